"""What a program that embeds text with its own layers has the kernel seam do:
the operators that a sibling of the built-in model, or a fine-tuned one, needs
beside the Q8_0 products.

Kinds of case (the key "kind"):
  attention  attention over packed sequences whose scores are capped by a tanh,
             biased by distance, or masked (causal, prefix, window, documents).
  norm       a block's post-norm, its gate and residual scale, the residual
             addition and the next block's pre-norm.
  adapters   low-rank adapters of many requests added to a shared projection's
             output, each sequence with its own adapter or none.

`run` computes them in plain torch operations, or, where `own` is true, by the
package's kernels.  exact() restates each from its definition in 64 bits.
"""
import functools
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def listed():
    return [
        # One short query through a windowed layer of the built-in model's shape.
        _attention("attention-1x32-f32", "f32", 3, 1, 256, 1, 32, 32, window=512),
        # A handful of queries, scores capped.
        _attention("attention-13-queries-f32", "f32", 3, 1, 256, 13, 5, 60, cap=50.0),
        # The throughput batch of documents, windowed.
        _attention("attention-64x512-f32", "f32", 3, 1, 256, 64, 512, 512, window=256),
        # Long documents behind an instruction that every token sees.
        _attention("attention-8-long-f16-prefix", "f16", 16, 8, 128, 8, 1024, 2048, causal=True, prefix=96),
        # Whole files through a causal model with capped scores.
        _attention("attention-4x4096-bf16-capped", "bf16", 32, 8, 128, 4, 4096, 4096, cap=50.0, causal=True),
        # Many documents packed into one row of an odd length, distance bias, padding behind them.
        _attention("attention-16391-docs-bf16", "bf16", 12, 12, 64, 1, 16391, 16391, alibi=True, docs=900),
        # One short query's residual step.
        _norm("norm-32x768-f32", "f32", 32, 768, 1, "sequence"),
        # The throughput batch's, a gate for each request.
        _norm("norm-32768x768-f32", "f32", 32768, 768, 64, "sequence"),
        # A wide model's, layer-scaled, an odd number of rows.
        _norm("norm-20001x5120-bf16", "bf16", 20001, 5120, 9, "shared"),
        # One new token of each of 64 requests, nearly all with adapters of their own.
        _adapters("adapters-64-single-bf16", "bf16", 4096, 4096, 16, 48, 64, 1, 1),
        # A mixed batch through the built-in model's Q|K|V projection, one adapter a task.
        _adapters("adapters-256-ragged-f32", "f32", 768, 1280, 16, 8, 256, 8, 512),
        # Documents through a wide up-projection, large ranks.
        _adapters("adapters-32x512-bf16", "bf16", 2048, 8192, 64, 12, 32, 512, 512),
    ]


def _attention(name, dtype, heads, kv_heads, hd, n, lo, hi, cap=0.0, causal=False, prefix=0, window=0, alibi=False,
               docs=0):
    return {"name": name, "kind": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "hd": hd, "n": n,
            "lo": lo, "hi": hi, "cap": cap, "causal": causal, "prefix": prefix, "window": window, "alibi": alibi,
            "docs": docs}


def _norm(name, dtype, rows, cols, n, gate):
    return {"name": name, "kind": "norm", "dtype": dtype, "rows": rows, "cols": cols, "n": n, "gate": gate}


def _adapters(name, dtype, k, cols, rank, count, n, lo, hi):
    return {"name": name, "kind": "adapters", "dtype": dtype, "in": k, "out": cols, "rank": rank, "count": count,
            "n": n, "lo": lo, "hi": hi}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    pick = rng.random()
    dtype = rng.choice(("f32", "f16", "bf16"))
    if pick < 0.5:
        hd = rng.choice((64, 128, 256, 8 * rng.randint(4, 31)))
        kv_heads = rng.choice((1, 1, 2, 4, 8))
        heads = kv_heads * rng.randint(1, 4)
        lo = _log_int(rng, 1, 2048)
        hi = min(4096, lo * rng.randint(1, 3))
        most = min(40000, 10**9 // (heads * hi))
        n = _log_int(rng, 1, max(1, most // hi))
        causal = rng.random() < 0.5
        c = _attention("", dtype, heads, kv_heads, hd, n, lo, hi,
                       cap=rng.choice((0.0, 0.0, 20.0, 50.0)), causal=causal,
                       prefix=_log_int(rng, 1, 256) if causal and rng.random() < 0.5 else 0,
                       window=_log_int(rng, 1, 1024) if rng.random() < 0.3 else 0,
                       alibi=rng.random() < 0.3, docs=_log_int(rng, 8, 1024) if rng.random() < 0.3 else 0)
    elif pick < 0.72:
        rows = _log_int(rng, 1, 30000)
        cols = rng.choice((768, 1152, rng.randint(1, 1024), 8 * rng.randint(16, 640)))
        c = _norm("", dtype, rows, cols, rng.randint(1, min(rows, 100)), rng.choice(("none", "shared", "sequence")))
    else:
        k, cols = 8 * _log_int(rng, 16, 512), 8 * _log_int(rng, 16, 1024)
        lo = _log_int(rng, 1, 512)
        hi = lo * rng.randint(1, 2)
        c = _adapters("", dtype, k, cols, _log_int(rng, 4, 64), _log_int(rng, 1, 32), _log_int(rng, 1, max(1, 16000 // hi)),
                      lo, hi)
    del c["name"]
    return c


# ---- the batch --------------------------------------------------------------


def _lengths(case):
    """The sequences' lengths: those of the case, whatever the seed."""
    r = np.random.RandomState(case["n"] * 131 + case["lo"])
    if case["hi"] > 16 * case["lo"]:  # a mixed batch
        return np.exp(r.uniform(math.log(case["lo"]), math.log(case["hi"]), case["n"])).astype(np.int64)
    return r.randint(case["lo"], case["hi"] + 1, case["n"]).astype(np.int64)


def _cuts(rows, n):
    """`rows` rows as n sequences of different lengths, one row at least each."""
    r = np.random.RandomState(rows)
    inner = np.sort(r.permutation(rows - 1)[: n - 1] + 1) if n > 1 else np.zeros(0, np.int64)
    return np.diff(np.concatenate([[0], inner, [rows]])).astype(np.int64)


def _offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def _docs(case, rows):
    """Documents of about case["docs"] tokens one after another; a thirtieth of the rows is padding."""
    r = np.random.RandomState(case["docs"])
    used, ids, at = rows - rows // 30, np.full(rows, -1, np.int32), 0
    k = 0
    while at < used:
        m = int(r.randint(1, 2 * case["docs"]))
        ids[at:min(used, at + m)] = k
        at, k = at + m, k + 1
    return ids


def _slopes(heads):
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


def _chosen(case):
    """Each sequence's adapter; a tenth of them has none."""
    r = np.random.RandomState(case["count"] + case["n"])
    return np.where(r.uniform(size=case["n"]) < 0.1, -1, r.randint(0, case["count"], case["n"])).astype(np.int32)


@functools.lru_cache(maxsize=None)
def _kernels():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-semantica_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from semantica_gpu import Context, kernels
    return Context(0), kernels


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))
    t = DTYPES[case["dtype"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * by).to(t)

    if case["kind"] == "attention":
        lens = _lengths(case)
        off, hd = _offsets(lens), case["hd"]
        rows = int(off[-1])
        # Normed and rotated queries and keys; values as a projection gives them.
        unit = torch.nn.functional.normalize
        q = unit(torch.randn(rows, case["heads"], hd, generator=g, device="cuda"), dim=-1) * hd ** 0.5
        k = unit(torch.randn(rows, case["kv_heads"], hd, generator=g, device="cuda"), dim=-1) * hd ** 0.5
        k = k * 2.0  # scores with a deviation of two
        return {"case": case, "longest": int(lens.max()), "off": torch.from_numpy(off).cuda(),
                "q": q.reshape(rows, -1).to(t), "k": k.reshape(rows, -1).to(t),
                "v": normal(rows, case["kv_heads"] * hd, by=3.0),
                "slopes": torch.tensor(_slopes(case["heads"]), device="cuda") if case["alibi"] else None,
                "docs": torch.from_numpy(_docs(case, rows)).cuda() if case["docs"] else None,
                "prefix": torch.full((case["n"],), case["prefix"], dtype=torch.int32, device="cuda")
                if case["prefix"] else None,
                "out": torch.empty(rows, case["heads"] * hd, dtype=t, device="cuda")}
    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        gates = {"none": 0, "shared": 1, "sequence": case["n"]}[case["gate"]]
        # A residual stream some columns of which are much larger than the rest.
        h = torch.randn(rows, cols, generator=g, device="cuda")
        h[:, ::97] *= 8.0
        return {"case": case, "off": torch.from_numpy(_offsets(_cuts(rows, case["n"]))).cuda(), "h": h.to(t),
                "x": normal(rows, cols, by=2.0),
                "post": 1.0 + 0.2 * torch.randn(cols, generator=g, device="cuda"),
                "pre": 1.0 + 0.2 * torch.randn(cols, generator=g, device="cuda"),
                "gate": 0.5 + 0.3 * torch.randn(gates, cols, generator=g, device="cuda") if gates else None,
                "xn": torch.empty(rows, cols, dtype=t, device="cuda"),
                "sum": torch.empty(rows, cols, dtype=t, device="cuda")}
    off = _offsets(_lengths(case))
    rows, r = int(off[-1]), case["rank"]
    st = {"case": case, "off": torch.from_numpy(off).cuda(), "chosen": torch.from_numpy(_chosen(case)).cuda(),
          "x": normal(rows, case["in"]), "base": normal(rows, case["out"]),
          "a": normal(case["count"], r, case["in"], by=case["in"] ** -0.5),
          "b": normal(case["count"], case["out"], r, by=r ** -0.5),
          "scales": 0.5 + torch.rand(case["count"], generator=g, device="cuda"),
          "dst": torch.empty(rows, case["out"], dtype=t, device="cuda")}
    if own:  # laid out once, as a program keeps it
        ctx, kernels = _kernels()
        st["bank"] = kernels.AdapterBank(ctx, st["a"], st["b"], st["scales"])
    return st


# ---- the operators in plain form --------------------------------------------


def _row_sequence(off, rows):
    """The sequence of each row."""
    return torch.searchsorted(off[1:].long(), torch.arange(rows, device=off.device), right=True)


def _attention_plain(st):
    case = st["case"]
    heads, kv_heads, hd, longest = case["heads"], case["kv_heads"], case["hd"], st["longest"]
    rows, group = st["q"].shape[0], case["heads"] // case["kv_heads"]
    off = st["off"].long()
    n = off.shape[0] - 1
    pos = torch.arange(longest, device="cuda")
    there = pos < (off[1:] - off[:-1])[:, None]  # [n, longest]
    at = torch.where(there, off[:-1, None] + pos, 0)
    # [n, kv_heads, group, longest, hd] and [n, kv_heads, longest, hd]
    q = st["q"].float().reshape(rows, kv_heads, group, hd)[at].permute(0, 2, 3, 1, 4).contiguous()
    k = st["k"].float().reshape(rows, kv_heads, hd)[at].permute(0, 2, 3, 1).contiguous()
    v = st["v"].float().reshape(rows, kv_heads, hd)[at].permute(0, 2, 1, 3).contiguous()
    s = torch.matmul(q.reshape(n, kv_heads, group * longest, hd), k).mul_(hd ** -0.5)
    if case["cap"]:
        s = torch.tanh_(s.div_(case["cap"])).mul_(case["cap"])
    s = s.reshape(n, kv_heads, group, longest, longest)
    far = (pos[:, None] - pos[None, :])  # query - key
    if case["alibi"]:
        s -= st["slopes"].reshape(kv_heads, group, 1, 1) * far.abs()
    seen = there[:, :, None] & there[:, None, :]
    if case["causal"]:
        back = far >= 0
        if case["prefix"]:
            back = back | (pos < st["prefix"][:, None])[:, None, :]
        seen = seen & back
    if case["window"]:
        seen = seen & (far.abs() < case["window"])
    if case["docs"]:
        d = st["docs"][at]
        seen = seen & (d[:, :, None] == d[:, None, :]) & (d >= 0)[:, :, None]
    seen = seen[:, None, None]
    s = s.masked_fill_(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = torch.exp_(s.sub_(torch.where(top > float("-inf"), top, 0.0)))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.reshape(n, kv_heads, group * longest, longest), v)
    o = o.reshape(n, kv_heads, group, longest, hd) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4)[there].reshape(rows, heads * hd).to(st["out"].dtype)


def _norm_plain(st):
    def rms(v, w):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * w

    y = rms(st["x"].float(), st["post"])
    if st["case"]["gate"] == "shared":
        y = y * st["gate"]
    elif st["case"]["gate"] == "sequence":
        y = y * st["gate"][_row_sequence(st["off"], y.shape[0])]
    h = st["h"].float() + 0.5 * y
    return {"xn": rms(h, st["pre"]).to(st["xn"].dtype), "sum": h.to(st["xn"].dtype)}


def _adapters_plain(st):
    a, b, x = st["a"].float(), st["b"].float(), st["x"].float()
    count, r, k = a.shape
    mine = st["chosen"][_row_sequence(st["off"], x.shape[0])]
    # Every adapter's low-rank rows at once; each row keeps those of its own.
    u = torch.matmul(x, a.reshape(count * r, k).t()).reshape(-1, count, r) * st["scales"][:, None]
    u = torch.where((mine[:, None] == torch.arange(count, device="cuda"))[:, :, None], u, 0.0)
    delta = torch.matmul(u.reshape(-1, count * r), b.permute(0, 2, 1).reshape(count * r, -1))
    return (st["base"].float() + delta).to(st["dst"].dtype)


def run(st):
    case = st["case"]
    if not own:
        return {"attention": _attention_plain, "norm": _norm_plain, "adapters": _adapters_plain}[case["kind"]](st)
    ctx, kernels = _kernels()
    if case["kind"] == "attention":
        kernels.attention_masked(ctx, st["out"], st["q"], st["k"], st["v"], case["heads"], case["kv_heads"], st["off"],
                                 softcap=case["cap"], slopes=st["slopes"], doc_ids=st["docs"], causal=case["causal"],
                                 prefix=st["prefix"], window=case["window"])
        return st["out"]
    if case["kind"] == "norm":
        gates = {"gate": st["gate"], "offsets": st["off"] if case["gate"] == "sequence" else None}
        kernels.block_norm(ctx, st["xn"], st["sum"], st["x"], st["h"], st["post"], st["pre"], EPS, scale=0.5, **gates)
        return {"xn": st["xn"], "sum": st["sum"]}
    kernels.adapters_apply(ctx, st["dst"], st["base"], st["bank"], st["x"], st["off"], st["chosen"])
    return st["dst"]


# ---- what a pass cannot do without -------------------------------------------


def _pairs(case):
    """Visible (query, key) pairs of one head."""
    total = 0
    lens = _lengths(case)
    ids = _docs(case, int(lens.sum())) if case["docs"] else None
    first = 0
    for s in (int(v) for v in lens):
        i = np.arange(s)
        low, high = np.zeros(s, np.int64), np.full(s, s)
        if case["causal"]:
            high = np.minimum(s, np.maximum(i + 1, case["prefix"]))
        if case["window"]:
            low, high = np.maximum(low, i - case["window"] + 1), np.minimum(high, i + case["window"])
        if ids is not None:  # documents lie one after another
            d = ids[first:first + s]
            low = np.maximum(low, np.searchsorted(np.where(d < 0, 1 << 30, d), d, "left"))
            high = np.minimum(high, np.searchsorted(np.where(d < 0, 1 << 30, d), d, "right"))
            high = np.where(d < 0, low, high)
        total += int(np.maximum(high - low, 0).sum())
        first += s
    return total


def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "attention":
        rows = int(_lengths(case).sum())
        return {"bytes": size * rows * case["hd"] * 2 * (case["heads"] + case["kv_heads"]),
                "flops": 4.0 * case["hd"] * case["heads"] * _pairs(case)}
    if case["kind"] == "norm":
        return {"bytes": 4 * size * case["rows"] * case["cols"], "flops": 12.0 * case["rows"] * case["cols"]}
    lens, mine = _lengths(case), _chosen(case)
    rows, active, used = int(lens.sum()), int(lens[mine >= 0].sum()), len(set(mine[mine >= 0].tolist()))
    both = case["in"] + case["out"]
    return {"bytes": size * (rows * (both + case["out"]) + used * case["rank"] * both),
            "flops": 2.0 * active * case["rank"] * both + rows * case["out"]}


# ---- the definitions in 64 bits -----------------------------------------------


def _exact_attention(case, st):
    hd, group = case["hd"], case["heads"] // case["kv_heads"]
    q, k, v = (st[n].double() for n in ("q", "k", "v"))
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    off = st["off"].tolist()
    for i in range(case["n"]):
        a, b = off[i], off[i + 1]
        place = torch.arange(a, b, device="cuda")
        for r0 in range(a, b, 4096):
            r1 = min(b, r0 + 4096)
            gap = place[r0 - a:r1 - a, None] - place[None, :]
            hide = torch.zeros_like(gap, dtype=torch.bool)
            if case["causal"]:
                hide |= (gap < 0) & (place - a >= case["prefix"])
            if case["window"]:
                hide |= gap.abs() >= case["window"]
            if case["docs"]:
                hide |= st["docs"][r0:r1, None] != st["docs"][a:b]
                hide |= st["docs"][r0:r1, None] < 0
            for h in range(case["heads"]):
                mine, theirs = slice(h * hd, (h + 1) * hd), slice(h // group * hd, (h // group + 1) * hd)
                z = q[r0:r1, mine] @ k[a:b, theirs].t().contiguous() / math.sqrt(hd)
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                if case["alibi"]:
                    z = z - st["slopes"][h].double() * gap.abs()
                z = torch.softmax(z.masked_fill(hide, -float("inf")), -1).nan_to_num(0.0)
                out[r0:r1, mine] = z @ v[a:b, theirs]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(case, st)
    if case["kind"] == "norm":
        x, h, lens = st["x"].double(), st["h"].double(), _cuts(case["rows"], case["n"])
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["cols"] + EPS) * st["post"].double()
        if case["gate"] != "none":
            gate = st["gate"].double()
            y = y * (gate if case["gate"] == "shared" else torch.repeat_interleave(gate, torch.from_numpy(lens).cuda(), 0))
        h = h + y / 2
        return {"xn": h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["cols"] + EPS) * st["pre"].double(), "sum": h}
    out, off = st["base"].double(), st["off"].tolist()
    for i, c in enumerate(_chosen(case).tolist()):
        if c >= 0:
            u = st["x"][off[i]:off[i + 1]].double() @ st["a"][c].double().t().contiguous()
            out[off[i]:off[i + 1]] += float(st["scales"][c]) * (u @ st["b"][c].double().t().contiguous())
    return out
