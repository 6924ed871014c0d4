"""What a program that answers requests behind documents kept on the GPU has the
kernel seam do: a causal sibling of the built-in model runs a document or an
instruction once, keeps its keys and values, and runs every request's own tokens
behind them, down to one token at a time, with weights of 4 bits.

Kinds of case (the key "kind"):
  write      new tokens' keys and values into a cache of 8 bits (or of the
             type itself), and back out of it.
  read       kept rows out of the cache.
  attention  queries of a batch whose sequences share long prefixes, over the
             prefix and each sequence's own tokens, all in the cache.
  products   a few rows times a matrix of 4-bit weights with group scales.

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


def listed():
    return [
        # One new token of one request of the built-in model's shape, behind a document.
        _attention("attention-1x1-f32", "f32", 3, 1, 256, 0, 1, 1, 1, 8, [1536]),
        # One new token of each of 64 requests behind one long instruction.
        _attention("attention-64-tokens-bf16-int8", "bf16", 32, 8, 128, 8, 64, 1, 1, 512, [8192]),
        # The same of four requests behind a whole book.
        _attention("attention-4-long-bf16-int8", "bf16", 32, 8, 128, 8, 4, 1, 16, 64, [131072]),
        # Passages of two documents, each read behind its own, windowed.
        _attention("attention-40-passages-f32-window", "f32", 3, 1, 256, 0, 40, 100, 400, 400, [2048, 1111], window=512),
        # Candidates scored behind a long shared context.
        _attention("attention-32x512-bf16", "bf16", 32, 8, 128, 0, 32, 512, 512, 512, [8192]),
        # One step's new keys and values of 64 requests.
        _rows("write-64-tokens-bf16", "write", "bf16", 8, 128, 8, 64, 1, 1),
        # The throughput batch's.
        _rows("write-64x512-f32", "write", "f32", 1, 256, 8, 64, 512, 512),
        # A short instruction's rows, to be kept elsewhere.
        _rows("read-100-f16", "read", "f16", 1, 256, 8, 1, 100, 100),
        # A book's.
        _rows("read-131072-bf16", "read", "bf16", 8, 128, 8, 1, 131072, 131072),
        # One token through the built-in model's gate and up projections.
        _products("products-1x768-f32", "f32", 1, 768, 2304, 32, False),
        # One token through a wide model's square projection.
        _products("products-1x8192-f16", "f16", 1, 8192, 8192, 32, False),
        # One token of each of 16 requests through a wide up-projection.
        _products("products-16x4096-bf16", "bf16", 16, 4096, 16384, 128, True),
    ]


def _attention(name, dtype, heads, kv_heads, hd, bits, n, lo, hi, past, prefixes, window=0, cap=0.0, causal=True):
    """n sequences of lo .. hi new tokens; past: a sequence's keys are up to so many (its new tokens' at least)."""
    return {"name": name, "kind": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "hd": hd,
            "bits": bits, "n": n, "lo": lo, "hi": hi, "past": past, "prefixes": ",".join(map(str, prefixes)),
            "window": window, "cap": cap, "causal": causal}


def _rows(name, kind, dtype, kv_heads, hd, bits, n, lo, hi):
    return {"name": name, "kind": kind, "dtype": dtype, "kv_heads": kv_heads, "hd": hd, "bits": bits, "n": n, "lo": lo,
            "hi": hi}


def _products(name, dtype, rows, k, cols, group, zeros):
    return {"name": name, "kind": "products", "dtype": dtype, "rows": rows, "in": k, "out": cols, "group": group,
            "zeros": zeros}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    pick = rng.random()
    dtype = rng.choice(("f32", "f16", "bf16"))
    hd = rng.choice((64, 128, 256, 8 * rng.randint(4, 31)))
    kv_heads = rng.choice((1, 1, 2, 4, 8))
    bits = rng.choice((0, 8))
    if pick < 0.5:
        heads = kv_heads * rng.randint(1, 8)
        prefixes = [_log_int(rng, 1, 65536) for _ in range(rng.choice((1, 1, 2, 3)))]
        lo = _log_int(rng, 1, 512)
        hi = lo * rng.randint(1, 2)
        if rng.random() < 0.4:
            lo = hi = 1
        most = 5 * 10**11 // (heads * hd * (max(prefixes) + hi + 400))  # rows
        n = min(512, _log_int(rng, 1, max(1, min(most, 16000) // hi)))
        c = _attention("", dtype, heads, kv_heads, hd, bits, n, lo, hi, hi + _log_int(rng, 1, 400), prefixes,
                       window=_log_int(rng, 16, 4096) if rng.random() < 0.25 else 0,
                       cap=rng.choice((0.0, 0.0, 20.0, 50.0)), causal=rng.random() < 0.8)
    elif pick < 0.75:
        lo = _log_int(rng, 1, 1024)
        hi = lo * rng.randint(1, 2)
        n = _log_int(rng, 1, max(1, 30000 // hi))
        c = _rows("", rng.choice(("write", "read")), dtype, kv_heads, hd, bits, n, lo, hi)
    else:
        group = rng.choice((32, 64, 128))
        k = group * _log_int(rng, 256 // group, 8192 // group)
        c = _products("", dtype, _log_int(rng, 1, 64), k, _log_int(rng, 128, 16384), group, rng.random() < 0.5)
    del c["name"]
    return c


# ---- the batch --------------------------------------------------------------


def _prefixes(case):
    return [int(p) for p in case["prefixes"].split(",")]


def _lengths(case):
    """The sequences' new tokens: those of the case, whatever the seed."""
    return np.random.RandomState(case["n"] * 131 + case["lo"]).randint(case["lo"], case["hi"] + 1, case["n"])


def _keys(case):
    """The sequences' own keys, the new tokens' among them."""
    lens = _lengths(case)
    r = np.random.RandomState(case["n"] + case["past"])
    return np.array([r.randint(m, max(m, case["past"]) + 1) for m in lens.tolist()])


def _offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def _shared(case):
    """Sequences of each prefix, as offsets: about as many for each."""
    count = len(_prefixes(case))
    return np.array([case["n"] * p // count for p in range(count + 1)], np.int32)


def _slots(lens):
    """Ranges of slots one after another, an odd gap between them; and the slots in all."""
    starts = np.cumsum(np.concatenate([[0], np.asarray(lens[:-1]) + 5])).astype(np.int32)
    return starts, int(starts[-1] + lens[-1])


@functools.lru_cache(maxsize=None)
def _kernels():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-semantica_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from semantica_gpu import Context, kernels
    return Context(0), kernels


def _gpu(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _most(x):
    return torch.full((), 127.0, dtype=torch.float64, device=x.device)


def _quantize(x, heads):
    """Rows of each head as codes of -127 .. 127 and a scale."""
    x = x.reshape(x.shape[0], heads, -1)
    # (A quotient in 64 bits: a float32 tensor over a number is its product with a rounded reciprocal.)
    scale = (x.double().abs().amax(-1, keepdim=True) / _most(x)).float().clamp_min(2.0 ** -126)
    return torch.round(x.double() / scale.double()).clamp_(-127, 127).to(torch.int8), scale


def _kept(case, k, v):
    """What the cache holds, in plain tensors: the values, or codes and scales of each head."""
    if case["bits"] == 0:
        return {"k": k, "v": v}
    (kc, ks), (vc, vs) = _quantize(k, case["kv_heads"]), _quantize(v, case["kv_heads"])
    return {"k": kc, "ks": ks, "v": vc, "vs": vs}


def _drawn(case, seed):
    """The dense inputs: x, codes, scales and zeros of products, or q (attention's), k and v."""
    g = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))
    t = DTYPES[case["dtype"]]

    def normal(*shape, by=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * by

    if case["kind"] == "products":
        k, cols, groups = case["in"], case["out"], case["in"] // case["group"]
        codes = torch.randint(0, 256, (cols, k // 2), generator=g, device="cuda", dtype=torch.uint8)
        scales = ((0.5 + torch.rand(cols, groups, generator=g, device="cuda")) * (k ** -0.5 / 4)).half()
        zeros = torch.randint(4, 12, (cols, groups), generator=g, device="cuda", dtype=torch.uint8)
        return normal(case["rows"], k).to(t), codes, scales, zeros if case["zeros"] else None
    kv_heads, hd = case["kv_heads"], case["hd"]
    rows = int(_lengths(case).sum())
    if case["kind"] != "attention":
        k, v = normal(rows, kv_heads * hd, by=2.0), normal(rows, kv_heads * hd, by=3.0)
        k[:, ::97] *= 8  # channels much larger than the rest
        return None, k.to(t), v.to(t)
    _, slots = _slots(_prefixes(case) + _keys(case).tolist())
    # Normed and rotated queries and keys, scores with a deviation of two; values as a projection gives them.
    unit = torch.nn.functional.normalize
    q = unit(normal(rows, case["heads"], hd), dim=-1) * hd ** 0.5
    k = unit(normal(slots, kv_heads, hd), dim=-1) * (2.0 * hd ** 0.5)
    return q.reshape(rows, -1).to(t), k.reshape(slots, -1).to(t), normal(slots, kv_heads * hd, by=3.0).to(t)


def prepare(case, seed):
    st, t = {"case": case}, DTYPES[case["dtype"]]
    if case["kind"] == "products":
        st["x"], st["codes"], st["scales"], st["zeros"] = _drawn(case, seed)
        if own:  # laid out once, as a program keeps it
            ctx, kernels = _kernels()
            st["weight"] = kernels.Q4Weight(ctx, st["codes"], st["scales"], st["zeros"])
            st["dst"] = torch.empty(case["rows"], case["out"], dtype=t, device="cuda")
        return st
    q, k, v = _drawn(case, seed)
    lens = _lengths(case)
    if case["kind"] != "attention":
        starts, slots = _slots(lens)
        st.update(off=_gpu(_offsets(lens)), starts=_gpu(starts), slots=slots)
        if own:
            ctx, kernels = _kernels()
            st["cache"] = kernels.KVCache(ctx, slots, case["kv_heads"], case["hd"], t, bits=case["bits"])
            st["k_out"], st["v_out"] = torch.empty_like(k), torch.empty_like(v)
        if case["kind"] == "write":
            return dict(st, k=k, v=v)
        if own:
            kernels.kv_cache_write(ctx, st["cache"], k, v, st["off"], st["starts"])
            return st
        at = _row_slots(st, k.shape[0])
        return dict(st, kept={n: torch.zeros((slots,) + x.shape[1:], dtype=x.dtype, device="cuda").index_copy_(0, at, x)
                              for n, x in _kept(case, k, v).items()})
    keys, prefixes = _keys(case), _prefixes(case)
    starts, slots = _slots(prefixes + keys.tolist())
    st.update(q=q, off=_gpu(_offsets(lens)), starts=_gpu(starts[len(prefixes):]), lengths=_gpu(keys.astype(np.int32)),
              shared=_gpu(_shared(case)), prefix_starts=_gpu(starts[:len(prefixes)]),
              prefix_lengths=_gpu(np.asarray(prefixes, np.int32)))
    if own:
        ctx, kernels = _kernels()
        st["cache"] = kernels.KVCache(ctx, slots, case["kv_heads"], case["hd"], t, bits=case["bits"])
        kernels.kv_cache_write(ctx, st["cache"], k, v, _gpu(np.array([0, slots], np.int32)), _gpu(np.zeros(1, np.int32)))
        st["out"] = torch.empty_like(q)
        return st
    return dict(st, kept=_kept(case, k, v), keys=keys, lens=lens, places=starts)


# ---- the operators in plain form --------------------------------------------


def _row_slots(st, rows):
    """The slot of each row."""
    off = st["off"].long()
    r = torch.arange(rows, device="cuda")
    i = torch.searchsorted(off[1:], r, right=True)
    return st["starts"].long()[i] + r - off[i]


def _values(kept, name, at):
    """Rows `at` of what is kept, in 32 bits: [rows, kv_heads * hd]."""
    x = kept[name][at].float()
    if name + "s" in kept:
        x = (x * kept[name + "s"][at]).reshape(x.shape[0], -1)
    return x


def _write_plain(st):
    case, t = st["case"], st["k"].dtype
    at = _row_slots(st, st["k"].shape[0])
    cache = {n: torch.zeros((st["slots"],) + x.shape[1:], dtype=x.dtype, device="cuda").index_copy_(0, at, x)
             for n, x in _kept(case, st["k"], st["v"]).items()}
    return {"k": _values(cache, "k", at).to(t), "v": _values(cache, "v", at).to(t)}


def _read_plain(st):
    t = DTYPES[st["case"]["dtype"]]
    at = _row_slots(st, int(_lengths(st["case"]).sum()))
    return {"k": _values(st["kept"], "k", at).to(t), "v": _values(st["kept"], "v", at).to(t)}


def _attention_plain(st):
    case = st["case"]
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["hd"]
    group, n = heads // kv_heads, case["n"]
    prefixes, shared, off = _prefixes(case), _shared(case), _offsets(st["lens"])
    out = torch.empty_like(st["q"])

    def scores(q, k):
        s = torch.matmul(q, k).mul_(hd ** -0.5)
        return torch.tanh_(s.div_(case["cap"])).mul_(case["cap"]) if case["cap"] else s

    for p, plen in enumerate(prefixes):
        k = _values(st["kept"], "k", slice(st["places"][p], st["places"][p] + plen)).reshape(plen, kv_heads, hd)
        v = _values(st["kept"], "v", slice(st["places"][p], st["places"][p] + plen)).reshape(plen, kv_heads, hd)
        k, v = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
        # Some sequences at a time, so that their scores fit.
        step = max(1, 2 * 10**9 // (4 * heads * case["hi"] * (plen + case["past"])))
        for a in range(shared[p], shared[p + 1], step):
            b = min(shared[p + 1], a + step)
            lens, keys = st["lens"][a:b], st["keys"][a:b]
            m, lq, lk = b - a, int(lens.max()), int(keys.max())
            qpos, kpos = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
            lens, keys = _gpu(lens), _gpu(keys)
            there, has = qpos < lens[:, None], kpos < keys[:, None]
            at = torch.where(there, _gpu(off[a:b]).long()[:, None] + qpos, 0)
            slot = torch.where(has, st["starts"][a:b].long()[:, None] + kpos, 0).reshape(-1)
            q = st["q"].float().reshape(-1, kv_heads, group, hd)[at].permute(2, 0, 3, 1, 4).contiguous()
            ok = _values(st["kept"], "k", slot).reshape(m, lk, kv_heads, hd).permute(2, 0, 3, 1).contiguous()
            ov = _values(st["kept"], "v", slot).reshape(m, lk, kv_heads, hd).permute(2, 0, 1, 3).contiguous()
            # [kv_heads, m, group, lq, keys]: the prefix's, then the own
            s0 = scores(q.reshape(kv_heads, -1, hd), k).reshape(kv_heads, m, group, lq, plen)
            s1 = scores(q.reshape(kv_heads, m, group * lq, hd), ok).reshape(kv_heads, m, group, lq, lk)
            pos = (keys - lens)[:, None] + qpos  # a query's place among the own keys
            seen = has[:, None, :].expand(m, lq, lk)
            gap = pos[:, :, None] - kpos
            if case["causal"]:
                seen = seen & (gap >= 0)
            if case["window"]:
                seen = seen & (gap.abs() < case["window"])
                far = plen + pos[:, :, None] - torch.arange(plen, device="cuda") >= case["window"]
                s0 = s0.masked_fill_(far[None, :, None], float("-inf"))
            s1 = s1.masked_fill_(~seen[None, :, None], float("-inf"))
            top = torch.maximum(s0.amax(-1, keepdim=True), s1.amax(-1, keepdim=True))
            top = torch.where(top > float("-inf"), top, 0.0)
            s0, s1 = torch.exp_(s0.sub_(top)), torch.exp_(s1.sub_(top))
            total = s0.sum(-1, keepdim=True) + s1.sum(-1, keepdim=True)
            o = torch.matmul(s0.reshape(kv_heads, -1, plen), v).reshape(kv_heads, m, group, lq, hd)
            o = o + torch.matmul(s1.reshape(kv_heads, m, -1, lk), ov).reshape(kv_heads, m, group, lq, hd)
            o = (o / torch.where(total > 0, total, 1.0)).permute(1, 3, 0, 2, 4)
            out[int(off[a]):int(off[b])] = o[there].reshape(-1, heads * hd).to(out.dtype)
    return out


def _products_plain(st):
    codes, scales, cols = st["codes"], st["scales"].float(), st["case"]["out"]
    w = torch.stack([codes & 15, codes >> 4], -1).reshape(cols, scales.shape[1], -1).float()
    w = (w - (st["zeros"].float()[..., None] if st["zeros"] is not None else 8.0)) * scales[..., None]
    return torch.matmul(st["x"].float(), w.reshape(cols, -1).t()).to(st["x"].dtype)


def run(st):
    case = st["case"]
    if not own:
        return {"write": _write_plain, "read": _read_plain, "attention": _attention_plain,
                "products": _products_plain}[case["kind"]](st)
    ctx, kernels = _kernels()
    if case["kind"] == "products":
        kernels.matmul_q4(ctx, st["dst"], st["weight"], st["x"])
        return st["dst"]
    if case["kind"] == "attention":
        kernels.attention_shared(ctx, st["out"], st["q"], st["cache"], case["heads"], st["off"], st["starts"],
                                 st["lengths"], st["shared"], st["prefix_starts"], st["prefix_lengths"],
                                 softcap=case["cap"], causal=case["causal"], window=case["window"])
        return st["out"]
    if case["kind"] == "write":
        kernels.kv_cache_write(ctx, st["cache"], st["k"], st["v"], st["off"], st["starts"])
    kernels.kv_cache_read(ctx, st["k_out"], st["v_out"], st["cache"], st["off"], st["starts"])
    return {"k": st["k_out"], "v": st["v_out"]}


# ---- what a pass cannot do without -------------------------------------------


def _pairs(case):
    """Visible (query, key) pairs of one head."""
    total, shared = 0, _shared(case)
    for p, plen in enumerate(_prefixes(case)):
        for i in range(shared[p], shared[p + 1]):
            m, keys = int(_lengths(case)[i]), int(_keys(case)[i])
            pos = plen + keys - m + np.arange(m)
            high = pos + 1 if case["causal"] else np.full(m, plen + keys)
            low = np.zeros(m, np.int64)
            if case["window"]:
                low, high = np.maximum(low, pos - case["window"] + 1), np.minimum(high, pos + case["window"])
            total += int(np.maximum(high - low, 0).sum())
    return total


def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "products":
        rows, k, cols, groups = case["rows"], case["in"], case["out"], case["in"] // case["group"]
        return {"bytes": size * rows * (k + cols) + cols * (k // 2 + groups * (3 if case["zeros"] else 2)),
                "flops": 2.0 * rows * k * cols}
    row = 2 * case["kv_heads"] * (case["hd"] * (1 if case["bits"] else size) + (4 if case["bits"] else 0))  # kept
    rows = int(_lengths(case).sum())
    if case["kind"] == "attention":
        # Every key that some query sees, once; queries and outputs.
        slots = int(_keys(case).sum())
        for p in _prefixes(case):
            slots += min(p, case["window"] + int(_keys(case).max())) if case["window"] else p
        return {"bytes": slots * row + 2 * size * rows * case["heads"] * case["hd"],
                "flops": 4.0 * case["hd"] * case["heads"] * _pairs(case)}
    values = 2 * case["kv_heads"] * case["hd"]
    passes = 2 if case["kind"] == "write" else 1
    return {"bytes": rows * (passes * (row + size * values)), "flops": 2.0 * passes * rows * values}


# ---- the definitions in 64 bits -----------------------------------------------


def _stored(case, x):
    """The values that the cache stands for, [rows, kv_heads, hd]."""
    x = x.double().reshape(x.shape[0], case["kv_heads"], case["hd"])
    if case["bits"] == 0:
        return x
    # The scale is a float32: 127th of the largest magnitude, no subnormal.
    scale = torch.clamp((x.abs().max(-1)[0] / _most(x)).float().double(), min=2.0 ** -126)[..., None]
    return torch.clamp(torch.round(x / scale), -127, 127) * scale


def _exact_attention(case, seed):
    q, k, v = _drawn(case, seed)
    k, v, hd, heads = _stored(case, k), _stored(case, v), case["hd"], case["heads"]
    q = q.reshape(q.shape[0], heads, hd)
    prefixes, shared, off = _prefixes(case), _shared(case).tolist(), _offsets(_lengths(case)).tolist()
    keys = _keys(case).tolist()
    places, _ = _slots(prefixes + keys)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for p, plen in enumerate(prefixes):
        for i in range(shared[p], shared[p + 1]):
            at = torch.cat([torch.arange(places[p], places[p] + plen),
                            torch.arange(places[len(prefixes) + i], places[len(prefixes) + i] + keys[i])]).cuda()
            there = torch.arange(plen + keys[i], device="cuda")
            mine = plen + keys[i] - (off[i + 1] - off[i]) + torch.arange(off[i + 1] - off[i], device="cuda")
            gap = mine[:, None] - there[None, :]
            hide = torch.zeros_like(gap, dtype=torch.bool)
            if case["causal"]:
                hide |= gap < 0
            if case["window"]:
                hide |= gap.abs() >= case["window"]
            for j in range(case["kv_heads"]):
                group = heads // case["kv_heads"]
                some = slice(j * group, (j + 1) * group)
                kt, vj = k[at, j].t().contiguous(), v[at, j]
                z = q[off[i]:off[i + 1], some].double().transpose(0, 1).reshape(-1, hd) @ kt / math.sqrt(hd)
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                z = z.reshape(group, -1, z.shape[-1]).masked_fill(hide, -float("inf"))
                w = torch.softmax(z, -1).nan_to_num(0.0)
                out[off[i]:off[i + 1], some] = (w.reshape(-1, w.shape[-1]) @ vj).reshape(group, -1, hd).transpose(0, 1)
    return out.reshape(out.shape[0], -1)


def exact(case, seed):
    if case["kind"] == "attention":
        # About 10^13 operations and a pass over the scores a second; a few hundred calls a sequence and head.
        return _exact_attention(case, seed) if case["n"] * case["kv_heads"] < 4000 else None
    if case["kind"] in ("write", "read"):
        _, k, v = _drawn(case, seed)
        return {n: _stored(case, x).reshape(x.shape) for n, x in (("k", k), ("v", v))}
    x, codes, scales, zeros = _drawn(case, seed)
    w = torch.empty(case["out"], case["in"], dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = codes % 16, torch.div(codes, 16, rounding_mode="floor")
    w -= 8.0 if zeros is None else torch.repeat_interleave(zeros.double(), case["group"], 1)
    w *= torch.repeat_interleave(scales.double(), case["group"], 1)
    return x.double() @ w.t().contiguous()
