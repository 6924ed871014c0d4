"""sg_attention_masked, sg_block_norm and sg_adapters_apply against their
definitions in 64 bits, and what they refuse.

Tolerances, element by element, count roundings.  u(T) is half a step of the
output's type; f = 2^-24 half a step of float32, in which every sum is formed.
"""
import ctypes
import math
import sys

import numpy as np
import pytest

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -24, "bf16": 2.0 ** -126}  # the types' own floor
F = 2.0 ** -24


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def dt(name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rand(g, *shape, by=1.0, dtype="f32"):
    return (torch.randn(*shape, generator=g) * by).to(dt(dtype))


def offsets(lens, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(lens)]).astype(np.int32))


def close(got, want, tol, what):
    got = got.double().cpu()
    err = (got - want).abs()
    ok = (err <= tol) | (got == want) | (torch.isnan(got) & torch.isnan(want))
    worst = (err / tol.clamp_min(1e-300)).nan_to_num(math.inf)[~ok]
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} off, up to {float(worst.max()):.3g} tolerances"


# ---- attention -----------------------------------------------------------------


def attention_ref(q, k, v, off, heads, kv_heads, scale=0.0, softcap=0.0, slopes=None, doc_ids=None, causal=False,
                  prefix=None, window=0):
    """The definition in 64 bits, and the mean of |v| and the scores' size that the tolerance needs.
    Rows of no sequence are NaN."""
    rows, hd = q.shape[0], q.shape[1] // heads
    q, k, v = (t.double().reshape(rows, -1, hd) for t in (q, k, v))
    scale = scale or 1.0 / math.sqrt(hd)
    out = torch.full((rows, heads, hd), math.nan, dtype=torch.float64)
    mean, size = torch.zeros(rows, heads, hd, dtype=torch.float64), torch.zeros(rows, heads, 1, dtype=torch.float64)
    off = off.tolist()
    for i, (a, b) in enumerate(zip(off[:-1], off[1:])):
        if a == b:
            continue
        at = torch.arange(b - a)
        gap = (at[:, None] - at[None, :]).abs()
        seen = torch.ones(b - a, b - a, dtype=torch.bool)
        if causal:
            seen &= (at[None, :] <= at[:, None]) | (at[None, :] < (int(prefix[i]) if prefix is not None else 0))
        if window:
            seen &= gap < window
        if doc_ids is not None:
            d = doc_ids[a:b]
            seen &= (d[:, None] == d[None, :]) & (d[:, None] >= 0)
        for h in range(heads):
            kh, vh = k[a:b, h * kv_heads // heads], v[a:b, h * kv_heads // heads]
            # Hidden keys' contents do not count, so they are zeros here.
            s = torch.einsum("id,jd->ij", q[a:b, h], kh.clone().nan_to_num(0, 0, 0))
            big = torch.einsum("id,jd->ij", q[a:b, h].abs(), kh.abs().nan_to_num(0, 0, 0)) * scale
            s = s * scale
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - slopes[h].double() * gap
                big = big + slopes[h].double() * gap * seen
            s = s.masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            vz = vh.nan_to_num(0, 0, 0)
            out[a:b, h] = p @ vz
            mean[a:b, h] = p @ vz.abs()
            size[a:b, h, 0] = (big * (p > 2.0 ** -40)).amax(-1)
    return out.reshape(rows, -1), mean.reshape(rows, -1), size.expand(rows, heads, hd).reshape(rows, -1)


def attention_tol(dtype, hd, out, mean, size, softcap=0.0):
    # A score: hd products and sums of float32 (float32 operands as two fp16 halves:
    # 2^-21 of each product for the dropped terms) and some ten roundings behind it;
    # an error of d in a score is one of 2 d in a weight relative to the sum.
    products = (hd + 16) * F + (2.0 ** -21 if dtype == "f32" else 0.0)
    score = products * size + 16 * F * (size + 1) + softcap * 2.0 ** -22
    # The weights' rounding to the type, the values' halves, the sums over the keys.
    weights = {"f32": 2.0 ** -20, "f16": U["f16"], "bf16": U["bf16"]}[dtype] + 2048 * F
    # 16-bit weights are summed as they are multiplied, p_j (1 + d_j) with |d_j| <= u, so the
    # result is off by sum_j p_j d_j (v_j - o) / sum_j p_j (1 + d_j), at most
    # u (mean |v| + |o|) / (1 - u): the sum's own share is the u |o|.
    total = 0.0 if dtype == "f32" else U[dtype] * (1 + 2 * U[dtype])
    return (U[dtype] + total) * out.abs() + (2 * score + weights * (1 + 2 * U[dtype])) * mean + TINY[dtype]


def run_attention(ctx, q, k, v, off, heads, kv_heads, fill=7.0, **kw):
    from semantica_gpu import kernels
    dev = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in kw.items()}
    out = torch.full(q.shape, fill, dtype=q.dtype, device="cuda")
    kernels.attention_masked(ctx, out, q.cuda(), k.cuda(), v.cuda(), heads, kv_heads, off.cuda(), **dev)
    return out.cpu()


def check_attention(ctx, seed, dtype, heads, kv_heads, hd, lens, first=0, behind=0, by=1.0, **kw):
    g = gen(seed)
    off = offsets(lens, first)
    rows = int(off[-1]) + behind
    q, k = rand(g, rows, heads * hd, by=by, dtype=dtype), rand(g, rows, kv_heads * hd, dtype=dtype)
    v = rand(g, rows, kv_heads * hd, by=2.0, dtype=dtype)
    say("attention", dtype, "heads", heads, kv_heads, "hd", hd, "lens", list(lens)[:8], "rows", rows, sorted(kw))
    got = run_attention(ctx, q, k, v, off, heads, kv_heads, **kw)
    want, mean, size = attention_ref(q, k, v, off, heads, kv_heads, **kw)
    there = torch.zeros(rows, dtype=torch.bool)
    there[first:int(off[-1])] = True
    assert bool((got[~there] == 7.0).all()), "rows of no sequence were written"
    close(got[there], want[there], attention_tol(dtype, hd, want, mean, size, kw.get("softcap", 0.0))[there], "attention")


MASKS = {
    "plain": {},
    "scale": {"scale": 0.31},
    "cap": {"softcap": 5.0},
    "causal": {"causal": True},
    "window": {"window": 9},
    "causal-window": {"causal": True, "window": 1},
}


def mask_of(name, heads, lens, first, behind):
    if name in MASKS:
        return dict(MASKS[name])
    rows = first + int(np.sum(lens)) + behind
    r = np.random.RandomState(rows)
    if name == "slopes":
        return {"slopes": torch.tensor([2.0 ** -(h + 1) for h in range(heads)], dtype=torch.float32)}
    if name == "prefix":
        return {"causal": True, "prefix": torch.tensor(r.randint(0, 40, len(lens)).astype(np.int32))}
    if name == "documents":  # one after another, some padding
        return {"doc_ids": torch.tensor(np.where(r.uniform(size=rows) < 0.1, -1, np.arange(rows) // 11).astype(np.int32))}
    if name == "mixed-documents":  # in no order, some rows see themselves alone, some nothing
        return {"doc_ids": torch.tensor(r.randint(-1, 4, rows).astype(np.int32)), "causal": True}
    assert name == "all"
    return {"doc_ids": torch.tensor((np.arange(rows) // 29).astype(np.int32)), "causal": True, "window": 20,
            "prefix": torch.tensor(r.randint(0, 9, len(lens)).astype(np.int32)), "softcap": 3.0,
            "slopes": torch.tensor([0.3 / (h + 1) for h in range(heads)], dtype=torch.float32)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mask", ["plain", "scale", "cap", "causal", "window", "causal-window", "slopes", "prefix",
                                  "documents", "mixed-documents", "all"])
def test_attention_masks(gpu_ctx, dtype, mask):
    """Few rows (the waves share them and split the keys): every mask, at the dims of each LDS layout."""
    for hd, heads, kv_heads in ((64, 4, 2), (128, 3, 1), (256, 3, 1)):
        lens = [1, 0, 5, 33, 0, 64, 131]
        check_attention(gpu_ctx, hd, dtype, heads, kv_heads, hd, lens, first=3, behind=4,
                        **mask_of(mask, heads, lens, 3, 4))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("mask", ["plain", "causal", "all", "mixed-documents"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_many_rows(gpu_ctx, dtype, mask, hd):
    """Rows enough for the form whose waves hold 32 rows each."""
    heads, kv_heads = 24, 8
    lens = [700, 1, 0, 257, 31, 32, 33] + [60] * 25 + [3] * 100
    check_attention(gpu_ctx, hd + 1, dtype, heads, kv_heads, hd, lens, first=1, behind=2,
                    **mask_of(mask, heads, lens, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [8, 40, 72, 136, 200, 248])
def test_attention_odd_head_dims(gpu_ctx, dtype, hd):
    check_attention(gpu_ctx, hd, dtype, 2, 1, hd, [17, 40, 1], causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attention_long_sequence(gpu_ctx, dtype):
    """Many tiles, running maxima that rise late, documents that end inside tiles and far apart."""
    lens = [3001]
    check_attention(gpu_ctx, 5, dtype, 2, 1, 64, lens, by=4.0)
    ids = torch.tensor((np.arange(3001) // 700).astype(np.int32))
    ids[:40] = 4  # the last document's other half, 2800 keys away
    check_attention(gpu_ctx, 6, dtype, 2, 1, 128, lens, doc_ids=ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_reads_slices_of_one_projection(gpu_ctx, dtype):
    """q, k and v as columns of one fused tensor, out as columns of a wider one."""
    from semantica_gpu import kernels
    heads, kv_heads, hd, off = 3, 1, 64, offsets([50, 13])
    g = gen(4)
    qkv = rand(g, 63, (heads + 2 * kv_heads) * hd + 8, dtype=dtype).cuda()
    wide = torch.full((63, heads * hd + 16), 7.0, dtype=dt(dtype), device="cuda")
    q, k, v = qkv[:, :192], qkv[:, 192:256], qkv[:, 256:320]
    kernels.attention_masked(gpu_ctx, wide[:, 8:200], q, k, v, heads, kv_heads, off.cuda(), causal=True)
    want, mean, size = attention_ref(q.cpu(), k.cpu(), v.cpu(), off, heads, kv_heads, causal=True)
    close(wide[:, 8:200], want, attention_tol(dtype, hd, want, mean, size), "attention")
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 200:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_attention_ignores_hidden_contents(gpu_ctx, dtype, hd, bad):
    """Infinities and NaN in keys and values that a query does not see leave its output alone:
    the next sequence's, a padding token's, a later key's."""
    heads, kv_heads, lens = 2, 1, [40, 70, 20]
    g, off = gen(8), offsets([40, 70, 20])
    q, k, v = (rand(g, 130, c * hd, dtype=dtype) for c in (heads, kv_heads, kv_heads))
    ids = torch.zeros(130, dtype=torch.int32)
    ids[60:63] = -1
    hide = [60, 61, 62, 109]  # padding, and the last key of the second sequence
    k[hide, :5], v[hide, 3:] = bad, bad
    kw = {"doc_ids": ids, "causal": True}
    got = run_attention(gpu_ctx, q, k, v, off, heads, kv_heads, **kw)
    want, mean, size = attention_ref(q, k, v, off, heads, kv_heads, **kw)
    fine = torch.ones(130, dtype=torch.bool)
    fine[109] = False  # it sees itself
    close(got[fine], want[fine], attention_tol(dtype, hd, want, mean, size)[fine], "attention")
    assert bool((got[60:63] == 0).all()), "padding comes out as zeros"
    if math.isnan(bad):
        assert bool(torch.isnan(got[109]).all())


@pytest.mark.gpu
def test_attention_visible_infinity_reaches_its_columns_alone(gpu_ctx):
    """An infinite value that is seen is in its own column of the queries that see it."""
    for dtype in ("f32", "bf16"):
        g, off = gen(9), offsets([33, 20])
        q, k, v = (rand(g, 53, 64, dtype=dtype) for _ in range(3))
        v[10, 7] = math.inf
        got = run_attention(gpu_ctx, q, k, v, off, 1, 1, causal=True).double()
        v0 = v.clone()
        v0[10, 7] = 0
        want, mean, size = attention_ref(q, k, v0, off, 1, 1, causal=True)
        tol = attention_tol(dtype, 64, want, mean, size)
        assert bool((got[10:33, 7] == math.inf).all())
        got[10:33, 7] = want[10:33, 7]
        close(got, want, tol, "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("qs,ks,vs", [(1e-20, 1e20, 1.0), (1e25, 1e-25, 1e-30), (1.0, 1.0, 1e-6), (1.0, 1.0, 1e12),
                                      (1.0, 1.0, 1e30), (1e30, 1e-30, 1.0)])
def test_attention_float32_range(gpu_ctx, hd, qs, ks, vs):
    """float32 operands far outside fp16's range, and values whose rows differ by many powers of ten."""
    g, off = gen(10), offsets([45, 90])
    q, k, v = rand(g, 135, hd) * qs, rand(g, 135, hd) * ks, rand(g, 135, hd) * vs
    v[::3] *= 1e-5
    v[1::7] = 0
    k[5] = 0
    got = run_attention(gpu_ctx, q, k, v, off, 1, 1, window=60)
    want, mean, size = attention_ref(q, k, v, off, 1, 1, window=60)
    close(got, want, attention_tol("f32", hd, want, mean, size), "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_large_scores(gpu_ctx, dtype):
    """Scores in the hundreds: one key takes all, and nothing overflows."""
    g, off = gen(11), offsets([64, 100])
    q, k, v = rand(g, 164, 128, by=40.0, dtype=dtype), rand(g, 164, 128, dtype=dtype), rand(g, 164, 128, dtype=dtype)
    for kw in ({}, {"slopes": torch.tensor([50.0])}):
        got = run_attention(gpu_ctx, q, k, v, off, 1, 1, **kw)
        want, mean, size = attention_ref(q, k, v, off, 1, 1, **kw)
        close(got, want, attention_tol(dtype, 128, want, mean, size), "attention")


# ---- norms ----------------------------------------------------------------------


def norm_ref(x, h, post, pre, eps, gate, scale, seq):
    x, h = x.double(), h.double()
    y = x
    if post is not None:
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * post.double()
    if gate is not None:
        y = y * (gate.double()[seq] if seq is not None else gate.double())
    y = scale * y
    s = h + y
    if pre is None:
        return s, None, h.abs() + y.abs(), None
    inv = torch.rsqrt((s * s).mean(-1, keepdim=True) + eps)
    return s, s * inv * pre.double(), h.abs() + y.abs(), (h.abs() + y.abs()) * inv * pre.double().abs()


def check_norm(ctx, dtype, rows, cols, lens=None, first=0, gate=False, post=True, pre=True, pad=0, in_place=False, seed=0):
    from semantica_gpu import kernels
    g = gen(seed + rows + cols)
    say("norm", dtype, rows, cols, "lens", lens, "gate", gate, post, pre, "pad", pad, in_place)

    def rowsof(t):  # rows of a wider tensor: strides and alignment of their own
        w = torch.full((rows, cols + pad), 7.0, dtype=t.dtype, device="cuda")
        w[:, pad // 2:pad // 2 + cols] = t.cuda()
        return w[:, pad // 2:pad // 2 + cols]

    x, h = rand(g, rows, cols, by=3.0, dtype=dtype), rand(g, rows, cols, dtype=dtype)
    wp, wn = (1 + 0.1 * torch.randn(cols, generator=g) for _ in range(2))
    off = offsets(lens, first) if lens is not None else None
    there = torch.ones(rows, dtype=torch.bool)
    seq = None
    if off is not None:
        there[:] = False
        there[first:int(off[-1])] = True
        seq = torch.zeros(rows, dtype=torch.long)
        seq[there] = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    gt = torch.randn(*((len(lens), cols) if off is not None else (cols,)), generator=g) if gate else None
    xd, hd_ = rowsof(x), rowsof(h)
    sum_ = hd_ if in_place else rowsof(torch.full((rows, cols), 7.0, dtype=dt(dtype)))
    xn = (xd if in_place else rowsof(torch.full((rows, cols), 7.0, dtype=dt(dtype)))) if pre else None
    kernels.block_norm(ctx, xn, sum_, xd, hd_, wp.cuda() if post else None, wn.cuda() if pre else None, 1e-6,
                       gate=gt.cuda() if gate else None, scale=0.25, offsets=off.cuda() if off is not None else None)
    s, n, size, nsize = norm_ref(x, h, wp if post else None, wn if pre else None, 1e-6, gt, 0.25, seq)
    # The mean of cols squares: cols roundings at most, half of that in its root; ten more behind it.
    rel = (cols / 2 + 10) * F
    tiny = TINY[dtype]
    close(sum_.cpu()[there], s[there], (U[dtype] * s.abs() + rel * size + tiny)[there], "sum")
    if pre:
        close(xn.cpu()[there], n[there], (U[dtype] * n.abs() + 2 * rel * nsize + tiny)[there], "xn")
    if off is not None and not in_place:
        assert bool((sum_.cpu()[~there] == 7).all()), "rows of no sequence were written"
        assert xn is None or bool((xn.cpu()[~there] == 7).all())
    if pad:
        base = sum_._base
        assert bool((base[:, :pad // 2] == 7).all()) and bool((base[:, pad // 2 + cols:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cols", [1, 3, 8, 64, 100, 255, 256, 768, 1152, 1000, 2048, 2056, 2047, 4096, 5120, 6008, 8192, 8191])
def test_norm_columns(gpu_ctx, dtype, cols):
    check_norm(gpu_ctx, dtype, 5, cols, lens=[2, 0, 1, 1], first=1, gate=True)
    check_norm(gpu_ctx, dtype, 3, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kw", [{"gate": True}, {"post": False}, {"pre": False}, {"post": False, "pre": False, "gate": True},
                                {"pad": 16}, {"pad": 6}, {"in_place": True}, {"in_place": True, "pad": 6}])
@pytest.mark.parametrize("rows,cols", [(1, 768), (37, 768), (9000, 96), (700, 2500)])
def test_norm_forms(gpu_ctx, dtype, kw, rows, cols):
    check_norm(gpu_ctx, dtype, rows, cols, **kw)
    if rows > 30:
        check_norm(gpu_ctx, dtype, rows, cols, lens=[1, 0, 0, 7, rows - 15, 3], first=2, **kw)


@pytest.mark.gpu
def test_norm_many_sequences_and_bad_rows(gpu_ctx):
    """A gate for each of thousands of sequences; a row that is not finite stays alone."""
    from semantica_gpu import kernels
    check_norm(gpu_ctx, "f32", 9001, 100, lens=[0, 1, 0] * 3000, first=1, gate=True)
    x, h = torch.randn(50, 768, device="cuda"), torch.randn(50, 768, device="cuda")
    w = torch.ones(768, device="cuda")
    outs = []
    for bad in (False, True):
        if bad:
            x[7, 3], h[9, 1] = math.nan, math.inf
        xn, s = torch.empty_like(x), torch.empty_like(x)
        kernels.block_norm(gpu_ctx, xn, s, x, h, w, w, 1e-6)
        outs.append((xn.cpu(), s.cpu()))
    rest = [i for i in range(50) if i not in (7, 9)]
    for a, b in zip(*outs):
        assert torch.equal(a[rest], b[rest])
    assert bool(torch.isnan(outs[1][0][7]).all())


# ---- adapters --------------------------------------------------------------------


def adapters_ref(x, base, a, b, scales, off, ids):
    out, size = base.double().clone(), base.double().abs()
    off = off.tolist()
    for i, c in enumerate(ids.tolist()):
        s = slice(off[i], off[i + 1])
        if 0 <= c < a.shape[0]:
            u = x[s].double() @ a[c].double().T
            out[s] += float(scales[c]) * (u @ b[c].double().T)
            size[s] += abs(float(scales[c])) * (x[s].double().abs() @ a[c].double().abs().T @ b[c].double().abs().T)
    return out, size


def adapter_case(dtype, k, n, rank, count, lens, first=0, behind=0, seed=0, by=1.0):
    g = gen(seed + k + n)
    off = offsets(lens, first)
    rows = int(off[-1]) + behind
    ids = torch.tensor(np.random.RandomState(rows).randint(-1, count + 1, len(lens)).astype(np.int32))  # count: no adapter
    return {"x": rand(g, rows, k, dtype=dtype, by=by), "base": rand(g, rows, n, dtype=dtype),
            "a": rand(g, count, rank, k, by=k ** -0.5, dtype=dtype), "b": rand(g, count, n, rank, dtype=dtype),
            "scales": torch.rand(count, generator=g) * 2 - 0.5, "off": off, "ids": ids}


def run_adapters(ctx, c, in_place=False):
    from semantica_gpu import kernels
    bank = kernels.AdapterBank(ctx, c["a"].cuda(), c["b"].cuda(), c["scales"].cuda())
    base = c["base"].cuda()
    dst = base if in_place else torch.full_like(base, 7.0)
    kernels.adapters_apply(ctx, dst, base, bank, c["x"].cuda(), c["off"].cuda(), c["ids"].cuda())
    got = dst.cpu()
    bank.close()
    return got


def check_adapters(ctx, dtype, k, n, rank, count, lens, first=0, behind=0, in_place=False, **kw):
    say("adapters", dtype, k, n, "rank", rank, "count", count, "lens", list(lens)[:8])
    c = adapter_case(dtype, k, n, rank, count, lens, first, behind, **kw)
    got = run_adapters(ctx, c, in_place)
    want, size = adapters_ref(c["x"], c["base"], c["a"], c["b"], c["scales"], c["off"], c["ids"])
    there = torch.zeros(got.shape[0], dtype=torch.bool)
    there[first:int(c["off"][-1])] = True
    # k + rank roundings of float32 at most, and (16-bit types) u as two halves: 2^-17 of it.
    rel = (k + rank + 32) * F + (0 if dtype == "f32" else 2.0 ** -16)
    close(got[there], want[there], (U[dtype] * want.abs() + rel * size + TINY[dtype])[there], "adapters")
    if not in_place:
        assert bool((got[~there] == 7).all()), "rows of no sequence were written"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [1, 4, 16, 17, 32, 64, 100, 256])
def test_adapters_ranks(gpu_ctx, dtype, rank):
    check_adapters(gpu_ctx, dtype, 768, 1280, rank, 5, [3, 0, 1, 40, 1, 17], first=2, behind=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k,n", [(8, 8), (40, 24), (136, 1000), (4096, 264), (776, 4104)])
def test_adapters_dims(gpu_ctx, dtype, k, n):
    check_adapters(gpu_ctx, dtype, k, n, 16, 3, [20, 5], in_place=True)
    check_adapters(gpu_ctx, dtype, k, n, 24, 40, [1] * 70, behind=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rank", [16, 48, 64, 128])
def test_adapters_many_rows(gpu_ctx, dtype, rank):
    """Rows enough for workgroups of two and of four row tiles."""
    check_adapters(gpu_ctx, dtype, 136, 200, rank, 9, [700, 1, 2, 3] + [97] * 80)
    check_adapters(gpu_ctx, dtype, 64, 72, rank, 9, [5] * 3500, first=7, behind=9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [7, 20, 48])
def test_adapters_many_short_sequences(gpu_ctx, dtype, rank):
    """Several adapters in every 16 rows, more than a workgroup takes at a time."""
    check_adapters(gpu_ctx, dtype, 1000, 72, rank, 9, [3] * 4000 + [0, 1, 2] * 20, first=1, behind=2)


@pytest.mark.gpu
def test_adapters_keep_to_their_rows(gpu_ctx):
    """One request's NaN, in its input or in its adapter, stays with it."""
    for dtype in ("f32", "f16"):
        c = adapter_case(dtype, 96, 80, 8, 4, [1] * 16)
        c["ids"] = torch.tensor([0, 1, 2, 3] * 4, dtype=torch.int32)
        clean = run_adapters(gpu_ctx, c)
        c["a"][1, 0, 3], c["b"][2, 5, 1], c["x"][4, 9] = math.nan, math.inf, math.nan
        got = run_adapters(gpu_ctx, c)
        rest = [i for i in range(16) if i % 4 not in (1, 2) and i != 4]
        assert torch.equal(got[rest], clean[rest])
        assert bool(torch.isnan(got[4]).all()) and bool(torch.isnan(got[1::4]).all())


@pytest.mark.gpu
def test_adapters_keep_to_their_rows_in_large_batches(gpu_ctx):
    """The same where a workgroup multiplies several adapters together."""
    for dtype in ("f32", "bf16"):
        c = adapter_case(dtype, 96, 80, 8, 6, [2] * 8000)
        c["ids"] = torch.arange(8000, dtype=torch.int32) % 6
        clean = run_adapters(gpu_ctx, c)
        c["a"][1, 0, 3], c["b"][2, 5, 1], c["x"][8, 9] = math.nan, math.inf, math.nan
        got = run_adapters(gpu_ctx, c)
        rest = torch.ones(16000, dtype=torch.bool)
        for i in (1, 2):
            rest[2 * i::12] = rest[2 * i + 1::12] = False
        rest[8] = False
        assert torch.equal(got[rest], clean[rest])
        assert bool(torch.isnan(got[8]).all()) and bool(torch.isnan(got[2::12]).all())


@pytest.mark.gpu
def test_adapters_large_values_in_fp16(gpu_ctx):
    """A low-rank value past fp16's range on the way to an output within it."""
    c = adapter_case("f16", 512, 64, 8, 2, [9, 9])
    c["ids"] = torch.tensor([0, 1], dtype=torch.int32)
    c["x"], c["a"] = c["x"] * 100, c["a"] * 500
    c["b"] = c["b"] * 2.0 ** -10
    c["a"][1] *= 2.0 ** -9
    got = run_adapters(gpu_ctx, c)
    want, size = adapters_ref(c["x"], c["base"], c["a"], c["b"], c["scales"], c["off"], c["ids"])
    close(got, want, U["f16"] * want.abs() + (600 * F + 2.0 ** -16) * size + TINY["f16"], "adapters")


# ---- what else may be in the tensors, and how else they may be called --------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("big", [1e4, 1e30])
def test_attention_ignores_large_hidden_contents(gpu_ctx, dtype, hd, big):
    """Finite values far above a query's own in what it does not see: padding first in its
    sequence, and later keys that grow."""
    if dtype == "f16" and big > 6e4:
        pytest.skip("past the type's range")
    for rows in (90, 2000):
        g, off = gen(21), offsets([rows])
        q, k, v = (rand(g, rows, c * hd, dtype=dtype) for c in (6, 2, 2))
        ids = torch.zeros(rows, dtype=torch.int32)
        ids[:33] = -1
        k[:33], v[:33] = big, -big
        k[70], v[70, ::2] = big, big
        v[80] = 0
        kw = {"doc_ids": ids, "causal": True}
        say("large hidden", dtype, hd, big, rows)
        got = run_attention(gpu_ctx, q, k, v, off, 6, 2, **kw)
        want, mean, size = attention_ref(q[:70], k[:70], v[:70], offsets([70]), 6, 2, doc_ids=ids[:70], causal=True)
        close(got[:70], want, attention_tol(dtype, hd, want, mean, size), "attention")
        assert bool((got[:33] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 256])
def test_attention_values_that_grow_and_fade(gpu_ctx, hd):
    """Causal float32 rows whose values rise, then fall, by tens of powers of ten."""
    g, off = gen(22), offsets([300, 300])
    q, k, v = rand(g, 600, hd), rand(g, 600, hd), rand(g, 600, hd)
    v[:300] *= (10.0 ** torch.linspace(-30, 30, 300))[:, None]
    v[300:] *= (10.0 ** torch.linspace(30, -30, 300))[:, None]
    for kw in ({"causal": True}, {"window": 3}):
        got = run_attention(gpu_ctx, q, k, v, off, 1, 1, **kw)
        want, mean, size = attention_ref(q, k, v, off, 1, 1, **kw)
        close(got, want, attention_tol("f32", hd, want, mean, size), "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [1e-3, 0.3, 50.0, 55.0, 60.0, 3e4, 1e6, 1e30])
def test_attention_caps_of_any_size(gpu_ctx, dtype, cap):
    """tanh from saturation to the identity, and queries whose scores all lie at the cap's
    lower end over values of any size."""
    g, off = gen(23), offsets([70, 40])
    q, k, v = rand(g, 110, 128, by=6.0, dtype=dtype), rand(g, 110, 128, dtype=dtype), rand(g, 110, 128, dtype=dtype)
    q[5], k[:70, :64] = -200.0, k[:70, :64].abs() + 1  # a row of the lowest scores
    for by in (1.0,) if dtype == "f16" else (1.0, 1e-20):
        vs = (v.float() * by).to(v.dtype)
        got = run_attention(gpu_ctx, q, k, vs, off, 2, 2, softcap=cap)
        want, mean, size = attention_ref(q, k, vs, off, 2, 2, softcap=cap)
        # (A score off by d ahead of the cap is off by d at most behind it.)
        close(got, want, attention_tol(dtype, 64, want, mean, size, min(cap, float(size.max()))), "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (16, 2), (24, 8)])
def test_attention_heads_dealt_over_the_xcds(gpu_ctx, dtype, heads, kv_heads):
    check_attention(gpu_ctx, 24, dtype, heads, kv_heads, 64, [3, 200, 131], causal=True)
    check_attention(gpu_ctx, 25, dtype, heads, kv_heads, 64, [1] * 40 + [700])


@pytest.mark.gpu
def test_attention_long_documents_scan(gpu_ctx):
    """More tiles than one look at the document ids covers, a document in two halves far apart."""
    rows, hd = 140001, 8
    g = gen(26)
    q, k, v = (rand(g, rows, hd, dtype="f16") for _ in range(3))
    ids = (torch.arange(rows) // 37 + 1).to(torch.int32)
    ids[:20] = 0
    ids[-21:] = 0
    got = run_attention(gpu_ctx, q, k, v, offsets([rows]), 1, 1, doc_ids=ids)
    for doc in (0, 1, 500, 1891, 3782, int(ids.max())):
        at = (ids == doc).nonzero()[:, 0]
        want, mean, size = attention_ref(q[at], k[at], v[at], offsets([len(at)]), 1, 1)
        close(got[at], want, attention_tol("f16", hd, want, mean, size), f"document {doc}")


def layer_calls(ctx, dtype="bf16", seed=0):
    """Each operator once, over buffers of its own: [(name, call(stream), inputs, outputs)]."""
    from semantica_gpu import kernels
    g, off = gen(seed), offsets([40, 0, 1, 90, 300], first=3)
    rows, offd = 440, offsets([40, 0, 1, 90, 300], first=3).cuda()
    assert int(off[-1]) <= rows
    t = lambda cols, by=1.0: rand(g, rows, cols, by=by, dtype=dtype).cuda()
    q, k, v, o = t(512), t(128), t(128), t(512)
    ids = torch.tensor([0, 1, -1, 2, 1], dtype=torch.int32).cuda()
    a, b = rand(g, 3, 16, 512, by=0.05, dtype=dtype).cuda(), rand(g, 3, 768, 16, dtype=dtype).cuda()
    bank = kernels.AdapterBank(ctx, a, b, torch.tensor([0.5, 1.0, 2.0]).cuda())
    base, dst = t(768), t(768)
    work = torch.empty(bank.work_bytes(rows), dtype=torch.uint8, device="cuda")
    x, h, s, n = t(768, 3.0), t(768), t(768), t(768)
    wp, wn, gate = (torch.randn(*z, generator=g).cuda() for z in ((768,), (768,), (5, 768)))
    slopes = torch.rand(4, generator=g).cuda()
    torch.cuda.synchronize()
    return [
        ("attention", lambda stream=None: kernels.attention_masked(ctx, o, q, k, v, 4, 1, offd, softcap=8.0, slopes=slopes,
                                                                   causal=True, stream=stream), [q, k, v], [o]),
        ("adapters", lambda stream=None: kernels.adapters_apply(ctx, dst, base, bank, q, offd, ids, work=work, stream=stream),
         [q, base], [dst]),
        ("norm", lambda stream=None: kernels.block_norm(ctx, n, s, x, h, wp, wn, 1e-6, gate=gate, offsets=offd, stream=stream),
         [x, h], [s, n])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_replayed_graphs_equal_eager_calls(gpu_ctx, dtype):
    """One graph of all three operators, replayed with new inputs, eager calls and
    synchronizations between; a second graph with its own workspace beside it."""
    sets = [layer_calls(gpu_ctx, dtype, seed) for seed in (1, 2)]
    graphs = []
    for calls in sets:
        for _, call, _, _ in calls:
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        say("capturing", dtype)
        with torch.cuda.graph(graph):
            for _, call, _, _ in calls:
                call()
        graphs.append(graph)
    for rep in range(4):
        for calls, graph in zip(sets, graphs):
            say("replay", rep)
            for _, _, ins, outs in calls:
                for t in ins:
                    t.copy_(torch.randn(t.shape, generator=gen(rep)).to(t.dtype))
                for t in outs:
                    t.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for _, _, _, outs in calls for t in outs]
            for _, call, _, outs in calls:
                for t in outs:
                    t.fill_(7.0)
                call()
            torch.cuda.synchronize()
            want = [t for _, _, _, outs in calls for t in outs]
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_from_two_threads_on_two_streams(gpu_ctx):
    """Two threads, each on a stream of its own with outputs and workspace of its own."""
    import threading
    sets = [layer_calls(gpu_ctx, "f32", 5), layer_calls(gpu_ctx, "bf16", 6)]
    alone = []
    for calls in sets:
        for _, call, _, _ in calls:
            call()
        torch.cuda.synchronize()
        alone.append([t.clone() for _, _, _, outs in calls for t in outs])
    streams = [torch.cuda.Stream() for _ in sets]
    wrong = []

    def work(i):
        try:
            for _ in range(20):
                for _, call, _, _ in sets[i]:
                    call(streams[i].cuda_stream)
            streams[i].synchronize()
        except Exception as e:  # pragma: no cover
            wrong.append(e)

    for calls in sets:
        for _, _, _, outs in calls:
            for t in outs:
                t[3:434] = 0
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for calls, want in zip(sets, alone):
        for a, b in zip([t for _, _, _, outs in calls for t in outs], want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_no_rows_and_empty_sequences(gpu_ctx, dtype):
    """No rows, no sequence with a row, and rows before and behind the only one."""
    from semantica_gpu import kernels
    check_attention(gpu_ctx, 31, dtype, 2, 1, 64, [0, 0, 0], first=2, behind=5)
    check_attention(gpu_ctx, 32, dtype, 2, 1, 64, [1], causal=True)
    check_attention(gpu_ctx, 33, dtype, 2, 1, 64, [0, 1, 0], first=1, behind=1, window=1)
    check_norm(gpu_ctx, dtype, 4, 768, lens=[0, 0], first=2, gate=True)
    check_adapters(gpu_ctx, dtype, 64, 64, 8, 2, [0, 0, 0], first=2, behind=5)
    none = torch.empty(0, 64, dtype=dt(dtype), device="cuda")
    off, ids = offsets([0, 0]).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda")
    kernels.attention_masked(gpu_ctx, none, none, none, none, 1, 1, off)
    kernels.block_norm(gpu_ctx, none, none, none, none, None, torch.ones(64, device="cuda"), 1e-6, offsets=off)
    bank = kernels.AdapterBank(gpu_ctx, torch.zeros(1, 8, 64, dtype=dt(dtype), device="cuda"),
                               torch.zeros(1, 64, 8, dtype=dt(dtype), device="cuda"), torch.ones(1, device="cuda"))
    kernels.adapters_apply(gpu_ctx, none, none, bank, none, off, ids)
    bank.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_single_row_of_a_wider_tensor(gpu_ctx, dtype):
    """A single row's stride does not matter, whatever the tensor that it is cut from."""
    from semantica_gpu import kernels
    wide = torch.randn(2, 203, device="cuda").to(dt(dtype))
    q = wide[:1, 8:136]
    out = torch.empty(1, 128, dtype=dt(dtype), device="cuda")
    kernels.attention_masked(gpu_ctx, out, q, q, q, 2, 2, offsets([1]).cuda())
    # One key, weight 1: its value.  float32 values are held as two halves of 11 bits, off by
    # 2^-11 of 2^-11 at most (2^-37 of the row's largest where the second is subnormal), and
    # the division and the scaling back are four roundings; 16-bit values pass unchanged.
    tol = 2.0 ** -21 * q.abs() + 2.0 ** -37 * q.abs().max() if dtype == "f32" else 0.0 * q.abs()
    close(out, q.double().cpu(), tol.double().cpu(), "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("off", [[5, 2, 9, 1], [-7, 400, 3, 1 << 30], [-(1 << 31), (1 << 31) - 1, 0, 64], [64, 64, 64, 64]])
def test_offsets_and_ids_that_make_no_sense(gpu_ctx, off):
    """Whatever device arrays hold, nothing outside the tensors is touched (every index
    that is formed from them is clamped)."""
    from semantica_gpu import kernels
    rows = 64
    wide = [torch.full((rows + 2, 144), 7.0, device="cuda") for _ in range(3)]
    o, s, n = (w[1:-1, 8:136] for w in wide)
    q = torch.randn(rows, 128, device="cuda")
    offd = torch.tensor(off, dtype=torch.int64).to(torch.int32).cuda()
    ids = torch.tensor([-9, 1 << 30, 3], dtype=torch.int32).cuda()
    docs = torch.randint(-(1 << 31), (1 << 31) - 1, (rows,), generator=gen(1)).to(torch.int32).cuda()
    say("offsets", off)
    kernels.attention_masked(gpu_ctx, o, q, q, q, 2, 2, offd, causal=True, prefix=ids, doc_ids=docs)
    torch.cuda.synchronize()
    kernels.block_norm(gpu_ctx, n, s, q, q, None, torch.ones(128, device="cuda"), 1e-6,
                       gate=torch.ones(3, 128, device="cuda"), offsets=offd)
    torch.cuda.synchronize()
    bank = kernels.AdapterBank(gpu_ctx, torch.ones(2, 8, 128, device="cuda"), torch.ones(2, 128, 8, device="cuda"),
                               torch.ones(2, device="cuda"))
    kernels.adapters_apply(gpu_ctx, o, q, bank, q, offd, ids)
    torch.cuda.synchronize()
    bank.close()
    for w in wide:
        assert bool((w[0] == 7).all()) and bool((w[-1] == 7).all())
        assert bool((w[:, :8] == 7).all()) and bool((w[:, 136:] == 7).all())


@pytest.mark.gpu
def test_rows_past_32_bits(gpu_ctx):
    """Rows that lie more than 2^32 bytes and 2^31 elements into their tensors."""
    from semantica_gpu import kernels
    rows, ld = 600, 1 << 22
    g, off = gen(41), offsets([rows])
    wide = torch.empty(rows, ld, dtype=torch.float16, device="cuda")
    cols = {n: rand(g, rows, 64, dtype="f16") for n in ("q", "k", "v", "h")}
    at = {n: wide[:, 64 * i:64 * i + 64] for i, n in enumerate(cols)}
    for n, t in cols.items():
        at[n].copy_(t.cuda())
    far = torch.empty(rows, ld, dtype=torch.float16, device="cuda")[:, 8:72]
    say("attention, strides of 2^22")
    kernels.attention_masked(gpu_ctx, far, at["q"], at["k"], at["v"], 1, 1, off.cuda())
    want, mean, size = attention_ref(cols["q"], cols["k"], cols["v"], off, 1, 1)
    close(far, want, attention_tol("f16", 64, want, mean, size), "attention")
    say("norm")
    w = torch.randn(64, generator=g)
    xn = torch.empty(rows, 64, dtype=torch.float16, device="cuda")
    kernels.block_norm(gpu_ctx, xn, far, at["q"], at["h"], w.cuda(), w.cuda(), 1e-6)
    s, n, ssize, nsize = norm_ref(cols["q"], cols["h"], w, w, 1e-6, None, 1.0, None)
    close(far, s, U["f16"] * s.abs() + 42 * F * ssize + TINY["f16"], "sum")
    close(xn, n, U["f16"] * n.abs() + 84 * F * nsize + TINY["f16"], "xn")
    say("adapters")
    a, b = rand(g, 2, 8, 64, by=0.1, dtype="f16"), rand(g, 2, 64, 8, dtype="f16")
    scales, ids = torch.tensor([0.5, 2.0]), torch.tensor([1], dtype=torch.int32)
    bank = kernels.AdapterBank(gpu_ctx, a.cuda(), b.cuda(), scales.cuda())
    kernels.adapters_apply(gpu_ctx, far, at["h"], bank, at["q"], off.cuda(), ids.cuda())
    want, size = adapters_ref(cols["q"], cols["h"], a, b, scales, off, ids)
    close(far, want, U["f16"] * want.abs() + (104 * F + 2.0 ** -16) * size + TINY["f16"], "adapters")
    bank.close()


@pytest.mark.gpu
def test_a_layer_with_adapters(gpu_ctx):
    """The operators as one layer uses them, around the Q8_0 products: queries and keys from
    shared weights with a low-rank change for each request, normed and rotated, masked attention,
    the output product with its own adapters, the residual step.  Each result is checked
    against its definition on what came before it."""
    from semantica_gpu import kernels, synth
    lens, hidden, heads, kv_heads, hd = [1, 37, 300, 2, 90], 768, 3, 1, 256
    g, rng = gen(51), np.random.default_rng(51)
    off, host_off = offsets(lens), np.concatenate([[0], np.cumsum(lens)])
    rows, offd = int(off[-1]), offsets(lens).cuda()
    x, h = rand(g, rows, hidden).cuda(), rand(g, rows, hidden).cuda()
    ids = torch.tensor([0, -1, 2, 1, 0], dtype=torch.int32)
    scales = torch.tensor([0.5, 1.0, 2.0])

    def product(t, n):
        """t @ w of Q8_0 weights, the shared part of a projection; and adapters for it."""
        k = t.shape[1]
        w = kernels.Q8Weight(gpu_ctx, synth.q8_0_random(rng, n, k), n, k)
        q = torch.empty(t.shape, dtype=torch.int8, device="cuda")
        scale, y = torch.empty(len(lens), device="cuda"), torch.empty(rows, n, device="cuda")
        kernels.quantize_symmetric_int8(gpu_ctx, t, host_off, q, scale)
        kernels.matmul_q8_0(gpu_ctx, y, w, q, scale.repeat_interleave(torch.tensor(lens, device="cuda")))
        shared = y.cpu()
        a, b = rand(g, 3, 16, k, by=k ** -0.5), rand(g, 3, n, 16)
        bank = kernels.AdapterBank(gpu_ctx, a.cuda(), b.cuda(), scales.cuda())
        kernels.adapters_apply(gpu_ctx, y, y, bank, t, offd, ids.cuda())
        want, size = adapters_ref(t.cpu(), shared, a, b, scales, off, ids)
        close(y, want, U["f32"] * want.abs() + (k + 48) * F * size + TINY["f32"], "adapters")
        bank.close()
        w.close()
        return y

    q, k, v = product(x, heads * hd), product(x, kv_heads * hd), product(x, kv_heads * hd)
    one = torch.ones(hd, device="cuda")
    kernels.qknorm_rope(gpu_ctx, q, k, one, one, heads, kv_heads, hd, 1e-6, 10000.0, 2048, host_off)
    o = torch.empty(rows, heads * hd, device="cuda")
    kw = {"softcap": 20.0, "causal": True, "window": 128}
    kernels.attention_masked(gpu_ctx, o, q, k, v, heads, kv_heads, offd, **kw)
    want, mean, size = attention_ref(q.cpu(), k.cpu(), v.cpu(), off, heads, kv_heads, **kw)
    close(o, want, attention_tol("f32", hd, want, mean, size, 20.0), "attention")
    y = product(o, hidden)
    wp, wn, gate = (torch.randn(*z, generator=g) for z in ((hidden,), (hidden,), (len(lens), hidden)))
    before, xn = h.cpu(), torch.empty_like(h)
    kernels.block_norm(gpu_ctx, xn, h, y, h, wp.cuda(), wn.cuda(), 1e-6, gate=gate.cuda(), offsets=offd)
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    s, n, ssize, nsize = norm_ref(y.cpu(), before, wp, wn, 1e-6, gate, 1.0, seq)
    rel = (hidden / 2 + 10) * F
    close(h, s, U["f32"] * s.abs() + rel * ssize, "sum")
    close(xn, n, U["f32"] * n.abs() + 2 * rel * nsize, "xn")


@pytest.mark.gpu
def test_adapters_work_refusals(gpu_ctx):
    from semantica_gpu import SemanticaError, kernels
    bank = kernels.AdapterBank(gpu_ctx, torch.zeros(1, 8, 64, device="cuda"), torch.zeros(1, 64, 8, device="cuda"),
                               torch.ones(1, device="cuda"))
    x, off, ids = torch.zeros(32, 64, device="cuda"), offsets([32]).cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    need = bank.work_bytes(32)
    dst, big = torch.zeros(32, 64, device="cuda"), torch.zeros(need + 64, dtype=torch.uint8, device="cuda")
    kernels.adapters_apply(gpu_ctx, dst, x, bank, x, off, ids, work=big[:need])
    inside = torch.zeros(32 * 64 + need, device="cuda")
    for work, to, word in ((big[:need - 1], dst, "bytes"), (big[8:], dst, "aligned"), (big[:0], dst, "bytes"),
                           (inside.view(torch.uint8), inside[:2048].view(32, 64), "work overlaps"), (big, x, "overlaps x")):
        with pytest.raises(SemanticaError, match=word):
            kernels.adapters_apply(gpu_ctx, to, dst if to is x else x, bank, x, off, ids, work=work)
    bank.close()
    with pytest.raises(SemanticaError, match="NULL"):
        kernels.adapters_apply(gpu_ctx, dst, x, bank, x, off, ids, work=big)


# ---- refusals (no device is touched) -----------------------------------------------


FAKE = ctypes.create_string_buffer(4096)


def _addr(at=0):
    base = (ctypes.addressof(FAKE) + 15) & ~15
    return ctypes.c_void_p(base + at)


def _refused(rc, word):
    from semantica_gpu import _lib
    assert rc == _lib.SG_ERR_INVALID
    assert word in _lib.load().sg_last_error().decode(), _lib.load().sg_last_error()


ATT = dict(out=1 << 40, ldo=256, q=2 << 40, ldq=256, k=3 << 40, ldk=128, v=4 << 40, ldv=128, dtype=1, heads=2, kv=1, hd=128,
           rows=10, off=5 << 40, n_seq=1)


@pytest.mark.parametrize("change,mask,word", [
    ({"out": None}, {}, "NULL"), ({"q": None}, {}, "NULL"), ({"dtype": 3}, {}, "element type"),
    ({"heads": 3, "kv": 2}, {}, "heads"), ({"heads": 0}, {}, "heads"), ({"kv": 0}, {}, "heads"), ({"hd": 12}, {}, "head_dim"),
    ({"hd": 264}, {}, "head_dim"), ({"hd": 0}, {}, "head_dim"), ({"rows": -1}, {}, "rows"), ({"off": None}, {}, "seq_offsets"),
    ({"n_seq": 0}, {}, "seq_offsets"), ({"n_seq": (1 << 30) + 1}, {}, "2^30"), ({"ldq": 255}, {}, "stride"), ({"ldk": 129}, {}, "aligned"), ({"v": (4 << 40) + 8}, {}, "aligned"),
    ({"ldo": 260}, {}, "aligned"), ({"out": 2 << 40}, {}, "overlaps"), ({"out": (3 << 40) - 16}, {}, "overlaps"),
    ({"ldk": (1 << 22) + 8}, {}, "2^22"), ({"ldq": 1 << 40}, {}, "stride"),
    ({}, {"scale": math.nan}, "scale"), ({}, {"softcap": -1.0}, "softcap"), ({}, {"softcap": math.inf}, "softcap"),
    ({}, {"window": -1}, "window"), ({}, {"prefix": 6 << 40}, "causal")])
def test_attention_refusals(change, mask, word):
    from semantica_gpu import _lib
    c = {**ATT, **change}
    m = _lib.AttnMask(**mask)
    _refused(_lib.load().sg_attention_masked(_addr(), c["out"], c["ldo"], c["q"], c["ldq"], c["k"], c["ldk"], c["v"], c["ldv"],
                                             c["dtype"], c["heads"], c["kv"], c["hd"], c["rows"], c["off"], c["n_seq"],
                                             ctypes.byref(m), None), word)


NORM = dict(xn=1 << 40, ldxn=64, sum=2 << 40, lds=64, x=3 << 40, ldx=64, h=4 << 40, ldh=64, dtype=0, rows=10, cols=64,
            post=5 << 40, pre=6 << 40, eps=1e-6, gate=None, scale=1.0, off=None, n_seq=0)


@pytest.mark.parametrize("change,word", [
    ({"sum": None}, "NULL"), ({"x": None}, "NULL"), ({"h": None}, "NULL"), ({"pre": None}, "w_pre"), ({"xn": None}, "xn"),
    ({"dtype": -1}, "element type"), ({"cols": 0}, "cols"), ({"cols": 8193}, "cols"), ({"rows": -1}, "rows"),
    ({"eps": -1.0}, "eps"), ({"eps": math.nan}, "eps"), ({"scale": math.inf}, "scale"), ({"n_seq": 1}, "n_seq"),
    ({"off": 7 << 40}, "seq_offsets"), ({"ldx": 63}, "stride"), ({"sum": 1 << 40}, "overlaps"),
    ({"sum": (4 << 40) + 4}, "overlaps"), ({"xn": 3 << 40, "ldxn": 65}, "overlaps"), ({"x": (3 << 40) + 2}, "aligned"),
    ({"dtype": 2, "h": (4 << 40) + 1}, "aligned")])
def test_norm_refusals(change, word):
    from semantica_gpu import _lib
    c = {**NORM, **change}
    _refused(_lib.load().sg_block_norm(_addr(), c["xn"], c["ldxn"], c["sum"], c["lds"], c["x"], c["ldx"], c["h"], c["ldh"],
                                       c["dtype"], c["rows"], c["cols"], c["post"], c["pre"], c["eps"], c["gate"], c["scale"],
                                       c["off"], c["n_seq"], None), word)


BANK = dict(a=1 << 40, b=2 << 40, scales=3 << 40, dtype=0, n=4, rank=8, k=64, out=64)


@pytest.mark.parametrize("change,word", [
    ({"a": None}, "NULL"), ({"scales": None}, "NULL"), ({"dtype": 7}, "element type"), ({"n": 0}, "n_adapters"),
    ({"rank": 0}, "rank"), ({"rank": 257}, "rank"), ({"k": 60}, "multiples of 8"), ({"out": 4}, "multiples of 8"),
    ({"out": 0}, "multiples of 8"), ({"n": 1 << 30, "rank": 256, "k": 1 << 16}, "too many"),
    ({"n": (1 << 31) - 1, "rank": 256, "k": 1 << 24, "out": 1 << 24}, "too many")])
def test_bank_refusals(change, word):
    from semantica_gpu import _lib
    c = {**BANK, **change}
    h = ctypes.c_void_p()
    _refused(_lib.load().sg_adapter_bank_create(_addr(), c["a"], c["b"], c["scales"], c["dtype"], c["n"], c["rank"], c["k"],
                                                c["out"], None, ctypes.byref(h)), word)
    assert not h.value


def test_adapters_null_arguments():
    from semantica_gpu import _lib
    lib = _lib.load()
    size = ctypes.c_size_t()
    _refused(lib.sg_adapters_work_bytes(None, 1, ctypes.byref(size)), "NULL")
    _refused(lib.sg_adapters_apply(_addr(), 1, 8, 1, 8, None, 1, 8, 1, 1, 1, 1, 1, 1, None), "NULL")
    lib.sg_adapter_bank_free(None)


def test_no_rows_need_no_tensors():
    from semantica_gpu import _lib
    lib = _lib.load()
    assert lib.sg_attention_masked(_addr(), None, 64, None, 64, None, 64, None, 64, 0, 1, 1, 64, 0, 1, 1, None, None) == 0
    assert lib.sg_block_norm(_addr(), None, 0, None, 64, None, 64, None, 64, 0, 0, 64, None, None, 1e-6, None, 1.0, None, 0,
                             None) == 0


class _Ctx:  # tensors in host memory count as this one's device, so that only the later checks refuse them
    device = -1

    def __init__(self):
        from semantica_gpu import _lib
        self.lib, self.handle = _lib.load(), _addr()


@pytest.mark.parametrize("change,word", [
    ({"q": (10, 130)}, "columns for 4 heads"), ({"k": (10, 16)}, "k: shape"), ({"v": (9, 32)}, "v: shape"),
    ({"out": (10, 136)}, "out: shape"), ({"k": "half"}, "k: torch.float16 beside"), ({"v": "turned"}, "contiguous"),
    ({"q": "long"}, "float32, float16 or bfloat16"), ({"slopes": (3,)}, "slopes: 4"), ({"doc_ids": (9,)}, "doc_ids"),
    ({"prefix": (2,)}, "prefix"), ({"offsets": "long"}, "offsets")])
def test_attention_wrapper_refusals(change, word):
    from semantica_gpu import kernels
    shapes = {"out": (10, 128), "q": (10, 128), "k": (10, 32), "v": (10, 32), "offsets": (2,)}
    kw = {}
    for n, to in {**shapes, **change}.items():
        t = torch.zeros(shapes.get(n, to) if isinstance(to, str) else to)
        if n in ("offsets", "doc_ids", "prefix"):
            t = t.to(torch.int32)
        if to == "half":
            t = t.half()
        if to == "long":
            t = t.long()
        if to == "turned":
            t = torch.zeros(t.shape[::-1]).t()
        kw[n] = t
    if change.get("q") == "long":
        for n in ("out", "k", "v"):
            kw[n] = kw[n].long()
    args = [kw.pop(n) for n in ("out", "q", "k", "v")]
    with pytest.raises(ValueError, match=word):
        kernels.attention_masked(_Ctx(), *args, 4, 1, kw.pop("offsets"), **kw)


def test_wrappers_refuse_other_devices_and_shapes():
    from semantica_gpu import kernels
    ctx, t, w = _Ctx(), torch.zeros(4, 64), torch.zeros(64)
    with pytest.raises(ValueError, match="w_post"):
        kernels.block_norm(ctx, None, t, t, t, torch.zeros(63), None, 1e-6)
    with pytest.raises(ValueError, match="gate"):
        kernels.block_norm(ctx, None, t, t, t, w, None, 1e-6, gate=w, offsets=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="h: shape"):
        kernels.block_norm(ctx, None, t, t, t[:3], w, None, 1e-6)
    with pytest.raises(ValueError, match="b: shape"):
        kernels.AdapterBank(ctx, torch.zeros(2, 8, 64), torch.zeros(2, 64, 4), torch.zeros(2))
    with pytest.raises(ValueError, match="scales"):
        kernels.AdapterBank(ctx, torch.zeros(2, 8, 64), torch.zeros(2, 64, 8), torch.zeros(3))
    ctx.device = 0
    with pytest.raises(ValueError, match="device"):
        kernels.block_norm(ctx, None, t, t, t, w, None, 1e-6)
    with pytest.raises(ValueError, match="device"):
        kernels.attention_masked(ctx, t, t, t, t, 1, 1, torch.zeros(2, dtype=torch.int32))


# ---- queries near zero, biases of any sign and size --------------------------------------


def check_bias(ctx, dtype, hd, lens, heads, kv_heads, slopes, by=None, v_by=1.0, **kw):
    g, off = gen(61), offsets(lens)
    rows = int(off[-1])
    q, k, v = (rand(g, rows, c * hd, dtype=dtype) for c in (heads, kv_heads, kv_heads))
    v = (v.float() * v_by).to(v.dtype)
    for i, f in enumerate(by or ()):  # every seventh row each
        q[i::7] = (q[i::7].float() * f).to(q.dtype)
    slopes = torch.tensor([slopes[h % len(slopes)] for h in range(heads)], dtype=torch.float32)
    say("bias", dtype, "hd", hd, "lens", lens, "heads", heads, kw)
    got = run_attention(ctx, q, k, v, off, heads, kv_heads, slopes=slopes, **kw)
    want, mean, _ = attention_ref(q, k, v, off, heads, kv_heads, slopes=slopes, **kw)
    # A score's size, at most: the products' (the cap, if that is less) and the farthest key's bias.
    scale = abs(kw.get("scale") or hd ** -0.5)
    dots = scale * float(q.double().abs().max() * k.double().abs().max()) * hd
    size = torch.full_like(mean, min(dots, kw.get("softcap") or dots) + float(slopes.abs().max()) * max(lens))
    close(got, want, attention_tol(dtype, hd, want, mean, size), "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens,heads,kv_heads", [([90, 40], 4, 2), ([700, 300], 24, 8)])
def test_attention_bias_of_queries_near_zero(gpu_ctx, dtype, hd, lens, heads, kv_heads):
    """Queries of zeros and of tiny values: the bias alone makes their weights.  In the form
    whose waves share rows and in the other; masked, and under a cap."""
    by, slopes = (0.0, 1e-38, 1e-36, 1e-30, 1e-22), (0.5, 2.0 ** -4, 2.0 ** -8)
    check_bias(gpu_ctx, dtype, hd, lens, heads, kv_heads, slopes, by)
    check_bias(gpu_ctx, dtype, hd, lens, heads, kv_heads, slopes, by, causal=True, window=50, scale=-0.2)
    check_bias(gpu_ctx, dtype, hd, lens, heads, kv_heads, slopes, by, softcap=5.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1e-39, 1e-37, -1e-30, 1e-6, 3e5])
def test_attention_bias_beside_scales_of_any_size(gpu_ctx, dtype, scale):
    """A scale that leaves nothing of the scores but the bias, or makes one key take all."""
    check_bias(gpu_ctx, dtype, 64, [90, 140], 4, 2, (0.5, 2.0 ** -6), scale=scale)
    check_bias(gpu_ctx, dtype, 64, [90, 140], 4, 2, (0.5, 2.0 ** -6), (0.0,), scale=scale, causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cap", [0.0, 20.0, 50.0])
@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (24, 8)])
def test_attention_bias_that_grows_with_distance(gpu_ctx, dtype, cap, heads, kv_heads):
    """Negative slopes: far keys weigh most, and scores leave float32's exponents in powers of
    two (90 at slope 0.1, 225 at 0.25) ahead of the softmax."""
    for v_by in (0.05, 1e-3):
        check_bias(gpu_ctx, dtype, 64, [900], heads, kv_heads, (-0.1, -0.25), v_by=v_by, softcap=cap)
    check_bias(gpu_ctx, dtype, 128, [330, 900], heads, kv_heads, (-0.1, 0.1), softcap=cap, causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 256])
def test_attention_values_at_the_types_end(gpu_ctx, dtype, hd):
    """Values whose sum over the keys leaves float32's range, though no mean of them does."""
    g, off = gen(62), offsets([50, 70])
    q, k, v = (rand(g, 120, hd, dtype=dtype) for _ in range(3))
    v = torch.sign(v) * 3.2e38
    v[:, ::3] = 3.2e38
    assert bool(torch.isfinite(v).all())
    got = run_attention(gpu_ctx, q, k, v, off, 1, 1)
    want, mean, size = attention_ref(q, k, v, off, 1, 1)
    # (careful_row's weights are float32 whatever the type: a division more each.)
    close(got, want, attention_tol(dtype, hd, want, mean, size) + 4 * F * mean, "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("odd", [1.0, math.inf, math.nan])
def test_attention_scores_of_minus_infinity(gpu_ctx, dtype, odd):
    """Visible keys whose scores are all -inf weigh nothing, as hidden ones do: zeros, whatever
    their values are."""
    g, off = gen(63), offsets([40])
    q, k, v = (rand(g, 40, 64, dtype=dtype) for _ in range(3))
    q[:, 0] = q[:, 0].abs() + 0.5
    k[:3, 0], v[:3, 5] = -math.inf, odd
    got = run_attention(gpu_ctx, q, k, v, off, 1, 1, causal=True)
    assert bool((got[:3] == 0).all())
    if odd == 1.0:
        want, mean, size = attention_ref(q[3:], k[3:], v[3:], offsets([37]), 1, 1, causal=True)
        close(got[3:], want, attention_tol(dtype, 64, want, mean, size), "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,k,rank", [("bf16", 4096, 16), ("bf16", 2048, 64), ("f32", 4096, 16), ("f16", 776, 100),
                                          ("f32", 64, 8)])
def test_adapters_workspace_of_the_largest_batch_serves_all(gpu_ctx, dtype, k, rank):
    """Smaller batches may be split into more parts: a workspace for more rows is enough
    for them, and what they get does not depend on its size."""
    from semantica_gpu import kernels
    c = adapter_case(dtype, k, 72, rank, 3, [2064], seed=3)
    bank = kernels.AdapterBank(gpu_ctx, c["a"].cuda(), c["b"].cuda(), c["scales"].cuda())
    x, base = c["x"].cuda(), c["base"].cuda()
    counts = sorted({0, 1, 2, 15, 16, 17, 33000, 40000} | {16 * t + d for t in range(1, 140) for d in (-1, 0, 1)})
    needs = [bank.work_bytes(rows) for rows in counts]
    assert needs == sorted(needs)
    largest = torch.empty(bank.work_bytes(2064), dtype=torch.uint8, device="cuda")
    ids = torch.tensor([1], dtype=torch.int32, device="cuda")
    for rows in (1, 16, 17, 200, 512, 1000, 1024, 1365, 2048, 2064):
        say("workspace", dtype, k, rank, "rows", rows)
        got, want = (torch.full_like(base[:rows], 7.0) for _ in range(2))
        off = offsets([rows]).cuda()
        kernels.adapters_apply(gpu_ctx, got, base[:rows], bank, x[:rows], off, ids, work=largest)
        kernels.adapters_apply(gpu_ctx, want, base[:rows], bank, x[:rows], off, ids)
        assert torch.equal(got, want)
        true, size = adapters_ref(c["x"][:rows], c["base"][:rows], c["a"], c["b"], c["scales"], offsets([rows]), ids.cpu())
        rel = (k + rank + 32) * F + (0 if dtype == "f32" else 2.0 ** -16)
        close(got, true, U[dtype] * true.abs() + rel * size + TINY[dtype], "adapters")
    bank.close()


@pytest.mark.gpu
def test_a_refused_bank_leaves_no_error_behind(gpu_ctx):
    """More adapters than the device's memory holds, then calls that succeed: this library's
    and torch's."""
    from semantica_gpu import _lib
    lib = _lib.load()
    c = adapter_case("f32", 96, 80, 8, 4, [1] * 16)
    clean = run_adapters(gpu_ctx, c)
    some, h = torch.zeros(64, device="cuda"), ctypes.c_void_p()
    for _ in range(2):
        # A: 2^24 adapters x 16 ranks x 1024 float32, 2^40 bytes.  The allocation is the first step.
        rc = lib.sg_adapter_bank_create(gpu_ctx.handle, some.data_ptr(), some.data_ptr(), some.data_ptr(), 0, 1 << 24, 16,
                                        1024, 64, None, ctypes.byref(h))
        assert rc == _lib.SG_ERR_NOMEM and not h.value
        for name, call, _, outs in layer_calls(gpu_ctx):
            say(name, "after a refused allocation")
            call()
        assert float((some + 1).sum()) == 64
    assert torch.equal(run_adapters(gpu_ctx, c), clean)


@pytest.mark.gpu
def test_a_call_does_not_report_an_earlier_error(gpu_ctx):
    """An error that another call of the thread left behind (a device that is not there) stays
    that call's."""
    from semantica_gpu import _lib
    calls = layer_calls(gpu_ctx)
    hip = _lib.load()  # (its symbols reach the HIP runtime that it is linked to)
    try:
        for name, call, _, _ in calls:
            assert hip.hipSetDevice(1 << 20) != 0
            say(name, "after another call's error")
            call()
    finally:
        hip.hipGetLastError()
    torch.cuda.synchronize()


# ---- the forms that only large batches take ------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [16, 32, 48, 64])
def test_adapters_of_33000_rows(gpu_ctx, dtype, rank):
    """A thousand workgroups of two row tiles and more: tiles of one adapter, and several in
    every tile."""
    check_adapters(gpu_ctx, dtype, 136, 72, rank, 9, [33000], first=5, behind=3)
    check_adapters(gpu_ctx, dtype, 136, 72, rank, 9, [3] * 10000 + [1, 0, 2999, 33], first=1, behind=9)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rank,rows", [(16, 33000), (32, 33000), (64, 33000), (100, 33000), (256, 17000)])
def test_adapters_over_wide_slices(gpu_ctx, dtype, rank, rows):
    """2048 slices of 256 columns and more in the second product, the last one narrow, with
    ranks that the first product leaves ready and with larger ones."""
    check_adapters(gpu_ctx, dtype, 64, 520, rank, 7, [rows - 1003, 3, 500, 500], behind=1)
    check_adapters(gpu_ctx, dtype, 64, 520, rank, 7, [5] * (rows // 5), in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [16, 32, 48, 100])
def test_adapters_over_wide_slices_of_one_tile(gpu_ctx, dtype, rank):
    """The same with rows too few for two tiles to a workgroup."""
    check_adapters(gpu_ctx, dtype, 64, 2056, rank, 5, [4000, 1, 99], first=1)
    check_adapters(gpu_ctx, dtype, 64, 2056, rank, 5, [2] * 2100, behind=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,cols,rows", [("f32", 1100, 5000), ("bf16", 2100, 5000), ("f16", 4104, 4300),
                                             ("f32", 5000, 2300), ("f32", 4097, 2300)])
def test_norm_rows_one_after_another(gpu_ctx, dtype, cols, rows):
    """Workgroups that share a row's sums and take several rows in turn, some of no sequence."""
    check_norm(gpu_ctx, dtype, rows, cols, lens=[1, 0, 0, 7, rows - 15, 3], first=2, gate=True)
    check_norm(gpu_ctx, dtype, rows, cols, lens=[1] * 700 + [rows - 2000], first=650, gate=True, post=False)
    check_norm(gpu_ctx, dtype, rows, cols, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [8, 40, 72, 136, 200, 248])
def test_attention_odd_head_dims_many_rows(gpu_ctx, dtype, hd):
    """Head dims that fill no layout, with rows enough for waves of their own rows."""
    lens = [300, 1, 0, 400, 63]
    check_attention(gpu_ctx, hd, dtype, 24, 8, hd, lens, first=1, behind=2, **mask_of("all", 24, lens, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("at", [1, 2, 3])
def test_attention_document_ids_at_any_alignment(gpu_ctx, at):
    """Ids that start inside a 16-byte piece, one look over many tiles and a ragged end."""
    rows, hd = 5003, 8
    g = gen(64)
    q, k, v = (rand(g, rows, hd, dtype="bf16") for _ in range(3))
    ids = (torch.arange(rows) // 61).to(torch.int32)
    ids[100:120] = -1
    wide = torch.zeros(rows + at, dtype=torch.int32)
    wide[at:] = ids
    from semantica_gpu import kernels
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    kernels.attention_masked(gpu_ctx, out, q.cuda(), k.cuda(), v.cuda(), 1, 1, offsets([rows]).cuda(),
                             doc_ids=wide.cuda()[at:], causal=True)
    out = out.cpu()
    assert bool((out[100:120] == 0).all())
    for doc in (0, 1, 40, int(ids.max())):
        to = (ids == doc).nonzero()[:, 0]
        want, mean, size = attention_ref(q[to], k[to], v[to], offsets([len(to)]), 1, 1, causal=True)
        close(out[to], want, attention_tol("bf16", hd, want, mean, size), f"document {doc}")


# ---- float32's bits -----------------------------------------------------------------------
# float32 attention holds q, k, the weights and the values as two fp16 halves each and drops
# the products of two low halves.  A half is off by 2^-12 of it at most, so an operand of two
# by 2^-22 (2^-12 2^-11 and the low half's own 11 bits: 2^-23), and what is dropped is 2^-22 of a
# product at most.  Over the terms of a sum these are of either sign: with normal q and k a
# score (of deviation 1) is off by some 2^-22 for each of q, k and the dropped part, a weight by
# as much, and an output of many keys, relative to the outputs' size, by those of the scores,
# the weights, the values and the dropped part again: sqrt(6) 2^-22, and float32's sums of
# hd products and of the keys, a few 2^-24.  Together below 2^-20.  The limit is twice that; any
# one low half left out is off by 2^-12 / sqrt(3) / 2 and more (2^-14).
FLOAT32_L2 = 2.0 ** -19


def halves(x, low=True):
    """x as two fp16 halves, its rows brought to 2^13 .. 2^14 first."""
    e = torch.floor(torch.log2(x.abs().amax(-1, keepdim=True)))
    y = x * 2.0 ** (13 - e)
    hi = y.half().double()
    lo = (y - hi).half().double() if low else torch.zeros_like(hi)
    return hi, lo, 2.0 ** (e - 13)


def attention_in_halves(q, k, v, without=""):
    """One sequence and head as the float32 kernel multiplies it, `without` a low half."""
    qh, ql, qe = halves(q.double(), "q" not in without)
    kh, kl, ke = halves(k.double(), "k" not in without)
    vh, vl, ve = halves(v.double(), "v" not in without)
    s = (qh @ kh.T + qh @ kl.T + ql @ kh.T) * qe * ke.T / math.sqrt(q.shape[1])
    p = torch.exp(s - s.amax(-1, keepdim=True))
    w = p * ve.T
    by = 2.0 ** (5 - torch.floor(torch.log2(w.amax(-1, keepdim=True))))
    wh = (w * by).half().double()
    wl = (w * by - wh).half().double() if "p" not in without else torch.zeros_like(wh)
    return (wh @ vh + wh @ vl + wl @ vh) / by / p.sum(-1, keepdim=True)


def l2(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_float32_limit_tells_a_lost_half(hd):
    g = gen(hd)
    q, k, v = (rand(g, 300, hd) for _ in range(3))
    want, _, _ = attention_ref(q, k, v, offsets([300]), 1, 1)
    assert l2(attention_in_halves(q, k, v), want) < FLOAT32_L2 / 2
    for half in "qkpv":
        assert l2(attention_in_halves(q, k, v, half), want) > 4 * FLOAT32_L2, half


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens,heads,kv_heads", [([300, 90], 3, 1), ([1501], 2, 1), ([700, 333], 24, 8)])
def test_attention_keeps_float32s_bits(gpu_ctx, hd, lens, heads, kv_heads):
    g, off = gen(65), offsets(lens)
    rows = int(off[-1])
    q, k, v = (rand(g, rows, c * hd) for c in (heads, kv_heads, kv_heads))
    slopes = torch.tensor([2.0 ** -(4 + h % 4) for h in range(heads)])
    for kw in ({}, {"causal": True, "softcap": 20.0}, {"softcap": 2.0}, {"slopes": slopes, "window": 200}):
        got = run_attention(gpu_ctx, q, k, v, off, heads, kv_heads, **kw)
        want, _, _ = attention_ref(q, k, v, off, heads, kv_heads, **kw)
        say("float32 bits", hd, lens, sorted(kw), l2(got, want))
        assert l2(got, want) < FLOAT32_L2


# ---- tensors that are columns of one -------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_outputs_beside_their_inputs_in_one_tensor(gpu_ctx, dtype):
    """Inputs and outputs as columns of one wide tensor, in any order; what lies between stays."""
    from semantica_gpu import kernels
    g, rows, off = gen(71), 70, offsets([50, 20])
    t = dt(dtype)

    def wide(*cols):
        """One tensor of these widths side by side, eight columns of sevens behind each."""
        w = torch.full((rows, sum(cols) + 8 * len(cols)), 7.0, dtype=t, device="cuda")
        at = np.concatenate([[0], np.cumsum([c + 8 for c in cols])])
        parts = [w[:, a:a + c] for a, c in zip(at, cols)]
        for p in parts:
            p.copy_(rand(g, *p.shape).to(t).cuda())
        return parts, [w[:, a + c:a + c + 8] for a, c in zip(at, cols)]

    (out, k, q, v), gaps = wide(128, 64, 128, 64)
    kernels.attention_masked(gpu_ctx, out, q, k, v, 2, 1, off.cuda(), causal=True)
    want, mean, size = attention_ref(q.cpu(), k.cpu(), v.cpu(), off, 2, 1, causal=True)
    close(out, want, attention_tol(dtype, 64, want, mean, size), "attention")
    assert all(bool((p == 7).all()) for p in gaps)

    (xn, x, s, h), gaps = wide(96, 96, 96, 96)
    w = torch.randn(96, generator=g)
    kernels.block_norm(gpu_ctx, xn, s, x, h, w.cuda(), w.cuda(), 1e-6)
    ws, wn, ssize, nsize = norm_ref(x.cpu(), h.cpu(), w, w, 1e-6, None, 1.0, None)
    close(s, ws, U[dtype] * ws.abs() + 58 * F * ssize + TINY[dtype], "sum")
    close(xn, wn, U[dtype] * wn.abs() + 116 * F * nsize + TINY[dtype], "xn")
    assert all(bool((p == 7).all()) for p in gaps)

    (x, dst, base), gaps = wide(64, 72, 72)
    a, b = rand(g, 2, 8, 64, by=0.1, dtype=dtype), rand(g, 2, 72, 8, dtype=dtype)
    scales, ids = torch.tensor([0.5, 2.0]), torch.tensor([1, 0], dtype=torch.int32)
    bank = kernels.AdapterBank(gpu_ctx, a.cuda(), b.cuda(), scales.cuda())
    kernels.adapters_apply(gpu_ctx, dst, base, bank, x, off.cuda(), ids.cuda())
    want, size = adapters_ref(x.cpu(), base.cpu(), a, b, scales, off, ids)
    close(dst, want, U[dtype] * want.abs() + (104 * F + 2.0 ** -16) * size + TINY[dtype], "adapters")
    assert all(bool((p == 7).all()) for p in gaps)
    bank.close()


# heads of 128 in float16: 256 columns of out and q, 128 of k and v; all of them columns of one
# tensor of 1024, q's first.
BESIDE = {**ATT, **{n: 1024 for n in ("ldo", "ldq", "ldk", "ldv")}, "q": 2 << 40, "out": (2 << 40) + 2 * 256,
          "k": (2 << 40) + 2 * 512, "v": (2 << 40) + 2 * 640}


@pytest.mark.parametrize("change", [
    {"out": (2 << 40) + 2 * 248}, {"out": (2 << 40) + 2 * 264}, {"out": (2 << 40) + 2 * 760},
    {"out": (2 << 40) + 2 * (1024 + 248)}, {"out": (2 << 40) - 2 * 248}, {"out": (2 << 40) + 2 * (8 * 1024 + 776)},
    {"ldo": 512}])
def test_attention_refuses_columns_that_meet(change):
    """A piece of 16 bytes too far to either side, in the same row or another; another stride."""
    from semantica_gpu import _lib
    c = {**BESIDE, **change}
    _refused(_lib.load().sg_attention_masked(_addr(), c["out"], c["ldo"], c["q"], c["ldq"], c["k"], c["ldk"], c["v"], c["ldv"],
                                             c["dtype"], c["heads"], c["kv"], c["hd"], c["rows"], c["off"], c["n_seq"], None,
                                             None), "overlaps")


@pytest.mark.gpu
def test_default_workspace_is_the_streams_own(gpu_ctx):
    """A workspace for another stream is not memory that the current one gave back and may
    still be writing."""
    from semantica_gpu import kernels
    c = adapter_case("f32", 64, 72, 32, 3, [20000], seed=5)
    bank = kernels.AdapterBank(gpu_ctx, c["a"].cuda(), c["b"].cuda(), c["scales"].cuda())
    x, base, off, ids = c["x"].cuda(), c["base"].cuda(), c["off"].cuda(), torch.tensor([1], dtype=torch.int32, device="cuda")
    need, dst, side = bank.work_bytes(20000), torch.full_like(base, 7.0), torch.cuda.Stream()

    class Spy:  # takes the call's workspace and runs nothing
        handle, device = gpu_ctx.handle, gpu_ctx.device

        def __init__(self):
            self.lib = self

        def sg_adapters_apply(self, *args):
            self.work, self.bytes = args[12], args[13]
            return 0

    spy = Spy()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    back = torch.empty(need, dtype=torch.uint8, device="cuda")
    at = back.data_ptr()
    del back
    seen = []
    for _ in range(2):
        kernels.adapters_apply(spy, dst, base, bank, x, off, ids, stream=side.cuda_stream)
        assert spy.bytes >= need and abs(spy.work - at) >= need
        seen.append(spy.work)
    assert seen[0] == seen[1]  # in order on its own stream
    kernels.adapters_apply(spy, dst, base, bank, x, off, ids)
    assert spy.work == at
    side.wait_stream(torch.cuda.current_stream())
    kernels.adapters_apply(gpu_ctx, dst, base, bank, x, off, ids, stream=side.cuda_stream)
    side.synchronize()
    c["ids"] = ids.cpu()
    want, size = adapters_ref(c["x"], c["base"], c["a"], c["b"], c["scales"], c["off"], c["ids"])
    close(dst, want, U["f32"] * want.abs() + 128 * F * size + TINY["f32"], "adapters")
    bank.close()


@pytest.mark.gpu
def test_banks_collected_during_a_capture(gpu_ctx):
    """By the capturing thread and by another: the graph is whole, and the memory comes back
    with the next bank that is made or closed."""
    import threading
    from semantica_gpu import kernels
    calls = layer_calls(gpu_ctx, "bf16", 7)
    for _, call, _, _ in calls:
        call()
    torch.cuda.synchronize()
    want = [t.clone() for _, _, _, outs in calls for t in outs]
    a, b, scales = (torch.zeros(s, device="cuda") for s in ((2048, 16, 1024), (2048, 1024, 16), (2048,)))
    banks = [kernels.AdapterBank(gpu_ctx, a, b, scales) for _ in range(2)]
    last = kernels.AdapterBank(gpu_ctx, a[:1], b[:1], scales[:1])
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    graph = torch.cuda.CUDAGraph()
    say("capturing")
    with torch.cuda.graph(graph):
        calls[0][1]()
        banks.pop()
        calls[1][1]()
        other = threading.Thread(target=banks.clear)
        other.start()
        other.join()
        calls[2][1]()
    last.close()
    assert torch.cuda.mem_get_info()[0] >= free + 4 * (a.numel() + b.numel())
    for _ in range(3):
        for _, _, _, outs in calls:
            for t in outs:
                t.fill_(7.0)
        say("replay")
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip([t for _, _, _, outs in calls for t in outs], want):
            assert torch.equal(x[3:434], y[3:434])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bank_of_more_pieces_than_packing_threads(gpu_ctx, dtype):
    """Over 2^24 pieces of 16 bytes in both arrays, which the packing threads take in turn."""
    from semantica_gpu import kernels
    n, rank, wide = (1100, 16, 16384) if dtype == "bf16" else (550, 16, 16384)
    g = gen(81)
    by = torch.randn(n, generator=g)
    a0, b0 = rand(g, rank, wide, by=wide ** -0.5, dtype=dtype), rand(g, wide, rank, dtype=dtype)
    a = (a0.cuda() * by.to(a0.dtype).cuda()[:, None, None]).contiguous()
    b = (b0.cuda() * by.flip(0).to(b0.dtype).cuda()[:, None, None]).contiguous()
    assert a.numel() * a.element_size() > 16 << 24
    say("bank", dtype, a.numel() * a.element_size() * 2 >> 20, "MiB")
    scales = torch.rand(n, generator=g) + 0.5
    bank = kernels.AdapterBank(gpu_ctx, a, b, scales.cuda())
    ids = torch.tensor([0, 1, n // 2, n - 2, n - 1], dtype=torch.int32)
    off, rows = offsets([2, 1, 3, 1, 2]), 9
    x, base = rand(g, rows, wide, dtype=dtype), rand(g, rows, wide, dtype=dtype)
    dst = torch.empty(rows, wide, dtype=dt(dtype), device="cuda")
    kernels.adapters_apply(gpu_ctx, dst, base.cuda(), bank, x.cuda(), off.cuda(), ids.cuda())
    bank.close()
    used = ids.long()
    want, size = adapters_ref(x, base, a[used].cpu(), b[used].cpu(), scales[used], off, torch.arange(5))
    rel = (wide + rank + 32) * F + (0 if dtype == "f32" else 2.0 ** -16)
    close(dst, want, U[dtype] * want.abs() + rel * size + TINY[dtype], "adapters")


@pytest.mark.parametrize("change", [
    {"heads": 64, "kv": 1, "hd": 8, "rows": 1 << 26}, {"heads": 65535, "kv": 1, "hd": 8, "rows": 1 << 21},
    {"heads": 1, "kv": 1, "hd": 8, "rows": (1 << 31) - (1 << 17), "dtype": 0}])
def test_attention_refuses_more_than_a_launch(change):
    """2^32 threads and more."""
    from semantica_gpu import _lib
    c = {**ATT, **change, "ldo": 8 * 65536, "ldq": 8 * 65536}
    _refused(_lib.load().sg_attention_masked(_addr(), c["out"], c["ldo"], c["q"], c["ldq"], c["k"], c["ldk"], c["v"], c["ldv"],
                                             c["dtype"], c["heads"], c["kv"], c["hd"], c["rows"], c["off"], c["n_seq"], None,
                                             None), "one launch")


@pytest.mark.parametrize("n", [1 << 31, (1 << 32) + 8])
def test_wrappers_refuse_counts_past_32_bits(n):
    """Counts that would lose their upper bits on the way to the C ABI."""
    from semantica_gpu import kernels
    ctx, off = _Ctx(), torch.zeros(2, dtype=torch.int32)
    rows, cols = torch.zeros(1, 64).expand(n, 64), torch.zeros(1, 1).expand(1, n)
    one, w = torch.zeros(1, 64), torch.zeros(64)

    class Bank:
        in_dim, out_dim, dtype, handle = 64, 64, torch.float32, None

        def work_bytes(self, rows):
            return 16

    for call in (lambda: kernels.attention_masked(ctx, rows, rows, rows, rows, 1, 1, off),
                 lambda: kernels.attention_masked(ctx, cols, cols, cols, cols, 1, 1, off),
                 lambda: kernels.attention_masked(ctx, one, one, one, one, 1, 1, torch.zeros(1, dtype=torch.int32).expand(n)),
                 lambda: kernels.block_norm(ctx, None, rows, rows, rows, w, None, 1e-6),
                 lambda: kernels.block_norm(ctx, None, cols, cols, cols, None, None, 1e-6),
                 lambda: kernels.adapters_apply(ctx, rows, rows, Bank(), rows, off, off[:1]),
                 lambda: kernels.AdapterBank(ctx, torch.zeros(1, 1, 8).expand(n, 1, 8), torch.zeros(1, 8, 1).expand(n, 8, 1), w),
                 lambda: kernels.AdapterBank.work_bytes(Bank(), n)):
        with pytest.raises(ValueError, match="more than a call takes"):
            call()


@pytest.mark.parametrize("window", [-1, -(1 << 32), -(1 << 32) + 5])
def test_attention_wrapper_refuses_any_negative_window(window):
    from semantica_gpu import SemanticaError, kernels
    t = torch.zeros(0, 64)
    with pytest.raises(SemanticaError, match="window"):
        kernels.attention_masked(_Ctx(), t, t, t, t, 1, 1, torch.zeros(2, dtype=torch.int32), window=window, stream=0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 72, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(3, 1), (24, 8)])
def test_attention_does_not_read_padding_rows(gpu_ctx, dtype, hd, heads, kv_heads):
    """What lies before the first sequence and behind the last: keys and values of NaN there give
    the very bits that zeros give, so no row is computed again for them."""
    lens = [50, 1, 300, 97]
    g, off = gen(91), offsets(lens, first=5)
    rows = int(off[-1]) + 90
    q, k, v = (rand(g, rows, c * hd, dtype=dtype) for c in (heads, kv_heads, kv_heads))
    slopes = torch.tensor([2.0 ** -(2 + h % 5) for h in range(heads)])
    for kw in ({}, {"causal": True, "window": 70, "softcap": 9.0, "slopes": slopes}):
        outs = []
        q[:5] = q[int(off[-1]):] = math.nan
        for fill in (0.0, math.nan):
            for t in (k, v):
                t[:5] = t[int(off[-1]):] = fill
            outs.append(run_attention(gpu_ctx, q, k, v, off, heads, kv_heads, **kw))
        assert torch.equal(*outs)
        inside = slice(5, int(off[-1]))
        want, mean, size = attention_ref(q, k, v, off, heads, kv_heads, **kw)
        close(outs[0][inside], want[inside], attention_tol(dtype, hd, want, mean, size, kw.get("softcap", 0.0))[inside],
              "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(2, 1), (24, 8)])
@pytest.mark.parametrize("qs,ks", [(1e-34, 1e33), (1e33, 1e-34), (1e-30, 3e33), (3e33, 1e-30)])
def test_attention_of_opposite_powers(gpu_ctx, hd, heads, kv_heads, qs, ks):
    """float32 queries and keys of far-apart powers of two, all in one direction or against it:
    the scores are small, what they are made of is not."""
    g, off = gen(92), offsets([300, 90])
    rows = 390
    q = (1 + torch.rand(rows, heads * hd, generator=g)) * torch.where(torch.rand(rows, 1, generator=g) < 0.5, -qs, qs)
    k = (1 + torch.rand(rows, kv_heads * hd, generator=g)) * torch.where(torch.rand(rows, 1, generator=g) < 0.5, -ks, ks)
    v = rand(g, rows, kv_heads * hd)
    for kw in ({}, {"softcap": 3.0, "causal": True}, {"scale": 1e-5 if qs * ks > 1 else 0.0}):
        got = run_attention(gpu_ctx, q, k, v, off, heads, kv_heads, **kw)
        want, mean, size = attention_ref(q, k, v, off, heads, kv_heads, **kw)
        close(got, want, attention_tol("f32", hd, want, mean, size, kw.get("softcap", 0.0)), "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,cols", [("f32", 20000, 40), ("bf16", 20000, 72), ("f32", 5000, 1100), ("f32", 2300, 4200)])
def test_norm_passes_over_runs_of_empty_sequences(gpu_ctx, dtype, rows, cols):
    """Runs of empty sequences between rows that one workgroup takes in turn: a few, hundreds,
    and more than a lookup's first step covers; rows of no sequence at both ends."""
    lens = [1] * 5 + [0] * 3 + [2] + [0] * 70 + [1, 1] + [0] * 5000 + [rows // 2] + [0] * 64 + [1] + [0] * 700 + [3] + [0] * 9
    lens = [0] * 90 + lens + [rows - 3 - sum(lens) - 4] + [0] * 300
    check_norm(gpu_ctx, dtype, rows, cols, lens=lens, first=3, gate=True)
    check_norm(gpu_ctx, dtype, rows, cols, lens=lens[:-301], first=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,rank", [([9, 20, 3], 16), ([1] * 40, 100), ([9000, 8000], 32)])
@pytest.mark.parametrize("by_x,by_b", [(1e-34, 1e35), (1e-20, 1e25), (1e25, 1e-30), (1e-34, 1.0)])
def test_adapters_of_far_apart_powers(gpu_ctx, dtype, lens, rank, by_x, by_b):
    """Small low-rank values against large weights and the other way round."""
    c = adapter_case(dtype, 64, 72, rank, 2, lens, seed=7, by=by_x)
    c["b"] = (c["b"].float() * by_b).to(c["b"].dtype)
    c["ids"] = torch.arange(len(lens), dtype=torch.int32) % 2
    say("adapters", dtype, lens[:4], rank, by_x, by_b)
    got = run_adapters(gpu_ctx, c)
    want, size = adapters_ref(c["x"], c["base"], c["a"], c["b"], c["scales"], c["off"], c["ids"])
    rel = (64 + rank + 32) * F + (0 if dtype == "f32" else 2.0 ** -16)
    close(got, want, U[dtype] * want.abs() + rel * size + TINY[dtype], "adapters")
