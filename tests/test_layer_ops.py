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
    ({"n_seq": 0}, {}, "seq_offsets"), ({"ldq": 255}, {}, "stride"), ({"ldk": 129}, {}, "aligned"), ({"v": (4 << 40) + 8}, {}, "aligned"),
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
    ({"sum": (4 << 40) + 4}, "overlaps"), ({"xn": 3 << 40, "ldxn": 65}, "overlaps")])
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
    ({"out": 0}, "multiples of 8"), ({"n": 1 << 30, "rank": 256, "k": 1 << 16}, "too many")])
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
