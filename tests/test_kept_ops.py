"""What answers requests behind kept text, against its definitions in 64 bits, and what it
refuses: sg_kv_cache_write, sg_kv_cache_read, sg_attention_shared, sg_matmul_q4.

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


def ints(a):
    return torch.tensor(np.asarray(a, np.int64).astype(np.int32))


def offsets(lens, first=0):
    return ints(np.concatenate([[first], first + np.cumsum(lens)]))


def same(got, want, what):
    """Equal, NaN for NaN."""
    got, want = got.cpu(), want.cpu()
    ok = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} differ"


def close(got, want, tol, what):
    got = got.double().cpu()
    err = (got - want).abs()
    ok = (err <= tol) | (got == want) | (torch.isnan(got) & torch.isnan(want))
    worst = (err / tol.clamp_min(1e-300)).nan_to_num(math.inf)[~ok]
    assert bool(ok.all()), f"{what}: {int((~ok).sum())} of {ok.numel()} off, up to {float(worst.max()):.3g} tolerances"


# ---- the cache --------------------------------------------------------------------


def kept_ref(x, kv_heads, bits):
    """What a cache stands for, in 64 bits and as it is read: [rows, kv_heads * hd] each."""
    if bits == 0:
        return x.double(), x
    y = x.double().reshape(x.shape[0], kv_heads, -1)
    top = y.abs().amax(-1, keepdim=True)  # (NaN where a NaN is)
    scale = (top / 127).float().double().clamp_min(2.0 ** -126)  # 53 bits round to 24 as the quotient does
    scale = torch.where(torch.isfinite(top), scale, math.nan)
    y = torch.round(y / scale).clamp(-127, 127) * scale
    return y.reshape(x.shape), y.float().to(x.dtype).reshape(x.shape)


def make_cache(ctx, slots, kv_heads, hd, dtype, bits):
    from semantica_gpu import kernels
    return kernels.KVCache(ctx, slots, kv_heads, hd, dt(dtype), bits=bits)


def fill_cache(ctx, cache, k, v):
    from semantica_gpu import kernels
    kernels.kv_cache_write(ctx, cache, k.cuda(), v.cuda(), ints([0, k.shape[0]]).cuda(), ints([0]).cuda())


def read_cache(ctx, cache):
    from semantica_gpu import kernels
    k = torch.empty(cache.slots, cache.n_kv_heads * cache.head_dim, dtype=cache.dtype, device="cuda")
    v = torch.empty_like(k)
    kernels.kv_cache_read(ctx, k, v, cache, ints([0, cache.slots]).cuda(), ints([0]).cuda())
    return k.cpu(), v.cpu()


def check_rows(ctx, seed, dtype, bits, kv_heads, hd, lens, starts, slots, first=0, behind=0):
    """Rows in over what was there, everything out; the later of two sequences keeps a slot."""
    from semantica_gpu import kernels
    say("rows", dtype, bits, "heads", kv_heads, "hd", hd, "lens", list(lens)[:8], "starts", list(starts)[:8], "slots", slots)
    g = gen(seed)
    off = offsets(lens, first)
    rows = int(off[-1]) + behind
    k, v = rand(g, rows, kv_heads * hd, by=3.0, dtype=dtype), rand(g, rows, kv_heads * hd, dtype=dtype)
    k0, v0 = rand(g, slots, kv_heads * hd, dtype=dtype), rand(g, slots, kv_heads * hd, by=2.0, dtype=dtype)
    cache = make_cache(ctx, slots, kv_heads, hd, dtype, bits)
    try:
        fill_cache(ctx, cache, k0, v0)
        kernels.kv_cache_write(ctx, cache, k.cuda(), v.cuda(), off.cuda(), ints(starts).cuda())
        want_k, want_v = kept_ref(k0, kv_heads, bits)[1].clone(), kept_ref(v0, kv_heads, bits)[1].clone()
        rk, rv = kept_ref(k, kv_heads, bits)[1], kept_ref(v, kv_heads, bits)[1]
        back_k, back_v = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
        for i, s in enumerate(starts):
            for r in range(int(off[i]), int(off[i + 1])):
                at = s + r - int(off[i])
                if s >= 0 and at < slots:
                    want_k[at], want_v[at] = rk[r], rv[r]
        for i, s in enumerate(starts):
            for r in range(int(off[i]), int(off[i + 1])):
                at = s + r - int(off[i])
                there = s >= 0 and at < slots
                back_k[r] = want_k[at] if there else 0
                back_v[r] = want_v[at] if there else 0
        got_k, got_v = read_cache(ctx, cache)
        same(got_k, want_k, "keys")
        same(got_v, want_v, "values")
        out_k, out_v = torch.full_like(k, 7.0).cuda(), torch.full_like(v, 7.0).cuda()
        kernels.kv_cache_read(ctx, out_k, out_v, cache, off.cuda(), ints(starts).cuda())
        same(out_k, back_k, "keys read")
        same(out_v, back_v, "values read")
    finally:
        cache.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("hd", [8, 64, 72, 128, 200, 256])
def test_rows(gpu_ctx, dtype, bits, hd):
    """Ranges that begin and end anywhere in a tile, empty sequences, rows of none, one slot at a time."""
    check_rows(gpu_ctx, hd, dtype, bits, 2, hd, [1, 0, 5, 33, 70, 1, 3], [9, 4, 100, 131, 30, 0, 65], 171, first=3, behind=4)
    check_rows(gpu_ctx, hd, dtype, bits, 3, hd, [1], [0], 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
def test_rows_many(gpu_ctx, dtype, bits):
    """Rows enough for workgroups of 32 of them."""
    check_rows(gpu_ctx, 3, dtype, bits, 8, 128, [1900, 31, 0, 33, 400], [7, 2000, 0, 2100, 2133], 2600, first=2, behind=3)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [0, 8])
def test_rows_outside_and_twice(gpu_ctx, bits):
    """Starts below zero and ends past the cache; slots that several sequences name."""
    check_rows(gpu_ctx, 5, "bf16", bits, 2, 64, [10, 40, 3, 9], [-1, 30, 64, 2**31 - 5], 64)
    check_rows(gpu_ctx, 6, "f32", bits, 2, 64, [20, 20, 1, 7], [5, 10, 12, 3], 64)
    lens = [1] * 300 + [40]
    check_rows(gpu_ctx, 7, "f16", bits, 8, 64, lens, [i % 17 for i in range(300)] + [9], 64)
    r = np.random.RandomState(1)
    lens = [30] * 80
    check_rows(gpu_ctx, 8, "f16", bits, 8, 64, lens, r.randint(-5, 600, 80).tolist(), 610)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_codes_at_borders(gpu_ctx, dtype):
    """Values halfway between codes, next to halfway, tiny, huge, zero."""
    g = gen(2)
    hd, rows = 64, 600
    top = (127 * 2.0 ** torch.randint(-8, 8, (rows, 1), generator=g).double()) * torch.where(
        torch.rand(rows, 1, generator=g) < 0.5, 1.0, 1.0 + torch.rand(rows, 1, generator=g))
    half = torch.randint(-127, 127, (rows, hd), generator=g).double() + 0.5
    k = (half * top / 127).to(dt(dtype))
    k[:, :1] = top.to(dt(dtype))
    bits = {torch.float32: torch.int32}.get(dt(dtype), torch.int16)
    v = (k.view(bits) + torch.randint(-1, 2, (rows, hd), generator=g).to(bits)).view(dt(dtype))  # one step aside
    if dtype != "f16":
        k[0], k[1], k[2] = 1e-44, 3e38, 0.0
        k[3] = torch.linspace(-1e-37, 1e-37, hd).to(dt(dtype))
    cache = make_cache(gpu_ctx, rows, 1, hd, dtype, 8)
    fill_cache(gpu_ctx, cache, k, v)
    got_k, got_v = read_cache(gpu_ctx, cache)
    cache.close()
    same(got_k, kept_ref(k, 1, 8)[1], "keys")
    same(got_v, kept_ref(v, 1, 8)[1], "values")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
def test_rows_not_finite(gpu_ctx, dtype, bits):
    """An infinity or a NaN is that slot's and head's alone, and goes when it is written over."""
    g = gen(8)
    k, v = rand(g, 40, 128, dtype=dtype), rand(g, 40, 128, dtype=dtype)
    clean_k, clean_v = k.clone(), v.clone()
    k[3, 7], v[5, 64 + 3], v[33, 0], k[33, 70] = math.nan, math.inf, -math.inf, math.inf
    cache = make_cache(gpu_ctx, 40, 2, 64, dtype, bits)
    fill_cache(gpu_ctx, cache, k, v)
    got_k, got_v = read_cache(gpu_ctx, cache)
    same(got_k, kept_ref(k, 2, bits)[1], "keys")
    same(got_v, kept_ref(v, 2, bits)[1], "values")
    fill_cache(gpu_ctx, cache, clean_k, clean_v)
    got_k, got_v = read_cache(gpu_ctx, cache)
    cache.close()
    same(got_k, kept_ref(clean_k, 2, bits)[1], "keys")
    same(got_v, kept_ref(clean_v, 2, bits)[1], "values")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_one_projection(gpu_ctx, dtype):
    """k and v as columns of one tensor, in and out."""
    from semantica_gpu import kernels
    g = gen(4)
    qkv = rand(g, 50, 64 + 2 * 128 + 8, dtype=dtype).cuda()
    cache = make_cache(gpu_ctx, 70, 2, 64, dtype, 8)
    off, starts = offsets([20, 30]).cuda(), ints([33, 1]).cuda()
    kernels.kv_cache_write(gpu_ctx, cache, qkv[:, 64:192], qkv[:, 192:320], off, starts)
    wide = torch.full((50, 320), 7.0, dtype=dt(dtype), device="cuda")
    kernels.kv_cache_read(gpu_ctx, wide[:, 16:144], wide[:, 144:272], cache, off, starts)
    cache.close()
    same(wide[:, 16:144], kept_ref(qkv[:, 64:192].cpu(), 2, 8)[1], "keys")
    same(wide[:, 144:272], kept_ref(qkv[:, 192:320].cpu(), 2, 8)[1], "values")
    assert bool((wide[:, :16] == 7).all()) and bool((wide[:, 272:] == 7).all())


# ---- attention ----------------------------------------------------------------------


def shared_ref(q, k, v, off, heads, kv_heads, starts, lengths, shared=None, prefix_starts=None, prefix_lengths=None,
               scale=0.0, softcap=0.0, causal=True, window=0):
    """The definition in 64 bits over what the cache stands for, and the mean of |v| and the
    scores' size that the tolerance needs.  Rows of no sequence are NaN."""
    rows, hd, slots = q.shape[0], q.shape[1] // heads, k.shape[0]
    q, k, v = q.double().reshape(rows, heads, hd), k.reshape(slots, kv_heads, hd), v.reshape(slots, kv_heads, hd)
    scale = scale or 1.0 / math.sqrt(hd)
    out = torch.full((rows, heads, hd), math.nan, dtype=torch.float64)
    mean, size = torch.zeros(rows, heads, hd, dtype=torch.float64), torch.zeros(rows, heads, 1, dtype=torch.float64)

    def slots_of(start, length):
        start, length = int(start), int(length)
        return list(range(start, start + length)) if start >= 0 and length > 0 and start + length <= slots else []

    for i in range(off.shape[0] - 1):
        a, b = int(off[i]), int(off[i + 1])
        if a == b:
            continue
        at = []
        for p in range(shared.shape[0] - 1 if shared is not None else 0):
            if int(shared[p]) <= i < int(shared[p + 1]):
                at = slots_of(prefix_starts[p], prefix_lengths[p])
        at = torch.tensor(at + slots_of(starts[i], lengths[i]), dtype=torch.long)
        pos = at.shape[0] - (b - a) + torch.arange(b - a)
        gap = pos[:, None] - torch.arange(at.shape[0])[None, :]
        seen = torch.ones_like(gap, dtype=torch.bool)
        if causal:
            seen &= gap >= 0
        if window:
            seen &= gap.abs() < window
        some = seen.any(0)  # hidden slots' contents do not count
        for h in range(heads):
            kh, vh = k[at, h * kv_heads // heads], v[at, h * kv_heads // heads]
            kh, vh = torch.where(some[:, None], kh, 0.0), torch.where(some[:, None], vh, 0.0)
            s = q[a:b, h] @ kh.t() * scale
            big = q[a:b, h].abs() @ kh.abs().t() * abs(scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            s = s.masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0) if bool(torch.isfinite(kh).all()) else softmax_seen(s, seen)
            vz = vh.nan_to_num(0, 0, 0)
            o = p @ vz
            for j in torch.nonzero(~torch.isfinite(vh).all(-1)).flatten().tolist():  # by themselves, where seen
                o = o + torch.where(seen[:, j, None], p[:, j, None] * vh[j] - p[:, j, None] * vz[j], 0.0)
            out[a:b, h] = o
            mean[a:b, h] = p.nan_to_num(0.0) @ vz.abs()
            size[a:b, h, 0] = (big.nan_to_num(0, 0, 0) * (p > 2.0 ** -40)).amax(-1) if at.shape[0] else 0.0
    return out.reshape(rows, -1), mean.reshape(rows, -1), size.expand(rows, heads, hd).reshape(rows, -1)


def softmax_seen(s, seen):
    """softmax where a row that sees a score of NaN is NaN, and one that sees nothing zeros."""
    p = torch.softmax(s, -1)
    none = ~(seen & ~(s == -math.inf)).any(-1, keepdim=True)
    return torch.where(none, 0.0, p)


def shared_tol(dtype, bits, hd, keys, out, mean, size, softcap=0.0):
    # A score: hd products and sums of float32 and some ten roundings behind it (codes are exact,
    # their scales are float32); an error of d in a score is one of 2 d in a weight relative to
    # the sum.
    score = (hd + 16) * F * size + 16 * F * (size + 1) + softcap * 2.0 ** -22
    # The weights' rounding for the second product (float32: none; fp16 over codes: two bf16
    # halves), a weight's own roundings, the sums over the keys (half of the keys' number is
    # far more additions than any one sum has in a row), as many joins.
    own = {"f32": 0.0, "f16": U["f16"] if bits == 0 else 2.0 ** -16, "bf16": U["bf16"]}[dtype]
    weights = own + (keys / 2 + 64) * F
    return 1.01 * U[dtype] * out.abs() + (2 * score + weights) * mean * (1 + 2 * own) + weights * F * out.abs() + \
        (keys / 2 + 64) * F * out.abs() + TINY[dtype]


def run_shared(ctx, q, cache, heads, off, fill=7.0, **kw):
    from semantica_gpu import kernels
    dev = {n: (t.cuda() if isinstance(t, torch.Tensor) else t) for n, t in kw.items()}
    out = torch.full(q.shape, fill, dtype=q.dtype, device="cuda")
    kernels.attention_shared(ctx, out, q.cuda(), cache, heads, off.cuda(), **dev)
    return out.cpu()


def ranges(lens, gap=3, first=5):
    """Starts of ranges one after another, and the slots in all."""
    starts = first + np.cumsum(np.concatenate([[0], np.asarray(lens[:-1], np.int64) + gap])) if len(lens) else np.zeros(0)
    return starts.astype(np.int64), int(starts[-1] + lens[-1] + 2) if len(lens) else 1


def check_shared(ctx, seed, dtype, bits, heads, kv_heads, hd, queries, lengths, plens=(), shared=None, first=0, behind=0,
                 by=1.0, poison=None, **kw):
    say("shared", dtype, bits, "heads", heads, kv_heads, "hd", hd, "queries", list(queries)[:6], "lengths",
        list(lengths)[:6], "prefixes", list(plens), kw)
    g = gen(seed)
    off = offsets(queries, first)
    rows = int(off[-1]) + behind
    places, slots = ranges(list(plens) + list(lengths))
    q = rand(g, rows, heads * hd, by=by, dtype=dtype)
    k, v = rand(g, slots, kv_heads * hd, dtype=dtype), rand(g, slots, kv_heads * hd, by=2.0, dtype=dtype)
    if poison is not None:  # what lies around the ranges
        out_of = torch.ones(slots, dtype=torch.bool)
        for s, m in zip(places, list(plens) + list(lengths)):
            out_of[int(s):int(s) + m] = False
        k[out_of], v[out_of] = poison, poison
    cache = make_cache(ctx, slots, kv_heads, hd, dtype, bits)
    keys = dict(starts=ints(places[len(plens):]), lengths=ints(lengths))
    if len(plens):
        if shared is None:
            shared = [0] + [len(queries) * (p + 1) // len(plens) for p in range(len(plens))]
        keys.update(shared=ints(shared), prefix_starts=ints(places[:len(plens)]), prefix_lengths=ints(plens))
    try:
        fill_cache(ctx, cache, k, v)
        got = run_shared(ctx, q, cache, heads, off, **keys, **kw)
    finally:
        cache.close()
    kr, vr = kept_ref(k, kv_heads, bits)[0], kept_ref(v, kv_heads, bits)[0]
    want, mean, size = shared_ref(q, kr, vr, off, heads, kv_heads, **keys, **kw)
    there = torch.zeros(rows, dtype=torch.bool)
    there[first:int(off[-1])] = True
    assert bool((got[~there] == 7.0).all()), "rows of no sequence were written"
    most = max([0] + [int(p) for p in plens]) + max([0] + [int(m) for m in lengths])
    close(got[there], want[there], shared_tol(dtype, bits, hd, most, want, mean, size, kw.get("softcap", 0.0))[there],
          "attention")


MASKS = {
    "causal": {},
    "whole": {"causal": False},
    "scale": {"scale": -0.31},
    "cap": {"softcap": 5.0},
    "window": {"window": 9},
    "window-whole": {"window": 40, "causal": False, "softcap": 30.0},
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("mask", list(MASKS))
def test_shared_masks(gpu_ctx, dtype, bits, mask):
    """Every mask in each form: few pairs of both kinds, many of both, many behind the prefix and few own."""
    for hd, heads, kv_heads in ((64, 4, 2), (128, 3, 1), (256, 3, 1)):
        check_shared(gpu_ctx, hd, dtype, bits, heads, kv_heads, hd, [1, 0, 2, 3], [7, 0, 70, 40], [83], first=3, behind=4,
                     **MASKS[mask])
        check_shared(gpu_ctx, hd + 1, dtype, bits, heads, kv_heads, hd, [33, 40, 64, 70], [33, 45, 64, 170], [150, 31],
                     first=2, behind=1, **MASKS[mask])
        check_shared(gpu_ctx, hd + 2, dtype, bits, heads, kv_heads, hd, [1] * 90, [1 + i % 50 for i in range(90)],
                     [200, 65], **MASKS[mask])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
def test_shared_few_behind_many_prefixes(gpu_ctx, dtype, bits):
    """Few pairs behind each prefix (more prefixes than sequences), many of each sequence."""
    check_shared(gpu_ctx, 1, dtype, bits, 2, 1, 64, [50, 40], [50, 60], [5, 40, 33, 70, 12, 9], shared=[0, 0, 1, 1, 2, 2, 2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_shared_many_rows(gpu_ctx, dtype, bits, hd):
    """More (row, head) than are joined one by one: sequences that fill jobs of their own, whole
    and cut; hundreds of short ones behind shared prefixes, few and many pairs of each."""
    check_shared(gpu_ctx, 1, dtype, bits, 8, 2, hd, [300, 170, 0, 200], [340, 170, 9, 230], [333, 90], first=1, behind=2)
    check_shared(gpu_ctx, 2, dtype, bits, 8, 2, hd, [2] * 170, [2 + i % 40 for i in range(170)], [300, 61, 0])
    check_shared(gpu_ctx, 3, dtype, bits, 8, 2, hd, [1] * 300, [i % 70 for i in range(300)], window=33)
    check_shared(gpu_ctx, 4, dtype, bits, 4, 2, hd, [30] * 20, [60] * 20, [130], causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
def test_shared_long(gpu_ctx, dtype, bits):
    """A prefix split over the GPU for one query, and for a few; running maxima that rise late."""
    check_shared(gpu_ctx, 2, dtype, bits, 8, 2, 128, [1], [3], [20011], by=3.0)
    check_shared(gpu_ctx, 3, dtype, bits, 3, 1, 256, [1, 1, 2], [30, 5, 7], [5000], by=3.0)
    check_shared(gpu_ctx, 4, dtype, bits, 4, 1, 64, [1] * 40, [9] * 40, [6001], by=4.0)
    check_shared(gpu_ctx, 5, dtype, bits, 2, 1, 64, [300], [4001], by=4.0)  # no prefix


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("hd", [8, 40, 72, 136, 200, 248])
def test_shared_odd_head_dims(gpu_ctx, dtype, bits, hd):
    check_shared(gpu_ctx, hd, dtype, bits, 2, 1, hd, [3, 1], [17, 40], [61])
    check_shared(gpu_ctx, hd, dtype, bits, 6, 2, hd, [40, 21], [41, 40], [61])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [0, 8])
def test_shared_edges(gpu_ctx, bits):
    """No own keys, empty prefixes, more queries than keys, sequences behind no prefix, ranges outside the cache."""
    for dtype in ("f32", "bf16"):
        check_shared(gpu_ctx, 1, dtype, bits, 2, 1, 64, [3, 2, 4], [0, 0, 9], [40, 0], shared=[0, 1, 3])
        check_shared(gpu_ctx, 2, dtype, bits, 2, 1, 64, [60, 5], [20, 1], [10], shared=[0, 1])
        check_shared(gpu_ctx, 3, dtype, bits, 2, 1, 64, [60, 5], [20, 1], [10], shared=[0, 1], causal=False, window=4)
        check_shared(gpu_ctx, 4, dtype, bits, 2, 1, 64, [1, 2, 3, 4], [5, 6, 7, 8], [33, 70], shared=[1, 2, 3])
    from semantica_gpu import kernels  # noqa: F401
    g = gen(9)
    k, v, q = rand(g, 64, 64, dtype="f32"), rand(g, 64, 64, dtype="f32"), rand(g, 4, 128, dtype="f32")
    cache = make_cache(gpu_ctx, 64, 1, 64, "f32", bits)
    fill_cache(gpu_ctx, cache, k, v)
    kr, vr = kept_ref(k, 1, bits)[0], kept_ref(v, 1, bits)[0]
    off = offsets([1, 1, 2])
    keys = dict(starts=ints([-1, 60, 10]), lengths=ints([5, 5, 2**31 - 1]), shared=ints([0, 2, 3]),
                prefix_starts=ints([3, 2**31 - 1]), prefix_lengths=ints([20, 20]))
    got = run_shared(gpu_ctx, q, cache, 2, off, **keys)
    want, mean, size = shared_ref(q, kr, vr, off, 2, 1, **keys)
    cache.close()
    assert bool((got[2:] == 0).all())
    close(got, want, shared_tol("f32", bits, 64, 64, want, mean, size), "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_shared_hidden_slots(gpu_ctx, dtype, bits, bad):
    """Infinities and NaN around the ranges, and in later tokens of the same sequence."""
    for queries, lengths in (([1, 2], [7, 40]), ([40, 64], [50, 64])):
        check_shared(gpu_ctx, 3, dtype, bits, 2, 1, 64, queries, lengths, [45], poison=bad)
    # A bad token in the middle of a sequence: earlier queries do not see it, later ones do.
    for n, hd in ((6, 64), (90, 128)):
        g = gen(n)
        q = rand(g, n, 2 * hd, dtype=dtype)
        k, v = rand(g, n + 40, hd, dtype=dtype), rand(g, n + 40, hd, dtype=dtype)
        v[40 + n // 2, 3] = bad
        cache = make_cache(gpu_ctx, n + 40, 1, hd, dtype, bits)
        fill_cache(gpu_ctx, cache, k, v)
        keys = dict(starts=ints([40]), lengths=ints([n]), shared=ints([0, 1]), prefix_starts=ints([1]),
                    prefix_lengths=ints([35]))
        got = run_shared(gpu_ctx, q, cache, 2, offsets([n]), **keys)
        cache.close()
        kr, vr = kept_ref(k, 1, bits)[0], kept_ref(v, 1, bits)[0]
        want, mean, size = shared_ref(q, kr, vr, offsets([n]), 2, 1, **keys)
        assert bool(torch.isfinite(got[:n // 2]).all()) and not bool(torch.isfinite(got[n // 2:]).all(-1).any())
        fin = torch.isfinite(want)
        same(torch.isfinite(got.float()), fin, "which are finite")
        if bits == 0:
            same(got[~fin].double(), want[~fin], "infinities")
        tol = shared_tol(dtype, bits, hd, n + 35, want.nan_to_num(0, 0, 0), mean, size)
        close(got[fin], want[fin], tol[fin], "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
def test_shared_visible_not_finite(gpu_ctx, dtype, bits):
    """A NaN in a key reaches the queries that see it and no others; scores of -infinity alone give zeros."""
    n, hd = 40, 64
    for pick in ("key", "lowest"):
        g = gen(7)
        q, k, v = rand(g, n, hd, dtype=dtype), rand(g, n, hd, dtype=dtype), rand(g, n, hd, dtype=dtype)
        if pick == "key":
            k[11] = math.nan
        elif bits == 0:
            k[:] = -math.inf
            q = q.abs() + dt(dtype).itemsize
        else:
            continue
        cache = make_cache(gpu_ctx, n, 1, hd, dtype, bits)
        fill_cache(gpu_ctx, cache, k, v)
        got = run_shared(gpu_ctx, q, cache, 1, offsets([n]), starts=ints([0]), lengths=ints([n]))
        cache.close()
        if pick == "key":
            assert bool(torch.isfinite(got[:11]).all()) and bool(torch.isnan(got[11:]).all())
        else:
            assert bool((got == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,limit", [("f32", 3e-6), ("f16", 6e-4), ("bf16", 5e-3)])
@pytest.mark.parametrize("bits", [0, 8])
def test_shared_error_norm(gpu_ctx, dtype, limit, bits):
    """The error's norm: a lost half of a weight, or a key counted twice, would show.

    float32: 320 products and scales of a score of size 20 at most, off by about the root of
    their number times f each, 2e-7 absolutely, so 4e-7 in a weight; 16-bit types: their
    output's and their weights' rounding, u / sqrt(3) each."""
    g = gen(11)
    n, hd, plen = 50, 128, 3001
    q = rand(g, n, 4 * hd, dtype=dtype)
    k, v = rand(g, plen + n, hd, dtype=dtype), rand(g, plen + n, hd, dtype=dtype)
    cache = make_cache(gpu_ctx, plen + n, 1, hd, dtype, bits)
    fill_cache(gpu_ctx, cache, k, v)
    kr, vr = kept_ref(k, 1, bits)[0], kept_ref(v, 1, bits)[0]
    for queries, own in (([n], [n]), ([1] * 5, [3] * 5)):
        off = offsets(queries)
        starts = plen + np.concatenate([[0], np.cumsum(own)[:-1]])
        keys = dict(starts=ints(starts), lengths=ints(own), shared=ints([0, len(own)]), prefix_starts=ints([0]),
                    prefix_lengths=ints([plen]))
        rows = int(off[-1])
        got = run_shared(gpu_ctx, q[:rows], cache, 4, off, **keys)
        want, _, _ = shared_ref(q[:rows], kr, vr, off, 4, 1, **keys)
        err = float((got.double() - want).norm() / want.norm())
        say("error", dtype, bits, rows, err)
        assert err < limit
    cache.close()


@pytest.mark.gpu
def test_shared_far_apart_scales(gpu_ctx):
    """Values of far-apart powers of two: a query that sees small ones alone keeps their bits."""
    hd, n = 64, 64
    for dtype in ("f32", "f16", "bf16"):
        for bits in (0, 8):
            g = gen(3)
            q, k, v = rand(g, n, hd, dtype=dtype), rand(g, n, hd, dtype=dtype), rand(g, n, hd, dtype=dtype)
            v[:32] *= 2.0 ** -12 if dtype == "f16" else 2.0 ** -60
            v[32:] *= 2.0 ** 12 if dtype == "f16" else 2.0 ** 60
            cache = make_cache(gpu_ctx, n, 1, hd, dtype, bits)
            fill_cache(gpu_ctx, cache, k, v)
            kr, vr = kept_ref(k, 1, bits)[0], kept_ref(v, 1, bits)[0]
            off = offsets([n])
            got = run_shared(gpu_ctx, q, cache, 1, off, starts=ints([0]), lengths=ints([n]))
            cache.close()
            want, mean, size = shared_ref(q, kr, vr, off, 1, 1, ints([0]), ints([n]))
            close(got, want, shared_tol(dtype, bits, hd, n, want, mean, size), "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("scale", [3e5, 1e9, -1e15])
def test_shared_large_scores(gpu_ctx, dtype, bits, scale):
    """Scores so large that one step of float32 is more than any weight: the keys of the largest share the answer.

    Products of -1, 0 and 1 are whole numbers (times a scale of codes that is the same for all keys), so
    keys tie exactly, their weights are 1, and all others' zero.  What is left is the values' weights'
    rounding (bf16 over codes: half a step, fp16: two halves of bf16), the sums' and the result's."""
    g = gen(17)
    heads, kv_heads, hd, plen = 4, 2, 64, 300
    for queries, lengths in (([1, 2, 1], [40, 3, 70]), ([70, 40], [70, 90])):
        rows, slots = sum(queries), plen + sum(lengths)
        q = torch.randint(-1, 2, (rows, heads * hd), generator=g).to(dt(dtype))
        k = torch.randint(-1, 2, (slots, kv_heads * hd), generator=g).to(dt(dtype))
        v = rand(g, slots, kv_heads * hd, dtype=dtype)
        cache = make_cache(gpu_ctx, slots, kv_heads, hd, dtype, bits)
        fill_cache(gpu_ctx, cache, k, v)
        off = offsets(queries)
        keys = dict(starts=ints(plen + np.concatenate([[0], np.cumsum(lengths)[:-1]])), lengths=ints(lengths),
                    shared=ints([0, len(queries)]), prefix_starts=ints([0]), prefix_lengths=ints([plen]), scale=scale)
        got = run_shared(gpu_ctx, q, cache, heads, off, **keys)
        cache.close()
        kr, vr = kept_ref(k, kv_heads, bits)[0], kept_ref(v, kv_heads, bits)[0]
        want, mean, _ = shared_ref(q, kr, vr, off, heads, kv_heads, **keys)
        own = 0.0 if bits == 0 else {"f32": 0.0, "f16": 2.0 ** -16, "bf16": U["bf16"]}[dtype]
        close(got, want, 1.01 * U[dtype] * want.abs() + (1.01 * own + 400 * F) * mean, "attention")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", [("f32", 0), ("f16", 8), ("bf16", 0)])
def test_shared_lists(gpu_ctx, dtype, bits):
    """A hundred tokens behind one prefix, longer and longer, then with many own keys: the prefix read again
    with every sequence, by itself beside the own keys in narrow jobs and in wide ones, and each in its own."""
    for plen, own in ((300, 40), (3000, 40), (12000, 40), (8000, 1500)):
        check_shared(gpu_ctx, plen, dtype, bits, 4, 1, 64, [1] * 100, [own - i % 30 for i in range(100)], [plen])
    check_shared(gpu_ctx, 5, dtype, bits, 8, 2, 64, [1, 2, 0, 1] * 20, [9, 70, 3, 2] * 20, [2500, 40, 0, 3000], window=1500)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,bits", [("f32", 0), ("bf16", 8)])
def test_shared_many_sequences(gpu_ctx, dtype, bits):
    """Thousands of sequences and hundreds of prefixes: more than a plan keeps at hand."""
    n = 2100
    check_shared(gpu_ctx, 1, dtype, bits, 2, 1, 64, [1] * n, [i % 7 for i in range(n)], [700])
    check_shared(gpu_ctx, 2, dtype, bits, 2, 1, 64, [i % 3 for i in range(n)], [i % 9 for i in range(n)],
                 [p * 13 % 70 for p in range(520)], first=2, behind=3)
    check_shared(gpu_ctx, 3, dtype, bits, 2, 2, 64, [2] * 30, [5] * 30, [40] * 600, shared=[min(p // 15, 30) for p in range(601)],
                 window=20)


# ---- 4-bit weights -------------------------------------------------------------------------


def q4_make(g, out_dim, in_dim, group, scale="f16", zeros=False):
    codes = torch.randint(0, 256, (out_dim, in_dim // 2), generator=g, dtype=torch.uint8)
    scales = ((torch.rand(out_dim, in_dim // group, generator=g) + 0.2) * 0.1).to(dt(scale))
    z = torch.randint(0, 16, (out_dim, in_dim // group), generator=g, dtype=torch.uint8) if zeros else None
    return codes, scales, z


def q4_dense(codes, scales, z):
    w = torch.stack([codes % 16, codes // 16], -1).reshape(codes.shape[0], scales.shape[1], -1).double()
    w = (w - (z.double()[..., None] if z is not None else 8.0)) * scales.double()[..., None]
    return w.reshape(codes.shape[0], -1)


def q4_tol(dtype, x, w, out):
    # The result's rounding; an inner sum of up to 3 * 128 products, the groups' sum, the eight
    # waves': fewer than in_dim / 8 + 400 additions of float32 in a row, and a scaling.
    size = x.double().nan_to_num(0, 0, 0).abs() @ w.abs().t()
    return 1.01 * U[dtype] * out.abs() + (x.shape[1] / 8 + 400) * F * size + TINY[dtype]


def check_q4(ctx, seed, dtype, rows, out_dim, in_dim, group, scale="f16", zeros=False, x=None):
    from semantica_gpu import kernels
    say("q4", dtype, rows, out_dim, in_dim, group, scale, zeros)
    g = gen(seed)
    codes, scales, z = q4_make(g, out_dim, in_dim, group, scale, zeros)
    x = rand(g, rows, in_dim, dtype=dtype) if x is None else x
    wt = kernels.Q4Weight(ctx, codes.cuda(), scales.cuda(), z.cuda() if zeros else None)
    wide = torch.full((rows, out_dim + 5), 7.0, dtype=dt(dtype), device="cuda")
    try:
        kernels.matmul_q4(ctx, wide[:, 3:3 + out_dim], wt, x.cuda())
    finally:
        wt.close()
    w = q4_dense(codes, scales, z)
    want = x.double() @ w.t()
    close(wide[:, 3:3 + out_dim], want, q4_tol(dtype, x, w, want), "products")
    assert bool((wide[:, :3] == 7).all()) and bool((wide[:, 3 + out_dim:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_q4(gpu_ctx, dtype, group, zeros):
    """Rows of each form, outputs that end inside a tile, inputs that end inside a block."""
    for rows, out_dim, groups in ((1, 1, 1), (1, 100, 3), (2, 33, 24), (16, 130, 5), (17, 64, 9), (33, 70, 40),
                                  (64, 16, 2), (130, 49, 7), (5, 16401, 2)):
        check_q4(gpu_ctx, rows, dtype, rows, out_dim, groups * group, group, ("f16", "f32", "bf16")[rows % 3], zeros)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_q4_many_outputs(gpu_ctx, dtype):
    """Two and four tiles of outputs to a workgroup, the last one's in part."""
    for rows, out_dim in ((1, 8200), (3, 8200), (16, 8217), (1, 16390), (3, 16390), (17, 8200), (40, 12000), (700, 770), (530, 250)):
        for group in (32, 64, 128):
            check_q4(gpu_ctx, rows, dtype, rows, out_dim, 384, group, "f16" if rows < 40 else "f32", rows in (3, 40))


@pytest.mark.gpu
def test_q4_exact_weights(gpu_ctx):
    """Weights of zero take nothing, however large the input beside them; float32 rows keep their bits."""
    from semantica_gpu import kernels
    for dtype in ("f32", "f16", "bf16"):
        for rows in (1, 40):
            g = gen(rows)
            codes, scales, _ = q4_make(g, 40, 256, 32)
            codes = codes & 0xf0 | 8  # even inputs' weights are zero
            x = rand(g, rows, 256, dtype=dtype)
            x[:, ::2] = 6e4 if dtype == "f16" else 1e30
            w = q4_dense(codes, scales, None)
            wt = kernels.Q4Weight(gpu_ctx, codes.cuda(), scales.cuda())
            dst = torch.empty(rows, 40, dtype=dt(dtype), device="cuda")
            kernels.matmul_q4(gpu_ctx, dst, wt, x.cuda())
            wt.close()
            want = x.double() @ w.t()
            close(dst, want, q4_tol(dtype, x[:, 1::2], w[:, 1::2], want), "products")
    # One weight a row: the product's own rounding and no other.
    g = gen(1)
    codes = torch.full((32, 64), 0x88, dtype=torch.uint8)
    codes[:, 0] = 0x89  # weight one for input 0
    x = torch.zeros(16, 128)
    x[:, 0] = torch.randn(16, generator=g) * 2.0 ** torch.arange(-120, 120, 15).float()
    wt = kernels.Q4Weight(gpu_ctx, codes.cuda(), torch.ones(32, 4, device="cuda"))
    dst = torch.empty(16, 32, device="cuda")
    kernels.matmul_q4(gpu_ctx, dst, wt, x.cuda())
    wt.close()
    # Parts of eight bits: the third holds what lies 16 to 23 places below the first bit, the second
    # 8 to 15, and a part is lost where it falls below bf16's smallest normal number (as part of
    # a subnormal or for a matrix core that takes those as zeros).  So nothing is lost of an input of
    # 2^-102 or more, and less than 2^-126 by each of two parts of a smaller one.
    want = x[:, :1].expand(16, 32)
    big = want.abs() >= 2.0 ** -102
    same(dst.cpu()[big], want[big], "float32 rows")
    assert bool(((dst.cpu().double() - want.double()).abs() <= 2.0 ** -125).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_q4_not_finite(gpu_ctx, dtype):
    """An infinity or a NaN is its row's alone; an infinity times a weight that is not zero is one."""
    from semantica_gpu import kernels
    g = gen(5)
    codes, scales, _ = q4_make(g, 48, 128, 64)
    codes[:, 3] = 0x9f  # weights 7 and 1 for inputs 6 and 7
    x = rand(g, 20, 128, dtype=dtype)
    x[4, 6], x[9, 11] = math.inf, math.nan
    wt = kernels.Q4Weight(gpu_ctx, codes.cuda(), scales.cuda())
    dst = torch.empty(20, 48, dtype=dt(dtype), device="cuda")
    kernels.matmul_q4(gpu_ctx, dst, wt, x.cuda())
    wt.close()
    got = dst.cpu().float()
    assert bool((got[4] == math.inf).all()) and bool(torch.isnan(got[9]).all())
    rest = torch.ones(20, dtype=torch.bool)
    rest[4] = rest[9] = False
    w = q4_dense(codes, scales, None)
    want = x[rest].double() @ w.t()
    close(got[rest], want, q4_tol(dtype, x[rest], w, want), "products")


@pytest.mark.gpu
def test_q4_from_gguf_blocks(gpu_ctx):
    """Raw Q4_0 blocks: the same products as their codes and scales."""
    from semantica_gpu import kernels
    r = np.random.RandomState(3)
    out_dim, in_dim = 50, 224
    d = (r.uniform(0.001, 0.1, (out_dim, in_dim // 32)) * r.choice([-1, 1], (out_dim, in_dim // 32))).astype(np.float16)
    q = r.randint(0, 16, (out_dim, in_dim // 32, 32)).astype(np.uint8)
    raw = np.concatenate([d[..., None].view(np.uint8), q[..., :16] | q[..., 16:] << 4], -1)
    w = torch.from_numpy(((q.astype(np.float64) - 8) * d.astype(np.float64)[..., None]).reshape(out_dim, in_dim))
    x = rand(gen(2), 3, in_dim)
    wt = kernels.Q4Weight.from_q4_0(gpu_ctx, raw, out_dim, in_dim)
    dst = torch.empty(3, out_dim, device="cuda")
    kernels.matmul_q4(gpu_ctx, dst, wt, x.cuda())
    wt.close()
    want = x.double() @ w.t()
    close(dst, want, q4_tol("f32", x, w, want), "products")


# ---- refusals ---------------------------------------------------------------------------


def test_refusals_without_a_gpu():
    """Argument checks come before any device call."""
    from semantica_gpu import _lib
    lib = _lib.load()
    out, size = ctypes.c_void_p(), ctypes.c_size_t()
    bad = _lib.SG_ERR_INVALID
    assert lib.sg_kv_cache_create(None, 10, 1, 64, 0, 8, None, ctypes.byref(out)) == bad
    assert lib.sg_kv_cache_write(None, None, None, 0, None, 0, 1, None, 1, None, None) == bad
    assert lib.sg_kv_cache_read(None, None, None, 0, None, 0, 1, None, 1, None, None) == bad
    assert lib.sg_kv_cache_bytes(None, ctypes.byref(size)) == bad
    assert lib.sg_attention_shared_work_bytes(None, 1, 1, 1, 1, ctypes.byref(size)) == bad
    keys = _lib.SharedKeys()
    assert lib.sg_attention_shared(None, None, 0, None, 0, None, 1, 1, None, 1, keys, None, 0, None) == bad
    assert b"NULL" in lib.sg_last_error()
    lib.sg_kv_cache_free(None)
    assert lib.sg_q4_weight_create(None, None, None, 0, None, 1, 32, 32, None, ctypes.byref(out)) == bad
    assert lib.sg_q4_weight_create_q4_0(None, None, 1, 32, ctypes.byref(out)) == bad
    assert lib.sg_matmul_q4(None, None, 0, None, None, 0, 0, 1, None) == bad
    lib.sg_q4_weight_free(None)


def refused(call, *words):
    from semantica_gpu import _lib
    with pytest.raises((ValueError, _lib.SemanticaError)) as e:
        call()
    assert all(w in str(e.value) for w in words), str(e.value)


@pytest.mark.gpu
def test_refusals(gpu_ctx):
    """What a call cannot do it says, and it leaves the outputs alone."""
    from semantica_gpu import kernels
    bf16, f32 = torch.bfloat16, torch.float32
    refused(lambda: kernels.KVCache(gpu_ctx, 10, 1, 64, torch.int8), "float32")
    refused(lambda: kernels.KVCache(gpu_ctx, 10, 1, 64, bf16, bits=4), "bits 4")
    refused(lambda: kernels.KVCache(gpu_ctx, 0, 1, 64, bf16), "slots 0")
    refused(lambda: kernels.KVCache(gpu_ctx, 10, 0, 64, bf16), "0 key heads")
    for hd in (0, 12, 264):
        refused(lambda: kernels.KVCache(gpu_ctx, 10, 1, hd, bf16), "head_dim")
    cache = kernels.KVCache(gpu_ctx, 40, 2, 64, bf16)
    assert cache.nbytes == 2 * 2 * (2 * 32 * 64 + 256)
    off, starts = offsets([3]).cuda(), ints([0]).cuda()
    k = torch.zeros(3, 128, dtype=bf16, device="cuda")
    refused(lambda: kernels.kv_cache_write(gpu_ctx, cache, k.float(), k, off, starts), "k")
    refused(lambda: kernels.kv_cache_write(gpu_ctx, cache, k[:, :64], k, off, starts), "shape")
    refused(lambda: kernels.kv_cache_write(gpu_ctx, cache, k, k.cpu(), off, starts), "device")
    refused(lambda: kernels.kv_cache_write(gpu_ctx, cache, k, k, off.long(), starts), "offsets")
    refused(lambda: kernels.kv_cache_write(gpu_ctx, cache, k, k, off, ints([0, 1]).cuda()), "starts")
    refused(lambda: kernels.kv_cache_read(gpu_ctx, k, k, cache, off, starts), "overlaps")
    odd = torch.zeros(3, 140, dtype=bf16, device="cuda")
    refused(lambda: kernels.kv_cache_write(gpu_ctx, cache, odd[:, 1:129], k, off, starts), "16")
    q, out = torch.zeros(3, 256, dtype=bf16, device="cuda"), torch.full((3, 256), 7.0, dtype=bf16, device="cuda")
    lengths = ints([3]).cuda()

    def attend(o=out, x=q, heads=4, **kw):
        kernels.attention_shared(gpu_ctx, o, x, cache, heads, off, starts, lengths, **kw)

    refused(lambda: attend(heads=3), "q: shape")
    refused(lambda: attend(o=q), "overlaps")
    refused(lambda: attend(x=q.float()), "q")
    refused(lambda: attend(window=-1), "window")
    refused(lambda: attend(softcap=-1.0), "softcap")
    refused(lambda: attend(scale=math.nan), "scale")
    refused(lambda: attend(scale=1e30), "scale")
    refused(lambda: attend(shared=ints([0, 1]).cuda()), "shared")
    refused(lambda: attend(shared=ints([0, 1]).cuda(), prefix_starts=ints([0, 1]).cuda(), prefix_lengths=ints([1]).cuda()), "prefix_starts")
    size = cache.work_bytes(4, 3, 1, 0)
    refused(lambda: attend(work=torch.empty(size - 1, dtype=torch.uint8, device="cuda")), "work")
    refused(lambda: attend(work=torch.empty(size + 8, dtype=torch.uint8, device="cuda")[8:]), "work")
    refused(lambda: cache.work_bytes(3, 3, 1, 0), "heads")
    refused(lambda: cache.work_bytes(4, -1, 1, 0), "rows")
    for more in ((4, 4, 1, 0), (4, 3, 2, 0), (4, 3, 1, 5)):
        assert cache.work_bytes(*more) >= size
    assert bool((out == 7).all())
    three = kernels.KVCache(gpu_ctx, 40, 3, 64, bf16)
    refused(lambda: kernels.attention_shared(gpu_ctx, out, q, three, 4, off, starts, lengths), "heads")
    three.close()
    cache.close()
    codes, scales = torch.zeros(8, 64, dtype=torch.uint8, device="cuda"), torch.ones(8, 4, dtype=torch.float16, device="cuda")
    refused(lambda: kernels.Q4Weight(gpu_ctx, codes, scales[:, :3]), "scales")
    refused(lambda: kernels.Q4Weight(gpu_ctx, codes, torch.ones(8, 8, device="cuda")), "group 16")
    refused(lambda: kernels.Q4Weight(gpu_ctx, codes.int(), scales), "codes")
    refused(lambda: kernels.Q4Weight(gpu_ctx, codes, scales.double()), "float")
    refused(lambda: kernels.Q4Weight(gpu_ctx, codes, scales, codes), "zeros")
    refused(lambda: kernels.Q4Weight.from_q4_0(gpu_ctx, np.zeros(17, np.uint8), 1, 32), "Q4_0")
    w = kernels.Q4Weight(gpu_ctx, codes, scales)
    x, dst = torch.zeros(2, 128, device="cuda"), torch.zeros(2, 8, device="cuda")
    refused(lambda: kernels.matmul_q4(gpu_ctx, dst, w, x[:, :64]), "x: shape")
    refused(lambda: kernels.matmul_q4(gpu_ctx, dst.half(), w, x), "dst")
    refused(lambda: kernels.matmul_q4(gpu_ctx, x[:, :8], w, x), "overlaps")
    wide = torch.zeros(2, 132, device="cuda")
    refused(lambda: kernels.matmul_q4(gpu_ctx, dst, w, wide[:, 1:129]), "16")
    w.close()
    del f32


@pytest.mark.gpu
def test_nothing_to_do(gpu_ctx):
    """Calls without rows, and sequences without rows."""
    from semantica_gpu import kernels
    cache = make_cache(gpu_ctx, 40, 1, 64, "bf16", 8)
    none = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda")
    off, starts = offsets([0, 0]).cuda(), ints([0, 5]).cuda()
    kernels.kv_cache_write(gpu_ctx, cache, none, none, off, starts)
    kernels.kv_cache_read(gpu_ctx, none, none.clone(), cache, off, starts)
    kernels.attention_shared(gpu_ctx, none, none.clone(), cache, 1, off, starts, ints([3, 3]).cuda())
    some = torch.full((4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    kernels.attention_shared(gpu_ctx, some, some.clone(), cache, 1, off, starts, ints([3, 3]).cuda())
    kernels.kv_cache_read(gpu_ctx, some, some.clone(), cache, off, starts)
    assert bool((some == 7).all())
    w = kernels.Q4Weight(gpu_ctx, torch.zeros(8, 16, dtype=torch.uint8, device="cuda"), torch.ones(8, 1, device="cuda"))
    kernels.matmul_q4(gpu_ctx, torch.zeros(0, 8, device="cuda"), w, torch.zeros(0, 32, device="cuda"))
    w.close()
    cache.close()


# ---- together, and as programs run them -------------------------------------------------------


class Served:
    """A document kept once, and sequences that grow behind it a token at a time."""

    def __init__(self, ctx, dtype, bits, seed, n=5, heads=8, kv_heads=2, hd=64, wide=256, doc=77, room=9):
        from semantica_gpu import kernels
        self.ctx, self.dtype, self.bits, self.n, self.heads, self.kv_heads, self.hd = ctx, dtype, bits, n, heads, kv_heads, hd
        self.g, self.wide, self.doc, self.room = gen(seed), wide, doc, room
        made = {m: q4_make(self.g, c, k, 64, "f16", True)
                for m, (c, k) in {"qkv": ((heads + 2 * kv_heads) * hd, wide), "o": (wide, heads * hd)}.items()}
        self.dense = {m: q4_dense(*v) for m, v in made.items()}
        self.w = {m: kernels.Q4Weight(ctx, *(t.cuda() for t in v)) for m, v in made.items()}
        self.slots = doc + n * room
        self.cache = make_cache(ctx, self.slots, kv_heads, hd, dtype, bits)
        self.kept = torch.zeros(2, self.slots, kv_heads * hd, dtype=dt(dtype))
        self.off, self.starts = offsets([1] * n).cuda(), ints([doc + i * room for i in range(n)]).cuda()
        self.lengths, self.slot = ints([0] * n).cuda(), self.starts.clone()
        self.shared = [ints([0, n]).cuda(), ints([0]).cuda(), ints([doc]).cuda()]
        d = dt(dtype)
        self.x = torch.empty(n, wide, dtype=d, device="cuda")
        self.qkv = torch.empty(n, (heads + 2 * kv_heads) * hd, dtype=d, device="cuda")
        self.att = torch.empty(n, heads * hd, dtype=d, device="cuda")
        self.y = torch.empty(n, wide, dtype=d, device="cuda")
        self.work = torch.empty(self.cache.work_bytes(heads, n, n, 1), dtype=torch.uint8, device="cuda")

    def parts(self, qkv):
        a, b = self.heads * self.hd, (self.heads + self.kv_heads) * self.hd
        return qkv[:, :a], qkv[:, a:b], qkv[:, b:]

    def document(self):
        from semantica_gpu import kernels
        x = rand(self.g, self.doc, self.wide, dtype=self.dtype)
        qkv = torch.empty(self.doc, self.qkv.shape[1], dtype=self.x.dtype, device="cuda")
        kernels.matmul_q4(self.ctx, qkv, self.w["qkv"], x.cuda())
        _, k, v = self.parts(qkv)
        kernels.kv_cache_write(self.ctx, self.cache, k, v, offsets([self.doc]).cuda(), ints([0]).cuda())
        self.kept[0, :self.doc], self.kept[1, :self.doc] = k.cpu(), v.cpu()

    def step(self):
        """One token of each sequence, in the tensors of the object."""
        from semantica_gpu import kernels
        kernels.matmul_q4(self.ctx, self.qkv, self.w["qkv"], self.x)
        q, k, v = self.parts(self.qkv)
        kernels.kv_cache_write(self.ctx, self.cache, k, v, self.off, self.slot)
        self.lengths += 1
        self.slot += 1
        kernels.attention_shared(self.ctx, self.att, q, self.cache, self.heads, self.off, self.starts, self.lengths,
                                 *self.shared, work=self.work)
        kernels.matmul_q4(self.ctx, self.y, self.w["o"], self.att)

    def check(self, t):
        """What step t left, each part from the values that it was given."""
        x, qkv, att, y = (a.cpu() for a in (self.x, self.qkv, self.att, self.y))
        want = x.double() @ self.dense["qkv"].t()
        close(qkv, want, q4_tol(self.dtype, x, self.dense["qkv"], want), "projection")
        q, k, v = self.parts(qkv)
        for i in range(self.n):
            at = self.doc + i * self.room + t
            self.kept[0, at], self.kept[1, at] = k[i], v[i]
        kr, vr = (kept_ref(a, self.kv_heads, self.bits)[0] for a in self.kept)
        lengths = ints([t + 1] * self.n)
        want, mean, size = shared_ref(q, kr, vr, self.off.cpu(), self.heads, self.kv_heads, self.starts.cpu(), lengths,
                                      *(a.cpu() for a in self.shared))
        close(att, want, shared_tol(self.dtype, self.bits, self.hd, self.doc + t + 1, want, mean, size), "attention")
        want = att.double() @ self.dense["o"].t()
        close(y, want, q4_tol(self.dtype, att, self.dense["o"], want), "output")

    def close(self):
        self.cache.close()
        for w in self.w.values():
            w.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
def test_served_tokens(gpu_ctx, dtype, bits):
    """Projection, cache, attention behind a kept document and output, token by token."""
    s = Served(gpu_ctx, dtype, bits, 21)
    s.document()
    for t in range(4):
        s.x.copy_(rand(s.g, s.n, s.wide, dtype=dtype))
        s.step()
        s.check(t)
    s.close()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [0, 8])
def test_served_tokens_by_a_replayed_graph(gpu_ctx, bits):
    """One captured step serves every token: lengths and slots are read on the device.  Eager work
    and synchronizations lie between the replays, and a cache that is dropped meanwhile is kept
    until the capture is over."""
    from semantica_gpu import kernels
    s = Served(gpu_ctx, "bf16", bits, 22)
    s.document()
    s.x.zero_()
    s.step()  # (first calls ask for their LDS)
    s.lengths.zero_()
    s.slot.copy_(s.starts)
    torch.cuda.synchronize()
    dropped = kernels.KVCache(gpu_ctx, 10, 1, 64, torch.bfloat16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        del dropped
        s.step()
    for t in range(6):
        s.x.copy_(rand(s.g, s.n, s.wide, dtype="bf16"))
        graph.replay()
        torch.cuda.synchronize()
        s.check(t)
        got = s.att.clone()
        q, _, _ = s.parts(s.qkv)
        again = torch.empty_like(s.att)
        kernels.attention_shared(gpu_ctx, again, q, s.cache, s.heads, s.off, s.starts, s.lengths, *s.shared)
        same(again, got, "eager and replayed")
    s.close()


@pytest.mark.gpu
def test_streams_and_threads(gpu_ctx):
    """Calls on streams of their own at once, from threads, with the default workspace and one of
    their own: the bits of a call by itself."""
    import threading
    from semantica_gpu import kernels
    g = gen(31)
    n, heads, kv_heads, hd, plen = 40, 8, 2, 128, 4000
    k, v = rand(g, plen + n, kv_heads * hd, dtype="f16"), rand(g, plen + n, kv_heads * hd, dtype="f16")
    cache = make_cache(gpu_ctx, plen + n, kv_heads, hd, "f16", 8)
    fill_cache(gpu_ctx, cache, k, v)
    qs = [rand(g, n, heads * hd, dtype="f16").cuda() for _ in range(4)]
    off, starts, lengths = offsets([1] * n).cuda(), ints(range(plen, plen + n)).cuda(), ints([1] * n).cuda()
    shared = [ints([0, n]).cuda(), ints([0]).cuda(), ints([plen]).cuda()]
    want = []
    for q in qs:
        want.append(torch.empty_like(q))
        kernels.attention_shared(gpu_ctx, want[-1], q, cache, heads, off, starts, lengths, *shared)
    torch.cuda.synchronize()
    got = [[torch.empty_like(q) for _ in range(5)] for q in qs]
    errors = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            own = torch.empty(cache.work_bytes(heads, n, n, 1), dtype=torch.uint8, device="cuda")
            torch.cuda.synchronize()
            for j, out in enumerate(got[i]):
                if j % 2:
                    kernels.attention_shared(gpu_ctx, out, qs[i], cache, heads, off, starts, lengths, *shared, work=own,
                                             stream=stream.cuda_stream)
                else:
                    kernels.attention_shared(gpu_ctx, out, qs[i], cache, heads, off, starts, lengths, *shared,
                                             stream=stream.cuda_stream)
            stream.synchronize()
        except Exception as e:  # pragma: no cover
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for w, outs in zip(want, got):
        for o in outs:
            same(o, w, "beside other calls")
    cache.close()


@pytest.mark.gpu
def test_numbers_that_make_no_sense(gpu_ctx):
    """Offsets, starts and lengths of any value: nothing outside the tensors is touched."""
    from semantica_gpu import kernels
    r = np.random.RandomState(4)
    rows, slots, heads, kv_heads, hd, n, n_prefix = 50, 100, 4, 2, 64, 12, 3
    for bits in (0, 8):
        cache = make_cache(gpu_ctx, slots, kv_heads, hd, "bf16", bits)
        pool = torch.full((rows + 2, heads * hd), 7.0, dtype=torch.bfloat16, device="cuda")
        k = torch.full((rows + 2, kv_heads * hd), 7.0, dtype=torch.bfloat16, device="cuda")
        v = k.clone()
        q = torch.randn(rows, heads * hd, device="cuda").bfloat16()
        for trial in range(30):
            def some(m):
                lim = int(r.choice([60, 200, 2**31 - 1]))
                return ints(r.randint(-lim, lim, m)).cuda()
            say("trial", bits, trial)
            off, starts, lengths, shared = some(n + 1), some(n), some(n), some(n_prefix + 1)
            kernels.kv_cache_write(gpu_ctx, cache, q[:, :128], q[:, 128:], off, starts)
            kernels.kv_cache_read(gpu_ctx, k[1:-1], v[1:-1], cache, off, starts)
            kernels.attention_shared(gpu_ctx, pool[1:-1], q, cache, heads, off, starts, lengths, shared, some(n_prefix),
                                     some(n_prefix), window=int(r.choice([0, 5])), causal=bool(r.randint(2)))
            torch.cuda.synchronize()
        for t in (pool, k, v):
            assert bool((t[0] == 7).all()) and bool((t[-1] == 7).all())
        cache.close()


@pytest.mark.gpu
def test_slots_past_32_bits(gpu_ctx):
    """A cache of 20 GB: the last slots of the last head lie past every 32-bit offset."""
    from semantica_gpu import kernels
    slots, kv_heads, hd, n = 1_250_000, 8, 256, 70
    cache = make_cache(gpu_ctx, slots, kv_heads, hd, "f32", 0)
    assert cache.nbytes > 2**34
    g = gen(41)
    k, v, q = rand(g, n, kv_heads * hd), rand(g, n, kv_heads * hd), rand(g, n, kv_heads * hd)
    off, starts = offsets([n]).cuda(), ints([slots - n]).cuda()
    kernels.kv_cache_write(gpu_ctx, cache, k.cuda(), v.cuda(), off, starts)
    ko, vo = torch.empty_like(k).cuda(), torch.empty_like(v).cuda()
    kernels.kv_cache_read(gpu_ctx, ko, vo, cache, off, starts)
    same(ko, k, "keys")
    same(vo, v, "values")
    for queries in ([n], [1]):
        rows = sum(queries)
        got = run_shared(gpu_ctx, q[:rows], cache, kv_heads, offsets(queries), starts=ints([slots - n]), lengths=ints([n]))
        want, mean, size = shared_ref(q[:rows], k.double(), v.double(), offsets(queries), kv_heads, kv_heads, ints([0]), ints([n]))
        close(got, want, shared_tol("f32", 0, hd, n, want, mean, size), "attention")
    cache.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_shared_columns_of_wider_tensors(gpu_ctx, dtype):
    """q as columns of a projection, out as columns of a wider tensor, rows far apart."""
    from semantica_gpu import kernels
    g = gen(6)
    heads, kv_heads, hd = 3, 1, 72
    for queries, lengths in (([2, 1], [20, 5]), ([50, 13], [50, 33])):
        off = offsets(queries)
        rows = int(off[-1])
        wide = rand(g, rows, heads * hd + 40, dtype=dtype).cuda()
        out = torch.full((rows, heads * hd + 16), 7.0, dtype=dt(dtype), device="cuda")
        k, v = rand(g, 100, hd, dtype=dtype), rand(g, 100, hd, dtype=dtype)
        cache = make_cache(gpu_ctx, 100, kv_heads, hd, dtype, 0)
        fill_cache(gpu_ctx, cache, k, v)
        keys = dict(starts=ints([3, 60]), lengths=ints(lengths))
        kernels.attention_shared(gpu_ctx, out[:, 8:8 + heads * hd], wide[:, 32:32 + heads * hd], cache, heads, off.cuda(),
                                 **{n: t.cuda() for n, t in keys.items()})
        cache.close()
        want, mean, size = shared_ref(wide[:, 32:32 + heads * hd].cpu(), k.double(), v.double(), off, heads, kv_heads, **keys)
        close(out[:, 8:8 + heads * hd], want, shared_tol(dtype, 0, hd, 60, want, mean, size), "attention")
        assert bool((out[:, :8] == 7).all()) and bool((out[:, 8 + heads * hd:] == 7).all())
