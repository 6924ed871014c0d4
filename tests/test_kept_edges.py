"""Kept keys and values and 4-bit products where their answers are easiest to lose: NaN of every
payload, infinities beside scores of any size, rows by the hundred thousand, workspaces to the
byte, first calls inside a capture.
"""
import ctypes
import math
import os
import subprocess
import sys

import numpy as np
import pytest

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None

from test_kept_ops import (close, dt, fill_cache, gen, ints, kept_ref, make_cache, offsets, q4_dense, q4_make, q4_tol, rand,
                           read_cache, run_shared, same, say, shared_ref, shared_tol)


# Quiet and signalling, of both signs, payloads in either half of the bits.
NANS = (0x7f800001, 0xff800001, 0x7f80ffff, 0x7f810000, 0x7fc00000, 0xffc00001, 0x7fffffff)


def nan_of(bits):
    return torch.from_numpy(np.array([bits], np.uint32).view(np.int32)).view(torch.float32)


@pytest.mark.gpu
def test_q4_nan_of_any_payload(gpu_ctx):
    """A NaN is a NaN in every result of its row; the other rows are as they would be."""
    from semantica_gpu import kernels
    g = gen(5)
    for rows, out_dim, group in ((8, 48, 64), (40, 33, 32), (40, 16400, 128)):
        codes, scales, _ = q4_make(g, out_dim, 256, group)
        x = rand(g, rows, 256)
        for i, bits in enumerate(NANS):
            x.view(torch.int32)[i, 37 * i + 1] = nan_of(bits).view(torch.int32)
        assert bool(torch.isnan(x).any(-1)[:len(NANS)].all())
        wt = kernels.Q4Weight(gpu_ctx, codes.cuda(), scales.cuda())
        dst = torch.empty(rows, out_dim, device="cuda")
        kernels.matmul_q4(gpu_ctx, dst, wt, x.cuda())
        wt.close()
        assert bool(torch.isnan(dst[:len(NANS)]).all()), "a NaN was lost"
        w = q4_dense(codes, scales, None)
        want = x[len(NANS):].double() @ w.t()
        close(dst[len(NANS):], want, q4_tol("f32", x[len(NANS):], w, want), "products")


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_shared_query_nan_of_any_payload(gpu_ctx, bits, sign):
    """A NaN in a query makes its row of that head NaN, whichever sign the keys have there, and no other row."""
    g = gen(6)
    for hd, queries, n in ((64, 9, 70), (128, 150, 300), (256, 9, 40), (256, 100, 150)):
        q, k, v = rand(g, queries, 2 * hd), rand(g, n, hd), rand(g, n, hd)
        for i, b in enumerate(NANS):
            q.view(torch.int32)[i, 5 * i + 3] = nan_of(b).view(torch.int32)
            k[:, 5 * i + 3] = sign * (0.5 + k[:, 5 * i + 3].abs())
        cache = make_cache(gpu_ctx, n, 1, hd, "f32", bits)
        fill_cache(gpu_ctx, cache, k, v)
        off, keys = offsets([queries]), dict(starts=ints([0]), lengths=ints([n]))
        got = run_shared(gpu_ctx, q, cache, 2, off, **keys)
        cache.close()
        m = len(NANS)
        assert bool(torch.isnan(got[:m, :hd]).all()), "a NaN was lost"
        kr, vr = kept_ref(k, 1, bits)[0], kept_ref(v, 1, bits)[0]
        want, mean, size = shared_ref(q.nan_to_num(0.0), kr, vr, off, 2, 1, **keys)
        tol = shared_tol("f32", bits, hd, n, want, mean, size)
        close(got[m:], want[m:], tol[m:], "other rows")
        close(got[:m, hd:], want[:m, hd:], tol[:m, hd:], "other heads")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rise", [20.0, 200.0])
def test_shared_infinite_values_anywhere(gpu_ctx, dtype, rise):
    """An infinity in a value that is seen is the dim's result, wherever the large scores lie: before it,
    behind it, in another piece; a NaN where both infinities are seen.

    Scores are 0 but for two keys of `rise` in powers of e: their weights are 2^29 or 2^288 times the
    infinite value's, which falls below float32 and, as a number of 64 bits, not below zero."""
    g = gen(23)
    hd, heads = 64, 2
    for queries, plen, n in (([3], 0, 200), ([1, 2], 9000, 70), ([100], 0, 700), ([90, 70], 1500, 130)):
        slots = plen + n * len(queries)
        rows = sum(queries)
        q = torch.zeros(rows, heads * hd, dtype=dt(dtype))
        q[:, ::hd] = 1.0
        k, v = torch.zeros(slots, hd, dtype=dt(dtype)), rand(g, slots, hd, dtype=dtype)
        keys = dict(starts=ints([plen + i * n for i in range(len(queries))]), lengths=ints([n] * len(queries)), causal=False,
                    scale=1.0)
        if plen:
            keys.update(shared=ints([0, len(queries)]), prefix_starts=ints([0]), prefix_lengths=ints([plen]))
        first = [plen + i * n for i in range(len(queries))]
        last = [plen + i * n + n - 1 for i in range(len(queries))]
        for name, large, plus, minus in (
                ("before", [0] + first, last, []), ("behind", last, [0] + first, []),
                ("between", [slots // 2] + [f + n // 2 for f in first], [0] + first + last, []),
                ("both", [slots // 2] + [f + n // 2 for f in first], [0] + first, last)):
            kk, vv = k.clone(), v.clone()
            kk[large, 0] = rise
            vv[plus, 3], vv[minus, 3] = math.inf, -math.inf
            cache = make_cache(gpu_ctx, slots, 1, hd, dtype, 0)
            fill_cache(gpu_ctx, cache, kk, vv)
            off = offsets(queries)
            say("infinite", name, dtype, rise, queries, plen, n)
            got = run_shared(gpu_ctx, q, cache, heads, off, **keys)
            cache.close()
            dim = got.reshape(rows, heads, hd)[:, :, 3].float()
            if name == "both":
                assert bool(torch.isnan(dim).all())
            else:
                assert bool((dim == math.inf).all()), f"{name}: {dim.flatten()[:8]}"
            vv[plus, 3], vv[minus, 3] = 0.0, 0.0
            want, mean, size = shared_ref(q, kk.double(), vv.double(), off, heads, 1, **keys)
            rest = torch.ones(heads * hd, dtype=torch.bool)
            rest[3::hd] = False
            tol = shared_tol(dtype, 0, hd, plen + n, want, mean, size)
            if dtype == "f16":
                # A weight of fp16 is a multiple of 2^-24 after its factor of 2^6: off by 2^-31 of the largest, in
                # the sum of the weights as in that of the values.
                tol = tol + (plen + n) * 2.0 ** -31 * (vv.double().abs().max() + want.abs())
            close(got[:, rest], want[:, rest], tol[:, rest], "other dims")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_shared_infinite_values_of_hopeless_keys(gpu_ctx, dtype):
    """A value counts if its key is seen, though its score be -infinity: the infinity is the dim's
    result in every cut of the work, unless no score is above -infinity (zeros)."""
    g = gen(24)
    hd = 64
    for queries, n in ((1, 5), (1, 3000), (60, 500)):
        q = torch.zeros(queries, hd, dtype=dt(dtype))
        q[:, 0] = 1.0
        for at in (0, 1, n // 2, n - 1):
            k, v = torch.zeros(n, hd, dtype=dt(dtype)), rand(g, n, hd, dtype=dtype)
            low = slice(at // 32 * 32, min(n - 1, at // 32 * 32 + 32)) if n > 32 else slice(at, at + 1)
            k[low, 0] = -math.inf
            v[at, 3] = math.inf
            cache = make_cache(gpu_ctx, n, 1, hd, dtype, 0)
            fill_cache(gpu_ctx, cache, k, v)
            keys = dict(starts=ints([0]), lengths=ints([n]), causal=False)
            got = run_shared(gpu_ctx, q, cache, 1, offsets([queries]), **keys).float()
            assert bool((got[:, 3] == math.inf).all()), (n, at, got[:, 3])
            got[:, 3] = 0
            assert bool(torch.isfinite(got).all())
            k[:, 0] = -math.inf
            fill_cache(gpu_ctx, cache, k, v)
            got = run_shared(gpu_ctx, q, cache, 1, offsets([queries]), **keys)
            cache.close()
            assert bool((got == 0).all()), "only scores of -infinity"


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [1, 60])
def test_shared_nan_values_of_hopeless_keys(gpu_ctx, queries):
    """Codes: a key whose score is -infinity has no weight, whatever its value holds, in a tile that is seen
    whole and in one that is seen in part; with any other score a value's NaN is the row's."""
    g = gen(25)
    hd = 64
    q = torch.zeros(queries, hd)
    q[:, 0] = 1e25
    for n, at in ((32, 7), (64, 40), (5, 2), (45, 40), (90, 3)):
        k, v = torch.zeros(n + 3, hd), rand(g, n + 3, hd)
        v[at, 9] = math.nan
        v[n + 1, 9] = math.nan  # behind what is seen
        cache = make_cache(gpu_ctx, n + 3, 1, hd, "f32", 8)
        fill_cache(gpu_ctx, cache, k, v)
        off, keys = offsets([queries]), dict(starts=ints([0]), lengths=ints([n]), causal=False)
        got = run_shared(gpu_ctx, q, cache, 1, off, **keys)
        assert bool(torch.isnan(got).all()), (n, at)
        k[at, 0] = -1e15  # a score of -1e40
        fill_cache(gpu_ctx, cache, k, v)
        got = run_shared(gpu_ctx, q, cache, 1, off, **keys)
        cache.close()
        assert bool(torch.isfinite(got).all()), (n, at)
        v[at], v[n + 1] = 0.0, 0.0
        want, mean, size = shared_ref(q, kept_ref(k, 1, 8)[0], kept_ref(v, 1, 8)[0], off, 1, 1, **keys)
        close(got, want, shared_tol("f32", 8, hd, n, want, mean, size), "attention")


def check_many_rows(ctx, seed, dtype, bits, kv_heads, hd, lens, starts, slots, first=0, behind=0):
    """Rows in and out, bit for bit; the later of two sequences keeps a slot."""
    from semantica_gpu import kernels
    say("many rows", dtype, bits, "heads", kv_heads, "hd", hd, "sequences", len(lens), "rows", int(np.sum(lens)), "slots", slots)
    g = gen(seed)
    off = offsets(lens, first)
    rows = int(off[-1]) + behind
    k, v = rand(g, rows, kv_heads * hd, by=3.0, dtype=dtype), rand(g, rows, kv_heads * hd, dtype=dtype)
    kr, vr = kept_ref(k, kv_heads, bits)[1], kept_ref(v, kv_heads, bits)[1]
    seq = np.repeat(np.arange(len(lens)), lens)
    row = np.arange(first, int(off[-1]))
    at = np.asarray(starts, np.int64)[seq] + row - off.numpy()[seq]
    there = (np.asarray(starts)[seq] >= 0) & (at < slots)
    owner = np.full(slots, -1)
    np.maximum.at(owner, at[there], row[there])  # rows of later sequences are higher
    owner = torch.from_numpy(owner)

    def kept(x):
        return torch.where((owner >= 0)[:, None], x[owner.clamp_min(0)], torch.zeros((), dtype=x.dtype))

    def back(x):
        y = torch.full_like(x, 7.0)
        seen = kept(x)[torch.from_numpy(np.where(there, at, 0))]
        y[first:int(off[-1])] = torch.where(torch.from_numpy(there)[:, None], seen, torch.zeros((), dtype=x.dtype))
        return y

    cache = make_cache(ctx, slots, kv_heads, hd, dtype, bits)
    try:
        kernels.kv_cache_write(ctx, cache, k.cuda(), v.cuda(), off.cuda(), ints(starts).cuda())
        out_k, out_v = torch.full_like(k, 7.0).cuda(), torch.full_like(v, 7.0).cuda()
        kernels.kv_cache_read(ctx, out_k, out_v, cache, off.cuda(), ints(starts).cuda())
        got_k, got_v = read_cache(ctx, cache)
    finally:
        cache.close()
    same(got_k, kept(kr), "keys")
    same(got_v, kept(vr), "values")
    same(out_k, back(kr), "keys read")
    same(out_v, back(vr), "values read")


def parts_of(r, rows, n):
    """Lengths of n sequences of so many rows, some of them empty."""
    cuts = np.sort(r.randint(0, rows + 1, n - 1))
    return np.diff(np.concatenate([[0], cuts, [rows]]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("kv_heads,hd,rows", [(8, 64, 17003), (3, 24, 45001), (9, 16, 44017), (1, 64, 140003), (1, 8, 530011)])
def test_rows_of_several_blocks_and_heads_a_workgroup(gpu_ctx, dtype, bits, kv_heads, hd, rows):
    """Workgroups that go over several heads, the last of them fewer, or over several blocks of rows:
    ends inside a block, gaps, slots named twice, starts and ends outside the cache."""
    r = np.random.RandomState(kv_heads * hd)
    # One after another with odd gaps; the last sequences before the cache, past it and over earlier ones.
    lens = parts_of(r, rows, 37)
    starts = np.cumsum(lens) - lens + 5 * np.arange(37) + 3
    slots = int(starts[-1] + lens[-1] + 40)
    starts[30], starts[33] = -2, starts[33] + 41
    starts[32] = slots - 5
    starts[34:] = np.maximum(starts[[1, 9, 20]] + 7, 0)
    check_many_rows(gpu_ctx, rows, dtype, bits, kv_heads, hd, lens, starts, slots, first=3, behind=29)
    # In whole, from a slot within a run of four, to the cache's last one.
    check_many_rows(gpu_ctx, rows + 1, dtype, bits, kv_heads, hd, [rows], [1], rows + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [0, 8])
def test_many_single_rows(gpu_ctx, bits):
    """Tens of thousands of tokens, each a sequence: slots in any order, some named by several."""
    r = np.random.RandomState(3)
    n = 17000
    check_many_rows(gpu_ctx, 4, "bf16", bits, 8, 64, [1] * n, r.randint(-3, 20000, n), 19990)


@pytest.mark.gpu
def test_workspace_to_the_byte(gpu_ctx):
    """Calls stay inside the bytes that they ask for, also those of a larger batch's workspace or of a smaller
    call in it, whatever the plan takes; without prefixes no (row, head) has a place of its own there."""
    from semantica_gpu import kernels
    g = gen(30)
    for dtype, bits, hd, heads, kv_heads in (("bf16", 8, 128, 4, 2), ("f32", 0, 64, 3, 1), ("f16", 0, 256, 8, 1), ("f32", 8, 256, 4, 2)):
        slots = 4000
        cache = make_cache(gpu_ctx, slots, kv_heads, hd, dtype, bits)
        fill_cache(gpu_ctx, cache, rand(g, slots, kv_heads * hd, dtype=dtype), rand(g, slots, kv_heads * hd, dtype=dtype))
        for queries, prefixes in (([1], 0), ([1], 1), ([1] * 60, 1), ([1] * 60, 3), ([300], 1), ([300, 1, 40], 1), ([40] * 20, 1),
                                  ([700, 300], 0), ([2] * 400, 2), ([129] * 9, 4)):
            rows, n = sum(queries), len(queries)
            keys = dict(starts=ints([i * 3 for i in range(n)]).cuda(), lengths=ints([m + 5 for m in queries]).cuda())
            if prefixes:
                keys.update(shared=ints([n * p // prefixes for p in range(prefixes + 1)]).cuda(),
                            prefix_starts=ints([1500 + 13 * p for p in range(prefixes)]).cuda(),
                            prefix_lengths=ints([2000 >> (p % 3 * 3) for p in range(prefixes)]).cuda())
            q, off = rand(g, rows, heads * hd, dtype=dtype).cuda(), offsets(queries).cuda()
            need = cache.work_bytes(heads, rows, n, prefixes)
            assert need <= cache.work_bytes(heads, rows + 1, n, prefixes) and need <= cache.work_bytes(heads, rows, n + 1, prefixes)
            assert need <= cache.work_bytes(heads, rows, n, prefixes + 1)
            say("workspace", dtype, bits, hd, "queries", queries[:3], n, "prefixes", prefixes, need)
            outs = []
            for size in (need, cache.work_bytes(heads, rows + 999, n + 7, prefixes + 1)):
                buf = torch.full((size + 512,), 0xa5, dtype=torch.uint8, device="cuda")
                out = torch.empty_like(q)
                kernels.attention_shared(gpu_ctx, out, q, cache, heads, off, work=buf[256:256 + size], **keys)
                assert bool((buf[:256] == 0xa5).all()) and bool((buf[256 + need:] == 0xa5).all()), "bytes around the workspace"
                outs.append(out)
            same(outs[1], outs[0], "in a larger workspace")
        cache.close()


@pytest.mark.gpu
def test_workspace_of_large_batches(gpu_ctx):
    """It grows with the rows that a plan may leave apart: none without prefixes, and so many of each
    sequence behind one, not with every row of long prompts."""
    cache = make_cache(gpu_ctx, 64, 8, 128, "bf16", 0)
    own = 16384 * 32 * 128 * 4  # a float32 output of every (row, head)
    beside = cache.work_bytes(32, 16384, 32, 0)
    behind = cache.work_bytes(32, 16384, 32, 1)
    short = cache.work_bytes(32, 16384, 16384, 1)
    cache.close()
    assert beside < 110e6
    assert beside < behind < beside + 2.1 * own / 4
    assert short > 2 * own




@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads", [1, 2, 3, 5, 8, 9, 17, 1000])
def test_rows_up_to_the_launch(gpu_ctx, kv_heads):
    """rows * n_kv_heads up to 2^30 is no reason to refuse a call, and what one launch does not take is.  (Rows that
    are not aligned are refused behind that check and before anything is done.)"""
    from semantica_gpu import _lib
    lib = gpu_ctx.lib
    k = torch.zeros(64, device="cuda")
    off, starts = ints([0, 1]).cuda(), ints([0]).cuda()

    def says(cache, rows):
        r = lib.sg_kv_cache_write(gpu_ctx.handle, cache.handle, ctypes.c_void_p(k.data_ptr() + 8), 16 * kv_heads,
                                  ctypes.c_void_p(k.data_ptr()), 16 * kv_heads, rows, ctypes.c_void_p(off.data_ptr()), 1,
                                  ctypes.c_void_p(starts.data_ptr()), None)
        assert r == _lib.SG_ERR_INVALID
        return lib.sg_last_error().decode()

    for dtype in ("f32", "bf16"):
        for bits in (0, 8):
            cache = make_cache(gpu_ctx, 8, kv_heads, 8, dtype, bits)
            try:
                # Workgroups of 256 threads take 16 rows of float32 as it is and 32 of others, of up to eight heads.
                assert "16-byte aligned" in says(cache, 2**30 // kv_heads)
                blocks = 16 if dtype == "f32" and bits == 0 else 32
                if kv_heads >= 8:
                    most = (2**24 - 1) // -(-kv_heads // 8) * blocks
                    if most < 2**31 - 2**16:
                        assert "16-byte aligned" in says(cache, most)
                        assert "launch" in says(cache, most + 1)
            finally:
                cache.close()


FIRST_CALLS = r"""
import sys
sys.path.insert(0, sys.argv[1])
import torch
from semantica_gpu import Context, kernels
ctx = Context(0)
dev = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
torch.manual_seed(1)
for dtype in (torch.float32, torch.float16, torch.bfloat16):
    for hd in (64, 128, 256):
        for bits in (0, 8):
            for queries in (2, 150):  # narrow jobs, wide ones
                n = queries + 200
                cache = kernels.KVCache(ctx, n, 1, hd, dtype, bits=bits)
                w = kernels.Q4Weight(ctx, torch.randint(0, 256, (hd, hd // 2), dtype=torch.uint8, device="cuda"),
                                     torch.rand(hd, hd // 32, device="cuda").half())
                k, v, q = (torch.randn(m, hd, device="cuda").to(dtype) for m in (n, n, queries))
                o, y, kb, vb = (torch.zeros_like(t) for t in (q, q, k, v))
                work = torch.empty(cache.work_bytes(1, queries, 1, 0), dtype=torch.uint8, device="cuda")
                every, some, zero, length = dev(0, n), dev(0, queries), dev(0), dev(n)

                def step():
                    kernels.kv_cache_write(ctx, cache, k, v, every, zero)
                    kernels.kv_cache_read(ctx, kb, vb, cache, every, zero)
                    kernels.attention_shared(ctx, o, q, cache, 1, some, zero, length, work=work)
                    kernels.matmul_q4(ctx, y, w, o)

                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step()
                for t in range(3):
                    k.normal_(), v.normal_(), q.normal_()
                    graph.replay()
                    torch.cuda.synchronize()
                    got = [x.clone() for x in (o, y, kb, vb)]
                    for x in (o, y, kb, vb):
                        x.zero_()
                    step()
                    torch.cuda.synchronize()
                    for x, a in zip((o, y, kb, vb), got):
                        assert bool((x == a).all()) and bool(torch.isfinite(a).all()) and bool((a != 0).any())
                cache.close()
                w.close()
            print(dtype, hd, bits, flush=True)
ctx.close()
print("first calls captured", flush=True)
"""


@pytest.mark.gpu
def test_first_calls_inside_a_capture():
    """A program's first call of each kernel may be the one that it captures: in a process of its own."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "go-semantica_amd")
    r = subprocess.run([sys.executable, "-u", "-c", FIRST_CALLS, at], capture_output=True, text=True, timeout=110)
    say(r.stdout[-2000:], r.stderr[-2000:])
    assert r.returncode == 0 and "first calls captured" in r.stdout
