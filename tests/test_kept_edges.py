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
