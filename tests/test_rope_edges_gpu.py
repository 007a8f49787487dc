"""Edges of the rotary append into a paged cache."""
from __future__ import annotations

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import paged_oracle as R
import tasft_b200 as T

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = Path(__file__).resolve().parent.parent

# the first call of a process, which no earlier one has given a larger limit
WIDE = """
import sys
import torch
import tasft_b200 as T
rot, dtype, mixed = int(sys.argv[1]), getattr(torch, sys.argv[2]), sys.argv[3] == "mixed"
x = torch.ones(3, 4, 256, device="cuda").to(dtype)
kp, vp = (torch.zeros(1, 16, 1, 256, device="cuda", dtype=dtype) for _ in range(2))
ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
freq, _ = T.rope_inv_freq(rot, device="cuda")
out, _ = T.rope_append_paged(x[:, :2], x[:, 2:3], x[:, 3:], freq, kp, vp, ints(0).view(1, 1), ints(0, 3), ints(3), 3,
                             interleaved=mixed)
torch.cuda.synchronize()
assert torch.equal(out[0], x[0, :2]) and torch.equal(vp[0, :3, 0], x[:, 3]) and (out[1] != x[1, :2]).any()
"""


@pytest.mark.parametrize("rot", [176, 192, 208])
@pytest.mark.parametrize("dtype,mixed", [("bfloat16", "half"), ("float16", "mixed"), ("float32", "half")])
def test_first_call_of_a_process_at_wide_rotations(rot, dtype, mixed):
    """64 rows of cos and sin and the kernel's own tables pass 48 KB from rot = 192 on."""
    env = dict(os.environ, PYTHONPATH=str(ROOT))
    got = subprocess.run([sys.executable, "-c", WIDE, str(rot), dtype, mixed], env=env, capture_output=True, text=True,
                         timeout=300)
    assert got.returncode == 0, got.stderr[-2000:]


def batch(new, ctx, Hq, Hk, D, page, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kp, vp, table, cu, kv_len = R.layout(new, ctx, page, Hk, D, dtype, DEV, g)
    rows = torch.randn(sum(new), Hq + 2 * Hk, D, generator=g, device=DEV).to(dtype)
    freq, _ = T.rope_inv_freq(D, device=DEV)
    return rows[:, :Hq], rows[:, Hq:Hq + Hk], rows[:, Hq + Hk:], freq, kp, vp, table, cu, kv_len


def test_means_that_have_no_place_are_reported():
    """A third block of a sequence, and room for the means of two: nothing is written beside them."""
    for n, nbk, bit in ((100, 2, 0), (101, 2, 1), (101, 3, 0), (1, 1, 1)):
        args = batch([n], [28], 4, 2, 64, 16, torch.bfloat16)
        if n == 1:
            args = batch([n], [64], 4, 2, 64, 16, torch.bfloat16)
        space = torch.full((3, 2, nbk, 64), 5.0, device=DEV)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        T.rope_append_paged(*args, n, pooled_k=space[1:2], err=err)
        assert int(err.item()) == bit, (n, nbk)
        assert (space[0] == 5).all() and (space[2] == 5).all()
        # without means there is nothing to report
        err.zero_()
        T.rope_append_paged(*args, n, err=err)
        assert int(err.item()) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_without_a_page_take_no_part_in_a_mean(dtype):
    """A key mean is that of what the cache holds: new rows whose page is not there are not in it, as
    earlier ones are not."""
    q, k, v, freq, kp, vp, table, cu, kv_len = batch([40], [24], 4, 2, 64, 16, dtype, seed=1)
    for gone in (0, 2, 3):  # rows 0 to 15 came earlier, 32 to 47 and 48 to 63 are new
        t = table.clone()
        t[0, gone] = -1 if gone == 2 else kp.shape[0]
        k1, means = kp.clone(), torch.zeros(1, 2, 1, 64, device=DEV)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        T.rope_append_paged(q, k, v, freq, k1, vp.clone(), t, cu, kv_len, 40, pooled_k=means, err=err)
        assert int(err.item()) & 1
        held = R.cached(k1, table[0], 64).double()
        held[16 * gone:16 * gone + 16] = 0
        # 63 fp32 additions, each at most half a step off
        tol = 64 * 2.0 ** -24 * held.abs().sum(0) / 64
        assert ((means[0, :, 0].double() - held.sum(0) / 64).abs() <= tol).all()
