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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("new,ctx", [([1], [0]), ([1], [100]), ([37, 1, 0, 150], [50, 63, 0, 20]), ([64, 63], [64, 1])])
def test_means_over_the_new_queries_alone(dtype, new, ctx):
    q, k, v, freq, kp, vp, table, cu, kv_len = batch(new, ctx, 6, 2, 64, 16, dtype, seed=2)
    nbk = max((n + c + 63) // 64 for n, c in zip(new, ctx))
    means = [torch.zeros(len(new), 2, nbk, 64, device=DEV) for _ in range(2)]
    args = (q, k, v, freq, kp, vp, table, cu, kv_len, max(new))
    out, pooled = T.rope_append_paged(*args, pooled_k=means[0], query_mean="new")
    _, padded = T.rope_append_paged(*args, pooled_k=means[1])
    assert torch.equal(means[0], means[1])  # key means are over what the cache holds either way
    at = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        for i in range(pooled.shape[2]):
            lo, hi = max((c // 64 + i) * 64, c) - c, min((c // 64 + i + 1) * 64, c + n) - c
            if hi <= lo:
                assert (pooled[b, :, i] == 0).all() and (padded[b, :, i] == 0).all()
                continue
            rows = out[at + lo:at + hi].double()
            # 63 fp32 additions, 1 / rows and the product, each at most half a step off
            tol = 66 * 2.0 ** -24 * rows.abs().mean(0)
            assert ((pooled[b, :, i].double() - rows.mean(0)).abs() <= tol).all()
            if hi - lo == 1:
                assert torch.equal(pooled[b, :, i], out[at + lo].float())
            if hi - lo == 64:
                assert torch.equal(pooled[b, :, i], padded[b, :, i])
        at += n


def test_query_mean_is_one_of_two():
    args = batch([3], [5], 4, 2, 64, 16, torch.bfloat16)
    with pytest.raises(T.KernelError):
        T.rope_append_paged(*args, 3, query_mean="rows")


def test_chunks_of_whole_blocks_choose_as_the_whole_prompt_does():
    """The gate's lists for a prompt do not depend on how it was cut, as long as blocks stay whole; in a
    cut one every row of its parts still has a mean of full weight."""
    Hq, Hk, D, n = 8, 2, 128, 700
    q, k, v, freq, kp, vp, table, cu, kv_len = batch([n], [0], Hq, Hk, D, 16, torch.bfloat16, seed=5)
    torch.manual_seed(5)
    gate = T.AttnGate(Hq, D, block_size=64, is_causal=False).to(DEV)
    torch.nn.init.normal_(gate.gate_proj_out.weight, std=1.0)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731

    def lists(cuts):
        means, got, weight = torch.zeros(1, Hk, 11, D, device=DEV), {}, []
        for lo, hi in zip(cuts[:-1], cuts[1:]):
            c, m = ints(0, hi - lo), hi - lo
            _, pooled = T.rope_append_paged(q[lo:hi], k[lo:hi], v[lo:hi], freq, kp, vp, table, c, ints(hi), m, pooled_k=means,
                                            query_mean="new")
            with torch.no_grad():
                soft = gate.forward_pooled(pooled, means, pooled.shape[2] * 64, 11 * 64).soft_scores
            kept = T.select_blocks(soft, Hk, c, ints(hi), 4)
            for i in range((hi - 1) // 64 - lo // 64 + 1):
                got[lo // 64 + i, lo] = kept.idx[0, :, i].tolist()
                weight.append(pooled[0, :, i].abs().mean().item())
        return got, weight

    whole, _ = lists([0, n])
    for cuts in ([0, 64, 320, n], [0, 384, 448, n]):
        got, _ = lists(cuts)
        assert {key[0]: x for key, x in got.items()} == {key[0]: x for key, x in whole.items()}
    _, weight = lists([0, 100, 101, 300, n])
    _, full = lists([0, 640])
    assert min(weight) >= 0.9 * min(full)  # (a mean of fewer random rows is larger, a sum over 64 smaller)


@pytest.mark.parametrize("cu", [[0, 4, 90, 12, 20], [-4, 4, 8, 12, 16], [30, 20, 10, 4, 0],
                                [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5, 9], [1, -2 ** 31, 4, 5, 3]])
def test_row_ranges_that_make_no_sense_are_left_out(cu):
    """Ends before starts by so much that their difference wraps to a small number among them."""
    q, k, v, freq, kp, vp, table, _, kv_len = batch([4, 4, 4, 13], [50, 60, 70, 0], 6, 2, 64, 16, torch.bfloat16)
    k1, v1, out = kp.clone(), vp.clone(), torch.full_like(q, 7.0, memory_format=torch.contiguous_format)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    T.rope_append_paged(q, k, v, freq, k1, v1, table, torch.tensor(cu, device=DEV).to(torch.int32), kv_len, 4, out=out,
                        err=err)
    assert int(err.item()) == 1
    fits = [0 <= cu[b] <= cu[b + 1] <= 25 and cu[b + 1] - cu[b] <= 4 for b in range(4)]
    row = torch.zeros(25, dtype=torch.bool, device=DEV)
    page = torch.zeros(kp.shape[0], dtype=torch.bool, device=DEV)
    for b in range(4):
        if fits[b]:
            row[cu[b]:cu[b + 1]] = True
            page[table[b][table[b] >= 0].long()] = True
    assert (out[~row] == 7).all()
    assert torch.equal(k1[~page], kp[~page]) and torch.equal(v1[~page], vp[~page])


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 256), (torch.float32, 128)])
def test_rows_that_no_sequence_accounts_for_are_zero_in_a_new_tensor(dtype, D):
    """Padding before and behind the sequences, a sequence that does not fit: 0 in a new tensor, left as
    they were in one that is given."""
    new, ctx = [40, 1, 0, 170, 5], [30, 90, 0, 0, 64]
    g = torch.Generator(device=DEV).manual_seed(4)
    kp, vp, table, cu, kv_len = R.layout(new, ctx, 16, 2, D, dtype, DEV, g)
    rows = torch.randn(sum(new) + 9, 10, D, generator=g, device=DEV).to(dtype)
    q, k, v = rows[:, :6], rows[:, 6:8], rows[:, 8:]
    freq, _ = T.rope_inv_freq(D, device=DEV)
    cu = cu + 3
    want = None
    for gone in ([], [0], [1, 4], [3], [0, 1, 3, 4]):
        n = kv_len.clone()
        n[gone] = 10 ** 6
        dead = torch.ones(rows.shape[0], dtype=torch.bool, device=DEV)
        for b in range(5):
            if b not in gone:
                dead[int(cu[b]):int(cu[b + 1])] = False
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        torch.full_like(q, 7.0, memory_format=torch.contiguous_format)  # where the new tensor is likely to come
        out, _ = T.rope_append_paged(q, k, v, freq, kp, vp, table, cu, n, 170, err=err)
        assert int(err.item()) == (1 if gone else 0)
        want = out.clone() if want is None else want
        assert (out[dead] == 0).all() and torch.equal(out[~dead], want[~dead])
        mine = torch.full((rows.shape[0], 6, D), 3.0, device=DEV, dtype=dtype)
        T.rope_append_paged(q, k, v, freq, kp, vp, table, cu, n, 170, out=mine)
        assert (mine[dead] == 3).all() and torch.equal(mine[~dead], want[~dead])


@pytest.mark.parametrize("cu", [[0, 4, 90, 12, 20], [-4, 4, 8, 12, 16], [30, 20, 10, 4, 0], [0, 0, 0, 0, 0],
                                [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5, 9]])
def test_row_ranges_that_make_no_sense_leave_nothing_unset(cu):
    q, k, v, freq, kp, vp, table, _, kv_len = batch([4, 4, 4, 13], [50, 60, 70, 0], 6, 2, 64, 16, torch.bfloat16)
    torch.full_like(q, 7.0, memory_format=torch.contiguous_format)
    out, _ = T.rope_append_paged(q, k, v, freq, kp, vp, table, torch.tensor(cu, device=DEV).to(torch.int32), kv_len, 4)
    assert torch.isfinite(out).all() and (out != 7).all()
