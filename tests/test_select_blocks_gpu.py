"""Kept blocks by score against a sort, exactly: ties, floors, odd lengths, masked scores."""
from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as R
import tasft_b200 as T

pytestmark = pytest.mark.gpu
DEV = "cuda"


def batch(new, ctx):
    cu = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    return cu, torch.tensor([n + c for n, c in zip(new, ctx)], dtype=torch.int32, device=DEV)


def check(scores, hk, new, ctx, top_k, **kw):
    cu, kv_len = batch(new, ctx)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = T.select_blocks(scores, hk, cu, kv_len, top_k, err=err, **kw)
    idx, cnt = R.choose(scores, hk, new, ctx, top_k, **kw)
    assert int(err.item()) == 0
    assert torch.equal(got.cnt.cpu(), cnt)
    assert torch.equal(got.idx.cpu(), idx)


def scores(B, H, rows, nbk, seed=0, levels=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = torch.randn(B, H, rows, nbk, generator=g, device=DEV)
    return torch.round(s * levels) / levels if levels else s


@pytest.mark.parametrize("nbk", [1, 2, 31, 33, 128, 129, 500, 513, 2048, 2049])
@pytest.mark.parametrize("top_k", [1, 2, 7, 64])
def test_lengths(nbk, top_k):
    new, ctx = [100, 1, 70], [max(0, nbk * 64 - 100), 0, max(0, nbk * 32 - 70)]
    new = [min(n, nbk * 64 - c) for n, c in zip(new, ctx)]
    check(scores(3, 4, 3, nbk, nbk), 2, new, ctx, top_k)


@pytest.mark.parametrize("levels", [1, 2, 8])
def test_ties_go_to_the_lowest_index(levels):
    check(scores(2, 4, 4, 300, 1, levels), 4, [200, 190], [300 * 64 - 200, 9000], 40)
    check(torch.zeros(1, 2, 1, 700, device=DEV), 1, [1], [700 * 64 - 1], 100)


def test_gate_scores_close_to_a_half():
    s = torch.sigmoid(0.01 * scores(2, 28, 2, 512, 2))
    check(s, 4, [128, 1], [512 * 64 - 128, 20000], 51)
    check(s, 4, [128, 1], [512 * 64 - 128, 20000], 51, tau=0.5)


@pytest.mark.parametrize("first,local,top_k", [(0, 1, 5), (4, 3, 5), (4, 3, 9), (1, 8, 2), (300, 300, 4)])
def test_forced_blocks(first, local, top_k):
    check(scores(2, 2, 6, 250, 3), 1, [290, 1], [3000, 250 * 64 - 1], top_k, first=first, local=local)


@pytest.mark.parametrize("block,nbk", [(32, 40), (128, 300), (1, 600)])
def test_other_block_sizes(block, nbk):
    new, ctx = [3 * block, 1, 2], [nbk * block - 3 * block, 5 * block, 0]
    check(scores(3, 6, 4, nbk, 11), 3, new, ctx, 6, block=block)
    with pytest.raises(T.KernelError):
        T.select_blocks(scores(1, 1, 1, 8), 1, *batch([1], [5]), 3, block=48)


def test_masked_and_odd_scores():
    s = scores(1, 2, 1, 200, 4)
    s[:, 0, :, 5:90] = -math.inf
    s[:, 1, :, 5:60] = float("nan")
    s[:, :, :, 100] = math.inf
    s[:, :, :, 101] = torch.finfo(torch.float32).min
    s[:, :, :, 102] = -0.0
    s[:, :, :, 103] = 0.0
    for k in (3, 30, 120, 200):
        check(s, 1, [1], [200 * 64 - 1], k)
        check(s, 2, [1], [200 * 64 - 1], k)
    check(torch.full((1, 1, 1, 150), -math.inf, device=DEV), 1, [1], [150 * 64 - 1], 50)


def test_strided_scores_empty_sequences_and_decode_lists():
    s = scores(4, 8, 3, 140, 5)
    new, ctx = [1, 0, 100, 64], [5000, 0, 64, 30]
    check(s.transpose(0, 1).contiguous().transpose(0, 1), 2, new, ctx, 20)
    check(s[:, :, :, 10:130], 2, new, ctx, 20)
    cu, kv_len = batch([1] * 4, [5000, 64, 100, 4])
    kept = T.select_blocks(s[:, :, :1], 2, cu, kv_len, 9)
    # one row per sequence: what the single-token decode takes
    g = torch.Generator(device=DEV).manual_seed(6)
    kp, vp, table, _, _ = R.layout([1] * 4, [5000, 64, 100, 4], 16, 2, 128, torch.bfloat16, DEV, g, fill=0.0)
    q = torch.randn(4, 8, 128, generator=g, device=DEV).to(torch.bfloat16)
    # (that call looks up whole 64-token blocks, so its table names pages behind the last token too)
    whole = torch.nn.functional.pad(table, (0, -table.shape[1] % 4)).clamp(min=0)
    one = T.bsa_decode_paged(q, kp, vp, whole, kv_len, T.KeptBlocks(kept.idx[:, :, 0], kept.cnt[:, :, 0]))
    two = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 1, kept)
    o, a = R.attend(q, kp, vp, table, [1] * 4, [5000, 64, 100, 4], (kept.idx, kept.cnt))
    bound = R.attend_bound(o, a, torch.bfloat16, 5001)
    assert ((one.double() - o).abs() <= bound).all() and ((two.double() - o).abs() <= bound).all()


def test_lengths_that_do_not_fit_are_reported():
    s = scores(2, 2, 1, 10, 7)
    cu, kv_len = batch([1, 1], [639, 640])  # the second needs an eleventh block
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    kept = T.select_blocks(s, 2, cu, kv_len, 4, err=err)
    assert int(err.item()) & 1
    assert kept.cnt[0].min().item() == 4 and (kept.cnt[1] == 0).all() and (kept.idx[1] == -1).all()
    # more rows than the scores have
    cu, kv_len = batch([1, 66], [0, 63])
    err.zero_()
    kept = T.select_blocks(s, 2, cu, kv_len, 4, err=err)
    assert int(err.item()) & 1 and kept.cnt[0].min().item() == 1 and (kept.cnt[1] == 0).all() and (kept.idx[1] == -1).all()
