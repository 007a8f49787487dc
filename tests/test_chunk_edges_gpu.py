"""Edges of the attention of new tokens over a paged cache."""
from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as R
import tasft_b200 as T

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run_list(entries, heads, ctx=639, seed=13, new=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kp, vp, table, cu, kv_len = R.layout([new], [ctx], 16, 1, 64, torch.bfloat16, DEV, g)
    q = torch.randn(new, 4, 64, generator=g, device=DEV).to(torch.bfloat16)
    idx = torch.tensor(entries, dtype=torch.int32, device=DEV).view(1, 1, 1, -1).repeat(1, heads, 1, 1)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    cnt = torch.full((1, heads, 1), len(entries), dtype=torch.int32, device=DEV)
    out = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, new, T.KeptBlocks(idx, cnt), err=err)
    return out, int(err.item()), (q, kp, vp, table)


@pytest.mark.parametrize("heads", [1, 4])
@pytest.mark.parametrize("entries,kept,bits", [
    ([0, 3, 2, 3, 9], [0, 3, 9], 4), ([0, 5, 2, 4, 9], [0, 5, 9], 4), ([3, 0, 1, 2, 3, 4], [3, 4], 4),
    ([5, -1, 5, 9], [5, 9], 5), ([-3, 0, 3, -1, 2, 9], [0, 3, 9], 5), ([9, 9, 9], [9], 4),
])
def test_an_entry_not_above_all_before_it_is_skipped(heads, entries, kept, bits):
    """Not only above its neighbour: a block that comes twice counts once, in both layouts of lists."""
    want, none, _ = run_list(kept, heads)
    got, err, _ = run_list(entries, heads)
    assert none == 0 and err == bits
    assert torch.equal(got, want)


@pytest.mark.parametrize("heads", [1, 4])
def test_order_is_kept_across_warps_segments_and_pieces(heads):
    """A long list with a block far ahead of its place: what it overtakes is skipped, however the
    list is cut among CTAs."""
    blocks = 600
    for at, jump in ((40, 300), (31, 33), (32, 590), (130, 400), (0, 200)):
        entries = list(range(blocks))
        entries.insert(at, jump)
        kept = list(range(at)) + list(range(jump, blocks))
        got, err, (q, kp, vp, table) = run_list(entries, heads, ctx=64 * blocks - 1)
        assert err == 4
        idx = torch.tensor(kept, dtype=torch.int32, device=DEV).view(1, 1, 1, -1)
        cnt = torch.full((1, 1, 1), len(kept), dtype=torch.int32, device=DEV)
        o, a = R.attend(q, kp, vp, table, [1], [64 * blocks - 1], (idx, cnt))
        assert ((got.double() - o).abs() <= R.attend_bound(o, a, torch.bfloat16, 64 * blocks)).all(), (at, jump)


@pytest.mark.parametrize("ctx,D", [(60000, 64), (30000, 128), (9000, 64)])
@pytest.mark.parametrize("top", [0, 4000])
def test_many_small_probabilities_in_half_precision(ctx, D, top):
    """One key far above the others (25.4 in base 2), whose values are 0: the output is the sum of the
    small ones, each below half the smallest fp16. Held as 2^6 p, a p is off by at most 2^-31 absolute.
    One tile a CTA, so that tiles stay whole: the same sequence as often as there are SMs."""
    n, B = ctx + 1, torch.cuda.get_device_properties(0).multi_processor_count
    g = torch.Generator(device=DEV).manual_seed(3)
    kp, vp, table, _, _ = R.layout([1], [ctx], 64, 2, D, torch.float16, DEV, g)
    kp.zero_()
    vp.copy_(1 + torch.rand(vp.shape, generator=g, device=DEV))
    page, row = int(table[0, top // 64]), top % 64
    kp[page, row, :, 0] = 1.0
    vp[page, row] = 0.0
    q = torch.zeros(B, 4, D, device=DEV, dtype=torch.float16)
    q[:, :, 0] = 2.0
    scale = 25.4 * math.log(2.0) / 2.0
    out = T.bsa_chunk_paged(q, kp, vp, table.repeat(B, 1), torch.arange(B + 1, dtype=torch.int32, device=DEV),
                            torch.full((B,), n, dtype=torch.int32, device=DEV), 1, scale=scale)
    o, a = R.attend(q[:1], kp, vp, table, [1], [ctx], scale=scale)
    # half a step of the result, 2^-31 for each p (2^6 2^-25.4 is below the normal numbers of fp16)
    # against a sum of at least 1, and 2^-14 for fp32 scores, exponentials and sums, as in attend_bound
    bound = 2.0 ** -11 * o.abs() + 2.0 ** -14 * a + n * 2.0 ** -31 * vp.max().item() + 2.0 ** -25
    assert ((out.double() - o).abs() <= bound).all()
