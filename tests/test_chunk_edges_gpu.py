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


def packed(new, ctx, D=128, page=16, seed=7):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kp, vp, table, cu, kv_len = R.layout(new, ctx, page, 2, D, torch.bfloat16, DEV, g)
    q = torch.randn(sum(new) + 9, 8, D, generator=g, device=DEV).to(torch.bfloat16)
    return q, kp, vp, table, cu, kv_len, g


def used_memory(like):
    """Leaves values where the next tensor of this size is likely to come."""
    torch.full_like(like, 7.0, memory_format=torch.contiguous_format)


@pytest.mark.parametrize("lists", [None, "kv", "q"])
@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_no_sequence_accounts_for_are_zero_in_a_new_tensor(lists, D):
    """Padding before and behind the sequences, a sequence that does not fit, all of them: 0 in a new
    tensor, left as they were in one that is given; the other rows as ever."""
    new, ctx = [40, 1, 0, 70, 5], [300, 900, 0, 0, 64]
    q, kp, vp, table, cu, kv_len, g = packed(new, ctx, D)
    kept = None
    if lists:
        kept = T.KeptBlocks(*R.random_lists(new, ctx, 2 if lists == "kv" else 8, 15, DEV, g, 0.6))
    cu = cu + 3  # three rows before, six behind
    good = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 70, kept)
    o, a = R.attend(q[3:119], kp, vp, table, new, ctx, None if kept is None else (kept.idx, kept.cnt))
    assert ((good[3:119].double() - o).abs() <= R.attend_bound(o, a, torch.bfloat16, 901)).all()
    for gone in ([], [0], [1, 4], [3], [0, 1, 3, 4]):
        n = kv_len.clone()
        n[gone] = 10 ** 6
        dead = torch.ones(q.shape[0], dtype=torch.bool, device=DEV)
        for b in range(5):
            if b not in gone:
                dead[int(cu[b]):int(cu[b + 1])] = False
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        used_memory(q)
        out = T.bsa_chunk_paged(q, kp, vp, table, cu, n, 70, kept, err=err)
        assert int(err.item()) == (1 if gone else 0)
        assert (out[dead] == 0).all() and torch.isfinite(out).all()
        o_dead, a_dead = o.clone(), a.clone()
        live = ~dead[3:119]
        assert ((out[3:119].double() - o_dead).abs()[live] <= R.attend_bound(o_dead, a_dead, torch.bfloat16, 901)[live]).all()
        mine = torch.full_like(q, 3.0)
        T.bsa_chunk_paged(q, kp, vp, table, cu, n, 70, kept, out=mine)
        assert (mine[dead] == 3).all() and torch.equal(mine[~dead], out[~dead])


@pytest.mark.parametrize("cu", [[0, 4, 90, 12, 20], [-4, 4, 8, 12, 16], [30, 20, 10, 4, 0], [0, 0, 0, 0, 0],
                                [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 5, 9]])
def test_row_ranges_that_make_no_sense_leave_nothing_unset(cu):
    q, kp, vp, table, _, kv_len, g = packed([4, 4, 4, 4], [50, 60, 70, 0])
    used_memory(q)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = T.bsa_chunk_paged(q, kp, vp, table, torch.tensor(cu, device=DEV).to(torch.int32), kv_len, 4, err=err)
    assert torch.isfinite(out).all() and (out != 7).all()
    assert int(err.item()) == (0 if cu == [0] * 5 else 1)


def test_padding_of_a_captured_step_follows_the_lengths():
    q, kp, vp, table, cu, kv_len, g = packed([33, 1, 1], [500, 900, 40])
    T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 33)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 33)
    for new in ([33, 1, 1], [2, 7, 0], [0, 0, 0], [30, 5, 9]):
        cu.copy_(torch.tensor([sum(new[:b]) for b in range(4)], dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        n = sum(new)
        assert (out[n:] == 0).all()
        total = kv_len.tolist()
        o, a = R.attend(q[:n], kp, vp, table, new, [t - m for t, m in zip(total, new)])
        assert ((out[:n].double() - o).abs() <= R.attend_bound(o, a, torch.bfloat16, 901)).all()
