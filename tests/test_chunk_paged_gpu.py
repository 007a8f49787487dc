"""Attention of a chunk of new tokens over a paged cache, against the formula in fp64."""
from __future__ import annotations

import math

import pytest
import torch

import paged_oracle as R
import tasft_b200 as T

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case(new, ctx, Hq, Hk, D, page, dtype, seed=0, fill=float("nan")):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kp, vp, table, cu, kv_len = R.layout(new, ctx, page, Hk, D, dtype, DEV, g, fill=fill)
    q = torch.randn(sum(new), Hq, D, generator=g, device=DEV).to(dtype)
    return q, kp, vp, table, cu, kv_len, g


def check(new, ctx, Hq, Hk, D, page, dtype, lists=None, seed=0, **kw):
    """lists: None, or (heads, density, own, empty)."""
    q, kp, vp, table, cu, kv_len, g = case(new, ctx, Hq, Hk, D, page, dtype, seed)
    kept = None
    if lists is not None:
        heads, density, own, empty = lists
        width = max((n + c + 63) // 64 for n, c in zip(new, ctx))
        kept = T.KeptBlocks(*R.random_lists(new, ctx, heads, width, DEV, g, density, own, empty))
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, max(max(new), 1), kept, err=err, **kw)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    o, a = R.attend(q, kp, vp, table, new, ctx, None if kept is None else (kept.idx, kept.cnt), kw.get("scale"))
    off = (out.double() - o).abs()
    keys = max(n + c for n, c in zip(new, ctx))
    bound = R.attend_bound(o, a, dtype, keys)
    assert torch.isfinite(out.float()).all()
    assert (off <= bound).all(), f"off by {(off / bound).max().item():.3g} of the bound"
    return out


@pytest.mark.parametrize("new,ctx", [
    ([1], [0]), ([1], [1]), ([1], [63]), ([1], [64]), ([2], [62]), ([64], [0]), ([65], [63]), ([130], [0]),
    ([1], [4000]), ([17], [2100]), ([300], [777]),
])
def test_one_sequence_every_block(new, ctx):
    check(new, ctx, 8, 2, 128, 16, torch.bfloat16)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (4, 4), (8, 4), (6, 2), (28, 4), (16, 2), (10, 2), (12, 1), (64, 1)])
@pytest.mark.parametrize("lists", [None, "kv", "q"])
def test_head_layouts(Hq, Hk, lists):
    spec = None if lists is None else ((Hk if lists == "kv" else Hq), 0.4, True, 0.0)
    check([70, 1, 33], [200, 555, 0], Hq, Hk, 128, 32, torch.bfloat16, spec, seed=1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lists", [None, "kv", "q"])
def test_types_and_pages(dtype, D, page, lists):
    spec = None if lists is None else ((2 if lists == "kv" else 6), 0.5, True, 0.0)
    check([5, 1, 100], [100, 831, 61], 6, 2, D, page, dtype, spec, seed=2)


@pytest.mark.parametrize("lists", ["kv", "q"])
def test_rows_that_keep_nothing(lists):
    heads = 2 if lists == "kv" else 8
    check([200, 1, 1, 90], [300, 640, 0, 64], 8, 2, 128, 16, torch.bfloat16, (heads, 0.2, False, 0.3), seed=3)


def test_nothing_kept_at_all_gives_zero():
    q, kp, vp, table, cu, kv_len, _ = case([9, 1], [500, 70], 8, 2, 128, 16, torch.bfloat16)
    kept = T.KeptBlocks(torch.full((2, 2, 2, 9), -1, dtype=torch.int32, device=DEV),
                        torch.zeros(2, 2, 2, dtype=torch.int32, device=DEV))
    out = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 9, kept)
    assert (out == 0).all()


def test_many_sequences_and_empty_ones():
    new = [1 if i % 3 else 0 for i in range(301)]
    new[7] = 129
    ctx = [(37 * i) % 400 if n else 0 for i, n in enumerate(new)]
    check(new, ctx, 8, 2, 64, 16, torch.bfloat16, seed=4)
    check(new, ctx, 8, 2, 64, 16, torch.bfloat16, (2, 0.4, True, 0.0), seed=4)


@pytest.mark.parametrize("lists", [None, "kv", "q"])
def test_more_sequences_than_the_table_with_tiles_in_pieces(lists):
    """Two sequences per entry of the kernel's table, a few of them long enough to be cut."""
    new = [0] * 290
    ctx = [0] * 290
    for b, (n, c) in {3: (1, 15000), 4: (40, 70), 100: (70, 9000), 101: (1, 1), 288: (2, 20000), 289: (1, 63)}.items():
        new[b], ctx[b] = n, c
    spec = None if lists is None else ((2 if lists == "kv" else 8), 0.7, True, 0.0)
    check(new, ctx, 8, 2, 64, 64, torch.bfloat16, spec, seed=18)


@pytest.mark.parametrize("n,ctx", [(2048, 0), (700, 5000), (1, 7000)])
@pytest.mark.parametrize("Hq,Hk", [(4, 4), (7, 1)])
def test_tiles_of_many_lengths_in_pieces(n, ctx, Hq, Hk):
    check([n], [ctx], Hq, Hk, 128, 32, torch.float16, seed=19)
    check([n], [ctx], Hq, Hk, 128, 32, torch.float16, (Hk, 0.8, True, 0.05), seed=20)


@pytest.mark.parametrize("lists", [None, "kv", "q"])
def test_long_context_is_split(lists):
    spec = None if lists is None else ((4 if lists == "kv" else 28), 0.6, True, 0.0)
    check([1], [32767], 28, 4, 128, 16, torch.bfloat16, spec, seed=5)
    check([3, 1], [20000, 9], 28, 4, 128, 64, torch.bfloat16, spec, seed=6)


def test_longer_than_a_list_segment():
    check([130], [12000], 4, 1, 128, 64, torch.bfloat16, seed=7)
    check([130] * 9, [9000 + 64 * i for i in range(9)], 8, 8, 64, 128, torch.bfloat16, (8, 0.7, True, 0.0), seed=8)


def test_chunks_equal_the_whole():
    """The same prompt in one chunk or in pieces: every row within the same bounds, and the packed
    prefill without a cache agrees."""
    n, Hq, Hk, D, page = 1000, 8, 2, 128, 64
    q, kp, vp, table, cu, kv_len, _ = case([n], [0], Hq, Hk, D, page, torch.bfloat16, 9)
    o, a = R.attend(q, kp, vp, table, [n], [0])
    bound = R.attend_bound(o, a, torch.bfloat16, n)
    at = 0
    for m in (1, 63, 64, 200, 1, 671):
        part = T.bsa_chunk_paged(q[at:at + m], kp, vp, table, torch.tensor([0, m], dtype=torch.int32, device=DEV),
                                 torch.tensor([at + m], dtype=torch.int32, device=DEV), m)
        assert ((part.double() - o[at:at + m]).abs() <= bound[at:at + m]).all(), (at, m)
        at += m
    assert at == n
    k, v = R.cached(kp, table[0], n), R.cached(vp, table[0], n)
    nb = math.ceil(n / 64)
    full = torch.ones(1, Hk, nb, nb, dtype=torch.bool, device=DEV)
    whole = T.BlockSparseFlashAttention(64).forward_varlen(q, k, v, cu, n, full)
    assert ((whole.double() - o).abs() <= bound).all()


def test_strided_q_and_out_and_rows_outside_are_left():
    new, ctx, Hq, Hk, D = [5, 40], [77, 300], 8, 2, 128
    q, kp, vp, table, cu, kv_len, g = case(new, ctx, Hq, Hk, D, 32, torch.bfloat16, 10)
    rows = torch.randn(60, Hq + 4, D, generator=g, device=DEV).to(torch.bfloat16)
    rows[:45, :Hq] = q
    buf = torch.full((60, 2 * Hq, D), 7.0, device=DEV, dtype=torch.bfloat16)
    got = T.bsa_chunk_paged(rows[:, :Hq], kp, vp, table, cu, kv_len, 40, out=buf[:, :Hq])
    o, a = R.attend(q, kp, vp, table, new, ctx)
    assert ((got[:45].double() - o).abs() <= R.attend_bound(o, a, torch.bfloat16, 340)).all()
    assert (buf[45:] == 7).all() and (buf[:, Hq:] == 7).all()
    # an interleaved page pool: K and V of a page beside one another
    both = torch.stack((kp, vp), 1)
    again = T.bsa_chunk_paged(q, both[:, 0], both[:, 1], table, cu, kv_len, 40)
    assert torch.equal(again, got[:45])


def test_scale_and_large_scores():
    check([66, 1], [900, 130], 8, 2, 128, 16, torch.bfloat16, scale=0.5, seed=11)
    check([66, 1], [900, 130], 8, 2, 64, 16, torch.float16, scale=0.02, seed=11)


def test_bad_entries_are_reported_and_skipped():
    new, ctx = [40, 8], [200, 300]
    q, kp, vp, table, cu, kv_len, g = case(new, ctx, 8, 2, 128, 16, torch.bfloat16, 12)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    good = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 40, err=err)
    assert int(err.item()) == 0
    bad = table.clone()
    bad[0, 3] = kp.shape[0] + 5
    bad[0, 4] = -7
    out = T.bsa_chunk_paged(q, kp, vp, bad, cu, kv_len, 40, err=err)
    assert int(err.item()) & 1
    assert torch.equal(out[40:], good[40:])
    # the missing pages' 32 keys drop out of the softmax
    gone = torch.zeros(240, dtype=torch.bool, device=DEV)
    gone[48:80] = True
    k, v = (R.cached(x, table[0], 240)[:, 0].double() for x in (kp, vp))
    s = q[:40, 0].double() @ k.T / math.sqrt(128)
    pos = 200 + torch.arange(40, device=DEV)
    see = (torch.arange(240, device=DEV) <= pos.view(-1, 1)) & ~gone
    p = torch.softmax(torch.where(see, s, -math.inf), 1)
    o, a = p @ v, p @ v.abs()
    assert ((out[:40, 0].double() - o).abs() <= R.attend_bound(o, a, torch.bfloat16, 240)).all()


def test_lists_that_do_not_ascend_or_leave_the_range():
    q, kp, vp, table, cu, kv_len, g = case([1], [639], 4, 1, 64, 16, torch.bfloat16, 13)
    def run(entries, heads=1):
        idx = torch.tensor(entries, dtype=torch.int32, device=DEV).view(1, 1, 1, -1).repeat(1, heads, 1, 1)
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 1,
                                T.KeptBlocks(idx, torch.full((1, heads, 1), len(entries), dtype=torch.int32, device=DEV)),
                                err=err)
        return out, int(err.item())
    for heads in (1, 4):
        good, e = run([0, 3, 9], heads)
        assert e == 0
        for entries, bit in (([0, 3, 3, 9], 4), ([-2, 0, 3, 9], 1), ([0, 3, 2, 9], 4)):
            out, e = run(entries, heads)
            assert e & bit and torch.equal(out, good), entries
        # past the row's own block: nothing kept there. (A longer list may be cut into slices whose
        # maxima, and with them the roundings of p, differ: the bound holds, not the bits.)
        out, e = run([0, 3, 9, 10, 1000000], heads)
        kept = torch.tensor([[[[0, 3, 9]]]], dtype=torch.int32, device=DEV), torch.full((1, 1, 1), 3, device=DEV)
        o, a = R.attend(q, kp, vp, table, [1], [639], kept)
        assert e == 0 and ((out.double() - o).abs() <= R.attend_bound(o, a, torch.bfloat16, 640)).all()


def test_sequences_that_do_not_fit_are_left_out():
    new, ctx = [4, 4, 4], [50, 60, 70]
    q, kp, vp, table, cu, kv_len, g = case(new, ctx, 8, 2, 64, 16, torch.bfloat16, 14)
    good = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 4)
    for wrong in (3, 10 ** 6, -1):
        n = kv_len.clone()
        n[1] = wrong
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = torch.full_like(q, 3.0)
        T.bsa_chunk_paged(q, kp, vp, table, cu, n, 4, out=out, err=err)
        assert int(err.item()) & 1
        assert torch.equal(out[:4], good[:4]) and torch.equal(out[8:], good[8:]) and (out[4:8] == 3).all()
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    T.bsa_chunk_paged(q, kp, vp, table, torch.tensor([0, 4, 90, 12], dtype=torch.int32, device=DEV), kv_len, 4, err=err)
    assert int(err.item()) & 1


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("lists", [None, "kv", "q"])
@pytest.mark.parametrize("n", [100, 2])
def test_values_not_finite_reach_only_rows_that_see_them(dtype, D, lists, n):
    """Infinities and NaN of K and V at some positions: rows before them, and rows whose lists skip
    their block, are as if they were not there; rows that see them give what the sums give."""
    new, ctx, Hq, Hk = [n], [230], 4, 2
    q, kp, vp, table, cu, kv_len, g = case(new, ctx, Hq, Hk, D, 16, dtype, 16)
    total = n + 230
    kept = None
    if lists is not None:
        kept = T.KeptBlocks(*R.random_lists(new, ctx, Hk if lists == "kv" else Hq, 6, DEV, g, 0.6))
        kept = T.KeptBlocks(kept.idx, kept.cnt)
    bad = {total - 1: (3, math.inf), total - 2: (3, -math.inf), 231: (7, math.nan), 70: (D - 1, -math.inf)}
    vz = vp.clone()
    at = lambda t: (int(table[0, t // 16]), t % 16)  # noqa: E731
    for t, (d, x) in bad.items():
        vp[at(t)[0], at(t)[1], :, d] = x
        vz[at(t)[0], at(t)[1], :, d] = 0.0
    o, a = R.attend(q, kp, vz, table, new, ctx, None if kept is None else (kept.idx, kept.cnt))
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, n, kept, err=err)
    assert int(err.item()) == 0
    bound = R.attend_bound(o, a, dtype, total)
    want = o.clone()
    pos = 230 + torch.arange(n, device=DEV)
    for h in range(Hq):
        for t, (d, x) in bad.items():
            see = pos >= t
            if kept is not None:
                lists_h = kept.idx[0, h if lists == "q" else h // 2].long()
                see = see & (lists_h == t // 64).any(1)[pos // 64 - 230 // 64]
            want[see, h, d] += x
    finite = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), finite)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out.double()[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)])
    assert ((out.double() - o).abs()[finite] <= bound[finite]).all()
    # keys that are not finite, behind every row's mask but the last one's
    kp[at(total - 1)[0], at(total - 1)[1]] = math.nan
    again = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, n, kept)
    assert torch.equal(again[:-1].nan_to_num(5), out[:-1].nan_to_num(5))


def test_a_query_that_is_nan_gives_nan():
    q, kp, vp, table, cu, kv_len, g = case([40], [100], 4, 2, 128, 16, torch.bfloat16, 17)
    good = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 40)
    q[7, 2] = math.nan
    out = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 40)
    assert torch.isnan(out[7, 2]).all()
    out[7, 2] = good[7, 2]
    assert torch.equal(out, good)


def test_no_tokens_and_odd_strides_of_single_axes():
    q, kp, vp, table, cu, kv_len, g = case([3, 2], [40, 9], 4, 1, 64, 16, torch.bfloat16, 21)
    none = T.bsa_chunk_paged(q[:0], kp, vp, table, torch.zeros_like(cu), kv_len, 3)
    assert none.shape == (0, 4, 64)
    want = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 3)
    one = torch.as_strided(q[4:5], (1, 4, 64), (3, 64, 1))  # one token: its stride says nothing
    got = T.bsa_chunk_paged(one, kp, vp, table[1:], torch.tensor([0, 1], dtype=torch.int32, device=DEV), kv_len[1:], 1)
    assert torch.equal(got, want[4:5])
    flat = torch.empty(q.numel() + 1, device=DEV, dtype=q.dtype)
    off = flat[1:].view(q.shape)  # not on a 16-byte boundary
    off.copy_(q)
    assert torch.equal(T.bsa_chunk_paged(off, kp, vp, table, cu, kv_len, 3), want)


def test_graph_replay_follows_its_inputs():
    new, ctx = [33, 1, 1], [500, 900, 40]
    q, kp, vp, table, cu, kv_len, g = case(new, ctx, 8, 2, 128, 16, torch.bfloat16, 15)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 33, out=out)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, 33, out=out)
    # fewer cached tokens and another split of the rows, in the same tensors
    kv_len.copy_(torch.tensor([400, 31, 30], dtype=torch.int32))
    cu.copy_(torch.tensor([0, 2, 33, 35], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    o, a = R.attend(q, kp, vp, table, [2, 31, 2], [398, 0, 28])
    assert ((out.double() - o).abs() <= R.attend_bound(o, a, torch.bfloat16, 600)).all()


@pytest.mark.parametrize("lists", [None, "kv", "q"])
@pytest.mark.parametrize("new,ctx", [([1, 90, 300], [4000, 0, 700]), ([1], [6000]), ([513], [5000])])
def test_out_may_be_q(lists, new, ctx):
    """Each tile reads its own rows of q before it writes them, tiles in pieces are written last."""
    q, kp, vp, table, cu, kv_len, g = case(new, ctx, 8, 2, 128, 16, torch.bfloat16, seed=21)
    kept = None
    if lists is not None:
        width = max((n + c + 63) // 64 for n, c in zip(new, ctx))
        kept = T.KeptBlocks(*R.random_lists(new, ctx, 2 if lists == "kv" else 8, width, DEV, g, 0.5, True, 0.0))
    want = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, max(new), kept)
    got = T.bsa_chunk_paged(q, kp, vp, table, cu, kv_len, max(new), kept, out=q)
    assert got is q and torch.equal(got, want)
