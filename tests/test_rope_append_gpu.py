"""Rotary embedding into a paged cache with the gate's block means, against the formula in fp64."""
from __future__ import annotations

import pytest
import torch

import paged_oracle as R
import tasft_b200 as T

pytestmark = pytest.mark.gpu
DEV = "cuda"


def case(new, ctx, Hq, Hk, D, page, dtype, rot, scaling=None, base=10000.0, seed=0, fill=float("nan")):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kp, vp, table, cu, kv_len = R.layout(new, ctx, page, Hk, D, dtype, DEV, g, fill=fill)
    rows = torch.randn(sum(new), Hq + 2 * Hk, D, generator=g, device=DEV).to(dtype)
    freq, factor = T.rope_inv_freq(rot, base, scaling, device=DEV)
    return rows, kp, vp, table, cu, kv_len, freq, factor


def rotated_bound(x, dtype, factor=1.0):
    """One rounding to the type (half a step of the result) and the fp32 products: each of the two is
    off by at most 3 half steps of fp32 (cos, factor, product) and their sum by one more, against
    the pair's length, which a rotation by ``factor`` keeps at most sqrt(2) factor max|x|."""
    u = torch.finfo(dtype).eps / 2
    return u * x.abs() + 8 * 2.0 ** -24 * (x.abs() + 1.5 * factor * x.abs().amax(-1, keepdim=True)) + 1e-30


def check(new, ctx, Hq, Hk, D, page, dtype, rot, interleaved=False, scaling=None, base=10000.0, seed=0, nbk=None):
    rows, kp, vp, table, cu, kv_len, freq, factor = case(new, ctx, Hq, Hk, D, page, dtype, rot, scaling, base, seed)
    q, k, v = rows[:, :Hq], rows[:, Hq:Hq + Hk], rows[:, Hq + Hk:]
    kp0, vp0 = kp.clone(), vp.clone()
    nbk = nbk or max((n + c + 63) // 64 for n, c in zip(new, ctx))
    means = torch.full((len(new), Hk, nbk, D), 5.0, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, pooled_q = T.rope_append_paged(q, k, v, freq, kp, vp, table, cu, kv_len, max(max(new), 1),
                                        interleaved=interleaved, attention_scaling=factor, pooled_k=means, err=err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    written = torch.zeros(kp.shape[:2], dtype=torch.bool, device=DEV)
    at = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        if n == 0:
            assert (pooled_q[b] == 0).all() and (means[b] == 5).all()
            continue
        pos = c + torch.arange(n, device=DEV)
        sl = slice(at, at + n)
        for got, x in ((out[sl], q[sl]), (R.cached(kp, table[b], n + c)[c:], k[sl])):
            want = R.rotate(x, pos, freq, factor, interleaved)
            assert ((got.double() - want).abs() <= rotated_bound(want, dtype, factor)).all()
            assert torch.equal(got[..., rot:], x[..., rot:])
        assert torch.equal(R.cached(vp, table[b], n + c)[c:], v[sl])
        written[table[b].long()[pos // page], pos % page] = True
        # means of the values as held: 64 fp32 additions, each at most half a step off
        first, last = c // 64, (c + n - 1) // 64
        keys = R.cached(kp, table[b], n + c).double()
        for i, blk in enumerate(range(first, last + 1)):
            rows_k = keys[blk * 64:(blk + 1) * 64]
            tol = 65 * 2.0 ** -24 * rows_k.abs().sum(0) / 64 + 1e-30
            assert ((means[b, :, blk].double() - rows_k.sum(0) / 64).abs() <= tol).all()
            lo, hi = max(blk * 64, c) - c, min((blk + 1) * 64, c + n) - c
            rows_q = out[at + lo:at + hi].double()
            tol = 65 * 2.0 ** -24 * rows_q.abs().sum(0) / 64 + 1e-30
            assert ((pooled_q[b, :, i].double() - rows_q.sum(0) / 64).abs() <= tol).all()
        assert (pooled_q[b, :, last - first + 1:] == 0).all()
        assert (means[b, :, :first] == 5).all() and (means[b, :, last + 1:] == 5).all()
        at += n
    # nothing else in the pools changed
    assert torch.equal(kp[~written].nan_to_num(9), kp0[~written].nan_to_num(9))
    assert torch.equal(vp[~written].nan_to_num(9), vp0[~written].nan_to_num(9))
    return out


LLAMA3 = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
              original_max_position_embeddings=8192)
YARN = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)


@pytest.mark.parametrize("new,ctx", [([1], [0]), ([1], [63]), ([1], [64]), ([64], [0]), ([65], [63]), ([129], [1]),
                                     ([1, 0, 200, 3], [5000, 0, 37, 64])])
def test_lengths(new, ctx):
    check(new, ctx, 8, 2, 128, 16, torch.bfloat16, 128)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (64, 64), (64, 16), (96, 32), (256, 256), (32, 0), (80, 80)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_types_and_layouts(dtype, D, rot, interleaved):
    if rot == 0:
        rows, kp, vp, table, cu, kv_len, _, _ = case([40], [50], 4, 2, D, 32, dtype, 2)
        out, _ = T.rope_append_paged(rows[:, :4], rows[:, 4:6], rows[:, 6:], torch.empty(0, device=DEV), kp, vp, table,
                                     cu, kv_len, 40, interleaved=interleaved)
        assert torch.equal(out, rows[:, :4])
        assert torch.equal(R.cached(kp, table[0], 90)[50:], rows[:, 4:6])
        return
    check([70, 1], [30, 200], 4, 2, D, 32, dtype, rot, interleaved, seed=1)


@pytest.mark.parametrize("scaling", [None, dict(rope_type="linear", factor=4.0), LLAMA3, YARN])
def test_far_positions(scaling):
    # fp32 angles have lost their fraction here: the result still matches the exact angle
    check([130, 1], [1_000_000, 131_000], 2, 1, 128, 128, torch.float32, 128, scaling=scaling, base=500000.0, seed=2)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hk", [(28, 4), (32, 8), (3, 3), (1, 1)])
def test_pages_and_heads(page, Hq, Hk):
    check([77, 5, 1], [100, 0, 1030], Hq, Hk, 64, page, torch.bfloat16, 64, seed=3)


def test_pieces_equal_the_whole():
    """Appending in pieces leaves the same cache and the same key means, bit for bit."""
    rows, kp, vp, table, cu, kv_len, freq, f = case([300], [0], 8, 2, 128, 16, torch.bfloat16, 128, seed=4)
    args = dict(attention_scaling=f)
    m1, m2 = torch.zeros(1, 2, 5, 128, device=DEV), torch.zeros(1, 2, 5, 128, device=DEV)
    k1, v1, k2, v2 = kp.clone(), vp.clone(), kp.clone(), vp.clone()
    whole, _ = T.rope_append_paged(rows[:, :8], rows[:, 8:10], rows[:, 10:], freq, k1, v1, table, cu, kv_len, 300,
                                   pooled_k=m1, **args)
    at, parts = 0, []
    for n in (1, 62, 1, 64, 100, 72):
        r = rows[at:at + n]
        parts.append(T.rope_append_paged(r[:, :8], r[:, 8:10], r[:, 10:], freq, k2, v2, table,
                                         torch.tensor([0, n], dtype=torch.int32, device=DEV),
                                         torch.tensor([at + n], dtype=torch.int32, device=DEV), n, pooled_k=m2, **args)[0])
        at += n
    assert at == 300
    assert torch.equal(torch.cat(parts), whole)
    assert torch.equal(k1.nan_to_num(9), k2.nan_to_num(9)) and torch.equal(v1.nan_to_num(9), v2.nan_to_num(9))
    assert torch.allclose(m1, m2, rtol=0, atol=65 * 2.0 ** -24 * 4)


def test_no_tokens_give_means_of_zero():
    rows, kp, vp, table, cu, kv_len, freq, f = case([4], [30], 4, 2, 64, 16, torch.bfloat16, 64, seed=7)
    means = torch.full((1, 2, 2, 64), 5.0, device=DEV)
    k0 = kp.clone()
    out, pooled_q = T.rope_append_paged(rows[:0, :4], rows[:0, 4:6], rows[:0, 6:], freq, kp, vp, table, torch.zeros_like(cu),
                                        kv_len, 3, pooled_k=means)
    assert out.shape == (0, 4, 64) and (pooled_q == 0).all() and (means == 5).all()
    assert torch.equal(kp.nan_to_num(9), k0.nan_to_num(9))


def test_in_place_and_fp32_frequencies():
    rows, kp, vp, table, cu, kv_len, freq, f = case([90], [10], 4, 4, 64, 16, torch.float16, 64, seed=5)
    q = rows[:, :4].contiguous()
    want, none = T.rope_append_paged(q, rows[:, 4:8], rows[:, 8:], freq.float(), kp, vp, table, cu, kv_len, 90)
    assert none is None
    got, _ = T.rope_append_paged(q, rows[:, 4:8], rows[:, 8:], freq.float(), kp, vp, table, cu, kv_len, 90, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want)
    flat = torch.empty(rows.numel() + 1, device=DEV, dtype=rows.dtype)
    off = flat[1:].view(rows.shape)  # not on a 16-byte boundary
    off.copy_(rows)
    again, _ = T.rope_append_paged(off[:, :4], off[:, 4:8], off[:, 8:], freq.float(), kp, vp, table, cu, kv_len, 90)
    assert torch.equal(again, want)


def test_bad_pages_and_sequences_write_nothing():
    new, ctx = [10, 10], [60, 60]
    rows, kp, vp, table, cu, kv_len, freq, f = case(new, ctx, 4, 2, 64, 16, torch.bfloat16, 64, seed=6, fill=0.0)
    q, k, v = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    for breakage in ("page", "length", "cu"):
        t, n, c = table.clone(), kv_len.clone(), cu.clone()
        if breakage == "page":
            t[0, 3:5] = kp.shape[0]
        elif breakage == "length":
            n[0] = 9
        else:
            c[0] = -4
        k1, v1, err = kp.clone(), vp.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
        T.rope_append_paged(q, k, v, freq, k1, v1, t, c, n, 10, err=err)
        torch.cuda.synchronize()
        assert int(err.item()) & 1
        row = table[0].long()
        assert torch.equal(k1[row[3:5]], kp[row[3:5]]) and torch.equal(v1[row[3:5]], vp[row[3:5]])
        assert torch.equal(R.cached(v1, table[1], 70)[60:], v[10:])
