"""Host side of the paged serving operators: refusals, sizes and rotary frequencies (no GPU)."""
from __future__ import annotations

import ctypes as C
import math

import pytest
import torch

import tasft_b200 as T
from tasft_b200 import _lib as L


def chunk_args(**kw):
    a = L.ChunkArgs(q=4096, k_pages=4096, v_pages=4096, out=4096, block_table=4096, cu_seqlens=4096, kv_len=4096,
                    B=2, T=5, Hq=8, Hk=2, D=128, block=64, dtype=L.BF16, max_q=4, max_pages=4, page_size=16,
                    num_pages=9, scale=0.1, workspace=4096, workspace_bytes=1 << 20)
    a.q_stride[:] = a.o_stride[:] = [1024, 128]
    a.k_stride[:] = a.v_stride[:] = [4096, 256, 128, 1]
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(B=0), -1), (dict(T=-1), -1), (dict(Hq=7), -1), (dict(Hk=0), -1), (dict(max_q=0), -1), (dict(max_pages=0), -1),
    (dict(num_pages=0), -1), (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(kv_len=None), -1),
    (dict(cu_seqlens=None), -1), (dict(block_table=None), -1), (dict(k_pages=None), -1), (dict(out=None), -1),
    (dict(kept_idx=4096), -1), (dict(kept_idx=4096, kept_cnt=4096, Hm=3, nb_q=2, nb_w=4), -1),
    (dict(kept_idx=4096, kept_cnt=4096, Hm=2, nb_q=1, nb_w=4), -1),
    (dict(kept_idx=4096, kept_cnt=4096, Hm=2, nb_q=2, nb_w=0), -1),
    (dict(dtype=L.F32), -2), (dict(D=96), -2), (dict(block=32), -2), (dict(page_size=48), -2), (dict(page_size=256), -2),
    (dict(out=4100), -2), (dict(Hq=130), -2), (dict(max_pages=1 << 26), -5), (dict(workspace=None), -4),
    (dict(workspace_bytes=0), -4),
])
def test_chunk_refusals(change, status):
    assert L.lib().tasft_bsa_chunk_paged_fwd(C.byref(chunk_args(**change)), None) == status


def test_chunk_without_tokens_launches_nothing():
    before = L.launch_count()
    assert L.lib().tasft_bsa_chunk_paged_fwd(C.byref(chunk_args(T=0, q=None, out=None)), None) == 0
    assert L.launch_count() == before


def test_chunk_null_and_workspace():
    lib = L.lib()
    for fn in ("tasft_bsa_chunk_paged_fwd", "tasft_rope_append_paged", "tasft_select_blocks"):
        assert getattr(lib, fn)(None, None) == -1
    assert lib.tasft_chunk_workspace_size(0, 1, 8, 2, 128, 1, 0) == -1
    assert lib.tasft_chunk_workspace_size(1, 1, 7, 2, 128, 1, 0) == -1
    assert lib.tasft_chunk_workspace_size(1, 1, 130, 2, 128, 1, 0) == -2
    one, many = (lib.tasft_chunk_workspace_size(b, b, 32, 8, 128, 1, 0) for b in (1, 64))
    assert 0 < one <= many < 16 << 20  # single tokens: few rows per split item


def rope_args(**kw):
    a = L.RopeAppendArgs(q=4096, k=4096, v=4096, q_out=4096, k_pages=4096, v_pages=4096, inv_freq=4096,
                         block_table=4096, cu_seqlens=4096, kv_len=4096, factor=1.0, B=2, T=5, Hq=8, Hk=2, D=128, rot=128,
                         block=64, dtype=L.BF16, max_q=4, max_pages=4, page_size=16, num_pages=9, NBq=2, NBk=4)
    a.q_stride[:] = a.k_in_stride[:] = a.v_in_stride[:] = a.o_stride[:] = [1024, 128]
    a.k_stride[:] = a.v_stride[:] = [4096, 256, 128, 1]
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(B=0), -1), (dict(T=-1), -1), (dict(Hq=7), -1), (dict(max_q=0), -1), (dict(page_size=0), -1), (dict(rot=-2), -1),
    (dict(rot=144), -1), (dict(inv_freq=None), -1), (dict(NBq=1), -1), (dict(pooled_k=4096, NBk=0), -1), (dict(q=None), -1),
    (dict(k_pages=None), -1), (dict(block=32), -2), (dict(dtype=7), -2), (dict(D=120, rot=16), -2), (dict(rot=24), -2),
    (dict(D=512), -2), (dict(q=4104), -2), (dict(pooled_q=4100), -2), (dict(max_pages=1 << 28), -5), (dict(B=70000), -5),
])
def test_rope_refusals(change, status):
    assert L.lib().tasft_rope_append_paged(C.byref(rope_args(**change)), None) == status


def select_args(**kw):
    a = L.SelectArgs(scores=4096, cu_seqlens=4096, kv_len=4096, B=2, Hq=8, Hk=2, NBq=1, NBk=50, block=64, top_k=8,
                     first=1, local=1, width=8, kept_idx=4096, kept_cnt=4096)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("change,status", [
    (dict(scores=None), -1), (dict(kept_cnt=None), -1), (dict(B=0), -1), (dict(Hq=9), -1), (dict(NBk=0), -1),
    (dict(top_k=0), -1), (dict(first=-1), -1), (dict(local=0), -1), (dict(width=7), -1), (dict(first=9, width=9), -1),
    (dict(NBk=16385, width=8), -5), (dict(block=48), -2), (dict(B=70000), -5),
])
def test_select_refusals(change, status):
    assert L.lib().tasft_select_blocks(C.byref(select_args(**change)), None) == status


def test_calls_refuse_host_tensors():
    x = torch.zeros(4, 8, 128, dtype=torch.bfloat16)
    p = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, 2, dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: T.bsa_chunk_paged(x, p, p, i, torch.zeros(3), n, 4),
                 lambda: T.rope_append_paged(x, x, x, torch.zeros(64), p, p, i, torch.zeros(3), n, 4),
                 lambda: T.select_blocks(torch.zeros(2, 8, 1, 4), 2, torch.zeros(3), n, 4)):
        with pytest.raises(T.KernelError):
            call()


def test_chunk_rows():
    for n in range(1, 300):
        assert T.chunk_rows(n) == max((c % 64 + n + 63) // 64 for c in range(64))


def test_frequencies():
    f, a = T.rope_inv_freq(128, 10000.0)
    assert a == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([10000.0 ** (-i / 64) for i in range(64)], dtype=torch.float64), rtol=1e-14)
    g, _ = T.rope_inv_freq(128, 10000.0, {"type": "linear", "factor": 4})
    assert torch.equal(g, f / 4)
    # llama3: short wavelengths kept, long ones divided, a monotone blend between
    s = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
             original_max_position_embeddings=8192)
    f, _ = T.rope_inv_freq(128, 500000.0)
    g, _ = T.rope_inv_freq(128, 500000.0, s)
    wave = 2 * math.pi / f
    assert torch.equal(g[wave < 8192 / 4], f[wave < 8192 / 4])
    assert torch.equal(g[wave > 8192], f[wave > 8192] / 8)
    ratio = f / g
    assert ((ratio[1:] - ratio[:-1]) >= -1e-12).all() and ratio.max() == 8.0 and ((ratio > 1.01) & (ratio < 7.9)).any()
    # yarn: pairs that turn more than 32 times in the original context are kept, less than once divided
    s = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)
    f, _ = T.rope_inv_freq(128, 1e6)
    g, a = T.rope_inv_freq(128, 1e6, s)
    turns = 32768 * f / (2 * math.pi)
    assert a == pytest.approx(0.1 * math.log(4) + 1)
    assert torch.equal(g[turns > 40], f[turns > 40]) and torch.allclose(g[turns < 0.9], f[turns < 0.9] / 4, rtol=1e-14)
    assert T.rope_inv_freq(128, 1e6, dict(s, attention_factor=1.25))[1] == 1.25
    for bad in ({"rope_type": "longrope"}, {"rope_type": "linear"}, {"rope_type": "linear", "factor": 0.5},
                {"rope_type": "llama3", "factor": 8.0}):
        with pytest.raises(T.ValidationError):
            T.rope_inv_freq(64, 10000.0, bad)
    with pytest.raises(T.ValidationError):
        T.rope_inv_freq(63)


@pytest.mark.parametrize("max_q", [2**31 - 126, 2**31 - 1])
def test_rows_for_the_largest_counts_do_not_wrap(max_q):
    """Too few rows for so many new tokens, although max_q + 126 leaves 32 bits."""
    lists = dict(kept_idx=4096, kept_cnt=4096, Hm=2, nb_q=2, nb_w=4)
    assert L.lib().tasft_bsa_chunk_paged_fwd(C.byref(chunk_args(max_q=max_q, **lists)), None) == -1
    assert L.lib().tasft_rope_append_paged(C.byref(rope_args(max_q=max_q)), None) == -1


@pytest.mark.parametrize("fields", [dict(max_q=2**31), dict(B=-(2**31) - 1), dict(scale=1e300)])
def test_numbers_that_do_not_fit_their_field_are_refused(fields):
    values = []
    for name, kind in L.ChunkArgs._fields_:
        values += [fields.get(name, 0)] * getattr(kind, "_length_", 1)
    with pytest.raises(T.KernelError):
        L.packed(L.ChunkArgs)(*values)


def test_an_infinite_scale_is_refused():
    assert L.lib().tasft_bsa_chunk_paged_fwd(C.byref(chunk_args(scale=math.inf)), None) == -1
