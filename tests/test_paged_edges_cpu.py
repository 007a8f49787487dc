"""Edges of the paged serving calls that their host side decides (no GPU)."""
from __future__ import annotations

import ctypes as C

import pytest

from tasft_b200 import _lib as L


def chunk_args(**kw):
    a = L.ChunkArgs(q=4096, k_pages=4096, v_pages=4096, out=4096, block_table=4096, cu_seqlens=4096, kv_len=4096,
                    B=2, T=5, Hq=8, Hk=2, D=128, block=64, dtype=L.BF16, max_q=4, max_pages=4, page_size=16,
                    num_pages=9, scale=0.1, workspace=4096, workspace_bytes=1 << 30)
    a.q_stride[:] = a.o_stride[:] = [1024, 128]
    a.k_stride[:] = a.v_stride[:] = [4096, 256, 128, 1]
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("at", [4096 + 4, 4096 + 8, 4096 + 16, 4096 + 48])
def test_a_workspace_off_32_byte_boundaries_is_refused(at):
    """Partial results are stored 32 bytes at a time."""
    assert L.lib().tasft_bsa_chunk_paged_fwd(C.byref(chunk_args(workspace=at)), None) == -4
