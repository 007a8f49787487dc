"""Edges of the paged serving calls that their host side decides (no GPU)."""
from __future__ import annotations

import ctypes as C
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import tasft_b200 as T
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


def yarn(i, dim, base, factor, original, fast=32.0, slow=1.0, truncate=True):
    """Frequency i from the definition: pairs that turn more than ``fast`` times within the original
    context stay, those that turn less than ``slow`` times are divided, a ramp over i between."""
    def place(turns):  # the i (not whole) whose pair turns so often
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
    lo, hi = place(fast), place(slow)
    if truncate:
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, dim - 1)
    part = min(1.0, max(0.0, (i - lo) / (hi - lo)))
    f = base ** (-2 * i / dim)
    return f * (1 - part) + f / factor * part


@pytest.mark.parametrize("dim,base,factor,original", [(64, 150000.0, 32.0, 4096), (128, 1e6, 4.0, 32768),
                                                      (64, 10000.0, 40.0, 4096)])
@pytest.mark.parametrize("extra", [{}, {"truncate": True}, {"truncate": False}, {"beta_fast": 16.0, "truncate": False},
                                   {"beta_slow": 2.0}])
def test_yarn_frequencies_with_their_options(dim, base, factor, original, extra):
    f, a = T.rope_inv_freq(dim, base, dict(rope_type="yarn", factor=factor, original_max_position_embeddings=original,
                                           **extra))
    want = [yarn(i, dim, base, factor, original, extra.get("beta_fast", 32.0), extra.get("beta_slow", 1.0),
                 extra.get("truncate", True)) for i in range(dim // 2)]
    assert torch.allclose(f, torch.tensor(want, dtype=torch.float64), rtol=1e-12, atol=0)
    assert a == pytest.approx(0.1 * math.log(factor) + 1, rel=1e-15)


def test_yarn_factor_on_cos_and_sin():
    s = dict(rope_type="yarn", factor=40.0, original_max_position_embeddings=4096)
    m = lambda c: 0.1 * c * math.log(40.0) + 1  # noqa: E731
    for extra, want in (({}, m(1)), ({"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0),
                        ({"mscale": 0.707, "mscale_all_dim": 1.0}, m(0.707) / m(1)), ({"mscale": 1.0}, m(1)),
                        ({"mscale": 1.0, "mscale_all_dim": 0.0}, m(1)), ({"mscale": None, "mscale_all_dim": None}, m(1)),
                        ({"mscale": 1.0, "mscale_all_dim": 2.0, "attention_factor": 1.25}, 1.25)):
        assert T.rope_inv_freq(64, 10000.0, dict(s, **extra))[1] == pytest.approx(want, rel=1e-15), extra
    assert T.rope_inv_freq(64, 10000.0, dict(s, factor=1.0, mscale=1.0, mscale_all_dim=0.5))[1] == 1.0
    # one of the two alone means different things to different models
    for extra in ({"mscale": 0.707}, {"mscale_all_dim": 1.0}, {"mscale": 0.707, "mscale_all_dim": 0.0}):
        with pytest.raises(T.ValidationError):
            T.rope_inv_freq(64, 10000.0, dict(s, **extra))


LLAMA3 = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
              original_max_position_embeddings=8192)
YARN = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=32768)


@pytest.mark.parametrize("scaling", [None, {"rope_type": "linear", "factor": 4.0}, LLAMA3, YARN])
def test_options_that_would_change_the_result_are_not_dropped(scaling):
    """An option that nothing here computes is refused; one that says what the call says already, or
    that belongs to another kind, is not."""
    s = scaling or {"rope_type": "default"}
    want = T.rope_inv_freq(64, 5e5, scaling)
    for extra in ({"rope_theta": 5e5}, {"partial_rotary_factor": 0.5}, {"type": s["rope_type"]}, {"unknown": None},
                  {"finetuned": True}, {"original_max_position_embeddings": 32768 if s is YARN else 8192}):
        got = T.rope_inv_freq(64, 5e5, {**s, **extra})
        assert torch.equal(got[0], want[0]) and got[1] == want[1]
    for extra in ({"rope_theta": 1e4}, {"mrope_section": [16, 24, 24]}, {"attn_factor": 1.2},
                  {"long_factor": [1.0] * 32}, {"extrapolation_factor": 0.5}):
        with pytest.raises(T.ValidationError):
            T.rope_inv_freq(64, 5e5, {**s, **extra})


@pytest.mark.parametrize("args", [
    (64, math.nan), (64, math.inf), (64, 1.0, YARN), (64, 1e4, {**YARN, "original_max_position_embeddings": 0}),
    (64, 1e4, {**YARN, "original_max_position_embeddings": -4096}), (64, 1e4, {**YARN, "beta_fast": -1.0}),
    (64, 1e4, {**YARN, "factor": math.inf}), (64, 1e4, {**YARN, "factor": math.nan}),
    (64, 1e4, {**YARN, "beta_slow": math.inf}), (64, 1e4, {**LLAMA3, "original_max_position_embeddings": math.inf}),
    (64, 1e4, {**LLAMA3, "low_freq_factor": math.nan}), (64, 1e4, {**YARN, "attention_factor": math.nan}),
    (64, 1e4, {**YARN, "factor": "wide"}), (64, 1e4, {**YARN, "mscale": 1.0, "mscale_all_dim": -3.0}),
])
def test_numbers_without_a_meaning_are_refused(args):
    with pytest.raises(T.ValidationError):
        T.rope_inv_freq(*args)


def test_options_that_are_not_known_are_refused():
    a = L.RopeAppendArgs(q=4096, k=4096, v=4096, q_out=4096, k_pages=4096, v_pages=4096, inv_freq=4096,
                         block_table=4096, cu_seqlens=4096, kv_len=4096, factor=1.0, B=2, T=5, Hq=8, Hk=2, D=128, rot=128,
                         block=64, dtype=L.BF16, max_q=4, max_pages=4, page_size=16, num_pages=9, NBq=2, NBk=4)
    for options in (1 << 10, -1):
        assert L.lib().tasft_rope_append_paged_opt(C.byref(a), options, None) == -1
        assert L.lib().tasft_bsa_chunk_paged_fwd_opt(C.byref(chunk_args()), options, None) == -1
    assert L.lib().tasft_rope_append_paged_opt(None, 0, None) == L.lib().tasft_bsa_chunk_paged_fwd_opt(None, 0, None) == -1


@pytest.mark.parametrize("cname,pyname", [("tasft_rope_append_args", "RopeAppendArgs"), ("tasft_select_args", "SelectArgs"),
                                          ("tasft_chunk_args", "ChunkArgs")])
def test_argument_blocks_match_the_header(tmp_path, cname, pyname):
    """Fields where the compiler lays them out, as ctypes and as packed bytes."""
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    cls = getattr(L, pyname)
    header = Path(L.__file__).resolve().parent.parent / "include" / "tasft_b200.h"
    lines = ["#include <stddef.h>", "#include <stdio.h>", f'#include "{header}"', "int main(void) {",
             f'  printf("%zu\\n", sizeof({cname}));']
    lines += [f'  printf("%zu\\n", offsetof({cname}, {name}));' for name, _ in cls._fields_] + ["  return 0;", "}"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-std=c11", "-o", str(exe), str(tmp_path / "layout.c")], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [C.sizeof(cls)] + [getattr(cls, name).offset for name, _ in cls._fields_]
    values, block, n = [], cls(), 0
    for name, kind in cls._fields_:
        many = getattr(kind, "_length_", 0)
        mine = [n + i + 1 for i in range(max(many, 1))]
        n += len(mine)
        values += mine
        if many:
            getattr(block, name)[:] = mine
        else:
            setattr(block, name, mine[0])
    assert L.packed(cls)(*values) == bytes(block)
