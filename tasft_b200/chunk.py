"""A serving step over a paged KV cache with chunked prompts: rotary append, block choice and
attention of the new tokens.

New capability: the reference's vLLM backend flattens prefill tokens into one sequence without
a cache and hands decode to a dense kernel (``tasft/inference/vllm_patch.py:172-196``). Here a
batch is the new tokens of B sequences packed along the token axis, chunks of prompts and single
tokens alike: sequence b is rows ``cu_seqlens[b]:cu_seqlens[b+1]``, the last of its ``kv_len[b]``
tokens, cached in the pages ``block_table[b]``. Blocks are 64 tokens; row i of a sequence's block
means, scores and lists stands for the i-th block that its new tokens touch, block
``(kv_len[b] - new) // 64 + i``, of at most :func:`chunk_rows` rows.

A step of one layer::

    q, pooled_q = rope_append_paged(q, k, v, inv_freq, k_pages, v_pages, table, cu, kv_len, max_new,
                                    pooled_k=means)
    soft = gate.forward_pooled(pooled_q, means, ...).soft_scores
    kept = select_blocks(soft, Hk, cu, kv_len, top_k)
    out = bsa_chunk_paged(q, k_pages, v_pages, table, cu, kv_len, max_new, kept)
"""
from __future__ import annotations

import math

import torch

from tasft_b200 import _lib as L
from tasft_b200.exceptions import KernelError, ValidationError
from tasft_b200.types import KeptBlocks

BLOCK = 64


def chunk_rows(max_new: int) -> int:
    """Most 64-token blocks that ``max_new`` consecutive tokens touch."""
    return (max_new + 126) // BLOCK


def rope_inv_freq(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None,
                  device=None) -> tuple[torch.Tensor, float]:
    """Rotary frequencies ``[rotary_dim / 2]`` (fp64, radians per position) and the factor on cos and
    sin, for :func:`rope_append_paged`. ``scaling`` is a model configuration's dictionary, with the
    kind under ``rope_type`` (or ``type``):

    * ``default``: ``f_i = base^(-2i / rotary_dim)``;
    * ``linear``: ``f_i / factor``;
    * ``llama3``: with ``t_i = original_max_position_embeddings * f_i / 2pi`` turns within the
      original context and ``b = clip((t_i - low_freq_factor) / (high_freq_factor -
      low_freq_factor), 0, 1)``: ``f_i (b + (1 - b) / factor)``;
    * ``yarn``: with ``d(t) = rotary_dim * ln(original / (2pi t)) / (2 ln base)``, ``lo =
      max(floor(d(beta_fast)), 0)``, ``hi = min(ceil(d(beta_slow)), rotary_dim - 1)`` and ``r =
      clip((i - lo) / (hi - lo), 0, 1)``: ``f_i ((1 - r) + r / factor)``; cos and sin are scaled by
      ``attention_factor``, ``0.1 ln(factor) + 1`` unless given.
    """
    if rotary_dim <= 0 or rotary_dim % 2 or base <= 0:
        raise ValidationError("rotary_dim must be even and positive, base positive",
                              context={"rotary_dim": rotary_dim, "base": base})
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = float(base) ** (-2.0 * i / rotary_dim)
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    attention = 1.0
    if kind == "default":
        pass
    elif kind in ("linear", "llama3", "yarn"):
        need = {"linear": ("factor",),
                "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
                "yarn": ("factor", "original_max_position_embeddings")}[kind]
        missing = [n for n in need if scaling.get(n) is None]
        if missing or not float(scaling["factor"]) >= 1.0:
            raise ValidationError(f"rope scaling '{kind}' needs {', '.join(need)}, factor at least 1",
                                  context={"scaling": dict(scaling)})
        factor = float(scaling["factor"])
        if kind == "linear":
            f = f / factor
        elif kind == "llama3":
            low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
            if not high > low:
                raise ValidationError("high_freq_factor must be above low_freq_factor",
                                      context={"scaling": dict(scaling)})
            turns = float(scaling["original_max_position_embeddings"]) * f / (2 * math.pi)
            blend = ((turns - low) / (high - low)).clamp(0.0, 1.0)
            f = f * (blend + (1 - blend) / factor)
        else:
            original = float(scaling["original_max_position_embeddings"])

            def dim_of(t: float) -> float:
                return rotary_dim * math.log(original / (2 * math.pi * t)) / (2 * math.log(base))

            lo = max(math.floor(dim_of(float(scaling.get("beta_fast") or 32.0))), 0)
            hi = min(math.ceil(dim_of(float(scaling.get("beta_slow") or 1.0))), rotary_dim - 1)
            ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
            f = f * ((1 - ramp) + ramp / factor)
            given = scaling.get("attention_factor")
            attention = float(given) if given is not None else (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
    else:
        raise ValidationError(f"unknown rope scaling '{kind}'", context={"scaling": dict(scaling)})
    return (f if device is None else f.to(device)), attention


def _batch(name: str, device, block_table, cu_seqlens, kv_len):
    """The batch's int32 index tensors on the tensors' device, contiguous."""
    B = kv_len.shape[0] if kv_len.ndim == 1 else -1
    if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] != B + 1 or B <= 0 or (
            block_table is not None and (block_table.ndim != 2 or block_table.shape[0] != B)):
        raise KernelError(f"{name}: expects cu_seqlens [B + 1], kv_len [B] and block_table [B, max_pages]",
                          context={"cu_seqlens": list(cu_seqlens.shape), "kv_len": list(kv_len.shape),
                                   "table": None if block_table is None else list(block_table.shape)})
    out = []
    for t in (block_table, cu_seqlens, kv_len):
        if t is not None:
            if t.device != device:
                raise KernelError(f"{name}: tensors on different devices",
                                  context={"device": str(device), "got": str(t.device)})
            if t.dtype != torch.int32:
                t = t.to(torch.int32)
            if not t.is_contiguous():
                t = t.contiguous()
        out.append(t)
    return B, *out


def _check_pages(name: str, q, k_pages, v_pages) -> None:
    if q.ndim != 3 or k_pages.ndim != 4 or k_pages.shape != v_pages.shape or k_pages.shape[3] != q.shape[2] \
            or k_pages.shape[2] == 0 or q.shape[1] == 0 or q.shape[1] % k_pages.shape[2]:
        raise KernelError(f"{name}: expects q [T, Hq, D] and pages [num_pages, page_size, Hk, D], Hq a multiple of Hk",
                          context={"q": list(q.shape), "k_pages": list(k_pages.shape), "v_pages": list(v_pages.shape)})
    if k_pages.dtype != q.dtype or v_pages.dtype != q.dtype:
        raise KernelError(f"{name}: q and the pages must have one dtype",
                          context={"q": str(q.dtype), "k": str(k_pages.dtype), "v": str(v_pages.dtype)})
    if k_pages.device != q.device or v_pages.device != q.device:
        raise KernelError(f"{name}: tensors on different devices",
                          context={"q": str(q.device), "k": str(k_pages.device), "v": str(v_pages.device)})


def _check_err(name: str, device, err) -> None:
    if err is not None and (err.dtype != torch.int32 or err.numel() < 1 or err.device != device):
        raise KernelError(f"{name}: err must be an int32 tensor on the same device",
                          context={"dtype": str(err.dtype), "device": str(err.device)})


def rope_append_paged(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    inv_freq: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    kv_len: torch.Tensor,
    max_new: int,
    *,
    interleaved: bool = False,
    attention_scaling: float = 1.0,
    pooled_k: torch.Tensor | None = None,
    block: int = BLOCK,
    out: torch.Tensor | None = None,
    err: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotate the new tokens at their positions, append k and v to the cache and keep the gate's
    block means (``tasft_rope_append_paged``).

    q ``[T, Hq, D]``, k, v ``[T, Hk, D]`` (slices of a fused projection are fine), ``inv_freq``
    ``[rot / 2]`` fp64 or fp32 as :func:`rope_inv_freq` gives it: the first ``rot`` columns of a head
    turn, in pairs ``(i, i + rot/2)`` or, ``interleaved``, ``(2i, 2i + 1)``; cos and sin are multiplied
    by ``attention_scaling``. ``max_new``: most new tokens of a sequence. With ``pooled_k`` (fp32
    ``[B, Hk, NBk, D]``, updated in place: the mean of every key block that got new tokens) also
    computes the means of the new queries. Returns ``(q, pooled_q)``: rotated q (``out``, which may
    be q itself) and fp32 ``[B, Hq, chunk_rows(max_new), D]`` or None, for
    :meth:`AttnGate.forward_pooled`. f32 / bf16 / f16; D and rot multiples of 16 (8 in f32), D up to
    256. The packed, paged counterpart of :func:`qkv_rope_pool`, which takes cos and sin as tables."""
    name = "rope_append_paged"
    L.require_cuda(q, k, v, inv_freq, k_pages, v_pages, block_table, cu_seqlens, kv_len)
    _check_pages(name, q, k_pages, v_pages)
    T, Hq, D = q.shape
    num_pages, page_size, Hk, _ = k_pages.shape
    if k.shape != (T, Hk, D) or v.shape != k.shape or k.dtype != q.dtype or v.dtype != q.dtype:
        raise KernelError(f"{name}: expects k, v [T, Hk, D] in q's dtype",
                          context={"q": list(q.shape), "k": list(k.shape), "v": list(v.shape)})
    if block != BLOCK or max_new <= 0:
        raise KernelError(f"{name}: block must be {BLOCK}, max_new positive",
                          context={"block": block, "max_new": max_new})
    if inv_freq.ndim != 1 or inv_freq.dtype not in (torch.float64, torch.float32):
        raise KernelError(f"{name}: inv_freq must be [rot / 2], fp64 or fp32",
                          context={"shape": list(inv_freq.shape), "dtype": str(inv_freq.dtype)})
    dev = q.device
    B, table, cu, kvl = _batch(name, dev, block_table, cu_seqlens, kv_len)
    _check_err(name, dev, err)
    rows = chunk_rows(max_new)
    nbk = 0
    pooled_q = None
    if pooled_k is not None:
        if pooled_k.ndim != 4 or pooled_k.dtype != torch.float32 or not pooled_k.is_contiguous() or \
                pooled_k.device != dev or pooled_k.shape[:2] != (B, Hk) or pooled_k.shape[3] != D:
            raise KernelError(f"{name}: pooled_k must be contiguous fp32 [B, Hk, NBk, D]",
                              context={"pooled_k": list(pooled_k.shape), "dtype": str(pooled_k.dtype)})
        nbk = pooled_k.shape[2]
        pooled_q = torch.empty(B, Hq, rows, D, dtype=torch.float32, device=dev)
    if out is None:
        out = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1:
        raise KernelError(f"{name}: out must match q", context={"q": list(q.shape), "out": list(out.shape)})
    q, k, v = (x if x.stride(2) == 1 else x.contiguous() for x in (q, k, v))
    freq = inv_freq if inv_freq.is_contiguous() else inv_freq.contiguous()
    with L.on_device(q):
        args = L.RopeAppendArgs(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            L.I64x2(*q.stride()[:2]), L.I64x2(*k.stride()[:2]), L.I64x2(*v.stride()[:2]), L.I64x2(*out.stride()[:2]),
            L.strides4(k_pages), L.strides4(v_pages), freq.data_ptr(), table.data_ptr(), cu.data_ptr(), kvl.data_ptr(),
            L.ptr(pooled_q), L.ptr(pooled_k), float(attention_scaling), B, T, Hq, Hk, D, 2 * freq.shape[0], block,
            L.dtype_code(q), int(max_new), table.shape[1], page_size, num_pages, rows, nbk, int(interleaved),
            int(freq.dtype == torch.float64), L.ptr(err))
        L.check(L.lib().tasft_rope_append_paged(args, L.stream_ptr(dev)), "tasft_rope_append_paged",
                shape=[B, T, Hq, Hk, D], page_size=page_size)
    return out, pooled_q


def select_blocks(
    scores: torch.Tensor,
    num_kv_heads: int,
    cu_seqlens: torch.Tensor,
    kv_len: torch.Tensor,
    top_k: int,
    *,
    tau: float | None = None,
    first: int = 1,
    local: int = 1,
    block: int = BLOCK,
    err: torch.Tensor | None = None,
) -> KeptBlocks:
    """Kept blocks by score for the new tokens of a packed batch (``tasft_select_blocks``).

    ``scores`` fp32 ``[B, Hq, NBq, NBk]`` (gate scores; row i as in the module's notes). Each row
    keeps its ``first`` blocks, the ``local`` blocks up to its own and the best of the others,
    ``top_k`` in all; a block's score is the highest of its group's query heads, ties go to the
    lowest index, scores of -inf or NaN, or below ``tau`` where given, are not chosen. Returns
    ascending lists ``[B, Hk, NBq, min(NBk, max(top_k, first + local))]`` for
    :func:`bsa_chunk_paged`; rows that no new token falls in keep nothing. For
    :func:`bsa_decode_paged` take row 0 (``idx[:, :, 0]``, ``cnt[:, :, 0]``). Beside
    :func:`threshold_scores`, which keeps by threshold alone."""
    name = "select_blocks"
    L.require_cuda(scores, cu_seqlens, kv_len)
    if scores.ndim != 4 or scores.dtype != torch.float32 or num_kv_heads <= 0 or scores.shape[1] % num_kv_heads:
        raise KernelError(f"{name}: expects fp32 scores [B, Hq, NBq, NBk], Hq a multiple of num_kv_heads",
                          context={"scores": list(scores.shape), "dtype": str(scores.dtype), "Hk": num_kv_heads})
    if top_k <= 0 or first < 0 or local < 1 or block <= 0:
        raise ValidationError(f"{name}: top_k and local must be positive, first not negative",
                              context={"top_k": top_k, "first": first, "local": local, "block": block})
    dev = scores.device
    B, _, cu, kvl = _batch(name, dev, None, cu_seqlens, kv_len)
    if scores.shape[0] != B:
        raise KernelError(f"{name}: scores and kv_len disagree about the batch",
                          context={"scores": list(scores.shape), "kv_len": list(kv_len.shape)})
    _check_err(name, dev, err)
    if scores.stride(3) != 1:
        scores = scores.contiguous()
    _, Hq, nbq, nbk = scores.shape
    width = min(nbk, max(top_k, first + local))
    idx = torch.empty(B, num_kv_heads, nbq, width, dtype=torch.int32, device=dev)
    cnt = torch.empty(B, num_kv_heads, nbq, dtype=torch.int32, device=dev)
    with L.on_device(scores):
        args = L.SelectArgs(
            scores.data_ptr(), L.I64x3(*scores.stride()[:3]), cu.data_ptr(), kvl.data_ptr(), B, Hq, num_kv_heads, nbq,
            nbk, block, min(top_k, nbk), min(first, nbk), min(local, nbk), int(tau is not None),
            0.0 if tau is None else float(tau), width, idx.data_ptr(), cnt.data_ptr(), L.ptr(err))
        L.check(L.lib().tasft_select_blocks(args, L.stream_ptr(dev)), "tasft_select_blocks",
                shape=[B, Hq, num_kv_heads, nbq, nbk])
    return KeptBlocks(idx, cnt)


def bsa_chunk_paged(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens: torch.Tensor,
    kv_len: torch.Tensor,
    max_new: int,
    kept: KeptBlocks | None = None,
    block: int = BLOCK,
    *,
    scale: float | None = None,
    out: torch.Tensor | None = None,
    err: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of the new tokens of a packed batch over a paged KV cache
    (``tasft_bsa_chunk_paged_fwd``), causal: a token sees its sequence's cached keys up to its
    own, in the blocks its list keeps (all of them without ``kept``).

    q ``[T, Hq, D]``, pages ``[num_pages, page_size, Hk, D]`` with the new keys and values already
    in them (:func:`rope_append_paged`), ``kept`` lists ``[B, Hk or Hq, NBq, W]`` with at least
    ``chunk_rows(max_new)`` rows, ascending. ``scale`` defaults to ``1 / sqrt(D)``. Returns
    ``[T, Hq, D]`` (``out``; rows outside all sequences stay as they were); a token with nothing
    kept gets 0. ``err``: optional int32 error word, see ``include/tasft_b200.h``. bf16 / f16, D 64
    or 128, page size 16, 32, 64 or 128. What the cache holds from ``kv_len`` on, or in blocks no
    list keeps, is never read into the result; a non-finite value of a kept block's own token
    spreads as the softmax formula has it. Beside :func:`bsa_decode_paged` (one token per sequence) and
    :meth:`BlockSparseFlashAttention.forward_varlen` (no cache)."""
    name = "bsa_chunk_paged"
    L.require_cuda(q, k_pages, v_pages, block_table, cu_seqlens, kv_len)
    _check_pages(name, q, k_pages, v_pages)
    T, Hq, D = q.shape
    num_pages, page_size, Hk, _ = k_pages.shape
    dev = q.device
    B, table, cu, kvl = _batch(name, dev, block_table, cu_seqlens, kv_len)
    _check_err(name, dev, err)
    if max_new <= 0:
        raise KernelError(f"{name}: max_new must be positive", context={"max_new": max_new})
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise KernelError(f"{name}: scale must be positive and finite", context={"scale": scale})
    idx = cnt = None
    hm = rows = width = 0
    if kept is not None:
        idx, cnt = kept.idx, kept.cnt
        if idx.ndim != 4 or idx.shape[0] != B or idx.shape[1] not in (Hq, Hk) or cnt.shape != idx.shape[:3] or \
                idx.shape[2] < chunk_rows(max_new) or idx.shape[3] == 0 or idx.device != dev or cnt.device != dev:
            raise KernelError(f"{name}: kept lists must be [B, Hk or Hq, at least {chunk_rows(max_new)}, W]",
                              context={"idx": list(idx.shape), "cnt": list(cnt.shape)})
        if idx.dtype != torch.int32 or not idx.is_contiguous():
            idx = idx.to(torch.int32).contiguous()
        if cnt.dtype != torch.int32 or not cnt.is_contiguous():
            cnt = cnt.to(torch.int32).contiguous()
        _, hm, rows, width = idx.shape
    if out is None:
        out = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1:
        raise KernelError(f"{name}: out must match q", context={"q": list(q.shape), "out": list(out.shape)})
    if q.stride(2) != 1 or q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
        q = q.contiguous()
    lib = L.lib()
    with L.on_device(q):
        nbytes = lib.tasft_chunk_workspace_size(B, T, Hq, Hk, D, max_new, hm)
        if nbytes < 0:
            L.check(int(nbytes), "tasft_chunk_workspace_size", shape=[B, T, Hq, Hk, D])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        args = L.ChunkArgs(
            q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), L.I64x2(*q.stride()[:2]),
            L.I64x2(*out.stride()[:2]), L.strides4(k_pages), L.strides4(v_pages), table.data_ptr(), cu.data_ptr(),
            kvl.data_ptr(), L.ptr(idx), L.ptr(cnt), B, T, Hq, Hk, D, block, L.dtype_code(q), max_new, table.shape[1],
            page_size, num_pages, hm, rows, width, scale, ws.data_ptr(), nbytes, L.ptr(err))
        L.check(lib.tasft_bsa_chunk_paged_fwd(args, L.stream_ptr(dev)), "tasft_bsa_chunk_paged_fwd",
                shape=[B, T, Hq, Hk, D], page_size=page_size)
    return out


__all__ = ["bsa_chunk_paged", "chunk_rows", "rope_append_paged", "rope_inv_freq", "select_blocks"]
