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
                                    pooled_k=means, query_mean="new")
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
      max(floor(d(beta_fast)), 0)``, ``hi = min(ceil(d(beta_slow)), rotary_dim - 1)`` (neither rounded
      where ``truncate`` is false) and ``r = clip((i - lo) / (hi - lo), 0, 1)``: ``f_i ((1 - r) + r /
      factor)``. Cos and sin are scaled by ``attention_factor`` where given; with ``m(c) = 0.1 c
      ln(factor) + 1``, by ``m(mscale) / m(mscale_all_dim)`` where both are, else by ``m(1)``. (What
      such a model multiplies its softmax scale with is the caller's, as ``scale`` of
      :func:`bsa_chunk_paged`.) One of the two alone, where that is not ``m(1)`` either way of reading
      it, is refused.

    Options of the other kinds are passed over, as is one that is None. Any other option would change
    the result and is refused, a ``rope_theta`` that is not ``base`` among them.
    """
    if rotary_dim <= 0 or rotary_dim % 2 or not 0.0 < base < math.inf:
        raise ValidationError("rotary_dim must be even and positive, base positive",
                              context={"rotary_dim": rotary_dim, "base": base})
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    f = float(base) ** (-2.0 * i / rotary_dim)
    scaling = scaling or {}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    strange = [n for n, x in scaling.items() if n not in _SCALING and x is not None]
    if strange or scaling.get("rope_theta") not in (None, base):
        raise ValidationError(f"rope scaling '{kind}': {', '.join(strange) or 'rope_theta'} would change the result",
                              context={"scaling": dict(scaling), "base": base})
    attention = 1.0
    if kind == "default":
        pass
    elif kind in ("linear", "llama3", "yarn"):
        need = {"linear": ("factor",),
                "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
                "yarn": ("factor", "original_max_position_embeddings")}[kind]
        missing = [n for n in need if scaling.get(n) is None]
        if missing or not _number(scaling, "factor") >= 1.0:
            raise ValidationError(f"rope scaling '{kind}' needs {', '.join(need)}, factor at least 1",
                                  context={"scaling": dict(scaling)})
        factor = _number(scaling, "factor")
        if kind == "linear":
            f = f / factor
        elif kind == "llama3":
            low, high = _number(scaling, "low_freq_factor"), _number(scaling, "high_freq_factor")
            if not high > low:
                raise ValidationError("high_freq_factor must be above low_freq_factor",
                                      context={"scaling": dict(scaling)})
            turns = _number(scaling, "original_max_position_embeddings") * f / (2 * math.pi)
            blend = ((turns - low) / (high - low)).clamp(0.0, 1.0)
            f = f * (blend + (1 - blend) / factor)
        else:
            original = _number(scaling, "original_max_position_embeddings")
            fast, slow = (_number(scaling, n) if scaling.get(n) else x for n, x in (("beta_fast", 32.0), ("beta_slow", 1.0)))
            if not (original > 0 and fast > 0 and slow > 0 and base > 1):
                raise ValidationError("yarn needs a base above 1, original length and betas above 0",
                                      context={"scaling": dict(scaling), "base": base})

            def dim_of(t: float) -> float:
                return rotary_dim * math.log(original / (2 * math.pi * t)) / (2 * math.log(base))

            lo, hi = dim_of(fast), dim_of(slow)
            if scaling.get("truncate") is None or scaling["truncate"]:
                lo, hi = math.floor(lo), math.ceil(hi)
            lo, hi = max(lo, 0), min(hi, rotary_dim - 1)
            ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
            f = f * ((1 - ramp) + ramp / factor)
            attention = _yarn_attention(scaling, factor)
    else:
        raise ValidationError(f"unknown rope scaling '{kind}'", context={"scaling": dict(scaling)})
    return (f if device is None else f.to(device)), attention


# what a scaling dictionary may hold; a kind takes no notice of the other kinds' options
_SCALING = frozenset((
    "rope_type", "type", "factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor",
    "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate",
    "rope_theta",             # the base: as the call's
    "partial_rotary_factor",  # in rotary_dim already
    "finetuned",              # how the weights came about
))


def _number(scaling: dict, name: str) -> float:
    try:
        x = float(scaling[name])
    except (TypeError, ValueError):
        x = math.nan
    if not math.isfinite(x):
        raise ValidationError(f"rope scaling: {name} must be a finite number", context={"scaling": dict(scaling)})
    return x


def _yarn_attention(scaling: dict, factor: float) -> float:
    """The factor on cos and sin of ``yarn``."""
    given, part, whole = (_number(scaling, n) if scaling.get(n) is not None else None
                          for n in ("attention_factor", "mscale", "mscale_all_dim"))

    def m(c: float) -> float:
        return 0.1 * c * math.log(factor) + 1.0

    if given is not None:
        return given
    if part and whole and part > 0 and whole > 0:
        return m(part) / m(whole)
    if whole or part not in (None, 1.0):
        raise ValidationError("yarn needs mscale and mscale_all_dim together (or attention_factor)",
                              context={"scaling": dict(scaling)})
    return m(1.0)


_rope_args = L.packed(L.RopeAppendArgs)
_select_args = L.packed(L.SelectArgs)
_chunk_args = L.packed(L.ChunkArgs)


def _index(name: str, t: torch.Tensor, gpu: int, n: int, ndim: int = 1) -> torch.Tensor:
    """An index tensor ``[n]`` (``[n, any]``) on the batch's device as contiguous int32."""
    if t.get_device() != gpu or t.dim() != ndim or t.size(0) != n:
        raise KernelError(f"{name}: expects cu_seqlens [B + 1], kv_len [B] and block_table [B, max_pages] on one device",
                          context={"shape": list(t.shape), "rows": n, "device": str(t.device)})
    return t if t.dtype is torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _check_pages(name: str, gpu: int, q, qs, k_pages, ks, v_pages) -> None:
    if len(qs) != 3 or len(ks) != 4 or ks != v_pages.shape or ks[3] != qs[2] or not ks[2] or not qs[1] or qs[1] % ks[2]:
        raise KernelError(f"{name}: expects q [T, Hq, D] and pages [num_pages, page_size, Hk, D], Hq a multiple of Hk",
                          context={"q": list(qs), "k_pages": list(ks), "v_pages": list(v_pages.shape)})
    if k_pages.dtype is not q.dtype or v_pages.dtype is not q.dtype:
        raise KernelError(f"{name}: q and the pages must have one dtype",
                          context={"q": str(q.dtype), "k": str(k_pages.dtype), "v": str(v_pages.dtype)})
    if gpu < 0 or k_pages.get_device() != gpu or v_pages.get_device() != gpu:
        raise KernelError(f"{name}: tensors must be on one CUDA device",
                          context={"q": str(q.device), "k": str(k_pages.device), "v": str(v_pages.device)})


def _err_ptr(name: str, gpu: int, err) -> int:
    if err is None:
        return 0
    if err.dtype is not torch.int32 or err.numel() < 1 or err.get_device() != gpu:
        raise KernelError(f"{name}: err must be an int32 tensor on the same device",
                          context={"dtype": str(err.dtype), "device": str(err.device)})
    return err.data_ptr()


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
    query_mean: str = "block",
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
    ``[B, Hk, NBk, D]``, updated in place: the mean of every key block that got new tokens; one from
    NBk on is left out and reported in ``err``) also computes the means of the new queries: with
    ``query_mean="block"`` the sum of a block's new rows over all 64 (the others count as zeros, as the
    padding behind a whole sequence does where :class:`AttnGate` pools it), with ``"new"`` their own
    mean. A gate trained on whole sequences has seen means of full blocks: give it ``"new"`` where
    chunks or single tokens leave blocks in part (a token's sum over 64 hardly moves its scores).
    Returns ``(q, pooled_q)``: rotated q (a new tensor, 0 in rows that no sequence accounts for, or
    ``out``, which may be q itself and where such rows are not written) and fp32 ``[B, Hq,
    chunk_rows(max_new), D]`` or None, for :meth:`AttnGate.forward_pooled`. f32 / bf16 / f16; D and rot multiples of 16 (8 in f32), D up to
    256. The packed, paged counterpart of :func:`qkv_rope_pool`, which takes cos and sin as tables."""
    name = "rope_append_paged"
    gpu, qs, ks = q.get_device(), q.shape, k_pages.shape
    _check_pages(name, gpu, q, qs, k_pages, ks, v_pages)
    T, Hq, D = qs
    num_pages, page_size, Hk, _ = ks
    dtype = q.dtype
    if k.shape != (T, Hk, D) or v.shape != (T, Hk, D) or k.dtype is not dtype or v.dtype is not dtype or \
            k.get_device() != gpu or v.get_device() != gpu:
        raise KernelError(f"{name}: expects k, v [T, Hk, D] in q's dtype and on its device",
                          context={"q": list(qs), "k": list(k.shape), "v": list(v.shape)})
    if block != BLOCK or max_new <= 0 or query_mean not in ("block", "new"):
        raise KernelError(f"{name}: block must be {BLOCK}, max_new positive, query_mean 'block' or 'new'",
                          context={"block": block, "max_new": max_new, "query_mean": query_mean})
    f64 = inv_freq.dtype is torch.float64
    if inv_freq.dim() != 1 or not (f64 or inv_freq.dtype is torch.float32) or inv_freq.get_device() != gpu:
        raise KernelError(f"{name}: inv_freq must be [rot / 2], fp64 or fp32, on the same device",
                          context={"shape": list(inv_freq.shape), "dtype": str(inv_freq.dtype)})
    dev = q.device
    B = kv_len.numel()
    kvl = _index(name, kv_len, gpu, B)
    cu = _index(name, cu_seqlens, gpu, B + 1)
    table = _index(name, block_table, gpu, B, 2)
    err_ptr = _err_ptr(name, gpu, err)
    rows = chunk_rows(max_new)
    nbk = pq_ptr = pk_ptr = 0
    pooled_q = None
    if pooled_k is not None:
        ps = pooled_k.shape
        if len(ps) != 4 or ps[0] != B or ps[1] != Hk or ps[3] != D or pooled_k.dtype is not torch.float32 or \
                not pooled_k.is_contiguous() or pooled_k.get_device() != gpu:
            raise KernelError(f"{name}: pooled_k must be contiguous fp32 [B, Hk, NBk, D] on the same device",
                              context={"pooled_k": list(ps), "dtype": str(pooled_k.dtype)})
        nbk = ps[2]
        pooled_q = torch.empty(B, Hq, rows, D, dtype=torch.float32, device=dev)
        pq_ptr, pk_ptr = pooled_q.data_ptr(), pooled_k.data_ptr()
    options = L.ROPE_MEAN_NEW if query_mean == "new" else 0
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        options |= L.ZERO_REST
    elif out.shape != qs or out.dtype is not dtype or out.get_device() != gpu or out.stride(2) != 1:
        raise KernelError(f"{name}: out must match q", context={"q": list(qs), "out": list(out.shape)})
    per16 = 16 // dtype.itemsize
    (q, qt), (k, kt), (v, vt) = _rows(q, per16), _rows(k, per16), _rows(v, per16)
    freq = inv_freq if inv_freq.is_contiguous() else inv_freq.contiguous()
    args = _rope_args(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
        qt[0], qt[1], kt[0], kt[1], vt[0], vt[1], out.stride(0), out.stride(1), *k_pages.stride(), *v_pages.stride(),
        freq.data_ptr(), table.data_ptr(), cu.data_ptr(), kvl.data_ptr(), pq_ptr, pk_ptr, attention_scaling,
        B, T, Hq, Hk, D, 2 * freq.numel(), block, L.dtype_code(q), max_new, table.size(1), page_size, num_pages, rows,
        nbk, interleaved, f64, err_ptr)
    rc = L.launch(L.lib().tasft_rope_append_paged_opt, gpu, args, options)
    if rc:
        L.check(rc, "tasft_rope_append_paged", shape=[B, T, Hq, Hk, D], page_size=page_size)
    return out, pooled_q


def _rows(x: torch.Tensor, per16: int):
    """x as rows on 16-byte boundaries with contiguous columns (a copy where it is not), and its strides."""
    st = x.stride()
    if st[2] != 1 or st[0] % per16 or st[1] % per16 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        st = x.stride()
    return x, st


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
    gpu, shape = scores.get_device(), scores.shape
    if len(shape) != 4 or scores.dtype is not torch.float32 or num_kv_heads <= 0 or shape[1] % num_kv_heads or gpu < 0:
        raise KernelError(f"{name}: expects fp32 scores [B, Hq, NBq, NBk] on a CUDA device, Hq a multiple of num_kv_heads",
                          context={"scores": list(shape), "dtype": str(scores.dtype), "Hk": num_kv_heads,
                                   "device": str(scores.device)})
    if top_k <= 0 or first < 0 or local < 1 or block <= 0:
        raise ValidationError(f"{name}: top_k and local must be positive, first not negative",
                              context={"top_k": top_k, "first": first, "local": local, "block": block})
    B, Hq, nbq, nbk = shape
    st = scores.stride()
    if st[3] != 1:
        scores = scores.contiguous()
        st = scores.stride()
    kvl = _index(name, kv_len, gpu, B)
    cu = _index(name, cu_seqlens, gpu, B + 1)
    err_ptr = _err_ptr(name, gpu, err)
    width = min(nbk, max(top_k, first + local))
    dev = scores.device
    idx = torch.empty(B, num_kv_heads, nbq, width, dtype=torch.int32, device=dev)
    cnt = torch.empty(B, num_kv_heads, nbq, dtype=torch.int32, device=dev)
    args = _select_args(
        scores.data_ptr(), st[0], st[1], st[2], cu.data_ptr(), kvl.data_ptr(), B, Hq, num_kv_heads, nbq, nbk, block,
        min(top_k, nbk), min(first, nbk), min(local, nbk), tau is not None, 0.0 if tau is None else tau, width,
        idx.data_ptr(), cnt.data_ptr(), err_ptr)
    rc = L.launch(L.lib().tasft_select_blocks, gpu, args)
    if rc:
        L.check(rc, "tasft_select_blocks", shape=[B, Hq, num_kv_heads, nbq, nbk])
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
    ``[T, Hq, D]``: a new tensor, 0 in rows that no sequence accounts for (outside all of them, or of
    one whose lengths do not fit), or ``out``, which may be q itself and where such rows stay as they
    were. A token with nothing kept gets 0. ``err``: optional int32 error word, see
    ``include/tasft_b200.h``. bf16 / f16, D 64 or 128, page size 16, 32, 64 or 128. What the cache holds from ``kv_len`` on, behind a
    token's own position or in blocks its list does not keep never reaches its row, infinities
    and NaN neither. Beside :func:`bsa_decode_paged` (one token per sequence) and
    :meth:`BlockSparseFlashAttention.forward_varlen` (no cache)."""
    name = "bsa_chunk_paged"
    gpu, qs, ks = q.get_device(), q.shape, k_pages.shape
    _check_pages(name, gpu, q, qs, k_pages, ks, v_pages)
    T, Hq, D = qs
    num_pages, page_size, Hk, _ = ks
    B = kv_len.numel()
    kvl = _index(name, kv_len, gpu, B)
    cu = _index(name, cu_seqlens, gpu, B + 1)
    table = _index(name, block_table, gpu, B, 2)
    err_ptr = _err_ptr(name, gpu, err)
    if max_new <= 0:
        raise KernelError(f"{name}: max_new must be positive", context={"max_new": max_new})
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    elif not (scale > 0.0 and math.isfinite(scale)):
        raise KernelError(f"{name}: scale must be positive and finite", context={"scale": scale})
    idx_ptr = cnt_ptr = hm = rows = width = 0
    if kept is not None:
        idx, cnt = kept.idx, kept.cnt
        ls = idx.shape
        if len(ls) != 4 or ls[0] != B or ls[1] not in (Hq, Hk) or cnt.shape != ls[:3] or ls[2] < chunk_rows(max_new) or \
                not ls[3] or idx.get_device() != gpu or cnt.get_device() != gpu:
            raise KernelError(f"{name}: kept lists must be [B, Hk or Hq, at least {chunk_rows(max_new)}, W] on one device",
                              context={"idx": list(ls), "cnt": list(cnt.shape)})
        if idx.dtype is not torch.int32 or not idx.is_contiguous():
            idx = idx.to(torch.int32).contiguous()
        if cnt.dtype is not torch.int32 or not cnt.is_contiguous():
            cnt = cnt.to(torch.int32).contiguous()
        idx_ptr, cnt_ptr = idx.data_ptr(), cnt.data_ptr()
        _, hm, rows, width = ls
    if gpu != torch._C._cuda_getDevice():  # the workspace is sized for the current device
        with torch.cuda.device(gpu):
            return bsa_chunk_paged(q, k_pages, v_pages, table, cu, kvl, max_new, kept, block, scale=scale, out=out, err=err)
    options = 0
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        options = L.ZERO_REST
    elif out.shape != qs or out.dtype is not q.dtype or out.get_device() != gpu or out.stride(2) != 1:
        raise KernelError(f"{name}: out must match q", context={"q": list(qs), "out": list(out.shape)})
    q, st = _rows(q, 8)
    lib = L.lib()
    nbytes = lib.tasft_chunk_workspace_size(B, T, Hq, Hk, D, max_new, hm)
    if nbytes < 0:
        L.check(int(nbytes), "tasft_chunk_workspace_size", shape=[B, T, Hq, Hk, D])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    args = _chunk_args(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), st[0], st[1], out.stride(0), out.stride(1),
        *k_pages.stride(), *v_pages.stride(), table.data_ptr(), cu.data_ptr(), kvl.data_ptr(), idx_ptr, cnt_ptr, B, T, Hq,
        Hk, D, block, L.dtype_code(q), max_new, table.size(1), page_size, num_pages, hm, rows, width, scale, ws.data_ptr(),
        nbytes, err_ptr)
    rc = L.launch(lib.tasft_bsa_chunk_paged_fwd_opt, gpu, args, options)
    if rc:
        L.check(rc, "tasft_bsa_chunk_paged_fwd", shape=[B, T, Hq, Hk, D], page_size=page_size)
    return out


__all__ = ["bsa_chunk_paged", "chunk_rows", "rope_append_paged", "rope_inv_freq", "select_blocks"]
