"""``fmha.shared_prefix_attention``: attention of a batch whose sequences share their first keys.

Sequences behind one system prompt, samples drawn from one prompt, beams: with the keys of the prefix in every sequence's own cache
(or page table) decode attention reads them once per sequence.  Here a group's prefix is read once for all of its rows, on the tensor
cores, and joined with the attention over the sequences' own keys (``csrc/shared_prefix.cu``, ``xfb200_shared_prefix_forward``).
The prefix and the own keys are described by two bias objects of this package over the same queries.  No counterpart in the reference; the
same result is what :func:`memory_efficient_attention_partial` over both parts and :func:`merge_attentions` give.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple, Union

import torch

from ... import _lib
from . import attn_bias as ab
from . import b200_splitk, front
from .b200_splitk import _DTYPE_CODE, _geometry
from .common import Inputs, InputsFp8

# testing aids of the kernel's bounded waits (see xfb200_shared_prefix_params); both 0 in production
_WAIT_BUDGET_KCYCLES = 0
_DEBUG_FLAGS = 0

_PREFIX_BIASES = (ab.BlockDiagonalPaddedKeysMask, ab.PagedBlockDiagonalPaddedKeysMask)
_DECODE_BIASES = (
    ab.BlockDiagonalPaddedKeysMask,
    ab.BlockDiagonalCausalWithOffsetPaddedKeysMask,
    ab.PagedBlockDiagonalPaddedKeysMask,
    ab.PagedBlockDiagonalCausalWithOffsetPaddedKeysMask,
    ab.BlockDiagonalGappyKeysMask,
    ab.BlockDiagonalCausalWithOffsetGappyKeysMask,
    ab.PagedBlockDiagonalGappyKeysMask,
    ab.PagedBlockDiagonalCausalWithOffsetGappyKeysMask,
)
_OWN_BIASES = _DECODE_BIASES + (ab.BlockDiagonalMask, ab.BlockDiagonalCausalMask, ab.BlockDiagonalCausalFromBottomRightMask)


def _check(query, prefix_key, prefix_value, prefix_bias, key, value, attn_bias, scale, out_dtype, k_words, v_words) -> None:
    name = "shared_prefix_attention"
    if query.ndim not in (4, 5) or any(t.ndim != query.ndim for t in (prefix_key, prefix_value, key, value)):
        raise ValueError(f"{name}: query, keys and values must all be [1, M, H, K] or all be [1, M, G, H, K]")
    if type(prefix_bias) not in _PREFIX_BIASES:
        raise ValueError(f"{name}: prefix_bias must be a BlockDiagonalPaddedKeysMask or a PagedBlockDiagonalPaddedKeysMask, got {type(prefix_bias)}")
    if type(attn_bias) not in _OWN_BIASES:
        raise ValueError(f"{name}: attn_bias type {type(attn_bias)} (block-diagonal masks over the own keys, without windows)")
    if query.shape[0] != 1 or prefix_key.shape[0] != 1 or key.shape[0] != 1:
        raise ValueError(f"{name}: expected batch size 1, sequences are concatenated")
    total = query.shape[1]
    for what, bias in (("prefix_bias", prefix_bias), ("attn_bias", attn_bias)):
        if bias.q_seqinfo.seqstart_py[-1] != total:
            raise ValueError(f"{name}: {what} describes {bias.q_seqinfo.seqstart_py[-1]} queries, query has {total}")
        if bias.q_seqinfo.seqstart.device != query.device or bias.k_seqinfo.seqstart.device != query.device:
            raise ValueError(f"{name}: {what} must be on the device of query")
    if prefix_value.shape != prefix_key.shape or prefix_key.shape[2:] != query.shape[2:]:
        raise ValueError(f"{name}: prefix_key {tuple(prefix_key.shape)} and prefix_value {tuple(prefix_value.shape)} must be [1, rows, ...] with the heads of query {tuple(query.shape)}")
    if key.shape[:-1] != value.shape[:-1] or key.shape[2:-1] != query.shape[2:-1]:
        raise ValueError(f"{name}: key {tuple(key.shape)} and value {tuple(value.shape)} must have the heads of query {tuple(query.shape)}")
    if prefix_key.dtype != query.dtype or prefix_value.dtype != query.dtype:
        raise ValueError(f"{name}: the prefix must have the dtype of query, got {prefix_key.dtype}, {prefix_value.dtype}")
    if (k_words is None) != (v_words is None) or (k_words is not None and not key.dtype == value.dtype == torch.int32):
        raise ValueError(f"{name}: k_fp8_scale_shift and v_fp8_scale_shift go together, with int32 words as key and value, got {key.dtype}, {value.dtype}")
    if any(t.device != query.device for t in (prefix_key, prefix_value, key, value)):
        raise ValueError(f"{name}: all tensors must be on one device")
    rows, slots = prefix_key.shape[1], len(prefix_bias.q_seqinfo.seqstart_py) - 1
    if isinstance(prefix_bias, ab.PagedBlockDiagonalPaddedKeysMask):
        t, page = prefix_bias.block_tables, prefix_bias.page_size
        if t.dtype != torch.int32 or t.ndim != 2 or t.shape[0] != slots or t.stride(1) != 1 or t.device != query.device:
            raise ValueError(f"{name}: prefix_bias.block_tables must be an int32 [groups, pages] tensor with unit inner stride on the device of query")
        if rows % page:
            raise ValueError(f"{name}: the {rows} rows of the prefix must be a whole number of pages of {page}")
        if page % 8:
            raise NotImplementedError(f"{name}: pages of the prefix must be a multiple of 8 tokens, got {page}")
    elif prefix_bias.k_seqinfo.padding * slots > rows:
        raise ValueError(f"{name}: prefix_bias describes {slots} slots of {prefix_bias.k_seqinfo.padding} keys, prefix_key has {rows} rows")
    if query.dtype not in (torch.bfloat16, torch.float16) or query.shape[-1] not in (64, 128):
        raise NotImplementedError(f"{name}: bf16 or f16 and head dim 64 or 128, got {query.dtype}, {query.shape[-1]}")
    if out_dtype not in _DTYPE_CODE:
        raise ValueError(f"{name}: output_dtype {out_dtype}")
    if scale is not None and not scale > 0:
        raise NotImplementedError(f"{name}: scale must be positive, got {scale}")
    for what, t in (("query", query), ("prefix_key", prefix_key), ("prefix_value", prefix_value)):
        if t.stride(-1) != 1 or any(s % 8 for n, s in zip(t.shape[1:-1], t.stride()[1:-1]) if n > 1) or (t.numel() and t.data_ptr() % 16):
            raise NotImplementedError(f"{name}: rows of {what} must be contiguous and start on 16-byte boundaries")


def _split_k(batch: int, kv_bound: int, kv_heads: int, row_bytes: int, rows: int, quantised: bool) -> int:
    """``xfb200_shared_prefix_split_k`` with its arguments in the order of ``FwOp.get_split_k``."""
    return _lib.load().xfb200_shared_prefix_split_k(batch, kv_bound, kv_heads, rows, row_bytes, quantised)


def _debug_check(prefix_bias, rows: int) -> None:
    lens, bound = prefix_bias.k_seqinfo.seqlen.cpu().tolist(), prefix_bias.k_seqinfo.padding
    if isinstance(prefix_bias, ab.PagedBlockDiagonalPaddedKeysMask):
        table, page = prefix_bias.block_tables.cpu(), prefix_bias.page_size
        bound = table.shape[1] * page
        for g, n in enumerate(lens):
            used = table[g, : -(-max(n, 0) // page)]
            if used.numel() and (int(used.min()) < 0 or int(used.max()) >= rows // page):
                raise ValueError(f"prefix_bias.block_tables[{g}] names a page outside the pool of {rows // page} pages")
    if any(n < 0 or n > bound for n in lens):
        raise ValueError(f"kv_seqlen {lens} of the prefix does not fit {bound} keys")


def shared_prefix_attention(
    query: torch.Tensor,
    prefix_key: torch.Tensor,
    prefix_value: torch.Tensor,
    prefix_bias: Union[ab.BlockDiagonalPaddedKeysMask, ab.PagedBlockDiagonalPaddedKeysMask],
    key: torch.Tensor,
    value: torch.Tensor,
    attn_bias,
    scale: Optional[float] = None,
    *,
    return_lse: bool = False,
    output_dtype: Optional[torch.dtype] = None,
    k_fp8_scale_shift: Optional[torch.Tensor] = None,
    v_fp8_scale_shift: Optional[torch.Tensor] = None,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``softmax(q [K_prefix, K_own]^T * scale) [V_prefix, V_own]``, own keys masked as ``attn_bias`` says.

    ``query [1, M, (G,) H, K]`` holds the tokens of all sequences.  ``prefix_bias`` (``BlockDiagonalPaddedKeysMask`` or
    ``PagedBlockDiagonalPaddedKeysMask``) puts them into groups: its ``q_seqlen`` are the tokens of each group (one entry: the whole
    batch), its ``kv_seqlen`` the prefix lengths, its slots or page tables where ``prefix_key`` / ``prefix_value [1, rows, (G,) H, K]`` hold them (pages a multiple of 8
    tokens; the pool may be the one of the own keys).  Every token sees the whole prefix of its group; an empty prefix is fine.
    ``attn_bias`` describes ``key`` / ``value``, the sequences' own keys, as for :func:`memory_efficient_attention_forward`:
    padded, paged or gappy caches, causal or not; up to 64 query rows per kv head and sequence run on the decode kernel, with int4 row-wise
    caches (int32 words) and fp8 row-wise ones (with ``k_fp8_scale_shift`` / ``v_fp8_scale_shift``, see :class:`InputsFp8`)
    too; otherwise, and for ``BlockDiagonalMask`` and its causal forms, the prefill kernels run, which read 16-bit keys that are not paged.  Masks with windows are refused: a window would have to count the prefix.

    One KV head for several query heads is given expanded (head stride 0), for the prefix and the own keys alike.  bf16 or f16, K of 64 or 128,
    ``scale > 0``.  Lengths, starts and page tables are read on the device, so a captured call may be replayed after they changed, as long as no group has more
    tokens than the largest one had at the capture.  A token with neither prefix nor own keys gets zeros and ``-inf``.

    It pays from some 16000 keys on that are not read again (prefix keys times sequences but one); below that, decode attention over page tables that
    repeat the prefix's pages is sooner done (32 query heads on 8 kv heads of 128, 2 sequences behind 4096 keys: 10.4 us, here 15.5).  Where a prefill kernel runs, the
    call holds two fp32 rows of K elements for every query row while it runs, one of the own keys and one or more of the prefix.

    Returns the output, with ``return_lse`` ``(out, lse [1, (G,) H, M])``.  No gradients.
    """
    if not _WAIT_BUDGET_KCYCLES and not _DEBUG_FLAGS:
        # the host front takes the call unless something about it is unusual, an input that requires grad among the rest (csrc/front.cpp)
        done = front.shared_prefix(query, prefix_key, prefix_value, prefix_bias, key, value, attn_bias, scale, output_dtype, return_lse, k_fp8_scale_shift, v_fp8_scale_shift)
        if done is not None:
            return done if return_lse else done[0]
    if torch.is_grad_enabled() and (query.requires_grad or prefix_key.requires_grad or prefix_value.requires_grad or key.requires_grad or value.requires_grad):
        raise NotImplementedError("shared_prefix_attention: an input requires grad, and the backward pass is outside this library; call it under torch.no_grad()")
    out_dtype = output_dtype or query.dtype
    _check(query, prefix_key, prefix_value, prefix_bias, key, value, attn_bias, scale, out_dtype, k_fp8_scale_shift, v_fp8_scale_shift)
    if query.device.type != "cuda":
        raise ValueError(f"shared_prefix_attention needs CUDA tensors, got device={query.device}")
    fp8 = k_fp8_scale_shift is not None or v_fp8_scale_shift is not None
    extra = dict(k_fp8_scale_shift=k_fp8_scale_shift, v_fp8_scale_shift=v_fp8_scale_shift) if fp8 else {}
    # (the own keys as a call of their own would see them: its checks, its errors)
    inp = (InputsFp8 if fp8 else Inputs)(query, key, value, attn_bias, 0.0, scale, torch.float32, True, **extra)
    inp.validate_inputs()
    q, pk, pv, broadcast = _geometry(Inputs(query, prefix_key, prefix_value))
    _, ok, ov, own_broadcast = _geometry(inp)
    if broadcast != own_broadcast:
        raise ValueError("shared_prefix_attention: the kv heads of the prefix and of the own keys must be given alike (both expanded, or neither)")
    _, M, G, H, D = q.shape
    if not broadcast and G > 1 and H > 1 and any(t.stride(2) != H * t.stride(3) for t in (q, pk, pv)):
        raise NotImplementedError("shared_prefix_attention: head axes (G, H) of non-broadcast keys must flatten to one stride")
    out = torch.empty((1, M, G, H, D), dtype=out_dtype, device=query.device)
    lse = torch.empty((G, H, M), dtype=torch.float32, device=query.device) if return_lse else None

    if M > 0:
        with torch.cuda.device(query.device):
            lib = _lib.load()
            p = _lib.SharedPrefixParams()
            p.q, p.k, p.v, p.out = q.data_ptr(), pk.data_ptr(), pv.data_ptr(), out.data_ptr()
            p.lse = lse.data_ptr() if lse is not None else None
            qi, ki = prefix_bias.q_seqinfo, prefix_bias.k_seqinfo
            p.seqstart_q, p.seqlen_k = qi.seqstart.data_ptr(), ki.seqlen.data_ptr()
            p.dtype, p.out_dtype = _DTYPE_CODE[query.dtype], _DTYPE_CODE[out_dtype]
            p.groups, p.max_q, p.total_q, p.head_dim = len(qi.seqstart_py) - 1, qi.max_seqlen, M, D
            p.kv_padding = ki.padding
            if isinstance(prefix_bias, ab.PagedBlockDiagonalPaddedKeysMask):
                t = prefix_bias.block_tables
                p.block_tables, p.block_table_stride, p.page_size = t.data_ptr(), t.stride(0), prefix_bias.page_size
                p.kv_padding = t.shape[1] * prefix_bias.page_size
            p.kv_rows = pk.shape[1]
            if p.kv_rows == 0:
                p.kv_padding = 0
            p.q_stride_m, p.k_stride_m, p.v_stride_m, p.o_stride_m = q.stride(1), pk.stride(1), pv.stride(1), out.stride(1)
            if broadcast:
                p.kv_heads, p.q_per_kv = G, H
                p.q_stride_g, p.q_stride_h = q.stride(2), q.stride(3)
                p.k_stride_g, p.v_stride_g = pk.stride(2), pv.stride(2)
                p.o_stride_g, p.o_stride_h, p.lse_stride_g, p.lse_stride_h = H * D, D, H * M, M
            else:
                p.kv_heads, p.q_per_kv = G * H, 1
                hs = lambda t: t.stride(3) if H > 1 else t.stride(2)
                p.q_stride_g, p.k_stride_g, p.v_stride_g = hs(q), hs(pk), hs(pv)
                p.o_stride_g, p.lse_stride_g = D, M
            for f, n in (("q_stride_m", M), ("q_stride_g", p.kv_heads), ("q_stride_h", p.q_per_kv), ("k_stride_g", p.kv_heads), ("v_stride_g", p.kv_heads),
                         ("k_stride_m", p.kv_rows), ("v_stride_m", p.kv_rows)):
                if n <= 1:
                    setattr(p, f, 0 if f.endswith(("g", "h")) else D)  # the stride of an extent-1 axis is meaningless
            p.scale = inp.scale_float
            p.wait_budget_kcycles, p.debug_flags = _WAIT_BUDGET_KCYCLES, _DEBUG_FLAGS
            if _lib.debug_checks():
                _debug_check(prefix_bias, p.kv_rows)
            own = None
            if type(attn_bias) in _DECODE_BIASES and not b200_splitk.FwOp.not_supported_reasons(inp):
                own = b200_splitk.FwOp.params(inp, ok, ov, q, own_broadcast, _split_k if b200_splitk.FwOp.SPLIT_K is None else None)
                p.own = C.pointer(own)
            else:
                from . import _run_forward

                own_out, own_lse = _run_forward(inp, None, needs_lse=True)
                own_out, own_lse = (own_out, own_lse) if query.ndim == 5 else (own_out.unsqueeze(2), own_lse.unsqueeze(1))
                if own_lse.stride(-1) != 1 and M > 1:
                    own_lse = own_lse.contiguous()
                p.own_out, p.own_lse = own_out.data_ptr(), own_lse.data_ptr()
                p.own_stride_m = own_out.stride(1)
                if broadcast:
                    p.own_stride_g, p.own_stride_h, p.own_lse_stride_g, p.own_lse_stride_h = own_out.stride(2), own_out.stride(3), own_lse.stride(1), own_lse.stride(2)
                else:
                    p.own_stride_g, p.own_lse_stride_g = D, own_lse.stride(2) if H > 1 else own_lse.stride(1)
            nbytes = lib.xfb200_shared_prefix_scratch_bytes(C.byref(p))
            scratch = torch.empty((max(nbytes, 256),), dtype=torch.uint8, device=query.device)
            p.scratch = scratch.data_ptr()
            rc = lib.xfb200_shared_prefix_forward(C.byref(p), C.c_void_p(torch.cuda.current_stream(query.device).cuda_stream))
            _lib.check(rc, "shared_prefix_attention")
            if _lib.check_status_after_every_call():
                from . import b200

                b200.check_device_status(query.device)
                b200_splitk.check_device_status(query.device)

    if query.ndim == 4:
        out = out[:, :, 0]
    if lse is None:
        return out
    return out, (lse[None] if query.ndim == 5 else lse)
