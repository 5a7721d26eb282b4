"""Host-side refusals of shared_prefix_attention, checked without a GPU."""

import ctypes as C

import pytest
import torch

from xformers_b200 import _lib
from xformers_b200.ops import fmha, shared_prefix_attention

ab = fmha.attn_bias


def _args(**kw):
    a = dict(
        query=torch.zeros(1, 4, 2, 3, 64, dtype=torch.bfloat16),
        prefix_key=torch.zeros(1, 32, 2, 1, 64, dtype=torch.bfloat16).expand(-1, -1, -1, 3, -1),
        key=torch.zeros(1, 40, 2, 1, 64, dtype=torch.bfloat16).expand(-1, -1, -1, 3, -1),
        prefix_bias=ab.BlockDiagonalPaddedKeysMask.from_seqlens(q_seqlen=[1, 3], kv_padding=16, kv_seqlen=[3, 16]),
        attn_bias=ab.BlockDiagonalCausalWithOffsetPaddedKeysMask.from_seqlens(q_seqlen=[1] * 4, kv_padding=10, kv_seqlen=[1, 2, 3, 4]),
    )
    a.update(kw)
    a.setdefault("prefix_value", a["prefix_key"])
    a.setdefault("value", a["key"])
    return a


_PAGED = ab.PagedBlockDiagonalPaddedKeysMask
_TABLE = torch.zeros(2, 2, dtype=torch.int32)


@pytest.mark.parametrize("kw,error,match", [
    (dict(query=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), ValueError, "must all be"),
    (dict(prefix_bias=ab.BlockDiagonalCausalWithOffsetPaddedKeysMask.from_seqlens(q_seqlen=[4], kv_padding=16, kv_seqlen=[3])), ValueError, "prefix_bias must be"),
    (dict(attn_bias=ab.BlockDiagonalCausalLocalAttentionPaddedKeysMask.from_seqlens_local([1] * 4, 10, [1] * 4, 3)), ValueError, "without windows"),
    (dict(attn_bias=None), ValueError, "attn_bias type"),
    (dict(attn_bias=torch.zeros(1, 2, 3, 4, 40)), ValueError, "attn_bias type"),
    (dict(prefix_bias=ab.BlockDiagonalPaddedKeysMask.from_seqlens(q_seqlen=[1, 2], kv_padding=16, kv_seqlen=[3, 16])), ValueError, "prefix_bias describes 3 queries"),
    (dict(attn_bias=ab.BlockDiagonalPaddedKeysMask.from_seqlens(q_seqlen=[1] * 5, kv_padding=8, kv_seqlen=[1] * 5)), ValueError, "attn_bias describes 5 queries"),
    (dict(prefix_value=torch.zeros(1, 31, 2, 3, 64, dtype=torch.bfloat16)), ValueError, "prefix_key .* and prefix_value"),
    (dict(prefix_key=torch.zeros(1, 32, 3, 2, 64, dtype=torch.bfloat16)), ValueError, "the heads of query"),
    (dict(key=torch.zeros(1, 40, 2, 2, 64, dtype=torch.bfloat16)), ValueError, "the heads of query"),
    (dict(prefix_key=torch.zeros(1, 32, 2, 3, 64, dtype=torch.float16)), ValueError, "dtype of query"),
    (dict(prefix_bias=ab.BlockDiagonalPaddedKeysMask.from_seqlens(q_seqlen=[1, 3], kv_padding=17, kv_seqlen=[3, 16])), ValueError, "2 slots of 17 keys"),
    (dict(prefix_bias=_PAGED.from_seqlens([1, 3], [3, 16], _TABLE, 24)), ValueError, "whole number of pages"),
    (dict(prefix_bias=_PAGED.from_seqlens([1, 3], [3, 4], _TABLE, 4)), NotImplementedError, "multiple of 8 tokens"),
    (dict(prefix_bias=_PAGED.from_seqlens([1, 3], [3, 16], _TABLE.long(), 8)), ValueError, "block_tables must be an int32"),
    (dict(scale=0.0), NotImplementedError, "scale must be positive"),
    (dict(scale=float("nan")), NotImplementedError, "scale must be positive"),
    (dict(output_dtype=torch.float64), ValueError, "output_dtype"),
    (dict(prefix_key=torch.zeros(1, 32, 2, 1, 68, dtype=torch.bfloat16)[..., :64].expand(-1, -1, -1, 3, -1)), NotImplementedError, "16-byte boundaries"),
    (dict(prefix_key=torch.zeros(1, 32, 2, 1, 128, dtype=torch.bfloat16)[..., ::2].expand(-1, -1, -1, 3, -1)), NotImplementedError, "16-byte boundaries"),
    (dict(query=torch.zeros(1 + 4 * 2 * 3 * 64, dtype=torch.bfloat16)[1:].view(1, 4, 2, 3, 64)), NotImplementedError, "16-byte boundaries"),
    (dict(), ValueError, "needs CUDA tensors"),
])
def test_refusals(kw, error, match):
    with pytest.raises(error, match=match):
        shared_prefix_attention(**_args(**kw))


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.bfloat16, 96), (torch.bfloat16, 256)])
def test_types_and_head_dims(dtype, d):
    x = torch.zeros(1, 4, 1, d, dtype=dtype)
    bias = ab.BlockDiagonalPaddedKeysMask.from_seqlens(q_seqlen=[4], kv_padding=4, kv_seqlen=[4])
    with pytest.raises(NotImplementedError, match="head dim 64 or 128"):
        shared_prefix_attention(x, x, x, bias, x, x, bias)


def test_gradients_are_refused():
    a = _args()
    a["query"].requires_grad_()
    with pytest.raises(NotImplementedError, match="backward pass"):
        shared_prefix_attention(**a)


def test_c_entry_refuses_before_it_launches():
    lib = _lib.load()
    call = lambda p: lib.xfb200_shared_prefix_forward(None if p is None else C.byref(p), None)
    assert call(None) == _lib.XFB200_E_INVALID
    p = _lib.SharedPrefixParams()
    assert call(p) == _lib.XFB200_E_INVALID
    p.groups = p.kv_heads = p.q_per_kv = 1
    assert call(p) == _lib.XFB200_OK  # no query
    p.total_q = p.max_q = 4
    p.head_dim, p.scale, p.kv_padding, p.kv_rows, p.dtype = 128, 1.0, 16, 16, _lib.BF16
    assert call(p) == _lib.XFB200_E_INVALID  # null tensors
    for n in ("q", "k", "v", "out", "seqstart_q", "seqlen_k", "own_out", "own_lse", "scratch"):
        setattr(p, n, 256)
    own = _lib.DecodeParams()
    for field, value, code in (
        ("head_dim", 96, _lib.XFB200_E_UNSUPPORTED), ("dtype", _lib.F32, _lib.XFB200_E_INVALID), ("out_dtype", 9, _lib.XFB200_E_INVALID),
        ("scale", 0.0, _lib.XFB200_E_UNSUPPORTED), ("own", C.pointer(own), _lib.XFB200_E_INVALID), ("own_out", None, _lib.XFB200_E_INVALID),
        ("own_lse", None, _lib.XFB200_E_INVALID), ("scratch", 128, _lib.XFB200_E_INVALID), ("scratch", None, _lib.XFB200_E_INVALID), 
        ("kv_rows", 0, _lib.XFB200_E_INVALID), ("kv_rows", 1 << 31, _lib.XFB200_E_INVALID), ("q_stride_m", 4, _lib.XFB200_E_INVALID), ("k", 264, _lib.XFB200_E_INVALID),
        ("total_q", 1 << 30, _lib.XFB200_E_UNSUPPORTED), ("own_stride_m", 2, _lib.XFB200_E_INVALID), ("own_beside", 2, _lib.XFB200_E_INVALID), ("own_out", 264, _lib.XFB200_E_INVALID),
    ):
        old = None if field == "own" else getattr(p, field)
        setattr(p, field, value)
        assert call(p) == code, field
        assert b"shared_prefix" in lib.xfb200_last_error()
        setattr(p, field, old)
    p.own_out = None
    for field, value in (("batch", -2), ("mq", 0), ("split_k", 0), ("split_k", 1025), ("kv_padding", 0), ("window_size", 3), ("q_per_kv", 2)):
        own.batch, own.mq, own.kv_heads, own.q_per_kv, own.head_dim, own.split_k, own.kv_padding, own.window_size = 2, 2, 1, 1, 128, 1, 1, 0
        setattr(own, field, value)
        if field == "batch":
            own.mq = -2
        p.own = C.pointer(own)
        assert call(p) == _lib.XFB200_E_INVALID, field
        assert b"own keys" in lib.xfb200_last_error()
    p.own, p.own_out = None, 256
    p.block_tables = 256
    for page, code in ((0, _lib.XFB200_E_INVALID), (12, _lib.XFB200_E_UNSUPPORTED)):
        p.page_size = page
        assert call(p) == code
    d = _lib.DecodeParams()
    d.batch = d.mq = d.kv_heads = d.q_per_kv = d.split_k = d.kv_padding = 1
    d.q = d.k = d.v = d.out = 256
    d.head_dim = 128
    d.flags = 8
    assert lib.xfb200_decode_forward(C.byref(d), None) == _lib.XFB200_E_INVALID
    d.flags = 1
    assert lib.xfb200_decode_forward(C.byref(d), None) == _lib.XFB200_E_INVALID  # no scratch
    assert lib.xfb200_decode_forward_static_scratch(C.byref(d), None) == _lib.XFB200_E_INVALID


def test_scratch():
    """Room for the own partials, and a slot for every block of rows and every CTA."""
    lib = _lib.load()
    p = _lib.SharedPrefixParams()
    assert lib.xfb200_shared_prefix_scratch_bytes(None) == 0 == lib.xfb200_shared_prefix_scratch_bytes(C.byref(p))
    p.groups, p.kv_heads, p.q_per_kv, p.total_q, p.max_q, p.head_dim, p.kv_padding = 1, 2, 4, 5, 5, 64, 300
    up = lambda n: -(-n // 256) * 256
    slots, rows = 2 + 2 * 3, 20
    assert lib.xfb200_shared_prefix_scratch_bytes(C.byref(p)) == up(32) + up(slots * rows * 64 * 4) + up(slots * rows * 4)
    own = _lib.DecodeParams()
    own.batch, own.mq, own.kv_heads, own.q_per_kv, own.head_dim, own.split_k = 5, 1, 2, 4, 64, 3
    p.own = C.pointer(own)
    part = 5 * 3 * 2 * 4
    assert lib.xfb200_shared_prefix_scratch_bytes(C.byref(p)) == up(32) + up(slots * rows * 64 * 4) + up(slots * rows * 4) + up(part * 64 * 4) + up(part * 4)


@pytest.mark.parametrize("words", [0, 17, 32])
@pytest.mark.parametrize("batch,pad,layout", [(4, 4096, (8, 4)), (8, 8192, (8, 8)), (1, 700, (1, 16)), (128, 2056, (8, 8)), (40, 300, (4, 7))])
def test_both_paths_cut_the_own_keys_alike(words, batch, pad, layout):
    """The chunks that the Python path asks for are those of the C rule, whose arguments the host front passes in C order."""
    from xformers_b200.ops.fmha import b200_splitk, common, shared_prefix

    G, H = layout
    q = torch.zeros(1, batch, G, H, 128, dtype=torch.bfloat16)
    key = torch.zeros(1, 1, G, 1, words or 128, dtype=torch.int32 if words else q.dtype).expand(-1, batch * pad, -1, H, -1)
    bias = ab.BlockDiagonalCausalWithOffsetPaddedKeysMask.from_seqlens(q_seqlen=[1] * batch, kv_padding=pad, kv_seqlen=[pad] * batch)
    extra = {f"{n}_fp8_scale_shift": torch.zeros(1, 1, G, H, dtype=torch.int32).expand(-1, batch * pad, -1, -1) for n in "kv"} if words == 32 else {}
    inp = (common.InputsFp8 if extra else common.Inputs)(q, key, key, bias, 0.0, None, torch.float32, True, **extra)
    q5, k5, v5, broadcast = b200_splitk._geometry(inp)
    p = b200_splitk.FwOp.params(inp, k5, v5, q5, broadcast, shared_prefix._split_k)
    rows, row_bytes = H, (words or 64) * 4
    assert p.split_k == _lib.load().xfb200_shared_prefix_split_k(batch, pad, G, rows, row_bytes, int(words > 0))
    assert b200_splitk.FwOp.params(inp, k5, v5, q5, broadcast).split_k == _lib.load().xfb200_decode_split_k(batch, pad, G, rows, row_bytes, int(words > 0))


def test_the_rule_gets_its_arguments_in_c_order(monkeypatch):
    from xformers_b200.ops.fmha import shared_prefix

    seen, lib = {}, _lib.load()

    def rule(batch, kv_bound, kv_heads, rows, row_bytes, quantised):
        seen.update(rows=rows, row_bytes=row_bytes, kv_heads=kv_heads)
        return 1

    monkeypatch.setattr(lib, "xfb200_shared_prefix_split_k", rule)
    assert shared_prefix._split_k(3, 100, 2, 256, 12, False) == 1
    assert seen == dict(rows=12, row_bytes=256, kv_heads=2)


_WORDS = torch.zeros(1, 40, 2, 3, dtype=torch.int32)


@pytest.mark.parametrize("k_words,v_words,as_words", [(_WORDS, None, True), (None, _WORDS, True), (_WORDS, _WORDS, False), (_WORDS, None, False)])
def test_scale_words_without_what_they_scale_are_refused(k_words, v_words, as_words):
    """Not left out of account: words for one of both, or beside 16-bit keys."""
    a = _args()
    if as_words:
        a["key"] = a["value"] = torch.zeros(1, 40, 2, 1, 16, dtype=torch.int32).expand(-1, -1, -1, 3, -1)
    with pytest.raises(ValueError, match="k_fp8_scale_shift and v_fp8_scale_shift go together"):
        shared_prefix_attention(**a, k_fp8_scale_shift=k_words, v_fp8_scale_shift=v_words)


def test_prefill_refuses_another_launch_order():
    lib = _lib.load()
    p = _lib.PrefillParams()
    p.batch = p.mq = p.mkv = p.total_q = p.groups = p.heads_per_group = 1
    p.head_dim, p.dtype, p.out_dtype, p.window_left = 64, _lib.BF16, _lib.BF16, -1
    p.q = p.k = p.v = p.out = 256
    for value in (-1, 2):
        p.in_order = value
        assert lib.xfb200_prefill_forward(C.byref(p), None) == _lib.XFB200_E_INVALID
        assert b"in_order" in lib.xfb200_last_error()
