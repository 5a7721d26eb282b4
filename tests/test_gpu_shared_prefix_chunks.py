"""shared_prefix_attention where a sequence's own keys are cut into several chunks: the Python path and the host front give the same bits, and both what the definition says."""

import pytest
import torch

import oracle
from test_gpu_shared_prefix import Case
from xformers_b200 import _lib
from xformers_b200.ops import shared_prefix_attention

pytestmark = pytest.mark.gpu


def _quantise(c, fmt):
    """Own keys of the case in a quantised format: words, what they stand for, scale / shift words by name."""
    raw = [torch.randn(x.shape, generator=torch.Generator().manual_seed(i)) for i, x in enumerate((c.own.k, c.own.v))]
    if fmt == "int4":
        words = [oracle.quantize_kv_int4(x.to(c.dt)).cuda() for x in raw]
        return words, [oracle.dequantize_kv_int4(w.cpu()).cuda() for w in words], {}
    words, held, extra = [], [], {}
    for n, x in zip("kv", raw):
        q8, scale, shift = oracle.quantize_fp8_asymmetric(x.reshape(-1, c.d))
        ss = oracle.combine_scale_shift(scale, shift)
        held.append(oracle.dequantize_fp8_asymmetric(q8, *oracle.split_scale_shift(ss)).view(x.shape).cuda())
        words.append(oracle.pack_fp8_words(q8).view(*x.shape[:-1], c.d // 4).cuda())
        extra[f"{n}_fp8_scale_shift"] = ss.view(x.shape[:-1]).cuda().expand(-1, -1, -1, c.H)
    return words, held, extra


@pytest.mark.parametrize("fmt", ["16 bits", "int4", "fp8"])
@pytest.mark.parametrize("own_page", [0, 16])
@pytest.mark.parametrize("new,own_pad,layout", [(1, 4096, ("gqa", 8, 4)), (1, 3008, ("gqa", 1, 16)), (3, 2000, ("gqa", 2, 7))])
def test_front_and_python_path_agree_over_chunks(fmt, own_page, new, own_pad, layout, monkeypatch):
    lens = [own_pad - 16, 700, new, 1333]
    c = Case([new * 4], [300], [new] * 4, lens, layout=layout, own_page=own_page, own_pad=own_pad, seed=own_pad)
    bytes_ = {"16 bits": 256, "int4": 68, "fp8": 128}[fmt]
    assert _lib.load().xfb200_shared_prefix_split_k(4, own_pad, c.G, new * c.H, bytes_, int(fmt != "16 bits")) > 1
    if fmt == "16 bits":
        words, held, extra = (c.own.k, c.own.v), (c.own.k, c.own.v), {}
    else:
        words, held, extra = _quantise(c, fmt)

    def call():
        wide = (w.expand(*c.own.expand(w)) for w in words)
        return shared_prefix_attention(c.q, *c.prefix.views(), c.prefix_bias, *wide, c.bias, return_lse=True, **extra)

    a = call()
    monkeypatch.setattr(_lib, "front", None)
    b = call()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # (a quantised cache: V times its scale is rounded to f16 as well, a half step more)
    c.check(a, c.reference(own=held), slack=1.0 if fmt == "16 bits" else 2.0)


@pytest.mark.parametrize("q_len", [[1, 1, 1], [40, 3, 70]])
@pytest.mark.parametrize("both", [True, False])
def test_scale_words_beside_16_bit_keys_are_refused(q_len, both):
    c = Case([sum(q_len)], [300], q_len, [90, 30, 70], seed=3)
    words = torch.zeros(1, c.own.k.shape[1], 2, 4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="go together"):
        c.call(k_fp8_scale_shift=words, v_fp8_scale_shift=words if both else None)
