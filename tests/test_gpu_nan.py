"""NaN among the keys that a query sees reaches its output and its log-sum-exp, and nothing else: the softmax of a row with NaN among its scores is NaN.

Each case puts NaN where a kernel could lose it -- the only key of a sequence, a key that is alone in a sub-tile of 16, in a chunk, the newest one of many -- and
compares everything that does not see it with the same call without, bit for bit."""

import pytest
import torch

import oracle
from test_gpu_shared_prefix import Case
from xformers_b200.ops import fmha
from xformers_b200.ops.fmha import attn_bias as ab

pytestmark = pytest.mark.gpu
S = fmha.b200_splitk
NAN_WORD = 0x7E007E00  # scale and shift of a quantised row: fp16 NaN
# keys of the sequences, and which of them is NaN (None: none of them)
LENS, BAD = [1, 17, 129, 700, 700, 40, 0], [0, 16, 128, 699, 3, None, None]



def _check(out, lse, clean, clean_lse, bad):
    """out [tokens, ..], lse [.., tokens], `bad` [tokens]: rows that see NaN."""
    assert bool(out[bad].isnan().all()) and bool(lse[..., bad].isnan().all())
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[..., ~bad], clean_lse[..., ~bad])


class Decode:
    def __init__(self, fmt, group, mq=1, d=128, kv_heads=2, pad=704):
        gen = torch.Generator().manual_seed(group)
        dt = torch.float16 if fmt == "f16" else torch.bfloat16
        self.fmt, self.group, self.pad, n = fmt, group, pad, len(LENS)
        self.q = torch.randn(1, n * mq, kv_heads, group, d, generator=gen).to(dt).cuda()
        x = [torch.randn(1, n * pad, kv_heads, 1, d, generator=gen).to(dt) for _ in range(2)]
        self.groups = 4 if fmt == "int4 groups" else 1
        if fmt.startswith("int4"):
            x = [oracle.quantize_kv_int4(t, self.groups) for t in x]
        self.words = None
        if fmt == "fp8":
            held = [oracle.quantize_fp8_asymmetric(t.float().reshape(-1, d)) for t in x]
            self.words = [oracle.combine_scale_shift(s, h).view(1, n * pad, kv_heads, 1).cuda() for _, s, h in held]
            x = [oracle.pack_fp8_words(q8).view(1, n * pad, kv_heads, 1, d // 4) for q8, _, _ in held]
        self.k, self.v = (t.contiguous().cuda() for t in x)
        mask = ab.BlockDiagonalPaddedKeysMask if mq == 1 else ab.BlockDiagonalCausalWithOffsetPaddedKeysMask
        self.bias = mask.from_seqlens(q_seqlen=[mq] * n, kv_padding=pad, kv_seqlen=LENS, device="cuda")

    def spoil(self):
        for i, t in enumerate(BAD):
            if t is None:
                continue
            if self.fmt == "fp8":
                self.words[0][0, i * self.pad + t] = NAN_WORD
            elif self.groups > 1 or self.fmt == "int4":
                self.k[0, i * self.pad + t, ..., : self.groups] = NAN_WORD
            else:
                self.k[0, i * self.pad + t] = float("nan")

    def call(self, split_k):
        op = type("Op", (S.FwOp,), {"SPLIT_K": split_k, "NUM_GROUPS": self.groups})
        wide = lambda t: t.expand(-1, -1, -1, self.group, *t.shape[4:])
        if self.words is None:
            out, lse = fmha.memory_efficient_attention_forward_requires_grad(self.q, wide(self.k), wide(self.v), self.bias, op=op)
        else:
            inp = S.InputsFp8(query=self.q, key=wide(self.k), value=wide(self.v), attn_bias=self.bias, k_fp8_scale_shift=wide(self.words[0]), v_fp8_scale_shift=wide(self.words[1]))
            out, ctx = fmha._memory_efficient_attention_forward_requires_grad(inp, op=op)
            lse = ctx.lse
        return out[0], lse[0]


@pytest.mark.parametrize("fmt", ["bf16", "f16", "int4", "int4 groups", "fp8"])
@pytest.mark.parametrize("split_k", [None, 1, 5])
@pytest.mark.parametrize("group", [1, 8, 40])
def test_decode(fmt, split_k, group):
    c = Decode(fmt, group)
    clean = c.call(split_k)
    assert not clean[0].isnan().any() and bool((clean[1][..., 6] == float("-inf")).all())
    c.spoil()
    _check(*c.call(split_k), *clean, torch.tensor([t is not None for t in BAD], device="cuda"))


@pytest.mark.parametrize("fmt", ["bf16", "int4", "fp8"])
@pytest.mark.parametrize("split_k", [1, 5])
def test_decode_newest_key_is_hidden_from_the_first_query(fmt, split_k):
    """Two queries a sequence: the last key is NaN for the second one only."""
    c = Decode(fmt, 4, mq=2)
    clean = c.call(split_k)
    c.spoil()
    bad = [False] * 14
    for i, (n, t) in enumerate(zip(LENS, BAD)):
        for j in range(2):
            bad[2 * i + j] = t is not None and t < n - 1 + j
    _check(*c.call(split_k), *clean, torch.tensor(bad, device="cuda"))


@pytest.mark.parametrize("fmt", ["bf16", "int4", "fp8"])
@pytest.mark.parametrize("split_k", [1, 5])
def test_decode_nan_in_a_query(fmt, split_k):
    c = Decode(fmt, 8)
    clean, clean_lse = c.call(split_k)
    c.q[0, 4, 1, 3, 7] = float("nan")
    out, lse = c.call(split_k)
    assert bool(out[4, 1, 3].isnan().all()) and bool(lse[1, 3, 4].isnan())
    out[4, 1, 3], lse[1, 3, 4] = clean[4, 1, 3], clean_lse[1, 3, 4]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("prefix", [0, 1, 300])
@pytest.mark.parametrize("lens,bad,pad", [(LENS, BAD, 704), (LENS, BAD, 4000), ([1, 17, 64, 33, 40, 0], [0, 16, 63, None, 5, None], 64)])
@pytest.mark.parametrize("page", [0, 16])
def test_own_keys_behind_a_shared_prefix(prefix, lens, bad, pad, page):
    """The decode kernel's partials, one or several to a sequence, joined with those of a prefix or without one."""
    n = len(lens)
    c = Case([n], [prefix], [1] * n, lens, own_pad=pad, own_page=page, page=page, seed=prefix + pad)
    clean, clean_lse = c.call(return_lse=True)
    c.check((clean, clean_lse))
    for i, t in enumerate(bad):
        if t is not None:
            c.own.k[0, c.own.where[i][t]] = float("nan")
    out, lse = c.call(return_lse=True)
    _check(out[0], lse[0], clean[0], clean_lse[0], torch.tensor([t is not None for t in bad], device="cuda"))


@pytest.mark.parametrize("prefix", [0, 1, 300])
@pytest.mark.parametrize("q_len,kv_len", [([7, 1, 40, 12, 9], [7, 300, 60, 12, 30]), ([150, 1, 200, 70, 9], [150, 5, 260, 200, 9])])
@pytest.mark.parametrize("through_front", [True, False])
def test_prefill_of_own_keys_behind_a_shared_prefix(prefix, q_len, kv_len, through_front, monkeypatch):
    """Unequal token counts: the partials are a prefill kernel's.  NaN in the only key that a token sees, among others, in the newest key, in a hidden value."""
    from xformers_b200 import _lib

    if not through_front:
        monkeypatch.setattr(_lib, "front", None)
    c = Case([sum(q_len)], [prefix], q_len, kv_len, seed=prefix + len(q_len))
    clean, clean_lse = c.call(return_lse=True)
    c.check((clean, clean_lse))
    at = [0, kv_len[1] - 1, kv_len[2] // 2, kv_len[3] - 1, None]
    bad = []
    for i, (n, m, t) in enumerate(zip(q_len, kv_len, at)):
        bad += [t is not None and m - n + j >= t for j in range(n)]
        if t is not None:
            c.own.k[0, c.own.where[i][t]] = float("nan")
    out, lse = c.call(return_lse=True)
    _check(out[0], lse[0], clean[0], clean_lse[0], torch.tensor(bad, device="cuda"))


@pytest.mark.parametrize("prefix", [0, 300])
def test_tokens_without_own_keys_on_the_prefill_path(prefix):
    """A sequence without own keys, and tokens ahead of the first own key of theirs, whose tile holds NaN that only later tokens see."""
    c = Case([60], [prefix], [9, 11, 40], [9, 0, 25], seed=31)
    clean, clean_lse = c.call(return_lse=True)
    c.check((clean, clean_lse))
    if prefix == 0:
        assert bool((clean[0, 9:35] == 0).all()) and bool((clean_lse[..., 9:35] == float("-inf")).all())
    c.own.k[0, c.own.where[2][24]] = c.own.v[0, c.own.where[2][24]] = float("nan")  # of the last token alone
    out, lse = c.call(return_lse=True)
    assert torch.equal(out[:, :35], clean[:, :35]) and torch.equal(lse[..., :59], clean_lse[..., :59])
    assert bool(out[:, 59].isnan().all()) and bool(lse[..., 59].isnan().all())


@pytest.mark.parametrize("op", ["FwOp_Tcgen05_Persistent", "FwOp_Tcgen05_M256", "FwOp_Generic"])
@pytest.mark.parametrize("d", [64, 128])
def test_prefill(op, d):
    """The log-sum-exp of a row that sees NaN is NaN, in each of the prefill kernels."""
    gen = torch.Generator().manual_seed(d)
    q_len, kv_len = [300, 5, 130], [300, 70, 133]
    q = torch.randn(1, sum(q_len), 4, d, generator=gen).bfloat16().cuda()
    k, v = (torch.randn(1, sum(kv_len), 4, d, generator=gen).bfloat16().cuda() for _ in range(2))
    bias = ab.BlockDiagonalCausalFromBottomRightMask.from_seqlens(q_len, kv_len, device="cuda")
    run = lambda: [x[0] for x in fmha.memory_efficient_attention_forward_requires_grad(q, k, v, bias, op=getattr(fmha.b200, op))]
    clean = run()
    k[0, 0], k[0, 300 + 69], k[0, 370 + 100] = (float("nan"),) * 3
    bad = [True] * 300 + [False] * 4 + [True] + [3 + j >= 100 for j in range(130)]
    _check(*run(), *clean, torch.tensor(bad, device="cuda"))
