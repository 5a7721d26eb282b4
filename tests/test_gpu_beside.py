"""shared_prefix_attention reads its prefix beside the kernel that reads the own keys.  Whatever wrote their inputs right ahead of the call -- a copy, or a kernel of this
library that lets the next one begin early -- has to be seen by both, in eager calls and in captured ones."""

import pytest
import torch

from test_gpu_shared_prefix import Case
from xformers_b200.ops import norm_rope_padded

pytestmark = pytest.mark.gpu

CASES = {
    # own keys on the decode kernel, its CTAs in several waves
    "decode": dict(tokens=[130], prefix=[900], q_len=[1] * 130, kv_len=[1 + 7 * i % 600 for i in range(130)], layout=("gqa", 4, 4), own_pad=640),
    "decode, many groups": dict(tokens=[3] * 12, prefix=[300 + 50 * i for i in range(12)], q_len=[1] * 36, kv_len=[1 + 11 * i for i in range(36)], layout=("gqa", 2, 8), own_pad=640),
    "prefill": dict(tokens=[211], prefix=[1500], q_len=[150, 11, 50], kv_len=[150, 70, 333], layout=("gqa", 4, 3), own_pad=400),
}


def _buffers(c):
    return [c.q, c.prefix.k, c.prefix.v, c.own.k, c.own.v, c.prefix_bias.k_seqinfo.seqlen, c.bias.k_seqinfo.seqlen]


def _versions(c, n):
    """Other contents of the same shapes: values shifted along the tokens' features, shorter lengths."""
    out = []
    for i in range(n):
        x = [t.roll(i, -1) for t in _buffers(c)[:5]]
        out.append(x + [(t - 5 * i).clamp_min(1) if t is c.prefix_bias.k_seqinfo.seqlen else t.clone() for t in _buffers(c)[5:]])
    return out


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("captured", [False, True])
def test_inputs_written_right_ahead(name, captured):
    c = Case(**CASES[name], seed=1)
    versions, want = _versions(c, 3), []
    for v in versions:
        for t, x in zip(_buffers(c), v):
            t.copy_(x)
        torch.cuda.synchronize()
        want.append(c.call(return_lse=True))
        torch.cuda.synchronize()
    assert not torch.equal(want[0][0], want[1][0])

    def steps(n):
        got = []
        for i in range(n):
            for t, x in zip(_buffers(c), versions[i % 3]):
                t.copy_(x)
            got.append(c.call(return_lse=True))
        return got

    if not captured:
        got = steps(30)
        torch.cuda.synchronize()
    else:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = steps(6)
        for _ in range(5):
            for t in _buffers(c)[:5]:
                t.zero_()
            graph.replay()
        torch.cuda.synchronize()
    for i, pair in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(pair, want[i % 3])), i


@pytest.mark.parametrize("captured", [False, True])
def test_behind_a_kernel_that_lets_the_next_one_begin(captured):
    """The append writes queries and own keys; the attention behind it is launched while it runs."""
    c = Case([130], [900], [1] * 130, [1 + 7 * i % 600 for i in range(130)], layout=("gqa", 4, 4), own_page=16, seed=2)
    x = [[torch.randn(1, 130, 4, h, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(10 * i + h + j)).bfloat16() for j, h in enumerate((4, 1, 1))] for i in range(3)]

    def step(i):
        q = norm_rope_padded(*x[i % 3], c.own.k, c.own.v, c.bias, out_q=c.q)
        assert q.data_ptr() == c.q.data_ptr()
        return c.call(return_lse=True)

    want = []
    for i in range(3):
        norm_rope_padded(*x[i], c.own.k, c.own.v, c.bias, out_q=c.q)
        torch.cuda.synchronize()
        want.append(c.call(return_lse=True))
        torch.cuda.synchronize()
    assert not torch.equal(want[0][0], want[1][0])
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [step(i) for i in range(9)]
        for _ in range(5):
            c.q.zero_()
            graph.replay()
    else:
        got = [step(i) for i in range(60)]
    torch.cuda.synchronize()
    for i, pair in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(pair, want[i % 3])), i
