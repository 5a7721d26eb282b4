"""Lengths that are written right ahead of a decode call with several chunks a sequence: its merge, which looks at them early, goes by the new ones."""

import pytest
import torch

from xformers_b200.ops import fmha
from xformers_b200.ops.fmha import attn_bias as ab

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("batch,pad,group", [(4, 4096, 4), (40, 1500, 8)])
def test_lengths_change_between_calls(batch, pad, group, captured):
    gen = torch.Generator().manual_seed(batch)
    q = torch.randn(1, batch, 2, group, 128, generator=gen).bfloat16().cuda()
    k, v = (torch.randn(1, batch * pad, 2, 1, 128, generator=gen).bfloat16().cuda().expand(-1, -1, -1, group, -1) for _ in range(2))
    bias = ab.BlockDiagonalPaddedKeysMask.from_seqlens(q_seqlen=[1] * batch, kv_padding=pad, kv_seqlen=[pad] * batch, device="cuda")
    op = type("Op", (fmha.b200_splitk.FwOp,), {"SPLIT_K": 7})
    lens = [torch.randint(0, pad + 1, (batch,), generator=gen).int().cuda() for _ in range(5)]
    lens[3].fill_(0), lens[4].fill_(pad)
    out = lambda: fmha.memory_efficient_attention_forward_requires_grad(q, k, v, bias, op=op)

    def call(n):
        bias.k_seqinfo.seqlen.copy_(n)
        return out()

    want = []
    for n in lens:
        bias.k_seqinfo.seqlen.copy_(n)
        torch.cuda.synchronize()
        want.append(out())
        torch.cuda.synchronize()
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [call(n) for n in lens]
        for _ in range(5):
            graph.replay()
    else:
        got = [call(lens[i % 5]) for i in range(50)]
    torch.cuda.synchronize()
    for i, (o, l) in enumerate(got):
        assert torch.equal(o, want[i % 5][0]) and torch.equal(l, want[i % 5][1]), i
    assert bool((want[3][0] == 0).all()) and bool((want[3][1] == float("-inf")).all())
