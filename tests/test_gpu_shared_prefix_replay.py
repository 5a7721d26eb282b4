"""A captured shared_prefix_attention call whose tokens move between groups before the replay: group starts, prefix lengths and page tables are read on the device, and only the
most tokens of a group and the size of a slot or table belong to the capture."""

import pytest
import torch

from test_gpu_shared_prefix import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", [("gqa", 2, 4), ("mqa", 1, 16), ("mha", 1, 3)])
@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("tokens,prefix,later", [
    ([9, 3, 0, 5], [700, 300, 500, 0], [([0, 9, 5, 3], [1, 129, 700, 3]), ([1, 1, 9, 6], [0, 0, 257, 700]), ([0, 0, 8, 9], [700, 700, 0, 0])]),
    ([100, 30], [400, 900], [([30, 100], [900, 128]), ([65, 65], [0, 900])]),
    ([3] + [2] * 38 + [1], [200] * 40, [([1, 3] + [2] * 38, [7 * i for i in range(28)] + [0] * 12), ([3, 3, 0] + [2] * 37, [200, 0, 128] + [129] * 37)]),
])
def test_tokens_in_other_groups(tokens, prefix, later, page, layout):
    c = Case(tokens, prefix, [1] * sum(tokens), [1 + 3 * i % 40 for i in range(sum(tokens))], layout=layout, page=page, own_page=page, seed=len(tokens))
    c.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = c.call(return_lse=True)
    for groups, lens in later:
        c.tokens, c.prefix.lens = groups, lens
        c.prefix_bias.q_seqinfo.seqstart.copy_(torch.tensor([0] + groups).cumsum(0).int())
        c.prefix_bias.k_seqinfo.seqlen.copy_(torch.tensor(lens, dtype=torch.int32))
        for g, n in enumerate(lens):
            t = torch.arange(n, device="cuda")
            c.prefix.where[g] = c.prefix.table[g].long()[t // page] * page + t % page if page else g * c.prefix.pad + t
            for x in (c.prefix.k, c.prefix.v):
                x[0, c.prefix.where[g]] = torch.randn(n, *x.shape[2:], device="cuda").to(x.dtype)
        graph.replay()
        torch.cuda.synchronize()
        c.check(got)
