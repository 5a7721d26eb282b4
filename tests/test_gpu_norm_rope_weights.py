"""norm_rope_padded with a weight of one kind only: a missing one counts as ones, to which the offset is added like to any other."""

import pytest
import torch

from test_gpu_norm_rope import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("missing", ["qw", "kw"])
@pytest.mark.parametrize("offset", [0.0, 1.0])
@pytest.mark.parametrize("q_len", [[2, 1, 3], [400, 1, 90]])
def test_one_weight_missing(missing, offset, q_len):
    c = Case(q_len, [n + 5 for n in q_len], 410, seed=21)
    setattr(c, missing, None)
    out, ck, _ = c.run(offset=offset)
    # the same as ones given
    setattr(c, missing, torch.ones(128, dtype=c.dtype))
    same, ck2, _ = c.run(offset=offset)
    assert torch.equal(out, same) and torch.equal(ck, ck2)
