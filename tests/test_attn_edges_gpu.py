"""GPU: calls of the softmax-attention operators at the edges of what they allow."""
import numpy as np
import pytest
import torch

from attn_util import D, on, prefill_inputs
from conftest import load_pkg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [np.float32(1e-6), np.float64(1e-6), torch.tensor(1e-6), 0, 1],
                         ids=["float32", "float64", "tensor", "0", "1"])
def test_eps_of_any_number_type_on_every_call(cuda, eps):
    """A call whose plan is kept takes what the first one took, with the same result."""
    pkg = load_pkg()
    g = on(prefill_inputs([9], 4, 2, seed=1), cuda)
    w = torch.ones(D, device=cuda)
    pos, table = torch.arange(9, device=cuda), pkg.rope_table(9, 64, device=cuda)
    kw = [dict(eps=eps)] * 3 + [dict(eps=float(eps))]
    q, k = zip(*(pkg.attn_qk_norm_rope(g["q"], g["k"], pos, table, w, w, **x) for x in kw))
    for x in (q, k):
        assert all(torch.equal(x[0], y) for y in x[1:])
