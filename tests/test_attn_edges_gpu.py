"""GPU: calls of the softmax-attention operators at the edges of what they allow."""
import pytest
import torch

from attn_util import check, on, prefill_inputs
from conftest import load_pkg
from oracle import attn_oracle as A

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[300], [5, 1, 3], [2500]])
def test_rows_whose_scores_are_all_minus_infinity(cuda, lens):
    """They give zeros, as rows that see nothing do, in every kernel, whole and joined.  The
    other rows agree with the oracle as ever (not bit for bit with a call without such rows: the
    32 rows of a warp choose together how their exponentials are taken)."""
    pkg = load_pkg()
    d = prefill_inputs(lens, 4, 2, seed=2)
    d["k"][..., 0] = 1.0
    ref, size = A.prefill(d["q"], d["k"], d["v"], d["cu"])
    g = on(d, cuda)
    rows = [i for i in (0, 5, 8, 200, 299, 2400) if i < sum(lens)]
    g["q"][rows, 1] = 0.0
    g["q"][rows, 1, 0] = float("-inf")  # -inf * 1 + 0 * the rest
    out = pkg.attn_prefill(g["q"], g["k"], g["v"], g["cu"])
    assert (out[rows, 1] == 0).all()
    ref[rows, 1], size[rows, 1] = 0, 0
    check(out, ref, size)
