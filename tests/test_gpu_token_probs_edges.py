"""Log probabilities of tokens and their gradient where the rows, what comes back to them or their number is out of the ordinary."""
import math

import pytest
import torch

from gpu_util import announce
from test_gpu_token_probs import INF, logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def P():
    from ml import primitives
    return primitives


@pytest.mark.parametrize("cols", [3, 300, 9001])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_with_nothing_in_them_have_no_gradient_whatever_comes_back(P, cols, dtype):
    """A loss that takes lse or the log probability itself, its square say, hands an infinity or a NaN back to a row whose lse is -inf: zeros there, and the other rows as without it."""
    announce("token_log_probs_backward of nothing %s" % ((cols, dtype),))
    x, t = logits(6, cols, dtype, seed=30)
    x[1::2] = -INF
    x, t = x.cuda(), t.cuda()
    _, entropy, lse = P.token_log_probs(x, t, want_entropy=True, want_lse=True)
    d = torch.randn(6, generator=torch.Generator().manual_seed(31)).cuda()
    for bad in (-INF, INF, math.nan):
        spoiled = d.clone()
        spoiled[1::2] = bad
        for which in ("logp", "entropy", "lse", "logp entropy lse"):
            grad = lambda v: P.token_log_probs_backward(v if "logp" in which else None, x, t, lse, d_entropy=v if "entropy" in which else None,
                                                        entropy=entropy if "entropy" in which else None, d_lse=v if "lse" in which else None)
            got, want = grad(spoiled), grad(d)
            assert (got[1::2] == 0).all(), (bad, which)
            assert torch.equal(got[::2], want[::2]), (bad, which)
