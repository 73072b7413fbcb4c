"""Log probabilities of tokens and their gradient where the rows, what comes back to them or their number is out of the ordinary."""
import math

import pytest
import torch

from gpu_util import announce
from test_gpu_token_probs import INF, U, bounds, exact, exact_backward, logits

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


# more rows than 2^32 work items would hold if every one took a wave, or a workgroup of 512
@pytest.mark.parametrize("rows,cols,top", [((1 << 26) + 5, 8, 0), ((1 << 23) + 3, 40, 2)])
def test_very_many_short_rows(P, rows, cols, top):
    announce("token_log_probs many rows %s" % ((rows, cols, top),))
    x, t = logits(1021, cols, "bf16", seed=32)
    x, t = x.cuda(), t.cuda()
    many = -(-rows // 1021)
    out = P.token_log_probs(x.repeat(many, 1)[:rows], t.repeat(many)[:rows], top=top, want_entropy=True, want_lse=True)
    few = P.token_log_probs(x.repeat(20, 1), t.repeat(20), top=top, want_entropy=True, want_lse=True)
    for a, b in zip(out, few):
        assert a.shape[0] == rows and torch.equal(a[:1021], b[:1021]) and torch.equal(a[-(rows % 1021):], b[:rows % 1021])
        last = rows // 1021 * 1021
        assert torch.equal(a[last - 1021 * 7:last], b[:1021 * 7])
    if top == 0:
        grad = P.token_log_probs_backward(out[0], x.repeat(many, 1)[:rows], t.repeat(many)[:rows], out[2])
        want = P.token_log_probs_backward(few[0], x.repeat(20, 1), t.repeat(20), few[2])
        assert torch.equal(grad[last - 1021:last], want[:1021]) and torch.equal(grad[last:], want[:rows - last])


@pytest.mark.parametrize("offset", [0.0, 1e3, -1e3, 1e4, -1e4])
@pytest.mark.parametrize("cols", [40, 1003, 9001])
def test_gradient_of_logits_that_have_an_offset_in_common(P, offset, cols):
    """Against the gradient of the logits themselves in 64 bits, forward and backward together: the rounding of lse is an error of ln p, |lse| 2^-24, and so is what the logarithm and the sum
    behind it are off; what the gradient adds to that is the bound of its own test."""
    announce("token_log_probs_backward offset %s" % ((offset, cols),))
    x, t = logits(5, cols, "f32", seed=33)
    x = x + offset
    d = [torch.randn(5, generator=torch.Generator().manual_seed(34 + k)) for k in range(3)]
    _, entropy, lse = P.token_log_probs(x.cuda(), t.cuda(), want_entropy=True, want_lse=True)
    got = P.token_log_probs_backward(d[0].cuda(), x.cuda(), t.cuda(), lse, d_entropy=d[1].cuda(), entropy=entropy, d_lse=d[2].cuda()).cpu().double()
    _, want_entropy, want_lse, p = exact(x, t)
    want, of_grad = exact_backward(x, t, want_lse, d[0], d[1], want_entropy, d[2])
    y = x.double() - want_lse[:, None]
    # of ln s: its sum (as in `bounds`, without the rounding of lse) and 4 roundings of the logarithm, which is ln(cols) at most; then lse's own
    far = (p * (y - y.amax(1, keepdim=True)).abs()).sum(1) * 1.4427
    of_lse = (want_lse.abs() + 2 * far + 8 + cols / 64 + 64 + 4 * math.log(cols) + 4) * U
    _, of_entropy = bounds(x, want_lse, p)
    size = d[0].abs()[:, None] + d[2].abs()[:, None] + d[1].abs()[:, None] * (y.abs() + want_entropy[:, None] + 1)
    bound = of_grad + p * size * of_lse[:, None] * 1.01 + p * (d[1].abs() * of_entropy)[:, None]
    off = (got - want).abs()
    assert (off <= bound + U * (want.abs() + bound)).all(), ((off / bound).max().item(), off.max().item())
