"""The activations of the gated block where they are small: the lower tails of GELU and SiLU, against the definitions in 64 bits, with bounds relative to what they are."""
import math

import pytest
import torch

from gpu_util import announce
from test_gpu_gated import TINY, TYPES, U, activation, rounded

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    from ml import matmul
    return matmul


def of_activation(g, name):
    """How far act(g) and act'(g) computed in f32 may be off, relative to their parts, so that a tail that comes out as 0 is seen; TINY times 256: what is lost below the smallest normal number.
    SiLU, s = 1 / (1 + e^-g): the argument of the exponential is g times a rounded constant, rounded (2 |g| roundings of its result), the exponential, the sum and the reciprocal are 2 each, g s
    one: (3 |g| + 16) U with some to spare.  Slope s (1 + g (1 - s)): the same of s, of 1 - s an absolute error of s's, and the sum's.
    GELU, g erfc(-g / sqrt 2) / 2: the argument is g times a rounded constant, rounded, which erfc below 0 multiplies by up to g^2; erfc itself is within 16 units in the last place (32 U).
    Slope: that of Phi and, of g phi, an exponential whose argument g^2 / 2 is rounded three times."""
    a = g.abs()
    if name == "relu":
        return torch.zeros_like(g), torch.zeros_like(g)
    if name == "silu":
        s = torch.sigmoid(g)
        e = (3 * a + 16) * U
        return a * s * e + 256 * TINY, s * (1 + a) * (2 * e + 8 * U) + 256 * TINY
    below, density = 0.5 * torch.special.erfc(-g / math.sqrt(2.0)), torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
    e = (32 + 3 * g.square()) * U
    return a * below * (e + 4 * U) + 256 * TINY, below * e + a * density * (2 * g.square() + 12) * U + 4 * U * (below + a * density) + 256 * TINY


def numbers(dtype):
    """Numbers of the type from -85 to 12, most of them between -13 and 3."""
    return torch.cat((torch.linspace(-85, -13, 300), torch.linspace(-13, 3, 3000), torch.linspace(3, 12, 100))).to(TYPES[dtype]).unique()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 130])
def test_results(M, act, dtype, n):
    """One number of a row of A is g, another one 1, and the weights pick them: both products are exact, so the result is the activation's own.  1 column: four waves share K; 130: tiles."""
    announce("matmul_abt_gated tails %s" % ((act, dtype, n),))
    g = numbers(dtype)
    x = torch.zeros((len(g), 8), dtype=g.dtype)
    x[:, 0], x[:, 1] = g, 1
    gate, up = torch.zeros((n, 8), dtype=g.dtype), torch.zeros((n, 8), dtype=g.dtype)
    gate[:, 0], up[:, 1] = 1, 1
    c = M.matmul_abt_gated(x.cuda(), gate.cuda(), up.cuda(), activation=act).cpu()
    want, of = activation(g.double(), act)[0], of_activation(g.double(), act)[0]
    off, bound = (c.double() - want[:, None]).abs(), (of + rounded(want.abs() + of, g.dtype))[:, None]
    worst = (off / bound).amax(1).argmax()
    assert (off <= bound).all(), (g[worst].item(), c[worst, 0].item(), want[worst].item())


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_gradients(M, act, dtype):
    """One column, whose weights are two different unit vectors: dA holds dg and du themselves."""
    announce("matmul_abt_gated_backward tails %s" % ((act, dtype),))
    g = numbers(dtype)
    gate, up = torch.zeros((1, 8), dtype=g.dtype), torch.zeros((1, 8), dtype=g.dtype)
    gate[:, 0], up[:, 1] = 1, 1
    ones = torch.ones((len(g), 1), dtype=g.dtype).cuda()
    x = torch.zeros((len(g), 8), dtype=g.dtype).cuda()
    da = M.matmul_abt_gated_backward(ones, x, gate.cuda(), up.cuda(), (g[:, None].cuda(), ones), activation=act, want_weight_grads=False)[0].cpu()
    for got, want, of, what in zip((da[:, 1], da[:, 0]), activation(g.double(), act), of_activation(g.double(), act), ("du", "dg")):
        # (dg and du are rounded to the type, and so is what their product by 1 is; f16 has 0 below its smallest number either time)
        bound = of + 2 * rounded(want.abs() + of, g.dtype)
        off = (got.double() - want).abs()
        worst = (off / bound).argmax()
        assert (off <= bound).all(), (what, g[worst].item(), got[worst].item(), want[worst].item())
    assert (da[:, 2:] == 0).all()


@pytest.mark.parametrize("m,n,k", [(70, 130, 72), (300, 700, 264)])
def test_a_loss_scaled_beyond_f16_is_seen_in_its_rows_alone(M, m, n, k):
    """dg above 65504 is an infinity: infinite or NaN in its row of dA and of dB_gate, whichever side of the products it is on; the others have the bits that they have without it."""
    announce("matmul_abt_gated_backward f16 range %s" % ((m, n, k),))
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda a, b, s=1.0: (torch.randn((a, b), generator=g, device="cuda") * s).half()
    x, gate, up, dc, kept = r(m, k), r(n, k, 0.1), r(n, k, 0.1), r(m, n), (r(m, n), r(m, n))
    row, col = m - 3, n - 2
    dc[row, col], kept[0][row, col], kept[1][row, col] = 1.0, 1.0, 2.0
    clean = M.matmul_abt_gated_backward(dc, x, gate, up, kept)
    dc[row, col], kept[1][row, col] = 3000.0, 30.0        # dg = 3000 * 30 * silu'(1) = 83500, du = 3000 * silu(1) = 2193
    da, dg, du = M.matmul_abt_gated_backward(dc, x, gate, up, kept)
    others = lambda t, i: torch.cat((t[:i], t[i + 1:]))
    assert not da[row].isfinite().any() and torch.equal(others(da, row), others(clean[0], row))
    assert not dg[col].isfinite().any() and torch.equal(others(dg, col), others(clean[1], col))
    assert du.isfinite().all() and torch.equal(others(du, col), others(clean[2], col))


def test_a_sum_beyond_f16_is_kept_as_an_infinity(M):
    """C is computed of the f32 sums; the gradients at an infinite gate are NaN in its row of dA and its column's row of dB_gate, and nowhere else."""
    announce("matmul_abt_gated f16 range of what is kept")
    m, n, k = 70, 130, 72
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda a, b, s=1.0: (torch.randn((a, b), generator=g, device="cuda") * s).half()
    x, gate, up, dc = r(m, k), r(n, k, 0.1), r(n, k, 0.1), r(m, n)
    x[:, :2], gate[:, :2], up[:, :2] = 0, 0, 0
    row, col = m - 3, n - 2
    _, clean = M.matmul_abt_gated(x, gate, up, keep=torch.float16)
    x[row], gate[col], up[col] = 0, 0, 0
    x[row, 0], gate[col, 0], x[row, 1], up[col, 1] = 300, 300, 0.25, 1.0          # g = 90000, u = 0.25
    c, kept = M.matmul_abt_gated(x, gate, up, keep=torch.float16)
    # (f16 counts in steps of 16 from 2^14 to 2^15: 22500 = 1406.25 * 16 is rounded to 1406 * 16)
    assert c[row, col].item() == 22496 and kept[0][row, col].item() == math.inf and kept[1][row, col].item() == 0.25
    kept = tuple(torch.where((torch.arange(m, device="cuda") == row)[:, None] & (torch.arange(n, device="cuda") == col), a, b) for a, b in zip(kept, clean))
    da, dg, du = M.matmul_abt_gated_backward(dc, x, gate, up, kept)
    others = lambda t, i: torch.cat((t[:i], t[i + 1:]))
    assert da[row].isnan().all() and not others(da, row).isnan().any()
    assert dg[col].isnan().all() and not others(dg, col).isnan().any() and not others(du, col).isnan().any()
