"""Every kernel of the log probabilities and of their gradient against the definitions in 64 bits: what a row's width, the number of rows, alternatives, the entropy and the size of the result
choose, in every type.  tests/test_gpu_kernels_reached.py counts them."""
import pytest
import torch

from gpu_util import announce
from test_gpu_token_probs import INF, TYPES, U, bounds, exact, exact_backward, same_where_special

pytestmark = pytest.mark.gpu

PIECE = {"f32": 4, "f16": 8, "bf16": 8}             # numbers in 16 bytes

# (rows, pieces of 16 bytes): lanes of a wave that hold a row in one to sixteen pieces each, workgroups of 256 and of 512, and both for chunks of a row
FORWARD = [(37, 3), (37, 11), (37, 27), (37, 55), (37, 101), (37, 203), (37, 401), (4099, 1000), (300, 1501), (100, 3001), (300, 5003), (100, 17501), (128, 32768)]
# with alternatives: workgroups of 256 and of 512, for rows and for chunks
ALTERNATIVES = [(300, 55), (300, 1501), (100, 1501), (300, 5003), (100, 17501)]
# of the gradient: 4, 16 or 64 lanes of a wave, workgroups of 256
GRADIENT = [3, 11, 27, 55, 101, 203, 700]


@pytest.fixture(scope="module")
def P():
    from ml import primitives
    return primitives


def columns(pieces, dtype):
    """A row that ends inside its last piece; in 16-bit types rows so begin anywhere."""
    return pieces * PIECE[dtype] - (3 if pieces % 2 else 1)


def rows_of(rows, cols, dtype, streamed):
    """`rows`, or as many as give a result that does not stay in the caches (32 MiB)."""
    return (32 << 20) // (cols * TYPES[dtype].itemsize) + 3 if streamed else rows


def inputs(rows, cols, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn((rows, cols), generator=g, device="cuda") * 3).to(TYPES[dtype])
    t = torch.randint(0, cols, (rows,), generator=g, device="cuda").int()
    t[rows // 2] = -1
    if rows > 5:
        x[1] = -INF
        x[3, : cols // 2] = -INF
    return x, t


def check(got, want, bound, what):
    fine = same_where_special(got, want)
    off = (got.double() - want).abs()
    assert (off <= bound)[fine].all(), (what, (off / bound)[fine].max().item())


@pytest.mark.parametrize("rows,pieces", FORWARD)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_forward(P, rows, pieces, dtype):
    cols = columns(pieces, dtype)
    announce("token_log_probs kernels %s" % ((rows, cols, dtype),))
    x, t = inputs(rows, cols, dtype, 40)
    logp, entropy, lse = P.token_log_probs(x, t, want_entropy=True, want_lse=True)
    alone, lse_alone = P.token_log_probs(x, t, want_lse=True)
    want_logp, want_entropy, want_lse, p = exact(x, t)
    of_lse, of_entropy = bounds(x, want_lse, p)
    for got in (logp, alone):
        check(got, want_logp, of_lse + 2 * U * want_logp.abs().nan_to_num(0, 0, 0), "logp")
    for got in (lse, lse_alone):
        check(got, want_lse, of_lse, "lse")
    check(entropy, want_entropy, of_entropy + 2 * U * want_entropy.abs().nan_to_num(0), "entropy")


@pytest.mark.parametrize("rows,pieces", ALTERNATIVES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top", [1, 5, 32])
def test_alternatives(P, rows, pieces, dtype, top):
    cols = columns(pieces, dtype)
    announce("token_log_probs kernels top %s" % ((rows, cols, dtype, top),))
    x, t = inputs(rows, cols, dtype, 41)
    logp, entropy, values, ids = P.token_log_probs(x, t, top=top, want_entropy=True)
    without = P.token_log_probs(x, t, top=top)
    assert torch.equal(without[0], logp) and torch.equal(without[1], values) and torch.equal(without[2], ids)
    want_logp, want_entropy, want_lse, p = exact(x, t)
    of_lse, of_entropy = bounds(x, want_lse, p)
    check(logp, want_logp, of_lse + 2 * U * want_logp.abs().nan_to_num(0, 0, 0), "logp")
    check(entropy, want_entropy, of_entropy + 2 * U * want_entropy.abs().nan_to_num(0), "entropy")
    order, at = torch.sort(x.float(), dim=1, descending=True, stable=True)
    want_ids = torch.where(order[:, :top] > -INF, at[:, :top].int(), -1)
    assert torch.equal(ids, want_ids)
    want = torch.where(want_ids >= 0, torch.stack([exact(x, want_ids[:, j])[0] for j in range(top)], 1), -INF)
    check(values, want, of_lse[:, None] + 2 * U * want.abs().nan_to_num(0, 0, 0), "alternatives")


@pytest.mark.parametrize("pieces", GRADIENT)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("streamed", [False, True])
def test_gradient(P, pieces, dtype, streamed):
    cols = columns(pieces, dtype)
    rows = rows_of(37, cols, dtype, streamed)
    announce("token_log_probs_backward kernels %s" % ((rows, cols, dtype),))
    x, t = inputs(rows, cols, dtype, 42)
    _, entropy, lse, _ = exact(x, t)
    lse, entropy = lse.float(), entropy.float()
    g = torch.Generator(device="cuda").manual_seed(43)
    d_logp, d_entropy, d_lse = (torch.randn(rows, generator=g, device="cuda") for _ in range(3))
    info = torch.finfo(x.dtype)
    for of_entropy in (False, True):
        more = (d_entropy, entropy) if of_entropy else (None, None)
        want, bound = exact_backward(x, t, lse, d_logp, more[0], more[1], d_lse)
        got = P.token_log_probs_backward(d_logp, x, t, lse, d_entropy=more[0], entropy=more[1], d_lse=d_lse)
        assert got.dtype == x.dtype and got.shape == x.shape
        check(got, want, bound + info.eps / 2 * (want.abs() + bound) + info.tiny * info.eps, "gradient")
