"""Layer norm and its gradients on the GPU against float64, with bounds counted from the roundings.

u = 2^-24 is half a step of f32.  A sum of n terms added along chains of d additions is off by at most d u times the sum of their
magnitudes; a row's longest chain is 64 elements of a lane, 6 steps over a wave and 15 over the waves."""
import numpy as np
import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CHAIN = 64 + 6 + 15 + 1                  # and the product by 1 / cols; 1 / cols itself is off by u
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# one lane, one wave, several; a piece of 16 bytes more or less; every width of group and the widest row
SHAPES = [(1, 1), (1, 2), (3, 7), (5, 8), (257, 9), (1000, 24), (70, 33), (4, 64), (131, 65), (515, 128), (35, 200), (7, 255), (300, 512), (2, 513), (9, 1003), (33, 1024), (513, 1025), (16, 2047),
          (1, 4096), (5, 4097), (600, 2500), (4, 6000), (6, 8192), (3, 8200), (2, 12001), (2, 16383), (3, 16384)]


@pytest.fixture(scope="module")
def P():
    from ml import primitives
    return primitives


def half_step(t):
    return torch.finfo(t).eps / 2


def make(rows, cols, t, wt, seed, offset=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, cols), generator=g, dtype=torch.float64) * torch.exp(torch.randn((cols,), generator=g, dtype=torch.float64))
         + offset * torch.randn((rows, 1), generator=g, dtype=torch.float64)).to(t)
    w = (1 + 0.2 * torch.randn((cols,), generator=g, dtype=torch.float64)).to(wt)
    b = (0.2 * torch.randn((cols,), generator=g, dtype=torch.float64)).to(wt)
    dy = torch.randn((rows, cols), generator=g, dtype=torch.float64).to(t)
    return x, w, b, dy


def forward64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = (x - mean) * rstd
    y = h * (1 if w is None else w.double()) + (0 if b is None else b.double())
    return y, mean, rstd, h


def check_forward(P, x, w, b, eps):
    t = x.dtype
    y, mean, rstd = P.layer_norm(x.cuda(), None if w is None else w.cuda(), None if b is None else b.cuda(), eps=eps, want_stats=True)
    torch.cuda.synchronize()
    want, m, r, h = forward64(x, w, b, eps)
    big = x.double().abs().mean(-1, keepdim=True)
    d_mean = (CHAIN + 1) * U * big + U * m.abs()
    assert ((mean.cpu().double() - m[:, 0]).abs() <= d_mean[:, 0] + 1e-45).all()
    # the variance: every (x - mean)^2 is off by 2 (d_mean + u |x - mean|) |x - mean| + u of itself; the mean's error adds its square;
    # a chain of additions, the product by 1 / cols, + eps; half of that for the root, u each for it and for 1 /
    var = 1 / r ** 2 - eps
    dev = (x.double() - m).abs().mean(-1, keepdim=True)
    d_var = 2 * d_mean * dev + d_mean ** 2 + (CHAIN + 6) * U * var + U * (var + eps)
    rel_rstd = d_var / (2 * (var + eps)) * (1 + d_var / (var + eps)) + 2 * U
    assert ((rstd.cpu().double() - r[:, 0]).abs() <= (rel_rstd * r)[:, 0] * 1.001).all()
    aw = 1 if w is None else w.double().abs()
    d_h = r * (d_mean + U * (x.double() - m).abs()) * (1 + rel_rstd) + h.abs() * (rel_rstd + U)
    f32 = aw * d_h + U * (aw * h.abs()) + U * want.abs()
    bound = f32 + half_step(t) * (want.abs() + f32) + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    off = (y.cpu().double() - want).abs()
    assert (off <= bound * 1.001).all(), float((off / bound).max())
    return mean, rstd


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("types", ["f32 f32", "bf16 f32", "bf16 bf16", "f16 f32", "f16 f16"])
def test_forward(P, shape, types):
    t, wt = (TYPES[n] for n in types.split())
    announce("layer_norm %s %s" % (shape, types))
    x, w, b, _ = make(*shape, t, wt, 1)
    check_forward(P, x, w, b, 1e-5)


def test_forward_without_weights_and_with_one_of_them(P):
    announce("layer_norm without weights")
    x, w, b, _ = make(37, 200, torch.bfloat16, torch.float32, 2)
    check_forward(P, x, None, None, 1e-6)
    check_forward(P, x, w, None, 1e-6)
    check_forward(P, x, None, b, 1e-6)


def test_rows_far_from_zero_and_constant_rows(P):
    announce("layer_norm far from zero")
    x, w, b, _ = make(16, 1024, torch.float32, torch.float32, 3, offset=1000.0)
    check_forward(P, x, w, b, 1e-5)
    x = torch.full((5, 96), 3.25)                     # every mean is exact: the squares are zeros
    y, mean, rstd = P.layer_norm(x.cuda(), eps=0.25, want_stats=True)
    assert (y.cpu() == 0).all() and (mean.cpu() == 3.25).all() and (rstd.cpu() == 2.0).all()


def test_bad_numbers_stay_in_their_row(P):
    announce("layer_norm NaN and inf")
    x, w, b, _ = make(12, 700, torch.bfloat16, torch.bfloat16, 4)
    good = P.layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu()
    x[3, 5] = float("nan")
    x[7, 699] = float("inf")
    y = P.layer_norm(x.cuda(), w.cuda(), b.cuda()).cpu()
    keep = [r for r in range(12) if r not in (3, 7)]
    assert torch.equal(y[keep], good[keep]) and y[3].isnan().all() and y[7].isnan().any()


def test_leading_dimensions_and_in_place(P):
    announce("layer_norm in place")
    x, w, b, _ = make(24, 72, torch.float32, torch.float32, 5)
    x, w, b = x.cuda().view(2, 3, 4, 72), w.cuda(), b.cuda()
    y, mean, rstd = P.layer_norm(x, w, b, want_stats=True)
    assert y.shape == x.shape and mean.shape == rstd.shape == (2, 3, 4)
    z = x.clone()
    assert P.layer_norm(z, w, b, out=z) is z and torch.equal(y, z)
    dy = torch.randn_like(x)
    dx, dw, db = P.layer_norm_backward(dy, x, mean, rstd, w)
    dz = dy.clone()
    assert P.layer_norm_backward(dz, x, mean, rstd, w, out=dz)[0] is dz and torch.equal(dx, dz)


@pytest.mark.parametrize("cols", [3, 9, 203, 1003, 2501, 5003, 9001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_in_place_at_widths_that_end_inside_a_piece(P, cols, dtype):
    """The last piece of such a row overlaps the one before it."""
    announce("layer_norm in place %d %s" % (cols, dtype))
    x, w, b, dy = (v.cuda() for v in make(131, cols, TYPES[dtype], torch.float32, 10))
    y, mean, rstd = P.layer_norm(x, w, b, want_stats=True)
    z, dz = x.clone(), dy.clone()
    P.layer_norm(z, w, b, out=z)
    dx = P.layer_norm_backward(dy, x, mean, rstd, w)[0]
    P.layer_norm_backward(dz, x, mean, rstd, w, out=dz)
    assert torch.equal(y, z) and torch.equal(dx, dz)


def backward64(dy, x, mean, rstd, w):
    h = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    d = dy.double()
    g = d * (1 if w is None else w.double())
    a, b = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    return rstd.double()[:, None] * (g - a - h * b), (d * h).sum(0), d.sum(0), g, h, a, b


def check_backward(P, dy, x, mean, rstd, w):
    rows, cols = x.shape
    t = x.dtype
    dev = lambda v: None if v is None else v.cuda()
    dx, dw, db = P.layer_norm_backward(dev(dy), dev(x), dev(mean), dev(rstd), dev(w))
    torch.cuda.synchronize()
    want, want_w, want_b, g, h, a, b = backward64(dy, x, mean, rstd, w)
    r = rstd.double()[:, None]
    # h: two roundings; g: one; their product one more; the sums a chain each
    d_a = (CHAIN + 3) * U * g.abs().mean(-1, keepdim=True)
    d_b = (CHAIN + 7) * U * (g * h).abs().mean(-1, keepdim=True)
    f32 = r * (U * g.abs() + d_a + h.abs() * d_b + 4 * U * (h * b).abs() + 3 * U * (g.abs() + a.abs() + (h * b).abs())) + U * want.abs()
    bound = f32 + half_step(t) * (want.abs() + f32) + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    off = (dx.cpu().double() - want).abs()
    assert (off <= bound * 1.001).all(), float((off / bound).max())
    # over the rows: those of a group one after the other, up to 4 joins, a 1/8 of up to 256 workgroups, 8 waves
    chain = -(-rows // min(rows, 256)) + 4 + 32 + 8
    d = dy.double()
    for got, exact, size, extra in ((dw, want_w, (d * h).abs().sum(0), 4), (db, want_b, d.abs().sum(0), 0)):
        off = (got.cpu().double() - exact).abs()
        assert (off <= (chain + extra) * U * size * 1.001 + 1e-45).all(), float((off / size).max() / U)
    return dx, dw, db


@pytest.mark.parametrize("shape", SHAPES + [(5001, 96), (2049, 4096), (600, 8208), (530, 12001), (520, 16384)])
@pytest.mark.parametrize("types", ["f32 f32", "bf16 f32", "bf16 bf16", "f16 f32", "f16 f16"])
def test_backward(P, shape, types):
    t, wt = (TYPES[n] for n in types.split())
    announce("layer_norm_backward %s %s" % (shape, types))
    x, w, b, dy = make(*shape, t, wt, 6)
    _, mean, rstd, _ = forward64(x, w, b, 1e-5)
    check_backward(P, dy, x, mean[:, 0].float(), rstd[:, 0].float(), w)


def test_backward_without_weights_or_their_gradients(P):
    announce("layer_norm_backward variants")
    x, w, b, dy = make(300, 264, torch.bfloat16, torch.float32, 7)
    _, mean, rstd, _ = forward64(x, w, b, 1e-5)
    mean, rstd = mean[:, 0].float(), rstd[:, 0].float()
    check_backward(P, dy, x, mean, rstd, None)
    dx, dw, db = check_backward(P, dy, x, mean, rstd, w)
    alone = P.layer_norm_backward(dy.cuda(), x.cuda(), mean.cuda(), rstd.cuda(), w.cuda(), want_weight_grads=False)
    assert torch.equal(alone[0], dx) and alone[1] is None and alone[2] is None
    again = P.layer_norm_backward(dy.cuda(), x.cuda(), mean.cuda(), rstd.cuda(), w.cuda())
    assert all(torch.equal(p, q) for p, q in zip(again, (dx, dw, db)))          # the same sums in the same order


def test_gradients_against_differences(P):
    """d loss / d x, w, b of loss = sum(y * c) from the calls, against central differences of the same function in float64."""
    announce("layer_norm gradients by differences")
    x, w, b, c = make(4, 24, torch.float32, torch.float32, 8)
    y, mean, rstd = P.layer_norm(x.cuda(), w.cuda(), b.cuda(), want_stats=True)
    dx, dw, db = (v.cpu().double() for v in P.layer_norm_backward(c.cuda(), x.cuda(), mean, rstd, w.cuda()))
    loss = lambda x, w, b: float((forward64(x, w, b, 1e-5)[0] * c.double()).sum())
    x, w, b = x.double(), w.double(), b.double()
    step = 1e-6                           # differences: step^2 of the third derivative, and 2^-53 of the loss over the step
    for grad, at, which in ((dx, x, 0), (dw, w, 1), (db, b, 2)):
        for i in range(0, at.numel(), 5):
            args = [x, w, b]
            ends = []
            for s in (step, -step):
                moved = at.clone()
                moved.view(-1)[i] += s
                ends.append(loss(*(moved if k == which else v for k, v in enumerate(args))))
            slope = (ends[0] - ends[1]) / (2 * step)
            assert abs(slope - float(grad.view(-1)[i])) < 1e-5 * (1 + abs(slope))


def test_captured_and_on_another_stream(P):
    announce("layer_norm captured")
    x, w, b, dy = (v.cuda() for v in make(260, 520, torch.bfloat16, torch.float32, 9))

    def step():
        y, mean, rstd = P.layer_norm(x, w, b, want_stats=True)
        return (y, mean, rstd) + P.layer_norm_backward(dy, x, mean, rstd, w)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for k in range(3):
        x.normal_()
        dy.normal_()
        graph.replay()
        want = step()                     # eager work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, kept)), k


def test_offsets_past_32_bits(P):
    """More than 2^31 elements: the last rows are those of a call on them alone."""
    announce("layer_norm 131080 x 16384 f16")
    rows, cols = 131080, 16384
    x = torch.empty((rows, cols), dtype=torch.float16, device="cuda")
    x[:8].normal_()
    x[8:-8].zero_()
    x[-8:].normal_()
    y = P.layer_norm(x)
    assert torch.equal(y[-8:], P.layer_norm(x[-8:].clone())) and torch.equal(y[:8], P.layer_norm(x[:8].clone()))
    assert (y[rows // 2] == 0).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_of_one_number(P, dtype):
    """Sums of equal numbers of 16 bits are exact in f32, bf16 of any width and f16 up to 8192 columns: such rows are exactly zero behind the mean.  f32 rows
    are as far from it as the sum's roundings put the mean."""
    t = TYPES[dtype]
    for rows, cols in ((200, 1003), (40, 96), (3, 8192), (600, 5001), (2, 7909), (5, 7), (2, 16384 if dtype == "bf16" else 4099)):
        announce("layer_norm rows of one number %d x %d %s" % (rows, cols, dtype))
        g = torch.Generator().manual_seed(11)
        value = (torch.randn((rows, 1), generator=g) * 100).to(t)
        b = torch.randn((cols,), generator=g)
        y, mean, rstd = (v.cpu() for v in P.layer_norm(value.expand(rows, cols).contiguous().cuda(), None, b.cuda(), eps=0.25, want_stats=True))
        if dtype == "f32":
            off = (CHAIN + 2) * U * value.double().abs()
            assert ((mean.double() - value[:, 0].double()).abs() <= off[:, 0]).all()
            assert ((y.double() - b.double()).abs() <= off * 2 * 1.001 + 2 * U * (b.double().abs() + off * 2)).all()      # (x - mean, times a rstd of at most 2, plus b)
        else:
            assert torch.equal(mean, value[:, 0].float()) and (rstd == 2).all() and torch.equal(y, b.to(t).expand(rows, cols))
