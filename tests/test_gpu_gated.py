"""The gated feed-forward block and its gradients on the GPU against the definitions in 64 bits, with bounds that count the roundings."""
import math

import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
F8 = torch.float8_e4m3fn
U = 2.0 ** -24                        # a rounding of f32
TINY = 2.0 ** -126


@pytest.fixture(scope="module")
def M():
    from ml import matmul
    return matmul


def operands(m, n, k, dtype, seed=0, with_dc=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda a, b, s: (torch.randn((a, b), generator=g, device="cuda") * s).to(TYPES[dtype])
    x, gate, up = r(m, k, 1.0), r(n, k, 1.5 / math.sqrt(k)), r(n, k, 1.0 / math.sqrt(k))
    return (x, gate, up, r(m, n, 1.0)) if with_dc else (x, gate, up)


def activation(g, name):
    """act(g), act'(g) in f64."""
    if name == "relu":
        return torch.relu(g), (g > 0).double()
    if name == "gelu":
        below = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
        return g * below, below + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return g * s, s * (1 + g * torch.sigmoid(-g))


def of_activation(g):
    """What act and act' computed in f32 are off: a few roundings of numbers up to 1 + |g|, and an exponential whose argument, up to g^2, is rounded
    (where the argument is above 100 it is 0 or infinite either way)."""
    return 8 * U * (1 + g.abs()) * (1 + (g * g).clamp(max=128) / 4)


def rounded(v, dtype):
    """How far a number of `dtype` may be from v, of which it is the rounding; f16 has numbers below its smallest normal one."""
    info = torch.finfo(dtype)
    return v.abs() * (info.eps / 2) + info.tiny * info.eps / 2


def products(x, gate, up):
    """g, u in f64, and bounds of f32 sums of them: any order of K products and sums is within (K + 1) roundings of the sum of magnitudes."""
    x, gate, up = x.double(), gate.double(), up.double()
    k = x.shape[1]
    return x @ gate.t(), x @ up.t(), (k + 1) * U * (x.abs() @ gate.abs().t()), (k + 1) * U * (x.abs() @ up.abs().t())


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    ok = off <= bound
    assert ok.all(), (what, tuple((~ok).nonzero()[0].tolist()), (off / bound).max().item(), off.max().item(), int((~ok).sum()))


def values(q, scale, cols):
    return q[:, :cols].double() * scale.double().repeat_interleave(128, 1)[:, :cols]


def check_kept_f8(q, scale, v, of_v, what):
    m, n = v.shape
    assert q.dtype == F8 and q.shape == (m, -(-n // 16) * 16) and scale.shape == (m, -(-n // 128))
    assert (q[:, n:].float() == 0).all(), what + ": padding"
    pad = lambda t: torch.nn.functional.pad(t, (0, -n % 128)).unflatten(1, (-1, 128)).amax(2)
    most, of_most = pad(v.abs()), pad(of_v)
    want = (most / 448).clamp(min=TINY)
    within(scale, want, of_most / 448 + 2 * U * want, what + ": scale")
    # a code is the nearest one to v over its scale, half a step off: 2^-4 of the value, or of the smallest normal number 2^-6; v is of_v off
    each = (want + of_most / 448).repeat_interleave(128, 1)[:, :n]
    within(values(q, scale, n), v, 2.0 ** -4 * torch.maximum(v.abs() + of_v, each * 2.0 ** -6) * (1 + 2.0 ** -4) + of_v + 4 * U * v.abs(), what)


def check_forward(M, x, gate, up, act, keep=None):
    out = M.matmul_abt_gated(x, gate, up, activation=act, keep=keep)
    torch.cuda.synchronize()
    c, kept = out if keep is not None else (out, None)
    g, u, of_g, of_u = products(x, gate, up)
    a, _ = activation(g, act)
    of_a = 1.2 * of_g + of_activation(g)                # (no slope is above 1.13)
    want = a * u
    bound = a.abs() * of_u + u.abs() * of_a + of_a * of_u + 2 * U * want.abs()
    assert c.dtype == x.dtype and c.shape == want.shape
    within(c, want, bound + rounded(want.abs() + bound, x.dtype), "c")
    if keep is None:
        return c, None
    if keep == F8:
        check_kept_f8(kept[0], kept[1], g, of_g, "gate")
        check_kept_f8(kept[2], kept[3], u, of_u, "up")
    else:
        for t, v, of, what in ((kept[0], g, of_g, "gate"), (kept[1], u, of_u, "up")):
            assert t.dtype == x.dtype and t.shape == v.shape
            within(t, v, of + rounded(v.abs() + of, x.dtype), what)
    return c, kept


def check_backward(M, dc, x, gate, up, kept, act, **want):
    n = gate.shape[0]
    got = M.matmul_abt_gated_backward(dc, x, gate, up, kept, activation=act, **want)
    torch.cuda.synchronize()
    g, u = (kept[0].double(), kept[1].double()) if len(kept) == 2 else (values(kept[0], kept[1], n), values(kept[2], kept[3], n))
    if len(kept) == 4:                                  # (a number of 8 bits times its scale is a f32)
        g, u = g.float().double(), u.float().double()
    a, slope = activation(g, act)
    d = dc.double()
    dg, du = d * u * slope, d * a
    of_dg = d.abs() * u.abs() * (of_activation(g) + 4 * U * slope.abs())
    of_du = d.abs() * (of_activation(g) + 4 * U * a.abs())
    of_dg, of_du = of_dg + rounded(dg.abs() + of_dg, x.dtype), of_du + rounded(du.abs() + of_du, x.dtype)
    xd, gd, ud = x.double(), gate.double(), up.double()

    def check_one(t, parts, adds, what):
        want = sum(p @ q for p, _, q in parts)
        bound = sum(of @ q.abs() + (adds + 2) * U * ((p.abs() + of) @ q.abs()) for p, of, q in parts)
        assert t.dtype == x.dtype and t.shape == want.shape
        within(t, want, bound + rounded(want.abs() + bound, x.dtype), what)

    if got[0] is not None:
        check_one(got[0], ((dg, of_dg, gd), (du, of_du, ud)), 2 * n, "da")
    if got[1] is not None:
        check_one(got[1], ((dg.t(), of_dg.t(), xd),), x.shape[0], "db_gate")
        check_one(got[2], ((du.t(), of_du.t(), xd),), x.shape[0], "db_up")
    return got


# every tile and its ends: rows, columns and K of one, below, at and above the tiles and K-tiles
SMALL = [(1, 1, 8), (1, 33, 64), (2, 16, 16), (3, 130, 72), (17, 128, 128), (16, 2667, 1000), (33, 300, 56), (49, 129, 40), (64, 128, 64), (65, 257, 200), (128, 64, 192), (255, 129, 1000),
         (300, 700, 264), (129, 513, 520)]
# every tile where there are many, whole and not
LARGE = [(2048, 1664, 64), (2047, 1663, 72), (4096, 1664, 128), (4095, 1663, 200), (512, 2736, 1024), (511, 2735, 1000), (1024, 2736, 1024), (1021, 2731, 520), (2048, 4096, 256),
         (2043, 4099, 264), (1, 4096, 2048), (15, 4099, 2056), (40, 4096, 512), (97, 2737, 1032)]


@pytest.mark.parametrize("m,n,k", SMALL + LARGE)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_forward(M, m, n, k, dtype):
    for act in ("silu", "gelu", "relu"):
        announce("matmul_abt_gated %s" % ((m, n, k, dtype, act),))
        check_forward(M, *operands(m, n, k, dtype), act)


@pytest.mark.parametrize("m,n,k", SMALL + LARGE)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("keep", ["whole", "f8"])
def test_kept(M, m, n, k, dtype, keep):
    announce("matmul_abt_gated keep %s" % ((m, n, k, dtype, keep),))
    x, gate, up = operands(m, n, k, dtype, seed=1)
    c, _ = check_forward(M, x, gate, up, "silu", keep=F8 if keep == "f8" else x.dtype)
    assert c.shape == (m, n)


# large tiles and, for the rows behind them, smaller ones
@pytest.mark.parametrize("m,n,k", [(5043, 1542, 8), (1795, 4555, 72), (2389, 3359, 128), (3440, 2411, 200), (3000, 5461, 64)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("keep", ["none", "whole", "f8"])
def test_rows_in_two_tiles(M, m, n, k, dtype, keep):
    announce("matmul_abt_gated two tiles %s" % ((m, n, k, dtype, keep),))
    x, gate, up = operands(m, n, k, dtype, seed=11)
    check_forward(M, x, gate, up, "silu", keep={"none": None, "whole": x.dtype, "f8": F8}[keep])


def test_f32_in_multiples_of_four(M):
    for m, n, k in ((5, 7, 4), (70, 130, 12), (100, 65, 36)):
        announce("matmul_abt_gated f32 %s" % ((m, n, k),))
        x, gate, up, dc = operands(m, n, k, "f32", with_dc=True)
        _, kept = check_forward(M, x, gate, up, "gelu", keep=x.dtype)
        check_backward(M, dc, x, gate, up, kept, "gelu")


# for the gradients: rows, columns and inner width each below, at and above a tile, with every other small
BACK = [(1, 1, 8), (2, 40, 16), (64, 64, 64), (65, 63, 72), (63, 65, 56), (128, 128, 128), (129, 31, 200), (300, 700, 264), (37, 2667, 1000), (1000, 33, 24),
        (2048, 40, 1664), (2047, 41, 1672), (4096, 64, 3336), (4095, 65, 3336), (70, 1024, 1664), (71, 1023, 1672), (70, 2048, 3336), (72, 2047, 3336),
        # sums that several workgroups share, on every tile: of long N, of many rows, of both
        (64, 4096, 256), (65, 5461, 264), (250, 4096, 256), (256, 5461, 2048), (509, 4099, 1032), (2048, 2736, 1024), (2043, 2731, 1032), (4096, 1024, 512), (8191, 257, 136), (8192, 1024, 128),
        (16384, 256, 256), (4099, 4099, 264), (8192, 1024, 512), (8192, 512, 4096), (16384, 512, 4096), (2048, 5461, 2048), (2048, 512, 4096), (2043, 509, 4104)]


@pytest.mark.parametrize("m,n,k", BACK)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_backward(M, m, n, k, dtype, act):
    announce("matmul_abt_gated_backward %s" % ((m, n, k, dtype, act),))
    x, gate, up, dc = operands(m, n, k, dtype, seed=2, with_dc=True)
    g = torch.Generator(device="cuda").manual_seed(3)
    kept = tuple((torch.randn((m, n), generator=g, device="cuda") * 1.5).to(x.dtype) for _ in range(2))
    check_backward(M, dc, x, gate, up, kept, act)


@pytest.mark.parametrize("m,n,k", BACK)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_backward_from_8_bits(M, m, n, k, dtype):
    announce("matmul_abt_gated_backward 8 bits %s" % ((m, n, k, dtype),))
    x, gate, up, dc = operands(m, n, k, dtype, seed=4, with_dc=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    kept = sum((tuple(M.quantize_blocks(torch.randn((m, n), generator=g, device="cuda"))) for _ in range(2)), ())
    check_backward(M, dc, x, gate, up, kept, "silu")


# both products with every tile, and what their sizes lead to: shares of K of either or both, the input's workgroups first or the weights'
PLANS_16 = [(29, 359, 2888), (1033, 1027, 32), (3370, 197, 56), (1083, 434, 64), (2118, 296, 48), (2181, 70, 200), (7391, 43, 96), (22, 1541, 896), (4668, 859,
     8), (186, 160, 3824), (412, 20, 3672), (4325, 252, 200), (1296, 22, 1160), (124, 1530, 160), (375, 2712, 40), (4099, 460, 16), (2646, 360, 32),
     (267, 258, 3688), (586, 271, 3600), (9565, 1, 3224), (18, 2006, 920), (237, 1586, 1056), (1164, 528, 3392), (2790, 20, 936), (2844, 7, 1576), (4,
     2467, 3496), (652, 2449, 1040), (10658, 1743, 160)]
PLANS_32 = [(29, 359, 2888), (262, 48, 2408), (551, 182, 312), (7391, 43, 96), (60, 3056, 176), (237, 4767, 32), (75, 134, 3512), (412, 20, 3672), (2181, 70,
     200), (1307, 60, 384), (179, 586, 288), (838, 4719, 8), (1083, 434, 64), (2118, 296, 48)]


@pytest.mark.parametrize("m,n,k,dtype", [p + ("bf16",) for p in PLANS_16] + [p + ("f16",) for p in PLANS_16[::3]] + [p + ("f32",) for p in PLANS_32])
def test_backward_of_every_plan(M, m, n, k, dtype):
    announce("matmul_abt_gated_backward plans %s" % ((m, n, k, dtype),))
    x, gate, up, dc = operands(m, n, k, dtype, seed=6, with_dc=True)
    g = torch.Generator(device="cuda").manual_seed(7)
    kept = tuple((torch.randn((m, n), generator=g, device="cuda") * 1.5).to(x.dtype) for _ in range(2))
    both = check_backward(M, dc, x, gate, up, kept, "silu")
    da, _, _ = M.matmul_abt_gated_backward(dc, x, gate, up, kept, want_weight_grads=False)
    _, db_gate, db_up = M.matmul_abt_gated_backward(dc, x, gate, up, kept, want_input_grad=False)
    assert torch.equal(da, both[0]) and torch.equal(db_gate, both[1]) and torch.equal(db_up, both[2])


def test_gradients_one_by_one(M):
    announce("matmul_abt_gated_backward parts")
    x, gate, up, dc = operands(100, 130, 72, "bf16", with_dc=True)
    _, kept = M.matmul_abt_gated(x, gate, up, keep=x.dtype)
    both = check_backward(M, dc, x, gate, up, kept, "silu")
    da, none, none2 = check_backward(M, dc, x, gate, up, kept, "silu", want_weight_grads=False)
    assert none is None and none2 is None and torch.equal(da, both[0])
    none, dg, du = check_backward(M, dc, x, gate, up, kept, "silu", want_input_grad=False)
    assert none is None and torch.equal(dg, both[1]) and torch.equal(du, both[2])


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradient_is_that_of_differences(M, act):
    """Along a direction of all three operands, from the definition in f64 at both sides."""
    announce("matmul_abt_gated_backward differences " + act)
    x, gate, up, dc = operands(33, 70, 40, "f32", seed=6, with_dc=True)
    _, kept = M.matmul_abt_gated(x, gate, up, activation=act, keep=torch.float32)
    grads = M.matmul_abt_gated_backward(dc, x, gate, up, kept, activation=act)
    g = torch.Generator(device="cuda").manual_seed(7)
    v = [torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64) * t.double().std() for t in (x, gate, up)]

    def loss(step):
        a, b, c = (t.double() + step * w for t, w in zip((x, gate, up), v))
        return (activation(a @ b.t(), act)[0] * (a @ c.t()) * dc.double()).sum()

    step = 1e-4
    want = (loss(step) - loss(-step)) / (2 * step)
    # three steps of Richardson's say what the differences themselves are off: their error goes with step^2
    off = ((loss(2 * step) - loss(-2 * step)) / (4 * step) - want).abs()
    along = sum((t.double() * w).sum() for t, w in zip(grads, v))
    sizes = sum((t.double() * w).abs().sum() for t, w in zip(grads, v))
    assert abs(along - want) <= off + 1e-5 * sizes, (along, want, off, sizes)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_infinities_and_nans_stay_in_their_rows_and_columns(M, dtype):
    """A row of A with a NaN spoils that row of C, a row of a weight that column: nothing else, not where tiles and K-tiles end inside the operands either."""
    announce("matmul_abt_gated special " + dtype)
    for m, n, k in ((70, 130, 72), (65, 129, 200)):
        x, gate, up, dc = operands(m, n, k, dtype, seed=8, with_dc=True)
        clean, kept_clean = M.matmul_abt_gated(x, gate, up, keep=x.dtype)
        _, kept8_clean = M.matmul_abt_gated(x, gate, up, keep=F8)
        grads_clean = M.matmul_abt_gated_backward(dc, x, gate, up, kept_clean)
        x2, gate2, up2 = x.clone(), gate.clone(), up.clone()
        x2[m - 1, k - 1] = math.nan
        gate2[n - 1, 0] = math.inf
        up2[n - 2, k - 1] = math.nan
        c, kept = M.matmul_abt_gated(x2, gate2, up2, keep=x.dtype)
        _, kept8 = M.matmul_abt_gated(x2, gate, up, keep=F8)
        torch.cuda.synchronize()
        assert torch.equal(c[:m - 1, :n - 2], clean[:m - 1, :n - 2])
        assert torch.equal(kept[0][:m - 1, :n - 1], kept_clean[0][:m - 1, :n - 1]) and torch.equal(kept[1][:m - 1, :n - 2], kept_clean[1][:m - 1, :n - 2])
        assert c[m - 1].isnan().all() and c[:m - 1, n - 2].isnan().all()
        assert torch.equal(kept8[0][:m - 1].float(), kept8_clean[0][:m - 1].float()) and kept8[1][m - 1].isnan().all() and (kept8[0][:, n:].float() == 0).all()
        # the last weights' rows do not touch the gradients of the others, and a row of dC only its own row of dA
        dc2 = dc.clone()
        dc2[m - 1] = math.nan
        da = M.matmul_abt_gated_backward(dc2, x, gate, up, kept_clean)[0]
        _, dg, du = M.matmul_abt_gated_backward(dc, x, gate2, up2, tuple(t.clone().index_fill_(1, torch.tensor([n - 1], device="cuda"), math.nan) for t in kept_clean))
        torch.cuda.synchronize()
        assert torch.equal(da[:m - 1], grads_clean[0][:m - 1]) and da[m - 1].isnan().all()
        assert torch.equal(dg[:n - 1], grads_clean[1][:n - 1]) and torch.equal(du[:n - 1], grads_clean[2][:n - 1]) and dg[n - 1].isnan().all()


def test_blocks_of_zeros(M):
    announce("matmul_abt_gated zeros")
    x, gate, up, dc = operands(70, 260, 64, "bf16", with_dc=True)
    gate[128:256] = 0
    x[3] = 0
    c, kept = M.matmul_abt_gated(x, gate, up, keep=F8)
    torch.cuda.synchronize()
    assert (c[:, 128:256] == 0).all() and (c[3] == 0).all() and (kept[1][:, 1] == TINY).all() and (kept[0][3].float() == 0).all()
    check_backward(M, dc, x, gate, up, kept, "silu")


def test_results_behind_four_gib(M):
    announce("matmul_abt_gated past 2^31 elements")
    m, n, k = 300000, 8200, 8
    x, gate, up = operands(m, n, k, "bf16", seed=9)
    c = M.matmul_abt_gated(x, gate, up)
    few = M.matmul_abt_gated(x[-8:].contiguous(), gate, up)
    torch.cuda.synchronize()
    assert torch.equal(c[-8:], few)                      # one K-tile: one order of the sum in every kernel
    del c
    # the workspace of the backward pass is larger still
    dc = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
    dc[-8:] = 1
    kept = (torch.full((m, n), 0.5, dtype=torch.bfloat16, device="cuda"),) * 2
    da, dg, du = M.matmul_abt_gated_backward(dc, x, gate, up, kept)
    small = M.matmul_abt_gated_backward(dc[-8:].contiguous(), x[-8:].contiguous(), gate, up, tuple(t[-8:].contiguous() for t in kept))
    torch.cuda.synchronize()
    assert (da[:-8] == 0).all() and torch.equal(da[-8:], small[0])
    assert torch.equal(dg, small[1]) and torch.equal(du, small[2])


# more workgroups than a launch of 1024 work items each could hold
def test_f32_results_of_many_tiles(M):
    announce("matmul_abt_gated 4194368 tiles")
    m, n, k = 1 << 20, 8193, 4
    x, gate, up = operands(m, n, k, "f32", seed=10)
    c = M.matmul_abt_gated(x, gate, up, "relu")
    for rows in (slice(0, 40), slice(m // 2 - 3, m // 2 + 70), slice(m - 40, m)):
        few = M.matmul_abt_gated(x[rows].contiguous(), gate, up, "relu")
        assert torch.equal(c[rows], few)                 # one K-tile: one order of the sum in every kernel


# ---- as they are used ----

def test_repeats_bit_for_bit_and_on_two_streams(M):
    announce("matmul_abt_gated two streams")
    x, gate, up, dc = operands(200, 300, 136, "bf16", seed=10, with_dc=True)

    def step(keep):
        c, kept = M.matmul_abt_gated(x, gate, up, keep=keep)
        return (c, *kept, *M.matmul_abt_gated_backward(dc, x, gate, up, kept))

    first = {k: step(k) for k in (torch.bfloat16, F8)}
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for k in range(6):
        keep = (torch.bfloat16, F8)[k % 2]
        with torch.cuda.stream(streams[k // 2 % 2]):
            got.append((keep, step(keep)))
    torch.cuda.synchronize()
    for keep, out in got:
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(out, first[keep]))


def test_captured_and_replayed(M):
    announce("matmul_abt_gated graph")
    x, gate, up, dc = operands(130, 300, 72, "f16", seed=11, with_dc=True)

    def step():
        c, kept = M.matmul_abt_gated(x, gate, up, keep=F8)
        return (c, *M.matmul_abt_gated_backward(dc, x, gate, up, kept), M.matmul_abt_gated(x, gate, up, "gelu"))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        x.copy_(operands(130, 300, 72, "f16", seed=20 + k)[0])
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), k


@pytest.mark.parametrize("keep", [None, torch.float32, F8])
def test_recorded_calls_are_those_of_python(M, keep):
    from ml import _lib
    announce("matmul_abt_gated recorded")
    x, gate, up, dc = operands(20, 50, 32, "f32", seed=12, with_dc=True)

    def step():
        if keep is None:
            return (M.matmul_abt_gated(x, gate, up),)
        c, kept = M.matmul_abt_gated(x, gate, up, keep=keep)
        return (c, *kept, *M.matmul_abt_gated_backward(dc, x, gate, up, kept))

    whole = step()
    tape = _lib.start_tape()
    try:
        own = step()
    finally:
        _lib.stop_tape()
    assert len(tape.calls) == (1 if keep is None else 2)
    assert all(a.dtype == b.dtype and torch.equal(a.float(), b.float()) for a, b in zip(whole, own))


def test_a_training_step_of_a_block_and_its_loss(M):
    """Norm, gated block, the products below and above it, the loss over a vocabulary, and back: every gradient against the same graph in f64 by
    autograd, whose one difference is the rounding of what is handed on."""
    from ml import primitives as P
    announce("a block and its loss")
    t, k, n, v = 70, 64, 176, 1003
    g = torch.Generator(device="cuda").manual_seed(13)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    x, w, b = r(t, k), 1 + 0.2 * r(k), 0.2 * r(k)
    gate, up, down, head = r(n, k) / 8, r(n, k) / 8, r(k, n) / 13, r(v, k) / 8
    tokens = torch.randint(0, v, (t,), generator=g, device="cuda").int()
    tokens[::9] = -1
    h, mean, rstd = P.layer_norm(x, w, b, want_stats=True)
    c, kept = M.matmul_abt_gated(h, gate, up, keep=torch.float32)
    y = M.matmul_abt(c, down)
    logits = M.matmul_abt(y, head)
    logp, entropy, lse = P.token_log_probs(logits, tokens, want_entropy=True, want_lse=True)
    loss = -(logp.sum() + 0.1 * entropy.sum())
    ones = torch.full((t,), -1.0, device="cuda")
    dl = P.token_log_probs_backward(ones, logits, tokens, lse, d_entropy=0.1 * ones, entropy=entropy)
    dy = dl @ head                                       # (1003 columns are no multiple of 16 bytes)
    dc = M.matmul_abt(dy, down.t().contiguous())
    dh, dgate, dup = M.matmul_abt_gated_backward(dc, h, gate, up, kept)
    dx, dw, db = P.layer_norm_backward(dh, x, mean, rstd, w)
    leaves = [p.double().requires_grad_() for p in (x, w, b, gate, up)]
    xd, wd, bd, gd, ud = leaves
    hd = torch.nn.functional.layer_norm(xd, (k,), wd, bd)
    logits_d = (torch.nn.functional.silu(hd @ gd.t()) * (hd @ ud.t())) @ down.double().t() @ head.double().t()
    logs = torch.log_softmax(logits_d, 1)
    picked = logs.gather(1, tokens.long().clamp(min=0)[:, None])[:, 0]
    loss_d = -(torch.where(tokens >= 0, picked, 0.0).sum() + 0.1 * -(logs.exp() * logs).sum())
    loss_d.backward()
    # f32 throughout: some 1000 roundings behind each other of sums whose terms do not cancel by more than a factor of some hundred
    assert abs(loss.double() - loss_d) <= 1e-5 * abs(loss_d)
    for got, leaf, name in zip((dx, dw, db, dgate, dup), leaves, ("x", "w", "b", "gate", "up")):
        off = (got.double() - leaf.grad).norm() / leaf.grad.norm()
        assert off <= 2e-5, (name, off)
