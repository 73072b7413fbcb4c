"""8-bit blocks and their product on the GPU against float64, with bounds counted from the roundings."""
import math

import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


@pytest.fixture(scope="module")
def M():
    from ml import matmul
    return matmul


def blocks(n):
    return -(-n // 128)


# ---- quantize_blocks -----------------------------------------------------------------------------

def scales64(x, high, most):
    """The scales of x (f64, CPU) in blocks of `high` x 128, as f32."""
    rows, cols = x.shape
    r, c = blocks(rows) * 128 if high == 128 else rows, blocks(cols) * 128
    pad = torch.zeros((r, c), dtype=torch.float64)
    pad[:rows, :cols] = x
    amax = pad.view(r // high, high, c // 128, 128).abs().amax((1, 3))
    # (f64 holds the quotient of two f32 numbers closely enough that rounding it to f32 is rounding the quotient)
    return torch.clamp((amax / most).float(), min=2.0 ** -126)


def spread(s, rows, cols, high):
    return s.repeat_interleave(128, 1)[:, :cols].repeat_interleave(high, 0)[:rows]


def check_form(q, scale, x, high, f8):
    rows, cols = x.shape
    t, most = F8[f8], torch.finfo(F8[f8]).max
    assert q.dtype == t and tuple(q.shape) == (rows, -(-cols // 16) * 16)
    want = scales64(x, high, most)
    assert torch.equal(scale.cpu(), want)
    got = q.cpu().float().double()
    assert (got[:, cols:] == 0).all()
    quotient = x / spread(want, rows, cols, high).double()
    nearest = quotient.float().to(t).double()
    # as near to the quotient as its nearest number, or as one that is a rounding of f32 further off
    assert ((got[:, :cols] - quotient).abs() <= (nearest - quotient).abs() + 2 * U * quotient.abs()).all()


QUANT_SHAPES = [(1, 1), (1, 128), (2, 129), (17, 16), (128, 128), (127, 255), (130, 1003), (1003, 130), (256, 384), (5, 4096), (300, 17)]


@pytest.mark.parametrize("shape", QUANT_SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("high,f8", [(1, "e4m3"), (1, "e5m2"), (128, "e4m3"), (128, "e5m2")])
def test_quantize(M, shape, dtype, high, f8):
    announce("quantize_blocks %s %s %d %s" % (shape, dtype, high, f8))
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(shape, generator=g) * torch.exp(2 * torch.randn((shape[1],), generator=g))).to(TYPES[dtype])
    d = x.cuda()
    q, s = M.quantize_blocks(d, (high, 128), F8[f8])
    check_form(q, s, x.double(), high, f8)
    qt, st = M.quantize_blocks(d, (high, 128), F8[f8], transpose=True)
    check_form(qt, st, x.double().t().contiguous(), high, f8)
    both = M.quantize_blocks(d, (high, 128), F8[f8], transpose="both")
    for p, w in zip(both, (q, s, qt, st)):
        assert torch.equal(p.view(torch.uint8), w.view(torch.uint8))


@pytest.mark.parametrize("rows,cols", [(2053, 4099), (8200, 4500)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_transposed_in_many_tiles(M, rows, cols, dtype):
    announce("quantize_blocks transposed %d x %d %s" % (rows, cols, dtype))
    x = torch.randn((rows, cols), generator=torch.Generator().manual_seed(2)).to(TYPES[dtype])
    d = x.cuda()
    q, s = M.quantize_blocks(d, transpose=True)
    check_form(q, s, x.t().contiguous().double(), 1, "e4m3")
    both = M.quantize_blocks(d, transpose="both")
    assert torch.equal(both[2].view(torch.uint8), q.view(torch.uint8)) and torch.equal(both[3], s)


def test_quantize_every_8_bit_number_and_every_tie(M):
    """Numbers of the type times a power of two come back, and those half-way between two go to the even one."""
    announce("quantize_blocks ties")
    for f8, t in F8.items():
        codes = torch.arange(256, dtype=torch.uint8).view(t).float()
        values = codes[codes.isfinite()].unique()
        ties = (values[1:] + values[:-1]) / 2
        most = torch.finfo(t).max
        for v, want in ((values, values), (ties, ties.to(t).float())):
            rows = torch.zeros((len(v), 128))
            rows[:, 5] = v
            rows[:, 99] = most                                 # fixes the scale at 1
            q, s = M.quantize_blocks((rows * 0.25).cuda(), dtype=t)
            assert (s.cpu() == 0.25).all() and torch.equal(q.cpu().float()[:, 5], want)


def test_quantize_zeros_tiny_and_huge_numbers(M):
    announce("quantize_blocks extremes")
    x = torch.zeros((6, 256))
    x[1] = 1e-44                                               # subnormal f32
    x[2] = 3.3e38
    x[3, :128] = torch.linspace(-1e-38, 1e-38, 128)
    x[4, 7] = 2.0 ** -126
    x[5] = torch.linspace(-1, 1, 256) * 1e30
    for f8 in F8:
        for high in (1, 128):
            q, s = M.quantize_blocks(x.cuda(), (high, 128), F8[f8])
            check_form(q, s, x.double(), high, f8)
    assert (M.quantize_blocks(torch.zeros((3, 40)).cuda())[0].cpu().view(torch.uint8) == 0).all()


def test_quantize_bad_numbers_stay_in_their_block(M):
    announce("quantize_blocks NaN and inf")
    x = torch.randn((140, 300), generator=torch.Generator().manual_seed(3))
    good = M.quantize_blocks(x.cuda(), transpose="both")
    y = x.clone()
    y[3, 130] = float("nan")
    y[139, 7] = float("-inf")
    q, s, qt, st = (v.cpu() for v in M.quantize_blocks(y.cuda(), transpose="both"))
    f = q.float()
    assert f[3, 128:256].isnan().all() and f[139, :128].isnan().all() and s[3, 1].isnan() and s[139, 0].isinf()
    bad = torch.zeros(f.shape, dtype=torch.bool)
    bad[3, 128:256] = bad[139, :128] = True
    assert torch.equal(f[~bad], good[0].cpu().float()[~bad])
    ft = qt.float()
    assert ft[130, :128].isnan().all() and ft[7, 128:140].isnan().all() and st[130, 0].isnan() and st[7, 1].isinf()
    assert not ft[131].isnan().any() and not ft[130, 128:].isnan().any()
    q, s = (v.cpu() for v in M.quantize_blocks(y.cuda(), (128, 128)))
    assert q.float()[:128, 128:256].isnan().all() and s[0, 1].isnan() and s[1, 0].isinf() and not q.float()[:128, :128].isnan().any()


def test_quantize_offsets_past_32_bits(M):
    announce("quantize_blocks 131200 x 16400 f16")
    rows, cols = 131200, 16400
    x = torch.empty((rows, cols), dtype=torch.float16, device="cuda")
    x[:128].normal_()
    x[128:-128].zero_()
    x[-128:].normal_()
    q, s, qt, st = M.quantize_blocks(x, transpose="both")
    for part, at in ((slice(0, 128), 0), (slice(rows - 128, rows), blocks(rows) - 1)):
        a, b, at_, bt = M.quantize_blocks(x[part].clone(), transpose="both")
        assert torch.equal(q[part].view(torch.uint8), a.view(torch.uint8)) and torch.equal(s[part], b)
        assert torch.equal(qt[:, part].contiguous().view(torch.uint8), at_.view(torch.uint8)) and torch.equal(st[:, at], bt[:, 0])


# ---- matmul_abt_scaled ---------------------------------------------------------------------------

def operands(m, n, k, wide, fa, fb, seed, whole=False):
    """Operands and scales on the CPU; whole: small integers and powers of two, whose sums are exact in f32."""
    g = torch.Generator().manual_seed(seed)
    if whole:
        a, b = (torch.randint(-4, 5, (r, k), generator=g).float() for r in (m, n))
        power = lambda *shape: torch.exp2(torch.randint(-1, 2, shape, generator=g).float())
        sa, sb = power(m, blocks(k)), power(blocks(n) if wide else n, blocks(k))
    else:
        a, b = (torch.randn((r, k), generator=g) * torch.finfo(F8[f]).max / 6 for r, f in ((m, fa), (n, fb)))
        a, b = (v.clamp(-torch.finfo(F8[f]).max, torch.finfo(F8[f]).max) for v, f in ((a, fa), (b, fb)))
        sa = torch.rand((m, blocks(k)), generator=g) + 0.5
        sb = (torch.rand((blocks(n) if wide else n, blocks(k)), generator=g) + 0.5) * 1e-3
    return a.to(F8[fa]), sa, b.to(F8[fb]), sb


def product64(a, sa, b, sb):
    """(the sum, the sum of the magnitudes) in f64 on the GPU."""
    m, n, k = a.shape[0], b.shape[0], a.shape[1]
    da = a.cuda().double() * spread(sa, m, k, 1).cuda().double()
    db = b.cuda().double() * spread(sb, n, k, 1 if sb.shape[0] == n else 128).cuda().double()
    return da @ db.t(), da.abs() @ db.abs().t()


# every kernel: few rows, few tiles, full ones; sides that are no multiple of a tile, K below a block, behind one, and with a tail of one chunk
PRODUCTS = [(1, 1, 16), (1, 128, 128), (1, 4096, 1040), (2, 130, 112), (7, 33, 272), (16, 256, 4096), (17, 100, 144), (31, 515, 2064), (33, 48, 128), (49, 1003, 528),
            (64, 64, 640), (65, 17, 384), (100, 300, 1168), (128, 128, 128), (129, 257, 272), (1000, 1500, 400), (2304, 1153, 272), (1537, 2050, 144),
            (2048, 2304, 1024), (4100, 3000, 528), (1, 24700, 272), (20, 24580, 1168), (49, 25001, 2576), (64, 32768, 128), (4224, 4112, 144)]


@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_of_whole_numbers_is_exact(M, m, n, k, wide):
    """Every element of A, B and both scales counts: sums of integers times powers of two have no rounding."""
    announce("matmul_abt_scaled whole %d %d %d %s" % (m, n, k, wide))
    a, sa, b, sb = operands(m, n, k, wide, "e4m3", "e4m3", 2, whole=True)
    want, size = product64(a, sa, b, sb)
    assert float(size.max()) < 2 ** 22                  # in quarters: below 2^24 of them
    a, sa, b, sb = (v.cuda() for v in (a, sa, b, sb))
    for out in (torch.float32, torch.bfloat16, torch.float16):
        c = M.matmul_abt_scaled(a, sa, b, sb, out_dtype=out)
        assert c.dtype == out and torch.equal(c, want.float().to(out)), (out, (c.double() - want).abs().max())


@pytest.mark.parametrize("types", ["e4m3 e4m3", "e5m2 e4m3", "e4m3 e5m2", "e5m2 e5m2"])
@pytest.mark.parametrize("m,n,k,wide", [(1, 500, 4096, True), (20, 300, 1040, False), (50, 1000, 528, True), (300, 200, 272, False), (2048, 2100, 656, True),
                                        (2100, 2048, 400, False), (17, 25001, 656, False), (3, 24704, 144, True)])
def test_product(M, m, n, k, wide, types):
    fa, fb = types.split()
    announce("matmul_abt_scaled %s" % ((m, n, k, wide, types),))
    a, sa, b, sb = operands(m, n, k, wide, fa, fb, 3)
    want, size = product64(a, sa, b, sb)
    # within a block 128 additions that may cut off instead of rounding, a whole step of f32 each; then two roundings of the scales' product and one per block
    bound = (128 * 2 + 2 + blocks(k) + 8) * U * size
    # 16-bit results: of eight consecutive products what lies below 2^-13 of the largest's power of two is cut off beforehand
    cut = 8 * 2.0 ** -13 * largest_of_eights(a, sa, b, sb)
    a, sa, b, sb = (v.cuda() for v in (a, sa, b, sb))
    off = (M.matmul_abt_scaled(a, sa, b, sb).double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
    for t in (torch.bfloat16, torch.float16):
        off = (M.matmul_abt_scaled(a, sa, b, sb, out_dtype=t).double() - want).abs()
        fine = want.abs() < 60000
        assert (off <= bound + cut + torch.finfo(t).eps / 2 * (want.abs() + bound + cut) + torch.finfo(t).smallest_normal * torch.finfo(t).eps)[fine].all()


def largest_of_eights(a, sa, b, sb):
    """The sum over groups of eight consecutive k of the largest magnitude of their products, scales and all, f64 on the GPU."""
    m, n, k = a.shape[0], b.shape[0], a.shape[1]
    da = (a.cuda().float() * spread(sa, m, k, 1).cuda()).abs()
    db = (b.cuda().float() * spread(sb, n, k, 1 if sb.shape[0] == n else 128).cuda()).abs()
    total = torch.zeros((m, n), device="cuda")
    for at in range(0, k, 8):
        most = torch.zeros((m, n), device="cuda")
        for j in range(at, at + 8):
            most = torch.maximum(most, da[:, j, None] * db[None, :, j])
        total += most
    return total.double() * 1.001


def test_product_of_the_smallest_numbers(M):
    """The subnormal numbers of both types count in full."""
    announce("matmul_abt_scaled subnormal numbers")
    for fa, fb in (("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2"), ("e4m3", "e4m3")):
        for m, n in ((5, 64), (2304, 2304)):
            g = torch.Generator().manual_seed(12)
            small = {"e4m3": (2.0 ** -9, 15), "e5m2": (2.0 ** -16, 7)}       # the smallest number, and how many of them have its step
            draw = lambda r, f: (torch.randint(-small[f][1], small[f][1] + 1, (r, 272), generator=g).float() * small[f][0]).to(F8[f])
            a, b = draw(m, fa).cuda(), draw(n, fb).cuda()
            one = lambda r: torch.ones((r, 3), device="cuda")
            want = a.double() @ b.double().t()
            assert torch.equal(M.matmul_abt_scaled(a, one(m), b, one(n)).double(), want)
            big = 2.0 ** 20                                                  # (so that bf16 results are not subnormal)
            c = M.matmul_abt_scaled(a, one(m) * big, b, one(n), out_dtype=torch.bfloat16)
            assert torch.equal(c, (want * big).float().to(torch.bfloat16))


@pytest.mark.parametrize("m,n,k", [(1, 259, 272), (40, 130, 400), (200, 301, 144), (2051, 2303, 272)])
@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
def test_product_epilogue(M, m, n, k, out):
    """Bias, ReLU and beta C, exact in whole numbers; a width that is no multiple of four leaves what stands behind C alone."""
    announce("matmul_abt_scaled epilogue %s" % ((m, n, k, out),))
    a, sa, b, sb = operands(m, n, k, True, "e4m3", "e4m3", 4, whole=True)
    want, _ = product64(a, sa, b, sb)
    a, sa, b, sb = (v.cuda() for v in (a, sa, b, sb))
    g = torch.Generator().manual_seed(5)
    bias = torch.randint(-50, 51, (n,), generator=g).float().cuda()
    old = torch.randint(-50, 51, (m, n), generator=g).to(TYPES[out])
    backing = torch.full((m * n + 64,), 7.0, dtype=TYPES[out], device="cuda")
    c = backing[:m * n].view(m, n)
    c.copy_(old)
    assert M.matmul_abt_scaled(a, sa, b, sb, c=c, beta=0.5, bias=bias, relu=True) is c
    expected = (want + 0.5 * old.cuda().double() + bias.double()).clamp(min=0)
    assert torch.equal(c, expected.float().to(TYPES[out])) and (backing[m * n:] == 7).all()
    # beta = 0: what C held is not read
    c.fill_(float("nan"))
    M.matmul_abt_scaled(a, sa, b, sb, c=c, bias=bias)
    assert torch.equal(c, (want + bias.double()).float().to(TYPES[out])) and (backing[m * n:] == 7).all()


def test_product_of_bad_numbers(M):
    """A NaN in A is a row of NaNs, one in B a column; an infinite scale does not reach other rows."""
    announce("matmul_abt_scaled NaN")
    for m, n in ((9, 70), (300, 2300), (2300, 2050)):
        a, sa, b, sb = operands(m, n, 272, False, "e4m3", "e4m3", 6)
        codes = a.view(torch.uint8).clone()
        codes[m // 2, 271] = 0x7f
        a, sa, b, sb = codes.view(a.dtype).cuda(), sa.cuda(), b.cuda(), sb.cuda()
        sb[n - 1, 1] = float("inf")
        c = M.matmul_abt_scaled(a, sa, b, sb)
        bad = torch.zeros((m, n), dtype=torch.bool, device="cuda")
        bad[m // 2] = bad[:, n - 1] = True
        assert c[m // 2].isnan().all() and not c[:, n - 1].isfinite().any() and c[~bad].isfinite().all()


def test_a_row_does_not_depend_on_the_others(M):
    announce("matmul_abt_scaled rows")
    for m, n, k in ((13, 100, 656), (2304, 2304, 272), (40, 25000, 272)):
        a, sa, b, sb = (v.cuda() for v in operands(m, n, k, True, "e4m3", "e4m3", 7))
        c = M.matmul_abt_scaled(a, sa, b, sb)
        order = torch.randperm(m, device="cuda")
        shuffled = M.matmul_abt_scaled(a.view(torch.uint8)[order].view(a.dtype), sa[order], b, sb)
        assert torch.equal(shuffled, c[order])


def test_product_captured_and_on_another_stream(M):
    announce("matmul_abt_scaled captured")
    xs = [torch.randn((m, 528), device="cuda") for m in (3, 60, 2200)]
    w = torch.randn((2304, 528), device="cuda")
    w8, sw = M.quantize_blocks(w, (128, 128))

    def step():
        return [M.matmul_abt_scaled(*M.quantize_blocks(x), w8, sw, out_dtype=torch.bfloat16) for x in xs]
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
        for x in xs:
            x.normal_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, kept)), k


def test_a_layer_and_its_gradients(M):
    """y = x W^T, dx = dy W and dW = dy^T x in 8 bits.  Every operand is off by at most half a step of its type relative to the block's
    largest number: 2^-4 of an element, or 2^-10 of the largest (e4m3: 2^-9 times half); e5m2 2^-3, or 2^-17."""
    announce("a layer in 8 bits")
    m, n, k = 272, 400, 528
    g = torch.Generator().manual_seed(8)
    x, w, dy = (torch.randn(s, generator=g) for s in ((m, k), (n, k), (m, n)))
    x8, sx, xt, sxt = M.quantize_blocks(x.cuda(), transpose="both")
    w8, sw, wt, swt = M.quantize_blocks(w.cuda(), (128, 128), transpose="both")
    d8, sd, dt, sdt = M.quantize_blocks(dy.cuda(), dtype=torch.float8_e5m2, transpose="both")
    off4 = lambda v: v.double().abs() * 2.0 ** -4 + float(v.abs().max()) / 448 * 2.0 ** -10
    off5 = lambda v: v.double().abs() * 2.0 ** -3 + float(v.abs().max()) / 57344 * 2.0 ** -17
    for got, p, q, dp, dq in ((M.matmul_abt_scaled(x8, sx, w8, sw), x, w.t(), off4(x), off4(w).t()),
                              (M.matmul_abt_scaled(d8, sd, wt, swt), dy, w, off5(dy), off4(w)),
                              (M.matmul_abt_scaled(dt, sdt, xt, sxt), dy.t(), x, off5(dy).t(), off4(x))):
        p, q = p.double(), q.double()
        bound = dp @ q.abs() + p.abs() @ dq + dp @ dq + 300 * U * ((p.abs() + dp) @ (q.abs() + dq))
        off = (got.cpu().double() - p @ q).abs()
        assert (off <= bound).all()
        assert float(off.norm() / (p @ q).norm()) > 1e-3       # (8 bits were used at all)


def test_weight_gradients_add_up(M):
    """dW over two half batches with beta = 1 is dW over the whole one, in whole numbers."""
    announce("matmul_abt_scaled beta 1")
    a, sa, b, sb = (v.cuda() for v in operands(144, 208, 512, False, "e5m2", "e4m3", 9, whole=True))
    whole = M.matmul_abt_scaled(a, sa, b, sb)
    dw = torch.zeros((144, 208), device="cuda")
    for at in (0, 256):
        part = lambda v, s: (v.view(torch.uint8)[:, at:at + 256].contiguous().view(v.dtype), s[:, at // 128:at // 128 + 2].contiguous())
        M.matmul_abt_scaled(*part(a, sa), *part(b, sb), c=dw, beta=1.0)
    assert torch.equal(dw, whole)


def test_small_products_beside_large_ones_that_cancel(M):
    """Of every eight products along K two are 2^16 and -2^16, the others integers of at most 9: what is left is exact in f32, so every type of C is its
    rounding.  A sum that keeps fewer bits than f32 (13 below the largest of eight, say) has none of it."""
    for m, n in ((5, 64), (40, 130), (200, 301), (49, 25001), (2304, 2304), (4224, 4112)):
        for fa, fb, wide in (("e4m3", "e4m3", True), ("e5m2", "e4m3", False)):
            announce("matmul_abt_scaled cancelling products %s" % ((m, n, fa, fb, wide),))
            g = torch.Generator().manual_seed(13)
            k = 272
            a, b = (torch.randint(-3, 4, (r, k), generator=g).float() for r in (m, n))
            for at in range(0, k, 8):
                p, q = (at + torch.randperm(8, generator=g)[:2]).tolist()
                sign = torch.randint(0, 2, (m,), generator=g) * 512. - 256.
                a[:, p], a[:, q], b[:, p], b[:, q] = sign, -sign, 256., 256.
            power = lambda *shape: torch.exp2(torch.randint(-1, 2, shape, generator=g).float())
            a, sa, b, sb = a.to(F8[fa]), power(m, 3), b.to(F8[fb]), power(blocks(n) if wide else n, 3)
            want, _ = product64(a, sa, b, sb)
            a, sa, b, sb = (v.cuda() for v in (a, sa, b, sb))
            for out in (torch.float32, torch.bfloat16, torch.float16):
                c = M.matmul_abt_scaled(a, sa, b, sb, out_dtype=out)
                assert torch.equal(c, want.float().to(out)), (m, n, out, float((c.double() - want).abs().max()))


@pytest.mark.parametrize("types", ["e4m3 e4m3", "e5m2 e4m3", "e5m2 e5m2"])
@pytest.mark.parametrize("m,n,k,wide", [(1, 500, 4096, True), (50, 1000, 528, True), (300, 200, 272, False), (2048, 2304, 656, True), (4224, 4112, 400, False)])
def test_16_bit_results_are_roundings_of_f32_sums(M, m, n, k, wide, types):
    fa, fb = types.split()
    announce("matmul_abt_scaled 16 bits %s" % ((m, n, k, wide, types),))
    a, sa, b, sb = operands(m, n, k, wide, fa, fb, 14)
    want, size = product64(a, sa, b, sb)
    bound = (128 * 2 + 2 + blocks(k) + 8) * U * size            # of the f32 sums, as in test_product
    a, sa, b, sb = (v.cuda() for v in (a, sa, b, sb))
    for t in (torch.bfloat16, torch.float16):
        off = (M.matmul_abt_scaled(a, sa, b, sb, out_dtype=t).double() - want).abs()
        fine = want.abs() < 60000
        allowed = bound + torch.finfo(t).eps / 2 * (want.abs() + bound) + torch.finfo(t).smallest_normal * torch.finfo(t).eps
        assert (off <= allowed)[fine].all(), float((off / allowed)[fine].max())


@pytest.mark.parametrize("wide", [True, False])
def test_scales_far_apart(M, wide):
    """Only the product of two scales has to be a number of f32: neither times the sum alone does.  Everything here is exact."""
    for m, n in ((5, 64), (40, 130), (200, 301), (49, 25001), (2304, 2304), (4224, 4112)):
        announce("matmul_abt_scaled scales far apart %s" % ((m, n, wide),))
        a, sa, b, sb = operands(m, n, 272, wide, "e5m2", "e5m2", 15, whole=True)
        for step, up in ((1.0, 125), (1.0, -125), (2.0 ** -16, 125), (2.0 ** -16, -125)):
            x, y = (a.float() * step).to(a.dtype), (b.float() * step).to(b.dtype)
            far, near = sa * 2.0 ** up, sb * 2.0 ** -up
            want, _ = product64(x, far, y, near)
            c = M.matmul_abt_scaled(x.cuda(), far.cuda(), y.cuda(), near.cuda())
            assert torch.equal(c.double(), want), (m, n, step, up)


@pytest.mark.parametrize("bad", ["inf", "-inf", "nan"])
@pytest.mark.parametrize("f8", ["e4m3", "e5m2"])
@pytest.mark.parametrize("high", [1, 128])
def test_padding_is_zeros_beside_bad_numbers(M, high, f8, bad):
    """An infinity or a NaN in the last block of a row makes its numbers NaNs, zeros among them, and leaves the columns behind them zeros."""
    for dtype in TYPES:
        for rows, cols in ((1, 1), (3, 7), (140, 300), (131, 1003), (2, 12), (260, 133)):
            announce("quantize_blocks padding %s" % ((rows, cols, high, f8, bad, dtype),))
            x = torch.randn((rows, cols), generator=torch.Generator().manual_seed(17)).to(TYPES[dtype])
            x[rows // 2, cols // 2] = 0
            x[rows - 1, cols - 1] = float(bad)
            for transpose in (False, True, "both"):
                forms = [v.cpu() for v in M.quantize_blocks(x.cuda(), (high, 128), F8[f8], transpose=transpose)]
                for i, form in enumerate(zip(forms[::2], forms[1::2])):
                    q, scale, y = form[0].view(torch.uint8), form[1], x if transpose is False or (transpose == "both" and i == 0) else x.t()
                    assert (q[:, y.shape[1]:] == 0).all() and not scale[-1, -1].isfinite()
                    last = slice((y.shape[0] - 1) // 128 * 128, None) if high == 128 else slice(y.shape[0] - 1, None)
                    assert form[0].float()[last, (y.shape[1] - 1) // 128 * 128:y.shape[1]].isnan().all()


# Loops long enough that every stage of LDS, those of the scales among them, is filled again and again, with a tail of K; on 256 compute units these
# are the 16 x 16, 32 x 32 and 64 x 64 split tiles, then 128 x 128 and 128 x 256
@pytest.mark.parametrize("wide", [True, False])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 8208), (9, 300, 12304), (20, 3000, 8208), (100, 515, 12304), (49, 12850, 8208), (2048, 2304, 1040), (2048, 2304, 2320),
                                   (2100, 2241, 4176), (4224, 4112, 1040), (4100, 2200, 2320), (4096, 2304, 4112)])
def test_product_of_many_blocks_is_exact(M, m, n, k, wide):
    announce("matmul_abt_scaled many blocks %s" % ((m, n, k, wide),))
    a, sa, b, sb = operands(m, n, k, wide, "e4m3", "e5m2", 16, whole=True)
    want, size = product64(a, sa, b, sb)
    assert float(size.max()) < 2 ** 22                  # in quarters: below 2^24 of them
    a, sa, b, sb = (v.cuda() for v in (a, sa, b, sb))
    for out in (torch.float32, torch.bfloat16):
        c = M.matmul_abt_scaled(a, sa, b, sb, out_dtype=out)
        assert torch.equal(c, want.float().to(out)), (out, (c.double() - want).abs().max())


def test_a_layer_and_its_gradients_at_odd_sizes(M):
    """What both operands of a product are padded with are zeros of the same width: the three products have the shapes and values of the plain ones."""
    announce("a layer in 8 bits, odd sizes")
    m, n, k = 261, 133, 515
    g = torch.Generator().manual_seed(18)
    x, w, dy = (torch.randint(-3, 4, s, generator=g).float() for s in ((m, k), (n, k), (m, n)))
    for v in (x, w, dy):                                        # scales of 1 or powers of two: 448 or 57344 in every block
        v[::64, ::64] = 448.
    dy[dy == 448.] = 57344.
    x8, sx, xt, sxt = M.quantize_blocks(x.cuda(), (1, 128), transpose="both")
    w8, sw, wt, swt = M.quantize_blocks(w.cuda(), (128, 128), transpose="both")
    d8, sd, dt, sdt = M.quantize_blocks(dy.cuda(), dtype=torch.float8_e5m2, transpose="both")
    back = lambda q, s, rows, cols: q.cpu().double()[:, :cols] * spread(s.cpu(), rows, cols, 1 if s.shape[0] == rows else 128).double()
    for got, a, b in ((M.matmul_abt_scaled(x8, sx, w8, sw), back(x8, sx, m, k), back(w8, sw, n, k)),
                      (M.matmul_abt_scaled(d8, sd, wt, swt), back(d8, sd, m, n), back(wt, swt, k, n)),
                      (M.matmul_abt_scaled(dt, sdt, xt, sxt), back(dt, sdt, n, m), back(xt, sxt, k, m))):
        assert got.shape == (a.shape[0], b.shape[0])
        size = a.abs() @ b.abs().t()
        assert ((got.cpu().double() - a @ b.t()).abs() <= (128 * 2 + 2 + 5 + 8) * U * size).all()      # (as in test_product)


def test_relu_makes_a_nan_zero(M):
    announce("matmul_abt_scaled NaN and ReLU")
    for m, n in ((9, 70), (40, 130), (300, 2301), (2304, 2304)):
        a, sa, b, sb = operands(m, n, 272, True, "e4m3", "e4m3", 19)
        codes = a.view(torch.uint8).clone()
        codes[m // 2, 271] = 0x7f
        a, sa, b, sb = codes.view(a.dtype).cuda(), sa.cuda(), b.cuda(), sb.cuda()
        for out in (torch.float32, torch.bfloat16, torch.float16):
            c = M.matmul_abt_scaled(a, sa, b, sb, relu=True, out_dtype=out)
            assert (c[m // 2] == 0).all() and torch.equal(c, M.matmul_abt_scaled(a, sa, b, sb, out_dtype=out).nan_to_num(0, math.inf).clamp(min=0))


@pytest.mark.parametrize("m,n,k", [(70016, 32771, 32), (5, 140011, 16400), (140011, 130, 16400), (40, 140011, 16400)])
def test_product_offsets_past_32_bits(M, m, n, k):
    """More than 2^31 elements of C, of B or of A: the corners are those of a product of them alone, in whole numbers."""
    announce("matmul_abt_scaled %d x %d x %d" % (m, n, k))
    g = torch.Generator(device="cuda").manual_seed(20)
    draw = lambda r: torch.randint(-3, 4, (r, k), generator=g, device="cuda", dtype=torch.int8).to(torch.float8_e4m3fn)
    scale = lambda r: torch.exp2(torch.randint(-1, 2, (r, blocks(k)), generator=g, device="cuda").float())
    a, sa, b, sb = draw(m), scale(m), draw(n), scale(n)
    c = M.matmul_abt_scaled(a, sa, b, sb, out_dtype=torch.bfloat16)
    ends = lambda r: torch.arange(r, device="cuda").unique() if r <= 300 else torch.cat([torch.arange(130, device="cuda"), torch.arange(r - 130, r, device="cuda")])
    rows, cols = ends(m), ends(n)
    part = lambda v, at: v.view(torch.uint8)[at].view(v.dtype)
    want, _ = product64(part(a, rows), sa[rows], part(b, cols), sb[cols])
    assert torch.equal(c[rows][:, cols], want.float().bfloat16())
