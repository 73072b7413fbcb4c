"""Log probabilities of tokens, entropies and alternatives, and their gradient, on the GPU against the definitions in 64 bits."""
import math

import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24                        # a rounding of f32
INF = math.inf


@pytest.fixture(scope="module")
def P():
    from ml import primitives
    return primitives


def logits(rows, cols, dtype, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, cols), generator=g) * spread).to(TYPES[dtype])
    t = (torch.rand(rows, generator=g) * cols).int().clamp(max=cols - 1)
    return x, t


def exact(x, tokens):
    """(logp, entropy, lse, p, what E|ln p| and the like are made of) of the definitions in f64, on the CPU."""
    x = x.double()
    cols = x.shape[1]
    m = torch.where(x.isnan(), -INF, x).amax(1)
    none = (x == -INF).all(1)
    y = x - torch.where(none, 0.0, m)[:, None]           # (NaN at an infinity, as the documentation has it; of a row of the lowest numbers 0, where x - lse would lose the rest)
    s = torch.where(none, 1.0, torch.exp(y).sum(1))
    p = torch.exp(y) / s[:, None]
    entropy = torch.where(none, 0.0, torch.log(s) - torch.where(p == 0, 0.0, p * y).sum(1))
    lse = m + torch.log(s)
    counts = (tokens >= 0) & (tokens < cols)
    at = (y - torch.log(s)[:, None]).gather(1, tokens.long().clamp(0, cols - 1)[:, None])[:, 0]
    logp = torch.where(counts, torch.where(none, -INF, at), 0.0)
    return logp, entropy, lse, p


def bounds(x, lse, p):
    """(of lse, of entropy): every term of s and w is an exp2 of a rounded product, (|y| + 4) roundings and the same again for the unit's own error, and a lane
    adds at most cols / 64 of them behind each other, and some 64 more where lanes, waves and chunks join; the logarithm and its sum with m are a few more."""
    x = x.double()
    cols = x.shape[1]
    m = x.amax(1, keepdim=True)
    far = torch.where(p > 0, (x - m).abs().nan_to_num(0, 0, 0), 0.0) * 1.4427
    mean, square = (p * far).sum(1), (p * far * far).sum(1)
    adds = cols / 64 + 64
    of_sum = U * (2 * mean + 8 + adds)
    of_lse = of_sum + 4 * U * (1 + lse.abs().nan_to_num(0, 0, 0) + m[:, 0].abs().nan_to_num(0, 0, 0))
    return of_lse, of_sum * (2 + mean) + 2 * U * square + 8 * U * (1 + mean)


def same_where_special(got, want):
    """Infinities and NaNs in the same places; True where numbers are to be compared."""
    assert torch.equal(got.isnan(), want.isnan()), (got, want)
    want = want.float().double()                         # (a difference of logits may be no f32)
    inf = want.isinf()
    assert torch.equal(got.double()[inf], want[inf])
    return ~(inf | want.isnan())


def check_forward(P, x, tokens, top=0, **more):
    out = P.token_log_probs(x.cuda(), tokens.cuda(), top=top, want_entropy=True, want_lse=True, **more)
    torch.cuda.synchronize()
    logp, entropy, lse = (t.cpu() for t in out[:3])
    want_logp, want_entropy, want_lse, p = exact(x, tokens)
    of_lse, of_entropy = bounds(x, want_lse, p)
    for name, got, want, bound in (("logp", logp, want_logp, of_lse + 2 * U * want_logp.abs().nan_to_num(0, 0, 0)), ("lse", lse, want_lse, of_lse),
                                   ("entropy", entropy, want_entropy, of_entropy + 2 * U * want_entropy.abs().nan_to_num(0))):
        fine = same_where_special(got, want)
        off = (got.double() - want).abs()[fine]
        assert (off <= bound[fine]).all(), (name, off.max(), bound[fine][off.argmax()])
    if top:
        check_top(x, out[3].cpu(), out[4].cpu(), top, of_lse)
    return logp, entropy, lse


def check_top(x, values, ids, top, of_lse):
    v = torch.where(x.isnan(), -INF, x.float())
    order, at = torch.sort(v, dim=1, descending=True, stable=True)
    k = min(top, x.shape[1])
    want_ids = torch.full((x.shape[0], top), -1, dtype=torch.int32)
    want_ids[:, :k] = torch.where(order[:, :k] > -INF, at[:, :k].int(), -1)
    assert torch.equal(ids, want_ids), (ids[(ids != want_ids).any(1)][:2], want_ids[(ids != want_ids).any(1)][:2])
    want = torch.stack([exact(x, want_ids[:, j])[0] for j in range(top)], 1)
    want = torch.where(want_ids >= 0, want, -INF)
    fine = same_where_special(values, want)
    off = (values.double() - want).abs()
    assert (off <= of_lse[:, None] + 2 * U * want.abs())[fine].all(), off[fine].max()


# rows of every kernel: a few lanes, a wave in one to four pieces, workgroups, chunks of a row; ends inside a piece
SHAPES = [(1, 1), (5, 3), (7, 31), (3, 64), (4, 65), (9, 128), (2, 129), (6, 255), (5, 256), (3, 257), (2, 511), (11, 1003), (4, 1024), (3, 1025), (2, 2048), (3, 2049), (1, 4097),
          (2, 8191), (3, 8193), (1, 32003), (600, 4099), (2, 50257), (1, 131072), (1, 262147)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_forward(P, rows, cols, dtype):
    announce("token_log_probs %s" % ((rows, cols, dtype),))
    x, t = logits(rows, cols, dtype)
    t[rows // 2:rows // 2 + 1] = -1
    check_forward(P, x, t)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (4, 64), (2, 100), (5, 1003), (3, 2049), (1, 8193), (2, 32003), (1, 131072), (520, 4099)])
@pytest.mark.parametrize("top", [1, 5, 32])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_alternatives(P, rows, cols, top, dtype):
    announce("token_log_probs top %s" % ((rows, cols, top, dtype),))
    x, t = logits(rows, cols, dtype, seed=1)
    check_forward(P, x, t, top=top)


@pytest.mark.parametrize("cols", [7, 300, 5000, 20000])
@pytest.mark.parametrize("top", [0, 20])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_rows_with_little_or_nothing_in_them(P, cols, top, dtype):
    announce("token_log_probs special rows %s" % ((cols, top, dtype),))
    x, t = logits(12, cols, dtype, seed=2)
    low = torch.finfo(TYPES[dtype]).min
    x[0] = -INF                                        # nothing
    x[1] = -INF
    x[1, cols - 1] = 2.0                               # one token
    x[2] = low                                         # all alike, at the lowest number
    x[3] = low
    x[3, [0, cols // 2, cols - 1]] = torch.tensor([1.0, 3.0, 2.0]).to(x.dtype)
    x[4] = 0.5                                         # all alike
    x[5, cols // 3] = math.nan
    x[6, cols // 2] = INF
    x[7, ::2] = -INF
    x[8] = -0.0
    x[8, 1::3] = 0.0                                   # zeros of both signs are equal
    x[9] = low
    x[9, 3] = -low                                     # a difference that is no number of the type
    x[10] = math.nan
    x[11, 2:] = -INF
    t[:8] = torch.tensor([0, cols - 1, 1, 0, cols // 2, 0, cols // 2, 0], dtype=torch.int32)
    t[11] = cols                                       # outside
    check_forward(P, x, t, top=top)


def test_large_logits_gathered_in_few_lanes(P):
    """More candidates for the alternatives than a workgroup keeps a list of: the largest logits stand where one lane in 64 looks."""
    for dtype, piece in (("f32", 4), ("bf16", 8)):
        announce("token_log_probs gathered " + dtype)
        g = torch.Generator().manual_seed(3)
        cols = 262144
        x = torch.randn((2, cols), generator=g).to(TYPES[dtype])
        lane = torch.arange(cols) // piece % 64
        x[:, lane == 5] += 20
        rows = x.cuda().repeat(260, 1)                 # more than two rows to a unit: none is split
        out = P.token_log_probs(rows, torch.zeros(520, dtype=torch.int32, device="cuda"), top=32)
        torch.cuda.synchronize()
        order, at = torch.sort(x.float(), dim=1, descending=True, stable=True)
        assert torch.equal(out[2].cpu(), at[:, :32].int().repeat(260, 1))


# rows in chunks, whose own alternatives meet: the largest logits all in one chunk, a few in each, alike, or fewer than are asked for
@pytest.mark.parametrize("rows,cols", [(2, 69474), (1, 32003), (90, 6001), (200, 4100), (1, 131072)])
@pytest.mark.parametrize("top", [1, 2, 7, 31, 32])
def test_alternatives_of_chunks(P, rows, cols, top):
    announce("token_log_probs top of chunks %s" % ((rows, cols, top),))
    x, t = logits(rows, cols, "bf16", seed=21)
    at = torch.arange(cols)
    for row in range(0, rows, 2):
        kind = row // 2 % 5 if rows > 10 else (top + row) % 5
        if kind == 0:
            x[row] = (at / 256).to(x.dtype)                                 # the last chunk's, many alike
        elif kind == 1:
            x[row] = ((at * 7919) % 251).to(x.dtype)                        # every chunk has some of the largest
        elif kind == 2:
            x[row] = 1.25
        elif kind == 3:
            x[row] = torch.where(at % (cols // 20) == 3, x[row], torch.full_like(x[row], -INF))
        else:
            x[row, 1000:1040] = 30 + torch.arange(40).flip(0).to(x.dtype) / 4  # one chunk's alone
    check_forward(P, x, t, top=top)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_every_value_sorted(P, dtype):
    announce("token_log_probs sorted " + dtype)
    for descending in (False, True):
        x = torch.linspace(-8, 8, 30000).to(TYPES[dtype]).sort(descending=descending).values.repeat(2, 1)
        check_forward(P, x.contiguous(), torch.tensor([0, 29999], dtype=torch.int32), top=32)


def test_what_is_wanted_and_shapes(P):
    announce("token_log_probs results")
    x, t = logits(6, 500, "f32")
    x, t = x.cuda().view(2, 3, 500), t.cuda().view(2, 3)
    alone = P.token_log_probs(x, t)
    assert alone.shape == (2, 3) and alone.dtype == torch.float32
    logp, entropy, lse, values, ids = P.token_log_probs(x, t, top=3, want_entropy=True, want_lse=True)
    assert values.shape == ids.shape == (2, 3, 3) and ids.dtype == torch.int32 and entropy.shape == lse.shape == (2, 3)
    logp, lse = P.token_log_probs(x, t, want_lse=True)
    assert torch.equal(logp, alone)
    logp, values, ids = P.token_log_probs(x, t, top=2)
    assert values.shape == (2, 3, 2)


# ---- the gradient ----

def exact_backward(x, tokens, lse, d_logp, d_entropy, entropy, d_lse):
    x = x.double()
    cols = x.shape[1]
    none = lse == -INF
    y = x - torch.where(none, 0.0, lse.double())[:, None]
    p = torch.where(none[:, None], 0.0, torch.exp(y))
    counts = ((tokens >= 0) & (tokens < cols) & ~none).double()
    g = (d_logp.double() if d_logp is not None else torch.zeros_like(lse, dtype=torch.float64)) * counts
    d = -p * g[:, None]
    f = g.abs()[:, None].expand_as(p)
    if d_entropy is not None:
        t = torch.where(p > 0, y, 0.0) + entropy.double()[:, None]
        d = d - d_entropy.double()[:, None] * p * t
        f = f + d_entropy.double().abs()[:, None] * (y.abs().nan_to_num(0, 0, 0) + entropy.double().abs()[:, None])
    if d_lse is not None:
        d = d + d_lse.double()[:, None] * p
        f = f + d_lse.double().abs()[:, None]
    d = d.scatter_add(1, tokens.long().clamp(0, cols - 1)[:, None], g[:, None])
    # p: an exp2 of (x - lse) log2 e, which is rounded twice, and the unit's own error; then a few products and sums of factors as large as f
    y = torch.where(p > 0, y, 0.0).abs()
    return d, p * f * (4 * y + 16) * U


def check_backward(P, x, tokens, which, seed=5, out=False):
    g = torch.Generator().manual_seed(seed)
    rows = x.shape[0]
    _, entropy, lse, _ = exact(x, tokens)
    lse, entropy = lse.float(), entropy.float()
    d_logp, d_entropy, d_lse = (torch.randn(rows, generator=g) if w in which else None for w in ("logp", "entropy", "lse"))
    want, bound = exact_backward(x, tokens, lse, d_logp, d_entropy, entropy, d_lse)
    c = lambda v: None if v is None else v.cuda()
    xg = x.cuda()
    got = P.token_log_probs_backward(c(d_logp), xg, tokens.cuda(), c(lse), d_entropy=c(d_entropy), entropy=c(entropy) if d_entropy is not None else None, d_lse=c(d_lse),
                                     out=xg if out else None)
    torch.cuda.synchronize()
    assert got.dtype == x.dtype and got.shape == x.shape
    info = torch.finfo(x.dtype)
    fine = same_where_special(got.cpu(), want)
    off = (got.cpu().double() - want).abs()
    limit = bound + info.eps / 2 * (want.abs() + bound) + info.tiny * info.eps
    assert (off <= limit)[fine].all(), (off[fine].max(), (off / limit)[fine].max())
    return got


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_backward(P, rows, cols, dtype):
    announce("token_log_probs_backward %s" % ((rows, cols, dtype),))
    x, t = logits(rows, cols, dtype, seed=4)
    t[rows // 2:rows // 2 + 1] = cols
    check_backward(P, x, t, ("logp",))
    check_backward(P, x, t, ("logp", "entropy", "lse"), out=True)


@pytest.mark.parametrize("which", [("logp",), ("entropy",), ("lse",), ("logp", "lse"), ("entropy", "lse")])
def test_backward_of_each(P, which):
    announce("token_log_probs_backward of %s" % (which,))
    for rows, cols in ((5, 40), (3, 700), (2, 9001)):
        check_backward(P, *logits(rows, cols, "f32", seed=6), which)


def test_backward_of_nothing_is_zeros(P):
    announce("token_log_probs_backward of nothing")
    x, t = logits(3, 100, "f32")
    assert (P.token_log_probs_backward(None, x.cuda(), t.cuda(), torch.zeros(3).cuda()).cpu() == 0).all()


@pytest.mark.parametrize("cols", [40, 9001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_backward_of_special_rows(P, cols, dtype):
    announce("token_log_probs_backward special rows %s" % ((cols, dtype),))
    x, t = logits(6, cols, dtype, seed=7)
    x[0] = -INF
    x[1, 1:] = -INF
    x[2, ::2] = -INF
    x[3] = torch.finfo(x.dtype).min
    t[:4] = torch.tensor([0, 0, 2, 1], dtype=torch.int32)      # (row 2's token is masked)
    got = check_backward(P, x, t, ("logp", "entropy", "lse")).cpu()
    assert (got[0] == 0).all()


@pytest.mark.parametrize("entropy", [False, True])
def test_gradient_is_that_of_differences(P, entropy):
    """d/dx of sum(a logp) + sum(b H) + sum(c lse) along a direction, from the definitions at both sides."""
    announce("token_log_probs_backward differences")
    x, t = logits(4, 300, "f32", seed=8)
    t[1] = -1
    g = torch.Generator().manual_seed(9)
    a, b, c = (torch.randn(4, generator=g) for _ in range(3))
    v = torch.randn((4, 300), generator=g).double()

    def loss(z):
        logp, h, lse, _ = exact(z, t)
        return (a * logp).sum() + (c * lse).sum() + ((b * h).sum() if entropy else 0)

    step = 1e-5
    want = (loss(x.double() + step * v) - loss(x.double() - step * v)) / (2 * step)
    _, h, lse = P.token_log_probs(x.cuda(), t.cuda(), want_entropy=True, want_lse=True)
    got = P.token_log_probs_backward(a.cuda(), x.cuda(), t.cuda(), lse, d_entropy=b.cuda() if entropy else None, entropy=h if entropy else None, d_lse=c.cuda())
    along = (got.cpu().double() * v).sum()
    # the differences are off by step^2 of a third derivative below 100, the gradient by its bound, some 2e-6 of 300 entries of each row
    assert abs(along - want) <= 1e-8 * 100 + 2e-5 * (1 + abs(want)), (along, want)


# ---- as they are used ----

def test_rows_behind_four_gib(P):
    announce("token_log_probs past 2^31 elements")
    rows, cols = 70000, 32003
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    last, t = logits(2, cols, "bf16", seed=10)
    x[-2:] = last.cuda()
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    tokens[-2:] = t.cuda()
    logp, entropy, lse, values, ids = P.token_log_probs(x, tokens, top=4, want_entropy=True, want_lse=True)
    want_logp, want_entropy, want_lse, p = exact(last, t)
    of_lse, of_entropy = bounds(last, want_lse, p)
    assert ((logp[-2:].cpu() - want_logp).abs() <= of_lse + 2 * U * want_logp.abs()).all() and ((entropy[-2:].cpu() - want_entropy).abs() <= 2 * of_entropy).all()
    check_top(last, values[-2:].cpu(), ids[-2:].cpu(), 4, of_lse)
    d = torch.zeros(rows, device="cuda")
    d[-2:] = 1.0
    grad = P.token_log_probs_backward(d, x, tokens, lse, out=x)
    want, bound = exact_backward(last, t, want_lse.float(), torch.ones(2), None, None, None)
    assert ((grad[-2:].cpu().double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound) + 4 * U).all()
    assert (grad[:-2].abs().amax() == 0).item()


def test_repeats_bit_for_bit_and_on_two_streams(P):
    announce("token_log_probs two streams")
    x, t = logits(8, 40000, "bf16", seed=11)
    x, t = x.cuda(), t.cuda()
    first = P.token_log_probs(x, t, top=20, want_entropy=True, want_lse=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            got.append(P.token_log_probs(x, t, top=20, want_entropy=True, want_lse=True))
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, first))


def test_captured_and_replayed(P):
    announce("token_log_probs graph")
    x, t = logits(4, 33000, "f32", seed=12)
    x, t = x.cuda(), t.cuda()
    d = torch.ones(4, device="cuda")

    def step():
        out = P.token_log_probs(x, t, top=5, want_entropy=True, want_lse=True)
        return (*out, P.token_log_probs_backward(d, x, t, out[2], d_entropy=d, entropy=out[1]))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        x.copy_(logits(4, 33000, "f32", seed=20 + k)[0])
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), k


def test_recorded_calls_are_those_of_python(P):
    """Calls that the extension does as a whole, and the Python functions' own way, which a recording takes."""
    from ml import _lib
    announce("token_log_probs recorded")
    x, t = logits(3, 9000, "f16", seed=13)
    x, t = x.cuda(), t.cuda()
    d = torch.ones(3, device="cuda")
    whole = P.token_log_probs(x, t, top=5, want_entropy=True, want_lse=True)
    grad = P.token_log_probs_backward(d, x, t, whole[2])
    tape = _lib.start_tape()
    try:
        own = P.token_log_probs(x, t, top=5, want_entropy=True, want_lse=True)
        own_grad = P.token_log_probs_backward(d, x, t, own[2])
    finally:
        _lib.stop_tape()
    assert len(tape.calls) == 2 and all(torch.equal(a, b) for a, b in zip(whole, own)) and torch.equal(grad, own_grad)
    for v in own:
        v.zero_()
    tape.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(whole, own))


def test_penalised_logits_to_log_probabilities(P):
    """A decoding step: penalties and a mask, the token, its log probability and the alternatives, all of the same logits."""
    announce("penalize_logits, then token_log_probs")
    x, _ = logits(3, 20011, "bf16", seed=14)
    g = torch.Generator().manual_seed(15)
    mask = torch.randint(-2 ** 31, 2 ** 31, (3, -(-20011 // 32)), generator=g).int()
    mask[2] = 0
    out, token = P.penalize_logits(x.cuda(), temperature=torch.full((3,), 0.7).cuda(), mask=mask.cuda(), want_token=True)
    logp, values, ids = P.token_log_probs(out, token, top=3)
    torch.cuda.synchronize()
    assert torch.equal(ids[:, 0], token) and torch.equal(values[:2, 0], logp[:2])
    assert token[2].item() == -1 and logp[2].item() == 0 and ids[2].tolist() == [-1] * 3 and (values[2] == -INF).all()
    want = exact(out.cpu(), token.cpu())[0]
    assert ((logp.cpu() - want).abs() <= 1e-4).all()
