"""Penalties, biases, temperature and masks on logits, on the GPU against the same steps on the CPU: every step is a single f32 operation,
so values are equal, bit for bit, and so are the tokens chosen."""
import math

import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def P():
    from ml import primitives
    return primitives


def plain(logits, tokens=None, lengths=None, prompt_lengths=None, repetition=None, presence=None, frequency=None, temperature=None,
          bias_ids=None, bias=None, mask=None):
    """Row by row in f32 on the CPU; numbers of a token once each, biases in their order."""
    x = logits.float().clone()
    rows, cols = x.shape
    chosen = torch.full((rows,), -1, dtype=torch.int32)
    for r in range(rows):
        if tokens is not None:
            n = tokens.shape[1] if lengths is None else max(0, min(int(lengths[r]), tokens.shape[1]))
            p = 0 if prompt_lengths is None else max(0, min(int(prompt_lengths[r]), n))
            valid = lambda t: t[(t >= 0) & (t < cols)].long()
            seen = torch.bincount(valid(tokens[r, :n]), minlength=cols) > 0
            count = torch.bincount(valid(tokens[r, p:n]), minlength=cols)
            if repetition is not None:
                x[r] = torch.where(seen, torch.where(x[r] > 0, x[r] / repetition[r], x[r] * repetition[r]), x[r])
            if frequency is not None:
                x[r] = torch.where(count > 0, x[r] - frequency[r] * count.float(), x[r])
            if presence is not None:
                x[r] = torch.where(count > 0, x[r] - presence[r], x[r])
        if bias is not None:
            sums = {}
            for j, b in zip(bias_ids[r].tolist(), bias[r]):
                if 0 <= j < cols:
                    sums[j] = sums[j] + b if j in sums else b
            for j, b in sums.items():
                x[r, j] = x[r, j] + b
        if temperature is not None and float(temperature[r]) > 0:
            x[r] = x[r] / temperature[r]
        if mask is not None:
            words = mask.reshape(-1, mask.shape[-1])[r if mask.numel() > mask.shape[-1] else 0]
            j = torch.arange(cols)
            x[r] = torch.where((words[j // 32].long() >> (j % 32)) & 1 != 0, x[r], -math.inf)
        v = x[r].nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        best = v.max()
        if best > -math.inf:
            chosen[r] = int((v == best).nonzero()[0])
    return x, chosen


def inputs(rows, cols, history, n_bias, seed, dtype="f32"):
    g = torch.Generator().manual_seed(seed)
    u = lambda *shape: torch.rand(shape, generator=g)
    kw = dict(repetition=u(rows) + 0.75, presence=u(rows) - 0.25, frequency=u(rows) * 0.3, temperature=u(rows) * 2,
              mask=torch.randint(-2 ** 31, 2 ** 31, (rows, -(-cols // 32)), generator=g).int())
    if history:
        kw["tokens"] = (u(rows, history) ** 3 * cols).int().clamp(max=cols - 1)
        kw["lengths"] = (u(rows) * (history + 2)).int()        # some at zero, some past the end
        kw["prompt_lengths"] = (u(rows) * history).int() - 1
        kw["tokens"][:, ::7] = -1
        kw["tokens"][:, 3::11] = cols + 5
    if n_bias:
        kw["bias_ids"] = (u(rows, n_bias) * cols).int().clamp(max=cols - 1)
        kw["bias"] = torch.randn((rows, n_bias), generator=g)
        kw["bias_ids"][:, ::5] = -1
    return (torch.randn((rows, cols), generator=g) * 3).to(TYPES[dtype]), kw


def check(P, logits, kw, **more):
    got, token = P.penalize_logits(logits.cuda(), **{k: v.cuda() for k, v in kw.items()}, want_token=True, **more)
    torch.cuda.synchronize()
    want, chosen = plain(logits, **kw)
    got = got.cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    assert same.all(), (got[~same][:4], want[~same][:4], int((~same).sum()))
    assert torch.equal(token.cpu(), chosen)


# one column, ends inside a piece, a word of the mask and a chunk; several chunks
@pytest.mark.parametrize("rows,cols,history,n_bias", [(1, 1, 3, 1), (3, 2, 5, 2), (5, 31, 40, 3), (4, 33, 0, 0), (2, 1000, 100, 20), (7, 1003, 1, 0), (3, 8192, 2000, 300),
                                                      (2, 8193, 513, 7), (1, 32003, 2001, 16), (3, 50257, 700, 2047), (2, 131072, 4096, 64), (300, 96, 9, 4)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_everything_at_once(P, rows, cols, history, n_bias, dtype):
    announce("penalize_logits %s" % ((rows, cols, history, n_bias, dtype),))
    check(P, *inputs(rows, cols, history, n_bias, 1, dtype))


@pytest.mark.parametrize("leave", ["repetition", "presence", "frequency", "temperature", "mask", "lengths", "prompt_lengths", "tokens", "bias"])
def test_each_step_can_be_left_out(P, leave):
    announce("penalize_logits without " + leave)
    x, kw = inputs(3, 9001, 300, 40, 2)
    gone = {"tokens": ("tokens", "lengths", "prompt_lengths"), "bias": ("bias", "bias_ids")}.get(leave, (leave,))
    check(P, x, {k: v for k, v in kw.items() if k not in gone})


@pytest.mark.parametrize("only", ["repetition", "presence", "frequency", "temperature", "mask", "bias", "nothing"])
def test_each_step_alone(P, only):
    announce("penalize_logits only " + only)
    x, kw = inputs(3, 777, 200, 40, 3)
    keep = {"repetition": ("tokens", "lengths", "repetition"), "presence": ("tokens", "presence"), "frequency": ("tokens", "prompt_lengths", "frequency"),
            "bias": ("bias", "bias_ids"), "nothing": ()}.get(only, (only,))
    check(P, x, {k: v for k, v in kw.items() if k in keep})


def test_masks_that_leave_little_or_nothing(P):
    announce("penalize_logits masks")
    x, kw = inputs(4, 20000, 50, 5, 4)
    kw["mask"].zero_()
    kw["mask"][1, 624] = -2 ** 31                       # the last column of all
    kw["mask"][2, 0] = 1
    check(P, x, kw)
    kw["mask"] = kw["mask"][1].clone()                  # one row for all
    check(P, x, kw)
    kw["mask"] = kw["mask"].view(1, -1)
    check(P, x, kw)


def test_infinities_nans_and_the_lowest_number(P):
    announce("penalize_logits infinities")
    x, kw = inputs(8, 9000, 100, 10, 5)
    x[0] = -math.inf
    x[1] = float("nan")
    x[2, ::3] = float("nan")
    x[3, 8999] = math.inf
    x[4] = torch.finfo(torch.float32).min
    x[5] = -0.0
    x[6, 17] = math.inf
    x[7, 100:] = -math.inf
    kw["mask"].fill_(-1)
    kw["mask"][6, 0] = ~(1 << 17)                       # an infinity in a masked place
    check(P, x, kw)
    kw["mask"][2] = 0x49249249                          # and NaNs
    check(P, x, kw)


def test_equal_logits_give_the_lowest_index(P):
    announce("penalize_logits ties")
    for cols in (5, 640, 8191, 30001):
        x = torch.zeros((3, cols))
        x[1, cols // 2:] = 1
        x[2, -1] = 1
        _, token = P.penalize_logits(x.cuda(), want_token=True)
        assert token.tolist() == [0, cols // 2, cols - 1]


def test_a_bias_given_twice_and_a_history_of_one_token(P):
    announce("penalize_logits duplicates")
    x, kw = inputs(3, 500, 3000, 60, 6)
    kw["bias_ids"][:, 10:] = 77                         # fifty times, in their order
    kw["tokens"].fill_(77)
    kw["lengths"].fill_(3000)
    check(P, x, kw)
    kw["lengths"] = torch.tensor([0, 1, -5], dtype=torch.int32)
    check(P, x, kw)


def test_a_history_longer_than_a_row(P):
    announce("penalize_logits long history")
    x, kw = inputs(2, 300, 100001, 0, 7)
    check(P, x, kw)


def test_temperatures_of_zero_leave_a_row_as_it_is(P):
    announce("penalize_logits temperature")
    x, kw = inputs(5, 400, 0, 0, 8)
    kw["temperature"] = torch.tensor([0.0, -1.0, float("nan"), 1e-30, 3.0])
    check(P, x, kw)


def test_in_place_and_leading_dimensions(P):
    announce("penalize_logits in place")
    x, kw = inputs(6, 8300, 30, 4, 9)
    want, chosen = plain(x, **kw)
    d = {k: v.cuda().view(2, 3, *v.shape[1:]) for k, v in kw.items()}
    y = x.cuda().view(2, 3, 8300)
    out, token = P.penalize_logits(y, **d, out=y, want_token=True)
    assert out is y and torch.equal(y.cpu().view(6, -1), want) and token.shape == (2, 3) and torch.equal(token.cpu().view(-1), chosen)


def test_captured_and_on_another_stream(P):
    announce("penalize_logits captured")
    x, kw = inputs(3, 20001, 60, 8, 10)
    x, kw = x.cuda(), {k: v.cuda() for k, v in kw.items()}
    want = P.penalize_logits(x, **kw, want_token=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = P.penalize_logits(x, **kw, want_token=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, other))
    graphs, kept = [], []
    for _ in range(2):                                  # two graphs, replayed one after the other: nothing of theirs is shared
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            kept.append(P.penalize_logits(x, **kw, want_token=True))
    for k in range(3):
        x.normal_()
        kw["tokens"].random_(0, 20001)
        for graph in graphs:
            graph.replay()
        want = P.penalize_logits(x, **kw, want_token=True)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for got in kept for p, q in zip(want, got)), k


@pytest.mark.parametrize("rows,cols,history", [(40, 32003, 900), (129, 8191, 0), (300, 33001, 4097)])       # (large chunks; the last results are streamed)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_many_rows_of_several_chunks(P, rows, cols, history, dtype):
    announce("penalize_logits %s" % ((rows, cols, history, dtype),))
    check(P, *inputs(rows, cols, history, 5, 3, dtype))


def test_offsets_past_32_bits(P):
    """More than 2^31 logits: the last rows are those of a call on them alone."""
    announce("penalize_logits 16400 x 131072 bf16")
    rows, cols = 16400, 131072
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    x[-3:].normal_()
    tokens = torch.randint(0, cols, (rows, 50), device="cuda", dtype=torch.int32)
    penalty = torch.full((rows,), 1.5, device="cuda")
    out, token = P.penalize_logits(x, tokens=tokens, repetition=penalty, presence=penalty, want_token=True)
    want = P.penalize_logits(x[-3:].clone(), tokens=tokens[-3:].clone(), repetition=penalty[-3:].clone(), presence=penalty[-3:].clone(), want_token=True)
    assert torch.equal(out[-3:], want[0]) and torch.equal(token[-3:], want[1])


def test_from_a_hidden_state_to_a_token(P):
    """norm -> 8-bit product with the vocabulary's weights -> penalties and mask -> the framework's own sampling, for a batch and for its
    last row alone: the chain of calls that a decoding step makes, eager and captured."""
    from ml import matmul
    announce("norm, product, logits, sample")
    g = torch.Generator(device="cuda").manual_seed(11)
    rows, width, vocabulary = 5, 528, 1000
    h = torch.randn((rows, width), generator=g, device="cuda").bfloat16()
    w = torch.randn((width,), generator=g, device="cuda").bfloat16()
    head = torch.randn((vocabulary, width), generator=g, device="cuda")
    head8, head_scale = matmul.quantize_blocks(head, (128, 128))
    tokens = torch.randint(0, vocabulary, (rows, 12), generator=g, device="cuda", dtype=torch.int32)
    penalty = torch.rand((rows,), generator=g, device="cuda") + 1
    mask = torch.randint(-2 ** 31, 2 ** 31, (rows, 32), generator=g, device="cuda", dtype=torch.int64).int()
    u = torch.rand((rows,), generator=g, device="cuda").clamp_(min=1e-6)

    def step(pick=slice(None)):
        n = P.layer_norm(h[pick], w)
        n8, s = matmul.quantize_blocks(n)
        logits = matmul.matmul_abt_scaled(n8, s, head8, head_scale)
        out, token = P.penalize_logits(logits, tokens=tokens[pick], repetition=penalty[pick], presence=penalty[pick], mask=mask[pick], want_token=True)
        probs, sample = P.softmax_and_discrete_sampling(out, u[pick])
        return n, logits, out, token, probs, sample
    n, logits, out, token, probs, sample = step()
    # against the plain chain; the norm's output is taken as it is, the 8-bit steps are bounded as in a layer (2^-4 and 2^-10 of the largest)
    nd, hd = n.double(), head.double()
    off = lambda v: v.abs() * 2.0 ** -4 + v.abs().max() / 448 * 2.0 ** -10
    bound = off(nd) @ hd.abs().t() + nd.abs() @ off(hd).t() + off(nd) @ off(hd).t()
    assert ((logits.double() - nd @ hd.t()).abs() <= bound * 1.001).all()
    want, chosen = plain(logits.cpu(), tokens=tokens.cpu(), repetition=penalty.cpu(), presence=penalty.cpu(), mask=mask.cpu())
    assert torch.equal(out.cpu(), want) and torch.equal(token.cpu(), chosen) and torch.equal(P.argmax(out).int(), token)
    assert (probs[out == -math.inf] == 0).all() and (out.gather(1, sample.long()[:, None]) > -math.inf).all()
    # a row alone takes the same kernels here: the same bits
    one = step(slice(rows - 1, rows))
    assert all(torch.equal(p[-1:], q) for p, q in zip((n, logits, out, token, probs, sample), one))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for k in range(3):
        h.normal_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, kept)), k


@pytest.mark.parametrize("rows,cols", [(1, 32003), (3, 2100), (40, 32003), (2, 9000)])
@pytest.mark.parametrize("kind", ["padding", "pairs", "runs", "few", "all", "one"])
def test_biases_of_ids_that_repeat(P, rows, cols, kind):
    """Their sum in their order: numbers of which most orders round differently."""
    for n in (2, 64, 65, 300, 2047):
        announce("penalize_logits repeated ids %s" % ((rows, cols, kind, n),))
        g = torch.Generator().manual_seed(12)
        ids = torch.stack([torch.randperm(cols, generator=g)[:n] if n <= cols else torch.randint(0, cols, (n,), generator=g) for _ in range(rows)])
        if kind == "padding":
            ids[:, n // 2:] = ids[:, :1]
        elif kind == "pairs":
            ids[:, n // 2:n // 2 * 2] = ids[:, :n // 2].flip(1)
        elif kind == "runs":
            ids = ids.sort(1).values // 7 * 7
        elif kind == "few":
            ids = ids % 5 * (cols // 5)
        elif kind == "all":
            ids[:] = cols - 1
        else:
            ids[:, -1] = ids[:, 0]
        kw = dict(bias_ids=ids.int(), bias=torch.randn((rows, n), generator=g) * torch.exp2(torch.randint(-12, 13, (rows, n), generator=g).float()))
        kw["bias_ids"][:, 1::9] = -1
        check(P, torch.randn((rows, cols), generator=g), kw)
