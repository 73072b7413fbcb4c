"""The calls that the extension makes as a whole (csrc/host.cpp) against the same calls as the Python functions make them step by step -- recording a tape takes
that way -- and what neither takes."""
import pytest
import torch

from gpu_util import announce

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn


def calls():
    from ml import matmul as M, primitives as P
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    i = lambda most, *s: torch.randint(0, most, s, generator=g, device="cuda", dtype=torch.int32)
    x, w, b = r(6, 40, 200), r(200), r(200)
    y, mean, rstd = P.layer_norm(x, w, want_stats=True)
    a8, sa = M.quantize_blocks(r(70, 272))
    b8, sb = M.quantize_blocks(r(130, 272), (128, 128))
    c8, sc = M.quantize_blocks(r(130, 272), dtype=torch.float8_e5m2)
    logits, tokens, each = r(3, 9000), i(9000, 3, 50), torch.rand((3,), generator=g, device="cuda") + 0.5
    return {
        "norm": lambda: P.layer_norm(x),
        "norm weights": lambda: P.layer_norm(x, w, b, 1e-3, want_stats=True),
        "norm bias": lambda: P.layer_norm(x.bfloat16(), None, b.bfloat16()),
        "norm 16 bits": lambda: P.layer_norm(x.half(), w, b),
        "backward": lambda: P.layer_norm_backward(x, x, mean, rstd),
        "backward weights": lambda: P.layer_norm_backward(x.bfloat16(), x.bfloat16(), mean, rstd, w.bfloat16()),
        "quantize": lambda: M.quantize_blocks(x[0]),
        "quantize transposed": lambda: M.quantize_blocks(x[0].half(), (128, 128), torch.float8_e5m2, True),
        "quantize both": lambda: M.quantize_blocks(x[0].bfloat16(), transpose="both"),
        "product": lambda: M.matmul_abt_scaled(a8, sa, b8, sb),
        "product bias": lambda: M.matmul_abt_scaled(a8, sa, c8, sc, bias=r(130).zero_() + 1, relu=True, out_dtype=torch.bfloat16),
        "logits": lambda: P.penalize_logits(logits),
        "logits everything": lambda: P.penalize_logits(logits.half(), tokens, i(50, 3).zero_() + 40, i(50, 3).zero_() + 9, each, each, each, each, i(9000, 3, 7).zero_(), r(3, 7).zero_() + 2,
                                                       i(2 ** 31 - 1, 3, 282).zero_() + 0x5a5a5a5a, want_token=True),
        "logits empty": lambda: P.penalize_logits(logits, tokens[:, :0].contiguous(), bias_ids=tokens[:, :0].contiguous(), bias=logits[:, :0].contiguous(), want_token=True),
    }


@pytest.mark.parametrize("name", ["norm", "norm weights", "norm bias", "norm 16 bits", "backward", "backward weights", "quantize", "quantize transposed", "quantize both", "product",
                                  "product bias", "logits", "logits everything", "logits empty"])
def test_whole_and_step_by_step(name):
    from ml import _lib
    announce("whole call: " + name)
    f = calls()[name]
    flat = lambda r: [t.view(torch.uint8) for t in (r if isinstance(r, tuple) else (r,))]
    shapes = lambda r: [(t.shape, t.dtype) for t in (r if isinstance(r, tuple) else (r,))]
    whole = f()
    tape = _lib.start_tape()
    try:
        steps = f()
    finally:
        _lib.stop_tape()
    assert len(tape.calls) == 1 and shapes(whole) == shapes(steps)
    assert all(torch.equal(p, q) for p, q in zip(flat(whole), flat(steps)))
    kept = [t.clone() for t in flat(steps)]
    for t in flat(steps):
        t.zero_()
    tape.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(flat(steps), kept))


def test_what_is_not_taken_raises():
    from ml import matmul as M, primitives as P
    announce("whole calls: refusals")
    x, w = torch.randn((4, 64), device="cuda"), torch.randn((64,), device="cuda")
    a8, sa = M.quantize_blocks(x)
    stats = torch.zeros((4,), device="cuda")
    for error, text, f in ((ValueError, "contiguous", lambda: P.layer_norm(x.t())), (ValueError, "GPU", lambda: P.layer_norm(x, w.cpu())), (ValueError, "weight must", lambda: P.layer_norm(x, w[:3])),
                           (TypeError, "f32, f16", lambda: P.layer_norm(x.double())), (RuntimeError, "16384", lambda: P.layer_norm(torch.zeros((1, 16385), device="cuda"))),
                           (RuntimeError, "eps", lambda: P.layer_norm(x, eps=-1.0)), (RuntimeError, "NULL", lambda: P.layer_norm(x[:0])), (RuntimeError, "16-byte", lambda: P.layer_norm(x.view(-1)[1:].view(3, 85))),
                           (ValueError, "dy must", lambda: P.layer_norm_backward(x.half(), x, stats, stats)), (TypeError, "mean must have dtype", lambda: P.layer_norm_backward(x, x, stats.half(), stats)),
                           (ValueError, "contiguous", lambda: M.quantize_blocks(x.t())), (ValueError, "block", lambda: M.quantize_blocks(x, (64, 64))), (ValueError, "empty", lambda: M.quantize_blocks(x[:, :0])),
                           (AssertionError, "K dimension", lambda: M.matmul_abt_scaled(a8, sa, a8.view(torch.uint8)[:, :32].contiguous().view(F8), sa)),
                           (TypeError, "dtype", lambda: M.matmul_abt_scaled(a8, sa.half(), a8, sa)), (RuntimeError, "multiple of 16", lambda: M.matmul_abt_scaled(
                               *2 * (a8.view(torch.uint8)[:, :40].contiguous().view(F8), sa))), (TypeError, "C must", lambda: M.matmul_abt_scaled(a8, sa, a8, sa, out_dtype=torch.float64)),
                           (TypeError, "tokens must have dtype", lambda: P.penalize_logits(x, tokens=torch.zeros((4, 3), device="cuda", dtype=torch.int64))),
                           (ValueError, "one entry", lambda: P.penalize_logits(x, repetition=stats[:2])), (ValueError, "need tokens", lambda: P.penalize_logits(x, lengths=torch.zeros((4,), device="cuda", dtype=torch.int32)))):
        with pytest.raises(error, match=text):
            f()
    assert torch.equal(P.layer_norm(x, eps=1), P.layer_norm(x, eps=1.0))          # (an integer goes the long way)
    for mask in (torch.full((4, 2), -1, device="cuda", dtype=torch.int32), torch.full((2, 2, 3), -1, device="cuda", dtype=torch.int32)):      # (rows in another shape than the logits')
        with pytest.raises(ValueError, match="mask must"):
            P.penalize_logits(x.view(2, 2, 64), mask=mask)


def test_a_transpose_of_0_or_1_is_false_or_true():
    from ml import matmul as M
    announce("quantize_blocks transpose=0, 1")
    x = torch.randn((40, 200), device="cuda")
    for flag in (0, 1):
        for got, want in zip(M.quantize_blocks(x, transpose=flag), M.quantize_blocks(x, transpose=bool(flag)), strict=True):
            assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


def test_gradients_are_not_asked_of_the_outputs():
    from ml import primitives as P
    announce("whole calls: requires_grad")
    x = torch.randn((4, 64), device="cuda", requires_grad=True)
    assert not P.layer_norm(x).requires_grad
