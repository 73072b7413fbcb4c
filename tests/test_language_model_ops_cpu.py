"""What layer norm, the 8-bit products and the penalties on logits refuse, without a GPU: in Python by shape and type, at the C entry points by pointer, type and
size, before any device work."""
import ctypes as C

import pytest
import torch

F8 = torch.float8_e4m3fn
P = C.c_void_p(0x1000)
ODD = C.c_void_p(0x1004)


@pytest.fixture(scope="module")
def L():
    from ml import _lib
    return _lib


def call(L, name, order, good, **kw):
    rc = getattr(L.lib, name)(*[kw.get(k, good[k]) for k in order.split()], None)
    return rc, L.lib.sp_last_error_string().decode()


def test_layer_norm_refusals(L):
    order = "dtype wdtype x weight bias y mean rstd rows cols eps"
    good = dict(dtype=2, wdtype=0, x=P, weight=P, bias=P, y=P, mean=P, rstd=P, rows=4, cols=64, eps=1e-5)
    for kw, code, text in ((dict(x=None), -1, "x is NULL"), (dict(y=None), -1, "y is NULL"), (dict(weight=ODD), -3, "16-byte"), (dict(mean=ODD), -3, "16-byte"),
                           (dict(dtype=7), -4, "dtype"), (dict(wdtype=1), -4, "weights"), (dict(rows=0), -2, "positive"), (dict(cols=0), -2, "positive"),
                           (dict(cols=16385), -2, "16384"), (dict(rows=1 << 41), -2, "too large"), (dict(eps=-1.0), -5, "eps"), (dict(eps=float("nan")), -5, "eps"),
                           (dict(eps=float("inf")), -5, "eps")):
        rc, said = call(L, "sp_layer_norm", order, good, **kw)
        assert rc == code and text in said, (kw, rc, said)


def test_layer_norm_backward_refusals(L):
    order = "dtype wdtype dy x mean rstd weight dx dw db rows cols ws bytes"
    need = L.lib.sp_layer_norm_backward_workspace_bytes(4, 64)
    assert need == 4 * 2 * 64 * 4 and L.lib.sp_layer_norm_backward_workspace_bytes(1 << 20, 64) <= 1024 * 2 * 64 * 4
    assert L.lib.sp_layer_norm_backward_workspace_bytes(0, 64) == 0 and L.lib.sp_layer_norm_backward_workspace_bytes(4, 16385) == 0
    good = dict(dtype=2, wdtype=0, dy=P, x=P, mean=P, rstd=P, weight=P, dx=P, dw=P, db=P, rows=4, cols=64, ws=P, bytes=need)
    for kw, code, text in ((dict(dy=None), -1, "dy"), (dict(mean=None), -1, "mean"), (dict(rstd=None), -1, "rstd"), (dict(dx=None), -1, "dx"), (dict(dx=ODD), -3, "16-byte"),
                           (dict(dw=None), -5, "both"), (dict(ws=None), -1, "workspace"), (dict(bytes=need - 1), -5, "workspace"), (dict(dtype=0, wdtype=2), -4, "weights"),
                           (dict(cols=20000), -2, "16384")):
        rc, said = call(L, "sp_layer_norm_backward", order, good, **kw)
        assert rc == code and text in said, (kw, rc, said)


def test_quantize_refusals(L):
    order = "dtype f8 high x q s qt st rows cols"
    good = dict(dtype=2, f8=8, high=1, x=P, q=P, s=P, qt=None, st=None, rows=4, cols=64)
    for kw, code, text in ((dict(x=None), -1, "x is NULL"), (dict(q=None, s=None), -1, "q and q_t"), (dict(s=None), -1, "go together"), (dict(qt=P), -1, "go together"),
                           (dict(q=ODD), -3, "16-byte"), (dict(dtype=8), -4, "dtype"), (dict(f8=0), -4, "f8"), (dict(high=64), -5, "1 or 128"), (dict(rows=0), -2, "positive"),
                           (dict(rows=(1 << 31) + 1), -2, "too large")):
        rc, said = call(L, "sp_quantize_blocks", order, good, **kw)
        assert rc == code and text in said, (kw, rc, said)


def test_scaled_product_refusals(L):
    order = "fa fb out a sa b sb high c bias m n k beta flags"
    good = dict(fa=8, fb=9, out=0, a=P, sa=P, b=P, sb=P, high=128, c=P, bias=None, m=4, n=64, k=64, beta=0.0, flags=0)
    for kw, code, text in ((dict(a=None), -1, "A is NULL"), (dict(sb=None), -1, "scale_b"), (dict(c=ODD), -3, "16-byte"), (dict(bias=ODD), -3, "16-byte"), (dict(fa=2), -4, "e4m3"),
                           (dict(out=8), -4, "C must"), (dict(high=2), -5, "1 or 128"), (dict(flags=0x100), -5, "flags"), (dict(m=0), -2, "positive"), (dict(k=0), -2, "positive"),
                           (dict(k=72), -2, "multiple of 16"), (dict(k=(1 << 23) + 16), -2, "too large"), (dict(m=1 << 31), -2, "too large")):
        rc, said = call(L, "sp_gemm_abt_scaled", order, good, **kw)
        assert rc == code and text in said, (kw, rc, said)


def test_logits_refusals(L):
    order = "dtype x out token tokens lengths prompts history rep pres freq temp ids bias n mask mask_rows rows cols ws bytes"
    need = L.lib.sp_logits_penalize_workspace_bytes(4, 100000)
    assert need >= 4 * 8 and L.lib.sp_logits_penalize_workspace_bytes(0, 5) == 0
    good = dict(dtype=2, x=P, out=C.c_void_p(0x2000), token=P, tokens=P, lengths=P, prompts=P, history=5, rep=P, pres=P, freq=P, temp=P, ids=P, bias=P, n=3, mask=P, mask_rows=4,
                rows=4, cols=100000, ws=P, bytes=need)
    for kw, code, text in ((dict(x=None), -1, "logits"), (dict(out=None), -1, "out"), (dict(temp=ODD), -3, "16-byte"), (dict(dtype=9), -4, "dtype"), (dict(rows=0), -2, "positive"),
                           (dict(cols=1 << 31), -2, "too large"), (dict(rows=1 << 30), -2, "too large"), (dict(out=P), -5, "overwritten"), (dict(history=1 << 20), -2, "history"),
                           (dict(history=-1), -2, "history"), (dict(n=2048), -2, "n_bias"), (dict(tokens=None), -1, "tokens"), (dict(bias=None), -1, "go together"),
                           (dict(mask_rows=3), -2, "mask_rows"), (dict(ws=None), -1, "workspace"), (dict(bytes=need - 1), -5, "workspace")):
        rc, said = call(L, "sp_logits_penalize", order, good, **kw)
        assert rc == code and text in said, (kw, rc, said)


def test_python_refusals():
    from ml import matmul, primitives
    x, w = torch.zeros((4, 64)), torch.zeros(64)
    stat = torch.zeros(4)
    a, sa = torch.zeros((4, 64)).to(F8), torch.zeros((4, 1))
    b, sb = torch.zeros((200, 64)).to(F8), torch.zeros((2, 1))
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    N, Bk, Q, G, Lo = primitives.layer_norm, primitives.layer_norm_backward, matmul.quantize_blocks, matmul.matmul_abt_scaled, primitives.penalize_logits
    for error, text, f in (
            (TypeError, "f32, f16 or bf16", lambda: N(x.double())), (ValueError, "2 dimensions", lambda: N(w)), (ValueError, "weight must be", lambda: N(x, w[:5])),
            (TypeError, "weight must be", lambda: N(x, w.half())), (TypeError, "one dtype", lambda: N(x.half(), w.half(), w)), (ValueError, "out must", lambda: N(x, out=x.half())),
            (ValueError, "GPU", lambda: N(x)), (ValueError, "GPU", lambda: N(x, w)), (ValueError, "dy must", lambda: Bk(x[:2], x, stat, stat)), (ValueError, "one entry", lambda: Bk(x, x, stat[:2], stat)),
            (ValueError, "GPU", lambda: Bk(x, x, stat, stat)),
            (ValueError, "2-D", lambda: Q(w)), (TypeError, "f32, f16 or bf16", lambda: Q(x.double())), (TypeError, "float8", lambda: Q(x, dtype=torch.float16)),
            (ValueError, "block must", lambda: Q(x, (1, 64))), (ValueError, "transpose", lambda: Q(x, transpose="yes")), (ValueError, "empty", lambda: Q(x[:0])), (ValueError, "GPU", lambda: Q(x)),
            (ValueError, "2-D", lambda: G(a, stat, b, sb)), (TypeError, "float8", lambda: G(x, sa, b, sb)), (AssertionError, "K dimension", lambda: G(a[:, :32], sa, b, sb)),
            (ValueError, "scale_a", lambda: G(a, sa[:3], b, sb)), (ValueError, "scale_b", lambda: G(a, sa, b, sb[:1])), (AssertionError, "beta", lambda: G(a, sa, b, sb, beta=1.0)),
            (AssertionError, "C tensor", lambda: G(a, sa, b, sb, c=x)), (TypeError, "out_dtype", lambda: G(a, sa, b, sb, c=torch.zeros((4, 200)), out_dtype=torch.float16)),
            (TypeError, "C must", lambda: G(a, sa, b, sb, out_dtype=torch.float64)), (ValueError, "bias", lambda: G(a, sa, b, sb, bias=w)), (ValueError, "GPU", lambda: G(a, sa, b, sb)),
            (TypeError, "logits", lambda: Lo(x.double())), (ValueError, "out must", lambda: Lo(x, out=x[:2])), (ValueError, "one entry", lambda: Lo(x, repetition=stat[:2])),
            (ValueError, "tokens must", lambda: Lo(x, tokens=i32(3, 5))), (ValueError, "need tokens", lambda: Lo(x, lengths=i32(4))), (ValueError, "go together", lambda: Lo(x, bias=x)),
            (ValueError, "bias_ids and bias", lambda: Lo(x, bias=x, bias_ids=i32(4, 3))), (ValueError, "mask must", lambda: Lo(x, mask=i32(4, 3))), (ValueError, "mask must", lambda: Lo(x, mask=i32(3, 2))),
            (ValueError, "mask must", lambda: Lo(x.view(2, 2, 64), mask=i32(4, 2))), (ValueError, "mask must", lambda: Lo(torch.zeros((2, 3, 64)), mask=i32(3, 2, 2))),
            (ValueError, "GPU", lambda: Lo(x)), (ValueError, "GPU", lambda: Lo(x, tokens=i32(4, 5)))):
        with pytest.raises(error, match=text):
            f()
