"""What the gated block and the log probabilities of tokens refuse, without a GPU: in Python by shape and type, at the C entry points by pointer, type and
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


def refuses(L, name, order, good, cases):
    for kw, code, text in cases:
        rc = getattr(L.lib, name)(*[kw.get(k, good[k]) for k in order.split()], None)
        said = L.lib.sp_last_error_string().decode()
        assert rc == code and text in said, (kw, rc, said)


def test_gated_refusals(L):
    order = "dtype act a bg bu c kept gate gs up us m n k"
    good = dict(dtype=2, act=0, a=P, bg=P, bu=P, c=P, kept=8, gate=P, gs=P, up=P, us=P, m=4, n=130, k=64)
    refuses(L, "sp_gemm_abt_gated", order, good, (
        (dict(a=None), -1, "A is NULL"), (dict(bg=None), -1, "B_gate is NULL"), (dict(bu=None), -1, "B_up is NULL"), (dict(c=None), -1, "C is NULL"), (dict(a=ODD), -3, "16-byte"),
        (dict(gate=ODD), -3, "16-byte"), (dict(us=ODD), -3, "16-byte"), (dict(dtype=8), -4, "dtype"), (dict(kept=9), -4, "kept"), (dict(kept=1), -4, "kept"), (dict(act=3), -5, "activation"),
        (dict(act=-1), -5, "activation"), (dict(up=None), -1, "go together"), (dict(gate=None), -1, "go together"), (dict(gs=None), -1, "scales"), (dict(us=None), -1, "scales"),
        (dict(m=0), -2, "positive"), (dict(n=0), -2, "positive"), (dict(k=-8), -2, "positive"), (dict(k=60), -2, "multiple of 8"), (dict(dtype=0, kept=0, k=6), -2, "multiple of 4"),
        (dict(m=1 << 31), -2, "too large"), (dict(n=(1 << 21) + 1), -2, "too large"), (dict(k=(1 << 22) + 8), -2, "too large"), (dict(dtype=0, kept=0, k=(1 << 21) + 4), -2, "too large")))


def test_gated_backward_refusals(L):
    order = "dtype act dc a bg bu kept gate gs up us da dg du m n k ws bytes"
    size = L.lib.sp_gemm_abt_gated_backward_workspace_bytes
    need = size(2, 4, 130, 64)
    assert need >= 4 * 2 * 192 * 2 and size(0, 4, 130, 64) >= 4 * 2 * 192 * 4
    assert size(2, 8192, 8192, 2048) == 8192 * 2 * 8192 * 2                   # enough tiles: no partial sums
    assert size(2, 0, 130, 64) == 0 and size(2, 4, -1, 64) == 0 and size(2, 4, 130, 0) == 0
    good = dict(dtype=2, act=0, dc=P, a=P, bg=P, bu=P, kept=8, gate=P, gs=P, up=P, us=P, da=P, dg=P, du=P, m=4, n=130, k=64, ws=P, bytes=need)
    refuses(L, "sp_gemm_abt_gated_backward", order, good, (
        (dict(dc=None), -1, "dC is NULL"), (dict(a=None), -1, "A is NULL"), (dict(gate=None), -1, "gate is NULL"), (dict(up=None), -1, "up is NULL"), (dict(da=ODD), -3, "16-byte"),
        (dict(dtype=7), -4, "dtype"), (dict(kept=0), -4, "kept"), (dict(act=9), -5, "activation"), (dict(gs=None), -1, "scales"), (dict(dg=None), -5, "both or neither"),
        (dict(da=None, dg=None, du=None), -1, "no gradient"), (dict(m=0), -2, "positive"), (dict(k=12), -2, "multiple of 8"), (dict(ws=None), -1, "workspace"),
        (dict(bytes=need - 1), -5, "workspace"), (dict(m=1 << 30), -2, "too large")))


def test_token_refusals(L):
    order = "dtype x tokens logp entropy lse top top_logp top_ids rows cols ws bytes"
    need = L.lib.sp_token_log_probs_workspace_bytes(1, 100000, 5)
    assert need > 0 and L.lib.sp_token_log_probs_workspace_bytes(0, 100000, 5) == 0 and L.lib.sp_token_log_probs_workspace_bytes(1, 100000, 33) == 0
    assert L.lib.sp_token_log_probs_workspace_bytes(1 << 16, 100000, 5) == 0
    good = dict(dtype=2, x=P, tokens=P, logp=P, entropy=P, lse=P, top=5, top_logp=P, top_ids=P, rows=1, cols=100000, ws=P, bytes=need)
    refuses(L, "sp_token_log_probs", order, good, (
        (dict(x=None), -1, "logits"), (dict(tokens=None), -1, "tokens"), (dict(logp=None), -1, "logp"), (dict(entropy=ODD), -3, "16-byte"), (dict(dtype=9), -4, "dtype"), (dict(rows=0), -2, "positive"),
        (dict(cols=0), -2, "positive"), (dict(cols=(1 << 30) + 1), -2, "too large"), (dict(rows=1 << 31), -2, "too large"), (dict(rows=1 << 24), -2, "too large"), (dict(top=33), -5, "top"),
        (dict(top=-1), -5, "top"), (dict(top_ids=None), -1, "top_logp"), (dict(ws=None), -1, "workspace"), (dict(bytes=need - 1), -5, "workspace")))
    order = "dtype x tokens lse entropy d_logp d_entropy d_lse dx rows cols"
    good = dict(dtype=2, x=P, tokens=P, lse=P, entropy=P, d_logp=P, d_entropy=P, d_lse=P, dx=P, rows=4, cols=1000)
    refuses(L, "sp_token_log_probs_backward", order, good, (
        (dict(x=None), -1, "logits"), (dict(tokens=None), -1, "tokens"), (dict(lse=None), -1, "lse"), (dict(dx=None), -1, "d_logits"), (dict(d_lse=ODD), -3, "16-byte"), (dict(dtype=9), -4, "dtype"),
        (dict(entropy=None), -1, "entropy"), (dict(rows=0), -2, "positive"), (dict(cols=(1 << 30) + 1), -2, "too large"), (dict(rows=(1 << 31) - 1, cols=1 << 20), -2, "too large")))


def test_python_refusals():
    from ml import matmul, primitives
    G, B, T, D = matmul.matmul_abt_gated, matmul.matmul_abt_gated_backward, primitives.token_log_probs, primitives.token_log_probs_backward
    a, w, dc = torch.zeros((4, 64)), torch.zeros((130, 64)), torch.zeros((4, 130))
    kept, kept8 = (dc, dc), (torch.zeros((4, 144)).to(F8), torch.zeros((4, 2)), torch.zeros((4, 144)).to(F8), torch.zeros((4, 2)))
    x, t, r = torch.zeros((4, 64)), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    for error, text, f in (
            (ValueError, "2-D", lambda: G(a[0], w, w)), (TypeError, "dtypes", lambda: G(a.half(), w, w)), (TypeError, "dtypes", lambda: G(a.double(), w.double(), w.double())),
            (ValueError, "one shape", lambda: G(a, w, w[:5])), (AssertionError, "K dimension", lambda: G(a[:, :32], w, w)), (ValueError, "activation", lambda: G(a, w, w, "tanh")),
            (ValueError, "activation", lambda: G(a, w, w, ["silu"])), (TypeError, "keep", lambda: G(a, w, w, keep=torch.float16)), (TypeError, "keep", lambda: G(a, w, w, keep=torch.float8_e5m2)),
            (ValueError, "GPU", lambda: G(a, w, w)), (ValueError, "dc must", lambda: B(dc[:3], a, w, w, kept)), (ValueError, "dc must", lambda: B(dc.half(), a, w, w, kept)),
            (ValueError, "kept must", lambda: B(dc, a, w, w, dc)), (ValueError, "kept must", lambda: B(dc, a, w, w, (dc,))), (ValueError, "kept gate", lambda: B(dc, a, w, w, (dc[:3], dc))),
            (ValueError, "kept up", lambda: B(dc, a, w, w, (dc, dc.half()))), (ValueError, "kept gate", lambda: B(dc, a, w, w, (dc, r, dc, r))),
            (ValueError, "kept gate_scale", lambda: B(dc, a, w, w, (kept8[0], r, kept8[2], kept8[3]))), (ValueError, "kept up_scale", lambda: B(dc, a, w, w, kept8[:3] + (r,))),
            (ValueError, "no gradient", lambda: B(dc, a, w, w, kept, want_input_grad=False, want_weight_grads=False)), (ValueError, "GPU", lambda: B(dc, a, w, w, kept)),
            (ValueError, "GPU", lambda: B(dc, a, w, w, kept8)), (ValueError, "activation", lambda: B(dc, a, w, w, kept, activation="elu")),
            (TypeError, "logits", lambda: T(x.double(), t)), (ValueError, "2 dimensions", lambda: T(x[0], t)), (ValueError, "one entry", lambda: T(x[:0], t[:0])), (ValueError, "one entry per row", lambda: T(x, t[:2])),
            (ValueError, "top", lambda: T(x, t, top=33)), (ValueError, "top", lambda: T(x, t, top=-1)), (ValueError, "GPU", lambda: T(x, t)), (TypeError, "logits", lambda: D(r, x.double(), t, r)),
            (ValueError, "one entry per row", lambda: D(r[:2], x, t, r)), (ValueError, "one entry per row", lambda: D(r, x, t, r[:2])), (ValueError, "lse is needed", lambda: D(r, x, t, None)),
            (ValueError, "needs the entropy", lambda: D(r, x, t, r, d_entropy=r)), (ValueError, "out must", lambda: D(r, x, t, r, out=x.half())), (ValueError, "GPU", lambda: D(r, x, t, r))):
        with pytest.raises(error, match=text):
            f()
