"""Memory and sizes that the gated block and the log probabilities of tokens refuse, and how near they go to that, without a GPU: what is taken ends at the missing device."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses of the calls that are taken are made up")

TAKEN, ARG, SHAPE = -7, -5, -2        # (TAKEN: nothing was refused, and then no device is there)


@pytest.fixture(scope="module")
def L():
    from ml import _lib
    return _lib


class Caller:
    """An entry point with arguments that are right, and what another value of some of them leads to."""

    def __init__(self, L, name, order, good):
        self.L, self.name, self.order, self.good = L, name, order.split(), good

    def __call__(self, **other):
        assert set(other) <= set(self.good)
        rc = getattr(self.L.lib, self.name)(*[other.get(k, self.good[k]) for k in self.order], None)
        said = self.L.lib.sp_last_error_string().decode()
        return rc, said


def places(**sizes):
    """Addresses behind each other without a gap but for the 16-byte alignment, in an order of their own."""
    at, out = 1 << 40, {}
    for name, size in sizes.items():
        out[name] = C.c_void_p(at)
        at += -(-size // 16) * 16
    return out


def sweep(call, sizes, outs, may_meet):
    """Every result moved over every other piece of memory, by its first and by its last 16 bytes: refused but for the pairs in may_meet; side by side all is taken."""
    rc, said = call()
    assert rc == TAKEN, said
    address = lambda n: call.good[n].value
    for o in outs:
        for other in sizes:
            if other == o:
                continue
            for at in (address(other), address(other) + sizes[other] - 16 & ~15, address(other) - (sizes[o] - 1 & ~15)):
                meets = [n for n in sizes if n != o and at < address(n) + sizes[n] and address(n) < at + sizes[o]]
                rc, said = call(**{o: C.c_void_p(at)})
                bad = [n for n in meets if not may_meet(o, n)]
                if bad:
                    assert rc == ARG and "overlap" in said and o in said and any(n in said for n in bad), (o, other, meets, rc, said)
                else:
                    assert rc == TAKEN, (o, other, meets, said)


@pytest.mark.parametrize("dtype,kept", [(2, 2), (0, 0), (1, 8), (0, 8)])
def test_gated_results_over_operands(L, dtype, kept):
    m, n, k = 37, 300, 64
    es, f8 = (4 if dtype == 0 else 2), kept == 8
    factor, scales = (m * 304, m * 3 * 4) if f8 else (m * n * es, 0)
    sizes = dict(A=m * k * es, C=m * n * es, gate=factor, B_gate=n * k * es, up=factor, B_up=n * k * es)
    if f8:
        sizes.update(gate_scale=scales, up_scale=scales)
    p = places(**sizes)
    good = {**dict(dtype=dtype, act=0, kept=kept, gate_scale=None, up_scale=None, m=m, n=n, k=k), **p}
    call = Caller(L, "sp_gemm_abt_gated", "dtype act A B_gate B_up C kept gate gate_scale up up_scale m n k", good)
    sweep(call, sizes, [o for o in ("C", "gate", "up", "gate_scale", "up_scale") if o in sizes], lambda o, other: False)
    assert call(B_up=p["B_gate"])[0] == TAKEN                # (operands are read alone)


@pytest.mark.parametrize("dtype,kept", [(2, 2), (0, 0), (1, 8), (0, 8)])
def test_gated_gradients_over_operands(L, dtype, kept):
    m, n, k = 37, 300, 64
    es, f8 = (4 if dtype == 0 else 2), kept == 8
    factor, scales = (m * 304, m * 3 * 4) if f8 else (m * n * es, 0)
    need = L.lib.sp_gemm_abt_gated_backward_workspace_bytes(dtype, m, n, k)
    sizes = dict(dC=m * n * es, A=m * k * es, dA=m * k * es, B_gate=n * k * es, dB_up=n * k * es, B_up=n * k * es, dB_gate=n * k * es, workspace=need, gate=factor, up=factor)
    if f8:
        sizes.update(gate_scale=scales, up_scale=scales)
    p = places(**sizes)
    good = {**dict(dtype=dtype, act=0, kept=kept, gate_scale=None, up_scale=None, m=m, n=n, k=k, bytes=need + 4096), **p}      # (what is more than needed is not looked at)
    call = Caller(L, "sp_gemm_abt_gated_backward", "dtype act dC A B_gate B_up kept gate gate_scale up up_scale dA dB_gate dB_up m n k workspace bytes", good)
    early = {"dC", "gate", "up", "gate_scale", "up_scale"}            # read before any gradient is written
    sweep(call, sizes, ["dA", "dB_gate", "dB_up", "workspace"], lambda o, other: o != "workspace" and other in early)
    # what is not wanted is nowhere
    assert call(dA=None)[0] == TAKEN and call(dB_gate=None, dB_up=None)[0] == TAKEN


@pytest.mark.parametrize("dtype,top,cols", [(2, 5, 9001), (0, 0, 300), (1, 32, 70), (0, 0, 40000)])
def test_log_probabilities_over_logits(L, dtype, top, cols):
    rows = 37
    need = L.lib.sp_token_log_probs_workspace_bytes(rows, cols, top)
    sizes = dict(logp=rows * 4, logits=rows * cols * (4 if dtype == 0 else 2), entropy=rows * 4, tokens=rows * 4, lse=rows * 4)
    if top:
        sizes.update(top_logp=rows * top * 4, top_ids=rows * top * 4)
    if need:
        sizes.update(workspace=need)
    call = tokens_forward(L, dtype=dtype, rows=rows, cols=cols, top=top, bytes=need, **places(**sizes))
    sweep(call, sizes, [o for o in sizes if o not in ("logits", "tokens")], lambda o, other: False)


@pytest.mark.parametrize("dtype,cols", [(2, 9001), (0, 300), (1, 7)])
def test_their_gradient_over_what_it_reads(L, dtype, cols):
    rows = 37
    numbers = rows * cols * (4 if dtype == 0 else 2)
    sizes = dict(logits=numbers, tokens=rows * 4, lse=rows * 4, d_logits=numbers, entropy=rows * 4, d_logp=rows * 4, d_entropy=rows * 4, d_lse=rows * 4)
    call = tokens_backward(L, dtype=dtype, rows=rows, cols=cols, **places(**sizes))
    assert call(d_logits=call.good["logits"])[0] == TAKEN
    for away in (16, 32, numbers - 16 & ~15):
        for at in (call.good["logits"].value + away, call.good["logits"].value - away):
            rc, said = call(d_logits=C.c_void_p(at))
            assert rc == ARG and "d_logits and logits overlap" in said
    del sizes["logits"]                                   # (the others, at places that the logits do not reach)
    call.good["logits"] = C.c_void_p(1 << 30)
    sweep(call, sizes, ["d_logits"], lambda o, other: False)
    # without d_entropy nobody looks at the entropy
    assert call(d_entropy=None, d_logits=call.good["entropy"], entropy=call.good["entropy"], d_logp=None, d_lse=None)[0] == TAKEN


def tokens_forward(L, **other):
    p = {n: C.c_void_p((1 << 44) + (i << 50)) for i, n in enumerate(("logits", "tokens", "logp", "entropy", "lse", "top_logp", "top_ids", "workspace"))}      # (far apart)
    good = {**dict(dtype=2, top=0, rows=1, cols=16, bytes=1 << 40), **p, **other}
    return Caller(L, "sp_token_log_probs", "dtype logits tokens logp entropy lse top top_logp top_ids rows cols workspace bytes", good)


def tokens_backward(L, **other):
    p = {n: C.c_void_p((1 << 44) + (i << 50)) for i, n in enumerate(("logits", "tokens", "lse", "entropy", "d_logp", "d_entropy", "d_lse", "d_logits"))}
    good = {**dict(dtype=2, rows=1, cols=16), **p, **other}
    return Caller(L, "sp_token_log_probs_backward", "dtype logits tokens lse entropy d_logp d_entropy d_lse d_logits rows cols", good)


# lanes to a row: 4 to 64 of a wave, a workgroup of 256 or 512
@pytest.mark.parametrize("dtype,cols,top,lanes", [(2, 32, 0, 4), (0, 64, 0, 4), (2, 256, 0, 16), (1, 1024, 0, 16), (2, 1032, 0, 64), (2, 8192, 0, 64), (0, 4096, 0, 64), (2, 64, 1, 256), (2, 8200, 0, 256),
                                                  (2, 16384, 0, 256), (2, 16385, 0, 512), (0, 20000, 5, 512)])
def test_log_probabilities_take_as_many_rows_as_a_launch_holds(L, dtype, cols, top, lanes):
    """A launch holds fewer than 2^32 work items: the last number of rows that fits is taken, one more is refused here and not by the launch."""
    most = min((1 << 32) - 256, ((1 << 31) - 1) * lanes) // lanes
    assert tokens_forward(L, dtype=dtype, cols=cols, top=top, rows=most)()[0] == TAKEN
    rc, said = tokens_forward(L, dtype=dtype, cols=cols, top=top, rows=most + 1)()
    assert rc == SHAPE and "too large" in said


@pytest.mark.parametrize("dtype,cols,lanes", [(2, 32, 4), (0, 64, 4), (1, 1024, 16), (2, 1032, 64), (2, 2048, 64), (2, 2056, 256), (0, 4100, 512)])
def test_their_gradient_too(L, dtype, cols, lanes):
    most = ((1 << 32) - 256) // lanes
    assert tokens_backward(L, dtype=dtype, cols=cols, rows=most)()[0] == TAKEN
    rc, said = tokens_backward(L, dtype=dtype, cols=cols, rows=most + 1)()
    assert rc == SHAPE and "too large" in said
