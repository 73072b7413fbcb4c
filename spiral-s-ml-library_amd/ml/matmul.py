"""Host surface of the tiled GEMM (reference: ml/matmul/run.spi, generated ml/matmul/run.py).

`matmul_tf32(a_trans, b_trans, alpha, a, b, beta, c)` keeps the reference's name and argument
order (ml/matmul/run.spi:25); `main()` / `main_body()` keep the self-test meaning of the generated
module (random A, B, C of 8192 x 8192 x 4096, compare against a library GEMM, return the max
absolute difference; ml/matmul/run.spi:28-58).  The multiplication itself runs in
libspiral_mi355.so (sp_gemm_abt).
"""
import ctypes as C

import torch

from . import _lib
from ._lib import check, lib, ptr, stream_ptr


def matmul_config_tf32(a_trans, b_trans, m, n, k, dtype=torch.float32):
    """Tile configuration chosen for a shape (counterpart of ml/matmul/run.spi:8-19).
    Returns dict(m_tile, n_tile, k_tile, threads); m_tile == 0 means one thread per output."""
    out = [C.c_int32() for _ in range(4)]
    check(lib.sp_gemm_config(_lib.DTYPES[dtype], m, n, k, *[C.byref(o) for o in out]))
    return dict(zip(("m_tile", "n_tile", "k_tile", "threads"), (o.value for o in out)))


def matmul_config_batched(batch, m, n, k, dtype=torch.float32):
    """The same for one launch over `batch` matrices, with k_parts, the partial sums over K behind an output (0: one thread)."""
    out = [C.c_int32() for _ in range(5)]
    check(lib.sp_gemm_batched_config(_lib.DTYPES[dtype], m, n, k, batch, *[C.byref(o) for o in out]))
    return dict(zip(("m_tile", "n_tile", "k_tile", "threads", "k_parts"), (o.value for o in out)))


def matmul_abt(a, b, c=None, alpha=1.0, beta=0.0, bias=None, relu=False, out_dtype=None, force_generic=False):
    """C = alpha * A . B^T + beta * C (+ bias, ReLU).  a: (M, K), b: (N, K), both row-major and of
    the same dtype (f32, f16 or bf16).  `c` is updated in place and returned; when it is None a new
    (M, N) tensor of `out_dtype` (default f32) is allocated by torch (beta must then be 0)."""
    if a.dim() != 2 or b.dim() != 2:
        raise ValueError("a and b must be 2-D")
    if a.dtype != b.dtype or a.dtype not in _lib.DTYPES:
        raise TypeError("a and b must share one of the dtypes f32/f16/bf16")
    m, k = a.shape
    n, kb = b.shape
    assert k == kb, "The K dimension of the A and B tensors must match."
    if c is None:
        assert beta == 0.0, "beta != 0 needs an existing C"
        c = torch.empty((m, n), dtype=out_dtype or torch.float32, device=a.device)
    assert c.shape[0] == m, "The M dimension of the A and C tensors must match."
    assert c.shape[1] == n, "The N dimension of the B and C tensors must match."
    assert alpha != 0, "The alpha must not be zero."
    flags = (_lib.GEMM_RELU if relu else 0) | (_lib.GEMM_FORCE_GENERIC if force_generic else 0)
    check(lib.sp_gemm_abt(_lib.DTYPES[a.dtype], _lib.DTYPES[c.dtype], ptr(a, name="a"), ptr(b, name="b"),
                          ptr(c, name="c"), ptr(bias, torch.float32, "bias"), m, n, k, float(alpha), float(beta),
                          flags, stream_ptr()))
    return c


def matmul_abt_batched(a, b, c=None, alpha=1.0, beta=0.0, bias=None, relu=False, out_dtype=None, force_generic=False):
    """C[e] = alpha * A[e] . B[e]^T + beta * C[e] for every batch member in ONE launch.  a: (E, M, K) or (M, K)
    (shared by all members), b: (E, N, K) or (N, K), at least one of them batched; c: (E, M, N).  This is the
    loop `graph_run_host model {ensemble}` makes around a `matmul_ensemble` layer (ml/layers.spi:336-344,468-471).
    In f32 every member is bit-identical to `matmul_abt` on it alone; in 16 bit a batch may add up K in another order."""
    if a.dtype != b.dtype or a.dtype not in _lib.DTYPES:
        raise TypeError("a and b must share one of the dtypes f32/f16/bf16")
    if a.dim() not in (2, 3) or b.dim() not in (2, 3) or (a.dim() == 2 and b.dim() == 2):
        raise ValueError("a is (E, M, K) or (M, K), b is (E, N, K) or (N, K), and one of them must carry the batch")
    e = a.shape[0] if a.dim() == 3 else b.shape[0]
    if a.dim() == 3 and b.dim() == 3:
        assert a.shape[0] == b.shape[0], "The batch dimensions of the A and B tensors must match."
    m, k = a.shape[-2:]
    n, kb = b.shape[-2:]
    assert k == kb, "The K dimension of the A and B tensors must match."
    if c is None:
        assert beta == 0.0, "beta != 0 needs an existing C"
        c = torch.empty((e, m, n), dtype=out_dtype or torch.float32, device=a.device)
    assert tuple(c.shape) == (e, m, n), "The dimensions of the C tensor must be (batch, M, N)."
    assert alpha != 0, "The alpha must not be zero."
    flags = (_lib.GEMM_RELU if relu else 0) | (_lib.GEMM_FORCE_GENERIC if force_generic else 0)
    check(lib.sp_gemm_abt_batched(_lib.DTYPES[a.dtype], _lib.DTYPES[c.dtype], ptr(a, name="a"), ptr(b, name="b"),
                                  ptr(c, name="c"), ptr(bias, torch.float32, "bias"), m, n, k, e,
                                  m * k if a.dim() == 3 else 0, n * k if b.dim() == 3 else 0, m * n, float(alpha),
                                  float(beta), flags, stream_ptr()))
    return c


def _blocks(n):
    return -(-n // 128)


def _on_device_of(what, *tensors):
    """The device index all of `tensors` (None passed over) live on: a launch on another device than theirs would read foreign memory."""
    index = None
    for t in tensors:
        if t is not None and t.is_cuda:
            if index is None:
                index = t.device.index
            elif t.device.index != index:
                raise ValueError("%s: the tensors live on different devices" % what)
    return index


def quantize_blocks(x, block=(1, 128), dtype=torch.float8_e4m3fn, transpose=False):
    """x (rows, cols) f32, f16 or bf16 in 8-bit blocks with an f32 scale each (sp_quantize_blocks): (q, scale), the operand of
    `matmul_abt_scaled`.  `block` is (1, 128), for activations, or (128, 128), for weights; a block's scale is its largest magnitude over the
    type's largest number.  q is (rows, cols rounded up to a multiple of 16), zeros behind the columns of x; scale (rows or ceil(rows / 128),
    ceil(cols / 128)).  transpose=True gives the same of the transpose of x, transpose="both" reads x once and gives
    (q, scale, q_t, scale_t): what a layer's forward product and the gradients of its input (weights) or its weights (activations) take."""
    if transpose in (False, True):
        transpose = bool(transpose)                                # (0 and 1 are taken for them)
    if (block == (1, 128) or block == (128, 128)) and (transpose in (False, True) or transpose == "both"):
        done = lib.whole_quantize_blocks(x, block[0], dtype, transpose is not True, transpose is not False)
        if done is not None:
            return done
    if x.dim() != 2:
        raise ValueError("x must be 2-D")
    if x.dtype not in _lib.DTYPES:
        raise TypeError("x must be f32, f16 or bf16, got %s" % x.dtype)
    if dtype not in _lib.F8_TYPES:
        raise TypeError("dtype must be torch.float8_e4m3fn or torch.float8_e5m2, got %s" % dtype)
    block = tuple(block)
    if block not in ((1, 128), (128, 128)):
        raise ValueError("block must be (1, 128) or (128, 128), got %r" % (block,))
    if transpose not in (False, True, "both"):
        raise ValueError("transpose must be False, True or \"both\", got %r" % (transpose,))
    rows, cols = x.shape
    if rows == 0 or cols == 0:
        raise ValueError("x must not be empty, got %d x %d" % (rows, cols))
    address = ptr(x, name="x")
    if x.device.index != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return quantize_blocks(x, block, dtype, transpose)
    out = []
    for r, c, wanted in ((rows, cols, transpose is not True), (cols, rows, transpose is not False)):
        if wanted:
            out += [torch.empty((r, (c + 15) // 16 * 16), dtype=dtype, device=x.device),
                    torch.empty((r if block[0] == 1 else _blocks(r), _blocks(c)), dtype=torch.float32, device=x.device)]
        else:
            out += [None, None]
    check(lib.sp_quantize_blocks(_lib.DTYPES[x.dtype], _lib.F8_TYPES[dtype], block[0], address, ptr(out[0]), ptr(out[1]), ptr(out[2]),
                                 ptr(out[3]), rows, cols, stream_ptr()))
    return tuple(t for t in out if t is not None)


def matmul_abt_scaled(a, scale_a, b, scale_b, c=None, beta=0.0, bias=None, relu=False, out_dtype=None):
    """C = A . B^T + beta * C (+ bias, ReLU) of 8-bit operands with a scale for each block of 128 along K (sp_gemm_abt_scaled): the
    numbers a (M, K), b (N, K), e4m3 or e5m2, and their scales as `quantize_blocks` gives them.  scale_a is (M, ceil(K / 128)), scale_b
    (N, ceil(K / 128)) or, in blocks of 128 x 128, (ceil(N / 128), ceil(K / 128)).  `c` (f32, f16 or bf16) is updated in place and returned; when it
    is None a new (M, N) tensor of `out_dtype` (default f32) is allocated by torch (beta must then be 0).  Sums are f32, whatever the type of C;
    ReLU makes a NaN 0, as in `matmul_abt`.

    A layer y = x . W^T and its gradients, with dy, x and W of M x N, M x K and N x K:
        x8, sx, xt, sxt = quantize_blocks(x, transpose="both");  w8, sw, wt, swt = quantize_blocks(W, (128, 128), transpose="both")
        d8, sd, dt, sdt = quantize_blocks(dy, dtype=torch.float8_e5m2, transpose="both")
        y = matmul_abt_scaled(x8, sx, w8, sw);  dx = matmul_abt_scaled(d8, sd, wt, swt);  dW = matmul_abt_scaled(dt, sdt, xt, sxt)
    for any M, N and K: both operands of a product have the same padding."""
    if c is None and beta == 0.0:
        done = lib.whole_matmul_abt_scaled(a, scale_a, b, scale_b, bias, relu, out_dtype or torch.float32)
        if done is not None:
            return done
    if a.dim() != 2 or b.dim() != 2 or scale_a.dim() != 2 or scale_b.dim() != 2:
        raise ValueError("a, b and their scales must be 2-D")
    if a.dtype not in _lib.F8_TYPES or b.dtype not in _lib.F8_TYPES:
        raise TypeError("a and b must be torch.float8_e4m3fn or torch.float8_e5m2, got %s and %s" % (a.dtype, b.dtype))
    m, k = a.shape
    n, kb = b.shape
    assert k == kb, "The K dimension of the A and B tensors must match."
    if tuple(scale_a.shape) != (m, _blocks(k)):
        raise ValueError("scale_a must be (M, ceil(K / 128)) = (%d, %d), got %s" % (m, _blocks(k), tuple(scale_a.shape)))
    if tuple(scale_b.shape) not in ((n, _blocks(k)), (_blocks(n), _blocks(k))):
        raise ValueError("scale_b must be (N, ceil(K / 128)) = (%d, %d) or (ceil(N / 128), ceil(K / 128)) = (%d, %d), got %s"
                         % (n, _blocks(k), _blocks(n), _blocks(k), tuple(scale_b.shape)))
    if c is None:
        assert beta == 0.0, "beta != 0 needs an existing C"
        out = out_dtype or torch.float32
    else:
        assert tuple(c.shape) == (m, n), "The dimensions of the C tensor must be (M, N)."
        out = c.dtype
        if out_dtype is not None and out_dtype != out:
            raise TypeError("out_dtype is %s, c is %s" % (out_dtype, out))
    if out not in _lib.DTYPES:
        raise TypeError("C must be f32, f16 or bf16, got %s" % out)
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError("bias must be (N,) = (%d,), got %s" % (n, tuple(bias.shape)))
    addresses = (ptr(a, name="a"), ptr(scale_a, torch.float32, "scale_a"), ptr(b, name="b"), ptr(scale_b, torch.float32, "scale_b"))
    bias_at = ptr(bias, torch.float32, "bias")
    device = _on_device_of("matmul_abt_scaled", a, scale_a, b, scale_b, c, bias)
    if device != torch.cuda.current_device():
        with torch.cuda.device(device):
            return matmul_abt_scaled(a, scale_a, b, scale_b, c, beta, bias, relu, out_dtype)
    if c is None:
        c = torch.empty((m, n), dtype=out, device=a.device)
    check(lib.sp_gemm_abt_scaled(_lib.F8_TYPES[a.dtype], _lib.F8_TYPES[b.dtype], _lib.DTYPES[out], *addresses,
                                 1 if scale_b.shape[0] == n else 128, ptr(c, name="c"), bias_at, m, n, k, float(beta),
                                 _lib.GEMM_RELU if relu else 0, stream_ptr()))
    return c


def _gated_operands(a, b_gate, b_up, activation):
    """(M, N, K) of a gated block's operands, which have one type."""
    if a.dim() != 2 or b_gate.dim() != 2 or b_up.dim() != 2:
        raise ValueError("a, b_gate and b_up must be 2-D")
    if a.dtype not in _lib.DTYPES or b_gate.dtype != a.dtype or b_up.dtype != a.dtype:
        raise TypeError("a, b_gate and b_up must share one of the dtypes f32/f16/bf16, got %s, %s and %s" % (a.dtype, b_gate.dtype, b_up.dtype))
    if b_gate.shape != b_up.shape:
        raise ValueError("b_gate and b_up must have one shape, got %s and %s" % (tuple(b_gate.shape), tuple(b_up.shape)))
    assert a.shape[1] == b_gate.shape[1], "The K dimension of the A and B tensors must match."
    if not isinstance(activation, str) or activation not in _lib.ACTIVATIONS:
        raise ValueError("activation must be \"silu\", \"gelu\" or \"relu\", got %r" % (activation,))
    return a.shape[0], b_gate.shape[0], a.shape[1]


def matmul_abt_gated(a, b_gate, b_up, activation="silu", keep=None):
    """The gated feed-forward block C = act(A . B_gate^T) * (A . B_up^T) in one launch (sp_gemm_abt_gated), next to `matmul_abt` with its ReLU.  a (M, K), b_gate and
    b_up (N, K): f32, f16 or bf16, the type of C (M, N); sums, activation ("silu", "gelu", the one with erf, or "relu") and product are f32.

    keep: what `matmul_abt_gated_backward` is to find of the two products, (c, kept) then.  keep=a.dtype: kept is (gate, up), (M, N) each; keep=torch.float8_e4m3fn, a quarter to half of
    that: (gate, gate_scale, up, up_scale), in the (1, 128) blocks of `quantize_blocks`."""
    done = lib.whole_matmul_abt_gated(a, b_gate, b_up, _lib.ACTIVATIONS.get(activation) if isinstance(activation, str) else None, keep)
    if done is not None:
        return done
    m, n, k = _gated_operands(a, b_gate, b_up, activation)
    f8 = keep == torch.float8_e4m3fn
    if keep is not None and keep != a.dtype and not f8:
        raise TypeError("keep must be None, %s or torch.float8_e4m3fn, got %s" % (a.dtype, keep))
    addresses = ptr(a, name="a"), ptr(b_gate, name="b_gate"), ptr(b_up, name="b_up")
    if _on_device_of("matmul_abt_gated", a, b_gate, b_up) != torch.cuda.current_device():
        with torch.cuda.device(a.device):
            return matmul_abt_gated(a, b_gate, b_up, activation, keep)
    new = lambda r, c, dtype: torch.empty((r, c), dtype=dtype, device=a.device)
    c = new(m, n, a.dtype)
    gate = gate_scale = up = up_scale = None
    kept = ()
    if f8:
        gate, up = (new(m, (n + 15) // 16 * 16, keep) for _ in range(2))
        gate_scale, up_scale = (new(m, _blocks(n), torch.float32) for _ in range(2))
        kept = gate, gate_scale, up, up_scale
    elif keep is not None:
        kept = gate, up = new(m, n, keep), new(m, n, keep)
    check(lib.sp_gemm_abt_gated(_lib.DTYPES[a.dtype], _lib.ACTIVATIONS[activation], *addresses, ptr(c), _lib.SP_F8_E4M3 if f8 else _lib.DTYPES[a.dtype], ptr(gate),
                                ptr(gate_scale), ptr(up), ptr(up_scale), m, n, k, stream_ptr()))
    return c if keep is None else (c, kept)


def matmul_abt_gated_backward(dc, a, b_gate, b_up, kept, activation="silu", want_input_grad=True, want_weight_grads=True):
    """The gradients of `matmul_abt_gated` (sp_gemm_abt_gated_backward): (da, db_gate, db_up), of the type of a, from dc (M, N), the operands and what the forward call kept.  They
    are those at the numbers that were kept, with dg and du rounded to the type of a on the way: in f16 one above 65504 is an infinity, so a loss is scaled for them, too.  da is None with want_input_grad=False, db_gate and db_up with want_weight_grads=False."""
    if want_input_grad is True and want_weight_grads is True and type(kept) is tuple and len(kept) in (2, 4):
        done = lib.whole_matmul_abt_gated_backward(dc, a, b_gate, b_up, kept[0], kept[1] if len(kept) == 4 else None, kept[-2] if len(kept) == 4 else kept[1],
                                                   kept[3] if len(kept) == 4 else None, _lib.ACTIVATIONS.get(activation) if isinstance(activation, str) else None)
        if done is not None:
            return done
    m, n, k = _gated_operands(a, b_gate, b_up, activation)
    if dc.shape != (m, n) or dc.dtype != a.dtype:
        raise ValueError("dc must be (M, N) = (%d, %d) of %s, got %s of %s" % (m, n, a.dtype, tuple(dc.shape), dc.dtype))
    if not isinstance(kept, (tuple, list)) or len(kept) not in (2, 4):
        raise ValueError("kept must be what matmul_abt_gated returned beside its result: (gate, up) or (gate, gate_scale, up, up_scale)")
    gate, gate_scale, up, up_scale = kept if len(kept) == 4 else (kept[0], None, kept[1], None)
    f8 = len(kept) == 4
    shape, dtype = ((m, (n + 15) // 16 * 16), torch.float8_e4m3fn) if f8 else ((m, n), a.dtype)
    for t, name in ((gate, "gate"), (up, "up")):
        if tuple(t.shape) != shape or t.dtype != dtype:
            raise ValueError("the kept %s must be %s of %s, got %s of %s" % (name, shape, dtype, tuple(t.shape), t.dtype))
    if f8:
        for t, name in ((gate_scale, "gate_scale"), (up_scale, "up_scale")):
            if tuple(t.shape) != (m, _blocks(n)):
                raise ValueError("the kept %s must be %s, got %s" % (name, (m, _blocks(n)), tuple(t.shape)))
    if not want_input_grad and not want_weight_grads:
        raise ValueError("no gradient is wanted")
    f32 = torch.float32
    addresses = ptr(dc, name="dc"), ptr(a, name="a"), ptr(b_gate, name="b_gate"), ptr(b_up, name="b_up")
    kept_at = ptr(gate, name="gate"), ptr(gate_scale, f32, "gate_scale"), ptr(up, name="up"), ptr(up_scale, f32, "up_scale")
    if _on_device_of("matmul_abt_gated_backward", dc, a, b_gate, b_up, gate, gate_scale, up, up_scale) != torch.cuda.current_device():
        with torch.cuda.device(a.device):
            return matmul_abt_gated_backward(dc, a, b_gate, b_up, kept, activation, want_input_grad, want_weight_grads)
    da = torch.empty_like(a) if want_input_grad else None
    db_gate, db_up = (torch.empty_like(b_gate) if want_weight_grads else None for _ in range(2))
    bytes_ = lib.sp_gemm_abt_gated_backward_workspace_bytes(_lib.DTYPES[a.dtype], m, n, k)
    workspace = torch.empty((bytes_,), dtype=torch.uint8, device=a.device)                  # of this call alone: calls may overlap
    check(lib.sp_gemm_abt_gated_backward(_lib.DTYPES[a.dtype], _lib.ACTIVATIONS[activation], *addresses, _lib.SP_F8_E4M3 if f8 else _lib.DTYPES[a.dtype], *kept_at,
                                         ptr(da), ptr(db_gate), ptr(db_up), m, n, k, ptr(workspace), bytes_, stream_ptr()))
    return da, db_gate, db_up


def _transposed(x):
    """Materialise x^T with the library's transpose kernel (4-byte elements only)."""
    if x.dtype != torch.float32:
        raise NotImplementedError("transposed operands are supported for f32 only")
    rows, cols = x.shape
    out = torch.empty((cols, rows), dtype=x.dtype, device=x.device)
    check(lib.sp_transpose_inner_b32(ptr(x), ptr(out), 1, rows, cols, stream_ptr()))
    return out


def matmul_tf32(a_trans, b_trans, alpha, a, b, beta, c):
    """`matmul_tf32 a_trans b_trans alpha a b beta c` (ml/matmul/run.spi:25): c <- alpha * op(a) .
    op(b) + beta * c.  The native layout is a_trans=False, b_trans=True (A (M,K), B (N,K)); the
    other three are brought to it by one transpose kernel.  Products are full f32 here, not TF32."""
    if a_trans:
        a = _transposed(a)       # stored (K, M) -> (M, K)
    if not b_trans:
        b = _transposed(b)       # stored (K, N) -> (N, K)
    return matmul_abt(a, b, c, alpha, beta)


def main_body(m=512 * 16, n=512 * 16, k=512 * 8, seed=12344321):
    """The reference self-test (ml/matmul/run.spi:28-58): C <- A . B^T + C on N(0,1) f32 inputs,
    compared against a library GEMM (torch.matmul here, cuBLAS through CuPy there).  Returns the
    max absolute difference as a 0-d tensor."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    mc = torch.randn((m, n), generator=gen, device="cuda", dtype=torch.float32)
    mb = torch.randn((n, k), generator=gen, device="cuda", dtype=torch.float32)
    ma = torch.randn((m, k), generator=gen, device="cuda", dtype=torch.float32)
    d = torch.matmul(ma, mb.t()) + mc
    matmul_tf32(False, True, 1.0, ma, mb, 1.0, mc)
    return torch.max(torch.abs(mc - d))


def main():
    r = main_body()
    torch.cuda.current_stream().synchronize()  # surface device faults here, like the reference does
    return float(r)


if __name__ == "__main__":
    print(main())
