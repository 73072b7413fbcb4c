"""Forward results of the gated block that do not stay in the caches (more than 32 MiB each), with the factors kept beside them: rows of whole lines, whose factors are streamed too, and others."""
import pytest

from gpu_util import announce
from test_gpu_gated import F8, check_forward, operands

pytestmark = pytest.mark.gpu

# rows of whole lines of 128 bytes, and not; the first and the last in tiles of two sizes
SIZES_16 = [(4099, 4160, 72), (4099, 5461, 72), (8193, 2624, 520), (5043, 4544, 8), (5008, 5461, 264)]
SIZES_32 = [(2053, 4128, 72), (2053, 4111, 72)]


@pytest.fixture(scope="module")
def M():
    from ml import matmul
    return matmul


@pytest.mark.parametrize("m,n,k,dtype", [s + (t,) for t in ("f16", "bf16") for s in SIZES_16] + [s + ("f32",) for s in SIZES_32])
@pytest.mark.parametrize("keep", ["none", "whole", "f8"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_streamed(M, m, n, k, dtype, keep, act):
    announce("matmul_abt_gated streamed %s" % ((m, n, k, dtype, keep, act),))
    x, gate, up = operands(m, n, k, dtype, seed=14)
    assert m * n * x.element_size() > 32 << 20
    check_forward(M, x, gate, up, act, keep={"none": None, "whole": x.dtype, "f8": F8}[keep])
