"""The size lists of the gated block's and the log probabilities' tests launch every kernel that the library has of them, in every type: a rule that chooses otherwise shows here."""
import re
import subprocess

import pytest
import torch

import test_gpu_gated as gated
import test_gpu_token_probs_kernels as tokens
from gpu_util import announce

pytestmark = pytest.mark.gpu


def kernels_of_the_library(pattern):
    from ml import _lib
    symbols = subprocess.run(["nm", "-C", "--defined-only", _lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    names = {re.sub(r"\(.*", "", line.split("__device_stub__")[1]) for line in symbols.split("\n") if "__device_stub__" in line}
    return {n for n in names if re.match(pattern, n)}


def kernels_of(run):
    from torch.profiler import ProfilerActivity, profile
    with profile(activities=[ProfilerActivity.CUDA], acc_events=True) as p:
        run()
        torch.cuda.synchronize()
    names = [e.name for e in p.events()]
    if not any("kernel" in n for n in names):
        pytest.skip("the profiler names no kernels here")
    return {m.group(1) for m in (re.search(r"sp::((?:gated|token)\w+(?:<[^>]*>)?)", n) for n in names) if m}


def test_log_probabilities():
    from ml import primitives as P
    announce("kernels of token_log_probs")

    def run():
        for dtype in tokens.PIECE:
            for rows, pieces in tokens.FORWARD:
                x, t = tokens.inputs(rows, tokens.columns(pieces, dtype), dtype, 40)
                P.token_log_probs(x, t, want_entropy=True, want_lse=True), P.token_log_probs(x, t)
            for rows, pieces in tokens.ALTERNATIVES:
                x, t = tokens.inputs(rows, tokens.columns(pieces, dtype), dtype, 41)
                P.token_log_probs(x, t, top=5, want_entropy=True), P.token_log_probs(x, t, top=5)
            for pieces in tokens.GRADIENT:
                for streamed in (False, True):
                    cols = tokens.columns(pieces, dtype)
                    x, t = tokens.inputs(tokens.rows_of(37, cols, dtype, streamed), cols, dtype, 42)
                    d = torch.zeros(x.shape[0], device="cuda")
                    P.token_log_probs_backward(d, x, t, d), P.token_log_probs_backward(d, x, t, d, d_entropy=d, entropy=d)

    launched = kernels_of(run)
    there = kernels_of_the_library(r"token_(probs|grad)")
    assert len(there) > 100 and launched >= there, sorted(there - launched)


def test_gated_block():
    from ml import matmul as M
    announce("kernels of matmul_abt_gated")

    def run():
        for dtype, t in gated.TYPES.items():
            for m, n, k in gated.SMALL + gated.LARGE + [(3000, 5461, 64)]:
                x, gate, up = gated.operands(m, n, k, dtype)
                for keep in (None, t, gated.F8):
                    M.matmul_abt_gated(x, gate, up, keep=keep)
            for m, n, k in gated.BACK:
                x, gate, up, dc = gated.operands(m, n, k, dtype, with_dc=True)
                M.matmul_abt_gated_backward(dc, x, gate, up, (dc, dc))
                if m < 100:
                    q, scale = M.quantize_blocks(dc)
                    M.matmul_abt_gated_backward(dc, x, gate, up, (q, scale, q, scale))

    launched = kernels_of(run)
    there = kernels_of_the_library("gated_")
    assert len(there) > 40 and launched >= there, sorted(there - launched)
