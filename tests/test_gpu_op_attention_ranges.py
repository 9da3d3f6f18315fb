"""Attention at the ends of its ranges: scores in the thousands, and the largest number of problems of a call."""
import math

import pytest
import torch

import tests.test_gpu_encoder as base
from tests.test_gpu_encoder import compare, d2p, inputs, reference, run_attention  # noqa: F401  (d2p: fixture)

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype,D,Lq,Lk", [(FP, 64, 130, 140), (BF, 128, 130, 300), (FP, 64, 1, 700)])
def test_scores_in_the_thousands(d2p, cuda_device, monkeypatch, dtype, D, Lq, Lk):  # noqa: F811
    """Only the fp32 term of the tolerance grows, by 8 units of the scores' magnitudes: the roundings to 16 bits are of the same
    size as with small scores."""
    q, k, v, do, _ = inputs(1, Lq, Lk, 2, 2, D, dtype, cuda_device, seed=7)
    size = float((torch.einsum("bihd,bjhd->bhij", q.double().abs(), k.double().abs()) * 40.0).max())
    monkeypatch.setattr(base, "F32", base.F32 + size * 2.0 ** -21)
    val, tol = reference(q, k, v, None, None, False, 40.0, 128, do)
    # (a gradient of dO V^T less its own mean: what is left of rows with one key is fp32's rounding of the two)
    compare(run_attention(d2p, q, k, v, do, None, None, False, scale=40.0), val, tol)


@pytest.mark.parametrize("Lq,Lk,causal", [(1, 9, True), (20, 20, False)])
def test_the_most_problems(d2p, cuda_device, Lq, Lk, causal):  # noqa: F811
    B, H, D = 65535, 2, 8
    q, k, v, do, bias = inputs(B, Lq, Lk, H, 1, D, BF, cuda_device, 4)
    lengths = torch.stack([torch.arange(B) % (Lq + 1), torch.arange(B) % (Lk + 1)], 1).to(torch.int32).to(cuda_device)
    got = run_attention(d2p, q, k, v, do, bias, lengths, causal, 16)
    picked = [0, 1, 777, 32768, 32769, 50000, B - 2, B - 1]
    val, tol = reference(q[picked], k[picked], v[picked], bias, lengths[picked], causal, 1 / math.sqrt(D), 16, do[picked])
    compare({n: got[n][picked] for n in ("out", "dq", "dk", "dv")}, val, tol)
    assert torch.isfinite(got["dbias"]).all()
