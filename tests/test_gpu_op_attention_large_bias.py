"""Attention with biases of large size: tables of lowest values and of -1e9, as masks are written, alone in a row and beside
others, near the diagonal and past the last edge; outputs and gradients against the 64-bit definition.

Only differences of a row's scores matter, so the tolerances are those of moderate scores (tests/test_gpu_encoder.py: scores of up to
~30; the scale here makes them that large).  Within a row the entries are either equal or so far apart that one side weighs
nothing: their difference in fp32 is exact or of no account."""
import math

import pytest
import torch

from tests.test_gpu_encoder import compare, d2p, inputs, reference, run_attention  # noqa: F401  (d2p: fixture)

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
LOWEST = "lowest"


def table(kind, nb, heads, dtype, dev):
    """[nb, heads]: head 0 as `kind` says, the others ordinary."""
    g = torch.Generator().manual_seed(5)
    t = torch.randn(nb, heads, generator=g)
    whole, value = kind
    value = torch.finfo(dtype).min if value == LOWEST else value
    if whole:
        t[:, 0] = value
    else:            # all but the nearest buckets of either side, so that distant rows meet nothing else
        t[2:nb // 2, 0] = value
        t[nb // 2 + 2:, 0] = value
    return t.to(dtype).to(dev)


@pytest.mark.parametrize("dtype,bias_dtype", [(BF, BF), (BF, F32), (FP, F32), (FP, FP)])
@pytest.mark.parametrize("kind", [(True, LOWEST), (True, -1e9), (True, 1e9), (True, -3e4), (False, LOWEST), (False, -1e9), (False, -3e4)])
@pytest.mark.parametrize("shape", [(1, 1, 150, 2, 2, 64), (2, 150, 400, 4, 2, 64), (1, 300, 40, 2, 1, 128), (1, 3, 5000, 2, 1, 128),
                                   (1, 40, 3000, 2, 2, 64)])
def test_large_biases(d2p, cuda_device, shape, kind, dtype, bias_dtype):  # noqa: F811
    B, Lq, Lk, H, Hkv, D = shape
    if kind[1] != LOWEST and abs(kind[1]) > torch.finfo(bias_dtype).max:
        kind = (kind[0], math.copysign(6e4, kind[1]))
    q, k, v, do, _ = inputs(B, Lq, Lk, H, Hkv, D, dtype, cuda_device, seed=Lk)
    bias = table(kind, 8, H, bias_dtype, cuda_device)
    scale = 6.0 / math.sqrt(D)   # scores of deviation 6
    for causal in (False, True):
        val, tol = reference(q, k, v, bias, None, causal, scale, 16, do)
        got = run_attention(d2p, q, k, v, do, bias, None, causal, 16, scale)
        compare(got, val, tol)
        alone = d2p.attention(q, k, v, bias=bias, causal=causal, max_distance=16, scale=scale)
        compare({"out": alone}, val, tol)


def test_scores_of_their_own_within_a_masked_row(d2p, cuda_device):  # noqa: F811
    """A row all of whose keys carry -1e9 is the softmax of its scores, like the row of the same call without a bias."""
    q, k, v, do, _ = inputs(1, 200, 300, 2, 2, 64, FP, cuda_device)
    flat = torch.full((8, 2), -1e9, device=cuda_device)
    val, tol = reference(q, k, v, None, None, False, 0.75, 16, do)
    got = run_attention(d2p, q, k, v, do, flat, None, False, 16, 0.75)
    compare({n: got[n] for n in ("out", "dq", "dk", "dv")}, val, tol)


@pytest.mark.parametrize("dtype,causal", [(BF, False), (FP, True)])
def test_large_biases_on_a_full_device(d2p, cuda_device, dtype, causal):  # noqa: F811
    """Several items a CTA, uneven lengths, heads with and without large entries."""
    B, L, H, Hkv, D = 40, 500, 16, 4, 64
    q, k, v, do, _ = inputs(B, L, L, H, Hkv, D, dtype, cuda_device, seed=3)
    bias = table((False, -1e9), 8, H, F32, cuda_device)
    bias[:, 6] = bias[:, 0]
    bias[:, 9] = torch.finfo(F32).min
    lengths = torch.tensor([[(b * 37) % (L + 1), (b * 53 + 20) % (L + 1)] for b in range(B)], dtype=torch.int32, device=cuda_device)
    val, tol = reference(q, k, v, bias, lengths, causal, 0.5, 16, do)
    compare(run_attention(d2p, q, k, v, do, bias, lengths, causal, 16, 0.5), val, tol)
