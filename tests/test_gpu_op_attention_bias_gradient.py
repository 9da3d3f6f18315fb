"""The bias table's gradient: buckets of no weight, and sums over many items a CTA."""
import math

import pytest
import torch

from tests.test_gpu_encoder import compare, d2p, inputs, reference, run_attention  # noqa: F401  (d2p: fixture)

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype,D", [(BF, 64), (FP, 128)])
def test_a_masked_bucket_has_no_gradient(d2p, cuda_device, dtype, D, causal):  # noqa: F811
    """Buckets of -inf take no weight, so their gradient is nothing at all, wide or narrow, beside buckets that have some."""
    q, k, v, do, bias = inputs(3, 500, 450, 4, 2, D, dtype, cuda_device, 32, seed=D, bias_dtype=torch.float32)
    masked = torch.tensor([3, 11, 12, 14, 15, 20, 28, 31] if not causal else [2, 9, 18, 19, 27, 30, 31], device=cuda_device)
    bias[masked] = -math.inf
    val, tol = reference(q, k, v, bias, None, causal, D ** -0.5, 128, do)
    got = run_attention(d2p, q, k, v, do, bias, None, causal)
    assert not got["dbias"][masked].any(), got["dbias"][masked]
    compare(got, val, tol)


@pytest.mark.parametrize("B,L,H,Hkv,D,dtype,causal,ragged", [
    (64, 512, 8, 8, 64, BF, False, True), (48, 512, 16, 4, 128, BF, True, True), (40, 384, 16, 4, 64, FP, True, False),
    (96, 300, 8, 4, 80, FP, False, True), (2, 2048, 16, 8, 64, BF, True, False)])
def test_bias_gradient_on_a_full_device(d2p, cuda_device, B, L, H, Hkv, D, dtype, causal, ragged):  # noqa: F811
    """A CTA sums several items, in order of their work: all outputs of all problems against the reference."""
    q, k, v, do, bias = inputs(B, L, L, H, Hkv, D, dtype, cuda_device, 32, seed=B, bias_dtype=torch.float32)
    lengths = None
    if ragged:
        ls = [(7 * b * L) // (8 * B) for b in range(B)]
        lengths = torch.tensor([[x, min(L, x + b % 3)] for b, x in enumerate(ls)], dtype=torch.int32, device=cuda_device)
    val, tol = reference(q, k, v, bias, lengths, causal, D ** -0.5, 128, do)
    compare(run_attention(d2p, q, k, v, do, bias, lengths, causal), val, tol)
