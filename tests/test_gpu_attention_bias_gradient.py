"""The bias table's gradient: buckets of no weight."""
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
