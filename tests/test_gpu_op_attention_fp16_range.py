"""Attention's gradients in fp16 from small and from large gradients of the output: what is formed on the way has its own
exponent, so that only the results' rounding is fp16's.  Tolerances: tests/test_gpu_encoder.py's, whose terms scale with the
gradient, half the spacing of fp16's subnormals for the results, and nothing absolute beside it."""
import math

import pytest
import torch

from tests.test_gpu_encoder import TINY, d2p, inputs, reference, run_attention  # noqa: F401  (d2p: fixture)

pytestmark = pytest.mark.gpu
FP = torch.float16


def held(got, val, tol, names):
    for n in names:
        assert torch.isfinite(got[n]).all(), (n, "not finite")
        bad = (got[n].double() - val[n]).abs() > tol[n] + 1.01 * TINY[got[n].dtype]
        assert not bad.any(), (n, int(bad.sum()), bad.nonzero()[:3].tolist())


@pytest.mark.parametrize("small", [2.0 ** -10, 2.0 ** -16])
@pytest.mark.parametrize("B,Lq,Lk,H,Hkv,D,causal,nb,lens", [
    (2, 500, 500, 4, 2, 64, False, 0, [[500, 500], [130, 400]]), (1, 300, 900, 4, 4, 128, False, 16, None),
    (2, 400, 400, 2, 1, 80, True, 16, [[400, 400], [399, 17]]), (48, 300, 300, 16, 16, 64, True, 16, None)])
def test_small_gradients(d2p, cuda_device, B, Lq, Lk, H, Hkv, D, causal, nb, lens, small):  # noqa: F811
    """The problems' gradients differ in size, as far as `small`; a CTA takes several of them where there are many."""
    q, k, v, do, bias = inputs(B, Lq, Lk, H, Hkv, D, FP, cuda_device, nb, seed=D, bias_dtype=torch.float32)
    do[0] *= small
    do[-1] *= small
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    got = run_attention(d2p, q, k, v, do, bias, lengths, causal)
    picked = sorted({0, B // 2, B - 1}) if B > 4 else list(range(B))
    val, tol = reference(q[picked], k[picked], v[picked], bias, None if lens is None else lengths[picked], causal, 1 / math.sqrt(D), 128, do[picked])
    held({n: x[picked] if n != "dbias" else x for n, x in got.items()}, val, tol, ["out", "dq", "dk", "dv"] + (["dbias"] if nb and B <= 4 else []))


@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 64), (4, 2, 128)])
def test_large_gradients(d2p, cuda_device, H, Hkv, D):  # noqa: F811
    """dO V^T beyond 65504, the results within it."""
    q, k, v, do, _ = inputs(2, 16, 16, H, Hkv, D, FP, cuda_device)
    v, do = v * 60, do * 300
    val, tol = reference(q, k, v, None, None, False, 0.01, 128, do)
    assert val["dq"].abs().max() < 60000 and val["dk"].abs().max() < 60000
    got = run_attention(d2p, q, k, v, do, None, None, False, scale=0.01)
    held(got, val, tol, ["out", "dq", "dk", "dv"])


def test_gradients_of_nothing_and_of_nan(d2p, cuda_device):  # noqa: F811
    """A gradient of zeros gives zeros; one problem's NaN stays there."""
    q, k, v, do, _ = inputs(2, 150, 170, 4, 2, 64, FP, cuda_device)
    got = run_attention(d2p, q, k, v, do * 0, None, None, False)
    assert not any(got[n].any() for n in ("dq", "dk", "dv"))
    clean = run_attention(d2p, q, k, v, do, None, None, False)
    do[1, 3, 0, 5] = math.nan
    got = run_attention(d2p, q, k, v, do, None, None, False)
    for n in ("dq", "dk", "dv"):
        assert torch.equal(got[n][0], clean[n][0]) and torch.isnan(got[n][1]).any(), n
