"""The encoder operators (d2p_b200/csrc/enc_*.cu) on the GPU against 64-bit evaluations.

attention: the reference is the definition in fp64 with its gradients by formula.  Tolerances, per entry, from
the roundings the operator makes (u: half a unit of the inputs' type, 2^-8 for bf16 and 2^-11 for fp16):
the output is rounded once (u |o|) and the probabilities are rounded before their product (u sum p |v|);
dS is rounded before its products (u |dS|) and takes delta = sum dO o from the rounded output
(p u sum |dO| |o|).  F32 of the same magnitudes covers fp32 sums and exponentials: scores of size up to ~30 in
fp32 are off by 2^-23 * 30 * 2 ~ 7e-6 relative in p.
The gradients' formulas are themselves checked against central differences in fp64.
"""
import ctypes
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = 2e-5
# half the spacing of a type's subnormals: the least an entry's rounding is off by
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def d2p(cuda_device):
    import d2p_b200

    return d2p_b200


def bucket_table(nb, max_distance, two_sided, far):
    """bucket[d + far] of d in [-far, far], from the definition in whole numbers."""
    side = nb // 2 if two_sided else nb
    e = side // 2
    c = side - e

    def one(n):
        if n < e:
            return n
        t = 0
        n = min(n, max_distance)
        while t + 1 < c and n ** c * e ** (t + 1) >= max_distance ** (t + 1) * e ** c:
            t += 1
        return e + t

    return torch.tensor([(one(-d) if d <= 0 else (side + one(d) if two_sided else one(0))) for d in range(-far, far + 1)])


def reference(q, k, v, bias, lengths, causal, scale, max_distance, grad=None):
    """fp64 outputs and, with grad, gradients; each with the magnitudes its tolerance is made of."""
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    dev = q.device
    names = ["out"] + (["dq", "dk", "dv"] + (["dbias"] if bias is not None else []) if grad is not None else [])
    shapes = {"out": q.shape, "dq": q.shape, "dk": k.shape, "dv": v.shape}
    if bias is not None:
        shapes["dbias"] = bias.shape
    val = {n: torch.zeros(shapes[n], dtype=torch.float64, device=dev) for n in names}
    tol = {n: torch.zeros(shapes[n], dtype=torch.float64, device=dev) for n in names}
    u = U[q.dtype]
    far = Lq + Lk
    table = bucket_table(bias.shape[0], max_distance, not causal, far).to(dev) if bias is not None else None
    for b in range(B):
        lq, lk = (Lq, Lk) if lengths is None else (int(lengths[b, 0]), int(lengths[b, 1]))
        if lq == 0 or lk == 0:
            continue
        Q, K, V = q[b, :lq].double(), k[b, :lk].double().repeat_interleave(G, 1), v[b, :lk].double().repeat_interleave(G, 1)
        rel = torch.arange(lk, device=dev)[None] - torch.arange(lq, device=dev)[:, None] - (lk - lq if causal else 0)
        s = torch.einsum("ihd,jhd->hij", Q, K) * scale
        if bias is not None:
            bu = table[rel + far]
            s = s + bias.double()[bu].permute(2, 0, 1)
        if causal:
            s = torch.where(rel > 0, -math.inf, s)
        m = s.amax(-1, keepdim=True)
        e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
        l = e.sum(-1, keepdim=True)
        p = e / torch.where(l == 0, 1.0, l)
        o = torch.einsum("hij,jhd->ihd", p, V)
        mag = torch.einsum("hij,jhd->ihd", p, V.abs())
        val["out"][b, :lq] = o
        tol["out"][b, :lq] = u * o.abs() + (1.02 * u + F32) * mag
        if grad is None:
            continue
        g = grad[b, :lq].double()
        dp = torch.einsum("ihd,jhd->hij", g, V)
        delta = (g * o).sum(-1).t()[..., None]
        ds = p * (dp - delta)
        # |dS error|: its rounding, delta from the rounded output, fp32 of the magnitudes
        slack = (g.abs() * (mag * (2 * u + F32))).sum(-1).t()[..., None]
        gmag = torch.einsum("ihd,jhd->hij", g.abs(), V.abs())
        raw = p * slack + F32 * p * (gmag + delta.abs())
        es = 1.02 * u * ds.abs() + raw
        dq = torch.einsum("hij,jhd->ihd", ds, K) * scale
        val["dq"][b, :lq] = dq
        tol["dq"][b, :lq] = u * dq.abs() + 1.02 * torch.einsum("hij,jhd->ihd", es, K.abs()) * scale
        dk = torch.einsum("hij,ihd->jhd", ds, Q) * scale
        ek = 1.02 * torch.einsum("hij,ihd->jhd", es, Q.abs()) * scale
        dv = torch.einsum("hij,ihd->jhd", p, g)
        ev = (1.02 * u + F32) * torch.einsum("hij,ihd->jhd", p, g.abs())
        for n, x, ex in (("dk", dk, ek), ("dv", dv, ev)):
            x, ex = x.reshape(lk, Hkv, G, D).sum(2), ex.reshape(lk, Hkv, G, D).sum(2)
            val[n][b, :lk] = x
            tol[n][b, :lk] = u * x.abs() + ex
        if bias is not None:
            flat = bu.reshape(-1)
            val["dbias"].index_add_(0, flat, ds.permute(1, 2, 0).reshape(-1, H))
            tol["dbias"].index_add_(0, flat, (raw + F32 * ds.abs()).permute(1, 2, 0).reshape(-1, H))
    if grad is not None and bias is not None:
        tol["dbias"] += U[bias.dtype] * val["dbias"].abs()
    return val, tol


def inputs(B, Lq, Lk, H, Hkv, D, dtype, dev, nb=0, seed=0, bias_dtype=None):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(B, Lq, H, D, generator=g).to(dtype).to(dev)
    k = torch.randn(B, Lk, Hkv, D, generator=g).to(dtype).to(dev)
    v = torch.randn(B, Lk, Hkv, D, generator=g).to(dtype).to(dev)
    do = torch.randn(B, Lq, H, D, generator=g).to(dtype).to(dev)
    bias = torch.randn(nb, H, generator=g).to(bias_dtype or dtype).to(dev) if nb else None
    return q, k, v, do, bias


def compare(got, val, tol):
    for n, x in got.items():
        assert torch.isfinite(x).all(), (n, "not finite")
        err = (x.double() - val[n]).abs()
        bad = err > tol[n] + 1e-7
        assert not bad.any(), (n, int(bad.sum()), float((err / (tol[n] + 1e-7)).max()), bad.nonzero()[:4].tolist())


def run_attention(d2p, q, k, v, do, bias, lengths, causal, max_distance=128, scale=None):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (q, k, v, bias)]
    out = d2p.attention(*leaves[:3], bias=leaves[3], lengths=lengths, causal=causal, max_distance=max_distance, scale=scale)
    out.backward(do)
    got = {"out": out.detach(), "dq": leaves[0].grad, "dk": leaves[1].grad, "dv": leaves[2].grad}
    if bias is not None:
        got["dbias"] = leaves[3].grad
    return got


BF, FP = torch.bfloat16, torch.float16
CASES = [
    # B, Lq, Lk, H, Hkv, D, dtype, causal, buckets, max_distance, lengths
    (1, 1, 1, 1, 1, 8, BF, False, 0, 128, None),
    (2, 3, 5, 2, 1, 16, FP, True, 4, 16, None),
    (2, 100, 120, 4, 4, 64, BF, False, 32, 128, [[100, 120], [37, 3]]),
    (1, 128, 128, 2, 2, 64, BF, False, 0, 128, None),
    (2, 129, 65, 2, 1, 64, BF, True, 0, 128, None),               # queries past the keys: empty causal rows
    (3, 257, 193, 6, 3, 128, FP, False, 16, 64, [[257, 193], [0, 60], [131, 0]]),
    (2, 300, 300, 4, 2, 128, BF, True, 32, 200, [[300, 300], [300, 131]]),
    (1, 70, 1000, 2, 2, 40, BF, False, 32, 300, [[70, 999]]),
    (2, 513, 77, 4, 4, 80, FP, False, 8, 1000, [[513, 77], [385, 64]]),
    (1, 1000, 515, 2, 1, 32, BF, True, 64, 1024, None),
    (2, 640, 640, 3, 3, 64, BF, False, 32, 128, [[640, 600], [511, 640]]),
    (4, 16, 2000, 8, 1, 128, BF, True, 0, 128, None),
    (1, 200, 190, 1, 1, 120, FP, True, 2, 2, None),
]


@pytest.mark.parametrize("case", CASES, ids=["-".join(str(x).replace("torch.", "") for x in c[:9]) for c in CASES])
def test_attention_and_gradients(d2p, cuda_device, case):
    B, Lq, Lk, H, Hkv, D, dtype, causal, nb, md, lens = case
    q, k, v, do, bias = inputs(B, Lq, Lk, H, Hkv, D, dtype, cuda_device, nb, seed=Lq + Lk)
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda_device) if lens else None
    val, tol = reference(q, k, v, bias, lengths, causal, 1 / math.sqrt(D), md, do)
    compare(run_attention(d2p, q, k, v, do, bias, lengths, causal, md), val, tol)


SPLIT = [   # few rows and many keys: the keys split over CTAs, the splits' results joined
    (2, 40, 3000, 2, 1, 64, BF, True, 32, 128, [[40, 3000], [17, 700]]),
    (1, 130, 2500, 2, 2, 128, FP, False, 16, 64, [[130, 2100]]),
    (1, 300, 4000, 1, 1, 64, FP, True, 0, 128, None),
    (2, 90, 1030, 4, 4, 80, BF, False, 0, 128, [[90, 1030], [40, 1]]),
    (3, 1, 9000, 4, 2, 64, BF, True, 16, 200, [[1, 9000], [1, 300], [0, 5]]),
    (1, 2, 20000, 4, 1, 128, FP, False, 0, 128, None),
    (2, 1, 5000, 3, 3, 40, BF, True, 32, 64, [[1, 4999], [1, 0]]),
]


@pytest.mark.parametrize("case", SPLIT, ids=["-".join(str(x).replace("torch.", "") for x in c[:9]) for c in SPLIT])
def test_attention_split_keys(d2p, cuda_device, case):
    B, Lq, Lk, H, Hkv, D, dtype, causal, nb, dist, lengths = case
    q, k, v, do, bias = inputs(B, Lq, Lk, H, Hkv, D, dtype, cuda_device, nb, seed=Lk)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    if lengths is not None:
        for b, (lq, lk) in enumerate(lengths):   # what lies outside is never used
            q[b, lq:], do[b, lq:], k[b, lk:], v[b, lk:] = math.nan, math.nan, math.inf, math.nan
    val, tol = reference(q, k, v, bias, ln, causal, D ** -0.5, dist, do)
    got = run_attention(d2p, q, k, v, do, bias, ln, causal, dist)
    compare(got, val, tol)
    alone = d2p.attention(q, k, v, bias=bias, lengths=ln, causal=causal, max_distance=dist)
    compare({"out": alone}, val, tol)
    assert torch.equal(alone, d2p.attention(q, k, v, bias=bias, lengths=ln, causal=causal, max_distance=dist))


def test_reference_gradients_by_differences(cuda_device):
    """The fp64 formulas the gradients are judged by, against central differences of the fp64 output."""
    q, k, v, do, bias = inputs(1, 6, 7, 2, 1, 8, torch.bfloat16, cuda_device, 8, seed=3)
    val, _ = reference(q, k, v, bias, None, False, 0.4, 16, do)
    base = {"dq": q, "dk": k, "dv": v, "dbias": bias}
    for name, arg in (("dq", 0), ("dk", 1), ("dv", 2), ("dbias", 3)):
        for at in (0, 5, 11):
            side = []
            for sign in (1, -1):
                args = [t.double() for t in (q, k, v, bias)]
                args[arg].view(-1)[at] += sign * 1e-5
                U64 = U.setdefault(torch.float64, 2.0 ** -53)
                assert U64
                o = reference(*args, None, False, 0.4, 16)[0]["out"]
                side.append(float((o * do.double()).sum()))
            want = float(val[name].view(-1)[at])
            assert abs((side[0] - side[1]) / 2e-5 - want) < 1e-6 * max(1.0, abs(want)), (name, at, base[name].shape)


@pytest.mark.parametrize("Lq,G", [(1, 1), (1, 8), (2, 4), (1, 16), (5, 3)])
@pytest.mark.parametrize("Lk", [1, 63, 64, 65, 700, 4111])
def test_attention_few_queries(d2p, cuda_device, Lq, G, Lk):
    """Serving's forms: one or a few query rows over a cache, no gradient."""
    for dtype, D, nb, causal in ((torch.bfloat16, 64, 32, True), (torch.float16, 128, 0, True), (torch.bfloat16, 80, 32, False)):
        q, k, v, _, bias = inputs(3, Lq, Lk, 2 * G, 2, D, dtype, cuda_device, nb, seed=Lk)
        lengths = torch.tensor([[Lq, Lk], [min(1, Lq), (Lk + 1) // 2], [Lq, 0]], dtype=torch.int32, device=cuda_device)
        val, tol = reference(q, k, v, bias, lengths, causal, 1 / math.sqrt(D), 128)
        compare({"out": d2p.attention(q, k, v, bias=bias, lengths=lengths, causal=causal)}, val, tol)


@pytest.mark.parametrize("Lq,Lk", [(1, 300), (200, 210)])
def test_attention_ignores_what_lies_outside(d2p, cuda_device, Lq, Lk):
    """NaN and infinities past the lengths, in every input and in the output's gradient, change nothing; rows and
    gradients there are exact zeros."""
    q, k, v, do, bias = inputs(3, Lq, Lk, 4, 2, 64, torch.bfloat16, cuda_device, 16)
    lens = [[Lq, Lk - 7], [max(1, Lq - 70), 130], [0, 5]]
    lengths = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    clean = run_attention(d2p, q, k, v, do, bias, lengths, False)
    plain = d2p.attention(q, k, v, bias=bias, lengths=lengths)
    for b, (lq, lk) in enumerate(lens):
        q[b, lq:], do[b, lq:] = math.nan, math.inf
        k[b, lk:], v[b, lk:] = math.inf, math.nan
        if lq == 0:
            k[b], v[b] = math.nan, math.nan
    dirty = run_attention(d2p, q, k, v, do, bias, lengths, False)
    for n in clean:
        assert torch.equal(clean[n], dirty[n]), n
    for b, (lq, lk) in enumerate(lens):
        assert not clean["out"][b, lq:].any() and not clean["dq"][b, lq:].any()
        assert not clean["dk"][b, lk:].any() and not clean["dv"][b, lk:].any()
    assert torch.equal(plain, d2p.attention(q, k, v, bias=bias, lengths=lengths))


@pytest.mark.parametrize("Lq", [1, 150])
def test_attention_extreme_bias(d2p, cuda_device, Lq):
    """A bucket of -inf masks its keys, a table of lowest values leaves the row uniform, all -inf leaves zeros."""
    q, k, v, do, bias = inputs(1, Lq, 150, 2, 2, 64, torch.bfloat16, cuda_device, 8)
    b1 = bias.clone()
    b1[0], b1[3] = -math.inf, -math.inf
    val, tol = reference(q, k, v, b1, None, False, 0.125, 16, do)
    got = run_attention(d2p, q, k, v, do, b1, None, False, 16)
    compare(got, val, tol)
    low = torch.full_like(bias, torch.finfo(torch.bfloat16).min)
    out = d2p.attention(q, k, v, bias=low)
    mean = v.double().mean(1, keepdim=True).expand(1, Lq, 2, 64)
    mag = v.double().abs().mean(1, keepdim=True)
    assert ((out.double() - mean).abs() <= 2.0 ** -8 * mean.abs() + (2.0 ** -7 + F32) * mag).all()
    got = run_attention(d2p, q, k, v, do, torch.full_like(bias, -math.inf), None, False)
    for n in ("out", "dq", "dk", "dv", "dbias"):
        assert not got[n].any(), n


@pytest.mark.parametrize("scale", [40.0, 1e-4])
def test_attention_score_range(d2p, cuda_device, scale):
    """Scores in the thousands (one key takes the row) and near zero.  The fp32 scores are off by 2^-23 of their
    size, so a probability by up to 2^-22 * 40 * 64 * ln-units: the tolerance grows by that much of the magnitudes."""
    q, k, v, do, _ = inputs(1, 130, 140, 2, 2, 64, torch.float16, cuda_device)
    val, tol = reference(q, k, v, None, None, False, scale, 128, do)
    size = float((torch.einsum("bihd,bjhd->bhij", q.double().abs(), k.double().abs()) * scale).max())
    more = 1 + size * 2.0 ** -21 / F32
    got = run_attention(d2p, q, k, v, do, None, None, False, scale=scale)
    mag = {n: x.abs().max() for n, x in val.items()}
    compare(got, val, {n: t * more + 2.0 ** -21 * size * mag[n] for n, t in tol.items()})


def test_bias_gradient_of_cancelling_buckets(d2p, cuda_device):
    """Nearly all the weight in the last bucket: its dS sum to what the others' leave, far below their terms, and an
    error of a row's delta would show there whole.  fp32 table, so nothing rounds the result.  The 1280 rows' deltas from
    an output rounded to bf16 are off by about 2^-9 |dO||o| / 8 each, independently: sqrt(1280) 2^-9 of a term together,
    some 7 %; with out's rest kept 2^-17 of it, and what is left are fp32's 1e-6 of the terms: 1e-3 allowed."""
    q, k, v, do, bias = inputs(2, 640, 640, 4, 4, 64, torch.bfloat16, cuda_device, 16, seed=8, bias_dtype=torch.float32)
    bias = bias * 0
    bias[15] = 6.0
    val, _ = reference(q, k, v, bias, None, True, 0.125, 16, do)
    got = run_attention(d2p, q, k, v, do, bias, None, True, 16)["dbias"].double()
    scale = val["dbias"].abs().amax(0)
    assert ((got - val["dbias"]).abs() <= 1e-3 * scale).all(), ((got - val["dbias"]).abs() / scale).max()


def test_attention_strided_views(d2p, cuda_device):
    """Heads inside one projection, head-major storage, an odd offset (copied) and an expanded gradient."""
    g = torch.Generator().manual_seed(5)
    for off in (0, 1):
        flat = torch.randn(2 * 90 * 8 * 64 + 8, generator=g).to(torch.bfloat16).to(cuda_device)
        qkv = flat[off:off + 2 * 90 * 8 * 64].view(2, 90, 8, 64)
        q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
        a = run_attention(d2p, q, k, v, torch.ones(1, device=cuda_device, dtype=torch.bfloat16).expand(2, 90, 4, 64), None, None, True)
        c = [t.clone(memory_format=torch.contiguous_format) for t in (q, k, v)]
        b = run_attention(d2p, *c, torch.ones(2, 90, 4, 64, device=cuda_device, dtype=torch.bfloat16), None, None, True)
        for n in a:
            assert torch.equal(a[n], b[n]), (off, n)
    major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in c]
    out = d2p.attention(*major, causal=True)
    assert torch.equal(out, d2p.attention(*c, causal=True))


def test_attention_of_broadcast_inputs(d2p, cuda_device):
    """Keys and values expanded over the batch and over heads: copied, and their gradients summed where they came from."""
    q, k, v, do, bias = inputs(3, 70, 90, 4, 2, 64, torch.bfloat16, cuda_device, 8)
    k1, v1 = k[:1, :, :1].clone().requires_grad_(True), v[:1, :, :1].clone().requires_grad_(True)
    d2p.attention(q, k1.expand_as(k), v1.expand_as(v), bias=bias.clone().requires_grad_(True)).backward(do)   # (as below)
    got = run_attention(d2p, q, k1.detach().expand_as(k).contiguous(), v1.detach().expand_as(v).contiguous(), do, bias, None, False)
    for leaf, name in ((k1, "dk"), (v1, "dv")):   # (a sum of six bf16 terms, itself rounded once or per axis)
        want = got[name].double().sum((0, 2), keepdim=True)
        mag = got[name].double().abs().sum((0, 2), keepdim=True)
        assert ((leaf.grad.double() - want).abs() <= 2 * U[torch.bfloat16] * mag + 1e-7).all()


def test_second_derivatives(d2p, cuda_device):
    """Attention's and the norms' gradients say that they are not differentiable; dropout's is the operator itself."""
    q, k, v, do, _ = inputs(1, 20, 20, 2, 2, 64, torch.bfloat16, cuda_device)
    leaf = q.clone().requires_grad_(True)
    (dq,) = torch.autograd.grad(d2p.attention(leaf, k, v), leaf, do, create_graph=True)
    assert torch.equal(dq.detach(), run_attention(d2p, q, k, v, do, None, None, False)["dq"])
    with pytest.raises(RuntimeError, match="differentiated again"):
        dq.float().sum().backward()
    w, ang = torch.ones(64, device=cuda_device), torch.rand(20, 32, device=cuda_device)
    (dq,) = torch.autograd.grad(d2p.qk_norm_rope(leaf, k, w.bfloat16(), w.bfloat16(), ang.cos(), ang.sin())[0], leaf, do, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        dq.float().sum().backward()
    x, g = torch.randn(999, device=cuda_device, requires_grad=True), torch.randn(999, device=cuda_device, requires_grad=True)
    y = d2p.dropout_add(x, None, 0.3, 5)
    (dx,) = torch.autograd.grad(y, x, g, create_graph=True)
    (dg,) = torch.autograd.grad(dx, g, x.detach())
    assert torch.equal(dg, y.detach())


def test_attention_is_repeatable(d2p, cuda_device):
    q, k, v, do, bias = inputs(4, 500, 480, 4, 2, 64, torch.bfloat16, cuda_device, 32)
    a = run_attention(d2p, q, k, v, do, bias, None, False)
    for _ in range(3):
        b = run_attention(d2p, q, k, v, do, bias, None, False)
        for n in a:
            assert torch.equal(a[n], b[n]), n


@pytest.mark.parametrize("B,L,H,Hkv,D,causal,ragged", [
    (2, 2048, 16, 4, 128, True, False), (1, 4096, 8, 8, 128, False, False), (2, 2048, 16, 16, 64, True, False),
    (64, 512, 8, 2, 128, True, True), (64, 512, 8, 8, 64, False, True), (96, 300, 8, 4, 80, False, True)])
def test_attention_on_a_full_device_is_repeatable(d2p, cuda_device, B, L, H, Hkv, D, causal, ragged):
    """Enough work for CTAs to take several row tiles, and for every wait to matter: the same bits again and again."""
    q, k, v, do, bias = inputs(B, L, L, H, Hkv, D, torch.bfloat16, cuda_device, 32, seed=B)
    lengths = None
    if ragged:
        ls = [(7 * b * L) // (8 * B) for b in range(B)]
        lengths = torch.tensor([[x, min(L, x + b % 3)] for b, x in enumerate(ls)], dtype=torch.int32, device=cuda_device)
    a = run_attention(d2p, q, k, v, do, bias, lengths, causal)
    for _ in range(8):
        b = run_attention(d2p, q, k, v, do, bias, lengths, causal)
        for n in a:
            assert torch.equal(a[n], b[n]), n
    picked = [0, B // 2, B - 1]
    part = lengths[picked] if ragged else None
    val, tol = reference(q[picked], k[picked], v[picked], bias, part, causal, D ** -0.5, 128, do[picked])
    compare({n: a[n][picked] for n in ("out", "dq", "dk", "dv")}, val, tol)


def test_attention_float32_bias_and_out_of_range_lengths(d2p, cuda_device):
    q, k, v, do, bias = inputs(2, 140, 150, 2, 2, 64, torch.bfloat16, cuda_device, 32, bias_dtype=torch.float32)
    wild = torch.tensor([[1000, 1000], [-3, 4]], dtype=torch.int32, device=cuda_device)
    held = torch.tensor([[140, 150], [0, 4]], dtype=torch.int32, device=cuda_device)
    val, tol = reference(q, k, v, bias, held, False, 0.125, 128, do)
    got = run_attention(d2p, q, k, v, do, bias, wild, False)
    assert got["dbias"].dtype == torch.float32
    compare(got, val, tol)


@pytest.mark.parametrize("shape", [(0, 4, 4), (2, 0, 4), (2, 4, 0), (0, 0, 0)])
def test_attention_empty_axes(d2p, cuda_device, shape):
    B, Lq, Lk = shape
    q, k, v, do, bias = inputs(B, Lq, Lk, 2, 1, 64, torch.bfloat16, cuda_device, 8)
    got = run_attention(d2p, q, k, v, do, bias, None, False)
    for n, x in got.items():
        assert not x.any(), n
    assert got["out"].shape == q.shape and got["dbias"].shape == bias.shape


def test_attention_long_cache_offsets(d2p, cuda_device):
    """A cache whose later problems lie past 2^31 elements."""
    B, Lk, Hkv, D = 3, 1 << 20, 8, 128
    k = torch.empty(B, Lk, Hkv, D, dtype=torch.bfloat16, device=cuda_device)
    v = torch.empty_like(k)
    g = torch.Generator().manual_seed(1)
    tail = torch.randn(2, 500, Hkv, D, generator=g).to(torch.bfloat16).to(cuda_device)
    k[2, :500], v[2, :500] = tail[0], tail[1]
    k[1, -500:], v[1, -500:] = tail[0], tail[1]
    q = torch.randn(B, 1, 16, D, generator=g).to(torch.bfloat16).to(cuda_device)
    lengths = torch.tensor([[0, 0], [0, 0], [1, 500]], dtype=torch.int32, device=cuda_device)
    out = d2p.attention(q, k, v, lengths=lengths, causal=True)
    want = d2p.attention(q[2:], tail[:1], tail[1:], causal=True)
    assert torch.equal(out[2:], want)
    k[1, :-500], v[1, :-500] = 0, 0
    k[1, :-500, :, 0] = -100.0
    q[1] = 0
    q[1, :, :, 0] = 100.0
    lengths = torch.tensor([[0, 0], [1, Lk], [0, 0]], dtype=torch.int32, device=cuda_device)
    out = d2p.attention(q, k, v, lengths=lengths, causal=True)
    val, tol = reference(q[1:2], tail[:1], tail[1:], None, None, True, 1 / math.sqrt(D), 128)   # the others weigh e^-800
    compare({"out": out[1:2]}, val, tol)


def test_operators_on_another_stream(d2p, cuda_device):
    q, k, v, do, bias = inputs(2, 300, 300, 4, 2, 64, torch.bfloat16, cuda_device, 16)
    want = run_attention(d2p, q, k, v, do, bias, None, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_attention(d2p, q, k, v, do, bias, None, False)
        y = d2p.dropout_add(q, q, 0.3, 7)
    torch.cuda.current_stream().wait_stream(side)
    for n in want:
        assert torch.equal(want[n], got[n]), n
    assert torch.equal(y, d2p.dropout_add(q, q, 0.3, 7))


def test_operators_in_a_graph(d2p, cuda_device):
    q, k, v, _, bias = inputs(2, 1, 900, 4, 2, 64, torch.bfloat16, cuda_device, 16)
    lengths = torch.tensor([[1, 900], [1, 450]], dtype=torch.int32, device=cuda_device)
    w = torch.ones(64, device=cuda_device)
    ang = torch.rand(64, 32, device=cuda_device)

    def step():
        a, b = d2p.qk_norm_rope(q, q, w, w, ang.cos(), ang.sin())
        return d2p.dropout_add(d2p.attention(a, k, v, bias=bias, lengths=lengths, causal=True), b, 0.2, 3)

    want = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------- head norms with rotation
def rope_reference(x, w, cos, sin, pos, eps, g=None):
    R = 2 * cos.shape[1]
    x, w = x.double(), w.double()
    c, s = cos.double()[pos][:, :, None], sin.double()[pos][:, :, None]

    def turn(y, s):
        a, b = y[..., :R // 2], y[..., R // 2:R]
        return torch.cat([a * c - b * s, b * c + a * s, y[..., R:]], -1)

    def size(y):   # sum of the magnitudes of turn's terms
        a, b = y[..., :R // 2].abs(), y[..., R // 2:R].abs()
        return torch.cat([a * c.abs() + b * s.abs(), b * c.abs() + a * s.abs(), y[..., R:].abs()], -1)

    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    xh = x * r
    y, ymag = turn(xh * w, s), size(xh * w)
    if g is None:
        return y, ymag
    u = turn(g.double(), -s)
    umag = size(g.double())
    t = u * w
    dot = (t * xh).mean(-1, keepdim=True)
    dx = r * (t - xh * dot)
    dxmag = r * ((umag * w.abs()) + xh.abs() * (umag * w.abs() * xh.abs()).mean(-1, keepdim=True))
    return y, ymag, dx, dxmag, (u * xh).sum((0, 1, 2)), (umag * xh.abs()).sum((0, 1, 2))


ROPE = [
    # B, L, H, Hkv, D, R, dtype, weight dtype, positions
    (1, 1, 1, 1, 16, 16, torch.float32, torch.float32, None),
    (2, 7, 3, 1, 64, 64, torch.bfloat16, torch.bfloat16, "2d"),
    (3, 50, 4, 2, 128, 64, torch.float16, torch.float32, "1d"),
    (2, 33, 5, 5, 80, 32, torch.bfloat16, torch.float32, "int64"),
    (1, 200, 2, 1, 256, 256, torch.float32, torch.float32, "2d"),
    (2, 90, 8, 8, 32, 0, torch.float16, torch.float16, None),
    (16, 300, 4, 1, 48, 16, torch.bfloat16, torch.bfloat16, None),
]


@pytest.mark.parametrize("case", ROPE, ids=["-".join(str(x).replace("torch.", "") for x in c) for c in ROPE])
def test_qk_norm_rope(d2p, cuda_device, case):
    """Per entry: one rounding of the result (u) and fp32 sums of the magnitudes; a weight's gradient sums N rows
    in fp32 (partial sums of at most a few hundred rows, then of blocks): 1e-6 of the magnitudes per factor."""
    B, L, H, Hkv, D, R, dtype, wdt, how = case
    g = torch.Generator().manual_seed(L)
    P = 500
    qkv = (torch.randn(B, L, H + Hkv + 1, D, generator=g) * 2).to(dtype).to(cuda_device)
    q, k = qkv[:, :, :H].detach().requires_grad_(True), qkv[:, :, H:H + Hkv].detach().requires_grad_(True)
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=g)).to(wdt).to(cuda_device).requires_grad_(True) for _ in range(2))
    ang = torch.rand(P, R // 2, generator=g) * 100
    cos, sin = ang.cos().to(cuda_device), ang.sin().to(cuda_device)
    pos = torch.arange(L).expand(B, L)
    arg = None
    if how == "1d":
        arg = torch.randint(0, P, (L,), generator=g, dtype=torch.int32)
        pos = arg.long().expand(B, L)
    elif how:
        arg = torch.randint(0, P, (B, L), generator=g, dtype=torch.int64 if how == "int64" else torch.int32)
        pos = arg.long()
    yq, yk = d2p.qk_norm_rope(q, k, qw, kw, cos, sin, positions=None if arg is None else arg.to(cuda_device), eps=1e-5)
    gq, gk = (torch.randn(B, L, h, D, generator=g).to(dtype).to(cuda_device) for h in (H, Hkv))
    torch.autograd.backward((yq, yk), (gq, gk))
    u = U[dtype]
    for x, w, y, gr in ((q, qw, yq, gq), (k, kw, yk, gk)):
        ry, rm, rdx, rdm, rdw, rwm = rope_reference(x.detach(), w.detach(), cos, sin, pos.to(cuda_device), 1e-5, gr)
        assert ((y.double() - ry).abs() <= u * ry.abs() + 2e-6 * rm.abs() + 1e-7).all()
        assert ((x.grad.double() - rdx).abs() <= u * rdx.abs() + 4e-6 * rdm + 1e-7).all()
        assert ((w.grad.double() - rdw).abs() <= U[wdt] * rdw.abs() + 4e-6 * rwm + 1e-7).all()


def test_qk_norm_rope_gradient_by_differences():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, 2, 1, 16, generator=g).double()
    w = torch.rand(16, generator=g).double()
    ang = torch.rand(4, 4, generator=g)
    pos = torch.tensor([[3, 1]])
    gr = torch.randn(1, 2, 1, 16, generator=g)
    full = rope_reference(x, w, ang.cos(), ang.sin(), pos, 1e-5, gr)
    for at in (0, 6, 31):
        side = []
        for sign in (1, -1):
            xp = x.clone()
            xp.view(-1)[at] += sign * 1e-6
            side.append(float((rope_reference(xp, w, ang.cos(), ang.sin(), pos, 1e-5)[0] * gr.double()).sum()))
        assert abs((side[0] - side[1]) / 2e-6 - float(full[2].view(-1)[at])) < 1e-6


def test_qk_norm_rope_positions_are_held_in_the_table(d2p, cuda_device):
    q = torch.randn(1, 4, 2, 32, device=cuda_device)
    w = torch.ones(32, device=cuda_device)
    ang = torch.rand(10, 16, device=cuda_device)
    wild = torch.tensor([[-5, 3, 10, 1 << 30]], dtype=torch.int32, device=cuda_device)
    held = wild.clamp(0, 9)
    a = d2p.qk_norm_rope(q, q, w, w, ang.cos(), ang.sin(), positions=wild)
    b = d2p.qk_norm_rope(q, q, w, w, ang.cos(), ang.sin(), positions=held)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    e = d2p.qk_norm_rope(q[:, :0], q[:, :0], w, w, ang.cos(), ang.sin())
    assert e[0].shape == (1, 0, 2, 32)


@pytest.mark.parametrize("B,L,H,Hkv", [(1, 3, 2, 1), (2, 7, 3, 2), (40, 300, 6, 5)])
def test_qk_norm_rope_without_eps(d2p, cuda_device, B, L, H, Hkv):
    """With eps = 0 a group of threads without a row would divide by zero: the weights' gradients take nothing from it."""
    g = torch.Generator().manual_seed(L)
    D = 48
    x = [torch.randn(B, L, h, D, generator=g).to(torch.bfloat16).to(cuda_device).requires_grad_(True) for h in (H, Hkv)]
    w = [torch.rand(D, generator=g).to(cuda_device).requires_grad_(True) for _ in range(2)]
    ang = torch.rand(L, 8, generator=g).to(cuda_device)
    y = d2p.qk_norm_rope(*x, *w, ang.cos(), ang.sin(), eps=0.0)
    gr = [torch.randn(B, L, h, D, generator=g).to(torch.bfloat16).to(cuda_device) for h in (H, Hkv)]
    torch.autograd.backward(y, gr)
    pos = torch.arange(L, device=cuda_device).expand(B, L)
    for i in range(2):   # (tolerances: test_qk_norm_rope's)
        ref = rope_reference(x[i].detach(), w[i].detach(), ang.cos(), ang.sin(), pos, 0.0, gr[i])
        assert ((x[i].grad.double() - ref[2]).abs() <= U[torch.bfloat16] * ref[2].abs() + 4e-6 * ref[3] + 1e-7).all()
        assert ((w[i].grad.double() - ref[4]).abs() <= U[torch.float32] * ref[4].abs() + 4e-6 * ref[5] + 1e-7).all()


def test_qk_norm_rope_zero_rows_and_empty_batches(d2p, cuda_device):
    w = torch.ones(64, device=cuda_device, requires_grad=True)
    ang = torch.rand(10, 32, device=cuda_device)
    q = torch.zeros(2, 3, 2, 64, device=cuda_device, requires_grad=True)
    y, _ = d2p.qk_norm_rope(q, q, w, w, ang.cos(), ang.sin())
    assert not y.any()
    y.sum().backward()
    assert torch.isfinite(q.grad).all() and not w.grad.any()
    q = torch.zeros(0, 3, 2, 64, device=cuda_device, requires_grad=True)
    w2 = torch.ones(64, device=cuda_device, requires_grad=True)
    a, b = d2p.qk_norm_rope(q, q, w2, w2, ang.cos(), ang.sin())
    (a.sum() + b.sum()).backward()
    assert a.shape == q.shape and not w2.grad.any()


# ---------------------------------------------------------------------------- dropout
def philox_words(n, seed, offset):
    out = []
    for block in range((n + 3) // 4):
        c = [block & 0xFFFFFFFF, block >> 32, offset & 0xFFFFFFFF, offset >> 32]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        out += c
    return out[:n]


def test_philox_known_answers():
    """The published generator's known answers (Random123: philox4x32-10, zero counter and key)."""
    assert philox_words(4, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 7, 8, 1003, 40000])
def test_dropout_add(d2p, cuda_device, dtype, n):
    g = torch.Generator().manual_seed(n)
    p, seed, offset = 0.3, (1 << 61) + 12345, (1 << 40) + 3
    x = torch.randn(n, generator=g).to(dtype).to(cuda_device).requires_grad_(True)
    r = torch.randn(n, generator=g).to(dtype).to(cuda_device).requires_grad_(True)
    go = torch.randn(n, generator=g).to(dtype).to(cuda_device)
    y = d2p.dropout_add(x, r, p, seed, offset)
    y.backward(go)
    keep = torch.tensor([w >= int(p * 2 ** 32) for w in philox_words(n, seed, offset)], device=cuda_device)
    want = r.detach().double() + torch.where(keep, x.detach().double() / (1 - p), 0.0)
    mag = r.detach().double().abs() + x.detach().double().abs() / (1 - p)
    u = U[dtype]
    assert ((y.detach().double() - want).abs() <= u * want.abs() + 2.0 ** -22 * mag).all()
    dx = torch.where(keep, go.double() / (1 - p), 0.0)
    assert ((x.grad.double() - dx).abs() <= (u + 2.0 ** -22) * dx.abs() + TINY[dtype]).all()
    assert torch.equal(x.grad != 0, keep & (go != 0)) and torch.equal(r.grad, go)
    plain = d2p.dropout_add(x.detach(), None, p, seed, offset)
    assert torch.equal(plain != 0, keep & (x.detach() != 0))


def test_dropout_rate_and_edges(d2p, cuda_device):
    x = torch.ones(1 << 20, device=cuda_device)
    for p in (0.0, 0.1, 0.5, 0.999):
        kept = float((d2p.dropout_add(x, None, p, 11) != 0).double().mean())
        assert abs(kept - (1 - p)) <= 5 * math.sqrt(p * (1 - p) / x.numel()) + 1e-9
    assert not torch.equal(d2p.dropout_add(x, None, 0.5, 11, 0), d2p.dropout_add(x, None, 0.5, 11, 1))
    bad = torch.full((64,), math.nan, device=cuda_device)
    y = d2p.dropout_add(bad, torch.zeros_like(bad), 0.5, 4)
    keep = torch.tensor([w >= 1 << 31 for w in philox_words(64, 4, 0)], device=cuda_device)
    assert torch.equal(torch.isnan(y), keep)   # a dropped NaN is gone
    assert d2p.dropout_add(x[:0], None, 0.5, 1).numel() == 0
    # a view at an odd offset, and a transposed one: elements count in row-major order
    odd = torch.randn(1025, device=cuda_device).to(torch.bfloat16)
    assert torch.equal(d2p.dropout_add(odd[1:], odd[1:], 0.4, 9), d2p.dropout_add(odd[1:].clone(), odd[1:].clone(), 0.4, 9))
    m = torch.randn(30, 50, device=cuda_device)
    assert torch.equal(d2p.dropout_add(m.t(), None, 0.4, 9), d2p.dropout_add(m.t().contiguous(), None, 0.4, 9))


def test_no_wait_gave_up(d2p, cuda_device):
    """Every bounded wait of the attention kernels so far in this process ended by what it waited for."""
    q, k, v, do, bias = inputs(2, 300, 300, 4, 2, 64, torch.bfloat16, cuda_device, 16)
    run_attention(d2p, q, k, v, do, bias, None, False)
    torch.cuda.synchronize()
    lib = ctypes.CDLL(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "d2p_b200", "libd2p_b200.so"))
    n = ctypes.c_ulonglong(77)
    lib.d2p_attention_gave_up.restype = ctypes.c_int
    lib.d2p_attention_gave_up.argtypes = [ctypes.POINTER(ctypes.c_ulonglong)]
    assert lib.d2p_attention_gave_up(ctypes.byref(n)) == 0
    assert n.value == 0


# ---------------------------------------------------------------------------- the C ABI's refusals, the kernels that run
def test_c_abi_refuses(cuda_device):
    lib = ctypes.CDLL(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "d2p_b200", "libd2p_b200.so"))
    f = lib.d2p_dropout_add
    f.restype = ctypes.c_int
    f.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_ulonglong, ctypes.c_double,
                  ctypes.c_ulonglong, ctypes.c_ulonglong, ctypes.c_void_p, ctypes.c_void_p]
    x = torch.zeros(8, device=cuda_device)
    assert f(x.data_ptr(), None, 0, 8, 1.0, 0, 0, x.data_ptr(), None) == 1001
    assert f(x.data_ptr(), None, 0, 8, math.nan, 0, 0, x.data_ptr(), None) == 1001
    assert f(x.data_ptr(), None, 5, 8, 0.5, 0, 0, x.data_ptr(), None) == 1001
    assert f(None, None, 0, 8, 0.5, 0, 0, x.data_ptr(), None) == 1001
    assert f(None, None, 0, 0, 0.5, 0, 0, None, None) == 0


def test_operators_refuse(d2p, cuda_device):
    q, k, v, _, bias = inputs(1, 8, 8, 4, 2, 64, torch.bfloat16, cuda_device, 8)
    op = torch.ops.d2p_b200.attention_forward
    for args in ((q.cpu(), k, v, None, None, [], 1.0, False, False, False),
                 (q, k, v, bias, None, [1, 2], 1.0, False, False, False),          # edges for another number of buckets
                 (q, k, v, bias, None, [3, 2, 1], 1.0, False, False, False),       # edges that fall
                 (q, k, v, bias, None, [1, 2, 5000], 1.0, False, False, False),    # past the reach
                 (q, k, v, None, None, [], -1.0, False, False, False),
                 (q, k, v, None, torch.zeros(1, 2, device=cuda_device), [], 1.0, False, False, False)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            op(*args)
    with pytest.raises(RuntimeError):
        torch.ops.d2p_b200.dropout_add(q, q.float(), 0.1, 1, 0)


def test_example_trains(cuda_device):
    """examples/encode_align.py: the four operators and the alignment in one training loop."""
    import importlib.util

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "encode_align.py")
    spec = importlib.util.spec_from_file_location("encode_align", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    losses = module.train(60, report=None)
    assert all(math.isfinite(x) for x in losses) and sum(losses[-10:]) < 0.5 * sum(losses[:10])
