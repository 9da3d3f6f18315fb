"""The encoder operators' host side, without a GPU: bucket edges, refusals, shapes of fake tensors, the C ABI's checks."""
import ctypes
import math
import os

import pytest
import torch

import d2p_b200 as d2p

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF = torch.bfloat16


@pytest.fixture(scope="module")
def lib():
    return ctypes.CDLL(os.path.join(ROOT, "d2p_b200", "libd2p_b200.so"))


# ---------------------------------------------------------------- buckets
@pytest.mark.parametrize("nb,md,two", [(32, 128, True), (16, 64, True), (32, 200, False), (4, 16, False), (64, 1024, False),
                                       (2, 2, False), (8, 1000, True), (8, 5, True)])
def test_bucket_edges_are_the_definition(nb, md, two):
    """Every distance's bucket by its edges against the definition with exact whole-number comparisons, and with
    logarithms in fp64 wherever these are not within 1e-9 of a whole number."""
    edges = d2p.relative_bucket_edges(nb, md, two)
    side = nb // 2 if two else nb
    e, c = side // 2, side - side // 2
    assert len(edges) == side - 1 and list(edges) == sorted(edges)
    for n in range(md + 5):
        got = sum(x <= n for x in edges)
        if n < e:
            assert got == n
            continue
        whole = max(t for t in range(c) if n ** c * e ** t >= md ** t * e ** c)
        assert got == e + whole, n
        real = math.log(n / e) / math.log(md / e) * c
        if abs(real - round(real)) > 1e-9:
            assert got == min(e + int(real), side - 1), n


def test_bucket_edges_refuse():
    for args in ((7, 128, True), (2, 128, True), (1, 128, False), (130, 128, True), (66, 128, False), (32, 8, True), (32, 1025, True)):
        with pytest.raises(ValueError):
            d2p.relative_bucket_edges(*args)


# ---------------------------------------------------------------- refusals before any launch
def test_attention_refuses():
    q, k = torch.zeros(2, 5, 4, 64, dtype=BF), torch.zeros(2, 7, 2, 64, dtype=BF)
    with pytest.raises(TypeError, match="bfloat16"):
        d2p.attention(q.float(), k.float(), k.float())
    with pytest.raises(TypeError, match="bfloat16"):
        d2p.attention(q, k.half(), k)
    with pytest.raises(ValueError, match="must be"):
        d2p.attention(q, k, k[:, :6])
    with pytest.raises(ValueError, match="must be"):
        d2p.attention(q[0], k, k)
    with pytest.raises(ValueError, match="multiple"):
        d2p.attention(q[:, :, :3], k, k)
    with pytest.raises(ValueError, match="head size"):
        d2p.attention(q[..., :60], k[..., :60], k[..., :60])
    big = torch.zeros(1, 1, 1, 136, dtype=BF)
    with pytest.raises(ValueError, match="head size"):
        d2p.attention(big, big, big)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            d2p.attention(q, k, k, scale=scale)
    with pytest.raises(ValueError, match="bias"):
        d2p.attention(q, k, k, bias=torch.zeros(32, 3, dtype=BF))
    with pytest.raises(TypeError, match="bias"):
        d2p.attention(q, k, k, bias=torch.zeros(32, 4, dtype=torch.float16))
    with pytest.raises(ValueError, match="even"):
        d2p.attention(q, k, k, bias=torch.zeros(31, 4, dtype=BF))
    with pytest.raises(ValueError, match="max_distance"):
        d2p.attention(q, k, k, bias=torch.zeros(32, 4, dtype=BF), max_distance=4)
    for lengths in (torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="lengths"):
            d2p.attention(q, k, k, lengths=lengths)


def test_qk_norm_rope_refuses():
    q, k, w, t = torch.zeros(2, 5, 4, 64), torch.zeros(2, 5, 2, 64), torch.ones(64), torch.zeros(9, 32)
    with pytest.raises(ValueError, match="must be"):
        d2p.qk_norm_rope(q, k[:, :4], w, w, t, t)
    with pytest.raises(TypeError, match="float32"):
        d2p.qk_norm_rope(q, k.to(BF), w, w, t, t)
    with pytest.raises(ValueError, match="head size"):
        d2p.qk_norm_rope(q[..., :40], k[..., :40], w[:40], w[:40], t[:, :8], t[:, :8])
    with pytest.raises(ValueError, match="weight"):
        d2p.qk_norm_rope(q, k, w[:32], w, t, t)
    with pytest.raises(TypeError, match="weights"):
        d2p.qk_norm_rope(q, k, w.to(BF), w.to(BF), t, t)
    with pytest.raises(ValueError, match="cos and sin"):
        d2p.qk_norm_rope(q, k, w, w, t.double(), t.double())
    with pytest.raises(ValueError, match="multiple of 16"):
        d2p.qk_norm_rope(q, k, w, w, t[:, :12], t[:, :12])
    with pytest.raises(ValueError, match="rows"):
        d2p.qk_norm_rope(q, k, w, w, t[:4], t[:4])
    with pytest.raises(ValueError, match="positions"):
        d2p.qk_norm_rope(q, k, w, w, t, t, positions=torch.zeros(2, 5))
    with pytest.raises(ValueError, match="positions"):
        d2p.qk_norm_rope(q, k, w, w, t, t, positions=torch.zeros(5, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="eps"):
        d2p.qk_norm_rope(q, k, w, w, t, t, eps=-1.0)


def test_dropout_add_refuses():
    x = torch.zeros(4, 4)
    with pytest.raises(TypeError):
        d2p.dropout_add(x.double(), None, 0.1, 0)
    with pytest.raises(ValueError, match="residual"):
        d2p.dropout_add(x, x[:2], 0.1, 0)
    for p in (-0.1, 1.0, math.nan):
        with pytest.raises(ValueError, match="p must be"):
            d2p.dropout_add(x, None, p, 0)
    with pytest.raises(ValueError, match="seed"):
        d2p.dropout_add(x, None, 0.1, 1 << 63)
    with pytest.raises(ValueError, match="offset"):
        d2p.dropout_add(x, None, 0.1, 0, -1)


def test_no_cpu_kernels():
    q, w, t = torch.zeros(1, 4, 2, 64, dtype=BF), torch.ones(64), torch.zeros(9, 32)
    for call in (lambda: d2p.attention(q, q, q), lambda: d2p.qk_norm_rope(q, q, w, w, t, t), lambda: d2p.dropout_add(q, q, 0.1, 0)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_public_names():
    for name in ("attention", "qk_norm_rope", "dropout_add", "relative_bucket_edges"):
        assert name in d2p.__all__ and callable(getattr(d2p, name))


# ---------------------------------------------------------------- fake tensors
def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    ops = torch.ops.d2p_b200
    with FakeTensorMode() as mode:
        q, k = (mode.from_tensor(torch.empty(2, n, h, 64, dtype=BF)) for n, h in ((5, 4), (7, 2)))
        b = mode.from_tensor(torch.empty(32, 4))
        assert d2p.attention(q, k, k, bias=b).shape == q.shape
        out, lse, rest = ops.attention_forward(q, k, k, b, None, d2p.relative_bucket_edges(32), 0.125, False, True, True)
        assert out.shape == q.shape and lse.shape == (2, 4, 5) and lse.dtype == torch.float32 and rest.shape == q.shape
        g = ops.attention_backward(q, q, k, k, b, None, d2p.relative_bucket_edges(32), 0.125, False, out, lse, rest, True)
        assert [tuple(t.shape) for t in g] == [(2, 5, 4, 64), (2, 7, 2, 64), (2, 7, 2, 64), (32, 4)] and g[3].dtype == torch.float32
        x, t, w = mode.from_tensor(torch.empty(2, 5, 2, 64, dtype=BF)), mode.from_tensor(torch.empty(9, 32)), mode.from_tensor(torch.empty(64))
        a, c = d2p.qk_norm_rope(q, x, w, w, t, t)
        assert a.shape == q.shape and c.shape == x.shape
        assert [tuple(r.shape) for r in ops.qk_norm_rope_backward(q, x, q, x, w, w, t, t, None, 1e-6)] == [(2, 5, 4, 64), (2, 5, 2, 64), (64,), (64,)]
        assert d2p.dropout_add(q, q, 0.1, 3).shape == q.shape


# ---------------------------------------------------------------- C ABI
class AttentionArgs(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("q_stride", ctypes.c_longlong * 3),
                ("k_stride", ctypes.c_longlong * 3), ("v_stride", ctypes.c_longlong * 3), ("bias", ctypes.c_void_p),
                ("lengths", ctypes.c_void_p), ("bucket_edges", ctypes.POINTER(ctypes.c_int)), ("n_edges", ctypes.c_int),
                ("bias_dtype", ctypes.c_int), ("B", ctypes.c_int), ("Lq", ctypes.c_int), ("Lk", ctypes.c_int), ("H", ctypes.c_int),
                ("Hkv", ctypes.c_int), ("D", ctypes.c_int), ("dtype", ctypes.c_int), ("causal", ctypes.c_int), ("scale", ctypes.c_float)]


def attention_args(**over):
    a = AttentionArgs(q=4096, k=4096, v=4096, B=1, Lq=4, Lk=4, H=2, Hkv=1, D=64, dtype=1, scale=0.125)
    for n in ("q_stride", "k_stride", "v_stride"):
        setattr(a, n, (ctypes.c_longlong * 3)(512, 128, 64))
    for n, v in over.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("over,code", [
    ({"H": 3, "Hkv": 2}, 1001), ({"Hkv": 0}, 1001), ({"B": -1}, 1001), ({"D": 60}, 1001), ({"D": 136}, 1001), ({"dtype": 0}, 1001),
    ({"scale": 0.0}, 1001), ({"scale": float("nan")}, 1001), ({"q": 4097}, 1001), ({"k": None}, 1001),
    ({"q_stride": (ctypes.c_longlong * 3)(512, 100, 64)}, 1001), ({"bias": 4096, "n_edges": 64}, 1001),
    ({"bias": 4096, "n_edges": 2, "bucket_edges": (ctypes.c_int * 2)(3, 2)}, 1001), ({"bias": 4096, "bias_dtype": 2}, 1001),
    ({"lengths": 4098}, 1001), ({"bias": 4098}, 1001),
    ({"B": 70000}, 1003), ({"B": 0}, 0), ({"Lq": 0}, 0)])
def test_c_abi_checks_attention(lib, over, code):
    f = lib.d2p_attention_forward
    f.restype = ctypes.c_int
    f.argtypes = [ctypes.POINTER(AttentionArgs), ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    a = attention_args(**over)
    assert f(ctypes.byref(a), None, None, None, None, 0, None) == code
    b = lib.d2p_attention_backward
    b.restype = ctypes.c_int
    b.argtypes = [ctypes.POINTER(AttentionArgs)] + [ctypes.c_void_p] * 9 + [ctypes.c_size_t, ctypes.c_void_p]
    if code:
        assert b(ctypes.byref(a), *[None] * 9, 0, None) == code


def test_c_abi_checks_outputs(lib):
    f = lib.d2p_attention_forward
    f.restype = ctypes.c_int
    f.argtypes = [ctypes.POINTER(AttentionArgs), ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    a = attention_args()
    assert f(ctypes.byref(a), None, None, None, None, 0, None) == 1001          # no output
    assert f(ctypes.byref(a), 4100, None, None, None, 0, None) == 1001          # output off a 16-byte boundary
    assert f(ctypes.byref(a), 4096, None, 4104, None, 0, None) == 1001          # rest off one
    assert f(ctypes.byref(a), 4096, 4098, None, None, 0, None) == 1001          # lse off a word
    d = lib.d2p_dropout_add
    d.restype = ctypes.c_int
    d.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_ulonglong, ctypes.c_double, ctypes.c_ulonglong,
                  ctypes.c_ulonglong, ctypes.c_void_p, ctypes.c_void_p]
    assert d(None, None, 0, 0, 0.5, 1, 1, None, None) == 0
    assert d(None, None, 0, 4, 0.5, 1, 1, None, None) == 1001
    assert d(None, None, 0, 0, 1.5, 1, 1, None, None) == 1001
    assert d(4097, None, 1, 4, 0.5, 1, 1, 4096, None) == 1001                   # off an element's boundary
    assert d(4096, None, 0, 4, 0.5, 1, 1, 4098, None) == 1001


class NormRopeArgs(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k")] + [("q_stride", ctypes.c_longlong * 3), ("k_stride", ctypes.c_longlong * 3)] + [
        (n, ctypes.c_void_p) for n in ("q_weight", "k_weight", "cos", "sin", "positions")] + [("position_batch_stride", ctypes.c_longlong)] + [
        (n, ctypes.c_int) for n in ("positions_int64", "P", "B", "L", "H", "Hkv", "D", "R", "dtype", "weight_dtype")] + [("eps", ctypes.c_float)]


@pytest.mark.parametrize("over", [
    {"D": 24}, {"D": 272}, {"R": 80}, {"R": 8}, {"L": 9}, {"cos": None}, {"q": 4104}, {"q_weight": 4100}, {"sin": 4104}, {"eps": -1.0},
    {"eps": float("nan")}, {"q_stride": (ctypes.c_longlong * 3)(512, 132, 64)}, {"positions": 4098}, {"B": -1}])
def test_c_abi_checks_norm_rope(lib, over):
    a = NormRopeArgs(q=4096, k=4096, q_weight=4096, k_weight=4096, cos=4096, sin=4096, P=8, B=1, L=4, H=2, Hkv=1, D=64, R=64, dtype=1,
                     weight_dtype=1, eps=1e-6)
    for n in ("q_stride", "k_stride"):
        setattr(a, n, (ctypes.c_longlong * 3)(512, 128, 64))
    for n, v in over.items():
        setattr(a, n, v)
    f = lib.d2p_norm_rope_forward
    f.restype = ctypes.c_int
    f.argtypes = [ctypes.POINTER(NormRopeArgs)] + [ctypes.c_void_p] * 3
    assert f(ctypes.byref(a), 4096, 4096, None) == 1001
    b = lib.d2p_norm_rope_backward
    b.restype = ctypes.c_int
    b.argtypes = [ctypes.POINTER(NormRopeArgs)] + [ctypes.c_void_p] * 7 + [ctypes.c_size_t, ctypes.c_void_p]
    assert b(ctypes.byref(a), *[4096] * 7, 1 << 30, None) == 1001
