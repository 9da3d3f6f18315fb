"""Encoder operators: what a network in front of the alignment runs to make its embeddings.

``attention`` (with a learned relative position bias by buckets), ``qk_norm_rope`` and ``dropout_add`` are
hand-written kernels (d2p_b200/csrc/enc_*.cu) with their gradients, over the same ragged batches and
``lengths`` [B, 2] as the alignment operators.  The reference has no such operators: it takes the score plane
(d2p/sw.py:247).  They are dispatcher ops under ``torch.ops.d2p_b200`` with shapes for fake tensors; there is
no CPU kernel.
"""
from __future__ import annotations

import functools
import math
from typing import Optional, Tuple

import torch

from . import _ops  # noqa: F401  the native extension (fails loudly if missing)

# the operators with their gradients (autograd nodes in csrc/torch_bindings.cpp)
_ops_attention = torch.ops.d2p_b200.attention.default
_ops_qk_norm_rope = torch.ops.d2p_b200.qk_norm_rope.default
_ops_dropout_add = torch.ops.d2p_b200.dropout_add.default

_MAX_PROBLEMS = 65535   # of a launch's grid
_MAX_REACH = 1024
_MAX_SIDE = 64


@functools.lru_cache(maxsize=64)
def relative_bucket_edges(num_buckets: int, max_distance: int = 128, two_sided: bool = True) -> Tuple[int, ...]:
    """Distances at which each bucket of a side but the first begins.

    With two_sided, keys after the query take the second half of the ``num_buckets``; a side then has ``s =
    num_buckets / 2`` buckets, otherwise ``s = num_buckets``.  Distances below ``e = s // 2`` have a bucket each;
    the rest are spaced by their logarithm, distance n in bucket ``e + floor(log(n / e) / log(max_distance / e)
    (s - e))``, at most s - 1.  Computed in whole numbers, so an edge never depends on a rounded logarithm."""
    if two_sided and num_buckets % 2:
        raise ValueError(f"a two-sided bias needs an even number of buckets, got {num_buckets}")
    side = num_buckets // 2 if two_sided else num_buckets
    if not 2 <= side <= _MAX_SIDE:
        raise ValueError(f"buckets per side must be in [2, {_MAX_SIDE}], got {side}")
    e = side // 2
    if not e < max_distance <= _MAX_REACH:
        raise ValueError(f"max_distance must be in ({e}, {_MAX_REACH}], got {max_distance}")
    c = side - e
    edges = list(range(1, e + 1))
    n = e
    for t in range(1, c):
        while n ** c * e ** t < max_distance ** t * e ** c:
            n += 1
        edges.append(n)
    return tuple(edges)


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    lengths: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    causal: bool = False,
    max_distance: int = 128,
) -> torch.Tensor:
    """softmax(scale q k^T + bias) v over a ragged batch: [B, Lq, H, D], with gradients to q, k, v and bias.

    q [B, Lq, H, D], k and v [B, Lk, Hkv, D], bfloat16 or float16, D a multiple of 8 up to 128; H is a multiple
    of Hkv, query head h reads key head ``h // (H // Hkv)``; B and H up to 65535.  Any strides (rows that are not whole 16-byte units
    are copied).  ``lengths`` [B, 2] int32: (queries, keys) of each problem, clamped to the padded sizes on the
    device; rows past them are zero, and what q, k, v hold there is never used.  ``causal`` aligns the last query
    with the last key (query i at position i + lk - lq) and masks later keys; a row left without keys is zero.
    (A NaN or infinity in a live key's v reaches masked rows of its tile too, as 0 x inf does in the plain product.)
    ``bias`` [num_buckets, H] (q's dtype or float32) adds bias[bucket, h] by relative position
    (``relative_bucket_edges``; two-sided unless causal).  -inf masks a bucket; a row all of whose keys carry one large
    entry (-1e9) is the softmax of its scores.  ``scale`` defaults to 1 / sqrt(D) and must be positive.
    """
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("attention: q must be [B, Lq, H, D] and k, v [B, Lk, Hkv, D]")
    if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("attention: q, k and v must all be bfloat16 or all float16")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError("attention: the heads of q must be a multiple of those of k and v")
    if q.shape[0] > _MAX_PROBLEMS or q.shape[2] > _MAX_PROBLEMS:
        raise ValueError(f"attention: at most {_MAX_PROBLEMS} problems and heads a call, got {q.shape[0]} and {q.shape[2]}")
    if not 8 <= q.shape[3] <= 128 or q.shape[3] % 8:
        raise ValueError(f"attention: the head size must be a multiple of 8, at most 128, got {q.shape[3]}")
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    if not (scale > 0.0 and scale <= 1e30):
        raise ValueError(f"attention: scale must be positive and finite, got {scale}")
    edges: Tuple[int, ...] = ()
    if bias is not None:
        if bias.dim() != 2 or bias.shape[1] != q.shape[2]:
            raise ValueError(f"attention: bias must be [num_buckets, {q.shape[2]}], got {tuple(bias.shape)}")
        if bias.dtype not in (q.dtype, torch.float32):
            raise TypeError("attention: bias must be float32 or of q's dtype")
        edges = relative_bucket_edges(int(bias.shape[0]), int(max_distance), not causal)
    if lengths is not None and (lengths.dtype != torch.int32 or tuple(lengths.shape) != (q.shape[0], 2)):
        raise ValueError("attention: lengths must be int32 [B, 2]")
    return _ops_attention(q, k, v, bias, lengths, edges, scale, bool(causal))


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor,
    k_weight: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    positions: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each head of q [B, L, H, D] and k [B, L, Hkv, D], then the position rotation, in one pass;
    gradients to q, k and the weights.

    ``y = x / sqrt(mean(x^2) + eps) * weight``; the first R = 2 cos.shape[1] elements turn in pairs (d, d + R / 2):
    ``(a cos - b sin, b cos + a sin)`` with cos, sin [P, R / 2] float32 (no gradient) at the token's position:
    ``positions`` [B, L] or [L] (int32 or int64, clamped to the table on the device) or 0 .. L - 1.  float32,
    bfloat16 or float16; D a multiple of 16 up to 256, R a multiple of 16 up to D; weights [D] float32 or q's dtype.
    """
    if q.dim() != 4 or k.dim() != 4 or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("qk_norm_rope: q must be [B, L, H, D] and k [B, L, Hkv, D]")
    if q.dtype not in (torch.float32, torch.bfloat16, torch.float16) or k.dtype != q.dtype:
        raise TypeError("qk_norm_rope: q and k must both be float32, bfloat16 or float16")
    D = q.shape[3]
    if D < 16 or D > 256 or D % 16:
        raise ValueError(f"qk_norm_rope: the head size must be a multiple of 16, at most 256, got {D}")
    if tuple(q_weight.shape) != (D,) or tuple(k_weight.shape) != (D,):
        raise ValueError("qk_norm_rope: q_weight and k_weight must be [D]")
    if q_weight.dtype != k_weight.dtype or q_weight.dtype not in (torch.float32, q.dtype):
        raise TypeError("qk_norm_rope: the weights must both be float32 or of q's dtype")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("qk_norm_rope: cos and sin must be float32 [P, R / 2]")
    if 2 * cos.shape[1] > D or cos.shape[1] % 8:
        raise ValueError("qk_norm_rope: 2 * cos.shape[1] must be a multiple of 16, at most D")
    if positions is None:
        if cos.shape[1] and q.shape[1] > cos.shape[0]:
            raise ValueError(f"qk_norm_rope: {q.shape[1]} positions but cos and sin have {cos.shape[0]} rows")
    elif positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in (
            tuple(q.shape[:2]), tuple(q.shape[1:2])):
        raise ValueError("qk_norm_rope: positions must be int32 or int64 [B, L] or [L]")
    if not eps >= 0.0:
        raise ValueError(f"qk_norm_rope: eps must not be negative, got {eps}")
    return _ops_qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, float(eps))


def dropout_add(
    x: torch.Tensor,
    residual: Optional[torch.Tensor],
    p: float,
    seed: int,
    offset: int = 0,
) -> torch.Tensor:
    """residual + dropout(x, p): kept elements are x / (1 - p), dropped ones nothing.  float32, bfloat16 or
    float16, any shape; ``residual`` of x's shape and dtype, or None.

    The mask comes from a counter-based generator (Philox4x32-10) and is never stored: element e (in row-major
    order) is kept where word e % 4 of the block with counter (e / 4, offset) and key ``seed`` is at least
    floor(p 2^32).  Equal seed and offset give equal masks; a step draws a new one by another offset.  0 <= seed,
    offset < 2^63 and 0 <= p < 1."""
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError("dropout_add: x must be float32, bfloat16 or float16")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("dropout_add: residual must have x's shape and dtype")
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout_add: p must be in [0, 1), got {p}")
    for name, value in (("seed", seed), ("offset", offset)):
        if not 0 <= value < 2 ** 63:
            raise ValueError(f"dropout_add: {name} must be in [0, 2^63), got {value}")
    # (symbols of a trace stay what they are)
    seed, offset = (v if isinstance(v, torch.SymInt) else int(v) for v in (seed, offset))
    return _ops_dropout_add(x, residual, float(p), seed, offset)


def _attention_forward_fake(q, k, v, bias, lengths, bucket_edges, scale, causal, want_lse, want_rest):
    lse = q.new_empty((q.shape[0] if want_lse else 0, q.shape[2], q.shape[1]), dtype=torch.float32)
    return q.new_empty(q.shape), lse, q.new_empty((q.shape[0] if want_rest else 0, *q.shape[1:]))


def _attention_fake(q, k, v, bias, lengths, bucket_edges, scale, causal):
    return q.new_empty(q.shape)


def _attention_backward_fake(grad, q, k, v, bias, lengths, bucket_edges, scale, causal, out, lse, rest, want_bias):
    db = bias.new_empty(bias.shape) if want_bias else q.new_empty((0, 0))
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape), db


def _qk_norm_rope_fake(q, k, q_weight, k_weight, cos, sin, positions, eps):
    return q.new_empty(q.shape), k.new_empty(k.shape)


def _qk_norm_rope_backward_fake(grad_q, grad_k, q, k, q_weight, k_weight, cos, sin, positions, eps):
    return q.new_empty(q.shape), k.new_empty(k.shape), q_weight.new_empty(q_weight.shape), k_weight.new_empty(k_weight.shape)


def _dropout_add_fake(x, residual, p, seed, offset):
    return x.new_empty(x.shape)


for _name, _fake in (("attention", _attention_fake), ("attention_forward", _attention_forward_fake), ("attention_backward", _attention_backward_fake),
                     ("qk_norm_rope", _qk_norm_rope_fake), ("qk_norm_rope_forward", _qk_norm_rope_fake), ("qk_norm_rope_backward", _qk_norm_rope_backward_fake),
                     ("dropout_add", _dropout_add_fake), ("dropout_add_forward", _dropout_add_fake)):
    torch.library.register_fake("d2p_b200::" + _name)(_fake)
