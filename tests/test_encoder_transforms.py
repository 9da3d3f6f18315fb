"""The encoder operators under forward-mode derivatives, with fake CUDA tensors (no GPU): a tangent is refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

import d2p_b200 as d2p

BF = torch.bfloat16


def operands():
    def new(*shape, dtype=BF):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    return {
        "attention": (lambda q, k, v, bias: d2p.attention(q, k, v, bias=bias), [new(2, 5, 4, 64), new(2, 7, 2, 64), new(2, 7, 2, 64), new(32, 4)]),
        "qk_norm_rope": (d2p.qk_norm_rope, [new(2, 5, 4, 64), new(2, 5, 2, 64), new(64), new(64), new(9, 32, dtype=torch.float32),
                                            new(9, 32, dtype=torch.float32)]),
        "dropout_add": (lambda x, r: d2p.dropout_add(x, r, 0.1, 7), [new(4, 5), new(4, 5)]),
    }


@pytest.mark.parametrize("name", ["attention", "qk_norm_rope", "dropout_add"])
def test_tangents_are_refused(name):
    with FakeTensorMode():
        call, args = operands()[name]
        for at in range(len(args)):
            for requires_grad in (False, True):
                with fwAD.dual_level():
                    a = list(args)
                    a[at] = fwAD.make_dual(a[at].clone().requires_grad_(requires_grad), torch.empty_like(a[at]))
                    with pytest.raises(RuntimeError, match="not implemented"):
                        call(*a)
                    with torch.no_grad(), pytest.raises(RuntimeError, match="not implemented"):
                        call(*a)
            with pytest.raises(RuntimeError, match="not implemented"):
                torch.func.jvp(lambda x: call(*args[:at], x, *args[at + 1:]), (args[at],), (torch.empty_like(args[at]),))
        with fwAD.dual_level():   # (no input with a tangent)
            out = call(*args)
        assert (out if isinstance(out, torch.Tensor) else out[0]).shape == args[0].shape
