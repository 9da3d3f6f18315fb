"""The encoder operators under forward-mode derivatives and under tracing, with fake CUDA tensors (no GPU): a tangent is refused,
never dropped, and a step's seed and offset are no constants of a graph."""
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


@pytest.mark.parametrize("train", [False, True])
def test_seed_and_offset_stay_symbols(train):
    from torch._dynamo.source import ConstantSource
    from torch.fx.experimental.symbolic_shapes import DimDynamic, ShapeEnv

    env = ShapeEnv()

    def symbol(value, name):
        source = ConstantSource(name)
        return env.create_symintnode(env.create_symbol(value, source, dynamic_dim=DimDynamic.DYNAMIC), hint=value, source=source)

    with FakeTensorMode(shape_env=env):
        x = torch.empty(4, 5, device="cuda", requires_grad=train)
        y = d2p.dropout_add(x, x, 0.1, symbol(9, "seed"), symbol(7, "offset"))
        assert y.shape == x.shape and y.requires_grad == train   # (its backward pass needs a device)
    assert not [g.expr for g in env.guards if "Eq" in str(g.expr)]


def test_a_step_is_no_new_graph():
    """The offset of each step: a constant at first, then a symbol, and no third graph."""
    graphs = []

    def backend(module, example):
        graphs.append(module)
        return module.forward

    torch._dynamo.reset()
    step = torch.compile(lambda x, offset: d2p.dropout_add(x, x, 0.1, 5, offset) + 1, backend=backend, fullgraph=True)
    with FakeTensorMode():
        x = torch.empty(4, 5, device="cuda")
        for offset in range(5, 12):
            assert step(x, offset).shape == x.shape
    assert len(graphs) == 2
