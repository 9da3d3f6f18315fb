"""dropout_add within torch.compile, forward and backward: an offset of its own each step, with the graphs of two."""
import pytest
import torch

from tests.test_gpu_encoder import d2p  # noqa: F401  (fixture)

pytestmark = pytest.mark.gpu


def test_dropout_steps_compiled(d2p, cuda_device):  # noqa: F811
    from torch._dynamo.backends.common import aot_autograd

    graphs = []

    def keep(module, example):
        graphs.append(module)
        return module.forward

    def step(x, r, offset):
        return d2p.dropout_add(x * 2, r, 0.3, 11, offset)

    torch._dynamo.reset()
    compiled = torch.compile(step, backend=aot_autograd(fw_compiler=keep, bw_compiler=keep), fullgraph=True)
    g = torch.Generator().manual_seed(1)
    x, r, do = (torch.randn(33, 50, generator=g).to(cuda_device) for _ in range(3))
    for offset in range(3, 10):
        outs = []
        for f in (step, compiled):
            a, b = x.clone().requires_grad_(True), r.clone().requires_grad_(True)
            y = f(a, b, offset)
            y.backward(do)
            outs.append((y.detach(), a.grad, b.grad))
        assert all(torch.equal(u, v) for u, v in zip(*outs)), offset
    assert len(graphs) <= 4   # forward and backward, with a constant and with a symbol
