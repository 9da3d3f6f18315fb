"""Attention's gradients captured in a CUDA graph: the chain of launches (the items' order, the statistics, both passes) replayed
over other lengths and values gives the bits of a call outside the graph."""
import pytest
import torch

from tests.test_gpu_encoder import d2p, inputs, run_attention  # noqa: F401  (d2p: fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,L,H,Hkv,D,causal,nb,dtype", [
    (64, 512, 8, 8, 64, False, 32, torch.bfloat16),      # several items a CTA in both passes, in order of their work
    (48, 512, 16, 4, 128, True, 16, torch.bfloat16),     # several items a CTA of the queries alone
    (1, 2048, 16, 4, 128, True, 0, torch.bfloat16),      # the keys' items leave SMs free, on which the queries' begin
    (2, 100, 4, 4, 64, False, 8, torch.bfloat16),
    (64, 512, 8, 2, 64, True, 16, torch.float16),        # (with the launches for the operands' exponents)
    (1, 300, 4, 2, 128, False, 0, torch.float16)])
def test_gradients_replayed(d2p, cuda_device, B, L, H, Hkv, D, causal, nb, dtype):  # noqa: F811
    q, k, v, do, bias = inputs(B, L, L, H, Hkv, D, dtype, cuda_device, nb, seed=L)
    lengths = torch.full((B, 2), L, dtype=torch.int32, device=cuda_device)
    leaves = [t.requires_grad_(True) for t in (q, k, v, bias) if t is not None]

    def step():
        out = d2p.attention(q, k, v, bias=bias, lengths=lengths, causal=causal)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    g = torch.Generator().manual_seed(L)
    for turn in range(4):
        short = torch.randint(0, L + 1, (B, 2), generator=g, dtype=torch.int32)
        if B == 1:   # (causal: no row left without keys)
            short[:, 0], short[:, 1] = L - L // 7 * turn, L - L // 10 * turn
        with torch.no_grad():
            lengths.copy_(short)
            q.copy_(torch.randn(q.shape, generator=g).to(q.dtype))
            do.copy_((torch.randn(do.shape, generator=g) * 2.0 ** (-4 * turn)).to(do.dtype))
        for _ in range(2):
            graph.replay()
        want = run_attention(d2p, q.detach(), k.detach(), v.detach(), do, None if bias is None else bias.detach(), lengths, causal)
        for x, n in zip(got, ("out", "dq", "dk", "dv", "dbias")):
            assert torch.equal(x, want[n]), (turn, n)
