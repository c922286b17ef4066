"""Calls of the sequence operators that no backward can follow: leaves that require gradients, under no_grad."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def test_a_forward_without_gradients_is_captured_while_an_eager_graph_lives():
    """Only the backward of a capture meets the leaf's gradient accumulator, and under no_grad there is none."""
    from ts_trajgen_amd import ops
    p = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    x = torch.randn(40, 2, 64, device=DEV, requires_grad=True)
    w = torch.randn(300, 128, device=DEV, requires_grad=True)
    target = torch.randint(0, 300, (40,), device=DEV)

    def forward():
        a = ops.causal_attention(x, x, x, p)
        return ops.linear_cross_entropy(ops.dropout(a, 0.3, 1).view(40, 128), w, target, reduction='none')
    kept = forward()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        out = forward()
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kept)
    with pytest.raises(RuntimeError, match='eager autograd graph'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            forward()
    grads = torch.autograd.grad(kept.sum(), [x, w])
    assert all(torch.isfinite(t).all() for t in grads)


def test_an_encoder_forward_without_gradients_is_captured_while_an_eager_graph_lives():
    from ts_trajgen_amd.generator.gat import GATLayerImp3
    torch.manual_seed(5)
    layer = GATLayerImp3(8, 16, 2, DEV, concat=True, dropout_prob=0.5).to(DEV).train(True)
    layer.dropout_rng = (1, 0, 2)
    edges = torch.cat([torch.randint(0, 50, (2, 200)), torch.arange(50).repeat(2, 1)], dim=1).to(DEV)
    x = torch.randn(50, 8, device=DEV, requires_grad=True)
    kept, _ = layer((x, edges))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        out, _ = layer((x, edges))
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, kept)


@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
def test_a_forward_without_gradients_keeps_nothing_for_one(dt):
    """16-bit attention writes what rounding took off its result for the backward alone."""
    from ts_trajgen_amd import ops
    p = torch.tensor([0, 4000], dtype=torch.int32, device=DEV)
    x = torch.randn(4000, 8, 64, device=DEV).to(dt)
    need = []
    for y, grad in ((x, True), (x.clone().requires_grad_(True), False)):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        with torch.set_grad_enabled(grad):
            out = ops.causal_attention(y, y, y, p)
        need.append(torch.cuda.max_memory_allocated() - before)
        assert not out.requires_grad
        del out
    assert need[0] == need[1]
