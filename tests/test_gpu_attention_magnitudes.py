"""Gradients of attention where upstream gradients are small, large or of very different size per sequence, against the 64-bit
form.

Tolerances as in test_gpu_ops.py: 2 u for the two roundings of 16-bit types (u = eps / 2), 1e-5 for f32, and for f16 results
half of its fixed step, 2^-25, per element."""
import math

import pytest
import torch

from test_gpu_ops import bound_of, plain_attention, ptr, rel

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def attention_grads(dt, lens, heads, kv_heads, dim, by, seed=0, v_by=1.0, k_lens=None):
    """by: the size of d_out per sequence.  Gradients here and in 64 bits."""
    from ts_trajgen_amd import ops
    g = torch.Generator().manual_seed(seed)
    k_lens = k_lens or lens
    qp, kp = ptr(lens), ptr(k_lens)
    mk = lambda n, h, s=1.0: (torch.randn(n, h, dim, generator=g) * s).to(dt)  # noqa: E731
    q, k, v = mk(qp[-1], heads), mk(kp[-1], kv_heads), mk(kp[-1], kv_heads, v_by)
    do = torch.randn(qp[-1], heads, dim, generator=g) * torch.repeat_interleave(torch.tensor(by), torch.tensor(lens)).view(-1, 1, 1)
    do = do.clamp(-torch.finfo(dt).max, torch.finfo(dt).max).to(dt)
    leaves = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
    tq, tk = (torch.tensor(p, dtype=torch.int32, device=DEV) for p in (qp, kp))
    out = ops.causal_attention(*leaves, tq, tk)
    got = torch.autograd.grad(out, leaves, do.to(DEV))
    return got, plain_attention(q, k, v, qp, kp, dim ** -0.5, do)[1:], qp, kp


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('by', [1e-4, 1e-3, 1.0, 1.5e4])
@pytest.mark.parametrize('lens,heads,kv_heads,dim', [([1500], 2, 1, 128), ([1100, 1300], 2, 2, 64), ([1200], 1, 1, 256), ([37, 5, 120, 64], 4, 2, 128)])
def test_attention_gradients_of_small_and_large_upstream_gradients(dt, by, lens, heads, kv_heads, dim):
    """Means over thousands of positions, and scaled losses."""
    got, want, _, _ = attention_grads(dt, lens, heads, kv_heads, dim, [by] * len(lens), seed=dim)
    for what, a, e in zip(('dq', 'dk', 'dv'), got, want):
        if dt == torch.float16:              # sums beyond its largest number are infinite, and only those
            a, e = a.clamp(-65504.0, 65504.0), e.clamp(-65504.0, 65504.0)
        assert rel(a, e) < bound_of(dt, e), (what, rel(a, e), bound_of(dt, e))


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_attention_sequences_of_very_different_upstream_gradients(dt, dim):
    """Packed side by side in the same tiles; each sequence for itself."""
    lens, by = [40, 300, 17, 1, 200, 90], [1e-4, 1.0, 3e3, 1.0, 1e-2, 3e2]
    got, want, qp, kp = attention_grads(dt, lens, 4, 2, dim, by, seed=dim)
    for s in range(len(lens)):
        for what, a, e, p in zip(('dq', 'dk', 'dv'), got, want, (qp, kp, kp)):
            a, e = a[p[s]:p[s + 1]], e[p[s]:p[s + 1]]
            if float(e.norm()) < 1e-9:       # one position attends to itself: its scores have no gradient
                assert float(a.double().norm()) <= 1e-3 * by[s] * torch.finfo(dt).eps * math.sqrt(e.numel()) + 1e-5 * by[s]
                continue
            assert rel(a, e) < bound_of(dt, e), (s, what, rel(a, e), bound_of(dt, e))


def test_attention_f16_gradients_of_large_values():
    """Values in the thousands under small upstream gradients, and the walk over the rows in stretches."""
    for v_by, by in ((4e3, 1e-2), (1e-3, 1e3)):
        got, want, _, _ = attention_grads(torch.float16, [2300], 2, 1, 64, [by], seed=5, v_by=v_by)
        for what, a, e in zip(('dq', 'dk', 'dv'), got, want):
            assert rel(a, e) < bound_of(torch.float16, e), (v_by, what, rel(a, e), bound_of(torch.float16, e))


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('by', [1e-3, 1.0])
@pytest.mark.parametrize('heads,kv_heads,dim', [(16, 1, 64), (16, 1, 128), (32, 2, 128), (16, 1, 256)])
def test_attention_gradients_of_short_sequences_under_many_heads(dt, by, heads, kv_heads, dim):
    """Fewer than 1024 positions in the mean, but walks long enough to be cut into stretches: both at once."""
    got, want, _, _ = attention_grads(dt, [500, 700], heads, kv_heads, dim, [by, by], seed=heads + dim)
    for what, a, e in zip(('dq', 'dk', 'dv'), got, want):
        assert rel(a, e) < bound_of(dt, e), (what, rel(a, e), bound_of(dt, e))


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('dim', [64, 128, 256])
def test_attention_gradients_in_a_captured_graph(dt, dim):
    """Replayed with upstream gradients of another size each time, between eager calls."""
    from ts_trajgen_amd import ops
    lens = [77, 600, 5]
    p = torch.tensor(ptr(lens), dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(dim)
    q, k, v = (torch.randn(sum(lens), h, dim, generator=g, device=DEV).to(dt).requires_grad_(True) for h in (8, 1, 1))
    base = torch.randn(sum(lens), 8, dim, generator=g, device=DEV)
    do = torch.zeros(sum(lens), 8, dim, device=DEV, dtype=dt)

    def step():
        out = ops.causal_attention(q, k, v, p)
        return (out.detach(),) + torch.autograd.grad(out, [q, k, v], do)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for by in (1e-4, 1.0, 5e3, 1e-2):
        do.copy_(base * by)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(captured, step()):
            assert torch.equal(a, e)
