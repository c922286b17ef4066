"""Gradients of the cross entropy where upstream gradients are small, large or of very different size per row, against the 64-bit
form, judged row by row.

Tolerances as in test_gpu_ops.py: 2 u for the two roundings of 16-bit types (u = eps / 2), 1e-5 for f32, and for f16 results
half of its fixed step, 2^-25, per element."""
import math

import pytest
import torch

from test_gpu_ops import bound_of, entropy_case, plain_cross_entropy, rel

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rows_within(got, want, dt, factor=1.0):
    """Every row for itself."""
    got, want = got.detach().double().cpu(), want.double()
    assert torch.isfinite(got).all()
    err, norm = (got - want).norm(dim=1), want.norm(dim=1)
    fixed = 2.0 ** -25 * math.sqrt(want.shape[1]) if dt == torch.float16 else 0.0
    over = err - factor * ((1e-5 if dt == torch.float32 else torch.finfo(dt).eps + 2e-6) * norm + fixed)
    worst = int(over.argmax())
    assert float(over[worst]) <= 0.0, (worst, float(err[worst]), float(norm[worst]))


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('t,v,k', [(61, 1000, 256), (150, 3001, 100), (2500, 9001, 64)])
def test_cross_entropy_rows_of_very_different_upstream_gradients(dt, t, v, k):
    """reduction 'none' with upstream gradients over 12 decades (f16, whose dh has to hold them: 7), in no order, some negative,
    some zero."""
    from ts_trajgen_amd import ops
    h, w, b, target = entropy_case(dt, t, v, k, seed=t)
    low, high = (-3, 4) if dt == torch.float16 else (-12, 0)
    g = torch.Generator().manual_seed(t)
    up = torch.logspace(low, high, t)[torch.randperm(t, generator=g)] * (1 - 2 * (torch.rand(t, generator=g) < 0.3).float())
    up[::17] = 0.0
    rows = ops.linear_cross_entropy(h, w, target, bias=b, reduction='none')
    got = torch.autograd.grad(rows, [h, w, b], up.to(DEV))
    _, dh, dw, db = plain_cross_entropy(h, w, b, target, -100, up)
    rows_within(got[0], dh, dt)
    rows_within(got[1], dw, dt)
    assert rel(got[2], db) < bound_of(dt, db)


@pytest.mark.parametrize('dt', TYPES)
def test_cross_entropy_one_large_upstream_gradient_over_small_ones(dt):
    """One row of 1 among rows of 1e-6 whose targets nothing else says anything about: their rows of dW are those rows' alone but
    for the large row's probabilities."""
    from ts_trajgen_amd import ops
    t, v, k = 200, 1500, 64
    h, w, b, target = entropy_case(dt, t, v, k, seed=3, ignored=0.0)
    target = torch.arange(t).to(DEV)
    up = torch.full((t,), 1e-6 if dt != torch.float16 else 1.0)
    up[7] = 1.0 if dt != torch.float16 else 1e4
    rows = ops.linear_cross_entropy(h, w, target, bias=b, reduction='none')
    got = torch.autograd.grad(rows, [h, w, b], up.to(DEV))
    _, dh, dw, db = plain_cross_entropy(h, w, b, target, -100, up)
    rows_within(got[0], dh, dt)
    rows_within(got[1], dw, dt)
    assert rel(got[2], db) < bound_of(dt, db)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('by', [1e-30, 1e30])
def test_cross_entropy_tiny_and_huge_upstream_gradients(dt, by):
    """All of one size, at the ends of f32 (bf16 and f32; f16 results hold neither)."""
    from ts_trajgen_amd import ops
    if dt == torch.float16:
        by = {1e-30: 2.0 ** -8, 1e30: 2.0 ** 14}[by]
    h, w, b, target = entropy_case(dt, 90, 700, 64, seed=6)
    up = torch.rand(90, generator=torch.Generator().manual_seed(1)) * by + by
    rows = ops.linear_cross_entropy(h, w, target, bias=b, reduction='none')
    got = torch.autograd.grad(rows, [h, w, b], up.to(DEV))
    _, dh, dw, db = plain_cross_entropy(h, w, b, target, -100, up)
    rows_within(got[0], dh, dt)
    rows_within(got[1], dw, dt)
    assert rel(got[2], db) < bound_of(dt, db)


@pytest.mark.parametrize('dt', TYPES)
def test_cross_entropy_rows_of_different_upstream_gradients_over_several_pieces(dt):
    """30000 rows x 8001 entries: two pieces of the vocabulary in 16 bits, three in f32."""
    from ts_trajgen_amd import ops
    t, v, k = 30000, 8001, 16
    g = torch.Generator(device=DEV).manual_seed(1)
    h = torch.randn(t, k, generator=g, device=DEV).to(dt).requires_grad_(True)
    w = (torch.randn(v, k, generator=g, device=DEV) * 0.3).to(dt).requires_grad_(True)
    b = (torch.randn(v, generator=g, device=DEV) * 0.3).to(dt).requires_grad_(True)
    target = torch.randint(0, v, (t,), generator=g, device=DEV)
    low, high = (-3, 3) if dt == torch.float16 else (-12, 0)
    up = torch.logspace(low, high, t, device=DEV)[torch.randperm(t, generator=g, device=DEV)]
    rows = ops.linear_cross_entropy(h, w, target, bias=b, reduction='none')
    got = torch.autograd.grad(rows, [h, w, b], up)
    with torch.no_grad():
        dz = torch.log_softmax(h.double() @ w.double().t() + b.double(), dim=1)
        assert rel(rows, -dz.gather(1, target.unsqueeze(1)).squeeze(1)) < 1e-5
        dz.exp_()
        dz[torch.arange(t, device=DEV), target] -= 1.0
        dz *= up.double().unsqueeze(1)
        dh, dw, db = (x.cpu() for x in (dz @ w.double(), dz.t() @ h.double(), dz.sum(0)))
    rows_within(got[0], dh, dt)
    rows_within(got[1], dw, dt)
    assert rel(got[2], db) < bound_of(dt, db)


@pytest.mark.parametrize('dt', TYPES)
def test_cross_entropy_upstream_gradients_of_zero_and_single_rows(dt):
    from ts_trajgen_amd import ops
    h, w, b, target = entropy_case(dt, 80, 600, 72, seed=2, ignored=0.0)
    rows = ops.linear_cross_entropy(h, w, target, bias=b, reduction='none')
    for g in torch.autograd.grad(rows, [h, w, b], torch.zeros(80, device=DEV), retain_graph=True):
        assert float(g.abs().sum()) == 0.0
    up = torch.zeros(80)
    up[61] = -3e-5 if dt != torch.float16 else -3.0        # one row alone: its gradients are what a call of it alone gives
    got = torch.autograd.grad(rows, [h, w, b], up.to(DEV))
    _, *want = plain_cross_entropy(h, w, b, target, -100, up)
    for a, e in zip(got, want):
        assert rel(a, e) < bound_of(dt, e)
    assert float(got[0][:61].abs().sum()) == 0.0 and float(got[0][62:].abs().sum()) == 0.0


@pytest.mark.parametrize('dt', TYPES)
def test_cross_entropy_per_row_in_a_captured_graph(dt):
    """Replayed with other upstream gradients of other sizes each time, between eager calls."""
    from ts_trajgen_amd import ops
    h, w, b, target = entropy_case(dt, 100, 700, 64, seed=10)
    up = torch.zeros(100, device=DEV)

    def step():
        rows = ops.linear_cross_entropy(h, w, target, bias=b, reduction='none')
        return (rows.detach(),) + torch.autograd.grad(rows, [h, w, b], up)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for n in range(4):
        up.copy_(torch.logspace(-3 - n, 2 * n, 100))
        g.replay()
        torch.cuda.synchronize()
        for a, e in zip(captured, step()):
            assert torch.equal(a, e)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('t,v,k,reduction', [(2048, 1300, 64, 'mean'), (5000, 300, 256, 'none'), (20000, 2049, 100, 'sum'), (2100, 257, 512, 'mean')])
def test_cross_entropy_many_rows_over_few_entries(dt, t, v, k, reduction):
    """dW has a handful of tiles and a long sum there, which is cut into stretches of the rows."""
    from ts_trajgen_amd import ops
    h, w, b, target = entropy_case(dt, t, v, k, seed=t, ignored=0.1)
    g = torch.Generator().manual_seed(t)
    loss = ops.linear_cross_entropy(h, w, target, bias=b, reduction=reduction)
    up = torch.rand(t, generator=g) + 0.5 if reduction == 'none' else torch.tensor(1.7)
    got = torch.autograd.grad(loss, [h, w, b], up.to(DEV))
    n = float((target != -100).sum())
    d_row = up if reduction == 'none' else torch.full((t,), 1.7 / (n if reduction == 'mean' else 1.0))
    _, *want = plain_cross_entropy(h, w, b, target, -100, d_row)
    for a, e in zip(got, want):
        assert rel(a, e) < bound_of(dt, e)


@pytest.mark.parametrize('h_by,w_by', [(1e-36, 1.0), (1e-3, 1e-33), (1e18, 1e-18)])
def test_cross_entropy_states_and_weights_at_the_ends_of_f32(h_by, w_by):
    """Their planes are brought to f16's range by powers of two as far out as 2^126, which come off the gradients without passing through
    f32's smallest numbers on the way."""
    from ts_trajgen_amd import ops
    h, w, b, target = entropy_case(torch.float32, 70, 500, 64, seed=6, h_by=h_by, w_by=w_by / 8, ignored=0.1)
    loss = ops.linear_cross_entropy(h, w, target, bias=b, reduction='sum')
    got = torch.autograd.grad(loss, [h, w, b])
    _, *want = plain_cross_entropy(h, w, b, target, -100, torch.ones(70))
    for a, e in zip(got, want):
        rows_within(a if a.dim() == 2 else a.unsqueeze(0), e if e.dim() == 2 else e.unsqueeze(0), torch.float32)
