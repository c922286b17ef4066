"""The framework's own training paths over the sequence operators, on MI355X: function G fitted on packed trajectories, and the
road encoder with its dropouts recomputed from a counter.

Tolerances: both sides of the encoder's comparison run the same f32 sums in the same order, apart from the compiler's choice of
fused operations (one step of 2^-24 per product): 1e-6 of the largest value.  Function G is compared with the same modules in
64 bits on the CPU: chained f32 sums of up to ~1000 terms through an LSTM of a dozen steps, sqrt(n) 2^-24 < 2e-6 each: 2e-5."""
import numpy as np
import pytest
import torch

from test_gpu_ops import keep_of

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def function_g(roads=1000, times=200, road=32, time=16, hidden=64, p=0.0, layers=1):
    from ts_trajgen_amd.generator.function_g_fc import FunctionGFC
    torch.manual_seed(3)
    return FunctionGFC({'road_emb_size': road, 'time_emb_size': time, 'hidden_size': hidden, 'lstm_layer_num': layers,
                        'dropout_p': p, 'dis_weight': 0.5},
                       {'road_num': roads, 'road_pad': roads - 1, 'time_size': times, 'time_pad': times - 1})


def trajectories(lens, roads=1000, times=200, front=0, tail=0):
    g = torch.Generator().manual_seed(7)
    n = sum(lens) + front + tail
    ptr = torch.tensor(np.cumsum([front] + list(lens)), dtype=torch.int32)
    return (torch.randint(0, roads - 1, (n,), generator=g), torch.randint(0, times - 1, (n,), generator=g), ptr)


def plain_loss(m, loc, tim, ptr, masks=None):
    """m in 64 bits on the CPU; masks: the two dropouts' factors."""
    x = torch.cat([m.road_emb(loc), m.time_emb(tim)], dim=1)
    if masks is not None:
        x = x * masks[0]
    total, count = x.new_zeros(()), 0
    for s in range(len(ptr) - 1):
        i, j = int(ptr[s]), int(ptr[s + 1])
        if j - i < 2:
            continue
        h = m.lstm(x[i:j].unsqueeze(0))[0][0]
        score = (h @ h.t()).masked_fill(torch.ones(j - i, j - i).triu(1).bool(), float('-inf'))
        a = torch.softmax(score, dim=1) @ h
        if masks is not None:
            a = a * masks[1][i:j]
        z = m.out_fc(a[:-1])
        total = total + torch.nn.functional.cross_entropy(z, loc[i + 1:j], reduction='sum')
        count += j - i - 1
    return total / count


@pytest.mark.parametrize('p,layers', [(0.0, 1), (0.6, 1), (0.1, 2)])
def test_function_g_over_packed_trajectories(p, layers):
    lens = [12, 1, 0, 7, 33, 2]
    m = function_g(p=p, layers=layers)
    loc, tim, ptr = trajectories(lens, front=3, tail=4)
    n, seed, step = loc.numel(), 77, 5
    masks = None
    if p:
        masks = [(keep_of(n * w, p, seed, site, step).double() / (1 - p)).reshape(n, w) for site, w in ((0, 48), (1, 64))]
    ref = function_g(p=p, layers=layers).double()
    want = plain_loss(ref, loc, tim, ptr, masks)
    want.backward()
    m = m.to(DEV).train(True)
    got = m.trajectory_loss(loc, tim, ptr, seed=seed, step=step)
    got.backward()
    assert abs(float(got.detach()) - float(want.detach())) <= 2e-5 * float(want.detach())
    refs = dict(ref.named_parameters())
    for k, w in m.named_parameters():
        if k.startswith('intra_attn'):
            assert w.grad is None
            continue
        r = refs[k].grad
        err = float((w.grad.double().cpu() - r).norm() / r.norm())
        assert err <= 2e-5, (k, err)
    # every step has its own masks, the same step the same
    with torch.no_grad():
        again = m.trajectory_loss(loc, tim, ptr, seed=seed, step=step)
        other = m.trajectory_loss(loc, tim, ptr, seed=seed, step=step + 1)
        assert torch.equal(again, got.detach()) and (p == 0) == torch.equal(other, got.detach())
        # a target of one's own, and the sums
        rows = m.train(False).trajectory_loss(loc, tim, ptr, target=torch.full((n,), 4), reduction='none')
        assert rows.shape == (n,) and (rows[:3] == 0).all() and (rows[-4:] == 0).all() and (rows[3:-4] > 0).all()


def test_function_g_refuses_what_it_cannot_fit():
    m = function_g().to(DEV)
    loc, tim, ptr = trajectories([5, 6])
    for bad in [(loc + 1000, tim, ptr), (loc, tim - 300, ptr), (loc, tim[:-1], ptr), (loc, tim, ptr.long()), (loc, tim, ptr + 1),
                (loc, tim, ptr.flip(0)), (loc[:0], tim[:0], ptr * 0), (loc, tim, ptr[:1])]:
        with pytest.raises(ValueError):
            m.trajectory_loss(*bad)
    with pytest.raises(ValueError):
        m.trajectory_loss(loc, tim, ptr, target=loc[:3])
    with pytest.raises(RuntimeError):
        function_g().trajectory_loss(loc, tim, ptr)


def encoder(fin, fo, heads, concat, p=0.6):
    from ts_trajgen_amd.generator.gat import GATLayerImp3
    torch.manual_seed(5)
    return GATLayerImp3(fin, fo, heads, DEV, concat=concat, dropout_prob=p).to(DEV).train(True)


def run_encoder(layer, x, edges, up):
    x = x.detach().requires_grad_(True)
    out, _ = layer((x, edges))
    grads = torch.autograd.grad(out, [x] + list(layer.parameters()), up, allow_unused=True)
    return [out.detach()] + [g for g in grads if g is not None]


@pytest.mark.parametrize('fin,fo,heads,concat', [(12, 16, 5, True), (16, 16, 1, False), (9, 7, 3, True), (64, 300, 2, True)])
@pytest.mark.parametrize('on_device', [False, True])
def test_encoder_masks_from_the_counter(fin, fo, heads, concat, on_device):
    n, e, p, seed, site, step = 131, 400, 0.6, 0xABCDEF0123456789, 11, 4
    g = torch.Generator().manual_seed(1)
    # loops of one's own keep every node's softmax non-empty; node 130 has nothing else
    edges = torch.cat([torch.randint(0, n - 1, (2, e), generator=g), torch.arange(n).repeat(2, 1)], dim=1).to(DEV)
    x = torch.randn(n, fin, generator=g).to(DEV)
    up = torch.randn(n, heads * fo if concat else fo, generator=g).to(DEV)
    layer = encoder(fin, fo, heads, concat, p)
    order = layer._train_graph(edges, n, x.device)[5].cpu()
    e_all = edges.shape[1]
    scale = np.float32(1.0 / (1.0 - p))
    m_in, m_proj, by_slot = [keep_of(rows * w, p, seed, site + i, step).float().reshape(rows, w) * scale
                             for i, (rows, w) in enumerate([(n, fin), (n, heads * fo), (e_all, heads)])]
    m_att = torch.empty(e_all, heads)
    m_att[order] = by_slot
    layer.dropout_masks = (m_in, m_proj, m_att)
    want = run_encoder(layer, x, edges, up)
    with pytest.raises(ValueError):
        layer.dropout_rng = (seed, site, step)
        layer((x, edges))
    layer.dropout_masks = None
    layer.dropout_rng = (seed, site, torch.tensor([step], device=DEV) if on_device else step)
    got = run_encoder(layer, x, edges, up)
    assert len(got) == len(want) >= 5
    for a, b in zip(got, want):
        assert float((a - b).abs().max()) <= 1e-6 * float(b.abs().max())
    layer.dropout_rng = (seed, site, step + 1)
    assert not torch.equal(run_encoder(layer, x, edges, up)[0], got[0])
    for bad in [(1 << 64, 0, 0), (0, -1, 0), (0, (1 << 32) - 2, 0), (0, 0, -1), (0, 0, torch.zeros(1, dtype=torch.int64))]:
        layer.dropout_rng = bad
        with pytest.raises(ValueError):
            layer((x, edges))


def test_encoder_step_advanced_before_its_backward_is_an_error():
    layer = encoder(8, 8, 2, True)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    layer.dropout_rng = (1, 0, step)
    edges = torch.arange(9, device=DEV).repeat(2, 1)
    out, _ = layer((torch.randn(9, 8, device=DEV, requires_grad=True), edges))
    step += 1
    with pytest.raises(RuntimeError):
        out.sum().backward()


def test_encoder_graph_goes_with_its_output():
    import gc
    from ts_trajgen_amd import ops
    layer = encoder(8, 8, 2, True)
    layer.dropout_rng = (1, 0, 0)
    edges = torch.arange(9, device=DEV).repeat(2, 1)
    gc.collect()
    before = len(ops._LIVE)
    gc.disable()
    try:
        out, _ = layer((torch.randn(9, 8, device=DEV, requires_grad=True), edges))
        assert len(ops._LIVE) == before + 1
        out.sum().backward()
        del out
        assert len(ops._LIVE) == before
    finally:
        gc.enable()


def test_encoder_saved_tensors_that_hooks_move_elsewhere():
    layer = encoder(8, 8, 2, True)
    edges = torch.randint(0, 50, (2, 200), generator=torch.Generator().manual_seed(2)).to(DEV)
    x = torch.randn(50, 8, device=DEV, requires_grad=True)

    def loss():
        layer.dropout_rng = (1, 0, torch.tensor([3], device=DEV))
        return (layer((x, edges))[0] ** 2).sum()
    leaves = [x, layer.linear_proj.weight, layer.bias]
    want = torch.autograd.grad(loss(), leaves)
    with torch.autograd.graph.save_on_cpu():
        value = loss()
    layer.dropout_rng = None
    junk = [torch.full((n,), float('nan'), device=DEV) for n in (2, 400, 800) for _ in range(20)]
    for a, e in zip(torch.autograd.grad(value, leaves), want):
        assert torch.equal(a, e)
    del junk


@pytest.mark.parametrize('hidden', [50, 320])
def test_function_g_of_other_widths(hidden):
    loc, tim, ptr = trajectories([12, 40, 2])
    ref = function_g(hidden=hidden).double()
    want = plain_loss(ref, loc, tim, ptr)
    want.backward()
    m = function_g(hidden=hidden).to(DEV).train(True)
    got = m.trajectory_loss(loc, tim, ptr)
    got.backward()
    assert abs(float(got.detach()) - float(want.detach())) <= 2e-5 * float(want.detach())
    for (k, w), r in zip(m.named_parameters(), ref.parameters()):
        if r.grad is not None:
            assert float((w.grad.double().cpu() - r.grad).norm() / r.grad.norm()) <= 2e-5, k


@pytest.mark.parametrize('auto', [torch.float16, torch.bfloat16])
def test_function_g_under_autocast(auto):
    """The recurrence then runs in 16 bits, and out_fc goes with it as torch's own linear would.  Logits are 64 products of states below 1
    and weights below 1/8: three roundings of 2^-11 on each are 64 / 8 * 3 * 2^-11 = 0.012, and states off by 8 * 2^-11 (four
    roundings a step, halved by every forget gate) 64 / 8 * 2^-8 = 0.03; a loss is the difference of two: 0.1 (the recurrence is
    f16 under both)."""
    loc, tim, ptr = trajectories([12, 40, 2])
    m = function_g().to(DEV).train(True)
    want = m.trajectory_loss(loc, tim, ptr).detach()
    with torch.autocast('cuda', auto):
        got = m.trajectory_loss(loc, tim, ptr)
    assert got.dtype == torch.float32 and abs(float(got.detach()) - float(want)) <= 0.1
    got.backward()
    for k, w in m.named_parameters():
        if not k.startswith('intra_attn'):
            assert w.grad.dtype == torch.float32 and torch.isfinite(w.grad).all() and float(w.grad.abs().max()) > 0.0
