"""The sequence operators (ts_trajgen_amd.ops) on MI355X against plain 64-bit forms on the CPU.

Tolerances.  One rounding to a type is off by at most half a step, u = eps / 2 (bf16 2^-8, fp16 2^-11, f32 2^-24).
An output that is a sum of products of which one factor was rounded to the type (probabilities, score gradients) and which
is rounded itself is off, in the 2-norm over the tensor, by at most u for each of the two roundings: 2 u, and the f32
accumulation of n terms adds at most n 2^-24 in the worst case and about sqrt(n) 2^-24 in earnest.  The bounds below are
relative 2-norms: 2 u + 2e-6 for 16-bit types; for f32 a handful of chained sums of up to ~1000 terms, each about
sqrt(n) 2^-24 < 2e-6, gives 1e-5 with room for the exponential's own 1e-7."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def bound(dt):
    return 1e-5 if dt == torch.float32 else torch.finfo(dt).eps + 2e-6


def bound_of(dt, want):
    """f16 below 2^-14 has a fixed step of 2^-24: an element is off by up to half of it however small it is (gradients of means
    over hundreds of rows lie there), which is 2^-25 sqrt(n) in the 2-norm over n elements, on top of bound()."""
    norm = float(want.norm())
    return bound(dt) + (2.0 ** -25 * math.sqrt(want.numel()) / norm if dt == torch.float16 and norm else 0.0)


def rel(x, y):
    x, y = x.detach().double().cpu(), y.detach().double().cpu()
    assert x.shape == y.shape and torch.isfinite(x).all()
    n = float(y.norm())
    return float((x - y).norm()) / n if n else float(x.norm())


# ---------------------------------------------------------------------------------------------------------- dropout
def keep_of(n, p, seed, site, step):
    """Philox4x32-10 in Python integers via numpy uint64."""
    m = np.uint64(0xFFFFFFFF)
    b = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [b & m, b >> np.uint64(32), np.full_like(b, site), np.full_like(b, step)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        x, y = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(y >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), y & m, (x >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), x & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.from_numpy(np.stack(c, 1).reshape(-1)[:n] >= np.uint64(int(p * 4294967296.0)))


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('n,p', [(1, 0.5), (3, 0.6), (8, 0.1), (2049, 0.25), (100003, 0.6), (64, 0.0), (64, 1.0)])
def test_dropout_matches_the_generator(dt, n, p):
    from ts_trajgen_amd import ops
    seed, site, step = 0xDEADBEEF12345678, 7, 0xFFFFFFF0
    x = torch.randn(n, device=DEV).to(dt).requires_grad_(True)
    y = ops.dropout(x, p, seed, site, step)
    dy = torch.randn(n, device=DEV).to(dt)
    dx, = torch.autograd.grad(y, x, dy)
    keep = keep_of(n, p, seed, site, step) if p < 1.0 else torch.zeros(n, dtype=torch.bool)
    by = 1.0 / (1.0 - p) if p < 1.0 else 0.0
    for out, src in ((y, x), (dx, dy)):
        want = torch.where(keep, src.detach().cpu().float() * by, torch.zeros(())).to(dt)
        assert torch.equal(out.detach().cpu(), want)


def test_dropout_views_steps_and_masked_values():
    from ts_trajgen_amd import ops
    base = torch.randn(65, 131, device=DEV)
    x = base.t()[3:, 1:]                                   # transposed, offset view: numbered by its own shape
    y = ops.dropout(x, 0.5, 11, 2, 5)
    keep = keep_of(x.numel(), 0.5, 11, 2, 5).view(x.shape)
    assert torch.equal(y.cpu(), torch.where(keep, x.cpu() * 2.0, torch.zeros(())))
    one = ops.dropout(base.flatten()[1:], 0.5, 11, 2, 5)   # base address not 16-byte aligned
    assert torch.equal(one.cpu(), torch.where(keep_of(one.numel(), 0.5, 11, 2, 5), base.flatten()[1:].cpu() * 2.0, torch.zeros(())))
    counter = torch.tensor([5], dtype=torch.int64, device=DEV)
    assert torch.equal(ops.dropout(x, 0.5, 11, 2, counter), y)
    bad = torch.full((64,), float('nan'), device=DEV)
    z = ops.dropout(bad, 0.5, 3).cpu()
    assert torch.equal(torch.isnan(z), keep_of(64, 0.5, 3, 0, 0))     # a dropped NaN is 0
    assert ops.dropout(torch.empty(0, 4, device=DEV), 0.5, 3).shape == (0, 4)
    x = torch.randn(16, device=DEV, requires_grad=True)
    y = ops.dropout(x, 0.5, 1, 0, counter)
    counter.add_(1)
    with pytest.raises(RuntimeError):                      # the step was advanced before the backward
        y.sum().backward()


def test_dropout_in_a_captured_graph_advances_with_its_counter():
    from ts_trajgen_amd import ops
    x = torch.randn(5000, device=DEV, requires_grad=True)
    dy = torch.randn(5000, device=DEV)
    counter = torch.zeros(1, dtype=torch.int64, device=DEV)
    ops.dropout(dy, 0.3, 9, 1, counter)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.dropout(x, 0.3, 9, 1, counter)
        dx, = torch.autograd.grad(y, x, dy)
        counter.add_(1)
    for n in range(4):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.dropout(x, 0.3, 9, 1, n))
        assert torch.equal(dx, ops.dropout(dy, 0.3, 9, 1, n))


# -------------------------------------------------------------------------------------------------------- attention
def plain_attention(q, k, v, qp, kp, scale, do=None):
    """64-bit, one sequence and one head at a time, only over the keys a row sees."""
    q, k, v = q.detach().double().cpu(), k.detach().double().cpu(), v.detach().double().cpu()
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    do = None if do is None else do.double().cpu()
    group = q.shape[1] // k.shape[1]
    for s in range(len(qp) - 1):
        lq, lk = qp[s + 1] - qp[s], kp[s + 1] - kp[s]
        seen = torch.arange(lk).unsqueeze(0) <= torch.arange(lq).unsqueeze(1) + (lk - lq)
        some = seen.any(dim=1, keepdim=True)
        for h in range(q.shape[1]):
            rq, rk, m = slice(qp[s], qp[s + 1]), slice(kp[s], kp[s + 1]), h // group
            if lq == 0 or lk == 0:
                continue
            z = (q[rq, h] @ k[rk, m].t() * scale).masked_fill(~seen, -math.inf)
            p = torch.where(some, torch.softmax(z, dim=1), torch.zeros((), dtype=torch.double))
            out[rq, h] = p @ v[rk, m]
            if do is not None:
                g = do[rq, h]
                ds = p * (g @ v[rk, m].t() - (g * out[rq, h]).sum(1, keepdim=True)) * scale
                dq[rq, h] = ds @ k[rk, m]
                dk[rk, m] += ds.t() @ q[rq, h]
                dv[rk, m] += p.t() @ g
    return out, dq, dk, dv


def ptr(lens):
    return [0] + list(np.cumsum(lens))


def attend(dt, q_lens, k_lens, heads, kv_heads, dim, scale=None, tail=0, grad=True, seed=0, spread=1.0):
    from ts_trajgen_amd import ops
    g = torch.Generator().manual_seed(seed)
    qp, kp = ptr(q_lens), ptr(k_lens)
    same = q_lens is k_lens
    mk = lambda n, h: (torch.randn(n + tail, h, dim, generator=g) * spread).to(dt).to(DEV).requires_grad_(grad)  # noqa: E731
    q, k, v = mk(qp[-1], heads), mk(kp[-1], kv_heads), mk(kp[-1], kv_heads)
    tq = torch.tensor(qp, dtype=torch.int32, device=DEV)
    tk = None if same else torch.tensor(kp, dtype=torch.int32, device=DEV)
    out = ops.causal_attention(q, k, v, tq, tk, scale)
    do = torch.randn(q.shape, generator=g).to(dt) if grad else None
    want = plain_attention(q, k, v, qp, kp, scale or dim ** -0.5, do)
    assert rel(out, want[0]) < bound(dt)
    assert float(out.detach()[qp[-1]:].abs().sum()) == 0.0
    if grad:
        got = torch.autograd.grad(out, [q, k, v], do.to(DEV))
        for a, b in zip(got, want[1:]):
            assert rel(a, b) < bound(dt)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('dim', [8, 40, 64, 100, 128, 192, 256])
def test_attention_widths(dt, dim):
    lens = [1, 0, 37, 128, 3, 0, 161]
    attend(dt, lens, lens, 4, 2, dim, seed=dim)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('dim', [320, 500, 512])
def test_attention_wide_heads(dt, dim):
    lens = [5, 1, 70]
    attend(dt, lens, lens, 2, 1, dim, seed=dim)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('heads,kv_heads', [(1, 1), (3, 1), (8, 8), (10, 2), (16, 1)])
def test_attention_groups_of_heads(dt, heads, kv_heads):
    lens = [2, 130, 65]
    attend(dt, lens, lens, heads, kv_heads, 64, seed=heads)


@pytest.mark.parametrize('dt', TYPES)
def test_attention_many_short_trajectories(dt):
    lens = [int(n) for n in np.random.RandomState(3).randint(0, 40, 200)]
    attend(dt, lens, lens, 1, 1, 256, scale=1.0, seed=5, spread=0.25)


@pytest.mark.parametrize('dt', TYPES)
def test_attention_rows_over_longer_and_shorter_keys(dt):
    # the rest of a prompt over a cache, rows without any key (more queries than keys), keys without queries
    attend(dt, [5, 70, 9, 0, 3, 2], [90, 70, 4, 12, 0, 300], 4, 2, 128, seed=1)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('heads,kv_heads,dim', [(8, 1, 64), (8, 2, 128), (1, 1, 256), (6, 2, 40), (24, 2, 128), (16, 1, 512)])
def test_attention_single_rows_over_long_keys(dt, heads, kv_heads, dim):
    attend(dt, [1, 1, 0, 2, 1], [1500, 33, 70, 700, 1], heads, kv_heads, dim, seed=dim, grad=dim <= 256)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('lens,heads,kv_heads,dim', [([3100], 2, 1, 64), ([1700, 1500], 4, 2, 128), ([2000], 1, 1, 256), ([4000], 1, 1, 40)])
def test_attention_long_sequences(dt, lens, heads, kv_heads, dim):
    # few long sequences: the backward's walk over the rows is cut into stretches
    attend(dt, lens, lens, heads, kv_heads, dim, seed=dim)


def test_attention_rows_behind_the_last_sequence_are_zero_and_unread():
    from ts_trajgen_amd import ops
    for dt in TYPES:
        attend(dt, [9, 140], [9, 140], 2, 1, 64, tail=70)
        q = torch.randn(300, 2, 64, device=DEV).to(dt)
        q[100:] = float('nan')
        p = torch.tensor([0, 40, 100], dtype=torch.int32, device=DEV)
        out = ops.causal_attention(q, q, q, p)
        assert torch.isfinite(out).all() and float(out[100:].abs().sum()) == 0.0
        assert torch.equal(out[:100], ops.causal_attention(q[:100], q[:100], q[:100], p))


def test_attention_views_are_read_by_their_strides():
    from ts_trajgen_amd import ops
    p = torch.tensor([0, 50, 177], dtype=torch.int32, device=DEV)
    for dt in TYPES:
        qkv = torch.randn(177, 3, 4, 64, device=DEV).to(dt)
        q, k, v = qkv.unbind(1)                                             # rows 3 * 4 * 64 apart
        ref = ops.causal_attention(q.contiguous(), k.contiguous(), v.contiguous(), p)
        assert torch.equal(ops.causal_attention(q, k, v, p), ref)
        turned = torch.randn(4, 177, 64, device=DEV).to(dt).transpose(0, 1)  # head-major memory
        assert torch.equal(ops.causal_attention(turned, k, v, p), ops.causal_attention(turned.contiguous(), k, v, p))
        odd = torch.randn(177 * 4 * 64 + 1, device=DEV).to(dt)[1:].view(177, 4, 64)   # not 16-byte aligned
        assert torch.equal(ops.causal_attention(odd, k, v, p), ops.causal_attention(odd.clone(), k, v, p))
        wide = torch.randn(177, 1, 64, device=DEV).to(dt).expand(177, 4, 64)  # broadcast heads: stride 0
        x = wide.clone().requires_grad_(True)
        y = torch.randn(177, 1, 64, device=DEV).to(dt).requires_grad_(True)
        a = ops.causal_attention(x, y.expand(177, 4, 64), y.expand(177, 4, 64), p)
        b = ops.causal_attention(x, y.expand(177, 4, 64).contiguous(), y.expand(177, 4, 64).contiguous(), p)
        assert torch.equal(a, b)
        a.backward(torch.ones_like(a))
        assert y.grad.shape == y.shape and torch.isfinite(y.grad.float()).all()


def test_attention_single_rows_read_subnormal_keys():
    # keys below f16's smallest normal number still have their products
    from ts_trajgen_amd import ops
    g = torch.Generator().manual_seed(4)
    q = (torch.randn(1, 4, 64, generator=g) * 1e4).half()      # inside f16: its largest is 65504
    k = (torch.randn(300, 1, 64, generator=g) * 1e-5).half()
    v = torch.randn(300, 1, 64, generator=g).half()
    want = plain_attention(q, k, v, [0, 1], [0, 300], 1.0)[0]
    out = ops.causal_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV),
                               torch.tensor([0, 300], dtype=torch.int32, device=DEV), 1.0)
    assert rel(out, want) < bound(torch.float16)


def test_attention_extreme_scores():
    # one key dominates by more than f32's exponent range, and scores of the lowest finite size
    from ts_trajgen_amd import ops
    p = torch.tensor([0, 64], dtype=torch.int32, device=DEV)
    q = torch.zeros(64, 1, 64, device=DEV)
    k = torch.zeros(64, 1, 64, device=DEV)
    v = torch.randn(64, 1, 64, device=DEV)
    q[..., 0] = 1.0
    k[:, 0, 0] = -3.0e38
    k[5, 0, 0] = -1.0e38
    out = ops.causal_attention(q, k, v, p, scale=1.0)
    assert torch.allclose(out[:5, 0], torch.stack([v[:i + 1, 0].mean(0) for i in range(5)]), atol=1e-5)
    assert torch.allclose(out[5:, 0], v[5, 0].expand(59, 64), atol=1e-6)


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('lens,broken,heads,kv_heads,dim', [
    ([5, 9, 3, 20], 1, 2, 1, 32), ([5, 9, 3, 20], 1, 4, 2, 128), ([40, 1, 0, 70, 33], 3, 2, 2, 256),
    ([30, 300, 40, 200], 1, 4, 2, 128), ([1000, 900, 1100], 1, 4, 1, 64), ([2500, 2700], 0, 8, 1, 128)])
def test_attention_values_that_are_not_finite_stay_in_their_sequence(dt, lens, broken, heads, kv_heads, dim):
    """Infinities and NaN in one sequence's operands: every other sequence gives what it gives without them, rows before
    the first broken key do too, and rows that see one say so.  What it gives: a row's running reference moves when that of
    any row of its wave has to, so a neighbour's scores decide between references and hence between roundings; both
    results are within bound() of the true one, and so within twice that of each other."""
    from ts_trajgen_amd import ops
    g = torch.Generator().manual_seed(3)
    n, p = sum(lens), ptr(lens)
    q, k, v, do = [torch.randn(n, x, dim, generator=g).to(dt) for x in (heads, kv_heads, kv_heads, heads)]
    i, j = int(p[broken]), int(p[broken + 1])
    q[int(p[broken + 1]) - 1, :, 0] = 1.0      # an infinite key is then a score of +inf
    others = torch.ones(n, dtype=torch.bool)
    others[i:j] = False

    def run(q, k, v, do):
        q, k, v = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
        o = ops.causal_attention(q, k, v, torch.tensor(p, dtype=torch.int32, device=DEV))
        return [x.cpu() for x in [o.detach()] + list(torch.autograd.grad(o, (q, k, v), do.to(DEV)))]
    want = run(q, k, v, do)
    # the sequence's last row is broken in each operand in turn
    for at, value in [(0, float('nan')), (1, float('inf')), (2, float('nan')), (2, float('-inf')), (3, float('inf'))]:
        ops_ = [x.clone() for x in (q, k, v, do)]
        ops_[at][j - 1, 0, dim // 2 if at == 2 else 0] = value
        got = run(*ops_)
        for what, a, b in zip(('out', 'dq', 'dk', 'dv'), got, want):
            assert rel(a[others], b[others]) <= 2 * bound_of(dt, b[others]), (at, value, what)
            if what in ('out', 'dq'):       # rows before the broken one do not see it
                assert rel(a[i:j - 1], b[i:j - 1]) <= 2 * bound_of(dt, b[i:j - 1]), (at, value, what)
        if at < 3:
            assert not torch.isfinite(got[0][j - 1, 0]).all()
        if at == 2:     # only that column, and only the heads over that key
            bad = ~torch.isfinite(got[0][j - 1])
            group = heads // kv_heads
            assert bad[:group, dim // 2].all() and int(bad.sum()) == group
    # a whole sequence of them
    ops_ = [x.clone() for x in (q, k, v, do)]
    for x in ops_:
        x[i:j] = float('nan')
    for a, b in zip(run(*ops_), want):
        assert rel(a[others], b[others]) <= 2 * bound_of(dt, b[others]) and torch.isnan(a[i:j]).all()


def test_attention_gradient_against_differences():
    from ts_trajgen_amd import ops
    torch.manual_seed(0)
    p = torch.tensor([0, 7, 20], dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn(20, h, 16, device=DEV, requires_grad=True) for h in (4, 2, 2))
    w = torch.randn(20, 4, 16, device=DEV)
    grads = torch.autograd.grad((ops.causal_attention(q, k, v, p) * w).sum(), [q, k, v])
    for i, (x, g) in enumerate(zip((q, k, v), grads)):
        d = torch.randn_like(x)
        e = 1e-2
        args = [[t.detach().clone() for t in (q, k, v)] for _ in range(2)]
        args[0][i] += e * d
        args[1][i] -= e * d
        hi, lo = (float((plain_attention(*a, [0, 7, 20], [0, 7, 20], 0.25)[0] * w.double().cpu()).sum()) for a in args)
        # central difference of the 64-bit form: off by e^2 / 6 of the third derivative (order 1 here)
        assert abs((hi - lo) / (2 * e) - float((g * d).sum())) < 1e-3 * (1.0 + abs(hi - lo) / (2 * e))


def test_attention_repeats_bit_for_bit_on_streams_and_in_graphs():
    from ts_trajgen_amd import ops
    lens = [77, 300, 5]
    p = torch.tensor(ptr(lens), dtype=torch.int32, device=DEV)
    for dt in (torch.float32, torch.bfloat16):
        q, k, v = (torch.randn(382, h, 64, device=DEV).to(dt).requires_grad_(True) for h in (4, 2, 2))
        do = torch.randn(382, 4, 64, device=DEV).to(dt)

        def step():
            out = ops.causal_attention(q, k, v, p)
            return (out.detach(),) + torch.autograd.grad(out, [q, k, v], do)     # no eager graph outlives the call
        first = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            third = step()
        for _ in range(3):
            for t in third:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            for a, b, c in zip(first, second, third):
                assert torch.equal(a, b) and torch.equal(a, c)


def test_capture_over_a_living_eager_graph_is_refused():
    from ts_trajgen_amd import ops
    p = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    x = torch.randn(40, 2, 64, device=DEV, requires_grad=True)
    kept = ops.causal_attention(x, x, x, p)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='eager autograd graph'):
        with torch.cuda.graph(g):
            ops.causal_attention(x, x, x, p)
    with pytest.raises(RuntimeError, match='eager autograd graph'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.dropout(x, 0.5, 1)
    want, = torch.autograd.grad(kept, x, torch.ones_like(kept))
    del kept
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.causal_attention(x, x, x, p)
        dx, = torch.autograd.grad(out, x, torch.ones_like(out))
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(dx, want)


# ---------------------------------------------------------------------------------------------------- cross entropy
def plain_cross_entropy(h, w, b, target, ignore, d_row):
    """64-bit losses per row, and the gradients for the row gradients d_row."""
    h, w = h.detach().double().cpu(), w.detach().double().cpu()
    b = torch.zeros(w.shape[0], dtype=torch.double) if b is None else b.detach().double().cpu()
    target, d_row = target.cpu(), d_row.double().cpu()
    used = target != ignore
    h = torch.where(used.unsqueeze(1), h, torch.zeros((), dtype=torch.double))
    lp = torch.log_softmax(h @ w.t() + b, dim=1)
    at = torch.where(used, target, 0)
    rows = torch.where(used, -lp.gather(1, at.unsqueeze(1)).squeeze(1), torch.zeros((), dtype=torch.double))
    dz = lp.exp()
    dz[torch.arange(len(at)), at] -= 1.0
    dz = dz * (d_row * used).unsqueeze(1)
    return rows, dz @ w, dz.t() @ h, dz.sum(0)


def entropy_case(dt, t, v, k, bias=True, reduction='mean', ignored=0.2, seed=0, h_by=1.0, w_by=None, spread=None):
    g = torch.Generator().manual_seed(seed)
    h = torch.tanh(torch.randn(t, k, generator=g)) * h_by
    if spread is not None:
        h = h * spread(t).unsqueeze(1)
    h = h.to(dt).to(DEV).requires_grad_(True)
    w = (torch.randn(v, k, generator=g) * (w_by or 1.5 / math.sqrt(k))).to(dt).to(DEV).requires_grad_(True)
    b = (torch.randn(v, generator=g) * 0.5).to(dt).to(DEV).requires_grad_(True) if bias else None
    target = torch.randint(0, v, (t,), generator=g)
    target[torch.rand(t, generator=g) < ignored] = -100
    target[0] = v - 1
    return h, w, b, target.to(DEV)


def check_entropy(dt, h, w, b, target, reduction='mean'):
    from ts_trajgen_amd import ops
    loss = ops.linear_cross_entropy(h, w, target, bias=b, reduction=reduction)
    up = torch.randn(loss.shape, generator=torch.Generator().manual_seed(1)).to(DEV) if reduction == 'none' else torch.full((), 1.7, device=DEV)
    got = torch.autograd.grad(loss, [h, w] + ([b] if b is not None else []), up)
    used = target != -100
    n = float(used.sum())
    d_row = up if reduction == 'none' else torch.full((len(target),), 1.7 / (n if reduction == 'mean' else 1.0), device=DEV)
    rows, dh, dw, db = plain_cross_entropy(h, w, b, target, -100, d_row)
    want = rows if reduction == 'none' else rows.sum() / (n if reduction == 'mean' else 1.0)
    # the loss itself is f32: products of exact operands, one rounding per addition
    assert rel(loss, want) < 1e-5
    for a, e in zip(got, (dh, dw, db)):
        assert rel(a, e) < bound_of(dt, e), (a.shape, rel(a, e))
    return loss, got


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('t,v,k', [(1, 1, 8), (1, 300, 64), (61, 1000, 256), (129, 129, 72), (300, 5003, 100), (128, 128, 128),
                                   (257, 4097, 320), (5, 11096, 256), (700, 640, 1000), (64, 2048, 3),
                                   (2500, 9001, 64), (4100, 8200, 260)])
def test_cross_entropy_sizes(dt, t, v, k):
    check_entropy(dt, *entropy_case(dt, t, v, k, seed=t + v))


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
@pytest.mark.parametrize('bias', [True, False])
def test_cross_entropy_reductions(dt, reduction, bias):
    check_entropy(dt, *entropy_case(dt, 200, 1500, 128, bias=bias, seed=3), reduction=reduction)


@pytest.mark.parametrize('dt', TYPES)
def test_cross_entropy_of_sharp_and_flat_rows(dt):
    check_entropy(dt, *entropy_case(dt, 150, 2000, 64, w_by=2.0, seed=4), reduction='sum')       # logits up to ~60
    check_entropy(dt, *entropy_case(dt, 150, 2000, 64, w_by=1e-3, seed=5), reduction='mean')     # almost uniform
    check_entropy(torch.float32, *entropy_case(torch.float32, 150, 2000, 64, h_by=1e-6, w_by=1e4, seed=6), reduction='mean')
    check_entropy(torch.float32, *entropy_case(torch.float32, 90, 700, 64, seed=7, spread=lambda t: torch.logspace(-3, 1, t)), reduction='none')


@pytest.mark.parametrize('dt', TYPES)
def test_cross_entropy_several_pieces(dt, monkeypatch):
    # 40000 rows: 2^31 bytes of dz are a piece of 26624 (16-bit) or 13312 (f32) entries
    g = torch.Generator(device=DEV).manual_seed(1)
    t, v, k = 40000, 27000, 16
    from ts_trajgen_amd import ops
    h = torch.randn(t, k, generator=g, device=DEV).to(dt).requires_grad_(True)
    w = (torch.randn(v, k, generator=g, device=DEV) * 0.3).to(dt).requires_grad_(True)
    b = (torch.randn(v, generator=g, device=DEV) * 0.3).to(dt).requires_grad_(True)
    target = torch.randint(0, v, (t,), generator=g, device=DEV)
    loss = ops.linear_cross_entropy(h, w, target, bias=b)
    got = torch.autograd.grad(loss, [h, w, b])
    with torch.no_grad():
        z = h.double() @ w.double().t() + b.double()
        lp = torch.log_softmax(z, dim=1)
        assert rel(loss, -lp.gather(1, target.unsqueeze(1)).mean()) < 1e-5
        dz = lp.exp_()
        dz[torch.arange(t, device=DEV), target] -= 1.0
        dz /= t
        for a, e in zip(got, (dz @ w.double(), dz.t() @ h.double(), dz.sum(0))):
            assert rel(a, e) < bound_of(dt, e)


@pytest.mark.parametrize('dt', TYPES)
def test_cross_entropy_rows_left_out_hold_anything(dt):
    from ts_trajgen_amd import ops
    h, w, b, target = entropy_case(dt, 130, 900, 64, seed=8)
    loss, grads = check_entropy(dt, h, w, b, target)
    bad = h.detach().clone()
    bad[target == -100] = float('nan')
    bad[torch.nonzero(target == -100)[0]] = float('inf')
    bad.requires_grad_(True)
    loss2 = ops.linear_cross_entropy(bad, w, target, bias=b)
    got = torch.autograd.grad(loss2, [bad, w, b], torch.full((), 1.7, device=DEV))
    assert torch.equal(loss, loss2)
    for a, e in zip(got, grads):
        assert torch.equal(a, e)
    assert float(got[0][target == -100].abs().sum()) == 0.0


@pytest.mark.parametrize('dt', TYPES)
@pytest.mark.parametrize('value', [float('nan'), float('inf')])
def test_cross_entropy_rows_that_are_not_finite_spoil_only_themselves(dt, value):
    """A state, and an upstream gradient, that are not finite: the other rows' losses and dh are what they are without.  All of
    it is small (2^-20), so that a scale taken from the broken value would lose it."""
    from ts_trajgen_amd import ops
    h, w, b, target = entropy_case(dt, 130, 900, 64, seed=12, ignored=0.0, h_by=2.0 ** -6 if dt == torch.float16 else 2.0 ** -20)
    up = torch.rand(130, generator=torch.Generator().manual_seed(2)).to(DEV) * 2.0 ** -10 + 2.0 ** -12
    keep = torch.arange(130) != 17

    def run(h, up):
        h = h.detach().requires_grad_(True)
        rows = ops.linear_cross_entropy(h, w, target, bias=b, reduction='none')
        return rows.detach(), torch.autograd.grad(rows, h, up)[0]
    rows, dh = run(h, up)
    _, want, _, _ = plain_cross_entropy(h, w, b, target, -100, up)
    assert rel(dh, want) < bound_of(dt, want)
    bad = h.detach().clone()
    bad[17, 3] = value
    rows2, dh2 = run(bad, up)
    assert torch.isnan(rows2[17]) and rel(rows2[keep], rows[keep]) < 2e-5
    assert torch.isnan(dh2[17].float()).all() and rel(dh2[keep], want[keep]) < bound_of(dt, want[keep])
    up2 = up.clone()
    up2[17] = value
    rows2, dh2 = run(h, up2)
    assert torch.equal(rows2, rows) and rel(dh2[keep], want[keep]) < bound_of(dt, want[keep])
    assert not torch.isfinite(dh2[17].float()).any()


def test_cross_entropy_masked_entries_empty_means_and_bad_targets():
    from ts_trajgen_amd import ops
    for dt in TYPES:
        h, w, b, target = entropy_case(dt, 40, 300, 64, seed=9, ignored=0.0)
        with torch.no_grad():
            b[7:200] = float('-inf')                    # entries that cannot be chosen
        target = torch.where((target >= 7) & (target < 200), torch.full_like(target, 3), target)
        loss = ops.linear_cross_entropy(h, w, target, bias=b)
        want, dh, dw, db = plain_cross_entropy(h, w, b, target, -100, torch.full((40,), 1 / 40.0))
        got = torch.autograd.grad(loss, [h, w, b])
        assert rel(loss, want.mean()) < 1e-5
        for a, e in zip(got, (dh, dw, db)):
            assert rel(a, e) < bound_of(dt, e)
        assert float(got[1][7:200].abs().sum()) == 0.0
        with torch.no_grad():
            b.fill_(torch.finfo(dt).min)                # the type's lowest value everywhere: uniform
        none = torch.full_like(target, -100)
        rows = ops.linear_cross_entropy(h, w, none, reduction='none')
        assert float(rows.detach().abs().sum()) == 0.0
        assert math.isnan(float(ops.linear_cross_entropy(h, w, none)))
        off = target.clone()
        off[5] = 300
        rows = ops.linear_cross_entropy(h, w, off, reduction='none')
        assert torch.isnan(rows[5]) and torch.isfinite(rows[torch.arange(40, device=DEV) != 5]).all()
        off[5] = -1
        dh, = torch.autograd.grad(ops.linear_cross_entropy(h, w, off, reduction='sum'), [h])
        assert torch.isnan(dh[5].float()).all() and torch.isfinite(dh[torch.arange(40, device=DEV) != 5].float()).all()


def test_cross_entropy_views_and_repeats():
    from ts_trajgen_amd import ops
    for dt in TYPES:
        h, w, b, target = entropy_case(dt, 100, 700, 64, seed=10)
        wide = torch.randn(100, 200, device=DEV).to(dt)
        hv = wide[:, 24:88]                             # rows 200 apart
        a = ops.linear_cross_entropy(hv, w, target, bias=b, reduction='none')
        assert torch.equal(a, ops.linear_cross_entropy(hv.contiguous(), w, target, bias=b, reduction='none'))
        assert torch.equal(ops.linear_cross_entropy(hv, w.t().contiguous().t(), target, bias=b, reduction='none'), a)
        assert torch.equal(ops.linear_cross_entropy(wide[:, 23:87], w, target, reduction='none'),
                           ops.linear_cross_entropy(wide[:, 23:87].contiguous(), w, target, reduction='none'))
        one = torch.randn(1, 64, device=DEV).to(dt).requires_grad_(True)
        loss = ops.linear_cross_entropy(one.expand(100, 64), w, target, bias=b)
        loss.backward()
        assert one.grad.shape == one.shape
        w.grad = b.grad = None

        def step():
            loss = ops.linear_cross_entropy(h, w, target, bias=b)
            return (loss.detach(),) + torch.autograd.grad(loss, [h, w, b])
        del loss, a
        first = step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            third = step()
        for _ in range(3):
            for t in third:
                t.zero_()
            g.replay()
            torch.cuda.synchronize()
            second = step()
            for x, y, z in zip(first, second, third):
                assert torch.equal(x, y) and torch.equal(x, z)


def test_cross_entropy_gradient_against_differences():
    from ts_trajgen_amd import ops
    h, w, b, target = entropy_case(torch.float32, 30, 50, 16, seed=11)
    loss = ops.linear_cross_entropy(h, w, target, bias=b)
    grads = torch.autograd.grad(loss, [h, w, b])
    n = float((target != -100).sum())
    for i, g in enumerate(grads):
        d = torch.randn_like(g)
        args = [[x.detach().clone() for x in (h, w, b)] for _ in range(2)]
        args[0][i] += 1e-3 * d
        args[1][i] -= 1e-3 * d
        hi, lo = (float(plain_cross_entropy(*a, target, -100, torch.ones(30))[0].sum()) / n for a in args)
        # e^2 / 6 of the third derivative, and f32 rounding of the shifted arguments over 2 e
        assert abs((hi - lo) / 2e-3 - float((g * d).sum())) < 1e-3 * (1.0 + abs(hi - lo) / 2e-3)


def test_the_operators_together_over_packed_trajectories():
    """states -> dropout -> attention -> dropout -> loss, as function G is fitted, against autograd through 64-bit forms."""
    from ts_trajgen_amd import ops
    lens = [5, 1, 33, 20]
    n, width, vocab = sum(lens), 64, 400
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(n, width, generator=g) * 0.5).to(DEV).requires_grad_(True)
    w = (torch.randn(vocab, width, generator=g) * 0.2).to(DEV).requires_grad_(True)
    b = (torch.randn(vocab, generator=g) * 0.2).to(DEV).requires_grad_(True)
    target = torch.randint(0, vocab, (n,), generator=g).to(DEV)
    target[torch.tensor(np.cumsum(lens) - 1)] = -100
    p = torch.tensor(ptr(lens), dtype=torch.int32, device=DEV)

    def fused():
        s = ops.dropout(x, 0.3, 5, 0, 1)
        a = ops.causal_attention(s.unsqueeze(1), s.unsqueeze(1), s.unsqueeze(1), p, scale=1.0).squeeze(1)
        return ops.linear_cross_entropy(ops.dropout(a, 0.3, 5, 1, 1), w, target, bias=b)
    loss = fused()
    got = torch.autograd.grad(loss, [x, w, b])
    xd, wd, bd = (t.detach().double().cpu().requires_grad_(True) for t in (x, w, b))
    s = xd * keep_of(n * width, 0.3, 5, 0, 1).view(n, width) / 0.7
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    pos = torch.arange(n)
    z = (s @ s.t()).masked_fill((seq.unsqueeze(1) != seq) | (pos.unsqueeze(1) < pos), -math.inf)
    a = (torch.softmax(z, 1) @ s) * keep_of(n * width, 0.3, 5, 1, 1).view(n, width) / 0.7
    want = torch.nn.functional.cross_entropy(a @ wd.t() + bd, target.cpu())
    assert rel(loss, want) < 1e-5
    for a, e in zip(got, torch.autograd.grad(want, [xd, wd, bd])):
        assert rel(a, e) < 1e-5


@pytest.mark.parametrize('dt', TYPES)
def test_saved_tensors_that_hooks_move_elsewhere(dt):
    """Under save_on_cpu everything saved leaves its memory, which other tensors then take."""
    from ts_trajgen_amd import ops
    g = torch.Generator().manual_seed(9)
    p = torch.tensor(ptr([40, 3, 90]), dtype=torch.int32)
    x = torch.randn(133, 2, 36, generator=g).to(dt).to(DEV).requires_grad_(True)
    h, w, b, target = entropy_case(dt, 133, 500, 72, seed=4)
    step = torch.tensor([6], device=DEV)

    def losses():
        a = ops.causal_attention(x * 1.0, x * 0.5, x, p.to(DEV))
        y = ops.dropout(a.reshape(133, 72) * h, 0.3, 5, 2, step.clone())
        return ops.linear_cross_entropy(y, w, target.clone(), bias=b)
    want = torch.autograd.grad(losses(), [x, h, w, b])
    with torch.autograd.graph.save_on_cpu():
        loss = losses()
    junk = [torch.full((n,), float('nan'), device=DEV) for n in (50, 133, 400, 5000, 20000, 40000) for _ in range(20)]
    got = torch.autograd.grad(loss, [x, h, w, b])
    for a, e in zip(got, want):
        assert torch.equal(a, e)
    del junk
