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
