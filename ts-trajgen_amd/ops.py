"""Operators over sequences on the HIP kernels of libtsg.so, differentiable under torch's autograd.

    dropout(x, p, seed, site, step)                        mask recomputed from a counter, never stored
    causal_attention(q, k, v, seq_ptr, kv_ptr, scale)      packed sequences, grouped heads, forward and backward

They take tensors on a HIP device (f32, bf16 or f16), run on torch's current stream of that device, allocate their results and
workspaces through torch's allocator and never synchronise, so they can be captured in a graph (forward and backward
together; drop eager results that still hold an autograd graph of the same leaves first, which is checked).  Wrong shapes, types or
devices raise ValueError / TypeError / RuntimeError before anything is launched; there is no CPU fallback.  Gradients are
first order: differentiating a gradient raises.
"""
import ctypes as C
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _on_device(what, *tensors):
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not torch.is_tensor(t):
            raise TypeError('%s takes tensors, got %s' % (what, type(t).__name__))
        if not t.is_cuda:
            raise RuntimeError('%s needs CUDA/HIP tensors (no CPU fallback)' % what)
        if dev is not None and t.device != dev:
            raise ValueError('%s: tensors on %s and %s' % (what, dev, t.device))
        dev = t.device
    return dev


def _dtype(what, *tensors):
    dt = tensors[0].dtype
    if dt not in DTYPES:
        raise TypeError('%s takes f32, bf16 or f16, got %s' % (what, dt))
    for t in tensors:
        if t is not None and t.dtype != dt:
            raise TypeError('%s: mixed types %s and %s' % (what, dt, t.dtype))
    return DTYPES[dt]


def _hold_leaves(*leaves):
    """The gradient accumulators of the leaves, to be held over the call that uses them.

    Capturing a backward while an eager autograd graph of the same leaf is alive ends the process: the accumulator that graph
    keeps is tied to the stream it was made on, and joining that stream breaks the capture.  So every eager call leaves its
    stream on the accumulators, and a call under capture that finds another one refuses."""
    held = []
    if not torch.is_grad_enabled():
        return held
    here = torch.cuda.current_stream().cuda_stream
    capturing = torch.cuda.is_current_stream_capturing()
    for t in leaves:
        if t is None or not t.requires_grad or not t.is_leaf:
            continue
        node = torch.autograd.graph.get_gradient_edge(t).node
        if capturing and node.metadata.get('ts_trajgen_amd.stream', here) != here:
            raise RuntimeError('capture of a backward while an eager autograd graph of the same leaf is alive: drop the '
                               'eager results (del, or .detach() what is kept) before capturing')
        node.metadata['ts_trajgen_amd.stream'] = here
        held.append(node)
    return held


# ---------------------------------------------------------------------------------------------------------- dropout
def _drop(x, p, seed, site, step):
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    x = x.contiguous()
    d = _lib.DropoutDesc()
    d.n, d.dtype, d.site, d.seed, d.p = x.numel(), DTYPES[x.dtype], site, seed, p
    if torch.is_tensor(step):
        d.step_dev = _lib.ptr(step)
    else:
        d.step = step
    d.x, d.y = _lib.ptr(x), _lib.ptr(y)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().tsg_dropout(C.byref(d), _lib.current_stream()), 'tsg_dropout')
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, site, step):
        ctx.cfg = (p, seed, site)
        if torch.is_tensor(step):
            ctx.save_for_backward(step)     # advancing it before the backward is an error that autograd reports
        else:
            ctx.step = step
        return _drop(x, p, seed, site, step)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed, site = ctx.cfg
        step = ctx.saved_tensors[0] if ctx.saved_tensors else ctx.step
        return _drop(dy, p, seed, site, step), None, None, None, None


def check_rng(what, p, seed, site, step, dev):
    if not 0.0 <= p <= 1.0:
        raise ValueError('%s: p is a probability, got %r' % (what, p))
    if not 0 <= seed < 1 << 64:
        raise ValueError('%s: seed is a 64-bit unsigned number, got %r' % (what, seed))
    if not 0 <= site < 1 << 32:
        raise ValueError('%s: site is a 32-bit unsigned number, got %r' % (what, site))
    if torch.is_tensor(step):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != dev:
            raise ValueError('%s: step is a number or one int64 on the device of x' % what)
    elif not 0 <= step < 1 << 32:
        raise ValueError('%s: step is a 32-bit unsigned number, got %r' % (what, step))


def dropout(x, p, seed, site=0, step=0):
    """y = x / (1 - p) where kept, 0 where dropped, elements numbered in row-major order of x's shape.

    What is dropped depends on (seed, site, step) and the element's number alone (Philox4x32-10, include/tsg.h): the same
    call gives the same mask, so the backward recomputes it.  Give every dropout of a model its own `site` and every
    training step its own `step`.  `step` may be an int64 tensor of one element on x's device, whose low 32 bits count:
    a captured graph advances it in place (after the backward; autograd refuses the backward otherwise)."""
    dev = _on_device('dropout', x)
    _dtype('dropout', x)
    p, seed, site = float(p), int(seed), int(site)
    step = step if torch.is_tensor(step) else int(step)
    check_rng('dropout', p, seed, site, step, dev)
    held = _hold_leaves(x)
    y = _Dropout.apply(x, p, seed, site, step)
    del held
    return y


# -------------------------------------------------------------------------------------------------------- attention
def _fits(x, per):
    """Whether the kernels can read x [rows][heads][dim] where it lies."""
    return (x.stride(2) == 1 and x.shape[2] % per == 0 and x.stride(0) % per == 0 and x.stride(1) % per == 0
            and x.data_ptr() % 16 == 0)


def _laid_out(x, per, dim):
    """x as the kernels read it: 16-byte aligned rows, width padded with zeros to `dim`."""
    if x.shape[2] == dim and _fits(x, per):
        return x
    if x.shape[2] == dim:
        return x.contiguous() if x.contiguous().data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)
    return torch.nn.functional.pad(x, (0, dim - x.shape[2]))


def _attn_desc(q, k, v, q_ptr, k_ptr, scale, out, stats):
    d = _lib.AttnDesc()
    d.dtype, d.n_seq = DTYPES[q.dtype], q_ptr.numel() - 1
    d.heads, d.kv_heads, d.dim, d.scale = q.shape[1], k.shape[1], q.shape[2], scale
    d.n_q, d.n_k = q.shape[0], k.shape[0]
    d.q_ptr, d.k_ptr = _lib.ptr(q_ptr), _lib.ptr(k_ptr)
    for name, t in (('q', q), ('k', k), ('v', v), ('out', out)):
        setattr(d, name, _lib.ptr(t))
        setattr(d, name + '_row', t.stride(0))
        setattr(d, name + '_head', t.stride(1))
    d.stats = _lib.ptr(stats)
    return d


class _CausalAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_ptr, k_ptr, scale):
        L = _lib.lib()
        dim, per = q.shape[2], 4 if q.dtype == torch.float32 else 8
        wide = -(-dim // per) * per
        ql, kl, vl = (_laid_out(t.detach(), per, wide) for t in (q, k, v))
        out = torch.empty((q.shape[0], q.shape[1], wide), dtype=q.dtype, device=q.device)
        stats = torch.empty((q.shape[1], q.shape[0], 2), dtype=torch.float32, device=q.device)
        d = _attn_desc(ql, kl, vl, q_ptr, k_ptr, scale, out, stats)
        need = C.c_size_t()
        _lib.check(L.tsg_attn_workspace(C.byref(d), C.byref(need)), 'tsg_attn_workspace')
        if need.value:
            ws = torch.empty(need.value, dtype=torch.uint8, device=q.device)
            d.workspace, d.workspace_bytes = _lib.ptr(ws), need.value
        if q.shape[0] and k.shape[0]:
            with torch.cuda.device(q.device):
                _lib.check(L.tsg_attn_forward(C.byref(d), _lib.current_stream()), 'tsg_attn_forward')
        else:
            out.zero_()
        if any(ctx.needs_input_grad[:3]):
            ctx.scale, ctx.dim = scale, dim
            res = out if wide == dim else out[..., :dim].contiguous()
            ctx.save_for_backward(q, k, v, q_ptr, k_ptr, res, stats)
            return res
        return out if wide == dim else out[..., :dim].contiguous()

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        q, k, v, q_ptr, k_ptr, out, stats = ctx.saved_tensors
        dim, per = ctx.dim, 4 if q.dtype == torch.float32 else 8
        wide = -(-dim // per) * per
        ql, kl, vl, ol, gl = (_laid_out(t.detach(), per, wide) for t in (q, k, v, out, d_out))
        dq, dk, dv = (torch.empty(t.shape[:2] + (wide,), dtype=t.dtype, device=t.device) for t in (q, k, v))
        if q.shape[0] and k.shape[0]:
            d = _attn_desc(ql, kl, vl, q_ptr, k_ptr, ctx.scale, ol, stats)
            delta = torch.empty(stats.shape[:2], dtype=torch.float32, device=q.device)
            d.d_out, d.d_out_row, d.d_out_head = _lib.ptr(gl), gl.stride(0), gl.stride(1)
            for name, t in (('dq', dq), ('dk', dk), ('dv', dv)):
                setattr(d, name, _lib.ptr(t))
                setattr(d, name + '_row', t.stride(0))
                setattr(d, name + '_head', t.stride(1))
            d.delta = _lib.ptr(delta)
            with torch.cuda.device(q.device):
                _lib.check(_lib.lib().tsg_attn_backward(C.byref(d), _lib.current_stream()), 'tsg_attn_backward')
        else:
            for t in (dq, dk, dv):
                t.zero_()
        return tuple(t if wide == dim else t[..., :dim].contiguous() for t in (dq, dk, dv)) + (None, None, None)


def _check_ptr(name, p, dev):
    if p.dtype != torch.int32 or p.dim() != 1 or p.numel() < 1 or not p.is_contiguous():
        raise ValueError('causal_attention: %s is a contiguous int32 vector of sequence starts, one more than sequences' % name)


def causal_attention(q, k, v, seq_ptr, kv_ptr=None, scale=None):
    """Causal softmax attention over packed sequences: softmax(scale q k) v, differentiable in q, k and v.

    q [n_q][heads][dim], k and v [n_k][kv_heads][dim], heads a multiple of kv_heads (query head h reads key-value head
    h // (heads / kv_heads)); any strides, copied first where the kernels cannot read them in place.  Sequence s has the
    rows seq_ptr[s] .. seq_ptr[s+1] of q and kv_ptr[s] .. kv_ptr[s+1] of k and v (kv_ptr None: the same positions);
    its last row sees its last key, and a row i places before that i keys fewer.  So a whole prompt, the rest of one, or a
    single new position over what has been kept are the same call.  The pointers are int32 on the device and are
    not checked there (that would wait for the device): starts outside the tensors are clamped.  Rows that see
    nothing, and rows behind the last sequence, give zeros.  scale defaults to 1 / sqrt(dim) and is positive; function G's
    attention (function_g_fc.py:31-35) is one head with scale 1.  dim <= 512."""
    kv_ptr = seq_ptr if kv_ptr is None else kv_ptr
    dev = _on_device('causal_attention', q, k, v, seq_ptr, kv_ptr)
    _dtype('causal_attention', q, k, v)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError('causal_attention: q [n_q][heads][dim] and k, v [n_k][kv_heads][dim], got %s, %s, %s'
                         % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if not 1 <= q.shape[2] <= 512:
        raise ValueError('causal_attention: heads of 1 to 512, got %d' % q.shape[2])
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError('causal_attention: %d heads over %d key-value heads' % (q.shape[1], k.shape[1]))
    _check_ptr('seq_ptr', seq_ptr, dev)
    _check_ptr('kv_ptr', kv_ptr, dev)
    if seq_ptr.numel() != kv_ptr.numel():
        raise ValueError('causal_attention: %d and %d sequences' % (seq_ptr.numel() - 1, kv_ptr.numel() - 1))
    if seq_ptr is kv_ptr and q.shape[0] != k.shape[0]:
        raise ValueError('causal_attention: %d queries at %d positions need a kv_ptr' % (q.shape[0], k.shape[0]))
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError('causal_attention: scale is positive, got %r' % scale)
    held = _hold_leaves(q, k, v)
    out = _CausalAttention.apply(q, k, v, seq_ptr, kv_ptr, scale)
    del held
    return out
