"""Operators over sequences on the HIP kernels of libtsg.so, differentiable under torch's autograd.

    dropout(x, p, seed, site, step)                        mask recomputed from a counter, never stored
    causal_attention(q, k, v, seq_ptr, kv_ptr, scale)      packed sequences, grouped heads, forward and backward
    linear_cross_entropy(h, weight, target, bias, ...)     loss over a large vocabulary, logits never kept

They take tensors on a HIP device (f32, bf16 or f16), run on torch's current stream of that device, allocate their results and
workspaces through torch's allocator and never synchronise, so they can be captured in a graph (forward and backward
together; drop eager results that still hold an autograd graph of the same leaves first, which is checked for leaves that these
operators took themselves; or a forward under no_grad).  Wrong shapes, types or
devices raise ValueError / TypeError / RuntimeError before anything is launched; there is no CPU fallback.  Gradients are
first order: differentiating a gradient raises.
"""
import ctypes as C
import math
import threading
import weakref

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


def _stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev.index)     # torch.cuda.current_stream(dev).cuda_stream without the object


def _ptr(t):
    return None if t is None else t.data_ptr()


_ENTRIES = {}


def _call(entry, d, dev):
    """entry(d, the current stream of dev) of libtsg, with dev current: a call is a few microseconds of host time all told."""
    fn = _ENTRIES.get(entry) or _ENTRIES.setdefault(entry, getattr(_lib.lib(), entry))
    if torch._C._cuda_getDevice() == dev.index:
        rc = fn(C.byref(d), _stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(C.byref(d), _stream(dev))
    if rc:
        _lib.check(rc, entry)


_LIVE = weakref.WeakSet()     # the operators' own nodes in autograd graphs that are alive
_LIVE_LOCK = threading.Lock()


def _enter(ctx, *inputs):
    """Notes a node, its leaves and the stream it was made on.

    Capturing a backward while an eager autograd graph of the same leaf is alive ends the process: the leaf's gradient
    accumulator is tied to the stream that graph was made on, and joining that stream breaks the capture.  So a call under
    capture that finds a living node of another stream over one of its leaves refuses."""
    leaves = {id(t) for t in inputs if t is not None and t.requires_grad and t.is_leaf}
    if not leaves:
        return
    here = _stream(inputs[0].device)
    if torch.cuda.is_current_stream_capturing():
        with _LIVE_LOCK:
            nodes = list(_LIVE)
        for node in nodes:
            if node.stream != here and not leaves.isdisjoint(node.leaves):
                raise RuntimeError('capture of a backward while an eager autograd graph of the same leaf is alive: drop the '
                                   'eager results (del, or .detach() what is kept) before capturing')
    ctx.leaves, ctx.stream = leaves, here
    with _LIVE_LOCK:
        _LIVE.add(ctx)


def _inputs(*tensors):
    """As an operator's node takes them: under no_grad no backward follows, and a node has nothing to note or keep for one."""
    if torch.is_grad_enabled():
        return tensors
    return [t.detach() if t is not None and t.requires_grad else t for t in tensors]


def _save(ctx, *tensors):
    """Everything a backward reads goes through autograd's saved tensors: hooks may move it or bring it back from elsewhere (then
    the operands may be written meanwhile), and a backward that does not keep its graph lets go of it."""
    ctx.save_for_backward(*tensors)
    ctx.like = [None if t is None else (t.shape, t.dtype, t.device) for t in tensors]


def _saved(what, ctx):
    """The saved tensors.  What a hook brings back has other addresses and strides; other shapes, types or devices would be read
    as what they are not."""
    tensors = ctx.saved_tensors
    now = [None if t is None else (t.shape, t.dtype, t.device) for t in tensors]
    if now != ctx.like:
        raise RuntimeError('%s: saved tensors %s came back as %s' % (what, ctx.like, now))
    return tensors


# ---------------------------------------------------------------------------------------------------------- dropout
def _drop(x, p, seed, site, step):
    x = x.contiguous()
    y = torch.empty_like(x)
    on_device = torch.is_tensor(step)
    _call('tsg_dropout', _lib.DropoutDesc(x.numel(), DTYPES[x.dtype], site, 0 if on_device else step, 0, seed, p,
                                          step.data_ptr() if on_device else None, x.data_ptr(), y.data_ptr()), x.device)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed, site, step):
        _enter(ctx, x)
        ctx.cfg = (p, seed, site)
        if torch.is_tensor(step):
            _save(ctx, step)                # advancing it before the backward is an error that autograd reports
            ctx.step = None
        else:
            ctx.step = step
        return _drop(x, p, seed, site, step)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed, site = ctx.cfg
        step = _saved('dropout', ctx)[0] if ctx.step is None else ctx.step
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
    return _Dropout.apply(*_inputs(x), p, seed, site, step)


# -------------------------------------------------------------------------------------------------------- attention
def _laid_out(x, per, dim):
    """x [rows][heads][width] as the kernels read it: 16-byte aligned rows, width padded with zeros to `dim`."""
    if x.shape[2] != dim:
        return torch.nn.functional.pad(x, (0, dim - x.shape[2]))
    row, head, one = x.stride()
    if (one == 1 and row % per == 0 and head % per == 0 and row * x.element_size() < 1 << 24 and x.data_ptr() % 16 == 0):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _attn_desc(q, k, v, q_ptr, k_ptr, scale, out, stats, rest):
    a, b, c, e = q.stride(), k.stride(), v.stride(), out.stride()
    return _lib.AttnDesc(DTYPES[q.dtype], q_ptr.numel() - 1, q.shape[1], k.shape[1], q.shape[2], scale, q.shape[0], k.shape[0],
                         q_ptr.data_ptr(), k_ptr.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                         a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1], stats.data_ptr(), _ptr(rest))


def _sizes(entry, d):
    """Workspace bytes of the forward and of the backward."""
    sizes = C.c_size_t(), C.c_size_t()
    _lib.check(getattr(_lib.lib(), entry)(C.byref(d), C.byref(sizes[0]), C.byref(sizes[1])), entry)
    return sizes[0].value, sizes[1].value


def _workspace(d, need, dev):
    if not need:
        d.workspace, d.workspace_bytes = None, 0
        return None
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    return ws


class _CausalAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_ptr, k_ptr, scale):
        _enter(ctx, q, k, v)
        dev, dim, per = q.device, q.shape[2], 4 if q.dtype == torch.float32 else 8
        wide = -(-dim // per) * per
        n_q, heads = q.shape[0], q.shape[1]
        train = any(ctx.needs_input_grad[:3])
        out = torch.empty((n_q, heads, wide), dtype=q.dtype, device=dev)
        stats = torch.empty(3 * heads * n_q, dtype=torch.float32, device=dev)      # [heads][n_q][2], then delta [heads][n_q]
        rest = torch.empty_like(out) if train and per == 8 else None
        ctx.need = None
        if n_q and k.shape[0]:
            ql, kl, vl = _laid_out(q, per, wide), _laid_out(k, per, wide), _laid_out(v, per, wide)
            d = _attn_desc(ql, kl, vl, q_ptr, k_ptr, scale, out, stats, rest)
            sizes = _sizes('tsg_attn_workspace', d)
            ws = _workspace(d, sizes[0], dev)  # noqa: F841  (held until the launches are on the stream)
            _call('tsg_attn_forward', d, dev)
            if train:
                ctx.need, ctx.desc = sizes[1], d
                ctx.strides = ql.stride(), kl.stride(), vl.stride(), out.stride()
                _save(ctx, ql, kl, vl, q_ptr, None if k_ptr is q_ptr else k_ptr, out, stats, rest)
        else:
            out.zero_()
        ctx.size = n_q, k.shape[0], heads, k.shape[1], dim, wide, per
        return out if wide == dim else out[..., :dim].contiguous()

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        n_q, n_k, heads, kv_heads, dim, wide, per = ctx.size
        dev, dt = d_out.device, d_out.dtype
        dq = torch.empty((n_q, heads, wide), dtype=dt, device=dev)
        dk = torch.empty((n_k, kv_heads, wide), dtype=dt, device=dev)
        dv = torch.empty_like(dk)
        if ctx.need is not None:
            q, k, v, q_ptr, k_ptr, out, stats, rest = _saved('causal_attention', ctx)
            # the forward's sizes; every address anew, and the strides where a hook brought back others
            d, at = _lib.AttnDesc.from_buffer_copy(ctx.desc), [t.data_ptr() for t in (q, k, v, out)]
            if (at[0] | at[1] | at[2] | at[3]) & 15 or (q.stride(), k.stride(), v.stride(), out.stride()) != ctx.strides:
                q, k, v, out = [_laid_out(t, per, wide) for t in (q, k, v, out)]
                at = [t.data_ptr() for t in (q, k, v, out)]
                (d.q_row, d.q_head), (d.k_row, d.k_head), (d.v_row, d.v_head), (d.out_row, d.out_head) = [
                    t.stride()[:2] for t in (q, k, v, out)]
            q_ptr, stats = q_ptr.contiguous(), stats.contiguous()
            k_ptr = q_ptr if k_ptr is None else k_ptr.contiguous()
            rest = None if rest is None else rest.contiguous()
            d.q, d.k, d.v, d.out = at
            d.q_ptr, d.k_ptr, d.stats, d.out_rest = q_ptr.data_ptr(), k_ptr.data_ptr(), stats.data_ptr(), _ptr(rest)
            gl = _laid_out(d_out, per, wide)
            d.d_out, d.dq, d.dk, d.dv = gl.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
            d.delta = d.stats + 8 * heads * n_q
            d.d_out_row, d.d_out_head = gl.stride(0), gl.stride(1)
            d.dq_row, d.dk_row, d.dv_row = heads * wide, kv_heads * wide, kv_heads * wide
            d.dq_head = d.dk_head = d.dv_head = wide
            ws = _workspace(d, ctx.need, dev)  # noqa: F841
            _call('tsg_attn_backward', d, dev)
        else:
            for t in (dq, dk, dv):
                t.zero_()
        if wide != dim:
            dq, dk, dv = (t[..., :dim].contiguous() for t in (dq, dk, dv))
        return dq, dk, dv, None, None, None


def _check_ptr(name, p):
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
    _on_device('causal_attention', q, k, v, seq_ptr, kv_ptr)
    _dtype('causal_attention', q, k, v)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[2] != k.shape[2]:
        raise ValueError('causal_attention: q [n_q][heads][dim] and k, v [n_k][kv_heads][dim], got %s, %s, %s'
                         % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if not 1 <= q.shape[2] <= 512:
        raise ValueError('causal_attention: heads of 1 to 512, got %d' % q.shape[2])
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError('causal_attention: %d heads over %d key-value heads' % (q.shape[1], k.shape[1]))
    _check_ptr('seq_ptr', seq_ptr)
    _check_ptr('kv_ptr', kv_ptr)
    if seq_ptr.numel() != kv_ptr.numel():
        raise ValueError('causal_attention: %d and %d sequences' % (seq_ptr.numel() - 1, kv_ptr.numel() - 1))
    if seq_ptr is kv_ptr and q.shape[0] != k.shape[0]:
        raise ValueError('causal_attention: %d queries at %d positions need a kv_ptr' % (q.shape[0], k.shape[0]))
    scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError('causal_attention: scale is positive, got %r' % scale)
    return _CausalAttention.apply(*_inputs(q, k, v), seq_ptr, kv_ptr, scale)


# ---------------------------------------------------------------------------------------------------- cross entropy
REDUCTIONS = {'none': 0, 'sum': 1, 'mean': 2}


def _rows_for(x, wide):
    """x [rows][width] as the kernels read it: rows 16-byte aligned, padded with zeros to `wide`."""
    per = 4 if x.dtype == torch.float32 else 8
    if x.shape[1] != wide:
        return torch.nn.functional.pad(x, (0, wide - x.shape[1]))
    if x.stride(1) == 1 and x.stride(0) >= wide and x.stride(0) % per == 0 and x.stride(0) < 1 << 21 and x.data_ptr() % 16 == 0:
        return x
    return x.clone(memory_format=torch.contiguous_format)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, w, bias, target, ignore, reduction):
        _enter(ctx, h, w, bias)
        dev, rows, wide = h.device, h.shape[0], -(-h.shape[1] // 8) * 8
        hl, wl = _rows_for(h, wide), _rows_for(w, wide)
        bl = None if bias is None else bias.contiguous()
        tl = target.contiguous()
        store = torch.empty(3 * rows + 2, dtype=torch.float32, device=dev)
        loss = torch.empty(rows if reduction == 0 else (), dtype=torch.float32, device=dev)
        at = store.data_ptr()        # [rows][2] stats, [rows] losses, [2] scales of f32 operands
        d = _lib.XentDesc(DTYPES[h.dtype], wide, reduction, 0, rows, w.shape[0], ignore, hl.data_ptr(), wl.data_ptr(), _ptr(bl),
                          max(hl.stride(0), wide), max(wl.stride(0), wide), tl.data_ptr(),
                          loss.data_ptr() if reduction == 0 else at + 8 * rows, loss.data_ptr(), at,
                          at + 12 * rows if h.dtype == torch.float32 else None)
        sizes = _sizes('tsg_xent_workspace', d)
        ws = _workspace(d, sizes[0], dev)  # noqa: F841
        _call('tsg_xent_forward', d, dev)
        if any(ctx.needs_input_grad[:3]):
            ctx.cfg, ctx.desc = (h.shape[1], wide, sizes[1]), d
            _save(ctx, hl, wl, bl, tl, store)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, d_loss):
        width, wide, need = ctx.cfg
        h, w, bias, target, store = _saved('linear_cross_entropy', ctx)
        dev, rows, dt = h.device, h.shape[0], h.dtype
        h, w, target, store = _rows_for(h, wide), _rows_for(w, wide), target.contiguous(), store.contiguous()
        bias = None if bias is None else bias.contiguous()
        d_loss = d_loss.contiguous()
        dh = torch.empty((rows, wide), dtype=dt, device=dev)
        dw = torch.empty((w.shape[0], wide), dtype=dt, device=dev)
        db = None if bias is None else torch.empty(w.shape[0], dtype=dt, device=dev)
        d = _lib.XentDesc.from_buffer_copy(ctx.desc)         # the forward's sizes; every address and stride anew
        d.h, d.w, d.bias, d.target, d.stats = h.data_ptr(), w.data_ptr(), _ptr(bias), target.data_ptr(), store.data_ptr()
        d.h_row, d.w_row = max(h.stride(0), wide), max(w.stride(0), wide)
        d.row_loss, d.loss, d.scales = None, None, d.stats + 12 * rows if dt == torch.float32 else None
        d.d_loss, d.dh, d.dw, d.dbias = d_loss.data_ptr(), dh.data_ptr(), dw.data_ptr(), _ptr(db)
        d.dh_row = d.dw_row = wide
        ws = _workspace(d, need, dev)  # noqa: F841
        _call('tsg_xent_backward', d, dev)
        if wide != width:
            dh, dw = dh[:, :width].contiguous(), dw[:, :width].contiguous()
        return dh, dw, db, None, None, None


def linear_cross_entropy(h, weight, target, bias=None, ignore_index=-100, reduction='mean'):
    """Cross entropy of softmax(h weight^T + bias) against target, differentiable in h, weight and bias, without the
    [rows][vocabulary] logits being kept (their gradient exists in pieces of the vocabulary, in the backward only: a quarter of the logits,
    between 384 MiB and 2 GiB).

    h [rows][hidden], weight [vocabulary][hidden] (function G's out_fc.weight, function_g_fc.py:134), bias [vocabulary] or
    None, all of one type (f32, bf16 or f16); target int64 [rows].  The loss is f32: per row ('none'), their sum
    ('sum') or their mean over the rows whose target is not ignore_index ('mean'; NaN when there is none).  Rows with
    ignore_index have loss 0 and add nothing to any gradient.  A target outside the vocabulary cannot be refused without
    waiting for the device: it makes its row's loss and gradients NaN."""
    _on_device('linear_cross_entropy', h, weight, bias, target)
    _dtype('linear_cross_entropy', h, weight, bias)
    if h.dim() != 2 or weight.dim() != 2 or h.shape[1] != weight.shape[1] or h.shape[1] < 1:
        raise ValueError('linear_cross_entropy: h [rows][hidden] and weight [vocabulary][hidden], got %s and %s'
                         % (tuple(h.shape), tuple(weight.shape)))
    if h.shape[0] < 1 or weight.shape[0] < 1:
        raise ValueError('linear_cross_entropy: at least one row and one entry, got %d and %d' % (h.shape[0], weight.shape[0]))
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError('linear_cross_entropy: bias of %d entries, got %s' % (weight.shape[0], tuple(bias.shape)))
    if target.dtype != torch.int64 or tuple(target.shape) != (h.shape[0],):
        raise ValueError('linear_cross_entropy: target is int64 [rows], got %s %s' % (target.dtype, tuple(target.shape)))
    if reduction not in REDUCTIONS:
        raise ValueError("linear_cross_entropy: reduction is 'none', 'sum' or 'mean', got %r" % (reduction,))
    return _LinearCrossEntropy.apply(*_inputs(h, weight, bias), target, int(ignore_index), REDUCTIONS[reduction])
