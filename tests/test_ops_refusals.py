"""What the sequence operators (ts_trajgen_amd.ops) refuse before anything is launched: no GPU needed."""
import ctypes as C

import pytest
import torch

from ts_trajgen_amd import _lib, ops


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 64)
    p = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        ops.dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        ops.causal_attention(x, x, x, p)
    with pytest.raises(TypeError):
        ops.dropout([1.0], 0.5, 1)


@pytest.mark.parametrize('kw', [dict(p=-0.1), dict(p=1.5), dict(p=float('nan')), dict(seed=-1), dict(seed=1 << 64),
                                dict(site=1 << 32), dict(step=-1), dict(step=1 << 32),
                                dict(step=torch.zeros(2, dtype=torch.int64)), dict(step=torch.zeros(1))])
def test_dropout_generator_arguments(kw):
    a = dict(p=0.5, seed=1, site=0, step=0)
    a.update(kw)
    with pytest.raises(ValueError):
        ops.check_rng('dropout', a['p'], a['seed'], a['site'], a['step'], torch.device('cpu'))


def _dropout(**kw):
    d = _lib.DropoutDesc()
    d.n, d.dtype, d.p, d.x, d.y = 8, 0, 0.5, 4096, 4096
    for k, v in kw.items():
        setattr(d, k, v)
    return _lib.lib().tsg_dropout(C.byref(d), None)


def test_dropout_descriptor():
    assert _lib.lib().tsg_dropout(None, None) == -1
    assert _dropout(n=0) == 0
    for kw in (dict(n=-1), dict(dtype=3), dict(p=1.5), dict(p=float('nan')), dict(x=None), dict(y=None)):
        assert _dropout(**kw) == -1


def _attn(entry='tsg_attn_forward', **kw):
    d = _lib.AttnDesc()
    d.dtype, d.n_seq, d.heads, d.kv_heads, d.dim, d.scale, d.n_q, d.n_k = 1, 1, 4, 2, 64, 0.125, 10, 10
    for n in ('q_ptr', 'k_ptr', 'q', 'k', 'v', 'out', 'stats', 'd_out', 'dq', 'dk', 'dv', 'delta'):
        setattr(d, n, 4096)
    for n in ('q', 'k', 'v', 'out', 'd_out', 'dq', 'dk', 'dv'):
        setattr(d, n + '_row', 256)
        setattr(d, n + '_head', 64)
    for k, v in kw.items():
        setattr(d, k, v)
    return getattr(_lib.lib(), entry)(C.byref(d), None)


@pytest.mark.parametrize('kw,rc', [
    (dict(dtype=7), -1), (dict(heads=3), -1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(dim=0), -1),
    (dict(dim=20), -1), (dict(dim=520), -3), (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float('nan')), -1),
    (dict(scale=float('inf')), -1), (dict(n_seq=-1), -1), (dict(n_k=-1), -1), (dict(q=None), -1), (dict(v=None), -1),
    (dict(out=None), -1), (dict(stats=None), -1), (dict(q_ptr=None), -1), (dict(k=4100), -1), (dict(q_row=252), -1),
    (dict(v_head=-64), -1), (dict(n_q=1 << 31), -3), (dict(n_k=1 << 30, kv_heads=4), -3), (dict(n_q=1, n_k=100000), -2)])
def test_attention_descriptor(kw, rc):
    assert _attn(**kw) == rc


def test_attention_backward_descriptor():
    for kw in (dict(d_out=None), dict(dq=None), dict(dk=None), dict(dv=4), dict(delta=None), dict(d_out_row=3)):
        assert _attn('tsg_attn_backward', **kw) == -1


def _xent(entry='tsg_xent_forward', **kw):
    d = _lib.XentDesc()
    d.dtype, d.hidden, d.reduction, d.n_rows, d.n_vocab, d.ignore_index = 0, 64, 2, 10, 100, -100
    for n in ('h', 'w', 'bias', 'target', 'row_loss', 'loss', 'stats', 'scales', 'd_loss', 'dh', 'dw', 'dbias', 'workspace'):
        setattr(d, n, 4096)
    d.h_row = d.w_row = d.dh_row = d.dw_row = 64
    for k, v in kw.items():
        setattr(d, k, v)
    return getattr(_lib.lib(), entry)(C.byref(d), None)


@pytest.mark.parametrize('kw,rc', [
    (dict(dtype=3), -1), (dict(hidden=0), -1), (dict(hidden=60), -1), (dict(reduction=3), -1), (dict(n_rows=0), -1),
    (dict(n_rows=-1), -1), (dict(n_vocab=0), -1), (dict(n_rows=1 << 31), -3), (dict(n_vocab=1 << 31), -3), (dict(h=None), -1),
    (dict(w=None), -1), (dict(target=None), -1), (dict(stats=None), -1), (dict(row_loss=None), -1), (dict(loss=None), -1), (dict(scales=None), -1),
    (dict(h=4100), -1), (dict(h_row=56), -1), (dict(w_row=66), -1), (dict(workspace=None), -2), (dict(workspace_bytes=8), -2)])
def test_cross_entropy_descriptor(kw, rc):
    assert _xent(**kw) == rc


def test_cross_entropy_backward_descriptor():
    for kw in (dict(d_loss=None), dict(dh=None), dict(dw=None), dict(dbias=None), dict(dh_row=8), dict(dh_row=66), dict(dh=4100), dict(dw_row=8), dict(dw_row=66), dict(dw=4100)):
        assert _xent('tsg_xent_backward', **kw) == -1
    assert _xent('tsg_xent_backward', workspace_bytes=100) == -2


def test_cross_entropy_refuses_cpu_tensors():
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        ops.linear_cross_entropy(torch.zeros(2, 8), torch.zeros(5, 8), torch.zeros(2, dtype=torch.int64))


def test_attention_backward_of_one_long_sequence_needs_its_workspace():
    assert _attn('tsg_attn_backward', n_q=4096, n_k=4096) == -2
    assert _attn('tsg_attn_backward', n_q=4096, n_k=4096, workspace=4104, workspace_bytes=1 << 40) == -2


def test_encoder_entries_with_a_generator_refuse_before_any_launch():
    import ctypes as C
    from ts_trajgen_amd import _lib
    L = _lib.lib()
    for entry in (L.tsg_gat_train_forward_rng, L.tsg_gat_train_backward_rng):
        d, ok = _lib.GatTrain(), _lib.GatDropout(0.5, 1, 0, 0, None)
        assert entry(None, C.byref(ok), None) < 0
        assert entry(C.byref(d), None, None) < 0
        assert entry(C.byref(d), C.byref(ok), None) < 0         # an empty description of the layer
        for bad in [(-0.1, 1, 0), (1.5, 1, 0), (float('nan'), 1, 0), (0.5, 1, (1 << 32) - 2)]:
            assert entry(C.byref(d), C.byref(_lib.GatDropout(*bad, 0, None)), None) < 0
        for mask in ('m_in', 'm_proj', 'm_att'):                # masks, or a generator
            d = _lib.GatTrain()
            setattr(d, mask, 4096)
            assert entry(C.byref(d), C.byref(ok), None) < 0


def test_live_dropouts_of_function_g_need_a_step():
    """The same step draws the same masks, so a caller who gives none would train on one mask for ever."""
    from ts_trajgen_amd.generator.function_g_fc import FunctionGFC
    conf = {'road_emb_size': 8, 'time_emb_size': 8, 'hidden_size': 16, 'lstm_layer_num': 1, 'dropout_p': 0.5, 'dis_weight': 0.5}
    m = FunctionGFC(conf, {'road_num': 20, 'road_pad': 19, 'time_size': 20, 'time_pad': 19}).train(True)
    loc, ptr = torch.zeros(4, dtype=torch.int64), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match='step'):
        m.trajectory_loss(loc, loc, ptr)
    with pytest.raises(RuntimeError, match='HIP device'):       # the parameters are not on a device: the next check
        m.trajectory_loss(loc, loc, ptr, step=0)
    with pytest.raises(RuntimeError, match='HIP device'):
        m.train(False).trajectory_loss(loc, loc, ptr)
    m.dropout_p = 0.0
    with pytest.raises(RuntimeError, match='HIP device'):
        m.train(True).trajectory_loss(loc, loc, ptr)


@pytest.mark.parametrize('dtype,rows,vocab,hidden', [(0, 8192, 40307, 256), (1, 16384, 50021, 1024), (2, 16384, 50021, 512), (1, 65536, 131072, 512)])
@pytest.mark.parametrize('reduction', [0, 2])
def test_cross_entropy_workspace_is_a_fraction_of_the_logits(dtype, rows, vocab, hidden, reduction):
    """The logits' gradient exists for a piece of the vocabulary at a time: 384 MiB, next to what grows with h and W alone
    (f32: their two planes; dh in f32; with reduction 0 h once more; dW in f32 where its rows are cut, of one piece)."""
    d = _lib.XentDesc()
    d.dtype, d.hidden, d.reduction, d.n_rows, d.n_vocab = dtype, hidden, reduction, rows, vocab
    fwd, bwd = C.c_size_t(), C.c_size_t()
    assert _lib.lib().tsg_xent_workspace(C.byref(d), C.byref(fwd), C.byref(bwd)) == 0
    each = 4 if dtype == 0 else 2
    logits = rows * vocab * each
    assert bwd.value < 0.5 * logits and fwd.value < 0.1 * logits
    assert bwd.value < (384 << 20) + 4 * hidden * (8 * vocab + 12 * rows)
