"""FunctionGFC drop-in (function G; reference: generator/function_g_fc.py:105-136 constructor).

Holds the reference's parameters under the reference's names (`road_emb`, `time_emb`, `lstm`,
`intra_attn.w1/w2/w3` -- unused by the reference too, function_g_fc.py:17-19 -- and `out_fc`).  The
arithmetic (incremental LSTM cell on MFMA, attention over the prefix, gathered out_fc rows) lives in
libtsg.so and is driven by GeneratorV4 / the engine, which need G and H together; `forward` / `predict` /
`predict_g` (function_g_fc.py:138-221) return G's share of that evaluation.  `trajectory_loss` fits function G on whole
trajectories: the next road at every position, over all roads, differentiable (ts_trajgen_amd.ops)."""
import torch
import torch.nn as nn

from .. import ops


class IntraAttention(nn.Module):
    def __init__(self, hidden_size):
        super().__init__()
        self.hidden_size = hidden_size
        self.w1 = nn.Linear(in_features=hidden_size, out_features=1, bias=False)
        self.w2 = nn.Linear(in_features=hidden_size, out_features=hidden_size, bias=False)
        self.w3 = nn.Linear(in_features=hidden_size, out_features=hidden_size, bias=False)


class FunctionGFC(nn.Module):
    def __init__(self, config, data_feature):
        super().__init__()
        self.road_emb_size = config['road_emb_size']
        self.time_emb_size = config['time_emb_size']
        self.hidden_size = config['hidden_size']
        self.lstm_layer_num = config['lstm_layer_num']
        self.dropout_p = config['dropout_p']
        self.dis_weight = config['dis_weight']
        self.input_size = self.road_emb_size + self.time_emb_size
        self.road_emb = nn.Embedding(num_embeddings=data_feature['road_num'], embedding_dim=self.road_emb_size,
                                     padding_idx=data_feature['road_pad'])
        self.time_emb = nn.Embedding(num_embeddings=data_feature['time_size'], embedding_dim=self.time_emb_size,
                                     padding_idx=data_feature['time_pad'])
        self.lstm = nn.LSTM(input_size=self.input_size, hidden_size=self.hidden_size,
                            num_layers=self.lstm_layer_num, batch_first=True)
        self.intra_attn = IntraAttention(hidden_size=self.hidden_size)
        self.dropout = nn.Dropout(p=self.dropout_p)
        self.out_fc = nn.Linear(in_features=self.hidden_size, out_features=data_feature['road_num'])

    def predict_g(self, trace_loc, trace_time, des, candidate_set, candidate_dis, trace_mask=None):
        """softmax over the candidates of function G alone (function_g_fc.py:206-221); same arguments."""
        from .generator_v4 import owner_of
        owner = owner_of(self, 'function_g')
        if owner is None:
            raise RuntimeError('FunctionGFC.predict_g runs through the device tables of its GeneratorV4: '
                               'construct the module as GeneratorV4(config, data_feature).function_g')
        return owner.predict_parts(trace_loc, trace_time, des, candidate_set, candidate_dis, trace_mask)[1]

    def forward(self, trace_loc, trace_time, des, candidate_set, candidate_dis, trace_mask=None, train=True):
        """The candidates' scores before the softmax: out_fc(attention-pooled LSTM state)[candidate_set]
        (function_g_fc.py:138-187), for a module in inference mode (the dropouts of :160,182 are then the
        identity; `train` is unused by the reference too).  Computed by the scoring kernel, which gathers only
        the candidates' rows of out_fc."""
        if self.training:
            raise NotImplementedError('FunctionGFC.forward with live dropout (training) is outside the generation '
                                      'path: call .train(False) first (our_model_generate.py:399)')
        from .generator_v4 import owner_of
        owner = owner_of(self, 'function_g')
        if owner is None:
            raise RuntimeError('FunctionGFC.forward runs through the device tables of its GeneratorV4: '
                               'construct the module as GeneratorV4(config, data_feature).function_g')
        return owner.predict_parts(trace_loc, trace_time, des, candidate_set, candidate_dis, trace_mask,
                                   logits=True)[3]

    def predict(self, trace_loc, trace_time, des, candidate_set, candidate_dis, trace_mask=None):
        """softmax of forward() over the candidates (function_g_fc.py:189-204)."""
        return self.predict_g(trace_loc, trace_time, des, candidate_set, candidate_dis, trace_mask)

    def trajectory_loss(self, trace_loc, trace_time, seq_ptr, target=None, reduction='mean', seed=0, step=None):
        """Cross entropy of the next road at every position of packed trajectories, over all roads (the score of
        function_g_fc.py:155-184 before its gather, at every prefix at once).

        trace_loc and trace_time hold the trajectories one behind the other ([n] integers), seq_ptr ([n_seq + 1] int32)
        their starts.  target ([n] int64, -100 = not counted) defaults to the next road of the same trajectory; positions of
        no trajectory never count.  In training mode the dropouts of function_g_fc.py:160,182 are live, drawn from the
        counter (seed, site 0 and 1, step): every training step needs a step of its own, and a call without one is refused.
        hidden_size is at most 512 (ops.causal_attention).  In inference mode torch's recurrence has no backward.  The call waits for the
        device once: it looks at the lengths and ids."""
        drop = self.dropout_p if self.training else 0.0
        if drop and step is None:
            raise ValueError('trajectory_loss: the dropouts are live, give every training step a step of its own (the same step '
                             'drops the same elements)')
        dev = self.out_fc.weight.device
        if dev.type != 'cuda':
            raise RuntimeError('FunctionGFC.trajectory_loss needs its parameters on a HIP device (no CPU fallback)')
        loc, tim, ptr = trace_loc.to(dev).long(), trace_time.to(dev).long(), seq_ptr.to(dev)
        if loc.dim() != 1 or loc.shape != tim.shape or not loc.numel():
            raise ValueError('trajectory_loss: trace_loc and trace_time are [n], n >= 1, got %s and %s'
                             % (tuple(loc.shape), tuple(tim.shape)))
        if ptr.dim() != 1 or ptr.dtype != torch.int32 or ptr.numel() < 2:
            raise ValueError('trajectory_loss: seq_ptr is int32 [n_seq + 1], n_seq >= 1')
        if target is not None and (target.shape != loc.shape or target.dtype != torch.int64):
            raise ValueError('trajectory_loss: target is int64 [n]')
        n = loc.shape[0]
        lens = ptr[1:] - ptr[:-1]
        first, end, least, longest, loc0, loc1, tim0, tim1 = torch.stack(
            [v.long() for v in (ptr[0], ptr[-1], lens.min(), lens.max(), loc.min(), loc.max(), tim.min(), tim.max())]).tolist()
        if first < 0 or end > n or least < 0:
            raise ValueError('trajectory_loss: seq_ptr does not grow inside [0, %d]' % n)
        if loc0 < 0 or loc1 >= self.road_emb.num_embeddings or tim0 < 0 or tim1 >= self.time_emb.num_embeddings:
            raise ValueError('trajectory_loss: an id is outside its embedding')
        at = torch.arange(n, device=dev, dtype=torch.int32)
        inside = (at >= first) & (at < end)
        seq = (torch.searchsorted(ptr, at, right=True) - 1).clamp_(0, ptr.numel() - 2)
        pos = torch.where(inside, at - ptr[seq], torch.zeros_like(at)).long()
        if target is None:
            target = torch.where(pos == lens[seq] - 1, torch.full_like(loc, -100), torch.roll(loc, -1))
        target = torch.where(inside, target.to(dev), torch.full_like(loc, -100))
        x = torch.cat([self.road_emb(loc), self.time_emb(tim)], dim=1)
        if drop:
            x = ops.dropout(x, drop, seed, site=0, step=step)
        # the recurrence runs over the padded batch; what it computes behind a trajectory's end is never looked at
        grid = (ptr[:-1].long().unsqueeze(1) + torch.arange(max(longest, 1), device=dev)).clamp_(max=n - 1)
        h = self.lstm(x[grid])[0][seq, pos]
        q = h.unsqueeze(1)
        a = ops.causal_attention(q, q, q, ptr, scale=1.0).squeeze(1)
        if drop:
            a = ops.dropout(a, drop, seed, site=1, step=step)
        # one type: under autocast the recurrence's, as a linear layer would have it
        return ops.linear_cross_entropy(a, self.out_fc.weight.to(a.dtype), target, bias=self.out_fc.bias.to(a.dtype), reduction=reduction)
