"""ModelBiLSTM's forward pass as a training step needs it: the graph of models.py:178-240 with its dropouts (models.py:137-157,
:234-236), over the operators of train_ops.py.  ModelBiLSTM.train() switches to it; eval() goes back to the inference kernels.

What is left to torch is elementwise: relu, dropout, the final softmax, concatenation."""
from __future__ import annotations

import torch
from torch.nn import functional as F

from . import train_ops as ops

_NAMES = ("weight_ih", "weight_hh", "bias_ih", "bias_hh")


def _bilstm(model, p, prefix, layers, x, h0, c0):
    """the layers of one nn.LSTM(batch_first, bidirectional, dropout): dropout on what a layer hands to the next one"""
    for k in range(layers):
        if k and model.dropout_rate:
            x = F.dropout(x, model.dropout_rate)
        weights = [p["%s.%s_l%d%s" % (prefix, name, k, way)] for way in ("", "_reverse") for name in _NAMES]
        x = ops.lstm(x, weights, None if h0 is None else h0[2 * k:2 * k + 2], None if c0 is None else c0[2 * k:2 * k + 2])[0]
    return x


def forward(model, p, kmer, base_means, base_stds, base_signal_lens, signals, init_states):
    """(logits, probabilities) of model's parameters p (name -> leaf tensor on its GPU)"""
    dev, L = torch.device("cuda", model._device_index()), model.seq_len
    states = init_states or {}

    def feature(t, name):
        if t is None or not t.is_cuda or t.device != dev:
            raise RuntimeError("ModelBiLSTM.forward: %s must live on %s (no CPU path)" % (name, dev))
        return t

    def initial(name, layers, hidden, n):
        # init_hidden (models.py:169-176): N(0, 1) from torch's generator, unless the caller or the model says otherwise
        for s in ("h_", "c_"):
            t = states.get(s + name)
            if t is not None:
                t = t.to(device=dev, dtype=torch.float32)
                if tuple(t.shape) != (2 * layers, n, hidden):
                    raise ValueError("initial state %s has shape %s, expected %s" % (s + name, tuple(t.shape), (2 * layers, n, hidden)))
            elif init_states is None and model.init_state == "randn":
                t = torch.randn(2 * layers, n, hidden, device=dev)
            yield t

    parts = []
    if model.module != "signal_bilstm":
        means = feature(base_means, "base_means")
        n = means.shape[0]
        column = lambda t, name: feature(t, name).reshape(n, L, 1).float()
        x = [column(means, "base_means"), column(base_stds, "base_stds")]
        if model.is_base:
            codes = feature(kmer, "kmer").reshape(n, L)
            x.insert(0, ops.embedding(codes if codes.dtype in ops.TOKEN_TYPES else codes.float(), p["embed.weight"]))
        if model.is_signallen:
            x.append(column(base_signal_lens, "base_signal_lens"))
        hidden = p["fc_seq.weight"].shape[0]
        x = _bilstm(model, p, "lstm_seq", model.num_layers2, torch.cat(x, 2), *initial("seq", model.num_layers2, hidden, n))
        parts.append(F.relu(ops.linear(x, p["fc_seq.weight"], p["fc_seq.bias"])))
    if model.module != "seq_bilstm":
        x = feature(signals, "signals")
        n = x.shape[0]
        hidden = p["fc_signal.weight"].shape[0]
        x = _bilstm(model, p, "lstm_signal", model.num_layers2, x.reshape(n, L, model.signal_len).float(), *initial("sig", model.num_layers2, hidden, n))
        parts.append(F.relu(ops.linear(x, p["fc_signal.weight"], p["fc_signal.bias"])))
    H = model.hidden_size
    x = parts[0] if len(parts) == 1 else torch.cat(parts, 2)
    x = _bilstm(model, p, "lstm_comb", model.num_layers1, x, *initial("comb", model.num_layers1, H, n))
    x = torch.cat((x[:, -1, :H], x[:, 0, H:]), 1)
    drop = (lambda t: F.dropout(t, model.dropout_rate)) if model.dropout_rate else (lambda t: t)
    x = F.relu(drop(ops.linear(drop(x), p["fc1.weight"], p["fc1.bias"])))
    logits = ops.linear(x, p["fc2.weight"], p["fc2.bias"])
    return logits, torch.softmax(logits, 1)
