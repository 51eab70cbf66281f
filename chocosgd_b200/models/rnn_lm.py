"""Word-level LSTM language model: embedding -> dropout -> LSTM stack -> dropout -> decoder,
optional weight tying, uniform(-0.1, 0.1) init (``dl_code/pcode/models/rnn_lm.py:7-75``).

``nffn > 0`` puts a gated feed-forward block of that hidden width (``layers.FeedForwardBlock``) behind the LSTM stack; the
reference has no counterpart, and without it the model is the reference's."""
from __future__ import annotations

import torch
import torch.nn as nn

from . import layers as L


class RNNLM(nn.Module):
    def __init__(self, ntoken, ninp, nhid, nlayers, dropout=0.5, tie_weights=False, weight_norm=False,
                 nffn=0, ffn_act="silu"):
        super().__init__()
        self.ntoken, self.ninp, self.nhid, self.nlayers = ntoken, ninp, nhid, nlayers
        self.drop = L.Dropout(dropout)
        self.encoder = L.Embedding(ntoken, ninp)
        self.rnn = L.LSTM(ninp, nhid, nlayers, dropout=dropout, batch_first=False)
        self.ffn = L.FeedForwardBlock(nhid, nffn, ffn_act, dropout) if nffn > 0 else None
        self.decoder = L.Linear(nhid, ntoken)
        if tie_weights:
            if nhid != ninp:
                raise ValueError("When using the tied flag, nhid must be equal to emsize")
            self.decoder.weight = self.encoder.weight
            if hasattr(self.encoder, "tie_to_other_gradient"):
                self.encoder.tie_to_other_gradient()   # the decoder yields a dense gradient of the shared matrix
        self.init_weights()

    def init_weights(self):
        r = 0.1
        self.encoder.weight.data.uniform_(-r, r)
        self.decoder.bias.data.zero_()
        self.decoder.weight.data.uniform_(-r, r)

    def forward(self, input, hidden):
        emb = self.drop(self.encoder(input))
        output, hidden = self.rnn(emb, hidden)
        if self.ffn is not None:
            output = self.ffn(output)
        output = self.drop(output)
        decoded = self.decoder(output.reshape(output.size(0) * output.size(1), output.size(2)))
        return decoded.view(output.size(0), output.size(1), decoded.size(1)), hidden

    def init_hidden(self, bsz):
        w = next(self.parameters())
        return (w.new_zeros(self.nlayers, bsz, self.nhid), w.new_zeros(self.nlayers, bsz, self.nhid))

    def repackage_hidden(self, h):
        """Detach the hidden state from its history (truncated BPTT)."""
        if isinstance(h, torch.Tensor):
            return h.detach()
        return tuple(self.repackage_hidden(v) for v in h)
