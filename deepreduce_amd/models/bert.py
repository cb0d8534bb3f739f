"""BERT-base encoder (masked-LM head) — for BASELINE.json config 5
(top-k 0.1%, deepreduce='both').  Written directly: 12 layers, hidden 768,
12 heads, ~110M params at vocab 30522.  Uses torch SDPA (Flash-attention
path on ROCm) on whole rows with learned positions, and ops.attention where
rows pack several documents or positions are rotary or distances.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops


class EncoderLayer(nn.Module):
    def __init__(self, hidden: int, heads: int, ffn: int, dropout: float = 0.0):
        super().__init__()
        self.heads = heads
        self.qkv = nn.Linear(hidden, hidden * 3)
        self.proj = nn.Linear(hidden, hidden)
        self.ln1 = nn.LayerNorm(hidden)
        self.fc1 = nn.Linear(hidden, ffn)
        self.fc2 = nn.Linear(ffn, hidden)
        self.ln2 = nn.LayerNorm(hidden)

    def forward(self, x, documents=None, rotary=None, slopes=None):
        b, s, h = x.shape
        qkv = self.qkv(x).view(b, s, 3, self.heads, h // self.heads)
        if documents is None and rotary is None and slopes is None:
            q, k, v = (qkv[:, :, i].transpose(1, 2) for i in range(3))
            attn = F.scaled_dot_product_attention(q, k, v)
            attn = attn.transpose(1, 2).reshape(b, s, h)
        else:
            q, k, v = qkv.unbind(2)
            if rotary is not None:
                q, k = ops.rotary(q, k, *rotary)
            attn = ops.attention(q, k, v, documents=documents, slopes=slopes).reshape(b, s, h)
        x = self.ln1(x + self.proj(attn))
        x = self.ln2(x + self.fc2(F.gelu(self.fc1(x))))
        return x


def document_positions(documents: torch.Tensor) -> torch.Tensor:
    """int64 [B, S]: each token's place in its run of equal document numbers."""
    at = torch.arange(documents.shape[1], device=documents.device).expand(documents.shape)
    starts = torch.ones_like(documents, dtype=torch.bool)
    starts[:, 1:] = documents[:, 1:] != documents[:, :-1]
    return at - torch.where(starts, at, torch.zeros_like(at)).cummax(1).values


class BertBase(nn.Module):
    """positions: 'learned' (an embedding of max_len positions), 'rotary' or
    'distance' (a bias of the attention scores, a slope for each head); the
    last two have no parameters and no longest row."""

    def __init__(self, vocab: int = 30522, hidden: int = 768, layers: int = 12,
                 heads: int = 12, ffn: int = 3072, max_len: int = 512,
                 positions: str = "learned"):
        super().__init__()
        if positions not in ("learned", "rotary", "distance"):
            raise ValueError(f"positions must be 'learned', 'rotary' or 'distance', "
                             f"got {positions!r}")
        self.positions, self.heads, self.max_len = positions, heads, max_len
        self.tok = nn.Embedding(vocab, hidden)
        if positions == "learned":
            self.pos = nn.Embedding(max_len, hidden)
        self.ln = nn.LayerNorm(hidden)
        self.layers = nn.ModuleList(EncoderLayer(hidden, heads, ffn) for _ in range(layers))
        self.head = nn.Linear(hidden, vocab, bias=False)
        self.head.weight = self.tok.weight  # tied
        # rotary frequencies or slopes by device, not part of the state: they
        # keep their type whatever the parameters are cast to
        self._constants = {}
        self._constant(self.tok.weight.device)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        # made where the model moves to, so that no captured call has to
        self._constant(self.tok.weight.device)
        return self

    def forward(self, ids: torch.Tensor, documents: torch.Tensor | None = None) -> torch.Tensor:
        """documents: int32 [B, S] for packed rows, the document of each token
        (a run of equal numbers) and a negative number for padding.  Documents
        do not see each other, and positions restart with each."""
        b, s = ids.shape
        pos = (torch.arange(s, device=ids.device).unsqueeze(0) if documents is None
               else document_positions(documents))
        x, rotary, slopes = self.tok(ids), None, None
        if self.positions == "learned":
            if s > self.max_len:
                raise ValueError(f"rows of {s} tokens, learned positions for {self.max_len}")
            x = x + self.pos(pos)
        elif self.positions == "rotary":
            rotary = (pos.expand(b, s), self._constant(ids.device))
        else:
            slopes = self._constant(ids.device)
        x = self.ln(x)
        for layer in self.layers:
            x = layer(x, documents, rotary, slopes)
        return self.head(x)

    @torch.inference_mode(False)  # constants made in an evaluation serve training too
    def _constant(self, device):
        if self.positions == "learned" or device.type == "meta":
            return None
        if device not in self._constants:
            if self.positions == "rotary":
                value = ops.rotary_frequencies(self.tok.embedding_dim // self.heads)
            else:  # slopes from 1/2 to 2^-8 or so, each head's a fixed part of the last
                value = torch.tensor([2.0 ** (-8.0 * (h + 1) / self.heads)
                                      for h in range(self.heads)], dtype=torch.float32)
            self._constants[device] = value.to(device)
        return self._constants[device]
