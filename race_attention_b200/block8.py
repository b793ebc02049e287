"""A causal RACE decoder whose linear layers run in 8 bits: the 8-bit operators,
the norm with the residual's addition and RACE attention as they are used
together.

The block is the pre-norm block of the reference (RACEBlock, misc/race.py:176-206)
with root-mean-square norms, one projection for q, k and v, and no biases.  It
passes (branch, residual) from one block to the next, so that each norm adds
the branch before it; nothing else reads or writes the residual.

Training: activations and the residual in bfloat16, weights in float32, both
quantised inside each product.  Serving (``hold()``, eval mode, no_grad): weights
are held in 8 bits and a norm hands its rows to the next product in 8 bits, so
no higher-precision copy of them is written.

``python -m race_attention_b200.block8`` trains a small decoder on a synthetic
task and then serves it.
"""
from __future__ import annotations

import torch
from torch import nn

from .fp8 import Fp8Linear, RMSNorm
from .race import BatchedACE


class RACEBlock8(nn.Module):
    """forward(x, residual) -> (x, residual): the branch that the next norm adds
    and the residual so far.  x, residual: [B, T, width] bfloat16 or float32."""

    def __init__(self, width: int, heads: int, K: int = 2, L: int = 5, hidden: int = 0, device=None):
        super().__init__()
        if width % heads:
            raise ValueError("width must be a multiple of heads")
        self.heads, self.d_k = heads, width // heads
        hidden = hidden or 4 * width
        self.norm1 = RMSNorm(width, device=device)
        self.qkv = Fp8Linear(width, 3 * width, device=device)
        self.ace = BatchedACE(self.d_k, K, L, 1, device=device or "cpu").to(device)
        self.out = Fp8Linear(width, width, device=device)
        self.norm2 = RMSNorm(width, device=device)
        self.up = Fp8Linear(width, hidden, device=device)
        self.down = Fp8Linear(hidden, width, device=device)

    def _serving(self) -> bool:
        return not self.training and self.qkv.held is not None and not torch.is_grad_enabled()

    def forward(self, x, residual=None):
        B, T, W = x.shape
        dtype, served = x.dtype, self._serving()
        y = self.norm1(x, residual, quantize=served)
        y, h = (y, x) if residual is None else y
        q, k, v = self.qkv(y, out_dtype=dtype).view(B, T, 3, self.heads, self.d_k).unbind(2)
        a = self.ace(*(z.unsqueeze(0) for z in (k, v, q)))[0]
        a = self.out(a.reshape(B, T, W), out_dtype=dtype)
        y, h = self.norm2(a, h, quantize=served)
        z = nn.functional.gelu(self.up(y, out_dtype=dtype))
        return self.down(z, out_dtype=dtype).view(B, T, W), h


class RACEDecoder8(nn.Module):
    """Token embedding, blocks and a tied output layer: [B, T] tokens to logits
    [B, T, vocab] in bfloat16."""

    def __init__(self, vocab: int, width: int, heads: int, layers: int, K: int = 2, L: int = 5, device=None):
        super().__init__()
        self.embed = nn.Embedding(vocab, width, device=device)
        nn.init.normal_(self.embed.weight, std=0.02)
        self.blocks = nn.ModuleList(RACEBlock8(width, heads, K, L, device=device) for _ in range(layers))
        self.norm = RMSNorm(width, device=device)
        self.head = Fp8Linear(width, vocab, device=device)
        self.head.weight = self.embed.weight

    def _layers(self):
        return [m for m in self.modules() if isinstance(m, Fp8Linear)]

    def hold(self) -> "RACEDecoder8":
        """Holds every weight in 8 bits for serving."""
        for m in self._layers():
            m.hold()
        return self

    def release(self) -> "RACEDecoder8":
        for m in self._layers():
            m.release()
        return self

    def forward(self, tokens):
        x, h = self.embed(tokens).to(torch.bfloat16), None
        for block in self.blocks:
            x, h = block(x, h)
        served = self.blocks[0]._serving()
        y, _ = self.norm(x, h, quantize=served)
        return self.head(y, out_dtype=torch.bfloat16).view(*tokens.shape, -1)


def train(model: RACEDecoder8, steps: int, batch: int = 8, tokens: int = 128, lr: float = 1e-3,
          state_bits: int = 8, seed: int = 0):
    """Trains on counting modulo the vocabulary (the next token is the last one
    plus a step that a sequence keeps) and returns the losses."""
    from .optim import AdamW
    dev = model.embed.weight.device
    vocab = model.embed.num_embeddings
    g = torch.Generator(device=dev).manual_seed(seed)
    opt = AdamW(model.parameters(), lr=lr, betas=(0.9, 0.95), weight_decay=0.0, state_bits=state_bits, seed=seed)
    losses = []
    for _ in range(steps):
        start = torch.randint(0, vocab, (batch, 1), generator=g, device=dev)
        by = torch.randint(1, 4, (batch, 1), generator=g, device=dev)
        seq = (start + by * torch.arange(tokens + 1, device=dev)) % vocab
        logits = model(seq[:, :-1])
        loss = nn.functional.cross_entropy(logits.float().flatten(0, 1), seq[:, 1:].flatten())
        loss.backward()
        opt.step()
        opt.zero_grad()
        losses.append(loss.detach())
    return [float(x) for x in losses]


def main() -> None:
    torch.manual_seed(0)
    model = RACEDecoder8(vocab=256, width=384, heads=6, layers=2, device="cuda")
    losses = train(model, steps=100)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} in {len(losses)} steps, states in 8 bits")
    model.eval().hold()
    seq = torch.arange(129, device="cuda")[None] * 2 % 256
    with torch.no_grad():
        logits = model(seq[:, :-1])
    loss = nn.functional.cross_entropy(logits.float().flatten(0, 1), seq[:, 1:].flatten())
    print(f"served with weights held in 8 bits: loss {float(loss):.3f} on a new sequence")


if __name__ == "__main__":
    main()
