"""A decoder from per-Gaussian features and an image's embedding to colours.

Large outdoor captures change their exposure, white balance and light from image to
image, which SH coefficients cannot follow.  ``AppearanceDecoder`` keeps a small
feature row with every Gaussian and one embedding per training image, and turns
them into an RGB offset of the SH colour: a residual block (layer norm, gated
feed-forward block, dropout) and a gated feed-forward block to the output, all in
``decoder_ops``'s kernels.  The embedding enters through the blocks' biases, where
it costs one small product an image instead of columns of every Gaussian's row.
TideGS has no counterpart.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor, nn

from .decoder_ops import dropout, gated_ffn, layer_norm


class _GatedBlock(nn.Module):
    """Layer norm and a gated feed-forward block whose hidden biases an embedding shifts."""

    def __init__(self, width: int, hidden: int, out: int, embedding: int):
        super().__init__()
        self.norm_weight = nn.Parameter(torch.ones(width))
        self.norm_bias = nn.Parameter(torch.zeros(width))
        self.w_gate = nn.Parameter(torch.randn(hidden, width) * width ** -0.5)
        self.w_up = nn.Parameter(torch.randn(hidden, width) * width ** -0.5)
        self.w_down = nn.Parameter(torch.randn(out, hidden) * hidden ** -0.5)
        self.b_down = nn.Parameter(torch.zeros(out))
        # rows 0 .. hidden - 1 shift the gate, the others the other factor
        self.shift = nn.Linear(embedding, 2 * hidden)

    def forward(self, x: Tensor, embedding: Tensor) -> Tensor:
        b_gate, b_up = self.shift(embedding).to(x.dtype).chunk(2)
        h = layer_norm(x, self.norm_weight.to(x.dtype), self.norm_bias.to(x.dtype))
        return gated_ffn(h, *(w.to(x.dtype) for w in (self.w_gate, self.w_up, self.w_down)),
                         b_gate, b_up, self.b_down.to(x.dtype))


class AppearanceDecoder(nn.Module):
    """RGB offsets [n, 3] (float32) of the Gaussians whose features [n, width] are given.

    ``dtype`` is the element type of the decoder's products; its parameters stay
    float32.  In training the residual branch drops a share ``p`` of its values: the
    mask follows from ``seed`` and the ``step`` of the call alone, so calls that are to
    differ (two images of one optimizer step) have steps of their own.
    """

    def __init__(self, images: int, width: int = 64, hidden: int = 256, embedding: int = 32,
                 p: float = 0.1, seed: int = 0, dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.embeddings = nn.Embedding(images, embedding)
        self.block = _GatedBlock(width, hidden, width, embedding)
        self.head = _GatedBlock(width, hidden, 3, embedding)
        nn.init.zeros_(self.head.w_down)  # starts at the SH colour
        self.p, self.seed, self.dtype = p, seed, dtype

    def forward(self, features: Tensor, image: int, step: Optional[int] = None) -> Tensor:
        x = features.to(self.dtype)
        embedding = self.embeddings.weight[image]
        h = self.block(x, embedding)
        if self.training and self.p > 0:
            if step is None:
                raise ValueError("training draws its dropout mask from the step: pass step=")
            x = dropout(h, self.p, self.seed, offset=step, residual=x)
        else:
            x = x + h
        return self.head(x, embedding).float()
