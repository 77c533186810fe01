"""A table of label vectors, looked up and scaled (label queries, label-by-label detectors; the reference has
none).  ROCm tensors run the HIP kernels, forward and backward; CPU tensors the host path.
"""
import torch
from torch import nn

from .. import core
from .. import hostpath
from ..metrics import on_host


def scaled_embedding(ids, weight, scale=1.0, padding_idx=None):
    """``scale * weight[ids]``: ids (int32 / int64, any shape) -> ids.shape + (D,), weight [V, D] in float32,
    bfloat16 or float16.

    The product is taken in 32 bits and rounded once.  An id outside [0, V) reads zeros.  The table's gradient is
    dense, each label's rows added in 32 bits in an order that the call's ids and sizes fix (the same bits every time for
    the same ids; other ids beside a label's may change its last bits), zeros where a label did not occur and for
    ``padding_idx``, whose row is looked up like any other."""
    r = core.label_call('label_embed', weight, ids, weight, float(scale), padding_idx)
    if r is not None:
        return r
    pad = core.embedding_arguments(ids, weight, scale, padding_idx)
    if on_host(ids, weight):
        return hostpath.scaled_embedding(ids, weight, scale, pad)
    return core.scaled_embedding(ids, weight, scale, pad)


class ScaledEmbedding(nn.Module):
    """``scaled_embedding`` with its table as ``weight``, normally distributed with deviation 1 / sqrt(D) and zeros
    for ``padding_idx``; ``scale`` defaults to sqrt(D)."""

    def __init__(self, num_embeddings, embedding_dim, scale=None, padding_idx=None, device=None, dtype=None):
        super().__init__()
        self.num_embeddings, self.embedding_dim = num_embeddings, embedding_dim
        self.scale = float(embedding_dim) ** 0.5 if scale is None else float(scale)
        self.padding_idx = padding_idx
        self.weight = nn.Parameter(torch.empty(num_embeddings, embedding_dim, device=device, dtype=dtype))
        nn.init.normal_(self.weight, std=float(max(embedding_dim, 1)) ** -0.5)
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx] = 0

    def forward(self, ids):
        return scaled_embedding(ids, self.weight, self.scale, self.padding_idx)

    def extra_repr(self):
        return '%d, %d, scale=%g, padding_idx=%s' % (self.num_embeddings, self.embedding_dim, self.scale,
                                                     self.padding_idx)
