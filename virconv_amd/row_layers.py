"""Row-wise layers on the HIP operators: layer norm, and a linear layer with one weight matrix per row group.

They take (N, C) feature rows and so run inside ``spconv.SparseSequential`` (``LayerNorm``) or on what the RoI stage pools (both)."""
from __future__ import annotations

import math

import torch
from torch import nn

from . import ops


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last axis (one number as ``normalized_shape``), same parameters and state_dict, as ops.layer_norm."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(normalized_shape, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm: normalises the last axis only, got normalized_shape {self.normalized_shape}")

    def forward(self, x):
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"LayerNorm: rows of {x.shape[-1]} channels, expected {self.normalized_shape[0]}")
        return ops.layer_norm(x, self.weight, self.bias, self.eps)


class GroupedLinear(nn.Module):
    """``groups`` linear layers, one per row group: rows sorted by group, ``offsets`` (groups + 1) their bounds on the GPU."""

    def __init__(self, groups, in_features, out_features, bias=True, device=None, dtype=None):
        super().__init__()
        if groups < 1 or in_features < 1 or out_features < 1:
            raise ValueError(f"GroupedLinear: {groups} groups of {in_features} -> {out_features}")
        self.groups, self.in_features, self.out_features = int(groups), int(in_features), int(out_features)
        self.weight = nn.Parameter(torch.empty(groups, out_features, in_features, device=device, dtype=dtype))
        if bias:
            self.bias = nn.Parameter(torch.empty(groups, out_features, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self):
        bound = 1.0 / math.sqrt(self.in_features)   # nn.Linear's
        nn.init.uniform_(self.weight, -bound, bound)
        if self.bias is not None:
            nn.init.uniform_(self.bias, -bound, bound)

    def forward(self, x, offsets):
        return ops.grouped_linear(x, self.weight, offsets, self.bias)

    def extra_repr(self):
        return f"groups={self.groups}, in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
