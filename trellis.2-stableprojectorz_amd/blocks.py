"""Sparse blocks around the conv: SparseLinear, the ConvNeXt block, group norm and the block of
differential attention.

  SparseLinear            src/sparse/ops/linear.ts:9-29 (nn.Linear per voxel; the TS port
                          multiplies by the (out,in) weight untransposed)
  SparseConvNeXtBlock3d   src/models/sparse_unet_vae_decoder.ts:48-78 and its use at :119-134:
                          h = conv(x); h = LN(h); h = h W0^T + b0; h = silu(LN(h)); out = x + h W2^T + b2
                          (LayerNorm without affine, eps 1e-6, as the TS block calls it)
  SparseGroupNorm, SparseDiffAttentionBlock3d
                          over each sample's voxels; no counterpart in the reference, whose blocks
                          normalize rows (src/sparse/ops/norm.ts:10-140) and attend with one map
                          (src/sparse/ops/attention.ts:24-79)

Each step is one C-ABI call: the conv (tsc_conv, map cached on x), tsc_layernorm (SiLU fused into
the second one), and tsc_linear (hipBLASLt GEMM with the bias epilogue; the second linear takes
the block input as its residual operand, so the skip add costs no extra pass).
"""
from __future__ import annotations

import torch

from . import ops
from .conv3d import SparseConv3d
from .sparse_tensor import SparseTensor


class SparseLinear:
    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None):
        if weight.dim() != 2:
            raise ValueError("weight must be (out_channels, in_channels)")
        self.weight = weight.contiguous()
        self.bias = None if bias is None else bias.contiguous()

    def forward(self, x: SparseTensor) -> SparseTensor:
        return x.replace(ops.sparse_linear(x.feats, self.weight, self.bias))

    __call__ = forward


class SparseGroupNorm:
    """Group norm of each sample's voxels, optionally with SiLU (ops.group_norm over x.cu_rows, so
    x's rows have to be grouped by sample)."""

    def __init__(self, num_groups: int, weight: torch.Tensor | None = None,
                 bias: torch.Tensor | None = None, eps: float = 1e-5, silu: bool = False):
        self.num_groups, self.eps, self.silu = num_groups, eps, silu
        self.weight = None if weight is None else weight.contiguous()
        self.bias = None if bias is None else bias.contiguous()

    def forward(self, x: SparseTensor) -> SparseTensor:
        cu = x.cu_rows
        return x.replace(ops.group_norm(x.feats, self.num_groups, self.weight, self.bias, cu,
                                        self.eps, self.silu))

    __call__ = forward


class SparseDiffAttentionBlock3d:
    """x + out(diff_attention(qkv(group_norm(x)))) over each sample's voxels, x's rows grouped by
    sample: group norm, one linear layer for q, k and v (read in place as row slices), differential
    attention, and the output layer with the skip as its residual.  qkv weight (3 C, C), out weight
    (C, C), lam float32 (num_heads), C = num_heads * 64 or 128.  Attention's result goes to the
    output layer as it is: no norm per head after the difference, no factor of 1 - lambda's start.
    Without gradients: its linear layers have none (group_norm and sparse_diff_attention do, around
    another library's linear layers)."""

    def __init__(self, num_heads: int, num_groups: int, norm_weight: torch.Tensor | None,
                 norm_bias: torch.Tensor | None, qkv_weight: torch.Tensor,
                 qkv_bias: torch.Tensor | None, lam: torch.Tensor, out_weight: torch.Tensor,
                 out_bias: torch.Tensor | None, eps: float = 1e-5):
        self.num_heads, self.lam = num_heads, lam
        self.norm = SparseGroupNorm(num_groups, norm_weight, norm_bias, eps)
        self.qkv = SparseLinear(qkv_weight, qkv_bias)
        self.out = SparseLinear(out_weight, out_bias)

    @torch.no_grad()
    def forward(self, x: SparseTensor) -> SparseTensor:
        n, c = x.feats.shape
        cu = x.cu_rows
        longest = max(stop - start for start, stop in x.layout)
        qkv = self.qkv(self.norm(x)).feats.view(n, 3, self.num_heads, c // self.num_heads)
        h = ops.sparse_diff_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], self.lam, cu,
                                      max_seqlen_q=longest, max_seqlen_kv=longest)
        return x.replace(ops.sparse_linear(h.view(n, c), self.out.weight, self.out.bias,
                                           residual=x.feats))

    __call__ = forward


class SparseConvNeXtBlock3d:
    def __init__(self, conv_weight: torch.Tensor, conv_bias: torch.Tensor | None,
                 linear0_weight: torch.Tensor, linear0_bias: torch.Tensor | None,
                 linear2_weight: torch.Tensor, linear2_bias: torch.Tensor | None,
                 eps: float = 1e-6):
        self.conv = SparseConv3d(conv_weight, conv_bias)
        self.linear0 = SparseLinear(linear0_weight, linear0_bias)
        self.linear2 = SparseLinear(linear2_weight, linear2_bias)
        self.eps = eps

    def forward(self, x: SparseTensor) -> SparseTensor:
        h = self.conv.forward(x).feats
        ops.layer_norm(h, eps=self.eps, out=h)
        h = ops.sparse_linear(h, self.linear0.weight, self.linear0.bias)
        ops.layer_norm(h, eps=self.eps, silu=True, out=h)
        out = ops.sparse_linear(h, self.linear2.weight, self.linear2.bias, residual=x.feats)
        return x.replace(out)

    __call__ = forward
