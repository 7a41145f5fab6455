"""Projections with 4-bit weights and group scales on fp16 or bf16 activations.

No counterpart in the reference, whose projections are INT8
(patches/tp_qwen3vl.py:25-134): the text encoder's projections of a few rows
take the time of their weights' bytes, which 4 bits halve. A weight is
scale * (code - zero) with one scale (and zero, 8 by default) per group of
inputs of each row.

Codes are packed eight to a 32-bit word: the word's nibbles 0-3, from the low
end, hold inputs 0, 2, 4, 6 of its eight, nibbles 4-7 inputs 1, 3, 5, 7 (so
that a shift and a mask leave two neighbouring inputs in a word's halves).
"""
import torch
from torch import nn

from . import _abi, kernels

_NIBBLE_OF_INPUT = (0, 4, 1, 5, 2, 6, 3, 7)


def _check_groups(features, group_size):
    if group_size not in (32, 64) and (group_size <= 0 or group_size % 128):
        raise ValueError('group sizes are 32, 64 and multiples of 128')
    if features <= 0 or features % group_size:
        raise ValueError('the input features must be a positive multiple of the group size')


def pack(codes):
    """int32 [N, K / 8] words of codes [N, K] (integers 0 to 15)."""
    if codes.ndim != 2 or codes.shape[1] % 8 or codes.is_floating_point():
        raise ValueError('codes must be integers [N, K] with K a multiple of 8')
    c = codes.to(torch.int64).reshape(codes.shape[0], -1, 8)
    if c.numel() and (int(c.min()) < 0 or int(c.max()) > 15):
        raise ValueError('codes are 0 to 15')
    shifts = torch.tensor([4 * i for i in _NIBBLE_OF_INPUT], dtype=torch.int64, device=c.device)
    word = (c << shifts).sum(-1)
    return torch.where(word >= 2 ** 31, word - 2 ** 32, word).to(torch.int32)


def unpack(words):
    """uint8 [N, K] codes of pack()'s words."""
    if words.ndim != 2 or words.dtype != torch.int32:
        raise ValueError('words must be int32 [N, K / 8]')
    shifts = torch.tensor([4 * i for i in _NIBBLE_OF_INPUT], dtype=torch.int32, device=words.device)
    return ((words[:, :, None] >> shifts) & 15).to(torch.uint8).reshape(words.shape[0], -1)


def _scales(step, dtype):
    """Steps (fp32) as values of dtype, never 0: to the nearest, but in the subnormal
    range (where that may be a good part of a step) never below."""
    info = torch.finfo(dtype)
    spacing = info.smallest_normal * info.eps
    scale = step.to(dtype).float()
    short = (scale < step) & (scale < info.smallest_normal)
    return torch.where(short, scale + spacing, scale).clamp_min(spacing)


def quantize_weight(weight, group_size=128, *, symmetric=True, dtype=torch.float16):
    """(codes, scales, zeros) of a weight [N, K]: round to nearest within each
    group of group_size inputs, with the scale already rounded to dtype.
    symmetric: scale = absmax / 7, zeros None (8); else the group's range,
    widened to hold 0, over 15 steps with a zero of its own. Scales may be
    subnormal, so that small weights (those that carry a residual divisor, say)
    keep their steps: below the smallest normal a scale that would fall short is
    the next one up, at most one spacing (2^-24 in fp16) more."""
    if weight.ndim != 2:
        raise ValueError('weight must be [N, K]')
    _check_groups(weight.shape[1], group_size)
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError('scales must be float16 or bfloat16')
    n, k = weight.shape
    w = weight.detach().float().reshape(n, k // group_size, group_size)
    if symmetric:
        scale = _scales(w.abs().amax(-1) / 7, dtype)
        zero = torch.full_like(scale, 8)
    else:
        low, high = w.amin(-1).clamp_max(0), w.amax(-1).clamp_min(0)
        scale = _scales((high - low) / 15, dtype)
        zero = (-low / scale).round().clamp(0, 15)
    if not bool(torch.isfinite(scale).all()):
        raise ValueError(f'weights that are not finite, or whose scale {dtype} does not hold')
    codes = ((w / scale[:, :, None]).round() + zero[:, :, None]).clamp(0, 15).to(torch.uint8)
    return (pack(codes.reshape(n, k)), scale.t().contiguous().to(dtype),
            None if symmetric else zero.t().contiguous().to(torch.uint8))


def dequantize_weight(codes, scales, zeros=None):
    """fp32 [N, K] weights."""
    c = unpack(codes).float().reshape(codes.shape[0], scales.shape[0], -1)
    z = 8.0 if zeros is None else zeros.float().t()[:, :, None]
    return ((c - z) * scales.float().t()[:, :, None]).reshape(codes.shape[0], -1)


def linear(x, codes, scales, zeros=None, *, bias=None, residual=None, gated=False, out=None):
    """x [.., K] times the 4-bit weight; see kernels.linear_w4. Inference only."""
    if out is None:
        y = _abi.native().linear_w4(x, codes, scales, zeros, bias, residual, gated)
        if y is not None:
            return y
    return kernels.linear_w4(x, codes, scales, zeros, bias=bias, residual=residual, gated=gated, out=out)


class LinearW4(nn.Module):
    """A projection with 4-bit weights, optionally gated (silu(gate) * up of a
    packed [2 F, K] weight). Buffers: codes, scales, zeros, bias."""

    def __init__(self, in_features, out_features, *, group_size=128, zeros=False, bias=False, gated=False,
                 dtype=torch.float16, device=None):
        super().__init__()
        _check_groups(in_features, group_size)
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError('scales must be float16 or bfloat16')
        if gated and out_features % 2:
            raise ValueError('a gated projection has gate and up halves')
        self.in_features, self.out_features, self.group_size, self.gated = in_features, out_features, group_size, gated
        dev = torch.device(device) if device is not None else torch.device('cuda', 0)
        groups = in_features // group_size
        self.register_buffer('codes', torch.zeros((out_features, in_features // 8), dtype=torch.int32, device=dev))
        self.register_buffer('scales', torch.zeros((groups, out_features), dtype=dtype, device=dev))
        self.register_buffer('zeros', torch.full((groups, out_features), 8, dtype=torch.uint8, device=dev)
                             if zeros else None)
        self.register_buffer('bias', torch.zeros(out_features, dtype=dtype, device=dev) if bias else None)

    @torch.no_grad()
    def load_weight(self, weight, bias=None):
        """Quantize a floating weight [N, K] (and bias [N]) into the buffers."""
        if tuple(weight.shape) != (self.out_features, self.in_features):
            raise ValueError('weight must be [out_features, in_features]')
        if (bias is None) != (self.bias is None):
            raise ValueError('a bias goes into a module that was made with one')
        codes, scales, zeros = quantize_weight(weight, self.group_size, symmetric=self.zeros is None,
                                               dtype=self.scales.dtype)
        self.codes.copy_(codes)
        self.scales.copy_(scales)
        if zeros is not None:
            self.zeros.copy_(zeros)
        if bias is not None:
            self.bias.copy_(bias)
        return self

    def forward(self, x, *, residual=None):
        return linear(x, self.codes, self.scales, self.zeros, bias=self.bias, residual=residual, gated=self.gated)
