"""Linears with 4-bit weights and group scales, activations as they come, on the HIP kernels (ops.linear_i4).

`apply_int4_weights(model)` swaps every nn.Linear under `model` (optionally filtered) in place, as quant.apply_dynamic_quant does for int8:
a quarter of the half types' weight bytes, which is what a step over few rows reads.  Where int8 quantises the activations and rounds
nothing else, here the weights alone lose bits; the products run in the activations' own type.
"""

import warnings
from typing import Callable, Optional, Tuple

import torch
import torch.nn as nn

from . import ops
from .tools import replace_with_custom_fn_if_matches_filter


def quantize_weight_int4(weight: torch.Tensor, group_size: int = 128, zero_points: bool = False,
                         dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(N, K) float -> (codes uint8 (N, K/2), scales (groups, N) of `dtype`, zeros uint8 (groups, N) or None), as ops.linear_i4 takes them.

    Over each group of `group_size` inputs of an output, in fp32: without zero points scale = absmax / 7 and code = round(w / scale) + 8, 1 to
    15; with them scale = (max(w, 0) - min(w, 0)) / 15, zero = round(-min(w, 0) / scale) and code = round(w / scale) + zero, 0 to 15.  The scale is rounded to
    `dtype` (the weight's own by default, bfloat16 for a float32 weight) before the codes are made, so that these are the nearest to the weights
    that the product sees.  A group of zeros has scale 1.  K must be a multiple of 8; the last group may be shorter."""
    if weight.dim() != 2 or not weight.is_floating_point() or weight.shape[1] % 8 != 0 or weight.numel() == 0:
        raise ValueError("the weight must be a floating-point (N, K) tensor with K a multiple of 8")
    if group_size <= 0 or group_size % 32 != 0:
        raise ValueError(f"groups must be a multiple of 32 inputs, got {group_size}")
    if dtype is None:
        dtype = weight.dtype if weight.dtype in (torch.bfloat16, torch.float16) else torch.bfloat16
    N, K = weight.shape
    groups = -(-K // group_size)
    w = nn.functional.pad(weight.detach().to(torch.float32), (0, groups * group_size - K)).view(N, groups, group_size)
    low, high = w.amin(-1).clamp_max(0.0), w.amax(-1).clamp_min(0.0)
    scale = (high - low) / 15.0 if zero_points else torch.maximum(high, -low) / 7.0
    tiny = torch.finfo(dtype).smallest_normal
    scale = torch.where(scale > 0, scale.clamp_min(tiny), torch.ones_like(scale)).to(dtype)
    step = scale.to(torch.float32)
    zero = torch.round(-low / step).clamp_(0, 15) if zero_points else torch.full_like(step, 8.0)
    codes = (torch.round(w / step.unsqueeze(-1)) + zero.unsqueeze(-1)).clamp_(0, 15).to(torch.uint8).view(N, -1)[:, :K]
    return ((codes[:, 0::2] | codes[:, 1::2] << 4).contiguous(), scale.t().contiguous(),
            zero.to(torch.uint8).t().contiguous() if zero_points else None)


def dequantize_weight_int4(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor], group_size: int) -> torch.Tensor:
    """The fp32 (N, K) weight that quantize_weight_int4's tensors stand for."""
    N, K = codes.shape[0], 2 * codes.shape[1]
    c = torch.stack((codes & 15, codes >> 4), -1).view(N, K).to(torch.float32)
    of = torch.arange(K, device=codes.device) // group_size
    zero = 8.0 if zeros is None else zeros.to(torch.float32).t()[:, of]
    return (c - zero) * scales.to(torch.float32).t()[:, of]


class Int4Linear(nn.Module):
    """A Linear whose weight is held as `codes`, `scales` and, with zero points, `zeros` (see ops.linear_i4).

    The scales follow the module's dtype between the half types, and the kernels compute in it: inputs of another floating type are cast on the way in and
    the result back.  A module cast to a wider type keeps them as they are; a cast that takes scales out of the new type's range warns.
    The fp32 bias is kept as int32 bit patterns (`bias_bits`), which no cast of the module rounds; a state dict that carries an nn.Linear's float
    `bias` is folded into it on load.  `weight` is the dequantised weight.  There is no backward pass and no CPU route."""

    def __init__(self, in_features: int, out_features: int, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor],
                 bias: Optional[torch.Tensor], group_size: int) -> None:
        super().__init__()
        self.in_features, self.out_features, self.group_size = in_features, out_features, group_size
        self.register_buffer("codes", codes)
        self.register_buffer("scales", scales)
        self.register_buffer("zeros", zeros)
        self.register_buffer("bias_bits", None if bias is None else bias.detach().to(torch.float32, copy=True).contiguous().view(torch.int32))

    @classmethod
    def from_float(cls, linear: nn.Linear, group_size: int = 128, zero_points: bool = False) -> "Int4Linear":
        codes, scales, zeros = quantize_weight_int4(linear.weight, group_size, zero_points)
        return cls(linear.in_features, linear.out_features, codes, scales, zeros, linear.bias, group_size)

    def _apply(self, fn, *args, **kwargs):
        scales = self.scales
        super()._apply(fn, *args, **kwargs)
        if self.scales.dtype not in (torch.bfloat16, torch.float16):
            self.scales = self.scales.to(scales.dtype)  # (there and back is exact)
        elif self.scales.dtype != scales.dtype and not self.scales.is_meta:
            scales = scales.to(self.scales.device)
            lost = (self.scales.isinf() & scales.isfinite()) | ((self.scales == 0) & (scales != 0))
            if lost.any():
                warnings.warn(f"{int(lost.sum())} scales of a 4-bit Linear are outside {self.scales.dtype}: their weights are now 0 or not finite", stacklevel=2)
        return self

    @property
    def bias(self) -> Optional[torch.Tensor]:
        return None if self.bias_bits is None else self.bias_bits.view(torch.float32)

    @property
    def weight(self) -> torch.Tensor:
        return dequantize_weight_int4(self.codes, self.scales, self.zeros, self.group_size)

    def _load_from_state_dict(self, state_dict, prefix, *args, **kwargs):
        if prefix + "bias" in state_dict and self.bias_bits is not None:  # (without a bias here it is an entry too many)
            value = state_dict.pop(prefix + "bias")
            if prefix + "bias_bits" not in state_dict:
                state_dict[prefix + "bias_bits"] = value.detach().to(torch.float32).contiguous().view(torch.int32)
        super()._load_from_state_dict(state_dict, prefix, *args, **kwargs)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = ops.linear_i4(x if x.dtype == self.scales.dtype else x.to(self.scales.dtype), self.codes, self.scales, self.zeros, self.bias,
                          group_size=self.group_size)
        return y if y.dtype == x.dtype else y.to(x.dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, int4 weights in groups of {self.group_size}"


def apply_int4_weights(model: nn.Module, filter_fn: Optional[Callable[[nn.Module, str], bool]] = None, group_size: int = 128,
                       zero_points: bool = False) -> None:
    """Swap every nn.Linear under `model` (for which filter_fn(module, fqn) holds, if given) for Int4Linear, in place.  Nothing is swapped where one of them
    cannot be: inputs that are no multiple of 8, weights that are not floating-point."""
    chosen = lambda mod, fqn: isinstance(mod, nn.Linear) and (filter_fn is None or filter_fn(mod, fqn))
    for fqn, mod in model.named_modules(remove_duplicate=False):  # (under each of its names, as the swap goes by them)
        if fqn and chosen(mod, fqn) and (mod.in_features % 8 != 0 or mod.weight.numel() == 0 or not mod.weight.is_floating_point()):
            raise ValueError(f"{fqn}: a 4-bit Linear needs a multiple of 8 inputs and a floating-point weight, got {mod.in_features} and {mod.weight.dtype}")
    replace_with_custom_fn_if_matches_filter(model, lambda linear: Int4Linear.from_float(linear, group_size, zero_points), chosen)
