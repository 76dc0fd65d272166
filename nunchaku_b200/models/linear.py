"""``SVDQW4A4Linear``: the module-level drop-in (mirror of ``nunchaku/models/linear.py:9-135``).

Same constructor, parameter names, shapes and dtypes as the reference, so a reference
``state_dict`` loads unchanged; the packed parameters keep the reference's memory order.

``W8A8Linear``: a linear layer with 8-bit weights (one scale per output channel) and 8-bit activations (one scale per token).
"""
from __future__ import annotations

import torch
from torch import nn

from ..ops.gemm import invalidate_prepared, svdq_gemm_w4a4_cuda
from ..ops.quantize import svdq_quantize_w4a4_act_fuse_lora_cuda
from ..ops.w8a8 import gemm_w8a8, quantize_w8a8


class SVDQW4A4Linear(nn.Module):
    def __init__(
        self,
        in_features: int,
        out_features: int,
        rank: int = 32,
        bias: bool = True,
        precision: str = "int4",
        act_unsigned: bool = False,
        torch_dtype: torch.dtype = torch.bfloat16,
        device: str | torch.device | None = None,
    ):
        super().__init__()
        if device is None:
            device = torch.device("cpu")
        self.in_features = in_features
        self.out_features = out_features
        self.rank = rank
        self.precision = precision
        self.torch_dtype = torch_dtype
        if precision == "nvfp4":
            self.group_size = 16
        elif precision == "int4":
            self.group_size = 64
        else:
            raise ValueError(f"Invalid precision: {precision}")

        def p(*shape, dtype=torch_dtype, grad=False):
            return nn.Parameter(torch.empty(*shape, dtype=dtype, device=device), requires_grad=grad)

        self.qweight = p(out_features, in_features // 2, dtype=torch.int8)
        self.bias = p(out_features) if bias else None
        self.wscales = p(
            in_features // self.group_size, out_features,
            dtype=torch_dtype if precision == "int4" else torch.float8_e4m3fn,
        )
        self.smooth_factor = p(in_features)
        self.smooth_factor_orig = p(in_features)
        self.proj_down = p(in_features, rank)
        self.proj_up = p(out_features, rank)
        self.wtscale = None
        self.wcscales = None
        if precision == "nvfp4":
            self.wtscale = nn.Parameter(torch.ones(1, dtype=torch_dtype, device=device), requires_grad=False)
            self.wcscales = nn.Parameter(torch.ones(out_features, dtype=torch_dtype, device=device), requires_grad=False)
        self.act_unsigned = act_unsigned

    @classmethod
    def from_linear(cls, linear: nn.Linear, **kwargs):
        in_features = kwargs.pop("in_features", linear.in_features)
        return cls(
            in_features=in_features, out_features=linear.out_features, bias=linear.bias is not None,
            torch_dtype=linear.weight.dtype, device=linear.weight.device, **kwargs,
        )

    def _load_from_state_dict(self, *args, **kwargs):
        # the GEMM keeps a re-tiled copy of the packed weights next to `qweight`; new values make it stale
        super()._load_from_state_dict(*args, **kwargs)
        self.invalidate_prepared_weights()

    def invalidate_prepared_weights(self) -> None:
        """Call after changing any packed parameter by a route that bypasses torch's version counter
        (``param.data.copy_()``, ``param.data = ...``): the next forward re-tiles the weights."""
        invalidate_prepared(self.qweight)

    def forward(self, x: torch.Tensor, output: torch.Tensor | None = None) -> torch.Tensor:
        batch_size, seq_len, channels = x.shape
        x = x.view(batch_size * seq_len, channels)
        if output is None:
            output = torch.empty(batch_size * seq_len, self.out_features, dtype=x.dtype, device=x.device)
        quantized_x, ascales, lora_act_out = self.quantize(x)
        output = self.forward_quant(quantized_x, ascales, lora_act_out, output)
        return output.view(batch_size, seq_len, -1)

    def quantize(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        return svdq_quantize_w4a4_act_fuse_lora_cuda(
            x, lora_down=self.proj_down, smooth=self.smooth_factor, fp4=self.precision == "nvfp4"
        )

    def forward_quant(
        self,
        quantized_x: torch.Tensor,
        ascales: torch.Tensor,
        lora_act: torch.Tensor,
        output: torch.Tensor | None = None,
    ) -> torch.Tensor:
        if output is None:
            output = torch.empty(
                quantized_x.shape[0], self.out_features, dtype=self.proj_up.dtype, device=quantized_x.device
            )
        svdq_gemm_w4a4_cuda(
            act=quantized_x, wgt=self.qweight, out=output, ascales=ascales, wscales=self.wscales,
            lora_act_in=lora_act, lora_up=self.proj_up, bias=self.bias, fp4=self.precision == "nvfp4",
            alpha=self.wtscale, wcscales=self.wcscales, act_unsigned=self.act_unsigned,
        )
        return output

    def __repr__(self):
        return (
            f"SVDQW4A4Linear(in_features={self.in_features}, out_features={self.out_features}, "
            f"rank={self.rank}, precision={self.precision}, act_unsigned={self.act_unsigned})"
        )


class W8A8Linear(nn.Module):
    """``y = x W^T + bias`` through :func:`nunchaku_b200.ops.gemm_w8a8`: ``qweight`` int8 [out, in] with ``wscales`` fp32 [out] (the plain
    row-major order, nothing packed), activations quantised per token.  ``in_features`` a multiple of 16 up to 16384, ``out_features`` of 8."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, torch_dtype: torch.dtype = torch.bfloat16,
                 device: str | torch.device | None = None):
        super().__init__()
        if in_features % 16 or in_features > 16384 or out_features % 8:
            raise ValueError("in_features must be a multiple of 16 up to 16384 and out_features of 8")
        device = torch.device("cpu") if device is None else device
        self.in_features, self.out_features, self.torch_dtype = in_features, out_features, torch_dtype
        self.qweight = nn.Parameter(torch.zeros(out_features, in_features, dtype=torch.int8, device=device), requires_grad=False)
        self.wscales = nn.Parameter(torch.zeros(out_features, dtype=torch.float32, device=device), requires_grad=False)
        self.bias = nn.Parameter(torch.zeros(out_features, dtype=torch_dtype, device=device), requires_grad=False) if bias else None

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: nn.Linear) -> "W8A8Linear":
        """Quantise a bf16 / fp16 ``nn.Linear`` that is on the GPU: one symmetric scale per output channel."""
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, linear.weight.dtype, linear.weight.device)
        codes, scales = quantize_w8a8(linear.weight.detach())
        m.qweight.copy_(codes)
        m.wscales.copy_(scales)
        if m.bias is not None:
            m.bias.copy_(linear.bias)
        return m

    def quantize(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        return quantize_w8a8(x)

    def forward_quant(self, codes: torch.Tensor, scales: torch.Tensor, output: torch.Tensor | None = None) -> torch.Tensor:
        return gemm_w8a8(codes, self.qweight, scales, self.wscales, bias=self.bias, out=output, out_dtype=self.torch_dtype)

    def forward(self, x: torch.Tensor, output: torch.Tensor | None = None) -> torch.Tensor:
        codes, scales = self.quantize(x)
        return self.forward_quant(codes, scales, output)

    def __repr__(self):
        return f"W8A8Linear(in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None})"
