"""A decode step with microscaled linear layers: weights in e2m1 blocks, a quarter of their bf16 bytes and
half of ``DecodeBlock``'s e4m3 ones, and the activations quantised to blocks in front of each product
(no counterpart in the reference, whose weights are bf16 or fp32: models/llama_block.py:82-105).

Five products of a step read their operands as blocks: the norms and the SwiGLU write theirs directly, the
attention's output is quantised by a launch of its own. The residual stream stays bf16.
"""
from __future__ import annotations

import torch

from . import abi, ops
from .paged import PagedDecodeBlock


class MxDecodeBlock(PagedDecodeBlock):
    """``PagedDecodeBlock`` with weights in e2m1 blocks of 32 along k; ``bits`` 8 (e4m3) or 4 (e2m1) are the
    activations' elements. intermediate is a multiple of 32, hidden at most 65536. ``effective_weights`` are the
    values that the codes stand for; there is no ``out32``, the sums are rounded to the bf16 stream once.
    ``fold_gain`` makes no difference: a norm always applies its gain as it quantises."""

    def __init__(self, state_dict: dict[str, torch.Tensor], *, bits: int = 8, **options) -> None:
        if bits not in (4, 8):
            raise abi.HipBackendError("MxDecodeBlock", abi.TH_ERR_INVALID, f"activations of {bits} bits; 4 or 8")
        if options.get("intermediate", 0) % 32 or options.get("hidden", 0) > 65536:
            raise abi.HipBackendError("MxDecodeBlock", abi.TH_ERR_INVALID, f"intermediate {options.get('intermediate')} must be whole "
                                      f"blocks of 32, hidden {options.get('hidden')} at most 65536")
        self.bits = bits
        super().__init__(state_dict, **options)

    def _load_projections(self, sd: dict[str, torch.Tensor], fold_gain: bool) -> None:
        dev, B = self.device, self.B

        def proj(names: list[str]) -> tuple[torch.Tensor, torch.Tensor]:
            w = torch.cat([sd[n] for n in names]).to(dev)   # nn.Linear [out, in]: one row an output column
            codes, scales = ops.mx_empty(*w.shape, bits=4, device=dev)
            ops.mx_quantize(w, codes, scales)
            values = ops.mx_dequantize(codes, scales, w).cpu()
            self._eff.update(zip(names, values.split([sd[n].shape[0] for n in names])))
            return codes, scales

        self.wqkv = proj(["attn.q_proj.weight", "attn.k_proj.weight", "attn.v_proj.weight"])
        self.wo = proj(["attn.o_proj.weight"])
        self.wgu = proj(["mlp.gate_proj.weight", "mlp.up_proj.weight"])
        self.wd = proj(["mlp.down_proj.weight"])
        self.normed = ops.mx_empty(B, self.D, bits=self.bits, device=dev)
        self.attended = ops.mx_empty(B, self.H * self.hd, bits=self.bits, device=dev)
        self.gated = ops.mx_empty(B, self.F, bits=self.bits, device=dev)

    def _project(self, x: torch.Tensor) -> None:
        ops.mx_rmsnorm(x, self.g1, self.eps, *self.normed)
        ops.mx_gemm(*self.normed, *self.wqkv, self.qkv)

    def _after_attention(self, x: torch.Tensor) -> torch.Tensor:
        ops.mx_quantize(self.attn, *self.attended)
        ops.mx_gemm(*self.attended, *self.wo, self.x1, residual=x)
        ops.mx_rmsnorm(self.x1, self.g2, self.eps, *self.normed)
        ops.mx_swiglu(*self.normed, *self.wgu, *self.gated)
        return ops.mx_gemm(*self.gated, *self.wd, self.out, residual=self.x1)

    def weight_bytes(self) -> int:
        return sum(t.numel() for p in (self.wqkv, self.wo, self.wgu, self.wd) for t in p)
