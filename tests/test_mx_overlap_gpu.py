"""Operands of the mx_ calls in shared buffers: those whose rows lie apart are taken, those that meet refused."""

from __future__ import annotations

import pytest
import torch

import mx_oracle

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def operands(m, n, k, gpu):
    g = torch.Generator().manual_seed(m)
    out = []
    for rows, bits in ((m, 8), (n, 4)):
        q, s = mx_oracle.quantized(torch.randint(-4, 5, (rows, k), generator=g), bits)
        out += [mx_oracle.encode(q, bits).to(gpu), s.to(torch.uint8).to(gpu)]
    return out


def exact(a, sa, w, sw):
    return mx_oracle.values(a, sa) @ mx_oracle.values(w, sw).t()


@pytest.mark.parametrize("m", [5, 700])
def test_results_over_what_is_read_are_refused(gpu, m):
    from torch_helion.hip import abi, ops

    a, sa, w, sw = operands(m, 512, 256, gpu)
    codes, _ = ops.mx_empty(m, 256, bits=8)
    held = torch.zeros(m, 520, dtype=BF16, device=gpu)
    x, gain = torch.zeros(m, 256, dtype=BF16, device=gpu), torch.ones(256, device=gpu)
    for call in (lambda: ops.mx_swiglu(a, sa, w, sw, codes, sa),                                       # scales over scales that are read
                 lambda: ops.mx_swiglu(a, sa, w, sw, a, torch.empty_like(sa)),
                 lambda: ops.mx_gemm(a, sa, w, sw, held[:, :512], residual=held[:, 1:513]),             # a residual a column further on
                 lambda: ops.mx_gemm(a[1:], sa[1:], w, sw, held[1:, :512], residual=held[:-1, :512]),   # and a row before
                 lambda: ops.mx_rmsnorm(x[1:], gain, 1e-5, codes[1:], torch.empty_like(sa)[1:], sum_out=x[:-1]),
                 lambda: ops.mx_quantize(x[:, :128], x.view(torch.uint8)[:, 240:368].view(torch.float8_e4m3fn), torch.empty_like(sa)[:, :4]),
                 lambda: ops.mx_dequantize(codes[:, :128], sa[:, :4], codes.view(BF16)[:, :128])):
        with pytest.raises(abi.HipBackendError, match="memory of"):
            call()


@pytest.mark.parametrize("m", [5, 700])
def test_rows_between_each_other_are_taken(gpu, m):
    """A residual and the result as columns of one buffer; activations and the result's scales in another."""
    from torch_helion.hip import ops

    a, sa, w, sw = operands(m, 512, 256, gpu)
    held = torch.zeros(m, 1024, dtype=BF16, device=gpu)
    held[:, 512:] = torch.randint(-64, 65, (m, 512), generator=torch.Generator().manual_seed(1)).to(BF16)
    ops.mx_gemm(a, sa, w, sw, held[:, :512], residual=held[:, 512:])
    ref = exact(a, sa, w, sw)
    assert torch.equal(held[:, :512].cpu(), (ref + held[:, 512:].cpu().double()).to(BF16))
    buf = torch.zeros(m, 256 + 16 + 16, dtype=torch.uint8, device=gpu)
    buf[:, :256] = a.view(torch.uint8)
    codes, want = ops.mx_empty(m, 256, bits=8), ops.mx_empty(m, 256, bits=8)
    ops.mx_swiglu(a, sa, w, sw, *want)
    ops.mx_swiglu(buf[:, :256].view(a.dtype), sa, w, sw, codes[0], buf[:, 260:268])
    assert torch.equal(codes[0].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(buf[:, 260:268], want[1])
    assert torch.equal(buf[:, :256], a.view(torch.uint8)) and not buf[:, 256:260].any() and not buf[:, 268:].any()
