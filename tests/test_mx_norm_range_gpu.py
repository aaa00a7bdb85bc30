"""th_mx_rmsnorm of finite rows whose squares leave fp32's range: the blocks of the formula in 64 bits.

Such a row is summed again in units of a power of two, so the bound is the one of other rows (test_mx_gpu.NORM): the
scaled squares are rounded as the others are, and those that underflow (of values 2^-46 beside one of 2^56 at least) do not count."""

from __future__ import annotations

import pytest
import torch

import mx_oracle
from conftest import announce
from test_mx_gpu import BF16, F32, NORM, empty, gen

pytestmark = pytest.mark.gpu

# one width of every instance: waves a row, chunks a lane
COLS = [40, 512, 2048, 4096, 8000, 16384, 32768, 40000]


def check(gpu, x, eps, bits, what, residual=None):
    from torch_helion.hip import ops

    announce(f"mx_rmsnorm range {what} {tuple(x.shape)} {x.dtype} eps={eps} bits={bits}")
    rows, cols = x.shape
    gain = 1.0 + 0.3 * torch.rand(cols, generator=gen(cols))
    codes, scales = empty(rows, cols, bits, gpu)
    ops.mx_rmsnorm(x.to(gpu), gain.to(gpu), eps, codes, scales, residual=None if residual is None else residual.to(gpu))
    h = x.double() if residual is None else (x.float() + residual.float()).to(x.dtype).double()
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + torch.tensor(eps, dtype=F32).double()) * gain.double()
    mx_oracle.assert_blocks_within(codes, scales, y, NORM * y.abs(), bits, what)


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("bits", [8, 4])
def test_huge_rows(gpu, cols, dtype, bits):
    """From the least that overflows to the largest numbers there are, ordinary rows between them, and one large value alone."""
    x = torch.randn(9, cols, generator=gen(cols)).double()
    top = x.abs().amax(1, keepdim=True)
    x = x / top * torch.tensor([2.0 ** e for e in (0, 62, 63, 64, 80, 100, 126, 127.99, 3)], dtype=torch.float64)[:, None]
    x[8] = 0.0
    x[8, cols // 2] = -2.0 ** 127
    x[4, : cols // 2] *= 2.0 ** -70      # small values beside huge ones
    check(gpu, x.to(dtype), 1e-5, bits, "huge")
    check(gpu, (x / 4).to(dtype), 1e-5, bits, "huge, with a residual", residual=(x / 2).to(dtype))


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("eps", [0.0, 1e-42, 1e-38, 1e-30])
def test_tiny_rows_with_a_tiny_eps(gpu, cols, dtype, eps):
    """Down to rows of subnormal numbers. (eps held to fp32, where 1e-42 is a subnormal of few bits.)"""
    x = torch.randn(6, cols, generator=gen(cols + 1)).double()
    x = x / x.abs().amax(1, keepdim=True) * torch.tensor([2.0 ** e for e in (-60, -64, -70, -100, -120, 0)], dtype=torch.float64)[:, None]
    check(gpu, x.to(dtype), eps, 8, "tiny")


def test_infinities_and_zeros_stay_what_they_were(gpu):
    """An infinity makes its block NaN and the row's others zeros; a row of zeros is zeros, and without eps NaN (0 / 0)."""
    from torch_helion.hip import ops

    x = torch.randn(4, 256, generator=gen(1)) * 2.0 ** 100
    x[1, 40], x[2] = float("inf"), 0.0
    gain = torch.ones(256, device=gpu)
    for eps in (1e-5, 0.0):
        codes, scales = empty(4, 256, 8, gpu)
        ops.mx_rmsnorm(x.to(gpu), gain, eps, codes, scales)
        s, q = scales.cpu(), mx_oracle.elements(codes)
        assert s[1, 1] == 255 and (q[1, [0, 2, 3, 4, 5, 6, 7]] == 0).all() and (s[1, [0, 2, 3, 4, 5, 6, 7]] == 0).all()
        assert (q[2] == 0).all() and (s[2] == (255 if eps == 0.0 else 0)).all()
        assert (s[[0, 3]] < 255).all() and q[[0, 3]].any()
