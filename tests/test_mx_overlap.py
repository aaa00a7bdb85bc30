"""What the th_mx_ calls write shares no memory with what they read: by ranges of bytes, row by row (no GPU)."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from test_mx import ENTRY, SWIGLU, _desc, lib  # noqa: F401


def status(lib, name, over):  # noqa: F811
    """What the call says; a product's form query says it without a device."""
    if torch.cuda.is_available() and name != "MxGemmDesc":
        pytest.skip("a GPU is present, and these pointers are no memory")
    if name == "MxGemmDesc":
        return lib.th_mx_gemm_form(bytes(_desc(name, **over)), (C.c_int32 * 2)())
    return getattr(lib, ENTRY[name])(bytes(_desc(name, **over)), None)


# rows=4: x 4096 + 512 (bf16), codes 8192 + 128 or 256, scales 12288 + 8, gain 16384 + 256; gemm: a 4096 + 256, a_scales 8192 + 8,
# w 12288 + 64 * 32, w_scales 16384 + 128, out 20480 + 4 * 128 (swiglu: + 256, out_scales 24576 + 8)
@pytest.mark.parametrize("name,over", [
    ("MxQuantizeDesc", dict(codes=4096 + 16)), ("MxQuantizeDesc", dict(codes=4096 - 112)), ("MxQuantizeDesc", dict(scales=4096 + 511)),
    ("MxQuantizeDesc", dict(scales=8192 + 127)), ("MxQuantizeDesc", dict(scales=8192 - 7)), ("MxQuantizeDesc", dict(codes=4096 + 128, ld_codes=256)),
    ("MxDequantizeDesc", dict(out=8192 + 2)), ("MxDequantizeDesc", dict(out=8192 - 510)), ("MxDequantizeDesc", dict(out=12288 + 6)),
    ("MxDequantizeDesc", dict(out=12288 - 256)),
    ("MxRmsNormDesc", dict(codes=4096 + 64)), ("MxRmsNormDesc", dict(scales=4096 + 100)), ("MxRmsNormDesc", dict(scales=8192 + 200)),
    ("MxRmsNormDesc", dict(scales=16384 + 255)), ("MxRmsNormDesc", dict(residual=8192 + 128, ld_residual=64)),
    ("MxRmsNormDesc", dict(sum_out=4096 + 2, ld_sum_out=64)), ("MxRmsNormDesc", dict(sum_out=4096 + 128, ld_sum_out=64)),
    ("MxRmsNormDesc", dict(residual=20480, ld_residual=64, sum_out=20480 - 128, ld_sum_out=64)),
    ("MxRmsNormDesc", dict(sum_out=16384 - 508, ld_sum_out=64)), ("MxRmsNormDesc", dict(sum_out=12288 + 4, ld_sum_out=64)),
    ("MxGemmDesc", dict(out=4096 + 254)), ("MxGemmDesc", dict(out=8192 + 4)), ("MxGemmDesc", dict(out=8192)),
    ("MxGemmDesc", dict(out=12288 + 2046)), ("MxGemmDesc", dict(out=16384 - 510)), ("MxGemmDesc", dict(out=16384)),
    ("MxGemmDesc", dict(residual=20480 + 2, ld_residual=64)), ("MxGemmDesc", dict(residual=20480 + 128, ld_residual=64)),
    ("MxGemmDesc", dict(residual=20480 - 128, ld_residual=64)),
    ("MxGemmDesc", dict(SWIGLU, out_scales=8192)), ("MxGemmDesc", dict(SWIGLU, out_scales=8192 + 7)), ("MxGemmDesc", dict(SWIGLU, out_scales=4096)),
    ("MxGemmDesc", dict(SWIGLU, out_scales=12288 + 4095)), ("MxGemmDesc", dict(SWIGLU, out_scales=16384 + 255)),
    ("MxGemmDesc", dict(SWIGLU, out_scales=20480 + 255)), ("MxGemmDesc", dict(SWIGLU, out=8192 - 16)), ("MxGemmDesc", dict(SWIGLU, out=16384 + 128)),
])
def test_shared_memory_is_refused(lib, name, over):  # noqa: F811
    from torch_helion.hip import abi

    assert status(lib, name, over) == abi.TH_ERR_INVALID and "memory of" in abi.last_error(lib), abi.last_error(lib)


# rows of one tensor between those of another: columns of a wider one; other strides whose rows do not meet
@pytest.mark.parametrize("name,over", [
    ("MxQuantizeDesc", dict(ld_x=128, codes=4096 + 128, ld_codes=256)), ("MxQuantizeDesc", dict(ld_codes=64, scales=8192 + 32, ld_scales=64)),
    ("MxQuantizeDesc", dict(ld_x=128, codes=4096 + 128 + 256, ld_codes=512)), ("MxQuantizeDesc", dict(codes=4096 + 512)),
    ("MxDequantizeDesc", dict(ld_codes=256, out=8192 + 64 + 2, ld_out=128)),
    ("MxRmsNormDesc", dict(sum_out=4096, ld_sum_out=64)), ("MxRmsNormDesc", dict(ld_x=128, sum_out=4096 + 128, ld_sum_out=128)),
    ("MxRmsNormDesc", dict(residual=4096, ld_residual=64, sum_out=4096, ld_sum_out=64)),
    ("MxRmsNormDesc", dict(rows=1, sum_out=4096, ld_sum_out=96)),
    ("MxGemmDesc", dict(residual=20480, ld_residual=64)), ("MxGemmDesc", dict(ld_out=128, residual=20480 + 128, ld_residual=128)),
    ("MxGemmDesc", dict(ld_a=512, out=4096 + 64, ld_out=256)), ("MxGemmDesc", dict(rows=1, residual=20480, ld_residual=96)),
    ("MxGemmDesc", dict(SWIGLU, ld_out=128, out_scales=20480 + 64, ld_out_scales=128)),
])
def test_rows_between_others_are_taken(lib, name, over):  # noqa: F811
    from torch_helion.hip import abi

    want = abi.TH_OK if name == "MxGemmDesc" else abi.TH_ERR_NOT_INIT
    assert status(lib, name, over) == want, abi.last_error(lib)


def test_every_pair_of_strides(lib):  # noqa: F811
    """Two tensors of rows of a few bytes, at every offset and stride, against the bytes they stand for."""
    from torch_helion.hip import abi

    base = 1 << 20

    def held(p, rows, ld, width):
        return {p + i * ld + j for i in range(rows) for j in range(width)}

    met = apart = 0
    for ld_codes in (16, 32, 48):
        for ld_scales in (1, 3, 16, 20, 32, 50):
            for rows in (1, 2, 3, 5):
                for off in range(-60, 160, 3):
                    over = dict(rows=rows, cols=32, ld_x=32, x=1 << 30, codes=base, ld_codes=ld_codes, scales=base + off, ld_scales=ld_scales)
                    got = status(lib, "MxQuantizeDesc", over)
                    share = bool(held(base, rows, ld_codes, 16) & held(base + off, rows, ld_scales, 1))
                    met, apart = met + share, apart + (not share)
                    assert got == (abi.TH_ERR_INVALID if share else abi.TH_ERR_NOT_INIT), (over, abi.last_error(lib))
    assert met > 200 and apart > 200
