"""th_mx_gemm_form on the CPU: which form th_mx_gemm takes, for 256 compute units."""

from __future__ import annotations

import pytest
import torch

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def lib():
    from torch_helion.hip import abi

    if not abi.library_path().exists():
        pytest.skip("libth_hip.so not built (run __graft_entry__.build())")
    if torch.cuda.is_available():
        pytest.skip("the card's compute units count; this checks the choice for 256")
    return abi.load()


def form(m, n, nb, bits=8, swiglu=False, scales_at=0):
    from torch_helion.hip import ops

    def sides(rows, wide):
        s = torch.empty(rows * nb + scales_at, dtype=torch.uint8)[scales_at:].view(rows, nb)
        c = torch.empty(rows, wide, dtype=torch.uint8)
        return c, s
    a, sa = sides(m, nb * 4 * bits)
    w, sw = sides(2 * n if swiglu else n, 16 * nb)
    a = a if bits == 4 else a.view(E4M3)
    if swiglu:
        return ops.mx_swiglu_form(a, sa, w, sw, *ops.mx_empty(m, n, bits=8, device="cpu"))
    return ops.mx_gemm_form(a, sa, w, sw, torch.empty(m, n, dtype=torch.bfloat16))


# the sizes at which every form was timed, and the fastest or one within 8 % of it
@pytest.mark.parametrize("m,n,nb,bits,swiglu,forms", [
    (1, 6144, 128, 8, False, {0}), (64, 4096, 128, 8, False, {0}), (64, 14336, 128, 8, False, {1}), (256, 4096, 128, 8, False, {1}),
    (512, 4096, 128, 8, False, {1, 2}), (512, 14336, 128, 8, False, {3}), (2048, 4096, 128, 8, False, {3}),
    (2048, 14336, 128, 8, False, {4}), (333, 2050, 43, 8, False, {1}), (2048, 4096, 127, 8, False, {3}),
    (64, 4096, 128, 4, False, {0}), (64, 14336, 128, 4, False, {1}), (512, 4096, 128, 4, False, {2}), (2048, 4096, 128, 4, False, {3}),
    (2048, 14336, 128, 4, False, {4}), (1, 14336, 128, 8, True, {0}), (64, 14336, 128, 8, True, {2}), (512, 14336, 128, 8, True, {4}),
    (64, 14336, 128, 4, True, {2}), (256, 14336, 128, 4, True, {3}), (1024, 14336, 128, 4, True, {4})])
def test_the_choice(m, n, nb, bits, swiglu, forms):
    got, bytewise = form(m, n, nb, bits, swiglu)
    assert got in forms and bytewise == (nb % 4 != 0)


def test_scales_at_odd_addresses_are_loaded_byte_by_byte():
    assert form(2048, 4096, 8, scales_at=4)[1] is False
    for at in (1, 2, 3):
        got, bytewise = form(2048, 4096, 8, scales_at=at)
        assert bytewise and got != 4


def test_refusals():
    from torch_helion.hip import abi, ops

    a, s = torch.empty(4, 64, dtype=E4M3), torch.empty(4, 2, dtype=torch.uint8)
    w, sw = torch.empty(6, 32, dtype=torch.uint8), torch.empty(6, 2, dtype=torch.uint8)
    with pytest.raises(abi.HipBackendError):
        ops.mx_gemm_form(a, s, w, sw, torch.empty(4, 7))
    with pytest.raises(abi.HipBackendError):
        ops.mx_swiglu_form(a, s, w, sw, *ops.mx_empty(4, 32, bits=8, device="cpu"))
    assert abi.load().th_mx_gemm_form(None, None) == abi.TH_ERR_INVALID
