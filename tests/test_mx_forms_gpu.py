"""th_mx_gemm in every form it has (th_mx_gemm_form), each test on the form that it names.

The operands are such that every sum is exact in fp32, in whatever order: elements of a whole numbers up to 4 (e4m3) or
multiples of 1/2 up to 6 (e2m1), of w multiples of 1/2 up to 6, every block with a scale of its own of 1/2, 1 or 2. Products
are multiples of 2^-4 (1/2 * 1/2 * 1/4) up to 144 (6 * 6 * 4), a sum of 1152 of them is below 2^18, in all 22 bits. So are sums with a
residual in eighths up to 8. fp32 results equal the sums of 64 bits, bf16 ones those rounded once; a SwiGLU is off by
(|g| + 8) 2^-23 of itself at most (the exponential's argument is rounded once: |g| 2^-24, and two more steps; then the
sum, the reciprocal and two products)."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

import mx_oracle
from conftest import announce

pytestmark = pytest.mark.gpu

E4M3, BF16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32
# (form, least rows): the ring has instances for up to 8, 16 and 32 rows, and takes 32 a workgroup
FORMS = {"ring": (0, 1), "ring9": (0, 9), "ring17": (0, 17), "ring33": (0, 33), "64x64": (1, 1), "64x128": (2, 1), "128x256": (3, 1),
         "256x256": (4, 1)}
ROWS = [1, 8, 9, 17, 33, 67, 130, 200, 257, 333, 515, 700, 1001, 1500, 2049, 3001, 4099, 6001, 8193, 16385]
OUTS = [70, 418, 801, 1058, 2083, 4130, 5217, 7010, 14338]


def size_of(name, nb, bits, swiglu, odd):
    """(rows, outs) of the smallest call among ROWS x OUTS (with swiglu whole blocks) that runs in this form."""
    from torch_helion.hip import abi

    lib = abi.init_device(0)
    d, got = abi.MxGemmDesc(), (C.c_int32 * 2)()
    d.blocks, d.a_dtype, d.swiglu = nb, abi.TH_F4E2M1 if bits == 4 else abi.TH_F8E4M3, swiglu
    d.a, d.a_scales, d.w, d.w_scales, d.out = 1 << 44, 2 << 44 | odd, 3 << 44, 4 << 44, 5 << 44
    d.ld_a, d.ld_w, d.ld_a_scales, d.ld_w_scales = nb * 4 * bits, nb * 16, nb, nb
    d.out_dtype = abi.TH_F8E4M3 if swiglu else abi.TH_F32
    if swiglu:
        d.out_scales, d.ld_out_scales = 6 << 44, 1 << 20
    form, least = FORMS[name]
    for m, n in sorted(((m, n // 32 * 32 if swiglu else n) for m in ROWS if m >= least for n in OUTS), key=lambda t: t[0] * t[1]):
        d.rows, d.outs, d.ld_out = m, n, max(n, 1 << 20)
        abi.check(lib.th_mx_gemm_form(bytes(d), got), "th_mx_gemm_form")
        if got[0] == form:
            return m, n
    raise AssertionError(f"no size of {nb} blocks runs in form {name}")


def gen(gpu, seed):
    return torch.Generator(device=gpu).manual_seed(seed)


def operand(rows, nb, bits, g, gpu, shift=0):
    """(codes, scales, values) of one side; bits 8: whole numbers up to 4."""
    s = torch.randint(126 + shift, 129 + shift, (rows, nb), generator=g, dtype=torch.uint8, device=gpu)
    if bits == 8:
        x = torch.randint(-4, 5, (rows, 32 * nb), generator=g, device=gpu).double()
        codes = x.to(E4M3)
    else:
        codes = torch.randint(0, 256, (rows, 16 * nb), generator=g, dtype=torch.uint8, device=gpu)
        table = torch.cat([mx_oracle.grid(4), -mx_oracle.grid(4)]).to(gpu)
        x = table[torch.stack([codes & 15, codes >> 4], -1).long()].flatten(1)
    return codes, s, x * torch.exp2(s.double() - 127).repeat_interleave(32, 1)


def placed(t, layout, gpu, more=0):
    """t inside wider rows of 0xff. "apart": codes 16 bytes in, scales 4, strides in whole dwords; "odd": scales 3 bytes in, at
    odd strides."""
    if layout == "plain":
        return t
    raw = t.view(torch.uint8)
    wide = raw.shape[1] % 16 == 0 and raw.shape[1] >= 16 and t.dtype is E4M3 or more
    if wide:
        first, stride = 16, raw.shape[1] + 16 + more
    elif layout == "apart":
        first, stride = 4, -(-raw.shape[1] // 4) * 4 + 8
    else:
        first, stride = 3, raw.shape[1] + 7
    held = torch.full((raw.shape[0], stride), 0xff, dtype=torch.uint8, device=gpu)
    held[:, first:first + raw.shape[1]] = raw
    return held[:, first:first + raw.shape[1]].view(t.dtype)


def product(a, w):
    return a @ w.t().contiguous()


def make(form, nb, bits, layout, gpu, *, swiglu=False, seed=0):
    m, n = size_of(form, nb, bits, swiglu, layout == "odd")
    g = gen(gpu, seed + 100 * list(FORMS).index(form) + nb)
    a, sa, x = operand(m, nb, bits, g, gpu)
    w, sw, y = operand(2 * n if swiglu else n, nb, 4, g, gpu, -6 if swiglu else 0)
    return m, n, g, (a, sa, x), (w, sw, y)


def laid(a, sa, w, sw, layout, gpu):
    return placed(a, layout, gpu, 32), placed(sa, layout, gpu), placed(w, layout, gpu, 64), placed(sw, layout, gpu)


def check(form, nb, bits, dtype, gpu, *, layout="plain", residual=False, in_place=False):
    from torch_helion.hip import ops

    m, n, g, (a, sa, x), (w, sw, y) = make(form, nb, bits, layout, gpu)
    announce(f"mx_gemm form {form} m={m} n={n} blocks={nb} bits={bits} {dtype} {layout} residual={residual} in_place={in_place}")
    pad = 0 if layout == "plain" else 5
    held = torch.full((m, n + 2 * pad), 7.0, dtype=dtype, device=gpu)
    out = held[:, pad:pad + n]
    ref, r = product(x, y), None
    if residual:
        r = torch.randint(-64, 65, (m, n), generator=g, device=gpu).to(dtype) / 8
        ref += r.double()
        if in_place:
            out.copy_(r)
            r = out
    args = laid(a, sa, w, sw, layout, gpu)
    assert ops.mx_gemm_form(*args, out, residual=r) == (FORMS[form][0], nb % 4 != 0 or layout == "odd")
    assert ops.mx_gemm(*args, out, residual=r) is out
    assert torch.equal(out, ref.to(dtype))
    assert (held[:, :pad] == 7).all() and (held[:, pad + n:] == 7).all()


def forms(blocks):
    """Every form with every number of blocks that it takes."""
    return [(f, nb) for f in FORMS for nb in blocks if f != "256x256" or nb % 4 == 0]


# (the ring's four-stage waves and the tiles' rings of three and four stages: fewer stages than these, as many, and more)
@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("form,nb", forms([1, 2, 3, 4, 5, 8, 9, 12, 15, 16, 17, 20, 24, 30, 36]))
def test_stages(gpu, form, nb, bits):
    check(form, nb, bits, F32, gpu, residual=nb % 2 == 1)
    check(form, nb, bits, BF16, gpu, residual=nb % 2 == 0)


# (scales at odd addresses take the smaller forms)
LAYOUTS = [(f, nb, layout) for f, nb in forms([8, 13, 20]) for layout in ("apart", "odd") if (f, layout) != ("256x256", "odd")]


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("form,nb,layout", LAYOUTS)
def test_strides_and_in_place(gpu, form, nb, bits, layout):
    check(form, nb, bits, BF16, gpu, layout=layout, residual=True, in_place=True)
    check(form, nb, bits, F32, gpu, layout=layout, residual=True, in_place=True)
    check(form, nb, bits, F32, gpu, layout=layout)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("form,nb", forms([4, 13, 20]))
def test_nan_blocks_and_elements(gpu, form, nb, bits):
    from torch_helion.hip import ops

    m, n, _, (a, sa, x), (w, sw, y) = make(form, nb, bits, "plain", gpu)
    announce(f"mx_gemm NaN in form {form} m={m} n={n} blocks={nb} bits={bits}")
    nan = torch.zeros(m, n, dtype=torch.bool, device=gpu)
    sa[m // 2, nb - 1], sw[n // 3, 0], sw[n - 1, nb - 1] = 255, 255, 255
    nan[m // 2], nan[:, n // 3], nan[:, n - 1] = True, True, True
    if bits == 8 and m > 1:
        a.view(torch.uint8)[m - 1, 32 * nb - 1] = 0xff
        nan[m - 1] = True
    out = torch.zeros(m, n, device=gpu)
    ops.mx_gemm(a, sa, w, sw, out)
    assert ops.mx_gemm_form(a, sa, w, sw, out)[0] == FORMS[form][0]
    assert torch.equal(torch.isnan(out), nan)
    assert torch.equal(out[~nan], product(x, y).float()[~nan])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("form,nb", forms([4, 13]))
def test_far_scales(gpu, form, nb, bits):
    """Rows and columns of scales from 2^-127 to 2^127: sums stay exact whose partial sums are within fp32's normal numbers, that
    is whose magnitudes add up to less than 2^127 (no partial sum is more), and that are over 2^-100 (unscaled they are
    below 2^18 and multiples of 2^-2, so that none of their bits is below 2^-120)."""
    from torch_helion.hip import ops

    m, n, g, (a, sa, x), (w, sw, y) = make(form, nb, bits, "plain", gpu)
    announce(f"mx_gemm far scales in form {form} m={m} n={n} blocks={nb} bits={bits}")
    x, y = (t * torch.exp2(127.0 - s.double()).repeat_interleave(32, 1) for t, s in ((x, sa), (y, sw)))
    ra = torch.randint(0, 255, (m, 1), generator=g, dtype=torch.uint8, device=gpu)
    rw = torch.randint(100, 150, (n, 1), generator=g, dtype=torch.uint8, device=gpu)
    ra[0], rw[0], rw[1] = 0, 254, 0
    ra[-1] = 254
    sa, sw = ra.repeat(1, nb), rw.repeat(1, nb)
    out = torch.zeros(m, n, device=gpu)
    ops.mx_gemm(a, sa, w, sw, out)
    unit = torch.exp2(ra.double() - 127) * torch.exp2(rw.double() - 127).t()
    ref = product(x, y) * unit
    plain = (ref.abs() > 2.0 ** -100) & (product(x.abs(), y.abs()) * unit < 2.0 ** 127)
    assert plain[-1].any() and (m == 1 or plain[:, 0].any())    # (of one row the only scale is the largest)
    assert torch.equal(out[plain], ref.float()[plain])


def check_swiglu(form, nb, bits, out_bits, gpu, layout="plain"):
    from torch_helion.hip import ops

    m, n, _, (a, sa, x), (w, sw, y) = make(form, nb, bits, layout, gpu, swiglu=True)
    announce(f"mx_swiglu form {form} m={m} outs={n} blocks={nb} bits={bits} -> {out_bits} {layout}")
    codes, scales = (placed(t.fill_(0x55), layout, gpu, more)
                     for t, more in zip((t.view(torch.uint8) for t in ops.mx_empty(m, n, bits=out_bits)), (16, 0)))
    codes = codes if out_bits == 4 else codes.view(E4M3)
    args = laid(a, sa, w, sw, layout, gpu)
    assert ops.mx_swiglu_form(*args, codes, scales) == (FORMS[form][0], nb % 4 != 0 or layout == "odd")
    ops.mx_swiglu(*args, codes, scales)
    # (some hundred rows: every row of a workgroup's tile, and the last ones)
    at = torch.cat([torch.arange(0, m, max(1, m // 300)), torch.arange(max(0, m - 40), m)]).to(gpu)
    p, q = product(x[at], y).split(n, 1)
    z = p * torch.sigmoid(p) * q
    mx_oracle.assert_blocks_within(codes[at].cpu(), scales[at].cpu(), z.cpu(), ((p.abs() + 8) * 2.0 ** -23 * z.abs()).cpu(), out_bits)
    for t in (codes.view(torch.uint8), scales):
        if t.stride(0) > t.shape[1]:    # what lies between the rows stays
            rest = t.as_strided((m - 1, t.stride(0) - t.shape[1]), (t.stride(0), 1), t.storage_offset() + t.shape[1])
            assert (rest == 0xff).all()


@pytest.mark.parametrize("bits,out_bits", [(8, 8), (8, 4), (4, 8), (4, 4)])
@pytest.mark.parametrize("form,nb", [(f, nb) for f, nb in forms([1, 3, 4, 5, 8, 13, 20]) if f != "64x64"])
def test_swiglu(gpu, form, nb, bits, out_bits):
    check_swiglu(form, nb, bits, out_bits, gpu)


@pytest.mark.parametrize("bits,out_bits", [(8, 8), (8, 4), (4, 8), (4, 4)])
@pytest.mark.parametrize("form,nb,layout", [x for x in LAYOUTS if x[0] != "64x64"])
def test_swiglu_strides(gpu, form, nb, bits, out_bits, layout):
    check_swiglu(form, nb, bits, out_bits, gpu, layout)


@pytest.mark.parametrize("form,nb", [("ring33", 36), ("64x64", 13), ("64x128", 12), ("128x256", 12), ("128x256", 13), ("256x256", 20)])
def test_two_streams_and_a_graph(gpu, form, nb):
    """Calls at once on two streams, and replays of a graph between eager calls: equal bits each time."""
    from torch_helion.hip import ops

    m, n, g, (a, sa, x), (w, sw, y) = make(form, nb, 8, "plain", gpu)
    announce(f"mx_gemm form {form} m={m} n={n} blocks={nb}: streams and a graph")
    want = product(x, y).float()
    torch.cuda.synchronize()
    outs = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            for _ in range(3):
                outs.append(torch.empty(m, n, device=gpu))
                ops.mx_gemm(a, sa, w, sw, outs[-1])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    out, graph = torch.zeros(m, n, device=gpu), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.mx_gemm(a, sa, w, sw, out)
    for _ in range(3):
        a.copy_(operand(m, nb, 8, g, gpu)[0])
        want = product(a.double() * torch.exp2(sa.double() - 127).repeat_interleave(32, 1), y).float()
        graph.replay()
        eager = torch.empty_like(out)
        ops.mx_gemm(a, sa, w, sw, eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(eager, want)
        out.zero_()
