"""Rotary positions and the paged KV cache: th_rope, th_paged_append, th_paged_attention and
th_page_copy against plain 64-bit implementations.

Tolerances are bounds of the arithmetic, elementwise. u(t) = torch.finfo(t).eps / 2 is a rounding's
half step. A rotated value a c - b s is off by (|a| + |b|) times ROT = 6e-7: the fraction of a turn is
rounded to 2^-25 (1.9e-7 of angle), sine and cosine to two steps of 2^-24 (1.2e-7), the scale, the two
products and the sum to one each (2.4e-7). An attention output is off by u(bf16) from its own rounding
and, against A = sum_j p_j |v_j|, by u(bf16) from the rounded p_j plus twice the score error, which is
head_dim 2^-22 scale sum_i |q_i k_i| for an fp32 accumulation in any order (twice its bound), 2^-20
softcap for the capped tanh, and 2^-20 for the exponential and the bias.
"""

from __future__ import annotations

import math

import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu

ROT = 6e-7
E4M3 = torch.float8_e4m3fn
BF16 = torch.bfloat16


def u(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def rope64(x, positions, freqs, interleaved=False, scale=1.0, inverse=False):
    """(rotated, |a| + |b| of each element's pair) of x [t, h, d], float64 on the CPU."""
    x = x.double()
    n = freqs.numel()
    ang = positions.double()[:, None, None] * freqs.double() * (-1.0 if inverse else 1.0)
    cos, sin = ang.cos() * scale, ang.sin() * scale
    ia = torch.arange(n) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else n)
    y, mag = x.clone(), torch.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
    mag[..., ia] = mag[..., ib] = (a.abs() + b.abs()) * scale
    return y, mag


def assert_within(got, ref, tol, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    over = ((got - ref).abs() - tol).max().item()
    assert over <= 0.0, f"{what}: {over:.3e} over the bound"


# ------------------------------------------------------------------ rope
@pytest.mark.parametrize("t,h,d,rot,interleaved,dtype,idx", [
    (1, 1, 64, 64, False, torch.bfloat16, torch.int32), (1, 32, 128, 128, False, torch.bfloat16, torch.int64),
    (65, 8, 128, 64, True, torch.bfloat16, torch.int32), (33, 3, 96, 40, False, torch.float32, torch.int64),
    (17, 5, 80, 80, True, torch.float32, torch.int32), (9, 2, 18, 6, False, torch.bfloat16, torch.int32),
    (257, 12, 64, 32, False, torch.float32, torch.int32), (40, 1, 256, 256, True, torch.bfloat16, torch.int32),
    (5, 2, 1024, 1024, False, torch.float32, torch.int32), (1000, 32, 128, 128, False, torch.bfloat16, torch.int32),
    (3, 7, 5, 2, True, torch.float32, torch.int32), (301, 4, 128, 104, False, torch.bfloat16, torch.int32),
])
def test_rope(gpu, t, h, d, rot, interleaved, dtype, idx):
    from torch_helion.hip import ops

    announce(f"rope t={t} h={h} d={d} rot={rot} interleaved={interleaved} {dtype}")
    g = gen(t * 7 + d)
    x = torch.randn(t, h * d, generator=g).to(dtype)
    pos = torch.randint(0, 5000, (t,), generator=g, dtype=idx)
    f = ops.rope_frequencies(rot, 10000.0)
    ref, mag = rope64(x.view(t, h, d), pos, f, interleaved, 1.25)
    out = torch.full((t, h * d), float("nan"), dtype=dtype, device=gpu)
    xd = x.to(gpu)
    ops.rope(xd, pos.to(gpu), f.to(gpu), out, head_dim=d, interleaved=interleaved, scale=1.25)
    torch.cuda.synchronize()
    half = u(dtype) if dtype == torch.bfloat16 else 0.0
    assert_within(out.view(t, h, d), ref, ROT * mag + half * ref.abs() + 1e-30, "rope")
    assert torch.equal(out.view(t, h, d)[..., rot:].cpu(), x.view(t, h, d)[..., rot:])
    ops.rope(xd, pos.to(gpu), f.to(gpu), xd, head_dim=d, interleaved=interleaved, scale=1.25)
    assert torch.equal(xd, out)


@pytest.mark.parametrize("first", [0, (1 << 31) - 600, -70000])
def test_rope_far_positions(gpu, first):
    """Angles of far (and negative) positions keep their accuracy: reduced in 64 bits. The reference's own
    product position * frequency is off by 2^-53 of up to 2^31 radians."""
    from torch_helion.hip import ops

    announce(f"rope far positions from {first}")
    t, h, d = 600, 2, 64
    x = torch.randn(t, h * d, generator=gen(3))
    pos = torch.arange(first, first + t, dtype=torch.int64)
    f = ops.rope_frequencies(d, 500000.0)
    ref, mag = rope64(x.view(t, h, d), pos, f)
    out = torch.empty(t, h * d, device=gpu)
    ops.rope(x.to(gpu), pos.to(gpu), f.to(gpu), out, head_dim=d)
    assert_within(out.view(t, h, d), ref, (ROT + 2e-6 * (abs(first) > 1 << 30)) * mag + 1e-30)


@pytest.mark.parametrize("t,h,d,rot", [((1 << 24) + 5, 1, 6, 2), ((1 << 23) + 5, 33, 64, 64)])
def test_rope_of_more_workgroups_than_one_dimension_holds(gpu, t, h, d, rot):
    """A workgroup a token and more tokens than a launch takes along x, in place: the first, the last and those
    beside the powers of two."""
    from torch_helion.hip import ops

    announce(f"rope of {t} tokens h={h} d={d}")
    f = ops.rope_frequencies(rot, 10000.0)
    ids = torch.tensor([0, 1, (1 << 23) - 1, 1 << 23, t - 6, t - 5, t - 1], device=gpu)
    x = torch.full((t, h * d), 0.5, dtype=torch.bfloat16, device=gpu)
    x[ids] = torch.randn(len(ids), h * d, generator=gen(8)).to(torch.bfloat16).to(gpu)
    pos = torch.arange(t, dtype=torch.int32, device=gpu)
    before = x[ids].cpu()
    ops.rope(x, pos, f.to(gpu), x, head_dim=d)
    ref, mag = rope64(before.view(-1, h, d), pos[ids].cpu(), f)
    assert_within(x[ids].view(-1, h, d), ref, ROT * mag + u(torch.bfloat16) * ref.abs() + 1e-30)
    del x
    torch.cuda.empty_cache()


def test_rope_strided_rows_and_a_stream(gpu):
    """Column slices of a wider projection (rows not 16-byte aligned among them), on a side stream."""
    from torch_helion.hip import ops

    announce("rope on strided rows")
    for col, dtype in ((64, torch.bfloat16), (3, torch.bfloat16), (5, torch.float32)):
        wide = torch.randn(50, 64 * 6 + 11, generator=gen(col)).to(dtype).to(gpu)
        pos, f = torch.arange(50, dtype=torch.int32, device=gpu), ops.rope_frequencies(64, 10000.0, device=gpu)
        x = wide[:, col:col + 256]
        before = wide.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.rope(x, pos, f, x, head_dim=64)
        torch.cuda.current_stream().wait_stream(s)
        ref, mag = rope64(before[:, col:col + 256].reshape(50, 4, 64).cpu(), pos.cpu(), f.cpu())
        assert_within(x.reshape(50, 4, 64), ref, ROT * mag + u(dtype) * ref.abs() + 1e-30)
        assert torch.equal(wide[:, :col], before[:, :col]) and torch.equal(wide[:, col + 256:], before[:, col + 256:])


def test_rope_inverse_is_the_gradient(gpu):
    """inverse on the output's gradient against the formula's gradient in float64 and against differences."""
    from torch_helion.hip import ops

    announce("rope gradient")
    t, h, d, rot = 12, 3, 32, 24
    f = ops.rope_frequencies(rot, 10000.0)
    pos = torch.randint(0, 1000, (t,), generator=gen(1), dtype=torch.int32)
    x = torch.randn(t, h * d, generator=gen(2))
    go = torch.randn(t, h * d, generator=gen(3))
    xx = x.double().requires_grad_()
    y = rope64_plain(xx.view(t, h, d), pos, f, 0.9)
    (ref,) = torch.autograd.grad((y * go.view(t, h, d).double()).sum(), xx)
    got = torch.empty(t, h * d, device=gpu)
    ops.rope(go.to(gpu), pos.to(gpu), f.to(gpu), got, head_dim=d, scale=0.9, inverse=True)
    mag = go.view(t, h, d).abs().amax(-1, keepdim=True).double().expand(t, h, d).reshape(t, -1) * 2
    assert_within(got, ref, ROT * mag)
    # the map is linear: a difference along a direction is exact up to the two calls' roundings
    dx = torch.randn(t, h * d, generator=gen(4))
    outs = []
    for s in (1.0, -1.0):
        o = torch.empty(t, h * d, device=gpu)
        ops.rope((x + s * dx).to(gpu), pos.to(gpu), f.to(gpu), o, head_dim=d, scale=0.9)
        outs.append(o.double().cpu())
    along = ((outs[0] - outs[1]) / 2 * go.double()).sum().item()
    assert abs(along - (got.double().cpu() * dx.double()).sum().item()) < 1e-6 * t * h * d


def rope64_plain(x, pos, f, scale):
    n = f.numel()
    ang = pos.double()[:, None, None] * f
    a, b = x[..., :n], x[..., n:2 * n]
    return torch.cat([(a * ang.cos() - b * ang.sin()) * scale, (b * ang.cos() + a * ang.sin()) * scale, x[..., 2 * n:]], -1)


# ------------------------------------------------------------------ append
def paged(rows, row_pages, page_size, hk, d, dtype, g, gpu, spare=3, head_major=False):
    """(k_cache, v_cache, table) with random contents; the table's pages in a random order."""
    pages = rows * row_pages + spare
    shape = (pages, hk, page_size, d) if head_major else (pages, page_size, hk, d)
    caches = [torch.randn(shape, generator=g).to(dtype).to(gpu) for _ in range(2)]
    if head_major:
        caches = [c.transpose(1, 2) for c in caches]
    table = torch.randperm(pages, generator=g)[:rows * row_pages].view(rows, row_pages).to(torch.int32).to(gpu)
    return caches[0], caches[1], table


@pytest.mark.parametrize("hq,hk,d,rot,interleaved,ps,in_dtype,cache,head_major", [
    (32, 8, 128, 128, False, 16, torch.float32, BF16, False), (8, 8, 64, 64, False, 32, torch.bfloat16, BF16, True),
    (4, 1, 128, 64, True, 64, torch.bfloat16, E4M3, False), (0, 4, 64, 0, False, 16, torch.float32, E4M3, True),
    (6, 2, 96, 40, False, 8, torch.bfloat16, BF16, False), (3, 3, 20, 10, True, 1, torch.float32, E4M3, False),
    (12, 4, 128, 128, False, 256, torch.bfloat16, E4M3, False), (5, 2, 64, 0, False, 32, torch.float32, BF16, False), (1, 1, 128, 104, False, 32, torch.float32, BF16, False),
])
def test_append(gpu, hq, hk, d, rot, interleaved, ps, in_dtype, cache, head_major):
    """Ragged prompts, some padded tokens: the slots written, and nothing else."""
    from torch_helion.hip import ops

    announce(f"append hq={hq} hk={hk} d={d} rot={rot} ps={ps} {in_dtype} -> {cache} head_major={head_major}")
    g = gen(hq * 31 + d + ps)
    new, past = [1, 2 * ps + 3, 0, 37], [0, 5, 9, 3 * ps - 1]
    rows = torch.tensor([r for r, n in enumerate(new) for _ in range(n)], dtype=torch.int32)
    pos = torch.tensor([p + i for n, p in zip(new, past) for i in range(n)], dtype=torch.int32)
    pos[2] = -1                                                       # a padded token
    t, width = pos.numel(), -(-(max(p + n for n, p in zip(new, past))) // ps)
    kc, vc, table = paged(4, width, ps, hk, d, cache, g, gpu, head_major=head_major)
    kc0, vc0 = kc.float().cpu(), vc.float().cpu()
    qkv = torch.randn(t, (hq + 2 * hk) * d, generator=g).to(in_dtype)
    qkv[2] = float("nan")
    qd, kd, vd = qkv.to(gpu).split([hq * d, hk * d, hk * d], 1)
    scales = {}
    if cache == E4M3:
        scales = {n: (torch.rand(hk, generator=g) + 0.01).to(gpu) for n in ("k_scale", "v_scale")}
    f = ops.rope_frequencies(rot, 10000.0) if rot else None
    q_out = torch.full((t, max(hq * d, 1)), 7.0, dtype=BF16, device=gpu)
    bad = torch.zeros(1, dtype=torch.int32, device=gpu)
    ops.paged_append(kd, vd, pos.to(gpu), kc, vc, table, rows=rows.to(gpu), freqs=None if f is None else f.to(gpu),
                     interleaved=interleaved, rope_scale=1.1, q=qd if hq else None, q_out=q_out[:, :hq * d] if hq else None,
                     n_invalid=bad, **scales)
    torch.cuda.synchronize()
    assert bad.item() == 0
    q, k, v = (x.reshape(t, -1, d) for x in qkv.split([hq * d, hk * d, hk * d], 1))
    zero = torch.zeros_like(k, dtype=torch.float64)
    ref_k, mag_k = rope64(k, pos, f, interleaved, 1.1) if rot else (k.double(), zero)
    live = pos >= 0
    if hq:
        ref_q, mag_q = rope64(q, pos, f, interleaved, 1.1) if rot else (q.double(), torch.zeros_like(q).double())
        assert_within(q_out[live.to(gpu)].view(-1, hq, d), ref_q[live], (ROT * mag_q + u(BF16) * ref_q.abs() + 1e-30)[live], "q")
        assert (q_out[2] == 7.0).all()
    page = table.cpu()[rows.long(), pos.clamp(min=0).long() // ps].long()
    slot = (pos % ps).long()
    for got, was, ref, mag, sc in ((kc, kc0, ref_k, mag_k, "k_scale"), (vc, vc0, v.double(), zero, "v_scale")):
        got = got.float().cpu()
        if cache == E4M3:
            s = scales[sc].double().cpu()[:, None]
            ref, mag = (ref / s).clamp(-448, 448), mag / s
            # one step of the division's reciprocal, then half an e4m3 step (absolute 2^-10 below 2^-6)
            tol = (ROT * mag + 2.0 ** -22 * ref.abs()) * (1 + u(E4M3)) + torch.clamp(u(E4M3) * ref.abs(), min=2.0 ** -10)
        else:
            tol = ROT * mag + u(BF16) * ref.abs() + 1e-30
        assert_within(got[page[live], slot[live]], ref[live], tol[live], sc[0])
        touched = torch.zeros(got.shape[:2], dtype=torch.bool)
        touched[page[live], slot[live]] = True
        assert torch.equal(got[~touched], was[~touched])


def test_append_leaves_out_what_lies_outside(gpu):
    """Rows and positions outside the table and pages outside the cache: left out and counted, the
    queries rotated all the same."""
    from torch_helion.hip import ops

    announce("append out of range")
    hk, d, ps = 2, 64, 16
    kc, vc, table = paged(3, 2, ps, hk, d, BF16, gen(0), gpu)
    table[1, 0], table[1, 1] = -1, kc.shape[0]
    kc0, vc0 = kc.clone(), vc.clone()
    rows = torch.tensor([0, 1, 1, 3, -1, 2, 0], dtype=torch.int32, device=gpu)
    pos = torch.tensor([3, 0, 16, 0, 0, 32, -5], dtype=torch.int32, device=gpu)
    k = torch.randn(7, hk * d, generator=gen(1)).to(BF16).to(gpu)
    q_out = torch.zeros_like(k)
    bad = torch.zeros(1, dtype=torch.int32, device=gpu)
    f = ops.rope_frequencies(d, 10000.0, device=gpu)
    ops.paged_append(k, k, pos, kc, vc, table, rows=rows, freqs=f, q=k, q_out=q_out, n_invalid=bad)
    torch.cuda.synchronize()
    assert bad.item() == 5
    page = int(table[0, 0])
    assert torch.equal(vc[page, 3].reshape(-1), k[0])
    for got, was in ((kc, kc0), (vc, vc0)):
        got = got.clone()
        got[page, 3] = was[page, 3]
        assert torch.equal(got, was)
    ref, mag = rope64(k.view(7, hk, d).cpu(), pos.cpu(), f.cpu())
    assert_within(q_out.view(7, hk, d)[:6], ref[:6], (ROT * mag + u(BF16) * ref.abs())[:6] + 1e-30)
    assert (q_out[6] == 0).all()


@pytest.mark.parametrize("dtype,cache", [(BF16, E4M3), (torch.float32, BF16)])
def test_large_calls_equal_their_halves(gpu, dtype, cache):
    """Calls past 128 MB go past the caches: the same bits as two calls of half the tokens each, which do not."""
    from torch_helion.hip import ops

    announce(f"large rope and append {dtype} -> {cache}")
    t, hq, hk, d, ps = 6000 if dtype == torch.float32 else 9000, 24, 8, 128, 64
    g = torch.Generator(device=gpu).manual_seed(4)
    qkv = torch.randn(t, (hq + 2 * hk) * d, generator=g, device=gpu).to(dtype)
    q, k, v = qkv.split([hq * d, hk * d, hk * d], 1)
    f = ops.rope_frequencies(96, 10000.0, device=gpu)
    pos, rows = torch.arange(t, dtype=torch.int32, device=gpu), torch.zeros(t, dtype=torch.int32, device=gpu)
    pages = -(-t // ps)
    table = torch.randperm(pages, generator=g, device=gpu).view(1, pages).to(torch.int32)
    results = []
    for parts in (1, 2):
        caches = [torch.zeros(pages, ps, hk, d, device=gpu).to(cache) for _ in range(2)]
        q_out = torch.zeros(t, hq * d, dtype=BF16, device=gpu)
        turned = torch.zeros_like(qkv)
        for s in torch.arange(t, device=gpu).tensor_split(parts):
            a, b = int(s[0]), int(s[-1]) + 1
            ops.paged_append(k[a:b], v[a:b], pos[a:b], *caches, table, rows=rows[a:b], freqs=f, q=q[a:b], q_out=q_out[a:b])
            ops.rope(qkv[a:b], pos[a:b], f, turned[a:b], head_dim=d)
        results.append((*caches, q_out, turned))
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_special_values(gpu):
    """An e4m3 cache saturates, infinities too, and keeps NaN."""
    from torch_helion.hip import ops

    announce("append special values")
    x = torch.zeros(1, 64, device=gpu)
    x[0, :5] = torch.tensor([1e9, -1e9, float("inf"), float("-inf"), float("nan")])
    kc = torch.zeros(1, 16, 1, 64, device=gpu).to(E4M3)
    vc = torch.zeros_like(kc)
    ops.paged_append(x, x, torch.zeros(1, dtype=torch.int32, device=gpu), kc, vc,
                     torch.zeros(1, 1, dtype=torch.int32, device=gpu))
    for c in (kc, vc):
        got = c[0, 0, 0].float().cpu()
        assert got[:4].tolist() == [448.0, -448.0, 448.0, -448.0] and torch.isnan(got[4]) and (got[5:] == 0).all()


# ------------------------------------------------------------------ attention
def attention64(q, kc, vc, table, pos, rows, scale, window=0, softcap=0.0, slopes=None, ks=None, vs=None):
    """(o, A = sum p |v|, score error bound) [t, h, d]; everything float64 on the CPU, one token at a time."""
    t, h, d = q.shape
    pages, ps, hk, _ = kc.shape
    o, mag, err = torch.zeros(t, h, d, dtype=torch.float64), torch.zeros(t, h, d, dtype=torch.float64), torch.zeros(t, h, 1, dtype=torch.float64)
    cap = table.shape[1] * ps
    for i in range(t):
        r, p = (i if rows is None else int(rows[i])), int(pos[i])
        if not 0 <= r < table.shape[0]:
            continue
        j = torch.arange(max(0, p + 1 - window) if window else 0, max(min(p + 1, cap), 0))
        pg = table[r].long()[j // ps]
        j, pg = j[(pg >= 0) & (pg < pages)], pg[(pg >= 0) & (pg < pages)]
        if not j.numel():
            continue
        for m in range(h):
            kv = m * hk // h
            keys = kc[pg, j % ps, kv].double() * (1.0 if ks is None else ks[kv].double())
            vals = vc[pg, j % ps, kv].double() * (1.0 if vs is None else vs[kv].double())
            s = keys @ q[i, m].double() * scale
            err[i, m] = d * 2.0 ** -22 * scale * (keys.abs() @ q[i, m].double().abs()).max() + 2.0 ** -20 * (1 + softcap)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if slopes is not None:
                s = s - slopes[m].double() * (p - j).double()
            w = torch.softmax(s, 0)
            o[i, m], mag[i, m] = w @ vals, w @ vals.abs()
    return o, mag, err


def check_attention(gpu, lens, hq, hk, d, ps, *, cache=BF16, rows=None, window=0, softcap=0.0, slopes=False, seed=0,
                    head_major=False, poison=True, amplitude=1.0, row_pages=0):
    from torch_helion.hip import ops

    g = gen(seed + 17 * d + ps)
    t, n_rows = len(lens), (len(lens) if rows is None else max(rows) + 1)
    width = max(1, -(-max(lens) // ps), row_pages)
    kc, vc, table = paged(n_rows, width, ps, hk, d, cache, g, gpu, head_major=head_major)
    pos = torch.tensor(lens, dtype=torch.int32) - 1
    rt = None if rows is None else torch.tensor(rows, dtype=torch.int32)
    if poison:  # unused slots and pages hold NaN, unused table entries lie outside
        seen = torch.zeros(kc.shape[:2], dtype=torch.bool)
        tab = table.cpu()
        for i, n in enumerate(lens):
            j = torch.arange(max(0, n - window) if window else 0, max(n, 0))
            seen[tab[i if rows is None else rows[i]].long()[j // ps], j % ps] = True
        for c in (kc, vc):
            c.copy_(torch.where(seen.to(gpu)[:, :, None, None], c.float(), float("nan")).to(c.dtype))
        page_seen = seen.any(1)
        table = torch.where(page_seen[tab.long()], tab, torch.full_like(tab, 1 << 30)).to(gpu)
    q = (torch.randn(t, hq * d, generator=g) * amplitude).to(BF16)
    sl = torch.rand(hq, generator=g) * 0.2 if slopes else None
    sc = {n: (torch.rand(hk, generator=g) + 0.5) for n in ("k_scale", "v_scale")} if cache == E4M3 else {}
    out = torch.full((t, hq * d), float("nan"), dtype=BF16, device=gpu)
    scale = d ** -0.5
    ops.paged_attention(q.to(gpu), kc, vc, table, pos.to(gpu), out, scale=scale, rows=None if rt is None else rt.to(gpu),
                        window=window, softcap=softcap, slopes=None if sl is None else sl.to(gpu),
                        **{n: x.to(gpu) for n, x in sc.items()})
    torch.cuda.synchronize()
    ref, mag, err = attention64(q.view(t, hq, d), kc.float().cpu(), vc.float().cpu(), table.cpu(), pos, rt, scale, window,
                                softcap, sl, sc.get("k_scale"), sc.get("v_scale"))
    assert_within(out.view(t, hq, d), ref, u(BF16) * (ref.abs() + mag) * (1 + 2 * u(BF16)) + 2 * err * mag + 1e-30)
    for i, n in enumerate(lens):
        if n <= 0:
            assert (out[i] == 0).all()


@pytest.mark.parametrize("lens,hq,hk,d,ps", [
    ([1], 4, 1, 128, 16), ([0], 8, 2, 64, 16), ([300], 32, 8, 128, 16), ([1, 2, 15, 16, 17, 31, 32, 33, 0, 127, 128, 129], 8, 2, 128, 16),
    ([63, 64, 65, 255, 256, 257, 1000, 3], 12, 12, 64, 32), ([2049, 5, 700], 16, 1, 128, 256), ([511, 513], 6, 2, 64, 64),
    ([5000], 8, 1, 64, 16), ([77] * 40, 4, 4, 128, 32), ([900, 1, 0, 450], 48, 2, 128, 64), ([333, 40], 64, 1, 64, 16),
    ([20000, 3, 1000], 8, 2, 128, 128),
])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_attention(gpu, lens, hq, hk, d, ps, cache):
    announce(f"paged attention lens={lens[:12]} hq={hq} hk={hk} d={d} ps={ps} {cache}")
    check_attention(gpu, lens, hq, hk, d, ps, cache=cache)


@pytest.mark.parametrize("window,softcap,slopes,cache", [
    (1, 0.0, False, BF16), (16, 0.0, False, BF16), (100, 0.0, False, E4M3), (0, 20.0, False, BF16), (0, 0.0, True, BF16),
    (257, 5.0, True, E4M3), (4096, 30.0, True, BF16),
])
def test_attention_window_cap_and_bias(gpu, window, softcap, slopes, cache):
    announce(f"paged attention window={window} softcap={softcap} slopes={slopes} {cache}")
    check_attention(gpu, [1, 99, 100, 101, 640, 0, 2000], 12, 4, 64, 32, window=window, softcap=softcap, slopes=slopes,
                    cache=cache, amplitude=6.0)
    check_attention(gpu, [31, 1500], 4, 4, 128, 16, window=window, softcap=softcap, slopes=slopes, cache=cache, amplitude=6.0)


@pytest.mark.parametrize("window,softcap,slopes,cache", [(1500, 0.0, False, BF16), (2100, 10.0, True, E4M3), (1030, 0.0, True, BF16)])
def test_attention_long_windows(gpu, window, softcap, slopes, cache):
    """Windows of more tiles than the pair form takes, ahead of, at and past the lengths' ends."""
    announce(f"paged attention long window={window} {cache}")
    check_attention(gpu, [window - 1, 3000, window, window + 1, 0, window + 16, 2999], 4, 2, 64, 16, window=window, softcap=softcap,
                    slopes=slopes, cache=cache, amplitude=4.0)


def test_attention_rows_and_head_major_pages(gpu):
    """Several tokens of one row (a speculated run), rows in any order, pages laid out head by head."""
    announce("paged attention with rows")
    check_attention(gpu, [500, 501, 502, 503, 20, 64, 65], 8, 2, 128, 32, rows=[2, 2, 2, 2, 0, 1, 1], head_major=True)
    check_attention(gpu, [40, 41, 900], 4, 4, 64, 16, rows=[1, 1, 0], head_major=True, cache=E4M3)


def test_attention_cap_far_above_the_scores(gpu):
    """The largest cap leaves scores of a few units nearly as they are; the bound's 2^-20 softcap is then 1e-3."""
    from torch_helion.hip import ops

    announce("paged attention, a cap far above the scores")
    kc, vc, table = paged(2, 40, 16, 2, 64, BF16, gen(12), gpu)
    q = (torch.randn(2, 4 * 64, generator=gen(13)) * 2).to(BF16)
    pos = torch.tensor([630, 99], dtype=torch.int32)
    out = torch.empty_like(q, device=gpu)
    ops.paged_attention(q.to(gpu), kc, vc, table, pos.to(gpu), out, scale=0.125, softcap=1024.0)
    ref, mag, err = attention64(q.view(2, 4, 64), kc.float().cpu(), vc.float().cpu(), table.cpu(), pos, None, 0.125, softcap=1024.0)
    assert_within(out.view(2, 4, 64), ref, u(BF16) * (ref.abs() + mag) * (1 + 2 * u(BF16)) + 2 * err * mag)


@pytest.mark.parametrize("row_pages", [20, 200])
def test_attention_onto_its_queries(gpu, row_pages):
    """out may be q, in both forms."""
    from torch_helion.hip import ops

    announce(f"paged attention onto its queries, rows of {row_pages} pages")
    kc, vc, table = paged(9, row_pages, 16, 4, 64, BF16, gen(14), gpu)
    q = torch.randn(9, 12 * 64, generator=gen(15)).to(BF16).to(gpu)
    pos = torch.tensor([0, 319, 5, -1, 100, 250, 16, 31, 200], dtype=torch.int32, device=gpu)
    out = torch.empty_like(q)
    ops.paged_attention(q, kc, vc, table, pos, out, scale=0.125)
    ops.paged_attention(q, kc, vc, table, pos, q, scale=0.125)
    assert torch.equal(q, out)


def test_attention_outside_the_table(gpu):
    """A position past the table sees the table's keys; a row outside it sees none; pages outside the cache
    are left out, also where that leaves nothing."""
    from torch_helion.hip import ops

    announce("paged attention out of range")
    hq, hk, d, ps = 4, 2, 64, 16
    kc, vc, table = paged(4, 3, ps, hk, d, BF16, gen(5), gpu)
    table[1, 1], table[2] = -1, kc.shape[0]
    rows = torch.tensor([0, 1, 2, 4, -1, 3], dtype=torch.int32)
    pos = torch.tensor([1000, 40, 40, 5, 5, -3], dtype=torch.int32)
    q = torch.randn(6, hq * d, generator=gen(6)).to(BF16)
    out = torch.full((6, hq * d), float("nan"), dtype=BF16, device=gpu)
    ops.paged_attention(q.to(gpu), kc, vc, table, pos.to(gpu), out, scale=0.125, rows=rows.to(gpu))
    ref, mag, err = attention64(q.view(6, hq, d), kc.float().cpu(), vc.float().cpu(), table.cpu(), pos, rows, 0.125)
    assert_within(out.view(6, hq, d), ref, u(BF16) * (ref.abs() + mag) * (1 + 2 * u(BF16)) + 2 * err * mag + 1e-30)
    assert (out[2:] == 0).all() and (out[:2] != 0).any(1).all()
    # a bias by distance far past the table: the distances' differences are what counts
    far = torch.full((1,), 2147483647, dtype=torch.int32)
    slopes = torch.full((hq,), 0.25)
    ops.paged_attention(q[:1].to(gpu), kc, vc, table, far.to(gpu), out[:1], scale=0.125, slopes=slopes.to(gpu))
    ref, mag, err = attention64(q[:1].view(1, hq, d), kc.float().cpu(), vc.float().cpu(), table.cpu(), far, None, 0.125, slopes=slopes)
    assert_within(out[:1].view(1, hq, d), ref, u(BF16) * (ref.abs() + mag) * (1 + 2 * u(BF16)) + 2 * err * mag + 1e-30)


@pytest.mark.parametrize("lens,hq,hk,d,ps,cache", [
    ([1], 32, 8, 128, 16, BF16), ([0, 0, 0], 4, 2, 64, 32, BF16), ([301], 32, 8, 128, 16, E4M3), ([1, 0, 17, 640, 0], 12, 4, 64, 64, E4M3),
    ([5] * 300, 3, 1, 64, 16, BF16), ([1000, 31, 33] * 30, 16, 16, 128, 32, BF16), ([700, 650], 40, 2, 128, 16, BF16)])
def test_attention_short_rows_in_long_tables(gpu, lens, hq, hk, d, ps, cache):
    """Tables with room for 8192 keys take the line form whatever the lengths: fewer tiles than waves, tokens
    without keys first, last and between, more tokens than a workgroup has threads' runs of one."""
    announce(f"paged attention, long tables, lens={lens[:6]} hq={hq} hk={hk} d={d} ps={ps} {cache}")
    check_attention(gpu, lens, hq, hk, d, ps, cache=cache, row_pages=8192 // ps, poison=len(lens) < 100)


@pytest.mark.parametrize("tokens,hq,hk,d,room,cache", [
    (70, 16, 8, 128, 64, BF16),      # 560 pairs of two tiles: two waves
    (150, 8, 8, 64, 64, BF16),       # 1200 pairs of one tile: one wave
    (139, 16, 8, 128, 128, BF16),    # 1112 pairs of four tiles: one wave, four tiles in turn
    (21, 6, 3, 64, 512, E4M3),       # 64-byte rows: an XCD takes a token, the last five in order
    (300, 4, 4, 64, 128, E4M3),
    (275, 8, 8, 64, 1024, BF16),     # from 512 MB of room on: 2200 pairs of 16 tiles
    (260, 32, 16, 128, 256, E4M3),   # 4160 pairs of 4 tiles past the caches
    (1100, 8, 8, 64, 512, E4M3),     # 8800 pairs of 4 tiles: one wave, tokens to the XCDs in turn
])
def test_attention_many_pairs(gpu, tokens, hq, hk, d, room, cache):
    """Every number of waves a pair can get and both orders of the pairs; few pages hold the keys of all."""
    announce(f"paged attention, {tokens} tokens of {hk} kv heads d={d} room={room} {cache}")
    rows = [i % 7 for i in range(tokens)]
    lens = [1 + (37 * i) % room for i in range(tokens)]
    check_attention(gpu, lens, hq, hk, d, 16, rows=rows, cache=cache, row_pages=room // 16, poison=False, seed=tokens)


def test_attention_many_tokens_of_one_row(gpu):
    """700 tokens of one row (a prompt's tail): several tokens to each run of the line's prefix sums."""
    announce("paged attention, 700 tokens of a row")
    check_attention(gpu, list(range(200, 900)), 2, 1, 64, 64, rows=[0] * 700, row_pages=32)


def test_attention_extreme_scores(gpu):
    """Scores of +-1e4 and a NaN query: the first come out as the formula's, the second as NaN in its row alone."""
    from torch_helion.hip import ops

    announce("paged attention extreme scores")
    check_attention(gpu, [700, 3], 4, 2, 64, 16, amplitude=3000.0)
    kc, vc, table = paged(2, 3, 16, 1, 64, BF16, gen(8), gpu)
    q = torch.randn(2, 64, generator=gen(9)).to(BF16).to(gpu)
    q[0, 5] = float("nan")
    out = torch.empty_like(q)
    ops.paged_attention(q, kc, vc, table, torch.tensor([40, 40], dtype=torch.int32, device=gpu), out, scale=0.125)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()


def test_attention_offsets_past_32_bits(gpu):
    """A pool of more than 2^31 elements (4.3 GB per tensor), the pages at its end."""
    from torch_helion.hip import ops

    announce("paged attention and append past 2^32 bytes")
    ps, hk, d, pages = 256, 8, 128, 8300
    kc = torch.zeros(pages, ps, hk, d, dtype=BF16, device=gpu)
    vc = torch.zeros_like(kc)
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device=gpu)
    n = 600
    k, v = (torch.randn(n, hk * d, generator=gen(i)).to(BF16) for i in (1, 2))
    q = torch.randn(1, 32 * d, generator=gen(3)).to(BF16)
    pos = torch.arange(n, dtype=torch.int32, device=gpu)
    ops.paged_append(k.to(gpu), v.to(gpu), pos, kc, vc, table, rows=torch.zeros(n, dtype=torch.int32, device=gpu))
    out = torch.empty(1, 32 * d, dtype=BF16, device=gpu)
    ops.paged_attention(q.to(gpu), kc, vc, table, pos[-1:].contiguous(), out, scale=d ** -0.5)
    assert torch.equal(kc[pages - 1].reshape(ps, -1).cpu(), k[:ps]) and torch.equal(vc[pages - 3, :n - 2 * ps].reshape(-1, hk * d).cpu(), v[2 * ps:])
    small = [x.view(1, n, hk, d) for x in (k, v)]
    ref, mag, err = attention64(q.view(1, 32, d), torch.nn.functional.pad(small[0].float(), (0, 0, 0, 0, 0, 1024 - n)),
                                torch.nn.functional.pad(small[1].float(), (0, 0, 0, 0, 0, 1024 - n)),
                                torch.zeros(1, 1, dtype=torch.int32), torch.tensor([n - 1]), None, d ** -0.5)
    assert_within(out.view(1, 32, d), ref, u(BF16) * (ref.abs() + mag) * (1 + 2 * u(BF16)) + 2 * err * mag + 1e-30)
    ops.copy_pages(kc, vc, torch.tensor([pages - 1], dtype=torch.int32, device=gpu), torch.tensor([pages - 2], dtype=torch.int32, device=gpu))
    assert torch.equal(kc[pages - 2], kc[pages - 1]) and torch.equal(vc[pages - 2], vc[pages - 1])


# ------------------------------------------------------------------ page copies
@pytest.mark.parametrize("layers,pages,n,ps,hk,d,dtype", [
    (1, 4, 1, 16, 1, 64, BF16), (3, 40, 13, 16, 8, 128, BF16), (2, 9, 4, 1, 3, 16, E4M3), (5, 30, 10, 64, 5, 128, E4M3),
    (None, 12, 5, 32, 2, 64, BF16), (2, 7, 0, 16, 1, 64, BF16),
])
def test_copy_pages(gpu, layers, pages, n, ps, hk, d, dtype):
    from torch_helion.hip import ops

    announce(f"copy pages layers={layers} pages={pages} n={n} ps={ps} hk={hk} d={d} {dtype}")
    g = gen(pages + n)
    shape = (() if layers is None else (layers,)) + (pages, ps, hk, d)
    kc, vc = (torch.randn(shape, generator=g).to(dtype).to(gpu) for _ in range(2))
    order = torch.randperm(pages, generator=g).to(torch.int32)
    src, dst = order[:n].contiguous(), order[n:2 * n].contiguous()
    table = torch.randint(-2, pages + 3, (6, 5), generator=g, dtype=torch.int32)
    wide = torch.full((6, 9), 123456, dtype=torch.int32)
    wide[:, :5] = table
    wide = wide.to(gpu)
    page_map = torch.arange(pages, dtype=torch.int32)
    page_map[src.long()] = dst
    ref = []
    for c in (kc, vc):
        r = c.view(torch.uint8).clone()
        r5 = r if layers is not None else r[None]
        r5[:, dst.long().to(gpu)] = r5[:, src.long().to(gpu)]
        ref.append(r)
    ops.copy_pages(kc, vc, src.to(gpu), dst.to(gpu), page_table=wide[:, :5], page_map=page_map.to(gpu))
    torch.cuda.synchronize()
    for c, r in zip((kc, vc), ref):
        assert torch.equal(c.view(torch.uint8), r)
    named = torch.tensor([[int(page_map[p]) if 0 <= p < pages else p for p in row] for row in table.tolist()], dtype=torch.int32)
    assert torch.equal(wide[:, :5].cpu(), named) and (wide[:, 5:] == 123456).all()


def test_copy_pages_of_more_workgroups_than_one_dimension_holds(gpu):
    """2^22 + 3 pages of 16 bytes in one layer's two caches: past 2^23 workgroups, and a table renamed behind them."""
    from torch_helion.hip import ops

    announce("copy of 2^22 + 3 pages")
    n = (1 << 22) + 3
    caches = [torch.randint(0, 1 << 14, (2 * n, 1, 1, 8), dtype=torch.int16, device=gpu).view(torch.bfloat16) for _ in range(2)]
    order = torch.randperm(n, device=gpu)
    src, dst = order.to(torch.int32), torch.arange(n, 2 * n, dtype=torch.int32, device=gpu)
    table = torch.arange(2 * n, dtype=torch.int32, device=gpu).view(2, n)
    ops.copy_pages(*caches, src, dst, page_table=table, page_map=torch.arange(2 * n, dtype=torch.int32, device=gpu).flip(0).contiguous())
    for c in caches:
        raw = c.view(torch.int16)
        assert torch.equal(raw[n:], raw[:n][order])
    assert torch.equal(table.flatten(), torch.arange(2 * n, dtype=torch.int32, device=gpu).flip(0))


def test_copy_pages_skips_what_lies_outside(gpu):
    from torch_helion.hip import ops

    announce("copy pages out of range")
    kc = torch.randn(2, 6, 16, 2, 64, generator=gen(0)).to(BF16).to(gpu)
    vc = torch.randn(2, 6, 16, 2, 64, generator=gen(1)).to(BF16).to(gpu)
    k0, v0 = kc.clone(), vc.clone()
    src = torch.tensor([-1, 6, 0, 2, 3], dtype=torch.int32, device=gpu)
    dst = torch.tensor([1, 1, 6, 2, 5], dtype=torch.int32, device=gpu)
    ops.copy_pages(kc, vc, src, dst)
    k0[:, 5], v0[:, 5] = k0[:, 3], v0[:, 3]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)


# ------------------------------------------------------------------ together, captured
@pytest.mark.parametrize("row_pages", [8, 40])
def test_append_and_attention_in_a_graph(gpu, row_pages):
    """A decode step captured once and replayed with new positions, tokens and page tables, other work
    between the replays: each replay gives the eager calls' bits."""
    from torch_helion.hip import ops

    announce(f"paged step in a graph, rows of {row_pages} pages")
    n, hq, hk, d, ps = 5, 8, 2, 128, 16
    g = gen(11)
    kc, vc, table = paged(n, row_pages, ps, hk, d, BF16, g, gpu)
    k2, v2 = kc.clone(), vc.clone()
    f = ops.rope_frequencies(d, 10000.0, device=gpu)
    qkv = torch.zeros(n, (hq + 2 * hk) * d, device=gpu)
    pos = torch.zeros(n, dtype=torch.int32, device=gpu)
    q_out = torch.zeros(n, hq * d, dtype=BF16, device=gpu)
    out, q2, out2 = torch.zeros_like(q_out), torch.zeros_like(q_out), torch.zeros_like(q_out)
    ws = torch.empty(max(ops.paged_attention_workspace_bytes(n, hq, hk, d, row_pages * ps), 16), dtype=torch.uint8, device=gpu)

    def step(kc, vc, q_out, out, ws):
        q, k, v = qkv.split([hq * d, hk * d, hk * d], 1)
        ops.paged_append(k, v, pos, kc, vc, table, freqs=f, q=q, q_out=q_out)
        ops.paged_attention(q_out, kc, vc, table, pos, out, scale=d ** -0.5, workspace=ws)

    step(kc, vc, q_out, out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(kc, vc, q_out, out, ws)
    kc.copy_(k2)
    vc.copy_(v2)
    for i in range(4):
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        pos.copy_(torch.tensor([3 + i, 127, -1, 31 + i, 60 + 16 * i], dtype=torch.int32))
        table[0], table[1] = table[1].clone(), table[0].clone()
        graph.replay()
        ws.fill_(255)                                 # the workspace holds nothing between calls
        step(k2, v2, q2, out2, None)
        torch.cuda.synchronize()
        for a, b in ((kc, k2), (vc, v2), (out, out2)):
            assert torch.equal(a, b)
        live = [0, 1, 3, 4]
        assert torch.equal(q_out[live], q2[live])
