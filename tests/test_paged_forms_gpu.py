"""The accuracy of th_paged_attention's probabilities and of th_paged_append's 8-bit stores.

Bounds are elementwise, against 64 bits, in the terms of tests/test_paged_gpu.py: u(t) is a rounding's
half step, A = sum_j p_j |v_j|, and a score is off by head_dim 2^-22 scale sum_i |q_i k_i| (an fp32 sum
in any order) and 2^-20 softcap; 2^-20 stands for the exponential.
"""

from __future__ import annotations

import pytest
import torch

from conftest import announce
from test_paged_gpu import BF16, E4M3, assert_within, gen, paged, u

pytestmark = pytest.mark.gpu


def attention64(q, kc, vc, table, pos, rows, scale, window=0, softcap=0.0, slopes=None, ks=None, vs=None):
    """(o, A, score error bound) [t, h, d] on the CPU from float64 on the device, a token at a time."""
    t, h, d = q.shape
    pages, ps, hk, _ = kc.shape
    dev, keys = kc.device, table.shape[1] * ps
    one = torch.ones(hk, device=dev)
    o, mag = (torch.zeros(t, h, d, dtype=torch.float64, device=dev) for _ in range(2))
    err = torch.zeros(t, h, 1, dtype=torch.float64, device=dev)
    where, at = pos.tolist(), list(range(t)) if rows is None else rows.tolist()
    for i, (p, r) in enumerate(zip(where, at)):
        if not 0 <= r < table.shape[0]:
            continue
        j = torch.arange(max(0, p + 1 - window) if window else 0, max(min(p + 1, keys), 0), device=dev)
        pg = table[r].long()[j // ps]
        j, pg = j[(pg >= 0) & (pg < pages)], pg[(pg >= 0) & (pg < pages)]
        if not j.numel():
            continue
        k, v = ((c[pg, j % ps].double() * (one if f is None else f).double()[:, None]).transpose(0, 1).contiguous()
                for c, f in ((kc, ks), (vc, vs)))
        mine = q[i].to(dev).double().view(hk, -1, d)
        kt = k.transpose(1, 2).contiguous()
        s = mine @ kt * scale
        err[i] = (d * 2.0 ** -22 * scale * (mine.abs() @ kt.abs()).amax(-1) + 2.0 ** -20 * (1 + softcap)).view(h, 1)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if slopes is not None:
            s = s - slopes.to(dev).double().view(hk, -1, 1) * (p - j).double()
        w = torch.softmax(s, -1)
        o[i], mag[i] = (w @ v).view(h, d), (w @ v.abs()).view(h, d)
    return o.cpu(), mag.cpu(), err.cpu()


def p_step(cache) -> float:
    """What a probability of the second product is off by, relative to it: two bf16 halves over a bf16
    cache (the second one's half step of what the first left over), one fp16 over an e4m3 cache."""
    return u(BF16) ** 2 if cache == BF16 else u(torch.float16)


# ------------------------------------------------------------------ probabilities
@pytest.mark.parametrize("room", [32, 8192])         # the pair and the line form
@pytest.mark.parametrize("hq,hk,d", [(8, 2, 64), (32, 8, 128), (20, 1, 128)])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_probabilities_keep_their_accuracy(gpu, cache, hq, hk, d, room):
    """Values that cancel (each second one is its neighbour's negative) leave the probabilities' own rounding in
    the output: off by p_step of A, not by u(bf16). The fp32 sums of n <= 32 keys are off by n 2^-23."""
    from torch_helion.hip import ops

    announce(f"paged attention, cancelling values, {cache} hq={hq} hk={hk} d={d} room={room}")
    lens = [1, 2, 2, 2, 2, 4, 4, 4, 6, 10, 16, 32] * 4
    g = gen(d + hq + room)
    kc, vc, table = paged(len(lens), room // 16, 16, hk, d, cache, g, gpu)
    vc[:, 1::2] = (-vc[:, 0::2].float()).to(cache)
    q = (torch.randn(len(lens), hq * d, generator=g) * 0.3).to(BF16)
    pos = torch.tensor(lens, dtype=torch.int32) - 1
    out = torch.empty(len(lens), hq * d, dtype=BF16, device=gpu)
    ops.paged_attention(q.to(gpu), kc, vc, table, pos.to(gpu), out, scale=d ** -0.5)
    torch.cuda.synchronize()
    ref, mag, err = attention64(q.view(-1, hq, d), kc, vc, table, pos, None, d ** -0.5)
    tol = u(BF16) * ref.abs() + mag * (1 + u(BF16)) * (2 * err + p_step(cache) + 32 * 2.0 ** -23) + 1e-30
    assert_within(out.view(-1, hq, d), ref, tol)


@pytest.mark.parametrize("room", [8192, 131072])
@pytest.mark.parametrize("cache,top", [(BF16, 18.0), (BF16, 26.0), (E4M3, 18.0), (E4M3, 22.0)])
def test_many_keys_of_little_weight_are_not_lost(gpu, cache, top, room):
    """One key of weight 1 and value 0 over all the others of weight e^-top: their sum is the output. The smallest
    step of an fp16 p is 2^-38 of the largest one's, so off by half of it, 2^-39, a key."""
    from torch_helion.hip import ops

    announce(f"paged attention, {room} keys of weight e^-{top}, {cache}")
    d, ps = 64, 64
    kc = torch.zeros(room // ps, ps, 1, d, device=gpu).to(cache)
    vc = torch.full((room // ps, ps, 1, d), 448.0, device=gpu).to(cache)
    kc[5, 7, 0, 0], vc[5, 7] = top, 0.0
    table = torch.arange(room // ps, dtype=torch.int32, device=gpu)[None]
    q = torch.zeros(1, d)
    q[0, 0] = 1.0
    pos = torch.tensor([room - 1], dtype=torch.int32, device=gpu)
    out = torch.empty(1, d, dtype=BF16, device=gpu)
    ops.paged_attention(q.to(BF16).to(gpu), kc, vc, table, pos, out, scale=1.0)
    ref, mag, err = attention64(q.view(1, 1, d), kc, vc, table, pos, None, 1.0)
    tol = u(BF16) * ref + mag * (1 + u(BF16)) * (2 * err + p_step(cache) + room * 2.0 ** -23)
    if cache == E4M3:
        tol = tol + room * 2.0 ** -39 * 448.0
    assert (tol < 0.05 * ref).all()
    assert_within(out.view(1, 1, d), ref, tol)


# ------------------------------------------------------------------ 8-bit stores
@pytest.mark.parametrize("in_dtype", [BF16, torch.float32])
@pytest.mark.parametrize("head_major", [False, True])   # head-major pages here are not whole pieces: one element a time
def test_append_divides_by_the_scale(gpu, in_dtype, head_major):
    """Halfway between two e4m3 values the quotient x / scale goes to the even one, bit for bit as torch's;
    a product with the rounded reciprocal lands beside the middle."""
    from torch_helion.hip import ops

    announce(f"append, quotients halfway between two e4m3 values, {in_dtype} head_major={head_major}")
    scales = torch.tensor([7.0, 3.0, 0.4375, 1.75, 5.0, 448.0, 1.0, 0.875])
    hk, d = len(scales), 64
    half = torch.cat([(torch.arange(17, 32, 2) / 16) * 2.0 ** e for e in range(-5, 11)])
    half = torch.cat([half, -half]).view(-1, 1, d)                    # four tokens of 64 values
    x = (half * scales[:, None]).to(BF16)                             # exact: five bits by at most three
    ref = (x.float() / scales[:, None]).clamp(-448, 448).to(E4M3)
    assert ((x.float() * (1 / scales[:, None])).clamp(-448, 448).to(E4M3).view(torch.uint8) != ref.view(torch.uint8)).sum() > 30
    n = x.shape[0]
    shape = (2, hk, 16, d + 3) if head_major else (2, 16, hk, d)
    caches = [torch.zeros(shape, device=gpu).to(E4M3)[..., :d] for _ in range(2)]
    if head_major:
        caches = [c.transpose(1, 2) for c in caches]
    rows = x.to(in_dtype).reshape(n, hk * d).to(gpu)
    ops.paged_append(rows, rows, torch.arange(n, dtype=torch.int32, device=gpu), *caches,
                     torch.tensor([[1]], dtype=torch.int32, device=gpu), rows=torch.zeros(n, dtype=torch.int32, device=gpu),
                     k_scale=scales.to(gpu), v_scale=scales.to(gpu))
    for c in caches:
        assert torch.equal(c[1, :n].contiguous().view(torch.uint8).cpu(), ref.view(torch.uint8))
