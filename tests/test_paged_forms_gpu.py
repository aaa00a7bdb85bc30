"""The paged entry points in the forms that their cases take: the accuracy of the attention's probabilities
and of the 8-bit stores, batches over which the attention's waves take several tiles and tokens each, the
inverse rotation by whole pieces, and the options of the cache and the block.

Bounds are elementwise, against 64 bits, in the terms of tests/test_paged_gpu.py: u(t) is a rounding's
half step, A = sum_j p_j |v_j|, and a score is off by head_dim 2^-22 scale sum_i |q_i k_i| (an fp32 sum
in any order), 2^-20 softcap and, with a bias, 2^-21 of the largest one (three roundings of it); 2^-20
stands for the exponential. The fp32 sums over n keys are off by n 2^-23 of A.
"""

from __future__ import annotations

import pytest
import torch

from conftest import announce
from test_paged_gpu import BF16, E4M3, ROT, assert_within, gen, paged, rope64, u

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
            err[i] += 2.0 ** -21 * slopes.to(dev).double().abs().view(h, 1) * (j[-1] - j[0] + 128)
            s = s - slopes.to(dev).double().view(hk, -1, 1) * (p - j).double()
        w = torch.softmax(s, -1)
        o[i], mag[i] = (w @ v).view(h, d), (w @ v.abs()).view(h, d)
    return o.cpu(), mag.cpu(), err.cpu()


def p_step(cache) -> float:
    """What a probability of the second product is off by, relative to it: two bf16 halves over a bf16
    cache (the second one's half step of what the first left over, at most 2^-7: it is taken 2^-8 below p
    and rounded), one fp16 over an e4m3 cache."""
    return u(BF16) * 2.0 ** -7 if cache == BF16 else u(torch.float16)


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


@pytest.mark.parametrize("room", [64, 8192])
@pytest.mark.parametrize("n,amplitude", [(1, 1.0), (2, 0.0), (60, 0.0), (60, 1.0), (33, 4.0)])
def test_infinite_values_stay_infinite(gpu, n, amplitude, room):
    """An infinity among the values a token sees is its output there, of its sign; the other dims are finite. Weights
    of one key alone, of equal keys (powers of two, whose second half is none) and of any."""
    from torch_helion.hip import ops

    announce(f"paged attention, infinite values, {n} keys room={room} amplitude={amplitude}")
    d = 64
    kc, vc, table = paged(1, room // 16, 16, 2, d, BF16, gen(n), gpu)
    page = int(table[0, (n - 1) // 16])
    vc[page, (n - 1) % 16, :, 3], vc[page, (n - 1) % 16, :, 40] = float("inf"), float("-inf")
    q = (torch.randn(1, 8 * d, generator=gen(5)) * amplitude).to(BF16).to(gpu)
    out = torch.empty_like(q)
    ops.paged_attention(q, kc, vc, table, torch.tensor([n - 1], dtype=torch.int32, device=gpu), out, scale=d ** -0.5)
    out = out.view(8, d).float().cpu()
    assert (out[:, 3] == float("inf")).all() and (out[:, 40] == float("-inf")).all()
    out[:, 3] = out[:, 40] = 0.0
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("room", [64, 8192])
@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("top", [2.0 ** e for e in (20, 24, 25, 26, 27, 28, 29, 40, 100)])
def test_scores_whose_steps_are_large(gpu, cache, top, room):
    """The largest score at top and at 1.5 top, the others a few steps of an fp32 of that size below it or far
    away: an exact score (one product of powers of two) leaves weight 1, split evenly, on the keys that have it."""
    from torch_helion.hip import ops

    announce(f"paged attention, scores of {top}, {cache} room={room}")
    d, ps, n = 64, 16, 60
    kc = torch.zeros(room // ps, ps, 2, d, device=gpu)
    at = torch.tensor([1.0, -1.0, 0.5, 0.0, 0.875, 1.0])
    for j in range(n):
        kc[j // ps, j % ps, :, 0] = at[j % 6]
    vc = torch.randn(room // ps, ps, 2, d, generator=gen(int(top) % 97)).to(gpu).to(cache)
    kc = kc.to(cache)
    table = torch.arange(room // ps, dtype=torch.int32, device=gpu)[None]
    q = torch.zeros(1, 4, d)
    q[0, :, 0] = torch.tensor([top, 1.5 * top, -top, -1.5 * top])
    pos = torch.tensor([n - 1], dtype=torch.int32, device=gpu)
    out = torch.empty(1, 4 * d, dtype=BF16, device=gpu)
    ops.paged_attention(q.view(1, -1).to(BF16).to(gpu), kc, vc, table, pos, out, scale=1.0)
    torch.cuda.synchronize()
    best = [[j for j in range(n) if at[j % 6] == (1.0 if h < 2 else -1.0)] for h in range(4)]
    ref = torch.stack([torch.stack([vc[j // ps, j % ps, h // 2].double().cpu() for j in js]).mean(0) for h, js in enumerate(best)])
    mag = torch.stack([torch.stack([vc[j // ps, j % ps, h // 2].double().cpu().abs() for j in js]).mean(0) for h, js in enumerate(best)])
    assert_within(out.view(4, d), ref, u(BF16) * ref.abs() + mag * (1 + u(BF16)) * n * 2.0 ** -23 + 1e-30)


# ------------------------------------------------------------------ the line form
def tiles_and_groups(gpu, lens, hq, hk, d, cache, window=0):
    """(tiles of all tokens, groups of waves that they are dealt out to, keys of a tile) of the line form."""
    keys = 8192 // (d * torch.empty(0, dtype=cache).element_size())
    blocks = hk * -(-(hq // hk) // 16)
    first = [max(0, n - window) // 16 * 16 if window else 0 for n in lens]
    cus = torch.cuda.get_device_properties(gpu).multi_processor_count
    return sum(-(-(n - a) // keys) for n, a in zip(lens, first) if n > 0), cus * 8 // blocks, keys


def check_line(gpu, lens, hq, hk, d, cache, *, room, rows=None, window=0, softcap=0.0, slopes=False, amplitude=1.0, least=2.0, seed=0,
               ps=16):
    """A call in the line form with at least ``least`` tiles for each group of waves, against 64 bits; NaN in every
    slot that no token sees and in the workspace; a second call gives the same bits."""
    from torch_helion.hip import ops

    tiles, groups, _ = tiles_and_groups(gpu, lens, hq, hk, d, cache, window)
    assert tiles >= least * groups, (tiles, groups)
    g = gen(seed + 31 * d + hq)
    t, n_rows = len(lens), (len(lens) if rows is None else max(rows) + 1)
    kc, vc, table = paged(n_rows, room // ps, ps, hk, d, cache, g, gpu)
    pos = torch.tensor(lens, dtype=torch.int32) - 1
    rt = None if rows is None else torch.tensor(rows, dtype=torch.int32)
    seen = torch.zeros(kc.shape[:2], dtype=torch.bool, device=gpu)
    for i, n in enumerate(lens):
        j = torch.arange(max(0, n - window) if window else 0, max(n, 0), device=gpu)
        seen[table[i if rows is None else rows[i]].long()[j // ps], j % ps] = True
    for c in (kc, vc):
        c.copy_(torch.where(seen[:, :, None, None], c.float(), float("nan")).to(cache))
    table = torch.where(seen.any(1)[table.long()], table, torch.full_like(table, -1))
    q = (torch.randn(t, hq * d, generator=g) * amplitude).to(BF16)
    sl = torch.rand(hq, generator=g) * 0.1 if slopes else None
    sc = {n: (torch.rand(hk, generator=g) + 0.5).to(gpu) for n in ("k_scale", "v_scale")} if cache == E4M3 else {}
    size = ops.paged_attention_workspace_bytes(t, hq, hk, d, room, window=window, dtype=cache, device=gpu)
    assert size > 0                                                  # the line form: the pair form needs none
    outs = []
    for _ in range(2):
        out = torch.full((t, hq * d), float("nan"), dtype=BF16, device=gpu)
        ops.paged_attention(q.to(gpu), kc, vc, table, pos.to(gpu), out, scale=d ** -0.5, rows=None if rt is None else rt.to(gpu),
                            window=window, softcap=softcap, slopes=None if sl is None else sl.to(gpu),
                            workspace=torch.full((size,), 255, dtype=torch.uint8, device=gpu), **sc)
        outs.append(out)
    torch.cuda.synchronize()
    assert torch.equal(*outs)
    ref, mag, err = attention64(q.view(t, hq, d), kc, vc, table, pos, rt, d ** -0.5, window, softcap, sl, sc.get("k_scale"), sc.get("v_scale"))
    most = max(lens)
    tol = u(BF16) * ref.abs() + mag * (1 + u(BF16)) * (2 * err + p_step(cache) + most * 2.0 ** -23) + 1e-30
    if cache == E4M3:
        tol = tol + most * 2.0 ** -39 * 448.0
    assert_within(outs[0].view(t, hq, d), ref, tol)
    empty = [i for i, n in enumerate(lens) if n <= 0]
    assert (outs[0][empty] == 0).all()


@pytest.mark.parametrize("group", [1, 3, 4, 8, 16, 20])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_line_of_cut_tokens(gpu, cache, d, group):
    """320 pairs of ragged lengths over 64 groups: waves go from token to token, past empty ones, and the parts of
    cut tokens are joined by workgroups of several heads (8 heads of 128 dims at most, a second block of 4 heads at
    group 20, rows that no head takes at group 3)."""
    announce(f"paged attention, cut tokens, {cache} d={d} group={group}")
    keys = tiles_and_groups(gpu, [], 1, 1, d, cache)[2]
    lens = [0, int(40.3 * keys), 1, int(30.9 * keys), 0, int(60.5 * keys), 17 * keys, 33 * keys + 1, 25 * keys - 1, 0]
    check_line(gpu, lens, 32 * group, 32, d, cache, room=64 * keys, least=3)


@pytest.mark.parametrize("lens,hq,hk,d,cache,room", [
    ([100003, 17], 8, 2, 128, BF16, 100016),               # few heads: the join by 32 dims
    ([70001], 4, 1, 64, E4M3, 70016), ([0, 150000, 0], 3, 1, 64, BF16, 150000),
    ([3000, 2999, 2047, 0, 4000, 2500], 64, 8, 128, BF16, 4096),   # fewer than 256 pairs: a head a workgroup
    ([9000, 5000, 0, 7001], 48, 16, 64, E4M3, 9008),
])
def test_line_of_few_tokens(gpu, lens, hq, hk, d, cache, room):
    announce(f"paged attention, few tokens, lens={lens} hq={hq} hk={hk} d={d} {cache}")
    check_line(gpu, lens, hq, hk, d, cache, room=room, least=0.2)


@pytest.mark.parametrize("d,cache", [(64, BF16), (128, BF16), (64, E4M3), (128, E4M3)])
def test_line_cut_at_its_tokens_ends(gpu, d, cache):
    """Stretches that end where tokens end: 32 tokens of four tiles for 32 groups (each finished by its group), 16 of
    eight (each two whole stretches), and the same with one tile more at the front (every cut moves by a little)."""
    announce(f"paged attention, even stretches, d={d} {cache}")
    _, groups, keys = tiles_and_groups(gpu, [], 64, 64, d, cache)
    for lens in ([4 * keys] * groups, [8 * keys] * (groups // 2), [1] + [4 * keys] * groups, [keys] + [0, 8 * keys] * (groups // 2)):
        check_line(gpu, lens, 64, 64, d, cache, room=33 * keys, rows=[i % 3 for i in range(len(lens))], least=4)


@pytest.mark.parametrize("window,softcap,slopes,d,cache,hq,hk", [
    (1500, 0.0, False, 128, BF16, 128, 32), (2500, 20.0, True, 64, BF16, 96, 32), (4400, 0.0, True, 64, E4M3, 64, 32),
    (2300, 5.0, False, 128, E4M3, 128, 32), (0, 30.0, True, 128, BF16, 32, 32), (0, 8.0, False, 64, E4M3, 160, 32),
    (0, 0.0, True, 128, E4M3, 64, 16), (1100, 1.0, True, 128, BF16, 640, 32),
])
def test_line_with_window_cap_and_bias(gpu, window, softcap, slopes, d, cache, hq, hk):
    announce(f"paged attention, line, window={window} softcap={softcap} slopes={slopes} d={d} {cache} hq={hq}")
    keys = tiles_and_groups(gpu, [], 1, 1, d, cache)[2]
    top = 80 * keys
    w = window or top // 2
    lens = [0, top, w - 1, w, w + 1, 0, w + 16, 1, top - 15, 3 * w // 2, 0, 0, top // 3, top - 1]
    check_line(gpu, lens, hq, hk, d, cache, room=top, window=window, softcap=softcap, slopes=slopes, amplitude=4.0)


@pytest.mark.parametrize("tokens,hq,hk,d,cache,top", [
    (513, 8, 4, 64, BF16, 2200), (1300, 2, 1, 64, BF16, 3000), (1024, 6, 2, 128, E4M3, 1500), (1500, 4, 4, 128, BF16, 900),
    (600, 20, 1, 64, E4M3, 5000),
])
def test_line_of_many_tokens(gpu, tokens, hq, hk, d, cache, top):
    """More than 512 tokens (several of them to a thread that counts their tiles), with empty ones at the front, at
    the end, at both ends of such runs and whole runs of them; seven rows hold the keys."""
    announce(f"paged attention, {tokens} tokens, hq={hq} hk={hk} d={d} {cache}")
    keys = tiles_and_groups(gpu, [], 1, 1, d, cache)[2]
    run = -(-tokens // 512)
    lens = [1 + (i * 7919) % top for i in range(tokens)]
    for i in range(tokens):
        if i < 11 or i >= tokens - 5 or i % (5 * run) == 0 or i % (7 * run) == run - 1 or 40 * run <= i < 47 * run:
            lens[i] = 0
    check_line(gpu, lens, hq, hk, d, cache, room=-(-max(top, 33 * keys) // 64) * 64, rows=[i % 7 for i in range(tokens)], ps=64)


@pytest.mark.parametrize("tokens,hk", [(700, 1), (1200, 8)])
def test_line_of_many_short_tokens(gpu, tokens, hk):
    """More than 512 tokens of a tile at most, most of them empty: fewer tiles than waves."""
    announce(f"paged attention, {tokens} short tokens of {hk} kv heads")
    lens = [(1 + i % 60) * (i % 17 == 3) for i in range(tokens)]
    tiles, groups, _ = tiles_and_groups(gpu, lens, 2 * hk, hk, 64, BF16)
    assert tiles < groups
    check_line(gpu, lens, 2 * hk, hk, 64, BF16, room=4096, rows=[i % 5 for i in range(tokens)], least=0)


# ------------------------------------------------------------------ the inverse rotation
@pytest.mark.parametrize("t,h,d,rot,interleaved,dtype,idx", [
    (70, 32, 128, 128, False, BF16, torch.int32), (33, 8, 128, 64, True, BF16, torch.int64), (129, 4, 64, 64, False, torch.float32, torch.int32),
    (16, 12, 128, 128, True, torch.float32, torch.int64), (17, 3, 128, 104, False, BF16, torch.int32), (9, 5, 64, 40, True, BF16, torch.int32),
])
def test_rope_inverse_by_whole_pieces(gpu, t, h, d, rot, interleaved, dtype, idx):
    """The first four have rows and rotated halves in whole 16-byte pieces, the last two go element by element:
    the gradient is the transpose of the formula's matrix, and turning there and back gives scale^2 x."""
    from torch_helion.hip import ops

    announce(f"rope inverse t={t} h={h} d={d} rot={rot} interleaved={interleaved} {dtype}")
    g = gen(t + rot)
    go = torch.randn(t, h * d, generator=g).to(dtype)
    pos = torch.randint(0, 5000, (t,), generator=g, dtype=idx)
    f = ops.rope_frequencies(rot, 10000.0)
    x = torch.zeros(t, h, d, dtype=torch.float64, requires_grad=True)
    n = rot // 2
    ia = torch.arange(n) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else n)
    ang = pos.double()[:, None, None] * f
    a, b = x[..., ia], x[..., ib]
    ga, gb = go.double().view(t, h, d)[..., ia], go.double().view(t, h, d)[..., ib]
    turned = ((a * ang.cos() - b * ang.sin()) * ga + (b * ang.cos() + a * ang.sin()) * gb).sum() * 1.25
    (ref,) = torch.autograd.grad(turned + (x[..., rot:] * go.double().view(t, h, d)[..., rot:]).sum(), x)
    _, mag = rope64(go.view(t, h, d), pos, f, interleaved, 1.25, inverse=True)
    half = u(dtype) if dtype == BF16 else 0.0
    got = torch.full((t, h * d), float("nan"), dtype=dtype, device=gpu)
    kw = dict(head_dim=d, interleaved=interleaved, scale=1.25)
    ops.rope(go.to(gpu), pos.to(gpu), f.to(gpu), got, inverse=True, **kw)
    assert_within(got.view(t, h, d), ref, ROT * mag + half * ref.abs() + 1e-30)
    there, back = torch.empty_like(got), torch.empty_like(got)
    ops.rope(go.to(gpu), pos.to(gpu), f.to(gpu), there, **kw)
    ops.rope(there, pos.to(gpu), f.to(gpu), back, inverse=True, **kw)
    want = go.double().view(t, h, d).clone()
    want[..., :rot] *= 1.25 ** 2
    # the first turn's roundings, turned back and scaled, then the second's own
    assert_within(back.view(t, h, d), want, (2 * ROT + 2 * half) * 1.25 * 2 * mag + half * want.abs() + 1e-30)


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


# ------------------------------------------------------------------ options of the cache and the block
@pytest.mark.parametrize("cache_type,options", [
    (BF16, dict(window=20, softcap=4.0)), (BF16, dict(rope_scale=1.2)), (E4M3, dict(window=33, rope_scale=0.9, softcap=15.0)),
    (E4M3, {}),
])
def test_block_options_and_scaled_pages(gpu, cache_type, options):
    """A step of the block with a window, a cap, a scaled rotation of frequencies of its own and, for an e4m3 cache,
    scales: what it stores and attends against 64 bits from its own projections; a captured step gives its bits."""
    from targets.llama_block import LlamaBlockConfig
    from test_e2e_gpu import _decode_case
    from torch_helion.hip import ops
    from torch_helion.hip.paged import PagedDecodeBlock, PagedKVCache

    announce(f"paged block {cache_type} {options}")
    cfg = LlamaBlockConfig(batch=5, seq=80, causal=True, dtype=BF16, rope_theta=500000.0, hidden=256, heads=4, kv_heads=2, intermediate=512)
    sd, x, *_ = _decode_case(cfg, cfg.seq, seed=4)
    hk, d, layer = cfg.n_kv, cfg.head_dim, 1
    g = gen(6)
    sc = {n: torch.rand(2, hk, generator=g) * 0.02 + 0.01 for n in ("k_scale", "v_scale")} if cache_type == E4M3 else {}
    cache = PagedKVCache(layers=2, pages=40, page_size=16, kv_heads=hk, head_dim=d, rows=6, max_len=128, dtype=cache_type, device=gpu, **sc)
    freqs = ops.rope_frequencies(d - 16, 10000.0, scaling="linear", factor=2.0)
    blk = PagedDecodeBlock(sd, hidden=cfg.hidden, heads=cfg.heads, kv_heads=hk, intermediate=cfg.intermediate, eps=cfg.eps,
                           rope_theta=cfg.rope_theta, batch=cfg.batch, cache=cache, layer=layer, freqs=freqs, **options)
    pos = [70, 0, -1, 31, 100]
    rows = [cache.open() for _ in range(5)]
    for r, p in zip(rows, pos):
        if p >= 0:
            cache.extend({r: p + 1})
            kv = [torch.randn(p + 1, hk * d, generator=g).to(BF16).to(gpu) for _ in range(2)]
            cache.append(layer, *kv, torch.arange(p + 1, dtype=torch.int32, device=gpu),
                         rows=torch.full((p + 1,), r, dtype=torch.int32, device=gpu))
    pt, rt = (torch.tensor(a, dtype=torch.int32, device=gpu) for a in (pos, rows))
    xs = x.to(gpu)
    blk.step(xs, pt, rt)
    torch.cuda.synchronize()
    q, k, v = (a.reshape(5, -1, d) for a in blk.qkv.cpu().split([cfg.heads * d, hk * d, hk * d], 1))
    scale = options.get("rope_scale", 1.0)
    live = [i for i, p in enumerate(pos) if p >= 0]
    at = pt.cpu()[live]
    (rq, mq), (rk, mk) = (rope64(a[live], at, freqs, False, scale) for a in (q, k))
    assert_within(blk.q.view(5, -1, d)[live], rq, ROT * mq + u(BF16) * rq.abs() + 1e-30, "q")
    page = torch.tensor([cache.book.pages[rows[i]][pos[i] // 16] for i in live])
    for pages, ref, mag, name in ((cache.k, rk, mk, "k_scale"), (cache.v, v[live].double(), torch.zeros_like(rk), "v_scale")):
        tol = ROT * mag + u(BF16) * ref.abs() + 1e-30
        if cache_type == E4M3:
            s = sc[name][layer].double()[:, None]
            ref, mag = (ref / s).clamp(-448, 448), mag / s
            tol = (ROT * mag + 2.0 ** -23 * ref.abs()) * (1 + u(E4M3)) + torch.clamp(u(E4M3) * ref.abs(), min=2.0 ** -10)
        assert_within(pages[layer].float().cpu()[page, at.long() % 16], ref, tol, name)
    mine = {n: s[layer].to(gpu) for n, s in sc.items()}
    ref, mag, err = attention64(blk.q.view(5, -1, d), cache.k[layer], cache.v[layer], cache.page_table, pt, rt, d ** -0.5,
                                options.get("window", 0), options.get("softcap", 0.0), None, mine.get("k_scale"), mine.get("v_scale"))
    tol = u(BF16) * ref.abs() + mag * (1 + u(BF16)) * (2 * err + p_step(cache_type) + 128 * 2.0 ** -23) + 1e-30
    assert_within(blk.attn.view(5, -1, d), ref, tol, "attention")
    assert blk.n_invalid.item() == 0 and torch.isfinite(blk.out32).all()
    want = [t.clone() for t in (blk.out32, cache.k.view(torch.uint8), cache.v.view(torch.uint8))]
    blk.capture(xs, pt, rt)
    for _ in range(3):
        blk.out32.zero_()
        blk.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((blk.out32, cache.k.view(torch.uint8), cache.v.view(torch.uint8)), want))
