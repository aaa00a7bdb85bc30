"""The paged cache as a decode loop uses it: PagedKVCache and PagedDecodeBlock.

The block's bars are those of the contiguous decode step's test: 2e-2 normalised, and in max-abs twice the
bf16 rounding floor (the oracle's step with bf16 storage against the unrounded one).
"""

from __future__ import annotations

import pytest
import torch

from conftest import announce
from test_e2e_gpu import _decode_case, _spec_quantised

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
E4M3 = torch.float8_e4m3fn


def _block_and_cache(gpu, which: str, dtype=BF16, layers: int = 2, layer: int = 1, seed: int = 3):
    from targets.llama_block import LlamaBlockConfig
    from torch_helion.hip.paged import PagedDecodeBlock, PagedKVCache

    h = dict(small=dict(hidden=256, heads=4, kv_heads=2, intermediate=512),
             medium=dict(hidden=1024, heads=8, kv_heads=2, intermediate=2048))[which]
    cfg = LlamaBlockConfig(batch=5, seq=80, causal=True, dtype=BF16, rope_theta=500000.0, **h)
    sd, x, kc, vc = _decode_case(cfg, cfg.seq, seed=seed)
    cache = PagedKVCache(layers=layers, pages=40, page_size=16, kv_heads=cfg.n_kv, head_dim=cfg.head_dim, rows=6, max_len=2048,
                         dtype=dtype, device=gpu)
    blk = PagedDecodeBlock(sd, hidden=cfg.hidden, heads=cfg.heads, kv_heads=cfg.n_kv, intermediate=cfg.intermediate, eps=cfg.eps,
                           rope_theta=cfg.rope_theta, batch=cfg.batch, cache=cache, layer=layer)
    return cfg, sd, x, kc, vc, cache, blk


@pytest.mark.parametrize("which", ["small", "medium"])
def test_paged_step_vs_oracle(gpu, which):
    """Five rows at positions of their own, one of them unused, in cache rows of another order."""
    from oracle.llama import decode_step

    announce(f"paged decode step {which}")
    cfg, sd, x, kc, vc, cache, blk = _block_and_cache(gpu, which)
    w_spec = _spec_quantised(sd)
    pos = [70, 0, -1, 31, 16]
    rows = [cache.open() for _ in range(5)][::-1]
    cache.extend({r: p for r, p in zip(rows, pos) if p > 0})
    for i, (r, p) in enumerate(zip(rows, pos)):                      # the earlier keys and values, already rotated
        if p > 0:
            cache.append(1, kc[i, :p].reshape(p, -1).to(gpu), vc[i, :p].reshape(p, -1).to(gpu),
                         torch.arange(p, dtype=torch.int32, device=gpu), rows=torch.full((p,), r, dtype=torch.int32, device=gpu))
    cache.extend([r for r, p in zip(rows, pos) if p >= 0])
    pt, rt = (torch.tensor(a, dtype=torch.int32, device=gpu) for a in (pos, rows))
    blk.step(x.to(gpu), pt, rt)
    torch.cuda.synchronize()
    assert blk.n_invalid.item() == 0 and (cache.k[0].float() == 0).all() and (cache.v[0].float() == 0).all()
    kw = dict(heads=cfg.heads, kv_heads=cfg.n_kv, eps=cfg.eps, theta=cfg.rope_theta)
    out = blk.out32.cpu().double()
    size = cache.k.shape[2]
    for i, (r, p) in enumerate(zip(rows, pos)):
        if p < 0:
            assert torch.isfinite(out[i]).all() and (blk.attn[i] == 0).all()
            continue
        one = lambda **s: decode_step(x[i:i + 1], w_spec, kc[i:i + 1], vc[i:i + 1], p, **kw, **s)
        ref, kn, vn = one()
        ref_b, kn_b, vn_b = one(storage=BF16)
        err, floor = (out[i] - ref[0]).abs().max().item(), (ref_b - ref).abs().max().item()
        assert err / ref.abs().max().item() < 2e-2 and err <= 2 * floor, (i, err, floor)
        page = cache.book.pages[r][p // size]
        for pages, want, want_b in ((cache.k, kn, kn_b), (cache.v, vn, vn_b)):
            got = pages[1, page, p % size].double().cpu().reshape(want.shape)
            assert (got - want).abs().max().item() <= 2 * (want_b - want).abs().max().item()
        assert torch.equal(cache.k[1, cache.book.pages[r]].reshape(-1, cfg.n_kv, cfg.head_dim)[:p].cpu(), kc[i, :p])


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_captured_steps_equal_eager_ones(gpu, dtype):
    """A graph captured once and replayed over steps at which rows grow, start and end and pages move, against an
    eager block with a cache of its own: the same bits in outputs and pages."""
    announce(f"paged decode loop, captured, {dtype}")
    cfg, _, x, *_, cache, blk = _block_and_cache(gpu, "small", dtype)
    *_, cache2, eager = _block_and_cache(gpu, "small", dtype)
    xs = x.to(gpu).clone()
    positions = torch.full((5,), -1, dtype=torch.int32, device=gpu)
    rows = torch.zeros(5, dtype=torch.int32, device=gpu)
    blk.capture(xs, positions, rows)
    g = torch.Generator().manual_seed(1)
    live: dict[int, int] = {}                                         # slot of the batch -> cache row
    for step in range(40):
        for c in (cache, cache2):
            mine = dict(live)
            if step % 3 == 0 and len(mine) < 5:
                slot = min(set(range(5)) - set(mine))
                mine[slot] = c.fork(mine[min(mine)]) if step % 2 and mine else c.open()
            if step in (13, 26):
                c.close(mine.pop(max(mine)))
            if step in (14, 27):
                c.compact()
            c.extend(list(mine.values()))
        live = mine
        assert cache.book.pages == cache2.book.pages
        pos = [cache.length(live[i]) - 1 if i in live else -1 for i in range(5)]
        positions.copy_(torch.tensor(pos, dtype=torch.int32))
        rows.copy_(torch.tensor([live.get(i, 0) for i in range(5)], dtype=torch.int32))
        xs.copy_(torch.randn(xs.shape, generator=g).to(BF16))
        blk.replay()
        eager.step(xs, positions, rows)
        torch.cuda.synchronize()
        assert torch.equal(blk.out32, eager.out32), step
        assert torch.equal(cache.page_table, cache2.page_table)
        for a, b in ((cache.k, cache2.k), (cache.v, cache2.v)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), step
    assert max(pos) > 32 and blk.n_invalid.item() == eager.n_invalid.item() == 0


def test_forks_and_compaction_keep_every_row(gpu):
    """A prompt, forks that go their own ways, closed rows, a compaction: each row's keys read back through the
    page table are its own, and the attention's outputs keep their bits over the move."""
    from torch_helion.hip.paged import PagedKVCache

    announce("forks and compaction")
    hk, d, layers = 2, 64, 3
    cache = PagedKVCache(layers=layers, pages=24, page_size=16, kv_heads=hk, head_dim=d, rows=5, max_len=160, device=gpu)
    g = torch.Generator().manual_seed(2)
    tokens: dict[int, torch.Tensor] = {}

    def add(new: dict[int, int]):
        before = {r: cache.length(r) for r in new}
        cache.extend(new)
        for layer in range(layers):
            kv = [torch.randn(sum(new.values()), hk * d, generator=g).to(BF16) for _ in range(2)]
            pos = torch.cat([torch.arange(before[r], before[r] + n) for r, n in new.items()]).to(torch.int32)
            rows = torch.cat([torch.full((n,), r) for r, n in new.items()]).to(torch.int32)
            cache.append(layer, kv[0].to(gpu), kv[1].to(gpu), pos.to(gpu), rows=rows.to(gpu))
            for r in new:
                mine = torch.stack([t[rows == r] for t in kv])        # [2, n, hk * d]
                old = tokens.get((r, layer), mine[:, :0])
                tokens[(r, layer)] = torch.cat([old, mine], 1)

    def check():
        for (r, layer), want in tokens.items():
            pages = cache.page_table[r].long()
            pages = pages[pages >= 0]
            for c, w in zip((cache.k, cache.v), want):
                assert torch.equal(c[layer, pages].reshape(-1, hk * d)[:w.shape[0]].cpu(), w), (r, layer)

    def attend(**kw):
        live = sorted({r for r, _ in tokens})
        q = torch.randn(len(live), 4 * d, generator=torch.Generator().manual_seed(5)).to(BF16).to(gpu)
        out = torch.empty_like(q)
        cache.attend(1, q, torch.tensor([cache.length(r) - 1 for r in live], dtype=torch.int32, device=gpu), out, scale=0.125,
                     rows=torch.tensor(live, dtype=torch.int32, device=gpu), **kw)
        return out

    a, b = cache.open(), cache.open()
    add({a: 40, b: 70})
    forks = [cache.fork(a) for _ in range(3)]
    for r in forks:
        for layer in range(layers):
            tokens[(r, layer)] = tokens[(a, layer)]
    assert 24 - cache.free_pages == 3 + 5
    add({forks[0]: 1, a: 2, forks[2]: 20})
    assert 24 - cache.free_pages == 3 + 5 + 3 + 1                     # three copies of the last page, one new page
    check()
    cache.close(b)
    cache.shrink(forks[1], 17)
    tokens = {(r, layer): w[:, :17] if r == forks[1] else w for (r, layer), w in tokens.items() if r != b}
    out = attend()
    assert torch.equal(attend(max_keys=60), out)                      # no row is longer: a narrower table, the same keys
    used = 24 - cache.free_pages
    assert cache.compact() == used and int(cache.page_table.max()) == used - 1
    check()
    assert torch.equal(attend(), out)
    add({forks[1]: 1})                                                # writes into a page it shares with row a
    check()
