"""Serving from a paged key-value cache: the operators, as cases that can be timed and compared.

Four operators that a decode loop over a paged cache is made of, each through its entry point in
``torch_helion.hip.ops`` and in a plain form of elementary torch operations:

  rope          rotary positions of a [tokens, heads * head_dim] tensor, every token at its own position;
  append        rotates the new keys (and queries) and stores keys and values into their cache pages;
  attention     one query per row against the pages of its sequence;
  copy          pages copied to other pages in every layer (forks), or moved with the page tables
                renamed (compaction).

A cache is ``[pages, page_size, kv_heads, head_dim]`` (copies: with a layer axis in front). Row r of a
page table lists the pages of sequence r; its unused tail holds -1. A token stands at ``positions[t]``
of sequence ``rows[t]`` (row t where there are no rows) and sees the keys at 0 .. positions[t]; a
position of -1 marks a padded row.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

_PKG = str(Path(__file__).resolve().parents[1] / "torch-helion_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

own = False

DEV = "cuda:0"
E4M3_MAX = 448.0
_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


# ------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # the queries of one decode step of 64 sequences at positions of their own: a launch's latency
        dict(name="rope_step", kind="rope", tokens=64, heads=32, head_dim=128, rot_dim=128, interleaved=False,
             stretch=1.0, far=4096, dtype="bfloat16"),
        # 8 x 2048 prompt tokens at far positions of a stretched context, half of each head, adjacent pairs
        dict(name="rope_prompt_far", kind="rope", tokens=16384, heads=32, head_dim=128, rot_dim=64, interleaved=True,
             stretch=8.0, far=131072, dtype="bfloat16"),
        # the append of a decode step: 64 sequences, one new token each, from the projection's fp32 output
        dict(name="append_step", kind="append", seqs=64, new_lo=1, new_hi=1, past=4000, heads=32, kv_heads=8,
             head_dim=128, page_size=16, rot_dim=128, interleaved=False, dtype="float32", cache="bfloat16"),
        # ragged prompts of 8 sequences entering an 8-bit cache
        dict(name="append_prompts_e4m3", kind="append", seqs=8, new_lo=501, new_hi=3500, past=700, heads=32, kv_heads=8,
             head_dim=128, page_size=64, rot_dim=128, interleaved=False, dtype="bfloat16", cache="e4m3"),
        # one user, a few hundred tokens in: latency
        dict(name="attention_one_short", kind="attention", seqs=1, len_lo=301, len_hi=301, padded=0, heads=32,
             kv_heads=8, head_dim=128, page_size=16, window=0, softcap=0.0, slopes=False, cache="bfloat16"),
        # the decode configuration's batch of 64 against up to 4096 keys, in small pages
        dict(name="attention_batch", kind="attention", seqs=64, len_lo=2048, len_hi=4096, padded=0, heads=32,
             kv_heads=8, head_dim=128, page_size=16, window=0, softcap=0.0, slopes=False, cache="bfloat16"),
        # an 8-bit cache, lengths from one token to 8192 and some slots of the batch unused
        dict(name="attention_batch_e4m3", kind="attention", seqs=64, len_lo=1, len_hi=8191, padded=5, heads=32,
             kv_heads=8, head_dim=128, page_size=64, window=0, softcap=0.0, slopes=False, cache="e4m3"),
        # two long documents: the work is one long axis
        dict(name="attention_long", kind="attention", seqs=2, len_lo=100003, len_hi=131072, padded=0, heads=32,
             kv_heads=8, head_dim=128, page_size=256, window=0, softcap=0.0, slopes=False, cache="bfloat16"),
        # 64-wide heads without sharing, a sliding window, capped scores and a bias by distance
        dict(name="attention_window_capped", kind="attention", seqs=24, len_lo=333, len_hi=4001, padded=1, heads=12,
             kv_heads=12, head_dim=64, page_size=32, window=1000, softcap=30.0, slopes=True, cache="bfloat16"),
        # 16 forked sequences get copies of their partly filled last pages in all 4 layers
        dict(name="copy_forks", kind="copy", layers=4, pages=512, moved=16, page_size=16, kv_heads=8, head_dim=128,
             rename=False, cache="bfloat16"),
        # a third of a pool moved together, with the page tables renamed
        dict(name="copy_compaction", kind="copy", layers=8, pages=2048, moved=683, page_size=32, kv_heads=8,
             head_dim=128, rename=True, cache="bfloat16"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    """An integer in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["rope", "append", "attention", "attention", "attention", "copy"])
    d = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128, 256])
    cache = rng.choice(["bfloat16", "bfloat16", "e4m3"])
    if kind == "rope":
        return dict(kind=kind, tokens=_log_int(rng, 1, 12000), heads=rng.choice([1, 8, 12, 32]), head_dim=d,
                    rot_dim=rng.choice([d, d, d // 2, d - 24]), interleaved=rng.random() < 0.5,
                    stretch=rng.choice([1.0, 4.0, 8.0]), far=_log_int(rng, 100, 1 << 20),
                    dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    if kind == "append":
        new = _log_int(rng, 1, 1500)
        return dict(kind=kind, seqs=_log_int(rng, 1, 64 if new < 200 else 8), new_lo=max(1, new // 3), new_hi=new,
                    past=_log_int(rng, 1, 3000), heads=kv * rng.choice([1, 4, 8]), kv_heads=kv, head_dim=d,
                    page_size=page, rot_dim=rng.choice([d, d, d // 2]), interleaved=rng.random() < 0.3,
                    dtype=rng.choice(["float32", "bfloat16"]), cache=cache)
    if kind == "attention":
        seqs = _log_int(rng, 1, 128)
        hi = _log_int(rng, 2, min(100000, 200000 // seqs))
        return dict(kind=kind, seqs=seqs, len_lo=rng.randint(1, hi), len_hi=hi, padded=rng.choice([0, 0, seqs // 4]),
                    heads=kv * rng.choice([1, 3, 4, 8, 16]), kv_heads=kv, head_dim=d, page_size=page,
                    window=rng.choice([0, 0, _log_int(rng, 16, 4096)]), softcap=rng.choice([0.0, 0.0, 20.0]),
                    slopes=rng.random() < 0.3, cache=cache)
    pages = _log_int(rng, 64, 2048 * 16 // page)
    return dict(kind="copy", layers=rng.randint(1, 8), pages=pages, moved=_log_int(rng, 1, pages // 3), page_size=page,
                kv_heads=kv, head_dim=d, rename=rng.random() < 0.5, cache=cache)


# ------------------------------------------------------------------ inputs
def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g: torch.Generator, shape, dtype: torch.dtype) -> torch.Tensor:
    if dtype == torch.float8_e4m3fn:
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16).to(dtype)
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _freqs(rot_dim: int, stretch: float) -> torch.Tensor:
    """Radians per position of the rot_dim / 2 pairs, float64; a stretched context divides the slow ones'
    by ``stretch``: those that turn less than once in 4096 positions, and in part those up to 32 times."""
    f = 500000.0 ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=DEV) / rot_dim)
    if stretch == 1.0:
        return f
    keep = ((f * (4096 / (2 * math.pi)) - 1.0) / 31.0).clamp(0.0, 1.0)
    return f * (keep + (1.0 - keep) / stretch)


def _spread(lo: int, hi: int, n: int, g: torch.Generator) -> torch.Tensor:
    """n whole numbers evenly over [lo, hi] (hi where there is one), in an order of the seed's."""
    at = torch.linspace(lo, hi, n, dtype=torch.float64, device=DEV).round() if n > 1 else \
        torch.tensor([hi], dtype=torch.float64, device=DEV)
    return at[torch.randperm(n, generator=g, device=DEV)].to(torch.int32)


def _table(lengths: torch.Tensor, longest: int, page_size: int, pages: int, g: torch.Generator) -> torch.Tensor:
    """Page table of sequences of these lengths: pages in an order of the seed's, -1 past each sequence's end."""
    n, width = lengths.numel(), -(-longest // page_size)
    table = torch.randperm(pages, generator=g, device=DEV)[:n * width].view(n, width).to(torch.int32)
    used = (lengths + page_size - 1) // page_size
    return table.masked_fill(torch.arange(width, device=DEV)[None] >= used[:, None], -1).contiguous()


def _scales(case: dict, g: torch.Generator) -> dict:
    """One scale per kv head of an 8-bit cache."""
    if case["cache"] != "e4m3":
        return {}
    return {n: torch.rand(case["kv_heads"], generator=g, device=DEV) * 0.5 + 0.75 for n in ("k_scale", "v_scale")}


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed)
    kind = case["kind"]
    if kind == "rope":
        s = {"x": _randn(g, (case["tokens"], case["heads"] * case["head_dim"]), _DTYPES[case["dtype"]]),
             "positions": torch.randint(0, case["far"], (case["tokens"],), generator=g, device=DEV, dtype=torch.int32),
             "freqs": _freqs(case["rot_dim"], case["stretch"]),
             "scale": 1.0 + 0.1 * math.log(case["stretch"])}
        return {"case": case, **s, "out": torch.empty_like(s["x"])}
    cache = _DTYPES[case["cache"]]
    row = (case["page_size"], case["kv_heads"], case["head_dim"])
    if kind == "copy":
        order = torch.randperm(case["pages"], generator=g, device=DEV).to(torch.int32)
        n = case["moved"]
        src, dst = order[:n].contiguous(), order[n:2 * n].contiguous()
        page_map = torch.arange(case["pages"], device=DEV, dtype=torch.int32)
        page_map[src.long()] = dst
        rest = torch.cat([src, order[2 * n:]])          # the pages in use before a compaction; dst's are free
        width = -(-rest.numel() // 8)
        table = torch.full((8 * width,), -1, device=DEV, dtype=torch.int32)
        table[:rest.numel()] = rest
        shape = (case["layers"], case["pages"]) + row
        return {"case": case, "k_cache": _randn(g, shape, cache), "v_cache": _randn(g, shape, cache), "src": src,
                "dst": dst, "page_table": table.view(8, width), "page_map": page_map}
    if kind == "append":
        new = _spread(case["new_lo"], case["new_hi"], case["seqs"], g)
        past = torch.randint(0, case["past"] + 1, (case["seqs"],), generator=g, device=DEV, dtype=torch.int32)
        tokens = _tokens(case)
        rows = torch.repeat_interleave(torch.arange(case["seqs"], device=DEV, dtype=torch.int32), new.long(), output_size=tokens)
        first = torch.cumsum(new, 0) - new
        positions = (torch.arange(tokens, device=DEV) - first[rows.long()] + past[rows.long()]).to(torch.int32)
        longest = case["past"] + case["new_hi"]
        pages = case["seqs"] * -(-longest // case["page_size"])
        table = _table(past + new, longest, case["page_size"], pages, g)
        qkv = _randn(g, (tokens, (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]), _DTYPES[case["dtype"]])
        q, k, v = qkv.split([n * case["head_dim"] for n in (case["heads"], case["kv_heads"], case["kv_heads"])], 1)
        return {"case": case, "q": q, "k": k, "v": v, "rows": rows, "positions": positions, "page_table": table,
                "freqs": _freqs(case["rot_dim"], 1.0), "k_cache": _randn(g, (pages,) + row, cache),
                "v_cache": _randn(g, (pages,) + row, cache), "scales": _scales(case, g),
                "q_out": torch.empty(q.shape, device=DEV, dtype=torch.bfloat16)}
    lengths = _spread(case["len_lo"], case["len_hi"], case["seqs"], g)
    if case["padded"]:
        lengths[torch.randperm(case["seqs"], generator=g, device=DEV)[:case["padded"]]] = 0
    pages = case["seqs"] * -(-case["len_hi"] // case["page_size"])
    slopes = 2.0 ** (-8.0 * torch.arange(1, case["heads"] + 1, device=DEV) / case["heads"]) if case["slopes"] else None
    q = _randn(g, (case["seqs"], case["heads"] * case["head_dim"]), torch.bfloat16)
    return {"case": case, "q": q, "positions": lengths - 1, "slopes": slopes,
            "page_table": _table(lengths, case["len_hi"], case["page_size"], pages, g),
            "k_cache": _randn(g, (pages,) + row, cache), "v_cache": _randn(g, (pages,) + row, cache),
            "scales": _scales(case, g), "out": torch.empty_like(q)}


def _tokens(case: dict) -> int:
    """The new tokens of an append case: the sum that _spread's numbers have for every seed."""
    lo, hi, n = case["new_lo"], case["new_hi"], case["seqs"]
    return int(torch.linspace(lo, hi, n, dtype=torch.float64).round().sum()) if n > 1 else hi


# ------------------------------------------------------------------ one pass
def _turn(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, head_dim: int, interleaved: bool,
          scale: float = 1.0) -> torch.Tensor:
    """The first 2 * len(freqs) dims of each head rotated, in fp32; the angles in 64 bits."""
    angle = positions.double()[:, None, None] * freqs
    cos, sin = (angle.cos() * scale).float(), (angle.sin() * scale).float()
    x = x.float().view(x.shape[0], -1, head_dim)
    r = 2 * freqs.numel()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _store(cache: torch.Tensor, page: torch.Tensor, slot: torch.Tensor, x: torch.Tensor, scale: torch.Tensor | None) -> None:
    if scale is not None:
        x = (x / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    cache[page, slot] = x.to(cache.dtype)


def _gathered(cache: torch.Tensor, table: torch.Tensor, scale: torch.Tensor | None) -> torch.Tensor:
    """[sequences, kv_heads, keys, head_dim] in fp32: every page that the table has room for."""
    x = cache[table.long().clamp(min=0)].flatten(1, 2).float()
    if scale is not None:
        x = x * scale[:, None]
    return x.transpose(1, 2).contiguous()


def run(state: dict):
    case = state["case"]
    kind = case["kind"]
    if own:
        from torch_helion.hip import ops

        if kind == "rope":
            return ops.rope(state["x"], state["positions"], state["freqs"], state["out"], head_dim=case["head_dim"],
                            interleaved=case["interleaved"], scale=state["scale"])
        if kind == "append":
            ops.paged_append(state["k"], state["v"], state["positions"], state["k_cache"], state["v_cache"],
                             state["page_table"], rows=state["rows"], freqs=state["freqs"],
                             interleaved=case["interleaved"], q=state["q"], q_out=state["q_out"], **state["scales"])
            return state["q_out"], state["k_cache"], state["v_cache"]
        if kind == "attention":
            return ops.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["page_table"],
                                       state["positions"], state["out"], scale=case["head_dim"] ** -0.5,
                                       window=case["window"], softcap=case["softcap"], slopes=state["slopes"],
                                       **state["scales"])
        named = dict(page_table=state["page_table"], page_map=state["page_map"]) if case["rename"] else {}
        ops.copy_pages(state["k_cache"], state["v_cache"], state["src"], state["dst"], **named)
        return state["k_cache"], state["v_cache"], state["page_table"]

    if kind == "rope":
        x = state["x"]
        turned = _turn(x, state["positions"], state["freqs"], case["head_dim"], case["interleaved"], state["scale"])
        return turned.reshape(x.shape).to(x.dtype)
    if kind == "append":
        d, scales = case["head_dim"], state["scales"]
        pos = state["positions"].long()
        page = state["page_table"][state["rows"].long(), pos // case["page_size"]].long()
        slot = pos % case["page_size"]
        k = _turn(state["k"], pos, state["freqs"], d, case["interleaved"])
        _store(state["k_cache"], page, slot, k, scales.get("k_scale"))
        _store(state["v_cache"], page, slot, state["v"].float().view(k.shape), scales.get("v_scale"))
        q = _turn(state["q"], pos, state["freqs"], d, case["interleaved"])
        return q.reshape(state["q"].shape).to(torch.bfloat16), state["k_cache"], state["v_cache"]
    if kind == "attention":
        keys = _gathered(state["k_cache"], state["page_table"], state["scales"].get("k_scale"))
        n, hk, width, d = keys.shape
        q = state["q"].float().view(n, hk, -1, d)
        s = (q @ keys.transpose(2, 3).contiguous()) * d ** -0.5                      # [n, hk, group, width]
        if case["softcap"]:
            s = torch.tanh(s / case["softcap"]) * case["softcap"]
        back = state["positions"][:, None] - torch.arange(width, device=DEV)          # how far a key lies behind
        if case["slopes"]:
            s = s - state["slopes"].float().view(hk, -1, 1) * back[:, None, None].float()
        seen = back >= 0
        if case["window"]:
            seen = seen & (back < case["window"])
        s = s.masked_fill(~seen[:, None, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
        o = p @ _gathered(state["v_cache"], state["page_table"], state["scales"].get("v_scale"))
        return (o / p.sum(-1, keepdim=True).clamp(min=1e-30)).reshape(n, -1).to(torch.bfloat16)
    src, dst = state["src"].long(), state["dst"].long()
    for cache in (state["k_cache"], state["v_cache"]):
        cache[:, dst] = cache[:, src]
    if case["rename"]:
        table = state["page_table"]
        table.copy_(torch.where(table >= 0, state["page_map"][table.long().clamp(min=0)], table))
    return state["k_cache"], state["v_cache"], state["page_table"]


# ------------------------------------------------------------------ what a pass cannot do without
def _seen_keys(case: dict) -> float:
    """Keys that all rows together see; which rows are padded is the seed's, so those count as the mean."""
    n, w = case["seqs"], case["window"]
    lens = torch.linspace(case["len_lo"], case["len_hi"], n, dtype=torch.float64).round() if n > 1 else \
        torch.tensor([float(case["len_hi"])], dtype=torch.float64)
    if w:
        lens = lens.clamp(max=w)
    return float(lens.mean()) * (n - case["padded"])


def work(case: dict) -> dict:
    kind, d = case["kind"], case["head_dim"]
    size = {"float32": 4, "bfloat16": 2, "e4m3": 1}
    if kind == "rope":
        n = case["tokens"] * case["heads"] * d
        return {"bytes": 2 * n * size[case["dtype"]] + 4 * case["tokens"],
                "flops": 3.0 * case["tokens"] * case["heads"] * case["rot_dim"]}
    c = size[case["cache"]]
    if kind == "append":
        t = _tokens(case)
        read = t * (case["heads"] + 2 * case["kv_heads"]) * d * size[case["dtype"]]
        return {"bytes": read + t * d * (2 * case["heads"] + 2 * c * case["kv_heads"]) + 8 * t,
                "flops": 3.0 * t * (case["heads"] + case["kv_heads"]) * case["rot_dim"]}
    if kind == "attention":
        keys = _seen_keys(case)
        return {"bytes": keys * (2 * c * case["kv_heads"] * d + 4 / case["page_size"]) + 4 * case["seqs"] * case["heads"] * d,
                "flops": 4.0 * keys * case["heads"] * d}
    page = case["page_size"] * case["kv_heads"] * d * c
    return {"bytes": 4.0 * case["layers"] * case["moved"] * page + 8 * case["moved"]
            + (8.0 * (case["pages"] - case["moved"]) if case["rename"] else 0), "flops": 0}


# ------------------------------------------------------------------ the same in 64 bits
def _turned64(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, interleaved: bool, scale: float) -> torch.Tensor:
    """x [t, h, d] in float64 as complex numbers times scale * exp(i position freq)."""
    n = freqs.numel()
    first = torch.arange(n, device=DEV) * (2 if interleaved else 1)
    second = first + (1 if interleaved else n)
    w = torch.polar(torch.full((positions.numel(), n), scale, dtype=torch.float64, device=DEV), torch.outer(positions.double(), freqs))
    z = torch.complex(x[..., first], x[..., second]) * w[:, None]
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _attended64(state: dict) -> torch.Tensor:
    """One row after the other: its keys by their pages, the softmax of its scores, the values' mean."""
    case = state["case"]
    d, size, hk = case["head_dim"], case["page_size"], case["kv_heads"]
    group = case["heads"] // hk
    ks = state["scales"].get("k_scale", torch.ones(hk, device=DEV)).double()
    vs = state["scales"].get("v_scale", torch.ones(hk, device=DEV)).double()
    out = torch.zeros(case["seqs"], case["heads"], d, dtype=torch.float64, device=DEV)
    q = state["q"].double().view(case["seqs"], case["heads"], d)
    for r, last in enumerate(state["positions"].tolist()):
        if last < 0:
            continue
        first = max(0, last + 1 - case["window"]) if case["window"] else 0
        at = torch.arange(first, last + 1, device=DEV)
        pages = state["page_table"][r].long()[at // size]
        for h in range(hk):
            keys = state["k_cache"][pages, at % size, h].double() * ks[h]
            values = state["v_cache"][pages, at % size, h].double() * vs[h]
            for m in range(h * group, (h + 1) * group):
                s = (keys @ q[r, m]) / math.sqrt(d)
                if case["softcap"]:
                    s = case["softcap"] * torch.tanh(s / case["softcap"])
                if case["slopes"]:
                    s = s - state["slopes"][m].double() * (last - at).double()
                out[r, m] = torch.softmax(s, 0) @ values
    return out.view(case["seqs"], -1)


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind, d = case["kind"], case["head_dim"]
    if kind == "rope":
        x = state["x"].double()
        y = _turned64(x.view(x.shape[0], -1, d), state["positions"], state["freqs"], case["interleaved"], state["scale"])
        return y.view(x.shape)
    if kind == "attention":
        return _attended64(state)
    if kind == "copy":
        to = dict(zip(state["src"].tolist(), state["dst"].tolist()))
        names = [[to.get(p, p) if case["rename"] else p for p in row] for row in state["page_table"].tolist()]
        whole = [c.double() for c in (state["k_cache"], state["v_cache"])]
        return *(c.index_copy_(1, state["dst"].long(), c.index_select(1, state["src"].long())) for c in whole), \
            torch.tensor(names, dtype=torch.int32, device=DEV)
    pos, size = state["positions"].long(), case["page_size"]
    flat = state["page_table"][state["rows"].long(), pos // size].long() * size + pos % size
    new = {n: state[n].double().view(pos.numel(), -1, d) for n in "qkv"}
    for n in "qk":
        new[n] = _turned64(new[n], state["positions"], state["freqs"], case["interleaved"], 1.0)
    caches = []
    for n in "kv":
        whole = state[n + "_cache"].double()
        if state["scales"]:
            new[n] = (new[n] / state["scales"][n + "_scale"].double()[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
        whole.view(-1, *whole.shape[2:]).index_copy_(0, flat, new[n])
        caches.append(whole)
    return new["q"].reshape(pos.numel(), -1), caches[0], caches[1]
