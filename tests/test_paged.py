"""The rotary and paged-cache entry points on the CPU: struct layouts, frequencies, refusals.

No call here reaches a device: each fails its argument checks, or stops where the library or the
tensor's device is missing.
"""

from __future__ import annotations

import ctypes as C
import functools
import math
import subprocess
from pathlib import Path

import pytest
import torch

REPO = Path(__file__).resolve().parents[1]
HEADER = REPO / "include" / "th_hip.h"
STRUCTS = {"th_rope_desc": "RopeDesc", "th_paged_append_desc": "PagedAppendDesc", "th_paged_attn_desc": "PagedAttnDesc",
           "th_page_copy_desc": "PageCopyDesc"}


@pytest.fixture(scope="module")
def lib():
    from torch_helion.hip import abi

    if not abi.library_path().exists():
        pytest.skip("libth_hip.so not built (run __graft_entry__.build())")
    return abi.load()


def test_struct_layouts_match_the_header(tmp_path):
    from torch_helion.hip import abi

    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "th_hip.h"', "int main(void){"]
    for cname, pyname in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in getattr(abi, pyname)._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines()
    got = {tuple(line.split()[:2]): int(line.split()[2]) for line in out}
    for cname, pyname in STRUCTS.items():
        st = getattr(abi, pyname)
        assert got[(cname, "size")] == C.sizeof(st)
        for f, _ in st._fields_:
            assert got[(cname, f)] == getattr(st, f).offset, (cname, f)


# ------------------------------------------------------------------ frequencies
def test_rope_frequencies():
    from torch_helion.hip import abi, ops

    f = ops.rope_frequencies(8, 10000.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    assert torch.allclose(ops.rope_frequencies(8, 10000.0, scaling="linear", factor=4.0), f / 4, rtol=1e-15)
    ntk = ops.rope_frequencies(8, 10000.0, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], 0.001 / 4, rel_tol=1e-12)
    parts = ops.rope_frequencies(128, 500000.0, scaling="by_parts", factor=8.0, original_len=8192, low=1.0, high=4.0)
    plain = ops.rope_frequencies(128, 500000.0)
    turns = plain * 8192 / (2 * math.pi)
    assert torch.equal(parts[turns > 4], plain[turns > 4])
    assert torch.allclose(parts[turns < 1], plain[turns < 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and (parts[mid] < plain[mid]).all() and (parts[mid] > plain[mid] / 8).all()
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(scaling="other"), dict(scaling="by_parts"),
                dict(scaling="linear", factor=0.0), dict(rot_dim=2, scaling="ntk", factor=2.0)):
        with pytest.raises(abi.HipBackendError):
            ops.rope_frequencies(**{"rot_dim": 8, "theta": 10000.0, **bad})


# ------------------------------------------------------------------ refusals of the C entries
def rope_desc(abi):
    d = abi.RopeDesc()
    d.tokens, d.heads, d.head_dim, d.rot_dim, d.dtype, d.positions_dtype, d.scale = 4, 2, 64, 64, abi.TH_BF16, abi.TH_I32, 1.0
    d.x, d.ld_x, d.positions, d.freqs, d.out, d.ld_out = 4096, 128, 8192, 12288, 16384, 128
    return d


def append_desc(abi):
    d = abi.PagedAppendDesc()
    d.tokens, d.heads_q, d.heads_kv, d.head_dim, d.rot_dim = 4, 4, 2, 64, 64
    d.in_dtype, d.cache_dtype, d.page_size, d.n_rows, d.row_pages, d.pages, d.scale = abi.TH_BF16, abi.TH_BF16, 16, 4, 2, 9, 1.0
    d.positions, d.page_table, d.ld_page_table, d.freqs = 4096, 8192, 2, 12288
    d.q, d.ld_q, d.q_out, d.ld_q_out, d.k, d.ld_k, d.v, d.ld_v = 16384, 256, 20480, 256, 24576, 128, 28672, 128
    d.k_cache, d.k_stride_page, d.k_stride_t, d.k_stride_h = 32768, 2048, 128, 64
    d.v_cache, d.v_stride_page, d.v_stride_t, d.v_stride_h = 65536, 2048, 128, 64
    return d


def attn_desc(abi):
    d = abi.PagedAttnDesc()
    d.tokens, d.heads_q, d.heads_kv, d.head_dim, d.cache_dtype, d.page_size = 4, 4, 2, 64, abi.TH_BF16, 16
    d.n_rows, d.row_pages, d.pages, d.scale = 4, 2, 9, 0.125
    d.positions, d.page_table, d.ld_page_table, d.q, d.ld_q, d.o, d.ld_o = 4096, 8192, 2, 16384, 256, 20480, 256
    d.k_cache, d.k_stride_page, d.k_stride_t, d.k_stride_h = 32768, 2048, 128, 64
    d.v_cache, d.v_stride_page, d.v_stride_t, d.v_stride_h = 65536, 2048, 128, 64
    d.workspace, d.workspace_bytes = 131072, 1 << 40
    return d


def copy_desc(abi):
    d = abi.PageCopyDesc()
    d.layers, d.n, d.pages, d.page_bytes = 2, 3, 9, 4096
    d.k_cache, d.k_layer_bytes, d.k_page_bytes = 4096, 65536, 4096
    d.v_cache, d.v_layer_bytes, d.v_page_bytes = 262144, 65536, 4096
    d.src, d.dst, d.page_table, d.ld_page_table, d.n_rows, d.row_pages, d.page_map = 8192, 8256, 12288, 2, 4, 2, 16384
    return d


REFUSED = [
    ("th_rope", rope_desc, [
        ({"rot_dim": 63}, "rot_dim"), ({"rot_dim": 66}, "rot_dim"), ({"rot_dim": 0}, "rot_dim"), ({"dtype": 2}, "dtype"),
        ({"positions_dtype": 0}, "positions dtype"), ({"head_dim": 2048, "rot_dim": 64}, "head_dim"), ({"heads": 0}, "heads"),
        ({"ld_x": 127}, "row stride"), ({"ld_out": 64}, "row stride"), ({"out": 4096, "ld_out": 256}, "in place"),
        ({"freqs": 0}, "null"), ({"positions": 0}, "null"), ({"tokens": -1}, "tokens"), ({"tokens": 1 << 31}, "tokens")]),
    ("th_paged_append", append_desc, [
        ({"rot_dim": 5}, "rot_dim"), ({"rot_dim": 66}, "rot_dim"), ({"page_size": 24}, "page_size"), ({"page_size": 0}, "page_size"),
        ({"cache_dtype": 0}, "cache_dtype"), ({"in_dtype": 3}, "in_dtype"), ({"heads_kv": 0}, "heads"), ({"heads_q": -1}, "heads"),
        ({"n_rows": 0}, "page table"), ({"ld_page_table": 1}, "page table"), ({"pages": 0}, "page table"),
        ({"ld_k": 64}, "row stride"), ({"ld_q": 64}, "row stride"), ({"q_out": 16384, "ld_q_out": 512}, "in place"),
        ({"q_out": 16384, "in_dtype": 0}, "in place"), ({"k_stride_h": 32}, "cache stride"), ({"v_stride_t": 0}, "cache stride"),
        ({"k_scale": 4096}, "e4m3"), ({"tokens": 5}, "exceed the table"), ({"freqs": 0}, "null"), ({"q": 0}, "null"),
        ({"page_table": 0}, "null")]),
    ("th_paged_attention", attn_desc, [
        ({"heads_q": 5}, "multiple"), ({"head_dim": 96}, "head_dim"), ({"cache_dtype": 0}, "cache_dtype"), ({"page_size": 8}, "page_size"),
        ({"page_size": 48}, "page_size"), ({"row_pages": 0}, "page table"), ({"window": -1}, "window"), ({"softcap": -1.0}, "softcap"),
        ({"softcap": float("nan")}, "softcap"), ({"softcap": 1025.0}, "softcap"), ({"softcap": 1e-39}, "softcap"), ({"tokens": 65536}, "tokens"), ({"ld_q": 255}, "row strides"), ({"ld_q": 260}, "16 bytes"),
        ({"k_stride_h": 68}, "16 bytes"), ({"v_stride_page": 2050}, "16 bytes"), ({"cache_dtype": 3, "k_stride_t": 136}, "16 bytes"),
        ({"k_stride_t": 1 << 23}, "token strides"), ({"q": 16392}, "16-byte"), ({"v_cache": 65544}, "16-byte"), ({"v_scale": 4096}, "e4m3"),
        ({"tokens": -1}, "tokens"), ({"tokens": 5}, "exceed the table"), ({"positions": 0}, "null"), ({"o": 0}, "null"),
        ({"row_pages": 1 << 27, "ld_page_table": 1 << 27}, "2^30")]),
    ("th_page_copy", copy_desc, [
        ({"layers": 0}, "sizes"), ({"n": -1}, "sizes"), ({"page_bytes": 4104}, "16"), ({"k_cache": 4104}, "16"),
        ({"k_page_bytes": 2048}, "page stride"), ({"v_layer_bytes": 0}, "layer stride"), ({"page_map": 0}, "page table"),
        ({"ld_page_table": 1}, "page table"), ({"src": 0}, "null"), ({"n": 1 << 30, "page_bytes": 16}, "one launch")]),
]


@pytest.mark.parametrize("entry,make,over,message", [(e, m, o, s) for e, m, cases in REFUSED for o, s in cases])
def test_refusals(lib, entry, make, over, message):
    from torch_helion.hip import abi

    d = make(abi)
    for name, value in over.items():
        setattr(d, name, value)
    assert getattr(lib, entry)(C.byref(d), None) == abi.TH_ERR_INVALID
    text = abi.last_error(lib)
    assert text.startswith(entry) and message in text, text


@pytest.mark.parametrize("entry,make,empty", [
    ("th_rope", rope_desc, {"tokens": 0, "x": 0, "positions": 0}), ("th_paged_append", append_desc, {"tokens": 0, "k": 0}),
    ("th_paged_attention", attn_desc, {"tokens": 0, "q": 0, "workspace": 0}),
    ("th_page_copy", copy_desc, {"n": 0, "page_table": 0, "src": 0})])
def test_null_empty_and_valid_descriptors(lib, entry, make, empty):
    """A null descriptor is refused, an empty call is a no-op, a valid one passes every check (and stops at the
    missing th_init where there is no GPU)."""
    from torch_helion.hip import abi

    fn = getattr(lib, entry)
    assert fn(None, None) == abi.TH_ERR_INVALID
    d = make(abi)
    if not torch.cuda.is_available():
        assert fn(C.byref(d), None) == abi.TH_ERR_NOT_INIT, abi.last_error(lib)
    for name, value in empty.items():
        setattr(d, name, value)
    assert fn(C.byref(d), None) == abi.TH_OK, abi.last_error(lib)


def test_workspace_query(lib):
    from torch_helion.hip import abi, ops

    good = dict(tokens=4, heads_q=8, heads_kv=2, head_dim=64, cache_dtype=abi.TH_BF16, max_keys=4096, window=0)
    query = lambda **kw: lib.th_paged_attention_workspace_bytes(*{**good, **kw}.values())
    for bad in ({"tokens": -1}, {"heads_q": 0}, {"heads_kv": 3}, {"head_dim": 96}, {"heads_kv": 0}, {"cache_dtype": abi.TH_F32},
                {"max_keys": 0}, {"window": -1}, {"max_keys": 1 << 30}):
        assert query(**bad) == -1, bad
    assert query() > 0 and query(tokens=0) == 0
    # 16 tiles of 8 KiB of keys at most: 1024 keys of 64 bf16 dims, 2048 of e4m3; a window of w can touch w + 15
    assert query(max_keys=1024) == 0 and query(max_keys=1040) > 0
    assert query(max_keys=2048, cache_dtype=abi.TH_F8E4M3) == 0
    assert query(window=1009) == 0 and query(window=1010) > 0
    # up to 32 tiles from 128 pairs on
    assert query(max_keys=2048, tokens=63) > 0 and query(max_keys=2048, tokens=64) == 0 and query(max_keys=2064, tokens=64) > 0
    assert ops.paged_attention_workspace_bytes(4, 8, 2, 64, 4096) == query()
    with pytest.raises(abi.HipBackendError):
        ops.paged_attention_workspace_bytes(4, 8, 3, 64, 4096)


# ------------------------------------------------------------------ refusals of the Python layer
def tensors():
    t, hk, d = 4, 2, 64
    kc = torch.zeros(9, 16, hk, d, dtype=torch.bfloat16)
    return dict(k=torch.zeros(t, hk * d, dtype=torch.bfloat16), v=torch.zeros(t, hk * d, dtype=torch.bfloat16),
                positions=torch.zeros(t, dtype=torch.int32), k_cache=kc, v_cache=torch.zeros_like(kc),
                page_table=torch.zeros(t, 2, dtype=torch.int32), q=torch.zeros(t, 4 * d, dtype=torch.bfloat16),
                out=torch.zeros(t, 4 * d, dtype=torch.bfloat16), freqs=torch.zeros(d // 2, dtype=torch.float64))


@pytest.mark.parametrize("change,message", [
    ({"positions": torch.zeros(4, dtype=torch.int64)}, "positions"), ({"positions": torch.zeros(3, dtype=torch.int32)}, "positions"),
    ({"positions": torch.zeros(8, dtype=torch.int32)[::2]}, "positions"), ({"page_table": torch.zeros(4, 2)}, "page_table"),
    ({"v_cache": torch.zeros(9, 16, 2, 32, dtype=torch.bfloat16)}, "caches"), ({"rows": torch.zeros(4, dtype=torch.int64)}, "rows"),
    ({"k_cache": torch.zeros(9, 16, 64, 2, dtype=torch.bfloat16).transpose(2, 3)}, "contiguous"),
    ({"k_scale": torch.ones(3)}, "k_scale"), ({}, "HIP device"),
])
def test_paged_argument_checks(change, message):
    from torch_helion.hip import abi, ops

    a = {**tensors(), **change}
    rest = {n: a[n] for n in ("rows", "k_scale") if n in a}
    with pytest.raises(abi.HipBackendError, match=message):
        ops.paged_append(a["k"], a["v"], a["positions"], a["k_cache"], a["v_cache"], a["page_table"], freqs=a["freqs"], **rest)
    with pytest.raises(abi.HipBackendError, match=message):
        ops.paged_attention(a["q"], a["k_cache"], a["v_cache"], a["page_table"], a["positions"], a["out"], scale=1.0, **rest)


def test_more_argument_checks():
    from torch_helion.hip import abi, ops

    a = tensors()
    append = lambda **kw: ops.paged_append(**{**{n: a[n] for n in ("k", "v", "positions", "k_cache", "v_cache", "page_table")}, **kw})
    attend = lambda **kw: ops.paged_attention(**{**{n: a[n] for n in ("q", "k_cache", "v_cache", "page_table", "positions", "out")},
                                                 "scale": 1.0, **kw})
    rope = lambda **kw: ops.rope(**{**dict(x=a["q"], positions=a["positions"], freqs=a["freqs"], out=a["out"], head_dim=64), **kw})
    copy = lambda **kw: ops.copy_pages(**{**dict(k_cache=a["k_cache"], v_cache=a["v_cache"], src=a["positions"], dst=a["positions"]), **kw})
    for call, kw, message in (
            (append, {"v": a["v"].float()}, "v must be"), (append, {"q": a["q"]}, "q_out"), (append, {"freqs": a["freqs"].float()}, "freqs"),
            (append, {"k": a["k"][:, :64]}, "k must be"), (append, {"k": a["k"][:1].expand(4, -1)}, "row stride|HIP device"),
            (append, {"q": a["q"][:, :100], "q_out": a["q"]}, "heads"), (attend, {"q": a["q"].float()}, "q must be .* torch.bfloat16"),
            (attend, {"slopes": torch.ones(3)}, "slopes"), (attend, {"window": 1 << 32}, "window"), (attend, {"window": -1}, "window"), (attend, {"out": a["out"][:3]}, "out must be"),
            (rope, {"head_dim": 60}, "heads"), (rope, {"scale": 1e40}, "out of range"), (rope, {"positions": a["positions"].float()}, "int32 or int64"),
            (rope, {"out": a["out"].float()}, "out must be"), (rope, {}, "HIP device"), (copy, {"src": a["positions"][:2]}, "dst"),
            (copy, {"page_table": a["page_table"]}, "page_map"), (copy, {"k_cache": a["k_cache"][:, :8], "v_cache": a["v_cache"][:, :8]}, "HIP device"),
            (copy, {"k_cache": a["k_cache"][:, ::2], "v_cache": a["v_cache"][:, ::2]}, "dense"), (copy, {}, "HIP device")):
        with pytest.raises(abi.HipBackendError, match=message):
            call(**kw)


# ------------------------------------------------------------------ who holds which page
def page_book(**kw):
    from torch_helion.hip.paged import PageBook

    return PageBook(**{**dict(pages=12, page_size=4, rows=4, row_pages=6), **kw})


def snapshot(book):
    return (list(book.refs), sorted(book.free), sorted(book.free_rows), {r: list(p) for r, p in book.pages.items()}, dict(book.length))


@pytest.mark.parametrize("seed", range(6))
def test_page_book_against_token_lists(seed):
    """Random opens, forks, extensions, cuts, closes and compactions: every row reads back its own
    tokens from the pages it is said to hold, and the counts add up; a refused call changes nothing."""
    import random

    from torch_helion.hip import abi

    rng = random.Random(seed)
    book = page_book(pages=rng.choice([5, 12, 30]), page_size=rng.choice([1, 4, 16]))
    content = {p: [None] * book.page_size for p in range(len(book.refs))}
    tokens: dict[int, list[int]] = {}
    stamp, refused = 0, 0
    for _ in range(400):
        act = rng.choice(["open", "fork", "extend", "extend", "extend", "extend", "shrink", "close", "compact"])
        before = snapshot(book)
        rows = list(tokens)
        try:
            if act == "open":
                tokens[book.open()] = []
            elif act == "fork" and rows:
                r = rng.choice(rows)
                tokens[book.fork(r)] = list(tokens[r])
            elif act == "extend" and rows:
                counts = {r: rng.choice([0, 1, 1, 1, rng.randint(2, 9)]) for r in rng.sample(rows, rng.randint(1, len(rows)))}
                copies, entries = book.extend(counts)
                table = {(r, i): p for r, i, p in entries}
                for a, b in copies:
                    content[b] = list(content[a])
                for r, n in counts.items():
                    for i in range(n):
                        stamp += 1
                        at = len(tokens[r]) // book.page_size
                        page = book.pages[r][at]
                        assert table.get((r, at), page) == page and book.refs[page] == 1
                        content[page][len(tokens[r]) % book.page_size] = stamp
                        tokens[r].append(stamp)
            elif act == "shrink" and rows:
                r = rng.choice(rows)
                n = rng.randint(0, len(tokens[r]))
                book.shrink(r, n)
                del tokens[r][n:]
            elif act == "close" and rows:
                r = rng.choice(rows)
                book.close(r)
                del tokens[r]
            elif act == "compact":
                moves = book.compact()
                assert not {a for a, _ in moves} & {b for _, b in moves}
                for a, b in moves:
                    content[b] = list(content[a])
                used = sum(r > 0 for r in book.refs)
                assert all(r > 0 for r in book.refs[:used]) and not any(book.refs[used:])
        except abi.HipBackendError:
            refused += 1
            assert snapshot(book) == before
        for r, want in tokens.items():
            assert book.length[r] == len(want) and len(book.pages[r]) == -(-len(want) // book.page_size)
            got = [content[p][i] for p in book.pages[r] for i in range(book.page_size)][:len(want)]
            assert got == want
        held = [p for pages in book.pages.values() for p in pages]
        assert [held.count(p) for p in range(len(book.refs))] == book.refs
        assert sorted(book.free) == [p for p, n in enumerate(book.refs) if n == 0] and len(set(held) & set(book.free)) == 0
    assert refused > 0


def test_page_book_refusals():
    from torch_helion.hip import abi
    from torch_helion.hip.paged import PagedKVCache

    book = page_book(pages=3, page_size=4, rows=2, row_pages=2)
    row = book.open()
    for call, message in ((lambda: book.extend({row: 9}), "exceed the table"), (lambda: book.extend({5: 1}), "not open"),
                          (lambda: book.extend({row: -1}), "tokens"), (lambda: book.fork(7), "not open"), (lambda: book.close(7), "not open"),
                          (lambda: book.shrink(row, 1), "tokens")):
        with pytest.raises(abi.HipBackendError, match=message):
            call()
    book.extend({row: 8})
    other = book.fork(row)
    with pytest.raises(abi.HipBackendError, match="no free row"):
        book.open()
    book.shrink(other, 6)
    assert book.extend({other: 1}) == ([(1, 2)], [(other, 1, 2)])       # its last page was shared
    book.close(row)
    row = book.open()
    with pytest.raises(abi.HipBackendError, match="pages needed"):
        book.extend({row: 5})
    assert book.length[row] == 0 and book.free == [1]
    sizes = dict(layers=1, pages=4, page_size=16, kv_heads=1, head_dim=64, rows=1, max_len=64)
    for change, message in (({"device": "cpu"}, "HIP device"),):
        with pytest.raises(abi.HipBackendError, match=message):
            PagedKVCache(**{**sizes, **change})


# ------------------------------------------------------------------ several devices
class Devices:
    """Stands for several devices: which one is current, and a library whose answers depend on it. As in the
    library, th_init makes its device the current one."""

    def __init__(self, monkeypatch):
        from torch_helion.hip import abi, ops

        self.current = 0
        outer = self

        class Guard:
            def __init__(self, device):
                self.to = device if isinstance(device, int) else torch.device(device).index

            def __enter__(self):
                self.was, outer.current = outer.current, self.to

            def __exit__(self, *_):
                outer.current = self.was

        class Lib:
            def th_paged_attention_workspace_bytes(self, *sizes):
                return 1000 + outer.current

        def init_device(device):
            outer.current = device
            return Lib()

        monkeypatch.setattr(abi, "load", lambda path=None: Lib())
        monkeypatch.setattr(abi, "init_device", init_device)
        monkeypatch.setattr(torch.cuda, "device", Guard)
        monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)
        ops._paged_workspace.cache_clear()
        monkeypatch.setattr(ops, "_paged_workspace", functools.lru_cache(maxsize=8)(ops._paged_workspace.__wrapped__))


def test_workspace_is_asked_of_its_device(monkeypatch):
    """The answer is the device's own, not the first one's, and the current device stays what it was."""
    from torch_helion.hip import abi, ops

    devices = Devices(monkeypatch)
    for current in (0, 2, 0, 1):
        devices.current = current
        assert ops.paged_attention_workspace_bytes(4, 8, 2, 64, 4096) == 1000 + current
        assert devices.current == current
    for device in (1, "cuda:2", torch.device("cuda", 3), "cuda"):
        devices.current = 0
        index = 0 if device == "cuda" else torch.device("cuda", device).index if isinstance(device, int) else torch.device(device).index
        assert ops.paged_attention_workspace_bytes(4, 8, 2, 64, 4096, device=device) == 1000 + index
        assert devices.current == 0
    with pytest.raises(abi.HipBackendError, match="HIP device"):
        ops.paged_attention_workspace_bytes(4, 8, 2, 64, 4096, device="cpu")
    assert ops._paged_workspace(5, 4, 8, 2, 64, 4096, 0, torch.bfloat16) == 1005 and devices.current == 0


def test_paged_decode_block_on_another_device(monkeypatch):
    """Built and stepped with its cache's device current, and the current one left as it was."""
    from torch_helion.hip import decode, ops, paged

    devices = Devices(monkeypatch)
    seen = []
    note = lambda *a, **k: seen.append(devices.current)

    class Cache:
        device = torch.device("cuda", 1)
        k = torch.zeros(1, 4, 16, 2, 64)
        page_table = torch.zeros(3, 4, dtype=torch.int32)
        append = attend = staticmethod(note)

    def build(self, state_dict, *, device, batch, **_):
        note()
        self.device, self.B, self.D, self.H, self.Hkv, self.hd, self.eps = device, batch, 256, 4, 2, 64, 1e-5
        self.wqkv = self.g1 = self.q = self.attn = self.attn_ws = self.n_invalid = None
        self.qkv = torch.zeros(batch, 8 * 64)

    monkeypatch.setattr(decode.DecodeBlock, "__init__", build)
    monkeypatch.setattr(decode.DecodeBlock, "_gemm", note)
    monkeypatch.setattr(decode.DecodeBlock, "_after_attention", note)
    blk = paged.PagedDecodeBlock({}, hidden=256, heads=4, kv_heads=2, intermediate=512, eps=1e-5, rope_theta=1e4, batch=3, cache=Cache())
    x, pos = torch.zeros(3, 256, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    blk.step(x, pos)
    assert seen == [1] * 5 and devices.current == 0
    devices.current = 1
    blk.step(x, pos)
    assert seen == [1] * 9 and devices.current == 1

    asked = []
    monkeypatch.setattr(ops, "paged_attention_workspace_bytes", lambda *a, device=None, **k: asked.append(device) or 0)
    monkeypatch.setattr(torch, "empty", lambda *a, **k: None)
    monkeypatch.setattr(torch, "zeros", lambda *a, **k: None)
    blk.device, blk.max_len, blk.freqs = Cache.device, 64, Cache.k
    monkeypatch.setattr(torch.Tensor, "to", lambda self, *a: self)
    blk._allocate_cache()
    assert asked == [Cache.device]


def test_attention_onto_its_queries_needs_their_stride(lib):
    """With another stride a token's output would lie on queries that are still to be read; one token has none."""
    from torch_helion.hip import abi

    for tokens, ld_o, status in ((4, 512, abi.TH_ERR_INVALID), (4, 256, None), (1, 512, None)):
        d = attn_desc(abi)
        d.tokens, d.o, d.ld_o = tokens, d.q, ld_o
        if status is None:
            if torch.cuda.is_available():
                continue
            status = abi.TH_ERR_NOT_INIT
        assert lib.th_paged_attention(C.byref(d), None) == status
        if status == abi.TH_ERR_INVALID:
            assert "in place" in abi.last_error(lib)
