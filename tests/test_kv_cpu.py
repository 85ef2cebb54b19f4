"""The attention half without a GPU: the page book's bookkeeping, the C ABI's refusals, the Python side's checks."""
import contextlib
import ctypes
import math
import random

import pytest
import torch

from engines.qwen36 import Rotary
from gguf import hip
from gguf.hbm_cache import HBMKVCache, OutOfPages, PageBook
from oracle import kv_ref

FAKE = 0x10000  # a non-NULL, aligned address that is never dereferenced


# -- the page book ---------------------------------------------------------------------------------------------------


def check_book(book):
    """Every page is free, or used as often as sequences hold it; sequences hold just the pages that their tokens need."""
    uses = [0] * book.pages
    for length, pages in book.sequences.values():
        assert len(pages) == -(-length // book.page_tokens) and len(set(pages)) == len(pages)
        for p in pages:
            uses[p] += 1
    assert uses == book.uses
    assert sorted(book.free_pages) == [p for p in range(book.pages) if not uses[p]]


class Contents:
    """What a device would hold, by the book's copies and a writer that writes where the book says."""

    def __init__(self, book):
        self.book, self.page, self.want = book, [[None] * book.page_tokens for _ in range(book.pages)], {}

    def copy(self, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for a, b in zip(src, dst):
            self.page[b] = list(self.page[a])

    def grow(self, seqs, counts, stamp):
        self.copy(*self.book.grow(seqs, counts))
        for s, n in zip(seqs, counts):
            length, pages = self.book.sequences[s]
            for t in range(length - n, length):
                self.page[pages[t // self.book.page_tokens]][t % self.book.page_tokens] = (stamp, s, t)
                self.want.setdefault(s, []).append((stamp, s, t))

    def check(self):
        for s, (length, pages) in self.book.sequences.items():
            got = [self.page[pages[t // self.book.page_tokens]][t % self.book.page_tokens] for t in range(length)]
            assert got == self.want.get(s, []), f"sequence {s}"


@pytest.mark.parametrize("seed", range(8))
def test_page_book_random(seed):
    """Random lives of sequences: what each one reads is always what was written for it, whatever was forked, cut, freed,
    copied and compacted in between."""
    rng = random.Random(seed)
    book = PageBook(40, 16)
    c = Contents(book)
    for i in range(400):
        live = list(book.sequences)
        what = rng.choice(("new", "grow", "grow", "grow", "fork", "free", "truncate", "compact"))
        if what == "new" or not live:
            c.want[book.new()] = []
        elif what == "grow":
            seqs = rng.sample(live, rng.randint(1, min(4, len(live))))
            counts = [rng.choice((0, 1, 1, 5, 16, 33)) for _ in seqs]
            before = {s: [v[0], list(v[1])] for s, v in book.sequences.items()}
            try:
                c.grow(seqs, counts, i)
            except OutOfPages:
                assert before == book.sequences
                book.free(rng.choice(live))
        elif what == "fork":
            s = rng.choice(live)
            c.want[book.fork(s)] = list(c.want[s])
        elif what == "free":
            book.free(rng.choice(live))
        elif what == "truncate":
            s = rng.choice(live)
            n = rng.randint(0, book.length(s))
            book.truncate(s, n)
            c.want[s] = c.want[s][:n]
        else:
            c.copy(*book.compact())
            assert all(p < book.used() for v in book.sequences.values() for p in v[1])
        check_book(book)
        c.check()


def test_page_book_takes_the_lowest():
    book = PageBook(8, 16)
    a, b = book.new(), book.new()
    assert book.grow([a, b], [20, 1]) == ([], []) and book.sequences[a][1] == [0, 1] and book.sequences[b][1] == [2]
    book.free(a)
    d = book.new()
    book.grow([d], [40])
    assert book.sequences[d][1] == [0, 1, 3]


def test_page_book_shared_last_page():
    """Of a page that n sequences share and all write, n - 1 take copies; of one that only some write, each of those."""
    book = PageBook(8, 16)
    a = book.new()
    book.grow([a], [20])
    b, c = book.fork(a), book.fork(a)
    src, dst = book.grow([a, b, c], [1, 1, 1])
    assert src == [1, 1] and dst == [2, 3] and book.sequences[c][1] == [0, 1]
    e = book.fork(a)
    assert book.grow([e], [1]) == ([2], [4]) and book.grow([a], [1]) == ([], [])
    f = book.fork(a)
    book.truncate(f, 16)
    assert book.grow([f], [1]) == ([], [])  # the page behind whole shared ones is its own


def test_page_book_refuses():
    book = PageBook(2, 16)
    a = book.new()
    for bad in (lambda: book.grow([a, a], [1, 1]), lambda: book.grow([a], [-1]), lambda: book.grow([a], [1, 2]),
                lambda: book.truncate(a, 1), lambda: book.truncate(a, -1)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: book.grow([7], [1]), lambda: book.free(7), lambda: book.fork(7), lambda: book.length(7)):
        with pytest.raises(KeyError):
            bad()
    with pytest.raises(OutOfPages):
        book.grow([a], [33])
    assert book.used() == 0 and book.length(a) == 0


# -- the C ABI -------------------------------------------------------------------------------------------------------


def cache_struct(**over):
    s = hip.WlKvCache(FAKE, FAKE, FAKE, FAKE, 8, 2, 2, 64, 16, 0, 0)
    for k, v in over.items():
        setattr(s, k, v)
    return s


def batch_struct(**over):
    b = hip.WlKvBatch(FAKE, FAKE, 4, 6, 2, 4, 3, 0)
    for k, v in over.items():
        setattr(b, k, v)
    return b


def test_struct_layout():
    assert ctypes.sizeof(hip.WlKvCache) == 4 * 8 + 8 + 6 * 4 == 64
    assert ctypes.sizeof(hip.WlKvBatch) == 4 * 8 + 4 * 4 == 48
    assert ctypes.sizeof(hip.WlRopeTensor) == 6 * 8 + 2 * 4 == 56


BAD_CACHES = [({"k": None}, -3), ({"v_scale": None}, -3), ({"type": 2}, -13), ({"head_dim": 96}, -13), ({"page_tokens": 8}, -13),
              ({"page_tokens": 48}, -13), ({"page_tokens": 2048}, -13), ({"pages": 0}, -2), ({"pages": 1 << 31}, -2),
              ({"layers": 0}, -2), ({"kv_heads": 0}, -2), ({"reserved": 1}, -2), ({"v": FAKE + 8}, -4), ({"k_scale": FAKE + 2}, -4)]
BAD_BATCHES = [({"table": None}, -3), ({"cu": None}, -3), ({"seqs": 0}, -2), ({"seqs": 65536}, -2), ({"table_width": 0}, -2),
               ({"table_stride": 3}, -2), ({"tokens": 0}, -2), ({"max_count": 0}, -2), ({"max_count": 7}, -2), ({"reserved": 1}, -2),
               ({"cu": FAKE + 2}, -4)]


def calls(cache, batch, layer=0):
    lib = hip.library()
    c, b = ctypes.byref(cache), ctypes.byref(batch)
    return [lib.wl_kv_append(c, layer, FAKE, 128, 64, FAKE, 128, 64, b, FAKE, None),
            lib.wl_kv_attend(c, layer, FAKE, 256, 64, 4, b, FAKE, 64, 0.125, 1, FAKE, None, 0, None)]


@pytest.mark.parametrize("over,code", BAD_CACHES)
def test_bad_caches(over, code):
    lib, cache = hip.library(), cache_struct(**over)
    assert lib.wl_kv_check(ctypes.byref(cache)) == code and calls(cache, batch_struct()) == [code, code]
    assert lib.wl_kv_copy(ctypes.byref(cache), FAKE, FAKE, 1, None) == code
    assert lib.wl_kv_attend_workspace_bytes(ctypes.byref(cache), 4, ctypes.byref(batch_struct()), 64) == 0


@pytest.mark.parametrize("over,code", BAD_BATCHES)
def test_bad_batches(over, code):
    assert calls(cache_struct(), batch_struct(**over)) == [code, code]


def test_bad_calls():
    lib = hip.library()
    c, b = ctypes.byref(cache_struct()), ctypes.byref(batch_struct())
    assert calls(cache_struct(), batch_struct(), layer=2) == [-2, -2] and calls(cache_struct(), batch_struct(), layer=-1) == [-2, -2]
    append = lambda k=FAKE, v=FAKE, start=FAKE: lib.wl_kv_append(c, 0, k, 128, 64, v, 128, 64, b, start, None)  # noqa: E731
    assert append(k=None) == append(v=None) == append(start=None) == -3 and append(k=FAKE + 1) == append(start=FAKE + 2) == -4

    def attend(q=FAKE, heads=4, batch=b, length=FAKE, bound=64, scale=0.125, out=FAKE, ws=None, n=0):
        return lib.wl_kv_attend(c, 0, q, 256, 64, heads, batch, length, bound, scale, 1, out, ws, n, None)
    assert attend(q=None) == attend(length=None) == attend(out=None) == -3
    assert attend(q=FAKE + 1) == attend(out=FAKE + 8) == attend(length=FAKE + 1) == -4
    assert attend(heads=3) == attend(heads=0) == attend(bound=-1) == -2
    assert attend(scale=-1.0) == attend(scale=math.inf) == attend(scale=math.nan) == -2
    long = ctypes.byref(batch_struct(table_width=64, table_stride=64))
    need = lib.wl_kv_attend_workspace_bytes(c, 4, long, 1024)
    assert need > 0 and attend(batch=long, bound=1024) == attend(batch=long, bound=1024, ws=FAKE, n=need - 1) == -6
    assert attend(batch=long, bound=1024, ws=FAKE + 4, n=need) == -6
    huge = ctypes.byref(batch_struct(seqs=65535, table_width=1 << 20, table_stride=1 << 20))
    assert attend(batch=huge) == -2  # more tiles than 31 bits count


@pytest.mark.parametrize("src,dst,code", [([0], [8], -14), ([-1], [2], -14), ([8], [2], -14), ([0, 1], [3, 3], -14),
                                          ([0, 1], [1, 2], -14), ([4], [4], -14)])
def test_bad_copies(src, dst, code):
    a, b = ((ctypes.c_int32 * len(x))(*x) for x in (src, dst))
    assert hip.library().wl_kv_copy(ctypes.byref(cache_struct()), a, b, len(src), None) == code


def test_copy_counts():
    lib, c = hip.library(), ctypes.byref(cache_struct())
    one = (ctypes.c_int32 * 1)(0)
    assert lib.wl_kv_copy(c, None, None, 0, None) == 0 and lib.wl_kv_copy(c, None, one, 1, None) == -3
    assert lib.wl_kv_copy(c, one, one, -1, None) == lib.wl_kv_copy(c, one, one, 9, None) == -2


def test_bad_rope():
    lib = hip.library()

    def call(q={}, k=None, dtype=1, tokens=4, dim=64, rotary=32, pos=FAKE, inv=FAKE, axes=3, sections=(6, 5, 5), inter=1):  # noqa: B006
        def tensor(over):
            t = hip.WlRopeTensor(FAKE, FAKE, 256, 64, 256, 64, 4, 0)
            for n, v in over.items():
                setattr(t, n, v)
            return ctypes.byref(t)
        return lib.wl_rope(tensor(q), None if k is None else tensor(k), dtype, tokens, dim, rotary, pos, 4, inv, axes,
                           (ctypes.c_int32 * len(sections))(*sections), inter, 1.0, None)
    assert call(dtype=2) == -7 and call(q={"in_": None}) == call(q={"out": None}) == call(k={"in_": None}) == -3
    assert call(pos=None) == call(inv=None) == -3 and call(pos=FAKE + 4) == call(inv=FAKE + 4) == call(q={"in_": FAKE + 1}) == -4
    assert call(dtype=0, q={"out": FAKE + 2}) == -4
    for bad in (dict(tokens=0), dict(dim=1), dict(dim=2048), dict(rotary=33), dict(rotary=66), dict(rotary=0), dict(axes=0),
                dict(axes=5, sections=(4, 4, 4, 4, 0)), dict(sections=(6, 5, 4)), dict(sections=(16, 1, -1)), dict(sections=(4, 5, 7)),
                dict(q={"heads": 0}), dict(k={"heads": 0}), dict(q={"reserved": 1})):
        assert call(**bad) == -2, bad


def test_error_strings():
    for code in (-13, -14):
        assert hip.library().wl_error_string(code) != hip.library().wl_error_string(-99)


# -- the Python side -------------------------------------------------------------------------------------------------


def test_pages_refuse():
    z = torch.zeros
    ok = dict(k=z(1, 2, 1, 16, 64, dtype=torch.int8), v=z(1, 2, 1, 64, 16, dtype=torch.int8), k_scale=z(1, 2, 1), v_scale=z(1, 2, 1))
    hip.KVPages(**ok)
    for bad in (dict(k=z(1, 2, 1, 16, 64)), dict(v=z(1, 2, 1, 16, 64, dtype=torch.int8)), dict(v=z(1, 2, 1, 64, 16)),
                dict(k_scale=z(1, 2)), dict(v_scale=z(1, 2, 2)), dict(k_scale=z(1, 2, 1, dtype=torch.float64)),
                dict(k=z(1, 2, 1, 64, 16, dtype=torch.int8).transpose(3, 4)),
                dict(k=z(1, 2, 1, 16, 96, dtype=torch.int8), v=z(1, 2, 1, 96, 16, dtype=torch.int8)),
                dict(k=z(1, 2, 1, 24, 64, dtype=torch.int8), v=z(1, 2, 1, 64, 24, dtype=torch.int8))):
        with pytest.raises(ValueError):
            hip.KVPages(**{**ok, **bad})


def test_call_checks():
    """What the wrappers refuse before they reach the library (on tensors of the CPU, which they take for a device's)."""
    z = torch.zeros
    p = hip.KVPages.empty(1, 4, 2, 64, 16, device="cpu")
    k, q = z(3, 2, 64, dtype=torch.bfloat16), z(3, 4, 64, dtype=torch.bfloat16)
    i = dict(dtype=torch.int32)
    good = dict(table=z(1, 2, **i), cu=z(2, **i))
    for bad in (dict(table=z(1, 2)), dict(table=z(2, **i)), dict(cu=z(3, **i)), dict(cu=z(2, dtype=torch.int64)), dict(cu=z(4, **i)[::2]),
                dict(table=z(1, 4, **i)[:, ::2]), dict(cu=[0, 3])):
        a = {**good, **bad}
        with pytest.raises(ValueError):
            hip.kv_append(p, 0, k, k, a["table"], z(1, **i), a["cu"])
        with pytest.raises(ValueError):
            hip.kv_attend(p, 0, q, a["table"], z(1, **i), a["cu"])
    for bad in (k.float(), z(3, 1, 64, dtype=torch.bfloat16), z(3, 2, 32, dtype=torch.bfloat16), z(2, 2, 64, dtype=torch.bfloat16), None,
                z(3, 2, 128, dtype=torch.bfloat16)[:, :, ::2]):
        with pytest.raises(ValueError):
            hip.kv_append(p, 0, k, bad, good["table"], z(1, **i), good["cu"])
    for bad in (q.float(), z(3, 3, 64, dtype=torch.bfloat16), z(3, 0, 64, dtype=torch.bfloat16), z(3, 4, 32, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            hip.kv_attend(p, 0, bad, good["table"], z(1, **i), good["cu"])
    for out in (q.float(), z(2, 4, 64, dtype=torch.bfloat16), z(3, 4, 128, dtype=torch.bfloat16)[:, :, :64]):
        with pytest.raises(ValueError):
            hip.kv_attend(p, 0, q, good["table"], z(1, **i), good["cu"], out=out)
    with pytest.raises(ValueError):
        hip.kv_copy(p, [0, 1], [2])
    with pytest.raises(ValueError):
        hip.rope(z(2, 1, 64), None, z(2, dtype=torch.int64), z(8, dtype=torch.float64))  # not on a GPU


def test_rotary():
    r = Rotary(256, 64, 1e7, (11, 11, 10), device="cpu")
    assert r.inv_freq.dtype == torch.float64 and float(r.inv_freq[0]) == 1.0
    assert float(r.inv_freq[16]) == pytest.approx(1e7 ** -0.5, rel=1e-15)
    assert r.positions(torch.arange(5)).shape == (3, 5)
    for bad in (dict(rotary_dim=63), dict(rotary_dim=512), dict(sections=(11, 11, 11), rotary_dim=64), dict(inv_freq=[1.0], rotary_dim=64)):
        with pytest.raises(ValueError):
            Rotary(256, device="cpu", **bad)


# -- the oracle's own pieces -----------------------------------------------------------------------------------------


def test_oracle_rounding():
    assert kv_ref.bf16_not_below(1.0) == 1.0 and kv_ref.bf16_not_below(1.0 + 2.0 ** -20) == 1.0 + 2.0 ** -7
    x = torch.linspace(-448, 448, 30001, dtype=torch.float64)
    assert torch.equal(kv_ref.nearest(x, torch.float8_e4m3fn), x.to(torch.float32).to(torch.float8_e4m3fn).double())
    tiny = torch.linspace(-0.03, 0.03, 30001, dtype=torch.float64)
    assert torch.equal(kv_ref.nearest(tiny, torch.float8_e4m3fn), tiny.to(torch.float32).to(torch.float8_e4m3fn).double())


def test_table_rows_lie_apart(monkeypatch):
    """A table whose rows overlap in memory (an expanded one) is refused: the kernels step from row to row by at least its
    width. Of one sequence the stride between rows means nothing."""
    z = torch.zeros
    p = hip.KVPages.empty(1, 4, 2, 64, 16, device="cpu")
    k, q = z(3, 2, 64, dtype=torch.bfloat16), z(3, 4, 64, dtype=torch.bfloat16)
    strides = []
    monkeypatch.setattr("gguf.hip.kv._launch", lambda index, call, *args: strides.extend(
        a.table_stride for a in args if isinstance(a, hip.WlKvBatch)))
    i = dict(dtype=torch.int32)
    for table in (z(1, 2, **i).expand(3, 2), z(4, **i).as_strided((3, 2), (1, 1)), z(1, 1, **i).expand(3, 1)):
        with pytest.raises(ValueError, match="apart"):
            hip.kv_append(p, 0, k, k, table, z(3, **i), z(4, **i))
        with pytest.raises(ValueError, match="apart"):
            hip.kv_attend(p, 0, q, table, z(3, **i), z(4, **i))
    assert not strides
    for table, want in ((z(3, 2, **i), 2), (z(3, 5, **i)[:, :2], 5), (z(5, **i)[:2][None], 2), (z(3, 1, **i), 1)):
        hip.kv_append(p, 0, k, k, table, z(len(table), **i), z(len(table) + 1, **i))
        assert strides.pop() == want


def test_cpu_tensors_are_not_launched(monkeypatch):
    """Calls that are right but for their device, on a machine that may well have a GPU: an error, and no kernel."""
    z = torch.zeros
    p = hip.KVPages.empty(1, 4, 2, 64, 16, device="cpu")
    k, q, i = z(3, 2, 64, dtype=torch.bfloat16), z(3, 4, 64, dtype=torch.bfloat16), dict(dtype=torch.int32)

    class Calls:
        wl_kv_append = wl_kv_attend = wl_kv_copy = staticmethod(lambda *args: pytest.fail("reached the library"))
        wl_kv_attend_workspace_bytes = staticmethod(lambda *args: 0)

    monkeypatch.setattr("gguf.hip.kv.library", lambda: Calls)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    for call in (lambda: hip.kv_append(p, 0, k, k, z(1, 2, **i), z(1, **i), z(2, **i)),
                 lambda: hip.kv_attend(p, 0, q, z(1, 2, **i), z(1, **i), z(2, **i)), lambda: hip.kv_copy(p, [0], [1])):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_copied_pages_stay_the_pages_named(monkeypatch):
    """Page numbers are cut to 32 bits for the library: none may become another one on the way."""
    import numpy as np
    p = hip.KVPages.empty(1, 4, 2, 64, 16, device="cpu")
    got = []
    monkeypatch.setattr("gguf.hip.kv._launch", lambda index, call, pages, src, dst, n: got.extend(
        (ctypes.c_int32 * n).from_address(a)[:] for a in (src, dst)))
    for bad in (np.array([2 ** 32 + 1]), np.array([2 ** 31], dtype=np.uint32), [-1], [1.5], [True], [2 ** 70], np.array([-2 ** 32])):
        with pytest.raises(ValueError):
            hip.kv_copy(p, bad, [2])
        with pytest.raises(ValueError):
            hip.kv_copy(p, [2], bad)
    hip.kv_copy(p, [], [])
    assert not got
    for kind in (list, np.array, lambda x: np.array(x, dtype=np.int32), lambda x: np.array(x, dtype=np.uint8),
                 lambda x: np.array([v for n in x for v in (n, 9)], dtype=np.int32)[::2]):
        hip.kv_copy(p, kind([0, 1]), kind([2, 3]))
        assert got == [[0, 1], [2, 3]]
        got.clear()


def test_step_needs_all_its_rows(monkeypatch):
    cache = HBMKVCache(1, 4, 2, 64, 16, device="cpu")
    step = cache.step([cache.new(), cache.new()], [3, 2])
    calls = []
    monkeypatch.setattr("gguf.hbm_cache.kv_append", lambda *args, **kw: calls.append("append"))
    monkeypatch.setattr("gguf.hbm_cache.kv_attend", lambda *args, **kw: calls.append("attend"))
    k = torch.zeros(7, 2, 64, dtype=torch.bfloat16)
    for rows in (0, 4):
        with pytest.raises(ValueError, match="5 tokens"):
            cache.append(0, step, k[:rows], k[:rows])
        with pytest.raises(ValueError, match="5 tokens"):
            cache.attend(0, step, k[:rows])
    assert not calls
    for rows in (5, 7):  # all of them, and a padded batch
        cache.append(0, step, k[:rows], k[:rows])
        cache.attend(0, step, k[:rows])
    assert calls == ["append", "attend"] * 2


def test_launch_limits():
    """Sizes that no launch holds are refused before one is made (2^32 threads along an axis)."""
    lib = hip.library()
    c = cache_struct()
    huge = dict(tokens=2 ** 31 - 1, max_count=2 ** 31 - 1)
    assert calls(c, batch_struct(**huge)) == [-2, -2]
    tensor = ctypes.byref(hip.WlRopeTensor(FAKE, FAKE, 256, 64, 256, 64, 4, 0))
    sections = (ctypes.c_int32 * 1)(16)
    assert lib.wl_rope(tensor, None, 1, 2 ** 24, 64, 32, FAKE, 4, FAKE, 1, sections, 1, 1.0, None) == -2
    wide = cache_struct(kv_heads=256)
    many = batch_struct(seqs=65535)
    assert lib.wl_kv_attend(ctypes.byref(wide), 0, FAKE, 256, 64, 256, ctypes.byref(many), FAKE, 64, 0.125, 1, FAKE, None, 0, None) == -2
    long = batch_struct(seqs=65535, tokens=2 ** 26, max_count=2 ** 26)  # of the form for many rows
    assert lib.wl_kv_attend(ctypes.byref(c), 0, FAKE, 256, 64, 4, ctypes.byref(long), FAKE, 64, 0.125, 1, FAKE, FAKE, 2 ** 40, None) == -2
    # a scale that times log2 e is infinite
    assert lib.wl_kv_attend(ctypes.byref(c), 0, FAKE, 256, 64, 4, ctypes.byref(batch_struct()), FAKE, 64, 3e38, 1, FAKE, None, 0, None) == -2


def test_out_is_not_q():
    p = hip.KVPages.empty(1, 4, 2, 64, 16, device="cpu")
    q, i = torch.zeros(3, 4, 64, dtype=torch.bfloat16), dict(dtype=torch.int32)
    with pytest.raises(ValueError, match="not q's memory"):
        hip.kv_attend(p, 0, q, torch.zeros(1, 2, **i), torch.zeros(1, **i), torch.zeros(2, **i), out=q)


def test_numbers_keep_their_value(monkeypatch):
    """The library takes 32-bit numbers: a layer or a count that does not fit is refused, not cut to another one."""
    z = torch.zeros
    p = hip.KVPages.empty(2, 4, 2, 64, 16, device="cpu")
    k, q, i = z(3, 2, 64, dtype=torch.bfloat16), z(3, 4, 64, dtype=torch.bfloat16), dict(dtype=torch.int32)
    launched = []
    monkeypatch.setattr("gguf.hip.kv._launch", lambda index, call, *args: launched.append(args[1]))
    args = (z(1, 2, **i), z(1, **i), z(2, **i))
    for layer in (2, -1, 2 ** 32, 2 ** 32 + 1, -2 ** 32, 2 ** 64 + 1):
        with pytest.raises(ValueError, match="layer"):
            hip.kv_append(p, layer, k, k, *args)
        with pytest.raises(ValueError, match="layer"):
            hip.kv_attend(p, layer, q, *args)
    for count in (-1, 1 - 2 ** 32, 2 - 2 ** 64):
        with pytest.raises(ValueError, match="max_count"):
            hip.kv_append(p, 0, k, k, *args, max_count=count)
        with pytest.raises(ValueError, match="max_count"):
            hip.kv_attend(p, 0, q, *args, max_count=count)
    for length in (-1, 64 - 2 ** 64):
        with pytest.raises(ValueError, match="max_length"):
            hip.kv_attend(p, 0, q, *args, max_length=length)
    assert not launched
    for layer in (0, 1):
        hip.kv_append(p, layer, k, k, *args, max_count=2 ** 40)
        hip.kv_attend(p, layer, q, *args, max_count=2 ** 40, max_length=2 ** 70)
    assert launched == [0, 0, 1, 1]


@pytest.mark.parametrize("side", ["q", "k"])
@pytest.mark.parametrize("heads,token,head,apart", [
    (4, 256, 64, True), (4, 1000, 64, True), (4, 64, 64 * 5, True), (1, 64, 0, True), (1, 64, 7, True), (4, -256, 64, True),
    (4, 256, -64, True), (2, 150, 100, False), (3, 160, 64, False), (2, 192, 64, True), (2, 64, 96, False), (4, 0, 64, False),
    (4, 256, 0, False), (4, 63, 64 * 5, False), (4, 255, 64, False), (4, 256, 63, False), (4, 256, 32, False), (4, -255, 64, False),
    (2, 128, 320, True), (2, 128, 340, False), (2, 128, 319, False), (8, 128, 192, False)])
def test_rope_rows_lie_apart(side, heads, token, head, apart):
    """Results whose tokens or heads share memory would be written twice, in no order: refused before anything is launched. What
    overlaps is worked out from every pair of rows."""
    tokens, dim = 5, 64
    at = sorted(t * token + h * head for t in range(tokens) for h in range(heads))
    assert apart == all(b - a >= dim for a, b in zip(at, at[1:]))
    lib, sections = hip.library(), (ctypes.c_int32 * 1)(16)
    good = hip.WlRopeTensor(FAKE, FAKE, 256, 64, 256, 64, 4, 0)
    over = hip.WlRopeTensor(3 * FAKE, 3 * FAKE, 256, 64, token, head, heads, 0)
    # positions on no 8-byte address are refused behind the tensors: what a call ends with whose tensors are right
    rc = lib.wl_rope(over if side == "q" else good, over if side == "k" else None, 1, tokens, dim, 32, FAKE + 4, tokens, FAKE, 1,
                     sections, 1, 1.0, None)
    assert rc == (-4 if apart else -2)
    one = lib.wl_rope(over if side == "q" else good, over if side == "k" else None, 1, 1, dim, 32, FAKE + 4, 1, FAKE, 1, sections, 1,
                      1.0, None)
    assert one == (-4 if heads == 1 or abs(head) >= dim else -2)  # of one token the stride between tokens means nothing


def test_out_overlaps_q():
    """out in the memory of q's rows is refused wherever they meet, before anything is launched; between the rows, or beside them,
    it may lie. Against every pair of elements."""
    lib, rng = hip.library(), random.Random(3)
    c = cache_struct(kv_heads=1)
    seen = [0, 0]
    for _ in range(3000):
        tokens, heads = rng.randint(1, 5), rng.randint(1, 4)
        token, head = (rng.choice((0, 64, 72, 128, 256, 300, 1000, 2000, -64, -256, -700)) for _ in range(2))
        at = 8 * rng.randint(-400, 400)  # out's beginning behind q's, in elements
        rows = {t * token + h * head for t in range(tokens) for h in range(heads)}
        meet = any(r < at + tokens * heads * 64 and r + 64 > at for r in rows)
        b = batch_struct(tokens=tokens, max_count=1, table_width=64, table_stride=64)
        args = (FAKE, token, head, heads, ctypes.byref(b), FAKE, 1024, 0.125, 1, FAKE + 2 * at)
        need = lib.wl_kv_attend_workspace_bytes(ctypes.byref(c), heads, ctypes.byref(b), 1024)
        assert need
        if meet:
            assert lib.wl_kv_attend(ctypes.byref(c), 0, *args, FAKE, need, None) == -11
        elif not torch.cuda.is_available():  # nothing stands in the way of a launch, which ends without a device
            assert lib.wl_kv_attend(ctypes.byref(c), 0, *args, FAKE, need, None) > 0
        seen[meet] += 1
    assert min(seen) > 500


def test_counts_are_whole(monkeypatch):
    """Fractions of tokens are refused with nothing changed (they were cut to whole ones, or left a book of fractions)."""
    book = PageBook(4, 16)
    a = book.new()
    book.grow([a], [20])
    for bad in (1.5, 0.999, float("nan"), float("inf"), "1", None):
        with pytest.raises((ValueError, TypeError)):
            book.grow([a], [bad])
        with pytest.raises((ValueError, TypeError)):
            book.truncate(a, bad)
        assert book.length(a) == 20 and book.sequences[a][1] == [0, 1]
    cache = HBMKVCache(1, 8, 2, 64, 16, device="cpu")
    s = cache.new()
    step = cache.step([s], [3], width=4)
    for bad in ([1.5], [3.5], ["3"]):
        with pytest.raises((ValueError, TypeError)):
            cache.step([s], bad)
        with pytest.raises((ValueError, TypeError)):
            cache.refresh(step, [s], bad)
        assert cache.length(s) == 3
    import numpy as np
    for one in (1, 1.0, np.int32(1), np.float32(1), torch.tensor(1)):
        cache.step([s], [one])
    cache.truncate(s, np.int64(4))
    cache.truncate(s, 2.0)
    assert cache.length(s) == 2 and type(cache.length(s)) is int
    check_book(cache.book)


def test_nothing_is_booked_under_capture(monkeypatch):
    """step, refresh and compact upload tables or move pages that the book counts as moved at once: under capture, where nothing
    runs, they are refused with nothing changed."""
    cache = HBMKVCache(1, 8, 2, 64, 16, device="cpu")
    a, b = cache.new(), cache.new()
    step = cache.step([a], [20], width=4)
    cache.step([b], [3])
    cache.truncate(a, 0)
    cache.step([a], [1])
    before = {s: [v[0], list(v[1])] for s, v in cache.book.sequences.items()}
    monkeypatch.setattr("torch.cuda.is_current_stream_capturing", lambda: True)
    monkeypatch.setattr("torch.cuda.device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(cache.pages, "index", 0)
    monkeypatch.setattr("gguf.hbm_cache.kv_copy", lambda *args: pytest.fail("copied"))
    for call in (lambda: cache.step([a], [1]), lambda: cache.refresh(step, [a], [20]), lambda: cache.compact()):
        with pytest.raises(RuntimeError, match="captur"):
            call()
        assert before == cache.book.sequences
    check_book(cache.book)


@pytest.mark.parametrize("after", range(4))
def test_steps_whose_tables_do_not_arrive(monkeypatch, after):
    """An upload that fails (no memory, say) leaves no token counted that no step can write."""
    cache = HBMKVCache(1, 8, 2, 64, 16, device="cpu")
    a, b = cache.new(), cache.new()
    step = cache.step([a, b], [10, 40], width=4)
    real, left = torch.from_numpy, [after]

    def upload(array):
        if not left[0]:
            raise RuntimeError("out of memory")
        left[0] -= 1
        return real(array)
    monkeypatch.setattr(torch, "from_numpy", upload)
    for call in (lambda: cache.step([b, a], [20, 7]), lambda: cache.refresh(step, [b, a], [10, 40])):
        left[0] = min(after, 2) if "refresh" in call.__code__.co_names else after
        with pytest.raises(RuntimeError, match="memory"):
            call()
        assert (cache.length(a), cache.length(b), cache.book.used()) == (10, 40, 4)
        check_book(cache.book)


def test_padding_rows_are_zeros(monkeypatch):
    """Rows behind the step's tokens, which no kernel writes, come out as zeros where the cache makes the result: what goes on
    through a layer (its projection, the next one's router) is not what the memory held before."""
    cache = HBMKVCache(1, 4, 2, 64, 16, device="cpu")
    step = cache.step([cache.new(), cache.new()], [3, 2])
    outs = []

    def attend(pages, layer, q, *args, out=None, **kw):
        out = torch.full(q.shape, float("nan"), dtype=q.dtype) if out is None else out  # memory that held something else
        outs.append(out)
        out[:5] = 1.0
        return out
    monkeypatch.setattr("gguf.hbm_cache.kv_attend", attend)
    wide = torch.zeros(8, 4, 128, dtype=torch.bfloat16)
    for q in (wide[:5, :, :64], wide[:8, :, :64], wide[:8, :, :64].contiguous()):
        got = cache.attend(0, step, q)
        assert got is outs.pop() and got.shape == q.shape and got.is_contiguous()
        assert (got[:5] == 1).all() and (got[5:] == 0).all()
    mine = torch.full((8, 4, 64), 7.0, dtype=torch.bfloat16)
    assert cache.attend(0, step, wide[..., :64], out=mine) is mine and (mine[5:] == 7).all()  # the caller's own stay


class FakeStreams:
    """Streams as clocks: what each one's work so far is known to come after. Every call of the cache is checked against all before
    it: a write comes after everything, a read after every write."""

    def __init__(self):
        self.current, self.capturing, self.clocks, self.log, self.held = 0, False, {}, [], []

    def stream(self, raw):
        outer = self

        class Stream:
            cuda_stream = raw

            def wait_stream(self, other):
                mine, theirs = (outer.clocks.setdefault(s, {}) for s in (raw, other.cuda_stream))
                for s, t in theirs.items():
                    mine[s] = max(mine.get(s, 0), t)
        return Stream()

    def work(self, writes):
        if self.capturing:
            return
        clock = self.clocks.setdefault(self.current, {})
        for s, t, wrote in self.log:
            assert not (writes or wrote) or clock.get(s, 0) >= t, f"stream {self.current} does not wait for stream {s}"
        clock[self.current] = clock.get(self.current, 0) + 1
        self.log.append((self.current, clock[self.current], writes))


@pytest.mark.parametrize("seed", range(6))
def test_calls_on_several_streams_keep_their_order(monkeypatch, seed):
    """Pages that a call reads or writes are another call's before it, which the caller cannot see (forks share them, freed ones are
    used again): work on one cache is ordered as its calls are, whatever streams they come on; reads beside reads are not."""
    rng, fake = random.Random(seed), FakeStreams()
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: fake.current, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index=None: fake.stream(fake.current))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: fake.capturing)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: fake.held.append((t, s.cuda_stream)))
    monkeypatch.setattr("gguf.hbm_cache.kv_append", lambda *args, **kw: fake.work(True))
    monkeypatch.setattr("gguf.hbm_cache.kv_attend", lambda *args, **kw: fake.work(False))
    monkeypatch.setattr("gguf.hbm_cache.kv_copy", lambda pages, src, dst: fake.work(True) if len(src) else None)
    empty = hip.KVPages.empty

    def made(*args):
        pages = empty(*args[:-1], device="cpu")
        pages.index = 0
        fake.work(True)  # the zeros
        return pages
    monkeypatch.setattr("gguf.hbm_cache.KVPages.empty", made)
    cache = HBMKVCache(1, 400, 2, 64, 16)
    live, steps, x = [], [], torch.zeros(64, 2, 64, dtype=torch.bfloat16)
    for _ in range(300):
        fake.current = rng.choice((0, 0, 11, 22, 33)) if rng.random() < 0.5 else fake.current
        fake.capturing = rng.random() < 0.1
        what = rng.choice(("step", "append", "attend", "attend", "attend", "fork", "free", "compact", "refresh"))
        if fake.capturing and what in ("step", "compact", "refresh"):
            continue
        if what == "step" or not steps:
            if fake.capturing:
                continue
            live.append(cache.new() if not live or rng.random() < 0.5 else cache.fork(rng.choice(live)))
            step = cache.step(live[-1:], [rng.randint(1, 20)], width=100)
            steps = steps[-3:] + [(step, live[-1], fake.current)]
        elif what == "append":
            cache.append(0, rng.choice(steps)[0], x, x)
        elif what == "attend":
            step, _, made_on = rng.choice(steps)
            cache.attend(0, step, x)
            if fake.current != made_on and not fake.capturing:  # its tables are not to be used again before this is done
                for t in (step.table, step.start, step.length, step.cu):
                    assert any(u is t and s == fake.current for u, s in fake.held)
        elif what == "refresh":
            step, seq, _ = rng.choice(steps)
            if seq in live and cache.length(seq) < 1000:
                cache.refresh(step, [seq], step.counts)
                fake.work(True)  # the graph's replay, on this stream
        elif what == "fork" and live:
            live.append(cache.fork(rng.choice(live)))
        elif what == "free" and len(live) > 4:
            cache.free(live.pop(rng.randrange(len(live))))
        elif what == "compact":
            cache.compact()
    # two streams that only read wait for the last write, not for each other
    fake.capturing, fake.current = False, 0
    step = cache.step([live[-1]], [1])
    cache.append(0, step, x, x)
    for fake.current in (11, 22, 11, 22):
        cache.attend(0, step, x)
    assert fake.clocks[11].get(22, 0) < fake.log[-1][1] and fake.clocks[22].get(11, 0) < fake.log[-2][1]


def test_a_step_that_was_not_run_is_taken_back():
    """Where a layer fails, truncating to the lengths before it takes the step back: the book is as after that, whether pages were
    begun, filled or copied for it, and the next step writes the same positions."""
    book = PageBook(12, 16)
    c = Contents(book)
    a, b = book.new(), book.new()
    c.want[a], c.want[b] = [], []
    c.grow([a], [20], 0)
    f = book.fork(a)
    c.want[f] = list(c.want[a])
    before = {s: book.length(s) for s in (a, b, f)}
    for counts in ((1, 40, 13), (12, 16, 1)):
        c.copy(*book.grow([a, b, f], list(counts)))  # and nothing is written
        for s, n in zip((a, b, f), counts):
            book.truncate(s, book.length(s) - n)
        assert {s: book.length(s) for s in (a, b, f)} == before
        check_book(book)
        c.check()
    c.grow([a, b, f], [3, 3, 3], 1)
    c.check()
    check_book(book)


def test_rotary_frequencies_stay_in_64_bits():
    """Frequencies given as plain numbers: a fp32 one is off by 2^-25 of itself, 3e-3 of a turn's angle at position 10^6."""
    want = [0.1, 1 / 3, 7e-5, 1.0]
    for given in (want, tuple(want), torch.tensor(want, dtype=torch.float64), __import__("numpy").array(want)):
        assert Rotary(8, 8, inv_freq=given, device="cpu").inv_freq.tolist() == want


@pytest.mark.parametrize("width", [2.5, 4.0, "4", 1 << 40])
def test_widths_that_make_no_table(width):
    """No table comes of such a width: nothing is counted."""
    cache = HBMKVCache(1, 8, 2, 64, 16, device="cpu")
    a = cache.new()
    cache.step([a], [3])
    with pytest.raises((TypeError, ValueError, MemoryError)):
        cache.step([a], [20], width=width)
    assert cache.length(a) == 3 and cache.book.used() == 1
    check_book(cache.book)


def test_rope_results_apart_from_the_other_tensor():
    """q's result where k is read or written, or k's where q is read, would be read or written in no order."""
    lib, sections = hip.library(), (ctypes.c_int32 * 1)(16)

    def call(q, k):
        q, k = (hip.WlRopeTensor(a, b, 256, 64, 256, 64, 4, 0) for a, b in (q, k))
        return lib.wl_rope(q, k, 1, 4, 64, 32, FAKE + 4, 4, FAKE, 1, sections, 1, 1.0, None)
    a, b, c, d = (FAKE * i for i in (1, 2, 3, 4))
    for q, k in (((a, b), (c, b)), ((a, b), (b, c)), ((a, b), (c, a)), ((a, a), (a, a)), ((a, a), (a, b)), ((a, b), (a, a))):
        assert call(q, k) == -11
    for q, k in (((a, b), (c, d)), ((a, a), (b, b)), ((a, a), (b, c)), ((a, b), (a, c))):
        assert call(q, k) == -4  # the positions, which are looked at last
