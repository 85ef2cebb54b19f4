"""Drafts and sliding windows without a GPU: what the C ABI and the Python side refuse, the page book's part in keeping accepted
tokens, the oracle's own pieces."""
import ctypes
import math
import random

import pytest
import torch

from engines.qwen36 import HipAttention, Rotary
from engines.qwen36.attention_hip import head_norm
from gguf import hip
from gguf.hbm_cache import HBMKVCache, PageBook
from oracle import kv_ref
from test_kv_cpu import BAD_BATCHES, BAD_CACHES, FAKE, batch_struct, cache_struct


def masked(cache=None, batch=None, layer=0, q=FAKE, heads=4, length=FAKE, bound=64, scale=0.125, out=FAKE, ws=None, n=0, **mask):
    m = hip.WlKvMask(None, 0, 0, 0)
    for name, v in mask.items():
        setattr(m, name, v)
    c, b = ctypes.byref(cache or cache_struct()), ctypes.byref(batch or batch_struct())
    return hip.library().wl_kv_attend_masked(c, layer, q, 256, 64, heads, b, length, bound, scale, ctypes.byref(m), out, ws, n, None)


def tree(batch=None, parents=FAKE, start=FAKE, out=FAKE, words=1, positions=FAKE):
    return hip.library().wl_kv_tree(ctypes.byref(batch or batch_struct(table=None)), parents, start, out, words, positions, None)


def keep(cache=None, batch=None, start=FAKE, kept=FAKE):
    return hip.library().wl_kv_keep(ctypes.byref(cache or cache_struct()), ctypes.byref(batch or batch_struct()), start, kept, None)


def test_struct_layout():
    assert hip.library().wl_abi_version() & 0xFFFF >= 5
    assert ctypes.sizeof(hip.WlKvMask) == 32


@pytest.mark.parametrize("over,code", BAD_CACHES)
def test_bad_caches(over, code):
    cache = cache_struct(**over)
    assert masked(cache, window=5) == keep(cache) == code
    m = hip.WlKvMask(None, 0, 5, 0)
    assert hip.library().wl_kv_attend_masked_workspace_bytes(ctypes.byref(cache), 4, ctypes.byref(batch_struct()), 64, ctypes.byref(m)) == 0


@pytest.mark.parametrize("over,code", BAD_BATCHES)
def test_bad_batches(over, code):
    batch = batch_struct(**over)
    assert masked(batch=batch, window=5) == keep(batch=batch) == code
    if not any(n.startswith("table") for n in over):
        assert tree(batch_struct(**{"table": None, "table_width": -5, "table_stride": 0, **over})) == code


def test_bad_masks():
    for bad in (dict(window=-1), dict(window=5, sinks=-1), dict(sinks=-1), dict(tree=FAKE, tree_stride=0), dict(tree=FAKE, tree_stride=1 << 31),
                dict(tree=FAKE, tree_stride=1, window=2)):  # max_count is 3
        assert masked(**bad) == -2, bad
    assert masked(tree=FAKE + 4, tree_stride=1) == -4
    wide = batch_struct(tokens=100, max_count=65)
    assert masked(batch=wide, tree=FAKE, tree_stride=1) == -2
    ok = dict(window=5, sinks=2)
    assert masked(q=None, **ok) == masked(length=None, **ok) == masked(out=None, **ok) == -3
    assert masked(q=FAKE + 1, **ok) == masked(out=FAKE + 8, **ok) == masked(length=FAKE + 1, **ok) == -4
    assert masked(heads=3, **ok) == masked(bound=-1, **ok) == masked(scale=math.nan, **ok) == masked(layer=2, **ok) == -2
    assert masked(out=FAKE, **ok) == -11  # q's memory
    long = batch_struct(table_width=64, table_stride=64)

    def need(**m):
        return hip.library().wl_kv_attend_masked_workspace_bytes(ctypes.byref(cache_struct()), 4, ctypes.byref(long), 1024,
                                                                 ctypes.byref(hip.WlKvMask(*m.values())))
    assert need(tree=None, stride=0, window=-1, sinks=0) == 0
    whole = need(tree=None, stride=0, window=0, sinks=0)
    assert whole == hip.library().wl_kv_attend_workspace_bytes(ctypes.byref(cache_struct()), 4, ctypes.byref(long), 1024) > 0
    assert need(tree=FAKE, stride=1, window=0, sinks=0) == whole and need(tree=None, stride=0, window=100, sinks=4) < whole
    assert masked(batch=long, bound=1024, window=1000) == masked(batch=long, bound=1024, ws=FAKE + 4, n=1 << 30, window=1000) == -6


@pytest.mark.parametrize("window,before,heads,cut", [
    (1024, 4096, 16, False), (1024, 0, 16, False), (3000, 0, 16, False), (3000, 1024, 16, False), (3584, 0, 16, True), (3840, 0, 16, True),
    (3840, 1024, 16, False), (3840, 10 ** 6, 16, False), (3840, 0, 32, False)])
def test_windowed_prompts_that_are_cut(window, before, heads, cut):
    """4096 tokens on two heads are one round of row tiles with 16 query heads: they are cut where the first rows' windows are so far from
    full that the last row tile would run on alone."""
    cache = cache_struct(kv_heads=2, head_dim=256, page_tokens=64, pages=1 << 20)
    width = -(-(4096 + before) // 64)
    batch = batch_struct(tokens=4096, max_count=4096, seqs=1, table_width=width, table_stride=width)
    need = hip.library().wl_kv_attend_masked_workspace_bytes(ctypes.byref(cache), heads, ctypes.byref(batch), 4096 + before,
                                                             ctypes.byref(hip.WlKvMask(None, 0, window, 4)))
    assert (need > 0) == cut


def test_bad_trees():
    assert tree(parents=None) == tree(start=None) == tree(out=None) == tree(positions=None) == tree(batch_struct(cu=None)) == -3
    assert tree(parents=FAKE + 2) == tree(start=FAKE + 2) == tree(out=FAKE + 4) == tree(positions=FAKE + 4) == -4
    assert tree(words=0) == tree(batch_struct(tokens=100, max_count=65)) == tree(words=1 << 31) == tree(words=1 << 62) == -2
    assert hip.library().wl_kv_tree(None, FAKE, FAKE, FAKE, 1, FAKE, None) == -3


def test_bad_keeps():
    assert keep(start=None) == keep(kept=None) == -3 and keep(start=FAKE + 2) == keep(kept=FAKE + 1) == -4


def test_bad_norm_rope():
    def call(qw=FAKE, kw=None, wtype=0, eps=1e-6, dtype=1, tokens=4, q={}, k=None, sections=(6, 5, 5)):  # noqa: B006
        def tensor(over):
            t = hip.WlRopeTensor(FAKE, FAKE, 256, 64, 256, 64, 4, 0)
            for n, v in over.items():
                setattr(t, n, v)
            return ctypes.byref(t)
        return hip.library().wl_norm_rope(tensor(q), None if k is None else tensor(k), dtype, tokens, 64, 32, FAKE, 4, FAKE, 3,
                                          (ctypes.c_int32 * len(sections))(*sections), 1, 1.0, qw, kw, wtype, eps, 1, None)
    assert call(dtype=2) == call(wtype=2) == -7 and call(q={"in_": None}) == call(k={"out": None}) == -3
    assert call(qw=FAKE + 2) == call(kw=FAKE + 2) == call(wtype=1, kw=FAKE + 1) == call(q={"in_": FAKE + 1}) == -4
    assert call(eps=-1e-6) == call(eps=math.nan) == call(eps=math.inf) == call(tokens=0) == call(sections=(6, 5, 4)) == -2
    assert call(k={}) == -11 and call(q={"out_token_stride": 32}) == -2


# -- the Python side -------------------------------------------------------------------------------------------------


def test_attend_mask_checks(monkeypatch):
    z, i = torch.zeros, dict(dtype=torch.int32)
    p = hip.KVPages.empty(1, 4, 2, 64, 16, device="cpu")
    q, table, length, cu = z(70, 4, 64, dtype=torch.bfloat16), z(1, 2, **i), z(1, **i), z(2, **i)
    got = []
    monkeypatch.setattr("gguf.hip.kv._launch", lambda index, call, *args: got.extend(a for a in args if isinstance(a, hip.WlKvMask)))
    good = z(70, 2, dtype=torch.int64)
    for bad in (dict(window=0), dict(window=-1), dict(window=5, sinks=-1), dict(sinks=3), dict(window=5, causal=False),
                dict(tree=good, causal=False), dict(tree=good, sinks=2), dict(tree=good.int()), dict(tree=good[:69]), dict(tree=good[:, :1]),
                dict(tree=good[:, 0]), dict(tree=z(70, 4, dtype=torch.int64)[:, ::2]), dict(tree=z(1, 2, dtype=torch.int64).expand(70, 2)),
                dict(tree=good, window=69), dict(tree=[[1, 0]] * 70)):
        with pytest.raises(ValueError):
            hip.kv_attend(p, 0, q, table, length, cu, **bad)
    with pytest.raises(TypeError):
        hip.kv_attend(p, 0, q, table, length, cu, window=5.5)
    assert not got
    hip.kv_attend(p, 0, q, table, length, cu, window=10 ** 15, sinks=10 ** 15, tree=z(70, 9, dtype=torch.int64)[:, 3:5])
    assert got[0].tree_stride == 9 and got[0].window == got[0].sinks == 2 ** 31
    hip.kv_attend(p, 0, q, table, length, cu, tree=good[:, :1], max_count=64, window=64)
    assert got[1].tree_stride == 2 and got[1].window == 64
    hip.kv_attend(p, 0, q, table, length, cu)
    assert len(got) == 2


def test_a_window_over_several_trees_goes_by_max_count(monkeypatch):
    z, i = torch.zeros, dict(dtype=torch.int32)
    p = hip.KVPages.empty(1, 4, 2, 64, 16, device="cpu")
    args = (p, 0, z(128, 4, 64, dtype=torch.bfloat16), z(2, 2, **i), z(2, **i), z(3, **i))
    launched = []
    monkeypatch.setattr("gguf.hip.kv._launch", lambda *a: launched.append(a))
    with pytest.raises(ValueError, match="128 tokens.*max_count"):
        hip.kv_attend(*args, tree=z(128, 2, dtype=torch.int64), window=100)
    with pytest.raises(ValueError, match="2 words.*max_count 128"):
        hip.kv_attend(*args, tree=z(128, 1, dtype=torch.int64), window=100)
    assert not launched
    hip.kv_attend(*args, tree=z(128, 1, dtype=torch.int64), window=100, max_count=64)
    assert len(launched) == 1


def test_tree_and_keep_checks():
    z, i = torch.zeros, dict(dtype=torch.int32)
    p = hip.KVPages.empty(1, 4, 2, 64, 16, device="cpu")
    for parents, start, cu in ((z(4), z(1, **i), z(2, **i)), (z(4, 1, **i), z(1, **i), z(2, **i)), (z(4, **i), z(1), z(2, **i)),
                               (z(4, **i), z(1, **i), z(3, **i)), (z(8, **i)[::2], z(1, **i), z(2, **i)), (z(4, **i), z(2, **i)[::2], z(2, **i)),
                               ([0], z(1, **i), z(2, **i))):
        with pytest.raises(ValueError):
            hip.kv_tree(parents, start, cu)
    with pytest.raises(ValueError):
        hip.kv_tree(z(4, **i), z(1, **i), z(2, **i), max_count=-1)
    with pytest.raises(ValueError, match="GPU"):
        hip.kv_tree(z(4, **i), z(1, **i), z(2, **i))
    assert [t.shape[0] for t in hip.kv_tree(z(0, **i), z(1, **i), z(2, **i))] == [0, 0]
    for kept, table, start, cu in ((z(3), z(1, 2, **i), z(1, **i), z(2, **i)), (z(6, **i)[::2], z(1, 2, **i), z(1, **i), z(2, **i)),
                                   (z(3, **i), z(1, 2), z(1, **i), z(2, **i)), (z(3, **i), z(1, 2, **i), z(2, **i), z(2, **i)),
                                   (z(3, **i), z(1, 2, **i), z(1, **i), z(3, **i)), (z(3, 1, **i), z(1, 2, **i), z(1, **i), z(2, **i))):
        with pytest.raises(ValueError):
            hip.kv_keep(p, table, start, kept, cu)
    with pytest.raises(ValueError, match="GPU"):
        hip.kv_keep(p, z(1, 2, **i), z(1, **i), z(3, **i), z(2, **i))


# -- keeping some of a step's tokens ---------------------------------------------------------------------------------


def test_book_moves():
    book = PageBook(10, 16)
    a, b, c = book.new(), book.new(), book.new()
    book.grow([a, b, c], [40, 20, 3])
    assert book.moves([a, b, c], [20, 5, 0], [[0, 4, 18], [0, 1, 2], []]) == [([1, 2], 4, [0, 4, 18])]
    assert book.moves([a], [8], [[7]]) == [([2], 0, [7])] and book.moves([], [], []) == []
    f = book.fork(a)
    assert book.moves([a, f], [20, 8], [[0, 1], []]) == []  # nothing moves
    for s in (a, f):
        with pytest.raises(ValueError, match="another"):
            book.moves([s], [8], [[1]])
    book.grow([f], [1])  # takes a copy of the last page, of which the other sequence is left alone
    assert book.moves([a, f], [8, 9], [[1], [2, 3]]) == [([2], 0, [1]), ([6], 0, [2, 3])]
    with pytest.raises(ValueError, match="another"):
        book.moves([a], [10], [[2, 3]])
    before = str(vars(book))
    for bad in (([a, a], [1, 1], [[], []]), ([a], [1, 2], [[]]), ([a], [1], []), ([a], [41], [[]]), ([a], [-1], [[]]), ([a], [5], [[5]]),
                ([a], [5], [[-1]]), ([a], [5], [[1, 1]]), ([a], [5], [[2, 1]]), ([a], [5], [[0.5]]), ([a], [2.5], [[0]]), ([a], [5], ["12"])):
        with pytest.raises(ValueError):
            book.moves(*bad)
    with pytest.raises(KeyError):
        book.moves([77], [0], [[]])
    assert str(vars(book)) == before


@pytest.mark.parametrize("seed", range(4))
def test_cache_keeps(seed, monkeypatch):
    """HBMKVCache.keep over random lives of sequences, on a cache of the CPU whose kernels are written out: what each sequence reads
    is what was kept for it."""
    rng = random.Random(seed)
    cache = HBMKVCache(1, 40, 1, 64, 16, device="cpu")
    held = [[None] * 16 for _ in range(40)]

    def move(pages, table, start, kept, cu, max_count=None):
        assert pages is cache.pages and all(t.dtype is torch.int32 for t in (table, start, kept, cu))
        lists = [kept[int(cu[b]):int(cu[b + 1])].tolist() for b in range(len(start))]
        assert max_count == max(map(len, lists))
        for row, first, mine in zip(table.tolist(), start.tolist(), lists):
            place = lambda t: (row[t // 16], t % 16)  # noqa: E731
            read = [held[p][t] for p, t in (place(first + j) for j in mine)]
            for i, x in enumerate(read):
                p, t = place(first + i)
                held[p][t] = x

    def copy(pages, src, dst):
        for a, b in zip(src, dst):
            held[b] = list(held[a])
    monkeypatch.setattr("gguf.hbm_cache.kv_keep", move)
    monkeypatch.setattr("gguf.hbm_cache.kv_copy", copy)
    want = {cache.new(): [] for _ in range(3)}
    for i in range(200):
        live = list(want)
        what = rng.choice(("draft", "draft", "draft", "fork", "free", "compact"))
        if what == "draft":
            seqs = rng.sample(live, rng.randint(1, min(3, len(live))))
            counts = [rng.choice((0, 1, 7, 16, 30)) for _ in seqs]
            if cache.book.used() > 25:
                continue
            cache.step(seqs, counts)
            for s, n in zip(seqs, counts):
                length, pages = cache.book.sequences[s]
                for t in range(length - n, length):
                    held[pages[t // 16]][t % 16] = (i, s, t)
            kept = [sorted(rng.sample(range(n), rng.randint(0, n))) for n in counts]
            for s, n, k in zip(seqs, counts, kept):
                first = cache.length(s) - n
                want[s] = want[s] + [(i, s, first + j) for j in k]
            cache.keep(seqs, counts, kept)
        elif what == "fork" and len(live) < 5:
            s = rng.choice(live)
            want[cache.fork(s)] = list(want[s])
        elif what == "free" and len(live) > 2:
            s = rng.choice(live)
            cache.free(s)
            del want[s]
        elif what == "compact":
            cache.compact()
        for s, tokens in want.items():
            length, pages = cache.book.sequences[s]
            assert [held[pages[t // 16]][t % 16] for t in range(length)] == tokens and len(pages) == -(-length // 16)


def test_cache_keep_refuses_before_it_moves(monkeypatch):
    cache = HBMKVCache(1, 8, 1, 64, 16, device="cpu")
    a, b = cache.new(), cache.new()
    cache.step([a, b], [20, 20])
    monkeypatch.setattr("gguf.hbm_cache.kv_keep", lambda *args, **kw: pytest.fail("moved"))
    for bad in (([a, b], [10, 10], [[1], [3, 2]]), ([a], [21], [[1]]), ([a, a], [1, 1], [[], []])):
        with pytest.raises(ValueError):
            cache.keep(*bad)
    assert cache.length(a) == cache.length(b) == 20
    cache.keep([a, b], [10, 4], [[0, 1, 2], []])  # nothing moves
    assert cache.length(a) == 13 and cache.length(b) == 16

    def fails(*args, **kw):
        raise RuntimeError("the device")
    monkeypatch.setattr("gguf.hbm_cache.kv_keep", fails)
    with pytest.raises(RuntimeError):
        cache.keep([a, b], [5, 4], [[1], [0]])
    assert cache.length(a) == 13 and cache.length(b) == 16


def test_cache_passes_masks_on(monkeypatch):
    cache = HBMKVCache(1, 8, 2, 64, 16, device="cpu")
    step = cache.step([cache.new()], [3])
    seen = []
    monkeypatch.setattr("gguf.hbm_cache.kv_attend", lambda *args, **kw: seen.append(kw))
    monkeypatch.setattr("gguf.hbm_cache.kv_tree", lambda *args, **kw: seen.append((args, kw)))
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    cache.attend(0, step, q, window=7, sinks=2, tree="masks")
    assert (seen[0]["window"], seen[0]["sinks"], seen[0]["tree"]) == (7, 2, "masks")
    parents = torch.zeros(3, dtype=torch.int32)
    cache.tree(step, parents)
    assert seen[1] == ((parents, step.start, step.cu), dict(max_count=3))
    with pytest.raises(ValueError, match="3 tokens"):
        cache.tree(step, parents[:2])


# -- the oracle's own pieces -----------------------------------------------------------------------------------------


def test_oracle_masks():
    masks, positions = kv_ref.tree([-1, 0, 0, 2, -1, 5], [7], [0, 6], 1)
    assert [kv_ref.drafted(m, 6) for m in masks] == [[0], [0, 1], [0, 2], [0, 2, 3], [4], [5]]
    assert positions.tolist() == [7, 8, 8, 9, 7, 7]
    g = torch.Generator().manual_seed(0)
    k, v = torch.randint(-127, 128, (4, 1, 16, 64), generator=g).to(torch.int8), torch.randint(-127, 128, (4, 1, 64, 16), generator=g).to(torch.int8)
    one = torch.ones(4, 1) / 50
    q = torch.randn(6, 1, 64, generator=g).to(torch.bfloat16)
    args = (k, v, one, one, q, torch.arange(4)[None], torch.tensor([50]), torch.tensor([0, 6]))
    plain, _ = kv_ref.attend(*args)
    chain = torch.tensor([[(2 << i) - 1] for i in range(6)])
    assert torch.equal(kv_ref.attend(*args, tree=chain)[0], plain) and torch.equal(kv_ref.attend(*args, window=50)[0], plain)
    assert torch.equal(kv_ref.attend(*args, window=10, sinks=40)[0], plain)
    short, _ = kv_ref.attend(*args, window=1)
    assert torch.allclose(short[2, 0], v[2, 0, :, 14].double() / 50 * one.double()[0, 0] * 50)  # the row's own token alone


def test_oracle_keep_and_norm():
    g = torch.Generator().manual_seed(1)
    pool = torch.randint(-127, 128, (1, 2, 1, 16, 64), generator=g).to(torch.int8)
    scale = torch.tensor([[[0.5], [0.25]]])
    out, now = kv_ref.keep(pool, scale, torch.tensor([[0, 1]]), [10], [0, 3, 12], [0, 3], 16)
    assert torch.equal(now, scale.double()) and torch.equal(out[0, 0, 0, 11], pool[0, 0, 0, 13].double())
    assert torch.equal(out[0, 0, 0, 12], (pool[0, 1, 0, 6].double() / 2).round())
    assert torch.equal(out[0, 0, 0, 13:], pool[0, 0, 0, 13:].double()) and torch.equal(out[0, 1], pool[0, 1].double())
    x = torch.randn(3, 2, 8, generator=g, dtype=torch.float64)
    y = kv_ref.norm(x, torch.zeros(8), 0.0)
    assert torch.allclose(y.square().mean(-1), torch.ones(3, 2, dtype=torch.float64))
    assert torch.allclose(kv_ref.norm(x, torch.full((8,), 3.0), 0.0, False), 3 * y)


def test_rotary_has_normed():
    assert callable(Rotary(64, device="cpu").normed)


def test_a_rotary_of_its_own_turns_behind_the_norms():
    class Reversed(Rotary):
        def __call__(self, q, k, positions):
            return q.flip(-1), k.flip(-1)

    gen = torch.Generator().manual_seed(5)
    q, k = (torch.randn(3, n, 64, generator=gen).bfloat16() for n in (4, 2))
    wq, wk = (torch.randn(64, generator=gen) for _ in range(2))
    got = Reversed(64, device="cpu").normed(q, k, torch.arange(3), wq, wk, 1e-6)
    for g, x, w in zip(got, (q, k), (wq, wk)):
        assert torch.equal(g, head_norm(x, w, 1e-6).flip(-1))


@pytest.mark.parametrize("q_shape,k_shape", [((1, 64), (1, 64)), ((1,), (1,)), ((4, 64), (2, 64)), ((), (64,)), ((64,), (2, 64)), ((64,), (64,))])
def test_norm_weights_of_any_shape(q_shape, k_shape, monkeypatch):
    """Weights that head_norm takes are taken behind Rotary.normed too; [head_dim] alone in one pass."""
    gen = torch.Generator().manual_seed(6)
    q, k = (torch.randn(3, n, 64, generator=gen).bfloat16() for n in (4, 2))
    wq, wk = (torch.randn(shape, generator=gen) for shape in (q_shape, k_shape))
    monkeypatch.setattr("engines.qwen36.attention_hip.rope", lambda q, k, *args, **kw: (q.flip(-1), k.flip(-1)))
    monkeypatch.setattr("engines.qwen36.attention_hip.norm_rope", lambda *args, **kw: "one pass")
    got = Rotary(64, device="cpu").normed(q, k, torch.arange(3), wq, wk, 1e-6)
    if q_shape == k_shape == (64,):
        assert got == "one pass"
    else:
        assert all(torch.equal(g, head_norm(x, w, 1e-6).flip(-1)) for g, x, w in zip(got, (q, k), (wq, wk)))


def test_a_rotary_that_passes_attributes_on_turns_behind_the_norms(monkeypatch):
    """A wrapper that looks every other attribute up in a Rotary has a `normed` by that, which knows nothing of the wrapper's rotation."""
    class Shifted:
        def __init__(self, inner):
            self.inner = inner

        def __getattr__(self, name):
            return getattr(self.inner, name)

        def __call__(self, q, k, positions):
            return q + positions.sum(), k - positions.sum()

    gen = torch.Generator().manual_seed(7)
    p, dim = "layers.0.self_attn", 64
    weights = {f"{p}.{n}_proj.weight": torch.randn(rows, 32, generator=gen).bfloat16() for n, rows in (("q", 4 * dim), ("k", 2 * dim), ("v", 2 * dim))}
    weights[f"{p}.o_proj.weight"] = torch.randn(32, 4 * dim, generator=gen).bfloat16()
    weights.update({f"{p}.{n}_norm.weight": torch.randn(dim, generator=gen) for n in "qk"})
    eng = HipAttention()
    eng.prefix, eng.weights, eng.rotary = "", weights, Shifted(Rotary(dim, device="cpu"))
    cache = eng.kv_cache = HBMKVCache(1, 4, 2, dim, 16, device="cpu")
    seen = {}
    monkeypatch.setattr(cache, "append", lambda layer, step, k, v: seen.update(k=k))
    monkeypatch.setattr(cache, "attend", lambda layer, step, q, **kw: seen.setdefault("q", q))
    monkeypatch.setattr("engines.qwen36.attention_hip.norm_rope", lambda q, k, *args, **kw: (q, k))
    x, positions = torch.randn(3, 32, generator=gen).bfloat16(), torch.tensor([[1, 2, 3]])
    eng.hip_attention(x, 0, 0, cache.step([cache.new()], [3]), positions)
    for name, heads, sign in (("q", 4, 1), ("k", 2, -1)):
        y = torch.nn.functional.linear(x, weights[f"{p}.{name}_proj.weight"]).view(3, heads, dim)
        assert torch.equal(seen[name], head_norm(y, weights[f"{p}.{name}_norm.weight"], 1e-6) + sign * 6)


def test_book_moves_past_a_shared_page():
    """A page that another sequence has too, in which the first kept tokens just stay, is left out of what moves."""
    book = PageBook(10, 16)
    a = book.new()
    book.grow([a], [8])
    book.grow([a], [40])  # drafts, from the middle of page 0 to the end of page 2
    f = book.fork(a)
    book.truncate(f, 16)  # has page 0 alone
    stay = list(range(8))
    assert book.moves([a], [40], [stay + [10, 11, 39]]) == [([1, 2], 0, [2, 3, 31])]
    assert book.moves([a], [40], [stay + [8, 11, 39]]) == [([1, 2], 0, [0, 3, 31])]
    assert book.moves([a], [40], [list(range(24)) + [30]]) == [([2], 0, [6])]
    for kept in ([0, 2], [1], stay[:7] + [8]):
        with pytest.raises(ValueError, match="another"):
            book.moves([a], [40], [kept])
    book.truncate(f, 0)
    assert book.moves([a], [40], [[0, 2]]) == [([0, 1, 2], 8, [0, 2])]
