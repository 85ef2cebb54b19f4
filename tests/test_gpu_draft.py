"""What decoding with drafts and sliding windows takes of the attention half, on the GPU: attention with a window and sinks,
attention for drafted trees, the trees' masks and positions, accepted tokens moved up in the cache bit for bit, norms with rotary
positions; against oracle/kv_ref.py in 64 bits."""
import math
import random

import numpy as np
import pytest
import torch

from oracle import kv_ref
from test_gpu_kv import cu_of, gen, i32, random_pages, table_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.int8, torch.float8_e4m3fn]
SHAPES = [  # q heads, kv heads, dim, page
    (16, 2, 256, 64), (32, 8, 128, 32), (8, 8, 64, 16), (6, 1, 64, 128), (3, 1, 256, 32), (20, 1, 128, 64)]


def check_masked(hip, pages, layer, q, table, length, cu, rows=None, **kw):
    """kv_attend against the oracle: every row, or just `rows` where all would take the oracle long (each as a call of its own)."""
    cache = [t[layer].cpu() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    assert hip.kv_attend(pages, layer, q, table, length, cu, out=out, **kw) is out
    torch.cuda.synchronize()
    got, bounds = out.cpu().double(), cu.cpu().tolist()
    ref = {n: kw[n] for n in ("scale", "window", "sinks") if n in kw}
    if rows is not None:
        for b, i in rows:
            n = bounds[b + 1] - bounds[b]
            at = bounds[b] + i
            want, tol = kv_ref.attend(*cache, q[at:at + 1].cpu(), table[b:b + 1].cpu(), length[b:b + 1].cpu() - (n - 1 - i), torch.tensor([0, 1]), **ref)
            assert ((got[at] - want[0]).abs() <= tol[0]).all(), (b, i)
        return out
    if "tree" in kw:
        ref["tree"] = kw["tree"].cpu()
    want, tol = kv_ref.attend(*cache, q.cpu(), table.cpu(), length.cpu(), cu.cpu(), max_count=kw.get("max_count"), **ref)
    owned = torch.zeros(q.shape[0], dtype=torch.bool)
    for b in range(len(bounds) - 1):
        lo = min(max(bounds[b], 0), q.shape[0])
        owned[lo:lo + min(max(bounds[b + 1], lo) - lo, q.shape[0] - lo, kw.get("max_count") or q.shape[0])] = True
    assert (got[~owned] == 7.0).all()  # rows of no sequence stay as they were
    want, got, tol = want[owned], got[owned], tol[owned]
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places than expected"
    err = torch.where(torch.isnan(want), 0.0, (got - want).abs())
    worst = float((err / (tol + 1e-300)).nan_to_num(0.0).max()) if err.numel() else 0.0
    assert (err <= tol.nan_to_num(0.0)).all(), f"off by {worst:.2f} of the bound"
    return out


# -- windows ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("counts,lengths", [((1,), (1,)), ((1, 1, 1), (65, 700, 3)), ((2, 1, 2), (130, 1, 2)), ((1, 0, 1, 1), (0, 50, 129, 257)),
                                            ((5, 33, 1), (5, 100, 190)), ((17,), (300,))])
@pytest.mark.parametrize("window,sinks", [(1, 0), (60, 4), (64, 64), (100, 130)])
def test_window(hip, dtype, heads, kv_heads, dim, page, counts, lengths, window, sinks):
    g = gen(sum(lengths) + dim + window)
    need = sum(-(-n // page) for n in lengths)
    pages = random_pages(hip, g, 2, need + 2, kv_heads, page, dim, dtype)
    table = table_of(g, lengths, page, need + 2)
    q = (1.5 * torch.randn(sum(counts), heads, dim, generator=g)).to(torch.bfloat16).to(DEV)
    check_masked(hip, pages, 1, q, table, i32(lengths), cu_of(counts), max_count=max(counts), window=window, sinks=sinks)


@pytest.mark.parametrize("count", [1, 3, 24])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (31, 32), (33, 5), (500, 0), (501, 7), (10 ** 12, 3), (5, 10 ** 12)])
def test_window_edges(hip, count, window, sinks):
    """Windows and sinks that end at tiles' and pages' ends, meet, cover everything; rows that stand before the sequence's beginning;
    lengths behind the table's pages."""
    g = gen(31)
    lengths = (500, 64 + count, 1, 1000)
    pages = random_pages(hip, g, 1, 26, 2, 64, 128, torch.int8)
    table = table_of(g, (500, 64 + count, 1, 640), 64, 26)
    q = torch.randn(4 * count, 8, 128, generator=g).to(torch.bfloat16).to(DEV)
    check_masked(hip, pages, 0, q, table, i32(lengths), cu_of([count] * 4), max_count=count, window=window, sinks=sinks)
    check_masked(hip, pages, 0, q, table, i32(lengths), cu_of([count] * 4), max_count=count, window=window, sinks=sinks, max_length=1)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32), (256, 128)])
@pytest.mark.parametrize("count", [1, 20])
def test_window_keeps_out_what_it_hides(hip, dim, page, count):
    """NaN bytes, NaN scales and missing pages between the sinks and the window reach no row: what kept pages of a sequence whose
    middle was given away may hold."""
    g = gen(32)
    length, window, sinks = 900, 100, 5
    pages = random_pages(hip, g, 1, -(-length // page) + 1, 2, page, dim, torch.float8_e4m3fn)
    table = table_of(g, (length,), page, -(-length // page) + 1)
    q = torch.randn(count, 8, dim, generator=g).to(torch.bfloat16).to(DEV)
    args = dict(max_count=count, window=window, sinks=sinks)
    want = check_masked(hip, pages, 0, q, table, i32([length]), i32([0, count]), **args)
    first = length - count + 1 - window  # that the first row sees
    raw_k, raw_v = pages.k.view(torch.uint8), pages.v.view(torch.uint8)
    for c in range(-(-length // page)):
        p, lo, hi = int(table[0, c]), max(sinks - c * page, 0), min(first - c * page, page)
        if hi > lo:
            raw_k[0, p, :, lo:hi], raw_v[0, p, :, :, lo:hi] = 0x7F, 0x7F
        if lo == 0 and hi == page:
            pages.k_scale[0, p], pages.v_scale[0, p] = math.nan, math.nan
    assert torch.equal(want, hip.kv_attend(pages, 0, q, table, i32([length]), i32([0, count]), **args))
    table[0, -(-sinks // page):first // page] = -1
    assert torch.equal(want, hip.kv_attend(pages, 0, q, table, i32([length]), i32([0, count]), **args))
    table[0, 0] = 2 ** 31 - 1  # the sinks' page itself
    check_masked(hip, pages, 0, q, table, i32([length]), i32([0, count]), **args)


def test_window_many_sequences(hip):
    g = gen(33)
    rng = np.random.default_rng(33)
    lengths = [int(x) for x in rng.integers(0, 900, 150)]
    lengths[77], lengths[149] = 5000, 3000
    counts = [int(x) for x in rng.integers(0, 3, 150)]
    need = sum(-(-n // 64) for n in lengths)
    pages = random_pages(hip, g, 1, need, 2, 64, 64, torch.int8)
    table = table_of(g, lengths, 64, need)
    q = torch.randn(sum(counts), 6, 64, generator=g).to(torch.bfloat16).to(DEV)
    args = (q, table, i32(lengths), cu_of(counts))
    a = check_masked(hip, pages, 0, *args, max_count=2, window=700, sinks=3)
    assert torch.equal(a, hip.kv_attend(pages, 0, *args, max_count=2, window=700, sinks=3))
    for bound in (1, 64, 10 ** 6):
        check_masked(hip, pages, 0, *args, max_count=2, window=700, sinks=3, max_length=bound)
    check_masked(hip, pages, 0, *args, window=300, sinks=100)  # no bound of the rows: the form for many


@pytest.mark.parametrize("heads,kv_heads,dim,counts,lengths,window,sinks", [
    (16, 2, 256, (512,), (9512,), 1000, 4), (32, 8, 128, (301, 180, 65, 256, 37), (1700, 999, 65, 1300, 437), 333, 7),
    (8, 1, 64, (700,), (30000,), 8000, 100), (4, 4, 256, (1100, 300), (1500, 5000), 77, 0), (16, 2, 256, (1,), (40000,), 20000, 64)])
def test_window_prompts(hip, heads, kv_heads, dim, counts, lengths, window, sinks):
    """Long rows and long windows, cut into pieces: rows of every part of them."""
    g = gen(34)
    need = sum(-(-n // 64) for n in lengths)
    pages = random_pages(hip, g, 1, need, kv_heads, 64, dim, torch.int8)
    table = table_of(g, lengths, 64, need)
    q = torch.randn(sum(counts), heads, dim, generator=g).to(torch.bfloat16).to(DEV)
    rows = [(b, i) for b, n in enumerate(counts) for i in sorted({0, min(1, n - 1), n // 3, n // 2, min(255, n - 1), max(n - 2, 0), n - 1})]
    check_masked(hip, pages, 0, q, table, i32(lengths), cu_of(counts), rows, max_count=max(counts), max_length=max(lengths),
                 window=window, sinks=sinks)


@pytest.mark.parametrize("window", [3500, 3800])
def test_windowed_prompt_without_history(hip, window):
    """A first prompt whose row tiles fill the CUs once, in a window nearly as long: cut into pieces; rows of every part."""
    g = gen(36)
    n = 3900
    pages = random_pages(hip, g, 1, 61, 2, 64, 64, torch.int8)
    table = table_of(g, (n,), 64, 61)
    q = torch.randn(n, 16, 64, generator=g).to(torch.bfloat16).to(DEV)
    rows = [(0, i) for i in (0, 1, 255, 1000, window - 1, window, window + 4, n - 2, n - 1)]
    args = (q, table, i32([n]), cu_of((n,)))
    out = check_masked(hip, pages, 0, *args, rows, max_count=n, max_length=n, window=window, sinks=4)
    assert torch.equal(out, hip.kv_attend(pages, 0, *args, max_count=n, max_length=n, window=window, sinks=4))


def test_window_of_everything_is_attention(hip):
    g = gen(35)
    pages = random_pages(hip, g, 1, 20, 2, 32, 128, torch.int8)
    table = table_of(g, (300, 250), 32, 20)
    for counts in ((1, 1), (40, 11)):
        q = torch.randn(sum(counts), 8, 128, generator=g).to(torch.bfloat16).to(DEV)
        args = (pages, 0, q, table, i32([300, 250]), cu_of(counts))
        check_masked(hip, *args, max_count=max(counts), window=300)
        if sum(counts) == 2:  # one form: the same bits
            assert torch.equal(hip.kv_attend(*args, max_count=1, window=300), hip.kv_attend(*args, max_count=1))


# -- trees -----------------------------------------------------------------------------------------------------------


def random_tree(rng, n, deep=0.5):
    return [-1 if i == 0 or rng.random() < 0.05 else i - 1 if rng.random() < deep else rng.randrange(i) for i in range(n)]


@pytest.mark.parametrize("counts,max_count,words,seed", [((1,), None, 1, 0), ((5, 0, 64, 3), 64, 1, 1), ((65, 2), 65, 2, 2), ((7, 300), None, 5, 3),
                                                         ((9, 4), 5, 1, 4), ((64, 64), 64, 1, 5)])
def test_tree_masks(hip, counts, max_count, words, seed):
    rng = random.Random(seed)
    parents = [p for n in counts for p in random_tree(rng, n)] + [0, 0, 0]  # padding behind
    for i in rng.sample(range(len(parents)), min(len(parents), 4)):  # no parents: itself, later ones, any number
        parents[i] = rng.choice((len(parents) + 3, -7, 2 ** 31 - 1, -2 ** 31, i))
    start = [rng.randrange(10 ** 6) for _ in counts]
    tree, positions = hip.kv_tree(i32(parents), i32(start), cu_of(counts), max_count=max_count)
    want, at = kv_ref.tree(parents, start, [0] + list(np.cumsum(counts)), -(-(max_count or len(parents)) // 64), max_count)
    assert tree.shape[1] == want.shape[1] >= words
    assert torch.equal(tree.cpu(), want) and torch.equal(positions.cpu(), at)


def test_tree_masks_of_long_drafts(hip):
    """More rows than are kept at hand: a chain, and a bush."""
    rng = random.Random(6)
    n = 4500
    parents = [i - 1 for i in range(n)] + [-1 if i == 0 else rng.randrange(max(0, i - 300), i) for i in range(n)]
    tree, positions = hip.kv_tree(i32(parents), i32([3, 10]), i32([0, n, 2 * n]), max_count=n)
    bits = torch.from_numpy(np.unpackbits(tree.cpu().numpy().view(np.uint8), axis=1, bitorder="little")).bool()
    assert torch.equal(bits[:n, :n], torch.ones(n, n, dtype=torch.bool).tril()) and not bits[:, n:].any()
    assert torch.equal(positions[:n].cpu(), 3 + torch.arange(n))
    for i in range(n, 2 * n, 97):
        line, j = [i - n], i - n
        while parents[n + j] >= 0:
            j = parents[n + j]
            line.append(j)
        assert bits[i].nonzero()[:, 0].tolist() == sorted(line) and int(positions[i]) == 10 + len(line) - 1


@pytest.mark.parametrize("cu", [(2, 5, 9), (-4, 5, 1000), (0, 9, 4)])
def test_tree_masks_out_of_range(hip, cu):
    parents = [-1, 0, 1, -1, 0, 1, 1, 0, 2, 3, 0, 1]
    tree, positions = hip.kv_tree(i32(parents), i32([100, 200]), i32(cu))
    if cu[1] <= cu[2]:
        want, at = kv_ref.tree(parents, [100, 200], cu, 1)
        assert torch.equal(tree.cpu(), want) and torch.equal(positions.cpu(), at)


@pytest.mark.parametrize("cu,known", [((0, 9, 4), (0, 4)), ((6, 2, 3), (0, 0)), ((0, 70, 10), (0, 10)), ((3, 2 ** 31 - 1, -5), (0, 0))])
def test_tree_masks_of_a_cu_that_decreases(hip, cu, known):
    """cu must not decrease. Where it does all the same: rows that one part alone has a say in are right, those behind every sequence
    zeros, and nothing is written outside."""
    import ctypes
    n, words, guard = 80, 2, 64
    parents = [-1, 0, 1, -1, 0, 1, 1, 0, 2, 3] * 8
    space = torch.full((2 * guard + n * words,), 0x5A5A5A5A, dtype=torch.int64, device=DEV)
    at = torch.full((2 * guard + n,), 0x5A5A5A5A, dtype=torch.int64, device=DEV)
    where, starts, up = i32(cu), i32([100, 200]), i32(parents)
    batch = hip.WlKvBatch(None, where.data_ptr(), 1, n, 2, 1, n, 0)
    assert hip.library().wl_kv_tree(ctypes.byref(batch), up.data_ptr(), starts.data_ptr(), space[guard:].data_ptr(), words,
                                    at[guard:].data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    for t, size in ((space, n * words), (at, n)):
        assert (t[:guard] == 0x5A5A5A5A).all() and (t[guard + size:] == 0x5A5A5A5A).all()
    tree, positions = space[guard:guard + n * words].view(n, words).cpu(), at[guard:guard + n].cpu()
    want, places = kv_ref.tree(parents, [100, 200], cu, words)
    rows = slice(*known)
    assert torch.equal(tree[rows], want[rows]) and torch.equal(positions[rows], places[rows])
    behind = min(max(max(cu), 0), n)
    assert not tree[behind:].any() and not positions[behind:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("counts,starts", [((1,), (0,)), ((2, 1, 2), (63, 0, 300)), ((5, 16, 1), (0, 100, 64)), ((17, 0, 33), (5, 9, 130)),
                                           ((64,), (200,)), ((70, 2), (0, 61))])
def test_tree(hip, dtype, heads, kv_heads, dim, page, counts, starts):
    g, rng = gen(sum(starts) + dim), random.Random(dim + sum(counts))
    lengths = [c + s for c, s in zip(counts, starts)]
    need = sum(-(-n // page) for n in lengths)
    pages = random_pages(hip, g, 2, need + 2, kv_heads, page, dim, dtype)
    table = table_of(g, lengths, page, need + 2)
    q = (1.5 * torch.randn(sum(counts), heads, dim, generator=g)).to(torch.bfloat16).to(DEV)
    parents = [p for n in counts for p in random_tree(rng, n)]
    tree, _ = hip.kv_tree(i32(parents), i32(starts), cu_of(counts), max_count=max(counts))
    check_masked(hip, pages, 1, q, table, i32(lengths), cu_of(counts), max_count=max(counts), tree=tree)


@pytest.mark.parametrize("count", [2, 16, 40, 130])
@pytest.mark.parametrize("group", [1, 4])
def test_tree_any_bits(hip, count, group):
    """Masks that no tree makes: no bit at all (with nothing before the draft: zeros), later rows, bits behind the sequence's rows,
    wider rows than needed; sequences with fewer rows than max_count; a draft of which the beginning is cut off."""
    g = gen(41)
    counts, lengths = (count, count // 2, count, 1), (count, 200, 70 + count, count // 2)
    pages = random_pages(hip, g, 1, 30, 2, 32, 64, torch.float8_e4m3fn)
    table = table_of(g, lengths, 32, 30)
    rows, words = sum(counts) + 3, -(-count // 64) + 2
    wide = torch.randint(-2 ** 63, 2 ** 63 - 1, (rows, words + 3), generator=g).to(DEV)
    wide[0] = 0
    wide[sum(counts[:3])] = 0
    q = torch.randn(rows, 2 * group, 64, generator=g).to(torch.bfloat16).to(DEV)
    out = check_masked(hip, pages, 0, q, table, i32(lengths), cu_of(counts), max_count=count, tree=wide[:, 1:words + 1])
    if count > 1:
        assert (out[0] == 0).all()
    check_masked(hip, pages, 0, q, table, i32(lengths), cu_of(counts), max_count=max(count - 1, 1), tree=wide[:, :words])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,group,window,sinks", [(1, 8, 5, 1), (4, 4, 60, 0), (16, 1, 16, 4), (40, 4, 64, 70), (70, 2, 100, 3), (16, 8, 1000, 5)])
def test_tree_in_a_window(hip, dtype, count, group, window, sinks):
    g, rng = gen(42), random.Random(count)
    counts, starts = (count, max(count // 2, 1), count), (0, 70, 700)
    lengths = [c + s for c, s in zip(counts, starts)]
    pages = random_pages(hip, g, 1, 40, 2, 32, 128, dtype)
    table = table_of(g, lengths, 32, 40)
    parents = [p for n in counts for p in random_tree(rng, n, 0.9)]
    tree, _ = hip.kv_tree(i32(parents), i32(starts), cu_of(counts), max_count=count)
    q = torch.randn(sum(counts), 2 * group, 128, generator=g).to(torch.bfloat16).to(DEV)
    check_masked(hip, pages, 0, q, table, i32(lengths), cu_of(counts), max_count=count, window=window, sinks=sinks, tree=tree)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,group", [(16, 1), (40, 1), (60, 4), (130, 4)])
def test_tree_keeps_out_what_it_hides(hip, dtype, count, group):
    """A page of drafted tokens whose scales are NaN reaches exactly the rows that see one of its tokens; pages that are not there
    nobody; a row's own page among them leaves it what is in the others."""
    g, rng = gen(45), random.Random(45)
    start = 48
    pages = random_pages(hip, g, 1, 14, 2, 16, 64, dtype)
    table = table_of(g, (start + count,), 16, 14)
    # two trees side by side: rows of one see nothing of the other
    half = count // 2
    parents = [max(i - 1 - rng.randrange(3), -1) if i < half else -1 if i == half else max(i - 1 - rng.randrange(2), half) for i in range(count)]
    tree, _ = hip.kv_tree(i32(parents), i32([start]), i32([0, count]))
    q = torch.randn(count, 2 * group, 64, generator=g).to(torch.bfloat16).to(DEV)
    args = (q, table, i32([start + count]), i32([0, count]))
    page = int(table[0, (start + half) // 16 if half % 16 == 0 else (start + half) // 16 + 1]) if half >= 16 else int(table[0, start // 16])
    for scale, head in ((pages.k_scale, 0), (pages.v_scale, 1)):
        was = float(scale[0, page, head])
        scale[0, page, head] = math.nan
        out = check_masked(hip, pages, 0, *args, tree=tree)
        if half >= 16:
            assert torch.isfinite(out[:8].float()).all() and torch.isnan(out[-1, head * group].float()).all()
        scale[0, page, head] = was
    missing = table.clone()
    missing[0, (start + count - 1) // 16], missing[0, 1] = -1, 2 ** 31 - 1
    check_masked(hip, pages, 0, q, missing, *args[2:], tree=tree)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32), (256, 128)])
@pytest.mark.parametrize("count,group,width", [(3, 4, None), (24, 1, None), (70, 2, None), (30, 8, 300), (130, 4, 300), (300, 1, 300)])
@pytest.mark.parametrize("window", [None, 400])
def test_tree_keeps_out_drafts_that_no_row_sees(hip, dim, page, count, group, width, window):
    """NaN bytes of drafted tokens whose bits no row of their sequence has, as of slots that nobody wrote, reach no row, in the form for
    few rows and in the one for many (a wide table makes the call look long)."""
    g, rng = gen(46), random.Random(46)
    counts, lengths = (count, count // 2 + 1, count), (count + 55, count // 2 + 1, count + 300)
    need = sum(-(-n // page) for n in lengths)
    pages = random_pages(hip, g, 1, need, 2, page, dim, torch.float8_e4m3fn)
    table = table_of(g, lengths, page, need, width and width * 64 // page)
    words = -(-count // 64)
    bits = torch.randint(-2 ** 63, 2 ** 63 - 1, (sum(counts), words), generator=g)
    hidden, at = [], 0
    for n in counts:
        hidden.append(sorted({0, n - 1, n // 2} | {j for j in range(n) if rng.random() < 0.3}) if n > 3 else [n - 1])
        for j in hidden[-1]:
            bits[at:at + n, j // 64] &= ~(1 << j % 64) if j % 64 < 63 else 2 ** 63 - 1
        at += n
    q = torch.randn(sum(counts), 2 * group, dim, generator=g).to(torch.bfloat16).to(DEV)
    kw = dict(max_count=count, tree=bits.to(DEV))
    if window:
        kw.update(window=window, sinks=3)
    want = hip.kv_attend(pages, 0, q, table, i32(lengths), cu_of(counts), **kw)
    for b, n in enumerate(counts):
        for j in hidden[b]:
            pos = lengths[b] - n + j
            p, t = int(table[b, pos // page]), pos % page
            pages.k.view(torch.uint8)[0, p, :, t], pages.v.view(torch.uint8)[0, p, :, :, t] = 0x7F, 0xFF if j % 2 else 0x7F
    assert torch.equal(want, hip.kv_attend(pages, 0, q, table, i32(lengths), cu_of(counts), **kw))
    if count <= 70:
        check_masked(hip, pages, 0, q, table, i32(lengths), cu_of(counts), **kw)


def test_tree_of_one_chain_is_causal(hip):
    g = gen(43)
    pages = random_pages(hip, g, 1, 20, 2, 64, 256, torch.int8)
    table = table_of(g, (500, 400), 64, 20)
    for n in (1, 2, 30):
        q = torch.randn(2 * n, 16, 256, generator=g).to(torch.bfloat16).to(DEV)
        tree, positions = hip.kv_tree(i32([i - 1 for i in range(n)] * 2), i32([500 - n, 400 - n]), cu_of((n, n)), max_count=n)
        args = (pages, 0, q, table, i32([500, 400]), cu_of((n, n)))
        out = check_masked(hip, *args, max_count=n, tree=tree)
        want, tol = kv_ref.attend(*(t[0].cpu() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)), q.cpu(), table.cpu(), i32([500, 400]).cpu(),
                                  cu_of((n, n)).cpu())
        assert ((out.cpu().double() - want).abs() <= tol).all()
        if n <= 2:  # one form: the same bits
            assert torch.equal(out, hip.kv_attend(*args, max_count=n))
        assert positions.tolist() == list(range(500 - n, 500)) + list(range(400 - n, 400))


@pytest.mark.parametrize("heads,kv_heads,dim,counts,held,page", [(16, 2, 256, (64,), (32000,), 64), (32, 8, 128, (61, 7, 30), (2001, 3000, 900), 32),
                                                                 (8, 8, 64, (256, 100), (5000, 10), 16)])
def test_tree_behind_long_caches(hip, heads, kv_heads, dim, counts, held, page):
    """Caches that are cut into many pieces, a few rows of each tree against the oracle on what they see."""
    g, rng = gen(44), random.Random(44)
    lengths = [c + h for c, h in zip(counts, held)]
    need = sum(-(-n // page) for n in lengths)
    pages = random_pages(hip, g, 1, need, kv_heads, page, dim, torch.int8)
    table = table_of(g, lengths, page, need)
    q = torch.randn(sum(counts), heads, dim, generator=g).to(torch.bfloat16).to(DEV)
    parents = [p for n in counts for p in random_tree(rng, n)]
    tree, _ = hip.kv_tree(i32(parents), i32(held), cu_of(counts), max_count=max(counts))
    args = (pages, 0, q, table, i32(lengths), cu_of(counts))
    out = hip.kv_attend(*args, max_count=max(counts), max_length=max(lengths), tree=tree)
    assert torch.equal(out, hip.kv_attend(*args, max_count=max(counts), max_length=max(lengths), tree=tree))
    cache = [t[0].cpu() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    at = 0
    for b, n in enumerate(counts):
        for i in sorted({n // 2, n - 1}):
            want, tol = _tree_row(cache, q[at + i], table[b], lengths[b], n, tree[at + i])
            assert ((out[at + i].cpu().double() - want).abs() <= tol).all(), (b, i)
        at += n


def _tree_row(cache, q, table, length, n, words):
    """One drafted row by the oracle: its sequence's tokens that it does not see taken out of the cache, the last one seen last."""
    k, v, ks, vs = cache
    page = k.shape[2]
    seen = list(range(length - n)) + [length - n + j for j in kv_ref.drafted(words.cpu(), n)]
    at = torch.tensor(seen)
    p = table.cpu().long()[at // page]
    # one page a token: the oracle takes any page size
    one = [k[p, :, at % page][:, :, None], v[p, :, :, at % page][..., None], ks[p], vs[p]]
    want, tol = kv_ref.attend(*one, q[None].cpu(), torch.arange(len(seen))[None], torch.tensor([len(seen)]), torch.tensor([0, 1]))
    return want[0], tol[0]


# -- keeping accepted tokens ------------------------------------------------------------------------------------------


def check_keep(hip, pages, table, start, keep, cu, max_count=None):
    want = {name: kv_ref.keep(getattr(pages, name).cpu(), getattr(pages, name + "_scale").cpu(), table.cpu(), start.cpu(), keep.cpu(),
                              cu.cpu(), pages.page_tokens, name == "v", max_count) for name in "kv"}
    hip.kv_keep(pages, table, start, keep, cu, max_count=max_count)
    torch.cuda.synchronize()
    for name in "kv":
        np.testing.assert_array_equal(getattr(pages, name + "_scale").cpu().double().numpy(), want[name][1].numpy(), name + " scale")
        np.testing.assert_array_equal(getattr(pages, name).cpu().double().numpy(), want[name][0].numpy(), name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page,counts,starts,kept", [
    (256, 64, (16,), (700,), ((0, 3, 7, 8),)), (256, 64, (64, 30), (60, 63), ((0, 5, 6, 20, 63), (1, 29))),
    (128, 16, (40, 5, 1, 64), (5, 16, 0, 31), (tuple(range(0, 40, 2)), (), (0,), tuple(range(10, 64)))),
    (64, 32, (100, 3), (31, 0), (tuple(range(1, 100)), (0, 1, 2))), (64, 1024, (30,), (1010,), (tuple(range(0, 30, 2)),)),
    (128, 128, (250,), (7,), (tuple(range(100, 250)),))])
def test_keep(hip, dtype, dim, page, counts, starts, kept):
    g = gen(dim + page + 50)
    lengths = [c + s for c, s in zip(counts, starts)]
    need = sum(-(-n // page) for n in lengths)
    pages = random_pages(hip, g, 3, need + 1, 2, page, dim, dtype)
    for name in ("k_scale", "v_scale"):  # pages whose scales lie far apart: some grow, by a lot
        t = getattr(pages, name)
        t.mul_(torch.pow(2.0, torch.randint(-9, 10, t.shape, generator=g)).to(DEV))
    table = table_of(g, lengths, page, need + 1)
    check_keep(hip, pages, table, i32(starts), i32([j for k in kept for j in k]), cu_of([len(k) for k in kept]),
               max(map(len, kept)) if dim == 64 else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page,count,start,every", [(256, 256, 400, 37, 3), (64, 1024, 1500, 900, 5), (128, 512, 700, 500, 17), (256, 16, 150, 9, 1)])
def test_keep_many(hip, dtype, dim, page, count, start, every):
    """More tokens of a page than are held at a time, from few or many groups of 16: pages whose scale grows, and that do not."""
    g, rng = gen(dim + page + 51), random.Random(every)
    lengths = (start + count, start + count // 2)
    need = sum(-(-n // page) for n in lengths)
    pages = random_pages(hip, g, 1, need + 1, 2, page, dim, dtype)
    pages.k_scale.mul_(torch.pow(2.0, torch.randint(-4, 5, pages.k_scale.shape, generator=g)).to(DEV))
    table = table_of(g, lengths, page, need + 1)
    kept = [sorted(rng.sample(range(n), max(n // every - 1, 1))) for n in (count, count // 2)]
    check_keep(hip, pages, table, i32([start] * 2), i32([j for k in kept for j in k]), cu_of([len(k) for k in kept]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_keep_moves_bytes_inside_a_page(hip, dtype):
    """What stays in its page keeps its bytes, whatever its scale, one of more bits than bf16's among them; nothing else changes."""
    g = gen(51)
    pages = random_pages(hip, g, 2, 3, 2, 64, 128, dtype)
    pages.k_scale.mul_(1.2345678)
    pages.v_scale.div_(3)
    before = [t.view(torch.int8).clone() if t.dim() == 5 else t.clone() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    hip.kv_keep(pages, i32([[2, 0]]), i32([70]), i32([0, 2, 3, 9, 40]), i32([0, 5]))
    before[0][:, 0, :, 6:11] = before[0][:, 0][:, :, [6, 8, 9, 15, 46]]
    before[1][:, 0, :, :, 6:11] = before[1][:, 0][..., [6, 8, 9, 15, 46]]
    for t, w in zip((pages.k, pages.v, pages.k_scale, pages.v_scale), before):
        assert torch.equal(t.view(torch.int8) if t.dim() == 5 else t, w)


@pytest.mark.parametrize("dtype", DTYPES)
def test_keep_special_scales(hip, dtype):
    """Pages of scale 0, a zero page that receives values (stray bytes before them become zeros), NaN scales on either side, values
    past fp32's range, missing source and target pages."""
    g = gen(52)
    for case in range(6):
        pages = random_pages(hip, g, 1, 6, 1, 16, 64, dtype)
        ks, vs = pages.k_scale[0, :, 0], pages.v_scale[0, :, 0]
        table = i32([[0, 1, 2], [3, 4, 5]])
        if case == 0:
            ks[0], vs[1], ks[4], vs[5] = 0.0, 0.0, 0.0, 0.0
        elif case == 1:
            ks[0], vs[1], ks[5] = math.nan, math.nan, math.nan
        elif case == 2:
            ks[1], vs[2], ks[3] = 3e38, 2.0 ** 125, 1e-30
        elif case == 3:
            table[0, 1], table[1, 0] = -1, 77
        elif case == 4:
            ks[:], vs[:] = 0.0, math.nan
        check_keep(hip, pages, table, i32([5, 15]), i32([0, 9, 12, 13, 14, 30, 0, 1, 2, 20]), i32([0, 6, 10]))


@pytest.mark.parametrize("starts,keep,cu,max_count", [
    ((0, 40), (3, 4, 9, 0, 1, 5), (0, 3, 6), None),                      # sequence 1 lies behind its table
    ((10, 31), (8, 40, 100, 2 ** 31 - 1, 1, 5), (0, 4, 6), None),        # sources behind the table stay where they are
    ((4, 9), (5, 0, -3, 20, 2, 2, 2, 9), (0, 4, 8), None),               # less than their number: they stay; one token twice; out of order
    ((4, 9), (1, 2, 3, 4, 5, 6, 7, 8), (0, 6, 8), 4),                    # entries beyond max_count are none
    ((4, 9), (1, 2, 3, 4, 5, 6, 7, 8), (-3, 4, 1000), None), ((4, 9), (1, 2, 3, 4, 5, 6, 7, 8), (6, 2, 8), None),
    ((-7, 2 ** 31 - 2), (1, 2, 3, 4, 5, 6, 7, 8), (0, 4, 8), None)])
def test_keep_out_of_range(hip, starts, keep, cu, max_count):
    g = gen(53)
    pages = random_pages(hip, g, 2, 7, 2, 16, 64, torch.int8)
    check_keep(hip, pages, i32([[1, 5, 3], [0, 2, 6]]), i32(starts), i32(keep), i32(cu), max_count)


def test_keep_past_32_bits(hip):
    """Pages whose bytes lie more than 2^32 into the cache: the same bits as on a small cache that holds just them."""
    g = gen(54)
    total, page, dim = 150_000, 64, 256
    far = hip.KVPages(*(torch.empty(1, total, 2, *t, dtype=torch.int8, device=DEV) for t in ((page, dim), (dim, page))),
                      *(torch.zeros(1, total, 2, device=DEV) for _ in range(2)))
    small = random_pages(hip, g, 1, 3, 2, page, dim, torch.int8)
    ids = [total - 1, 5, total - 1000]
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(far, name)[:, ids] = getattr(small, name)
    keep, cu = i32([0, 9, 30, 66, 100]), i32([0, 5])
    hip.kv_keep(small, i32([[0, 1, 2]]), i32([62]), keep, cu)
    hip.kv_keep(far, i32([ids]), i32([62]), keep, cu)
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(far, name)[:, ids], getattr(small, name)), name
    tree, _ = hip.kv_tree(i32([-1] * 5), i32([130]), cu)
    q = torch.randn(5, 16, dim, generator=g).to(torch.bfloat16).to(DEV)
    for kw in (dict(tree=tree), dict(window=50, sinks=3)):
        outs = [hip.kv_attend(p, 0, q, i32([t]), i32([135]), cu, **kw) for p, t in ((small, [0, 1, 2]), (far, ids))]
        assert torch.equal(*outs)


# -- norms with positions ---------------------------------------------------------------------------------------------


def check_norm_rope(x, got, weight, eps, zero_centered, positions, inv_freq, sections, interleaved, scale=1.0):
    y = kv_ref.norm(x.cpu(), None if weight is None else weight.cpu(), eps, zero_centered)
    want = kv_ref.rope(y, positions.cpu(), inv_freq.cpu(), sections, interleaved, scale)
    half, dim = inv_freq.shape[0], x.shape[-1]
    # a normed value: the sum of dim squares in fp32 (its error halves in the root), a root, a quotient, two products, 1 + w
    per = (dim / 2 + 8) * 2.0 ** -24
    pair = y.abs().clone()
    pair[..., :2 * half] = (pair[..., :half] + pair[..., half:2 * half]).repeat(1, 1, 2) * abs(scale)
    # cosine and sine within 2^-21 of a turn's exact ones, three fp32 roundings; one rounding to the type
    turned = torch.zeros_like(pair)
    turned[..., :2 * half] = 2.0 ** -20
    tol = pair * (per + turned) * 1.01 + want.abs() * torch.finfo(x.dtype).eps / 2
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,half,sections,interleaved", [
    (1, 16, 2, 256, 32, (11, 11, 10), True), (37, 16, 2, 256, 32, (11, 11, 10), True), (5, 3, 1, 128, 64, (16, 24, 24), False),
    (9, 4, 4, 64, 32, (32,), False), (6, 2, 1, 80, 15, (5, 5, 5), True), (3, 1, 1, 6, 1, (1, 0), True), (4, 2, 2, 64, 20, (5, 5, 5, 5), True),
    (3, 9, 1, 1024, 512, (512,), True), (2, 2, 1, 1000, 8, (4, 4), True), (2, 1, 1, 2, 1, (1,), True)])
@pytest.mark.parametrize("layout", ["dense", "gated", "odd"])
def test_norm_rope(hip, dtype, tokens, heads, kv_heads, dim, half, sections, interleaved, layout):
    g = gen(tokens + dim)
    extra = {"dense": 0, "gated": dim, "odd": 1}[layout]
    q = (3 * torch.randn(tokens, heads, dim + extra, generator=g)).to(dtype).to(DEV)[..., :dim]
    k = torch.randn(tokens, kv_heads, dim + extra, generator=g).to(dtype).to(DEV)[..., :dim]
    weights = [(0.5 * torch.randn(dim, generator=g)).to(torch.bfloat16 if layout == "odd" else torch.float32).to(DEV) for _ in range(2)]
    positions = torch.randint(-50, 1 << 20, (len(sections), tokens), generator=g).to(DEV)
    inv_freq = torch.pow(1e6, -torch.arange(half, dtype=torch.float64) / half).to(DEV)
    q0, k0 = q.clone(), k.clone()
    args = dict(sections=sections, interleaved=interleaved, scale=1.25)
    for wq, wk, eps, zero in ((*weights, 1e-6, True), (weights[0], None, 1e-3, False), (None, weights[1], 0.0, True), (None, None, 2.0, False)):
        rq, rk = hip.norm_rope(q, k, positions, inv_freq, wq, wk, eps=eps, zero_centered=zero, **args)
        assert rq.is_contiguous() and torch.equal(q, q0) and torch.equal(k, k0)
        check_norm_rope(q, rq, wq, eps, zero, positions, inv_freq, sections, interleaved, 1.25)
        check_norm_rope(k, rk, wk, eps, zero, positions, inv_freq, sections, interleaved, 1.25)
    iq, none = hip.norm_rope(q, None, positions, inv_freq, None, None, eps=2.0, out=(q, None), **args)
    assert none is None and iq is q and torch.equal(q, rq)  # in place, alone: the same bits


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,half", [(2051, 3, 1, 256, 32), (4099, 1, 2, 64, 32), (2049, 2, 1, 512, 64)])
def test_norm_rope_many_tokens(hip, tokens, heads, kv_heads, dim, half):
    """More tokens than a workgroup each holds at once, an odd number of them; against the oracle, and the same bits as in smaller calls."""
    g = gen(tokens)
    q, k = (torch.randn(tokens, h, dim, generator=g).to(torch.bfloat16).to(DEV) for h in (heads, kv_heads))
    w = [torch.randn(dim, generator=g).to(DEV) for _ in range(2)]
    p, f = torch.arange(tokens, device=DEV) * 7, torch.pow(1e6, -torch.arange(half, dtype=torch.float64, device=DEV) / half)
    rq, rk = hip.norm_rope(q, k, p, f, *w)
    check_norm_rope(q, rq, w[0], 1e-6, True, p[None], f, (half,), True)
    check_norm_rope(k, rk, w[1], 1e-6, True, p[None], f, (half,), True)
    for part in (slice(0, 1), slice(1000, 2000), slice(tokens - 3, tokens)):
        sq, sk = hip.norm_rope(q[part], k[part], p[part], f, *w)
        assert torch.equal(sq, rq[part]) and torch.equal(sk, rk[part])


def test_norm_rope_small_and_large_values(hip):
    """Rows of zeros, of values whose squares leave eps nothing to do, and of values that are nothing beside it; NaN and infinities
    stay in their head."""
    g = gen(61)
    x = torch.randn(6, 2, 64, generator=g)
    x[0] = 0
    x[1] *= 1e15
    x[2] *= 1e-15
    x[4, 0, 3], x[5, 1, 60] = math.nan, math.inf
    q = x.to(torch.bfloat16).to(DEV)
    p, f = torch.arange(6, device=DEV), torch.ones(8, dtype=torch.float64, device=DEV)
    w = torch.zeros(64, device=DEV)
    got, _ = hip.norm_rope(q, None, p, f, w)
    check_norm_rope(q[:4], got[:4], w, 1e-6, True, p[None, :4], f, (8,), True)
    assert (got[0] == 0).all() and torch.isnan(got[4, 0].float()).all()
    assert torch.isfinite(got[4, 1].float()).all() and torch.isfinite(got[5, 0].float()).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_norm_rope_of_one_head_knows_no_other(hip, dtype, dim):
    """A head's bits are those of a call of its own, whatever stands beside it: zeros without eps, values whose squares all but vanish."""
    g = gen(62)
    x = torch.randn(40, 3, dim, generator=g)
    x[:20, 1] *= 1e-17
    x[20:, 2] = 0
    q = x.to(dtype).to(DEV)
    w, f, p = torch.randn(dim, generator=g).to(DEV), torch.ones(16, dtype=torch.float64, device=DEV), torch.arange(40, device=DEV)
    for eps in (0.0, 1e-32, 1e-6):
        got, _ = hip.norm_rope(q, None, p, f, w, eps=eps)
        for i in range(40):
            for h in range(3):
                alone, _ = hip.norm_rope(q[i:i + 1, h:h + 1], None, p[i:i + 1], f, w, eps=eps)
                assert torch.equal(alone[0, 0].view(torch.uint8), got[i, h].view(torch.uint8)), (eps, i, h)


def test_norm_rope_refusals(hip):
    q = torch.zeros(2, 1, 64, device=DEV)
    f, p = torch.ones(8, dtype=torch.float64, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    w = torch.zeros(64, device=DEV)
    for bad in (dict(q_weight=w[:32]), dict(q_weight=w.double()), dict(q_weight=w.cpu()), dict(q_weight=w, k_weight=w.bfloat16()),
                dict(q_weight=torch.zeros(128, device=DEV)[::2]), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf), dict(q_weight=w[None]),
                dict(sections=(4, 3))):
        with pytest.raises(ValueError):
            hip.norm_rope(q, q.clone(), p, f, **bad)
    for bad in (q.half(), q.cpu(), q[..., :8]):
        with pytest.raises(ValueError):
            hip.norm_rope(bad, None, p, f)


# -- workspaces -------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("count,window", [(1, 900), (8, None), (64, None), (300, 500)])
def test_masked_workspaces(hip, count, window):
    """A workspace of the size that is asked for, whatever it holds, gives the bits of one from the allocator; a smaller one is refused."""
    import ctypes
    g, rng = gen(72), random.Random(72)
    pages = random_pages(hip, g, 1, 150, 2, 64, 128, torch.int8)
    table = table_of(g, (4000, 3000), 64, 150)
    length, cu = i32([4000, 3000]), cu_of((count, count))
    q = torch.randn(2 * count, 8, 128, generator=g).to(torch.bfloat16).to(DEV)
    kw = dict(window=window, sinks=3) if window else dict(tree=hip.kv_tree(i32(random_tree(rng, count) * 2), length - count, cu, max_count=count)[0])
    want = hip.kv_attend(pages, 0, q, table, length, cu, max_count=count, **kw)
    tree = kw.get("tree")
    mask = hip.WlKvMask(tree.data_ptr() if tree is not None else None, tree.shape[1] if tree is not None else 0, window or 0, 3 if window else 0)
    batch = hip.WlKvBatch(table.data_ptr(), cu.data_ptr(), table.stride(0), 2 * count, 2, table.shape[1], count, 0)
    need = hip.library().wl_kv_attend_masked_workspace_bytes(pages.ref, 8, ctypes.byref(batch), table.shape[1] * 64, ctypes.byref(mask))
    assert need > 0
    space = torch.full((need + 64,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(want, hip.kv_attend(pages, 0, q, table, length, cu, max_count=count, workspace=space[:need], **kw))
    assert (space[need:] == 255).all()
    with pytest.raises(ValueError):
        hip.kv_attend(pages, 0, q, table, length, cu, max_count=count, workspace=space[:need - 16], **kw)


# -- captured ---------------------------------------------------------------------------------------------------------


def test_two_graphs_of_a_draft(hip):
    """Two captured steps (norms and positions, tree, attention with and without a window, accepted tokens moved), replayed in turn
    with other inputs, eager calls and synchronizations in between: the eager calls' bits every time."""
    g, rng = gen(71), random.Random(71)
    page, dim, n = 32, 128, 20
    f = torch.pow(1e6, -torch.arange(32, dtype=torch.float64, device=DEV) / 32)
    w = torch.randn(dim, generator=g).to(DEV)

    def fresh():
        return dict(q=torch.randn(2 * n, 8, dim, generator=g).to(torch.bfloat16), k=torch.randn(2 * n, 2, dim, generator=g).to(torch.bfloat16),
                    parents=torch.tensor(random_tree(rng, n) + random_tree(rng, n), dtype=torch.int32),
                    start=torch.tensor([rng.randrange(900), rng.randrange(40)], dtype=torch.int32),
                    keep=torch.tensor(sorted(rng.sample(range(n), 6)) + sorted(rng.sample(range(n), 3)), dtype=torch.int32))

    pools = [random_pages(hip, g, 2, 32, 2, page, dim, torch.int8) for _ in range(2)]
    mirrors = [hip.KVPages(*(getattr(p, name).clone() for name in ("k", "v", "k_scale", "v_scale"))) for p in pools]
    table = table_of(g, (920, 60), page, 32, width=30)
    cu, kept = cu_of((n, n)), i32([0, 6, 9])
    states = [{name: t.to(DEV) for name, t in fresh().items()} for _ in range(2)]

    def call(pages, s):
        tree, positions = hip.kv_tree(s["parents"], s["start"], cu, max_count=n)
        q, k = hip.norm_rope(s["q"], s["k"], positions, f, w, w)
        hip.kv_append(pages, 0, k, k, table, s["start"], cu, max_count=n)
        length = s["start"] + n
        a = hip.kv_attend(pages, 0, q, table, length, cu, max_count=n, max_length=920, tree=tree)
        b = hip.kv_attend(pages, 0, q, table, length, cu, max_count=n, max_length=920, tree=tree, window=100, sinks=4)
        hip.kv_keep(pages, table, s["start"], s["keep"], kept, max_count=6)
        return torch.stack((a, b)), positions
    for p, m, s in zip(pools, mirrors, states):  # once before the capture, on both alike
        call(p, s)
        call(m, s)
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[i]):
            got.append(call(pools[i], states[i]))
    for turn in range(6):
        want = []
        for i in (0, 1) if turn % 2 else (1, 0):
            for name, t in fresh().items():
                states[i][name].copy_(t)
            want.append((i, call(mirrors[i], states[i])))
            if turn % 3 == 0:
                torch.cuda.synchronize()
            graphs[i].replay()
        torch.cuda.synchronize()
        for i, (a, positions) in want:
            assert torch.equal(got[i][0], a) and torch.equal(got[i][1], positions), f"turn {turn}"
            for name in ("k", "v", "k_scale", "v_scale"):
                assert torch.equal(getattr(pools[i], name), getattr(mirrors[i], name)), f"turn {turn}, {name}"
