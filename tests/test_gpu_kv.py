"""The paged 8-bit key/value cache on the GPU: append bit for bit, attention within the bound that its roundings give, page
copies, rotary positions; against oracle/kv_ref.py in 64 bits."""
import math

import numpy as np
import pytest
import torch

from oracle import kv_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def gen(seed):
    return torch.Generator().manual_seed(seed)


def random_pages(hip, g, layers, pages, heads, page, dim, dtype):
    """A cache of random values (on the GPU), every block with a scale of its own."""
    top = kv_ref.LARGEST[dtype]

    def values(*tail):
        x = (torch.randn(layers, pages, heads, *tail, generator=g) * top / 4).clamp(-top, top)
        return (x.round() if dtype == torch.int8 else x).to(dtype).to(DEV)

    def scales():
        return (torch.exp(0.5 * torch.randn(layers, pages, heads, generator=g)) * 4 / top).to(torch.bfloat16).float().to(DEV)

    return hip.KVPages(values(page, dim), values(dim, page), scales(), scales())


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cu_of(counts):
    return i32([0] + list(np.cumsum(counts)))


def table_of(g, lengths, page, pages, width=None):
    """Pages for sequences of these lengths, in random order; entries that no token needs point outside the cache."""
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(pages, generator=g).tolist()
    width = max(max(need), 1) if width is None else width
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1 if at % 2 else 2 ** 31 - 1] * (width - n))
        at += n
    assert at <= pages
    return i32(table)


# -- append ----------------------------------------------------------------------------------------------------------


def check_append(hip, pages, layer, k, v, table, start, cu, max_count=None, equal_nan=True):
    want = {}
    for name, new, is_v in (("k", k, False), ("v", v, True)):
        want[name] = kv_ref.append(getattr(pages, name)[layer].cpu(), getattr(pages, name + "_scale")[layer].cpu(), new.cpu(),
                                   table.cpu(), start.cpu(), cu.cpu(), pages.page_tokens, is_v, max_count)
    others = [getattr(pages, n).view(torch.int8).clone() if n in "kv" else getattr(pages, n).clone()
              for n in ("k", "v", "k_scale", "v_scale")]
    hip.kv_append(pages, layer, k, v, table, start, cu, max_count=max_count)
    torch.cuda.synchronize()
    for name in ("k", "v"):
        pool, scale = want[name]
        np.testing.assert_array_equal(getattr(pages, name + "_scale")[layer].cpu().double().numpy(), scale.numpy(), name + " scale")
        np.testing.assert_array_equal(getattr(pages, name)[layer].cpu().double().numpy(), pool.numpy(), name)
    for n, was in zip(("k", "v", "k_scale", "v_scale"), others):  # the other layers
        now = getattr(pages, n).view(torch.int8) if n in "kv" else getattr(pages, n)
        for l in range(pages.layers):
            assert l == layer or torch.equal(now[l], was[l])


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dim,page,counts,starts", [
    (256, 64, (1,), (0,)), (256, 64, (1, 1, 1), (63, 64, 17)), (128, 16, (37, 1, 0, 16), (5, 31, 3, 16)),
    (64, 32, (100, 3), (47, 0)), (64, 1024, (5,), (1020,)), (256, 32, (129,), (31,)), (128, 64, (64, 65, 63), (0, 64, 1))])
@pytest.mark.parametrize("layout", ["fused", "dense", "odd"])
def test_append(hip, dtype, dim, page, counts, starts, layout):
    g = gen(dim + page)
    pages = random_pages(hip, g, 2, 12, 2, page, dim, dtype)
    table = table_of(g, [c + s for c, s in zip(counts, starts)], page, 12)
    total = sum(counts)
    x = torch.randn(total, 2, 2, dim, generator=g)
    x[:, 0] *= 1 + 20 * (torch.rand(dim, generator=g) < 0.05)  # some channels make older scales grow
    x = x.to(torch.bfloat16).to(DEV)
    if layout == "dense":
        k, v = x[:, 0].contiguous(), x[:, 1].contiguous()
    elif layout == "odd":  # rows that start on any even address
        wide = torch.zeros(total, 2, 2, dim + 3, dtype=torch.bfloat16, device=DEV)
        wide[..., 1:dim + 1] = x
        k, v = wide[:, 0, :, 1:dim + 1], wide[:, 1, :, 1:dim + 1]
    else:
        k, v = x[:, 0], x[:, 1]
    check_append(hip, pages, 1, k, v, table, i32(starts), cu_of(counts))


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_append_token_by_token(hip, dtype):
    """The scale of a page grows with its tokens, by powers of two; a value stays within one final step of what it was."""
    g = gen(3)
    pages = hip.KVPages.empty(1, 3, 1, 64, 32, dtype)
    table = i32([[2, 0]])
    x = (torch.randn(40, 1, 64, generator=g) * torch.logspace(-3, 2, 40)[:, None, None]).to(torch.bfloat16).to(DEV)
    for t in range(40):
        check_append(hip, pages, 0, x[t:t + 1], -x[t:t + 1], table, i32([t]), i32([0, 1]))
    for t in range(40):
        p = (2, 0)[t // 32]
        got = pages.k[0, p, 0, t % 32].cpu().double() * float(pages.k_scale[0, p, 0])
        step = float(pages.k_scale[0, p, 0]) * (1 if dtype == torch.int8 else 2.0 ** -9)
        want = x[t, 0].cpu().double()
        assert ((got - want).abs() <= step + (0 if dtype == torch.int8 else 2.0 ** -4) * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_append_special_values(hip, dtype):
    """Blocks of zeros, a zero block that gets values, NaN, infinities, the largest and smallest bf16; scales that tie."""
    pages = hip.KVPages.empty(1, 4, 1, 64, 16, dtype)
    table = i32([[0], [1], [2], [3]])
    big = torch.finfo(torch.bfloat16).max
    rows = torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    rows[1, 0, 5], rows[2, 0, :3], rows[3, 0, :4] = math.nan, torch.tensor([big, -big, 1.0]), torch.tensor([127.0, 63.5, 0.5, -1.5])
    check_append(hip, pages, 0, rows.to(DEV), (rows * 0.5).to(DEV), table, i32([0] * 4), i32([0, 1, 2, 3, 4]))
    assert math.isnan(float(pages.k_scale[0, 1, 0])) and float(pages.k_scale[0, 0, 0]) == 0
    rows = torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    rows[0, 0, 1], rows[1, 0, 0], rows[2, 0, 0], rows[3, 0, 7] = 1e-39, 3.0, math.inf, 128.0
    check_append(hip, pages, 0, rows.to(DEV), rows.to(DEV), table, i32([1] * 4), i32([0, 1, 2, 3, 4]))
    assert math.isnan(float(pages.k_scale[0, 1, 0])) and math.isnan(float(pages.k_scale[0, 2, 0]))


def test_append_zero_scale_forgets_stray_bytes(hip):
    """A block of scale 0 holds zeros whatever its bytes are; they are zero bytes once it gets a scale."""
    pages = hip.KVPages.empty(1, 1, 1, 64, 16)
    pages.k.fill_(77)
    pages.v.fill_(-5)
    check_append(hip, pages, 0, *(torch.ones(1, 1, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2)), i32([[0]]), i32([3]),
                 i32([0, 1]))
    assert not pages.k[0, 0, 0, :3].any() and not pages.v[0, 0, 0, :, :3].any()


@pytest.mark.parametrize("counts,starts,cu,max_count", [
    ((3, 3), (0, 40), (0, 3, 6), None),        # sequence 1 lies behind its table
    ((3, 3), (14, 15), (0, 3, 6), None),       # both cross into a page that is not there
    ((9, 4), (0, 0), (0, 9, 13), 5),           # rows beyond max_count are dropped
    ((9, 4), (0, 0), (-4, 9, 1000), None),     # offsets outside the rows
    ((9, 4), (0, 0), (6, 2, 13), None),        # a sequence that ends before it begins is empty
    ((9, 4), (-7, 2 ** 31 - 2), (0, 9, 13), None)])
def test_append_out_of_range(hip, counts, starts, cu, max_count):
    g = gen(9)
    pages = random_pages(hip, g, 1, 3, 2, 16, 64, torch.int8)
    table = i32([[1, -1], [0, 3]])
    x = torch.randn(13, 2, 64, generator=g).to(torch.bfloat16).to(DEV)
    check_append(hip, pages, 0, x, x * 2, table, i32(starts), i32(cu), max_count)


# -- attend ----------------------------------------------------------------------------------------------------------


def check_attend(hip, pages, layer, q, table, length, cu, **kw):
    ref = {n: kw[n] for n in ("scale", "causal", "max_count") if n in kw}
    if "weight_roundings" in kw:
        ref["weight_roundings"] = kw.pop("weight_roundings")
    want, tol = kv_ref.attend(pages.k[layer].cpu(), pages.v[layer].cpu(), pages.k_scale[layer].cpu(), pages.v_scale[layer].cpu(),
                              q.cpu(), table.cpu(), length.cpu(), cu.cpu(), **ref)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    got = hip.kv_attend(pages, layer, q, table, length, cu, out=out, **kw)
    torch.cuda.synchronize()
    assert got is out
    got = got.cpu().double()
    free = torch.isnan(want).all(2)
    owned = torch.zeros(q.shape[0], dtype=torch.bool)
    bounds = cu.cpu().tolist()
    for b in range(len(bounds) - 1):
        lo = min(max(bounds[b], 0), q.shape[0])
        n = min(max(bounds[b + 1], lo) - lo, q.shape[0] - lo, kw.get("max_count") or q.shape[0])
        owned[lo:lo + n] = True
    assert (got[~owned] == 7.0).all()  # rows of no sequence stay as they were
    want, got, tol, free = want[owned], got[owned], tol[owned], free[owned]
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places than expected"
    err = torch.where(torch.isnan(want), 0.0, (got - want).abs())
    worst = (err / (tol + 1e-300)).nan_to_num(0.0).max() if err.numel() else 0
    assert (err <= tol.nan_to_num(0.0)).all(), f"off by {float(worst):.2f} of the bound"
    return out


SHAPES = [  # q heads, kv heads, dim, page
    (16, 2, 256, 64), (32, 8, 128, 32), (8, 8, 64, 16), (6, 1, 64, 128), (3, 1, 256, 32), (20, 1, 128, 64)]


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("counts,lengths", [
    ((1,), (1,)), ((1,), (64,)), ((1, 1, 1), (65, 700, 3)), ((2, 1, 2), (130, 1, 2)), ((1, 0, 1, 1), (0, 50, 129, 257)),
    ((5, 33, 1), (5, 100, 190)), ((17,), (300,))])
def test_attend(hip, dtype, heads, kv_heads, dim, page, counts, lengths):
    g = gen(sum(lengths) + dim)
    need = sum(-(-n // page) for n in lengths)
    pages = random_pages(hip, g, 2, need + 2, kv_heads, page, dim, dtype)
    table = table_of(g, lengths, page, need + 2)
    q = (1.5 * torch.randn(sum(counts), heads, dim, generator=g)).to(torch.bfloat16).to(DEV)
    check_attend(hip, pages, 1, q, table, i32(lengths), cu_of(counts), max_count=max(counts))


@pytest.mark.parametrize("counts,lengths", [((7, 3), (3, 3)), ((40, 2), (11, 0)), ((3,), (200,))])
@pytest.mark.parametrize("causal", [True, False])
def test_attend_rows_without_tokens(hip, counts, lengths, causal):
    """More new rows than tokens: the first ones stand before the sequence's beginning and see nothing."""
    g = gen(4)
    pages = random_pages(hip, g, 1, 8, 2, 64, 128, torch.int8)
    table = table_of(g, lengths, 64, 8)
    q = torch.randn(sum(counts), 8, 128, generator=g).to(torch.bfloat16).to(DEV)
    out = check_attend(hip, pages, 0, q, table, i32(lengths), cu_of(counts), causal=causal, scale=0.3)
    if causal and counts[0] > lengths[0]:
        assert (out[:counts[0] - lengths[0]] == 0).all()


@pytest.mark.parametrize("count", [1, 24])
def test_attend_strided_and_padded(hip, count):
    """q as a slice of wider rows (aligned, and not), rows behind the last sequence, a table wider than its rows' use."""
    g = gen(5)
    pages = random_pages(hip, g, 1, 12, 2, 32, 256, torch.float8_e4m3fn)
    lengths = (90, 33 + count)
    table = table_of(g, lengths, 32, 12, width=9)
    wide = torch.randn(2 * count + 5, 8, 2 * 256 + 8, generator=g).to(torch.bfloat16).to(DEV)
    for cut in (0, 1, 8):
        check_attend(hip, pages, 0, wide[:, :, cut:cut + 256], table, i32(lengths), cu_of((count, count)), max_count=count)
    padded = torch.cat((table, table), 1)[:, :9]
    check_attend(hip, pages, 0, wide[:, :, :256], padded, i32(lengths), cu_of((count, count)), max_count=count, max_length=70)


@pytest.mark.parametrize("count", [1, 20])
def test_attend_nan_stays_where_it_is(hip, count):
    """e4m3 bytes that nobody wrote (NaN codes behind the length, in spare pages) reach no row; a block whose scale is NaN
    reaches exactly the rows that see a token of it; missing pages are seen by nobody."""
    g = gen(6)
    lengths = (75, 130, 40)
    pages = random_pages(hip, g, 1, 10, 2, 32, 64, torch.float8_e4m3fn)
    table = table_of(g, lengths, 32, 10)
    raw_k, raw_v = pages.k.view(torch.uint8), pages.v.view(torch.uint8)
    used = set()
    for b, n in enumerate(lengths):
        for c in range(-(-n // 32)):
            p = int(table[b, c])
            used.add(p)
            raw_k[0, p, :, max(0, n - 32 * c):] = 0x7F
            raw_v[0, p, :, :, max(0, n - 32 * c):] = 0xFF
    for p in set(range(10)) - used:
        raw_k[0, p], raw_v[0, p] = 0x7F, 0x7F
        pages.k_scale[0, p], pages.v_scale[0, p] = math.nan, math.nan
    q = torch.randn(3 * count, 4, 64, generator=g).to(torch.bfloat16).to(DEV)
    args = (i32(lengths), cu_of((count,) * 3))
    out = check_attend(hip, pages, 0, q, table, *args)
    assert torch.isfinite(out.float()).all()
    missing = table.clone()
    missing[1, 2], missing[2, 0] = -1, 10
    check_attend(hip, pages, 0, q, missing, *args)
    pages.v_scale[0, int(table[1, 4]), 1] = math.nan  # tokens 128, 129 of sequence 1, second kv head
    out = check_attend(hip, pages, 0, q, table, *args)
    assert torch.isnan(out[2 * count - 1, 2:].float()).all() and torch.isfinite(out[2 * count - 1, :2].float()).all()


def test_attend_many_sequences(hip):
    """More sequences than lanes, of all lengths, some without rows: shares of the split that begin and end anywhere."""
    g = gen(7)
    rng = np.random.default_rng(7)
    lengths = [int(x) for x in rng.integers(0, 300, 150)]
    lengths[77], lengths[149] = 2000, 1500
    counts = [int(x) for x in rng.integers(0, 3, 150)]
    need = sum(-(-n // 64) for n in lengths)
    pages = random_pages(hip, g, 1, need, 2, 64, 64, torch.int8)
    table = table_of(g, lengths, 64, need)
    q = torch.randn(sum(counts), 6, 64, generator=g).to(torch.bfloat16).to(DEV)
    a = check_attend(hip, pages, 0, q, table, i32(lengths), cu_of(counts), max_count=2)
    for bound in (1, 64, 10 ** 6):  # a bound of the lengths only steers the split
        check_attend(hip, pages, 0, q, table, i32(lengths), cu_of(counts), max_count=2, max_length=bound)
    assert torch.equal(a, hip.kv_attend(pages, 0, q, table, i32(lengths), cu_of(counts), max_count=2))  # the same bits


@pytest.mark.parametrize("dim,count", [(256, 1), (128, 40), (256, 70)])
def test_attend_long(hip, dim, count):
    """A cache long enough that one sequence is shared by many workgroups; weights that pick few tokens."""
    g = gen(8)
    n = 20011
    pages = random_pages(hip, g, 1, n // 64 + 2, 1, 64, dim, torch.int8)
    table = table_of(g, (n,), 64, n // 64 + 2)
    q = (4 * torch.randn(count, 2, dim, generator=g)).to(torch.bfloat16).to(DEV)
    check_attend(hip, pages, 0, q, table, i32([n]), i32([0, count]))


@pytest.mark.parametrize("heads,kv_heads,dim,counts,lengths", [
    (16, 2, 256, (512,), (16512,)), (32, 8, 128, (301, 180, 65, 256, 37), (1700, 999, 65, 1300, 437)), (8, 1, 64, (700,), (30000,)),
    (4, 4, 256, (1100, 300), (1500, 5000))])
def test_attend_prompts_in_pieces(hip, heads, kv_heads, dim, counts, lengths):
    """Prompts whose caches are cut into about a piece a CU, by shares that the device chooses: rows of every part of them."""
    g = gen(18)
    need = sum(-(-n // 64) for n in lengths)
    pages = random_pages(hip, g, 1, need, kv_heads, 64, dim, torch.int8)
    table = table_of(g, lengths, 64, need)
    q = torch.randn(sum(counts), heads, dim, generator=g).to(torch.bfloat16).to(DEV)
    out = hip.kv_attend(pages, 0, q, table, i32(lengths), cu_of(counts), max_count=max(counts), max_length=max(lengths)).cpu().double()
    cache = [x[0].cpu() for x in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    at = 0
    for b, (n, length) in enumerate(zip(counts, lengths)):
        for i in sorted({0, 1, n // 3, n // 2, min(255, n - 1), n - 2, n - 1}):
            want, tol = kv_ref.attend(*cache, q[at + i:at + i + 1].cpu(), table[b:b + 1].cpu(), torch.tensor([length - n + i + 1]),
                                      torch.tensor([0, 1]))
            assert ((out[at + i] - want[0]).abs() <= tol[0]).all(), (b, i)
        at += n


@pytest.mark.parametrize("count", [1, 24])
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_attend_scales_far_out(hip, count, dtype):
    """V's scales from where weights still are normal bf16 values to where sums would leave fp32, zeros among them, K's of 0 and nearly: a sequence
    of each, and one with a mixture, whose largest pages drown the others."""
    g = gen(11)
    v_scales = (2.0 ** -100, 1e-30, 2.0 ** -61, 2.0 ** -60, 2.0 ** -59, 2.0 ** 59, 2.0 ** 60, 2.0 ** 61, 1e25, 0.0)
    n = len(v_scales)
    pages = random_pages(hip, g, 1, 2 * n + 6, 2, 32, 128, dtype)
    for i, s in enumerate(v_scales):
        pages.v_scale[0, 2 * i:2 * i + 2] = s
    for i, s in enumerate((1.0, 0.0, 1e-30, 2.0 ** -60, 1e25, 3.0)):
        pages.v_scale[0, 2 * n + i] = s
    pages.k_scale[0, 4:6], pages.k_scale[0, 8], pages.k_scale[0, 2 * n + 1] = 0.0, 0.0, 1e-38
    table = torch.full((n + 1, 6), -1, dtype=torch.int32)
    table[:n, :2] = torch.arange(2 * n).view(n, 2)
    table[n] = torch.arange(2 * n, 2 * n + 6)
    lengths = [61 - i for i in range(n)] + [190]
    q = torch.randn((n + 1) * count, 8, 128, generator=g).to(torch.bfloat16).to(DEV)
    # the form for many rows rounds weights twice where a scale is that far out
    check_attend(hip, pages, 0, q, table.to(DEV), i32(lengths), cu_of([count] * (n + 1)), max_count=count,
                 weight_roundings=1 if count == 1 else 2)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("max_count", [2, 30])
def test_attend_rows_beyond_max_count(hip, causal, max_count):
    """What an append with the same max_count has left: rows beyond it are not there for either."""
    g = gen(12)
    counts = (max_count + 3, 1, max_count + 40)
    lengths = (200, 5, max_count + 1)
    pages = random_pages(hip, g, 1, 12, 2, 32, 64, torch.int8)
    table = table_of(g, lengths, 32, 12)
    q = torch.randn(sum(counts), 8, 64, generator=g).to(torch.bfloat16).to(DEV)
    check_attend(hip, pages, 0, q, table, i32(lengths), cu_of(counts), max_count=max_count, causal=causal)


@pytest.mark.parametrize("count", [2, 24])
def test_attend_shared_pages(hip, count):
    """Sequences on the same pages (forks), with other lengths."""
    g = gen(13)
    pages = random_pages(hip, g, 1, 12, 2, 32, 64, torch.float8_e4m3fn)
    table = table_of(g, (300,), 32, 12).repeat(3, 1)
    q = torch.randn(3 * count, 8, 64, generator=g).to(torch.bfloat16).to(DEV)
    check_attend(hip, pages, 0, q, table, i32((300, 299, 40)), cu_of([count] * 3), max_count=count)


def test_attend_many_ragged_prompts(hip):
    """The form for many rows over hundreds of sequences, some without rows, some without tokens; no bound of the rows given."""
    g = gen(14)
    rng = np.random.default_rng(14)
    counts = [int(x) for x in rng.integers(0, 8, 300)]
    counts[100], counts[299] = 150, 40
    lengths = [c + int(x) for c, x in zip(counts, rng.integers(0, 60, 300))]
    lengths[5] = 0
    need = sum(-(-n // 16) for n in lengths)
    pages = random_pages(hip, g, 1, need, 2, 16, 64, torch.int8)
    table = table_of(g, lengths, 16, need)
    q = torch.randn(sum(counts) + 3, 8, 64, generator=g).to(torch.bfloat16).to(DEV)
    check_attend(hip, pages, 0, q, table, i32(lengths), cu_of(counts))
    check_attend(hip, pages, 0, q, table, i32(lengths), cu_of(counts), causal=False)


@pytest.mark.parametrize("page,dim,total", [(64, 256, 140_000), (16, 128, 1_100_000)])
def test_past_32_bits(hip, page, dim, total):
    """Pages whose bytes lie more than 2^32 into the cache: the same bits as on a small cache that holds just them."""
    g = gen(15)
    assert total * 2 * page * dim > 2 ** 32
    far = hip.KVPages(*(torch.empty(1, total, 2, *t, dtype=torch.int8, device=DEV) for t in ((page, dim), (dim, page))),
                      *(torch.zeros(1, total, 2, device=DEV) for _ in range(2)))
    ids = [total - 1, total - 2, 0, total - 1000, total // 2 + 1, total - 77, 5, total - 3]
    small = hip.KVPages.empty(1, len(ids), 2, dim, page)
    for t in (far.k, far.v):
        t[:, ids] = 0
    rows = 3 * page + 5
    x = torch.randn(rows + 40, 2, 2, dim, generator=g).to(torch.bfloat16).to(DEV)
    table = torch.tensor([[0, 1, 2, 3], [4, 5, 6, -1]], dtype=torch.int32)
    numbers = torch.tensor(ids + [-1], dtype=torch.int32)
    cu = cu_of((rows, 40))
    outs = []
    for pages, t in ((small, table.to(DEV)), (far, numbers[table.long()].to(DEV))):
        hip.kv_append(pages, 0, x[:, 0], x[:, 1], t, i32([0, 3]), cu)
        outs.append([hip.kv_attend(pages, 0, q, t, i32([rows, 43]), c, max_count=m) for q, c, m in (
            (torch.randn(2, 8, dim, generator=gen(16)).to(torch.bfloat16).to(DEV), i32([0, 1, 2]), 1),
            (torch.randn(60, 8, dim, generator=gen(17)).to(torch.bfloat16).to(DEV), i32([0, 35, 60]), 35))])
    assert all(torch.equal(a, b) and torch.isfinite(a.float()).all() for a, b in zip(*outs))
    hip.kv_copy(far, [ids[0], 5], [total // 3, ids[7]])
    hip.kv_copy(small, [0, 6], [4, 7])
    for name in ("k", "v", "k_scale", "v_scale"):
        a, b = getattr(small, name)[0], getattr(far, name)[0]
        for i, n in enumerate(ids[:4] + [total // 3] + ids[5:]):
            assert torch.equal(a[i], b[n]), (name, i)


# -- copy ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("layers,heads,dim,page,n", [(3, 2, 64, 16, 7), (1, 1, 256, 64, 300), (2, 3, 128, 1024, 2)])
def test_copy(hip, layers, heads, dim, page, n):
    g = gen(n)
    total = 2 * n + 3
    pages = random_pages(hip, g, layers, total, heads, page, dim, torch.float8_e4m3fn)
    order = torch.randperm(total, generator=g).numpy()
    src, dst = order[:n].copy(), order[n:2 * n].copy()
    src[-1] = src[0]  # one page may be copied to several
    want = [t.view(torch.int8).clone() if t.dim() == 5 else t.clone() for t in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    for t in want:
        t[:, torch.from_numpy(dst).to(DEV)] = t[:, torch.from_numpy(src).to(DEV)]
    hip.kv_copy(pages, src, dst)
    for t, name in zip(want, ("k", "v", "k_scale", "v_scale")):
        now = getattr(pages, name)
        assert torch.equal(now.view(torch.int8) if now.dim() == 5 else now, t), name


def test_copy_refuses_on_the_host(hip):
    pages = hip.KVPages.empty(1, 8, 1, 64, 16)
    for src, dst in (([0], [8]), ([-1], [2]), ([0, 1], [3, 3]), ([0, 1], [1, 2]), ([4], [4]), ([0, 1], [2])):
        with pytest.raises(ValueError):
            hip.kv_copy(pages, src, dst)
    hip.kv_copy(pages, [], [])


# -- rope ------------------------------------------------------------------------------------------------------------


def check_rope(hip, x, got, positions, inv_freq, sections, interleaved, scale=1.0):
    want = kv_ref.rope(x.cpu(), positions.cpu(), inv_freq.cpu(), sections, interleaved, scale)
    got = got.cpu()
    half = inv_freq.shape[0]
    a = x.cpu().double().abs()
    pair = torch.zeros_like(a)
    pair[..., :2 * half] = (a[..., :half] + a[..., half:2 * half]).repeat(1, 1, 2)
    # cosine and sine within 2^-21 of a turn's exact ones, three fp32 roundings, one rounding to the type
    tol = abs(scale) * pair * 2.0 ** -20 + want.abs() * torch.finfo(x.dtype).eps / 2
    tol[..., 2 * half:] = 0
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,half,sections,interleaved", [
    (1, 16, 2, 256, 32, (11, 11, 10), True), (37, 16, 2, 256, 32, (11, 11, 10), True), (5, 3, 1, 128, 64, (16, 24, 24), False),
    (9, 4, 4, 64, 32, (32,), False), (6, 2, 1, 80, 15, (5, 5, 5), True), (3, 1, 1, 6, 1, (1, 0), True), (4, 2, 2, 64, 20, (5, 5, 5, 5), True)])
@pytest.mark.parametrize("layout", ["dense", "gated", "odd"])
def test_rope(hip, dtype, tokens, heads, kv_heads, dim, half, sections, interleaved, layout):
    g = gen(tokens + dim)
    extra = {"dense": 0, "gated": dim, "odd": 1}[layout]
    q = torch.randn(tokens, heads, dim + extra, generator=g).to(dtype).to(DEV)[..., :dim]
    k = torch.randn(tokens, kv_heads, dim + extra, generator=g).to(dtype).to(DEV)[..., :dim]
    positions = torch.randint(-50, 1 << 20, (len(sections), tokens), generator=g).to(DEV)
    inv_freq = torch.pow(1e6, -torch.arange(half, dtype=torch.float64) / half).to(DEV)
    q0, k0 = q.clone(), k.clone()
    rq, rk = hip.rope(q, k, positions, inv_freq, sections=sections, interleaved=interleaved, scale=1.25)
    assert rq.is_contiguous() and torch.equal(q, q0) and torch.equal(k, k0)
    check_rope(hip, q, rq, positions, inv_freq, sections, interleaved, 1.25)
    check_rope(hip, k, rk, positions, inv_freq, sections, interleaved, 1.25)
    iq, none = hip.rope(q, None, positions, inv_freq, sections=sections, interleaved=interleaved, scale=1.25, out=(q, None))
    assert none is None and iq is q and torch.equal(q, rq)  # in place: the same bits


def test_rope_refusals(hip):
    q = torch.zeros(2, 1, 64, device=DEV)
    f = torch.ones(8, dtype=torch.float64, device=DEV)
    p = torch.zeros(3, 2, dtype=torch.int64, device=DEV)
    for sections in ((8, 1, 0), (1, 3, 4), (4, 4), (9, -1, 0)):
        with pytest.raises(ValueError):
            hip.rope(q, None, p, f, sections=sections)
    for bad in (lambda: hip.rope(q.half(), None, p, f, sections=(3, 3, 2)), lambda: hip.rope(q, q.bfloat16(), p, f, sections=(3, 3, 2)),
                lambda: hip.rope(q, None, p.int(), f, sections=(3, 3, 2)), lambda: hip.rope(q, None, p, f.float(), sections=(3, 3, 2)),
                lambda: hip.rope(q, None, p[:, :1], f, sections=(3, 3, 2)), lambda: hip.rope(q[..., :8], None, p, f, sections=(3, 3, 2)),
                lambda: hip.rope(q.cpu(), None, p, f, sections=(3, 3, 2)), lambda: hip.rope(q, torch.zeros(3, 1, 64, device=DEV), p, f, sections=(3, 3, 2))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("counts", [(4, 2, 3), (70, 3, 33)])
def test_attend_length_beyond_the_table(hip, counts, page):
    """Lengths that the table has no pages for: the tokens behind its width are not there, and the rows stand at the positions
    that the lengths say, so the last ones see all that is there."""
    g = gen(19)
    pages = random_pages(hip, g, 1, 10, 2, page, 64, torch.int8)
    table = table_of(g, (3 * page,) * 3, page, 10)
    q = torch.randn(sum(counts), 8, 64, generator=g).to(torch.bfloat16).to(DEV)
    for beyond in (1, counts[0] - 2, 2 ** 31 - 1 - 3 * page):
        check_attend(hip, pages, 0, q, table, i32([3 * page + beyond, 3 * page - 1, 3 * page + 2]), cu_of(counts), max_count=max(counts))


def test_rope_into_rows_that_share_memory(hip):
    q = torch.randn(4, 2, 64, device=DEV)
    f, p = torch.ones(32, dtype=torch.float64, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    one = torch.zeros(1, 2, 64, device=DEV)
    for out in (one.expand(4, 2, 64), torch.zeros(4, 1, 64, device=DEV).expand(4, 2, 64),
                torch.zeros(1000, device=DEV).as_strided((4, 2, 64), (100, 50, 1))):
        before = out.clone()
        with pytest.raises(ValueError):
            hip.rope(q, None, p, f, out=(out, None))
        with pytest.raises(ValueError):
            hip.rope(q, q, p, f, out=(None, out))
        assert torch.equal(out, before)
    with pytest.raises(ValueError):
        hip.rope(one.expand(4, 2, 64), None, p, f, out=(one.expand(4, 2, 64), None))  # in place
    a, _ = hip.rope(one.expand(4, 2, 64), None, p, f)  # to be read they may
    assert torch.equal(a, torch.zeros_like(q))
    apart = torch.zeros(2, 4, 64, device=DEV).transpose(0, 1)  # heads outermost
    assert torch.equal(hip.rope(q, None, p, f, out=(apart, None))[0], hip.rope(q, None, p, f)[0])


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("dim,page,counts,starts", [(256, 128, (300,), (37,)), (64, 1024, (1500,), (3,)), (128, 512, (700, 513), (0, 511)),
                                                    (256, 1024, (2100,), (1023,))])
@pytest.mark.parametrize("layout", ["fused", "odd"])
def test_append_large_blocks(hip, dtype, dim, page, counts, starts, layout):
    """Blocks with more new values than the threads keep (16384): what is beyond is read a second time."""
    g = gen(dim + page + 1)
    pages = random_pages(hip, g, 1, 6, 2, page, dim, dtype)
    table = table_of(g, [c + s for c, s in zip(counts, starts)], page, 6)
    wide = torch.randn(sum(counts), 2, 2, dim + (3 if layout == "odd" else 0), generator=g)
    wide[:, 0] *= 1 + 20 * (torch.rand(wide.shape[-1], generator=g) < 0.05)
    wide[-1, :, :, 5] = 90.0  # the largest of the last block is in its last row
    x = wide.to(torch.bfloat16).to(DEV)[..., 1 if layout == "odd" else 0:][..., :dim]
    check_append(hip, pages, 0, x[:, 0], x[:, 1], table, i32(starts), cu_of(counts))


@pytest.mark.parametrize("count", [1, 20])
@pytest.mark.parametrize("dim,page", [(256, 64), (128, 64), (64, 128), (256, 32), (128, 1024)])
def test_attend_nan_stays_where_it_is_on_whole_pages(hip, dim, page, count):
    """As on small pages, where a page holds whole tiles: stray e4m3 NaN bytes reach no row, a NaN scale just the rows that see its
    block, missing pages nobody."""
    g = gen(21)
    lengths = [n * page // 32 for n in (75, 130, 40)]
    pages = random_pages(hip, g, 1, 10, 2, page, dim, torch.float8_e4m3fn)
    table = table_of(g, lengths, page, 10)
    raw_k, raw_v = pages.k.view(torch.uint8), pages.v.view(torch.uint8)
    used = set()
    for b, n in enumerate(lengths):
        for c in range(-(-n // page)):
            p = int(table[b, c])
            used.add(p)
            raw_k[0, p, :, max(0, n - page * c):] = 0x7F
            raw_v[0, p, :, :, max(0, n - page * c):] = 0xFF
    for p in set(range(10)) - used:
        raw_k[0, p], raw_v[0, p] = 0x7F, 0x7F
        pages.k_scale[0, p], pages.v_scale[0, p] = math.nan, math.nan
    q = torch.randn(3 * count, 4, dim, generator=g).to(torch.bfloat16).to(DEV)
    args = (i32(lengths), cu_of((count,) * 3))
    for causal in (True, False):
        out = check_attend(hip, pages, 0, q, table, *args, causal=causal)
        assert torch.isfinite(out.float()).all()
        missing = table.clone()
        missing[1, 2], missing[2, 0], missing[0, 0] = -1, 10, 2 ** 31 - 1
        check_attend(hip, pages, 0, q, missing, *args, causal=causal)
    last = int(table[1, 4])
    for scale, head in ((pages.v_scale, 1), (pages.k_scale, 0)):
        scale[0, last, head] = math.nan  # the last tokens of sequence 1
        out = check_attend(hip, pages, 0, q, table, *args)
        assert torch.isnan(out[2 * count - 1, 2 * head:2 * head + 2].float()).all()
    seen = torch.isnan(check_attend(hip, pages, 0, q, table, *args).float())
    assert seen[2 * count - 1].all() and not seen[:count].any() and not seen[2 * count:].any()


@pytest.mark.parametrize("dim,kv_heads,seqs", [(64, 8, 64), (128, 8, 64), (64, 16, 33)])
def test_attend_one_long_sequence_among_many(hip, dim, kv_heads, seqs):
    """As many short (sequence, kv head)s as leave nothing to be cut, and a long one among them."""
    g = gen(22)
    lengths = [7 + i % 90 for i in range(seqs)]
    lengths[seqs // 2] = 6000
    need = sum(-(-n // 64) for n in lengths)
    pages = random_pages(hip, g, 1, need, kv_heads, 64, dim, torch.int8)
    table = table_of(g, lengths, 64, need)
    q = torch.randn(5 * seqs, 4 * kv_heads, dim, generator=g).to(torch.bfloat16).to(DEV)
    check_attend(hip, pages, 0, q, table, i32(lengths), cu_of([5] * seqs), max_count=5)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("heads,kv_heads,dim,count", [(16, 2, 256, 1), (16, 2, 256, 40), (32, 8, 128, 4), (32, 8, 128, 30), (8, 8, 64, 20)])
def test_attend_error_as_a_whole(hip, dtype, heads, kv_heads, dim, count):
    """The 2-norm of the error over that of the result, for a long cache, where the largest possible error says little. Independent
    values: rounding the result leaves 2^-8 / sqrt(3) at most (an error spread evenly over a step, of the smallest significand), and
    rounding the weights as much again, since weights and result have the same relative spread."""
    g = gen(23)
    lengths, seqs = (3000, 2500), 2
    pages = random_pages(hip, g, 1, 90, kv_heads, 64, dim, dtype)
    table = table_of(g, lengths, 64, 90)
    q = torch.randn(count * seqs, heads, dim, generator=g).to(torch.bfloat16).to(DEV)
    out = hip.kv_attend(pages, 0, q, table, i32(lengths), cu_of([count] * seqs), max_count=count).cpu().double()
    want, _ = kv_ref.attend(pages.k[0].cpu(), pages.v[0].cpu(), pages.k_scale[0].cpu(), pages.v_scale[0].cpu(), q.cpu(), table.cpu(),
                            i32(lengths).cpu(), cu_of([count] * seqs).cpu())
    assert (out - want).norm() <= 2 ** 0.5 * 2.0 ** -8 / 3 ** 0.5 * want.norm()


@pytest.mark.parametrize("dim,kv_heads,group,seqs,count,far", [
    (64, 16, 4, 33, 5, (9000, 8300)), (128, 8, 4, 70, 5, (5000, 4100, 4500)), (256, 2, 8, 260, 3, (2100, 4000)), (128, 8, 2, 40, 200, (6000,))])
def test_attend_long_ones_are_cut(hip, dim, kv_heads, group, seqs, count, far):
    """From 512 (row tile, kv head)s on, where the bound of the lengths allows for long ones: some are, among short ones, ones without
    rows and ones without tokens. The same with a bound that is far too small (nothing is cut) or none, and with any workspace."""
    g = gen(24)
    rng = np.random.default_rng(24)
    lengths = [int(x) for x in rng.integers(0, 120, seqs)]
    counts = [int(x) for x in rng.integers(0, count + 1, seqs)]
    for i, n in enumerate(far):
        lengths[5 + 7 * i], counts[5 + 7 * i] = n, count
    lengths[seqs - 1], counts[0] = 0, 0
    need = sum(-(-n // 64) for n in lengths)
    pages = random_pages(hip, g, 1, need, kv_heads, 64, dim, torch.float8_e4m3fn)
    table = table_of(g, lengths, 64, need)
    q = torch.randn(sum(counts), group * kv_heads, dim, generator=g).to(torch.bfloat16).to(DEV)
    args = (q, table, i32(lengths), cu_of(counts))
    rows_of = [5 + 7 * i for i in range(len(far))]
    bounds = args[3].tolist()
    out = hip.kv_attend(pages, 0, *args, max_count=count)
    some = sorted({r for b in rows_of for r in (bounds[b], bounds[b + 1] - 1)} | set(range(0, q.shape[0], max(1, q.shape[0] // 60))))
    cache = [x[0].cpu() for x in (pages.k, pages.v, pages.k_scale, pages.v_scale)]
    for r in some:
        b = next(b for b in range(seqs) if bounds[b] <= r < bounds[b + 1])
        seen = lengths[b] - (bounds[b + 1] - 1 - r)
        want, tol = kv_ref.attend(*cache, q[r:r + 1].cpu(), table[b:b + 1].cpu(), torch.tensor([max(seen, 0)]), torch.tensor([0, 1]))
        assert ((out[r].cpu().double() - want[0]).abs() <= tol[0]).all(), (r, b)
    assert torch.equal(out, hip.kv_attend(pages, 0, *args, max_count=count, max_length=max(far)))
    ws = torch.full((300 << 20,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(out, hip.kv_attend(pages, 0, *args, max_count=count, workspace=ws))
    uncut = hip.kv_attend(pages, 0, *args, max_count=count, max_length=64)
    # both lie within their bound of the exact result: 2^-8 of themselves and of the mean weighted value
    assert (out.float() - uncut.float()).abs().max() <= 2.0 ** -5 * out.float().abs().max()
