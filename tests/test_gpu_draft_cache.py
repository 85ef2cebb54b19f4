"""Drafts and windows on HBMKVCache and HipAttention as a model's loop uses them: trees drafted, checked and partly kept, round after
round, on several sequences, forks and streams; against oracle/kv_ref.py on the cache's own contents."""
import random
import types

import pytest
import torch
import torch.nn.functional as F

from gguf.hbm_cache import HBMKVCache
from oracle import kv_ref
from test_gpu_draft import random_tree
from test_gpu_kv_cache import assert_within, bf16, engine, oracle_attend, stored, worst

pytestmark = pytest.mark.gpu
DEV = "cuda"


def path_to(tree, node):
    line = [node]
    while tree[line[0]] >= 0:
        line.insert(0, tree[line[0]])
    return line


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 3)])
def test_rounds_of_drafts(hip, dtype, window, sinks):
    """Trees of drafts appended, attended, and a path of each kept: what the cache then holds are the kept tokens' own keys and
    values. A value is rounded when it is written, when it moves, and by less than one step in all when its page's scale grows."""
    rng, g = random.Random(3), torch.Generator().manual_seed(3)
    cache = HBMKVCache(layers=2, pages=60, kv_heads=2, head_dim=64, page_tokens=16, dtype=dtype)
    seqs = [cache.new() for _ in range(3)]
    kept = {s: [(torch.empty(0, 2, 64), torch.empty(0, 2, 64))] * 2 for s in seqs}
    largest = 0.0
    for turn in range(14):
        live = rng.sample(seqs, rng.randint(1, 3))
        counts = [rng.choice((1, 7, 20, 40)) for _ in live]
        trees = [random_tree(rng, n) for n in counts]
        step = cache.step(live, counts)
        tree, positions = cache.tree(step, torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=DEV))
        want = [cache.length(s) - n + len(path_to(t, i)) - 1 for s, n, t in zip(live, counts, trees) for i in range(n)]
        assert positions.tolist() == want
        new = []
        for layer in range(2):
            k, v, q = bf16(g, sum(counts), 2, 64), bf16(g, sum(counts), 2, 64), bf16(g, sum(counts), 6, 64)
            cache.append(layer, step, k, v)
            limits = dict(window=window, sinks=sinks) if window else {}
            assert_within(cache.attend(layer, step, q, tree=tree, **limits), *oracle_attend(cache, layer, step, q, tree=tree.cpu(), **limits))
            new.append((k.float().cpu(), v.float().cpu()))
        largest = max(largest, float(cache.pages.k_scale.max()), float(cache.pages.v_scale.max()))
        accepted = [path_to(t, rng.randrange(n))[:rng.randint(0, n)] for t, n in zip(trees, counts)]
        cache.keep(live, counts, accepted)
        at = 0
        for s, n, a in zip(live, counts, accepted):
            rows = [at + i for i in a]
            kept[s] = [tuple(torch.cat((o, x[rows])) for o, x in zip(old, kv)) for old, kv in zip(kept[s], new)]
            at += n
        for s in seqs:
            assert cache.length(s) == len(kept[s][0][0])
            if not cache.length(s):
                continue
            for layer in range(2):
                for (x, step_size), want in zip(stored(cache, layer, s), kept[s][layer]):
                    want = want.double()
                    # int8: a step of the page it was written into, half a one of its own, and one for its growth; e4m3: half a
                    # step of its magnitude three times (each of what the last left), or of the smallest values' steps
                    tol = largest + 1.5 * step_size if dtype == torch.int8 else 3.4 * 2.0 ** -4 * want.abs() + 2.0 ** -9 * (largest + 1.5 * step_size)
                    assert ((x - want).abs() <= tol).all(), f"turn {turn}, sequence {s}, layer {layer}"
    # decoding goes on behind them
    step = cache.step(seqs, [1, 1, 1])
    q = bf16(g, 3, 6, 64)
    cache.append(0, step, bf16(g, 3, 2, 64), bf16(g, 3, 2, 64))
    assert_within(cache.attend(0, step, q), *oracle_attend(cache, 0, step, q))


def test_keep_beside_forks(hip):
    """A fork made before the draft keeps its tokens; one made behind it makes keep() refuse, with nothing changed."""
    g = torch.Generator().manual_seed(4)
    cache = HBMKVCache(1, 20, 2, 64, 16)
    a = cache.new()
    step = cache.step([a], [20])
    cache.append(0, step, bf16(g, 20, 2, 64), bf16(g, 20, 2, 64))
    b = cache.fork(a)
    before = [x.clone() for x, _ in stored(cache, 0, b)]
    step = cache.step([a], [30])
    cache.append(0, step, bf16(g, 30, 2, 64), 9 * bf16(g, 30, 2, 64))
    drafted = [x.clone() for x, _ in stored(cache, 0, a)]
    c = cache.fork(a)
    with pytest.raises(ValueError, match="another"):
        cache.keep([a], [30], [[1, 2, 29]])
    assert all(torch.equal(x, y) for (x, _), y in zip(stored(cache, 0, a), drafted)) and cache.length(a) == 50
    cache.free(c)
    cache.keep([a], [30], [[1, 2, 29]])
    assert cache.length(a) == 23 and all(torch.equal(x, y) for (x, _), y in zip(stored(cache, 0, b), before))
    for (x, step_size), y in zip(stored(cache, 0, a), drafted):
        assert ((x[20:] - y[[21, 22, 49]]).abs() <= 1.5 * step_size[20:]).all()


def test_keep_is_not_captured(hip):
    cache = HBMKVCache(1, 4, 2, 64, 16)
    a = cache.new()
    cache.step([a], [10])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            cache.keep([a], [5], [[3]])
    graph.replay()
    torch.cuda.synchronize()
    assert cache.length(a) == 10


@pytest.mark.parametrize("seed", [0, 1])
def test_drafts_on_changing_streams(hip, seed):
    """The same rounds of drafts on one stream and on three in turn, without a synchronization: the same answers and the same cache."""
    streams = [torch.cuda.current_stream()] + [torch.cuda.Stream() for _ in range(2)]
    g = torch.Generator().manual_seed(21)
    k, v, q = bf16(g, 4000, 2, 128), bf16(g, 4000, 2, 128), bf16(g, 4000, 16, 128)
    parents = torch.tensor(random_tree(random.Random(seed), 64), dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()

    def lives(changing):
        rng, which = random.Random(seed), random.Random(seed + 50)

        def move():
            torch.cuda.set_stream(streams[which.randrange(3) if changing else 0])
        cache = HBMKVCache(2, 200, 2, 128, 64)
        torch.cuda.synchronize()
        seqs, outs = [cache.new() for _ in range(3)], []
        step = cache.step(seqs, [900, 2000, 50])
        for layer in range(2):
            cache.append(layer, step, k[:2950], v[:2950])
        for _ in range(20):
            move()
            n, at = rng.randint(2, 64), rng.randint(0, 3000)
            live = rng.sample(seqs, rng.randint(1, 3))
            rows = slice(at, at + n * len(live))
            step = cache.step(live, [n] * len(live))
            move()
            tree, _ = cache.tree(step, parents[:n].repeat(len(live)))
            for layer in range(2):
                cache.append(layer, step, k[rows], v[rows])
                outs.append(cache.attend(layer, step, q[rows], tree=tree))
                outs.append(cache.attend(layer, step, q[rows], window=200, sinks=4))
            move()
            cache.keep(live, [n] * len(live), [sorted(rng.sample(range(n), rng.randint(0, n))) for _ in live])
        torch.cuda.set_stream(streams[0])
        torch.cuda.synchronize()
        return outs, [getattr(cache.pages, name) for name in ("k", "v", "k_scale", "v_scale")]
    want, pools = lives(False)
    try:
        for _ in range(3):
            got, mine = lives(True)
            assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))
            assert all(torch.equal(a, b) for a, b in zip(mine, pools))
    finally:
        torch.cuda.set_stream(streams[0])


def test_padded_draft(hip):
    """Padding rows behind a step's tokens: no bits, position 0, and zeros from attend."""
    g = torch.Generator().manual_seed(5)
    cache = HBMKVCache(1, 20, 2, 64, 16)
    seqs = [cache.new(), cache.new()]
    step = cache.step(seqs, [40, 5])
    cache.append(0, step, bf16(g, 45, 2, 64), bf16(g, 45, 2, 64))
    step = cache.step(seqs, [6, 4])
    parents = torch.tensor([-1, 0, 0, 1, 1, 2, -1, 0, 1, 2, 5, 5, 5], dtype=torch.int32, device=DEV)
    tree, positions = cache.tree(step, parents)
    assert not tree[10:].any() and not positions[10:].any()
    q = bf16(g, 13, 8, 64)
    cache.append(0, step, bf16(g, 13, 2, 64), bf16(g, 13, 2, 64))
    for kw in (dict(tree=tree), dict(window=7, sinks=2), dict(tree=tree, window=7)):
        full = torch.full((100000,), float("nan"), device=DEV, dtype=torch.bfloat16)
        del full
        out = cache.attend(0, step, q, **kw)
        assert (out[10:] == 0).all()
        ref = {n: x.cpu() if n == "tree" else x for n, x in kw.items()}
        want, tol = oracle_attend(cache, 0, step, q, **ref)
        assert_within(out[:10], want[:10], tol[:10])


@pytest.mark.parametrize("gated,norm", [(True, True), (False, True), (True, False)])
def test_engine_drafts(hip, monkeypatch, gated, norm):
    """HipAttention over a prompt, a drafted tree and what is kept of it, in a window and without: queries and keys against the
    norms' and positions' formulas in 64 bits, attention against the oracle on the cache's contents."""
    g, rng = torch.Generator().manual_seed(16), random.Random(16)
    eng, heads, dim = engine(g, gated, False, norm)
    cache, p, seen = eng.kv_cache, "model.layers.3.self_attn", {}
    append, attend, linear = cache.append, cache.attend, F.linear

    def append_(layer, step, k, v):
        seen["k"] = k
        return append(layer, step, k, v)

    def attend_(layer, step, q, **kw):
        seen["q"], seen["kw"], seen["o"] = q, kw, attend(layer, step, q, **kw)
        return seen["o"]

    def linear_(x, w):
        name = next(n for n in ("q", "k", "v", "o") if eng.weights[f"{p}.{n}_proj.weight"] is w)
        seen[name + " proj"] = linear(x, w)
        return seen[name + " proj"]
    cache.append, cache.attend = append_, attend_
    monkeypatch.setattr("engines.qwen36.attention_hip.F", types.SimpleNamespace(linear=linear_))
    seqs = [cache.new(), cache.new()]
    for turn, counts in enumerate(((30, 11), (20, 9), (1, 1), (33, 2))):
        n, trees = sum(counts), [random_tree(rng, c) for c in counts]
        starts = [cache.length(s) for s in seqs]
        step = cache.step(seqs, counts)
        drafts = turn % 2 == 1
        if drafts:
            tree, ids = cache.tree(step, torch.tensor([x for t in trees for x in t], dtype=torch.int32, device=DEV))
        else:
            tree, ids = None, torch.cat([torch.arange(a, a + c) for a, c in zip(starts, counts)])
        kw = dict(window=35, sinks=2, tree=tree) if turn != 1 else dict(tree=tree)
        positions = eng.rotary.positions(ids)
        y = eng.hip_attention(bf16(g, n, 256), 3, 0, step, positions, **kw)
        assert y.shape == (n, 256) and all(seen["kw"].get(name) is x or seen["kw"].get(name) == x for name, x in kw.items())
        wide = seen["q proj"].cpu().double()
        raw = {"q": wide.view(n, heads, 2, dim)[:, :, 0] if gated else wide.view(n, heads, dim), "k": seen["k proj"].cpu().double().view(n, 2, dim)}
        for name in "qk":
            z = kv_ref.norm(raw[name], eng.weights[f"{p}.{name}_norm.weight"], 1e-6) if norm else raw[name]
            want = kv_ref.rope(z, positions.cpu(), eng.rotary.inv_freq.cpu(), (6, 5, 5), True)
            pair = z.abs().clone()
            pair[..., :32] = (pair[..., :16] + pair[..., 16:32]).repeat(1, 1, 2)
            # the norm in fp32 (64 squares, a root, products), cosine and sine; one rounding to bf16
            bound = pair * (2.0 ** -20 + 40 * 2.0 ** -24) * 1.01 + want.abs() * 2.0 ** -8
            assert worst(seen[name], want, bound) <= 1
            if norm:
                assert worst(seen[name], kv_ref.rope(raw[name], positions.cpu(), eng.rotary.inv_freq.cpu(), (6, 5, 5), True), bound) > 10
        ref = {name: x.cpu() if name == "tree" else x for name, x in kw.items() if x is not None}
        assert worst(seen["o"], *oracle_attend(cache, 0, step, seen["q"], **ref)) <= 1
        if drafts:
            assert worst(seen["o"], *oracle_attend(cache, 0, step, seen["q"])) > 4  # what no mask would give
            cache.keep(seqs, counts, [path_to(t, c - 1) for t, c in zip(trees, counts)])
            assert [cache.length(s) for s in seqs] == [a + len(path_to(t, c - 1)) for a, t, c in zip(starts, trees, counts)]


@pytest.mark.parametrize("shapes", [((1, 64), (1, 64)), ((1,), (1,)), ((8, 64), (2, 64)), ((64,), (1, 64))])
def test_engine_norm_weights_of_any_shape(hip, shapes):
    """Norm weights that are not one vector for all heads go through HipAttention: the layer's result is that of the norms in front of
    the rotary positions."""
    outs = []
    for own in (False, True):
        g = torch.Generator().manual_seed(18)
        eng, heads, dim = engine(g, True, False, True)
        p = "model.layers.3.self_attn"
        for name, shape, n in zip("qk", shapes, (heads, 2)):
            shape = tuple(n if x == 8 else x for x in shape)
            eng.weights[f"{p}.{name}_norm.weight"] = (0.3 * torch.randn(shape, generator=g)).to(DEV)
        if own:  # a rotary that knows nothing of norms
            inner = eng.rotary
            eng.rotary = lambda q, k, positions: inner(q, k, positions)
        step = eng.kv_cache.step([eng.kv_cache.new()], [21])
        outs.append(eng.hip_attention(bf16(g, 21, 256), 3, 0, step, torch.arange(21, device=DEV).expand(3, -1).contiguous()))
    assert torch.equal(*outs) and torch.isfinite(outs[0].float()).all()


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_keep_past_a_shared_page(hip, dtype):
    """A fork made behind the draft that shares just a page whose kept tokens stay in their places: keep() moves the others, and the
    fork's tokens stay as they are."""
    g = torch.Generator().manual_seed(6)
    cache = HBMKVCache(2, 20, 2, 64, 16, dtype=dtype)
    a = cache.new()
    for n in (8, 40):
        step = cache.step([a], [n])
        for layer in range(2):
            cache.append(layer, step, bf16(g, n, 2, 64), bf16(g, n, 2, 64))
    f = cache.fork(a)
    cache.truncate(f, 16)
    drafted = [[x.clone() for x, _ in stored(cache, layer, a)] for layer in range(2)]
    kept = list(range(8)) + [10, 11, 39]
    cache.keep([a], [40], [kept])
    assert cache.length(a) == 19 and cache.length(f) == 16
    for layer in range(2):
        for (x, step_size), (y, _), was in zip(stored(cache, layer, a), stored(cache, layer, f), drafted[layer]):
            assert torch.equal(x[:16], was[:16]) and torch.equal(y, was[:16])
            want = was[[8 + i for i in kept[8:]]]
            # rounded once, to half a step, of a quotient in fp32
            tol = 0.501 * step_size[16:] if dtype == torch.int8 else 1.001 * (2.0 ** -4 * want.abs() + 2.0 ** -10 * step_size[16:])
            assert ((x[16:] - want).abs() <= tol).all()


def test_what_is_refused_under_capture_is_named(hip):
    cache = HBMKVCache(1, 4, 2, 64, 16)
    a = cache.new()
    cache.step([a], [10])
    torch.cuda.synchronize()
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        x.add_(1)
        for name, call in (("step", lambda: cache.step([a], [1])), ("compact", cache.compact), ("keep", lambda: cache.keep([a], [5], [[3]]))):
            with pytest.raises(RuntimeError, match=rf"{name}\(\).* cannot be captured"):
                call()
    torch.cuda.synchronize()
    assert cache.length(a) == 10
