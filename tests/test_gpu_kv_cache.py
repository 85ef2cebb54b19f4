"""HBMKVCache, the rotary positions and HipAttention together on the GPU, as a model's loop uses them: prompts, decoding,
forks, truncation, compaction, HIP graphs, several streams; against oracle/kv_ref.py on the cache's own contents."""
import random
import types

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from engines.qwen36 import HipAttention, Rotary
from gguf import synth
from gguf.hbm_cache import HBMKVCache, OutOfPages
from gguf.hip import GGMLWeight, kv_attend
from oracle import kv_ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bf16(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).to(DEV)


def oracle_attend(cache, layer, step, q, **kw):
    p = cache.pages
    return kv_ref.attend(p.k[layer].cpu(), p.v[layer].cpu(), p.k_scale[layer].cpu(), p.v_scale[layer].cpu(), q.cpu(),
                         step.table.cpu(), step.length.cpu(), step.cu.cpu(), **kw)


def assert_within(got, want, tol):
    err = (got.cpu().double() - want).abs()
    assert (err <= tol).all(), f"off by {float((err / (tol + 1e-300)).max()):.2f} of the bound"


def stored(cache, layer, seq):
    """(keys, values) of a sequence as the cache holds them, fp64 [tokens, kv_heads, head_dim], and each value's step."""
    p, (length, pages) = cache.pages, cache.book.sequences[seq]
    ids = torch.tensor(pages, dtype=torch.long)
    out = []
    for pool, scale, flip in ((p.k, p.k_scale, False), (p.v, p.v_scale, True)):
        x, s = pool[layer].cpu().double()[ids], scale[layer].cpu().double()[ids]
        x = x.transpose(2, 3) if flip else x
        tokens = lambda y: y.transpose(1, 2).reshape(-1, *y.shape[1:2], y.shape[3])[:length]  # noqa: E731
        out.append((tokens(x * s[:, :, None, None]), tokens((s[:, :, None, None] * torch.ones_like(x)))))
    return out


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_lives_of_sequences(hip, dtype):
    """Prompts, single tokens, forks, cuts, frees and compactions in random order: every live sequence holds its own keys and
    values, each within one step of its block, and attends to just those."""
    rng, g = random.Random(5), torch.Generator().manual_seed(5)
    cache = HBMKVCache(layers=2, pages=12, kv_heads=2, head_dim=64, page_tokens=16, dtype=dtype)
    kept = {}  # seq -> [(k, v) of each layer]
    full = 0
    for i in range(90):
        live = list(kept)
        what = rng.choice(("new", "fork", "truncate", "free", "compact") + 6 * ("step",))
        if what == "new" or not live:
            kept[cache.new()] = [(torch.empty(0, 2, 64), torch.empty(0, 2, 64))] * 2
        elif what == "step":
            seqs = rng.sample(live, rng.randint(1, min(3, len(live))))
            counts = [rng.choice((1, 1, 3, 17, 40)) for _ in seqs]
            try:
                step = cache.step(seqs, counts)
            except OutOfPages:
                full += 1
                s = rng.choice(live)
                cache.free(s)
                del kept[s]
                continue
            for layer in range(2):
                k, v = bf16(g, sum(counts), 2, 64, scale=1 + i % 4), bf16(g, sum(counts), 2, 64)
                q = bf16(g, sum(counts), 6, 64)
                cache.append(layer, step, k, v)
                out = cache.attend(layer, step, q)
                assert_within(out, *oracle_attend(cache, layer, step, q))
                at = 0
                for s, n in zip(seqs, counts):
                    old = kept[s][layer]
                    new = tuple(torch.cat((o, x[at:at + n].float().cpu())) for o, x in zip(old, (k, v)))
                    kept[s] = [new if l == layer else kept[s][l] for l in range(2)]
                    at += n
        elif what == "fork":
            s = rng.choice(live)
            kept[cache.fork(s)] = list(kept[s])
        elif what == "truncate":
            s = rng.choice(live)
            n = rng.randint(0, cache.length(s))
            cache.truncate(s, n)
            kept[s] = [tuple(x[:n] for x in kv) for kv in kept[s]]
        elif what == "free":
            s = rng.choice(live)
            cache.free(s)
            del kept[s]
        else:
            cache.compact()
            assert all(p < cache.book.used() for v in cache.book.sequences.values() for p in v[1])
        for s, layers in kept.items():
            assert cache.length(s) == len(layers[0][0])
            if not cache.length(s):
                continue
            for layer in range(2):
                for (x, step_size), want in zip(stored(cache, layer, s), layers[layer]):
                    # int8: under one step of the final scale. e4m3: half a step of its own magnitude (2^-4), and where a
                    # grown scale pushed it below the normal ones, one of the smallest steps (2^-9) of the final scale
                    tol = step_size if dtype == torch.int8 else 2.0 ** -4 * want.double().abs() + 2.0 ** -9 * step_size
                    assert ((x - want.double()).abs() <= tol).all(), f"sequence {s}, layer {layer}"
    assert full  # the cache did run out of pages on the way


def test_prompt_by_pages(hip):
    """A prompt in chunks that end with pages leaves the same bytes as the prompt at once, and the same answers."""
    g = torch.Generator().manual_seed(6)
    k, v, q = bf16(g, 300, 2, 128), bf16(g, 300, 2, 128), bf16(g, 300, 8, 128)
    caches = [HBMKVCache(1, 8, 2, 128, 64) for _ in range(2)]
    a, b = (c.new() for c in caches)
    step = caches[0].step([a], [300])
    caches[0].append(0, step, k, v)
    whole = caches[0].attend(0, step, q)
    parts = []
    for lo, hi in ((0, 64), (64, 256), (256, 300)):
        step = caches[1].step([b], [hi - lo])
        caches[1].append(0, step, k[lo:hi], v[lo:hi])
        parts.append(caches[1].attend(0, step, q[lo:hi]))
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(caches[0].pages, name), getattr(caches[1].pages, name))
    want, tol = oracle_attend(caches[0], 0, _as_step(caches[0], a, 300), q)
    assert_within(whole, want, tol)
    assert_within(torch.cat(parts), want, tol)


def _as_step(cache, seq, count):
    class S:
        pass
    s, (length, pages) = S(), cache.book.sequences[seq]
    s.table, s.length = torch.tensor([pages], dtype=torch.int32), torch.tensor([length], dtype=torch.int32)
    s.cu = torch.tensor([0, count], dtype=torch.int32)
    return s


def test_decode_graph(hip):
    """One decode step (rotary, append, attend over two layers) captured once and replayed for later tokens after refresh(),
    with eager work and synchronizations in between: the same bits as eager steps on a cache of its own."""
    g = torch.Generator().manual_seed(7)
    rotary = Rotary(256, 64, 1e7, (11, 11, 10))
    prompt, T = (70, 33, 128), 3
    caches, seqs = [HBMKVCache(2, 24, 2, 256, 64) for _ in range(2)], []
    filled = [(bf16(g, sum(prompt), 2, 256), bf16(g, sum(prompt), 2, 256)) for _ in range(2)]
    for c in caches:
        ids = [c.new() for _ in prompt]
        seqs.append(ids)
        s = c.step(ids, prompt)
        for layer in range(2):
            c.append(layer, s, *filled[layer])

    def run(cache, step, x, positions):
        outs = []
        for layer in range(2):
            q, k = rotary(x[layer][0], x[layer][1], positions)
            cache.append(layer, step, k, x[layer][2])
            outs.append(cache.attend(layer, step, q))
        return torch.stack(outs)

    def fresh():
        return [(bf16(g, T, 16, 256), bf16(g, T, 2, 256), bf16(g, T, 2, 256)) for _ in range(2)]

    inputs = fresh()
    positions = rotary.positions(torch.tensor(prompt))
    step = caches[0].step(seqs[0], [1] * T, width=6)
    first = caches[1].step(seqs[1], [1] * T, width=6)
    want = run(caches[1], first, inputs, positions)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = run(caches[0], step, inputs, positions)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    for i in range(1, 9):
        new = fresh()
        for old, x in zip(inputs, new):
            for a, b in zip(old, x):
                a.copy_(b)
        positions.add_(1)
        caches[0].refresh(step, seqs[0], [1] * T)
        want = run(caches[1], caches[1].step(seqs[1], [1] * T, width=6), inputs, positions)
        if i % 3 == 0:
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), f"replay {i}"
    with pytest.raises(ValueError):
        caches[0].refresh(step, seqs[0], [2] * T)
    with pytest.raises(ValueError):
        caches[0].step([seqs[0][0]], [400], width=6)


def test_streams_and_workspaces(hip):
    """Calls on two streams at once on one cache, each with its own workspace from the allocator, and with one given."""
    g = torch.Generator().manual_seed(8)
    cache = HBMKVCache(1, 200, 2, 128, 64)
    ids = [cache.new() for _ in range(3)]
    step = cache.step(ids, [3000, 5000, 77])
    cache.append(0, step, bf16(g, 8077, 2, 128), bf16(g, 8077, 2, 128))
    step = cache.step(ids, [1, 1, 1])
    cache.append(0, step, bf16(g, 3, 2, 128), bf16(g, 3, 2, 128))
    qs = [bf16(g, 3, 16, 128) for _ in range(6)]
    want = [cache.attend(0, step, q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for i, q in enumerate(qs):
            with torch.cuda.stream(streams[i % 2]):
                got.append(cache.attend(0, step, q))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    args = (cache.pages, 0, qs[0], step.table, step.length, step.cu)
    ws = torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV)
    assert torch.equal(kv_attend(*args, max_count=1, workspace=ws), want[0])  # whatever the workspace held
    for bad in (ws[:64], ws.view(torch.int8), ws.cpu()):
        with pytest.raises(ValueError):
            kv_attend(*args, max_count=1, workspace=bad)


def test_two_prompt_graphs(hip):
    """Two captured calls of many rows that leave partial results in workspaces of their own, replayed in turn with other
    inputs and lengths, eager calls and synchronizations in between: the eager calls' bits every time."""
    g = torch.Generator().manual_seed(12)
    cache = HBMKVCache(1, 80, 2, 128, 64)
    seqs = [cache.new(), cache.new()]
    first = cache.step(seqs, [2500, 1300])
    cache.append(0, first, bf16(g, 3800, 2, 128), bf16(g, 3800, 2, 128))
    lengths = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ((2500, 1300), (900, 1100))]
    cus = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ((0, 40, 60), (0, 5, 25))]
    qs = [bf16(g, 60, 16, 128), bf16(g, 25, 16, 128)]

    def call(i):
        return kv_attend(cache.pages, 0, qs[i], first.table, lengths[i], cus[i], max_count=40, max_length=2500)
    want = [call(i) for i in range(2)]
    graphs, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for i in range(2):
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[i]):
            got.append(call(i))
    for turn in range(6):
        for i in (0, 1) if turn % 2 else (1, 0):
            qs[i].copy_(bf16(g, *qs[i].shape))
            lengths[i].sub_(turn * 31)
            want[i] = call(i)
            if turn % 3 == 0:
                torch.cuda.synchronize()
            graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"turn {turn}"


class TinyEngine(HipAttention):
    prefix = "model."

    def __init__(self, weights, cache, rotary):
        self.weights, self.kv_cache, self.rotary = weights, cache, rotary


def engine(g, gated, quantized, norm):
    hidden, heads, kv_heads, dim = 256, 4, 2, 64
    p = "model.layers.3.self_attn"
    rows = {"q_proj": (2 if gated else 1) * heads * dim, "k_proj": kv_heads * dim, "v_proj": kv_heads * dim, "o_proj": hidden}
    w = {}
    for i, (name, n) in enumerate(rows.items()):
        if quantized and name != "o_proj":
            raw = synth.q4_k_blocks(np.random.default_rng(i), n * hidden // 256)
            w[f"{p}.{name}.weight"] = GGMLWeight(torch.from_numpy(raw.reshape(-1)).to(DEV), "Q4_K", (n, hidden))
        else:
            w[f"{p}.{name}.weight"] = bf16(g, n, heads * dim if name == "o_proj" else hidden, scale=hidden ** -0.5)
    if norm:
        w[f"{p}.q_norm.weight"], w[f"{p}.k_norm.weight"] = (0.1 * torch.randn(dim, generator=g) for _ in range(2))
    return TinyEngine(w, HBMKVCache(1, 16, kv_heads, dim, 16), Rotary(dim, 32, 1e6, (6, 5, 5))), heads, dim


@pytest.mark.parametrize("gated,quantized,norm", [(True, False, True), (False, False, False), (True, True, True)])
def test_engine_attention(hip, gated, quantized, norm):
    """HipAttention over a ragged prompt and decode steps, against its formula in 64 bits on the projections' own outputs and the
    cache's own contents."""
    g = torch.Generator().manual_seed(9)
    eng, heads, dim = engine(g, gated, quantized, norm)
    cache, p = eng.kv_cache, "model.layers.3.self_attn"
    seqs = [cache.new(), cache.new()]
    at = [0, 0]
    for counts in ((21, 9), (1, 1), (1, 3)):
        n = sum(counts)
        x = bf16(g, n, 256, scale=2.0 ** -9 if quantized else 1.0)
        step = cache.step(seqs, counts)
        ids = torch.cat([torch.arange(a, a + c) for a, c in zip(at, counts)])
        at = [a + c for a, c in zip(at, counts)]
        positions = eng.rotary.positions(torch.stack((ids, ids // 3, ids % 5)))
        y = eng.hip_attention(x, 3, 0, step, positions)
        assert y.shape == (n, 256) and y.dtype == torch.bfloat16
        wide = F.linear(x, eng.weights[f"{p}.q_proj.weight"]).cpu()
        q, gate = wide.view(n, heads, 2, dim).unbind(2) if gated else (wide.view(n, heads, dim), None)
        q64 = q.double()
        if norm:
            q64 = q64 * torch.rsqrt(q64.square().mean(-1, keepdim=True) + 1e-6) * (1 + eng.weights[f"{p}.q_norm.weight"].double())
            q64 = q64.to(torch.float32).to(torch.bfloat16).double()
        turned = kv_ref.rope(q64, positions.cpu(), eng.rotary.inv_freq.cpu(), (6, 5, 5), True)
        want, tol = oracle_attend(cache, 0, step, turned.to(torch.float32).to(torch.bfloat16))
        # q's norm and rotation round to bf16 twice, perhaps to the other neighbour (2^-7 of each value, 2^-6 together): scores
        # move by at most that times sum |q k|, weights by twice as much, relatively
        keys, values = zip(*[[z[0].abs().max() for z in stored(cache, 0, s)] for s in seqs])
        move = 2.0 ** -6 * turned.abs().sum(-1, keepdim=True) * float(max(keys)) * dim ** -0.5
        tol = tol + torch.expm1(2 * move) * float(max(values))
        o, tol = want, tol
        if gated:
            s = torch.sigmoid(gate.double())
            o, tol = o * s, tol * s + 2.0 ** -7 * (o * s).abs()
        w = eng.weights[f"{p}.o_proj.weight"].cpu().double()
        ref = o.reshape(n, -1) @ w.T
        bound = (tol + 2.0 ** -8 * o.abs()).reshape(n, -1) @ w.abs().T + 2.0 ** -8 * ref.abs() + 1e-6
        assert_within(y, ref, bound)


def test_engine_attention_refuses(hip):
    g = torch.Generator().manual_seed(10)
    eng, _, _ = engine(g, True, False, True)
    step = eng.kv_cache.step([eng.kv_cache.new()], [2])
    eng.weights["model.layers.3.self_attn.k_proj.weight"] = bf16(g, 192, 256)
    with pytest.raises(ValueError):
        eng.hip_attention(bf16(g, 2, 256), 3, 0, step, eng.rotary.positions(torch.arange(2)))


@pytest.mark.parametrize("counts,pad", [((3, 1), 12), ((40, 9), 15)])
def test_padded_layer(hip, monkeypatch, counts, pad):
    """A layer over a batch with padding rows behind its tokens: the tokens' rows have the bits of the call without padding, the
    others come out as zeros, whatever the allocator's memory held. Projections in 64 bits, rounded once, since a library's product
    may add up in another order for another number of rows."""
    monkeypatch.setattr(F, "linear", lambda x, w: (x.double() @ w.double().T).to(torch.bfloat16))
    g, n, outs = torch.Generator().manual_seed(14), sum(counts), []
    x = bf16(g, n + pad, 256)
    for rows in (n, n + pad):
        eng = engine(torch.Generator().manual_seed(11), True, False, False)[0]
        step = eng.kv_cache.step([eng.kv_cache.new() for _ in counts], counts)
        positions = eng.rotary.positions(torch.arange(rows))
        full = [torch.full((rows * 256,), float("nan"), device=DEV, dtype=torch.bfloat16) for _ in range(8)]
        del full
        outs.append(eng.hip_attention(x[:rows], 3, 0, step, positions))
    assert torch.equal(outs[1][:n], outs[0]) and outs[0].abs().max() > 0
    assert (outs[1][n:] == 0).all()


@pytest.mark.parametrize("seed", [0, 1])
def test_calls_on_changing_streams(hip, seed):
    """The same lives of sequences (prompts, forks, single tokens, frees, compactions, a replayed graph) on one stream and on three in
    turn, without a synchronization: the same answers and the same cache, bit for bit."""
    streams = [torch.cuda.current_stream()] + [torch.cuda.Stream() for _ in range(2)]
    g = torch.Generator().manual_seed(20)
    k, v, q = bf16(g, 4000, 2, 128), bf16(g, 4000, 2, 128), bf16(g, 4000, 16, 128)
    torch.cuda.synchronize()

    def lives(changing):
        rng, which = random.Random(seed), random.Random(seed + 50)
        cache = HBMKVCache(1, 300, 2, 128, 64)
        torch.cuda.synchronize()
        live, outs = [], []
        decoded, graph = cache.new(), torch.cuda.CUDAGraph()
        step = cache.step([decoded], [1], width=4)
        cache.append(0, step, k[:1], v[:1])
        cache.attend(0, step, q[:1])
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            cache.append(0, step, k[:1], v[:1])
            answer = cache.attend(0, step, q[:1])
        graph.replay()
        for i in range(60):
            torch.cuda.set_stream(streams[which.randrange(3) if changing else 0])
            what = rng.choice(("new", "fork", "token", "token", "token", "free", "compact", "replay"))
            if what == "replay" and cache.length(decoded) < 250:
                cache.refresh(step, [decoded], [1])
                graph.replay()
                outs.append(answer.clone())
                continue
            if what in ("compact", "free") and len(live) > 3:
                if what == "free":
                    cache.free(live.pop(rng.randrange(len(live))))
                else:
                    cache.compact()
                continue
            if what == "fork" and live:
                live.append(cache.fork(rng.choice(live)))
                continue
            if what == "new" or not live:
                live.append(cache.new())
                seqs, counts = live[-1:], [rng.randint(500, 3000)]
            else:
                seqs = rng.sample(live, min(len(live), 3))
                counts = [rng.randint(1, 3) for _ in seqs]
            if cache.book.used() > 220:
                cache.free(live.pop(0))
                continue
            n, at = sum(counts), rng.randint(0, 900)
            s = cache.step(seqs, counts)
            cache.append(0, s, k[at:at + n], v[at:at + n])
            if changing:
                torch.cuda.set_stream(streams[which.randrange(3)])
            outs.append(cache.attend(0, s, q[at:at + n]))
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


def worst(got, want, bound):
    """The largest error over its bound."""
    return float(((got.cpu().double() - want).abs() / (bound + 1e-300)).max())


@pytest.mark.parametrize("gated,quantized,norm", [(True, False, True), (False, False, False), (True, True, True), (True, False, False)])
def test_engine_attention_link_by_link(hip, monkeypatch, gated, quantized, norm):
    """HipAttention's every link against its formula in 64 bits, each on what the link before it gave, so that a bound holds just the
    link's own roundings; and what a wrong link would give lies far outside of it: a result of zeros, a query that is not turned,
    one that is not normed, attention to later tokens, a gate left out, the gate's half taken for the query's."""
    g = torch.Generator().manual_seed(15)
    eng, heads, dim = engine(g, gated, quantized, norm)
    cache, p, seen = eng.kv_cache, "model.layers.3.self_attn", {}
    turn, append, attend, linear = eng.rotary, cache.append, cache.attend, F.linear

    def rotary(q, k, positions):
        seen["q in"], seen["k in"] = q, k
        seen["q"], seen["k"] = turn(q, k, positions)
        return seen["q"], seen["k"]

    def append_(layer, step, k, v):
        seen["k kept"], seen["v kept"] = k, v
        return append(layer, step, k, v)

    def attend_(layer, step, q, **kw):
        seen["q asked"], seen["o"] = q, attend(layer, step, q, **kw)
        return seen["o"].clone()

    def linear_(x, w):
        name = next(n for n in ("q", "k", "v", "o") if eng.weights[f"{p}.{n}_proj.weight"] is w)
        seen[name + " from"], seen[name + " proj"] = x, linear(x, w)
        return seen[name + " proj"]
    eng.rotary, cache.append, cache.attend = rotary, append_, attend_
    monkeypatch.setattr("engines.qwen36.attention_hip.F", types.SimpleNamespace(linear=linear_))

    def normed(x, name):
        w = eng.weights.get(f"{p}.{name}_norm.weight")
        return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
    seqs, at = [cache.new(), cache.new()], [0, 0]
    for counts in ((21, 9), (1, 1), (1, 3), (17, 2)):
        n = sum(counts)
        x = bf16(g, n, 256, scale=2.0 ** -9 if quantized else 1.0)
        step = cache.step(seqs, counts)
        ids = torch.cat([torch.arange(a, a + c) for a, c in zip(at, counts)])
        at = [a + c for a, c in zip(at, counts)]
        positions = turn.positions(torch.stack((ids, ids // 3, ids % 5)))
        y = eng.hip_attention(x, 3, 0, step, positions)
        # the projections of x (quantized ones have tests of their own): 256 products in fp32, one rounding
        for name in "qkv":
            assert torch.equal(seen[name + " from"], x)
            if not quantized:
                w = eng.weights[f"{p}.{name}_proj.weight"].cpu().double()
                want = x.cpu().double() @ w.T
                bound = 2.0 ** -8 * want.abs() + 2.0 ** -14 * (x.cpu().double().abs() @ w.T.abs())  # 257 * 2^-23 < 2^-14
                assert worst(seen[name + " proj"], want, bound) <= 1
        # each head's query, its gate behind it; norms in fp32 (64 squares, a root, two products: under 2^-16), one rounding
        wide = seen["q proj"].cpu().double()
        q, gate = wide.view(n, heads, 2, dim).unbind(2) if gated else (wide.view(n, heads, dim), None)
        k = seen["k proj"].cpu().double().view(n, 2, dim)
        for name, raw in (("q", q), ("k", k)):
            want = normed(raw, name)
            bound = (2.0 ** -8 + 2.0 ** -15) * want.abs() if norm else 0 * want
            assert worst(seen[name + " in"], want, bound) <= 1
            if norm:
                assert worst(seen[name + " in"], raw, bound) > 10
        if gated:
            assert worst(seen["q in"], normed(gate, "q"), (2.0 ** -8 + 2.0 ** -15) * want.abs().max()) > 10
        # positions
        for name in "qk":
            z = seen[name + " in"].cpu().double()
            want = kv_ref.rope(z, positions.cpu(), turn.inv_freq.cpu(), (6, 5, 5), True)
            pair = torch.zeros_like(z)
            pair[..., :32] = (z[..., :16].abs() + z[..., 16:32].abs()).repeat(1, 1, 2)
            bound = pair * 2.0 ** -20 + want.abs() * 2.0 ** -8
            assert worst(seen[name], want, bound) <= 1
        assert seen["q asked"] is seen["q"] and seen["k kept"] is seen["k"]
        assert torch.equal(seen["v kept"], seen["v proj"].view(n, 2, dim))
        # attention over what the cache holds
        want, tol = oracle_attend(cache, 0, step, seen["q"])
        assert worst(seen["o"], want, tol) <= 1
        assert worst(torch.zeros_like(want), want, tol) > 10
        assert worst(seen["o"], *oracle_attend(cache, 0, step, seen["q in"])) > 4
        assert worst(seen["o"], *oracle_attend(cache, 0, step, seen["q"].flip(1))) > 10
        if max(counts) > 4:
            assert worst(seen["o"], *oracle_attend(cache, 0, step, seen["q"], causal=False)) > 10
        # the gate: a sigmoid and a product in fp32, one rounding; then 256 products in fp32 and one rounding
        o = seen["o"].cpu().double()
        w = eng.weights[f"{p}.o_proj.weight"].cpu().double()
        if gated:
            o = o * torch.sigmoid(gate)
        o = o.reshape(n, -1)
        assert worst(seen["o from"], o, (2.0 ** -8 + 2.0 ** -20) * o.abs() if gated else 0 * o) <= 1
        if gated:
            assert worst(seen["o from"], seen["o"].cpu().double().reshape(n, -1), 2.0 ** -7 * o.abs()) > 10
        z = seen["o from"].cpu().double()
        want = z @ w.T
        assert worst(y, want, 2.0 ** -8 * want.abs() + 2.0 ** -14 * (z.abs() @ w.T.abs())) <= 1
        assert torch.equal(y, seen["o proj"])
