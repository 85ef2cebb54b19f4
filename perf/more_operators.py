"""What decoding with drafts and with sliding windows adds to the attention half of a decoder layer, timed.

Kinds of case:
  norm    queries and keys normed head by head (RMS, zero-centred weights) and turned by their positions, in one pass
  window  grouped-query attention over the paged 8-bit cache in which a row sees the last `window` tokens up to its own, and the
          sequence's first `sinks`
  tree    the same over the whole cache for a tree of drafted tokens: a row sees the tokens before the draft, its ancestors in the
          tree and itself; the tree is given by every node's parent, and its positions are worked out with it
  keep    the drafted tokens that were accepted move up in the cache, behind the last token before the draft, on all layers

The cache: k [layers, pages, kv_heads, page_tokens, head_dim], v [layers, pages, kv_heads, head_dim, page_tokens] (int8 or
float8_e4m3fn), k_scale and v_scale fp32 [layers, pages, kv_heads]; a value is byte * scale. A token that moves to another page
is its value divided by that page's scale, rounded to nearest even; where the page's scale does not reach the largest of the
tokens kept in it, it grows by the smallest power of two that does, and the bytes before the draft are divided by that."""
import math
import os
import random
import sys

import torch

own = False

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
DEVICE = "cuda"


def _hip():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "willow-v2_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from gguf import hip
    return hip


# -- cases ---------------------------------------------------------------------------------------------------------


def _norm(tokens, heads=16, kv_heads=2, dim=256, rotary=64, gated=True, bf16=True):
    return {"kind": "norm", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "gated": gated, "bf16": bf16}


def _window(seqs, count, history, window, sinks, dtype="int8", heads=16, kv_heads=2, dim=256, page=64, ragged=False):
    return {"kind": "window", "seqs": seqs, "count": count, "history": history, "window": window, "sinks": sinks, "ragged": ragged,
            "type": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page}


def _tree(seqs, count, history, dtype="int8", heads=16, kv_heads=2, dim=256, page=64, ragged=False):
    return {"kind": "tree", "seqs": seqs, "count": count, "history": history, "ragged": ragged, "type": dtype, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def _keep(seqs, count, accepted, history, layers, dtype="int8", kv_heads=2, dim=256, page=64, ragged=False):
    return {"kind": "keep", "seqs": seqs, "count": count, "accepted": accepted, "history": history, "layers": layers,
            "ragged": ragged, "type": dtype, "kv_heads": kv_heads, "dim": dim, "page": page}


def listed():
    return [
        # one decode step of 64 conversations; q beside its gate in the projection's rows
        dict(_norm(64), name="norm_64"),
        # a prefill chunk with images in it, the benchmark's size
        dict(_norm(4096), name="norm_4096"),
        # a ragged batch of prompts kept in fp32, every value of a head turned
        dict(_norm(777, heads=32, kv_heads=8, dim=128, rotary=128, gated=False, bf16=False), name="norm_fp32"),
        # interactive decoding far into a conversation, on a layer that looks back 1000 tokens
        dict(_window(1, 1, 20000, 1000, 4), name="window_1"),
        # batched serving: 64 conversations of very different lengths
        dict(_window(64, 1, 16000, 4096, 4, ragged=True), name="window_64"),
        # ragged prompts behind earlier turns in one call, smaller heads and pages
        dict(_window(5, 301, 1500, 333, 7, "e4m3", heads=32, kv_heads=8, dim=128, page=32, ragged=True), name="window_ragged"),
        # a prefill chunk behind another
        dict(_window(1, 4096, 4096, 1024, 4), name="window_4096"),
        # one user's drafts of 16 tokens checked at once, behind some hundred tokens
        dict(_tree(1, 16, 776), name="tree_16"),
        # a few users with trees of up to 61 tokens
        dict(_tree(7, 61, 2001, "e4m3", heads=32, kv_heads=8, dim=128, page=32, ragged=True), name="tree_ragged"),
        # 64 drafted tokens far into a long document
        dict(_tree(1, 64, 32000), name="tree_long"),
        # what one user's verification accepted of its tree, in the ten attention layers
        dict(_keep(1, 16, 5, 776, 10), name="keep_1"),
        # the same of 64 conversations with trees of 64 tokens, which mostly reach over a page's end
        dict(_keep(64, 64, 12, 2000, 10, ragged=True), name="keep_64"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 5e14)


def draw(rng: random.Random):
    kind = rng.choice(("norm", "window", "window", "tree", "tree", "keep"))
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        heads, kv_heads, dim = rng.choice(((16, 2, 256), (16, 2, 256), (32, 8, 128), (8, 8, 64), (24, 8, 128), (6, 1, 64)))
        page, dtype = rng.choice((16, 32, 64, 64, 128)), rng.choice(("int8", "e4m3"))
        ragged = rng.random() < 0.6
        if kind == "norm":
            case = _norm(_spread(rng, 1, 4096), heads, kv_heads, dim, rng.choice((dim, dim // 2, dim // 4)), rng.random() < 0.5,
                         rng.random() < 0.7)
        elif kind == "keep":
            count = rng.randint(2, 9) if rng.random() < 0.3 else _spread(rng, 10, 256)
            case = _keep(_spread(rng, 1, 64), count, rng.randint(1, min(count, 24)), rng.choice((0, _spread(rng, 1, 8192))),
                         _spread(rng, 1, 10), dtype, kv_heads, dim, page, ragged)
            if case["seqs"] * (case["history"] + count + page) * kv_heads * dim * case["layers"] > 64 * 2100 * 512 * 10:
                continue
        else:
            if kind == "window":
                count = rng.choice((1, 1, rng.randint(2, 9), _spread(rng, 10, 4096)))
                case = _window(_spread(rng, 1, 64), count, rng.choice((0, _spread(rng, 1, 65536))), _spread(rng, 1, 8192),
                               rng.choice((0, 1, 4, rng.randint(5, 200))), dtype, heads, kv_heads, dim, page, ragged)
            else:
                count = rng.choice((1, rng.randint(2, 9), _spread(rng, 10, 256), _spread(rng, 10, 256)))
                case = _tree(_spread(rng, 1, 64), count, rng.choice((0, _spread(rng, 1, 32768))), dtype, heads, kv_heads, dim, page,
                             ragged)
            # the plain form pads every sequence to the longest, and keeps all scores
            if case["seqs"] * (case["history"] + count) * kv_heads * dim > 64 * 16384 * 512:
                continue
            if case["seqs"] * (case["history"] + count) * count * heads > 8200 * 4100 * 16:
                continue
        if _cost(case) <= most:
            return case


def _sizes(case):
    """(new tokens, tokens held before) of each sequence: the case's own, or spread below them where it is ragged."""
    n, top, past = case["seqs"], case["count"], case["history"]
    if not case["ragged"]:
        return [top] * n, [past] * n
    rng = random.Random(n * 7919 + top * 31 + past)
    counts = [_spread(rng, max(1, top // 8), top) for _ in range(n)]
    held = [_spread(rng, max(1, past // 64), past) if past else 0 for _ in range(n)]
    counts[0], held[-1] = top, past
    return counts, held


def _parents(case):
    """A drafted tree for each sequence, as every node's parent (-1: the last token before the draft), parents first: mostly
    narrow and some levels deep, as drafts that a small model ranks are."""
    rng = random.Random(case["seqs"] * 104729 + case["count"] * 37 + case["history"])
    trees = []
    for n in _sizes(case)[0]:
        depth, tree = [], []
        for i in range(n):
            parent = -1 if i == 0 or rng.random() < 0.04 else max(rng.randrange(i), rng.randrange(i)) if rng.random() < 0.6 else rng.randrange(i)
            tree.append(parent)
            depth.append(0 if parent < 0 else depth[parent] + 1)
        trees.append(tree)
    return trees


def _kept(case, seed):
    """The accepted ones of each sequence's drafted tokens, in order: a path down its tree, which begins with its first node."""
    rng = random.Random(seed * 611953 + case["seqs"] * 37 + case["count"])
    kept = []
    for b, n in enumerate(_sizes(case)[0]):
        a = min(n, case["accepted"] if b == 0 else rng.randint(0, case["accepted"]))
        kept.append([0] + sorted(rng.sample(range(1, n), a - 1)) if a else [])
    return kept


def _seen(case):
    """(visible pairs of row and token, tokens that some row sees) over all sequences."""
    pairs = tokens = 0
    if case["kind"] == "tree":
        for tree, held in zip(_parents(case), _sizes(case)[1]):
            depth = []
            for p in tree:
                depth.append(0 if p < 0 else depth[p] + 1)
            pairs += sum(depth) + len(tree) * (held + 1)
            tokens += held + len(tree)
        return pairs, tokens
    window, sinks = case["window"], case["sinks"]
    for n, held in zip(*_sizes(case)):
        pairs += sum(min(p + 1, window) + min(sinks, max(0, p + 1 - window)) for p in range(held, held + n))
        first = max(0, held + 1 - window)
        tokens += held + n - first + min(first, sinks)
    return pairs, tokens


def work(case):
    kind = case["kind"]
    if kind == "norm":
        values = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * values * case["dim"] * (2 if case["bf16"] else 4) + 12 * case["tokens"],
                "flops": values * (4 * case["dim"] + 3 * case["rotary"])}
    if kind == "keep":
        moved = sum(map(len, _kept(case, 0))) * case["layers"] * case["kv_heads"] * case["dim"]
        return {"bytes": 4 * moved, "flops": 4 * moved}
    pairs, tokens = _seen(case)
    return {"bytes": 2 * tokens * case["kv_heads"] * case["dim"] + -(-tokens // case["page"]) * (8 * case["kv_heads"] + 4)
            + 4 * sum(_sizes(case)[0]) * case["heads"] * case["dim"], "flops": 4 * case["dim"] * case["heads"] * pairs}


# -- inputs --------------------------------------------------------------------------------------------------------


def _pool(case, gen, layers, pages):
    """Random cache contents: bell-shaped values that fill most of a byte's range, scales of trained models' spread."""
    dtype, page = TYPES[case["type"]], case["page"]
    shape = (layers, pages, case["kv_heads"])

    def values(*tail):
        out = torch.empty(*shape, *tail, dtype=dtype, device=DEVICE)
        for layer in out:
            x = torch.randn(layer.shape, generator=gen, device=DEVICE)
            layer.copy_((x * 36).round().clamp(-127, 127) if dtype == torch.int8 else (x * 110).clamp(-448, 448))
        return out

    def scales():
        s = torch.exp(0.4 * torch.randn(shape, generator=gen, device=DEVICE)) * (4.0 / LARGEST[dtype])
        return s.to(torch.bfloat16).float()

    return values(page, case["dim"]), values(case["dim"], page), scales(), scales()


def _tables(counts, held, page, gen, spare=3):
    """Each sequence's pages, drawn from the whole cache in no order; -1 behind its last."""
    need = [-(-(c + h) // page) for c, h in zip(counts, held)]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    at = torch.arange(max(need), device=DEVICE)
    n = torch.tensor(need, device=DEVICE)
    first = torch.cumsum(n, 0) - n
    table = torch.where(at < n[:, None], order[(first[:, None] + at).clamp(max=pages - 1)], -1)
    return table.to(torch.int32).contiguous(), pages


def _whole(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    kind = case["kind"]
    state = {"case": case}
    if kind == "norm":
        T, half, dim = case["tokens"], case["rotary"] // 2, case["dim"]
        dtype = torch.bfloat16 if case["bf16"] else torch.float32
        # projections whose heads differ in size
        loud = torch.exp(0.7 * randn(case["heads"] + case["kv_heads"], 1))
        q = (randn(T, case["heads"], (2 if case["gated"] else 1) * dim) * loud[:case["heads"]]).to(dtype)
        state["q"], state["k"] = q[:, :, :dim], (randn(T, case["kv_heads"], dim) * loud[case["heads"]:]).to(dtype)
        state["q_weight"], state["k_weight"] = 0.4 * randn(dim), 0.4 * randn(dim)
        # text with runs of images in it, far into a long context: three axes that differ inside an image
        time = torch.arange(T, device=DEVICE) + 100_000
        grid = torch.randint(0, 64, (2, T), generator=gen, device=DEVICE) * (torch.arange(T, device=DEVICE) // 97 % 2)
        state["positions"] = torch.stack((time, time + grid[0], time + grid[1])).to(torch.int64)
        state["inv_freq"] = torch.pow(1e7, -torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
        state["sections"] = ((half + 2) // 3, (half + 1) // 3, half // 3)
        return state
    counts, held = _sizes(case)
    state["table"], pages = _tables(counts, held, case["page"], gen)
    state["start"] = _whole(held)
    rows = counts
    if kind == "keep":
        kept = _kept(case, seed)
        rows = list(map(len, kept))
        state["keep"] = _whole([i for k in kept for i in k])
    else:
        state["length"] = _whole([c + h for c, h in zip(counts, held)])
        state["max_length"] = max(c + h for c, h in zip(counts, held))
        # keys and queries whose scores spread over several units, as trained heads' do
        state["q"] = (1.6 * randn(sum(counts), case["heads"], case["dim"])).to(torch.bfloat16)
    state["cu"] = _whole([sum(rows[:i]) for i in range(len(rows) + 1)])
    state["max_count"] = max(rows)
    if kind == "tree":
        trees = _parents(case)
        rng = random.Random(seed)
        for tree in trees:  # another tree for another seed, of the same depths
            depth = [0] * len(tree)
            for i, p in enumerate(tree):
                depth[i] = 0 if p < 0 else depth[p] + 1
                if p >= 0:
                    tree[i] = rng.choice([j for j in range(i) if depth[j] == depth[p]])
        state["parents"] = _whole([p for tree in trees for p in tree])
    state["k"], state["v"], state["k_scale"], state["v_scale"] = _pool(case, gen, case.get("layers", 1), pages)
    if own:  # the handle that a program keeps
        state["pages"] = _hip().KVPages(state["k"], state["v"], state["k_scale"], state["v_scale"])
    return state


# -- the plain forms -----------------------------------------------------------------------------------------------


def _plain_norm(x, weight, s):
    rotary = s["case"]["rotary"]
    half = rotary // 2
    j = torch.arange(half, device=x.device)
    _, height, width = s["sections"]
    axis = torch.where((j % 3 == 1) & (j < 3 * height), 1, torch.where((j % 3 == 2) & (j < 3 * width), 2, 0))
    angle = s["positions"][axis].double().T * s["inv_freq"]  # [T, half]
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * (1 + weight)
    a, b, rest = y[..., :half], y[..., half:rotary], y[..., rotary:]
    return torch.cat((a * c - b * sn, b * c + a * sn, rest), 2).to(x.dtype)


def _plain_tree(s):
    """Every node's ancestors and itself: truth values [B, count, count], the masks as 64-bit words [tokens, words], and the
    positions [tokens]."""
    cu, parents = s["cu"].long(), s["parents"].long()
    n = cu[1:] - cu[:-1]
    top = s["max_count"]
    i = torch.arange(top, device=cu.device)
    there = i < n[:, None]
    own_parent = torch.where(there, parents[(cu[:-1, None] + i).clamp(max=len(parents) - 1)], -1)
    line = torch.eye(top, top + 1, device=cu.device).repeat(len(n), 1, 1)  # column `top`: past a root
    line.scatter_(2, torch.where(own_parent < 0, top, own_parent)[..., None], 1.0)
    line = line[..., :top]
    for _ in range((top - 1).bit_length()):  # ancestors 1, 3, 7, .. steps up
        line = torch.matmul(line, line).clamp(max=1.0)
    line = (line > 0) & there[..., None]
    words = -(-top // 64)
    bits = torch.zeros(len(n), top, words * 64, dtype=torch.int64, device=cu.device)
    bits[..., :top] = line
    masks = (bits.view(len(n), top, words, 64) << torch.arange(64, device=cu.device)).sum(3)
    positions = s["start"].long()[:, None] + line.sum(2) - 1
    return line, masks[there], positions[there]


def _plain_attend(s, seen_of):
    """seen_of(position [B, count, 1] of each row, token j, first new token [B, 1, 1]) -> which rows see which tokens."""
    k, v, table, length, cu = s["k"][0], s["v"][0], s["table"].long().clamp(min=0), s["length"].long(), s["cu"].long()
    q = s["q"]
    B, W = table.shape
    H, D, page = k.shape[1], k.shape[3], k.shape[2]
    G = q.shape[1] // H
    keys = (k[table].float() * s["k_scale"][0][table][..., None, None]).permute(0, 2, 1, 3, 4).reshape(B, H, W * page, D)
    values = (v[table].float() * s["v_scale"][0][table][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, H, W * page, D)
    n = cu[1:] - cu[:-1]
    i = torch.arange(s["max_count"], device=q.device)
    at = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    rows = q[at].float().reshape(B, len(i), H, G, D).permute(0, 2, 1, 3, 4).reshape(B, H, len(i) * G, D)
    scores = torch.matmul(rows, keys.transpose(2, 3)) * D ** -0.5
    first = (length - n)[:, None, None]
    j = torch.arange(W * page, device=q.device)
    seen = seen_of(first + i[:, None], j, first) & (j < length[:, None, None])
    seen = seen.repeat_interleave(G, 1)[:, None]
    scores.masked_fill_(~seen, float("-inf"))
    top = scores.amax(3, keepdim=True)
    p = scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(3, keepdim=True)
    o = torch.matmul(p, values) / torch.where(total == 0, 1.0, total)
    o = o.reshape(B, H, len(i), G, D).permute(0, 2, 1, 3, 4).reshape(B, len(i), H * G, D)
    return o[i < n[:, None]].to(torch.bfloat16)


def _plain_window(s):
    window, sinks = s["case"]["window"], s["case"]["sinks"]
    return _plain_attend(s, lambda at, j, first: (j <= at) & ((j > at - window) | (j < sinks)))


def _round_up_bf16(x):
    """The smallest bfloat16 value that is not below x (fp32, not negative), as fp32."""
    bits = x.view(torch.int32)
    return ((bits + 0xFFFF) & -65536).view(torch.float32)


def _plain_keep(s, pool, scale, token_dim):
    """One of K and V, all layers: the kept tokens' values gathered, the pages that they belong into requantized and put back."""
    table, cu, start, keep = s["table"].long(), s["cu"].long(), s["start"].long(), s["keep"].long()
    page, dtype = s["case"]["page"], pool.dtype
    top = LARGEST[dtype]
    n = cu[1:] - cu[:-1]
    if len(keep) == 0:
        return
    b = torch.repeat_interleave(torch.arange(len(n), device=keep.device), n)
    to = start[b] + torch.arange(len(keep), device=keep.device) - cu[b]
    at = start[b] + keep
    tokens = pool.transpose(3, 4) if token_dim == 4 else pool  # [L, pages, H, page, D]
    where = table[b, at // page]
    x = tokens[:, where, :, at % page].float() * scale[:, where].transpose(0, 1)[..., None]  # [rows, L, H, D]
    column = (start // page)[:, None] + torch.arange((s["max_count"] + page - 1) // page + 1, device=keep.device)
    holds = (column * page < (start + n)[:, None]) & (n > 0)[:, None]
    pb, pc = torch.nonzero(holds, as_tuple=True)
    ids = table[pb, column[pb, pc]]  # the pages that kept tokens belong into
    position = column[pb, pc][:, None] * page + torch.arange(page, device=keep.device)  # [P, page]
    fresh = (position >= start[pb][:, None]) & (position < (start + n)[pb][:, None])
    rows = x[(cu[pb][:, None] + position - start[pb][:, None]).clamp(0, len(keep) - 1)]  # [P, page, L, H, D]
    rows = torch.where(fresh[..., None, None, None], rows, 0.0).permute(2, 0, 3, 1, 4)  # [L, P, H, page, D]
    amax = rows.abs().amax((3, 4))
    old = scale[:, ids]
    alone = _round_up_bf16(amax / torch.full_like(amax, top))  # by a tensor: a quotient rounded once
    reach = old * top
    grow = torch.ceil(torch.log2(torch.where((amax > reach) & (reach > 0), amax / reach, 1.0)))
    grow = torch.where(torch.ldexp(reach, grow - 1) >= amax, grow - 1, grow).clamp(min=0)
    grow = torch.where(torch.ldexp(reach, grow) < amax, grow + 1, grow)
    now = torch.where(old > 0, torch.ldexp(old, grow), alone)
    grow = torch.where(old > 0, grow, 0.0)
    before = tokens[:, ids].float()
    shrunk = torch.ldexp(before, -grow[..., None, None])
    per = rows / torch.where(now > 0, now, 1.0)[..., None, None]
    if dtype == torch.int8:
        shrunk, per = shrunk.round(), per.round()
    older = position < start[pb][:, None]  # what lies behind the kept tokens stays as it is
    out = torch.where(fresh[:, None, :, None], per, torch.where(older[:, None, :, None], shrunk, before)).to(dtype)
    tokens[:, ids] = out
    scale[:, ids] = now


def run(state):
    kind, case = state["case"]["kind"], state["case"]
    if kind == "norm":
        if own:
            return _hip().norm_rope(state["q"], state["k"], state["positions"], state["inv_freq"], state["q_weight"],
                                    state["k_weight"], eps=1e-6, sections=state["sections"])
        return _plain_norm(state["q"], state["q_weight"], state), _plain_norm(state["k"], state["k_weight"], state)
    if kind == "window":
        if own:
            return _hip().kv_attend(state["pages"], 0, state["q"], state["table"], state["length"], state["cu"],
                                    max_count=state["max_count"], max_length=state["max_length"], window=case["window"],
                                    sinks=case["sinks"])
        return _plain_window(state)
    if kind == "tree":  # a step's first attention layer: the masks are made for the step, all its layers take them
        if own:
            masks, positions = _hip().kv_tree(state["parents"], state["start"], state["cu"], max_count=state["max_count"])
            out = _hip().kv_attend(state["pages"], 0, state["q"], state["table"], state["length"], state["cu"],
                                   max_count=state["max_count"], max_length=state["max_length"], tree=masks)
        else:
            line, masks, positions = _plain_tree(state)

            def seen(at, j, first):
                drafted = line.gather(2, (j - first).clamp(0, line.shape[2] - 1).expand(-1, line.shape[1], -1))
                return (j < first) | ((j < first + line.shape[2]) & drafted)
            out = _plain_attend(state, seen)
        return {"out": out, "masks": masks, "positions": positions}
    if own:
        _hip().kv_keep(state["pages"], state["table"], state["start"], state["keep"], state["cu"], max_count=state["max_count"])
    else:
        _plain_keep(state, state["k"], state["k_scale"], 3)
        _plain_keep(state, state["v"], state["v_scale"], 4)
    # the cache itself: whole numbers (or e4m3 values) and the scales that they are multiples of
    return {"k": state["k"], "v": state["v"], "k_scale": state["k_scale"], "v_scale": state["v_scale"]}


# -- in 64 bits ----------------------------------------------------------------------------------------------------


def _exact_norm(s):
    half = s["case"]["rotary"] // 2
    counts = list(s["sections"])
    axis = [0] * half
    for a in (1, 2):
        for j in range(a, 3 * counts[a], 3):
            axis[j] = a
    angle = torch.stack([s["positions"][a].double() * s["inv_freq"][j] for j, a in enumerate(axis)], 1)[:, None]
    out = []
    for x, w in ((s["q"].double(), s["q_weight"].double()), (s["k"].double(), s["k_weight"].double())):
        y = x / ((x * x).sum(2, keepdim=True) / x.shape[2] + 1e-6).sqrt() * (w + 1)
        z = torch.complex(y[..., :half], y[..., half:2 * half]) * torch.polar(torch.ones_like(angle), angle)
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_attend(s, hidden_of):
    """hidden_of(sequence, its rows, its length) -> truth values [rows, length]: what a row does not see."""
    case = s["case"]
    G, page = case["heads"] // case["kv_heads"], case["page"]
    out = []
    bounds = s["cu"].tolist()
    for b, length in enumerate(s["length"].tolist()):
        ids = s["table"][b, :-(-length // page)].long()
        k = (s["k"][0][ids].double() * s["k_scale"][0][ids].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :length]
        v = (s["v"][0][ids].double() * s["v_scale"][0][ids].double()[..., None, None]).transpose(2, 3).transpose(0, 1).flatten(1, 2)[:, :length]
        q = s["q"][bounds[b]:bounds[b + 1]].double()
        o = torch.empty_like(q)
        hidden = hidden_of(b, q.shape[0], length)
        for h in range(case["heads"]):
            a = (q[:, h] @ k[h // G].T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
            o[:, h] = torch.softmax(a, 1) @ v[h // G]
        out.append(o)
    return torch.cat(out)


def _exact_window(s):
    window, sinks = s["case"]["window"], s["case"]["sinks"]

    def hidden(b, n, length):
        at, j = torch.arange(length - n, length, device=DEVICE)[:, None], torch.arange(length, device=DEVICE)[None]
        return (j > at) | ((j <= at - window) & (j >= sinks))
    return _exact_attend(s, hidden)


def _exact_tree(s):
    bounds, parents, starts = s["cu"].tolist(), s["parents"].tolist(), s["start"].tolist()
    words = -(-s["max_count"] // 64)
    lines, masks, positions = [], [], []
    for b, start in enumerate(starts):
        tree = parents[bounds[b]:bounds[b + 1]]
        line = []
        for i, p in enumerate(tree):
            line.append((line[p] if p >= 0 else []) + [i])
            number = sum(1 << j for j in line[i])
            masks.append([(w - (1 << 64) if w >> 63 else w) for w in (number >> 64 * k & (1 << 64) - 1 for k in range(words))])
            positions.append(start + len(line[i]) - 1)
        lines.append(line)

    def hidden(b, n, length):
        out = torch.zeros(n, length, dtype=torch.bool)
        out[:, length - n:] = True
        for i, line in enumerate(lines[b]):
            out[i, [length - n + j for j in line]] = False
        return out.to(DEVICE)
    return {"out": _exact_attend(s, hidden), "masks": torch.tensor(masks, dtype=torch.int64, device=DEVICE),
            "positions": torch.tensor(positions, dtype=torch.int64, device=DEVICE)}


def _bf16_not_below(x):
    """The smallest value with 8 significant bits that is not below x (a float, positive)."""
    m, e = math.frexp(x)
    return math.ldexp(math.ceil(m * 256), e - 8)


def _nearest(x, dtype):
    """x (fp64, within the type's range) rounded to nearest even."""
    if dtype == torch.int8:
        return x.round()
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 4).clamp(min=-9))
    return (x / step).round() * step


def _exact_keep(s):
    case = s["case"]
    page, dtype = case["page"], TYPES[case["type"]]
    top = LARGEST[dtype]
    bounds, starts, table, keep = s["cu"].tolist(), s["start"].tolist(), s["table"].tolist(), s["keep"].tolist()
    if case["layers"] * sum(n // page + 2 for n in (b - a for a, b in zip(bounds, bounds[1:])) if n) > 3000:
        return None
    got = {}
    for name in ("k", "v"):
        pool, scale = s[name].double(), s[name + "_scale"].double()
        if name == "v":
            pool = pool.transpose(3, 4).contiguous()
        was, was_scale = pool.clone(), scale.clone()
        for b, start in enumerate(starts):
            mine = keep[bounds[b]:bounds[b + 1]]
            for c in range(start // page, -(-(start + len(mine)) // page) if mine else 0):
                lo, hi = max(start, c * page), min(start + len(mine), (c + 1) * page)
                p, held = table[b][c], lo - c * page
                at = [start + mine[t - start] for t in range(lo, hi)]
                source = [table[b][t // page] for t in at]
                part = torch.stack([was[:, q, :, t % page] * was_scale[:, q][..., None] for q, t in zip(source, at)], 2)  # [L, H, n, D]
                largest = part.abs().amax((2, 3)).tolist()
                for l in range(case["layers"]):
                    for h in range(case["kv_heads"]):
                        before, a = float(was_scale[l, p, h]), largest[l][h]
                        now = before
                        if before > 0:
                            while now * top < a:
                                now *= 2
                            pool[l, p, h, :held] = _nearest(pool[l, p, h, :held] * (before / now), dtype)
                        else:
                            now = _bf16_not_below(a / top) if a > 0 else 0.0
                        scale[l, p, h] = now
                        pool[l, p, h, held:held + hi - lo] = _nearest(part[l, h] / (now or 1.0), dtype)
        got[name + "_scale"] = scale
        if name == "v":
            pool = pool.transpose(3, 4)
        got[name] = pool.to(torch.int8) if dtype == torch.int8 else pool
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "window": _exact_window, "tree": _exact_tree, "keep": _exact_keep}[case["kind"]](s)
