"""The attention half of a decoder layer, timed: rotary positions with several axes, writing keys and values into a paged
8-bit cache, attention over that cache from one token to a prompt, and moving the cache's pages.

Kinds of case:
  attend  grouped-query attention of `count` new tokens a sequence over pages of int8 or e4m3 values, one scale for each
          page and kv head (causal; the new tokens are the last ones in the cache)
  append  new keys and values quantized into the cache, behind what their sequences hold
  rope    q and k rotated by positions on three axes (time, height, width), interleaved over the frequencies
  copy    pages copied inside the cache, all layers at once: what forking and compacting do

The cache: k [layers, pages, kv_heads, page_tokens, head_dim], v [layers, pages, kv_heads, head_dim, page_tokens] (int8 or
float8_e4m3fn), k_scale and v_scale fp32 [layers, pages, kv_heads]; a value is byte * scale. A page's scale is the smallest
bfloat16 s with M * s >= max |x| over the page's tokens (M = 127 or 448), a value's byte x / s rounded to nearest even.
When tokens join a page that holds some, its scale grows by the smallest power of two that covers the new ones, and
the older bytes are divided by it and rounded to nearest even."""
import math
import os
import random
import sys

import numpy as np
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


def _attend(seqs, count, history, dtype="int8", heads=16, kv_heads=2, dim=256, page=64, ragged=False):
    return {"kind": "attend", "seqs": seqs, "count": count, "history": history, "ragged": ragged, "type": dtype, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def _append(seqs, count, history, dtype="int8", kv_heads=2, dim=256, page=64, ragged=False):
    return {"kind": "append", "seqs": seqs, "count": count, "history": history, "ragged": ragged, "type": dtype,
            "kv_heads": kv_heads, "dim": dim, "page": page}


def _rope(tokens, heads=16, kv_heads=2, dim=256, rotary=64, gated=True, bf16=True):
    return {"kind": "rope", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "gated": gated, "bf16": bf16}


def _copy(copies, pages, layers, dtype="int8", kv_heads=2, dim=256, page=64):
    return {"kind": "copy", "copies": copies, "pages": pages, "layers": layers, "type": dtype, "kv_heads": kv_heads,
            "dim": dim, "page": page}


def listed():
    return [
        # interactive decoding: one sequence, one token, a conversation of some hundred tokens
        dict(_attend(1, 1, 776), name="attend_1"),
        # a drafted continuation of four tokens checked at once, a few users, smaller pages and heads
        dict(_attend(7, 4, 2001, "e4m3", heads=32, kv_heads=8, dim=128, page=32, ragged=True), name="attend_verify"),
        # batched serving: 64 conversations of very different lengths
        dict(_attend(64, 1, 16000, ragged=True), name="attend_64"),
        # one user far into a long document
        dict(_attend(1, 1, 131070, "e4m3"), name="attend_long"),
        # short ragged prompts, some behind an earlier turn, in one call
        dict(_attend(5, 301, 1500, "e4m3", heads=32, kv_heads=8, dim=128, page=32, ragged=True), name="prefill_ragged"),
        # a prefill chunk from nothing, the benchmark's size
        dict(_attend(1, 4096, 0), name="prefill_4096"),
        # one decode step's new keys and values of 64 sequences
        dict(_append(64, 1, 16000, ragged=True), name="append_64"),
        # a prefill chunk's keys and values behind a first turn that ends inside a page
        dict(_append(1, 4096, 1001), name="append_4096"),
        # one decode step of 64 sequences; q beside its gate in the projection's rows
        dict(_rope(64), name="rope_64"),
        # a prefill chunk with images in it
        dict(_rope(4096), name="rope_4096"),
        # 16 forked sequences take copies of the last pages they share, in the ten attention layers
        dict(_copy(16, 256, 10), name="copy_tails"),
        # compaction: the live pages of a fragmented cache move into its holes
        dict(_copy(900, 2048, 4), name="copy_compact"),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 4e12, w["flops"] / 5e14)


def draw(rng: random.Random):
    kind = rng.choice(("attend", "attend", "attend", "append", "rope", "copy"))
    most = max(_cost(c) for c in listed() if c["kind"] == kind)
    while True:
        heads, kv_heads, dim = rng.choice(((16, 2, 256), (16, 2, 256), (32, 8, 128), (8, 8, 64), (24, 8, 128), (6, 1, 64)))
        page, dtype = rng.choice((16, 32, 64, 64, 128)), rng.choice(("int8", "e4m3"))
        ragged = rng.random() < 0.6
        if kind == "attend":
            count = rng.choice((1, 1, rng.randint(2, 9), _spread(rng, 10, 4096)))
            case = _attend(_spread(rng, 1, 64), count, rng.choice((0, _spread(rng, 1, 131072))), dtype, heads, kv_heads, dim, page, ragged)
            # the plain form pads every sequence to the longest, and keeps all scores
            if case["seqs"] * (case["history"] + count) * kv_heads * dim > 64 * 16384 * 512:
                continue
            if case["seqs"] * (case["history"] + count) * count * heads > 4200 * 4200 * 16:
                continue
        elif kind == "append":
            count = rng.choice((1, rng.randint(2, 9), _spread(rng, 10, 4096)))
            case = _append(_spread(rng, 1, 64), count, rng.choice((0, _spread(rng, 1, 16384))), dtype, kv_heads, dim, page, ragged)
            if case["seqs"] * (case["history"] + count) * kv_heads * dim > 64 * 16384 * 512:
                continue
        elif kind == "rope":
            case = _rope(_spread(rng, 1, 4096), heads, kv_heads, dim, rng.choice((dim, dim // 2, dim // 4)), rng.random() < 0.5,
                         rng.random() < 0.7)
        else:
            copies = _spread(rng, 1, 900)
            case = _copy(copies, 2 * copies + rng.randint(1, 300), _spread(rng, 1, 10), dtype, kv_heads, dim, page)
            if case["pages"] * case["layers"] * page * kv_heads * dim * 2 > 1 << 30:
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


def _pairs(count, held):
    """How many (query, key) pairs the causal mask leaves of `count` tokens behind `held`."""
    return count * held + count * (count + 1) // 2


def work(case):
    kind = case["kind"]
    if kind in ("attend", "append"):
        counts, held = _sizes(case)
        new = sum(counts) * case["kv_heads"] * case["dim"]
    if kind == "attend":
        tokens = sum(counts) + sum(held)
        pages = sum(-(-(c + h) // case["page"]) for c, h in zip(counts, held))
        return {"bytes": 2 * tokens * case["kv_heads"] * case["dim"] + pages * (8 * case["kv_heads"] + 4)
                + 4 * sum(counts) * case["heads"] * case["dim"],
                "flops": 4 * case["dim"] * case["heads"] * sum(map(_pairs, counts, held))}
    if kind == "append":
        return {"bytes": 6 * new, "flops": 4 * new}
    if kind == "rope":
        values = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * values * case["dim"] * (2 if case["bf16"] else 4) + 12 * case["tokens"], "flops": 3 * values * case["rotary"]}
    page = 2 * case["kv_heads"] * (case["page"] * case["dim"] + 4)
    return {"bytes": 2 * case["copies"] * case["layers"] * page, "flops": 0}


# -- inputs --------------------------------------------------------------------------------------------------------


def _pool(case, gen, layers, pages):
    """Random cache contents: bell-shaped values that fill most of a byte's range, scales of trained models' spread."""
    dtype, page = TYPES[case["type"]], case["page"]
    shape = (layers, pages, case["kv_heads"])

    def values(*tail):
        if dtype == torch.int8:
            out = torch.empty(*shape, *tail, dtype=dtype, device=DEVICE)
            for layer in out:
                layer.copy_((torch.randn(layer.shape, generator=gen, device=DEVICE) * 36).round().clamp(-127, 127))
            return out
        out = torch.empty(*shape, *tail, dtype=dtype, device=DEVICE)
        for layer in out:
            layer.copy_((torch.randn(layer.shape, generator=gen, device=DEVICE) * 110).clamp(-448, 448))
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


def prepare(case, seed):
    gen = torch.Generator(DEVICE).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    kind = case["kind"]
    state = {"case": case}
    if kind in ("attend", "append"):
        counts, held = _sizes(case)
        state["table"], pages = _tables(counts, held, case["page"], gen)
        layers = 1
        total = sum(counts)
        state["cu"] = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=DEVICE)
        state["start"] = torch.tensor(held, dtype=torch.int32, device=DEVICE)
        state["length"] = torch.tensor([c + h for c, h in zip(counts, held)], dtype=torch.int32, device=DEVICE)
        state["max_count"], state["max_length"] = max(counts), max(c + h for c, h in zip(counts, held))
    elif kind == "copy":
        layers, pages = case["layers"], case["pages"]
        order = np.random.default_rng(seed).permutation(pages).astype(np.int32)
        state["src"], state["dst"] = order[:case["copies"]].copy(), order[case["copies"]:2 * case["copies"]].copy()
    if kind != "rope":
        state["k"], state["v"], state["k_scale"], state["v_scale"] = _pool(case, gen, layers, pages)
        if own:  # the handle that a program keeps
            state["pages"] = _hip().KVPages(state["k"], state["v"], state["k_scale"], state["v_scale"])
    if kind == "attend":
        # keys and queries whose scores spread over several units, as trained heads' do
        state["q"] = (1.6 * randn(total, case["heads"], case["dim"])).to(torch.bfloat16)
    elif kind == "append":
        # keys with a few strong channels, values without; the projections' outputs side by side in one row
        loud = 1 + 7 * (torch.rand(case["dim"], generator=gen, device=DEVICE) < 0.03).float()
        kv = randn(total, 2, case["kv_heads"], case["dim"])
        kv[:, 0] *= loud
        kv = kv.to(torch.bfloat16)
        state["new_k"], state["new_v"] = kv[:, 0], kv[:, 1]
    elif kind == "rope":
        T, half = case["tokens"], case["rotary"] // 2
        dtype = torch.bfloat16 if case["bf16"] else torch.float32
        q = randn(T, case["heads"], (2 if case["gated"] else 1) * case["dim"]).to(dtype)
        state["q"], state["rotated_k"] = q[:, :, :case["dim"]], randn(T, case["kv_heads"], case["dim"]).to(dtype)
        # text with runs of images in it, far into a long context: three axes that differ inside an image
        time = torch.arange(T, device=DEVICE) + 100_000
        grid = torch.randint(0, 64, (2, T), generator=gen, device=DEVICE) * (torch.arange(T, device=DEVICE) // 97 % 2)
        state["positions"] = torch.stack((time, time + grid[0], time + grid[1])).to(torch.int64)
        state["inv_freq"] = torch.pow(1e7, -torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
        state["sections"] = ((half + 2) // 3, (half + 1) // 3, half // 3)
    return state


# -- the plain forms -----------------------------------------------------------------------------------------------


def _plain_attend(s):
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
    position = (length - n)[:, None] + i  # [B, count]
    j = torch.arange(W * page, device=q.device)
    seen = (j <= position[..., None]) & (j < length[:, None, None])
    seen = seen.repeat_interleave(G, 1)[:, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(3, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(3, keepdim=True)
    o = torch.matmul(p, values) / torch.where(total == 0, 1.0, total)
    o = o.reshape(B, H, len(i), G, D).permute(0, 2, 1, 3, 4).reshape(B, len(i), H * G, D)
    return o[i < n[:, None]].to(torch.bfloat16)


def _round_up_bf16(x):
    """The smallest bfloat16 value that is not below x (fp32, not negative), as fp32."""
    bits = x.view(torch.int32)
    return ((bits + 0xFFFF) & -65536).view(torch.float32)


def _plain_append(s, new, pool, scale, token_dim):
    """One of K and V: the touched pages gathered, requantized and put back."""
    table, cu, start = s["table"].long(), s["cu"].long(), s["start"].long()
    page, dtype = s["case"]["page"], pool.dtype
    top = LARGEST[dtype]
    n = cu[1:] - cu[:-1]
    first = start // page
    touched = (s["max_count"] + page - 1) // page + 1
    column = first[:, None] + torch.arange(touched, device=new.device)
    position = column[..., None] * page + torch.arange(page, device=new.device)  # [B, touched, page]
    fresh = (position >= start[:, None, None]) & (position < (start + n)[:, None, None])
    b, c = torch.nonzero(fresh.any(2), as_tuple=True)
    fresh, position = fresh[b, c], position[b, c]
    ids = table[b, column[b, c]]
    x = new.float()[(cu[b][:, None] + position - start[b][:, None]).clamp(0, new.shape[0] - 1)]  # [P, page, H, D]
    x = torch.where(fresh[..., None, None], x, 0.0).permute(0, 2, 1, 3)  # [P, H, page, D]
    amax = x.abs().amax((2, 3))
    old = scale[ids]
    kept = (position[:, 0] < start[b])[:, None]  # the page holds older tokens
    alone = _round_up_bf16(amax / torch.full_like(amax, top))  # by a tensor: a quotient rounded once
    reach = old * top
    grow = torch.ceil(torch.log2(torch.where((amax > reach) & (reach > 0), amax / reach, 1.0)))
    grow = torch.where(torch.ldexp(reach, grow - 1) >= amax, grow - 1, grow).clamp(min=0)
    grow = torch.where(torch.ldexp(reach, grow) < amax, grow + 1, grow)
    now = torch.where(kept & (old > 0), torch.ldexp(old, grow), alone)
    grow = torch.where(kept & (old > 0), grow, 0.0)
    before = pool[ids].float()
    if token_dim == 3:
        before = before.transpose(2, 3)
    shrunk = torch.ldexp(before, -grow[..., None, None])
    per = x / torch.where(now > 0, now, 1.0)[..., None, None]
    if dtype == torch.int8:
        shrunk, per = shrunk.round(), per.round()
    older = position < start[b][:, None]  # what lies behind the new tokens stays as it is
    out = torch.where(fresh[:, None, :, None], per, torch.where(older[:, None, :, None], shrunk, before)).to(dtype)
    if token_dim == 3:
        out = out.transpose(2, 3)
    pool[ids] = out
    scale[ids] = now


def _plain_rope(x, s):
    rotary = s["case"]["rotary"]
    half = rotary // 2
    j = torch.arange(half, device=x.device)
    _, height, width = s["sections"]
    axis = torch.where((j % 3 == 1) & (j < 3 * height), 1, torch.where((j % 3 == 2) & (j < 3 * width), 2, 0))
    angle = s["positions"][axis].double().T * s["inv_freq"]  # [T, half]
    c, sn = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b, rest = x[..., :half].float(), x[..., half:rotary].float(), x[..., rotary:].float()
    return torch.cat((a * c - b * sn, b * c + a * sn, rest), 2).to(x.dtype)


def _plain_copy(s):
    src, dst = (torch.from_numpy(s[n]).to(DEVICE).long() for n in ("src", "dst"))
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    s["k_scale"][:, dst] = s["k_scale"][:, src]
    s["v_scale"][:, dst] = s["v_scale"][:, src]


def run(state):
    kind = state["case"]["kind"]
    if kind == "attend":
        if own:
            return _hip().kv_attend(state["pages"], 0, state["q"], state["table"], state["length"], state["cu"],
                                    max_count=state["max_count"], max_length=state["max_length"])
        return _plain_attend(state)
    if kind == "rope":
        if own:
            return _hip().rope(state["q"], state["rotated_k"], state["positions"], state["inv_freq"], sections=state["sections"])
        return _plain_rope(state["q"], state), _plain_rope(state["rotated_k"], state)
    if kind == "append":
        if own:
            _hip().kv_append(state["pages"], 0, state["new_k"], state["new_v"], state["table"], state["start"], state["cu"],
                             max_count=state["max_count"])
        else:
            _plain_append(state, state["new_k"], state["k"][0], state["k_scale"][0], 2)
            _plain_append(state, state["new_v"], state["v"][0], state["v_scale"][0], 3)
    elif own:
        _hip().kv_copy(state["pages"], state["src"], state["dst"])
    else:
        _plain_copy(state)
    # the cache itself: whole numbers (or e4m3 values) and the scales that they are multiples of
    return {"k": state["k"], "v": state["v"], "k_scale": state["k_scale"], "v_scale": state["v_scale"]}


# -- in 64 bits ----------------------------------------------------------------------------------------------------


def _exact_attend(s):
    case = s["case"]
    G, D, page = case["heads"] // case["kv_heads"], case["dim"], case["page"]
    out = []
    bounds = s["cu"].tolist()
    for b, length in enumerate(s["length"].tolist()):
        ids = s["table"][b, :-(-length // page)].long()
        k = (s["k"][0][ids].double() * s["k_scale"][0][ids].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :length]
        v = (s["v"][0][ids].double() * s["v_scale"][0][ids].double()[..., None, None]).transpose(2, 3).transpose(0, 1).flatten(1, 2)[:, :length]
        q = s["q"][bounds[b]:bounds[b + 1]].double()
        n = q.shape[0]
        o = torch.empty_like(q)
        last = torch.arange(length - n, length, device=q.device)
        hidden = torch.arange(length, device=q.device)[None] > last[:, None]
        for h in range(case["heads"]):
            a = (q[:, h] @ k[h // G].T / math.sqrt(D)).masked_fill(hidden, -math.inf)
            o[:, h] = torch.softmax(a, 1) @ v[h // G]
        out.append(o)
    return torch.cat(out)


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


def _exact_append(s):
    case = s["case"]
    page, dtype = case["page"], TYPES[case["type"]]
    top = LARGEST[dtype]
    bounds, starts, table = s["cu"].tolist(), s["start"].tolist(), s["table"].tolist()
    if len(starts) * (s["max_count"] // page + 2) > 1500:
        return None
    got = {}
    for name, new in (("k", s["new_k"]), ("v", s["new_v"])):
        pool, scale = s[name][0].double(), s[name + "_scale"][0].double()
        if name == "v":
            pool = pool.transpose(2, 3).contiguous()
        for b, start in enumerate(starts):
            x = new[bounds[b]:bounds[b + 1]].double()
            end = start + x.shape[0]
            for c in range(start // page, -(-end // page)):
                lo, hi = max(start, c * page), min(end, (c + 1) * page)
                part = x[lo - start:hi - start].transpose(0, 1)
                p = table[b][c]
                held = lo - c * page
                largest = part.abs().amax((1, 2)).tolist()
                for h, a in enumerate(largest):
                    before = float(scale[p, h]) if held else 0.0
                    if before > 0:
                        now = before
                        while now * top < a:
                            now *= 2
                        pool[p, h, :held] = _nearest(pool[p, h, :held] * (before / now), dtype)
                    else:
                        now = _bf16_not_below(a / top) if a > 0 else 0.0
                    scale[p, h] = now
                    pool[p, h, held:held + hi - lo] = _nearest(part[h] / (now or 1.0), dtype)
        got[name + "_scale"] = scale[None].to(torch.float64)
        if name == "v":
            pool = pool.transpose(2, 3)
        got[name] = pool[None].to(torch.int8) if dtype == torch.int8 else pool[None]
    return got


def _exact_rope(s):
    half = s["case"]["rotary"] // 2
    counts = list(s["sections"])
    axis = [0] * half
    for a in (1, 2):
        for j in range(a, 3 * counts[a], 3):
            axis[j] = a
    angle = torch.stack([s["positions"][a].double() * s["inv_freq"][j] for j, a in enumerate(axis)], 1)[:, None]
    out = []
    for x in (s["q"].double(), s["rotated_k"].double()):
        y = x.clone()
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.polar(torch.ones_like(angle), angle)
        y[..., :half], y[..., half:2 * half] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_copy(s):
    got = {}
    for name in ("k", "v", "k_scale", "v_scale"):
        pool = s[name] if s[name].dtype == torch.int8 else s[name].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pool[:, b].copy_(pool[:, a])
        got[name] = pool
    return got


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "attend":
        return _exact_attend(s)
    if kind == "append":
        return _exact_append(s)
    return _exact_rope(s) if kind == "rope" else _exact_copy(s)
