"""The attention half's operators in plain torch on the CPU, in 64 bits: the paged 8-bit cache's append, attention over it,
rotary positions behind a norm, trees of drafts and their accepted tokens. Written from the definitions, one block, row or frequency at a time; used by the tests only."""
import math

import torch

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def bf16_not_below(x: float) -> float:
    """The smallest bfloat16 value that is not below x >= 0: 8 significant bits, at least 2^-133 apart."""
    if x == 0:
        return 0.0
    e = max(math.frexp(x)[1] - 8, -133)
    return math.ldexp(math.ceil(math.ldexp(x, -e)), e)


def nearest(x: torch.Tensor, dtype) -> torch.Tensor:
    """x (fp64) rounded to nearest even in int8 or e4m3, as fp64."""
    if dtype == torch.int8:
        return x.round()
    _, e = torch.frexp(x)
    step = torch.pow(2.0, (e - 4).clamp(min=-9).double())
    return (x / step).round() * step


def grown(old: float, reach: float, top: float) -> float:
    """old times the smallest power of two with which it reaches top."""
    now = old
    while now * reach < top:
        now *= 2
    return now


def append(pool, scale, new, table, start, cu, page_tokens, v=False, max_count=None):
    """One layer's K (or V) pool [pages, heads, page_tokens, dim] (V: [.., dim, page_tokens]) and scale [pages, heads] on
    the CPU -> (pool, scale) after the append, the pool's values as fp64."""
    top = LARGEST[pool.dtype]
    dtype = pool.dtype
    out, sc = pool.double(), scale.double().clone()
    out = out.transpose(2, 3).clone() if v else out.clone()
    pages = pool.shape[0]
    for b in range(len(start)):
        lo = min(max(int(cu[b]), 0), new.shape[0])
        n = min(max(int(cu[b + 1]), lo) - lo, new.shape[0] - lo, new.shape[0] if max_count is None else max_count)
        at = max(int(start[b]), 0)
        col = at // page_tokens
        while n and col * page_tokens < at + n:
            p = int(table[b, col]) if col < table.shape[1] else -1
            t0, t1 = max(at, col * page_tokens), min(at + n, (col + 1) * page_tokens)
            col += 1
            if not 0 <= p < pages:
                continue
            rows = new[lo + t0 - at:lo + t1 - at].double()
            i0, i1 = t0 % page_tokens, t0 % page_tokens + t1 - t0
            for h in range(pool.shape[1]):
                x = rows[:, h]
                a = float(x.abs().max())
                old = float(sc[p, h]) if i0 else 0.0
                if not math.isfinite(a):
                    now = math.nan
                elif math.isnan(old):
                    now = old
                elif old > 0:
                    now = grown(old, top, a)
                    out[p, h, :i0] = nearest(out[p, h, :i0] * (old / now), dtype)
                else:
                    now = bf16_not_below(a / top)
                    if i0 and now > 0:
                        out[p, h, :i0] = 0
                sc[p, h] = now
                out[p, h, i0:i1] = nearest(x / now, dtype) if now > 0 else 0.0
    return (out.transpose(2, 3) if v else out), sc


def attend(k, v, k_scale, v_scale, q, table, length, cu, scale=None, causal=True, max_count=None, weight_roundings=1, window=None, sinks=0,
           tree=None):
    """window, sinks, tree (int64 [tokens, words]): what a causal call's rows see. k, v, scales: one layer on the CPU. -> (out fp64 [tokens, heads, dim] with NaN in rows that belong to no sequence, the
    bound of |error| of a bf16 result whose scores and sums are fp32 and whose weights are rounded to bf16, so many times)."""
    pages, kv_heads, page, dim = k.shape
    group = q.shape[1] // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    tol = torch.zeros(q.shape, dtype=torch.float64)
    for b in range(len(length)):
        lo = min(max(int(cu[b]), 0), q.shape[0])
        n = min(max(int(cu[b + 1]), lo) - lo, q.shape[0] - lo, q.shape[0] if max_count is None else max_count)
        total = min(max(int(length[b]), 0), table.shape[1] * page)
        ids = [int(p) for p in table[b, :-(-total // page)]]
        there = torch.tensor([0 <= p < pages for p in ids for _ in range(page)], dtype=torch.bool)[:total]
        use = torch.tensor([p if 0 <= p < pages else 0 for p in ids], dtype=torch.long)
        for h in range(q.shape[1]):
            g = h // group
            K = (k[use, g].double() * k_scale[use, g].double()[:, None, None]).reshape(-1, dim)[:total]
            V = (v[use, g].double() * v_scale[use, g].double()[:, None, None]).transpose(1, 2).reshape(-1, dim)[:total]
            for i in range(n):
                begin = int(length[b]) - n
                seen = there.clone()
                if tree is not None:
                    own = drafted(tree[lo + i], n)
                    seen[max(begin, 0):] = False
                    for j in own:
                        if 0 <= begin + j < total:
                            seen[begin + j] = there[begin + j]
                    at = begin + max(len(own) - 1, 0)
                else:
                    at = begin + i
                    if causal:
                        seen[max(at + 1, 0):] = False
                if window is not None:
                    seen[min(sinks, total):max(at + 1 - window, min(sinks, total), 0)] = False
                keep = seen.nonzero()[:, 0]
                x = q[lo + i, h].double()
                if len(keep) == 0:
                    out[lo + i, h] = 0
                    continue
                Kk, Vk = K[keep], V[keep]
                s = Kk @ x * scale
                w = torch.softmax(s, 0)
                o = w @ Vk
                out[lo + i, h] = o
                # a score: dim products added in fp32, then two multiplications; its exponential: 2 steps of the argument
                slack = (dim + 4) * 2.0 ** -23 * float((Kk.abs() @ x.abs()).max()) * abs(scale) + 2.0 ** -21 * float(s.abs().max())
                # a weight is rounded to bf16 (2^-8), the sums are fp32; the result is rounded once more
                per = weight_roundings * 2.0 ** -8 + 2 * slack + (len(keep) + 8) * 2.0 ** -23
                tol[lo + i, h] = 2.0 ** -8 * o.abs() + per * (w @ Vk.abs())
    return out, tol


def drafted(words, n):
    """The rows below n whose bits are set in a row's words."""
    return [j for j in range(min(n, 64 * len(words))) if int(words[j // 64]) >> j % 64 & 1]


def tree(parents, start, cu, words, max_count=None):
    """-> (masks int64 [tokens, words], positions int64 [tokens]) of drafted trees, zeros in rows of no sequence."""
    masks, positions = torch.zeros(len(parents), words, dtype=torch.int64), torch.zeros(len(parents), dtype=torch.int64)
    for b in range(len(start)):
        lo = min(max(int(cu[b]), 0), len(parents))
        n = min(max(int(cu[b + 1]), lo) - lo, len(parents) - lo, len(parents) if max_count is None else max_count)
        for i in range(n):
            line = [i]
            while 0 <= int(parents[lo + line[-1]]) < line[-1]:
                line.append(int(parents[lo + line[-1]]))
            for w in range(words):
                bits = sum(1 << j % 64 for j in line if j // 64 == w)
                masks[lo + i, w] = bits - (1 << 64) if bits >> 63 else bits
            positions[lo + i] = int(start[b]) + len(line) - 1
    return masks, positions


def keep(pool, scale, table, start, keep, cu, page_tokens, v=False, max_count=None):
    """K (or V) of all layers [layers, pages, heads, page_tokens, dim] (V: [.., dim, page_tokens]) and scale [layers, pages, heads] on
    the CPU -> (pool as fp64, scale) with each sequence's kept tokens moved up, read before any is written."""
    dtype, top = pool.dtype, LARGEST[pool.dtype]
    old, sc = (pool.double().transpose(3, 4) if v else pool.double()).clone(), scale.double()
    out, now_sc, pages = old.clone(), sc.clone(), pool.shape[1]

    def page(b, pos):
        p = int(table[b, pos // page_tokens]) if pos // page_tokens < table.shape[1] else -1
        return p if 0 <= p < pages else None
    for b in range(len(start)):
        lo = min(max(int(cu[b]), 0), len(keep))
        n = min(max(int(cu[b + 1]), lo) - lo, len(keep) - lo, len(keep) if max_count is None else max_count)
        first = max(int(start[b]), 0)
        moves = {}  # target page -> [(place in it, source page, place in it)]
        for i in range(n):
            source, target = first + max(int(keep[lo + i]), i), first + i
            if page(b, target) is not None and page(b, source) is not None:
                moves.setdefault(target // page_tokens, []).append((target % page_tokens, page(b, source), source % page_tokens))
        for column, tokens in moves.items():
            p, held = page(b, column * page_tokens), max(first - column * page_tokens, 0)
            for layer in range(pool.shape[0]):
                for h in range(pool.shape[2]):
                    x = torch.stack([old[layer, s, h, t] * sc[layer, s, h] for _, s, t in tokens])
                    a, was = float(x.abs().max()), float(sc[layer, p, h])
                    if not math.isfinite(a) or a >= 2.0 ** 128:
                        now = math.nan
                    elif math.isnan(was):
                        now = was
                    elif was > 0:
                        now = grown(was, top, a)
                        out[layer, p, h, :held] = nearest(old[layer, p, h, :held] * (was / now), dtype)
                    else:
                        now = bf16_not_below(a / top)
                        if now > 0:
                            out[layer, p, h, :held] = 0
                    now_sc[layer, p, h] = now
                    for (t, _, _), y in zip(tokens, x):
                        out[layer, p, h, t] = nearest(y / now, dtype) if now > 0 else 0.0
    return (out.transpose(3, 4) if v else out), now_sc


def norm(x, weight, eps, zero_centered=True):
    """Each head's x / sqrt(mean(x^2) + eps) * w in fp64."""
    x = x.double()
    w = 1.0 if weight is None else weight.double() + (1.0 if zero_centered else 0.0)
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w


def rope(x, positions, inv_freq, sections, interleaved, scale=1.0):
    """x [tokens, heads, dim] on the CPU -> fp64; positions [axes, tokens]."""
    half = inv_freq.shape[0]
    axis = []
    for j in range(half):
        if interleaved:
            a = j % len(sections)
            axis.append(a if a and j < len(sections) * sections[a] else 0)
        else:
            axis.append(next(i for i in range(len(sections)) if j < sum(sections[:i + 1])))
    y = x.double().clone()
    for j, a in enumerate(axis):
        angle = positions[a].double() * inv_freq[j].double()
        c, s = torch.cos(angle)[:, None] * scale, torch.sin(angle)[:, None] * scale
        p, r = x[..., j].double(), x[..., half + j].double()
        y[..., j], y[..., half + j] = p * c - r * s, r * c + p * s
    return y
