"""The attention half's operators in plain torch on the CPU, in 64 bits: the paged 8-bit cache's append, attention over it,
rotary positions. Written from the definitions, one block, row or frequency at a time; used by the tests only."""
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


def attend(k, v, k_scale, v_scale, q, table, length, cu, scale=None, causal=True, max_count=None, weight_roundings=1):
    """k, v, scales: one layer on the CPU. -> (out fp64 [tokens, heads, dim] with NaN in rows that belong to no sequence, the
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
                seen = min(total, max(int(length[b]) - n + i + 1, 0)) if causal else total
                keep = there[:seen].nonzero()[:, 0]
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
