"""The attention half's operators: rotary positions, the paged 8-bit key/value cache and attention over it, trees of drafted
tokens in it.

The reference keeps keys and values in a bf16 tensor per layer that grows in blocks of 256 positions and runs torch's
attention on it (engines/base.py:213-216,328-367). Here the cache is pages of bytes with one scale for each page and kv
head, shared by any number of sequences through page tables (gguf.hbm_cache keeps those), half the bytes of bf16 to read for
every decoded token. All calls only enqueue work on the current stream of their tensors' device and read page tables,
lengths and row offsets on the GPU, so they may be captured into a HIP graph.
"""
import ctypes
import functools

import numpy as np
import torch

from . import DTYPE_BF16, DTYPE_F32, KV_E4M3, KV_INT8, WlKvBatch, WlKvCache, WlKvMask, WlRopeTensor, check, library

TYPES = {torch.int8: KV_INT8, torch.float8_e4m3fn: KV_E4M3}


def _launch(index, call, *args):
    """call(*args, stream) with device `index` current (a launch goes to the current device) and its current stream."""
    if index < 0:
        raise ValueError("the tensors must be on the GPU (got tensors on the CPU)")
    if index == torch._C._cuda_getDevice():
        rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc)


def _refuse(t, name, device, dtype, shape):
    got = f"{t.dtype} {list(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
    raise ValueError(f"{name} must be a {dtype} tensor {shape} on {device} (got {got})")


# The checks below run before every launch, so each is one expression of cheap attributes; what is wrong is worked out
# after one has failed.


def _need(t, name, index, dtype, shape):
    """shape: what to say, one name or number a dimension."""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == index and t.dim() == len(shape)):
        _refuse(t, name, f"cuda:{index}", dtype, f"[{', '.join(map(str, shape))}]")


def _rows(t, name, index, dtype, heads, head_dim):
    """A [tokens, heads, head_dim] tensor whose head_dim is contiguous -> (tokens, heads, token stride, head stride)."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == index and t.dim() == 3:
        n, h, d = t.shape
        ts, hs, ds = t.stride()
        if d == head_dim and (ds == 1 or d == 1) and (heads is None or h == heads):
            return n, h, ts, hs
    _refuse(t, name, f"cuda:{index}", dtype, f"[tokens, {'heads' if heads is None else heads}, {head_dim}] with a contiguous last dimension")


def _in_cache(pages, layer):
    if not 0 <= layer < pages.layers:
        raise ValueError(f"layer {layer}: the cache has {pages.layers}")


class KVPages:
    """A paged key/value cache on one GPU, all layers: k int8 or float8_e4m3fn [layers, pages, kv_heads, page_tokens,
    head_dim], v of the same type [layers, pages, kv_heads, head_dim, page_tokens] (tokens innermost: the order in which the
    matrix core takes them), k_scale and v_scale fp32 [layers, pages, kv_heads], all contiguous. A value is its byte times its
    block's scale. head_dim 64, 128 or 256; page_tokens a power of two, 16 to 1024."""

    def __init__(self, k, v, k_scale, v_scale):
        if not isinstance(k, torch.Tensor) or k.dim() != 5 or k.dtype not in TYPES:
            raise ValueError("k must be an int8 or float8_e4m3fn tensor [layers, pages, kv_heads, page_tokens, head_dim]")
        layers, pages, heads, tokens, dim = k.shape
        _need(v, "v", k.get_device(), k.dtype, ("layers", "pages", "kv_heads", "head_dim", "page_tokens"))
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            _need(t, name, k.get_device(), torch.float32, ("layers", "pages", "kv_heads"))
            if tuple(t.shape) != (layers, pages, heads):
                raise ValueError(f"{name} must be [layers, pages, kv_heads] = {[layers, pages, heads]} (got {list(t.shape)})")
        if tuple(v.shape) != (layers, pages, heads, dim, tokens):
            raise ValueError(f"v must be [layers, pages, kv_heads, head_dim, page_tokens] = {[layers, pages, heads, dim, tokens]} "
                             f"(got {list(v.shape)})")
        if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            raise ValueError("the cache's tensors must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers, self.pages, self.kv_heads, self.page_tokens, self.head_dim = layers, pages, heads, tokens, dim
        self.dtype, self.device, self.index = k.dtype, k.device, k.get_device()
        s = WlKvCache()
        s.k, s.v, s.k_scale, s.v_scale = k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()
        s.pages, s.layers, s.kv_heads, s.page_tokens, s.head_dim = pages, layers, heads, tokens, dim
        s.type = TYPES[k.dtype]
        self.struct, self.ref = s, ctypes.byref(s)
        check(library().wl_kv_check(ctypes.byref(s)))

    @classmethod
    def empty(cls, layers: int, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64, dtype=torch.int8,
              device="cuda"):
        """A cache of zeros."""
        if dtype not in TYPES:
            raise ValueError("dtype must be torch.int8 or torch.float8_e4m3fn")

        def zeros(*tail):
            return torch.zeros(layers, pages, kv_heads, *tail, dtype=torch.int8, device=device).view(dtype)
        return cls(zeros(page_tokens, head_dim), zeros(head_dim, page_tokens),
                   *(torch.zeros(layers, pages, kv_heads, device=device) for _ in range(2)))

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.k_scale, self.v_scale))


def _batch(pages, table, cu, per_seq, name, tokens, max_count):
    """The WlKvBatch of one call; per_seq: start or length."""
    index = pages.index
    if not (isinstance(table, torch.Tensor) and table.dtype is torch.int32 and table.get_device() == index and table.dim() == 2):
        _refuse(table, "table", pages.device, torch.int32, "[sequences, pages]")
    seqs, width = table.shape
    row, step = table.stride()
    for t, what, n in ((cu, "cu", seqs + 1), (per_seq, name, seqs)):
        if not (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.get_device() == index and t.dim() == 1
                and t.shape[0] == n and t.is_contiguous()):
            _refuse(t, what, pages.device, torch.int32, f"[{n}] (table has {seqs} sequences), contiguous")
    if (step != 1 and width > 1) or (seqs > 1 and row < width):
        raise ValueError("the rows of table must be contiguous, and lie apart (not expanded)")
    if max_count is None or max_count > tokens:
        max_count = tokens
    if (seqs | width | tokens | max_count) >> 31:  # below 0, or more than the library's 32 bits: it would see another number
        raise ValueError(f"max_count {max_count} with {seqs} sequences of {width} pages and {tokens} rows")
    return WlKvBatch(table.data_ptr(), cu.data_ptr(), max(row, width), tokens, seqs, width,
                     max_count, 0)


def kv_append(pages: KVPages, layer: int, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
              cu: torch.Tensor, max_count: int = None):
    """Quantizes new keys and values of one layer into the cache: k, v bf16 [tokens, kv_heads, head_dim] (any strides over
    tokens and heads), sequence b's rows cu[b] .. cu[b + 1] to its positions start[b], start[b] + 1, ... of the pages in
    table[b] (int32 [seqs, width]; cu int32 [seqs + 1], start int32 [seqs]). max_count: the most rows any sequence has (rows
    beyond it are dropped; default: all rows). A page that begins among the rows gets the smallest bf16 scale that covers its
    rows, a page with older tokens its scale times the smallest power of two that does (its older bytes are divided by it and
    rounded); a NaN or an infinity makes its block's scale NaN. Rows whose page is not there (no table entry, or one outside
    the cache) are dropped. Pages written in one call must be distinct over its sequences."""
    _in_cache(pages, layer)
    n, _, k_token, k_head = _rows(k, "k", pages.index, torch.bfloat16, pages.kv_heads, pages.head_dim)
    rows, _, v_token, v_head = _rows(v, "v", pages.index, torch.bfloat16, pages.kv_heads, pages.head_dim)
    if n != rows:
        raise ValueError(f"k has {n} rows, v {rows}")
    b = _batch(pages, table, cu, start, "start", n, max_count)
    if n == 0 or b.seqs == 0:
        return
    _launch(pages.index, library().wl_kv_append, pages.ref, layer, k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head,
            b, start.data_ptr())


def _mask(n, index, b, causal, window, sinks, tree):
    """The WlKvMask of one call, or None."""
    if window is None and tree is None:
        if sinks:
            raise ValueError("sinks are what stays visible in front of a window")
        return None
    if not causal:
        raise ValueError("a window or a tree goes with causal=True")
    if window is not None and (window < 1 or sinks < 0):
        raise ValueError(f"window {window} with {sinks} sinks")
    if window is None and sinks:
        raise ValueError("sinks are what stays visible in front of a window")
    m = WlKvMask(None, 0, 0 if window is None else min(window, 1 << 31), min(sinks, 1 << 31))
    if tree is not None:
        _need(tree, "tree", index, torch.int64, (n, "words"))
        rows, words = tree.shape
        if rows != n or words * 64 < b.max_count or (words > 1 and tree.stride(1) != 1) or (n > 1 and tree.stride(0) < words):
            raise ValueError(f"tree must be [{n}, {-(-b.max_count // 64)} words or more] (max_count {b.max_count}) with contiguous rows "
                             f"that lie apart (got {list(tree.shape)}, strides {list(tree.stride())})")
        if window is not None and window < b.max_count:
            raise ValueError(f"a window of {window} would begin inside a tree of up to {b.max_count} tokens (max_count; without it all rows "
                             "of the call)")
        m.tree, m.tree_stride = tree.data_ptr(), max(tree.stride(0), words)
    return m


def kv_attend(pages: KVPages, layer: int, q: torch.Tensor, table: torch.Tensor, length: torch.Tensor, cu: torch.Tensor,
              max_count: int = None, max_length: int = None, scale: float = None, causal: bool = True,
              out: torch.Tensor = None, workspace: torch.Tensor = None, window: int = None, sinks: int = 0,
              tree: torch.Tensor = None) -> torch.Tensor:
    """Grouped-query attention of one layer: q bf16 [tokens, q_heads, head_dim] (any strides over tokens and heads) -> bf16
    [tokens, q_heads, head_dim]. Sequence b's rows are cu[b] .. cu[b + 1], the last of its length[b] tokens in the cache (so
    append them first); query head i reads kv head i / (q_heads / kv_heads). causal: a row sees the positions up to its own;
    otherwise all length[b]. A row that sees none is 0. scale (finite, not negative) defaults to head_dim ** -0.5. max_count: the
    most rows any sequence has (rows beyond it count as if they were not there; default: all rows, which costs calls of short
    sequences the form that is made for them); cu must not decrease; max_length: a bound of length that only steers how the
    work is split (default: what the table's width holds). Rows of no sequence stay as they are in `out` (which may not overlap
    q), and hold anything without it.
    workspace: a uint8 tensor that is large enough (wl_kv_attend_workspace_bytes; wl_kv_attend_masked_workspace_bytes with a
    window or a tree), for calls that do not overlap in time; by default it comes from torch's allocator, for this call and stream.
    window: a row sees the last `window` tokens up to its own alone, and the sequence's first `sinks`; only their pages are read.
    tree: int64 [tokens, words], words >= max_count / 64: the rows are drafted tokens, and of its sequence's own rows a row sees
    those whose bits are set (bit j % 64 of word j // 64 for row j; kv_tree makes them), all tokens before the rows as without it.
    With both, a row's position is its first row's plus the drafted tokens that it sees less one; the window has to hold a whole tree,
    max_count tokens: name that where a call has several sequences, since without it any of them may have all rows."""
    _in_cache(pages, layer)
    n, heads, token_stride, head_stride = _rows(q, "q", pages.index, torch.bfloat16, None, pages.head_dim)
    if heads == 0 or heads % pages.kv_heads:
        raise ValueError(f"{heads} query heads over {pages.kv_heads} kv heads")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif not (isinstance(out, torch.Tensor) and out.dtype is torch.bfloat16 and out.get_device() == pages.index
              and out.shape == q.shape and out.is_contiguous() and out.data_ptr() != q.data_ptr()):
        _refuse(out, "out", pages.device, torch.bfloat16, f"{list(q.shape)}, contiguous and not q's memory,")
    b = _batch(pages, table, cu, length, "length", n, max_count)
    if n == 0 or b.seqs == 0:
        return out
    longest = b.table_width * pages.page_tokens
    if max_length is not None and max_length < longest:
        if max_length < 0:
            raise ValueError(f"max_length {max_length}")
        longest = max_length
    lib = library()
    mask = _mask(n, pages.index, b, causal, window, sinks, tree)
    if mask is None:
        need = lib.wl_kv_attend_workspace_bytes(pages.ref, heads, b, longest)
    else:
        need = lib.wl_kv_attend_masked_workspace_bytes(pages.ref, heads, b, longest, mask)
    space = None
    if workspace is not None:
        if workspace.dtype is not torch.uint8 or workspace.get_device() != pages.index or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous uint8 tensor on the cache's device")
        space, need = workspace.data_ptr(), workspace.numel()
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=pages.device)
        space = workspace.data_ptr()
    _launch(pages.index, lib.wl_kv_attend if mask is None else lib.wl_kv_attend_masked, pages.ref, layer, q.data_ptr(), token_stride,
            head_stride, heads, b, length.data_ptr(), longest, pages.head_dim ** -0.5 if scale is None else scale,
            causal if mask is None else mask, out.data_ptr(), space, need)
    return out


def kv_tree(parents: torch.Tensor, start: torch.Tensor, cu: torch.Tensor, max_count: int = None):
    """A tree of drafted tokens for each sequence -> (tree, positions): int64 [tokens, words] masks as kv_attend takes them (a row's
    ancestors and itself) and int64 [tokens] positions, start[b] plus the number of a row's ancestors. parents: int32 [tokens], each
    row's parent among its sequence's rows cu[b] .. cu[b + 1], counted from 0, and before the row itself; anything else (-1) is a
    root, behind the last token before the draft. start, cu int32 [seqs], [seqs + 1]; max_count: the most rows any sequence has
    (words = max_count / 64 rounded up; rows beyond it are dropped; default: all rows); cu must not decrease (rows that two sequences
    then claim hold what either writes). Rows of no sequence get no bits and position 0. Once a step: every layer takes the same
    masks. Meant for drafts: the time grows with a sequence's rows times their depth."""
    index = parents.get_device() if isinstance(parents, torch.Tensor) else -1
    for t, name, dim in ((parents, "parents", "tokens"), (start, "start", "sequences"), (cu, "cu", "sequences + 1")):
        if not (isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.get_device() == index and t.dim() == 1 and t.is_contiguous()):
            _refuse(t, name, f"cuda:{index}", torch.int32, f"[{dim}], contiguous")
    n, seqs = parents.shape[0], start.shape[0]
    if cu.shape[0] != seqs + 1:
        raise ValueError(f"cu must be [{seqs + 1}] for {seqs} sequences (got {list(cu.shape)})")
    if max_count is None or max_count > n:
        max_count = n
    if (seqs | n | max_count) >> 31:
        raise ValueError(f"max_count {max_count} with {seqs} sequences and {n} rows")
    words = max(1, -(-max_count // 64))
    tree = torch.empty(n, words, dtype=torch.int64, device=parents.device)
    positions = torch.empty(n, dtype=torch.int64, device=parents.device)
    if n == 0 or seqs == 0:
        return tree.zero_(), positions.zero_()
    _launch(index, library().wl_kv_tree, WlKvBatch(None, cu.data_ptr(), 1, n, seqs, 1, max_count, 0), parents.data_ptr(),
            start.data_ptr(), tree.data_ptr(), words, positions.data_ptr())
    return tree, positions


def kv_keep(pages: KVPages, table: torch.Tensor, start: torch.Tensor, keep: torch.Tensor, cu: torch.Tensor, max_count: int = None):
    """Moves accepted tokens up in the cache, on every layer: for the i-th of keep's entries cu[b] .. cu[b + 1] (int32), the token at
    position start[b] + keep[..] of sequence b goes to position start[b] + i, as if all were read before any is written. Entries
    have to be at least i (less is taken as i: the token stays); increasing ones are the accepted tokens in order. What lies behind
    the last of them is no longer the sequence's (shorten its length), and stays as it is. A page that receives tokens keeps its
    scale, times the smallest power of two with which it covers the tokens kept in it; bytes that stay in a page whose scale stays
    move as they are. Tokens whose page is not there are not moved. A page that receives tokens belongs to one of the call's sequences
    alone."""
    index = pages.index
    _need(keep, "keep", index, torch.int32, ("rows",))
    n = keep.shape[0]
    if not keep.is_contiguous():
        raise ValueError("keep must be contiguous")
    b = _batch(pages, table, cu, start, "start", n, max_count)
    if n == 0 or b.seqs == 0:
        return
    _launch(index, library().wl_kv_keep, pages.ref, b, start.data_ptr(), keep.data_ptr())


def _page_numbers(x, name):
    """x as int32, unless a number would become another one by that."""
    a = np.asarray(x)
    if a.dtype != np.int32:
        if a.size and (a.dtype.kind not in "iu" or int(a.min()) < 0 or int(a.max()) >= 2 ** 31):
            raise ValueError(f"{name} must be page numbers")
        a = a.astype(np.int32)
    return np.ascontiguousarray(a)


def kv_copy(pages: KVPages, src, dst):
    """Copies pages src[i] -> dst[i] of every layer, bytes and scales. src, dst: page numbers on the host (lists or integer
    arrays); they travel in the kernels' arguments, so nothing is uploaded. Refused (ValueError): a page out of range, one
    written twice, one both read and written."""
    src, dst = _page_numbers(src, "src"), _page_numbers(dst, "dst")
    if src.ndim != 1 or src.shape != dst.shape:
        raise ValueError(f"src and dst must be lists of the same length (got {list(src.shape)} and {list(dst.shape)})")
    if src.shape[0] == 0:
        return
    _launch(pages.index, library().wl_kv_copy, pages.ref, src.ctypes.data, dst.ctypes.data, src.shape[0])


@functools.lru_cache(maxsize=64)
def _sections(sections):
    return (ctypes.c_int32 * len(sections))(*sections)


def _rotated_into(out, x, index, dim):
    """(token stride, head stride) of the tensor that x's rotated values go to."""
    n, _, token, head = _rows(out, "out", index, x.dtype, x.shape[1], dim)
    if n != x.shape[0] or (out.data_ptr() == x.data_ptr() and (token, head) != x.stride()[:2]):
        raise ValueError("out must have its tensor's shape, and its strides where it is the same memory")
    return token, head


def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections=None,
         interleaved: bool = True, scale: float = 1.0, out=None):
    """Rotary positions with several axes: q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] (or None), both bf16
    or both fp32 (any strides over tokens and heads), rotated into new tensors (or into `out`, a (q, k) pair, which may be
    q and k themselves, but not overlap them otherwise; rows of one that share memory are refused) -> (q, k).
    positions: int64 [axes, tokens] (or [tokens], one axis); inv_freq: fp64 [rotary_dim / 2], the angle of one position step;
    sections[i] of its frequencies belong to axis i, interleaved (axis i > 0 has the frequencies i, i + axes, i + 2 axes, ..; axis
    0 the rest) or one axis after the other. Value pairs (j, j + rotary_dim / 2) turn by positions[axis(j)] * inv_freq[j], taken in
    64 bits; cosine and sine are multiplied by `scale`; the rest of each head
    is copied. (engines/base.py:16-89 has the one-axis form.)"""
    return _rotate(library().wl_rope, q, k, positions, inv_freq, sections, interleaved, scale, out, ())


def norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, q_weight: torch.Tensor = None,
              k_weight: torch.Tensor = None, eps: float = 1e-6, zero_centered: bool = True, sections=None,
              interleaved: bool = True, scale: float = 1.0, out=None):
    """rope() on queries and keys that are normed first, each head by itself: x / sqrt(mean(x^2) + eps) * w, in fp32 up to the one
    rounding of the rotated values. w: 1 + weight with zero_centered (the reference's RMSNorm, engines/base.py:27-31), else weight;
    q_weight and k_weight [head_dim], both fp32 or both bf16, None: w = 1. The rest as in rope."""
    if not 0 <= eps < float("inf"):
        raise ValueError(f"eps {eps}")
    index, dim, kind, at = q.get_device(), q.shape[-1], None, []
    for w in (q_weight, k_weight):
        if w is None:
            at.append(None)
            continue
        kind = w.dtype if kind is None else kind
        if not (w.dtype is kind and w.get_device() == index and w.dim() == 1 and w.shape[0] == dim and w.is_contiguous()):
            _refuse(w, "q_weight" if not at else "k_weight", q.device, kind, f"[{dim}], contiguous,")
        at.append(w.data_ptr())
    if kind not in (None, torch.float32, torch.bfloat16):
        raise ValueError(f"the weights must be fp32 or bf16 (got {kind})")
    return _rotate(library().wl_norm_rope, q, k, positions, inv_freq, sections, interleaved, scale, out,
                   (*at, DTYPE_BF16 if kind is torch.bfloat16 else DTYPE_F32, eps, zero_centered))


def _rotate(call, q, k, positions, inv_freq, sections, interleaved, scale, out, more):
    """One call of wl_rope or wl_norm_rope; more: its arguments behind the scale."""
    dtype, index = q.dtype, q.get_device()
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise ValueError(f"q must be bf16 or fp32 (got {dtype})")
    if index < 0:
        raise ValueError(f"q must be on the GPU (got {q.device})")
    dim = q.shape[-1]
    n, heads, token, head = _rows(q, "q", index, dtype, None, dim)
    if positions.dim() == 1:
        positions = positions[None]
    if not (positions.dtype is torch.int64 and positions.get_device() == index and positions.dim() == 2):
        _refuse(positions, "positions", q.device, torch.int64, "[axes, tokens]")
    if not (inv_freq.dtype is torch.float64 and inv_freq.get_device() == index and inv_freq.dim() == 1 and inv_freq.is_contiguous()):
        _refuse(inv_freq, "inv_freq", q.device, torch.float64, "[rotary_dim / 2], contiguous")
    axes, cols = positions.shape
    axis_stride, step = positions.stride()
    half = inv_freq.shape[0]
    sections = (half,) if sections is None else tuple(sections)
    if len(sections) != axes or cols != n or (step != 1 and n > 1):
        raise ValueError(f"positions must be [{len(sections)}, {n}] (axes as in sections {sections}, q's tokens) with contiguous "
                         f"rows (got {list(positions.shape)})")
    q_out, k_out = (None, None) if out is None else out
    if q_out is None:
        q_out, to = torch.empty_like(q, memory_format=torch.contiguous_format), (heads * dim, dim)
    else:
        to = _rotated_into(q_out, q, index, dim)
    q_arg = WlRopeTensor(q.data_ptr(), q_out.data_ptr(), token, head, *to, heads, 0)
    k_arg = None
    if k is not None:
        rows, heads, token, head = _rows(k, "k", index, dtype, None, dim)
        if rows != n:
            raise ValueError(f"q has {n} rows, k {rows}")
        if k_out is None:
            k_out, to = torch.empty_like(k, memory_format=torch.contiguous_format), (heads * dim, dim)
        else:
            to = _rotated_into(k_out, k, index, dim)
        k_arg = WlRopeTensor(k.data_ptr(), k_out.data_ptr(), token, head, *to, heads, 0)
    if n:
        _launch(index, call, q_arg, k_arg, DTYPE_BF16 if dtype is torch.bfloat16 else DTYPE_F32, n, dim, 2 * half,
                positions.data_ptr(), axis_stride, inv_freq.data_ptr(), axes, _sections(sections), interleaved, scale, *more)
    return q_out, k_out
