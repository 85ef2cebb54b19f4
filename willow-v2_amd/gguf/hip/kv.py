"""The attention half's operators: rotary positions, the paged 8-bit key/value cache and attention over it.

The reference keeps keys and values in a bf16 tensor per layer that grows in blocks of 256 positions and runs torch's
attention on it (engines/base.py:213-216,328-367). Here the cache is pages of bytes with one scale for each page and kv
head, shared by any number of sequences through page tables (gguf.hbm_cache keeps those), half the bytes of bf16 to read for
every decoded token. All calls only enqueue work on the current stream of their tensors' device and read page tables,
lengths and row offsets on the GPU, so they may be captured into a HIP graph.
"""
import contextlib
import ctypes

import numpy as np
import torch

from . import DTYPE_BF16, DTYPE_F32, KV_E4M3, KV_INT8, WlKvBatch, WlKvCache, WlRopeTensor, _stream, check, library

TYPES = {torch.int8: KV_INT8, torch.float8_e4m3fn: KV_E4M3}


def _on_device(device):
    """The device made current where it is not (a launch goes to the current device)."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _need(t, name, device, dtype, dims=None):
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != dtype or (dims is not None and t.dim() != dims):
        got = f"{t.dtype} {list(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{name} must be a {'' if dims is None else f'{dims}-d '}{dtype} tensor on {device} (got {got})")


def _rows(t, name, device, dtype, heads, head_dim):
    """A [tokens, heads, head_dim] tensor whose head_dim is contiguous -> (pointer, token stride, head stride)."""
    _need(t, name, device, dtype, 3)
    if t.shape[2] != head_dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {head_dim}] (got {list(t.shape)})")
    if t.shape[2] > 1 and t.stride(2) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return t.data_ptr(), t.stride(0), t.stride(1)


class KVPages:
    """A paged key/value cache on one GPU, all layers: k int8 or float8_e4m3fn [layers, pages, kv_heads, page_tokens,
    head_dim], v of the same type [layers, pages, kv_heads, head_dim, page_tokens] (tokens innermost: the order in which the
    matrix core takes them), k_scale and v_scale fp32 [layers, pages, kv_heads], all contiguous. A value is its byte times its
    block's scale. head_dim 64, 128 or 256; page_tokens a multiple of 16 up to 1024."""

    def __init__(self, k, v, k_scale, v_scale):
        if not isinstance(k, torch.Tensor) or k.dim() != 5 or k.dtype not in TYPES:
            raise ValueError("k must be an int8 or float8_e4m3fn tensor [layers, pages, kv_heads, page_tokens, head_dim]")
        layers, pages, heads, tokens, dim = k.shape
        _need(v, "v", k.device, k.dtype, 5)
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            _need(t, name, k.device, torch.float32, 3)
            if tuple(t.shape) != (layers, pages, heads):
                raise ValueError(f"{name} must be [layers, pages, kv_heads] = {[layers, pages, heads]} (got {list(t.shape)})")
        if tuple(v.shape) != (layers, pages, heads, dim, tokens):
            raise ValueError(f"v must be [layers, pages, kv_heads, head_dim, page_tokens] = {[layers, pages, heads, dim, tokens]} "
                             f"(got {list(v.shape)})")
        if not all(t.is_contiguous() for t in (k, v, k_scale, v_scale)):
            raise ValueError("the cache's tensors must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers, self.pages, self.kv_heads, self.page_tokens, self.head_dim = layers, pages, heads, tokens, dim
        self.dtype, self.device = k.dtype, k.device
        s = WlKvCache()
        s.k, s.v, s.k_scale, s.v_scale = k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr()
        s.pages, s.layers, s.kv_heads, s.page_tokens, s.head_dim = pages, layers, heads, tokens, dim
        s.type = TYPES[k.dtype]
        self.struct = s
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
    _need(table, "table", pages.device, torch.int32, 2)
    _need(cu, "cu", pages.device, torch.int32, 1)
    _need(per_seq, name, pages.device, torch.int32, 1)
    seqs = table.shape[0]
    if cu.shape[0] != seqs + 1 or per_seq.shape[0] != seqs:
        raise ValueError(f"table has {seqs} sequences: cu must have {seqs + 1} entries (got {cu.shape[0]}) and {name} {seqs} "
                         f"(got {per_seq.shape[0]})")
    if not cu.is_contiguous() or not per_seq.is_contiguous() or (table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError(f"cu, {name} and the rows of table must be contiguous")
    b = WlKvBatch()
    b.table, b.cu = table.data_ptr(), cu.data_ptr()
    b.table_stride = table.stride(0) if seqs > 1 else max(table.stride(0), table.shape[1])
    b.tokens, b.seqs, b.table_width = tokens, seqs, table.shape[1]
    b.max_count = tokens if max_count is None else min(int(max_count), tokens)
    return b


def kv_append(pages: KVPages, layer: int, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
              cu: torch.Tensor, max_count: int = None):
    """Quantizes new keys and values of one layer into the cache: k, v bf16 [tokens, kv_heads, head_dim] (any strides over
    tokens and heads), sequence b's rows cu[b] .. cu[b + 1] to its positions start[b], start[b] + 1, ... of the pages in
    table[b] (int32 [seqs, width]; cu int32 [seqs + 1], start int32 [seqs]). max_count: the most rows any sequence has (rows
    beyond it are dropped; default: all rows). A page that begins among the rows gets the smallest bf16 scale that covers its
    rows, a page with older tokens its scale times the smallest power of two that does (its older bytes are divided by it and
    rounded); a NaN or an infinity makes its block's scale NaN. Rows whose page is not there (no table entry, or one outside
    the cache) are dropped. Pages written in one call must be distinct over its sequences."""
    kp, vp = (_rows(t, n, pages.device, torch.bfloat16, pages.kv_heads, pages.head_dim) for n, t in (("k", k), ("v", v)))
    if k.shape[0] != v.shape[0]:
        raise ValueError(f"k has {k.shape[0]} rows, v {v.shape[0]}")
    b = _batch(pages, table, cu, start, "start", k.shape[0], max_count)
    if k.shape[0] == 0 or b.seqs == 0:
        return
    with _on_device(pages.device):
        check(library().wl_kv_append(ctypes.byref(pages.struct), layer, *kp, *vp, ctypes.byref(b), start.data_ptr(),
                                     _stream(pages.device)))


def kv_attend(pages: KVPages, layer: int, q: torch.Tensor, table: torch.Tensor, length: torch.Tensor, cu: torch.Tensor,
              max_count: int = None, max_length: int = None, scale: float = None, causal: bool = True,
              out: torch.Tensor = None, workspace: torch.Tensor = None) -> torch.Tensor:
    """Grouped-query attention of one layer: q bf16 [tokens, q_heads, head_dim] (any strides over tokens and heads) -> bf16
    [tokens, q_heads, head_dim]. Sequence b's rows are cu[b] .. cu[b + 1], the last of its length[b] tokens in the cache (so
    append them first); query head i reads kv head i / (q_heads / kv_heads). causal: a row sees the positions up to its own;
    otherwise all length[b]. A row that sees none is 0. scale defaults to head_dim ** -0.5. max_count: the most rows any
    sequence has (rows beyond it are not computed; default: all rows); max_length: a bound of length that only steers how the
    work is split (default: what the table's width holds). Rows behind cu[-1] of `out` stay as they are. workspace: a uint8
    tensor of kv_attend_workspace bytes; by default it comes from torch's allocator, for this call and stream."""
    _rows(q, "q", pages.device, torch.bfloat16, None, pages.head_dim)
    heads = q.shape[1]
    if heads == 0 or heads % pages.kv_heads:
        raise ValueError(f"{heads} query heads over {pages.kv_heads} kv heads")
    if out is None:
        out = torch.empty(q.shape, dtype=torch.bfloat16, device=q.device)
    else:
        _need(out, "out", pages.device, torch.bfloat16, 3)
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {list(q.shape)} tensor")
    b = _batch(pages, table, cu, length, "length", q.shape[0], max_count)
    if q.shape[0] == 0 or b.seqs == 0:
        return out
    most = b.table_width * pages.page_tokens
    longest = most if max_length is None else min(int(max_length), most)
    lib = library()
    need = lib.wl_kv_attend_workspace_bytes(ctypes.byref(pages.struct), heads, ctypes.byref(b), longest)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    elif workspace.dtype != torch.uint8 or workspace.device != q.device or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous uint8 tensor on the cache's device")
    with _on_device(pages.device):
        check(lib.wl_kv_attend(ctypes.byref(pages.struct), layer, q.data_ptr(), q.stride(0), q.stride(1), heads,
                               ctypes.byref(b), length.data_ptr(), longest,
                               pages.head_dim ** -0.5 if scale is None else scale, int(causal), out.data_ptr(),
                               workspace.data_ptr() if workspace is not None else None,
                               workspace.numel() if workspace is not None else 0, _stream(pages.device)))
    return out


def kv_copy(pages: KVPages, src, dst):
    """Copies pages src[i] -> dst[i] of every layer, bytes and scales. src, dst: page numbers on the host (lists or integer
    arrays); they travel in the kernels' arguments, so nothing is uploaded. Refused (ValueError): a page out of range, one
    written twice, one both read and written."""
    src, dst = (np.ascontiguousarray(x, dtype=np.int32) for x in (src, dst))
    if src.ndim != 1 or src.shape != dst.shape:
        raise ValueError(f"src and dst must be lists of the same length (got {list(src.shape)} and {list(dst.shape)})")
    with _on_device(pages.device):
        check(library().wl_kv_copy(ctypes.byref(pages.struct), src.ctypes.data, dst.ctypes.data, src.shape[0],
                                   _stream(pages.device)))


def rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, sections=None,
         interleaved: bool = True, scale: float = 1.0, out=None):
    """Rotary positions with several axes: q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] (or None), both bf16
    or both fp32 (any strides over tokens and heads), rotated into new tensors (or into `out`, a (q, k) pair, which may be
    q and k themselves) -> (q, k). positions: int64 [axes, tokens] (or [tokens], one axis); inv_freq: fp64 [rotary_dim / 2],
    the angle of one position step; sections[i] of its frequencies belong to axis i, interleaved (axis i > 0 has the
    frequencies i, i + axes, i + 2 axes, ..; axis 0 the rest) or one axis after the other. Value pairs (j, j + rotary_dim / 2)
    turn by positions[axis(j)] * inv_freq[j], taken in 64 bits; cosine and sine are multiplied by `scale`; the rest of each head
    is copied. (engines/base.py:16-89 has the one-axis form.)"""
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"q must be bf16 or fp32 (got {q.dtype})")
    if not q.is_cuda:
        raise ValueError(f"q must be on the GPU (got {q.device})")
    positions = positions.reshape(1, -1) if positions.dim() == 1 else positions
    _need(positions, "positions", q.device, torch.int64, 2)
    _need(inv_freq, "inv_freq", q.device, torch.float64, 1)
    half, axes = inv_freq.shape[0], positions.shape[0]
    sections = (half,) if sections is None else tuple(int(s) for s in sections)
    if len(sections) != axes:
        raise ValueError(f"positions has {axes} axes, sections {len(sections)}")
    if positions.shape[1] != q.shape[0] or (positions.shape[1] > 1 and positions.stride(1) != 1) or not inv_freq.is_contiguous():
        raise ValueError(f"positions must be [axes, {q.shape[0]}] with contiguous rows, inv_freq contiguous")
    outs = (None, None) if out is None else out
    structs, got = [], []
    for name, x, y in (("q", q, outs[0]), ("k", k, outs[1])):
        if x is None:
            structs.append(None)
            got.append(None)
            continue
        p, ts, hs = _rows(x, name, q.device, q.dtype, None, q.shape[2])
        if x.shape[0] != q.shape[0]:
            raise ValueError(f"q has {q.shape[0]} rows, k {x.shape[0]}")
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if y is None else y
        yp, yts, yhs = _rows(y, "out", q.device, q.dtype, x.shape[1], q.shape[2])
        if y.shape != x.shape or (yp == p and (yts, yhs) != (ts, hs)):
            raise ValueError(f"out of {name} must have its shape (and its strides where it is the same memory)")
        structs.append(WlRopeTensor(p, yp, ts, hs, yts, yhs, x.shape[1], 0))
        got.append(y)
    if q.shape[0] == 0:
        return tuple(got)
    with _on_device(q.device):
        check(library().wl_rope(ctypes.byref(structs[0]), ctypes.byref(structs[1]) if structs[1] is not None else None,
                                DTYPE_BF16 if q.dtype == torch.bfloat16 else DTYPE_F32, q.shape[0], q.shape[2], 2 * half,
                                positions.data_ptr(), positions.stride(0), inv_freq.data_ptr(), axes,
                                (ctypes.c_int32 * axes)(*sections), int(interleaved), scale, _stream(q.device)))
    return tuple(got)
