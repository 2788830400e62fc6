"""Serving from 4-bit weights and a 4-bit key/value cache (the `q4` and `kv4` entry points of include/phobos_leaf.h).

    W  = q4_pack(codes, scales, zeros, group)                 # once
    gemv_q4(X, W, Y, group)                                   # beside `gemm`: a few rows against 4-bit weights

    cache = Kv4Cache.create(layers, n_pages, kv_heads, head_dim, group, page_tokens, max_seqs, table_width)
    kv4_extend(cache, slots, counts, shortfall, workspace=ws) # room for the new tokens; *shortfall != 0: nothing changed
    kv4_append(cache, layer, K, V, slots, indptr)             # per layer: the new tokens' keys and values
    kv4_attention(cache, layer, Q, O, scale, slots, indptr, workspace=ws)
    kv4_fork / kv4_free / kv4_compact                         # share or copy a sequence, give pages back, close gaps

Calls enqueue on the current (or given) stream; index arrays are int32 device tensors and are not read by the host.
"""
from __future__ import annotations

import ctypes

from . import (F16, F32, I8, I32, PH_ERR_INVALID, PH_ERR_UNSUPPORTED, PhobosError, PhTensor, _stream_ptr, _ws, check, lib)


class PhKv4Cache(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_void_p), ("refs", ctypes.c_void_p), ("tables", ctypes.c_void_p), ("lens", ctypes.c_void_p),
                ("layer_pitch", ctypes.c_int64), ("layers", ctypes.c_int32), ("n_pages", ctypes.c_int32),
                ("page_tokens", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("group", ctypes.c_int32), ("max_seqs", ctypes.c_int32), ("table_width", ctypes.c_int32)]


def _on_device(t, name: str) -> None:
    import torch
    if not t.is_cuda:
        raise PhobosError(PH_ERR_INVALID, f"{name} is not on a CUDA device")
    if t.device.index != torch.cuda.current_device():
        raise PhobosError(PH_ERR_INVALID, f"{name} lives on cuda:{t.device.index} but the current device is "
                                          f"cuda:{torch.cuda.current_device()}")


def _desc(t, name: str) -> PhTensor:
    """PhTensor of a rank-1/2 CUDA tensor of any element type these entry points know (no copy)."""
    import torch
    _on_device(t, name)
    codes = {torch.float16: F16, torch.float32: F32, torch.int8: I8, torch.uint8: I8, torch.int32: I32}
    if t.dtype not in codes:
        raise PhobosError(PH_ERR_UNSUPPORTED, f"{name}: element type {t.dtype}")
    if t.dim() not in (1, 2):
        raise PhobosError(PH_ERR_INVALID, f"{name}: rank {t.dim()}, expected 1 or 2")
    d = PhTensor(t.data_ptr(), codes[t.dtype], t.dim())
    for i in range(t.dim()):
        d.sizes[i], d.strides[i] = t.shape[i], t.stride(i)
    return d


def _ints(t, name: str, n: int | None = None):
    """Address of a contiguous int32 device tensor of at least n values (None stays None)."""
    import torch
    if t is None:
        return None
    _on_device(t, name)
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise PhobosError(PH_ERR_INVALID, f"{name}: expected a contiguous int32 tensor")
    if n is not None and t.numel() < n:
        raise PhobosError(PH_ERR_INVALID, f"{name}: {t.numel()} values, expected {n}")
    return t.data_ptr()


# ---- 4-bit weights ----------------------------------------------------------------------------
def q4_packed_bytes(N: int, K: int, group: int) -> int:
    return int(lib().phobos_q4_packed_bytes(N, K, group))


def q4_pack(codes, scales, zeros, group: int, out=None, stream=None):
    """Lays out codes [N, K] (one per byte, 0..15), scales and zeros [N, K/group] (f16; zeros None: 8) for gemv_q4."""
    import torch
    if out is None:
        need = q4_packed_bytes(codes.shape[0], codes.shape[1], group)
        out = torch.empty(need, dtype=torch.int8, device=codes.device)
    c, s, o = _desc(codes, "codes"), _desc(scales, "scales"), _desc(out, "packed")
    z = _desc(zeros, "zeros") if zeros is not None else None
    check(lib().phobos_q4_pack(ctypes.byref(c), ctypes.byref(s), ctypes.byref(z) if z else None, group, ctypes.byref(o),
                               _stream_ptr(stream)))
    return out


def gemv_q4(X, packed, Y, group: int, alpha: float = 1.0, beta: float = 0.0, stream=None) -> None:
    """Y[M,N] = alpha * X[M,K] W[N,K]^T + beta * Y, W = scale * (code - zero) in 4 bits; X f16, Y f16 or f32."""
    x, w, y = _desc(X, "X"), _desc(packed, "packed"), _desc(Y, "Y")
    check(lib().phobos_gemv_q4(ctypes.byref(x), ctypes.byref(w), ctypes.byref(y), alpha, beta, group, _stream_ptr(stream)))


# ---- the cache ------------------------------------------------------------------------------------
def kv4_page_bytes(kv_heads: int, head_dim: int, group: int, page_tokens: int) -> int:
    return int(lib().phobos_kv4_page_bytes(kv_heads, head_dim, group, page_tokens))


class Kv4Cache:
    """Keys and values of sequences in 4 bits: pages [layers, n_pages, page bytes] (8-bit), and int32 refs [n_pages],
    tables [max_seqs, table_width], lens [max_seqs].  Holds the tensors; the calls below change them in place."""

    def __init__(self, pages, refs, tables, lens, *, kv_heads: int, head_dim: int, group: int, page_tokens: int):
        for t, name in ((pages, "pages"), (refs, "refs"), (tables, "tables"), (lens, "lens")):
            _on_device(t, name)
        need = kv4_page_bytes(kv_heads, head_dim, group, page_tokens)
        if need == 0:
            raise PhobosError(PH_ERR_UNSUPPORTED, f"kv4: {kv_heads} heads of {head_dim} dims in groups of {group}, pages of "
                                                  f"{page_tokens} tokens")
        if pages.dim() != 3 or pages.element_size() != 1 or pages.shape[2] != need or pages.stride(2) != 1 or (
                pages.shape[1] > 1 and pages.stride(1) != need):
            raise PhobosError(PH_ERR_INVALID, f"pages: expected [layers, n_pages, {need}] bytes with whole pages side by side")
        if tables.dim() != 2 or lens.numel() != tables.shape[0] or refs.numel() != pages.shape[1]:
            raise PhobosError(PH_ERR_INVALID, "kv4: refs [n_pages], tables [max_seqs, table_width] and lens [max_seqs] do not agree")
        self.pages, self.refs, self.tables, self.lens = pages, refs, tables, lens
        self.kv_heads, self.head_dim, self.group, self.page_tokens = kv_heads, head_dim, group, page_tokens
        pitch = pages.stride(0) if pages.shape[0] > 1 else 0
        self.struct = PhKv4Cache(pages.data_ptr(), _ints(refs, "refs"), _ints(tables, "tables"), _ints(lens, "lens"), pitch,
                                 pages.shape[0], pages.shape[1], page_tokens, kv_heads, head_dim, group, tables.shape[0],
                                 tables.shape[1])

    @classmethod
    def create(cls, layers: int, n_pages: int, kv_heads: int, head_dim: int, group: int, page_tokens: int, max_seqs: int,
               table_width: int, device=None) -> "Kv4Cache":
        """An empty cache in newly allocated device memory."""
        import torch
        device = device if device is not None else torch.device("cuda", torch.cuda.current_device())
        i32 = dict(dtype=torch.int32, device=device)
        pages = torch.empty((layers, n_pages, kv4_page_bytes(kv_heads, head_dim, group, page_tokens)), dtype=torch.uint8, device=device)
        return cls(pages, torch.zeros(n_pages, **i32), torch.full((max_seqs, table_width), -1, **i32), torch.zeros(max_seqs, **i32),
                   kv_heads=kv_heads, head_dim=head_dim, group=group, page_tokens=page_tokens)


def _batch(cache: Kv4Cache, slots, indptr):
    _on_device(cache.pages, "the cache")
    n = slots.numel()
    return _ints(slots, "slots"), _ints(indptr, "indptr", n + 1), n


def kv4_append(cache: Kv4Cache, layer: int, K, V, slots, indptr=None, stream=None) -> None:
    """Quantises rows K, V [T, kv_heads * head_dim] into the places of the sequences' last tokens (see kv4_extend)."""
    s, i, n = _batch(cache, slots, indptr)
    k, v = _desc(K, "K"), _desc(V, "V")
    check(lib().phobos_kv4_append(ctypes.byref(cache.struct), layer, ctypes.byref(k), ctypes.byref(v), s, i, n, _stream_ptr(stream)))


def kv4_read(cache: Kv4Cache, layer: int, K, V, slots, indptr=None, stream=None) -> None:
    """The values of the sequences' last tokens into rows K, V: the inverse of kv4_append."""
    s, i, n = _batch(cache, slots, indptr)
    k, v = _desc(K, "K"), _desc(V, "V")
    check(lib().phobos_kv4_read(ctypes.byref(cache.struct), layer, ctypes.byref(k), ctypes.byref(v), s, i, n, _stream_ptr(stream)))


def kv4_attention_workspace_bytes(cache: Kv4Cache, T: int, n: int, q_heads: int) -> int:
    return int(lib().phobos_kv4_attention_workspace_bytes(ctypes.byref(cache.struct), T, n, q_heads))


def kv4_attention(cache: Kv4Cache, layer: int, Q, O, scale: float, slots, indptr=None, lse=None, window: int = 0, workspace=None,
                  stream=None) -> None:
    """O = softmax(scale q K^T) V over the cache; Q, O [T, q_heads * head_dim] f16.  The row of position p sees tokens
    j <= p (window > 0: only j > p - window); one that sees nothing gets zeros and lse -inf."""
    s, i, n = _batch(cache, slots, indptr)
    q, o = _desc(Q, "Q"), _desc(O, "O")
    l = _desc(lse, "lse") if lse is not None else None
    wp, wn = _ws(workspace)
    check(lib().phobos_kv4_attention(ctypes.byref(cache.struct), layer, ctypes.byref(q), ctypes.byref(o),
                                     ctypes.byref(l) if l else None, scale, window, s, i, n, wp, wn, _stream_ptr(stream)))


def kv4_pages_workspace_bytes(cache: Kv4Cache) -> int:
    return int(lib().phobos_kv4_pages_workspace_bytes(ctypes.byref(cache.struct)))


def kv4_extend(cache: Kv4Cache, slots, counts, shortfall, workspace=None, stream=None) -> None:
    """Room for counts[i] more tokens of slots[i], and the new lengths.  shortfall (int32 [1], device): 0 done, > 0 pages
    missing, -1 a wrong request; unless it is 0 nothing has changed and the rows must not be appended."""
    s, _, n = _batch(cache, slots, None)
    wp, wn = _ws(workspace)
    check(lib().phobos_kv4_extend(ctypes.byref(cache.struct), s, _ints(counts, "counts", n), n, _ints(shortfall, "shortfall", 1), wp, wn,
                                  _stream_ptr(stream)))


def kv4_fork(cache: Kv4Cache, src, dst, shortfall, deep: bool = False, workspace=None, stream=None) -> None:
    """The empty sequences dst[i] continue from src[i], sharing its pages, or (deep) with copies of them."""
    s, _, n = _batch(cache, src, None)
    wp, wn = _ws(workspace)
    check(lib().phobos_kv4_fork(ctypes.byref(cache.struct), s, _ints(dst, "dst", n), n, int(deep), _ints(shortfall, "shortfall", 1), wp, wn,
                                _stream_ptr(stream)))


def kv4_free(cache: Kv4Cache, slots, keep=None, stream=None) -> None:
    """Shortens slots[i] to keep[i] tokens (None: to none) and gives the pages behind them back."""
    s, _, n = _batch(cache, slots, None)
    check(lib().phobos_kv4_free(ctypes.byref(cache.struct), s, _ints(keep, "keep", n), n, _stream_ptr(stream)))


def kv4_compact(cache: Kv4Cache, live, workspace=None, stream=None) -> None:
    """Moves the pages in use to ids 0 .. live[0] - 1 in every layer."""
    _on_device(cache.pages, "the cache")
    wp, wn = _ws(workspace)
    check(lib().phobos_kv4_compact(ctypes.byref(cache.struct), _ints(live, "live", 1), wp, wn, _stream_ptr(stream)))
