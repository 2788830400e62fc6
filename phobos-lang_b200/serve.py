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
import struct

from . import (F16, F32, I8, I32, PH_ERR_INVALID, PH_ERR_UNSUPPORTED, PhobosError, PhTensor, check, lib)


class PhKv4Cache(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_void_p), ("refs", ctypes.c_void_p), ("tables", ctypes.c_void_p), ("lens", ctypes.c_void_p),
                ("layer_pitch", ctypes.c_int64), ("layers", ctypes.c_int32), ("n_pages", ctypes.c_int32),
                ("page_tokens", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("group", ctypes.c_int32), ("max_seqs", ctypes.c_int32), ("table_width", ctypes.c_int32)]


_PACK = struct.Struct("<Qiiqqqqq").pack     # PhTensor, as the C compiler lays it out
assert struct.calcsize("<Qiiqqqqq") == ctypes.sizeof(PhTensor)


_torch = None          # imported at the first call, as everywhere in this package
_CODES = {}
_get_device = _get_stream = None


def _load_torch():
    global _torch, _CODES, _get_device, _get_stream
    import torch
    _CODES = {torch.float16: F16, torch.float32: F32, torch.int8: I8, torch.uint8: I8, torch.int32: I32}
    # The raw getters cost a tenth of the documented ones (which build a Stream object, and check each time that CUDA is
    # up): much of a short call.  Where a torch lacks them the documented ones serve.
    torch.cuda.init()
    _get_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    _get_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)
    _torch = torch


def _device() -> int:
    if _torch is None:
        _load_torch()
    return _get_device()


def _stream(stream, device: int) -> int:
    if stream is None:
        return _get_stream(device)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _on_device(t, name: str, device: int) -> None:
    if t.get_device() != device:      # -1 for a CPU tensor
        if not t.is_cuda:
            raise PhobosError(PH_ERR_INVALID, f"{name} is not on a CUDA device")
        raise PhobosError(PH_ERR_INVALID, f"{name} lives on cuda:{t.device.index} but the current device is cuda:{device}")


def _desc(t, name: str, device: int) -> bytes:
    """A PhTensor, as bytes, of a rank-1/2 CUDA tensor of any element type these entry points know (no copy)."""
    if t.get_device() != device:
        _on_device(t, name, device)
    code = _CODES.get(t.dtype)
    if code is None:
        raise PhobosError(PH_ERR_UNSUPPORTED, f"{name}: element type {t.dtype}")
    size, stride = t.shape, t.stride()
    if len(size) == 2:
        return _PACK(t.data_ptr(), code, 2, size[0], size[1], stride[0], stride[1], 0)
    if len(size) == 1:
        return _PACK(t.data_ptr(), code, 1, size[0], 0, stride[0], 0, 0)
    raise PhobosError(PH_ERR_INVALID, f"{name}: rank {len(size)}, expected 1 or 2")


def byte_desc(t) -> PhTensor:
    """The descriptor of `launch` for a tensor that is not f16 or f32."""
    return PhTensor.from_buffer_copy(_desc(t, "tensor", _device()))


def _ints(t, name: str, device: int, n: int = 0):
    """Address of a contiguous int32 device tensor of at least n values (None stays None)."""
    if t is None:
        return None
    if t.get_device() != device:
        _on_device(t, name, device)
    if t.dtype is not _torch.int32 or not t.is_contiguous():
        raise PhobosError(PH_ERR_INVALID, f"{name}: expected a contiguous int32 tensor")
    if t.numel() < n:
        raise PhobosError(PH_ERR_INVALID, f"{name}: {t.numel()} values, expected {n}")
    return t.data_ptr()


def _space(workspace, device: int):
    if workspace is None:
        return None, 0
    _on_device(workspace, "workspace", device)
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


# ---- 4-bit weights ----------------------------------------------------------------------------
def q4_packed_bytes(N: int, K: int, group: int) -> int:
    return int(lib().phobos_q4_packed_bytes(N, K, group))


def q4_pack(codes, scales, zeros, group: int, out=None, stream=None):
    """Lays out codes [N, K] (one per byte, 0..15), scales and zeros [N, K/group] (f16; zeros None: 8) for gemv_q4."""
    import torch
    if out is None:
        need = q4_packed_bytes(codes.shape[0], codes.shape[1], group)
        out = torch.empty(need, dtype=torch.int8, device=codes.device)
    dev = _device()
    z = _desc(zeros, "zeros", dev) if zeros is not None else None
    check(lib().phobos_q4_pack(_desc(codes, "codes", dev), _desc(scales, "scales", dev), z, group, _desc(out, "packed", dev),
                               _stream(stream, dev)))
    return out


def gemv_q4(X, packed, Y, group: int, alpha: float = 1.0, beta: float = 0.0, stream=None) -> None:
    """Y[M,N] = alpha * X[M,K] W[N,K]^T + beta * Y, W = scale * (code - zero) in 4 bits; X f16, Y f16 or f32."""
    dev = _device()
    check(lib().phobos_gemv_q4(_desc(X, "X", dev), _desc(packed, "packed", dev), _desc(Y, "Y", dev), alpha, beta, group,
                               _stream(stream, dev)))


# ---- the cache ------------------------------------------------------------------------------------
def kv4_page_bytes(kv_heads: int, head_dim: int, group: int, page_tokens: int) -> int:
    return int(lib().phobos_kv4_page_bytes(kv_heads, head_dim, group, page_tokens))


class Kv4Cache:
    """Keys and values of sequences in 4 bits: pages [layers, n_pages, page bytes] (8-bit), and int32 refs [n_pages],
    tables [max_seqs, table_width], lens [max_seqs].  Holds the tensors; the calls below change them in place."""

    def __init__(self, pages, refs, tables, lens, *, kv_heads: int, head_dim: int, group: int, page_tokens: int):
        dev = _device()
        for t, name in ((pages, "pages"), (refs, "refs"), (tables, "tables"), (lens, "lens")):
            _on_device(t, name, dev)
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
        self.struct = PhKv4Cache(pages.data_ptr(), _ints(refs, "refs", dev), _ints(tables, "tables", dev), _ints(lens, "lens", dev), pitch,
                                 pages.shape[0], pages.shape[1], page_tokens, kv_heads, head_dim, group, tables.shape[0],
                                 tables.shape[1])
        self.address, self.device = ctypes.addressof(self.struct), dev

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
    dev = _device()
    if cache.device != dev:
        raise PhobosError(PH_ERR_INVALID, f"the cache lives on cuda:{cache.device} but the current device is cuda:{dev}")
    n = slots.numel()
    return dev, _ints(slots, "slots", dev), _ints(indptr, "indptr", dev, n + 1), n


def kv4_append(cache: Kv4Cache, layer: int, K, V, slots, indptr=None, stream=None) -> None:
    """Quantises rows K, V [T, kv_heads * head_dim] into the places of the sequences' last tokens (see kv4_extend)."""
    dev, s, i, n = _batch(cache, slots, indptr)
    check(lib().phobos_kv4_append(cache.address, layer, _desc(K, "K", dev), _desc(V, "V", dev), s, i, n, _stream(stream, dev)))


def kv4_read(cache: Kv4Cache, layer: int, K, V, slots, indptr=None, stream=None) -> None:
    """The values of the sequences' last tokens into rows K, V: the inverse of kv4_append."""
    dev, s, i, n = _batch(cache, slots, indptr)
    check(lib().phobos_kv4_read(cache.address, layer, _desc(K, "K", dev), _desc(V, "V", dev), s, i, n, _stream(stream, dev)))


def kv4_attention_workspace_bytes(cache: Kv4Cache, T: int, n: int, q_heads: int) -> int:
    return int(lib().phobos_kv4_attention_workspace_bytes(cache.address, T, n, q_heads))


def kv4_attention(cache: Kv4Cache, layer: int, Q, O, scale: float, slots, indptr=None, lse=None, window: int = 0, workspace=None,
                  stream=None) -> None:
    """O = softmax(scale q K^T) V over the cache; Q, O [T, q_heads * head_dim] f16.  The row of position p sees tokens
    j <= p (window > 0: only j > p - window); one that sees nothing gets zeros and lse -inf."""
    dev, s, i, n = _batch(cache, slots, indptr)
    l = _desc(lse, "lse", dev) if lse is not None else None
    wp, wn = _space(workspace, dev)
    check(lib().phobos_kv4_attention(cache.address, layer, _desc(Q, "Q", dev), _desc(O, "O", dev), l, scale, window, s, i, n, wp, wn,
                                     _stream(stream, dev)))


def kv4_pages_workspace_bytes(cache: Kv4Cache) -> int:
    return int(lib().phobos_kv4_pages_workspace_bytes(cache.address))


def kv4_extend(cache: Kv4Cache, slots, counts, shortfall, workspace=None, stream=None) -> None:
    """Room for counts[i] more tokens of slots[i], and the new lengths.  shortfall (int32 [1], device): 0 done, > 0 pages
    missing, -1 a wrong request; unless it is 0 nothing has changed and the rows must not be appended."""
    dev, s, _, n = _batch(cache, slots, None)
    wp, wn = _space(workspace, dev)
    check(lib().phobos_kv4_extend(cache.address, s, _ints(counts, "counts", dev, n), n, _ints(shortfall, "shortfall", dev, 1), wp, wn,
                                  _stream(stream, dev)))


def kv4_fork(cache: Kv4Cache, src, dst, shortfall, deep: bool = False, workspace=None, stream=None) -> None:
    """The empty sequences dst[i] continue from src[i], sharing its pages, or (deep) with copies of them."""
    dev, s, _, n = _batch(cache, src, None)
    wp, wn = _space(workspace, dev)
    check(lib().phobos_kv4_fork(cache.address, s, _ints(dst, "dst", dev, n), n, int(deep), _ints(shortfall, "shortfall", dev, 1), wp, wn,
                                _stream(stream, dev)))


def kv4_free(cache: Kv4Cache, slots, keep=None, stream=None) -> None:
    """Shortens slots[i] to keep[i] tokens (None: to none) and gives the pages behind them back."""
    dev, s, _, n = _batch(cache, slots, None)
    check(lib().phobos_kv4_free(cache.address, s, _ints(keep, "keep", dev, n), n, _stream(stream, dev)))


def kv4_compact(cache: Kv4Cache, live, workspace=None, stream=None) -> None:
    """Moves the pages in use to ids 0 .. live[0] - 1 in every layer."""
    dev, _, _, _ = _batch(cache, live, None)
    wp, wn = _space(workspace, dev)
    check(lib().phobos_kv4_compact(cache.address, _ints(live, "live", dev, 1), wp, wn, _stream(stream, dev)))
