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
import importlib.util
import sysconfig

from . import (F16, F32, I8, I32, PH_ERR_INVALID, PH_ERR_UNSUPPORTED, LIB_PATH, PhobosError, PhTensor, _stream_ptr, check, lib)


class PhKv4Cache(ctypes.Structure):
    _fields_ = [("pages", ctypes.c_void_p), ("refs", ctypes.c_void_p), ("tables", ctypes.c_void_p), ("lens", ctypes.c_void_p),
                ("layer_pitch", ctypes.c_int64), ("layers", ctypes.c_int32), ("n_pages", ctypes.c_int32),
                ("page_tokens", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("group", ctypes.c_int32), ("max_seqs", ctypes.c_int32), ("table_width", ctypes.c_int32)]


_bind = None           # the CPython module with the short calls (csrc/bind.cpp), loaded at the first call


def _load():
    """Loads csrc/bind.cpp's module and gives it what it calls; raises if it has not been built (no fallback exists)."""
    global _bind
    path = LIB_PATH.parent / ("_bind" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
    if not path.exists():
        raise ImportError(f"{path} is missing: build it with `python phobos-lang_b200/build.py`")
    import torch
    torch.cuda.init()
    spec = importlib.util.spec_from_file_location("_bind", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    L = lib()
    entries = tuple(ctypes.cast(getattr(L, "phobos_" + n), ctypes.c_void_p).value for n in
                    ("gemv_q4", "kv4_append", "kv4_read", "kv4_attention", "kv4_extend", "kv4_fork", "kv4_free", "kv4_compact"))
    # The raw getters cost a tenth of the documented ones, which build a Stream object and check each time that CUDA is up.
    # Where a torch lacks them the documented ones serve.
    device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
    stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
    module.setup(entries, (torch.float16, torch.float32, torch.int8, torch.uint8, torch.int32), PhobosError, device, stream)
    _bind = module
    return module


def _device() -> int:
    import torch
    return torch.cuda.current_device()


def _on_device(t, name: str, device: int) -> None:
    if not t.is_cuda:
        raise PhobosError(PH_ERR_INVALID, f"{name} is not on a CUDA device")
    if t.device.index != device:
        raise PhobosError(PH_ERR_INVALID, f"{name} lives on cuda:{t.device.index} but the current device is cuda:{device}")


def byte_desc(t, name: str = "tensor") -> PhTensor:
    """PhTensor of a rank-1/2 CUDA tensor of any element type these entry points know (no copy)."""
    import torch
    _on_device(t, name, _device())
    codes = {torch.float16: F16, torch.float32: F32, torch.int8: I8, torch.uint8: I8, torch.int32: I32}
    if t.dtype not in codes:
        raise PhobosError(PH_ERR_UNSUPPORTED, f"{name}: element type {t.dtype}")
    if t.dim() not in (1, 2):
        raise PhobosError(PH_ERR_INVALID, f"{name}: rank {t.dim()}, expected 1 or 2")
    d = PhTensor(t.data_ptr(), codes[t.dtype], t.dim())
    for i in range(t.dim()):
        d.sizes[i], d.strides[i] = t.shape[i], t.stride(i)
    return d


# ---- 4-bit weights ----------------------------------------------------------------------------
def q4_packed_bytes(N: int, K: int, group: int) -> int:
    return int(lib().phobos_q4_packed_bytes(N, K, group))


def q4_pack(codes, scales, zeros, group: int, out=None, stream=None):
    """Lays out codes [N, K] (one per byte, 0..15), scales and zeros [N, K/group] (f16; zeros None: 8) for gemv_q4."""
    import torch
    if out is None:
        need = q4_packed_bytes(codes.shape[0], codes.shape[1], group)
        out = torch.empty(need, dtype=torch.int8, device=codes.device)
    c, s, o = byte_desc(codes, "codes"), byte_desc(scales, "scales"), byte_desc(out, "packed")
    z = byte_desc(zeros, "zeros") if zeros is not None else None
    check(lib().phobos_q4_pack(ctypes.byref(c), ctypes.byref(s), ctypes.byref(z) if z is not None else None, group, ctypes.byref(o),
                               _stream_ptr(stream)))
    return out


def gemv_q4(X, packed, Y, group: int, alpha: float = 1.0, beta: float = 0.0, stream=None) -> None:
    """Y[M,N] = alpha * X[M,K] W[N,K]^T + beta * Y, W = scale * (code - zero) in 4 bits; X f16, Y f16 or f32."""
    rc = (_bind or _load()).gemv_q4(X, packed, Y, group, alpha, beta, stream)
    if rc:
        check(rc)


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
        import torch
        for t, name in ((refs, "refs"), (tables, "tables"), (lens, "lens")):
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise PhobosError(PH_ERR_INVALID, f"{name}: expected a contiguous int32 tensor")
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
        self.struct = PhKv4Cache(pages.data_ptr(), refs.data_ptr(), tables.data_ptr(), lens.data_ptr(), pitch,
                                 pages.shape[0], pages.shape[1], page_tokens, kv_heads, head_dim, group, tables.shape[0],
                                 tables.shape[1])
        self.address = ctypes.addressof(self.struct)
        self.handle = (self.address, dev)      # for csrc/bind.cpp

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


def kv4_append(cache: Kv4Cache, layer: int, K, V, slots, indptr=None, stream=None) -> None:
    """Quantises rows K, V [T, kv_heads * head_dim] into the places of the sequences' last tokens (see kv4_extend)."""
    rc = (_bind or _load()).rows(0, cache.handle, layer, K, V, slots, indptr, stream)
    if rc:
        check(rc)


def kv4_read(cache: Kv4Cache, layer: int, K, V, slots, indptr=None, stream=None) -> None:
    """The values of the sequences' last tokens into rows K, V: the inverse of kv4_append."""
    rc = (_bind or _load()).rows(1, cache.handle, layer, K, V, slots, indptr, stream)
    if rc:
        check(rc)


def kv4_attention_workspace_bytes(cache: Kv4Cache, T: int, n: int, q_heads: int) -> int:
    return int(lib().phobos_kv4_attention_workspace_bytes(cache.address, T, n, q_heads))


def kv4_attention(cache: Kv4Cache, layer: int, Q, O, scale: float, slots, indptr=None, lse=None, window: int = 0, workspace=None,
                  stream=None) -> None:
    """O = softmax(scale q K^T) V over the cache; Q, O [T, q_heads * head_dim] f16.  The row of position p sees tokens
    j <= p (window > 0: only j > p - window); one that sees nothing gets zeros and lse -inf."""
    rc = (_bind or _load()).attention(cache.handle, layer, Q, O, lse, scale, window, slots, indptr, workspace, stream)
    if rc:
        check(rc)


def kv4_pages_workspace_bytes(cache: Kv4Cache) -> int:
    return int(lib().phobos_kv4_pages_workspace_bytes(cache.address))


def kv4_extend(cache: Kv4Cache, slots, counts, shortfall, workspace=None, stream=None) -> None:
    """Room for counts[i] more tokens of slots[i], and the new lengths.  shortfall (int32 [1], device): 0 done, > 0 pages
    missing, -1 a wrong request; unless it is 0 nothing has changed and the rows must not be appended."""
    rc = (_bind or _load()).extend(cache.handle, slots, counts, shortfall, workspace, stream)
    if rc:
        check(rc)


def kv4_fork(cache: Kv4Cache, src, dst, shortfall, deep: bool = False, workspace=None, stream=None) -> None:
    """The empty sequences dst[i] continue from src[i], sharing its pages, or (deep) with copies of them."""
    rc = (_bind or _load()).fork(cache.handle, src, dst, int(deep), shortfall, workspace, stream)
    if rc:
        check(rc)


def kv4_free(cache: Kv4Cache, slots, keep=None, stream=None) -> None:
    """Shortens slots[i] to keep[i] tokens (None: to none) and gives the pages behind them back."""
    rc = (_bind or _load()).free(cache.handle, slots, keep, stream)
    if rc:
        check(rc)


def kv4_compact(cache: Kv4Cache, live, workspace=None, stream=None) -> None:
    """Moves the pages in use to ids 0 .. live[0] - 1 in every layer."""
    rc = (_bind or _load()).compact(cache.handle, live, workspace, stream)
    if rc:
        check(rc)
