"""Argument checks of the 4-bit entry points without a GPU: a bad call is refused before any device is asked for, a good
one only for want of a device (PH_ERR_DEVICE) on a machine that has none."""
import ctypes

import pytest


def desc(ph, dtype, *sizes, strides=None, ptr=0x10000, offset=0):
    d = ph.PhTensor(ptr, dtype, len(sizes))
    for i, n in enumerate(sizes):
        d.sizes[i] = n
    d.strides[0], d.strides[1] = strides or ((sizes[1], 1) if len(sizes) == 2 else (1, 0))
    d.offset = offset
    return ctypes.byref(d), d


def cache(ph, **over):
    from phobos_lang_b200.serve import PhKv4Cache
    v = dict(pages=0x20000, refs=0x30000, tables=0x40000, lens=0x50000, layer_pitch=1 << 20, layers=2, n_pages=8, page_tokens=16, kv_heads=2,
             head_dim=64, group=64, max_seqs=4, table_width=8)
    return PhKv4Cache(**(v | over))


def refused(ph, rc, code):
    assert rc == code, (rc, ph.last_error())
    assert ph.last_error()


def test_sizes(ph):
    assert ph.q4_packed_bytes(16, 128, 128) == 1024 + 64
    assert ph.q4_packed_bytes(17, 160, 32) == 2 * 2 * (1024 + 256)
    assert ph.q4_packed_bytes(1, 64, 64) == 1024 + 128
    for bad in ((0, 128, 128), (16, 0, 32), (16, 100, 32), (16, 128, 48), (-1, 128, 64), (1 << 40, 128, 64)):
        assert ph.q4_packed_bytes(*bad) == 0
    # 16 tokens of one head: codes of K and V, and a pair of f16 for each group of each
    assert ph.kv4_page_bytes(1, 128, 128, 16) == 16 * 128 + 128
    assert ph.kv4_page_bytes(8, 64, 32, 64) == 8 * 4 * (16 * 64 + 256)
    for bad in ((0, 128, 128, 16), (1, 96, 32, 16), (1, 64, 128, 16), (1, 64, 64, 24), (1, 64, 64, 8), (1, 64, 64, 512)):
        assert ph.kv4_page_bytes(*bad) == 0


def test_gemv_q4_refusals(ph):
    L, code = ph.lib(), ph.PH_ERR_INVALID
    x, xd = desc(ph, ph.F16, 4, 256)
    w, wd = desc(ph, ph.I8, ph.q4_packed_bytes(40, 256, 64))
    y, yd = desc(ph, ph.F32, 4, 40)
    call = lambda x=x, w=w, y=y, g=64: L.phobos_gemv_q4(x, w, y, 1.0, 0.0, g, None)  # noqa: E731
    keep = []

    def d(*a, **k):
        r = desc(ph, *a, **k)
        keep.append(r)
        return r[0]

    refused(ph, call(x=None), code)
    refused(ph, call(w=None), code)
    refused(ph, call(x=d(ph.F32, 4, 256)), ph.PH_ERR_UNSUPPORTED)
    refused(ph, call(y=d(ph.I32, 4, 40)), ph.PH_ERR_UNSUPPORTED)
    refused(ph, call(g=16), ph.PH_ERR_UNSUPPORTED)
    refused(ph, call(x=d(ph.F16, 4, 248)), ph.PH_ERR_UNSUPPORTED)
    refused(ph, call(y=d(ph.F32, 5, 40)), code)
    refused(ph, call(y=d(ph.F32, 4, 49)), code)                                # more rows of W than were packed
    refused(ph, call(y=d(ph.F32, 4, 40, strides=(39, 1))), code)
    refused(ph, call(y=d(ph.F32, 4, 40, strides=(1, 4))), code)
    refused(ph, call(y=d(ph.F32, 4, 40, ptr=0x10002)), code)
    refused(ph, call(x=d(ph.F16, 4, 256, strides=(260, 1))), code)
    refused(ph, call(x=d(ph.F16, 4, 256, ptr=0x10008)), code)
    refused(ph, call(x=d(ph.F16, 4, 256, offset=-8)), code)
    refused(ph, call(x=d(ph.F16, 4, 256, ptr=0)), code)
    refused(ph, call(w=d(ph.I8, ph.q4_packed_bytes(40, 256, 64), ptr=0x10004)), code)
    refused(ph, call(w=d(ph.F16, ph.q4_packed_bytes(40, 256, 64))), code)
    c, cd = desc(ph, ph.I8, 40, 256)
    s, sd = desc(ph, ph.F16, 40, 4)
    pack = lambda c=c, s=s, z=None, g=64, w=w: L.phobos_q4_pack(c, s, z, g, w, None)  # noqa: E731
    refused(ph, pack(s=d(ph.F16, 40, 5)), code)
    refused(ph, pack(s=d(ph.F32, 40, 4)), ph.PH_ERR_UNSUPPORTED)
    refused(ph, pack(z=d(ph.F16, 39, 4)), code)
    refused(ph, pack(c=d(ph.I32, 40, 256)), code)
    refused(ph, pack(g=100), ph.PH_ERR_UNSUPPORTED)
    refused(ph, pack(w=d(ph.I8, 1000)), code)


def test_cache_refusals(ph):
    L = ph.lib()
    one = ctypes.c_void_p(0x60000)
    ws = ctypes.c_void_p(0x70000)

    def free(c, n=1, slots=one):
        return L.phobos_kv4_free(ctypes.byref(c) if c is not None else None, slots, None, n, None)

    refused(ph, free(None), ph.PH_ERR_INVALID)
    for bad in (dict(head_dim=96), dict(group=48), dict(group=128), dict(page_tokens=20), dict(kv_heads=0), dict(table_width=1 << 21),
                dict(table_width=1 << 20, page_tokens=16, max_seqs=1, n_pages=8, layers=1, head_dim=32)):
        refused(ph, free(cache(ph, **bad)), ph.PH_ERR_UNSUPPORTED)
    for bad in (dict(pages=0), dict(refs=0), dict(tables=0), dict(lens=0), dict(layers=0), dict(n_pages=0), dict(max_seqs=0), dict(table_width=0),
                dict(pages=0x20008), dict(lens=0x50002), dict(layer_pitch=8), dict(layer_pitch=(1 << 20) + 8), dict(layer_pitch=-(1 << 20))):
        refused(ph, free(cache(ph, **bad)), ph.PH_ERR_INVALID)
    refused(ph, free(cache(ph), n=-1), ph.PH_ERR_INVALID)
    refused(ph, free(cache(ph), slots=None), ph.PH_ERR_INVALID)
    c = ctypes.byref(cache(ph))
    need = L.phobos_kv4_pages_workspace_bytes(c)
    assert need > 0 and L.phobos_kv4_pages_workspace_bytes(ctypes.byref(cache(ph, group=7))) == 0
    refused(ph, L.phobos_kv4_extend(c, one, one, 5, one, ws, need, None), ph.PH_ERR_INVALID)          # more rows than sequences
    refused(ph, L.phobos_kv4_extend(c, one, None, 1, one, ws, need, None), ph.PH_ERR_INVALID)
    refused(ph, L.phobos_kv4_extend(c, one, one, 1, None, ws, need, None), ph.PH_ERR_INVALID)
    refused(ph, L.phobos_kv4_extend(c, one, one, 1, one, ws, need - 1, None), ph.PH_ERR_WORKSPACE)
    refused(ph, L.phobos_kv4_extend(c, one, one, 1, one, None, need, None), ph.PH_ERR_WORKSPACE)
    refused(ph, L.phobos_kv4_fork(c, one, one, 1, 0, one, ctypes.c_void_p(0x70010), need, None), ph.PH_ERR_WORKSPACE)
    refused(ph, L.phobos_kv4_fork(c, one, None, 1, 1, one, ws, need, None), ph.PH_ERR_INVALID)
    refused(ph, L.phobos_kv4_compact(c, None, ws, need, None), ph.PH_ERR_INVALID)


def test_attention_and_row_refusals(ph):
    L = ph.lib()
    c = ctypes.byref(cache(ph))
    one, ws = ctypes.c_void_p(0x60000), ctypes.c_void_p(0x70000)
    keep = []

    def d(*a, **k):
        r = desc(ph, *a, **k)
        keep.append(r)
        return r[0]

    q, lse = d(ph.F16, 3, 256), d(ph.F32, 3, 4)
    need = L.phobos_kv4_attention_workspace_bytes(c, 3, 3, 4)
    assert need > 0 and L.phobos_kv4_attention_workspace_bytes(c, 3, 3, 3) == 0 and L.phobos_kv4_attention_workspace_bytes(c, -1, 3, 4) == 0
    att = lambda layer=0, q=q, o=q, l=lse, window=0, slots=one, ind=None, n=3, ws=ws, have=need: L.phobos_kv4_attention(  # noqa: E731
        c, layer, q, o, l, 0.1, window, slots, ind, n, ws, have, None)
    for bad in (dict(layer=2), dict(layer=-1), dict(q=None), dict(o=d(ph.F16, 2, 256)), dict(q=d(ph.F16, 3, 192), o=d(ph.F16, 3, 192)), dict(window=-1),
                dict(l=d(ph.F32, 3, 5)), dict(slots=None), dict(n=-1), dict(n=4), dict(q=d(ph.F16, 3, 256, strides=(257, 1))),
                dict(q=d(ph.F16, 256)), dict(slots=ctypes.c_void_p(0x60001))):
        refused(ph, att(**bad), ph.PH_ERR_INVALID)
    refused(ph, att(q=d(ph.F32, 3, 256)), ph.PH_ERR_UNSUPPORTED)
    refused(ph, att(l=d(ph.F16, 3, 4)), ph.PH_ERR_UNSUPPORTED)
    for bad in (dict(have=need - 1), dict(ws=None), dict(ws=ctypes.c_void_p(0x70080))):
        refused(ph, att(**bad), ph.PH_ERR_WORKSPACE)
    k = d(ph.F16, 3, 128)
    for f in (L.phobos_kv4_append, L.phobos_kv4_read):
        for bad in ((c, 5, k, k, one, None, 3), (c, 0, k, d(ph.F16, 3, 64), one, None, 3), (c, 0, k, d(ph.F16, 2, 128), one, None, 2), (c, 0, k, None, one, None, 3),
                    (c, 0, k, k, None, None, 3), (c, 0, k, k, one, None, 4), (None, 0, k, k, one, None, 3)):
            refused(ph, f(*bad, None), ph.PH_ERR_INVALID)
        refused(ph, f(c, 0, d(ph.F32, 3, 128), d(ph.F32, 3, 128), one, None, 3, None), ph.PH_ERR_UNSUPPORTED)


def test_good_calls_need_a_device(ph):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is here")
    x, xd = desc(ph, ph.F16, 4, 256)
    w, wd = desc(ph, ph.I8, ph.q4_packed_bytes(40, 256, 64))
    y, yd = desc(ph, ph.F32, 4, 40)
    refused(ph, ph.lib().phobos_gemv_q4(x, w, y, 1.0, 0.0, 64, None), ph.PH_ERR_DEVICE)
    c = ctypes.byref(cache(ph))
    refused(ph, ph.lib().phobos_kv4_free(c, ctypes.c_void_p(0x60000), None, 1, None), ph.PH_ERR_DEVICE)


def test_launch_by_name_needs_the_group(ph):
    x, xd = desc(ph, ph.F16, 4, 256)
    t = (ph.PhTensor * 3)(xd, desc(ph, ph.I8, ph.q4_packed_bytes(40, 256, 64))[1], desc(ph, ph.F32, 4, 40)[1])
    s = (ph.PhScalar * 2)(ph.scalar_f32(3, 1.0), ph.scalar_f32(4, 0.0))
    g = (ctypes.c_uint32 * 3)(1, 1, 1)
    refused(ph, ph.lib().phobos_launch(b"gemv_q4", t, 3, s, 2, g, g, -1, None, 0, None), ph.PH_ERR_INVALID)
    refused(ph, ph.lib().phobos_launch(b"gemv_q4", t, 2, s, 2, g, g, -1, None, 0, None), ph.PH_ERR_INVALID)


def test_the_short_calls_module_names_its_interpreter_and_is_left_out_without_headers(ph, tmp_path, capfd, monkeypatch):
    """The C library's build asks for no Python; the CPython module carries the interpreter's suffix, so that another
    interpreter does not load it, and without headers the library is all that is built."""
    import sysconfig

    import __graft_entry__ as entry
    build = entry._load_build_module()
    assert build.BIND.name == "_bind" + sysconfig.get_config_var("EXT_SUFFIX") != "_bind.so"
    assert build.build_bind(tmp_path / "x.so", headers=str(tmp_path)) is None
    assert "Python.h" in capfd.readouterr().err and not list(tmp_path.iterdir())
    # a build asks for the module apart from the library, and ends well without it
    monkeypatch.setattr(build, "BIND", tmp_path / "y.so")
    calls = []
    monkeypatch.setattr(build, "_build_lib", lambda *a: None)
    monkeypatch.setattr(build, "build_bind", lambda: calls.append(1))
    assert build.build() == build.LIB and calls == [1]
    # the calls then say what is missing
    from phobos_lang_b200 import serve
    monkeypatch.setattr(serve, "_bind", None)
    monkeypatch.setattr(serve, "LIB_PATH", tmp_path / "libphobos_leaf.so")
    with pytest.raises(ImportError, match="_bind"):
        serve.gemv_q4(None, None, None, 64)


SLEEPER = """
import ctypes, importlib.util, sys, threading, time
spec = importlib.util.spec_from_file_location("_bind", sys.argv[1])
bind = importlib.util.module_from_spec(spec)
spec.loader.exec_module(bind)

class Ints:                                # what the module asks of an int32 tensor
    dtype = "i32"
    get_device = lambda self: 0
    is_contiguous = lambda self: True
    numel = lambda self: 4
    data_ptr = lambda self: 4096
    element_size = lambda self: 4

usleep = ctypes.cast(ctypes.CDLL(None).usleep, ctypes.c_void_p).value
bind.setup((usleep,) * 8, ("f16", "f32", "i8", "u8", Ints.dtype), RuntimeError, lambda: 0, lambda d: 0)
ticks, stop = [], threading.Event()

def tick():
    while not stop.is_set():
        ticks.append(time.monotonic())
        time.sleep(0.001)

other = threading.Thread(target=tick)
other.start()
cache = (500000, 0)                        # the entry point's first argument: half a second
for call in (lambda: bind.free(cache, Ints(), None, None), lambda: bind.compact(cache, Ints(), None, None), lambda: bind.extend(cache, Ints(), Ints(), Ints(), None, None),
             lambda: bind.fork(cache, Ints(), Ints(), 0, Ints(), None, None)):
    t0 = time.monotonic()
    assert call() == 0
    t1 = time.monotonic()
    assert t1 - t0 >= 0.4, t1 - t0
    print(sum(t0 + 0.1 < t < t1 - 0.1 for t in list(ticks)))
stop.set()
other.join()
# two threads' calls are made one after another
t0 = time.monotonic()
both = [threading.Thread(target=lambda: bind.free(cache, Ints(), None, None)) for _ in range(2)]
for t in both:
    t.start()
for t in both:
    t.join()
assert time.monotonic() - t0 >= 0.9
"""


def test_other_threads_run_while_a_call_waits(ph):
    """An entry point that takes its time (here: usleep in their place) does not hold the interpreter's lock: a launch may
    wait for a host function that needs it.  Two threads' calls still do not mix their launches."""
    import subprocess
    import sys

    import __graft_entry__ as entry
    bind = entry._load_build_module().BIND
    r = subprocess.run([sys.executable, "-c", SLEEPER, str(bind)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    counts = [int(x) for x in r.stdout.split()]
    assert len(counts) == 4 and all(c > 0 for c in counts), counts


WORKSPACES = """
import importlib.util, sys
spec = importlib.util.spec_from_file_location("_bind", sys.argv[1])
bind = importlib.util.module_from_spec(spec)
spec.loader.exec_module(bind)
import torch

class Device:                              # a tensor in host memory that says it is on device 0
    def __init__(self, t):
        self.t, self.dtype = t, t.dtype

    def __getattr__(self, name):
        return (lambda: 0) if name == "get_device" else getattr(self.t, name)

class Refused(Exception):
    pass

import ctypes
called = []
entry = ctypes.CFUNCTYPE(ctypes.c_int, *[ctypes.c_void_p] * 5)(lambda cache, live, ws, n, stream: called.append(n) or 0)
bind.setup((ctypes.cast(entry, ctypes.c_void_p).value,) * 8, (torch.float16, torch.float32, torch.int8, torch.uint8, torch.int32), Refused, lambda: 0, lambda d: 0)
live = Device(torch.zeros(1, dtype=torch.int32))
space = torch.zeros(64, dtype=torch.uint8)
assert bind.compact((4096, 0), live, Device(space), None) == 0 and called == [64]
for view in (space[:1].expand(1 << 20), space.view(8, 8).t(), space[::2]):
    try:
        bind.compact((4096, 0), live, Device(view), None)
    except Refused as e:
        assert "workspace" in str(e)
    else:
        raise SystemExit(f"taken: {view.stride()}, {called}")
"""


def test_a_workspace_is_contiguous(ph):
    """A view that repeats its elements has fewer bytes behind its address than elements: not a workspace."""
    import subprocess
    import sys

    import __graft_entry__ as entry
    r = subprocess.run([sys.executable, "-c", WORKSPACES, str(entry._load_build_module().BIND)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
