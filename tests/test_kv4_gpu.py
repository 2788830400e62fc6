"""The 4-bit cache and the attention that reads it, on a B200, against the definition in 64 bits.

Tolerances.  Values: zero + scale * code is one f32 sum rounded to f16: half an f16 step of the value.
Attention: scores are f32 sums of exact products; with A = scale * sum |q| (|zero| + step * code) their error is at
most A * 2^-17 (D / 16 matrix steps cut to f32, the running sums, the change to powers of two), which is the relative
error of a weight and, with |lse| 2^-22, the error of lse.  A weight times a step is rounded to f16 once, 2^-11 of it
(2^-12 and less only where it is subnormal: below 2^-28 of the largest, counted as 2^-30 a token), and O to f16 once,
2^-11 of it, or 2^-25."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def quantise(x, G):
    """f64 definition on f16 rows [..., D]: scale, zero (f16) and codes."""
    import torch
    g = x.double().unflatten(-1, (-1, G))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / 15).half()
    s = scale.double()[..., None]
    code = torch.where(s > 0, ((g - lo[..., None]) / s.clamp_min(1e-30)).round().clamp(0, 15), torch.zeros_like(g))
    return scale, lo.half(), code


def value(x, G):
    scale, zero, code = quantise(x, G)
    return (zero.double()[..., None] + scale.double()[..., None] * code).flatten(-2)


class Setup:
    """A cache filled through the public calls, and the f64 values of every token that was appended."""

    def __init__(self, ph, dev, lens, Hkv, D, G, page, layers=1, extra_slots=2, spare=3, seed=0, order=None):
        import torch
        self.ph, self.dev, self.Hkv, self.D, self.G = ph, dev, Hkv, D, G
        n = len(lens)
        width = max(1, -(-max(lens + [1]) // page)) + 1
        pages = sum(-(-l // page) for l in lens) + spare
        self.cache = ph.Kv4Cache.create(layers, pages, Hkv, D, G, page, n + extra_slots, width)
        self.cache.pages.fill_(0xFF)          # what a page holds before it is written: f16 NaN everywhere
        self.ws = torch.empty(max(256, ph.kv4_pages_workspace_bytes(self.cache)), dtype=torch.uint8, device=dev)
        self.short = torch.full((1,), 77, dtype=torch.int32, device=dev)
        g = torch.Generator().manual_seed(seed)
        self.slots = torch.randperm(n + extra_slots, generator=g)[:n].to(dev, torch.int32)
        ph.kv4_extend(self.cache, self.slots, torch.tensor(lens, dtype=torch.int32, device=dev), self.short, workspace=self.ws)
        assert int(self.short) == 0
        T = sum(lens)
        self.lens = lens
        self.k = (torch.randn(T, Hkv * D, generator=g) * torch.exp(torch.randn(Hkv * D, generator=g) * 0.5)).half().to(dev)
        self.v = (torch.randn(T, Hkv * D, generator=g) + 0.3).half().to(dev)
        ind = [0]
        for l in lens:
            ind.append(ind[-1] + l)
        self.ind = ind
        for layer in range(layers):
            if T:
                ph.kv4_append(self.cache, layer, self.k, self.v, self.slots, torch.tensor(ind, dtype=torch.int32, device=dev))

    def kv(self, b):
        a, z = self.ind[b], self.ind[b + 1]
        f = lambda x: x[a:z].unflatten(1, (self.Hkv, self.D))  # noqa: E731
        return f(self.k), f(self.v)


def reference(setup, q, ind, rep, scale, window):
    """(o, lse, tolerance of o, tolerance of lse) in f64 for rows q [T, Hq * D]."""
    import torch
    H, D, G, dev = setup.Hkv, setup.D, setup.G, setup.dev
    T = q.shape[0]
    o = torch.zeros(T, H * rep, D, dtype=torch.float64, device=dev)
    lse = torch.full((T, H * rep), -math.inf, dtype=torch.float64, device=dev)
    to, tl = torch.zeros_like(o), torch.zeros_like(lse)
    for b, length in enumerate(setup.lens):
        a, z = ind[b], ind[b + 1]
        if a == z:
            continue
        kx, vx = setup.kv(b)
        ks, kz, kc = quantise(kx, G)
        vs, vz, vc = quantise(vx, G)
        spread = lambda s: s.double()[..., None].expand(*s.shape, G)  # noqa: E731
        k, v = (spread(kz) + spread(ks) * kc).flatten(-2), (spread(vz) + spread(vs) * vc).flatten(-2)
        ka, va = (spread(kz).abs() + spread(ks) * kc).flatten(-2), (spread(vs) * vc).flatten(-2)
        qq = q[a:z].double().view(z - a, H, rep, D)
        pos = torch.arange(length - (z - a), length, device=dev)
        tok = torch.arange(length, device=dev)
        see = tok[None] <= pos[:, None]
        if window:
            see &= tok[None] > pos[:, None] - window
        x = torch.einsum("ihrd,jhd->ihrj", qq, k) * scale
        A = torch.einsum("ihrd,jhd->ihrj", qq.abs(), ka) * abs(scale)
        x = x.masked_fill(~see[:, None, None], -math.inf)
        some = see.any(1)[:, None, None]
        m = x.amax(-1, keepdim=True) if length else x.sum(-1, keepdim=True)
        p = torch.exp(x - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
        l = p.sum(-1, keepdim=True)
        w = p / torch.where(l > 0, l, torch.ones_like(l))
        o[a:z] = torch.einsum("ihrj,jhd->ihrd", w, v).flatten(1, 2)
        lse[a:z] = torch.where(some, (m + l.log())[..., 0], torch.full_like(l[..., 0], -math.inf)).flatten(1, 2)
        e = (A * see[:, None, None]).amax(-1, keepdim=True) * 2.0 ** -17 + 2.0 ** -20 if length else 0 * l
        full = (v.abs() + va)
        to[a:z] = (2 * e * torch.einsum("ihrj,jhd->ihrd", w, full) + 2.0 ** -11 * torch.einsum("ihrj,jhd->ihrd", w, va)
                   + (2.0 ** -30 * va.amax(0)[None, :, None] * see.sum(1)[:, None, None, None] / l.clamp_min(1) if length else 0)).flatten(1, 2)
        tl[a:z] = (e[..., 0] + 2.0 ** -22 * lse[a:z].view(z - a, H, rep).abs().nan_to_num(0, 0, 0)).flatten(1, 2)
    to += 2.0 ** -11 * (o.abs() + to) + 2.0 ** -25
    return o.flatten(1), lse, to.flatten(1), tl


def attend(setup, q, ind, scale, window=0, layer=0, slots=None, o=None, stream=None):
    import torch
    ph, T = setup.ph, q.shape[0]
    Hq = q.shape[1] // setup.D
    o = torch.full_like(q, 7.0) if o is None else o
    lse = torch.full((T, Hq), 7.0, device=setup.dev)
    slots = setup.slots if slots is None else slots
    ws = torch.full((max(256, ph.kv4_attention_workspace_bytes(setup.cache, T, slots.numel(), Hq)),), 0xFF, dtype=torch.uint8, device=setup.dev)
    i = None if ind is None else torch.tensor(ind, dtype=torch.int32, device=setup.dev)
    ph.kv4_attention(setup.cache, layer, q, o, scale, slots, i, lse=lse, window=window, workspace=ws, stream=stream)
    return o, lse


def check(setup, new, rep, window=0, scale=None, seed=1, mult=1.0):
    import torch
    ind = [0]
    for x in new:
        ind.append(ind[-1] + x)
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(ind[-1] + 3, setup.Hkv * rep * setup.D, generator=g) * mult).half().to(setup.dev)
    scale = 1.0 / math.sqrt(setup.D) if scale is None else scale
    o, lse = attend(setup, q, ind, scale, window)
    assert setup.ph.device_status() == 0
    T = ind[-1]
    assert bool((o[T:] == 7.0).all()) and bool((lse[T:] == 7.0).all()), "rows behind the last sequence were written"
    wo, wl, to, tl = reference(setup, q, ind, rep, scale, window)
    gone = torch.isinf(wl[:T])
    assert torch.equal(torch.isinf(lse[:T]), gone)
    assert bool(((lse[:T].double() - wl[:T]).abs()[~gone] <= tl[:T][~gone]).all()), float((lse[:T].double() - wl[:T]).abs()[~gone].max())
    bad = (o[:T].double() - wo[:T]).abs() > to[:T]
    assert not bool(bad.any()), (int(bad.sum()), float(((o[:T].double() - wo[:T]).abs() / to[:T]).max()))
    assert bool((o[:T].view(T, -1, setup.D)[gone] == 0).all())
    return q, o, lse


LAYOUTS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)]


@pytest.mark.parametrize("D,G", LAYOUTS)
@pytest.mark.parametrize("page", [16, 64])
def test_append_then_read_gives_the_quantised_values(ph, dev, D, G, page):
    import torch
    s = Setup(ph, dev, [1, 50, 0, 129, 16], 3, D, G, page, layers=2, seed=D + G)
    T = s.k.shape[0]
    ind = torch.tensor(s.ind, dtype=torch.int32, device=dev)
    for layer in range(2):
        k, v = torch.full_like(s.k, 9.0), torch.full_like(s.v, 9.0)
        ph.kv4_read(s.cache, layer, k, v, s.slots, ind)
        for got, x in ((k, s.k), (v, s.v)):
            want = value(x.unflatten(1, (3, D)), G).flatten(1)
            assert bool(((got.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -24 * 2 + 2.0 ** -24 * want.abs()).all())
    assert ph.device_status() == 0 and T == s.ind[-1]


def test_many_rows_at_once(ph, dev):
    """Enough rows that whole units go through shared memory; ends of sequences that do not end a unit among them."""
    import torch
    for D, G in ((128, 32), (64, 64)):
        s = Setup(ph, dev, [3000, 1, 1200, 17], 3, D, G, 64, seed=G)
        ind = torch.tensor(s.ind, dtype=torch.int32, device=dev)
        k, v = torch.full_like(s.k, 9.0), torch.full_like(s.v, 9.0)
        ph.kv4_read(s.cache, 0, k, v, s.slots, ind)
        for got, x in ((k, s.k), (v, s.v)):
            want = value(x.unflatten(1, (3, D)), G).flatten(1)
            assert bool(((got.double() - want).abs() <= 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -23).all())
        small = torch.empty_like(s.k[:17]), torch.empty_like(s.v[:17])
        ph.kv4_read(s.cache, 0, *small, s.slots[3:], torch.tensor([0, 17], dtype=torch.int32, device=dev))
        assert torch.equal(small[0], k[-17:]) and torch.equal(small[1], v[-17:])
        check(s, [1, 1, 1, 1], 2)
    assert ph.device_status() == 0


@pytest.mark.parametrize("D,G", [(64, 32), (128, 128)])
def test_page_layout_is_the_documented_one(ph, dev, D, G):
    """The unit layout at the top of csrc/kv4.cuh, byte by byte; bytes of tokens that were not written stay."""
    import torch
    H, page, n = 2, 32, 27
    s = Setup(ph, dev, [n], H, D, G, page, extra_slots=0, spare=0)
    unit = 16 * D + 128 * (D // G)
    want = np.full((H, page // 16, unit), 0xFF, dtype=np.uint8)
    ng, W = D // G, D // 8
    for which, x in enumerate(s.kv(0)):
        scale, zero, code = (a.cpu().numpy() for a in quantise(x, G))
        code = code.reshape(n, H, D).astype(np.uint8)
        for j in range(n):
            for h in range(H):
                u, r = want[h, j // 16], j % 16
                for d in range(D):
                    if which == 0:
                        w, i = d // 8, d % 8
                        at, sh = (r >> 3) * 4 * D + ((r & 7) * 4 + w % 4) * W + w // 4 * 4 + i // 2, 4 * (i % 2)
                    else:
                        p, g, i = d // 32, d % 32 // 4, d % 4
                        at, sh = 8 * D + (r >> 3) * 4 * D + (4 * g + (r & 7) // 2) * W + 4 * p + 2 * (r & 1) + i // 2, 4 * (i % 2)
                    u[at] = (u[at] & (0xF0 if sh == 0 else 0x0F)) | (code[j, h, d] << sh)
                for q in range(ng):
                    at = 16 * D + which * 64 * ng + (r * ng + q) * 4
                    u[at:at + 4] = np.array([scale[j, h, q], zero[j, h, q]], dtype=np.float16).view(np.uint8)
    got = s.cache.pages[0, int(s.cache.tables[int(s.slots[0]), 0])].cpu().numpy().reshape(H, page // 16, unit)
    assert np.array_equal(got, want)


def test_quantising_special_groups(ph, dev):
    """Equal values, a range too small for a scale, f16's whole range, and values that are not finite."""
    import torch
    D, G = 64, 32
    s = Setup(ph, dev, [6], 1, D, G, 16)
    x = torch.randn(6, D, device=dev).half()
    x[0] = 3.25
    x[1, :G] = 1e-7
    x[1, 3] = 1.8e-7
    x[2, 0], x[2, 1] = 65504.0, -65504.0
    x[3, 5] = float("nan")
    x[4, 40] = float("inf")
    k, v = torch.empty_like(x), torch.empty_like(x)
    ph.kv4_append(s.cache, 0, x, x, s.slots, torch.tensor([0, 6], dtype=torch.int32, device=dev))
    ph.kv4_read(s.cache, 0, k, v, s.slots, torch.tensor([0, 6], dtype=torch.int32, device=dev))
    assert torch.equal(k.nan_to_num(5.0), v.nan_to_num(5.0))
    assert bool((k[0] == 3.25).all())
    assert bool((k[1, :G] == x[1, :G].min()).all())
    ok = torch.isfinite(x.unflatten(1, (-1, G))).all(-1).repeat_interleave(G, 1)
    assert torch.equal(torch.isnan(k), ~ok)
    want = value(torch.where(ok, x, torch.zeros_like(x)), G)
    assert bool(((k.double() - want).abs() <= 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -23)[ok].all())


@pytest.mark.parametrize("D,G", LAYOUTS)
@pytest.mark.parametrize("rep,page,lens", [(1, 16, [1, 15, 16, 17]), (4, 32, [100, 1, 63, 64, 65]), (8, 64, [300, 257]), (16, 128, [777]), (3, 16, [40, 2])])
def test_decode_rows(ph, dev, D, G, rep, page, lens):
    s = Setup(ph, dev, lens, 2, D, G, page, seed=rep)
    check(s, [1] * len(lens), rep)
    check(s, [1] * len(lens), rep, window=20, seed=2)


@pytest.mark.parametrize("D,G,rep,page", [(128, 128, 4, 16), (64, 32, 1, 64), (128, 32, 7, 128), (64, 64, 16, 32)])
def test_chunks_of_queries(ph, dev, D, G, rep, page):
    """Several query tokens a sequence: none, one, a few, as many as the sequence has, and more than it has (rows that
    see nothing)."""
    s = Setup(ph, dev, [70, 33, 200, 5, 130, 1], 2, D, G, page, seed=3)
    check(s, [0, 33, 17, 9, 100, 1], rep)
    check(s, [3, 1, 200, 5, 0, 4], rep, window=1, seed=4)
    check(s, [70, 30, 64, 0, 130, 0], rep, window=50, seed=5)


@pytest.mark.parametrize("D,G,Hkv,rep,lens", [(128, 128, 1, 8, [20000, 3, 7000]), (64, 64, 2, 4, [33000]), (128, 32, 8, 1, [5000, 4999, 1, 2500, 16, 1000, 777, 64, 65]),
                                              (128, 64, 1, 16, [9000, 100]), (64, 64, 1, 1, [120000])])
def test_long_and_uneven_sequences(ph, dev, D, G, Hkv, rep, lens):
    s = Setup(ph, dev, lens, Hkv, D, G, 64, seed=6)
    check(s, [1] * len(lens), rep)
    check(s, [2] + [1] * (len(lens) - 1), rep, mult=6.0, seed=7)      # peaked weights
    check(s, [1] * len(lens), rep, window=3333, seed=8)


def test_empty_sequences_and_batches(ph, dev):
    import torch
    s = Setup(ph, dev, [0, 20, 0], 2, 64, 64, 16)
    check(s, [1, 1, 2], 4)
    q = torch.randn(0, 2 * 64, device=dev).half()
    attend(s, q, [0, 0, 0, 0], 0.1)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    attend(s, torch.randn(2, 128, device=dev).half(), None, 0.1, slots=none)
    assert ph.device_status() == 0


def test_weights_over_a_wide_range_of_steps(ph, dev):
    """Values whose sizes differ by 2^20 between tokens and groups: small ones keep their bits when they come alone, and
    scores that grow along the sequence move the maximum."""
    import torch
    D, G, n = 128, 32, 200
    s = Setup(ph, dev, [n], 1, D, G, 16)
    for case in range(3):
        f = torch.ones(n, 1, device=dev)
        if case == 0:
            f = torch.exp2(torch.linspace(-14, 6, n, device=dev))[:, None]
        elif case == 1:
            f = torch.exp2(torch.linspace(6, -14, n, device=dev))[:, None]
        else:
            f = torch.full((n, 1), 2.0 ** -13, device=dev)
        s.v = (torch.randn(n, D, device=dev) * f).half()
        s.k = (torch.randn(n, D, device=dev) * torch.linspace(0.1, 4, n, device=dev)[:, None]).half()
        ph.kv4_append(s.cache, 0, s.k, s.v, s.slots, torch.tensor([0, n], dtype=torch.int32, device=dev))
        check(s, [n], 2, seed=case)
    check(s, [1], 2, scale=0.0)
    check(s, [3], 2, scale=-0.2)


def test_strides_no_indptr_and_no_lse(ph, dev):
    import torch
    lens = [37, 90, 2]
    s = Setup(ph, dev, lens, 2, 64, 32, 32, layers=3)
    n, w = len(lens), 2 * 4 * 64
    wide = torch.randn(n + 2, w + 40, device=dev).half()
    out = torch.full((n + 2, w + 16), 3.0, device=dev).half()
    q, o = wide[:, 8:8 + w], out[:, 8:8 + w]
    ws = torch.empty(max(256, ph.kv4_attention_workspace_bytes(s.cache, n, n, 8)), dtype=torch.uint8, device=dev)
    ph.kv4_attention(s.cache, 2, q, o, 0.125, s.slots, workspace=ws)
    wo, _, to, _ = reference(s, q[:n], [0, 1, 2, 3], 4, 0.125, 0)
    assert bool(((o[:n].double() - wo).abs() <= to).all())
    assert bool((out[n:] == 3.0).all()) and bool((out[:, :8] == 3.0).all()) and bool((out[:, 8 + w:] == 3.0).all())
    # rows of K and V out of a wider tensor, one token each
    kv = torch.randn(n, 2 * 128 + 8, device=dev).half()
    ph.kv4_append(s.cache, 1, kv[:, :128], kv[:, 128:256], s.slots)
    k, v = torch.empty(n, 128, device=dev).half(), torch.empty(n, 128, device=dev).half()
    ph.kv4_read(s.cache, 1, k, v, s.slots)
    want = value(kv[:, :128].unflatten(1, (2, 64)), 32).flatten(1)
    assert bool(((k.double() - want).abs() <= 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -23).all())


def test_a_nan_is_seen_only_by_rows_that_see_its_token(ph, dev):
    import torch
    n = 40
    s = Setup(ph, dev, [n], 1, 64, 64, 16)
    s.k[30, 3] = float("nan")
    s.v[35, 3] = float("inf")
    ph.kv4_append(s.cache, 0, s.k, s.v, s.slots, torch.tensor([0, n], dtype=torch.int32, device=dev))
    q = torch.randn(n, 128, device=dev).half()
    o, lse = attend(s, q, [0, n], 0.125)
    assert bool(torch.isfinite(o[:30]).all()) and bool(torch.isfinite(lse[:30]).all())
    assert bool(torch.isnan(o[30:]).all()) and bool(torch.isnan(lse[30:]).all())
    o, lse = attend(s, q, [0, n], 0.125, window=4)
    assert bool(torch.isfinite(o[:30]).all()) and bool(torch.isnan(lse[30:34]).all()) and bool(torch.isfinite(o[39:]).all())


def test_bad_slots_and_pages_are_not_followed(ph, dev):
    import torch
    lens = [60, 50, 40]
    s = Setup(ph, dev, lens, 2, 64, 64, 16)
    q = torch.randn(3, 4 * 64, device=dev).half()
    # (where sequences are cut depends on the batch, so a batch with another length in it agrees to rounding)
    want, _, tol, _ = reference(s, q, [0, 1, 2, 3], 2, 0.125, 0)
    near = lambda o, rows: bool(((o[rows].double() - want[rows]).abs() <= tol[rows]).all())  # noqa: E731
    assert near(attend(s, q, [0, 1, 2, 3], 0.125)[0], [0, 1, 2])
    assert ph.device_status() == 0
    for bad in (-1, 5, 2 ** 31 - 1):
        slots = s.slots.clone()
        slots[1] = bad
        o, lse = attend(s, q, [0, 1, 2, 3], 0.125, slots=slots)
        with pytest.raises(ph.PhobosError) as e:
            ph.device_status()
        assert e.value.code == ph.PH_ERR_INVALID
        assert near(o, [0, 2]) and bool((o[1] == 0).all()) and bool(torch.isinf(lse[1]).all())
        assert ph.device_status() == 0
    pages = s.cache.pages.clone()
    for bad in (-1, s.cache.refs.numel(), 2 ** 31 - 1):
        old = s.cache.tables[s.slots[0].long(), 1].clone()
        s.cache.tables[s.slots[0].long(), 1] = bad
        o, _ = attend(s, q, [0, 1, 2, 3], 0.125)
        with pytest.raises(ph.PhobosError):
            ph.device_status()
        assert near(o, [1, 2]) and bool(torch.isfinite(o[0]).all())
        keep = torch.tensor([0, 40], dtype=torch.int32, device=dev)
        kv = torch.randn(40, 128, device=dev).half()
        ph.kv4_append(s.cache, 0, kv, kv, s.slots[:1], keep)       # tokens 20..59: the ones of the bad page are left out
        with pytest.raises(ph.PhobosError):
            ph.device_status()
        k, v = torch.full_like(kv, 9.0), torch.full_like(kv, 9.0)
        ph.kv4_read(s.cache, 0, k, v, s.slots[:1], keep)
        with pytest.raises(ph.PhobosError):
            ph.device_status()
        assert bool((k[:12] == 0).all()) and bool(torch.isfinite(k).all())
        s.cache.tables[s.slots[0].long(), 1] = old
        s.cache.pages.copy_(pages)
    long = s.cache.lens.clone()
    s.cache.lens[s.slots[2].long()] = 10 ** 6     # a length that the table does not hold
    o, _ = attend(s, q, [0, 1, 2, 3], 0.125, window=64)
    with pytest.raises(ph.PhobosError):
        ph.device_status()
    assert near(o, [0, 1])
    s.cache.lens.copy_(long)
    # an indptr that does not ascend or leaves the rows: nothing outside is touched
    o = torch.full((6, 256), 7.0, device=dev).half()
    attend(s, q, [0, 9, -4, 2], 0.125, o=o[:3])
    assert bool((o[3:] == 7.0).all())
    try:
        ph.device_status()
    except ph.PhobosError:
        pass


def test_streams_graph_and_a_step_of_decoding(ph, dev):
    """extend, append in each layer, attend in each layer, as a decoder does, eagerly and as one captured graph that is
    replayed step after step; both give the same bytes as a cache that was filled at once."""
    import torch
    layers, lens, H, D, G, page = 2, [14, 31, 5], 2, 64, 32, 16
    steps, n = 20, 3
    torch.manual_seed(0)
    k = torch.randn(steps, layers, n, H * D, device=dev).half()
    q = torch.randn(steps, layers, n, 4 * D, device=dev).half()

    def fresh():
        s = Setup(ph, dev, lens, H, D, G, page, layers=layers, spare=8)
        t = s.cache.tables
        wide = torch.full((t.shape[0], t.shape[1] + 3), -1, dtype=torch.int32, device=dev)
        wide[:, :t.shape[1]] = t
        s.cache = ph.Kv4Cache(s.cache.pages, s.cache.refs, wide, s.cache.lens, kv_heads=H, head_dim=D, group=G, page_tokens=page)
        s.ws = torch.empty(max(256, ph.kv4_pages_workspace_bytes(s.cache), ph.kv4_attention_workspace_bytes(s.cache, n, n, 4)), dtype=torch.uint8, device=dev)
        return s

    one = torch.ones(n, dtype=torch.int32, device=dev)
    kk, qq, oo = torch.empty_like(k[0]), torch.empty_like(q[0]), torch.empty_like(q[0])

    def step(s):
        ph.kv4_extend(s.cache, s.slots, one, s.short, workspace=s.ws)
        for layer in range(layers):
            ph.kv4_append(s.cache, layer, kk[layer], kk[layer], s.slots)
            ph.kv4_attention(s.cache, layer, qq[layer], oo[layer], 0.125, s.slots, workspace=s.ws)

    a, outs = fresh(), []
    for i in range(steps):
        kk.copy_(k[i]); qq.copy_(q[i])
        step(a)
        assert int(a.short) == 0
        outs.append(oo.clone())
    assert a.cache.lens[a.slots.long()].tolist() == [l + steps for l in lens]
    s, graph = fresh(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(s)
    for i in range(steps):
        kk.copy_(k[i]); qq.copy_(q[i])
        graph.replay()
        assert torch.equal(oo, outs[i]), i
    assert ph.device_status() == 0
    # the last step against the definition
    for layer in range(layers):
        b = fresh()
        b.lens = [l + steps for l in lens]
        b.k = torch.cat([torch.cat([b.k[b.ind[j]:b.ind[j + 1]], k[:, layer, j]]) for j in range(n)])
        b.v = torch.cat([torch.cat([b.v[b.ind[j]:b.ind[j + 1]], k[:, layer, j]]) for j in range(n)])
        b.ind = [0, *np.cumsum(b.lens).tolist()]
        wo, _, to, _ = reference(b, q[-1, layer], [0, 1, 2, 3], 2, 0.125, 0)
        assert bool(((outs[-1][layer].double() - wo).abs() <= to).all())


def test_repeatable_and_alone_as_in_a_batch(ph, dev):
    """The same call twice gives the same bits."""
    import torch
    s = Setup(ph, dev, [3000, 17, 1200, 64], 4, 128, 128, 64, seed=9)
    q = torch.randn(4, 16 * 128, device=dev).half()
    o, lse = attend(s, q, [0, 1, 2, 3, 4], 0.09)
    for _ in range(5):
        o2, lse2 = attend(s, q, [0, 1, 2, 3, 4], 0.09)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_refusals(ph, dev):
    import torch
    s = Setup(ph, dev, [20], 2, 64, 64, 16)
    q = torch.randn(1, 256, device=dev).half()
    kv = torch.randn(1, 128, device=dev).half()
    need = ph.kv4_attention_workspace_bytes(s.cache, 1, 1, 4)
    ws = torch.empty(need + 256, dtype=torch.uint8, device=dev)
    att = lambda **k: ph.kv4_attention(s.cache, k.get("layer", 0), k.get("q", q), k.get("o", torch.empty_like(k.get("q", q))), 0.1, k.get("slots", s.slots),  # noqa: E731
                                       k.get("ind"), lse=k.get("lse"), window=k.get("window", 0), workspace=k.get("ws", ws))
    bad = [lambda: att(layer=1), lambda: att(layer=-1), lambda: att(q=q.float()), lambda: att(q=q[:, :192]), lambda: att(o=torch.empty(2, 256, device=dev).half()),
           lambda: att(window=-1), lambda: att(slots=s.slots.long()), lambda: att(slots=torch.zeros(2, dtype=torch.int32, device=dev)),
           lambda: att(lse=torch.empty(1, 3, device=dev)), lambda: att(lse=torch.empty(1, 4, device=dev).half()),
           lambda: att(ind=torch.zeros(1, dtype=torch.int32, device=dev)), lambda: att(q=torch.randn(1, 264, device=dev).half()[:, 4:260]),
           lambda: att(ws=None), lambda: ph.kv4_append(s.cache, 0, kv, kv, None), lambda: ph.kv4_append(s.cache, 0, kv.cpu(), kv, s.slots),
           lambda: ph.kv4_append(s.cache, 0, kv.double(), kv, s.slots), lambda: ph.kv4_append(s.cache, 0, kv[0], kv[0], s.slots), lambda: att(ws=ws[:need - 1]), lambda: att(ws=ws[8:]),
           lambda: ph.kv4_append(s.cache, 0, kv, kv[:, :64], s.slots), lambda: ph.kv4_append(s.cache, 0, kv.float(), kv.float(), s.slots),
           lambda: ph.kv4_append(s.cache, 3, kv, kv, s.slots), lambda: ph.kv4_read(s.cache, 0, kv[:0], kv, s.slots),
           lambda: ph.Kv4Cache.create(1, 4, 2, 96, 32, 16, 2, 4), lambda: ph.Kv4Cache.create(1, 4, 2, 64, 128, 16, 2, 4),
           lambda: ph.Kv4Cache.create(1, 4, 2, 64, 64, 24, 2, 4),
           lambda: ph.Kv4Cache(s.cache.pages[:, :, :-128], s.cache.refs, s.cache.tables, s.cache.lens, kv_heads=2, head_dim=64, group=64, page_tokens=16),
           lambda: ph.Kv4Cache(s.cache.pages, s.cache.refs[:-1], s.cache.tables, s.cache.lens, kv_heads=2, head_dim=64, group=64, page_tokens=16)]
    for i, f in enumerate(bad):
        with pytest.raises(ph.PhobosError):
            f()
            print("not refused:", i)
    att()
    assert ph.device_status() == 0


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 7, 10 ** 6, 97, 96, 95])
def test_windows_that_hide_nothing_or_little(ph, dev, window):
    """The largest windows, with more rows than tokens among the sequences, and windows around what the tables hold (96)."""
    s = Setup(ph, dev, [5, 70, 1, 80], 2, 64, 64, 16, seed=11)
    assert s.cache.tables.shape[1] * 16 == 96
    check(s, [9, 70, 4, 1], 4, window=window)
    check(s, [1, 1, 1, 1], 4, window=window, seed=2)


@pytest.mark.parametrize("length", [1, 700, 20000])
def test_values_over_the_whole_range_give_finite_outputs(ph, dev, length):
    """A group from -65504 to 65504 has the scale 8736 (131008 / 15 to f16), so that its code 15 stands for 65536: O has
    65504 there, as kv4_read gives.  One token, parts joined by a warp a row, and parts joined by a block.
    Weights off by 2^-11 of 8 scales either way leave code 15 above 65506 and code 0 within 8 * 8736 * 2^-11 < 35 and half an f16
    step, 16, of -65504."""
    import torch
    D, G = 64, 32
    s = Setup(ph, dev, [length], 1, D, G, 64, seed=12)
    s.v[:, 0::2], s.v[:, 1::2] = 65504.0, -65504.0
    ind = torch.tensor([0, length], dtype=torch.int32, device=dev)
    ph.kv4_append(s.cache, 0, s.k, s.v, s.slots, ind)
    k, v = torch.empty_like(s.k), torch.empty_like(s.v)
    ph.kv4_read(s.cache, 0, k, v, s.slots, ind)
    assert torch.equal(v, s.v)
    o, lse = attend(s, torch.randn(1, 2 * D, device=dev).half(), [0, 1], 0.125)
    assert ph.device_status() == 0 and bool(torch.isfinite(lse).all())
    assert bool((o[:, 0::2] == 65504.0).all()) and bool(((o[:, 1::2].float() + 65504.0).abs() <= 35 + 16).all())
    # a NaN is none of those
    s.v[0, 3] = float("nan")
    ph.kv4_append(s.cache, 0, s.k, s.v, s.slots, ind)
    o, _ = attend(s, torch.randn(1, 2 * D, device=dev).half(), [0, 1], 0.125)
    assert bool(torch.isnan(o.view(2, D)[:, :G]).all()) and bool(torch.isfinite(o.view(2, D)[:, G:]).all())


@pytest.mark.parametrize("D,G,rep,page", [(128, 128, 4, 64), (128, 32, 16, 128), (64, 64, 1, 16)])
def test_alone_and_in_a_batch(ph, dev, D, G, rep, page):
    """A sequence attended alone and in batches whose other sequences move the places where it is cut: each within the
    tolerance of the definition, and so within the sum of both of one another.  A window and several rows a sequence too."""
    import torch
    lens, new = [3000, 17, 1200, 64, 9000, 1], [1, 3, 1, 2, 1, 1]
    s = Setup(ph, dev, lens, 2, D, G, page, seed=21)
    ind = [0, *np.cumsum(new).tolist()]
    q = torch.randn(ind[-1], 2 * rep * D, generator=torch.Generator().manual_seed(22)).half().to(dev)
    scale = 1 / math.sqrt(D)
    for window in (0, 700):
        wo, wl, to, tl = reference(s, q, ind, rep, scale, window)
        near = lambda got, want, tol: bool(((got.double() - want).abs() <= tol).all())  # noqa: E731
        o, lse = attend(s, q, ind, scale, window)
        assert near(o, wo, to) and near(lse, wl, tl)
        for b in range(len(lens)):
            a, z = ind[b], ind[b + 1]
            o1, lse1 = attend(s, q[a:z].contiguous(), [0, z - a], scale, window, slots=s.slots[b:b + 1])
            assert near(o1, wo[a:z], to[a:z]) and near(lse1, wl[a:z], tl[a:z])
            assert near(o1, o[a:z].double(), 2 * to[a:z]) and near(lse1, lse[a:z].double(), 2 * tl[a:z])
        half = [4, 1, 0]
        i = [0]
        for b in half:
            i.append(i[-1] + new[b])
        rows = torch.cat([torch.arange(ind[b], ind[b + 1]) for b in half]).to(dev)
        o2, lse2 = attend(s, q[rows].contiguous(), i, scale, window, slots=s.slots[torch.tensor(half, device=dev)].contiguous())
        assert near(o2, wo[rows], to[rows]) and near(lse2, wl[rows], tl[rows])
    assert ph.device_status() == 0


def test_pages_beyond_four_gigabytes(ph, dev):
    """Offsets that pass 32 bits: pages and a second layer behind the first 2^32 bytes are written, read, attended, copied
    and moved like any others."""
    import torch
    H, D, G, page = 8, 128, 32, 256
    n_pages, seqs = 16500, 4
    c = ph.Kv4Cache.create(2, n_pages, H, D, G, page, seqs, 3)
    assert c.pages[0].numel() > 2 ** 32
    low = 16480
    c.refs[:low] = 1                                     # the pages in front are taken
    ws = torch.empty(max(ph.kv4_pages_workspace_bytes(c), ph.kv4_attention_workspace_bytes(c, 1, 1, 2 * H)), dtype=torch.uint8, device=dev)
    out = torch.zeros(1, dtype=torch.int32, device=dev)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    n, g = 600, torch.Generator().manual_seed(41)
    ph.kv4_extend(c, ints(2), ints(n), out, workspace=ws)
    assert int(out) == 0 and c.tables[2].tolist() == [low, low + 1, low + 2]
    k, v, q = (torch.randn(rows, heads * D, generator=g).half().to(dev) for rows, heads in ((n, H), (n, H), (1, 2 * H)))

    def right(slot, layer):
        for rows in (k, v):
            got = [torch.empty_like(k), torch.empty_like(v)]
            ph.kv4_read(c, layer, *got, ints(slot), ints(0, n))
            want = value(rows.unflatten(1, (H, D)), G).flatten(1)
            assert bool(((got[rows is v].double() - want).abs() <= 2.0 ** -11 * want.abs() * 1.001 + 2.0 ** -23).all())
        s = Setup.__new__(Setup)
        s.ph, s.dev, s.Hkv, s.D, s.G, s.lens, s.ind, s.k, s.v = ph, dev, H, D, G, [n], [0, n], k, v
        want, _, tol, _ = reference(s, q, [0, 1], 2, 0.09, 0)
        o = torch.empty_like(q)
        ph.kv4_attention(c, layer, q, o, 0.09, ints(slot), workspace=ws)
        assert bool(((o.double() - want).abs() <= tol).all())

    for layer in (0, 1):
        ph.kv4_append(c, layer, k, v, ints(2), ints(0, n))
    right(2, 0), right(2, 1)
    ph.kv4_fork(c, ints(2), ints(0), out, deep=True, workspace=ws)
    assert int(out) == 0 and c.tables[0].tolist() == [low + 3, low + 4, low + 5]
    ph.kv4_free(c, ints(2))
    right(0, 1)
    c.refs[:low] = 0                                     # now the copies are all there is: they move to the front
    ph.kv4_compact(c, out, workspace=ws)
    assert int(out) == 3 and c.tables[0].tolist() == [0, 1, 2]
    right(0, 0), right(0, 1)
    assert ph.device_status() == 0
