"""The 4-bit operators together, as a program that answers uses them: projections from 4-bit weights, the cache, branches of
a sequence, and the pages' housekeeping in between, against the same layer in 64 bits."""
import math

import pytest

pytestmark = pytest.mark.gpu


class Layer:
    """One attention layer: q, k, v and output projections in 4 bits, a cache for its keys and values."""

    def __init__(self, ph, dev, width=256, Hkv=2, rep=4, D=64, G=64, page=16, seqs=6, seed=0):
        import torch
        self.ph, self.dev, self.Hkv, self.rep, self.D, self.G = ph, dev, Hkv, rep, D, G
        g = torch.Generator().manual_seed(seed)
        self.w, self.packed = {}, {}
        for name, (n, k) in {"q": (Hkv * rep * D, width), "k": (Hkv * D, width), "v": (Hkv * D, width), "o": (width, Hkv * rep * D)}.items():
            code = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8).to(dev)
            scale = ((torch.rand(n, k // G, generator=g) + 0.5) * 0.25 / math.sqrt(k)).half().to(dev)
            zero = torch.randint(6, 10, (n, k // G), generator=g).half().to(dev)
            self.packed[name] = ph.q4_pack(code, scale, zero, G)
            self.w[name] = (scale.double()[..., None] * (code.double().unflatten(1, (-1, G)) - zero.double()[..., None])).flatten(1)
        self.cache = ph.Kv4Cache.create(1, 64, Hkv, D, G, page, seqs, 16)
        self.cache.pages.fill_(0xFF)
        self.ws = torch.empty(max(ph.kv4_pages_workspace_bytes(self.cache), ph.kv4_attention_workspace_bytes(self.cache, 64, seqs, Hkv * rep)),
                              dtype=torch.uint8, device=dev)
        self.short = torch.zeros(1, dtype=torch.int32, device=dev)
        self.k, self.v = [None] * seqs, [None] * seqs     # the rows that each sequence was given, f16

    def ints(self, v):
        import torch
        return torch.tensor(v, dtype=torch.int32, device=self.dev)

    def step(self, x, seqs, counts):
        """Rows x [T, width] f16 of sequences `seqs`, counts[i] each: the layer's f32 output."""
        import torch
        ph, T = self.ph, x.shape[0]
        proj = {n: torch.empty(T, self.w[n].shape[0], dtype=torch.float16, device=self.dev) for n in "qkv"}
        for n in "qkv":
            ph.gemv_q4(x, self.packed[n], proj[n], self.G)
        ind = [0]
        for c in counts:
            ind.append(ind[-1] + c)
        slots, i = self.ints(seqs), self.ints(ind)
        ph.kv4_extend(self.cache, slots, self.ints(counts), self.short, workspace=self.ws)
        ph.kv4_append(self.cache, 0, proj["k"], proj["v"], slots, i)
        o = torch.empty_like(proj["q"])
        ph.kv4_attention(self.cache, 0, proj["q"], o, 1 / math.sqrt(self.D), slots, i, workspace=self.ws)
        y = torch.empty(T, self.w["o"].shape[0], device=self.dev)
        ph.gemv_q4(o, self.packed["o"], y, self.G)
        assert int(self.short) == 0 and ph.device_status() == 0
        for s, a, b in zip(seqs, ind, ind[1:]):
            for mine, new in ((self.k, proj["k"][a:b]), (self.v, proj["v"][a:b])):
                mine[s] = new if mine[s] is None else torch.cat([mine[s], new])
        return y, proj, ind

    def want(self, x, seqs, proj, ind):
        """The layer in 64 bits on its own f16 projections, and those projections' distance from 64 bits."""
        import torch
        far = max(float((proj[n].double() - x.double() @ self.w[n].T).norm() / (x.double() @ self.w[n].T).norm()) for n in "qkv")
        out = []
        for s, a, b in zip(seqs, ind, ind[1:]):
            k, v = (self.value(t[s]).view(-1, self.Hkv, self.D) for t in (self.k, self.v))
            q = proj["q"][a:b].double().view(b - a, self.Hkv, self.rep, self.D)
            z = torch.einsum("ihrd,jhd->ihrj", q, k) / math.sqrt(self.D)
            n = k.shape[0]
            hide = torch.arange(n, device=self.dev)[None] > torch.arange(n - (b - a), n, device=self.dev)[:, None]
            p = torch.softmax(z.masked_fill(hide[:, None, None], -math.inf), -1)
            out.append(torch.einsum("ihrj,jhd->ihrd", p, v).flatten(1))
        return torch.cat(out) @ self.w["o"].T, far

    def value(self, x):
        import torch
        g = x.double().unflatten(1, (-1, self.G))
        lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        step = ((hi - lo) / 15).half().double()
        return torch.where(step > 0, lo + step * ((g - lo) / step.clamp_min(1e-30)).round().clamp(0, 15), lo).flatten(1)


def test_a_layer_answers_branches_and_is_compacted(ph, dev):
    import torch
    L = Layer(ph, dev)
    g = torch.Generator().manual_seed(5)
    rows = lambda n: torch.randn(n, 256, generator=g).half().to(dev)  # noqa: E731

    def go(seqs, counts):
        x = rows(sum(counts))
        y, proj, ind = L.step(x, seqs, counts)
        want, far = L.want(x, seqs, proj, ind)
        # f16 projections: half a step of each value, 2^-11, and f32 sums
        assert far <= 2.0 ** -11
        # the attention's f16 output (2^-11) and its f16 weights (2^-11 of values up to the group's whole range, which
        # averaging makes small): 2^-8 of the result's size covers both with the sizes of this layer
        assert float((y.double() - want).norm() / want.norm()) <= 2.0 ** -8

    go([4, 1], [37, 5])                                   # two prompts
    go([1, 4], [1, 1])
    L.ph.kv4_fork(L.cache, L.ints([4, 4]), L.ints([0, 2]), L.short, workspace=L.ws)
    L.ph.kv4_fork(L.cache, L.ints([1]), L.ints([3]), L.short, deep=True, workspace=L.ws)
    for s, f in ((0, 4), (2, 4), (3, 1)):
        L.k[s], L.v[s] = L.k[f], L.v[f]
    go([0, 2, 4, 3], [1, 3, 1, 1])                        # the branches part
    L.ph.kv4_free(L.cache, L.ints([4, 1]))
    L.k[4] = L.v[4] = L.k[1] = L.v[1] = None
    live = torch.zeros(1, dtype=torch.int32, device=dev)
    L.ph.kv4_compact(L.cache, live, workspace=L.ws)
    go([3, 0, 2], [1, 1, 1])
    L.ph.kv4_free(L.cache, L.ints([2]), keep=L.ints([30]))    # a rejected draft: the tail goes
    L.k[2], L.v[2] = L.k[2][:30], L.v[2][:30]
    go([2, 0, 1], [4, 1, 20])
    used = sum(-(-int(n) // 16) for n in L.cache.lens.tolist())
    assert int((L.cache.refs > 0).sum()) <= used and int(live) <= used + 6


def test_two_caches_on_two_streams(ph, dev):
    """Calls on different streams with workspaces of their own do not disturb one another."""
    import torch
    layers = [Layer(ph, dev, seed=s) for s in (1, 2)]
    x = [torch.randn(40, 256, device=dev).half() for _ in layers]
    alone = []
    for L, r in zip(layers, x):
        alone.append(L.step(r, [2], [40])[0])
    again = [Layer(ph, dev, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    torch.cuda.synchronize()
    for L, r, st in zip(again, x, streams):
        with torch.cuda.stream(st):
            q = torch.empty(40, 512, dtype=torch.float16, device=dev)
            kv = [torch.empty(40, 128, dtype=torch.float16, device=dev) for _ in "kv"]
            o, y = torch.empty_like(q), torch.empty(40, 256, device=dev)
            slots, ind = L.ints([2]), L.ints([0, 40])
            for _ in range(10):
                ph.gemv_q4(r, L.packed["q"], q, L.G)
                ph.gemv_q4(r, L.packed["k"], kv[0], L.G)
                ph.gemv_q4(r, L.packed["v"], kv[1], L.G)
                ph.kv4_free(L.cache, slots)
                ph.kv4_extend(L.cache, slots, L.ints([40]), L.short, workspace=L.ws)
                ph.kv4_append(L.cache, 0, kv[0], kv[1], slots, ind)
                ph.kv4_attention(L.cache, 0, q, o, 1 / 8, slots, ind, workspace=L.ws)
                ph.gemv_q4(o, L.packed["o"], y, L.G)
            outs.append(y)
    torch.cuda.synchronize()
    for a, b in zip(alone, outs):
        assert torch.equal(a, b)
    assert ph.device_status() == 0


def test_a_launch_that_fails_is_reported_once(ph, dev):
    """A launch that CUDA refuses (into the legacy stream while a stream that orders itself after it is being captured) is an
    error of that call alone: the next calls neither report it nor do without their work."""
    import torch
    from cuda.bindings import runtime
    L = Layer(ph, dev)
    x = torch.randn(3, 256, device=dev).half()
    y, again = torch.empty(3, 512, device=dev), torch.zeros(3, 512, device=dev)
    ph.gemv_q4(x, L.packed["q"], y, L.G)
    L.step(x, [2], [3])
    code = torch.randint(0, 16, (512, 256), dtype=torch.uint8, device=dev)
    scale = torch.rand(512, 4, device=dev).half()
    packed = ph.q4_pack(code, scale, None, L.G)
    out, slots = torch.zeros_like(packed), L.ints([2])
    q, o, o2 = torch.randn(1, 512, device=dev).half(), torch.empty(1, 512, device=dev).half(), torch.zeros(1, 512, device=dev).half()
    ph.kv4_attention(L.cache, 0, q, o, 0.125, slots, workspace=L.ws)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    calls = [lambda: ph.q4_pack(code, scale, None, L.G, out=out, stream=side), lambda: ph.kv4_attention(L.cache, 0, q, o2, 0.125, slots, workspace=L.ws, stream=side),
             lambda: ph.gemv_q4(x, L.packed["q"], again, L.G, stream=side)]
    for call in calls:
        err, stream = runtime.cudaStreamCreate()
        assert int(err) == 0
        assert int(runtime.cudaStreamBeginCapture(stream, runtime.cudaStreamCaptureMode.cudaStreamCaptureModeRelaxed)[0]) == 0
        try:
            with pytest.raises(ph.PhobosError) as e:
                ph.gemv_q4(x, L.packed["q"], y, L.G, stream=0)
            assert e.value.code == ph.PH_ERR_DEVICE
        finally:
            runtime.cudaStreamEndCapture(stream)
            runtime.cudaStreamDestroy(stream)
        call()
    torch.cuda.synchronize()
    assert torch.equal(out, packed) and torch.equal(o, o2) and torch.equal(y, again)
    assert ph.device_status() == 0
