"""Products with 4-bit weights (`gemv_q4`, `q4_pack`) on a B200 against the sum in 64 bits.

Tolerance: X and the codes are exact in f16 and their products exact in f32.  The matrix unit adds 16 products and the
running sum with an error of at most 2^-22 of what it adds (sums cut to f32, not rounded); a group's sum, the sum of x
times zero, and the sum over groups are one f32 rounding each.  With S = sum |x| scale (code + |zero|) that is at most
S (2 G/16 2^-22 + (3 + K/G + 40) 2^-24): the last 40 for joining partial sums.  An f16 Y adds half a step, 2^-11 |y|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _weights(N, K, G, seed, dev, zeros=True):
    import torch
    g = torch.Generator(device="cpu").manual_seed(seed)
    code = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8).to(dev)
    scale = (torch.rand(N, K // G, generator=g) * 0.1 + 1e-3).half().to(dev)
    zero = (torch.rand(N, K // G, generator=g) * 20 - 2).half().to(dev) if zeros else None
    return code, scale, zero


def _want(x, code, scale, zero, G):
    """The product and the bound's S, in f64."""
    s = scale.double().repeat_interleave(G, 1)
    z = zero.double().repeat_interleave(G, 1) if zero is not None else code.double() * 0 + 8
    w = s * (code.double() - z)
    return x.double() @ w.T, x.double().abs() @ (s * (code.double() + z.abs())).T


def _tol(S, y, K, G, half):
    t = S * (2 * G / 16 * 2.0 ** -22 + (43 + K / G) * 2.0 ** -24) + 1e-30
    return t + (y.abs() + t) * 2.0 ** -11 + 2.0 ** -25 if half else t


CASES = [(1, 16, 128, 128), (1, 1, 32, 32), (2, 17, 96, 32), (3, 130, 64, 64), (5, 33, 320, 64), (7, 8, 1152, 128), (8, 257, 2048, 128),
         (9, 100, 416, 32), (16, 64, 4096, 64), (17, 200, 640, 128), (33, 48, 1024, 32), (64, 96, 512, 128), (65, 31, 256, 64), (200, 40, 128, 128),
         (1, 4100, 1024, 128), (4, 2500, 8192, 64), (1, 24, 16384, 32),
         # sizes at which the tensor-core form is taken: each width of it, rows shared out along K, several groups of rows, a ragged K
         (11, 16387, 8192, 128), (30, 16011, 4096, 64), (64, 4100, 4096, 128), (200, 3001, 2048, 128), (61, 16500, 1056, 32)]


@pytest.mark.parametrize("M,N,K,G", CASES)
@pytest.mark.parametrize("out", ["f16", "f32"])
def test_gemv_q4_matches_the_sum(ph, dev, M, N, K, G, out):
    import torch
    g = torch.Generator().manual_seed(M * 7 + N)
    x = (torch.randn(M, K, generator=g) + 0.5).half().to(dev)
    code, scale, zero = _weights(N, K, G, N + K, dev, zeros=(M + N) % 2 == 1)
    w = ph.q4_pack(code, scale, zero, G)
    y = torch.full((M, N), float("nan"), dtype=torch.float16 if out == "f16" else torch.float32, device=dev)
    ph.gemv_q4(x, w, y, G)
    assert ph.device_status() == 0
    want, S = _want(x, code, scale, zero, G)
    assert bool(((y.double() - want).abs() <= _tol(S, want, K, G, out == "f16")).all())


def test_packed_layout_is_the_documented_one(ph, dev):
    """The block layout at the top of csrc/gemv_q4.cu, byte by byte."""
    import torch
    N, K, G = 18, 160, 32
    code, scale, zero = _weights(N, K, G, 3, dev)
    got = ph.q4_pack(code, scale, zero, G).cpu().numpy().view(np.uint8)
    c, s, z = code.cpu().numpy(), scale.cpu().numpy(), zero.cpu().numpy()
    block = 1024 + 64 * (128 // G)
    want = np.zeros(2 * 2 * block, dtype=np.uint8)
    for n in range(N):
        for k in range(K):
            base = (n // 16 * 2 + k // 128) * block
            r, kk = n % 16, k % 128
            S, t, e, i = kk // 32, kk % 32 // 8, kk % 8 // 4, kk % 4
            w, lane = 2 * S + e, 4 * (r % 8) + t
            at = base + w // 4 * 512 + lane * 16 + w % 4 * 4 + (0, 2, 1, 3)[i]
            want[at] |= c[n, k] << (4 * (r // 8))
        for q in range(K // G):
            at = (n // 16 * 2 + q * G // 128) * block + 1024 + ((q % (128 // G)) * 16 + n % 16) * 4
            want[at:at + 4] = np.array([s[n, q], z[n, q]], dtype=np.float16).view(np.uint8)
    assert np.array_equal(got, want)


def test_alpha_beta_strides_and_columns_behind_n(ph, dev):
    import torch
    M, N, K, G = 6, 45, 256, 64
    code, scale, zero = _weights(N, K, G, 9, dev)
    wide = torch.randn(M, K + 64, device=dev).half()
    x = wide[:, 32:32 + K]
    w = ph.q4_pack(code, scale, zero, G)
    for dt in (torch.float16, torch.float32):
        buf = torch.randn(M, N + 11, device=dev).to(dt)
        before = buf.clone()
        ph.gemv_q4(x, w, buf[:, 3:3 + N], G, alpha=0.5, beta=-2.0)
        want, S = _want(x, code, scale, zero, G)
        old = before[:, 3:3 + N].double()
        want = 0.5 * want - 2.0 * old
        tol = _tol(0.5 * S + 2 * old.abs(), want, K, G, dt == torch.float16)
        assert bool(((buf[:, 3:3 + N].double() - want).abs() <= tol).all())
        assert torch.equal(buf[:, :3], before[:, :3]) and torch.equal(buf[:, 3 + N:], before[:, 3 + N:])
        # beta = 0: what Y held is not read, not even a NaN
        buf.fill_(float("nan"))
        ph.gemv_q4(x, w, buf[:, 3:3 + N], G)
        assert bool(torch.isfinite(buf[:, 3:3 + N]).all()) and bool(torch.isnan(buf[:, :3]).all())


def test_tensor_core_form_strides_alpha_beta_and_graph(ph, dev):
    """The same where more than eight rows take the tensor-core form: rows of X out of a wider tensor, rows of Y too."""
    import torch
    M, N, K, G = 24, 16400, 4096, 128
    code, scale, zero = _weights(N, K, G, 2, dev)
    w = ph.q4_pack(code, scale, zero, G)
    wide = torch.randn(M, K + 128, device=dev).half()
    x = wide[:, 64:64 + K]
    want, S = _want(x, code, scale, zero, G)
    for dt in (torch.float16, torch.float32):
        buf = torch.randn(M + 1, N + 9, device=dev).to(dt)
        before = buf.clone()
        ph.gemv_q4(x, w, buf[:M, 5:5 + N], G, alpha=-1.5, beta=0.5)
        old = before[:M, 5:5 + N].double()
        tol = _tol(1.5 * S + 0.5 * old.abs(), -1.5 * want + 0.5 * old, K, G, dt == torch.float16)
        assert bool(((buf[:M, 5:5 + N].double() - (-1.5 * want + 0.5 * old)).abs() <= tol).all())
        assert torch.equal(buf[M:], before[M:]) and torch.equal(buf[:, :5], before[:, :5]) and torch.equal(buf[:, 5 + N:], before[:, 5 + N:])
    y, z = torch.empty(M, N, device=dev), torch.empty(M, N, device=dev)
    graph = torch.cuda.CUDAGraph()
    ph.gemv_q4(x, w, z, G)
    with torch.cuda.graph(graph):
        ph.gemv_q4(x, w, z, G)
        ph.gemv_q4(x[:7], w, z[:7], G)       # the other form right behind it
    wide.mul_(-0.5)
    graph.replay()
    ph.gemv_q4(x, w, y, G)
    ph.gemv_q4(x[:7], w, y[:7], G)
    assert torch.equal(y, z)
    # an infinity in one row of X stays there
    x[3, 9] = float("inf")
    ph.gemv_q4(x, w, y, G)
    keep = [i for i in range(M) if i != 3]
    assert torch.equal(y[keep][7:], z[keep][7:]) and bool(torch.isfinite(y[keep]).all()) and not bool(torch.isfinite(y[3]).any())
    assert ph.device_status() == 0


def test_extreme_values(ph, dev):
    """f16's largest and smallest x and scales: no product leaves f32, subnormals are not flushed."""
    import torch
    N, K, G = 32, 128, 128
    code = torch.arange(N * K, device=dev).remainder(16).to(torch.uint8).view(N, K)
    zero = torch.zeros(N, 1, device=dev).half()
    for xv, sv in ((65504.0, 65504.0), (6e-8, 1.0), (1.0, 6e-8), (6e-8, 6e-8)):
        x = torch.full((2, K), xv, device=dev).half()
        scale = torch.full((N, 1), sv, device=dev).half()
        y = torch.empty(2, N, device=dev)
        ph.gemv_q4(x, ph.q4_pack(code, scale, zero, G), y, G)
        want, S = _want(x, code, scale, zero, G)
        assert bool(((y.double() - want).abs() <= _tol(S, want, K, G, False)).all())
    # rows and outputs are apart: an infinity in one row of X stays there
    x = torch.ones(3, K, device=dev).half()
    x[1, 5] = float("inf")
    y = torch.empty(3, N, device=dev)
    ph.gemv_q4(x, ph.q4_pack(code, torch.ones(N, 1, device=dev).half(), zero, G), y, G)
    assert bool(torch.isfinite(y[[0, 2]]).all()) and not bool(torch.isfinite(y[1]).any())


def test_by_entry_name_stream_and_graph(ph, dev):
    import torch
    M, N, K, G = 3, 80, 512, 128
    code, scale, zero = _weights(N, K, G, 4, dev)
    x, w = torch.randn(M, K, device=dev).half(), ph.q4_pack(code, scale, zero, G)
    y = torch.empty(M, N, device=dev)
    ph.gemv_q4(x, w, y, G)
    z = torch.empty_like(y)
    group = ph.PhScalar(5, ph.I32, G)
    ph.launch("gemv_q4", [x, w, z], [ph.scalar_f32(3, 1.0), ph.scalar_f32(4, 0.0), group])
    assert torch.equal(y, z)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    z.zero_()
    torch.cuda.synchronize()
    ph.gemv_q4(x, w, z, G, stream=side)
    side.synchronize()
    assert torch.equal(y, z)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ph.gemv_q4(x, w, z, G)
    x.mul_(2)
    graph.replay()
    ph.gemv_q4(x, w, y, G)
    assert torch.equal(y, z)
    assert ph.device_status() == 0


def test_refusals(ph, dev):
    import torch
    N, K, G = 32, 256, 64
    code, scale, zero = _weights(N, K, G, 1, dev)
    x, w, y = torch.randn(4, K, device=dev).half(), ph.q4_pack(code, scale, zero, G), torch.empty(4, N, device=dev)
    bad = [lambda: ph.gemv_q4(x.float(), w, y, G), lambda: ph.gemv_q4(x, w, y.to(torch.int32), G), lambda: ph.gemv_q4(x, w, y, 48),
           lambda: ph.gemv_q4(x[:, :200], w, y, G), lambda: ph.gemv_q4(x[:3], w, y, G), lambda: ph.gemv_q4(x, w[:-16], y, G),
           lambda: ph.gemv_q4(x, w[4:], y, G), lambda: ph.gemv_q4(x[:, 1:257 - 64], w, y, G),
           lambda: ph.gemv_q4(x, w, y.t(), G), lambda: ph.q4_pack(code, scale[:, :-1], zero, G), lambda: ph.q4_pack(code, scale, zero[:-1], G),
           lambda: ph.q4_pack(code.int(), scale, zero, G), lambda: ph.q4_pack(code, scale.float(), zero, G),
           lambda: ph.q4_pack(code, scale, zero, G, out=w[:100]), lambda: ph.gemv_q4(x.cpu(), w, y, G)]
    for f in bad:
        with pytest.raises(ph.PhobosError):
            f()
    ph.gemv_q4(x[:0], w, y[:0], G)   # no rows: nothing to do
    assert ph.device_status() == 0


@pytest.mark.parametrize("M,N,K,G", [(64, 16384, 1152, 128), (64, 4096, 5504, 128), (64, 4096, 13696, 128)])
def test_tensor_core_form_with_a_half_filled_last_stage(ph, dev, M, N, K, G):
    """An odd number of 128-column blocks, or an odd share of them for each CTA of a cluster of two: the last stage holds one
    block instead of two, which must not release the stage before it in its slot.  The same bits in every call."""
    import torch
    g = torch.Generator().manual_seed(K)
    x = torch.randn(M, K, generator=g).half().to(dev)
    code, scale, zero = _weights(N, K, G, N + K, dev)
    w = ph.q4_pack(code, scale, zero, G)
    y, again = torch.empty(M, N, device=dev), torch.empty(M, N, device=dev)
    ph.gemv_q4(x, w, y, G)
    want, S = _want(x, code, scale, zero, G)
    assert bool(((y.double() - want).abs() <= _tol(S, want, K, G, False)).all())
    for _ in range(30):
        ph.gemv_q4(x, w, again, G)
        assert torch.equal(y, again)
    assert ph.device_status() == 0


@pytest.mark.parametrize("M,N,K,G", [(5, 70, 256, 32), (8, 5000, 384, 128), (1, 24, 16384, 64), (24, 16400, 1024, 128), (11, 16387, 512, 64), (64, 4100, 5504, 128),
                                     (64, 2048, 8192, 128)])
@pytest.mark.parametrize("out", ["f16", "f32"])
def test_infinities_are_those_of_the_definition(ph, dev, M, N, K, G, out):
    """inf and -inf in x, alone, in one group, in two, and a NaN: infinities of the weight's sign, NaN where a weight is zero or
    infinities cancel, and the rows without any as they are."""
    import torch
    g = torch.Generator().manual_seed(N)
    x = torch.randn(M, K, generator=g).half().to(dev)
    code, scale, _ = _weights(N, K, G, N + K, dev)
    zero = torch.randint(-3, 16, (N, K // G), generator=g).half().to(dev)
    scale[::3] *= -1
    scale[5] = 0
    inf = float("inf")
    x[0, 17] = inf
    if M > 4:
        x[1, K - 1] = -inf
        x[2, 3], x[2, 9], x[2, K - 20] = inf, -inf, inf
        x[3, 40], x[3, 41] = float("nan"), inf
    y = torch.randn(M, N, device=dev).to(torch.float16 if out == "f16" else torch.float32)
    old = y.double()
    ph.gemv_q4(x, ph.q4_pack(code, scale, zero, G), y, G, alpha=-0.5, beta=0.25)
    assert ph.device_status() == 0
    want, _ = _want(x, code, scale, zero, G)
    want = -0.5 * want + 0.25 * old
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    assert torch.equal(torch.isinf(y), torch.isinf(want)) and bool((y.double() == want)[torch.isinf(want)].all())
    assert bool(torch.isinf(want[0]).any()) and bool(torch.isnan(want[0]).any())
    ok = torch.isfinite(want)
    _, S = _want(x, code, scale.abs(), zero, G)
    S = 0.5 * S + 0.25 * old.abs()
    assert bool(((y.double() - want).abs() <= _tol(S, want, K, G, out == "f16"))[ok].all())


EDGES = """
import sys
sys.path.insert(0, {root!r})
import torch
import __graft_entry__ as entry
from cuda.bindings import runtime
ph = entry.load_package()
dev = torch.device("cuda:0")
calls = []
for M, N, K in ((24, 16400, 1024), (64, 2048, 8192), (3, 80, 512)):      # tcgen05, in clusters, warp-level
    code = torch.randint(0, 16, (N, K), device=dev, dtype=torch.uint8)
    w = ph.q4_pack(code, torch.rand(N, K // 128, device=dev).half(), None, 128)
    calls.append((torch.randn(M, K, device=dev).half(), w, torch.empty(M, N, device=dev)))
for c in calls:
    ph.gemv_q4(*c, 128)
graph = torch.cuda.CUDAGraph(keep_graph=True)
with torch.cuda.graph(graph):
    for c in calls + calls:
        ph.gemv_q4(*c, 128)
get = lambda *n: runtime.cudaGraphGetEdges_v2(runtime.cudaGraph_t(graph.raw_cuda_graph()), *n)
n = get()[-1]
_, _, _, data, _ = get(n)
print("edges", n, sum(int(d.type) == int(runtime.cudaGraphDependencyType.cudaGraphDependencyTypeProgrammatic) for d in data))
"""


@pytest.mark.parametrize("pdl", ["0", "1"])
def test_the_switch_for_early_starts_reaches_every_form(ph, dev, pdl):
    """PHOBOS_PDL=0 (read once, so in a process of its own) turns the early start off for all of gemv_q4's kernels: of the
    five edges between six captured calls none is then programmatic.  Without it some are (not all: capture puts ordinary
    edges in front of kernels in clusters)."""
    import os
    import subprocess
    import sys
    from pathlib import Path
    code = EDGES.replace("{root!r}", repr(str(Path(__file__).resolve().parent.parent)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=dict(os.environ, PHOBOS_PDL=pdl))
    assert r.returncode == 0, r.stderr[-2000:]
    word, edges, early = r.stdout.split()
    assert (word, edges) == ("edges", "5") and (int(early) > 0) == (pdl == "1")


# forms that the sizes above leave out: sixteen columns with G = 64, 32 columns with G = 32, 64 columns with G = 64, and shares
# along K for clusters of two and of four, with even, odd and unequal shares
MORE = [(9, 18766, 448, 64), (16, 18930, 2112, 64), (31, 56074, 160, 32), (32, 18930, 2080, 32), (48, 16390, 1152, 64), (64, 14133, 4096, 64),
        (64, 2048, 8192, 128), (58, 2220, 4736, 128), (29, 2327, 15232, 128), (128, 1125, 22272, 64), (29, 4608, 7680, 128), (61, 4619, 12160, 64),
        (2048, 51, 5120, 128)]


@pytest.mark.parametrize("M,N,K,G", MORE)
def test_tensor_core_forms_left(ph, dev, M, N, K, G):
    import torch
    g = torch.Generator().manual_seed(M + K)
    x = (torch.randn(M, K, generator=g) + 0.5).half().to(dev)
    code, scale, zero = _weights(N, K, G, N + K, dev, zeros=M % 2 == 0)
    w = ph.q4_pack(code, scale, zero, G)
    y, z = torch.full((M, N), float("nan"), device=dev), torch.full((M, N), float("nan"), device=dev)
    ph.gemv_q4(x, w, y, G)
    want, S = _want(x, code, scale, zero, G)
    assert bool(((y.double() - want).abs() <= _tol(S, want, K, G, False)).all())
    ph.gemv_q4(x, w, z, G)
    assert torch.equal(y, z) and ph.device_status() == 0


@pytest.mark.parametrize("G,K", [(128, 1152), (64, 448), (32, 416)])
@pytest.mark.parametrize("M,N", [(1, 5003), (7, 9401), (8, 9501), (2, 18901), (3, 20011), (1, 40007), (13, 9501)])
def test_warp_level_forms(ph, dev, M, N, G, K):
    """Shares of one to more than eight tiles a CTA: each shape of the warp-level kernel, with tiles and columns left over.
    (13 rows: the 128 and 64 groups may take the tensor-core form.)"""
    import torch
    g = torch.Generator().manual_seed(M + N)
    x = (torch.randn(M, K, generator=g) - 0.25).half().to(dev)
    code, scale, zero = _weights(N, K, G, N + K, dev, zeros=M != 2)
    w = ph.q4_pack(code, scale, zero, G)
    buf = torch.full((M, N + 3), float("nan"), device=dev)
    ph.gemv_q4(x, w, buf[:, 1:1 + N], G)
    want, S = _want(x, code, scale, zero, G)
    assert bool(((buf[:, 1:1 + N].double() - want).abs() <= _tol(S, want, K, G, False)).all())
    assert bool(torch.isnan(buf[:, [0, N + 1, N + 2]]).all()) and ph.device_status() == 0


@pytest.mark.parametrize("M", [1, 20])
def test_weights_beyond_four_gigabytes(ph, dev, M):
    """Packed weights of more than 2^32 bytes: the last rows of Y against the sum in 64 bits."""
    import torch
    N, K, G = 65541, 131072, 128
    code = torch.randint(0, 16, (N, K), dtype=torch.uint8, device=dev)
    scale = (torch.rand(N, K // G, device=dev) * 0.1 + 1e-3).half()
    zero = (torch.rand(N, K // G, device=dev) * 20 - 2).half()
    w = ph.q4_pack(code, scale, zero, G)
    assert w.numel() > 2 ** 32
    x = torch.randn(M, K, device=dev).half()
    y = torch.empty(M, N, device=dev)
    ph.gemv_q4(x, w, y, G)
    for a, z in ((0, 40), (32760, 32800), (N - 40, N)):
        want, S = _want(x, code[a:z], scale[a:z], zero[a:z], G)
        assert bool(((y[:, a:z].double() - want).abs() <= _tol(S, want, K, G, False)).all())
    assert ph.device_status() == 0
