"""Operators of serving from 4-bit weights and a 4-bit key/value cache: cases, plain forms and exact values.

A cache is a pool of pages; a page holds `page` tokens of all key/value heads of one layer, in units of 16 tokens of one head:
  K codes [8 D bytes] | V codes [8 D bytes] | K (scale, zero) [16 tokens][D / G] f16 pairs | V (scale, zero) the same
and a value is zero + scale * code, code in 0..15.  Codes stand in the order in which a warp feeds them to the matrix unit:
  K: token r = 8 h + g, dims 8 (4 j + t) .. + 7 are the 32-bit word at byte 4 D h + (4 g + t) D / 8 + 4 j, dim i in bits 4 i
  V: token r = 8 h + 2 t + l, dims 32 p + 4 g .. + 3 are the 16-bit word at byte 4 D h + (4 g + t) D / 8 + 4 p + 2 l, dim x in bits 4 x
Weights W[n, k] = scale[n, k / G] (code - zero[n, k / G]) stand in blocks of 16 rows x 128 columns (see pack_weights)."""
import importlib
import math

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # a projection of one token's hidden state: launch and memory latency count
        {"name": "gemv_1x4096x4096", "op": "gemv", "M": 1, "N": 4096, "K": 4096, "G": 128, "out": "f16", "zeros": False},
        # a few sequences through a layer with an uneven number of outputs, f32 results (as logits are kept)
        {"name": "gemv_5x11001x4096_f32", "op": "gemv", "M": 5, "N": 11001, "K": 4096, "G": 64, "out": "f32", "zeros": True},
        # a batch of 32 sequences through a large layer
        {"name": "gemv_32x16384x8192", "op": "gemv", "M": 32, "N": 16384, "K": 8192, "G": 128, "out": "f16", "zeros": True},
        # one sequence of a chat: one token appended and attended, small pages
        {"name": "attn_1x777", "op": "attn", "B": 1, "ctx": 777, "nq": 1, "Hkv": 8, "rep": 4, "D": 128, "G": 128, "page": 16, "window": 0},
        # a serving batch of uneven lengths, one token each
        {"name": "attn_64x8192", "op": "attn", "B": 64, "ctx": 8192, "nq": 1, "Hkv": 8, "rep": 4, "D": 128, "G": 128, "page": 64, "window": 0},
        # two long documents, fine groups, one key/value head for 16 query heads
        {"name": "attn_2x131072_g32", "op": "attn", "B": 2, "ctx": 131072, "nq": 1, "Hkv": 4, "rep": 16, "D": 128, "G": 32, "page": 128, "window": 0},
        # prompts in chunks of uneven size that continue cached text, sliding window
        {"name": "attn_chunk_3x4000", "op": "attn", "B": 3, "ctx": 4000, "nq": 500, "Hkv": 8, "rep": 4, "D": 64, "G": 64, "page": 32, "window": 1500},
        # the cache write of a decode step of 32 sequences, read back
        {"name": "append_32x1", "op": "append", "B": 32, "ctx": 2048, "nq": 1, "Hkv": 8, "rep": 1, "D": 128, "G": 128, "page": 64, "window": 0},
        # long prompts written into the cache, read back
        {"name": "append_4x8000", "op": "append", "B": 4, "ctx": 8191, "nq": 8000, "Hkv": 8, "rep": 1, "D": 128, "G": 32, "page": 64, "window": 0},
        # a search that branches every sequence and lets each branch grow: shared pages, last page copied on write
        {"name": "pages_branch_48", "op": "branch", "n": 48, "len": 1000, "add": 5, "layers": 16, "pages": 2048, "Hkv": 8, "D": 128, "G": 128, "page": 64},
        # sequences copied whole, to be edited apart
        {"name": "pages_copy_16", "op": "copy", "n": 16, "len": 2000, "add": 0, "layers": 16, "pages": 2048, "Hkv": 8, "D": 128, "G": 128, "page": 64},
        # half of the sequences leave, what remains moves to the front of the pool
        {"name": "pages_compact_40", "op": "compact", "n": 40, "len": 1500, "add": 0, "layers": 16, "pages": 1024, "Hkv": 8, "D": 128, "G": 128, "page": 64},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemv", "gemv", "gemv", "attn", "attn", "attn", "attn", "append", "append", "branch", "copy", "compact"])
    if op == "gemv":
        G, M = rng.choice([32, 64, 128]), _log(rng, 1, 64)
        K = G * max(1, _log(rng, 128, 16384) // G)
        N = min(_log(rng, 64, 32768), 16384 * 8192 // K)
        if M * N * K > 32 * 16384 * 8192:
            N = 32 * 16384 * 8192 // (M * K)
        return {"op": op, "M": M, "N": N, "K": K, "G": G, "out": rng.choice(["f16", "f32"]), "zeros": rng.random() < 0.5}
    if op in ("attn", "append"):
        D, Hkv = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
        G = rng.choice([g for g in (32, 64, 128) if g <= D])
        B, nq = _log(rng, 1, 64), rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 16, 500)])
        rep = rng.choice([1, 2, 3, 4, 5, 7, 8, 16]) if op == "attn" else 1
        ctx = max(nq, _log(rng, 1, 131072))
        ctx = max(nq, min(ctx, (1 << 19) * 8 // (B * Hkv)))
        if op == "attn" and nq > 1:  # the largest prompt chunk's work
            most = 3 * 500 * 4000 * 32 * 64
            B = max(1, min(B, most // (nq * ctx * Hkv * rep * D)))
            ctx = max(nq, min(ctx, most // (B * nq * Hkv * rep * D)))
            nq = min(nq, max(1, most // (B * ctx * Hkv * rep * D)))
        return {"op": op, "B": B, "ctx": ctx, "nq": nq, "Hkv": Hkv, "rep": rep, "D": D, "G": G, "page": rng.choice([16, 32, 64, 128]),
                "window": rng.choice([0, 0, _log(rng, 1, 4096)]) if op == "attn" else 0}
    page, length = rng.choice([16, 32, 64, 128]), _log(rng, 20, 2000)
    n = _log(rng, 1, 40)
    per = -(-length // page) + 1
    most = 16 * 1024 * 64  # tokens x layers of the largest pool that is moved
    layers = rng.choice([1, 4, 16])
    n = max(1, min(n, most // (2 * per * page * layers)))
    return {"op": op, "n": n, "len": length, "add": _log(rng, 1, 100) if op == "branch" else 0, "layers": layers, "pages": 2 * n * (per + 8) + rng.randint(1, 64),
            "Hkv": rng.choice([1, 2, 8]), "D": 128, "G": rng.choice([32, 128]), "page": page}


# ---- inputs ---------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def quantise(x, G):
    """f16 [..., D] -> codes uint8 [..., D], (scale, zero) f16 [..., D / G, 2]."""
    g = x.float().unflatten(-1, (-1, G))
    lo, hi = g.amin(-1), g.amax(-1)
    scale = ((hi - lo) / 15.0).half()
    s = scale.float()[..., None]
    code = torch.where(s > 0, ((g - lo[..., None]) / s).round(), torch.zeros_like(g)).clamp(0, 15)
    return code.flatten(-2).to(torch.uint8), torch.stack([scale, lo.half()], -1)


def values(code, par, G):
    """The f32 values that codes [..., D] with (scale, zero) [..., D / G, 2] stand for."""
    p = par.float()
    return (code.unflatten(-1, (-1, G)).float() * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def pack_pages(kc, vc, kp, vp):
    """Codes [pages, heads, page, D] and params [pages, heads, page, D / G, 2] -> pages as bytes [pages, page bytes]."""
    n, h, p, d = kc.shape
    u = p // 16
    k = kc.view(n, h, u, 2, 8, d // 32, 4, 4, 2)                            # half, g, j, t, byte, nibble
    k = (k[..., 0] | (k[..., 1] << 4)).permute(0, 1, 2, 3, 4, 6, 5, 7).reshape(n, h, u, 8 * d)
    v = vc.view(n, h, u, 2, 4, 2, d // 32, 8, 2, 2)                         # half, t, l, p, g, byte, nibble
    v = (v[..., 0] | (v[..., 1] << 4)).permute(0, 1, 2, 3, 7, 4, 6, 5, 8).reshape(n, h, u, 8 * d)
    par = [x.contiguous().view(torch.uint8).reshape(n, h, u, -1) for x in (kp, vp)]
    return torch.cat([k, v, *par], -1).reshape(n, -1)


def pack_weights(code, par, G):
    """Codes [N, K] and (scale, zero) [N, K / G, 2] -> blocks of 16 rows x 128 columns: 1024 bytes of codes, then [128 / G][16 rows] pairs.
    Rows g and g + 8 share bytes (low and high nibble); lane 4 g + t holds columns 32 s + 8 t .. + 7 of its rows, four to a word in the order
    0, 2, 1, 3, the words 2 s + e of a lane in two groups of four."""
    n, k = code.shape
    rows, cols = -(-n // 16), -(-k // 128)
    c = torch.zeros(rows * 16, cols * 128, dtype=torch.uint8, device=code.device)
    c[:n, :k] = code
    p = torch.zeros(rows * 16, cols * 128 // G, 2, dtype=torch.float16, device=code.device)
    p[:n, :k // G] = par
    c = c.view(rows, 2, 8, cols, 2, 2, 4, 2, 4)                             # tile, half, g, block, s / 2, s % 2, t, e, column
    c = (c[:, 0] | (c[:, 1] << 4))[..., [0, 2, 1, 3]]                       # tile, g, block, s / 2, s % 2, t, e, byte
    c = c.permute(0, 2, 3, 1, 5, 4, 6, 7).reshape(rows, cols, 1024)
    p = p.view(rows, 16, cols, 128 // G, 2).permute(0, 2, 3, 1, 4).contiguous().view(torch.uint8).reshape(rows, cols, -1)
    return torch.cat([c, p], -1).reshape(-1)


def _gemv_inputs(case, seed):
    g = _gen(seed)
    M, N, K, G = case["M"], case["N"], case["K"], case["G"]
    x = torch.randn(M, K, generator=g, device=DEV).half()
    code = torch.randint(0, 16, (N, K), generator=g, device=DEV, dtype=torch.uint8)
    scale = (torch.rand(N, K // G, generator=g, device=DEV) * 0.02 + 0.005).half()
    zero = torch.randint(5, 11, (N, K // G), generator=g, device=DEV).half() if case["zeros"] else torch.full((N, K // G), 8.0, device=DEV).half()
    return x, code, torch.stack([scale, zero], -1)


def _lengths(case, seed):
    """Lengths (with the new tokens) and numbers of new tokens of each sequence: a case's own set, in an order that goes by the seed."""
    r = torch.Generator().manual_seed(case["B"] * 1000003 + case["ctx"])
    B, ctx, nq = case["B"], case["ctx"], case["nq"]
    new = torch.randint(max(1, nq // 2), nq + 1, (B,), generator=r)
    new[0] = nq
    length = torch.maximum(new, torch.randint(1, ctx + 1, (B,), generator=r))
    length[0] = ctx
    order = torch.randperm(B, generator=torch.Generator().manual_seed(seed))
    return length[order], new[order]


def _pool_lengths(case):
    r = torch.Generator().manual_seed(case["n"] * 1000003 + case["len"])
    return torch.randint(max(1, case["len"] * 3 // 4), case["len"] + 1, (case["n"],), generator=r)


def _cache_inputs(case, seed):
    g, r = _gen(seed), torch.Generator().manual_seed(seed + 1)
    B, H, D, G, P = case["B"], case["Hkv"], case["D"], case["G"], case["page"]
    length, new = _lengths(case, seed)
    need = (length + P - 1) // P
    width, total = int(need.max()) + 1, int(need.sum()) + 5
    used = torch.arange(width)[None] < need[:, None]
    slots = torch.randperm(B + 3, generator=r)[:B]
    rows = torch.full((B, width), -1)
    rows[used] = torch.randperm(total, generator=r)[:int(need.sum())]
    tables = torch.full((B + 3, width), -1)
    tables[slots] = rows
    lens = torch.zeros(B + 3, dtype=torch.int64)
    lens[slots] = length
    refs = torch.zeros(total, dtype=torch.int64)
    refs[rows[used]] = 1
    spread = torch.exp(torch.randn(H, 1, D, generator=g, device=DEV) * 0.4)  # keys have channels of unlike size
    k = (torch.randn(total, H, P, D, generator=g, device=DEV, dtype=torch.float16) * spread.half())
    kc, kp = quantise(k, G)
    k = torch.randn(total, H, P, D, generator=g, device=DEV, dtype=torch.float16)
    vc, vp = quantise(k, G)
    # slots behind a sequence's end, and the places that the new tokens take, hold what memory happened to hold
    past = torch.zeros(total, P, dtype=torch.bool)
    past[rows[used]] = (torch.arange(width)[None, :, None] * P + torch.arange(P) < (length - new)[:, None, None])[used]
    stale = ~past.to(DEV)[:, None, :, None, None]
    kp, vp = kp.masked_fill(stale, float("nan")), vp.masked_fill(stale, float("nan"))
    T = int(new.sum())
    ind = torch.zeros(B + 1, dtype=torch.int64)
    ind[1:] = new.cumsum(0)
    kn = (torch.randn(T, H, D, generator=g, device=DEV) * spread[:, 0]).half()
    vn = torch.randn(T, H, D, generator=g, device=DEV).half()
    q = (torch.randn(T, H * case["rep"], D, generator=g, device=DEV) * 2.0).half()
    i32 = lambda t: t.to(DEV, torch.int32)  # noqa: E731
    return {"kc": kc, "kp": kp, "vc": vc, "vp": vp, "kn": kn.flatten(1), "vn": vn.flatten(1), "q": q.flatten(1), "tables": i32(tables), "lens": i32(lens),
            "refs": i32(refs), "slots": i32(slots), "ind": i32(ind), "longest": int(length.max()), "most": int(new.max())}


def _pages_inputs(case, seed):
    """A pool of sequences that fill part of it; one int32 tensor holds refs, lens and tables, so that a pass starts from the same ones."""
    g, r = _gen(seed), torch.Generator().manual_seed(seed)
    n, P, N = case["n"], case["page"], case["pages"]
    length = _pool_lengths(case)[torch.randperm(n, generator=r)]
    need = (length + P - 1) // P
    width = -(-(case["len"] + case["add"]) // P) + 1
    used = torch.arange(width)[None] < need[:, None]
    tables = torch.full((2 * n, width), -1, dtype=torch.int64)
    ids = torch.randperm(N, generator=r)[:int(need.sum())]
    tables[:n][used] = ids
    lens = torch.zeros(2 * n, dtype=torch.int64)
    lens[:n] = length
    refs = torch.zeros(N, dtype=torch.int64)
    refs[ids] = 1
    unit = 16 * case["D"] + 128 * (case["D"] // case["G"])
    pool = torch.randint(0, 256, (case["layers"], N, case["Hkv"] * P // 16 * unit), generator=g, device=DEV, dtype=torch.uint8)
    a, b = torch.randperm(n, generator=r), torch.randperm(n, generator=r)
    return {"pool": pool, "meta": torch.cat([refs, lens, tables.flatten()]).to(DEV, torch.int32), "src": a.to(DEV, torch.int32), "dst": (b + n).to(DEV, torch.int32),
            "gone": a[: (n + 1) // 2].to(DEV, torch.int32), "add": torch.full((n,), case["add"], device=DEV, dtype=torch.int32), "width": width}


def prepare(case, seed):
    s = {"case": case}
    if case["op"] == "gemv":
        x, code, par = _gemv_inputs(case, seed)
        s |= {"x": x, "code": code, "par": par, "packed": pack_weights(code, par, case["G"]),
              "y": torch.empty(case["M"], case["N"], device=DEV, dtype=torch.float16 if case["out"] == "f16" else torch.float32)}
    elif case["op"] in ("attn", "append"):
        s |= _cache_inputs(case, seed)
        s["pool"] = pack_pages(s["kc"], s["vc"], s["kp"], s["vp"])[None]
        s["o"], s["lse"] = torch.empty_like(s["q"]), torch.empty(s["q"].shape[0], case["Hkv"] * case["rep"], device=DEV)
        s["kr"], s["vr"] = torch.empty_like(s["kn"]), torch.empty_like(s["vn"])
    else:
        s |= _pages_inputs(case, seed)
        N, n = case["pages"], case["n"]
        s["now"] = s["meta"].clone()
        s["refs"], s["lens"], s["tables"] = s["now"][:N], s["now"][N:N + 2 * n], s["now"][N + 2 * n:].view(2 * n, s["width"])
        s["count"] = torch.zeros(1, device=DEV, dtype=torch.int32)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _plain_gemv(s):
    G = s["case"]["G"]
    p = s["par"].float()
    w = ((s["code"].unflatten(1, (-1, G)).float() - p[..., 1:2]) * p[..., 0:1]).flatten(1)
    return (s["x"].float() @ w.T).to(s["y"].dtype)


def _rows(s):
    """For each new row: its sequence, its index among the sequence's new rows, its position."""
    ind, lens = s["ind"].long(), s["lens"].long()[s["slots"].long()]
    row = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(ind[1:], row, right=True)
    i = row - ind[seq]
    return seq, i, lens[seq] - (ind[seq + 1] - ind[seq]) + i


def _plain_append(s):
    c = s["case"]
    seq, _, pos = _rows(s)
    page = s["tables"].long()[s["slots"].long()[seq], pos // c["page"]]
    at = pos % c["page"]
    kc, kp = quantise(s["kn"].unflatten(1, (c["Hkv"], c["D"])), c["G"])
    vc, vp = quantise(s["vn"].unflatten(1, (c["Hkv"], c["D"])), c["G"])
    s["kc"][page, :, at], s["kp"][page, :, at], s["vc"][page, :, at], s["vp"][page, :, at] = kc, kp, vc, vp
    return page, at


def _plain_attn(s):
    c = s["case"]
    H, R, D, P = c["Hkv"], c["rep"], c["D"], c["page"]
    _plain_append(s)
    seq, i, pos = _rows(s)
    slots, T = s["slots"].long(), s["longest"]
    tok = torch.arange(T, device=DEV)
    page = s["tables"].long()[slots][:, tok // P].clamp_min(0)              # [B, T]
    at = (tok % P).expand_as(page)
    live = (tok[None] < s["lens"].long()[slots][:, None])[..., None, None]
    k = torch.where(live, values(s["kc"][page, :, at], s["kp"][page, :, at], c["G"]), 0.0)  # [B, T, H, D]
    v = torch.where(live, values(s["vc"][page, :, at], s["vp"][page, :, at], c["G"]), 0.0)
    B = k.shape[0]
    q = torch.zeros(B, s["most"], H, R, D, device=DEV)
    q[seq, i] = s["q"].float().view(-1, H, R, D)
    far = torch.zeros(B, s["most"], device=DEV, dtype=torch.long)
    far[seq, i] = pos
    x = torch.einsum("bqhrd,bthd->bqhrt", q, k) * (1.0 / math.sqrt(D))
    see = tok[None, None] <= far[..., None]
    if c["window"]:
        see = see & (tok[None, None] > far[..., None] - c["window"])
    x = x.masked_fill(~see[:, :, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    o = torch.einsum("bqhrt,bthd->bqhrd", e / z, v)
    lse = (m + z.log())[..., 0]
    return {"o": o[seq, i].flatten(1).half(), "lse": lse[seq, i].flatten(1)}


def _plain_read(s):
    page, at = _plain_append(s)
    G = s["case"]["G"]
    return {"k": values(s["kc"][page, :, at], s["kp"][page, :, at], G).flatten(1).half(), "v": values(s["vc"][page, :, at], s["vp"][page, :, at], G).flatten(1).half()}


def _free_pages(refs):
    """The free pages in ascending order, then zeros; and their number."""
    n = refs.shape[0]
    free = refs == 0
    rank = torch.where(free, free.cumsum(0) - 1, n)
    return torch.zeros(n + 1, device=DEV, dtype=torch.long).scatter_(0, rank, torch.arange(n, device=DEV))[:n], free.sum()


def _plain_fork(s, deep):
    src, dst, P = s["src"].long(), s["dst"].long(), s["case"]["page"]
    need = (s["lens"][src].long() + P - 1) // P
    old = s["tables"][src].long()
    has = torch.arange(s["width"], device=DEV)[None] < need[:, None]
    if deep:
        pages, n_free = _free_pages(s["refs"])
        k = (has.flatten().cumsum(0) - 1).view_as(has).clamp_min(0)
        new = torch.where(has, pages[k.clamp_max(pages.shape[0] - 1)], -1)
        to = torch.where(has, new, old[:, :1]).flatten()                    # places without a page copy one onto itself
        s["pool"][:, to] = s["pool"][:, torch.where(has, old, old[:, :1]).flatten()]
        s["refs"].index_add_(0, to, has.flatten().int())
        short = (has.sum() - n_free).clamp_min(0)
    else:
        new = torch.where(has, old, -1)
        s["refs"].index_add_(0, new.clamp_min(0).flatten(), has.flatten().int())
        short = has.sum() * 0
    s["tables"][dst] = new.int()
    s["lens"][dst] = s["lens"][src]
    return short.int().view(1)


def _plain_extend(s, slots, add):
    P, slots, width = s["case"]["page"], slots.long(), s["width"]
    n = slots.shape[0]
    length = s["lens"][slots].long()
    have, need = (length + P - 1) // P, (length + add.long() + P - 1) // P
    last = s["tables"][slots, (have - 1).clamp_min(0)].long()
    part = (length % P != 0) & (add > 0)
    same = (last[:, None] == last[None]) & part[:, None] & part[None]
    before = (same & (torch.arange(n, device=DEV)[None] < torch.arange(n, device=DEV)[:, None])).sum(1)
    cow = part & (s["refs"][last.clamp_min(0)] - before > 1)
    fresh = need - have + cow
    start = fresh.cumsum(0) - fresh
    pages, n_free = _free_pages(s["refs"])
    col = torch.arange(width, device=DEV)[None]
    first = have - cow.long()
    new = (col >= first[:, None]) & (col < need[:, None])
    got = pages[(start[:, None] + col - first[:, None]).clamp(0, pages.shape[0] - 1)]
    table = torch.where(new, got, s["tables"][slots].long())
    to = torch.where(cow, pages[start.clamp_max(pages.shape[0] - 1)], last)
    s["pool"][:, to] = s["pool"][:, last]
    s["refs"].index_add_(0, last, -cow.int())
    s["refs"].index_add_(0, got.flatten(), new.flatten().int())
    s["tables"][slots] = table.int()
    s["lens"][slots] = (length + add).int()
    return (fresh.sum() - n_free).clamp_min(0).int().view(1)


def _plain_free(s, slots):
    slots, P = slots.long(), s["case"]["page"]
    has = torch.arange(s["width"], device=DEV)[None] < ((s["lens"][slots].long() + P - 1) // P)[:, None]
    s["refs"].index_add_(0, s["tables"][slots].long().clamp_min(0).flatten(), -has.flatten().int())
    s["tables"][slots] = -1
    s["lens"][slots] = 0


def _plain_compact(s):
    refs = s["refs"].long()
    n = refs.shape[0]
    ids, live = torch.arange(n, device=DEV), refs > 0
    count = live.sum()
    mover, hole = live & (ids >= count), ~live & (ids < count)
    end = torch.full((1,), n, device=DEV)
    holes = torch.zeros(n + 1, device=DEV, dtype=torch.long).scatter_(0, torch.where(hole, hole.cumsum(0) - 1, end), ids)
    movers = torch.zeros(n + 1, device=DEV, dtype=torch.long).scatter_(0, torch.where(mover, mover.cumsum(0) - 1, end), ids)
    to = torch.where(mover, holes[(mover.cumsum(0) - 1).clamp_min(0)], ids)
    of = torch.where(hole, movers[(hole.cumsum(0) - 1).clamp_min(0)], ids)
    s["pool"].copy_(s["pool"].index_select(1, of))
    s["refs"].copy_(torch.where(hole, refs[of], torch.where(mover, 0, refs)))
    table = s["tables"].long()
    s["tables"].copy_(torch.where(table >= 0, to[table.clamp_min(0)], -1))
    return count.int().view(1)


def _plain_pages(s):
    op = s["case"]["op"]
    if op == "compact":
        _plain_free(s, s["gone"])
        return _plain_compact(s)
    short = _plain_fork(s, op == "copy")
    return short if op == "copy" else _plain_extend(s, s["dst"], s["add"])


# ---- the framework's calls --------------------------------------------------------------------------------------------------
def _own(s):
    """The package, and what a program that serves keeps: the cache's handle and a workspace."""
    ph = importlib.import_module("phobos-lang_b200")
    if "cache" not in s and s["case"]["op"] != "gemv":
        c = s["case"]
        s["cache"] = ph.Kv4Cache(s["pool"], s["refs"], s["tables"], s["lens"], kv_heads=c["Hkv"], head_dim=c["D"], group=c["G"], page_tokens=c["page"])
        need = (ph.kv4_attention_workspace_bytes(s["cache"], s["q"].shape[0], c["B"], c["Hkv"] * c["rep"]) if c["op"] == "attn"
                else 0 if c["op"] == "append" else ph.kv4_pages_workspace_bytes(s["cache"]))
        s["ws"] = torch.empty(max(256, need), device=DEV, dtype=torch.uint8)
    return ph


def _own_pages(ph, s):
    op, cache, count, ws = s["case"]["op"], s["cache"], s["count"], s["ws"]
    if op == "compact":
        ph.kv4_free(cache, s["gone"])
        ph.kv4_compact(cache, count, workspace=ws)
    else:
        ph.kv4_fork(cache, s["src"], s["dst"], count, deep=op == "copy", workspace=ws)
        if op == "branch":
            ph.kv4_extend(cache, s["dst"], s["add"], count, workspace=ws)
    return count


def run(s):
    op = s["case"]["op"]
    if op == "gemv":
        if own:
            _own(s).gemv_q4(s["x"], s["packed"], s["y"], s["case"]["G"])
            return s["y"]
        return _plain_gemv(s)
    if op in ("attn", "append"):
        if own:
            ph, cache = _own(s), s["cache"]
            ph.kv4_append(cache, 0, s["kn"], s["vn"], s["slots"], s["ind"])
            if op == "append":
                ph.kv4_read(cache, 0, s["kr"], s["vr"], s["slots"], s["ind"])
                return {"k": s["kr"], "v": s["vr"]}
            ph.kv4_attention(cache, 0, s["q"], s["o"], 1.0 / math.sqrt(s["case"]["D"]), s["slots"], s["ind"], lse=s["lse"], window=s["case"]["window"], workspace=s["ws"])
            return {"o": s["o"], "lse": s["lse"]}
        return _plain_attn(s) if op == "attn" else _plain_read(s)
    s["now"].copy_(s["meta"])
    count = _own_pages(_own(s), s) if own else _plain_pages(s)
    return {"count": count, "refs": s["refs"], "lens": s["lens"], "tables": s["tables"], "pool": s["pool"]}


# ---- what it costs, and the exact values --------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "gemv":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": N * K // 2 + 4 * N * K // case["G"] + 2 * M * K + M * N * (2 if case["out"] == "f16" else 4), "flops": 2 * M * N * K}
    token = case["Hkv"] * (case["D"] + 8 * case["D"] // case["G"]) if "Hkv" in case else 0  # a cached token's bytes, K and V
    if op in ("attn", "append"):
        length, new = (t.double() for t in _lengths(case, 0))
        rows, kv = float(new.sum()), case["Hkv"] * case["D"] * 4
        if op == "append":
            return {"bytes": rows * (2 * kv + 2 * token), "flops": rows * kv}
        w = case["window"] or 1 << 40
        lo, hi = length - new + 1, length                                    # a row at the p-th place sees min(p, w) tokens
        upto = lambda p: torch.where(p <= w, p * (p + 1) / 2, w * (w + 1) / 2 + (p - w) * w)  # noqa: E731
        pairs = float((upto(hi) - upto(lo - 1)).sum())
        seen = float(torch.minimum(length, new - 1 + w).sum())
        q = rows * case["Hkv"] * case["rep"] * case["D"]
        return {"bytes": seen * token + rows * (kv + token) + 4 * q + 4 * q / case["D"], "flops": 4 * case["D"] * case["Hkv"] * case["rep"] * pairs}
    length = _pool_lengths(case)
    need, P = (length + case["page"] - 1) // case["page"], case["page"]
    if op == "copy":
        moved = int(need.sum())
    elif op == "branch":
        moved = int((length % P != 0).sum())
    else:
        live = int(need.sum()) - int(need[: (case["n"] + 1) // 2].sum())
        moved = int(live * (1 - live / case["pages"]))                       # live pages that stand behind the first `live` places
    meta = 4 * (case["pages"] + 2 * case["n"] * (-(-(case["len"] + case["add"]) // P) + 2))
    return {"bytes": 2 * moved * case["layers"] * P * token + 2 * meta, "flops": 0}


def _exact_quantised(x, G):
    g = x.double().unflatten(-1, (-1, G))
    lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
    step = ((hi - lo) / 15).half().double()
    return torch.where(step > 0, lo + step * torch.round((g - lo) / step).clamp(0, 15), lo).flatten(-2)


def exact(case, seed):
    op = case["op"]
    if op == "gemv":
        x, code, par = _gemv_inputs(case, seed)
        s, z = par[..., 0].double(), par[..., 1].double()
        y = torch.zeros(case["M"], case["N"], device=DEV, dtype=torch.float64)
        for k in range(case["K"] // case["G"]):
            cut = slice(k * case["G"], (k + 1) * case["G"])
            y += x[:, cut].double() @ ((code[:, cut].double() - z[:, k:k + 1]) * s[:, k:k + 1]).T
        return y
    if op not in ("attn", "append"):
        return None
    i = _cache_inputs(case, seed)
    H, R, D, G, P = case["Hkv"], case["rep"], case["D"], case["G"], case["page"]
    kn, vn = (_exact_quantised(i[x].unflatten(1, (H, D)), G) for x in ("kn", "vn"))
    if op == "append":
        return {"k": kn.flatten(1), "v": vn.flatten(1)}
    out, lse, ind = [], [], i["ind"].tolist()
    for b, slot in enumerate(i["slots"].tolist()):
        n, length = ind[b + 1] - ind[b], int(i["lens"][slot])
        pages = i["tables"][slot, :-(-length // P)].long()
        q = i["q"][ind[b]:ind[b + 1]].double().view(n, H, R, D)
        pos = torch.arange(length - n, length, device=DEV)
        tok = torch.arange(length, device=DEV)
        hide = tok[None] > pos[:, None]
        if case["window"]:
            hide |= tok[None] <= pos[:, None] - case["window"]
        for h in range(H):
            kv = []
            for c, p, fresh in (("kc", "kp", kn), ("vc", "vp", vn)):
                code = i[c][pages, h].double().view(-1, D // G, G)[:length]
                par = i[p][pages, h].double().view(-1, D // G, 2)[:length]
                x = (par[..., 1:2] + par[..., 0:1] * code).flatten(1)
                x[length - n:] = fresh[ind[b]:ind[b + 1], h]
                kv.append(x)
            a = (q[:, h].reshape(n * R, D) @ kv[0].T / math.sqrt(D)).view(n, R, length).masked_fill(hide[:, None], float("-inf"))
            lse.append(torch.logsumexp(a, -1))
            out.append((torch.exp(a - lse[-1][..., None]).reshape(n * R, length) @ kv[1]).view(n, R, D))
    split = lambda parts, last: torch.cat([torch.stack(parts[b * H:(b + 1) * H], 1).flatten(1) for b in range(case["B"])])  # noqa: E731
    return {"o": split(out, D), "lse": split(lse, 1)}
