"""Cases and plain forms of the operators around the paged 4-bit key/value cache (include/l3m_kernels.h).

  plan    l3m_kv4_plan_dev: block tables, free list, slot map and positions of one step from the requests' lengths
  qkv     l3m_qkv_rope_dev: RMS norm of each query and key head and the position rotation in one pass, keys and values
          written to the cache in 4 bits (read back by l3m_kv4_load_dev), or the rotated keys returned without a cache
  attend  l3m_kv4_attend_dev: causal attention of each request's newest tokens over its pages of the cache

`own` chooses what run() computes: False the plain form in torch, True the library's entry points.

The cache is made of tiles: 16 tokens of one head, groups of 32 of its head_dim values (the last group padded with
zeros). With NG groups a tile holds, in this order,
  key codes     [16 tokens][4 parts t][NG groups j][4 bytes]   nibble i (low first) is the value at 32*j + 8*t + i
  value codes   [16 tokens][8 parts g][NG groups j][2 bytes]   nibble i is the value at 32*j + 4*g + i
  key scales    [16 tokens][NG], value scales [16 tokens][NG]  f16 (q4_0) or e8m0 (mxfp4)
and the tiles lie [page][head][page / 16]. q4_0: (nibble - 8) * scale; mxfp4: e2m1(nibble) * 2^(scale - 127).
"""
import math

import numpy as np
import torch

own = False

TILE, GROUP = 16, 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DT = {"f32": 0, "bf16": 1, "q4_0": 3, "mxfp4": 4}
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
DEV = "cuda"


# ---- cases

def listed():
    return [
        # one decode step of a small server: 24 requests, one token each, a few of them over a page's end, two just ended
        dict(name="plan-decode-24", op="plan", reqs=24, prompt=False, max_kv=4096, page=32, odd=True),
        # a large step: 512 requests, a quarter of them new prompts, 64-token pages
        dict(name="plan-prefill-512", op="plan", reqs=512, prompt=True, max_kv=16384, page=64, odd=True),
        # SmolLM2-135M's heads (9 over 3, 64 wide), no q/k norm, float activations, one decode step of 4 requests
        dict(name="qkv-decode-4-f32", op="qkv", dtype="f32", cache="q4_0", tokens=4, heads=9, kv_heads=3, dim=64, page=16, rope="pairs", norm=False, store=True),
        # a decode step of 128 requests, 32 heads over 8, normed
        dict(name="qkv-decode-128-bf16", op="qkv", dtype="bf16", cache="q4_0", tokens=128, heads=32, kv_heads=8, dim=128, page=64, rope="halves", norm=True, store=True),
        # a prompt chunk into an mxfp4 cache
        dict(name="qkv-chunk-8191-mx", op="qkv", dtype="bf16", cache="mxfp4", tokens=8191, heads=32, kv_heads=8, dim=128, page=64, rope="halves", norm=True, store=True),
        # the rotation without a cache, stories15M's 48-wide heads
        dict(name="qkv-rope-4000-f32", op="qkv", dtype="f32", cache="q4_0", tokens=4000, heads=6, kv_heads=6, dim=48, page=16, rope="pairs", norm=True, store=False),
        # latency: one short request, SmolLM2's heads in float
        dict(name="attend-1x200-f32", op="attend", dtype="f32", cache="q4_0", reqs=1, kv=200, ragged=False, new=1, heads=9, kv_heads=3, dim=64, page=16, window=0),
        # an ordinary decode batch: 16 requests of uneven lengths
        dict(name="attend-16x2000-mx", op="attend", dtype="bf16", cache="mxfp4", reqs=16, kv=2000, ragged=True, new=1, heads=32, kv_heads=8, dim=128, page=32, window=0),
        # a full decode batch
        dict(name="attend-64x8192", op="attend", dtype="bf16", cache="q4_0", reqs=64, kv=8192, ragged=True, new=1, heads=32, kv_heads=8, dim=128, page=64, window=0),
        # one long context: few rows, a long axis
        dict(name="attend-1x250001", op="attend", dtype="bf16", cache="q4_0", reqs=1, kv=250001, ragged=False, new=1, heads=16, kv_heads=2, dim=128, page=128, window=0),
        # five drafted tokens a request under a sliding window, 96-wide heads
        dict(name="attend-draft-32x5-f32", op="attend", dtype="f32", cache="mxfp4", reqs=32, kv=3000, ragged=True, new=5, heads=16, kv_heads=4, dim=96, page=16, window=1000),
        # prompt chunks over what is cached already
        dict(name="attend-chunk-2x1024", op="attend", dtype="bf16", cache="q4_0", reqs=2, kv=6000, ragged=True, new=1024, heads=32, kv_heads=8, dim=128, page=64, window=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "qkv", "qkv", "attend", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 48, 64, 128])
    if op == "plan":
        return dict(op="plan", reqs=_log(rng, 1, 700), prompt=rng.random() < 0.5, max_kv=_log(rng, 40, 16384), page=page, odd=True)
    dims = [16, 24, 32, 40, 48, 64, 80, 96, 112, 128, 160, 192, 256]
    kv_heads, group = rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([1, 2, 3, 4, 5, 8, 12])
    case = dict(op=op, dtype=rng.choice(["f32", "bf16"]), cache=rng.choice(["q4_0", "mxfp4"]), heads=kv_heads * group, kv_heads=kv_heads, dim=rng.choice(dims), page=page)
    width = (case["heads"] + 2 * kv_heads) * case["dim"]
    if op == "qkv":
        most = max(64, min(8191, 8191 * 6144 // width // (2 if case["dtype"] == "f32" else 1)))
        return dict(case, tokens=_log(rng, 1, most), rope=rng.choice(["pairs", "halves", "none"]), norm=rng.random() < 0.6, store=rng.random() < 0.75)
    new = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 700)])
    reqs = _log(rng, 1, 96 if new < 10 else 4)
    row = kv_heads * case["dim"]
    # below the largest listed cases: about half a gigabyte of cache, 100 GFLOP of products
    most = min(200000, int(2.5e8 / (row * reqs)), int(2.5e10 / (reqs * new * case["heads"] * case["dim"])))
    kv = max(new, _log(rng, 1, max(64, most)))
    return dict(case, reqs=reqs, kv=kv, ragged=rng.random() < 0.8, new=new, window=rng.choice([0, 0, 0, _log(rng, 1, 4096)]))


# ---- inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _tile_bytes(case):
    ng = -(-case["dim"] // GROUP)
    return ng * (512 + 32 * (2 if case["cache"] == "q4_0" else 1))


def _cache(case, n_pages, g):
    """A cache whose codes and scales are those of roughly normal keys and values."""
    ng, kv_heads, dim = -(-case["dim"] // GROUP), case["kv_heads"], case["dim"]
    z = torch.erfinv(torch.linspace(-0.998, 0.998, 4096, dtype=torch.float64)) * math.sqrt(2)     # normal quantiles
    if case["cache"] == "q4_0":
        code = (z * 2.9).round().clamp(-8, 7).long() + 8
    else:
        mag = torch.tensor(E2M1, dtype=torch.float64)
        code = (z.abs()[:, None] * 2.2 - mag).abs().argmin(1)
        code = code + 8 * ((z < 0) & (code > 0)).long()
    pick = torch.randint(0, 4096, (2, 4096), generator=torch.Generator().manual_seed(1))
    byte = (code[pick[0]] | code[pick[1]] << 4).to(torch.uint8).to(DEV)
    tiles = (n_pages, kv_heads, case["page"] // TILE)
    data = torch.empty(tiles + (_tile_bytes(case),), dtype=torch.uint8, device=DEV)
    data[..., :512 * ng] = byte[torch.randint(0, 4096, tiles + (512 * ng,), device=DEV, generator=g)]
    if dim % GROUP:                                                                              # the padding of the last group
        k, v = data[..., :256 * ng].view(*tiles, 16, 4, ng, 4), data[..., 256 * ng:512 * ng].view(*tiles, 16, 8, ng, 2)
        zero, real = 0x88 if case["cache"] == "q4_0" else 0, dim % GROUP
        k[..., real // 8:, ng - 1, :] = zero
        v[..., real // 4:, ng - 1, :] = zero
    n = tiles + (32 * ng,)
    if case["cache"] == "q4_0":
        s = torch.randn(n, device=DEV, generator=g).mul_(0.25).exp_().mul_(0.32) * (torch.randint(0, 2, n, device=DEV, generator=g) * 2 - 1)
        data[..., 512 * ng:] = s.to(torch.float16).view(torch.uint8)
    else:
        data[..., 512 * ng:] = torch.randint(125, 128, n, device=DEV, generator=g).to(torch.uint8)
    return data


def _lengths(case, seed):
    """Lengths of an attention batch, newest tokens included, and how many of them are new."""
    r = np.random.default_rng(int(seed) + 5)
    n, kv, new = case["reqs"], case["kv"], case["new"]
    lens = r.integers(max(new, kv // 3), kv + 1, n) if case["ragged"] else np.full(n, kv)
    lens[r.integers(n)] = kv
    news = np.random.default_rng(n).integers(max(1, new // 2), new + 1, n) if case["ragged"] else np.full(n, new)      # the rows of q: the same for every seed
    news[0] = new
    return lens, news


def prepare(case, seed):
    state = {"plan": _prepare_plan, "qkv": _prepare_qkv, "attend": _prepare_attend}[case["op"]](case, seed)
    state["case"] = case
    if own:
        _handles(state)
    return state


def _prepare_plan(case, seed):
    r, page, n = np.random.default_rng(int(seed)), case["page"], case["reqs"]
    kv = r.integers(0, case["max_kv"] + 1, n)
    new = np.ones(n, dtype=np.int64)
    most = n + 5                                                      # rows of the batch: those behind the last request are padding
    if case["prompt"]:
        fresh = r.permutation(n)[:n // 4]
        kv[fresh] = 0
        new[fresh] = r.integers(1, max(2, case["max_kv"] // 4), n // 4)
        most += n // 4 * (case["max_kv"] // 4)
    ended = r.random(n) < 0.08
    new[ended] = -1
    new[r.random(n) < 0.03] = 0
    blocks = -(-(case["max_kv"] + max(1, case["max_kv"] // 4)) // page) + 1
    held, after = -(-kv // page), -(-(kv + np.maximum(new, 0)) // page)
    need = int((after - held).sum())
    n_free = need + int(r.integers(0, 64))
    n_pages = n * blocks + 64
    order = r.permutation(n_pages)
    tables = np.full((n, blocks), -1, dtype=np.int64)
    live = np.arange(blocks)[None, :] < held[:, None]
    tables[live] = order[:int(held.sum())]
    free = np.full(n_pages, -1, dtype=np.int64)
    free[:n_free] = order[int(held.sum()):int(held.sum()) + n_free]
    return dict(kv_len=_ints(kv), new_len=_ints(new), tables=_ints(tables), free=_ints(free), n_free=_ints([n_free]), page=page, n_pages=n_pages,
                n_free_out=_ints([0]), q_start=_ints([0] * (n + 1)), kv_total=_ints([0] * n), slot=_ints([0] * most), pos=_ints([0] * most), status=_ints([0]))


def _prepare_qkv(case, seed):
    g, r = _gen(seed), np.random.default_rng(int(seed))
    t, h, kh, d, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
    n_pos, n_pages = 8192, -(-t // page) + 3
    x = torch.randn(t, (h + 2 * kh) * d, device=DEV, generator=g)
    x *= 1 + 3 * torch.rand((h + 2 * kh) * d, device=DEV, generator=g) ** 4                       # a few strong channels
    x = x.to(TORCH[case["dtype"]])
    angle = torch.arange(n_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    pos = r.integers(0, n_pos, t)
    pos[r.integers(t)] = 0
    state = dict(x=x, pos=_ints(pos), slot=_ints(r.permutation(n_pages * page)[:t]), rope=torch.stack((angle.cos(), angle.sin()), -1).float().to(DEV).contiguous(),
                 q_norm=1 + 0.2 * torch.randn(d, device=DEV, generator=g) if case["norm"] else None,
                 k_norm=1 + 0.2 * torch.randn(d, device=DEV, generator=g) if case["norm"] else None,
                 q_out=torch.zeros(t, h, d, dtype=x.dtype, device=DEV), status=_ints([0]))
    shape = (t, kh, d)
    if case["store"]:
        state["data"] = torch.zeros(n_pages, kh, page // TILE, _tile_bytes(case), dtype=torch.uint8, device=DEV)
        state["k_read"], state["v_read"] = torch.zeros(shape, dtype=x.dtype, device=DEV), torch.zeros(shape, dtype=x.dtype, device=DEV)
    else:
        state["k_out"] = torch.zeros(shape, dtype=x.dtype, device=DEV)
    return state


def _prepare_attend(case, seed):
    g, r = _gen(seed), np.random.default_rng(int(seed))
    lens, news = _lengths(case, seed)
    held = -(-lens // case["page"])
    n_pages, blocks = int(held.sum()) + 2, int(held.max())
    tables = np.full((case["reqs"], blocks), -1, dtype=np.int64)
    tables[np.arange(blocks)[None, :] < held[:, None]] = r.permutation(n_pages)[:int(held.sum())]
    q_start = np.concatenate(([0], np.cumsum(news)))
    q = torch.randn(int(q_start[-1]), case["heads"], case["dim"], device=DEV, generator=g).to(TORCH[case["dtype"]])
    return dict(q=q, out=torch.zeros_like(q), data=_cache(case, n_pages, g), tables=_ints(tables), q_start=_ints(q_start), kv_len=_ints(lens),
                max_q=int(news.max()), max_kv=int(lens.max()), scale=case["dim"] ** -0.5, status=_ints([0]))


# ---- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state)
    return {"plan": _plain_plan, "qkv": _plain_qkv, "attend": _plain_attend}[op](state)


def _plain_plan(s):
    kv, new, page, n_pages = s["kv_len"].long(), s["new_len"].long(), s["page"], s["n_pages"]
    tables, free, (n, blocks), most = s["tables"].long(), s["free"].long(), s["tables"].shape, s["slot"].numel()
    held, count = (kv + page - 1) // page, new.clamp(min=0)
    after = (kv + count + page - 1) // page
    good = (kv >= 0) & (after <= blocks)
    # the pages of ended requests go back on the stack, in request order
    col = torch.arange(blocks, device=DEV)
    gone = torch.where(good & (new < 0), held, 0)
    before = s["n_free"].long() + gone.cumsum(0) - gone
    at = torch.where(col[None, :] < gone[:, None], before[:, None] + col, n_pages)
    stack = torch.cat((free, free.new_zeros(1))).scatter_(0, at.reshape(-1), tables.reshape(-1))[:n_pages]
    top = s["n_free"].long() + gone.sum()
    # new pages come off its top, in request order
    need = torch.where(good & (count > 0), after - held, 0)
    upto = need.cumsum(0)
    q_start = torch.cat((count.new_zeros(1), count.cumsum(0)))
    served = good & (new >= 0) & ((need == 0) | (upto <= top)) & (q_start[1:] <= most)
    nth = (upto - need)[:, None] + col - held[:, None]
    fresh = (col[None, :] >= held[:, None]) & (col[None, :] < after[:, None]) & (served & (need > 0))[:, None]
    tables = torch.where(fresh, stack[(top - 1 - nth).clamp(0, n_pages - 1)], tables)
    left = top - torch.where(served, upto, 0).amax()
    # every token's request, position and slot
    token = torch.arange(most, device=DEV)
    req = torch.searchsorted(q_start, token, right=True) - 1
    real = (req < n) & (token < q_start[-1])
    req = req.clamp(max=n - 1)
    real &= served[req]
    pos = kv[req] + token - q_start[req]
    slot = tables[req, (pos // page).clamp(0, blocks - 1)] * page + pos % page
    return [tables.int(), stack.int(), left.int(), q_start.int(), torch.where(served, kv + count, 0).int(), torch.where(real, slot, -1).int(), torch.where(real, pos, -1).int()]


def _rotate(x, s, turn, kind):
    """x [tokens, heads, dim] turned by its position, in x's precision."""
    if kind == "none":
        return x
    c, n = turn[..., 0][:, None], turn[..., 1][:, None]
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if kind == "pairs" else (x[..., :half], x[..., half:])
    a, b = a * c - b * n, a * n + b * c
    return torch.stack((a, b), -1).flatten(-2) if kind == "pairs" else torch.cat((a, b), -1)


def _quantised(u, factor, kind):
    """The values that 4 bits hold of u * factor (u [..., dim], one factor a row), in 64 bits. q4_0's codes do not depend on the
    factor and are taken before it, so that ties between values are exact."""
    dim, pad = u.shape[-1], -u.shape[-1] % GROUP
    u = torch.nn.functional.pad(u, (0, pad)).unflatten(-1, (-1, GROUP))
    factor = factor[..., None]
    mag = u.abs()
    top = mag.amax(-1, keepdim=True)
    if kind == "q4_0":
        first = torch.where(mag == top, torch.arange(GROUP, device=DEV), GROUP).amin(-1, keepdim=True)
        d = u.gather(-1, first) / -8                                   # the value of largest magnitude gets code 0
        code = torch.where(d != 0, torch.floor(u / torch.where(d != 0, d, 1) + 8.5), 8).clamp(0, 15)
        scale = (d * factor).float().clamp(-65504, 65504).half().double()
        return ((code - 8) * scale).flatten(-2)[..., :dim]
    y = u * factor
    top = top * factor
    e = torch.where(top > 0, torch.frexp(top).exponent - 1 + 125, 0).clamp(0, 254)
    step = torch.ldexp(torch.ones_like(top), e - 127)
    v, mags = (y / step).abs(), torch.tensor(E2M1, dtype=y.dtype, device=DEV)
    code = (v[..., None] > (mags[1:] + mags[:-1]) / 2).sum(-1)           # ties go to the smaller magnitude
    return (mags[code] * step * torch.where(y < 0, -1, 1)).flatten(-2)[..., :dim]


def _plain_qkv(s):
    case, x = s["case"], s["x"]
    t, h, kh, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    q, k, v = (a.unflatten(-1, (-1, d)) for a in x.split((h * d, kh * d, kh * d), -1))
    turn = s["rope"][s["pos"].long()]

    def normed(a, w):                                                  # the row's factor, and what it multiplies
        if w is None:
            return torch.ones_like(a[..., :1]), a
        return torch.rsqrt(a.square().mean(-1, keepdim=True) + 1e-6), a * w.to(a.dtype)

    f, u = normed(q.float(), s["q_norm"])
    q_out = (_rotate(u, s, turn, case["rope"]) * f).to(x.dtype)
    if not case["store"]:
        f, u = normed(k.float(), s["k_norm"])
        return [q_out, (_rotate(u, s, turn, case["rope"]) * f).to(x.dtype)]
    f, u = normed(k.double(), s["k_norm"])                             # codes and scales lie next to borders: 64 bits
    k_held = _quantised(_rotate(u, s, turn.double(), case["rope"]), f, case["cache"])
    v_held = _quantised(v.double(), torch.ones_like(f), case["cache"])
    return [q_out, k_held.float().to(x.dtype), v_held.float().to(x.dtype)]


def _values(codes, scales, kind):
    """codes [..., 16, 32 * NG] and scales (their bytes) [..., 16 * NG * width] as numbers in 32 bits."""
    if kind == "q4_0":
        return (codes.float() - 8).unflatten(-1, (-1, GROUP)) * scales.contiguous().view(torch.float16).float().unflatten(-1, (TILE, -1))[..., None]
    lut = torch.tensor(E2M1 + tuple(-m for m in E2M1), device=DEV)
    return lut[codes.int()].unflatten(-1, (-1, GROUP)) * torch.ldexp(torch.ones((), device=DEV), scales.int() - 127).unflatten(-1, (TILE, -1))[..., None]


def _plain_rows(s):
    """The requests' keys and values in 32 bits, padded to the longest: [request, head, token, dim]."""
    case = s["case"]
    ng, wide = -(-case["dim"] // GROUP), 16 * -(-case["dim"] // GROUP) * (2 if case["cache"] == "q4_0" else 1)
    tiles = s["data"][s["tables"].long().clamp(min=0)].transpose(1, 2)   # [request, head, block, tile, bytes]
    rows = []
    for at, parts, size, sc in ((0, 4, 4, 512 * ng), (256 * ng, 8, 2, 512 * ng + wide)):
        b = tiles[..., at:at + 256 * ng].unflatten(-1, (TILE, parts, ng, size))
        n = torch.stack((b & 15, b >> 4), -1).flatten(-2).transpose(-3, -2).flatten(-3)
        rows.append(_values(n, tiles[..., sc:sc + wide], case["cache"]).flatten(-2).flatten(2, 4)[..., :case["dim"]])
    return rows


def _plain_attend(s):
    case, q = s["case"], s["q"]
    kh, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    k, v = _plain_rows(s)
    start, kv = s["q_start"].long(), s["kv_len"].long()
    news = start[1:] - start[:-1]
    i = torch.arange(s["max_q"], device=DEV)
    row = (start[:-1, None] + i).clamp(max=q.shape[0] - 1)                                            # past a request's last row: any row, never taken
    x = q.float()[row].unflatten(2, (kh, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)                # [request, kv head, token * group, dim]
    scores = (x * s["scale"]) @ k.transpose(-1, -2)
    at = (kv - news)[:, None] + i                                                                    # the queries' positions
    j = torch.arange(k.shape[2], device=DEV)
    seen = (j <= at[..., None]) & (j < kv[:, None, None])
    if case["window"]:
        seen &= j > at[..., None] - case["window"]
    seen = seen[:, None, :, None, :].expand(-1, kh, -1, group, -1).flatten(2, 3)
    scores = scores.masked_fill_(~seen, -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = torch.exp(scores.sub_(torch.where(most == -math.inf, 0.0, most)))
    total = p.sum(-1, keepdim=True)
    # a token that nobody sees may hold anything: its values are left out, not multiplied by zero
    o = (p @ v.masked_fill_((j >= kv[:, None])[:, None, :, None], 0.0)) / torch.where(total > 0, total, 1.0)
    o = o.unflatten(2, (-1, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    token = torch.arange(q.shape[0], device=DEV)
    req = torch.searchsorted(start, token, right=True) - 1
    return o[req, token - start[req]].to(q.dtype)


# ---- the library's calls

def _ptr(t):
    return None if t is None else t.data_ptr()


def _handles(s):
    """What a user's program keeps: the library, the cache's handle and the calls' argument blocks."""
    import l3m_b200 as l3m
    case, s["lib"] = s["case"], l3m.lib()
    if case["op"] == "plan":
        s["call"] = l3m.Kv4Plan(n_req=s["kv_len"].numel(), max_blocks=s["tables"].shape[1], max_tokens=s["slot"].numel(), page=s["page"], n_pages=s["n_pages"],
                                kv_len=_ptr(s["kv_len"]), new_len=_ptr(s["new_len"]), tables=_ptr(s["tables"]), free_pages=_ptr(s["free"]), n_free=_ptr(s["n_free"]),
                                n_free_out=_ptr(s["n_free_out"]), q_start=_ptr(s["q_start"]), kv_total=_ptr(s["kv_total"]), slot=_ptr(s["slot"]), pos=_ptr(s["pos"]),
                                status=_ptr(s["status"]))
        return
    dt, d, kh = DT[case["dtype"]], case["dim"], case["kv_heads"]
    cache = l3m.Kv4(data=_ptr(s.get("data")), dtype=DT[case["cache"]], n_pages=s["data"].shape[0] if "data" in s else 0, page=case["page"], n_kv_heads=kh, head_dim=d)
    s["cache"] = cache
    if case["op"] == "qkv":
        x, h, size, wide = s["x"], case["heads"], s["x"].element_size(), s["x"].shape[1]
        base = _ptr(x)
        s["call"] = l3m.Qkv(dtype=dt, n_tokens=case["tokens"], n_heads=h, n_kv_heads=kh, head_dim=d, rope={"none": 0, "pairs": 1, "halves": 2}[case["rope"]], rot_dim=d,
                            n_pos=s["rope"].shape[0], eps=1e-6, q_norm=_ptr(s["q_norm"]), k_norm=_ptr(s["k_norm"]), rope_table=_ptr(s["rope"]), pos=_ptr(s["pos"]), slot=_ptr(s["slot"]),
                            q=base, k=base + h * d * size, v=base + (h + kh) * d * size, q_ld=wide, k_ld=wide, v_ld=wide, q_out=_ptr(s["q_out"]), k_out=_ptr(s.get("k_out")),
                            q_out_ld=h * d, k_out_ld=kh * d, status=_ptr(s["status"]))
        return
    q = s["q"]
    s["call"] = l3m.Kv4Attend(dtype=dt, n_heads=case["heads"], n_req=case["reqs"], max_blocks=s["tables"].shape[1], max_q=s["max_q"], max_kv=s["max_kv"], window=case["window"],
                              scale=s["scale"], q=_ptr(q), out=_ptr(s["out"]), q_ld=q.stride(0), out_ld=s["out"].stride(0), q_start=_ptr(s["q_start"]), kv_len=_ptr(s["kv_len"]),
                              tables=_ptr(s["tables"]), status=_ptr(s["status"]))
    s["scratch"] = torch.empty(max(16, s["lib"].l3m_kv4_attend_scratch(cache, s["call"])), dtype=torch.uint8, device=DEV)
    s["call"].scratch, s["call"].scratch_bytes = _ptr(s["scratch"]), s["scratch"].numel()


def _own(s):
    case, lib, stream = s["case"], s["lib"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "plan":
        rc = lib.l3m_kv4_plan_dev(s["call"], stream)
        out = [s["tables"], s["free"], s["n_free_out"], s["q_start"], s["kv_total"], s["slot"], s["pos"]]
    elif case["op"] == "attend":
        rc = lib.l3m_kv4_attend_dev(s["cache"], s["call"], stream)
        out = s["out"]
    elif case["store"]:
        rc = lib.l3m_qkv_rope_dev(s["cache"], s["call"], stream)
        rc = rc or lib.l3m_kv4_load_dev(s["cache"], s["call"].dtype, _ptr(s["k_read"]), _ptr(s["v_read"]), _ptr(s["slot"]), case["tokens"], stream)
        out = [s["q_out"], s["k_read"], s["v_read"]]
    else:
        rc = lib.l3m_qkv_rope_dev(None, s["call"], stream)
        out = [s["q_out"], s["k_out"]]
    if rc:
        raise RuntimeError(lib.l3m_cuda_error().decode())
    return out


# ---- what a pass cannot do without

def work(case):
    if case["op"] == "plan":
        n, blocks = case["reqs"], -(-case["max_kv"] // case["page"])
        new = n * 0.75 + n * 0.25 * case["max_kv"] / 8 if case["prompt"] else n
        return {"bytes": 16 * n + 8 * new + 4 * n * blocks * 0.08, "flops": 0}
    size, row = 4 if case["dtype"] == "f32" else 2, case["dim"] / 2 + -(-case["dim"] // GROUP) * (2 if case["cache"] == "q4_0" else 1)
    kh = case["kv_heads"]
    if case["op"] == "qkv":
        t, h, d = case["tokens"], case["heads"], case["dim"]
        kept = t * kh * (2 * row + 2 * d * size) if case["store"] else t * kh * d * size
        read = t * (h + (2 if case["store"] else 1) * kh) * d * size
        turn = 0 if case["rope"] == "none" else min(t, 8192) * d * 4
        return {"bytes": read + t * h * d * size + kept + turn + 8 * t, "flops": t * (h + kh) * d * 8}
    lens, news = _lengths(case, 0)
    seen = np.minimum(lens, case["window"] + news - 1) if case["window"] else lens                    # cached tokens that some query of the request sees
    first = lens - news
    if case["window"]:
        pairs = sum(int(np.minimum(np.arange(f, f + n) + 1, case["window"]).sum()) for f, n in zip(first, news))
    else:
        pairs = sum(int(n * f + n * (n + 1) // 2) for f, n in zip(first, news))
    t = int(news.sum())
    return {"bytes": float(seen.sum()) * kh * 2 * row + 2 * t * case["heads"] * case["dim"] * size, "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# ---- the definition in 64 bits, request by request and value by value

def exact(case, seed):
    if case["op"] == "plan":
        return None                                                    # whole numbers
    return {"qkv": _exact_qkv, "attend": _exact_attend}[case["op"]](prepare(case, seed))


def _exact_qkv(s):
    case = s["case"]
    t, h, kh, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    x, pos = s["x"].double().cpu().numpy().reshape(t, h + 2 * kh, d), s["pos"].cpu().numpy()
    turn = s["rope"].double().cpu().numpy()[pos]
    dims = np.arange(d)
    if case["rope"] == "pairs":
        mate, which, sign = dims ^ 1, dims // 2, np.where(dims % 2, 1.0, -1.0)
    else:
        mate, which, sign = (dims + d // 2) % d, dims % (d // 2), np.where(dims < d // 2, -1.0, 1.0)
    c, n = turn[:, which, 0][:, None], turn[:, which, 1][:, None] * sign

    def turned(a, w):
        f = np.ones(a.shape[:2]) if w is None else 1 / np.sqrt((a * a).mean(-1) + 1e-6)
        a = a if w is None else a * w.double().cpu().numpy()
        return f, a if case["rope"] == "none" else a * c + a[..., mate] * n

    def held(u, f):
        out = np.empty_like(u)
        for lo in range(0, d, GROUP):
            g = u[..., lo:lo + GROUP]
            at = np.abs(g).argmax(-1)[..., None]
            if case["cache"] == "q4_0":
                step = np.take_along_axis(g, at, -1) / -8.0
                code = np.where(step == 0, 8.0, np.clip(np.floor(np.divide(g, step, out=np.zeros_like(g), where=step != 0) + 8.5), 0, 15))
                out[..., lo:lo + GROUP] = (code - 8) * np.clip((step * f[..., None]).astype(np.float32), -65504, 65504).astype(np.float16).astype(np.float64)
            else:
                y = g * f[..., None]
                top = np.abs(np.take_along_axis(y, at, -1))
                step = np.where(top > 0, 2.0 ** np.clip(np.floor(np.log2(np.where(top > 0, top, 1.0))) - 2, -127, 127), 2.0 ** -127)
                a, m = np.abs(y) / step, np.zeros_like(y)
                for low, high in zip(E2M1, E2M1[1:]):
                    m[a > (low + high) / 2] = high
                out[..., lo:lo + GROUP] = m * step * np.sign(y)
        return out

    f, u = turned(x[:, :h], s["q_norm"])
    q_out = u * f[..., None]
    f, u = turned(x[:, h:h + kh], s["k_norm"])
    if not case["store"]:
        return [q_out, u * f[..., None]]
    v = x[:, h + kh:]
    return [q_out, held(u, f), held(v, np.ones(v.shape[:2]))]


def _exact_attend(s):
    case = s["case"]
    dim, page, kh, group = case["dim"], case["page"], case["kv_heads"], case["heads"] // case["kv_heads"]
    ng = -(-dim // GROUP)
    d = torch.arange(dim, device=DEV)
    j, r = d // GROUP, d % GROUP
    bytes_k, shift_k = (r // 8 * ng + j) * 4 + r % 8 // 2, r % 2 * 4
    bytes_v, shift_v = 256 * ng + (r // 4 * ng + j) * 2 + r % 4 // 2, r % 2 * 4
    q4 = case["cache"] == "q4_0"
    start, lens = s["q_start"].tolist(), s["kv_len"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    mags = torch.tensor(E2M1 + tuple(-m for m in E2M1), dtype=torch.float64, device=DEV)
    for n, kv in enumerate(lens):
        new = start[n + 1] - start[n]
        first = max(0, kv - new - case["window"] + 1) if case["window"] else 0
        tok = torch.arange(first, kv, device=DEV)
        if not tok.numel():
            continue
        where, within = s["tables"][n].long()[tok // page], tok % page
        tile, row = within // TILE, within % TILE
        step = max(1, kh * int(2e8) // max(1, kh * tok.numel() * max(dim, new * group)))
        for lo in range(0, kh, step):
            heads = torch.arange(lo, min(kh, lo + step), device=DEV)[:, None]
            raw = s["data"][where[None], heads, tile[None]]                                            # [head, token, tile's bytes]
            at = torch.arange(tok.numel(), device=DEV)
            kv_rows = []
            for part, (off, shift, stride) in enumerate(((bytes_k, shift_k, 16 * ng), (bytes_v, shift_v, 16 * ng))):
                code = (raw[:, at[:, None], row[:, None] * stride + off] >> shift.to(torch.uint8)) & 15
                cell = 512 * ng + (part * 16 + row[:, None]) * ng * (2 if q4 else 1) + j * (2 if q4 else 1)
                lowb = raw[:, at[:, None], cell].int()
                if q4:
                    scale = (lowb | raw[:, at[:, None], cell + 1].int() << 8).to(torch.int16).view(torch.float16).double()
                    kv_rows.append((code.double() - 8) * scale)
                else:
                    kv_rows.append(mags[code.long()] * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=DEV), (lowb - 127).double()))
                del code, lowb
            del raw
            k, v = kv_rows
            x = s["q"][start[n]:start[n + 1]].double().unflatten(1, (kh, group))[:, lo:lo + step]     # [new, head, group, dim]
            z = torch.einsum("nhgd,htd->hngt", x, k) * s["scale"]
            p = torch.arange(kv - new, kv, device=DEV)[:, None]
            hide = tok > p
            if case["window"]:
                hide |= tok <= p - case["window"]
            z = torch.softmax(z.masked_fill_(hide[None, :, None], -math.inf), -1)
            out[start[n]:start[n + 1]].unflatten(1, (kh, group))[:, lo:lo + step] = torch.einsum("hngt,htd->nhgd", z, v)
    return out
