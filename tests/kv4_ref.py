"""Plain restatements, in 64 bits, of the operators around the paged 4-bit cache (include/l3m_kernels.h):
the definitions that tests/test_kv4.py and tests/test_gpu_kv4.py hold the library to."""
import numpy as np

MAGS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
Q4, MX = 3, 4
NO_PAGES, BAD_LENGTH, NO_ROOM, BAD_PAGE, BAD_POS = 1, 2, 4, 8, 16


def blocks(dim):
    return -(-dim // 32)


def tile_bytes(dtype, dim):
    return blocks(dim) * (512 + 32 * (2 if dtype == Q4 else 1))


def plan(kv_len, new_len, tables, free_pages, n_free, page, max_tokens):
    """One step's bookkeeping, request by request. Returns a dict of everything l3m_kv4_plan_dev writes."""
    tables, stack = tables.copy(), free_pages.copy()
    n, width = tables.shape
    n_pages, status = len(stack), 0
    top = min(max(n_free, 0), n_pages)
    if top != n_free:
        status |= BAD_LENGTH
    for r in range(n):
        held = -(-int(kv_len[r]) // page)
        if new_len[r] < 0 and kv_len[r] >= 0 and held <= width:
            for b in range(held):
                if top == n_pages:
                    status |= BAD_LENGTH
                    break
                stack[top] = tables[r, b]
                top += 1
    left, wanted = top, 0
    q_start, total = np.zeros(n + 1, np.int32), np.zeros(n, np.int32)
    slot, pos = np.full(max_tokens, -1, np.int32), np.full(max_tokens, -1, np.int32)
    for r in range(n):
        kv, count = int(kv_len[r]), max(int(new_len[r]), 0)
        held, after = -(-kv // page), -(-(kv + count) // page)
        q_start[r + 1] = q_start[r] + count
        bad = kv < 0 or after > width or kv + count + page > 2 ** 31 - 1
        need = 0 if bad else after - held
        first, wanted = wanted, wanted + need
        status |= BAD_LENGTH if bad else 0
        pages_ok, rows_ok = need == 0 or wanted <= top, q_start[r + 1] <= max_tokens
        status |= (0 if pages_ok else NO_PAGES) | (NO_ROOM if count and not rows_ok else 0)
        if bad or new_len[r] < 0 or not pages_ok or not rows_ok:
            continue
        for i in range(need):
            tables[r, held + i] = stack[top - 1 - first - i]
        left = min(left, top - wanted) if need else left
        total[r] = kv + count
        for i in range(count):
            pos[q_start[r] + i] = kv + i
            there = 0 <= tables[r, (kv + i) // page] < n_pages
            slot[q_start[r] + i] = tables[r, (kv + i) // page] * page + (kv + i) % page if there else -1
            status |= 0 if there else BAD_PAGE
    return dict(tables=tables, free_pages=stack, n_free_out=left, q_start=q_start, kv_total=total, slot=slot, pos=pos, status=status)


def normed_rotated(x, w, eps, turn, rope, rot):
    """(what the row's factor multiplies, the factor) of x [tokens, heads, dim] in 64 bits; turn [tokens, rot / 2, 2]."""
    f = np.ones(x.shape[:2]) if w is None else 1 / np.sqrt((x * x).mean(-1) + eps)
    u = x.copy() if w is None else x * w
    if rope:
        c, s = turn[:, None, :, 0], turn[:, None, :, 1]
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if rope == 1 else (slice(0, rot // 2), slice(rot // 2, rot))
        first, second = u[..., a] * c - u[..., b] * s, u[..., a] * s + u[..., b] * c
        u[..., a], u[..., b] = first, second
    return u, f


def quantise(u, f, dtype):
    """u [..., dim] times its row's factor f in 4 bits: (codes [..., 32 * NG], scale bits [..., NG])."""
    dim = u.shape[-1]
    g = np.concatenate((u, np.zeros(u.shape[:-1] + (-dim % 32,))), -1).reshape(u.shape[:-1] + (blocks(dim), 32))
    f = f[..., None]
    top = np.take_along_axis(g, np.abs(g).argmax(-1)[..., None], -1)[..., 0]
    if dtype == Q4:
        d = top / -8
        safe = np.where(d != 0, d, 1)
        code = np.where(d[..., None] != 0, np.clip(np.floor(g / safe[..., None] + 8.5), 0, 15), 8)
        bits = np.clip(np.where(d != 0, d * f, 0).astype(np.float32), -65504, 65504).astype(np.float16).view(np.uint16)
        return code.astype(np.uint8).reshape(u.shape[:-1] + (32 * blocks(dim),)), bits
    m = np.abs(top * f)
    e = np.where(m > 0, np.clip(np.frexp(np.where(m > 0, m, 1))[1] - 1 + 125, 0, 254), 0)
    y = g * f[..., None]
    v = np.abs(y) / np.ldexp(1.0, e - 127)[..., None]
    mag = (v[..., None] > (MAGS[1:] + MAGS[:-1]) / 2).sum(-1)
    return (mag + 8 * ((y < 0) & (mag > 0))).astype(np.uint8).reshape(u.shape[:-1] + (32 * blocks(dim),)), e.astype(np.uint8)


def values(codes, bits, dtype):
    """The numbers that codes [..., 32 * NG] and scale bits [..., NG] stand for, in 64 bits."""
    with np.errstate(invalid="ignore"):
        c = codes.reshape(codes.shape[:-1] + (codes.shape[-1] // 32, 32)).astype(np.int64)
        if dtype == Q4:
            out = (c - 8) * bits.view(np.float16).astype(np.float64)[..., None]
        else:
            out = np.where(c & 8, -1, 1) * MAGS[c & 7] * np.ldexp(1.0, bits.astype(np.int64) - 127)[..., None]
    return out.reshape(codes.shape)


def put_row(data, slot, head, codes, bits, is_v, dtype, dim, page):
    """Write one row into the cache's bytes [pages, heads, page / 16, tile]."""
    ng, width = blocks(dim), 2 if dtype == Q4 else 1
    tile = data[slot // page, head, slot % page // 16]
    row = slot % 16
    for d in range(32 * ng):
        j, i = d // 32, d % 32
        at = 256 * ng + row * 16 * ng + (i // 4 * ng + j) * 2 + i % 4 // 2 if is_v else row * 16 * ng + (i // 8 * ng + j) * 4 + i % 8 // 2
        tile[at] = (tile[at] & 0x0F) | codes[d] << 4 if i % 2 else (tile[at] & 0xF0) | codes[d]
    at = (512 + (16 * width if is_v else 0)) * ng + row * ng * width
    tile[at:at + ng * width] = bits.view(np.uint8)


def get_rows(data, slots, head, is_v, dtype, dim, page):
    """The values [len(slots), dim] of cache rows, in 64 bits."""
    ng, width = blocks(dim), 2 if dtype == Q4 else 1
    slots = np.asarray(slots, np.int64)
    tile = data[slots // page, head, slots % page // 16]
    row, n = slots % 16, np.arange(len(slots))
    d = np.arange(32 * ng)
    j, i = d // 32, d % 32
    at = 256 * ng + (i // 4 * ng + j) * 2 + i % 4 // 2 if is_v else (i // 8 * ng + j) * 4 + i % 8 // 2
    codes = tile[n[:, None], row[:, None] * 16 * ng + at] >> (i % 2 * 4).astype(np.uint8) & 15
    at = (512 + (16 * width if is_v else 0)) * ng + row * ng * width
    bits = tile[n[:, None], at[:, None] + np.arange(ng * width)]
    bits = np.ascontiguousarray(bits).view(np.uint16) if dtype == Q4 else bits
    return values(codes, bits, dtype)[:, :dim]


def attend(q, q_start, kv_len, tables, data, dtype, dim, page, n_kv, scale, window=0):
    """Attention in 64 bits: (out, spread) with q's shape [rows, heads, dim]. spread is sum(p |v|) / sum(p), what a relative
    error of the probabilities is multiplied by. Rows outside q_start's range are NaN; a query that sees nothing is 0."""
    rows, heads, _ = q.shape
    out, spread = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    n_pages = data.shape[0]
    for r in range(len(kv_len)):
        lo, hi, kv = q_start[r], q_start[r + 1], int(kv_len[r])
        if hi == lo:
            continue
        tok = np.arange(kv)
        ids = tables[r][tok // page] if kv else tok
        tok = tok[(ids >= 0) & (ids < n_pages)]
        slots = tables[r][tok // page].astype(np.int64) * page + tok % page if len(tok) else tok
        pos = kv - (hi - lo) + np.arange(hi - lo)
        seen = tok[None] <= pos[:, None]
        if window:
            seen &= tok[None] > pos[:, None] - window
        any_seen = seen.any(0)
        tok, slots, seen = tok[any_seen], slots[any_seen], seen[:, any_seen]
        for h in range(n_kv):
            g = slice(h * (heads // n_kv), (h + 1) * (heads // n_kv))
            if not len(tok):
                out[lo:hi, g], spread[lo:hi, g] = 0, 0
                continue
            k, v = (get_rows(data, slots, h, is_v, dtype, dim, page) for is_v in (0, 1))
            s = np.where(seen[:, None], np.einsum("qgd,td->qgt", q[lo:hi, g].astype(np.float64), k) * scale, -np.inf)
            m = s.max(-1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(m), m, 0))
            total = p.sum(-1, keepdims=True)
            p /= np.where(total > 0, total, 1)
            out[lo:hi, g], spread[lo:hi, g] = p @ v, p @ np.abs(v)
    return out, spread
