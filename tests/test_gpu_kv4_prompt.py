"""Attention of prompt chunks over the paged 4-bit cache (bf16, many query rows a key/value head: the variant on the
fifth-generation tensor cores) against the plain 64-bit restatement.

Tolerance, element by element (want_and_tolerance). Keys and values are widened to f16, one rounding of code * scale: 2^-11 of it, and 2^-35
of the cache's largest scale for those that become subnormal (the largest is brought to 2^10 or more, subnormal
steps are 2^-24). Queries are bf16 times a power of two, exact but for subnormals: 2^-34 of the row's largest. So the score of token t is off
by at most
    e_t = 2^-11 scale sum |q k_t| + 2^-35 d_k scale sum |q| + 2^-34 max|q| scale sum |k_t|
and by what sums and products in f32 lose, less than 2^-17 scale sum |q k_t| + 2^-20 together. The probability p_t is off by the factor
e_t + sum p e in first order (2^-6 of it more for the second: e_t < 1/64 in these tests but the sharp one, which has its own), and the numerator's is
rounded to f16: 2^-11, or 2^-25 of a row's largest, 2^9 at least, where subnormal. With the values' rounding
    |error| <= 2^-8 |w| + sum p |v| (e_t + sum p e + 2^-10 + 2^-19) + n 2^-34 max|v| + 2^-35 d_v
where 2^-8 |w| is the result's rounding. Roundings do not conspire: over a whole result the error's norm has to stay below
2^-8 of the result's as well, where scores and values are of ordinary size (bf16's own rounding is 0.4 of that)."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import BF16, Api, batch, queries, random_cache

pytestmark = pytest.mark.gpu


class PromptApi(Api):
    """Calls that have to take this variant: it alone needs no scratch for long contexts."""

    def attend(self, cache, *args, **kw):
        got = super().attend(cache, *args, **kw)
        a = self.keep[3]
        longer = self.l3m.Kv4Attend(dtype=a.dtype, n_heads=a.n_heads, n_req=a.n_req, max_q=a.max_q, max_blocks=1 << 12, max_kv=1 << 16)
        assert self.lib.l3m_kv4_attend_scratch(C.byref(cache), C.byref(longer)) == 16
        return got


@pytest.fixture(scope="module")
def api(gpu):
    import torch
    return PromptApi(gpu, torch)


def top_scales(data, cdtype, dim):
    tail = np.ascontiguousarray(data[..., 512 * ref.blocks(dim):])
    half = tail.shape[-1] // 2
    out = []
    for part in (tail[..., :half], tail[..., half:]):
        s = np.abs(np.ascontiguousarray(part).view(np.float16).astype(np.float64)) if cdtype == ref.Q4 else np.ldexp(1.0, part.astype(np.int64) - 127)
        out.append(s[np.isfinite(s)].max(initial=0))
    return out


def want_and_tolerance(q, q_start, kv_len, tables, data, cdtype, dim, page, n_kv, scale, window=0):
    heads, n_pages = q.shape[1], data.shape[0]
    want, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    dk, dv = top_scales(data, cdtype, dim)
    for r in range(len(kv_len)):
        lo, hi, kv = int(q_start[r]), int(q_start[r + 1]), int(kv_len[r])
        if hi == lo:
            continue
        tok = np.arange(kv)
        ids = tables[r][tok // page] if kv else tok
        tok = tok[(ids >= 0) & (ids < n_pages)]
        pos = kv - (hi - lo) + np.arange(hi - lo)
        seen = tok[None] <= pos[:, None]
        if window:
            seen &= tok[None] > pos[:, None] - window
        tok, seen = tok[seen.any(0)], seen[:, seen.any(0)]
        slots = tables[r][tok // page].astype(np.int64) * page + tok % page if len(tok) else tok
        for h in range(n_kv):
            g = slice(h * (heads // n_kv), (h + 1) * (heads // n_kv))
            if not len(tok):
                want[lo:hi, g], tol[lo:hi, g] = 0, 0
                continue
            k, v = (ref.get_rows(data, slots, h, is_v, cdtype, dim, page) for is_v in (0, 1))
            qq, mask = q[lo:hi, g], seen[:, None]
            s = np.where(mask, np.einsum("qgd,td->qgt", qq, k) * scale, -np.inf)
            m = s.max(-1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(m), m, 0))
            total = p.sum(-1, keepdims=True)
            p /= np.where(total > 0, total, 1)
            a = np.abs(qq)
            e = scale * ((2.0 ** -11 + 2.0 ** -17) * np.einsum("qgd,td->qgt", a, np.abs(k)) + 2.0 ** -35 * dk * a.sum(-1)[..., None] + 2.0 ** -34 * a.max(-1)[..., None] * np.abs(k).sum(-1)) + 2.0 ** -20
            e = np.where(mask, e, 0) * (1 + 2.0 ** -6)
            w = p @ v
            off = (p * (e + (p * e).sum(-1, keepdims=True) + 2.0 ** -10 + 2.0 ** -19)) @ np.abs(v)
            want[lo:hi, g] = w
            tol[lo:hi, g] = np.where(total > 0, 2.0 ** -8 * np.abs(w) + off + len(tok) * 2.0 ** -34 * np.abs(v).max() + 2.0 ** -35 * dv, 0)
    return want, tol


def check(got, want, tol, norm=True):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol + 1e-38)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], float(np.abs(got - want)[bad].max()))
    if norm:
        assert np.linalg.norm(got - want) <= 2.0 ** -8 * np.linalg.norm(want)


# heads, kv heads, dim, page, cached lengths, new tokens: enough rows each for this variant
SHAPES = [
    (64, 64, 128, 64, [128] * 2, [128] * 2),                            # one tile of 128 rows each, no group
    (16, 4, 128, 32, [300, 200, 130, 1, 77, 64, 90, 400], [100, 64, 130, 1, 40, 30, 90, 64]),
    (30, 10, 64, 16, [300, 200, 130, 50], [100, 64, 130, 50]),          # a group of 3: tiles end inside a token's heads
    (30, 10, 48, 16, [129, 257, 255, 383], [129, 1, 63, 100]),           # dims that end inside a block, lengths beside steps
    (160, 16, 40, 48, [64, 65, 127, 128, 129, 2, 0, 33], [13, 10, 5, 1, 12, 2, 0, 3]),
    (64, 32, 104, 16, [60, 61], [60, 49]),
    (8, 2, 112, 128, [500] * 4, [129, 128, 127, 300]),
    (96, 96, 128, 16, [900], [97]),
]


@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("heads,kv_heads,dim,page,lens,news", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 70])
def test_prompt(api, cdtype, heads, kv_heads, dim, page, lens, news, window):
    rng = np.random.default_rng(dim + page)
    tables, q_start, n_pages = batch(rng, lens, news, page)
    host = random_cache(rng, cdtype, n_pages, kv_heads, page, dim)
    q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
    out, st = api.attend(api.cache(api.put(host), cdtype, page, kv_heads, dim), q, q_start, lens, tables, dim ** -0.5, window)
    assert st.item() == 0
    check(out, *want_and_tolerance(q64, q_start, lens, tables, host, cdtype, dim, page, kv_heads, float(np.float32(dim ** -0.5)), window))


@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
def test_prompt_rows_that_see_nothing_and_rows_of_nobody(api, cdtype):
    """More queries than cached tokens, nothing cached, no queries; rows of q behind the last request hold NaN and their results stay."""
    rng = np.random.default_rng(1)
    lens, news, heads, kh, dim, page = [0, 3, 20, 0, 50, 150], [130, 140, 0, 0, 9, 128], 16, 8, 64, 16
    tables, q_start, n_pages = batch(rng, lens, news, page)
    host = random_cache(rng, cdtype, n_pages, kh, page, dim)
    q, q64 = queries(api, rng, int(q_start[-1]) + 5, heads, dim, BF16)
    q[-5:] = float("nan")
    out, st = api.attend(api.cache(api.put(host), cdtype, page, kh, dim), q, q_start, lens, tables, 0.125, max_q=200)
    n = int(q_start[-1])
    assert (out[n:] == 123).all() and st.item() == 0
    want, tol = want_and_tolerance(q64, q_start, lens, tables, host, cdtype, dim, page, kh, 0.125)
    assert (want[:130 + 137] == 0).all() and (out[:130 + 137] == 0).all() and (want[130 + 137] != 0).any()
    check(out[:n], want[:n], tol[:n])


def test_prompt_windows_beyond_everything(api):
    rng = np.random.default_rng(13)
    lens, news, heads, kh, dim, page = [200, 50, 333], [130, 140, 128], 40, 40, 64, 16
    tables, q_start, n_pages = batch(rng, lens, news, page)
    host = random_cache(rng, ref.Q4, n_pages, kh, page, dim)
    q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
    want, tol = want_and_tolerance(q64, q_start, lens, tables, host, ref.Q4, dim, page, kh, 0.125)
    for window in (333, (1 << 31) - 1):
        check(api.attend(api.cache(api.put(host), ref.Q4, page, kh, dim), q, q_start, lens, tables, 0.125, window)[0], want, tol)


@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("window", [0, 21])
def test_prompt_ignores_what_nobody_sees(api, cdtype, window):
    """NaN and infinite scales behind a request's last token, outside the window and in pages of nobody: the same bits."""
    rng = np.random.default_rng(2)
    lens, new, heads, kh, page, dim = [277, 145, 64], 60, 80, 40, 32, 64
    tables, q_start, n_pages = batch(rng, lens, [new] * 3, page)
    host = random_cache(rng, cdtype, n_pages, kh, page, dim)
    bad, ng, width = host.copy(), 2, 2 if cdtype == ref.Q4 else 1
    seen = np.zeros((n_pages, page), bool)
    for r, n in enumerate(lens):
        for t in range(max(0, n - new - window + 1) if window else 0, n):
            seen[tables[r, t // page], t % page] = True
    for pg, t in np.argwhere(~seen):
        for at in (512 * ng, (512 + 16 * width) * ng):
            cell = at + t % 16 * ng * width
            bad[pg, :, t // 16, cell:cell + ng * width] = 0xFF if (pg + t) % 2 else 0x7C
        bad[pg, :, t // 16, t % 16 * 32:t % 16 * 32 + 32] = 0xF7
    q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
    outs = [api.attend(api.cache(api.put(d), cdtype, page, kh, dim), q, q_start, lens, tables, 0.125, window)[0] for d in (host, bad)]
    assert api.torch.equal(*outs)
    check(outs[1], *want_and_tolerance(q64, q_start, lens, tables, host, cdtype, dim, page, kh, 0.125, window))


def test_prompt_rows_that_do_not_see_a_bad_scale(api):
    """A token among the new ones with scales that are not finite: rows before it and other requests have the results without it."""
    rng = np.random.default_rng(12)
    lens, new, heads, kh, page, dim = [200, 150], 100, 64, 64, 16, 64
    for at, byte in ((160, 0x7C), (101, 0x7E), (199, 0xFF)):
        tables, q_start, n_pages = batch(rng, lens, [new] * 2, page)
        host = random_cache(rng, ref.Q4, n_pages, kh, page, dim)
        q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
        want, tol = want_and_tolerance(q64, q_start, lens, tables, host, ref.Q4, dim, page, kh, 0.125)
        for cell in (1024, 1024 + 64):
            cell += at % 16 * 4
            host[tables[0, at // page], :, 0, cell:cell + 4] = byte
        out, _ = api.attend(api.cache(api.put(host), ref.Q4, page, kh, dim), q, q_start, lens, tables, 0.125)
        before = at - (lens[0] - new)
        check(out[:before], want[:before], tol[:before])
        check(out[new:], want[new:], tol[new:])


@pytest.mark.parametrize("window", [0, 90])
def test_prompt_bad_pages_are_not_seen(api, window):
    rng = np.random.default_rng(3)
    lens, new, heads, kh, page, dim = [300, 190, 140], 70, 32, 16, 16, 128
    tables, q_start, n_pages = batch(rng, lens, [new] * 3, page)
    host = random_cache(rng, ref.Q4, n_pages, kh, page, dim)
    tables[0, 15], tables[0, 17], tables[0, 18], tables[1, :] = -1, n_pages, -(1 << 31), 1 << 30
    q, q64 = queries(api, rng, 3 * new, heads, dim, BF16)
    out, st = api.attend(api.cache(api.put(host), ref.Q4, page, kh, dim), q, q_start, lens, tables, 0.09, window)
    assert st.item() == ref.BAD_PAGE
    want, tol = want_and_tolerance(q64, q_start, lens, tables, host, ref.Q4, dim, page, kh, float(np.float32(0.09)), window)
    assert (want[new:2 * new] == 0).all() and (out[new:2 * new] == 0).all()
    check(out, want, tol)


@pytest.mark.parametrize("cdtype,lo", [(ref.Q4, v) for v in (2.0 ** -24, 2.0 ** -14, 0.01, 1.0, 4000.0)] + [(ref.MX, v) for v in (1, 30, 100, 127, 160, 230)])
@pytest.mark.parametrize("mixed", [False, True])
def test_prompt_scales_of_every_size(api, cdtype, lo, mixed):
    """The values' scales from the smallest to the largest that the formats have; the keys' with queries sized to match."""
    rng = np.random.default_rng(4)
    page, dim, lens, new, heads, kh = 32, 64, [275, 133], 100, 64, 64
    tables, q_start, n_pages = batch(rng, lens, [new, new], page)
    for values in (True, False):
        host = random_cache(rng, cdtype, n_pages, kh, page, dim)
        cells = 16 * 2 * (2 if cdtype == ref.Q4 else 1)
        scales = host[..., 1024 + cells:] if values else host[..., 1024:1024 + cells]
        if cdtype == ref.Q4:
            s = lo * np.exp2(rng.integers(0, 5, scales.shape[:-1] + (32,)))
            s = np.where(rng.random(s.shape) < 0.5, s, min(lo, 0.02)) if mixed else s
            top = 16 * lo
            scales[...] = s.astype(np.float16).view(np.uint8).reshape(scales.shape)
        else:
            e = lo + rng.integers(0, 5, scales.shape)
            top = 2.0 ** (lo + 4 - 127)
            scales[...] = np.where(rng.random(e.shape) < 0.5, e, min(lo, 120)) if mixed else e
        # scores of ordinary size: q k scale is 64 * size * (5 top) * scale at most
        scale = 0.125 if values else float(np.float32(2.0 ** -6 / min(top, 2.0 ** 100)))
        q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
        out, _ = api.attend(api.cache(api.put(host), cdtype, page, kh, dim), q, q_start, lens, tables, scale)
        check(out, *want_and_tolerance(q64, q_start, lens, tables, host, cdtype, dim, page, kh, scale), norm=not (mixed or lo in (2.0 ** -24, 1)))


@pytest.mark.parametrize("cdtype,size", [(ref.Q4, 1e30), (ref.Q4, 1e-30), (ref.MX, 1e30), (ref.MX, 1e-35), (ref.Q4, 1.0), (ref.MX, 0.0)])
def test_prompt_queries_of_every_size(api, cdtype, size):
    """Queries at both ends of their range with scores of ordinary size, queries whose values differ by 2^40, rows of zeros, a scale of 0."""
    rng = np.random.default_rng(5)
    page, dim, lens, new, heads, kh = 16, 64, [270, 141], 100, 64, 64
    tables, q_start, n_pages = batch(rng, lens, [new, new], page)
    host = random_cache(rng, cdtype, n_pages, kh, page, dim)
    q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16, size)
    if size == 1.0:
        q = api.torch.from_numpy(q64 * np.ldexp(1.0, rng.integers(-40, 1, q64.shape))).cuda().to(q.dtype)
        q[::3] = 0
        q64 = q.double().cpu().numpy()
    for scale in (float(np.float32(0.125 / size if size else 0.125)), 0.0):
        out, _ = api.attend(api.cache(api.put(host), cdtype, page, kh, dim), q, q_start, lens, tables, scale)
        check(out, *want_and_tolerance(q64, q_start, lens, tables, host, cdtype, dim, page, kh, scale))


@pytest.mark.parametrize("order", [1, -1, 0])
def test_prompt_sharp_scores(api, order):
    """Scores of hundreds that rise, fall or jump along the context, so that the softmax's reference moves at every half, never, or now and
    then. Keys of one code and scales of 11 bits: the products with the code 1 are exact in f16, and queries of 8 bits, so
    scores are exact but for the sums' roundings, 2^-23 of 2^10 sixty-four times at most: the probabilities are off by 2^-7 of
    themselves at the worst, and twice that with the sum's."""
    rng = np.random.default_rng(6)
    page, dim, n, new, heads, kh = 16, 64, 700, 130, 128, 128
    tables, q_start, n_pages = batch(rng, [n], [new], page)
    host = random_cache(rng, ref.Q4, n_pages, kh, page, dim)
    host[..., :512] = 0x99                                     # every key code 9: the value 1 times the scale
    for t in range(n):
        size = {1: t, -1: n - t, 0: int(rng.integers(n))}[order] / n
        tile = host[tables[0, t // page], :, t % page // 16]
        tile[:, 1024 + t % 16 * 4:1024 + t % 16 * 4 + 4] = np.array([size * 16] * 2, np.float16).view(np.uint8)
    q, q64 = queries(api, rng, new, heads, dim, BF16)
    q, q64 = q.abs(), np.abs(q64)
    out, _ = api.attend(api.cache(api.put(host), ref.Q4, page, kh, dim), q, q_start, [n], tables, 1.0)
    want, spread = ref.attend(q64, q_start, [n], tables, host, ref.Q4, dim, page, kh, 1.0)
    assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -6 + 2.0 ** -10) * spread).all()


def test_prompt_strides_alignment_and_the_same_bits_twice(api):
    """Queries and results inside wider matrices at addresses that are only 2-byte aligned: the spare columns stay, and the bits
    are those of the aligned call."""
    rng, t = np.random.default_rng(7), api.torch
    page, dim, heads, kh, lens, news = 16, 48, 40, 40, [250, 330, 7], [100, 133, 2]
    tables, q_start, n_pages = batch(rng, lens, news, page)
    host = random_cache(rng, ref.MX, n_pages, kh, page, dim)
    cache = api.cache(api.put(host), ref.MX, page, kh, dim)
    q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
    rows, width = q.shape[0], heads * dim
    want = api.attend(cache, q, q_start, lens, tables, 0.2)[0]
    check(want, *want_and_tolerance(q64, q_start, lens, tables, host, ref.MX, dim, page, kh, float(np.float32(0.2))))
    for pad, base in ((13, 1), (8, 0), (16, 4)):
        flat = t.full((rows * (width + pad) + base,), float("nan"), dtype=t.bfloat16, device="cuda")
        qs = flat.as_strided((rows, heads, dim), (width + pad, dim, 1), base)
        qs.copy_(q)
        for _ in range(2):
            space = t.full((rows * (width + pad) + base,), 5.0, dtype=t.bfloat16, device="cuda")
            out = space.as_strided((rows, heads, dim), (width + pad, dim, 1), base)
            api.attend(cache, qs, q_start, lens, tables, 0.2, out=out)
            assert t.equal(out, want)
            assert (space[base:].view(rows, width + pad)[:, width:] == 5).all() and (space[:base] == 5).all()


def test_prompt_on_two_streams_and_in_a_replayed_graph(api):
    """Two calls at once, and a captured call that is replayed with other queries, lengths and tables in the same places."""
    t, rng = api.torch, np.random.default_rng(8)
    jobs = []
    for cdtype, dim, kh in ((ref.Q4, 64, 20), (ref.MX, 128, 20)):
        lens, news, page = [400, 130, 260], [100, 130, 7], 16
        tables, q_start, n_pages = batch(rng, lens, news, page)
        host = random_cache(rng, cdtype, n_pages, kh, page, dim)
        q, _ = queries(api, rng, int(q_start[-1]), 2 * kh, dim, BF16)
        cache = api.cache(api.put(host), cdtype, page, kh, dim)
        out, _ = api.attend(cache, q, q_start, lens, tables, 0.1)
        t.cuda.synchronize()
        jobs.append((cache, api.keep, out, out.clone(), t.cuda.Stream(), host, tables))
    for job in jobs:
        job[2].zero_()
    t.cuda.synchronize()
    for _ in range(30):
        for cache, keep, _, _, s, _, _ in jobs:
            api.ok(api.lib.l3m_kv4_attend_dev(C.byref(cache), C.byref(keep[3]), s.cuda_stream))
    t.cuda.synchronize()
    for _, _, out, want, _, _, _ in jobs:
        assert t.equal(out, want)
    cache, keep, out, _, s, host, tables = jobs[0]
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph, stream=s):
        api.ok(api.lib.l3m_kv4_attend_dev(C.byref(cache), C.byref(keep[3]), t.cuda.current_stream().cuda_stream))
    q_start, lens = np.array([0, 60, 60, 190], np.int32), np.array([80, 9, 390], np.int32)
    shuffled = tables.copy()
    shuffled[2, :tables.shape[1]] = tables[0]
    q, q64 = queries(api, rng, keep[4].shape[0], 40, 64, BF16)
    for dst, src in ((keep[0][0], q_start), (keep[0][1], lens), (keep[0][2], shuffled)):
        dst.copy_(t.from_numpy(src))
    keep[4].copy_(q)
    out.fill_(7)
    for _ in range(2):
        graph.replay()
    t.cuda.synchronize()
    want, tol = want_and_tolerance(q64, q_start, lens, shuffled, host, ref.Q4, 64, 16, 20, float(np.float32(0.1)))
    check(out[:190], want[:190], tol[:190])
    assert (out[190:] == 7).all()
