"""The paged 4-bit cache on a B200 where calls are at the edge of what they allow, against the 64-bit restatements of kv4_ref.py.
Tolerances are those of test_gpu_kv4.py and test_gpu_kv4_prompt.py, where they are derived."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import (BF16, F32, Api, batch, check_attend, check_cache, check_rows, qkv_call, qkv_case, qkv_want, queries,
                          random_cache)
from test_gpu_kv4_prompt import check as check_prompt
from test_gpu_kv4_prompt import want_and_tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(scope="module")
def api(gpu, torch):
    return Api(gpu, torch)


def again(api, cache, **changes):
    """The last attention call once more with some arguments changed, its results' tensor filled with 123 first."""
    a, out, st = api.keep[3], api.keep[5], api.keep[2]
    for k, v in changes.items():
        setattr(a, k, v)
    out.fill_(123)
    api.ok(api.lib.l3m_kv4_attend_dev(C.byref(cache), C.byref(a), api.stream()))
    return out, st


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["whole", "split", "prompt"])
def test_rows_of_a_step_without_room_stay_outside(api, torch, dtype, kind):
    """A step that brings more rows than its tensors have, as the plan leaves it: q_start passes max_rows, the requests concerned have kv_total 0.
    Their rows inside are zeros, nothing behind max_rows is written, whatever is there in q, and the others are served."""
    if kind == "prompt" and dtype == F32:
        pytest.skip("prompt chunks on the fifth-generation tensor cores are bf16")
    rng = np.random.default_rng(40)
    heads, kh, dim, page, width = (80, 40, 64, 16, 30) if kind == "prompt" else (8, 2, 64, 16, 200 if kind == "split" else 40)
    kv, news = np.array([300, 20, 0, 410, 5], np.int32), np.array([130, 1, 40, 90, 3], np.int32)
    held = -(-kv // page)
    n_pages = int((-(-(kv + news) // page)).sum()) + 3
    tables, order, at = np.full((5, width), -1, np.int32), rng.permutation(n_pages).astype(np.int32), 0
    for r in range(5):
        tables[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    free = np.full(n_pages, -1, np.int32)
    free[:n_pages - at] = order[at:]
    for most in (171, 200, 264, 130):
        plan = api.plan(kv, news, tables, free, n_pages - at, page, most)
        want = ref.plan(kv, news, tables, free, n_pages - at, page, most)
        for k in ("q_start", "kv_total", "tables", "status"):
            assert np.array_equal(plan[k], want[k]), k
        total = int(plan["q_start"][-1])
        assert total == 264 and bool(plan["status"] & ref.NO_ROOM) == (most < total)
        host = random_cache(rng, ref.Q4, n_pages, kh, page, dim)
        q, q64 = queries(api, rng, total + 8, heads, dim, dtype)           # more rows than the call is told of, so that a stray access would land in them
        q[most:] = float("nan")
        cache = api.cache(api.put(host), ref.Q4, page, kh, dim)
        api.attend(cache, q, plan["q_start"], plan["kv_total"], plan["tables"], 0.125, max_q=130, max_kv=width * page)
        out, st = again(api, cache, max_rows=most)
        torch.cuda.synchronize()
        assert st.item() == 0 and (out[most:] == 123).all()
        q_start = np.minimum(plan["q_start"], most)
        rows = int(q_start[-1])
        if kind == "prompt":
            w, tol = want_and_tolerance(q64[:rows], q_start, plan["kv_total"], plan["tables"], host, ref.Q4, dim, page, kh, 0.125)
            check_prompt(out[:rows], w, tol)
        else:
            check_attend(out[:rows], *ref.attend(q64[:rows], q_start, plan["kv_total"], plan["tables"], host, ref.Q4, dim, page, kh, 0.125), dtype)
        for r in np.flatnonzero(plan["kv_total"] == 0):
            assert (out[q_start[r]:q_start[r + 1]] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_are_cut_off_do_not_move_the_others(api, dtype):
    """max_rows inside a served request: its rows before it have the positions, and the results, that they have in the whole call."""
    rng = np.random.default_rng(41)
    lens, news, page = [50, 90, 33], [7, 40, 5], 16
    tables, q_start, n_pages = batch(rng, lens, news, page)
    host = random_cache(rng, ref.MX, n_pages, 2, page, 64)
    q, _ = queries(api, rng, 52, 6, 64, dtype)
    cache = api.cache(api.put(host), ref.MX, page, 2, 64)
    for window in (0, 11):
        want = api.attend(cache, q, q_start, lens, tables, 0.125, window)[0].clone()
        for most in (1, 7, 8, 30, 47, 48, 52, 60):
            out, _ = again(api, cache, max_rows=most)
            assert api.torch.equal(out[:most], want[:most]) and (out[most:] == 123).all()


# ---- scales far apart

def scale_cells(host, cdtype, dim, is_v):
    """The scales of a random cache as a writable view [pages, heads, tiles, 16 tokens, blocks]: f16 numbers or e8m0 bytes."""
    ng, width = ref.blocks(dim), 2 if cdtype == ref.Q4 else 1
    lo = 512 * ng + (16 * ng * width if is_v else 0)
    part = host[..., lo:lo + 16 * ng * width]
    part = part.view(np.float16) if cdtype == ref.Q4 else part
    return np.lib.stride_tricks.as_strided(
        part, part.shape[:3] + (16, ng), part.strides[:3] + (part.strides[3] * ng, part.strides[3]))


def of_token(cells, tables, r, t, page):
    return cells[tables[r, t // page], :, t % page // 16, t % 16]


FAR = [(ref.Q4, 8), (ref.Q4, 12), (ref.Q4, 20), (ref.MX, 8), (ref.MX, 12), (ref.MX, 15), (ref.MX, 16), (ref.MX, 17), (ref.MX, 24), (ref.MX, 40)]


def far_case(rng, cdtype, lens, news, kh, page, dim):
    tables, q_start, n_pages = batch(rng, lens, news, page)
    host = random_cache(rng, cdtype, n_pages, kh, page, dim)
    return tables, q_start, host, scale_cells(host, cdtype, dim, False), scale_cells(host, cdtype, dim, True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype,gap", FAR)
@pytest.mark.parametrize("new", [1, 5, 40])
@pytest.mark.parametrize("dim,lens", [(64, [75, 40]), (128, [1500]), (160, [90])])
def test_values_whose_blocks_are_far_apart(api, dtype, cdtype, gap, new, dim, lens):
    """A head whose blocks of 32 dims differ in size by 2^gap from one to the next, the large one first or last, in all tokens."""
    rng = np.random.default_rng(gap + new)
    for order in (1, -1):
        tables, q_start, host, _, v = far_case(rng, cdtype, lens, [new] * len(lens), 2, 16, dim)
        step = (np.arange(ref.blocks(dim))[::order] * gap) if cdtype == ref.MX else np.minimum(np.arange(ref.blocks(dim))[::order] * gap, 24)
        if cdtype == ref.MX:
            v[...] = np.clip(200 - step - rng.integers(0, 4, v.shape), 1, 254)
        else:
            v[...] = (np.exp2(10.0 - step) * rng.uniform(1, 2, v.shape) * rng.choice([-1, 1], v.shape)).astype(np.float16)
        q, q64 = queries(api, rng, int(q_start[-1]), 4, dim, dtype)
        out, _ = api.attend(api.cache(api.put(host), cdtype, 16, 2, dim), q, q_start, lens, tables, dim ** -0.5)
        check_attend(out, *ref.attend(q64, q_start, lens, tables, host, cdtype, dim, 16, 2, dim ** -0.5), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype,gap", FAR)
@pytest.mark.parametrize("new", [1, 5, 40])
@pytest.mark.parametrize("lens", [[75, 40], [1500]])
def test_values_whose_tokens_are_far_apart(api, dtype, cdtype, gap, new, lens):
    """A few tokens whose values are 2^gap times the others' and which nobody attends to (their scores are a hundred below), in every block or in
    one; and tokens that get nearly everything while their values are 2^gap times smaller than the rest."""
    rng, dim, page = np.random.default_rng(100 + gap + new), 64, 16
    for kind in ("ignored", "ignored in a block", "favoured"):
        tables, q_start, host, k, v = far_case(rng, cdtype, lens, [new] * len(lens), 2, page, dim)
        low = 0.01 if cdtype == ref.Q4 else 110
        v[...] = (low * rng.uniform(1, 2, v.shape)).astype(np.float16) if cdtype == ref.Q4 else low + rng.integers(0, 3, v.shape)
        host[..., :512] = 0x99 if cdtype == ref.Q4 else 0x11                  # keys of one code: the scale decides
        k[...] = 0.01 if cdtype == ref.Q4 else 121
        for r, n in enumerate(lens):
            for t in rng.choice(n - new, min(3, n - new), replace=False):
                at, kt = of_token(v, tables, r, t, page), of_token(k, tables, r, t, page)
                big = min(low * 2.0 ** gap, 30000.0) if cdtype == ref.Q4 else low + gap
                if kind == "favoured":
                    at[...] = low * 2.0 ** -min(gap, 14) if cdtype == ref.Q4 else low - gap
                    kt[...] = 0.4 if cdtype == ref.Q4 else 127                  # a score of about 0.3 * 40 above the others
                elif kind == "ignored":
                    at[...] = big
                else:
                    at[:, 0] = big
                if kind != "favoured":
                    tile = host[tables[r, t // page], :, 0]
                    tile[:, t % 16 * 32:t % 16 * 32 + 32] = 0x00 if cdtype == ref.Q4 else 0xFF       # -8 or -6 times the scale
                    kt[...] = 1.0 if cdtype == ref.Q4 else 127
        q, q64 = queries(api, rng, int(q_start[-1]), 4, dim, dtype)
        q, q64 = q.abs(), np.abs(q64)
        out, _ = api.attend(api.cache(api.put(host), cdtype, page, 2, dim), q, q_start, lens, tables, 0.5)
        want, spread = ref.attend(q64, q_start, lens, tables, host, cdtype, dim, page, 2, 0.5)
        # A score is off by 2^-20 of sum |q k| scale at most. That is up to sum |q| * 0.4 * 0.5 here (0.5 * 0.5 with mxfp4), not the 5 of the usual
        # inputs, where the favoured tokens are concerned; a probability by its own score's and the others' mean.
        off = 2 * 2.0 ** -20 * 0.25 * np.abs(q64).sum(-1, keepdims=True) if kind == "favoured" else 0
        # And P times scale is held down to 2^-25 (in f16, or the second of two f16), where the largest P is 2^12 or more and the largest scale up to
        # four windows' steps below 2 (q4_0: 2^base, with P up to 2^(14 - base)): values of 8 steps are off by 2^-25 * 8 * 2^-12 * 4 of that scale.
        floor = max(lens) * 2.0 ** -32 * (0.02 if cdtype == ref.Q4 else 2.0 ** (low + 2 - 127)) if kind == "favoured" else 0
        unit = 2.0 ** (-10 if dtype == BF16 else -16)
        check_attend(out, want, spread * (1 + off / unit) + floor / unit, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("heads,new", [(4, 5), (8, 3), (4, 40)])
def test_scales_that_only_later_queries_see(api, dtype, cdtype, heads, new):
    """The last new token has the largest scales there are, or ones that are not finite: the queries before it have the results
    without it, although they share a tile of rows with the query that sees it."""
    rng, dim, page, lens = np.random.default_rng(new), 64, 16, [75, 1100 + new]
    for last in ((60000.0, np.inf, np.nan) if cdtype == ref.Q4 else (160, 200, 225, 255)):
        tables, q_start, host, k, v = far_case(rng, cdtype, lens, [new] * 2, 2, page, dim)
        q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, dtype)
        want, spread = ref.attend(q64, q_start, lens, tables, host, cdtype, dim, page, 2, 0.125)
        for r, n in enumerate(lens):
            of_token(v, tables, r, n - 1, page)[...] = last
            if not np.isfinite(last) or last == 255:
                of_token(k, tables, r, n - 1, page)[...] = last
        out, _ = api.attend(api.cache(api.put(host), cdtype, page, 2, dim), q, q_start, lens, tables, 0.125)
        for r in range(2):
            rows = slice(int(q_start[r]), int(q_start[r + 1]) - 1)
            check_attend(out[rows], want[rows], spread[rows], dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_beyond_the_sums_range_count_as_nothing(api, dtype):
    """A scale of 2^127 beside ones of 2^-3: the queries that do not see it may lose their values (sums have 32 bits) but get nothing else."""
    rng, dim, page, lens, new = np.random.default_rng(50), 64, 16, [75, 1140], 40
    tables, q_start, host, _, v = far_case(rng, ref.MX, lens, [new] * 2, 2, page, dim)
    q, q64 = queries(api, rng, int(q_start[-1]), 4, dim, dtype)
    _, spread = ref.attend(q64, q_start, lens, tables, host, ref.MX, dim, page, 2, 0.125)
    for r, n in enumerate(lens):
        of_token(v, tables, r, n - 1, page)[...] = 254
    out, st = api.attend(api.cache(api.put(host), ref.MX, page, 2, dim), q, q_start, lens, tables, 0.125)
    for r in range(2):
        rows = slice(int(q_start[r]), int(q_start[r + 1]) - 1)
        assert (np.abs(out[rows].double().cpu().numpy()) <= spread[rows] * (1 + 2.0 ** -7)).all()
    assert st.item() == 0


# ---- prompt chunks

def prompt_want(q, q_start, kv_len, tables, data, cdtype, dim, page, n_kv, scale, window=0):
    """want_and_tolerance() of test_gpu_kv4_prompt.py without the terms that are relative to the cache's largest scale: what keys and values lose as
    f16 numbers is 2^-11 of themselves, however large another one is. P is off by 2^-34 of a row's largest, or by all of itself."""
    heads, n_pages = q.shape[1], data.shape[0]
    want, tol = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    for r in range(len(kv_len)):
        lo, hi, kv = int(q_start[r]), int(q_start[r + 1]), int(kv_len[r])
        tok, pos = np.arange(kv), kv - (hi - lo) + np.arange(hi - lo)
        seen = tok[None] <= pos[:, None]
        if window:
            seen &= tok[None] > pos[:, None] - window
        slots = tables[r][tok // page].astype(np.int64) * page + tok % page
        for h in range(n_kv):
            g = slice(h * (heads // n_kv), (h + 1) * (heads // n_kv))
            k, v = (ref.get_rows(data, slots, h, is_v, cdtype, dim, page) for is_v in (0, 1))
            with np.errstate(invalid="ignore"):
                k, v = np.where(np.isfinite(k), k, 0), np.where(np.isfinite(v), v, 0)
            qq, mask = q[lo:hi, g], seen[:, None]
            s = np.where(mask, np.einsum("qgd,td->qgt", qq, k) * scale, -np.inf)
            m = s.max(-1, keepdims=True)
            p = np.exp(s - np.where(np.isfinite(m), m, 0))
            total = p.sum(-1, keepdims=True)
            p /= np.where(total > 0, total, 1)
            e = scale * ((2.0 ** -11 + 2.0 ** -17) * np.einsum("qgd,td->qgt", np.abs(qq), np.abs(k)) + 2.0 ** -34 * np.abs(qq).max(-1)[..., None] * np.abs(k).sum(-1)) + 2.0 ** -20
            e = np.where(mask & (p > 0), e, 0) * (1 + 2.0 ** -6)
            w = p @ v
            want[lo:hi, g] = w
            tol[lo:hi, g] = 2.0 ** -8 * np.abs(w) + (p * (e + (p * e).sum(-1, keepdims=True) + 2.0 ** -10 + 2.0 ** -19) + np.minimum(p, 2.0 ** -34)) @ np.abs(v)
    return want, tol


def takes_prompt_kernel(api, cache):
    """The last call went to the kernel for prompt chunks: it alone needs no scratch for long contexts."""
    a = api.keep[3]
    longer = api.l3m.Kv4Attend(dtype=a.dtype, n_heads=a.n_heads, n_req=a.n_req, max_q=a.max_q, max_blocks=1 << 12, max_kv=1 << 16)
    return api.lib.l3m_kv4_attend_scratch(C.byref(cache), C.byref(longer)) == 16


@pytest.mark.parametrize("dim,heads,kh", [(64, 64, 64), (128, 32, 32)])
@pytest.mark.parametrize("at", [160, 101, 199])
def test_prompt_rows_before_an_mxfp4_scale_that_is_not_finite(api, dim, heads, kh, at):
    rng, page, lens, new = np.random.default_rng(at), 16, [200, 150], 100
    tables, q_start, host, k, v = far_case(rng, ref.MX, lens, [new] * 2, kh, page, dim)
    q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
    want, tol = prompt_want(q64, q_start, lens, tables, host, ref.MX, dim, page, kh, 0.125)
    for cells in (k, v):
        of_token(cells, tables, 0, at, page)[...] = 255
    cache = api.cache(api.put(host), ref.MX, page, kh, dim)
    out, _ = api.attend(cache, q, q_start, lens, tables, 0.125)
    assert takes_prompt_kernel(api, cache)
    before = at - (lens[0] - new)
    check_prompt(out[:before], want[:before], tol[:before])
    check_prompt(out[new:], want[new:], tol[new:])


WIDE = [(ref.Q4, 20), (ref.Q4, 28), (ref.MX, 20), (ref.MX, 33), (ref.MX, 35), (ref.MX, 60)]


@pytest.mark.parametrize("cdtype,gap", WIDE)
@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("dim,heads,kh,lens,new", [(64, 64, 32, [300, 150], 100), (104, 48, 16, [200, 130], 130), (128, 32, 32, [260, 120], 120), (48, 90, 30, [129, 257], 129)])
def test_prompt_scales_far_apart(api, cdtype, gap, window, dim, heads, kh, lens, new):
    """Values' blocks 2^gap apart in all tokens; tokens whose values are 2^gap times the others' and which nobody attends to; and keys whose blocks are
    far apart, with queries that are zero in the large one. Below and above the reach of widened numbers, which is 2^24 (q4_0) and 2^34 (mxfp4)."""
    rng, page = np.random.default_rng(gap + dim), 16
    ng = ref.blocks(dim)
    for kind in ("value blocks", "ignored tokens", "key blocks"):
        tables, q_start, host, k, v = far_case(rng, cdtype, lens, [new] * 2, kh, page, dim)
        q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
        scale = float(np.float32(0.125))
        if kind == "ignored tokens":
            q, q64 = q.abs(), np.abs(q64)
            for r, n in enumerate(lens):
                for t in rng.choice(n, 5, replace=False):
                    of_token(v, tables, r, t, page)[...] = 0.001 * 2.0 ** min(gap, 25) if cdtype == ref.Q4 else 124 + gap
                    tile = host[tables[r, t // page], :, t % page // 16]
                    tile[:, t % 16 * 16 * ng:t % 16 * 16 * ng + 16 * ng] = 0x00 if cdtype == ref.Q4 else 0xFF
                    of_token(k, tables, r, t, page)[...] = 4.0 if cdtype == ref.Q4 else 130
            if cdtype == ref.Q4:
                ordinary = np.abs(v) < 30
                v[...] = np.where(ordinary, v * np.float16(2.0 ** -9), v)
        else:
            cells = v if kind == "value blocks" else k
            for j in range(1, ng):
                cells[..., j] = (cells[..., j] * 2.0 ** (-gap / 2)).astype(np.float16) if cdtype == ref.Q4 else cells[..., j] - gap // 2
            cells[..., 0] = cells[..., 0] * np.float16(2.0 ** (gap / 2)) if cdtype == ref.Q4 else cells[..., 0] + (gap + 1) // 2
            if kind == "key blocks":
                q[..., :32] = 0
                q64 = q.double().cpu().numpy()
                scale = float(np.float32(0.1 * 2.0 ** (gap / 2)))
        cache = api.cache(api.put(host), cdtype, page, kh, dim)
        out, st = api.attend(cache, q, q_start, lens, tables, scale, window)
        assert takes_prompt_kernel(api, cache) and st.item() == 0
        check_prompt(out, *prompt_want(q64, q_start, lens, tables, host, cdtype, dim, page, kh, scale, window), norm=False)


@pytest.mark.parametrize("cdtype,big", [(ref.Q4, 60000.0), (ref.MX, 160), (ref.MX, 200), (ref.MX, 254)])
def test_prompt_scales_that_only_later_queries_see(api, cdtype, big):
    """A token in the middle of a chunk with the largest scales there are: the queries before it, in the same tiles of rows, do not know."""
    rng, dim, page, lens, new, heads, kh = np.random.default_rng(3), 64, 16, [200, 150], 100, 64, 64
    for at in (101, 160, 199):
        tables, q_start, host, k, v = far_case(rng, cdtype, lens, [new] * 2, kh, page, dim)
        if cdtype == ref.Q4:
            k *= np.float16(2.0 ** -12)
            v *= np.float16(2.0 ** -12)
        scale = 0.125 * (4096 if cdtype == ref.Q4 else 1)
        q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
        want, tol = prompt_want(q64, q_start, lens, tables, host, cdtype, dim, page, kh, scale)
        for cells in (k, v):
            of_token(cells, tables, 0, at, page)[...] = big
        cache = api.cache(api.put(host), cdtype, page, kh, dim)
        out, _ = api.attend(cache, q, q_start, lens, tables, scale)
        assert takes_prompt_kernel(api, cache)
        before = at - (lens[0] - new)
        check_prompt(out[:before], want[:before], tol[:before], norm=False)
        check_prompt(out[new:], want[new:], tol[new:], norm=False)


def test_prompt_scales_far_apart_with_strides_bad_pages_and_rows_that_see_nothing(api, torch):
    """The same contexts where they meet the rest: spare columns, odd addresses, pages outside the cache, more queries than tokens."""
    rng, dim, page, lens, news, heads, kh = np.random.default_rng(4), 48, 16, [0, 3, 250, 180], [60, 70, 133, 100], 60, 30
    tables, q_start, host, k, v = far_case(rng, ref.MX, lens, news, kh, page, dim)
    v[..., 0] += 60
    tables[2, 3], tables[2, 15] = -1, host.shape[0]
    q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, BF16)
    rows, width, cache = q.shape[0], heads * dim, api.cache(api.put(host), ref.MX, page, kh, dim)
    flat = torch.full((rows * (width + 13) + 1,), float("nan"), dtype=torch.bfloat16, device="cuda")
    qs = flat.as_strided((rows, heads, dim), (width + 13, dim, 1), 1)
    qs.copy_(q)
    space = torch.full((rows * (width + 13) + 1,), 5.0, dtype=torch.bfloat16, device="cuda")
    out, st = api.attend(cache, qs, q_start, lens, tables, 0.2, out=space.as_strided((rows, heads, dim), (width + 13, dim, 1), 1))
    assert takes_prompt_kernel(api, cache) and st.item() == ref.BAD_PAGE
    assert (space[1:].view(rows, width + 13)[:, width:] == 5).all() and (out[:60] == 0).all() and (out[60:127] == 0).all()
    want, spread = ref.attend(q64, q_start, lens, tables, host, ref.MX, dim, page, kh, float(np.float32(0.2)))
    # plain sums in 32 bits: a score of |q k| scale below 2^4 is off by 2^-17 at most, a probability by 2^-16, and the result is rounded to bf16
    assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -14 * spread).all()
    api.attend(cache, q, q_start, lens, tables, 0.2)
    assert torch.equal(api.keep[5], out)


# ---- plan

def test_plans_of_two_host_threads(api, torch):
    """Two threads plan steps of very different sizes on streams of their own, many times: no call of one is refused for the other's, and both
    have their results."""
    import threading
    rng, page, jobs = np.random.default_rng(60), 16, []
    for n in (16384, 1):
        kv, new = rng.integers(0, 33, n).astype(np.int32), np.ones(n, np.int32)
        held, after = -(-kv // page), -(-(kv + 1) // page)
        order = rng.permutation(int(after.sum()) + 5).astype(np.int32)
        tables = np.full((n, 3), -1, np.int32)
        tables[np.arange(3)[None] < held[:, None]] = order[:int(held.sum())]
        free = np.concatenate((order[int(held.sum()):], np.full(int(held.sum()), -1, np.int32)))
        n_free = len(order) - int(held.sum())
        want = ref.plan(kv, new, tables, free, n_free, page, n)
        t = {k: api.put(np.asarray(v, np.int32)) for k, v in dict(kv_len=kv, new_len=new, tables=tables, free_pages=free, n_free=[n_free]).items()}
        for k, size in dict(n_free_out=1, q_start=n + 1, kv_total=n, slot=n, pos=n, status=1).items():
            t[k] = torch.zeros(size, dtype=torch.int32, device="cuda")
        jobs.append((api.l3m.Kv4Plan(n_req=n, max_blocks=3, max_tokens=n, page=page, n_pages=len(free), **{k: v.data_ptr() for k, v in t.items()}), t, want, torch.cuda.Stream(), []))
    torch.cuda.synchronize()

    def work(args, stream, bad):
        for _ in range(3000):
            if api.lib.l3m_kv4_plan_dev(C.byref(args), stream.cuda_stream):
                bad.append(api.lib.l3m_cuda_error())

    threads = [threading.Thread(target=work, args=(args, stream, bad)) for args, _, _, stream, bad in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    for _, t, want, _, bad in jobs:
        assert not bad, bad[:3]
        for k in ("tables", "q_start", "kv_total", "slot", "pos"):
            assert np.array_equal(t[k].cpu().numpy(), want[k]), k
        assert t["n_free_out"].item() == want["n_free_out"] and t["status"].item() == 0


# ---- q, k, v

def put_x(api, c, x):
    """Other inputs for a case of qkv_case(), as its type holds them."""
    t = api.torch
    host = t.from_numpy(x).to(t.float32 if c["dtype"] == F32 else t.bfloat16)
    c["buf"][c["shift"]:] = host.reshape(-1).cuda()
    c["x"] = host.double().numpy()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("eps", [1e-5, 1e-38, 0.0])
@pytest.mark.parametrize("dim,rope,heads,kh", [(64, 0, 3, 2), (64, 2, 3, 2), (128, 1, 5, 3), (256, 2, 1, 1), (24, 2, 9, 5)])
def test_norms_of_rows_whose_squares_leave_32_bits(api, dtype, cdtype, eps, dim, rope, heads, kh):
    """Rows from the type's smallest to its largest values, some with one value far above the others: norms, keys and cache are those of the definition
    in 64 bits, with a cache and without, in place and not."""
    rng = np.random.default_rng(70 + dim)
    sizes = [1e-42, 1e-38, 1e-30, 1e-23, 1e-20, 1e-16, 1.0, 1e15, 1e17, 1.5e18, 1e19, 1e25, 1e37, 8e37]
    for store, in_place in ((True, False), (False, False), (True, True)):
        c = qkv_case(api, rng, dtype, cdtype, len(sizes) + 4, heads, kh, dim, rope, dim if rope else 0, True)
        c["eps"] = float(np.float32(eps))
        x = rng.standard_normal(c["x"].shape).clip(-3, 3)
        x[np.abs(x) < 0.01] = 0.01
        x[:len(sizes)] *= np.array(sizes)[:, None]
        x[-4, ::dim] = 2.0 ** 60
        x[-3, ::dim] = 2.0 ** 66
        x[-2] *= np.exp2(rng.integers(-60, 60, x.shape[1]))
        put_x(api, c, x)
        q, k, v = qkv_want(c)
        got_q, got_k, data, status, _ = qkv_call(api, c, store=store, in_place=in_place)
        assert status == 0
        for got, (u, f) in ((got_q, q), (got_k, k)):                       # a row of zeros (what bf16 makes of 1e-42) without eps is 0 / 0, stored as 0
            none = ~np.isfinite(f)
            got = got.reshape(u.shape)
            assert np.isnan(got[none]).all()
            got[none], u[none], f[none] = 0, 0, 1
            check_rows(got, u, f, c)
        if store:
            check_cache(data, c, k, v)
        else:
            assert (data == 0x5A).all()


@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("factor", [0.01, 1.4, 100.0, 2.0 ** 30])
@pytest.mark.parametrize("rope,rot", [(1, 128), (2, 128), (2, 96)])
def test_rotation_tables_that_carry_a_factor(api, cdtype, factor, rope, rot):
    """cos and sin times a factor, as tables for long contexts have them: codes and scales are still those of exact arithmetic, for rows enough that
    some lie within the rotation's rounding of a border."""
    rng = np.random.default_rng(80 + rot)
    c = qkv_case(api, rng, F32, cdtype, 2500, 1, 4, 128, rope, rot, True, page=64)
    c["turn"] = (c["turn"] * factor).astype(np.float32)
    q, k, v = qkv_want(c)
    got_q, _, data, _, _ = qkv_call(api, c)
    for is_v, (u, f) in enumerate((k, v)):
        codes, bits = ref.quantise(u, f, cdtype)
        want = ref.values(codes, bits, cdtype)
        for h in range(4):
            assert np.array_equal(ref.get_rows(data, c["slot"], h, is_v, cdtype, 128, 64), want[:, h])
    u, f = q
    pair = np.abs(u)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if rope == 1 else (slice(0, rot // 2), slice(rot // 2, rot))
    pair[..., a] = pair[..., b] = 2 * (pair[..., a] + pair[..., b])
    assert (np.abs(got_q.reshape(u.shape) - u * f[..., None]) <= 2.0 ** -24 * np.abs(u * f[..., None]) + 2.0 ** -19 * pair * f[..., None]).all()


@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("factor", [1.0, 1.4, 100.0, 2.0 ** 30])
@pytest.mark.parametrize("norm", [True, False])
def test_rotations_that_cancel(api, cdtype, factor, norm):
    """Keys whose first half cancels in the rotation but for 2^-22 to 2^-12 of it: what is left is a block of its own, with codes and a scale that 32 bits
    do not have, whatever factor the table carries."""
    rng = np.random.default_rng(85)
    c = qkv_case(api, rng, F32, cdtype, 700, 1, 2, 64, 2, 64, norm, page=64)
    c["turn"] = (c["turn"] * factor).astype(np.float32)
    x, turn = c["x"].copy(), c["turn"].astype(np.float64)[c["pos"]]
    w = c["w"][1].astype(np.float64) if norm else np.ones(64)
    for h in range(2):
        at = 64 + 64 * h
        size = rng.standard_normal((700, 32)) * np.exp2(-rng.integers(12, 23, (700, 1)).astype(float))
        x[:, at:at + 32] = x[:, at + 32:at + 64] * w[32:] * turn[..., 1] * (1 + size) / np.where(np.abs(turn[..., 0]) > 1e-3 * factor, turn[..., 0], factor) / w[:32]
    put_x(api, c, x)
    q, k, v = qkv_want(c)
    _, _, data, _, _ = qkv_call(api, c)
    for is_v, (u, f) in enumerate((k, v)):
        codes, bits = ref.quantise(u, f, cdtype)
        want = ref.values(codes, bits, cdtype)
        for h in range(2):
            assert np.array_equal(ref.get_rows(data, c["slot"], h, is_v, cdtype, 64, 64), want[:, h])


# ---- sums over long contexts

@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("heads,dim,flat", [(1, 32, True), (2, 32, False), (8, 64, True)])
def test_many_tokens_in_every_share(api, dtype, cdtype, heads, dim, flat):
    """16 requests of up to four million tokens, the same 16 pages over and over, so that a warp sums thousands of tiles: the result is that of
    the 16 pages once, within the tolerance of short contexts. Scores are all alike (scale 0) or random."""
    rng, page, times = np.random.default_rng(90 + heads), 4096, 64 if dim == 32 else 32
    host = random_cache(rng, cdtype, 16, 1, page, dim)
    tables = np.stack([np.concatenate([rng.permutation(16) for _ in range(times)]) for _ in range(16)]).astype(np.int32)
    lens, q_start = [16 * times * page] * 16, np.arange(17)
    q, q64 = queries(api, rng, 16, heads, dim, dtype)
    scale = 0.0 if flat else 0.25
    out, st = api.attend(api.cache(api.put(host), cdtype, page, 1, dim), q, q_start, lens, tables, scale)
    assert st.item() == 0
    once = [16 * page] * 16
    want, spread = ref.attend(q64, q_start, once, tables[:, :16], host, cdtype, dim, page, 1, scale)
    check_attend(out, want, spread, dtype)
    # and not further off, over all, than the 16 pages once: sums in 32 bits, rounded to nearest, of a few thousand terms a warp lose 2^-24 of themselves
    # each, 2^-12 at the very worst, and the values' sum is 200 times smaller than the spread that this is relative to
    short, _ = api.attend(api.cache(api.put(host), cdtype, page, 1, dim), q, q_start, once, tables, scale)
    off = [np.linalg.norm(x.double().cpu().numpy() - want) for x in (out, short)]
    assert off[0] <= 1.1 * off[1] + (2.0 ** -20 * np.linalg.norm(spread) if dtype == F32 else 0), off


@pytest.mark.parametrize("dim", [64, 128])
def test_bf16_queries_enter_the_scores_whole(api, torch, dim):
    """Neighbouring query values of 8 bits whose combinations have more than 11: scores are those of the queries themselves. One query whose large values
    cancel exactly over keys of one code, but for a few dims: a query off by 2^-12 would move the scores by far more than is left."""
    rng, page, n = np.random.default_rng(95), 16, 400
    tables, q_start, n_pages = batch(rng, [n], [1], page)
    host = random_cache(rng, ref.Q4, n_pages, 1, page, dim)
    ng = ref.blocks(dim)
    host[..., :256 * ng] = 0xFF                                              # key codes 15: 7 times the scale
    scale_cells(host, ref.Q4, dim, False)[...] = rng.integers(1, 33, (n_pages, 1, 1, 16, 1)).astype(np.float16)      # one for all blocks of a token
    big = rng.integers(128, 256, (8, dim // 4)) * np.exp2(rng.integers(-3, 3, (8, dim // 4)))
    q64 = np.zeros((1, 8, dim))
    q64[0, :, 0::4], q64[0, :, 1::4] = big, rng.integers(128, 256, big.shape) * np.exp2(rng.integers(-3, 3, big.shape))
    q64[0, :, 2::4], q64[0, :, 3::4] = -q64[0, :, 1::4], -q64[0, :, 0::4]
    q64[0, :, 0] += np.where(q64[0, :, 0] >= 256, 2.0, 1.0)
    q = torch.from_numpy(q64).to(torch.bfloat16).cuda()
    q64 = q.double().cpu().numpy()
    out, _ = api.attend(api.cache(api.put(host), ref.Q4, page, 1, dim), q, q_start, [n], tables, 0.02)
    want, spread = ref.attend(q64, q_start, [n], tables, host, ref.Q4, dim, page, 1, 0.02)
    # Products of whole numbers below 2^22 in units of 2^-3: sums in 32 bits are exact up to 2^21, and lose 2^-24 of sum |q k| = 2^18 at the
    # most per block and step; scores are off by 2^-4 * 0.02 then, P by 2^-9.
    assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -8 + 2.0 ** -10) * spread).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("dim,heads,kh,wide", [(dim, 8, 1, wide) for dim in (24, 64, 96, 128) for wide in (False, True)] + [(160, 7, 1, False), (192, 4, 2, False), (224, 8, 1, False), (256, 3, 1, False)])
def test_scales_far_apart_in_every_variant(api, dtype, cdtype, dim, heads, kh, wide):
    """Each number of blocks, 8 and 16 rows to a tile (the call's bounds decide, lengths are short): blocks 2^10 apart, some tokens 2^16 (q4_0: 2^9) above their
    neighbours, in a context with a window and without, through pages in any order."""
    rng, page, lens, news = np.random.default_rng(dim), 16, [333, 40, 1200], [20, 3, 33]
    ng = ref.blocks(dim)
    width = 40000 // page * 16 if wide else 80
    for window in (0, 100):
        tables, q_start, n_pages = batch(rng, lens, news, page, width=width)
        host = random_cache(rng, cdtype, n_pages, kh, page, dim)
        v = scale_cells(host, cdtype, dim, True)
        up = (rng.random(v.shape[:4] + (1,)) < 0.1) * 1
        if cdtype == ref.MX:
            v[...] = 200 - 10 * np.arange(ng) + 16 * up + rng.integers(0, 3, v.shape)
        else:
            v[...] = (np.exp2(5.0 - np.minimum(10 * np.arange(ng), 16) + 9 * up) * rng.uniform(1, 2, v.shape)).astype(np.float16)
        q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, dtype)
        out, st = api.attend(api.cache(api.put(host), cdtype, page, kh, dim), q, q_start, lens, tables, dim ** -0.5, window, max_kv=width * page)
        want, spread = ref.attend(q64, q_start, lens, tables, host, cdtype, dim, page, kh, dim ** -0.5, window)
        if dtype == BF16 and cdtype == ref.Q4:
            # q4_0's codes enter bf16 results as f16 subnormals, n * 2^-24, and 8 is taken off behind. A product's 17 terms (16 tokens and the sum so
            # far) are aligned by their exponents, a subnormal's being -14, and cut off 24 bits below: by 2^-14 of the largest p * scale of the 16 tokens
            # each, in units of a code. So a result is off by 17 * 2^-14 < 1.1 * 2^-10 of sum p * scale, a token whose value is 0 included, which the
            # spread does not know.
            ones = host.copy()
            ones[..., 256 * ng:512 * ng] = 0x99
            scale = ref.attend(q64, q_start, lens, tables, ones, cdtype, dim, page, kh, dim ** -0.5, window)[0]
            spread = spread + 1.1 * scale
        check_attend(out, want, spread, dtype)
        assert st.item() == 0
