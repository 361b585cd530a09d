"""The paged 4-bit cache on a B200 against plain 64-bit restatements (kv4_ref.py): bookkeeping and cache bytes exactly,
norms, rotations and attention within what their roundings can be off by.

Tolerances. A result rounded once to bf16 is off by at most 2^-8 of it, to f32 by 2^-24. q_out and k_out: a norm's sum of up to
256 squares, a root, a division and at most five products and sums in f32, each at most 2^-24 of the pair's magnitude
|a| + |b|: 2^-19 of it covers them. Attention with f32 in and out: a score is off by at most 2^-20 of sum |q k| scale (about 5 with
the inputs here: every product's operands hold 22 bits or more, sums of a block are truncated to 2^-23 at most four times), so the
probabilities by 2^-17; the products with the values add at most 2^-19 and exp 2^-22: 2^-16 of
sum(p |v|) / sum(p) covers them. With bf16 in and out the products of probability and scale are rounded once to 11 bits,
2^-11 of that sum, and the result to bf16: 2^-8 of it, and 2^-10 of the sum."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu
F32, BF16 = 0, 1


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


class Api:
    """The library's calls on torch tensors."""

    def __init__(self, lib, torch):
        import l3m_b200
        self.lib, self.torch, self.l3m = lib, torch, l3m_b200

    def put(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a)).cuda()

    def ok(self, rc):
        assert rc == 0, self.lib.l3m_cuda_error()

    def stream(self):
        return self.torch.cuda.current_stream().cuda_stream

    def cache(self, data, dtype, page, heads, dim, n_pages=None):
        c = self.l3m.Kv4(data=data.data_ptr(), dtype=dtype, n_pages=data.shape[0] if n_pages is None else n_pages, page=page, n_kv_heads=heads, head_dim=dim)
        c.owner = data                                        # the tensor lives as long as its handle
        return c

    def plan(self, kv_len, new_len, tables, free_pages, n_free, page, max_tokens):
        t = {k: self.put(np.asarray(v, np.int32)) for k, v in dict(kv_len=kv_len, new_len=new_len, tables=tables, free_pages=free_pages, n_free=[n_free]).items()}
        n, width = tables.shape
        for k, size in dict(n_free_out=1, q_start=n + 1, kv_total=n, slot=max_tokens, pos=max_tokens, status=1).items():
            t[k] = self.torch.full((size,), 0 if k == "status" else -77, dtype=self.torch.int32, device="cuda")
        args = self.l3m.Kv4Plan(n_req=n, max_blocks=width, max_tokens=max_tokens, page=page, n_pages=len(free_pages), **{k: v.data_ptr() for k, v in t.items()})
        self.ok(self.lib.l3m_kv4_plan_dev(C.byref(args), self.stream()))
        out = {k: v.cpu().numpy() for k, v in t.items()}
        return {**out, "n_free_out": int(out["n_free_out"][0]), "status": int(out["status"][0])}

    def attend(self, cache, q, q_start, kv_len, tables, scale, window=0, max_q=None, max_kv=None, out=None, q_ld=None):
        t = self.torch
        heads, dim = q.shape[-2:]
        out = t.full((q.shape[0], heads, dim), 123.0, dtype=q.dtype, device="cuda") if out is None else out
        st, dev = t.zeros(1, dtype=t.int32, device="cuda"), [self.put(np.asarray(a, np.int32)) for a in (q_start, kv_len, tables)]
        lens = np.diff(q_start)
        a = self.l3m.Kv4Attend(dtype=F32 if q.dtype == t.float32 else BF16, n_heads=heads, n_req=len(kv_len), max_blocks=tables.shape[1], max_q=max(lens, default=0) if max_q is None else max_q,
                               max_kv=min(max(kv_len, default=0), tables.shape[1] * cache.page) if max_kv is None else max_kv, window=window, scale=scale, q=q.data_ptr(), out=out.data_ptr(),
                               q_ld=q.stride(0), out_ld=out.stride(0), q_start=dev[0].data_ptr(), kv_len=dev[1].data_ptr(), tables=dev[2].data_ptr(), status=st.data_ptr())
        scratch = t.full((max(16, self.lib.l3m_kv4_attend_scratch(C.byref(cache), C.byref(a))),), 0xA5, dtype=t.uint8, device="cuda")
        a.scratch, a.scratch_bytes = scratch.data_ptr(), scratch.numel()
        self.ok(self.lib.l3m_kv4_attend_dev(C.byref(cache), C.byref(a), self.stream()))
        self.keep = (dev, scratch, st, a, q, out)
        return out, st


@pytest.fixture(scope="module")
def api(gpu, torch):
    return Api(gpu, torch)


# ---- plan

def plan_case(rng, n, page, width, n_pages, prompts, ended=0.1):
    kv = rng.integers(0, width * page // 2 + 1, n)
    kv[rng.random(n) < 0.2] = 0
    new = np.where(rng.random(n) < prompts, rng.integers(0, width * page // 2 + 1, n), 1)
    new[rng.random(n) < ended] = -1
    held = -(-kv // page)
    order = rng.permutation(n_pages)
    tables = np.full((n, width), -5, np.int32)
    at = 0
    for r in range(n):
        tables[r, :held[r]] = order[at:at + held[r]]
        at += held[r]
    free = np.full(n_pages, -9, np.int32)
    free[:n_pages - at] = order[at:]
    return kv.astype(np.int32), new.astype(np.int32), tables, free, n_pages - at


def same_plan(got, want):
    for k, v in want.items():
        assert np.array_equal(got[k], v), (k, got[k], v)


@pytest.mark.parametrize("n,page,width", [(1, 16, 3), (3, 48, 5), (33, 16, 9), (257, 64, 4), (1024, 16, 6), (1025, 16, 6), (2500, 32, 3)])
@pytest.mark.parametrize("prompts", [0.0, 0.5])
def test_plan(api, n, page, width, prompts):
    rng = np.random.default_rng(n + page)
    kv, new, tables, free, n_free = plan_case(rng, n, page, width, n * width + 7, prompts)
    total = int(np.maximum(new, 0).sum())
    for most in (total, total + 5):
        want = ref.plan(kv, new, tables, free, n_free, page, most)
        assert want["status"] == 0
        same_plan(api.plan(kv, new, tables, free, n_free, page, most), want)


def test_plan_when_pages_rows_or_lengths_run_out(api):
    rng = np.random.default_rng(9)
    for trial in range(12):
        n, page, width = int(rng.integers(2, 60)), 16, 8
        kv, new, tables, free, n_free = plan_case(rng, n, page, width, n * width, 0.6, ended=0.05)
        total = int(np.maximum(new, 0).sum())
        short = int(rng.integers(0, n_free + 1)) // 3
        kv2 = kv.copy()
        kv2[rng.integers(n)] = -3 if trial % 3 else page * width + 1
        for args in ((kv, new, tables, free, short, page, total), (kv, new, tables, free, n_free, page, total // 2), (kv2, new, tables, free, n_free, page, total)):
            want = ref.plan(*args)
            same_plan(api.plan(*args), want)
    assert ref.plan(kv2, new, tables, free, n_free, page, total)["status"] & ref.BAD_LENGTH


@pytest.mark.parametrize("n_free", [-1, 99])
def test_plan_with_a_bad_free_count(api, n_free):
    kv, new = np.array([0, 20], np.int32), np.array([5, 1], np.int32)
    tables, free = np.array([[-1, -1, -1], [3, 4, -1]], np.int32), np.arange(6, dtype=np.int32)
    want = ref.plan(kv, new, tables, free, n_free, 16, 6)
    assert want["status"] & ref.BAD_LENGTH
    same_plan(api.plan(kv, new, tables, free, n_free, 16, 6), want)


def test_plan_returning_more_pages_than_the_pool_has(api):
    kv, new = np.array([40, 40, 3], np.int32), np.array([-1, -1, 30], np.int32)
    tables, free = np.array([[0, 1, 2], [3, 4, 5], [6, -1, -1]], np.int32), np.arange(8, dtype=np.int32)
    want = ref.plan(kv, new, tables, free, 5, 16, 32)
    assert want["status"] & ref.BAD_LENGTH
    same_plan(api.plan(kv, new, tables, free, 5, 16, 32), want)


def test_plan_leaves_out_pages_that_are_none(api):
    """Ids outside the cache in a request's own pages or on the free list: their slots are -1, nothing wraps into the cache."""
    for bad in (6, -3, 1 << 28, -(1 << 31), (1 << 31) - 1):
        kv, new = np.array([14, 20, 0], np.int32), np.array([3, 2, 20], np.int32)
        tables, free = np.array([[bad, -1, -1], [3, 4, -1], [-1, -1, -1]], np.int32), np.array([0, 1, bad, 2, 5, 5], np.int32)
        want = ref.plan(kv, new, tables, free, 5, 16, 30)
        assert want["status"] == ref.BAD_PAGE and (want["slot"][:2] == -1).all()
        same_plan(api.plan(kv, new, tables, free, 5, 16, 30), want)


def test_plan_of_no_requests(api):
    got = api.plan(np.zeros(0), np.zeros(0), np.zeros((0, 4), np.int32), np.arange(6), 6, 16, 3)
    assert got["n_free_out"] == 6 and list(got["q_start"]) == [0] and list(got["slot"]) == [-1] * 3 and got["status"] == 0


# ---- q, k, v

def half_step(dtype):
    return 2.0 ** -8 if dtype == BF16 else 2.0 ** -24


def qkv_case(api, rng, dtype, cdtype, tokens, heads, kv_heads, dim, rope, rot, norm, page=16, pad=0, shift=0, ties=False):
    """Inputs as slices of one matrix with `pad` spare columns, its base `shift` elements off; positions with 0 among them."""
    t, width = api.torch, (heads + 2 * kv_heads) * dim + pad
    x = rng.standard_normal((tokens, width)) * np.exp(rng.standard_normal(width))
    if ties:                                                  # few bits a value: values on the borders of codes, equal magnitudes of both signs
        x = np.round(x * 4) / 4
    x[:, :min(8, width)] = 0
    host = t.from_numpy(x).to(t.float32 if dtype == F32 else t.bfloat16)
    buf = t.zeros(tokens * width + shift, dtype=host.dtype, device="cuda")
    buf[shift:] = host.reshape(-1).cuda()
    n_pos = 64
    turn = np.stack((np.cos(np.outer(np.arange(n_pos), 0.7 ** np.arange(max(1, rot // 2)))), np.sin(np.outer(np.arange(n_pos), 0.7 ** np.arange(max(1, rot // 2))))), -1).astype(np.float32)
    turn = turn[:, :rot // 2]
    pos = rng.integers(0, n_pos, tokens).astype(np.int32)
    pos[:2] = 0
    n_pages = -(-tokens // page) + 2
    slot = rng.permutation(n_pages * page)[:tokens].astype(np.int32)
    w = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if norm else None for _ in "qk"]
    return dict(x=host.double().numpy(), buf=buf, shift=shift, width=width, turn=turn, pos=pos, slot=slot, w=w, n_pages=n_pages, page=page, dtype=dtype, cdtype=cdtype, tokens=tokens, heads=heads,
                kv_heads=kv_heads, dim=dim, rope=rope, rot=rot, eps=1e-5, n_pos=n_pos)


def qkv_call(api, c, store=True, k_out=True, in_place=False, out_pad=0):
    t, d, h, kh = api.torch, c["dim"], c["heads"], c["kv_heads"]
    size, base = c["buf"].element_size(), c["buf"].data_ptr() + c["shift"] * c["buf"].element_size()
    dev = {k: api.put(c[k]) for k in ("turn", "pos", "slot")}
    w = [None if a is None else api.put(a) for a in c["w"]]
    q_out = t.full((c["tokens"], h * d + out_pad), 7.0, dtype=c["buf"].dtype, device="cuda")
    k_res = t.full((c["tokens"], kh * d + out_pad), 7.0, dtype=c["buf"].dtype, device="cuda")
    data = t.full((c["n_pages"], kh, c["page"] // 16, ref.tile_bytes(c["cdtype"], d)), 0x5A, dtype=t.uint8, device="cuda")
    st = t.zeros(1, dtype=t.int32, device="cuda")
    a = api.l3m.Qkv(dtype=c["dtype"], n_tokens=c["tokens"], n_heads=h, n_kv_heads=kh, head_dim=d, rope=c["rope"], rot_dim=c["rot"], n_pos=c["n_pos"], eps=c["eps"],
                    q_norm=w[0].data_ptr() if w[0] is not None else None, k_norm=w[1].data_ptr() if w[1] is not None else None, rope_table=dev["turn"].data_ptr() or None, pos=dev["pos"].data_ptr(),
                    slot=dev["slot"].data_ptr(), q=base, k=base + h * d * size, v=base + (h + kh) * d * size, q_ld=c["width"], k_ld=c["width"], v_ld=c["width"],
                    q_out=base if in_place else q_out.data_ptr(), k_out=(base + h * d * size if in_place else k_res.data_ptr()) if k_out else None,
                    q_out_ld=c["width"] if in_place else h * d + out_pad, k_out_ld=c["width"] if in_place else kh * d + out_pad, status=st.data_ptr())
    cache = api.cache(data, c["cdtype"], c["page"], kh, d)
    api.ok(api.lib.l3m_qkv_rope_dev(C.byref(cache) if store else None, C.byref(a), api.stream()))
    if in_place:
        rows = c["buf"][c["shift"]:].view(c["tokens"], c["width"])
        q_out, k_res = rows[:, :h * d], rows[:, h * d:(h + kh) * d]
    return q_out.double().cpu().numpy(), k_res.double().cpu().numpy(), data.cpu().numpy(), int(st.item()), (cache, data)


def qkv_want(c):
    d, h, kh, n = c["dim"], c["heads"], c["kv_heads"], c["tokens"]
    parts = np.split(c["x"][:, :(h + 2 * kh) * d], [h * d, (h + kh) * d], 1)
    q, k, v = (p.reshape(n, -1, d) for p in parts)
    turn = c["turn"].astype(np.float64)[np.clip(c["pos"], 0, c["n_pos"] - 1)]
    w = [None if a is None else a.astype(np.float64) for a in c["w"]]
    return (ref.normed_rotated(q, w[0], c["eps"], turn, c["rope"], c["rot"]), ref.normed_rotated(k, w[1], c["eps"], turn, c["rope"], c["rot"]), (v, np.ones(v.shape[:2])))


def pair_size(u, rope, rot):
    """|a| + |b| of each value's pair, what a rotation's rounding errors are relative to."""
    m = np.abs(u)
    if rope:
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if rope == 1 else (slice(0, rot // 2), slice(rot // 2, rot))
        both = m[..., a] + m[..., b]
        m = m.copy()
        m[..., a], m[..., b] = 2 * both, 2 * both
    return m


def check_rows(got, u, f, c):
    want = u * f[..., None]
    tol = half_step(c["dtype"]) * np.abs(want) + 2.0 ** -19 * pair_size(u, c["rope"], c["rot"]) * f[..., None] + 1e-37
    got = got.reshape(want.shape)
    assert (np.abs(got - want) <= tol).all(), np.max((np.abs(got - want) - tol))


def check_cache(data, c, k, v, rows=None):
    want = np.full_like(data, 0x5A)
    for is_v, (u, f) in enumerate((k, v)):
        codes, bits = ref.quantise(u, f, c["cdtype"])
        for t in range(c["tokens"]) if rows is None else rows:
            for h in range(c["kv_heads"]):
                ref.put_row(want, int(c["slot"][t]), h, codes[t, h], bits[t, h], is_v, c["cdtype"], c["dim"], c["page"])
    assert np.array_equal(data, want), f"{(data != want).sum()} bytes of the cache differ"


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("dim,rope,rot,norm", [(8, 1, 8, True), (16, 2, 16, False), (24, 2, 24, True), (32, 1, 20, True), (40, 2, 40, True), (48, 1, 48, False), (64, 2, 64, True), (64, 1, 64, True),
                                               (64, 0, 0, True), (96, 2, 64, True), (128, 2, 128, True), (128, 1, 128, False), (128, 2, 36, True), (160, 2, 160, True), (256, 1, 256, True),
                                               (256, 2, 256, False), (64, 1, 0, False)])
def test_qkv(api, dtype, cdtype, dim, rope, rot, norm):
    rng = np.random.default_rng(dim * 10 + rope)
    for tokens, heads, kv_heads, page, pad, shift in ((1, 2, 1, 16, 0, 0), (37, 3, 3, 48, 0, 0), (19, 4, 2, 16, 3, 1)):
        c = qkv_case(api, rng, dtype, cdtype, tokens, heads, kv_heads, dim, rope, rot, norm, page, pad, shift)
        q, k, v = qkv_want(c)
        got_q, got_k, data, status, _ = qkv_call(api, c, out_pad=pad)
        assert status == 0
        check_rows(got_q[:, :heads * dim], *q, c)
        check_rows(got_k[:, :kv_heads * dim], *k, c)
        assert (got_q[:, heads * dim:] == 7).all() and (got_k[:, kv_heads * dim:] == 7).all()
        check_cache(data, c, k, v)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("rope", [0, 1, 2])
def test_qkv_values_on_the_borders_of_codes(api, dtype, cdtype, rope):
    """Values of few bits, unnormed: many lie exactly between two codes or tie for the largest of their block, and rows at position 0
    stay such after the rotation. The cache has the codes of exact arithmetic."""
    rng = np.random.default_rng(5)
    c = qkv_case(api, rng, dtype, cdtype, 300, 1, 2, 64, rope, 64 if rope else 0, False, ties=True)
    c["pos"][::2] = 0
    q, k, v = qkv_want(c)
    _, _, data, _, _ = qkv_call(api, c)
    check_cache(data, c, k, v)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_qkv_many_rows(api, dtype):
    """Enough normed and rotated keys that some lie within a few 2^-24 of a border between codes."""
    rng = np.random.default_rng(6)
    for cdtype in (ref.Q4, ref.MX):
        c = qkv_case(api, rng, dtype, cdtype, 1500, 1, 4, 128, 2, 128, True, page=64)
        q, k, v = qkv_want(c)
        _, _, data, _, handle = qkv_call(api, c)
        for is_v, (u, f) in enumerate((k, v)):
            codes, bits = ref.quantise(u, f, cdtype)
            want = ref.values(codes, bits, cdtype)
            for h in range(4):
                assert np.array_equal(ref.get_rows(data, c["slot"], h, is_v, cdtype, 128, 64), want[:, h])


def test_qkv_in_place_and_without_a_cache(api):
    rng = np.random.default_rng(7)
    for dtype in (F32, BF16):
        for rope in (1, 2):
            c = qkv_case(api, rng, dtype, ref.Q4, 23, 4, 2, 64, rope, 64, True)
            q, k, v = qkv_want(c)
            got_q, got_k, data, _, _ = qkv_call(api, c, store=True, in_place=True)
            check_rows(got_q, *q, c)
            check_rows(got_k, *k, c)
            check_cache(data, c, k, v)
            c = qkv_case(api, rng, dtype, ref.Q4, 23, 4, 2, 64, rope, 64, True)
            q, k, v = qkv_want(c)
            got_q, got_k, data, _, _ = qkv_call(api, c, store=False)
            check_rows(got_q, *q, c)
            check_rows(got_k, *k, c)
            assert (data == 0x5A).all()


def test_qkv_padding_bad_positions_and_slots(api):
    """Rows with a negative position, and with a position outside the table, are left as they were; a negative slot stores nothing, one past
    the cache is reported."""
    rng = np.random.default_rng(8)
    for dtype in (F32, BF16):
        c = qkv_case(api, rng, dtype, ref.Q4, 40, 2, 2, 48, 1, 48, True)
        c["pos"][[3, 39]] = -1
        c["pos"][5] = 64
        c["slot"][7] = -1
        c["slot"][9] = c["n_pages"] * 16
        q, k, v = qkv_want(c)
        got_q, got_k, data, status, _ = qkv_call(api, c)
        assert status == ref.BAD_POS | ref.BAD_PAGE
        out = np.isin(np.arange(40), [3, 5, 39])
        assert (got_q[out] == 7).all() and (got_k[out] == 7).all()
        for got, (u, f) in ((got_q, q), (got_k, k)):
            check_rows(got[~out], u[~out], f[~out], c)
        check_cache(data, c, k, v, rows=[t for t in range(40) if t not in (3, 5, 7, 9, 39)])


def test_qkv_extreme_values(api):
    """Zeros, the type's largest and smallest values, and NaN: a NaN is stored as zero, scales end at f16's largest."""
    rng = np.random.default_rng(10)
    for cdtype in (ref.Q4, ref.MX):
        c = qkv_case(api, rng, F32, cdtype, 12, 1, 1, 64, 0, 0, False)
        x = c["x"]
        x[0], x[1], x[2] = 0, 3e38, 1e-42
        x[3] *= 1e30
        x[4] *= 1e-30
        x[5] *= np.ldexp(1.0, rng.integers(-60, 60, x.shape[1]))
        x[6, 70], x[6, 140] = np.nan, np.nan
        x = x.astype(np.float32).astype(np.float64)
        c["buf"][:] = api.torch.from_numpy(x).reshape(-1).float().cuda()
        c["x"] = np.nan_to_num(x)
        q, k, v = qkv_want(c)
        _, _, data, _, _ = qkv_call(api, c)
        check_cache(data, c, k, v)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype,dim,page", [(ref.Q4, 64, 16), (ref.MX, 64, 48), (ref.Q4, 40, 32), (ref.MX, 256, 16), (ref.Q4, 8, 64)])
def test_load(api, dtype, cdtype, dim, page):
    rng = np.random.default_rng(dim)
    t, heads, n_pages = api.torch, 3, 5
    host = rng.integers(0, 256, (n_pages, heads, page // 16, ref.tile_bytes(cdtype, dim)), dtype=np.uint8)
    if cdtype == ref.Q4:                                                                        # every scale's bits finite
        view = host[..., 512 * ref.blocks(dim):].view(np.uint16)
        view[...] = np.where(view & 0x7C00 == 0x7C00, view & 0x83FF, view)
    else:
        host[..., 512 * ref.blocks(dim):] = rng.integers(0, 252, host[..., 512 * ref.blocks(dim):].shape)
    data, slots = api.put(host), rng.integers(0, n_pages * page, 77).astype(np.int32)
    slots[5], slots[6] = -1, n_pages * page
    k, v = (t.full((77, heads, dim), 9.0, dtype=t.float32 if dtype == F32 else t.bfloat16, device="cuda") for _ in "kv")
    dev, cache = api.put(slots), api.cache(data, cdtype, page, heads, dim)
    api.ok(api.lib.l3m_kv4_load_dev(C.byref(cache), dtype, k.data_ptr(), v.data_ptr(), dev.data_ptr(), 77, api.stream()))
    good = np.ones(77, bool)
    good[[5, 6]] = False
    for is_v, got in enumerate((k, v)):
        assert (got[~t.from_numpy(good).cuda()] == 9).all()
        for h in range(heads):
            want = t.from_numpy(ref.get_rows(host, slots[good], h, is_v, cdtype, dim, page)).float().to(got.dtype).cuda()
            assert t.equal(got[t.from_numpy(good).cuda(), h], want)
    only = t.full_like(k, 9.0)
    api.ok(api.lib.l3m_kv4_load_dev(C.byref(cache), dtype, None, only.data_ptr(), dev.data_ptr(), 77, api.stream()))
    assert t.equal(only, v)


# ---- attention

def random_cache(rng, cdtype, n_pages, heads, page, dim, scale=0.3):
    """Bytes of a cache of roughly normal values, every scale finite."""
    ng = ref.blocks(dim)
    data = np.empty((n_pages, heads, page // 16, ref.tile_bytes(cdtype, dim)), np.uint8)
    pair = rng.integers(0, 256, 4096).astype(np.uint8) if cdtype == ref.MX else ((rng.normal(8, 2.6, 4096).round().clip(0, 15).astype(np.uint8)) | (rng.normal(8, 2.6, 4096).round().clip(0, 15).astype(np.uint8) << 4))
    data[..., :512 * ng] = pair[rng.integers(0, 4096, data[..., :512 * ng].shape)]
    tail = data[..., 512 * ng:]
    if cdtype == ref.Q4:
        s = (rng.lognormal(0, 0.3, tail.shape[:-1] + (32 * ng,)) * scale * rng.choice([-1, 1], tail.shape[:-1] + (32 * ng,))).astype(np.float16)
        tail[...] = s.view(np.uint8).reshape(tail.shape)
    else:
        tail[...] = rng.integers(124, 127, tail.shape)
    return data


def batch(rng, lens, news, page, n_extra=2, width=None):
    lens = np.asarray(lens)
    held = -(-lens // page)
    n_pages = int(held.sum()) + n_extra
    width = max(1, int(held.max(initial=0))) if width is None else width
    tables = np.full((len(lens), width), -1, np.int32)
    order, at = rng.permutation(n_pages), 0
    for r, b in enumerate(held):
        tables[r, :b] = order[at:at + b]
        at += b
    return tables, np.concatenate(([0], np.cumsum(news))).astype(np.int32), n_pages


def queries(api, rng, rows, heads, dim, dtype, size=1.0):
    q = api.torch.from_numpy(rng.standard_normal((rows, heads, dim)) * size).to(api.torch.float32 if dtype == F32 else api.torch.bfloat16)
    return q.cuda(), q.double().numpy()


def check_attend(got, want, spread, dtype):
    got = got.double().cpu().numpy()
    tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * spread if dtype == BF16 else 2.0 ** -16 * spread
    bad = ~(np.abs(got - want) <= tol + 1e-30)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], float(np.abs(got - want)[bad].max()))


SHAPES = [(1, 1, 16), (2, 1, 24), (4, 4, 32), (6, 6, 48), (9, 3, 64), (5, 1, 64), (8, 2, 40), (8, 1, 80), (16, 4, 96), (32, 8, 128), (12, 1, 128), (24, 2, 64), (7, 1, 160), (4, 2, 192), (8, 1, 256), (3, 1, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
def test_attend_one_token_each(api, dtype, cdtype, heads, kv_heads, dim):
    rng = np.random.default_rng(heads * 1000 + dim)
    for page, lens in ((16, [1, 2, 15, 16, 17, 33, 64, 200]), (48, [300, 47, 48, 49]), (128, [513])):
        tables, q_start, n_pages = batch(rng, lens, [1] * len(lens), page)
        host = random_cache(rng, cdtype, n_pages, kv_heads, page, dim)
        q, q64 = queries(api, rng, len(lens), heads, dim, dtype)
        data = api.put(host)
        out, st = api.attend(api.cache(data, cdtype, page, kv_heads, dim), q, q_start, lens, tables, dim ** -0.5)
        check_attend(out, *ref.attend(q64, q_start, lens, tables, host, cdtype, dim, page, kv_heads, dim ** -0.5), dtype)
        assert st.item() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 16), (9, 3, 64), (6, 6, 48), (8, 2, 128), (16, 2, 96), (12, 1, 64), (4, 1, 256)])
def test_attend_several_tokens(api, dtype, cdtype, heads, kv_heads, dim):
    """Chunks of every kind in one batch: one token, a few, whole prompts, more than a tile, one request with none."""
    rng = np.random.default_rng(heads + dim)
    for page, lens, news in ((16, [5, 40, 130, 77, 3], [5, 1, 130, 9, 0]), (64, [200, 400], [67, 33]), (32, [64], [64])):
        for window in (0, 1, 7, 50):
            tables, q_start, n_pages = batch(rng, lens, news, page)
            host = random_cache(rng, cdtype, n_pages, kv_heads, page, dim)
            q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, dtype)
            out, _ = api.attend(api.cache(api.put(host), cdtype, page, kv_heads, dim), q, q_start, lens, tables, dim ** -0.5, window)
            api.torch.cuda.synchronize()
            check_attend(out, *ref.attend(q64, q_start, lens, tables, host, cdtype, dim, page, kv_heads, dim ** -0.5, window), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("cdtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 16), (9, 3, 64), (6, 6, 48), (16, 4, 128), (16, 2, 96)])
def test_attend_many_rows_over_long_tables(api, dtype, cdtype, heads, kv_heads, dim):
    """Chunks whose rows go 16 to a tile of the cache: work enough by the bounds that the call gives, the tables' width (cut into shares
    and joined) or the number of requests (whole), while the lengths at hand are of every size."""
    rng = np.random.default_rng(heads + dim)
    for lens, news, page, width in (([300, 41, 2, 700, 0, 130], [100, 33, 5, 16, 0, 130], 16, 20000 // kv_heads), ([900, 64], [13, 64], 64, 40000 // kv_heads), (list(rng.integers(1, 200, 400)), [16] * 400, 64, 16)):
        for window in (0, 150):
            tables, q_start, n_pages = batch(rng, lens, news, page, width=width)
            host = random_cache(rng, cdtype, n_pages, kv_heads, page, dim)
            q, q64 = queries(api, rng, int(q_start[-1]), heads, dim, dtype)
            out, st = api.attend(api.cache(api.put(host), cdtype, page, kv_heads, dim), q, q_start, lens, tables, dim ** -0.5, window, max_kv=width * page)
            want, spread = ref.attend(q64, q_start, lens, tables, host, cdtype, dim, page, kv_heads, dim ** -0.5, window)
            got, extra = out.double().cpu().numpy(), 0.0
            if dtype == BF16 and cdtype == ref.Q4:
                # Codes enter as n0 + 16 n1, at most 255, and the parts and the offset are taken off the sums behind: what the f32 sums lose
                # is relative to 255 P times scale, not to the values (a token whose value is 0 loses it, too). A product of 16 tokens
                # adds to them with a truncation of 2^-23 of the largest term and one of the sum: 255 * 2^-22 < 2^-14 of
                # sum(p |scale|) / sum(p) <= the largest scale, for each of a warp's products: two a pair of tiles, every fourth pair at least.
                scales = np.ascontiguousarray(host[..., 544 * ref.blocks(dim):]).view(np.float16)
                extra = 2 * -(-max(lens) // (4 * 32)) * 2.0 ** -14 * float(np.abs(scales).max())
            tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -10 * spread + extra if dtype == BF16 else 2.0 ** -16 * spread
            bad = ~(np.abs(got - want) <= tol + 1e-30)
            assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], float(np.abs(got - want)[bad].max()))
            assert st.item() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens,heads,kv_heads,dim", [([20011], 4, 1, 64), ([9000, 1, 30, 5000], 8, 2, 128), ([4097] * 3, 6, 6, 48)])
def test_attend_long(api, dtype, lens, heads, kv_heads, dim):
    rng = np.random.default_rng(len(lens))
    for cdtype in (ref.Q4, ref.MX):
        tables, q_start, n_pages = batch(rng, lens, [1] * len(lens), 64)
        host = random_cache(rng, cdtype, n_pages, kv_heads, 64, dim)
        q, q64 = queries(api, rng, len(lens), heads, dim, dtype)
        data = api.put(host)
        out, _ = api.attend(api.cache(data, cdtype, 64, kv_heads, dim), q, q_start, lens, tables, dim ** -0.5, max_kv=tables.shape[1] * 64)
        check_attend(out, *ref.attend(q64, q_start, lens, tables, host, cdtype, dim, 64, kv_heads, dim ** -0.5), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attend_rows_that_see_nothing_and_rows_of_nobody(api, dtype):
    """kv_len 0, queries before position 0 (more queries than cached tokens), requests without queries, and rows of q behind the last
    request: zeros for the first two, untouched for the last."""
    rng = np.random.default_rng(3)
    for cdtype in (ref.Q4, ref.MX):
        lens, news = np.array([0, 3, 20, 0, 50]), [2, 7, 0, 0, 1]
        tables, q_start, n_pages = batch(rng, lens, news, 16)
        host = random_cache(rng, cdtype, n_pages, 2, 16, 64)
        q, q64 = queries(api, rng, int(q_start[-1]) + 4, 4, 64, dtype)
        q[-4:] = float("nan")
        out, st = api.attend(api.cache(api.put(host), cdtype, 16, 2, 64), q, q_start, lens, tables, 0.125, max_q=9)
        assert (out[-4:] == 123).all()
        n = int(q_start[-1])
        want, spread = ref.attend(q64, q_start, lens, tables, host, cdtype, 64, 16, 2, 0.125)
        assert (want[:2] == 0).all() and (want[2:6] == 0).all() and (want[6] != 0).any()
        check_attend(out[:n], want[:n], spread[:n], dtype)
        assert st.item() == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attend_windows_beyond_everything(api, dtype):
    """A window as long as the context or as long as an int goes leaves nothing out, for queries before position 0 either."""
    rng = np.random.default_rng(31)
    lens, news = [40, 3, 600], [1, 30, 9]
    tables, q_start, n_pages = batch(rng, lens, news, 16)
    host = random_cache(rng, ref.Q4, n_pages, 2, 16, 64)
    q, q64 = queries(api, rng, int(q_start[-1]), 4, 64, dtype)
    want, spread = ref.attend(q64, q_start, lens, tables, host, ref.Q4, 64, 16, 2, 0.125)
    for window in (600, 1 << 30, (1 << 31) - 1):
        out, _ = api.attend(api.cache(api.put(host), ref.Q4, 16, 2, 64), q, q_start, lens, tables, 0.125, window)
        check_attend(out, want, spread, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 40])
def test_attend_ignores_what_nobody_sees(api, dtype, new):
    """Slots behind a request's last token, tokens outside the window and pages of nobody hold the worst bytes there are (NaN and
    infinite scales): the result's bits do not depend on them."""
    rng = np.random.default_rng(4)
    for cdtype in (ref.Q4, ref.MX):
        for window in (0, 21):
            lens, page = [77, 45, 64], 32
            tables, q_start, n_pages = batch(rng, lens, [new] * 3, page)
            host = random_cache(rng, cdtype, n_pages, 2, page, 64)
            bad = host.copy()
            seen = np.zeros((n_pages, page), bool)
            for r, n in enumerate(lens):
                for t in range(max(0, n - new - window + 1) if window else 0, n):
                    seen[tables[r, t // page], t % page] = True
            ng, width = 2, 2 if cdtype == ref.Q4 else 1
            for pg, t in np.argwhere(~seen):
                for at in (512 * ng, (512 + 16 * width) * ng):
                    cell = at + t % 16 * ng * width
                    bad[pg, :, t // 16, cell:cell + ng * width] = 0xFF if (pg + t) % 2 else 0x7C
                bad[pg, :, t // 16, t % 16 * 32:t % 16 * 32 + 32] = 0xF7
            q, q64 = queries(api, rng, int(q_start[-1]), 6, 64, dtype)
            outs = [api.attend(api.cache(d, cdtype, page, 2, 64), q, q_start, lens, tables, 0.125, window)[0] for d in (api.put(host), api.put(bad))]
            assert api.torch.equal(*outs)
            check_attend(outs[0], *ref.attend(q64, q_start, lens, tables, host, cdtype, 64, page, 2, 0.125, window), dtype)


@pytest.mark.parametrize("new", [1, 30])
def test_attend_bad_pages_are_not_seen(api, new):
    rng = np.random.default_rng(5)
    lens, page = [100, 90], 16
    tables, q_start, n_pages = batch(rng, lens, [new, new], page)
    host = random_cache(rng, ref.Q4, n_pages, 1, page, 64)
    tables[0, 2], tables[0, 5], tables[1, :] = -1, n_pages, 1 << 30
    q, q64 = queries(api, rng, 2 * new, 3, 64, F32)
    out, st = api.attend(api.cache(api.put(host), ref.Q4, page, 1, 64), q, q_start, lens, tables, 0.125)
    assert st.item() == ref.BAD_PAGE
    want, spread = ref.attend(q64, q_start, lens, tables, host, ref.Q4, 64, page, 1, 0.125)
    assert (want[new:] == 0).all()
    check_attend(out, want, spread, F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 24])
def test_attend_scales_of_every_size(api, dtype, new):
    """Scales from the smallest to the largest the formats have, in values and in keys (queries sized to match), block by block of each token."""
    rng = np.random.default_rng(6)
    page, dim, lens = 32, 64, [75, 33]
    for cdtype, lows in ((ref.Q4, (2.0 ** -24, 2.0 ** -14, 0.01, 1.0, 4000.0)), (ref.MX, (1, 30, 100, 127, 160, 230))):
        for lo in lows:
            for mixed in (False, True):
                tables, q_start, n_pages = batch(rng, lens, [new, new], page)
                host = random_cache(rng, cdtype, n_pages, 2, page, dim)
                cells = 16 * 2 * (2 if cdtype == ref.Q4 else 1)
                v_scales = host[..., 1024 + cells:]
                if cdtype == ref.Q4:
                    s = lo * np.exp2(rng.integers(0, 5, v_scales.shape[:-1] + (32,)))
                    s = np.where(rng.random(s.shape) < 0.5, s, 0.02) if mixed else s
                    v_scales[...] = s.astype(np.float16).view(np.uint8).reshape(v_scales.shape)
                else:
                    e = lo + rng.integers(0, 5, v_scales.shape)
                    v_scales[...] = np.where(rng.random(e.shape) < 0.5, e, 120) if mixed else e
                q, q64 = queries(api, rng, int(q_start[-1]), 4, dim, dtype)
                out, _ = api.attend(api.cache(api.put(host), cdtype, page, 2, dim), q, q_start, lens, tables, 0.125)
                want, spread = ref.attend(q64, q_start, lens, tables, host, cdtype, dim, page, 2, 0.125)
                check_attend(out, want, spread, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("new", [1, 24])
def test_attend_queries_of_every_size(api, dtype, new):
    """Queries and key scales at both ends of their range with products of ordinary size, queries whose values differ by 2^40, zero queries,
    and a scale of 0 (a plain mean)."""
    rng = np.random.default_rng(7)
    page, dim, lens = 16, 64, [70, 41]
    tables, q_start, n_pages = batch(rng, lens, [new, new], page)
    rows = int(q_start[-1])
    for cdtype, size in ((ref.Q4, 1e30), (ref.Q4, 1e-30), (ref.MX, 1e30), (ref.MX, 1e-35), (ref.Q4, 1.0), (ref.Q4, 0.0)):
        host = random_cache(rng, cdtype, n_pages, 2, page, dim)
        q, q64 = queries(api, rng, rows, 4, dim, dtype, size)
        if size == 1.0:
            q64 = q64 * np.ldexp(1.0, rng.integers(-40, 1, q64.shape))
            q = api.torch.from_numpy(q64).cuda().to(q.dtype)
            q64 = q.double().cpu().numpy()
        scale = np.float32(0.125 / size if size else 0.125)
        out, _ = api.attend(api.cache(api.put(host), cdtype, page, 2, dim), q, q_start, lens, tables, float(scale))
        check_attend(out, *ref.attend(q64, q_start, lens, tables, host, cdtype, dim, page, 2, float(scale)), dtype)
        out, _ = api.attend(api.cache(api.put(host), cdtype, page, 2, dim), q, q_start, lens, tables, 0.0)
        check_attend(out, *ref.attend(q64, q_start, lens, tables, host, cdtype, dim, page, 2, 0.0), dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attend_sharp_scores(api, dtype):
    """Scores that differ by hundreds, rising and falling along the context: the running maximum moves at every step or never. The scores
    reach 2^9 in magnitude, so f32 scores are off by up to 2^-20 * 2^11 (sum |q k|): the probabilities of near ties by 2^-9."""
    rng = np.random.default_rng(8)
    page, dim, n = 16, 32, 400
    for order in (1, -1, 0):
        tables, q_start, n_pages = batch(rng, [n], [1], page)
        host = random_cache(rng, ref.Q4, n_pages, 1, page, dim)
        for t in range(n):
            size = {1: t, -1: n - t, 0: rng.integers(n)}[order] / n
            ref.put_row(host, int(tables[0, t // page]) * page + t % page, 0, np.full(32, 9, np.uint8), np.array([size * 16], np.float16).view(np.uint16), 0, ref.Q4, dim, page)
        q, q64 = queries(api, rng, 1, 2, dim, dtype)
        q64 = np.abs(q64)
        q = api.torch.from_numpy(q64).to(q.dtype).cuda()
        out, _ = api.attend(api.cache(api.put(host), ref.Q4, page, 1, dim), q, q_start, [n], tables, 1.0)
        want, spread = ref.attend(q64, q_start, [n], tables, host, ref.Q4, dim, page, 1, 1.0)
        assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -8 * spread + 2.0 ** -8 * np.abs(want)).all()


def test_attend_strides_and_the_same_bits_twice(api):
    """Queries and outputs inside wider matrices, at addresses that are not 16-byte aligned; the spare columns stay, and two calls agree bit for bit."""
    rng, t = np.random.default_rng(9), api.torch
    page, dim, heads, lens, news = 16, 40, 6, [50, 130, 7], [1, 33, 2]
    tables, q_start, n_pages = batch(rng, lens, news, page)
    host = random_cache(rng, ref.MX, n_pages, 2, page, dim)
    for dtype in (F32, BF16):
        kind, rows, width = t.float32 if dtype == F32 else t.bfloat16, int(q_start[-1]), heads * dim
        big = t.from_numpy(rng.standard_normal((rows, width + 13))).to(kind).cuda()
        flat = t.empty(rows * (width + 13) + 1, dtype=kind, device="cuda")
        flat[1:] = big.reshape(-1)
        q = flat[1:].as_strided((rows, heads, dim), (width + 13, dim, 1), 1)
        outs = []
        for _ in range(2):
            space = t.full((rows * (width + 5) + 1,), 5.0, dtype=kind, device="cuda")
            api.attend(api.cache(api.put(host), ref.MX, page, 2, dim), q, q_start, lens, tables, 0.2, out=space.as_strided((rows, heads, dim), (width + 5, dim, 1), 1))
            outs.append(space)
        assert t.equal(*outs)
        got = outs[0][1:].view(rows, width + 5)
        assert (got[:, width:] == 5).all() and outs[0][0] == 5
        check_attend(got[:, :width].reshape(rows, heads, dim), *ref.attend(big[:, :width].reshape(rows, heads, dim).double().cpu().numpy(), q_start, lens, tables, host, ref.MX, dim, page, 2, 0.2), dtype)


def test_offsets_past_32_bits(api):
    """A cache of 5 GB: pages near its end hold the tokens, written by the store, read by the load and by attention."""
    rng, t = np.random.default_rng(11), api.torch
    page, dim, heads = 64, 128, 8
    per = ref.tile_bytes(ref.Q4, dim) * heads * page // 16
    n_pages = 5 * 10 ** 9 // per
    data = t.empty(n_pages, heads, page // 16, ref.tile_bytes(ref.Q4, dim), dtype=t.uint8, device="cuda")
    n, x = 100, rng.standard_normal((100, (8 + 16) * dim))
    tables = np.array([[n_pages - 1, n_pages - 3]], np.int32)
    slot = np.concatenate((np.arange(64) + (n_pages - 1) * page, np.arange(36) + (n_pages - 3) * page)).astype(np.int32)
    dev, d_slot, d_pos = t.from_numpy(x).float().cuda(), api.put(slot), api.put(np.arange(n, dtype=np.int32))
    q_out = t.zeros(n, 8 * dim, device="cuda")
    cache = api.cache(data, ref.Q4, page, heads, dim)
    a = api.l3m.Qkv(dtype=F32, n_tokens=n, n_heads=8, n_kv_heads=heads, head_dim=dim, pos=d_pos.data_ptr(), slot=d_slot.data_ptr(), q=dev.data_ptr(), k=dev.data_ptr() + 8 * dim * 4,
                    v=dev.data_ptr() + 16 * dim * 4, q_ld=24 * dim, k_ld=24 * dim, v_ld=24 * dim, q_out=q_out.data_ptr(), q_out_ld=8 * dim)
    api.ok(api.lib.l3m_qkv_rope_dev(C.byref(cache), C.byref(a), api.stream()))
    kv = [t.zeros(n, heads, dim, device="cuda") for _ in "kv"]
    api.ok(api.lib.l3m_kv4_load_dev(C.byref(cache), F32, kv[0].data_ptr(), kv[1].data_ptr(), d_slot.data_ptr(), n, api.stream()))
    rows = x.astype(np.float32).astype(np.float64).reshape(n, 24, dim)
    for i, got in enumerate(kv):
        part = rows[:, 8 + 8 * i:16 + 8 * i]
        assert np.array_equal(got.double().cpu().numpy(), ref.values(*ref.quantise(part, np.ones(part.shape[:2]), ref.Q4), ref.Q4))
    for new in (1, n):
        q = q_out[n - new:].view(new, 8, dim)
        out, _ = api.attend(cache, q, np.array([0, new]), [n], tables, 0.1)
        small = np.stack([data[p].cpu().numpy() for p in (n_pages - 1, n_pages - 3)])
        check_attend(out, *ref.attend(q.double().cpu().numpy(), [0, new], [n], np.array([[0, 1]]), small, ref.Q4, dim, page, heads, 0.1), F32)
    del data


# ---- together

@pytest.mark.parametrize("dtype,cdtype", [(F32, ref.Q4), (BF16, ref.MX)])
@pytest.mark.parametrize("graph", [False, True])
def test_serving_steps(api, dtype, cdtype, graph):
    """Plan, store and attend as a server calls them, step after step, on a stream of its own: prompts, then single tokens over page ends,
    a request that ends and one that takes its place. With `graph` the steps after the prompts are one captured graph, replayed. Every
    step's bookkeeping, cache and attention are the restatements'."""
    t, rng = api.torch, np.random.default_rng(20)
    n, page, width, heads, kh, dim, most, n_pages = 3, 16, 6, 6, 2, 64, 48, 14
    kind = t.float32 if dtype == F32 else t.bfloat16
    i32 = dict(dtype=t.int32, device="cuda")
    s = t.cuda.Stream()
    kv, new, tables = t.zeros(n, **i32), t.zeros(n, **i32), t.full((n, width), -1, **i32)
    free, top, slot, pos, q_start, total, st = t.arange(n_pages, **i32), [t.tensor([n_pages], **i32), t.zeros(1, **i32)], t.zeros(most, **i32), t.zeros(most, **i32), t.zeros(n + 1, **i32), t.zeros(n, **i32), t.zeros(1, **i32)
    x = t.zeros(most, (heads + 2 * kh) * dim, dtype=kind, device="cuda")
    q_out, out = t.zeros(most, heads, dim, dtype=kind, device="cuda"), t.full((most, heads, dim), 55.0, dtype=kind, device="cuda")
    data = t.zeros(n_pages, kh, 1, ref.tile_bytes(cdtype, dim), dtype=t.uint8, device="cuda")
    turn = np.stack((np.cos(np.outer(np.arange(128), 0.8 ** np.arange(dim // 2))), np.sin(np.outer(np.arange(128), 0.8 ** np.arange(dim // 2)))), -1).astype(np.float32)
    d_turn, w = api.put(turn), [(1 + 0.2 * rng.standard_normal(dim)).astype(np.float32) for _ in "qk"]
    d_w, size, cache = [api.put(a) for a in w], x.element_size(), api.cache(data, cdtype, page, kh, dim)
    P = lambda a: a.data_ptr()      # noqa: E731
    plan = api.l3m.Kv4Plan(n_req=n, max_blocks=width, max_tokens=most, page=page, n_pages=n_pages, kv_len=P(kv), new_len=P(new), tables=P(tables), free_pages=P(free), n_free=P(top[0]),
                           n_free_out=P(top[1]), q_start=P(q_start), kv_total=P(total), slot=P(slot), pos=P(pos), status=P(st))
    qkv = api.l3m.Qkv(dtype=dtype, n_tokens=most, n_heads=heads, n_kv_heads=kh, head_dim=dim, rope=2, rot_dim=dim, n_pos=128, eps=1e-6, q_norm=P(d_w[0]), k_norm=P(d_w[1]), rope_table=P(d_turn),
                      pos=P(pos), slot=P(slot), q=P(x), k=P(x) + heads * dim * size, v=P(x) + (heads + kh) * dim * size, q_ld=x.shape[1], k_ld=x.shape[1], v_ld=x.shape[1], q_out=P(q_out),
                      q_out_ld=heads * dim, status=P(st))
    att = api.l3m.Kv4Attend(dtype=dtype, n_heads=heads, n_req=n, max_blocks=width, max_q=most, max_kv=width * page, scale=0.125, q=P(q_out), out=P(out), q_ld=heads * dim, out_ld=heads * dim,
                            q_start=P(q_start), kv_len=P(total), tables=P(tables), status=P(st))
    scratch = t.empty(max(16, api.lib.l3m_kv4_attend_scratch(C.byref(cache), C.byref(att))), dtype=t.uint8, device="cuda")
    att.scratch, att.scratch_bytes = P(scratch), scratch.numel()

    def step():
        api.ok(api.lib.l3m_kv4_plan_dev(C.byref(plan), s.cuda_stream))
        top[0].copy_(top[1])
        api.ok(api.lib.l3m_qkv_rope_dev(C.byref(cache), C.byref(qkv), s.cuda_stream))
        api.ok(api.lib.l3m_kv4_attend_dev(C.byref(cache), C.byref(att), s.cuda_stream))

    w_kv, w_tables, w_free, w_top = np.zeros(n, np.int32), np.full((n, width), -1, np.int32), np.arange(n_pages, dtype=np.int32), n_pages
    w_data, w_out, captured = np.zeros(data.shape, np.uint8), np.full((most, heads, dim), 55.0), None
    steps = [[17, 5, 0], [1, 1, 20]] + [[1, 1, 1]] * 13 + [[1, -1, 1], [1, 30, 1], [1, 1, 1], [-1, -1, -1]]
    with t.cuda.stream(s):
        for count, news in enumerate(steps):
            fresh = t.from_numpy(rng.standard_normal(x.shape)).to(kind)
            x.copy_(fresh)
            kv.copy_(t.from_numpy(w_kv))
            new.copy_(t.tensor(news, dtype=t.int32))
            s.synchronize()
            if graph and count >= 2:
                if captured is None:
                    captured = t.cuda.CUDAGraph()
                    with t.cuda.graph(captured, stream=s):
                        step()
                captured.replay()
            else:
                step()
            s.synchronize()
            want = ref.plan(w_kv, np.array(news), w_tables, w_free, w_top, page, most)
            assert want["status"] == 0 and st.item() == 0
            for k, got in dict(tables=tables, free_pages=free, q_start=q_start, kv_total=total, slot=slot, pos=pos).items():
                assert np.array_equal(got.cpu().numpy(), want[k]), (count, k)
            assert top[0].item() == want["n_free_out"]
            rows = int(want["q_start"][-1])
            x64 = fresh.double().numpy()[:rows].reshape(rows, heads + 2 * kh, dim)
            turned = [ref.normed_rotated(x64[:, lo:hi], w[i].astype(np.float64), 1e-6, turn.astype(np.float64)[want["pos"][:rows]], 2, dim) for i, (lo, hi) in enumerate(((0, heads), (heads, heads + kh)))]
            for is_v, (u, f) in enumerate((turned[1], (x64[:, heads + kh:], np.ones((rows, kh))))):
                codes, bits = ref.quantise(u, f, cdtype)
                for i in range(rows):
                    for h in range(kh):
                        ref.put_row(w_data, int(want["slot"][i]), h, codes[i, h], bits[i, h], is_v, cdtype, dim, page)
            assert np.array_equal(data.cpu().numpy(), w_data), count
            q64 = q_out.double().cpu().numpy()[:rows]
            u, f = turned[0]
            assert (np.abs(q64 - u * f[..., None]) <= (half_step(dtype) + 2.0 ** -17) * pair_size(u, 2, dim) * f[..., None]).all()
            o, spread = ref.attend(q64, want["q_start"], want["kv_total"], want["tables"], w_data, cdtype, dim, page, kh, 0.125)
            got = out.double().cpu().numpy()
            assert np.array_equal(got[rows:], w_out[rows:]), "rows behind the last request changed"
            if rows:
                check_attend(out[:rows], o[:rows], spread[:rows], dtype)
            w_out = got
            w_kv = np.where(np.array(news) < 0, 0, want["kv_total"]).astype(np.int32)
            w_tables, w_free, w_top = want["tables"], want["free_pages"], want["n_free_out"]
    del captured


def test_calls_on_two_streams_at_once(api):
    """Two attentions on two streams, each with its scratch, interleaved many times: each gives what it gives alone."""
    t, rng = api.torch, np.random.default_rng(30)
    jobs = []
    for lens, page, dim, heads, kh, dtype in (([3000, 10], 32, 64, 8, 2, F32), ([700] * 6, 16, 128, 8, 1, BF16)):
        tables, q_start, n_pages = batch(rng, lens, [1] * len(lens), page)
        host = random_cache(rng, ref.Q4, n_pages, kh, page, dim)
        q, q64 = queries(api, rng, len(lens), heads, dim, dtype)
        data = api.put(host)
        cache = api.cache(data, ref.Q4, page, kh, dim)
        out, _ = api.attend(cache, q, q_start, lens, tables, 0.1)
        t.cuda.synchronize()
        jobs.append((cache, api.keep, out, out.clone(), t.cuda.Stream(), data, q))
    for _, _, out, _, _, _, _ in jobs:
        out.zero_()
    t.cuda.synchronize()
    for _ in range(50):
        for cache, keep, out, _, s, _, _ in jobs:
            api.ok(api.lib.l3m_kv4_attend_dev(C.byref(cache), C.byref(keep[3]), s.cuda_stream))
    t.cuda.synchronize()
    for _, _, out, want, _, _, _ in jobs:
        assert t.equal(out, want)
