"""The paged 4-bit cache's entry points on the CPU: sizes, and every refusal (arguments are checked before anything touches a GPU)."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref


@pytest.fixture(scope="module")
def lib():
    import l3m_b200
    return l3m_b200.lib()


def cache(**kw):
    import l3m_b200
    return l3m_b200.Kv4(**{**dict(data=4096, dtype=ref.Q4, n_pages=8, page=16, n_kv_heads=2, head_dim=64), **kw})


BAD_CACHES = [(dict(dtype=2), b"dtype"), (dict(dtype=5), b"dtype"), (dict(head_dim=0), b"head_dim"), (dict(head_dim=12), b"head_dim"), (dict(head_dim=264), b"head_dim"),
              (dict(n_kv_heads=0), b"n_kv_heads"), (dict(page=0), b"page"), (dict(page=24), b"page"), (dict(page=8192), b"page"), (dict(n_pages=-1), b"2^31"),
              (dict(n_pages=1 << 27), b"2^31"), (dict(data=None), b"aligned"), (dict(data=4104), b"aligned")]


@pytest.mark.parametrize("dtype", [ref.Q4, ref.MX])
@pytest.mark.parametrize("dim", [8, 32, 40, 64, 96, 128, 256])
def test_page_bytes(lib, dtype, dim):
    for heads, page in ((1, 16), (3, 64), (8, 48)):
        assert lib.l3m_kv4_page_bytes(dtype, heads, dim, page) == ref.tile_bytes(dtype, dim) * heads * page // 16


def test_page_bytes_of_no_cache_is_zero(lib):
    for args in ((2, 1, 64, 16), (3, 0, 64, 16), (3, 1, 12, 16), (3, 1, 64, 20)):
        assert lib.l3m_kv4_page_bytes(*args) == 0


def plan(**kw):
    import l3m_b200
    base = dict(n_req=2, max_blocks=4, max_tokens=8, page=16, n_pages=8)
    base.update({f: 64 * (i + 1) for i, f in enumerate(("kv_len", "new_len", "tables", "free_pages", "n_free", "n_free_out", "q_start", "kv_total", "slot", "pos"))})
    return l3m_b200.Kv4Plan(**{**base, **kw})


@pytest.mark.parametrize("change,why", [
    (dict(n_req=-1), b"n_req"), (dict(n_req=16385), b"n_req"), (dict(page=8), b"page"), (dict(page=40), b"page"), (dict(max_tokens=-1), b"negative"), (dict(max_tokens=(1 << 30) + 1), b"2^30"), (dict(max_blocks=-1), b"negative"),
    (dict(n_pages=-1), b"negative"), (dict(n_pages=1 << 28), b"2^31")] + [(dict([(f, None)]), b"missing") for f in
    ("kv_len", "new_len", "tables", "free_pages", "n_free", "n_free_out", "q_start", "kv_total", "slot", "pos")] + [
    (dict(n_free_out=64 * 5), b"must not be"), (dict(kv_total=64), b"must not be"), (dict(kv_total=128), b"must not be"), (dict(kv_len=66), b"aligned")])
def test_plan_refuses(lib, change, why):
    assert lib.l3m_kv4_plan_dev(C.byref(plan(**change)), None) == -1
    assert b"l3m_kv4_plan_dev" in lib.l3m_cuda_error() and why in lib.l3m_cuda_error(), lib.l3m_cuda_error()


def qkv(**kw):
    import l3m_b200
    base = dict(dtype=0, n_tokens=4, n_heads=4, n_kv_heads=2, head_dim=64, rope=1, rot_dim=64, n_pos=32, eps=1e-5, q_norm=64, k_norm=64, rope_table=64, pos=64, slot=64, q=64, k=64, v=64,
                q_ld=512, k_ld=512, v_ld=512, q_out=64, k_out=64, q_out_ld=256, k_out_ld=128)
    return l3m_b200.Qkv(**{**base, **kw})


@pytest.mark.parametrize("change,why", [
    (dict(dtype=2), b"dtype"), (dict(n_tokens=-1), b"counts"), (dict(n_heads=-1), b"counts"), (dict(n_kv_heads=1 << 17), b"counts"), (dict(head_dim=20), b"head_dim"), (dict(rope=3), b"rope"),
    (dict(rot_dim=63), b"rot_dim"), (dict(rot_dim=66), b"rot_dim"), (dict(rope_table=None), b"table"), (dict(rope_table=68), b"8-byte"), (dict(eps=-1.0), b"eps"), (dict(eps=float("nan")), b"eps"),
    (dict(n_kv_heads=4), b"another"), (dict(head_dim=32, rot_dim=32), b"another"), (dict(k=None), b"needs"), (dict(v=None), b"needs"), (dict(slot=None), b"needs"), (dict(pos=None), b"pos"),
    (dict(q=None), b"q_out"), (dict(q_out=None), b"q_out"), (dict(q_ld=255), b"stride"), (dict(k_ld=127), b"stride"), (dict(v_ld=127), b"stride"), (dict(q_out_ld=255), b"stride"),
    (dict(k_out_ld=127), b"stride"), (dict(q=66), b"aligned"), (dict(q_norm=66), b"aligned"), (dict(pos=66), b"aligned"), (dict(status=66), b"aligned"), (dict(dtype=1, v=65), b"aligned")])
def test_qkv_refuses(lib, change, why):
    c = cache()
    assert lib.l3m_qkv_rope_dev(C.byref(c), C.byref(qkv(**change)), None) == -1
    assert b"l3m_qkv_rope_dev" in lib.l3m_cuda_error() and why in lib.l3m_cuda_error(), lib.l3m_cuda_error()


def test_qkv_without_a_cache_needs_k_for_k_out(lib):
    assert lib.l3m_qkv_rope_dev(None, C.byref(qkv(k=None)), None) == -1 and b"k_out needs k" in lib.l3m_cuda_error()
    assert lib.l3m_qkv_rope_dev(None, C.byref(qkv(n_tokens=0, pos=None)), None) == 0


def attend(**kw):
    import l3m_b200
    base = dict(dtype=0, n_heads=4, n_req=2, max_blocks=4, max_q=1, max_kv=64, window=0, scale=0.1, q=64, out=128, q_ld=256, out_ld=256, q_start=64, kv_len=64, tables=64, scratch=64,
                scratch_bytes=1 << 40)
    return l3m_b200.Kv4Attend(**{**base, **kw})


@pytest.mark.parametrize("change,why", [
    (dict(dtype=3), b"dtype"), (dict(n_heads=3), b"n_heads"), (dict(n_heads=0), b"n_heads"), (dict(n_req=-1), b"negative"), (dict(max_q=-1), b"negative"), (dict(max_kv=-1), b"negative"),
    (dict(window=-1), b"negative"), (dict(max_q=(1 << 28) + 1), b"2^30"), (dict(scale=-3e38), b"scale"), (dict(status=66), b"aligned"), (dict(max_kv=65), b"max_kv"), (dict(scale=float("inf")), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(q=None), b"missing"), (dict(out=None), b"missing"),
    (dict(q_start=None), b"missing"), (dict(kv_len=None), b"missing"), (dict(tables=None), b"missing"), (dict(q_ld=255), b"stride"), (dict(out_ld=255), b"stride"), (dict(q=66), b"aligned"),
    (dict(tables=65), b"aligned"), (dict(scratch=None), b"scratch"), (dict(scratch=72), b"scratch"), (dict(scratch_bytes=1), b"scratch")])
def test_attend_refuses(lib, change, why):
    c = cache()
    assert lib.l3m_kv4_attend_dev(C.byref(c), C.byref(attend(**change)), None) == -1
    assert b"l3m_kv4_attend_dev" in lib.l3m_cuda_error() and why in lib.l3m_cuda_error(), lib.l3m_cuda_error()


@pytest.mark.parametrize("change,why", BAD_CACHES)
def test_bad_caches_are_refused(lib, change, why):
    c = cache(**change)
    for call in (lambda: lib.l3m_kv4_attend_dev(C.byref(c), C.byref(attend()), None), lambda: lib.l3m_qkv_rope_dev(C.byref(c), C.byref(qkv()), None),
                 lambda: lib.l3m_kv4_load_dev(C.byref(c), 0, 64, 64, 64, 1, None)):
        assert call() == -1 and why in lib.l3m_cuda_error(), lib.l3m_cuda_error()


def test_a_cache_of_too_many_tiles_is_refused(lib):
    c = cache(n_pages=1 << 16, n_kv_heads=1 << 15)
    assert lib.l3m_kv4_load_dev(C.byref(c), 0, 64, 64, 64, 1, None) == -1 and b"2^31 tiles" in lib.l3m_cuda_error()


def test_plan_restatement_leaves_out_bad_pages_and_lengths_at_the_end_of_int32():
    tables = np.array([[7, 1, -1], [2, -1, -1]], np.int32)
    got = ref.plan(np.array([20, 3], np.int32), np.array([13, 1], np.int32), tables, np.array([0, 3, 4, 5, 0, 0], np.int32), 4, 16, 16)
    assert got["status"] == 0 and list(got["slot"][:13]) == [1 * 16 + 4 + i for i in range(12)] + [5 * 16]
    got = ref.plan(np.array([14, 3], np.int32), np.array([3, 1], np.int32), tables, np.array([0, 3, 4, 5, 0, 0], np.int32), 4, 16, 16)
    assert got["status"] == ref.BAD_PAGE and list(got["slot"][:4]) == [-1, -1, 5 * 16, 2 * 16 + 3]
    got = ref.plan(np.array([2 ** 31 - 17], np.int32), np.array([1], np.int32), np.zeros((1, 1), np.int32), np.zeros(1, np.int32), 0, 16, 1)
    assert got["status"] & ref.BAD_LENGTH


def test_null_arguments_are_refused(lib):
    c = cache()
    assert lib.l3m_kv4_plan_dev(None, None) == -1 and lib.l3m_qkv_rope_dev(None, None, None) == -1
    assert lib.l3m_kv4_attend_dev(None, C.byref(attend()), None) == -1 and lib.l3m_kv4_attend_dev(C.byref(c), None, None) == -1
    assert lib.l3m_kv4_load_dev(None, 0, 64, 64, 64, 1, None) == -1


@pytest.mark.parametrize("args,why", [((2, 64, 64, 64, 1), b"dtype"), ((0, 64, 64, None, 1), b"slots"), ((0, 66, 64, 64, 1), b"aligned"), ((0, 64, 64, 64, -1), b"negative")])
def test_load_refuses(lib, args, why):
    c = cache()
    assert lib.l3m_kv4_load_dev(C.byref(c), *args, None) == -1 and why in lib.l3m_cuda_error()


def test_nothing_to_do_launches_nothing(lib):
    c = cache()
    assert lib.l3m_kv4_load_dev(C.byref(c), 0, 64, 64, None, 0, None) == 0
    assert lib.l3m_kv4_load_dev(C.byref(c), 0, None, None, None, 5, None) == 0
    assert lib.l3m_kv4_attend_dev(C.byref(c), C.byref(attend(n_req=0, q=None)), None) == 0
    assert lib.l3m_kv4_attend_dev(C.byref(c), C.byref(attend(max_q=0)), None) == 0


def test_scratch_size(lib):
    c = cache()
    assert lib.l3m_kv4_attend_scratch(C.byref(c), C.byref(attend())) >= 16
    assert lib.l3m_kv4_attend_scratch(C.byref(c), C.byref(attend(n_heads=3))) == 0
    assert lib.l3m_kv4_attend_scratch(C.byref(c), C.byref(attend(q=None, out=None, scratch=None, scratch_bytes=0))) >= 16


def test_scratch_size_of_prompt_chunks(lib):
    """Long contexts need scratch for their split, but for bf16 chunks of thousands of rows at 33 .. 64 and 97 .. 128 dims, which are not split."""
    def size(dim, **kw):
        c = cache(head_dim=dim, n_kv_heads=4)
        return lib.l3m_kv4_attend_scratch(C.byref(c), C.byref(attend(**dict(dict(n_heads=16, dtype=1, n_req=4, max_q=1024, max_blocks=4096, max_kv=65536), **kw))))
    assert size(128) == size(104) == size(64) == size(40) == 16
    for kw in (dict(dtype=0), dict(max_q=8), dict(n_req=1, max_q=256)):
        assert size(128, **kw) > 16
    assert size(96) > 16 and size(32) > 16 and size(136) > 16
    assert size(128, n_req=1 << 21) > 16 and size(128, max_q=1 << 24) > 16
    assert size(128, max_q=0) > 16 and size(128, n_req=0) > 16
