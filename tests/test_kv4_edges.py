"""The paged 4-bit cache on the CPU: what a step that does not fit leaves behind, and refusals of calls at the edges of the contract."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref
from test_kv4 import attend, cache, lib, qkv  # noqa: F401


def test_a_plan_without_room_counts_rows_past_its_tensors():
    """q_start goes on counting behind max_tokens, so whoever takes rows from it has to be told where the tensors end."""
    tables = np.array([[0, -1], [1, -1], [2, -1]], np.int32)
    got = ref.plan(np.array([3, 2, 1], np.int32), np.array([4, 5, 6], np.int32), tables, np.array([3, 4, 5], np.int32), 3, 16, 10)
    assert got["status"] == ref.NO_ROOM and list(got["q_start"]) == [0, 4, 9, 15] and list(got["kv_total"]) == [7, 7, 0]


def test_attend_refuses_a_negative_row_count(lib):  # noqa: F811
    c = cache()
    assert lib.l3m_kv4_attend_dev(C.byref(c), C.byref(attend(max_rows=-1)), None) == -1 and b"negative" in lib.l3m_cuda_error()
    assert lib.l3m_kv4_attend_scratch(C.byref(c), C.byref(attend(max_rows=-1))) == 0
    assert lib.l3m_kv4_attend_scratch(C.byref(c), C.byref(attend(max_rows=3))) >= 16


@pytest.mark.parametrize("change", [dict(q_out=64, q_out_ld=256, q_ld=512), dict(q_out=64, q_out_ld=768), dict(q_out=4096, k_out=64, k_out_ld=128)])
def test_qkv_in_place_refuses_another_stride(lib, change):  # noqa: F811
    """A row's result would land on rows that are still to be read."""
    c = cache()
    base = dict(q=64, q_out=4096, k=64, k_out=8192, k_ld=512)
    assert lib.l3m_qkv_rope_dev(C.byref(c), C.byref(qkv(**{**base, **change})), None) == -1
    assert b"in place" in lib.l3m_cuda_error(), lib.l3m_cuda_error()
