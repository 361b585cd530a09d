"""The paged 4-bit cache on a B200 where calls are at the edge of what they allow, against the 64-bit restatements of kv4_ref.py.
Tolerances are those of test_gpu_kv4.py and test_gpu_kv4_prompt.py, where they are derived."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import BF16, F32, Api, batch, check_attend, queries, random_cache
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
