"""The paged-cache operators without a GPU: what they refuse, rotations that cannot be made, and their index arithmetic.

The refused calls carry addresses that no call may touch."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest

import jetsonfabric_amd as jf
from jetsonfabric_amd import _capi
from jetsonfabric_amd._capi import check

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT = 1 << 20  # an aligned address; nothing is there


def rows(**kw):
    return _capi.Rows(**{"data": AT, "row_stride": 256, "head_stride": 64, "n_rows": 3, "n_head": 4, "head_dim": 64,
                         "type": 2, **kw})


def cache(**kw):
    return _capi.PagedCache(**{"k": AT, "v": AT, "weights": AT, "positions": AT, "page_stride": 4096, "head_stride": 1024,
                               "slot_stride": 64, "n_pages": 9, "page_size": 16, "n_head_kv": 4, "head_dim": 64, "type": 2,
                               "device": 0, **kw})


def batch(**kw):
    return _capi.PagedBatch(**{"table": AT, "lengths": AT, "row_starts": AT, "n_seq": 2, "table_stride": 4, "max_rows": 3,
                               "max_length": 64, **kw})


def refused(call, match):
    with pytest.raises(jf.InvalidArgument, match=match):
        check(call())


BAD_CACHES = [({"k": None}, "aligned"), ({"v": AT + 8}, "aligned"), ({"type": 1}, "f16 or bf16"), ({"type": 9}, "f16 or bf16"),
              ({"n_pages": 0}, "pages"), ({"n_pages": 1 << 31}, "pages"), ({"page_size": 24}, "power of two"),
              ({"page_size": 0}, "power of two"), ({"page_size": 1 << 17}, "power of two"), ({"n_head_kv": 0}, "heads"),
              ({"head_dim": 60}, "head dim"), ({"head_dim": 264}, "head dim"), ({"head_dim": 0}, "head dim"),
              ({"slot_stride": 65}, "strides"), ({"head_stride": -1024}, "strides"), ({"page_stride": 4100}, "strides"),
              ({"slot_stride": 56}, "overlap"), ({"head_stride": 8}, "overlap"), ({"page_stride": 0}, "overlap"),
              ({"weights": AT + 2}, "aligned"), ({"positions": AT + 1}, "aligned")]
BAD_BATCHES = [({"table": None}, "table, lengths"), ({"lengths": None}, "table, lengths"),
               ({"row_starts": None}, "row starts"), ({"max_length": 65}, "max_length"), ({"table_stride": 3}, "max_length"),
               ({"table_stride": 1 << 31, "max_length": (1 << 31) - 1}, "2\\^31"), ({"max_rows": 1 << 31}, "2\\^31"),
               ({"n_seq": 1 << 24}, "sequences")]


def _append(c=None, b=None, k=None, v=None, rope=None, positions=AT):
    return jf.library().jfh_paged_append(ctypes.byref(c or cache()), ctypes.byref(b or batch()), ctypes.byref(k or rows()),
                                         ctypes.byref(v or rows()), rope, positions, None)


@pytest.mark.parametrize("change,match", BAD_CACHES)
def test_caches_are_checked(change, match):
    refused(lambda: _append(c=cache(**change)), match)


@pytest.mark.parametrize("change,match", BAD_BATCHES)
def test_batches_are_checked(change, match):
    refused(lambda: _append(b=batch(**change)), match)


@pytest.mark.parametrize("change,match", [
    ({"data": None}, "k rows are missing"), ({"data": AT + 1}, "aligned"), ({"type": 1, "data": AT + 2}, "aligned"),
    ({"type": 0}, "value type"), ({"type": 4}, "value type"), ({"n_head": 3}, "heads and head dim"),
    ({"head_dim": 32}, "heads and head dim"), ({"n_head": 0}, "no heads"), ({"row_stride": -1}, "negative stride"),
    ({"n_rows": 4}, "same rows"), ({"n_rows": 1 << 31}, "more rows"), ({"n_head": 65536, "head_dim": 512}, "too many values")])
def test_appended_rows_are_checked(change, match):
    refused(lambda: _append(k=rows(**change)), match)


def test_appends_ask_for_positions():
    refused(lambda: _append(positions=None), "positions are required")
    refused(lambda: _append(c=cache(positions=None), positions=None, rope=jf.Rope(64).handle), "positions are required")
    refused(lambda: _append(positions=AT + 2), "aligned")
    refused(lambda: _append(rope=jf.Rope(66).handle), "more values than a head")


def _attend(c=None, b=None, q=None, out=None, scale=0.125, lse=AT, space=AT, size=1 << 40):
    return jf.library().jfh_paged_attention(ctypes.byref(c or cache()), ctypes.byref(b or batch()), ctypes.byref(q or rows()),
                                            scale, 1, ctypes.byref(out or rows()), lse, space, size, None)


@pytest.mark.parametrize("change,match", BAD_CACHES)
def test_attended_caches_are_checked(change, match):
    refused(lambda: _attend(c=cache(**change)), match)


@pytest.mark.parametrize("change,match", BAD_BATCHES)
def test_attended_batches_are_checked(change, match):
    refused(lambda: _attend(b=batch(**change)), match)


@pytest.mark.parametrize("change,match", [
    ({"type": 3}, "cache's type"), ({"type": 1}, "cache's type"), ({"head_dim": 32}, "head dim"), ({"n_head": 6}, "multiple of"),
    ({"data": AT + 8}, "16-byte"), ({"row_stride": 260}, "16-byte"), ({"head_stride": 4}, "16-byte"), ({"n_rows": 2}, "same rows"),
    ({"n_head": 8}, "same rows and heads"), ({"n_rows": (1 << 31) - 1}, "more rows"), ({"data": None}, "missing")])
def test_attention_rows_are_checked(change, match):
    refused(lambda: _attend(q=rows(**change)), match)
    if "same rows" not in match:
        refused(lambda: _attend(out=rows(**change)), match)


def test_attention_arguments_are_checked():
    for scale in (0.0, -1.0, float("nan"), float("inf"), 3e38):
        refused(lambda: _attend(scale=scale), "score scale")
    refused(lambda: _attend(lse=AT + 2), "lse")
    long = {"b": batch(n_seq=1, table_stride=4096, max_length=65536), "c": cache(page_size=16)}
    need = ctypes.c_size_t()
    check(jf.library().jfh_paged_attention_workspace(ctypes.byref(long["c"]), ctypes.byref(long["b"]), ctypes.byref(rows()),
                                                     ctypes.byref(need)))
    assert need.value > 0
    refused(lambda: _attend(**long, size=need.value - 1), f"needs {need.value} bytes")
    refused(lambda: _attend(**long, space=None), "workspace")
    refused(lambda: _attend(**long, space=AT + 4), "16-byte")
    check(_attend(q=rows(n_rows=0), out=rows(n_rows=0)))
    check(_attend(b=batch(n_seq=0)))


def _weigh(c=None, b=None, q=None, scale=0.125, lse=AT, space=AT, size=1 << 40):
    return jf.library().jfh_paged_weigh(ctypes.byref(c or cache()), ctypes.byref(b or batch()), ctypes.byref(q or rows()),
                                        lse, scale, 1, space, size, None)


def _evict(c=None, b=None, budget=8, first=4, recent=2, space=AT, size=1 << 40):
    return jf.library().jfh_paged_evict(ctypes.byref(c or cache()), ctypes.byref(b or batch()), budget, first, recent, space,
                                        size, None)


@pytest.mark.parametrize("change,match", BAD_CACHES)
def test_weighed_and_cut_caches_are_checked(change, match):
    refused(lambda: _weigh(c=cache(**change)), match)
    refused(lambda: _evict(c=cache(**change)), match)


@pytest.mark.parametrize("change,match", BAD_BATCHES)
def test_weighed_and_cut_batches_are_checked(change, match):
    refused(lambda: _weigh(b=batch(**change)), match)
    if "row_starts" not in change and "max_rows" not in change:
        refused(lambda: _evict(b=batch(**change)), match)


def test_weigh_arguments_are_checked():
    refused(lambda: _weigh(c=cache(weights=None)), "needs weights")
    refused(lambda: _weigh(lse=None), "lse")
    refused(lambda: _weigh(scale=0.0), "score scale")
    refused(lambda: _weigh(q=rows(type=3)), "cache's type")
    many = {"q": rows(n_rows=4000, n_head=28), "b": batch(n_seq=1, max_rows=4000)}
    need = ctypes.c_size_t()
    check(jf.library().jfh_paged_weigh_workspace(ctypes.byref(cache()), ctypes.byref(many["b"]), ctypes.byref(many["q"]),
                                                 ctypes.byref(need)))
    assert need.value > 0
    refused(lambda: _weigh(**many, size=need.value - 1), f"needs {need.value} bytes")
    refused(lambda: _weigh(**many, space=None), "workspace")
    refused(lambda: _weigh(**many, space=AT + 8), "16-byte")
    check(_weigh(q=rows(n_rows=0)))
    check(_weigh(b=batch(max_length=0)))


def test_evict_arguments_are_checked():
    refused(lambda: _evict(c=cache(weights=None)), "weights and positions")
    refused(lambda: _evict(c=cache(positions=None)), "weights and positions")
    refused(lambda: _evict(budget=0), "budget")
    refused(lambda: _evict(budget=1 << 31), "budget")
    refused(lambda: _evict(first=1 << 31), "protected")
    refused(lambda: _evict(recent=(1 << 32) - 1), "protected")
    need = ctypes.c_size_t()
    check(jf.library().jfh_paged_evict_workspace(ctypes.byref(cache()), ctypes.byref(batch(row_starts=None)), 8,
                                                 ctypes.byref(need)))
    assert need.value == 2 * 4 * (1 + 2 * 8) * 4  # lists of 8 moves for 2 sequences of 4 heads
    refused(lambda: _evict(size=need.value - 1), f"needs {need.value} bytes")
    refused(lambda: _evict(space=None), "workspace")
    refused(lambda: _evict(space=AT + 8), "16-byte")
    check(_evict(budget=64, space=None, size=0))  # no sequence is longer
    check(_evict(b=batch(n_seq=0)))


def test_missing_arguments_are_refused():
    lib = jf.library()
    assert lib.jfh_paged_append(None, ctypes.byref(batch()), ctypes.byref(rows()), ctypes.byref(rows()), None, AT, None).code == 1
    assert lib.jfh_paged_append(ctypes.byref(cache()), None, ctypes.byref(rows()), ctypes.byref(rows()), None, AT, None).code == 1
    assert lib.jfh_paged_append(ctypes.byref(cache()), ctypes.byref(batch()), None, ctypes.byref(rows()), None, AT, None).code == 1
    assert lib.jfh_rope_rotate(None, ctypes.byref(rows()), AT, ctypes.byref(rows()), 0, None).code == 1
    assert lib.jfh_rope_create(None, ctypes.byref(ctypes.c_void_p())).code == 1
    lib.jfh_rope_destroy(None)


def test_steps_without_rows_or_sequences_do_nothing():
    check(_append(k=rows(n_rows=0, data=None), v=rows(n_rows=0, data=None)))
    check(_append(b=batch(n_seq=0, table=None, lengths=None, row_starts=None)))
    none = rows(n_rows=0, data=None)
    check(jf.library().jfh_rope_rotate(jf.Rope(64).handle, ctypes.byref(none), None, ctypes.byref(none), 0, None))


@pytest.mark.parametrize("kw,match", [
    ({"n_rot": 0}, "even number"), ({"n_rot": 7}, "even number"), ({"n_rot": 258}, "even number"),
    ({"base": 1.0}, "base"), ({"base": float("nan")}, "base"), ({"scaling": "linear", "factor": 0.5}, "factor"),
    ({"scaling": "yarn", "factor": float("inf")}, "factor"), ({"scaling": "ntk", "n_rot": 2, "factor": 2.0}, "more than one pair"),
    ({"scaling": "yarn", "factor": 2.0, "original_context": 0}, "original context"),
    ({"scaling": "yarn", "factor": 2.0, "beta_fast": 0.5}, "beta_fast"),
    ({"scaling": "yarn", "factor": 2.0, "beta_slow": 0.0}, "beta_fast"),
    ({"scaling": "yarn", "factor": 2.0, "attention_factor": -1.0}, "attention factor")])
def test_rotations_are_checked(kw, match):
    with pytest.raises(jf.InvalidArgument, match=match):
        jf.Rope(**{"n_rot": 64, **kw})


def test_rotation_names_are_checked():
    with pytest.raises(ValueError, match="layout"):
        jf.Rope(64, layout="pairs")
    with pytest.raises(ValueError, match="scaling"):
        jf.Rope(64, scaling="dynamic")


def _rotate(x, y, rope=None, positions=AT):
    rope = rope or jf.Rope(64)
    return jf.library().jfh_rope_rotate(rope.handle, ctypes.byref(x), positions, ctypes.byref(y), 0, None)


def test_rotated_rows_are_checked():
    refused(lambda: _rotate(rows(), rows(n_head=5)), "same rows, heads")
    refused(lambda: _rotate(rows(), rows(head_dim=128)), "same rows, heads")
    refused(lambda: _rotate(rows(head_dim=32), rows(head_dim=32)), "more values than a head")
    refused(lambda: _rotate(rows(), rows(row_stride=512)), "in place")
    refused(lambda: _rotate(rows(), rows(type=3)), "in place")
    refused(lambda: _rotate(rows(), rows(data=AT + 4096), positions=None), "positions")
    refused(lambda: _rotate(rows(), rows(data=AT + 4096, type=7)), "value type")


def test_index_arithmetic_cpp_tests():
    exe = os.path.join(ROOT, "tests", "cpp", "paged_test")
    subprocess.run(["make", "-C", os.path.join(ROOT, "tests", "cpp"), "paged_test"], check=True, capture_output=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "paged tests passed" in r.stdout


def test_tensors_are_checked():
    import torch

    with pytest.raises(ValueError, match="on GPU|on one GPU"):
        jf.Rope(64).rotate(torch.zeros(2, 1, 64), torch.zeros(2, dtype=torch.int32))
    pages = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        jf.PagedCache(pages, pages)
    with pytest.raises(ValueError, match="equal strides"):
        jf.PagedCache(pages, pages.float())
    with pytest.raises(ValueError, match="GPU"):
        jf.PagedBatch(torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                      torch.zeros(2, dtype=torch.int32), 1, 64)


def test_calls_without_a_gpu_are_device_errors():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    calls = [_append, _attend, _weigh, _evict, lambda: _rotate(rows(), rows(data=AT + 4096))]
    for call in calls:
        with pytest.raises(jf.JfhError) as e:
            check(call())
        assert e.value.code == 6
