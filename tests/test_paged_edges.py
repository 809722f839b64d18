"""The paged-cache operators without a GPU, where bounds and handles decide."""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest

import jetsonfabric_amd as jf
from jetsonfabric_amd import _capi
from jetsonfabric_amd._capi import check
from tests.test_paged import AT, _append, _attend, _evict, _weigh, batch, cache, refused, rows

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_bounds_cpp_tests():
    exe = os.path.join(ROOT, "tests", "cpp", "paged_bounds_test")
    subprocess.run(["make", "-C", os.path.join(ROOT, "tests", "cpp"), "paged_bounds_test"], check=True, capture_output=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "paged bounds tests passed" in r.stdout


LONGEST = (1 << 31) - 65537  # kernels' loops step by up to 65536 slots in 32 bits


@pytest.mark.parametrize("length", [LONGEST + 1, (1 << 31) - 1025, (1 << 31) - 1])
@pytest.mark.parametrize("call", [_append, _attend, _weigh, _evict])
def test_lengths_that_a_loop_could_step_out_of_are_refused(call, length):
    refused(lambda: call(b=batch(table_stride=1 << 28, max_length=length)), "max_length exceeds 2\\^31 - 65537")


def test_the_longest_sequences_have_workspaces():
    lib, need = jf.library(), ctypes.c_size_t()
    long = batch(n_seq=1, table_stride=1 << 28, max_length=LONGEST)
    check(lib.jfh_paged_attention_workspace(ctypes.byref(cache()), ctypes.byref(long), ctypes.byref(rows()), ctypes.byref(need)))
    check(lib.jfh_paged_weigh_workspace(ctypes.byref(cache()), ctypes.byref(long), ctypes.byref(rows()), ctypes.byref(need)))
    check(lib.jfh_paged_evict_workspace(ctypes.byref(cache()), ctypes.byref(long), 8, ctypes.byref(need)))
    assert need.value == 4 * (1 + 2 * 8) * 4


def test_a_closed_rotation_has_no_handle():
    rope = jf.Rope(64)
    assert rope.handle
    rope.close()
    rope.close()
    with pytest.raises(jf.InvalidArgument, match="closed"):
        rope.handle
    x = rows()
    with pytest.raises(jf.InvalidArgument, match="a rotation is required"):
        check(jf.library().jfh_rope_rotate(rope._h, ctypes.byref(x), AT, ctypes.byref(x), 0, None))


@pytest.mark.parametrize("handle,names", [(jf.PagedCache, ("k", "v", "weights", "positions", "device")),
                                          (jf.PagedBatch, ("table", "lengths", "row_starts", "device"))])
def test_tensors_of_a_handle_cannot_be_exchanged(handle, names):
    """A handle has passed their addresses on: another tensor in their place would free them under the kernels."""
    for name in names:
        with pytest.raises(AttributeError):
            setattr(object.__new__(handle), name, None)


def test_tensors_that_require_gradients_are_refused():
    """No operator has a backward pass: a gradient would be lost without a word."""
    import torch

    x, positions = torch.zeros(2, 1, 64, requires_grad=True), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="x requires a gradient"):
        jf.Rope(64).rotate(x, positions)
    with torch.no_grad(), pytest.raises(ValueError, match="on GPU"):  # as any tensor
        jf.Rope(64).rotate(x, positions)
    with pytest.raises(ValueError, match="out requires a gradient|on GPU"):
        jf.Rope(64).rotate(x.detach(), positions, out=x)


@pytest.mark.parametrize("kw", [{"n_rot": (1 << 32) + 64}, {"n_rot": -64}, {"original_context": (1 << 32) + 4096}, {"n_rot": 64 - (1 << 32)}])
def test_numbers_beyond_32_bits_are_refused_not_cut(kw):
    with pytest.raises(jf.InvalidArgument, match="must be 0 to 2\\^32 - 1"):
        jf.Rope(**{"n_rot": 64, "scaling": "yarn", "factor": 2.0, **kw})


@pytest.mark.parametrize("change", [{"row_stride": 0}, {"head_stride": 0}, {"row_stride": 0, "head_stride": 0}, {"head_stride": 56},
                                    {"row_stride": 64}, {"row_stride": 248}, {"row_stride": 64, "head_stride": 128}])
def test_rows_that_overlap_are_not_written(change):
    """Three rows of four heads of 64 values; an expanded tensor has stride 0."""
    out = rows(data=AT + (1 << 16), **change)
    refused(lambda: _attend(out=out), "out's strides let its rows overlap")
    x = rows()
    call = lambda: jf.library().jfh_rope_rotate(jf.Rope(64).handle, ctypes.byref(x), AT, ctypes.byref(out), 0, None)  # noqa: E731
    refused(call, "y's strides let its rows overlap")


@pytest.mark.parametrize("change", [{"row_stride": 512}, {"row_stride": 64, "head_stride": 192}])
def test_attention_in_place_keeps_its_strides(change):
    refused(lambda: _attend(out=rows(**change)), "in place must keep")


@pytest.mark.parametrize("change", [{}, {"row_stride": 64, "head_stride": 192}, {"row_stride": 64, "head_stride": 256},
                                    {"row_stride": 1 << 40}, {"head_stride": 64, "row_stride": 264},
                                    {"n_rows": 1, "row_stride": 0}, {"n_head": 4, "n_rows": 1, "row_stride": 8}])
def test_other_layouts_of_rows_are_written(change):
    """Not refused for their layout: the next check, of the workspace's size, is."""
    long = {"b": batch(n_seq=1, table_stride=4096, max_length=65536), "space": None}
    refused(lambda: _attend(q=rows(n_rows=change.get("n_rows", 3)), out=rows(data=AT + (1 << 16), **change), **long), "bytes of workspace")
