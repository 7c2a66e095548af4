"""The paged views leave the library as other callers of it know it. Arrays only look like device tensors; no GPU."""
import ctypes as C

from goinfer_b200 import abi
from test_paged import _cache, _packed, _rows, _view, host, i32, lib  # noqa: F401


def test_a_view_changes_no_other_callers_functions(lib, host):  # noqa: F811
    before = {op: getattr(lib, "b200_paged_" + op).argtypes for op in ("plan", "append", "select", "attend")}
    view = _view(lib, host)
    assert {op: getattr(lib, "b200_paged_" + op).argtypes for op in before} == before
    # one that leaves the conversion to ctypes: a null pointer, given as such for every argument
    null = C.POINTER(abi.PagedCache)()
    for op in before:
        assert getattr(lib, "b200_paged_" + op)(host, null, null, None, None, 0, 0, 0, 0, None, 0, None) == abi.BAD_ARGUMENT
    try:
        view.plan(i32(2), i32(2), _packed())
    except Exception as e:
        assert e.status == abi.CUDA_ERROR
    assert lib.b200_paged_plan(host, C.byref(_cache()), C.byref(_rows()), C.c_void_p(1 << 20), C.c_void_p(1 << 20)) == abi.CUDA_ERROR
