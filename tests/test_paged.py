"""The paged-cache calls without a GPU: address rules, struct layouts, and every refusal of the C entry points and of the
Python views (nothing is queued by a refused call)."""
import ctypes as C
import os
import re
import subprocess

import pytest

from goinfer_b200 import abi
from goinfer_b200.paged import PagedCache, PagedRows
from goinfer_b200.resident import ResidentError

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from goinfer_b200 import build, resident
    build.build()
    return resident.load_library()


@pytest.fixture(scope="module")
def host(lib):
    """A context without a device: calls that pass their checks end with CUDA_ERROR."""
    ctx = C.c_void_p()
    assert lib.b200_debug_open_host(C.byref(ctx)) == abi.OK
    yield ctx
    lib.b200_close(ctx)


def test_struct_layouts():
    assert C.sizeof(abi.PagedCache) == 7 * 8 + 6 * 4 and abi.PagedCache.n_blocks.offset == 56
    assert C.sizeof(abi.PagedRows) == 5 * 8 + 2 * 4 and abi.PagedRows.n_rows.offset == 40
    text = open(os.path.join(ROOT, "integration", "b200", "lib.go")).read()
    assert "unsafe.Sizeof(pagedCacheC{}) != 80" in text and "unsafe.Sizeof(pagedRowsC{}) != 48" in text


def test_address_rules_of_bad_pages_and_rows(tmp_path):
    """The rules every kernel asks before it forms an address, compiled for the host."""
    src = tmp_path / "rules.cpp"
    src.write_text(r"""
#include <assert.h>
#include <limits.h>
#include "paged.cuh"
int main() {
    const int n = 100;
    const int bad[] = {INT_MIN, -2, -1, 0, n, n + 1, INT_MAX};
    for (int b : bad) assert(!paged_block_ok(b, n));
    assert(paged_block_ok(1, n) && paged_block_ok(n - 1, n) && !paged_block_ok(1, 1));
    assert(paged_row_ok(0, 0, 1) && paged_row_ok(6, INT_MAX, 7));
    assert(!paged_row_ok(-1, 0, 7) && !paged_row_ok(7, 0, 7) && !paged_row_ok(INT_MIN, 0, 7) && !paged_row_ok(INT_MAX, 0, 7) && !paged_row_ok(0, -1, 7));
    assert(paged_visible(0, 16, 8) == 1 && paged_visible(15, 16, 8) == 1 && paged_visible(16, 16, 8) == 2);
    assert(paged_visible(127, 16, 8) == 8 && paged_visible(128, 16, 8) == 8 && paged_visible(INT_MAX, 16, 8) == 8 && paged_visible(5, 256, 1) == 1);
    assert(paged_tile(1 << 20, 7, 8, 64, 128) == (((size_t)1 << 23) + 7) * 64 * 128);
    for (int br = 16; br <= 256; br += 16) {
        const unsigned d = paged_divisor(br);
        for (unsigned k = 0; k < 5000000; k++) {
            const unsigned x = k < 100000 ? k : k % 3 == 0 ? (k * 2654435761u) >> 1 : k % 3 == 1 ? (k * 429u) / br * br : (k * 429u) / br * br + br - 1;
            if (x >= 0x80000000u) continue;
            assert(paged_div(x, d) == x / br && paged_div_up(x, d) == (x + (unsigned)br - 1) / br);
        }
        for (unsigned x = 0x7fffffffu; x > 0x7fffffffu - 100000; x--) assert(paged_div(x, d) == x / br && paged_div_up(x, d) == (x + (unsigned)br - 1) / br);
    }
    return 0;
}
""")
    exe = tmp_path / "rules"
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "goinfer_b200", "csrc"), "-I", "/usr/local/cuda/include", str(src), "-o", str(exe)], check=True)
    subprocess.run([str(exe)], check=True)


def test_every_kernel_waits_for_the_one_before_it():
    """The paged kernels start while the kernel ahead of them still runs: each must wait before its first statement that reads."""
    n = 0
    for name in ("paged.cu", "paged_select.cu", "paged_attend.cu"):
        text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "goinfer_b200", "csrc", name)).read())
        assert "<<<" not in text and "__restrict__" not in text and "__ldg" not in text and ".nc." not in text
        for m in re.finditer(r"__global__[^{]*\{", text):
            n += 1
            body = text[m.end():].lstrip()
            body = re.sub(r"^extern __shared__[^;]*;\s*", "", body)
            assert re.match(r"(pdl_trigger\(\);\s*)?pdl_wait\(\);", body), m.group(0)
    assert n == 5


A = 1 << 20  # an aligned address that no call reads


def _cache(**kw):
    d = dict(k_pool=A, v_pool=A, key_bounds=A, block_table=A, seq_blocks=A, free_blocks=A, free_count=A, n_blocks=9, n_seqs=2, max_blocks=4, block_rows=16,
             n_kv_heads=2, head_dim=64)
    d.update(kw)
    return abi.PagedCache(*[d[f[0]] for f in abi.PagedCache._fields_])


def _rows(**kw):
    d = dict(seq_row0=A, row_slot=A, row_pos=A, slot_map=A, status=A, n_rows=3, _pad=0)
    d.update(kw)
    return abi.PagedRows(*[d[f[0]] for f in abi.PagedRows._fields_])


def _plan(lib, ctx, c, r, kv_len=A, n_new=A):
    return lib.b200_paged_plan(ctx, C.byref(c), C.byref(r), C.c_void_p(kv_len), C.c_void_p(n_new))


def _append(lib, ctx, c, r, k=A, ldk=128, v=A, ldv=128):
    return lib.b200_paged_append(ctx, C.byref(c), C.byref(r), C.c_void_p(k), ldk, C.c_void_p(v), ldv)


def _select(lib, ctx, c, r, q=A, ldq=512, heads=8, first=1, recent=1, n=4, sel=A):
    return lib.b200_paged_select(ctx, C.byref(c), C.byref(r), C.c_void_p(q), ldq, heads, first, recent, n, C.c_void_p(sel))


def _attend(lib, ctx, c, r, q=A, ldq=512, heads=8, scale=0.0, cap=0.0, sel=A, n=4, out=A, ldo=512):
    return lib.b200_paged_attend(ctx, C.byref(c), C.byref(r), C.c_void_p(q), ldq, heads, C.c_float(scale), C.c_float(cap), C.c_void_p(sel), n,
                                 C.c_void_p(out), ldo)


CALLS = {"plan": _plan, "append": _append, "select": _select, "attend": _attend}
ANY_CACHE = [dict(block_table=None), dict(block_table=A + 2), dict(n_seqs=0), dict(max_blocks=0), dict(n_blocks=1), dict(block_rows=0), dict(block_rows=8),
             dict(block_rows=24), dict(block_rows=272), dict(n_blocks=1 << 27), dict(max_blocks=1 << 28)]
POOLS = [dict(k_pool=None), dict(v_pool=None), dict(k_pool=A + 8), dict(v_pool=A + 8), dict(head_dim=96), dict(head_dim=256), dict(n_kv_heads=0), dict(key_bounds=A + 8)]
NAN, INF = float("nan"), float("inf")
REFUSED = (
    [(op, dict(c), {}, {}) for op in CALLS for c in ANY_CACHE] +
    [(op, {}, dict(n_rows=n), {}) for op in CALLS for n in (-1, (1 << 27) + 1)] +
    [(op, {}, r, {}) for op in ("plan", "select", "attend") for r in (dict(row_slot=None), dict(row_pos=None), dict(row_slot=A + 1), dict(row_pos=A + 1))] +
    [(op, {}, r, {}) for op in ("plan", "append") for r in (dict(slot_map=None), dict(slot_map=A + 2))] +
    [("plan", c, {}, {}) for c in (dict(seq_blocks=None), dict(free_blocks=None), dict(free_count=None), dict(seq_blocks=A + 1), dict(free_blocks=A + 1),
                                   dict(free_count=A + 1), dict(n_seqs=16385), dict(n_seqs=16384, max_blocks=1 << 17))] +
    [("plan", {}, r, {}) for r in (dict(seq_row0=None), dict(status=None), dict(seq_row0=A + 1), dict(status=A + 1))] +
    [("plan", {}, {}, a) for a in (dict(kv_len=None), dict(n_new=None), dict(kv_len=A + 2), dict(n_new=A + 2))] +
    [(op, c, {}, {}) for op in ("append", "attend") for c in POOLS] +
    [("append", {}, {}, a) for a in (dict(k=None), dict(v=None), dict(k=A + 4), dict(v=A + 4), dict(ldk=124), dict(ldv=124), dict(ldk=130), dict(ldv=130))] +
    [("select", c, {}, {}) for c in (dict(key_bounds=None), dict(key_bounds=A + 8), dict(head_dim=32), dict(n_kv_heads=-1), dict(max_blocks=24577))] +
    [("select", {}, {}, a) for a in (dict(q=None), dict(q=A + 4), dict(ldq=508), dict(ldq=514), dict(heads=0), dict(heads=7), dict(heads=18, ldq=2048), dict(first=-1), dict(recent=0),
                                     dict(first=4), dict(n=0), dict(n=2049), dict(sel=None), dict(sel=A + 2), dict(first=0x7fffffff, recent=0x7fffffff))] +
    [("attend", {}, {}, a) for a in (dict(q=None), dict(q=A + 4), dict(ldq=508), dict(ldq=514), dict(heads=0), dict(heads=7), dict(heads=18, ldq=2048, ldo=2048), dict(n=0), dict(n=2049),
                                     dict(sel=None), dict(sel=A + 2), dict(out=None), dict(out=A + 8), dict(ldo=508), dict(ldo=514), dict(scale=-1.0), dict(scale=NAN),
                                     dict(scale=INF), dict(cap=-1.0), dict(cap=1e-38), dict(cap=NAN), dict(cap=INF))])


@pytest.mark.parametrize("op,cache,rows,args", REFUSED, ids=lambda x: x if isinstance(x, str) else ",".join(f"{k}={v}" for k, v in x.items()) or "-")
def test_refused_calls(lib, host, op, cache, rows, args):
    assert CALLS[op](lib, host, _cache(**cache), _rows(**rows), **args) == abi.BAD_ARGUMENT
    text = lib.b200_last_error(host).decode()
    assert text.startswith("b200_paged_" + op), text
    assert CALLS[op](lib, None, _cache(), _rows()) == abi.BAD_ARGUMENT


@pytest.mark.parametrize("op", CALLS)
def test_accepted_calls_reach_the_device(lib, host, op):
    assert CALLS[op](lib, host, _cache(), _rows()) == abi.CUDA_ERROR
    assert "no device" in lib.b200_last_error(host).decode()
    null = C.POINTER(abi.PagedCache)()
    assert getattr(lib, "b200_paged_" + op)(host, null, null, None, None, 0, 0, 0, 0, None, 0, None) == abi.BAD_ARGUMENT


def test_a_step_without_rows_is_no_work(lib, host):
    empty = dict(n_rows=0, row_slot=None, row_pos=None, slot_map=None)
    assert _append(lib, host, _cache(), _rows(**empty), k=None, v=None) == abi.OK
    assert _select(lib, host, _cache(), _rows(**empty), q=None, sel=None) == abi.OK
    assert _attend(lib, host, _cache(), _rows(**empty), q=None, sel=None, out=None) == abi.OK
    assert _plan(lib, host, _cache(), _rows(**empty)) == abi.CUDA_ERROR  # sequences may still be retired


# ---- the Python views, over arrays that only look like device tensors -------------------------------------------------


class Array:
    class device:
        def __init__(self, index):
            self.type, self.index = "cuda", index

        def __str__(self):
            return f"cuda:{self.index}"

    def __init__(self, shape, dtype="torch.float32", device=0, stride=None):
        self.shape, self.dtype, self.device = tuple(shape), dtype, Array.device(device)
        dense, n = [], 1
        for s in reversed(self.shape):
            dense.insert(0, n)
            n *= s
        self._dense, self._stride, self._n = tuple(dense), tuple(stride or dense), n

    def get_device(self):
        return self.device.index

    def stride(self):
        return self._stride

    def is_contiguous(self):
        return self._stride == self._dense

    def data_ptr(self):
        return A



class FakeOps:
    def __init__(self, lib, ctx):
        self.lib, self.ctx, self.drv = lib, ctx, self
        self.device = 0

    def last_error(self):
        return self.lib.b200_last_error(self.ctx).decode()


def i32(*shape, **kw):
    return Array(shape, "torch.int32", **kw)


def f16(*shape, **kw):
    return Array(shape, "torch.float16", **kw)


def _view(lib, host, **kw):
    d = dict(block_table=i32(2, 4), seq_blocks=i32(2), free_blocks=i32(9), free_count=i32(1), block_rows=16, k_pool=f16(9, 2, 16, 64), v_pool=f16(9, 2, 16, 64),
             key_bounds=f16(9, 2, 2, 64))
    d.update(kw)
    return PagedCache(FakeOps(lib, host), **d)


def _packed(**kw):
    d = dict(row_slot=i32(3), row_pos=i32(3), slot_map=i32(3), seq_row0=i32(3), status=i32(4))
    d.update(kw)
    return PagedRows(**d)


@pytest.mark.parametrize("kw", [dict(block_table=i32(2, 4, 1)), dict(block_table=Array((2, 4), "torch.int64")), dict(block_table=i32(2, 4, device=1)),
                                dict(block_table=i32(2, 4, stride=(8, 1))), dict(seq_blocks=i32(3)), dict(free_count=i32(2)), dict(k_pool=f16(9, 2, 32, 64)),
                                dict(k_pool=f16(8, 2, 16, 64)), dict(v_pool=f16(9, 1, 16, 64)), dict(v_pool=None), dict(k_pool=None),
                                dict(k_pool=Array((9, 2, 16, 64), "torch.bfloat16")), dict(key_bounds=f16(9, 2, 1, 64)), dict(k_pool=f16(9, 2, 64)),
                                dict(k_pool=None, v_pool=None, key_bounds=f16(9, 64))])
def test_views_refuse_arrays_that_do_not_fit(lib, host, kw):
    with pytest.raises(ResidentError) as e:
        _view(lib, host, **kw)
    assert e.value.status == abi.BAD_ARGUMENT


def _raises(want, f, *a, **kw):
    with pytest.raises(ResidentError) as e:
        f(*a, **kw)
    assert e.value.status == want, e.value


def test_views_refuse_calls_that_do_not_fit(lib, host):
    c, r = _view(lib, host), _packed()
    bad = abi.BAD_ARGUMENT
    for kw in (dict(row_pos=i32(4)), dict(slot_map=i32(2)), dict(status=i32(3)), dict(row_slot=Array((3,), "torch.int64"), row_pos=i32(3)), dict(row_pos=i32(3, device=1))):
        _raises(bad, _packed, **kw)
    _raises(bad, c.plan, i32(2), i32(2), _packed(seq_row0=i32(4)))
    _raises(bad, c.plan, i32(3), i32(2), r)
    _raises(bad, c.plan, i32(2), Array((2,), "torch.int64"), r)
    _raises(bad, c.plan, i32(2), i32(2), PagedRows(i32(3), i32(3)))
    kv, q, sel, out = Array((3, 2, 64)), Array((3, 8, 64)), i32(3, 2, 4), Array((3, 512))
    for k, v in ((Array((4, 2, 64)), kv), (Array((3, 128), "torch.float16"), kv), (Array((3, 1, 64)), Array((3, 1, 64))), (kv, Array((3, 64))), (kv, Array((3,))),
                 (Array((3, 2, 64), stride=(256, 128, 1)), kv), (Array((3, 2, 64), stride=(128, 64, 2)), kv), (Array((3, 2, 64), device=1), kv)):
        _raises(bad, c.append, r, k, v)
    _raises(bad, c.append, PagedRows(i32(3), i32(3)), kv, kv)
    away = PagedRows(*(i32(3, device=1) for _ in range(3)))
    _raises(bad, c.append, away, kv, kv)
    _raises(bad, c.select, away, q, sel)
    _raises(bad, c.attend, away, q, sel, out)
    _raises(bad, PagedRows, i32(3, device=-1), i32(3, device=-1))
    for f in (lambda q, s, o=out: c.select(r, q, s), lambda q, s, o=out: c.attend(r, q, s, o)):
        _raises(bad, f, Array((3, 8, 60)), sel)
        _raises(bad, f, Array((2, 8, 64)), sel)
        _raises(bad, f, Array((3, 8, 64), "torch.float64"), sel)
        _raises(bad, f, q, i32(3, 1, 4))
        _raises(bad, f, q, Array((3, 2, 4), "torch.int64"))
        _raises(bad, f, q, i32(3, 2, 4, device=1))
        _raises(abi.CUDA_ERROR, f, q, sel)  # accepted, and the context has no device
    _raises(bad, c.attend, r, q, sel, Array((3, 256)))
    _raises(bad, c.attend, r, q, sel, Array((3, 512), stride=(512, 2)))
    _raises(bad, c.attend, r, q, sel, out, scale=-1.0)
    _raises(bad, c.select, r, q, sel, n_first=4, n_recent=1)
    _raises(bad, c.select, r, q, sel, n_first=0, n_recent=0)
    plan_only = _view(lib, host, k_pool=None, v_pool=None, key_bounds=None)
    _raises(abi.CUDA_ERROR, plan_only.plan, i32(2), i32(2), r)
    _raises(bad, plan_only.append, r, kv, kv)
    _raises(bad, plan_only.select, r, q, i32(3, 0, 4))
    _raises(bad, _view(lib, host, key_bounds=None).select, r, q, sel)
    _raises(bad, _view(lib, host, k_pool=None, v_pool=None).attend, r, q, sel, out)
    _raises(abi.CUDA_ERROR, c.append, r, kv, Array((3, 128)))
    _raises(abi.CUDA_ERROR, c.append, r, Array((3, 128), stride=(640, 1)), Array((3, 128), stride=(640, 1)))
    _raises(bad, c.append, r, Array((3, 128), stride=(642, 1)), Array((3, 128), stride=(640, 1)))
    _raises(bad, c.append, r, kv, Array((3, 2, 64), stride=(64, 64, 1)))
    _raises(bad, c.select, r, q, Array((3,), "torch.int32"))
    _raises(bad, c.attend, PagedRows(i32(2), i32(2)), q, i32(2, 2, 4), out)
