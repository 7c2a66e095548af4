"""A paged KV cache in the caller's own device memory: the b200_paged_* entry points over device arrays.

`PagedCache` is one layer's pools with the block tables and the free stack that every layer shares; `PagedRows` the packed
rows of a step. Both are views: they check the arrays once and keep references to them, so a step costs one foreign call per
operator. Arrays are anything with torch's tensor attributes (data_ptr, shape, stride, dtype, get_device, is_contiguous); the
module itself imports no tensor library.

    ops = Ops(0, stream=torch.cuda.current_stream().cuda_stream or 1)      # 1: the legacy default stream
    cache = PagedCache(ops, table, seq_blocks, free_blocks, free_count, 16, k_pool, v_pool, key_bounds)
    rows = PagedRows(row_slot, row_pos, slot_map, seq_row0, status)
    cache.plan(kv_len, n_new, rows)
    cache.append(rows, k, v)
    cache.select(rows, q, sel)
    cache.attend(rows, q, sel, out)

Work is queued on the stream of `ops`, whatever the caller's current stream is; the two have to be ordered by the caller.
Wrong arguments raise ResidentError with B200_BAD_ARGUMENT before anything is queued. What the lengths ask of the pool is
known on the device only: `rows.status` says whether a plan went through (include/b200_resident.h).
"""
from __future__ import annotations

import ctypes as C

from . import abi
from .resident import ResidentError


def _refuse(text: str):
    raise ResidentError(abi.BAD_ARGUMENT, text)


_vp, _i, _f = C.c_void_p, C.c_int, C.c_float
# Foreign functions of this module's own: argument types set on the library's would hold for every other caller of it too.
_CALLS = (("b200_paged_plan", C.CFUNCTYPE(_i, _vp, _vp, _vp, _vp, _vp)), ("b200_paged_append", C.CFUNCTYPE(_i, _vp, _vp, _vp, _vp, _i, _vp, _i)),
          ("b200_paged_select", C.CFUNCTYPE(_i, _vp, _vp, _vp, _vp, _i, _i, _i, _i, _i, _vp)),
          ("b200_paged_attend", C.CFUNCTYPE(_i, _vp, _vp, _vp, _vp, _i, _i, _f, _f, _vp, _i, _vp, _i)))

_F32, _F16, _I32 = "torch.float32", "torch.float16", "torch.int32"
_I32_MAX = 2**31 - 1
_names: dict = {}  # dtype -> its text: formatting one costs more than a whole check


def _is(dtype, name: str) -> bool:
    text = _names.get(dtype)
    if text is None:
        text = _names[dtype] = str(dtype)
    return text == name


def _array(name: str, a, dtype: str, shape, device: int) -> int:
    """Address of a contiguous device array of this type and shape (None entries of shape: any extent)."""
    if a.shape == shape and _names.get(a.dtype) == dtype and a.get_device() == device and a.is_contiguous():
        return a.data_ptr()
    if not _is(a.dtype, dtype):
        _refuse(f"{name} has type {a.dtype}, not {dtype}")
    if len(a.shape) != len(shape) or any(w is not None and n != w for n, w in zip(a.shape, shape)):
        _refuse(f"{name} has shape {tuple(a.shape)}, not {tuple('any' if w is None else w for w in shape)}")
    if a.get_device() != device:
        _refuse(f"{name} is on {a.device}, the context on cuda:{device}")
    if not a.is_contiguous():
        _refuse(f"{name} is not contiguous")
    return a.data_ptr()


def _int(name: str, n: int) -> int:
    """n, for a 32-bit integer of the C call, which a foreign call would cut to its low bits."""
    if n > _I32_MAX or n < -_I32_MAX:
        _refuse(f"{name} is {n}, past 32 bits")
    return n


def _packed(name: str, a, n_rows: int, device: int):
    """Address, row stride and row width of a f32 [n_rows][...] device array whose rows are contiguous."""
    shape, stride = a.shape, a.stride()
    if n_rows > 1 and stride and stride[0] > _I32_MAX:
        _refuse(f"the rows of {name} lie {stride[0]} values apart, past 32 bits")
    if len(shape) == 2 and stride[1] == 1 and shape[0] == n_rows and _names.get(a.dtype) == _F32 and a.get_device() == device:
        return a.data_ptr(), stride[0] if n_rows > 1 else shape[1], shape[1]
    if len(shape) < 2 or shape[0] != n_rows or not _is(a.dtype, _F32) or a.get_device() != device:
        _refuse(f"{name} is {a.dtype} {tuple(shape)} on {a.device}, not f32 with {n_rows} rows on cuda:{device}")
    width = 1
    for n, st in zip(shape[:0:-1], stride[:0:-1]):
        if n != 1 and st != width:
            _refuse(f"the rows of {name} are not contiguous (shape {tuple(shape)}, strides {stride})")
        width *= n
    return a.data_ptr(), stride[0] if n_rows > 1 else width, width


class PagedRows:
    """The packed rows of a step: row_slot, row_pos [n_rows] int32, and what plan and append need besides."""

    def __init__(self, row_slot, row_pos, slot_map=None, seq_row0=None, status=None):
        device = row_slot.get_device()
        if device < 0:
            _refuse(f"row_slot is on {row_slot.device}")
        i32 = _I32
        slots = _array("row_slot", row_slot, i32, (None,), device)
        row0 = None if seq_row0 is None else _array("seq_row0", seq_row0, i32, (None,), device)
        n = _int("the number of rows", row_slot.shape[0])
        self.n_rows, self.device = n, device
        self.n_seqs = None if seq_row0 is None else _int("the number of sequences", seq_row0.shape[0] - 1)
        self._keep = (row_slot, row_pos, slot_map, seq_row0, status)
        self.row_slot, self.row_pos, self.slot_map, self.seq_row0, self.status = self._keep
        self.c = abi.PagedRows(row0, slots, _array("row_pos", row_pos, i32, (n,), device),
                               None if slot_map is None else _array("slot_map", slot_map, i32, (n,), device),
                               None if status is None else _array("status", status, i32, (4,), device), n, 0)
        self._c = C.addressof(self.c)


class PagedCache:
    """block_table [n_seqs][max_blocks], seq_blocks [n_seqs], free_blocks [n_blocks], free_count [1], all int32; k_pool, v_pool
    fp16 [n_blocks][n_kv_heads][block_rows][head_dim]; key_bounds fp16 [n_blocks][n_kv_heads][2][head_dim]. A cache without
    pools plans, one without key_bounds selects nothing and keeps no bounds as it appends."""

    def __init__(self, ops, block_table, seq_blocks, free_blocks, free_count, block_rows: int, k_pool=None, v_pool=None, key_bounds=None):
        self.ops, self.device = ops, ops.drv.device
        dev, i32, f16 = self.device, _I32, _F16
        self._keep = (block_table, seq_blocks, free_blocks, free_count, k_pool, v_pool, key_bounds)
        table = _array("block_table", block_table, i32, (None, None), dev)
        stack = _array("free_blocks", free_blocks, i32, (None,), dev)
        self.n_seqs, max_blocks = (_int("an extent of block_table", n) for n in block_table.shape)
        n_blocks = _int("the number of blocks", free_blocks.shape[0])
        _int("block_rows", block_rows)
        kv = hd = 0
        if k_pool is not None or v_pool is not None:
            if k_pool is None or v_pool is None:
                _refuse("k_pool and v_pool come together")
            if len(k_pool.shape) != 4:
                _refuse(f"k_pool has shape {tuple(k_pool.shape)}, not [n_blocks][n_kv_heads][block_rows][head_dim]")
            kv, hd = k_pool.shape[1], k_pool.shape[3]
        elif key_bounds is not None:
            if len(key_bounds.shape) != 4:
                _refuse(f"key_bounds has shape {tuple(key_bounds.shape)}, not [n_blocks][n_kv_heads][2][head_dim]")
            kv, hd = key_bounds.shape[1], key_bounds.shape[3]
        _int("the number of kv heads", kv), _int("head_dim", hd)
        pool = lambda name, a: None if a is None else _array(name, a, f16, (n_blocks, kv, block_rows, hd), dev)  # noqa: E731
        self.block_rows, self.n_kv_heads, self.head_dim = block_rows, kv, hd
        self.c = abi.PagedCache(pool("k_pool", k_pool), pool("v_pool", v_pool),
                                None if key_bounds is None else _array("key_bounds", key_bounds, f16, (n_blocks, kv, 2, hd), dev), table,
                                _array("seq_blocks", seq_blocks, i32, (self.n_seqs,), dev), stack,
                                _array("free_count", free_count, i32, (1,), dev), n_blocks, self.n_seqs, max_blocks, block_rows, kv, hd)
        self._c, self._drv = C.addressof(self.c), ops.drv
        self._plan, self._append, self._select, self._attend = (proto((name, ops.lib)) for name, proto in _CALLS)

    def _raise(self, st: int):
        raise ResidentError(st, self.ops.drv.last_error())

    def _here(self, rows: PagedRows) -> int:
        if rows.device != self.device:
            _refuse(f"the rows are on cuda:{rows.device}, the cache is on cuda:{self.device}")
        return rows.n_rows

    def _heads(self, name: str, width: int) -> int:
        if self.head_dim == 0 or width % self.head_dim:
            _refuse(f"{name} has {width} values a row, not whole heads of {self.head_dim}")
        return width // self.head_dim

    def plan(self, kv_len, n_new, rows: PagedRows):
        self._here(rows)
        if rows.n_seqs != self.n_seqs:
            _refuse(f"rows are for {rows.n_seqs} sequences, the cache has {self.n_seqs}")
        shape, device = (self.n_seqs,), self.device
        st = self._plan(self._drv.ctx.value, self._c, rows._c, _array("kv_len", kv_len, _I32, shape, device), _array("n_new", n_new, _I32, shape, device))
        if st:
            self._raise(st)

    def append(self, rows: PagedRows, k, v):
        n, device = self._here(rows), self.device
        pk, ldk, wk = _packed("k", k, n, device)
        pv, ldv, wv = _packed("v", v, n, device)
        if wk != self.n_kv_heads * self.head_dim or wv != wk:
            _refuse(f"k {tuple(k.shape)} and v {tuple(v.shape)} must have {self.n_kv_heads} heads of {self.head_dim} a row")
        st = self._append(self._drv.ctx.value, self._c, rows._c, pk, ldk, pv, ldv)
        if st:
            self._raise(st)

    def select(self, rows: PagedRows, q, sel, n_first: int = 1, n_recent: int = 1):
        n, device = self._here(rows), self.device
        pq, ldq, width = _packed("q", q, n, device)
        n_select = sel.shape[-1] if sel.shape else 0
        ps = _array("sel", sel, _I32, (n, self.n_kv_heads, n_select), device)
        if n_select > _I32_MAX or not -_I32_MAX <= n_first <= _I32_MAX or not -_I32_MAX <= n_recent <= _I32_MAX:
            _refuse(f"lists of {n_select} blocks with the first {n_first} and the last {n_recent}")
        st = self._select(self._drv.ctx.value, self._c, rows._c, pq, ldq, self._heads("q", width), n_first, n_recent, n_select, ps)
        if st:
            self._raise(st)

    def attend(self, rows: PagedRows, q, sel, out, scale: float = 0.0, softcap: float = 0.0):
        n, device = self._here(rows), self.device
        pq, ldq, width = _packed("q", q, n, device)
        po, ldo, wide = _packed("out", out, n, device)
        if wide != width:
            _refuse(f"out has shape {tuple(out.shape)}, q {tuple(q.shape)}")
        n_select = sel.shape[-1] if sel.shape else 0
        ps = _array("sel", sel, _I32, (n, self.n_kv_heads, n_select), device)
        if n_select > _I32_MAX:
            _refuse(f"lists of {n_select} blocks")
        st = self._attend(self._drv.ctx.value, self._c, rows._c, pq, ldq, self._heads("q", width), scale, softcap, ps, n_select, po, ldo)
        if st:
            self._raise(st)
