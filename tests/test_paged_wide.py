"""The paged views refuse numbers that the C calls' 32-bit integers do not hold (ctypes would cut them off): strides and lengths of 2^31 and
more, counts and block sizes that would come out as other, valid ones. Arrays only look like device tensors; no GPU."""
import pytest

from goinfer_b200 import abi
from goinfer_b200.resident import ResidentError
from test_paged import Array, FakeOps, _packed, _view, f16, host, i32, lib  # noqa: F401

W = 1 << 32


def _refused(f, *a, **kw):
    with pytest.raises(ResidentError) as e:
        f(*a, **kw)
    assert e.value.status == abi.BAD_ARGUMENT, e.value


def test_row_strides(lib, host):  # noqa: F811
    c, r = _view(lib, host), _packed()
    kv, q, sel, out = Array((3, 128)), Array((3, 512)), i32(3, 2, 4), Array((3, 512))
    for wide in (W + 128, 1 << 31):
        far = Array((3, 128), stride=(wide, 1))
        _refused(c.append, r, far, kv)
        _refused(c.append, r, kv, far)
        _refused(c.append, r, Array((3, 2, 64), stride=(wide, 64, 1)), kv)
    for wide in (W + 512, 1 << 31):
        far = Array((3, 512), stride=(wide, 1))
        _refused(c.select, r, far, sel)
        _refused(c.attend, r, far, sel, out)
        _refused(c.attend, r, q, sel, far)
        _refused(c.attend, r, q, sel, Array((3, 8, 64), stride=(wide, 64, 1)))


def test_counts(lib, host):  # noqa: F811
    c, r = _view(lib, host), _packed()
    q, sel = Array((3, 512)), i32(3, 2, 4)
    _refused(c.select, r, q, sel, n_first=W + 1)
    _refused(c.select, r, q, sel, n_recent=W + 1)
    _refused(c.select, r, q, sel, n_first=1 - W)
    _refused(c.select, r, q, i32(3, 2, W + 4))
    _refused(c.attend, r, q, i32(3, 2, W + 4), Array((3, 512)))


def test_lengths(lib, host):  # noqa: F811
    n = W + 3
    _refused(_packed, row_slot=i32(n), row_pos=i32(n), slot_map=i32(n))
    _refused(_packed, seq_row0=i32(n))
    _refused(_view, lib, host, free_blocks=i32(W + 9), k_pool=f16(W + 9, 2, 16, 64), v_pool=f16(W + 9, 2, 16, 64), key_bounds=f16(W + 9, 2, 2, 64))
    _refused(_view, lib, host, block_table=i32(2, W + 4))
    _refused(_view, lib, host, block_table=i32(W + 2, 4), seq_blocks=i32(W + 2))
    _refused(_view, lib, host, block_rows=W + 16, k_pool=None, v_pool=None)
    _refused(_view, lib, host, k_pool=f16(9, W + 2, 16, 64), v_pool=f16(9, W + 2, 16, 64), key_bounds=None)


def test_arrays_without_extents(lib, host):  # noqa: F811
    c, r = _view(lib, host), _packed()
    q, sel, none = Array((3, 512)), i32(3, 2, 4), i32()
    for kw in (dict(row_slot=none), dict(row_pos=none), dict(slot_map=none), dict(seq_row0=none), dict(status=none)):
        _refused(_packed, **kw)
    for kw in (dict(block_table=none), dict(seq_blocks=none), dict(free_blocks=none), dict(free_count=none), dict(k_pool=f16()), dict(v_pool=f16()),
               dict(key_bounds=f16())):
        _refused(_view, lib, host, **kw)
    _refused(c.plan, none, i32(2), r)
    _refused(c.append, r, Array(()), Array((3, 128)))
    _refused(c.select, r, Array(()), sel)
    _refused(c.select, r, q, none)
    _refused(c.attend, r, q, none, Array((3, 512)))
    _refused(c.attend, r, q, sel, Array(()))


def test_the_stride_of_a_single_row_does_not_count(lib, host):  # noqa: F811
    c, r = _view(lib, host), _packed(row_slot=i32(1), row_pos=i32(1), slot_map=i32(1))
    far = Array((1, 128), stride=(W + 128, 1))
    for call in (lambda: c.append(r, far, far), lambda: c.select(r, Array((1, 8, 64), stride=(W, 64, 1)), i32(1, 2, 4)),
                 lambda: c.attend(r, Array((1, 512), stride=(W, 1)), i32(1, 2, 4), Array((1, 512)))):
        with pytest.raises(ResidentError) as e:
            call()
        assert e.value.status == abi.CUDA_ERROR, e.value  # accepted, and the context has no device
