"""The paged attention over keys whose weights lie far apart, against the same sums in 64 bits.

Values are positive here, so that nothing cancels and every weight's relative error reaches the result unhidden. With
u = 2^-22 (what two fp16 parts leave of a value) and X the largest scale * sum |q k| of the case, to first order:
  a score, and with it the maximum it is held against, is off by 2 u X (the split of the query, the fp32 sum): a weight by 4 u X;
  a factor exp(-a) is off by (2 + 1.2 a) units of 2^-23: a weight's own, a few rescales' (at most four that are not 1), two joins',
  whose arguments add up to at most 2 X: 1.2 u X + 7 u; its own split u; the sums 2 u;
numerator and denominator both: 2 u (5.2 X + 10) <= u (11 X + 20)."""
import numpy as np
import pytest

from test_gpu_paged import _views, dev, ops  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -22


def _exact(q, k, v, scale):
    """f64: q [rows][kv][G][hd], k and v [rows][kv][keys][hd] -> result, largest scale * sum |q k|."""
    q, k, v = q.double(), k.double(), v.double()
    x = torch.matmul(q, k.transpose(-1, -2)) * scale
    return torch.matmul(torch.softmax(x, -1), v), (torch.matmul(q.abs(), k.abs().transpose(-1, -2)) * scale).max().item()


# one row (clusters of CTAs), rows enough that a CTA has the whole list, lists of one tile, of a tile a warp and of many; sizes between
SINK_SHAPES = [(1, 1, 1, 64, 16, 1), (1, 2, 4, 128, 16, 3), (2, 1, 8, 64, 32, 5), (1, 8, 4, 128, 16, 64), (70, 8, 4, 128, 16, 33), (180, 4, 2, 64, 48, 11), (90, 4, 5, 64, 16, 70)]


@pytest.mark.parametrize("rows,kv,G,hd,br,n", SINK_SHAPES)
@pytest.mark.parametrize("gap", [6.0, 12.0, 17.0, 18.5, 30.0])
@pytest.mark.parametrize("value", [0.0, 0.02, 1.0])
def test_attend_one_key_above_all_others(ops, rows, kv, G, hd, br, n, gap, value):  # noqa: F811
    """One key of the first block scores `gap` above the middle of all others, whose weights together stay in the result."""
    torch.manual_seed(rows + n)
    keys = n * br
    k = torch.randn(rows * n + 1, kv, br, hd, device="cuda").half()
    v = (1 + torch.rand(rows * n + 1, kv, br, hd, device="cuda")).half()
    table = np.arange(1, rows * n + 1, dtype=np.int32).reshape(rows, n)
    q = torch.randn(rows, kv, G, hd, device="cuda")
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    first = torch.from_numpy(table[:, 0]).cuda().long()
    k[first, :, 5] = 0.0
    k[first, :, 5, 0] = gap * hd ** 0.5 / 4.0
    v[first, :, 5] = value
    cache, packed = _views(ops, table, np.arange(rows), np.full(rows, keys - 1), br, rows * n + 1, k, v)
    out = torch.empty(rows, kv, G, hd, device="cuda")
    cache.attend(packed, q, dev(np.tile(np.arange(n, dtype=np.int32), (rows, kv, 1))), out)
    torch.cuda.synchronize()
    flat = lambda a: a[dev(table).long()].transpose(1, 2).reshape(rows, kv, keys, hd)  # noqa: E731
    want, X = _exact(q, flat(k), flat(v), hd ** -0.5)
    err, bound = ((out.double() - want).abs() / want).max().item(), U * (11 * X + 20)
    assert err <= bound, (err, bound)


@pytest.mark.parametrize("rows,kv,G,hd,br,n", SINK_SHAPES)
def test_attend_weights_of_every_size(ops, rows, kv, G, hd, br, n):  # noqa: F811
    """The larger a key's score, the smaller its value: keys from 0 to 100 below the largest, in every tile, all count alike in one
    dim of the result or another. (fp32 itself may lose weights below 2^-126, 87 below the largest: that much of a value below 2.)"""
    torch.manual_seed(rows * n)
    keys = n * br
    below = (torch.rand(rows * n + 1, kv, br, device="cuda") * 100)
    below[:, :, 3] = 0.0
    k = torch.randn(rows * n + 1, kv, br, hd, device="cuda").half() * 0.25
    k[..., 0] = (-below * hd ** 0.5 / 4.0).half()
    below = -k[..., 0].double() * 4 / hd ** 0.5  # what fp16 made of it
    v = torch.zeros(rows * n + 1, kv, br, hd, dtype=torch.float16, device="cuda")
    dim = (below / 100 * (hd - 1)).long().clamp_max(hd - 1)  # a dim for each range of distances: 1.6 or 0.8 wide
    v.scatter_(3, dim[..., None], 1 + torch.rand(dim.shape, device="cuda").half()[..., None])
    table = np.arange(1, rows * n + 1, dtype=np.int32).reshape(rows, n)
    q = torch.randn(rows, kv, G, hd, device="cuda") * 0.25
    q[..., 0] = 4.0
    cache, packed = _views(ops, table, np.arange(rows), np.full(rows, keys - 1), br, rows * n + 1, k, v)
    out = torch.empty(rows, kv, G, hd, device="cuda")
    cache.attend(packed, q, dev(np.tile(np.arange(n, dtype=np.int32), (rows, kv, 1))), out)
    torch.cuda.synchronize()
    flat = lambda a: a[dev(table).long()].transpose(1, 2).reshape(rows, kv, keys, hd)  # noqa: E731
    want, X = _exact(q, flat(k), flat(v), hd ** -0.5)
    bound = U * (11 * X + 20)
    assert ((out.double() - want).abs() <= bound * want + keys * 2.0 ** -125).all(), (((out.double() - want).abs() / want.clamp_min(1e-35)).max().item(), bound)
    assert (out[want > keys * 2.0 ** -124] > 0).all()


@pytest.mark.parametrize("rows,kv,G,hd,br,n", SINK_SHAPES)
@pytest.mark.parametrize("small", [1e-3, 1e-5, 1e-7])
def test_attend_small_queries_against_large_keys(ops, rows, kv, G, hd, br, n, small):  # noqa: F811
    """One dim of the keys is thousands of times the others, and the query is `small` there. A query is kept to 2^-36 of the head's
    largest where that is more than 2^-22 of it: a score may be off by F = 2^-36 max|q| scale sum |k| besides, the maximum too, and both enter
    numerator and denominator."""
    torch.manual_seed(rows + 7 * n)
    keys = n * br
    k = (torch.randn(rows * n + 1, kv, br, hd, device="cuda") * 0.05).half()
    k[..., 9] = ((torch.rand(rows * n + 1, kv, br, device="cuda") * 2 - 1) * 6e4).half()
    v = (1 + torch.rand(rows * n + 1, kv, br, hd, device="cuda")).half()
    table = np.arange(1, rows * n + 1, dtype=np.int32).reshape(rows, n)
    q = torch.randn(rows, kv, G, hd, device="cuda")
    q[..., 9] = small * (1 + torch.rand(rows, kv, G, device="cuda"))
    cache, packed = _views(ops, table, np.arange(rows), np.full(rows, keys - 1), br, rows * n + 1, k, v)
    out = torch.empty(rows, kv, G, hd, device="cuda")
    cache.attend(packed, q, dev(np.tile(np.arange(n, dtype=np.int32), (rows, kv, 1))), out, scale=0.125)
    torch.cuda.synchronize()
    flat = lambda a: a[dev(table).long()].transpose(1, 2).reshape(rows, kv, keys, hd)  # noqa: E731
    want, X = _exact(q, flat(k), flat(v), 0.125)
    F = 2.0 ** -36 * q.abs().max().item() * 0.125 * k.double().abs().sum(-1).max().item()
    err, bound = ((out.double() - want).abs() / want).max().item(), U * (11 * X + 20) + 4 * F
    assert err <= bound, (err, bound)


@pytest.mark.parametrize("rows,kv,G,hd,br,n", SINK_SHAPES)
def test_attend_keys_of_minus_infinity(ops, rows, kv, G, hd, br, n):  # noqa: F811
    """A key value below -65520 is stored as -inf; against a query above zero its score is -inf and its weight 0. A row whose keys
    all are so has no weight and gives 0; one key at +inf gives NaN, as inf - inf does."""
    torch.manual_seed(rows + 3 * n)
    keys = n * br
    k = torch.randn(rows * n + 1, kv, br, hd, device="cuda").half()
    v = (1 + torch.rand(rows * n + 1, kv, br, hd, device="cuda")).half()
    table = np.arange(1, rows * n + 1, dtype=np.int32).reshape(rows, n)
    k[..., 7] = torch.where(torch.rand(k.shape[:-1], device="cuda") < 0.4, -np.inf, k[..., 7].float()).half()
    k[..., 2::4, 11] = -np.inf
    k[..., ::4, (7, 11)] = -1.0
    q = torch.randn(rows, kv, G, hd, device="cuda")
    q[..., 7], q[..., 11] = 1.0, 1.2  # 1.0 has nothing in its lower part, 1.2 something below zero
    assert (q[..., 11].half().float() - q[..., 11] > 0).all()
    k[-1, -1, :, 7] = -np.inf
    none = n == 1  # the last row and head sees that block alone
    cache, packed = _views(ops, table, np.arange(rows), np.full(rows, keys - 1), br, rows * n + 1, k, v)
    out = torch.empty(rows, kv, G, hd, device="cuda")
    sel = dev(np.tile(np.arange(n, dtype=np.int32), (rows, kv, 1)))
    cache.attend(packed, q, sel, out)
    torch.cuda.synchronize()
    flat = lambda a: a[dev(table).long()].transpose(1, 2).reshape(rows, kv, keys, hd)  # noqa: E731
    want, _ = _exact(q, flat(k), flat(v), hd ** -0.5)
    if none:
        assert want[-1, -1].isnan().all() and out[-1, -1].eq(0).all()
        want[-1, -1] = 0.0
    _, X = _exact(q, flat(k.nan_to_num(neginf=0.0)), flat(v), hd ** -0.5)
    assert ((out.double() - want).abs() <= U * (11 * X + 20) * want).all()
    k[int(table[0, 0]), 0, 0, 7] = np.inf
    cache.attend(packed, q, sel, out)
    torch.cuda.synchronize()
    assert out[0, 0].isnan().all() and not out[1:].isnan().any()
