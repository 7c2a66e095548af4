"""The decode attention over keys whose weights lie far apart (paged, at most 512 keys a split, four warps a split), against 64 bits.

Values are positive, so that nothing cancels. u = 2^-22, X the largest scale * sum |q k|. As derived for the attention over listed blocks
(test_gpu_paged_values.py), numerator and denominator together are off by u (11 X + 20); besides, the matrix unit cuts off what it adds
to, by at most 2 u a step of 16 products: two steps a tile, eight tiles a warp: 32 u. A weight below 2^-18 of the largest of its
warp's keys (128 at most) is kept to 2^-40 of that one, which weighs 1 at most; values are at most 2."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -22


@pytest.fixture(scope="module")
def ops():
    from goinfer_b200.ops import Ops
    return Ops(0)


@pytest.mark.parametrize("n_keys,heads,kv,hd,br", [([7], 2, 1, 64, 16), ([64, 33], 8, 8, 128, 16), ([512, 300, 200], 32, 8, 128, 32), ([1300, 2048], 16, 2, 64, 64), ([700], 4, 2, 128, 16)])
@pytest.mark.parametrize("gap", [6.0, 12.0, 17.0, 18.5])
@pytest.mark.parametrize("value", [0.0, 0.02, 1.0])
def test_one_key_above_all_others(ops, n_keys, heads, kv, hd, br, gap, value):
    rng = np.random.default_rng(heads * hd)
    rows, most, G = len(n_keys), max(n_keys), heads // kv
    q = rng.normal(0, 1, (rows, kv, G, hd)).astype(np.float32)
    k = rng.normal(0, 1, (rows, most, kv, hd)).astype(np.float16).astype(np.float32)
    v = (1 + rng.random((rows, most, kv, hd))).astype(np.float16).astype(np.float32)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[:, 5] = 0.0
    k[:, 5, :, 0] = np.float16(gap * hd ** 0.5 / 4.0)
    v[:, 5] = np.float16(value)
    got = ops.attention(q.reshape(rows, -1), k.reshape(rows, most, -1), v.reshape(rows, most, -1), np.array(n_keys, np.int32), heads, kv, hd, block_rows=br, klass=2)
    got = np.asarray(got, np.float64).reshape(rows, kv, G, hd)
    for r, n in enumerate(n_keys):
        kk, vv, qq = (a.astype(np.float64) for a in (k[r, :n], v[r, :n], q[r]))
        x = np.einsum("hgd,khd->hgk", qq, kk) * hd ** -0.5
        X = (np.einsum("hgd,khd->hgk", np.abs(qq), np.abs(kk)) * hd ** -0.5).max()
        w = np.exp(x - x.max(-1, keepdims=True))
        want = np.einsum("hgk,khd->hgd", w / w.sum(-1, keepdims=True), vv)
        over = (np.abs(got[r] - want) - U * (11 * X + 52) * want - min(n, 128) * 2.0 ** -40 * 2).max()
        assert over <= 0, (r, over, (np.abs(got[r] - want) / want).max(), U * (11 * X + 52))
