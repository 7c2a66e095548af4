"""The prefill attention of short runs (mma.sync) over keys whose weights lie far apart, against 64 bits.

Values are positive, so that nothing cancels. u = 2^-22, X the largest scale * sum |q k|. As derived for the attention over listed blocks
(test_gpu_paged_values.py), numerator and denominator together are off by u (11 X + 20); besides, the matrix unit cuts off what it
adds to, by at most 2 u a step of 16 products, two steps for 16 keys. A weight below 2^-18 of its row's largest is kept to 2^-40 of that
one, which weighs 1 at most; values are at most 2."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -22


@pytest.fixture(scope="module")
def ops():
    from goinfer_b200.ops import Ops
    return Ops(0)


@pytest.mark.parametrize("rows,pos0,heads,kv,hd,br", [(17, 30, 2, 1, 64, 16), (40, 0, 8, 8, 128, 16), (33, 300, 32, 8, 128, 32), (100, 500, 8, 2, 64, 64)])
@pytest.mark.parametrize("gap", [6.0, 12.0, 17.0, 18.5])
@pytest.mark.parametrize("value", [0.0, 0.02, 1.0])
def test_one_key_above_all_others(ops, rows, pos0, heads, kv, hd, br, gap, value):
    rng = np.random.default_rng(heads * hd)
    keys, G = pos0 + rows, heads // kv
    q = rng.normal(0, 1, (rows, kv, G, hd)).astype(np.float32)
    k = rng.normal(0, 1, (keys, kv, hd)).astype(np.float16).astype(np.float32)
    v = (1 + rng.random((keys, kv, hd))).astype(np.float16).astype(np.float32)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[0] = 0.0
    k[0, :, 0] = np.float16(gap * hd ** 0.5 / 4.0)
    v[0] = np.float16(value)
    got = ops.prefill_attention(q.reshape(rows, -1), k.reshape(keys, -1), v.reshape(keys, -1), pos0, heads, kv, hd, block_rows=br)
    got = np.asarray(got, np.float64).reshape(rows, kv, G, hd)
    for r in range(rows):
        n = pos0 + r + 1
        kk, vv, qq = (a.astype(np.float64) for a in (k[:n], v[:n], q[r]))
        x = np.einsum("hgd,khd->hgk", qq, kk) * hd ** -0.5
        X = (np.einsum("hgd,khd->hgk", np.abs(qq), np.abs(kk)) * hd ** -0.5).max()
        w = np.exp(x - x.max(-1, keepdims=True))
        want = np.einsum("hgk,khd->hgd", w / w.sum(-1, keepdims=True), vv)
        bound = U * (11 * X + 20 + 4 * -(-n // 16))
        over = (np.abs(got[r] - want) - bound * want - n * 2.0 ** -40 * 2).max()
        assert over <= 0, (r, over, (np.abs(got[r] - want) / np.maximum(want, 1e-30)).max(), bound)
