"""The paged selection where hundreds of blocks are in doubt and one CTA of a cluster gathers and chooses alone: an infinite bound of the
scores' error, equal scores, scores that differ behind their 30th bit, against a stable sort of the scores in 64 bits."""
import numpy as np
import pytest

from test_gpu_paged import _select_reference, _views, dev, ops  # noqa: F401

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("rows,kv,G,hd,max_blocks,n_first,n_recent,n", [(1, 1, 4, 128, 300, 1, 1, 64), (1, 8, 4, 128, 514, 1, 1, 100), (2, 2, 8, 64, 400, 0, 2, 7),
                                                                     (3, 1, 5, 128, 511, 2, 1, 400), (1, 2, 1, 64, 260, 1, 1, 255)])
@pytest.mark.parametrize("kind", ["nan", "inf", "equal", "near", "nan and bad pages"])
def test_select_with_hundreds_in_doubt(ops, rows, kv, G, hd, max_blocks, n_first, n_recent, n, kind):  # noqa: F811
    rng = np.random.default_rng(max_blocks + G)
    n_blocks, br = rows * max_blocks + 1, 16
    bounds = np.sort(rng.normal(0, 1, (n_blocks, kv, 2, hd)), axis=2).astype(np.float16)
    q = rng.normal(0, 1, (rows, kv * G * hd)).astype(np.float32)
    table = (1 + np.arange(rows * max_blocks, dtype=np.int32)).reshape(rows, max_blocks)
    if kind.startswith("nan"):  # in the last head of each group: all scores of its kv head count as the largest
        q.reshape(rows, kv, G, hd)[:, :, -1, 9] = np.nan
    if kind == "inf":  # in some bounds: those scores are the largest or the lowest, the rest are ordered in f64
        bounds[rng.random(n_blocks) < 0.1, :, 1, 3] = np.inf
        bounds[rng.random(n_blocks) < 0.1, :, 0, 4] = -np.inf
    if kind in ("equal", "near"):
        bounds[:] = bounds[0]
    if kind == "near":
        q.reshape(rows, kv, G, hd)[..., 0] = 2.0 ** -29
        bounds[:, :, 1, 0] = np.abs(rng.normal(0, 1, (n_blocks, kv)))
    if kind == "nan and bad pages":
        table[rng.random(table.shape) < 0.5] = 0
        table[rng.random(table.shape) < 0.1] = n_blocks
    slot, pos = np.arange(rows, dtype=np.int32), np.full(rows, max_blocks * br - 1, np.int32)
    cache, packed = _views(ops, table, slot, pos, br, n_blocks, key_bounds=torch.from_numpy(bounds).cuda())
    before = np.full((rows, kv, n), -7, np.int32)
    for _ in range(3):  # (what another call left in shared memory is no part of the answer)
        sel = dev(before)
        cache.select(packed, torch.from_numpy(q).cuda(), sel, n_first=n_first, n_recent=n_recent)
        torch.cuda.synchronize()
        np.testing.assert_array_equal(sel.cpu().numpy(), _select_reference(q, bounds, table, slot, pos, br, kv, n_first, n_recent, n, before))


@pytest.mark.parametrize("rows,kv,G,hd,max_blocks,n", [(1, 2, 4, 128, 90, 12), (3, 1, 8, 64, 700, 40), (40, 2, 2, 64, 30, 9)])
def test_select_scores_of_minus_infinity_are_the_lowest(ops, rows, kv, G, hd, max_blocks, n):  # noqa: F811
    """A block whose keys are all -inf in a dim where every query is above zero scores -inf: no more than an unmapped block, and less
    than every other one. With too few others the lower of these is taken."""
    rng = np.random.default_rng(max_blocks)
    n_blocks, br = rows * max_blocks + 1, 16
    bounds = np.sort(rng.normal(0, 1, (n_blocks, kv, 2, hd)), axis=2).astype(np.float16)
    q = rng.normal(0, 1, (rows, kv, G, hd)).astype(np.float32)
    q[..., 4] = np.abs(q[..., 4]) + 0.1
    table = (1 + np.arange(rows * max_blocks, dtype=np.int32)).reshape(rows, max_blocks)
    others = rng.permutation(max_blocks - 2)[:n // 2] + 1  # fewer than there is room for
    low = np.setdiff1d(np.arange(1, max_blocks - 1), others)
    bounds[table[:, low[::2]], :, :, 4] = -np.inf
    table[:, low[1::2]] = 0
    slot, pos = np.arange(rows, dtype=np.int32), np.full(rows, max_blocks * br - 1, np.int32)
    cache, packed = _views(ops, table, slot, pos, br, n_blocks, key_bounds=torch.from_numpy(bounds).cuda())
    sel = torch.zeros(rows, kv, n, dtype=torch.int32, device="cuda")
    cache.select(packed, torch.from_numpy(q.reshape(rows, -1)).cuda(), sel)
    torch.cuda.synchronize()
    want = np.sort(np.concatenate(([0, max_blocks - 1], others, low[:n - 2 - len(others)])))
    assert (sel.cpu().numpy() == want).all()
