"""The paged-cache operators on the GPU against plain implementations in 64 bits: plan against a list-based block allocator,
append and select exactly, attend to a derived bound, a step of all four captured into a graph, and two graphs at once.

Attend's tolerance. u = 2^-22 is the relative residue of a value split into two fp16 parts (two roundings of 2^-11). A score
is off by at most u * scale * sum |q k| (the split of q) and as much again for its fp32 sum (its terms' roundings of 2^-24 do
not line up over up to 128 of them: taken as u); that is e_x = 2 u X, X the largest scale * sum |q k| of the case (a softcap only shrinks it). A
weight is then off by e_x, by __expf (2 + 1.2 |x| ulp of 2^-23 <= u (1 + X), |x - max| <= 2 X), by its own split (u), by the
running rescale and by the fp32 sums (u each); numerator and denominator both carry it. Relative to the result's 2-norm that is
2 * u * (2 X + 1 + X + 3) = u * (6 X + 8); the largest single deviation is held to eight times that of the row's rms."""
import ctypes as C
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from goinfer_b200 import abi

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ops():
    from goinfer_b200.ops import Ops
    return Ops(0, stream=1)  # the legacy default stream, torch's own


def dev(a, dtype=np.int32):
    return torch.from_numpy(np.ascontiguousarray(a, dtype)).cuda()


class Pool:
    """Device arrays of a cache, and the list-based allocator that says what they should hold."""

    def __init__(self, ops, n_seqs, max_blocks, n_blocks, br, n_rows, rng, **pools):
        from goinfer_b200.paged import PagedCache, PagedRows
        self.br, self.n_rows, self.n_blocks = br, n_rows, n_blocks
        self.table = np.zeros((n_seqs, max_blocks), np.int32)
        self.blocks = np.zeros(n_seqs, np.int32)
        self.free = list(map(int, rng.permutation(n_blocks - 1) + 1))
        stack = np.zeros(n_blocks, np.int32)
        stack[:len(self.free)] = self.free
        self.d = dict(table=dev(self.table), blocks=dev(self.blocks), stack=dev(stack), count=dev([len(self.free)]))
        self.r = dict(slot=torch.full((n_rows,), 77, dtype=torch.int32, device="cuda"), row0=torch.full((n_seqs + 1,), 77, dtype=torch.int32, device="cuda"),
                      status=torch.zeros(4, dtype=torch.int32, device="cuda"))
        self.r["pos"], self.r["map"] = self.r["slot"].clone(), self.r["slot"].clone()
        self.cache = PagedCache(ops, self.d["table"], self.d["blocks"], self.d["stack"], self.d["count"], br, **pools)
        self.rows = PagedRows(self.r["slot"], self.r["pos"], self.r["map"], self.r["row0"], self.r["status"])

    def plan(self, kv_len, n_new):
        kv_len, n_new = np.asarray(kv_len, np.int64), np.asarray(n_new, np.int64)
        self.cache.plan(dev(kv_len), dev(n_new), self.rows)
        want = (kv_len + n_new + self.br - 1) // self.br
        bad = (kv_len < 0) | (n_new < 0) | (kv_len + n_new > self.table.shape[1] * self.br) | (kv_len > self.blocks.astype(np.int64) * self.br)
        live = [(-1, -1, -1)] * self.n_rows
        row0 = np.zeros(len(kv_len) + 1, np.int64)
        if bad.any() or n_new.sum() > self.n_rows:
            status = [3, 0, len(self.free), int(bad.argmax()) if bad.any() else len(bad)]
        elif (missing := int(np.maximum(0, want - self.blocks).sum()) - int(np.maximum(0, self.blocks - want).sum()) - len(self.free)) > 0:
            status = [2, 0, len(self.free), missing]
        else:
            for i in range(len(want) - 1, -1, -1):
                for p in range(self.blocks[i] - 1, want[i] - 1, -1):
                    self.free.append(int(self.table[i, p]))
                    self.table[i, p] = 0
            for i in range(len(want)):
                for p in range(self.blocks[i], want[i]):
                    self.table[i, p] = self.free.pop()
            self.blocks = want.astype(np.int32)
            row0[1:] = np.cumsum(n_new)
            rows = [(i, pos, int(self.table[i, pos // self.br]) * self.br + pos % self.br)
                    for i in range(len(want)) for pos in range(kv_len[i], kv_len[i] + n_new[i])]
            live = rows + live[len(rows):]
            status = [0, len(rows), len(self.free), 0]
        torch.cuda.synchronize()
        assert self.r["status"].tolist() == status
        assert np.array_equal(self.d["table"].cpu().numpy(), self.table) and np.array_equal(self.d["blocks"].cpu().numpy(), self.blocks)
        assert self.d["count"].item() == len(self.free) and self.d["stack"][:len(self.free)].tolist() == self.free
        assert self.r["row0"].tolist() == row0.tolist()
        got = torch.stack((self.r["slot"], self.r["pos"], self.r["map"]), 1).cpu().numpy()
        assert np.array_equal(got, np.array(live).reshape(-1, 3))
        return status[0]


@pytest.mark.parametrize("n_seqs,max_blocks,br,n_rows", [(1, 1, 16, 4), (3, 40, 16, 700), (37, 9, 48, 300), (1030, 7, 256, 9000), (2500, 6, 16, 30000),
                                                         (16384, 2, 16, 20000)])
def test_plan_follows_a_list_allocator(ops, n_seqs, max_blocks, br, n_rows):
    rng = np.random.default_rng(n_seqs)
    p = Pool(ops, n_seqs, max_blocks, 1 + int(0.6 * n_seqs * max_blocks) + 2, br, n_rows, rng)
    length, codes = np.zeros(n_seqs, np.int64), []
    for step in range(12):
        keep = length - np.where(rng.random(n_seqs) < 0.3, rng.integers(0, 3 * br, n_seqs), 0)
        keep = np.where(rng.random(n_seqs) < 0.1, 0, np.maximum(keep, 0))
        new = rng.integers(0, max(2, 2 * n_rows // n_seqs), n_seqs)
        new = np.minimum(np.where(rng.random(n_seqs) < 0.4, 0, new), max_blocks * br - keep)
        if step % 4 == 3:
            new[:] = max_blocks * br - keep  # more blocks than there are, or more rows than the arrays hold
        codes.append(p.plan(keep, new))
        if codes[-1] == 0:
            length = keep + new
    p.plan(np.zeros(n_seqs), np.zeros(n_seqs))
    assert len(p.free) == p.n_blocks - 1
    assert 0 in codes
    if n_seqs > 3:
        assert {2, 3} & set(codes)


def test_plan_refuses_on_the_device(ops):
    rng = np.random.default_rng(5)
    p = Pool(ops, 4, 6, 13, 16, 100, rng)
    assert p.plan([0, 0, 0, 0], [20, 0, 33, 1]) == 0
    for keep, new in (([20, -1, 33, 1], [0, 0, 0, 0]), ([20, 0, 33, 1], [0, 0, 0, -1]), ([20, 0, 33, 1], [0, 97, 0, 0]), ([33, 0, 33, 1], [0, 0, 0, 0]),
                      ([20, 1, 33, 1], [0, 0, 0, 0]), ([20, 0, 33, 1], [25, 25, 25, 26]), ([2**31 - 1] * 4, [2**31 - 1] * 4), ([-2**31] * 4, [-2**31] * 4)):
        assert p.plan(keep, new) == 3
    assert p.plan([20, 0, 33, 1], [0, 96, 0, 0]) == 0 and len(p.free) == 0
    assert p.plan([20, 96, 33, 1], [13, 0, 0, 0]) == 2
    assert p.plan([32, 96, 48, 16], [0, 0, 0, 0]) == 0
    assert p.plan([32, 0, 48, 16], [13, 80, 0, 0]) == 0  # what one sequence gives back serves another
    # a free count that cannot be is refused, and nothing is read behind the stack
    for count in (-1, 14, 2**31 - 1):
        p.d["count"].fill_(count)
        before = [t.clone() for t in p.d.values()]
        p.cache.plan(dev([32, 80, 48, 16]), dev([0, 0, 0, 0]), p.rows)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(before, p.d.values()))
        assert p.r["status"].tolist() == [3, 0, count, 4]


def test_plan_growing_and_giving_back_restores_the_stack(ops):
    rng = np.random.default_rng(6)
    p = Pool(ops, 50, 20, 900, 16, 16000, rng)
    keep = rng.integers(0, 100, 50)
    p.plan(np.zeros(50), keep)
    stack, table = list(p.free), p.table.copy()
    p.plan(keep, rng.integers(0, 200, 50))
    p.plan(keep, np.zeros(50))
    assert p.free == stack and np.array_equal(p.table, table)


def _bounds(pool, page, last):
    with np.errstate(invalid="ignore"):
        keys = pool[page, :, :last + 1].astype(np.float32)
        return np.stack((keys.min(1), keys.max(1)), 1).astype(np.float16)  # NaN wins in numpy's min and max as well


@pytest.mark.parametrize("kv,hd,br", [(8, 128, 16), (4, 64, 32), (1, 64, 48), (9, 128, 256), (2, 128, 64)])
@pytest.mark.parametrize("bounded", [True, False])
def test_append_stores_rows_and_bounds(ops, kv, hd, br, bounded):
    rng = np.random.default_rng(kv * br)
    n_blocks, n_seqs = 14, 3
    k_pool = rng.normal(0, 1, (n_blocks, kv, br, hd)).astype(np.float16)
    v_pool = rng.normal(0, 1, k_pool.shape).astype(np.float16)
    k_pool[:, :, ::3] = np.nan  # stale rows must not show in any bound
    bounds = rng.normal(0, 1, (n_blocks, kv, 2, hd)).astype(np.float16)
    dk, dv, db = (torch.from_numpy(a).cuda() for a in (k_pool, v_pool, bounds))
    p = Pool(ops, n_seqs, 4, n_blocks, br, 3 * br + 9, rng, k_pool=dk, v_pool=dv, key_bounds=db if bounded else None)
    keep = np.zeros(n_seqs, np.int64)
    for new in ([1, 0, br + 3], [1, br - 1, 2], [br - 2, 2, 1], [0, 0, 0], [5, 1, 2 * br - 7]):
        assert p.plan(keep, new) == 0
        keep = keep + new
        x = torch.empty(p.n_rows, 3, kv * hd, device="cuda").normal_()  # k and v inside a wider row
        x[0, 0, 0], x[0, 0, 1], x[0, 1, 2], x[min(2, p.n_rows - 1), 0, hd - 1] = 7e4, -7e4, 3e-8, float("nan")
        k, v = x[:, 0], x[:, 1]
        p.cache.append(p.rows, k, v)
        torch.cuda.synchronize()
        with np.errstate(over="ignore"):
            hk, hv = k.cpu().numpy().astype(np.float16).reshape(-1, kv, hd), v.cpu().numpy().astype(np.float16).reshape(-1, kv, hd)
        last = {}
        for r, at in enumerate(p.r["map"].tolist()):
            if at >= 0:
                k_pool[at // br, :, at % br], v_pool[at // br, :, at % br] = hk[r], hv[r]
                last[at // br] = at % br
        if bounded:
            for page, row in last.items():
                bounds[page] = _bounds(k_pool, page, row)
        for got, want in ((dk, k_pool), (dv, v_pool), (db, bounds)):
            np.testing.assert_array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("kv,hd,br,news", [(2, 64, 16, (901, 0, 777)), (8, 128, 32, (300, 13, 500)), (1, 128, 64, (2049, 1, 2700)), (3, 64, 16, (5000, 1, 17))])
def test_append_of_many_rows(ops, kv, hd, br, news):
    """Prompts: a CTA looks for runs among several rows, runs begin and end anywhere among them."""
    rng = np.random.default_rng(br)
    torch.manual_seed(br)
    n_blocks = sum(-(-(n + br) // br) for n in news) + 4
    k_pool = torch.full((n_blocks, kv, br, hd), float("nan"), dtype=torch.float16, device="cuda")
    v_pool, bounds = torch.zeros_like(k_pool), torch.zeros(n_blocks, kv, 2, hd, dtype=torch.float16, device="cuda")
    p = Pool(ops, 3, max(news) // br + 2, n_blocks, br, sum(news) + 40, rng, k_pool=k_pool, v_pool=v_pool, key_bounds=bounds)
    assert p.plan([0, 0, 0], [5, 2, 0]) == 0
    x = torch.randn(p.n_rows, kv, hd, device="cuda")
    p.cache.append(p.rows, x, x)
    assert p.plan([5, 2, 0], news) == 0
    y = torch.randn(p.n_rows, kv, hd, device="cuda")
    p.cache.append(p.rows, y, -y)
    torch.cuda.synchronize()
    r = 0
    for s, (first, new, old) in enumerate(zip((5, 2, 0), news, ([0, 5], [5, 7], [7, 7]))):
        keys = torch.cat((x[old[0]:old[1]], y[r:r + new])).half()
        r += new
        for b in range(-(-len(keys) // br)):
            page, part = int(p.table[s, b]), keys[b * br:(b + 1) * br]
            assert torch.equal(k_pool[page, :, :len(part)], part.transpose(0, 1))
            if len(keys) > b * br + (first if b == 0 else 0):  # written to by the second step
                assert torch.equal(v_pool[page, :, max(0, first - b * br):len(part)], -part[max(0, first - b * br):].transpose(0, 1))
            assert torch.equal(bounds[page], torch.stack((part.amin(0), part.amax(0)), 1))
    assert k_pool[0].isnan().all() and bounds[0].eq(0).all()


def test_append_leaves_bad_slots_out(ops):
    rng = np.random.default_rng(1)
    pool = torch.zeros(6, 2, 16, 64, dtype=torch.float16, device="cuda")
    other, bounds = pool.clone(), torch.zeros(6, 2, 2, 64, dtype=torch.float16, device="cuda")
    p = Pool(ops, 2, 4, 6, 16, 7, rng, k_pool=pool, v_pool=other, key_bounds=bounds)
    p.r["map"].copy_(dev([0, 15, -1, -2**31, 6 * 16, 2**31 - 1, 5 * 16 + 15]))  # the null block, idle rows, past the pool, one good row
    k = torch.ones(7, 2, 64, device="cuda")
    p.cache.append(p.rows, k, 2 * k)
    torch.cuda.synchronize()
    assert pool[:5].eq(0).all() and other[:5].eq(0).all() and bounds[:5].eq(0).all()
    assert pool[5, :, 15].eq(1).all() and pool[5, :, :15].eq(0).all() and other[5, :, 15].eq(2).all()
    assert bounds[5, :, 0].eq(0).all() and bounds[5, :, 1].eq(1).all()


def _select_reference(q, bounds, table, slot, pos, br, kv, n_first, n_recent, n, before):
    out = before.copy()
    n_blocks, top = bounds.shape[0], np.finfo(np.float64).max
    for r in range(len(slot)):
        if slot[r] < 0 or slot[r] >= len(table) or pos[r] < 0:
            continue
        have = min(pos[r] // br, table.shape[1] - 1) + 1
        page = table[slot[r], :have]
        good = (page > 0) & (page < n_blocks)
        for h in range(kv):
            if have <= n:
                chosen = np.arange(have)
            else:
                qh = q[r].astype(np.float64).reshape(kv, -1, bounds.shape[-1])[h]
                b = bounds[np.where(good, page, 0), h].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = (qh[None] * np.where(qh[None] > 0, b[:, 1][:, None], b[:, 0][:, None])).sum(-1).max(1)  # NaN wins in numpy's max
                s = np.where(good, np.nan_to_num(s, nan=top, posinf=top, neginf=-top), -top)
                middle = np.arange(n_first, have - n_recent)
                order = middle[np.argsort(-s[middle], kind="stable")]
                chosen = np.sort(np.concatenate((np.arange(n_first), order[:n - n_first - n_recent], np.arange(have - n_recent, have))))
            out[r, h] = -1
            out[r, h, :len(chosen)] = chosen
    return out


def _context(rng, rows, max_blocks, br, n_blocks):
    table = rng.integers(1, n_blocks, (rows, max_blocks)).astype(np.int32)
    slot = rng.permutation(rows).astype(np.int32)
    pos = rng.integers(0, max_blocks * br, rows).astype(np.int32)
    pos[0] = max_blocks * br - 1
    return table, slot, pos


def _views(ops, table, slot, pos, br, n_blocks, k_pool=None, v_pool=None, key_bounds=None):
    from goinfer_b200.paged import PagedCache, PagedRows
    z = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    return PagedCache(ops, dev(table), z(len(table)), z(n_blocks), z(1), br, k_pool, v_pool, key_bounds), PagedRows(dev(slot), dev(pos))


SELECT_SHAPES = [(1, 2, 1, 64, 16, 300, 1, 1, 8), (5, 3, 2, 128, 16, 70, 1, 1, 9), (2, 1, 3, 64, 48, 700, 0, 1, 33), (3, 2, 4, 128, 32, 2100, 2, 3, 256),
                 (40, 8, 4, 128, 16, 90, 1, 1, 64), (4, 1, 5, 64, 16, 129, 1, 2, 3), (3, 1, 6, 128, 64, 65, 3, 4, 64), (2, 2, 7, 128, 16, 333, 1, 1, 2),
                 (7, 2, 8, 128, 16, 530, 1, 1, 100), (1, 1, 8, 64, 16, 5000, 1, 1, 2048), (300, 1, 1, 64, 16, 12, 1, 1, 5), (1, 1, 2, 64, 16, 24576, 1, 1, 700),
                 # clusters of 8 with three CTAs an SM, of 4 where those of 8 do not fit, pairs, and single CTAs
                 (12, 4, 8, 64, 16, 600, 1, 2, 40), (18, 4, 2, 64, 16, 600, 2, 1, 40), (9, 8, 4, 128, 16, 520, 1, 1, 30), (20, 8, 5, 128, 16, 130, 1, 1, 24),
                 (40, 8, 2, 128, 16, 70, 0, 1, 9), (300, 1, 8, 64, 32, 66, 1, 1, 9)]


@pytest.mark.parametrize("rows,kv,G,hd,br,max_blocks,n_first,n_recent,n", SELECT_SHAPES)
@pytest.mark.parametrize("kind", ["spread", "ties", "outliers"])
def test_select_takes_the_best_blocks(ops, rows, kv, G, hd, br, max_blocks, n_first, n_recent, n, kind):
    rng = np.random.default_rng(rows * max_blocks + G)
    n_blocks = min(rows * max_blocks + 1, 9000)
    centre, reach = rng.normal(0, 1, (n_blocks, kv, hd)), np.abs(rng.normal(0, 1, (n_blocks, kv, hd)))
    bounds = np.stack((centre - reach, centre + reach), 2).astype(np.float16)
    if kind == "outliers":  # a few blocks and one dim far off: the range of the scores says little about most of them
        centre[rng.random(n_blocks) < 0.02] *= 400
        centre[:, :, 5] *= 30
        bounds = np.stack((centre - reach, centre + reach), 2).astype(np.float16)
    if kind == "ties":
        bounds = bounds[rng.integers(0, 4, n_blocks)]  # four kinds of blocks: most decisions are ties
    q = rng.normal(0, 1, (rows, kv * G * hd)).astype(np.float32)
    table, slot, pos = _context(rng, rows, max_blocks, br, n_blocks)
    if rows > 2:
        slot[1] = -1
        pos[2] = 0
    cache, packed = _views(ops, table, slot, pos, br, n_blocks, key_bounds=torch.from_numpy(bounds).cuda())
    before = rng.integers(-9, 0, (rows, kv, n)).astype(np.int32)
    sel = dev(before)
    wide = torch.zeros(rows, kv * G * hd + 12, device="cuda")
    wide[:, :kv * G * hd] = torch.from_numpy(q).cuda()
    cache.select(packed, wide[:, :kv * G * hd], sel, n_first=n_first, n_recent=n_recent)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(sel.cpu().numpy(), _select_reference(q, bounds, table, slot, pos, br, kv, n_first, n_recent, n, before))


@pytest.mark.parametrize("max_blocks", [80, 900])
def test_select_values_out_of_the_ordinary(ops, max_blocks):
    """Zeros of both signs, subnormal and largest fp16 bounds, infinities and NaN in the bounds and in q, bad pages, equal rows,
    positions past the table, and scores that agree to 30 bits."""
    rng = np.random.default_rng(3)
    rows, kv, G, hd, br, n = 12, 2, 2, 64, 16, 20
    n_blocks = 200
    bounds = np.sort(rng.normal(0, 1, (n_blocks, kv, 2, hd)), axis=2).astype(np.float16)
    bounds[1:8] = 0.0
    bounds[8:12] = -0.0
    bounds[12:20] *= np.float16(6e-8)
    bounds[20:30] = np.where(bounds[20:30] > 0, 65504, -65504).astype(np.float16)
    bounds[30, :, 1, 3], bounds[31, 0, 0, 5], bounds[32, 1, 1, 7], bounds[33, :, 0, 9] = np.inf, -np.inf, np.nan, np.nan
    bounds[40:60] = bounds[40]
    bounds[41:60, :, 1, 0] = np.nextafter(bounds[40, :, 1, 0], np.float16(9))  # one last place of one dim apart
    q = rng.normal(0, 1, (rows, kv * G * hd)).astype(np.float32)
    q[:, ::7] = 0.0
    q[3] *= 1e-30
    q[4] *= 1e30
    q[5, 3], q[6, 70], q[7, 9] = np.inf, -np.inf, np.nan
    q[8] = 0.0
    q[:, 0] = 1e-6  # the bound that is one place apart hardly counts
    table, slot, pos = _context(rng, rows, max_blocks, br, n_blocks)
    table[:, 5], table[:, 6], table[:, 7], table[:, 8] = 0, -3, n_blocks, 2**31 - 1
    table[slot[9]] = 0          # nothing mapped: every score is the lowest
    pos[:] = max_blocks * br - 1
    pos[10], pos[11] = 2**31 - 1, max_blocks * br + 5
    cache, packed = _views(ops, table, slot, pos, br, n_blocks, key_bounds=torch.from_numpy(bounds).cuda())
    before = np.full((rows, kv, n), -7, np.int32)
    sel = dev(before)
    cache.select(packed, torch.from_numpy(q).cuda(), sel)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(sel.cpu().numpy(), _select_reference(q, bounds, table, slot, pos, br, kv, 1, 1, n, before))


def _attend_reference(q, k_pool, v_pool, table, slot, pos, br, sel, scale, cap, before):
    """f64 on the GPU; -> result, the largest scale * sum |q k| of a case."""
    out, worst = before.double().clone(), 0.0
    n_blocks, kv, _, hd = k_pool.shape
    for r in range(len(slot)):
        if slot[r] < 0 or slot[r] >= len(table) or pos[r] < 0:
            continue
        have = min(pos[r] // br, table.shape[1] - 1) + 1
        for h in range(kv):
            qh = q[r].double().reshape(kv, -1, hd)[h]
            named = [b for b in sel[r, h].tolist() if 0 <= b < have and 0 < table[slot[r], b] < n_blocks]
            pages = torch.tensor([int(table[slot[r], b]) for b in named], dtype=torch.long, device="cuda")
            key = (torch.tensor(named, dtype=torch.long, device="cuda")[:, None] * br + torch.arange(br, device="cuda")).reshape(-1)
            seen = key <= int(pos[r])
            o = torch.zeros(qh.shape, dtype=torch.float64, device="cuda")
            if seen.any():
                k, v = k_pool[pages, h].reshape(-1, hd)[seen].double(), v_pool[pages, h].reshape(-1, hd)[seen].double()
                x = qh @ k.T * scale
                worst = max(worst, (qh.abs() @ k.abs().T * scale).max().item())
                if cap:
                    x = cap * torch.tanh(x / cap)
                o = torch.softmax(x, -1) @ v
            out[r].view(kv, -1, hd)[h] = o
    return out, worst


def _close(got, want, worst):
    u, got = 2.0 ** -22, got.double()
    bound = u * (6 * worst + 8)
    err = (got - want).norm() / want.norm()
    assert err <= bound, (err.item(), bound)
    rms = want.pow(2).mean(-1, keepdim=True).sqrt()
    assert ((got - want).abs() <= 8 * bound * torch.maximum(rms, want.abs())).all()


ATTEND_SHAPES = [(1, 1, 1, 64, 16, 1, 1, 0.0), (1, 8, 4, 128, 16, 500, 64, 0.0), (3, 2, 2, 128, 48, 30, 7, 0.0), (5, 1, 3, 64, 256, 4, 4, 20.0),
                 (4, 2, 5, 128, 16, 40, 33, 0.0), (2, 3, 6, 64, 32, 25, 25, 5.0), (9, 1, 7, 128, 64, 9, 6, 0.0), (33, 8, 8, 128, 16, 20, 12, 0.0),
                 (200, 4, 8, 64, 32, 12, 5, 0.0), (1, 1, 2, 128, 16, 2048, 2048, 0.0),
                 # clusters of 8 (three and four an SM), 4, 2, and single CTAs at head_dim 64; of 4 and 2 at 128
                 (12, 4, 4, 64, 16, 80, 64, 0.0), (17, 4, 2, 64, 16, 80, 64, 0.0), (20, 4, 3, 64, 16, 80, 64, 7.0), (40, 4, 4, 64, 32, 40, 33, 0.0),
                 (90, 4, 2, 64, 16, 40, 30, 0.0), (8, 8, 4, 128, 16, 80, 64, 0.0), (9, 8, 2, 128, 16, 80, 64, 0.0)]


@pytest.mark.parametrize("rows,kv,G,hd,br,max_blocks,n,cap", ATTEND_SHAPES)
def test_attend_over_listed_blocks(ops, rows, kv, G, hd, br, max_blocks, n, cap):
    rng = np.random.default_rng(rows + max_blocks)
    torch.manual_seed(rows)
    n_blocks = min(rows * max_blocks + 1, 4000)
    k_pool = torch.randn(n_blocks, kv, br, hd, device="cuda").half()
    v_pool = torch.randn(n_blocks, kv, br, hd, device="cuda").half()
    q = torch.randn(rows, kv * G * hd + 8, device="cuda")[:, :kv * G * hd]
    table, slot, pos = _context(rng, rows, max_blocks, br, n_blocks)
    sel = rng.integers(0, max_blocks, (rows, kv, n)).astype(np.int32)
    sel[rng.random(sel.shape) < 0.1] = -1
    if rows > 2:
        slot[1], pos[2] = -1, 0
        sel[2, :, 0] = 0
    if rows > 8:
        sel[4], sel[5, :, :] = -1, max_blocks   # lists that name nothing
        sel[6, :, 1] = sel[6, :, 0]             # named twice
        sel[7] = 2**31 - 1
        pos[8] = 2**31 - 1
    cache, packed = _views(ops, table, slot, pos, br, n_blocks, k_pool, v_pool)
    out = torch.full((rows, kv * G * hd + 4), 9.0, device="cuda")
    before = out[:, :kv * G * hd].clone()
    cache.attend(packed, q, dev(sel), out[:, :kv * G * hd], softcap=cap)
    torch.cuda.synchronize()
    want, worst = _attend_reference(q, k_pool, v_pool, table, slot, pos, br, sel, hd ** -0.5, cap, before)
    _close(out[:, :kv * G * hd], want, worst)
    assert out[:, kv * G * hd:].eq(9).all()
    if rows > 2:
        assert out[1].eq(9).all()
    if rows > 8:
        assert out[[4, 5, 7], :kv * G * hd].eq(0).all()


def test_attend_does_not_read_what_lies_behind_the_position(ops):
    """NaN and infinities in the rows behind a position, in the null block and in blocks that the list does not name."""
    kv, G, hd, br = 2, 4, 128, 32
    torch.manual_seed(2)
    k_pool = torch.randn(9, kv, br, hd, device="cuda").half()
    v_pool = torch.randn(9, kv, br, hd, device="cuda").half()
    table = np.array([[1, 2, 3, 4], [5, 6, 0, 40], [7, 8, -1, 9]], np.int32)
    pos = np.array([3 * br + 4, br + br - 2, br], np.int32)
    for pool, bad in ((k_pool, float("nan")), (v_pool, float("inf"))):
        pool[0], pool[2] = bad, bad
        pool[4, :, 5:], pool[6, :, br - 1:], pool[8, :, 1:] = bad, bad, bad
    sel = np.tile(np.array([0, 2, 3, 1], np.int32), (3, kv, 1))
    sel[0, :, 3] = -1
    q = torch.randn(3, kv * G * hd, device="cuda")
    cache, packed = _views(ops, table, np.arange(3), pos, br, 9, k_pool, v_pool)
    out = torch.empty(3, kv * G * hd, device="cuda")
    cache.attend(packed, q, dev(sel), out, scale=0.05)
    torch.cuda.synchronize()
    want, worst = _attend_reference(q, k_pool, v_pool, table, np.arange(3), pos, br, sel, 0.05, 0.0, out)
    _close(out, want, worst)


def test_attend_queries_of_any_size(ops):
    """|q| far beyond and far below fp16's range: the product with the keys is brought back by the scale or the keys."""
    kv, G, hd, br = 1, 4, 64, 16
    torch.manual_seed(4)
    v_pool = torch.randn(5, kv, br, hd, device="cuda").half()
    table, sel = np.array([[1, 2, 3, 4]], np.int32), np.arange(4, dtype=np.int32).reshape(1, 1, 4)
    for size, key_size, scale in ((1e6, 1.0, 1e-7), (1e20, 1.0, 1e-21), (1e-9, 1.0, 1e8), (3.0, 6e4, 1e-6), (1e-30, 1.0, 1e30), (1e-37, 1.0, 1e37), (1e37, 0.1, 1e-36), (0.0, 1.0, 1.0)):
        k_pool = (torch.randn(5, kv, br, hd, device="cuda") * key_size).clamp(-65000, 65000).half()
        q = torch.randn(1, kv * G * hd, device="cuda") * size
        cache, packed = _views(ops, table, [0], [60], br, 5, k_pool, v_pool)
        out = torch.empty(1, kv * G * hd, device="cuda")
        cache.attend(packed, q, dev(sel), out, scale=scale)
        torch.cuda.synchronize()
        want, worst = _attend_reference(q, k_pool, v_pool, table, [0], [60], br, sel, float(np.float32(scale)), 0.0, out)
        _close(out, want, worst)


def test_attend_softcap_from_the_smallest_to_the_largest_scores(ops):
    """Sixteen keys of score x against one of score 0: the weights are 16 / (16 + exp(-c)) and the rest, c = cap * tanh(x / cap).
    tanh is held to 2^-21 of its value, a weight to that of c plus 2^-21 each for exp, the split into two halves and the sums."""
    hd, br, cap = 64, 16, 8.0
    x = torch.cat((torch.logspace(-6, 4, 26, dtype=torch.float64), torch.tensor([0.55, 0.5999, 0.6, 0.6001, 0.7]).double() * cap))
    x = torch.cat((x, -x)).cuda().half()
    n = len(x)
    k_pool = torch.zeros(n + 2, 1, br, hd, dtype=torch.float16, device="cuda")
    v_pool = torch.zeros_like(k_pool)
    k_pool[1:n + 1, 0, :, 0] = x[:, None]
    v_pool[1:n + 1, 0, :, 0], v_pool[n + 1, 0, :, 1] = 1.0, 1.0
    q = torch.zeros(n, hd, device="cuda")
    q[:, 0] = 1.0
    table = np.array([[i + 1, n + 1] for i in range(n)], np.int32)
    cache, packed = _views(ops, table, np.arange(n), np.full(n, br), br, n + 2, k_pool, v_pool)
    out = torch.empty(n, hd, device="cuda")
    cache.attend(packed, q, dev(np.tile(np.array([0, 1], np.int32), (n, 1, 1))), out, scale=1.0, softcap=cap)
    torch.cuda.synchronize()
    c = cap * torch.tanh(x.double() / cap)
    want = 16 / (16 + torch.exp(-c))
    bound = 2.0 ** -21 * c.abs() + 3 * 2.0 ** -21
    assert ((out[:, 0].double() - want).abs() <= bound * want).all()
    assert ((out[:, 1].double() - (1 - want)).abs() <= bound * (1 - want)).all()
    assert out[:, 2:].eq(0).all()


def test_attend_offsets_past_32_bits(ops):
    """A pool of more than 2^31 values: the last block lies 4 GB behind the first."""
    kv, G, hd, br = 8, 2, 128, 64
    n_blocks = 2**31 // (kv * br * hd) + 9
    pool = torch.empty(n_blocks, kv, br, hd, dtype=torch.float16, device="cuda")
    bounds = torch.zeros(n_blocks, kv, 2, hd, dtype=torch.float16, device="cuda")
    pages = [1, n_blocks - 1, n_blocks // 2, n_blocks - 2]
    pool[pages] = torch.randn(4, kv, br, hd, device="cuda").half()
    table, sel = np.array([pages], np.int32), np.tile(np.arange(4, dtype=np.int32), (1, kv, 1))
    cache, packed = _views(ops, table, [0], [4 * br - 1], br, n_blocks, pool, pool, bounds)
    from goinfer_b200.paged import PagedRows
    k = torch.randn(1, kv * hd, device="cuda")
    at = (n_blocks - 2) * br + br - 1
    cache.append(PagedRows(dev([0]), dev([4 * br - 1]), dev([at])), k, k)
    q, out = torch.randn(1, kv * G * hd, device="cuda"), torch.empty(1, kv * G * hd, device="cuda")
    cache.attend(packed, q, dev(sel), out)
    torch.cuda.synchronize()
    assert torch.equal(pool[n_blocks - 2, :, br - 1], k.reshape(kv, hd).half())
    assert torch.equal(bounds[n_blocks - 2, :, 1], pool[n_blocks - 2].amax(1))
    want, worst = _attend_reference(q, pool, pool, table, [0], [4 * br - 1], br, sel, hd ** -0.5, 0.0, out)
    _close(out, want, worst)


@pytest.mark.parametrize("rows,kv,G,hd,br,max_blocks,n", [(2, 2, 4, 128, 16, 700, 90), (70, 4, 8, 64, 32, 40, 20)])
def test_calls_give_the_same_bits_again(ops, rows, kv, G, hd, br, max_blocks, n):
    rng = np.random.default_rng(rows)
    torch.manual_seed(rows)
    n_blocks = 3000
    k_pool = torch.randn(n_blocks, kv, br, hd, device="cuda").half()
    v_pool = torch.randn(n_blocks, kv, br, hd, device="cuda").half()
    bounds = torch.stack((k_pool.amin(2), k_pool.amax(2)), 2).contiguous()
    table, slot, pos = _context(rng, rows, max_blocks, br, n_blocks)
    cache, packed = _views(ops, table, slot, pos, br, n_blocks, k_pool, v_pool, bounds)
    q = torch.randn(rows, kv * G, hd, device="cuda")  # heads as a dimension of their own, in q and in out
    results = []
    for _ in range(5):
        sel = torch.full((rows, kv, n), -1, dtype=torch.int32, device="cuda")
        out = torch.zeros_like(q)
        cache.select(packed, q, sel)
        cache.attend(packed, q, sel, out)
        results.append((sel, out))
    torch.cuda.synchronize()
    assert all(torch.equal(a, results[0][0]) and torch.equal(b, results[0][1]) for a, b in results)
    want, worst = _attend_reference(q.reshape(rows, -1), k_pool, v_pool, table, slot, pos, br, results[0][0].cpu().numpy(), hd ** -0.5, 0.0, out.reshape(rows, -1))
    _close(out.reshape(rows, -1), want, worst)


def test_the_last_sequences_are_retired_by_a_plan_without_rows(ops):
    p = Pool(ops, 3, 5, 20, 16, 0, np.random.default_rng(0))
    full = len(p.free)
    grown = Pool(ops, 3, 5, 20, 16, 90, np.random.default_rng(0))
    grown.plan([0, 0, 0], [20, 40, 30])
    for a, b in ((p.d[k], grown.d[k]) for k in p.d):
        a.copy_(b)
    p.table, p.blocks, p.free = grown.table.copy(), grown.blocks.copy(), list(grown.free)
    assert p.plan([20, 0, 30], [0, 0, 0]) == 0 and p.plan([0, 0, 0], [0, 0, 0]) == 0 and len(p.free) == full
    assert p.plan([0, 0, 0], [1, 0, 0]) == 3  # a row, and no room for it


def test_refused_calls_queue_nothing_and_the_device_stays(ops):
    from goinfer_b200.resident import ResidentError
    cache, packed = _views(ops, np.ones((2, 4), np.int32), [0, 1], [3, 60], 16, 9, torch.zeros(9, 2, 16, 64, dtype=torch.float16, device="cuda"),
                           torch.zeros(9, 2, 16, 64, dtype=torch.float16, device="cuda"))
    q, sel, out = torch.randn(2, 256, device="cuda"), torch.zeros(2, 2, 4, dtype=torch.int32, device="cuda"), torch.full((2, 256), 5.0, device="cuda")
    before, device = ops.launch_count(), torch.cuda.current_device()
    for f in (lambda: cache.attend(packed, q, sel, out, softcap=-1.0), lambda: cache.select(packed, q, sel), lambda: cache.attend(packed, q[:, :250], sel, out),
              lambda: cache.append(packed, q[:, :128], q[:, 128:]), lambda: cache.attend(packed, q.cpu(), sel, out)):
        with pytest.raises(ResidentError) as e:
            f()
        assert e.value.status == abi.BAD_ARGUMENT
    torch.cuda.synchronize()
    assert ops.launch_count() == before and out.eq(5).all()
    cache.attend(packed, q, sel, out)
    torch.cuda.synchronize()
    assert ops.launch_count() == before + 1 and torch.cuda.current_device() == device and out.eq(0).all()


class Step:
    """Four operators as a decode step runs them, on a stream of its own."""

    def __init__(self, seed, n_seqs=6, kv=2, G=4, hd=128, br=16, max_blocks=40, n=10, n_rows=50):
        from goinfer_b200.ops import Ops
        self.stream = torch.cuda.Stream()
        self.ops = Ops(0, stream=self.stream.cuda_stream)
        self.rng = np.random.default_rng(seed)
        self.shape = (n_seqs, kv, G, hd, br, max_blocks, n, n_rows)
        n_blocks = n_seqs * max_blocks + 1
        f16 = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")  # noqa: E731
        self.k, self.v, self.b = f16(n_blocks, kv, br, hd), f16(n_blocks, kv, br, hd), f16(n_blocks, kv, 2, hd)
        self.p = Pool(self.ops, n_seqs, max_blocks, n_blocks, br, n_rows, self.rng, k_pool=self.k, v_pool=self.v, key_bounds=self.b)
        self.len, self.new = dev(np.zeros(n_seqs)), dev(np.zeros(n_seqs))
        self.x = torch.zeros(n_rows, (G + 2) * kv * hd, device="cuda")  # q | k | v of a row
        self.sel = torch.zeros(n_rows, kv, n, dtype=torch.int32, device="cuda")
        self.out = torch.zeros(n_rows, G * kv * hd, device="cuda")
        torch.cuda.synchronize()

    def call(self):
        _, kv, G, hd, *_ = self.shape
        c, w = self.p.cache, kv * hd
        c.plan(self.len, self.new, self.p.rows)
        c.append(self.p.rows, self.x[:, G * w:(G + 1) * w], self.x[:, (G + 1) * w:])
        c.select(self.p.rows, self.x[:, :G * w], self.sel)
        c.attend(self.p.rows, self.x[:, :G * w], self.sel, self.out)

    def capture(self):
        self.call()  # nothing to set up, but a program warms up
        self.stream.synchronize()
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self.stream):
            self.call()

    def feed(self, length, new, x):
        self.len.copy_(dev(length))
        self.new.copy_(dev(new))
        self.x.copy_(x)
        torch.cuda.synchronize()


def _run(step, seed, replay, rounds=7):
    n_seqs, kv, G, hd, br, max_blocks, n, n_rows = step.shape
    rng = np.random.default_rng(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    length, results = np.zeros(n_seqs, np.int64), []
    keys = {}  # what each sequence holds: position -> (k row, v row)
    for i in range(rounds):
        new = rng.integers(0, n_rows // n_seqs + 1, n_seqs)
        if i == 3:
            length[0], length[1] = 0, max(0, length[1] - 5)  # one sequence ends, one is rewound
        if i == 5:
            new[:] = n_rows                                     # too many rows: the step does nothing
        x = torch.randn(step.x.shape, generator=gen, device="cuda")
        step.feed(length, new, x)
        step.out.fill_(3.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(step.stream):
            step.graph.replay() if replay else step.call()
        step.stream.synchronize()
        results.append((step.out.clone(), step.sel.clone(), step.p.r["status"].clone()))
        if i == 5:
            assert step.p.r["status"][0].item() == 3 and step.out.eq(3).all()
            continue
        r, w = 0, kv * hd
        for s in range(n_seqs):
            for pos in range(length[s], length[s] + new[s]):
                keys[s, pos] = (x[r, G * w:(G + 1) * w].half().double(), x[r, (G + 1) * w:].half().double())
                r += 1
        # every row against the keys it selected, out of what was stored for its sequence
        r = 0
        for s in range(n_seqs):
            for pos in range(length[s], length[s] + new[s]):
                for h in range(kv):
                    blocks = [b for b in step.sel[r, h].tolist() if b >= 0]
                    assert blocks == sorted(set(blocks)) and blocks[-1] == pos // br and len(blocks) == min(n, pos // br + 1)
                    at = [p for b in blocks for p in range(b * br, min((b + 1) * br, pos + 1))]
                    k = torch.stack([keys[s, p][0].reshape(kv, hd)[h] for p in at])
                    v = torch.stack([keys[s, p][1].reshape(kv, hd)[h] for p in at])
                    qh = x[r, :G * w].double().reshape(kv, G, hd)[h]
                    o = torch.softmax(qh @ k.T * hd ** -0.5, -1) @ v
                    _close(step.out[r].reshape(kv, G, hd)[h], o, (qh.abs() @ k.abs().T * hd ** -0.5).max().item())
                r += 1
        assert step.out[r:].eq(3).all()
        length = length + new
    return results


@pytest.mark.parametrize("replay", [False, True])
def test_the_four_operators_as_a_decode_step(ops, replay):
    step = Step(1, max_blocks=12, n=3)
    if replay:
        step.capture()
    _run(step, 11, replay)


def test_the_first_call_of_a_process_may_be_captured(tmp_path):
    """Whatever a kernel asks of the device once (limits, how many clusters fit) is allowed while a stream captures."""
    prog = tmp_path / "first.py"
    prog.write_text("""
import torch
from goinfer_b200.ops import Ops
from goinfer_b200.paged import PagedCache, PagedRows
rows, kv, G, hd, br, n = 20, 4, 2, 64, 16, 32
side = torch.cuda.Stream()
ops = Ops(0, stream=side.cuda_stream)
i32 = dict(dtype=torch.int32, device="cuda")
k, v = (torch.randn(rows * n + 1, kv, br, hd, device="cuda").half() for _ in range(2))
bounds = torch.zeros(rows * n + 1, kv, 2, hd, dtype=torch.float16, device="cuda")
table = torch.arange(1, rows * n + 1, **i32).reshape(rows, n)
packed = PagedRows(torch.arange(rows, **i32), torch.full((rows,), n * br - 1, **i32), torch.zeros(rows, **i32))
cache = PagedCache(ops, table, torch.full((rows,), n, **i32), torch.zeros(rows * n + 1, **i32), torch.zeros(1, **i32), br, k, v, bounds)
q, sel = torch.randn(rows, kv * G * hd, device="cuda"), torch.empty(rows, kv, n, **i32)
outs = [torch.zeros(rows, kv * G * hd, device="cuda") for _ in range(2)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    cache.select(packed, q, sel, n_first=1, n_recent=1)
    cache.attend(packed, q, sel, outs[0])
graph.replay()
torch.cuda.synchronize()
with torch.cuda.stream(side):
    cache.attend(packed, q, sel, outs[1])
torch.cuda.synchronize()
assert outs[0].abs().sum() > 0 and torch.equal(outs[0], outs[1])
""")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, str(prog)], env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


def test_two_captured_steps_at_once_share_nothing(ops):
    """Two steps' graphs replayed on two streams without an order between them give what each gives alone, bit for bit."""
    alone = []
    for seed in (1, 2):
        s = Step(seed, max_blocks=30)
        s.capture()
        alone.append(_run(s, 20 + seed, True, 3))
    steps = [Step(seed, max_blocks=30) for seed in (1, 2)]
    for s in steps:
        s.capture()
    rngs = [np.random.default_rng(20 + seed) for seed in (1, 2)]
    gens = [torch.Generator("cuda").manual_seed(20 + seed) for seed in (1, 2)]
    lengths = [np.zeros(6, np.int64) for _ in steps]
    for i in range(3):
        for s, rng, gen, length in zip(steps, rngs, gens, lengths):
            new = rng.integers(0, 50 // 6 + 1, 6)
            s.feed(length, new, torch.randn(s.x.shape, generator=gen, device="cuda"))
            s.out.fill_(3.0)
            length += new
        torch.cuda.synchronize()
        for _ in range(20):  # the same step again writes the same rows
            for s in steps:
                with torch.cuda.stream(s.stream):
                    s.graph.replay()
        torch.cuda.synchronize()
        for s, a in zip(steps, alone):
            assert torch.equal(s.out, a[i][0]) and torch.equal(s.sel, a[i][1])


def test_a_full_list_gives_dense_attention(ops):
    """Every block named: the result of b200_attention_noalloc on the same pools."""
    rows, kv, G, hd, br, max_blocks = 9, 4, 2, 128, 16, 50
    rng = np.random.default_rng(8)
    torch.manual_seed(8)
    n_blocks = rows * max_blocks + 1
    k_pool = torch.randn(n_blocks, kv, br, hd, device="cuda").half()
    v_pool = torch.randn(n_blocks, kv, br, hd, device="cuda").half()
    table = (rng.permutation(n_blocks - 1) + 1).reshape(rows, max_blocks).astype(np.int32)
    slot, pos = rng.permutation(rows).astype(np.int32), rng.integers(0, max_blocks * br, rows).astype(np.int32)
    q = torch.randn(rows, kv * G * hd, device="cuda")
    bounds = torch.stack((k_pool.amin(2), k_pool.amax(2)), 2).contiguous()
    cache, packed = _views(ops, table, slot, pos, br, n_blocks, k_pool, v_pool, bounds)
    sel = torch.empty(rows, kv, max_blocks, dtype=torch.int32, device="cuda")
    out, dense = torch.empty_like(q), torch.empty_like(q)
    launches = ops.launch_count()
    cache.select(packed, q, sel)
    cache.attend(packed, q, sel, out)
    assert ops.launch_count() == launches + 2
    dt, ds, dp = dev(table), dev(slot), dev(pos)
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    assert ops.lib.b200_attention_noalloc(ops.ctx, p(q), kv * G * hd, rows, kv * G, kv, hd, C.c_float(0), C.c_float(0), p(ds), p(dp), max_blocks * br, p(k_pool),
                                          p(v_pool), p(dt), max_blocks, br, p(dense)) == abi.OK
    torch.cuda.synchronize()
    x = (q.reshape(rows, kv, G, hd).abs().amax() * hd * k_pool.abs().amax().float() * hd ** -0.5).item()
    _close(out, dense.double(), min(x, math.sqrt(hd) * 1.0))


def test_the_documented_step_runs():
    """The step of the integration guide, as it stands there, over two steps of eight sequences."""
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    code = text[text.index("import torch\nfrom goinfer_b200.ops import Ops\nfrom goinfer_b200.paged"):]
    setup, step = code[:code.index("```")].split("layers[0].plan", 1)
    env = {}
    exec(setup, env)
    length = torch.zeros(8, dtype=torch.int32, device="cuda")
    for new in ([5, 0, 17, 1, 2, 3, 4, 8], [1, 1, 1, 1, 1, 1, 1, 1]):
        env.update(kv_len=length, n_new=dev(new), k=torch.randn(64, 8, 128, device="cuda"), v=torch.randn(64, 8, 128, device="cuda"),
                   q=torch.randn(64, 32, 128, device="cuda"))
        exec("layers[0].plan" + step, env)
        torch.cuda.synchronize()
        assert env["rows"].status.tolist()[:2] == [0, sum(new)]
        length = length + dev(new)
    # a sequence's second step sees what the first stored, in both layers' pools
    r, cache = 2, env["layers"][1]
    keys = cache._keep[4][env["table"][2, :2].long()].transpose(1, 2).reshape(32, 8, 128)[:18]
    values = cache._keep[5][env["table"][2, :2].long()].transpose(1, 2).reshape(32, 8, 128)[:18]
    x = torch.einsum("hgd,khd->hgk", env["q"][r].double().reshape(8, 4, 128), keys.double()) * 128 ** -0.5
    want = torch.einsum("hgk,khd->hgd", torch.softmax(x, -1), values.double()).reshape(32, 128)
    _close(env["out"][r], want, torch.einsum("hgd,khd->hgk", env["q"][r].double().reshape(8, 4, 128).abs(), keys.double().abs()).max().item() * 128 ** -0.5)


def test_the_microbenchmark_runs(capsys, monkeypatch):
    import json
    import sys
    from goinfer_b200 import microbench
    monkeypatch.setattr(sys, "argv", "microbench paged --rows 5 --ctx-lo 40 --ctx-hi 900 --heads 8 --kv-heads 2 --head-dim 64 --select 9 --iters 2".split())
    microbench.main()
    lines = [json.loads(line) for line in capsys.readouterr().out.splitlines()]
    assert [x["kernel"] for x in lines] == ["paged plan", "paged append", "paged select", "paged attend"]
    assert all(x["plan_status"][:2] == [0, 5] and x["ms_per_launch"] > 0 for x in lines)
