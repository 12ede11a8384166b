"""Chunks over selected blocks where their tiles of rows can go wrong: long lists, wide tables and long sequences, against the
formulas in 64 bits (tests/sparse_ref.py)."""
import numpy as np
import pytest
import torch

import sparse_ref as S
from gpu_util import log_case
from rllm_amd import ops
from test_gpu_sparse_select import check, key_like, queries

pytestmark = pytest.mark.gpu


def normal(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32))


@pytest.mark.parametrize("kind,kv,hq,hkv,d,k,width,n", [
    ("bf16", "bf16", 8, 2, 256, 1024, 32000, 520),      # the list leaves LDS for two waves, whose windows hold the blocks' bits
    ("bf16", "bf16", 8, 2, 256, 1024, 65000, 520),      # and do not
    ("f16", "e4m3", 4, 4, 256, 256, 40000, 1030),
    ("f16", "f16", 4, 4, 256, 201, 32896, 1030),        # the most that two waves hold, and one more
    ("f16", "f16", 4, 4, 256, 201, 32897, 1030),
    ("bf16", "e5m2", 4, 4, 32, 32, 8448, 1030),         # the same for four waves
    ("bf16", "bf16", 4, 4, 32, 32, 8449, 1030)])
def test_tiles_under_wide_tables(dev, kind, kv, hq, hkv, d, k, width, n):
    """A sequence as long as a wide table, most rows with a few of its blocks, some with lists as long as they may be that have
    little in common.  The table names few blocks again and again."""
    rng = np.random.default_rng(width + k)
    new = [n - 21, 17]
    lens = [16 * width - 3, 16 * 40 + 5]
    nb = 97
    bt = torch.from_numpy(rng.integers(0, nb, (2, width)).astype(np.int32))
    kc, vc = (S.store(normal(rng, nb, hkv, d, 16), kv) for _ in range(2))
    q = normal(rng, n, hq, d).to(S.HALF[kind])
    qsl = [2, 2 + new[0], 2 + sum(new)]
    sel = torch.full((n, hkv, k), -1, dtype=torch.int32)
    for t, s, pos in S.rows(lens, qsl, n):
        nv = pos // 16 + 1
        long = 34 <= t < 39 or t == qsl[1] - 1                   # rows of two tiles, and the longest row
        for h in range(hkv if not long else 1):
            m = min(nv, k if long else int(rng.integers(0, 7)))
            sel[t, h, :m] = torch.from_numpy(np.sort(rng.permutation(nv)[:m]).astype(np.int32))
            if m and rng.random() < 0.5:
                sel[t, h, m - 1] = nv - 1                        # the row's own block
    ks, vs = (0.5, 0.75) if kv in S.FP8 else (1.0, 1.0)
    ref, mag, spread = S.attend(q, S.values(kc, kv), S.values(vc, kv), bt, lens, qsl, sel, d ** -0.5, ks, vs)
    out = torch.full_like(q, 3.0).to(dev)
    log_case(f"attend rows={n} hq={hq} hkv={hkv} d={d} k={k} width={width} {kind} {kv}")
    kw = dict(k_scale=ks, v_scale=vs, **S.fp8(kv)) if kv in S.FP8 else {}
    ops.paged_sparse(q.to(dev), kc.to(dev), vc.to(dev), bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), sel.to(dev),
                     d ** -0.5, query_start_loc=torch.tensor(qsl, dtype=torch.int32, device=dev), out=out, **kw)
    S.check_attend(out, ref, mag, spread, kind, d, 16 * k)
    left = ref[:, 0, 0].isnan()
    assert (out.cpu()[left] == 3.0).all() and int(left.sum()) == n - sum(new)

# ---------------------------------------------------------------------------
# selection: rows of a chunk in tiles
# ---------------------------------------------------------------------------

GROUPS = [(2, 2), (4, 2), (3, 1), (8, 2), (9, 1), (16, 1)]      # heads of a group: 1, 2, 3, 4, 9, 16


def chunks_of(rng, hq, hkv, blocks=70, bs=16):
    """Lengths and new tokens of two sequences, two tiles of rows at least each (64 * 4 (row, head) pairs a tile, heads of a group
    as a power of two); (lens, query_start_loc, rows, table, blocks in the pool)."""
    tile = 256 // (1 << (hq // hkv - 1).bit_length())
    new = [2 * tile + 3, tile + 1]
    lens = [max(blocks * bs, new[0]) - 2, blocks * bs // 2 + new[1]]
    bt, nb = S.tables(rng, lens, bs)
    return lens, [1, 1 + new[0], 1 + sum(new)], sum(new) + 4, bt, nb


def bounds_that_nearly_tie(rng, nb, hkv, d, kind):
    """Scores that differ by far less than an f32 sum's rounding: + 6400 - 6400 + a little, for queries as near_tie_queries has
    them."""
    kb = np.broadcast_to(rng.standard_normal(d) * 0.1, (nb, hkv, 2, d)).copy()
    kb[..., 0], kb[..., 1] = 100.0, -100.0
    kb[..., 2] = rng.permutation(nb)[:, None, None] * 2.0 ** -9
    return torch.from_numpy(kb).to(S.HALF[kind])


def near_tie_queries(rng, n, hq, d, kind):
    q = normal(rng, n, hq, d).to(S.HALF[kind])
    q[..., 0], q[..., 1], q[..., 2] = 64.0, 64.0, 2.0 ** -10
    return q


@pytest.mark.parametrize("hq,hkv", GROUPS)
def test_select_ties(dev, hq, hkv):
    rng = np.random.default_rng(hq)
    lens, qsl, n, bt, nb = chunks_of(rng, hq, hkv)
    q, kb = queries(rng, n, hq, 64, "bf16"), key_like(rng, nb, hkv, 64, "bf16")
    kb[bt[0, 5:60:3].long()] = kb[int(bt[0, 7])].clone()
    check(dev, q, kb, "bf16", bt, lens, 16, 9, 1, 1, qsl, what="some alike")
    check(dev, torch.zeros_like(q), kb, "bf16", bt, lens, 16, 9, 0, 1, qsl, what="zero queries")
    kb[:] = kb[3].clone()
    check(dev, q, kb, "bf16", bt, lens, 16, 9, 1, 2, qsl, what="all alike")
    check(dev, q, torch.zeros_like(kb), "bf16", bt, lens, 16, 9, 0, 1, qsl, what="zero bounds")


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv", GROUPS)
def test_select_scores_that_f32_cannot_tell_apart(dev, kind, hq, hkv):
    rng = np.random.default_rng(hq + 100)
    lens, qsl, n, bt, nb = chunks_of(rng, hq, hkv)
    q, kb = near_tie_queries(rng, n, hq, 64, kind), bounds_that_nearly_tie(rng, nb, hkv, 64, kind)
    for k in (3, 20, 50):
        check(dev, q, kb, kind, bt, lens, 16, k, 1, 1, qsl, what="near ties")
    # 250 blocks: more between the border's two sides than are scored again at once
    lens, qsl, n, bt, nb = chunks_of(rng, hq, hkv, 250)
    n = 60
    check(dev, near_tie_queries(rng, n, hq, 64, kind), bounds_that_nearly_tie(rng, nb, hkv, 64, kind), kind, bt[:1], lens[:1], 16, 99,
          1, 1, [1, 59], what="more near ties")


@pytest.mark.parametrize("hq,hkv", GROUPS)
def test_select_near_ties_before_a_block_that_is_not_finite(dev, hq, hkv):
    """NaN or an infinity in a block that only the last rows see (and that stands among the first candidates' 64 blocks): the rows
    before it are still the 64-bit scores'."""
    rng = np.random.default_rng(hq + 200)
    tile = 256 // (1 << (hq // hkv - 1).bit_length())
    new = max(2 * tile + 3, 16 * 16)
    lens, qsl, n = [max(62 * 16, new + 16 * 20) - 2, 500], [1, 1 + new, 1 + new + 40], new + 45
    bt, nb = S.tables(rng, lens, 16)
    q = near_tie_queries(rng, n, hq, 64, "bf16")
    late = (lens[0] - 1) // 16 - 2
    assert (lens[0] - new) // 16 + 8 < late < 64
    for bad in (float("nan"), -float("nan"), float("inf")):
        kb = bounds_that_nearly_tie(rng, nb, hkv, 64, "bf16")
        kb[int(bt[0, late]), :, 1, 9] = bad
        for k in (3, 12):
            check(dev, q, kb, "bf16", bt, lens, 16, k, 1, 1, qsl, what=f"a late {bad}")


@pytest.mark.parametrize("hq,hkv", GROUPS)
def test_select_values_that_are_not_finite(dev, hq, hkv):
    rng = np.random.default_rng(hq + 300)
    lens, qsl, n, bt, nb = chunks_of(rng, hq, hkv)
    kb = key_like(rng, nb, hkv, 64, "bf16")
    nan, inf = float("nan"), float("inf")
    kb[int(bt[0, 50]), :, 1, 5] = nan
    kb[int(bt[0, 20]), :, 0, 5] = nan
    kb[int(bt[0, 10]), :, 1, 7] = inf
    kb[int(bt[0, 11]), :, 0, 7] = -inf
    kb[int(bt[0, 12])], kb[int(bt[0, 13])] = inf, -inf
    q = queries(rng, n, hq, 64, "bf16")
    for k in (3, 6, 20):
        check(dev, q, kb, "bf16", bt, lens, 16, k, 1, 1, qsl, what="non-finite bounds")
    q[::3, hq - 1, 7] = 0.0
    q[1::7, 0, 9] = nan
    q[2::7, hq // 2, 9] = inf
    check(dev, q, kb, "bf16", bt, lens, 16, 6, 1, 1, qsl, what="non-finite queries")
    big = key_like(rng, nb, hkv, 64, "bf16") * 2.0 ** 126
    check(dev, queries(rng, n, hq, 64, "bf16") * 64, big, "bf16", bt, lens, 16, 20, 1, 1, qsl, what="scores past f32")


@pytest.mark.parametrize("hq,hkv", GROUPS)
@pytest.mark.parametrize("queries_by,bounds_by", [(-20, -120), (-40, -120), (-60, -100), (-126, -126), (60, -130), (-130, 100)])
def test_select_scores_below_f32(dev, hq, hkv, queries_by, bounds_by):
    """Scores below f32's range, subnormal bf16 queries and bounds: a chunk, and its last rows as decode rows."""
    rng = np.random.default_rng(hq + 400)
    lens, qsl, n, bt, nb = chunks_of(rng, hq, hkv)
    kb = key_like(rng, nb, hkv, 64, "bf16") * 2.0 ** bounds_by
    q = queries(rng, n, hq, 64, "bf16") * 2.0 ** queries_by
    assert bool(kb.any()) and bool(q.any())
    check(dev, q, kb, "bf16", bt, lens, 16, 10, 1, 1, qsl, what=f"2^{queries_by} by 2^{bounds_by}")
    check(dev, q[:2], kb, "bf16", bt, lens, 16, 10, 1, 1, what=f"2^{queries_by} by 2^{bounds_by}, a row a sequence")


@pytest.mark.parametrize("hq,hkv", GROUPS)
def test_select_f16_and_e5m2_subnormals(dev, hq, hkv):
    rng = np.random.default_rng(hq + 500)
    lens, qsl, n, bt, nb = chunks_of(rng, hq, hkv)
    for kv in ("f16", "e5m2"):
        x = normal(rng, nb, hkv, 2, 64).sort(2).values * 2.0 ** -16
        q = queries(rng, n, hq, 64, "f16")
        check(dev, q, S.store(x, kv), kv, bt, lens, 16, 12, 1, 1, qsl, what="subnormal bounds")
        check(dev, q * 2.0 ** -14, S.store(x * 2.0 ** 17, kv), kv, bt, lens, 16, 12, 1, 1, qsl, what="subnormal queries")


@pytest.mark.parametrize("hq,hkv", GROUPS)
def test_select_unused_entries(dev, hq, hkv):
    rng = np.random.default_rng(hq + 600)
    lens, qsl, n, bt, nb = chunks_of(rng, hq, hkv)
    kb, q = key_like(rng, nb, hkv, 64, "bf16"), queries(rng, n, hq, 64, "bf16")
    bt[0, rng.permutation(70)[:50]] = -1
    bt[0, 3], bt[0, 40], bt[1, 0] = nb, 1 << 30, -7
    for k in (4, 9, 30):
        check(dev, q, kb, "bf16", bt, lens, 16, k, 2, 2, qsl)
    check(dev, q, kb, "bf16", bt[:, :25].contiguous(), lens, 16, 6, 1, 1, qsl, what="a table narrower than the lengths")


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (16, 1)])
def test_select_more_blocks_than_registers_hold(dev, hq, hkv):
    rng = np.random.default_rng(hq + 700)
    blocks, n = 8192 + 300, 40
    lens, qsl = [blocks * 16 - 3, 60], [0, n - 6, n - 4]
    bt, nb = S.tables(rng, lens, 16)
    q, kb = queries(rng, n, hq, 32, "bf16"), key_like(rng, nb, hkv, 32, "bf16")
    check(dev, q, kb, "bf16", bt, lens, 16, 100, 1, 2, qsl)
    check(dev, near_tie_queries(rng, n, hq, 32, "bf16"), bounds_that_nearly_tie(rng, nb, hkv, 32, "bf16"), "bf16", bt, lens, 16, 100, 1,
          2, qsl, what="near ties")
    kb[int(bt[0, 8200]), 0, 1, 3] = float("nan")
    check(dev, q, kb, "bf16", bt, lens, 16, 100, 1, 2, qsl, what="NaN")


def test_select_lists_of_one_wave_each(dev):
    """2048 lists and more, of up to 2047 blocks: every register of a lane."""
    rng = np.random.default_rng(800)
    hq, hkv, n = 8, 8, 262
    lens, qsl = [2047 * 16 - 1, 1000 * 16, 33], [0, 200, 258, 260]
    bt, nb = S.tables(rng, lens, 16)
    q, kb = queries(rng, n, hq, 32, "bf16"), key_like(rng, nb, hkv, 32, "bf16")
    check(dev, q, kb, "bf16", bt, lens, 16, 64, 1, 2, qsl)
    check(dev, near_tie_queries(rng, n, hq, 32, "bf16"), bounds_that_nearly_tie(rng, nb, hkv, 32, "bf16"), "bf16", bt, lens, 16, 64, 1,
          2, qsl, what="near ties")


@pytest.mark.parametrize("hq", [8, 24])
def test_select_near_ties_over_several_slabs(dev, hq):
    """Near ties and a late NaN in a call that works through its rows in parts: as under a narrow table, and by the formula."""
    rng = np.random.default_rng(hq + 900)
    hkv, width, new = 8, 16384, [901, 1, 1300, 40]
    lens = [1500, 2000, 1300, 900]
    small, nb = S.tables(rng, lens, 16)
    qsl = np.concatenate([[0], np.cumsum(new)]).tolist()
    n = qsl[-1]
    kb, q = bounds_that_nearly_tie(rng, nb, hkv, 32, "bf16"), near_tie_queries(rng, n, hq, 32, "bf16")
    kb[int(small[2, 60]), :, 1, 9] = float("nan")
    assert n * hkv * width * 4 > ops.lib().rllm_select_blocks_workspace_size(n, hkv, width)
    bt = torch.full((4, width), -1, dtype=torch.int32, device=dev)
    bt[:, :small.shape[1]] = small.to(dev)
    args = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (lens, qsl)]
    wide, narrow = (ops.select_blocks(q.to(dev), kb.to(dev), t, args[0], 16, 8, validate=False, query_start_loc=args[1]).cpu()
                    for t in (bt, small.to(dev)))
    assert torch.equal(wide, narrow)
    for t in list(range(0, n, 53)) + [900, 901, 902, 1524, 1525, 1526, 1527, n - 41, n - 1]:
        s = int(np.searchsorted(qsl, t, side="right")) - 1
        one = S.select(q[t:t + 1], S.values(kb, "bf16"), small[s:s + 1], [lens[s] - (qsl[s + 1] - 1 - t)], None, 16, 8, 1, 1)
        assert torch.equal(wide[t:t + 1], one), t


def test_select_more_lists_than_a_launch_has_threads_for(dev):
    """2^26 lists and some, under a table no wider than they are."""
    n, hkv = (1 << 23) + 3, 8
    q = torch.ones((n, hkv, 32), dtype=torch.bfloat16, device=dev)
    kb = torch.zeros((1, hkv, 2, 32), dtype=torch.bfloat16, device=dev)
    bt = torch.zeros((n, 1), dtype=torch.int32, device=dev)
    lens = torch.arange(n, dtype=torch.int32, device=dev) % 3       # 0, 1 and 2 keys
    out = torch.full((n, hkv, 1), -7, dtype=torch.int32, device=dev)
    log_case(f"select rows={n} hkv={hkv} d=32 width=1")
    ops.select_blocks(q, kb, bt, lens, 16, 1, num_first=0, out=out, validate=False)
    want = torch.where(lens > 0, 0, -1)
    assert bool((out[:, :, 0] == want[:, None]).all())
