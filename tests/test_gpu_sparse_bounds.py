"""Key bounds of cache blocks and the append that keeps them, against tests/sparse_ref.py: equal, element by element."""
import numpy as np
import pytest
import torch

import sparse_ref as S
from gpu_util import RawStream, log_case
from rllm_amd import FP8_ROUND_NEAREST_EVEN, FP8_ROUND_TOWARD_ZERO, ops

pytestmark = pytest.mark.gpu


def cache(rng, nb, hkv, d, bs, kv):
    return S.store(torch.from_numpy(rng.standard_normal((nb, hkv, d, bs)).astype(np.float32)) * 2, kv)


@pytest.mark.parametrize("kv", ["bf16", "f16", "e4m3", "e5m2"])
@pytest.mark.parametrize("hkv,d,bs", [(1, 32, 16), (8, 128, 16), (3, 96, 32), (5, 64, 64), (2, 256, 128), (4, 160, 16)])
def test_bounds(dev, kv, hkv, d, bs):
    rng = np.random.default_rng(d + bs)
    lens = [0, 1, bs - 1, bs, bs + 1, 5 * bs + 7, 3 * bs, -4]
    bt, nb = S.tables(rng, lens, bs, width=6)
    bt[5, 1], bt[5, 2], bt[6, 0] = -1, nb, nb + 1000          # unused entries
    kc = cache(rng, nb, hkv, d, bs, kv)
    raw = S.values(kc, kv)
    raw[torch.from_numpy(rng.random(raw.shape) < 0.1)] = 0
    raw = torch.where(torch.from_numpy(rng.random(raw.shape) < 0.05), -0.0, raw)
    for s, L in enumerate(lens):                               # rows behind the last key hold what was there before
        if L > 0 and L % bs and 0 <= bt[s, L // bs] < nb:
            raw[int(bt[s, L // bs]), :, :, L % bs:] = float("nan")
    kc = S.store(raw.float(), kv)
    before = S.store(torch.full((nb, hkv, 2, d), 5.0), kv)
    kb, kct = before.to(dev), kc.to(dev)
    log_case(f"bounds hkv={hkv} d={d} bs={bs} {kv}")
    lt = torch.tensor(lens, dtype=torch.int32, device=dev)
    assert ops.key_bounds(kct, kb, bt.to(dev), lt, validate=False, **S.fp8(kv)) is kb
    ref = S.bounds(S.values(before, kv), S.values(kc, kv), bt, lens, bs)
    assert S.same_values(S.values(kb, kv), ref)
    assert torch.equal(kct.cpu().view(torch.uint8), kc.view(torch.uint8))
    # from a position on
    first = [0, 0, 0, bs, bs, 2 * bs + 3, 9 * bs, 0]
    kb = before.to(dev)
    ops.key_bounds(kct, kb, bt.to(dev), lt, first_positions=torch.tensor(first, dtype=torch.int32, device=dev),
                   validate=False, **S.fp8(kv))
    assert S.same_values(S.values(kb, kv), S.bounds(S.values(before, kv), S.values(kc, kv), bt, lens, bs, first))


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_bounds_keep_nan_and_infinities(dev, kv):
    rng = np.random.default_rng(8)
    kc = S.values(cache(rng, 3, 2, 64, 16, kv), kv)
    kc[0, 0, 3, 5], kc[1, 1, 7, 2] = float("nan"), -float("nan")
    if kv == "bf16":
        kc[2, 0, 9, 1], kc[2, 0, 10, 1] = float("inf"), -float("inf")
    kc = S.store(kc.float(), kv)
    kb = ops.new_key_bounds(kc.to(dev))
    ops.key_bounds(kc.to(dev), kb, torch.tensor([[0, 1, 2]], dtype=torch.int32, device=dev),
                   torch.tensor([48], dtype=torch.int32, device=dev), **S.fp8(kv))
    got = S.values(kb, kv)
    assert got[0, 0, :, 3].isnan().any() and got[1, 1, :, 7].isnan().any()
    rest = S.bounds(S.values(kb, kv), S.values(kc, kv), torch.tensor([[0, 1, 2]]), [48], 16)
    ok = ~rest.isnan().any(2, keepdim=True).expand_as(rest)
    assert torch.equal(got[ok], rest[ok])


def test_many_blocks_of_wide_tables(dev):
    # more table entries than workgroups, most of them unused
    rng = np.random.default_rng(3)
    lens = [16 * 900 + 3] + [5] * 29
    bt, nb = S.tables(rng, lens, 16, width=1000)
    kc = cache(rng, nb, 1, 32, 16, "bf16")
    kb = ops.new_key_bounds(kc.to(dev))
    ops.key_bounds(kc.to(dev), kb, bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev))
    assert torch.equal(S.values(kb, "bf16"), S.bounds(torch.zeros(kb.shape).double(), S.values(kc, "bf16"), bt, lens, 16))


def test_bounds_move_with_their_blocks(dev):
    rng = np.random.default_rng(5)
    kc, vc = (cache(rng, 6, 2, 64, 16, "bf16").to(dev) for _ in range(2))
    kb = ops.new_key_bounds(kc)
    bt = torch.tensor([[4, 1]], dtype=torch.int32, device=dev)
    ops.key_bounds(kc, kb, bt, torch.tensor([32], dtype=torch.int32, device=dev))
    pairs = torch.tensor([[4, 0], [1, 5]], dtype=torch.int64, device=dev)
    ops.copy_blocks([kc], [vc], pairs)
    # a bounds array is moved as a cache of its own
    ops.copy_blocks([kb], [kb.clone()], pairs)
    fresh = ops.new_key_bounds(kc)
    ops.key_bounds(kc, fresh, torch.tensor([[0, 5]], dtype=torch.int32, device=dev),
                   torch.tensor([32], dtype=torch.int32, device=dev))
    assert torch.equal(kb[[0, 5]], fresh[[0, 5]])


def state(rng, lens, new, hq, hkv, d, bs, kind, kv, qsl_tail=0, width=0):
    """Caches with old tokens and their bounds, new tokens' q, k, v, and tables for both."""
    total = [a + b for a, b in zip(lens, new)]
    bt, nb = S.tables(rng, total, bs, width=width)
    kc, vc = cache(rng, nb, hkv, d, bs, kv), cache(rng, nb, hkv, d, bs, kv)
    kb = S.values(S.store(torch.full((nb, hkv, 2, d), 9.0), kv), kv)      # of no block yet, as the type holds it
    kb = S.bounds(kb, S.values(kc, kv), bt, lens, bs)
    n = sum(new) + qsl_tail
    q, k, v = (torch.from_numpy(rng.standard_normal((n, h, d)).astype(np.float32)).to(S.HALF[kind]) for h in (hq, hkv, hkv))
    return total, bt, kc, vc, kb, q, k, v


def run_append(dev, total, bt, kc, vc, kb, q, k, v, qsl, cos, sin, kv, in_place=False, scales=(1.0, 1.0), nearest=False):
    t = [x.to(dev) for x in (kc, vc, S.store(kb.float(), kv))]
    qd = q.to(dev)
    q_out = qd if in_place else torch.full_like(qd, 3.0)
    kw = dict(k_scale=scales[0], v_scale=scales[1], **S.fp8(kv)) if kv in S.FP8 else {}
    got = ops.rope_and_append(qd, k.to(dev), v.to(dev), *t, bt.to(dev), torch.tensor(total, dtype=torch.int32, device=dev),
                              cos.to(dev), sin.to(dev), q_out=q_out, validate=False,
                              query_start_loc=None if qsl is None else torch.tensor(qsl, dtype=torch.int32, device=dev),
                              fp8_rounding=FP8_ROUND_NEAREST_EVEN if nearest else FP8_ROUND_TOWARD_ZERO, **kw)
    assert got is q_out
    torch.cuda.synchronize()
    return q_out.cpu(), [x.cpu() for x in t]


def check_append(dev, total, bt, kc, vc, kb, q, k, v, qsl, cos, sin, kv, **kw):
    got_q, (gk, gv, gb) = run_append(dev, total, bt, kc, vc, kb, q, k, v, qsl, cos, sin, kv, **kw)
    scales, nearest = kw.get("scales", (1.0, 1.0)), kw.get("nearest", False)
    rk, rv, rb = kc.clone(), vc.clone(), kb.clone()
    ref_q = S.append(q, k, v, rk, rv, rb, bt, total, qsl, cos, sin, kv, *scales, nearest)
    have = [t for t, _, _ in S.rows(total, qsl, q.shape[0])]
    left = [t for t in range(q.shape[0]) if t not in have]
    assert torch.equal(got_q[have].view(torch.int16), ref_q[have].view(torch.int16))
    if left:
        assert torch.equal(got_q[left], q[left] if kw.get("in_place") else torch.full_like(q[left], 3.0))
    assert torch.equal(gk.view(torch.uint8), rk.view(torch.uint8)) and torch.equal(gv.view(torch.uint8), rv.view(torch.uint8))
    assert S.same_values(S.values(gb, kv), rb)


@pytest.mark.parametrize("kind,kv", S.TYPES)
@pytest.mark.parametrize("hq,hkv,d,bs", [(4, 1, 32, 16), (32, 8, 128, 16), (6, 3, 96, 32), (2, 2, 256, 64), (5, 5, 224, 128)])
def test_append_a_token_a_sequence(dev, kind, kv, hq, hkv, d, bs):
    rng = np.random.default_rng(d * 7 + bs)
    cos, sin = ops.rope_cache_tables(700, d, 10000.0)
    lens = [0, 1, bs - 1, bs, bs + 1, 3 * bs + 5, 2 * bs - 1] + rng.integers(0, 4 * bs, 14).tolist()
    st = state(rng, lens, [1] * len(lens), hq, hkv, d, bs, kind, kv)
    log_case(f"append d={d} bs={bs} {kind} {kv}")
    check_append(dev, *st, None, cos, sin, kv, scales=(0.37, 0.25))
    check_append(dev, *st, None, cos, sin, kv, scales=(0.37, 0.25), nearest=True, in_place=True)


@pytest.mark.parametrize("kind,kv", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e5m2")])
@pytest.mark.parametrize("hq,hkv,d,bs", [(4, 2, 64, 16), (8, 2, 128, 32), (3, 1, 256, 64), (2, 2, 192, 128)])
def test_append_chunks(dev, kind, kv, hq, hkv, d, bs):
    """Runs that start and end anywhere in a block, of none, one and many tokens, across the 16-token groups of the list;
    rows before the first sequence's and behind the last one's."""
    rng = np.random.default_rng(d + 3 * bs)
    cos, sin = ops.rope_cache_tables(1000, d, 10000.0)
    lens = [0, 5, 0, bs, 2 * bs - 3, 16, 7]
    new = [3, 2 * bs + 9, 0, 1, 5, bs, 40]
    total, bt, kc, vc, kb, q, k, v = state(rng, lens, new, hq, hkv, d, bs, kind, kv, qsl_tail=9)
    qsl = (4 + np.concatenate([[0], np.cumsum(new)])).tolist()
    log_case(f"append chunk d={d} bs={bs} {kind} {kv}")
    check_append(dev, total, bt, kc, vc, kb, q, k, v, qsl, cos, sin, kv)
    qsl = (np.concatenate([[0], np.cumsum(new)])).tolist()
    check_append(dev, total, bt, kc, vc, kb, q, k, v, qsl, cos, sin, kv, scales=(2.0, 0.7), nearest=True)


def test_append_padding_holes_and_limits(dev):
    rng = np.random.default_rng(77)
    cos, sin = ops.rope_cache_tables(50, 64, 10000.0)          # fewer positions than tokens: clamped
    lens, new = [10, 60, 0, 30, 20], [30, 20, 4, 6, 1]
    total, bt, kc, vc, kb, q, k, v = state(rng, lens, new, 4, 2, 64, 16, "bf16", "bf16")
    qsl = np.concatenate([[0], np.cumsum(new)]).tolist()
    bt[0, 1], bt[1, 4], bt[3, 2] = -1, kc.shape[0], 1 << 30    # tokens without a block
    check_append(dev, total, bt, kc, vc, kb, q, k, v, qsl, cos, sin, "bf16")
    total[2], total[3] = 2, 3                                   # more new tokens than the length: the first ones have no place
    check_append(dev, total, bt, kc, vc, kb, q, k, v, qsl, cos, sin, "bf16")
    total[1], total[4] = 0, -5
    check_append(dev, total, bt, kc, vc, kb, q, k, v, qsl, cos, sin, "bf16")
    check_append(dev, total, bt[:, :2].contiguous(), kc, vc, kb, q, k, v, qsl, cos, sin, "bf16")   # tokens past the table
    # a padded decode batch
    check_append(dev, [17, 0, 0, 33, 1], bt, kc, vc, kb, q[:5], k[:5], v[:5], None, cos, sin, "bf16")


def test_append_without_q_and_step_by_step(dev):
    """Chunks and single tokens lead to the caches and bounds of one chunk, and those to key_bounds'."""
    rng = np.random.default_rng(12)
    cos, sin = (x.to(dev) for x in ops.rope_cache_tables(300, 128, 10000.0))
    T = 150
    bt, nb = S.tables(rng, [T], 32)
    bt = bt.to(dev)
    k, v = (torch.from_numpy(rng.standard_normal((T, 4, 128)).astype(np.float32)).to(torch.float16).to(dev) for _ in range(2))
    ends = [[T], [1, 2, 15, 16, 17, 40, 64, 101, 102, T], list(range(1, T + 1))]
    got = []
    for cut in ends:
        kc, vc = (torch.full((nb, 4, 128, 32), 7.0, dtype=torch.float16, device=dev) for _ in range(2))
        kb = ops.new_key_bounds(kc)
        a = 0
        for e in cut:
            qsl = torch.tensor([0, e - a], dtype=torch.int32, device=dev)
            assert ops.rope_and_append(None, k[a:e], v[a:e], kc, vc, kb, bt, torch.tensor([e], dtype=torch.int32, device=dev),
                                       cos, sin, query_start_loc=qsl) is None
            a = e
        fresh = ops.new_key_bounds(kc)
        ops.key_bounds(kc, fresh, bt, torch.tensor([T], dtype=torch.int32, device=dev))
        assert torch.equal(fresh, kb)
        got.append((kc, vc, kb))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("kv", ["e4m3", "e5m2"])
@pytest.mark.parametrize("scale", [1.0, 0.37, 2.0 ** -7])
def test_every_16_bit_value_into_an_fp8_cache(dev, kind, kv, scale):
    """All 65536 patterns as values, in both roundings; as keys unrotated (position 0)."""
    x = torch.from_numpy(np.arange(65536, dtype=np.uint16).view(np.int16)).view(S.HALF[kind]).view(2048, 1, 32)
    cos, sin = ops.rope_cache_tables(4, 32, 10000.0)
    for nearest in (True, False):
        n = 2048
        bt = torch.arange(n, dtype=torch.int32)[:, None]        # a block for each token, the first of its sequence
        kc, vc = (torch.full((n, 1, 32, 16), 9, dtype=torch.uint8, device=dev) for _ in range(2))
        kb = ops.new_key_bounds(kc)
        ops.rope_and_append(None, x.to(dev), x.to(dev), kc, vc, kb, bt.to(dev), torch.ones(n, dtype=torch.int32, device=dev),
                            cos.to(dev), sin.to(dev), k_scale=scale, v_scale=scale, validate=False, **S.fp8(kv),
                            fp8_rounding=FP8_ROUND_NEAREST_EVEN if nearest else FP8_ROUND_TOWARD_ZERO)
        want = S.encode(x.float(), kv, scale, nearest)[:, 0]
        assert torch.equal(vc[:, 0, :, 0].cpu(), want)
        # rotation by 0 leaves a finite pair as it is, but for the sign of zeros
        fine = torch.isfinite(x.float().view(n, 2, 16)).all(1).repeat(1, 2)
        got, k = kc[:, 0, :, 0].cpu(), want.clone()
        k[(k & 0x7F) == 0], got[(got & 0x7F) == 0] = 0, 0
        assert torch.equal(got[fine], k[fine])


def test_append_on_a_stream_and_replayed(dev):
    rng = np.random.default_rng(9)
    cos, sin = ops.rope_cache_tables(300, 64, 10000.0)
    lens = rng.integers(0, 90, 40).tolist()
    total, bt, kc, vc, kb, q, k, v = state(rng, lens, [1] * 40, 4, 2, 64, 16, "bf16", "bf16")
    want_q, want = run_append(dev, total, bt, kc, vc, kb, q, k, v, None, cos, sin, "bf16")
    d = [x.to(dev) for x in (q, k, v, kc, vc, kb.to(torch.bfloat16), bt, torch.tensor(total, dtype=torch.int32), cos, sin)]
    q_out = torch.zeros_like(d[0])
    start = [x.clone() for x in d[3:6]]
    with RawStream() as st:
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ops.rope_and_append(*d, q_out=q_out, validate=False)
        for _ in range(3):
            for x, s in zip(d[3:6], start):
                x.copy_(s)
            q_out.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(q_out.cpu(), want_q)
            assert all(torch.equal(x.cpu(), w) for x, w in zip(d[3:6], want))
