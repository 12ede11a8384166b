"""Selected blocks against the scores in 64 bits (tests/sparse_ref.py): the same lists, ties to the lowest block."""
import threading

import numpy as np
import pytest
import torch

import sparse_ref as S
from gpu_util import RawStream, log_case
from rllm_amd import KernelError, ops

pytestmark = pytest.mark.gpu


def key_like(rng, nb, hkv, d, kv, width=1.0):
    lo = rng.standard_normal((nb, hkv, d)) * 1.5
    hi = lo + rng.random((nb, hkv, d)) * width
    return S.store(torch.from_numpy(np.stack((lo, hi), 2).astype(np.float32)), kv)


def queries(rng, n, hq, d, kind):
    return torch.from_numpy(rng.standard_normal((n, hq, d)).astype(np.float32)).to(S.HALF[kind])


def check(dev, q, kb, kv, bt, lens, bs, k, first=1, last=1, qsl=None, what="", **kw):
    n, hkv = q.shape[0], kb.shape[1]
    ref = S.select(q, S.values(kb, kv), bt, lens, qsl, bs, k, first, last)
    out = torch.full((n, hkv, k), -7, dtype=torch.int32, device=dev)
    log_case(f"select rows={n} hq={q.shape[1]} hkv={hkv} d={q.shape[2]} bs={bs} k={k} width={bt.shape[1]} {kv} {what}")
    qt = None if qsl is None else torch.tensor(qsl, dtype=torch.int32, device=dev)
    got = ops.select_blocks(q.to(dev), kb.to(dev), bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), bs, k,
                            num_first=first, num_last=last, query_start_loc=qt, out=out, validate=False, **S.fp8(kv), **kw)
    assert got is out
    assert torch.equal(out.cpu(), ref), what
    return out


@pytest.mark.parametrize("kind,kv", S.TYPES)
@pytest.mark.parametrize("hq,hkv,d,bs", [(4, 1, 32, 16), (32, 8, 128, 16), (6, 2, 96, 32), (20, 1, 64, 64), (48, 1, 160, 16),
                                         (2, 2, 256, 128), (7, 1, 192, 16), (16, 1, 224, 32)])
def test_decode_rows(dev, kind, kv, hq, hkv, d, bs):
    rng = np.random.default_rng(d + bs + hq)
    lens = [0, 1, bs, bs + 1, 9 * bs, 9 * bs + 1, 40 * bs - 3, 150 * bs, -2, 70 * bs + 1]
    bt, nb = S.tables(rng, lens, bs)
    kb = key_like(rng, nb, hkv, d, kv)
    q = queries(rng, len(lens), hq, d, kind)
    check(dev, q, kb, kv, bt, lens, bs, 9, 2, 3)
    check(dev, q, kb, kv, bt, lens, bs, 1, 0, 1)
    check(dev, q, kb, kv, bt, lens, bs, 64, 0, 2)
    check(dev, q, kb, kv, bt, lens, bs, 200, 1, 1)              # every list is the whole sequence


@pytest.mark.parametrize("kind,kv", [("bf16", "bf16"), ("f16", "f16"), ("f16", "e4m3")])
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 8, 128, 16), (6, 2, 64, 32), (20, 1, 96, 16), (2, 2, 256, 16), (5, 1, 32, 64),
                                         (4, 2, 160, 32), (16, 1, 224, 16), (9, 1, 192, 16)])
def test_chunk_rows(dev, kind, kv, hq, hkv, d, bs):
    rng = np.random.default_rng(d * 3 + hq)
    lens, new = [30 * bs + 5, 90 * bs, 17, 11 * bs + 1, 300], [1, 37, 17, 0, 9]
    bt, nb = S.tables(rng, lens, bs)
    kb = key_like(rng, nb, hkv, d, kv)
    qsl = (3 + np.concatenate([[0], np.cumsum(new)])).tolist()
    q = queries(rng, sum(new) + 8, hq, d, kind)
    check(dev, q, kb, kv, bt, lens, bs, 8, 1, 2, qsl)
    lens[2], lens[4] = 5, 0                                     # more rows than keys, and none
    check(dev, q, kb, kv, bt, lens, bs, 5, 0, 1, qsl)


def test_unused_entries_are_in_no_list(dev):
    rng = np.random.default_rng(4)
    lens = [60 * 16, 60 * 16 - 5, 6 * 16, 30 * 16]
    bt, nb = S.tables(rng, lens, 16)
    bt[0, rng.permutation(60)[:45]] = -1
    bt[1, 0], bt[1, 59], bt[1, 30] = nb, -3, 1 << 30
    bt[2, 2] = -1
    bt[3, :] = -1
    kb = key_like(rng, nb, 2, 64, "bf16")
    check(dev, queries(rng, 4, 8, 64, "bf16"), kb, "bf16", bt, lens, 16, 20, 2, 2)
    # a table narrower than the lengths
    check(dev, queries(rng, 4, 8, 64, "bf16"), kb, "bf16", bt[:, :40].contiguous(), lens, 16, 12, 1, 1)


@pytest.mark.parametrize("kind,kv", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e5m2")])
def test_ties_go_to_the_lowest_block(dev, kind, kv):
    rng = np.random.default_rng(6)
    lens = [100 * 16, 77 * 16 - 1, 100 * 16]
    bt, nb = S.tables(rng, lens, 16)
    kb = key_like(rng, nb, 2, 128, kv)
    q = queries(rng, 3, 8, 128, kind)
    base = kb[int(bt[0, 7])].clone()
    kb[bt[0, 10:90:3].long()] = base                            # 27 blocks of one score
    check(dev, q, kb, kv, bt, lens, 16, 15, 1, 1, what="some alike")
    kb[:] = base
    check(dev, q, kb, kv, bt, lens, 16, 15, 1, 1, what="all alike")
    check(dev, torch.zeros_like(q), key_like(rng, nb, 2, 128, kv), kv, bt, lens, 16, 15, 0, 1, what="zero queries")
    check(dev, q, torch.zeros_like(kb), kv, bt, lens, 16, 15, 0, 1, what="zero bounds")
    check(dev, q, -torch.zeros_like(kb) if kv in S.HALF else torch.full_like(kb, 0x80), kv, bt, lens, 16, 15, 0, 1)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_scores_that_f32_cannot_tell_apart(dev, kind):
    """Scores around the border that differ by far less than an f32 sum's rounding, in both halves of the 64-bit key, with large
    parts that cancel."""
    rng = np.random.default_rng(21)
    nb, d = 400, 128
    lens = [nb * 16]
    bt, _ = S.tables(rng, lens, 16, spare=0)
    q = queries(rng, 1, 4, d, kind)
    q[0, :, 0], q[0, :, 1], q[0, :, 2] = 64.0, 64.0, 2.0 ** -10
    base = rng.standard_normal(d) * 0.1
    kb = np.broadcast_to(base, (nb, 1, 2, d)).copy()
    kb[..., 0] = 100.0                                           # + 6400 - 6400 + a little
    kb[..., 1] = -100.0
    kb[..., 2] = rng.permutation(nb)[:, None, None] * 2.0 ** -9
    kb = torch.from_numpy(kb).to(S.HALF[kind])
    assert len(set(S.scores(q[0].double(), kb[:, 0].double()).tolist())) > 200
    for k in (3, 30, 77, 200):
        check(dev, q, kb, kind, bt, lens, 16, k, 1, 1, what="near ties")
    kb[:, :, :, 2] = (torch.arange(nb) % 2 * 2.0 ** -14)[:, None, None]
    check(dev, q, kb, kind, bt, lens, 16, 50, 1, 1, what="two values")


def test_values_that_are_not_finite(dev):
    rng = np.random.default_rng(31)
    lens = [90 * 16]
    bt, nb = S.tables(rng, lens, 16)
    kb = key_like(rng, nb, 1, 64, "bf16")
    nan, inf = float("nan"), float("inf")
    kb[int(bt[0, 50]), 0, 1, 5] = nan
    kb[int(bt[0, 20]), 0, 0, 5] = nan
    kb[int(bt[0, 30]), 0, 1, 7] = inf
    kb[int(bt[0, 31]), 0, 0, 7] = -inf
    kb[int(bt[0, 32]), 0] = inf
    kb[int(bt[0, 33]), 0] = -inf
    q = queries(rng, 1, 4, 64, "bf16")
    for k in (3, 5, 8, 40):
        check(dev, q, kb, "bf16", bt, lens, 16, k, 1, 1, what="non-finite bounds")
    q[0, 2, 7] = 0.0
    check(dev, q, kb, "bf16", bt, lens, 16, 6, 1, 1, what="zero times infinity")
    q[0, 1, 9] = nan
    check(dev, q, kb, "bf16", bt, lens, 16, 6, 1, 1, what="a query with NaN")
    q[0, 1, 9] = inf
    check(dev, q, kb, "bf16", bt, lens, 16, 6, 1, 1, what="an infinite query")
    big = key_like(rng, nb, 1, 64, "bf16") * 2.0 ** 126
    check(dev, queries(rng, 1, 4, 64, "bf16") * 64, big, "bf16", bt, lens, 16, 20, 1, 1, what="scores past f32")
    tiny = key_like(rng, nb, 1, 64, "bf16") * 2.0 ** -120
    check(dev, queries(rng, 1, 4, 64, "bf16") * 2.0 ** -20, tiny, "bf16", bt, lens, 16, 20, 1, 1, what="scores below f32")


def test_f16_and_e5m2_subnormals_count(dev):
    rng = np.random.default_rng(32)
    lens = [120 * 16]
    bt, nb = S.tables(rng, lens, 16)
    for kv in ("f16", "e5m2"):
        kb = torch.from_numpy(np.sort(rng.standard_normal((nb, 1, 2, 64)), axis=2).astype(np.float32)) * 2.0 ** -16
        kb = S.store(kb, kv)
        q = queries(rng, 1, 4, 64, "f16")
        check(dev, q, kb, kv, bt, lens, 16, 30, 1, 1, what="subnormal bounds")
        check(dev, q * 2.0 ** -14, S.store(S.values(kb, kv).float() * 2.0 ** 17, kv), kv, bt, lens, 16, 30, 1, 1, what="subnormal queries")


@pytest.mark.parametrize("blocks", [8192 + 3, 8195 + 700, 20000])
def test_more_blocks_than_lds_holds(dev, blocks):
    rng = np.random.default_rng(blocks)
    lens = [blocks * 16 - 7, 5000 * 16, 3]
    bt, nb = S.tables(rng, lens, 16, spare=0)
    kb = key_like(rng, nb, 1, 32, "bf16")
    q = queries(rng, 3, 2, 32, "bf16")
    check(dev, q, kb, "bf16", bt, lens, 16, 100, 1, 2)
    check(dev, q, kb, "bf16", bt, lens, 16, 4096, 1, 2)
    kb[:] = kb[0].clone()
    check(dev, q, kb, "bf16", bt, lens, 16, 100, 1, 2, what="all alike")


def test_more_scratch_than_a_slab(dev):
    """Wide tables and many rows: the call works through its rows in parts."""
    rng = np.random.default_rng(2)
    n, width = 3000, 16384
    lens = rng.integers(1, 30 * 16, n).tolist()
    small, nb = S.tables(rng, lens, 16)
    kb, q = key_like(rng, nb, 8, 32, "bf16"), queries(rng, n, 8, 32, "bf16")
    size = ops.lib().rllm_select_blocks_workspace_size(n, 8, width)
    assert n * 8 * width * 4 > size >= 1 << 30
    bt = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    bt[:, :small.shape[1]] = small.to(dev)
    out = ops.select_blocks(q.to(dev), kb.to(dev), bt, torch.tensor(lens, dtype=torch.int32, device=dev), 16, 8, validate=False)
    ref = S.select(q, S.values(kb, "bf16"), small, lens, None, 16, 8, 1, 1)
    assert torch.equal(out.cpu(), ref)


def test_a_chunk_with_more_scratch_than_a_slab(dev):
    """The same for tiles of rows, cut by the parts' ends."""
    rng = np.random.default_rng(22)
    new, width = [901, 1, 1300, 40], 16384
    lens = [1500, 2000, 1300, 900]
    small, nb = S.tables(rng, lens, 16)
    qsl = np.concatenate([[0], np.cumsum(new)]).tolist()
    n = qsl[-1]
    kb, q = key_like(rng, nb, 8, 32, "bf16"), queries(rng, n, 16, 32, "bf16")
    assert n * 8 * width * 4 > ops.lib().rllm_select_blocks_workspace_size(n, 8, width)
    bt = torch.full((4, width), -1, dtype=torch.int32, device=dev)
    bt[:, :small.shape[1]] = small.to(dev)
    out = ops.select_blocks(q.to(dev), kb.to(dev), bt, torch.tensor(lens, dtype=torch.int32, device=dev), 16, 8, validate=False,
                            query_start_loc=torch.tensor(qsl, dtype=torch.int32, device=dev))
    wide = out.cpu()
    narrow = ops.select_blocks(q.to(dev), kb.to(dev), small.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), 16, 8,
                               query_start_loc=torch.tensor(qsl, dtype=torch.int32, device=dev)).cpu()
    assert torch.equal(wide, narrow)                            # every row; some of them against the formula
    for t in list(range(0, n, 97)) + [900, 901, 902, n - 41, n - 1]:
        s = int(np.searchsorted(qsl, t, side="right")) - 1
        one = S.select(q[t:t + 1], S.values(kb, "bf16"), small[s:s + 1], [lens[s] - (qsl[s + 1] - 1 - t)], None, 16, 8, 1, 1)
        assert torch.equal(wide[t:t + 1], one), t


def test_workspace_of_the_largest_serves_the_smaller(dev):
    rng = np.random.default_rng(14)
    lens = [200 * 16] * 6
    bt, nb = S.tables(rng, lens, 16)
    kb, q = key_like(rng, nb, 2, 64, "bf16"), queries(rng, 6, 8, 64, "bf16")
    ws = torch.full((ops.lib().rllm_select_blocks_workspace_size(6, 2, 200),), 0xA5, dtype=torch.uint8, device=dev)
    for n, w in ((6, 200), (1, 200), (3, 150), (6, 31)):
        check(dev, q[:n], kb, "bf16", bt[:n, :w].contiguous(), lens[:n], 16, 9, workspace=ws)
    with pytest.raises(KernelError):
        check(dev, q, kb, "bf16", bt, lens, 16, 9, workspace=ws[:-16])


def test_captured_and_replayed(dev):
    rng = np.random.default_rng(15)
    lens = [150 * 16, 90 * 16 + 3]
    bt, nb = S.tables(rng, lens, 16)
    kb, q = key_like(rng, nb, 2, 64, "bf16").to(dev), queries(rng, 2, 8, 64, "bf16").to(dev)
    args = (kb, bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), 16, 20)
    other = queries(rng, 2, 8, 64, "bf16").to(dev)
    want = [ops.select_blocks(x, *args) for x in (q, other)]
    assert not torch.equal(*want)
    with RawStream() as st:
        torch.cuda.synchronize()
        out = torch.zeros_like(want[0])
        g = torch.cuda.CUDAGraph()
        with pytest.raises(KernelError) as e:                   # the stream has no scratch yet
            with torch.cuda.graph(g, stream=st):
                ops.select_blocks(q, *args, out=out, validate=False)
        assert e.value.code == 900
        torch.cuda.synchronize()
        ops.select_blocks(q, *args, out=out, validate=False, stream=st)
        torch.cuda.synchronize()
        held = q.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ops.select_blocks(held, *args, out=out, validate=False)
        for x, w in ((q, want[0]), (other, want[1]), (q, want[0])):
            held.copy_(x)
            out.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)
            assert torch.equal(ops.select_blocks(x, *args), w)


def test_two_threads_on_one_stream(dev):
    rng = np.random.default_rng(16)
    lens = [400 * 16] * 5
    bt, nb = S.tables(rng, lens, 16)
    kb, t = key_like(rng, nb, 2, 64, "bf16").to(dev), bt.to(dev)
    lt = torch.tensor(lens, dtype=torch.int32, device=dev)
    qs = [queries(rng, 5, 8, 64, "bf16").to(dev) for _ in range(2)]
    want = [ops.select_blocks(q, kb, t, lt, 16, 33) for q in qs]
    outs, wrong, errors = [torch.zeros_like(w) for w in want], torch.zeros(2, dtype=torch.int64, device=dev), []
    torch.cuda.synchronize()

    def work(i, st):
        try:
            with torch.cuda.stream(st):
                for _ in range(60):
                    ops.select_blocks(qs[i], kb, t, lt, 16, 33, out=outs[i], validate=False, stream=st)
                    wrong[i] += (outs[i] != want[i]).any()
        except Exception as e:
            errors.append(e)

    with RawStream() as st:
        threads = [threading.Thread(target=work, args=(i, st)) for i in range(2)]
        for th in threads:
            th.start()
        for th in threads:
            th.join(timeout=60)
        torch.cuda.synchronize()
    assert not errors and wrong.tolist() == [0, 0]
