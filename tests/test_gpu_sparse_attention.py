"""Attention over listed blocks against a 64-bit softmax (tests/sparse_ref.py), and a run of the four operators together."""
import numpy as np
import pytest
import torch

import sparse_ref as S
from gpu_util import RawStream, log_case
from rllm_amd import ops

pytestmark = pytest.mark.gpu
SCALES = (0.5, 0.75)     # of an FP8 cache


def pool(rng, nb, hkv, d, bs, kv):
    return [S.store(torch.from_numpy(rng.standard_normal((nb, hkv, d, bs)).astype(np.float32)), kv) for _ in range(2)]


def queries(rng, n, hq, d, kind):
    return torch.from_numpy(rng.standard_normal((n, hq, d)).astype(np.float32)).to(S.HALF[kind])


def lists(rng, bt, lens, qsl, n, hkv, bs, k, holes=True):
    """Random lists, rising, as long as they may be, shorter and empty ones among them."""
    sel = torch.full((n, hkv, k), -1, dtype=torch.int32)
    for t, s, pos in S.rows(lens, qsl, n):
        nv = 0 if pos < 0 else min(pos // bs + 1, bt.shape[1])
        for h in range(hkv):
            m = min(nv, k if rng.random() < 0.7 else int(rng.integers(0, k + 1)))
            sel[t, h, :m] = torch.from_numpy(np.sort(rng.permutation(nv)[:m]).astype(np.int32))
    return sel


def check(dev, q, kc, vc, kind, kv, bt, lens, sel, bs, scale, qsl=None, what=""):
    ks, vs = SCALES if kv in S.FP8 else (1.0, 1.0)
    ref, mag, spread = S.attend(q, S.values(kc, kv), S.values(vc, kv), bt, lens, qsl, sel, scale, ks, vs)
    out = torch.full_like(q, 3.0).to(dev)
    log_case(f"attend rows={q.shape[0]} hq={q.shape[1]} hkv={kc.shape[1]} d={q.shape[2]} bs={bs} k={sel.shape[2]} {kind} {kv} {what}")
    kw = dict(k_scale=ks, v_scale=vs, **S.fp8(kv)) if kv in S.FP8 else {}
    qt = None if qsl is None else torch.tensor(qsl, dtype=torch.int32, device=dev)
    got = ops.paged_sparse(q.to(dev), kc.to(dev), vc.to(dev), bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                           sel.to(dev), scale, query_start_loc=qt, out=out, validate=False, **kw)
    assert got is out
    S.check_attend(out, ref, mag, spread, kind, q.shape[2], sel.shape[2] * bs, what)
    left = ref[:, 0, 0].isnan()
    assert (out.cpu()[left] == 3.0).all()
    return out


@pytest.mark.parametrize("kind,kv", S.TYPES)
@pytest.mark.parametrize("hq,hkv,d,bs", [(4, 1, 32, 16), (32, 8, 128, 16), (6, 2, 96, 32), (20, 1, 64, 64), (48, 1, 160, 16),
                                         (2, 2, 256, 128), (7, 1, 192, 16), (16, 1, 224, 32)])
def test_decode_rows(dev, kind, kv, hq, hkv, d, bs):
    rng = np.random.default_rng(d * 5 + hq)
    lens = [0, 1, bs, bs + 1, 9 * bs, 20 * bs - 3, 33 * bs, -2, 25 * bs + 1]
    bt, nb = S.tables(rng, lens, bs)
    kc, vc = pool(rng, nb, hkv, d, bs, kv)
    q = queries(rng, len(lens), hq, d, kind)
    for k in (1, 5, 19, 40):
        check(dev, q, kc, vc, kind, kv, bt, lens, lists(rng, bt, lens, None, len(lens), hkv, bs, k), bs, d ** -0.5)


@pytest.mark.parametrize("kind,kv", [("bf16", "bf16"), ("f16", "f16"), ("f16", "e4m3"), ("bf16", "e5m2")])
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 8, 128, 16), (6, 2, 64, 32), (20, 1, 96, 16), (2, 2, 256, 64)])
def test_chunk_rows(dev, kind, kv, hq, hkv, d, bs):
    rng = np.random.default_rng(d * 3 + hq)
    lens, new = [12 * bs + 5, 30 * bs, 17, 11 * bs + 1, 300], [1, 21, 17, 0, 9]
    bt, nb = S.tables(rng, lens, bs)
    kc, vc = pool(rng, nb, hkv, d, bs, kv)
    qsl = (3 + np.concatenate([[0], np.cumsum(new)])).tolist()
    n = sum(new) + 8
    q = queries(rng, n, hq, d, kind)
    check(dev, q, kc, vc, kind, kv, bt, lens, lists(rng, bt, lens, qsl, n, hkv, bs, 12), bs, d ** -0.5, qsl)
    lens[2], lens[4] = 5, 0                                     # more rows than keys, and none
    check(dev, q, kc, vc, kind, kv, bt, lens, lists(rng, bt, lens, qsl, n, hkv, bs, 12), bs, d ** -0.5, qsl)


def chunk(rng, lens, new, hq, hkv, d, bs, kind, kv):
    bt, nb = S.tables(rng, lens, bs)
    qsl = (2 + np.concatenate([[0], np.cumsum(new)])).tolist()
    n = sum(new) + 5
    return bt, pool(rng, nb, hkv, d, bs, kv), qsl, n, queries(rng, n, hq, d, kind)


@pytest.mark.parametrize("kind,kv,hq,hkv,d,bs,n", [
    ("bf16", "bf16", 32, 8, 128, 16, 150), ("f16", "e4m3", 24, 8, 128, 32, 150), ("bf16", "e5m2", 16, 16, 32, 16, 280),
    ("f16", "f16", 16, 8, 64, 64, 300), ("bf16", "bf16", 28, 4, 96, 128, 150), ("f16", "f16", 16, 2, 256, 16, 270),
    ("f16", "e5m2", 32, 8, 224, 16, 140), ("bf16", "e4m3", 32, 8, 96, 16, 140)])
def test_tiles_of_rows(dev, kind, kv, hq, hkv, d, bs, n):
    """Chunks whose rows share a workgroup: lists that overlap in part, that end where each row does, and empty ones; runs that end
    inside a tile, a sequence without rows, more rows than keys."""
    rng = np.random.default_rng(d + n)
    new = [n // 2 + 1, 0, 1, n // 3, 7, n - n // 2 - n // 3 - 9]
    lens = [9 * bs + 3 + new[0], 40, 1, 200 + new[3], 4, new[5]]
    bt, (kc, vc), qsl, rows, q = chunk(rng, lens, new, hq, hkv, d, bs, kind, kv)
    assert rows >= 2 * len(lens)
    sel = lists(rng, bt, lens, qsl, rows, hkv, bs, 7)
    check(dev, q, kc, vc, kind, kv, bt, lens, sel, bs, d ** -0.5, qsl)
    bt[0, 2], bt[3, 1], bt[5, 0] = -1, kc.shape[0], -7          # unused entries among the listed
    check(dev, q, kc, vc, kind, kv, bt, lens, sel, bs, 0.0, qsl)
    sel[:] = torch.from_numpy(rng.integers(-2, 12, tuple(sel.shape)).astype(np.int32))   # lists that do not rise
    check(dev, q, kc, vc, kind, kv, bt, lens, sel, bs, -d ** -0.5, qsl)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_rows_of_a_tile_do_not_see_each_other_s_blocks(dev, kv):
    rng = np.random.default_rng(91)
    lens, new = [400], [160]
    bt, (kc, vc), qsl, n, q = chunk(rng, lens, new, 32, 8, 64, 16, "bf16", kv)
    sel = lists(rng, bt, lens, qsl, n, 8, 16, 9)
    sel = torch.where(sel == 5, 6, sel)                         # now and then 6 twice: the second attends nothing
    kc, vc = S.values(kc, kv), S.values(vc, kv)
    kc[int(bt[0, 5])] = float("nan")
    vc[int(bt[0, 5])] = float("nan")
    vc[int(bt[0, 24]), :, :, 15] = float("nan")                 # the chunk's last key: the other rows stand before it
    some = sel.clone()
    hit = torch.zeros(n, dtype=torch.bool)
    hit[rng.permutation(n - 10)[:20]] = True
    some[hit, :, 0], some[hit, :, 1:] = 5, -1
    kc, vc = S.store(kc.float(), kv), S.store(vc.float(), kv)
    ks, vs = SCALES if kv in S.FP8 else (1.0, 1.0)
    ref, mag, spread = S.attend(q, S.values(kc, kv), S.values(vc, kv), bt, lens, qsl, some, 0.125, ks, vs)
    ref = torch.where(torch.isnan(ref), float("nan"), ref)
    kw = dict(k_scale=ks, v_scale=vs, **S.fp8(kv)) if kv in S.FP8 else {}
    out = ops.paged_sparse(q.to(dev), kc.to(dev), vc.to(dev), bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                           some.to(dev), 0.125, query_start_loc=torch.tensor(qsl, dtype=torch.int32, device=dev), validate=False, **kw)
    S.check_attend(out, ref, mag, spread, "bf16", 64, 9 * 16, "beside rows with NaN")
    rows = torch.arange(n)
    assert out.cpu()[hit & (rows >= 2) & (rows < 162)].isnan().all()


def test_what_is_not_attended_is_not_looked_at(dev):
    """NaN and infinities behind the last key, in unlisted blocks, in blocks of unused entries."""
    rng = np.random.default_rng(3)
    for kv in ("bf16", "e4m3"):
        lens = [100, 37, 160]
        bt, nb = S.tables(rng, lens, 16)
        kc, vc = (S.values(x, kv) for x in pool(rng, nb, 2, 64, 16, kv))
        sel = torch.tensor([[0, 3, 6, -1], [1, 2, -1, -1], [0, 5, 9, 12]], dtype=torch.int32)[:, None].repeat(1, 2, 1)
        keep = torch.zeros((nb, 16), dtype=torch.bool)
        for s, L in enumerate(lens):
            for j in sel[s, 0].tolist():
                if 0 <= j < (L + 15) // 16:
                    keep[int(bt[s, j]), :max(0, min(16, L - 16 * j))] = True
        for c, bad in ((kc, float("nan")), (vc, float("nan") if kv == "e4m3" else float("inf"))):
            c.copy_(torch.where(keep[:, None, None], c, torch.full_like(c, bad)))
        kc, vc = S.store(kc.float(), kv), S.store(vc.float(), kv)
        q = queries(rng, 3, 8, 64, "bf16")
        check(dev, q, kc, vc, "bf16", kv, bt, lens, sel, 16, 0.125)


def test_entries_that_attend_nothing(dev):
    rng = np.random.default_rng(13)
    lens = [200, 200, 200, 200]
    bt, nb = S.tables(rng, lens, 16)
    bt[1, 3], bt[1, 5] = -1, nb + 3
    kc, vc = pool(rng, nb, 1, 64, 16, "f16")
    sel = torch.tensor([[2, 2, 2, 7, 7, -1], [3, 4, 5, 6, -1, -1], [0, 13, 1 << 20, -5, -1, 2], [-1, -1, 4, 4, 3, 12]],
                       dtype=torch.int32)[:, None]
    check(dev, queries(rng, 4, 4, 64, "f16"), kc, vc, "f16", "f16", bt, lens, sel, 16, 0.125)
    none = torch.full_like(sel, -1)
    out = check(dev, queries(rng, 4, 4, 64, "f16"), kc, vc, "f16", "f16", bt, lens, none, 16, 0.125)
    assert (out == 0).all()
    # a table narrower than the lengths, and none at all
    check(dev, queries(rng, 4, 4, 64, "f16"), kc, vc, "f16", "f16", bt[:, :5].contiguous(), lens, sel, 16, 0.125)
    with pytest.raises(ValueError):
        ops.paged_sparse(queries(rng, 4, 4, 64, "f16").to(dev), kc.to(dev), vc.to(dev), bt.clamp(-1, nb - 1).to(dev),
                         torch.tensor(lens, dtype=torch.int32, device=dev), sel.to(dev), 0.125)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_scales_and_large_scores(dev, kind):
    rng = np.random.default_rng(23)
    lens = [300, 77]
    bt, nb = S.tables(rng, lens, 16)
    kc, vc = pool(rng, nb, 2, 64, 16, kind)
    q = queries(rng, 2, 8, 64, kind)
    sel = lists(rng, bt, lens, None, 2, 2, 16, 15)
    for scale in (-0.125, 0.0, 1e-6, 4.0):
        check(dev, q, kc, vc, kind, kind, bt, lens, sel, 16, scale, what=f"scale {scale}")
    # one key far ahead of the others: its value comes out, whatever the size of the score
    kc[int(bt[0, 2]), :, :, 4] = 100.0
    kc[int(bt[1, 1]), :, :, 3] = 100.0
    sel = torch.tensor([[0, 2, 5], [0, 1, -1]], dtype=torch.int32)[:, None].repeat(1, 2, 1)
    q = q.abs() + 0.5
    for scale in (1.0, 1e4, 1e9, 1e20, 1e30):
        out = ops.paged_sparse(q.to(dev), kc.to(dev), vc.to(dev), bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                               sel.to(dev), scale)
        for s, (b, o) in enumerate(((int(bt[0, 2]), 4), (int(bt[1, 1]), 3))):
            want = vc[b, :, :, o].repeat_interleave(4, 0)
            assert torch.allclose(out[s].cpu().float(), want.float(), rtol=2.0 ** -7, atol=1e-6), scale


def test_a_key_that_is_not_finite_shows(dev):
    rng = np.random.default_rng(24)
    lens = [100, 100]
    bt, nb = S.tables(rng, lens, 16)
    kc, vc = pool(rng, nb, 1, 64, 16, "bf16")
    kc[int(bt[0, 1]), 0, 3, 3] = float("nan")
    vc[int(bt[1, 1]), 0, 9, 3] = float("inf")
    sel = torch.tensor([[0, 1, 6], [0, 1, 6]], dtype=torch.int32)[:, None]
    q = queries(rng, 2, 4, 64, "bf16")
    args = (q.to(dev), kc.to(dev), vc.to(dev), bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), sel.to(dev))
    assert all(ops.paged_sparse(*args, scale)[0].isnan().all() for scale in (1e9, -1e9, 1e30))
    out = ops.paged_sparse(*args, 0.125).cpu()
    assert out[0].isnan().all()
    assert not out[1, :, 9].isfinite().any() and out[1, :, 10:].isfinite().all() and out[1, :, :9].isfinite().all()


@pytest.mark.parametrize("kind,kv,hq,hkv,d,bs,k", [("bf16", "bf16", 32, 8, 128, 16, 64), ("f16", "e4m3", 20, 1, 64, 32, 40),
                                                   ("f16", "f16", 2, 2, 256, 128, 9), ("bf16", "e5m2", 6, 2, 96, 16, 300)])
def test_few_rows_over_several_workgroups(dev, kind, kv, hq, hkv, d, bs, k):
    """Lists cut between workgroups that the last to end joins: the same bits every time, also where the lists are short; and as
    a graph, with the stream's scratch and without."""
    rng = np.random.default_rng(k)
    lens = [k * bs + 40, 1, 5 * bs + 3, 0]
    bt, nb = S.tables(rng, lens, bs)
    kc, vc = pool(rng, nb, hkv, d, bs, kv)
    q = queries(rng, 4, hq, d, kind)
    sel = lists(rng, bt, lens, None, 4, hkv, bs, k)
    out = check(dev, q, kc, vc, kind, kv, bt, lens, sel, bs, d ** -0.5)
    ref = S.attend(q, S.values(kc, kv), S.values(vc, kv), bt, lens, None, sel, d ** -0.5, *(SCALES if kv in S.FP8 else (1.0, 1.0)))
    args = [x.to(dev) for x in (q, kc, vc, bt, torch.tensor(lens, dtype=torch.int32), sel)]
    kw = dict(k_scale=SCALES[0], v_scale=SCALES[1], **S.fp8(kv)) if kv in S.FP8 else {}
    for _ in range(5):
        assert torch.equal(ops.paged_sparse(*args, d ** -0.5, **kw), out)
    with RawStream() as st:
        torch.cuda.synchronize()
        got = [torch.zeros_like(out) for _ in range(2)]
        graphs = []
        for g in got:                                           # first without scratch, then with
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=st):
                ops.paged_sparse(*args, d ** -0.5, out=g, validate=False, **kw)
            torch.cuda.synchronize()
            ops.paged_sparse(*args, d ** -0.5, validate=False, stream=st, **kw)
            torch.cuda.synchronize()
        for _ in range(3):
            for g, x in zip(graphs, got):
                x.fill_(float("nan"))
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                S.check_attend(x, *ref, kind, d, k * bs, "replayed")
            assert torch.equal(got[1], out)
            assert torch.equal(ops.paged_sparse(*args, d ** -0.5, **kw), out)


def test_few_rows_on_two_streams_at_once(dev):
    """Each stream has scratch of its own: calls of different inputs that overlap give what they give alone."""
    rng = np.random.default_rng(77)
    lens = [2000, 1300]
    bt, nb = S.tables(rng, lens, 16)
    kc, vc = (x.to(dev) for x in pool(rng, nb, 8, 128, 16, "bf16"))
    t, lt = bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    work = []
    for _ in range(2):
        q, sel = queries(rng, 2, 32, 128, "bf16").to(dev), lists(rng, bt, lens, None, 2, 8, 16, 60).to(dev)
        want = ops.paged_sparse(q, kc, vc, t, lt, sel, 0.09)
        work.append((q, sel, want, [torch.zeros_like(want) for _ in range(20)]))
    torch.cuda.synchronize()
    with RawStream() as a, RawStream() as b:
        for i in range(20):
            for st, (q, sel, _, outs) in zip((a, b), work):
                ops.paged_sparse(q, kc, vc, t, lt, sel, 0.09, out=outs[i], validate=False, stream=st)
        torch.cuda.synchronize()
    for _, _, want, outs in work:
        assert all(torch.equal(x, want) for x in outs)


@pytest.mark.parametrize("d,hkv,rows", [(256, 1, 2), (128, 1, 2), (256, 4, 40), (128, 4, 40)])
def test_the_longest_lists(dev, d, hkv, rows):
    """4096 entries, beside the windows of wide heads; also as a graph on a stream without scratch."""
    rng = np.random.default_rng(d + hkv)
    lens = [70000, 30] + [400] * (rows - 2)
    bt, nb = S.tables(rng, lens, 16)
    kc, vc = pool(rng, nb, hkv, d, 16, "bf16")
    q = queries(rng, rows, 2 * hkv, d, "bf16")
    sel = lists(rng, bt, lens, None, rows, hkv, 16, 4096)
    sel[0, 0] = torch.arange(4096) + 200
    sel[0, -1, 4000:] = -1
    out = check(dev, q, kc, vc, "bf16", "bf16", bt, lens, sel, 16, d ** -0.5)
    args = [x.to(dev) for x in (q, kc, vc, bt, torch.tensor(lens, dtype=torch.int32), sel)]
    with RawStream() as st:
        torch.cuda.synchronize()
        got = torch.zeros_like(out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ops.paged_sparse(*args, d ** -0.5, out=got, validate=False)
        g.replay()
        torch.cuda.synchronize()
    assert ((got - out).float().abs() <= 2.0 ** -7 * out.float().abs() + 1e-6).all()


def test_whole_lists_match_the_dense_kernels(dev):
    rng = np.random.default_rng(33)
    lens = [500, 3, 999, 160]
    bt, nb = S.tables(rng, lens, 16)
    kc, vc = (x.to(dev) for x in pool(rng, nb, 4, 128, 16, "bf16"))
    q, lt, t = queries(rng, 4, 16, 128, "bf16").to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), bt.to(dev)
    sel = torch.arange(64, dtype=torch.int32, device=dev).repeat(4, 4, 1)
    sel = torch.where(sel < (lt[:, None, None] + 15) // 16, sel, -1)
    a, b = ops.paged_sparse(q, kc, vc, t, lt, sel, 0.1), ops.paged_decode(q, kc, vc, t, lt, 0.1)
    # two roundings to bf16, and the dense kernel's weights rounded to it
    assert ((a - b).float().abs() <= 2.0 ** -7 * b.float().abs() + 2.0 ** -8 * vc.float().abs().max()).all()


def test_caches_past_32_bits(dev):
    """Blocks whose offsets pass 2^32 bytes in every cache and in the bounds."""
    rng = np.random.default_rng(43)
    hkv, d, bs = 8, 256, 16
    nb = (1 << 32) // (hkv * 2 * d) + 50                        # bounds of one byte an element
    kc = torch.zeros((nb, hkv, d, bs), dtype=torch.uint8, device=dev)
    vc, kb = torch.zeros_like(kc), ops.new_key_bounds(kc)
    lens = [10 * bs + 5]
    blocks = [nb - 1 - 3 * i for i in range(11)]
    bt = torch.tensor([blocks], dtype=torch.int32)
    small = pool(rng, 11, hkv, d, bs, "e4m3")
    at = torch.tensor(blocks, device=dev)
    kc[at], vc[at] = (x.to(dev) for x in small)
    lt = torch.tensor(lens, dtype=torch.int32, device=dev)
    ops.key_bounds(kc, kb, bt.to(dev), lt, **S.fp8("e4m3"))
    near = torch.arange(11, dtype=torch.int32)[None]
    ref = S.bounds(torch.zeros((11, hkv, 2, d)).double(), S.values(small[0], "e4m3"), near, lens, bs)
    assert torch.equal(S.values(kb[at], "e4m3"), ref)
    q = queries(rng, 1, 16, d, "bf16")
    sel = ops.select_blocks(q.to(dev), kb, bt.to(dev), lt, bs, 6, **S.fp8("e4m3"))
    assert torch.equal(sel.cpu(), S.select(q, ref, near, lens, None, bs, 6, 1, 1))
    out = ops.paged_sparse(q.to(dev), kc, vc, bt.to(dev), lt, sel, 0.1, k_scale=SCALES[0], v_scale=SCALES[1], **S.fp8("e4m3"))
    r = S.attend(q, *(S.values(x, "e4m3") for x in small), near, lens, None, sel.cpu(), 0.1, *SCALES)
    S.check_attend(out, *r, "bf16", d, 6 * bs, "past 2^32")
    # a new token there
    cos, sin = (x.to(dev) for x in ops.rope_cache_tables(200, d))
    k, v = (queries(rng, 1, hkv, d, "bf16") for _ in range(2))
    lt += 1
    ops.rope_and_append(None, k.to(dev), v.to(dev), kc, vc, kb, bt.to(dev), lt, cos, sin, **S.fp8("e4m3"))
    S.append(q, k, v, small[0], small[1], ref, near, [lens[0] + 1], None, cos.cpu(), sin.cpu(), "e4m3")
    assert torch.equal(kc[at].cpu(), small[0]) and torch.equal(vc[at].cpu(), small[1])
    assert torch.equal(S.values(kb[at], "e4m3"), ref)


@pytest.mark.parametrize("kind,kv", [("bf16", "bf16"), ("f16", "e4m3")])
def test_a_run_of_steps(dev, kind, kv):
    """Prompts appended in chunks, then decode steps: append, select, attend, each against the formulas; the decode step once
    more as a replayed graph."""
    rng = np.random.default_rng(55)
    hq, hkv, d, bs, k = 8, 2, 64, 16, 6
    steps = [[70, 0, 33], [61, 130, 0], [0, 7, 1]] + [[1, 1, 1]] * 3
    total = [sum(x) for x in zip(*steps)]
    bt, nb = S.tables(rng, total, bs)
    t = bt.to(dev)
    kc, vc = (x.to(dev) for x in pool(rng, nb, hkv, d, bs, kv))
    kb = ops.new_key_bounds(kc)
    cos, sin = ops.rope_cache_tables(300, d, 10000.0)
    dcos, dsin = cos.to(dev), sin.to(dev)
    ks, vs = SCALES if kv in S.FP8 else (1.0, 1.0)
    kw = dict(k_scale=ks, v_scale=vs, **S.fp8(kv)) if kv in S.FP8 else {}
    rk, rv, rb = kc.cpu(), vc.cpu(), S.values(kb, kv)
    lens = [0, 0, 0]
    for i, new in enumerate(steps):
        lens = [a + b for a, b in zip(lens, new)]
        n = sum(new)
        qsl = None if i > 2 else np.concatenate([[0], np.cumsum(new)]).tolist()
        qt = None if qsl is None else torch.tensor(qsl, dtype=torch.int32, device=dev)
        lt = torch.tensor(lens, dtype=torch.int32, device=dev)
        q, kk, vv = (queries(rng, n, h, d, kind) for h in (hq, hkv, hkv))
        qd, kd, vd = (x.to(dev) for x in (q, kk, vv))
        qr = ops.rope_and_append(qd, kd, vd, kc, vc, kb, t, lt, dcos, dsin, query_start_loc=qt, **kw)
        sel = ops.select_blocks(qr, kb, t, lt, bs, k, num_first=1, num_last=2, query_start_loc=qt, **S.fp8(kv))
        out = ops.paged_sparse(qr, kc, vc, t, lt, sel, d ** -0.5, query_start_loc=qt, **kw)
        ref_q = S.append(q, kk, vv, rk, rv, rb, bt, lens, qsl, cos, sin, kv, ks, vs)
        assert torch.equal(qr.cpu(), ref_q) and S.same_values(S.values(kb, kv), rb)
        ref_sel = S.select(ref_q, rb, bt, lens, qsl, bs, k, 1, 2)
        assert torch.equal(sel.cpu(), ref_sel)
        r = S.attend(ref_q, S.values(rk, kv), S.values(rv, kv), bt, lens, qsl, ref_sel, d ** -0.5, ks, vs)
        S.check_attend(out, *r, kind, d, k * bs, f"step {i}")
    ws = torch.empty(ops.lib().rllm_select_blocks_workspace_size(3, hkv, t.shape[1]), dtype=torch.uint8, device=dev)
    got = [torch.zeros_like(x) for x in (qr, sel, out)]

    def step():
        ops.rope_and_append(qd, kd, vd, kc, vc, kb, t, lt, dcos, dsin, q_out=got[0], validate=False, **kw)
        ops.select_blocks(got[0], kb, t, lt, bs, k, num_first=1, num_last=2, out=got[1], workspace=ws, validate=False, **S.fp8(kv))
        ops.paged_sparse(got[0], kc, vc, t, lt, got[1], d ** -0.5, out=got[2], validate=False, **kw)

    with RawStream() as st:
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            step()                                              # the stream's scratch, as the default stream has it
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            step()
        for _ in range(3):
            for x in got:
                x.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, (qr, sel, out)))
            assert torch.equal(ops.paged_sparse(qr, kc, vc, t, lt, sel, d ** -0.5, **kw), out)
