"""Chunked-prefill attention over the MXFP4 cache on the GPU against the 64-bit
formulation, and the operators of a serving step together."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
from rllm_amd import ops
from gpu_util import RawStream, log_case
from test_gpu_mxfp4_decode import DT, tables

pytestmark = pytest.mark.gpu
# a bf16 weight is off by at most half a step, 2^-8; two bf16 terms by 2^-17
WEIGHT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -16}


def case(rng, new, ctx, hq, hkv, d, bs, kind, dev, width=None):
    bt, nb = tables(rng, ctx, bs, width=width)
    kc, vc = M.Cache.random(rng, nb, hkv, d, bs), M.Cache.random(rng, nb, hkv, d, bs)
    q = torch.from_numpy(rng.standard_normal((sum(new), hq, d))).to(DT[kind]).to(dev)
    qsl = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return q, kc, vc, bt, np.array(ctx, np.int32), qsl


def dev_args(q, kc, vc, bt, lens, qsl, dev):
    return (q, torch.from_numpy(kc.pages()).to(dev), torch.from_numpy(vc.pages()).to(dev), torch.from_numpy(bt).to(dev),
            torch.from_numpy(lens).to(dev), torch.from_numpy(qsl).to(dev))


def reference(q, kc, vc, bt, lens, qsl, scale):
    x = q.cpu().double().numpy()
    parts = [M.attend(x[qsl[s]:qsl[s + 1]], kc, vc, bt[s], int(lens[s]), int(qsl[s + 1] - qsl[s]), scale)
             for s in range(len(lens))]
    return [np.concatenate([p[i] for p in parts]) for i in range(3)]


def run_and_check(rng, new, ctx, hq, hkv, d, bs, kind, dev, width=None, edit=None, validate=True):
    c = case(rng, new, ctx, hq, hkv, d, bs, kind, dev, width)
    if edit:
        edit(*c)
    what = f"prefill new={new[:5]} ctx={ctx[:5]} hq={hq} hkv={hkv} d={d} bs={bs} {kind}"
    log_case(what)
    out = ops.paged_prefill_mxfp4(*dev_args(*c, dev), 1 / np.sqrt(d), validate=validate)
    ref, mag, big = reference(*c, 1 / np.sqrt(d))
    M.check_attention(out.float().cpu().numpy(), ref, mag, big, kind, WEIGHT[kind], what)
    return out, c


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("new,ctx,hq,hkv,d,bs", [
    ([1], [1], 1, 1, 32, 16),
    ([5, 0, 1, 64], [5, 30, 77, 64], 8, 2, 64, 16),
    ([117], [117], 32, 8, 64, 16),
    ([130, 3], [430, 3], 24, 8, 128, 32),
    ([65], [64 + 65], 28, 4, 96, 48),
    ([300], [300], 4, 1, 128, 16),
    ([40, 41], [81, 500], 6, 2, 160, 16),
    ([33], [97], 16, 16, 192, 64),
    ([20, 90], [220, 90], 3, 1, 224, 16),
    ([100], [1000], 10, 2, 256, 16),
    ([12], [700], 48, 1, 128, 4096),
])
def test_shapes(dev, kind, new, ctx, hq, hkv, d, bs):
    run_and_check(np.random.default_rng(sum(ctx) + d), new, ctx, hq, hkv, d, bs, kind, dev)


def test_many_sequences(dev):
    rng = np.random.default_rng(1)
    new = rng.integers(0, 30, 150).tolist()     # more than a wave's 64, some without tokens
    ctx = [n + int(c) for n, c in zip(new, rng.integers(0, 60, 150))]
    run_and_check(rng, new, ctx, 4, 2, 64, 16, "bf16", dev)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_few_tokens_on_a_long_context_are_split(dev, kind):
    rng = np.random.default_rng(2)
    run_and_check(rng, [4, 1], [3001, 64], 8, 2, 128, 16, kind, dev)
    run_and_check(rng, [9], [2000], 4, 1, 64, 32, kind, dev, width=2000)    # a table far wider than the context


def test_missing_blocks_short_contexts_and_narrow_tables(dev):
    rng = np.random.default_rng(3)

    def drop(q, kc, vc, bt, lens, qsl):
        bt[0, 2:6] = -1
        bt[1, :] = -1
        bt[2, 0] = 10 ** 6
        lens[3] = 20         # fewer keys than new tokens: the first ones see nothing
        lens[4] = 0
    out, c = run_and_check(rng, [70, 10, 20, 40, 5], [200, 40, 60, 40, 5], 8, 2, 128, 16, "bf16", dev, edit=drop,
                           validate=False)
    assert not out[70:80].view(torch.int16).any() and not out[100:120].view(torch.int16).any()
    # positions past the table's width see the keys it holds
    c = case(rng, [30], [64], 4, 1, 64, 16, "bf16", dev)
    c[4][0] = 94
    a = dev_args(*c, dev)
    out = ops.paged_prefill_mxfp4(*a, 0.125, validate=False)
    ref = M.attend(c[0].cpu().double().numpy(), c[1], c[2], c[3][0], 64, 0, 0.125)[0]
    full = [M.attend(c[0][i:i + 1].cpu().double().numpy(), c[1], c[2], c[3][0], 64, 1, 0.125) for i in range(30)]
    M.check_attention(out.float().cpu().numpy(), *(np.concatenate([f[j] for f in full]) for j in range(3)), "bf16",
                      WEIGHT["bf16"], "past the table")
    assert ref.shape == (30, 4, 64)


def test_stale_rows_are_not_read_into_the_result(dev):
    rng = np.random.default_rng(4)

    def poison(q, kc, vc, bt, lens, qsl):
        used = np.zeros((kc.shape[0], kc.shape[3]), bool)
        for s, n in enumerate(lens):
            for t in range(n):
                used[bt[s, t // 16], t % 16] = True
        for c in (kc, vc):
            c.scales.transpose(0, 2, 1, 3)[~used] = 255
            c.codes.transpose(0, 2, 1, 3)[~used] = 15
    run_and_check(rng, [1, 17, 40], [1, 47, 240], 8, 2, 128, 16, "bf16", dev, edit=poison)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("cached", [0, 1500])
def test_nan_reaches_only_the_rows_that_see_it(dev, kind, cached):
    rng = np.random.default_rng(5)
    n = 80 if not cached else 8          # the long one is split over its keys
    c = case(rng, [n], [cached + n], 8, 2, 128, 16, kind, dev)
    q, kc, vc, bt, lens, qsl = c
    at = cached + n // 2 + 1             # a value of kv head 1, elements 64..95
    vc.scales[bt[0, at // 16], 1, at % 16, 2] = 255
    ak = cached + n - 2                  # a key of kv head 0
    kc.scales[bt[0, ak // 16], 0, ak % 16, 0] = 255
    qi = cached and 3 or 20
    q[qi, 5, 7] = float("inf")
    nan = torch.isnan(ops.paged_prefill_mxfp4(*dev_args(*c, dev), 0.09).cpu()).numpy()
    want = np.zeros_like(nan)
    want[n // 2 + 1:, 4:, 64:96] = True
    want[n - 2:, :4] = True
    want[qi, 5] = True
    assert np.array_equal(nan, want)


def test_rows_outside_every_sequence_stay(dev):
    rng = np.random.default_rng(6)
    for new, ctx in (([20, 7], [20, 90]), ([3], [2500])):       # whole, and split over the keys
        c = case(rng, new, ctx, 8, 2, 64, 16, "bf16", dev)
        q = torch.cat([c[0], torch.randn((13, 8, 64), device=dev).bfloat16()])
        out = torch.full_like(q, 7.0)
        a = dev_args(*c, dev)
        ops.paged_prefill_mxfp4(q, *a[1:], 0.125, out=out, validate=False)
        ref, mag, big = reference(*c, 0.125)
        n = sum(new)
        M.check_attention(out[:n].float().cpu().numpy(), ref, mag, big, "bf16", WEIGHT["bf16"], "padded")
        assert (out[n:] == 7.0).all()


def test_streams_and_capture(dev):
    rng = np.random.default_rng(7)
    for new, ctx in (([50, 20], [300, 20]), ([6], [3000])):
        c = case(rng, new, ctx, 8, 2, 128, 16, "bf16", dev)
        a = dev_args(*c, dev)
        ref, mag, big = reference(*c, 0.088)
        eager = ops.paged_prefill_mxfp4(*a, 0.088)
        for warm in (False, True):
            with RawStream() as st:
                st.wait_stream(torch.cuda.current_stream())
                out = torch.zeros_like(eager)
                if warm:
                    ops.paged_prefill_mxfp4(*a, 0.088, stream=st, out=out, validate=False)
                    torch.cuda.synchronize()
                    assert torch.equal(out, eager)
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=st):
                    ops.paged_prefill_mxfp4(*a, 0.088, out=out, validate=False)
                for i in range(3):
                    out.fill_(float("nan"))
                    torch.cuda.synchronize()
                    g.replay()
                    torch.cuda.synchronize()
                    M.check_attention(out.float().cpu().numpy(), ref, mag, big, "bf16", WEIGHT["bf16"], f"replay {i}")
                    assert torch.equal(ops.paged_prefill_mxfp4(*a, 0.088), eager)


def test_a_chunk_and_decode_steps_together(dev):
    """A prompt in two chunks, then decode steps: rotate and write, attend, read
    back, against the formulation fed with the same rows."""
    rng = np.random.default_rng(8)
    hq, hkv, d, bs, scale = 8, 2, 128, 16, 1 / np.sqrt(128)
    lens = [90, 37]
    nblk = [8, 4]
    perm = rng.permutation(12).astype(np.int32)
    bt = np.full((2, 8), -1, np.int32)
    bt[0, :8], bt[1, :4] = perm[:8], perm[8:]
    kt, vt = (ops.mxfp4_cache(12, hkv, d, bs, dev) for _ in range(2))
    kc, vc = M.Cache(12, hkv, d, bs), M.Cache(12, hkv, d, bs)
    cos, sin = ops.rope_cache_tables(200, d, 500000.0, device=dev)
    cn, sn = cos.cpu().numpy(), sin.cpu().numpy()
    tbt = torch.from_numpy(bt).to(dev)
    done = [0, 0]

    def step(new):
        n = sum(new)
        pos = np.concatenate([np.arange(done[s], done[s] + new[s]) for s in range(2)])
        slots = np.concatenate([[bt[s, p // bs] * bs + p % bs for p in range(done[s], done[s] + new[s])] for s in range(2)])
        slots = slots.astype(np.int64)
        q, k, v = (torch.from_numpy(rng.standard_normal((n, h, d))).bfloat16().to(dev) for h in (hq, hkv, hkv))
        qr = ops.rope_and_cache_mxfp4(q, k, v, kt, vt, torch.from_numpy(slots).to(dev),
                                      torch.from_numpy(pos.astype(np.int32)).to(dev), cos, sin)
        from test_gpu_mxfp4_cache import rotate_f32
        kc.write(rotate_f32(k.float().cpu().numpy(), cn[pos][:, None], sn[pos][:, None]).astype(np.float64), slots)
        vc.write(v.cpu().double().numpy(), slots)
        for s in range(2):
            done[s] += new[s]
        sl = torch.tensor(done, dtype=torch.int32, device=dev)
        if max(new) == 1:
            out = ops.paged_decode_mxfp4(qr, kt, vt, tbt, sl, scale)
            w = 2.0 ** -16
        else:
            qsl = torch.tensor([0, new[0], n], dtype=torch.int32, device=dev)
            out = ops.paged_prefill_mxfp4(qr, kt, vt, tbt, sl, qsl, scale)
            w = WEIGHT["bf16"]
        x = qr.cpu().double().numpy()
        parts, p = [], 0
        for s in range(2):
            parts.append(M.attend(x[p:p + new[s]], kc, vc, bt[s], done[s], new[s], scale))
            p += new[s]
        M.check_attention(out.float().cpu().numpy(), *(np.concatenate([y[i] for y in parts]) for i in range(3)), "bf16",
                          w, f"step {new}")

    step([60, 37])
    step([30, 0])
    assert done == lens
    for _ in range(4):
        step([1, 1])
    assert np.array_equal(kt.cpu().numpy(), kc.pages()) and np.array_equal(vt.cpu().numpy(), vc.pages())
    back = np.array([bt[0, t // bs] * bs + t % bs for t in range(done[0])], np.int64)
    ko, vo = ops.read_cache_mxfp4(kt, vt, torch.from_numpy(back).to(dev), head_dim=d, dtype=torch.bfloat16)
    assert np.array_equal(ko.cpu().double().numpy(), kc.rows(back)) and np.array_equal(vo.cpu().double().numpy(), vc.rows(back))
    assert nblk == [8, 4]
