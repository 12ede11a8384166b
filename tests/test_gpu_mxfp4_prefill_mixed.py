"""Chunked prefill over the MXFP4 cache where sequences of few new tokens are taken apart
from those of many, and where contexts are cut between workgroups: against the 64-bit
formulation."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
from rllm_amd import ops
from gpu_util import RawStream
from test_gpu_mxfp4_decode import case as decode_case, dev_args as decode_args
from test_gpu_mxfp4_prefill import WEIGHT, case, dev_args, reference, run_and_check

pytestmark = pytest.mark.gpu
# 24 sequences of 8 kv heads: few and many new tokens, none, contexts shorter than them
NEW = [1, 300, 1, 0, 2, 8, 9, 40, 1, 0, 1, 1, 16, 17, 1, 3, 1, 70, 1, 1, 2, 0, 1, 33]
CTX = [900, 400, 1, 50, 2, 2000, 30, 40, 33, 0, 64, 65, 1016, 17, 31, 700, 32, 1270, 500, 16, 3, 10, 1, 300]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("new,ctx,hq,hkv,d,bs", [
    ([1], [1], 1, 1, 32, 16),
    ([5, 0, 1, 64], [5, 30, 77, 64], 8, 2, 64, 16),
    ([130, 3], [430, 3], 24, 8, 128, 32),
    ([65], [64 + 65], 28, 4, 96, 48),
    ([40, 41], [81, 500], 6, 2, 160, 16),
    ([33], [97], 16, 16, 192, 64),
    ([20, 90], [220, 90], 3, 1, 224, 16),
    ([100], [1000], 10, 2, 256, 16),
])
def test_tables_far_wider_than_the_contexts(dev, kind, new, ctx, hq, hkv, d, bs):
    run_and_check(np.random.default_rng(sum(ctx) + d), new, ctx, hq, hkv, d, bs, kind, dev, width=1500 // bs)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 8, 64, 16), (24, 8, 128, 32), (8, 8, 96, 16), (48, 8, 256, 64), (160, 8, 32, 16)])
def test_few_and_many_new_tokens_in_one_batch(dev, kind, hq, hkv, d, bs):
    run_and_check(np.random.default_rng(d), NEW, CTX, hq, hkv, d, bs, kind, dev)


@pytest.mark.parametrize("new,hq,hkv", [(1, 8, 2), (4, 8, 2), (8, 32, 4)])
def test_more_sequences_than_a_wave_has_lanes(dev, new, hq, hkv):
    rng = np.random.default_rng(new)
    ctx = rng.integers(new, 1200, 140).tolist()
    run_and_check(rng, [new] * 140, ctx, hq, hkv, 64, 16, "bf16", dev)


def test_missing_blocks_and_short_contexts(dev):
    def drop(q, kc, vc, bt, lens, qsl):
        bt[0, 2:6] = -1
        bt[5, 100:] = -1
        bt[8, :] = -1
        bt[12, 0] = 10 ** 6
        lens[15] = 2         # fewer keys than new tokens: the first sees nothing
        lens[16] = 0
    out, c = run_and_check(np.random.default_rng(3), NEW, CTX, 32, 8, 64, 16, "bf16", dev, edit=drop, validate=False)
    qsl = c[5]
    for t in (qsl[8], qsl[15], qsl[16]):
        assert not out[t].view(torch.int16).any()


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_stale_rows_and_nan(dev, kind):
    rng = np.random.default_rng(5)
    c = case(rng, NEW, CTX, 16, 8, 128, 16, kind, dev)
    q, kc, vc, bt, lens, qsl = c
    used = np.zeros((kc.shape[0], kc.shape[3]), bool)
    for s, n in enumerate(lens):
        for t in range(n):
            used[bt[s, t // 16], t % 16] = True
    for x in (kc, vc):
        x.scales.transpose(0, 2, 1, 3)[~used] = 255
        x.codes.transpose(0, 2, 1, 3)[~used] = 15
    want = np.zeros(tuple(q.shape), bool)
    for s in (5, 7, 15, 17):                 # 8 new on 1992, 40 fresh, 3 on 697, 70 on 1200
        n, cached = NEW[s], CTX[s] - NEW[s]
        at = cached + n // 2                 # a value of kv head 1, elements 64..95
        vc.scales[bt[s, at // 16], 1, at % 16, 2] = 255
        want[qsl[s] + n // 2:qsl[s + 1], 2:4, 64:96] = True
        at = cached + n - 1                  # a key of kv head 7, which the last token sees
        kc.scales[bt[s, at // 16], 7, at % 16, 0] = 255
        want[qsl[s + 1] - 1, 14:] = True
        q[qsl[s], 5, 7] = float("inf")
        want[qsl[s], 5] = True
    out = ops.paged_prefill_mxfp4(*dev_args(*c, dev), 0.09).float().cpu().numpy()
    assert np.array_equal(np.isnan(out), want)


def test_rows_behind_the_last_sequence_stay_and_replays_agree(dev):
    c = case(np.random.default_rng(6), NEW, CTX, 32, 8, 64, 16, "bf16", dev)
    q = torch.cat([c[0], torch.randn((13, 32, 64), device=dev).bfloat16()])
    a = (q,) + dev_args(*c, dev)[1:]
    ref, mag, big = reference(*c, 0.125)
    eager = torch.full_like(q, 7.0)
    ops.paged_prefill_mxfp4(*a, 0.125, out=eager, validate=False)
    for warm in (False, True):
        with RawStream() as st:
            st.wait_stream(torch.cuda.current_stream())
            out = torch.full_like(q, 7.0)
            if warm:
                ops.paged_prefill_mxfp4(*a, 0.125, stream=st, out=out, validate=False)
                torch.cuda.synchronize()
                assert torch.equal(out, eager)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                ops.paged_prefill_mxfp4(*a, 0.125, out=out, validate=False)
            for i in range(3):
                out.fill_(7.0)
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                n = sum(NEW)
                M.check_attention(out[:n].float().cpu().numpy(), ref, mag, big, "bf16", WEIGHT["bf16"], f"replay {i}")
                assert (out[n:] == 7.0).all()
                again = torch.full_like(q, 7.0)
                ops.paged_prefill_mxfp4(*a, 0.125, out=again, validate=False)
                assert torch.equal(again, eager)


@pytest.mark.parametrize("new", [0, 1, 40])
def test_nan_of_a_part_with_next_to_no_weight(dev, new):
    """A context's first half scores 399 (in log2) below its second; a NaN value there still
    reaches the outputs, as it does where the context is not cut into parts."""
    rng = np.random.default_rng(8)
    if new:
        c = case(rng, [new], [4000], 8, 2, 128, 16, "bf16", dev)
        q, kc, vc, bt, lens, qsl = c
    else:
        c = decode_case(rng, [4000], 8, 2, 128, 16, "bf16", dev)
        q, kc, vc, bt, lens = c
    q.fill_(4.0)
    for t in range(4000):
        b, r = bt[0, t // 16], t % 16
        kc.codes[b, :, r] = 15 if t < 2000 else 0        # -6 or 0
        kc.scales[b, :, r] = 127
    vc.scales[bt[0, 50 // 16], 1, 50 % 16, 2] = 255      # of a score of -399 in log2
    want = np.zeros(tuple(q.shape), bool)
    want[:, 4:, 64:96] = True
    out = ops.paged_prefill_mxfp4(*dev_args(*c, dev), 0.09) if new else ops.paged_decode_mxfp4(*decode_args(*c, dev), 0.09)
    assert np.array_equal(torch.isnan(out).cpu().numpy(), want)


@pytest.mark.parametrize("new,ctx,wide", [([40, 3], [200, 64], 0), ([90, 40], [200, 64], 40), ([4], [230], 40)])
def test_long_cache_past_32_bits(dev, new, ctx, wide):
    """The contexts' blocks lie past 2^32 bytes; tables of their own width and far wider ones."""
    rng = np.random.default_rng(17)
    nb, hkv, d, bs = 70000, 8, 256, 32
    kt, vt = (ops.mxfp4_cache(nb, hkv, d, bs, dev) for _ in range(2))
    kc, vc = M.Cache.random(rng, 12, hkv, d, bs), M.Cache.random(rng, 12, hkv, d, bs)
    kt[nb - 12:] = torch.from_numpy(kc.pages()).to(dev)
    vt[nb - 12:] = torch.from_numpy(vc.pages()).to(dev)
    bt = np.full((len(new), 8 + wide), -1, np.int32)
    for s in range(len(new)):
        bt[s, :8] = rng.permutation(12)[:8]
    q = torch.from_numpy(rng.standard_normal((sum(new), 16, d))).to(torch.bfloat16).to(dev)
    lens, qsl = np.array(ctx, np.int32), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    far = np.where(bt >= 0, bt + nb - 12, -1).astype(np.int32)
    out = ops.paged_prefill_mxfp4(q, kt, vt, *(torch.from_numpy(x).to(dev) for x in (far, lens, qsl)), 0.06)
    ref, mag, big = reference(q, kc, vc, bt, lens, qsl, 0.06)
    M.check_attention(out.float().cpu().numpy(), ref, mag, big, "bf16", WEIGHT["bf16"], "past 32 bits")
