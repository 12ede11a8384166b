"""Decode attention over the MXFP4 cache on the GPU against the 64-bit formulation."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
from rllm_amd import ops
from gpu_util import RawStream, log_case

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}
# two bf16 terms a weight: 2^-17 of it; exp2 and the f32 sums are off by a few 2^-23
WEIGHT = 2.0 ** -16


def tables(rng, lens, bs, extra=2, width=None):
    nblk = [(max(n, 0) + bs - 1) // bs for n in lens]
    nb = sum(nblk) + extra
    perm = rng.permutation(nb).astype(np.int32)
    bt = np.full((len(lens), width or max(max(nblk), 1)), -1, np.int32)
    p = 0
    for s, n in enumerate(nblk):
        bt[s, :n] = perm[p:p + n]
        p += n
    return bt, nb


def case(rng, lens, hq, hkv, d, bs, kind, dev, width=None, qmul=1.0):
    bt, nb = tables(rng, lens, bs, width=width)
    kc, vc = M.Cache.random(rng, nb, hkv, d, bs), M.Cache.random(rng, nb, hkv, d, bs)
    q = torch.from_numpy(rng.standard_normal((len(lens), hq, d)) * qmul).to(DT[kind]).to(dev)
    return q, kc, vc, bt, np.array(lens, np.int32)


def dev_args(q, kc, vc, bt, lens, dev):
    return (q, torch.from_numpy(kc.pages()).to(dev), torch.from_numpy(vc.pages()).to(dev), torch.from_numpy(bt).to(dev),
            torch.from_numpy(lens).to(dev))


def reference(q, kc, vc, bt, lens, scale):
    x = q.cpu().double().numpy()
    parts = [M.attend(x[s:s + 1], kc, vc, bt[s], int(lens[s]), 1, scale) for s in range(len(lens))]
    return [np.concatenate([p[i] for p in parts]) for i in range(3)]


def run_and_check(rng, lens, hq, hkv, d, bs, kind, dev, width=None, qmul=1.0, scale=None, edit=None, validate=True):
    c = case(rng, lens, hq, hkv, d, bs, kind, dev, width, qmul)
    if edit:
        edit(*c)
    scale = 1 / np.sqrt(d) if scale is None else scale
    what = f"decode lens={lens[:6]} hq={hq} hkv={hkv} d={d} bs={bs} {kind}"
    log_case(what)
    out = ops.paged_decode_mxfp4(*dev_args(*c, dev), scale, validate=validate)
    ref, mag, big = reference(*c, scale)
    M.check_attention(out.float().cpu().numpy(), ref, mag, big, kind, WEIGHT, what)
    return out, c


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("lens,hq,hkv,d,bs", [
    ([1], 1, 1, 32, 16),
    ([0, 1, 15, 16, 17, 31, 32, 33], 8, 2, 64, 16),
    ([700], 32, 8, 128, 16),
    ([130, 5, 0, 1000, 64], 24, 8, 128, 32),
    ([257, 96], 7, 1, 96, 48),
    ([1023], 28, 4, 160, 16),
    ([300, 2], 16, 16, 192, 64),
    ([77, 555], 6, 3, 224, 16),
    ([2000], 40, 8, 256, 16),
    ([65], 48, 2, 128, 16),         # 24 query heads a kv head: two groups
    ([400], 33, 1, 64, 4096),       # 33: three groups, one block
])
def test_shapes(dev, kind, lens, hq, hkv, d, bs):
    run_and_check(np.random.default_rng(sum(lens) + d), lens, hq, hkv, d, bs, kind, dev)


def test_many_sequences(dev):
    rng = np.random.default_rng(9)
    lens = rng.integers(0, 90, 200).tolist()     # more than a wave's 64 lengths
    run_and_check(rng, lens, 4, 2, 64, 16, "bf16", dev)


@pytest.mark.parametrize("lo", [1, 150])
def test_many_short_rows(dev, lo):
    # a row or more for every two waves of the chip: workgroups of two waves, several rows each
    rng = np.random.default_rng(22)
    lens = rng.integers(lo, 150, 150, endpoint=True).tolist()
    run_and_check(rng, lens, 16, 8, 64, 16, "bf16", dev)
    run_and_check(rng, lens[:140], 16, 8, 160, 32, "f16", dev)


@pytest.mark.parametrize("lens", [[64] * 9, [1, 700, 33, 64, 2], [3000] + [40] * 20, [0, 0, 5000]])
def test_equal_and_unequal_parts(dev, lens):
    # rows cut at multiples of one part, and a list cut into equal shares
    rng = np.random.default_rng(23)
    run_and_check(rng, lens, 8, 2, 128, 16, "bf16", dev)


def test_long_row_cut_between_workgroups(dev):
    rng = np.random.default_rng(10)
    run_and_check(rng, [9001, 40], 4, 1, 128, 16, "bf16", dev)
    run_and_check(rng, [9001, 0, 777], 5, 1, 64, 32, "f16", dev, width=1000)   # a table far wider than the contexts


def test_missing_blocks_and_narrow_tables(dev):
    rng = np.random.default_rng(11)

    def drop(q, kc, vc, bt, lens):
        bt[0, 3:9] = -1              # holes
        bt[1, :] = -1                # nothing left
        bt[2, 1] = 10 ** 6           # past the cache
        lens[3] = 10 ** 6            # past the table
        lens[4] = -7
    out, _ = run_and_check(rng, [300, 100, 90, 64, 33], 8, 2, 128, 16, "bf16", dev, edit=drop, validate=False)
    assert not out[1].view(torch.int16).any() and not out[4].view(torch.int16).any()


def test_stale_rows_and_unused_blocks_are_not_read_into_the_result(dev):
    # NaN scales and wild codes behind the contexts' ends and in unused blocks
    rng = np.random.default_rng(12)

    def poison(q, kc, vc, bt, lens):
        used = np.zeros((kc.shape[0], kc.shape[3]), bool)
        for s, n in enumerate(lens):
            for t in range(n):
                used[bt[s, t // 16], t % 16] = True
        for c in (kc, vc):
            sc = c.scales.transpose(0, 2, 1, 3)
            sc[~used] = 255
            co = c.codes.transpose(0, 2, 1, 3)
            co[~used] = 15
    run_and_check(rng, [1, 17, 47, 240], 8, 2, 128, 16, "bf16", dev, edit=poison)


def test_nan_in_a_visible_row_reaches_its_outputs_only(dev):
    rng = np.random.default_rng(13)
    q, kc, vc, bt, lens = case(rng, [40, 50], 4, 2, 64, 16, "bf16", dev)
    vc.scales[bt[0, 1], 1, 3, 1] = 255       # value of sequence 0, kv head 1, elements 32..63
    kc.scales[bt[1, 0], 0, 2, 0] = 255       # key of sequence 1, kv head 0
    out = ops.paged_decode_mxfp4(*dev_args(q, kc, vc, bt, lens, dev), 0.125).float().cpu().numpy()
    nan = np.isnan(out)
    want = np.zeros_like(nan)
    want[0, 2:, 32:] = True
    want[1, :2] = True
    assert np.array_equal(nan, want)
    # a query that is not finite
    q[0, 0, 5] = float("inf")
    q[1, 3, 0] = float("nan")
    out = ops.paged_decode_mxfp4(*dev_args(q, kc, vc, bt, lens, dev), 0.125).float().cpu().numpy()
    assert np.isnan(out[0, 0]).all() and np.isnan(out[1, 3]).all() and np.isfinite(out[0, 1]).all()


def test_scales_of_every_size(dev):
    # large and tiny keys, values and queries; a softmax of one key; negative and zero scale
    rng = np.random.default_rng(14)

    def grow(kf, vf):
        def edit(q, kc, vc, bt, lens):
            kc.scales[...] = np.clip(kc.scales.astype(int) + kf, 1, 254)
            vc.scales[...] = np.clip(vc.scales.astype(int) + vf, 1, 254)
        return edit
    run_and_check(rng, [200, 3], 8, 2, 128, 16, "bf16", dev, edit=grow(0, 100))
    run_and_check(rng, [200, 3], 8, 2, 128, 16, "bf16", dev, edit=grow(0, -100))
    run_and_check(rng, [200, 3], 8, 2, 128, 16, "bf16", dev, edit=grow(40, 0), qmul=2.0 ** -40)
    run_and_check(rng, [200, 3], 8, 2, 128, 16, "bf16", dev, edit=grow(-60, 0), qmul=2.0 ** 60)
    run_and_check(rng, [200, 3], 8, 2, 128, 16, "f16", dev, scale=-0.1)
    run_and_check(rng, [200, 3], 8, 2, 128, 16, "f16", dev, scale=0.0)


def test_same_bits_every_time_streams_and_workspaces(dev):
    rng = np.random.default_rng(15)
    c = case(rng, [5000, 10, 900, 33], 8, 2, 128, 16, "bf16", dev)
    a = dev_args(*c, dev)
    first = ops.paged_decode_mxfp4(*a, 0.088)
    L = ops.lib()
    need = L.rllm_paged_attention_decode_mxfp4_workspace_size(4, 8, 2, 128, 16, a[3].shape[1])
    ws = torch.zeros(need, dtype=torch.uint8, device=dev)
    for _ in range(20):
        assert torch.equal(first, ops.paged_decode_mxfp4(*a, 0.088))
        assert torch.equal(first, ops.paged_decode_mxfp4(*a, 0.088, workspace=ws))
    torch.cuda.synchronize()
    assert not ws[: 16384].any(), "arrival counters are back at zero"
    with RawStream() as st, RawStream() as st2:
        st.wait_stream(torch.cuda.current_stream())
        st2.wait_stream(torch.cuda.current_stream())
        outs = []
        for _ in range(10):
            outs.append(ops.paged_decode_mxfp4(*a, 0.088, stream=st, out=torch.empty_like(first)))
            outs.append(ops.paged_decode_mxfp4(*a, 0.088, stream=st2, out=torch.empty_like(first)))
        torch.cuda.synchronize()
        assert all(torch.equal(first, o) for o in outs)


def test_one_workspace_for_calls_of_every_size(dev):
    # few workgroups, then many, then few: no call's partials under another's counters
    rng = np.random.default_rng(21)
    cases = [([1500], 4, 1, 256), ([2000, 900, 60] * 8, 32, 8, 128), ([3000], 4, 1, 64), ([5000] * 6, 16, 4, 128)]
    L, built, need = ops.lib(), [], 0
    for lens, hq, hkv, d in cases:
        c = case(rng, lens, hq, hkv, d, 16, "bf16", dev)
        a = dev_args(*c, dev)
        need = max(need, L.rllm_paged_attention_decode_mxfp4_workspace_size(len(lens), hq, hkv, d, 16, a[3].shape[1]))
        built.append((a, reference(*c, 0.09)))
    ws = torch.zeros(need, dtype=torch.uint8, device=dev)
    for i in (0, 1, 2, 3, 2, 1, 0, 3, 1):
        a, (ref, mag, big) = built[i]
        for w in (ws, None):
            out = ops.paged_decode_mxfp4(*a, 0.09, workspace=w)
            M.check_attention(out.float().cpu().numpy(), ref, mag, big, "bf16", WEIGHT, f"case {i}")
    assert not ws[: 16384].any()


def test_captured_with_and_without_scratch(dev):
    rng = np.random.default_rng(16)
    c = case(rng, [3000, 70], 8, 2, 128, 16, "bf16", dev)
    a = dev_args(*c, dev)
    ref, mag, big = reference(*c, 0.088)
    eager = ops.paged_decode_mxfp4(*a, 0.088)
    for warm in (False, True):
        with RawStream() as st:
            st.wait_stream(torch.cuda.current_stream())
            out = torch.zeros_like(eager)
            if warm:
                with torch.cuda.stream(st):
                    ops.paged_decode_mxfp4(*a, 0.088)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                ops.paged_decode_mxfp4(*a, 0.088, out=out, validate=False)
            for i in range(4):
                out.fill_(float("nan"))
                torch.cuda.synchronize()
                g.replay()
                torch.cuda.synchronize()
                M.check_attention(out.float().cpu().numpy(), ref, mag, big, "bf16", WEIGHT, f"replay {i} warm={warm}")
                assert torch.equal(ops.paged_decode_mxfp4(*a, 0.088), eager)
                if warm:
                    assert torch.equal(out, eager)


def test_long_cache_past_32_bits(dev):
    # the context's blocks lie past 2^32 bytes
    rng = np.random.default_rng(17)
    nb, hkv, d, bs = 70000, 8, 256, 32
    kt = ops.mxfp4_cache(nb, hkv, d, bs, dev)
    vt = ops.mxfp4_cache(nb, hkv, d, bs, dev)
    lens = np.array([200, 64], np.int32)
    kc, vc = M.Cache.random(rng, 12, hkv, d, bs), M.Cache.random(rng, 12, hkv, d, bs)
    kt[nb - 12:] = torch.from_numpy(kc.pages()).to(dev)
    vt[nb - 12:] = torch.from_numpy(vc.pages()).to(dev)
    bt = rng.permutation(12).astype(np.int32)[:7]
    bt = np.stack([bt, np.roll(bt, 2)])
    q = torch.from_numpy(rng.standard_normal((2, 8, d))).to(torch.bfloat16).to(dev)
    out = ops.paged_decode_mxfp4(q, kt, vt, torch.from_numpy(bt + nb - 12).to(dev), torch.from_numpy(lens).to(dev), 0.06)
    ref, mag, big = reference(q, kc, vc, bt, lens, 0.06)
    M.check_attention(out.float().cpu().numpy(), ref, mag, big, "bf16", WEIGHT, "past 32 bits")
