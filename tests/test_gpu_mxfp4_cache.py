"""MXFP4 cache rows on the GPU against the 64-bit formulation (tests/mxfp4_ref.py):
the write, the rotation fused with it, and the read, byte for byte."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
from rllm_amd import ops
from gpu_util import log_case

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def rows16(rng, n, hkv, d, kind, dev):
    """16-bit rows whose blocks spread over the exponent range, zeros and borders of two codes among them."""
    x = rng.standard_normal((n, hkv, d // 32, 32))
    x *= np.exp2(rng.integers(-12, 12, (n, hkv, d // 32, 1)))
    grid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.5, 0.0, -0.0])
    border = rng.random((n, hkv, d // 32, 1)) < 0.4
    e = np.exp2(rng.integers(-10, 10, (n, hkv, d // 32, 1)).astype(np.float64))
    x = np.where(border, rng.choice(grid, x.shape) * rng.choice([-1.0, 1.0], x.shape) * e, x)
    x[rng.random((n, hkv, d // 32)) < 0.1] = 0.0
    return torch.from_numpy(x.reshape(n, hkv, d)).to(DT[kind]).to(dev)


def f64(t):
    return t.detach().cpu().double().numpy()


def pool(rng, nb, hkv, d, bs, dev):
    c = M.Cache.random(rng, nb, hkv, d, bs)
    return c, torch.from_numpy(c.pages()).to(dev)


def same_bits(a, b):
    return np.array_equal(a.cpu().view(torch.int16).numpy(), b.cpu().view(torch.int16).numpy())


def slots_of(rng, n, nb, bs, skip=0.1):
    s = rng.permutation(nb * bs)[:n].astype(np.int64)
    s[rng.random(n) < skip] = -1
    if n > 3:
        s[1] = nb * bs + 5      # a block past the cache
        s[2] = -(1 << 40)
    return s


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n,hkv,d,bs", [(1, 1, 32, 16), (3, 2, 64, 16), (37, 8, 128, 16), (65, 3, 96, 32),
                                        (9, 5, 160, 48), (130, 4, 256, 64), (17, 1, 224, 4096)])
def test_write_and_read(dev, kind, n, hkv, d, bs):
    rng = np.random.default_rng(n * 1000 + d)
    nb = max(2, 2 * n // bs + 2)
    kc, kt = pool(rng, nb, hkv, d, bs, dev)
    vc, vt = pool(rng, nb, hkv, d, bs, dev)
    k, v = rows16(rng, n, hkv, d, kind, dev), rows16(rng, n, hkv, d, kind, dev)
    slots = slots_of(rng, n, nb, bs)
    log_case(f"write n={n} hkv={hkv} d={d} bs={bs} {kind}")
    ops.reshape_and_cache_mxfp4(k, v, kt, vt, torch.from_numpy(slots).to(dev))
    kc.write(f64(k), slots)
    vc.write(f64(v), slots)
    torch.cuda.synchronize()
    assert np.array_equal(kt.cpu().numpy(), kc.pages()), "key pages"      # untouched rows among them
    assert np.array_equal(vt.cpu().numpy(), vc.pages()), "value pages"
    # read: every slot written, some twice, some skipped
    back = np.concatenate([slots, slots[::-1], rng.integers(0, nb * bs, 11)])
    for out in ("bf16", "f16"):
        ko, vo = ops.read_cache_mxfp4(kt, vt, torch.from_numpy(back).to(dev), head_dim=d, dtype=DT[out])
        for got, ref in ((ko, kc), (vo, vc)):
            want = torch.from_numpy(ref.rows(back)).to(DT[out])    # rounded to nearest even once
            assert same_bits(got, want), out


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_every_16_bit_pattern(dev, kind):
    # each pattern as one block's whole content, and beside a block's largest value
    bits = np.arange(65536, dtype=np.uint16).astype(np.int16)
    x = torch.from_numpy(bits).view(DT[kind])
    rows = x[:, None, None].expand(65536, 1, 32).contiguous()
    mixed = rows.clone()
    mixed[:, :, 7] = 1.5
    mixed[:, :, 31] = -0.375
    for r in (rows, mixed):
        n = r.shape[0]
        kt = ops.mxfp4_cache(n // 16, 1, 32, 16, dev)
        vt = torch.zeros_like(kt)
        slots = torch.arange(n, dtype=torch.int64, device=dev)
        ops.reshape_and_cache_mxfp4(r.to(dev), r.neg().to(dev), kt, vt, slots)
        ref = M.Cache(n // 16, 1, 32, 16)
        c, e = M.quantise(f64(r))
        ref.codes, ref.scales = c.reshape(n // 16, 16, 1, 32).transpose(0, 2, 1, 3), e.reshape(n // 16, 16, 1, 1).transpose(0, 2, 1, 3)
        assert np.array_equal(kt.cpu().numpy(), ref.pages())
        c, e = M.quantise(f64(r.neg()))
        ref.codes, ref.scales = c.reshape(n // 16, 16, 1, 32).transpose(0, 2, 1, 3), e.reshape(n // 16, 16, 1, 1).transpose(0, 2, 1, 3)
        assert np.array_equal(vt.cpu().numpy(), ref.pages())


def test_read_every_code_and_scale(dev):
    # 256 scale bytes (NaN and 2^-127 among them) x 16 codes, to both types
    nb = 16
    ref = M.Cache(nb, 1, 32, 16)
    ref.codes[...] = np.tile(np.arange(16, dtype=np.uint8), 2)
    ref.scales[...] = np.arange(256, dtype=np.uint8).reshape(nb, 1, 16, 1)
    kt = torch.from_numpy(ref.pages()).to(dev)
    slots = torch.arange(256, dtype=torch.int64, device=dev)
    for out in ("bf16", "f16"):
        ko, _ = ops.read_cache_mxfp4(kt, kt, slots, head_dim=32, dtype=DT[out])
        want = torch.from_numpy(ref.rows(np.arange(256))).to(DT[out])
        got, nan = ko.cpu(), torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        assert same_bits(got[~nan], want[~nan]), out


def rotate_f32(x, cos, sin):
    """Each product and sum rounded to f32."""
    a, b = np.split(x.astype(np.float32), 2, axis=-1)
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n,hq,hkv,d,bs,inplace", [(1, 4, 1, 64, 16, False), (33, 32, 8, 128, 16, True),
                                                   (7, 3, 3, 192, 32, False), (20, 0, 2, 128, 16, False),
                                                   (5, 14, 2, 256, 64, True)])
def test_rope_and_write(dev, kind, n, hq, hkv, d, bs, inplace):
    rng = np.random.default_rng(n + d)
    nb = n // bs + 3
    kc, kt = pool(rng, nb, hkv, d, bs, dev)
    vc, vt = pool(rng, nb, hkv, d, bs, dev)
    k, v = (torch.from_numpy(rng.standard_normal((n, hkv, d))).to(DT[kind]).to(dev) for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((n, hq, d))).to(DT[kind]).to(dev) if hq else None
    cos, sin = ops.rope_cache_tables(500, d, 10000.0, device=dev)
    pos = rng.integers(-2, 503, n).astype(np.int32)    # clamped to the table
    slots = slots_of(rng, n, nb, bs)
    log_case(f"rope n={n} hq={hq} hkv={hkv} d={d} bs={bs} {kind}")
    q0 = None if q is None else q.clone()
    got = ops.rope_and_cache_mxfp4(q, k, v, kt, vt, torch.from_numpy(slots).to(dev), torch.from_numpy(pos).to(dev), cos,
                                   sin, q_out=q if inplace else None)
    p = np.clip(pos, 0, 499)
    c, s = cos.cpu().numpy()[p][:, None], sin.cpu().numpy()[p][:, None]
    kr = rotate_f32(k.float().cpu().numpy(), c, s)
    kc.write(kr.astype(np.float64), slots)
    vc.write(f64(v), slots)
    assert np.array_equal(kt.cpu().numpy(), kc.pages()), "key pages"
    assert np.array_equal(vt.cpu().numpy(), vc.pages()), "value pages"
    if q is None:
        assert got is None
        return
    want = torch.from_numpy(rotate_f32(q0.float().cpu().numpy(), c, s)).to(DT[kind])
    assert same_bits(got, want)
    assert got is q if inplace else same_bits(q, q0)


def test_copy_swap_and_zero_move_whole_blocks(dev):
    # the block movers take these caches as they are
    rng = np.random.default_rng(3)
    kc, kt = pool(rng, 6, 2, 64, 16, dev)
    vc, vt = pool(rng, 6, 2, 64, 16, dev)
    ops.copy_blocks([kt], [vt], torch.tensor([[1, 4], [0, 5]], dtype=torch.int64, device=dev))
    assert torch.equal(kt[4], kt[1]) and torch.equal(vt[5], vt[0])
    assert np.array_equal(kt[:4].cpu().numpy(), kc.pages()[:4])
    rec = torch.zeros((2, 1, 2, kt[0].numel()), dtype=torch.uint8).pin_memory()
    ids = torch.tensor([2, 3], dtype=torch.int64, device=dev)
    ops.swap_out([kt], [vt], ids, rec)
    torch.cuda.synchronize()
    assert np.array_equal(rec[1, 0, 1].numpy(), vc.pages()[3].ravel())
    kt[2:4] = 0
    ops.swap_in([kt], [vt], ids, rec)
    torch.cuda.synchronize()
    assert np.array_equal(kt[2:4].cpu().numpy(), kc.pages()[2:4])
    z = ops.mxfp4_cache(2, 1, 64, 16, dev)
    ko, vo = ops.read_cache_mxfp4(z, z, torch.arange(32, device=dev), head_dim=64, dtype=torch.bfloat16)
    assert not ko.view(torch.int16).any() and not vo.view(torch.int16).any()


def test_slots_past_32_bits(dev):
    # a cache of more than 2^32 bytes: rows at its end
    nb, hkv, d, bs = 70000, 8, 256, 32     # 4.9e9 bytes
    kt = ops.mxfp4_cache(nb, hkv, d, bs, dev)
    n = 40
    k = torch.randn((n, hkv, d), device=dev, dtype=torch.bfloat16)
    slots = torch.arange(nb * bs - n, nb * bs, dtype=torch.int64, device=dev)
    ops.reshape_and_cache_mxfp4(k, k, kt, kt, slots)
    ref = M.values(*M.quantise(f64(k)))
    ko, _ = ops.read_cache_mxfp4(kt, kt, slots, head_dim=d, dtype=torch.bfloat16)
    assert np.array_equal(f64(ko), ref)
    assert not kt[: nb - 2].any()
