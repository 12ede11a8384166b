"""The MXFP4 entry points' host-side checks (no GPU work), and the 64-bit
formulation they are tested against."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
import rllm_amd
from rllm_amd import ops

P = 0x1000   # never dereferenced: validation fails first


def write(n=4, hkv=8, d=128, bs=16, nb=10, dt=1, kc=P, vc=P, k=P, v=P, sm=P):
    return rllm_amd.lib().rllm_cache_write_mxfp4(kc, vc, k, v, sm, n, hkv, d, bs, nb, dt, 0)


def read(n=4, hkv=8, d=128, bs=16, nb=10, dt=1, kc=P, vc=P, k=P, v=P, sm=P):
    return rllm_amd.lib().rllm_cache_read_mxfp4(k, v, kc, vc, sm, n, hkv, d, bs, nb, dt, 0)


def rope(n=4, hq=32, hkv=8, d=128, bs=16, nb=10, maxp=100, dt=1, q=P, qo=P, k=P, v=P, kc=P, vc=P, sm=P, pos=P, cs=P,
         sn=P):
    return rllm_amd.lib().rllm_rope_cache_write_mxfp4(qo, q, k, v, kc, vc, sm, pos, cs, sn, n, hq, hkv, d, bs, nb, maxp,
                                                      dt, 0)


def decode(b=4, hq=32, hkv=8, d=128, bs=16, maxb=4, nb=10, scale=0.1, dt=1, ws=None, wsb=0, o=P, q=P, kc=P, vc=P, bt=P,
           sl=P):
    return rllm_amd.lib().rllm_paged_attention_decode_mxfp4(o, q, kc, vc, bt, sl, b, hq, hkv, d, bs, maxb, nb, scale, dt,
                                                            ws, wsb, 0)


@pytest.mark.parametrize("f", [write, read, rope])
def test_row_operators_refuse(f):
    for bad in (dict(hkv=0), dict(hkv=1025), dict(d=0), dict(d=48), dict(d=288), dict(bs=0), dict(bs=8), dict(bs=24),
                dict(bs=8192), dict(nb=-1), dict(dt=2), dict(dt=-1), dict(kc=0), dict(vc=0), dict(k=0), dict(v=0),
                dict(sm=0), dict(kc=P + 8), dict(vc=P + 4), dict(k=P + 2), dict(v=P + 8), dict(n=1 << 31)):
        assert f(**bad) == 1, bad
    assert f(n=0, kc=0) == 0 and f(n=-3) == 0      # empty work


def test_rope_refuses():
    for bad in (dict(d=96), dict(d=32), dict(hq=-1), dict(hq=1025), dict(maxp=0), dict(q=0), dict(qo=0), dict(q=P + 8),
                dict(qo=P + 4), dict(pos=0), dict(cs=0), dict(sn=0), dict(cs=P + 4), dict(sn=P + 8)):
        assert rope(**bad) == 1, bad


def test_decode_refuses():
    for bad in (dict(hkv=0), dict(hq=0), dict(hq=30), dict(hq=2048, hkv=1024), dict(d=40), dict(d=512), dict(bs=8),
                dict(maxb=-1), dict(maxb=1 << 25), dict(bs=4096, maxb=1 << 16), dict(nb=0), dict(nb=-1), dict(b=(1 << 20) + 1),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(dt=2), dict(o=0), dict(q=0), dict(kc=0),
                dict(vc=0), dict(bt=0), dict(sl=0), dict(kc=P + 8), dict(vc=P + 1), dict(q=P + 2), dict(o=P + 2)):
        assert decode(**bad) == 1, bad
    assert decode(b=0, o=0) == 0 and decode(b=-1) == 0


def prefill(b=2, t=10, hq=32, hkv=8, d=128, bs=16, maxb=4, nb=10, scale=0.1, dt=1, o=P, q=P, kc=P, vc=P, bt=P, sl=P,
            qsl=P):
    return rllm_amd.lib().rllm_paged_attention_prefill_mxfp4(o, q, kc, vc, bt, sl, qsl, b, t, hq, hkv, d, bs, maxb, nb,
                                                             scale, dt, 0)


def test_prefill_refuses():
    for bad in (dict(hkv=0), dict(hq=0), dict(hq=30), dict(d=40), dict(d=512), dict(bs=8), dict(maxb=-1),
                dict(maxb=1 << 25), dict(nb=0), dict(b=(1 << 20) + 1), dict(t=(1 << 26) + 1), dict(scale=float("nan")),
                dict(dt=3), dict(o=0), dict(q=0), dict(kc=0), dict(vc=0), dict(bt=0), dict(sl=0), dict(qsl=0),
                dict(kc=P + 8), dict(vc=P + 8), dict(q=P + 8), dict(o=P + 4)):
        assert prefill(**bad) == 1, bad
    assert prefill(b=0, o=0) == 0 and prefill(t=0) == 0


def test_launches_past_the_devices_limit_are_refused():
    n = (1 << 31) - 1                                # 2^32 threads and more
    assert write(n=n, hkv=1024) == 1 and read(n=n, hkv=1024) == 1 and rope(n=n, hkv=1024) == 1
    assert prefill(b=1 << 20, t=1 << 26, hq=1024, hkv=1024, maxb=1) == 1
    for f in (decode, prefill):                      # finite, but not in units of log2
        assert f(scale=3e38) == 1


def test_sizes():
    L = rllm_amd.lib()
    assert L.rllm_mxfp4_page_bytes(128, 16) == 16 * (64 + 4) == M.page_bytes(128, 16)
    assert L.rllm_mxfp4_page_bytes(96, 32) == M.page_bytes(96, 32)
    assert L.rllm_mxfp4_page_bytes(100, 16) == -1 and L.rllm_mxfp4_page_bytes(128, 20) == -1
    assert ops.mxfp4_cache(3, 2, 64, 16, "cpu").shape == (3, 2, 16 * 34)
    with pytest.raises(ValueError):
        ops.mxfp4_cache(3, 2, 64, 8, "cpu")
    W = L.rllm_paged_attention_decode_mxfp4_workspace_size
    assert W(0, 32, 8, 128, 16, 4) == 0 and W(4, 30, 8, 128, 16, 4) == -1 and W(4, 32, 8, 100, 16, 4) == -1


def test_front_end_refuses():
    kc = ops.mxfp4_cache(4, 2, 64, 16, "cpu")
    k = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    s = torch.zeros(3, dtype=torch.int64)
    for a in ((k, k[:2], kc, kc, s), (k, k, kc, kc[:2], s), (k, k, kc, kc, s.int()), (k, k, kc, kc, s[:2]),
              (k[:, :1].contiguous(), k[:, :1].contiguous(), kc, kc, s), (k, k, kc.view(torch.int8), kc, s),
              (k, k, kc[..., :-16].contiguous(), kc[..., :-16].contiguous(), s)):
        with pytest.raises(ValueError):
            ops.reshape_and_cache_mxfp4(*a)
    with pytest.raises(TypeError):
        ops.reshape_and_cache_mxfp4(k.float(), k.float(), kc, kc, s)
    with pytest.raises(ValueError):          # not on a GPU
        ops.reshape_and_cache_mxfp4(k, k, kc, kc, s)
    with pytest.raises(ValueError):
        ops.read_cache_mxfp4(kc, kc, s)
    with pytest.raises(ValueError):
        ops.read_cache_mxfp4(kc, kc, s, out_key=k)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    bt, sl = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for a in ((q[0], kc, kc, bt, sl, 1.0), (q, kc, kc, bt[:1], sl, 1.0), (q[..., :32].contiguous(), kc, kc, bt, sl, 1.0),
              (q, kc, kc, bt, sl, 1.0)):
        with pytest.raises(ValueError):
            ops.paged_decode_mxfp4(*a)
        with pytest.raises(ValueError):
            ops.paged_prefill_mxfp4(*a[:5], torch.zeros(3, dtype=torch.int32), 1.0)
    with pytest.raises(TypeError):
        ops.paged_decode_mxfp4(q, kc, kc, bt.long(), sl, 1.0)


def test_reference_quantiser():
    x = np.zeros((2, 32))
    x[0, :10] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -0.26, -0.0]
    c, e = M.quantise(x)
    assert e.tolist() == [[127], [1]]
    assert M.values(c, e)[0, :10].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, -0.5, 0]
    assert c[0, 9] == 8
    x[1, 3] = np.inf
    assert M.quantise(x)[1].tolist() == [[127], [255]]
    page = M.Cache.random(np.random.default_rng(0), 2, 3, 64, 16)
    again = M.Cache.from_pages(page.pages(), 64, 16)
    assert np.array_equal(again.codes, page.codes) and np.array_equal(again.scales, page.scales)
