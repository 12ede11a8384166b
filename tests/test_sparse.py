"""Refusals of the operators over selected cache blocks, on the host and before any launch; the scratch's size."""
import itertools

import pytest
import torch

import rllm_amd
from rllm_amd import ops

P = 0x1000   # never dereferenced: validation fails first


def bounds(L, kb=P, kc=P, bt=P, lens=P, n=2, hkv=8, d=128, bs=16, maxb=4, nb=10, kv=1):
    return L.rllm_key_bounds(kb, kc, bt, lens, None, n, hkv, d, bs, maxb, nb, kv, 0)


def append(L, q_out=P, q=P, k=P, kc=P, kb=P, lens=P, qsl=None, cos=P, n=2, rows=2, hq=32, hkv=8, d=128, bs=16, maxb=4, nb=10,
           maxp=100, dt=1, kv=1, ks=1.0, rounding=0):
    return L.rllm_rope_cache_append(q_out, q, k, P, kc, P, kb, P, lens, qsl, cos, P, n, rows, hq, hkv, d, bs, maxb, nb, maxp,
                                    dt, kv, ks, 1.0, rounding, 0)


def select(L, sel=P, q=P, kb=P, bt=P, qsl=None, n=2, rows=2, hq=32, hkv=8, d=128, bs=16, maxb=40, nb=10, k=8, first=1, last=1,
           dt=1, kv=1, ws=P, ws_bytes=1 << 20):
    return L.rllm_select_blocks(sel, q, kb, bt, P, qsl, n, rows, hq, hkv, d, bs, maxb, nb, k, first, last, dt, kv, ws, ws_bytes, 0)


def attend(L, out=2 * P, q=P, kc=P, sel=P, qsl=None, n=2, rows=2, hq=32, hkv=8, d=128, bs=16, maxb=40, nb=10, k=8, scale=0.1,
           dt=1, kv=1, ks=1.0, vs=1.0):
    return L.rllm_paged_attention_sparse(out, q, kc, P, P, P, qsl, sel, n, rows, hq, hkv, d, bs, maxb, nb, k, scale, dt, kv, ks,
                                         vs, 0)


SHAPES = [dict(d=120), dict(d=0), dict(d=288), dict(bs=8), dict(bs=48), dict(bs=256), dict(hkv=0), dict(hkv=2048),
          dict(maxb=-1), dict(maxb=1 << 30), dict(nb=-1)]


@pytest.mark.parametrize("call", [bounds, append, select, attend])
def test_shapes_are_refused(call):
    L = rllm_amd.lib()
    for bad in SHAPES:
        if call is bounds and bad.get("maxb") == -1:
            continue                                            # empty work
        assert call(L, **bad) == 1, bad
    assert call(L, n=0) == 0 and call(L, n=-3) == 0
    assert call(L, kv=7) == 1 and call(L, kv=-1) == 1


def test_arguments_are_refused():
    L = rllm_amd.lib()
    for bad in (dict(kb=None), dict(kc=None), dict(bt=None), dict(lens=None), dict(kb=P + 8), dict(kc=P + 2)):
        assert bounds(L, **bad) == 1, bad
    assert bounds(L, maxb=0) == 0
    for bad in (dict(k=None), dict(kc=None), dict(kb=None), dict(lens=None), dict(cos=None), dict(q=None), dict(q_out=None),
                dict(k=P + 8), dict(kc=P + 4), dict(cos=P + 4), dict(q=P + 2), dict(rows=3), dict(hq=-1), dict(maxp=0),
                dict(dt=2), dict(dt=0), dict(kv=2, ks=0.0), dict(kv=2, ks=float("inf")), dict(kv=3, rounding=2)):
        assert append(L, **bad) == 1, bad
    assert append(L, rows=0) == 0
    for bad in (dict(sel=None), dict(q=None), dict(kb=None), dict(bt=None), dict(rows=3), dict(hq=30), dict(hq=0), dict(k=0),
                dict(k=4097), dict(first=-1), dict(last=0), dict(first=8), dict(first=3, last=6), dict(dt=0), dict(dt=3),
                dict(q=P + 8), dict(kb=P + 8), dict(ws=P + 8), dict(ws_bytes=100)):
        assert select(L, **bad) == 1, bad
    for bad in (dict(out=None), dict(q=None), dict(kc=None), dict(sel=None), dict(rows=3), dict(hq=30), dict(k=0), dict(k=4097),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(kv=2, ks=float("nan")), dict(kv=2, vs=float("inf")),
                dict(kv=2, ks=3e38, scale=10.0), dict(dt=0), dict(out=P + 8), dict(kc=P + 8), dict(out=P),
                dict(rows=1 << 25, qsl=P)):
        assert attend(L, **bad) == 1, bad


def test_workspace_size():
    size = rllm_amd.lib().rllm_select_blocks_workspace_size
    assert size(0, 8, 100) == 0
    assert size(-1, 8, 100) == size(4, 0, 100) == size(4, 2048, 100) == size(4, 8, -1) == size(1 << 25, 8, 1) == -1
    rows, widths = (1, 2, 7, 64, 255, 256, 257, 300, 301, 4000, 1 << 20), (0, 1, 63, 64, 65, 511, 512, 513, 2000, 8192, 8193, 100000)
    s = {(r, w): size(r, 8, w) for r in rows for w in widths}
    for (r0, w0), (r1, w1) in itertools.product(s, s):
        if r0 <= r1 and w0 <= w1:
            assert s[r0, w0] <= s[r1, w1], (r0, w0, r1, w1)
    assert all(s[r, w] >= r * 8 * w * 4 or s[r, w] == 1 << 30 for r, w in s)


def test_the_front_end_names_what_is_wrong():
    kc = torch.zeros((4, 2, 64, 16), dtype=torch.bfloat16)
    kb = ops.new_key_bounds(kc)
    assert kb.shape == (4, 2, 2, 64) and kb.dtype == torch.bfloat16
    bt, lens = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q, k = torch.zeros((3, 4, 64), dtype=torch.bfloat16), torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    cos = torch.zeros((10, 32))
    sel = torch.zeros((3, 2, 1), dtype=torch.int32)
    with pytest.raises(ValueError, match="current GPU"):
        ops.key_bounds(kc, kb, bt, lens)
    with pytest.raises(ValueError, match="k_bounds"):
        ops.key_bounds(kc, kb[:3], bt, lens)
    with pytest.raises(ValueError, match="k_bounds"):
        ops.key_bounds(kc, kb.half(), bt, lens)
    with pytest.raises(TypeError, match="int32"):
        ops.key_bounds(kc, kb, bt.long(), lens)
    with pytest.raises(ValueError, match="block_size"):
        ops.key_bounds(kc[..., :8], kb, bt, lens)
    with pytest.raises(ValueError, match="one row a sequence"):
        ops.rope_and_append(None, k[:2], k[:2], kc, kc, kb, bt, lens, cos, cos)
    with pytest.raises(ValueError, match="cos/sin"):
        ops.rope_and_append(q, k, k, kc, kc, kb, bt, lens, cos[:, :16], cos)
    with pytest.raises(ValueError, match="current GPU"):
        ops.rope_and_append(q, k, k, kc, kc, kb, bt, lens, cos, cos)
    with pytest.raises(ValueError, match="q_out without q"):
        ops.rope_and_append(None, k, k, kc, kc, kb, bt, lens, cos, cos, q_out=q)
    with pytest.raises(TypeError, match="16-bit cache"):
        ops.rope_and_append(q.half(), k.half(), k.half(), kc, kc, kb, bt, lens, cos, cos)
    with pytest.raises(ValueError, match="query_start_loc"):
        ops.select_blocks(q, kb, bt, lens, 16, 2, query_start_loc=lens)
    with pytest.raises(TypeError, match="dtype of q"):
        ops.select_blocks(q.half(), kb, bt, lens, 16, 2)
    with pytest.raises(ValueError, match="uint8"):
        ops.select_blocks(q, kb.view(torch.uint8)[..., :64].contiguous(), bt, lens, 16, 2)
    with pytest.raises(ValueError, match="out must be"):
        ops.select_blocks(q, kb, bt, lens, 16, 2, out=sel)
    with pytest.raises(ValueError, match="selected"):
        ops.paged_sparse(q, kc, kc, bt, lens, sel[:2], 0.1)
    with pytest.raises(ValueError, match="must not be q"):
        ops.paged_sparse(q, kc, kc, bt, lens, sel, 0.1, out=q)
    with pytest.raises(ValueError, match="head_dim"):
        ops.paged_sparse(q[..., :32], kc, kc, bt, lens, sel, 0.1)
    with pytest.raises(ValueError, match="current GPU"):
        ops.paged_sparse(q, kc, kc, bt, lens, sel, 0.1)
