"""Chunks over selected blocks where their tiles of rows can go wrong: long lists, wide tables and long sequences, against the
formulas in 64 bits (tests/sparse_ref.py)."""
import numpy as np
import pytest
import torch

import sparse_ref as S
from gpu_util import log_case
from rllm_amd import ops

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
