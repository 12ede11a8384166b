"""Attention over the MXFP4 cache on the GPU within the bound of tests/mxfp4_accuracy.py:
every route with all its terms of queries and weights."""
import numpy as np
import pytest
import torch

import mxfp4_accuracy as A
from rllm_amd import ops
from gpu_util import log_case
from test_gpu_mxfp4_decode import case as decode_case, dev_args as decode_args
from test_gpu_mxfp4_prefill import case, dev_args

pytestmark = pytest.mark.gpu


def check(out, c, new, scale, kind, weight, what):
    q, kc, vc, bt, lens = c[:5]
    x, got = q.cpu().double().numpy(), out.cpu().double().numpy()
    parts, p = [], 0
    for s, n in enumerate(new):
        parts.append(A.exact(x[p:p + n], *A.visible(kc, vc, bt[s], int(lens[s])), n, scale, weight))
        p += n
    e = A.excess(got, *(np.concatenate([y[i] for y in parts]) for i in range(2)), kind)
    print(f"[excess] {what}: {e:.2f}", flush=True)
    assert e < 2, f"{what}: {e:.2f} times the bound"


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("lens,hq,hkv,d", [
    ([700], 32, 8, 128),
    ([1023, 64, 5], 24, 8, 64),
    ([2000], 32, 8, 256),
    ([9001, 333], 32, 4, 128),                # cut between workgroups
    ([40, 130, 90] * 45, 32, 8, 96),          # many short rows: workgroups of two waves
])
def test_decode(dev, kind, lens, hq, hkv, d):
    c = decode_case(np.random.default_rng(sum(lens) + d), lens, hq, hkv, d, 16, kind, dev)
    what = f"decode lens={lens[:3]} hq={hq} hkv={hkv} d={d} {kind}"
    log_case(what)
    out = ops.paged_decode_mxfp4(*decode_args(*c, dev), 1 / np.sqrt(d))
    check(out, c, [1] * len(lens), 1 / np.sqrt(d), kind, A.TWO_TERMS, what)


# (new tokens, contexts, heads, head_dim, table width in tokens or 0, weight terms of bf16): short
# chunks and calls over short tables have two terms, long chunks one; f16 two in all
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("new,ctx,hq,hkv,d,width,terms", [
    ([120], [600], 32, 8, 64, 0, 2),
    ([4] * 64, [500 + 3 * s for s in range(64)], 32, 8, 128, 1200, 2),
    ([300, 70], [1500, 2000], 32, 8, 128, 0, 1),               # keys split between workgroups
    ([500] * 5, [1100 + 10 * s for s in range(5)], 32, 8, 64, 0, 1),
    ([150] * 9, [1200] * 9, 16, 4, 256, 0, 1),
])
def test_chunks(dev, kind, new, ctx, hq, hkv, d, width, terms):
    c = case(np.random.default_rng(sum(ctx) + d), new, ctx, hq, hkv, d, 16, kind, dev, width // 16 or None)
    what = f"chunks new={new[:3]} ctx={ctx[:3]} hq={hq} hkv={hkv} d={d} {kind}"
    log_case(what)
    out = ops.paged_prefill_mxfp4(*dev_args(*c, dev), 1 / np.sqrt(d))
    check(out, c, new, 1 / np.sqrt(d), kind, A.ONE_TERM if terms == 1 and kind == "bf16" else A.TWO_TERMS, what)
