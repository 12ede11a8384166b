"""Chunks over the MXFP4 cache whose contexts are far shorter than their new tokens, in
batches whose query tiles go by falling key counts: rows without a key are zeros."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
from rllm_amd import ops
from gpu_util import log_case
from test_gpu_mxfp4_prefill import WEIGHT, case, dev_args, reference

pytestmark = pytest.mark.gpu


# (new tokens, contexts, q heads, kv heads, head_dim): more workgroups than the GPU has CUs,
# at most four rounds, and contexts more than a key tile (64) short of the new tokens
@pytest.mark.parametrize("new,ctx,hq,hkv,d,kind", [
    ([300, 600, 700], [0, 100, 500], 32, 32, 64, "bf16"),
    ([300, 600, 700], [236, 535, 636], 32, 32, 64, "f16"),       # one step of keys short, and less
    ([200, 333, 900], [200, 1, 0], 32, 16, 256, "f16"),
    ([512] * 8, [512, 0, 300, 447, 448, 449, 64, 900], 32, 8, 32, "bf16"),
])
def test_rows_without_keys_in_a_longest_first_batch(dev, new, ctx, hq, hkv, d, kind):
    rng = np.random.default_rng(sum(ctx) + d)
    c = case(rng, new, ctx, hq, hkv, d, 16, kind, dev)
    what = f"no keys new={new} ctx={ctx} hq={hq} hkv={hkv} d={d} {kind}"
    log_case(what)
    out = torch.full_like(c[0], float("nan"))
    ops.paged_prefill_mxfp4(*dev_args(*c, dev), 1 / np.sqrt(d), out=out)
    ref, mag, big = reference(*c, 1 / np.sqrt(d))
    M.check_attention(out.float().cpu().numpy(), ref, mag, big, kind, WEIGHT[kind], what)
    qsl = c[5]
    for s, (n, x) in enumerate(zip(new, ctx)):
        assert not out[qsl[s]:qsl[s] + max(n - x, 0)].view(torch.int16).any()
