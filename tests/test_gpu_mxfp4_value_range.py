"""Values at both ends of the MXFP4 cache's range, under softmax weights that are taken
against a running max behind the true one: sums of large values stay finite where the
weights' own would, and the smallest values keep their bits."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
from rllm_amd import ops
from gpu_util import log_case

pytestmark = pytest.mark.gpu
HQ, HKV, D, BS = 8, 2, 128, 16


# rise: scores of a half of the 64-key tiles, in log2, above the others'; the running maxima
# of decode and short chunks follow from 8 on, those of long chunks from a lane's sum of 2^8
@pytest.mark.parametrize("end", ["large", "small"])
@pytest.mark.parametrize("seqs,new,ctx,rise", [(1, 0, 700, 7.0), (200, 0, 700, 7.0), (2, 0, 9000, 7.0),
                                               (60, 4, 700, 7.0), (1, 300, 700, 7.0), (1, 300, 1500, 2.9),
                                               (3, 700, 1500, 2.9), (1, 90, 4000, 2.9)])
def test_values_at_the_ends_of_the_range(dev, seqs, new, ctx, rise, end):
    rng = np.random.default_rng(ctx + new)
    nb = (ctx + BS - 1) // BS
    kc, vc = M.Cache(nb, HKV, D, BS), M.Cache(nb, HKV, D, BS)
    high = np.repeat(rng.random(ctx // 64 + 1) < 0.5, 64)[:nb * BS].reshape(nb, 1, BS, 1)
    kc.codes[...] = np.where(high, 2, 0)                         # 1 or 0
    kc.scales[...] = 127
    scale = rise * np.log(2.0) / D                               # queries of ones
    vc.codes[...] = 2 + rng.integers(0, 2, vc.codes.shape)       # 1 or 1.5
    # ctx * 1.5 * 2^e < 2^128, past it with weights of 2^rise; or the smallest scale a write makes
    vc.scales[...] = 127 + 127 - int(np.ceil(np.log2(ctx))) if end == "large" else 1
    n = max(new, 1)
    bt = np.arange(nb, dtype=np.int32)
    ref = M.attend(np.ones((n, HQ, D)), kc, vc, bt, ctx, n, scale)
    q = torch.ones((seqs * n, HQ, D), dtype=torch.bfloat16, device=dev)
    a = (q, *(torch.from_numpy(x).to(dev) for x in (kc.pages(), vc.pages(), np.tile(bt, (seqs, 1)),
                                                    np.full(seqs, ctx, np.int32))))
    what = f"{end} values seqs={seqs} new={new} ctx={ctx}"
    log_case(what)
    if new:
        qsl = torch.arange(seqs + 1, dtype=torch.int32, device=dev) * new
        out = ops.paged_prefill_mxfp4(*a, qsl, scale)
    else:
        out = ops.paged_decode_mxfp4(*a, scale)
    # one or two bf16 terms a weight
    M.check_attention(out.float().cpu().numpy(), *(np.tile(x, (seqs,) + (1,) * (x.ndim - 1)) for x in ref), "bf16",
                      2.0 ** -8 if new else 2.0 ** -16, what)
