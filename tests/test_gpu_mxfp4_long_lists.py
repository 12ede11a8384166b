"""Attention over the MXFP4 cache without scratch (captured on a stream that the library has
not seen), a workgroup a row, where the list of all rows' 32-token items comes close to the
2^31 that it is counted in: the workgroup of the last, longest row stops at its end."""
import numpy as np
import pytest
import torch

import mxfp4_ref as M
from rllm_amd import ops
from gpu_util import RawStream, log_case

pytestmark = pytest.mark.gpu
WEIGHT = 2.0 ** -16     # two bf16 terms a weight
ROWS, BLOCKS, BS, D = 4000, 4194, 4096, 32
ITEMS = BLOCKS * BS // 32


@pytest.mark.parametrize("chunks", [False, True])
def test_last_row_of_a_list_near_its_limit(dev, chunks):
    assert ROWS * (ITEMS + 9) < 2 ** 31 < (ROWS + 1) * ITEMS     # allowed; one row more would not be
    rng = np.random.default_rng(41)
    kc, vc = M.Cache.random(rng, 4, 1, D, BS), M.Cache.random(rng, 4, 1, D, BS)
    q = torch.from_numpy(rng.standard_normal((ROWS, 1, D))).bfloat16().to(dev)
    lens = rng.integers(1, 100, ROWS).astype(np.int32)
    lens[-1] = BLOCKS * BS
    bt = torch.full((ROWS, BLOCKS), -1, dtype=torch.int32, device=dev)
    bt[:, 0] = 1
    bt[-1, 0], bt[-1, -1] = 2, 3         # all between them is missing
    a = (q, *(torch.from_numpy(x).to(dev) for x in (kc.pages(), vc.pages())), bt, torch.from_numpy(lens).to(dev))
    out = torch.zeros_like(q)
    log_case(f"list near 2^31, chunks={chunks}")
    with RawStream() as st:
        st.wait_stream(torch.cuda.current_stream())
        qsl = torch.arange(ROWS + 1, dtype=torch.int32, device=dev)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            if chunks:
                ops.paged_prefill_mxfp4(*a, qsl, 0.18, out=out, validate=False)
            else:
                ops.paged_decode_mxfp4(*a, 0.18, out=out, validate=False)
        x = q.cpu().double().numpy()
        one = np.array([1], np.int32)
        parts = [M.attend(x[s:s + 1], kc, vc, one, int(lens[s]), 1, 0.18) for s in range(ROWS - 1)]
        parts.append(M.attend(x[-1:], kc, vc, np.array([2, 3], np.int32), 2 * BS, 1, 0.18))
        ref = [np.concatenate([p[i] for p in parts]) for i in range(3)]
        for i in range(2):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            M.check_attention(out.float().cpu().numpy(), *ref, "bf16", WEIGHT, f"replay {i}")
