"""The decode workspace over the MXFP4 cache: one sized for the largest batch and the widest
table serves every smaller call, and so does the library's own buffer."""
import itertools

import numpy as np
import pytest
import torch

import mxfp4_ref as M
from rllm_amd import ops
from gpu_util import RawStream
from test_gpu_mxfp4_decode import WEIGHT, case, dev_args, reference

pytestmark = pytest.mark.gpu


def size(n, hq, hkv, d, bs, maxb):
    return ops.lib().rllm_paged_attention_decode_mxfp4_workspace_size(n, hq, hkv, d, bs, maxb)


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (8, 1, 64), (16, 4, 256), (48, 1, 32)])
def test_size_never_falls_with_the_batch_or_the_table(dev, hq, hkv, d):
    batches, tables = (1, 2, 31, 64, 127, 128, 129, 256, 700, 1024), (0, 1, 3, 16, 127, 128, 129, 512, 2000)
    s = {(n, t): size(n, hq, hkv, d, 16, t) for n in batches for t in tables}
    for (n0, t0), (n1, t1) in itertools.product(s, s):
        if n0 <= n1 and t0 <= t1:
            assert s[n0, t0] <= s[n1, t1], (n0, t0, n1, t1)
    assert all(size(n, hq, hkv, d, 32, t // 2) <= s[n, t] for n in batches for t in tables)


def test_narrow_tables_on_a_workspace_of_wide_ones(dev):
    # many rows over narrow tables take two-wave workgroups, twice as many as of four
    rng = np.random.default_rng(51)
    lens = rng.integers(1, 150, 150).tolist()
    c = case(rng, lens, 16, 8, 64, 16, "bf16", dev)
    a = dev_args(*c, dev)
    ref = reference(*c, 0.125)
    wide = torch.full((150, 2000), -1, dtype=torch.int32, device=dev)
    wide[:, :a[3].shape[1]] = a[3]
    w = a[:3] + (wide, a[4])
    ws = torch.zeros(size(150, 16, 8, 64, 16, 2000), dtype=torch.uint8, device=dev)
    for args in (w, a, w, a):
        out = ops.paged_decode_mxfp4(*args, 0.125, workspace=ws)
        M.check_attention(out.float().cpu().numpy(), *ref, "bf16", WEIGHT, "one workspace")
    with pytest.raises(Exception):
        ops.paged_decode_mxfp4(*a, 0.125, workspace=ws[:16384 + 1024])
    # the library's buffer, warmed by the wide table, serves a captured narrow call: the
    # eager call's bits, with rows cut between workgroups as there
    lens = [2000] + [30] * 149
    c = case(rng, lens, 16, 8, 64, 16, "bf16", dev)
    a = dev_args(*c, dev)
    wide = torch.full((150, 2000), -1, dtype=torch.int32, device=dev)
    wide[:, :a[3].shape[1]] = a[3]
    eager = ops.paged_decode_mxfp4(*a, 0.125)
    M.check_attention(eager.float().cpu().numpy(), *reference(*c, 0.125), "bf16", WEIGHT, "eager")
    with RawStream() as st:
        st.wait_stream(torch.cuda.current_stream())
        ops.paged_decode_mxfp4(*a[:3], wide, a[4], 0.125, stream=st)
        torch.cuda.synchronize()
        out = torch.zeros_like(eager)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            ops.paged_decode_mxfp4(*a, 0.125, out=out, validate=False)
        for _ in range(3):
            out.fill_(float("nan"))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)
            assert torch.equal(ops.paged_decode_mxfp4(*a, 0.125), eager)
