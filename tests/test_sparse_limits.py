"""Sizes and lists of the operators over selected blocks that the host refuses before any launch."""
import pytest
import torch

import rllm_amd
from rllm_amd import ops

P = 0x1000   # never dereferenced: validation fails first
INVALID = 1


def attend(rows, hq, hkv, qsl=P, n=1, maxb=40):
    return rllm_amd.lib().rllm_paged_attention_sparse(2 * P, P, P, P, P, P, qsl, P, n, rows, hq, hkv, 128, 16, maxb, 10, 8, 0.1, 1, 1,
                                                      1.0, 1.0, 0)


def append(rows, hq, hkv):
    return rllm_amd.lib().rllm_rope_cache_append(P, P, P, P, P, P, P, P, P, P, P, P, 1, rows, hq, hkv, 128, 16, 40, 10, 100, 1, 1, 1.0,
                                                 1.0, 0, 0)


def test_launches_past_the_limit_of_threads_are_refused():
    for rows, hq, hkv in ((1 << 24, 1, 1), (1 << 21, 8, 8), (1 << 18, 1024, 1), (1 << 22, 64, 64), (1 << 24, 1024, 1024)):
        assert attend(rows, hq, hkv, None, rows) == INVALID, (rows, hq, hkv)
        assert attend(rows, hq, hkv, n=rows // 2 + 1) == INVALID, (rows, hq, hkv)
    for rows, hq, hkv in ((1 << 24, 32, 8), (1 << 24, 0, 17), (1 << 23, 1, 17), (1 << 20, 1024, 1024)):
        assert append(rows, hq, hkv) == INVALID, (rows, hq, hkv)


def test_lists_that_do_not_rise_or_go_on_after_their_end_are_refused():
    for good in ([0, 3, 9], [4, -1, -1], [-1, -1, -1], [7, 8, -1], [5]):
        ops._validate_lists(torch.tensor(good, dtype=torch.int32)[None, None])
    for bad in ([-1, 3, -1], [2, -1, 3], [-7, -7, 0], [3, 3, -1], [4, 2, 5], [0, 1, 0]):
        with pytest.raises(ValueError, match="must rise"):
            ops._validate_lists(torch.tensor([[1, 2, 3], bad], dtype=torch.int32)[:, None])
