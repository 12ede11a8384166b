"""Sizes of the operators over selected blocks that the host refuses before any launch."""
import rllm_amd

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
