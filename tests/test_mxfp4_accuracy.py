"""The bound on the MXFP4 attention's own error (tests/mxfp4_accuracy.py) holds for the
kernels' arithmetic and not for the same with a term of a query or of a weight left out."""
import numpy as np
import pytest

import mxfp4_accuracy as A
import mxfp4_ref as M


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("ctx,n,hq,hkv,d", [(700, 1, 32, 8, 128), (1023, 1, 24, 8, 64), (2000, 1, 32, 8, 256),
                                            (9001, 1, 32, 4, 128), (300, 5, 8, 2, 96)])
def test_a_lost_term_passes_the_bound(kind, ctx, n, hq, hkv, d):
    rng = np.random.default_rng(ctx + d)
    nb = (ctx + 15) // 16
    kc, vc = M.Cache.random(rng, nb, hkv, d, 16), M.Cache.random(rng, nb, hkv, d, 16)
    k, v = A.visible(kc, vc, rng.permutation(nb), ctx)
    q = A.rounded(rng.standard_normal((n, hq, d)), kind)
    scale, terms = 1 / np.sqrt(d), 2 if kind == "bf16" else 3
    out, dev = A.exact(q, k, v, n, scale, A.TWO_TERMS)
    assert A.excess(A.emulate(q, k, v, n, scale, kind, terms, 2), out, dev, kind) < 1
    for q_terms, p_terms in ((terms, 1), (terms - 1, 2), (terms - 1, 1)):
        assert A.excess(A.emulate(q, k, v, n, scale, kind, q_terms, p_terms), out, dev, kind) > 2, (q_terms, p_terms)
    # one weight term is what long bf16 chunks have, and no less
    out, dev = A.exact(q, k, v, n, scale, A.ONE_TERM)
    assert A.excess(A.emulate(q, k, v, n, scale, kind, terms, 1), out, dev, kind) < 1
    assert A.excess(A.emulate(q, k, v, n, scale, kind, 1, 1), out, dev, kind) > 2
