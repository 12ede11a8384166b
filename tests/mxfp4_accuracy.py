"""How exact the attention over the MXFP4 cache is before its output is rounded, from
64 bits (numpy): a bound that the loss of one term of a query or a weight does not pass.

An output is RN(o + e), o the exact value, e what the kernel's own arithmetic adds.  Where e
is small against ulp, the spacing of the output's type, the output mostly equals RN(o), and
differs by one step with probability |e| / ulp: over a position of o in its step that is
even, E (got - RN(o))^2 = ulp^2 (k^2 + f (2k + 1)) <= e^2 + ulp |e| for |e| = (k + f) ulp.
What e is made of, as standard deviations over independent errors a key:

  weights   w sqrt(sum_j p_j^2 v_j^2).  A rounding to bf16 (8 bits) is off by an even error of
            at most 2^-8 of the value, deviation 2^-8 / sqrt(3): w = that for one term, and
            the product of two such for the second term of two, 2^-16 / 3.
  scores    s sqrt(sum_j p_j^2 (v_j - o)^2), s the error of a score: 2^-16 of the scores' rms
            (the block-scaled product's sums, four times what random tiles show; the query's
            terms are exact here) and 2^-20 (f32 products with the scale and differences of
            exponents up to 2^4 at 2^-24 each).
  sums      2^-21 |o|: a few f32 roundings of 2^-24 and exp2's.

The 2-norm of got - RN(o) over an output may be twice what these give: the bound's own
fluctuation (tens of steps or more are off in every case tested) and the errors that are
not quite independent.  Losing the second weight term makes w 400 times as large, a query
term s a hundred times or more: norms 6 to 100 times what the bound gives."""
import numpy as np
import torch

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
BITS = {"bf16": 7, "f16": 10}
ONE_TERM, TWO_TERMS = 2.0 ** -8 / np.sqrt(3), 2.0 ** -16 / 3


def rounded(x, kind):
    return torch.from_numpy(np.ascontiguousarray(x, np.float64)).to(DT[kind]).double().numpy()


def visible(kc, vc, table, ctx):
    """Keys and values float64 [ctx, hkv, d] of a sequence whose blocks are all there."""
    bs = kc.shape[3]
    t = np.arange(ctx)
    slots = table[t // bs].astype(np.int64) * bs + t % bs
    return kc.rows(slots), vc.rows(slots)


def exact(q, k, v, n, scale, weight):
    """q [n, hq, d], the last n of the keys' tokens (float64) -> o and e's deviation [n, hq, d]."""
    ctx, hkv, d = k.shape
    hq = q.shape[1]
    out, dev = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(hq):
        s = q[:, h] @ k[:, h // (hq // hkv)].T * scale
        x = v[:, h // (hq // hkv)]
        seen = np.arange(ctx)[None, :] <= ctx - n + np.arange(n)[:, None]
        rms = np.sqrt((s * s * seen).sum(1, keepdims=True) / seen.sum(1, keepdims=True))
        p = np.exp(np.where(seen, s, -np.inf) - np.where(seen, s, -np.inf).max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        p2 = p * p
        o, v2, v1 = p @ x, p2 @ (x * x), p2 @ x
        spread = np.sqrt(np.maximum(v2 - 2 * o * v1 + o * o * p2.sum(1, keepdims=True), 0.0))
        out[:, h] = o
        dev[:, h] = weight * np.sqrt(v2) + (2.0 ** -16 * rms + 2.0 ** -20) * spread + 2.0 ** -21 * np.abs(o)
    return out, dev


def excess(got, out, dev, kind):
    """The 2-norm of got - RN(out) against what dev gives; a kernel stays below 2."""
    with np.errstate(divide="ignore"):
        ulp = np.exp2(np.maximum(np.floor(np.log2(np.abs(out))), -14.0 if kind == "f16" else -126.0) - BITS[kind])
    off = np.asarray(got, np.float64) - rounded(out, kind)
    return np.linalg.norm(off) / np.sqrt((dev * dev + ulp * dev).sum())


# ---- the kernels' arithmetic with a given number of terms, on the CPU ----

def query_terms(q, terms):
    """Rows q (float64, 16-bit values) as the sum of `terms` E4M3 values a row's power of two apart."""
    amax = np.abs(q).max(-1, keepdims=True)
    unit = np.exp2(np.floor(np.log2(np.maximum(amax, 1e-300))) - 7)
    rest, total = q / unit, np.zeros_like(q)
    for t in range(terms):
        x = torch.from_numpy(rest).float().to(torch.float8_e4m3fn).double().numpy()
        total += x * 16.0 ** -t
        rest = (rest - x) * 16
    return total * unit


def weight_terms(p, terms):
    total = np.zeros_like(p)
    for _ in range(terms):
        total += rounded(p - total, "bf16")
    return total


def emulate(q, k, v, n, scale, kind, q_terms, p_terms):
    ctx, hkv, d = k.shape
    hq = q.shape[1]
    out = np.zeros(q.shape)
    for h in range(hq):
        s = query_terms(q[:, h], q_terms) @ k[:, h // (hq // hkv)].T * scale
        seen = np.arange(ctx)[None, :] <= ctx - n + np.arange(n)[:, None]
        s = np.where(seen, s, -np.inf)
        p = np.exp(s - s.max(1, keepdims=True))
        out[:, h] = weight_terms(p, p_terms) @ v[:, h // (hq // hkv)] / p.sum(1, keepdims=True)
    return rounded(out, kind)
