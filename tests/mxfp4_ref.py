"""Plain formulation of the MXFP4 KV cache and the attention over it, in 64 bits
(numpy).  Independent of the library: quantisation by distance to the code
values, attention by dense softmax."""
import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def page_bytes(d, bs):
    return bs * d // 2 + bs * d // 32


def quantise(x):
    """float64 [..., d] -> codes uint8 [..., d], scale bytes uint8 [..., d/32]."""
    b = x.reshape(x.shape[:-1] + (-1, 32))
    finite = np.isfinite(b).all(-1)
    safe = np.where(finite[..., None], b, 0.0)
    amax = np.abs(safe).max(-1)
    with np.errstate(divide="ignore"):
        e = np.where(amax > 0, np.floor(np.log2(np.maximum(amax, 1e-320))) - 2, -126.0)
    e = np.clip(e, -126, 127)
    y = np.abs(safe) / np.exp2(e)[..., None]
    dist = np.abs(y[..., None] - VALUES)
    best = dist.min(-1, keepdims=True)
    near = dist == best                      # one code, or two at a tie: take the even one
    first = near.argmax(-1)
    second = 7 - near[..., ::-1].argmax(-1)
    code = np.where(first % 2 == 0, first, second)
    code = np.where(y >= 6, 7, code) + 8 * np.signbit(safe)
    byte = np.where(finite, e + 127, 255)
    code = np.where(finite[..., None], code, 0)
    return code.reshape(x.shape).astype(np.uint8), byte.astype(np.uint8)


def values(codes, scales):
    """codes [..., d], scale bytes [..., d/32] -> float64 [..., d]."""
    v = VALUES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    f = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(f, 32, axis=-1)


class Cache:
    """Code and scale rows of a pool, [nb, hkv, bs, ...], packed into pages by ``pages``."""

    def __init__(self, nb, hkv, d, bs, codes=None, scales=None):
        self.shape = (nb, hkv, d, bs)
        self.codes = np.zeros((nb, hkv, bs, d), np.uint8) if codes is None else codes
        self.scales = np.zeros((nb, hkv, bs, d // 32), np.uint8) if scales is None else scales

    @classmethod
    def random(cls, rng, nb, hkv, d, bs, spread=1.0):
        x = rng.standard_normal((nb, hkv, bs, d)) * np.exp(spread * 0.5 * rng.standard_normal((1, hkv, 1, d)))
        return cls(nb, hkv, d, bs, *quantise(x))

    @classmethod
    def from_pages(cls, pages, d, bs):
        nb, hkv, _ = pages.shape
        c = pages[..., :bs * d // 2].reshape(nb, hkv, bs, d // 2)
        codes = np.stack([c & 15, c >> 4], -1).reshape(nb, hkv, bs, d)
        return cls(nb, hkv, d, bs, codes, pages[..., bs * d // 2:].reshape(nb, hkv, bs, d // 32).copy())

    def pages(self):
        nb, hkv, d, bs = self.shape
        c = (self.codes[..., 0::2] | (self.codes[..., 1::2] << 4)).reshape(nb, hkv, -1)
        return np.concatenate([c, self.scales.reshape(nb, hkv, -1)], -1)

    def write(self, x, slots):
        """Rows x [n, hkv, d] (float64) to the slots; negative or far ones are skipped."""
        nb, hkv, d, bs = self.shape
        c, e = quantise(x)
        for t, s in enumerate(slots):
            if 0 <= s < nb * bs:
                self.codes[s // bs, :, s % bs] = c[t]
                self.scales[s // bs, :, s % bs] = e[t]

    def rows(self, slots):
        """float64 [n, hkv, d]; zeros for skipped slots."""
        nb, hkv, d, bs = self.shape
        out = np.zeros((len(slots), hkv, d))
        for t, s in enumerate(slots):
            if 0 <= s < nb * bs:
                out[t] = values(self.codes[s // bs, :, s % bs], self.scales[s // bs, :, s % bs])
        return out


def attend(q, kc, vc, table, ctx, n, scale):
    """The last n of ctx tokens' queries q [n, hq, d] (float64), causal ->
    (out, out over |v|, sum over d of |q k| scale at its largest), float64."""
    nb, hkv, d, bs = kc.shape
    _, hq, _ = q.shape
    g = hq // hkv
    ctx = min(ctx, len(table) * bs)
    slots = np.array([-1 if not 0 <= table[t // bs] < nb else table[t // bs] * bs + t % bs for t in range(max(ctx, 0))],
                     np.int64)
    pos = np.nonzero(slots >= 0)[0]
    k, v = kc.rows(slots[pos]), vc.rows(slots[pos])
    out, mag, big = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    return _attend(q, k, v, pos, ctx, n, scale, g, out, mag, big)


def _attend(q, k, v, pos, ctx, n, scale, g, out, mag, big):
    for h in range(q.shape[1]):
        kv = h // g
        s = q[:, h] @ k[:, kv].T * scale
        a = np.abs(q[:, h]) @ np.abs(k[:, kv]).T * abs(scale)
        for i in range(n):
            see = pos <= ctx - n + i
            if not see.any():
                continue
            x = s[i, see]
            with np.errstate(invalid="ignore"):
                p = np.exp(x - x.max())
                p /= p.sum()
            out[i, h] = p @ v[see, kv]
            mag[i, h] = p @ np.abs(v[see, kv])
            big[i, h] = a[i, see].max()
    return out, mag, big


# A rounding to 16 bits is off by at most half a step, eps / 2 of the value.
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def check_attention(got, ref, mag, big, kind, weight_err, what):
    """|got - ref| <= half a step of ref (the output's rounding)
    + mag * (weight_err + 2 * 2^-12 big): weights off by weight_err relative to
    themselves, and by the scores' error, which the block-scaled product keeps
    below 2^-12 of the sum of its terms' magnitudes (random codes, terms and scales
    over nine powers of two; a score off by s moves a normalised weight by at most
    2 s).  Subnormal f16 outputs: half their spacing, 2^-25.  Over a whole output
    the errors are of random sign: the 2-norm stays within half a step (plus
    weight_err) of the reference's, plus 2^-12 of mag's for the scores."""
    got = np.asarray(got, np.float64)
    step = HALF_STEP[kind]
    tol = step * np.abs(ref) + mag * (weight_err + 2.0 ** -11 * big[..., None]) + (2.0 ** -25 if kind == "f16" else 0)
    err = np.abs(got - ref)
    assert np.isfinite(got).all(), f"{what}: non-finite output"
    assert (err <= tol).all(), f"{what}: max err {err.max():.3e}, {int((err > tol).sum())} of {err.size} past the tolerance"
    norm = np.linalg.norm(ref)
    off = np.linalg.norm(got - ref)
    assert off <= (step + weight_err) * norm + 2.0 ** -12 * np.linalg.norm(mag) + 1e-30, \
        f"{what}: 2-norm off by {off / max(norm, 1e-30):.3e}"
