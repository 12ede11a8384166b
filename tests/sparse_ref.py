"""Plain formulation, in 64 bits, of attention over selected cache blocks: the bounds of a
block's keys, the append, the selection and the attention.  Torch on the CPU, a row at a
time, written from the operators' definitions alone."""
import math

import numpy as np
import torch

import oracle as O
import rllm_amd

HALF = {"bf16": torch.bfloat16, "f16": torch.float16}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
CODE = {"e4m3": rllm_amd.DTYPE_FP8_E4M3, "e5m2": rllm_amd.DTYPE_FP8_E5M2}
ORACLE = {"bf16": O.BF16, "f16": O.F16, "e4m3": O.FP8_E4M3, "e5m2": O.FP8_E5M2}
TYPES = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e5m2"), ("f16", "e4m3"), ("bf16", "e5m2")]


def fp8(kv):
    """Keyword arguments that an FP8 cache needs."""
    return {"kv_dtype": CODE[kv]} if kv in CODE else {}


def store(x, kv):
    """f32 values to a cache tensor as the framework takes it (FP8: bytes, to the nearest)."""
    if kv in HALF:
        return x.to(HALF[kv])
    big = 448.0 if kv == "e4m3" else 57344.0
    return x.clamp(-big, big).to(FP8[kv]).view(torch.uint8)


def values(t, kv):
    """What a cache tensor holds, float64 on the CPU."""
    t = t.detach().cpu()
    return (t.view(FP8[kv]) if kv in FP8 else t).double()


def tables(rng, lens, bs, spare=3, width=0):
    """(block tables int32 [n, width], blocks in the pool): scattered distinct blocks."""
    nblk = [(max(int(n), 0) + bs - 1) // bs for n in lens]
    nb = sum(nblk) + spare
    perm = rng.permutation(nb)
    bt = np.full((len(nblk), max(max(nblk), 1, width)), -1, np.int32)
    p = 0
    for s, n in enumerate(nblk):
        bt[s, :n] = perm[p:p + n]
        p += n
    return torch.from_numpy(bt), nb


def rows(lens, qsl, num_rows):
    """(row, sequence, position) of every row that a sequence has."""
    out = []
    for s, L in enumerate(lens):
        a, b = (s, s + 1) if qsl is None else (int(qsl[s]), int(qsl[s + 1]))
        out += [(t, s, int(L) - (b - t)) for t in range(a, min(b, num_rows))]
    return out


def usable(bt, s, j, nb):
    return 0 <= j < bt.shape[1] and 0 <= int(bt[s, j]) < nb


def bounds(kb, kc, bt, lens, bs, first=None):
    """The bounds after key_bounds: kb float64 [nb, hkv, 2, d] before, kc float64 [nb, hkv, d, bs]."""
    kb = kb.clone()
    for s, L in enumerate(lens):
        for j in range(min((max(int(L), 0) + bs - 1) // bs, bt.shape[1])):
            if first is not None and (j + 1) * bs <= int(first[s]):
                continue
            if usable(bt, s, j, kc.shape[0]):
                x = kc[int(bt[s, j])][:, :, :min(int(L) - j * bs, bs)]
                kb[int(bt[s, j])] = torch.stack((x.amin(2), x.amax(2)), 1)
    return kb


def rotate(x, pos, cos, sin):
    """f32 [h, d] at a position: each product and the sum rounded to f32."""
    p = min(max(pos, 0), cos.shape[0] - 1)
    a, b = x.float().chunk(2, -1)
    c, s = cos[p], sin[p]
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def encode(x, kv, scale, nearest):
    if kv in HALF:
        return x.to(HALF[kv])
    y = (x / scale).contiguous().numpy()
    e = O.encode_fp8_rne(y, ORACLE[kv]) if nearest else O.encode(y, ORACLE[kv])
    return torch.from_numpy(e)


def append(q, k, v, kc, vc, kb, bt, lens, qsl, cos, sin, kv, k_scale=1.0, v_scale=1.0, nearest=False):
    """Appends in place into CPU copies (cache tensors as the framework takes them, kb float64); returns
    the rotated q (rows that no sequence has: zeros)."""
    nb, hkv, d, bs = kc.shape
    q_out = torch.zeros_like(q)
    started = {}
    for t, s, pos in rows(lens, qsl, k.shape[0]):
        q_out[t] = rotate(q[t], pos, cos, sin).to(q.dtype)
        j = pos // bs
        if pos < 0 or not usable(bt, s, j, nb):
            continue
        b, off = int(bt[s, j]), pos % bs
        kc[b, :, :, off] = encode(rotate(k[t], pos, cos, sin), kv, k_scale, nearest)
        vc[b, :, :, off] = encode(v[t].float(), kv, v_scale, nearest)
        x = values(kc[b, :, :, off], kv)
        if off == 0:
            kb[b, :, 0], kb[b, :, 1] = x, x
        else:
            kb[b, :, 0], kb[b, :, 1] = torch.minimum(kb[b, :, 0], x), torch.maximum(kb[b, :, 1], x)
        started[b] = True
    return q_out


def scores(q, kb):
    """q float64 [g, d], kb float64 [n, 2, d] -> [n]."""
    x = q[None] * kb[:, 0, None]
    y = q[None] * kb[:, 1, None]
    return torch.maximum(x, y).sum(-1).amax(1)


def select(q, kb, bt, lens, qsl, bs, k, first, last):
    """The lists [rows, hkv, k]; rows that no sequence has are -7.  kb float64."""
    n, hq, d = q.shape
    nb, hkv = kb.shape[:2]
    out = torch.full((n, hkv, k), -7, dtype=torch.int32)
    for t, s, pos in rows(lens, qsl, n):
        nv = 0 if pos < 0 else min(pos // bs + 1, bt.shape[1])
        ok = [j for j in range(nv) if usable(bt, s, j, nb)]
        for h in range(hkv):
            if nv <= k:
                took = ok
            else:
                took = [j for j in ok if j < first or j >= nv - last]
                rest = [j for j in ok if first <= j < nv - last]
                qg = q[t].double().view(hkv, hq // hkv, d)[h]
                sc = scores(qg, kb[bt[s, rest].long(), h]).tolist() if rest else []
                rank = sorted(zip(rest, sc), key=lambda e: (0 if math.isnan(e[1]) else 1, -e[1] if not math.isnan(e[1]) else 0, e[0]))
                took = sorted(took + [j for j, _ in rank[:k - len(took)]])
            out[t, h, :len(took)] = torch.tensor(took, dtype=torch.int32)
            out[t, h, len(took):] = -1
    return out


def attend(q, kc, vc, bt, lens, qsl, sel, scale, k_scale=1.0, v_scale=1.0):
    """(outputs, sum of |weight value|, largest sum of |scale q k|, keys), float64 [rows, hq, ...]; rows that no
    sequence has: NaN.  kc, vc float64."""
    n, hq, d = q.shape
    nb, hkv, _, bs = kc.shape
    g = hq // hkv
    out = torch.full((n, hq, d), float("nan"), dtype=torch.float64)
    mag, spread = torch.zeros((n, hq, d), dtype=torch.float64), torch.zeros((n, hq, 1), dtype=torch.float64)
    for t, s, pos in rows(lens, qsl, n):
        for h in range(hkv):
            keys, before = [], -1
            for j in sel[t, h].tolist():
                if j <= before:
                    break
                if usable(bt, s, j, nb) and j * bs <= pos:
                    keys += [(int(bt[s, j]), o) for o in range(min(bs, pos + 1 - j * bs))]
                before = j
            hs = slice(h * g, (h + 1) * g)
            if not keys:
                out[t, hs] = 0
                continue
            b, o = (torch.tensor(x) for x in zip(*keys))
            kk, vv = kc[b, h, :, o] * k_scale, vc[b, h, :, o] * v_scale
            qg = q[t, hs].double()
            p = torch.softmax(qg @ kk.T * scale, -1)
            out[t, hs] = p @ vv
            mag[t, hs] = p @ vv.abs()
            spread[t, hs] = ((qg.abs() @ kk.abs().T) * abs(scale)).amax(-1, keepdim=True)
    return out, mag, spread


def check_attend(got, ref, mag, spread, kind, d, keys, what=""):
    """Half a step of the output's rounding; and of the values' weighted magnitude: the scores' error (D + 8 roundings of
    2^-24 relative to sum |q k|, twice, as a score and its maximum move), the pair of 16-bit terms of a weight
    (2^-16), the f32 sums (2^-23 a key for numerator and denominator) and 2^-20 for exp2."""
    got, half = got.detach().cpu().double(), torch.finfo(HALF[kind]).eps / 2
    rel = 2 * (d + 8) * 2.0 ** -24 * spread + 2.0 ** -16 + keys * 2.0 ** -23 + 2.0 ** -20
    tol = ref.abs() * half + mag * rel * (1 + half) + torch.finfo(HALF[kind]).smallest_normal * half
    live = ~torch.isnan(ref)
    off = ((got - ref).abs() / tol)[live]
    assert torch.isfinite(got[live]).all(), what
    assert off.numel() == 0 or float(off.max()) <= 1.0, (what, float(off.max()))


def same_values(a, b):
    return bool(((a == b) | (a.isnan() & b.isnan())).all())
