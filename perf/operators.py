"""The microscaled 4-bit (MXFP4) KV cache and the attention that reads it, as measurable cases.

Five operators: the slot-mapped cache write that quantises as it writes, the
same fused with the rotary embedding, the read of cache rows back to 16 bits,
decode attention and chunked-prefill attention over the cache.

The cache of one layer and one of K / V is uint8 [num_blocks, num_kv_heads,
page], page = block_size * head_dim * 17 / 32 bytes: first block_size rows of
head_dim / 2 bytes (element 2i in the low four bits of byte i, 2i + 1 in the
high ones; sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4,
6), then block_size rows of head_dim / 32 scale bytes e, one per 32 elements.
An element stands for code * 2^(e - 127); e = 255 makes its 32 elements NaN.
A row's block of 32 with largest magnitude a is written with
e = clamp(floor(log2 a) - 2 + 127, 1, 254) and each element as the nearest
code, ties to the even one, at most 6; a block that holds an infinity or a NaN
is written with e = 255 and codes 0.

``own`` false: the plain form of each operator in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
HALF = {"bf16": torch.bfloat16, "f16": torch.float16}
ROPE_THETA = 500000.0
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _write(name, rope, runs, run_min, run_max, hq, hkv, d, bs=16, dtype="bf16", lens=0):
    """runs sequences, each writing run_min..run_max consecutive new tokens."""
    c = {"kind": "rope" if rope else "write", "runs": runs, "run_min": run_min, "run_max": run_max, "hq": hq,
         "hkv": hkv, "d": d, "bs": bs, "dtype": dtype, "lens": lens}
    return dict(c, name=name) if name else c


def _read(name, batch, ctx_min, ctx_max, hkv, d, bs=16, dtype="bf16", lens=0):
    c = {"kind": "read", "batch": batch, "ctx_min": ctx_min, "ctx_max": ctx_max, "hkv": hkv, "d": d, "bs": bs,
         "dtype": dtype, "lens": lens}
    return dict(c, name=name) if name else c


def _decode(name, batch, ctx_min, ctx_max, hq, hkv, d, bs=16, dtype="bf16", lens=0):
    c = {"kind": "decode", "batch": batch, "ctx_min": ctx_min, "ctx_max": ctx_max, "hq": hq, "hkv": hkv, "d": d,
         "bs": bs, "dtype": dtype, "lens": lens}
    return dict(c, name=name) if name else c


def _prefill(name, prompts, new_min, new_max, cached, hq, hkv, d, bs=16, dtype="bf16", lens=0):
    c = {"kind": "prefill", "prompts": prompts, "new_min": new_min, "new_max": new_max, "cached": cached,
         "hq": hq, "hkv": hkv, "d": d, "bs": bs, "dtype": dtype, "lens": lens}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token for each of 64 sequences, written and read back: latency
        _write("write_step", False, 64, 1, 1, 32, 8, 128),
        # a scheduler's step of prompts of uneven length, f16 as in the f16 entry points
        _write("write_prompts", False, 8, 300, 2000, 32, 8, 128, dtype="f16", lens=3),
        # the same step for a model that rotates: q, k and the cache in one pass
        _write("rope_step", True, 64, 1, 1, 32, 8, 128),
        # the rotation and cache write of a chunk of prompts
        _write("rope_chunk", True, 8, 512, 512, 32, 8, 128),
        # one short context taken back to 16 bits (a cache handed to another path)
        _read("read_short", 1, 777, 777, 8, 64, dtype="f16"),
        # a batch of contexts of mixed age taken back to 16 bits
        _read("read_batch", 16, 1000, 8000, 8, 128, bs=32, lens=5),
        # a single chat, where launches and latency count
        _decode("decode_one", 1, 700, 700, 32, 8, 128),
        # a serving batch of chats of mixed age on an 8B-size layer
        _decode("decode_mixed", 64, 128, 4096, 32, 8, 128, lens=2),
        # long documents under a model whose query heads group in threes, f16, 32-token blocks
        _decode("decode_long", 24, 4000, 32000, 24, 8, 128, bs=32, dtype="f16", lens=4),
        # one short fresh prompt of a small model with 64-wide heads
        _prefill("prefill_short", 1, 117, 117, 0, 32, 8, 64, dtype="f16"),
        # a scheduler's chunk of prompts whose first part is cached already
        _prefill("prefill_chunk", 8, 512, 512, 2048, 32, 8, 128),
        # long prompts, a chunk of each at a time: the largest
        _prefill("prefill_long", 2, 1500, 2048, 14000, 32, 8, 128, bs=32, lens=6),
    ]


_HEADS = [(32, 8), (32, 8), (16, 4), (8, 2), (4, 1), (32, 32), (32, 4), (24, 8), (28, 4), (40, 8), (48, 8), (16, 16)]
_DIMS = [64, 96, 128, 128, 128, 192, 256]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "rope", "read", "decode", "decode", "prefill", "prefill"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    bs = rng.choice([16, 16, 32, 64])
    lens = rng.randrange(1 << 16)
    hq, hkv = rng.choice(_HEADS)
    d = rng.choice(_DIMS)
    if kind in ("write", "rope"):
        if kind == "rope":
            d = rng.choice([64, 128, 128, 256])
        if rng.random() < 0.4:   # a decode step: one token per sequence
            return _write(None, kind == "rope", _log_int(rng, 1, 256), 1, 1, hq, hkv, d, bs, dtype, lens)
        runs, run = _log_int(rng, 1, 8), _log_int(rng, 16, 2000)
        while runs * run * hkv * d > 8 * 2000 * 1024:
            run = run * 2 // 3
        return _write(None, kind == "rope", runs, rng.choice([run, max(1, run // 10)]), run, hq, hkv, d, bs, dtype,
                      lens)
    if kind == "read":
        batch, ctx = _log_int(rng, 1, 64), _log_int(rng, 16, 8000)
        while batch * ctx * hkv * d > 16 * 8000 * 1024:
            ctx = ctx * 2 // 3
        return _read(None, batch, rng.choice([ctx, max(1, ctx // 8)]), ctx, hkv, d, bs, dtype, lens)
    if kind == "decode":
        batch, ctx = _log_int(rng, 1, 256), _log_int(rng, 32, 32000)
        while batch * ctx * hkv * d > 24 * 24000 * 1024:
            if ctx > 2048 or batch == 1:
                ctx = ctx * 2 // 3
            else:
                batch = batch * 2 // 3
        return _decode(None, batch, rng.choice([ctx, max(1, ctx // 2), max(1, ctx // 32)]), ctx, hq, hkv, d, bs,
                       dtype, lens)
    prompts, new = _log_int(rng, 1, 8), _log_int(rng, 16, 2048)
    cached = rng.choice([0, _log_int(rng, 16, 14000)])
    while 4.0 * hq * d * prompts * new * (cached + new / 2) > 4e11 or hq * prompts * new * (cached + new) > 2e9:
        if cached > 512:
            cached = cached * 2 // 3
        else:
            new = new * 2 // 3
    return _prefill(None, prompts, rng.choice([new, max(1, new // 20)]), new, cached, hq, hkv, d, bs, dtype, lens)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _lens(case, n, lo, hi):
    r = np.random.default_rng([0x4D58, case["lens"], n, lo, hi])
    return r.integers(lo, hi, size=n, endpoint=True).astype(np.int64)


def _ctx_lens(case):
    return _lens(case, case["batch"], case["ctx_min"], case["ctx_max"])


def _prefill_lens(case):
    new = _lens(case, case["prompts"], case["new_min"], case["new_max"])
    return new, new + case["cached"]


def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed & 0x7FFFFFFF)
    return g


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)


def _keys(g, n, hkv, d, dtype):
    """Keys: some channels of a head are larger than others, as after a projection and a rotation."""
    return (_randn(g, (n, hkv, d)) * torch.exp(0.6 * _randn(g, (1, hkv, d)))).to(dtype)


def _tables(rng, lens, bs):
    """Scattered block ids, as a block pool hands them out: (tables, blocks in the pool)."""
    nblk = [(int(n) + bs - 1) // bs for n in lens]
    pool = int(math.ceil(1.1 * sum(nblk))) + 1
    perm = rng.permutation(pool).astype(np.int32)
    bt = np.full((len(nblk), max(nblk)), -1, np.int32)
    p = 0
    for s, n in enumerate(nblk):
        bt[s, :n] = perm[p:p + n]
        p += n
    return bt, pool


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)


def _fill_caches(case, g, pool):
    """K and V pools of quantised random rows, a part of the blocks at a time."""
    hkv, d, bs = case["hkv"], case["d"], case["bs"]
    page = bs * d * 17 // 32
    chan = torch.exp(0.6 * _randn(g, (1, hkv, d)))
    caches = []
    step = max(1, (1 << 25) // (hkv * d * bs))
    for factor in (chan, None):
        cache = torch.empty((pool, hkv, page), dtype=torch.uint8, device=DEVICE)
        codes, scales = _parts(cache, d, bs)
        for b in range(0, pool, step):
            n = min(step, pool - b)
            x = _randn(g, (n * bs, hkv, d))
            if factor is not None:
                x *= factor
            c, e = _quantise(x)
            codes[b:b + n] = c.view(n, bs, hkv, d // 2).transpose(1, 2)
            scales[b:b + n] = e.view(n, bs, hkv, d // 32).transpose(1, 2)
        caches.append(cache)
    return caches


def _slots(bt, s, p, bs):
    return bt[s, p // bs].astype(np.int64) * bs + p % bs


def prepare(case, seed):
    kind, dt = case["kind"], HALF[case["dtype"]]
    g = _gen(seed)
    rng = np.random.default_rng([seed & 0x7FFFFFFF, 23])
    hkv, d, bs = case["hkv"], case["d"], case["bs"]
    st = {"case": case}
    if kind in ("write", "rope"):
        runs = _lens(case, case["runs"], case["run_min"], case["run_max"])
        # decode tokens land anywhere in their sequence's last block; prompt
        # chunks start at the front of a block, as a scheduler cuts them
        if case["run_max"] == 1:
            start = rng.integers(0, 4096, size=case["runs"])
        else:
            start = rng.integers(0, 4096 // bs, size=case["runs"]) * bs
        first = start // bs * bs
        bt, pool = _tables(rng, start + runs - first, bs)
        slots, pos, back = [], [], []
        for s, n in enumerate(runs.tolist()):
            p = np.arange(start[s], start[s] + n)
            slots.append(_slots(bt, s, p - first[s], bs))
            pos.append(p)
            # the blocks that the run touches, their other rows among them
            back.append(_slots(bt, s, np.arange((start[s] + n - first[s] + bs - 1) // bs * bs), bs))
        st["slots"], st["back"] = _dev(np.concatenate(slots)), _dev(np.concatenate(back))
        n = int(runs.sum())
        st["k"], st["v"] = _keys(g, n, hkv, d, dt), _randn(g, (n, hkv, d), dt)
        st["kc"], st["vc"] = _fill_caches(case, g, pool)
        st["k_out"] = torch.empty((st["back"].numel(), hkv, d), dtype=dt, device=DEVICE)
        st["v_out"] = torch.empty_like(st["k_out"])
        if kind == "rope":
            st["q"] = _randn(g, (n, case["hq"], d), dt)
            st["q_out"] = torch.empty_like(st["q"])
            st["pos"] = _dev(np.concatenate(pos).astype(np.int32))
            inv = ROPE_THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
            ang = torch.arange(8192, dtype=torch.float64)[:, None] * inv[None, :]
            st["cos"], st["sin"] = ang.cos().float().to(DEVICE), ang.sin().float().to(DEVICE)
        return st
    if kind == "read":
        lens = _ctx_lens(case)
        bt, pool = _tables(rng, lens, bs)
        st["back"] = _dev(np.concatenate([_slots(bt, s, np.arange(n), bs) for s, n in enumerate(lens.tolist())]))
        st["kc"], st["vc"] = _fill_caches(case, g, pool)
        st["k_out"] = torch.empty((st["back"].numel(), hkv, d), dtype=dt, device=DEVICE)
        st["v_out"] = torch.empty_like(st["k_out"])
        return st
    if kind == "decode":
        lens = _ctx_lens(case)
        rows = case["batch"]
    else:
        new, lens = _prefill_lens(case)
        rows = int(new.sum())
        st["qsl"] = _dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
    bt, pool = _tables(rng, lens, bs)
    st["q"] = _randn(g, (rows, case["hq"], d), dt)
    st["bt"], st["lens"] = _dev(bt), _dev(lens.astype(np.int32))
    st["kc"], st["vc"] = _fill_caches(case, g, pool)
    st["out"] = torch.empty_like(st["q"])
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _parts(cache, d, bs):
    """The code rows [nb, hkv, bs, d/2] and the scale rows [nb, hkv, bs, d/32] of a cache, as views."""
    nb, hkv, page = cache.shape
    c = bs * d // 2
    codes = cache.as_strided((nb, hkv, bs, d // 2), (hkv * page, page, d // 2, 1), cache.storage_offset())
    scales = cache.as_strided((nb, hkv, bs, d // 32), (hkv * page, page, d // 32, 1), cache.storage_offset() + c)
    return codes, scales


def _quantise(x):
    """f32 [..., d] -> code bytes [..., d/2] and scale bytes [..., d/32]."""
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(b).all(-1, keepdim=True)
    e = (torch.frexp(amax)[1] - 3).clamp(-126, 127)    # frexp's mantissa is in [0.5, 1); of 0 it gives exponent 0
    e = torch.where(amax > 0, e, -126)
    y = torch.where(ok, torch.ldexp(b, -e), 0.0)
    a = y.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = code + 8 * (torch.signbit(y)).to(torch.uint8)
    code = code.flatten(-2)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    return packed, torch.where(ok, e + 127, 255).squeeze(-1).to(torch.uint8)


def _values(codes, scales):
    """Code bytes [..., d/2] and scale bytes [..., d/32] -> f32 [..., d]."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float32, device=codes.device)
    pairs = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    x = table[pairs.int()].unflatten(-1, (-1, 32))
    e = scales.int()
    f = torch.where(e == 255, float("nan"), torch.ldexp(torch.ones((), device=codes.device), e - 127))
    return (x * f.unsqueeze(-1)).flatten(-2)


def _plain_write(case, cache, x, slots):
    codes, scales = _parts(cache, case["d"], case["bs"])
    blk, off = slots // case["bs"], slots % case["bs"]
    c, e = _quantise(x)
    codes[blk, :, off] = c
    scales[blk, :, off] = e


def _plain_read(case, cache, slots):
    codes, scales = _parts(cache, case["d"], case["bs"])
    blk, off = slots // case["bs"], slots % case["bs"]
    return _values(codes[blk, :, off], scales[blk, :, off]).to(HALF[case["dtype"]])


def _plain_rotate(x, cos, sin):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_context(case, cache, bt):
    """The padded contexts f32 [batch, hkv, tokens, d] that the tables name."""
    codes, scales = _parts(cache, case["d"], case["bs"])
    bt = bt.long().clamp(min=0)
    return _values(codes[bt], scales[bt]).transpose(1, 2).flatten(2, 3)


def _plain_attend(q, k, v, last, scale):
    """q f32 [batch, hkv, rows, d] over k, v [batch, hkv, tokens, d]; row r sees tokens 0..last[batch, r]."""
    s = torch.matmul(q, k.transpose(2, 3)) * scale
    seen = torch.arange(k.shape[2], device=q.device) <= last[:, None, :, None]
    s = s.masked_fill_(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    s = s.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    z = s.sum(-1, keepdim=True)
    return torch.matmul(s, v) / torch.where(z == 0, 1.0, z)


def _plain_decode(st):
    case = st["case"]
    b, hq, d = st["q"].shape
    hkv = case["hkv"]
    q = st["q"].float().view(b, hkv, hq // hkv, d)
    k, v = (_plain_context(case, st[c], st["bt"]) for c in ("kc", "vc"))
    last = (st["lens"].long() - 1)[:, None].expand(b, hq // hkv)
    return _plain_attend(q, k, v, last, _scale(case)).reshape(b, hq, d).to(st["q"].dtype)


def _plain_prefill(st):
    case = st["case"]
    t, hq, d = st["q"].shape
    hkv, g = case["hkv"], hq // case["hkv"]
    qsl, lens = st["qsl"].long(), st["lens"].long()
    b, longest = lens.numel(), case["new_max"]
    new = qsl[1:] - qsl[:-1]
    tok = torch.arange(t, device=DEVICE)
    seq = torch.bucketize(tok, qsl[1:], right=True)
    i = tok - qsl[seq]
    q = torch.zeros((b, longest, hkv, g, d), device=DEVICE)
    q[seq, i] = st["q"].float().view(t, hkv, g, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(b, hkv, g * longest, d)
    last = ((lens - new)[:, None] + torch.arange(longest, device=DEVICE)).clamp(max=case["cached"] + longest - 1)
    k, v = (_plain_context(case, st[c], st["bt"]) for c in ("kc", "vc"))
    o = _plain_attend(q, k, v, last.repeat(1, g), _scale(case))
    o = o.view(b, hkv, g, longest, d).permute(0, 3, 1, 2, 4)
    return o[seq, i].reshape(t, hq, d).to(st["q"].dtype)


def _scale(case):
    return 1.0 / math.sqrt(case["d"])


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from rllm_amd import ops
        if kind == "write":
            ops.reshape_and_cache_mxfp4(st["k"], st["v"], st["kc"], st["vc"], st["slots"])
        elif kind == "rope":
            ops.rope_and_cache_mxfp4(st["q"], st["k"], st["v"], st["kc"], st["vc"], st["slots"], st["pos"],
                                     st["cos"], st["sin"], q_out=st["q_out"])
        if kind in ("write", "rope", "read"):
            ops.read_cache_mxfp4(st["kc"], st["vc"], st["back"], out_key=st["k_out"], out_value=st["v_out"])
            return ((st["q_out"],) if kind == "rope" else ()) + (st["k_out"], st["v_out"])
        if kind == "decode":
            return ops.paged_decode_mxfp4(st["q"], st["kc"], st["vc"], st["bt"], st["lens"], _scale(case),
                                          out=st["out"], validate=False)
        return ops.paged_prefill_mxfp4(st["q"], st["kc"], st["vc"], st["bt"], st["lens"], st["qsl"], _scale(case),
                                       out=st["out"], validate=False)
    if kind == "decode":
        return _plain_decode(st)
    if kind == "prefill":
        return _plain_prefill(st)
    first = ()
    if kind in ("write", "rope"):
        k = st["k"].float()
        if kind == "rope":
            cos, sin = (st[t][st["pos"].long()][:, None, :] for t in ("cos", "sin"))
            first = (_plain_rotate(st["q"], cos, sin).to(st["q"].dtype),)
            k = _plain_rotate(st["k"], cos, sin)
        _plain_write(case, st["kc"], k, st["slots"])
        _plain_write(case, st["vc"], st["v"].float(), st["slots"])
    return first + (_plain_read(case, st["kc"], st["back"]), _plain_read(case, st["vc"], st["back"]))


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kind, d = case["kind"], case["d"]
    row16, row4 = case["hkv"] * d * 2 * 2, case["hkv"] * d * 2 * 17 // 32   # K and V of a token
    if kind in ("write", "rope"):
        runs = _lens(case, case["runs"], case["run_min"], case["run_max"])
        n = int(runs.sum())
        back = int(((runs + case["bs"] - 1) // case["bs"]).sum()) * case["bs"]
        per = row16 + row4 + 8
        if kind == "rope":
            per += case["hq"] * d * 4 + d * 4 + 4
        return {"bytes": n * per + back * (row4 + row16 + 8),
                "flops": n * (case["hq"] + case["hkv"]) * d * 3 if kind == "rope" else 0}
    if kind == "read":
        return {"bytes": int(_ctx_lens(case).sum()) * (row4 + row16 + 8), "flops": 0}
    if kind == "decode":
        ctx = _ctx_lens(case).tolist()
        new = [1] * len(ctx)
    else:
        new, ctx = (a.tolist() for a in _prefill_lens(case))
    pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(new, ctx))
    table = sum((c + case["bs"] - 1) // case["bs"] for c in ctx) * 4
    return {"bytes": int(sum(ctx) * row4 + sum(new) * case["hq"] * d * 4 + table + 4 * len(ctx)),
            "flops": int(4 * d * case["hq"] * pairs)}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _exact_round(x):
    """float64 [n, hkv, d] -> the values that the cache holds for them."""
    out = torch.empty_like(x)
    for b in range(0, x.shape[-1], 32):
        y = x[..., b:b + 32]
        a = y.abs().max(dim=-1, keepdim=True).values
        unit = torch.exp2((torch.floor(torch.log2(a.clamp(min=1e-300))) - 2).clamp(-126, 127))
        m = (y / unit).abs()
        step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0)).double()
        out[..., b:b + 32] = torch.sign(y) * torch.clamp(torch.round(m / step) * step, max=6.0) * unit
    return out


def _exact_rows(case, cache, blocks, offs):
    """The rows (blocks[i], offs[i]) of a cache, float64 [n, hkv, d]."""
    d, bs = case["d"], case["bs"]
    pages = cache[blocks]
    at = torch.arange(blocks.numel(), device=cache.device)
    raw = pages[..., :bs * d // 2].reshape(-1, case["hkv"], bs, d // 2)[at, :, offs].long()
    e = pages[..., bs * d // 2:].reshape(-1, case["hkv"], bs, d // 32)[at, :, offs].double()
    out = torch.empty((blocks.numel(), case["hkv"], d), dtype=torch.float64, device=cache.device)
    for half in (0, 1):
        c = (raw >> (4 * half)) & 15
        exp, man = (c >> 1) & 3, (c & 1).double()
        mag = torch.where(exp == 0, man / 2, (1 + man / 2) * torch.exp2((exp - 1).double()))
        out[..., half::2] = torch.where(c >= 8, -mag, mag)
    return out * torch.exp2(e - 127).repeat_interleave(32, dim=-1)


def _exact_back(case, st, new):
    """The rows read back after `new` (float64, or None where it has no 64-bit value) went to the slots."""
    blk, off = st["back"] // case["bs"], st["back"] % case["bs"]
    out = []
    for cache, x in zip((st["kc"], st["vc"]), new):
        if x is None:
            out.append(None)
            continue
        rows = _exact_rows(case, cache, blk, off)
        if x is not False:
            where = torch.full((int(st["back"].max()) + 1,), -1, dtype=torch.long, device=DEVICE)
            where[st["back"]] = torch.arange(st["back"].numel(), device=DEVICE)
            rows[where[st["slots"]]] = _exact_round(x)
        out.append(rows)
    return tuple(out)


def _exact_attend(case, st, q, table, ctx):
    """q [n, hq, d]: the last n of ctx tokens, causal -> float64 [n, hq, d]."""
    n, hq, d = q.shape
    hkv, bs, g = case["hkv"], case["bs"], hq // case["hkv"]
    t = torch.arange(ctx, device=q.device)
    k, v = (_exact_rows(case, st[c], table[t // bs].long(), t % bs).permute(1, 0, 2).contiguous()
            for c in ("kc", "vc"))
    kt = k.transpose(1, 2).contiguous()
    out = torch.empty((n, hq, d), dtype=torch.float64, device=q.device)
    step = max(1, (1 << 27) // (hq * ctx))
    for i in range(0, n, step):
        m = min(step, n - i)
        qq = q[i:i + m].double().view(m, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * m, d)
        s = torch.matmul(qq, kt) * _scale(case)
        pos = torch.arange(ctx - n + i, ctx - n + i + m, device=q.device).repeat(g)
        s.masked_fill_(t[None, None, :] > pos[None, :, None], float("-inf"))
        o = torch.matmul(torch.softmax(s, dim=-1), v)
        out[i:i + m] = o.view(hkv, g, m, d).permute(2, 0, 1, 3).reshape(m, hq, d)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "read":
        return _exact_back(case, st, (False, False))
    if kind == "write":
        return _exact_back(case, st, (st["k"].double(), st["v"].double()))
    if kind == "rope":
        # the rotated keys are rounded to 32 bits before they are quantised: a
        # value at a border of two codes may go either way in 64
        cos, sin = (st[t][st["pos"].long()].double()[:, None, :] for t in ("cos", "sin"))
        a, b = st["q"].double().chunk(2, dim=-1)
        q = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        return (q,) + _exact_back(case, st, (None, st["v"].double()))
    lens = st["lens"].tolist()
    if kind == "decode":
        return torch.cat([_exact_attend(case, st, st["q"][s:s + 1], st["bt"][s], c) for s, c in enumerate(lens)])
    qsl = st["qsl"].tolist()
    return torch.cat([_exact_attend(case, st, st["q"][qsl[s]:qsl[s + 1]], st["bt"][s], c)
                      for s, c in enumerate(lens)])
