"""Attention over selected cache blocks, and the cache that says which to select, as measurable cases.

Four operators over the paged 16-bit and FP8 caches [num_blocks, num_kv_heads,
head_dim, block_size]:

bounds  For every block that a sequence's keys 0 .. seq_len - 1 reach, the smallest
        and the largest key of each channel over the rows that hold keys:
        k_bounds [num_blocks, num_kv_heads, 2, head_dim], in the cache's own type.
append  The new tokens' rotation (by halves, in f32), their write into the caches at
        the places that the block table gives, and the bounds of the blocks written.
select  For each query (the last n tokens of a sequence; n = 1 in a decode step) and
        kv head, the blocks to attend: of the nv = ceil(len / block_size) blocks
        that the query sees, the first num_first, the last num_last and, by falling
            score(b) = max over the group's heads of sum_d max(q_d lo_bd, q_d hi_bd),
        as many others as num_selected leaves room for; of equal ones the lowest.
        The score is an upper bound of q . k over the block's keys.  Block numbers
        rise along a list, -1 fills it up.
attend  softmax(scale * q . K) V over the keys of the listed blocks that the query sees.

``own`` false: the plain form of each operator in elementary torch operations.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
HALF = {"bf16": torch.bfloat16, "f16": torch.float16}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
ROPE_THETA = 500000.0
K_SCALE, V_SCALE = 0.125, 0.0234375   # an FP8 cache's scales: 448 of them hold the largest key and value
FIRST, LAST = 1, 2                       # blocks of a sequence that every query attends


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _case(name, kind, batch, ctx_min, ctx_max, new_min=0, new_max=0, hq=32, hkv=8, d=128, bs=16, dtype="bf16", kv="",
          k=0, lens=0):
    """batch sequences of ctx_min..ctx_max cached tokens, and new_min..new_max new ones each (in append and,
    where not 0, in select and attend, whose queries they are); kv "": a cache of dtype."""
    c = {"kind": kind, "batch": batch, "ctx_min": ctx_min, "ctx_max": ctx_max, "new_min": new_min, "new_max": new_max,
         "hq": hq, "hkv": hkv, "d": d, "bs": bs, "dtype": dtype, "kv": kv, "k": k, "lens": lens}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one sequence whose blocks came back from host memory without their bounds
        _case("bounds_swap", "bounds", 1, 777, 777, d=64, dtype="f16"),
        # a batch whose caches another write filled, 32-token blocks
        _case("bounds_batch", "bounds", 16, 1000, 8000, bs=32, lens=1),
        # one new token for each of 64 sequences: latency
        _case("append_step", "append", 64, 100, 4000, 1, 1, lens=2),
        # a scheduler's step of fresh prompts of uneven length, f16
        _case("append_prompts", "append", 8, 0, 0, 300, 2000, dtype="f16", lens=3),
        # the next chunk of each of eight prompts, into an FP8 cache
        _case("append_chunk_fp8", "append", 8, 700, 2000, 512, 512, kv="e4m3", lens=4),
        # one long chat: latency
        _case("select_one", "select", 1, 20000, 20000, k=64),
        # a serving batch of long documents of mixed age
        _case("select_batch", "select", 64, 4000, 32000, k=64, lens=5),
        # chunks of two long prompts: every new token selects for itself
        _case("select_chunk", "select", 2, 20000, 26000, 200, 512, k=64, lens=6),
        # one long chat: latency
        _case("attend_one", "attend", 1, 20000, 20000, k=64),
        # the serving batch's attention
        _case("attend_batch", "attend", 64, 4000, 32000, k=128, lens=7),
        # an FP8 cache of 32-token blocks under query heads that group in threes, f16
        _case("attend_fp8", "attend", 48, 2000, 16000, hq=24, bs=32, dtype="f16", kv="e4m3", k=96, lens=8),
        # the chunks' attention, every new token over its own blocks
        _case("attend_chunk", "attend", 2, 20000, 26000, 200, 512, k=64, lens=9),
    ]


_HEADS = [(32, 8), (32, 8), (16, 4), (8, 2), (4, 1), (32, 32), (32, 4), (24, 8), (28, 4), (40, 8), (48, 8), (16, 16)]
_DIMS = [64, 96, 128, 128, 128, 192, 256]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["bounds", "append", "append", "select", "select", "select", "attend", "attend", "attend"])
    dtype, kv = rng.choice(["bf16", "bf16", "f16"]), rng.choice(["", "", "e4m3", "e5m2"])
    bs, d = rng.choice([16, 16, 32, 64]), rng.choice(_DIMS)
    hq, hkv = rng.choice(_HEADS)
    lens = rng.randrange(1 << 16)
    low = rng.choice([1, 2, 8])
    batch, ctx, new, k = _log_int(rng, 1, 128), _log_int(rng, 16, 32000), 0, 0
    if kind == "append":
        new = rng.choice([1, _log_int(rng, 8, 2000)])
        ctx = rng.choice([0, _log_int(rng, 16, 4000)])
        if new > 1:
            batch = min(batch, 8)
        while batch * (ctx + new) * hkv * d > 1.2e8 or batch * new * (hq + 2 * hkv) * d > 1.2e8:
            ctx, new = ctx * 2 // 3, max(1, new * 2 // 3) if ctx < 512 or new > ctx else new
    elif kind != "bounds":
        k = _log_int(rng, 4, 256)
        if kind == "select":   # more blocks than are selected
            low, ctx = min(low, 2), max(ctx, 48 * bs)
        if rng.random() < 0.3:
            new, batch = _log_int(rng, 2, 512), _log_int(rng, 1, 3)
            while batch * new * max(hq, 2 * hkv) * (ctx / bs) * d > 8e10 or batch * new * hkv * k * bs * d > 1.1e9:
                if k > 32:
                    k = k * 2 // 3
                elif new > 16:
                    new = new * 2 // 3
                else:
                    ctx = ctx * 2 // 3
    if kind == "bounds":
        while batch * ctx * hkv * d > 1.4e8:
            batch, ctx = (batch, ctx * 2 // 3) if ctx > 2048 or batch == 1 else (batch * 2 // 3, ctx)
    elif kind != "append":
        while batch * ctx * hkv * d > 1.6e9 or batch * k * bs * hkv * d > 1.3e8:
            batch, k = (batch * 2 // 3, k) if batch > 1 else (batch, max(4, k * 2 // 3))
    if kind == "select":
        ctx = max(ctx, 48 * bs)
        k = max(8, min(k, ctx // bs // 3))
    return _case(None, kind, batch, ctx // low, ctx, max(1, new // low) if new else 0, new, hq, hkv, d, bs, dtype, kv, k, lens)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _ints(case, n, lo, hi, tag):
    r = np.random.default_rng([0x5B0C, case["lens"], n, lo, hi, tag])
    return r.integers(lo, hi, size=n, endpoint=True).astype(np.int64)


def _lengths(case):
    """(tokens before the call's new ones, queries or new tokens of each sequence)."""
    ctx = _ints(case, case["batch"], case["ctx_min"], case["ctx_max"], 0)
    if case["new_max"] == 0:   # a decode step's query is the last cached token's
        return np.maximum(ctx, 1) - 1, np.ones(case["batch"], np.int64)
    return ctx, _ints(case, case["batch"], case["new_min"], case["new_max"], 1)


def _gen(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed & 0x7FFFFFFF)
    return g


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)


def _dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(DEVICE)


def _tables(rng, lens, bs):
    """Scattered block ids, as a block pool hands them out: (tables, blocks in the pool)."""
    nblk = [(int(n) + bs - 1) // bs for n in lens]
    pool = int(math.ceil(1.1 * sum(nblk))) + 1
    perm = rng.permutation(pool).astype(np.int32)
    bt = np.full((len(nblk), max(max(nblk), 1)), -1, np.int32)
    p = 0
    for s, n in enumerate(nblk):
        bt[s, :n] = perm[p:p + n]
        p += n
    return bt, pool


def _stored(case):
    return FP8[case["kv"]] if case["kv"] else HALF[case["dtype"]]


def _own_type(case, t):
    """What the framework takes: FP8 caches are bytes."""
    return t.view(torch.uint8) if case["kv"] else t


def _cache(case, g, pool, chan, scale):
    """A pool of random rows in the cache's type, a part of the blocks at a time."""
    hkv, d, bs = case["hkv"], case["d"], case["bs"]
    out = torch.empty((pool, hkv, d, bs), dtype=_stored(case), device=DEVICE)
    step = max(1, (1 << 27) // (hkv * d * bs))
    for b in range(0, pool, step):
        x = _randn(g, (min(step, pool - b), hkv, d, bs))
        if chan is not None:
            x *= chan[None, :, :, None]
        out[b:b + step] = _to_cache(case, x, scale)
    return out


def _fill(bt, lens, pool, bs):
    """Rows that hold keys, of every block of the pool."""
    fill = np.zeros(pool, np.int64)
    for s, n in enumerate(lens):
        nb = (int(n) + bs - 1) // bs
        fill[bt[s, :nb]] = np.minimum(int(n) - bs * np.arange(nb), bs)
    return _dev(fill)


def _selection(case, g, nv, k):
    """Lists of blocks [rows, hkv, k] as consecutive queries make them: 64 of them draw from 2 k blocks."""
    rows, most = nv.numel(), int(nv.max())
    blk = torch.arange(most, device=DEVICE)
    u = torch.rand((rows, case["hkv"], most), generator=g, device=DEVICE)
    if case["new_max"]:
        t = torch.rand(((rows + 63) // 64, case["hkv"], most), generator=g, device=DEVICE)
        keep = torch.zeros_like(t).scatter_(2, t.topk(min(2 * k, most), dim=2).indices, 1.0)
        u = u + keep.repeat_interleave(64, 0)[:rows]
    fixed = (blk < FIRST) | (blk >= nv[:, None, None] - LAST)
    u = torch.where(fixed, 4.0, u).masked_fill_(blk >= nv[:, None, None], -1.0)
    val, idx = u.topk(min(k, most), dim=2)
    idx = torch.where(val < 0, most, idx).sort(dim=2).values
    idx = torch.where(idx == most, -1, idx)
    return torch.nn.functional.pad(idx, (0, k - idx.shape[2]), value=-1).int().contiguous()


def prepare(case, seed):
    kind, dt = case["kind"], HALF[case["dtype"]]
    g = _gen(seed)
    rng = np.random.default_rng([seed & 0x7FFFFFFF, 29])
    hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["bs"]
    ctx, new = _lengths(case)
    lens, rows = ctx + new, int(new.sum())
    bt, pool = _tables(rng, lens, bs)
    st = {"case": case, "bt": _dev(bt), "lens": _dev(lens.astype(np.int32)), "pool": pool}
    st["qsl"] = _dev(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)) if case["new_max"] > 1 else None
    chan = torch.exp(0.6 * _randn(g, (hkv, d)))   # some channels of a head's keys are larger than others
    if kind == "bounds":
        st["kc"] = _own_type(case, _cache(case, g, pool, chan, K_SCALE))
        st["kb"] = torch.zeros_like(st["kc"][..., :2]).transpose(2, 3).contiguous()
        return st
    pos = torch.cat([torch.arange(c, c + n) for c, n in zip(ctx.tolist(), new.tolist())]).to(DEVICE)
    if kind == "append":
        kc, vc = _cache(case, g, pool, chan, K_SCALE), _cache(case, g, pool, None, V_SCALE)
        st["kb"] = _own_type(case, _plain_bounds(case, kc, _fill(bt, ctx, pool, bs)))
        st["kc"], st["vc"] = _own_type(case, kc), _own_type(case, vc)
        st["q"], st["v"] = _randn(g, (rows, hq, d), dt), _randn(g, (rows, hkv, d), dt)
        st["k"] = (_randn(g, (rows, hkv, d)) * chan).to(dt)
        st["q_out"] = torch.empty_like(st["q"])
        inv = ROPE_THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        ang = torch.arange(8192, dtype=torch.float64)[:, None] * inv[None, :]
        st["cos"], st["sin"] = ang.cos().float().to(DEVICE), ang.sin().float().to(DEVICE)
        return st
    # queries of neighbouring tokens are alike, and point where some keys do
    base = _randn(g, (case["batch"], hq, d)) * 0.8
    seq = torch.repeat_interleave(torch.arange(case["batch"]), torch.from_numpy(new)).to(DEVICE)
    st["q"] = (base[seq] + 0.6 * _randn(g, (rows, hq, d))).to(dt)
    if kind == "select":
        kc = _cache(case, g, pool, chan, K_SCALE)
        st["kb"] = _own_type(case, _plain_bounds(case, kc, _fill(bt, lens, pool, bs)))
        return st
    st["kc"], st["vc"] = (_own_type(case, _cache(case, g, pool, c, s)) for c, s in ((chan, K_SCALE), (None, V_SCALE)))
    st["sel"] = _selection(case, g, pos // bs + 1, case["k"])
    st["out"] = torch.empty_like(st["q"])
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _plain_bounds(case, cache, fill):
    """Bounds [pool, hkv, 2, d] of the first fill[b] rows of every block (zeros where there are none)."""
    x = cache.float()
    held = torch.arange(case["bs"], device=DEVICE) < fill[:, None, None, None]
    lo = x.masked_fill(~held, float("inf")).amin(-1)
    hi = x.masked_fill(~held, float("-inf")).amax(-1)
    some = fill[:, None, None, None] > 0
    return torch.where(some, torch.stack((lo, hi), 2), 0.0).to(cache.dtype)


def _typed(case, t):
    return t.view(_stored(case))


def _rows(st):
    """(sequence, position) of every query or new token."""
    b = st["lens"].numel()
    if st["qsl"] is None:
        return torch.arange(b, device=DEVICE), st["lens"].long() - 1
    qsl = st["qsl"].long()
    t = torch.arange(st["q"].shape[0], device=DEVICE)
    seq = torch.bucketize(t, qsl[1:], right=True)
    return seq, st["lens"].long()[seq] - qsl[seq + 1] + t


def _filled(st, lens):
    """Rows that hold keys, of every block of the pool, by the table."""
    bs, bt = st["case"]["bs"], st["bt"]
    n = (lens.long()[:, None] - bs * torch.arange(bt.shape[1], device=DEVICE)).clamp(0, bs)
    fill = torch.zeros(st["pool"] + 1, dtype=torch.long, device=DEVICE)
    return fill.scatter_(0, torch.where(n > 0, bt.long(), st["pool"]).flatten(), n.flatten())[:-1]


def _plain_rotate(x, cos, sin):
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _to_cache(case, x, scale):
    if not case["kv"]:
        return x.to(HALF[case["dtype"]])
    return (x / scale).clamp(-LARGEST[case["kv"]], LARGEST[case["kv"]]).to(FP8[case["kv"]])


def _plain_append(st):
    case = st["case"]
    seq, pos = _rows(st)
    cos, sin = (st[t][pos][:, None, :] for t in ("cos", "sin"))
    blk, off = st["bt"].long()[seq, pos // case["bs"]], pos % case["bs"]
    _typed(case, st["kc"])[blk, :, :, off] = _to_cache(case, _plain_rotate(st["k"], cos, sin), K_SCALE)
    _typed(case, st["vc"])[blk, :, :, off] = _to_cache(case, st["v"].float(), V_SCALE)
    q = _plain_rotate(st["q"], cos, sin).to(st["q"].dtype)
    # the blocks that each sequence's new tokens reach; where it reaches fewer than others, its last one again
    first = st["lens"].long() - (1 if st["qsl"] is None else (st["qsl"][1:] - st["qsl"][:-1]).long())
    j = first[:, None] // case["bs"] + torch.arange((max(1, case["new_max"]) - 1) // case["bs"] + 2, device=DEVICE)
    j = torch.minimum(j, (st["lens"].long()[:, None] - 1) // case["bs"])
    ids = torch.gather(st["bt"].long(), 1, j).flatten()
    fill = (st["lens"].long()[:, None] - j * case["bs"]).clamp(max=case["bs"]).flatten()
    _typed(case, st["kb"])[ids] = _plain_bounds(case, _typed(case, st["kc"])[ids], fill)
    return q, _typed(case, st["kc"]), _typed(case, st["vc"]), _typed(case, st["kb"])


def _plain_select(st):
    case = st["case"]
    b, hkv, d, k = st["lens"].numel(), case["hkv"], case["d"], case["k"]
    seq, pos = _rows(st)
    rows, most, n = pos.numel(), st["bt"].shape[1], max(1, case["new_max"])
    i = torch.zeros_like(pos) if st["qsl"] is None else torch.arange(rows, device=DEVICE) - st["qsl"].long()[seq]
    q = torch.zeros((b, n, hkv, case["hq"] // hkv, d), dtype=torch.float64, device=DEVICE)
    q[seq, i] = st["q"].double().view(rows, hkv, -1, d)
    q = torch.cat((q.clamp(max=0.0), q.clamp(min=0.0)), -1).transpose(1, 2).reshape(b, hkv, -1, 2 * d)
    bounds = _typed(case, st["kb"])[st["bt"].long().clamp(min=0)].double()              # [b, most, hkv, 2, d]
    bounds = bounds.permute(0, 2, 3, 4, 1).reshape(b, hkv, 2 * d, most).contiguous()
    s = torch.matmul(q, bounds).view(b, hkv, n, -1, most).amax(3)
    s = s.transpose(1, 2)[seq, i]                                                        # [rows, hkv, most]
    blk, nv = torch.arange(most, device=DEVICE), (pos // case["bs"] + 1)[:, None, None]
    s = s.masked_fill((blk < FIRST) | (blk >= nv - LAST), float("inf")).masked_fill(blk >= nv, float("-inf"))
    val, idx = torch.sort(s, dim=2, descending=True, stable=True)
    idx = torch.where(val[..., :k] == float("-inf"), most, idx[..., :k]).sort(dim=2).values
    idx = torch.where(idx == most, -1, idx)
    return torch.nn.functional.pad(idx, (0, k - idx.shape[2]), value=-1).int()


def _plain_attend(st):
    case = st["case"]
    hkv, d, bs = case["hkv"], case["d"], case["bs"]
    seq, pos = _rows(st)
    rows, sel = pos.numel(), st["sel"].long()
    blk = torch.gather(st["bt"].long()[seq][:, None, :].expand(-1, hkv, -1), 2, sel.clamp(min=0))
    head = torch.arange(hkv, device=DEVICE)[None, :, None]
    k = _typed(case, st["kc"])[blk, head].float().transpose(2, 3).flatten(3)             # [rows, hkv, d, keys]
    v = _typed(case, st["vc"])[blk, head].float().transpose(3, 4).flatten(2, 3)          # [rows, hkv, keys, d]
    k_scale, v_scale = (K_SCALE, V_SCALE) if case["kv"] else (1.0, 1.0)
    q = st["q"].float().view(rows, hkv, -1, d)
    s = torch.matmul(q, k) * (_scale(case) * k_scale)
    at = sel[..., None] * bs + torch.arange(bs, device=DEVICE)
    seen = ((sel[..., None] >= 0) & (at <= pos[:, None, None, None])).flatten(2)[:, :, None]
    s = s.masked_fill_(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) * (v_scale / torch.where(z == 0, 1.0, z))
    return o.reshape(rows, case["hq"], d).to(st["q"].dtype)


def _scale(case):
    return 1.0 / math.sqrt(case["d"])


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        from rllm_amd import DTYPE_FP8_E4M3, DTYPE_FP8_E5M2, FP8_ROUND_NEAREST_EVEN, ops
        fp8 = {}
        if case["kv"]:
            fp8 = {"kv_dtype": DTYPE_FP8_E4M3 if case["kv"] == "e4m3" else DTYPE_FP8_E5M2}
        scales = {"k_scale": K_SCALE, "v_scale": V_SCALE} if case["kv"] else {}
        if kind == "bounds":
            ops.key_bounds(st["kc"], st["kb"], st["bt"], st["lens"], validate=False, **fp8)
            return _typed(case, st["kb"])
        if kind == "append":
            ops.rope_and_append(st["q"], st["k"], st["v"], st["kc"], st["vc"], st["kb"], st["bt"], st["lens"],
                                st["cos"], st["sin"], query_start_loc=st["qsl"], q_out=st["q_out"], validate=False,
                                fp8_rounding=FP8_ROUND_NEAREST_EVEN, **fp8, **scales)
            return st["q_out"], _typed(case, st["kc"]), _typed(case, st["vc"]), _typed(case, st["kb"])
        if kind == "select":
            return ops.select_blocks(st["q"], st["kb"], st["bt"], st["lens"], case["bs"], case["k"], num_first=FIRST,
                                     num_last=LAST, query_start_loc=st["qsl"], validate=False, **fp8)
        return ops.paged_sparse(st["q"], st["kc"], st["vc"], st["bt"], st["lens"], st["sel"], _scale(case),
                                query_start_loc=st["qsl"], out=st["out"], validate=False, **fp8, **scales)
    if kind == "bounds":
        return _plain_bounds(case, _typed(case, st["kc"]), _filled(st, st["lens"]))
    if kind == "append":
        return _plain_append(st)
    if kind == "select":
        return _plain_select(st)
    return _plain_attend(st)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    kind, hq, hkv, d, bs, k = (case[x] for x in ("kind", "hq", "hkv", "d", "bs", "k"))
    e = 1 if case["kv"] else 2
    ctx, new = _lengths(case)
    lens, rows = ctx + new, int(new.sum())
    nblk = (lens + bs - 1) // bs
    bound = hkv * 2 * d * e                    # of a block
    table = 4 * int(nblk.sum()) + 4 * len(lens)
    if kind == "bounds":
        return {"bytes": int(lens.sum()) * hkv * d * e + int(nblk.sum()) * bound + table, "flops": 0}
    if kind == "append":
        touched = nblk - ctx // bs
        old = int((ctx % bs > 0).sum())         # blocks whose bounds go on
        per = (2 * hq + 2 * hkv) * d * 2 + 2 * hkv * d * e + d * 4
        return {"bytes": rows * per + (int(touched.sum()) + old) * bound + 4 * int(touched.sum()),
                "flops": rows * (hq + hkv) * d * 3}
    pos = np.concatenate([np.arange(c, c + n) for c, n in zip(ctx.tolist(), new.tolist())])
    nv = pos // bs + 1
    if kind == "select":
        return {"bytes": int(nblk.sum()) * bound + table + rows * (hq * d * 2 + hkv * k * 4),
                "flops": int(nv.sum()) * hq * d * 2}
    took = np.minimum(nv, k)
    keys = took * bs - (bs - 1 - pos % bs)
    blocks = int(took.sum())                    # distinct ones of each sequence and kv head
    if case["new_max"] > 1:
        blocks = int(sum(n * (1 - (1 - min(1.0, 2 * k / n)) ** (m / 64.0)) if m > 64 else min(n, 2 * k)
                         for n, m in zip(nblk.tolist(), new.tolist())))
    return {"bytes": blocks * bs * hkv * d * 2 * e + rows * (hq * d * 4 + hkv * k * 4) + table,
            "flops": int(keys.sum()) * hq * d * 4}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def _exact_bounds(case, values, bt, lens, out):
    """Writes the bounds of every block of the tables over out [pool, hkv, 2, d], a sequence at a time."""
    bs = case["bs"]
    for s, n in enumerate(lens.tolist()):
        nb = n // bs
        if nb:
            x = values[bt[s, :nb].long()]
            out[bt[s, :nb].long()] = torch.stack((x.min(dim=3).values, x.max(dim=3).values), 2)
        if n % bs:
            x = values[int(bt[s, nb])][:, :, :n % bs]
            out[int(bt[s, nb])] = torch.stack((x.min(dim=2).values, x.max(dim=2).values), 1)
    return out


def _exact_stored(case, x, scale):
    """float64 values as an FP8 cache holds them, to the nearest; as they are for a 16-bit one."""
    if not case["kv"]:
        return x
    bits, least = (3, -6) if case["kv"] == "e4m3" else (2, -14)
    x = x / scale
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** least))) - bits)
    return torch.clamp(torch.round(x / step) * step, -LARGEST[case["kv"]], LARGEST[case["kv"]])


def _exact_append(case, st):
    kc, vc, old = (st[t].view(_stored(case)).double() for t in ("kc", "vc", "kb"))
    ctx, new = _lengths(case)
    half, bs, row = case["d"] // 2, case["bs"], 0
    q_all = torch.empty(st["q"].shape, dtype=torch.float64, device=DEVICE)
    touched = []
    for s in range(case["batch"]):
        c, n = int(ctx[s]), int(new[s])
        p = torch.arange(c, c + n, device=DEVICE)
        cos, sin = (st[t][c:c + n].double()[:, None, :] for t in ("cos", "sin"))
        q, k = (st[t][row:row + n].double() for t in ("q", "k"))
        q_all[row:row + n, :, :half] = q[..., :half] * cos - q[..., half:] * sin
        q_all[row:row + n, :, half:] = q[..., half:] * cos + q[..., :half] * sin
        k = torch.cat((k[..., :half] * cos - k[..., half:] * sin, k[..., half:] * cos + k[..., :half] * sin), -1)
        blk = st["bt"][s].long()[p // bs]
        kc[blk, :, :, p % bs] = _exact_stored(case, k, K_SCALE)
        vc[blk, :, :, p % bs] = _exact_stored(case, st["v"][row:row + n].double(), V_SCALE)
        touched.append(blk.unique())
        row += n
    touched = torch.cat(touched)
    full = _exact_bounds(case, kc, st["bt"], st["lens"], old.clone())
    old[touched] = full[touched]
    return q_all, kc, vc, old


def _exact_attend(case, st):
    hkv, g, d, bs = case["hkv"], case["hq"] // case["hkv"], case["d"], case["bs"]
    ctx, new = _lengths(case)
    ks, vs = (K_SCALE, V_SCALE) if case["kv"] else (1.0, 1.0)
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=DEVICE)
    row = 0
    for s in range(case["batch"]):
        c, n = int(ctx[s]), int(new[s])
        ids = st["bt"][s].long()
        step = max(1, (1 << 27) // (hkv * case["k"] * bs * d))
        for a in range(0, n, step):
            m = min(step, n - a)
            sel = st["sel"][row + a:row + a + m].long()
            key = (sel.clamp(min=0)[..., None] * bs + torch.arange(bs, device=DEVICE)).flatten(2)
            ok = (sel >= 0).repeat_interleave(bs, 2) & (key <= c + a + torch.arange(m, device=DEVICE)[:, None, None])
            h = torch.arange(hkv, device=DEVICE)[None, :, None]
            kk = st["kc"].view(_stored(case))[ids[key // bs], h, :, key % bs].double() * ks       # [m, hkv, keys, d]
            q = st["q"][row + a:row + a + m].double().view(m, hkv, g, d)
            w = torch.matmul(kk, q.transpose(2, 3).contiguous()) / math.sqrt(d)
            w = torch.softmax(torch.where(ok[..., None], w, -math.inf), dim=2).transpose(2, 3).contiguous()
            vv = st["vc"].view(_stored(case))[ids[key // bs], h, :, key % bs].double() * vs
            out[row + a:row + a + m] = torch.matmul(w, vv).view(m, case["hq"], d)
        row += n
    return out


def exact(case, seed):
    if case["kind"] == "select":
        return None   # whole numbers
    st = prepare(case, seed)
    if case["kind"] == "bounds":
        kb = torch.zeros(st["kb"].shape, dtype=torch.float64, device=DEVICE)
        return _exact_bounds(case, st["kc"].view(_stored(case)).double(), st["bt"], st["lens"], kb)
    return _exact_append(case, st) if case["kind"] == "append" else _exact_attend(case, st)
