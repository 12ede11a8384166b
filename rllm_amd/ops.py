"""torch-tensor front end of the C ABI, used by the tests and the benchmark.

torch supplies device memory and the current HIP stream; every computation is
one of the library's gfx950 kernels.  Shapes, dtypes, devices and (optionally)
block-table bounds are checked on the host before any launch, so a kernel
never sees operands that disagree with its grid.
"""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import DTYPE_BF16, DTYPE_F16, DTYPE_FP8_E4M3, DTYPE_FP8_E5M2, FP8_ROUND_TOWARD_ZERO, call, lib

_TORCH_16 = {torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}


# A small call's GPU work ends before its Python does, so the checks below first
# test everything at once on plain ints and flags; only a call that fails there
# goes through them one by one, for the error that says which (the host time of
# a decode call 12.0 -> 9.0 us, 3.2 of it the launch).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream: Optional[torch.cuda.Stream]) -> int:
    if stream is not None:
        return int(stream.cuda_stream)
    if _raw_stream is not None and torch.cuda.is_initialized():
        return _raw_stream(torch._C._cuda_getDevice())   # no Stream object is made
    return int(torch.cuda.current_stream().cuda_stream)


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _dense_on_one_gpu(*tensors: torch.Tensor) -> bool:
    dev = tensors[0].get_device()
    if not tensors[0].is_cuda:
        return False
    for t in tensors:
        if t.get_device() != dev or not t.is_contiguous():
            return False
    return True


def _like(out: torch.Tensor, q: torch.Tensor) -> bool:
    return out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous() and out.device == q.device


def _kv_code(cache: torch.Tensor, kv_dtype: Optional[int]) -> int:
    code = _TORCH_16.get(cache.dtype)
    if code is not None:
        if kv_dtype is not None and kv_dtype != code:
            raise ValueError("kv_dtype disagrees with the cache tensor dtype")
        return code
    if cache.dtype == torch.uint8:
        if kv_dtype not in (DTYPE_FP8_E4M3, DTYPE_FP8_E5M2):
            raise ValueError("a uint8 cache needs kv_dtype FP8_E4M3 or FP8_E5M2")
        return kv_dtype
    raise TypeError(f"unsupported cache dtype {cache.dtype}")


def _check_common(q, k_cache, v_cache, block_tables, seq_lens, nseq_dim0):
    if (_dense_on_one_gpu(q, k_cache, v_cache, block_tables, seq_lens) and q.ndim == 3 and k_cache.ndim == 4
            and k_cache.shape == v_cache.shape and k_cache.dtype == v_cache.dtype
            and block_tables.dtype == torch.int32 and seq_lens.dtype == torch.int32 and block_tables.ndim == 2
            and block_tables.shape[0] == nseq_dim0 and seq_lens.shape == (nseq_dim0,)
            and q.shape[2] == k_cache.shape[2] and q.dtype in _TORCH_16):
        return
    dev = q.device
    if dev.type != "cuda":
        raise ValueError("tensors must live on a GPU")
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("block_tables", block_tables),
                    ("seq_lens", seq_lens)):
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, q on {dev}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if not q.is_contiguous():
        raise ValueError("q must be contiguous")
    if q.dim() != 3 or k_cache.dim() != 4 or k_cache.shape != v_cache.shape:
        raise ValueError("q [*, Hq, D] and caches [nb, Hkv, D, bs] of equal shape required")
    if k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache dtypes differ")
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_tables and seq_lens must be int32")
    if block_tables.dim() != 2 or block_tables.shape[0] != nseq_dim0 or seq_lens.shape != (nseq_dim0,):
        raise ValueError("block_tables [num_seqs, max_blocks] and seq_lens [num_seqs] required")
    if q.shape[2] != k_cache.shape[2]:
        raise ValueError("head_dim of q and caches differ")
    if q.dtype not in _TORCH_16:
        raise TypeError("q must be float16 or bfloat16")


def validate_tables(block_tables: torch.Tensor, seq_lens: torch.Tensor, num_blocks: int,
                    block_size: int) -> None:
    """Every table entry a sequence's context reaches must be < num_blocks
    (negative entries are skipped by the kernels)."""
    bt = block_tables.detach().cpu()
    sl = seq_lens.detach().cpu()
    maxb = bt.shape[1]
    for s in range(bt.shape[0]):
        n = min((max(int(sl[s]), 0) + block_size - 1) // block_size, maxb)
        if n and int(bt[s, :n].max()) >= num_blocks:
            raise ValueError(f"block table of sequence {s} points past the cache")


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 block_tables: torch.Tensor, seq_lens: torch.Tensor, scale: float, *,
                 kv_dtype: Optional[int] = None, k_scale: float = 1.0, v_scale: float = 1.0,
                 partition_size: int = 0, out: Optional[torch.Tensor] = None,
                 workspace: Optional[torch.Tensor] = None, validate: bool = True,
                 stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Decode attention through rllm_paged_attention_decode_ex."""
    B, hq, d = q.shape
    _check_common(q, k_cache, v_cache, block_tables, seq_lens, B)
    nb, hkv, d2, bs = k_cache.shape
    kv = _kv_code(k_cache, kv_dtype)
    qd = _TORCH_16[q.dtype]
    if kv in (DTYPE_F16, DTYPE_BF16) and kv != qd:
        raise TypeError("a 16-bit cache must have the dtype of q")
    if validate:
        validate_tables(block_tables, seq_lens, nb, bs)
    if out is None:
        out = torch.empty_like(q)
    elif not _like(out, q):
        raise ValueError("out must be a contiguous tensor like q")
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    call("rllm_paged_attention_decode_ex", _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache),
         _ptr(block_tables), _ptr(seq_lens), B, hq, hkv, d, bs, block_tables.shape[1], scale,
         qd, kv, k_scale, v_scale, partition_size, _ptr(workspace), ws_bytes, _stream(stream))
    return out


def paged_decode_prefix(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        block_tables: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                        num_prefix_blocks: int, *, kv_dtype: Optional[int] = None, k_scale: float = 1.0,
                        v_scale: float = 1.0, out: Optional[torch.Tensor] = None, validate: bool = True,
                        stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Decode of a batch whose tables share their first num_prefix_blocks
    entries, through rllm_paged_attention_decode_prefix_ex (the prefix is
    attended once for the batch, then merged with each sequence's rest)."""
    B, hq, d = q.shape
    _check_common(q, k_cache, v_cache, block_tables, seq_lens, B)
    nb, hkv, d2, bs = k_cache.shape
    kv = _kv_code(k_cache, kv_dtype)
    qd = _TORCH_16[q.dtype]
    if kv in (DTYPE_F16, DTYPE_BF16) and kv != qd:
        raise TypeError("a 16-bit cache must have the dtype of q")
    if validate:
        validate_tables(block_tables, seq_lens, nb, bs)
        if num_prefix_blocks:
            bt = block_tables.cpu()
            if not bool((bt[:, :num_prefix_blocks] == bt[:1, :num_prefix_blocks]).all()):
                raise ValueError("the tables do not share their first num_prefix_blocks entries")
    if out is None:
        out = torch.empty_like(q)
    elif not _like(out, q):
        raise ValueError("out must be a contiguous tensor like q")
    call("rllm_paged_attention_decode_prefix_ex", _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache),
         _ptr(block_tables), _ptr(seq_lens), B, hq, hkv, d, bs, block_tables.shape[1], scale,
         qd, kv, k_scale, v_scale, num_prefix_blocks, _stream(stream))
    return out


def paged_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  query_start_loc: torch.Tensor, scale: float, *, kv_dtype: Optional[int] = None,
                  k_scale: float = 1.0, v_scale: float = 1.0, out: Optional[torch.Tensor] = None,
                  validate: bool = True,
                  stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Chunked-prefill attention through rllm_paged_attention_prefill_ex."""
    T, hq, d = q.shape
    B = seq_lens.shape[0]
    _check_common(q, k_cache, v_cache, block_tables, seq_lens, B)
    if query_start_loc.dtype != torch.int32 or query_start_loc.shape != (B + 1,) or \
            query_start_loc.device != q.device:
        raise ValueError("query_start_loc must be int32 [num_seqs + 1] on the device of q")
    nb, hkv, d2, bs = k_cache.shape
    kv = _kv_code(k_cache, kv_dtype)
    qd = _TORCH_16[q.dtype]
    if kv in (DTYPE_F16, DTYPE_BF16) and kv != qd:
        raise TypeError("a 16-bit cache must have the dtype of q")
    if validate:
        validate_tables(block_tables, seq_lens, nb, bs)
        qsl = query_start_loc.detach().cpu()
        if int(qsl[0]) != 0 or int(qsl[-1]) != T or bool((qsl[1:] < qsl[:-1]).any()):
            raise ValueError("query_start_loc must rise from 0 to num_tokens")
    if out is None:
        out = torch.empty_like(q)
    call("rllm_paged_attention_prefill_ex", _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache),
         _ptr(block_tables), _ptr(seq_lens), _ptr(query_start_loc), B, T, hq, hkv, d, bs,
         block_tables.shape[1], scale, qd, kv, k_scale, v_scale, _stream(stream))
    return out


def paged_mixed(prefill_q: torch.Tensor, prefill_block_tables: torch.Tensor, prefill_seq_lens: torch.Tensor,
                query_start_loc: torch.Tensor, decode_q: torch.Tensor, decode_block_tables: torch.Tensor,
                decode_seq_lens: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, scale: float, *,
                kv_dtype: Optional[int] = None, k_scale: float = 1.0, v_scale: float = 1.0,
                prefill_out: Optional[torch.Tensor] = None, decode_out: Optional[torch.Tensor] = None,
                validate: bool = True, stream: Optional[torch.cuda.Stream] = None):
    """One step's attention over a mixed batch through rllm_paged_attention_mixed_ex:
    the prefill group (as paged_prefill's arguments) and the decode group (as
    paged_decode's) over the same caches.  Returns (prefill_out, decode_out)."""
    T, hq, d = prefill_q.shape
    Bp = prefill_seq_lens.shape[0]
    Bd = decode_q.shape[0]
    _check_common(prefill_q, k_cache, v_cache, prefill_block_tables, prefill_seq_lens, Bp)
    _check_common(decode_q, k_cache, v_cache, decode_block_tables, decode_seq_lens, Bd)
    if decode_q.shape[1:] != (hq, d) or decode_q.dtype != prefill_q.dtype:
        raise ValueError("the two groups' queries must have the same heads, head_dim and dtype")
    if query_start_loc.dtype != torch.int32 or query_start_loc.shape != (Bp + 1,) or \
            query_start_loc.device != prefill_q.device:
        raise ValueError("query_start_loc must be int32 [num_prefill_seqs + 1] on the device of q")
    nb, hkv, d2, bs = k_cache.shape
    kv = _kv_code(k_cache, kv_dtype)
    qd = _TORCH_16[prefill_q.dtype]
    if kv in (DTYPE_F16, DTYPE_BF16) and kv != qd:
        raise TypeError("a 16-bit cache must have the dtype of q")
    if validate:
        validate_tables(prefill_block_tables, prefill_seq_lens, nb, bs)
        validate_tables(decode_block_tables, decode_seq_lens, nb, bs)
        qsl = query_start_loc.detach().cpu()
        if int(qsl[0]) != 0 or int(qsl[-1]) != T or bool((qsl[1:] < qsl[:-1]).any()):
            raise ValueError("query_start_loc must rise from 0 to num_prefill_tokens")
    if prefill_out is None:
        prefill_out = torch.empty_like(prefill_q)
    if decode_out is None:
        decode_out = torch.empty_like(decode_q)
    for o, ref in ((prefill_out, prefill_q), (decode_out, decode_q)):
        if not _like(o, ref):
            raise ValueError("outputs must be contiguous tensors like their queries")
    call("rllm_paged_attention_mixed_ex", _ptr(prefill_out), _ptr(prefill_q), _ptr(prefill_block_tables),
         _ptr(prefill_seq_lens), _ptr(query_start_loc), Bp, T, prefill_block_tables.shape[1], _ptr(decode_out),
         _ptr(decode_q), _ptr(decode_block_tables), _ptr(decode_seq_lens), Bd, decode_block_tables.shape[1],
         _ptr(k_cache), _ptr(v_cache), hq, hkv, d, bs, scale, qd, kv, k_scale, v_scale, _stream(stream))
    return prefill_out, decode_out


def reshape_and_cache(new_key: torch.Tensor, new_value: torch.Tensor, k_cache: torch.Tensor,
                      v_cache: torch.Tensor, slot_mapping: torch.Tensor, *,
                      kv_dtype: Optional[int] = None, k_scale: float = 1.0, v_scale: float = 1.0,
                      fp8_rounding: int = FP8_ROUND_TOWARD_ZERO,
                      stream: Optional[torch.cuda.Stream] = None) -> None:
    """Slot-mapped cache write through rllm_cache_write_{bf16,f16,fp8_ex}.
    ``fp8_rounding``: FP8_ROUND_TOWARD_ZERO (the reference contract) or
    FP8_ROUND_NEAREST_EVEN."""
    if new_key.shape != new_value.shape or new_key.dim() != 3:
        raise ValueError("new_key/new_value must be [num_tokens, Hkv, D]")
    n, hkv, d = new_key.shape
    nb, hkv2, d2, bs = k_cache.shape
    if (hkv, d) != (hkv2, d2) or k_cache.shape != v_cache.shape:
        raise ValueError("token rows do not match the cache layout")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (n,):
        raise ValueError("slot_mapping must be int64 [num_tokens]")
    if not _dense_on_one_gpu(new_key, new_value, k_cache, v_cache, slot_mapping):
        for t in (new_key, new_value, k_cache, v_cache, slot_mapping):
            if not t.is_contiguous() or t.device != new_key.device:
                raise ValueError("tensors must be contiguous and on one device")
    kv = _kv_code(k_cache, kv_dtype)
    ind = _TORCH_16.get(new_key.dtype)
    if ind is None or new_value.dtype != new_key.dtype:
        raise TypeError("new_key/new_value must be float16 or bfloat16")
    st = _stream(stream)
    if kv in (DTYPE_F16, DTYPE_BF16):
        if kv != ind:
            raise TypeError("16-bit cache dtype must equal the input dtype")
        name = "rllm_cache_write_bf16" if kv == DTYPE_BF16 else "rllm_cache_write_f16"
        call(name, _ptr(k_cache), _ptr(v_cache), _ptr(new_key), _ptr(new_value),
             _ptr(slot_mapping), n, hkv, d, bs, nb, st)
    else:
        call("rllm_cache_write_fp8_ex", _ptr(k_cache), _ptr(v_cache), _ptr(new_key),
             _ptr(new_value), _ptr(slot_mapping), n, hkv, d, bs, nb, ind, k_scale, v_scale,
             kv, fp8_rounding, st)


def rope_cache_tables(max_position: int, head_dim: int, theta: float = 10000.0,
                      device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """cos / sin tables float32 [max_position, head_dim // 2] from the
    library's host builder ``rllm_rope_tables`` (RotaryEmbedding::new,
    crates/rllm-model/src/rope.rs:13-33), moved to ``device`` if given."""
    cos = torch.empty((max_position, head_dim // 2), dtype=torch.float32)
    sin = torch.empty_like(cos)
    call("rllm_rope_tables", _ptr(cos), _ptr(sin), max_position, head_dim, theta)
    if device is not None:
        cos, sin = cos.to(device), sin.to(device)
    return cos, sin


def rope_and_cache(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                   k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                   positions: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                   q_out: Optional[torch.Tensor] = None, kv_dtype: Optional[int] = None,
                   k_scale: float = 1.0, v_scale: float = 1.0,
                   fp8_rounding: int = FP8_ROUND_TOWARD_ZERO,
                   stream: Optional[torch.cuda.Stream] = None) -> Optional[torch.Tensor]:
    """Rotate q and k by halves (crates/rllm-model/src/rope.rs:57-82) and write
    the rotated key and v into the paged caches, through
    ``rllm_rope_cache_write``.  Returns the rotated q (``q_out``, which may be
    ``q`` itself for an in-place rotation), or None when q is None."""
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError("k/v must be [num_tokens, Hkv, D] of one shape")
    n, hkv, d = k.shape
    nb, hkv2, d2, bs = k_cache.shape
    if (hkv, d) != (hkv2, d2) or k_cache.shape != v_cache.shape:
        raise ValueError("token rows do not match the cache layout")
    dt = _TORCH_16.get(k.dtype)
    if dt is None or v.dtype != k.dtype:
        raise TypeError("k/v must be float16 or bfloat16")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (n,):
        raise ValueError("slot_mapping must be int64 [num_tokens]")
    if positions.dtype != torch.int32 or positions.shape != (n,):
        raise ValueError("positions must be int32 [num_tokens]")
    if cos.dtype != torch.float32 or sin.shape != cos.shape or sin.dtype != cos.dtype \
            or cos.dim() != 2 or cos.shape[1] != d // 2:
        raise ValueError("cos/sin must be float32 [max_position, head_dim // 2]")
    hq = 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != d or q.dtype != k.dtype:
            raise ValueError("q must be [num_tokens, Hq, D] of the k dtype")
        hq = q.shape[1]
        if q_out is None:
            q_out = torch.empty_like(q)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise ValueError("q_out must match q")
    kv = _kv_code(k_cache, kv_dtype)
    if kv in (DTYPE_F16, DTYPE_BF16) and kv != dt:
        raise TypeError("16-bit cache dtype must equal the input dtype")
    tensors = [k, v, k_cache, v_cache, slot_mapping, positions, cos, sin]
    if q is not None:
        tensors += [q, q_out]
    if not _dense_on_one_gpu(*tensors):
        for t in tensors:
            if not t.is_contiguous() or t.device != k.device:
                raise ValueError("tensors must be contiguous and on one device")
    call("rllm_rope_cache_write_ex", _ptr(q_out) if q is not None else 0, _ptr(q), _ptr(k), _ptr(v),
         _ptr(k_cache), _ptr(v_cache), _ptr(slot_mapping), _ptr(positions), _ptr(cos), _ptr(sin),
         n, hq, hkv, d, bs, nb, cos.shape[0], dt, kv, k_scale, v_scale, fp8_rounding, _stream(stream))
    return q_out if q is not None else None


def mxfp4_cache(num_blocks: int, num_kv_heads: int, head_dim: int, block_size: int, device) -> torch.Tensor:
    """A zeroed MXFP4 cache uint8 [num_blocks, num_kv_heads, page] (keys or values
    of one layer; layout in include/rllm_kernels.h)."""
    page = lib().rllm_mxfp4_page_bytes(head_dim, block_size)
    if page < 0:
        raise ValueError("head_dim must be a multiple of 32 up to 256, block_size a multiple of 16 up to 4096")
    return torch.zeros((num_blocks, num_kv_heads, page), dtype=torch.uint8, device=device)


def _check_mxfp4_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, hkv: int, d: int) -> None:
    """A pair of MXFP4 caches of hkv heads and head_dim d, or an error."""
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8 or k_cache.dim() != 3 \
            or k_cache.shape != v_cache.shape:
        raise ValueError("MXFP4 caches are uint8 [num_blocks, Hkv, page] of equal shape")
    row = d // 32 * 17
    bs = k_cache.shape[2] // row if row else 0
    if d % 32 or k_cache.shape[1] != hkv or bs < 16 or bs % 16 or bs * row != k_cache.shape[2]:
        raise ValueError("the caches' heads and page do not fit the heads and head_dim")


def _on_current_gpu(*tensors: torch.Tensor) -> bool:
    """Contiguous tensors of the current device (device numbers as ints: no device objects are made)."""
    dev = tensors[0].get_device()
    if dev < 0 or dev != torch.cuda.current_device():
        return False
    for t in tensors:
        if t.get_device() != dev or not t.is_contiguous():
            return False
    return True


def _all_dense(*tensors: torch.Tensor) -> None:
    if not _on_current_gpu(*tensors):
        raise ValueError("tensors must be contiguous and on the current GPU")


def _mxfp4_rows(key, value, k_cache, v_cache, slot_mapping):
    """Checks of the row operators; returns (n, Hkv, D, block size, blocks, dtype code)."""
    shape, cache = key.shape, k_cache.shape
    dt = _TORCH_16.get(key.dtype)
    # at once, as for the other operators; what fails goes on to the error that says which
    if (dt is not None and len(shape) == 3 and len(cache) == 3 and value.shape == shape and v_cache.shape == cache
            and value.dtype is key.dtype and k_cache.dtype is torch.uint8 and v_cache.dtype is torch.uint8
            and slot_mapping.dtype is torch.int64 and slot_mapping.shape == shape[:1]
            and _on_current_gpu(key, value, k_cache, v_cache, slot_mapping)):
        n, hkv, d = shape
        nb, heads, page = cache
        row = d // 32 * 17
        if heads == hkv and d % 32 == 0 and row and page % (16 * row) == 0 and page:
            return n, hkv, d, page // row, nb, dt
    if key.dim() != 3 or value.shape != key.shape:
        raise ValueError("key and value rows must be [num_tokens, Hkv, D] of one shape")
    if dt is None or value.dtype != key.dtype:
        raise TypeError("key and value rows must be float16 or bfloat16")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != shape[:1]:
        raise ValueError("slot_mapping must be int64 [num_tokens]")
    _check_mxfp4_caches(k_cache, v_cache, shape[1], shape[2])
    raise ValueError("tensors must be contiguous and on the current GPU")


def reshape_and_cache_mxfp4(new_key: torch.Tensor, new_value: torch.Tensor, k_cache: torch.Tensor,
                            v_cache: torch.Tensor, slot_mapping: torch.Tensor, *,
                            stream: Optional[torch.cuda.Stream] = None) -> None:
    """Slot-mapped write into MXFP4 caches, quantising as it writes, through
    rllm_cache_write_mxfp4."""
    n, hkv, d, bs, nb, dt = _mxfp4_rows(new_key, new_value, k_cache, v_cache, slot_mapping)
    call("rllm_cache_write_mxfp4", _ptr(k_cache), _ptr(v_cache), _ptr(new_key), _ptr(new_value), _ptr(slot_mapping),
         n, hkv, d, bs, nb, dt, _stream(stream))


def read_cache_mxfp4(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor, *,
                     head_dim: Optional[int] = None, dtype: Optional[torch.dtype] = None,
                     out_key: Optional[torch.Tensor] = None, out_value: Optional[torch.Tensor] = None,
                     stream: Optional[torch.cuda.Stream] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows slot_mapping names of MXFP4 caches as 16-bit (key, value)
    [num_tokens, Hkv, D], through rllm_cache_read_mxfp4; rows of negative slots are
    zeros.  Give out_key and out_value, or head_dim and dtype."""
    if (out_key is None) != (out_value is None):
        raise ValueError("give both out_key and out_value or neither")
    if out_key is None:
        if head_dim is None or dtype is None or k_cache.dim() != 3 or slot_mapping.dim() != 1:
            raise ValueError("without outputs, head_dim and dtype are needed, 3-d caches and 1-d slots")
        out_key = torch.empty((slot_mapping.shape[0], k_cache.shape[1], head_dim), dtype=dtype, device=k_cache.device)
        out_value = torch.empty_like(out_key)
    elif (head_dim is not None and head_dim != out_key.shape[-1]) or (dtype is not None and dtype != out_key.dtype):
        raise ValueError("head_dim and dtype disagree with the outputs")
    n, hkv, d, bs, nb, dt = _mxfp4_rows(out_key, out_value, k_cache, v_cache, slot_mapping)
    call("rllm_cache_read_mxfp4", _ptr(out_key), _ptr(out_value), _ptr(k_cache), _ptr(v_cache), _ptr(slot_mapping),
         n, hkv, d, bs, nb, dt, _stream(stream))
    return out_key, out_value


def rope_and_cache_mxfp4(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                         v_cache: torch.Tensor, slot_mapping: torch.Tensor, positions: torch.Tensor,
                         cos: torch.Tensor, sin: torch.Tensor, *, q_out: Optional[torch.Tensor] = None,
                         stream: Optional[torch.cuda.Stream] = None) -> Optional[torch.Tensor]:
    """rope_and_cache over MXFP4 caches, through rllm_rope_cache_write_mxfp4: q and
    k rotated in f32, q rounded once, k quantised from f32.  Returns the rotated q
    (``q_out``, which may be ``q`` itself), or None when q is None."""
    n, hkv, d, bs, nb, dt = _mxfp4_rows(k, v, k_cache, v_cache, slot_mapping)
    if positions.dtype != torch.int32 or positions.shape != (n,):
        raise ValueError("positions must be int32 [num_tokens]")
    if cos.dtype != torch.float32 or sin.shape != cos.shape or sin.dtype != cos.dtype \
            or cos.dim() != 2 or cos.shape[1] != d // 2:
        raise ValueError("cos/sin must be float32 [max_position, head_dim // 2]")
    hq = 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != d or q.dtype != k.dtype:
            raise ValueError("q must be [num_tokens, Hq, D] of the k dtype")
        hq = q.shape[1]
        if q_out is None:
            q_out = torch.empty_like(q)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype:
            raise ValueError("q_out must match q")
        _all_dense(positions, cos, sin, q, q_out)
    elif q_out is not None:
        raise ValueError("q_out without q")
    else:
        _all_dense(positions, cos, sin)
    call("rllm_rope_cache_write_mxfp4", _ptr(q_out), _ptr(q), _ptr(k), _ptr(v), _ptr(k_cache), _ptr(v_cache),
         _ptr(slot_mapping), _ptr(positions), _ptr(cos), _ptr(sin), n, hq, hkv, d, bs, nb, cos.shape[0], dt,
         _stream(stream))
    return q_out


def _mxfp4_attention(q, k_cache, v_cache, block_tables, seq_lens, out):
    """Checks the attention operators share; returns (rows, Hq, Hkv, D, sequences,
    table width, block size, blocks, dtype code, out)."""
    shape, cache, table = q.shape, k_cache.shape, block_tables.shape
    dt = _TORCH_16.get(q.dtype)
    if out is None:
        out = torch.empty_like(q)
    if (dt is not None and len(shape) == 3 and len(cache) == 3 and len(table) == 2 and v_cache.shape == cache
            and out.shape == shape and out.dtype is q.dtype and k_cache.dtype is torch.uint8
            and v_cache.dtype is torch.uint8 and block_tables.dtype is torch.int32 and seq_lens.dtype is torch.int32
            and seq_lens.shape == table[:1] and _on_current_gpu(q, k_cache, v_cache, block_tables, seq_lens, out)):
        rows, hq, d = shape
        nb, hkv, page = cache
        row = d // 32 * 17
        if d % 32 == 0 and row and page % (16 * row) == 0 and page:
            return rows, hq, hkv, d, table[0], table[1], page // row, nb, dt, out
    if q.dim() != 3 or k_cache.dim() != 3:
        raise ValueError("q [*, Hq, D] and MXFP4 caches [nb, Hkv, page] required")
    if dt is None:
        raise TypeError("q must be float16 or bfloat16")
    if block_tables.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise TypeError("block_tables and seq_lens must be int32")
    if block_tables.dim() != 2 or seq_lens.shape != table[:1]:
        raise ValueError("block_tables [num_seqs, max_blocks] and seq_lens [num_seqs] required")
    if not _like(out, q):
        raise ValueError("out must be a contiguous tensor like q")
    _check_mxfp4_caches(k_cache, v_cache, cache[1], shape[2])
    raise ValueError("tensors must be contiguous and on the current GPU")


def paged_decode_mxfp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                       seq_lens: torch.Tensor, scale: float, *, out: Optional[torch.Tensor] = None,
                       workspace: Optional[torch.Tensor] = None, validate: bool = True,
                       stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Decode attention over MXFP4 caches through rllm_paged_attention_decode_mxfp4."""
    n, hq, hkv, d, b, maxb, bs, nb, dt, out = _mxfp4_attention(q, k_cache, v_cache, block_tables, seq_lens, out)
    if n != b:
        raise ValueError("one query a sequence required")
    if validate:
        validate_tables(block_tables, seq_lens, nb, bs)
    ws_bytes = 0
    if workspace is not None:
        _all_dense(q, workspace)
        ws_bytes = workspace.numel() * workspace.element_size()
    call("rllm_paged_attention_decode_mxfp4", _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables),
         _ptr(seq_lens), b, hq, hkv, d, bs, maxb, nb, scale, dt, _ptr(workspace), ws_bytes,
         _stream(stream))
    return out


def paged_prefill_mxfp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                        seq_lens: torch.Tensor, query_start_loc: torch.Tensor, scale: float, *,
                        out: Optional[torch.Tensor] = None, validate: bool = True,
                        stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Chunked-prefill attention over MXFP4 caches through rllm_paged_attention_prefill_mxfp4."""
    t, hq, hkv, d, b, maxb, bs, nb, dt, out = _mxfp4_attention(q, k_cache, v_cache, block_tables, seq_lens, out)
    if query_start_loc.dtype != torch.int32 or query_start_loc.shape != (b + 1,) or \
            query_start_loc.get_device() != q.get_device() or not query_start_loc.is_contiguous():
        raise ValueError("query_start_loc must be contiguous int32 [num_seqs + 1] on the device of q")
    if validate:
        validate_tables(block_tables, seq_lens, nb, bs)
        qsl = query_start_loc.detach().cpu()
        if int(qsl[0]) != 0 or int(qsl[-1]) != t or bool((qsl[1:] < qsl[:-1]).any()):
            raise ValueError("query_start_loc must rise from 0 to num_tokens")
    call("rllm_paged_attention_prefill_mxfp4", _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables),
         _ptr(seq_lens), _ptr(query_start_loc), b, t, hq, hkv, d, bs, maxb, nb, scale, dt,
         _stream(stream))
    return out


def new_key_bounds(k_cache: torch.Tensor) -> torch.Tensor:
    """Zeroed key bounds [num_blocks, Hkv, 2, D] for a key cache [num_blocks, Hkv, D, bs], in its type."""
    if k_cache.dim() != 4:
        raise ValueError("a key cache [num_blocks, Hkv, D, bs] required")
    nb, hkv, d, _ = k_cache.shape
    return torch.zeros((nb, hkv, 2, d), dtype=k_cache.dtype, device=k_cache.device)


def _check_rows(rows: int, block_tables, seq_lens, query_start_loc, device: int) -> int:
    """Checks of what places rows in sequences; returns the number of sequences."""
    if block_tables.dtype is not torch.int32 or seq_lens.dtype is not torch.int32:
        raise TypeError("block_tables and seq_lens must be int32")
    table = block_tables.shape
    if len(table) != 2 or seq_lens.shape != table[:1]:
        raise ValueError("block_tables [num_seqs, max_blocks] and seq_lens [num_seqs] required")
    if query_start_loc is None:
        if rows != table[0]:
            raise ValueError("without query_start_loc there is one row a sequence")
    elif query_start_loc.dtype is not torch.int32 or query_start_loc.shape != (table[0] + 1,) \
            or query_start_loc.get_device() != device or not query_start_loc.is_contiguous():
        raise ValueError("query_start_loc must be contiguous int32 [num_seqs + 1] on the device of the rows")
    return table[0]


def _validate_rows(rows: int, block_tables, seq_lens, query_start_loc, num_blocks: int, block_size: int) -> None:
    validate_tables(block_tables, seq_lens, num_blocks, block_size)
    if query_start_loc is not None:
        qsl = query_start_loc.detach().cpu()
        if int(qsl[0]) < 0 or int(qsl[-1]) > rows or bool((qsl[1:] < qsl[:-1]).any()):
            raise ValueError("query_start_loc must rise, within the rows")


def _sparse_shape(d: int, bs: int) -> None:
    if d % 32 or not 0 < d <= 256 or bs not in (16, 32, 64, 128):
        raise ValueError("head_dim must be a multiple of 32 up to 256, block_size 16, 32, 64 or 128")


def _check_bounds(k_bounds: torch.Tensor, nb: int, hkv: int, d: int, dtype: torch.dtype) -> None:
    if k_bounds.shape != (nb, hkv, 2, d) or k_bounds.dtype is not dtype:
        raise ValueError("k_bounds must be [num_blocks, Hkv, 2, D] of the cache's type")


def key_bounds(k_cache: torch.Tensor, k_bounds: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor, *,
               first_positions: Optional[torch.Tensor] = None, kv_dtype: Optional[int] = None, validate: bool = True,
               stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Brings up to date the bounds of the blocks that the sequences' keys reach (of those that end
    past first_positions, int32 [num_seqs], if given), through rllm_key_bounds; returns k_bounds."""
    if k_cache.dim() != 4:
        raise ValueError("a key cache [num_blocks, Hkv, D, bs] required")
    nb, hkv, d, bs = k_cache.shape
    kv = _kv_code(k_cache, kv_dtype)
    _sparse_shape(d, bs)
    _check_bounds(k_bounds, nb, hkv, d, k_cache.dtype)
    b = _check_rows(seq_lens.shape[0], block_tables, seq_lens, None, k_cache.get_device())
    _all_dense(k_cache, k_bounds, block_tables, seq_lens)
    if first_positions is not None:
        if first_positions.dtype is not torch.int32 or first_positions.shape != (b,):
            raise ValueError("first_positions must be int32 [num_seqs]")
        _all_dense(k_cache, first_positions)
    if validate:
        validate_tables(block_tables, seq_lens, nb, bs)
    call("rllm_key_bounds", _ptr(k_bounds), _ptr(k_cache), _ptr(block_tables), _ptr(seq_lens), _ptr(first_positions),
         b, hkv, d, bs, block_tables.shape[1], nb, kv, _stream(stream))
    return k_bounds


def rope_and_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                    v_cache: torch.Tensor, k_bounds: torch.Tensor, block_tables: torch.Tensor,
                    seq_lens: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                    query_start_loc: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
                    kv_dtype: Optional[int] = None, k_scale: float = 1.0, v_scale: float = 1.0,
                    fp8_rounding: int = FP8_ROUND_TOWARD_ZERO, validate: bool = True,
                    stream: Optional[torch.cuda.Stream] = None) -> Optional[torch.Tensor]:
    """Rotates q and k by halves at their positions, writes the sequences' new keys and values where the block
    tables say, and keeps the bounds of the blocks written, through rllm_rope_cache_append.  seq_lens count the
    new tokens; without query_start_loc each sequence has one.  Returns the rotated q (``q_out``, which
    may be ``q`` itself), or None when q is None."""
    rows, cache, table, dtype, cache_dtype = k.shape, k_cache.shape, cos.shape, k.dtype, k_cache.dtype   # each read once
    if len(rows) != 3 or v.shape != rows or len(cache) != 4:
        raise ValueError("k/v [num_tokens, Hkv, D] of one shape and caches [nb, Hkv, D, bs] required")
    n, hkv, d = rows
    nb, hkv2, d2, bs = cache
    if hkv != hkv2 or d != d2 or v_cache.shape != cache or v_cache.dtype is not cache_dtype:
        raise ValueError("token rows do not match the cache layout")
    dt = _TORCH_16.get(dtype)
    if dt is None or v.dtype is not dtype:
        raise TypeError("k/v must be float16 or bfloat16")
    kv = _kv_code(k_cache, kv_dtype)
    if kv in (DTYPE_F16, DTYPE_BF16) and kv != dt:
        raise TypeError("16-bit cache dtype must equal the input dtype")
    _sparse_shape(d, bs)
    _check_bounds(k_bounds, nb, hkv, d, cache_dtype)
    b = _check_rows(n, block_tables, seq_lens, query_start_loc, k.get_device())
    if cos.dtype is not torch.float32 or sin.shape != table or sin.dtype is not torch.float32 \
            or len(table) != 2 or table[1] != d // 2:
        raise ValueError("cos/sin must be float32 [max_position, head_dim // 2]")
    hq = 0
    if q is not None:
        queries = q.shape
        if len(queries) != 3 or queries[0] != n or queries[2] != d or q.dtype is not dtype:
            raise ValueError("q must be [num_tokens, Hq, D] of the k dtype")
        hq = queries[1]
        if q_out is None:
            q_out = torch.empty_like(q)
        elif q_out.shape != queries or q_out.dtype is not dtype:
            raise ValueError("q_out must match q")
        _all_dense(k, v, k_cache, v_cache, k_bounds, block_tables, seq_lens, cos, sin, q, q_out)
    elif q_out is not None:
        raise ValueError("q_out without q")
    else:
        _all_dense(k, v, k_cache, v_cache, k_bounds, block_tables, seq_lens, cos, sin)
    if validate:
        _validate_rows(n, block_tables, seq_lens, query_start_loc, nb, bs)
    call("rllm_rope_cache_append", _ptr(q_out), _ptr(q), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
         k_bounds.data_ptr(), block_tables.data_ptr(), seq_lens.data_ptr(), _ptr(query_start_loc), cos.data_ptr(),
         sin.data_ptr(), b, n, hq, hkv, d, bs, block_tables.shape[1], nb, table[0], dt, kv, k_scale, v_scale, fp8_rounding,
         _stream(stream))
    return q_out


def select_blocks(q: torch.Tensor, k_bounds: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                  block_size: int, num_selected: int, *, num_first: int = 1, num_last: int = 1,
                  query_start_loc: Optional[torch.Tensor] = None, kv_dtype: Optional[int] = None,
                  out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                  validate: bool = True, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """The blocks that each query row and kv head attends, int32 [num_rows, Hkv, num_selected] (rising,
    then -1): the first num_first, the last num_last and those of the largest upper bound of q . k, through
    rllm_select_blocks.  Without query_start_loc each sequence has one row, its last token."""
    if q.dim() != 3 or k_bounds.dim() != 4:
        raise ValueError("q [*, Hq, D] and k_bounds [nb, Hkv, 2, D] required")
    rows, hq, d = q.shape
    nb, hkv = k_bounds.shape[:2]
    dt = _TORCH_16.get(q.dtype)
    if dt is None:
        raise TypeError("q must be float16 or bfloat16")
    kv = _kv_code(k_bounds, kv_dtype)
    if kv in (DTYPE_F16, DTYPE_BF16) and kv != dt:
        raise TypeError("16-bit bounds must have the dtype of q")
    _sparse_shape(d, block_size)
    _check_bounds(k_bounds, nb, hkv, d, k_bounds.dtype)
    b = _check_rows(rows, block_tables, seq_lens, query_start_loc, q.get_device())
    if out is None:
        out = torch.empty((rows, hkv, num_selected), dtype=torch.int32, device=q.device)
        _all_dense(q, k_bounds, block_tables, seq_lens)
    elif out.shape != (rows, hkv, num_selected) or out.dtype is not torch.int32:
        raise ValueError("out must be int32 [num_rows, Hkv, num_selected]")
    else:
        _all_dense(q, k_bounds, block_tables, seq_lens, out)
    ws_bytes = 0
    if workspace is not None:
        _all_dense(q, workspace)
        ws_bytes = workspace.numel() * workspace.element_size()
    if validate:
        _validate_rows(rows, block_tables, seq_lens, query_start_loc, nb, block_size)
    call("rllm_select_blocks", _ptr(out), _ptr(q), _ptr(k_bounds), _ptr(block_tables), _ptr(seq_lens),
         _ptr(query_start_loc), b, rows, hq, hkv, d, block_size, block_tables.shape[1], nb, num_selected, num_first,
         num_last, dt, kv, _ptr(workspace), ws_bytes, _stream(stream))
    return out


def _validate_lists(selected: torch.Tensor) -> None:
    s = selected.detach().cpu()
    before, after = s[..., :-1], s[..., 1:]
    if bool(((after >= 0) & ((after <= before) | (before < 0))).any()):
        raise ValueError("the blocks of a list must rise, with nothing but -1 after them")


def paged_sparse(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 seq_lens: torch.Tensor, selected: torch.Tensor, scale: float, *,
                 query_start_loc: Optional[torch.Tensor] = None, kv_dtype: Optional[int] = None, k_scale: float = 1.0,
                 v_scale: float = 1.0, out: Optional[torch.Tensor] = None, validate: bool = True,
                 stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Attention of each query row over the keys it sees in the blocks that selected [num_rows, Hkv, n]
    lists for it (as select_blocks returns them), through rllm_paged_attention_sparse.  ``out`` is not ``q``."""
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape or v_cache.dtype is not k_cache.dtype:
        raise ValueError("q [*, Hq, D] and caches [nb, Hkv, D, bs] of equal shape and type required")
    rows, hq, d = q.shape
    nb, hkv, d2, bs = k_cache.shape
    dt = _TORCH_16.get(q.dtype)
    if dt is None:
        raise TypeError("q must be float16 or bfloat16")
    if d != d2:
        raise ValueError("head_dim of q and caches differ")
    kv = _kv_code(k_cache, kv_dtype)
    if kv in (DTYPE_F16, DTYPE_BF16) and kv != dt:
        raise TypeError("a 16-bit cache must have the dtype of q")
    _sparse_shape(d, bs)
    b = _check_rows(rows, block_tables, seq_lens, query_start_loc, q.get_device())
    if selected.dtype is not torch.int32 or selected.dim() != 3 or selected.shape[:2] != (rows, hkv):
        raise ValueError("selected must be int32 [num_rows, Hkv, n]")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype is not q.dtype:
        raise ValueError("out must be a contiguous tensor like q")
    elif out.data_ptr() == q.data_ptr() and out.numel():
        raise ValueError("out must not be q")
    _all_dense(q, k_cache, v_cache, block_tables, seq_lens, selected, out)
    if validate:
        _validate_rows(rows, block_tables, seq_lens, query_start_loc, nb, bs)
        _validate_lists(selected)
    call("rllm_paged_attention_sparse", _ptr(out), _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(block_tables),
         _ptr(seq_lens), _ptr(query_start_loc), _ptr(selected), b, rows, hq, hkv, d, bs, block_tables.shape[1], nb,
         selected.shape[2], scale, dt, kv, k_scale, v_scale, _stream(stream))
    return out


def layer_table(caches, device) -> torch.Tensor:
    """DEVICE uint64 array of the per-layer cache base addresses, the form
    rllm_cache_copy_blocks / rllm_cache_swap_{out,in} take.  Build it once per
    cache allocation and keep it alive while calls use it."""
    return torch.tensor([int(c.data_ptr()) for c in caches], dtype=torch.int64).to(device)


def _block_geometry(key_caches, value_caches):
    if not key_caches or len(key_caches) != len(value_caches):
        raise ValueError("need one key and one value cache per layer")
    c0 = key_caches[0]
    for c in list(key_caches) + list(value_caches):
        if c.shape != c0.shape or c.dtype != c0.dtype or c.device != c0.device or not c.is_contiguous():
            raise ValueError("all layer caches must share shape, dtype and device, contiguous")
    nb = c0.shape[0]
    return nb, c0[0].numel() * c0.element_size()


def copy_blocks(key_caches, value_caches, block_pairs: torch.Tensor, *, tables=None,
                stream: Optional[torch.cuda.Stream] = None) -> None:
    """Copy-on-write data movement: block src -> dst of every (src, dst) row of
    the int64 [n, 2] device tensor, in every layer's key and value cache
    (rllm_cache_copy_blocks).  ``tables`` = (key, value) from layer_table()."""
    nb, nbytes = _block_geometry(key_caches, value_caches)
    if block_pairs.dtype != torch.int64 or block_pairs.dim() != 2 or block_pairs.shape[1] != 2 \
            or not block_pairs.is_contiguous():
        raise ValueError("block_pairs must be contiguous int64 [n, 2]")
    dev = key_caches[0].device
    kt, vt = tables if tables is not None else (layer_table(key_caches, dev), layer_table(value_caches, dev))
    call("rllm_cache_copy_blocks", _ptr(kt), _ptr(vt), len(key_caches), _ptr(block_pairs),
         block_pairs.shape[0], nb, nbytes, _stream(stream))


def _swap(name, key_caches, value_caches, block_ids, records, slots, tables, stream):
    nb, nbytes = _block_geometry(key_caches, value_caches)
    L = len(key_caches)
    if block_ids.dtype != torch.int64 or block_ids.dim() != 1 or not block_ids.is_contiguous():
        raise ValueError("block_ids must be contiguous int64 [n]")
    if records.dtype != torch.uint8 or records.device.type != "cpu" or not records.is_pinned() \
            or not records.is_contiguous() or records.dim() != 4 \
            or tuple(records.shape[1:]) != (L, 2, nbytes):
        raise ValueError(f"records must be pinned contiguous uint8 [R, {L}, 2, {nbytes}]")
    if slots is not None and (slots.dtype != torch.int64 or slots.shape != block_ids.shape):
        raise ValueError("slots must be int64 like block_ids")
    dev = key_caches[0].device
    kt, vt = tables if tables is not None else (layer_table(key_caches, dev), layer_table(value_caches, dev))
    call(name, _ptr(kt), _ptr(vt), L, _ptr(block_ids), block_ids.shape[0], nb, nbytes, _ptr(slots),
         records.shape[0], _ptr(records), _stream(stream))


def swap_out(key_caches, value_caches, block_ids: torch.Tensor, records: torch.Tensor, *,
             slots: Optional[torch.Tensor] = None, tables=None,
             stream: Optional[torch.cuda.Stream] = None) -> None:
    """Blocks -> pinned host records [R, layers, 2, block_nbytes]
    (rllm_cache_swap_out); synchronise before reading ``records``."""
    _swap("rllm_cache_swap_out", key_caches, value_caches, block_ids, records, slots, tables, stream)


def swap_in(key_caches, value_caches, block_ids: torch.Tensor, records: torch.Tensor, *,
            slots: Optional[torch.Tensor] = None, tables=None,
            stream: Optional[torch.cuda.Stream] = None) -> None:
    """Pinned host records -> blocks (rllm_cache_swap_in)."""
    _swap("rllm_cache_swap_in", key_caches, value_caches, block_ids, records, slots, tables, stream)


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, *, out: Optional[torch.Tensor] = None,
            stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """RmsNorm::forward (crates/rllm-model/src/layers.rs:128-140) over the last
    dimension, through rllm_rmsnorm_ex."""
    dt = _TORCH_16.get(x.dtype)
    if dt is None or weight.dtype != x.dtype or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise ValueError("x and weight must share a 16-bit dtype; weight is [hidden]")
    out = torch.empty_like(x) if out is None else out
    if not _dense_on_one_gpu(x, weight, out):
        for t in (x, weight, out):
            if not t.is_contiguous() or t.device != x.device:
                raise ValueError("tensors must be contiguous and on one device")
    call("rllm_rmsnorm_ex", _ptr(out), _ptr(x), _ptr(weight), x.shape[-1], x.numel(), eps, dt, _stream(stream))
    return out


def silu_mul(gate: torch.Tensor, up: torch.Tensor, *, out: Optional[torch.Tensor] = None,
             stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """silu(gate) * up in the activation dtype (crates/rllm-model/src/
    layers.rs:214-220), through rllm_silu_mul_ex."""
    dt = _TORCH_16.get(gate.dtype)
    if dt is None or up.dtype != gate.dtype or up.shape != gate.shape:
        raise ValueError("gate and up must share a shape and a 16-bit dtype")
    out = torch.empty_like(gate) if out is None else out
    if not _dense_on_one_gpu(gate, up, out):
        for t in (gate, up, out):
            if not t.is_contiguous() or t.device != gate.device:
                raise ValueError("tensors must be contiguous and on one device")
    call("rllm_silu_mul_ex", _ptr(out), _ptr(gate), _ptr(up), gate.numel(), dt, _stream(stream))
    return out
