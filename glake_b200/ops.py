"""Custom-op layer with the reference's call signatures
(GLakeServe/vllm/_custom_ops.py:34-52, :238-252 and the flash_attn_2_cuda.fwd_kvcache
call at GLakeServe/vllm/attention/backends/xformers.py:407-430), forwarding to
libvtensor's C ABI.  Tensors are only unwrapped to pointers and strides here; all
work happens in the CUDA kernels.  Non-CUDA tensors are rejected: there is no
CPU path.
"""
import contextlib
import ctypes
import functools
from ctypes import byref, c_size_t, c_void_p

import torch

from ._lib import VT_KV_BF16, VT_KV_FP8_E4M3, VT_KV_INT4, check, lib

_workspaces = {}


# Host time per call matters for short sequences (the kernels take a few microseconds), hence: addresses go to ctypes as
# plain integers, the device is only switched when it is not the current one, sizes that the library computes from
# shapes alone are remembered.
def _stream():
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _ptr(t):
    return t.data_ptr() if t is not None else None


_SAME_DEVICE = contextlib.nullcontext()


def _on(device):
    """Context in which ``device`` is the current device."""
    index = device.index
    return _SAME_DEVICE if index is None or index == torch.cuda.current_device() else torch.cuda.device(device)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(call, *shape):
    need = c_size_t()
    check(getattr(lib, call)(*shape, byref(need)), call)
    return need.value


def _require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("glake_b200 ops need CUDA tensors: there is no CPU fallback")


def _kv_dtype(kv_cache_dtype):
    if kv_cache_dtype in ("auto", "bf16", "bfloat16", None):
        return VT_KV_BF16
    if kv_cache_dtype in ("fp8", "fp8_e4m3"):
        return VT_KV_FP8_E4M3
    if kv_cache_dtype == "int4":
        return VT_KV_INT4
    raise RuntimeError(f"unsupported kv_cache_dtype {kv_cache_dtype!r} (bf16, fp8_e4m3 and int4 only)")


def kv_row_bytes(num_kv_heads, head_size, kv_cache_dtype="auto"):
    """Bytes of one token's K (or V) row of all kv heads in a range of this cache type."""
    n = c_size_t()
    check(lib.vt_kv_row_bytes(num_kv_heads, head_size, _kv_dtype(kv_cache_dtype), byref(n)), "vt_kv_row_bytes")
    return n.value


def new_workspace(device, batch, num_heads, head_size, max_seq_len, scored=False):
    """A private, zero-filled scratch buffer for ``decode_step(..., workspace=...)``; ``scored`` adds
    the room that ``scores=`` needs."""
    call = "vt_decode_scored_workspace_bytes" if scored else "vt_decode_attn_workspace_bytes"
    return torch.zeros(_workspace_bytes(call, batch, num_heads, head_size, int(max_seq_len)), dtype=torch.uint8, device=device)


def _device_index(device):
    return device.index if device.index is not None else torch.cuda.current_device()


def _scratch(device, nbytes):
    """Scratch cached per device and stream and grown on demand: calls of one stream run back to back, calls of two
    streams may overlap.  While the stream is being captured the buffer belongs to the capture instead: a graph must
    not hold the address of a buffer that a later, larger call replaces, nor share one with another graph."""
    index = _device_index(device)
    with _on(device):
        if torch.cuda.is_current_stream_capturing():
            return torch.empty(max(nbytes, 1 << 10), dtype=torch.uint8, device=device)
    key = (index, torch._C._cuda_getCurrentRawStream(index))
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = buf
    return buf


def attn_workspace(device, batch, num_heads, head_size, max_seq_len):
    """Scratch for the split-K partials, cached per device and stream and grown on demand.
    One buffer serves every layer because layers run back to back on one stream."""
    return _scratch(device, _workspace_bytes("vt_decode_attn_workspace_bytes", batch, num_heads, head_size, int(max_seq_len)))


def reshape_and_cache(key, value, key_cache, value_cache, slot_m, slot_mapping, seq_lens, cache_seq_lens,
                      max_seq_len, num_kv_heads, head_size, kv_cache_dtype="auto", k_scale=None, v_scale=None):
    """Append K/V rows into the slots' contiguous ranges.

    Positional arguments as in the reference (csrc/cache.h:18-29): ``key_cache`` /
    ``value_cache`` are int64 device tensors of base addresses indexed by slot id,
    ``slot_m`` the per-entry destination byte offsets, ``slot_mapping`` the slot
    ids, ``max_seq_len`` 1 for decode.  The keyword arguments add the fp8 e4m3
    cache and the 4-bit cache (``"int4"``: an e4m3 scale per 32 dims, see vt_append) with
    per-kv-head scales (float32 device tensors of num_kv_heads, for both from :func:`kv_scales`)."""
    _require_cuda(key, value, key_cache, value_cache, slot_m, slot_mapping)
    if key.dtype != torch.bfloat16 or value.dtype != torch.bfloat16:
        raise RuntimeError("reshape_and_cache: key/value must be bfloat16")
    key = key.view(-1, num_kv_heads, head_size) if key.dim() == 2 else key
    value = value.view(-1, num_kv_heads, head_size) if value.dim() == 2 else value
    if key.stride(2) != 1 or key.stride(1) != head_size or value.stride(2) != 1 or value.stride(1) != head_size:
        raise RuntimeError("reshape_and_cache: key/value rows must be contiguous [kv_heads, head_size]")
    batch = slot_mapping.numel()
    with _on(key.device):
        check(lib.vt_append(_ptr(key), _ptr(value), key.stride(0), value.stride(0), _ptr(key_cache),
                            _ptr(value_cache), _ptr(slot_m), _ptr(slot_mapping), _ptr(seq_lens),
                            _ptr(cache_seq_lens), int(max_seq_len), batch, num_kv_heads, head_size,
                            _kv_dtype(kv_cache_dtype), _ptr(k_scale), _ptr(v_scale), _stream()), "vt_append")


VT_ROPE_WRITE_KEY = 1


def rotary_embedding_and_cache(positions, query, key, value, head_size, cos_sin_cache, is_neox, key_cache,
                               value_cache, slot_m, slot_mapping, seq_lens, cache_seq_lens, max_seq_len,
                               num_kv_heads, kv_cache_dtype="auto", k_scale=None, v_scale=None, write_key=False):
    """``rotary_embedding`` (GLakeServe/vllm/_custom_ops.py:81-90) and
    ``reshape_and_cache`` in one launch: ``query`` is rotated in place, the rotated
    key and the value rows go straight into the slots' ranges.  The first seven
    arguments are rotary_embedding's (plus ``value``), the rest reshape_and_cache's.
    ``key`` itself is only rewritten with ``write_key=True``."""
    _require_cuda(positions, query, key, value, cos_sin_cache, key_cache, value_cache, slot_m, slot_mapping)
    if not (query.dtype == key.dtype == value.dtype == cos_sin_cache.dtype == torch.bfloat16):
        raise RuntimeError("rotary_embedding_and_cache: bfloat16 tensors only")
    q2 = query.view(-1, query.shape[-1])
    k2 = key.view(-1, key.shape[-1])
    v2 = value.view(-1, value.shape[-1])
    if q2.stride(1) != 1 or k2.stride(1) != 1 or v2.stride(1) != 1 or not cos_sin_cache.is_contiguous():
        raise RuntimeError("rotary_embedding_and_cache: rows must be contiguous")
    if q2.shape[-1] % head_size or k2.shape[-1] != num_kv_heads * head_size or v2.shape[-1] != k2.shape[-1]:
        raise RuntimeError("rotary_embedding_and_cache: inconsistent head counts")
    with _on(query.device):
        check(lib.vt_rope_append(_ptr(positions), _ptr(q2), q2.stride(0), q2.shape[-1] // head_size, _ptr(k2), _ptr(v2),
                                 k2.stride(0), v2.stride(0), _ptr(cos_sin_cache), cos_sin_cache.shape[1],
                                 1 if is_neox else 0, _ptr(key_cache), _ptr(value_cache), _ptr(slot_m),
                                 _ptr(slot_mapping), _ptr(seq_lens), _ptr(cache_seq_lens), int(max_seq_len),
                                 slot_mapping.numel(), num_kv_heads, head_size, _kv_dtype(kv_cache_dtype),
                                 _ptr(k_scale), _ptr(v_scale), VT_ROPE_WRITE_KEY if write_key else 0, _stream()),
              "vt_rope_append")


def rms_norm(out, input, weight, epsilon):
    """out = rms_norm(input) * weight (GLakeServe/vllm/_custom_ops.py:104-106)."""
    _require_cuda(out, input, weight)
    if not (out.dtype == input.dtype == weight.dtype == torch.bfloat16):
        raise RuntimeError("rms_norm: bfloat16 tensors only")
    hidden = input.shape[-1]
    x, o = input.view(-1, hidden), out.view(-1, hidden)
    if x.stride(1) != 1 or o.stride(1) != 1:
        raise RuntimeError("rms_norm: rows must be contiguous")
    with _on(input.device):
        check(lib.vt_rms_norm(_ptr(o), _ptr(x), _ptr(weight), float(epsilon), x.shape[0], hidden, x.stride(0),
                              o.stride(0), _stream()), "vt_rms_norm")


def fused_add_rms_norm(input, residual, weight, epsilon):
    """residual += input; input = rms_norm(residual) * weight, both in place
    (GLakeServe/vllm/_custom_ops.py:109-111)."""
    _require_cuda(input, residual, weight)
    if not (input.dtype == residual.dtype == weight.dtype == torch.bfloat16):
        raise RuntimeError("fused_add_rms_norm: bfloat16 tensors only")
    if not (input.is_contiguous() and residual.is_contiguous()):
        raise RuntimeError("fused_add_rms_norm: contiguous tensors only")
    hidden = input.shape[-1]
    with _on(input.device):
        check(lib.vt_fused_add_rms_norm(_ptr(input), _ptr(residual), _ptr(weight), float(epsilon),
                                        input.numel() // hidden, hidden, _stream()), "vt_fused_add_rms_norm")


def kv_scales(x, num_kv_heads, head_size):
    """Per-kv-head scale = amax / 448 of x ([tokens, kv_heads, head_size] bf16)."""
    _require_cuda(x)
    x = x.view(-1, num_kv_heads, head_size)
    out = torch.empty(num_kv_heads, dtype=torch.float32, device=x.device)
    with _on(x.device):
        check(lib.vt_kv_scales(_ptr(x), x.stride(0), x.shape[0], num_kv_heads, head_size, _ptr(out), _stream()),
              "vt_kv_scales")
    return out


def _check_scores(scores, num_kv_heads, device, what):
    if scores.dim() != 3 or scores.dtype != torch.float32 or scores.shape[1] != num_kv_heads or scores.stride(2) != 1:
        raise RuntimeError(f"{what}: scores must be float32 [slots, kv_heads, rows] with contiguous rows")
    if scores.device != device:
        raise RuntimeError(f"{what}: scores must be on the device of the other tensors")


def _scored(out, query, key, value, slot_m, k_table, v_table, num_kv_heads, scale, seq_lens, max_seq_len, slot_ids,
            kv_dtype, k_scale, v_scale, lse, scores, workspace=None):
    batch, num_heads, head_size = query.shape
    _require_cuda(scores)
    _check_scores(scores, num_kv_heads, query.device, "scores")
    ws = workspace
    if ws is None:
        ws = _scratch(query.device, _workspace_bytes("vt_decode_scored_workspace_bytes", batch, num_heads, head_size, int(max_seq_len)))
    with _on(query.device):
        check(lib.vt_decode_step_scored(_ptr(out), out.stride(0), _ptr(query), query.stride(0), _ptr(key), _ptr(value),
                                        key.stride(0) if key is not None else 0,
                                        value.stride(0) if value is not None else 0, _ptr(slot_m), (int(k_table)),
                                        (int(v_table)), _ptr(slot_ids), _ptr(seq_lens), batch, num_heads,
                                        num_kv_heads, head_size, int(max_seq_len), float(scale), kv_dtype, _ptr(k_scale),
                                        _ptr(v_scale), _ptr(lse), _ptr(scores), scores.stride(0), scores.stride(1),
                                        scores.shape[2], _ptr(ws), ws.numel(), _stream()), "vt_decode_step_scored")


def _decode(out, query, k_table, v_table, num_kv_heads, scale, seq_lens, max_seq_len, slot_ids, kv_dtype,
            k_scale, v_scale, lse, num_splits, maps=None):
    batch, num_heads, head_size = query.shape
    ws = attn_workspace(query.device, batch, num_heads, head_size, max_seq_len)
    if maps is not None and num_splits == 0:
        # plain attention through the tensor-map entry point (no rows to append)
        with _on(query.device):
            check(lib.vt_decode_step_tma(_ptr(out), out.stride(0), _ptr(query), query.stride(0), None, None, 0, 0, None,
                                         (int(k_table)), (int(v_table)), _ptr(slot_ids), _ptr(seq_lens),
                                         batch, num_heads, num_kv_heads, head_size, int(max_seq_len), float(scale),
                                         kv_dtype, _ptr(k_scale), _ptr(v_scale), _ptr(lse), _ptr(ws), ws.numel(), 0,
                                         _ptr(maps), _stream()), "vt_decode_step_tma")
        return
    with _on(query.device):
        check(lib.vt_decode_attn(_ptr(out), out.stride(0), _ptr(query), query.stride(0), (int(k_table)),
                                 (int(v_table)), _ptr(slot_ids), _ptr(seq_lens), batch, num_heads,
                                 num_kv_heads, head_size, int(max_seq_len), float(scale), kv_dtype, _ptr(k_scale),
                                 _ptr(v_scale), _ptr(lse), _ptr(ws), ws.numel(), int(num_splits), _stream()),
              "vt_decode_attn")


def paged_attention_v1(out, query, key_cache, value_cache, num_kv_heads, scale, seq_lens, block_size, max_seq_len,
                       alibi_slopes, kv_cache_dtype, kv_scale, slot_mapping, k_scale=None, v_scale=None,
                       num_splits=0, maps=None, scores=None):
    """Decode attention with the reference's vTensor signature (csrc/ops.h:6-19):
    ``key_cache`` / ``value_cache`` are the device addresses (ints) of the per-layer
    pointer tables, ``slot_mapping`` the slot ids.  ``block_size`` must be 1 (the
    token-major contiguous layout, vllm/attention/ops/paged_attn.py:105).  ``maps`` (from
    :func:`decode_maps`, fp8 cache) selects the tcgen05 kernel where the head counts allow.
    ``scores`` (float32 ``[slots, kv_heads, rows]``) also receives the softmax weight of every cached
    row, summed over the q heads of its kv head: ``scores[slot, j, t] += ...`` (``maps`` then stay
    unused, and ``num_splits`` must be 0)."""
    _require_cuda(out, query, seq_lens, slot_mapping, maps)
    if alibi_slopes is not None:
        raise RuntimeError("paged_attention_v1: ALiBi is not supported on the vTensor path")
    if block_size != 1:
        raise RuntimeError("paged_attention_v1: the vTensor layout is block_size 1")
    if query.dtype != torch.bfloat16 or out.dtype != torch.bfloat16:
        raise RuntimeError("paged_attention_v1: bf16 only")
    kvd = _kv_dtype(kv_cache_dtype)
    if kvd != VT_KV_BF16 and k_scale is None:
        k_scale = torch.full((num_kv_heads,), float(kv_scale), dtype=torch.float32, device=query.device)
        v_scale = k_scale
    if scores is not None:
        if num_splits:
            raise RuntimeError("paged_attention_v1: scores needs num_splits = 0")
        _scored(out, query, None, None, None, key_cache, value_cache, num_kv_heads, scale, seq_lens, max_seq_len,
                slot_mapping, kvd, k_scale, v_scale, None, scores)
        return
    _decode(out, query, key_cache, value_cache, num_kv_heads, scale, seq_lens, max_seq_len, slot_mapping, kvd,
            k_scale, v_scale, None, num_splits, maps)


def fwd_kvcache(q, k_table_ptr, v_table_ptr, max_seq_len, num_kv_heads, batch, slot_mapping, k_new, v_new,
                seq_lens, rotary_cos, rotary_sin, cache_batch_idx, block_table, alibi_slopes, out, softmax_scale,
                causal, window_left, window_right, rotary_interleaved, num_splits, kv_cache_dtype="auto",
                k_scale=None, v_scale=None, scores=None):
    """The 22-positional-argument call the reference's backend makes into its
    flash-attention fork (xformers.py:407-430): q ``[B, 1, H, D]``, pointer-table
    addresses, ``slot_mapping`` slot ids, ``seq_lens`` int32.  Returns ``(out, lse)``
    with out ``[B, 1, H, D]`` and lse ``[B, H, 1]`` float32.  ``scores`` accumulates the weights as in
    :func:`paged_attention_v1` (single-token form).  The arguments the
    reference always passes as None / -1 must be None / -1 here."""
    _require_cuda(q, slot_mapping, seq_lens)
    for name, v in (("k_new", k_new), ("v_new", v_new), ("rotary_cos", rotary_cos), ("rotary_sin", rotary_sin),
                    ("cache_batch_idx", cache_batch_idx), ("block_table", block_table),
                    ("alibi_slopes", alibi_slopes)):
        if v is not None:
            raise RuntimeError(f"fwd_kvcache: {name} is not supported on the vTensor path")
    if window_left != -1 or window_right != -1:
        raise RuntimeError("fwd_kvcache: sliding window is not supported")
    if q.dim() != 4:
        raise RuntimeError("fwd_kvcache: q must be [B, S, H, D]")
    if q.shape[1] != 1:
        if scores is not None:
            raise RuntimeError("fwd_kvcache: scores needs seqlen_q == 1 (prompt_scores serves prompts)")
        # prefix-extend form (xformers.py:362-385): S new tokens per sequence, causal over the range
        if not causal:
            raise RuntimeError("fwd_kvcache: seqlen_q > 1 needs causal=True")
        b, s, h, d = q.shape
        qc = q.contiguous().view(b * s, h, d)
        o = out if out is not None else torch.empty(b, s, h, d, dtype=q.dtype, device=q.device)
        q_lens = torch.full((b,), s, dtype=torch.int32, device=q.device)
        q_start = torch.arange(b, dtype=torch.int32, device=q.device) * s
        prefill_attention(o.view(b * s, h, d), qc, k_table_ptr, v_table_ptr, num_kv_heads, softmax_scale,
                          slot_mapping, seq_lens, q_lens, q_start, s, kv_cache_dtype=kv_cache_dtype, k_scale=k_scale,
                          v_scale=v_scale)
        return o, None
    b, _, h, d = q.shape
    q3 = q.view(b, h, d) if q.is_contiguous() else q[:, 0]
    o = out if out is not None else torch.empty(b, 1, h, d, dtype=q.dtype, device=q.device)
    lse = torch.empty(b, h, dtype=torch.float32, device=q.device)
    if scores is not None:
        _scored(o.view(b, h, d), q3, None, None, None, k_table_ptr, v_table_ptr, num_kv_heads, softmax_scale, seq_lens,
                max_seq_len, slot_mapping, _kv_dtype(kv_cache_dtype), k_scale, v_scale, lse, scores)
        return o, lse.unsqueeze(-1)
    _decode(o.view(b, h, d), q3, k_table_ptr, v_table_ptr, num_kv_heads, softmax_scale, seq_lens, max_seq_len,
            slot_mapping, _kv_dtype(kv_cache_dtype), k_scale, v_scale, lse, 0)
    return o, lse.unsqueeze(-1)


def decode_step(out, query, key, value, key_cache, value_cache, slot_m, slot_mapping, seq_lens, max_seq_len,
                num_kv_heads, scale, kv_cache_dtype="auto", k_scale=None, v_scale=None, lse=None, overlap=False,
                workspace=None, maps=None, clean_scratch=False, scores=None):
    """``reshape_and_cache`` (decode form) + ``paged_attention_v1`` in one call; one
    kernel launch for a bf16 cache.  ``key_cache`` / ``value_cache`` are the device
    addresses of the layer's pointer tables (ints), ``slot_m`` the destination byte
    offsets, ``slot_mapping`` the slot ids, ``seq_lens`` the contexts INCLUDING the
    appended token.  query/out ``[B, H, D]``, key/value ``[B, KVH, D]`` bf16.
    ``overlap=True`` lets the launch overlap the previous ``decode_step`` on the
    stream (VT_STEP_OVERLAP): only for a different layer's ranges, see vtensor.h;
    ``overlap="early_kv"`` (VT_STEP_EARLY_KV) is the form for inputs that the preceding
    kernel produces: cache rows stream early, q / key / value are read after it finished.
    Pass a private zero-filled ``workspace`` (uint8 tensor) in both cases.
    ``maps`` (from :func:`decode_maps`, fp8 cache only) selects the tcgen05 kernel where
    the head counts allow; other shapes run as without it.  ``clean_scratch=True``
    (VT_STEP_CLEAN_SCRATCH): ``workspace`` is private, was zero-filled once and is used by
    nothing but these calls, so the call need not clear its counters first.  ``scores``
    accumulates the weights as in :func:`paged_attention_v1`; the overlap forms do not apply then,
    and ``workspace`` comes from ``new_workspace(..., scored=True)``."""
    _require_cuda(out, query, key, value, slot_m, slot_mapping, seq_lens, maps)
    batch, num_heads, head_size = query.shape
    key = key.view(batch, num_kv_heads, head_size)
    value = value.view(batch, num_kv_heads, head_size)
    if overlap and workspace is None:
        raise RuntimeError("decode_step(overlap=True) needs a private zero-filled workspace")
    if scores is not None:
        if overlap:
            raise RuntimeError("decode_step: scores excludes overlap")
        _scored(out, query, key, value, slot_m, key_cache, value_cache, num_kv_heads, scale, seq_lens, max_seq_len,
                slot_mapping, _kv_dtype(kv_cache_dtype), k_scale, v_scale, lse, scores, workspace)
        return
    ws = workspace if workspace is not None else attn_workspace(query.device, batch, num_heads, head_size,
                                                                max_seq_len)
    flags = (2 if overlap == "early_kv" else (1 if overlap else 0)) | (4 if clean_scratch else 0)
    if clean_scratch and workspace is None:
        raise RuntimeError("decode_step(clean_scratch=True) needs a private zero-filled workspace")
    if maps is not None:
        with _on(query.device):
            check(lib.vt_decode_step_tma(_ptr(out), out.stride(0), _ptr(query), query.stride(0), _ptr(key), _ptr(value),
                                         key.stride(0), value.stride(0), _ptr(slot_m), (int(key_cache)),
                                         (int(value_cache)), _ptr(slot_mapping), _ptr(seq_lens), batch,
                                         num_heads, num_kv_heads, head_size, int(max_seq_len), float(scale),
                                         _kv_dtype(kv_cache_dtype), _ptr(k_scale), _ptr(v_scale), _ptr(lse), _ptr(ws),
                                         ws.numel(), flags, _ptr(maps), _stream()), "vt_decode_step_tma")
        return
    with _on(query.device):
        check(lib.vt_decode_step(_ptr(out), out.stride(0), _ptr(query), query.stride(0), _ptr(key), _ptr(value),
                                 key.stride(0), value.stride(0), _ptr(slot_m), (int(key_cache)),
                                 (int(value_cache)), _ptr(slot_mapping), _ptr(seq_lens), batch, num_heads,
                                 num_kv_heads, head_size, int(max_seq_len), float(scale), _kv_dtype(kv_cache_dtype),
                                 _ptr(k_scale), _ptr(v_scale), _ptr(lse), _ptr(ws), ws.numel(), flags, _stream()),
              "vt_decode_step")


def step_is_fused(kv_cache_dtype):
    """Whether decode_step on the persistent schedule is ONE launch for this cache type: the
    attention kernel appends the new rows itself (bf16: copied, fp8 and int4: quantised on the way)."""
    return _kv_dtype(kv_cache_dtype) in (VT_KV_BF16, VT_KV_FP8_E4M3, VT_KV_INT4)


def prefill_tma_supported(num_kv_heads):
    """Whether ``prefill_maps`` / the TMA prefill path take this kv-head count (a
    32-token box must never straddle a 2 MiB chunk)."""
    return num_kv_heads & (num_kv_heads - 1) == 0 and num_kv_heads * 32 <= 8192


def prefill_maps(k_bases, v_bases, num_kv_heads, head_size, max_tokens, device):
    """Device table of TMA tensor maps for ``prefill_attention(..., maps=...)``:
    ``k_bases[i]`` / ``v_bases[i]`` are slot i's range bases of one layer
    (``getKeyDevicePtr`` / ``getValueDevicePtr``).  Valid while the slots live."""
    n = len(k_bases)
    kb = (ctypes.c_uint64 * n)(*[int(x) for x in k_bases])
    vb = (ctypes.c_uint64 * n)(*[int(x) for x in v_bases])
    host = torch.empty(n * 256 + 64, dtype=torch.uint8)
    off = (-host.data_ptr()) % 64
    with _on(device):
        check(lib.vt_prefill_maps_encode(kb, vb, n, num_kv_heads, head_size, int(max_tokens),
                                         c_void_p(host.data_ptr() + off)), "vt_prefill_maps_encode")
    return host[off: off + n * 256].to(device)


def decode_tma_supported(num_heads, num_kv_heads, kv_cache_dtype):
    """Whether ``decode_step(..., maps=...)`` runs the tcgen05 kernel for this shape (fp8 cache,
    kv heads a power of two >= 8, at most 4 q heads per kv head); other shapes ignore the maps."""
    g = num_heads // num_kv_heads
    return (_kv_dtype(kv_cache_dtype) == VT_KV_FP8_E4M3 and num_kv_heads % 8 == 0
            and num_kv_heads & (num_kv_heads - 1) == 0 and num_kv_heads <= 256 and g in (1, 2, 4))


def decode_maps(k_bases, v_bases, num_kv_heads, head_size, max_tokens, device, kv_cache_dtype="fp8"):
    """Device table of TMA tensor maps for ``decode_step(..., maps=...)`` over fp8 ranges:
    ``k_bases[i]`` / ``v_bases[i]`` are slot i's range bases of one layer.  Valid while the slots live."""
    n = len(k_bases)
    kb = (ctypes.c_uint64 * n)(*[int(x) for x in k_bases])
    vb = (ctypes.c_uint64 * n)(*[int(x) for x in v_bases])
    host = torch.empty(n * 256 + 64, dtype=torch.uint8)
    off = (-host.data_ptr()) % 64
    with _on(device):
        check(lib.vt_decode_maps_encode(kb, vb, n, num_kv_heads, head_size, _kv_dtype(kv_cache_dtype), int(max_tokens),
                                        c_void_p(host.data_ptr() + off)), "vt_decode_maps_encode")
    return host[off: off + n * 256].to(device)


def widen_fp8_ranges(key_cache, value_cache, num_kv_heads, head_size, slot_mapping, seq_lens, k_scale, v_scale,
                     pad_rows=64, kv_cache_dtype="fp8_e4m3"):
    """Dense bf16 copies of the slots' fp8 (or, with ``kv_cache_dtype="int4"``, 4-bit) rows for the prompt kernels: returns
    (k_bases, v_bases, holder) where ``k_bases`` / ``v_bases`` are int64 device tensors
    of one scratch range address per batch entry (usable as pointer tables with slot ids
    0..B-1) and ``holder`` keeps the scratch alive.  Every entry's range is padded to a
    multiple of ``pad_rows`` rows so that whole-tile fetches at its ragged end stay
    inside the buffer.  Synchronises once to learn the context lengths."""
    lens = [int(x) for x in seq_lens.tolist()]
    row = num_kv_heads * head_size
    padded = [(n + pad_rows - 1) // pad_rows * pad_rows + pad_rows for n in lens]
    total = sum(padded)
    dev = seq_lens.device
    buf = torch.zeros(2, max(total, 1), row, dtype=torch.bfloat16, device=dev)
    starts, acc = [], 0
    for n in padded:
        starts.append(acc)
        acc += n
    kb = torch.tensor([buf[0].data_ptr() + s * row * 2 for s in starts], dtype=torch.int64, device=dev)
    vb = torch.tensor([buf[1].data_ptr() + s * row * 2 for s in starts], dtype=torch.int64, device=dev)
    if _kv_dtype(kv_cache_dtype) == VT_KV_INT4:
        dequantize_ranges(buf[0].view(-1, num_kv_heads, head_size), buf[1].view(-1, num_kv_heads, head_size), key_cache,
                          value_cache, num_kv_heads, slot_mapping, seq_lens,
                          torch.tensor(starts, dtype=torch.int32, device=dev), max(lens) if lens else 0, kv_cache_dtype,
                          k_scale, v_scale)
        return kb, vb, (buf, padded)
    with _on(dev):
        check(lib.vt_kv_widen((int(key_cache)), (int(value_cache)), _ptr(slot_mapping), _ptr(seq_lens),
                              len(lens), num_kv_heads, head_size, max(lens) if lens else 0, _ptr(k_scale), _ptr(v_scale),
                              _ptr(kb), _ptr(vb), _stream()), "vt_kv_widen")
    return kb, vb, (buf, padded)


def dequantize_ranges(key_out, value_out, key_cache, value_cache, num_kv_heads, slot_mapping, seq_lens, row_start,
                      max_seq_len, kv_cache_dtype="fp8_e4m3", k_scale=None, v_scale=None):
    """Reads a quantised cache back: rows ``0 .. seq_lens[i]`` of entry i's ranges as bf16 rows
    ``row_start[i] ..`` of ``key_out`` / ``value_out`` ([rows, kv_heads, head_size], contiguous; one
    of the two may be None).  ``key_cache`` / ``value_cache`` are pointer-table addresses (ints),
    ``seq_lens`` / ``row_start`` int32, ``max_seq_len`` a host bound of ``seq_lens``."""
    outs = [t for t in (key_out, value_out) if t is not None]
    if not outs:
        raise RuntimeError("dequantize_ranges: no output")
    _require_cuda(*outs, slot_mapping, seq_lens, row_start, k_scale, v_scale)
    head_size = outs[0].shape[-1]
    for t in outs:
        if t.dtype != torch.bfloat16 or not t.is_contiguous() or t.numel() % (num_kv_heads * head_size):
            raise RuntimeError("dequantize_ranges: outputs must be contiguous bfloat16 [rows, kv_heads, head_size]")
    if slot_mapping.dtype != torch.int64 or seq_lens.dtype != torch.int32 or row_start.dtype != torch.int32:
        raise RuntimeError("dequantize_ranges: slot_mapping must be int64, seq_lens and row_start int32")
    with _on(outs[0].device):
        check(lib.vt_kv_dequant((int(key_cache)), (int(value_cache)), _ptr(slot_mapping), _ptr(seq_lens),
                                _ptr(row_start), slot_mapping.numel(), num_kv_heads, head_size, int(max_seq_len),
                                _kv_dtype(kv_cache_dtype), _ptr(k_scale), _ptr(v_scale), _ptr(key_out), _ptr(value_out),
                                _stream()), "vt_kv_dequant")


def prefill_attention(out, query, key_cache, value_cache, num_kv_heads, scale, slot_mapping, seq_lens, q_lens,
                      q_start, max_q_len, maps=None, kv_cache_dtype="auto", k_scale=None, v_scale=None):
    """Causal attention of the new tokens over the slots' whole ranges (the new rows
    already appended with ``reshape_and_cache``).  query/out ``[tokens, H, D]`` bf16,
    ``key_cache`` / ``value_cache`` the pointer-table addresses (ints), ``seq_lens``
    the contexts including the new tokens, ``q_lens`` / ``q_start`` int32 per entry.
    With ``maps`` (from :func:`prefill_maps`) K/V tiles are fetched by TMA tensor copies.
    An fp8 e4m3 or int4 cache (``kv_cache_dtype``, per-kv-head ``k_scale`` / ``v_scale``) is first
    widened into bf16 scratch ranges (:func:`widen_fp8_ranges`), over which the same
    kernels run, with tensor maps of the scratch where the head count allows."""
    _require_cuda(out, query, slot_mapping, seq_lens, q_lens, q_start, maps)
    if query.dtype != torch.bfloat16:
        raise RuntimeError("prefill_attention: bf16 only")
    n, num_heads, head_size = query.shape
    holder = None
    if _kv_dtype(kv_cache_dtype) != VT_KV_BF16:
        if k_scale is None or v_scale is None:
            raise RuntimeError(f"prefill_attention: an {kv_cache_dtype} cache needs k_scale and v_scale")
        kb, vb, holder = widen_fp8_ranges(key_cache, value_cache, num_kv_heads, head_size, slot_mapping, seq_lens,
                                          k_scale, v_scale, kv_cache_dtype=kv_cache_dtype)
        batch = slot_mapping.numel()
        key_cache, value_cache = kb.data_ptr(), vb.data_ptr()
        slot_mapping = torch.arange(batch, dtype=torch.int64, device=query.device)
        maps = None
        if prefill_tma_supported(num_kv_heads):
            maps = prefill_maps(kb.tolist(), vb.tolist(), num_kv_heads, head_size, max(holder[1]), query.device)
        holder = (holder, kb, vb, slot_mapping, maps)
    args = (_ptr(out), out.stride(0), _ptr(query), query.stride(0), (int(key_cache)),
            (int(value_cache)), _ptr(slot_mapping), _ptr(seq_lens), _ptr(q_lens),
            _ptr(q_start), slot_mapping.numel(), num_heads, num_kv_heads, head_size,
            int(max_q_len), float(scale), VT_KV_BF16, None)
    with _on(query.device):
        if maps is None:
            check(lib.vt_prefill_attn(*args, _stream()), "vt_prefill_attn")
        else:
            check(lib.vt_prefill_attn_tma(*args, _ptr(maps), _stream()), "vt_prefill_attn_tma")
    if holder is not None:
        # the scratch must outlive the kernels queued above: torch's allocator reuses a freed
        # block only in stream order on the stream that allocated it, which is this one
        del holder


def prompt_scores(scores, query, key_cache, num_kv_heads, scale, slot_mapping, seq_lens, q_lens, q_start, max_seq_len,
                  window, kv_cache_dtype="auto", k_scale=None):
    """Adds the attention weights of a prompt's last queries to ``scores``: what
    :func:`paged_attention_v1` with ``scores`` adds per decode step, for the last
    ``min(window, q_lens[i])`` of entry i's new tokens at once.  ``query`` ``[tokens, H, D]`` bf16,
    ``key_cache`` the address of the K pointer table, ``seq_lens`` / ``q_lens`` / ``q_start`` as in
    :func:`prefill_attention` (after the rows were appended).  A quantised cache is read back into
    bf16 scratch first (``k_scale`` needed), at most 1 GiB of it at a time."""
    _require_cuda(scores, query, slot_mapping, seq_lens, q_lens, q_start, k_scale)
    if query.dtype != torch.bfloat16 or query.dim() != 3 or query.stride(2) != 1 or query.stride(1) != query.shape[2]:
        raise RuntimeError("prompt_scores: query must be bfloat16 [tokens, heads, head_size] with contiguous rows")
    if slot_mapping.dtype != torch.int64 or any(t.dtype != torch.int32 for t in (seq_lens, q_lens, q_start)):
        raise RuntimeError("prompt_scores: slot_mapping must be int64, seq_lens, q_lens and q_start int32")
    _check_scores(scores, num_kv_heads, query.device, "prompt_scores")
    _, num_heads, head_size = query.shape
    batch, max_seq_len = slot_mapping.numel(), int(max_seq_len)
    dtype = _kv_dtype(kv_cache_dtype)
    step, table, range_ids = max(batch, 1), (int(key_cache)), None
    if dtype != VT_KV_BF16:
        if k_scale is None:
            raise RuntimeError(f"prompt_scores: an {kv_cache_dtype} cache needs k_scale")
        row = num_kv_heads * head_size * 2
        step = max(1, min(step, (1 << 30) // max(1, max_seq_len * row)))
        rows = torch.empty(step * max_seq_len, num_kv_heads, head_size, dtype=torch.bfloat16, device=query.device)
        range_ids = torch.arange(step, dtype=torch.int64, device=query.device)
        bases = range_ids * (max_seq_len * row) + rows.data_ptr()
        starts = (range_ids * max_seq_len).to(torch.int32)
        table = _ptr(bases)
    for b in range(0, batch, step):
        n = min(step, batch - b)
        slots, lens, qn, qs = slot_mapping, seq_lens, q_lens, q_start
        if n < batch:
            slots, lens, qn, qs = (t[b:b + n] for t in (slot_mapping, seq_lens, q_lens, q_start))
        need = _workspace_bytes("vt_prompt_scores_workspace_bytes", n, num_heads, num_kv_heads, head_size, max_seq_len, int(window))
        if range_ids is not None:
            dequantize_ranges(rows, None, key_cache, 0, num_kv_heads, slots, lens, starts[:n], max_seq_len, kv_cache_dtype,
                              k_scale)
        ws = _scratch(query.device, need)
        with _on(query.device):
            check(lib.vt_prompt_scores(_ptr(scores), scores.stride(0), scores.stride(1), scores.shape[2], _ptr(query),
                                       query.stride(0), table, _ptr(slots), _ptr(range_ids), _ptr(lens),
                                       _ptr(qn), _ptr(qs), n, num_heads, num_kv_heads, head_size, max_seq_len, int(window),
                                       float(scale), _ptr(ws), ws.numel(), _stream()), "vt_prompt_scores")


def evict_rows(scores, key_cache, value_cache, num_kv_heads, slot_mapping, seq_lens, max_seq_len, budget, sink=0, recent=0,
               kv_cache_dtype="auto", scores_out=None, head_size=128):
    """Cuts every sequence longer than ``budget`` rows to ``budget``: per kv head the first ``sink``
    rows, the last ``recent`` and the heaviest of the others by ``scores`` stay (equal weights: the
    lower row) and move to the front of their range in their old order; the scores move along
    (``scores_out``, default in place) and the ones behind become 0.  Returns the old row numbers
    int32 ``[B, kv_heads, budget]``, -1 behind the rows of a shorter sequence.  The slots of a call
    must be distinct.  Afterwards the sequences have ``min(seq_lens, budget)`` rows; telling the
    allocator is the caller's part (``VTensorCacheEngine.evict`` does both)."""
    _require_cuda(scores, scores_out, slot_mapping, seq_lens)
    if slot_mapping.dtype != torch.int64 or seq_lens.dtype != torch.int32:
        raise RuntimeError("evict_rows: slot_mapping must be int64, seq_lens int32")
    _check_scores(scores, num_kv_heads, slot_mapping.device, "evict_rows")
    out = scores if scores_out is None else scores_out
    if out.shape != scores.shape or out.stride() != scores.stride() or out.dtype != scores.dtype or out.device != scores.device:
        raise RuntimeError("evict_rows: scores_out must be laid out as scores")
    batch, dtype = slot_mapping.numel(), _kv_dtype(kv_cache_dtype)
    kept = torch.empty(batch, num_kv_heads, int(budget), dtype=torch.int32, device=scores.device)
    ws = _scratch(scores.device, _workspace_bytes("vt_evict_workspace_bytes", batch, num_kv_heads, int(budget), dtype))
    with _on(scores.device):
        check(lib.vt_evict_rows(_ptr(scores), _ptr(out), scores.stride(0), scores.stride(1), scores.shape[2],
                                (int(key_cache)), (int(value_cache)), _ptr(slot_mapping), _ptr(seq_lens),
                                batch, num_kv_heads, head_size, int(max_seq_len), int(budget), int(sink), int(recent), dtype,
                                _ptr(kept), _ptr(ws), ws.numel(), _stream()), "vt_evict_rows")
    return kept


def attn_plan(batch, num_heads, num_kv_heads, max_seq_len, kv_cache_dtype="auto", num_splits=0):
    """(tokens per partition, partitions per sequence, kernel variant) the library
    picks for this problem size."""
    a, b, c = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    check(lib.vt_decode_attn_plan(batch, num_heads, num_kv_heads, max_seq_len, _kv_dtype(kv_cache_dtype),
                                  num_splits, byref(a), byref(b), byref(c)), "vt_decode_attn_plan")
    return a.value, b.value, c.value


_VARIANTS = {None: -1, "auto": -1, "simt": 0, "mma": 1, "flat": 2}


def set_attn_tuning(variant="auto", part_tokens=0):
    """Process-wide planner override for benchmarks and tests: ``variant`` one of
    auto / simt / mma / flat, ``part_tokens`` tokens per split-K partition (0 = auto)."""
    check(lib.vt_attn_set_tuning(_VARIANTS[variant], int(part_tokens)), "vt_attn_set_tuning")


def workspace_status(workspace):
    """VT_OK (0) unless an attention kernel using this scratch buffer gave up on a
    bounded wait.  Synchronises the current stream."""
    code = ctypes.c_int()
    with _on(workspace.device):
        check(lib.vt_decode_attn_status(_ptr(workspace), _stream(), byref(code)), "vt_decode_attn_status")
    return code.value


def attn_status(device=None):
    """VT_OK (0) unless an attention kernel's bounded wait ran out since the
    workspace was created.  Synchronises the current stream."""
    dev = torch.cuda.current_device() if device is None else _device_index(device)
    return max((workspace_status(ws) for (index, _), ws in list(_workspaces.items()) if index == dev), default=0)
