"""``tri_tier._C`` drop-in: the reference extension's Python surface over the gfx950 C ABI.

Same names, argument names, defaults and exception classes as the reference
module (csrc/bindings.cpp:317-626). The compute runs in
``libtritiercache_amd.so`` on the current HIP device, on torch's current stream.

Argument conventions follow the reference's ``get_contiguous_ptr``
(bindings.cpp:25-97): every tensor argument may be a raw integer address, a
torch tensor (must be contiguous) or a C-contiguous buffer-protocol object
(numpy array, memoryview). Device memory (ROCm tensors, device addresses) is
used in place. Host memory (CPU tensors, numpy arrays, host addresses) is
staged through device memory and, for output arguments, copied back before the
call returns, so the reference's host-side callers and tests keep working.

Differences from the reference, all documented in the C header:
  * the zero-copy getters return ROCm tensors viewing device memory (the
    reference returns numpy arrays viewing host memory);
  * num_q_heads must be a multiple of num_kv_heads and head_dim a multiple of
    16 of at most 256 (ValueError otherwise).
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import torch

from . import _lib

_L = _lib.load()

__all__ = [
    "TriTierCacheEngine",
    "fused_attention_decode",
    "fused_attention_decode_shared",
    "quantize_k_block",
    "quantize_v_block",
    "dequantize_k",
    "dequantize_v",
    "qk_norm_rope",
    "device_count",
    "version",
]


def device_count() -> int:
    return int(_L.tt_device_count())


def version() -> str:
    return _L.tt_version().decode()


def _require_gpu() -> None:
    if device_count() == 0 or not torch.cuda.is_available():
        raise RuntimeError("tritiercache_amd: no HIP device is visible; the gfx950 kernels need an MI355X GPU.")


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _is_fp16(dtype_str: str, scale_obj) -> bool:
    """bindings.cpp:130-136: "fp16" selects half metadata, as does a scale
    object whose dtype string names float16/half."""
    fp16 = dtype_str == "fp16"
    dt = getattr(scale_obj, "dtype", None)
    if dt is not None:
        s = str(dt)
        if "float16" in s or "half" in s:
            fp16 = True
    return fp16


class _Staging:
    """Resolves arguments to device addresses, staging host memory."""

    def __init__(self, sized=False):
        self._writeback = []
        self._keep = []
        self._sized = sized  # tensors must hold the bytes that the call reads or writes

    def ptr(self, obj, name: str, nbytes: int, writable: bool = False, nullable: bool = False) -> int:
        if obj is None:
            if nullable:
                return 0
            raise ValueError(f"Argument '{name}' cannot be None.")
        if isinstance(obj, int) and not isinstance(obj, bool):
            if obj == 0:
                if nullable:
                    return 0
                raise ValueError(f"Argument '{name}' pointer address is NULL.")
            if int(_L.tt_pointer_kind(C.c_void_p(obj))) == 1:
                return obj
            return self._stage_raw(obj, nbytes, writable)
        if isinstance(obj, torch.Tensor):
            if not obj.is_contiguous():
                raise ValueError(
                    f"Argument '{name}' PyTorch tensor is not contiguous in memory. Call .contiguous() before passing.")
            if self._sized and obj.numel() * obj.element_size() < nbytes:
                raise ValueError(f"Argument '{name}' tensor holds {obj.numel() * obj.element_size()} bytes, the call "
                                 f"needs {nbytes}.")
            if obj.is_cuda:
                p = obj.data_ptr()
                if p == 0 and not nullable:
                    raise ValueError(f"Argument '{name}' tensor data pointer is NULL.")
                return p
            return self._stage_tensor(obj, writable)
        if hasattr(obj, "data_ptr") and hasattr(obj, "is_contiguous"):
            if not obj.is_contiguous():
                raise ValueError(
                    f"Argument '{name}' PyTorch tensor is not contiguous in memory. Call .contiguous() before passing.")
            return int(obj.data_ptr())
        try:
            arr = np.asarray(memoryview(obj))
        except TypeError:
            raise ValueError(
                f"Argument '{name}' has unsupported type '{type(obj)}'. Expected PyTorch tensor, NumPy array, buffer "
                "object, or integer memory address.") from None
        if not arr.flags["C_CONTIGUOUS"]:
            raise ValueError(f"Argument '{name}' buffer is not C-contiguous in memory.")
        if writable and not arr.flags["WRITEABLE"]:
            raise ValueError(f"Argument '{name}' buffer is read-only.")
        return self._stage_numpy(arr, writable)

    def _device_copy(self, host_u8: torch.Tensor) -> torch.Tensor:
        dev = torch.empty(max(host_u8.numel(), 1), dtype=torch.uint8, device="cuda")
        if host_u8.numel():
            dev[: host_u8.numel()].copy_(host_u8)
        self._keep.append(dev)
        return dev

    def _stage_numpy(self, arr: np.ndarray, writable: bool) -> int:
        u8 = torch.from_numpy(arr.reshape(-1).view(np.uint8))
        dev = self._device_copy(u8)
        if writable:
            self._writeback.append(("numpy", arr, dev))
        return dev.data_ptr()

    def _stage_tensor(self, t: torch.Tensor, writable: bool) -> int:
        u8 = t.reshape(-1).view(torch.uint8)
        dev = self._device_copy(u8)
        if writable:
            self._writeback.append(("tensor", t, dev))
        return dev.data_ptr()

    def _stage_raw(self, addr: int, nbytes: int, writable: bool) -> int:
        buf = (C.c_uint8 * max(nbytes, 1)).from_address(addr)
        u8 = torch.from_numpy(np.frombuffer(buf, dtype=np.uint8, count=nbytes))
        dev = self._device_copy(u8)
        if writable:
            self._writeback.append(("raw", addr, dev, nbytes))
        return dev.data_ptr()

    def finish(self) -> None:
        if not self._writeback:
            return
        torch.cuda.current_stream().synchronize()
        for item in self._writeback:
            kind = item[0]
            if kind == "numpy":
                _, arr, dev = item
                n = arr.nbytes
                flat = arr.reshape(-1).view(np.uint8)
                flat[:] = dev[:n].cpu().numpy()
            elif kind == "tensor":
                _, t, dev = item
                n = t.numel() * t.element_size()
                t.reshape(-1).view(torch.uint8).copy_(dev[:n].cpu())
            else:
                _, addr, dev, n = item
                host = dev[:n].cpu().numpy()
                C.memmove(addr, host.ctypes.data, n)
        self._writeback.clear()
        self._keep.clear()


def fused_attention_decode(Q_ptr, dense_K_ptr, dense_V_ptr, dense_count, PBS_K_Packed_ptr, PBS_K_Scales_ptr,
                           PBS_K_Zeroes_ptr, PBS_V_Packed_ptr, PBS_V_Scales_ptr, PBS_V_Zeroes_ptr, PBS_token_ids_ptr,
                           num_blocks, num_q_heads, num_kv_heads, head_dim, attn_output_ptr,
                           mean_attn_weights_ptr=None, k_group_size=16, pbs_metadata_dtype="fp32"):
    """Fused decode attention over dense KV and 2-bit packed KV (bindings.cpp:99-178)."""
    dense_count, num_blocks = int(dense_count), int(num_blocks)
    Hq, Hkv, D, kgs = int(num_q_heads), int(num_kv_heads), int(head_dim), int(k_group_size)
    if dense_count < 0:
        raise ValueError("dense_count must be non-negative.")
    if num_blocks < 0:
        raise ValueError("num_blocks must be non-negative.")
    if Hq <= 0 or Hkv <= 0 or D <= 0:
        raise ValueError("num_q_heads, num_kv_heads, and head_dim must be positive integers.")
    _require_gpu()
    fp16 = _is_fp16(pbs_metadata_dtype, PBS_K_Scales_ptr)
    msz = 2 if fp16 else 4
    kvs = Hkv * D
    W = max(kgs // 16, 1)
    st = _Staging()
    nd0, nb0 = dense_count == 0, num_blocks == 0
    q = st.ptr(Q_ptr, "Q", Hq * D * 4)
    dk = st.ptr(dense_K_ptr, "dense_K", dense_count * kvs * 4, nullable=nd0)
    dv = st.ptr(dense_V_ptr, "dense_V", dense_count * kvs * 4, nullable=nd0)
    kp = st.ptr(PBS_K_Packed_ptr, "PBS_K_Packed", num_blocks * W * kvs * 4, nullable=nb0)
    vp = st.ptr(PBS_V_Packed_ptr, "PBS_V_Packed", num_blocks * kgs * Hkv * (D // 16) * 4, nullable=nb0)
    ids = st.ptr(PBS_token_ids_ptr, "PBS_token_ids", num_blocks * kgs * 8, nullable=nb0)
    out = st.ptr(attn_output_ptr, "attn_output", Hq * D * 4, writable=True)
    total = dense_count + num_blocks * kgs
    mw = st.ptr(mean_attn_weights_ptr, "mean_attn_weights", total * 4, writable=True, nullable=True)
    ks = st.ptr(PBS_K_Scales_ptr, "PBS_K_Scales", num_blocks * kvs * msz, nullable=nb0)
    kz = st.ptr(PBS_K_Zeroes_ptr, "PBS_K_Zeroes", num_blocks * kvs * msz, nullable=nb0)
    vs = st.ptr(PBS_V_Scales_ptr, "PBS_V_Scales", num_blocks * kgs * Hkv * msz, nullable=nb0)
    vz = st.ptr(PBS_V_Zeroes_ptr, "PBS_V_Zeroes", num_blocks * kgs * Hkv * msz, nullable=nb0)
    rc = _L.tt_fused_attention_decode(q, dk, dv, dense_count, kp, ks, kz, vp, vs, vz, ids, num_blocks, Hq, Hkv, D,
                                      out, mw or None, kgs, int(fp16), _stream())
    _lib.check(rc, "fused_attention_decode")
    st.finish()


_BATCH_FIELDS = ("Q", "dense_K", "dense_V", "dense_count", "PBS_K_Packed", "PBS_K_Scales", "PBS_K_Zeroes",
                 "PBS_V_Packed", "PBS_V_Scales", "PBS_V_Zeroes", "PBS_token_ids", "num_blocks", "attn_output",
                 "mean_attn_weights")


def _fill_tiers(st, s, e, Hkv, D, kgs, msz):
    """The tiers and counts of `e` (a dict with the keys of _BATCH_FIELDS) into the tt_decode_seq `s`."""
    kvs = Hkv * D
    W = max(kgs // 16, 1)
    nd, nb = int(e.get("dense_count", 0)), int(e.get("num_blocks", 0))
    if nd < 0:
        raise ValueError("dense_count must be non-negative.")
    if nb < 0:
        raise ValueError("num_blocks must be non-negative.")
    nd0, nb0 = nd == 0, nb == 0
    s.dense_K = st.ptr(e.get("dense_K"), "dense_K", nd * kvs * 4, nullable=nd0) or None
    s.dense_V = st.ptr(e.get("dense_V"), "dense_V", nd * kvs * 4, nullable=nd0) or None
    s.PBS_K_Packed = st.ptr(e.get("PBS_K_Packed"), "PBS_K_Packed", nb * W * kvs * 4, nullable=nb0) or None
    s.PBS_K_Scales = st.ptr(e.get("PBS_K_Scales"), "PBS_K_Scales", nb * kvs * msz, nullable=nb0) or None
    s.PBS_K_Zeroes = st.ptr(e.get("PBS_K_Zeroes"), "PBS_K_Zeroes", nb * kvs * msz, nullable=nb0) or None
    s.PBS_V_Packed = st.ptr(e.get("PBS_V_Packed"), "PBS_V_Packed", nb * kgs * Hkv * (D // 16) * 4,
                            nullable=nb0) or None
    s.PBS_V_Scales = st.ptr(e.get("PBS_V_Scales"), "PBS_V_Scales", nb * kgs * Hkv * msz, nullable=nb0) or None
    s.PBS_V_Zeroes = st.ptr(e.get("PBS_V_Zeroes"), "PBS_V_Zeroes", nb * kgs * Hkv * msz, nullable=nb0) or None
    s.PBS_token_ids = st.ptr(e.get("PBS_token_ids"), "PBS_token_ids", nb * kgs * 8, nullable=nb0) or None
    s.dense_count, s.num_blocks = nd, nb


def _fill_seq(st, s, e, Hq, Hkv, D, kgs, msz):
    """One sequence of a batch: its query, tiers and outputs."""
    s.Q = st.ptr(e.get("Q"), "Q", Hq * D * 4)
    _fill_tiers(st, s, e, Hkv, D, kgs, msz)
    s.attn_output = st.ptr(e.get("attn_output"), "attn_output", Hq * D * 4, writable=True)
    s.mean_attn_weights = st.ptr(e.get("mean_attn_weights"), "mean_attn_weights",
                                 (s.dense_count + s.num_blocks * kgs) * 4, writable=True, nullable=True) or None


def fused_attention_decode_batched(batch, num_q_heads, num_kv_heads, head_dim, k_group_size=16,
                                   pbs_metadata_dtype="fp32"):
    """One decode step of many sequences in one split-K launch (plus one merge launch).

    `batch` holds one entry per sequence: a dict with the keys of
    ``_BATCH_FIELDS`` or a tuple in that order, i.e. the per-sequence
    arguments of fused_attention_decode (bindings.cpp:99-178); each
    sequence's outputs equal that call's. The sequences share the head
    counts, head_dim, k_group_size and metadata dtype. No counterpart in the
    reference, whose callers loop over sequences."""
    Hq, Hkv, D, kgs = int(num_q_heads), int(num_kv_heads), int(head_dim), int(k_group_size)
    if Hq <= 0 or Hkv <= 0 or D <= 0:
        raise ValueError("num_q_heads, num_kv_heads, and head_dim must be positive integers.")
    _require_gpu()
    entries = [dict(e) if isinstance(e, dict) else dict(zip(_BATCH_FIELDS, e)) for e in batch]
    if not entries:
        return
    fp16 = _is_fp16(pbs_metadata_dtype, entries[0].get("PBS_K_Scales"))
    msz = 2 if fp16 else 4
    st = _Staging()
    seqs = (_lib.DecodeSeq * len(entries))()
    for s, e in zip(seqs, entries):
        _fill_seq(st, s, e, Hq, Hkv, D, kgs, msz)
    n = len(entries)
    ws_bytes = int(_L.tt_batched_decode_workspace_bytes(seqs, n, Hq, Hkv, D, kgs))
    if ws_bytes == 0:
        _lib.check(_lib.TT_ERR_INVALID_ARGUMENT, "fused_attention_decode_batched")
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device="cuda")
    raw = np.frombuffer(bytes(seqs), dtype=np.uint8)
    seqs_dev = torch.from_numpy(raw.copy()).cuda()
    rc = _L.tt_fused_attention_decode_batched(seqs, seqs_dev.data_ptr(), n, Hq, Hkv, D, kgs, int(fp16), ws.data_ptr(),
                                              ws_bytes, _stream())
    _lib.check(rc, "fused_attention_decode_batched")
    st.finish()


def fused_attention_decode_shared(prefix, batch, num_q_heads, num_kv_heads, head_dim, k_group_size=16,
                                  pbs_metadata_dtype="fp32"):
    """One decode step of sequences that share a prefix (a common system prompt or document): every sequence attends
    to the prefix's tokens and its own in one softmax, and the prefix is unpacked and multiplied once for all of them
    (a short one, or that of few sequences, once for each). No counterpart in the reference.

    `prefix`: a dict with the tier keys of ``_BATCH_FIELDS`` (dense_K .. num_blocks without Q and the outputs), e.g.
    ``TriTierCache.as_prefix()``. `batch`: the sequences as in fused_attention_decode_batched, each with its own
    tiers behind the prefix (counts of 0 where it has none); mean_attn_weights receives the weights of its own tokens.
    Attended keys and values and the queries must be finite. Runs on the device of the queries."""
    Hq, Hkv, D, kgs = int(num_q_heads), int(num_kv_heads), int(head_dim), int(k_group_size)
    if Hq <= 0 or Hkv <= 0 or D <= 0:
        raise ValueError("num_q_heads, num_kv_heads, and head_dim must be positive integers.")
    pre = dict(prefix)
    if pre.get("mean_attn_weights") is not None:
        raise ValueError("the prefix has no mean attention weights.")
    _require_gpu()
    entries = [dict(e) if isinstance(e, dict) else dict(zip(_BATCH_FIELDS, e)) for e in batch]
    if not entries:
        return
    q = entries[0].get("Q")
    with torch.cuda.device(q.device if isinstance(q, torch.Tensor) and q.is_cuda else torch.cuda.current_device()):
        _decode_shared(pre, entries, Hq, Hkv, D, kgs, pbs_metadata_dtype)


def _decode_shared(pre, entries, Hq, Hkv, D, kgs, pbs_metadata_dtype):
    scales = pre.get("PBS_K_Scales")
    fp16 = _is_fp16(pbs_metadata_dtype, scales if scales is not None else entries[0].get("PBS_K_Scales"))
    msz = 2 if fp16 else 4
    st = _Staging(sized=True)
    p = _lib.DecodeSeq()
    _fill_tiers(st, p, pre, Hkv, D, kgs, msz)
    seqs = (_lib.DecodeSeq * len(entries))()
    for s, e in zip(seqs, entries):
        _fill_seq(st, s, e, Hq, Hkv, D, kgs, msz)
    n = len(entries)
    ws_bytes = int(_L.tt_shared_decode_workspace_bytes(C.byref(p), seqs, n, Hq, Hkv, D, kgs))
    if ws_bytes == 0:
        _lib.check(_lib.TT_ERR_INVALID_ARGUMENT, "fused_attention_decode_shared")
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device="cuda")
    seqs_dev = torch.from_numpy(np.frombuffer(bytes(seqs), dtype=np.uint8).copy()).cuda()
    rc = _L.tt_fused_attention_decode_shared(C.byref(p), seqs, seqs_dev.data_ptr(), n, Hq, Hkv, D, kgs, int(fp16),
                                             ws.data_ptr(), ws_bytes, _stream())
    _lib.check(rc, "fused_attention_decode_shared")
    st.finish()


def quantize_k_block(K, packed, scale, zero, num_heads, head_dim, k_group_size=16, pbs_metadata_dtype="fp32"):
    """2-bit per-channel quantisation of one K block (bindings.cpp:180-212)."""
    H, D, kgs = int(num_heads), int(head_dim), int(k_group_size)
    _require_gpu()
    fp16 = _is_fp16(pbs_metadata_dtype, scale)
    msz = 2 if fp16 else 4
    st = _Staging()
    k = st.ptr(K, "K", kgs * H * D * 4)
    p = st.ptr(packed, "packed", (kgs // 16) * H * D * 4, writable=True)
    s = st.ptr(scale, "scale", H * D * msz, writable=True)
    z = st.ptr(zero, "zero", H * D * msz, writable=True)
    _lib.check(_L.tt_quantize_k_block(k, p, s, z, 1, H, D, kgs, int(fp16), _stream()), "quantize_k_block")
    st.finish()


def quantize_k_blocks(K, packed, scale, zero, num_blocks, num_heads, head_dim, k_group_size=16,
                      pbs_metadata_dtype="fp32"):
    """Batched quantize_k_block over `num_blocks` consecutive blocks (one launch)."""
    nb, H, D, kgs = int(num_blocks), int(num_heads), int(head_dim), int(k_group_size)
    _require_gpu()
    fp16 = _is_fp16(pbs_metadata_dtype, scale)
    msz = 2 if fp16 else 4
    st = _Staging()
    k = st.ptr(K, "K", nb * kgs * H * D * 4)
    p = st.ptr(packed, "packed", nb * (kgs // 16) * H * D * 4, writable=True)
    s = st.ptr(scale, "scale", nb * H * D * msz, writable=True)
    z = st.ptr(zero, "zero", nb * H * D * msz, writable=True)
    _lib.check(_L.tt_quantize_k_block(k, p, s, z, nb, H, D, kgs, int(fp16), _stream()), "quantize_k_blocks")
    st.finish()


def quantize_v_block(V, packed, scale, zero, num_heads, head_dim, chunk_size=16, pbs_metadata_dtype="fp32"):
    """2-bit per-token quantisation of one V block (bindings.cpp:214-246)."""
    H, D, ch = int(num_heads), int(head_dim), int(chunk_size)
    _require_gpu()
    fp16 = _is_fp16(pbs_metadata_dtype, scale)
    msz = 2 if fp16 else 4
    st = _Staging()
    v = st.ptr(V, "V", ch * H * D * 4)
    p = st.ptr(packed, "packed", ch * H * ((D + 15) // 16) * 4, writable=True)
    s = st.ptr(scale, "scale", ch * H * msz, writable=True)
    z = st.ptr(zero, "zero", ch * H * msz, writable=True)
    _lib.check(_L.tt_quantize_v_block(v, p, s, z, ch, H, D, int(fp16), _stream()), "quantize_v_block")
    st.finish()


def dequantize_k(packed, scale, zero, out, num_blocks, num_heads, head_dim, k_group_size=16,
                 pbs_metadata_dtype="fp32"):
    """Dequantise K blocks: x = fmaf(q, scale, zero) (bindings.cpp:248-281)."""
    nb, H, D, kgs = int(num_blocks), int(num_heads), int(head_dim), int(k_group_size)
    _require_gpu()
    fp16 = _is_fp16(pbs_metadata_dtype, scale)
    msz = 2 if fp16 else 4
    st = _Staging()
    p = st.ptr(packed, "packed", nb * (kgs // 16) * H * D * 4)
    s = st.ptr(scale, "scale", nb * H * D * msz)
    z = st.ptr(zero, "zero", nb * H * D * msz)
    o = st.ptr(out, "out", nb * kgs * H * D * 4, writable=True)
    _lib.check(_L.tt_dequantize_k(p, s, z, o, nb, H, D, kgs, int(fp16), _stream()), "dequantize_k")
    st.finish()


def dequantize_v(packed, scale, zero, out, total_tokens, num_heads, head_dim, pbs_metadata_dtype="fp32"):
    """Dequantise V tokens (bindings.cpp:283-315)."""
    n, H, D = int(total_tokens), int(num_heads), int(head_dim)
    _require_gpu()
    fp16 = _is_fp16(pbs_metadata_dtype, scale)
    msz = 2 if fp16 else 4
    st = _Staging()
    p = st.ptr(packed, "packed", n * H * ((D + 15) // 16) * 4)
    s = st.ptr(scale, "scale", n * H * msz)
    z = st.ptr(zero, "zero", n * H * msz)
    o = st.ptr(out, "out", n * H * D * 4, writable=True)
    _lib.check(_L.tt_dequantize_v(p, s, z, o, n, H, D, int(fp16), _stream()), "dequantize_v")
    st.finish()


_DTYPES = {torch.float32: _lib.TT_DTYPE_F32, torch.float16: _lib.TT_DTYPE_F16, torch.bfloat16: _lib.TT_DTYPE_BF16}


def _rows(t, name: str, heads=None, like=None) -> torch.Tensor:
    """A ROCm tensor [tokens, heads, head_dim] whose channels are adjacent (other strides are free)."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"Argument '{name}' must be a tensor [tokens, heads, head_dim].")
    if t.dtype not in _DTYPES:
        raise ValueError(f"Argument '{name}' must be float32, float16 or bfloat16, got {t.dtype}.")
    if t.shape[2] > 1 and t.numel() and t.stride(2) != 1:
        raise ValueError(f"Argument '{name}' must have adjacent channels (stride 1 in its last dimension).")
    if like is not None and (t.dtype != like.dtype or t.shape[2] != like.shape[2]):
        raise ValueError(f"Argument '{name}' must have the type and head_dim of its kind: {like.dtype}, {like.shape[2]}.")
    if heads is not None and t.shape[1] != heads:
        raise ValueError(f"Argument '{name}' must have {heads} heads, got {t.shape[1]}.")
    return t


def qk_norm_rope(q, k, v=None, cos=None, sin=None, positions=None, q_weight=None, k_weight=None, eps=1e-6,
                 out_dtype=None, rows=None, q_out=None, k_out=None, v_out=None):
    """The norm of each query and key head, the position rotation and the cast, in one launch; no
    counterpart in the reference (its patch runs the model file's modules, patch_model.py:98-116).

    q [tokens, num_q_heads, head_dim], k and v [tokens, num_kv_heads, head_dim] (v may be None): ROCm tensors of one
    type, any strides with adjacent channels (views of a joint projection, transposed ones). cos, sin [table rows,
    rotary_dim]: a multiple of 16 channels is rotated, the first half of them against the second (rotate-half),
    the rest passes; None: no rotation. positions [tokens] int64: each token's row of the tables (None: row t; a position outside them makes
    the token's queries and keys NaN). q_weight, k_weight [head_dim]: weights of the RMS norms, None for no norm.
    rows [tokens] int64: the row of k_out and v_out that takes the token's keys and values (None: row t; -1 or any
    row that is not there: not stored). Outputs that are not given are allocated in out_dtype (q's type where that is None); with
    rows, k_out and v_out are the caller's. No backward pass: inputs that record gradients are refused. Returns (q_out, k_out,
    v_out or None)."""
    q = _rows(q, "q")
    tokens, hq, d = q.shape
    if tokens >= 2 ** 31:
        raise ValueError(f"Argument 'q' must have fewer than 2^31 tokens, got {tokens}.")
    k = _rows(k, "k", like=q)
    hkv = k.shape[1]
    ins = {"q": q, "k": k}
    if v is not None:
        ins["v"] = _rows(v, "v", hkv, q)
    for name, x in ins.items():
        if x.shape[0] != tokens:
            raise ValueError(f"Argument '{name}' must have {tokens} tokens, got {x.shape[0]}.")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin must both be given or both be None.")
    if v is None and v_out is not None:
        raise ValueError("v_out without v.")
    small = {"cos": cos, "sin": sin, "positions": positions, "rows": rows, "q_weight": q_weight, "k_weight": k_weight}
    for name, x in small.items():
        if x is not None and not isinstance(x, torch.Tensor):
            raise ValueError(f"Argument '{name}' must be a tensor.")
    rot = 0
    if cos is not None:
        if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != sin.dtype or cos.dtype not in _DTYPES:
            raise ValueError("cos and sin must be [table rows, rotary_dim] of one type: float32, float16 or bfloat16.")
        rot = cos.shape[1]
        if cos.stride() != sin.stride() or (rot > 1 and cos.stride(1) != 1):
            raise ValueError("cos and sin must have the same strides and adjacent channels.")
    for name in ("positions", "rows"):
        x = small[name]
        if x is not None and (x.dtype != torch.int64 or x.shape != (tokens,) or not x.is_contiguous()):
            raise ValueError(f"Argument '{name}' must be a contiguous int64 tensor [{tokens}].")
    wdt = {x.dtype for x in (q_weight, k_weight) if x is not None}
    for name in ("q_weight", "k_weight"):
        x = small[name]
        if x is not None and (x.dtype not in _DTYPES or x.shape != (d,) or not x.is_contiguous() or len(wdt) > 1):
            raise ValueError("q_weight and k_weight must be contiguous [head_dim] tensors of one type.")
    if rows is not None and (k_out is None or (v is not None and v_out is None)):
        raise ValueError("with rows, k_out and v_out are the caller's tensors.")
    if torch.is_grad_enabled() and any(isinstance(x, torch.Tensor) and x.requires_grad
                                       for x in (q, k, v, cos, sin, q_weight, k_weight, q_out, k_out, v_out)):
        raise ValueError("qk_norm_rope has no backward pass: call it under torch.no_grad() or on detached tensors.")
    _require_gpu()
    odt = out_dtype
    if odt is None:
        given = [x for x in (q_out, k_out, v_out) if x is not None]
        odt = given[0].dtype if given else q.dtype
    if odt not in _DTYPES:
        raise ValueError(f"out_dtype must be float32, float16 or bfloat16, got {odt}.")
    outs = {}
    for name, x, h in (("q_out", q_out, hq), ("k_out", k_out, hkv), ("v_out", v_out, hkv)):
        if name == "v_out" and v is None:
            continue
        if x is None:
            x = torch.empty((tokens, h, d), dtype=odt, device=q.device)
        x = _rows(x, name, h)
        if x.dtype != odt or x.shape[2] != d:
            raise ValueError(f"Argument '{name}' must be {odt} with head_dim {d}.")
        if (name == "q_out" or rows is None) and x.shape[0] < tokens:
            raise ValueError(f"Argument '{name}' must have a row for each of the {tokens} tokens.")
        outs[name] = x
    if v is not None and outs["v_out"].shape[0] != outs["k_out"].shape[0]:
        raise ValueError("k_out and v_out must have the same number of rows.")
    tensors = {**ins, **outs, **{n: x for n, x in small.items() if x is not None}}
    for name, x in tensors.items():
        if not x.is_cuda or x.device != q.device:
            raise ValueError(f"Argument '{name}' must be a ROCm tensor on the device of q.")
    a = _lib.QkRope()
    for name, x in tensors.items():
        setattr(a, name, x.data_ptr() or None)
    for name, x in {**ins, **outs}.items():
        setattr(a, name + "_token_stride", x.stride(0))
        setattr(a, name + "_head_stride", x.stride(1))
    a.tokens, a.num_q_heads, a.num_kv_heads, a.head_dim, a.rotary_dim, a.eps = tokens, hq, hkv, d, rot, float(eps)
    a.out_rows = outs["k_out"].shape[0]
    if cos is not None:
        a.table_rows, a.table_stride, a.table_dtype = cos.shape[0], cos.stride(0), _DTYPES[cos.dtype]
        if cos.shape[0] == 1:
            a.table_stride = rot
    a.in_dtype, a.out_dtype = _DTYPES[q.dtype], _DTYPES[odt]
    a.weight_dtype = _DTYPES[wdt.pop()] if wdt else _lib.TT_DTYPE_F32
    with torch.cuda.device(q.device):
        _lib.check(_L.tt_qk_norm_rope(C.byref(a), _stream()), "qk_norm_rope")
    return outs["q_out"], outs["k_out"], outs.get("v_out")


class _DeviceView:
    """__cuda_array_interface__ holder: torch.as_tensor keeps it (and through
    it the engine) alive for as long as the tensor lives."""

    def __init__(self, ptr: int, shape, typestr: str, owner):
        self._owner = owner
        self.__cuda_array_interface__ = {
            "shape": tuple(int(s) for s in shape),
            "typestr": typestr,
            "data": (int(ptr), False),
            "version": 3,
            "strides": None,
        }


_BUFFERS = {
    "S_K": 0, "S_V": 1, "RW_K": 2, "RW_V": 3, "HH_K": 4, "HH_V": 5, "HH_token_ids": 6, "HH_scores": 7, "WR_K": 8,
    "WR_V": 9, "WR_token_ids": 10, "PBS_K_Packed": 11, "PBS_K_Scales": 12, "PBS_K_Zeroes": 13, "PBS_V_Packed": 14,
    "PBS_V_Scales": 15, "PBS_V_Zeroes": 16, "PBS_token_ids": 17, "global_attn_scores": 18,
    "mean_attn_weights": 19,
}


class TriTierCacheEngine:
    """Device-resident tier engine (bindings.cpp:384-626, cache_engine.cpp)."""

    _COUNTER_NAMES = None

    def __init__(self, num_q_heads, num_kv_heads, head_dim, max_seq_len, sink_size=4, rw_size=64, h_ratio=0.1,
                 score_decay=0.999, update_interval=16, k_group_size=16, pbs_metadata_dtype="fp16"):
        _require_gpu()
        self._h = None
        h = C.c_void_p()
        self._pbs_metadata_dtype = str(pbs_metadata_dtype)
        rc = _L.tt_engine_create(C.byref(h), int(num_q_heads), int(num_kv_heads), int(head_dim), int(max_seq_len),
                                 int(sink_size), int(rw_size), float(h_ratio), float(score_decay),
                                 int(update_interval), int(k_group_size), self._pbs_metadata_dtype.encode(),
                                 _stream())
        _lib.check(rc, "TriTierCacheEngine")
        self._h = h
        self.h_ratio = float(np.float32(h_ratio))
        self.score_decay = float(np.float32(score_decay))
        c = self.counters()
        for k in ("num_q_heads", "num_kv_heads", "head_dim", "max_seq_len", "sink_size", "rw_size",
                  "update_interval", "k_group_size", "chunk_size", "quant_head_dim", "max_hh"):
            setattr(self, "_" + k, c[k])

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            _L.tt_engine_destroy(h)
            self._h = None

    # ---- configuration (read-only) ----
    num_q_heads = property(lambda self: self._num_q_heads)
    num_kv_heads = property(lambda self: self._num_kv_heads)
    head_dim = property(lambda self: self._head_dim)
    max_seq_len = property(lambda self: self._max_seq_len)
    sink_size = property(lambda self: self._sink_size)
    rw_size = property(lambda self: self._rw_size)
    update_interval = property(lambda self: self._update_interval)
    k_group_size = property(lambda self: self._k_group_size)
    chunk_size = property(lambda self: self._chunk_size)
    quant_head_dim = property(lambda self: self._quant_head_dim)
    max_hh = property(lambda self: self._max_hh)
    pbs_metadata_dtype = property(lambda self: self._pbs_metadata_dtype)
    use_fp16_meta = property(lambda self: self._pbs_metadata_dtype == "fp16")

    # ---- counters (read from the device; synchronises the current stream) ----
    def counters(self) -> dict:
        if TriTierCacheEngine._COUNTER_NAMES is None:
            TriTierCacheEngine._COUNTER_NAMES = _L.tt_engine_counter_names().decode().split()
        out = np.zeros(23, np.int64)
        _lib.check(_L.tt_engine_counters(self._h, out.ctypes.data, _stream()), "counters")
        return dict(zip(TriTierCacheEngine._COUNTER_NAMES, (int(x) for x in out)))

    pbs_allocated_blocks = property(lambda self: self.counters()["pbs_allocated_blocks"])
    s_count = property(lambda self: self.counters()["s_count"])
    rw_count = property(lambda self: self.counters()["rw_count"])
    rw_head_index = property(lambda self: self.counters()["rw_head_index"])
    hh_count = property(lambda self: self.counters()["hh_count"])
    wr_count = property(lambda self: self.counters()["wr_count"])
    pbs_count = property(lambda self: self.counters()["pbs_count"])
    pbs_blocks_used = property(lambda self: self.counters()["pbs_blocks_used"])
    total_processed_tokens = property(lambda self: self.counters()["total_processed_tokens"])
    total_evictions = property(lambda self: self.counters()["total_evictions"])
    last_calc_pos = property(lambda self: self.counters()["last_calc_pos"])

    # ---- compute ----
    def step(self, q_ptr, k_ptr, v_ptr, out_ptr):
        """Ingest one token, attend, feed back scores (cache_engine.cpp:397-541)."""
        st = _Staging()
        Hq, Hkv, D = self._num_q_heads, self._num_kv_heads, self._head_dim
        q = st.ptr(q_ptr, "Q", Hq * D * 4)
        k = st.ptr(k_ptr, "K_new", Hkv * D * 4)
        v = st.ptr(v_ptr, "V_new", Hkv * D * 4)
        o = st.ptr(out_ptr, "attn_output", Hq * D * 4, writable=True)
        _lib.check(_L.tt_engine_step(self._h, q, k, v, o, _stream()), "step")
        st.finish()

    def step_deferred(self, q_ptr, k_ptr, v_ptr, out_ptr, prev=None):
        """step() for engines stepped one after another (a model's layers): this
        step runs up to its merged attention output and leaves its mean attention
        weights and score feedback pending; the pending feedback of `prev`
        (another TriTierCacheEngine on the same device, or None) runs in this
        step's finalize launch. A pending feedback also runs at the start of any
        later call on its engine, or in flush_feedback()."""
        if prev is self:
            raise ValueError("prev must be another engine.")
        st = _Staging()
        Hq, Hkv, D = self._num_q_heads, self._num_kv_heads, self._head_dim
        q = st.ptr(q_ptr, "Q", Hq * D * 4)
        k = st.ptr(k_ptr, "K_new", Hkv * D * 4)
        v = st.ptr(v_ptr, "V_new", Hkv * D * 4)
        o = st.ptr(out_ptr, "attn_output", Hq * D * 4, writable=True)
        ph = prev._h if prev is not None else None
        _lib.check(_L.tt_engine_step_deferred(self._h, q, k, v, o, ph, _stream()), "step_deferred")
        st.finish()

    def flush_feedback(self):
        """Runs this engine's pending mean weights and score feedback, if any."""
        _lib.check(_L.tt_engine_flush_feedback(self._h, _stream()), "flush_feedback")

    def step_with_weights(self, q_ptr, k_ptr, v_ptr, out_ptr) -> torch.Tensor:
        """step() that also returns this step's per-head softmax weights
        [num_q_heads, visible] in the engine's visible order."""
        st = _Staging()
        Hq, Hkv, D = self._num_q_heads, self._num_kv_heads, self._head_dim
        q = st.ptr(q_ptr, "Q", Hq * D * 4)
        k = st.ptr(k_ptr, "K_new", Hkv * D * 4)
        v = st.ptr(v_ptr, "V_new", Hkv * D * 4)
        o = st.ptr(out_ptr, "attn_output", Hq * D * 4, writable=True)
        # the step adds the new token, and a waiting-room flush makes up to
        # one more chunk of tokens visible
        cap = self.visible() + 1 + self._chunk_size
        w = torch.empty((Hq, cap), dtype=torch.float32, device="cuda")
        vis = C.c_int(0)
        _lib.check(_L.tt_engine_step_weights(self._h, q, k, v, o, w.data_ptr(), cap, C.byref(vis), _stream()),
                   "step_with_weights")
        st.finish()
        return w[:, : vis.value]

    def prefill(self, k_ptr, v_ptr, q_len):
        """Bulk prompt ingest (cache_engine.cpp:271-395)."""
        q_len = int(q_len)
        if q_len < 0:
            raise ValueError("q_len must be non-negative.")
        st = _Staging()
        n = q_len * self._num_kv_heads * self._head_dim * 4
        k = st.ptr(k_ptr, "K_all", n, nullable=q_len == 0)
        v = st.ptr(v_ptr, "V_all", n, nullable=q_len == 0)
        _lib.check(_L.tt_engine_prefill(self._h, k, v, q_len, _stream()), "prefill")
        st.finish()

    def ingest(self, k_ptr, v_ptr):
        """Tier maintenance only: ring ingest / eviction / routing / flush."""
        st = _Staging()
        n = self._num_kv_heads * self._head_dim * 4
        k = st.ptr(k_ptr, "K_new", n)
        v = st.ptr(v_ptr, "V_new", n)
        _lib.check(_L.tt_engine_ingest(self._h, k, v, _stream()), "ingest")
        st.finish()

    def feedback(self, mean_attn_weights):
        """Decayed score feedback with caller-supplied mean weights [visible]."""
        n = self.visible()
        size = getattr(mean_attn_weights, "numel", None)
        size = size() if callable(size) else getattr(mean_attn_weights, "size", None)
        if isinstance(size, int) and size < n:
            raise ValueError(f"mean_attn_weights has {size} elements; the engine attends {n} tokens.")
        st = _Staging()
        w = st.ptr(mean_attn_weights, "mean_attn_weights", n * 4)
        _lib.check(_L.tt_engine_feedback(self._h, w, _stream()), "feedback")
        st.finish()

    def visible(self) -> int:
        v = C.c_int(0)
        _lib.check(_L.tt_engine_visible(self._h, C.byref(v), _stream()), "visible")
        return int(v.value)

    def get_buffer_bytes(self) -> int:
        """The reference's tier-byte accounting (cache_engine.cpp:543-568)."""
        v = C.c_size_t(0)
        _lib.check(_L.tt_engine_buffer_bytes(self._h, C.byref(v), _stream()), "get_buffer_bytes")
        return int(v.value)

    # ---- zero-copy device views (bindings.cpp:461-626) ----
    def _view(self, name: str, shape, typestr: str) -> torch.Tensor:
        p = C.c_void_p()
        n = C.c_int64(0)
        es = C.c_int(0)
        _lib.check(_L.tt_engine_buffer(self._h, _BUFFERS[name], C.byref(p), C.byref(n), C.byref(es), _stream()),
                   name)
        assert int(np.prod(shape)) == n.value, (name, shape, n.value)
        if n.value == 0:
            return torch.empty(shape, dtype=torch.uint16 if typestr == "<u2" else {
                "<f4": torch.float32, "<i4": torch.int32, "<i8": torch.int64}[typestr], device="cuda")
        return torch.as_tensor(_DeviceView(p.value, shape, typestr, self), device="cuda")

    def _meta(self):
        return "<u2" if self.use_fp16_meta else "<f4"

    def get_global_attn_scores(self):
        return self._view("global_attn_scores", (self._max_seq_len,), "<f4")

    def get_S_K(self):
        return self._view("S_K", (self._sink_size, self._num_kv_heads, self._head_dim), "<f4")

    def get_S_V(self):
        return self._view("S_V", (self._sink_size, self._num_kv_heads, self._head_dim), "<f4")

    def get_RW_K(self):
        return self._view("RW_K", (self._rw_size, self._num_kv_heads, self._head_dim), "<f4")

    def get_RW_V(self):
        return self._view("RW_V", (self._rw_size, self._num_kv_heads, self._head_dim), "<f4")

    def get_HH_K(self):
        return self._view("HH_K", (self._max_hh, self._num_kv_heads, self._head_dim), "<f4")

    def get_HH_V(self):
        return self._view("HH_V", (self._max_hh, self._num_kv_heads, self._head_dim), "<f4")

    def get_HH_token_ids(self):
        return self._view("HH_token_ids", (self._max_hh,), "<i8")

    def get_HH_scores(self):
        return self._view("HH_scores", (self._max_hh,), "<f4")

    def get_WR_K(self):
        return self._view("WR_K", (self._chunk_size, self._num_kv_heads, self._head_dim), "<f4")

    def get_WR_V(self):
        return self._view("WR_V", (self._chunk_size, self._num_kv_heads, self._head_dim), "<f4")

    def get_WR_token_ids(self):
        return self._view("WR_token_ids", (self._chunk_size,), "<i8")

    def get_PBS_K_Packed(self):
        nb = self.pbs_allocated_blocks
        return self._view("PBS_K_Packed", (nb, self._k_group_size // 16, self._num_kv_heads, self._head_dim), "<i4")

    def get_PBS_K_Scales(self):
        nb = self.pbs_allocated_blocks
        return self._view("PBS_K_Scales", (nb, self._num_kv_heads, self._head_dim), self._meta())

    def get_PBS_K_Zeroes(self):
        nb = self.pbs_allocated_blocks
        return self._view("PBS_K_Zeroes", (nb, self._num_kv_heads, self._head_dim), self._meta())

    def get_PBS_V_Packed(self):
        nb = self.pbs_allocated_blocks
        return self._view("PBS_V_Packed", (nb * self._chunk_size, self._num_kv_heads, self._quant_head_dim), "<i4")

    def get_PBS_V_Scales(self):
        nb = self.pbs_allocated_blocks
        return self._view("PBS_V_Scales", (nb * self._chunk_size, self._num_kv_heads, 1), self._meta())

    def get_PBS_V_Zeroes(self):
        nb = self.pbs_allocated_blocks
        return self._view("PBS_V_Zeroes", (nb * self._chunk_size, self._num_kv_heads, 1), self._meta())

    def get_mean_attn_weights(self):
        """Mean attention weights of the last step, in visible order (engine extra)."""
        return self._view("mean_attn_weights", (self.visible(),), "<f4")

    def get_PBS_token_ids(self):
        nb = self.pbs_allocated_blocks
        return self._view("PBS_token_ids", (nb * self._chunk_size,), "<i8")
