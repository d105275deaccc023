"""Torch-facing wrappers over the C ABI (device pointers, strides, current stream).

These are thin: validate what the reference validates, hand raw pointers to the
library, raise on a non-zero status.  Every op runs its CUDA kernel; tensors on
the CPU are rejected (there is no CPU path in the product).
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import numpy as np
import torch

from ._lib import check, lib

HEAD_DIM = 128
DEFAULT_MROPE_SECTION = (16, 24, 24)  # Qwen2.5-VL rope_scaling.mrope_section


_raw_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    """Handle of the current device's current stream.  Read raw (no torch.cuda.Stream object,
    no device-availability probe): it is on every launch's host path."""
    if _raw_device is not None and _raw_stream is not None:
        return _raw_stream(_raw_device())
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor | None) -> int:
    """Device address of ``t`` (0 for None); every C-ABI argument is declared ``void*``."""
    return 0 if t is None else t.data_ptr()


def _require_cuda(*ts: torch.Tensor) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("vlcache_b200 ops run on CUDA tensors only (no CPU fallback)")


def num_sms() -> int:
    return int(lib().vlc_num_sms())


def device_error(reset: bool = True) -> int:
    """Synchronise and return (and by default clear) the library's device error word."""
    return int(lib().vlc_get_device_error(1 if reset else 0))


# --------------------------------------------------------------------------- scatter
def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slot_mapping: torch.Tensor) -> None:
    """``k_cache.view(-1, D)[slot_mapping[i]] = key[i]`` (and V); slot -1 is skipped.

    Same contract and assertions as nanovllm/layers/attention.py:33-40.
    """
    N, num_heads, head_dim = key.shape
    D = num_heads * head_dim
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert k_cache.stride(1) == D and v_cache.stride(1) == D
    assert slot_mapping.numel() == N
    _require_cuda(key, value, k_cache, v_cache, slot_mapping)
    assert key.dtype == torch.bfloat16 and k_cache.dtype == torch.bfloat16
    assert slot_mapping.dtype == torch.int32
    num_slots = k_cache.numel() // D
    st = lib().vlc_store_kvcache(_ptr(key), key.stride(0), _ptr(value), value.stride(0), _ptr(k_cache),
                                 _ptr(v_cache), _ptr(slot_mapping), N, D, num_slots, _stream())
    check("vlc_store_kvcache", st)


# --------------------------------------------------------------------------- rotary + scatter
def _rope_args(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, cos_sin_cache: torch.Tensor):
    N, H, D = query.shape
    Hk = key.shape[1]
    assert key.shape[0] == N and key.shape[2] == D and positions.numel() == N
    assert query.stride(-1) == 1 and query.stride(1) == D and key.stride(-1) == 1 and key.stride(1) == D
    assert query.dtype == torch.bfloat16 and key.dtype == torch.bfloat16
    assert positions.dtype == torch.int64 and positions.is_contiguous()
    assert cos_sin_cache.dtype == torch.float32 and cos_sin_cache.is_contiguous()
    assert cos_sin_cache.shape[-1] == D and cos_sin_cache.numel() == cos_sin_cache.shape[0] * D
    return N, H, Hk, D, cos_sin_cache.shape[0]


def rotary_embedding(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor,
                     cos_sin_cache: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotate-half RoPE of ``query`` [N, H, D] and ``key`` [N, Hk, D] at ``positions``.

    Semantics of nanovllm/layers/rotary_embedding.py:37-48 (``cos_sin_cache[positions]``
    split into cos | sin, ``apply_rotary_emb`` :6-14 in fp32, result in bf16); returns new
    tensors like the reference.  ``cos_sin_cache`` is the reference's buffer
    ([max_position, 1, D] fp32) or the same values as [max_position, D].
    """
    _require_cuda(positions, query, key, cos_sin_cache)
    N, H, Hk, D, max_pos = _rope_args(positions, query, key, cos_sin_cache)
    q_out = torch.empty((N, H, D), dtype=query.dtype, device=query.device)
    k_out = torch.empty((N, Hk, D), dtype=key.dtype, device=key.device)
    st = lib().vlc_rope_store_kvcache(_ptr(positions), _ptr(query), query.stride(0), _ptr(q_out), q_out.stride(0),
                                      _ptr(key), key.stride(0), None, 0, _ptr(cos_sin_cache), max_pos, D, None,
                                      None, None, 0, _ptr(k_out), k_out.stride(0), N, H, Hk, D, _stream())
    check("vlc_rope_store_kvcache", st)
    return q_out, k_out


def rope_store_kvcache(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                       cos_sin_cache: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       slot_mapping: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """RoPE of ``query`` and ``key`` fused with the paged KV scatter: returns the roped
    query (into ``out`` when given; ``out`` may be ``query``) and writes the roped key
    and the value rows to ``k_cache`` / ``v_cache`` row ``slot_mapping[i]`` (-1 skipped).

    One launch for what the reference does in two steps: ``rotary_emb(positions, q, k)``
    (rotary_embedding.py:37-48) and ``store_kvcache`` (attention.py:10-40, with its
    stride assertions :33-40).  The key's K rows reach the cache roped, bit-identical to
    roping then scattering.
    """
    _require_cuda(positions, query, key, value, cos_sin_cache, k_cache, v_cache, slot_mapping)
    N, H, Hk, D, max_pos = _rope_args(positions, query, key, cos_sin_cache)
    assert value.shape == key.shape and value.stride(-1) == 1 and value.stride(1) == D
    assert value.dtype == torch.bfloat16 and k_cache.dtype == torch.bfloat16 and v_cache.dtype == torch.bfloat16
    row = Hk * D
    assert k_cache.stride(1) == row and v_cache.stride(1) == row    # as store_kvcache (attention.py:33-40)
    assert k_cache.is_contiguous() and v_cache.is_contiguous()
    assert slot_mapping.dtype == torch.int32 and slot_mapping.numel() == N and slot_mapping.is_contiguous()
    if out is None:
        out = torch.empty((N, H, D), dtype=query.dtype, device=query.device)
    assert out.shape == (N, H, D) and out.stride(-1) == 1 and out.stride(1) == D
    num_slots = k_cache.numel() // row
    st = lib().vlc_rope_store_kvcache(_ptr(positions), _ptr(query), query.stride(0), _ptr(out), out.stride(0),
                                      _ptr(key), key.stride(0), _ptr(value), value.stride(0), _ptr(cos_sin_cache),
                                      max_pos, D, _ptr(k_cache), _ptr(v_cache), _ptr(slot_mapping), num_slots,
                                      None, 0, N, H, Hk, D, _stream())
    check("vlc_rope_store_kvcache", st)
    return out


# --------------------------------------------------------------------------- M-RoPE shift
def mrope_shift(k_cache: torch.Tensor, v_cache: torch.Tensor | None, src_slots: torch.Tensor,
                dst_slots: torch.Tensor | None, delta_thw, mrope_section=DEFAULT_MROPE_SECTION,
                rope_theta: float = 1e6) -> None:
    """Re-rotate reused K rows of one layer by an M-RoPE position delta.

    ``k_cache``/``v_cache`` are one layer's ``[num_blocks, block_size, Hk, D]`` (or
    ``[num_slots, Hk, D]``) caches.  With ``dst_slots`` None the rotation is in place;
    otherwise K rows move (rotated) to ``dst_slots`` and V rows move verbatim.
    """
    _require_cuda(k_cache, v_cache, src_slots, dst_slots)
    assert k_cache.dtype == torch.bfloat16 and k_cache.is_contiguous()
    assert src_slots.dtype == torch.int32 and (dst_slots is None or dst_slots.dtype == torch.int32)
    Hk, hd = k_cache.shape[-2], k_cache.shape[-1]
    num_slots = k_cache.numel() // (Hk * hd)
    n = src_slots.numel()
    if dst_slots is not None:
        assert dst_slots.numel() == n
    d = (ctypes.c_int32 * 3)(*[int(x) for x in delta_thw])
    sec = (ctypes.c_int32 * 3)(*[int(x) for x in mrope_section])
    st = lib().vlc_mrope_shift(_ptr(k_cache), _ptr(v_cache), 0, 1, int(num_slots), int(Hk), int(hd),
                               _ptr(src_slots), _ptr(dst_slots), n, d, sec, float(rope_theta), _stream())
    check("vlc_mrope_shift", st)


def mrope_shift_all_layers(kv_cache: torch.Tensor, src_slots: torch.Tensor, dst_slots: torch.Tensor | None,
                           delta_thw, mrope_section=DEFAULT_MROPE_SECTION, rope_theta: float = 1e6) -> None:
    """Shift reused image rows of every layer of a ``[2, L, NB, BS, Hk, D]`` cache in one launch."""
    assert kv_cache.dim() == 6 and kv_cache.is_contiguous()
    L = kv_cache.shape[1]
    per_layer = kv_cache[0, 0].numel()
    k0 = kv_cache[0, 0]
    v0 = kv_cache[1, 0]
    Hk, hd = kv_cache.shape[4], kv_cache.shape[5]
    num_slots = kv_cache.shape[2] * kv_cache.shape[3]
    _require_cuda(kv_cache, src_slots, dst_slots)
    n = src_slots.numel()
    d = (ctypes.c_int32 * 3)(*[int(x) for x in delta_thw])
    sec = (ctypes.c_int32 * 3)(*[int(x) for x in mrope_section])
    st = lib().vlc_mrope_shift(_ptr(k0), _ptr(v0) if dst_slots is not None else ctypes.c_void_p(0),
                               per_layer, L, num_slots, Hk, hd, _ptr(src_slots), _ptr(dst_slots), n, d, sec,
                               float(rope_theta), _stream())
    check("vlc_mrope_shift", st)


# --------------------------------------------------------------------------- prefill
@dataclass
class PrefillPlan:
    """Host plan (numpy int32) plus its device copy and workspace size (bytes), and the key
    rows and sequences it was built for.  Behind a windowed plan, at ``lows_at``, stands the first key of each
    sequence that its first row's window shows (-1: it has no rows)."""
    host: np.ndarray
    dev: torch.Tensor | None
    workspace_bytes: int
    total_k: int = 0
    num_seqs: int = 0
    lows_at: int | None = None

    @property
    def host_ptr(self) -> int:
        """Address of ``host`` (cached: the launch path passes it on every call)."""
        p = self.__dict__.get("_host_ptr")
        if p is None:
            p = self.__dict__["_host_ptr"] = int(self.host.ctypes.data)
        return p

    @property
    def grid(self) -> int:
        return int(self.host[2])

    @property
    def num_units(self) -> int:
        return int(self.host[3])

    @property
    def num_parts(self) -> int:
        return int(self.host[4])

    @property
    def num_merges(self) -> int:
        return int(self.host[5])

    def split_tiles(self) -> list[tuple[int, int, int]]:
        """(first query row, query rows, KV head) of every tile whose keys are split over
        several units (its output goes through the log-sum-exp merge of partials)."""
        off, n = int(self.host[14]), self.num_merges
        rec = self.host[off:off + 8 * n].reshape(n, 8) if n else np.zeros((0, 8), np.int32)
        return [(int(r[0]), int(r[1]), int(r[2])) for r in rec]


PLAN_WINDOW, PLAN_SINKS = 22, 23   # of a plan's header (csrc/plan.h)
PREFILL_DEFAULT, PREFILL_PAIRS, PREFILL_QUADS = 0, 1, 2


def set_prefill_kernel(mode: int) -> None:
    """Unit kind of the prefill plans built from now on: ``PREFILL_PAIRS`` (two query tiles
    per unit on one SM), ``PREFILL_QUADS`` (four tiles per unit on a CTA pair) or
    ``PREFILL_DEFAULT``.  Each plan records its kind; the launch follows the plan."""
    check("vlc_prefill_set_kernel", lib().vlc_prefill_set_kernel(int(mode)))


def build_prefill_plan(cu_seqlens_q, cu_seqlens_k, num_heads: int, num_kv_heads: int, head_dim: int = HEAD_DIM,
                       num_sms: int = 0, device: torch.device | str | None = None, causal: bool = True,
                       window: int | None = None, sinks: int = 0, parts: torch.dtype | None = None) -> PrefillPlan:
    """Plan the warm-prefill attention launch from HOST cu_seqlens (lists/arrays/CPU tensors).
    ``causal=False`` plans the non-causal varlen attention (every row sees all keys of its
    sequence); ``head_dim`` may be 80..128 in steps of 16.  ``window`` > 0: a row at position t sees
    key j <= t iff j > t - window or j < ``sinks``; pages that no row sees are not read (their
    block-table entries may be -1).
    ``parts``: the type in which tiles that several CTAs share are kept until they are joined,
    torch.bfloat16 or torch.float32 (error against 64 bits 2.7e-3 or 1.7e-3; 48 rows behind 8000 keys 23.9 or
    27.8 us, and positive softmax scales only).  Unless said, fp32 where ``window`` is given, 0 (every key is
    visible, as without) among them, and bf16 else, as ``layers.attention`` plans layers without a window.
    A ``window`` above 0 and non-causal plans have one type only, fp32 and bf16."""
    if parts not in (None, torch.bfloat16, torch.float32):
        raise ValueError("parts: torch.bfloat16 or torch.float32")
    if (parts == torch.bfloat16 and window) or (parts == torch.float32 and not causal):
        raise ValueError("parts: fp32 under a window, bf16 in a non-causal plan")
    if parts is not None and not window:
        window = 0 if parts == torch.float32 else None
    cq = np.ascontiguousarray(np.asarray(cu_seqlens_q, dtype=np.int32))
    ck = np.ascontiguousarray(np.asarray(cu_seqlens_k, dtype=np.int32))
    nseq = len(cq) - 1
    assert len(ck) == nseq + 1
    L = lib()
    sms = int(num_sms) if num_sms else (L.vlc_num_sms() if device is not None else 148)
    cap = L.vlc_attention_plan_capacity(cq.ctypes.data, ck.ctypes.data, nseq, num_heads, num_kv_heads,
                                        1 if causal else 0, sms)
    if cap < 0:
        raise ValueError("invalid prefill metadata (cu_seqlens / heads)")
    plan = np.empty(int(cap), dtype=np.int32)   # (the planner writes all that it uses; zeroing 15 MB took 0.7 ms)
    used = ctypes.c_int64(0)
    sizes = (cq.ctypes.data, ck.ctypes.data, nseq, num_heads, num_kv_heads, head_dim, 1 if causal else 0)
    room = (sms, plan.ctypes.data, int(cap), ctypes.byref(used))
    if window is None:
        check("vlc_attention_plan", L.vlc_attention_plan(*sizes, *room))
    else:
        check("vlc_attention_plan_window", L.vlc_attention_plan_window(*sizes, int(window), int(sinks), *room))
    plan = plan[: used.value].copy()
    ws = int(L.vlc_prefill_workspace_size(plan.ctypes.data))
    lows_at = None
    if plan[PLAN_WINDOW] > 0:
        rows, keys = np.diff(cq), np.diff(ck)
        lows = np.where(rows > 0, np.maximum(0, keys - rows - int(plan[PLAN_WINDOW]) + 1), -1).astype(np.int32)
        lows_at, plan = len(plan), np.concatenate((plan, lows))
    dev = None
    if device is not None:
        dev = torch.from_numpy(plan).pin_memory().to(device, non_blocking=True)
    return PrefillPlan(host=plan, dev=dev, workspace_bytes=ws, total_k=int(ck[-1]), num_seqs=nseq,
                       lows_at=lows_at)


def prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, block_tables: torch.Tensor | None,
                      plan: PrefillPlan, softmax_scale: float, out: torch.Tensor | None = None,
                      workspace: torch.Tensor | None = None, k_new: torch.Tensor | None = None,
                      v_new: torch.Tensor | None = None) -> torch.Tensor:
    """Causal (bottom-right) varlen attention — the flash_attn_varlen_func contract.

    Paged: ``k``/``v`` are one layer's ``[num_blocks, block_size, Hk, D]`` caches and
    ``block_tables`` maps sequences to pages.  Contiguous (``block_tables`` None): ``k``/``v``
    are ``[total_k, Hk, D]`` (any token stride) laid out by cu_seqlens_k.
    The kernel is a programmatic dependent launch of the previous kernel on the
    stream: that kernel may produce q/k/v and ``block_tables``, but not the plan.

    Paged with ``k_new``/``v_new`` (the step's in-flight ``[total_q, Hk, D]`` rows, row i
    for query row i): sequences with q_len == k_len read their keys from those rows and
    start without waiting for the previous kernel, which may then only write the cache
    (the KV scatter, an ordinary launch) — ``vlc_prefill_attn_inflight``.
    """
    _require_cuda(q, k, v, block_tables)
    assert q.dtype == torch.bfloat16 and k.dtype == torch.bfloat16 and v.dtype == torch.bfloat16
    total_q, H, hd = q.shape
    assert q.stride(2) == 1 and q.stride(1) == hd
    Hk = k.shape[-2]
    assert k.stride(-1) == 1 and k.stride(-2) == hd and v.stride(-1) == 1 and v.stride(-2) == hd
    if block_tables is not None:
        assert k.dim() == 4 and k.is_contiguous() and v.is_contiguous()
        block_size = k.shape[1]
        rows = k.shape[0] * k.shape[1]
        k_stride = v_stride = Hk * hd
        assert block_tables.dtype == torch.int32 and block_tables.stride(-1) == 1
        bt_ptr, bt_stride = _ptr(block_tables), block_tables.stride(0)
    else:
        assert k.dim() == 3 and v.dim() == 3 and k.shape[0] == v.shape[0]
        block_size, rows = 0, k.shape[0]
        k_stride, v_stride = k.stride(0), v.stride(0)
        bt_ptr, bt_stride = ctypes.c_void_p(0), 0
    if out is None:
        out = torch.empty(total_q, H, hd, dtype=q.dtype, device=q.device)
    assert out.stride(2) == 1 and out.stride(1) == hd
    if plan.dev is None or plan.dev.device != q.device:
        plan.dev = torch.from_numpy(plan.host).to(q.device)
    if plan.workspace_bytes > 0 and (workspace is None or workspace.numel() * workspace.element_size()
                                     < plan.workspace_bytes):
        workspace = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=q.device)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    if k_new is not None:
        assert block_tables is not None and v_new is not None, "in-flight K/V go with a paged cache"
        _require_cuda(k_new, v_new)
        assert k_new.dim() == 3 and v_new.dim() == 3 and k_new.shape[1:] == (Hk, hd) and v_new.shape[1:] == (Hk, hd)
        assert k_new.shape[0] == v_new.shape[0] >= total_q
        assert k_new.stride(-1) == 1 and k_new.stride(-2) == hd and v_new.stride(-1) == 1 and v_new.stride(-2) == hd
        st = lib().vlc_prefill_attn_inflight(_ptr(q), q.stride(0), total_q, H, _ptr(k), _ptr(v), k_stride, v_stride,
                                             rows, Hk, hd, bt_ptr, bt_stride, block_size, _ptr(plan.dev),
                                             plan.host_ptr, float(softmax_scale), _ptr(out), out.stride(0),
                                             _ptr(workspace), ws_bytes, _ptr(k_new), _ptr(v_new), k_new.stride(0),
                                             v_new.stride(0), k_new.shape[0], _stream())
        check("vlc_prefill_attn_inflight", st)
        return out
    st = lib().vlc_prefill_attn(_ptr(q), q.stride(0), total_q, H, _ptr(k), _ptr(v), k_stride, v_stride, rows,
                                Hk, hd, bt_ptr, bt_stride, block_size, _ptr(plan.dev), plan.host_ptr,
                                float(softmax_scale), _ptr(out), out.stride(0), _ptr(workspace), ws_bytes,
                                _stream())
    check("vlc_prefill_attn", st)
    return out


# --------------------------------------------------------------------------- decode
def decode_workspace_bytes(num_seqs: int, num_heads: int, num_kv_heads: int, max_context_len: int) -> int:
    return int(lib().vlc_decode_workspace_size(num_seqs, num_heads, num_kv_heads, max_context_len))


def decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, max_context_len: int, softmax_scale: float,
                     out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """One-token paged decode (flash_attn_with_kvcache contract); q/out are ``[B, H, D]``."""
    _require_cuda(q, k_cache, v_cache, block_tables, context_lens)
    if q.dim() == 4:
        q = q.squeeze(1)
    B, H, hd = q.shape
    assert q.stride(2) == 1 and q.stride(1) == hd
    Hk = k_cache.shape[-2]
    block_size = k_cache.shape[1] if k_cache.dim() == 4 else 256
    num_slots = k_cache.numel() // (Hk * hd)
    assert context_lens.dtype == torch.int32 and block_tables.dtype == torch.int32
    if out is None:
        out = torch.empty(B, H, hd, dtype=q.dtype, device=q.device)
    need = decode_workspace_bytes(B, H, Hk, max_context_len)
    if need > 0 and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    st = lib().vlc_decode_attn(_ptr(q), q.stride(0), B, H, _ptr(k_cache), _ptr(v_cache), num_slots, Hk, hd,
                               _ptr(block_tables), block_tables.stride(0), block_size, _ptr(context_lens),
                               int(max_context_len), float(softmax_scale), _ptr(out), out.stride(0),
                               _ptr(workspace), ws_bytes, _stream())
    check("vlc_decode_attn", st)
    return out


# --------------------------------------------------------------------------- metadata
VSEQ_INTS, REUSE_INTS = 7, 8


def warm_metadata(desc: torch.Tensor, num_vseqs: int, reuse_offset: int, num_reuse: int, table_offset: int,
                  block_size: int, total_q: int, total_slots: int, table_rows: int, table_width: int,
                  total_reuse: int):
    """Device warm-prefill metadata from one int32 descriptor buffer ``desc`` =
    [virtual-sequence descriptors][reuse descriptors at reuse_offset][flat block tables at
    table_offset] (layout in include/vlcache_b200.h, vlc_warm_metadata).  Returns
    (positions int64, slot_mapping int32, block_tables int32 or None, src_slots, dst_slots)."""
    _require_cuda(desc)
    assert desc.dtype == torch.int32 and desc.is_contiguous()
    dev = desc.device
    positions = torch.empty(total_q, dtype=torch.int64, device=dev)
    slots = torch.empty(total_slots, dtype=torch.int32, device=dev)
    tables = torch.empty(table_rows, table_width, dtype=torch.int32, device=dev) if table_rows > 0 else None
    src = torch.empty(total_reuse, dtype=torch.int32, device=dev)
    dst = torch.empty(total_reuse, dtype=torch.int32, device=dev)
    base = desc.data_ptr()
    st = lib().vlc_warm_metadata(ctypes.c_void_p(base), num_vseqs, ctypes.c_void_p(base + 4 * reuse_offset),
                                 num_reuse, ctypes.c_void_p(base + 4 * table_offset), block_size,
                                 _ptr(positions), _ptr(slots) if total_slots > 0 else ctypes.c_void_p(0),
                                 _ptr(tables), table_width if tables is not None else 0, _ptr(src), _ptr(dst),
                                 _stream())
    check("vlc_warm_metadata", st)
    return positions, slots, tables, src, dst


# --------------------------------------------------------------------------- linear layers
LINEAR, SILU_MUL, QKV_ROPE = 0, 1, 2
_LINEAR_WS: dict = {}


def linear_workspace(kind: int, m: int, n: int, k: int, device) -> tuple[torch.Tensor | None, int]:
    """The stream-K workspace of a linear launch: one zeroed buffer per device, grown to
    the largest size asked for (each launch leaves it zeroed; launches on one stream never
    overlap).  Returns (tensor, bytes)."""
    need = int(lib().vlc_linear_workspace_size(kind, m, n, k))
    if need <= 0:
        return None, 0
    dev = torch.device(device)
    key = (dev.type, dev.index if dev.index is not None else torch.cuda.current_device())
    ws = _LINEAR_WS.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.zeros(need, dtype=torch.uint8, device=dev)
        _LINEAR_WS[key] = ws
    return ws, ws.numel()


def set_linear_kernel(mode: int) -> None:
    """GEMM kernel of the linear ops, process-wide: 0 automatic (a cost model picks per
    shape), 1 single-SM 128 x 256 tiles (stream-K where it pays), 2 CTA pairs
    (tcgen05.mma.cta_group::2, 256 x 256), 3 single-SM 128 x 128, 4 single-SM 128 x 224
    (plain linear only; the fused epilogues fall back to pairs)."""
    check("vlc_linear_set_kernel", lib().vlc_linear_set_kernel(int(mode)))


def reset_linear_workspaces() -> None:
    """Zero the cached stream-K workspaces (after a recorded device error)."""
    for ws in _LINEAR_WS.values():
        ws.zero_()


def _linear_args(x: torch.Tensor, weight: torch.Tensor):
    _require_cuda(x, weight)
    assert x.dim() == 2 and weight.dim() == 2 and x.shape[1] == weight.shape[1]
    assert x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16
    assert x.stride(1) == 1 and weight.stride(1) == 1
    return x.shape[0], x.shape[1]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
           out: torch.Tensor | None = None, stream_k: bool = True) -> torch.Tensor:
    """``F.linear(x, weight, bias)`` for bf16 ``x`` [m, k] and ``weight`` [n, k] on the
    tcgen05 GEMM (nanovllm/layers/linear.py:73, :154); ``stream_k=False`` runs whole
    output tiles per CTA (no workspace)."""
    m, k = _linear_args(x, weight)
    n = weight.shape[0]
    if bias is not None:
        _require_cuda(bias)
        assert bias.dtype == torch.bfloat16 and bias.is_contiguous() and bias.numel() == n
    if out is None:
        out = torch.empty(m, n, dtype=x.dtype, device=x.device)
    assert out.shape == (m, n) and out.stride(1) == 1
    ws, ws_bytes = linear_workspace(LINEAR, m, n, k, x.device) if stream_k else (None, 0)
    st = lib().vlc_linear(_ptr(x), x.stride(0), _ptr(weight), weight.stride(0), _ptr(bias), _ptr(out),
                          out.stride(0), m, n, k, _ptr(ws), ws_bytes, _stream())
    check("vlc_linear", st)
    return out


def linear_silu_mul(x: torch.Tensor, gate_up_weight: torch.Tensor, out: torch.Tensor | None = None,
                    stream_k: bool = True) -> torch.Tensor:
    """``SiluAndMul()(F.linear(x, gate_up_weight))`` in one kernel: ``gate_up_weight`` is
    [2 I, k] (gate rows then up rows); returns silu(gate) * up, [m, I]
    (nanovllm/models/qwen3.py:112-114, nanovllm/layers/activation.py:8-14)."""
    m, k = _linear_args(x, gate_up_weight)
    assert gate_up_weight.shape[0] % 2 == 0
    inter = gate_up_weight.shape[0] // 2
    if out is None:
        out = torch.empty(m, inter, dtype=x.dtype, device=x.device)
    assert out.shape == (m, inter) and out.stride(1) == 1
    ws, ws_bytes = linear_workspace(SILU_MUL, m, inter, k, x.device) if stream_k else (None, 0)
    st = lib().vlc_linear_silu_mul(_ptr(x), x.stride(0), _ptr(gate_up_weight), gate_up_weight.stride(0), _ptr(out),
                                   out.stride(0), m, inter, k, _ptr(ws), ws_bytes, _stream())
    check("vlc_linear_silu_mul", st)
    return out


def qkv_rope_store_kvcache(x: torch.Tensor, qkv_weight: torch.Tensor, qkv_bias: torch.Tensor | None,
                           positions: torch.Tensor, cos_sin_cache: torch.Tensor, k_cache: torch.Tensor,
                           v_cache: torch.Tensor, slot_mapping: torch.Tensor, num_heads: int, num_kv_heads: int,
                           q_out: torch.Tensor | None = None, stream_k: bool = True) -> torch.Tensor:
    """The QKV projection of the recomputed rows, its bias, the rotary embedding and the
    KV scatter in one kernel; returns the roped q [m, num_heads, 128] and writes the
    roped k and the v rows to the paged cache at ``slot_mapping`` (-1 skipped).
    Same result as ``qkv = F.linear(x, W, b)``; split; ``rotary_emb(positions, q, k)``;
    ``store_kvcache(k, v, ...)`` (nanovllm/models/qwen3.py:75-84), up to the GEMM's
    accumulation order."""
    m, hidden = _linear_args(x, qkv_weight)
    D = HEAD_DIM
    assert qkv_weight.shape[0] == (num_heads + 2 * num_kv_heads) * D
    _require_cuda(qkv_bias, positions, cos_sin_cache, k_cache, v_cache, slot_mapping)
    if qkv_bias is not None:
        assert qkv_bias.dtype == torch.bfloat16 and qkv_bias.is_contiguous()
    assert positions.dtype == torch.int64 and positions.is_contiguous() and positions.numel() == m
    assert cos_sin_cache.dtype == torch.float32 and cos_sin_cache.is_contiguous()
    assert cos_sin_cache.shape[-1] == D and cos_sin_cache.numel() == cos_sin_cache.shape[0] * D
    row = num_kv_heads * D
    assert k_cache.is_contiguous() and v_cache.is_contiguous()
    assert tuple(k_cache.shape[-2:]) == (num_kv_heads, D) and tuple(v_cache.shape) == tuple(k_cache.shape)
    assert slot_mapping.dtype == torch.int32 and slot_mapping.numel() == m and slot_mapping.is_contiguous()
    if q_out is None:
        q_out = torch.empty(m, num_heads, D, dtype=x.dtype, device=x.device)
    assert q_out.shape == (m, num_heads, D) and q_out.stride(2) == 1 and q_out.stride(1) == D
    ws, ws_bytes = linear_workspace(QKV_ROPE, m, qkv_weight.shape[0], hidden, x.device) if stream_k else (None, 0)
    st = lib().vlc_qkv_rope_store_kvcache(_ptr(x), x.stride(0), _ptr(qkv_weight), qkv_weight.stride(0),
                                          _ptr(qkv_bias), _ptr(positions), _ptr(cos_sin_cache),
                                          cos_sin_cache.shape[0], _ptr(q_out), q_out.stride(0), _ptr(k_cache),
                                          _ptr(v_cache), _ptr(slot_mapping), k_cache.numel() // row, m, hidden,
                                          num_heads, num_kv_heads, D, _ptr(ws), ws_bytes, _stream())
    check("vlc_qkv_rope_store_kvcache", st)
    return q_out


# --------------------------------------------------------------------------- content hash
def _header_buf(header: bytes):
    hb = bytes(header)
    return ctypes.create_string_buffer(hb, max(1, len(hb))), len(hb)


def content_hash_device_async(data: torch.Tensor, header: bytes = b"",
                              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Tree-XXH64 digest (include/vlcache_b200.h, vlc_content_hash_*) of a CUDA tensor's
    bytes with ``header``, as a one-element int64 device tensor (the uint64 bit pattern),
    computed on the current stream without any host synchronisation."""
    _require_cuda(data)
    assert data.is_contiguous(), "hash a contiguous tensor"
    nbytes = data.numel() * data.element_size()
    need = int(lib().vlc_content_hash_workspace_size(nbytes))
    if workspace is None or workspace.numel() * workspace.element_size() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=data.device)
    out = torch.empty(1, dtype=torch.int64, device=data.device)
    hb, hl = _header_buf(header)
    st = lib().vlc_content_hash_device(_ptr(data), nbytes, hb, hl, _ptr(workspace),
                                       workspace.numel() * workspace.element_size(), _ptr(out), _stream())
    check("vlc_content_hash_device", st)
    return out


def content_hash(data: torch.Tensor | np.ndarray, header: bytes = b"", num_threads: int = 0) -> int:
    """Tree-XXH64 digest of a tensor's bytes as a Python int: on the GPU when the tensor
    lives there (one 8-byte read back), else on the host threads."""
    if torch.is_tensor(data) and data.is_cuda:
        return int(content_hash_device_async(data, header).item()) & (2 ** 64 - 1)
    arr = np.ascontiguousarray(data.numpy() if torch.is_tensor(data) else data)
    hb, hl = _header_buf(header)
    out = ctypes.c_uint64(0)
    st = lib().vlc_content_hash_host(ctypes.c_void_p(arr.ctypes.data), arr.nbytes, hb, hl, num_threads,
                                     ctypes.byref(out))
    check("vlc_content_hash_host", st)
    return int(out.value)


def xxh64(data: bytes | np.ndarray, seed: int = 0) -> int:
    """Plain XXH64 of host bytes (the tree's primitive)."""
    arr = np.frombuffer(bytes(data), dtype=np.uint8) if not isinstance(data, np.ndarray) else \
        np.ascontiguousarray(data).reshape(-1).view(np.uint8)
    return int(lib().vlc_xxh64(ctypes.c_void_p(arr.ctypes.data if arr.size else 0), arr.size, seed))


# --------------------------------------------------------------------------- several-axes rotary
def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _device(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """Index of the CUDA device that all the tensors are on."""
    dev = first.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensors on {first.device} and {t.device}: one call takes one device")
    if dev < 0:
        raise ValueError("vlcache_b200 ops run on CUDA tensors only (no CPU fallback)")
    return dev


def _launch(dev: int, name: str, *args) -> None:
    """Call a C-ABI entry point on device ``dev`` and its current stream (the last argument)."""
    fn = getattr(lib(), name)
    if dev == (_raw_device() if _raw_device is not None else torch.cuda.current_device()):
        status = fn(*args, _stream())
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _stream())
    if status != 0:
        check(name, status)


def _rows(t: torch.Tensor, name: str) -> tuple[int, int, int, int]:
    """(tokens, heads, head_dim, token stride) of bf16 rows [tokens, heads, head_dim] with
    contiguous heads (any token stride)."""
    shape, stride = t.shape, t.stride()
    if t.dtype != torch.bfloat16 or len(shape) != 3:
        raise ValueError(f"{name}: bf16 [tokens, heads, head_dim]")
    n, h, d = shape
    if stride[2] != 1 or (h > 1 and stride[1] != d):
        raise ValueError(f"{name}: the heads of a token must be contiguous")
    return n, h, d, stride[0] if n > 1 else h * d


_INT3 = ctypes.c_int32 * 3
_SECTIONS: dict = {}   # pairs per axis -> the C array of them


def _sections(sections):
    sections = tuple(sections)
    array = _SECTIONS.get(sections)
    if array is None:
        if len(_SECTIONS) > 64:
            _SECTIONS.clear()
        array = _SECTIONS[sections] = (ctypes.c_int32 * len(sections))(*[int(x) for x in sections])
    return array


def _rotary_args(positions, cos_sin_cache, sections, n: int, d: int):
    """Positions and table of the rotating ops; returns (axis stride, axes, sections array, table rows)."""
    if sections is None:
        _need(positions.dim() == 1, "positions [tokens] (or [axes, tokens] with mrope_section)")
        sections = (d // 2,)
    array = _sections(sections)
    axes = len(array)
    shape, stride = positions.shape, positions.stride()
    _need(shape == (axes, n) or (axes == 1 and shape == (n,)), f"positions: [{axes}, {n}]")
    _need(positions.dtype == torch.int64 and (n <= 1 or stride[-1] == 1), "positions: int64, tokens contiguous")
    rows = cos_sin_cache.shape[0]
    _need(cos_sin_cache.dtype == torch.float32 and cos_sin_cache.is_contiguous() and cos_sin_cache.shape[-1] == d
          and cos_sin_cache.numel() == rows * d, "cos_sin_cache: contiguous fp32 [positions, (1,) head_dim]")
    return stride[0] if axes > 1 else n, axes, array, rows   # stride 0: one row of positions for every axis


def _q_out(query: torch.Tensor, out: torch.Tensor | None) -> tuple[torch.Tensor, int]:
    """The output in query's shape, a new one unless given, and its token stride."""
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
        return out, out.shape[1] * out.shape[2]
    _need(out.shape == query.shape, "out: query's shape")
    return out, _rows(out, "out")[3]


def _kv_rows(key: torch.Tensor, value: torch.Tensor, n: int, d: int) -> tuple[int, int, int]:
    """(KV heads, key's token stride, value's) of n tokens' key and value rows."""
    nk, hk, dk, ks = _rows(key, "key")
    nv, hv, dv, vs = _rows(value, "value")
    if nk != n or dk != d:
        raise ValueError("query and key: the same tokens and head_dim")
    if nv != n or hv != hk or dv != d:
        raise ValueError("value: key's shape")
    return hk, ks, vs


def _slots(slot_mapping: torch.Tensor, n: int) -> None:
    _need(slot_mapping.dtype == torch.int32 and slot_mapping.numel() == n and slot_mapping.is_contiguous(),
          "slot_mapping: contiguous int32, one per token")


def mrotary_embedding(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, cos_sin_cache: torch.Tensor,
                      mrope_section=DEFAULT_MROPE_SECTION) -> tuple[torch.Tensor, torch.Tensor]:
    """Rotate-half RoPE of ``query`` [N, H, D] and ``key`` [N, Hk, D] at ``positions``
    [axes, N] (time, height, width): pair j takes the position of the axis whose section of
    ``mrope_section`` (pairs per axis, summing to D / 2) holds it.  Returns new tensors;
    with equal positions on all axes they are ``rotary_embedding``'s, bit for bit."""
    dev = _device(query, positions, key, cos_sin_cache)
    n, h, d, qs = _rows(query, "query")
    nk, hk, dk, ks = _rows(key, "key")
    _need(nk == n and dk == d, "query and key: the same tokens and head_dim")
    axis, axes, sec, max_pos = _rotary_args(positions, cos_sin_cache, mrope_section, n, d)
    q_out, k_out = _q_out(query, None)[0], _q_out(key, None)[0]
    _launch(dev, "vlc_mrope_store_kvcache", positions.data_ptr(), axis, axes, sec, query.data_ptr(), qs,
            q_out.data_ptr(), h * d, key.data_ptr(), ks, None, 0, cos_sin_cache.data_ptr(), max_pos, None, None, None,
            0, k_out.data_ptr(), hk * d, n, h, hk, d)
    return q_out, k_out


def mrope_store_kvcache(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                        cos_sin_cache: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        slot_mapping: torch.Tensor, mrope_section=DEFAULT_MROPE_SECTION,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """``mrotary_embedding`` fused with the paged KV scatter, in one launch: returns the
    rotated query (into ``out`` when given; it may be ``query``) and writes the rotated key
    and the value rows to ``k_cache`` / ``v_cache`` row ``slot_mapping[i]`` (-1 skipped)."""
    dev = _device(query, positions, key, value, cos_sin_cache, k_cache, v_cache, slot_mapping, out)
    n, h, d, qs = _rows(query, "query")
    hk, ks, vs = _kv_rows(key, value, n, d)
    axis, axes, sec, max_pos = _rotary_args(positions, cos_sin_cache, mrope_section, n, d)
    shape = k_cache.shape
    _need(k_cache.dtype == torch.bfloat16 and v_cache.dtype == torch.bfloat16 and k_cache.is_contiguous()
          and v_cache.is_contiguous() and shape == v_cache.shape and shape[-2:] == (hk, d),
          "k_cache / v_cache: contiguous bf16 [.., num_kv_heads, head_dim]")
    _slots(slot_mapping, n)
    out, os = _q_out(query, out)
    _launch(dev, "vlc_mrope_store_kvcache", positions.data_ptr(), axis, axes, sec, query.data_ptr(), qs,
            out.data_ptr(), os, key.data_ptr(), ks, value.data_ptr(), vs, cos_sin_cache.data_ptr(), max_pos,
            k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), k_cache.numel() // (hk * d), None, 0, n,
            h, hk, d)
    return out


# --------------------------------------------------------------------------- the KV cache in 4 bits
FP4_ROW_BYTES = 72   # of one head's row: 64 of e2m1 codes, 8 of e4m3 scales (include/vlcache_b200.h)


def _fp4_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, dims: int = 3) -> tuple[int, int, int]:
    """(pages, KV heads, block size) of 4-bit caches uint8 [pages, Hk, block * 72], or with
    ``dims`` 4 of layers of them."""
    shape = k_cache.shape
    if k_cache.dtype != torch.uint8 or v_cache.dtype != torch.uint8 or len(shape) != dims:
        raise ValueError("a 4-bit cache is uint8 [pages, num_kv_heads, block_size * 72]")
    _need(v_cache.shape == shape, "k_cache and v_cache: the same shape")
    dense = (shape[-2] * shape[-1], shape[-1], 1)   # of a layer; layers may lie apart
    for t in (k_cache, v_cache):
        if t.stride()[-3:] != dense and not (t if dims == 3 or shape[0] == 0 else t[0]).is_contiguous():
            raise ValueError("4-bit caches must be contiguous")
    return shape[-3], shape[-2], _fp4_block(shape[-1])


def _tables(block_tables: torch.Tensor, num_seqs: int) -> tuple[int, int]:
    """(row stride, width) of int32 block tables [num_seqs, width]."""
    shape, stride = block_tables.shape, block_tables.stride()
    if block_tables.dtype != torch.int32 or len(shape) != 2 or shape[0] != num_seqs:
        raise ValueError(f"block_tables: int32 [{num_seqs}, width]")
    width = shape[1]
    _need(width <= 1 or stride[1] == 1, "block_tables: rows must be contiguous")
    return (stride[0] if num_seqs > 1 else width), width


def store_kvcache_fp4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slot_mapping: torch.Tensor, k_scale: float = 1.0, v_scale: float = 1.0) -> None:
    """``store_kvcache`` into a 4-bit cache (uint8 [pages, Hk, block * 72]): each group of 16
    dims becomes e2m1 codes and an e4m3 scale.  ``k_scale`` / ``v_scale``: the cache's
    powers of two (include/vlcache_b200.h says how values are held).  The slots of a call differ
    (of two rows for one slot, codes and scales could come from either)."""
    dev = _device(key, value, k_cache, v_cache, slot_mapping)
    n, hk, d, ks = _rows(key, "key")
    _need(value.shape == key.shape, "value: key's shape")
    vs = _rows(value, "value")[3]
    pages, heads, block = _fp4_caches(k_cache, v_cache)
    _need(heads == hk, "the caches' num_kv_heads")
    _slots(slot_mapping, n)
    _launch(dev, "vlc_store_kvcache_fp4", key.data_ptr(), ks, value.data_ptr(), vs, k_cache.data_ptr(),
            v_cache.data_ptr(), slot_mapping.data_ptr(), pages, block, float(k_scale), float(v_scale), n, hk, d)


def rope_store_kvcache_fp4(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                           cos_sin_cache: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           slot_mapping: torch.Tensor, mrope_section=None, k_scale: float = 1.0,
                           v_scale: float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """``rope_store_kvcache`` (or, with ``mrope_section``, ``mrope_store_kvcache``) into a 4-bit
    cache, in one launch: returns the rotated query; the rotated key, rounded to bf16, and
    the value are quantised into row ``slot_mapping[i]`` (-1 skipped), the same bytes as
    rotating first and ``store_kvcache_fp4`` after."""
    dev = _device(query, positions, key, value, cos_sin_cache, k_cache, v_cache, slot_mapping, out)
    n, h, d, qs = _rows(query, "query")
    hk, ks, vs = _kv_rows(key, value, n, d)
    axis, axes, sec, max_pos = _rotary_args(positions, cos_sin_cache, mrope_section, n, d)
    pages, heads, block = _fp4_caches(k_cache, v_cache)
    _need(heads == hk, "the caches' num_kv_heads")
    _slots(slot_mapping, n)
    out, os = _q_out(query, out)
    _launch(dev, "vlc_rope_store_kvcache_fp4", positions.data_ptr(), axis, axes, sec, query.data_ptr(), qs,
            out.data_ptr(), os, key.data_ptr(), ks, value.data_ptr(), vs, cos_sin_cache.data_ptr(), max_pos,
            k_cache.data_ptr(), v_cache.data_ptr(), slot_mapping.data_ptr(), pages, block, float(k_scale),
            float(v_scale), n, h, hk, d)
    return out


def gather_kvcache_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                       cu_seqlens_k: torch.Tensor, total_k: int, k_scale: float = 1.0, v_scale: float = 1.0,
                       k_out: torch.Tensor | None = None,
                       v_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The values of a 4-bit cache's keys and values, in bf16 (exact): row cu_seqlens_k[b] + j
    of the outputs [total_k, Hk, 128] is key j of sequence b.  With caches of several layers
    ([layers, pages, Hk, block * 72], e.g. ``kv_cache[0]``, ``kv_cache[1]``) the outputs are
    [layers, total_k, Hk, 128].  ``total_k`` is cu_seqlens_k's last entry, on the host."""
    dev = _device(k_cache, v_cache, block_tables, cu_seqlens_k, k_out, v_out)
    many = k_cache.dim() == 4
    pages, hk, block = _fp4_caches(k_cache, v_cache, 4 if many else 3)
    layers = k_cache.shape[0] if many else 1
    layer_stride = k_cache.stride(0) if layers > 1 else 0
    _need(layers <= 1 or v_cache.stride(0) == layer_stride, "k_cache and v_cache: the same layer stride")
    _need(cu_seqlens_k.dtype == torch.int32 and cu_seqlens_k.dim() == 1 and cu_seqlens_k.is_contiguous()
          and cu_seqlens_k.numel() >= 1, "cu_seqlens_k: contiguous int32 [num_seqs + 1]")
    seqs, total_k = cu_seqlens_k.numel() - 1, int(total_k)
    stride, width = _tables(block_tables, seqs)
    shape = (layers, total_k, hk, HEAD_DIM) if many else (total_k, hk, HEAD_DIM)
    for t in (k_out, v_out):
        if t is not None and (t.shape != shape or t.dtype != torch.bfloat16 or not t.is_contiguous()):
            raise ValueError(f"k_out / v_out: contiguous bf16 {list(shape)}")
    if k_out is None:
        k_out = torch.empty(*shape, dtype=torch.bfloat16, device=k_cache.device)
    if v_out is None:
        v_out = torch.empty_like(k_out)
    row = hk * HEAD_DIM
    _launch(dev, "vlc_gather_kvcache_fp4", k_cache.data_ptr(), v_cache.data_ptr(), layer_stride, layers, pages, block,
            hk, HEAD_DIM, block_tables.data_ptr(), stride, width, cu_seqlens_k.data_ptr(), seqs, total_k,
            float(k_scale), float(v_scale), k_out.data_ptr(), v_out.data_ptr(), row, total_k * row)
    return k_out, v_out


def _fp4_block(page_bytes: int) -> int:
    """Block size of a 4-bit page of that many bytes a head."""
    block = page_bytes // FP4_ROW_BYTES
    _need(block > 0 and page_bytes == block * FP4_ROW_BYTES, "a 4-bit page is block_size * 72 bytes a head")
    return block


def _shift_fp4(dev, k, v, layers, layer_stride, shape, src_slots, dst_slots, delta_thw, mrope_section,
               rope_theta) -> None:
    pages, hk, page_bytes = shape
    n = src_slots.numel()
    for t in (src_slots, dst_slots):
        _need(t is None or (t.dtype == torch.int32 and t.is_contiguous() and t.numel() == n),
              "src_slots / dst_slots: contiguous int32 of one length")
    _need(len(delta_thw) == 3 and len(mrope_section) == 3, "delta_thw and mrope_section: (t, h, w)")
    d = _INT3(*[int(x) for x in delta_thw])
    _launch(dev, "vlc_mrope_shift_fp4", k, v, layer_stride, layers, pages, _fp4_block(page_bytes), hk, HEAD_DIM,
            src_slots.data_ptr(), _ptr(dst_slots), n, d, _sections(mrope_section), float(rope_theta))


def mrope_shift_fp4(kv_cache: torch.Tensor, src_slots: torch.Tensor, dst_slots: torch.Tensor | None, delta_thw,
                    mrope_section=DEFAULT_MROPE_SECTION, rope_theta: float = 1e6) -> None:
    """``mrope_shift_all_layers`` in a 4-bit cache uint8 [2, L, pages, Hk, block * 72], one
    launch: K rows of ``src_slots`` turned by the position delta to ``dst_slots`` (None: in
    place), V rows copied.  A turned row is rounded to bf16 and quantised again; groups of
    16 pairs whose delta is 0 keep their bits, so a zero delta copies.  Destinations differ, and
    none may be another row's source (``engine.kv_cache.check_reuse_slots``)."""
    dev = _device(kv_cache, src_slots, dst_slots)
    shape, stride = kv_cache.shape, kv_cache.stride()
    _need(kv_cache.dtype == torch.uint8 and len(shape) == 5 and shape[0] == 2 and kv_cache.is_contiguous(),
          "kv_cache: contiguous uint8 [2, layers, pages, Hk, block * 72]")
    k = kv_cache.data_ptr()
    _shift_fp4(dev, k, k + stride[0], shape[1], stride[1], shape[2:], src_slots, dst_slots, delta_thw, mrope_section,
               rope_theta)


def mrope_shift_layer_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor | None, src_slots: torch.Tensor,
                          dst_slots: torch.Tensor | None, delta_thw, mrope_section=DEFAULT_MROPE_SECTION,
                          rope_theta: float = 1e6) -> None:
    """``mrope_shift_fp4`` of one layer's caches uint8 [pages, Hk, block * 72] (``v_cache`` None:
    K alone)."""
    dev = _device(k_cache, v_cache, src_slots, dst_slots)
    _fp4_caches(k_cache, k_cache if v_cache is None else v_cache)
    _shift_fp4(dev, k_cache.data_ptr(), _ptr(v_cache), 1, 0, k_cache.shape, src_slots, dst_slots, delta_thw,
               mrope_section, rope_theta)


def decode_fp4_workspace_bytes(num_seqs: int, num_heads: int, num_kv_heads: int, max_context_len: int) -> int:
    return int(lib().vlc_decode_fp4_workspace_size(num_seqs, num_heads, num_kv_heads, max_context_len))


def decode_attention_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                         context_lens: torch.Tensor, max_context_len: int, softmax_scale: float,
                         k_scale: float = 1.0, v_scale: float = 1.0, out: torch.Tensor | None = None,
                         workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``decode_attention`` over a 4-bit cache: one query token per sequence, q / out [B, H, 128]
    (q may be [B, 1, H, 128]); sequences of length 0 give zeros, a head whose query holds an infinity
    or a NaN gives NaN.  ``max_context_len`` bounds the lengths on the host and sizes the grid;
    ``workspace``: ``decode_fp4_workspace_bytes``, contiguous and 32-byte aligned, one per call in
    flight."""
    dev = _device(q, k_cache, v_cache, block_tables, context_lens, out, workspace)
    if q.dim() == 4:
        _need(q.shape[1] == 1, "q: one token per sequence")
        q = q.squeeze(1)
    b, h, d, qs = _rows(q, "q")
    pages, hk, block = _fp4_caches(k_cache, v_cache)
    stride, width = _tables(block_tables, b)
    _need(context_lens.dtype == torch.int32 and context_lens.numel() == b and context_lens.is_contiguous(),
          "context_lens: contiguous int32, one per sequence")
    out, os = _q_out(q, out)
    max_context_len = int(max_context_len)
    _need(0 <= max_context_len <= 1 << 30, "max_context_len: 0 .. 2^30")
    need = lib().vlc_decode_fp4_workspace_size(b, h, hk, max_context_len)
    if need > 0 and (workspace is None or workspace.nbytes < need):
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    _need(workspace is None or workspace.is_contiguous(), "workspace: contiguous")
    _launch(dev, "vlc_decode_attn_fp4", q.data_ptr(), qs, b, h, k_cache.data_ptr(), v_cache.data_ptr(), pages, block,
            hk, d, block_tables.data_ptr(), stride, width, context_lens.data_ptr(), max_context_len,
            float(softmax_scale), float(k_scale), float(v_scale), out.data_ptr(), os, _ptr(workspace),
            0 if workspace is None else workspace.nbytes)
    return out


def prefill_fp4_workspace_bytes(plan: PrefillPlan, num_kv_heads: int) -> int:
    """Workspace of ``prefill_attention_fp4``: the plan's, and the keys and values in bf16."""
    return _round_up(plan.workspace_bytes, 256) + 2 * plan.total_k * num_kv_heads * HEAD_DIM * 2


def _round_up(n: int, to: int) -> int:
    return (n + to - 1) // to * to


def prefill_attention_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                          cu_seqlens_k: torch.Tensor, plan: PrefillPlan, softmax_scale: float, k_scale: float = 1.0,
                          v_scale: float = 1.0, out: torch.Tensor | None = None,
                          workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``prefill_attention`` over a 4-bit cache: the sequences' keys and values are read back
    to bf16 once (``gather_kvcache_fp4``, exact), then the tcgen05 attention kernel runs on
    them.  A prompt's query tiles share each key, so each is converted once.  The read-back
    writes 512 bytes a key and KV head: 12 MB for one warm 4K-image request of 2 KV heads, which
    stay in L2 (4 of 24 us), 222 MB for 64 warm 1080p requests, which do not (48 of 263 us).  Under a plan's
    window, keys that no row sees are not read (their block-table entries may be -1).  As in
    ``prefill_attention``, P and the partial outputs of split tiles are bf16 (off by 2^-8 of
    themselves at most, each), where the 4-bit decode keeps P in f16 and its parts in fp32.
    ``cu_seqlens_k``: the plan's, on the device; ``workspace``: ``prefill_fp4_workspace_bytes``,
    256-byte aligned, one per call in flight."""
    dev = _device(q, k_cache, v_cache, block_tables, cu_seqlens_k, out, workspace)
    n, h, d, qs = _rows(q, "q")
    pages, hk, block = _fp4_caches(k_cache, v_cache)
    seqs, total_k = plan.num_seqs, plan.total_k
    _need(cu_seqlens_k.dtype == torch.int32 and cu_seqlens_k.is_contiguous() and cu_seqlens_k.numel() == seqs + 1,
          "cu_seqlens_k: contiguous int32, the plan's sequences")
    stride, width = _tables(block_tables, seqs)
    out, os = _q_out(q, out)
    if n == 0 and plan.num_units == 0:
        return out
    need = prefill_fp4_workspace_bytes(plan, hk)
    if workspace is None or workspace.nbytes < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    _need(workspace.is_contiguous(), "workspace: contiguous")
    if plan.dev is None or plan.dev.device != q.device:
        plan.dev = torch.from_numpy(plan.host).to(q.device)
    row = hk * HEAD_DIM
    k = workspace.data_ptr() + _round_up(plan.workspace_bytes, 256)
    v = k + 2 * total_k * row
    gather = (k_cache.data_ptr(), v_cache.data_ptr(), 0, 1, pages, block, hk, d, block_tables.data_ptr(), stride, width,
              cu_seqlens_k.data_ptr(), seqs, total_k, float(k_scale), float(v_scale), k, v, row, 0)
    if plan.lows_at is None:
        _launch(dev, "vlc_gather_kvcache_fp4", *gather)
    else:   # (keys that no row sees, whose pages may be gone, are left out)
        _launch(dev, "vlc_gather_seen_kvcache_fp4", *gather, plan.dev.data_ptr() + 4 * plan.lows_at,
                int(plan.host[PLAN_SINKS]))
    _launch(dev, "vlc_prefill_attn", q.data_ptr(), qs, n, h, k, v, row, row, total_k, hk, d, None, 0, 0,
            plan.dev.data_ptr(), plan.host_ptr, float(softmax_scale), out.data_ptr(), os, workspace.data_ptr(),
            plan.workspace_bytes)
    return out


# --------------------------------------------------------------------------- pages
def copy_kv_pages(kv_cache: torch.Tensor, src_pages: torch.Tensor, dst_pages: torch.Tensor) -> None:
    """Page ``dst_pages[i]`` becomes a copy of page ``src_pages[i]`` in every layer's K and V, in
    one launch: ``kv_cache[:, :, dst] = kv_cache[:, :, src]`` for a cache [2, L, pages, ...] of
    either format.  Pages of the lists (device int32) are copied in no order: destinations
    differ and none is another pair's source (``engine.page_pool`` makes such lists); pairs
    of -1 are skipped."""
    dev = _device(kv_cache, src_pages, dst_pages)
    _need(kv_cache.dim() >= 4 and kv_cache.is_contiguous(), "kv_cache: contiguous [2, layers, pages, ...]")
    n = src_pages.numel()
    for t in (src_pages, dst_pages):
        _need(t.dtype == torch.int32 and t.is_contiguous() and t.numel() == n,
              "src_pages / dst_pages: contiguous int32 of one length")
    shape = kv_cache.shape
    page = math.prod(shape[3:]) * kv_cache.element_size()   # (of a dim of size 1 the stride may be anything)
    _launch(dev, "vlc_copy_pages", kv_cache.data_ptr(), shape[2] * page, shape[0] * shape[1], page, shape[2],
            src_pages.data_ptr(), dst_pages.data_ptr(), n)


def remap_block_tables(block_tables: torch.Tensor, page_map: torch.Tensor) -> None:
    """Every entry p of the device block tables becomes ``page_map[p]`` (int32 [pages]); -1 stays."""
    dev = _device(block_tables, page_map)
    rows = block_tables.shape[0]
    stride, width = _tables(block_tables, rows)
    _need(page_map.dtype == torch.int32 and page_map.dim() == 1 and page_map.is_contiguous(),
          "page_map: contiguous int32 [pages]")
    _launch(dev, "vlc_remap_block_tables", block_tables.data_ptr(), stride, rows, width, page_map.data_ptr(),
            page_map.numel())


# --------------------------------------------------------------------------- a decode step with drafted tokens
_compiled = None


def _binding():
    """The compiled binding (checks, allocations and launches of the ops below in C++)."""
    global _compiled
    if _compiled is None:
        lib()   # raises where the kernels' library is missing
        from . import _binding as module
        _compiled = module
    return _compiled


def decode_window_workspace_bytes(num_seqs: int, num_tokens: int, num_heads: int, num_kv_heads: int,
                                  max_context_len: int, window: int = 0, sinks: int = 0) -> int:
    return int(lib().vlc_decode_window_workspace_size(num_seqs, num_tokens, num_heads, num_kv_heads, max_context_len,
                                                      window, sinks))


def decode_attention_window(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                            context_lens: torch.Tensor, max_context_len: int, softmax_scale: float, window: int = 0,
                            sinks: int = 0, out: torch.Tensor | None = None,
                            workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``decode_attention`` for the last ``n`` tokens of each sequence (drafted tokens to verify) and
    with a sliding window: q / out [B, n, H, 128] (or [B, H, 128]: n = 1), row r being token
    ``context_lens[b] - n + r``, whose key is in the cache.  The row at position t sees key j <= t iff
    ``window`` is 0, j > t - window or j < ``sinks``; pages that no row sees are not read (their
    block-table entries may be -1).  At most 128 rows n * H / Hk.  Tokens before a sequence's first
    and sequences of length 0 give zeros, a head whose query holds an infinity or a NaN gives NaN.
    ``max_context_len`` bounds the lengths on the host and sizes the grid; ``workspace``:
    ``decode_window_workspace_bytes``, contiguous, one per call in flight."""
    return (_compiled or _binding()).decode_attention_window(q, k_cache, v_cache, block_tables, context_lens,
                                                             max_context_len, softmax_scale, window, sinks, out,
                                                             workspace)


def step_metadata(context_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor,
                  free_pages: torch.Tensor, num_free: torch.Tensor, block_size: int, total_rows: int, window: int = 0,
                  sinks: int = 0) -> tuple[torch.Tensor, ...]:
    """Block tables and slot maps of a step, built on the device from the sequences' lengths, without a
    host read (so that it can be captured): sequence i of ``context_lens[i]`` tokens takes
    ``new_lens[i]`` more (a ``context_lens[i]`` below 0: an idle place of the batch, whose
    ``new_lens[i]`` rows have position 0 and slot -1, and which takes no page and has length 0 after).

    Missing entries (below 0) of ``block_tables`` [B, width] where they fall are filled from the end of
    the free list (``free_pages[:num_free]``, sequences in order), then pages wholly behind the
    ``window`` and the ``sinks`` go back to it; the three are updated in place (all int32).  Returns
    (positions int64 [total_rows], slot_mapping int32 [total_rows], cu_seqlens_q, cu_seqlens_k [B + 1],
    the lengths with the new tokens [B]); rows behind the last have position 0 and slot -1.
    ``total_rows`` bounds the new tokens on the host.  Pages that the list does not have, positions
    past the table and rows past ``total_rows`` are recorded (``device_error``) and have slot -1 or are
    left out (include/vlcache_b200.h).  The tables' pages are their own: forked requests, which share
    pages, stay with ``engine.page_pool``.  Any kernel may follow on the stream, the prefill too, which starts before
    this one has ended but reads the tables behind it."""
    return (_compiled or _binding()).step_metadata(context_lens, new_lens, block_tables, free_pages, num_free, block_size,
                                                   total_rows, window, sinks)


def verify_drafts(drafts: torch.Tensor, target_probs: torch.Tensor, draft_probs: torch.Tensor | None,
                  u: torch.Tensor, u_last: torch.Tensor, context_lens: torch.Tensor | None = None,
                  block_tables: torch.Tensor | None = None,
                  block_size: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Speculative sampling's verification, from given random numbers: draft i of each sequence
    (``drafts`` int64 [B, K], -1 from a sequence's end on) is accepted iff ``u[b, i] * draft_probs[b, i,
    d] < target_probs[b, i, d]``, up to the first refusal; then one token is sampled at ``u_last[b]``, from
    max(target - draft, 0) at the refused draft or from the target's row behind the last accepted one.

    ``target_probs`` [B, K + 1, vocabulary] and ``draft_probs`` [B, K, vocabulary] are of one type (fp32,
    bf16 or fp16); without ``draft_probs`` (drafts looked up, not sampled) a draft has probability 1,
    and refused it counts 0.  ``u`` [B, K] and ``u_last`` [B] are fp32 in [0, 1).  Returns (tokens int64
    [B, K + 1]: the accepted drafts, the sampled token, then -1; emitted int32 [B]: accepted + 1).
    ``context_lens`` (int32 [B], when given) is moved on by emitted in place: the step's first token and
    the accepted drafts are in the cache then (idle places, below 0, stay).  With the step's
    ``block_tables`` [B, width] and ``block_size`` (and ``context_lens``) that is so also where the free list ran out or
    a table ended: from the first row without a page on there are no drafts, and a sequence whose first row has
    none emits nothing (emitted 0, tokens -1, its length stays); its next step begins with the same token.
    Sums are whole numbers (include/vlcache_b200.h), so the answer is the same in every run and
    whatever the order of summation.  At most 31 drafts and 2^18 tokens of vocabulary."""
    return (_compiled or _binding()).verify_drafts(drafts, target_probs, draft_probs, u, u_last, context_lens, block_tables,
                                                   block_size)
