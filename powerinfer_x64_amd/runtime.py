"""torch-tensor front end of libpi_attn.so (include/pi_attn.h).

torch provides device memory and the stream; every computation runs in the
library's HIP kernels.  Calls are issued on torch's current stream so they
order with surrounding torch work.  Errors raise PiError subclasses that
mirror the reference's BackendError (src/runtime/mod.rs:6-18).
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

import numpy as np
import torch

from . import _abi

F32, F16, BF16 = 0, 1, 2
MODULO, GROUPED = 0, 1
PAGE_TOKENS = 16
ROPE_LAYOUTS = {"pairs": 0, "halves": 1}
ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}

_DTYPE_CODE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


class PiError(RuntimeError):
    code = -1


class InvalidArg(PiError):
    code = 1


class OutOfMemory(PiError):
    code = 2


class InvalidKernel(PiError):
    code = 3


class DeviceError(PiError):
    code = 4


class Unsupported(PiError):
    code = 5


_ERRORS = {c.code: c for c in (InvalidArg, OutOfMemory, InvalidKernel, DeviceError, Unsupported)}


# The handle of torch.cuda.current_stream(device) without its Stream object: 0.1 against 2 us, on
# every call.  Not a public name of torch: without it stream() takes the public way.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _vp(t: Optional[torch.Tensor]):
    """A tensor's address for a void* argument (an int: the signatures convert it)."""
    return None if t is None else t.data_ptr()


def _need(t: torch.Tensor, name: str, dtype=None, shape=None, dev=None):
    if not isinstance(t, torch.Tensor):
        raise InvalidArg(f"{name}: expected a torch.Tensor")
    if dev is not None and t.device != dev:
        raise InvalidArg(f"{name}: on {t.device}, expected {dev}")
    if dtype is not None and t.dtype != dtype:
        raise InvalidArg(f"{name}: dtype {t.dtype}, expected {dtype}")
    if shape is not None and t.shape != tuple(shape):
        raise InvalidArg(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise InvalidArg(f"{name}: must be contiguous")


class Device:
    """One pi_handle bound to a GPU (GpuDevice / GpuResources, src/cuda/mod.rs:141-460)."""

    def __init__(self, device: int = 0):
        self.lib = _abi.load()
        self.index = device
        self.torch_device = torch.device("cuda", device)
        h = ctypes.c_void_p()
        rc = self.lib.pi_create(device, ctypes.byref(h))
        if rc != 0:
            raise _ERRORS.get(rc, PiError)(self.lib.pi_last_error(None).decode())
        self.h = h
        torch.cuda.init()  # _raw_stream reads torch's current stream without checking

    def close(self):
        if self.h:
            self.lib.pi_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def stream(self):
        if _raw_stream is not None:
            return _raw_stream(self.index)
        return torch.cuda.current_stream(self.torch_device).cuda_stream

    def check(self, rc: int):
        if rc != 0:
            raise _ERRORS.get(rc, PiError)(self.lib.pi_last_error(self.h).decode())

    def sync(self):
        self.check(self.lib.pi_sync(self.h, self.stream()))


class KvPool:
    """Paged KV cache in HBM: 16-token pages, one K and one V block per (page, kv head)."""

    def __init__(self, dev: Device, n_pages: int, n_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.float16, page_tokens: int = PAGE_TOKENS):
        self.dev = dev
        self.n_pages, self.n_kv_heads, self.head_dim = n_pages, n_kv_heads, head_dim
        self.dtype = dtype
        p = ctypes.c_void_p()
        code = _DTYPE_CODE.get(dtype, -1)
        dev.check(dev.lib.pi_kv_pool_create(dev.h, n_pages, page_tokens, n_kv_heads, head_dim,
                                            code, ctypes.byref(p)))
        self.p = p

    @property
    def nbytes(self) -> int:
        return int(self.dev.lib.pi_kv_pool_bytes(self.p))

    def close(self):
        if self.p:
            self.dev.lib.pi_kv_pool_destroy(self.p)
            self.p = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def append(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
               start_pos: torch.Tensor):
        """k, v: [n_seq, n_tok, n_kv_heads, head_dim] (f32/f16/bf16)."""
        d = self.dev
        if k.dim() != 4 or k.shape[2:] != (self.n_kv_heads, self.head_dim):
            raise InvalidArg(f"k: shape {tuple(k.shape)}")
        for name, t in (("k", k), ("v", v)):
            _need(t, name, dtype=k.dtype, shape=k.shape, dev=d.torch_device)
        n_seq, n_tok = k.shape[:2]
        _need(page_table, "page_table", torch.int32, dev=d.torch_device)
        _need(start_pos, "start_pos", torch.int32, (n_seq,), d.torch_device)
        if page_table.dim() != 2 or page_table.shape[0] < n_seq:
            raise InvalidArg(f"page_table: shape {tuple(page_table.shape)}")
        d.check(d.lib.pi_kv_append(d.h, self.p, _vp(k), _vp(v), _DTYPE_CODE.get(k.dtype, -1),
                                   _vp(page_table), page_table.shape[1], _vp(start_pos), n_seq,
                                   n_tok, d.stream()))

    def read(self, page_table: torch.Tensor, seq: int, start: int, n_tok: int):
        d = self.dev
        _need(page_table, "page_table", torch.int32, dev=d.torch_device)
        ko = torch.empty((n_tok, self.n_kv_heads, self.head_dim), dtype=torch.float32,
                         device=d.torch_device)
        vo = torch.empty_like(ko)
        d.check(d.lib.pi_kv_read(d.h, self.p, _vp(page_table), page_table.shape[1], seq, start,
                                 n_tok, _vp(ko), _vp(vo), d.stream()))
        return ko, vo


class AttnLayer:
    """LayerCache of one attention layer for one sequence, on the device
    (src/model/mod.rs:73-106), with the forward step of src/model/mod.rs:1035-1196 on host
    slices (numpy float32), as the reference's InferenceContext::forward hands them over."""

    def __init__(self, dev: Device, max_tokens: int, n_heads: int, n_kv_heads: int,
                 head_dim: int, kv_dtype: torch.dtype = torch.float16, q_norm_w=None,
                 k_norm_w=None, eps: float = 1e-6, rope_dim: int = None,
                 rope_base: float = 1e6, sections=None, gqa_mode: int = MODULO,
                 q_head_dim: int = None, v_head_dim: int = None):
        """head_dim is the key head width; q_head_dim (>= head_dim) and v_head_dim default to
        it (src/model/mod.rs:976-982: the three may differ)."""
        self.dev = dev
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self.q_head_dim = head_dim if q_head_dim is None else q_head_dim
        self.v_head_dim = head_dim if v_head_dim is None else v_head_dim
        qn = None if q_norm_w is None else np.ascontiguousarray(q_norm_w, np.float32).reshape(-1)
        kn = None if k_norm_w is None else np.ascontiguousarray(k_norm_w, np.float32).reshape(-1)
        for name, w in (("q_norm_w", qn), ("k_norm_w", kn)):
            if w is not None and w.size != head_dim:
                raise InvalidArg(f"{name}: expected {head_dim} values, got {w.size}")
        sec = None if sections is None else (ctypes.c_int32 * 4)(*[int(x) for x in sections])
        p = ctypes.c_void_p()
        dev.check(dev.lib.pi_attn_layer_create_dims(
            dev.h, max_tokens, n_heads, n_kv_heads, self.q_head_dim, head_dim, self.v_head_dim,
            _DTYPE_CODE.get(kv_dtype, -1),
            None if qn is None else qn.ctypes.data_as(ctypes.c_void_p),
            None if kn is None else kn.ctypes.data_as(ctypes.c_void_p), float(eps),
            head_dim if rope_dim is None else rope_dim, float(rope_base), sec, gqa_mode,
            ctypes.byref(p)))
        self.p = p

    def close(self):
        if self.p:
            self.dev.lib.pi_attn_layer_destroy(self.p)
            self.p = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def seq_len(self) -> int:
        return int(self.dev.lib.pi_attn_layer_seq_len(self.p))

    def reset(self):
        self.dev.lib.pi_attn_layer_reset(self.p)

    def forward(self, q: np.ndarray, k: np.ndarray, v: np.ndarray, gate=None):
        """q [n, Hq, Dq], k [n, Hkv, D], v [n, Hkv, Dv] float32 (q, k normalised / rotated in
        place); gate like q; returns out [n, Hq, D]."""
        n = q.shape[0]
        for name, a, h, d in (("q", q, self.n_heads, self.q_head_dim),
                              ("k", k, self.n_kv_heads, self.head_dim),
                              ("v", v, self.n_kv_heads, self.v_head_dim)):
            if (not isinstance(a, np.ndarray) or a.dtype != np.float32 or
                    not a.flags.c_contiguous or a.shape != (n, h, d)):
                raise InvalidArg(f"{name}: expected C-contiguous float32 [{n}, {h}, {d}]")
        g = None
        if gate is not None:
            g = np.ascontiguousarray(gate, np.float32)
            if g.shape != q.shape:
                raise InvalidArg(f"gate: shape {g.shape}")
        out = np.empty((n, self.n_heads, self.head_dim), np.float32)
        vp = lambda a: None if a is None else a.ctypes.data_as(ctypes.c_void_p)
        self.dev.check(self.dev.lib.pi_attn_layer_forward(self.dev.h, self.p, vp(q), vp(k), vp(v),
                                                          vp(g), n, vp(out)))
        return out

    def forward_dev(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
        """The same step on device tensors (f32, q / gate [n, Hq, Dq], k [n, Hkv, D],
        v [n, Hkv, Dv]; q and k normalised / rotated in place), enqueued on torch's current
        stream; returns out [n, Hq, D]."""
        d = self.dev
        n = q.shape[0]
        _need(q, "q", torch.float32, (n, self.n_heads, self.q_head_dim), d.torch_device)
        _need(k, "k", torch.float32, (n, self.n_kv_heads, self.head_dim), d.torch_device)
        _need(v, "v", torch.float32, (n, self.n_kv_heads, self.v_head_dim), d.torch_device)
        if gate is not None:
            _need(gate, "gate", torch.float32, q.shape, d.torch_device)
        shp = (n, self.n_heads, self.head_dim)
        if out is None:
            out = torch.empty(shp, dtype=torch.float32, device=q.device)
        _need(out, "out", torch.float32, shp, d.torch_device)
        d.check(d.lib.pi_attn_layer_forward_dev(d.h, self.p, _vp(q), _vp(k), _vp(v), _vp(gate), n,
                                                _vp(out), d.stream()))
        return out


class GdnLayer:
    """Gated-DeltaNet layer of one sequence, on the device: the rolling conv state and the
    recurrent state (src/model/mod.rs:122-127), with the step of src/model/mod.rs:750-932 on
    host slices (numpy float32): conv1d + SiLU, q / k / v split, gates, the delta rule and
    RMSNormGated."""

    def __init__(self, dev: Device, n_k_heads: int, n_v_heads: int, k_hd: int, v_hd: int,
                 conv_w, ssm_a, dt_bias, norm_w, eps: float = 1e-6):
        self.dev = dev
        self.hk, self.hv, self.dk, self.dv = n_k_heads, n_v_heads, k_hd, v_hd
        self.conv_dim = 2 * n_k_heads * k_hd + n_v_heads * v_hd
        w = np.ascontiguousarray(conv_w, np.float32)
        if w.ndim != 2 or w.shape[0] != self.conv_dim:
            raise InvalidArg(f"conv_w: expected [{self.conv_dim}, d_conv], got {w.shape}")
        arrs = [np.ascontiguousarray(a, np.float32).reshape(-1) for a in (ssm_a, dt_bias, norm_w)]
        for name, a, m in zip(("ssm_a", "dt_bias", "norm_w"), arrs, (n_v_heads, n_v_heads, v_hd)):
            if a.size != m:
                raise InvalidArg(f"{name}: expected {m} values, got {a.size}")
        vp = lambda a: a.ctypes.data_as(ctypes.c_void_p)
        p = ctypes.c_void_p()
        dev.check(dev.lib.pi_gdn_layer_create(dev.h, n_k_heads, n_v_heads, k_hd, v_hd,
                                              w.shape[1], vp(w), vp(arrs[0]), vp(arrs[1]),
                                              vp(arrs[2]), float(eps), ctypes.byref(p)))
        self.p = p

    def close(self):
        if self.p:
            self.dev.lib.pi_gdn_layer_destroy(self.p)
            self.p = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def reset(self):
        self.dev.check(self.dev.lib.pi_gdn_layer_reset(self.dev.h, self.p))

    def forward(self, qkv: np.ndarray, z: np.ndarray, beta_raw: np.ndarray, a_raw: np.ndarray):
        """qkv [n, conv_dim], z [n, Hv, Dv], beta_raw, a_raw [n, Hv] float32; returns the
        gated, normalised output [n, Hv, Dv]."""
        n = qkv.shape[0]
        for name, a, shp in (("qkv", qkv, (n, self.conv_dim)), ("z", z, (n, self.hv, self.dv)),
                             ("beta_raw", beta_raw, (n, self.hv)), ("a_raw", a_raw, (n, self.hv))):
            if (not isinstance(a, np.ndarray) or a.dtype != np.float32 or
                    not a.flags.c_contiguous or a.shape != shp):
                raise InvalidArg(f"{name}: expected C-contiguous float32 {list(shp)}")
        out = np.empty((n, self.hv, self.dv), np.float32)
        vp = lambda a: a.ctypes.data_as(ctypes.c_void_p)
        self.dev.check(self.dev.lib.pi_gdn_layer_forward(self.dev.h, self.p, vp(qkv), vp(z),
                                                         vp(beta_raw), vp(a_raw), n, vp(out)))
        return out

    def forward_dev(self, qkv: torch.Tensor, z: torch.Tensor, beta_raw: torch.Tensor,
                    a_raw: torch.Tensor, out: Optional[torch.Tensor] = None):
        """The same step on device f32 tensors, enqueued on torch's current stream."""
        d = self.dev
        n = qkv.shape[0]
        for name, t, shp in (("qkv", qkv, (n, self.conv_dim)), ("z", z, (n, self.hv, self.dv)),
                             ("beta_raw", beta_raw, (n, self.hv)), ("a_raw", a_raw, (n, self.hv))):
            _need(t, name, torch.float32, shp, d.torch_device)
        if out is None:
            out = torch.empty((n, self.hv, self.dv), dtype=torch.float32, device=qkv.device)
        _need(out, "out", torch.float32, (n, self.hv, self.dv), d.torch_device)
        d.check(d.lib.pi_gdn_layer_forward_dev(d.h, self.p, _vp(qkv), _vp(z), _vp(beta_raw),
                                               _vp(a_raw), n, _vp(out), d.stream()))
        return out


class TqPool:
    """TurboQuant compressed KV cache (CompressedKVCache, src/turboquant/mod.rs:408-566) in
    16-token pages: ceil(head_dim/2)-byte 3-bit + QJL key records with f32 norms, f16
    values; head_dim 1..256."""

    def __init__(self, dev: Device, n_pages: int, n_kv_heads: int, head_dim: int = 128,
                 page_tokens: int = PAGE_TOKENS):
        self.dev = dev
        self.n_pages, self.n_kv_heads, self.head_dim = n_pages, n_kv_heads, head_dim
        self.KEY_BYTES = (4 * head_dim + 7) // 8
        p = ctypes.c_void_p()
        dev.check(dev.lib.pi_tq_pool_create(dev.h, n_pages, page_tokens, n_kv_heads, head_dim,
                                            ctypes.byref(p)))
        self.p = p

    @property
    def nbytes(self) -> int:
        return int(self.dev.lib.pi_tq_pool_bytes(self.p))

    def close(self):
        if self.p:
            self.dev.lib.pi_tq_pool_destroy(self.p)
            self.p = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def append(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor,
               start_pos: torch.Tensor):
        """k, v: [n_seq, n_tok, n_kv_heads, head_dim] f32."""
        d = self.dev
        if k.dim() != 4 or k.shape[2:] != (self.n_kv_heads, self.head_dim):
            raise InvalidArg(f"k: shape {tuple(k.shape)}")
        for name, t in (("k", k), ("v", v)):
            _need(t, name, dtype=torch.float32, shape=k.shape, dev=d.torch_device)
        n_seq, n_tok = k.shape[:2]
        _need(page_table, "page_table", torch.int32, dev=d.torch_device)
        _need(start_pos, "start_pos", torch.int32, (n_seq,), d.torch_device)
        if page_table.dim() != 2 or page_table.shape[0] < n_seq:
            raise InvalidArg(f"page_table: shape {tuple(page_table.shape)}")
        d.check(d.lib.pi_tq_append(d.h, self.p, _vp(k), _vp(v), _vp(page_table),
                                   page_table.shape[1], _vp(start_pos), n_seq, n_tok, d.stream()))

    def read(self, page_table: torch.Tensor, seq: int, start: int, n_tok: int):
        """(keys [n_tok, Hkv, ceil(head_dim/2)] uint8, norms [n_tok, Hkv] f32, values
        [n_tok, Hkv, head_dim] f16)."""
        d = self.dev
        _need(page_table, "page_table", torch.int32, dev=d.torch_device)
        ko = torch.empty((n_tok, self.n_kv_heads, self.KEY_BYTES), dtype=torch.uint8,
                         device=d.torch_device)
        no = torch.empty((n_tok, self.n_kv_heads), dtype=torch.float32, device=d.torch_device)
        vo = torch.empty((n_tok, self.n_kv_heads, self.head_dim), dtype=torch.float16,
                         device=d.torch_device)
        d.check(d.lib.pi_tq_read(d.h, self.p, _vp(page_table), page_table.shape[1], seq, start,
                                 n_tok, _vp(ko), _vp(no), _vp(vo), d.stream()))
        return ko, no, vo


def tq_generate(dim: int, seed: int):
    """Host only: (rotation, QJL matrix) of TurboQuant::new(bits, dim, dim, seed)."""
    lib = _abi.load()
    rot = np.empty((dim, dim), dtype=np.float32)
    qjl = np.empty((dim, dim), dtype=np.float32)
    rc = lib.pi_tq_generate(dim, seed, rot.ctypes.data_as(ctypes.c_void_p),
                            qjl.ctypes.data_as(ctypes.c_void_p))
    if rc != 0:
        raise _ERRORS.get(rc, PiError)(lib.pi_last_error(None).decode())
    return rot, qjl


def tq_attn_decode(dev: Device, q: torch.Tensor, pool: TqPool, page_table: torch.Tensor,
                   ctx_len: torch.Tensor, gqa_mode: int = MODULO,
                   gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """q [B, Hq, D] f32 -> out [B, Hq, D] f32 over each sequence's compressed cache."""
    _need(q, "q", torch.float32, dev=dev.torch_device)
    b, hq, dh = q.shape
    if dh != pool.head_dim:
        raise InvalidArg(f"q head_dim {dh} != pool head_dim {pool.head_dim}")
    _need(page_table, "page_table", torch.int32, dev=dev.torch_device)
    if page_table.dim() != 2 or page_table.shape[0] != b:
        raise InvalidArg(f"page_table: shape {tuple(page_table.shape)}")
    _need(ctx_len, "ctx_len", torch.int32, (b,), dev.torch_device)
    if gate is not None:
        _need(gate, "gate", torch.float32, q.shape, dev.torch_device)
    if out is None:
        out = torch.empty_like(q)
    _need(out, "out", torch.float32, q.shape, dev.torch_device)
    dev.check(dev.lib.pi_tq_attn_decode(dev.h, _vp(q), pool.p, _vp(page_table),
                                        page_table.shape[1], _vp(ctx_len), b, hq, gqa_mode,
                                        _vp(gate), _vp(out), dev.stream()))
    return out


def head_rmsnorm(dev: Device, x: torch.Tensor, w: torch.Tensor, eps: float):
    """In place: every row of the last dimension of x (f32) is RMS-normalised and scaled by w."""
    _need(x, "x", torch.float32, dev=dev.torch_device)
    dim = x.shape[-1]
    _need(w, "w", torch.float32, (dim,), dev.torch_device)
    dev.check(dev.lib.pi_head_rmsnorm(dev.h, _vp(x), _vp(w), x.numel() // dim, dim, dim,
                                      float(eps), dev.stream()))
    return x


def rope(dev: Device, q: torch.Tensor, k: Optional[torch.Tensor], pos: torch.Tensor,
         rope_dim: int, base: float, sections: Optional[Sequence[int]] = None):
    """In place on q [n_tok, Hq, D] and k [n_tok, Hkv, D] (f32) at positions pos [n_tok]."""
    _need(q, "q", torch.float32, dev=dev.torch_device)
    n_tok, hq, dh = q.shape
    hkv = 1
    if k is not None:
        _need(k, "k", torch.float32, dev=dev.torch_device)
        if k.shape[0] != n_tok or k.shape[2] != dh:
            raise InvalidArg(f"k: shape {tuple(k.shape)}")
        hkv = k.shape[1]
    _need(pos, "pos", torch.int32, (n_tok,), dev.torch_device)
    sec = None
    if sections is not None:
        sec = (ctypes.c_int32 * 4)(*[int(s) for s in sections])
    dev.check(dev.lib.pi_rope(dev.h, _vp(q), _vp(k), _vp(pos), n_tok, hq, hkv, dh, rope_dim,
                              float(base), sec, dev.stream()))
    return q, k


def attn_decode(dev: Device, q: torch.Tensor, pool: KvPool, page_table: torch.Tensor,
                ctx_len: torch.Tensor, gqa_mode: int = MODULO, scale: Optional[float] = None,
                gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """q [B, Hq, D] f32 -> out [B, Hq, D] f32 over each sequence's ctx_len[b] cached tokens."""
    _need(q, "q", torch.float32, dev=dev.torch_device)
    b, hq, dh = q.shape
    if dh != pool.head_dim:
        raise InvalidArg(f"q head_dim {dh} != pool head_dim {pool.head_dim}")
    _need(page_table, "page_table", torch.int32, dev=dev.torch_device)
    if page_table.dim() != 2 or page_table.shape[0] != b:
        raise InvalidArg(f"page_table: shape {tuple(page_table.shape)}")
    _need(ctx_len, "ctx_len", torch.int32, (b,), dev.torch_device)
    if gate is not None:
        _need(gate, "gate", torch.float32, q.shape, dev.torch_device)
    if out is None:
        out = torch.empty_like(q)
    _need(out, "out", torch.float32, q.shape, dev.torch_device)
    if scale is None:
        scale = 1.0 / math.sqrt(dh)
    dev.check(dev.lib.pi_attn_decode(dev.h, _vp(q), pool.p, _vp(page_table), page_table.shape[1],
                                     _vp(ctx_len), b, hq, gqa_mode, float(scale), _vp(gate),
                                     _vp(out), dev.stream()))
    return out


def attn_prefill(dev: Device, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                 causal: bool = True, gqa_mode: int = MODULO, scale: Optional[float] = None,
                 out: Optional[torch.Tensor] = None):
    """q [B, S, Hq, D], k/v [B, S, Hkv, D] (bf16/f16) -> out [B, S, Hq, D] f32."""
    _need(q, "q", dev=dev.torch_device)
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise Unsupported(f"q: dtype {q.dtype} (bf16 or f16)")
    bsz, s, hq, dh = q.shape
    _need(k, "k", q.dtype, dev=dev.torch_device)
    hkv = k.shape[2]
    _need(k, "k", q.dtype, (bsz, s, hkv, dh), dev.torch_device)
    _need(v, "v", q.dtype, (bsz, s, hkv, dh), dev.torch_device)
    if out is None:
        out = torch.empty((bsz, s, hq, dh), dtype=torch.float32, device=q.device)
    _need(out, "out", torch.float32, (bsz, s, hq, dh), dev.torch_device)
    if scale is None:
        scale = 1.0 / math.sqrt(dh)
    dev.check(dev.lib.pi_attn_prefill(dev.h, _vp(q), _vp(k), _vp(v), _DTYPE_CODE[q.dtype], bsz,
                                      s, hq, hkv, dh, 1 if causal else 0, gqa_mode, float(scale),
                                      _vp(out), dev.stream()))
    return out


def attn_prefill_paged(dev: Device, q: torch.Tensor, pool: KvPool, page_row: torch.Tensor,
                       start_pos: int, gqa_mode: int = MODULO, scale: Optional[float] = None,
                       out: Optional[torch.Tensor] = None):
    """A chunk continuing a sequence: q [n, Hq, D] at positions start_pos .. start_pos + n - 1
    over the sequence's pages (page_row: int32 [max_pages]; the chunk's K/V appended first)
    -> out [n, Hq, D] f32.  q is f16 for an f16 pool, f32 for an f32 pool."""
    _need(q, "q", pool.dtype, dev=dev.torch_device)
    n, hq, dh = q.shape
    if dh != pool.head_dim:
        raise InvalidArg(f"q head_dim {dh} != pool head_dim {pool.head_dim}")
    _need(page_row, "page_row", torch.int32, dev=dev.torch_device)
    if out is None:
        out = torch.empty((n, hq, dh), dtype=torch.float32, device=q.device)
    _need(out, "out", torch.float32, (n, hq, dh), dev.torch_device)
    if scale is None:
        scale = 1.0 / math.sqrt(dh)
    dev.check(dev.lib.pi_attn_prefill_paged(dev.h, _vp(q), pool.p, _vp(page_row), page_row.numel(),
                                            int(start_pos), n, hq, gqa_mode, float(scale), _vp(out),
                                            dev.stream()))
    return out


def gdn_gates(dev: Device, beta_raw, a_raw, ssm_a, dt_bias):
    """beta_raw/a_raw [n_tok, Hv], ssm_a/dt_bias [Hv] (f32) -> (beta, g)."""
    n_tok, hv = beta_raw.shape
    for name, t, shp in (("beta_raw", beta_raw, (n_tok, hv)), ("a_raw", a_raw, (n_tok, hv)),
                         ("ssm_a", ssm_a, (hv,)), ("dt_bias", dt_bias, (hv,))):
        _need(t, name, torch.float32, shp, dev.torch_device)
    beta = torch.empty_like(beta_raw)
    g = torch.empty_like(beta_raw)
    dev.check(dev.lib.pi_gdn_gates(dev.h, _vp(beta_raw), _vp(a_raw), _vp(ssm_a), _vp(dt_bias),
                                   _vp(beta), _vp(g), n_tok, hv, dev.stream()))
    return beta, g


def _gdn_check(dev, q, k, v, beta, g, state, lead):
    hk, dk = q.shape[-2:]
    hv, dv = v.shape[-2:]
    _need(q, "q", torch.float32, (lead, hk, dk), dev.torch_device)
    _need(k, "k", torch.float32, (lead, hk, dk), dev.torch_device)
    _need(v, "v", torch.float32, (lead, hv, dv), dev.torch_device)
    _need(beta, "beta", torch.float32, (lead, hv), dev.torch_device)
    _need(g, "g", torch.float32, (lead, hv), dev.torch_device)
    return hk, hv, dk, dv


def gdn_decode(dev: Device, q, k, v, beta, g, state, out=None):
    """One step per sequence: q/k [B, Hk, Dk] raw, v [B, Hv, Dv], beta/g [B, Hv],
    state [B, Hv, Dk, Dv] (in/out)."""
    b = q.shape[0]
    hk, hv, dk, dv = _gdn_check(dev, q, k, v, beta, g, state, b)
    _need(state, "state", torch.float32, (b, hv, dk, dv), dev.torch_device)
    if out is None:
        out = torch.empty((b, hv, dv), dtype=torch.float32, device=q.device)
    _need(out, "out", torch.float32, (b, hv, dv), dev.torch_device)
    dev.check(dev.lib.pi_gdn_decode(dev.h, _vp(q), _vp(k), _vp(v), _vp(beta), _vp(g), _vp(state),
                                    _vp(out), b, hk, hv, dk, dv, dev.stream()))
    return out


def gdn_prefill(dev: Device, q, k, v, beta, g, state, out=None, chunk: int = 64):
    """n_tok tokens of one sequence: q/k [T, Hk, Dk], v [T, Hv, Dv], beta/g [T, Hv],
    state [Hv, Dk, Dv] (in/out)."""
    t = q.shape[0]
    hk, hv, dk, dv = _gdn_check(dev, q, k, v, beta, g, state, t)
    _need(state, "state", torch.float32, (hv, dk, dv), dev.torch_device)
    if out is None:
        out = torch.empty((t, hv, dv), dtype=torch.float32, device=q.device)
    _need(out, "out", torch.float32, (t, hv, dv), dev.torch_device)
    dev.check(dev.lib.pi_gdn_prefill(dev.h, _vp(q), _vp(k), _vp(v), _vp(beta), _vp(g),
                                     _vp(state), _vp(out), t, hk, hv, dk, dv, chunk,
                                     dev.stream()))
    return out


def ssm_forward(dev: Device, x, ssm_conv1d, ssm_a, ssm_dt_bias, ssm_alpha, ssm_beta, ssm_out,
                state: np.ndarray, d_inner: int, d_state: int, d_conv: int) -> np.ndarray:
    """ssm::ssm_forward (src/ssm/mod.rs:40-157) on host slices, computed on the GPU: returns
    y [d_inner] and updates `state` (float32 [d_state * d_inner], C-contiguous) in place.
    ssm_conv1d, ssm_beta and ssm_out pick the reference's branches by their lengths."""
    f = lambda a: np.ascontiguousarray(np.asarray(a, np.float32).reshape(-1))  # noqa: E731
    x, w, a, bias, alpha, beta, out_w = (f(v) for v in (x, ssm_conv1d, ssm_a, ssm_dt_bias,
                                                        ssm_alpha, ssm_beta, ssm_out))
    if (not isinstance(state, np.ndarray) or state.dtype != np.float32 or
            not state.flags.c_contiguous or state.size != d_state * d_inner):
        raise InvalidArg(f"state: expected C-contiguous float32 of {d_state * d_inner} values")
    for name, arr, n in (("x", x, d_inner), ("ssm_dt_bias", bias, d_inner),
                         ("ssm_a", a, d_state * d_inner), ("ssm_alpha", alpha, d_inner * d_inner)):
        if arr.size != n:
            raise InvalidArg(f"{name}: expected {n} values, got {arr.size}")
    y = np.empty(d_inner, np.float32)
    vp = lambda arr: arr.ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    dev.check(dev.lib.pi_ssm_forward(dev.h, vp(y), vp(x), vp(w), w.size, vp(a), vp(bias),
                                     vp(alpha), vp(beta), beta.size, vp(out_w), out_w.size,
                                     vp(state), d_inner, d_state, d_conv))
    return y


def attention_head(dev: Device, q: np.ndarray, k_cache: np.ndarray, v_cache: np.ndarray,
                   seq_len: int, head_dim: int) -> np.ndarray:
    """ops::attention_head (src/ops.rs:213-247) on host slices, computed on the GPU."""
    q = np.ascontiguousarray(q, dtype=np.float32)
    k = np.ascontiguousarray(k_cache, dtype=np.float32)
    v = np.ascontiguousarray(v_cache, dtype=np.float32)
    if q.size < head_dim or k.size < seq_len * head_dim or v.size < seq_len * head_dim:
        raise InvalidArg("attention_head: slice shorter than seq_len * head_dim")
    out = np.zeros(head_dim, dtype=np.float32)
    fp = ctypes.POINTER(ctypes.c_float)
    dev.check(dev.lib.pi_ops_attention_head(dev.h, out.ctypes.data_as(fp), q.ctypes.data_as(fp),
                                            k.ctypes.data_as(fp), v.ctypes.data_as(fp), seq_len,
                                            head_dim))
    return out


def gdn_conv1d(dev: Device, x, conv_state, w, out=None):
    """Depthwise causal conv1d + SiLU: x [n_seq, n_tok, conv_dim], conv_state
    [n_seq, d_conv-1, conv_dim] (in/out), w [conv_dim, d_conv] -> out like x."""
    n_seq, n_tok, conv_dim = x.shape
    d_conv = w.shape[1]
    _need(x, "x", torch.float32, dev=dev.torch_device)
    _need(conv_state, "conv_state", torch.float32, (n_seq, d_conv - 1, conv_dim), dev.torch_device)
    _need(w, "w", torch.float32, (conv_dim, d_conv), dev.torch_device)
    if out is None:
        out = torch.empty_like(x)
    _need(out, "out", torch.float32, x.shape, dev.torch_device)
    dev.check(dev.lib.pi_gdn_conv1d(dev.h, _vp(x), _vp(conv_state), _vp(w), _vp(out), n_seq, n_tok,
                                    conv_dim, d_conv, dev.stream()))
    return out


def gdn_rmsnorm_gated(dev: Device, o, z, w, eps: float):
    """In place on o [..., n_v_heads, v_hd]: o * rsqrt(mean(o^2) + eps) * w * silu(z)."""
    hv, dv = o.shape[-2:]
    _need(o, "o", torch.float32, dev=dev.torch_device)
    _need(z, "z", torch.float32, o.shape, dev.torch_device)
    _need(w, "w", torch.float32, (dv,), dev.torch_device)
    rows = o.numel() // (hv * dv)
    dev.check(dev.lib.pi_gdn_rmsnorm_gated(dev.h, _vp(o), _vp(z), _vp(w), rows, hv, dv, float(eps),
                                           dev.stream()))
    return o


def attn_prologue(dev: Device, q, k, v, pool: KvPool, page_table, start_pos, q_norm_w=None,
                  k_norm_w=None, eps: float = 1e-6, rope_dim: int = 0, rope_base: float = 10000.0,
                  sections: Optional[Sequence[int]] = None):
    """Norm + RoPE + append for q [n_seq, n_tok, Hq, D], k/v [n_seq, n_tok, Hkv, D]
    (f32; q and k rewritten in place, k and v appended at start_pos[s] + t)."""
    n_seq, n_tok, hq, dh = q.shape
    _need(q, "q", torch.float32, dev=dev.torch_device)
    _need(k, "k", torch.float32, (n_seq, n_tok, pool.n_kv_heads, pool.head_dim), dev.torch_device)
    _need(v, "v", torch.float32, k.shape, dev.torch_device)
    if dh != pool.head_dim:
        raise InvalidArg(f"q head_dim {dh} != pool head_dim {pool.head_dim}")
    _need(page_table, "page_table", torch.int32, dev=dev.torch_device)
    _need(start_pos, "start_pos", torch.int32, (n_seq,), dev.torch_device)
    for name, w in (("q_norm_w", q_norm_w), ("k_norm_w", k_norm_w)):
        if w is not None:
            _need(w, name, torch.float32, (dh,), dev.torch_device)
    sec = None if sections is None else (ctypes.c_int32 * 4)(*[int(s) for s in sections])
    dev.check(dev.lib.pi_attn_prologue(dev.h, _vp(q), _vp(k), _vp(v), _vp(q_norm_w), _vp(k_norm_w),
                                       float(eps), int(rope_dim), float(rope_base), sec, pool.p,
                                       _vp(page_table), page_table.shape[1], _vp(start_pos), n_seq,
                                       n_tok, hq, dev.stream()))
    return q, k


# ---- rotary plans and the 4-bit cache ------------------------------------------------------


def rope_freqs(rope_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
               orig_ctx: float = 4096, params: Optional[Sequence[float]] = None):
    """Host only: (rope_dim / 2 rotary frequencies in float64, the factor of cos and sin).  `params`
    are yarn's (fast, slow) turns, by default (32, 1), or bands' (low, high) turns, by default (1, 4)."""
    if scaling not in ROPE_SCALINGS:
        raise InvalidArg(f"scaling: {scaling!r} (one of {', '.join(ROPE_SCALINGS)})")
    p = [] if scaling == "none" else [float(factor)]
    if scaling in ("yarn", "bands"):
        two = (32.0, 1.0) if scaling == "yarn" else (1.0, 4.0)
        p += [float(orig_ctx), *(float(x) for x in (two if params is None else params))]
    elif params is not None:
        raise InvalidArg(f"params: scaling {scaling!r} takes none")
    lib = _abi.load()
    f = np.zeros(max(int(rope_dim) // 2, 1), np.float64)
    m = ctypes.c_double()
    rc = lib.pi_rope_scaled_freqs(int(rope_dim), float(base), ROPE_SCALINGS[scaling],
                                  (ctypes.c_double * len(p))(*p) if p else None, len(p), f.ctypes.data,
                                  ctypes.addressof(m))
    if rc != 0:
        raise _ERRORS.get(rc, PiError)(lib.pi_last_error(None).decode())
    return f, m.value


class RopePlan:
    """Rotary frequencies on the device, for rope_apply and Q4Pool.append.  layout "halves" pairs channels
    (i, i + rope_dim / 2), "pairs" (2i, 2i + 1); scaling and its arguments as rope_freqs, or the
    frequencies themselves (`freqs`, rope_dim / 2 values, and `mscale`)."""

    def __init__(self, dev: Device, rope_dim: int, base: float = 10000.0, layout: str = "halves",
                 scaling: str = "none", factor: float = 1.0, orig_ctx: float = 4096,
                 params: Optional[Sequence[float]] = None, freqs=None, mscale: Optional[float] = None):
        self.p = None
        self.dev, self.rope_dim, self.layout = dev, int(rope_dim), layout
        if layout not in ROPE_LAYOUTS:
            raise InvalidArg(f"layout: {layout!r} (one of {', '.join(ROPE_LAYOUTS)})")
        if freqs is None:
            f, m = rope_freqs(rope_dim, base, scaling, factor, orig_ctx, params)
        else:
            f, m = np.ascontiguousarray(freqs, np.float64).reshape(-1), 1.0
            if f.size != self.rope_dim // 2:
                raise InvalidArg(f"freqs: expected {self.rope_dim // 2} values, got {f.size}")
        self.freqs, self.mscale = f, m if mscale is None else float(mscale)
        p = ctypes.c_void_p()
        dev.check(dev.lib.pi_rope_plan_create(dev.h, self.rope_dim, ROPE_LAYOUTS[layout], f.ctypes.data,
                                              self.mscale, ctypes.byref(p)))
        self.p = p

    def close(self):
        if self.p:
            self.dev.lib.pi_rope_plan_destroy(self.p)
            self.p = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _rows(t: torch.Tensor, name: str, dtype, shape, dev):
    """A tensor of head rows [n, heads, D] at any strides of its first two dimensions: its address and them."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == dev:
        st, sh, sd = t.stride()
        if sd == 1 or shape[2] <= 1:
            return t.data_ptr(), st, sh
        raise InvalidArg(f"{name}: the last dimension must be contiguous")
    if not isinstance(t, torch.Tensor):
        raise InvalidArg(f"{name}: expected a torch.Tensor")
    if t.device != dev:
        raise InvalidArg(f"{name}: on {t.device}, expected {dev}")
    if t.dtype != dtype:
        raise InvalidArg(f"{name}: dtype {t.dtype}, expected {dtype}")
    raise InvalidArg(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")


def _new_rows(t: torch.Tensor):
    """A new contiguous tensor like t, and what _rows would give for it."""
    t = torch.empty_like(t, memory_format=torch.contiguous_format)
    st, sh, _ = t.stride()
    return t, (t.data_ptr(), st, sh)


def _table(t: torch.Tensor, name: str, dtype, shape, dev):
    """A contiguous tensor's address (None: None)."""
    if t is None:
        return None
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == dev and t.is_contiguous()):
        _need(t, name, dtype, shape, dev)
    return t.data_ptr()


def _pages(page_table, n_seq, dev):
    """The page table's address and columns."""
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2:
        raise InvalidArg("page_table: expected a torch.Tensor [n_seq, max_pages]")
    rows, cols = page_table.shape
    if rows < n_seq:
        raise InvalidArg(f"page_table: shape {(rows, cols)}")
    return _table(page_table, "page_table", torch.int32, (rows, cols), dev), cols


def _float_rows(t, name):
    """The dtype code of a tensor of head rows."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise InvalidArg(f"{name}: expected a torch.Tensor [n, heads, D]")
    code = _DTYPE_CODE.get(t.dtype)
    if code is None:
        raise Unsupported(f"{name}: dtype {t.dtype} (f32, f16 or bf16)")
    return code


def rope_apply(dev: Device, plan: RopePlan, q: torch.Tensor, k: Optional[torch.Tensor], pos: torch.Tensor,
               q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None):
    """q [n, Hq, D] and k [n, Hkv, D] (f32 / f16 / bf16, D contiguous, any other strides) rotated at
    positions pos int32 [n], into q_out and k_out: new tensors (contiguous) by default, or q and k
    themselves for a rotation in place.  Returns (q_out, k_out)."""
    code, td, dt, shape = _float_rows(q, "q"), dev.torch_device, q.dtype, q.shape
    n, hq, d = shape
    if not plan.p:
        raise InvalidArg("plan: closed")
    qp = _rows(q, "q", dt, shape, td)
    if q_out is None:
        q_out, qo = _new_rows(q)
    else:
        qo = _rows(q_out, "q_out", dt, shape, td)
    kp = ko = (None, 0, 0)
    hkv = 0
    if k is not None:
        _float_rows(k, "k")
        hkv = k.shape[1]
        shape = (n, hkv, d)
        kp = _rows(k, "k", dt, shape, td)
        if k_out is None:
            k_out, ko = _new_rows(k)
        else:
            ko = _rows(k_out, "k_out", dt, shape, td)
    rc = dev.lib.pi_rope_apply(dev.h, plan.p, code, n, d, _table(pos, "pos", torch.int32, (n,), td), *qp, hq, *qo, *kp, hkv,
                               *ko, dev.stream())
    if rc:
        dev.check(rc)
    return q_out, k_out


class Q4Pool:
    """Paged KV cache held in 4 bits (include/pi_attn.h): groups of 32 channels with an f16 scale, 4.5 bits
    a value; 16-token pages addressed by the caller's page table, head_dim 64, 128 or 256."""

    def __init__(self, dev: Device, n_pages: int, n_kv_heads: int, head_dim: int,
                 page_tokens: int = PAGE_TOKENS):
        self.p = None
        self.dev = dev
        self._ws_bytes = {}
        self.n_pages, self.n_kv_heads, self.head_dim = n_pages, n_kv_heads, head_dim
        p = ctypes.c_void_p()
        dev.check(dev.lib.pi_q4_pool_create(dev.h, n_pages, page_tokens, n_kv_heads, head_dim,
                                            ctypes.byref(p)))
        self.p = p

    @property
    def nbytes(self) -> int:
        return int(self.dev.lib.pi_q4_pool_bytes(self.p))

    def close(self):
        if self.p:
            self.dev.lib.pi_q4_pool_destroy(self.p)
            self.p = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def append(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, start_pos: torch.Tensor,
               tok_start: Optional[torch.Tensor] = None, plan: Optional[RopePlan] = None,
               q: Optional[torch.Tensor] = None, q_norm_w: Optional[torch.Tensor] = None,
               k_norm_w: Optional[torch.Tensor] = None, eps: float = 1e-6,
               q_out: Optional[torch.Tensor] = None, values: bool = False):
        """Appends k, v [n, Hkv, D] (f32 / f16 / bf16, D contiguous, any other strides): sequence s's rows
        tok_start[s] .. tok_start[s + 1] - 1 (int32 [n_seq + 1]; None: one row a sequence) go to positions
        start_pos[s] ... of page_table's row s, k normed by k_norm_w and rotated by plan on the way.  With q
        [n, Hq, D], returns it normed and rotated (q_out: another tensor than q, a new one by default);
        with `values`, (q_out, k, v) with the f16 [n, Hkv, D] values that the cache now holds (rows of no
        sequence stay uninitialised)."""
        d, td = self.dev, self.dev.torch_device
        if plan is not None and not plan.p:
            raise InvalidArg("plan: closed")  # (a null plan is no rotation)
        code = _float_rows(k, "k")
        dt, n, dh = k.dtype, k.shape[0], self.head_dim
        shape = (n, self.n_kv_heads, dh)
        kp = _rows(k, "k", dt, shape, td)
        vp = _rows(v, "v", dt, shape, td)
        n_seq = start_pos.shape[0] if isinstance(start_pos, torch.Tensor) and start_pos.dim() == 1 else -1
        pt, cols = _pages(page_table, n_seq, td)
        sp = _table(start_pos, "start_pos", torch.int32, (n_seq,), td)
        ts = _table(tok_start, "tok_start", torch.int32, (n_seq + 1,), td)
        qp = qo = (None, 0, 0)
        hq = 0
        if q is not None:
            _float_rows(q, "q")
            hq = q.shape[1]
            qp = _rows(q, "q", dt, (n, hq, dh), td)
            if q_out is None:
                q_out, qo = _new_rows(q)
            else:
                qo = _rows(q_out, "q_out", dt, (n, hq, dh), td)
        qw = _table(q_norm_w, "q_norm_w", torch.float32, (dh,), td)
        kw = _table(k_norm_w, "k_norm_w", torch.float32, (dh,), td)
        k_val = torch.empty(shape, dtype=torch.float16, device=td) if values else None
        v_val = torch.empty(shape, dtype=torch.float16, device=td) if values else None
        rc = d.lib.pi_q4_append(d.h, self.p, None if plan is None else plan.p, code, n, ts, sp, n_seq, pt, cols, *qp, hq, *qo,
                                *kp, *vp, qw, kw, float(eps), _vp(k_val), _vp(v_val), d.stream())
        if rc:
            d.check(rc)
        return (q_out, k_val, v_val) if values else q_out

    def _record_shapes(self, n):
        hk, d = self.n_kv_heads, self.head_dim
        return ((torch.uint8, (n, hk, d // 2)), (torch.float16, (n, hk, d // 32))) * 2

    def read(self, page_table: torch.Tensor, seq: int, start: int, n_tok: int):
        """(k_codes, k_scales, v_codes, v_scales) of positions start .. start + n_tok - 1 of sequence seq:
        uint8 [n_tok, Hkv, D / 2], even channel in the low bits, and f16 [n_tok, Hkv, D / 32]."""
        d = self.dev
        _need(page_table, "page_table", torch.int32, dev=d.torch_device)
        if page_table.dim() != 2 or not 0 <= seq < page_table.shape[0]:
            raise InvalidArg(f"seq {seq} of page_table {tuple(page_table.shape)}")
        out = [torch.empty(s, dtype=t, device=d.torch_device) for t, s in self._record_shapes(max(int(n_tok), 0))]
        d.check(d.lib.pi_q4_read(d.h, self.p, page_table.data_ptr(), page_table.shape[1], int(seq), int(start),
                                 int(n_tok), *(t.data_ptr() for t in out), d.stream()))
        return tuple(out)

    def write(self, page_table: torch.Tensor, seq: int, start: int, k_codes: torch.Tensor,
              k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor):
        """Puts records that `read` gave back into the pages."""
        d = self.dev
        _need(page_table, "page_table", torch.int32, dev=d.torch_device)
        if page_table.dim() != 2 or not 0 <= seq < page_table.shape[0]:
            raise InvalidArg(f"seq {seq} of page_table {tuple(page_table.shape)}")
        n = k_codes.shape[0] if isinstance(k_codes, torch.Tensor) and k_codes.dim() else 0
        args = (k_codes, k_scales, v_codes, v_scales)
        for name, t, (dt, shp) in zip(("k_codes", "k_scales", "v_codes", "v_scales"), args, self._record_shapes(n)):
            _need(t, name, dt, shp, d.torch_device)
        d.check(d.lib.pi_q4_write(d.h, self.p, page_table.data_ptr(), page_table.shape[1], int(seq), int(start), n,
                                  *(t.data_ptr() for t in args), d.stream()))


def _q4_attn(entry, dev, q, pool, page_table, n_seq, ts, pos, max_tok, max_ctx, gqa_mode, scale, gate, out, ws):
    code, td, dt, shape = _float_rows(q, "q"), dev.torch_device, q.dtype, q.shape
    n, hq, dh = shape
    qp = _table(q, "q", dt, shape, td)
    if dh != pool.head_dim:
        raise InvalidArg(f"q head_dim {dh} != pool head_dim {pool.head_dim}")
    pt, max_pages = _pages(page_table, n_seq, td)
    gp = _table(gate, "gate", dt, shape, td)
    if out is None:
        out = torch.empty_like(q)
    op = _table(out, "out", dt, shape, td)
    max_ctx = 0 if max_ctx is None else int(max_ctx)
    key = (code, n, n_seq, max_tok, max_pages, max_ctx, hq, gqa_mode)
    need = pool._ws_bytes.get(key)  # a function of the sizes alone
    if need is None:
        size = ctypes.c_size_t()
        dev.check(dev.lib.pi_q4_attn_ws_bytes(dev.h, pool.p, *key, ctypes.byref(size)))
        if len(pool._ws_bytes) >= 4096:
            pool._ws_bytes.clear()
        need = pool._ws_bytes[key] = size.value
    wp, wn = None, 0
    if ws is not None:
        if not isinstance(ws, torch.Tensor) or ws.device != td or not ws.is_contiguous():
            raise InvalidArg("ws: expected a contiguous torch.Tensor on the device")
        wp, wn = ws.data_ptr(), ws.numel() * ws.element_size()
    elif need:  # torch's allocator keeps it with the stream, and with the graph under capture
        ws = torch.empty(need, dtype=torch.uint8, device=td)
        wp, wn = ws.data_ptr(), need
    if scale is None:
        scale = 1.0 / math.sqrt(dh)
    if ts is None:
        rc = entry(dev.h, pool.p, qp, code, pt, max_pages, max_ctx, pos, n, hq, gqa_mode, scale, gp, op, wp, wn, dev.stream())
    else:
        rc = entry(dev.h, pool.p, qp, code, n, ts, pos, n_seq, max_tok, pt, max_pages, max_ctx, hq, gqa_mode, scale, gp, op, wp,
                   wn, dev.stream())
    if rc:
        dev.check(rc)
    return out


def q4_attn_decode(dev: Device, q: torch.Tensor, pool: Q4Pool, page_table: torch.Tensor, ctx_len: torch.Tensor,
                   gqa_mode: int = MODULO, scale: Optional[float] = None, gate: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None, max_ctx: Optional[int] = None,
                   ws: Optional[torch.Tensor] = None):
    """q [B, Hq, D] (f32 / f16 / bf16) -> out like q, over each sequence's ctx_len[b] tokens of the 4-bit cache.
    max_ctx: a bound of ctx_len (default: the table's row).  ws: a workspace of the caller's; by default
    the call takes one from torch's allocator."""
    b = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() else 0
    if ctx_len is None:
        raise InvalidArg("ctx_len: expected a torch.Tensor")
    cl = _table(ctx_len, "ctx_len", torch.int32, (b,), dev.torch_device)
    return _q4_attn(dev.lib.pi_q4_attn_decode, dev, q, pool, page_table, b, None, cl, 1, max_ctx, gqa_mode, scale,
                    gate, out, ws)


def q4_attn_prefill(dev: Device, q: torch.Tensor, pool: Q4Pool, page_table: torch.Tensor, start_pos: torch.Tensor,
                    tok_start: torch.Tensor, max_tok: Optional[int] = None, gqa_mode: int = MODULO,
                    scale: Optional[float] = None, gate: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, max_ctx: Optional[int] = None,
                    ws: Optional[torch.Tensor] = None):
    """A chunk of tokens a sequence, causal: q [n, Hq, D], sequence s's rows tok_start[s] .. tok_start[s + 1] - 1
    at positions start_pos[s] ... (their keys appended first) -> out like q.  max_tok: no sequence has more
    rows (default: n; a close bound launches fewer workgroups).  Rows of no sequence are left as they were in `out`."""
    n_seq = start_pos.shape[0] if isinstance(start_pos, torch.Tensor) and start_pos.dim() == 1 else -1
    n = q.shape[0] if isinstance(q, torch.Tensor) and q.dim() else 0
    if start_pos is None or tok_start is None:
        raise InvalidArg("start_pos and tok_start: expected torch.Tensors")
    sp = _table(start_pos, "start_pos", torch.int32, (n_seq,), dev.torch_device)
    ts = _table(tok_start, "tok_start", torch.int32, (n_seq + 1,), dev.torch_device)
    return _q4_attn(dev.lib.pi_q4_attn_prefill, dev, q, pool, page_table, n_seq, ts, sp,
                    n if max_tok is None else int(max_tok), max_ctx, gqa_mode, scale, gate, out, ws)
