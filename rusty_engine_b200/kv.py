"""The paged 8-bit KV cache next to the MoE layer, and the operators that serve a block with it.

* ``extend_tables`` / ``KVBatch``  -- block tables and slot maps, built on the GPU from lengths
* ``Rope``                         -- rotary positions (src/infer.rs:90-145), both layouts, part of
  the head, scaled for long contexts
* ``KVCache.append`` / ``read``    -- keys and values into 8-bit codes with a scale per block of
  tokens and head (rope of q and k with it), and back
* ``KVCache.attend``               -- attention over the cache (src/forward.rs:218-283) for prompts,
  prompt chunks and single tokens, any mix of them in one call

One step of a server:  ``step = batch.extend(new_lens, total)``, then per block of the model
``q = cache.append(k, v, step.slots, rope=rope, positions=step.positions, q=q)`` and
``ctx = cache.attend(q, batch.table, batch.lens, step.cu)``; ``batch.release(done)`` when requests
end.  Calls are stream-ordered on the current stream (or ``stream=``) and wait for nothing, so a
step can be captured in a CUDA graph; lengths live on the GPU only.  Shape and type errors raise
``EngineError``; what only the device can see (a slot out of range, a key that is not finite) is
kept in the handle's status word, which ``check()`` reads and raises.  Tensors are float32,
float16 or bfloat16 CUDA tensors [tokens, heads, head_dim] whose last dimension is contiguous.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import enum
import math
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np

from . import _lib
from .moe import EngineError, _call, _require_cuda, _stream, torch

_binding = None


def _ops():
    """The native entry for torch tensors (binding/kv_ops.cpp); raises if it was not built."""
    global _binding
    if _binding is None:
        import importlib.util
        import os

        _lib.load()
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_kv_ops.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with `python -m rusty_engine_b200.build`")
        spec = importlib.util.spec_from_file_location("_kv_ops", path)
        m = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(m)
        m.setup(EngineError, _call)
        _binding = m
    return _binding


@contextlib.contextmanager
def _on(stream, *tensors):
    """Calls made here run on `stream` and allocate their outputs there; the tensors' memory is kept
    from being reused before the stream is done with it."""
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    with torch.cuda.stream(stream):
        yield


class RopeLayout(enum.IntEnum):
    Interleaved = 0  # pairs (x[2i], x[2i + 1])
    Half = 1         # pairs (x[i], x[i + rot_dim / 2]), rusty-engine's NeoX rotate-half


class RopeScaling(enum.IntEnum):
    NoScaling = 0
    Linear = 1
    Yarn = 2


class CacheCode(enum.IntEnum):
    Int8 = 0
    E4M3 = 1


@dataclass(frozen=True)
class RopeConfig:
    """rmoe_rope_desc: angle of pair i at position p is p * base^(-2i / rot_dim), scaled."""

    rot_dim: int
    base: float = 1e6
    layout: RopeLayout = RopeLayout.Half
    scaling: RopeScaling = RopeScaling.NoScaling
    factor: float = 1.0
    orig_ctx: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    mscale: float = 0.0  # factor of cos and sin; 0: the scaling's own
    freq_factors: Optional[Sequence[float]] = None


def _int32(x, what, like, n):
    if x.dtype != torch.int32 or not x.is_contiguous() or x.device != like.device or x.numel() != n:
        raise EngineError(f"{what}: {n} contiguous int32 on {like.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x.data_ptr()


class Rope:
    """Rotary positions 0 .. max_pos - 1 (rmoe_rope_create): the table of cosines and sines."""

    def __init__(self, cfg: RopeConfig, max_pos: int, device: Optional[int] = None):
        _require_cuda()
        self.cfg, self.max_pos = cfg, max_pos
        self.device = torch.cuda.current_device() if device is None else device
        d = _lib.RopeDesc()
        d.rot_dim, d.layout, d.scaling, d.max_pos = cfg.rot_dim, int(cfg.layout), int(cfg.scaling), max_pos
        d.base, d.factor, d.beta_fast, d.beta_slow, d.mscale = cfg.base, cfg.factor, cfg.beta_fast, cfg.beta_slow, cfg.mscale
        d.orig_ctx, d.device = cfg.orig_ctx, self.device
        if cfg.freq_factors is not None:
            ff = np.ascontiguousarray(cfg.freq_factors, dtype=np.float32)
            if ff.shape != (cfg.rot_dim // 2,):
                raise EngineError(f"freq_factors: {ff.shape}, expected ({cfg.rot_dim // 2},)")
            d.freq_factors = ff.ctypes.data
        h = C.c_void_p()
        L = _lib.load()
        _call(L.rmoe_rope_create(C.byref(d), C.byref(h)))
        self._h, self._p, self._apply = h, h.value, _ops().rope_apply

    def apply(self, q, positions, k=None, *, out=None, k_out=None, inverse: bool = False, stream=None):
        """q (and k) [tokens, heads, head_dim] turned by positions [tokens] (int32); returns the
        turned q, or (q, k) when k is given.  `out=q` turns in place.  inverse: turns back."""
        if stream is not None:
            with _on(stream, q, positions, k, out, k_out):
                return self.apply(q, positions, k, out=out, k_out=k_out, inverse=inverse)
        return self._apply(self._open(), self.device, q, positions, k, out, k_out, inverse)

    def _open(self):
        if not self._p:  # 0 would be taken for "no rope"
            raise EngineError("the rope is closed")
        return self._p

    def check(self):
        """Raises if a call so far met a position outside the table (synchronises)."""
        _call(_lib.load().rmoe_rope_status(self._h))

    def close(self):
        if getattr(self, "_h", None) is not None and self._h.value:
            _lib.load().rmoe_rope_destroy(self._h)
            self._h, self._p = C.c_void_p(), 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


@dataclass
class KVStep:
    """What extend made for one step: cu [R + 1], positions and slots [tokens], and the lengths
    [R] and free-stack height [1] afterwards (all int32)."""

    cu: "torch.Tensor"
    positions: "torch.Tensor"
    slots: "torch.Tensor"
    lens: "torch.Tensor"
    n_free: "torch.Tensor"


def extend_tables(table, lens, new_lens, free, n_free, total: int, block_size: int, *, stream=None) -> KVStep:
    """rmoe_kv_extend: request r, holding lens[r] tokens, adds new_lens[r]; `total` is the batch's
    token count (slots past the requests' tokens are -1).  New blocks come off the stack
    free[:n_free] in request order and are written into `table` [R, max_blocks]; a request that
    cannot have all its blocks gets none: its slots are -1 and its length stays."""
    if stream is not None:
        with _on(stream, table, lens, new_lens, free, n_free):
            return extend_tables(table, lens, new_lens, free, n_free, total, block_size)
    return KVStep(*_ops().extend(table, lens, new_lens, free, n_free, total, block_size))


class KVBatch:
    """The requests in flight: table [R, max_blocks], lens [R] and the free-block stack, on the GPU."""

    def __init__(self, max_requests: int, max_blocks: int, n_blocks: int, block_size: int, device=None):
        _require_cuda()
        dev = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        self.block_size = block_size
        self.table = torch.full((max_requests, max_blocks), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.free = torch.arange(n_blocks - 1, -1, -1, dtype=torch.int32, device=dev)
        self.n_free = torch.full((1,), n_blocks, dtype=torch.int32, device=dev)

    def extend(self, new_lens, total: int, *, stream=None) -> KVStep:
        """extend_tables on this batch; lens and the stack move on (in place, so that a step captured in
        a CUDA graph is the next step at every replay)."""
        if stream is not None:
            with _on(stream, self.table, self.lens, new_lens, self.free, self.n_free):
                return self.extend(new_lens, total)
        step = extend_tables(self.table, self.lens, new_lens, self.free, self.n_free, total, self.block_size)
        torch._foreach_copy_([self.lens, self.n_free], [step.lens, step.n_free])
        return step

    def release(self, done, *, stream=None):
        """rmoe_kv_release: requests with done[r] != 0 (int32 [R]) give their blocks back."""
        if stream is not None:
            with _on(stream, self.table, self.lens, self.free, done, self.n_free):
                return self.release(done)
        R, mb = self.table.shape
        with torch.cuda.device(self.table.device):
            out = torch.empty_like(self.n_free)
            args = _lib.KV_RELEASE_ARGS.pack(self.table.data_ptr(), self.lens.data_ptr(), self.free.data_ptr(),
                                             _int32(done, "done", self.table, R), self.n_free.data_ptr(), out.data_ptr(),
                                             R, mb, self.block_size, self.free.numel())
            _call(_lib.load().rmoe_kv_release(args, _stream()))
        self.n_free.copy_(out)


class KVCache:
    """One layer's keys and values: codes [n_blocks, n_kv_heads, block_size, head_dim] in 8 bits and
    one f32 scale per block and head (rmoe_kv_create)."""

    def __init__(self, n_blocks: int, block_size: int, n_kv_heads: int, head_dim: int,
                 code: CacheCode = CacheCode.Int8, device: Optional[int] = None):
        _require_cuda()
        dev = torch.device("cuda", torch.cuda.current_device() if device is None else device)
        dt = torch.int8 if code == CacheCode.Int8 else torch.float8_e4m3fn
        if min(n_blocks, block_size, n_kv_heads, head_dim) < 1:
            raise EngineError(f"cache of {n_blocks} blocks x {n_kv_heads} heads x {block_size} x {head_dim}")
        z = lambda: torch.zeros((n_blocks, n_kv_heads, block_size, head_dim), dtype=torch.uint8, device=dev).view(dt)  # noqa: E731
        s = lambda: torch.zeros((n_blocks, n_kv_heads), dtype=torch.float32, device=dev)  # noqa: E731
        self._bind(z(), z(), s(), s())

    @classmethod
    def from_buffers(cls, k, v, k_scale, v_scale) -> "KVCache":
        """A cache over the caller's tensors: int8 or float8_e4m3fn codes and f32 scales."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, ks, vs):
        codes = {torch.int8: CacheCode.Int8, torch.float8_e4m3fn: CacheCode.E4M3}
        if k.dtype not in codes or k.dim() != 4 or not k.is_cuda:
            raise EngineError(f"cache codes: int8 or float8_e4m3fn [blocks, heads, block, dim] on CUDA, got {k.dtype} "
                              f"{tuple(k.shape)} on {k.device}")
        for name, t, shape, dt in (("v", v, k.shape, k.dtype), ("k_scale", ks, k.shape[:2], torch.float32),
                                   ("v_scale", vs, k.shape[:2], torch.float32)):
            if t.shape != shape or t.dtype != dt or t.device != k.device:
                raise EngineError(f"{name}: {t.dtype} {tuple(t.shape)} on {t.device} beside k {k.dtype} {tuple(k.shape)}")
        for name, t in (("k", k), ("v", v), ("k_scale", ks), ("v_scale", vs)):
            if not t.is_contiguous():
                raise EngineError(f"{name}: cache memory must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = k, v, ks, vs
        self.code, self.device = codes[k.dtype], k.device.index
        self.n_blocks, self.n_kv_heads, self.block_size, self.head_dim = k.shape
        d = _lib.KvDesc()
        d.n_blocks, d.block_size, d.n_kv_heads, d.head_dim = self.n_blocks, self.block_size, self.n_kv_heads, self.head_dim
        d.code, d.device = int(self.code), self.device
        d.k, d.v, d.k_scale, d.v_scale = k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr()
        h = C.c_void_p()
        L = _lib.load()
        _call(L.rmoe_kv_create(C.byref(d), C.byref(h)))
        ops = _ops()
        self._h, self._p, self._append, self._read, self._attend = h, h.value, ops.append, ops.read, ops.attend
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._like = {dt: torch.empty(0, dtype=dt, device=k.device) for dt in (torch.float32, torch.float16, torch.bfloat16)}

    def append(self, k, v, slots, *, rope: Optional[Rope] = None, positions=None, q=None, q_out=None, stream=None):
        """Writes k and v [tokens, n_kv_heads, head_dim] at `slots` (int32, -1 skips); the tokens of one
        block in one run of consecutive slots, as extend gives them.  With a rope, k is turned by
        `positions` first, and so is q where given; returns the turned q."""
        if stream is not None:
            with _on(stream, k, v, slots, positions, q, q_out):
                return self.append(k, v, slots, rope=rope, positions=positions, q=q, q_out=q_out)
        return self._append(self._open(), self.device, self.n_kv_heads, self.head_dim, k, v, slots,
                            0 if rope is None else rope._open(), positions, q, q_out)

    def read(self, slots, dtype=None, *, stream=None):
        """(k, v) of cached tokens [slots, n_kv_heads, head_dim], code * scale, as `dtype` (float32)."""
        like = self._like.get(torch.float32 if dtype is None else dtype)
        if like is None:
            raise EngineError(f"read as {dtype}: float32, float16 or bfloat16")
        if stream is not None:
            with _on(stream, slots):
                return self.read(slots, dtype)
        return self._read(self._open(), self.k, slots, like)

    def attend(self, q, table, lens, cu, *, scale: Optional[float] = None, window: int = 0, max_new: Optional[int] = None,
               out=None, return_lse: bool = False, stream=None):
        """Attention of q [tokens, q heads, head_dim]: request r, with lens[r] cached tokens in
        blocks table[r], has the queries cu[r] .. cu[r + 1) at its last positions.  Causal; with a
        window, each query sees that many keys at most.  scale: 1 / sqrt(head_dim) by default.
        max_new: an upper bound of any request's new tokens, where known (chooses kernels only).
        Only reads the cache: calls on different streams may overlap (each stream has a workspace of
        its own; of graphs captured on the same stream one may run at a time).
        Returns out (as q), or (out, lse [tokens, q heads] f32)."""
        if stream is not None:
            with _on(stream, q, table, lens, cu, out):
                return self.attend(q, table, lens, cu, scale=scale, window=window, max_new=max_new, out=out,
                                   return_lse=return_lse)
        return self._attend(self._open(), self.device, self.head_dim, q, table, lens, cu, self._scale if scale is None else scale,
                            window, max_new or 0, out, return_lse)

    def _open(self):
        if not self._p:
            raise EngineError("the cache is closed")
        return self._p

    def check(self):
        """Raises if a call so far met a device error (synchronises and clears it)."""
        _call(_lib.load().rmoe_kv_status(self._h))

    def close(self):
        if getattr(self, "_h", None) is not None and self._h.value:
            _lib.load().rmoe_kv_destroy(self._h)
            self._h, self._p = C.c_void_p(), 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
