"""Attention with a sliding window and sinks over a KV ring (host side of trx_attn_window).

`KVRing` holds the K and V rows of one layer on the GPU in the decoder's layout (fp16, position p in
slot p below `pin`, else in a ring of the most recent positions; firmware/hybrid.c:156-181) and
attends the next positions over them: any number at once (a prompt's chunk) or one (decoding).
Queries, keys, values and outputs are numpy arrays, copied to the GPU and back by each call, which waits for
it; a program whose data is on the GPU calls trx_attn_window with its own pointers, stream and workspace.
"""

import ctypes
import math

import numpy as np

from . import _lib
from . import layout as L

_DTYPES = {L.KIND_F32: np.float32, L.KIND_F16: np.float16}


class KVRing:
    """The ring of one layer: `slots` rows per kv head, the first `pin` positions kept. A query at
    position t sees the positions u <= t with u < sinks or u > t - window (by default every one that
    the ring holds: sinks = pin, window = slots - pin). kind: the type of queries, gates and
    outputs (layout.KIND_F32 or KIND_F16)."""

    def __init__(self, n_head, n_kv_head, head_dim, slots, pin=4, window=None, sinks=None, scale=None,
                 kind=L.KIND_F32):
        if kind not in _DTYPES:
            raise ValueError(f"kind {kind} is not KIND_F32 or KIND_F16")
        self.n_head, self.n_kv, self.hd, self.slots = int(n_head), int(n_kv_head), int(head_dim), int(slots)
        self.dtype = _DTYPES[kind]
        q, kv = self.n_head * self.hd, self.n_kv * self.hd
        shape = dict(
            kind=kind, n_head=self.n_head, n_kv_head=self.n_kv, head_dim=self.hd, slots=self.slots, pin=int(pin),
            window=int(self.slots - pin if window is None else window), sinks=int(pin if sinks is None else sinks),
            q_stride=q, kv_stride=kv, out_stride=q, gate_stride=q, gate_head_stride=self.hd)
        for name, v in shape.items():              # (ctypes would take them modulo 2^32)
            if not -2**31 <= v < 2**31:
                raise ValueError(f"{name} {v} is not an int32")
        self.shape = _lib.AttnWindowShape(scale=1.0 / math.sqrt(self.hd) if scale is None else scale, **shape)
        self.work, self.work_n = None, 0           # the workspace, of calls of up to work_n positions
        self._workspace(1)                         # refuses an unsupported shape before any allocation
        self.position = 0                          # of the next row
        self.kcache = _lib.DeviceBuffer(2 * kv * self.slots)
        self.vcache = _lib.DeviceBuffer(2 * kv * self.slots)
        for c in (self.kcache, self.vcache):
            c.zero()
        _lib.synchronize()

    def _workspace(self, n):
        if n > self.work_n:
            size = ctypes.c_size_t()
            _lib.call("trx_attn_window_geometry", ctypes.byref(self.shape), n, ctypes.byref(size))
            if size.value and (self.work is None or self.work.nbytes < size.value):
                self.work = _lib.DeviceBuffer(size.value)
            self.work_n = n
        return self.work.ptr if self.work else None

    def attend(self, q, k, v, gate=None):
        """Outputs [n, n_head, head_dim] of the next n positions: q (and gate) [n, n_head, head_dim], k
        and v [n, n_kv_head, head_dim] (rounded to fp16, as the ring holds them; k rotated). The rows
        take their slots and the position moves on by n."""
        q = np.ascontiguousarray(np.asarray(q, dtype=self.dtype).reshape(-1, self.n_head, self.hd))
        n = q.shape[0]
        k = np.ascontiguousarray(np.asarray(k, dtype=np.float16).reshape(-1, self.n_kv, self.hd))
        v = np.ascontiguousarray(np.asarray(v, dtype=np.float16).reshape(-1, self.n_kv, self.hd))
        if k.shape[0] != n or v.shape[0] != n:
            raise ValueError(f"{n} queries, {k.shape[0]} keys, {v.shape[0]} values")
        if gate is not None:
            gate = np.ascontiguousarray(np.asarray(gate, dtype=self.dtype).reshape(-1, self.n_head, self.hd))
            if gate.shape[0] != n:
                raise ValueError(f"{n} queries, {gate.shape[0]} gates")
        if n == 0:
            return np.empty((0, self.n_head, self.hd), dtype=self.dtype)
        work = self._workspace(n)
        qb, kb, vb = (_lib.DeviceBuffer.from_array(a) for a in (q, k, v))
        gb = _lib.DeviceBuffer.from_array(gate) if gate is not None else None
        out = _lib.DeviceBuffer(q.nbytes)
        _lib.call("trx_attn_window", ctypes.byref(self.shape), n, self.position, None, qb.ptr, kb.ptr, vb.ptr,
                  self.kcache.ptr, self.vcache.ptr, gb.ptr if gb else None, out.ptr, work, None)
        _lib.synchronize()
        self.position += n
        return out.download(self.dtype, q.size).reshape(q.shape)

    def rows(self):
        """(K, V) as the ring holds them, fp16 [n_kv_head, slots, head_dim]."""
        return tuple(c.download(np.float16, self.n_kv * self.slots * self.hd).reshape(self.n_kv, self.slots, self.hd)
                     for c in (self.kcache, self.vcache))

    def reset(self):
        """Position 0 again (rows of earlier positions are not read any more)."""
        self.position = 0
