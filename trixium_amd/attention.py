"""Attention over KV caches: a sliding window and sinks over a ring (host side of trx_attn_window), drafts behind
a prefix that they share (trx_attn_shared), a cache that keeps the rows that got most of the attention
(trx_attn_mass, trx_kv_evict).

`KVRing` holds the K and V rows of one layer on the GPU in the decoder's layout (fp16, position p in
slot p below `pin`, else in a ring of the most recent positions; firmware/hybrid.c:156-181) and
attends the next positions over them: any number at once (a prompt's chunk) or one (decoding).
Queries, keys, values and outputs are numpy arrays, copied to the GPU and back by each call, which waits for
it; a program whose data is on the GPU calls the C entry points with its own pointers, stream and workspace.
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


def _int32s(**values):
    for name, v in values.items():                 # (ctypes would take them modulo 2^32)
        if not -2**31 <= v < 2**31:
            raise ValueError(f"{name} {v} is not an int32")
    return values


def _strides(n_head, n_kv, hd):
    return dict(q_stride=n_head * hd, kv_stride=n_kv * hd, out_stride=n_head * hd, gate_stride=n_head * hd,
                gate_head_stride=hd)


class _Rows:
    """What the caches below share: the shape's checks, arrays as the kernels take them, a workspace."""

    def __init__(self, n_head, n_kv_head, head_dim, kind):
        if kind not in _DTYPES:
            raise ValueError(f"kind {kind} is not KIND_F32 or KIND_F16")
        self.n_head, self.n_kv, self.hd, self.kind = int(n_head), int(n_kv_head), int(head_dim), kind
        self.dtype = _DTYPES[kind]
        self.work = None

    def _workspace(self, name, *args):
        size = ctypes.c_size_t()
        _lib.call(name, ctypes.byref(self.shape), *args, ctypes.byref(size))
        if self.work is None or self.work.nbytes < size.value:
            self.work = _lib.DeviceBuffer(size.value)
        return self.work.ptr

    def _inputs(self, lead, q, k, v, gate):
        q, gate = (None if a is None else np.ascontiguousarray(np.asarray(a, dtype=self.dtype)) for a in (q, gate))
        k, v = (np.ascontiguousarray(np.asarray(a, dtype=np.float16)) for a in (k, v))
        if q.ndim != lead + 2:
            raise ValueError(f"queries of shape {q.shape}")
        rows = q.shape[:lead]
        for name, a, heads in (("queries", q, self.n_head), ("keys", k, self.n_kv), ("values", v, self.n_kv),
                               ("gates", gate, self.n_head)):
            if a is not None and a.shape != (*rows, heads, self.hd):
                raise ValueError(f"{name} of shape {a.shape}, expected {(*rows, heads, self.hd)}")
        return q, k, v, gate


class SharedPrefix(_Rows):
    """Drafts of one prompt (host side of trx_attn_shared): the prompt's K and V rows (fp16 [n_kv_head, rows,
    head_dim], k rotated) once for all, and a tail of up to `tail_slots` rows for each of `batch` drafts. The
    firmware decodes one sequence (firmware/infer.c:2001); drafts are drawn by `sampling.sample`, a row each."""

    def __init__(self, n_head, n_kv_head, head_dim, k, v, batch, tail_slots, scale=None, kind=L.KIND_F32):
        super().__init__(n_head, n_kv_head, head_dim, kind)
        k, v = (np.ascontiguousarray(np.asarray(a, dtype=np.float16)) for a in (k, v))
        if k.ndim != 3 or k.shape[::2] != (self.n_kv, self.hd) or v.shape != k.shape:
            raise ValueError(f"keys of shape {k.shape} and values of shape {v.shape}")
        self._begin(k.shape[1], batch, tail_slots, scale)
        self.kprefix, self.vprefix = (_lib.DeviceBuffer.from_array(a) for a in (k, v))
        _lib.synchronize()

    def _begin(self, prefix, batch, tail_slots, scale):
        self.prefix, self.batch, self.tail_slots = int(prefix), int(batch), int(tail_slots)
        sizes = _int32s(kind=self.kind, n_head=self.n_head, n_kv_head=self.n_kv, head_dim=self.hd, prefix_slots=self.prefix,
                        tail_slots=self.tail_slots, batch=self.batch, **_strides(self.n_head, self.n_kv, self.hd))
        if sizes.pop("batch") < 1:
            raise ValueError(f"{batch} drafts")
        self.shape = _lib.AttnSharedShape(scale=1.0 / math.sqrt(self.hd) if scale is None else scale, **sizes)
        self._workspace("trx_attn_shared_geometry", self.batch, 1, self.prefix)  # refuses a shape before any allocation
        self.lengths = np.zeros(self.batch, np.int32)
        size = 2 * self.batch * self.n_kv * self.tail_slots * self.hd
        self.ktail, self.vtail = _lib.DeviceBuffer(size), _lib.DeviceBuffer(size)
        for t in (self.ktail, self.vtail):
            t.zero()

    def attend(self, q, k, v, gate=None, counts=None):
        """Outputs [batch, n, n_head, head_dim] of each draft's next n rows: q (and gate) [batch, n, n_head, head_dim],
        k and v [batch, n, n_kv_head, head_dim]. counts: how many of its rows a draft takes (all of them; outputs of
        the others are 0). The rows go to the drafts' tails."""
        q, k, v, gate = self._inputs(2, q, k, v, gate)
        if q.shape[0] != self.batch:
            raise ValueError(f"{q.shape[0]} drafts, not {self.batch}")
        n = q.shape[1]
        counts = np.full(self.batch, n) if counts is None else np.asarray(counts)
        if counts.shape != (self.batch,) or counts.dtype.kind not in "iu" or (counts < 0).any() or (counts > n).any():
            raise ValueError(f"counts {counts} of {n} rows")
        if (self.lengths + counts > self.tail_slots).any():
            raise ValueError(f"tails of {(self.lengths + counts).max()} rows in {self.tail_slots} slots")
        if n == 0:
            return np.empty(q.shape, self.dtype)
        work = self._workspace("trx_attn_shared_geometry", self.batch, n, self.prefix)
        qb, kb, vb, lb, cb, out = (_lib.DeviceBuffer.from_array(a) for a in (q, k, v, self.lengths, counts.astype(np.int32),
                                                                          np.zeros_like(q)))
        gb = _lib.DeviceBuffer.from_array(gate) if gate is not None else None
        _lib.call("trx_attn_shared", ctypes.byref(self.shape), self.batch, n, self.prefix, lb.ptr, cb.ptr, qb.ptr, kb.ptr,
                  vb.ptr, self.kprefix.ptr, self.vprefix.ptr, self.ktail.ptr, self.vtail.ptr, gb.ptr if gb else None,
                  out.ptr, work, None)
        _lib.synchronize()
        self.lengths = (self.lengths + counts).astype(np.int32)
        return out.download(self.dtype, q.size).reshape(q.shape)

    def cut(self, lengths):
        """Tails of `lengths` rows (none longer than it is): what was proposed and not taken goes."""
        lengths = np.asarray(lengths)
        if lengths.shape != (self.batch,) or lengths.dtype.kind not in "iu" or (lengths < 0).any() or (lengths > self.lengths).any():
            raise ValueError(f"lengths {lengths} of tails of {self.lengths}")
        self.lengths = lengths.astype(np.int32)

    def rows(self, draft):
        """(K, V) of a draft's tail, fp16 [n_kv_head, rows, head_dim]."""
        size = self.n_kv * self.tail_slots * self.hd
        draft = range(self.batch)[draft]
        return tuple(t.download(np.float16, size, offset=2 * size * draft)
                     .reshape(self.n_kv, self.tail_slots, self.hd)[:, :self.lengths[draft]] for t in (self.ktail, self.vtail))


class KVMass(_Rows):
    """The cache of one layer that adds up the probabilities that each row gets (host side of trx_attn_mass) and keeps
    the rows that got most (trx_kv_evict), where the firmware's ring drops the oldest (firmware/hybrid.c:156-181):
    `slots` rows per kv head, `count` of them held."""

    def __init__(self, n_head, n_kv_head, head_dim, slots, scale=None, kind=L.KIND_F32):
        super().__init__(n_head, n_kv_head, head_dim, kind)
        self.slots = int(slots)
        sizes = _int32s(kind=kind, n_head=self.n_head, n_kv_head=self.n_kv, head_dim=self.hd, slots=self.slots,
                        **_strides(self.n_head, self.n_kv, self.hd))
        self.shape = _lib.AttnMassShape(scale=1.0 / math.sqrt(self.hd) if scale is None else scale, **sizes)
        self._workspace("trx_attn_mass_geometry", 1)           # refuses an unsupported shape before any allocation
        self.reset()
        rows = self.n_kv * self.slots
        self.kcache, self.vcache, self.mass, self.position = (
            _lib.DeviceBuffer(size * rows) for size in (2 * self.hd, 2 * self.hd, 4, 4))
        for b in (self.kcache, self.vcache, self.mass, self.position):
            b.zero()
        _lib.synchronize()

    def reset(self):
        """No rows, position 0 again."""
        self.count = self.next = 0                             # rows held; the next row's position

    def attend(self, q, k, v, gate=None):
        """Outputs [n, n_head, head_dim] of the next n positions: q (and gate) [n, n_head, head_dim], k and v [n,
        n_kv_head, head_dim] (k rotated). The rows go behind those held; all masses grow."""
        q, k, v, gate = self._inputs(1, q, k, v, gate)
        n = q.shape[0]
        if self.count + n > self.slots:
            raise ValueError(f"{self.count} rows and {n} new ones in {self.slots} slots")
        if n == 0:
            return np.empty(q.shape, self.dtype)
        work = self._workspace("trx_attn_mass_geometry", n)
        qb, kb, vb = (_lib.DeviceBuffer.from_array(a) for a in (q, k, v))
        gb, out = _lib.DeviceBuffer.from_array(gate) if gate is not None else None, _lib.DeviceBuffer(q.nbytes)
        _lib.call("trx_attn_mass", ctypes.byref(self.shape), n, self.count, self.next, None, qb.ptr, kb.ptr, vb.ptr,
                  self.kcache.ptr, self.vcache.ptr, self.mass.ptr, self.position.ptr, gb.ptr if gb else None, out.ptr,
                  work, None)
        _lib.synchronize()
        self.count += n
        self.next += n
        return out.download(self.dtype, q.size).reshape(q.shape)

    def evict(self, keep, sinks=4, recent=0):
        """Keeps `keep` rows of each kv head: the first `sinks` positions and the last `recent` before the others,
        then the largest masses. Of more than `keep` rows at such positions (sinks + recent > keep) those in the lowest
        slots stay."""
        _int32s(keep=keep, sinks=sinks, recent=recent)
        work = self._workspace("trx_kv_evict_geometry")
        _lib.call("trx_kv_evict", ctypes.byref(self.shape), self.count, self.next, None, keep, sinks, recent, self.kcache.ptr,
                  self.vcache.ptr, self.mass.ptr, self.position.ptr, work, None)
        _lib.synchronize()
        self.count = min(self.count, int(keep))

    def rows(self):
        """(K, V) of the rows held, fp16 [n_kv_head, count, head_dim]."""
        return tuple(b.download(np.float16, self.n_kv * self.slots * self.hd)
                     .reshape(self.n_kv, self.slots, self.hd)[:, :self.count] for b in (self.kcache, self.vcache))

    def masses(self):
        """float32 [n_kv_head, count]."""
        return self.mass.download(np.float32, self.n_kv * self.slots).reshape(self.n_kv, self.slots)[:, :self.count]

    def positions(self):
        """int32 [n_kv_head, count]: the position of each row held."""
        return self.position.download(np.int32, self.n_kv * self.slots).reshape(self.n_kv, self.slots)[:, :self.count]

    def share(self, batch, tail_slots):
        """Drafts behind a copy of the rows held, made on the GPU."""
        s = SharedPrefix.__new__(SharedPrefix)
        _Rows.__init__(s, self.n_head, self.n_kv, self.hd, self.kind)
        s._begin(self.count, batch, tail_slots, self.shape.scale)
        size = 2 * self.count * self.hd
        s.kprefix, s.vprefix = _lib.DeviceBuffer(self.n_kv * size), _lib.DeviceBuffer(self.n_kv * size)
        for g in range(self.n_kv if size else 0):
            for to, frm in ((s.kprefix, self.kcache), (s.vprefix, self.vcache)):
                _lib.call("trx_memcpy_d2d", to.ptr + g * size, frm.ptr + g * 2 * self.slots * self.hd, size, None)
        _lib.synchronize()
        return s
