"""Attention with a sliding window and sinks over a KV ring (trx_attn_window) against its definition in
64 bits over absolute positions, from single tokens to chunks longer than the window, and what it
refuses.

Tolerance, per output element, from the arithmetic (A = sum of p |v| over the seen keys, S = the largest
sum over dims of scale |q k|, N seen keys): a score is off by S (2^-21 + head_dim 2^-24) (the query's
two planes or fp16 itself, fp32 sums), its exponent by 2^-21 more, which moves a probability and the
total by twice that; the sums add N 2^-24 A; the probabilities' planes 2^-22 A in fp32, half a step
(2^-11 A) in fp16, where those below fp16's steps lose 2^-32 max |v| each, and the result is rounded
by 2^-11 of itself. The gate multiplies by a value of error 2^-21."""

import ctypes

import numpy as np
import pytest

from trixium_amd import _lib, layout as L

F32, F16 = L.KIND_F32, L.KIND_F16
DT = {F32: np.float32, F16: np.float16}


class Case:
    """A ring with its history by absolute position, and what the operator has to give."""

    def __init__(self, heads, kv, hd, slots, pin, window, sinks, kind=F32, seed=0, scale=None):
        self.heads, self.kv, self.hd, self.slots = heads, kv, hd, slots
        self.pin, self.window, self.sinks, self.kind = pin, window, sinks, kind
        self.scale = np.float32(1.0 / np.sqrt(hd) if scale is None else scale)
        self.rng = np.random.default_rng(seed)
        self.K = np.zeros((0, kv, hd), np.float16)
        self.V = np.zeros((0, kv, hd), np.float16)

    def slot(self, p):
        return p if p < self.pin else self.pin + (p - self.pin) % (self.slots - self.pin)

    def rows(self, n, size=1.0):
        r = self.rng
        q = (1.5 * size * r.standard_normal((n, self.heads, self.hd))).astype(DT[self.kind])
        k = r.standard_normal((n, self.kv, self.hd)).astype(np.float16)
        v = r.standard_normal((n, self.kv, self.hd)).astype(np.float16)
        return q, k, v

    def extend(self, n):
        _, k, v = self.rows(n)
        self.K, self.V = np.concatenate([self.K, k]), np.concatenate([self.V, v])

    def ring(self, fill=0.0):
        """The caches after the history; slots without a position hold `fill`."""
        kc = np.full((self.kv, self.slots, self.hd), fill, np.float16)
        vc = kc.copy()
        for p in range(self.K.shape[0]):
            kc[:, self.slot(p)], vc[:, self.slot(p)] = self.K[p], self.V[p]
        return kc, vc

    def expect(self, q, k, v, gate=None):
        """(outputs, tolerances) in 64 bits of the next rows over the history."""
        pos = self.K.shape[0]
        K = np.concatenate([self.K, k]).astype(np.float64)
        V = np.concatenate([self.V, v]).astype(np.float64)
        n, half = q.shape[0], self.kind == F16
        out = np.empty((n, self.heads, self.hd))
        tol = np.empty_like(out)
        for r in range(n):
            t = pos + r
            u = np.arange(t + 1)
            u = u[(u < self.sinks) | (u > t - self.window)]
            for h in range(self.heads):
                g = h // (self.heads // self.kv)
                qd = q[r, h].astype(np.float64)
                s = float(self.scale) * (K[u, g] @ qd)
                S = float(self.scale) * (np.abs(K[u, g]) @ np.abs(qd)).max()
                p = np.exp(s - s.max())
                p /= p.sum()
                A = p @ np.abs(V[u, g])
                o = p @ V[u, g]
                e = A * (2 * (S * (2.0**-21 + self.hd * 2.0**-24) + 2.0**-21) + u.size * 2.0**-24 + 2.0**-22)
                if half:
                    e += A * 2.0**-11 + u.size * 2.0**-32 * np.abs(V[u, g]).max()
                if gate is not None:
                    sg = 1.0 / (1.0 + np.exp(-gate[r, h].astype(np.float64)))
                    o, e = o * sg, e * sg + np.abs(o) * 2.0**-21
                if half:
                    e += np.abs(o) * 2.0**-11 + 2.0**-25
                out[r, h], tol[r, h] = o, e
        return out, tol

    def c_shape(self, **kw):
        q, kv = self.heads * self.hd, self.kv * self.hd
        d = dict(kind=self.kind, n_head=self.heads, n_kv_head=self.kv, head_dim=self.hd, slots=self.slots, pin=self.pin,
                 window=self.window, sinks=self.sinks, q_stride=q, kv_stride=kv, out_stride=q, gate_stride=q,
                 gate_head_stride=self.hd, scale=float(self.scale))
        d.update(kw)
        return _lib.AttnWindowShape(**d)


def _geometry(shape, n):
    size = ctypes.c_size_t()
    _lib.call("trx_attn_window_geometry", ctypes.byref(shape), n, ctypes.byref(size))
    return size.value


def _call(c, q, k, v, kc, vc, gate=None, pos=None, pos_dev=None, stream=None, shape=None):
    """One call on device copies; (out, K ring, V ring) back."""
    B = _lib.DeviceBuffer
    shape = shape or c.c_shape()
    n = k.shape[0]
    bufs = [B.from_array(a) for a in (q, k, v, kc, vc)]
    gb = B.from_array(gate) if gate is not None else None
    out = B.from_array(np.full(n * shape.out_stride, 77, DT[c.kind]))
    work = B(max(_geometry(shape, n), 1))
    pd = B.from_array(np.array([pos_dev], np.int32)) if pos_dev is not None else None
    _lib.synchronize()
    _lib.call("trx_attn_window", ctypes.byref(shape), n, c.K.shape[0] if pos is None else pos, pd.ptr if pd else None,
              *(b.ptr for b in bufs), gb.ptr if gb else None, out.ptr, work.ptr, stream)
    _lib.synchronize(stream)
    shp = (c.kv, c.slots, c.hd)
    return (out.download(DT[c.kind], n * shape.out_stride).reshape(n, shape.out_stride),
            bufs[3].download(np.float16, kc.size).reshape(shp), bufs[4].download(np.float16, vc.size).reshape(shp))


def _check(c, n, fill=0.0, gated=False):
    q, k, v = c.rows(n)
    gate = c.rng.standard_normal(q.shape).astype(DT[c.kind]) if gated else None
    kc, vc = c.ring(fill)
    out, kc1, vc1 = _call(c, q, k, v, kc, vc, gate)
    want, tol = c.expect(q, k, v, gate)
    err = np.abs(out.reshape(want.shape).astype(np.float64) - want)
    assert (err <= tol).all(), (float(np.nanmax(err / tol)), np.argwhere(~(err <= tol))[:4].tolist())
    c.K, c.V = np.concatenate([c.K, k]), np.concatenate([c.V, v])
    ek, ev = c.ring(fill)
    assert np.array_equal(kc1.view(np.uint16), ek.view(np.uint16)) and np.array_equal(vc1.view(np.uint16), ev.view(np.uint16))
    return float((err / tol).max())


# Refusals (no GPU) -----------------------------------------------------------------------------------


@pytest.mark.parametrize("change,what", [
    (dict(head_dim=96), b"head_dim"), (dict(n_kv_head=0), b"n_head"), (dict(n_head=5), b"n_head"),
    (dict(pin=-1), b"pin"), (dict(pin=64), b"pin"), (dict(slots=(1 << 30) + 1), b"slots"), (dict(sinks=5), b"sinks"),
    (dict(sinks=-1), b"sinks"), (dict(window=0), b"window"), (dict(window=61), b"window"), (dict(scale=0.0), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(q_stride=252), b"q_stride"),
    (dict(q_stride=258), b"q_stride"), (dict(kv_stride=132), b"kv_stride"), (dict(out_stride=255), b"out_stride"),
    (dict(kind=L.KIND_Q8), b"kind")])
def test_geometry_refuses(change, what):
    c = Case(4, 2, 64, 64, 4, 60, 4)
    lib = _lib.lib()
    size = ctypes.c_size_t()
    shape = c.c_shape(**change)
    assert lib.trx_attn_window_geometry(ctypes.byref(shape), 3, ctypes.byref(size)) == _lib.TRX_E_INVALID
    assert what in lib.trx_last_error()
    fake = ctypes.c_void_p(256)
    assert lib.trx_attn_window(ctypes.byref(shape), 3, 0, None, fake, fake, fake, fake, fake, None, fake, fake,
                               None) == _lib.TRX_E_INVALID
    assert what in lib.trx_last_error()


def test_geometry_refuses_more_positions_than_a_grid_holds():
    shape = Case(32, 8, 128, slots=64, pin=4, window=60, sinks=4).c_shape()
    size = ctypes.c_size_t()
    geometry = _lib.lib().trx_attn_window_geometry
    assert geometry(ctypes.byref(shape), 2**20, ctypes.byref(size)) == _lib.TRX_OK
    assert geometry(ctypes.byref(shape), 2**20 + 1, ctypes.byref(size)) == _lib.TRX_E_INVALID
    assert geometry(ctypes.byref(shape), -1, ctypes.byref(size)) == _lib.TRX_E_INVALID


def test_call_refuses_bad_arguments():
    c = Case(4, 2, 64, 64, 4, 60, 4)
    lib, shape = _lib.lib(), c.c_shape()
    fake, odd = ctypes.c_void_p(256), ctypes.c_void_p(264)

    def call(n=1, pos=0, q=fake, k=fake, v=fake, kc=fake, vc=fake, gate=None, out=fake, work=fake, sh=shape):
        return lib.trx_attn_window(ctypes.byref(sh), n, pos, None, q, k, v, kc, vc, gate, out, work, None)

    for kw, what in ((dict(pos=-1), b"position"), (dict(n=2, pos=2**31 - 2), b"position"), (dict(n=-1), b"positions"),
                     (dict(n=1 << 27), b"positions"), (dict(q=None), b"null"), (dict(k=None), b"null"),
                     (dict(vc=None), b"null"), (dict(out=None), b"null"), (dict(q=odd), b"aligned"),
                     (dict(kc=odd), b"aligned"), (dict(out=odd), b"aligned"), (dict(gate=odd), b"aligned"),
                     (dict(gate=fake, sh=c.c_shape(gate_head_stride=32)), b"gate"),
                     (dict(gate=fake, sh=c.c_shape(gate_stride=192)), b"gate"),
                     (dict(work=odd), b"aligned")):
        assert call(**kw) == _lib.TRX_E_INVALID, kw
        assert what in lib.trx_last_error(), (kw, lib.trx_last_error())
    long = Case(4, 2, 64, 4096, 4, 4092, 4).c_shape()
    assert _geometry(long, 1) > 0                       # its keys are split: a workspace is needed
    assert call(work=None, sh=long) == _lib.TRX_E_INVALID and b"workspace" in lib.trx_last_error()
    assert call(n=0, q=None) == _lib.TRX_OK             # nothing to do
    assert lib.trx_attn_window(None, 1, 0, None, *[fake] * 5, None, fake, fake, None) == _lib.TRX_E_INVALID
    assert lib.trx_attn_window_geometry(ctypes.byref(shape), 1, None) == _lib.TRX_E_INVALID
    from trixium_amd.attention import KVRing
    with pytest.raises(ValueError):
        KVRing(4, 2, 64, 64, kind=L.KIND_Q8)
    with pytest.raises(_lib.TrxError):
        KVRing(4, 2, 64, 64, pin=4, window=61)


# Results (GPU) ---------------------------------------------------------------------------------------


GEOMETRIES = [  # heads, kv heads, head dim
    (4, 2, 64), (6, 1, 256), (4, 4, 128), (16, 1, 64), (5, 1, 128), (8, 2, 256), (33, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("geo", GEOMETRIES, ids=str)
def test_single_tokens_and_chunks(geo, kind):
    """From an empty ring: a first token, chunks of odd sizes across the window's and the ring's ends."""
    c = Case(*geo, slots=83, pin=4, window=41, sinks=3, kind=kind, seed=1)
    worst = 0.0
    for n in (1, 1, 5, 33, 1, 40, 2, 9, 67, 1):
        print(geo, kind, "position", c.K.shape[0], "n", n, flush=True)
        worst = max(worst, _check(c, n, gated=n % 2 == 0))
    print(f"worst error {worst:.3f} of the tolerance")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("pin,sinks,window,slots", [(0, 0, 1, 1), (0, 0, 7, 7), (1, 1, 1, 2), (9, 0, 50, 200),
                                                    (64, 64, 64, 128), (40, 37, 3, 64), (4, 4, 300, 304)])
def test_windows_and_sinks(pin, sinks, window, slots, kind):
    c = Case(4, 2, 64, slots, pin, window, sinks, kind=kind, seed=2)
    for n in (3, 1, 30, 70, 1, 130, 17):
        print(pin, sinks, window, slots, "position", c.K.shape[0], "n", n, flush=True)
        _check(c, n)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("geo,n", [((4, 2, 128), 1), ((6, 1, 256), 1), ((4, 2, 64), 3), ((4, 1, 128), 45),
                                   ((6, 1, 256), 130), ((4, 2, 64), 300)], ids=str)
def test_long_windows_split_over_blocks(geo, n, kind):
    c = Case(*geo, slots=2500, pin=4, window=2300, sinks=4, kind=kind, seed=3)
    c.extend(3200)
    print(geo, n, "workspace", _geometry(c.c_shape(), n), flush=True)
    _check(c, n, gated=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("n", [1, 40])
def test_hidden_infinities_and_nans_stay_hidden(kind, n):
    """Slots without a position hold NaN; so do rows that left the window but not the ring; a later row
    of the chunk holds infinities and NaN that the earlier queries must not see."""
    c = Case(4, 2, 64, 200, 4, 50, 2, kind=kind, seed=4)
    _check(c, 30, fill=np.nan)
    c.extend(60)
    c.K[20:35], c.V[20:35] = np.nan, np.inf               # outside every window from position 90 on
    c.K[2:4], c.V[2:4] = -np.inf, np.nan                  # pinned, but no sinks
    _check(c, n, fill=np.nan)
    if n == 1:
        return
    q, k, v = c.rows(n)
    bad = 17
    k[bad], v[bad, :, 5], v[bad, :, 9], v[bad + 1, :, 9], v[bad, 1, 40] = 3.0, np.inf, np.inf, -np.inf, np.nan
    kc, vc = c.ring(np.nan)
    out, _, _ = _call(c, q, k, v, kc, vc)
    out = out.reshape(n, 4, 64)
    finite_v = np.where(np.isfinite(v), v, np.float16(0))
    want, tol = c.expect(q, k, finite_v)
    touched = np.zeros(out.shape, bool)
    touched[bad:, :, 5] = touched[bad:, :, 9] = touched[bad:, 2:, 40] = True
    assert (np.abs(out - want)[~touched] <= tol[~touched]).all()
    assert (out[bad:, :, 5] == np.inf).all()
    assert (out[bad, :, 9] == np.inf).all() and np.isnan(out[bad + 1:, :, 9]).all()
    assert np.isnan(out[bad:, 2:, 40]).all()


@pytest.mark.gpu
def test_a_nan_query_or_seen_key_shows_in_its_rows_only():
    c = Case(4, 2, 64, 200, 4, 50, 4, seed=5)
    c.extend(120)
    q, k, v = c.rows(20)
    q[3, 1, 7] = np.nan
    k[10, 0, 0] = np.nan
    out, _, _ = _call(c, q, k, v, *c.ring())
    out = out.reshape(20, 4, 64)
    bad = np.zeros((20, 4), bool)
    bad[3, 1] = True
    bad[10:, :2] = True                                    # kv head 0 serves query heads 0 and 1
    assert np.isnan(out[bad]).all() and np.isfinite(out[~bad]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4])
def test_queries_of_any_magnitude(size):
    """fp32 queries far from 1 keep their precision (an exponent per query): the scale undoes it."""
    c = Case(4, 2, 64, 128, 4, 100, 4, seed=6, scale=0.125 / size if size > 1 else 0.125)
    c.extend(60)
    q, k, v = c.rows(9, size)
    out, _, _ = _call(c, q, k, v, *c.ring())
    want, tol = c.expect(q, k, v)
    assert (np.abs(out.reshape(want.shape) - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("n", [1, 37])
def test_strides(kind, n):
    """Rows inside wider ones (a fused projection's), gates beside each head; nothing else is written."""
    c = Case(4, 2, 64, 100, 4, 60, 4, kind=kind, seed=7)
    c.extend(150)
    q, k, v = c.rows(n)
    gate = c.rng.standard_normal(q.shape).astype(DT[kind])
    wide = np.full((n, 4 * 64 + 16), 9, DT[kind])
    wide[:, :256] = q.reshape(n, -1)
    kv = np.full((2, n, 2 * 64 + 8), 9, np.float16)
    kv[0, :, :128], kv[1, :, :128] = k.reshape(n, -1), v.reshape(n, -1)
    gw = np.full((n, 4, 128), 9, DT[kind])
    gw[:, :, :64] = gate
    shape = c.c_shape(q_stride=272, kv_stride=136, out_stride=260, gate_stride=512, gate_head_stride=128)
    out, _, _ = _call(c, wide, kv[0], kv[1], *c.ring(), gate=gw, shape=shape)
    want, tol = c.expect(q, k, v, gate)
    assert (np.abs(out[:, :256].reshape(want.shape) - want) <= tol).all()
    assert (out[:, 256:] == 77).all()


@pytest.mark.gpu
def test_position_on_the_device_and_captured_graph():
    """A captured call replayed at the position that the device holds then, on a stream of its own,
    with other work between the replays; positions that the ring cannot hold leave everything."""
    c = Case(4, 2, 64, 90, 4, 70, 4, seed=8)
    c.extend(200)
    B = _lib.DeviceBuffer
    shape, n = c.c_shape(), 3
    kc, vc = c.ring()
    s = ctypes.c_void_p()
    _lib.call("trx_stream_create", ctypes.byref(s))
    kb, vb, out, pos = B.from_array(kc), B.from_array(vc), B(n * 256 * 4), B(4)
    qb, kn, vn, work = B(n * 256 * 4), B(n * 128 * 2), B(n * 128 * 2), B(max(_geometry(shape, n), 1))
    _lib.synchronize()
    _lib.call("trx_graph_begin", s)
    _lib.call("trx_attn_window", ctypes.byref(shape), n, -5, pos.ptr, qb.ptr, kn.ptr, vn.ptr, kb.ptr, vb.ptr, None,
              out.ptr, work.ptr, s)
    ex = ctypes.c_void_p()
    _lib.call("trx_graph_end", s, ctypes.byref(ex))
    for rep in range(4):
        q, k, v = c.rows(n)
        qb.upload(q, s), kn.upload(k, s), vn.upload(v, s), pos.upload(np.array([c.K.shape[0]], np.int32), s)
        _lib.call("trx_graph_launch", ex, s)
        _lib.synchronize(s)
        want, tol = c.expect(q, k, v)
        got = out.download(np.float32, n * 256).reshape(want.shape)
        assert (np.abs(got - want) <= tol).all(), rep
        c.K, c.V = np.concatenate([c.K, k]), np.concatenate([c.V, v])
        assert np.array_equal(kb.download(np.float16).reshape(kc.shape), c.ring()[0])
        _check(Case(4, 2, 64, 90, 4, 70, 4, seed=9 + rep), 5)       # an eager call between the replays
    before = kb.download(np.float16)
    for bad in (-1, 2**31 - 2):
        out.upload(np.full(n * 256, 5, np.float32), s), pos.upload(np.array([bad], np.int32), s)
        _lib.call("trx_graph_launch", ex, s)
        _lib.synchronize(s)
        assert (out.download(np.float32, n * 256) == 5).all()
        assert np.array_equal(kb.download(np.float16).view(np.uint16), before.view(np.uint16))
    _lib.call("trx_graph_destroy", ex)
    _lib.call("trx_stream_destroy", s)


@pytest.mark.gpu
def test_offsets_past_four_gib():
    """The second kv head's rows near the end of a ring of 2^23 slots lie 4 GiB into the cache."""
    slots, kv, hd, n = 1 << 23, 2, 128, 6
    c = Case(4, kv, hd, slots, 4, 90, 4, seed=10)
    B = _lib.DeviceBuffer
    kb, vb = B(2 * kv * slots * hd), B(2 * kv * slots * hd)
    pos = 4 + 3 * (slots - 4) - 50                         # the window's last 40 rows and the call end before the seam
    q, k, v = c.rows(n)
    seen = [0, 1, 2, 3] + list(range(pos - 89, pos))
    _, K, V = c.rows(len(seen))
    for i, p in enumerate(seen):
        for g in range(kv):
            off = (g * slots + c.slot(p)) * hd * 2
            kb.upload(K[i, g], offset=off), vb.upload(V[i, g], offset=off)
    out, work = B(n * 4 * hd * 4), B(max(_geometry(c.c_shape(), n), 1))
    qb, kn, vn = (B.from_array(a) for a in (q, k, v))
    _lib.call("trx_attn_window", ctypes.byref(c.c_shape()), n, pos, None, qb.ptr, kn.ptr, vn.ptr, kb.ptr, vb.ptr, None,
              out.ptr, work.ptr, None)
    _lib.synchronize()
    # The same over a history that is short: the sinks, then the window.
    near = Case(4, kv, hd, slots, 4, 90, 4, seed=10)
    near.K, near.V = K, V
    want, tol = near.expect(q, k, v)
    assert (np.abs(out.download(np.float32, q.size).reshape(want.shape) - want) <= tol).all()
    for r in range(n):
        for g in range(kv):
            off = (g * slots + c.slot(pos + r)) * hd * 2
            assert off > (1 << 32) - (1 << 16) or g == 0
            assert np.array_equal(kb.download(np.float16, hd, offset=off), k[r, g])
            assert np.array_equal(vb.download(np.float16, hd, offset=off), v[r, g])


@pytest.mark.gpu
def test_kv_ring_object():
    from trixium_amd.attention import KVRing
    c = Case(4, 2, 64, 70, 4, 66, 4, seed=11)
    ring = KVRing(4, 2, 64, 70)
    for n in (50, 1, 1, 0, 40, 100, 1):
        q, k, v = c.rows(n)
        want, tol = c.expect(q, k, v)
        assert (np.abs(ring.attend(q, k, v) - want) <= tol).all()
        c.K, c.V = np.concatenate([c.K, k]), np.concatenate([c.V, v])
    assert ring.position == c.K.shape[0]
    assert all(np.array_equal(a, b) for a, b in zip(ring.rows(), c.ring()))
    with pytest.raises(ValueError):
        ring.attend(q, k[:0], v)


def _expect_by_head(c, q, k, v, gate):
    """Case.expect for many heads and rows at once: a kv head's scores as one matrix."""
    pos, n, rep, half = c.K.shape[0], q.shape[0], c.heads // c.kv, c.kind == F16
    K = np.concatenate([c.K, k]).astype(np.float64)
    V = np.concatenate([c.V, v]).astype(np.float64)
    t, u = pos + np.arange(n)[:, None], np.arange(pos + n)[None]
    seen = np.repeat((u <= t) & ((u < c.sinks) | (u > t - c.window)), rep, axis=0)
    N = seen.sum(1)[:, None]
    out = np.empty((n, c.heads, c.hd))
    tol = np.empty_like(out)
    for g in range(c.kv):
        hs = slice(g * rep, (g + 1) * rep)
        qd = q[:, hs].astype(np.float64).reshape(n * rep, c.hd)
        s = np.where(seen, float(c.scale) * (qd @ K[:, g].T), -np.inf)
        S = np.where(seen, float(c.scale) * (np.abs(qd) @ np.abs(K[:, g]).T), 0).max(1)[:, None]
        p = np.exp(s - s.max(1)[:, None])
        p /= p.sum(1)[:, None]
        A, o = p @ np.abs(V[:, g]), p @ V[:, g]
        e = A * (2 * (S * (2.0**-21 + c.hd * 2.0**-24) + 2.0**-21) + N * 2.0**-24 + 2.0**-22)
        if half:
            e += A * 2.0**-11 + N * 2.0**-32 * np.abs(V[:, g]).max()
        sg = 1.0 / (1.0 + np.exp(-gate[:, hs].astype(np.float64).reshape(o.shape)))
        o, e = o * sg, e * sg + np.abs(o) * 2.0**-21
        if half:
            e += np.abs(o) * 2.0**-11 + 2.0**-25
        out[:, hs], tol[:, hs] = o.reshape(n, rep, c.hd), e.reshape(n, rep, c.hd)
    return out, tol


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,hd,window,n", [
    (F32, 32, 2, 64, 1000, 325), (F32, 24, 2, 64, 600, 695), (F16, 64, 4, 64, 1000, 140), (F16, 64, 32, 64, 1000, 177),
    (F32, 64, 4, 128, 600, 140), (F32, 16, 4, 128, 2300, 180), (F32, 32, 32, 128, 100, 547), (F32, 16, 4, 128, 2300, 341),
    (F16, 32, 32, 128, 1000, 177), (F16, 8, 8, 128, 1000, 547), (F16, 64, 32, 128, 1000, 177), (F16, 32, 32, 128, 1000, 140),
    (F32, 64, 8, 256, 333, 140), (F32, 64, 4, 256, 333, 140), (F32, 32, 32, 256, 1000, 68), (F16, 64, 32, 256, 600, 54),
    (F16, 32, 8, 256, 1000, 82), (F16, 64, 4, 256, 200, 140), (F16, 64, 32, 256, 1000, 33)])
def test_many_columns(kind, heads, kv, hd, window, n):
    """Calls with enough columns for the blocks of two and of four waves of them, with and without splits of
    the keys, in each head size and type: the window across the ring's seam, slots that no position takes NaN.
    One value seen by some rows alone is an infinity, in a tile that other rows see whole."""
    c = Case(heads, kv, hd, slots=window + 90, pin=9, window=window, sinks=5, kind=kind, seed=11)
    pos = window + 300
    c.extend(pos)
    c.K[7], c.V[7] = np.nan, np.nan                       # pinned, no sink, outside every window
    q, k, v = c.rows(n)
    gate = c.rng.standard_normal(q.shape).astype(DT[kind])
    kc, vc = c.ring(np.nan)
    late = 300 + window // 2                              # leaves the window after row window // 2
    vc[:, c.slot(late), 3], vc[:, c.slot(late), hd - 1] = np.inf, -np.inf
    out, _, _ = _call(c, q, k, v, kc, vc, gate)
    out = out.reshape(n, heads, hd).astype(np.float64)
    c.K[7], c.V[7] = 0, 0
    want, tol = _expect_by_head(c, q, k, v, gate)
    sees = np.zeros(out.shape, bool)
    rows = pos + np.arange(n) - window < late
    sees[rows, :, 3] = sees[rows, :, hd - 1] = True
    assert (out[rows, :, 3] == np.inf).all() and (out[rows, :, hd - 1] == -np.inf).all()
    err = np.abs(out - want)[~sees] / tol[~sees]
    assert err.max() <= 1, float(err.max())
    print(f"worst error {err.max():.3f} of the tolerance")


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,hd,n", [(F32, 4, 2, 64, 1), (F32, 4, 2, 64, 37), (F16, 6, 1, 256, 5),
                                                (F16, 64, 4, 64, 140), (F32, 64, 4, 128, 140)])
def test_positions_up_to_the_largest(kind, heads, kv, hd, n):
    """Without pinned rows the outputs depend on the position's place in the ring alone: the last n positions
    that int32 holds give the bits of earlier ones at the same place; one more is refused."""
    R = 900
    c = Case(heads, kv, hd, slots=R, pin=0, window=800, sinks=0, kind=kind, seed=12)
    q, k, v = c.rows(n)
    _, kc, vc = c.rows(R)
    kc, vc = (np.ascontiguousarray(a.transpose(1, 0, 2)) for a in (kc, vc))
    top = 2**31 - 1 - n
    low = top - (top - 5000) // R * R
    a, b = (_call(c, q, k, v, kc, vc, pos=p) for p in (top, low))
    assert np.isfinite(a[0]).all()
    for x, y in zip(a, b):
        assert np.array_equal(x.view(np.uint8), y.view(np.uint8))
    with pytest.raises(_lib.TrxError):
        _call(c, q, k, v, kc, vc, pos=top + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,window,n", [(32, 8, 128, 60, 1), (6, 1, 256, 40, 5), (4, 2, 64, 50, 9),
                                                  (8, 8, 128, 90, 31)])
def test_few_columns_with_fp16_queries_round_once(heads, kv, hd, window, n):
    """A token's or a short turn's fp16 outputs are the fp32 result rounded: x + d rounds to a value whose distance
    from x is at most that of x rounded, plus 2 d. Queries with one element leave a score no sum over dims: d is
    the fp32 tolerance without it."""
    c = Case(heads, kv, hd, slots=window + 50, pin=4, window=window, sinks=4, kind=F16, seed=15, scale=1.0)
    c.extend(window + 99)
    pos = c.K.shape[0]
    q, k, v = c.rows(n)
    q[..., 1:] = 0
    out, _, _ = _call(c, q, k, v, *c.ring())
    out = out.reshape(n, heads, hd).astype(np.float64)
    K, V = (np.concatenate(a).astype(np.float64) for a in ((c.K, k), (c.V, v)))
    for r in range(n):
        u = np.r_[:4, pos + r - window + 1:pos + r + 1]
        for h in range(heads):
            s = K[u, h * kv // heads, 0] * float(q[r, h, 0])
            p = np.exp(s - s.max())
            p /= p.sum()
            Vu = V[u, h * kv // heads]
            x, d = p @ Vu, (p @ np.abs(Vu)) * (2 * (np.abs(s).max() + 1) * 2.0**-21 + u.size * 2.0**-24 + 2.0**-22)
            assert (np.abs(out[r, h] - x) <= np.abs(x.astype(np.float16).astype(np.float64) - x) + 2 * d).all(), (r, h)


# The workspace of a length holds every shorter one's --------------------------------------------------


@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("heads,kv,hd,window", [(32, 8, 128, 2048), (32, 8, 128, 4092), (24, 4, 256, 2044), (16, 8, 128, 1020),
                                                (4, 2, 64, 124), (64, 4, 64, 30000), (1, 1, 256, 1 << 20)])
def test_the_workspace_does_not_shrink_with_the_length(heads, kv, hd, window, kind):
    """geometry(n) is a bound for every call of up to n positions: it never falls as n grows, and below 64
    positions (each length's own figure) it is the largest so far."""
    shape = Case(heads, kv, hd, slots=window + 4, pin=4, window=window, sinks=4, kind=kind).c_shape()
    lengths = list(range(1, 700)) + [2**k + d for k in range(10, 15) for d in (-1, 0, 1, 17)]
    sizes = [_geometry(shape, n) for n in lengths]
    assert sizes == sorted(sizes)
    assert _geometry(shape, 0) == 0
    assert all(s % (heads * (hd + 2) * 4) == 0 for s in sizes)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("heads,kv,hd,window,longest", [(32, 8, 128, 2048, 700), (24, 4, 256, 2044, 700), (4, 2, 64, 900, 300)])
def test_one_workspace_for_a_prompt_and_its_rest(heads, kv, hd, window, longest, kind):
    """Sized for the longest call, used by shorter ones, whose keys may be split further: nothing is written behind
    it, and the results are those of a workspace of their own."""
    c = Case(heads, kv, hd, slots=window + 4, pin=4, window=window, sinks=4, kind=kind, seed=16)
    _, kc, vc = c.rows(c.slots)
    kc, vc = (np.ascontiguousarray(a.transpose(1, 0, 2)) for a in (kc, vc))
    B, shape, guard = _lib.DeviceBuffer, c.c_shape(), 1 << 20
    size = _geometry(shape, longest)
    work = B.from_array(np.full(size + guard, 0xA5, np.uint8))
    for n in (longest, 400, 300, 256, 200, 129, 64, 27, 3, 1):
        if n > longest:
            continue
        q, k, v = c.rows(n)
        want = _call(c, q, k, v, kc, vc, pos=3 * window)
        qb, kn, vn, kb, vb = (B.from_array(a) for a in (q, k, v, kc, vc))
        out = B(q.nbytes)
        _lib.call("trx_attn_window", ctypes.byref(shape), n, 3 * window, None, qb.ptr, kn.ptr, vn.ptr, kb.ptr, vb.ptr, None,
                  out.ptr, work.ptr, None)
        _lib.synchronize()
        assert np.array_equal(out.download(np.uint8, q.nbytes), want[0].view(np.uint8).ravel()), n
        assert (work.download(np.uint8, guard, offset=size) == 0xA5).all(), n


@pytest.mark.gpu
def test_kv_ring_object_keeps_its_workspace():
    """A long chunk, then shorter ones and single tokens over the same object."""
    from trixium_amd.attention import KVRing
    c = Case(4, 2, 64, 1004, 4, 1000, 4, seed=17)
    ring = KVRing(4, 2, 64, 1004)
    for n in (1, 900, 300, 27, 1):
        q, k, v = c.rows(n)
        want, tol = c.expect(q, k, v)
        assert (np.abs(ring.attend(q, k, v) - want) <= tol).all()
        c.K, c.V = np.concatenate([c.K, k]), np.concatenate([c.V, v])
    assert ring.work_n == 900 and ring.work.nbytes == _geometry(ring.shape, 900) >= _geometry(ring.shape, 300)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("heads,kv,hd,window,n", [(4, 2, 64, 2300, 1), (4, 2, 128, 200, 1), (6, 1, 256, 200, 9),
                                                  (64, 4, 128, 600, 140), (64, 4, 64, 1000, 140), (64, 8, 256, 333, 140),
                                                  (16, 4, 128, 2300, 180)])
def test_a_seen_infinity_far_below_the_largest_score(kind, heads, kv, hd, window, n):
    """One key's score is 860 powers of two above the others', whose probabilities vanish: the outputs are that
    key's values, and an infinity among the others' is an infinity, wherever the keys are cut into waves and
    splits. With fp16 queries some scores are -inf, a whole tile of them beside the infinity."""
    c = Case(heads, kv, hd, slots=window + 200, pin=4, window=window, sinks=4, kind=kind, seed=13, scale=1.0)
    c.extend(window + 250)
    c.K[:] = 0
    q, k, v = c.rows(n)
    q[:], k[:] = 0, 0
    q[..., 0] = 10
    pos, seen = c.K.shape[0], 250 + n - 1 + 4              # the first position that every query sees, and some
    top = pos - 40
    c.K[top, :, 0] = 60
    at = [2] + list(range(seen, top - 1, max(1, (top - seen) // 24)))
    for i, u in enumerate(at):
        c.V[u, :, 3 + i], c.V[u, :, hd - 1 - i] = np.inf, -np.inf
    if kind == F16:
        c.K[at[5] - 40:at[5] + 41, :, 0] = -np.inf
    kc, vc = c.ring()
    out, _, _ = _call(c, q, k, v, kc, vc)
    out = out.reshape(n, heads, hd).astype(np.float64)
    want = np.repeat(np.broadcast_to(c.V[top].astype(np.float64), (n, kv, hd)), heads // kv, axis=1).copy()
    for i in range(len(at)):
        want[..., 3 + i], want[..., hd - 1 - i] = np.inf, -np.inf
    bad = np.isinf(want)
    assert np.array_equal(out[bad], want[bad]), np.argwhere(bad & (out != want))[:6].tolist()
    # Sums of one term: its probability's planes (2^-22, or 2^-11), 1 / l and the product (2^-24 each), the result.
    eps = 2.0**-21 + (2.0**-10 if kind == F16 else 0)
    assert (np.abs(out[~bad] - want[~bad]) <= eps * np.abs(want[~bad])).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("heads,kv,hd,window,n", [(32, 8, 128, 4000, 1), (32, 8, 128, 4000, 27), (24, 4, 256, 1500, 301),
                                                  (64, 4, 64, 1000, 140)])
def test_repeated_calls_give_the_same_bits(kind, heads, kv, hd, window, n):
    """Over a ring whose replaced rows no query sees, the same call again gives the same outputs and ring."""
    c = Case(heads, kv, hd, slots=window + n + 4, pin=4, window=window, sinks=4, kind=kind, seed=14)
    q, k, v = c.rows(n)
    _, kc, vc = c.rows(c.slots)
    kc, vc = (np.ascontiguousarray(a.transpose(1, 0, 2)) for a in (kc, vc))
    first = _call(c, q, k, v, kc, vc, pos=2 * window)
    for _ in range(4):
        for a, b in zip(first, _call(c, q, k, v, first[1], first[2], pos=2 * window)):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("change", [dict(window=2**32 + 10), dict(sinks=2**32 + 1), dict(pin=2**32 + 4, sinks=4, window=60),
                                    dict(slots=2**32 + 64, window=60), dict(n_head=2**32 + 4), dict(head_dim=2**32 + 64)])
def test_kv_ring_refuses_what_int32_does_not_hold(change):
    from trixium_amd.attention import KVRing
    with pytest.raises(ValueError):
        KVRing(**{**dict(n_head=4, n_kv_head=2, head_dim=64, slots=64, pin=4), **change})
