"""Attention that adds up its probabilities (trx_attn_mass) against its definition in 64 bits, eviction by them
(trx_kv_evict) against a sort on the host, to the bit, the two and the drafts behind what stays as a program uses them,
and what they refuse.

Outputs: test_shared_prefix_gpu.py's tolerance. A mass adds probabilities: each is off by what an output's weight is
(S (2^-21 + head_dim 2^-24) + 2^-21 twice, N 2^-24 for the sums) and by what its second taking adds (the score in powers
of two and the reference, each rounded once and below 1.5 S: S 2^-22; the exponential, the reciprocal and their product
2^-21), the sum of T of them by T 2^-24, and adding it to the mass by 2^-24 of the result. Probabilities below 2^-126
may vanish."""

import ctypes

import numpy as np
import pytest

from trixium_amd import _lib, layout as L
from test_shared_prefix_gpu import attend64

F32, F16 = L.KIND_F32, L.KIND_F16
DT = {F32: np.float32, F16: np.float16}


class Cache:
    """A cache with masses, and what the operators have to make of it."""

    def __init__(self, heads, kv, hd, slots, kind=F32, seed=0, scale=None):
        self.heads, self.kv, self.hd, self.slots, self.kind = heads, kv, hd, slots, kind
        self.scale = np.float32(1.0 / np.sqrt(hd) if scale is None else scale)
        self.rng = r = np.random.default_rng(seed)
        self.K, self.V = (r.standard_normal((kv, slots, hd)).astype(np.float16) for _ in range(2))
        self.mass = r.lognormal(-1, 2, (kv, slots)).astype(np.float32)
        self.positions = r.integers(0, 1 << 20, (kv, slots)).astype(np.int32)

    def rows(self, n, size=1.0):
        r = self.rng
        q = (1.5 * size * r.standard_normal((n, self.heads, self.hd))).astype(DT[self.kind])
        k, v = (r.standard_normal((n, self.kv, self.hd)).astype(np.float16) for _ in range(2))
        return q, k, v

    def shape(self, **kw):
        q, kv = self.heads * self.hd, self.kv * self.hd
        d = dict(kind=self.kind, n_head=self.heads, n_kv_head=self.kv, head_dim=self.hd, slots=self.slots, q_stride=q,
                 kv_stride=kv, out_stride=q, gate_stride=q, gate_head_stride=self.hd, scale=float(self.scale))
        d.update(kw)
        return _lib.AttnMassShape(**d)

    def arrays(self):
        return self.K, self.V, self.mass, self.positions

    def attend(self, q, k, v, count, pos, gate=None, state=None, shape=None, stream=None):
        """One call on device copies; (out, K, V, mass, positions) back."""
        B, shape, n = _lib.DeviceBuffer, shape or self.shape(), k.shape[0]
        qb, kb, vb = (B.from_array(a) for a in (q, k, v))
        cache = [B.from_array(a) for a in self.arrays()]
        gb = B.from_array(gate) if gate is not None else None
        sb = B.from_array(np.asarray(state, np.int32)) if state is not None else None
        out, work = B.from_array(np.full(n * shape.out_stride, 77, DT[self.kind])), B(max(geometry(shape, n), 1))
        _lib.synchronize()
        _lib.call("trx_attn_mass", ctypes.byref(shape), n, count, pos, sb.ptr if sb else None, qb.ptr, kb.ptr, vb.ptr,
                  *(b.ptr for b in cache), gb.ptr if gb else None, out.ptr, work.ptr, stream)
        _lib.synchronize(stream)
        return (out.download(DT[self.kind], n * shape.out_stride).reshape(n, shape.out_stride),
                *(b.download(a.dtype, a.size).reshape(a.shape) for b, a in zip(cache, self.arrays())))

    def after(self, q, k, v, count, pos, gate=None):
        """(outputs, tolerances), and the cache moves on: K, V, positions; mass and its tolerance are returned too."""
        n = q.shape[0]
        end = count + n
        self.K[:, count:end], self.V[:, count:end] = k.transpose(1, 0, 2), v.transpose(1, 0, 2)
        self.positions[:, count:end] = pos + np.arange(n)
        out, tol, p, e = attend64(q, self.K[:, :end].transpose(1, 0, 2), self.V[:, :end].transpose(1, 0, 2),
                                  count + 1 + np.arange(n), self.scale, self.kind == F16, gate)
        rep = self.heads // self.kv
        mass, mtol = self.mass.astype(np.float64), np.zeros(self.mass.shape)
        for g in range(self.kv):
            given = p[:, g * rep:(g + 1) * rep].reshape(n * rep, end).sum(0)
            mass[g, :end] = np.where(np.arange(end) < count, mass[g, :end], 0) + given
            mtol[g, :end] = (e[:, g * rep:(g + 1) * rep].reshape(n * rep, end).sum(0) + given * n * rep * 2.0**-24
                             + mass[g, :end] * 2.0**-24 + n * rep * 2.0**-120)
        return out, tol, mass, mtol

    def check(self, n, count, pos=None, gated=False):
        pos = count if pos is None else pos
        q, k, v = self.rows(n)
        gate = self.rng.standard_normal(q.shape).astype(DT[self.kind]) if gated else None
        out, K, V, mass, positions = self.attend(q, k, v, count, pos, gate)
        want, tol, wm, mtol = self.after(q, k, v, count, pos, gate)
        err = np.abs(out.reshape(want.shape).astype(np.float64) - want)
        assert (err <= tol).all(), (float(np.nanmax(err / tol)), np.argwhere(~(err <= tol))[:4].tolist())
        assert np.array_equal(K.view(np.uint16), self.K.view(np.uint16)) and np.array_equal(V.view(np.uint16), self.V.view(np.uint16))
        assert np.array_equal(positions, self.positions)
        merr = np.abs(mass - wm)
        assert (merr <= mtol).all(), (float(np.nanmax(merr / np.maximum(mtol, 1e-300))), np.argwhere(~(merr <= mtol))[:4].tolist())
        self.mass = mass
        return float((err / tol).max()), float((merr[:, :count + n] / mtol[:, :count + n]).max())

    def evict(self, count, pos, keep, sinks, recent, state=None, stream=None):
        B, shape = _lib.DeviceBuffer, self.shape()
        cache = [B.from_array(a) for a in self.arrays()]
        sb = B.from_array(np.asarray(state, np.int32)) if state is not None else None
        work = B(evict_geometry(shape))
        _lib.synchronize()
        _lib.call("trx_kv_evict", ctypes.byref(shape), count, pos, sb.ptr if sb else None, keep, sinks, recent,
                  *(b.ptr for b in cache), work.ptr, stream)
        _lib.synchronize(stream)
        return [b.download(a.dtype, a.size).reshape(a.shape) for b, a in zip(cache, self.arrays())]

    def evicted(self, count, pos, keep, sinks, recent):
        """The cache after it, by a sort on the host."""
        arrays = [a.copy() for a in self.arrays()]
        if count <= keep:
            return arrays
        for g in range(self.kv):
            at, m = self.positions[g, :count].astype(np.int64), self.mass[g, :count].astype(np.float64)
            first = (at < sinks) | (at >= pos - recent)
            order = np.lexsort((np.arange(count), np.where(np.isnan(m), 0, -m), np.isnan(m) & ~first, ~first))
            order = np.concatenate([np.flatnonzero(first), order[first.sum():]])
            stays = np.zeros(count, bool)
            stays[order[:keep]] = True
            holes, moved = np.flatnonzero(~stays[:keep]), keep + np.flatnonzero(stays[keep:])
            for a in arrays:
                a[g, holes] = a[g, moved]
        return arrays

    def check_evict(self, count, pos, keep, sinks, recent, **kw):
        got, want = self.evict(count, pos, keep, sinks, recent, **kw), self.evicted(count, pos, keep, sinks, recent)
        for a, b, name in zip(got, want, ("K", "V", "mass", "positions")):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8)), (name, np.argwhere(a != b)[:5].tolist())
        self.K, self.V, self.mass, self.positions = got


def geometry(shape, n):
    size = ctypes.c_size_t()
    _lib.call("trx_attn_mass_geometry", ctypes.byref(shape), n, ctypes.byref(size))
    return size.value


def evict_geometry(shape):
    size = ctypes.c_size_t()
    _lib.call("trx_kv_evict_geometry", ctypes.byref(shape), ctypes.byref(size))
    return size.value


# Refusals (no GPU) -----------------------------------------------------------------------------------


@pytest.mark.parametrize("change,what", [
    (dict(head_dim=96), b"head_dim"), (dict(n_kv_head=0), b"n_head"), (dict(n_head=5), b"n_head"), (dict(slots=0), b"slots"),
    (dict(slots=(1 << 30) + 1), b"slots"), (dict(slots=(1 << 29) + 1), b"slots"), (dict(scale=-1.0), b"scale"), (dict(q_stride=252), b"q_stride"),
    (dict(q_stride=258), b"q_stride"), (dict(kv_stride=132), b"kv_stride"), (dict(out_stride=255), b"out_stride"),
    (dict(kind=L.KIND_Q8), b"kind")])
def test_geometry_refuses(change, what):
    c = Cache(4, 2, 64, 40)
    lib, size, fake = _lib.lib(), ctypes.c_size_t(), ctypes.c_void_p(256)
    shape = c.shape(**change)
    assert lib.trx_attn_mass_geometry(ctypes.byref(shape), 1, ctypes.byref(size)) == _lib.TRX_E_INVALID
    assert what in lib.trx_last_error(), lib.trx_last_error()
    assert lib.trx_attn_mass(ctypes.byref(shape), 1, 0, 0, None, *[fake] * 7, None, fake, fake, None) == _lib.TRX_E_INVALID
    assert what in lib.trx_last_error(), lib.trx_last_error()
    if what in (b"head_dim", b"n_head", b"slots"):
        assert lib.trx_kv_evict_geometry(ctypes.byref(shape), ctypes.byref(size)) == _lib.TRX_E_INVALID
        assert lib.trx_kv_evict(ctypes.byref(shape), 10, 10, None, 5, 0, 0, *[fake] * 5, None) == _lib.TRX_E_INVALID
        assert what in lib.trx_last_error(), lib.trx_last_error()


def test_attend_refuses_bad_arguments():
    c = Cache(4, 2, 64, 40)
    lib, shape, fake, odd = _lib.lib(), c.shape(), ctypes.c_void_p(256), ctypes.c_void_p(264)
    names = ("q", "k", "v", "kc", "vc", "mass", "positions", "gate", "out", "work")

    def call(n=1, count=0, pos=0, state=None, sh=shape, **kw):
        a = dict.fromkeys(names, fake) | dict(gate=None) | kw
        return lib.trx_attn_mass(ctypes.byref(sh), n, count, pos, state, *(a[x] for x in names), None)

    bad = [(dict(n=-1), b"rows"), (dict(n=1 << 22), b"rows"), (dict(n=41), b"slots"), (dict(count=-1), b"slots"), (dict(count=40), b"slots"),
           (dict(n=3, count=38), b"slots"), (dict(pos=-1), b"position"), (dict(n=2, pos=2**31 - 2), b"position"),
           (dict(mass=ctypes.c_void_p(258)), b"aligned"), (dict(positions=ctypes.c_void_p(258)), b"aligned"),
           (dict(state=ctypes.c_void_p(258)), b"aligned"), (dict(n=41, state=fake), b"slots"),
           (dict(gate=fake, sh=c.shape(gate_head_stride=32)), b"gate")]
    bad += [({x: None}, b"null") for x in names if x != "gate"]
    bad += [({x: odd}, b"aligned") for x in names if x not in ("mass", "positions")]
    for kw, what in bad:
        assert call(**kw) == _lib.TRX_E_INVALID, kw
        assert what in lib.trx_last_error(), (kw, lib.trx_last_error())
    assert call(n=0, q=None) == _lib.TRX_OK
    assert lib.trx_attn_mass(None, 1, 0, 0, None, *[fake] * 10, None) == _lib.TRX_E_INVALID
    assert lib.trx_attn_mass_geometry(ctypes.byref(shape), 1, None) == _lib.TRX_E_INVALID


def test_evict_refuses_bad_arguments():
    c = Cache(4, 2, 64, 40)
    lib, shape, fake = _lib.lib(), c.shape(), ctypes.c_void_p(256)
    names = ("kc", "vc", "mass", "positions", "work")

    def call(count=30, pos=100, state=None, keep=20, sinks=4, recent=8, **kw):
        a = dict.fromkeys(names, fake) | kw
        return lib.trx_kv_evict(ctypes.byref(shape), count, pos, state, keep, sinks, recent, *(a[x] for x in names), None)

    bad = [(dict(keep=0), b"keep"), (dict(keep=41), b"keep"), (dict(count=41), b"slots"), (dict(count=-1), b"slots"), (dict(pos=-1), b"position"),
           (dict(sinks=-1), b"sinks"), (dict(recent=-1), b"recent"), (dict(state=ctypes.c_void_p(258)), b"aligned"),
           (dict(kc=ctypes.c_void_p(264)), b"aligned"), (dict(vc=ctypes.c_void_p(264)), b"aligned"), (dict(work=ctypes.c_void_p(264)), b"aligned"),
           (dict(mass=ctypes.c_void_p(258)), b"aligned"), (dict(positions=ctypes.c_void_p(258)), b"aligned")]
    bad += [({x: None}, b"null") for x in names]
    for kw, what in bad:
        assert call(**kw) == _lib.TRX_E_INVALID, kw
        assert what in lib.trx_last_error(), (kw, lib.trx_last_error())
    assert call(count=20, kc=None) == _lib.TRX_OK               # nothing to do
    assert lib.trx_kv_evict(None, 30, 100, None, 20, 4, 8, *[fake] * 5, None) == _lib.TRX_E_INVALID
    assert lib.trx_kv_evict_geometry(None, None) == _lib.TRX_E_INVALID


@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (24, 4, 256), (16, 8, 128), (4, 2, 64), (40, 1, 64)])
def test_the_workspace_does_not_shrink_with_the_length(heads, kv, hd, kind):
    shape = Cache(heads, kv, hd, 1, kind).shape(slots=5000)
    sizes = [geometry(shape, n) for n in range(0, 1500)]
    assert sizes == sorted(sizes)


# Attention with masses (GPU) ----------------------------------------------------------------------------


GEOMETRIES = [  # heads, kv heads, head dim
    (4, 2, 64), (6, 1, 256), (4, 4, 128), (16, 1, 64), (5, 1, 128), (8, 2, 256), (33, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("geo", GEOMETRIES, ids=str)
def test_tokens_and_chunks(geo, kind):
    """From an empty cache: a first token, chunks of odd sizes, each with the masses of all that came before."""
    c = Cache(*geo, slots=400, kind=kind, seed=1)
    count, worst = 0, (0, 0)
    for n in (1, 1, 5, 33, 1, 40, 2, 9, 131, 1, 7):
        print(geo, kind, "count", count, "n", n, flush=True)
        worst = max(worst, c.check(n, count, pos=count + 1000, gated=n % 2 == 0))
        count += n
    print(f"worst errors {worst} of the tolerances")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("geo,count,n", [((4, 2, 128), 2300, 1), ((6, 1, 256), 2300, 1), ((4, 2, 64), 3200, 3), ((4, 1, 128), 2300, 45),
                                         ((6, 1, 256), 1500, 130), ((4, 2, 64), 2000, 300), ((32, 8, 128), 700, 1),
                                         ((64, 2, 64), 500, 70), ((24, 4, 256), 900, 27), ((16, 8, 128), 0, 257),
                                         ((32, 2, 128), 1000, 90), ((8, 1, 128), 600, 300)], ids=str)
def test_long_caches(geo, count, n, kind):
    """Keys split over blocks, and enough columns for the wide blocks."""
    c = Cache(*geo, slots=count + n + 17, kind=kind, seed=2)
    print(f"worst errors {c.check(n, count, gated=True)} of the tolerances")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("n", [1, 9, 60])
def test_slots_behind_the_rows_may_hold_anything(n, kind):
    """NaN and infinities behind the rows, in masses too; afterwards the new rows' masses are this call's alone."""
    c = Cache(4, 2, 64, 300, kind=kind, seed=3)
    c.K[:, 150:], c.V[:, 150:], c.mass[:, 150:] = np.nan, np.inf, np.nan
    c.check_rest = c.mass[:, 150 + n:].copy()
    q, k, v = c.rows(n)
    out, K, V, mass, positions = c.attend(q, k, v, 150, 9)
    want, tol, wm, mtol = c.after(q, k, v, 150, 9)
    assert (np.abs(out.reshape(want.shape) - want) <= tol).all()
    assert (np.abs(mass - wm)[:, :150 + n] <= mtol[:, :150 + n]).all()
    assert np.array_equal(K.view(np.uint16), c.K.view(np.uint16)) and np.array_equal(mass[:, 150 + n:].view(np.uint32), c.check_rest.view(np.uint32))
    assert np.array_equal(positions, c.positions)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("n", [1, 60])
def test_a_later_row_gives_nothing_to_an_earlier_one(n, kind):
    """A new key that would take all the attention leaves the rows before it, and their share of the masses, alone;
    an infinity in a value touches no mass; a NaN key shows in the masses of its own kv head alone."""
    c = Cache(4, 2, 64, 200, kind=kind, seed=4)
    q, k, v = c.rows(n)
    k[n - 1], v[n // 2, 0, 3] = 20.0, np.inf
    out, _, _, mass, _ = c.attend(q, k, v, 100, 100)
    inf = out.reshape(n, 4, 64)[:, :2, 3].copy()
    assert (inf[n // 2:] == np.inf).all() and np.isfinite(inf[:n // 2]).all()
    v[n // 2, 0, 3] = 0
    want, tol, wm, mtol = c.after(q, k, v, 100, 100)
    ok = np.ones(want.shape, bool)
    ok[n // 2:, :2, 3] = False
    assert (np.abs(out.reshape(want.shape) - want)[ok] <= tol[ok]).all()
    assert (np.abs(mass - wm)[:, :100 + n] <= mtol[:, :100 + n]).all()
    c.K[1, 50, 0] = np.nan
    out, _, _, mass, _ = c.attend(q, k, v, 100, 100)
    assert np.isnan(out.reshape(n, 4, 64)[:, 2:]).all() and np.isfinite(out.reshape(n, 4, 64)[:, :2]).all()
    assert np.isfinite(mass[0]).all() and np.isnan(mass[1, :100 + n]).all() and np.isfinite(mass[1, 100 + n:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("n", [1, 45])
def test_masses_sum_to_the_rows(n, kind):
    """Each position and head gives a mass of 1: over a cache of zeros the masses add up to their number. Both takings
    see the same scores, so that a share is off by the second one's roundings alone (S 2^-22 + 2^-21, S below 40 here)
    and the sums by N 2^-24 (N below 700 and as many again of the masses): less than 2^-13 in all."""
    c = Cache(8, 2, 128, 700, kind=kind, seed=5)
    c.mass[:] = 0
    q, k, v = c.rows(n)
    _, _, _, mass, _ = c.attend(q, k, v, 600, 600)
    assert np.abs(mass[:, :600 + n].astype(np.float64).sum(1) / (4 * n) - 1).max() <= 2.0**-13
    assert (mass[:, 600 + n:] == 0).all() and (mass[:, :600 + n] > 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4])
@pytest.mark.parametrize("n", [2, 40])
def test_queries_of_any_magnitude(size, n):
    c = Cache(4, 2, 64, 200, seed=6, scale=0.125 / size if size > 1 else 0.125)
    q, k, v = c.rows(n, size)
    out, _, _, mass, _ = c.attend(q, k, v, 120, 0)
    want, tol, wm, mtol = c.after(q, k, v, 120, 0)
    assert (np.abs(out.reshape(want.shape) - want) <= tol).all() and (np.abs(mass - wm) <= mtol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("n", [1, 37])
def test_strides(n, kind):
    c = Cache(4, 2, 64, 200, kind=kind, seed=7)
    q, k, v = c.rows(n)
    gate = c.rng.standard_normal(q.shape).astype(DT[kind])
    wide = np.full((n, 4 * 64 + 16), 9, DT[kind])
    wide[:, :256] = q.reshape(n, -1)
    kv = np.full((2, n, 2 * 64 + 8), 9, np.float16)
    kv[0, :, :128], kv[1, :, :128] = k.reshape(n, -1), v.reshape(n, -1)
    gw = np.full((n, 4, 128), 9, DT[kind])
    gw[:, :, :64] = gate
    shape = c.shape(q_stride=272, kv_stride=136, out_stride=260, gate_stride=512, gate_head_stride=128)
    out, K, _, mass, _ = c.attend(wide, kv[0], kv[1], 90, 90, gate=gw, shape=shape)
    want, tol, wm, mtol = c.after(q, k, v, 90, 90, gate)
    assert (np.abs(out[:, :256].reshape(want.shape) - want) <= tol).all() and (out[:, 256:] == 77).all()
    assert (np.abs(mass - wm) <= mtol).all() and np.array_equal(K, c.K)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("geo,n", [((32, 8, 128), 1), ((32, 8, 128), 27), ((24, 4, 256), 101), ((64, 4, 64), 140)], ids=str)
def test_repeated_calls_give_the_same_bits(geo, n, kind):
    c = Cache(*geo, slots=2000, kind=kind, seed=8)
    q, k, v = c.rows(n)
    first = c.attend(q, k, v, 1700, 5)
    for _ in range(3):
        for a, b in zip(first, c.attend(q, k, v, 1700, 5)):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_state_on_the_device_captured(n):
    """A captured token (or chunk) and an eviction, replayed while the rows and the position grow past the budget, with
    eager calls between the replays; a state out of range leaves everything as it is."""
    c = Cache(4, 2, 64, 330, seed=9)
    B, shape, keep = _lib.DeviceBuffer, c.shape(), 250
    s = ctypes.c_void_p()
    _lib.call("trx_stream_create", ctypes.byref(s))
    cache = [B.from_array(a) for a in c.arrays()]
    qb, kb, vb, out, sb = (B(x) for x in (n * 256 * 4, n * 128 * 2, n * 128 * 2, n * 256 * 4, 8))
    work, ework = B(geometry(shape, n)), B(evict_geometry(shape))
    _lib.synchronize()
    ex = [ctypes.c_void_p(), ctypes.c_void_p()]
    _lib.call("trx_graph_begin", s)
    _lib.call("trx_attn_mass", ctypes.byref(shape), n, -3, -3, sb.ptr, qb.ptr, kb.ptr, vb.ptr, *(b.ptr for b in cache), None, out.ptr,
              work.ptr, s)
    _lib.call("trx_graph_end", s, ctypes.byref(ex[0]))
    _lib.call("trx_graph_begin", s)
    _lib.call("trx_kv_evict", ctypes.byref(shape), -3, -3, sb.ptr, keep, 3, 20, *(b.ptr for b in cache), ework.ptr, s)
    _lib.call("trx_graph_end", s, ctypes.byref(ex[1]))
    count, pos = keep - n - 1, 700
    for rep in range(5):
        q, k, v = c.rows(n)
        for b, a in ((qb, q), (kb, k), (vb, v), (sb, np.array([count, pos], np.int32))):
            b.upload(a, s)
        _lib.call("trx_graph_launch", ex[0], s)
        _lib.synchronize(s)
        want, tol, wm, mtol = c.after(q, k, v, count, pos)
        assert (np.abs(out.download(np.float32, q.size).reshape(q.shape) - want) <= tol).all(), rep
        c.mass = cache[2].download(np.float32).reshape(c.mass.shape)
        assert (np.abs(c.mass - wm) <= mtol).all(), rep
        count, pos = count + n, pos + n
        sb.upload(np.array([count, pos], np.int32), s)
        _lib.call("trx_graph_launch", ex[1], s)
        _lib.synchronize(s)
        want = c.evicted(count, pos, keep, 3, 20)
        for b, a in zip(cache, want):
            assert np.array_equal(b.download(a.dtype).reshape(a.shape).view(np.uint8), a.view(np.uint8)), rep
        c.K, c.V, c.mass, c.positions = want
        count = min(count, keep)
        Cache(4, 2, 64, 90, seed=30 + rep).check(3, 40)                # an eager call between the replays
    before = [b.download(np.uint8) for b in cache]
    for bad in ((-1, 5), (331 - n, 5), (5, -1), (5, 2**31 - n)):
        sb.upload(np.array(bad, np.int32), s), out.upload(np.full(n * 256, 5, np.float32), s)
        _lib.call("trx_graph_launch", ex[0], s)
        _lib.synchronize(s)
        assert (out.download(np.float32, n * 256) == 5).all(), bad
        assert all(np.array_equal(a, b.download(np.uint8)) for a, b in zip(before, cache)), bad
    for bad in ((331, 5), (300, -1), (-5, 5), (keep, 5)):
        sb.upload(np.array(bad, np.int32), s)
        _lib.call("trx_graph_launch", ex[1], s)
        _lib.synchronize(s)
        assert all(np.array_equal(a, b.download(np.uint8)) for a, b in zip(before, cache)), bad
    for e in ex:
        _lib.call("trx_graph_destroy", e)
    _lib.call("trx_stream_destroy", s)


@pytest.mark.gpu
def test_one_workspace_for_a_prompt_and_its_rest():
    """Sized for the longest call, used by shorter ones: nothing is written behind it."""
    c, B, guard = Cache(32, 8, 128, 1500, seed=10), _lib.DeviceBuffer, 1 << 20
    shape = c.shape()
    size = geometry(shape, 700)
    work = B.from_array(np.full(size + guard, 0xA5, np.uint8))
    for n in (700, 300, 129, 64, 9, 8, 7, 3, 1):
        q, k, v = c.rows(n)
        want = c.attend(q, k, v, 800, 800)
        qb, kb, vb = (B.from_array(a) for a in (q, k, v))
        cache, out = [B.from_array(a) for a in c.arrays()], B(q.nbytes)
        _lib.call("trx_attn_mass", ctypes.byref(shape), n, 800, 800, None, qb.ptr, kb.ptr, vb.ptr, *(b.ptr for b in cache), None, out.ptr,
                  work.ptr, None)
        _lib.synchronize()
        assert np.array_equal(out.download(np.uint8, q.nbytes), want[0].view(np.uint8).ravel()), n
        assert np.array_equal(cache[2].download(np.uint8), want[3].view(np.uint8).ravel()), n
        assert (work.download(np.uint8, guard, offset=size) == 0xA5).all(), n


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,n", [(32, 8, 128, 1), (6, 1, 256, 5), (4, 2, 64, 9), (8, 8, 128, 31)])
def test_few_columns_with_fp16_queries_round_once(heads, kv, hd, n):
    """As test_shared_prefix_gpu.py's: up to 32 columns' fp16 outputs are the fp32 result rounded."""
    c = Cache(heads, kv, hd, 1500 + n, F16, seed=16, scale=1.0)
    q, k, v = c.rows(n)
    q[..., 1:] = 0
    out, *_ = c.attend(q, k, v, 1500, 1500)
    out = out.reshape(n, heads, hd).astype(np.float64)
    K, V = (np.concatenate([a[:, :1500], x.transpose(1, 0, 2)], axis=1).astype(np.float64) for a, x in ((c.K, k), (c.V, v)))
    for r in range(n):
        for h in range(heads):
            g, N = h * kv // heads, 1500 + r + 1
            s = K[g, :N, 0] * float(q[r, h, 0])
            p = np.exp(s - s.max())
            p /= p.sum()
            x, d = p @ V[g, :N], (p @ np.abs(V[g, :N])) * (2 * (np.abs(s).max() + 1) * 2.0**-21 + N * 2.0**-24 + 2.0**-22)
            assert (np.abs(out[r, h] - x) <= np.abs(x.astype(np.float16).astype(np.float64) - x) + 2 * d).all(), (r, h)


# Eviction (GPU) -------------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("kv,hd,slots,count,keep", [
    (2, 64, 1, 1, 1), (2, 64, 2, 2, 1), (1, 64, 65, 65, 64), (3, 128, 100, 90, 1), (2, 256, 300, 300, 150), (8, 128, 1100, 1024, 1023),
    (8, 128, 1100, 1025, 1000), (8, 128, 4096, 4096, 4095), (4, 256, 5000, 4999, 700), (2, 64, 33000, 32999, 32999 // 2),
    (2, 64, 70000, 66000, 65999), (1, 64, 140000, 139999, 130001), (40, 64, 900, 777, 700), (2, 64, 5000, 4097, 4032), (2, 64, 5000, 4097, 4033)])
def test_evict_matches_a_sort(kv, hd, slots, count, keep):
    c = Cache(kv, kv, hd, slots, seed=11)
    c.positions[:, :count] = np.stack([c.rng.permutation(2 * count)[:count] for _ in range(kv)])
    print(kv, hd, slots, count, keep, flush=True)
    c.check_evict(count, 2 * count, keep, sinks=min(4, keep), recent=keep // 10)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["equal", "zeros", "few values", "nan", "inf", "negative", "close", "bits"])
@pytest.mark.parametrize("keep", [1, 700, 1999])
def test_evict_orders_every_mass(keep, what):
    """Equal masses go by slot; NaN below every number, of both signs; -0 as 0; masses one bit apart."""
    c, n = Cache(2, 2, 64, 2100, seed=12), 2000
    m = c.mass[:, :n]
    if what == "equal":
        m[:] = 0.25
    elif what == "zeros":
        m[:] = np.where(c.rng.random(m.shape) < 0.5, 0.0, -0.0)
    elif what == "few values":
        m[:] = c.rng.integers(0, 3, m.shape)
    elif what == "nan":
        m[c.rng.random(m.shape) < 0.4] = np.nan
        m[c.rng.random(m.shape) < 0.2] = -np.nan
    elif what == "inf":
        m[c.rng.random(m.shape) < 0.4] = np.inf
        m[c.rng.random(m.shape) < 0.1] = -np.inf
    elif what == "negative":
        m[c.rng.random(m.shape) < 0.5] *= -1
    elif what == "close":
        m[:] = (np.float32(1.5).view(np.uint32) + c.rng.integers(0, 700, m.shape).astype(np.uint32)).view(np.float32)
    else:
        m[:] = c.rng.integers(0, 2**32, m.shape, dtype=np.uint64).astype(np.uint32).view(np.float32)
    for sinks, recent in ((0, 0), (200000, 30000)):
        c.check_evict(n, 1 << 20, keep, sinks, recent)


@pytest.mark.gpu
def test_evict_keeps_positions_first():
    """Rows at the first and last positions stay whatever their mass, NaN too; with more of them than stay, by slot."""
    c = Cache(3, 3, 64, 600, seed=13)
    for g in range(3):
        c.positions[g, :500] = c.rng.permutation(500)
    low = (c.positions < 5) | (c.positions >= 460)
    c.mass[low] = np.where(c.rng.random(low.sum()) < 0.5, 0, np.nan)
    before = c.positions.copy()
    c.check_evict(500, 500, 300, 5, 40)
    for g in range(3):
        assert set(range(5)) | set(range(460, 500)) <= set(c.positions[g, :300].tolist())
    c.check_evict(300, 500, 20, 5, 40)
    assert all(set(c.positions[g, :20].tolist()) <= set(range(5)) | set(range(460, 500)) for g in range(3))
    assert before.shape == c.positions.shape
    c.check_evict(20, 500, 20, 5, 40)                            # nothing to do
    c.check_evict(0, 500, 20, 5, 40)
    c.check_evict(20, 2**31 - 1, 7, 2**31 - 1, 2**31 - 1)


@pytest.mark.gpu
def test_evict_past_four_gib():
    """The second kv head's rows of a cache of 2^24 slots lie 4 GiB into it."""
    slots, hd, kv, n, B = (1 << 24) + 5, 128, 2, 90, _lib.DeviceBuffer
    c = Cache(kv, kv, hd, n, seed=14)
    c.positions[:, :n] = np.stack([c.rng.permutation(n) for _ in range(kv)])
    row = (2 * hd, 2 * hd, 4, 4)
    cache = [B(r * kv * slots) for r in row]
    for b, a, r in zip(cache, c.arrays(), row):
        for g in range(kv):
            b.upload(a[g], offset=r * g * slots)
    shape = c.shape(slots=slots)
    work = B(evict_geometry(shape))
    _lib.call("trx_kv_evict", ctypes.byref(shape), n, n, None, 50, 2, 9, *(b.ptr for b in cache), work.ptr, None)
    _lib.synchronize()
    for b, a, r in zip(cache, c.evicted(n, n, 50, 2, 9), row):
        for g in range(kv):
            assert np.array_equal(b.download(a.dtype, a[g].size, offset=r * g * slots).reshape(a[g].shape), a[g])


# As a program uses them ------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
def test_a_cache_under_a_budget_and_its_drafts(kind):
    """A prompt in two chunks, cut to a budget, tokens that each push one row out, then drafts behind what stays, whose
    next tokens are drawn from logits made of their outputs."""
    from trixium_amd import sampling
    from trixium_amd.attention import KVMass
    c = Cache(8, 2, 64, 300, kind=kind, seed=15)
    for a in c.arrays():
        a[:] = 0
    m = KVMass(8, 2, 64, 300, kind=kind)
    count = pos = 0
    for n, keep in ((150, 300), (140, 120), (1, 120), (1, 120), (1, 120), (7, 120)):
        q, k, v = c.rows(n)
        out = m.attend(q, k, v)
        want, tol, wm, mtol = c.after(q, k, v, count, pos)
        assert (np.abs(out - want) <= tol).all()
        count, pos = count + n, pos + n
        assert (np.abs(m.masses() - wm[:, :count]) <= mtol[:, :count]).all()
        c.mass[:, :count] = m.masses()
        c.K, c.V, c.mass, c.positions = c.evicted(count, pos, keep, 4, 30)
        m.evict(keep, sinks=4, recent=30)
        count = min(count, keep)
        assert m.count == count and m.next == pos
        for a, b in zip((*m.rows(), m.masses(), m.positions()), c.arrays()):
            assert np.array_equal(a, b[:, :count])
    d = m.share(5, 12)
    K, V = c.K[:, :count].transpose(1, 0, 2), c.V[:, :count].transpose(1, 0, 2)
    m.attend(*c.rows(3))                                          # the cache goes on; the drafts have a copy
    tails = [(np.zeros((0, 2, 64), np.float16),) * 2 for _ in range(5)]
    W = c.rng.standard_normal((8 * 64, 50))
    for n, counts in ((1, [1] * 5), (3, [3, 0, 1, 2, 3]), (1, [1] * 5)):
        q, k, v = c.rows(5 * n)
        out = d.attend(*(a.reshape(5, n, *a.shape[1:]) for a in (q, k, v)), counts=counts)
        for b in range(5):
            rows = slice(b * n, b * n + counts[b])
            tails[b] = tuple(np.concatenate([t, x[rows]]) for t, x in zip(tails[b], (k, v)))
            have = tails[b][0].shape[0] - counts[b]
            want, tol, _, _ = attend64(q[rows], np.concatenate([K, tails[b][0]]), np.concatenate([V, tails[b][1]]),
                                       count + have + 1 + np.arange(counts[b]), c.scale, kind == F16)
            assert (np.abs(out[b, :counts[b]] - want) <= tol).all()
        logits = out[:, 0].reshape(5, -1).astype(np.float32) @ W
        tokens, logp = sampling.sample(logits, c.rng.random(5), temperature=0.8, top_p=0.9)
        assert ((tokens >= 0) & (tokens < 50)).all() and (logp <= 0).all()
    m.reset()
    assert m.count == 0 and m.next == 0
    q, k, v = c.rows(2)
    out = m.attend(q, k, v)
    want, tol, _, _ = attend64(q, k, v, [1, 2], c.scale, kind == F16)
    assert (np.abs(out - want) <= tol).all()
    with pytest.raises(ValueError):
        m.attend(*c.rows(299))
    with pytest.raises(ValueError):
        m.attend(q, k[:1], v)
    with pytest.raises(ValueError):
        m.evict(2**32 + 3)
