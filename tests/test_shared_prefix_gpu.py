"""Attention of drafts behind a shared prefix (trx_attn_shared) against its definition in 64 bits, draft by
draft over the rows that each sees, and what it refuses.

Tolerance, per output element, from the arithmetic (A = sum of p |v| over the seen keys, S = the largest sum over
dims of scale |q k|, N seen keys): a score is off by S (2^-21 + head_dim 2^-24) (the query's two planes or fp16
itself, fp32 sums), its exponent by 2^-21 more, which moves a probability and the total by twice that; the sums and
the parts' join add N 2^-24 A; the probabilities' planes 2^-22 A in fp32, half a step (2^-11 A) in fp16, where those
below fp16's steps lose 2^-32 max |v| each, and the result is rounded by 2^-11 of itself. The gate multiplies by a
value of error 2^-21."""

import ctypes

import numpy as np
import pytest

from trixium_amd import _lib, layout as L

F32, F16 = L.KIND_F32, L.KIND_F16
DT = {F32: np.float32, F16: np.float16}


def attend64(q, K, V, lim, scale, half, gate=None):
    """(outputs, tolerances, probabilities, their tolerances) [rows, heads, ...] of queries [rows, heads, hd] over
    K, V [N, kv, hd], row r seeing the first lim[r] keys; probabilities [rows, heads, N]."""
    rows, heads, hd = q.shape
    N, kv = K.shape[:2]
    rep = heads // kv
    out, tol = np.empty((rows, heads, hd)), np.empty((rows, heads, hd))
    prob, ptol = np.zeros((rows, heads, N)), np.zeros((rows, heads, N))
    seen = np.repeat(np.arange(N)[None] < np.asarray(lim)[:, None], rep, axis=0)
    for g in range(kv):
        hs = slice(g * rep, (g + 1) * rep)
        qd = q[:, hs].astype(np.float64).reshape(rows * rep, hd)
        Kg, Vg = K[:, g].astype(np.float64), V[:, g].astype(np.float64)
        Kg, Vg = np.where(seen.any(0)[:, None], Kg, 0), np.where(seen.any(0)[:, None], Vg, 0)
        s = np.where(seen, float(scale) * (qd @ Kg.T), -np.inf)
        S = np.where(seen, float(scale) * (np.abs(qd) @ np.abs(Kg).T), 0).max(1)[:, None]
        n = seen.sum(1)[:, None]
        p = np.exp(s - s.max(1)[:, None])
        p /= p.sum(1)[:, None]
        A, o = p @ np.abs(Vg), p @ Vg
        rel = 2 * (S * (2.0**-21 + hd * 2.0**-24) + 2.0**-21) + n * 2.0**-24
        e = A * (rel + 2.0**-22)
        if half:
            e += A * 2.0**-11 + n * 2.0**-32 * np.abs(Vg).max()
        if gate is not None:
            sg = 1.0 / (1.0 + np.exp(-gate[:, hs].astype(np.float64).reshape(o.shape)))
            o, e = o * sg, e * sg + np.abs(o) * 2.0**-21
        if half:
            e += np.abs(o) * 2.0**-11 + 2.0**-25
        out[:, hs], tol[:, hs] = o.reshape(rows, rep, hd), e.reshape(rows, rep, hd)
        # (A probability again from its score: the score times log2 e and the reference, each rounded once.)
        prob[:, hs], ptol[:, hs] = (a.reshape(rows, rep, N) for a in (p, p * (rel + S * 2.0**-22 + 2.0**-21)))
    return out, tol, prob, ptol


class Drafts:
    def __init__(self, heads, kv, hd, batch, prefix, tail_slots, kind=F32, seed=0, scale=None, prefix_slots=None):
        self.heads, self.kv, self.hd, self.batch, self.prefix = heads, kv, hd, batch, prefix
        self.tail_slots, self.kind = tail_slots, kind
        self.prefix_slots = prefix if prefix_slots is None else prefix_slots
        self.scale = np.float32(1.0 / np.sqrt(hd) if scale is None else scale)
        self.rng = np.random.default_rng(seed)
        self.kp, self.vp = (self.rng.standard_normal((kv, self.prefix_slots, hd)).astype(np.float16) for _ in range(2))
        self.kt, self.vt = (self.rng.standard_normal((batch, kv, tail_slots, hd)).astype(np.float16) for _ in range(2))

    def rows(self, n, size=1.0):
        r, b = self.rng, self.batch
        q = (1.5 * size * r.standard_normal((b * n, self.heads, self.hd))).astype(DT[self.kind])
        k, v = (r.standard_normal((b * n, self.kv, self.hd)).astype(np.float16) for _ in range(2))
        return q, k, v

    def shape(self, **kw):
        q, kv = self.heads * self.hd, self.kv * self.hd
        d = dict(kind=self.kind, n_head=self.heads, n_kv_head=self.kv, head_dim=self.hd, prefix_slots=self.prefix_slots,
                 tail_slots=self.tail_slots, q_stride=q, kv_stride=kv, out_stride=q, gate_stride=q, gate_head_stride=self.hd,
                 scale=float(self.scale))
        d.update(kw)
        return _lib.AttnSharedShape(**d)

    def expect(self, q, k, v, lengths, counts, gate=None, fill=77):
        """Outputs (rows that do not count: fill), tolerances and the tails afterwards."""
        n = q.shape[0] // self.batch
        out, tol = np.full(q.shape, fill, np.float64), np.zeros(q.shape)
        kt, vt = self.kt.copy(), self.vt.copy()
        for b in range(self.batch):
            have, c = int(lengths[b]), int(counts[b])
            if not (0 < c <= n and 0 <= have <= self.tail_slots - c):
                continue
            at = slice(b * n, b * n + c)
            K, V = (np.concatenate([p[:, :self.prefix], t[b][:, :have], x[at].transpose(1, 0, 2)], axis=1).transpose(1, 0, 2)
                    for p, t, x in ((self.kp, self.kt, k), (self.vp, self.vt, v)))
            lim = self.prefix + have + 1 + np.arange(c)
            out[at], tol[at], _, _ = attend64(q[at], K, V, lim, self.scale, self.kind == F16, None if gate is None else gate[at])
            kt[b][:, have:have + c], vt[b][:, have:have + c] = k[at].transpose(1, 0, 2), v[at].transpose(1, 0, 2)
        return out, tol, kt, vt

    def call(self, q, k, v, lengths, counts=None, gate=None, shape=None, stream=None, n=None):
        """One call on device copies; (out, K tails, V tails) back."""
        B, shape = _lib.DeviceBuffer, shape or self.shape()
        n = k.shape[0] // self.batch if n is None else n
        bufs = [B.from_array(a) for a in (q, k, v, self.kp, self.vp, self.kt, self.vt)]
        lb, cb, gb = (B.from_array(np.asarray(a, d)) if a is not None else None
                      for a, d in ((lengths, np.int32), (counts, np.int32), (gate, DT[self.kind])))
        out = B.from_array(np.full(self.batch * n * shape.out_stride, 77, DT[self.kind]))
        work = B(geometry(shape, self.batch, n, self.prefix))
        _lib.synchronize()
        _lib.call("trx_attn_shared", ctypes.byref(shape), self.batch, n, self.prefix, lb.ptr, cb.ptr if cb else None,
                  *(b.ptr for b in bufs), gb.ptr if gb else None, out.ptr, work.ptr, stream)
        _lib.synchronize(stream)
        return (out.download(DT[self.kind], self.batch * n * shape.out_stride).reshape(self.batch * n, shape.out_stride),
                bufs[5].download(np.float16, self.kt.size).reshape(self.kt.shape),
                bufs[6].download(np.float16, self.vt.size).reshape(self.vt.shape))

    def check(self, n, lengths, counts=None, gated=False):
        q, k, v = self.rows(n)
        gate = self.rng.standard_normal(q.shape).astype(DT[self.kind]) if gated else None
        out, kt, vt = self.call(q, k, v, lengths, counts, gate)
        want, tol, ek, ev = self.expect(q, k, v, lengths, [n] * self.batch if counts is None else counts, gate)
        err = np.abs(out.reshape(want.shape).astype(np.float64) - want)
        assert (err <= tol).all(), (float(np.nanmax(err / np.maximum(tol, 1e-300))), np.argwhere(~(err <= tol))[:4].tolist())
        assert np.array_equal(kt.view(np.uint16), ek.view(np.uint16)) and np.array_equal(vt.view(np.uint16), ev.view(np.uint16))
        return float((err[tol > 0] / tol[tol > 0]).max(initial=0))


def geometry(shape, batch, n, prefix):
    size = ctypes.c_size_t()
    _lib.call("trx_attn_shared_geometry", ctypes.byref(shape), batch, n, prefix, ctypes.byref(size))
    return size.value


# Refusals (no GPU) -----------------------------------------------------------------------------------


@pytest.mark.parametrize("change,what", [
    (dict(head_dim=96), b"head_dim"), (dict(n_kv_head=0), b"n_head"), (dict(n_head=5), b"n_head"),
    (dict(n_head=2048, q_stride=2048 * 64, out_stride=2048 * 64), b"heads"),
    (dict(prefix_slots=-1), b"slots"), (dict(prefix_slots=(1 << 30) + 1), b"slots"), (dict(tail_slots=0), b"slots"),
    (dict(tail_slots=(1 << 30) + 1), b"slots"), (dict(tail_slots=(1 << 29) + 1), b"slots"),
    (dict(prefix_slots=(1 << 29) + 1), b"slots"), (dict(prefix_slots=39), b"prefix"), (dict(scale=0.0), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale"), (dict(q_stride=252), b"q_stride"),
    (dict(q_stride=258), b"q_stride"), (dict(kv_stride=132), b"kv_stride"), (dict(kv_stride=(1 << 22) + 8), b"kv_stride"),
    (dict(out_stride=255), b"out_stride"), (dict(kind=L.KIND_Q8), b"kind")])
def test_geometry_refuses(change, what):
    c = Drafts(4, 2, 64, 3, 40, 16)
    lib, size, fake = _lib.lib(), ctypes.c_size_t(), ctypes.c_void_p(256)
    shape = c.shape(**change)
    assert lib.trx_attn_shared_geometry(ctypes.byref(shape), 3, 1, 40, ctypes.byref(size)) == _lib.TRX_E_INVALID
    assert what in lib.trx_last_error(), lib.trx_last_error()
    assert lib.trx_attn_shared(ctypes.byref(shape), 3, 1, 40, fake, None, *[fake] * 7, None, fake, fake, None) == _lib.TRX_E_INVALID
    assert what in lib.trx_last_error(), lib.trx_last_error()


def test_call_refuses_bad_arguments():
    c = Drafts(4, 2, 64, 3, 40, 16)
    lib, shape, fake, odd = _lib.lib(), c.shape(), ctypes.c_void_p(256), ctypes.c_void_p(264)
    names = ("lengths", "counts", "q", "k", "v", "kp", "vp", "kt", "vt", "gate", "out", "work")

    def call(batch=3, n=1, prefix=40, sh=shape, **kw):
        a = dict.fromkeys(names, fake) | dict(counts=None, gate=None) | kw
        return lib.trx_attn_shared(ctypes.byref(sh), batch, n, prefix, *(a[x] for x in names), None)

    bad = [(dict(batch=-1), b"rows"), (dict(n=-1), b"rows"), (dict(batch=1 << 20, n=3), b"rows"), (dict(prefix=-1), b"prefix"),
           (dict(prefix=41), b"prefix"), (dict(lengths=ctypes.c_void_p(258)), b"aligned"), (dict(counts=ctypes.c_void_p(258)), b"aligned"),
           (dict(gate=fake, sh=c.shape(gate_head_stride=32)), b"gate"), (dict(gate=fake, sh=c.shape(gate_stride=192)), b"gate")]
    bad += [({x: None}, b"null") for x in names if x not in ("counts", "gate")]
    bad += [({x: odd}, b"aligned") for x in names if x not in ("lengths", "counts")]
    for kw, what in bad:
        assert call(**kw) == _lib.TRX_E_INVALID, kw
        assert what in lib.trx_last_error(), (kw, lib.trx_last_error())
    assert call(batch=0, q=None) == _lib.TRX_OK and call(n=0, q=None) == _lib.TRX_OK    # nothing to do
    assert lib.trx_attn_shared(None, 3, 1, 40, *[fake] * 12, None) == _lib.TRX_E_INVALID
    assert lib.trx_attn_shared_geometry(ctypes.byref(shape), 3, 1, 40, None) == _lib.TRX_E_INVALID


@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("heads,kv,hd", [(32, 8, 128), (24, 4, 256), (16, 8, 128), (4, 2, 64), (40, 1, 64)])
def test_the_workspace_grows_with_the_call(heads, kv, hd, kind):
    """A size holds every smaller call: it never falls as the drafts, the rows or the prefix grow."""
    shape = Drafts(heads, kv, hd, 1, 1, 1, kind).shape(prefix_slots=1 << 20, tail_slots=5000)
    for sizes in ([geometry(shape, b, 1, 4000) for b in range(1, 400)], [geometry(shape, 7, n, 4000) for n in range(1, 400)],
                  [geometry(shape, 7, 2, p) for p in list(range(0, 3000, 7)) + [1 << 20]]):
        assert sizes == sorted(sizes)


def test_python_form_refuses():
    from trixium_amd.attention import KVMass, SharedPrefix
    k = np.zeros((2, 5, 64), np.float16)
    for kw in (dict(kind=L.KIND_Q8), dict(batch=0), dict(tail_slots=2**32 + 4), dict(batch=2**32 + 1)):
        with pytest.raises(ValueError):
            SharedPrefix(**{**dict(n_head=4, n_kv_head=2, head_dim=64, k=k, v=k, batch=2, tail_slots=8), **kw})
    with pytest.raises(ValueError):
        SharedPrefix(4, 2, 64, k, k[:, :4], 2, 8)
    with pytest.raises(ValueError):
        SharedPrefix(4, 2, 64, k[:1], k[:1], 2, 8)
    with pytest.raises(_lib.TrxError):
        SharedPrefix(4, 2, 96, np.zeros((2, 5, 96)), np.zeros((2, 5, 96)), 2, 8)
    with pytest.raises(ValueError):
        KVMass(4, 2, 64, 2**32 + 8)


# Results (GPU) ---------------------------------------------------------------------------------------


GEOMETRIES = [  # heads, kv heads, head dim
    (4, 2, 64), (6, 1, 256), (4, 4, 128), (16, 1, 64), (5, 1, 128), (8, 2, 256), (33, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("geo", GEOMETRIES, ids=str)
def test_head_shapes(geo, kind):
    for batch, prefix, n in ((3, 45, 1), (9, 131, 1), (2, 64, 5), (1, 1, 1), (5, 0, 2)):
        c = Drafts(*geo, batch=batch, prefix=prefix, tail_slots=50, kind=kind, seed=1)
        lengths = c.rng.integers(0, 50 - n + 1, batch)
        lengths[0] = 0
        print(geo, kind, batch, prefix, n, lengths, flush=True)
        print(f"worst error {c.check(n, lengths, gated=n == 1):.3f} of the tolerance")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("batch,prefix,tail,n", [(1, 5000, 0, 1), (40, 700, 3, 1), (70, 333, 40, 1), (7, 900, 600, 3),
                                                 (3, 31, 33, 40), (2, 2000, 100, 70), (160, 64, 10, 1), (33, 129, 64, 4)])
def test_batches_and_lengths(batch, prefix, tail, n, kind):
    """From one draft to more than a block's columns; prefixes and tails that are split over blocks and that end
    inside a tile; drafts of all lengths, empty and full."""
    c = Drafts(8, 2, 128, batch, prefix, tail + n, kind=kind, seed=2)
    lengths = c.rng.integers(0, tail + 1, batch)
    lengths[0], lengths[-1] = 0, tail
    c.check(n, lengths)
    c.check(n, lengths, counts=c.rng.integers(0, n + 1, batch), gated=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,heads,kv,hd,batch,n", [(F32, 32, 4, 64, 50, 1), (F16, 32, 4, 64, 50, 1), (F32, 64, 2, 128, 9, 2),
                                                      (F16, 64, 2, 128, 9, 2), (F32, 24, 2, 256, 30, 1), (F16, 24, 2, 256, 30, 1),
                                                      (F32, 32, 2, 256, 3, 20), (F16, 32, 2, 256, 3, 20), (F32, 32, 2, 64, 3, 20),
                                                      (F16, 32, 2, 128, 3, 20), (F32, 32, 2, 128, 3, 37)])
def test_many_columns(kind, heads, kv, hd, batch, n):
    """Prefixes and tails of long turns that fill wide blocks of columns, with a hidden NaN behind each."""
    c = Drafts(heads, kv, hd, batch, 777, 260, kind=kind, seed=3, prefix_slots=800)
    c.kp[:, 777:], c.vp[:, 777:] = np.nan, np.inf
    lengths = c.rng.integers(0, 260 - n + 1, batch)
    for b in range(batch):
        c.kt[b][:, lengths[b]:], c.vt[b][:, lengths[b]:] = np.nan, -np.inf
    c.check(n, lengths, gated=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
def test_drafts_that_take_no_part(kind):
    """Counts of 0 and out of range, lengths negative and past the slots: rows and tails stay, whatever q, k, v and
    gate hold there; the others' results are what they are alone."""
    c = Drafts(4, 2, 64, 9, 100, 20, kind=kind, seed=4)
    lengths = np.array([3, -1, 20, 18, 5, 0, 2**31 - 1, -2**31, 17], np.int32)
    counts = np.array([3, 2, 1, 3, 0, 4, 1, 3, 3], np.int32)      # n is 3: the sixth is out of range
    q, k, v = c.rows(3)
    gate = c.rng.standard_normal(q.shape).astype(DT[kind])
    for b in range(9):
        behind = slice(b * 3 + (3 if b in (0, 8) else 0), b * 3 + 3)
        for a in (q, k, v, gate):
            a[behind] = np.nan
    out, kt, vt = c.call(q, k, v, lengths, counts, gate)
    want, tol, ek, ev = c.expect(q, k, v, lengths, counts, gate)
    assert (np.abs(out.reshape(want.shape) - want) <= tol).all()
    assert (want[3:24] == 77).all() and (want[:3] != 77).all() and (want[24:] != 77).all()
    assert np.array_equal(kt.view(np.uint16), ek.view(np.uint16)) and np.array_equal(vt.view(np.uint16), ev.view(np.uint16))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("batch,n", [(3, 2), (60, 1)])
def test_infinities_and_nans_stay_where_they_are_seen(kind, batch, n):
    """A value of the prefix that is infinite shows in every draft, one of a tail in that draft alone, one of a new row
    in the rows from it on; a NaN query in its own row."""
    c = Drafts(4, 2, 64, batch, 150, 70, kind=kind, seed=5)
    lengths = np.full(batch, 60)
    c.vp[0, 17, 3] = np.inf
    c.vt[1][1, 9, 5] = -np.inf
    q, k, v = c.rows(n)
    v[2 * n + n - 1, 0, 7] = np.nan
    q[0, 3, 0] = np.nan
    out, _, _ = c.call(q, k, v, lengths)
    out = out.reshape(-1, 4, 64)
    bad = np.zeros(out.shape, bool)
    assert (out[:, :2, 3] == np.inf).all()
    assert (out[n:2 * n, 2:, 5] == -np.inf).all()
    assert np.isnan(out[3 * n - 1, :2, 7]).all() and np.isnan(out[0, 3]).all()
    bad[:, :2, 3] = bad[n:2 * n, 2:, 5] = bad[3 * n - 1, :2, 7] = bad[0, 3] = True
    c.vp[0, 17, 3] = c.vt[1][1, 9, 5] = v[2 * n + n - 1, 0, 7] = q[0, 3, 0] = 0
    want, tol, _, _ = c.expect(q, k, v, lengths, [n] * batch)
    assert (np.abs(out - want)[~bad] <= tol[~bad]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4])
def test_queries_of_any_magnitude(size):
    c = Drafts(4, 2, 64, 5, 90, 20, seed=6, scale=0.125 / size if size > 1 else 0.125)
    q, k, v = c.rows(2, size)
    lengths = [0, 3, 18, 9, 1]
    out, _, _ = c.call(q, k, v, lengths)
    want, tol, _, _ = c.expect(q, k, v, lengths, [2] * 5)
    assert (np.abs(out.reshape(want.shape) - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("batch,n", [(3, 2), (40, 1), (2, 40)])
def test_strides(kind, batch, n):
    """Rows inside wider ones (a fused projection's), gates beside each head; nothing else is written."""
    c = Drafts(4, 2, 64, batch, 100, 60, kind=kind, seed=7, prefix_slots=130)
    q, k, v = c.rows(n)
    gate = c.rng.standard_normal(q.shape).astype(DT[kind])
    wide = np.full((batch * n, 4 * 64 + 16), 9, DT[kind])
    wide[:, :256] = q.reshape(batch * n, -1)
    kv = np.full((2, batch * n, 2 * 64 + 8), 9, np.float16)
    kv[0, :, :128], kv[1, :, :128] = k.reshape(batch * n, -1), v.reshape(batch * n, -1)
    gw = np.full((batch * n, 4, 128), 9, DT[kind])
    gw[:, :, :64] = gate
    lengths = c.rng.integers(0, 60 - n + 1, batch)
    shape = c.shape(q_stride=272, kv_stride=136, out_stride=260, gate_stride=512, gate_head_stride=128)
    out, kt, _ = c.call(wide, kv[0], kv[1], lengths, gate=gw, shape=shape, n=n)
    want, tol, ek, _ = c.expect(q, k, v, lengths, [n] * batch, gate)
    assert (np.abs(out[:, :256].reshape(want.shape) - want) <= tol).all()
    assert (out[:, 256:] == 77).all() and np.array_equal(kt, ek)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
@pytest.mark.parametrize("batch,n", [(5, 1), (64, 1), (3, 33)])
def test_repeated_calls_give_the_same_bits(kind, batch, n):
    c = Drafts(32, 8, 128, batch, 1500, 300, kind=kind, seed=8)
    q, k, v = c.rows(n)
    lengths = c.rng.integers(0, 300 - n + 1, batch)
    first = c.call(q, k, v, lengths)
    for _ in range(3):
        for a, b in zip(first, c.call(q, k, v, lengths)):
            assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.gpu
def test_a_draft_does_not_depend_on_the_others():
    """A draft's outputs are those that the window attention gives over its rows in one cache."""
    c = Drafts(8, 2, 128, 6, 300, 90, seed=9)
    q, k, v = c.rows(1)
    lengths = np.array([0, 5, 89, 31, 32, 33])
    out, _, _ = c.call(q, k, v, lengths)
    from trixium_amd.attention import KVRing
    for b in range(6):
        ring = KVRing(8, 2, 128, 500, pin=0)
        K, V = (np.concatenate([p, t[b][:, :lengths[b]]], axis=1).transpose(1, 0, 2) for p, t in ((c.kp, c.kt), (c.vp, c.vt)))
        ring.attend(np.zeros((K.shape[0], 8, 128)), K, V)
        want = ring.attend(q[b:b + 1], k[b:b + 1], v[b:b + 1])
        _, tol, _, _ = c.expect(q, k, v, lengths, [1] * 6)
        assert (np.abs(out[b].reshape(8, 128) - want[0]) <= 2 * tol[b]).all()


@pytest.mark.gpu
def test_captured_graph_follows_lengths_and_counts():
    """A captured call replayed with the lengths and counts that the device holds then, on a stream of its own,
    with other work between the replays."""
    c = Drafts(4, 2, 64, 5, 130, 40, seed=10)
    B, shape, n = _lib.DeviceBuffer, c.shape(), 3
    s = ctypes.c_void_p()
    _lib.call("trx_stream_create", ctypes.byref(s))
    kp, vp, kt, vt = (B.from_array(a) for a in (c.kp, c.vp, c.kt, c.vt))
    qb, kb, vb, out, lb, cb = (B(x) for x in (5 * n * 256 * 4, 5 * n * 128 * 2, 5 * n * 128 * 2, 5 * n * 256 * 4, 20, 20))
    work = B(geometry(shape, 5, n, 130))
    _lib.synchronize()
    _lib.call("trx_graph_begin", s)
    _lib.call("trx_attn_shared", ctypes.byref(shape), 5, n, 130, lb.ptr, cb.ptr, qb.ptr, kb.ptr, vb.ptr, kp.ptr, vp.ptr, kt.ptr,
              vt.ptr, None, out.ptr, work.ptr, s)
    ex = ctypes.c_void_p()
    _lib.call("trx_graph_end", s, ctypes.byref(ex))
    lengths = np.array([0, 1, 30, 40, 7])
    for rep in range(4):
        counts = c.rng.integers(0, n + 1, 5)
        q, k, v = c.rows(n)
        for b, a in ((qb, q), (kb, k), (vb, v), (lb, lengths.astype(np.int32)), (cb, counts.astype(np.int32)),
                     (out, np.full(q.shape, 77, np.float32))):
            b.upload(a, s)
        _lib.call("trx_graph_launch", ex, s)
        _lib.synchronize(s)
        want, tol, ek, ev = c.expect(q, k, v, lengths, counts)
        assert (np.abs(out.download(np.float32, q.size).reshape(q.shape) - want) <= tol).all(), rep
        assert np.array_equal(kt.download(np.float16).reshape(ek.shape), ek)
        c.kt, c.vt = ek, ev
        took = (counts > 0) & (lengths + counts <= 40)
        lengths = lengths + np.where(took, counts, 0)
        Drafts(4, 2, 64, 4, 50, 10, seed=20 + rep).check(2, [0, 3, 8, 1])     # an eager call between the replays
    _lib.call("trx_graph_destroy", ex)
    _lib.call("trx_stream_destroy", s)


@pytest.mark.gpu
def test_one_workspace_for_smaller_calls():
    """Sized for the largest call, used by smaller ones: nothing is written behind it."""
    guard, B = 1 << 20, _lib.DeviceBuffer
    big = Drafts(32, 8, 128, 48, 3000, 64, seed=11)
    size = geometry(big.shape(), 48, 2, 3000)
    work = B.from_array(np.full(size + guard, 0xA5, np.uint8))
    for batch, n, prefix in ((48, 2, 3000), (48, 1, 3000), (17, 2, 2999), (1, 1, 3000), (33, 1, 100), (2, 2, 0)):
        c = Drafts(32, 8, 128, batch, prefix, 64, seed=12, prefix_slots=3000)
        q, k, v = c.rows(n)
        lengths = c.rng.integers(0, 60, batch)
        want = c.call(q, k, v, lengths)
        bufs = [B.from_array(a) for a in (q, k, v, c.kp, c.vp, c.kt, c.vt)]
        lb, out = B.from_array(lengths.astype(np.int32)), B(q.nbytes)
        _lib.call("trx_attn_shared", ctypes.byref(c.shape()), batch, n, prefix, lb.ptr, None, *(b.ptr for b in bufs), None, out.ptr,
                  work.ptr, None)
        _lib.synchronize()
        assert np.array_equal(out.download(np.uint8, q.nbytes), want[0].view(np.uint8).ravel()), (batch, n, prefix)
        assert (work.download(np.uint8, guard, offset=size) == 0xA5).all(), (batch, n, prefix)


@pytest.mark.gpu
def test_offsets_past_four_gib():
    """The second kv head's prefix and the last draft's tail lie 4 GiB into their buffers."""
    hd, kv, B = 128, 2, _lib.DeviceBuffer
    slots, tail = (1 << 24) + 64, 1 << 22                       # 4 GiB a kv head's prefix; 2 GiB a draft's tail
    c = Drafts(4, kv, hd, 3, 100, 50, seed=13)
    kp, vp, kt, vt = B(2 * kv * slots * hd), B(2 * kv * slots * hd), B(2 * 3 * kv * tail * hd), B(2 * 3 * kv * tail * hd)
    lengths = np.array([0, 50, 41], np.int32)
    for g in range(kv):
        for buf, a in ((kp, c.kp), (vp, c.vp)):
            buf.upload(a[g], offset=2 * g * slots * hd)
        for b in range(3):
            for buf, a in ((kt, c.kt), (vt, c.vt)):
                buf.upload(a[b, g], offset=2 * (b * kv + g) * tail * hd)
    q, k, v = c.rows(1)
    shape = c.shape(prefix_slots=slots, tail_slots=tail)
    qb, kb, vb, lb = (B.from_array(a) for a in (q, k, v, lengths))
    out, work = B(q.nbytes), B(geometry(shape, 3, 1, 100))
    _lib.call("trx_attn_shared", ctypes.byref(shape), 3, 1, 100, lb.ptr, None, qb.ptr, kb.ptr, vb.ptr, kp.ptr, vp.ptr, kt.ptr, vt.ptr,
              None, out.ptr, work.ptr, None)
    _lib.synchronize()
    c.tail_slots = 51                                            # (the definition over the rows alone)
    c.kt, c.vt = (np.pad(a, ((0, 0), (0, 0), (0, 1), (0, 0))) for a in (c.kt, c.vt))
    want, tol, _, _ = c.expect(q, k, v, lengths, [1] * 3)
    assert (np.abs(out.download(np.float32, q.size).reshape(want.shape) - want) <= tol).all()
    for b in range(3):
        for g in range(kv):
            at = 2 * ((b * kv + g) * tail + int(lengths[b])) * hd
            assert np.array_equal(kt.download(np.float16, hd, offset=at), k[b, g])
            assert np.array_equal(vt.download(np.float16, hd, offset=at), v[b, g])


@pytest.mark.gpu
def test_shared_prefix_object():
    from trixium_amd.attention import SharedPrefix
    c = Drafts(4, 2, 64, 4, 70, 30, seed=14)
    d = SharedPrefix(4, 2, 64, c.kp, c.vp, 4, 30)
    c.kt[:], c.vt[:] = 0, 0
    lengths = np.zeros(4, int)
    for n, counts in ((1, None), (5, [5, 0, 2, 3]), (0, None), (3, None), (1, [1, 1, 0, 1])):
        q, k, v = c.rows(n)
        shaped = [a.reshape(4, n, *a.shape[1:]) for a in (q, k, v)]
        out = d.attend(*shaped, counts=counts)
        if n == 0:
            continue
        took = np.array([n] * 4 if counts is None else counts)
        want, tol, c.kt, c.vt = c.expect(q, k, v, lengths, took, fill=0)
        assert (np.abs(out.reshape(want.shape) - want) <= tol).all()
        lengths = lengths + took
        assert np.array_equal(d.lengths, lengths)
    for b in range(4):
        assert all(np.array_equal(x, t[b][:, :lengths[b]]) for x, t in zip(d.rows(b), (c.kt, c.vt)))
    d.cut([1, 0, 3, lengths[3]])
    lengths = np.array([1, 0, 3, lengths[3]])
    q, k, v = c.rows(2)
    out = d.attend(*(a.reshape(4, 2, *a.shape[1:]) for a in (q, k, v)))
    want, tol, _, _ = c.expect(q, k, v, lengths, [2] * 4)
    assert (np.abs(out.reshape(want.shape) - want) <= tol).all()
    for kw in (dict(counts=[3, 0, 0, 0]), dict(counts=[0.5] * 4), dict(counts=[1] * 3)):
        with pytest.raises(ValueError):
            d.attend(*(a.reshape(4, 2, *a.shape[1:]) for a in (q, k, v)), **kw)
    with pytest.raises(ValueError):
        d.attend(np.zeros((4, 40, 4, 64)), np.zeros((4, 40, 2, 64)), np.zeros((4, 40, 2, 64)))     # past the slots
    with pytest.raises(ValueError):
        d.cut([9] * 4)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,batch,n", [(32, 8, 128, 8, 1), (6, 1, 256, 5, 1), (4, 2, 64, 4, 4), (8, 8, 128, 3, 5)])
def test_few_columns_with_fp16_queries_round_once(heads, kv, hd, batch, n):
    """Up to 32 columns' fp16 outputs are the fp32 result rounded: x + d rounds to a value whose distance from x is at most
    that of x rounded, plus 2 d. Queries with one element leave a score no sum over dims: d is the fp32 tolerance
    without it."""
    c = Drafts(heads, kv, hd, batch, 1900, 60, F16, seed=15, scale=1.0)
    q, k, v = c.rows(n)
    q[..., 1:] = 0
    lengths = c.rng.integers(0, 60 - n + 1, batch)
    out, _, _ = c.call(q, k, v, lengths)
    out = out.reshape(batch * n, heads, hd).astype(np.float64)
    for r in range(batch * n):
        b, i = divmod(r, n)
        K, V = (np.concatenate([p, t[b][:, :lengths[b]], x[b * n:b * n + i + 1].transpose(1, 0, 2)], axis=1).astype(np.float64)
                for p, t, x in ((c.kp, c.kt, k), (c.vp, c.vt, v)))
        for h in range(heads):
            g = h * kv // heads
            s = K[g, :, 0] * float(q[r, h, 0])
            p = np.exp(s - s.max())
            p /= p.sum()
            x, d = p @ V[g], (p @ np.abs(V[g])) * (2 * (np.abs(s).max() + 1) * 2.0**-21 + s.size * 2.0**-24 + 2.0**-22)
            assert (np.abs(out[r, h] - x) <= np.abs(x.astype(np.float16).astype(np.float64) - x) + 2 * d).all(), (r, h)


@pytest.mark.gpu
def test_two_calls_at_once():
    """Two batches over one prefix on streams of their own, each with its workspace: the bits of each alone."""
    c = Drafts(32, 8, 128, 12, 3000, 90, seed=16)
    B, shape = _lib.DeviceBuffer, c.shape()
    calls = []
    kp, vp = B.from_array(c.kp), B.from_array(c.vp)
    for _ in range(2):
        q, k, v = c.rows(2)
        lengths = c.rng.integers(0, 89, 12)
        want = c.call(q, k, v, lengths)
        s = ctypes.c_void_p()
        _lib.call("trx_stream_create", ctypes.byref(s))
        bufs = [B.from_array(a) for a in (lengths.astype(np.int32), q, k, v, c.kt, c.vt)]
        calls.append((want, s, bufs, B(q.nbytes), B(geometry(shape, 12, 2, 3000))))
    _lib.synchronize()
    for _ in range(3):
        for want, s, (lb, qb, kb, vb, kt, vt), out, work in calls:
            _lib.call("trx_attn_shared", ctypes.byref(shape), 12, 2, 3000, lb.ptr, None, qb.ptr, kb.ptr, vb.ptr, kp.ptr, vp.ptr,
                      kt.ptr, vt.ptr, None, out.ptr, work.ptr, s)
        for want, s, bufs, out, work in calls:
            _lib.synchronize(s)
            assert np.array_equal(out.download(np.uint8, out.nbytes), want[0].view(np.uint8).ravel())
    for _, s, *_ in calls:
        _lib.call("trx_stream_destroy", s)
