"""Drafts behind a shared prefix (trx_attn_shared) and attention with masses (trx_attn_mass) at sizes whose columns fill
wide blocks, waves of two or four columns, against their definition in 64 bits; and masses of long chunks whose rows and
position are on the device. Tolerances: test_shared_prefix_gpu.py's and test_kv_mass_gpu.py's."""

import ctypes
import os
import subprocess

import numpy as np
import pytest

from trixium_amd import _lib, layout as L
from test_kv_mass_gpu import DT, Cache, geometry
from test_shared_prefix_gpu import Drafts

F32, F16 = L.KIND_F32, L.KIND_F16

# What the calls below are cut into: waves of columns (1: the kernel for few columns, 0: no prefix) of the prefix and of
# the tails, and for masses whether parts of the columns are added up.
SHARED = [  # kind, heads, kv heads, head dim, drafts, rows each, prefix, tail slots; waves of the prefix and of the tails
    (F32, 32, 8, 128, 48, 2, 3000, 64, 4, 1), (F16, 32, 8, 128, 48, 2, 3000, 64, 4, 1), (F32, 32, 8, 128, 12, 7, 6001, 207, 4, 1),
    (F16, 32, 8, 128, 12, 7, 6001, 207, 4, 1), (F32, 32, 8, 128, 3, 128, 500, 578, 4, 2), (F32, 64, 8, 128, 4, 64, 300, 300, 2, 2),
    (F16, 64, 8, 128, 4, 64, 300, 300, 4, 4), (F32, 24, 4, 256, 4, 100, 300, 400, 4, 4), (F16, 24, 4, 256, 4, 100, 300, 400, 4, 4),
    (F32, 24, 4, 256, 2, 200, 300, 300, 4, 2), (F16, 24, 4, 256, 2, 200, 300, 300, 4, 2), (F32, 64, 8, 64, 60, 2, 2000, 64, 4, 1),
    (F16, 64, 8, 64, 60, 2, 2000, 64, 4, 1), (F32, 64, 8, 64, 3, 128, 500, 400, 4, 4), (F16, 64, 8, 64, 3, 128, 500, 400, 4, 4),
    (F32, 32, 4, 64, 2, 200, 100, 800, 1, 2), (F16, 32, 4, 64, 2, 400, 100, 800, 1, 4), (F32, 32, 8, 128, 2, 300, 0, 900, 0, 4)]
MASS = [  # kind, heads, kv heads, head dim, rows, rows there; waves, several parts
    (F32, 32, 8, 128, 700, 800, 4, True), (F16, 32, 8, 128, 700, 800, 4, True), (F32, 32, 8, 128, 300, 300, 2, True),
    (F16, 32, 8, 128, 300, 300, 2, True), (F32, 16, 8, 128, 300, 800, 2, False), (F16, 16, 8, 128, 300, 800, 4, False),
    (F32, 24, 4, 256, 101, 1700, 4, True), (F16, 24, 4, 256, 101, 1700, 4, True), (F32, 24, 4, 256, 512, 0, 2, True),
    (F16, 24, 4, 256, 400, 100, 2, True), (F32, 64, 8, 64, 300, 900, 4, True), (F16, 64, 8, 64, 300, 900, 4, True),
    (F32, 64, 8, 64, 256, 500, 2, True), (F16, 32, 4, 64, 380, 500, 2, True)]
CAPTURED = [  # kind, heads, kv heads, head dim, rows, slots; waves, several parts
    (F32, 8, 1, 128, 200, 1500, 1, True), (F32, 4, 2, 64, 200, 1500, 1, False), (F32, 32, 8, 128, 160, 1500, 2, False),
    (F16, 24, 4, 256, 120, 1000, 2, True), (F16, 32, 8, 128, 160, 1500, 4, False)]
SLACK = 17                                          # slots behind the rows of MASS


def test_the_sizes_are_cut_as_they_are_meant(tmp_path):
    """The cut of every call below (the planner alone, no GPU): a changed estimate must not leave the wide blocks untested."""
    (tmp_path / "plan.cpp").write_text("""
#include "trx_attn_plan.h"
#include <cstdio>
int main() {
  trx::ArCall c;
  trx::ArCut prefix, tail;
  for (int half; scanf("%d%d%d%d%d%d%d%d%d", &half, &c.n_head, &c.n_kv, &c.hd, &c.batch, &c.n, &c.prefix, &c.slots, &c.keys) == 9;) {
    c.half_io = half;
    trx::ar_plan(c, prefix, tail);
    printf("%d %d %d %d\\n", c.prefix ? prefix.wq : 0, tail.wq, trx::ar_keeps(c, tail), trx::ar_mass_parts(c) > 1);
  }
}""")
    exe, src = str(tmp_path / "plan"), os.path.join(os.path.dirname(_lib.__file__), "csrc")
    subprocess.run(["g++", "-std=c++17", "-I", src, str(tmp_path / "plan.cpp"), "-o", exe], check=True)
    calls = [(*c[:8], c[7]) for c in SHARED]
    calls += [(*c[:4], 1, c[4], 0, c[5] + c[4] + SLACK, c[5] + c[4]) for c in MASS]
    calls += [(*c[:4], 1, c[4], 0, c[5], c[5]) for c in CAPTURED]
    lines = "".join(" ".join(str(int(x == F16)) if i == 0 else str(x) for i, x in enumerate(c)) + "\n" for c in calls)
    got = [tuple(map(int, x.split())) for x in subprocess.run([exe], input=lines, capture_output=True, text=True, check=True).stdout.splitlines()]
    assert len(got) == len(calls)
    for c, g in zip(SHARED, got):
        assert g[:2] == c[8:], (c, g)
    for c, g in zip(MASS + CAPTURED, got[len(SHARED):]):
        assert g == (0, c[6], 0, c[7]), (c, g)                      # none keeps its scores


def ident(c):
    return "-".join(str(x) for x in c)


@pytest.mark.gpu
@pytest.mark.parametrize("case", SHARED, ids=ident)
def test_drafts(case):
    """All rows, then ragged counts and a gate, with NaN and infinities behind the prefix and behind each draft's rows."""
    kind, heads, kv, hd, batch, n, prefix, slots = case[:8]
    c = Drafts(heads, kv, hd, batch, prefix, slots, kind, seed=23, prefix_slots=prefix + 40)
    c.kp[:, prefix:], c.vp[:, prefix:] = np.nan, np.inf
    lengths = c.rng.integers(0, slots - n + 1, batch)
    lengths[0], lengths[-1] = 0, slots - n
    for b in range(batch):
        c.kt[b][:, lengths[b]:], c.vt[b][:, lengths[b]:] = np.nan, -np.inf
    print(f"worst error {c.check(n, lengths):.3f} of the tolerance")
    counts = c.rng.integers(0, n + 1, batch)
    counts[0] = n
    print(f"worst error {c.check(n, lengths, counts=counts, gated=True):.3f} of the tolerance")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
def test_drafts_that_take_no_part(kind):
    """As test_shared_prefix_gpu.py's, where prefix and tails fill wide blocks."""
    c = Drafts(64, 8, 128, 6, 300, 300, kind, seed=24)
    n = 64
    lengths = np.array([7, -1, 237, 236, 100, 2**31 - 1], np.int32)
    counts = np.array([64, 64, 64, 64, 65, 9], np.int32)
    q, k, v = c.rows(n)
    for b in (1, 2, 4, 5):
        for a in (q, k, v):
            a[b * n:b * n + n] = np.nan
    out, kt, vt = c.call(q, k, v, lengths, counts)
    want, tol, ek, ev = c.expect(q, k, v, lengths, counts)
    assert (np.abs(out.reshape(want.shape) - want) <= tol).all()
    assert all((want[b * n:b * n + n] == 77).all() == (b in (1, 2, 4, 5)) for b in range(6))
    assert np.array_equal(kt.view(np.uint16), ek.view(np.uint16)) and np.array_equal(vt.view(np.uint16), ev.view(np.uint16))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
def test_infinities_and_nans_stay_where_they_are_seen(kind):
    """A value of the prefix that is infinite shows in every draft, one of a tail in that draft alone, one of a new row in the
    rows from it on; a NaN query in its own row."""
    c = Drafts(64, 8, 128, 4, 300, 300, kind, seed=25)
    n, lengths = 64, np.array([60, 200, 0, 236])
    q, k, v = c.rows(n)
    c.vp[0, 17, 3], c.vt[1][1, 9, 5] = np.inf, -np.inf
    v[2 * n + 40, 0, 7], q[5, 30, 0] = np.nan, np.nan
    out = c.call(q, k, v, lengths)[0].reshape(q.shape)
    bad = np.zeros(out.shape, bool)
    bad[:, :8, 3] = bad[n:2 * n, 8:16, 5] = bad[2 * n + 40:3 * n, :8, 7] = bad[5, 30] = True
    assert (out[:, :8, 3] == np.inf).all() and (out[n:2 * n, 8:16, 5] == -np.inf).all()
    assert np.isnan(out[2 * n + 40:3 * n, :8, 7]).all() and np.isnan(out[5, 30]).all()
    c.vp[0, 17, 3] = c.vt[1][1, 9, 5] = v[2 * n + 40, 0, 7] = q[5, 30, 0] = 0
    want, tol, _, _ = c.expect(q, k, v, lengths, [n] * 4)
    assert (np.abs(out - want)[~bad] <= tol[~bad]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("case", MASS, ids=ident)
def test_chunks(case):
    """Outputs, rows, positions and masses, with NaN and infinities behind the rows."""
    kind, heads, kv, hd, n, count = case[:6]
    c = Cache(heads, kv, hd, count + n + SLACK, kind, seed=26)
    end = count + n
    c.K[:, count:], c.V[:, count:], c.mass[:, count:] = np.nan, np.inf, np.nan
    rest = c.mass[:, end:].copy()
    q, k, v = c.rows(n)
    gate = c.rng.standard_normal(q.shape).astype(DT[kind])
    out, K, V, mass, positions = c.attend(q, k, v, count, count + 5, gate)
    want, tol, wm, mtol = c.after(q, k, v, count, count + 5, gate)
    err, merr = np.abs(out.reshape(want.shape) - want), np.abs(mass - wm)[:, :end]
    assert (err <= tol).all(), (float((err / tol).max()), np.argwhere(~(err <= tol))[:4].tolist())
    assert (merr <= mtol[:, :end]).all(), (float((merr / mtol[:, :end]).max()), np.argwhere(~(merr <= mtol[:, :end]))[:4].tolist())
    assert np.array_equal(mass[:, end:].view(np.uint32), rest.view(np.uint32))
    assert np.array_equal(K.view(np.uint16), c.K.view(np.uint16)) and np.array_equal(V.view(np.uint16), c.V.view(np.uint16))
    assert np.array_equal(positions, c.positions)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [F32, F16])
def test_a_later_row_gives_nothing_to_an_earlier_one(kind):
    """A new key that would take all the attention, an infinity in a value and a NaN key (of another kv head) show in the rows
    from them on alone; the infinity touches no mass, the key those of its kv head."""
    c, n, count = Cache(32, 8, 128, 617, kind, seed=27), 300, 300
    q, k, v = c.rows(n)
    k[n - 1, 0], v[n // 2, 0, 3], k[n - 20, 5, 1] = 20.0, np.inf, np.nan
    out, _, _, mass, _ = c.attend(q, k, v, count, count)
    out = out.reshape(q.shape)
    assert (out[n // 2:, :4, 3] == np.inf).all() and np.isnan(out[n - 20:, 20:24]).all()
    v[n // 2, 0, 3] = k[n - 20, 5, 1] = 0
    want, tol, wm, mtol = c.after(q, k, v, count, count)
    ok = np.ones(want.shape, bool)
    ok[n // 2:, :4, 3] = ok[n - 20:, 20:24] = False
    assert (np.abs(out - want)[ok] <= tol[ok]).all()
    others = [g for g in range(8) if g != 5]
    assert (np.abs(mass - wm)[others, :count + n] <= mtol[others, :count + n]).all()
    assert np.array_equal(mass[:, count + n:], wm[:, count + n:].astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("case", CAPTURED, ids=ident)
def test_state_on_the_device_captured(case):
    """A captured chunk whose grid is that of all slots, replayed over few rows and many, with eager calls between the replays;
    a state out of range leaves everything as it is."""
    kind, heads, kv, hd, n, slots = case[:6]
    c = Cache(heads, kv, hd, slots, kind, seed=28)
    B, shape, size = _lib.DeviceBuffer, c.shape(), DT[kind]().itemsize * n * heads * hd
    s, ex = ctypes.c_void_p(), ctypes.c_void_p()
    _lib.call("trx_stream_create", ctypes.byref(s))
    cache = [B.from_array(a) for a in c.arrays()]
    qb, kb, vb, out, sb, work = (B(x) for x in (size, 2 * n * kv * hd, 2 * n * kv * hd, size, 8, geometry(shape, n)))
    _lib.synchronize()
    _lib.call("trx_graph_begin", s)
    _lib.call("trx_attn_mass", ctypes.byref(shape), n, 0, 0, sb.ptr, qb.ptr, kb.ptr, vb.ptr, *(b.ptr for b in cache), None, out.ptr,
              work.ptr, s)
    _lib.call("trx_graph_end", s, ctypes.byref(ex))
    for rep, count in enumerate((0, 37, 300, slots - n, 150)):
        q, k, v = c.rows(n)
        for b, a in ((qb, q), (kb, k), (vb, v), (sb, np.array([count, 900 + count], np.int32))):
            b.upload(a, s)
        _lib.call("trx_graph_launch", ex, s)
        _lib.synchronize(s)
        want, tol, wm, mtol = c.after(q, k, v, count, 900 + count)
        assert (np.abs(out.download(DT[kind], q.size).reshape(q.shape) - want) <= tol).all(), count
        c.mass = cache[2].download(np.float32).reshape(c.mass.shape)
        assert (np.abs(c.mass - wm) <= mtol).all(), count
        assert all(np.array_equal(b.download(a.dtype).reshape(a.shape).view(np.uint8), a.view(np.uint8))
                   for b, a in zip(cache, c.arrays())), count
        Cache(4, 2, 64, 400, seed=40 + rep).check(200, 150)          # an eager call between the replays
    before = [b.download(np.uint8) for b in cache]
    for bad in ((-1, 5), (slots - n + 1, 5), (5, -1), (5, 2**31 - n), (2**31 - 1, 5)):
        sb.upload(np.array(bad, np.int32), s), out.upload(np.full(size, 5, np.uint8), s)
        _lib.call("trx_graph_launch", ex, s)
        _lib.synchronize(s)
        assert (out.download(np.uint8, size) == 5).all(), bad
        assert all(np.array_equal(a, b.download(np.uint8)) for a, b in zip(before, cache)), bad
    _lib.call("trx_graph_destroy", ex)
    _lib.call("trx_stream_destroy", s)


# (Short caches: the bound on the sums grows with the keys, and past some thousand would hide a rounded probability.)
def round_once(out, q, K, V, lim, scale):
    """Outputs [rows, heads, hd] of fp16 queries with one element over K, V [keys, kv heads, hd], row r seeing lim[r] keys:
    the fp32 result rounded. x + d rounds to a value whose distance from x is at most that of x rounded, plus 2 d; a score
    without a sum over dims leaves d the fp32 tolerance without it: the score and the exponent 2^-21 of S and of 1 each,
    twice (the probability and the total), the sums N 2^-24, the probabilities' planes 2^-22."""
    rows, heads, hd = q.shape
    worst = 0.0
    for h in range(heads):
        g = h * K.shape[1] // heads
        Kg, Vg = K[:, g, 0].astype(np.float64), V[:, g].astype(np.float64)
        s = float(scale) * np.outer(q[:, h, 0].astype(np.float64), Kg)
        s[np.arange(K.shape[0])[None] >= np.asarray(lim)[:, None]] = -np.inf
        S = np.where(np.isfinite(s), np.abs(s), 0).max(1)[:, None]
        p = np.exp(s - s.max(1)[:, None])
        p /= p.sum(1)[:, None]
        x, d = p @ Vg, (p @ np.abs(Vg)) * (2 * (S + 1) * 2.0**-21 + np.asarray(lim)[:, None] * 2.0**-24 + 2.0**-22)
        bound = np.abs(x.astype(np.float16).astype(np.float64) - x) + 2 * d
        err = np.abs(out[:, h].astype(np.float64) - x)
        assert (err <= bound).all(), (h, float((err / bound).max()), int((err > bound).sum()))
        worst = max(worst, float((err / bound).max()))
    return worst


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,batch,n,prefix,slots", [
    (64, 8, 128, 4, 64, 300, 300), (24, 4, 256, 4, 100, 300, 400), (64, 8, 64, 100, 8, 700, 60), (32, 8, 128, 160, 4, 500, 60)])
def test_drafts_with_fp16_queries_round_once(heads, kv, hd, batch, n, prefix, slots):
    """However many drafts share a call, their fp16 outputs are the fp32 result rounded."""
    c = Drafts(heads, kv, hd, batch, prefix, slots, F16, seed=21, scale=2.0)
    q, k, v = c.rows(n)
    q[..., 1:] = 0
    lengths = c.rng.integers(0, slots - n + 1, batch)
    out, _, _ = c.call(q, k, v, lengths)
    out = out.reshape(q.shape)
    for b in range(batch):
        at, have = slice(b * n, b * n + n), int(lengths[b])
        K, V = (np.concatenate([p, t[b][:, :have], x[at].transpose(1, 0, 2)], axis=1).transpose(1, 0, 2)
                for p, t, x in ((c.kp, c.kt, k), (c.vp, c.vt, v)))
        round_once(out[at], q[at], K, V, prefix + have + 1 + np.arange(n), c.scale)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,count,n", [(32, 8, 128, 300, 300), (24, 4, 256, 500, 256), (64, 8, 64, 500, 256), (16, 8, 128, 300, 500)])
def test_chunks_with_fp16_queries_round_once(heads, kv, hd, count, n):
    c = Cache(heads, kv, hd, count + n + 17, F16, seed=22, scale=2.0)
    q, k, v = c.rows(n)
    q[..., 1:] = 0
    out = c.attend(q, k, v, count, count)[0].reshape(q.shape)
    K, V = (np.concatenate([a[:, :count], x.transpose(1, 0, 2)], axis=1).transpose(1, 0, 2) for a, x in ((c.K, k), (c.V, v)))
    round_once(out, q, K, V, count + 1 + np.arange(n), c.scale)
