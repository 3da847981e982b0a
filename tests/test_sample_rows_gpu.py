"""Sampling from the whole vocabulary (trx_sample_rows) against its definition on the host, the masses as
the integers that the operator defines: filters, ties, masked and infinite logits, extreme settings
and uniform numbers, rows of any alignment; and what it refuses.

The host's exponentials differ from the device's by a unit of 2^-50 at most, so a mass may differ by one
unit of its last bit; a token could differ only where a border falls within that of a target, which
equal logits (whose masses are exact) never do. Log-probabilities: two 64-bit results rounded to
fp32, half a step (2^-24) each, plus 2^-40."""

import ctypes

import numpy as np
import pytest

from trixium_amd import _lib, layout as L
from trixium_amd.sampling import ROW, sample, settings

OFF = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)


def _frac(vocab):
    return min(51, 62 - (vocab - 1).bit_length())


def oracle(logits, u, temperature, top_k, top_p, min_p):
    """(token, log-probability) of one row."""
    x = np.asarray(logits).astype(np.float32).astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    V = x.size
    T, p, mp, u = (np.float32(v) for v in (temperature, top_p, min_p, u))
    top = x.max()
    if top == -np.inf:
        return -1, np.nan
    if not T > 0:
        return int(np.argmax(x)), 0.0
    frac = _frac(V)
    with np.errstate(all="ignore"):
        y = np.where(x == top, 0.0, -np.abs(top - x) * (1.0 / np.float64(T)))
        y = np.where(x == -np.inf, -np.inf, y)
        w = np.where(x == top, 1.0, np.where(np.isnan(y), 1.0, np.exp(y)))
        if top == np.inf:
            w = (x == np.inf).astype(np.float64)
    mass = [int(m) for m in np.rint(w * 2.0**frac)]
    order = [i for i in np.argsort(-x, kind="stable") if mass[i]]
    if 0 < top_k < V:
        order = order[:top_k]
    if 0 < p < 1:
        num, den = float(p).as_integer_ratio()
        total, run = sum(mass[i] for i in order), 0
        for j, i in enumerate(order):
            run += mass[i]
            if run * den >= num * total:
                order = order[:j + 1]
                break
    if 0 <= mp <= 1:
        num, den = float(mp).as_integer_ratio()
        order = [i for i in order if mass[i] * den >= num << frac]
    total, run = sum(mass[i] for i in order), 0
    uf = float(u) if u > 0 else 0.0                        # NaN too
    num, den = uf.as_integer_ratio() if uf < 1 else (total * 2 - 1, total * 2)
    for i in sorted(order):
        run += mass[i]
        if run * den > num * total:
            lw = 0.0 if top == np.inf else -(top - x[i]) / np.float64(T)
            return int(i), float(lw - np.log(total / 2.0**frac))
    raise AssertionError("no token")


def check(logits, u, **kw):
    kw = {**OFF, **kw}
    tok, lp = sample(logits, u, **kw)
    cols = np.broadcast_arrays(*(np.atleast_1d(kw[k]) for k in ROW.names), np.asarray(u))[:4]
    for r in range(len(tok)):
        t, l = oracle(logits[r], u[r], *(c[r] for c in cols))
        assert tok[r] == t, (r, int(tok[r]), t, [c[r] for c in cols], u[r])
        if t < 0:
            assert np.isnan(lp[r])
        else:
            assert abs(float(lp[r]) - l) <= 2.0**-23 * abs(l) + 2.0**-40, (r, lp[r], l)
    return tok


def _logits(rng, n, vocab, dtype=np.float32, spread=1.3):
    """As a language model's: falling with the logarithm of the rank, noise, a random order."""
    r = np.stack([rng.permutation(vocab) for _ in range(n)])
    return (11.0 - spread * np.log(r + 1.0) + 0.5 * rng.standard_normal((n, vocab))).astype(dtype)


MIX = [dict(temperature=0.8, top_p=0.9), dict(temperature=0.7, top_k=50), dict(temperature=1.0),
       dict(temperature=0.9, top_k=200, top_p=0.95, min_p=0.02), dict(temperature=1.3, min_p=0.05),
       dict(temperature=0.0), dict(temperature=1.5, top_k=7, top_p=0.3), dict(temperature=1.0, top_k=1),
       dict(temperature=2.5, top_p=0.999), dict(temperature=0.3, min_p=1.0), dict(temperature=1.0, top_p=1e-9),
       dict(temperature=1.7, top_k=5000), dict(temperature=3.0, top_k=9000, top_p=0.8),
       dict(temperature=1.0, top_k=10**9, top_p=0.7), dict(temperature=1.2, top_k=-3, top_p=2.0, min_p=-1.0)]


def _mixed(n):
    full = [{**OFF, **MIX[r % len(MIX)]} for r in range(n)]
    return {k: np.array([f[k] for f in full]) for k in ROW.names}


# The oracle and refusals (no GPU) ----------------------------------------------------------------------


def test_the_oracle_on_closed_forms():
    """Equal logits: u picks floor(u times the count). top_p keeps the first ceil(p V) of them, top_k the
    first k; two tokens d apart: the second's share is 1 / (1 + e^d)."""
    eq = np.zeros(10, np.float32)
    for u in (0.0, 0.05, 0.31, 0.999):
        assert oracle(eq, u, 1, 0, 1, 0)[0] == int(np.float32(u) * 10)
        assert oracle(eq, u, 1, 0, 0.5, 0)[0] == int(np.float32(u) * 5)
        assert oracle(eq, u, 1, 3, 1, 0)[0] == int(np.float32(u) * 3)
        assert oracle(eq, u, 1, 4, 0.5, 0)[0] == int(np.float32(u) * 2)
    two = np.array([0.0, 1.0], np.float32)
    low = 1 / (1 + np.e)
    assert oracle(two, low - 1e-3, 1, 0, 1, 0)[0] == 0 and oracle(two, low + 1e-3, 1, 0, 1, 0)[0] == 1
    assert abs(oracle(two, 0.9, 1, 0, 1, 0)[1] - np.log(1 - low)) < 1e-12
    assert oracle(two, 0.0, 1, 0, 1, 0.5)[0] == 1                      # e^-1 < 0.5
    assert oracle(two, 0.0, 0, 0, 1, 0) == (1, 0.0)


def test_refusals():
    lib, fake, size = _lib.lib(), ctypes.c_void_p(256), ctypes.c_size_t()
    for vocab, n, what in ((0, 1, b"vocab"), ((1 << 24) + 1, 1, b"vocab"), (100, -1, b"rows"), (100, (1 << 20) + 1, b"rows")):
        assert lib.trx_sample_rows_geometry(vocab, n, ctypes.byref(size)) == _lib.TRX_E_INVALID
        assert what in lib.trx_last_error()
    assert lib.trx_sample_rows_geometry(100, 1, None) == _lib.TRX_E_INVALID
    assert lib.trx_sample_rows_geometry(100, 4, ctypes.byref(size)) == _lib.TRX_OK and size.value > 0

    def call(lg=fake, kind=L.KIND_F32, n=1, vocab=100, ld=100, rows=fake, u=fake, tok=fake, lp=None, work=fake):
        return lib.trx_sample_rows(lg, kind, n, vocab, ld, rows, 0, u, tok, lp, work, None)

    p = ctypes.c_void_p
    for kw, what in ((dict(kind=L.KIND_Q8), b"kind"), (dict(ld=99), b"rows of"), (dict(vocab=0), b"vocab"),
                     (dict(n=-1), b"rows"), (dict(lg=None), b"null"), (dict(rows=None), b"null"), (dict(u=None), b"null"),
                     (dict(tok=None), b"null"), (dict(work=None), b"null"), (dict(lg=p(258)), b"aligned"),
                     (dict(lg=p(257), kind=L.KIND_F16), b"aligned"), (dict(work=p(264)), b"aligned"),
                     (dict(lp=p(258)), b"aligned")):
        assert call(**kw) == _lib.TRX_E_INVALID, kw
        assert what in lib.trx_last_error(), (kw, lib.trx_last_error())
    assert call(n=0, lg=None) == _lib.TRX_OK
    with pytest.raises(ValueError):
        sample(np.zeros(4, np.float32), [0.5])
    with pytest.raises(ValueError):
        sample(np.zeros((2, 4), np.float32), [0.5])
    with pytest.raises(ValueError):
        sample(np.zeros((2, 4), np.float32), [0.5, 0.5], top_k=np.array([1, 2, 3]))
    assert sample(np.zeros((0, 4), np.float32), [])[0].size == 0


def test_a_top_k_past_int32_is_off(monkeypatch):
    """2^32 + 5 is past every vocabulary, not 5."""
    assert settings(top_k=[2**32 + 5, -2**33 + 7, 7, 0])["top_k"].tolist() == [2**31 - 1, -1, 7, 0]
    assert settings(top_k=2**40 + 1)["top_k"].tolist() == [2**31 - 1]
    from trixium_amd.model import Decoder
    seen = []
    monkeypatch.setattr(_lib, "call", lambda name, *a: seen.append(a[2]))
    dec = Decoder.__new__(Decoder)
    dec._h = None
    for k in (2**32 + 5, -2**33 + 7, 40, 0):
        dec.set_vocab_sampling(top_k=k)
    assert seen[:4] == [2**31 - 1, -1, 40, 0]


@pytest.mark.parametrize("dtype", [np.uint8, np.int8, np.uint16, np.int16, np.uint32, np.int64, np.uint64, np.float16,
                                   np.float64, bool, object])
def test_settings_take_a_top_k_of_any_type(dtype):
    assert settings(top_k=np.array([1, 0], dtype))["top_k"].tolist() == [1, 0]
    if dtype in (np.uint32, np.int64, np.uint64, np.float64, object):
        assert settings(top_k=np.array([2**32 - 1, 50], dtype))["top_k"].tolist() == [2**31 - 1, 50]
    if dtype is object:
        assert settings(top_k=np.array([2**70], dtype))["top_k"].tolist() == [2**31 - 1]


# Results (GPU) ---------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab,n", [(1, 3), (2, 15), (7, 15), (300, 30), (2048, 30), (4097, 15), (20011, 30), (151936, 15)])
def test_rows_against_the_definition(vocab, n, dtype):
    rng = np.random.default_rng(vocab)
    print(vocab, n, dtype.__name__, flush=True)
    check(_logits(rng, n, vocab, dtype), rng.random(n).astype(np.float32), **_mixed(n))


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [0.02, 4.0])
def test_flat_and_steep_rows(spread):
    rng = np.random.default_rng(3)
    check(_logits(rng, 15, 30000, spread=spread), rng.random(15).astype(np.float32), **_mixed(15))


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [5, 1000, 4096, 40000])
def test_equal_logits(vocab):
    """Ties go by index; the masses are exact, so every border is."""
    us = np.array([0.0, 2.0**-24, 0.25, 0.5, 1 - 2.0**-24], np.float32)
    lg = np.full((us.size, vocab), -3.25, np.float32)
    for kw in (dict(), dict(top_p=0.5), dict(top_k=max(1, vocab // 3)), dict(top_k=max(2, vocab // 2), top_p=0.5),
               dict(top_p=0.125, temperature=1e-3), dict(min_p=1.0)):
        check(lg, us, **kw)
    lg[:, ::3] = 1.0                                       # two values
    for kw in (dict(), dict(top_p=0.5), dict(top_k=vocab // 3 + 2), dict(top_p=0.99, temperature=4.0)):
        check(lg, us, **kw)


@pytest.mark.gpu
def test_a_cluster_behind_an_outlier():
    """One step of the histogram holds nearly the whole vocabulary: the cut is found in the row itself."""
    rng = np.random.default_rng(5)
    lg = (1e-4 * rng.standard_normal((6, 30000))).astype(np.float32)
    lg[:, 777] = 40.0
    us = np.array([0.1, 0.4, 0.7, 0.9, 0.99, 0.5], np.float32)
    check(lg, us, temperature=8.0, top_p=0.9)
    check(lg, us, temperature=8.0, top_k=12345)
    check(lg, us, temperature=8.0, top_k=12345, top_p=0.6, min_p=1e-3)
    check(lg, us, temperature=8.0, top_k=6000, top_p=0.9999)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_masked_and_infinite_logits(dtype):
    rng = np.random.default_rng(6)
    n, V = 15, 5000
    lg = _logits(rng, n, V, dtype)
    hide = rng.random((n, V)) < 0.99
    low = np.finfo(dtype).min
    us = rng.random(n).astype(np.float32)
    for fill in (-np.inf, low, np.nan):
        check(np.where(hide, dtype(fill), lg), us, **_mixed(n))
    one = np.full((n, V), -np.inf, dtype)
    one[:, 4321] = low                                     # a single token left
    assert (check(one, us, **_mixed(n)) == 4321).all()
    one[:, 4321] = np.nan
    assert (check(one, us, **_mixed(n)) == -1).all()
    lg[:, [7, 4000, 4999]] = np.inf
    check(lg, us, **_mixed(n))
    big = np.where(hide, dtype(low), np.finfo(dtype).max).astype(dtype)
    check(big, us, **_mixed(n))
    zeros = np.where(hide, dtype(-0.0), dtype(0.0)).astype(dtype)      # equal: by index
    check(zeros, us, top_k=17)


@pytest.mark.gpu
def test_extreme_settings_and_uniforms():
    rng = np.random.default_rng(7)
    ts = np.array([1e-38, 1e-30, 1e-4, 50.0, 1e4, 1e38, np.inf, np.nan, -1.0, -np.inf], np.float32)
    lg = _logits(rng, ts.size, 3000)
    us = rng.random(ts.size).astype(np.float32)
    for kw in (dict(), dict(top_p=0.4), dict(top_k=100), dict(min_p=0.5)):
        check(lg, us, temperature=ts, **kw)
    us = np.array([0.0, 1e-45, 1e-30, 2.0**-24, 1 - 2.0**-24, 1.0, 2.0, np.inf, -1.0, np.nan], np.float32)
    for kw in (dict(), dict(top_p=0.4), dict(top_k=100), dict(min_p=0.5), dict(top_p=np.nan, min_p=np.nan)):
        check(lg, us, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_any_row_alignment_gives_the_same_tokens(dtype):
    """The same row at every offset from a 16-byte boundary, in rows wider than the vocabulary whose rest
    holds larger values."""
    rng = np.random.default_rng(8)
    V, ld, n = 9001, 9017, 16
    row, u = _logits(rng, 1, V, dtype)[0], np.float32(0.37)
    lg = np.full((n, ld), 30.0, dtype)
    lg[:, :V] = row
    B = _lib.DeviceBuffer
    size = ctypes.c_size_t()
    _lib.call("trx_sample_rows_geometry", V, n, ctypes.byref(size))
    lb, ub, work = B.from_array(lg), B.from_array(np.full(n, u)), B(size.value)
    for kw in (dict(temperature=0.8, top_p=0.9), dict(temperature=1.0), dict(temperature=1.0, top_k=40)):
        kw = {**OFF, **kw}
        rb, tok = B.from_array(settings(**kw)), B(4 * n)
        _lib.call("trx_sample_rows", lb.ptr, L.KIND_F16 if dtype == np.float16 else L.KIND_F32, n, V, ld, rb.ptr, 0,
                  ub.ptr, tok.ptr, None, work.ptr, None)
        _lib.synchronize()
        want = oracle(row, u, *(kw[k] for k in ROW.names))[0]
        assert (tok.download(np.int32, n) == want).all()


@pytest.mark.gpu
def test_captured_graph_reads_new_settings_and_numbers():
    rng = np.random.default_rng(9)
    n, V = 15, 7000
    B = _lib.DeviceBuffer
    size, s, ex = ctypes.c_size_t(), ctypes.c_void_p(), ctypes.c_void_p()
    _lib.call("trx_sample_rows_geometry", V, n, ctypes.byref(size))
    lb, ub, rb, tok, lp, work = B(4 * n * V), B(4 * n), B(16 * n), B(4 * n), B(4 * n), B(size.value)
    _lib.call("trx_stream_create", ctypes.byref(s))
    _lib.call("trx_graph_begin", s)
    _lib.call("trx_sample_rows", lb.ptr, L.KIND_F32, n, V, V, rb.ptr, 1, ub.ptr, tok.ptr, lp.ptr, work.ptr, s)
    _lib.call("trx_graph_end", s, ctypes.byref(ex))
    for rep in range(4):
        lg, us = _logits(rng, n, V), rng.random(n).astype(np.float32)
        kw = {k: np.roll(v, rep) for k, v in _mixed(n).items()}
        lb.upload(lg, s), ub.upload(us, s), rb.upload(settings(**kw), s)
        _lib.call("trx_graph_launch", ex, s)
        _lib.synchronize(s)
        got = tok.download(np.int32, n)
        assert got.tolist() == [oracle(lg[r], us[r], *(kw[k][r] for k in ROW.names))[0] for r in range(n)], rep
        assert np.array_equal(sample(lg, us, **kw)[0], got)            # eager work between the replays
    _lib.call("trx_graph_destroy", ex)
    _lib.call("trx_stream_destroy", s)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab,n", [(20011, 600), (9001, 2100), (33000, 129), (2**21 + 5, 2)])
def test_rows_cut_into_long_chunks(vocab, n, dtype):
    """Many rows and the longest ones take chunks of several rounds and parts: some rows of each setting
    against the definition, and every row's token again when the row is drawn alone with others."""
    rng = np.random.default_rng(vocab)
    lg = (4.0 * rng.standard_normal((n, vocab), dtype=np.float32)).astype(dtype)
    u = rng.random(n).astype(np.float32)
    kw = _mixed(n)
    tok, lp = sample(lg, u, **kw)
    some = rng.permutation(n)[:15]
    check(lg[some], u[some], **{k: v[some] for k, v in kw.items()})
    again, lp2 = sample(lg[some], u[some], **{k: v[some] for k, v in kw.items()})
    assert np.array_equal(tok[some], again) and np.array_equal(lp[some], lp2)
    for r in some[:4]:
        assert oracle(lg[r], u[r], *(kw[k][r] for k in ROW.names))[0] == tok[r]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_cuts_beside_tokens_without_mass(dtype):
    """The cut lies in the histogram's last step, where the tokens too far below the largest stand as well."""
    rng = np.random.default_rng(8)
    vocab = 6000
    lg = np.stack([rng.permutation(np.linspace(0, -60, vocab)) for _ in range(4)]).astype(dtype)
    lg[3, 17] = lg[3, 4000] = np.inf
    mass = [int(m) for m in np.rint(np.exp(lg[0].astype(np.float64)) * 2.0**_frac(vocab))]
    live = sum(m > 0 for m in mass)
    assert 1000 < live < vocab
    us = np.array([0.2, 0.6, 1 - 2.0**-24, 0.7], np.float32)
    for k in (live - 1, live, live + 1, live - 3):
        check(lg, us, top_k=k)
        check(lg, us, top_k=k, top_p=1 - 2.0**-24)
    check(lg, us, top_p=1 - 2.0**-24)
    check(lg, us, top_p=0.5, top_k=2)


@pytest.mark.gpu
def test_many_tokens_at_the_last_mass_of_none():
    """The smallest logits stand exactly where a mass is half a unit, which rounds to none, and share the
    histogram's last step with the cut: more of them than a gather holds must not push the others out. (The row's
    largest logit comes last, and is drawn but at u = 0, which takes the first token with a mass: everything else is
    below 2^-46 of the mass.)"""
    vocab, T = 9000, np.float32(float.fromhex("0x1.00000ep-1"))
    top, low = (float.fromhex(v) for v in ("0x1.0fb6c4p+4", "0x1.c22362p-22"))
    c2 = 1.44269504088896340736 / np.float64(T)
    assert np.float32(low) == low and (_frac(vocab) + 1) / c2 == top - low and (low - top) * c2 == -(_frac(vocab) + 1)
    lg = np.full((8, vocab), low, np.float32)
    lg[:, -1] = top
    lg[:, 100:104] = low + np.array([1e-3, 2e-3, 3e-3, 4e-3])
    us = np.linspace(0, 1 - 2.0**-24, 8).astype(np.float32)
    for kw in (dict(top_k=2), dict(top_k=3), dict(top_k=3, min_p=0.1), dict(top_k=2, top_p=0.999)):
        assert (check(lg, us, temperature=T, **kw)[1:] == vocab - 1).all()
