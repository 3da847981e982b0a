"""Drafts behind a shared prefix (trx_attn_shared) and attention with masses (trx_attn_mass) at sizes whose columns fill
wide blocks, waves of two or four columns, against their definition in 64 bits."""

import numpy as np
import pytest

from trixium_amd import layout as L
from test_kv_mass_gpu import Cache
from test_shared_prefix_gpu import Drafts

F32, F16 = L.KIND_F32, L.KIND_F16


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
