"""Sampling one token per row of logits from the whole vocabulary (host side of trx_sample_rows):
temperature, top-k, top-p and min-p, from given uniform numbers. The firmware's own sampler, which
draws among 32 candidates, is `Decoder.set_sampling` (firmware/infer.c:385-488). Logits and results are
numpy arrays, copied to the GPU and back by each call, which waits for it; a program whose logits are on the GPU
calls trx_sample_rows with its own pointers, stream and workspace, and the decoder does (set_vocab_sampling)."""

import ctypes

import numpy as np

from . import _lib
from . import layout as L

ROW = np.dtype([("temperature", np.float32), ("top_k", np.int32), ("top_p", np.float32), ("min_p", np.float32)])


def settings(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row's settings (scalars), or n rows' (arrays of n or scalars), as trx_sampling structs. top_k 0,
    top_p 1 and min_p 0 are off; temperature 0 takes the largest logit."""
    top_k = np.asarray(top_k)                      # (past int32: off, like every one past the vocabulary)
    top_k = np.clip(top_k.astype(np.int64 if top_k.dtype.kind in "bui" else np.float64), -1, 2**31 - 1)
    cols = np.broadcast_arrays(*(np.atleast_1d(a) for a in (temperature, top_k, top_p, min_p)))
    out = np.empty(cols[0].shape, dtype=ROW)
    for name, c in zip(ROW.names, cols):
        out[name] = c
    return out


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens int32 [n], log-probabilities float32 [n]) for logits [n, vocab] (float16, else taken as
    float32) and uniform numbers u [n]; the settings are scalars or arrays of n. A token of -1: the row
    has no logit above -inf."""
    lg = np.asarray(logits)
    lg = np.ascontiguousarray(lg if lg.dtype == np.float16 else lg.astype(np.float32))
    if lg.ndim != 2:
        raise ValueError(f"logits of shape {lg.shape}: rows of a vocabulary expected")
    n, vocab = lg.shape
    u = np.ascontiguousarray(np.asarray(u, dtype=np.float32).reshape(-1))
    rows = settings(temperature, top_k, top_p, min_p)
    if u.size != n or rows.size not in (1, n):
        raise ValueError(f"{n} rows of logits, {u.size} uniform numbers, settings for {rows.size}")
    size = ctypes.c_size_t()
    _lib.call("trx_sample_rows_geometry", vocab, n, ctypes.byref(size))
    if n == 0:
        return np.empty(0, np.int32), np.empty(0, np.float32)
    lb, ub, rb = (_lib.DeviceBuffer.from_array(a) for a in (lg, u, rows))
    tok, lp, work = _lib.DeviceBuffer(4 * n), _lib.DeviceBuffer(4 * n), _lib.DeviceBuffer(size.value)
    _lib.call("trx_sample_rows", lb.ptr, L.KIND_F16 if lg.dtype == np.float16 else L.KIND_F32, n, vocab, vocab, rb.ptr,
              int(rows.size == n), ub.ptr, tok.ptr, lp.ptr, work.ptr, None)
    _lib.synchronize()
    return tok.download(np.int32, n), lp.download(np.float32, n)
