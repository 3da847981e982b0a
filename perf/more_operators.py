"""Operators of caches that several drafts share or that keep less than they were given, over the
sizes that the configurations run.

`shared`: attention of the next positions of a batch of drafts of one prompt (`trx_attn_shared`). The
prompt's K and V rows, the prefix, stand once for all; each draft has a tail of its own. The i-th new
position of draft b sees the whole prefix, the lengths[b] rows of the draft's tail and the new rows
0 .. i; of n new positions a draft takes the first counts[b], whose K and V rows are appended to its
tail. Rows behind a draft's count are left as they were.

`mass`: attention of the next n positions over a cache of rows (`trx_attn_mass`), which also adds to
each row of K and V the probabilities that the positions and the heads of its kv head gave it: the
row's mass. A new row's mass begins with this call's. The new rows take the slots behind the last.

`evict`: of the `count` rows of each kv head of such a cache, `keep` stay (`trx_kv_evict`): the first
`sinks` positions and the last `recent` ones before any other, then the largest masses, equal ones by
slot. Rows that stay past slot `keep` take, in the order of their slots, the slots below it of rows
that go; K, V, mass and position move together and nothing past `keep` is written.
"""

import ctypes
import math

import numpy as np
import torch

own = False

# (heads, kv heads, head dim) of the shipped configurations.
MODELS = {"1.7b": (16, 8, 128), "8b": (32, 8, 128), "27b": (24, 4, 256), "tiny": (4, 2, 64)}
TYPES = {"f32": torch.float32, "f16": torch.float16}


def _shared(name, model, batch, n, prefix, tail, dtype, ragged=False, gated=False):
    return {"name": name, "op": "shared", "model": model, "batch": batch, "n": n, "prefix": prefix, "tail": tail,
            "type": dtype, "ragged": ragged, "gated": gated}


def _mass(name, model, n, count, slots, dtype, gated=False):
    return {"name": name, "op": "mass", "model": model, "n": n, "count": count, "slots": slots, "type": dtype,
            "gated": gated}


def _evict(name, model, count, keep, slots, sinks, recent):
    return {"name": name, "op": "evict", "model": model, "count": count, "keep": keep, "slots": slots, "sinks": sinks,
            "recent": recent}


def listed():
    return [
        # A few drafts of a short prompt, a token each: launch latency counts.
        _shared("drafts-1.7b", "1.7b", 4, 1, 1000, 40, "f32"),
        # The drafts of one prompt that sampled rows are drawn for, tails of ragged length.
        _shared("drafts-8b", "8b", 24, 1, 4001, 300, "f32"),
        # The hybrid's gated attention, six heads on a kv head.
        _shared("drafts-27b", "27b", 8, 1, 2047, 130, "f32", gated=True),
        # An offline run: many drafts behind a long prompt, tails of up to a thousand tokens.
        _shared("drafts-long-8b", "8b", 64, 1, 32768, 999, "f16"),
        # Proposed tokens of a dozen drafts checked at once, each draft with as many as it has.
        _shared("verify-8b", "8b", 12, 7, 6001, 200, "f16", ragged=True),
        # One token over a small model's full cache: launch latency counts.
        _mass("mass-token-1.7b", "1.7b", 1, 1019, 1024, "f32"),
        # One token over a long cache: the cache's bytes count.
        _mass("mass-token-long-8b", "8b", 1, 32700, 32768, "f16"),
        # A chat turn of ragged length through the hybrid's gated attention.
        _mass("mass-turn-27b", "27b", 27, 1900, 2048, "f32", gated=True),
        # A long prompt's chunk over what the chunks before it left.
        _mass("mass-chunk-8b", "8b", 1024, 2900, 4096, "f32"),
        # The same with queries and outputs in half precision, a ragged chunk over a longer cache.
        _mass("mass-chunk-half-8b", "8b", 1021, 7001, 8192, "f16"),
        # A full cache makes room for the next token.
        _evict("evict-one-8b", "8b", 4096, 4095, 4096, 4, 256),
        # A long prompt's cache is cut to a budget.
        _evict("evict-prompt-8b", "8b", 32768, 4096, 32768, 4, 512),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.random()
    model = rng.choice(("1.7b", "8b", "27b", "tiny"))
    heads, kv, dim = MODELS[model]
    dtype = rng.choice(("f32", "f32", "f16"))
    if kind < 0.45:
        batch = rng.choice((1, _log_int(rng, 2, 160), _log_int(rng, 2, 64), _log_int(rng, 2, 64)))
        n = rng.choice((1, 1, 1, rng.randint(2, 16)))
        prefix = rng.choice((_log_int(rng, 16, 32768), _log_int(rng, 256, 32768), _log_int(rng, 256, 8192), 0))
        tail = rng.choice((0, _log_int(rng, 1, 1000), _log_int(rng, 16, 1000)))
        most = 64 * 32 * 128 * 33268                                # a listed case's operations
        prefix = max(0, min(prefix, most // (batch * n * heads * dim) - tail))
        tail = min(tail, 64 * 8 * 128 * 999 // (batch * kv * dim))  # and its tails' bytes
        return _nameless(_shared("", model, batch, n, prefix, tail, dtype, n > 1 and rng.random() < 0.7,
                                 rng.random() < 0.3))
    if kind < 0.8:
        n = rng.choice((1, 1, _log_int(rng, 2, 40), _log_int(rng, 16, 1024), _log_int(rng, 16, 1024)))
        count = rng.choice((0, _log_int(rng, 1, 32768), _log_int(rng, 64, 32768), _log_int(rng, 64, 8192)))
        count = min(count, 1021 * 32 * 128 * 7001 // (n * heads * dim))
        return _nameless(_mass("", model, n, count, count + n + rng.choice((0, rng.randint(0, 500))), dtype,
                               rng.random() < 0.3))
    count = _log_int(rng, 64, 32768)
    keep = rng.choice((count - 1, rng.randint(1, count - 1), max(1, count - _log_int(rng, 1, 64)), max(1, count // 8)))
    recent = rng.randint(0, min(keep, 600))
    return _nameless(_evict("", model, count, keep, count + rng.choice((0, rng.randint(0, 500))),
                            min(keep - recent, rng.randint(0, 8)), recent))


def _nameless(case):
    del case["name"]
    return case


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own:
        _prepare_own(case, state)
    return state


def _inputs(case, seed):
    """Queries and keys as their norms and the rotation leave them (about unit variance a dim); slots
    behind the last row hold zeros."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 31)
    heads, kv, dim = MODELS[case["model"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "evict":
        count, slots = case["count"], case["slots"]
        s = {"kcache": normal(kv, slots, dim).half(), "vcache": normal(kv, slots, dim).half()}
        # Masses over many octaves, of some rows so little that none was left in the sum: 0.
        mass = torch.exp(2.5 * normal(kv, slots) - 3.0)
        mass[torch.rand((kv, slots), generator=gen, device="cuda") < 0.05] = 0.0
        # Positions of what earlier calls left: some are missing, and rows have moved.
        position = torch.empty((kv, slots), dtype=torch.int32, device="cuda")
        gone = torch.rand((kv, count), generator=gen, device="cuda") < 0.3
        position[:, :count] = torch.cumsum(1 + gone.int(), 1).int()
        position[:, :count] += 2 * count - position[:, count - 1:count]
        mixed = torch.argsort(torch.arange(count, device="cuda") + 0.2 * count * torch.rand((kv, count), generator=gen, device="cuda"))
        position[:, :count] = position[:, :count].gather(1, mixed)
        for name, t in (("mass", mass), ("positions", position)):
            t[:, count:] = 0
            s[name] = t
        s["kcache"][:, count:] = 0
        s["vcache"][:, count:] = 0
        return s
    t, n = TYPES[case["type"]], case["n"]
    rows = n * case.get("batch", 1)
    s = {"q": (1.5 * normal(rows, heads, dim)).to(t), "k": normal(rows, kv, dim).half(), "v": normal(rows, kv, dim).half(),
         "gate": normal(rows, heads, dim).to(t) if case["gated"] else None}
    if case["op"] == "shared":
        batch, tail = case["batch"], case["tail"]
        s["kprefix"], s["vprefix"] = (normal(kv, max(case["prefix"], 1), dim).half() for _ in range(2))
        s["ktail"], s["vtail"] = (normal(batch, kv, tail + n, dim).half() for _ in range(2))
        s["lengths"] = torch.randint(0, tail + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)
        s["counts"] = torch.randint(0, n + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32) if case["ragged"] else None
        behind = torch.arange(tail + n, device="cuda")[None, :] >= s["lengths"][:, None]
        for name in ("ktail", "vtail"):
            s[name].masked_fill_(behind[:, None, :, None], 0.0)
        return s
    slots, count = case["slots"], case["count"]
    s["kcache"], s["vcache"] = (normal(kv, slots, dim).half() for _ in range(2))
    s["mass"] = torch.exp(1.5 * normal(kv, slots) - 1.0)
    s["positions"] = torch.arange(slots, dtype=torch.int32, device="cuda").repeat(kv, 1)
    for name in ("kcache", "vcache", "mass", "positions"):
        s[name][:, count:] = 0
    return s


def run(state):
    op = state["case"]["op"]
    if own:
        return {"shared": _own_shared, "mass": _own_mass, "evict": _own_evict}[op](state)
    return {"shared": _plain_shared, "mass": _plain_mass, "evict": _plain_evict}[op](state)


# The framework's calls ------------------------------------------------------------------------------


def _prepare_own(case, s):
    """The shape, workspace and output buffers that a program keeps from call to call."""
    from trixium_amd import _lib
    from trixium_amd import layout as L
    heads, kv, dim = MODELS[case["model"]]
    strides = dict(n_head=heads, n_kv_head=kv, head_dim=dim, q_stride=heads * dim, kv_stride=kv * dim,
                   out_stride=heads * dim, gate_stride=heads * dim, gate_head_stride=dim, scale=1.0 / math.sqrt(dim),
                   kind=L.KIND_F16 if case.get("type") == "f16" else L.KIND_F32)
    size = ctypes.c_size_t()
    if case["op"] == "shared":
        s["shape"] = _lib.AttnSharedShape(prefix_slots=max(case["prefix"], 1), tail_slots=case["tail"] + case["n"], **strides)
        _lib.call("trx_attn_shared_geometry", ctypes.byref(s["shape"]), case["batch"], case["n"], case["prefix"],
                  ctypes.byref(size))
    else:
        s["shape"] = _lib.AttnMassShape(slots=case["slots"], **strides)
        if case["op"] == "mass":
            _lib.call("trx_attn_mass_geometry", ctypes.byref(s["shape"]), case["n"], ctypes.byref(size))
        else:
            _lib.call("trx_kv_evict_geometry", ctypes.byref(s["shape"]), ctypes.byref(size))
    s["workspace"] = torch.empty(max(size.value, 1), dtype=torch.uint8, device="cuda")
    if "q" in s:
        s["out"] = torch.zeros_like(s["q"])


def _pointer(t):
    return t.data_ptr() if t is not None else None


def _own_shared(s):
    from trixium_amd import _lib
    case = s["case"]
    _lib.call("trx_attn_shared", ctypes.byref(s["shape"]), case["batch"], case["n"], case["prefix"], s["lengths"].data_ptr(),
              _pointer(s["counts"]), s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["kprefix"].data_ptr(),
              s["vprefix"].data_ptr(), s["ktail"].data_ptr(), s["vtail"].data_ptr(), _pointer(s["gate"]),
              s["out"].data_ptr(), s["workspace"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return s["out"], s["ktail"], s["vtail"]


def _own_mass(s):
    from trixium_amd import _lib
    case = s["case"]
    _lib.call("trx_attn_mass", ctypes.byref(s["shape"]), case["n"], case["count"], case["count"], None, s["q"].data_ptr(),
              s["k"].data_ptr(), s["v"].data_ptr(), s["kcache"].data_ptr(), s["vcache"].data_ptr(), s["mass"].data_ptr(),
              s["positions"].data_ptr(), _pointer(s["gate"]), s["out"].data_ptr(), s["workspace"].data_ptr(),
              torch.cuda.current_stream().cuda_stream)
    return s["out"], s["kcache"], s["vcache"], s["mass"], s["positions"]


def _own_evict(s):
    from trixium_amd import _lib
    case = s["case"]
    _lib.call("trx_kv_evict", ctypes.byref(s["shape"]), case["count"], 2 * case["count"] + 1, None, case["keep"],
              case["sinks"], case["recent"], s["kcache"].data_ptr(), s["vcache"].data_ptr(), s["mass"].data_ptr(),
              s["positions"].data_ptr(), s["workspace"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return s["kcache"], s["vcache"], s["mass"], s["positions"]


# The plain forms ------------------------------------------------------------------------------------


def _gated(out, gate):
    return out if gate is None else out / (1.0 + torch.exp(-gate.float()))


def _plain_shared(s):
    case = s["case"]
    heads, kv, dim = MODELS[case["model"]]
    batch, n, P, rep = case["batch"], case["n"], case["prefix"], heads // kv
    slots = s["ktail"].shape[2]
    slot, new = torch.arange(slots, device="cuda"), torch.arange(n, device="cuda")
    counts = s["counts"] if s["counts"] is not None else torch.full((batch,), n, dtype=torch.int32, device="cuda")
    # The new rows into the tails first: row i of draft b stands in slot lengths[b] + i.
    at = slot[None] - s["lengths"][:, None]                                 # [batch, slots]: the new row of a slot
    fresh = ((at >= 0) & (at < counts[:, None]))[:, None, :, None]
    row = at.clamp(0, n - 1).long()[:, None, :, None].expand(batch, kv, slots, dim)
    for name, x in (("ktail", "k"), ("vtail", "v")):
        x = s[x].view(batch, n, kv, dim).transpose(1, 2).contiguous()
        s[name].copy_(torch.where(fresh, x.gather(2, row), s[name]))
    q = s["q"].float().view(batch, n, kv, rep, dim).permute(2, 0, 3, 1, 4)  # [kv, batch, rep, n, dim]
    kp, vp = s["kprefix"][:, :P].float(), s["vprefix"][:, :P].float()
    a = torch.matmul(q.reshape(kv, batch * rep * n, dim), kp.transpose(1, 2).contiguous())
    kt = s["ktail"].float().permute(1, 0, 3, 2).contiguous()                # [kv, batch, dim, slots]
    b = torch.matmul(q.reshape(kv, batch, rep * n, dim), kt)
    score = torch.cat([a.view(kv, batch, rep, n, P), b.view(kv, batch, rep, n, slots)], 4) / math.sqrt(dim)
    seen = slot[None, None] < (s["lengths"][:, None] + new[None] + 1)[:, :, None]       # [batch, n, slots]
    score[..., P:].masked_fill_(~seen[None, :, None], float("-inf"))
    p = torch.exp(score - score.amax(4, keepdim=True))
    p = p / p.sum(4, keepdim=True)
    out = torch.matmul(p[..., :P].reshape(kv, batch * rep * n, P), vp).view(kv, batch, rep * n, dim)
    vt = s["vtail"].float().transpose(0, 1).contiguous()
    out = out + torch.matmul(p[..., P:].reshape(kv, batch, rep * n, slots), vt)
    out = out.view(kv, batch, rep, n, dim).permute(1, 3, 0, 2, 4).reshape(batch * n, heads, dim)
    out = _gated(out, s["gate"])
    taken = (new[None] < counts[:, None]).reshape(batch * n, 1, 1)
    return torch.where(taken, out, torch.zeros_like(out)).to(s["q"].dtype), s["ktail"], s["vtail"]


def _plain_mass(s):
    case = s["case"]
    heads, kv, dim = MODELS[case["model"]]
    n, count, rep = case["n"], case["count"], heads // kv
    end = count + n
    s["kcache"][:, count:end] = s["k"].transpose(0, 1)
    s["vcache"][:, count:end] = s["v"].transpose(0, 1)
    s["positions"][:, count:end] = torch.arange(count, end, dtype=torch.int32, device="cuda")
    q = s["q"].float().view(n, kv, rep, dim).permute(1, 2, 0, 3).reshape(kv, rep * n, dim)
    K, V = s["kcache"][:, :end].float(), s["vcache"][:, :end].float()
    score = torch.matmul(q, K.transpose(1, 2).contiguous()).view(kv, rep, n, end) / math.sqrt(dim)
    later = torch.arange(end, device="cuda")[None] > count + torch.arange(n, device="cuda")[:, None]
    score = score.masked_fill(later, float("-inf"))
    p = torch.exp(score - score.amax(3, keepdim=True))
    p = (p / p.sum(3, keepdim=True)).view(kv, rep * n, end)
    out = torch.matmul(p, V).view(kv, rep, n, dim).permute(2, 0, 1, 3).reshape(n, heads, dim)
    given = p.sum(1)
    s["mass"][:, :count] += given[:, :count]
    s["mass"][:, count:end] = given[:, count:]
    return _gated(out, s["gate"]).to(s["q"].dtype), s["kcache"], s["vcache"], s["mass"], s["positions"]


def _plain_evict(s):
    case = s["case"]
    count, keep, pos = case["count"], case["keep"], 2 * case["count"] + 1
    kv, _, dim = s["kcache"].shape
    position = s["positions"][:, :count]
    first = (position < case["sinks"]) | (position >= pos - case["recent"])
    key = torch.where(first, torch.full_like(s["mass"][:, :count], float("inf")), s["mass"][:, :count])
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    stays = torch.zeros((kv, count), dtype=torch.bool, device="cuda").scatter_(1, order[:, :keep], True)
    slot = torch.arange(count, device="cuda")[None]
    # Slots of rows that go below keep, and of rows that stay past it, each in order, then the rest.
    to = torch.sort(torch.where(~stays & (slot < keep), slot, count + slot), 1).values
    frm = torch.sort(torch.where(stays & (slot >= keep), slot, count + slot), 1).values
    m = min(keep, count - keep)
    moved = (frm[:, :m] < count)
    # Where nothing moves any more, a slot past keep is written with itself.
    to, frm = to[:, :m], frm[:, :m] % count
    src = torch.where(moved, frm, torch.full_like(frm, count - 1))
    dst = torch.where(moved, to % count, torch.full_like(to, count - 1))
    for name in ("mass", "positions"):
        s[name].scatter_(1, dst, s[name].gather(1, src))
    for name in ("kcache", "vcache"):
        wide = src[:, :, None].expand(kv, m, dim)
        s[name].scatter_(1, dst[:, :, None].expand(kv, m, dim), s[name].gather(1, wide))
    return s["kcache"], s["vcache"], s["mass"], s["positions"]


# 64 bits ----------------------------------------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    return {"shared": _exact_shared, "mass": _exact_mass, "evict": _exact_evict}[case["op"]](case, s)


def _softmax64(e):
    e = torch.exp(e - e.max(dim=1).values[:, None])
    return e / e.sum(dim=1)[:, None]


def _exact_shared(case, s):
    """Draft by draft and head by head over the rows that it sees, put one behind the other."""
    heads, kv, dim = MODELS[case["model"]]
    n, P = case["n"], case["prefix"]
    lengths = s["lengths"].tolist()
    counts = s["counts"].tolist() if s["counts"] is not None else [n] * case["batch"]
    out = torch.zeros((case["batch"], n, heads, dim), dtype=torch.float64, device="cuda")
    kt, vt = s["ktail"].double(), s["vtail"].double()
    kn, vn = s["k"].view(-1, n, kv, dim), s["v"].view(-1, n, kv, dim)
    q = s["q"].view(-1, n, heads, dim)
    for b, (have, c) in enumerate(zip(lengths, counts)):
        if c == 0:
            continue
        for g in range(kv):
            K = torch.cat([s["kprefix"][g, :P], s["ktail"][b, g, :have], kn[b, :c, g]]).double()
            V = torch.cat([s["vprefix"][g, :P], s["vtail"][b, g, :have], vn[b, :c, g]]).double()
            for h in range(g * heads // kv, (g + 1) * heads // kv):
                e = q[b, :c, h].double() @ K.T / dim ** 0.5
                for i in range(c):
                    e[i, P + have + i + 1:] = -math.inf
                out[b, :c, h] = _softmax64(e) @ V
        kt[b, :, have:have + c] = kn[b, :c].double().transpose(0, 1)
        vt[b, :, have:have + c] = vn[b, :c].double().transpose(0, 1)
    out = out.view(-1, heads, dim)
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].double())
    return out, kt, vt


def _exact_mass(case, s):
    heads, kv, dim = MODELS[case["model"]]
    n, count = case["n"], case["count"]
    out = torch.empty((n, heads, dim), dtype=torch.float64, device="cuda")
    kc, vc, mass = s["kcache"].double(), s["vcache"].double(), s["mass"].double()
    kc[:, count:count + n], vc[:, count:count + n] = s["k"].double().transpose(0, 1), s["v"].double().transpose(0, 1)
    position = s["positions"].cpu().numpy()
    position[:, count:count + n] = np.arange(count, count + n)
    for h in range(heads):
        g = h * kv // heads
        for r in range(0, n, 128):
            m = min(n - r, 128)
            seen = count + r + m
            e = s["q"][r:r + m, h].double() @ kc[g, :seen].T / dim ** 0.5
            e += torch.full((m, seen), -math.inf, dtype=torch.float64, device="cuda").triu(count + r + 1)
            p = _softmax64(e)
            out[r:r + m, h] = p @ vc[g, :seen]
            mass[g, :seen] += p.sum(0)
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].double())
    return out, kc, vc, mass, torch.from_numpy(position)


def _exact_evict(case, s):
    """On the host: the rows of each kv head sorted by what keeps them."""
    count, keep, pos = case["count"], case["keep"], 2 * case["count"] + 1
    a = {name: t.cpu().numpy() for name, t in s.items()}
    for g in range(a["mass"].shape[0]):
        at = a["positions"][g, :count]
        first = (at < case["sinks"]) | (at >= pos - case["recent"])
        order = np.lexsort((np.arange(count), -a["mass"][g, :count].astype(np.float64), ~first))
        stays = set(order[:keep].tolist())
        holes = [i for i in range(keep) if i not in stays]
        for to, frm in zip(holes, sorted(i for i in stays if i >= keep)):
            for name in ("kcache", "vcache", "mass", "positions"):
                a[name][g, to] = a[name][g, frm]
    return tuple(torch.from_numpy(a[name] if name == "positions" else a[name].astype(np.float64))
                 for name in ("kcache", "vcache", "mass", "positions"))


def work(case):
    heads, kv, dim = MODELS[case["model"]]
    if case["op"] == "evict":
        # Masses and positions read once; the rows that are expected past keep read and written.
        moved = (case["count"] - case["keep"]) * case["keep"] / case["count"]
        return {"bytes": int(kv * (8 * case["count"] + 2 * moved * (4 * dim + 8))), "flops": kv * case["count"]}
    n, size = case["n"], 4 if case["type"] == "f32" else 2
    ends = 3 if case["gated"] else 2                                # q and out, and the gate
    if case["op"] == "mass":
        pairs = n * case["count"] + n * (n + 1) // 2
        moved = (ends * n * heads * dim * size + 4 * kv * dim * (case["count"] + 2 * n)
                 + 4 * kv * (2 * case["count"] + 2 * n))
        return {"bytes": moved, "flops": 4 * heads * dim * pairs + 2 * heads * pairs}
    # Tails and counts at their mean.
    batch, mean = case["batch"], case["tail"] / 2
    taken = n / 2 if case["ragged"] else n
    pairs = batch * taken * (case["prefix"] + mean + (taken + 1) / 2)
    moved = (ends * batch * taken * heads * dim * size + 4 * kv * dim * (case["prefix"] + batch * (mean + 2 * taken))
             + 4 * batch)
    return {"bytes": int(moved), "flops": int(4 * heads * dim * pairs)}
