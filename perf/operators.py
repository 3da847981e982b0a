"""Two operators of decoding past the context window, over the sizes that the configurations run.

`attend`: attention of the next n positions with a sliding window and a few first positions that
stay visible, over the ring of K and V rows that the decoder keeps (`trx_attn_window`). Position p
of the ring takes slot p where p < pin, else slot pin + (p - pin) % (slots - pin); a query at
position t sees the positions u <= t with u < sinks or u > t - window. The new rows of K and V
take their slots, so the ring is an output too.

`sample`: one token per row of logits from the whole vocabulary, by temperature, top-k, top-p and
min-p, from a given uniform number (`trx_sample_rows`). Tokens stand in the order of their logits,
largest first, equal ones by index; the first top_k stay, of those the smallest prefix that holds
top_p of their mass, of those the ones whose probability is at least min_p of the largest. The
token is the first in index order at which the mass that stayed passes u times its total; beside it
comes its log-probability among those that stayed.
"""

import ctypes
import math

import numpy as np
import torch

own = False

# (heads, kv heads, head dim, KV slots) of the shipped configurations.
MODELS = {"1.7b": (16, 8, 128, 1024), "8b": (32, 8, 128, 4096), "27b": (24, 4, 256, 2048), "tiny": (4, 2, 64, 128)}
VOCAB = {"1.7b": 151936, "8b": 151936, "27b": 248320, "tiny": 2048}
TYPES = {"f32": torch.float32, "f16": torch.float16}
# (temperature, top_k, top_p, min_p): a chat's nucleus, a short list, every filter at once, no
# filter at all, a floor alone, the largest logit.
SETTINGS = {"nucleus": (0.8, 0, 0.9, 0.0), "short": (0.7, 50, 1.0, 0.0), "all": (0.9, 200, 0.95, 0.02),
            "open": (1.0, 0, 1.0, 0.0), "floor": (1.3, 0, 1.0, 0.05), "greedy": (0.0, 0, 1.0, 0.0)}
MIXED = ("nucleus", "short", "all", "open", "floor", "nucleus", "all", "greedy")


def _attend(name, model, n, slots, pin, window, sinks, pos, dtype, gated=False):
    return {"name": name, "op": "attend", "model": model, "n": n, "slots": slots, "pin": pin, "window": window,
            "sinks": sinks, "pos": pos, "type": dtype, "gated": gated}


def listed():
    return [
        # One token of a small model whose window is full: launch latency counts.
        _attend("token-1.7b", "1.7b", 1, 1024, 4, 1020, 4, 9000, "f32"),
        # One token of the hybrid's gated attention, past its window, six heads on a kv head.
        _attend("token-27b", "27b", 1, 2048, 64, 1984, 64, 5001, "f32", True),
        # One token over a long ring: the cache's bytes count.
        _attend("token-long-8b", "8b", 1, 32768, 4, 32764, 4, 100003, "f16"),
        # A short chat turn of ragged length behind a full window, the first turn pinned.
        _attend("turn-8b", "8b", 27, 4096, 61, 4000, 61, 6007, "f32"),
        # A long prompt's chunk behind a window of half the ring.
        _attend("chunk-8b", "8b", 1024, 4096, 4, 2048, 4, 12288, "f32"),
        # The same with queries and outputs in half precision, a longer window, a ragged chunk.
        _attend("chunk-half-8b", "8b", 1021, 8192, 16, 6000, 16, 20011, "f16"),
        # A chunk of the hybrid's gated attention that begins inside the window's first filling.
        _attend("chunk-27b", "27b", 509, 2048, 4, 1500, 4, 700, "f32", True),
        # The tokenwise draw of a small model with the nucleus of a chat.
        {"name": "draw-1.7b", "op": "sample", "vocab": 151936, "n": 1, "settings": "nucleus", "type": "f32"},
        # The hybrid's larger vocabulary with every filter at once.
        {"name": "draw-27b", "op": "sample", "vocab": 248320, "n": 1, "settings": "all", "type": "f32"},
        # Drafts of one prompt, each row with settings of its own, logits in half precision (ties).
        {"name": "draw-rows-8b", "op": "sample", "vocab": 151936, "n": 24, "settings": "mixed", "type": "f16"},
        # Many rows from nuclei, as an offline sampling run has them.
        {"name": "draw-many-27b", "op": "sample", "vocab": 248320, "n": 160, "settings": "nucleus", "type": "f32"},
        # Many rows without a filter.
        {"name": "draw-open-8b", "op": "sample", "vocab": 151936, "n": 128, "settings": "open", "type": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    if rng.random() < 0.55:
        model = rng.choice(("1.7b", "8b", "27b", "tiny"))
        heads, kv, dim, _ = MODELS[model]
        n = rng.choice((1, 1, _log_int(rng, 2, 40), _log_int(rng, 16, 1024), _log_int(rng, 16, 1024)))
        pin = rng.choice((0, 4, 4, rng.randint(1, 64)))
        window = _log_int(rng, 16, 32768 if n == 1 else 6000)
        most = 68719476736 // (4 * heads * dim * n)                 # a listed chunk's work
        window = max(1, min(window, most))
        # Room for the chunk behind the window, so that a pass leaves what the next one reads.
        slots = pin + window + n - 1 + rng.choice((0, rng.randint(0, 700)))
        pos = rng.choice((0, rng.randint(0, slots), _log_int(rng, slots, 40 * slots)))
        return {"op": "attend", "model": model, "n": n, "slots": slots, "pin": pin, "window": window,
                "sinks": rng.randint(0, pin), "pos": pos, "type": rng.choice(("f32", "f32", "f16")),
                "gated": rng.random() < 0.3}
    vocab = rng.choice((151936, 248320, 2048, _log_int(rng, 500, 248320)))
    n = rng.choice((1, _log_int(rng, 1, 160), _log_int(rng, 1, 160)))
    return {"op": "sample", "vocab": vocab, "n": n, "settings": rng.choice(tuple(SETTINGS) + ("mixed", "mixed")),
            "type": rng.choice(("f32", "f32", "f16"))}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)
    state = _prepare_attend(case, gen) if case["op"] == "attend" else _prepare_sample(case, gen)
    state["case"] = case
    if own:
        _prepare_own(case, state)
    return state


def _prepare_attend(case, gen):
    """Queries and keys as their norms and the rotation leave them (about unit variance a dim), a
    ring that holds what came before."""
    heads, kv, dim, _ = MODELS[case["model"]]
    n, slots, t = case["n"], case["slots"], TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    state = {"q": (1.5 * normal(n, heads, dim)).to(t), "k": normal(n, kv, dim).half(), "v": normal(n, kv, dim).half(),
             "kcache": normal(kv, slots, dim).half(), "vcache": normal(kv, slots, dim).half(),
             "gate": normal(n, heads, dim).to(t) if case["gated"] else None}
    if case["pos"] < slots:                       # slots that no position has taken yet
        state["kcache"][:, case["pos"]:] = 0
        state["vcache"][:, case["pos"]:] = 0
    return state


def _prepare_sample(case, gen):
    """Logits that fall with the logarithm of the rank, as a language model's do, with noise on
    them, in a random order; and each row's settings."""
    n, V = case["n"], case["vocab"]
    fall = 0.9 + 0.9 * torch.rand((n, 1), generator=gen, device="cuda")
    rank = torch.empty((n, V), device="cuda")
    for r in range(n):
        rank[r] = torch.randperm(V, generator=gen, device="cuda").float() + 1.0
    logits = 12.0 - fall * rank.log_() + 0.5 * torch.randn((n, V), generator=gen, device="cuda")
    names = [MIXED[r % len(MIXED)] if case["settings"] == "mixed" else case["settings"] for r in range(n)]
    rows = [SETTINGS[name] for name in names]
    return {"logits": logits.to(TYPES[case["type"]]), "u": torch.rand(n, generator=gen, device="cuda"),
            "temperature": torch.tensor([r[0] for r in rows], device="cuda"),
            "top_k": torch.tensor([r[1] for r in rows], dtype=torch.int32, device="cuda"),
            "top_p": torch.tensor([r[2] for r in rows], device="cuda"),
            "min_p": torch.tensor([r[3] for r in rows], device="cuda")}


def run(state):
    if own:
        return _own_attend(state) if state["case"]["op"] == "attend" else _own_sample(state)
    return _plain_attend(state) if state["case"]["op"] == "attend" else _plain_sample(state)


# The framework's calls ------------------------------------------------------------------------------


def _prepare_own(case, state):
    """The shape, workspace and output buffers that a program keeps from call to call."""
    from trixium_amd import _lib
    from trixium_amd import layout as L
    kind = L.KIND_F32 if case["type"] == "f32" else L.KIND_F16
    size = ctypes.c_size_t()
    if case["op"] == "attend":
        heads, kv, dim, _ = MODELS[case["model"]]
        state["shape"] = _lib.AttnWindowShape(
            kind=kind, n_head=heads, n_kv_head=kv, head_dim=dim, slots=case["slots"], pin=case["pin"],
            window=case["window"], sinks=case["sinks"], q_stride=heads * dim, kv_stride=kv * dim,
            out_stride=heads * dim, gate_stride=heads * dim, gate_head_stride=dim, scale=1.0 / math.sqrt(dim))
        _lib.call("trx_attn_window_geometry", ctypes.byref(state["shape"]), case["n"], ctypes.byref(size))
        state["out"] = torch.empty_like(state["q"])
    else:
        state["kind"] = kind
        table = torch.stack([state["temperature"], state["top_k"].view(torch.float32), state["top_p"], state["min_p"]], 1)
        state["rows"] = table.contiguous()        # struct trx_sampling [n]
        _lib.call("trx_sample_rows_geometry", case["vocab"], case["n"], ctypes.byref(size))
        state["tokens"] = torch.empty(case["n"], dtype=torch.int32, device="cuda")
        state["logp"] = torch.empty(case["n"], device="cuda")
    state["workspace"] = torch.empty(max(size.value, 1), dtype=torch.uint8, device="cuda")


def _own_attend(s):
    from trixium_amd import _lib
    gate = s["gate"].data_ptr() if s["gate"] is not None else None
    _lib.call("trx_attn_window", ctypes.byref(s["shape"]), s["case"]["n"], s["case"]["pos"], None, s["q"].data_ptr(),
              s["k"].data_ptr(), s["v"].data_ptr(), s["kcache"].data_ptr(), s["vcache"].data_ptr(), gate,
              s["out"].data_ptr(), s["workspace"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return s["out"], s["kcache"], s["vcache"]


def _own_sample(s):
    from trixium_amd import _lib
    _lib.call("trx_sample_rows", s["logits"].data_ptr(), s["kind"], s["case"]["n"], s["case"]["vocab"], s["case"]["vocab"],
              s["rows"].data_ptr(), 1, s["u"].data_ptr(), s["tokens"].data_ptr(), s["logp"].data_ptr(),
              s["workspace"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return s["tokens"], s["logp"]


# The plain forms ------------------------------------------------------------------------------------


def _slot(case, u):
    return torch.where(u < case["pin"], u, case["pin"] + (u - case["pin"]) % (case["slots"] - case["pin"]))


def _plain_attend(s):
    case = s["case"]
    heads, kv, dim, _ = MODELS[case["model"]]
    n, pos = case["n"], case["pos"]
    # The positions that any query sees: the first ones, then the window from the first query's on.
    low = max(case["sinks"], pos - case["window"] + 1)
    first = torch.arange(min(case["sinks"], pos + n), device="cuda")
    seen = torch.cat([first, torch.arange(min(low, pos + n), pos + n, device="cuda")])
    old, new = seen[seen < pos], seen[seen >= pos] - pos
    K = torch.cat([s["kcache"][:, _slot(case, old)], s["k"][new].transpose(0, 1)], dim=1).float()
    V = torch.cat([s["vcache"][:, _slot(case, old)], s["v"][new].transpose(0, 1)], dim=1).float()
    rep = heads // kv
    q = s["q"].float().view(n, kv, rep, dim).permute(1, 2, 0, 3).reshape(kv, rep * n, dim)
    score = torch.matmul(q, K.transpose(1, 2).contiguous()).view(kv, rep, n, -1) / math.sqrt(dim)
    t = torch.arange(pos, pos + n, device="cuda")[:, None]
    mask = (seen <= t) & ((seen < case["sinks"]) | (seen > t - case["window"]))
    score = score.masked_fill(~mask, float("-inf"))
    p = torch.exp(score - score.amax(dim=3, keepdim=True))
    p = p / p.sum(dim=3, keepdim=True)
    out = torch.matmul(p.view(kv, rep * n, -1), V).view(kv, rep, n, dim).permute(2, 0, 1, 3).reshape(n, heads, dim)
    if s["gate"] is not None:
        out = out / (1.0 + torch.exp(-s["gate"].float()))
    # The rows that a later one of the same call does not replace, into their slots.
    last = torch.arange(pos, pos + n, device="cuda")
    last = last[(last < case["pin"]) | (last > pos + n - 1 - (case["slots"] - case["pin"]))]
    s["kcache"][:, _slot(case, last)] = s["k"][last - pos].transpose(0, 1)
    s["vcache"][:, _slot(case, last)] = s["v"][last - pos].transpose(0, 1)
    return out.to(s["q"].dtype), s["kcache"], s["vcache"]


def _plain_sample(s):
    """In 64 bits: the mass's sums run over the vocabulary, and a token changes at a border."""
    logits = s["logits"].double()
    n, V = logits.shape
    T = s["temperature"].double()[:, None]
    top = logits.amax(dim=1, keepdim=True)
    mass = torch.exp((logits - top) / torch.where(T > 0, T, torch.ones_like(T)))
    by_size, order = torch.sort(logits, dim=1, descending=True, stable=True)
    m = mass.gather(1, order)
    k = s["top_k"].long()[:, None]
    rank = torch.arange(V, device="cuda")[None, :]
    m = torch.where((k <= 0) | (rank < k), m, torch.zeros_like(m))
    before = torch.cumsum(m, dim=1)
    total = before[:, -1:].clone()
    before -= m
    p = s["top_p"].double()[:, None]
    stays = (m > 0) & ((p >= 1.0) | (before < p * total)) & (m >= s["min_p"].double()[:, None])
    kept = torch.zeros_like(m).scatter_(1, order, torch.where(stays, m, torch.zeros_like(m)))
    run_ = torch.cumsum(kept, dim=1)
    picked = (run_ <= s["u"].double()[:, None] * run_[:, -1:]).sum(dim=1)
    share = kept.gather(1, picked[:, None])[:, 0] / run_[:, -1]
    token = torch.where(T[:, 0] > 0, picked, order[:, 0])
    logp = torch.where(T[:, 0] > 0, torch.log(share), torch.zeros_like(share))
    return token.to(torch.int32), logp.to(torch.float32)


# 64 bits ----------------------------------------------------------------------------------------------


def exact(case, seed):
    return _exact_attend(case, seed) if case["op"] == "attend" else _exact_sample(case, seed)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)
    return _prepare_attend(case, gen) if case["op"] == "attend" else _prepare_sample(case, gen)


def _exact_attend(case, seed):
    """The ring unrolled to absolute positions, then each head and block of queries by the sum's
    definition, its scores taken relative to their largest."""
    s = _inputs(case, seed)
    heads, kv, dim, _ = MODELS[case["model"]]
    n, pos, pin, ring = case["n"], case["pos"], case["pin"], case["slots"] - case["pin"]
    where = {}
    for u in list(range(min(pin, pos))) + list(range(max(pin, pos - ring), pos)):
        where[u] = u if u < pin else pin + (u - pin) % ring
    seen = [u for u in range(min(case["sinks"], pos))]
    seen += [u for u in range(max(len(seen), pos - case["window"] + 1, 0), pos)]
    at = torch.tensor([where[u] for u in seen], dtype=torch.long, device="cuda")
    u = torch.tensor(seen + list(range(pos, pos + n)), dtype=torch.long, device="cuda")
    out = torch.empty((n, heads, dim), dtype=torch.float64, device="cuda")
    for h in range(heads):
        g = h * kv // heads
        K = torch.cat([s["kcache"][g][at], s["k"][:, g]]).double()
        V = torch.cat([s["vcache"][g][at], s["v"][:, g]]).double()
        for r in range(0, n, 256):
            t = torch.arange(pos + r, pos + min(n, r + 256), device="cuda")
            e = s["q"][r:r + 256, h].double() @ K.T / dim ** 0.5
            hidden = (u[None] > t[:, None]) | ((u[None] >= case["sinks"]) & (u[None] <= t[:, None] - case["window"]))
            e[hidden] = -math.inf
            e = torch.exp(e - e.max(dim=1).values[:, None])
            out[r:r + 256, h] = (e @ V) / e.sum(dim=1)[:, None]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].double())
    kc, vc = s["kcache"].double(), s["vcache"].double()
    slots = [p if p < pin else pin + (p - pin) % ring for p in range(pos, pos + n)]
    final = {slot: r for r, slot in enumerate(slots)}              # a slot's last row stays
    to = torch.tensor(list(final), device="cuda")
    frm = torch.tensor(list(final.values()), device="cuda")
    kc[:, to] = s["k"][frm].double().transpose(0, 1)
    vc[:, to] = s["v"][frm].double().transpose(0, 1)
    return out, kc, vc


def _exact_sample(case, seed):
    """Row by row on the host: the cut is looked for among the sorted values, then the draw goes
    over the vocabulary."""
    if case["n"] * case["vocab"] > 60_000_000:
        return None
    s = {k: v.cpu().numpy() for k, v in _inputs(case, seed).items()}
    tokens, logp = np.empty(case["n"], np.int32), np.zeros(case["n"])
    for r in range(case["n"]):
        x = s["logits"][r].astype(np.float64)
        if not s["temperature"][r] > 0:
            tokens[r] = int(np.flatnonzero(x == x.max())[0])
            continue
        w = np.exp((x - x.max()) / np.float64(s["temperature"][r]))
        rank = np.argsort(-x, kind="stable")
        if 0 < s["top_k"][r] < rank.size:
            rank = rank[:s["top_k"][r]]
        if s["top_p"][r] < 1:
            c = np.cumsum(w[rank])
            rank = rank[:int(np.searchsorted(c, np.float64(s["top_p"][r]) * c[-1])) + 1]
        rank = rank[w[rank] >= np.float64(s["min_p"][r])]
        rank = np.sort(rank)
        c = np.cumsum(w[rank])
        tokens[r] = rank[int(np.searchsorted(c, np.float64(s["u"][r]) * c[-1], side="right"))]
        logp[r] = math.log(w[tokens[r]] / c[-1])
    return torch.from_numpy(tokens), torch.from_numpy(logp)


def work(case):
    if case["op"] == "sample":
        # Every logit read once; a subtraction, a product, an exponential and a sum for each.
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": case["n"] * (case["vocab"] * size + 24), "flops": 4 * case["n"] * case["vocab"]}
    heads, kv, dim, _ = MODELS[case["model"]]
    n, pos, window, sinks = case["n"], case["pos"], case["window"], case["sinks"]
    pairs = 0
    for t in range(pos, pos + n):
        low = max(0, t - window + 1)
        pairs += t + 1 - low + min(sinks, low)
    old = pos - max(0, pos - window + 1) + min(sinks, max(0, pos - window + 1))
    size = 4 if case["type"] == "f32" else 2
    # q and out (and the gate), the rows seen before, the new rows read and stored in the ring.
    moved = n * heads * dim * size * (3 if case["gated"] else 2) + 2 * 2 * kv * dim * (old + 2 * n)
    return {"bytes": moved, "flops": 4 * heads * dim * pairs}
