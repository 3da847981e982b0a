"""Decoding past the KV window as a program runs it: prompts batched over the ring (trx_model_prefill's
chunks past max_ctx on the window attention) and tokens drawn from the whole vocabulary
(trx_model_set_vocab_sampling), against the float oracle's ring, against one position per forward, and
against the sampler's definition on the decoder's own logits."""

import numpy as np
import pytest

from oracle import sampler as S
from oracle.floatref import FloatRef
from test_sample_rows_gpu import oracle as draw
from trixium_amd import _lib, bons, configs as C

CAP, PIN = 20, 5
LOGIT_RTOL = 1e-2                       # the decoder's float tolerance


def _decoder(path, **kw):
    from trixium_amd.model import Decoder
    return Decoder.from_image(path, **kw)


def _tokens(golden, name, n):
    return ((golden[f"prompt/{name}"] + golden[f"fastref_tokens/{name}"]) * 4)[:n]


def _rel_err(got, ref):
    return float(np.max(np.abs(np.asarray(got, np.float64) - ref)) / np.max(np.abs(ref)))


def test_vocab_sampling_refuses_without_a_model():
    lib = _lib.lib()
    assert lib.trx_model_set_vocab_sampling(None, 1.0, 0, 1.0, 0.0, 1.0, 1) == _lib.TRX_E_INVALID


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiny-hybrid", "tiny-qwen3"])
@pytest.mark.parametrize("chunk", [4, 7, 64])
def test_chunks_over_the_ring_match_the_oracle(tiny_images, golden, name, chunk):
    """Feeds of every kind of length across and past a 20-slot window, chunks shorter and longer than it;
    a feed takes at most a window. Every feed's last logits are compared."""
    path = tiny_images[(name, True)]
    toks = _tokens(golden, name, 100)
    dec = _decoder(path, max_ctx=CAP, prefill_chunk=chunk)
    dec.set_kv_ring(1, PIN)
    dec.reset()
    ref = FloatRef(bons.BONSReader(path), kv_fp16=True)
    ref.set_kv_ring(CAP, PIN)
    ref.reset()
    at, worst = 0, 0.0
    for n in (13, 20, 1, 5, 20, 2, 19, 6, 14):
        a, b = dec.forward(toks[at:at + n]), ref.forward(toks[at:at + n])
        at += n
        err = _rel_err(a, b)
        worst = max(worst, err)
        assert err <= LOGIT_RTOL, (at, n, err)
        assert dec.position() == at - 1
    print(f"{name} chunk {chunk}: {at} positions, worst rel err {worst:.2e}")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", ["1.7b", "27b", "tiny-hybrid"])
def test_chunks_over_the_ring_equal_single_positions(shape):
    """The shipped widths: the same positions batched and one a forward, then a token and a checkpoint
    after them. The attention's two forms differ by fp32 rounding."""
    from trixium_amd.model import Decoder
    base = {"1.7b": C.QWEN3_1P7B, "27b": C.QWEN35_27B, "tiny-hybrid": C.TINY_HYBRID}[shape]
    layers = 4 if shape != "1.7b" else 2
    mc = base.replace(name=base.name + "-few", n_layer=layers, max_ctx=160, vocab=1024,
                      layer_types=base.layer_types[:layers])
    rng = np.random.default_rng(1)
    feeds = [rng.integers(0, 1024, n).tolist() for n in (150, 61, 160, 33)]
    got = []
    for chunk in (0, 48):
        dec = Decoder.synthetic(mc, seed=3, prefill_chunk=chunk)
        dec.set_kv_ring(1, 9)
        dec.reset()
        out = [dec.forward(f) for f in feeds]
        out.append(dec.forward([7]))
        dec.checkpoint()
        out.append(dec.forward([8]))
        dec.restore()
        assert np.array_equal(dec.forward([8]), out[-1])
        got.append(out)
        dec.close()
    errs = [_rel_err(b, a) for a, b in zip(*got)]
    print(shape, ["%.1e" % e for e in errs])
    assert max(errs) <= 2e-3


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(temperature=0.8, top_p=0.9), dict(temperature=1.2, top_k=40, min_p=0.02),
                                dict(temperature=0.7, top_k=300, top_p=0.95, repetition=1.3),
                                dict(temperature=0.0, repetition=1.5)], ids=str)
@pytest.mark.parametrize("use_graph", [True, False])
def test_draws_and_chunks_together(tiny_images, golden, kw, use_graph):
    """A conversation past the window: turns batched over the ring, replies drawn. Each drawn token is the
    definition's on the decoder's logits of its position (read back token by token), with the
    firmware's stream and the penalty over the last 64 tokens; and the replies generated in one
    call are the same."""
    name, seed = "tiny-hybrid", 4321
    path = tiny_images[(name, True)]
    turns = [_tokens(golden, name, 16), _tokens(golden, name, 31)[16:], [5, 9, 5, 9, 11]]
    full = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, repetition=1.0), **kw}

    def fresh():
        dec = _decoder(path, max_ctx=CAP, max_new=16, prefill_chunk=8, use_graph=use_graph)
        dec.set_kv_ring(1, PIN)
        dec.set_vocab_sampling(seed=seed, **kw)
        dec.reset()
        return dec

    dec = fresh()
    replies = [dec.generate(t, 12) for t in turns]
    dec.close()
    dec, rng, history = fresh(), seed, []
    for turn, reply in zip(turns, replies):
        feed = list(turn)
        for want in reply:
            got = dec.generate(feed, 1)[0]
            history += feed
            lg = dec.logits().copy()
            for t in set(history[-64:]) if full["repetition"] > 1 else ():
                r = np.float32(full["repetition"])
                lg[t] = lg[t] / r if lg[t] > 0 else lg[t] * r
            u = 0.0
            if full["temperature"] > 0:
                rng = S.xorshift32(rng)
                u = np.float32(rng >> 8) * np.float32(1.0 / 16777216.0)
            t, _ = draw(lg, u, full["temperature"], full["top_k"], full["top_p"], full["min_p"])
            assert got == t == want, (len(history), got, t, want)
            feed = [got]
        # The last token of a reply is not fed: the next turn follows it in the definition's loop too.
    assert dec.position() == len(history) - 1 > 2 * CAP
    dec.set_vocab_sampling(temperature=0.0)
    dec.reset()
    assert dec.generate(golden[f"prompt/{name}"], 4) == golden[f"fastref_tokens/{name}"][:4]


@pytest.mark.gpu
def test_the_penalty_reaches_back_over_calls(tiny_images, golden):
    """Tokens that an earlier call generated without feeding them count as the last 64's in the next call,
    for both samplers: with a penalty that forbids what it meets, three calls of greedy tokens repeat
    none."""
    name = "tiny-qwen3"
    for firmware in (False, True):
        dec = _decoder(tiny_images[(name, True)], max_new=16)
        if firmware:
            dec.set_sampling(0.0, 1.0, 1e30)
        else:
            dec.set_vocab_sampling(temperature=0.0, repetition=1e30)
        dec.reset()
        prompt = golden[f"prompt/{name}"][:4]
        seen = dec.generate(prompt, 12)
        for _ in range(2):
            seen += dec.generate([seen[-1]], 12)
        assert len(set(seen + prompt)) == len(seen) + len(set(prompt)), (firmware, seen)
        dec.close()


@pytest.mark.gpu
def test_checkpoint_replays_a_draw_and_samplers_switch(tiny_images, golden):
    name = "tiny-qwen3"
    dec = _decoder(tiny_images[(name, True)], max_new=32)
    prompt = golden[f"prompt/{name}"]
    dec.set_vocab_sampling(temperature=1.5, seed=99)
    dec.reset()
    dec.generate(prompt, 3)
    dec.checkpoint()
    a = dec.generate([1], 8)
    dec.restore()
    assert dec.generate([1], 8) == a
    # The firmware's sampler again, with the stream that the seed sets.
    dec.set_sampling(0.8, 0.9, 1.3, 1234)
    dec.reset()
    firm = dec.generate(prompt, 8)
    dec.set_vocab_sampling(temperature=1.5, top_k=5, repetition=1.2, seed=7)
    dec.set_sampling(0.8, 0.9, 1.3, 1234)
    dec.reset()
    assert dec.generate(prompt, 8) == firm
    dec.set_sampling()
    dec.reset()
    assert dec.generate(prompt, 8) == golden[f"fastref_tokens/{name}"][:8]


@pytest.mark.gpu
def test_chat_goes_on_past_the_window(tiny_images):
    """The chat loop on a hybrid: turns and replies past the window, batched and drawn; a turn longer than
    the window is refused as before."""
    from trixium_amd.chat import Chat

    class Words:
        im_end = 1023

        def turn(self, text, system, first, prev_closed):
            return [3 + len(w) for w in text.split()]

        encode = turn

        def stream_decoder(self):
            return lambda t: f"{t} "

    dec = _decoder(tiny_images[("tiny-hybrid", True)], max_ctx=CAP, max_new=1, prefill_chunk=16)
    dec.set_vocab_sampling(temperature=0.9, top_k=20, seed=5)
    chat = Chat(dec, Words(), max_reply=7)
    for i in range(6):
        got, _ = chat.reply("one two three four five six")
        assert 1 <= len(got) <= 7
    assert dec.position() > CAP
    with pytest.raises(ValueError):
        chat.reply("w " * (CAP + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("before,after", [
    (dict(temperature=0.0), dict(temperature=1.5)),
    (dict(temperature=0.9, top_k=1), dict(temperature=1.5)),
    (dict(temperature=0.0), dict(temperature=0.0, repetition=1e30)),
    (dict(temperature=1.5), "firmware"),
    ("firmware", dict(temperature=1.5, repetition=1.2))], ids=str)
def test_a_checkpoint_leaves_the_sampler_as_it_was_set_since(tiny_images, golden, before, after):
    """The random stream is part of the state, the settings are not: after a restore the sampler set since the
    checkpoint draws, and draws what it drew after the checkpoint."""
    name = "tiny-qwen3"
    dec = _decoder(tiny_images[(name, True)], max_new=32)

    def choose(s):
        if s == "firmware":
            dec.set_sampling(1.4, 1.0, 1.3)
        else:
            dec.set_vocab_sampling(**s)

    dec.set_vocab_sampling(temperature=1.0, seed=31)      # the stream
    choose(before)
    dec.reset()
    dec.generate(golden[f"prompt/{name}"], 3)
    dec.checkpoint()
    choose(after)
    a = dec.generate([1], 12)
    dec.restore()
    assert dec.generate([1], 12) == a
    assert len(set(a)) > 4                                # drawn, or penalised: not the greedy repeats
    dec.close()


@pytest.mark.gpu
def test_more_heads_than_the_window_attention_takes():
    """A model past the window attention's 1024 heads is stepped there, as one position a forward."""
    from trixium_amd.model import Decoder
    mc = C.TINY.replace(name="tiny-wide", n_head=1040, n_kv_head=130, n_layer=2, max_ctx=40)
    rng = np.random.default_rng(2)
    feeds = [rng.integers(0, mc.vocab, n).tolist() for n in (30, 25)]
    out = []
    for chunk in (0, 16):
        dec = Decoder.synthetic(mc, seed=3, prefill_chunk=chunk)
        dec.set_kv_ring(1, 4)
        dec.reset()
        out.append([dec.forward(f) for f in feeds])
        dec.close()
    assert max(_rel_err(b, a) for a, b in zip(*out)) <= 2e-3
