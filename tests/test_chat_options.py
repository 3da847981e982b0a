"""The chat command's choices of a sampler and of a prefill chunk, with the decoder replaced by a record of its
calls."""

import pytest

from trixium_amd import chat


class _Decoder:
    made = None

    @classmethod
    def from_image(cls, path, **kw):
        d = cls()
        d.kw, d.calls = kw, []
        cls.made = d
        return d

    def reset(self):
        pass

    def close(self):
        pass

    def set_sampling(self, *a, **kw):
        self.calls.append(("firmware", a, kw))

    def set_vocab_sampling(self, *a, **kw):
        self.calls.append(("vocab", a, kw))


@pytest.fixture
def run(monkeypatch):
    import trixium_amd.model
    import trixium_amd.tokenizer
    monkeypatch.setattr(trixium_amd.model, "Decoder", _Decoder)
    monkeypatch.setattr(trixium_amd.tokenizer.Tokenizer, "from_btok", classmethod(lambda cls, p: None))
    monkeypatch.setattr(chat.Chat, "reply", lambda self, *a, **k: ([], ""))

    def go(*opts):
        chat.main(["-m", "x", "-z", "y", "-p", "hi", *opts])
        return _Decoder.made

    return go


def test_samplers(run):
    assert run().calls == []
    assert run("-S", "0.8,0.9,1.1", "-s", "3").calls == [("firmware", (0.8, 0.9, 1.1), {"seed": 3})]
    assert run("-V", "0.8,40,0.9,0.02").calls == [("vocab", (0.8, 40, 0.9, 0.02, 1.0), {"seed": 0})]
    assert run("-V", "0.8,40,0.9,0.02,1.3", "-s", "9").calls == [("vocab", (0.8, 40, 0.9, 0.02, 1.3), {"seed": 9})]
    assert run("-c", "64").kw["prefill_chunk"] == 64 and run().kw["prefill_chunk"] == 0


@pytest.mark.parametrize("opts", [("-S", "1,1,1", "-V", "1,0,1,0"), ("-V", "1,0,1"), ("-V", "1,0,1,0,1,1")])
def test_refusals(run, opts):
    with pytest.raises(SystemExit):
        run(*opts)
