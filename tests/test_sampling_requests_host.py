"""How top_p, top_k and min_p reach the engine: request fields, sessions, the chat loop.  No GPU."""

import io
import json
import threading
import urllib.error
import urllib.request

import pytest
import torch

from megakernels_b200 import sampling, server
from megakernels_b200.chat import repl
from megakernels_b200.session import ChatSession


class Engine:
    """A `Megakernel` as a session sees it: replies with the bytes of 'ok' and the stop id, and notes what was asked of it."""

    mtp, mtp_h, device = None, None, "cpu"

    def __init__(self):
        self.asked = []

    def reset(self):
        pass

    def snapshot(self):
        return None

    def restore(self, snap):
        pass

    def prefill(self, tokens):
        return tokens[-1]

    def generate(self, prompt, **kw):
        self.asked.append(kw)
        yield from (111, 107, 256)


class Tokenizer:
    def encode(self, text):
        return list(text.encode())

    def decode(self, ids):
        return bytes(i for i in ids if i < 256).decode(errors="replace")


@pytest.fixture
def session(monkeypatch):
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    return ChatSession(Engine(), Tokenizer(), [256], [])


def test_filters_of_a_request():
    f = server.filters_of
    assert f({}) == {} and f({"top_p": 1, "top_k": 0, "min_p": 0}) == {} and f({"top_p": None, "top_k": -1}) == {}
    assert f({"top_p": 0.9, "top_k": "20", "min_p": 0.05}) == {"top_p": 0.9, "top_k": 20, "min_p": 0.05}
    for bad in ({"top_p": 0}, {"top_p": 1.5}, {"top_p": "x"}, {"top_k": -2}, {"min_p": 2}, {"min_p": float("nan")}):
        with pytest.raises(ValueError):
            f(bad)


def test_they_reach_the_engine_and_only_when_asked_for(session):
    ask = {"messages": [{"role": "user", "content": "hi"}], "temperature": 0.5, "seed": 3}
    assert server.complete(session, ask)["choices"][0]["message"]["content"] == "ok"
    assert server.complete(session, dict(ask, top_p=0.9, top_k=5))["choices"][0]["finish_reason"] == "stop"
    assert list(server.stream_chunks(session, dict(ask, min_p=0.1)))[-1]["choices"][0]["finish_reason"] == "stop"
    kw = [{k: v for k, v in a.items() if k in ("top_p", "top_k", "min_p")} for a in session.mk.asked]
    assert kw == [{}, {"top_p": 0.9, "top_k": 5}, {"min_p": 0.1}] and all(a["temperature"] == 0.5 and a["seed"] == 3 for a in session.mk.asked)


def test_a_request_that_means_nothing_is_refused(session):
    httpd = server.serve(session, port=0)
    threading.Thread(target=httpd.serve_forever, daemon=True).start()
    try:
        url = f"http://127.0.0.1:{httpd.server_address[1]}/v1/chat/completions"
        post = lambda body: urllib.request.urlopen(urllib.request.Request(url, json.dumps(body).encode()), timeout=20)     # noqa: E731
        msg = [{"role": "user", "content": "hi"}]
        for bad in (dict(top_p=2), dict(top_k=[1]), dict(min_p="no"), dict(top_p=0, stream=True)):
            with pytest.raises(urllib.error.HTTPError) as e:
                post(dict(messages=msg, **bad))
            assert e.value.code == 400
        assert not session.mk.asked
        assert json.loads(post(dict(messages=msg, top_p=0.5)).read())["choices"][0]["message"]["content"] == "ok"
    finally:
        httpd.shutdown()


def test_a_request_with_numbers_beyond_all_bounds_is_refused(session):
    """JSON as Python reads it has Infinity and NaN."""
    httpd = server.serve(session, port=0)
    threading.Thread(target=httpd.serve_forever, daemon=True).start()
    try:
        url = f"http://127.0.0.1:{httpd.server_address[1]}/v1/chat/completions"
        for bad in ('"top_k": Infinity', '"top_p": NaN', '"min_p": -Infinity', '"top_k": 1e400'):
            body = '{"messages": [{"role": "user", "content": "hi"}], %s}' % bad
            with pytest.raises(urllib.error.HTTPError) as e:
                urllib.request.urlopen(urllib.request.Request(url, body.encode()), timeout=20)
            assert e.value.code == 400
        assert not session.mk.asked
    finally:
        httpd.shutdown()


def test_the_chat_loop_passes_them_on(session):
    lines = iter(["hello", "/quit"])
    repl(session, inp=lambda _: next(lines), out=io.StringIO(), top_k=7, top_p=0.8, min_p=0.0)
    assert session.mk.asked[0]["top_k"] == 7 and session.mk.asked[0]["top_p"] == 0.8


def test_sampled_continuations_feed_their_own_choices(monkeypatch):
    """`continue_from` with a choice that needs no GPU: the arg-max."""
    monkeypatch.setattr(sampling, "sample", lambda logits, u, *s: sampling.Sample(logits.argmax(-1).int(), None, None))
    fed = []

    def step(tok):
        fed.append(tok.tolist())
        return torch.nn.functional.one_hot((tok.long() * 3 + 1) % 50, 50).float()

    out = sampling.continue_from(step, torch.tensor([2, 7]), 4, temperature=0.5, top_k=3, top_p=0.9, seed=1)
    assert out.tolist() == [[7, 22], [22, 17], [17, 2], [2, 7]] and fed == [[2, 7], [7, 22], [22, 17], [17, 2]]
    with pytest.raises(ValueError):
        sampling.continue_from(step, torch.tensor([1]), 1, top_p=0.0)
