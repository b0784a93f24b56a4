"""What the server answers to requests that cannot be had, and to faults of its own."""

import pytest
from starlette.testclient import TestClient
from test_api_server_cpu import make_engine

from easydel_b200.inference import InvalidRequest, SamplingParams
from easydel_b200.inference.esurge.server import eSurgeApiServer


@pytest.fixture(scope="module")
def engine():
    return make_engine()


@pytest.fixture
def client(engine):
    return TestClient(eSurgeApiServer(engine).app, raise_server_exceptions=False)


CHAT, TEXT = {"messages": [{"role": "user", "content": "hi"}]}, {"prompt": "hello"}


@pytest.mark.parametrize("path,body", [("/v1/chat/completions", CHAT), ("/v1/completions", TEXT), ("/v1/responses", {"input": "hi"})])
@pytest.mark.parametrize("bad", [{"logit_bias": {"4000": 1}}, {"logit_bias": {"x": 1}}, {"min_tokens": 9}, {"top_p": 3.0}])
def test_refused_requests(client, engine, path, body, bad):
    r = client.post(path, json={**body, "max_tokens": 4, **bad})
    assert r.status_code == 400 and r.json()["error"]["type"] == "invalid_request_error"
    assert not engine.scheduler.has_unfinished() and not engine._tracked


@pytest.mark.parametrize("path,body", [("/v1/chat/completions", CHAT), ("/v1/completions", TEXT), ("/v1/responses", {"input": "hi"})])
def test_faults_of_the_server_are_not_the_request_s(client, engine, monkeypatch, path, body):
    def boom(*a, **kw):
        raise ValueError("shapes do not fit")

    monkeypatch.setattr(engine, "generate", boom)
    r = client.post(path, json={**body, "max_tokens": 4})
    assert r.status_code == 500 and "shapes" not in r.text


def test_refusals_keep_their_type():
    assert issubclass(InvalidRequest, ValueError)
    with pytest.raises(InvalidRequest):
        SamplingParams(temperature=-1)


@pytest.mark.parametrize("path,body", [("/v1/chat/completions", CHAT), ("/v1/completions", TEXT), ("/v1/responses", {"input": "hi"})])
@pytest.mark.parametrize("bad", [{"logit_bias": {"4000": 1}}, {"logit_bias": {"-1": 1}}])
def test_refused_streams(client, engine, path, body, bad):
    r = client.post(path, json={**body, "max_tokens": 4, "stream": True, **bad})
    assert r.status_code == 400 and r.json()["error"]["type"] == "invalid_request_error"
    assert not engine.scheduler.has_unfinished() and not engine._tracked
    r = client.post(path, json={**body, "max_tokens": 4, "stream": True})
    assert r.status_code == 200 and r.headers["content-type"].startswith("text/event-stream")


def test_a_stream_ends_its_request_however_it_ends(engine):
    sp = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True)
    whole = engine.generate([5, 6, 7], sp)[0].outputs[0].token_ids
    outs = list(engine.stream([5, 6, 7], sp))
    assert outs[-1].finished and outs[-1].outputs[0].token_ids == whole and not engine._tracked
    with pytest.raises(InvalidRequest):
        engine.stream([], sp)
    for leave in (lambda s: s.close(), lambda s: (next(s), s.close()), lambda s: None, lambda s: next(s)):
        s = engine.stream([5, 6, 7], sp)
        assert engine.scheduler.has_unfinished()
        leave(s)
        del s
        assert not engine.scheduler.has_unfinished() and not engine._tracked
        assert len(engine._free_slots) == engine.runner.max_num_seqs
    s = engine.stream([5, 6, 7], sp)
    s.close()
    s.close()
    assert list(s) == []


def test_two_streams_at_once(engine):
    sp = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True)
    want = [engine.generate(p, sp)[0].outputs[0].token_ids for p in ([5, 6, 7], [9, 10])]
    a, b = engine.stream([5, 6, 7], sp), engine.stream([9, 10], sp)
    got = [list(a)[-1], list(b)[-1]]
    assert [o.outputs[0].token_ids for o in got] == want and not engine._tracked


def test_a_refused_request_of_a_batch_leaves_none_behind(engine):
    ok, bad = SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True), SamplingParams(logit_bias={4000: 1.0})
    for _ in range(2 * engine.runner.max_num_seqs):
        with pytest.raises(InvalidRequest):
            engine.generate([[5, 6], [7, 8], [9, 10]], [ok, ok, bad])
    assert not engine.scheduler.has_unfinished() and not engine._tracked and len(engine._free_slots) == engine.runner.max_num_seqs
    assert len(engine.generate([[5, 6], [7, 8]], ok)) == 2
