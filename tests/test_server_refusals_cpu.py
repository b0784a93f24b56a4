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
