"""Model.score and the server's /score on the CPU."""

import json

import pytest
import torch

from moe_engine import serve
from moe_engine.model import Model, ModelConfig
from test_serve import start

SMALL = dict(max_seq_length=32, vocab_size=300, num_layers=2, hidden_dim=32, num_heads=4, num_experts=4, top_k=2)


@pytest.fixture(scope="module")
def model():
    torch.manual_seed(0)
    return Model(ModelConfig(**SMALL)).eval()


def test_score_is_the_log_softmax_of_the_forward_pass(model):
    ids = torch.randint(0, 300, (20,))
    with torch.no_grad():
        logp = model(ids[None], model.new_cache())[0].double().log_softmax(-1)
    r = model.score(ids, top=4)
    assert torch.allclose(r.logprobs.double(), logp[:-1].gather(1, ids[1:, None])[:, 0], atol=1e-5)
    assert torch.allclose(r.entropy.double(), -(logp.exp() * logp).sum(-1)[:-1], atol=1e-5)
    assert torch.allclose(r.top_logprobs.double(), logp[:-1].topk(4).values, atol=1e-5)
    assert torch.equal(r.top_tokens, logp[:-1].topk(4).indices)
    cache = model.new_block_allocator(num_blocks=2, block_size=16).new_cache()
    paged = model.score(ids[None], cache=cache)
    assert torch.allclose(paged.logprobs, r.logprobs, atol=1e-5) and paged.top_tokens.shape == (19, 0)
    assert cache.position == 20


def test_one_token_has_nothing_to_score(model):
    r = model.score(torch.tensor([5]), top=2)
    assert r.logprobs.shape == (0,) and r.top_tokens.shape == (0, 2)


def test_score_refuses(model):
    ids = torch.zeros(3, dtype=torch.long)
    used = model.new_cache()
    model(ids[None], used)
    for args, kw, message in (((torch.zeros(2, 3),), {}, "batch size 1"), ((ids[:0],), {}, "at least one token"),
                              ((torch.zeros(33),), {}, "max_seq_length"), ((ids,), dict(top=-1), "top"),
                              ((ids,), dict(top=65), "top"), ((ids,), dict(cache=used), "fresh cache")):
        with pytest.raises(ValueError, match=message):
            model.score(*args, **kw)


def test_the_server_scores_and_returns_its_blocks(monkeypatch):
    for flags in ((), ("--cache", "paged")):
        client, ledger = start(monkeypatch, *flags)
        ids = [7, 300, 42, 9]
        body = client.post("/score", json={"prompt_ids": ids, "top": 3}).json()
        want = serve.model.score(torch.tensor(ids), top=3)
        assert body["token_ids"] == ids and body["logprobs"][0] is None and body["top"][0] == []
        assert body["logprobs"][1:] == pytest.approx(want.logprobs.tolist(), abs=1e-5)
        assert body["entropy"][1:] == pytest.approx(want.entropy.tolist(), abs=1e-5)
        assert [[t["token_id"] for t in row] for row in body["top"][1:]] == want.top_tokens.tolist()
        assert client.post("/score", json={"prompt": "hello"}).status_code == 200
        assert client.post("/score", json={"prompt_ids": [10**6]}).status_code == 400
        assert client.post("/score", json={"prompt_ids": [1] * 60}).status_code == 400
        assert client.post("/score", json={}).status_code == 422
        assert client.post("/score", json={"prompt_ids": [1], "top": 21}).status_code == 422
        assert ledger.balanced() and len(ledger.opened) == 2
        if flags:
            assert sorted(serve.allocator.free_blocks) == list(range(serve.allocator.num_blocks))


def test_values_json_cannot_hold_are_null(monkeypatch):
    client, _ = start(monkeypatch)
    bias = serve.model.output_projection.bias
    with torch.no_grad():
        bias[5] = float("-inf")
    body = json.loads(client.post("/score", json={"prompt_ids": [1, 5, 2]}).content)
    assert body["logprobs"][1] is None and body["logprobs"][2] is not None
