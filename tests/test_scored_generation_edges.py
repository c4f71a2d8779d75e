"""Scoring and the 8-bit cache as the framework's own paths use them: requests that were answered before they existed,
tokens outside the vocabulary, heads that are scored without their logits."""

import http.client
import json
import threading

import pytest
import torch

from optimus_dl_b200.core import conf


def _server():
    from optimus_dl_b200.recipe.serve import ServeConfig, ServeRecipe

    recipe = ServeRecipe(conf.merge(conf.create(ServeConfig()), conf.create({
        "serve": {"host": "127.0.0.1", "port": 0},
        "common": {"device": "cpu", "tokenizer": {"_name": "char_tokenize", "add_eos": False},
                   "model": {"_name": "llama2", "n_layer": 1, "n_head": 2, "n_embd": 32, "vocab_size": 258,
                             "sequence_length": 64, "intermediate_size": 64}}})))
    recipe.setup()
    httpd = recipe.make_server()
    threading.Thread(target=httpd.serve_forever, daemon=True).start()
    return httpd


def test_chats_with_fields_that_were_ignored_before_are_still_answered():
    httpd = _server()
    msgs = [{"role": "user", "content": "hi"}]

    def post(**fields):
        c = http.client.HTTPConnection("127.0.0.1", httpd.server_address[1], timeout=60)
        c.request("POST", "/v1/chat/completions", body=json.dumps({"messages": msgs, "max_tokens": 3, **fields}),
                  headers={"Content-Type": "application/json"})
        r = c.getresponse()
        return r.status, r.read().decode()

    try:
        for fields in (dict(logprobs=None), dict(logprobs=None, top_logprobs=None), dict(logprobs=False, top_logprobs=3)):
            status, body = post(**fields)
            assert status == 200 and json.loads(body)["choices"][0]["logprobs"] is None
        for fields in (dict(logprobs=None), dict(logprobs=False), dict(logprobs=True), dict(logprobs=True, top_logprobs=2)):
            status, body = post(stream=True, **fields)
            assert status == 200 and body.rstrip().endswith("[DONE]")
    finally:
        httpd.shutdown()
        httpd.server_close()


def _model(**kw):
    from optimus_dl_b200.models.llama2 import Llama, LlamaConfig

    torch.manual_seed(0)
    base = dict(n_layer=2, n_head=4, n_kv_head=2, n_embd=64, vocab_size=97, sequence_length=48, intermediate_size=128)
    return Llama(LlamaConfig(**{**base, **kw}))


@pytest.mark.parametrize("token", [-1, -100, 97, 1 << 40])
def test_scored_tokens_outside_the_vocabulary_are_refused(token):
    from optimus_dl_b200.eval.model import LLMBaselinesModel

    with pytest.raises(IndexError):
        LLMBaselinesModel(_model(), None)._score([([1, 2], [3]), ([1, 2], [5, token])])


def _scores(model, device="cpu"):
    from optimus_dl_b200.eval.model import LLMBaselinesModel

    g = torch.Generator().manual_seed(2)
    ids = lambda n: torch.randint(0, 97, (n,), generator=g).tolist()                             # noqa: E731
    pairs = [(ids(5), ids(3)), (ids(1), ids(40)), (ids(60), ids(2)), (ids(3), []), (ids(2), ids(1)), (ids(30), ids(60))]
    return LLMBaselinesModel(model, None, device=device, batch_size=4)._score(pairs)


def _check_scores(device, dtype, tol, **kw):
    """Scores without all logits, against those of a model whose forward pass forms them."""
    from optimus_dl_b200.models.llama2 import Llama

    class Whole(Llama):
        def head(self, x):
            return super().head(x)

    class Scored(Llama):
        def forward(self, *a, skip_lm_head=False, **kw):
            assert skip_lm_head, "logits of all positions"
            return super().forward(*a, skip_lm_head=True, **kw)

    model = _model(**kw).to(device, dtype)
    got = []
    for cls in (Scored, Whole):
        model.__class__ = cls
        got.append(_scores(model, device))
    for (a, ga), (b, gb) in zip(*got):
        assert abs(a - b) <= tol * (1 + abs(b)) and (ga == gb or dtype != torch.float32)
    assert got[0][3] == (0.0, True)


def test_scoring_forms_the_logits_of_scored_positions_only():
    _check_scores("cpu", torch.float32, 1e-5)


@pytest.mark.gpu
def test_scoring_forms_the_logits_of_scored_positions_only_on_the_gpu():
    """A logit may be rounded to the neighbouring bf16 number, 2^-8 of it; logits here are below 4."""
    _check_scores("cuda", torch.bfloat16, 2.0 ** -6, n_embd=256, n_kv_head=4)
