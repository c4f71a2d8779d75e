"""The 8-bit cache and token log probabilities together, as generation, GRPO, serving and evaluation use them."""

import json
import math
import threading

import pytest
import torch

from optimus_dl_b200.core import conf
from optimus_dl_b200.core.config_utils import non_resolving_instantiate
from optimus_dl_b200.core.registry import build
from optimus_dl_b200.models.gpt2 import GPT, GPTConfig
from optimus_dl_b200.models.llama2 import Llama, LlamaConfig
from optimus_dl_b200.models.olmo3 import Olmo3, Olmo3Config
from optimus_dl_b200.ops import decode_fp8 as d8
from optimus_dl_b200.recipe.generation import DecodeSession, generate, generate_stream


def _model(kind="llama", **kw):
    torch.manual_seed(0)
    base = dict(n_layer=2, n_head=4, n_embd=64, vocab_size=97)
    base.update(kw)
    if kind == "gpt2":
        return GPT(GPTConfig(block_size=96, **base))
    if kind == "olmo3":
        return Olmo3(Olmo3Config(n_kv_head=2, head_dim=16, sequence_length=96, intermediate_size=128, sliding_window=8,
                                 layer_types=["sliding_attention", "full_attention"], **base))
    return Llama(LlamaConfig(n_kv_head=2, sequence_length=96, intermediate_size=128, **base))


@pytest.mark.parametrize("kind", ["llama", "gpt2", "olmo3"])
def test_session_attends_over_all_rounded_tokens(kind, monkeypatch):
    """Every decode step is compared with attention over the unrounded keys and values of all tokens so far. A code is
    off by at most half a step, 2^-4 of the value or 2^-10 of its block's scale, whose 448-fold is at most twice the
    block's largest magnitude; raising a scale rounds again, each time relative to a scale twice as large, so all of
    them together stay below twice the last: e(x) <= 2^-3 |x| + 2^-9 s with s <= max|x| / 224. Scores are then off by
    d = scale * sum |q| e(k), probabilities by a factor in [e^-2d, e^2d]."""
    model = _model(kind).eval()
    calls = {}
    real_append, real_attend = d8.append_kv_fp8, d8.decode_attention_fp8
    seen = []

    def append(k, v, cache, lens, n_new=None):
        calls[id(cache)] = [k.clone(), v.clone()]
        real_append(k, v, cache, lens, n_new)

    def attend(q, kn, vn, cache, lens, *, scale=None, window=None):
        kv = calls[id(cache)]
        kv[0], kv[1] = torch.cat([kv[0], kn[:, None]], 1), torch.cat([kv[1], vn[:, None]], 1)
        out = real_attend(q, kn, vn, cache, lens, scale=scale, window=window)
        k, v = kv[0].double(), kv[1].double()
        T, rep = k.shape[1], q.shape[1] // k.shape[2]
        assert lens.tolist() == [T] * q.shape[0]
        first = max(0, T - window) if window else 0
        k, v = (x[:, first:].repeat_interleave(rep, 2) for x in (k, v))
        c = 1 / math.sqrt(q.shape[2])
        err = lambda x: 2.0 ** -3 * x.abs() + 2.0 ** -9 * x.abs().amax(dim=(1, 3), keepdim=True) / 224      # noqa: E731
        s = torch.einsum("bhd,bthd->bht", q.double(), k) * c
        p = torch.softmax(s, -1)
        want = torch.einsum("bht,bthd->bhd", p, v)
        d = (torch.einsum("bhd,bthd->bht", q.double().abs(), err(k)) * c).amax(-1)[..., None]
        tol = (torch.exp(2 * d) - 1) * torch.einsum("bht,bthd->bhd", p, v.abs() + err(v))
        tol = tol + torch.einsum("bht,bthd->bhd", p, err(v)) + 1e-6
        assert bool(((out.double() - want).abs() <= tol).all())
        seen.append(float(((out.double() - want).abs() / want.abs().amax()).max()))
        return out

    monkeypatch.setattr(d8, "append_kv_fp8", append)
    monkeypatch.setattr(d8, "decode_attention_fp8", attend)
    ids = torch.randint(0, 97, (3, 20), generator=torch.Generator().manual_seed(1))
    with DecodeSession(model, 3, 60, kv_cache_dtype="fp8") as sess, DecodeSession(_model(kind).eval(), 3, 60) as full:
        a, b = sess.prefill(ids), full.prefill(ids)
        assert torch.equal(a, b)                        # the prompt itself is attended to unrounded
        for i in range(30):
            a, b = sess.step(ids[:, i % 20]), full.step(ids[:, i % 20])
    assert len(seen) == 60 and 0 < max(seen)            # two layers, and codes do round


def test_kv_cache_dtype_is_checked():
    ids = torch.zeros(1, 4, dtype=torch.long)
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        generate(_model(), ids, 2, kv_cache_dtype="int4")
    with pytest.raises(ValueError, match="logprobs"):
        generate(_model(), ids, 2, logprobs=33)


@pytest.mark.parametrize("use_kv_cache", [True, False])
@pytest.mark.parametrize("k", [0, 4])
def test_generated_logprobs_are_those_of_the_full_forward(use_kv_cache, k):
    model = _model().eval()
    ids = torch.randint(0, 97, (3, 7), generator=torch.Generator().manual_seed(1))
    plain = generate(model, ids, 9, greedy=False, temperature=0.7, top_k=10, seed=3, use_kv_cache=use_kv_cache,
                     generator=torch.Generator().manual_seed(5))
    toks, scored = generate(model, ids, 9, greedy=False, temperature=0.7, top_k=10, seed=3, use_kv_cache=use_kv_cache,
                            generator=torch.Generator().manual_seed(5), logprobs=k)
    assert torch.equal(plain, toks)
    with torch.no_grad():
        full = torch.log_softmax(model(torch.cat([ids, toks], 1))["logits"][:, 6:-1].double(), -1)
    assert torch.allclose(scored.logp.double(), full.gather(-1, toks[..., None])[..., 0], atol=1e-4)
    assert torch.allclose(scored.entropy.double(), -(full.exp() * full).sum(-1), atol=1e-4)
    if k:
        assert scored.top_ids.shape == (3, 9, 4)
        assert torch.allclose(scored.top_logp.double(), full.topk(4, -1).values, atol=1e-4)
    else:
        assert scored.top_ids is None
    none, empty = generate(model, ids, 0, logprobs=k)
    assert none.shape == (3, 0) and empty.logp.shape == (3, 0)


def test_linear_token_loss_with_entropy_cpu():
    from optimus_dl_b200.ops.cross_entropy import linear_token_loss

    torch.manual_seed(0)
    x, w = torch.randn(12, 16, requires_grad=True), torch.randn(40, 16, requires_grad=True)
    tg, coef, ew = torch.randint(0, 40, (12,)), torch.randn(12), torch.randn(12)
    total, nll, ent = linear_token_loss(x, w, tg, lambda n, a, b: (coef[a:b] * n, coef[a:b]), entropy_weight=ew)
    total.backward()
    x2, w2 = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
    lp = torch.log_softmax(x2 @ w2.t(), -1)
    h = -(lp.exp() * lp).sum(-1)
    ref = -(coef * lp.gather(-1, tg[:, None])[:, 0]).sum() + (ew * h).sum()
    ref.backward()
    assert torch.allclose(total, ref, atol=1e-4) and torch.allclose(ent, h, atol=1e-5)
    assert torch.allclose(x.grad, x2.grad, atol=1e-4) and torch.allclose(w.grad, w2.grad, atol=1e-4)
    with pytest.raises(ValueError):
        linear_token_loss(x, w, tg, lambda n, a, b: (n, n), entropy_weight=ew[:5])


def _grpo(tmp_path, use_gpu=False, **grpo):
    head = 64 if use_gpu else 16
    return build("grpo_recipe", non_resolving_instantiate(conf.create({
        "_name": "base",
        "common": {"use_gpu": use_gpu, "output_path": str(tmp_path), "seed": 0,
                   "distributed": {"tp_size": 1, "sharding_world_size": 1}},
        "model": {"_name": "qwen3", "n_layer": 2, "n_head": 4, "n_kv_head": 2, "head_dim": head, "n_embd": 4 * head,
                  "vocab_size": 64, "sequence_length": 48, "intermediate_size": 128, "tie_word_embeddings": True},
        "model_transforms": [{"_name": "fully_shard"}] if use_gpu else [],
        "grpo": {"num_prompts": 4, "prompt_length": 6, "group_size": 4, "max_new_tokens": 20, "micro_batch_size": 8,
                 "rollout_batch_size": 8, **grpo},
        "optimization": {"iterations": 2, "optimizer": {"_name": "adamw", "lr": 1e-3, "weight_decay": 0.0,
                                                        **({} if use_gpu else {"fused": False})}},
    })))


def test_grpo_rolls_out_over_the_8_bit_cache_with_its_own_logprobs(tmp_path):
    recipe = _grpo(tmp_path, kv_cache_dtype="fp8", rollout_logprobs=True, entropy_coef=0.01, eos_token_id=3)
    recipe.run()
    assert len(recipe.history) == 2
    assert all(0 < h["entropy"] <= math.log(64) + 1e-4 and math.isfinite(h["loss"]) for h in recipe.history)


def test_rollout_logprobs_match_teacher_forcing(tmp_path):
    recipe = _grpo(tmp_path)
    model, _ = recipe._build_models(torch.device("cpu"), None)
    prompts = torch.randint(0, 64, (2, 6), generator=torch.Generator().manual_seed(0))
    torch.manual_seed(4)                   # the CPU's sampler draws from the global generator
    seqs, mask, logp = recipe.rollout_scored(model, prompts, 1)
    torch.manual_seed(4)
    assert torch.equal(seqs, recipe.rollout(model, prompts, 1)[0]) and logp.shape == mask.shape == (8, 20)
    assert torch.allclose(logp, recipe.token_logprobs(model, seqs, 6), atol=1e-4)


def test_served_logprobs():
    import http.client

    from optimus_dl_b200.recipe.serve import ServeConfig, ServeRecipe

    recipe = ServeRecipe(conf.merge(conf.create(ServeConfig()), conf.create({
        "serve": {"host": "127.0.0.1", "port": 0},
        "common": {"device": "cpu", "tokenizer": {"_name": "char_tokenize", "add_eos": False}, "kv_cache_dtype": "fp8",
                   "model": {"_name": "llama2", "n_layer": 2, "n_head": 2, "n_embd": 32, "vocab_size": 258,
                             "sequence_length": 64, "intermediate_size": 64}}})))
    recipe.setup()
    httpd = recipe.make_server()
    threading.Thread(target=httpd.serve_forever, daemon=True).start()

    def post(path, payload):
        c = http.client.HTTPConnection("127.0.0.1", httpd.server_address[1], timeout=60)
        c.request("POST", path, body=json.dumps(payload), headers={"Content-Type": "application/json"})
        r = c.getresponse()
        return r.status, json.loads(r.read())

    try:
        ask = {"prompt": "To be", "max_tokens": 8, "temperature": 0.0}
        status, out = post("/v1/completions", {**ask, "logprobs": 3})
        lp = out["choices"][0]["logprobs"]
        n = out["usage"]["completion_tokens"]
        assert status == 200 and len(lp["tokens"]) == len(lp["token_logprobs"]) == len(lp["text_offset"]) == n
        assert lp["text_offset"][0] == 5 and all(x <= 0 for x in lp["token_logprobs"])
        # greedy: the token is the most likely alternative (several tokens may decode to one text)
        assert all(abs(max(t.values()) - x) < 1e-6 for t, x in zip(lp["top_logprobs"], lp["token_logprobs"]))
        status, again = post("/v1/completions", ask)
        assert again["choices"][0]["logprobs"] is None and again["choices"][0]["text"] == out["choices"][0]["text"]
        msgs = [{"role": "user", "content": "hi"}]
        status, out = post("/v1/chat/completions", {"messages": msgs, "max_tokens": 4, "logprobs": True, "top_logprobs": 2})
        content = out["choices"][0]["logprobs"]["content"]
        assert status == 200 and len(content) == out["usage"]["completion_tokens"]
        assert all(len(c["top_logprobs"]) == 2 and c["logprob"] <= 0 for c in content)
        assert post("/v1/chat/completions", {"messages": msgs, "max_tokens": 4})[1]["choices"][0]["logprobs"] is None
        assert post("/v1/completions", {**ask, "logprobs": 21})[0] == 422
        assert post("/v1/completions", {**ask, "logprobs": 2, "stream": True})[0] == 422
    finally:
        httpd.shutdown()
        httpd.server_close()


def test_scoring_refuses_tokens_outside_the_vocabulary():
    from optimus_dl_b200.eval.model import LLMBaselinesModel

    lm = LLMBaselinesModel(_model(), None)
    (a,), (b,) = lm._score([([1, 2, 3], [4, 5])]), lm._score([([1, 2, 3, 4], [5])])
    with torch.no_grad():
        lp = torch.log_softmax(_model().eval()(torch.tensor([[1, 2, 3, 4]]))["logits"].double(), -1)
    assert abs(a[0] - float(lp[0, 2, 4] + lp[0, 3, 5])) < 1e-4 and abs(b[0] - float(lp[0, 3, 5])) < 1e-4
    with pytest.raises(IndexError):
        lm._score([([1, 2], [97])])


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["llama", "gpt2"])
def test_captured_steps_equal_eager_ones(kind):
    dev = torch.device("cuda")
    models = [_model(kind, n_embd=256, vocab_size=512).to(dev, torch.bfloat16).eval() for _ in range(2)]
    ids = torch.randint(0, 512, (3, 40), device=dev)
    with DecodeSession(models[0], 3, 96, kv_cache_dtype="fp8") as a, DecodeSession(models[1], 3, 96, kv_cache_dtype="fp8") as b:
        assert torch.equal(a.prefill(ids), b.prefill(ids))
        for i in range(40):
            assert torch.equal(a.step(ids[:, i]), b.step(ids[:, i], use_graph=False))
        for x, y in zip(a.layers, b.layers):
            assert torch.equal(x.fp8.k.view(torch.uint8), y.fp8.k.view(torch.uint8))
            assert torch.equal(x.fp8.v_scale, y.fp8.v_scale)


@pytest.mark.gpu
def test_sessions_refuse_what_has_no_kernel():
    model = _model(n_embd=64).to("cuda", torch.bfloat16)          # heads of 16
    with pytest.raises(ValueError, match="head dimension"):
        DecodeSession(model, 1, 8, kv_cache_dtype="fp8")


@pytest.mark.gpu
def test_stream_of_scored_tokens_on_the_gpu():
    model = _model(n_embd=256, vocab_size=512).to("cuda", torch.bfloat16).eval()
    ids = torch.randint(0, 512, (2, 30), device="cuda")
    steps = list(generate_stream(model, ids, 12, greedy=True, logprobs=5, kv_cache_dtype="fp8"))
    assert len(steps) == 12
    for tok, r in steps:
        assert torch.equal(r.top_ids[:, 0], tok) and torch.equal(r.top_logp[:, 0], r.logp)
    assert torch.equal(torch.stack([t for t, _ in steps], 1), generate(model, ids, 12, greedy=True, kv_cache_dtype="fp8"))


@pytest.mark.gpu
def test_grpo_on_the_gpu_with_both(tmp_path):
    recipe = _grpo(tmp_path, use_gpu=True, kv_cache_dtype="fp8", rollout_logprobs=True, entropy_coef=0.01)
    recipe.run()
    assert len(recipe.history) == 2
    assert all(0 < h["entropy"] <= math.log(64) + 1e-3 and math.isfinite(h["loss"]) for h in recipe.history)


@pytest.mark.gpu
def test_linear_token_loss_with_entropy_on_the_gpu():
    from optimus_dl_b200.ops.cross_entropy import linear_token_loss

    torch.manual_seed(0)
    T, D, V = 700, 256, 1003
    x = (torch.randn(T, D, device="cuda") * 0.5).bfloat16().requires_grad_(True)
    w = (torch.randn(V, D, device="cuda") * 0.2).bfloat16().requires_grad_(True)
    tg, coef, ew = torch.randint(0, V, (T,), device="cuda"), torch.randn(T, device="cuda"), torch.randn(T, device="cuda")
    total, nll, ent = linear_token_loss(x, w, tg, lambda n, a, b: (coef[a:b] * n, coef[a:b]), chunk_rows=256,
                                        entropy_weight=ew)
    total.backward()
    # the same on logits rounded to bf16, as the chunk holds them
    xd, wd = x.detach().double(), w.detach().double()
    z = (xd @ wd.t()).to(torch.bfloat16).double()
    lp = torch.log_softmax(z, -1)
    p, h = lp.exp(), -(lp.exp() * lp).sum(-1)
    # a product may round to the neighbouring bf16 logit: 2^-8 of the largest, in log p twice
    tol = float(z.abs().max()) * 2.0 ** -7
    assert float((nll.double() + lp.gather(-1, tg[:, None])[:, 0]).abs().max()) <= tol
    assert float((ent.double() - h).abs().max()) <= tol * (1 + float(h.max()))
    dz = coef.double()[:, None] * p - ew.double()[:, None] * p * (lp + h[:, None])
    dz = dz.scatter_add(-1, tg[:, None], -coef.double()[:, None])
    # dz is rounded to bf16 (2^-8) after the logits were (2^-8 of the largest in the exponent), and the products to bf16
    for got, want, size in ((x.grad, dz @ wd, dz.abs() @ wd.abs()), (w.grad, dz.t() @ xd, dz.abs().t() @ xd.abs())):
        slack = (2.0 ** -8 + 2 * tol) * size + 2.0 ** -8 * want.abs()
        assert bool(((got.double() - want).abs() <= slack).all())
