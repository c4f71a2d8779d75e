"""Token log probabilities, entropy and alternatives: the PyTorch statement on the CPU and the arguments it refuses,
the kernels on the GPU against the definition in 64 bits.

Tolerances.  fp32 statistics: u = (z - m) / T carries one rounding of the difference, one of the product and one of
the constant (3 * 2^-24 relative), the exponential and the logarithm 2^-21 relative or absolute near 1, and the sums
of at most 2^18 terms of one sign are taken in groups of 2^9 and less, so 2^-15 * 2^-24 * 2^9 < 2^-17 relative bounds
them generously: |error of log p| <= 4e-7 |u| + 2e-5, |error of H| <= 2e-5 (1 + H).  Gradients: the same error in the
exponent times a probability, plus half a step of the output type relative to the value.
"""

import math

import pytest
import torch

from optimus_dl_b200.ops import logprobs as lp

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def definition(logits, targets, top_k, temperature, d_logp=None, d_entropy=None):
    """Row by row in 64 bits, straight from the formulas."""
    z = logits.detach().double().cpu()
    t, vocab = targets.cpu(), z.shape[-1]
    out = {"logp": [], "entropy": [], "top_ids": [], "top_logp": [], "grad": [], "p": []}
    for i in range(z.shape[0]):
        live = z[i] > -math.inf
        if not live.any():
            log_p, p, h = torch.full((vocab,), -math.inf, dtype=torch.float64), torch.zeros(vocab).double(), 0.0
        else:
            u = (z[i] - z[i].max()) / temperature
            log_p = u - torch.log(torch.exp(u).sum())
            p = torch.exp(log_p)
            h = -float((p[live] * log_p[live]).sum())
        inside = 0 <= int(t[i]) < vocab
        out["logp"].append(float(log_p[t[i]]) if inside else 0.0)
        out["entropy"].append(h)
        order = sorted(range(vocab), key=lambda j: (-float(z[i, j]), j))[:top_k] if top_k else []
        out["top_ids"].append(order)
        out["top_logp"].append([float(log_p[j]) for j in order])
        if d_logp is not None:
            gl, gh = float(d_logp[i]) * inside * bool(live.any()), float(d_entropy[i])
            g = -gl * p
            g[live] -= gh * p[live] * (log_p[live] + h)
            if inside:
                g[t[i]] += gl
            out["grad"].append(g / temperature)
            out["p"].append(p)
    r = {k: torch.tensor(v, dtype=torch.float64) for k, v in out.items() if k not in ("grad", "p", "top_ids")}
    r["top_ids"] = torch.tensor(out["top_ids"])
    r["grad"], r["p"] = (torch.stack(out["grad"]), torch.stack(out["p"])) if d_logp is not None else (None, None)
    return r


def make(rows, vocab, dtype, seed=0, banned=0.0):
    torch.manual_seed(seed + 1)       # for what a test draws besides
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, vocab, generator=g) * 3).to(dtype)
    if banned:
        z[:, torch.rand(vocab, generator=g) < banned] = -math.inf
    t = torch.randint(0, vocab, (rows,), generator=g)
    return z, t


def compare(r, want, temperature=1.0, logits=None):
    span = 0.0
    if logits is not None:
        f = logits.detach().double().cpu()
        f = f[torch.isfinite(f)]
        span = float(f.max() - f.min()) / temperature if f.numel() else 0.0
    tol = 4e-7 * span + 2e-5
    for name in ("logp", "top_logp"):
        got = getattr(r, name)
        if got is None:
            continue
        got, w = got.detach().double().cpu(), want[name]
        fin = torch.isfinite(w)
        assert torch.equal(got[~fin], w[~fin]), name
        assert not fin.any() or float((got[fin] - w[fin]).abs().max()) <= tol, name
    h = r.entropy.detach().double().cpu()
    assert float(((h - want["entropy"]).abs() / (1 + want["entropy"])).max()) <= 2e-5 + 4e-7 * span
    if r.top_ids is not None:
        assert torch.equal(r.top_ids.cpu(), want["top_ids"])


def check_grad(got, want, dtype, d_logp, d_entropy, temperature):
    """Error in an element: p_j times the exponent's (at most 4e-5 here) times what p_j is multiplied with, and the
    output's rounding (its smallest normal value where that is absolute). At the token's own element g_l outweighs the
    rest: the fp32 sum rounds once, 1 / T once and the product with it once before the output does, 3 * 2^-24."""
    got, w, p = got.detach().double().cpu(), want["grad"], want["p"]
    log_p = torch.where(p > 0, torch.log(p), 0.0).abs()
    times = (d_logp.abs()[:, None] + d_entropy.abs()[:, None] * (log_p + want["entropy"][:, None] + 1)) / temperature
    tol = (1.01 * HALF_STEP[dtype] + 3 * 2.0 ** -24) * w.abs() + 4e-5 * p * times + torch.finfo(dtype).tiny
    assert bool(((got - w).abs() <= tol).all())


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("vocab,top_k,temperature", [(1, 1, 1.0), (7, 0, 1.0), (97, 5, 0.7), (1000, 32, 2.0)])
def test_statement_matches_definition(vocab, top_k, temperature):
    z, t = make(6, vocab, torch.float32, seed=vocab, banned=0.2 if vocab > 50 else 0.0)
    t[1], t[2] = -100, vocab
    z[3] = -math.inf
    z[4] = torch.finfo(torch.float32).min
    z.requires_grad_(True)
    d_logp, d_h = torch.randn(6), torch.randn(6)
    r = lp.token_logprobs(z, t, top_k=top_k, temperature=temperature)
    want = definition(z, t, top_k, temperature, d_logp, d_h)
    finite = z.detach().clone()
    finite[4] = 0
    compare(r, want, temperature, finite)
    torch.autograd.backward([r.logp, r.entropy], [d_logp, d_h])
    check_grad(z.grad, want, torch.float32, d_logp, d_h, temperature)


def test_gradient_against_differences():
    z, t = make(4, 11, torch.float64, seed=3)
    z = z.double().requires_grad_(True)
    t[2] = -100
    w = torch.randn(2, 4).double()

    def f(x):
        r = lp.token_logprobs(x, t, temperature=0.8)
        return (w[0] * r.logp + w[1] * r.entropy).sum()

    assert torch.autograd.gradcheck(f, (z,))


def test_nan_and_infinity():
    z, t = make(3, 9, torch.float32)
    z[0, 4], z[1, 5] = math.nan, math.inf
    r = lp.token_logprobs(z, t, top_k=2)
    assert torch.isnan(r.logp[:2]).all() and torch.isnan(r.entropy[:2]).all() and torch.isfinite(r.logp[2])
    assert int(r.top_ids[0, 0]) == 4 and int(r.top_ids[1, 0]) == 5


def test_statement_orders_doubles_by_all_their_bits():
    z = torch.ones(1, 5, dtype=torch.float64) + torch.tensor([0.0, 2e-12, 1e-12, 2e-12, -1e-12], dtype=torch.float64)
    assert lp.token_logprobs(z, torch.tensor([0]), top_k=5).top_ids.tolist() == [[1, 3, 2, 0, 4]]


def test_refusals():
    z, t = make(3, 9, torch.float32)
    for kw in (dict(top_k=-1), dict(top_k=10), dict(top_k=33), dict(temperature=0.0), dict(temperature=-1.0),
               dict(temperature=math.nan), dict(temperature=math.inf), dict(temperature=1e-7)):
        with pytest.raises(ValueError):
            lp.token_logprobs(z, t, **kw)
    with pytest.raises(ValueError):
        lp.token_logprobs(z, t[:2])
    with pytest.raises(TypeError):
        lp.token_logprobs(z, t.float())
    with pytest.raises(TypeError):
        lp.token_logprobs(z.long(), t)
    with pytest.raises(ValueError):
        lp.token_logprobs(z[:, :0], t)
    with pytest.raises(ValueError):
        lp.linear_token_logprobs(torch.randn(3, 4), torch.randn(9, 4), t, chunk_rows=0)


def test_linear_form_and_shapes():
    x, w = torch.randn(2, 5, 16), torch.randn(33, 16)
    t = torch.randint(0, 33, (2, 5))
    r = lp.linear_token_logprobs(x, w, t, top_k=3, chunk_rows=4)
    full = torch.log_softmax(x @ w.t(), -1)
    assert r.logp.shape == (2, 5) and r.top_ids.shape == (2, 5, 3)
    assert torch.allclose(r.logp, full.gather(-1, t[..., None])[..., 0], atol=1e-5)
    assert torch.allclose(r.top_logp, full.topk(3, -1).values, atol=1e-5)
    empty = lp.linear_token_logprobs(x[:0], w, t[:0], top_k=3)
    assert empty.logp.shape == (0, 5) and empty.top_ids.shape == (0, 5, 3)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_results_may_be_changed_in_place(device):
    """Masking the results in place, as losses do, neither fails nor changes the gradient of the others."""
    z, t = make(6, 301, torch.float32, seed=9)
    z, t = z.to(device), t.to(device)
    grads = []
    for in_place in (True, False):
        x = z.clone().requires_grad_(True)
        r = lp.token_logprobs(x, t, top_k=2)
        keep = torch.tensor([1.0, 0, 1, 1, 0, 1], device=device)
        logp, h = r.logp, r.entropy
        if in_place:
            logp.mul_(keep)
            h[2] = 0.0
            r.top_logp.zero_()
        else:
            logp, h = logp * keep, torch.where(torch.arange(6, device=device) == 2, 0.0, h)
        (logp.sum() + 2 * h.sum()).backward()
        grads.append(x.grad)
    assert torch.equal(*grads)


# ------------------------------------------------------------------------------------------------ GPU
CASES = [(1, 1, 1), (1, 2, 2), (3, 97, 5), (2, 2047, 32), (5, 4097, 20), (2, 8209, 32), (1, 50257, 20), (17, 50257, 1),
         (3, 128256, 20), (2, 200003, 32),
         (600, 97, 5), (601, 2053, 20)]         # rows for narrow CTAs


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top_k", CASES)
def test_kernel_matches_definition(rows, vocab, top_k, dtype):
    z, t = make(rows, vocab, dtype, seed=vocab, banned=0.25 if vocab > 2 else 0.0)
    if rows > 1:
        t[0] = -100
    if rows > 2:
        z[1] = -math.inf
    temperature = 0.8
    d_logp, d_h = torch.randn(rows), torch.randn(rows)
    want = definition(z, t, top_k, temperature, d_logp, d_h)
    zc = z.cuda().requires_grad_(True)
    r = lp.token_logprobs(zc, t.cuda(), top_k=top_k, temperature=temperature)
    compare(r, want, temperature, z)
    g, = torch.autograd.grad([r.logp, r.entropy], [zc], [d_logp.cuda(), d_h.cuda()])
    check_grad(g, want, dtype, d_logp, d_h, temperature)
    again = lp.token_logprobs(zc.detach(), t.cuda(), top_k=top_k, temperature=temperature)
    assert torch.equal(again.logp, r.logp.detach()) and torch.equal(again.top_ids, r.top_ids)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["up", "down", "same", "same_but_last", "lowest", "two_values", "steps"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_alternatives_of_ordered_and_equal_rows(kind, dtype):
    """Rows that list every position as a candidate, and rows of ties."""
    vocab = 70001
    z = {"up": torch.linspace(-4, 4, vocab), "down": torch.linspace(4, -4, vocab), "same": torch.zeros(vocab),
         "same_but_last": torch.zeros(vocab).index_fill_(0, torch.tensor([vocab - 1]), 1.0),
         "lowest": torch.full((vocab,), torch.finfo(dtype).min),
         "two_values": (torch.arange(vocab) % 7 == 3).float(),
         "steps": (torch.arange(vocab) // 64).float() * 0.01}[kind].to(dtype)
    z = z.repeat(700, 1)        # one CTA a row
    t = torch.full((700,), 5)
    want = definition(z[:1], t[:1], 32, 1.0)
    r = lp.token_logprobs(z.cuda(), t.cuda(), top_k=32)
    assert torch.equal(r.top_ids, r.top_ids[:1].expand_as(r.top_ids))
    compare(lp.TokenLogprobs(r.logp[:1], r.entropy[:1], r.top_logp[:1], r.top_ids[:1]), want, 1.0,
            None if kind == "lowest" else z[:1])
    few = lp.token_logprobs(z[:1].cuda(), t[:1].cuda(), top_k=32)       # a cluster a row
    assert torch.equal(few.top_ids.cpu(), want["top_ids"])


@pytest.mark.gpu
def test_kernel_nan_infinity_zero_signs():
    z, t = make(5, 5000, torch.float32)
    z[0, 4321], z[1, 77], z[2, 3] = math.nan, math.inf, -math.nan
    z[3] = 0.0
    z[3, ::2] = -0.0
    z[4, 4999], z[4, 17] = 1e-39, 50.0
    zc = z.cuda().requires_grad_(True)
    r = lp.token_logprobs(zc, t.cuda(), top_k=4)
    assert torch.isnan(r.logp[:3]).all() and torch.isnan(r.entropy[:3]).all() and torch.isfinite(r.logp[3:]).all()
    assert [int(x) for x in r.top_ids[:3, 0]] == [4321, 77, 3]
    assert r.top_ids[3].tolist() == [0, 1, 2, 3]
    g, = torch.autograd.grad(r.logp[3:].sum(), [zc])
    assert torch.isfinite(g[3:]).all()
    g, = torch.autograd.grad(lp.token_logprobs(zc, t.cuda()).entropy.sum(), [zc])
    assert torch.isnan(g[:3]).all() and torch.isfinite(g[3:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("temperature", [1.0, 0.5, 3.0])
def test_extreme_rows(dtype, temperature):
    """Rows of the lowest value, of it among banned tokens, with huge maxima, and far from zero."""
    vocab = 9001
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    z, t = make(8, vocab, dtype, seed=5)
    z[0] = low
    z[0, ::2] = -math.inf                  # half banned, the rest masked: uniform over the rest
    z[1] = low
    z[1, 4000:4010] = 1.0                  # a few live ones
    z[2, 77] = high
    z[3, 5:9] = high                       # four equals share it
    z[4] = (z[4].float() + 300).to(dtype)
    z[5] = (z[5].float() - 2000).to(dtype)
    z[6] = low
    t[:4] = torch.tensor([1, 4003, 77, 8])
    t[6] = 9000
    d_logp, d_h = torch.randn(8), torch.randn(8)
    want = definition(z, t, 4, temperature, d_logp, d_h)
    zc = z.cuda().requires_grad_(True)
    for k in (0, 4):
        r = lp.token_logprobs(zc, t.cuda(), top_k=k, temperature=temperature)
        err = (r.logp.detach().double().cpu() - want["logp"]).abs()
        assert bool((err <= 2e-5 + 4e-7 * (want["logp"].abs() + 20)).all())
        assert (r.entropy.detach().double().cpu() - want["entropy"]).abs().max() <= 1e-3 * (dtype != torch.float32) + 2e-4
    assert torch.equal(r.top_ids.cpu(), want["top_ids"])
    fin = torch.isfinite(want["top_logp"].float()) & (want["top_logp"] > -1e30)
    # an alternative 65504 below the maximum is 2^-24 of that off by its own rounding alone
    err = (r.top_logp.double().cpu() - want["top_logp"]).abs()
    assert bool((err <= 2e-5 + 4e-7 * (want["top_logp"].abs() + 20))[fin].all())
    g, = torch.autograd.grad([r.logp, r.entropy], [zc], [d_logp.cuda(), d_h.cuda()])
    assert torch.isfinite(g).all()
    check_grad(g, want, dtype, d_logp, d_h, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_shapes_and_expanded_gradients(dtype):
    base = torch.randn(6, 3, 1031, device="cuda").to(dtype)
    # the statement rounds its gradient to the type as the kernel does, from fp32 values 1e-5 apart at most
    near = dict(atol=2e-5, rtol=2 * HALF_STEP[dtype])
    t = torch.randint(0, 1000, (6, 3), device="cuda")
    for view in (base[..., 5:1005], base[..., 1:1001], base[::2].repeat_interleave(2, 0)[..., 31:1031],
                 base[:, :1, :1000].expand(6, 3, 1000), base.transpose(0, 1).contiguous().transpose(0, 1)[..., :1000],
                 base[..., :2000:2][..., :500]):
        tg = t % view.shape[-1]
        v = view.detach().clone().requires_grad_(True)
        x = view.detach().requires_grad_(True)
        r, w = lp.token_logprobs(x, tg, top_k=3), lp.token_logprobs_ref(v, tg, top_k=3)
        assert r.logp.shape == (6, 3) and r.top_ids.shape == (6, 3, 3)
        assert torch.equal(r.top_ids, w.top_ids)
        (r.logp.sum() + 0.5 * r.entropy.mean()).backward()
        (w.logp.sum() + 0.5 * w.entropy.mean()).backward()
        assert torch.allclose(r.logp, w.logp, atol=2e-5) and torch.allclose(x.grad, v.grad, **near)
    only = torch.randn(4, 50, device="cuda", requires_grad=True)
    lp.token_logprobs(only, torch.zeros(4, dtype=torch.int32, device="cuda")).entropy.sum().backward()
    assert torch.isfinite(only.grad).all()
    assert lp.token_logprobs(base[:0, 0], t[:0, 0], top_k=2).top_ids.shape == (0, 2)


@pytest.mark.gpu
def test_captured_and_replayed_on_another_stream():
    z = torch.randn(40, 50257, device="cuda").bfloat16()
    t = torch.randint(0, 50257, (40,), device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        lp.token_logprobs(z, t, top_k=5)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = lp.token_logprobs(z, t, top_k=5)
    for seed in range(3):
        z.copy_(torch.randn(40, 50257, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)))
        graph.replay()
        w = lp.token_logprobs_ref(z, t, top_k=5)
        assert torch.equal(r.top_ids, w.top_ids) and torch.allclose(r.logp, w.logp, atol=2e-5)


@pytest.mark.gpu
def test_rows_past_32_bits():
    """2^31 logits and more: the last rows are the ones whose offsets would wrap."""
    vocab, rows = 128256, 16800
    z = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    z[-3:] = torch.randn(3, vocab, device="cuda", generator=g).bfloat16()
    t = torch.arange(rows, device="cuda") % vocab
    r = lp.token_logprobs(z, t, top_k=3)
    w = lp.token_logprobs_ref(z[-3:], t[-3:], top_k=3)
    assert torch.equal(r.top_ids[-3:], w.top_ids) and torch.allclose(r.logp[-3:], w.logp, atol=2e-5)
    assert torch.allclose(r.entropy[:-3], torch.full((), math.log(vocab), device="cuda"), atol=1e-4)


@pytest.mark.gpu
def test_linear_form_on_the_gpu():
    x = torch.randn(300, 64, device="cuda").bfloat16()
    w = torch.randn(1003, 64, device="cuda").bfloat16()
    t = torch.randint(0, 1003, (300,), device="cuda")
    r = lp.linear_token_logprobs(x, w, t, top_k=4, chunk_rows=128)
    # logits are rounded to bf16: 2^-8 of the largest
    z = x.float() @ w.float().t()
    full = torch.log_softmax(z, -1)
    tol = float(z.abs().max()) * 2.0 ** -8 * 2
    assert (r.logp - full.gather(-1, t[:, None])[:, 0]).abs().max() <= tol
    assert (r.top_logp - full.topk(4, -1).values).abs().max() <= tol
