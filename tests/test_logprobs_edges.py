"""Token log probabilities at their edges: where tensors lie, magnitudes of logits, the ends of rows, ties, and the forms
over a head projection.

Tolerances, with u = (z - max z) / T in 64 bits and S = sum e^u. An exponent carries one rounding of c = log2 e / T, one of
the difference and one of the product in fp32, and the logarithm of one element the same again: 6 * 2^-24 |u| < 4e-7 |u|.
A reference's residue (at most 2^-4) cancels but for its own rounding. 2^x and log2 x are off by 2^-22 relative and
2^-21 absolute; a thread's sum of n terms of one sign by (n / 2) 2^-24 at most (it is two sums), n <= 2^9 for the rows
here, and joining 2^8 of them by 2^4 steps: together below 5e-5 of S and of sum u e^u. So
    |error of log p_j| <= 4e-7 |u_j| + 5e-5        |error of H| <= 5e-5 (1 + H) + 4e-7 (H + 1)
as sum p |u| <= H. An element of the gradient, -p_j (g_l + g_H (log p_j + H)) / T with g_l / T more at the token, is off by
p_j times the errors of log p_j and H times what p_j is multiplied with, and by half a step of its type. Exponentials below
2^-126 are flushed to 0, so p_j itself may be off by that much.
"""

import math

import pytest
import torch

from optimus_dl_b200.ops import logprobs as lp
from optimus_dl_b200.ops.cross_entropy import linear_token_loss

LARGEST = torch.finfo(torch.float32).max        # of a log probability; beyond, it is -inf
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def definition(z, t, temperature, d_logp, d_h):
    z, d_logp, d_h = z.detach().double().cpu(), d_logp.double().cpu()[:, None], d_h.double().cpu()[:, None]
    t = t.cpu()[:, None]
    top = z.amax(-1, keepdim=True)
    none = top == -math.inf
    u = (z - torch.where(none, 0.0, top)) / temperature
    log_s = torch.log(torch.where(none, 1.0, torch.exp(u).sum(-1, keepdim=True)))
    log_p = u - log_s
    p = torch.exp(log_p)
    h = -torch.where(p == 0, 0.0, p * log_p).sum(-1, keepdim=True)
    inside = (t >= 0) & (t < z.shape[-1])
    at = t.clamp(0, z.shape[-1] - 1)
    logp = torch.where(inside, log_p.gather(-1, at), 0.0)
    a = torch.where(inside & ~none, d_logp, 0.0)
    times = a.abs() + d_h.abs() * (torch.where(p == 0, 0.0, log_p).abs() + h + 1)
    g = -p * a - d_h * torch.where(p == 0, 0.0, p * (log_p + h))
    g = g.scatter_add(-1, at, a)
    off = 4e-7 * torch.where(u == -math.inf, 0.0, u).abs() + 5e-5
    # 2^x is 0 below 2^-126: such a p_j is off by all of itself
    slack = (p * (off + 6e-5 * (1 + h)) + torch.finfo(torch.float32).tiny) * times / temperature
    return dict(logp=logp[:, 0], h=h[:, 0], grad=g / temperature, slack=slack, u=torch.where(inside, u.gather(-1, at), 0.0)[:, 0],
                log_p=log_p)


def check(z, t, temperature, d_logp=None, d_h=None, top_k=0):
    """The kernels' results on the GPU against the definition; returns them."""
    rows = z.shape[0]
    g = torch.Generator().manual_seed(rows)
    d_logp = torch.randn(rows, generator=g) if d_logp is None else d_logp
    d_h = torch.randn(rows, generator=g) if d_h is None else d_h
    want = definition(z, t, temperature, d_logp, d_h)
    x = z.cuda().requires_grad_(True)
    r = lp.token_logprobs(x, t.cuda(), top_k=top_k, temperature=temperature)
    logp, h = r.logp.detach().double().cpu(), r.entropy.detach().double().cpu()
    fin = want["logp"].abs() <= LARGEST
    assert bool((logp[~fin] == -math.inf).all())
    err = ((logp - want["logp"]).abs() / (4e-7 * want["u"].abs() + 5e-5))[fin]
    assert not err.numel() or float(err.max()) <= 1, (err.argmax(), err.max())
    err = (h - want["h"]).abs() / (5.1e-5 * (1 + want["h"]))
    assert float(err.max()) <= 1, (err.argmax(), err.max())
    grad, = torch.autograd.grad([r.logp, r.entropy], [x], [d_logp.cuda(), d_h.cuda()])
    tol = want["slack"] + (1.01 * HALF_STEP[z.dtype] + 3 * 2.0 ** -24) * want["grad"].abs() + torch.finfo(z.dtype).tiny
    fits = want["grad"].abs() <= torch.finfo(z.dtype).max
    assert not torch.isnan(grad).any()
    err = ((grad.double().cpu() - want["grad"]).abs() / tol)[fits]
    assert bool((err <= 1).all()), (err.argmax(), err.max())
    if top_k:
        order = torch.sort(z.double(), dim=-1, descending=True, stable=True).indices[:, :top_k]
        assert torch.equal(r.top_ids.cpu(), order)
    return r, grad


# ------------------------------------------------------------------------------------------------ where tensors lie
def test_the_entropy_weight_has_to_be_where_the_rows_are():
    x, w = torch.randn(6, 16), torch.randn(9, 16)
    t, ew = torch.randint(0, 9, (6,)), torch.randn(6)
    zero = lambda n, a, b: (torch.zeros_like(n), torch.zeros_like(n))                          # noqa: E731
    linear_token_loss(x, w, t, zero, entropy_weight=ew)
    for bad in (dict(entropy_weight=ew.to("meta")), dict(entropy_weight=ew, t=t.to("meta")),
                dict(entropy_weight=ew, w=w.to("meta")), dict(entropy_weight=ew[:4], t=t[:4])):
        with pytest.raises(ValueError):
            linear_token_loss(x, bad.get("w", w), bad.get("t", t), zero, entropy_weight=bad["entropy_weight"])


def test_the_head_has_to_fit_the_rows_and_be_where_they_are():
    x, w, t = torch.randn(6, 16), torch.randn(9, 16), torch.randint(0, 9, (6,))
    for bad in (w.to("meta"), w[:, :8], w[0], w[None]):
        with pytest.raises(ValueError):
            lp.linear_token_logprobs(x, bad, t)


def test_the_head_projection_runs_on_the_rows_own_device(monkeypatch):
    """Of the two launches the product alone would go to the current device. Tensors without memory stand for those of a
    second GPU."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    entered, inside = [], []

    class On:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            entered.append(self.device)

        def __exit__(self, *exc):
            entered.pop()

    def product(a, b, out):
        inside.append(list(entered))

    def scores(z, t, **kw):
        n = z.new_empty(t.shape, dtype=torch.float32)
        return lp.TokenLogprobs(n, n, None, None)

    monkeypatch.setattr(lp._lib, "on_device", On)
    monkeypatch.setattr(lp.gemm, "gemm", product)
    monkeypatch.setattr(lp, "token_logprobs", scores)
    with FakeTensorMode():
        there = torch.device("cuda", 1)
        x, w = (torch.empty(n, 16, dtype=torch.bfloat16, device=there) for n in (6, 9))
        r = lp.linear_token_logprobs(x, w, torch.zeros(6, dtype=torch.int64, device=there), chunk_rows=4)
    assert r.logp.shape == (6,) and inside == [[there], [there]]


# ------------------------------------------------------------------------------------------------ the statement
def by_sorting(z, k):
    return torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]


@pytest.mark.parametrize("k", [1, 2, 5, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_the_statements_alternatives_are_those_of_a_stable_sort(dtype, k):
    g = torch.Generator().manual_seed(k)
    z = torch.randn(14, 3001, generator=g).to(dtype)
    z[1] = 0.0
    z[2] = (torch.arange(3001) % 5 == 0).to(dtype)
    z[3, 2000:] = 9.0
    z[4] = -math.inf
    z[5, ::3] = -math.inf
    z[6, 5:] = -math.inf
    z[7, 2999], z[8, ::100] = math.nan, math.nan
    z[9, 10], z[9, 20], z[9, 30] = math.inf, math.nan, math.inf
    z[10] = math.nan
    z[11, ::2] = -0.0
    z[11, 1::2] = 0.0
    z[12] = torch.finfo(dtype).min
    r = lp.token_logprobs_ref(z, torch.zeros(14, dtype=torch.int64), top_k=k)
    assert torch.equal(r.top_ids, by_sorting(z if dtype == torch.float64 else z.float(), k))
    rows = [0, 1, 2, 3, 11]
    want = torch.log_softmax(z[rows].double(), -1).gather(-1, r.top_ids[rows])
    assert torch.allclose(r.top_logp[rows].double(), want, atol=1e-5)


def test_the_statement_does_not_sort_rows_and_holds_no_copies_of_them(monkeypatch):
    """What scoring on the CPU costs: parts of a batch at a time, and sorts of what is listed only."""
    sizes, real = [], torch.sort
    monkeypatch.setattr(torch, "sort", lambda t, *a, **kw: (sizes.append(t.shape[-1]), real(t, *a, **kw))[1])
    monkeypatch.setattr(lp._TokenLogprobsRef, "CHUNK", 4000)
    z = torch.randn(3, 7, 1501)
    t = torch.randint(0, 1501, (3, 7))
    for k in (1, 4):
        r = lp.token_logprobs(z, t, top_k=k, temperature=0.7)
        want = torch.log_softmax(z.double() / 0.7, -1)
        assert torch.allclose(r.logp.double(), want.gather(-1, t[..., None])[..., 0], atol=1e-5)
        assert torch.allclose(r.entropy.double(), -(want.exp() * want).sum(-1), atol=1e-5)
        assert torch.equal(r.top_ids, z.topk(k, -1).indices)
    assert not sizes or max(sizes) <= 4


def test_the_statements_gradient_over_several_parts(monkeypatch):
    monkeypatch.setattr(lp._TokenLogprobsRef, "CHUNK", 30)
    z = torch.randn(2, 5, 11, dtype=torch.float64, requires_grad=True)
    t = torch.randint(0, 11, (2, 5))
    t[0, 1] = -100

    def f(x):
        r = lp.token_logprobs(x, t, temperature=0.8)
        return (r.logp * torch.arange(10.0).view(2, 5)).sum() + (r.entropy ** 2).sum()

    assert torch.autograd.gradcheck(f, (z,))
    r = lp.token_logprobs(z, t)
    with torch.no_grad():
        z.mul_(2)                  # the gradient is of what was scored
    g, = torch.autograd.grad(r.logp.sum(), z)
    p = torch.softmax(z.detach() / 2, -1)
    inside = (t >= 0)[..., None]
    want = inside * (torch.nn.functional.one_hot(t.clamp(min=0), 11) - p)
    assert torch.allclose(g, want)


# ------------------------------------------------------------------------------------------------ ends of rows, GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size,temperature", [(30.0, 1e-6), (7e5, 1.0), (60000.0, 0.1), (50.0, 7e-5)])
def test_a_maximum_at_either_end_of_a_row(dtype, size, temperature):
    """Alone with the distribution: its entropy is 0 wherever it stands, to what the logarithm and the reference's own
    rounding leave, 2^-20 of the exponent's residue (at most 2) and of 1."""
    if size > torch.finfo(dtype).max:
        pytest.skip("not a number of this type")
    for vocab in (1025, 1027, 4099, 20003):
        z = torch.zeros(24, vocab)
        for i in range(24):
            z[i, [0, 1, 2, 3, 6, 7, vocab // 2, vocab - 8, vocab - 7, vocab - 3, vocab - 2, vocab - 1][i % 12]] = size + i
        r = lp.token_logprobs(z.to(dtype).cuda(), z.argmax(-1).cuda(), temperature=temperature)
        assert float(r.entropy.abs().max()) <= 5e-5 and float(r.logp.abs().max()) <= 5e-5


# ------------------------------------------------------------------------------------------------ magnitudes, GPU
def masked_rows(dtype, vocab, temperature, fills):
    """Ordinary logits with a fill in the whole row, in a stretch of it, in the first or the last token, in every other
    token, beside its neighbour; and rows whose m c lies about the places where exponents are taken differently."""
    g = torch.Generator().manual_seed(vocab)
    rows = []
    for fill in fills:
        fill = torch.tensor(fill, dtype=torch.float64).to(dtype)
        if not torch.isfinite(fill):
            continue
        base = (torch.randn(6, vocab, generator=g) * 3).to(dtype)
        base[0] = fill
        base[1, vocab // 5:vocab // 5 + 16384] = fill
        base[2, 0] = fill
        base[3, -1] = fill
        base[4, ::2] = fill
        base[5] = fill
        base[5, 1::3] = torch.nextafter(fill.float(), torch.tensor(math.inf)).to(dtype) if dtype != torch.bfloat16 else \
            (fill.view(torch.int16) + 1).view(dtype)
        rows.append(base)
    for far in (2.0 ** 20, 2.0 ** 24, 2.0 ** 30, 2.0 ** 32):
        for sign in (1, -1):
            at = sign * far * temperature * math.log(2)
            if abs(at) < torch.finfo(dtype).max:
                rows.append((torch.randn(2, vocab, generator=g) * 3 * max(1.0, abs(at) * 2.0 ** -22) + at).to(dtype))
    return torch.cat(rows)


FILLS = [s * f for f in (1e5, 1e9, 3e9, 1e10, 1e12, 1e20, 1e25, 3e38) for s in (-1, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1.0, 0.5, 0.1, 1e-3, 1e-6, 1e6])
@pytest.mark.parametrize("vocab", [1025, 33001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_logits_of_any_finite_magnitude(dtype, vocab, temperature):
    fills = [s * f for f in (1000.0, 30000.0, 65504.0) for s in (-1, 1)] if dtype == torch.float16 else FILLS
    z = masked_rows(dtype, vocab, temperature, fills)
    t = torch.randint(0, vocab, (z.shape[0],), generator=torch.Generator().manual_seed(1))
    t[::7] = vocab - 1
    r, _ = check(z, t, temperature, top_k=3)
    few = lp.token_logprobs(z[:2].cuda(), t[:2].cuda(), temperature=temperature)             # a cluster a row
    many = lp.token_logprobs(z.repeat(12, 1).cuda(), t.repeat(12).cuda(), temperature=temperature)     # narrow CTAs
    for part in (few, lp.TokenLogprobs(many.logp[-z.shape[0]:], many.entropy[-z.shape[0]:], None, None)):
        n = part.logp.shape[0]
        want = definition(z[:n], t[:n], temperature, torch.zeros(n), torch.zeros(n))
        fin = want["logp"].abs() <= LARGEST
        assert bool(((part.logp.double().cpu() - want["logp"]).abs() <= 4e-7 * want["u"].abs() + 5e-5)[fin].all())
        assert bool(((part.entropy.double().cpu() - want["h"]).abs() <= 5.1e-5 * (1 + want["h"])).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_of_the_lowest_value_keep_their_log_probability(dtype):
    """It is that value itself here, less 0.7 to 6.2: within a rounding of each of two terms."""
    low = torch.finfo(dtype).min
    z = torch.full((3, 501), low, dtype=dtype)
    z[:, :2], z[1, 2:] = 0.0, 0.0
    z[1, 500] = low
    r = lp.token_logprobs(z.cuda(), torch.tensor([500, 500, 2]).cuda(), top_k=4)
    assert bool(((r.logp.double().cpu() - low).abs() <= 2.0 ** -23 * abs(low)).all())
    for got, want in ((r.top_logp[0, 2:], low), (r.top_logp[2, 3:], low), (r.top_logp[1], -math.log(500))):
        assert bool(((got.double().cpu() - want).abs() <= 2.0 ** -23 * abs(want) + 5e-5).all())


@pytest.mark.gpu
@pytest.mark.parametrize("temperature,g_h", [(1.0, 1e9), (1e-2, 1e5), (1e-4, 1e5), (1e-6, 1.0), (1e-6, 1e5), (1e6, 1e9)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients_of_banned_tokens_under_large_weights(dtype, temperature, g_h):
    """0 at a banned token, whatever the entropy's weight (a loss scale) and the temperature."""
    g = torch.Generator().manual_seed(3)
    z = (torch.randn(8, 4099, generator=g) * 3).to(dtype)
    z[:, torch.rand(4099, generator=g) < 0.3] = -math.inf
    z[1] = -math.inf
    z[2, :4000] = torch.finfo(dtype).min
    z[3, :2000] = -30000.0
    t = torch.randint(0, 4099, (8,), generator=g)
    d_logp, d_h = torch.randn(8, generator=g), torch.randn(8, generator=g) * g_h
    _, grad = check(z, t, temperature, d_logp, d_h)
    banned = (z == -math.inf) & (torch.arange(4099) != t[:, None])
    assert not grad.cpu()[banned].any()


# ------------------------------------------------------------------------------------------------ calls at once, replays
@pytest.mark.gpu
def test_two_threads_on_streams_of_their_own():
    import threading

    def work(seed, dtype):
        g = torch.Generator().manual_seed(seed)
        z = (torch.randn(70, 20011, generator=g) * 3).to(dtype).cuda().requires_grad_(True)
        t = torch.randint(0, 20011, (70,), generator=g).cuda()
        r = lp.token_logprobs(z, t, top_k=7)
        grad, = torch.autograd.grad(r.logp.sum() + 0.1 * r.entropy.sum(), z)
        return r.logp.detach(), r.entropy.detach(), r.top_ids, grad

    jobs = [(1, torch.bfloat16), (2, torch.float32)]
    want = [work(*j) for j in jobs]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i] = work(*jobs[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


@pytest.mark.gpu
def test_forward_and_gradient_captured_and_replayed_with_other_logits():
    rows, vocab = 33, 5003
    z = torch.empty(rows, vocab, device="cuda", dtype=torch.bfloat16)
    t = torch.randint(0, vocab, (rows,), device="cuda")
    ones = torch.ones(rows, device="cuda")

    def step(logits):
        x = logits.detach().requires_grad_(True)
        r = lp.token_logprobs(x, t)
        return r.logp.detach(), r.entropy.detach(), torch.autograd.grad([r.logp, r.entropy], [x], [ones, -ones])[0]

    z.normal_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(z)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(z)
    for scale in (1.0, 30.0, 1e10):
        z.normal_().mul_(scale)
        t.random_(0, vocab)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step(z)))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,chunk", [(1, 50257, 4096), (5, 1003, 2), (65, 33001, 64), (129, 4096, 4096)])
def test_few_and_many_rows_over_a_head(rows, vocab, chunk):
    """Logits are bf16 products; a product of 128 terms in fp32 may round to the neighbouring one."""
    torch.manual_seed(rows)
    x, w = torch.randn(rows, 128, device="cuda").bfloat16(), (torch.randn(vocab, 128, device="cuda") * 0.1).bfloat16()
    t = torch.randint(0, vocab, (rows,), device="cuda")
    r = lp.linear_token_logprobs(x, w, t, top_k=3, chunk_rows=chunk)
    z = x.double() @ w.double().t()
    want = torch.log_softmax(z, -1)
    tol = 2 * 2.0 ** -8 * float(z.abs().max()) + 1e-4
    assert float((r.logp.double() - want.gather(-1, t[:, None])[:, 0]).abs().max()) <= tol
    assert float((r.top_logp.double() - want.topk(3).values).abs().max()) <= tol
