"""Cases and plain forms of the operators behind sampling and scoring.

``logprobs``       ``ops.logprobs.token_logprobs``: log probabilities of given tokens, the entropy of each row's
                   distribution and its most likely alternatives, from a matrix of logits; with ``grad`` also the
                   gradient with respect to the logits.
``append``         ``ops.decode_fp8.append_kv_fp8``: new keys and values into a cache held in e4m3 with one
                   power-of-two scale for each block of tokens and head.
``attend``         ``ops.decode_fp8.decode_attention_fp8``: one query token per sequence; appends its key and value
                   to that cache and attends over it.

``run`` computes the plain forms (elementary torch operations in 32 bits) while ``own`` is false and calls the
framework where it is true; ``exact`` states the same definitions in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0
SCALE_EXP_MIN, SCALE_EXP_MAX = -112, 119     # exponents a block's scale is clamped to


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one served token: its log probability and the five alternatives that an answer lists beside it
        dict(name="answer-1x128256", op="logprobs", rows=1, vocab=128256, dtype="bf16", top_k=5, temperature=1.0,
             banned=False, grad=False),
        # one step of a rollout batch under a vocabulary mask, twenty alternatives
        dict(name="rollout-64x151936", op="logprobs", rows=64, vocab=151936, dtype="bf16", top_k=20, temperature=0.7,
             banned=True, grad=False),
        # scoring an evaluation batch in 32 bits: odd vocabulary, so rows start at any alignment; arg max only
        dict(name="eval-1000x50257", op="logprobs", rows=1000, vocab=50257, dtype="fp32", top_k=1, temperature=1.0,
             banned=False, grad=False),
        # scoring a whole training sequence
        dict(name="score-8192x128256", op="logprobs", rows=8192, vocab=128256, dtype="bf16", top_k=0, temperature=1.0,
             banned=False, grad=False),
        # policy objective with an entropy term: forward and gradient of a head chunk
        dict(name="train-4096x128256", op="logprobs", rows=4096, vocab=128256, dtype="bf16", top_k=0, temperature=1.0,
             banned=False, grad=True),
        # the same on a small ragged batch in 32 bits with banned tokens
        dict(name="train-257x50257", op="logprobs", rows=257, vocab=50257, dtype="fp32", top_k=0, temperature=0.8,
             banned=True, grad=True),
        # one decode step's keys and values
        dict(name="append-64x1", op="append", batch=64, tokens=1, held=1000, kv_heads=8, head_dim=128, block=64,
             dtype="bf16"),
        # the prompts of a batch, right-padded to the longest
        dict(name="prompt-8x8192", op="append", batch=8, tokens=8192, held=0, kv_heads=8, head_dim=128, block=64,
             dtype="bf16"),
        # one served sequence
        dict(name="attend-1x1009", op="attend", batch=1, longest=1009, heads=32, kv_heads=8, head_dim=128, block=64,
             window=0, dtype="bf16"),
        # a rollout batch: prompt of 256 and up to 512 new tokens
        dict(name="attend-64x768", op="attend", batch=64, longest=768, heads=16, kv_heads=8, head_dim=128, block=64,
             window=0, dtype="bf16"),
        # one query head per key head of 64
        dict(name="attend-128x1024", op="attend", batch=128, longest=1024, heads=12, kv_heads=12, head_dim=64, block=64,
             window=0, dtype="fp16"),
        # few sequences, long caches
        dict(name="attend-4x131072", op="attend", batch=4, longest=131072, heads=40, kv_heads=8, head_dim=128, block=64,
             window=0, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["logprobs", "logprobs", "append", "attend", "attend"])
    if op == "logprobs":
        grad = rng.random() < 0.4
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        vocab = rng.choice([_log_int(rng, 97, 152000), 50257, 50304, 128256, 151936])
        top_k = 0 if grad else min(rng.choice([0, 1, 5, 20, 32]), vocab)
        most = (1 << 30 if dtype == "fp32" else 1 << 31) // ((8 if top_k else 4 if grad else 2) * vocab)
        return dict(op=op, rows=_log_int(rng, 1, max(1, min(8192, most))), vocab=vocab, dtype=dtype, top_k=top_k,
                    temperature=rng.choice([1.0, 1.0, round(rng.uniform(0.3, 2.0), 2)]), banned=rng.random() < 0.3,
                    grad=grad)
    kv_heads, rep, hd = rng.choice([(8, 4, 128), (8, 5, 128), (8, 2, 128), (12, 1, 64), (2, 4, 64), (1, 8, 128),
                                    (2, 16, 128), (1, 24, 64), (4, 3, 256), (3, 2, 32)])
    block = rng.choice([16, 32, 64, 64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    batch = _log_int(rng, 1, 128)
    if op == "append":
        tokens = rng.choice([1, _log_int(rng, 1, max(1, min(8192, (1 << 26) // (batch * kv_heads * hd))))])
        held = rng.choice([0, rng.randrange(0, 1500)])
        return dict(op=op, batch=batch, tokens=tokens, held=held, kv_heads=kv_heads, head_dim=hd, block=block, dtype=dtype)
    longest = _log_int(rng, 1, max(1, min(131072, (1 << 29) // (batch * kv_heads * hd))))
    return dict(op=op, batch=batch, longest=longest, heads=kv_heads * rep, kv_heads=kv_heads, head_dim=hd, block=block,
                window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]), dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case):
    """Tokens each sequence of the batch adds (``append``) or holds after the step (``attend``): spread evenly from a
    quarter of the longest to the longest, and one idle slot in batches of eight or more."""
    n, top = case["batch"], case["tokens"] if case["op"] == "append" else case["longest"]
    low = max(1, top // 4)
    out = [top - (top - low) * i // max(1, n - 1) for i in range(n)]
    if n >= 8:
        out[-1] = 0
    return out


def _quantised(x, block):
    """Values ``[heads, tokens, dim]`` (32 bits, tokens a multiple of ``block``) as e4m3 codes and block scales."""
    heads, tokens, dim = x.shape
    y = x.view(heads, tokens // block, block, dim)
    scale = _needed_scale(y.abs().amax(dim=(2, 3)))
    codes = (y / scale[:, :, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return codes.view(heads, tokens, dim), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    state = dict(case=dict(case))
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.empty(rows, vocab, device="cuda", dtype=dtype)
        step = max(1, (1 << 27) // vocab)
        for r in range(0, rows, step):
            n = min(step, rows - r)
            part = normal(n, vocab) * 2.5
            # rows differ in how decided they are
            part *= 0.5 + torch.rand(n, 1, generator=gen, device="cuda")
            logits[r:r + n] = part.to(dtype)
        if case["banned"]:
            ban = torch.rand(vocab, generator=gen, device="cuda") < 0.3
            logits[:, ban] = -math.inf
            if rows > 1:
                logits[rows // 2] = -math.inf     # a row whose mask leaves nothing
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        targets[torch.rand(rows, generator=gen, device="cuda") < 0.05] = -100
        state.update(logits=logits, targets=targets)
        if case["grad"]:
            state.update(d_logp=normal(rows), d_entropy=normal(rows) * 0.1)
            if case["banned"]:
                # no token that counts is a banned one
                state["d_logp"] *= ~ban[targets.clamp(min=0)]
        return state

    batch, kv_heads, hd, block = case["batch"], case["kv_heads"], case["head_dim"], case["block"]
    added = torch.tensor(_lengths(case))
    added = added[torch.randperm(batch, generator=torch.Generator().manual_seed(seed))]
    if case["op"] == "append":
        tokens = case["tokens"]
        held = torch.randint(case["held"] * 3 // 4, case["held"] + 1, (batch,),
                             generator=torch.Generator().manual_seed(seed))
        capacity = case["held"] + tokens
        lens = held + added
        state.update(n_new=added.to("cuda", torch.int32))
    else:
        tokens, capacity, lens = 1, case["longest"], added
    blocks = -(-capacity // block)
    gain = torch.exp(normal(kv_heads, 1, hd) * 0.5)      # channels differ in size
    for name in ("k", "v"):
        store = torch.empty(batch, kv_heads, capacity, hd, dtype=torch.float8_e4m3fn, device="cuda")
        scale = torch.empty(batch, kv_heads, blocks, device="cuda")
        for b in range(batch):
            codes, scale[b] = _quantised(normal(kv_heads, blocks * block, hd) * gain, block)
            store[b] = codes[:, :capacity]
        state[name], state[name + "_scale"] = store, scale
    # keys and values lie behind the queries in rows of one projection
    width = kv_heads * hd
    q_width = case.get("heads", kv_heads) * hd
    rows = torch.empty(batch, tokens, q_width + 2 * width, dtype=dtype, device="cuda")
    rows[..., :q_width] = normal(batch, tokens, q_width).to(dtype)
    rows[..., q_width:q_width + width] = (normal(batch, tokens, kv_heads, hd) * gain[:, 0]).flatten(2).to(dtype)
    rows[..., q_width + width:] = (normal(batch, tokens, kv_heads, hd) * gain[:, 0]).flatten(2).to(dtype)
    state.update(k_new=rows[..., q_width:q_width + width].unflatten(2, (kv_heads, hd)),
                 v_new=rows[..., q_width + width:].unflatten(2, (kv_heads, hd)),
                 seq_lens=lens.to("cuda", torch.int32))
    if case["op"] == "attend":
        state.update(q=rows[:, 0, :q_width].unflatten(1, (case["heads"], hd)), k_new=state["k_new"][:, 0],
                     v_new=state["v_new"][:, 0])
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_logprobs(logits, targets, top_k, temperature, d_logp=None, d_entropy=None):
    """u = (z - max z) / T;  log p_t = u_t - log sum e^u;  H = log sum e^u - sum u e^u / sum e^u;
    the alternatives are the largest logits, equal ones by lowest index; a target outside the vocabulary gives 0;
    a row without any finite logit gives log probabilities of -inf and an entropy of 0."""
    vocab = logits.shape[-1]
    z = logits.float()
    top = z.amax(-1, keepdim=True)
    empty = top == -math.inf
    u = (z - torch.where(empty, 0.0, top)) / temperature
    e = torch.exp(u)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(torch.where(empty, 1.0, total))
    weighted = torch.where(u == -math.inf, 0.0, u * e).sum(-1, keepdim=True)
    entropy = log_total - weighted / torch.where(empty, 1.0, total)
    inside = (targets >= 0) & (targets < vocab)
    logp = u.gather(-1, targets.clamp(0, vocab - 1)[:, None]) - log_total
    out = {"logp": torch.where(inside, logp[:, 0], 0.0), "entropy": entropy[:, 0]}
    if top_k:
        bits = (z + 0.0).view(torch.int32)                                  # one zero
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()      # integers in the order of the values
        place = torch.arange(vocab, device=z.device)
        key = torch.topk(order * (1 << 32) + (vocab - 1 - place), top_k, dim=-1).values
        ids = vocab - 1 - key % (1 << 32)
        out["top_ids"] = ids
        out["top_logp"] = u.gather(-1, ids) - log_total
    if d_logp is not None:
        p = torch.where(empty, 0.0, e / total)
        log_p = u - log_total
        d_h = torch.where(p == 0, 0.0, -p * (log_p + entropy)) * d_entropy[:, None]
        g = d_h - p * (d_logp * inside)[:, None]
        g = g.scatter_add(-1, targets.clamp(0, vocab - 1)[:, None], (d_logp * inside * ~empty[:, 0])[:, None])
        out["grad"] = (g / temperature).to(logits.dtype)
    return out


def _needed_scale(amax):
    """The smallest power of two s with amax <= 448 s, its exponent clamped."""
    mantissa, exponent = torch.frexp(amax)                       # amax = mantissa 2^exponent, mantissa in [0.5, 1)
    exponent = exponent - 9 + (mantissa > 0.875).to(exponent.dtype)
    exponent = torch.where(amax > 0, exponent, SCALE_EXP_MIN).clamp(SCALE_EXP_MIN, SCALE_EXP_MAX)
    return torch.ldexp(torch.ones_like(amax), exponent)


def _plain_append(new, store, scale, lens, n_new, block):
    """Writes ``new[b, :n_new[b]]`` to the positions that end at ``lens[b]``. Every block that gains tokens takes the
    larger of the scale it had for the tokens it held and the scale that the new ones need; if that grew, the tokens
    it held are rounded again at the new scale."""
    batch, heads, capacity, dim = store.shape
    tokens = new.shape[1]
    start = (lens - n_new).long()
    first = start // block
    span = (tokens + 2 * block - 2) // block                     # blocks that a run of `tokens` can touch
    dev = store.device
    blk = first[:, None] + torch.arange(span, device=dev)                                      # [B, span]
    pos = blk[:, :, None] * block + torch.arange(block, device=dev)                            # [B, span, block]
    there = torch.arange(batch, device=dev)
    safe_pos = pos.clamp(max=capacity - 1).view(batch, -1)
    safe_blk = blk.clamp(max=scale.shape[2] - 1)
    is_old = (pos < start[:, None, None]).view(batch, 1, -1, 1)
    is_new = ((pos >= start[:, None, None]) & (pos < lens.long()[:, None, None])).view(batch, 1, -1, 1)
    old_scale = scale[there[:, None], :, safe_blk].transpose(1, 2)                             # [B, heads, span]
    codes = store[there[:, None], :, safe_pos].transpose(1, 2).float()                         # [B, heads, rows, dim]
    take = (safe_pos - start[:, None]).clamp(0, tokens - 1)
    values = new[there[:, None], take].transpose(1, 2).float()
    amax = torch.where(is_new, values.abs(), 0.0).view(batch, heads, span, block, dim).amax(dim=(3, 4))
    holds = is_old.view(batch, 1, span, block).any(-1)
    gains = is_new.view(batch, 1, span, block).any(-1)
    wanted = _needed_scale(amax)
    next_scale = torch.where(holds, torch.maximum(wanted, old_scale), wanted)
    rows = lambda s: s.repeat_interleave(block, dim=2)[..., None]                              # noqa: E731
    values = torch.where(is_new, values, codes * rows(old_scale)) / rows(next_scale)
    values = values.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    put = (is_new | is_old) & rows(gains)                                                      # [B, heads, rows, 1]
    # rows that are not written go where the first new token goes, with its value (row 0 as it is without new tokens)
    some = (n_new > 0).view(batch, 1, 1, 1)
    index = torch.where(n_new > 0, start - first * block, 0)
    anchor = values.view(torch.uint8)[there, :, index][:, :, None]
    anchor = torch.where(some, anchor, store.view(torch.uint8)[:, :, :1])
    target = torch.where(put[..., 0], safe_pos[:, None], torch.where(n_new > 0, start, 0)[:, None, None])
    head = torch.arange(heads, device=dev)[:, None]
    store.view(torch.uint8)[there[:, None, None], head, target] = torch.where(put, values.view(torch.uint8), anchor)
    kept = torch.where(some[..., 0], next_scale[:, :, :1], scale[:, :, :1])
    at = torch.where(gains, safe_blk[:, None], torch.where(n_new > 0, first, 0)[:, None, None]).expand(batch, heads, span)
    scale[there[:, None, None], head, at] = torch.where(gains, next_scale, kept)


def _plain_attend(q, store_k, scale_k, store_v, scale_v, lens, block, window):
    """softmax(q k / sqrt(dim)) v over the last ``window`` of the first ``lens[b]`` tokens; 0 where there are none."""
    batch, heads, dim = q.shape
    kv_heads, capacity = store_k.shape[1], store_k.shape[2]
    spread = lambda s: s.repeat_interleave(block, dim=2)[:, :, :capacity, None]                # noqa: E731
    k = store_k.float() * spread(scale_k)
    at = torch.arange(capacity, device=q.device)
    seen = at < lens[:, None]
    if window:
        seen &= at >= lens[:, None] - window
    seen = seen[:, None, None, :]
    qf = q.float().view(batch, kv_heads, heads // kv_heads, dim)
    s = (qf @ k.transpose(2, 3)) / math.sqrt(dim)
    del k
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p @ (store_v.float() * spread(scale_v))) / torch.where(total == 0, 1.0, total)
    return o.view(batch, heads, dim).to(q.dtype)


def run(state):
    case = state["case"]
    if case["op"] == "logprobs":
        logits, targets = state["logits"], state["targets"]
        if own:
            from optimus_dl_b200.ops.logprobs import token_logprobs

            if case["grad"]:
                logits = logits.detach().requires_grad_(True)
            r = token_logprobs(logits, targets, top_k=case["top_k"], temperature=case["temperature"])
            out = {"logp": r.logp.detach(), "entropy": r.entropy.detach()}
            if case["top_k"]:
                out.update(top_ids=r.top_ids, top_logp=r.top_logp)
            if case["grad"]:
                out["grad"], = torch.autograd.grad([r.logp, r.entropy], [logits], [state["d_logp"], state["d_entropy"]])
            return out
        return _plain_logprobs(logits, targets, case["top_k"], case["temperature"], state.get("d_logp"),
                               state.get("d_entropy"))
    k, v, k_scale, v_scale, lens = state["k"], state["v"], state["k_scale"], state["v_scale"], state["seq_lens"]
    held = {"k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}
    if own:
        from optimus_dl_b200.ops.decode_fp8 import Fp8KVCache, append_kv_fp8, decode_attention_fp8

        cache = Fp8KVCache(k.transpose(1, 2), v.transpose(1, 2), k_scale, v_scale, case["block"])
        if case["op"] == "append":
            append_kv_fp8(state["k_new"], state["v_new"], cache, lens, state["n_new"])
            return held
        out = decode_attention_fp8(state["q"], state["k_new"], state["v_new"], cache, lens,
                                   window=case["window"] or None)
        return {"out": out, **held}
    if case["op"] == "append":
        _plain_append(state["k_new"], k, k_scale, lens, state["n_new"], case["block"])
        _plain_append(state["v_new"], v, v_scale, lens, state["n_new"], case["block"])
        return held
    one = (lens > 0).int()
    _plain_append(state["k_new"][:, None], k, k_scale, lens, one, case["block"])
    _plain_append(state["v_new"][:, None], v, v_scale, lens, one, case["block"])
    return {"out": _plain_attend(state["q"], k, k_scale, v, v_scale, lens, case["block"], case["window"]), **held}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_logprobs(state):
    case, targets = state["case"], state["targets"]
    rows, vocab = state["logits"].shape
    out = {"logp": [], "entropy": []}
    if case["top_k"]:
        out.update(top_ids=[], top_logp=[])
    if case["grad"]:
        out["grad"] = []
    step = max(1, (1 << 26) // vocab)
    for r in range(0, rows, step):
        z = state["logits"][r:r + step].double() / case["temperature"]
        t = targets[r:r + step]
        logp = torch.log_softmax(z, dim=-1)                      # NaN in rows without a finite logit
        none = torch.isnan(logp[:, :1])
        logp = torch.where(none, -math.inf, logp)
        p = logp.exp()
        h = -torch.special.xlogy(p, p).sum(-1)
        counts = (t >= 0) & (t < vocab)
        picked = logp[torch.arange(len(t), device=t.device), torch.where(counts, t, 0)]
        out["logp"].append(torch.where(counts, picked, 0.0))
        out["entropy"].append(h)
        if case["top_k"]:
            ids = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]
            out["top_ids"].append(ids)
            out["top_logp"].append(torch.take_along_dim(logp, ids, -1))
        if case["grad"]:
            a = (state["d_logp"][r:r + step].double() * counts)[:, None]
            c = state["d_entropy"][r:r + step].double()[:, None]
            g = -p * a - c * (torch.special.xlogy(p, p) + p * h[:, None])
            hit = torch.zeros_like(g)
            hit[torch.arange(len(t), device=t.device), torch.where(counts, t, 0)] = 1.0
            out["grad"].append(torch.where(none, 0.0, g + hit * a) / case["temperature"])
    return {k: torch.cat(v) for k, v in out.items()}


def _exact_e4m3(x):
    """Round to the nearest e4m3 value, ties to even: three mantissa bits, smallest exponent -6."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_append(new, store, scale, lens, n_new, block):
    """Block by block; returns codes and scales in 64 bits."""
    codes, scale = store.double(), scale.double()
    for b, (end, n) in enumerate(zip(lens.tolist(), n_new.tolist())):
        start, at = end - n, end - n
        while at < end:
            j = at // block
            stop = min(end, (j + 1) * block)
            fresh = new[b, at - start:stop - start].double().transpose(0, 1)                   # [heads, n, dim]
            amax = fresh.abs().amax(dim=(1, 2))
            need = torch.full_like(amax, 2.0 ** SCALE_EXP_MIN)
            # less than the step between neighbouring inputs, more than the logarithm's own error
            exps = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448.0) - 1e-9).clamp(SCALE_EXP_MIN, SCALE_EXP_MAX)
            need = torch.where(amax > 0, torch.exp2(exps), need)
            if at > j * block:
                was = scale[b, :, j]
                grown = torch.maximum(was, need)
                part = codes[b, :, j * block:at]
                codes[b, :, j * block:at] = _exact_e4m3(part * (was / grown)[:, None, None])
                need = grown
            scale[b, :, j] = need
            codes[b, :, at:stop] = _exact_e4m3(fresh / need[:, None, None])
            at = stop
    return codes, scale


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(state)
    lens, block = state["seq_lens"], case["block"]
    if case["op"] == "append":
        k, k_scale = _exact_append(state["k_new"], state["k"], state["k_scale"], lens, state["n_new"], block)
        v, v_scale = _exact_append(state["v_new"], state["v"], state["v_scale"], lens, state["n_new"], block)
        return {"k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}
    one = (lens > 0).int()
    k, k_scale = _exact_append(state["k_new"][:, None], state["k"], state["k_scale"], lens, one, block)
    v, v_scale = _exact_append(state["v_new"][:, None], state["v"], state["v_scale"], lens, one, block)
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    rep = case["heads"] // case["kv_heads"]
    for b, n in enumerate(lens.tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        at = torch.arange(first, n, device="cuda") // block
        kb = k[b, :, first:n] * k_scale[b][:, at, None]
        vb = v[b, :, first:n] * v_scale[b][:, at, None]
        qb = state["q"][b].double().view(case["kv_heads"], rep, -1)
        w = torch.softmax(torch.einsum("hrd,htd->hrt", qb, kb) / math.sqrt(case["head_dim"]), dim=-1)
        out[b] = torch.einsum("hrt,htd->hrd", w, vb).flatten(0, 1)
    return {"out": out, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        # maximum, difference, exponential, two sums; the gradient adds the product with p and the entropy's part
        flops = n * (6 + (6 if case["grad"] else 0))
        return {"bytes": n * size * (2 if case["grad"] else 1) + case["rows"] * (16 + 12 * case["top_k"]), "flops": flops}
    heads, dim, block = case["kv_heads"], case["head_dim"], case["block"]
    lens = _lengths(case)
    if case["op"] == "append":
        n = sum(lens) * heads * dim * 2
        return {"bytes": n * (size + 1) + sum(-(-x // block) for x in lens) * heads * 8, "flops": 4 * n}
    seen = [min(x, case["window"] or x) for x in lens]
    held = sum(seen) * heads * dim * 2 + sum(-(-x // block) for x in seen) * heads * 8
    step = case["batch"] * (2 * case["heads"] + 2 * heads) * dim * size
    return {"bytes": held + step, "flops": 4 * sum(seen) * case["heads"] * dim}
