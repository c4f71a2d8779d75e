"""Log probabilities of given tokens, with entropy and the most likely alternatives.

For a row of logits ``z`` over ``V`` tokens, a token ``t`` and a temperature ``T``::

    log p_j = z_j / T - log sum_i exp(z_i / T)
    logp    = log p_t            entropy = - sum_j p_j log p_j            top = the k largest log p_j

``token_logprobs`` reads the logits once (``csrc/logprobs.cu``) and is differentiable in ``logp`` and ``entropy``;
``linear_token_logprobs`` does the same for a head projection without holding all logits. Both have PyTorch
statements with the same semantics for CPU runs and tests. The reference scores with ``log_softmax`` over whole
``[batch, tokens, vocab]`` logits (optimus_dl/modules/eval/model.py:69-165).

Rules, the same on every path:

* a token id outside ``[0, V)`` (such as the criterion's ignore index) marks a position without a token: its log
  probability is 0 and it gets no gradient; entropy and alternatives do not depend on the token;
* a banned token (logit ``-inf``) has probability 0 and adds nothing to the entropy; a row with nothing but banned
  tokens has log probabilities of ``-inf``, entropy 0 and no gradient;
* alternatives are ordered by logit, equal ones by lowest id;
* a row with a NaN or ``+inf`` gives NaN; NaN counts as the largest logit among the alternatives.
"""

from __future__ import annotations

import contextlib
import math
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import _lib, gemm

MAX_TOP_K = 32
_KERNEL_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_launch_forward = _lib.Packed("ob_logprobs_fwd", "QqqQQQQQQQqqqdQ")
_launch_backward = _lib.Packed("ob_logprobs_bwd", "QqqQQQQQQqqqdQ")


@dataclass
class TokenLogprobs:
    logp: torch.Tensor                 # log p(token), fp32, shape of the tokens
    entropy: torch.Tensor              # entropy of the row's distribution in nats, fp32, same shape
    top_logp: torch.Tensor | None      # [..., k] log probabilities of the k most likely tokens, most likely first
    top_ids: torch.Tensor | None       # [..., k] their ids, int64


def _check(rows_shape: torch.Size, vocab: int, floating: torch.Tensor, targets: torch.Tensor, top_k: int,
           temperature: float) -> None:
    if not floating.is_floating_point():
        raise TypeError(f"logits must be floating point, got {floating.dtype}")
    if targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool:
        raise TypeError(f"targets must be token ids of an integer type, got {targets.dtype}")
    if targets.shape != rows_shape:
        raise ValueError(f"targets have shape {tuple(targets.shape)}, the rows of logits {tuple(rows_shape)}")
    if targets.get_device() != floating.get_device():
        raise ValueError(f"targets are on {targets.device}, logits on {floating.device}")
    if vocab < 1:
        raise ValueError("logits need at least one token")
    if not 0 <= top_k <= min(MAX_TOP_K, vocab):
        raise ValueError(f"top_k must be between 0 and {min(MAX_TOP_K, vocab)}, got {top_k}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"temperature must be between 1e-6 and 1e6, got {temperature}")


def _largest(z: torch.Tensor, k: int) -> torch.Tensor:
    """Ids ``[rows, k]`` of the largest of ``z [rows, V]``: the largest first, equal ones by lowest id, NaN above all."""
    if k == 1:
        return z.argmax(-1, keepdim=True)          # the first of equal maxima
    # sorting whole rows for this takes 20 times the rest of the statement; topk orders equal values as it likes
    kth = torch.topk(z, k).values[:, -1:]
    if bool(torch.isnan(kth).any()):
        return torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]
    keep = ~(z < kth)                              # k of them, and what is equal to the last
    more = (keep.sum(-1) > k).nonzero()[:, 0]
    if len(more):
        some, last = z[more], kth[more]
        equal = some == last
        above = keep[more] & ~equal
        keep[more] = above | (equal & (equal.cumsum(-1) <= k - above.sum(-1, keepdim=True)))
    ids = keep.nonzero()[:, 1].view(-1, k)
    return ids.gather(-1, torch.sort(z.gather(-1, ids), dim=-1, descending=True, stable=True).indices)


class _TokenLogprobsRef(torch.autograd.Function):
    CHUNK = 1 << 20                                # logits taken at a time: what stays in a processor's cache

    @staticmethod
    def forward(ctx, logits, targets, top_k, temperature):
        shape, vocab = targets.shape, logits.shape[-1]
        wide = logits.dtype if logits.dtype == torch.float64 else torch.float32
        z2, at = logits.reshape(-1, vocab), targets.reshape(-1).long()
        rows = z2.shape[0]
        inside = (at >= 0) & (at < vocab)
        at = at.clamp(0, vocab - 1).unsqueeze(-1)
        new = lambda *size, dtype=wide: torch.empty(size, dtype=dtype, device=logits.device)    # noqa: E731
        results = [new(*shape), new(*shape)]           # no views of one another: they may be changed in place
        if top_k:
            results += [new(*shape, top_k), new(*shape, top_k, dtype=torch.int64)]
        logp, entropy, *listed = [r.view(rows, *r.shape[len(shape):]) for r in results]
        counts = new(rows, dtype=torch.bool)
        kept = new(rows, vocab) if ctx.needs_input_grad[0] else None
        step = max(1, _TokenLogprobsRef.CHUNK // vocab)
        for r in range(0, rows, step):
            part = slice(r, r + step)
            z = z2[part].to(wide)
            top = z.amax(-1, keepdim=True)
            none = top == -math.inf
            top = torch.where(none, 0.0, top)
            u = z - top
            if temperature != 1.0:
                u.div_(temperature)
            e = torch.exp(u)
            total = torch.where(none, 1.0, e.sum(-1, keepdim=True))
            log_total = torch.log(total)
            if kept is not None:
                torch.sub(u, log_total, out=kept[part])
            # a banned token adds 0 and not -inf * 0
            moment = e.mul_(u.clamp_(min=-1e6)).sum(-1, keepdim=True)
            entropy[part] = (log_total - moment / total)[:, 0]
            log_p = lambda ids: (z.gather(-1, ids) - top) / temperature - log_total             # noqa: E731
            logp[part] = torch.where(inside[part], log_p(at[part])[:, 0], 0.0)
            counts[part] = inside[part] & ~none[:, 0]
            if top_k:
                listed[1][part] = _largest(z, top_k)
                listed[0][part] = log_p(listed[1][part])
        if kept is not None:
            ctx.save_for_backward(kept.view(logits.shape), entropy.clone().view(*shape, 1), counts.view(shape),
                                  at.view(*shape, 1))                        # what is kept is not shared
        ctx.dtype, ctx.temperature = logits.dtype, temperature
        ctx.mark_non_differentiable(*results[2:])
        return (*results, None, None)[:4]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_logp, d_entropy, *_):
        log_p, entropy, counts, at = ctx.saved_tensors
        p = torch.exp(log_p)
        a = torch.where(counts, d_logp, 0.0).unsqueeze(-1)
        g = -p * a - d_entropy.unsqueeze(-1) * torch.where(p == 0, 0.0, p * (log_p + entropy))
        g = g.scatter_add(-1, at, a)
        return (g / ctx.temperature).to(ctx.dtype), None, None, None


def token_logprobs_ref(logits: torch.Tensor, targets: torch.Tensor, *, top_k: int = 0,
                       temperature: float = 1.0) -> TokenLogprobs:
    """PyTorch statement of :func:`token_logprobs`: in fp32, or in fp64 for fp64 logits."""
    return TokenLogprobs(*_TokenLogprobsRef.apply(logits, targets, top_k, temperature))


def _forward(z: torch.Tensor, targets: torch.Tensor, top_k: int, temperature: float, keep: bool):
    """Kernel call on ``z [rows, V]`` (unit column stride) and contiguous int64 ``targets [rows]``. Returns ``logp,
    entropy, top_logp, top_ids, kept``; with ``keep``, ``kept`` is what the gradient needs, none of it shared with the
    results: the maximum and log2 sum of every row as pairs, then the entropy."""
    rows, vocab = z.shape
    dev = z.device
    logp = torch.empty(rows, dtype=torch.float32, device=dev)
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    top_logp = top_ids = kept = None
    pairs = 0
    if keep:
        kept = torch.empty(3 * rows, dtype=torch.float32, device=dev)
        pairs = kept.data_ptr()
    if top_k:      # empty_strided: the cheapest way to a new tensor on the host
        top_logp = torch.empty_strided((rows, top_k), (top_k, 1), dtype=torch.float32, device=dev)
        top_ids = torch.empty_strided((rows, top_k), (top_k, 1), dtype=torch.int64, device=dev)
    with _lib.on_device(dev):
        _launch_forward(z.data_ptr(), z.stride(0), _KERNEL_DTYPES[z.dtype], targets.data_ptr(), logp.data_ptr(),
                        entropy.data_ptr(), pairs, pairs + 8 * rows, top_logp.data_ptr() if top_k else 0,
                        top_ids.data_ptr() if top_k else 0, rows, vocab, top_k, temperature, _lib.raw_stream(dev.index))
    return logp, entropy, top_logp, top_ids, kept


def _rows_fp32(g: torch.Tensor) -> torch.Tensor:
    return g if g.dtype == torch.float32 and g.is_contiguous() else g.to(torch.float32).contiguous()


def _backward(z: torch.Tensor, targets: torch.Tensor, kept: torch.Tensor, d_logp: torch.Tensor | None,
              d_entropy: torch.Tensor | None, temperature: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """``d loss / d z`` from what ``_forward`` kept; ``out`` may be ``z`` itself."""
    rows, vocab = z.shape
    if out is None:
        out = torch.empty_like(z, memory_format=torch.contiguous_format)
    # the converted gradients live until the launch has been queued
    d_logp = None if d_logp is None else _rows_fp32(d_logp)
    d_entropy = None if d_entropy is None else _rows_fp32(d_entropy)
    at = kept.data_ptr()
    with _lib.on_device(z.device):
        _launch_backward(z.data_ptr(), z.stride(0), _KERNEL_DTYPES[z.dtype], targets.data_ptr(), at, at + 8 * rows,
                         0 if d_logp is None else d_logp.data_ptr(),
                         0 if d_entropy is None else d_entropy.data_ptr(), out.data_ptr(), out.stride(0), rows, vocab,
                         temperature, _lib.raw_stream(z.device.index))
    return out


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, targets, top_k, temperature):
        logp, entropy, top_logp, top_ids, kept = _forward(z, targets, top_k, temperature, True)
        ctx.save_for_backward(z, targets, kept)
        ctx.temperature = temperature
        ctx.set_materialize_grads(False)
        if not top_k:
            return logp, entropy
        ctx.mark_non_differentiable(top_logp, top_ids)
        return logp, entropy, top_logp, top_ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_logp, d_entropy, *_):
        if d_logp is None and d_entropy is None:
            return None, None, None, None
        z, targets, kept = ctx.saved_tensors
        return _backward(z, targets, kept, d_logp, d_entropy, ctx.temperature), None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, top_k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities of ``targets [...]`` under ``logits [..., V]`` (see the module docstring).

    bf16, fp16 and fp32 logits of any row stride run in one kernel on CUDA; ``logp`` and ``entropy`` are
    differentiable, the alternatives (``top_k`` of them, at most 32) are not.
    """
    top_k, temperature = int(top_k), float(temperature)
    if logits.dim() < 1:
        raise ValueError("logits need a vocabulary dimension")
    vocab, shape = logits.shape[-1], targets.shape
    _check(logits.shape[:-1], vocab, logits, targets, top_k, temperature)
    if not (logits.is_cuda and logits.dtype in _KERNEL_DTYPES):
        return token_logprobs_ref(logits, targets, top_k=top_k, temperature=temperature)
    flat = len(shape) == 1
    z, tg = logits, targets
    if not flat:
        z, tg = z.reshape(-1, vocab), tg.reshape(-1)
    if z.stride(1) != 1 and vocab > 1:
        z = z.contiguous()
    if tg.dtype != torch.int64 or not tg.is_contiguous():
        tg = tg.to(torch.int64).contiguous()
    top_logp = top_ids = None
    if z.requires_grad and torch.is_grad_enabled():
        if top_k:
            logp, entropy, top_logp, top_ids = _TokenLogprobs.apply(z, tg, top_k, temperature)
        else:
            logp, entropy = _TokenLogprobs.apply(z, tg, 0, temperature)
    else:
        logp, entropy, top_logp, top_ids, _ = _forward(z, tg, top_k, temperature, False)
    if not flat:
        logp, entropy = logp.view(shape), entropy.view(shape)
        if top_k:
            top_logp, top_ids = top_logp.view(*shape, top_k), top_ids.view(*shape, top_k)
    return TokenLogprobs(logp, entropy, top_logp, top_ids)


@torch.no_grad()
def linear_token_logprobs(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, top_k: int = 0,
                          temperature: float = 1.0, chunk_rows: int = 4096) -> TokenLogprobs:
    """:func:`token_logprobs` of the logits ``x [..., d] @ weight [V, d]^T``, without gradients.

    Rows are taken ``chunk_rows`` at a time, so no more than a chunk of logits is held.
    """
    top_k, temperature = int(top_k), float(temperature)
    if x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise ValueError(f"a weight of {tuple(weight.shape)} does not fit rows of {tuple(x.shape)}")
    if weight.device != x.device:
        raise ValueError(f"weight is on {weight.device}, the rows on {x.device}")
    vocab = weight.shape[0]
    _check(x.shape[:-1], vocab, x, targets, top_k, temperature)
    if chunk_rows < 1:
        raise ValueError(f"chunk_rows must be positive, got {chunk_rows}")
    with _lib.on_device(x.device) if x.is_cuda else contextlib.nullcontext():
        return _linear_token_logprobs(x, weight, targets, top_k, temperature, chunk_rows)


def _linear_token_logprobs(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, top_k: int, temperature: float,
                           chunk_rows: int) -> TokenLogprobs:
    shape, d, vocab = targets.shape, x.shape[-1], weight.shape[0]
    x2, tg = x.reshape(-1, d), targets.reshape(-1)
    kernel = x.is_cuda and x.dtype == torch.bfloat16 and weight.dtype == torch.bfloat16 and d % 8 == 0
    if kernel:
        x2 = x2.contiguous()
    rows = x2.shape[0]
    ld = (vocab + 7) // 8 * 8
    buf = None
    parts = []
    for r0 in range(0, rows, chunk_rows):
        r1 = min(rows, r0 + chunk_rows)
        if kernel:
            if buf is None:
                buf = torch.empty((min(chunk_rows, rows), ld), dtype=torch.bfloat16, device=x.device)
            logits = buf[: r1 - r0, :vocab]
            gemm.gemm(x2[r0:r1], weight, out=logits)
        else:
            logits = F.linear(x2[r0:r1], weight)
        parts.append(token_logprobs(logits, tg[r0:r1], top_k=top_k, temperature=temperature))
    if not parts:
        parts.append(token_logprobs(x.new_empty((0, vocab)), tg, top_k=top_k, temperature=temperature))
    cat = lambda ts: ts[0] if len(ts) == 1 else torch.cat(ts)                                   # noqa: E731
    return TokenLogprobs(cat([p.logp for p in parts]).view(shape), cat([p.entropy for p in parts]).view(shape),
                         cat([p.top_logp for p in parts]).view(*shape, top_k) if top_k else None,
                         cat([p.top_ids for p in parts]).view(*shape, top_k) if top_k else None)
