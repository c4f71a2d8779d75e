"""Key / value cache held in 8 bits, and one-token attention over it.

The cache stores e4m3 codes and one fp32 scale for each block of tokens and kv head (keys and values apart): half the
bytes of the bf16 cache of :mod:`.decode`, which is what a decode step's time and a rollout's memory consist of.

    code = round_to_e4m3(x / s),  s = the smallest power of two with  max |x| over the block <= 448 s

(its exponent between -112 and 119). A block that gains tokens keeps its scale, unless the new ones need a larger one;
then the codes it holds are rounded again at the larger scale. Powers of two make every division exact, so the result
does not depend on how a value is computed. NaN stays NaN and infinities become NaN; neither sets a scale.

``append_kv_fp8`` writes new tokens (a padded batch of prompts, or one token each), ``decode_attention_fp8`` appends
one token per sequence and attends. CUDA runs ``csrc/kv_fp8.cu`` and ``csrc/attention_decode_fp8.cu`` for head
dimensions 32, 64, 128 and 256, any number of query heads per kv head and bf16 / fp16 queries; the ``*_ref`` functions
are the PyTorch statements of the same semantics and serve CPU runs, tests and whatever the kernels do not take.
"""

from __future__ import annotations

import functools
import math
from dataclasses import dataclass

import torch

from . import _lib

E4M3_MAX = 448.0
SCALE_EXP_MIN, SCALE_EXP_MAX = -112, 119
BLOCKS = (16, 32, 64, 128)
_HEAD_DIMS = (32, 64, 128, 256)
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_CACHE = "QQqqqQQqq"                     # as Fp8KVCache._args gives it
_launch_append = _lib.Packed("ob_kv_fp8_append", "QQqqqq" + _CACHE + "QQqqqqqqQQ")
_launch_attention = _lib.Packed("ob_attn_decode_fp8", "QqqQQqq" + _CACHE + "QQQqqqqqqdqQQ")


def has_kernel(head_dim: int, dtype: torch.dtype) -> bool:
    """Whether decode steps of this head dimension and model type run in the CUDA kernels."""
    return head_dim in _HEAD_DIMS and dtype in (torch.bfloat16, torch.float16)


def _strides(t: torch.Tensor) -> tuple[int, ...]:
    """Strides, 0 for dimensions of size 1 (whose stride means nothing)."""
    strides, shape = t.stride(), t.shape
    return tuple([s if n > 1 else 0 for n, s in zip(shape, strides)]) if 1 in shape else strides


@dataclass(frozen=True, eq=False)
class Fp8KVCache:
    """``k``, ``v``: logical ``[B, capacity, Hk, hd]`` float8_e4m3fn with a unit stride in the last dimension and any
    others (a head-major allocation viewed this way reads fastest); ``k_scale``, ``v_scale``: fp32
    ``[B, Hk, ceil(capacity / block)]`` with a unit stride in the blocks, powers of two (a cache that repeats a sequence
    or a head by a stride of 0, or has keys and values in one place, can be attended over, not written); ``block``: tokens that share a scale (16, 32, 64 or 128)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    block: int = 64

    def __post_init__(self) -> None:
        k, v, ks, vs, block = self.k, self.v, self.k_scale, self.v_scale, self.block
        if block not in BLOCKS:
            raise ValueError(f"block must be one of {BLOCKS}, got {block}")
        if k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
            raise TypeError(f"codes must be float8_e4m3fn, got {k.dtype} and {v.dtype}")
        if ks.dtype != torch.float32 or vs.dtype != torch.float32:
            raise TypeError(f"scales must be float32, got {ks.dtype} and {vs.dtype}")
        shape, strides, scale_strides = k.shape, _strides(k), _strides(ks)
        if 0 in shape[1:]:
            raise ValueError(f"a cache needs at least one token, head and dimension, got {tuple(shape)}")
        if (len(shape) != 4 or shape != v.shape or strides[3] != (shape[3] > 1)
                or (k.stride() != v.stride() and strides != _strides(v))):
            raise ValueError("k and v must be [B, capacity, Hk, hd] of the same shape and strides, contiguous in hd")
        B, capacity, Hk, hd = shape
        want = (B, Hk, -(-capacity // block))
        if (ks.shape != want or vs.shape != want or scale_strides[2] != (want[2] > 1)
                or (ks.stride() != vs.stride() and scale_strides != _strides(vs))):
            raise ValueError(f"k_scale and v_scale must be {want} of the same strides, contiguous in the blocks")
        dev = k.device
        if v.device != dev or ks.device != dev or vs.device != dev:
            raise ValueError("codes and scales must be on one device")
        codes_k, codes_v = k.data_ptr(), v.data_ptr()
        if dev.type == "cuda":
            sb, st, sh, _ = strides
            kernels = hd in _HEAD_DIMS and not (sb | st | sh | codes_k | codes_v) & 15
            geometry, status = (sb, st, sh, scale_strides[0], scale_strides[1]), _lib.status_word(dev)
        else:
            kernels, geometry, status = False, None, None
        shared = (codes_k == codes_v or ks.data_ptr() == vs.data_ptr()) and k.numel() > 0
        if 0 in strides or 0 in scale_strides:       # of a dimension of size 1, or of several elements in one place
            shared = shared or any(n > 1 and s == 0 for n, s in (*zip(shape, strides), *zip(want, scale_strides)))
        # the status word exists before any capture into a graph
        self.__dict__.update(_device=dev, _index=k.get_device(), _shape=tuple(shape), _kernels=kernels, _geometry=geometry,
                             _status=status, _shared=shared)

    def _args(self) -> tuple:
        """What describes the cache to the kernels: codes and their strides, scales and theirs."""
        sb, st, sh, cb, ch = self._geometry
        return (self.k.data_ptr(), self.v.data_ptr(), sb, st, sh, self.k_scale.data_ptr(), self.v_scale.data_ptr(), cb, ch)


def fp8_kv_cache(batch: int, max_len: int, n_kv_head: int, head_dim: int, *, block: int = 64,
                 device: torch.device | str | None = None) -> Fp8KVCache:
    """An empty cache, stored head-major."""
    if min(batch, max_len, n_kv_head, head_dim) < 1:
        raise ValueError("a cache needs at least one sequence, token, head and dimension")
    if block not in BLOCKS:
        raise ValueError(f"block must be one of {BLOCKS}, got {block}")
    shape = (batch, n_kv_head, max_len, head_dim)
    codes = [torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.full((batch, n_kv_head, -(-max_len // block)), 2.0 ** SCALE_EXP_MIN, device=device) for _ in range(2)]
    return Fp8KVCache(codes[0].permute(0, 2, 1, 3), codes[1].permute(0, 2, 1, 3), scales[0], scales[1], block)


def _check_new(k_new: torch.Tensor, v_new: torch.Tensor, cache: Fp8KVCache, want: tuple) -> None:
    if k_new.shape != want or v_new.shape != want:
        raise ValueError(f"new keys and values must be {want}, got {tuple(k_new.shape)} and {tuple(v_new.shape)}")
    if k_new.dtype != v_new.dtype or k_new.dtype not in _DTYPES:
        raise TypeError(f"new keys and values must share one of bf16, fp16, fp32: got {k_new.dtype}, {v_new.dtype}")
    if k_new.get_device() != cache._index or v_new.get_device() != cache._index:
        raise ValueError("new keys and values must be on the cache's device")
    if cache._shared:
        raise ValueError("sequences, tokens, heads or keys and values of this cache share memory: it can be read only")


def _check_counts(t: torch.Tensor, cache: Fp8KVCache, batch: int, what: str) -> None:
    if t.dtype != torch.int32 or t.shape != (batch,) or t.get_device() != cache._index or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 [{batch}] on the cache's device, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def _row_strides(t: torch.Tensor) -> tuple[torch.Tensor, tuple[int, ...]]:
    """``t`` and its strides, or those of a copy if its rows (last dimension) are not contiguous or do not start on
    16-byte boundaries."""
    strides = _strides(t)
    bits, size = t.data_ptr(), t.element_size()
    for s in strides[:-1]:
        bits |= s * size
    if strides[-1] != 1 or bits & 15:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = _strides(t)
    return t, strides


def _new_rows(k_new: torch.Tensor, v_new: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, tuple[int, ...]]:
    """New keys and values as the kernels take them: rows on 16-byte boundaries, the same strides for both."""
    if k_new.stride() == v_new.stride():
        strides, size = _strides(k_new), k_new.element_size()
        bits = k_new.data_ptr() | v_new.data_ptr()
        for s in strides[:-1]:
            bits |= s * size
        if strides[-1] == 1 and not bits & 15:
            return k_new, v_new, strides
    k_new, k_strides = _row_strides(k_new)
    v_new, v_strides = _row_strides(v_new)
    if k_strides != v_strides:
        k_new, v_new = k_new.contiguous(), v_new.contiguous()
        k_strides = _strides(k_new)
    return k_new, v_new, k_strides


def append_kv_fp8(k_new: torch.Tensor, v_new: torch.Tensor, cache: Fp8KVCache, seq_lens: torch.Tensor,
                  n_new: torch.Tensor | None = None) -> None:
    """Write ``k_new`` / ``v_new [B, T, Hk, hd]`` (bf16, fp16 or fp32) into the cache.

    ``seq_lens`` (int32 ``[B]``) counts the tokens of each sequence *including* the new ones; the last ``n_new[b]`` of
    them are ``k_new[b, :n_new[b]]`` (default: all ``T``, and none for a sequence of length 0). Rows behind a
    sequence's last token stay as they were. Counts that do not fit (``n_new`` outside ``[0, T]``, more new tokens than
    the sequence has, a length beyond the capacity) raise on the CPU; on CUDA the sequence is left as it was and
    ``ops._lib.check_status`` raises.
    """
    B, capacity, Hk, hd = cache._shape
    if k_new.dim() != 4:
        raise ValueError(f"new keys must be [B, T, Hk, hd], got {tuple(k_new.shape)}")
    T = k_new.shape[1]
    _check_new(k_new, v_new, cache, (B, T, Hk, hd))
    _check_counts(seq_lens, cache, B, "seq_lens")
    if n_new is not None:
        _check_counts(n_new, cache, B, "n_new")
    if T == 0:
        return
    if not cache._kernels:
        append_kv_fp8_ref(k_new, v_new, cache, seq_lens, n_new)
        return
    k_new, v_new, (nb, nt, nh, _) = _new_rows(k_new, v_new)
    with _lib.on_device(cache._device):
        _launch_append(k_new.data_ptr(), v_new.data_ptr(), _DTYPES[k_new.dtype], nb, nt, nh, *cache._args(),
                       seq_lens.data_ptr(), 0 if n_new is None else n_new.data_ptr(), B, T, Hk, hd, capacity, cache.block,
                       cache._status.data_ptr(), _lib.raw_stream(cache._index))


def needed_scale(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two ``s`` with ``amax <= 448 s``, its exponent clamped."""
    mantissa, exponent = torch.frexp(amax.float())               # mantissa in [0.5, 1); 448 = 0.875 * 2^9
    exponent = torch.where(amax > 0, exponent - 9 + (mantissa > 0.875).int(), SCALE_EXP_MIN)
    return torch.ldexp(torch.ones_like(mantissa), exponent.clamp(SCALE_EXP_MIN, SCALE_EXP_MAX))


def _to_codes(x: torch.Tensor) -> torch.Tensor:
    """Bytes of the e4m3 values nearest to ``x`` (fp32): finite ones saturate, infinities become NaN."""
    x = torch.where(torch.isinf(x), math.nan, x).clamp(-E4M3_MAX, E4M3_MAX)
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _append_one_ref(new: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, lens: torch.Tensor, n: torch.Tensor,
                    block: int) -> None:
    raw = codes.view(torch.uint8)
    for b in range(new.shape[0]):
        end = int(lens[b])
        start = at = end - int(n[b])
        while at < end:
            j = at // block
            row0, stop = j * block, min(end, (j + 1) * block)
            fresh = new[b, at - start:stop - start].float()                                   # [n, Hk, hd]
            size = torch.where(torch.isfinite(fresh), fresh.abs(), 0.0).amax(dim=(0, 2))
            s = needed_scale(size)
            if at > row0:
                was = scale[b, :, j].clone()
                s = torch.maximum(s, was)
                held = codes[b, row0:at].float() * (was / s)[:, None]
                raw[b, row0:at] = _to_codes(held)
            raw[b, at:stop] = _to_codes(fresh / s[:, None])
            scale[b, :, j] = s
            at = stop


@torch.no_grad()
def append_kv_fp8_ref(k_new: torch.Tensor, v_new: torch.Tensor, cache: Fp8KVCache, seq_lens: torch.Tensor,
                      n_new: torch.Tensor | None = None) -> None:
    """PyTorch statement of :func:`append_kv_fp8`, block by block."""
    T, capacity = k_new.shape[1], cache.k.shape[1]
    n = torch.where(seq_lens == 0, 0, T) if n_new is None else n_new
    bad = (n < 0) | (n > T) | (n > seq_lens) | (seq_lens > capacity)
    if bool(bad.any()):
        raise ValueError(f"sequences {bad.nonzero().flatten().tolist()}: the counts do not fit the cache")
    _append_one_ref(k_new, cache.k, cache.k_scale, seq_lens, n, cache.block)
    _append_one_ref(v_new, cache.v, cache.v_scale, seq_lens, n, cache.block)


def decode_attention_fp8(q: torch.Tensor, k_new: torch.Tensor | None, v_new: torch.Tensor | None, cache: Fp8KVCache,
                         seq_lens: torch.Tensor, *, scale: float | None = None,
                         window: int | None = None) -> torch.Tensor:
    """Attention of one query token per sequence against its 8-bit cache; the counterpart of
    :func:`.decode.decode_attention`.

    ``q``: ``[B, Hq, hd]`` (a strided view into a fused qkv row is fine); ``k_new`` / ``v_new [B, Hk, hd]``: the current
    token's, appended as token ``seq_lens[b] - 1`` first (``None`` if already stored); ``seq_lens``: int32 ``[B]``,
    counts *including* the current token, taken as the capacity where larger (the new token of such a sequence is not
    stored: that raises as in :func:`append_kv_fp8`); ``window``: attend to the last so many tokens only, 0 or None to
    all. A sequence of length 0 appends nothing and gives zeros. Returns ``[B, Hq, hd]`` of the type of ``q``, without
    a gradient.
    """
    B, capacity, Hk, hd = cache._shape
    shape = q.shape
    if len(shape) != 3 or shape[0] != B or shape[2] != hd or shape[1] % Hk:
        raise ValueError(f"q {tuple(shape)} does not fit a cache of {tuple(cache.k.shape)}")
    dtype, Hq = q.dtype, shape[1]
    if not dtype.is_floating_point:
        raise TypeError(f"q must be floating point, got {dtype}")
    if q.get_device() != cache._index:
        raise ValueError("q must be on the cache's device")
    _check_counts(seq_lens, cache, B, "seq_lens")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new come together")
    if k_new is not None:
        _check_new(k_new, v_new, cache, (B, Hk, hd))
        if k_new.dtype != dtype:
            raise TypeError(f"q and the new keys must have one type, got {dtype} and {k_new.dtype}")
    if window is not None and window < 0:
        raise ValueError(f"window must not be negative, got {window}")
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    if not (cache._kernels and has_kernel(hd, dtype)):
        return decode_attention_fp8_ref(q, k_new, v_new, cache, seq_lens, scale=scale, window=window)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if B == 0:
        return out
    if Hq == 0:
        if k_new is not None:
            append_kv_fp8(k_new[:, None], v_new[:, None], cache, seq_lens)
        return out
    q_batch, q_head, q_last = q.stride()
    if q_last != 1 or q_head != hd or (2 * q_batch | q.data_ptr()) & 15:
        q = q.clone(memory_format=torch.contiguous_format)
        q_batch = Hq * hd
    new_k = new_v = new_batch = new_head = 0
    if k_new is not None:
        k_new, v_new, (new_batch, new_head, _) = _new_rows(k_new, v_new)
        new_k, new_v = k_new.data_ptr(), v_new.data_ptr()
    ws = torch.empty(_workspace(B, Hq, Hk, hd, capacity), dtype=torch.uint8, device=cache._device)
    with _lib.on_device(cache._device):
        _launch_attention(q.data_ptr(), q_batch, _DTYPES[dtype], new_k, new_v, new_batch, new_head, *cache._args(),
                          seq_lens.data_ptr(), out.data_ptr(), ws.data_ptr(), B, Hq, Hk, hd, capacity, cache.block, scale,
                          window or 0, cache._status.data_ptr(), _lib.raw_stream(cache._index))
    return out


@functools.lru_cache(maxsize=256)
def _workspace(B: int, Hq: int, Hk: int, hd: int, capacity: int) -> int:
    return _lib.lib().ob_attn_decode_fp8_workspace(B, Hq, Hk, hd, capacity)


@torch.no_grad()
def decode_attention_fp8_ref(q, k_new, v_new, cache: Fp8KVCache, seq_lens, *, scale=None, window=None) -> torch.Tensor:
    """PyTorch statement of :func:`decode_attention_fp8` in fp32 (fp64 for fp64 queries); also appends."""
    B, Hq, hd = q.shape
    capacity, Hk = cache.k.shape[1], cache.k.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(hd)
    if k_new is not None:
        append_kv_fp8_ref(k_new[:, None], v_new[:, None], cache, seq_lens)
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    lens = seq_lens.long().clamp(0, capacity)
    pos = torch.arange(capacity, device=q.device)
    seen = pos < lens[:, None]
    if window:
        seen = seen & (pos >= lens[:, None] - int(window))
    block = pos // cache.block

    def values(codes, scales):                                     # [B, Hk, T, hd]; unseen rows may hold anything
        x = codes.to(wide).transpose(1, 2) * scales.to(wide)[:, :, block, None]
        return torch.where(seen[:, None, :, None], x, 0.0)

    s = q.to(wide).view(B, Hk, Hq // Hk, hd) @ values(cache.k, cache.k_scale).transpose(2, 3) * scale
    s = s.masked_fill(~seen[:, None, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = p @ values(cache.v, cache.v_scale) / torch.where(total == 0, 1.0, total)
    return o.reshape(B, Hq, hd).to(q.dtype)
