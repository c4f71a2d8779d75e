"""The 8-bit cache at its edges: layouts, ranges of scales, windows, what is refused and what must stay as it was.

Codes and scales have to be equal to the PyTorch statement's. Attention is compared with the definition in 64 bits.
Probabilities times value scales are rounded to f16 relative to the largest such product met (half a step, 2^-12, for
what lies above 2^-21 of it, else 2^-32 of it), exponentials and sums are fp32 (2^-20 and less): |error| <= 2^-11
sum p |v| / sum p + 2^-32 * 448 max(p s_v) / sum p + half a step of |out|.
"""

import math

import pytest
import torch

from optimus_dl_b200.ops import decode_fp8 as d8

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def same_cache(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in ((a.k, b.k), (a.v, b.v))) and \
        torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)


def test_rows_that_are_broadcast_along_the_head_dimension_are_laid_out():
    """What the kernels read is hd numbers from every row's first one on."""
    one = torch.tensor(3.0).bfloat16()
    for k in (one.expand(2, 2, 32), torch.randn(2, 5, 2, 1).half().expand(2, 5, 2, 32)):
        for v in (k, torch.zeros(k.shape, dtype=k.dtype)):
            a, b, strides = d8._new_rows(k, v)
            assert strides[-1] == 1 and a.stride(-1) == 1 and b.stride(-1) == 1
            assert torch.equal(a, k) and torch.equal(b, v)


def test_broadcast_codes_and_scales_are_refused():
    ok = d8.fp8_kv_cache(2, 40, 2, 32, block=16)
    flat = torch.zeros(2, 40, 2, 1, dtype=torch.uint8).view(torch.float8_e4m3fn).expand(2, 40, 2, 32)
    with pytest.raises(ValueError):
        d8.Fp8KVCache(flat, flat, ok.k_scale, ok.v_scale, 16)
    scale = torch.ones(2, 2, 1).expand(2, 2, 3)
    with pytest.raises(ValueError):
        d8.Fp8KVCache(ok.k, ok.v, scale, scale, 16)
    one = d8.fp8_kv_cache(2, 16, 2, 32, block=16)          # one block: its stride means nothing
    d8.Fp8KVCache(one.k, one.v, torch.ones(2, 2, 1).expand(2, 2, 1), one.v_scale, 16)


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_broadcast_rows_equal_their_contiguous_form(dtype):
    torch.manual_seed(0)
    B, Hk, hd, T = 3, 2, 64, 5
    lens = torch.tensor([5, 20, 33], dtype=torch.int32, device="cuda")
    rows = [torch.randn(B, T, Hk, 1, device="cuda").to(dtype).expand(B, T, Hk, hd),
            torch.randn(B, 1, 1, hd, device="cuda").to(dtype).expand(B, T, Hk, hd),
            torch.tensor(2.5, device="cuda").to(dtype).expand(B, T, Hk, hd)]
    for k in rows:
        for v in rows:
            a, b = (d8.fp8_kv_cache(B, 40, Hk, hd, block=16, device="cuda") for _ in range(2))
            d8.append_kv_fp8(k, v, a, lens)
            d8.append_kv_fp8(k.contiguous(), v.contiguous(), b, lens)
            assert same_cache(a, b)
            if dtype == torch.float32:
                continue
            q = torch.randn(B, 4, hd, device="cuda").to(dtype)
            out = d8.decode_attention_fp8(q, k[:, 0], v[:, 0], a, lens + 1)
            assert torch.equal(out, d8.decode_attention_fp8(q, k[:, 0].contiguous(), v[:, 0].contiguous(), b, lens + 1))
            assert same_cache(a, b)
