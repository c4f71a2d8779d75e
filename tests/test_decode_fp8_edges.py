"""The 8-bit cache at its edges: layouts, ranges of scales, windows, what is refused and what must stay as it was.

Codes and scales have to be equal to the PyTorch statement's. Attention is compared with the definition in 64 bits. The
kernel rounds p s_v (probability times value scale) to f16: by 2^-11 of itself at most while it is above 2^-21 of the
largest of its head, and by 2^-32 of that largest one below; codes are at most 448. Exponentials, scores and sums of fp32
add less than 2^-18. So |error| <= ((2^-11 + 2^-18) sum p |v| + n 2^-32 448 max(p s_v)) / sum p + half a step of |out|.
"""

import math

import pytest
import torch

from optimus_dl_b200.ops import decode_fp8 as d8

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def random_cache(B, capacity, Hk, hd, block, seed=0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    codes = [(torch.randn(B, Hk, capacity, hd, generator=g) * 60).clamp(-448, 448).to(torch.float8_e4m3fn).to(device)
             for _ in range(2)]
    nb = -(-capacity // block)
    scales = [torch.exp2(torch.randint(-9, -4, (B, Hk, nb), generator=g).float()).to(device) for _ in range(2)]
    return d8.Fp8KVCache(codes[0].permute(0, 2, 1, 3), codes[1].permute(0, 2, 1, 3), *scales, block)


def check_attention(q, cache, lens, window=None, scale=None, out=None):
    B, Hq, hd = q.shape
    Hk = cache.k.shape[2]
    c = 1 / math.sqrt(hd) if scale is None else scale
    if out is None:
        out = d8.decode_attention_fp8(q, None, None, cache, lens, window=window, scale=scale)
    for b in range(B):
        n = min(int(lens[b]), cache.k.shape[1])
        first = max(0, n - window) if window else 0
        if n <= 0:
            assert not out[b].any()
            continue
        j = torch.arange(first, n, device=q.device) // cache.block
        k = cache.k[b, first:n].double() * cache.k_scale[b][:, j].t()[..., None]
        sv = cache.v_scale[b][:, j].double()                                             # [Hk, n]
        v = cache.v[b, first:n].double() * sv.t()[..., None]
        s = torch.einsum("hrd,thd->hrt", q[b].double().view(Hk, Hq // Hk, hd), k) * c
        p = torch.softmax(s, -1)
        want = torch.einsum("hrt,thd->hrd", p, v).reshape(Hq, hd)
        size = torch.einsum("hrt,thd->hrd", p, v.abs()).reshape(Hq, hd)
        most = (p * sv[:, None]).amax(-1).reshape(Hq, 1)
        tol = (2.0 ** -11 + 2.0 ** -18) * size + (n - first) * 2.0 ** -32 * 448 * most + HALF_STEP[q.dtype] * want.abs()
        err = (out[b].double() - want).abs() / (tol + torch.finfo(q.dtype).tiny)
        assert bool((err <= 1).all()), (b, float(err.max()))
    return out


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


def test_neither_the_cache_nor_the_result_takes_part_in_a_gradient():
    cache = d8.fp8_kv_cache(2, 40, 2, 32, block=16)
    k, q = torch.randn(2, 3, 2, 32, requires_grad=True), torch.randn(2, 4, 32, requires_grad=True)
    lens = torch.tensor([3, 3], dtype=torch.int32)
    d8.append_kv_fp8(k, k, cache, lens)
    out = d8.decode_attention_fp8(q, k[:, 0], k[:, 0], cache, lens + 1)
    assert not any(t.requires_grad for t in (out, cache.k, cache.v, cache.k_scale, cache.v_scale))


def test_caches_that_share_memory_are_read_only():
    """Two sequences in one place would be written by two CTAs at once."""
    a = d8.fp8_kv_cache(1, 40, 1, 32, block=16)
    d8.append_kv_fp8(torch.randn(1, 40, 1, 32), torch.randn(1, 40, 1, 32), a, torch.tensor([40], dtype=torch.int32))
    own = d8.fp8_kv_cache(3, 40, 2, 32, block=16)
    shared = [d8.Fp8KVCache(a.k.expand(3, 40, 2, 32), a.v.expand(3, 40, 2, 32), a.k_scale.expand(3, 2, 3),
                            a.v_scale.expand(3, 2, 3), 16),
              d8.Fp8KVCache(own.k, own.v, a.k_scale.expand(3, 2, 3), a.v_scale.expand(3, 2, 3), 16),
              d8.Fp8KVCache(own.k, own.k, own.k_scale, own.v_scale, 16),
              d8.Fp8KVCache(own.k, own.v, own.k_scale, own.k_scale, 16)]
    new, q = torch.randn(3, 2, 2, 32), torch.randn(3, 4, 32)
    lens = torch.tensor([40, 17, 2], dtype=torch.int32)
    for cache in shared:
        with pytest.raises(ValueError, match="share memory"):
            d8.append_kv_fp8(new, new, cache, lens)
        with pytest.raises(ValueError, match="share memory"):
            d8.decode_attention_fp8(q, new[:, 0], new[:, 0], cache, lens)
        assert torch.isfinite(d8.decode_attention_fp8(q, None, None, cache, lens)).all()
    one = d8.decode_attention_fp8(q[:1], None, None, d8.Fp8KVCache(a.k.expand(1, 40, 2, 32), a.v.expand(1, 40, 2, 32),
                                                                   a.k_scale.expand(1, 2, 3), a.v_scale.expand(1, 2, 3), 16),
                                  lens[:1])
    assert torch.equal(d8.decode_attention_fp8(q, None, None, shared[0], lens)[:1], one)


def test_caches_without_anything_in_them_are_refused_but_for_an_empty_batch():
    for shape in ((2, 0, 2, 32), (2, 40, 0, 32), (2, 40, 2, 0)):
        codes = torch.zeros(shape, dtype=torch.uint8).view(torch.float8_e4m3fn)
        scales = torch.ones(shape[0], shape[2], -(-shape[1] // 16))
        with pytest.raises(ValueError, match="at least one"):
            d8.Fp8KVCache(codes, codes.clone(), scales, scales.clone(), 16)
    codes, scales = torch.zeros(0, 40, 2, 32, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(0, 2, 3)
    empty, none = d8.Fp8KVCache(codes, codes.clone(), scales, scales.clone(), 16), torch.zeros(0, dtype=torch.int32)
    rows = torch.zeros(0, 2, 32)
    assert d8.decode_attention_fp8(torch.zeros(0, 4, 32), rows, rows, empty, none).shape == (0, 4, 32)


def _step_without_query_heads(device):
    cache = d8.fp8_kv_cache(2, 40, 2, 32, block=16, device=device)
    new = torch.ones(2, 2, 32, device=device).bfloat16()
    lens = torch.tensor([1, 0], dtype=torch.int32, device=device)
    out = d8.decode_attention_fp8(new[:, :0], new, new, cache, lens)
    assert out.shape == (2, 0, 32)
    assert bool((cache.k[0, 0].float() == 256).all()) and not cache.k[1].float().any()


def test_a_step_without_query_heads_stores_its_token():
    _step_without_query_heads("cpu")


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
def test_a_step_without_query_heads_stores_its_token_on_the_gpu():
    _step_without_query_heads("cuda")


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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd,Hq,Hk", [(32, 3, 1), (64, 2, 2), (128, 8, 2), (128, 12, 1), (256, 4, 2)])
def test_a_block_of_large_values_and_no_probability_hides_nothing(hd, Hq, Hk, dtype):
    """Blocks whose values are up to 2^60 times the others', with scores 60 below them (p = 2^-86), wherever they lie: the
    result is that of the other blocks. And the other way round: p = 2^-14, but values that outweigh all others."""
    torch.manual_seed(4)
    B, capacity, block = 8, 12000, 16                  # several blocks a warp
    lens = torch.tensor([12000, 33, 17, 9000, 64, 11650, 0, 5001], dtype=torch.int32, device="cuda")
    q = torch.ones(B, Hq, hd, device="cuda").to(dtype) + 0.25 * torch.randn(B, Hq, hd, device="cuda").to(dtype)
    step = math.sqrt(hd) / hd
    for drop, ratio in ((60.0, 10), (60.0, 30), (60.0, 60), (10.0, 20), (10.0, 12)):
        if dtype == torch.float16 and drop < 60:
            ratio = min(ratio, 12)                     # results that this type holds
        for first, every in ((0, 4), (1, 2), (2, 7), (0, 10 ** 6)):
            cache = random_cache(B, capacity, Hk, hd, block)
            cache.k.view(torch.uint8).copy_((torch.randn(B, capacity, Hk, hd, device="cuda") * 4).to(
                torch.float8_e4m3fn).view(torch.uint8))
            cache.k_scale.fill_(2.0 ** -6)
            cache.v_scale.fill_(2.0 ** -8)
            s = 2.0 ** (math.ceil(math.log2(drop * step)) - 8)
            code = torch.full((), -drop * step / s, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8)
            large = torch.arange(capacity, device="cuda") // block % every == first
            cache.k.view(torch.uint8).copy_(torch.where(large[:, None, None], code, cache.k.view(torch.uint8)))
            cache.k_scale[:, :, first::every] = s
            cache.v_scale[:, :, first::every] = 2.0 ** (ratio - 8)
            check_attention(q, cache, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,Hq,Hk,window", [(128, 8, 2, 1), (128, 20, 1, 37), (64, 3, 3, 64), (32, 6, 2, 100), (256, 2, 2, 16)])
def test_tokens_before_the_window_are_not_looked_at(hd, Hq, Hk, window):
    """NaN codes on both sides of what a sequence may see."""
    torch.manual_seed(5)
    lens = torch.tensor([0, 1, 16, 63, 64, 65, 300, 333], dtype=torch.int32, device="cuda")
    cache = random_cache(8, 333, Hk, hd, 64)
    at = torch.arange(333, device="cuda")
    dead = (at >= lens[:, None]) | (at < lens[:, None] - window)
    for c in (cache.k, cache.v):
        c.view(torch.uint8).masked_fill_(dead[:, :, None, None], 0x7F)
    q = torch.randn(8, Hq, hd, device="cuda").bfloat16()
    check_attention(q, cache, lens, window=window)


@pytest.mark.gpu
def test_scores_beyond_fp32_leave_the_other_tokens():
    """A unit of tokens whose every score is -inf in fp32 (so its probabilities are 0), then ordinary ones."""
    cache = random_cache(2, 64, 1, 64, 16)
    cache.k.view(torch.uint8)[:, :16] = 0xFE                     # -448
    cache.k_scale[:, :, 0] = 2.0 ** 115
    q = torch.full((2, 2, 64), 1000.0, device="cuda").bfloat16()
    lens = torch.tensor([64, 16], dtype=torch.int32, device="cuda")
    cache.k.view(torch.uint8)[:, 16:] = 0
    out = d8.decode_attention_fp8(q, None, None, cache, lens)
    want = (cache.v[0, 16:, 0].double() * cache.v_scale[0, 0, 1:].double().repeat_interleave(16)[:, None]).mean(0)
    size = (cache.v[0, 16:, 0].double() * cache.v_scale[0, 0, 1:].double().repeat_interleave(16)[:, None]).abs().mean(0)
    assert bool(((out[0].double() - want).abs() <= 2.0 ** -10 * size + 2.0 ** -8 * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_value_scales_that_are_no_number_show_and_zeros_count_nothing(hd):
    torch.manual_seed(6)
    cache = random_cache(4, 200, 2, hd, 16)
    lens = torch.tensor([200, 100, 200, 200], dtype=torch.int32, device="cuda")
    cache.v_scale[0, 1, 3] = math.nan
    cache.v_scale[1, 0, 7:] = math.nan              # tokens 112 and on: not seen
    cache.v_scale[2, :, 1::2] = 0.0
    cache.v_scale[3] = 0.0
    q = torch.randn(4, 6, hd, device="cuda").bfloat16()
    out = d8.decode_attention_fp8(q, None, None, cache, lens)
    assert torch.isnan(out[0, 3:]).all() and torch.isfinite(out[0, :3]).all() and torch.isfinite(out[1:]).all()
    assert float(out[3].abs().max()) < 1e-30
    cache.v_scale[0, 1, 3] = 1.0
    cache.v_scale[1, 0, 7:] = 1.0
    cache.v_scale[3] = 1.0
    check_attention(q, cache, lens)


@pytest.mark.gpu
def test_captured_appends_replay_with_other_counts():
    B, T, Hk, hd = 5, 9, 2, 64
    k, v = (torch.empty(B, T, Hk, hd, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    lens, n = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    a, b = (d8.fp8_kv_cache(B, 100, Hk, hd, block=16, device="cuda") for _ in range(2))
    d8.append_kv_fp8(k, v, a, lens, n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d8.append_kv_fp8(k, v, a, lens, n)
    g = torch.Generator().manual_seed(0)
    for step in range(8):
        more = torch.randint(0, T + 1, (B,), generator=g).int()
        n.copy_(more)
        lens.add_(n)
        k.normal_().mul_(1 + step)
        v.normal_()
        graph.replay()
        d8.append_kv_fp8_ref(k, v, b, lens, n)
        assert same_cache(a, b)


@pytest.mark.gpu
def test_two_threads_step_over_caches_of_their_own():
    import threading

    def work(seed):
        g = torch.Generator().manual_seed(seed)
        cache = random_cache(3, 400, 2, 128, 64, seed)
        lens = torch.tensor([100, 0, 300], dtype=torch.int32, device="cuda")
        out = []
        for _ in range(20):
            q, kn, vn = (torch.randn(3, h, 128, generator=g).bfloat16().cuda() for h in (8, 2, 2))
            lens = lens + (lens > 0).int()
            out.append(d8.decode_attention_fp8(q, kn, vn, cache, lens))
        return torch.stack(out)

    want = [work(s) for s in (1, 2)]
    torch.cuda.synchronize()
    got = [None, None]

    def run(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = work(i + 1)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
