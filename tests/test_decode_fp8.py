"""The 8-bit key / value cache and one-token attention over it: the PyTorch statement on the CPU and what it refuses,
the kernels on the GPU against the definition in 64 bits on the same codes.

Tolerances.  Codes and scales have to be equal: every division is by a power of two and every rounding is to nearest
even.  Attention: probabilities are rounded to f16 (half a step, 2^-12 relative, taken twice for the exponential and
the sum in fp32), the output to its own type, so |error| <= 2^-11 sum p |v| / sum p + half a step of |out|.
"""

import math

import pytest
import torch

from optimus_dl_b200.ops import decode_fp8 as d8

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def nearest_e4m3(x):
    """By the list of all values: the nearest, ties to the even code."""
    codes = torch.arange(127, dtype=torch.uint8)
    table = codes.view(torch.float8_e4m3fn).double()
    d = (x.abs()[..., None] - table).abs()
    best = d.min(-1, keepdim=True).values
    tie = d == best
    even = tie & (codes % 2 == 0)
    pick = torch.where(tie.sum(-1) > 1, even.int().argmax(-1), tie.int().argmax(-1))
    return torch.copysign(table[pick], x)


def test_scale_is_the_smallest_power_of_two():
    amax = torch.tensor([448.0, 448.1, 1.0, 1.75, 1.7500001, 3.5, 0.0, 1e-38, 3.3e38, 2.0 ** -112 * 448, 2.0 ** -113 * 448])
    s = d8.needed_scale(amax).double()
    ok = (amax.double() <= 448 * s)
    half = (amax.double() > 224 * s)
    exps = torch.log2(s)
    assert torch.equal(exps, exps.round()) and ok[:8].all() and ok[9:].all()
    assert half[:6].all() and half[9]
    assert s[6] == s[7] == s[10] == 2.0 ** -112 and s[8] == 2.0 ** 119


def test_append_rounds_and_grows():
    torch.manual_seed(0)
    B, T, Hk, hd, block = 2, 21, 2, 32, 16
    cache = d8.fp8_kv_cache(B, 40, Hk, hd, block=block)
    k, v = torch.randn(B, T, Hk, hd), torch.randn(B, T, Hk, hd) * 1e-3
    n = torch.tensor([21, 5], dtype=torch.int32)
    d8.append_kv_fp8(k, v, cache, n, n)
    for b in range(B):
        for j in range(0, int(n[b]), block):
            part = k[b, j:min(j + block, int(n[b]))].double()
            s = d8.needed_scale(part.abs().amax(dim=(0, 2)).float()).double()
            assert torch.equal(cache.k_scale[b, :, j // block].double(), s)
            assert torch.equal(cache.k[b, j:j + part.shape[0]].double(), nearest_e4m3(part / s[:, None]))
    assert not cache.k[1, 5:].float().any() and not cache.k[0, 21:].float().any()
    # a larger token raises its block's scale and rounds the held codes again, and only there
    held, old = cache.k.clone(), cache.k_scale.clone()
    big = torch.full((B, Hk, hd), 900.0)
    big[:, 1] = 0.0
    lens = n + 1
    out = d8.decode_attention_fp8(torch.randn(B, 4, hd), big, big, cache, lens)
    assert out.shape == (B, 4, hd)
    for b in range(B):
        j = (int(lens[b]) - 1) // block
        lo, hi = j * block, int(lens[b]) - 1
        s = cache.k_scale[b, 0, j]
        assert s == 4.0 and torch.equal(cache.k_scale[b, 1], old[b, 1])
        again = nearest_e4m3(held[b, lo:hi, 0].double() * float(old[b, 0, j] / s))
        assert torch.equal(cache.k[b, lo:hi, 0].double(), again)
        assert torch.equal(cache.k[b, lo:hi, 1].float(), held[b, lo:hi, 1].float())
        assert torch.equal(cache.k[b, :lo].float(), held[b, :lo].float())


def test_nan_and_infinity_are_stored_as_nan():
    cache = d8.fp8_kv_cache(1, 16, 1, 32, block=16)
    k = torch.ones(1, 3, 1, 32)
    k[0, 0, 0, 0], k[0, 1, 0, 1], k[0, 2, 0, 2] = math.nan, math.inf, -math.inf
    d8.append_kv_fp8(k, torch.ones_like(k), cache, torch.tensor([3], dtype=torch.int32))
    f = cache.k[0, :3, 0].float()
    assert torch.isnan(f[0, 0]) and torch.isnan(f[1, 1]) and torch.isnan(f[2, 2])
    assert int(torch.isnan(f).sum()) == 3 and torch.isfinite(cache.k_scale).all()


def test_refusals():
    ok = d8.fp8_kv_cache(2, 8, 2, 32, block=16)
    k = torch.zeros(2, 3, 2, 32)
    n = torch.tensor([3, 3], dtype=torch.int32)
    for bad in (torch.tensor([9, 3]), torch.tensor([2, 3]), torch.tensor([3, -1])):
        with pytest.raises(ValueError):
            d8.append_kv_fp8(k, k, ok, bad.int())
    with pytest.raises(ValueError):
        d8.append_kv_fp8(k, k, ok, n, torch.tensor([4, 1], dtype=torch.int32))
    with pytest.raises(ValueError):
        d8.append_kv_fp8(k, k, ok, n.long())
    with pytest.raises(ValueError):
        d8.append_kv_fp8(k[:, :, :1], k[:, :, :1], ok, n)
    with pytest.raises(TypeError):
        d8.append_kv_fp8(k, k.half(), ok, n)
    with pytest.raises(TypeError):
        d8.append_kv_fp8(k.double(), k.double(), ok, n)
    q = torch.zeros(2, 4, 32)
    for bad_q in (torch.zeros(2, 3, 32), torch.zeros(1, 4, 32), torch.zeros(2, 4, 16), torch.zeros(2, 4, 1, 32)):
        with pytest.raises(ValueError):
            d8.decode_attention_fp8(bad_q, None, None, ok, n)
    with pytest.raises(ValueError):
        d8.decode_attention_fp8(q, k[:, 0], None, ok, n)
    with pytest.raises(ValueError):
        d8.decode_attention_fp8(q, None, None, ok, n, window=-1)
    with pytest.raises(TypeError):
        d8.decode_attention_fp8(q.half(), k[:, 0], k[:, 0], ok, n)
    for kw in (dict(block=48), dict(block=8), dict(block=256)):
        with pytest.raises(ValueError):
            d8.fp8_kv_cache(1, 8, 1, 32, **kw)
    with pytest.raises(ValueError):
        d8.fp8_kv_cache(0, 8, 1, 32)
    with pytest.raises(TypeError):
        d8.Fp8KVCache(ok.k.view(torch.uint8), ok.v, ok.k_scale, ok.v_scale, 16)
    with pytest.raises(TypeError):
        d8.Fp8KVCache(ok.k, ok.v, ok.k_scale.double(), ok.v_scale, 16)
    with pytest.raises(ValueError):
        d8.Fp8KVCache(ok.k, ok.v, ok.k_scale[:, :1], ok.v_scale[:, :1], 16)
    with pytest.raises(ValueError):
        d8.Fp8KVCache(ok.k, ok.v[:, :4], ok.k_scale, ok.v_scale, 16)


# ------------------------------------------------------------------------------------------------ GPU
def filled(B, capacity, Hk, hd, block, seed=0, token_major=False):
    """A cache with random codes and scales on the GPU, NaN codes everywhere a kernel must not look."""
    g = torch.Generator("cuda").manual_seed(seed)
    shape = (B, capacity, Hk, hd) if token_major else (B, Hk, capacity, hd)
    nb = -(-capacity // block)

    def one():
        c = (torch.randn(shape, generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
        c = c if token_major else c.permute(0, 2, 1, 3)
        return c, torch.exp2(torch.randint(-9, -4, (B, Hk, nb), generator=g, device="cuda").float())

    (k, ks), (v, vs) = one(), one()
    return d8.Fp8KVCache(k, v, ks, vs, block)


def spoil(cache, lens):
    """NaN codes behind every sequence's last token."""
    dead = torch.arange(cache.k.shape[1], device="cuda") >= lens[:, None]
    for c in (cache.k, cache.v):
        raw = c.view(torch.uint8)
        raw.masked_fill_(dead[:, :, None, None], 0x7F)


def exact(q, cache, lens, window, scale):
    B, Hq, hd = q.shape
    Hk = cache.k.shape[2]
    out, size = torch.zeros(2, B, Hq, hd, dtype=torch.float64)
    for b in range(B):
        n = min(int(lens[b]), cache.k.shape[1])
        first = max(0, n - window) if window else 0
        if n <= 0:
            continue
        j = torch.arange(first, n, device=q.device) // cache.block
        k = cache.k[b, first:n].double() * cache.k_scale[b][:, j].t()[..., None]
        v = cache.v[b, first:n].double() * cache.v_scale[b][:, j].t()[..., None]
        s = torch.einsum("hrd,thd->hrt", q[b].double().view(Hk, Hq // Hk, hd), k) * scale
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("hrt,thd->hrd", p, v).reshape(Hq, hd).cpu()
        size[b] = torch.einsum("hrt,thd->hrd", p, v.abs()).reshape(Hq, hd).cpu()
    return out, size


def assert_near(got, want, size):
    err = (got.double().cpu() - want).abs()
    tol = HALF_STEP[got.dtype] * want.abs() + 2.0 ** -11 * size + 1e-7
    assert bool((err <= tol).all()), float((err / tol).max())


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 200, 333]


@pytest.mark.gpu
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hd,Hq,Hk,block,window", [
    (128, 8, 2, 64, None), (128, 5, 1, 16, None), (64, 12, 12, 32, None), (64, 9, 1, 64, 40), (128, 40, 8, 128, 100),
    (128, 32, 2, 64, None), (128, 34, 2, 64, 1), (32, 6, 2, 16, None), (32, 24, 1, 128, 17), (256, 4, 2, 64, None),
    (256, 20, 1, 32, 64)])
def test_attention_matches_definition(hd, Hq, Hk, block, window, dtype, token_major):
    torch.manual_seed(1)
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    B = len(LENS)
    cache = filled(B, 333, Hk, hd, block, token_major=token_major)
    spoil(cache, lens)
    q = (torch.randn(B, Hq, hd, device="cuda") * 0.7).to(dtype)
    out = d8.decode_attention_fp8(q, None, None, cache, lens, window=window)
    want, size = exact(q, cache, lens, window, 1 / math.sqrt(hd))
    assert_near(out, want, size)
    assert torch.equal(out, d8.decode_attention_fp8(q, None, None, cache, lens, window=window))
    assert not out[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hd,Hk,block,T", [(128, 2, 64, 1), (128, 3, 64, 200), (64, 2, 16, 37), (32, 1, 16, 5),
                                           (256, 2, 128, 300), (32, 4, 128, 129)])
def test_append_matches_statement(hd, Hk, block, T, dtype):
    torch.manual_seed(2)
    B, capacity = 7, 333
    counts = [T, 0, 1, max(1, T // 2), T, min(T, 3), T - 1]
    held = [0, 9, 15, 16, min(33, capacity - T), capacity - min(T, 3), 0]
    n = torch.tensor(counts, dtype=torch.int32, device="cuda")
    lens = n + torch.tensor(held, dtype=torch.int32, device="cuda")
    cache = filled(B, capacity, Hk, hd, block)
    twin = d8.Fp8KVCache(cache.k.clone(), cache.v.clone(), cache.k_scale.clone(), cache.v_scale.clone(), block)
    rows = torch.randn(B, T, 3 * Hk * hd, device="cuda").to(dtype)
    rows[0, 0, -1], rows[4, 0, Hk * hd] = math.inf, math.nan
    k = rows[..., Hk * hd:2 * Hk * hd].unflatten(2, (Hk, hd)) * 3
    k[2] = 0
    k = torch.cat([rows[..., :Hk * hd], k.flatten(2)], -1)[..., Hk * hd:].unflatten(2, (Hk, hd))
    v = rows[..., 2 * Hk * hd:].unflatten(2, (Hk, hd))
    d8.append_kv_fp8(k, v, cache, lens, n)
    d8.append_kv_fp8_ref(k, v, twin, lens, n)
    for a, b in ((cache.k, twin.k), (cache.v, twin.v)):
        fa, fb = a.float(), b.float()
        assert torch.equal(torch.isnan(fa), torch.isnan(fb)) and torch.equal(fa.nan_to_num(), fb.nan_to_num())
    assert torch.equal(cache.k_scale, twin.k_scale) and torch.equal(cache.v_scale, twin.v_scale)
    keep = cache.k.clone()
    d8.append_kv_fp8(k, v, cache, lens, n)         # the same tokens again change nothing
    assert torch.equal(keep.view(torch.uint8), cache.k.view(torch.uint8))


@pytest.mark.gpu
def test_counts_that_do_not_fit_are_reported_and_leave_the_cache():
    from optimus_dl_b200.ops import _lib

    _lib.check_status()
    cache = filled(4, 50, 2, 64, 16)
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale)]
    k = torch.randn(4, 3, 2, 64, device="cuda").bfloat16()
    lens = torch.tensor([51, 2, -5, 4], dtype=torch.int32, device="cuda")
    n = torch.tensor([3, 3, 1, 4], dtype=torch.int32, device="cuda")
    d8.append_kv_fp8(k, k, cache, lens, n)
    after = [cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale]
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    with pytest.raises(_lib.KernelError):
        _lib.check_status()
    _lib.check_status()


@pytest.mark.gpu
def test_steps_match_the_statement_over_time():
    """Fill a cache token by token through the step, as generation does, next to the statement."""
    torch.manual_seed(3)
    B, Hq, Hk, hd, block = 3, 8, 2, 64, 16
    a, b = (d8.fp8_kv_cache(B, 70, Hk, hd, block=block, device="cuda") for _ in range(2))
    prompt = torch.randn(B, 19, 2 * Hk, hd, device="cuda").bfloat16()
    n = torch.tensor([19, 4, 0], dtype=torch.int32, device="cuda")
    for c, f in ((a, d8.append_kv_fp8), (b, d8.append_kv_fp8_ref)):
        f(prompt[:, :, :Hk], prompt[:, :, Hk:], c, n, n)
    lens = n.clone()
    for i in range(50):
        lens = lens + (lens > 0).int()
        row = (torch.randn(B, (Hq + 2 * Hk) * hd, device="cuda") * (1.0 + i % 7)).bfloat16()
        q = row[:, :Hq * hd].unflatten(1, (Hq, hd))
        kn, vn = row[:, Hq * hd:(Hq + Hk) * hd].unflatten(1, (Hk, hd)), row[:, (Hq + Hk) * hd:].unflatten(1, (Hk, hd))
        out = d8.decode_attention_fp8(q, kn, vn, a, lens)
        want = d8.decode_attention_fp8_ref(q.float(), kn.float(), vn.float(), b, lens)
        assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v_scale, b.v_scale)
        exact_out, size = exact(q, a, lens, None, 1 / math.sqrt(hd))
        assert_near(out, exact_out, size)
        assert float((want.double().cpu() - exact_out).abs().max()) < 1e-4


@pytest.mark.gpu
def test_values_of_very_different_blocks():
    """Scales 2^60 apart, a dominant token, and scores beyond f16."""
    cache = filled(2, 300, 1, 128, 16)
    cache.v_scale[0, 0] = torch.exp2(torch.linspace(-30, 30, 19, device="cuda").round())
    cache.v_scale[1, 0] = cache.v_scale[0, 0].flip(0)
    cache.k_scale[:] = 2.0
    q = torch.randn(2, 4, 128, device="cuda") * 1e3
    q[0, 0] *= 1e-30
    q[1, 1] *= 1e25
    q[1, 2] = 0
    q = q.bfloat16()
    lens = torch.tensor([300, 299], dtype=torch.int32, device="cuda")
    out = d8.decode_attention_fp8(q, None, None, cache, lens, scale=1e-5)
    assert torch.isfinite(out).all()
    want, size = exact(q, cache, lens, None, 1e-5)
    ok = torch.ones(2, 4, dtype=torch.bool)
    ok[1, 1] = False             # scores of 1e25: the two largest differ by rounding alone
    assert_near(out[ok.cuda()], want[ok], size[ok])


@pytest.mark.gpu
def test_nan_code_in_a_seen_token_shows():
    cache = filled(2, 64, 2, 64, 16)
    cache.k.view(torch.uint8)[0, 3, 1, 5] = 0x7F
    cache.v.view(torch.uint8)[1, 7, 0, 9] = 0xFF
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    out = d8.decode_attention_fp8(q, None, None, cache, torch.tensor([64, 20], dtype=torch.int32, device="cuda"))
    assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2]).all()
    assert torch.isnan(out[1, :2, 9]).all() and torch.isfinite(out[1, 2:]).all() and torch.isfinite(out[1, :2, :9]).all()


@pytest.mark.gpu
def test_many_sequences_and_lengths_beyond_the_capacity():
    B = 5003                      # more than one launch holds
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(0, 40, (B,), generator=g).int()
    lens[7] = 1000
    lens = lens.cuda()
    cache = filled(B, 33, 1, 32, 16)
    q = torch.randn(B, 2, 32, device="cuda").bfloat16()
    out = d8.decode_attention_fp8(q, None, None, cache, lens)
    ref = d8.decode_attention_fp8_ref(q.double(), None, None, cache, lens)
    cache.v.view(torch.uint8).bitwise_and_(0x7F)
    size = d8.decode_attention_fp8_ref(q.double(), None, None, cache, lens)
    assert_near(out, ref.cpu(), size.cpu())


@pytest.mark.gpu
def test_more_sequences_than_a_grid_dimension_holds():
    B = 70001
    cache = d8.fp8_kv_cache(B, 5, 1, 32, block=16, device="cuda")
    k = torch.randn(B, 2, 1, 32, device="cuda").bfloat16()
    lens = torch.full((B,), 2, dtype=torch.int32, device="cuda")
    d8.append_kv_fp8(k, -k, cache, lens)
    d8.append_kv_fp8(2 * k[:, :1], k[:, 1:], cache, lens + 1)
    s = d8.needed_scale(k.float().abs().amax(dim=(1, 2, 3)))
    grown = torch.maximum(s, d8.needed_scale(2 * k[:, 0].float().abs().amax(dim=(1, 2))))
    assert torch.equal(cache.k_scale[:, 0, 0], grown)
    first = (k.float() / s[:, None, None, None]).to(torch.float8_e4m3fn).float()
    want = (first * (s / grown)[:, None, None, None]).to(torch.float8_e4m3fn).float()
    assert torch.equal(cache.k[:, :2].float(), want)
    assert torch.equal(cache.k[:, 2].float(), (2 * k[:, 0].float() / grown[:, None, None]).to(torch.float8_e4m3fn).float())


@pytest.mark.gpu
def test_strides_of_single_dimensions_mean_nothing_and_odd_rows_are_copied():
    cache = filled(1, 50, 1, 64, 16)
    k = cache.k.as_strided(cache.k.shape, (7, 64, 3, 1))
    odd = d8.Fp8KVCache(k, cache.v, cache.k_scale.as_strided((1, 1, 4), (9, 5, 1)), cache.v_scale, 16)
    lens = torch.tensor([50], dtype=torch.int32, device="cuda")
    base = torch.randn(1, 3, 3 * 64 + 1, device="cuda").bfloat16()
    q, kn, vn = base[:, :, 1:65], base[:, :1, 65:129], base[:, 1:2, 129:193]
    out = d8.decode_attention_fp8(q, kn, vn, odd, lens)
    want = d8.decode_attention_fp8(q.contiguous(), kn.contiguous(), vn.contiguous(), cache, lens)
    assert torch.equal(out, want)
    ref, size = exact(q, cache, lens, None, 0.125)
    assert_near(out, ref, size)


@pytest.mark.gpu
def test_one_long_sequence_past_32_bit_offsets():
    """2.3 GB of codes for keys alone: the last tokens' offsets do not fit 32 bits."""
    T, Hk, hd = 1_100_003, 8, 256
    k = torch.zeros(1, Hk, T, hd, dtype=torch.uint8, device="cuda")
    v = torch.zeros_like(k)
    n = 70
    g = torch.Generator("cuda").manual_seed(0)
    tail = (torch.randn(2, 1, Hk, n, hd, generator=g, device="cuda") * 50).to(torch.float8_e4m3fn).view(torch.uint8)
    k[:, :, -n:], v[:, :, -n:] = tail[0], tail[1]
    blocks = -(-T // 64)
    s = torch.ones(1, Hk, blocks, device="cuda")
    cache = d8.Fp8KVCache(k.view(torch.float8_e4m3fn).permute(0, 2, 1, 3), v.view(torch.float8_e4m3fn).permute(0, 2, 1, 3),
                          s, s.clone(), 64)
    q = torch.randn(1, 16, hd, device="cuda").bfloat16()
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    out = d8.decode_attention_fp8(q, None, None, cache, lens, window=n, scale=0.01)
    want, size = exact(q, cache, lens, n, 0.01)
    assert_near(out, want, size)
    full = d8.decode_attention_fp8(q, None, None, cache, lens, scale=0.01)
    # every token before the tail scores 0 and holds 0
    s_tail = torch.einsum("hrd,htd->hrt", q.double().view(Hk, 2, hd), tail[0, 0].view(torch.float8_e4m3fn).double()) * 0.01
    v_tail = tail[1, 0].view(torch.float8_e4m3fn).double()
    top = s_tail.amax(-1, keepdim=True).clamp(min=0)
    e = torch.exp(s_tail - top)
    total = e.sum(-1, keepdim=True) + (T - n) * torch.exp(-top)
    want = (torch.einsum("hrt,htd->hrd", e, v_tail) / total).reshape(1, 16, hd)
    size = (torch.einsum("hrt,htd->hrd", e, v_tail.abs()) / total).reshape(1, 16, hd)
    # probabilities of up to 10^6 equal tokens are exact in f16 (powers of two times e^-top are not: counted in size)
    assert_near(full, want.cpu(), size.cpu())


@pytest.mark.gpu
def test_captured_steps_replay_with_new_lengths():
    B, Hq, Hk, hd = 4, 8, 2, 128
    cache = filled(B, 500, Hk, hd, 64)
    twin = d8.Fp8KVCache(cache.k.clone(), cache.v.clone(), cache.k_scale.clone(), cache.v_scale.clone(), 64)
    lens = torch.tensor([1, 100, 64, 0], dtype=torch.int32, device="cuda")
    q = torch.randn(B, Hq, hd, device="cuda").bfloat16()
    kv = torch.randn(2, B, Hk, hd, device="cuda").bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                    # on a stream of its own, into scratch
        d8.decode_attention_fp8(q, None, None, cache, lens)
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(d8.decode_attention_fp8(q, kv[0], kv[1], cache, lens))
    for step in range(4):
        lens.copy_(torch.tensor([2 + step, 101 + 90 * step, 65 + step, 0], dtype=torch.int32))
        q.normal_()
        kv.normal_()
        graphs[step % 2].replay()
        want = d8.decode_attention_fp8(q, kv[0], kv[1], twin, lens)
        assert torch.equal(outs[step % 2], want)
        assert torch.equal(cache.k.view(torch.uint8), twin.k.view(torch.uint8))
