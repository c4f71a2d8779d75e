// Attention of one query token per sequence over a cache of e4m3 codes with one power-of-two scale for each block of
// tokens and head (kv_fp8.cuh), with the append of the new token in front.
//
//   q     [B, Hq, HD]  bf16 / fp16          k, v  logical [B, capacity, Hk, HD] codes, any batch / token / head strides
//   out   [B, Hq, HD]  type of q            scales [B, Hk, blocks] fp32
//
//   out_h = sum_t p_t v_t s_v(t) / sum_t p_t,   p_t = exp(q_h . k_t s_k(t) / sqrt(HD) - max)
//
// The kernel is bound by the stream of codes (2 HD bytes per token and kv head).  What follows from that:
//
// * Codes go straight from global memory to registers with 16-byte loads, no shared memory in between.  The products
//   run transposed, S^T = K Q^T and O^T = V^T P^T, on 16 x 8 x 16 tensor-core tiles (mma.sync: a tile is far too small
//   for tcgen05): tokens are the M side of the first product and head dimensions that of the second, the up to 8 query
//   heads that share a kv head are the N side of both, so no row of a tile is padding.  The K side of either product
//   may be permuted freely, so each thread takes its 16 contiguous bytes as they come: for K as consecutive k pairs of
//   one token, for V as the same 16 dimensions of four tokens, whose bytes are interleaved with byte permutes.  e4m3
//   to f16 is one exact conversion for two codes; P gets from the accumulator layout of the first product to the
//   operand layout of the second with one 8 x 8 transpose (movmatrix) for 8 tokens.
// * q is scaled by a power of two per head so that its largest element lies in [2^14, 2^15): f16 then holds a bf16 or
//   fp16 q exactly down to 2^-28 of that.  Probabilities are held as p 2^15 s_v / r in f16, r being the largest
//   value scale met so far, so the smallest normal one is 2^-29 of the row's maximum and nothing overflows.  Scores,
//   maxima, sums and both accumulators are fp32.
// * Work is cut evenly, not by sequence: units of 16 tokens of one (sequence, kv head, group of query heads) are
//   numbered through the batch, every CTA takes an equal run of them and every warp an equal part of that.  A warp
//   that sees all units of a segment writes its output; parts are joined first inside the CTA through shared memory
//   (at most two per warp) and then, at most two per CTA, by a second kernel.  A ragged batch or a single long
//   sequence therefore keeps every SM busy to the end, and the workspace does not depend on the batch.
#include "kv_fp8.cuh"

namespace ob {
namespace decode_fp8 {

using namespace kvfp8;

constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr int UNIT = 16;                 // tokens
constexpr int MAX_BATCH = 4096;          // sequences per launch (their unit counts are held in shared memory)
constexpr int COMBINE_GROUPS = 8;

struct Params {
  const void* q; long long q_batch;      // elements; heads are contiguous
  const uint8_t *k, *v;
  long long batch, tok, head;            // bytes
  const float *k_scale, *v_scale;
  long long scale_batch, scale_head;
  const int* lens;
  void* out;
  float* part_o; float2* part_ml; int2* part_info;
  int B, Hq, Hk, rep, chunks, capacity, block_shift, window, min_units;
  float scale_log2;
};

template <int HD, int NT>
struct Slot {                            // one part of one segment: normalised output, maximum (log2), sum
  float o[8 * NT][HD];
  float m[8 * NT], l[8 * NT];
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// WORDS 32-bit words of codes from `p`, chunks of at most 16 bytes that lie `step` bytes apart; zeros when !ok.
template <int WORDS>
__device__ __forceinline__ void load_codes(uint32_t (&w)[WORDS], const uint8_t* p, int step, bool ok) {
#pragma unroll
  for (int i = 0; i < WORDS; ++i) w[i] = 0;
  if (!ok) return;
  if constexpr (WORDS == 1) {
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
  } else if constexpr (WORDS == 2) {
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3]) : "l"(p + i * step));
  }
}

__device__ __forceinline__ float load_q(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_q(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ uint32_t pack_out(float a, float b, const __nv_bfloat16*) { return pack_bf16x2(a, b); }
__device__ __forceinline__ uint32_t pack_out(float a, float b, const __half*) { return pack_half2(a, b); }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float f) { *p = __float2bfloat16(f); }
__device__ __forceinline__ void store_out(__half* p, float f) { *p = __float2half(f); }

__device__ __forceinline__ int clamp_len(int len, int capacity) { return min(max(len, 0), capacity); }
__device__ __forceinline__ int first_token(int len, int window) { return window > 0 && len > window ? len - window : 0; }

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(THREADS, NT == 1 && HD <= 128 ? 2 : 1) decode_kernel(const Params p) {
  constexpr int KS = HD / 16;            // k-steps of the first product = words of one token's codes per thread
  constexpr int VW = HD / 32;            // words of one token's values per thread
  constexpr int NH = 8 * NT;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  auto* slots = reinterpret_cast<Slot<HD, NT>*>(smem_raw);                       // [2 * WARPS]
  int* cum = reinterpret_cast<int*>(smem_raw + sizeof(Slot<HD, NT>) * 2 * WARPS);  // [B + 1] units per head
  __shared__ long long tag[2 * WARPS];
  __shared__ int scan[WARPS + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int HC = p.Hk * p.chunks;

  // units of every sequence, and their running sum
  const int per_thread = (p.B + THREADS - 1) / THREADS;
  int mine = 0;
  for (int i = 0; i < per_thread; ++i) {
    const int b = tid * per_thread + i;
    if (b < p.B) {
      const int len = clamp_len(p.lens[b], p.capacity);
      const int n = len > 0 ? (len + UNIT - 1) / UNIT - first_token(len, p.window) / UNIT : 0;
      cum[b + 1] = n;
      mine += n;
    }
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) scan[warp + 1] = incl;
  if (tid < 2 * WARPS) tag[tid] = -1;
  if (tid == 0) { scan[0] = 0; cum[0] = 0; }
  __syncthreads();
  int before = incl - mine;
  for (int w = 0; w < warp; ++w) before += scan[w + 1];
  for (int i = 0; i < per_thread; ++i) {
    const int b = tid * per_thread + i;
    if (b < p.B) { before += cum[b + 1]; cum[b + 1] = before; }
  }
  __syncthreads();

  // sequences without tokens give zeros
  for (int b = blockIdx.x; b < p.B; b += gridDim.x)
    if (cum[b + 1] == cum[b]) {
      T* o = static_cast<T*>(p.out) + (long long)b * p.Hq * HD;
      for (int i = tid; i < p.Hq * HD; i += THREADS) store_out(o + i, 0.f);
    }

  const long long total = (long long)cum[p.B] * HC;
  long long per = (total + gridDim.x - 1) / gridDim.x;
  if (per < p.min_units) per = p.min_units;
  const long long A = min(total, per * blockIdx.x), E = min(total, A + per);
  const long long per_warp = (E - A + WARPS - 1) / WARPS;
  const long long ua = min(E, A + per_warp * warp), ue = min(E, ua + per_warp);

  for (long long u = ua; u < ue;) {
    int lo = 0, hi = p.B;                // the sequence of unit u: cum[b] * HC <= u < cum[b + 1] * HC
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((long long)cum[mid] * HC <= u) lo = mid; else hi = mid;
    }
    const int b = lo, n = cum[b + 1] - cum[b];
    const long long rel = u - (long long)cum[b] * HC;
    const int hc = (int)(rel / n), u0 = (int)(rel - (long long)hc * n);
    const int u1 = (int)min((long long)n, u0 + (ue - u));
    const int hk = hc / p.chunks, chunk = hc - hk * p.chunks;
    const int len = clamp_len(p.lens[b], p.capacity), first = first_token(len, p.window);
    const int heads = min(NH, p.rep - chunk * NH), h0 = hk * p.rep + chunk * NH;

    // query heads as the B operand of the first product: k pairs of head g, dimensions as the codes are loaded
    uint32_t qf[NT][KS][2];
    float f_scale[NT][2];                // 2^x of this thread's two score columns (heads 2t, 2t + 1)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool live = nt * 8 + g < heads;
      const T* qp = static_cast<const T*>(p.q) + (long long)b * p.q_batch + (long long)(h0 + nt * 8 + (live ? g : 0)) * HD;
      float qv[KS][4];
      float amax = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = HD == 32 ? t * 8 + s * 4 : (s >> 2) * 64 + t * 16 + (s & 3) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          qv[s][e] = live ? load_q(qp + d + e) : 0.f;
          amax = fmaxf(amax, fabsf(qv[s][e]));
        }
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int ex = max((int)(__float_as_uint(amax) >> 23) - 127, -100);
      const float up = pow2(14 - ex), down = pow2(ex - 14) * p.scale_log2;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        qf[nt][s][0] = pack_half2(qv[s][0] * up, qv[s][1] * up);
        qf[nt][s][1] = pack_half2(qv[s][2] * up, qv[s][3] * up);
      }
      f_scale[nt][0] = __shfl_sync(0xffffffffu, down, 2 * t * 4);
      f_scale[nt][1] = __shfl_sync(0xffffffffu, down, (2 * t + 1) * 4);
    }

    float acc[NT][KS][4];
    float m[NT][2], l[NT][2], r = 0.f, inv_r = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) acc[nt][j][0] = acc[nt][j][1] = acc[nt][j][2] = acc[nt][j][3] = 0.f;
    }
    const uint8_t* kb = p.k + (long long)b * p.batch + (long long)hk * p.head + t * (HD >= 64 ? 16 : 8);
    const uint8_t* vb = p.v + (long long)b * p.batch + (long long)hk * p.head + g * (VW >= 4 ? 16 : VW * 4);
    const float* ks_p = p.k_scale + (long long)b * p.scale_batch + (long long)hk * p.scale_head;
    const float* vs_p = p.v_scale + (long long)b * p.scale_batch + (long long)hk * p.scale_head;
    const int unit0 = first / UNIT;

    for (int un = u0; un < u1; ++un) {
      const int tk = (unit0 + un) * UNIT;
      const bool whole = tk >= first && tk + UNIT <= len;
      auto seen = [&](int row) { return whole || (tk + row >= first && tk + row < len); };
      uint32_t ka[KS], kc[KS], va[4][VW];
      load_codes(ka, kb + (long long)(tk + g) * p.tok, 64, seen(g));
      load_codes(kc, kb + (long long)(tk + g + 8) * p.tok, 64, seen(g + 8));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 2 * t + (i & 1) + (i >> 1) * 8;
        load_codes(va[i], vb + (long long)(tk + row) * p.tok, 128, seen(row));
      }
      const float ks = ks_p[tk >> p.block_shift], vs = vs_p[tk >> p.block_shift];

      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const uint32_t a0 = to_half2(ka[i]), a1 = to_half2(kc[i]), a2 = to_half2_hi(ka[i]), a3 = to_half2_hi(kc[i]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma(s[nt], a0, a1, a2, a3, qf[nt][i][0], qf[nt][i][1]);
      }
      // raise the value reference if this block's scale is larger
      float drop = 1.f;
      if (vs > r) {
        drop = r * inverse_pow2(vs);
        r = vs;
        inv_r = inverse_pow2(vs);
      }
      const float w = vs * inv_r * 32768.f;
      uint32_t pf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float f0 = f_scale[nt][0] * ks, f1 = f_scale[nt][1] * ks;
        float x[4] = {s[nt][0] * f0, s[nt][1] * f1, s[nt][2] * f0, s[nt][3] * f1};
        if (!whole) {
          if (!seen(g)) x[0] = x[1] = -INFINITY;
          if (!seen(g + 8)) x[2] = x[3] = -INFINITY;
        }
        float m0 = fmaxf(x[0], x[2]), m1 = fmaxf(x[1], x[3]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
          m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
        }
        m0 = fmaxf(m0, m[nt][0]);
        m1 = fmaxf(m1, m[nt][1]);
        const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
        const float a0 = exp2_fast(m[nt][0] - b0), a1 = exp2_fast(m[nt][1] - b1);
        m[nt][0] = m0;
        m[nt][1] = m1;
        const float p0 = exp2_fast(x[0] - b0), p1 = exp2_fast(x[1] - b1), p2 = exp2_fast(x[2] - b0), p3 = exp2_fast(x[3] - b1);
        l[nt][0] = l[nt][0] * a0 + p0 + p2;
        l[nt][1] = l[nt][1] * a1 + p1 + p3;
        pf[nt][0] = transpose8(pack_half2(p0 * w, p1 * w));
        pf[nt][1] = transpose8(pack_half2(p2 * w, p3 * w));
        const float d0 = a0 * drop, d1 = a1 * drop;
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          acc[nt][j][0] *= d0; acc[nt][j][1] *= d1; acc[nt][j][2] *= d0; acc[nt][j][3] *= d1;
        }
      }
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        const uint32_t ab0 = __byte_perm(va[0][i], va[1][i], 0x5140), ab1 = __byte_perm(va[0][i], va[1][i], 0x7362);
        const uint32_t cd0 = __byte_perm(va[2][i], va[3][i], 0x5140), cd1 = __byte_perm(va[2][i], va[3][i], 0x7362);
        const uint32_t a0 = to_half2(ab0), a1 = to_half2_hi(ab0), a2 = to_half2(cd0), a3 = to_half2_hi(cd0);
        const uint32_t e0 = to_half2(ab1), e1 = to_half2_hi(ab1), e2 = to_half2(cd1), e3 = to_half2_hi(cd1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma(acc[nt][2 * i], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
          mma(acc[nt][2 * i + 1], e0, e1, e2, e3, pf[nt][0], pf[nt][1]);
        }
      }
    }

    // this warp's part of the segment: the whole of it is written out, a piece goes to shared memory
    const bool complete = u0 == 0 && u1 == n;
    const int slot = warp * 2 + (u0 == 0);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[nt][c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const int h = nt * 8 + 2 * t + c;
        const float inv = sum == 0.f ? 0.f : 1.f / sum * (1.f / 32768.f);
        if (complete) {
          if (h < heads) {
            T* o = static_cast<T*>(p.out) + ((long long)b * p.Hq + h0 + h) * HD;
#pragma unroll
            for (int i = 0; i < VW; ++i) {
              // words 4 and up of a 256-wide head lie 128 dimensions on
              const int d = (i >> 2) * 128 + g * (VW >= 4 ? 16 : VW * 4) + (i & 3) * 4;
              uint2 pk;
              pk.x = pack_out(acc[nt][2 * i][c] * inv * r, acc[nt][2 * i][c + 2] * inv * r, o);
              pk.y = pack_out(acc[nt][2 * i + 1][c] * inv * r, acc[nt][2 * i + 1][c + 2] * inv * r, o);
              *reinterpret_cast<uint2*>(o + d) = pk;
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < VW; ++i) {
            const int d = (i >> 2) * 128 + g * (VW >= 4 ? 16 : VW * 4) + (i & 3) * 4;
            *reinterpret_cast<float4*>(&slots[slot].o[h][d]) =
                make_float4(acc[nt][2 * i][c] * inv * r, acc[nt][2 * i][c + 2] * inv * r, acc[nt][2 * i + 1][c] * inv * r,
                            acc[nt][2 * i + 1][c + 2] * inv * r);
          }
          if (g == 0) { slots[slot].m[h] = m[nt][c]; slots[slot].l[h] = sum; }
        }
      }
    if (!complete && lane == 0) tag[slot] = (long long)b * HC + hc;
    u += u1 - u0;
  }
  __syncthreads();

  // join the parts of each segment inside the CTA; parts of one segment lie in neighbouring slots
  int2 info[2] = {make_int2(-1, 0), make_int2(-1, 0)};
  for (int i = 0; i < 2 * WARPS;) {
    const long long seg = tag[i];
    if (seg < 0) { ++i; continue; }
    int end = i + 1;
    while (end < 2 * WARPS && (tag[end] == seg || tag[end] < 0)) ++end;
    const int b = (int)(seg / HC), hc = (int)(seg - (long long)b * HC);
    const int hk = hc / p.chunks, chunk = hc - hk * p.chunks;
    const int n = cum[b + 1] - cum[b];
    const long long s0 = (long long)cum[b] * HC + (long long)hc * n, s1 = s0 + n;
    const bool complete = s0 >= A && s1 <= E;
    const int heads = min(NH, p.rep - chunk * NH), h0 = hk * p.rep + chunk * NH;
    const int which = s0 >= A;           // 1: the segment starts in this CTA
    const long long part = (long long)blockIdx.x * 2 + which;
    for (int e = tid; e < NH * HD; e += THREADS) {
      const int h = e / HD, d = e - h * HD;
      float top = -INFINITY;
      for (int j = i; j < end; ++j) if (tag[j] == seg) top = fmaxf(top, slots[j].m[h]);
      float num = 0.f, den = 0.f;
      for (int j = i; j < end; ++j)
        if (tag[j] == seg && slots[j].l[h] != 0.f) {
          const float wgt = exp2_fast(slots[j].m[h] - top) * slots[j].l[h];
          num += wgt * slots[j].o[h][d];
          den += wgt;
        }
      const float o = den == 0.f ? 0.f : num / den;
      if (complete) {
        if (h < heads) store_out(static_cast<T*>(p.out) + ((long long)b * p.Hq + h0 + h) * HD + d, o);
      } else {
        p.part_o[part * NH * HD + e] = o;
        if (d == 0) p.part_ml[part * NH + h] = make_float2(top, den);
      }
    }
    if (!complete) info[which] = make_int2((int)seg, which ? (int)((s1 - 1) / per) - (int)blockIdx.x : 0);
    i = end;
  }
  if (tid == 0) {
    p.part_info[2 * blockIdx.x] = info[0];
    p.part_info[2 * blockIdx.x + 1] = info[1];
  }
}

// Joins the parts of a segment that starts in CTA blockIdx.x and goes on in the CTAs behind it; one head per CTA here.
template <int HD, int NH, typename T>
__global__ void __launch_bounds__(COMBINE_GROUPS * 32) combine_kernel(const Params p) {
  constexpr int PER = HD / 32;
  __shared__ float so[COMBINE_GROUPS][HD];
  __shared__ float sm[COMBINE_GROUPS], sl[COMBINE_GROUPS];
  const int2 info = p.part_info[2 * blockIdx.x + 1];
  if (info.x < 0) return;
  const int HC = p.Hk * p.chunks;
  const int b = info.x / HC, hc = info.x - b * HC, hk = hc / p.chunks, chunk = hc - hk * p.chunks;
  const int h = blockIdx.y;
  if (chunk * NH + h >= p.rep) return;
  const int grp = threadIdx.x >> 5, lane = threadIdx.x & 31, count = info.y + 1;
  auto part_of = [&](int i) { return ((long long)blockIdx.x + i) * 2 + (i == 0); };
  float top = -INFINITY;
  for (int i = grp; i < count; i += COMBINE_GROUPS) top = fmaxf(top, p.part_ml[part_of(i) * NH + h].x);
  float acc[PER] = {}, den = 0.f;
#pragma unroll 4
  for (int i = grp; i < count; i += COMBINE_GROUPS) {
    const float2 ml = p.part_ml[part_of(i) * NH + h];
    const float* o = p.part_o + (part_of(i) * NH + h) * HD + lane;
    const float wgt = ml.y == 0.f ? 0.f : exp2_fast(ml.x - top) * ml.y;
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] += wgt * o[e * 32];
    den += wgt;
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) so[grp][e * 32 + lane] = acc[e];
  if (lane == 0) { sm[grp] = top; sl[grp] = den; }
  __syncthreads();
  for (int d = threadIdx.x; d < HD; d += COMBINE_GROUPS * 32) {
    float mx = -INFINITY, num = 0.f, sum = 0.f;
    for (int i = 0; i < COMBINE_GROUPS; ++i) mx = fmaxf(mx, sm[i]);
    for (int i = 0; i < COMBINE_GROUPS; ++i)
      if (sl[i] != 0.f) {
        const float wgt = exp2_fast(sm[i] - mx);
        num += wgt * so[i][d];
        sum += wgt * sl[i];
      }
    store_out(static_cast<T*>(p.out) + ((long long)b * p.Hq + hk * p.rep + chunk * NH + h) * HD + d, sum == 0.f ? 0.f : num / sum);
  }
}

template <int HD, int NT, typename T>
static int launch(const Params& p, int grid, cudaStream_t stream) {
  const size_t smem = sizeof(Slot<HD, NT>) * 2 * WARPS + sizeof(int) * (p.B + 1);
  auto kern = decode_kernel<HD, NT, T>;
  OB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kern<<<grid, THREADS, smem, stream>>>(p);
  OB_CUDA_CHECK(cudaGetLastError());
  combine_kernel<HD, 8 * NT, T><<<dim3(grid, min(8 * NT, p.rep)), COMBINE_GROUPS * 32, 0, stream>>>(p);
  return (int)cudaGetLastError();
}

// Two groups of 8 query heads per pass over the codes where the accumulators of both fit beside them.
static int groups(int rep, int hd) { return rep > 8 && hd <= 128 ? 2 : 1; }

template <typename T>
static int dispatch(const Params& p, int hd, int nt, int grid, cudaStream_t stream) {
  if (hd == 32) return nt == 1 ? launch<32, 1, T>(p, grid, stream) : launch<32, 2, T>(p, grid, stream);
  if (hd == 64) return nt == 1 ? launch<64, 1, T>(p, grid, stream) : launch<64, 2, T>(p, grid, stream);
  if (hd == 128) return nt == 1 ? launch<128, 1, T>(p, grid, stream) : launch<128, 2, T>(p, grid, stream);
  return launch<256, 1, T>(p, grid, stream);
}

// CTAs of a launch: two per SM, or one where the accumulators of a warp leave room for no more; fewer when the
// batch cannot hold that many runs of MIN_UNITS units.
constexpr int MIN_UNITS = 8;
static int grid_size(int B, int Hk, int rep, int hd, int capacity) {
  const int nt = groups(rep, hd), chunks = (rep + 8 * nt - 1) / (8 * nt);
  const long long most = (long long)B * Hk * chunks * ((capacity + UNIT - 1) / UNIT + 1);
  const long long want = (most + MIN_UNITS - 1) / MIN_UNITS, fit = nt == 1 && hd <= 128 ? 296 : 148;
  return (int)(want < fit ? want : fit);
}

}  // namespace decode_fp8
}  // namespace ob

using namespace ob::decode_fp8;

// Bytes of workspace that ob_attn_decode_fp8 needs for these sizes; < 0 for sizes it does not take.
extern "C" long long ob_attn_decode_fp8_workspace(int B, int Hq, int Hk, int hd, int capacity) {
  if (B <= 0 || Hk <= 0 || Hq <= 0 || Hq % Hk || hd < 32 || hd > 256 || (hd & (hd - 1)) || capacity <= 0) return -1;
  const int rep = Hq / Hk, nh = 8 * groups(rep, hd);
  const long long grid = grid_size(B < MAX_BATCH ? B : MAX_BATCH, Hk, rep, hd, capacity);
  return grid * 2 * ((long long)nh * hd * 4 + nh * 8 + 8);
}

// q_dtype: 0 = bf16, 1 = fp16 (also of k_new, v_new and out).  k_new / v_new may be null when the cache already holds
// the current token.  Strides of q, new rows and scales in elements, of the cache in bytes.
extern "C" int ob_attn_decode_fp8(const void* q, long long q_batch, int q_dtype, const void* k_new, const void* v_new,
                                  long long new_batch, long long new_head, void* k, void* v, long long batch, long long tok,
                                  long long head, void* k_scale, void* v_scale, long long scale_batch, long long scale_head,
                                  const void* lens, void* out, void* workspace, int B, int Hq, int Hk, int hd, int capacity,
                                  int block, float scale, int window, void* status, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (Hk <= 0 || Hq <= 0 || Hq % Hk || hd < 32 || hd > 256 || (hd & (hd - 1)) || capacity <= 0 || window < 0) return -1;
  if (block < 16 || block > 128 || (block & (block - 1)) || q_dtype < 0 || q_dtype > 1) return -1;
  if ((batch | tok | head) % 16) return -2;
  if (k_new) {
    const int rc = launch_append({k_new, v_new, new_batch, 0, new_head, k, v, batch, tok, head, (float*)k_scale,
                                  (float*)v_scale, scale_batch, scale_head, (const int*)lens, nullptr, (int*)status, B, 1,
                                  Hk, hd, capacity, block, 0, 0, 0}, q_dtype, stream);
    if (rc) return rc;
  }
  const int rep = Hq / Hk, nt = groups(rep, hd), nh = 8 * nt;
  int shift = 4;
  while ((1 << shift) < block) ++shift;
  for (int b0 = 0; b0 < B; b0 += MAX_BATCH) {
    const int nb = B - b0 < MAX_BATCH ? B - b0 : MAX_BATCH;
    const int grid = grid_size(nb, Hk, rep, hd, capacity);
    Params p;
    p.q = (const uint16_t*)q + (long long)b0 * q_batch; p.q_batch = q_batch;
    p.k = (const uint8_t*)k + (long long)b0 * batch; p.v = (const uint8_t*)v + (long long)b0 * batch;
    p.batch = batch; p.tok = tok; p.head = head;
    p.k_scale = (const float*)k_scale + (long long)b0 * scale_batch;
    p.v_scale = (const float*)v_scale + (long long)b0 * scale_batch;
    p.scale_batch = scale_batch; p.scale_head = scale_head;
    p.lens = (const int*)lens + b0;
    p.out = (uint16_t*)out + (long long)b0 * Hq * hd;
    p.part_o = (float*)workspace;
    p.part_ml = (float2*)(p.part_o + (long long)grid * 2 * nh * hd);
    p.part_info = (int2*)(p.part_ml + (long long)grid * 2 * nh);
    p.B = nb; p.Hq = Hq; p.Hk = Hk; p.rep = rep; p.chunks = (rep + nh - 1) / nh; p.capacity = capacity;
    p.block_shift = shift; p.window = window; p.min_units = MIN_UNITS;
    p.scale_log2 = scale * 1.4426950408889634f;
    const int rc = q_dtype == 0 ? dispatch<__nv_bfloat16>(p, hd, nt, grid, stream) : dispatch<__half>(p, hd, nt, grid, stream);
    if (rc) return rc;
  }
  return 0;
}
