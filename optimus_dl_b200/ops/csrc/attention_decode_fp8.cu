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
// * The products run transposed, S^T = K Q^T and O^T = V^T P^T, on 16 x 8 x 16 tensor-core tiles (mma.sync: a tile is
//   far too small for tcgen05): tokens are the M side of the first product and head dimensions that of the second, the
//   up to 8 query heads that share a kv head are the N side of both, so no row of a tile is padding.  The K side of
//   either product may be permuted freely, so each thread takes 16 contiguous bytes as they come: for K as consecutive k
//   pairs of one token, for V as the same 16 dimensions of four tokens, whose bytes are interleaved with byte permutes.
//   e4m3 to f16 is one exact conversion for two codes; P gets from the accumulator layout of the first product to the
//   operand layout of the second with one 8 x 8 transpose (movmatrix) for 8 tokens.
// * So every thread consumes exactly the bytes it asked for, and codes go straight from global memory to registers with
//   16-byte loads. The keys of the next unit of 16 tokens are loaded behind the first product of the current one, the
//   values behind its second; 16 warps on an SM with 2 to 4 KB each under way cover the latency (4 sequences of up to
//   131072 tokens, 40 / 8 heads of 128: 116 us for 671 MB, 0.89 of the measured copy bandwidth). The same bytes through
//   a two-stage cp.async ring in shared memory took 168 us: its reads add a second latency to every unit's chain.
// * q is scaled by a power of two per head so that its largest element lies in [2^14, 2^15): f16 then holds a bf16 or
//   fp16 q exactly down to 2^-28 of that.  The softmax runs against a reference that follows the maximum only when a
//   score exceeds it by more than 2^8, so most units need no reduction across lanes and no rescaling.  Probabilities
//   are held as p s_v 2^7 in f16 against a reference of their own, which follows the largest p s_v of the head in the same
//   way: at most 2^15, normal down to 2^-21 of the reference and nothing below 2^-32.  (Against the largest s_v alone, a
//   block with 2^31 times the scale of the others hid them even where its own p was nothing.)  Scores, references, sums
//   and both accumulators are fp32.
// * Work is cut evenly, not by sequence: units of 16 tokens of one (sequence, kv head, group of query heads) are
//   numbered through the batch, every CTA takes an equal run of them and every warp an equal part of that.  A warp
//   that sees all units of a segment writes its output; parts are joined first inside the CTA through shared memory
//   (at most two per warp) and then, at most two per CTA, by a second kernel.  A ragged batch or a single long
//   sequence therefore keeps every SM busy to the end, and the workspace does not depend on the batch.
// * The three launches of a step (append, attention, join) overlap: each starts while the one before it drains and
//   waits for its results only where it reads them (programmatic dependent launch).
#include "kv_fp8.cuh"
#include <atomic>
#include <string.h>

namespace ob {
namespace decode_fp8 {

using namespace kvfp8;

constexpr int WARPS = 8;
// CTAs per SM, as many as the registers of a warp's accumulators allow; at HD 64 one more, whose 80 registers spill 48
// bytes (60 loaded again) and which is faster all the same.  Measured at HD 128, 4 sequences of up to 131072 tokens:
// 2 x 8 warps 121 us, 1 x 12 129 us, 2 x 6 130 us; at HD 64, 128 of up to 1024: 3 x 8 36 us, 2 x 8 39 us.
template <int HD, int NT> constexpr int CTAS = NT > 1 || HD > 128 ? 1 : HD > 64 ? 2 : 3;
constexpr int THREADS = WARPS * 32;
constexpr int UNIT = 16;                 // tokens
constexpr int MAX_BATCH = 2048;          // sequences per launch (their lengths are held in shared memory)
constexpr float LAZY = 8.f;              // log2 of how far a score may exceed the reference
constexpr float P_SCALE = 7.f;           // log2 of what p s_v is held times: up to 2^8 it stays below 2^15 in f16
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
  int B, Hq, Hk, rep, chunks, capacity, block_shift, window, min_units, appended;
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
__device__ __forceinline__ float log2_fast(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
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

// WORDS 32-bit words of codes from `p`, in chunks of at most 16 bytes that lie `step` bytes apart.
template <int WORDS>
__device__ __forceinline__ void load_codes(uint32_t (&w)[WORDS], const uint8_t* p, int step) {
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
template <int WORDS>
__device__ __forceinline__ void load_codes_if(uint32_t (&w)[WORDS], const uint8_t* p, int step, bool ok) {
  if (ok) {
    load_codes(w, p, step);
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
  }
}
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_launch_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ float2 unpack_q(uint32_t u, const __nv_bfloat16*) { return unpack_bf16x2(u); }
__device__ __forceinline__ float2 unpack_q(uint32_t u, const __half*) { return half2_to_float2(u); }
__device__ __forceinline__ uint32_t pack_out(float a, float b, const __nv_bfloat16*) { return pack_bf16x2(a, b); }
__device__ __forceinline__ uint32_t pack_out(float a, float b, const __half*) { return pack_half2(a, b); }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float f) { *p = __float2bfloat16(f); }
__device__ __forceinline__ void store_out(__half* p, float f) { *p = __float2half(f); }

// PER consecutive numbers of one lane
template <int PER>
__device__ __forceinline__ void read_floats(float (&x)[PER], const float* p) {
  if constexpr (PER == 1) {
    x[0] = *p;
  } else if constexpr (PER == 2) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    x[0] = v.x; x[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + i);
      x[i] = v.x; x[i + 1] = v.y; x[i + 2] = v.z; x[i + 3] = v.w;
    }
  }
}
template <int PER>
__device__ __forceinline__ void write_floats(float* p, const float (&x)[PER]) {
  if constexpr (PER == 1) {
    *p = x[0];
  } else if constexpr (PER == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(x[0], x[1]);
  } else {
#pragma unroll
    for (int i = 0; i < PER; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  }
}
template <int PER, typename T>
__device__ __forceinline__ void write_out(T* p, const float (&x)[PER]) {
  if constexpr (PER == 1) {
    store_out(p, x[0]);
  } else {
#pragma unroll
    for (int i = 0; i < PER; i += 2) reinterpret_cast<uint32_t*>(p)[i / 2] = pack_out(x[i], x[i + 1], p);
  }
}

// a / b; 32 bits wide where that is enough, which is several times faster
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return (a | b) >> 31 ? a / b : (long long)((unsigned)a / (unsigned)b);
}
__device__ __forceinline__ int clamp_len(int len, int capacity) { return min(max(len, 0), capacity); }
__device__ __forceinline__ int first_token(int len, int window) { return window > 0 && len > window ? len - window : 0; }

template <int HD, int NT, typename T>
__global__ void __launch_bounds__(THREADS, CTAS<HD, NT>) decode_kernel(const __grid_constant__ Params p) {
  constexpr int KS = HD / 16;            // k-steps of the first product = words of one token's codes per thread
  constexpr int VW = HD / 32;            // words of one token's values per thread
  constexpr int NH = 8 * NT;
  constexpr int KCB = HD >= 64 ? 16 : 8, VCB = HD >= 128 ? 16 : HD / 8;      // bytes of a thread's key / value chunks
  extern __shared__ __align__(16) uint8_t smem_raw[];
  auto* slots = reinterpret_cast<Slot<HD, NT>*>(smem_raw);               // [2 * WARPS]: entered in the middle, left unfinished
  int* cum = reinterpret_cast<int*>(slots + 2 * WARPS);                  // [B + 1] units per head, summed up
  int* lens = cum + p.B + 1;                                             // [B]
  __shared__ int tag[2 * WARPS];         // the slots' segments, -1 = empty
  __shared__ int2 where[2 * WARPS], crossing[2];
  __shared__ int scan[WARPS + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int HC = p.Hk * p.chunks;
  let_next_launch_start();

  // units of every sequence, and their running sum
  const int per_thread = (p.B + THREADS - 1) / THREADS;
  int mine = 0;
  for (int i = 0; i < per_thread; ++i) {
    const int b = tid * per_thread + i;
    if (b < p.B) {
      const int len = clamp_len(p.lens[b], p.capacity);
      const int n = len > 0 ? (len + UNIT - 1) / UNIT - first_token(len, p.window) / UNIT : 0;
      lens[b] = len;
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
  if (tid < 2) crossing[tid] = make_int2(-1, 0);
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
  long long per = quotient(total + gridDim.x - 1, gridDim.x);
  if (per < p.min_units) per = p.min_units;
  const long long A = min(total, per * blockIdx.x), E = min(total, A + per);
  const long long per_warp = (E - A + WARPS - 1) / WARPS;
  const long long ua = min(E, A + per_warp * warp);
  const int count = (int)(min(E, ua + per_warp) - ua);      // units of this warp

  // the segment and position of the first unit: cum[b] * HC <= ua < cum[b + 1] * HC
  int b = 0, hc = 0, un = 0;
  if (count > 0) {
    for (int span = p.B; span > 1;) {    // 32 places a round
      const int step = (span + 31) >> 5, at = lane * step;
      const bool below = at < span && (long long)cum[b + at] * HC <= ua;
      const int skip = (__popc(__ballot_sync(0xffffffffu, below)) - 1) * step;
      b += skip;
      span = min(step, span - skip);
    }
    const long long rel = ua - (long long)cum[b] * HC;
    const int n = cum[b + 1] - cum[b];
    hc = (int)quotient(rel, n);
    un = (int)(rel - (long long)hc * n);
  }

  if (p.appended) wait_for_launch_before();      // codes and scales of the new token
  for (int done = 0; done < count;) {
    const int n = cum[b + 1] - cum[b], u0 = un, u1 = min(n, un + count - done);
    const int hk = p.chunks == 1 ? hc : hc / p.chunks, chunk = hc - hk * p.chunks;
    const int len = lens[b], first = first_token(len, p.window), unit0 = first / UNIT;
    const int heads = min(NH, p.rep - chunk * NH), h0 = hk * p.rep + chunk * NH;

    const long long tok = p.tok;
    const uint8_t *kp, *vp;
    {
      const long long base = (long long)b * p.batch + (long long)hk * p.head, tk = (long long)(unit0 + un) * UNIT;
      kp = p.k + base + (tk + g) * tok + t * KCB;
      vp = p.v + base + (tk + 2 * t) * tok + g * VCB;
    }
    const long long srow = (long long)b * p.scale_batch + (long long)hk * p.scale_head;
    const float *ks_p = p.k_scale + srow, *vs_p = p.v_scale + srow;
    uint32_t ka[KS], kc[KS], va[4][VW];
    float ks, vs;
    auto fetch_k = [&](int unit) {
      const int tk = (unit0 + unit) * UNIT;
      if (tk >= first && tk + UNIT <= len) {
        load_codes(ka, kp, 64);
        load_codes(kc, kp + 8 * tok, 64);
      } else {
        load_codes_if(ka, kp, 64, tk + g >= first && tk + g < len);
        load_codes_if(kc, kp + 8 * tok, 64, tk + g + 8 >= first && tk + g + 8 < len);
      }
      ks = ks_p[tk >> p.block_shift];
      kp += UNIT * tok;
    };
    auto fetch_v = [&](int unit) {
      const int tk = (unit0 + unit) * UNIT, row = tk + 2 * t;
      if (tk >= first && tk + UNIT <= len) {
        load_codes(va[0], vp, 128);
        load_codes(va[1], vp + tok, 128);
        load_codes(va[2], vp + 8 * tok, 128);
        load_codes(va[3], vp + 9 * tok, 128);
      } else {
        load_codes_if(va[0], vp, 128, row >= first && row < len);
        load_codes_if(va[1], vp + tok, 128, row + 1 >= first && row + 1 < len);
        load_codes_if(va[2], vp + 8 * tok, 128, row + 8 >= first && row + 8 < len);
        load_codes_if(va[3], vp + 9 * tok, 128, row + 9 >= first && row + 9 < len);
      }
      vs = vs_p[tk >> p.block_shift];
      vp += UNIT * tok;
    };
    fetch_k(un);
    fetch_v(un);

    // query heads as the B operand of the first product: k pairs of head g, dimensions as the codes are loaded
    uint32_t qf[NT][KS][2];
    float f_scale[NT][2];                // 2^x of this thread's two score columns (heads 2t, 2t + 1)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const bool live = nt * 8 + g < heads;
      const T* qp = static_cast<const T*>(p.q) + (long long)b * p.q_batch + (long long)(h0 + nt * 8 + (live ? g : 0)) * HD;
      uint2 raw[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = HD == 32 ? t * 8 + s * 4 : (s >> 2) * 64 + t * 16 + (s & 3) * 4;
        raw[s] = live ? *reinterpret_cast<const uint2*>(qp + d) : make_uint2(0, 0);
      }
      float amax = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const float2 x = unpack_q(raw[s].x, qp), y = unpack_q(raw[s].y, qp);
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int ex = max((int)(__float_as_uint(amax) >> 23) - 127, -100);
      const float up = pow2(14 - ex), down = pow2(ex - 14) * p.scale_log2;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const float2 x = unpack_q(raw[s].x, qp), y = unpack_q(raw[s].y, qp);
        qf[nt][s][0] = pack_half2(x.x * up, x.y * up);
        qf[nt][s][1] = pack_half2(y.x * up, y.y * up);
      }
      f_scale[nt][0] = __shfl_sync(0xffffffffu, down, 2 * t * 4);
      f_scale[nt][1] = __shfl_sync(0xffffffffu, down, (2 * t + 1) * 4);
    }

    float acc[NT][KS][4];
    float m[NT][2], l[NT][2], r[NT][2];        // reference of p (log2), sums of p, reference of p s_v 2^-7
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = r[nt][0] = r[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) acc[nt][j][0] = acc[nt][j][1] = acc[nt][j][2] = acc[nt][j][3] = 0.f;
    }

    for (; un < u1; ++un) {
      const int tk = (unit0 + un) * UNIT;
      const bool whole = tk >= first && tk + UNIT <= len;

      float s[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const uint32_t a0 = to_half2(ka[i]), a1 = to_half2(kc[i]), a2 = to_half2_hi(ka[i]), a3 = to_half2_hi(kc[i]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma(s[nt], a0, a1, a2, a3, qf[nt][i][0], qf[nt][i][1]);
      }
      const float ks_now = ks, vs_now = vs;
      if (un + 1 < u1) fetch_k(un + 1);
      // scores in log2 units; the references move only if one exceeds them by more than LAZY
      const float lift = max_nan(log2_fast(vs_now), -127.f);       // of the value scale; NaN where that is none
      bool high = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float f0 = f_scale[nt][0] * ks_now, f1 = f_scale[nt][1] * ks_now;
        s[nt][0] *= f0; s[nt][1] *= f1; s[nt][2] *= f0; s[nt][3] *= f1;
        if (!whole) {
          if (tk + g < first || tk + g >= len) s[nt][0] = s[nt][1] = -INFINITY;
          if (tk + g + 8 < first || tk + g + 8 >= len) s[nt][2] = s[nt][3] = -INFINITY;
        }
        high |= fmaxf(s[nt][0], s[nt][2]) - m[nt][0] > fminf(LAZY, r[nt][0] - (lift - P_SCALE - LAZY)) ||
                fmaxf(s[nt][1], s[nt][3]) - m[nt][1] > fminf(LAZY, r[nt][1] - (lift - P_SCALE - LAZY));
      }
      if (__any_sync(0xffffffffu, high)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float m0 = fmaxf(s[nt][0], s[nt][2]), m1 = fmaxf(s[nt][1], s[nt][3]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o));
            m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
          }
          const float n0 = fmaxf(m0, m[nt][0]), n1 = fmaxf(m1, m[nt][1]);
          // both references are -inf only while every score was -inf: nothing to scale then
          const float e0 = n0 == m[nt][0] ? 0.f : m[nt][0] - n0, e1 = n1 == m[nt][1] ? 0.f : m[nt][1] - n1;
          const float was0 = r[nt][0] + e0, was1 = r[nt][1] + e1;
          const float r0 = fmaxf(was0, m0 - n0 + (lift - P_SCALE)), r1 = fmaxf(was1, m1 - n1 + (lift - P_SCALE));
          const float d0 = r0 == was0 ? 1.f : exp2_fast(was0 - r0), d1 = r1 == was1 ? 1.f : exp2_fast(was1 - r1);
          l[nt][0] *= exp2_fast(e0);
          l[nt][1] *= exp2_fast(e1);
          m[nt][0] = n0;
          m[nt][1] = n1;
          r[nt][0] = r0;
          r[nt][1] = r1;
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            acc[nt][j][0] *= d0; acc[nt][j][1] *= d1; acc[nt][j][2] *= d0; acc[nt][j][3] *= d1;
          }
        }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float b0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], b1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
        const float p0 = exp2_fast(s[nt][0] - b0), p1 = exp2_fast(s[nt][1] - b1);
        const float p2 = exp2_fast(s[nt][2] - b0), p3 = exp2_fast(s[nt][3] - b1);
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        // s_v 2^7 against the second reference; as a number even where p is 0
        const float w0 = exp2_fast(min_nan(lift - r[nt][0], 120.f));
        const float w1 = exp2_fast(min_nan(lift - r[nt][1], 120.f));
        pf[nt][0] = transpose8(pack_half2(p0 * w0, p1 * w1));
        pf[nt][1] = transpose8(pack_half2(p2 * w0, p3 * w1));
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
      if (un + 1 < u1) fetch_v(un + 1);
    }

    // this warp's part of the segment: the whole of it is written out, a piece goes to shared memory
    const bool complete = u0 == 0 && u1 == n;
    const int which = u0 == 0;
    Slot<HD, NT>& part = slots[2 * warp + which];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[nt][c];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const int h = nt * 8 + 2 * t + c;
        const float inv = sum == 0.f ? 0.f : 1.f / sum, back = exp2_fast(r[nt][c]);
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          // words 4 and up of a 256-wide head lie 128 dimensions on
          const int d = (i >> 2) * 128 + g * VCB + (i & 3) * 4;
          const float x0 = acc[nt][2 * i][c] * inv * back, x1 = acc[nt][2 * i][c + 2] * inv * back;
          const float x2 = acc[nt][2 * i + 1][c] * inv * back, x3 = acc[nt][2 * i + 1][c + 2] * inv * back;
          if (!complete) {
            *reinterpret_cast<float4*>(&part.o[h][d]) = make_float4(x0, x1, x2, x3);
          } else if (h < heads) {
            T* o = static_cast<T*>(p.out) + ((long long)b * p.Hq + h0 + h) * HD + d;
            *reinterpret_cast<uint2*>(o) = make_uint2(pack_out(x0, x1, o), pack_out(x2, x3, o));
          }
        }
        if (!complete && g == 0) { part.m[h] = m[nt][c]; part.l[h] = sum; }
      }
    if (!complete && lane == 0) {
      // where the segment lies: its units are [s0, s1)
      const long long s0 = ua + done - u0, s1 = s0 + n;
      const bool starts = s0 >= A, inside = starts && s1 <= E;
      tag[2 * warp + which] = b * HC + hc;
      where[2 * warp + which] = make_int2(b * p.Hq + h0, heads | inside << 8 | starts << 9);
      // joined in this CTA for good, or with the CTAs behind that hold units up to s1
      if (!inside) crossing[starts] = make_int2(b * HC + hc, starts ? (int)quotient(s1 - 1, per) - (int)blockIdx.x : 0);
    }
    done += u1 - u0;
    if (done < count) {
      un = 0;
      if (++hc == HC) {
        hc = 0;
        do ++b; while (cum[b + 1] == cum[b]);
      }
    }
  }
  __syncthreads();

  // Join the parts of each segment inside the CTA, a warp for each segment and head: lane j holds the reference and sum
  // of slot j, every lane HD / 32 dimensions.
  constexpr int PER = HD / 32;
  static_assert(2 * WARPS <= 32, "one lane per slot");
  const int my_tag = lane < 2 * WARPS ? tag[lane] : -1;
  const int2 my_where = lane < 2 * WARPS ? where[lane] : make_int2(0, 0);
  int turn = warp;                       // this warp takes every WARPS-th (segment, head)
  for (unsigned todo = __ballot_sync(0xffffffffu, my_tag >= 0); todo;) {
    const int leader = __ffs(todo) - 1, seg = __shfl_sync(0xffffffffu, my_tag, leader);
    const unsigned members = __ballot_sync(0xffffffffu, my_tag == seg);
    todo &= ~members;
    const int out_row = __shfl_sync(0xffffffffu, my_where.x, leader), bits = __shfl_sync(0xffffffffu, my_where.y, leader);
    const int live = bits & 0xff;
    const long long part = (long long)blockIdx.x * 2 + (bits >> 9);
    int h = turn;
    for (; h < live; h += WARPS) {
      const float ref = my_tag == seg ? slots[lane].m[h] : -INFINITY, sum = my_tag == seg ? slots[lane].l[h] : 0.f;
      const float top = warp_max(ref);
      const float wgt = sum == 0.f ? 0.f : exp2_fast(ref - top) * sum;
      const float den = warp_sum(wgt), inv = den == 0.f ? 0.f : 1.f / den;
      float o[PER] = {};
      for (unsigned from = members; from; from &= from - 1) {
        const int j = __ffs(from) - 1;
        const float w = __shfl_sync(0xffffffffu, wgt, j);
        float x[PER];
        read_floats(x, &slots[j].o[h][lane * PER]);
        if (w != 0.f)
#pragma unroll
          for (int e = 0; e < PER; ++e) o[e] += w * x[e];
      }
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] *= inv;
      if (bits >> 8 & 1) {
        write_out(static_cast<T*>(p.out) + (long long)(out_row + h) * HD + lane * PER, o);
      } else {
        write_floats(p.part_o + (part * NH + h) * HD + lane * PER, o);
        if (lane == 0) p.part_ml[part * NH + h] = make_float2(top, den);
      }
    }
    turn = h - live;
  }
  if (tid < 2) p.part_info[2 * blockIdx.x + tid] = crossing[tid];
}

// Joins the parts of a segment that starts in CTA blockIdx.x and goes on in the CTAs behind it; one head per CTA here.
// At HD 32 the compiler spills 4 bytes at 32 registers.
template <int HD, int NH, typename T>
__global__ void __launch_bounds__(COMBINE_GROUPS * 32) combine_kernel(const __grid_constant__ Params p) {
  constexpr int PER = HD / 32;
  __shared__ float so[COMBINE_GROUPS][HD];
  __shared__ float sm[COMBINE_GROUPS], sl[COMBINE_GROUPS];
  wait_for_launch_before();
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

template <typename... Args>
static cudaError_t launch_behind(bool overlap, void (*kern)(Args...), dim3 grid, int threads, size_t smem, cudaStream_t stream,
                                 const Params& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int HD, int NT, typename T>
static int launch(const Params& p, int grid, cudaStream_t stream) {
  const size_t smem = sizeof(Slot<HD, NT>) * 2 * WARPS + sizeof(int) * (2 * p.B + 1);
  auto kern = decode_kernel<HD, NT, T>;
  // the largest it may ask for, told once for each device
  static std::atomic<unsigned long long> told{0};
  int device = 0;
  OB_CUDA_CHECK(cudaGetDevice(&device));
  const unsigned long long bit = 1ull << (device & 63);
  if (!(told.load(std::memory_order_relaxed) & bit)) {
    constexpr int most = sizeof(Slot<HD, NT>) * 2 * WARPS + sizeof(int) * (2 * MAX_BATCH + 1);
    OB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    told.fetch_or(bit, std::memory_order_relaxed);
  }
  OB_CUDA_CHECK(launch_behind(p.appended, kern, dim3(grid), THREADS, smem, stream, p));
  OB_CUDA_CHECK(launch_behind(true, combine_kernel<HD, 8 * NT, T>, dim3(grid, min(8 * NT, p.rep)), COMBINE_GROUPS * 32, 0,
                              stream, p));
  return 0;
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

// CTAs of a launch: as many as fit on the SMs at once (CTAS above), fewer when the batch cannot hold that many runs of
// MIN_UNITS units.
constexpr int MIN_UNITS = 8;
static int grid_size(int B, int Hk, int rep, int hd, int capacity) {
  const int nt = groups(rep, hd), chunks = (rep + 8 * nt - 1) / (8 * nt);
  const long long most = (long long)B * Hk * chunks * ((capacity + UNIT - 1) / UNIT + 1);
  const long long want = (most + MIN_UNITS - 1) / MIN_UNITS, fit = 148 * (nt > 1 || hd > 128 ? 1 : hd > 64 ? 2 : 3);
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

// One block of 8-byte arguments, in this order.  q_dtype: 0 = bf16, 1 = fp16 (also of k_new, v_new and out).  k_new /
// v_new may be null when the cache already holds the current token.  Strides of q, new rows and scales in elements, of
// the cache in bytes.
struct AttentionArgs {
  const void* q;
  long long q_batch, q_dtype;
  const void *k_new, *v_new;
  long long new_batch, new_head;
  void *k, *v;
  long long batch, tok, head;
  float *k_scale, *v_scale;
  long long scale_batch, scale_head;
  const int* lens;
  void *out, *workspace;
  long long B, Hq, Hk, hd, capacity, block;
  double scale;
  long long window;
  int* status;
  cudaStream_t stream;
};
static_assert(sizeof(AttentionArgs) == 29 * 8, "packed");

extern "C" int ob_attn_decode_fp8(const void* packed) {
  AttentionArgs a;
  memcpy(&a, packed, sizeof(a));
  if (a.B <= 0) return 0;
  if (a.B > 0x7fffffffLL || a.Hq > 65536 || a.capacity > 0x3fffffffLL || a.window < 0) return -1;
  const int B = (int)a.B, Hq = (int)a.Hq, Hk = (int)a.Hk, hd = (int)a.hd, capacity = (int)a.capacity, block = (int)a.block;
  const int q_dtype = (int)a.q_dtype, window = (int)(a.window < a.capacity ? a.window : 0);     // a wider one hides nothing
  if (Hk <= 0 || Hq <= 0 || Hq % Hk || hd < 32 || hd > 256 || (hd & (hd - 1)) || capacity <= 0) return -1;
  if (block < 16 || block > 128 || (block & (block - 1)) || q_dtype < 0 || q_dtype > 1) return -1;
  if ((a.batch | a.tok | a.head) % 16) return -2;
  if (a.k_new) {
    const int rc = launch_append({a.k_new, a.v_new, a.new_batch, 0, a.new_head, a.k, a.v, a.batch, a.tok, a.head, a.k_scale,
                                  a.v_scale, a.scale_batch, a.scale_head, a.lens, nullptr, a.status, B, 1, Hk, hd, capacity,
                                  block, 0, 0, 0, 0}, q_dtype, a.stream);
    if (rc) return rc;
  }
  const int rep = Hq / Hk, nt = groups(rep, hd), nh = 8 * nt;
  int shift = 4;
  while ((1 << shift) < block) ++shift;
  for (int b0 = 0; b0 < B; b0 += MAX_BATCH) {
    const int nb = B - b0 < MAX_BATCH ? B - b0 : MAX_BATCH;
    const int grid = grid_size(nb, Hk, rep, hd, capacity);
    Params p;
    p.q = (const uint16_t*)a.q + (long long)b0 * a.q_batch; p.q_batch = a.q_batch;
    p.k = (const uint8_t*)a.k + (long long)b0 * a.batch; p.v = (const uint8_t*)a.v + (long long)b0 * a.batch;
    p.batch = a.batch; p.tok = a.tok; p.head = a.head;
    p.k_scale = a.k_scale + (long long)b0 * a.scale_batch;
    p.v_scale = a.v_scale + (long long)b0 * a.scale_batch;
    p.scale_batch = a.scale_batch; p.scale_head = a.scale_head;
    p.lens = a.lens + b0;
    p.out = (uint16_t*)a.out + (long long)b0 * Hq * hd;
    p.part_o = (float*)a.workspace;
    p.part_ml = (float2*)(p.part_o + (long long)grid * 2 * nh * hd);
    p.part_info = (int2*)(p.part_ml + (long long)grid * 2 * nh);
    p.B = nb; p.Hq = Hq; p.Hk = Hk; p.rep = rep; p.chunks = (rep + nh - 1) / nh; p.capacity = capacity;
    p.block_shift = shift; p.window = window; p.min_units = MIN_UNITS;
    p.scale_log2 = (float)(a.scale * 1.4426950408889634);
    p.appended = a.k_new != nullptr && b0 == 0;      // the launch before is the append
    const int rc = q_dtype == 0 ? dispatch<__nv_bfloat16>(p, hd, nt, grid, a.stream) : dispatch<__half>(p, hd, nt, grid, a.stream);
    if (rc) return rc;
  }
  return 0;
}
