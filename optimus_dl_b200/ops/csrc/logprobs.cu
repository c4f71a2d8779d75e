// Log probabilities of given tokens, the entropy of each row's distribution and its most likely alternatives, from
// a matrix of logits [rows, V] (bf16, fp16 or fp32, any row stride), and the gradient of the first two.
//
//   u_j = (z_j - max z) / T      S = sum_j e^u_j      W = sum_j u_j e^u_j
//   log p_t = u_t - log S        H = log S - W / S
//   dz_j = ( g_l (delta_jt - p_j) - g_H p_j (log p_j + H) ) / T
//
// The forward reads every logit once: each thread keeps (m, S, W) for its share against its own running maximum m, and
// two such triples join as S = S_a 2^(r_a - r) + S_b 2^(r_b - r), W likewise after W_a += (r_a - r) S_a.  All
// exponents are in base 2 against r = m c rounded to fp32, c = log2 e / T: u = fma(z, c, -r) has one rounding, and what
// r lost against m c cancels in H and is put back into log S at the end.  At 1600 MHz, where the chip settles under
// power in a long run, the kernel is bound by instruction issue (the loads alone would take 5/6 of the time), so the
// loop is written for few instructions: packed fp32 pairs, 16-bit pair maxima, one fused operation per exponent.
//
// Where nothing may go wrong: a banned token (-inf) has to add 0 to W, not 0 * inf, so bf16 logits are raised to -1e30
// (a pair at a time) and the exponents of the other types to -200; 2^x is 0 there.  What r lost, up to half a unit in
// its last place, is the exponent of the maximum itself: at most 2^-5 while |r| is below 2^20, but 128, which 2^x does
// not hold, at 2^32 (a row masked with -1e10).  So from 2^20 on, where no ordinary row comes, the exponents are (z - m) c
// with that residue added, and from 2^24 on without it: the sums are against m itself then.  References of both sides of
// 2^20 are therefore of one kind, and a sum from beyond 2^24 is nothing beside one from below 2^20, so where the larger
// maximum's r is below 2^20 the shift between two sums is r_a - r.  The running maximum propagates NaN, and +inf is found
// at the end, so such rows give NaN as the formulas do.  A row without any logit above -inf has log probabilities of
// -inf, entropy 0 and no gradient.
//
// Alternatives: the k largest logits, equal ones by lowest index.  A candidate is one 64-bit number, the logit's
// order-preserving key above the complement of its index, so "better" is one integer comparison without ties.  The
// pass over the logits does no more for them than note, per thread, every batch's maximum (in shared memory) and the
// vector that holds the largest.  Afterwards the k-th best of the threads' maxima is a bound that at least k candidates
// reach; a thread reads those of its batches again whose maximum reaches it (little more than k in the whole CTA,
// unless logits are equal) and lists what reaches the bound, and the list is ranked by counting.  A list that overflows
// (thousands of equal logits in one thread's share) is replaced by k plain arg-max passes.
#include "common.cuh"
#include <cooperative_groups.h>
#include <string.h>

namespace ob {
namespace logprobs {

namespace cg = cooperative_groups;

constexpr int THREADS = 256;     // of the gradient's CTAs and, with few rows, of the forward's
constexpr int NARROW = 128;      // of the forward's with many rows
constexpr int UNROLL = 4;        // 16-byte loads in flight per thread
constexpr int MAX_TOPK = 32;
constexpr int CAP = 512;        // candidates a CTA can list
constexpr int MAX_CLUSTER = 8;
constexpr int LOOKS = 512;      // notes that the CTA looks behind together
constexpr int NOTES = 16;        // maxima a thread notes: one for each batch, or for 2, 4, 8... of longer slices
constexpr float FLOOR = -200.0f;       // of an exponent: 2^x is 0 in fp32
constexpr float FAR = 1048576.f;       // 2^20: a maximum with an r of this magnitude or more is treated apart
constexpr float FARTHER = 16777216.f;  // 2^24: from here on sums are against the maximum itself

using u64 = unsigned long long;

__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static constexpr uint32_t NONE = 0xff800000u;      // 32 bits of -inf
  static constexpr bool LIFTED = false;              // exponents have to be kept above FLOOR one by one
  __device__ static uint4 lift(const uint4& u, uint32_t = 0) { return u; }
  __device__ static uint32_t below(float) { return 0; }
  __device__ static void unpack(const uint4& u, float (&f)[N]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  __device__ static float max_of(const uint4& u) {
    float f[N];
    unpack(u, f);
    return max_nan(max_nan(f[0], f[1]), max_nan(f[2], f[3]));
  }
  __device__ static uint4 pack(const float (&f)[N]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  __device__ static float load(const float* p) { return *p; }
  __device__ static float cast(float f) { return f; }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t NONE = 0xff80ff80u;
  static constexpr bool LIFTED = true;
  __device__ static uint4 lift(const uint4& u, uint32_t low = 0xf14af14au) {         // at least -1e30, or `low` (a pair)
    return make_uint4(lift2(u.x, low), lift2(u.y, low), lift2(u.z, low), lift2(u.w, low));
  }
  __device__ static uint32_t lift2(uint32_t a, uint32_t low) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(low));
    return r;
  }
  __device__ static uint32_t below(float f) {            // a pair of f rounded down
    const uint32_t b = __bfloat16_as_ushort(__float2bfloat16_rd(f));
    return b << 16 | b;
  }
  __device__ static void unpack(const uint4& u, float (&f)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  __device__ static float max_of(const uint4& u) {       // two elements per instruction
    const uint32_t w = max2(max2(u.x, u.y), max2(u.z, u.w));
    return max_nan(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ static uint4 pack(const float (&f)[N]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
  __device__ static float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ static __nv_bfloat16 cast(float f) { return __float2bfloat16(f); }
};
template <> struct Vec<__half> {
  static constexpr int N = 8;
  static constexpr uint32_t NONE = 0xfc00fc00u;
  static constexpr bool LIFTED = false;
  __device__ static uint4 lift(const uint4& u, uint32_t = 0) { return u; }
  __device__ static uint32_t below(float) { return 0; }
  __device__ static void unpack(const uint4& u, float (&f)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x; f[2 * i + 1] = v.y;
    }
  }
  __device__ static float max_of(const uint4& u) {
    const uint32_t w = max2(max2(u.x, u.y), max2(u.z, u.w));
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return max_nan(v.x, v.y);
  }
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ static uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static uint4 pack(const float (&f)[N]) {
    return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
  }
  __device__ static float load(const __half* p) { return __half2float(*p); }
  __device__ static __half cast(float f) { return __float2half(f); }
};

// Candidate: order-preserving key (NaN above everything, one zero) over the complement of the index.  Integer
// arithmetic only, so values below the normal range keep their order.
__device__ __forceinline__ u64 candidate(float z, int idx) {
  uint32_t b = __float_as_uint(z);
  if ((b & 0x7fffffffu) > 0x7f800000u) b = 0x7fffffffu;
  if (b == 0x80000000u) b = 0u;
  const uint32_t key = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((u64)key << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ float candidate_value(u64 c) {
  const uint32_t key = (uint32_t)(c >> 32);
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
__device__ __forceinline__ int candidate_index(u64 c) { return (int)~(uint32_t)c; }

struct Sums { float m, s, w; };        // s and w against r = m c, from FARTHER on against m itself
// The exponent of the maximum itself: what r = m c rounded leaves of it.
__device__ __forceinline__ float residue(float m, float c) {
  const float r = __fmul_rn(m, c);
  return fabsf(r) < FARTHER ? fmaf(m, c, -r) : 0.f;
}
// log2 of the factor that takes sums of a maximum `a` to a larger one, `m`: the second form holds for any maxima, the
// first where |r| is below FAR.
__device__ __forceinline__ float shift(float a, float ra, float m, float r) {
  return a == m ? 0.f : fmaxf(ra - r, FLOOR);
}
__device__ __forceinline__ float shift_far(float a, float m, float c) {
  return a == m ? 0.f : fmaxf((a - m) * c - residue(a, c) + residue(m, c), FLOOR);
}
// Sums against another maximum, at least their own.
__device__ __forceinline__ void carry(Sums& a, float m, float c) {
  const float r = __fmul_rn(m, c);
  // lanes without a share (m = -inf) take the short way: they do not keep the others waiting
  const float d = fabsf(r) < FAR || m == -INFINITY ? shift(a.m, __fmul_rn(a.m, c), m, r) : shift_far(a.m, m, c);
  const float f = exp2_fast(d);
  a.w = f * (a.w + d * a.s);
  a.s *= f;
  a.m = m;
}
// The sums of LANES neighbouring lanes together, in each of them: the maximum first, then one shift for each lane.
template <int LANES>
__device__ __forceinline__ void join_lanes(Sums& a, float c) {
  float m = a.m;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  carry(a, m, c);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
  }
}

struct Params {
  const void* logits; long long ld;
  const long long* targets;
  float* logp; float* entropy;
  float2* stats; float* kept;                     // for the gradient: (max, log2 S) and the entropy once more
  float* top_logp; long long* top_ids;
  int rows, V, k, cluster;
  float c, inv_t;
};

// Not in base 2: log2 e times the type's lowest value is no fp32 number.
__device__ __forceinline__ float log_of(float z, float m, float inv_t, float log2s) {
  return (z - m) * inv_t - log2s * 0.6931471805599453f;
}

// Of a CTA that looks for alternatives.  Kept to some 28 KB: four CTAs of 54 KB left the SM so little of its L1 cache for
// the loads in flight that 1000 rows of 50257 fp32 took 54 us instead of 43.
template <int TH>
struct Scratch {
  u64 list[CAP], few[CAP], top[MAX_TOPK], merged[MAX_TOPK], warp_bound[TH / 32], kth;
  float note[NOTES][TH];
  int look[LOOKS];
  int listed, counted, looks;
};

// A lower bound of the k-th best of the CTA's candidates, one per thread; the first `active` threads have one (0
// elsewhere).  The r-th best of the lanes in each of W warps, r = ceil(k / W), and the least of those: r W >= k
// candidates reach it.  0 when there are too few to tell.  One barrier, before the result is read.
template <int TH>
__device__ __forceinline__ u64 bound(u64 best, int active, int k, u64* warp_bound) {
  const int warps = max(1, min(active, TH) >> 5), warp = threadIdx.x >> 5;
  if (warp < warps) {
    u64 w = 0;
    for (int i = (k + warps - 1) / warps; i > 0; --i) {
      const uint32_t key = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32));
      const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(best >> 32) == key ? (uint32_t)best : 0u);
      w = (u64)key << 32 | low;
      if (best == w) best = 0;
    }
    if ((threadIdx.x & 31) == 0) warp_bound[warp] = w;
  }
  __syncthreads();
  u64 b = warp_bound[0];
  for (int w = 1; w < warps; ++w) b = min(b, warp_bound[w]);
  return b;
}

// The k best of `n` candidates in `list` (0 = none), best first.  Barriers inside, none at the end; sc.counted is 0
// before.
template <int TH>
__device__ __forceinline__ void select_top(const u64* list, int n, int k, u64* top, Scratch<TH>& sc) {
  if (n > 64) {
    u64 best = 0;
    for (int i = threadIdx.x; i < n; i += TH) best = max(best, list[i]);
    const u64 b = bound<TH>(best, n, k, sc.warp_bound);
    for (int i = threadIdx.x; i < n; i += TH)
      if (list[i] >= b && list[i] != 0) sc.few[atomicAdd(&sc.counted, 1)] = list[i];
    __syncthreads();
    n = sc.counted;
    list = sc.few;
  }
  for (int i = threadIdx.x; i < n; i += TH) {
    const u64 mine = list[i];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += list[j] > mine;
    if (r < k && mine != 0) top[r] = mine;
  }
}

template <typename T, bool TOPK, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH) forward_kernel(const __grid_constant__ Params p) {
  static_assert(UNROLL == 4 && TH <= 256, "how a look is packed and shared out");
  constexpr int N = Vec<T>::N, STEP = TH * UNROLL;
  __shared__ Sums warp_sums[TH / 32];
  __shared__ Sums cta_sums;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  auto& sc = *reinterpret_cast<Scratch<TH>*>(smem_raw);          // TOPK only
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.cluster, rank = blockIdx.x - row * p.cluster;
  const T* z = static_cast<const T*>(p.logits) + (long long)row * p.ld;
  const float c = p.c;
  // elements before the first 16-byte boundary, whole vectors, elements after the last one
  const int head = min(p.V, (int)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T)));
  const int nv = (p.V - head) / N;
  const int v0 = (int)((long long)nv * rank / p.cluster), v1 = (int)((long long)nv * (rank + 1) / p.cluster);
  const char* zv = reinterpret_cast<const char*>(z + head);
  const char* at = zv + ((long long)v0 + tid) * 16;
  auto fetch = [&](int base, uint4 (&raw)[UNROLL]) {             // from `at`; what lies behind the slice reads as banned
    if (base + STEP <= v1) {
#pragma unroll
      for (int j = 0; j < UNROLL; ++j) raw[j] = load_once(at + j * TH * 16);
    } else {
#pragma unroll
      for (int j = 0; j < UNROLL; ++j) {
        raw[j] = make_uint4(Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE, Vec<T>::NONE);
        if (base + j * TH + tid < v1) raw[j] = load_once(at + j * TH * 16);
      }
    }
    at += STEP * 16;
  };
  uint4 raw[UNROLL], next[UNROLL];
  fetch(v0, raw);
  // the token's own logit is under way while the row is read
  float z_t = 0.f;
  bool inside = false;
  if (rank == 0 && tid == 0) {
    const long long t = p.targets[row];
    inside = t >= 0 && t < p.V;
    if (inside) z_t = Vec<T>::load(z + t);
  }
  if (TOPK) {
    if (tid == 0) { sc.listed = sc.counted = sc.looks = 0; sc.kth = 0; }
    if (tid < MAX_TOPK) sc.top[tid] = sc.merged[tid] = 0;
  }

  float m = -INFINITY, r = -INFINITY;
  float2 s2 = make_float2(0.f, 0.f), w2 = s2;
  const float2 cc = make_float2(c, c);
  int best_vec = v0 + tid;             // TOPK: a vector that holds this thread's maximum (or one behind it)
  int group = 0;                       // log2 of the batches that share a note
  if (TOPK)
    while ((v1 - v0 + STEP - 1) / STEP > NOTES << group) ++group;
  auto add = [&](int base, const uint4 (&raw)[UNROLL]) {
    float top_of[UNROLL], mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      top_of[j] = Vec<T>::max_of(raw[j]);
      mx = max_nan(mx, top_of[j]);
    }
    if (TOPK && !(mx <= m)) {
      best_vec = base + (UNROLL - 1) * TH + tid;
#pragma unroll
      for (int j = UNROLL - 2; j >= 0; --j) if (top_of[j] == mx) best_vec = base + j * TH + tid;
    }
    if (TOPK) {
      const int batch = (base - v0) / STEP;
      float& note = sc.note[batch >> group][tid];
      note = (batch & ((1 << group) - 1)) ? max_nan(note, mx) : mx;
    }
    mx = max_nan(mx, m);
    const float now = __fmul_rn(mx, c);
    auto raise = [&](float d) {                                  // the sums so far to the new maximum
      const float f = exp2_fast(d);
      w2 = fmul2(ffma2(make_float2(d, d), s2, w2), make_float2(f, f));
      s2 = fmul2(s2, make_float2(f, f));
      m = mx;
      r = now;
    };
    if (fabsf(now) < FAR) {
      raise(shift(m, r, mx, now));
      const float2 neg = make_float2(-r, -r);
#pragma unroll
      for (int j = 0; j < UNROLL; ++j) {
        float z8[N];
        Vec<T>::unpack(Vec<T>::lift(raw[j]), z8);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          float2 u = ffma2(make_float2(z8[e], z8[e + 1]), cc, neg);
          if (!Vec<T>::LIFTED) u = make_float2(fmaxf(u.x, FLOOR), fmaxf(u.y, FLOOR));
          const float2 x = make_float2(exp2_fast(u.x), exp2_fast(u.y));
          s2 = fadd2(s2, x);
          w2 = ffma2(u, x, w2);
        }
      }
    } else {
      raise(shift_far(m, mx, c));
      if (fabsf(m) < INFINITY) {
        const float rest = residue(m, c);
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
          float z8[N];
          Vec<T>::unpack(raw[j], z8);
#pragma unroll 1
          for (int k = 0; k < N; ++k) {            // one element a turn: code that is hardly ever run stays small
            const float u = fmaxf(fmaf(z8[0] - m, c, rest), FLOOR), x = exp2_fast(u);
            s2.x += x;
            w2.x = fmaf(u, x, w2.x);
#pragma unroll
            for (int e = 0; e + 1 < N; ++e) z8[e] = z8[e + 1];
          }
        }
      }
    }
  };
  for (int base = v0; base < v1; base += 2 * STEP) {       // two buffers in turn: one is added up, one under way
    fetch(base + STEP, next);
    add(base, raw);
    if (base + STEP >= v1) break;
    fetch(base + 2 * STEP, raw);
    add(base + STEP, next);
  }
  Sums st{m, s2.x + s2.y, w2.x + w2.y};
  const u64 mine = TOPK && v0 + tid < v1 ? candidate(st.m, head + best_vec * N + N - 1) : 0;
  // the ragged ends of the row: fewer than N elements each
  const int tail = p.V - head - nv * N;
  const int extra0 = rank == 0 ? head : 0, extra1 = rank == p.cluster - 1 ? tail : 0;
  const int extra_at = tid < extra0 ? tid : head + nv * N + (tid - extra0);
  float extra = -INFINITY;
  if (tid < extra0 + extra1) {
    extra = Vec<T>::load(z + extra_at);
    const float u = residue(extra, c), x = exp2_fast(u);       // NaN and +inf are found by the maximum
    if (extra != -INFINITY) {
      Sums end{extra, x, u * x};
      const float m = max_nan(st.m, extra);
      carry(st, m, c);
      carry(end, m, c);
      st.s += end.s;
      st.w += end.w;
    }
  }

  // one triple per CTA
  join_lanes<32>(st, c);
  if (lane == 0) warp_sums[warp] = st;
  __syncthreads();
  if (warp == 0) {
    Sums t = lane < TH / 32 ? warp_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
    join_lanes<TH / 32>(t, c);
    if (lane == 0) cta_sums = t;
  }
  if (TOPK) {
    // the k-th best of the threads' maxima
    const u64 rough = bound<TH>(mine, v1 - v0, p.k, sc.warp_bound);
    if (mine != 0 && mine >= rough) sc.list[atomicAdd(&sc.counted, 1)] = mine;
    __syncthreads();
    const int near = sc.counted;
    for (int i = tid; i < near; i += TH) {
      const u64 m = sc.list[i];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < near; ++j) r += sc.list[j] > m;
      if (r == p.k - 1) sc.kth = m;
    }
    __syncthreads();
    const u64 kth = sc.kth;
    const float kth_z = kth == 0 ? -INFINITY : candidate_value(kth);
    const int kth_at = kth == 0 ? 0x7fffffff : candidate_index(kth);
    auto push = [&](float f, int idx) {
      const u64 cand = candidate(f, idx);
      if (cand >= kth) {
        const int at = atomicAdd(&sc.listed, 1);
        if (at < CAP) sc.list[at] = cand;
      }
    };
    auto examine = [&](const uint4& u, int i) {
      const float mx = Vec<T>::max_of(u);
      if (mx < kth_z || (mx == kth_z && head + i * N > kth_at)) return;
      float f[N];
      Vec<T>::unpack(u, f);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (!(f[e] < kth_z)) push(f[e], head + i * N + e);
    };
    // notes that reach the bound, little more than k; their vectors are shared out over all threads
    const int notes = ((v1 - v0 + STEP - 1) / STEP + (1 << group) - 1) >> group;
    for (int n = 0; n < notes; ++n)
      if (!(sc.note[n][tid] < kth_z) && v0 + tid < v1) {
        const int at = atomicAdd(&sc.looks, 1);
        if (at < LOOKS) sc.look[at] = n << 8 | tid;
      }
    __syncthreads();
    const int looks = sc.looks, each = UNROLL << group;
    if (looks <= LOOKS) {
      for (int w = tid; w < looks * each; w += TH) {
        const int q = w >> (2 + group), look = sc.look[q];
        const int i = v0 + (((look >> 8) << group) * UNROLL + (w - q * each)) * TH + (look & 255);
        if (i < v1) examine(load_once(zv + (long long)i * 16), i);
      }
    } else {
      // Much of the slice reaches the bound: everyone looks at all of it, or, where nothing lies above (equal logits,
      // all banned), as far as the bound's index.
      const int end = cta_sums.m == kth_z ? min(v1, max(kth_at - head, 0) / N + 1) : v1;
#pragma unroll 1
      for (int w = v0 + tid; w < end; w += TH * UNROLL) {
#pragma unroll
        for (int j = 0; j < UNROLL; ++j)
          if (w + j * TH < end) raw[j] = load_once(zv + (long long)(w + j * TH) * 16);
#pragma unroll
        for (int j = 0; j < UNROLL; ++j)
          if (w + j * TH < end) examine(raw[j], w + j * TH);
      }
    }
    if (tid < extra0 + extra1) push(extra, extra_at);
    if (tid == 0) sc.counted = 0;
    __syncthreads();
    const int n = sc.listed;
    if (n <= CAP) {
      select_top(sc.list, n, p.k, sc.top, sc);
    } else {
      // more candidates than the list holds: k arg-max passes, each below the one before
      u64 limit = ~0ull;
      for (int r = 0; r < p.k; ++r) {
        u64 best = 0;
        for (int i = v0 + tid; i < v1; i += TH) {
          float f[N];
          Vec<T>::unpack(load_once(zv + (long long)i * 16), f);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const u64 cand = candidate(f[e], head + i * N + e);
            if (cand < limit && cand > best) best = cand;
          }
        }
        if (tid < extra0 + extra1) {
          const u64 cand = candidate(extra, extra_at);
          if (cand < limit && cand > best) best = cand;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        __syncthreads();
        if (lane == 0) sc.list[warp] = best;
        __syncthreads();
        best = sc.list[0];
        for (int i = 1; i < TH / 32; ++i) best = max(best, sc.list[i]);
        if (tid == 0) sc.top[r] = best;
        if (best == 0) break;
        limit = best;
      }
    }
  }
  __syncthreads();
  if (p.cluster > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    if (rank == 0) {
      if (warp == 0) {
        Sums t = lane < p.cluster ? *cl.map_shared_rank(&cta_sums, lane) : Sums{-INFINITY, 0.f, 0.f};
        join_lanes<MAX_CLUSTER>(t, c);
        if (lane == 0) warp_sums[0] = t;
      }
      if (TOPK) {
        const int n = p.cluster * p.k;
        for (int i = tid; i < n; i += TH) sc.list[i] = cl.map_shared_rank(sc.top, i / p.k)[i % p.k];
        if (tid == 0) sc.counted = 0;
        __syncthreads();
        select_top(sc.list, n, p.k, sc.merged, sc);
      }
    }
    cl.sync();            // no CTA leaves while its shared memory is read
    if (rank != 0) return;
  }
  const Sums total = p.cluster > 1 ? warp_sums[0] : cta_sums;
  const bool none = total.m == -INFINITY, broken = !(total.m < INFINITY);     // +inf and NaN
  const float sum_log2 = broken ? NAN : none ? 0.f : log2f(total.s);
  const float top_z = none ? 0.f : total.m;
  // against the maximum itself from here on
  const float log2s = sum_log2 - residue(top_z, c);
  if (tid == 0) {
    p.logp[row] = inside ? log_of(z_t, top_z, p.inv_t, log2s) : 0.f;
    const float h = none ? 0.f : (sum_log2 - total.w / total.s) * 0.6931471805599453f;
    p.entropy[row] = h;
    if (p.stats) {
      p.stats[row] = make_float2(total.m, log2s);
      p.kept[row] = h;
    }
  }
  if (TOPK && tid < p.k) {
    const u64 cand = p.cluster > 1 ? sc.merged[tid] : sc.top[tid];
    p.top_logp[(long long)row * p.k + tid] = log_of(candidate_value(cand), top_z, p.inv_t, log2s);
    p.top_ids[(long long)row * p.k + tid] = candidate_index(cand);
  }
}

// dz of one row's share: two batches of loads are in flight per thread, and the row's numbers are fetched behind the
// first.  Exponents as in the forward pass, v = log2 p = fma(z, c, -r) - log2 S, in packed pairs: with the plain form of
// a difference, a product, a clamp and a product per element the kernel issued 14.5 instructions per logit.  Rows are
// taken from the last to the first: a forward pass that ran just before left its last rows in the L2 cache.  `dz` may
// be the logits themselves (every element is read and written by the same thread).
template <typename T>
__global__ void __launch_bounds__(THREADS, 4)
backward_kernel(const T* logits, long long ld, const long long* __restrict__ targets, const float2* __restrict__ stats,
                const float* __restrict__ entropy, const float* __restrict__ d_logp, const float* __restrict__ d_entropy,
                T* dz, long long dz_ld, int rows, int V, int pieces, float c, float inv_t) {
  constexpr int N = Vec<T>::N, STEP = THREADS * UNROLL;
  const int up = blockIdx.x / pieces, piece = blockIdx.x - up * pieces, row = rows - 1 - up, tid = threadIdx.x;
  const T* z = logits + (long long)row * ld;
  T* g = dz + (long long)row * dz_ld;
  const int head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) / sizeof(T)));
  const int nv = (V - head) / N;
  const int v0 = (int)((long long)nv * piece / pieces), v1 = (int)((long long)nv * (piece + 1) / pieces);
  const bool aligned = (reinterpret_cast<uintptr_t>(z + head) & 15) == 0;
  const T* from = z + head + ((long long)v0 + tid) * N;
  T* to = g + head + ((long long)v0 + tid) * N;
  auto fetch = [&](int base, uint4 (&raw)[UNROLL]) {
    if (aligned && base + STEP <= v1) {
#pragma unroll
      for (int j = 0; j < UNROLL; ++j) raw[j] = load_once(from + j * THREADS * N);
    } else {
#pragma unroll
      for (int j = 0; j < UNROLL; ++j)
        if (base + j * THREADS + tid < v1) {
          if (aligned) {
            raw[j] = load_once(from + j * THREADS * N);
          } else {
            T tmp[N];
#pragma unroll
            for (int e = 0; e < N; ++e) tmp[e] = from[j * THREADS * N + e];
            memcpy(&raw[j], tmp, 16);
          }
        }
    }
    from += STEP * N;
  };
  uint4 raw[UNROLL], next[UNROLL];
  fetch(v0, raw);
  const float2 st = stats[row];
  const bool none = st.x == -INFINITY;
  const float m = none ? 0.f : st.x;
  const long long t64 = targets[row];
  const bool inside = t64 >= 0 && t64 < V;
  const int t = inside && !none ? (int)t64 : -1;
  const float gl = inside && d_logp ? d_logp[row] : 0.f, gh = d_entropy ? d_entropy[row] : 0.f;
  // p (log p + H) = p (v ln 2 + H) with v = log2 p: dz = -(p / T) (a + b v), a = g_l + g_H H, b = g_H ln 2
  const float a = none ? 0.f : -inv_t * (gl + gh * entropy[row]), b = none ? 0.f : -inv_t * gh * 0.6931471805599453f;
  const float r = __fmul_rn(m, c), log2s = st.y + residue(m, c);       // log2 S against r
  const bool apart = !(fabsf(r) < FAR);              // also NaN and infinities, whose log2 S is NaN
  // what the loop below seldom needs is read again: kept, it costs registers that the loop lacks
  auto at_token = [&] {
    float g = 0.f;
    if (d_logp) asm volatile("ld.global.f32 %0, [%1];" : "=f"(g) : "l"(d_logp + row));
    return g * inv_t;
  };
  auto grad = [&](float f) {                         // of one element, whatever the maximum
    float2 s;
    asm volatile("ld.global.v2.f32 {%0, %1}, [%2];" : "=f"(s.x), "=f"(s.y) : "l"(stats + row));
    const float v = max_nan((f - (s.x == -INFINITY ? 0.f : s.x)) * c - s.y, FLOOR);
    return exp2_fast(v) * fmaf(b, v, a);
  };
  const float2 cc = make_float2(c, c), neg_r = make_float2(-r, -r), neg_s = make_float2(-log2s, -log2s);
  const float2 aa = make_float2(a, a), bb = make_float2(b, b);
  // bf16: p is 0 300 below the maximum in the exponent, and b v stays a number there whatever g_H and T are (raised to
  // -1e30 as in the forward pass, a banned token had 0 * inf from |g_H| / T^2 of 3e8 on)
  const uint32_t low = Vec<T>::below(m - 300.f / c);
  auto put = [&](int base, const uint4 (&raw)[UNROLL]) {
    const bool full = base + STEP <= v1;
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int i = base + j * THREADS + tid;
      if (full || i < v1) {
        float f[N];
        if (!apart) {
          Vec<T>::unpack(Vec<T>::lift(raw[j], low), f);
#pragma unroll
          for (int e = 0; e < N; e += 2) {
            float2 v = fadd2(ffma2(make_float2(f[e], f[e + 1]), cc, neg_r), neg_s);
            if (!Vec<T>::LIFTED) v = make_float2(max_nan(v.x, FLOOR), max_nan(v.y, FLOOR));
            const float2 x = fmul2(make_float2(exp2_fast(v.x), exp2_fast(v.y)), ffma2(bb, v, aa));
            f[e] = x.x;
            f[e + 1] = x.y;
          }
        } else {
          Vec<T>::unpack(raw[j], f);
#pragma unroll 1
          for (int k = 0; k < N; ++k) {              // one element a turn: code that is hardly ever run stays small
            float x = f[0];
#pragma unroll
            for (int e = 0; e + 1 < N; ++e) f[e] = f[e + 1];
            f[N - 1] = grad(x);
          }
        }
        const unsigned off = (unsigned)(t - (head + i * N));       // t = -1 is never below N
        if (off < N)
#pragma unroll
          for (int e = 0; e < N; ++e) if (e == off) f[e] += at_token();
        *reinterpret_cast<uint4*>(to + j * THREADS * N) = Vec<T>::pack(f);
      }
    }
    to += STEP * N;
  };
  for (int base = v0; base < v1; base += 2 * STEP) {       // two buffers in turn
    fetch(base + STEP, next);
    put(base, raw);
    if (base + STEP >= v1) break;
    fetch(base + 2 * STEP, raw);
    put(base + STEP, next);
  }
  const int tail = V - head - nv * N;
  if (piece == 0 && tid < head + tail) {
    const int idx = tid < head ? tid : nv * N + tid;
    g[idx] = Vec<T>::cast(grad(Vec<T>::load(z + idx)) + (idx == t ? at_token() : 0.f));
  }
}

template <typename T, bool TOPK, int TH>
static int launch_forward(const Params& p, cudaStream_t stream) {
  auto kern = forward_kernel<T, TOPK, TH>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)p.rows * p.cluster));
  cfg.blockDim = dim3(TH);
  cfg.stream = stream;
  cfg.dynamicSmemBytes = TOPK ? sizeof(Scratch<TH>) : 0;
  static_assert(sizeof(Scratch<TH>) <= 48 * 1024, "what needs no asking");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, kern, p);
}

// Rows enough to fill the SMs four times over go to CTAs of 128 threads, eight to an SM: their latencies at the start
// and the end of a row overlap with more of the others. Measured, 128 against 256 threads: 1000 rows of 50257 fp32 37.6
// and 43.0 us, 4096 of 128256 bf16 with 20 alternatives 183 and 193, without 160 and 162, 8192 in a long run 365 and 375;
// but 257 rows of 50257 fp32 17.8 and 13.7, 64 of 151936 with 20 alternatives 17.3 and 15.7.
template <typename T>
static int run_forward(const Params& p, cudaStream_t stream) {
  if (p.rows >= 148 * 4) return p.k > 0 ? launch_forward<T, true, NARROW>(p, stream) : launch_forward<T, false, NARROW>(p, stream);
  return p.k > 0 ? launch_forward<T, true, THREADS>(p, stream) : launch_forward<T, false, THREADS>(p, stream);
}

// CTAs that share a row: as many as make two per SM with the rows there are, each with at least one full batch of
// loads.  Measured, V = 151936, k = 20, 64 rows: 20.6 us with 1, 15.8 with 2, 15.4 with 4, 16.9 with 8; 257 rows of
// 50257: 14.4 us with 1, 16.5 with 2; one row of 128256, k = 5: 14.4 us with 1, 8.9 with 8, 10.3 with 16.
static int pick_cluster(int rows, int V, int vec) {
  int cl = 1;
  while (cl < MAX_CLUSTER && (long long)rows * cl * 2 <= 148 * 2 && V / (cl * 2) >= THREADS * vec) cl *= 2;
  return cl;
}

}  // namespace logprobs
}  // namespace ob

using namespace ob::logprobs;

// Launchers take one block of 8-byte arguments, in this order.  dtype: 0 = bf16, 1 = fp16, 2 = fp32 (also of the
// gradient).
struct ForwardArgs {
  const void* logits;
  long long ld, dtype;
  const long long* targets;
  float *logp, *entropy;
  float2* stats;                // may be null, and with it:
  float* kept;
  float* top_logp;
  long long* top_ids;
  long long rows, V, top_k;
  double temperature;
  cudaStream_t stream;
};
struct BackwardArgs {
  const void* logits;
  long long ld, dtype;
  const long long* targets;
  const float2* stats;
  const float *entropy, *d_logp, *d_entropy;      // the last two may be null
  void* dz;
  long long dz_ld, rows, V;
  double temperature;
  cudaStream_t stream;
};
static_assert(sizeof(ForwardArgs) == 15 * 8 && sizeof(BackwardArgs) == 14 * 8, "packed");

extern "C" int ob_logprobs_fwd(const void* packed) {
  ForwardArgs a;
  memcpy(&a, packed, sizeof(a));
  const int rows = (int)a.rows, V = (int)a.V, top_k = (int)a.top_k, dtype = (int)a.dtype;
  if (a.rows > 0x7fffffffLL || a.V > 0x7fffffffLL) return -1;
  const double temperature = a.temperature;
  const cudaStream_t stream = a.stream;
  if (rows <= 0) return 0;
  if (V <= 0 || top_k < 0 || top_k > MAX_TOPK || top_k > V || !(temperature >= 1e-6 && temperature <= 1e6)) return -1;
  const int cl = pick_cluster(rows, V, dtype == 2 ? 4 : 8);
  if ((long long)rows * cl > 0x7fffffffLL) return -1;
  const Params p{a.logits, a.ld, a.targets, a.logp, a.entropy, a.stats, a.kept, a.top_logp, a.top_ids, rows, V, top_k, cl,
                 (float)(1.4426950408889634 / temperature), (float)(1.0 / temperature)};
  if (dtype == 0) return run_forward<__nv_bfloat16>(p, stream);
  if (dtype == 1) return run_forward<__half>(p, stream);
  if (dtype == 2) return run_forward<float>(p, stream);
  return -1;
}

extern "C" int ob_logprobs_bwd(const void* packed) {
  BackwardArgs a;
  memcpy(&a, packed, sizeof(a));
  const int rows = (int)a.rows, V = (int)a.V, dtype = (int)a.dtype;
  if (a.rows > 0x7fffffffLL || a.V > 0x7fffffffLL) return -1;
  const double temperature = a.temperature;
  if (rows <= 0) return 0;
  if (V <= 0 || !(temperature >= 1e-6 && temperature <= 1e6)) return -1;
  const int vec = dtype == 2 ? 4 : 8;
  // CTAs per row: four per SM, of half a batch of loads at least, and no more than 8 batches each.  Measured: one row of
  // 128256 bf16 18.5 us with 1, 6.2 with 8, 4.2 with 16; 1000 rows of 50257 42.5 us with 1, 45.2 with 4; 4096 rows of
  // 128256 340 us with 1 (16 batches), 336 with 2, 350 with 4; 2048 such rows in fp32 339 us with 1, 327 with 4.
  int pieces = 1;
  while (V / vec / (pieces * 2) >= THREADS * UNROLL / 2 &&
         ((long long)rows * pieces < 148 * 4 || V / vec / pieces > THREADS * UNROLL * 8))
    pieces *= 2;
  if ((long long)rows * pieces > 0x7fffffffLL) return -1;
  const float c = (float)(1.4426950408889634 / temperature), inv_t = (float)(1.0 / temperature);
  const unsigned grid = (unsigned)((long long)rows * pieces);
#define OB_LAUNCH(T)                                                                                                  \
  backward_kernel<T><<<grid, THREADS, 0, a.stream>>>((const T*)a.logits, a.ld, a.targets, a.stats, a.entropy, a.d_logp, \
                                                     a.d_entropy, (T*)a.dz, a.dz_ld, rows, V, pieces, c, inv_t)
  if (dtype == 0) OB_LAUNCH(__nv_bfloat16);
  else if (dtype == 1) OB_LAUNCH(__half);
  else if (dtype == 2) OB_LAUNCH(float);
  else return -1;
#undef OB_LAUNCH
  return (int)cudaGetLastError();
}
