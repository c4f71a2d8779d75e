// Log probabilities of given tokens, the entropy of each row's distribution and its most likely alternatives, from
// a matrix of logits [rows, V] (bf16, fp16 or fp32, any row stride), and the gradient of the first two.
//
//   u_j = (z_j - max z) / T      S = sum_j e^u_j      W = sum_j u_j e^u_j
//   log p_t = u_t - log S        H = log S - W / S
//   dz_j = ( g_l (delta_jt - p_j) - g_H p_j (log p_j + H) ) / T
//
// The forward reads every logit once: each thread keeps (m, S, W) for its share against its own running maximum m,
// and two such triples join as S = S_a 2^(m_a - m) + S_b 2^(m_b - m), W likewise after W_a += (m_a - m) S_a.  All
// exponents are in base 2 (u log2 e = (z - m) c with c = log2 e / T); sums and statistics are fp32.  Differences are
// taken before the product with c, so a row of the type's lowest value is a uniform row and not an overflow.
// Exponents are clamped at -200, where 2^x is 0 in fp32 anyway: a banned token (-inf) then adds 0 to W, not 0 * inf.
// The running maximum propagates NaN, and +inf is found at the end, so such rows give NaN as the formulas do.  A row
// without any logit above -inf has log probabilities of -inf, entropy 0 and no gradient.
//
// Alternatives: the k largest logits, equal ones by lowest index.  A candidate is one 64-bit number, the logit's
// order-preserving key above the complement of its index, so "better" is one integer comparison without ties.  After
// its first batch a CTA takes the k-th best of its threads' best candidates as a threshold: at least k candidates
// reach it, so nothing below it can be among the k largest.  From then on only candidates at or above the threshold
// go to a shared list (about k for every doubling of the positions seen; the threshold is raised after 4, 16, 64...
// batches), and the list is ranked at the end.  A list that overflows (rows sorted upwards) is replaced by k plain
// arg-max passes over the slice, which the L2 cache serves.
#include "common.cuh"
#include <cooperative_groups.h>

namespace ob {
namespace logprobs {

namespace cg = cooperative_groups;

constexpr int THREADS = 256;
constexpr int UNROLL = 4;        // 16-byte loads in flight per thread
constexpr int MAX_TOPK = 32;
constexpr int CAP = 1024;        // candidates a CTA can list
constexpr int MAX_CLUSTER = 16;
constexpr float FLOOR = -200.0f;

using u64 = unsigned long long;

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void unpack(const uint4& u, float (&f)[N]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  __device__ static uint4 pack(const float (&f)[N]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  __device__ static float load(const float* p) { return *p; }
  __device__ static float cast(float f) { return f; }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4& u, float (&f)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  }
  __device__ static uint4 pack(const float (&f)[N]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
  __device__ static float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ static __nv_bfloat16 cast(float f) { return __float2bfloat16(f); }
};
template <> struct Vec<__half> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4& u, float (&f)[N]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x; f[2 * i + 1] = v.y;
    }
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

struct Sums { float m, s, w; };
__device__ __forceinline__ void join(Sums& a, const Sums& b, float c) {
  const float m = max_nan(a.m, b.m);
  const float da = a.m == m ? 0.f : fmaxf((a.m - m) * c, FLOOR), db = b.m == m ? 0.f : fmaxf((b.m - m) * c, FLOOR);
  const float fa = exp2_fast(da), fb = exp2_fast(db);
  a.w = fa * (a.w + da * a.s) + fb * (b.w + db * b.s);
  a.s = fa * a.s + fb * b.s;
  a.m = m;
}

struct Params {
  const void* logits; long long ld;
  const long long* targets;
  float* logp; float* entropy; float2* stats;     // stats: (max, log2 S), what the gradient needs beside the entropy
  float* top_logp; long long* top_ids;
  int rows, V, k, cluster;
  float c;
};

__device__ __forceinline__ float log_of(float z, float m, float c, float log2s) {
  return ((z - m) * c - log2s) * 0.6931471805599453f;
}

// `n` candidates in `list` (0 = none): writes the k best to `top`, best first.  All threads of the CTA.
__device__ __forceinline__ void rank_into(const u64* list, int n, int k, u64* top) {
  for (int i = threadIdx.x; i < n; i += THREADS) {
    const u64 mine = list[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += list[j] > mine;
    if (r < k && mine != 0) top[r] = mine;
  }
}

template <typename T, bool TOPK>
__global__ void __launch_bounds__(THREADS, TOPK ? 3 : 4) forward_kernel(const Params p) {
  constexpr int N = Vec<T>::N;
  __shared__ Sums warp_sums[THREADS / 32];
  __shared__ Sums cta_sums;
  __shared__ u64 list[TOPK ? CAP : 1];
  __shared__ u64 top[TOPK ? MAX_TOPK : 1];
  __shared__ u64 merged[TOPK ? MAX_TOPK : 1];
  __shared__ u64 threshold;
  __shared__ int listed;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / p.cluster, rank = blockIdx.x - row * p.cluster;
  const T* z = static_cast<const T*>(p.logits) + (long long)row * p.ld;
  const float c = p.c;
  // elements before the first 16-byte boundary, whole vectors, elements after the last one
  const int head = min(p.V, (int)(((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T)));
  const int nv = (p.V - head) / N;
  const int v0 = (int)((long long)nv * rank / p.cluster), v1 = (int)((long long)nv * (rank + 1) / p.cluster);
  const char* zv = reinterpret_cast<const char*>(z + head);
  u64 tau = 0;            // the threshold as this thread last saw it, and its value for the quick test
  float tau_z = -INFINITY;
  if (TOPK) {
    if (tid == 0) { threshold = 0; listed = 0; }
    if (tid < MAX_TOPK) { top[tid] = 0; merged[tid] = 0; }
    __syncthreads();
  }
  auto push = [&](float f, int idx) {
    const u64 cand = candidate(f, idx);
    if (cand >= tau) {
      const int at = atomicAdd(&listed, 1);
      if (at < CAP) list[at] = cand;
    }
  };

  Sums st{-INFINITY, 0.f, 0.f};
  int batch = 0, next_refresh = 4;
  for (int base = v0; base < v1; base += THREADS * UNROLL, ++batch) {
    uint4 raw[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int i = base + j * THREADS + tid;
      if (i < v1) raw[j] = load_once(zv + (long long)i * 16);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      if (base + j * THREADS + tid < v1) {
        float f[N];
        Vec<T>::unpack(raw[j], f);
#pragma unroll
        for (int e = 0; e < N; ++e) mx = max_nan(mx, f[e]);
      }
    }
    Sums fresh{mx, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      if (base + j * THREADS + tid < v1) {
        float f[N];
        Vec<T>::unpack(raw[j], f);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float u = fmaxf((f[e] - mx) * c, FLOOR);
          const float x = exp2_fast(u);
          fresh.s += x;
          fresh.w = fmaf(u, x, fresh.w);
        }
      }
    }
    join(st, fresh, c);
    if (TOPK) {
      if (batch == 0) {
        u64 best = 0;
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
          const int i = base + j * THREADS + tid;
          if (i < v1) {
            float f[N];
            Vec<T>::unpack(raw[j], f);
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const u64 cand = candidate(f[e], head + i * N + e);
              if (cand > best) best = cand;
            }
          }
        }
        list[tid] = best;
        __syncthreads();
        int r = 0;
        for (int j = 0; j < THREADS; ++j) r += list[j] > best;
        if (best != 0 && r == p.k - 1) threshold = best;
        __syncthreads();
      } else if (batch == next_refresh) {
        next_refresh *= 4;
        __syncthreads();
        const int n = listed;
        if (n <= CAP)
          for (int i = tid; i < n; i += THREADS) {
            const u64 mine = list[i];
            int r = 0;
            for (int j = 0; j < n; ++j) r += list[j] > mine;
            if (r == p.k - 1) threshold = mine;
          }
        __syncthreads();
      }
      if (batch == 0 || batch * 4 == next_refresh) {
        tau = threshold;
        tau_z = tau == 0 ? -INFINITY : candidate_value(tau);
      }
      if (!(mx < tau_z)) {
#pragma unroll
        for (int j = 0; j < UNROLL; ++j) {
          const int i = base + j * THREADS + tid;
          if (i < v1) {
            float f[N];
            Vec<T>::unpack(raw[j], f);
#pragma unroll
            for (int e = 0; e < N; ++e)
              if (!(f[e] < tau_z)) push(f[e], head + i * N + e);
          }
        }
      }
    }
  }
  // the ragged ends of the row: fewer than N elements each
  const int tail = p.V - head - nv * N;
  const int extra0 = rank == 0 ? head : 0, extra1 = rank == p.cluster - 1 ? tail : 0;
  if (tid < extra0 + extra1) {
    const int idx = tid < extra0 ? tid : head + nv * N + (tid - extra0);
    const float f = Vec<T>::load(z + idx);
    const float u = f == f ? 0.f : f;      // e^0, or NaN
    join(st, Sums{f, 1.f + u, 0.f}, c);
    if (f == -INFINITY && st.m == -INFINITY) st = Sums{-INFINITY, 0.f, 0.f};
    if (TOPK) push(f, idx);
  }

  // one triple per CTA
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums b;
    b.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    b.w = __shfl_xor_sync(0xffffffffu, st.w, o);
    join(st, b, c);
  }
  if (lane == 0) warp_sums[warp] = st;
  __syncthreads();
  if (tid == 0) {
    Sums t = warp_sums[0];
    for (int i = 1; i < THREADS / 32; ++i) join(t, warp_sums[i], c);
    cta_sums = t;
  }
  if (TOPK) {
    const int n = listed;
    if (n <= CAP) {
      rank_into(list, n, p.k, top);
    } else {
      // more candidates than the list holds: k arg-max passes, each below the one before
      u64 limit = ~0ull;
      for (int r = 0; r < p.k; ++r) {
        u64 best = 0;
        for (int i = v0 + tid; i < v1; i += THREADS) {
          const uint4 raw = *reinterpret_cast<const uint4*>(zv + (long long)i * 16);
          float f[N];
          Vec<T>::unpack(raw, f);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const u64 cand = candidate(f[e], head + i * N + e);
            if (cand < limit && cand > best) best = cand;
          }
        }
        if (tid < extra0 + extra1) {
          const int idx = tid < extra0 ? tid : head + nv * N + (tid - extra0);
          const u64 cand = candidate(Vec<T>::load(z + idx), idx);
          if (cand < limit && cand > best) best = cand;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const u64 b = __shfl_xor_sync(0xffffffffu, best, o);
          if (b > best) best = b;
        }
        __syncthreads();
        if (lane == 0) list[warp] = best;
        __syncthreads();
        best = list[0];
        for (int i = 1; i < THREADS / 32; ++i) if (list[i] > best) best = list[i];
        if (tid == 0) top[r] = best;
        if (best == 0) break;
        limit = best;
      }
    }
  }
  __syncthreads();
  u64* chosen = top;
  if (p.cluster > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    if (rank == 0) {
      if (tid == 0) {
        Sums t = cta_sums;
        for (int r = 1; r < p.cluster; ++r) join(t, *cl.map_shared_rank(&cta_sums, r), c);
        warp_sums[0] = t;
      }
      if (TOPK) {
        const int n = p.cluster * p.k;
        for (int i = tid; i < n; i += THREADS) list[i] = cl.map_shared_rank(top, i / p.k)[i % p.k];
        __syncthreads();
        rank_into(list, n, p.k, merged);
        chosen = merged;
      }
    }
    cl.sync();            // no CTA leaves while its shared memory is read
    if (rank != 0) return;
    if (tid == 0) cta_sums = warp_sums[0];
    __syncthreads();
  }
  const Sums total = cta_sums;
  const bool none = total.m == -INFINITY, broken = !(total.m < INFINITY);     // +inf and NaN
  const float log2s = broken ? NAN : none ? 0.f : log2f(total.s);
  const float m = none ? 0.f : total.m;
  if (tid == 0) {
    const long long t = p.targets[row];
    float lp = 0.f;
    if (t >= 0 && t < p.V) lp = log_of(Vec<T>::load(z + t), m, c, log2s);
    p.logp[row] = lp;
    p.entropy[row] = none ? 0.f : (log2s - total.w / total.s) * 0.6931471805599453f;
    p.stats[row] = make_float2(total.m, log2s);
  }
  if (TOPK && tid < p.k) {
    const u64 cand = chosen[tid];
    p.top_logp[(long long)row * p.k + tid] = log_of(candidate_value(cand), m, c, log2s);
    p.top_ids[(long long)row * p.k + tid] = candidate_index(cand);
  }
}

// One thread handles UNROLL vectors of a row; the row's five numbers are the same for the whole CTA.  `dz` may be
// the logits themselves.
template <typename T>
__global__ void __launch_bounds__(THREADS)
backward_kernel(const T* logits, long long ld, const long long* __restrict__ targets,
                const float2* __restrict__ stats, const float* __restrict__ entropy, const float* __restrict__ d_logp,
                const float* __restrict__ d_entropy, T* dz, long long dz_ld, int V, int pieces, float c,
                float inv_t) {
  constexpr int N = Vec<T>::N;
  const int row = blockIdx.x / pieces, piece = blockIdx.x - row * pieces, tid = threadIdx.x;
  const T* z = logits + (long long)row * ld;
  T* g = dz + (long long)row * dz_ld;
  const float2 st = stats[row];
  const bool none = st.x == -INFINITY;
  const float m = none ? 0.f : st.x;
  const long long t64 = targets[row];
  const int t = t64 >= 0 && t64 < V && !none ? (int)t64 : -1;
  const float gl = (t64 >= 0 && t64 < V && d_logp) ? d_logp[row] : 0.f, gh = d_entropy ? d_entropy[row] : 0.f;
  // p (log p + H) = p (v ln 2 + H) with v = log2 p: dz = -(p / T) (a + b v), a = g_l + g_H H, b = g_H ln 2
  const float a = none ? 0.f : gl + gh * entropy[row], b = none ? 0.f : gh * 0.6931471805599453f;
  auto grad = [&](float f, int idx) {
    const float v = max_nan((f - m) * c - st.y, FLOOR);
    const float pr = exp2_fast(v);
    float r = -pr * fmaf(b, v, a);
    if (idx == t) r += gl;
    return r * inv_t;
  };
  const int head = min(V, (int)(((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) / sizeof(T)));
  const int nv = (V - head) / N;
  const bool aligned = (reinterpret_cast<uintptr_t>(z + head) & 15) == 0;
  const int base = piece * THREADS * UNROLL + tid;
  uint4 raw[UNROLL];
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    const int i = base + j * THREADS;
    if (i < nv) {
      if (aligned) {
        raw[j] = load_once(z + head + (long long)i * N);
      } else {
        T tmp[N];
#pragma unroll
        for (int e = 0; e < N; ++e) tmp[e] = z[head + (long long)i * N + e];
        memcpy(&raw[j], tmp, 16);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < UNROLL; ++j) {
    const int i = base + j * THREADS;
    if (i < nv) {
      float f[N];
      Vec<T>::unpack(raw[j], f);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = grad(f[e], head + i * N + e);
      *reinterpret_cast<uint4*>(g + head + (long long)i * N) = Vec<T>::pack(f);
    }
  }
  const int tail = V - head - nv * N;
  if (piece == 0 && tid < head + tail) {
    const int idx = tid < head ? tid : nv * N + tid;
    g[idx] = Vec<T>::cast(grad(Vec<T>::load(z + idx), idx));
  }
}

template <typename T>
static int run_forward(const Params& p, cudaStream_t stream) {
  auto kern = p.k > 0 ? forward_kernel<T, true> : forward_kernel<T, false>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)p.rows * p.cluster));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster > 1 ? 1 : 0;
  if (p.cluster > 8) OB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  return (int)cudaLaunchKernelEx(&cfg, kern, p);
}

// CTAs that share a row: enough for a few waves of the 148 SMs, but not less than one full batch of loads each.
static int pick_cluster(int rows, int V, int vec) {
  int cl = 1;
  while (cl < MAX_CLUSTER && (long long)rows * cl < 148 * 6 && V / (cl * 2) >= THREADS * vec) cl *= 2;
  return cl;
}

}  // namespace logprobs
}  // namespace ob

using namespace ob::logprobs;

// dtype: 0 = bf16, 1 = fp16, 2 = fp32 (also of the gradient).
extern "C" int ob_logprobs_fwd(const void* logits, long long ld, int dtype, const void* targets, void* logp, void* entropy,
                               void* stats, void* top_logp, void* top_ids, int rows, int V, int top_k, double temperature,
                               cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || top_k < 0 || top_k > MAX_TOPK || top_k > V || !(temperature > 0.0)) return -1;
  const int cl = pick_cluster(rows, V, dtype == 2 ? 4 : 8);
  if ((long long)rows * cl > 0x7fffffffLL) return -1;
  const Params p{logits, ld, (const long long*)targets, (float*)logp, (float*)entropy, (float2*)stats, (float*)top_logp,
                 (long long*)top_ids, rows, V, top_k, cl, (float)(1.4426950408889634 / temperature)};
  if (dtype == 0) return run_forward<__nv_bfloat16>(p, stream);
  if (dtype == 1) return run_forward<__half>(p, stream);
  if (dtype == 2) return run_forward<float>(p, stream);
  return -1;
}

extern "C" int ob_logprobs_bwd(const void* logits, long long ld, int dtype, const void* targets, const void* stats,
                               const void* entropy, const void* d_logp, const void* d_entropy, void* dz, long long dz_ld,
                               int rows, int V, double temperature, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (V <= 0 || !(temperature > 0.0)) return -1;
  const int vec = dtype == 2 ? 4 : 8;
  const int pieces = (V / vec + THREADS * UNROLL - 1) / (THREADS * UNROLL) + (V / vec == 0);
  if ((long long)rows * pieces > 0x7fffffffLL) return -1;
  const float c = (float)(1.4426950408889634 / temperature), inv_t = (float)(1.0 / temperature);
  const unsigned grid = (unsigned)((long long)rows * pieces);
#define OB_LAUNCH(T)                                                                                                  \
  backward_kernel<T><<<grid, THREADS, 0, stream>>>((const T*)logits, ld, (const long long*)targets, (const float2*)stats, \
                                                   (const float*)entropy, (const float*)d_logp, (const float*)d_entropy, \
                                                   (T*)dz, dz_ld, V, pieces, c, inv_t)
  if (dtype == 0) OB_LAUNCH(__nv_bfloat16);
  else if (dtype == 1) OB_LAUNCH(__half);
  else if (dtype == 2) OB_LAUNCH(float);
  else return -1;
#undef OB_LAUNCH
  return (int)cudaGetLastError();
}
