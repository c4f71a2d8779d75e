// Writes keys and values into a cache of e4m3 codes with one power-of-two scale for each block of tokens and head.
//
//   new      [B, T, Hk, hd]   bf16 / fp16 / fp32, any batch / token / head strides
//   cache    logical [B, capacity, Hk, hd] codes with any batch / token / head strides
//   scale    [B, Hk, blocks]  fp32
//
// Sequence b holds lens[b] tokens afterwards; the last n_new[b] of them are new[b, :n_new[b]].  One CTA owns one
// block of one head of one sequence (keys or values), so no two CTAs touch the same codes or scale: it reads the
// block's new rows once into registers, takes the largest finite magnitude, and writes codes and scale.  A block that
// already held tokens keeps its scale unless the new rows need a larger one; then the held rows are rounded again at
// the larger scale in the same CTA.  The kernel is bound by the stream of new rows (2 or 4 bytes read and 1 written
// per element); the CTA has one thread per 64 elements of a full block, so each thread has all its loads in flight.
// 8 prompts of up to 8192 tokens, 8 heads of 128, bf16: 40 us for 239 MB, 0.92 of the measured copy bandwidth (47 us
// while a chunk's row, bounds and address were computed anew each time: 12.5 instructions per element instead of 9.5).
// With half as many elements per thread 50 us, with several blocks per CTA 52 us and more.
#include "kv_fp8.cuh"
#include <string.h>

namespace ob {
namespace kvfp8 {

constexpr int CHUNKS = 8;      // chunks of 8 elements per thread
constexpr int ONE_WARPS = 4;   // rows per CTA when every sequence gets one token

// PER elements of a row per lane
template <int PER>
__device__ __forceinline__ void load_row(float (&x)[PER], const float* p) {
  if constexpr (PER == 1) x[0] = *p;
  else
#pragma unroll
    for (int i = 0; i < PER; i += 2) {
      const float2 v = *reinterpret_cast<const float2*>(p + i);
      x[i] = v.x; x[i + 1] = v.y;
    }
}
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float2 to_float2(uint32_t w, const __nv_bfloat16*) { return unpack_bf16x2(w); }
__device__ __forceinline__ float2 to_float2(uint32_t w, const __half*) { return half2_to_float2(w); }
template <int PER, typename T>
__device__ __forceinline__ void load_row(float (&x)[PER], const T* p) {
  if constexpr (PER == 1) x[0] = to_float(*p);
  else {
    uint32_t w[PER / 2];
    if constexpr (PER == 8) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
    else if constexpr (PER == 4) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) {
      const float2 v = to_float2(w[i], p);
      x[2 * i] = v.x; x[2 * i + 1] = v.y;
    }
  }
}
template <int PER>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[PER]) {
  if constexpr (PER == 1) *p = (uint8_t)to_codes(x[0], 0.f);
  else if constexpr (PER == 2) *reinterpret_cast<uint16_t*>(p) = (uint16_t)to_codes(x[0], x[1]);
  else
#pragma unroll
    for (int i = 0; i < PER; i += 4)
      *reinterpret_cast<uint32_t*>(p + i) = to_codes(x[i], x[i + 1]) | to_codes(x[i + 2], x[i + 3]) << 16;
}
template <int PER>
__device__ __forceinline__ void load_codes(float (&x)[PER], const uint8_t* p) {
  if constexpr (PER <= 2) {
    const float2 v = half2_to_float2(to_half2(PER == 1 ? *p : *reinterpret_cast<const uint16_t*>(p)));
    x[0] = v.x;
    if constexpr (PER == 2) x[1] = v.y;
  } else
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p + i);
      const float2 a = half2_to_float2(to_half2(w)), b = half2_to_float2(to_half2_hi(w));
      x[i] = a.x; x[i + 1] = a.y; x[i + 2] = b.x; x[i + 3] = b.y;
    }
}

// Eight elements.  abs_max: the largest magnitude as fp32 bits, which order infinities (and, where NaN is not passed
// over, NaN) above every number.
struct Chunk16 {
  uint4 u;
  __device__ void load(const void* p) { u = *static_cast<const uint4*>(p); }
  __device__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ uint32_t word(int i) const { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }
  __device__ uint32_t magnitude(int i) const { return word(i) & 0x7fff7fffu; }
  __device__ void poison16(uint32_t inf) {         // infinities become NaN
    uint32_t* w = &u.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((w[i] & 0x7fffu) == inf) w[i] |= 1u;
      if ((w[i] >> 16 & 0x7fffu) == inf) w[i] |= 0x10000u;
    }
  }
};
template <typename T> struct Chunk;
template <> struct Chunk<__nv_bfloat16> : Chunk16 {
  __device__ void poison() { poison16(0x7f80u); }
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {      // NaN gives way to a number
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ uint32_t abs_max() const {
    const uint32_t w = max2(max2(magnitude(0), magnitude(1)), max2(magnitude(2), magnitude(3)));
    return __float_as_uint(fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)));
  }
  __device__ float2 pair(int i) const { return make_float2(__uint_as_float(word(i) << 16), __uint_as_float(word(i) & 0xffff0000u)); }
};
template <> struct Chunk<__half> : Chunk16 {
  __device__ void poison() { poison16(0x7c00u); }
  __device__ static uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  __device__ uint32_t abs_max() const {
    const float2 f = half2_to_float2(max2(max2(magnitude(0), magnitude(1)), max2(magnitude(2), magnitude(3))));
    return __float_as_uint(fmaxf(f.x, f.y));
  }
  __device__ float2 pair(int i) const { return half2_to_float2(word(i)); }
};
template <> struct Chunk<float> {
  float4 a, b;
  __device__ void load(const void* p) {
    a = static_cast<const float4*>(p)[0];
    b = static_cast<const float4*>(p)[1];
  }
  __device__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ void poison() {
    float* f = &a.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) if (isinf(f[i])) f[i] = NAN;
    f = &b.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) if (isinf(f[i])) f[i] = NAN;
  }
  __device__ uint32_t abs_max() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = pair(i);
      m = max(m, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
    }
    return m;
  }
  __device__ float2 pair(int i) const {
    return i == 0 ? make_float2(a.x, a.y) : i == 1 ? make_float2(a.z, a.w) : i == 2 ? make_float2(b.x, b.y) : make_float2(b.z, b.w);
  }
};

template <typename T>
__global__ void __launch_bounds__(512, sizeof(T) == 4 ? 1 : 2) append_kernel(const __grid_constant__ AppendParams p) {
  __shared__ uint32_t warp_max_[2][16];
  const int tid = threadIdx.x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the attention launch may start its own set-up
  const int j = blockIdx.x, kv = blockIdx.y >= p.Hk, h = blockIdx.y - (kv ? p.Hk : 0), b = p.b0 + blockIdx.z;
  const int len = p.lens[b];
  const int n = p.n_new ? p.n_new[b] : (len == 0 ? 0 : p.T);
  const int start = len - n;
  if (n < 0 || n > p.T || start < 0 || len > p.capacity) {       // nothing of this sequence is touched
    if (tid == 0) atomicCAS(p.status, kStatusOk, kStatusBadArgs);
    return;
  }
  const int blk = (start >> p.block_shift) + j, row0 = blk << p.block_shift;
  const int lo = max(start, row0), hi = min(len, row0 + p.block);
  if (lo >= hi) return;
  const bool holds = lo > row0;
  const T* src = static_cast<const T*>(kv ? p.v_new : p.k_new) + (long long)b * p.new_batch + (long long)h * p.new_head;
  uint8_t* dst = static_cast<uint8_t*>(kv ? p.v : p.k) + (long long)b * p.batch + (long long)h * p.head;
  float* scale = (kv ? p.v_scale : p.k_scale) + (long long)b * p.scale_batch + (long long)h * p.scale_head + blk;
  const float was = holds ? *scale : 0.f;

  // round r of the block: this thread's chunk of row `row + r * rows`
  const int rows = blockDim.x >> p.row_shift, row = row0 + (tid >> p.row_shift), col = (tid & ((1 << p.row_shift) - 1)) * 8;
  Chunk<T> c[CHUNKS];
  {
    const T* from = src + (long long)(row - start) * p.new_tok + col;
    const long long step = rows * p.new_tok;
#pragma unroll
    for (int r = 0; r < CHUNKS; ++r, from += step) {
      if ((unsigned)(row + r * rows - lo) < (unsigned)(hi - lo)) c[r].load(from);
      else c[r].zero();
    }
  }
  auto block_max = [&](uint32_t m, int buf) {
    m = __reduce_max_sync(0xffffffffu, m);
    if ((tid & 31) == 0) warp_max_[buf][tid >> 5] = m;
    __syncthreads();           // the first one also: everyone has read the old scale
    for (int w = 0; w < blockDim.x / 32; ++w) m = max(m, warp_max_[buf][w]);
    return m;
  };
  uint32_t bits = 0;
#pragma unroll
  for (int r = 0; r < CHUNKS; ++r) bits = max(bits, c[r].abs_max());
  bits = block_max(bits, 0);
  const bool special = bits >= 0x7f800000u;                       // an infinity among them, or nothing but NaN
  if (special) {
    bits = 0;
#pragma unroll
    for (int r = 0; r < CHUNKS; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = c[r].pair(e);
        if (fabsf(f.x) < INFINITY) bits = max(bits, __float_as_uint(f.x) & 0x7fffffffu);
        if (fabsf(f.y) < INFINITY) bits = max(bits, __float_as_uint(f.y) & 0x7fffffffu);
      }
#pragma unroll
    for (int r = 0; r < CHUNKS; ++r) c[r].poison();               // an infinity becomes NaN, not a large number
    bits = block_max(bits, 1);
  }
  const float now = fmaxf(needed_scale(__uint_as_float(bits)), was), inv = inverse_pow2(now);
  uint8_t* to = dst + (long long)row * p.tok + col;
  const long long step = rows * p.tok;
#pragma unroll
  for (int r = 0; r < CHUNKS; ++r) {
    if ((unsigned)(row + r * rows - lo) >= (unsigned)(hi - lo)) continue;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = fmul2(c[r].pair(e), make_float2(inv, inv));
      w[e >> 1] |= to_codes(f.x, f.y) << (16 * (e & 1));
    }
    *reinterpret_cast<uint2*>(to + r * step) = make_uint2(w[0], w[1]);
  }
  if (holds && now > was) {            // held rows at the larger scale
    const float ratio = was * inv;
#pragma unroll 1
    for (int at = row; at < lo; at += rows, to += step) {
      const uint2 old = *reinterpret_cast<const uint2*>(to);
      const uint32_t o[2] = {old.x, old.y};
      uint32_t w[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = half2_to_float2(to_half2(o[e])), g = half2_to_float2(to_half2_hi(o[e]));
        w[e] = to_codes(f.x * ratio, f.y * ratio) | to_codes(g.x * ratio, g.y * ratio) << 16;
      }
      *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
    }
  }
  if (tid == 0) *scale = now;
}

// One token per sequence (T = 1), a warp for each row: the same rules, without a block-wide step.  A latency of two
// dependent loads, 1.8 us for 64 sequences of 8 heads of 128; where the scale grows the warp rounds the held rows again one
// by one, a memory latency each: 5.0 us with 15 held rows, 8.1 with 31, 13.8 with 63.
template <typename T, int HD>
__global__ void __launch_bounds__(ONE_WARPS * 32) append_one_kernel(const __grid_constant__ AppendParams p) {
  constexpr int PER = HD / 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31;
  // item = (b * 2 + kv) * Hk + head
  const long long item = (long long)blockIdx.x * ONE_WARPS + (threadIdx.x >> 5);
  if (item >= 2LL * p.B * p.Hk) return;
  unsigned i = (unsigned)item;
  const int h = i % p.Hk; i /= p.Hk;
  const int kv = i & 1, b = i >> 1;
  const T* src = static_cast<const T*>(kv ? p.v_new : p.k_new) + (long long)b * p.new_batch + (long long)h * p.new_head;
  float x[PER];
  load_row(x, src + lane * PER);
  const int len = p.lens[b], n = p.n_new ? p.n_new[b] : len != 0;
  if (n < 0 || n > 1 || len < n || len > p.capacity) {
    if (lane == 0) atomicCAS(p.status, kStatusOk, kStatusBadArgs);
    return;
  }
  if (n == 0) return;
  const int pos = len - 1, blk = pos >> p.block_shift, row0 = blk << p.block_shift;
  uint8_t* dst = static_cast<uint8_t*>(kv ? p.v : p.k) + (long long)b * p.batch + (long long)h * p.head + lane * PER;
  float* scale = (kv ? p.v_scale : p.k_scale) + (long long)b * p.scale_batch + (long long)h * p.scale_head + blk;
  const float was = pos > row0 ? *scale : 0.f;
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const uint32_t m = __float_as_uint(x[e]) & 0x7fffffffu;
    if (m < 0x7f800000u) bits = max(bits, m);
    else x[e] = NAN;                                              // an infinity becomes NaN, not a large number
  }
  bits = __reduce_max_sync(0xffffffffu, bits);
  const float now = fmaxf(needed_scale(__uint_as_float(bits)), was), inv = inverse_pow2(now);
#pragma unroll
  for (int e = 0; e < PER; ++e) x[e] *= inv;
  store_codes(dst + (long long)pos * p.tok, x);
  if (now > was) {
    if (lane == 0) *scale = now;
    const float ratio = was * inv;
    for (int row = row0; row < pos; ++row) {                      // rows that are held, at the larger scale
      uint8_t* at = dst + (long long)row * p.tok;
      load_codes(x, at);
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] *= ratio;
      store_codes(at, x);
    }
  }
}

template <typename T>
static int launch_one(const AppendParams& p, cudaStream_t stream) {
  const unsigned grid = (unsigned)((2LL * p.B * p.Hk + ONE_WARPS - 1) / ONE_WARPS);
  if (p.hd == 32) append_one_kernel<T, 32><<<grid, ONE_WARPS * 32, 0, stream>>>(p);
  else if (p.hd == 64) append_one_kernel<T, 64><<<grid, ONE_WARPS * 32, 0, stream>>>(p);
  else if (p.hd == 128) append_one_kernel<T, 128><<<grid, ONE_WARPS * 32, 0, stream>>>(p);
  else append_one_kernel<T, 256><<<grid, ONE_WARPS * 32, 0, stream>>>(p);
  return (int)cudaGetLastError();
}

int launch_append(AppendParams p, int dtype, cudaStream_t stream) {
  if (p.B <= 0 || p.T <= 0) return 0;
  p.span = (p.T + 2 * p.block - 2) / p.block;
  p.block_shift = p.row_shift = 0;
  while ((1 << p.block_shift) < p.block) ++p.block_shift;
  while ((8 << p.row_shift) < p.hd) ++p.row_shift;
  if (p.Hk > 0x7fff || 2LL * p.B * p.Hk > 0x7fffffffLL) return -1;
  if (p.T == 1)
    return dtype == 0 ? launch_one<__nv_bfloat16>(p, stream) : dtype == 1 ? launch_one<__half>(p, stream)
         : dtype == 2 ? launch_one<float>(p, stream) : -1;
  const int threads = max(32, min(512, p.block * p.hd / (8 * CHUNKS)));
  for (p.b0 = 0; p.b0 < p.B; p.b0 += 0xffff) {
    const dim3 grid(p.span, 2 * p.Hk, min(p.B - p.b0, 0xffff));
    if (dtype == 0) append_kernel<__nv_bfloat16><<<grid, threads, 0, stream>>>(p);
    else if (dtype == 1) append_kernel<__half><<<grid, threads, 0, stream>>>(p);
    else if (dtype == 2) append_kernel<float><<<grid, threads, 0, stream>>>(p);
    else return -1;
    OB_CUDA_CHECK(cudaGetLastError());
  }
  return 0;
}

}  // namespace kvfp8
}  // namespace ob

// One block of 8-byte arguments, in this order.  dtype: 0 = bf16, 1 = fp16, 2 = fp32.  Strides of the new rows and
// scales in elements, of the cache in bytes; rows of both start on 16-byte boundaries.
struct AppendArgs {
  const void *k_new, *v_new;
  long long dtype, new_batch, new_tok, new_head;
  void *k, *v;
  long long batch, tok, head;
  float *k_scale, *v_scale;
  long long scale_batch, scale_head;
  const int *lens, *n_new;      // n_new may be null
  long long B, T, Hk, hd, capacity, block;
  int* status;
  cudaStream_t stream;
};
static_assert(sizeof(AppendArgs) == 25 * 8, "packed");

extern "C" int ob_kv_fp8_append(const void* packed) {
  AppendArgs a;
  memcpy(&a, packed, sizeof(a));
  const int hd = (int)a.hd, block = (int)a.block;
  if (a.Hk <= 0 || hd < 32 || hd > 256 || (hd & (hd - 1)) || block < 16 || block > 128 || (block & (block - 1))) return -1;
  if (a.B > 0x7fffffffLL || a.T > 0x3fffffffLL || a.capacity > 0x3fffffffLL) return -1;
  if ((a.batch | a.tok | a.head) % 16) return -2;
  return ob::kvfp8::launch_append({a.k_new, a.v_new, a.new_batch, a.new_tok, a.new_head, a.k, a.v, a.batch, a.tok, a.head,
                                   a.k_scale, a.v_scale, a.scale_batch, a.scale_head, a.lens, a.n_new, a.status, (int)a.B,
                                   (int)a.T, (int)a.Hk, hd, (int)a.capacity, block, 0, 0, 0, 0},
                                  (int)a.dtype, a.stream);
}
