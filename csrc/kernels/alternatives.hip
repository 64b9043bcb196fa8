// Log-probabilities of given tokens, entropy and the best alternatives of every row of logits, and their gradient.
//
//   m = max l, z = c (l - m), S = sum exp z, mean = sum exp(z) z / S
//   logp = z_t - log S, H = log S - mean, top_i = z_id(i) - log S
// Everything is held relative to m: a common offset of the logits costs no bits, and rows of the type's lowest value do not overflow.
// The alternatives go by the logits as they are given (equal ones by index, a NaN counts as -inf), so no rounding of z can change
// their order. A row of -inf alone has log-probabilities of -inf, no entropy and no gradient.
#include "rt_common.h"

namespace rt {
namespace alt {

constexpr int MAX_TOP = 32;

__device__ __forceinline__ float get(const bf16_t* p) { return bf2f(*p); }
__device__ __forceinline__ float get(const float* p) { return *p; }
__device__ __forceinline__ void put(bf16_t* p, float v) { *p = f2bf(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

// a value and its place as one number: larger first, equal ones by the smaller index
__device__ __forceinline__ uint64_t order(float v, int i) {
  v = fmaxf(v, -INFINITY) + 0.f;  // NaN -> -inf, -0 -> 0
  const uint32_t u = __float_as_uint(v);
  return (uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~i;
}

// of a part of the row: largest l, sum exp z, sum exp(z) z (m = -inf: nothing but -inf and NaN, which make the sums NaN)
struct Sums { float m, s, t; };
__device__ __forceinline__ Sums merge(Sums a, Sums b, float c) {
  const float m = fmaxf(a.m, b.m);
  auto part = [&](Sums& p) {
    if (p.m == m || p.m == -INFINITY) return;
    const float d = c * (p.m - m), e = __expf(d);
    p.t = e > 0.f ? e * (p.t + d * p.s) : 0.f * p.s;  // d may be -inf
    p.s *= e;
  };
  part(a); part(b);
  return Sums{m, a.s + b.s, a.t + b.t};
}

template <typename T>
__global__ __launch_bounds__(256) void alternatives_kernel(const T* __restrict__ logits, long ld, const int64_t* __restrict__ tgt, float c,
                                                           int V, int top, float* __restrict__ logp, float* __restrict__ ent,
                                                           float* __restrict__ top_lp, int64_t* __restrict__ ids, float* __restrict__ stats) {
  __shared__ float sm[4][3];
  __shared__ uint64_t best[4];
  const long row = blockIdx.x;
  const T* const x = logits + row * ld;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  Sums a{-INFINITY, 0.f, 0.f};
  for (int i = tid; i < V; i += 256) {
    const float f = get(x + i);
    if (f != f) a.s += f;
    else if (f > -INFINITY) a = merge(a, Sums{f, f == INFINITY ? NAN : 1.f, 0.f}, c);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    a = merge(a, Sums{__shfl_xor(a.m, off, 64), __shfl_xor(a.s, off, 64), __shfl_xor(a.t, off, 64)}, c);
  if (lane == 0) { sm[wid][0] = a.m; sm[wid][1] = a.s; sm[wid][2] = a.t; }
  __syncthreads();
  a = Sums{sm[0][0], sm[0][1], sm[0][2]};
  for (int w = 1; w < 4; ++w) a = merge(a, Sums{sm[w][0], sm[w][1], sm[w][2]}, c);
  const bool none = a.m == -INFINITY && a.s == 0.f;
  const float ls = none ? 0.f : __logf(a.s), mean = none ? 0.f : a.t / a.s;
  auto log_prob = [&](float l) { return none ? -INFINITY : (l - a.m) * c - ls; };
  if (tid == 0) {
    const int64_t t = tgt ? tgt[row] : -1;
    logp[row] = t < 0 ? 0.f : t >= V ? NAN : log_prob(get(x + t));
    ent[row] = ls - mean;
    if (stats) { stats[row * 3] = none ? INFINITY : a.m; stats[row * 3 + 1] = ls; stats[row * 3 + 2] = mean; }
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < top; ++k) {  // the largest below the last one
    uint64_t b = 0;
    for (int i = tid; i < V; i += 256) {
      const uint64_t o = order(get(x + i), i);
      if (o < last && o > b) b = o;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)b, off, 64);
      b = o > b ? o : b;
    }
    __syncthreads();
    if (lane == 0) best[wid] = b;
    __syncthreads();
    last = max(max(best[0], best[1]), max(best[2], best[3]));
    if (tid == 0) {
      const int id = (int)~(uint32_t)last;
      ids[row * top + k] = id;
      top_lp[row * top + k] = log_prob(get(x + id));
    }
  }
}

// dl = c (up - p (sum up) - g_H p (z - mean)), up: the given token's and the alternatives' gradients at their places
template <typename T>
__global__ __launch_bounds__(256) void alternatives_bwd_kernel(const T* __restrict__ logits, long ld, const int64_t* __restrict__ tgt, float c,
                                                               int V, int top, const int64_t* __restrict__ ids,
                                                               const float* __restrict__ stats, const float* __restrict__ g_lp,
                                                               const float* __restrict__ g_ent, const float* __restrict__ g_top,
                                                               T* __restrict__ d, long ldd) {
  __shared__ int at[MAX_TOP + 1];
  __shared__ float up[MAX_TOP + 1];
  const long row = blockIdx.x;
  const T* const x = logits + row * ld;
  T* const dx = d + row * ldd;
  const int tid = threadIdx.x;
  const float m = stats[row * 3], ls = stats[row * 3 + 1], mean = stats[row * 3 + 2];
  if (tid <= top) {
    const int64_t t = tgt ? tgt[row] : -1;
    const bool given = tid < top || (t >= 0 && t < V);
    at[tid] = !given ? -1 : tid < top ? (int)ids[row * top + tid] : (int)t;
    up[tid] = !given ? 0.f : tid < top ? (g_top ? g_top[row * top + tid] : 0.f) : (g_lp ? g_lp[row] : 0.f);
  }
  __syncthreads();
  float total = 0.f;
  for (int k = 0; k <= top; ++k) total += up[k];
  const float ge = g_ent ? g_ent[row] : 0.f;
  const bool none = m == INFINITY && ls == 0.f;
  for (int i = tid; i < V; i += 256) {
    const float z = (get(x + i) - m) * c, p = __expf(z - ls);
    float o = z == -INFINITY ? 0.f : -p * (total + ge * (z - mean));
    for (int k = 0; k <= top; ++k)
      if (at[k] == i) o += up[k];
    put(dx + i, none ? 0.f : o * c);
  }
}

}  // namespace alt
}  // namespace rt

using namespace rt;
using namespace rt::alt;

extern "C" int rt_alternatives(int f32, const void* logits, long ld, const int64_t* tgt, float c, long T, int V, int top, float* logp, float* ent,
                               float* top_lp, int64_t* ids, float* stats, hipStream_t stream) {
  if (T == 0) return 0;
  if (top < 1 || top > MAX_TOP || top > V) return -1;
  if (f32)
    hipLaunchKernelGGL(alternatives_kernel<float>, dim3(T), dim3(256), 0, stream, (const float*)logits, ld, tgt, c, V, top, logp, ent, top_lp,
                       ids, stats);
  else
    hipLaunchKernelGGL(alternatives_kernel<bf16_t>, dim3(T), dim3(256), 0, stream, (const bf16_t*)logits, ld, tgt, c, V, top, logp, ent, top_lp,
                       ids, stats);
  RT_LAUNCH_CHECK();
  return 0;
}

extern "C" int rt_alternatives_bwd(int f32, const void* logits, long ld, const int64_t* tgt, float c, long T, int V, int top, const int64_t* ids,
                                   const float* stats, const float* g_lp, const float* g_ent, const float* g_top, void* d, long ldd,
                                   hipStream_t stream) {
  if (T == 0) return 0;
  if (top < 1 || top > MAX_TOP || top > V) return -1;
  if (f32)
    hipLaunchKernelGGL(alternatives_bwd_kernel<float>, dim3(T), dim3(256), 0, stream, (const float*)logits, ld, tgt, c, V, top, ids, stats, g_lp,
                       g_ent, g_top, (float*)d, ldd);
  else
    hipLaunchKernelGGL(alternatives_bwd_kernel<bf16_t>, dim3(T), dim3(256), 0, stream, (const bf16_t*)logits, ld, tgt, c, V, top, ids, stats,
                       g_lp, g_ent, g_top, (bf16_t*)d, ldd);
  RT_LAUNCH_CHECK();
  return 0;
}
