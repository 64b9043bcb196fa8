// Log-probabilities of given tokens, entropy and the best alternatives of every row of logits, and their gradient.
//
//   m = max l, z = c (l - m), S = sum exp z, mean = sum exp(z) z / S
//   logp = z_t - log S, H = log S - mean, top_i = z_id(i) - log S
// Everything is held relative to m: a common offset of the logits costs no bits, and rows of the type's lowest value do not overflow.
// The alternatives go by the logits as they are given (equal ones by index, a NaN counts as -inf), so no rounding of z can change
// their order. A row of -inf alone has log-probabilities of -inf, no entropy and no gradient.
#include "rt_common.h"

#include <algorithm>

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

__device__ __forceinline__ float value(uint64_t o) {
  const uint32_t u = (uint32_t)(o >> 32);
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

// 16 bytes of a row, wherever they start: rows of an odd pitch need no copy (loads take any address)
template <typename T> struct Chunk;
template <> struct Chunk<bf16_t> {
  static constexpr int E = 8;
  static __device__ __forceinline__ void open(const u32x4& w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint32_t word(const bf16_t* p, int n, int i) {  // word i of a chunk with n elements left
    const uint32_t none = 0xff80u;  // -inf
    return (2 * i < n ? (uint32_t)p[2 * i] : none) | (2 * i + 1 < n ? (uint32_t)p[2 * i + 1] : none) << 16;
  }
};
template <> struct Chunk<float> {
  static constexpr int E = 4;
  static __device__ __forceinline__ void open(const u32x4& w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ uint32_t word(const float* p, int n, int i) { return i < n ? __float_as_uint(p[i]) : 0xff800000u; }
};
// the chunk behind the last whole one: -inf past the row
template <typename T>
__device__ __forceinline__ u32x4 load_tail(const T* x, int c, int V) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = Chunk<T>::word(x + (long)c * Chunk<T>::E, V - c * Chunk<T>::E, i);
  return w;
}
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* x, int c, int V) {
  u32x4 w;
  if ((c + 1) * Chunk<T>::E <= V) __builtin_memcpy(&w, x + (long)c * Chunk<T>::E, 16);
  else w = load_tail(x, c, V);
  return w;
}

constexpr int CAP = 512;       // candidates that are ranked at once
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// One workgroup a row, which stays in registers: NC chunks a thread (0: it does not fit, and is read again from the caches).
// The alternatives without sorting: the best of each lane's elements over the waves makes 64 numbers of which no two are equal (value,
// then place), and the top-th of them is one that at least `top` elements reach. What reaches it is a little more than `top` elements (24 of 32000
// where 20 are wanted); each counts how many of the others are before it. Where they are more than CAP (rows made for it) the
// best are taken one by one. Bound by memory with many rows (4096 x 32000 in bf16: 56 us, 4.7 TB/s), by the exp of one CU's row and a chain of
// barriers with few (8 rows: 8 us).
template <typename T, int THREADS, int NC>
__global__ __launch_bounds__(THREADS, NC ? 1 : 8) void alternatives_kernel(const T* __restrict__ logits, long ld,
                                                                           const int64_t* __restrict__ tgt, float c, int V, int top,
                                                                           float* __restrict__ logp, float* __restrict__ ent,
                                                                           float* __restrict__ top_lp, int64_t* __restrict__ ids,
                                                                           float* __restrict__ stats) {
  constexpr int E = Chunk<T>::E, NW = THREADS / 64, KEEP = NC ? NC : 1, SHARE = 64 / NW;
  __shared__ float sm[3][NW];
  __shared__ uint64_t best[THREADS], cand[CAP], group[64], tau_s;
  __shared__ int ahead[NW][64];
  __shared__ int count;
  const long row = blockIdx.x;
  const T* const x = logits + row * ld;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, chunks = (V + E - 1) / E;
  // the given token's logit, with the row: behind the sums it would be two more trips to memory
  const int64_t given = tgt ? tgt[row] : -1;
  const float given_l = get(x + (given >= 0 && given < V ? given : 0));
  u32x4 data[KEEP];
  float top_of[KEEP];
  if constexpr (NC > 0) {
    const uint32_t none = E == 8 ? 0xff80ff80u : 0xff800000u;  // -inf: counts for nothing
    const int full = V / E;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int ch = k * THREADS + tid;
      data[k] = u32x4{none, none, none, none};
      if (ch < full) __builtin_memcpy(&data[k], x + (long)ch * E, 16);
    }
    if (full < chunks && tid == full % THREADS) {
      const u32x4 w = load_tail(x, full, V);
#pragma unroll
      for (int k = 0; k < NC; ++k)
        if (k == full / THREADS) data[k] = w;
    }
  }
  // f(turn, chunk, its elements) for the thread's chunks in order
  auto each = [&](auto f) {
    if constexpr (NC > 0) {
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        if (k * THREADS >= chunks) break;
        asm volatile("" : "+v"(data[k]));  // opened anew in each pass: kept open it takes twice the registers
        f(k, k * THREADS + tid, data[k]);
      }
    } else {
      int ch = tid;
      for (; ch + 3 * THREADS < V / E; ch += 4 * THREADS) {
        u32x4 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) __builtin_memcpy(&w[k], x + (long)(ch + k * THREADS) * E, 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) f(0, ch + k * THREADS, w[k]);
      }
      for (; ch < chunks; ch += THREADS) f(0, ch, load_chunk(x, ch, V));
    }
  };
  // the row's largest, and each thread's with the chunk where it lies
  float mine = -INFINITY;
  int where = tid;
  each([&](int k, int ch, const u32x4& w) {
    float f[E];
    Chunk<T>::open(w, f);
    float mx = -INFINITY;  // a NaN counts as this
#pragma unroll
    for (int i = 0; i < E; ++i) mx = fmaxf(mx, f[i]);
    top_of[k] = mx;
    if (mx > mine) { mine = mx; where = ch; }
  });
  best[tid] = tid < chunks ? order(mine, where) : 0;
  const float wm = wave_max(mine);
  if (lane == 0) sm[0][wid] = wm;
  if (tid == 0) count = 0;
  __syncthreads();
  float m = sm[0][0];
#pragma unroll
  for (int w = 1; w < NW; ++w) m = fmaxf(m, sm[0][w]);
  // the sums, in steps of log 2
  const float c2 = c * LOG2E, ref = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
  each([&](int, int, const u32x4& w) {
    float f[E];
    Chunk<T>::open(w, f);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float z = (f[i] - ref) * c2, e = __builtin_amdgcn_exp2f(z);
      s += e;
      t = fmaf(e, fmaxf(z, -1e30f), t);  // 0 for an element of -inf
    }
  });
  s = wave_sum(s);
  t = wave_sum(t);
  if (lane == 0) { sm[1][wid] = s; sm[2][wid] = t; }
  // the bound for the alternatives: each wave counts a share of the lanes' best that are before each lane's
  {
    uint64_t b = best[lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) b = max(b, best[w * 64 + lane]);
    const uint32_t lo = (uint32_t)b, hi = (uint32_t)(b >> 32);
    int before = 0;
#pragma unroll
    for (int i = 0; i < SHARE; ++i) {
      const int j = wid * SHARE + i;
      const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane(hi, j) << 32 | (uint32_t)__builtin_amdgcn_readlane(lo, j);
      before += o > b;
    }
    ahead[wid][lane] = before;
    if (wid == 0) group[lane] = b;
  }
  __syncthreads();
  s = sm[1][0];
  t = sm[2][0];
#pragma unroll
  for (int w = 1; w < NW; ++w) { s += sm[1][w]; t += sm[2][w]; }
  const bool none = m == -INFINITY && s == 0.f;
  const float ls = none ? 0.f : __logf(s), mean = none ? 0.f : t / s * LN2;
  auto log_prob = [&](float l) { return none ? -INFINITY : (l - ref) * c2 * LN2 - ls; };
  if (tid == 0) {
    logp[row] = given < 0 ? 0.f : given >= V ? NAN : log_prob(given_l);
    ent[row] = ls - mean;
    if (stats) { stats[row * 3] = none ? INFINITY : ref; stats[row * 3 + 1] = ls; stats[row * 3 + 2] = mean; }
  }
  if (wid == 0) {
    int before = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) before += ahead[w][lane];
    const uint64_t b = group[lane];
    // fewer lanes with elements than alternatives: everything is ranked
    if (__popcll(__ballot(b != 0)) < top) tau_s = 0;
    else if (before == top - 1) tau_s = b;
  }
  __syncthreads();
  const uint64_t tau = tau_s;
  const float tv = tau ? value(tau) : -INFINITY;
  const int tch = tau ? (int)~(uint32_t)tau : chunks;  // elements of value tv count up to this chunk
  auto look = [&](int ch, const u32x4& w) {
    float f[E];
    Chunk<T>::open(w, f);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float v = f[i] == f[i] ? f[i] : -INFINITY;
      if ((v > tv || (v == tv && ch <= tch)) && ch * E + i < V) {
        const int at = atomicAdd(&count, 1);
        if (at < CAP) cand[at] = order(v, ch * E + i);
      }
    }
  };
  if constexpr (NC > 0) {
    // a thread's chunks that reach the bound, seldom more than one: all threads of a wave look into theirs at once, read anew since
    // registers have no index (20 of 32000 over 4096 rows took a twelfth less than with a look into the registers turn by turn)
    unsigned hits = 0;
    const int q = tch >= tid ? (tch - tid) / THREADS : -1;
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (k * THREADS < chunks) hits |= (top_of[k] > tv || (top_of[k] == tv && k <= q) ? 1u : 0u) << k;
    for (; hits; hits &= hits - 1) {
      const int ch = __builtin_ctz(hits) * THREADS + tid;
      if (ch < chunks) look(ch, load_chunk(x, ch, V));
    }
  } else {
    each([&](int, int ch, const u32x4& w) { look(ch, w); });
  }
  __syncthreads();
  const int n = count;
  if (n <= CAP) {
    for (int i = tid; i < n; i += THREADS) {
      const uint64_t o = cand[i];
      int before = 0;
      int j = 0;
      for (; j + 8 <= n; j += 8) {  // eight under way: they come one by one otherwise, 50 of them in a microsecond
        uint64_t c8[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) c8[q] = cand[j + q];
#pragma unroll
        for (int q = 0; q < 8; ++q) before += c8[q] > o;
      }
      for (; j < n; ++j) before += cand[j] > o;
      if (before < top) {
        ids[row * top + before] = (int)~(uint32_t)o;
        top_lp[row * top + before] = log_prob(value(o));
      }
    }
    return;
  }
  uint64_t last = ~0ull;
  for (int q = 0; q < top; ++q) {  // the largest behind the last one
    uint64_t b = 0;
    for (int i = tid; i < V; i += THREADS) {
      const uint64_t o = order(get(x + i), i);
      if (o < last && o > b) b = o;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) b = max(b, (uint64_t)__shfl_xor((unsigned long long)b, off, 64));
    __syncthreads();
    if (lane == 0) best[wid] = b;
    __syncthreads();
    last = best[0];
#pragma unroll
    for (int w = 1; w < NW; ++w) last = max(last, best[w]);
    if (tid == 0) {
      ids[row * top + q] = (int)~(uint32_t)last;
      top_lp[row * top + q] = log_prob(value(last));
    }
  }
}

// dl = c (up - p (sum up) - g_H p (z - mean)), up: the given token's and the alternatives' gradients at their places. A row is read and
// written once; the places with gradients of their own, 33 at most, are written again behind the chunks that hold them. Bound by
// memory (2048 x 32002 in bf16: 44 us, 6 TB/s read and written, part of it from the cache that the forward filled).
template <typename T>
__global__ __launch_bounds__(256) void alternatives_bwd_kernel(const T* __restrict__ logits, long ld, const int64_t* __restrict__ tgt, float c,
                                                               int V, int top, const int64_t* __restrict__ ids,
                                                               const float* __restrict__ stats, const float* __restrict__ g_lp,
                                                               const float* __restrict__ g_ent, const float* __restrict__ g_top,
                                                               T* d, long ldd, int span) {
  constexpr int E = Chunk<T>::E;
  __shared__ float total_s;
  const long row = blockIdx.x;
  const T* const x = logits + row * ld;
  T* const dx = d + row * ldd;
  const int tid = threadIdx.x, chunks = (V + E - 1) / E, full = V / E;
  const int first = blockIdx.y * span, last = min(first + span, chunks), whole = min(last, full);
  u32x4 w[4];  // the first four chunks, on their way while the row's gradients are added
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k] = u32x4{};
    if (full) __builtin_memcpy(&w[k], x + (long)min(first + tid + k * 256, full - 1) * E, 16);
  }
  const float m = stats[row * 3], ls = stats[row * 3 + 1], mean = stats[row * 3 + 2];
  int place = -1;
  float up = 0.f, at_place = 0.f;
  if (tid < 64) {
    if (tid <= top) {
      const int64_t t = tid < top ? ids[row * top + tid] : tgt ? tgt[row] : -1;
      place = t >= 0 && t < V ? (int)t : -1;
      up = place < 0 ? 0.f : tid < top ? (g_top ? g_top[row * top + tid] : 0.f) : (g_lp ? g_lp[row] : 0.f);
      at_place = get(x + max(place, 0));
    }
    const float total = wave_sum(up);
    if (tid == 0) total_s = total;
    // a given token that is among the alternatives adds to its place there
    const int given = __builtin_amdgcn_readlane(place, top);
    const float given_up = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(up), top));
    const bool among = tid < top && place == given && given >= 0;
    if (among) up += given_up;
    if (__any(among) && tid == top) place = -1;
  }
  __syncthreads();
  const float total = total_s, ge = g_ent ? g_ent[row] : 0.f, c2 = c * LOG2E, ls2 = ls * LOG2E;
  const bool none = m == INFINITY && ls == 0.f;
  // -c p (total + g_H (z - mean)) with z in steps of log 2
  const float k1 = none ? 0.f : -c * (total - ge * mean), k2 = none ? 0.f : -c * ge * LN2;
  auto slope = [&](float l) {
    const float z = (l - m) * c2;
    return __builtin_amdgcn_exp2f(z - ls2) * fmaf(k2, fmaxf(z, -1e30f), k1);
  };
  auto one = [&](int ch, const u32x4& in) {
    float f[E];
    Chunk<T>::open(in, f);
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = slope(f[i]);
    if constexpr (E == 8) {
      const uint4 out = pack8(f);
      __builtin_memcpy(dx + (long)ch * E, &out, 16);
    } else {
      __builtin_memcpy(dx + (long)ch * E, f, 16);
    }
  };
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (first + tid + k * 256 < whole) one(first + tid + k * 256, w[k]);
  int ch = first + tid + 4 * 256;
  for (; ch + 3 * 256 < whole; ch += 4 * 256) {
#pragma unroll
    for (int k = 0; k < 4; ++k) __builtin_memcpy(&w[k], x + (long)(ch + k * 256) * E, 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) one(ch + k * 256, w[k]);
  }
  for (; ch < whole; ch += 256) {
    __builtin_memcpy(&w[0], x + (long)ch * E, 16);
    one(ch, w[0]);
  }
  if (last > full && tid < V - full * E) put(dx + full * E + tid, slope(get(x + full * E + tid)));  // less than a chunk
  __syncthreads();
  if (place >= first * E && place < last * E) put(dx + place, none ? 0.f : fmaf(c, up, slope(at_place)));
}

}  // namespace alt
}  // namespace rt

using namespace rt;
using namespace rt::alt;

template <typename T>
static int launch_alternatives(const T* x, long ld, const int64_t* tgt, float c, long rows, int V, int top, float* logp, float* ent, float* top_lp,
                               int64_t* ids, float* stats, hipStream_t stream) {
  const int chunks = (V + Chunk<T>::E - 1) / Chunk<T>::E;
#define ALT(THREADS, NC)                                                                                                                 \
  hipLaunchKernelGGL((alternatives_kernel<T, THREADS, NC>), dim3((unsigned)rows), dim3(THREADS), 0, stream, x, ld, tgt, c, V, top, logp, ent, \
                     top_lp, ids, stats)
  // up to a row a CU as many threads as the row feeds (8 rows of 32000 in bf16 8.9 us, with 256 threads 9.6); beyond, rows of 256 and 512 threads that
  // share a CU and wait at different times (300 rows 14.3 us, with 1024 threads 17.1; 1000 rows 22.6 and 35)
  const bool few = rows <= num_cus();
  if (chunks <= 256 * 4) ALT(256, 4);
  else if (few && chunks <= 1024 * 4) ALT(1024, 4);
  else if (!few && chunks <= 256 * 16) ALT(256, 16);
  else if (!few && chunks <= 512 * 16) ALT(512, 16);
  else if (chunks <= 1024 * 8) ALT(1024, 8);
  else if (chunks <= 1024 * 16) ALT(1024, 16);
  else ALT(1024, 0);
#undef ALT
  RT_LAUNCH_CHECK();
  return 0;
}

extern "C" int rt_alternatives(int f32, const void* logits, long ld, const int64_t* tgt, float c, long T, int V, int top, float* logp, float* ent,
                               float* top_lp, int64_t* ids, float* stats, hipStream_t stream) {
  if (T == 0) return 0;
  if (top < 1 || top > MAX_TOP || top > V) return -1;
  return f32 ? launch_alternatives((const float*)logits, ld, tgt, c, T, V, top, logp, ent, top_lp, ids, stats, stream)
             : launch_alternatives((const bf16_t*)logits, ld, tgt, c, T, V, top, logp, ent, top_lp, ids, stats, stream);
}

template <typename T>
static int launch_alternatives_bwd(const T* x, long ld, const int64_t* tgt, float c, long rows, int V, int top, const int64_t* ids,
                                   const float* stats, const float* g_lp, const float* g_ent, const float* g_top, T* d, long ldd,
                                   hipStream_t stream) {
  // a row goes to several workgroups where rows are few: eight of them a CU, with four chunks a thread at least (333 x 50272 in fp32 72 -> 28 us)
  const int chunks = (V + Chunk<T>::E - 1) / Chunk<T>::E;
  const int parts = (int)std::max(1L, std::min((8L * num_cus() + rows - 1) / rows, (long)(chunks + 1023) / 1024));
  const int span = ((chunks + parts - 1) / parts + 255) / 256 * 256;
  hipLaunchKernelGGL(alternatives_bwd_kernel<T>, dim3((unsigned)rows, (unsigned)((chunks + span - 1) / span)), dim3(256), 0, stream, x, ld, tgt, c,
                     V, top, ids, stats, g_lp, g_ent, g_top, d, ldd, span);
  RT_LAUNCH_CHECK();
  return 0;
}

extern "C" int rt_alternatives_bwd(int f32, const void* logits, long ld, const int64_t* tgt, float c, long T, int V, int top, const int64_t* ids,
                                   const float* stats, const float* g_lp, const float* g_ent, const float* g_top, void* d, long ldd,
                                   hipStream_t stream) {
  if (T == 0) return 0;
  if (top < 1 || top > MAX_TOP || top > V) return -1;
  return f32 ? launch_alternatives_bwd((const float*)logits, ld, tgt, c, T, V, top, ids, stats, g_lp, g_ent, g_top, (float*)d, ldd, stream)
             : launch_alternatives_bwd((const bf16_t*)logits, ld, tgt, c, T, V, top, ids, stats, g_lp, g_ent, g_top, (bf16_t*)d, ldd, stream);
}
