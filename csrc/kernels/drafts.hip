// Checking drafted tokens: the plan of a batch's token trees, attention of their nodes over the K/V cache, and the path that the
// model agrees with, appended to the cache of every layer. Up to 64 nodes a row: a node's ancestors are one 64-bit word, and a
// wave holds a row's tree with one node to a lane.
#include "rt_common.h"
#include "rt_paged.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace rt {
namespace drafts {

using paged::ld;
using paged::st;

constexpr int NODES = 64;

__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
  const uint32_t lo = __shfl((uint32_t)v, lane, 64), hi = __shfl((uint32_t)(v >> 32), lane, 64);
  return (uint64_t)hi << 32 | lo;
}

// ---------------------------------------------------------------------------------------------
// the plan: see[i] = bit i | see[parent[i]], pos[i] = pos0 + ancestors. Pointer doubling, 1, 2, 4, ... ancestors a round.
// ---------------------------------------------------------------------------------------------
__global__ __launch_bounds__(64) void draft_tree_kernel(const int* __restrict__ parent, const int* __restrict__ nodes,
                                                        const int* __restrict__ pos0, int N, int64_t* __restrict__ see,
                                                        int* __restrict__ pos) {
  const int b = blockIdx.x, i = threadIdx.x;
  const int n = nodes ? min(nodes[b], N) : N;
  int p = i < n ? parent[(long)b * N + i] : -1;
  if (p < 0 || p >= i) p = i;  // a root
  uint64_t s = 1ull << i;
#pragma unroll
  for (int r = 0; r < 6; ++r) {
    s |= lane64(s, p);
    p = __shfl(p, p, 64);
  }
  if (i < N) {
    see[(long)b * N + i] = i < n ? (int64_t)s : 0;
    pos[(long)b * N + i] = (pos0 ? pos0[b] : 0) + (i < n ? __popcll(s) - 1 : 0);
  }
}

// ---------------------------------------------------------------------------------------------
// attention, any size and type: one workgroup per (node, head, row), 256 keys at a time
// ---------------------------------------------------------------------------------------------
struct TreeArgs {
  const void* qkv; long ldq;            // [B N, (Hq + 2 Hkv) D] rotated rows of the nodes
  const void* kc; const void* vc;       // [B, Hkv, Smax, D]
  const float* ksc; const float* vsc; int SmaxP;  // scales [B, Hkv, SmaxP] of caches in e4m3 (keys' bytes in the order that decoding reads), or null
  const int* kv_len; const int* kv_start;
  const int64_t* see;                   // [B, N]
  void* o; long ldo;
  int B, N, Hq, Hkv, D, Smax, window;   // window 0: none
  float scale;
  int G; float per_G;                   // Hq / Hkv and 1 / G
  int sorted, blocks;                   // long rows first; workgroups for a key head's rows
  float part_cost, join_cost;           // in stages
  float* part; int S;                   // partials of at most S shares of a row's keys (part_of)
};

// the nodes that node i of row b sees; bits past the tree count for nothing
__device__ __forceinline__ uint64_t word(const TreeArgs& a, int b, int i) { return (uint64_t)a.see[(long)b * a.N + i] & ~0ull >> (NODES - a.N); }

template <typename T>
__global__ __launch_bounds__(256) void tree_any_kernel(TreeArgs a) {
  extern __shared__ float sm[];  // q [D], acc [D], p [256], sbuf [4]
  float* qs = sm;
  float* acc = qs + a.D;
  float* ps = acc + a.D;
  float* sbuf = ps + 256;
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, gh = h / (a.Hq / a.Hkv);
  const uint64_t mine = word(a, b, i);
  const T* const x = (const T*)a.qkv + (long)b * a.N * a.ldq;
  T* const o = (T*)a.o + ((long)b * a.N + i) * a.ldo + (long)h * a.D;
  const int depth = __popcll(mine) - 1, len = min(max(a.kv_len[b], 0), a.Smax);
  int lo = a.kv_start ? max(a.kv_start[b], 0) : 0;
  if (a.window) lo = max(lo, len + depth - a.window + 1);
  const int ctx = max(len - lo, 0), n = ctx + a.N;
  uint64_t near = mine;  // nodes less than `window` places before this one; a place is how many nodes one sees
  if (a.window && depth + 1 >= a.window)
    for (int j = 0; j < a.N; ++j)
      if (depth + 1 - (int)__popcll(word(a, b, j)) >= a.window) near &= ~(1ull << j);
  if (!near && (!mine || !ctx)) {  // no node, or one that a window leaves nothing of
    for (int c = tid; c < a.D; c += 256) st(o + c, 0.f);
    return;
  }
  const T* const kc = (const T*)a.kc + ((long)b * a.Hkv + gh) * a.Smax * a.D;
  const T* const vc = (const T*)a.vc + ((long)b * a.Hkv + gh) * a.Smax * a.D;
  for (int c = tid; c < a.D; c += 256) {
    qs[c] = ld(x + (long)i * a.ldq + (long)h * a.D + c);
    acc[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  __syncthreads();
  for (int j0 = 0; j0 < n; j0 += 256) {
    const int j = j0 + tid;
    bool sees = j < ctx;
    if (j >= ctx && j < n) sees = near >> (j - ctx) & 1;
    float s = -INFINITY;
    if (sees) {
      const T* kp = j < ctx ? kc + (long)(lo + j) * a.D : x + (long)(j - ctx) * a.ldq + (long)(a.Hq + gh) * a.D;
      float d = 0.f;
      for (int c = 0; c < a.D; ++c) d = fmaf(qs[c], ld(kp + c), d);
      s = d * a.scale;
    }
    const float mn = fmaxf(m, block_max(s, sbuf));
    const float mz = mn == -INFINITY ? 0.f : mn;
    const float alpha = expf(m - mz), p = sees ? expf(s - mz) : -1.f;
    ps[tid] = p;  // -1: a key that is not seen, whatever its value holds
    l = l * alpha + block_sum(sees ? p : 0.f, sbuf);
    m = mn;
    __syncthreads();
    const int cnt = min(256, n - j0);
    for (int c = tid; c < a.D; c += 256) {
      float y = acc[c] * alpha;
      for (int k = 0; k < cnt; ++k) {
        if (ps[k] < 0.f) continue;
        const int jk = j0 + k;
        y = fmaf(ps[k], ld(jk < ctx ? vc + (long)(lo + jk) * a.D + c : x + (long)(jk - ctx) * a.ldq + (long)(a.Hq + a.Hkv + gh) * a.D + c), y);
      }
      acc[c] = y;
    }
    __syncthreads();
  }
  for (int c = tid; c < a.D; c += 256) st(o + c, acc[c] / l);
}

// ---------------------------------------------------------------------------------------------
// attention in bf16 on matrix instructions
// ---------------------------------------------------------------------------------------------
// A workgroup takes one key head of a row: its queries (node r / G, head r % G of the group for row r of G N) against a share of the
// keys, in stages of SK keys that go to LDS by DMA while the stage before is multiplied. The context comes from the cache; the nodes'
// own keys are the last stage. S^T = K Q^T and O^T = V^T P^T: a query is a lane's column in both, so its maximum and sum lie in four
// lanes, and p goes from the scores' registers to the product's as it is (rounded to the cache's type: half a step of bf16 for each term,
// the sums in fp32). WR waves share the rows, RT tiles of 16 each, WK the keys of a stage.
// Shares of a long row's keys (cut(): by the lengths, which only the device knows) leave fp32 partials that a second launch joins.
// How many of a row's stages one part takes. Parts of `per` stages cost, in stages, per + part_cost * parts + join_cost: each part writes and reads
// partials of all rows of its key head, whatever its length. Measured: 16 nodes of one row over 4096 keys in 8 key heads (65 stages) 17.1 /
// 14.9 / 13.9 / 16.0 us in 8 / 16 / 22 / 33 parts, 48 rows of 150 to 1200 keys 31 / 44 / 50 in 1 / 2 / 3.
__host__ __device__ inline int stages_per_part(int stages, int most, float part_cost, float join_cost) {
  if (most <= 1 || stages <= 1) return stages > 1 ? stages : 1;
  int per = (int)(sqrtf(stages * part_cost) + 0.5f), least = (stages + most - 1) / most;
  per = per < least ? least : per;
  const int parts = (stages + per - 1) / per;
  return parts > 1 && per + part_cost * parts + join_cost < stages ? per : stages;
}

// nodes of a row (those that see nothing lie behind them, or between them in plans of a caller's own, whose masks may name rows behind the last
// node too); every lane of a wave has to be there
__device__ __forceinline__ int count_nodes(uint64_t see) {
  const uint64_t live = __ballot(see != 0);
  int n = live ? 64 - __builtin_clzll(live) : 0;
  while (__any(n < NODES && see >> n)) ++n;
  return n;
}

// full: stages that the context fills; rest: its last keys, which go into the nodes' stage where both fit there (and are of one type)
struct Cut { int lo, len, full, rest, tiles, parts, per; };
__device__ __forceinline__ Cut cut(const TreeArgs& a, int b, int n, int SK) {
  Cut c;
  c.len = min(max(a.kv_len[b], 0), a.Smax);
  c.lo = a.kv_start ? max(a.kv_start[b], 0) : 0;
  if (a.window) c.lo = max(c.lo, c.len - a.window + 1);
  c.lo = min(c.lo, c.len);
  c.full = (c.len - c.lo) / SK;
  c.rest = (c.len - c.lo) % SK;
  c.tiles = c.full + (c.rest > (a.ksc ? 0 : SK - n) ? 2 : 1);
  c.per = stages_per_part(c.tiles, a.S, a.part_cost, a.join_cost);
  c.parts = (c.tiles + c.per - 1) / c.per;
  return c;
}

// a part of a pair's rows: of each 16 of them the accumulators as the lanes hold them [D / 16][64][4], behind all of these (m, l) of each row
__device__ __forceinline__ int tiles16(const TreeArgs& a) { return (a.N * a.G + 15) / 16; }
__device__ __forceinline__ float* part_of(const TreeArgs& a, int D, int s, long pair) {
  return a.part + ((long)s * a.B * a.Hkv + pair) * ((long)tiles16(a) * 16 * (D + 2));
}

// r / G for a row r of a key head (under 64 G, G up to 4096: the error of the product is under 64 2^-23, and 1 / 2 G is more)
__device__ __forceinline__ int node_of_row(const TreeArgs& a, int r) { return (int)((r + 0.5f) * a.per_G); }

// of the nodes in w, those less than `window` places before the node that sees w; a place is how many nodes one sees (see: the word of this lane's
// node), so one that sees fewer than `window` has none farther. Every lane of a wave has to be there.
__device__ __forceinline__ uint64_t near_nodes(uint64_t w, uint64_t see, int window) {
  const int place = __popcll(w), other = __popcll(see);
  if (window && __any(place >= window))
    for (int j = 0; j < NODES; ++j)
      if (place - __builtin_amdgcn_readlane(other, j) >= window) w &= ~(1ull << j);
  return w;
}

// the row that has q longer ones before it (64 rows at most, one a lane)
__device__ __forceinline__ int longest(const TreeArgs& a, int q, int lane) {
  const int len = lane < a.B ? min(max(a.kv_len[lane], 0), a.Smax) : -1;
  int before = 0;
  for (int j = 0; j < a.B; ++j) {
    const int other = __builtin_amdgcn_readlane(len, j);
    before += other > len || (other == len && j < lane);
  }
  return __builtin_ctzll(__ballot(lane < a.B && before == q));
}

// one v_maximum3_f32 for two of these; fmaxf has each operand made canonical first. A NaN stays one.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// 16 B at an address of LDS and 16 B `second` behind it. An ordinary read would wait for every DMA to LDS that is under way.
template <int second>
__device__ __forceinline__ void read_pair(uint32_t at, u32x4& x, u32x4& y) {
  asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)" : "=&v"(x), "=&v"(y) : "v"(at), "i"(second) : "memory");
}

// where 16 bytes c of an e4m3 value lie in its row of a stage: eight keys in turn (4 g .. + 3 and 16 behind these) use all banks
__device__ __forceinline__ int v8_chunk(int key, int c) { return c ^ ((key >> 1 & 3) | (key >> 2 & 4)); }
// columns of eight keys' bytes each, of eight chunks of 16 (at: of chunk 0)
template <int offset>
__device__ __forceinline__ void read_columns8(uint32_t at, uint2 (&v)[8]) {
  asm volatile(
      "ds_read_b64_tr_b8 %0, %8 offset:%16\n\t"
      "ds_read_b64_tr_b8 %1, %9 offset:%16\n\t"
      "ds_read_b64_tr_b8 %2, %10 offset:%16\n\t"
      "ds_read_b64_tr_b8 %3, %11 offset:%16\n\t"
      "ds_read_b64_tr_b8 %4, %12 offset:%16\n\t"
      "ds_read_b64_tr_b8 %5, %13 offset:%16\n\t"
      "ds_read_b64_tr_b8 %6, %14 offset:%16\n\t"
      "ds_read_b64_tr_b8 %7, %15 offset:%16\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(at), "v"(at ^ 16), "v"(at ^ 32), "v"(at ^ 48), "v"(at ^ 64), "v"(at ^ 80), "v"(at ^ 96), "v"(at ^ 112), "i"(offset)
      : "memory");
}

// e4m3 byte e of four
__device__ __forceinline__ float fp8_at(uint32_t four, int e) {
  typedef __attribute__((ext_vector_type(2))) float f32x2_t;
  const f32x2_t f = e < 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(four, false) : __builtin_amdgcn_cvt_pk_f32_fp8(four, true);
  return f[e & 1];
}

// the largest of 16 lanes' values, in each of them (rotations within the 16 by 8, 4, 2, 1); NaN counts as the least
__device__ __forceinline__ float largest16(float x) {
  x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x128, 0xf, 0xf, false)));
  x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x124, 0xf, 0xf, false)));
  x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x122, 0xf, 0xf, false)));
  return fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x121, 0xf, 0xf, false)));
}

// a value of a row with this scale, as the row is read once it lies in an e4m3 cache
__device__ __forceinline__ float as_stored(float v, float scale) { return fp8_at(__builtin_amdgcn_cvt_pk_fp8_f32(v * (1.f / scale), 0.f, 0, false), 0) * scale; }

// The bound: 128 registers where two workgroups of eight waves share a CU (in e4m3, with 162: rows of 128 queries took an eighth more); elsewhere 256,
// without which the compiler keeps some in the matrix cores' file and moves them in each stage (32 rows of 5 nodes, 12 heads of 64: 11.3 us, with
// it 10.7; 64 rows of 64 nodes 209 and 205).
// STORED: the nodes' keys and values count as they will be once they lie in the e4m3 cache.
template <int D, int RT, int WR, int WK, int KT, bool KV8, bool STORED>
__global__ __launch_bounds__(64 * WR * WK, WR == 4 ? 4 : 2) void tree_mfma_kernel(TreeArgs a) {
  constexpr int NW = WR * WK, SK = WK * KT, ROWS = 16 * RT * WR, KB = SK * D * 2, DS = D / 32, DT = D / 16, KS = KT / 16, NC = D / 8;
  static_assert(KB / 1024 % NW == 0 && SK >= NODES && (KV8 || !STORED) && (!KV8 || (D == 128 && SK == 64 && NW >= 2)));
  __shared__ __attribute__((aligned(128))) char smem[4 * KB];
  __shared__ __attribute__((aligned(16))) float scales[KV8 ? 4 : 1][KV8 ? 2 * SK : 1];  // of a stage's keys, and of its values
  __shared__ unsigned bad[2][2];  // keys of the first stage, and of the nodes', whose values are not all numbers
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, r16 = lane & 15, g = lane >> 4, wr = wid % WR, wk = wid / WR;
  // (part, key head, row); where several workgroups share a key head's rows, the grid is (8 x these, all of the former by eight): blocks go to
  // the eight XCDs in turn, and those that read the same keys come eight later, to the same L2
  int s = blockIdx.x, gh = blockIdx.y, b = blockIdx.z, rb = 0;
  if (a.blocks > 1) {
    const int lin = blockIdx.y * 8 + (blockIdx.x & 7), pair = lin / a.S;
    s = lin % a.S;
    gh = pair % a.Hkv;
    b = pair / a.Hkv;
    rb = blockIdx.x >> 3;
    if (b >= a.B) return;
  }
  if (a.sorted) b = longest(a, b, lane);
  const int G = a.G;
  const uint64_t see = lane < a.N ? word(a, b, lane) : 0;
  const int n = count_nodes(see), M = n * G;
  const Cut ct = cut(a, b, n, SK);
  if (s >= ct.parts) return;
  const int t0 = s * ct.per, t1 = min(t0 + ct.per, ct.tiles);
  const int row0 = rb * ROWS + wr * 16 * RT;  // of this wave
  const bf16_t* const x = (const bf16_t*)a.qkv + (long)b * a.N * a.ldq;
  const long pair_at = (long)b * a.Hkv + gh;

  if (rb * ROWS < M) {
    bf16x8 qf[RT][DS];
    uint64_t sees[RT];
    int from[RT];       // first key of the context that the row sees
    bool sees_any[RT];  // set in steps, as a mask of the wave: as one expression it costs the loop below registers (64 rows of 64 nodes 194 -> 197 us)
    const int joint = !KV8 && ct.tiles == ct.full + 1 ? ct.rest : 0;
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      const int r = min(row0 + 16 * u + r16, a.N * G - 1), node = node_of_row(a, r);
      const bf16_t* const q = x + (long)node * a.ldq + (long)(gh * G + r - node * G) * D + 8 * g;
#pragma unroll
      for (int d = 0; d < DS; ++d) qf[u][d] = *(const bf16x8*)(q + 32 * d);
      const uint64_t w = lane64(see, node);
      sees_any[u] = w != 0;
      from[u] = a.window ? ct.len + (int)__popcll(w) - a.window : 0;
      // by the nodes' stage: its first `joint` keys are the context's last ones
      const uint64_t ctx = ~0ull << min(max(from[u] - (ct.len - joint), 0), 63) & ((1ull << joint) - 1);  // joint is 63 at most
      sees[u] = near_nodes(w, see, a.window) << joint | ctx;
      if (a.window && !sees[u] && max(from[u], ct.lo) >= ct.len) sees_any[u] = false;
    }
    f32x4 o[RT][DT];
    float m[RT], l[RT];
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      m[u] = -INFINITY; l[u] = 0.f;
#pragma unroll
      for (int c = 0; c < DT; ++c) o[u][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const long head = ((long)b * a.Hkv + gh) * a.Smax * D;
    const bf16_t* const kc = (const bf16_t*)a.kc + head + (long)ct.lo * D;
    const bf16_t* const vc = (const bf16_t*)a.vc + head + (long)ct.lo * D;
    const bf16_t* const nk = x + (long)(a.Hq + gh) * D;
    const bf16_t* const nv = nk + (long)a.Hkv * D;
    constexpr int NJ = KB / 1024 / NW;       // this wave's loads of the keys' (values') image
    uint32_t off[2 * NJ];
    int key_of[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int e = (j * NW + wid) * 64 + lane, key = e / NC;
      key_of[j] = key;
      off[j] = key * D * 2 + 16 * paged::kq_chunk<D>(key, e % NC);
      off[NJ + j] = key * D * 2 + 16 * paged::vv_chunk<D>(key, e % NC);
    }
    auto stage = [&](int tile, int buf) {
      char* const dst = smem + 2 * buf * KB + wid * 1024;
      if (!KV8 && tile < ct.full) {
        const long at = (long)tile * SK * D;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          paged::lds_dma16(kc + at, off[j], dst + j * NW * 1024);
          paged::lds_dma16(vc + at, off[NJ + j], dst + KB + j * NW * 1024);
        }
        asm volatile("; a whole stage");
        return;
      }
      // keys behind the last one repeat it: they are masked, and what lies there is nobody's
      const long at = (long)tile * SK * D;
      const bool own = tile == ct.tiles - 1;
      const int ctx = own ? joint : ct.rest;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const uint32_t ck = off[j] & (2 * D - 1), cv = off[NJ + j] & (2 * D - 1);
        // the comments keep the compiler from joining loads of different bases, each of which would become a loop over the bases
        if (!KV8 && (!own || key_of[j] < ctx)) {
          const uint32_t key = min(key_of[j], ctx - 1) * (D * 2);
          paged::lds_dma16(kc + at, key + ck, dst + j * NW * 1024);
          paged::lds_dma16(vc + at, key + cv, dst + KB + j * NW * 1024);
          asm volatile("; last keys of the context");
        }
        if (own && key_of[j] >= ctx) {
          const uint32_t key = min(key_of[j] - ctx, n - 1) * (uint32_t)(a.ldq * 2);
          paged::lds_dma16(nk, key + ck, dst + j * NW * 1024);
          paged::lds_dma16(nv, key + cv, dst + KB + j * NW * 1024);
          asm volatile("; nodes");
        }
      }
    };
    // An e4m3 cache: its stages go to LDS as they are, in a ring of four, three under way, and become bf16 (exact) where fragments are read.
    // The nodes' stage, in bf16, takes the half of the ring that the last of these is not in. Measured against a cache in bf16, captured: 64 rows of
    // 48 nodes over 100 to 700 keys in 32 key heads of one query each 74 us for 92, 16 rows of 32 nodes 37 for 45, where memory bounds these; 48 rows of 16
    // nodes in 8 heads of four 36 for 30, and 64 rows of 64 nodes over 1000 to 4000 keys 222 for 206 to 219 (by the card's power), where the instructions
    // do: each wave converts what it reads. (Converted once, in a pass over LDS with a barrier, the first three took 77, 49 and 38.)
    const int raw_end = min(t1, ct.tiles - 1);
    auto fetch = [&](int tile) {
      const int last = ct.len - ct.lo - tile * SK - 1, slot = tile - t0 & 3;
      const long at = head + ((long)ct.lo + (long)tile * SK) * D;
      char* const dst = smem + slot * KB + wid * 1024;
#pragma unroll
      for (int j = 0; j < NJ / 2; ++j) {
        const int e = (j * NW + wid) * 64 + lane, key = e / 8;
        const uint32_t row = min(key, last) * D;
        paged::lds_dma16((const char*)a.kc + at, row + 16 * paged::kq_chunk<64>(key, e % 8), dst + j * NW * 1024);
        paged::lds_dma16((const char*)a.vc + at, row + 16 * v8_chunk(key, e % 8), dst + KB / 2 + j * NW * 1024);
      }
      const long sc = pair_at * a.SmaxP + ct.lo + tile * SK;
      paged::lds_dma4(a.ksc + sc, 4 * min(lane, last), scales[slot]);  // by every wave: the same to the same place
      paged::lds_dma4(a.vsc + sc, 4 * min(lane, last), scales[slot] + SK);
    };
    constexpr int RAW_LOADS = NJ / 2 * 2 + 2;
    if (tid < 4) bad[tid / 2][tid & 1] = 0;
    // The queries are waited for here, once, behind the first stages (in each branch, where the compiler can count what is behind them). It does
    // not know what the turns wait for, and would put waits for all loads, the next stage's among them, in front of every product with them.
    auto have_queries = [&] {
#pragma unroll
      for (int u = 0; u < RT; ++u)
#pragma unroll
        for (int d = 0; d < DS; ++d) asm volatile("" : "+v"(qf[u][d]));
    };
    if (KV8 && t0 + 2 < raw_end) {
      fetch(t0);
      fetch(t0 + 1);
      fetch(t0 + 2);
      have_queries();
    } else if (KV8 && t0 + 1 < raw_end) {
      fetch(t0);
      fetch(t0 + 1);
      have_queries();
    } else if (KV8 && t0 < raw_end) {
      fetch(t0);
      have_queries();
    } else {
      stage(t0, KV8);
      have_queries();
    }
    int cur = KV8;
    // a stage that lies in LDS; MODE 0: every row sees all of its keys, 1: a window leaves out keys of the context for some, 2: the nodes'
    // own keys, 3: the context's last keys, repeated behind its end
    auto multiply = [&](auto mode, int t, char* image) {
      constexpr int MODE = decltype(mode)::value;
      constexpr bool RAW = KV8 && MODE != 2, SCALED = RAW || STORED;
      char* const Ks = image + wk * KT * D * (RAW ? 1 : 2);
      char* const Vs = Ks + (RAW ? KB / 2 : KB);
      const float* const scale_of = scales[RAW ? t - t0 & 3 : 0];
      f32x4 st[KS][RT];
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int u = 0; u < RT; ++u) st[k][u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (RAW) {
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int d = 0; d < DS; d += 2) {  // 16 bytes: this lane's eight elements of d and of d + 1
            const u32x4 w = *(const u32x4*)(Ks + paged::kq_off<64>(16 * k + r16, 2 * g + d / 2));
            const bf16x8 k0 = fp8x8_to_bf16(w[0], w[1]), k1 = fp8x8_to_bf16(w[2], w[3]);
#pragma unroll
            for (int u = 0; u < RT; ++u) {
              st[k][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, qf[u][d], st[k][u], 0, 0, 0);
              st[k][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, qf[u][d + 1], st[k][u], 0, 0, 0);
            }
          }
      } else {
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int d = 0; d < DS; ++d) {
          // the swizzle goes by the row within the stage: KT rows are a multiple of its period
          const bf16x8 kf = *(const bf16x8*)(Ks + paged::kq_off<D>(16 * k + r16, 4 * d + g));
#pragma unroll
          for (int u = 0; u < RT; ++u) st[k][u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[u][d], st[k][u], 0, 0, 0);
        }
      }
      const int key0 = wk * KT + 4 * g;  // of the stage: this lane's keys are key0 + 16 k + e
      if constexpr (SCALED) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const f32x4 sc = *(const f32x4*)&scale_of[key0 + 16 * k];
#pragma unroll
          for (int u = 0; u < RT; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) st[k][u][e] *= sc[e];
        }
      }
      if constexpr (MODE == 2) {
#pragma unroll
        for (int u = 0; u < RT; ++u)
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            const unsigned bits = (unsigned)(sees[u] >> (key0 + 16 * k));
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(bits >> e & 1)) st[k][u][e] = -INFINITY;
          }
      }
      if constexpr (MODE == 1 || MODE == 3) {
        const int first = ct.lo + t * SK + key0;
#pragma unroll
        for (int u = 0; u < RT; ++u)
#pragma unroll
          for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = first + 16 * k + e;
              if (key >= ct.len || (MODE == 1 && key < from[u])) st[k][u][e] = -INFINITY;
            }
      }
      bool grown = false;
      float mn[RT];
#pragma unroll
      for (int u = 0; u < RT; ++u) {
        float mx = st[0][u][0];
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = larger(mx, st[k][u][e]);
        mn[u] = larger(m[u], over_groups(mx, [](float p, float q) { return larger(p, q); }));
        // each row by its own growth, so that what a row gives does not depend on the rows beside it
        if ((mn[u] - m[u]) * a.scale <= 8.f || mn[u] == m[u]) mn[u] = m[u];
        else grown = true;
      }
      // the maximum that p is taken from follows the rows' own only by steps: up to 2^8 instead of 1 costs nothing in fp32, and o is seldom
      // multiplied
      if (__any(grown)) {
#pragma unroll
        for (int u = 0; u < RT; ++u) {
          const float mz = (mn[u] == -INFINITY ? 0.f : mn[u]) * a.scale;  // a row may see nothing of its first stages
          const float x = mn[u] == m[u] ? 1.f : paged::fexp2(m[u] * a.scale - mz);
          m[u] = mn[u];
          l[u] *= x;
#pragma unroll
          for (int c = 0; c < DT; ++c) o[u][c] *= x;
        }
      }
#pragma unroll
      for (int u = 0; u < RT; ++u) {
        const float mz = (m[u] == -INFINITY ? 0.f : m[u]) * a.scale;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = paged::fexp2(fmaf(st[k][u][e], a.scale, -mz));
            st[k][u][e] = p;
            sum += p;
          }
        l[u] += sum;  // of this lane's keys; the four lanes are added at the end
      }
      if constexpr (SCALED) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const f32x4 sc = *(const f32x4*)&scale_of[SK + key0 + 16 * k];
#pragma unroll
          for (int u = 0; u < RT; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) st[k][u][e] *= MODE == 0 || (MODE != 3 ? fabsf(sc[e]) < INFINITY : key0 + 16 * k + e < ct.rest) ? sc[e] : 0.f;
        }
      }
      bf16x8 pf[KT / 32][RT];
#pragma unroll
      for (int k = 0; k < KT / 32; ++k)
#pragma unroll
        for (int u = 0; u < RT; ++u) pf[k][u] = paged::pack_p(st[2 * k][u], st[2 * k + 1][u]);
      // 0 times the infinity that the last key's value may be is no number: its repetitions count as 0
      uint32_t real[KT / 32][4];
      if constexpr (MODE == 3)
#pragma unroll
        for (int k = 0; k < KT / 32; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int left = ct.rest - (key0 + 32 * k + 16 * (i / 2) + 2 * (i & 1));
            real[k][i] = left <= 0 ? 0 : left == 1 ? 0xffffu : ~0u;
          }
      auto of_keys = [&](bf16x8 v, int k) {
        if constexpr (MODE == 3) {
          u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] &= real[k][i];
          v = __builtin_bit_cast(bf16x8, w);
        }
        return v;
      };
      const int key_a = 4 * g + (lane >> 2 & 3), pcol = lane & 3;  // transposed reads: rows 16 apart have the same swizzle
      if constexpr (RAW) {
        // lane pairs read the 16 columns of keys 4 g .. + 3 and 16 behind these; the lane gets its column of the eight
        const int q = lane >> 1 & 7, key = 4 * g + (q & 3) + 16 * (q >> 2);
        const uint32_t at = lds_addr(Vs + key * D + 16 * v8_chunk(key, 0) + 8 * (lane & 1));
#pragma unroll
        for (int h = 0; h < KT / 32; ++h) {
          uint2 v[8];
          if (h == 0) read_columns8<0>(at, v);
          else read_columns8<32 * D>(at, v);
#pragma unroll
          for (int c = 0; c < DT; ++c) {
            const bf16x8 vf = of_keys(fp8x8_to_bf16(v[c & 7].x, v[c & 7].y), h);
#pragma unroll
            for (int u = 0; u < RT; ++u) o[u][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[h][u], o[u][c], 0, 0, 0);
          }
        }
        return;
      }
#pragma unroll
      for (int c = 0; c < DT; c += 4) {
        uint32_t va[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) va[k] = lds_addr(Vs + paged::vv_off<D>(key_a, 2 * (c + k) + (pcol >> 1)) + ((pcol & 1) << 3));
        if constexpr (KT == 64) {
          rt_s16x4 v[16];
          ds_tr16_frag4<16 * D * 2, 32 * D * 2, 48 * D * 2>(va[0], va[1], va[2], va[3], v);
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const bf16x8 vf = of_keys(paged::cat4(v[4 * k + 2 * h], v[4 * k + 2 * h + 1]), h);
#pragma unroll
              for (int u = 0; u < RT; ++u) o[u][c + k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[h][u], o[u][c + k], 0, 0, 0);
            }
        } else {
          const uint32_t at[8] = {va[0], va[0] + 32 * D, va[1], va[1] + 32 * D, va[2], va[2] + 32 * D, va[3], va[3] + 32 * D};
          rt_s16x4 v[8];
          ds_tr16_at8(at, v);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const bf16x8 vf = of_keys(paged::cat4(v[2 * k], v[2 * k + 1]), 0);
#pragma unroll
            for (int u = 0; u < RT; ++u) o[u][c + k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[0][u], o[u][c + k], 0, 0, 0);
          }
        }
      }
    };
    // The values of a stage that some row does not see all of: 0 times what is no number is none, so such values count as 0 in the product and
    // are added at the end for the rows that see them. These are the nodes' stage and, with a window, the first one (the last node's starts less
    // than NODES keys behind the first one's). The reads are of this kind because ordinary ones would wait for the next stage.
    auto only_numbers = [&](char* values, auto own) {
      constexpr bool raw = KV8 && !own.value;
      constexpr int second = raw ? KB / 4 : KB / 2;
#pragma unroll 1
      for (int e = 16 * tid; e < second; e += 16 * 64 * NW) {
        u32x4 w[2];
        read_pair<second>(lds_addr(values + e), w[0], w[1]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int key = (e + h * second) / (raw ? D : 2 * D);
          u32x4 x = w[h];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (raw) x[i] &= ~((((x[i] & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u) * 0xffu);
            else x[i] &= ((x[i] & 0x7f80u) == 0x7f80u ? 0xffff0000u : ~0u) & ((x[i] & 0x7f800000u) == 0x7f800000u ? 0xffffu : ~0u);
          }
          bool ill = x[0] != w[h][0] || x[1] != w[h][1] || x[2] != w[h][2] || x[3] != w[h][3];
          if (ill) *(u32x4*)(values + e + h * second) = x;
          if (raw || (STORED && key < n)) ill |= !(fabsf(scales[0][SK + key]) < INFINITY);
          if (ill) atomicOr(&bad[own.value][key / 32], 1u << (key % 32));
        }
      }
    };
    // The nodes' keys and values to e4m3 and back, with a scale each in the place of a stage that is done: as tree_accept stores them. 16 lanes a row,
    // each with 8 elements of its key and of its value, wherever the swizzle put these. Rows behind the nodes keep any scale: they are masked.
    // Measured, captured: one row of 8 nodes over 300 keys 9.7 -> 10.6 us, 64 rows of 48 nodes in 32 key heads 74 -> 78, 48 rows of 16 in 8 36.0 -> 36.4.
    auto round_nodes = [&](char* image) {
#pragma unroll 1
      for (int e = 16 * tid; e < n * 2 * D; e += 16 * 64 * NW) {
        float f[2][8], am[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          unpack8(*(const uint4*)(image + h * KB + e), f[h]);
          am[h] = fabsf(f[h][0]);
#pragma unroll
          for (int i = 1; i < 8; ++i) am[h] = fmaxf(am[h], fabsf(f[h][i]));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          am[h] = largest16(am[h]);
          const float sc = am[h] > 0.f ? am[h] / 448.f : 1.f;
          const uint2 q = f32x8_to_fp8(f[h], 1.f / sc);
          *(bf16x8*)(image + h * KB + e) = fp8x8_to_bf16(q.x, q.y);
          if ((tid & 15) == 0) scales[0][h * SK + e / (2 * D)] = sc;
        }
      }
    };
    auto turn = [&](auto mode, int t) {
      constexpr int MODE = decltype(mode)::value;
      if constexpr (KV8 && MODE != 2) {
        // this stage, not those behind it
        if (t + 2 < raw_end) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(2 * RAW_LOADS) : "memory");
        else if (t + 1 < raw_end) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(RAW_LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");  // ... of every wave, and the stage before is multiplied
        const int slot = t - t0 & 3;
        if constexpr (MODE == 1) {
          only_numbers(smem + slot * KB + KB / 2, std::false_type());
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          asm volatile("s_barrier" ::: "memory");
        }
        if (t + 3 < raw_end) {
          fetch(t + 3);
        } else if (t + 1 == raw_end && raw_end < t1) {
          cur = slot < 2;
          stage(t + 1, cur);
        }
        if (row0 < M) multiply(mode, t, smem + slot * KB);
        return;
      }
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // this stage, issued one ago
      asm volatile("s_barrier" ::: "memory");                      // ... by every wave; the other buffer is free
      if (MODE != 2 && t + 1 < t1) stage(t + 1, cur ^ 1);
      char* const image = smem + 2 * cur * KB;
      cur ^= 1;
      if constexpr (MODE == 2 && STORED) {
        round_nodes(image);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");
      }
      if constexpr (MODE == 1 || MODE == 2) {
        only_numbers(image + KB, std::bool_constant<MODE == 2>());
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");
      }
      if (row0 < M) multiply(mode, t, image);
    };
    int t = t0;
    if (a.window && t == 0 && t < min(t1, ct.tiles - 1)) turn(std::integral_constant<int, 1>(), t++);
    for (; t < min(t1, ct.full); ++t) turn(std::integral_constant<int, 0>(), t);
    if (t < min(t1, ct.tiles - 1)) turn(std::integral_constant<int, 3>(), t++);
    if (t < t1) turn(std::integral_constant<int, 2>(), t);
    for (int own = 0; own < 2; ++own) {
      const uint64_t ill = ((uint64_t)bad[own][1] << 32 | bad[own][0]) & (KT == 64 ? ~0ull : 0xffffffffull << (wk * KT));
      for (uint64_t w = ill; w; w &= w - 1) {
        const int key = __builtin_ctzll(w), i = own ? ct.full * SK + key : key;  // of the context, behind ct.lo
        const bool node = own && key >= joint;
        if (!own && ct.lo + i >= ct.len) break;
        const bf16_t* const v = (node ? nv + (long)(key - joint) * a.ldq : vc + (long)i * D) + 4 * g;
        const uint8_t* const v8 = (const uint8_t*)a.vc + head + ((long)ct.lo + i) * D + 4 * g;
        const float sc = KV8 && !own ? a.vsc[pair_at * a.SmaxP + ct.lo + i] : 1.f;
#pragma unroll
        for (int u = 0; u < RT; ++u)
          if (own ? sees[u] >> key & 1 : ct.lo + i >= from[u])
#pragma unroll
            for (int c = 0; c < DT; ++c) {
              const uint32_t four = KV8 && !own ? *(const uint32_t*)(v8 + 16 * c) : 0;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float f = KV8 && !own ? fp8_at(four, e) * sc : STORED ? as_stored(bf2f(v[16 * c + e]), scales[0][SK + key]) : bf2f(v[16 * c + e]);
                if (!(fabsf(f) < INFINITY)) o[u][c][e] += f;
              }
              asm volatile("" ::: "memory");  // this is seldom reached: few registers, not many loads at once
            }
      }
    }
#pragma unroll
    for (int u = 0; u < RT; ++u) l[u] = over_groups(l[u], [](float p, float q) { return p + q; });
    if constexpr (WK > 1) {  // the keys' shares, joined in order
      float* const sh = (float*)smem + wr * (4 * DT + 2) * 64 + lane;
      static_assert(WR * (4 * DT + 2) * 256 <= 4 * KB);
#pragma unroll
      for (int u = 0; u < RT; ++u)
        for (int k = 1; k < WK; ++k) {
          __syncthreads();
          if (wk == k) {
            sh[0] = m[u];
            sh[64] = l[u];
#pragma unroll
            for (int c = 0; c < DT; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) sh[(2 + 4 * c + e) * 64] = o[u][c][e];
          }
          __syncthreads();
          if (wk == 0) {
            const float mn = larger(m[u], sh[0]), mz = (mn == -INFINITY ? 0.f : mn) * a.scale;
            const float x0 = paged::fexp2(m[u] * a.scale - mz), x1 = paged::fexp2(sh[0] * a.scale - mz);
            m[u] = mn;
            l[u] = l[u] * x0 + sh[64] * x1;
#pragma unroll
            for (int c = 0; c < DT; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[u][c][e] = o[u][c][e] * x0 + sh[(2 + 4 * c + e) * 64] * x1;
          }
        }
    }
#pragma unroll
    for (int u = 0; u < RT; ++u) {
      if (wk) break;
      const int r = row0 + 16 * u + r16;
      if (ct.parts > 1) {
        if (row0 + 16 * u >= M) continue;
        float* const p = part_of(a, D, s, pair_at);
        if (g == 0) *(float2*)(p + tiles16(a) * 16 * D + 2 * r) = make_float2(m[u] * a.scale, l[u]);
        f32x4* const q = (f32x4*)(p + (long)(row0 + 16 * u) * D) + lane;
#pragma unroll
        for (int c = 0; c < DT; ++c) q[64 * c] = o[u][c];
      } else if (r < M) {
        const float inv = 1.f / l[u];
        const int node = node_of_row(a, r);
        bf16_t* const p = (bf16_t*)a.o + ((long)b * a.N + node) * a.ldo + (long)(gh * G + r - node * G) * D + 4 * g;
#pragma unroll
        for (int c = 0; c < DT; ++c)
          *(uint2*)(p + 16 * c) = sees_any[u] ? make_uint2(pack2bf(o[u][c][0] * inv, o[u][c][1] * inv), pack2bf(o[u][c][2] * inv, o[u][c][3] * inv))
                                          : make_uint2(0, 0);
      }
    }
  }
  if (s == 0) {  // rows that are no nodes
    for (int r = max(M, rb * ROWS) + wid; r < min(a.N * G, (rb + 1) * ROWS); r += NW) {
      bf16_t* const p = (bf16_t*)a.o + ((long)b * a.N + r / G) * a.ldo + (long)(gh * G + r % G) * D;
      if (lane < D / 4) *(uint2*)(p + 4 * lane) = make_uint2(0, 0);
    }
  }
}

// The parts of rows that were cut: WAVES waves for 16 rows' accumulators of 16 columns, eight parts each under way at once. The first
// eight are read before the lengths that say how many there are (what lies in the others is in the buffer, and not used): one trip to
// memory instead of two.
template <int D, int WAVES>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a, int SK) {
  __shared__ float sh[4][6][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, w = wid % WAVES, r16 = lane & 15, g = lane >> 4, G = a.G;
  const int tiles = tiles16(a);
  const long all = (long)a.B * a.Hkv * tiles * (D / 16), id = (long)blockIdx.x * (4 / WAVES) + wid / WAVES, at = min(id, all - 1);
  const int c = (int)(at % (D / 16)), tile = (int)(at / (D / 16) % tiles);
  const long pair = at / (D / 16) / tiles;
  const int b = (int)(pair / a.Hkv), gh = (int)(pair % a.Hkv), r = 16 * tile + r16;
  float m = -INFINITY, l = 0.f;
  f32x4 o{0.f, 0.f, 0.f, 0.f};
  int parts = a.S;
  const int n = count_nodes(lane < a.N ? word(a, b, lane) : 0);
  for (int s0 = 8 * w; s0 < parts; s0 += 8 * WAVES) {
    float2 ml[8];
    f32x4 po[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float* const q = part_of(a, D, min(s0 + k, a.S - 1), pair);
      ml[k] = *(const float2*)(q + tiles * 16 * D + 2 * r);
      po[k] = ((const f32x4*)(q + 16 * tile * D))[64 * c + lane];
    }
    parts = cut(a, b, n, SK).parts;
    float mx = m;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s0 + k < parts) mx = larger(mx, ml[k].x);
    const float mz = mx == -INFINITY ? 0.f : mx, old = paged::fexp2(m - mz);
    m = mx;
    l *= old;
    o *= old;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (s0 + k < parts) {
        const float x = paged::fexp2(ml[k].x - mz);
        l = fmaf(ml[k].y, x, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(po[k][e], x, o[e]);
      }
  }
  if constexpr (WAVES > 1) {
    sh[wid][0][lane] = m;
    sh[wid][1][lane] = l;
#pragma unroll
    for (int e = 0; e < 4; ++e) sh[wid][2 + e][lane] = o[e];
    __syncthreads();
    if (w) return;
    float mx = m;
#pragma unroll
    for (int k = 1; k < WAVES; ++k) mx = larger(mx, sh[wid + k][0][lane]);
    const float mz = mx == -INFINITY ? 0.f : mx, old = paged::fexp2(m - mz);
    l *= old;
    o *= old;
#pragma unroll
    for (int k = 1; k < WAVES; ++k) {
      const float x = paged::fexp2(sh[wid + k][0][lane] - mz);
      l = fmaf(sh[wid + k][1][lane], x, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(sh[wid + k][2 + e][lane], x, o[e]);
    }
  }
  if (id >= all || parts == 1 || r >= a.N * G) return;
  const bool node = word(a, b, r / G) != 0;  // others have no parts (windows that may leave nothing of a node are under a stage: never cut)
  const float inv = 1.f / l;
  *(uint2*)((bf16_t*)a.o + ((long)b * a.N + r / G) * a.ldo + (long)(gh * G + r % G) * D + 16 * c + 4 * g) =
      node ? make_uint2(pack2bf(o[0] * inv, o[1] * inv), pack2bf(o[2] * inv, o[3] * inv)) : make_uint2(0, 0);
}

// ---------------------------------------------------------------------------------------------
// the path that the model agrees with, and its keys and values into the caches. One workgroup per (row, layer), each of which walks
// the tree by itself: a step is a comparison over the wave's nodes.
// ---------------------------------------------------------------------------------------------
constexpr int LAYERS = 256;
struct AcceptArgs {
  const int* parent; const int64_t* see; const int64_t* tokens; const int64_t* choice; const int* kv_len;
  int* count; int* path; int64_t* next;
  void* kc; void* vc;                   // [L, B, Hkv, Smax, D], layers `layer` units apart
  long ldq, layer;
  float* ksc; float* vsc; long sc_layer; int SmaxP;  // scales [L, B, Hkv, SmaxP] of e4m3 caches, or null
  int B, N, L, Hq, Hkv, Smax, row;      // row: 16-byte (or single element) units of a head's row
  const void* drafts[LAYERS];           // [B N, (Hq + 2 Hkv) D] of every layer
};

// KV8: rows of 128 in bf16 to e4m3 with a scale each, rounded and ordered as a prompt's are
template <typename U, bool KV8>
__global__ __launch_bounds__(256) void tree_accept_kernel(AcceptArgs a) {
  __shared__ int path[NODES];
  __shared__ int steps;
  const int b = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x;
  const long at = (long)b * a.N;
  if (tid < 64) {
    const bool in = tid < a.N;
    const uint64_t see = in ? (uint64_t)a.see[at + tid] : 0;
    const int p = in ? a.parent[at + tid] : -1;
    const int64_t tok = in ? a.tokens[at + tid] : 0;
    const uint64_t choice = in ? (uint64_t)a.choice[at + tid] : 0;
    const bool child = see != 0 && p >= 0 && p < tid;
    const int room = a.Smax - max(a.kv_len[b], 0);
    int cur = 0, n = 0, mine = -1;
    int64_t last = -1;
    if (__ballot(see != 0) & 1 && room > 0) {
      for (;;) {  // nodes along a path rise: at most N steps
        if (tid == n) mine = cur;
        ++n;
        last = (int64_t)lane64(choice, cur);
        if (n == room) break;  // a node without a slot would be missing from the context of what follows it
        const uint64_t go = __ballot(child && p == cur && tok == last);
        if (!go) break;
        cur = __builtin_ctzll(go);
      }
    }
    path[tid] = mine;
    if (tid == 0) steps = n;
    if (layer == 0) {
      if (in) a.path[at + tid] = mine;
      if (tid == 0) { a.count[b] = n; a.next[b] = last; }
    }
  }
  __syncthreads();
  const int len = max(a.kv_len[b], 0), n = steps;
  const U* const x = (const U*)a.drafts[layer] + at * a.ldq;
  if constexpr (KV8) {
    const int c = tid & 15;  // 16 lanes a row
    for (int e = tid >> 4; e < n * a.Hkv * 2; e += 16) {
      const int kv = e & 1, g = e / 2 % a.Hkv, i = e / 2 / a.Hkv;
      float f[8];
      unpack8(((const uint4*)x)[path[i] * a.ldq + (long)(a.Hq + kv * a.Hkv + g) * 16 + c], f);
      float am = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) am = fmaxf(am, fabsf(f[q]));
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) am = fmaxf(am, __shfl_xor(am, o, 16));
      const float sc = am > 0.f ? am / 448.f : 1.f;
      const uint2 w = f32x8_to_fp8(f, 1.f / sc);
      const long slot = ((long)b * a.Hkv + g) * a.Smax + len + i;
      char* const at = (char*)(kv ? a.vc : a.kc) + layer * a.layer + slot * 128;
      *(uint2*)(at + (kv ? 8 * c : 32 * (c & 3) + 8 * (c >> 2))) = w;
      if (c == 0) (kv ? a.vsc : a.ksc)[layer * a.sc_layer + ((long)b * a.Hkv + g) * a.SmaxP + len + i] = sc;
    }
    return;
  }
  const long head = layer * a.layer + (long)b * a.Hkv * a.Smax * a.row;
  for (int e = tid; e < n * a.Hkv * a.row; e += 256) {
    const int i = e / (a.Hkv * a.row), r = e % (a.Hkv * a.row), g = r / a.row, c = r % a.row;
    const U* const src = x + path[i] * a.ldq + (long)(a.Hq + g) * a.row + c;
    const long dst = head + ((long)g * a.Smax + len + i) * a.row + c;
    ((U*)a.kc)[dst] = src[0];
    ((U*)a.vc)[dst] = src[(long)a.Hkv * a.row];
  }
}

}  // namespace drafts
}  // namespace rt

using namespace rt;
using namespace rt::drafts;

extern "C" int rt_draft_tree(const int* parent, const int* nodes, const int* pos0, int B, int N, int64_t* see, int* pos, hipStream_t stream) {
  if (N < 1 || N > NODES) return -1;
  if (B == 0) return 0;
  hipLaunchKernelGGL(draft_tree_kernel, dim3(B), dim3(64), 0, stream, parent, nodes, pos0, N, see, pos);
  RT_LAUNCH_CHECK();
  return 0;
}

constexpr int WIDE_ROWS = 192;  // rows of a key head that go to workgroups of 64

template <int D, int RT, int WR, int WK, int KT, bool KV8, bool STORED>
static void launch_tree_form(const TreeArgs& a, int rows, hipStream_t stream) {
  TreeArgs t = a;
  t.blocks = (rows + 16 * RT * WR - 1) / (16 * RT * WR);
  const dim3 grid = t.blocks == 1 ? dim3(a.S, a.Hkv, a.B) : dim3(8 * t.blocks, (unsigned)(((long)a.S * a.B * a.Hkv + 7) / 8));
  hipLaunchKernelGGL((tree_mfma_kernel<D, RT, WR, WK, KT, KV8, STORED>), grid, dim3(64 * WR * WK), 0, stream, t);
}
template <int D, bool KV8, bool STORED>
static int launch_tree(const TreeArgs& a, int rows, hipStream_t stream) {
  // waves by rows of 16, and two shares of each stage's keys: half the chain of a stage, and the shares are joined in LDS at the end (16 ungrouped
  // rows of 32 nodes 52 -> 47 us, 48 rows of 64 34 -> 31 against one share). Up to 192 rows go to workgroups of 64, two of them on a
  // CU, that read the same keys from L2 (32 rows of 128 over 500 to 2900 keys 56 us, in one workgroup of 8 waves with two tiles each 64); beyond, and
  // with few idle waves, two tiles a wave halve the reads of LDS (40 rows of 240 41 us against 46).
  if (rows <= 16) launch_tree_form<D, 1, 1, 2, 32, KV8, STORED>(a, rows, stream);
  else if (rows <= 32) launch_tree_form<D, 1, 2, 2, 32, KV8, STORED>(a, rows, stream);
  else if (rows <= WIDE_ROWS) launch_tree_form<D, 1, 4, 2, 32, KV8, STORED>(a, rows, stream);
  else launch_tree_form<D, 2, 8, 1, 64, KV8, STORED>(a, rows, stream);
  RT_LAUNCH_CHECK();
  return 0;
}

template <int D>
static void launch_join(const TreeArgs& a, long all, hipStream_t stream) {
  if (a.S <= 8) hipLaunchKernelGGL((tree_join_kernel<D, 1>), dim3((unsigned)((all + 3) / 4)), dim3(256), 0, stream, a, 64);
  else hipLaunchKernelGGL((tree_join_kernel<D, 4>), dim3((unsigned)all), dim3(256), 0, stream, a, 64);
}

// a part's time of all key heads and a join's, in stages (0.9 us of a workgroup that is alone on its CU, 2.4 with 256 rows)
static void tree_costs(int B, int N, int Hq, int Hkv, int D, float& part, float& join) {
  const int rows = N * (Hq / Hkv);
  const float stage = (rows <= WIDE_ROWS ? 0.9f : 2.4f) * (D == 64 ? 0.7f : 1.f);
  part = (float)B * Hkv * ((rows + 15) / 16 * 16) * (D + 2) * 8 / 4.5e6f / stage;
  join = 3.f / stage;
}

// Parts that a row's keys may be cut in at most: the partials that rt_tree_attention wants (0: sizes without matrix instructions). No more than
// fill the CUs once; 1, and no second launch, where a full cache would not gain a quarter by them (the launch costs 3 us also where no
// row turns out long enough).
extern "C" int rt_tree_parts(int B, int N, int Hq, int Hkv, int D, int Smax, int window) {
  if ((D != 64 && D != 128) || B == 0 || Hq / Hkv > 4096 || (long)B * Hkv > 500000) return 0;  // grids
  const int rows = N * (Hq / Hkv), blocks = B * Hkv * (rows <= WIDE_ROWS ? (rows + 63) / 64 : (rows + 255) / 256);
  const int stages = ((window ? std::min(Smax, window) : Smax) + 63) / 64 + 1;
  const int most = std::max(1, std::min((num_cus() + blocks / 2) / blocks, stages));
  float part, join;
  tree_costs(B, N, Hq, Hkv, D, part, join);
  const int per = stages_per_part(stages, most, part, join), parts = (stages + per - 1) / per;
  return per + part * parts + join < 0.75f * stages ? parts : 1;
}

extern "C" int rt_tree_attention(int f32, const void* qkv, long ldq, const void* kc, const void* vc, const float* ksc, const float* vsc, int SmaxP,
                                 const int* kv_len, const int* kv_start, const int64_t* see, void* o, long ldo, float* part, int S, int B, int N, int Hq, int Hkv, int D, int Smax,
                                 int window, float scale, int stored, hipStream_t stream) {
  if (B == 0) return 0;
  if (N < 1 || N > NODES || Hkv < 1 || Hq % Hkv || Hq > 65535 || B > 65535 || D < 1 || D > 512) return -1;
  TreeArgs a{qkv, ldq, kc, vc, ksc, vsc, SmaxP, kv_len, kv_start, see, o, ldo, B, N, Hq, Hkv, D, Smax, window, scale, Hq / Hkv, 1.f / (Hq / Hkv), 0, 1, 0.f, 0.f, part, S};
  if (stored && !ksc) return -1;
  if (ksc && (!vsc || D != 128 || SmaxP < Smax || S < 1)) return -1;
  if (S < 1) {
    const size_t shm = (2 * D + 256 + 4) * sizeof(float);
    if (f32) hipLaunchKernelGGL(tree_any_kernel<float>, dim3(N, Hq, B), dim3(256), shm, stream, a);
    else hipLaunchKernelGGL(tree_any_kernel<bf16_t>, dim3(N, Hq, B), dim3(256), shm, stream, a);
    RT_LAUNCH_CHECK();
    return 0;
  }
  if (f32 || (D != 64 && D != 128) || (S > 1 && !part)) return -1;
  a.scale = scale * 1.4426950408889634f;
  tree_costs(B, N, Hq, Hkv, D, a.part_cost, a.join_cost);
  const int rows = N * (Hq / Hkv);
  // Long rows first where a CU takes workgroups of 256 rows one after the other: 64 rows of 300 to 4000 keys in any order 177 us, as they come 230.
  // Smaller workgroups, of which several share a CU, only pay for the order (64 rows over 32 ungrouped heads 102 us, in order 110).
  a.sorted = rows > WIDE_ROWS && B > 1 && B <= 64 && (long)B * Hkv * S > num_cus();
  const int rc = ksc ? (stored ? launch_tree<128, true, true>(a, rows, stream) : launch_tree<128, true, false>(a, rows, stream))
                     : D == 128 ? launch_tree<128, false, false>(a, rows, stream) : launch_tree<64, false, false>(a, rows, stream);
  if (rc) return rc;
  if (S > 1) {
    const long all = (long)B * Hkv * ((rows + 15) / 16) * (D / 16);
    if (D == 128) launch_join<128>(a, all, stream);
    else launch_join<64>(a, all, stream);
    RT_LAUNCH_CHECK();
  }
  return 0;
}

extern "C" int rt_tree_accept(const int* parent, const int64_t* see, const int64_t* tokens, const int64_t* choice, const int* kv_len, int* count,
                              int* path, int64_t* next, const void* const* drafts, long ldq, void* kc, void* vc, long layer,
                              float* ksc, float* vsc, long sc_layer, int SmaxP, int B, int N, int L, int Hq,
                              int Hkv, int Smax, int D, int size, hipStream_t stream) {
  if (B == 0) return 0;
  if (N < 1 || N > NODES || L < 1 || L > LAYERS) return -1;
  AcceptArgs a{parent, see, tokens, choice, kv_len, count, path, next, kc, vc, ldq, layer, ksc, vsc, sc_layer, SmaxP, B, N, L, Hq, Hkv, Smax, D, {}};
  bool wide = (D * size) % 16 == 0 && (ldq * size) % 16 == 0 && layer * (ksc ? 1 : size) % 16 == 0 && (uintptr_t)kc % 16 == 0 && (uintptr_t)vc % 16 == 0;
  for (int i = 0; i < L; ++i) {
    a.drafts[i] = drafts[i];
    wide = wide && (uintptr_t)drafts[i] % 16 == 0;
  }
  if (ksc) {
    if (!vsc || D != 128 || SmaxP < Smax || !wide) return -1;
    a.ldq = ldq / 8;
    hipLaunchKernelGGL((tree_accept_kernel<uint4, true>), dim3(B, L), dim3(256), 0, stream, a);
  } else if (wide) {
    a.row = D * size / 16;
    a.ldq = ldq * size / 16;
    a.layer = layer * size / 16;
    hipLaunchKernelGGL((tree_accept_kernel<uint4, false>), dim3(B, L), dim3(256), 0, stream, a);
  } else if (size == 4) {
    hipLaunchKernelGGL((tree_accept_kernel<uint32_t, false>), dim3(B, L), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL((tree_accept_kernel<uint16_t, false>), dim3(B, L), dim3(256), 0, stream, a);
  }
  RT_LAUNCH_CHECK();
  return 0;
}
