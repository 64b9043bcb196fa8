// Checking drafted tokens: the plan of a batch's token trees, attention of their nodes over the K/V cache, and the path that the
// model agrees with, appended to the cache of every layer. Up to 64 nodes a row: a node's ancestors are one 64-bit word, and a
// wave holds a row's tree with one node to a lane.
#include "rt_common.h"
#include "rt_paged.h"

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
  const int* kv_len; const int* kv_start;
  const int64_t* see;                   // [B, N]
  void* o; long ldo;
  int B, N, Hq, Hkv, D, Smax, window;   // window 0: none
  float scale;
};

template <typename T>
__global__ __launch_bounds__(256) void tree_any_kernel(TreeArgs a) {
  extern __shared__ float sm[];  // q [D], acc [D], p [256], sbuf [4]
  float* qs = sm;
  float* acc = qs + a.D;
  float* ps = acc + a.D;
  float* sbuf = ps + 256;
  const int i = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, gh = h / (a.Hq / a.Hkv);
  const int64_t* see = a.see + (long)b * a.N;
  const uint64_t mine = see[i];
  const T* const x = (const T*)a.qkv + (long)b * a.N * a.ldq;
  T* const o = (T*)a.o + ((long)b * a.N + i) * a.ldo + (long)h * a.D;
  if (!mine) {
    for (int c = tid; c < a.D; c += 256) st(o + c, 0.f);
    return;
  }
  const int depth = __popcll(mine) - 1, len = min(max(a.kv_len[b], 0), a.Smax);
  int lo = a.kv_start ? max(a.kv_start[b], 0) : 0;
  if (a.window) lo = max(lo, len + depth - a.window + 1);
  const int ctx = max(len - lo, 0), n = ctx + a.N;
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
    if (j >= ctx && j < n) {
      const int node = j - ctx;
      sees = (mine >> node & 1) && !(a.window && depth + 1 - __popcll((uint64_t)see[node]) >= a.window);
    }
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
  for (int c = tid; c < a.D; c += 256) st(o + c, acc[c] / l);  // a node sees itself
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
  int B, N, L, Hq, Hkv, Smax, row;      // row: 16-byte (or single element) units of a head's row
  const void* drafts[LAYERS];           // [B N, (Hq + 2 Hkv) D] of every layer
};

template <typename U>
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
    int cur = 0, n = 0, mine = -1;
    int64_t last = -1;
    if (__ballot(see != 0) & 1) {
      for (;;) {  // nodes along a path rise: at most N steps
        if (tid == n) mine = cur;
        ++n;
        last = (int64_t)lane64(choice, cur);
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
  const int len = max(a.kv_len[b], 0), n = min(steps, a.Smax - len);  // slots that are there
  const U* const x = (const U*)a.drafts[layer] + at * a.ldq;
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

extern "C" int rt_tree_attention(int f32, const void* qkv, long ldq, const void* kc, const void* vc, const int* kv_len, const int* kv_start,
                                 const int64_t* see, void* o, long ldo, int B, int N, int Hq, int Hkv, int D, int Smax, int window,
                                 float scale, hipStream_t stream) {
  if (B == 0) return 0;
  if (N < 1 || N > NODES || Hkv < 1 || Hq % Hkv || Hq > 65535 || B > 65535 || D < 1 || D > 512) return -1;
  const TreeArgs a{qkv, ldq, kc, vc, kv_len, kv_start, see, o, ldo, B, N, Hq, Hkv, D, Smax, window, scale};
  const size_t shm = (2 * D + 256 + 4) * sizeof(float);
  if (f32) hipLaunchKernelGGL(tree_any_kernel<float>, dim3(N, Hq, B), dim3(256), shm, stream, a);
  else hipLaunchKernelGGL(tree_any_kernel<bf16_t>, dim3(N, Hq, B), dim3(256), shm, stream, a);
  RT_LAUNCH_CHECK();
  return 0;
}

extern "C" int rt_tree_accept(const int* parent, const int64_t* see, const int64_t* tokens, const int64_t* choice, const int* kv_len, int* count,
                              int* path, int64_t* next, const void* const* drafts, long ldq, void* kc, void* vc, long layer, int B, int N, int L, int Hq,
                              int Hkv, int Smax, int D, int size, hipStream_t stream) {
  if (B == 0) return 0;
  if (N < 1 || N > NODES || L < 1 || L > LAYERS) return -1;
  AcceptArgs a{parent, see, tokens, choice, kv_len, count, path, next, kc, vc, ldq, layer, B, N, L, Hq, Hkv, Smax, D, {}};
  bool wide = (D * size) % 16 == 0 && (ldq * size) % 16 == 0 && (layer * size) % 16 == 0 && (uintptr_t)kc % 16 == 0 && (uintptr_t)vc % 16 == 0;
  for (int i = 0; i < L; ++i) {
    a.drafts[i] = drafts[i];
    wide = wide && (uintptr_t)drafts[i] % 16 == 0;
  }
  if (wide) {
    a.row = D * size / 16;
    a.ldq = ldq * size / 16;
    a.layer = layer * size / 16;
    hipLaunchKernelGGL(tree_accept_kernel<uint4>, dim3(B, L), dim3(256), 0, stream, a);
  } else if (size == 4) {
    hipLaunchKernelGGL(tree_accept_kernel<uint32_t>, dim3(B, L), dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL(tree_accept_kernel<uint16_t>, dim3(B, L), dim3(256), 0, stream, a);
  }
  RT_LAUNCH_CHECK();
  return 0;
}
