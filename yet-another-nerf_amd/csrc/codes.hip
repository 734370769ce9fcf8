// Learned codes for gfx950: embedding lookup with scaling and dropout, its gradient by sorted ids, and dropout whose
// mask is a function of a Philox counter.
//
//   lookup   out[n, d] = f * table[ids[n], d] * keep(n D + d)                          f = scale / (1 - p)
//   gradient grad[v, d] = f * sum over n with ids[n] == v of keep(n D + d) * g[n, d]   (0 for the padding row)
//   dropout  y[e] = x[e] * keep(e) / (1 - p); its gradient is the same map
//
// keep(e) is 1 where word e % 4 of Philox4x32-10(key = seed, counter = (e / 4, offset)) is at least
// T = round(p 2^32): forward and backward evaluate it anew, so no mask is stored or read. A dropped element is 0
// whatever its input holds. Products and sums are fp32; each output is rounded once.
//
// The gradient sorts the positions by id with a stable sort, so the terms of a row are added in an order that only the
// ids fix: no float atomics, the same bits on every run.
#include <cmath>

#include "common.hpp"

namespace yanerf {

// ------------------------------------------------------------------------------------------ types
enum { kF32 = YANERF_TYPE_F32, kBf16 = YANERF_TYPE_BF16, kF16 = YANERF_TYPE_F16 };

inline int64_t type_bytes(int t) { return t == kF32 ? 4 : 2; }
inline bool type_ok(int t) { return t == kF32 || t == kBf16 || t == kF16; }

// f(T{}) with T the element type of `t`
template <typename F>
inline void with_type(int t, F&& f) {
  if (t == kF32) f(float{});
  else if (t == kBf16) f(__bf16{});
  else f(_Float16{});
}

// workgroups for `work` of them, bounded so that a launch stays under 2^32 threads (the kernels stride over the rest)
inline dim3 grid_for(int64_t work) { return dim3((unsigned)(work < (1 << 22) ? work : (1 << 22))); }

// ------------------------------------------------------------------------------------------ dropout mask
struct Mask {
  uint64_t seed, offset;
  const uint64_t* base;  // NULL, or a device u64 added to `offset`
  uint32_t threshold;    // T; kept iff word >= T
  int mode;              // 0 keep all, 1 by word, 2 drop all
};

inline Mask make_mask(double p, uint64_t seed, uint64_t offset, const uint64_t* base) {
  const double t = std::floor(p * 4294967296.0 + 0.5);
  Mask m{seed, offset, base, 0, 0};
  if (t >= 4294967296.0) m.mode = 2;
  else if (t > 0.0) {
    m.mode = 1;
    m.threshold = (uint32_t)t;
  }
  return m;
}

// 1 / (1 - p), 0 where everything is dropped
inline double mask_scale(double p, const Mask& m) { return m.mode == 2 ? 0.0 : 1.0 / (1.0 - p); }

__device__ __forceinline__ uint64_t mask_offset(const Mask& m) { return m.offset + (m.base ? *m.base : 0ull); }

__device__ __forceinline__ bool keep_at(const Mask& m, uint64_t off, uint64_t e) {
  if (m.mode != 1) return m.mode == 0;
  const u4 r = philox(m.seed, off, e >> 2);
  const uint32_t w = (e & 2) ? ((e & 1) ? r.w : r.z) : ((e & 1) ? r.y : r.x);
  return w >= m.threshold;
}

// ------------------------------------------------------------------------------------------ dropout
template <typename T>
__global__ void dropout_kernel(const T* x, T* y, int64_t n, Mask m, float f, uint64_t* used) {
  const uint64_t off = mask_offset(m);
  int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (e == 0 && used) *used = off;
  for (; e < n; e += (int64_t)gridDim.x * blockDim.x)
    y[e] = keep_at(m, off, (uint64_t)e) ? (T)((float)x[e] * f) : (T)0.0f;
}

// ------------------------------------------------------------------------------------------ lookup
template <typename TT, typename OT, typename IT>
__global__ void embedding_kernel(const TT* table, int64_t stride, const IT* ids, int64_t N, int64_t V, int64_t D,
                                 OT* out, Mask m, float f, uint64_t* used, int* oob) {
  const uint64_t off = mask_offset(m);
  int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (e == 0 && used) *used = off;
  for (; e < N * D; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t n = e / D, d = e - n * D;
    const int64_t id = (int64_t)ids[n];
    const bool bad = id < 0 || id >= V;
    if (bad && oob) *oob = 1;
    out[e] = (!bad && keep_at(m, off, (uint64_t)e)) ? (OT)((float)table[id * stride + d] * f) : (OT)0.0f;
  }
}

// ------------------------------------------------------------------------------------------ sort
// Stable least-significant-digit radix sort of (id, position) pairs. Ids that take no part in the gradient (outside
// the table, the padding row) get the key V, which sorts last. One pass: per-block digit counts, an exclusive scan of
// each digit's counts over the blocks, and a scatter in which a wave ranks equal digits by ballots, so that equal keys
// keep their order.
constexpr int kSortThreads = 256, kSortWaves = kSortThreads / 64, kSortItems = 16;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kBins = 256;

struct SortPlan {
  int passes, width;
  int64_t blocks;
};

inline SortPlan sort_plan(int64_t N, int64_t V) {
  int bits = 1;
  while (bits < 32 && (V >> bits)) ++bits;  // keys 0 .. V
  SortPlan s;
  s.passes = (bits + 7) / 8;
  s.width = (bits + s.passes - 1) / s.passes;
  s.blocks = (N + kSortTile - 1) / kSortTile;
  return s;
}

// first pass: keys come from the ids, positions are the indices themselves
template <typename IT>
struct KeyFromIds {
  const IT* ids;
  int64_t V, pad;
  __device__ __forceinline__ uint32_t key(int64_t i) const {
    const int64_t id = (int64_t)ids[i];
    return (uint32_t)((id < 0 || id >= V || id == pad) ? V : id);
  }
  __device__ __forceinline__ uint32_t pos(int64_t i) const { return (uint32_t)i; }
};
struct KeyFromPairs {
  const uint32_t *keys, *poss;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return keys[i]; }
  __device__ __forceinline__ uint32_t pos(int64_t i) const { return poss[i]; }
};

template <typename Src>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(Src src, int64_t N, int shift, int width,
                                                                  uint32_t* counts, int64_t blocks) {
  __shared__ uint32_t hist[kBins];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t mask = (1u << width) - 1;
  const int64_t base = (int64_t)blockIdx.x * kSortTile;
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * kSortThreads + threadIdx.x;
    if (i < N) atomicAdd(&hist[(src.key(i) >> shift) & mask], 1u);
  }
  __syncthreads();
  if (threadIdx.x <= mask) counts[threadIdx.x * blocks + blockIdx.x] = hist[threadIdx.x];
}

// exclusive scan of counts[digit][0 .. blocks) in place, one workgroup a digit; its sum into totals[digit]
__global__ __launch_bounds__(256) void sort_scan_kernel(uint32_t* counts, int64_t blocks, uint32_t* totals) {
  __shared__ uint32_t part[256];
  uint32_t* c = counts + (int64_t)blockIdx.x * blocks;
  uint32_t run = 0;
  for (int64_t b0 = 0; b0 < blocks; b0 += 256) {
    const int64_t b = b0 + threadIdx.x;
    const uint32_t v = b < blocks ? c[b] : 0u;
    part[threadIdx.x] = v;
    __syncthreads();
    for (int o = 1; o < 256; o <<= 1) {
      const uint32_t t = threadIdx.x >= (unsigned)o ? part[threadIdx.x - o] : 0u;
      __syncthreads();
      part[threadIdx.x] += t;
      __syncthreads();
    }
    if (b < blocks) c[b] = run + part[threadIdx.x] - v;
    run += part[255];
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

// lanes of this wave whose digit equals this lane's
__device__ __forceinline__ uint64_t wave_match(uint32_t digit, int width, bool valid) {
  uint64_t peers = __ballot(valid);
  for (int b = 0; b < width; ++b) {
    const uint64_t bal = __ballot((digit >> b) & 1);
    peers &= ((digit >> b) & 1) ? bal : ~bal;
  }
  return peers;
}

template <typename Src>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(Src src, int64_t N, int shift, int width,
                                                                    const uint32_t* counts, int64_t blocks,
                                                                    const uint32_t* totals, uint32_t* keys_out,
                                                                    uint32_t* pos_out) {
  __shared__ volatile uint32_t cnt[kSortWaves][kBins];  // a wave's count of each digit so far, then its first slot
  __shared__ uint32_t scan[kBins];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const uint32_t mask = (1u << width) - 1;
  for (int w = 0; w < kSortWaves; ++w) cnt[w][threadIdx.x] = 0;
  const uint32_t total = threadIdx.x <= mask ? totals[threadIdx.x] : 0u;
  scan[threadIdx.x] = total;
  __syncthreads();
  for (int o = 1; o < kBins; o <<= 1) {
    const uint32_t t = threadIdx.x >= (unsigned)o ? scan[threadIdx.x - o] : 0u;
    __syncthreads();
    scan[threadIdx.x] += t;
    __syncthreads();
  }
  const int64_t base = (int64_t)blockIdx.x * kSortTile + wave * (64 * kSortItems);
  uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * 64 + lane;
    key[j] = i < N ? src.key(i) : 0u;
  }
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const bool valid = base + j * 64 + lane < N;
    const uint32_t dig = (key[j] >> shift) & mask;
    const uint64_t peers = wave_match(dig, width, valid);
    const uint32_t below = __popcll(peers & ((1ull << lane) - 1));
    const uint32_t before = cnt[wave][dig];
    rank[j] = before + below;
    __builtin_amdgcn_wave_barrier();
    if (valid && below == 0) cnt[wave][dig] = before + __popcll(peers);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if (threadIdx.x <= mask) {
    uint32_t at = scan[threadIdx.x] - total + counts[threadIdx.x * blocks + blockIdx.x];
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = cnt[w][threadIdx.x];
      cnt[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSortItems; ++j) {
    const int64_t i = base + j * 64 + lane;
    if (i < N) {
      const uint32_t to = cnt[wave][(key[j] >> shift) & mask] + rank[j];
      keys_out[to] = key[j];
      pos_out[to] = src.pos(i);
    }
  }
}

// ------------------------------------------------------------------------------------------ gradient
__device__ __forceinline__ int64_t lower_bound(const uint32_t* keys, int64_t N, uint32_t v) {
  int64_t lo = 0, hi = N;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// one wave a row of the table: its terms in the order of their positions
template <typename GT, typename TT>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const GT* g, const uint32_t* keys, const uint32_t* pos,
                                                             int64_t N, int64_t V, int64_t D, Mask m, float f,
                                                             TT* grad) {
  const int lane = threadIdx.x & 63;
  const uint64_t off = mask_offset(m);
  for (int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); v < V; v += (int64_t)gridDim.x * 4) {
    const int64_t a = lower_bound(keys, N, (uint32_t)v), b = lower_bound(keys, N, (uint32_t)v + 1);
    for (int64_t d = lane; d < D; d += 64) {
      float s = 0.0f;
      for (int64_t i = a; i < b; ++i) {
        const int64_t e = (int64_t)pos[i] * D + d;
        if (keep_at(m, off, (uint64_t)e)) s += (float)g[e];
      }
      grad[v * D + d] = (TT)(s * f);
    }
  }
}

// ------------------------------------------------------------------------------------------ workspace
struct GradWs {
  int64_t counts, totals, keys[2], pos[2], bytes;
};

inline GradWs grad_ws(int64_t N, int64_t V) {
  const SortPlan s = sort_plan(N, V);
  GradWs w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  w.counts = take(kBins * s.blocks * 4);
  w.totals = take(kBins * 4);
  for (int i = 0; i < 2; ++i) {
    w.keys[i] = take(N * 4);
    w.pos[i] = take(N * 4);
  }
  w.bytes = at;
  return w;
}

template <typename Src>
inline void sort_pass(Src src, int64_t N, int pass, const SortPlan& s, char* ws, const GradWs& w, hipStream_t st) {
  uint32_t* counts = (uint32_t*)(ws + w.counts);
  uint32_t* totals = (uint32_t*)(ws + w.totals);
  const int shift = pass * s.width;
  hipLaunchKernelGGL(sort_count_kernel<Src>, dim3((unsigned)s.blocks), dim3(kSortThreads), 0, st, src, N, shift,
                     s.width, counts, s.blocks);
  hipLaunchKernelGGL(sort_scan_kernel, dim3(1u << s.width), dim3(256), 0, st, counts, s.blocks, totals);
  hipLaunchKernelGGL(sort_scatter_kernel<Src>, dim3((unsigned)s.blocks), dim3(kSortThreads), 0, st, src, N, shift,
                     s.width, counts, s.blocks, totals, (uint32_t*)(ws + w.keys[pass & 1]),
                     (uint32_t*)(ws + w.pos[pass & 1]));
}

// sizes that the kernels' 32-bit positions and keys, and the grids, hold
inline int embedding_sizes_ok(const char* what, int64_t N, int64_t V, int64_t D) {
  YN_CHECK(N >= 0 && V >= 0 && D >= 0, "%s: negative size", what);
  YN_CHECK(N < (1ll << 31) && V < (1ll << 31), "%s: N=%lld or V=%lld is 2^31 or more", what, (long long)N, (long long)V);
  YN_CHECK(D <= (1ll << 31) && (D == 0 || (N <= (1ll << 38) / D && V <= (1ll << 38) / D)),
           "%s: more than 2^38 elements", what);
  return 0;
}
inline int mask_args_ok(const char* what, double p) {
  YN_CHECK(p >= 0.0 && p <= 1.0, "%s: p=%g is not a probability", what, p);
  return 0;
}

}  // namespace yanerf

using namespace yanerf;

extern "C" {

int yanerf_dropout(const void* x, int type, int64_t n, double p, uint64_t seed, uint64_t offset,
                   const uint64_t* rng_base, uint64_t* rng_used, void* y, void* stream) {
  YN_CHECK(type_ok(type), "dropout: unknown element type %d", type);
  YN_CHECK(n >= 0 && n <= (1ll << 38), "dropout: n=%lld out of range", (long long)n);
  if (mask_args_ok("dropout", p)) return 1;
  if (n == 0) return 0;
  YN_CHECK(x && y, "dropout: null pointer");
  const Mask m = make_mask(p, seed, offset, rng_base);
  const float f = (float)mask_scale(p, m);
  with_type(type, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(dropout_kernel<T>, grid_for((n + 255) / 256), dim3(256), 0, as_stream(stream),
                       (const T*)x, (T*)y, n, m, f, rng_used);
  });
  YN_LAUNCH_CHECK("dropout");
  return 0;
}

int yanerf_embedding_forward(const void* table, int table_type, int64_t table_stride, const void* ids, int id_bytes,
                             int64_t N, int64_t V, int64_t D, double scale, double p, uint64_t seed, uint64_t offset,
                             const uint64_t* rng_base, uint64_t* rng_used, void* out, int out_type, int* oob,
                             void* stream) {
  YN_CHECK(type_ok(table_type) && type_ok(out_type), "embedding: unknown element type %d / %d", table_type, out_type);
  YN_CHECK(id_bytes == 4 || id_bytes == 8, "embedding: ids of %d bytes", id_bytes);
  if (embedding_sizes_ok("embedding", N, V, D) || mask_args_ok("embedding", p)) return 1;
  YN_CHECK(std::isfinite(scale), "embedding: scale is not finite");
  if (N == 0 || D == 0) return 0;
  YN_CHECK(V >= 1, "embedding: an empty table");
  YN_CHECK(table && ids && out, "embedding: null pointer");
  YN_CHECK(table_stride >= 0, "embedding: negative table stride");
  const Mask m = make_mask(p, seed, offset, rng_base);
  const float f = (float)(scale * mask_scale(p, m));
  with_type(table_type, [&](auto tt) {
    with_type(out_type, [&](auto ot) {
      using TT = decltype(tt);
      using OT = decltype(ot);
      const dim3 grid = grid_for((N * D + 255) / 256);
      if (id_bytes == 8)
        hipLaunchKernelGGL((embedding_kernel<TT, OT, int64_t>), grid, dim3(256), 0, as_stream(stream),
                           (const TT*)table, table_stride, (const int64_t*)ids, N, V, D, (OT*)out, m, f, rng_used, oob);
      else
        hipLaunchKernelGGL((embedding_kernel<TT, OT, int32_t>), grid, dim3(256), 0, as_stream(stream),
                           (const TT*)table, table_stride, (const int32_t*)ids, N, V, D, (OT*)out, m, f, rng_used, oob);
    });
  });
  YN_LAUNCH_CHECK("embedding");
  return 0;
}

int64_t yanerf_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t D) {
  if (embedding_sizes_ok("embedding_bwd_workspace", N, V, D)) return -1;
  return N == 0 || V == 0 || D == 0 ? 0 : grad_ws(N, V).bytes;
}

int yanerf_embedding_backward(const void* g, int g_type, const void* ids, int id_bytes, int64_t N, int64_t V,
                              int64_t D, int64_t padding_idx, double scale, double p, uint64_t seed, uint64_t offset,
                              const uint64_t* rng_base, void* grad_table, int table_type, void* workspace,
                              void* stream) {
  YN_CHECK(type_ok(table_type) && type_ok(g_type), "embedding_backward: unknown element type %d / %d", table_type,
           g_type);
  YN_CHECK(id_bytes == 4 || id_bytes == 8, "embedding_backward: ids of %d bytes", id_bytes);
  if (embedding_sizes_ok("embedding_backward", N, V, D) || mask_args_ok("embedding_backward", p)) return 1;
  YN_CHECK(std::isfinite(scale), "embedding_backward: scale is not finite");
  YN_CHECK(padding_idx >= -1 && padding_idx < (V > 0 ? V : 1), "embedding_backward: padding_idx=%lld outside the table",
           (long long)padding_idx);
  if (V == 0 || D == 0) return 0;
  YN_CHECK(grad_table, "embedding_backward: null pointer");
  YN_CHECK(N == 0 || (g && ids && workspace), "embedding_backward: null pointer");
  const Mask m = make_mask(p, seed, offset, rng_base);
  const float f = (float)(scale * mask_scale(p, m));
  hipStream_t st = as_stream(stream);
  char* ws = (char*)workspace;
  const GradWs w = grad_ws(N, V);
  const SortPlan s = sort_plan(N, V);
  if (N > 0)
    for (int pass = 0; pass < s.passes; ++pass) {
      if (pass > 0)
        sort_pass(KeyFromPairs{(const uint32_t*)(ws + w.keys[(pass - 1) & 1]),
                               (const uint32_t*)(ws + w.pos[(pass - 1) & 1])}, N, pass, s, ws, w, st);
      else if (id_bytes == 8)
        sort_pass(KeyFromIds<int64_t>{(const int64_t*)ids, V, padding_idx}, N, pass, s, ws, w, st);
      else
        sort_pass(KeyFromIds<int32_t>{(const int32_t*)ids, V, padding_idx}, N, pass, s, ws, w, st);
    }
  const int last = (s.passes - 1) & 1;
  with_type(g_type, [&](auto gt) {
    with_type(table_type, [&](auto tt) {
      using GT = decltype(gt);
      using TT = decltype(tt);
      hipLaunchKernelGGL((embedding_rows_kernel<GT, TT>), grid_for((V + 3) / 4), dim3(256), 0, st,
                         (const GT*)g, (const uint32_t*)(ws + w.keys[last]), (const uint32_t*)(ws + w.pos[last]), N, V,
                         D, m, f, (TT*)grad_table);
    });
  });
  YN_LAUNCH_CHECK("embedding_backward");
  return 0;
}

}  // extern "C"
