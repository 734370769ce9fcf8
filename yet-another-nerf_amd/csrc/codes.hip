// Learned codes for gfx950: embedding lookup with scaling and dropout, its gradient by sorted ids, and dropout whose
// mask is a function of a Philox counter.
//
//   lookup   out[n, d] = f * table[ids[n], d] * keep(n D + d)                          f = scale / (1 - p)
//   gradient grad[v, d] = f * sum over n with ids[n] == v of keep(n D + d) * g[n, d]   (0 for the padding row)
//   dropout  y[e] = x[e] * keep(e) / (1 - p); its gradient is the same map
//
// keep(e) is 1 where word e % 4 of Philox4x32-10(key = seed, counter = (e / 4, offset)) is at least
// T = round(p 2^32): forward and backward evaluate it anew, so no mask is stored or read. A dropped element is 0
// whatever its input holds. Sums are fp32, products with f too but the gradient's, which is taken in 64 bits; each output
// is rounded once more, to its type.
//
// The gradient groups the positions of each row with stable sorts, so the terms of a row are added in an order that the call
// fixes (its ids, sizes, types and alignment): no float atomics, the same bits on every run. Which way depends on the sizes:
//
//   N <= 4096, gradient <= 32 MB            one launch, each workgroup picks the ids of its own rows (own_rows_kernel)
//   V <= 32                                 one pass over g with a table a lane (dense_sum_kernel)
//   N > 16384, rows of g of <= 16 bytes     one partition that carries the rows along (bucket_sum_kernel)
//   the rest                                a sort of (id, position) pairs, then sums over pieces of the sorted list
//                                           (rank_sort_kernel to N = 16384, sort_scatter_kernel beyond; run_sum_kernel)
#include <cfloat>
#include <cmath>
#include <type_traits>

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

// f(I{}) with I the index type of `bytes`
template <typename F>
inline void with_index(int bytes, F&& f) {
  if (bytes == 8) f(int64_t{});
  else f(int32_t{});
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

// scale / (1 - p), 0 where everything is dropped
inline double mask_scale(double scale, double p, const Mask& m) { return m.mode == 2 ? 0.0 : scale / (1.0 - p); }

__device__ __forceinline__ uint64_t mask_offset(const Mask& m) { return m.offset + (m.base ? *m.base : 0ull); }

// keep of the elements 4 q .. 4 q + 3
struct Keep4 {
  bool k[4];
};
__device__ __forceinline__ Keep4 keep_group(const Mask& m, uint64_t off, uint64_t q) {
  if (m.mode != 1) {
    const bool k = m.mode == 0;
    return {{k, k, k, k}};
  }
  const u4 r = philox(m.seed, off, q);
  return {{r.x >= m.threshold, r.y >= m.threshold, r.z >= m.threshold, r.w >= m.threshold}};
}

// zeros where the VEC elements from e, a multiple of VEC, are dropped
template <int VEC>
__device__ __forceinline__ void apply_keep(const Mask& m, uint64_t off, int64_t e, float (&v)[VEC]) {
  if constexpr (VEC >= 4) {
#pragma unroll
    for (int q = 0; q < VEC / 4; ++q) {
      const Keep4 keep = keep_group(m, off, (uint64_t)(e >> 2) + q);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[4 * q + k] = keep.k[k] ? v[4 * q + k] : 0.0f;
    }
  } else {
    const Keep4 keep = keep_group(m, off, (uint64_t)(e >> 2));
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      const bool odd = VEC == 1 && (e & 1);
      const bool lo = odd ? keep.k[1] : keep.k[k], hi = odd ? keep.k[3] : keep.k[2 + k];
      v[k] = ((e & 2) ? hi : lo) ? v[k] : 0.0f;
    }
  }
}

// ------------------------------------------------------------------------------------------ vectors
template <int BYTES>
struct RawOf;
template <>
struct RawOf<2> {
  typedef uint16_t type;
};
template <>
struct RawOf<4> {
  typedef uint32_t type;
};
template <>
struct RawOf<8> {
  typedef uint32_t type __attribute__((ext_vector_type(2)));
};
template <>
struct RawOf<16> {
  typedef uint32_t type __attribute__((ext_vector_type(4)));
};

// VEC elements at p as floats: one load of up to 16 bytes where ALIGNED, else VEC loads
template <typename T, int VEC, bool ALIGNED, bool NT>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
  if constexpr (ALIGNED) {
    typedef typename RawOf<VEC * sizeof(T)>::type R;
    struct A {
      T t[VEC];
    };
    const R r = NT ? __builtin_nontemporal_load((const R*)p) : *(const R*)p;
    const A a = __builtin_bit_cast(A, r);
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = (float)a.t[k];
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = (float)p[k];
  }
}
template <typename T, int VEC, bool ALIGNED, bool NT>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (ALIGNED && VEC * sizeof(T) == 32) {
    const float lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
    store_vec<T, 4, true, NT>(p, lo);
    store_vec<T, 4, true, NT>(p + 4, hi);
  } else if constexpr (ALIGNED) {
    typedef typename RawOf<VEC * sizeof(T)>::type R;
    struct A {
      T t[VEC];
    };
    A a;
#pragma unroll
    for (int k = 0; k < VEC; ++k) a.t[k] = (T)v[k];
    const R r = __builtin_bit_cast(R, a);
    if (NT) __builtin_nontemporal_store(r, (R*)p);
    else *(R*)p = r;
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) p[k] = (T)v[k];
  }
}

// unsigned division by a number fixed for a launch, for dividends below 2^31: n / d = (n * mul) >> shift
struct Div {
  uint32_t d, mul;
  int shift;
};
inline Div make_div(int64_t d) {
  int s = 0;
  while ((1ll << s) < d) ++s;
  return {(uint32_t)d, (uint32_t)((1ull << (31 + s)) / (uint64_t)d + 1), 31 + s};
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, const Div& d) {
  return (uint32_t)(((uint64_t)n * d.mul) >> d.shift);
}

inline bool aligned(const void* p, int64_t bytes) { return ((uintptr_t)p & (uint64_t)(bytes - 1)) == 0; }

// ------------------------------------------------------------------------------------------ dropout
// Bound by the bytes of x and y: 16 bytes a lane each way, loaded before anything else is looked at, and one Philox call
// for every 4 elements hides behind them. A lane takes one vector: loops over more of them measured 10 % slower. 201 M bf16
// values: 142 to 145 us for a launch by itself, 5.6 TB/s, and 134 us for each of a row of launches (a copy of them by torch
// 151 us); 33.5 M fp32 values: 42 us, 6.4 TB/s.
template <typename T, bool ALIGNED, bool NT>
__global__ __launch_bounds__(256) void dropout_kernel(const T* x, T* y, int64_t n, int64_t first, Mask m, float f,
                                                      uint64_t* used) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t e = first + ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC;
  if (e >= n) return;
  float v[VEC];
  const bool whole = e + VEC <= n;
  if (whole) {
    load_vec<T, VEC, ALIGNED, NT>(x + e, v);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = e + k < n ? (float)x[e + k] : 0.0f;
  }
  const uint64_t off = mask_offset(m);
  if (e == 0 && used) *used = off;
#pragma unroll
  for (int k = 0; k < VEC; ++k) v[k] *= f;
  if (m.mode != 0) apply_keep<VEC>(m, off, e, v);
  if (whole) {
    store_vec<T, VEC, ALIGNED, NT>(y + e, v);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (e + k < n) y[e + k] = (T)v[k];
  }
}

// ------------------------------------------------------------------------------------------ flags
// The flag of ids outside their table that lookups without one of their own set: a variable of the library and not an
// allocation, so that it is there, cleared, before the first lookup (also where that one is captured into a graph) and never
// moves.
__device__ int id_flag = 0;

// lookups on other streams may set a flag while it is taken
__device__ __forceinline__ void set_flag(int* flag) {
  __hip_atomic_store(flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__global__ void take_flag_kernel(int* flag, int* taken) {
  *taken = __hip_atomic_exchange(flag, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ------------------------------------------------------------------------------------------ lookup
// A workgroup takes `rows` consecutive ids. Rows of whole vectors: lane t of the tile's rows * D / VEC vectors copies one,
// kUnroll of them in flight (1, 2 and 8 measured the same or up to 10 % slower). The ids and hot rows come from L1 / L2, so
// the output's bytes bound it: 640000 x 16 bf16 7.4 us (20 MB out), 6.3 M x 2 fp32 21 us (50 MB out, 8 bytes a lane);
// with dropout Philox does, 16384 x 1024 bf16 16.0 us.
constexpr int kUnroll = 4;

template <typename TT, typename OT, typename IT, int VEC, bool NT>
__global__ __launch_bounds__(256) void embedding_rows_of_vectors_kernel(const TT* table, int64_t stride, const IT* ids,
                                                                        int64_t N, int64_t V, Div dv, int rows, OT* out,
                                                                        Mask m, float f, uint64_t* used, int* oob) {
  const uint64_t off = mask_offset(m);
  if (blockIdx.x == 0 && threadIdx.x == 0 && used) *used = off;
  for (int64_t n0 = (int64_t)blockIdx.x * rows; n0 < N; n0 += (int64_t)gridDim.x * rows) {
    const uint32_t total = (uint32_t)(N - n0 < rows ? N - n0 : rows) * dv.d;
    for (uint32_t t0 = threadIdx.x; t0 < total; t0 += 256 * kUnroll) {
      float v[kUnroll][VEC];
      int64_t id[kUnroll];
      uint32_t col[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const uint32_t t = t0 + u * 256;
        if (t < total) {
          const uint32_t r = div_by(t, dv);
          col[u] = t - r * dv.d;
          id[u] = (int64_t)ids[n0 + r];
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (t0 + u * 256 < total) {
          if (id[u] >= 0 && id[u] < V) {
            load_vec<TT, VEC, true, false>(table + id[u] * stride + (int64_t)col[u] * VEC, v[u]);
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[u][k] *= f;
          } else {
            if (oob) set_flag(oob);
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[u][k] = 0.0f;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const uint32_t t = t0 + u * 256;
        if (t < total) {
          const int64_t i = n0 * dv.d + t;  // the vector's index in the output
          if (m.mode != 0) apply_keep<VEC>(m, off, i * VEC, v[u]);
          store_vec<OT, VEC, true, NT>(out + i * VEC, v[u]);
        }
      }
    }
  }
}

// Any other row length, stride or alignment: a lane takes 4 consecutive elements of the output, wherever rows begin, so
// that one Philox call still serves 4 of them and stores stay wide. `rows` is a multiple of 4. 10007 x 37 fp16: 4.2 us.
template <typename TT, typename OT, typename IT, bool ALIGNED>
__global__ __launch_bounds__(256) void embedding_any_rows_kernel(const TT* table, int64_t stride, const IT* ids,
                                                                 int64_t N, int64_t V, Div dd, int rows, OT* out, Mask m,
                                                                 float f, uint64_t* used, int* oob) {
  const uint64_t off = mask_offset(m);
  if (blockIdx.x == 0 && threadIdx.x == 0 && used) *used = off;
  for (int64_t n0 = (int64_t)blockIdx.x * rows; n0 < N; n0 += (int64_t)gridDim.x * rows) {
    const uint32_t total = (uint32_t)(N - n0 < rows ? N - n0 : rows) * dd.d;
    for (uint32_t t = threadIdx.x * 4; t < total; t += 256 * 4) {
      uint32_t r = div_by(t, dd), c = t - r * dd.d;
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[k] = 0.0f;
        if (t + k < total) {
          const int64_t id = (int64_t)ids[n0 + r];
          if (id >= 0 && id < V) v[k] = (float)table[id * stride + c] * f;
          else if (oob) set_flag(oob);
        }
        if (++c == dd.d) {
          c = 0;
          ++r;
        }
      }
      const int64_t e = n0 * dd.d + t;
      if (m.mode != 0) {
        const Keep4 keep = keep_group(m, off, (uint64_t)e >> 2);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = keep.k[k] ? v[k] : 0.0f;
      }
      if (t + 4 <= total) {
        store_vec<OT, 4, ALIGNED, false>(out + e, v);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (t + k < total) out[e + k] = (OT)v[k];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ sort
// Stable sorts of (id, position) pairs by id. Ids that take no part in the gradient (outside the table, the padding row)
// get a key past the table (`none`), which sorts last.
struct Pair {
  uint32_t key, pos;
};

// where keys come from: the ids (positions are the indices themselves), or pairs
template <typename IT>
struct KeyFromIds {
  const IT* ids;
  int64_t V, pad;
  uint32_t none;
  __device__ __forceinline__ Pair at(int64_t i) const {
    const int64_t id = (int64_t)ids[i];
    return {id < 0 || id >= V || id == pad ? none : (uint32_t)id, (uint32_t)i};
  }
};
struct KeyFromPairs {
  const Pair* pairs;
  __device__ __forceinline__ Pair at(int64_t i) const {
    return __builtin_bit_cast(Pair, *(const uint64_t*)(pairs + i));
  }
};
__device__ __forceinline__ void store_pair(Pair* to, Pair p) { *(uint64_t*)to = __builtin_bit_cast(uint64_t, p); }

// Long lists: least-significant-digit radix sort, digits of up to 10 bits. A pass counts the digits of each tile, scans each
// digit's counts over the tiles, and scatters: a wave ranks equal digits by ballots, so that equal keys keep their order,
// and a tile's pairs are first put in order in LDS, so that they leave as runs and not one by one. With no more than
// kFewTiles tiles the scatter reads the counts of all of them itself and the scan's launch is left out. Bound by the
// ranking's vector instructions (half the time) and the latency of its LDS counters: 2 M pairs of 300000 rows, two passes of
// 10 bits: 5.3 + 6.2 + 15.6 us a pass.
constexpr int64_t kFewTiles = 64;
// lanes and pairs a lane: small tiles while they are few, else 4096 by 8 waves (6.3 M pairs, 1024 bins: 512 x 8 52 us,
// 256 x 16 55, 1024 x 8 61, 512 x 16 71, 1024 x 16 109)
constexpr int kFewThreads = 256, kFewItems = 8, kTileThreads = 512, kTileItems = 8;

struct SortPlan {
  int passes, width, bins;
  bool few;
  int64_t tiles;
};

inline SortPlan sort_plan(int64_t N, int64_t V) {
  int bits = 1;
  while (bits < 32 && (V >> bits)) ++bits;  // keys 0 .. V
  SortPlan s;
  s.passes = (bits + 9) / 10;
  s.width = (bits + s.passes - 1) / s.passes;
  s.bins = s.width <= 8 ? 256 : 1024;
  s.few = N <= kFewTiles * kFewThreads * kFewItems;
  const int64_t tile = s.few ? kFewThreads * kFewItems : kTileThreads * kTileItems;
  s.tiles = (N + tile - 1) / tile;
  return s;
}

template <typename Src, int BINS, int THREADS, int ITEMS>
__global__ __launch_bounds__(THREADS) void sort_count_kernel(Src src, int64_t N, int shift, int width, uint32_t* counts) {
  // neighbouring ids often share a digit: copies of the counts, by lane, keep them from waiting for one another
  constexpr int COPIES = 4;
  __shared__ uint32_t hist[BINS * COPIES];
  for (int k = threadIdx.x; k < BINS * COPIES; k += THREADS) hist[k] = 0;
  __syncthreads();
  const uint32_t mask = (1u << width) - 1;
  const int64_t base = (int64_t)blockIdx.x * (THREADS * ITEMS) + threadIdx.x;
  uint32_t key[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) key[j] = base + j * THREADS < N ? src.at(base + j * THREADS).key : 0u;
#pragma unroll
  for (int j = 0; j < ITEMS; ++j)
    if (base + j * THREADS < N) atomicAdd(&hist[((key[j] >> shift) & mask) * COPIES + threadIdx.x % COPIES], 1u);
  __syncthreads();
  for (int k = threadIdx.x; k < BINS; k += THREADS) {
    uint32_t sum = 0;
#pragma unroll
    for (int c = 0; c < COPIES; ++c) sum += hist[k * COPIES + c];
    counts[(int64_t)blockIdx.x * BINS + k] = sum;
  }
}

// sum of v over the lanes before this one, of the whole workgroup's in `total`; part has a slot a wave
template <int WAVES>
__device__ __forceinline__ uint32_t block_exclusive_scan(uint32_t v, uint32_t* part, uint32_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = __shfl_up(inc, o, 64);
    if (lane >= o) inc += t;
  }
  __syncthreads();  // part may still be read from an earlier call
  if (lane == 63) part[wave] = inc;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    before += w < wave ? part[w] : 0u;
    total += part[w];
  }
  return before + inc - v;
}

// exclusive scan of counts[0 .. tiles)[digit] in place, 16 digits a workgroup, whose 64 parts take consecutive tiles; the
// digits' sums into totals
constexpr int kScanDigits = 16, kScanParts = 64, kScanThreads = kScanDigits * kScanParts;
__global__ __launch_bounds__(kScanThreads) void sort_scan_kernel(uint32_t* counts, int64_t tiles, int bins,
                                                                 uint32_t* totals) {
  __shared__ uint32_t sums[kScanParts][kScanDigits];
  const int dig = threadIdx.x % kScanDigits, part = threadIdx.x / kScanDigits;
  const int64_t per = (tiles + kScanParts - 1) / kScanParts;
  const int64_t begin = part * per, end = begin + per < tiles ? begin + per : tiles;
  uint32_t* c = counts + blockIdx.x * kScanDigits + dig;
  uint32_t sum = 0;
#pragma unroll 8
  for (int64_t t = begin; t < end; ++t) sum += c[t * bins];
  sums[part][dig] = sum;
  __syncthreads();
  uint32_t at = 0, total = 0;
#pragma unroll 16
  for (int q = 0; q < kScanParts; ++q) {
    at += q < part ? sums[q][dig] : 0u;
    total += sums[q][dig];
  }
  for (int64_t t = begin; t < end; t += 8) {  // loads of 8 before their stores, which the compiler cannot move them past
    uint32_t v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = t + k < end ? c[(t + k) * bins] : 0u;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (t + k < end) c[(t + k) * bins] = at;
      at += v[k];
    }
  }
  if (part == 0) totals[blockIdx.x * kScanDigits + dig] = total;
}

// what the wave's lanes wrote to LDS before is what they read from it after (LDS serves a wave in order; this keeps the
// compiler to it)
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// lanes of this wave whose digit, of `bits` bits, equals this lane's
__device__ __forceinline__ uint64_t wave_match(uint32_t digit, int bits, bool valid) {
  const uint64_t all = __ballot(valid);
  uint32_t lo = (uint32_t)all, hi = (uint32_t)(all >> 32);
  for (int b = 0; b < bits; ++b) {
    const uint64_t bal = __ballot((digit >> b) & 1);
    const uint32_t same = (digit >> b) & 1 ? 0u : ~0u;
    lo &= (uint32_t)bal ^ same;
    hi &= (uint32_t)(bal >> 32) ^ same;
  }
  return ((uint64_t)hi << 32) | lo;
}

struct StorePairs {
  Pair* out;
  __device__ __forceinline__ void operator()(int64_t to, Pair p) const { store_pair(out + to, p); }
};

template <typename Src, typename Dst, int BINS, int THREADS, int ITEMS>
__global__ __launch_bounds__(THREADS) void sort_scatter_kernel(Src src, int64_t N, int shift, int width,
                                                               const uint32_t* counts, int64_t tiles,
                                                               const uint32_t* totals, Dst dst) {
  constexpr int WAVES = THREADS / 64, PER = (BINS + THREADS - 1) / THREADS, TILE = THREADS * ITEMS;
  __shared__ union {
    uint32_t cnt[WAVES][BINS];  // a wave's count of each digit so far, then its first slot
    uint64_t sorted[TILE];      // the tile in order, once every lane knows its slots
  } u;
  __shared__ uint32_t delta[BINS];  // place in the output less place in the tile
  __shared__ uint32_t part[WAVES];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t mask = (1u << width) - 1;
  for (int k = tid; k < WAVES * BINS; k += THREADS) (&u.cnt[0][0])[k] = 0;
  const int64_t base = (int64_t)blockIdx.x * TILE;
  const int64_t mine = base + wave * (64 * ITEMS) + lane;
  Pair p[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) p[j] = mine + j * 64 < N ? src.at(mine + j * 64) : Pair{0, 0};
  // where this tile's digits go: the digit's own place, after the same digit of the tiles before
  uint32_t place[PER], sum = 0, all;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const uint32_t dig = tid * PER + k;
    uint32_t before = 0, total = 0;
    if (dig <= mask) {
      const uint32_t* c = counts + dig;
      if (totals) {
        before = c[(int64_t)blockIdx.x * BINS];
        total = totals[dig];
      } else {
#pragma unroll 8
        for (int t = 0; t < (int)tiles; ++t) {
          const uint32_t v = c[t * BINS];
          before += t < (int)blockIdx.x ? v : 0u;
          total += v;
        }
      }
    }
    place[k] = sum + before;
    sum += total;
  }
  const uint32_t digit_base = block_exclusive_scan<WAVES>(sum, part, all);
  __syncthreads();
  uint32_t rank[ITEMS];
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const bool valid = mine + j * 64 < N;
    const uint32_t dig = (p[j].key >> shift) & mask;
    const uint64_t peers = wave_match(dig, width, valid);
    const uint32_t below = __popcll(peers & ((1ull << lane) - 1));
    const uint32_t before = u.cnt[wave][dig];
    rank[j] = before + below;
    wave_fence();
    if (valid && below == 0) u.cnt[wave][dig] = before + __popcll(peers);
    wave_fence();
  }
  __syncthreads();
  sum = 0;
  uint32_t here[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    here[k] = sum;
    if (tid * PER + k < BINS) {
#pragma unroll
      for (int w = 0; w < WAVES; ++w) sum += u.cnt[w][tid * PER + k];
    }
  }
  const uint32_t first = block_exclusive_scan<WAVES>(sum, part, all);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int dig = tid * PER + k;
    if (dig >= BINS) break;
    uint32_t at = first + here[k];
    delta[dig] = digit_base + place[k] - at;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const uint32_t c = u.cnt[w][dig];
      u.cnt[w][dig] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) rank[j] += u.cnt[wave][(p[j].key >> shift) & mask];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < ITEMS; ++j)
    if (mine + j * 64 < N) u.sorted[rank[j]] = __builtin_bit_cast(uint64_t, p[j]);
  __syncthreads();
  const uint32_t held = (uint32_t)(N - base < TILE ? N - base : TILE);
#pragma unroll
  for (int j = 0; j < ITEMS; ++j) {
    const uint32_t i = tid + j * THREADS;
    if (i < held) {
      const Pair q = __builtin_bit_cast(Pair, u.sorted[i]);
      dst((int64_t)(delta[(q.key >> shift) & mask] + i), q);
    }
  }
}

// Short lists are sorted in one launch: the place of a pair is the number of pairs below it. Every workgroup places
// kRankTile pairs and holds all of them in LDS, as (key << 14) | index, so that they all differ. It deals them into bins
// (LDS atomics: the order inside a bin does not matter, only its members do); a pair's place is then the bin's start and the
// count of the bin's members below it. A wave compares one pair with 64 others in one v_cmp, whose lanes the scalar unit
// counts. Bins are as wide as 1/64 of their keys: word frequencies, which fall with the id, would put a third of the ids
// into the first of 2048 equal bins (38 us for 16384 ids; counting against all pairs 37). Bound by the latency of its LDS
// phases: 10007 ids 12.4 us, 16384 ids 17.4 us.
constexpr int kIndexBits = 14;
constexpr int64_t kRankMax = 1 << kIndexBits;
constexpr int kRankThreads = 1024, kRankWaves = kRankThreads / 64, kRankItems = 4, kRankTile = kRankWaves * kRankItems;
constexpr int kRankBins = 2048;
// The bin of a pair, rising with it: of 1 / 64 of the key (at most 1727), or, where a small table leaves bins over, of the
// key and the leading `index_bits` bits of the index (a row that every id names would otherwise fill one bin).
struct RankBins {
  int index_bits;
  __device__ __forceinline__ uint32_t operator()(uint32_t key, uint32_t index) const {
    if (index_bits) return (key << index_bits) | (index >> (kIndexBits - index_bits));
    const int e = key < 64 ? 0 : 25 - __builtin_clz(key);
    return (e << 6) + (key >> e);
  }
};
inline RankBins rank_bins(int64_t V) {  // keys 0 .. V
  int b = kIndexBits;
  while (b > 0 && ((V + 1) << b) > kRankBins) --b;
  return {b};
}

// LDS: all pairs by bin
template <typename IT, typename P>
__global__ __launch_bounds__(kRankThreads) void rank_sort_kernel(KeyFromIds<IT> src, int N, RankBins bins,
                                                                 Pair* out) {
  extern __shared__ __attribute__((aligned(16))) char rank_lds[];
  P* binned = (P*)rank_lds;
  // a bin is dealt out in COPIES parts, by lane: word frequencies fill some bins with a third of the ids, and atomics on
  // one address wait for one another
  constexpr int COPIES = sizeof(P) == 4 ? 4 : 2, PER = kRankBins * COPIES / kRankThreads;
  __shared__ uint32_t start[kRankBins + 1], next[kRankBins * COPIES];
  __shared__ uint32_t part[kRankWaves];
  const int tid = threadIdx.x, lane = tid & 63, copy = lane % COPIES;
  constexpr int R = (int)(kRankMax / kRankThreads);
  for (int k = tid; k < kRankBins * COPIES; k += kRankThreads) next[k] = 0;
  __syncthreads();
  uint32_t key[R], place[R];  // place: among the pairs of this part of the bin, in whatever order they come
#pragma unroll
  for (int j = 0; j < R; ++j) key[j] = tid + j * kRankThreads < N ? src.at(tid + j * kRankThreads).key : 0u;
#pragma unroll
  for (int j = 0; j < R; ++j)
    if (tid + j * kRankThreads < N)
      place[j] = atomicAdd(&next[bins(key[j], tid + j * kRankThreads) * COPIES + copy], 1u);
  __syncthreads();
  uint32_t c[PER], sum = 0, all;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    c[k] = next[tid * PER + k];
    sum += c[k];
  }
  uint32_t at = block_exclusive_scan<kRankWaves>(sum, part, all);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    next[tid * PER + k] = at;
    if ((tid * PER + k) % COPIES == 0) start[(tid * PER + k) / COPIES] = at;
    at += c[k];
  }
  if (tid == kRankThreads - 1) start[kRankBins] = at;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const int i = tid + j * kRankThreads;
    if (i < N) binned[next[bins(key[j], i) * COPIES + copy] + place[j]] = ((P)key[j] << kIndexBits) | (P)i;
  }
  __syncthreads();
  const int first = blockIdx.x * kRankTile + (tid >> 6) * kRankItems;
  uint32_t item[kRankItems];
#pragma unroll
  for (int t = 0; t < kRankItems; ++t) item[t] = src.at(first + t < N ? first + t : N - 1).key;
#pragma unroll
  for (int t = 0; t < kRankItems; ++t) {
    if (first + t >= N) return;
    const uint32_t k = __builtin_amdgcn_readfirstlane(item[t]);
    const P mine = ((P)k << kIndexBits) | (P)(first + t);
    const uint32_t bin = bins(k, first + t);
    const uint32_t begin = __builtin_amdgcn_readfirstlane(start[bin]);
    const uint32_t end = __builtin_amdgcn_readfirstlane(start[bin + 1]);
    uint32_t rank = begin;
    for (uint32_t i = begin; i < end; i += 256) {
      P other[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) other[u] = i + u * 64 + lane < end ? binned[i + u * 64 + lane] : ~(P)0;
#pragma unroll
      for (int u = 0; u < 4; ++u) rank += __popcll(__ballot(other[u] < mine));
    }
    if (lane == 0) store_pair(out + rank, {k, (uint32_t)(first + t)});
  }
}

// ------------------------------------------------------------------------------------------ gradient
// A run is the sorted positions of one row. Sorted positions are cut into equal pieces whatever the runs' lengths are, so
// that a row named by most ids costs no more than many rows named once: a group of lanes (one vector of columns a lane)
// adds a piece, writes the rows whose runs lie inside it, and leaves the sums of the runs that its ends cut, which are then
// joined in the order of the pieces. Pieces depend on the sizes and the vector's width, runs on the ids: nothing else changes
// the order of a sum.
template <typename GT, int VEC>
__device__ __forceinline__ void masked_term(const GT* g, int64_t D, uint32_t pos, int64_t d, const Mask& m, uint64_t off,
                                            float (&v)[VEC]) {
  const int64_t e = (int64_t)pos * D + d;
  load_vec<GT, VEC, (VEC > 1), false>(g + e, v);
  if (m.mode != 0) apply_keep<VEC>(m, off, e, v);
}

// f * sum. In 64 bits: f is often a simple fraction (32 / 0.9 = 320 / 9), so that sums of few terms give products that lie
// half a step of bf16 or fp16 from both neighbours, and a factor rounded to fp32 would move them off the half. One product
// an output element: the kernels' times do not show it.
__device__ __forceinline__ float scaled(float sum, double f) { return (float)((double)sum * f); }

template <typename TT, int VEC>
__device__ __forceinline__ void write_row(TT* grad, int64_t D, int64_t row, int64_t d, double f, const float (&acc)[VEC]) {
  float v[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) v[k] = scaled(acc[k], f);
  store_vec<TT, VEC, (VEC > 1), false>(grad + row * D + d, v);
}

// What a workgroup's groups leave for each other in LDS: the sum of the run that entered a piece (head) and of the one
// that leaves it (tail)
enum { kHead = 1, kThrough = 2, kTail = 4 };
template <int THREADS, int VEC>
struct RunEnds {
  float head[THREADS * VEC], tail[THREADS * VEC];
  uint8_t flags[THREADS];
};

// Adds the sorted positions [0, N) of `src` that this workgroup's groups hold: group q the `piece` from base + q * piece.
// src.pair(i) holds the key that orders the runs and the row of g, src.row(key) is the row of the table; a key of
// src.none() takes no part. The runs that enter or leave the workgroup's span go to heads / tails [D], which a workgroup
// with the whole of [0, N) never writes.
template <int THREADS, typename GT, typename TT, int VEC, typename Src>
__device__ __forceinline__ void sum_runs(RunEnds<THREADS, VEC>& ends, const Src& src, int64_t N, int64_t base, int piece,
                                         int lg, const GT* g, int64_t D, int64_t d, const Mask& m, uint64_t off, double f,
                                         TT* grad, float* heads, float* tails) {
  constexpr int U = 8;
  const int groups = THREADS >> lg, group = threadIdx.x >> lg, sub = threadIdx.x & ((1 << lg) - 1);
  const bool col = d < D;
  const int64_t a = base + (int64_t)group * piece;
  const int64_t b = a + piece < N ? a + piece : N;
  const uint32_t none = src.none();
  float acc[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
  int flag = 0;
  uint32_t cur = none;
  if (a < N) {
    cur = src.key(a);
    bool cut = a > 0 && src.key(a - 1) == cur;  // the run began in an earlier piece
    for (int64_t i = a; i < b; i += U) {
      Pair q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = i + u < b ? src.pair(i + u) : Pair{none, 0u};
      float v[U][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (q[u].key != none && col) {
          masked_term<GT, VEC>(g, D, q[u].pos, d, m, off, v[u]);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) v[u][k] = 0.0f;
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u < b) {
          if (q[u].key != cur) {
            if (cut) {
#pragma unroll
              for (int k = 0; k < VEC; ++k) ends.head[threadIdx.x * VEC + k] = acc[k];
              flag |= kHead;
            } else if (col) {
              write_row<TT, VEC>(grad, D, src.row(cur), d, f, acc);
            }
            cut = false;
            cur = q[u].key;
#pragma unroll
            for (int k = 0; k < VEC; ++k) acc[k] = 0.0f;
          }
#pragma unroll
          for (int k = 0; k < VEC; ++k) acc[k] += v[u][k];
        }
      }
    }
    const bool goes_on = b < N && src.key(b) == cur;
    if (cur != none) {
      if (cut) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) ends.head[threadIdx.x * VEC + k] = acc[k];
        flag |= goes_on ? kHead | kThrough : kHead;
      } else if (goes_on) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) ends.tail[threadIdx.x * VEC + k] = acc[k];
        flag |= kTail;
      } else if (col) {
        write_row<TT, VEC>(grad, D, src.row(cur), d, f, acc);
      }
    }
  }
  if (sub == 0) ends.flags[group] = (uint8_t)flag;
  __syncthreads();
  const bool from_before = group == 0 && (flag & kHead);
  // two runs may leave group 0: the one that came in (its sum goes to `heads`) and the one it starts
  for (int which = from_before ? 0 : 1; which < 2; ++which) {
    if (which == 1 && !(flag & kTail)) break;
    float s[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) s[k] = (which ? ends.tail : ends.head)[threadIdx.x * VEC + k];
    bool open = which == 1 || (flag & kThrough);
    for (int h = group + 1; h < groups && open; ++h) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[k] += ends.head[(threadIdx.x + ((h - group) << lg)) * VEC + k];
      open = ends.flags[h] & kThrough;
    }
    if (!col) continue;
    if (which == 0 || open) {
      float* to = (which ? tails : heads) + d;
#pragma unroll
      for (int k = 0; k < VEC; ++k) to[k] = s[k];
    } else {
      write_row<TT, VEC>(grad, D, src.row(cur), d, f, s);
    }
  }
}

// ---- short id lists: one launch. Every workgroup owns a set of table rows (and a chunk of their columns): it reads all
// ids, keeps the positions of its own rows in order, sorts them by row, adds their runs and writes zeros to its other
// rows. The rows come in groups of 2^lgroup neighbours dealt out to the workgroups in turn, so that the low ids, which
// word frequencies favour, spread over the chip. What it costs is that each workgroup reads every id (from L2). Bound by
// latency: 1 id of 100 x 32 fp32 4.6 us, 4096 ids of 100 x 48 fp32 8.9 us (a sort, sums and a join: 18 us in three launches).
constexpr int kOwnThreads = 512, kOwnWaves = kOwnThreads / 64;
constexpr int64_t kOwnMax = 4096;  // ids
constexpr int64_t kOwnTable = 32ll << 20;  // bytes of the gradient

struct OwnPlan {
  int lg;           // log2 of the lanes a group
  int64_t chunks;   // column chunks
  int lgroup, lown; // log2 of the rows a row group, of the owners of row groups
  int64_t slots;    // rows an owner has (some beyond the table)
  int cap;          // list entries, a power of two
  int64_t lds;      // bytes of list and presence bits
};

inline OwnPlan own_plan(int64_t N, int64_t V, int64_t D, int vec, int64_t g_bytes, int64_t t_bytes) {
  OwnPlan o;
  const int64_t dv = (D + vec - 1) / vec;
  o.lgroup = 0;
  while (((int64_t)1 << o.lgroup) * D * t_bytes < 128 && ((int64_t)1 << o.lgroup) < V) ++o.lgroup;
  // up to 16 lanes, 256 bytes of a row; fewer, but 4, where a small table would leave CUs idle
  const int64_t groups = (V + (1ll << o.lgroup) - 1) >> o.lgroup;
  o.lg = 0;
  while (o.lg < 4 && (1ll << o.lg) < dv) ++o.lg;
  while (o.lg > 2 && ((dv + (1 << o.lg) - 1) >> o.lg) * groups < 64) --o.lg;
  while (o.lg < 6 && ((dv + (1 << o.lg) - 1) >> o.lg) > 256) ++o.lg;
  o.chunks = (dv + (1 << o.lg) - 1) >> o.lg;
  // owners: one for every 32 KB of zeros or 8 KB of gradient rows, up to 1024 workgroups, then up to the next power of two
  // (fewer than 2048 workgroups where the columns make no more than 1024 chunks)
  const int64_t most = 1024 / o.chunks > 1 ? 1024 / o.chunks : 1;
  int64_t want = V * D * t_bytes / 32768;
  want = want > N * D * g_bytes / 8192 ? want : N * D * g_bytes / 8192;
  want = want < most ? want : most;
  o.lown = 0;
  while (((int64_t)1 << o.lown) < want && ((int64_t)1 << (o.lown + o.lgroup)) < V) ++o.lown;
  const int64_t deal = (int64_t)1 << (o.lown + o.lgroup);
  o.slots = (V + deal - 1) / deal << o.lgroup;
  o.cap = 1;
  while (o.cap < N) o.cap *= 2;
  o.lds = (int64_t)o.cap * 4 + (o.slots + 31) / 32 * 4;
  return o;
}
// the list packs (slot, index) into 32 bits, and list and presence bits share the LDS with RunEnds; large tables are left
// to the sorted path, whose zeros stream faster (100 ids of 500000 x 100 bf16: 29 us against 32; 4000 of 50000 x 1000: 37
// against 60)
// The other end, us for one launch against the other paths: with rows named evenly it wins up to 4096 ids (4096 of
// 5000 x 64 bf16 11.2 / 17.7, 50000 x 32 fp32 9.2 / 16.4) and, with the registers and LDS for more, beyond (8192: 15.3 / 19.5,
// 13.8 / 18.9); with word frequencies, where one owner has most positions, it is level at 2048 (17.7 / 17.8, 16.8 / 17.1), behind
// at 4096 (21.9 / 20.1, 21.8 / 19.6; 500 x 4 fp32 41.1 / 23.2) and further behind beyond (8192: 32.6 / 25.1, 30.1 / 23.3). Tables
// of up to 32 rows would be faster with a table a lane from about 1000 ids on (4096 of 17 x 64 bf16 21.6 / 9.5).
inline bool own_fits(int64_t N, int64_t table_bytes, const OwnPlan& o) {
  return N <= kOwnMax && table_bytes <= kOwnTable && o.slots < (1ll << (32 - kIndexBits)) && o.lds <= 100 * 1024;
}

// own_fits whatever the types and alignments (slots are at most V + 64 then): no workspace
inline bool own_always(int64_t N, int64_t V, int64_t D) {
  return N <= kOwnMax && V <= (1 << 17) && V * D * 4 <= kOwnTable;
}

struct OwnList {
  const uint32_t* list;
  OwnPlan o;
  uint32_t owner;
  __device__ __forceinline__ uint32_t none() const { return 0xffffffffu; }
  __device__ __forceinline__ uint32_t key(int64_t i) const { return list[i] >> kIndexBits; }
  __device__ __forceinline__ Pair pair(int64_t i) const {
    const uint32_t e = list[i];
    return {e >> kIndexBits, e & ((1u << kIndexBits) - 1)};
  }
  __device__ __forceinline__ int64_t row(uint32_t slot) const {
    return (((((int64_t)slot >> o.lgroup) << o.lown) + owner) << o.lgroup) + (slot & ((1u << o.lgroup) - 1));
  }
};

template <typename GT, typename TT, int VEC>
__global__ __launch_bounds__(kOwnThreads) void own_rows_kernel(const GT* g, const void* ids, int id_bytes, int N, int64_t V,
                                                               int64_t D, int64_t pad, OwnPlan o, Mask m, double f,
                                                               TT* grad) {
  extern __shared__ uint32_t shared[];
  __shared__ RunEnds<kOwnThreads, VEC> ends;
  __shared__ int wave_count[kOwnWaves], unsorted;
  uint32_t* list = shared;
  uint32_t* present = shared + o.cap;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t owner = blockIdx.x & ((1u << o.lown) - 1);
  const int64_t chunk = blockIdx.x >> o.lown;
  const OwnList src{list, o, owner};
  const uint32_t in_group = (1u << o.lgroup) - 1;
  for (int k = tid; k < (o.slots + 31) / 32; k += kOwnThreads) present[k] = 0;
  if (tid == 0) unsorted = 0;

  // 1. the positions of this owner's rows, in order: count, then place. A wave holds its consecutive ids in registers.
  constexpr int B = (int)(kOwnMax / kOwnThreads);
  const int span = ((N + kOwnWaves - 1) / kOwnWaves + 63) / 64 * 64;
  const int first = wave * span, end = first + span < N ? first + span : N;
  int64_t id[B];
#pragma unroll
  for (int u = 0; u < B; ++u) {
    const int i = first + u * 64 + lane;
    id[u] = i < end ? (id_bytes == 8 ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i]) : -1;
  }
  int64_t slot[B];  // -1: not this owner's
  int count = 0;
#pragma unroll
  for (int u = 0; u < B; ++u) {
    const int64_t grp = id[u] >> o.lgroup;
    const bool mine =
        id[u] >= 0 && id[u] < V && id[u] != pad && ((uint32_t)grp & ((1u << o.lown) - 1)) == owner;
    slot[u] = mine ? ((grp >> o.lown) << o.lgroup) + (id[u] & in_group) : -1;
    count += __popcll(__ballot(mine));
  }
  if (lane == 0) wave_count[wave] = count;
  __syncthreads();
  int at = 0, M = 0;
#pragma unroll
  for (int w = 0; w < kOwnWaves; ++w) {
    at += w < wave ? wave_count[w] : 0;
    M += wave_count[w];
  }
#pragma unroll
  for (int u = 0; u < B; ++u) {
    const uint64_t mine = __ballot(slot[u] >= 0);
    if (slot[u] >= 0) {
      list[at + __popcll(mine & ((1ull << lane) - 1))] =
          ((uint32_t)slot[u] << kIndexBits) | (uint32_t)(first + u * 64 + lane);
      atomicOr(&present[slot[u] >> 5], 1u << (slot[u] & 31));
    }
    at += __popcll(mine);
  }
  __syncthreads();

  // 2. zeros for the rows that no position names
  const int64_t d0 = (chunk << o.lg) * VEC;
  for (int64_t t = tid; t < (o.slots << o.lg); t += kOwnThreads) {
    const int64_t slot = t >> o.lg, d = d0 + (t & ((1 << o.lg) - 1)) * VEC;
    const int64_t row = src.row((uint32_t)slot);
    if (row < V && d < D && !(present[slot >> 5] >> (slot & 31) & 1)) {
      const float zero[VEC] = {};
      store_vec<TT, VEC, (VEC > 1), false>(grad + row * D + d, zero);
    }
  }

  // 3. sort by (slot, index): the entries differ, so any sort is stable. Often there is nothing to do.
  for (int i = tid; i + 1 < M; i += kOwnThreads)
    if (list[i] > list[i + 1]) unsorted = 1;
  __syncthreads();
  if (unsorted) {
    int n = 1;
    while (n < M) n *= 2;
    for (int i = M + tid; i < n; i += kOwnThreads) list[i] = 0xffffffffu;
    __syncthreads();
    for (int k = 2; k <= n; k *= 2) {
      for (int j = k / 2; j > 0; j /= 2) {
        for (int t = tid; t < n / 2; t += kOwnThreads) {
          const int i = ((t & ~(j - 1)) << 1) | (t & (j - 1));
          const uint32_t x = list[i], y = list[i + j];
          if ((x > y) == ((i & k) == 0)) {
            list[i] = y;
            list[i + j] = x;
          }
        }
        __syncthreads();
      }
    }
  }

  // 4. the runs
  const int groups = kOwnThreads >> o.lg;
  const int64_t d = d0 + (tid & ((1 << o.lg) - 1)) * VEC;
  const int piece = (M + groups - 1) / groups;
  sum_runs<kOwnThreads, GT, TT, VEC>(ends, src, M, 0, piece, o.lg, g, D, d, m, mask_offset(m), f, grad, nullptr, nullptr);
}

// ---- many ids of a small table: no sort. Every lane keeps a table of its own in LDS (all rows, its vector of columns) and
// adds the rows of g it is given, which are consecutive for a workgroup and so read once, in order and whole; lanes that
// hold the same columns are then added in order, and the workgroups' tables in a second launch. Neither the ids nor their
// distribution change what it costs. Tables of up to 32 rows, whose LDS lets a lane have 4 columns (a row more would halve
// them: 100 rows with 1 column a lane, 10^6 ids of 16 columns, took 104 us, sorting 73). Bound by the LDS additions, each of
// which waits for the one before: 131072 ids of 17 x 64 bf16 16.4 us and 3.9 us for the join (sorting: 34 us).
constexpr int kDenseThreads = 256;
constexpr int64_t kDenseRows = 32;

struct DensePlan {
  int vec;             // elements a lane, 0: the path does not fit
  int lg;              // log2 of the lanes a row of g
  int64_t chunks;      // column chunks
  int64_t rows, blocks;  // rows of g a workgroup, workgroups a chunk
  int64_t lds;
};

// vec: the most that the pointers and D allow; this path takes up to 4
inline DensePlan dense_plan(int64_t N, int64_t V, int64_t D, int vec) {
  DensePlan p{0, 0, 0, 0, 0, 0};
  vec = vec < 4 ? vec : 4;
  if (N <= kOwnMax || V > kDenseRows) return p;
  p.vec = vec;
  p.lds = V * kDenseThreads * vec * 4;
  const int64_t dv = (D + vec - 1) / vec;
  while (p.lg < 6 && (1ll << p.lg) < dv) ++p.lg;
  p.chunks = (dv + (1 << p.lg) - 1) >> p.lg;
  // as many workgroups as the chip holds at once, but 4 rows a lane
  int64_t per_cu = 160 * 1024 / p.lds;
  per_cu = per_cu > 8 ? 8 : per_cu;
  int64_t want = 256 * per_cu / p.chunks;
  want = want < 1 ? 1 : want;
  const int64_t least = (kDenseThreads >> p.lg) * 4;
  p.rows = (N + want - 1) / want;
  p.rows = p.rows > least ? p.rows : least;
  p.blocks = (N + p.rows - 1) / p.rows;
  return p;
}

template <typename GT, int VEC>
__global__ __launch_bounds__(kDenseThreads) void dense_sum_kernel(const GT* g, const void* ids, int id_bytes, int64_t N,
                                                                  int64_t V, int64_t D, int64_t pad, DensePlan p, Mask m,
                                                                  float* partial) {
  extern __shared__ float dense_table[];  // [row][lane][VEC]
  const int tid = threadIdx.x, groups = kDenseThreads >> p.lg, group = tid >> p.lg, sub = tid & ((1 << p.lg) - 1);
  const int64_t block = blockIdx.x % (uint32_t)p.blocks, chunk = blockIdx.x / (uint32_t)p.blocks;
  const int64_t d = ((chunk << p.lg) + sub) * VEC;
  for (int v = 0; v < (int)V; ++v)
#pragma unroll
    for (int k = 0; k < VEC; ++k) dense_table[(v * kDenseThreads + tid) * VEC + k] = 0.0f;
  const uint64_t off = mask_offset(m);
  const int64_t begin = block * p.rows, end = begin + p.rows < N ? begin + p.rows : N;
  constexpr int U = 8;
  for (int64_t n0 = begin + group; n0 < end; n0 += groups * U) {
    int64_t id[U];
    float v[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * groups;
      id[u] = -1;
      if (n < end && d < D) {
        id[u] = id_bytes == 8 ? ((const int64_t*)ids)[n] : (int64_t)((const int32_t*)ids)[n];
        load_vec<GT, VEC, (VEC > 1), false>(g + n * D + d, v[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (id[u] < 0 || id[u] >= V || id[u] == pad) continue;
      if (m.mode != 0) apply_keep<VEC>(m, off, (n0 + u * groups) * D + d, v[u]);
      float* a = dense_table + ((int)id[u] * kDenseThreads + tid) * VEC;
#pragma unroll
      for (int k = 0; k < VEC; ++k) a[k] += v[u][k];
    }
  }
  __syncthreads();
  for (int t = tid; t < (int)V << p.lg; t += kDenseThreads) {
    const int v = t >> p.lg, c = t & ((1 << p.lg) - 1);
    const int64_t e = ((chunk << p.lg) + c) * VEC;
    if (e >= D) continue;
    float s[VEC] = {};
    for (int q = 0; q < groups; ++q) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[k] += dense_table[(v * kDenseThreads + (q << p.lg) + c) * VEC + k];
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) partial[block * V * D + v * D + e + k] = s[k];
  }
}

// grad[k] = f * (the workgroups' tables in order), 2^lo elements a workgroup, whose other lanes take consecutive workgroups
constexpr int kDenseJoinThreads = 1024;
template <typename TT>
__global__ __launch_bounds__(kDenseJoinThreads) void dense_join_kernel(const float* partial, int64_t blocks, int64_t n, int lo,
                                                                       double f, TT* grad) {
  __shared__ float sums[kDenseJoinThreads];
  const int out = threadIdx.x & ((1 << lo) - 1), part = threadIdx.x >> lo, parts = kDenseJoinThreads >> lo;
  const int64_t k = ((int64_t)blockIdx.x << lo) + out;
  const int64_t per = (blocks + parts - 1) / parts, begin = part * per, end = begin + per < blocks ? begin + per : blocks;
  float s = 0.0f;
  if (k < n) {
#pragma unroll 8
    for (int64_t b = begin; b < end; ++b) s += partial[b * n + k];
  }
  sums[threadIdx.x] = s;
  __syncthreads();
  if (part != 0 || k >= n) return;
  for (int q = 1; q < parts; ++q) s += sums[(q << lo) + out];
  grad[k] = (TT)scaled(s, f);
}

// ---- long id lists: the sorted pairs in memory, a workgroup's runs cut by its neighbours' joined in a second launch.
// Bound by bytes where rows are long: 16384 ids of 50000 x 1024 bf16, 33 MB of g and 102 MB of gradient, 27.8 us, 4.9 TB/s;
// by the gather's cache lines where they are short (2 M rows of 16 bytes: 67 us). The join, 5 to 7 us, is latency.
struct RunPlan {
  int lg;          // log2 of the lanes a group
  int64_t chunks;  // column chunks of (1 << lg) vectors
  int piece;       // positions a group
  int64_t span, blocks;  // positions a workgroup, workgroups
};
constexpr int kRunThreads = 256, kRunSpan = 2048;

inline RunPlan run_plan(int64_t N, int64_t D, int vec) {
  RunPlan r;
  const int64_t dv = (D + vec - 1) / vec;
  r.lg = 0;
  while (r.lg < 6 && (1ll << r.lg) < dv) ++r.lg;
  r.chunks = (dv + (1 << r.lg) - 1) >> r.lg;
  const int64_t groups = kRunThreads >> r.lg;
  // enough workgroups for the chip, else longer pieces: fewer runs are cut
  const int64_t want = 2048 / r.chunks > 0 ? 2048 / r.chunks : 1;
  int64_t t = (N + groups * want - 1) / (groups * want);
  const int64_t most = kRunSpan / groups < 64 ? kRunSpan / groups : 64;
  t = t < 8 ? 8 : t > most ? most : t;
  r.piece = (int)(t / 8 * 8);
  r.span = groups * r.piece;
  r.blocks = (N + r.span - 1) / r.span;
  return r;
}

// a workgroup's span of the sorted pairs and their neighbours at both ends, in LDS; a gap after every 8 keeps the groups'
// pieces, which start at multiples of 8, on different banks
struct StagedPairs {
  const uint64_t* lds;
  int64_t base;
  uint32_t V;
  static __device__ __forceinline__ int slot(int i) { return i + (i >> 3); }
  __device__ __forceinline__ uint32_t none() const { return V; }
  __device__ __forceinline__ Pair pair(int64_t i) const {
    return __builtin_bit_cast(Pair, lds[slot((int)(i - base) + 8)]);
  }
  __device__ __forceinline__ uint32_t key(int64_t i) const { return pair(i).key; }
  __device__ __forceinline__ int64_t row(uint32_t key) const { return key; }
};

// first position of [lo, hi) whose key is not below v
__device__ __forceinline__ int64_t lower_bound(const Pair* pairs, int64_t lo, int64_t hi, uint32_t v) {
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (pairs[mid].key < v) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(256) void zeros_kernel(uint16_t* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

// Workgroups beyond the first r.blocks * r.chunks write zeros to the rows that no pair names, `rows` consecutive ones each
// (clearing the whole gradient beforehand writes the named rows twice, and could not share the chip with the sums).
constexpr int kAbsentRows = 1024;

template <typename GT, typename TT, int VEC>
__global__ __launch_bounds__(kRunThreads) void run_sum_kernel(const GT* g, const Pair* pairs, uint32_t V, int64_t N,
                                                              int64_t D, RunPlan r, Mask m, double f, TT* grad,
                                                              float* heads, float* tails, int rows, Div dv) {
  __shared__ RunEnds<kRunThreads, VEC> ends;
  __shared__ uint64_t staged[(kRunSpan + 16) / 8 * 9];
  const uint32_t sums = (uint32_t)(r.blocks * r.chunks);
  if (blockIdx.x >= sums) {
    uint8_t* named = (uint8_t*)staged;
    const int64_t row0 = (int64_t)(blockIdx.x - sums) * rows;
    const int here = (int)(V - row0 < rows ? V - row0 : rows);
    for (int k = threadIdx.x; k < here; k += kRunThreads) {
      const uint32_t row = (uint32_t)(row0 + k);
      const int64_t at = lower_bound(pairs, 0, N, row);
      named[k] = at < N && pairs[at].key == row;
    }
    __syncthreads();
    const float zero[VEC] = {};
    for (uint32_t t = threadIdx.x; t < (uint32_t)here * dv.d; t += kRunThreads)
      if (!named[div_by(t, dv)]) store_vec<TT, VEC, (VEC > 1), false>(grad + row0 * D + (int64_t)t * VEC, zero);
    return;
  }
  const int64_t block = blockIdx.x % (uint32_t)r.blocks, chunk = blockIdx.x / (uint32_t)r.blocks;
  const int64_t d = ((chunk << r.lg) + (threadIdx.x & ((1 << r.lg) - 1))) * VEC;
  const int64_t base = block * r.span;
  const uint64_t* in = (const uint64_t*)pairs;
  for (int k = threadIdx.x; k < r.span; k += kRunThreads)
    if (base + k < N) staged[StagedPairs::slot(k + 8)] = in[base + k];
  if (threadIdx.x == 0 && base > 0) staged[StagedPairs::slot(7)] = in[base - 1];
  if (threadIdx.x == 1 && base + r.span < N) staged[StagedPairs::slot((int)r.span + 8)] = in[base + r.span];
  __syncthreads();
  sum_runs<kRunThreads, GT, TT, VEC>(ends, StagedPairs{staged, base, V}, N, base, r.piece, r.lg, g, D, d, m,
                                     mask_offset(m), f, grad, heads + block * D, tails + block * D);
}

// the run that workgroup b of run_sum_kernel started and did not end: its tail and the heads of the workgroups after it
template <typename TT, int VEC>
__global__ __launch_bounds__(kRunThreads) void run_join_kernel(const Pair* pairs, int64_t N, uint32_t V, int64_t D,
                                                               RunPlan r, double f, TT* grad, const float* heads,
                                                               const float* tails) {
  const int64_t b = blockIdx.x % (uint32_t)r.blocks, next = (b + 1) * r.span;
  if (next >= N) return;
  const uint32_t key = pairs[next - 1].key;
  if (key == V || pairs[next].key != key) return;
  if (b > 0 && pairs[b * r.span].key == key && pairs[b * r.span - 1].key == key) return;  // it began earlier
  int64_t end = (b + 2) * r.span < N ? (b + 2) * r.span : N;
  if (pairs[end - 1].key == key) end = lower_bound(pairs, end, N, key + 1);
  else end = next + 1;  // ends inside the next workgroup
  const int64_t last = (end - 1) / r.span;
  __shared__ float part[kRunThreads * VEC];
  const int groups = kRunThreads >> r.lg, group = threadIdx.x >> r.lg, sub = threadIdx.x & ((1 << r.lg) - 1);
  const int64_t d = (((int64_t)(blockIdx.x / (uint32_t)r.blocks) << r.lg) + sub) * VEC;
  const bool col = d < D;
  float s[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) s[k] = 0.0f;
  if (col) {
#pragma unroll 4
    for (int64_t h = b + 1 + group; h <= last; h += groups) {
#pragma unroll
      for (int k = 0; k < VEC; ++k) s[k] += heads[h * D + d + k];
    }
  }
#pragma unroll
  for (int k = 0; k < VEC; ++k) part[threadIdx.x * VEC + k] = s[k];
  __syncthreads();
  if (group != 0 || !col) return;
#pragma unroll
  for (int k = 0; k < VEC; ++k) s[k] = tails[b * D + d + k];
  const int64_t used = last - b < groups ? last - b : groups;
  for (int q = 0; q < used; ++q) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) s[k] += part[(threadIdx.x + (q << r.lg)) * VEC + k];
  }
  write_row<TT, VEC>(grad, D, key, d, f, s);
}

// ---- long id lists of short rows (up to 16 bytes of g): gathering such rows one by one would fetch a cache line for each.
// One partition by ranges of table rows carries the rows of g along, dropout applied; then a workgroup streams a tile of a
// bucket, each wave into its own LDS table of the bucket's rows. Lanes of a wave that hold the same row add one after the
// other in the order of the lanes, so that the ids fix the sums' order. A bucket of more than one tile leaves its
// tiles' tables to a second launch. Every row of a bucket is written, so the gradient needs no zeros beforehand. 6.3 M ids of
// 512000 x 2 fp32: count 10, scan 11, partition 42, sums 46, join 7 us (sorting pairs and gathering: 270 us); the partition
// is bound like the sort's scatter, the sums by the turns of the lanes that share a row.
constexpr int kBucketThreads = 512, kBucketWaves = kBucketThreads / 64;
constexpr int64_t kBucketTile = 8192;    // positions a workgroup
constexpr int64_t kBucketFloats = 2048;  // a wave's table

struct BucketPlan {
  int lrows;        // log2 of a bucket's rows
  int64_t buckets;  // 0: the path does not fit
  int64_t max_tiles;
  int dm;           // elements a row of the tables and of the carried rows, a power of two
};

inline BucketPlan bucket_plan(int64_t N, int64_t V, int64_t D, int64_t g_bytes) {
  BucketPlan b{0, 0, 0, 1};
  if (D * g_bytes > 16) return b;
  while (b.dm < D) b.dm *= 2;
  // up to 1023 buckets (and one for the ids that take no part), as many as would hold half a tile each; more, of fewer ids,
  // where a bucket has all the rows that its table holds (16385 ids of 2000000 x 1: 977 buckets of 17 ids)
  int64_t most = N / (kBucketTile / 2);
  most = most < 1 ? 1 : most > 1023 ? 1023 : most;
  while (((V + (1ll << b.lrows) - 1) >> b.lrows) > most && ((2ll << b.lrows) * b.dm <= kBucketFloats)) ++b.lrows;
  const int64_t n = (V + (1ll << b.lrows) - 1) >> b.lrows;
  if (n > 1023) return b;
  b.buckets = n;
  b.max_tiles = n + N / kBucketTile;
  return b;
}

// the carried rows: DM elements of E bytes each, raw
template <typename E, int DM>
struct alignas(sizeof(E) * DM) Row {
  E e[DM];
};
template <typename E, int DM>
struct StoreRows {
  const E* g;
  int D;
  Mask m;
  uint32_t* keys;
  Row<E, DM>* rows;
  __device__ __forceinline__ void operator()(int64_t to, Pair p) const {
    Row<E, DM> r;
    const int64_t e = (int64_t)p.pos * D;
#pragma unroll
    for (int k = 0; k < DM; ++k) r.e[k] = k < D ? g[e + k] : (E)0;
    if (m.mode != 0) {
      const uint64_t off = mask_offset(m);
      Keep4 keep = keep_group(m, off, (uint64_t)e >> 2);
#pragma unroll
      for (int k = 0; k < DM; ++k) {
        if (k > 0 && ((e + k) & 3) == 0) keep = keep_group(m, off, (uint64_t)(e + k) >> 2);
        const bool lo = (e + k) & 1 ? keep.k[1] : keep.k[0], hi = (e + k) & 1 ? keep.k[3] : keep.k[2];
        if (!((e + k) & 2 ? hi : lo)) r.e[k] = (E)0;
      }
    }
    keys[to] = p.key;
    rows[to] = r;
  }
};

// first position, positions, and the tiles before it, of the bucket that holds tile `tile`
struct BucketTile {
  uint32_t bucket, first, count, tile, tiles, tiles_before;
};

template <typename GT, typename TT, int DM>
__global__ __launch_bounds__(kBucketThreads) void bucket_sum_kernel(const uint32_t* keys, const Row<GT, DM>* rows,
                                                                    const uint32_t* totals, BucketPlan b, int64_t V, int D,
                                                                    double f, TT* grad, float* partial,
                                                                    BucketTile* multi) {
  extern __shared__ float table[];  // [wave][row of the bucket][DM]
  __shared__ uint32_t part[kBucketWaves];
  __shared__ BucketTile me;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int floats = DM << b.lrows;
  for (int k = tid; k < kBucketWaves * floats; k += kBucketThreads) table[k] = 0.0f;
  if (tid == 0) me.bucket = 0xffffffffu;
  // which bucket, which of its tiles: 2 buckets a lane
  uint32_t cnt[2], nt[2], all;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    cnt[k] = tid * 2 + k < b.buckets ? totals[tid * 2 + k] : 0u;
    nt[k] = tid * 2 + k < b.buckets ? (cnt[k] > 0 ? (cnt[k] + (uint32_t)kBucketTile - 1) / (uint32_t)kBucketTile : 1u) : 0u;
  }
  uint32_t first = block_exclusive_scan<kBucketWaves>(cnt[0] + cnt[1], part, all);
  uint32_t tile0 = block_exclusive_scan<kBucketWaves>(nt[0] + nt[1], part, all);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (blockIdx.x >= tile0 && blockIdx.x < tile0 + nt[k])
      me = {(uint32_t)(tid * 2 + k), first, cnt[k], blockIdx.x - tile0, nt[k], tile0};
    first += cnt[k];
    tile0 += nt[k];
  }
  __syncthreads();
  const BucketTile t = me;
  if (t.bucket == 0xffffffffu) return;  // fewer tiles than the most there can be
  if (t.tile == 0 && tid == 0) multi[t.bucket] = t;
  // a wave's step takes 8 consecutive positions from each of 8 places of its part: neighbours often name the same row, and
  // lanes with the same row wait for one another, while 8 positions still make a whole sector to load
  constexpr int kPart = (int)(kBucketTile / kBucketWaves), kPlace = kPart / 8, U = 4;
  const uint32_t begin = t.tile * (uint32_t)kBucketTile + wave * kPart;
  for (int s0 = 0; s0 < kPlace / 8 && begin < t.count; s0 += U) {
    uint32_t slot[U];
    bool valid[U];
    Row<GT, DM> r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t i = begin + (lane >> 3) * kPlace + (s0 + u) * 8 + (lane & 7);
      valid[u] = i < t.count;
      slot[u] = 0;
      if (valid[u]) {
        slot[u] = keys[t.first + i] & ((1u << b.lrows) - 1);
        r[u] = rows[t.first + i];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint64_t peers = wave_match(slot[u], b.lrows, valid[u]);
      const int turn = valid[u] ? __popcll(peers & ((1ull << lane) - 1)) : -1;
      for (int now = 0; __ballot(turn >= now); ++now) {
        if (turn == now) {
          float* a = table + wave * floats + slot[u] * DM;
#pragma unroll
          for (int k = 0; k < DM; ++k) a[k] += (float)r[u].e[k];
        }
        wave_fence();
      }
    }
  }
  __syncthreads();
  const int64_t row0 = (int64_t)t.bucket << b.lrows;
  for (int k = tid; k < floats; k += kBucketThreads) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kBucketWaves; ++w) s += table[w * floats + k];
    if (t.tiles > 1) {
      partial[(int64_t)blockIdx.x * floats + k] = s;
    } else {
      const int64_t row = row0 + k / DM;
      const int d = k % DM;
      if (row < V && d < D) grad[row * D + d] = (TT)scaled(s, f);
    }
  }
}

// buckets of more than one tile: their tiles' tables, added in order; `split` workgroups a bucket
template <typename TT, int DM>
__global__ __launch_bounds__(256) void bucket_join_kernel(const float* partial, const BucketTile* multi, BucketPlan b,
                                                          int split, int64_t V, int D, double f, TT* grad) {
  __shared__ float sums[256];
  const uint32_t bucket = blockIdx.x / split;
  const BucketTile t = multi[bucket];
  if (t.tiles < 2) return;
  const int floats = DM << b.lrows;
  const int out = threadIdx.x & 63, part = threadIdx.x >> 6;  // 4 parts of the tiles
  const uint32_t per = (t.tiles + 3) / 4;
  const uint32_t begin = t.tiles_before + part * per, stop = t.tiles_before + t.tiles;
  const uint32_t end = begin + per < stop ? begin + per : stop;
  for (int k0 = (blockIdx.x % split) * 64; k0 < floats; k0 += split * 64) {
    const int k = k0 + out;
    float s = 0.0f;
    if (k < floats) {
#pragma unroll 8
      for (uint32_t q = begin; q < end; ++q) s += partial[(int64_t)q * floats + k];
    }
    __syncthreads();
    sums[threadIdx.x] = s;
    __syncthreads();
    const int64_t row = ((int64_t)t.bucket << b.lrows) + k / DM;
    const int d = k % DM;
    if (part == 0 && k < floats && row < V && d < D)
      grad[row * D + d] = (TT)scaled(((sums[out] + sums[64 + out]) + sums[128 + out]) + sums[192 + out], f);
  }
}

// ------------------------------------------------------------------------------------------ workspace
struct GradWs {
  int64_t counts, totals, pairs[2], heads, tails, bytes;
};

inline GradWs grad_ws(int64_t N, int64_t V, int64_t D) {
  const SortPlan s = sort_plan(N, V);
  GradWs w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  w.counts = take(s.bins * s.tiles * 4);
  w.totals = take(s.bins * 4);
  for (int i = 0; i < 2; ++i) w.pairs[i] = take(N * (int64_t)sizeof(Pair));
  int64_t blocks = 0;  // of whichever vector the pointers' alignment allows
  for (int vec : {1, 2, 4, 8}) {
    const int64_t b = run_plan(N, D, vec).blocks;
    blocks = b > blocks ? b : blocks;
  }
  w.heads = take(blocks * D * 4);
  w.tails = take(blocks * D * 4);
  w.bytes = at;
  return w;
}

struct BucketWs {
  int64_t counts, totals, keys, rows, partial, multi, bytes;
};

inline int64_t partition_tiles(int64_t N) { return (N + kTileThreads * kTileItems - 1) / (kTileThreads * kTileItems); }

inline BucketWs bucket_ws(int64_t N, const BucketPlan& b, int64_t g_bytes) {
  BucketWs w;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  w.counts = take(1024 * partition_tiles(N) * 4);
  w.totals = take(1024 * 4);
  w.keys = take(N * 4);
  w.rows = take(N * b.dm * g_bytes);
  w.partial = take(b.max_tiles * ((int64_t)b.dm << b.lrows) * 4);
  w.multi = take(1024 * (int64_t)sizeof(BucketTile));
  w.bytes = at;
  return w;
}

template <typename Src>
inline void sort_pass(Src src, int64_t N, int pass, const SortPlan& s, char* ws, const GradWs& w, hipStream_t st) {
  uint32_t* counts = (uint32_t*)(ws + w.counts);
  uint32_t* totals = s.tiles <= kFewTiles ? nullptr : (uint32_t*)(ws + w.totals);
  const int shift = pass * s.width;
  auto go = [&](auto bins, auto threads, auto items) {
    constexpr int BINS = decltype(bins)::value, THREADS = decltype(threads)::value, ITEMS = decltype(items)::value;
    hipLaunchKernelGGL((sort_count_kernel<Src, BINS, THREADS, ITEMS>), dim3((unsigned)s.tiles), dim3(THREADS), 0, st, src,
                       N, shift, s.width, counts);
    if (totals)
      hipLaunchKernelGGL(sort_scan_kernel, dim3(BINS / kScanDigits), dim3(kScanThreads), 0, st, counts, s.tiles, BINS,
                         totals);
    hipLaunchKernelGGL((sort_scatter_kernel<Src, StorePairs, BINS, THREADS, ITEMS>), dim3((unsigned)s.tiles),
                       dim3(THREADS), 0, st, src, N, shift, s.width, counts, s.tiles, totals,
                       StorePairs{(Pair*)(ws + w.pairs[pass & 1])});
  };
  using std::integral_constant;
  auto sized = [&](auto bins) {
    if (s.few) go(bins, integral_constant<int, kFewThreads>{}, integral_constant<int, kFewItems>{});
    else go(bins, integral_constant<int, kTileThreads>{}, integral_constant<int, kTileItems>{});
  };
  if (s.bins == 256) sized(integral_constant<int, 256>{});
  else sized(integral_constant<int, 1024>{});
}

// sorts the ids; returns which of the two buffers holds the pairs
template <typename IT>
inline int sort_ids(const IT* ids, int64_t N, int64_t V, int64_t pad, char* ws, const GradWs& w, hipStream_t st) {
  const SortPlan s = sort_plan(N, V);
  const KeyFromIds<IT> src{ids, V, pad, (uint32_t)V};
  if (N <= kRankMax) {
    const bool narrow = V < (1ll << (32 - kIndexBits));  // keys 0 .. V beside the index in 32 bits
    auto* k = narrow ? rank_sort_kernel<IT, uint32_t> : rank_sort_kernel<IT, uint64_t>;
    hipLaunchKernelGGL(k, dim3((unsigned)((N + kRankTile - 1) / kRankTile)), dim3(kRankThreads),
                       (unsigned)(N * (narrow ? 4 : 8)), st, src, (int)N, rank_bins(V),
                       (Pair*)(ws + w.pairs[0]));
    return 0;
  }
  for (int pass = 0; pass < s.passes; ++pass) {
    const int from = (pass - 1) & 1;
    if (pass == 0) sort_pass(src, N, pass, s, ws, w, st);
    else sort_pass(KeyFromPairs{(const Pair*)(ws + w.pairs[from])}, N, pass, s, ws, w, st);
  }
  return (s.passes - 1) & 1;
}

template <typename GT, typename TT, int DM, typename IT>
inline void bucket_gradient(const GT* g, const IT* ids, int64_t N, int64_t V, int64_t D, int64_t pad, const BucketPlan& b,
                            const Mask& m, double f, TT* grad, char* ws, hipStream_t st) {
  typedef typename std::conditional<sizeof(GT) == 4, uint32_t, uint16_t>::type E;
  const BucketWs w = bucket_ws(N, b, sizeof(GT));
  uint32_t *counts = (uint32_t*)(ws + w.counts), *totals = (uint32_t*)(ws + w.totals), *keys = (uint32_t*)(ws + w.keys);
  const int64_t tiles = partition_tiles(N);
  const KeyFromIds<IT> src{ids, V, pad, (uint32_t)(b.buckets << b.lrows)};
  hipLaunchKernelGGL((sort_count_kernel<KeyFromIds<IT>, 1024, kTileThreads, kTileItems>), dim3((unsigned)tiles),
                     dim3(kTileThreads), 0, st, src, N, b.lrows, 10, counts);
  hipLaunchKernelGGL(sort_scan_kernel, dim3(1024 / kScanDigits), dim3(kScanThreads), 0, st, counts, tiles, 1024, totals);
  const StoreRows<E, DM> dst{(const E*)g, (int)D, m, keys, (Row<E, DM>*)(ws + w.rows)};
  hipLaunchKernelGGL((sort_scatter_kernel<KeyFromIds<IT>, StoreRows<E, DM>, 1024, kTileThreads, kTileItems>),
                     dim3((unsigned)tiles), dim3(kTileThreads), 0, st, src, N, b.lrows, 10, counts, tiles, totals, dst);
  const unsigned lds = (unsigned)(kBucketWaves * ((int64_t)DM << b.lrows) * 4);
  float* partial = (float*)(ws + w.partial);
  BucketTile* multi = (BucketTile*)(ws + w.multi);
  hipLaunchKernelGGL((bucket_sum_kernel<GT, TT, DM>), dim3((unsigned)b.max_tiles), dim3(kBucketThreads), lds, st, keys,
                     (const Row<GT, DM>*)(ws + w.rows), totals, b, V, (int)D, f, grad, partial, multi);
  int64_t split = 2048 / b.buckets, most = (((int64_t)DM << b.lrows) + 63) / 64;
  split = split < 1 ? 1 : split > most ? most : split;
  hipLaunchKernelGGL((bucket_join_kernel<TT, DM>), dim3((unsigned)(b.buckets * split)), dim3(256), 0, st, partial, multi, b,
                     (int)split, V, (int)D, f, grad);
}

// sizes that the kernels' 32-bit positions and keys, and the grids, hold
inline int embedding_sizes_ok(const char* what, int64_t N, int64_t V, int64_t D) {
  YN_CHECK(N >= 0 && V >= 0 && D >= 0, "%s: negative size", what);
  YN_CHECK(N < (1ll << 31) && V < (1ll << 31), "%s: N=%lld or V=%lld is 2^31 or more", what, (long long)N, (long long)V);
  YN_CHECK(D <= (1ll << 24), "%s: D=%lld is more than 2^24", what, (long long)D);
  YN_CHECK(D == 0 || (N <= (1ll << 36) / D && V <= (1ll << 36) / D), "%s: more than 2^36 elements", what);
  return 0;
}
// rows a workgroup takes, so that it has about `work` units of `per_row` each (fewer where N of them leave CUs idle)
inline int tile_rows(int64_t N, int64_t per_row, int64_t work, int64_t multiple) {
  const int64_t spread = (N * per_row + 1023) / 1024;  // 4 workgroups a CU
  const int64_t w = spread < work ? (spread > 256 ? spread : 256) : work;
  const int64_t r = (w / per_row + multiple - 1) / multiple * multiple;
  return (int)(r < multiple ? multiple : r);
}
// outputs that leave no cache lines worth keeping (the Infinity Cache holds 256 MB) are stored non-temporally
inline bool streams_past_cache(int64_t bytes) { return bytes >= (64ll << 20); }
// The factor, 0 or a normal number of fp32, in which the lookup multiplies: beyond them 0 would become NaN, and below them the
// factor's own digits go
inline int factor_ok(const char* what, double f) {
  YN_CHECK(f == 0.0 || (std::fabs(f) >= FLT_MIN && std::fabs(f) <= FLT_MAX),
           "%s: the factor scale / (1 - p) = %g is outside the range of fp32", what, f);
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
  YN_CHECK(n >= 0 && n <= (1ll << 36), "dropout: n=%lld out of range", (long long)n);
  if (mask_args_ok("dropout", p)) return 1;
  YN_CHECK(!rng_used || rng_used != rng_base, "dropout: rng_used is rng_base");
  if (n == 0) return 0;
  YN_CHECK(x && y, "dropout: null pointer");
  const Mask m = make_mask(p, seed, offset, rng_base);
  const float f = (float)mask_scale(1.0, p, m);
  const bool al = aligned(x, 16) && aligned(y, 16), nt = streams_past_cache(n * type_bytes(type));
  with_type(type, [&](auto t) {
    using T = decltype(t);
    constexpr int VEC = 16 / sizeof(T);
    auto* k = !al ? dropout_kernel<T, false, false> : nt ? dropout_kernel<T, true, true> : dropout_kernel<T, true, false>;
    for (int64_t first = 0; first < n; first += 1ll << 32) {  // a launch holds fewer than 2^32 lanes
      const int64_t part = n - first < 1ll << 32 ? n - first : 1ll << 32;
      hipLaunchKernelGGL(k, dim3((unsigned)((part + 256 * VEC - 1) / (256 * VEC))), dim3(256), 0, as_stream(stream),
                         (const T*)x, (T*)y, first + part, first, m, f, rng_used);
    }
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
  YN_CHECK(!rng_used || rng_used != rng_base, "embedding: rng_used is rng_base");
  if (N == 0 || D == 0) return 0;
  YN_CHECK(V >= 1, "embedding: an empty table");
  YN_CHECK(table && ids && out, "embedding: null pointer");
  YN_CHECK(table_stride >= 0, "embedding: negative table stride");
  const Mask m = make_mask(p, seed, offset, rng_base);
  if (factor_ok("embedding", mask_scale(scale, p, m))) return 1;
  const float f = (float)mask_scale(scale, p, m);
  const int64_t wide = 16 / (type_bytes(table_type) > type_bytes(out_type) ? type_bytes(table_type) : type_bytes(out_type));
  auto fits = [&](int64_t vec) {
    return D % vec == 0 && table_stride % vec == 0 && aligned(table, vec * type_bytes(table_type)) &&
           aligned(out, vec * type_bytes(out_type));
  };
  const int64_t vec = fits(wide) ? wide : fits(4) ? 4 : fits(2) ? 2 : 0;
  const bool nt = streams_past_cache(N * D * type_bytes(out_type));
  with_type(table_type, [&](auto tt) {
    with_type(out_type, [&](auto ot) {
      using TT = decltype(tt);
      using OT = decltype(ot);
      with_index(id_bytes, [&](auto it) {
        using IT = decltype(it);
        if (vec) {
          constexpr int W = 16 / (sizeof(TT) > sizeof(OT) ? sizeof(TT) : sizeof(OT));
          const int rows = tile_rows(N, D / vec, 256 * kUnroll, 1);
          auto* k = vec == 2   ? (nt ? embedding_rows_of_vectors_kernel<TT, OT, IT, 2, true>
                                     : embedding_rows_of_vectors_kernel<TT, OT, IT, 2, false>)
                    : vec == 4 ? (nt ? embedding_rows_of_vectors_kernel<TT, OT, IT, 4, true>
                                   : embedding_rows_of_vectors_kernel<TT, OT, IT, 4, false>)
                             : (nt ? embedding_rows_of_vectors_kernel<TT, OT, IT, W, true>
                                   : embedding_rows_of_vectors_kernel<TT, OT, IT, W, false>);
          hipLaunchKernelGGL(k, grid_for((N + rows - 1) / rows), dim3(256), 0, as_stream(stream), (const TT*)table,
                             table_stride, (const IT*)ids, N, V, make_div(D / vec), rows, (OT*)out, m, f, rng_used, oob);
        } else {
          const int rows = tile_rows(N, D, 256 * 4 * kUnroll, 4);
          auto* k = aligned(out, 4 * sizeof(OT)) ? embedding_any_rows_kernel<TT, OT, IT, true>
                                                 : embedding_any_rows_kernel<TT, OT, IT, false>;
          hipLaunchKernelGGL(k, grid_for((N + rows - 1) / rows), dim3(256), 0, as_stream(stream), (const TT*)table,
                             table_stride, (const IT*)ids, N, V, make_div(D), rows, (OT*)out, m, f, rng_used, oob);
        }
      });
    });
  });
  YN_LAUNCH_CHECK("embedding");
  return 0;
}

int yanerf_id_flag(int** flag) {
  YN_CHECK(flag, "id_flag: null pointer");
  void* p = nullptr;
  const hipError_t e = hipGetSymbolAddress(&p, HIP_SYMBOL(id_flag));
  YN_CHECK(e == hipSuccess, "id_flag: %s", hipGetErrorString(e));
  *flag = (int*)p;
  return 0;
}

int yanerf_flag_take(int* flag, int* taken, void* stream) {
  YN_CHECK(flag && taken && flag != taken, "flag_take: null or equal pointers");
  hipLaunchKernelGGL(take_flag_kernel, dim3(1), dim3(1), 0, as_stream(stream), flag, taken);
  YN_LAUNCH_CHECK("flag_take");
  return 0;
}

int64_t yanerf_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t D) {
  if (embedding_sizes_ok("embedding_bwd_workspace", N, V, D)) return -1;
  if (N == 0 || V == 0 || D == 0 || own_always(N, V, D)) return 0;
  int64_t bytes = grad_ws(N, V, D).bytes;
  for (int vec : {1, 2, 4}) {
    const DensePlan p = dense_plan(N, V, D, vec);
    if (p.vec && p.blocks * V * D * 4 > bytes) bytes = p.blocks * V * D * 4;
  }
  for (int64_t gb : {2, 4}) {  // of whichever type g has
    const BucketPlan b = bucket_plan(N, V, D, gb);
    if (b.buckets) {
      const int64_t n = bucket_ws(N, b, gb).bytes;
      bytes = n > bytes ? n : bytes;
    }
  }
  return bytes;
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
  YN_CHECK(N == 0 || (g && ids && (workspace || own_always(N, V, D))), "embedding_backward: null pointer");
  YN_CHECK(aligned(workspace, 16), "embedding_backward: the workspace is not aligned to 16 bytes");
  const Mask m = make_mask(p, seed, offset, rng_base);
  const double f = mask_scale(scale, p, m);
  if (factor_ok("embedding_backward", f)) return 1;
  hipStream_t st = as_stream(stream);
  char* ws = (char*)workspace;
  if (N == 0) {
    const int64_t halves = V * D * type_bytes(table_type) / 2;
    hipLaunchKernelGGL(zeros_kernel, grid_for((halves + 2047) / 2048), dim3(256), 0, st, (uint16_t*)grad_table, halves);
    YN_LAUNCH_CHECK("embedding_backward");
    return 0;
  }
  // elements a lane: rows of g and of the gradient start at multiples of it, and loads are of up to 16 bytes
  const int64_t gb = type_bytes(g_type), tb = type_bytes(table_type);
  int vec = (int)(16 / gb);
  while (vec > 1 && (D % vec || !aligned(g, vec * gb) || !aligned(grad_table, vec * tb < 16 ? vec * tb : 16))) vec /= 2;
  auto launch = [&](auto gt, auto tt, auto vc) {
    using GT = decltype(gt);
    using TT = decltype(tt);
    constexpr int VEC = decltype(vc)::value;
    const OwnPlan o = own_plan(N < kOwnMax ? N : kOwnMax, V, D, VEC, gb, tb);
    if (own_fits(N, V * D * tb, o)) {
      hipLaunchKernelGGL((own_rows_kernel<GT, TT, VEC>), dim3((unsigned)(o.chunks << o.lown)), dim3(kOwnThreads),
                         (unsigned)o.lds, st, (const GT*)g, ids, id_bytes, (int)N, V, D, padding_idx, o, m, f,
                         (TT*)grad_table);
      return;
    }
    const BucketPlan b = bucket_plan(N, V, D, gb);
    const DensePlan p = dense_plan(N, V, D, VEC);
    if (p.vec) {
      float* partial = (float*)ws;
      auto go = [&](auto dc) {
        constexpr int DV = decltype(dc)::value;
        if constexpr (DV <= VEC)
          hipLaunchKernelGGL((dense_sum_kernel<GT, DV>), dim3((unsigned)(p.blocks * p.chunks)), dim3(kDenseThreads),
                             (unsigned)p.lds, st, (const GT*)g, ids, id_bytes, N, V, D, padding_idx, p, m, partial);
      };
      using std::integral_constant;
      if (p.vec == 1) go(integral_constant<int, 1>{});
      else if (p.vec == 2) go(integral_constant<int, 2>{});
      else go(integral_constant<int, 4>{});
      int lo = 0;
      while (lo < 6 && (1ll << lo) < V * D) ++lo;
      hipLaunchKernelGGL((dense_join_kernel<TT>), dim3((unsigned)((V * D + (1 << lo) - 1) >> lo)), dim3(kDenseJoinThreads),
                         0, st, partial, p.blocks, V * D, lo, f, (TT*)grad_table);
      return;
    }
    if (N > kRankMax && b.buckets) {
      with_index(id_bytes, [&](auto it) {
        using IT = decltype(it);
        auto go = [&](auto dm) {
          bucket_gradient<GT, TT, decltype(dm)::value>((const GT*)g, (const IT*)ids, N, V, D, padding_idx, b, m, f,
                                                       (TT*)grad_table, ws, st);
        };
        using std::integral_constant;
        if (b.dm == 1) go(integral_constant<int, 1>{});
        else if (b.dm == 2) go(integral_constant<int, 2>{});
        else if (b.dm == 4) go(integral_constant<int, 4>{});
        else if constexpr (sizeof(GT) == 2) go(integral_constant<int, 8>{});
      });
      return;
    }
    const GradWs w = grad_ws(N, V, D);
    const RunPlan r = run_plan(N, D, VEC);
    int at = 0;
    with_index(id_bytes, [&](auto it) { at = sort_ids((const decltype(it)*)ids, N, V, padding_idx, ws, w, st); });
    const Pair* pairs = (const Pair*)(ws + w.pairs[at]);
    float *heads = (float*)(ws + w.heads), *tails = (float*)(ws + w.tails);
    int64_t rows = 65536 / (D * tb) < V / 512 ? 65536 / (D * tb) : V / 512;  // 64 KB of zeros, or two workgroups a CU
    rows = rows < 1 ? 1 : rows > kAbsentRows ? kAbsentRows : rows;
    const unsigned sums = (unsigned)(r.blocks * r.chunks), zeros = (unsigned)((V + rows - 1) / rows);
    hipLaunchKernelGGL((run_sum_kernel<GT, TT, VEC>), dim3(sums + zeros), dim3(kRunThreads), 0, st, (const GT*)g, pairs,
                       (uint32_t)V, N, D, r, m, f, (TT*)grad_table, heads, tails, (int)rows, make_div(D / VEC));
    if (r.blocks > 1)
      hipLaunchKernelGGL((run_join_kernel<TT, VEC>), dim3(sums), dim3(kRunThreads), 0, st, pairs, N, (uint32_t)V, D, r, f,
                         (TT*)grad_table, heads, tails);
  };
  with_type(g_type, [&](auto gt) {
    with_type(table_type, [&](auto tt) {
      using std::integral_constant;
      if (vec == 1) launch(gt, tt, integral_constant<int, 1>{});
      else if (vec == 2) launch(gt, tt, integral_constant<int, 2>{});
      else if (vec == 4) launch(gt, tt, integral_constant<int, 4>{});
      else if constexpr (sizeof(gt) == 2) launch(gt, tt, integral_constant<int, 8>{});
    });
  });
  YN_LAUNCH_CHECK("embedding_backward");
  return 0;
}

}  // extern "C"
