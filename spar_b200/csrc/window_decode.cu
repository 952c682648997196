// Window attention of a few rows against a long cache (a decoding step): the mathematics stands at
// the top of window_attention.cu.
//
// The floor is one read of the visible keys and values, which all query heads of a key head share:
// a CTA takes up to 8 (fp32) or 16 (bf16) rows (heads of one group, times tokens) and a range of the
// visible keys, so that a cache row is loaded once for that many: by cp.async, two steps ahead (one step ahead
// in registers every step waited for memory: 4 TB/s), each lane into slots of shared memory that it
// alone reads, so nothing but its own copies is waited for. (32 caches, 4096 visible keys, 32/8 heads of
// 128 bf16: 115 us with a flushed L2, 4.7 TB/s of the 6.55 of a copy.) Each warp (or lane group) keeps its own running
// maximum, sum and output; they are joined in shared memory, and the ranges of one row over the shared
// memory of a cluster of up to eight CTAs, or, where it takes more to fill the machine, by a second
// launch. Both add in a fixed order.
//
// bf16, head_dim a multiple of 32: mma.sync m16n8k16 with the rows as M. Fragments come from 16-byte
// vectors of the cache without a shuffle, since the order of a product's K and N indices is free:
//   scores: thread (g, t) of a warp holds key g, elements 8 t .. 8 t + 7 of each 32: two K steps
//   output: thread (g, t) holds keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9, elements 8 g .. 8 g + 7 of each
//           64; product j takes element 8 g + j of each (two byte permutes)
// P enters as two bf16 planes (16 bits), so the only rounding to bf16 is the result's. (The products
// are a few percent of the time; the tcgen05 path would spend 128 rows on the 8 here.)
// fp32 and other head sizes: fused multiply-adds, a cache row over L lanes, sums by shuffles.
#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "tc.cuh"
#include "window.cuh"

namespace spar_b200 {
namespace window {
namespace {

constexpr int kThreads = 128;
constexpr int kKeys = 4;    // rows of the cache that a lane group takes at once
constexpr int kStages = 3;  // steps of the ring, two of them under way (96 KB an SM at head_dim 128)
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DecodeParams {
  WindowParams w;
  int rows, row_blocks, splits;  // rows: query heads of a group x tokens
  int lanes_log2;
  float scale_log2;
  float* partial;  // [batch * kv_heads * rows][splits][head_dim + 2]: output, maximum, sum; or
                   // null: the ranges are a cluster
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes of the cache into this lane's slot, or zeros.
__device__ __forceinline__ void copy16(uint4* slot, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(slot)), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <typename T>
constexpr int kVec = 16 / sizeof(T);

template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[kVec<T>]);
template <>
__device__ __forceinline__ void unpack<float>(const uint4& u, float (&v)[4]) {
  v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y);
  v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
}
template <>
__device__ __forceinline__ void unpack<__nv_bfloat16>(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// The keys that the rows of one sequence see together: the first `kept` tokens, then from `start`.
struct Range {
  int kept, start, total;
  __device__ __forceinline__ int key(int i) const { return i < kept ? i : start + i - kept; }
};
__device__ __forceinline__ Range range_of(const WindowParams& w, const Sequence& s) {
  Range r = {0, 0, 0};
  const int pa = max(s.p0, 0), pb = min(s.p0 + w.q_len - 1, s.n - 1);
  if (pb < pa) return r;
  r.start = max(0, pa - w.window + 1);
  r.kept = min(w.sinks, r.start);
  r.total = r.kept + pb - r.start + 1;
  return r;
}

// Whether row i sees a key (then its own).
__device__ __forceinline__ bool sees_any(const WindowParams& w, int b, int i) {
  const Sequence s = sequence_of(w, b);
  return s.p0 + i >= 0 && s.p0 + i < s.n;
}

// Shared-memory address of `p` in CTA `rank` of the cluster, and a load from there.
__device__ __forceinline__ float load_from(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(tc::map_to_rank(tc::smem_u32(p), rank)) : "memory");
  return v;
}

// Joins a CTA's `groups` partial results, shared [group][rr][head_dim + 2] (output, maximum, sum;
// written by the caller), into shared's first [rr][head_dim + 2], and those of the row's ranges: from
// the cluster's shared memory, or through `partial` where the join is a launch of its own.
template <typename T>
__device__ __forceinline__ void finish(const DecodeParams& p, float* shared, int groups, int rr, int b,
                                       int kh, int row0, int split) {
  const WindowParams& w = p.w;
  const int stride = w.head_dim + 2, rows = min(rr, p.rows - row0);
  float* weight = shared + groups * rr * stride;  // [row][group]: 2^(maximum - the row's)
  __syncthreads();
  for (int r = threadIdx.x; r < rows; r += kThreads) {
    float top = -INFINITY, total = 0.f;
    for (int g = 0; g < groups; ++g) top = fmaxf(top, shared[(g * rr + r) * stride + w.head_dim]);
    const float base_m = top == -INFINITY ? 0.f : top;
    for (int g = 0; g < groups; ++g) {
      const float* src = shared + (g * rr + r) * stride + w.head_dim;
      const float f = ex2(src[0] - base_m);
      weight[r * groups + g] = f;
      total += src[1] * f;
    }
    weight[rows * groups + 2 * r] = top;
    weight[rows * groups + 2 * r + 1] = total;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < rows * w.head_dim; x += kThreads) {
    const int r = x / w.head_dim, e = x - r * w.head_dim;
    float o = 0.f;
    for (int g = 0; g < groups; ++g) o += shared[(g * rr + r) * stride + e] * weight[r * groups + g];
    shared[r * stride + e] = o;  // this thread alone reads element e of row r
  }
  for (int r = threadIdx.x; r < rows; r += kThreads) {
    shared[r * stride + w.head_dim] = weight[rows * groups + 2 * r];
    shared[r * stride + w.head_dim + 1] = weight[rows * groups + 2 * r + 1];
  }
  if (p.partial) {
    __syncthreads();
    const uint64_t bk = static_cast<uint64_t>(b) * w.kv_heads + kh;
    for (int x = threadIdx.x; x < rows * stride; x += kThreads) {
      const int r = x / stride;
      p.partial[((bk * p.rows + row0 + r) * p.splits + split) * stride + x - r * stride] = shared[x];
    }
    return;
  }
  tc::cluster_sync();  // a cluster of one: a barrier of the CTA
  for (int x = split * kThreads + threadIdx.x; x < rows * w.head_dim; x += p.splits * kThreads) {
    const int r = x / w.head_dim, e = x - r * w.head_dim, row = row0 + r;
    const int i = row / w.group, h = kh * w.group + row - i * w.group;
    const float* at = shared + r * stride;
    float top = -INFINITY, total = 0.f, o = 0.f;
    for (int k = 0; k < p.splits; ++k) top = fmaxf(top, load_from(at + w.head_dim, k));
    const float base_m = top == -INFINITY ? 0.f : top;
    for (int k = 0; k < p.splits; ++k) {
      const float f = ex2(load_from(at + w.head_dim, k) - base_m);
      total += load_from(at + w.head_dim + 1, k) * f;
      o += load_from(at + e, k) * f;
    }
    put(row_out<T>(w.out, b, i, h) + e, sees_any(w, b, i) ? o / total : 0.f);
    if (e == 0 && w.lse)
      w.lse[(static_cast<uint64_t>(b) * w.heads + h) * w.q_len + i] = base_m * kLn2 + logf(total);
  }
  tc::cluster_sync();  // nobody leaves while its shared memory is read
}

template <typename T, int RR>
__global__ void __launch_bounds__(kThreads) window_decode_kernel(
    const __grid_constant__ DecodeParams p) {
  pdl_begin();
  constexpr int V = kVec<T>;
  extern __shared__ float shared[];
  const WindowParams& w = p.w;
  const int lanes = 1 << p.lanes_log2, l = threadIdx.x & (lanes - 1);
  const int group = threadIdx.x >> p.lanes_log2, groups = kThreads >> p.lanes_log2;
  const int split = blockIdx.x, bk = blockIdx.y / p.row_blocks;
  const int row0 = (blockIdx.y - bk * p.row_blocks) * RR;
  const int b = bk / w.kv_heads, kh = bk - b * w.kv_heads;
  const Sequence s = sequence_of(w, b);
  const Range range = range_of(w, s);
  // Whole steps of the CTA per range, the ranges equal within one step.
  const int step = groups * kKeys;
  const int per = (range.total + step * p.splits - 1) / (step * p.splits) * step;
  const int from = min(split * per, range.total), to = min(from + per, range.total);
  const bool in = l * V < w.head_dim;

  float q[RR][V], acc[RR][V], m[RR], sum[RR];
  int pos[RR];
#pragma unroll
  for (int r = 0; r < RR; ++r) {
    const int row = row0 + r, i = row / w.group, h = kh * w.group + row - i * w.group;
    pos[r] = s.p0 + i;
    if (row >= p.rows || pos[r] >= s.n) pos[r] = -1;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (in && row < p.rows) u = *reinterpret_cast<const uint4*>(row_ptr<T>(w.q, b, i, h) + l * V);
    unpack<T>(u, q[r]);
    m[r] = -INFINITY;
    sum[r] = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      q[r][e] *= p.scale_log2;
      acc[r][e] = 0.f;
    }
  }
  const T* kb = row_ptr<T>(w.k, b, 0, kh) + l * V;
  const T* vb = row_ptr<T>(w.v, b, 0, kh) + l * V;
  uint4* ring = reinterpret_cast<uint4*>(shared) + threadIdx.x;  // [stage][key, value][kKeys] slots
  auto fetch = [&](int base, int stage) {
    uint4* slot = ring + stage * 2 * kKeys * kThreads;
#pragma unroll
    for (int x = 0; x < kKeys; ++x) {
      const int i = base + group + x * groups;
      const bool there = i < to && in;
      const uint64_t key = static_cast<uint64_t>(there ? range.key(i) : 0);
      copy16(slot + x * kThreads, kb + key * w.k.token, there);
      copy16(slot + (kKeys + x) * kThreads, vb + key * w.v.token, there);
    }
    copies_commit();
  };
#pragma unroll
  for (int n = 0; n < kStages - 1; ++n) fetch(from + n * step, n);
  int stage = 0;
  for (int base = from; base < to; base += step) {
    float score[kKeys][RR];
    copies_wait<kStages - 2>();
    const uint4* slot = ring + stage * 2 * kKeys * kThreads;
#pragma unroll
    for (int x = 0; x < kKeys; ++x) {
      float k[V];
      unpack<T>(slot[x * kThreads], k);
#pragma unroll
      for (int r = 0; r < RR; ++r) {
        score[x][r] = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) score[x][r] = fmaf(q[r][e], k[e], score[x][r]);
      }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int x = 0; x < kKeys; ++x)
#pragma unroll
        for (int r = 0; r < RR; ++r) score[x][r] += __shfl_xor_sync(0xffffffffu, score[x][r], o);
    }
    fetch(base + (kStages - 1) * step, (stage + kStages - 1) % kStages);
    const int at = base + group;
#pragma unroll
    for (int x = 0; x < kKeys; ++x) {
      const int i = at + x * groups;
      const int key = i < to ? range.key(i) : INT_MAX;
#pragma unroll
      for (int r = 0; r < RR; ++r)
        if (key > pos[r] || (key <= pos[r] - w.window && key >= w.sinks)) score[x][r] = -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < RR; ++r) {
      float top = m[r];
#pragma unroll
      for (int x = 0; x < kKeys; ++x) top = fmaxf(top, score[x][r]);
      const float base_m = top == -INFINITY ? 0.f : top;
      const float f = ex2(m[r] - base_m);
      m[r] = top;
      sum[r] *= f;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[r][e] *= f;
#pragma unroll
      for (int x = 0; x < kKeys; ++x) {
        score[x][r] = ex2(score[x][r] - base_m);
        sum[r] += score[x][r];
      }
    }
#pragma unroll
    for (int x = 0; x < kKeys; ++x) {
      float v[V];
      unpack<T>(slot[(kKeys + x) * kThreads], v);
#pragma unroll
      for (int r = 0; r < RR; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r][e] = fmaf(score[x][r], v[e], acc[r][e]);
    }
    stage = (stage + 1) % kStages;
  }
  copies_wait<0>();
  __syncthreads();  // the ring's memory is reused

  // shared: [group][row][head_dim + 2]
  const int stride = w.head_dim + 2;
#pragma unroll
  for (int r = 0; r < RR; ++r) {
    float* dst = shared + (group * RR + r) * stride;
    if (in) {
#pragma unroll
      for (int e = 0; e < V; ++e) dst[l * V + e] = acc[r][e];
    }
    if (l == 0) {
      dst[w.head_dim] = m[r];
      dst[w.head_dim + 1] = sum[r];
    }
  }
  finish<T>(p, shared, groups, RR, b, kh, row0, split);
}

// ------------------------------------------------------------------------------- bf16 products
__device__ __forceinline__ void mma_m16n8k16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same with rows 8 .. 15 of A zero and of D dropped.
__device__ __forceinline__ void mma_m8n8k16(float (&d)[2], uint32_t a0, uint32_t a2, uint32_t b0,
                                            uint32_t b1) {
  const uint32_t z = 0;
  const float zero = 0.f;
  [[maybe_unused]] float x, y;
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %6, %5, %6}, "
      "{%7, %8}, {%0, %1, %9, %9};"
      : "+f"(d[0]), "+f"(d[1]), "=f"(x), "=f"(y)
      : "r"(a0), "r"(a2), "r"(z), "r"(b0), "r"(b1), "f"(zero));
}
template <int RB>
__device__ __forceinline__ void mma_rows(float (&d)[2 * RB], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (RB == 1)
    mma_m8n8k16(d, a[0], a[2], b0, b1);
  else
    mma_m16n8k16(d, a, b0, b1);
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// DB: blocks of 32 elements of a head; RB: blocks of 8 rows (1 or 2).
template <int DB, int RB>
__global__ void __launch_bounds__(kThreads) window_decode_mma_kernel(
    const __grid_constant__ DecodeParams p) {
  pdl_begin();
  using T = __nv_bfloat16;
  constexpr int VB = (DB + 1) / 2;  // blocks of 64 elements of a value row
  extern __shared__ float shared[];
  const WindowParams& w = p.w;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, bk = blockIdx.y / p.row_blocks;
  const int row0 = (blockIdx.y - bk * p.row_blocks) * 8 * RB;
  const int b = bk / w.kv_heads, kh = bk - b * w.kv_heads;
  const Sequence s = sequence_of(w, b);
  const Range range = range_of(w, s);
  constexpr int kStep = kThreads / 32 * 16;
  const int per = (range.total + kStep * p.splits - 1) / (kStep * p.splits) * kStep;
  const int from = min(split * per, range.total), to = min(from + per, range.total);

  uint32_t q[DB][2][RB][2];  // [block][K step][rows g, g + 8][first, second pair of the step]
  int pos[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int row = row0 + g + 8 * r, i = row / w.group, h = kh * w.group + row - i * w.group;
    pos[r] = s.p0 + i;
    if (row >= p.rows || pos[r] >= s.n) pos[r] = -1;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (row < p.rows) u = *reinterpret_cast<const uint4*>(row_ptr<T>(w.q, b, i, h) + d * 32 + t * 8);
      q[d][0][r][0] = u.x, q[d][0][r][1] = u.y, q[d][1][r][0] = u.z, q[d][1][r][1] = u.w;
    }
  }
  float acc[VB][8][2 * RB], m[RB], sum[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) m[r] = -INFINITY, sum[r] = 0.f;
#pragma unroll
  for (int d = 0; d < VB; ++d)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2 * RB; ++e) acc[d][j][e] = 0.f;

  const T* kb = row_ptr<T>(w.k, b, 0, kh) + t * 8;
  const T* vb = row_ptr<T>(w.v, b, 0, kh) + g * 8;
  constexpr int kSlots = 2 * DB + 4 * VB;
  uint4* ring = reinterpret_cast<uint4*>(shared) + threadIdx.x;  // [stage][slot]
  auto fetch = [&](int base, int stage) {
    uint4* slot = ring + stage * kSlots * kThreads;
#pragma unroll
    for (int x = 0; x < 2; ++x) {  // keys base + g, base + 8 + g
      const int i = base + 8 * x + g;
      const T* src = kb + static_cast<uint64_t>(i < to ? range.key(i) : 0) * w.k.token;
#pragma unroll
      for (int d = 0; d < DB; ++d) copy16(slot + (x * DB + d) * kThreads, src + d * 32, i < to);
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {  // keys base + 2t, + 1, + 8, + 9
      const int i = base + 2 * t + (x & 1) + (x >> 1) * 8;
      const T* src = vb + static_cast<uint64_t>(i < to ? range.key(i) : 0) * w.v.token;
#pragma unroll
      for (int d = 0; d < VB; ++d) {
        const bool there = i < to && (DB % 2 == 0 || d * 64 + g * 8 < DB * 32);
        copy16(slot + (2 * DB + x * VB + d) * kThreads, there ? src + d * 64 : vb, there);
      }
    }
    copies_commit();
  };
  int base = from + warp * 16, stage = 0;
#pragma unroll
  for (int n = 0; n < kStages - 1; ++n) fetch(base + n * kStep, n);
  for (; base < to; base += kStep) {
    copies_wait<kStages - 2>();
    const uint4* slot = ring + stage * kSlots * kThreads;
    float sc[2][2 * RB];  // [8 keys][row g: keys 2t, 2t + 1; row g + 8: the same]
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int e = 0; e < 2 * RB; ++e) sc[x][e] = 0.f;
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const uint32_t a0[4] = {q[d][0][0][0], RB > 1 ? q[d][0][RB - 1][0] : 0, q[d][0][0][1],
                                RB > 1 ? q[d][0][RB - 1][1] : 0};
        const uint32_t a1[4] = {q[d][1][0][0], RB > 1 ? q[d][1][RB - 1][0] : 0, q[d][1][0][1],
                                RB > 1 ? q[d][1][RB - 1][1] : 0};
        const uint4 k = slot[(x * DB + d) * kThreads];
        mma_rows<RB>(sc[x], a0, k.x, k.y);
        mma_rows<RB>(sc[x], a1, k.z, k.w);
      }
    }
    fetch(base + (kStages - 1) * kStep, (stage + kStages - 1) % kStages);
    // Keys of this thread's columns; the whole tile inside every row's window is the usual case.
    const int at = base + 2 * t;
    uint32_t hi[4] = {0, 0, 0, 0}, lo[4] = {0, 0, 0, 0};
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      float v[4] = {sc[0][2 * r], sc[0][2 * r + 1], sc[1][2 * r], sc[1][2 * r + 1]};
      float top = m[r];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int i = at + (x & 1) + (x >> 1) * 8;
        const int key = i < to ? range.key(i) : INT_MAX;
        if (key > pos[r] || (key <= pos[r] - w.window && key >= w.sinks)) v[x] = -INFINITY;
        v[x] *= p.scale_log2;
        top = fmaxf(top, v[x]);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float base_m = top == -INFINITY ? 0.f : top;
      if (__any_sync(0xffffffffu, top > m[r])) {
        const float f = ex2(m[r] - base_m);
        sum[r] *= f;
#pragma unroll
        for (int d = 0; d < VB; ++d)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            acc[d][j][2 * r] *= f;
            acc[d][j][2 * r + 1] *= f;
          }
      }
      m[r] = top;
      float rest[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        v[x] = ex2(v[x] - base_m);
        sum[r] += v[x];
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t u = pack_bf16(v[2 * x], v[2 * x + 1]);
        hi[2 * x + r] = u;
        rest[2 * x] = v[2 * x] - __uint_as_float(u << 16);
        rest[2 * x + 1] = v[2 * x + 1] - __uint_as_float(u & 0xffff0000u);
        lo[2 * x + r] = pack_bf16(rest[2 * x], rest[2 * x + 1]);
      }
    }
#pragma unroll
    for (int d = 0; d < VB; ++d) {
      uint32_t v[4][4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint4 u = slot[(2 * DB + x * VB + d) * kThreads];
        v[x][0] = u.x, v[x][1] = u.y, v[x][2] = u.z, v[x][3] = u.w;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t a = v[0][j / 2], c = v[1][j / 2], e = v[2][j / 2], f = v[3][j / 2];
        const uint32_t pick = j & 1 ? 0x7632 : 0x5410;
        const uint32_t b0 = __byte_perm(a, c, pick), b1 = __byte_perm(e, f, pick);
        mma_rows<RB>(acc[d][j], lo, b0, b1);
        mma_rows<RB>(acc[d][j], hi, b0, b1);
      }
    }
    stage = (stage + 1) % kStages;
  }
  copies_wait<0>();
  __syncthreads();  // the ring's memory is reused
  // A row's sum is spread over the four threads of its group; each has the row's maximum.
  // shared: [warp][row][head_dim + 2]
  const int stride = w.head_dim + 2;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    float total = sum[r];
    total += __shfl_xor_sync(0xffffffffu, total, 1);
    total += __shfl_xor_sync(0xffffffffu, total, 2);
    float* dst = shared + (warp * 8 * RB + g + 8 * r) * stride;
    if (t == 0) {
      dst[w.head_dim] = m[r];
      dst[w.head_dim + 1] = total;
    }
#pragma unroll
    for (int d = 0; d < VB; ++d)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int e = d * 64 + (2 * t + x) * 8 + j;
          if (DB % 2 == 0 || e < DB * 32) dst[e] = acc[d][j][2 * r + x];
        }
  }
  finish<T>(p, shared, kThreads / 32, 8 * RB, b, kh, row0, split);
}

// One CTA per row: the ranges' partials, added in an order that depends on the sizes alone. Groups of
// threads as wide as a head take every (number of groups)-th range.
constexpr int kJoinThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) window_join_kernel(const __grid_constant__ DecodeParams p,
                                                                   int width) {
  pdl_begin();
  extern __shared__ float weight[];  // [splits], then [kJoinThreads] sums
  __shared__ float scratch[32];
  const WindowParams& w = p.w;
  const int row = blockIdx.x, bk = blockIdx.y;
  const int b = bk / w.kv_heads, kh = bk - b * w.kv_heads;
  const int i = row / w.group, h = kh * w.group + row - i * w.group;
  const int stride = w.head_dim + 2;
  const float* src = p.partial + (static_cast<uint64_t>(bk) * p.rows + row) * p.splits * stride;
  float top = -INFINITY, total = 0.f;
  for (int s = threadIdx.x; s < p.splits; s += kJoinThreads) top = fmaxf(top, src[s * stride + w.head_dim]);
  top = block_max(top, scratch);
  const float base_m = top == -INFINITY ? 0.f : top;
  for (int s = threadIdx.x; s < p.splits; s += kJoinThreads) {
    const float f = ex2(src[s * stride + w.head_dim] - base_m);
    weight[s] = f;
    total += src[s * stride + w.head_dim + 1] * f;
  }
  total = block_sum(total, scratch);
  __syncthreads();
  const int e = threadIdx.x % width, group = threadIdx.x / width, groups = kJoinThreads / width;
  float o = 0.f;
  if (e < w.head_dim) {
#pragma unroll 8
    for (int s = group; s < p.splits; s += groups) o += src[s * stride + e] * weight[s];
  }
  float* sums = weight + p.splits;
  sums[threadIdx.x] = o;
  __syncthreads();
  if (group == 0 && e < w.head_dim) {
    for (int g = 1; g < groups; ++g) o += sums[g * width + e];
    put(row_out<T>(w.out, b, i, h) + e, sees_any(w, b, i) ? o / total : 0.f);
  }
  if (threadIdx.x == 0 && w.lse)
    w.lse[(static_cast<uint64_t>(b) * w.heads + h) * w.q_len + i] = base_m * kLn2 + logf(total);
}

constexpr int kMaxCluster = 8;

struct DecodePlan {
  bool mma;
  int rows, rr, row_blocks, splits, groups, lanes_log2;
  size_t smem;
};
DecodePlan decode_plan(const WindowParams& w, int device) {
  DecodePlan d;
  d.rows = w.group * w.q_len;
  d.mma = w.dtype == SPAR_B200_BFLOAT16 && w.head_dim % 32 == 0 && w.head_dim <= 128;
  d.rr = d.mma ? 8 : 1;
  while (d.rr < (d.mma ? 16 : 8) && d.rr < d.rows) d.rr *= 2;
  d.row_blocks = (d.rows + d.rr - 1) / d.rr;
  const int vec = w.dtype == SPAR_B200_FLOAT32 ? 4 : 8;
  d.lanes_log2 = 0;
  while ((1 << d.lanes_log2) * vec < w.head_dim) ++d.lanes_log2;
  d.groups = d.mma ? kThreads / 32 : kThreads >> d.lanes_log2;
  const int blocks = w.head_dim / 32;
  const size_t ring = static_cast<size_t>(kStages) * kThreads * 16 *
                      (d.mma ? 2 * blocks + 4 * ((blocks + 1) / 2) : 2 * kKeys);
  d.smem = std::max(ring, (static_cast<size_t>(d.groups) * d.rr * (w.head_dim + 2) + d.rr * (d.groups + 2)) *
                              sizeof(float));
  // Ranges so that the CTAs fill whole rounds of the machine: rounds x (keys of a range + what a
  // CTA's start and join cost, about 96 keys' time) at its least, none with less than two steps' keys.
  // Up to eight are joined inside a cluster.
  const int step = d.mma ? kThreads / 32 * 16 : d.groups * kKeys;
  const int64_t keys = std::min<int64_t>(w.kv_len, static_cast<int64_t>(w.window) + w.q_len + w.sinks);
  const int64_t ctas = static_cast<int64_t>(w.batch) * w.kv_heads * d.row_blocks;
  const int64_t slots = sm_count(device) * std::min<int64_t>(3, (227 << 10) / (d.smem + 1024));
  const int64_t most = std::max<int64_t>(1, std::min((2 * slots + ctas - 1) / ctas, keys / (2 * step)));
  int64_t best = INT64_MAX;
  d.splits = 1;
  for (int64_t rounds = (ctas + slots - 1) / slots; rounds <= (ctas * most + slots - 1) / slots; ++rounds) {
    // the most ranges of so many rounds, or fewer that are as long
    const int64_t longest = std::max<int64_t>(1, (keys + most - 1) / most);
    const int64_t n_most = std::max<int64_t>(1, std::min(most, rounds * slots / ctas));
    const int64_t range = std::max(longest, (keys + n_most - 1) / n_most);
    const int64_t cost = rounds * (range + 96);
    if (cost < best) best = cost, d.splits = static_cast<int>(std::max<int64_t>(1, (keys + range - 1) / range));
  }
  return d;
}

template <typename T>
cudaError_t launch_decode(void (*kernel)(DecodeParams), const DecodeParams& p, const DecodePlan& d,
                          int device, cudaStream_t stream) {
  cudaError_t e = raise_dynamic_smem(reinterpret_cast<const void*>(kernel), device, d.smem);
  if (e != cudaSuccess) return e;
  const unsigned y = static_cast<unsigned>(p.w.batch * p.w.kv_heads);
  const dim3 grid(p.splits, y * p.row_blocks);
  if (p.partial) {
    e = launch(kernel, grid, dim3(kThreads), d.smem, stream, p);
    if (e != cudaSuccess) return e;
    int width = 32;
    while (width < p.w.head_dim) width *= 2;
    return launch(window_join_kernel<T>, dim3(p.rows, y), dim3(kJoinThreads),
                  (p.splits + kJoinThreads) * sizeof(float), stream, p, width);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = d.smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int RB>
auto mma_kernel(int head_dim) -> void (*)(DecodeParams) {
  return head_dim == 32   ? window_decode_mma_kernel<1, RB>
         : head_dim == 64 ? window_decode_mma_kernel<2, RB>
         : head_dim == 96 ? window_decode_mma_kernel<3, RB>
                          : window_decode_mma_kernel<4, RB>;
}
template <typename T>
auto simt_kernel(int rr) -> void (*)(DecodeParams) {
  return rr == 1   ? window_decode_kernel<T, 1>
         : rr == 2 ? window_decode_kernel<T, 2>
         : rr == 4 ? window_decode_kernel<T, 4>
                   : window_decode_kernel<T, 8>;
}

}  // namespace

bool decode_supported(const WindowParams& w) {
  const int size = w.dtype == SPAR_B200_FLOAT32 ? 4 : 2, vec = 16 / size;
  const int64_t rows = static_cast<int64_t>(w.group) * w.q_len;
  // Up to 64 rows where the cache is long beside them: ranges of keys then fill the machine, which the
  // tiled path's few items do not (64 rows of 1024 keys, 8 x 4 heads of 64 bf16: 21 against 27 us; 40
  // rows of 4096 keys, 8 heads of 128 fp32: 93 against 309 us, as the tiled path splits the whole cache
  // into planes). Short caches are better tiled (64 rows of 64 keys, 32 x 32 heads of 128 bf16: 30
  // against 213 us). Rule and plan go by the cache's capacity, since the lengths are on the device: ranges
  // planned for 16384 keys of which 512 are used, 32/8 heads of 128 bf16, cost one cache 10.2 against 6.6
  // us, four 10.8 against 7.8, and 32, which fill the machine, nothing.
  const int64_t keys = std::min<int64_t>(w.kv_len, static_cast<int64_t>(w.window) + w.q_len + w.sinks);
  return rows > 0 && (rows <= 16 || (rows <= 64 && keys >= 8 * rows)) && w.head_dim % vec == 0 &&
         w.head_dim / vec <= 32 && w.kv_len > 0 &&
         static_cast<int64_t>(w.batch) * w.kv_heads * ((rows + 7) / 8) < 65536 &&
         tiled_view(w.q, size, w.batch, w.q_len, w.heads) &&
         tiled_view(w.k, size, w.batch, w.kv_len, w.kv_heads) &&
         tiled_view(w.v, size, w.batch, w.kv_len, w.kv_heads);
}

uint64_t decode_scratch_bytes(const WindowParams& w, int device) {
  const DecodePlan d = decode_plan(w, device);
  if (d.splits <= kMaxCluster) return 0;
  return static_cast<uint64_t>(w.batch) * w.kv_heads * d.rows * d.splits * (w.head_dim + 2) * sizeof(float);
}

cudaError_t decode_forward(const WindowParams& w, void* scratch, int device, cudaStream_t stream) {
  const DecodePlan d = decode_plan(w, device);
  DecodeParams p = {};
  p.w = w;
  p.rows = d.rows;
  p.row_blocks = d.row_blocks;
  p.splits = d.splits;
  p.lanes_log2 = d.lanes_log2;
  p.scale_log2 = w.scale * kLog2e;
  p.partial = d.splits > kMaxCluster ? static_cast<float*>(scratch) : nullptr;
  if (w.dtype == SPAR_B200_FLOAT32)
    return launch_decode<float>(simt_kernel<float>(d.rr), p, d, device, stream);
  return launch_decode<__nv_bfloat16>(d.mma ? (d.rr == 8 ? mma_kernel<1>(w.head_dim) : mma_kernel<2>(w.head_dim))
                                            : simt_kernel<__nv_bfloat16>(d.rr),
                                      p, d, device, stream);
}

}  // namespace window
}  // namespace spar_b200
