// Window attention of a few rows against a long cache (a decoding step): the mathematics stands at
// the top of window_attention.cu.
//
// The floor is one read of the visible keys and values, which all query heads of a key head share:
// a CTA takes up to RR rows (heads of one group, times tokens) and a range of the visible keys, so
// that a cache row is loaded once for all of them. A row of the cache is 16-byte vectors over L
// neighbouring lanes; each lane group walks its own keys, KB at a time, with its own running
// maximum, sum and output in registers (fp32), the next KB rows already on their way. Groups are
// joined in shared memory, and the ranges (as many as fill the machine) by a second launch that
// adds them in order.
#include <algorithm>

#include "common.cuh"
#include "kernels.cuh"
#include "window.cuh"

namespace spar_b200 {
namespace window {
namespace {

constexpr int kThreads = 128;
constexpr int kKeys = 4;  // rows of the cache in flight per lane group
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct DecodeParams {
  WindowParams w;
  int rows, row_blocks, splits;  // rows: query heads of a group x tokens
  int lanes_log2;
  float scale_log2;
  float* partial;  // [batch * kv_heads * rows][splits][head_dim + 2]: output, maximum, sum
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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
  uint4 ku[kKeys], vu[kKeys];
  auto fetch = [&](int base) {
#pragma unroll
    for (int x = 0; x < kKeys; ++x) {
      const int i = base + x * groups;
      ku[x] = vu[x] = make_uint4(0, 0, 0, 0);
      if (i < to && in) {
        const uint64_t key = static_cast<uint64_t>(range.key(i));
        ku[x] = __ldg(reinterpret_cast<const uint4*>(kb + key * w.k.token));
        vu[x] = __ldg(reinterpret_cast<const uint4*>(vb + key * w.v.token));
      }
    }
  };
  fetch(from + group);
  for (int base = from; base < to; base += step) {
    float score[kKeys][RR];
#pragma unroll
    for (int x = 0; x < kKeys; ++x) {
      float k[V];
      unpack<T>(ku[x], k);
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
    uint4 held[kKeys];
#pragma unroll
    for (int x = 0; x < kKeys; ++x) held[x] = vu[x];
    const int at = base + group;
    fetch(at + step);
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
      unpack<T>(held[x], v);
#pragma unroll
      for (int r = 0; r < RR; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[r][e] = fmaf(score[x][r], v[e], acc[r][e]);
    }
  }

  // Join the groups of the CTA: shared [group][row][head_dim + 2].
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
  __syncthreads();
  for (int r = 0; r < RR && row0 + r < p.rows; ++r) {
    const int row = row0 + r, i = row / w.group, h = kh * w.group + row - i * w.group;
    float top = -INFINITY, total = 0.f;
    for (int g = 0; g < groups; ++g) top = fmaxf(top, shared[(g * RR + r) * stride + w.head_dim]);
    const float base_m = top == -INFINITY ? 0.f : top;
    for (int g = 0; g < groups; ++g) {
      const float* src = shared + (g * RR + r) * stride + w.head_dim;
      total += src[1] * ex2(src[0] - base_m);
    }
    for (int e = threadIdx.x; e < w.head_dim; e += kThreads) {
      float o = 0.f;
      for (int g = 0; g < groups; ++g) {
        const float* src = shared + (g * RR + r) * stride;
        o += src[e] * ex2(src[w.head_dim] - base_m);
      }
      if (p.splits == 1)
        put(row_out<T>(w.out, b, i, h) + e, total > 0.f || total != total ? o / total : 0.f);
      else
        p.partial[((static_cast<uint64_t>(bk) * p.rows + row) * p.splits + split) * stride + e] = o;
    }
    if (threadIdx.x == 0) {
      if (p.splits == 1) {
        if (w.lse)
          w.lse[(static_cast<uint64_t>(b) * w.heads + h) * w.q_len + i] = base_m * kLn2 + logf(total);
      } else {
        float* dst = p.partial +
                     ((static_cast<uint64_t>(bk) * p.rows + row) * p.splits + split) * stride + w.head_dim;
        dst[0] = top;
        dst[1] = total;
      }
    }
  }
}

// One CTA per row: the ranges' partials added in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) window_join_kernel(const __grid_constant__ DecodeParams p) {
  pdl_begin();
  const WindowParams& w = p.w;
  const int row = blockIdx.x, bk = blockIdx.y;
  const int b = bk / w.kv_heads, kh = bk - b * w.kv_heads;
  const int i = row / w.group, h = kh * w.group + row - i * w.group;
  const int stride = w.head_dim + 2;
  const float* src = p.partial + (static_cast<uint64_t>(bk) * p.rows + row) * p.splits * stride;
  float top = -INFINITY, total = 0.f;
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, src[s * stride + w.head_dim]);
  const float base_m = top == -INFINITY ? 0.f : top;
  for (int s = 0; s < p.splits; ++s)
    total += src[s * stride + w.head_dim + 1] * ex2(src[s * stride + w.head_dim] - base_m);
  for (int e = threadIdx.x; e < w.head_dim; e += kThreads) {
    float o = 0.f;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) o += src[s * stride + e] * ex2(src[s * stride + w.head_dim] - base_m);
    put(row_out<T>(w.out, b, i, h) + e, total > 0.f || total != total ? o / total : 0.f);
  }
  if (threadIdx.x == 0 && w.lse)
    w.lse[(static_cast<uint64_t>(b) * w.heads + h) * w.q_len + i] = base_m * kLn2 + logf(total);
}

struct DecodePlan {
  int rows, rr, row_blocks, splits, lanes_log2;
};
DecodePlan decode_plan(const WindowParams& w, int device) {
  DecodePlan d;
  d.rows = w.group * w.q_len;
  d.rr = 1;
  while (d.rr < 8 && d.rr < d.rows) d.rr *= 2;
  d.row_blocks = (d.rows + d.rr - 1) / d.rr;
  const int vec = w.dtype == SPAR_B200_FLOAT32 ? 4 : 8;
  d.lanes_log2 = 0;
  while ((1 << d.lanes_log2) * vec < w.head_dim) ++d.lanes_log2;
  // Four CTAs per SM, none with less than two steps' keys.
  const int step = (kThreads >> d.lanes_log2) * kKeys;
  const int64_t keys = std::min<int64_t>(w.kv_len, static_cast<int64_t>(w.window) + w.q_len + w.sinks);
  const int64_t ctas = static_cast<int64_t>(w.batch) * w.kv_heads * d.row_blocks;
  const int64_t fill = (4 * sm_count(device) + ctas - 1) / ctas;
  d.splits = static_cast<int>(std::max<int64_t>(1, std::min(fill, keys / (2 * step))));
  return d;
}

template <typename T, int RR>
cudaError_t launch_decode(const DecodeParams& p, int device, cudaStream_t stream) {
  auto kernel = window_decode_kernel<T, RR>;
  const size_t smem = static_cast<size_t>(kThreads >> p.lanes_log2) * RR * (p.w.head_dim + 2) * sizeof(float);
  cudaError_t e = raise_dynamic_smem(reinterpret_cast<const void*>(kernel), device, smem);
  if (e != cudaSuccess) return e;
  const unsigned y = static_cast<unsigned>(p.w.batch * p.w.kv_heads);
  e = launch(kernel, dim3(p.splits, y * p.row_blocks), dim3(kThreads), smem, stream, p);
  if (e != cudaSuccess || p.splits == 1) return e;
  return launch(window_join_kernel<T>, dim3(p.rows, y), dim3(kThreads), 0, stream, p);
}

}  // namespace

bool decode_supported(const WindowParams& w) {
  const int size = w.dtype == SPAR_B200_FLOAT32 ? 4 : 2, vec = 16 / size;
  const int64_t rows = static_cast<int64_t>(w.group) * w.q_len;
  return rows > 0 && rows <= 32 && w.head_dim % vec == 0 && w.head_dim / vec <= 32 && w.kv_len > 0 &&
         static_cast<int64_t>(w.batch) * w.kv_heads * ((rows + 7) / 8) < 65536 &&
         tiled_view(w.q, size, w.batch, w.q_len, w.heads) &&
         tiled_view(w.k, size, w.batch, w.kv_len, w.kv_heads) &&
         tiled_view(w.v, size, w.batch, w.kv_len, w.kv_heads);
}

uint64_t decode_scratch_bytes(const WindowParams& w, int device) {
  const DecodePlan d = decode_plan(w, device);
  if (d.splits == 1) return 0;
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
  p.partial = static_cast<float*>(scratch);
  if (w.dtype == SPAR_B200_FLOAT32)
    return d.rr == 1   ? launch_decode<float, 1>(p, device, stream)
           : d.rr == 2 ? launch_decode<float, 2>(p, device, stream)
           : d.rr == 4 ? launch_decode<float, 4>(p, device, stream)
                       : launch_decode<float, 8>(p, device, stream);
  return d.rr == 1   ? launch_decode<__nv_bfloat16, 1>(p, device, stream)
         : d.rr == 2 ? launch_decode<__nv_bfloat16, 2>(p, device, stream)
         : d.rr == 4 ? launch_decode<__nv_bfloat16, 4>(p, device, stream)
                     : launch_decode<__nv_bfloat16, 8>(p, device, stream);
}

}  // namespace window
}  // namespace spar_b200
