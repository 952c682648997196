// Causal attention with a sliding window and first tokens that stay visible, forward and backward.
//
// Row i of sequence b stands at position p = first[b] + i and sees the keys
//   K(p) = { j : j <= p, j < n_b, and j > p - window or j < sinks }   (empty when p >= n_b).
//   s_j = scale q.k_j;  lse = ln sum exp(s_j);  out = sum exp(s_j - lse) v_j
// Backward with P_j = exp(s_j - lse), D = dout.out:
//   dv_j += P_j dout;  ds_j = P_j (dout.v_j - D);  dq = scale sum ds_j k_j;  dk_j += scale ds_j q
// where dk, dv of a key / value head sum over its group of query heads.
#include <cuda_bf16.h>

#include <cmath>

#include "common.cuh"
#include "kernels.cuh"
#include "window.cuh"

namespace spar_b200 {
namespace window {
namespace {

// ------------------------------------------------------------------------- any shape and stride
// One warp per row, lanes over the head's elements (E of them each), one pass over the visible
// keys with a running maximum and sum. Reads elements one by one, so it takes every head_dim,
// stride and alignment; it is the path of the rows that the tiled kernels cannot address. Bound by
// its instructions (five shuffles a dot product): 2 x 1023 x 8/4 heads of 100 bf16, window 256, 500 us
// forward and 1620 us backward, where the tiled kernels take 15 and 48 us for heads of 96.
constexpr int kRowWarps = 4;

template <typename T, int E>
__device__ __forceinline__ void load_row(float (&r)[E], const T* p, int dim, int lane) {
#pragma unroll
  for (int e = 0; e < E; ++e) r[e] = lane + 32 * e < dim ? as_float(p[lane + 32 * e]) : 0.f;
}
template <int E>
__device__ __forceinline__ float dot_row(const float (&a)[E], const float (&b)[E]) {
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) s += a[e] * b[e];
  return warp_sum(s);
}

// The unit of this warp among `units`, or false. Units may exceed the grid's x limit in no case:
// the host refuses such sizes.
__device__ __forceinline__ bool row_unit(uint64_t units, uint64_t& unit) {
  unit = static_cast<uint64_t>(blockIdx.x) * kRowWarps + (threadIdx.x >> 5);
  return unit < units;
}

template <typename T, int E>
__global__ void __launch_bounds__(kRowWarps * 32) row_forward_kernel(
    const __grid_constant__ WindowParams w) {
  pdl_begin();
  const int lane = threadIdx.x & 31;
  uint64_t unit;
  if (!row_unit(static_cast<uint64_t>(w.batch) * w.heads * w.q_len, unit)) return;
  const int i = static_cast<int>(unit % w.q_len);
  const int bh = static_cast<int>(unit / w.q_len), b = bh / w.heads, h = bh - b * w.heads;
  const int kh = h / w.group;
  const Sequence s = sequence_of(w, b);
  const int p = s.p0 + i;
  float q[E], acc[E];
  load_row<T, E>(q, row_ptr<T>(w.q, b, i, h), w.head_dim, lane);
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  float top = -INFINITY, sum = 0.f;
  if (p >= 0 && p < s.n) {
    const int near = max(0, p - w.window + 1);
    for (int j = min(near, w.sinks) > 0 ? 0 : near; j <= p; ++j) {
      if (j >= w.sinks && j < near) j = near;
      float k[E], v[E];
      load_row<T, E>(k, row_ptr<T>(w.k, b, j, kh), w.head_dim, lane);
      load_row<T, E>(v, row_ptr<T>(w.v, b, j, kh), w.head_dim, lane);
      const float x = dot_row<E>(q, k) * w.scale;
      if (x > top) {
        const float f = expf(top - x);  // (0 for the first key)
        sum *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= f;
        top = x;
      }
      const float pr = expf(x - (top == -INFINITY ? 0.f : top));
      sum += pr;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += pr * v[e];
    }
  }
  const bool empty = p < 0 || p >= s.n;
  T* o = row_out<T>(w.out, b, i, h);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + 32 * e < w.head_dim) put(o + lane + 32 * e, empty ? 0.f : acc[e] / sum);
  if (lane == 0 && w.lse) w.lse[unit] = empty ? -INFINITY : top + logf(sum);
}

// dq of one row, and its D for the key kernel.
template <typename T, int E>
__global__ void __launch_bounds__(kRowWarps * 32) row_backward_q_kernel(
    const __grid_constant__ WindowParams w) {
  pdl_begin();
  const int lane = threadIdx.x & 31;
  uint64_t unit;
  if (!row_unit(static_cast<uint64_t>(w.batch) * w.heads * w.q_len, unit)) return;
  const int i = static_cast<int>(unit % w.q_len);
  const int bh = static_cast<int>(unit / w.q_len), b = bh / w.heads, h = bh - b * w.heads;
  const int kh = h / w.group;
  const Sequence s = sequence_of(w, b);
  const int p = s.p0 + i;
  float acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (p >= 0 && p < s.n) {
    float q[E], o[E], g[E];
    load_row<T, E>(q, row_ptr<T>(w.q, b, i, h), w.head_dim, lane);
    load_row<T, E>(g, row_ptr<T>(w.dout, b, i, h), w.head_dim, lane);
    load_row<T, E>(o, row_ptr<T>(w.out, b, i, h), w.head_dim, lane);
    const float delta = dot_row<E>(g, o), lse = w.lse[unit];
    if (lane == 0) w.delta[unit] = delta;
    const int near = max(0, p - w.window + 1);
    for (int j = min(near, w.sinks) > 0 ? 0 : near; j <= p; ++j) {
      if (j >= w.sinks && j < near) j = near;
      float k[E], v[E];
      load_row<T, E>(k, row_ptr<T>(w.k, b, j, kh), w.head_dim, lane);
      load_row<T, E>(v, row_ptr<T>(w.v, b, j, kh), w.head_dim, lane);
      const float pr = expf(dot_row<E>(q, k) * w.scale - lse);
      const float ds = pr * (dot_row<E>(g, v) - delta) * w.scale;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += ds * k[e];
    }
  }
  T* o = row_out<T>(w.dq, b, i, h);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + 32 * e < w.head_dim) put(o + lane + 32 * e, acc[e]);
}

// dk, dv of one key: every row of the head group that sees it, heads then rows in order.
template <typename T, int E>
__global__ void __launch_bounds__(kRowWarps * 32) row_backward_kv_kernel(
    const __grid_constant__ WindowParams w) {
  pdl_begin();
  const int lane = threadIdx.x & 31;
  uint64_t unit;
  if (!row_unit(static_cast<uint64_t>(w.batch) * w.kv_heads * w.kv_len, unit)) return;
  const int j = static_cast<int>(unit % w.kv_len);
  const int bh = static_cast<int>(unit / w.kv_len), b = bh / w.kv_heads, kh = bh - b * w.kv_heads;
  const Sequence s = sequence_of(w, b);
  float dk[E], dv[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dk[e] = dv[e] = 0.f;
  if (j < s.n) {
    float k[E], v[E];
    load_row<T, E>(k, row_ptr<T>(w.k, b, j, kh), w.head_dim, lane);
    load_row<T, E>(v, row_ptr<T>(w.v, b, j, kh), w.head_dim, lane);
    // rows of positions j .. min(n, j + window) - 1, or j .. n - 1 for a first token
    const int64_t end = j < w.sinks ? s.n : min(static_cast<int64_t>(s.n), static_cast<int64_t>(j) + w.window);
    const int lo = max(0, j - s.p0);
    const int hi = static_cast<int>(min(static_cast<int64_t>(w.q_len), end - s.p0));
    for (int h = kh * w.group; h < (kh + 1) * w.group; ++h) {
      const uint64_t base = (static_cast<uint64_t>(b) * w.heads + h) * w.q_len;
      for (int i = lo; i < hi; ++i) {
        float q[E], g[E];
        load_row<T, E>(q, row_ptr<T>(w.q, b, i, h), w.head_dim, lane);
        load_row<T, E>(g, row_ptr<T>(w.dout, b, i, h), w.head_dim, lane);
        const float pr = expf(dot_row<E>(q, k) * w.scale - w.lse[base + i]);
        const float ds = pr * (dot_row<E>(g, v) - w.delta[base + i]) * w.scale;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          dv[e] += pr * g[e];
          dk[e] += ds * q[e];
        }
      }
    }
  }
  T* ok = row_out<T>(w.dk, b, j, kh);
  T* ov = row_out<T>(w.dv, b, j, kh);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + 32 * e < w.head_dim) {
      put(ok + lane + 32 * e, dk[e]);
      put(ov + lane + 32 * e, dv[e]);
    }
}

// ------------------------------------------------------------------------------- host side
// Strides over a single index never count, so that they cannot spoil an alignment rule.
View view_of(const SparB200Heads& v, uint64_t batch, uint64_t tokens, uint64_t heads) {
  return {static_cast<char*>(v.data), batch > 1 ? v.batch : 0, tokens > 1 ? v.token : 0,
          heads > 1 ? v.head : 0};
}

bool whole_words(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// An output whose rows lie on one another (a stride of zero) would be written by many at once.
bool shared_rows(const View& v, uint64_t batch, uint64_t tokens, uint64_t heads) {
  return (batch > 1 && !v.batch) || (tokens > 1 && !v.token) || (heads > 1 && !v.head);
}

bool whole_elements(const SparB200Heads& v, int dtype) {
  return v.data && reinterpret_cast<uintptr_t>(v.data) % (dtype == SPAR_B200_FLOAT32 ? 4 : 2) == 0;
}

bool valid_sizes(const SparB200WindowAttention* a) {
  if (!a) return false;
  if (a->dtype != SPAR_B200_FLOAT32 && a->dtype != SPAR_B200_BFLOAT16) return false;
  const uint64_t most = static_cast<uint64_t>(kMaxLength);
  if (a->q_len >= most || a->kv_len >= most || a->batch >= most || a->heads < 1 ||
      a->heads >= most || a->kv_heads < 1 || a->kv_heads > a->heads || a->heads % a->kv_heads)
    return false;
  if (a->head_dim < 1 || a->head_dim > kMaxHeadDim || a->window < 1) return false;
  if (a->scale != 0.0 && !(a->scale >= 1e-30 && a->scale <= 1e30)) return false;
  // rows and keys of all heads are numbered in 32 bits of warps and blocks
  if (a->batch * a->heads >= (1ull << 31)) return false;
  const uint64_t longest = a->q_len > a->kv_len ? a->q_len : a->kv_len;
  return longest == 0 || a->batch * a->heads <= ((1ull << 32) / longest);
}

bool make_params(const SparB200WindowAttention* a, bool backward, WindowParams& w) {
  if (!valid_sizes(a)) return false;
  const bool rows = a->batch && a->q_len, keys = a->batch && a->kv_len;
  if (rows && (!whole_elements(a->q, a->dtype) || !whole_elements(a->out, a->dtype))) return false;
  if (keys && (!whole_elements(a->k, a->dtype) || !whole_elements(a->v, a->dtype))) return false;
  if (backward) {
    if (rows && (!whole_elements(a->dout, a->dtype) || !whole_elements(a->dq, a->dtype) || !a->lse))
      return false;
    if (keys && (!whole_elements(a->dk, a->dtype) || !whole_elements(a->dv, a->dtype))) return false;
  }
  w = WindowParams{};
  w.q = view_of(a->q, a->batch, a->q_len, a->heads);
  w.k = view_of(a->k, a->batch, a->kv_len, a->kv_heads);
  w.v = view_of(a->v, a->batch, a->kv_len, a->kv_heads);
  w.out = view_of(a->out, a->batch, a->q_len, a->heads);
  w.dout = view_of(a->dout, a->batch, a->q_len, a->heads);
  w.dq = view_of(a->dq, a->batch, a->q_len, a->heads);
  w.dk = view_of(a->dk, a->batch, a->kv_len, a->kv_heads);
  w.dv = view_of(a->dv, a->batch, a->kv_len, a->kv_heads);
  if (rows && (shared_rows(w.out, a->batch, a->q_len, a->heads) ||
               (backward && shared_rows(w.dq, a->batch, a->q_len, a->heads))))
    return false;
  if (keys && backward && (shared_rows(w.dk, a->batch, a->kv_len, a->kv_heads) ||
                           shared_rows(w.dv, a->batch, a->kv_len, a->kv_heads)))
    return false;
  if (!whole_words(a->lse) || !whole_words(a->lengths) || !whole_words(a->first)) return false;
  // Outputs are written while other rows' inputs are still read (other overlaps are the caller's to
  // avoid: views of one packed buffer interleave).
  const char* in[5] = {rows ? w.q.data : nullptr, keys ? w.k.data : nullptr, keys ? w.v.data : nullptr,
                       backward && rows ? w.dout.data : nullptr, backward && rows ? w.out.data : nullptr};
  const char* out[3] = {rows ? (backward ? w.dq.data : w.out.data) : nullptr,
                        backward && keys ? w.dk.data : nullptr, backward && keys ? w.dv.data : nullptr};
  for (int i = 0; i < 3; ++i) {
    for (const char* p : in)
      if (out[i] && out[i] == p) return false;
    for (int j = 0; j < i; ++j)
      if (out[i] && out[i] == out[j]) return false;
  }
  w.lse = a->lse;
  w.lengths = a->lengths;
  w.first = a->first;
  w.batch = static_cast<int>(a->batch);
  w.q_len = static_cast<int>(a->q_len);
  w.kv_len = static_cast<int>(a->kv_len);
  w.heads = static_cast<int>(a->heads);
  w.kv_heads = static_cast<int>(a->kv_heads);
  w.group = w.heads / w.kv_heads;
  w.head_dim = static_cast<int>(a->head_dim);
  w.window = static_cast<int>(a->window < static_cast<uint64_t>(kMaxLength) ? a->window : kMaxLength);
  w.sinks = static_cast<int>(a->sinks < a->kv_len ? a->sinks : a->kv_len);
  w.dtype = a->dtype;
  w.scale = static_cast<float>(
      a->scale > 0.0 ? a->scale : 1.0 / std::sqrt(static_cast<double>(a->head_dim)));
  return true;
}

uint64_t round256(uint64_t bytes) { return (bytes + 255) & ~255ull; }

unsigned row_blocks(uint64_t units) {
  return static_cast<unsigned>((units + kRowWarps - 1) / kRowWarps);
}

template <typename T, int E>
cudaError_t row_forward(const WindowParams& w, cudaStream_t stream) {
  return launch(row_forward_kernel<T, E>,
                dim3(row_blocks(static_cast<uint64_t>(w.batch) * w.heads * w.q_len)),
                dim3(kRowWarps * 32), 0, stream, w);
}
template <typename T, int E>
cudaError_t row_backward(const WindowParams& w, cudaStream_t stream) {
  const uint64_t rows = static_cast<uint64_t>(w.batch) * w.heads * w.q_len;
  const uint64_t keys = static_cast<uint64_t>(w.batch) * w.kv_heads * w.kv_len;
  if (rows) {
    const cudaError_t e = launch(row_backward_q_kernel<T, E>, dim3(row_blocks(rows)),
                                 dim3(kRowWarps * 32), 0, stream, w);
    if (e != cudaSuccess) return e;
  }
  if (!keys) return cudaSuccess;
  return launch(row_backward_kv_kernel<T, E>, dim3(row_blocks(keys)), dim3(kRowWarps * 32), 0,
                stream, w);
}

template <typename T>
cudaError_t row_path(const WindowParams& w, bool backward, cudaStream_t stream) {
  if (w.head_dim <= 32) return backward ? row_backward<T, 1>(w, stream) : row_forward<T, 1>(w, stream);
  if (w.head_dim <= 64) return backward ? row_backward<T, 2>(w, stream) : row_forward<T, 2>(w, stream);
  if (w.head_dim <= 128) return backward ? row_backward<T, 4>(w, stream) : row_forward<T, 4>(w, stream);
  return backward ? row_backward<T, 8>(w, stream) : row_forward<T, 8>(w, stream);
}

}  // namespace
}  // namespace window
}  // namespace spar_b200

using namespace spar_b200;
using namespace spar_b200::window;

namespace {

// What a call will run, decided from its sizes, types and strides alone, so that the scratch it is
// asked for and the launch agree.
struct Plan {
  bool few, tiled;
  uint64_t delta_bytes, bytes;
};
Plan plan_of(const WindowParams& w, bool backward, int device) {
  Plan p;
  p.few = !backward && decode_supported(w);
  p.tiled = !p.few && tc_supported(w, backward);
  p.delta_bytes =
      backward ? round256(static_cast<uint64_t>(w.batch) * w.heads * w.q_len * sizeof(float)) : 0;
  p.bytes = p.delta_bytes + (p.few     ? decode_scratch_bytes(w, device)
                             : p.tiled ? tc_scratch_bytes(w, backward, device)
                                       : 0);
  return p;
}

}  // namespace

extern "C" uint64_t spar_b200_window_attention_scratch_bytes(const SparB200WindowAttention* a,
                                                             int backward, int device) {
  WindowParams w;
  if (!make_params(a, backward != 0, w) || !w.batch) return 0;
  return plan_of(w, backward != 0, device).bytes;
}

extern "C" SparCudaStatus spar_b200_window_attention_forward(const SparB200WindowAttention* a,
                                                             int device, void* stream) {
  WindowParams w;
  if (!make_params(a, false, w)) return invalid();
  if (!w.batch || !w.q_len) return ok();
  const Plan plan = plan_of(w, false, device);
  if (plan.bytes && (!a->scratch || (reinterpret_cast<uintptr_t>(a->scratch) & 255))) return invalid();
  DeviceScope scope(device);
  if (scope.error() != cudaSuccess) return runtime(scope.error());
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (plan.few)
    e = decode_forward(w, a->scratch, device, s);
  else if (plan.tiled)
    e = tc_forward(w, a->scratch, device, s);
  else
    e = w.dtype == SPAR_B200_FLOAT32 ? row_path<float>(w, false, s)
                                     : row_path<__nv_bfloat16>(w, false, s);
  return e == cudaSuccess ? launch_status() : runtime(e);
}

extern "C" SparCudaStatus spar_b200_window_attention_backward(const SparB200WindowAttention* a,
                                                              int device, void* stream) {
  WindowParams w;
  if (!make_params(a, true, w)) return invalid();
  if (!w.batch || (!w.q_len && !w.kv_len)) return ok();
  const Plan plan = plan_of(w, true, device);
  if (plan.bytes && (!a->scratch || (reinterpret_cast<uintptr_t>(a->scratch) & 255))) return invalid();
  w.delta = static_cast<float*>(a->scratch);
  DeviceScope scope(device);
  if (scope.error() != cudaSuccess) return runtime(scope.error());
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (plan.tiled)
    e = tc_backward(w, static_cast<char*>(a->scratch) + plan.delta_bytes, device, s);
  else
    e = w.dtype == SPAR_B200_FLOAT32 ? row_path<float>(w, true, s)
                                     : row_path<__nv_bfloat16>(w, true, s);
  return e == cudaSuccess ? launch_status() : runtime(e);
}
