// What the window-attention kernels share: one call's tensors and sizes, and what of them one
// sequence of the batch uses.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace spar_b200 {
namespace window {

constexpr int64_t kMaxLength = 1ll << 29;  // so that sums of two positions stay in 32 bits
constexpr uint64_t kMaxHeadDim = 256;

// A strided view of heads: element (b, t, h, e) at data + b*batch + t*token + h*head + e.
struct View {
  char* data;
  uint64_t batch, token, head;  // strides in elements
};

struct WindowParams {
  View q, k, v, out, dout, dq, dk, dv;
  float* lse;
  float* delta;  // [batch, heads, q_len] D
  const int32_t* lengths;
  const int32_t* first;
  int q_len, kv_len, heads, kv_heads, group, head_dim;
  int window, sinks;
  int batch;
  int dtype;
  float scale;
};

// What of one sequence of the batch the call's rows can see: its first n keys, which end with its length
// or with the last row's position (a cache's slots behind them may hold anything), and the position of
// its first row.
struct Sequence {
  int n, p0;
};
__device__ __forceinline__ Sequence sequence_of(const WindowParams& w, int b) {
  Sequence s;
  s.n = w.lengths ? min(max(__ldg(w.lengths + b), 0), w.kv_len) : w.kv_len;
  // Positions beyond +-2^29 see nothing, as every position at or behind the length does.
  const int far = 1 << 29;
  s.p0 = w.first ? min(max(__ldg(w.first + b), -far), far) : w.kv_len - w.q_len;
  s.n = min(s.n, max(s.p0 + w.q_len, 0));
  return s;
}

template <typename T>
__device__ __forceinline__ const T* row_ptr(const View& v, int b, int t, int h) {
  return reinterpret_cast<const T*>(v.data) + b * v.batch + t * v.token + h * v.head;
}
template <typename T>
__device__ __forceinline__ T* row_out(const View& v, int b, int t, int h) {
  return reinterpret_cast<T*>(v.data) + b * v.batch + t * v.token + h * v.head;
}
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// A view that TMA and 16-byte accesses can address: 16-byte rows, no broadcast dimension.
inline bool tiled_view(const View& v, int size, uint64_t batch, uint64_t tokens, uint64_t heads) {
  const uint64_t n = 16 / size;
  const uint64_t extent[3] = {batch, tokens, heads}, stride[3] = {v.batch, v.token, v.head};
  if (reinterpret_cast<uintptr_t>(v.data) & 15) return false;
  for (int i = 0; i < 3; ++i)
    if (extent[i] > 1 && (stride[i] % n || stride[i] == 0 || stride[i] * size >= (1ull << 40)))
      return false;
  return true;
}

// A few rows against a cache (window_decode.cu).
bool decode_supported(const WindowParams& w);
uint64_t decode_scratch_bytes(const WindowParams& w, int device);
cudaError_t decode_forward(const WindowParams& w, void* scratch, int device, cudaStream_t stream);

// Tensor-core path (window_tc.cu): whether it takes this call, its scratch, and the launches.
bool tc_supported(const WindowParams& w, bool backward);
uint64_t tc_scratch_bytes(const WindowParams& w, bool backward, int device);
cudaError_t tc_forward(const WindowParams& w, void* scratch, int device, cudaStream_t stream);
cudaError_t tc_backward(const WindowParams& w, void* scratch, int device, cudaStream_t stream);

}  // namespace window
}  // namespace spar_b200
