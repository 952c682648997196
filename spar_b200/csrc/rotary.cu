// Rotary positions (interleaved and half layouts, part of the head, scaled angle tables) and the
// per-head RMSNorm of queries and keys with the rotation in the same pass, forward and backward.
//
// Rotation of pair (a, b) at angle t: (a cos t - b sin t, b cos t + a sin t); turning back is the
// same with -sin, and is the rotation's backward pass.
// qk-norm (reference src/nn/attention.cpp:183-186, 208-215; src/nn/rmsnorm.cpp:50-52):
//   y = rotate(x r w), r = 1 / sqrt(mean(x^2) + eps) over the head.
//   g = rotate_back(dy);  dx = r (g w - x r mean(g w x r));  dw = sum over tokens, heads of g x r.
// All of them stream: x in, y out (backward: x and dy in, dx out) and the angle rows, which all
// heads of a token share. The floor is those bytes at the copy bandwidth.
//
// Layout: a head is split into vectors of 16 bytes (VEC elements; VEC = 1 for rows that are not
// aligned to 16 bytes). A slot is two vectors of one head that one lane holds: vectors v and
// v + half of the rotated part, so that both layouts' partners meet in one lane (half layout: the
// same element of both vectors; interleaved: neighbours inside each), then pairs of vectors of
// the part that passes. Heads take a power-of-two group of lanes, sums over a head are shuffles
// inside the group, and nothing but weight gradients leaves a warp.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "kernels.cuh"

namespace spar_b200 {
namespace {

constexpr uint64_t kMaxUnits = 1ull << 31;
constexpr int kBackwardThreads = 128;

// Exact quotient by a fixed divisor for dividends below 2^31: with 2^(s-1) < d <= 2^s and
// m = ceil(2^(31+s) / d) < 2^32, floor(n m / 2^(31+s)) = floor(n / d) since n (m d - 2^(31+s)) <
// 2^31 d <= 2^(31+s) (Granlund and Montgomery 1994).
struct Divider {
  uint32_t d, m, s;
  Divider() : d(1), m(0), s(0) {}
  explicit Divider(uint32_t divisor) : d(divisor), m(0), s(0) {
    while ((1ull << s) < d) ++s;
    m = static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> (31 + s));
  }
};

struct View {
  char* data;
  uint64_t batch, token, head;  // strides in elements
};

struct RotaryParams {
  View in[2], out[2], grad[2];  // queries, keys
  const float* weight[2];
  const float2* table;
  const int32_t* positions;
  int32_t* invalid;
  float* partial;
  uint64_t start, table_rows;
  uint32_t heads[2], chunks[2];  // heads, and groups of HP heads
  uint32_t tokens, seq, head_dim, pairs, slots, rotating;
  uint32_t lanes_log2;
  uint32_t blocks_q;  // backward: blocks below this index take queries, the others keys
  Divider by_seq, by_chunks, by_heads[2];
  float sine, eps, inv_dim;
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// VEC elements as loaded: one 16-byte access, or one element.
template <typename T, int VEC>
struct Raw {
  T e[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load_raw(const T* p) {
  Raw<T, VEC> r;
  if constexpr (VEC * sizeof(T) == 16) {
    const float4 f = __ldcs(reinterpret_cast<const float4*>(p));
    memcpy(&r, &f, 16);
  } else {
    r.e[0] = *p;
  }
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  Raw<T, VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r.e[i] = from_float<T>(v[i]);
  if constexpr (VEC * sizeof(T) == 16) {
    float4 f;
    memcpy(&f, &r, 16);
    *reinterpret_cast<float4*>(p) = f;
  } else {
    *p = r.e[0];
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void widen(const Raw<T, VEC>& r, float (&v)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] = to_float(r.e[i]);
}

// Where a slot's two vectors start in the head; b may not exist (the odd vector of the part that
// passes). `pair` is the first pair of vector a; of vector b in the interleaved layout.
struct Slot {
  uint32_t a, b, pair_a, pair_b;
  bool has_a, has_b, turns;
};

// FULL: the whole head turns and every lane of the group has a slot, the usual case, which then
// carries none of the tests.
template <int VEC, bool HALF, bool FULL>
__device__ __forceinline__ Slot slot_of(const RotaryParams& p, uint32_t s) {
  Slot o;
  o.has_a = FULL || s < p.slots;
  o.turns = FULL || s < p.rotating;
  if (o.turns) {
    if (HALF || VEC > 1) {  // vectors s and s + half of the rotated part
      o.a = s * VEC;
      o.b = s * VEC + p.pairs;
    } else {  // interleaved single elements
      o.a = 2 * s;
      o.b = 2 * s + 1;
    }
    o.has_b = true;
    o.pair_a = HALF || VEC == 1 ? s * VEC : s * (VEC / 2);
    o.pair_b = o.pair_a + p.pairs / 2;
  } else {
    // vectors v and v + (their number of slots) of the part that passes, so that neighbouring
    // lanes' accesses are neighbours
    o.a = 2 * p.pairs + (s - p.rotating) * VEC;
    o.b = o.a + (p.slots - p.rotating) * VEC;
    o.has_b = o.b < p.head_dim;
    o.pair_a = o.pair_b = 0;
  }
  return o;
}

// cos and sin of a slot: pair x of `cs` (half: element x of both vectors; interleaved: pairs
// 0 .. VEC/2 - 1 of vector a, then those of vector b).
template <int VEC, bool HALF>
__device__ __forceinline__ void load_angles(const RotaryParams& p, const Slot& s, uint64_t row,
                                            float2 (&cs)[VEC]) {
  const float2* t = p.table + row * p.pairs;
  if constexpr (VEC == 1) {
    cs[0] = __ldg(t + s.pair_a);
  } else {
#pragma unroll
    for (int x = 0; x < VEC; x += 2) {
      const uint32_t at = HALF || x < VEC / 2 ? s.pair_a + x : s.pair_b + x - VEC / 2;
      const float4 f = __ldg(reinterpret_cast<const float4*>(t + at));
      cs[x] = make_float2(f.x, f.y);
      cs[x + 1] = make_float2(f.z, f.w);
    }
  }
#pragma unroll
  for (int x = 0; x < VEC; ++x) cs[x].y *= p.sine;
}

template <int VEC, bool HALF>
__device__ __forceinline__ void turn(float (&a)[VEC], float (&b)[VEC], const float2 (&cs)[VEC],
                                     float sign) {
  if constexpr (HALF || VEC == 1) {
#pragma unroll
    for (int x = 0; x < VEC; ++x) {
      const float c = cs[x].x, s = cs[x].y * sign, u = a[x], w = b[x];
      a[x] = u * c - w * s;
      b[x] = w * c + u * s;
    }
  } else {
#pragma unroll
    for (int x = 0; x < VEC / 2; ++x) {
      float c = cs[x].x, s = cs[x].y * sign, u = a[2 * x], w = a[2 * x + 1];
      a[2 * x] = u * c - w * s;
      a[2 * x + 1] = w * c + u * s;
      c = cs[VEC / 2 + x].x, s = cs[VEC / 2 + x].y * sign, u = b[2 * x], w = b[2 * x + 1];
      b[2 * x] = u * c - w * s;
      b[2 * x + 1] = w * c + u * s;
    }
  }
}

// The table row of token t, or false when its position lies outside the table.
__device__ __forceinline__ bool row_of(const RotaryParams& p, uint32_t t, uint32_t in_seq,
                                       uint64_t& row) {
  if (p.positions) {
    const int32_t at = __ldg(p.positions + t);
    row = static_cast<uint64_t>(static_cast<int64_t>(at));  // negative: above every row count
  } else {
    row = p.start + in_seq;
  }
  return row < p.table_rows;
}

template <int VEC>
__device__ __forceinline__ void load_weights(const float* w, const Slot& s, float (&wa)[VEC],
                                             float (&wb)[VEC]) {
  const bool a = s.has_a, b = s.has_a && s.has_b;
  if constexpr (VEC == 1) {
    wa[0] = a ? __ldg(w + s.a) : 0.f;
    wb[0] = b ? __ldg(w + s.b) : 0.f;
  } else {
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < VEC; x += 4) {
      const float4 u = a ? __ldg(reinterpret_cast<const float4*>(w + s.a + x)) : none;
      const float4 v = b ? __ldg(reinterpret_cast<const float4*>(w + s.b + x)) : none;
      wa[x] = u.x, wa[x + 1] = u.y, wa[x + 2] = u.z, wa[x + 3] = u.w;
      wb[x] = v.x, wb[x + 1] = v.y, wb[x + 2] = v.z, wb[x + 3] = v.w;
    }
  }
}

__device__ __forceinline__ float group_sum(float v, uint32_t lanes) {
  for (uint32_t o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One lane group per (token, HP heads of queries or of keys): the heads of a chunk share the
// token's angles in registers and put 2 HP vectors in flight per lane before the first is used.
// U slots per lane (one but for unaligned rows).
// (Four blocks an SM where two heads of a group still leave the registers: 116 -> 108 us for the
// gradients of 3 x 8191 tokens of 40 heads of 128 bf16, half of each turned.)
template <typename T, int VEC, int U, int HP, bool HALF, bool NORM, bool FULL>
__global__ void __launch_bounds__(256, HP == 2 ? 4 : 1) rotary_kernel(const __grid_constant__ RotaryParams p) {
  pdl_begin();
  const uint32_t lanes = 1u << p.lanes_log2;
  const uint32_t l = threadIdx.x & (lanes - 1);
  const uint32_t all = p.chunks[0] + p.chunks[1];
  const uint32_t unit = static_cast<uint32_t>(
      (static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> p.lanes_log2);
  const bool live = unit < p.tokens * static_cast<uint64_t>(all);
  const uint32_t t = live ? p.by_chunks.quotient(unit) : 0;
  uint32_t chunk = live ? unit - t * all : 0;
  const int side = chunk >= p.chunks[0];
  if (side) chunk -= p.chunks[0];
  const uint32_t h0 = chunk * HP;
  const uint32_t n = live ? min(static_cast<uint32_t>(HP), p.heads[side] - h0) : 0;
  const uint32_t b = p.by_seq.quotient(t), in_seq = t - b * p.seq;
  const View& in = p.in[side];
  const View& out = p.out[side];
  const T* src = reinterpret_cast<const T*>(in.data) + b * in.batch + in_seq * in.token +
                 h0 * in.head;
  T* dst = reinterpret_cast<T*>(out.data) + b * out.batch + in_seq * out.token + h0 * out.head;
  uint64_t row = 0;
  const bool good = row_of(p, t, in_seq, row);  // under way; not looked at before the heads are too

  Raw<T, VEC> ra[U][HP], rb[U][HP];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Slot s = slot_of<VEC, HALF, FULL>(p, l + u * lanes);
#pragma unroll
    for (int h = 0; h < HP; ++h) {
      if (static_cast<uint32_t>(h) < n && s.has_a) {
        ra[u][h] = load_raw<T, VEC>(src + h * in.head + s.a);
        if (s.has_b) rb[u][h] = load_raw<T, VEC>(src + h * in.head + s.b);
      }
    }
  }
  if (!good && live && l == 0 && chunk == 0 && p.invalid) atomicExch(p.invalid, 1);
  float r[HP];
  if constexpr (NORM) {
#pragma unroll
    for (int h = 0; h < HP; ++h) {
      float ss = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Slot s = slot_of<VEC, HALF, FULL>(p, l + u * lanes);
        if (static_cast<uint32_t>(h) < n && s.has_a) {
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            const float v = to_float(ra[u][h].e[x]);
            ss += v * v;
          }
          if (s.has_b) {
#pragma unroll
            for (int x = 0; x < VEC; ++x) {
              const float v = to_float(rb[u][h].e[x]);
              ss += v * v;
            }
          }
        }
      }
      r[h] = rsqrtf(group_sum(ss, lanes) * p.inv_dim + p.eps);  // within two steps of fp32
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Slot s = slot_of<VEC, HALF, FULL>(p, l + u * lanes);
    if (!s.has_a || !n) continue;
    float2 cs[VEC];
    float wa[VEC], wb[VEC];
    if (s.turns && good) load_angles<VEC, HALF>(p, s, row, cs);
    if constexpr (NORM) load_weights<VEC>(p.weight[side], s, wa, wb);
#pragma unroll
    for (int h = 0; h < HP; ++h) {
      if (static_cast<uint32_t>(h) >= n) continue;
      float a[VEC], c[VEC];
      widen<T, VEC>(ra[u][h], a);
      if (s.has_b) widen<T, VEC>(rb[u][h], c);
      if constexpr (NORM) {
#pragma unroll
        for (int x = 0; x < VEC; ++x) {
          a[x] *= r[h] * wa[x];
          if (s.has_b) c[x] *= r[h] * wb[x];
        }
      }
      if (!good) {
#pragma unroll
        for (int x = 0; x < VEC; ++x) a[x] = c[x] = 0.f;
      } else if (s.turns) {
        turn<VEC, HALF>(a, c, cs, 1.f);
      }
      store_vec<T, VEC>(dst + h * out.head + s.a, a);
      if (s.has_b) store_vec<T, VEC>(dst + h * out.head + s.b, c);
    }
  }
}

// Backward of the norm and the rotation. Blocks are split between queries and keys in proportion
// to their heads and walk their (token, HB heads) units with the grid's stride, so a lane keeps the
// sums of its slots' weight gradients in registers for the whole launch; a block adds its lane
// groups' sums in a fixed order and leaves one partial row of head_dim floats. The heads of a unit
// share the token's angles and addresses, and put 4 HB vectors in flight per lane.
template <typename T, int VEC, int U, int HB, bool HALF, bool FULL>
__global__ void __launch_bounds__(kBackwardThreads) qk_norm_rotary_backward_kernel(
    const __grid_constant__ RotaryParams p) {
  pdl_begin();
  extern __shared__ float sums[];  // [groups of the block][head_dim]
  const uint32_t lanes = 1u << p.lanes_log2;
  const uint32_t l = threadIdx.x & (lanes - 1), group = threadIdx.x >> p.lanes_log2;
  const uint32_t groups = blockDim.x >> p.lanes_log2;
  const int side = blockIdx.x >= p.blocks_q;
  const uint32_t block = side ? blockIdx.x - p.blocks_q : blockIdx.x;
  const uint32_t blocks = side ? gridDim.x - p.blocks_q : p.blocks_q;
  const uint32_t heads = p.heads[side], chunks = p.chunks[side];
  const uint64_t units = static_cast<uint64_t>(p.tokens) * chunks;
  const View &in = p.in[side], &out = p.out[side], &grad = p.grad[side];
  float wa[U][VEC], wb[U][VEC], da[U][VEC], db[U][VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    load_weights<VEC>(p.weight[side], slot_of<VEC, HALF, FULL>(p, l + u * lanes), wa[u], wb[u]);
#pragma unroll
    for (int x = 0; x < VEC; ++x) da[u][x] = db[u][x] = 0.f;
  }
  for (uint64_t first = static_cast<uint64_t>(block) * groups; first < units;
       first += static_cast<uint64_t>(blocks) * groups) {  // every lane: the sums are whole-warp
    const uint64_t unit = first + group;
    const bool live = unit < units;
    const uint32_t t = live ? p.by_heads[side].quotient(static_cast<uint32_t>(unit)) : 0;
    const uint32_t h0 = live ? (static_cast<uint32_t>(unit) - t * chunks) * HB : 0;
    const uint32_t n = live ? min(static_cast<uint32_t>(HB), heads - h0) : 0;
    const uint32_t b = p.by_seq.quotient(t), in_seq = t - b * p.seq;
    uint64_t row = 0;
    const bool good = row_of(p, t, in_seq, row);
    const T* px = reinterpret_cast<const T*>(in.data) + b * in.batch + in_seq * in.token + h0 * in.head;
    const T* pg =
        reinterpret_cast<const T*>(grad.data) + b * grad.batch + in_seq * grad.token + h0 * grad.head;
    T* po = reinterpret_cast<T*>(out.data) + b * out.batch + in_seq * out.token + h0 * out.head;
    Raw<T, VEC> rxa[HB][U], rxb[HB][U], rga[HB][U], rgb[HB][U];
#pragma unroll
    for (int h = 0; h < HB; ++h)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Slot s = slot_of<VEC, HALF, FULL>(p, l + u * lanes);
        rxa[h][u] = rxb[h][u] = rga[h][u] = rgb[h][u] = Raw<T, VEC>{};
        if (static_cast<uint32_t>(h) >= n || !s.has_a) continue;
        rxa[h][u] = load_raw<T, VEC>(px + h * in.head + s.a);
        rga[h][u] = load_raw<T, VEC>(pg + h * grad.head + s.a);
        if (s.has_b) {
          rxb[h][u] = load_raw<T, VEC>(px + h * in.head + s.b);
          rgb[h][u] = load_raw<T, VEC>(pg + h * grad.head + s.b);
        }
      }
    if (!good && live && l == 0 && h0 == 0 && p.invalid) atomicExch(p.invalid, 1);
    float2 cs[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Slot s = slot_of<VEC, HALF, FULL>(p, l + u * lanes);
      if (s.turns) load_angles<VEC, HALF>(p, s, good ? row : 0, cs[u]);  // (the host sees to a row 0)
    }
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      float xa[U][VEC], xb[U][VEC], ga[U][VEC], gb[U][VEC];
      float ss = 0.f, dot = 0.f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Slot s = slot_of<VEC, HALF, FULL>(p, l + u * lanes);
        widen<T, VEC>(rxa[h][u], xa[u]);
        widen<T, VEC>(rxb[h][u], xb[u]);
        widen<T, VEC>(rga[h][u], ga[u]);
        widen<T, VEC>(rgb[h][u], gb[u]);
        if (s.turns) turn<VEC, HALF>(ga[u], gb[u], cs[u], -1.f);  // (unused where the position is not good)
#pragma unroll
        for (int x = 0; x < VEC; ++x) {
          ss += xa[u][x] * xa[u][x] + xb[u][x] * xb[u][x];
          dot += ga[u][x] * wa[u][x] * xa[u][x] + gb[u][x] * wb[u][x] * xb[u][x];
        }
      }
      for (uint32_t o = lanes >> 1; o > 0; o >>= 1) {
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
      const float r = rsqrtf(ss * p.inv_dim + p.eps);  // within two steps of fp32
      const float m = dot * r * p.inv_dim;             // mean(g w x r)
      if (static_cast<uint32_t>(h) >= n) continue;
      if (!good) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const Slot s = slot_of<VEC, HALF, FULL>(p, l + u * lanes);
          const float zero[VEC] = {};
          if (s.has_a) store_vec<T, VEC>(po + h * out.head + s.a, zero);
          if (s.has_a && s.has_b) store_vec<T, VEC>(po + h * out.head + s.b, zero);
        }
        continue;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Slot s = slot_of<VEC, HALF, FULL>(p, l + u * lanes);
        if (!s.has_a) continue;
        float oa[VEC], ob[VEC];
#pragma unroll
        for (int x = 0; x < VEC; ++x) {
          const float ua = xa[u][x] * r, ub = xb[u][x] * r;
          oa[x] = r * (ga[u][x] * wa[u][x] - ua * m);
          ob[x] = r * (gb[u][x] * wb[u][x] - ub * m);
          da[u][x] += ga[u][x] * ua;
          db[u][x] += gb[u][x] * ub;
        }
        store_vec<T, VEC>(po + h * out.head + s.a, oa);
        if (s.has_b) store_vec<T, VEC>(po + h * out.head + s.b, ob);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const Slot s = slot_of<VEC, HALF, FULL>(p, l + u * lanes);
    if (!s.has_a) continue;
#pragma unroll
    for (int x = 0; x < VEC; ++x) {
      sums[group * p.head_dim + s.a + x] = da[u][x];
      if (s.has_b) sums[group * p.head_dim + s.b + x] = db[u][x];
    }
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < p.head_dim; e += blockDim.x) {
    float v = 0.f;
    for (uint32_t g = 0; g < groups; ++g) v += sums[g * p.head_dim + e];
    p.partial[static_cast<uint64_t>(blockIdx.x) * p.head_dim + e] = v;
  }
}

// dweight[e] (+)= the sum of the partial rows: 32 columns a block, 32 rows of threads over the
// parts, added in a fixed order. blockIdx.y 0: queries (rows below parts_q), 1: keys.
__global__ void __launch_bounds__(1024) qk_weight_partials_kernel(float* dq, float* dk,
                                                                  const float* __restrict__ partial,
                                                                  uint32_t parts_q, uint32_t parts,
                                                                  uint32_t head_dim, int accumulate) {
  pdl_begin();
  __shared__ float red[32][33];
  const uint32_t x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const uint32_t e = blockIdx.x * 32 + x;
  const uint32_t lo = blockIdx.y ? parts_q : 0, hi = blockIdx.y ? parts : parts_q;
  float s = 0.f;
  if (e < head_dim) {
#pragma unroll 8
    for (uint32_t r = lo + y; r < hi; r += 32) s += partial[static_cast<uint64_t>(r) * head_dim + e];
  }
  red[y][x] = s;
  __syncthreads();
  s = warp_sum(red[x][y]);  // column blockIdx.x * 32 + y
  const uint32_t c = blockIdx.x * 32 + y;
  float* d = blockIdx.y ? dk : dq;
  if (x == 0 && c < head_dim && d) d[c] = accumulate ? d[c] + s : s;
}

// One thread per (pair, run of positions): the first angle's cos and sin, then rotations by one
// position in double (each adds ~2^-52, far below the fp32 result's 2^-25): four double operations
// per entry instead of ~100. The run is as long as leaves 32768 threads, 8 to 128 positions: 131072
// positions of 64 pairs take 12.2 us from a graph, of which the stores' floor is 10.2, and 17 as a call with
// a flushed L2: a chain of 128 steps on 256 blocks of 148 SMs. (Runs of 128 left a shorter table's few
// threads with the latency of 128 steps: 4096 positions 21 us a call, in runs of 8 9 us.)
__global__ void __launch_bounds__(256) rotary_table_kernel(float2* table, uint64_t rows,
                                                           uint32_t pairs, uint64_t start, uint32_t length,
                                                           SparB200RotaryScaling sc, double theta) {
  pdl_begin();
  const uint64_t idx = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const uint64_t run = idx / pairs;
  const uint32_t i = static_cast<uint32_t>(idx - run * pairs);
  const uint64_t r0 = run * length;
  if (r0 >= rows) return;
  double f = pow(theta, -static_cast<double>(i) / static_cast<double>(pairs));
  if (sc.kind == SPAR_B200_ROTARY_LINEAR) f /= sc.factor;
  if (sc.kind == SPAR_B200_ROTARY_PARTS) {
    const double turns = sc.original_length * f * 0.15915494309189535;  // 1 / (2 pi)
    const double g =
        fmin(fmax((turns - sc.slow_turns) / (sc.fast_turns - sc.slow_turns), 0.0), 1.0);
    f = f * g + f / sc.factor * (1.0 - g);
  }
  double c, s, dc, ds;
  sincos(static_cast<double>(start + r0) * f, &s, &c);
  sincos(f, &ds, &dc);
  const uint64_t n = min(static_cast<uint64_t>(length), rows - r0);
  float2* out = table + r0 * pairs + i;
  for (uint64_t r = 0; r < n; ++r) {
    out[r * pairs] = make_float2(static_cast<float>(c * sc.magnitude),
                                 static_cast<float>(s * sc.magnitude));
    const double next = c * dc - s * ds;
    s = s * dc + c * ds;
    c = next;
  }
}

// ------------------------------------------------------------------------------- host side
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool on4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Strides over a single index never count, so that they cannot spoil the alignment rule.
View view_of(const SparB200Heads& v, uint64_t batch, uint64_t seq, uint64_t heads) {
  return {static_cast<char*>(v.data), batch > 1 ? v.batch : 0, seq > 1 ? v.token : 0,
          heads > 1 ? v.head : 0};
}

// More blocks than run at once (four or five an SM), so that their ends do not fall together (2 x 4095
// tokens of 40 heads of 128 bf16, calls repeated: 4 an SM 76.5 us, 16 an SM 72.2 us).
constexpr int kBackwardBlocksPerSM = 16;

uint32_t backward_blocks(int device) {
  return static_cast<uint32_t>(sm_count(device)) * kBackwardBlocksPerSM;
}

// Shared checks; fills what the kernels of all three operators read.
bool make_params(const SparB200Rotary* r, bool norm, bool backward, int device, RotaryParams& p, bool& vec) {
  if (!r) return false;
  if (r->dtype != SPAR_B200_FLOAT32 && r->dtype != SPAR_B200_BFLOAT16) return false;
  if (r->layout != SPAR_B200_ROTARY_INTERLEAVED && r->layout != SPAR_B200_ROTARY_HALF) return false;
  if (r->head_dim < 1 || r->head_dim > 256 || r->rotary_dim < 2 || r->rotary_dim > r->head_dim ||
      (r->rotary_dim & 1))
    return false;
  if (r->heads < 1) return false;
  if (r->batch && r->seq &&
      (r->batch >= kMaxUnits || r->seq >= kMaxUnits || r->heads >= kMaxUnits ||
       r->kv_heads >= kMaxUnits || r->batch * r->seq >= kMaxUnits ||
       r->batch * r->seq * (r->heads + r->kv_heads) >= kMaxUnits))
    return false;
  if (norm && !(r->epsilon >= 0.0 && r->epsilon <= 1e30)) return false;
  if (backward && (!r->dq_weight || !r->scratch || !on16(r->scratch))) return false;
  if (backward && r->kv_heads) {
    if (!r->dk_weight) return false;
    const int64_t apart = r->dq_weight - r->dk_weight;  // both are written whole
    if (apart < static_cast<int64_t>(r->head_dim) && -apart < static_cast<int64_t>(r->head_dim)) return false;
  }
  if (!on4(r->positions) || !on4(r->invalid) || (backward && (!on4(r->dq_weight) || !on4(r->dk_weight))))
    return false;
  p = RotaryParams{};
  const uint64_t tokens = r->batch * r->seq;
  const int sides = r->kv_heads ? 2 : 1;
  const uint64_t v = r->dtype == SPAR_B200_FLOAT32 ? 4 : 8;
  vec = r->rotary_dim % (2 * v) == 0 && r->head_dim % v == 0 && on16(r->table);
  const SparB200Heads* in[2] = {&r->q, &r->k};
  const SparB200Heads* out[2] = {&r->q_out, &r->k_out};
  const SparB200Heads* grad[2] = {&r->dq, &r->dk};
  const float* weight[2] = {r->q_weight, r->k_weight};
  for (int s = 0; s < sides; ++s) {
    const uint64_t heads = s ? r->kv_heads : r->heads;
    p.in[s] = view_of(*in[s], r->batch, r->seq, heads);
    p.out[s] = view_of(*out[s], r->batch, r->seq, heads);
    p.grad[s] = view_of(*grad[s], r->batch, r->seq, heads);
    const View* views[3] = {&p.in[s], &p.out[s], &p.grad[s]};
    for (int x = 0; x < (backward ? 3 : 2); ++x) {
      if (tokens && !views[x]->data) return false;
      const uint64_t size = r->dtype == SPAR_B200_FLOAT32 ? 4 : 2;
      if (reinterpret_cast<uintptr_t>(views[x]->data) % size) return false;
      vec = vec && on16(views[x]->data) && views[x]->batch % v == 0 && views[x]->token % v == 0 &&
            views[x]->head % v == 0;
    }
    const View& o = p.out[s];  // rows on one another (a stride of zero) would be written by many at once
    if (tokens && ((r->batch > 1 && !o.batch) || (r->seq > 1 && !o.token) || (heads > 1 && !o.head)))
      return false;
    if (norm && tokens && (!weight[s] || !on4(weight[s]))) return false;
    vec = vec && (!norm || on16(weight[s]));
    p.weight[s] = weight[s];
  }
  // In place is element by element: the same data with the same strides, on its own side.
  for (int s = 0; tokens && s < sides; ++s)
    for (int other = 0; other < sides; ++other)
      for (const View* v : {&p.in[other], backward ? &p.grad[other] : nullptr}) {
        const View& o = p.out[s];
        if (v && v->data == o.data &&
            (other != s || v->batch != o.batch || v->token != o.token || v->head != o.head))
          return false;
      }
  if (tokens && sides == 2 && p.out[0].data == p.out[1].data) return false;
  if (tokens && !r->positions && (r->table_rows < r->seq || r->start > r->table_rows - r->seq))
    return false;
  const bool rows = !r->positions || r->table_rows;  // of the table, that a token may read
  if (tokens && ((rows && !r->table) || (reinterpret_cast<uintptr_t>(r->table) & 7))) return false;
  p.table = reinterpret_cast<const float2*>(r->table);
  p.table_rows = r->table_rows;
  p.positions = r->positions;
  p.start = r->start;
  p.invalid = r->invalid;
  p.heads[0] = static_cast<uint32_t>(r->heads);
  p.heads[1] = static_cast<uint32_t>(r->kv_heads);
  p.tokens = static_cast<uint32_t>(tokens);
  p.seq = static_cast<uint32_t>(r->seq);
  p.head_dim = static_cast<uint32_t>(r->head_dim);
  p.pairs = static_cast<uint32_t>(r->rotary_dim / 2);
  const uint32_t step = vec ? static_cast<uint32_t>(v) : 1;
  p.rotating = p.pairs / step;
  p.slots = p.rotating + ((p.head_dim - 2 * p.pairs) / step + 1) / 2;
  while ((1u << p.lanes_log2) < p.slots && p.lanes_log2 < 5) ++p.lanes_log2;
  p.sine = 1.f;
  p.eps = static_cast<float>(r->epsilon);
  p.inv_dim = 1.0f / static_cast<float>(r->head_dim);
  p.by_seq = Divider(p.seq ? p.seq : 1);
  p.partial = static_cast<float*>(r->scratch);
  // The backward loads row 0 for a position outside the table, without looking at it: the last row of
  // the scratch, which nobody writes, where the table has none. (A test in the kernel instead cost 2 x
  // 4095 tokens of 40 heads of 128 bf16, half layout, 72 -> 74 us.)
  if (backward && !r->table_rows)
    p.table = reinterpret_cast<const float2*>(p.partial + static_cast<uint64_t>(backward_blocks(device)) * p.head_dim);
  return true;
}

bool full_head(const RotaryParams& p) {
  return 2 * p.pairs == p.head_dim && p.slots == 1u << p.lanes_log2;
}

template <typename T, int VEC, int U, int HP, bool HALF, bool NORM, bool FULL = false>
cudaError_t launch_rotary(RotaryParams& p, cudaStream_t stream) {
  for (int s = 0; s < 2; ++s) p.chunks[s] = (p.heads[s] + HP - 1) / HP;
  p.by_chunks = Divider(p.chunks[0] + p.chunks[1]);
  const uint64_t threads = (static_cast<uint64_t>(p.tokens) * (p.chunks[0] + p.chunks[1]))
                           << p.lanes_log2;
  return launch(rotary_kernel<T, VEC, U, HP, HALF, NORM, FULL>,
                dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, stream, p);
}

template <typename T, int VEC, bool HALF, bool NORM>
cudaError_t launch_forward(RotaryParams& p, bool vec, int device, cudaStream_t stream) {
  if (!vec) return launch_rotary<T, 1, 4, 1, HALF, NORM>(p, stream);
  // heads of a lane group: as many as keep the registers for four blocks an SM (bf16 with norms: one
  // head 23 us, two 29 us for 4 x 4096 tokens of 20 heads of 64; fp32: four 45 us, one 50 us)
  constexpr int kHeads = VEC == 4 ? 4 : NORM ? 1 : 2;
  const uint64_t warps =
      (static_cast<uint64_t>(p.tokens) * (p.heads[0] + p.heads[1]) << p.lanes_log2) / 32;
  const bool many = warps >= static_cast<uint64_t>(sm_count(device)) * 64;
  if (full_head(p))
    return many ? launch_rotary<T, VEC, 1, kHeads, HALF, NORM, true>(p, stream)
                : launch_rotary<T, VEC, 1, 1, HALF, NORM, true>(p, stream);
  return many ? launch_rotary<T, VEC, 1, kHeads, HALF, NORM>(p, stream)
              : launch_rotary<T, VEC, 1, 1, HALF, NORM>(p, stream);
}

template <bool NORM>
SparCudaStatus run_forward(const SparB200Rotary* r, int device, void* stream) {
  RotaryParams p;
  bool vec = false;
  if (!make_params(r, NORM, false, device, p, vec)) return invalid();
  if (!p.tokens) return ok();
  if (!NORM && r->inverse) p.sine = -1.f;
  DeviceScope scope(device);
  if (scope.error() != cudaSuccess) return runtime(scope.error());
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool half = r->layout == SPAR_B200_ROTARY_HALF;
  cudaError_t e;
  if (r->dtype == SPAR_B200_FLOAT32)
    e = half ? launch_forward<float, 4, true, NORM>(p, vec, device, s)
             : launch_forward<float, 4, false, NORM>(p, vec, device, s);
  else
    e = half ? launch_forward<__nv_bfloat16, 8, true, NORM>(p, vec, device, s)
             : launch_forward<__nv_bfloat16, 8, false, NORM>(p, vec, device, s);
  return e == cudaSuccess ? launch_status() : runtime(e);
}

template <typename T, int VEC, int U, bool HALF, bool FULL>
cudaError_t launch_backward_as(RotaryParams& p, int device, cudaStream_t stream, uint32_t& grid) {
  constexpr int HB = VEC == 4 ? 2 : 1;
  const uint32_t groups = kBackwardThreads >> p.lanes_log2;
  uint64_t need[2];
  for (int s = 0; s < 2; ++s) {
    p.chunks[s] = (p.heads[s] + HB - 1) / HB;
    p.by_heads[s] = Divider(p.chunks[s] ? p.chunks[s] : 1);
    need[s] = (static_cast<uint64_t>(p.tokens) * p.chunks[s] + groups - 1) / groups;
  }
  const uint32_t most = backward_blocks(device);
  uint64_t nq = need[0], nk = need[1];
  if (nq + nk > most) {  // in proportion to the heads, at least one each
    nk = p.heads[1] ? std::max<uint64_t>(1, static_cast<uint64_t>(most) * p.heads[1] /
                                                (p.heads[0] + p.heads[1]))
                    : 0;
    nq = most - nk;
  }
  p.blocks_q = static_cast<uint32_t>(nq);
  grid = static_cast<uint32_t>(nq + nk);
  return launch(qk_norm_rotary_backward_kernel<T, VEC, U, HB, HALF, FULL>, dim3(grid), dim3(kBackwardThreads),
                groups * p.head_dim * sizeof(float), stream, p);
}

template <typename T, int VEC, int U, bool HALF>
cudaError_t launch_backward(RotaryParams& p, int device, cudaStream_t stream, uint32_t& grid) {
  if (VEC > 1 && full_head(p))
    return launch_backward_as<T, VEC, U, HALF, (VEC > 1)>(p, device, stream, grid);
  return launch_backward_as<T, VEC, U, HALF, false>(p, device, stream, grid);
}

}  // namespace
}  // namespace spar_b200

using namespace spar_b200;

extern "C" SparCudaStatus spar_b200_rotary_table(float* table, uint64_t rows, uint64_t rotary_dim,
                                                 double theta, uint64_t start,
                                                 const SparB200RotaryScaling* scaling, int device,
                                                 void* stream) {
  if (rotary_dim < 2 || (rotary_dim & 1) || rotary_dim > 256) return invalid();
  if (!(theta > 0.0) || !std::isfinite(theta)) return invalid();
  if (rows > (1ull << 40) || start > (1ull << 40)) return invalid();
  SparB200RotaryScaling sc = {};
  if (scaling) sc = *scaling;
  if (sc.kind < SPAR_B200_ROTARY_NONE || sc.kind > SPAR_B200_ROTARY_PARTS) return invalid();
  if (!std::isfinite(sc.magnitude) || sc.magnitude < 0.0) return invalid();
  if (sc.kind != SPAR_B200_ROTARY_NONE && !(sc.factor > 0.0 && std::isfinite(sc.factor)))
    return invalid();
  if (sc.kind == SPAR_B200_ROTARY_BASE) {
    if (rotary_dim <= 2) return invalid();
    const double d = static_cast<double>(rotary_dim);
    theta *= std::pow(sc.factor, d / (d - 2.0));
    if (!(theta > 0.0) || !std::isfinite(theta)) return invalid();
  }
  if (sc.kind == SPAR_B200_ROTARY_PARTS &&
      (!(sc.original_length > 0.0) || !std::isfinite(sc.original_length) ||
       !(sc.fast_turns > sc.slow_turns) || !std::isfinite(sc.fast_turns - sc.slow_turns)))
    return invalid();
  if (sc.magnitude == 0.0)
    sc.magnitude = sc.kind == SPAR_B200_ROTARY_PARTS && sc.factor > 1.0
                       ? 0.1 * std::log(sc.factor) + 1.0
                       : 1.0;
  if (rows == 0) return ok();
  if (!table || (reinterpret_cast<uintptr_t>(table) & 7)) return invalid();
  const uint64_t pairs = rotary_dim / 2;
  const uint64_t length = std::min<uint64_t>(128, std::max<uint64_t>(8, rows * pairs / 32768));
  const uint64_t threads = (rows + length - 1) / length * pairs;
  if ((threads + 255) / 256 > 0x7fffffffull) return invalid();
  DeviceScope scope(device);
  if (scope.error() != cudaSuccess) return runtime(scope.error());
  const cudaError_t e =
      launch(rotary_table_kernel, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0,
             static_cast<cudaStream_t>(stream), reinterpret_cast<float2*>(table), rows,
             static_cast<uint32_t>(pairs), start, static_cast<uint32_t>(length), sc, theta);
  return e == cudaSuccess ? launch_status() : runtime(e);
}

extern "C" SparCudaStatus spar_b200_rotary(const SparB200Rotary* r, int device, void* stream) {
  return run_forward<false>(r, device, stream);
}

extern "C" SparCudaStatus spar_b200_qk_norm_rotary_forward(const SparB200Rotary* r, int device,
                                                           void* stream) {
  return run_forward<true>(r, device, stream);
}

extern "C" uint64_t spar_b200_qk_norm_rotary_scratch_bytes(uint64_t head_dim, int device) {
  return (static_cast<uint64_t>(backward_blocks(device)) + 1) * head_dim * sizeof(float);
}

extern "C" SparCudaStatus spar_b200_qk_norm_rotary_backward(const SparB200Rotary* r, int device,
                                                            void* stream) {
  RotaryParams p;
  bool vec = false;
  if (!make_params(r, true, true, device, p, vec)) return invalid();
  DeviceScope scope(device);
  if (scope.error() != cudaSuccess) return runtime(scope.error());
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool half = r->layout == SPAR_B200_ROTARY_HALF;
  uint32_t grid = 0;
  cudaError_t e = cudaSuccess;
  if (p.tokens) {
    if (r->dtype == SPAR_B200_FLOAT32) {
      if (vec)
        e = half ? launch_backward<float, 4, 1, true>(p, device, s, grid)
                 : launch_backward<float, 4, 1, false>(p, device, s, grid);
      else
        e = half ? launch_backward<float, 1, 4, true>(p, device, s, grid)
                 : launch_backward<float, 1, 4, false>(p, device, s, grid);
    } else {
      if (vec)
        e = half ? launch_backward<__nv_bfloat16, 8, 1, true>(p, device, s, grid)
                 : launch_backward<__nv_bfloat16, 8, 1, false>(p, device, s, grid);
      else
        e = half ? launch_backward<__nv_bfloat16, 1, 4, true>(p, device, s, grid)
                 : launch_backward<__nv_bfloat16, 1, 4, false>(p, device, s, grid);
    }
    if (e != cudaSuccess) return runtime(e);
  }
  e = launch(qk_weight_partials_kernel, dim3((p.head_dim + 31) / 32, r->kv_heads ? 2 : 1),
             dim3(1024), 0, s, r->dq_weight, r->dk_weight, static_cast<const float*>(p.partial),
             p.blocks_q, grid, p.head_dim, r->accumulate ? 1 : 0);
  return e == cudaSuccess ? launch_status() : runtime(e);
}
