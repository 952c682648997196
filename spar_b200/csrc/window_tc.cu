// Window attention on the sm_100a tensor cores: tcgen05.mma kind::f16 over bf16 operands staged by
// TMA, accumulators in TMEM, the softmax in the warps that read the scores out of TMEM. The
// mathematics stands at the top of window_attention.cu; scores never reach memory.
//
// fp32 inputs run on the same kernels as three bf16 planes: x = x0 + x1 + x2 with x0, x1 the upper
// 16 bits of x and of x - x0, and x2 the rest (8 significant bits each, so the sum is exact for
// normal values). A product keeps the six pairs of planes above 2^-24 of it (x0y0; x0y1, x1y0;
// x1y1, x0y2, x2y0), issued smallest first so that the tensor cores' truncating accumulation
// cuts the small terms at their own size; the product over keys starts afresh for every key tile
// and tiles are added in fp32 registers, so no truncating accumulator spans more than one tile.
//
// One CTA per SM works through its items (two query tiles of 128 rows that share their key tiles:
// two heads of one key head where the group is even, else neighbouring tiles of one head).
// Warp 0 feeds key and value tiles by TMA, one thread of warp 1 issues every product, warps 4-7
// and 8-11 are the softmax of the two tiles (thread = row): while one tile's scores are
// exponentiated the other tile's products run. The keys of an item are its first tokens' tiles,
// then tiles that start exactly at the first key of the window, so a window of W keys under a tile
// of 128 rows costs ceil((W + 127) / BN) tiles. Every wait is bounded and leaves an error flag.
// bf16, 8192 tokens of 32/8 heads of 128, window 1024: 157 us, 825 TFLOP/s, where calls are repeated, and
// 181 us with other inputs every call and a flushed L2. One 128 x 128 tile (scores and P V) takes about
// 2000 cycles of an SM where its products take 1024 (tensor pipe active 50 %): the exponentials and
// packing of two softmax warps a scheduler bound it (sixteen warps, half the columns each: 270 us).
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>

#include "common.cuh"
#include "kernels.cuh"
#include "tc.cuh"
#include "window.cuh"

namespace spar_b200 {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();

namespace window {
namespace {

constexpr uint32_t kMaxSmem = 232448;
constexpr uint32_t kTmemCols = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kPolyShare = 2;        // of every 8 weights of an unmasked bf16 tile (see ex2_poly)
constexpr float kRescaleLog2 = 8.f;  // the running maximum moves only past this margin (P <= 2^8)

// The warp's number, told to the compiler as one value of the warp.
__device__ __forceinline__ int warp_index() {
  return __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
}

// Why a CTA gives up: the CTA's flag, and the one that spar_b200_attention_error reads.
struct Abort {
  volatile int* cta;
  int* device;
};
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, const Abort& abort) {
  if (tc::mbar_wait(bar, parity & 1)) return true;
  atomicExch(abort.device, 1);
  *abort.cta = 1;
  return false;
}

__device__ __forceinline__ uint8_t* align1024(uint8_t* p) {
  return reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Operand tiles in shared memory: per plane, DH / 64 boxes of `rows` rows x 64 elements (128 bytes,
// 128-byte swizzle). The same image is a K-major operand (rows = M or N, elements = K) and an
// MN-major one (elements = N, rows = K).
// Descriptors differ in their low words only (address and leading offset, in 16 bytes), so that a
// product's steps cost one addition each.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (tc::kLayoutSw128 << 29);
__device__ __forceinline__ uint64_t desc(uint32_t low) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(kDescHigh));
  return d;
}
__device__ __forceinline__ uint32_t kmajor_low(uint32_t addr) { return (addr >> 4) | (1u << 16); }
__host__ __device__ constexpr uint32_t kmajor_step(uint32_t rows, int plane, int boxes, int ks) {
  return (plane * boxes + (ks >> 2)) * rows * 8 + (ks & 3) * 2;
}
__device__ __forceinline__ uint32_t mnmajor_low(uint32_t addr, uint32_t rows) {
  return (addr >> 4) | ((rows * 8) << 16);
}
__host__ __device__ constexpr uint32_t mnmajor_step(uint32_t rows, int plane, int boxes, int ks) {
  return plane * boxes * rows * 8 + ks * 128;
}

// Pairs of planes of a product, smallest first: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0).
template <int NP>
constexpr int kProducts = NP == 1 ? 1 : 6;
template <int NP>
__host__ __device__ constexpr int plane_a(int i) { return NP == 1 ? 0 : (0x001102 >> (4 * i)) & 15; }
template <int NP>
__host__ __device__ constexpr int plane_b(int i) { return NP == 1 ? 0 : (0x010120 >> (4 * i)) & 15; }

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// The upper halves of two floats (their bf16 truncations), and what they leave.
__device__ __forceinline__ uint32_t take_upper(float& lo, float& hi) {
  const uint32_t a = __float_as_uint(lo), b = __float_as_uint(hi);
  lo -= __uint_as_float(a & 0xffff0000u);
  hi -= __uint_as_float(b & 0xffff0000u);
  return __byte_perm(a, b, 0x7632);
}

// Registers a thread of this warpgroup may use from here on (all its warps take part; the shares
// of all groups add up to the launch's).
template <int N>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

__device__ __forceinline__ float max_nan(float a, float b, float c) {  // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Bits 0 .. n - 1 (none below 0, all from 32 on).
__device__ __forceinline__ uint32_t below(int n) {
  return n >= 32 ? 0xffffffffu : (1u << max(n, 0)) - 1u;
}
// Scores whose bit is not set become -infinity.
__device__ __forceinline__ void hide32(uint32_t (&v)[32], uint32_t seen) {
#pragma unroll
  for (int e = 0; e < 32; ++e) v[e] = seen & (1u << e) ? v[e] : 0xff800000u;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t both(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x of two values on the FMA pipe (Cody and Waite): x = n + f with n the nearest integer, the
// polynomial 2^f ~ c0 + .. + c4 f^4 on [-1/2, 1/2] (minimax in relative error, 2.7e-6, fitted for
// this file), n added to the exponent. x is cut at -126. The special-function unit makes 16 values
// per cycle and SM, less than the score tiles need; a share of them goes this way.
__device__ __forceinline__ uint64_t ex2_poly(uint64_t x) {
  float2 v = halves(x);
  x = both(fmaxf(v.x, -126.f), fmaxf(v.y, -126.f));
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it leaves the integer in the low bits
  const uint64_t n = add2(x, both(kRound, kRound));
  const uint64_t f = add2(x, fma2(n, both(-1.f, -1.f), both(kRound, kRound)));
  uint64_t y = fma2(f, both(0.009570102f, 0.009570102f), both(0.05591786f, 0.05591786f));
  y = fma2(f, y, both(0.24024744f, 0.24024744f));
  y = fma2(f, y, both(0.6931218f, 0.6931218f));
  y = fma2(f, y, both(0.9999993f, 0.9999993f));
  const float2 e = halves(n), r = halves(y);
  return both(__uint_as_float(__float_as_uint(r.x) + (__float_as_uint(e.x) << 23)),
              __uint_as_float(__float_as_uint(r.y) + (__float_as_uint(e.y) << 23)));
}

// P = 2^(s scale - m) of 32 scores as 16 columns of bf16 pairs, rounded to nearest, and the sums of
// the unrounded values; the last kPoly of every 8 on the FMA pipe. (P in 8 bits is a choice: the product
// takes operands of one type, and a second plane would double P V and its packing. It leaves out 1.15 to
// 1.3 times as far off as its own rounding. A row's sum and lse have all bits but the polynomial's.)
template <int kPoly>
__device__ __forceinline__ void weights32(const uint32_t (&s)[32], uint64_t scale, uint64_t minus_m,
                                          uint64_t (&sums)[2], uint32_t (&u)[16]) {
#pragma unroll
  for (int e = 0; e < 32; e += 2) {
    const uint64_t x = fma2(both(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), scale, minus_m);
    uint64_t w;
    if (e % 8 >= 8 - kPoly) {
      w = ex2_poly(x);
    } else {
      const float2 t = halves(x);
      w = both(ex2(t.x), ex2(t.y));
    }
    sums[e / 2 % 2] = add2(sums[e / 2 % 2], w);
    const float2 t = halves(w);
    u[e / 2] = pack_bf16(t.x, t.y);
  }
}

// 64 consecutive values of a row as three planes of 32 bf16 operand columns.
__device__ __forceinline__ void store_planes(uint32_t taddr, uint32_t plane_cols, float (&v)[64]) {
#pragma unroll
  for (int pl = 0; pl < 3; ++pl) {
    uint32_t r[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) r[e] = take_upper(v[2 * e], v[2 * e + 1]);
    tc::tmem_store_32x32(taddr + pl * plane_cols, r);
  }
}

// 32 rows of results (lane = row) on their way to memory: 16-byte chunks into a box of 32 rows x 128
// bytes (128-byte swizzle, so that neighbouring lanes hit other banks), stored by TMA, which leaves
// out rows and elements outside the tensor. Stores straight from the registers, 16 bytes in each of
// 32 rows, took 4800 cycles per 128 x 128 tile.
struct Box {
  uint8_t* at;  // 4 KB of this warp, 1024-byte aligned
  // Columns col .. col + 31 of the row; NP = 1 packs them to bf16, and two calls fill a box.
  template <int NP>
  __device__ __forceinline__ void put(const CUtensorMap* map, const float (&o)[32], int col, int row,
                                      int head, int batch) const {
    const int lane = threadIdx.x & 31;
    const int chunk = NP == 1 ? (col & 32) / 8 : 0;
    if (chunk == 0) {
      if (lane == 0) tc::bulk_wait_read<0>();
      __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < (NP == 1 ? 4 : 8); ++i) {
      uint4 u;
      if constexpr (NP == 1)
        u = make_uint4(pack_bf16(o[8 * i], o[8 * i + 1]), pack_bf16(o[8 * i + 2], o[8 * i + 3]),
                       pack_bf16(o[8 * i + 4], o[8 * i + 5]), pack_bf16(o[8 * i + 6], o[8 * i + 7]));
      else
        u = make_uint4(__float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]),
                       __float_as_uint(o[4 * i + 2]), __float_as_uint(o[4 * i + 3]));
      *reinterpret_cast<uint4*>(at + lane * 128 + (((chunk + i) ^ (lane & 7)) << 4)) = u;
    }
    if (NP == 1 && chunk == 0) return;
    tc::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      tc::tma_store_5d(map, at, NP == 1 ? col - 32 : col, row, head, batch, 0);
      tc::bulk_commit();
    }
  }
};

struct TcParams {
  WindowParams w;
  CUtensorMap q, k, v, out;
  int* wait_flag;
  int tiles;        // query tiles of 128 rows
  int pair_heads;   // 1: items are (query tile, two heads); 0: (two query tiles, head)
  int items;
  int ksteps;       // K steps of 16 that cover head_dim
  float scale_log2;
};

// Which keys one item visits: `n` tiles of BN keys, the first `ns` over the first tokens (keys
// below `sinks`), the others from `start` on; query tile x uses the first-token tiles and tiles
// ns + a[x] .. ns + b[x] - 1 of the rest (none of any when `any[x]` is false).
struct Item {
  int b, kh, h[2], row[2];
  Sequence s;
  int ns, n, start;
  int a[2], b_end[2];
  bool any[2];
};

// Fills in the keys of an item whose heads and rows are set.
template <int QT, int BN, int TILE = 128>
__device__ __forceinline__ void place_keys(const WindowParams& w, Item& it) {
  it.kh = it.h[0] / w.group;
  it.s = sequence_of(w, it.b);
  int lo[2], hi[2], ulo = INT_MAX, uhi = -1;
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    const int rows = min(TILE, w.q_len - it.row[x]);
    const int pa = max(it.s.p0 + it.row[x], 0), pb = min(it.s.p0 + it.row[x] + rows - 1, it.s.n - 1);
    it.any[x] = rows > 0 && pb >= pa;
    lo[x] = max(0, pa - w.window + 1);
    hi[x] = pb;
    if (it.any[x]) {
      ulo = min(ulo, lo[x]);
      uhi = max(uhi, hi[x]);
    }
  }
  it.ns = it.n = it.start = 0;
  if (uhi < 0) return;
  const bool apart = w.sinks > 0 && ulo > w.sinks;
  it.start = w.sinks > 0 && !apart ? 0 : ulo;
  it.ns = apart ? (w.sinks + BN - 1) / BN : 0;
  it.n = it.ns + (uhi - it.start) / BN + 1;
#pragma unroll
  for (int x = 0; x < QT; ++x) {
    it.a[x] = w.sinks > 0 && !apart ? 0 : (lo[x] - it.start) / BN;
    it.b_end[x] = (hi[x] - it.start) / BN + 1;
  }
}

// The items' last rows first: they see the most keys.
template <int QT, int BN>
__device__ __forceinline__ Item item_of(const TcParams& p, int idx) {
  const WindowParams& w = p.w;
  Item it;
  int bh;
  if (QT == 2 && p.pair_heads) {
    const int pairs = w.heads / 2, per = w.batch * pairs, t = p.tiles - 1 - idx / per;
    bh = idx % per;
    it.b = bh / pairs;
    it.h[0] = (bh - it.b * pairs) * 2;
    it.h[1] = it.h[0] + 1;
    it.row[0] = it.row[1] = t * 128;
  } else {
    const int per = w.batch * w.heads, t = (p.tiles - 1) / QT - idx / per;
    bh = idx % per;
    it.b = bh / w.heads;
    it.h[0] = it.h[1] = bh - it.b * w.heads;
    it.row[0] = t * 128 * QT;
    it.row[1] = it.row[0] + 128;
  }
  place_keys<QT, BN>(w, it);
  return it;
}
// The item of one query tile, in the same order.
template <int BN, int TILE>
__device__ __forceinline__ Item item_of_tile(const WindowParams& w, int idx) {
  const int per = w.batch * w.heads, t = (w.q_len + TILE - 1) / TILE - 1 - idx / per;
  const int bh = idx % per;
  Item it;
  it.b = bh / w.heads;
  it.h[0] = bh - it.b * w.heads;
  it.row[0] = t * TILE;
  place_keys<1, BN, TILE>(w, it);
  return it;
}
// The next tile of query tile x from j on, or n.
__device__ __forceinline__ int next_tile(const Item& it, int x, int j) {
  if (j < it.ns) return j;
  j = max(j, it.ns + it.a[x]);
  return j < it.ns + it.b_end[x] ? j : it.n;
}
template <int BN>
__device__ __forceinline__ int key_of(const Item& it, int j) {
  return j < it.ns ? j * BN : it.start + (j - it.ns) * BN;
}

template <int DH, int NP, int QT, int BN, int KS, int VS>
struct Fwd {
  static constexpr uint32_t kQTile = NP * DH * 256;      // 128 rows
  static constexpr uint32_t kKTile = NP * DH * BN * 2;   // BN rows
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kK = kQ + QT * kQTile;
  static constexpr uint32_t kV = kK + KS * kKTile;
  static constexpr uint32_t kOut = kV + VS * kKTile;  // 4 KB per softmax warp
  static constexpr uint32_t kBar = kOut + QT * 16384;
  static constexpr uint32_t kSmem = kBar + 256 + 1024;
  static_assert(kSmem <= kMaxSmem, "forward shared memory");
  // TMEM columns of one query tile: scores, which P overwrites, then O of the current key tile
  // (NP = 1: of the item), then (NP = 3) the sum of the earlier tiles' O.
  static constexpr uint32_t kS = NP == 1 ? BN : (NP * BN / 2 > BN ? NP * BN / 2 : BN);
  static constexpr uint32_t kCols = kS + DH * (NP == 1 ? 1 : 2);
  static_assert(QT * kCols <= kTmemCols, "forward TMEM");
};

template <int DH, int NP, int QT, int BN, int KS, int VS>
__global__ void __launch_bounds__(128 + 128 * QT, 1) window_forward_kernel(
    const __grid_constant__ TcParams p) {
  using L = Fwd<DH, NP, QT, BN, KS, VS>;
  constexpr int kBoxes = DH / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* q_full = bars;         // [2]
  uint64_t* q_empty = bars + 2;    // [2]
  uint64_t* s_full = bars + 4;     // [2]
  uint64_t* p_full = bars + 6;     // [2]
  uint64_t* o_full = bars + 8;     // [2]
  uint64_t* o_empty = bars + 10;   // [2]
  uint64_t* p_rest = bars + 12;    // [2] NP = 1: the second half of P
  uint64_t* k_full = bars + 14;    // [KS]
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;  // [VS]
  uint64_t* v_empty = v_full + VS;
  uint64_t* drain = v_empty + VS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  const Abort abort_flag = {reinterpret_cast<volatile int*>(tmem_slot + 1), p.wait_flag};
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const WindowParams& w = p.w;

  if (threadIdx.x == 0) {
    for (int x = 0; x < 2; ++x) {
      tc::mbar_init(q_full + x, 1);
      tc::mbar_init(q_empty + x, 1);
      tc::mbar_init(s_full + x, 1);
      tc::mbar_init(p_full + x, 4);
      tc::mbar_init(p_rest + x, 4);
      tc::mbar_init(o_full + x, 1);
      tc::mbar_init(o_empty + x, 4);
    }
    for (int i = 0; i < KS; ++i) {
      tc::mbar_init(k_full + i, 1);
      tc::mbar_init(k_empty + i, 1);
    }
    for (int i = 0; i < VS; ++i) {
      tc::mbar_init(v_full + i, 1);
      tc::mbar_init(v_empty + i, 1);
    }
    tc::mbar_init(drain, 1);
    *abort_flag.cta = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, kTmemCols);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_begin();

  // Four warps that feed and four per query tile: the launch's registers (168 a thread of three
  // groups) are dealt out anew, 88 to the feeding group and 208 to each softmax group, whose
  // threads hold a whole row of 128 scores.
  if (warp < 4) {
    if constexpr (QT == 2) registers_down<88>();
    if (warp == 0) {
      // -------------------------------------------------------------- TMA producer
      if (tc::elect_one()) {
        tc::tma_prefetch(&p.q);
        tc::tma_prefetch(&p.k);
        tc::tma_prefetch(&p.v);
        uint32_t kn = 0, vn = 0, qn[2] = {0, 0};
        bool ok = true;
        for (int idx = blockIdx.x; idx < p.items && ok && !*abort_flag.cta; idx += gridDim.x) {
          const Item it = item_of<QT, BN>(p, idx);
#pragma unroll
          for (int x = 0; x < QT; ++x) {
            if (!it.any[x] || !ok) continue;
            if (!(ok = wait_or_abort(q_empty + x, qn[x] + 1, abort_flag))) break;
            tc::mbar_arrive_expect_tx(q_full + x, L::kQTile);
            ++qn[x];
            for (int pl = 0; pl < NP; ++pl)
              for (int c = 0; c < kBoxes; ++c)
                tc::tma_load_5d(smem + L::kQ + x * L::kQTile + (pl * kBoxes + c) * 16384, &p.q,
                                q_full + x, 64 * c, it.row[x], it.h[x], it.b, pl);
          }
          for (int j = 0; j < it.n && ok; ++j) {
            const int key = key_of<BN>(it, j);
            const uint32_t ks = kn % KS, vs = vn % VS;
            if (!(ok = wait_or_abort(k_empty + ks, kn / KS + 1, abort_flag))) break;
            tc::mbar_arrive_expect_tx(k_full + ks, L::kKTile);
            for (int pl = 0; pl < NP; ++pl)
              for (int c = 0; c < kBoxes; ++c)
                tc::tma_load_5d(smem + L::kK + ks * L::kKTile + (pl * kBoxes + c) * BN * 128, &p.k,
                                k_full + ks, 64 * c, key, it.kh, it.b, pl);
            ++kn;
            if (!(ok = wait_or_abort(v_empty + vs, vn / VS + 1, abort_flag))) break;
            tc::mbar_arrive_expect_tx(v_full + vs, L::kKTile);
            for (int pl = 0; pl < NP; ++pl)
              for (int c = 0; c < kBoxes; ++c)
                tc::tma_load_5d(smem + L::kV + vs * L::kKTile + (pl * kBoxes + c) * BN * 128, &p.v,
                                v_full + vs, 64 * c, key, it.kh, it.b, pl);
            ++vn;
          }
        }
        // Every load issued must have landed before the CTA exits: the last one of each barrier.
        for (int x = 0; x < QT; ++x)
          if (qn[x]) wait_or_abort(q_full + x, qn[x] - 1, abort_flag);
        for (uint32_t i = kn > KS ? kn - KS : 0; i < kn; ++i)
          wait_or_abort(k_full + i % KS, i / KS, abort_flag);
        for (uint32_t i = vn > VS ? vn - VS : 0; i < vn; ++i)
          wait_or_abort(v_full + i % VS, i / VS, abort_flag);
      }
      __syncwarp();
    } else if (warp == 1) {
      // -------------------------------------------------------------- product issuer
      if (tc::elect_one()) {
        const uint32_t idesc_s = tc::idesc_bf16(128, BN, 0, 0);
        const uint32_t idesc_o = tc::idesc_bf16(128, 16 * p.ksteps, 0, 1);
        const uint32_t q_addr = tc::smem_u32(smem + L::kQ), k_addr = tc::smem_u32(smem + L::kK),
                       v_addr = tc::smem_u32(smem + L::kV);
        uint32_t base = 0, qn[2] = {0, 0}, pn[2] = {0, 0}, on[2] = {0, 0};
        bool ok = true;
        for (int idx = blockIdx.x; idx < p.items && ok && !*abort_flag.cta; idx += gridDim.x) {
          const Item it = item_of<QT, BN>(p, idx);
          int issued[2] = {it.n, it.n};  // the last tile whose scores were issued; n: none ever
#pragma unroll
          for (int x = 0; x < QT; ++x)
            if (it.any[x]) issued[x] = -1;
          // Scores of tile j; K_j is free once every query tile that uses it has issued its own.
          auto scores = [&](int x, int j) -> bool {
            const uint32_t st = (base + j) % KS;
            if (!wait_or_abort(k_full + st, (base + j) / KS, abort_flag)) return false;
            tc::tc_fence_after();
            const uint32_t qa = kmajor_low(q_addr + x * L::kQTile), ka = kmajor_low(k_addr + st * L::kKTile);
            uint32_t acc = 0;
#pragma unroll
            for (int pr = 0; pr < kProducts<NP>; ++pr)
#pragma unroll
              for (int ks = 0; ks < DH / 16; ++ks)
                if (ks < p.ksteps) {
                  tc::mma_f16(tmem + x * L::kCols, desc(qa + kmajor_step(128, plane_a<NP>(pr), kBoxes, ks)),
                              desc(ka + kmajor_step(BN, plane_b<NP>(pr), kBoxes, ks)), idesc_s, acc);
                  acc = 1;
                }
            tc::mma_commit(s_full + x);
            issued[x] = j;
            const int y = x ^ 1;
            if (QT == 1 || !it.any[y] || next_tile(it, y, j) != j || issued[y] >= j)
              tc::mma_commit(k_empty + st);
            if (next_tile(it, x, j + 1) == it.n) tc::mma_commit(q_empty + x);
            return true;
          };
#pragma unroll
          for (int x = 0; x < QT; ++x) {
            if (!ok || !it.any[x]) continue;
            if (!(ok = wait_or_abort(q_full + x, qn[x], abort_flag))) break;
            ++qn[x];
            if (next_tile(it, x, 0) == 0) ok = scores(x, 0);
          }
          for (int j = 0; j < it.n && ok; ++j) {
            const uint32_t st = (base + j) % VS;
#pragma unroll
            for (int x = 0; x < QT; ++x) {
              if (!ok || !it.any[x]) continue;
              if (next_tile(it, x, j) == j) {
                if (!(ok = wait_or_abort(p_full + x, pn[x], abort_flag))) break;
                const bool first = next_tile(it, x, 0) == j;
                if (first && !(ok = wait_or_abort(o_empty + x, on[x] + 1, abort_flag))) break;
                if (!(ok = wait_or_abort(v_full + st, (base + j) / VS, abort_flag))) break;
                tc::tc_fence_after();
                uint32_t acc = NP == 1 && !first;
                const uint32_t va = mnmajor_low(v_addr + st * L::kKTile, BN);
#pragma unroll
                for (int pr = 0; pr < kProducts<NP>; ++pr)
#pragma unroll
                  for (int ks = 0; ks < BN / 16; ++ks) {
                    // The product over the first half of the keys runs while the second half's
                    // weights are made.
                    if (NP == 1 && ks == BN / 32) {
                      if (!(ok = wait_or_abort(p_rest + x, pn[x], abort_flag))) break;
                      tc::tc_fence_after();
                    }
                    tc::mma_f16_ts(tmem + x * L::kCols + L::kS,
                                   tmem + x * L::kCols + plane_a<NP>(pr) * (BN / 2) + ks * 8,
                                   desc(va + mnmajor_step(BN, plane_b<NP>(pr), kBoxes, ks)), idesc_o, acc);
                    acc = 1;
                  }
                if (!ok) break;
                ++pn[x];
                if (next_tile(it, x, j + 1) == it.n) {
                  tc::mma_commit(o_full + x);
                  ++on[x];
                }
              }
              // The next scores overwrite P, which the product above reads: one thread's products run
              // in the order of their issue. Never more than one tile ahead of the products over
              // keys, so that a query tile that skips tiles cannot wait for a stage still in use.
              if (j + 1 < it.n && next_tile(it, x, j + 1) == j + 1) ok = scores(x, j + 1);
            }
            if (ok) tc::mma_commit(v_empty + st);
          }
          base += it.n;
        }
        tc::mma_commit(drain);
        wait_or_abort(drain, 0, abort_flag);
      }
      __syncwarp();
    }
  } else {
    // -------------------------------------------------------------- softmax
    if constexpr (QT == 2) registers_up<208>();
    const int x = (warp >> 2) - 1;
    const uint32_t quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((quarter * 32) << 16) + x * L::kCols;
    const Box box = {smem + L::kOut + (warp - 4) * 4096};
    uint32_t base = 0, sn = 0, on = 0;
    bool ok = true;
    for (int idx = blockIdx.x; idx < p.items && ok; idx += gridDim.x) {
      const Item it = item_of<QT, BN>(p, idx);
      const int row = x ? it.row[1] : it.row[0], head = x ? it.h[1] : it.h[0];
      const bool any = x ? it.any[1] : it.any[0];
      const int from = it.ns + (x ? it.a[1] : it.a[0]), upto = it.ns + (x ? it.b_end[1] : it.b_end[0]);
      auto next = [&](int j) {  // as next_tile
        if (j < it.ns) return j;
        j = max(j, from);
        return j < upto ? j : it.n;
      };
      const int pos = it.s.p0 + row + r;
      const bool valid = row + r < w.q_len && pos >= 0 && pos < it.s.n;
      const int first_pos = it.s.p0 + row + static_cast<int>(quarter) * 32;  // of this warp
      float m = -INFINITY, sum = 0.f, pending = 0.f;
      int done = 0;
      if (any) {
        for (int j = next(0); j < it.n && ok; j = next(j + 1), ++done) {
          const int key = key_of<BN>(it, j);
          if (!(ok = wait_or_abort(s_full + x, sn, abort_flag))) break;
          ++sn;
          tc::tc_fence_after();
          if constexpr (NP > 1) {
            // s_full also tells that the product over the previous tile is complete.
            if (done) {
#pragma unroll 1
              for (int c = 0; c < DH / 32; ++c) {
                uint32_t o[32], a[32];
                tc::tmem_load_2x32(lanes + L::kS + c * 32, lanes + L::kS + DH + c * 32, o, a);
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const float u = __uint_as_float(o[e]);
                  o[e] = __float_as_uint(done > 1 ? fmaf(__uint_as_float(a[e]), pending, u) : u);
                }
                tc::tmem_store_32x32(lanes + L::kS + DH + c * 32, o);
              }
            }
          }
          uint32_t v[BN / 32][32];
          if constexpr (BN == 128)
            tc::tmem_load_4x32(lanes, v[0], v[1], v[2], v[3]);
          else
            tc::tmem_load_2x32(lanes, lanes + 32, v[0], v[1]);
          // Keys of this tile that this row sees: c <= last and (c >= near or c < kept).
          const bool all_seen = key + BN - 1 <= first_pos && first_pos + 31 < it.s.n && first_pos >= 0 &&
                                (j < it.ns ? key + BN <= w.sinks
                                           : key > first_pos + 31 - w.window || key + BN <= w.sinks);
          if (!all_seen) {
            int last = min(pos, it.s.n - 1) - key;
            if (j < it.ns) last = min(last, w.sinks - 1 - key);
            if (!valid) last = -1;
            const int near = pos - w.window + 1 - key, kept = w.sinks - key;
#pragma unroll
            for (int c = 0; c < BN / 32; ++c)
              hide32(v[c], below(last + 1 - c * 32) & (~below(near - c * 32) | below(kept - c * 32)));
          }
          float mxs[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) mxs[i] = -INFINITY;
#pragma unroll
          for (int c = 0; c < BN; c += 2)
            mxs[c / 2 & 7] = max_nan(mxs[c / 2 & 7], __uint_as_float(v[c / 32][c % 32]),
                                     __uint_as_float(v[c / 32][c % 32 + 1]));
          const float mx = max_nan(max_nan(mxs[0], mxs[1], mxs[2]), max_nan(mxs[3], mxs[4], mxs[5]),
                                   max_nan(mxs[6], mxs[7], mxs[7])) * p.scale_log2;
          // A score of +infinity or NaN makes the row NaN; the polynomial would not.
          if (!(mx < INFINITY)) sum = __int_as_float(0x7fffffff);
          const bool move = m == -INFINITY ? mx > m : mx > m + kRescaleLog2;
          float f = 1.f;
          if (move) {
            f = ex2(m - mx);
            m = mx;
            sum *= f;
          }
          if constexpr (NP == 1) {
            // O follows the new maximum (s_full: the last O += P V is complete).
            if (done && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
              for (int c = 0; c < DH / 32; ++c) {
                uint32_t o[32];
                tc::tmem_load_32x32(lanes + L::kS + c * 32, o);
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tc::tmem_store_32x32(lanes + L::kS + c * 32, o);
              }
            }
          } else {
            pending = f;
          }
          const float base_m = m == -INFINITY ? 0.f : m;
          // Value rows behind the sequence may hold anything, and 0 times NaN is NaN: clear them, and
          // those behind the first tokens in their tiles, which every row visits.
          const int held = min(it.s.n, j < it.ns ? w.sinks : w.kv_len) - key;
          if (held < BN && key + held < w.kv_len) {
            const uint32_t st = (base + j) % VS;
            if (!(ok = wait_or_abort(v_full + st, (base + j) / VS, abort_flag))) break;
            uint8_t* vt = smem + L::kV + st * L::kKTile;
            for (int i = max(0, held) * 8 + r; i < BN * 8; i += 128)
              for (int box = 0; box < NP * kBoxes; ++box)
                *reinterpret_cast<uint4*>(vt + box * BN * 128 + i * 16) = make_uint4(0, 0, 0, 0);
            tc::fence_proxy_async_smem();
          }
          if constexpr (NP == 1) {
            const uint64_t scale = both(p.scale_log2, p.scale_log2), minus_m = both(-base_m, -base_m);
            uint64_t sums[2] = {both(0.f, 0.f), both(0.f, 0.f)};
#pragma unroll
            for (int c = 0; c < BN / 32; ++c) {
              uint32_t u[16];
              if (all_seen)
                weights32<kPolyShare>(v[c], scale, minus_m, sums, u);
              else
                weights32<0>(v[c], scale, minus_m, sums, u);
              tc::tmem_store_32x16_async(lanes + c * 16, u);
              if (c == BN / 64 - 1 || c == BN / 32 - 1) {
                tc::tmem_store_wait();
                tc::tc_fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive((c == BN / 32 - 1 ? p_rest : p_full) + x);
              }
            }
            const float2 t = halves(add2(sums[0], sums[1]));
            sum += t.x + t.y;
          } else {
            float sums[4] = {0.f, 0.f, 0.f, 0.f};
            float pr[64];
#pragma unroll
            for (int c = 0; c < 64; ++c) {
              pr[c] = ex2(fmaf(__uint_as_float(v[c / 32][c % 32]), p.scale_log2, -base_m));
              sums[c & 3] += pr[c];
            }
            store_planes(lanes, BN / 2, pr);
            sum += (sums[0] + sums[1]) + (sums[2] + sums[3]);
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(p_full + x);
          }
        }
        if (!ok) break;
        if (!(ok = wait_or_abort(o_full + x, on, abort_flag))) break;
        ++on;
        tc::tc_fence_after();
      }
      base += it.n;
      const bool stored = row + r < w.q_len;
      // (a row that sees scores of -infinity alone is 0 / 0, whatever the polynomial makes of them)
      const float inv = !valid ? 0.f : m == -INFINITY ? __int_as_float(0x7fffffff) : 1.f / sum;
#pragma unroll 1
      for (int c = 0; c < DH / 32; ++c) {
        float o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0.f;
        if (any) {
          uint32_t u[32];
          if constexpr (NP == 1) {
            tc::tmem_load_32x32(lanes + L::kS + c * 32, u);
          } else {
            uint32_t a[32];
            tc::tmem_load_2x32(lanes + L::kS + c * 32, lanes + L::kS + DH + c * 32, u, a);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (done > 1) u[e] = __float_as_uint(fmaf(__uint_as_float(a[e]), pending, __uint_as_float(u[e])));
          }
          if (valid) {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(u[e]) * inv;
          }
        }
        if (row + quarter * 32 < w.q_len)
          box.put<NP>(&p.out, o, c * 32, row + quarter * 32, head, it.b);
      }
      if (any) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(o_empty + x);
      }
      if (stored && w.lse)
        w.lse[(static_cast<uint64_t>(it.b) * w.heads + head) * w.q_len + row + r] =
            valid ? m * kLn2 + logf(sum) : -INFINITY;
    }
    if (lane == 0) tc::bulk_wait_all();
    __syncwarp();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc(tmem, kTmemCols);
}

// ============================================================================ backward
// Two launches of one kernel, after D = rowsum(dout o out):
//   queries (KEYS = false)  stationary: 128 rows of q and dout; moving: 64 rows of k and v
//       S = q k^T, dP = dout v^T;  dS = P o (dP - D);  dq += dS k   (bf16: and P k, see Bwd::kCorrect)
//   keys (KEYS = true)      stationary: 128 rows of k and v; moving: 64 rows of q and dout, for
//       every query head of the group: S^T = k q^T, dP^T = v dout^T;  dv += P^T dout;  dk += dS^T q
// P = exp(S - lse) is recomputed on both sides, so every gradient element is summed in one CTA and
// no order is left to chance. P and dS replace S and dP in TMEM and are read there as the A operand.
// With two or three buffers of S and dP the next tiles' products run meanwhile. `scale` is applied to
// dq and dk at the end.
// First tokens are seen by every later row: their key tiles' rows are cut into chunks of
// `chunk` rows that are items of their own (and, where there are few key tiles, so are groups of
// query heads); such items leave fp32 partial sums that a last launch adds in order.
// bf16 rounds P and dS to bf16 for their products, as every such product takes bf16 operands: a second
// rounding of the size of the result's own. (Two planes would cost a product and the packing of each.)
// (2 x 4096 tokens of 16/4 heads of 64 bf16, window 512: 145 us with D and the partials, 138 without the
// sums that correct D; 1 x 8192 x 32/8 heads of 128, window 1024: 571, 523. Some 500 instructions a warp
// and tile at 5.4 cycles each, two warps a scheduler, are what bounds it. fp32, 16 x 1024 x 16 heads of
// 64, all keys: 870 us, bound by the six products. Calls repeated.)
constexpr int kMoving = 64;

struct BackwardParams {
  WindowParams w;
  CUtensorMap s1, s2, m1, m2;  // stationary and moving operands: q, dout / k, v or k, v / q, dout
  CUtensorMap out1, out2;      // dq, or dk and dv
  int* wait_flag;
  int* ticket;  // counts the items drawn beyond the first of each CTA; zero at the launch
  int items, tiles, ksteps;
  float scale_log2, inv_scale;
  // keys: the first `first_tiles` key tiles are cut into `chunks` row ranges, every tile into
  // `head_parts` groups of query heads.
  int first_tiles, chunks, chunk, head_parts;
  int tile;        // stationary rows of a tile
  float* partial;  // [part][2][tile][head_dim]: dk, dv
};

// Which part of the key side an item is: batch, key head, tile, rows, heads; `slot`: its partial,
// or -1 when it is the tile's only item.
struct KeyItem {
  int b, kh, key, row, jobs_per_head, head, heads, end;
  Sequence s;
  int64_t slot;
};
__device__ __forceinline__ KeyItem key_item(const BackwardParams& p, int idx) {
  const WindowParams& w = p.w;
  const int bk = w.batch * w.kv_heads, parts = p.chunks * p.head_parts;
  const int others = (p.tiles - p.first_tiles) * bk * p.head_parts;
  KeyItem it;
  int part, which, tile, from = 0, to = w.q_len;
  if (idx < others) {
    part = idx % p.head_parts;
    const int rest = idx / p.head_parts;
    which = rest % bk;
    tile = p.first_tiles + rest / bk;
    it.slot = p.head_parts > 1 ? static_cast<int64_t>(p.first_tiles) * bk * parts + idx : -1;
  } else {
    const int i = idx - others;
    part = i % parts;
    const int rest = i / parts;
    which = rest % bk;
    tile = rest / bk;
    from = (part / p.head_parts) * p.chunk;
    to = min(from + p.chunk, w.q_len);
    it.slot = parts > 1 ? i : -1;
    part %= p.head_parts;
  }
  it.b = which / w.kv_heads;
  it.kh = which - it.b * w.kv_heads;
  it.key = tile * p.tile;
  it.s = sequence_of(w, it.b);
  it.head = it.kh * w.group + w.group * part / p.head_parts;
  it.heads = it.kh * w.group + w.group * (part + 1) / p.head_parts - it.head;
  // rows that see a key of the tile: positions key .. last key + window - 1 (first tokens: n - 1)
  const int last_key = min(it.key + p.tile - 1, it.s.n - 1);
  const int far = it.key < w.sinks ? it.s.n - 1 : min(it.s.n - 1, last_key + w.window - 1);
  it.row = max(from, it.key - it.s.p0);
  it.end = min(to, far - it.s.p0 + 1);
  it.jobs_per_head =
      last_key >= it.key && it.end > it.row ? (it.end - it.row + kMoving - 1) / kMoving : 0;
  return it;
}

// OUT: which sums of the key side a launch makes (0 both, 1 dk, 2 dv).
template <bool KEYS, int DH, int NP, int ST, int OUT>
struct Bwd {
  // Buffers of S and dP: three where TMEM has room, so that the two softmax groups find their next
  // scores ready; not more than stages, as scores run that far ahead of the last use of a stage.
  static constexpr int kBuffers = NP > 1 ? (ST == 1 ? 1 : 2) : DH == 128 ? 2 : 3;
  static_assert(kBuffers <= ST, "stages");
  static constexpr uint32_t kStats = NP == 1 && DH == 64 ? 2 : 1;  // pairs of stationary operands
  // Stationary rows. Three planes of two operands of 128 columns leave room for 64 of the 128 rows of a
  // product: its other rows read whatever follows in shared memory, give results that nobody reads,
  // and multiply P and dS of zero.
  static constexpr int kTile = NP > 1 && DH == 128 ? 64 : 128;
  static constexpr uint32_t kStat = NP * DH * kTile * 2;      // one stationary operand
  static constexpr uint32_t kMov = NP * DH * kMoving * 2;     // one moving operand
  static constexpr uint32_t kA = 0;
  static constexpr uint32_t kB = kA + kStats * 2 * kStat;
  static constexpr uint32_t kOut = kB + ST * 2 * kMov;        // 4 KB per softmax warp
  // Keys, statistics of the moving rows. bf16: as a K step of the products themselves, operands of 16
  // more columns without swizzle (core matrices of 8 rows x 16 bytes, the two of a row group
  // neighbours): ones on the key side, [ST][2] tiles of three bf16 planes of -lse / scale and of -D
  // on the row side, so that S and dP arrive with them subtracted. (Read from shared memory by every
  // thread they took 620 of 2090 cycles a tile.) fp32: [ST][2][64] -lse log2 e, -D.
  static constexpr bool kAugment = KEYS && NP == 1;
  // Queries, bf16: D comes from the rounded `out`, so the rows of dS do not add up to zero. What a row
  // of the unrounded dS' = P o (dP - D') adds up to is D - D': dq = dS' k - (D - D') P k, and the key
  // side reads the D so corrected. (Without it dq and dk were 1.5 to 1.75 times as far off as their own
  // rounding, most where few keys are seen; with it sqrt 2, the rounding of dS.)
  static constexpr bool kCorrect = !KEYS && NP == 1;
  static constexpr uint32_t kOnes = kOut + 8 * 4096;
  static constexpr uint32_t kRows = kOnes + (kAugment ? 4096 : 0);
  static constexpr uint32_t kRowsBytes = kAugment ? 4096 : 512;  // of a stage
  static constexpr uint32_t kBar = kRows + (KEYS ? ST * kRowsBytes : kCorrect ? 1024 : 0);
  static constexpr uint32_t kSmem = kBar + 320 + 1024;
  static_assert((22 + 2 * ST) * 8 + 24 <= 320, "backward barriers");
  static_assert(kSmem <= kMaxSmem, "backward shared memory");
  // TMEM: buffers of S | dP (| the third planes of P and dS), then the products' sums: of the item, or
  // (NP = 3) of a tile, whose sum over tiles the softmax threads keep.
  static constexpr uint32_t kBuf = KEYS && NP > 1 ? 192 : 128;
  static constexpr uint32_t kAcc = kBuffers * kBuf;
  static constexpr uint32_t kOuts = (KEYS && OUT == 0) || kCorrect ? 2 : 1;
  static constexpr uint32_t kResults = KEYS ? kOuts : 1;
  static_assert(kAcc + kOuts * DH <= kTmemCols, "backward TMEM");
  // Which operands the softmax writes, and whether dS goes over dP (or over S, where P is not needed).
  static constexpr bool kP = KEYS ? OUT != 1 : kCorrect, kDs = OUT != 2;
  static constexpr int kDsAt = KEYS || kCorrect ? 1 : 0;
};

// Column (in a buffer) of plane pl of K step ks of the operand that overwrites S (which = 0) or dP
// (which = 1). Columns 32 g .. 32 g + 31 of S and dP are read by softmax group g alone, and it
// alone overwrites them (two steps of 16 values, 8 columns each, of two planes); third planes go
// to columns nobody reads.
template <bool KEYS>
__host__ __device__ constexpr uint32_t operand_col(int which, int pl, int ks) {
  const int g = ks >> 1, sub = (ks & 1) * 8;
  if (pl < 2) return which * 64 + g * 32 + pl * 16 + sub;
  return KEYS ? 128 + which * 32 + g * 16 + sub : 64 + g * 32 + sub;
}

// Three bf16 planes of a float as the first elements of a 16-byte row of a core matrix.
__device__ __forceinline__ uint4 plane_row(float v) {
  float rest = 0.f, x = v;
  const uint32_t first = take_upper(x, rest) & 0xffffu, second = take_upper(x, rest) << 16;
  return make_uint4(first | second, take_upper(x, rest) & 0xffffu, 0, 0);
}
__device__ __forceinline__ uint32_t core_row(int row) { return (row >> 3) * 256 + (row & 7) * 16; }
// Descriptor of a 16-column K-major operand of such core matrices.
__device__ __forceinline__ uint64_t core_desc(uint32_t addr) { return tc::smem_desc(addr, 128, 256, 0); }

template <bool KEYS, int DH, int NP, int ST, int OUT>
__global__ void __launch_bounds__(384, 1) window_backward_kernel(
    const __grid_constant__ BackwardParams p) {
  using L = Bwd<KEYS, DH, NP, ST, OUT>;
  constexpr int kBoxes = DH / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBar);
  uint64_t* a_full = bars;         // [2]
  uint64_t* a_empty = bars + 2;    // [2]
  uint64_t* s_full = bars + 4;     // [3]
  uint64_t* pd_full = bars + 7;    // [3]
  uint64_t* sum_full = bars + 10;  // the products of a tile (NP = 3) or item are complete
  uint64_t* sum_empty = bars + 11;
  uint64_t* drain = bars + 12;
  uint64_t* m_full = bars + 13;    // [ST]
  uint64_t* m_empty = m_full + ST;
  uint64_t* item_full = m_empty + ST;  // [4]
  uint64_t* item_empty = item_full + 4;
  uint64_t* row_sums = item_empty + 4;  // both groups' sums of dS are there
  volatile int* items = reinterpret_cast<volatile int*>(row_sums + 1);  // [4]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(row_sums + 1) + 4;
  const Abort abort_flag = {reinterpret_cast<volatile int*>(tmem_slot + 1), p.wait_flag};
  const int warp = warp_index(), lane = threadIdx.x & 31;
  const WindowParams& w = p.w;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(a_full + i, 1);
      tc::mbar_init(a_empty + i, 1);
    }
    for (int i = 0; i < 3; ++i) {
      tc::mbar_init(s_full + i, 1);
      tc::mbar_init(pd_full + i, NP == 1 ? 4 : 8);
    }
    tc::mbar_init(sum_full, 1);
    tc::mbar_init(sum_empty, 8);
    tc::mbar_init(drain, 1);
    for (int i = 0; i < ST; ++i) {
      tc::mbar_init(m_full + i, KEYS ? 2 : 1);  // TMA, and the rows' statistics
      tc::mbar_init(m_empty + i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      tc::mbar_init(item_full + i, 1);
      tc::mbar_init(item_empty + i, 1 + 8);  // the issuer, the softmax warps
    }
    tc::mbar_init(row_sums, 8);
    *abort_flag.cta = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, kTmemCols);
    tc::tmem_relinquish();
  }
  if constexpr (L::kAugment) {  // ones in the columns of the three planes; zeros behind them
    for (int i = threadIdx.x; i < 128 * 2; i += blockDim.x)
      *reinterpret_cast<uint4*>(smem + L::kOnes + core_row(i >> 1) + (i & 1) * 128) =
          i & 1 ? make_uint4(0, 0, 0, 0) : make_uint4(0x3f803f80u, 0x3f80u, 0, 0);
    for (int i = threadIdx.x; i < ST * 2 * kMoving; i += blockDim.x)
      *reinterpret_cast<uint4*>(smem + L::kRows + i / kMoving * 2048 + core_row(i % kMoving) + 128) =
          make_uint4(0, 0, 0, 0);
    tc::fence_proxy_async_smem();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  pdl_begin();

  // Items are drawn from a counter when the producer is done with the one before (their costs differ,
  // and a fixed share left a third of the SMs with half the work), and handed on through `items`.
  auto take = [&](uint32_t tn, int& idx) -> bool {
    if (!wait_or_abort(item_full + (tn & 3), tn / 4, abort_flag)) return false;
    idx = items[tn & 3];
    return true;
  };

  // Moving tiles of an item; both sides number them 0 .. n - 1.
  auto jobs_of = [&](int idx, Item& q, KeyItem& k) -> int {
    if constexpr (KEYS) {
      k = key_item(p, idx);
      return k.jobs_per_head * k.heads;
    } else {
      q = item_of_tile<kMoving, L::kTile>(w, idx);
      return q.n;
    }
  };

  // As in the forward: 88 registers a thread for the four feeding warps, 208 for the eight others.
  if (warp < 4) {
    registers_down<88>();
    if (warp == 0) {
      // -------------------------------------------------------------- TMA producer (whole warp)
      if (lane == 0) {
        tc::tma_prefetch(&p.s1);
        tc::tma_prefetch(&p.s2);
        tc::tma_prefetch(&p.m1);
        tc::tma_prefetch(&p.m2);
      }
      uint32_t an = 0, mn = 0;
      bool ok = true;
      for (uint32_t tn = 0; ok && !*abort_flag.cta; ++tn) {
        if (!(ok = wait_or_abort(item_empty + (tn & 3), tn / 4 + 1, abort_flag))) break;
        int idx = blockIdx.x;
        if (tn && lane == 0) idx = static_cast<int>(gridDim.x) + atomicAdd(p.ticket, 1);
        idx = __shfl_sync(0xffffffffu, idx, 0);
        if (lane == 0) {
          items[tn & 3] = idx;
          tc::mbar_arrive(item_full + (tn & 3));
        }
        __syncwarp();
        if (idx >= p.items) break;
        Item q;
        KeyItem k;
        const int n = jobs_of(idx, q, k);
        if (!n) continue;
        const int b = KEYS ? k.b : q.b;
        const uint32_t as = an % L::kStats;
        if (!(ok = wait_or_abort(a_empty + as, an / L::kStats + 1, abort_flag))) break;
        ++an;
        if (lane == 0) {
          tc::mbar_arrive_expect_tx(a_full + as, 2 * L::kStat);
          for (int pl = 0; pl < NP; ++pl)
            for (int c = 0; c < kBoxes; ++c) {
              uint8_t* dst = smem + L::kA + as * 2 * L::kStat + (pl * kBoxes + c) * L::kTile * 128;
              const int row = KEYS ? k.key : q.row[0], h = KEYS ? k.kh : q.h[0];
              tc::tma_load_5d(dst, &p.s1, a_full + as, 64 * c, row, h, b, pl);
              tc::tma_load_5d(dst + L::kStat, &p.s2, a_full + as, 64 * c, row, h, b, pl);
            }
        }
        __syncwarp();
        for (int i = 0; i < n && ok; ++i, ++mn) {
          const uint32_t st = mn % ST;
          if (!(ok = wait_or_abort(m_empty + st, mn / ST + 1, abort_flag))) break;
          int row, h;
          if constexpr (KEYS) {
            const int head = i / k.jobs_per_head;
            row = k.row + (i - head * k.jobs_per_head) * kMoving;
            h = k.head + head;
          } else {
            row = key_of<kMoving>(q, i);
            h = q.kh;
          }
          if (lane == 0) {
            tc::mbar_arrive_expect_tx(m_full + st, 2 * L::kMov);
            for (int pl = 0; pl < NP; ++pl)
              for (int c = 0; c < kBoxes; ++c) {
                uint8_t* dst = smem + L::kB + st * 2 * L::kMov + (pl * kBoxes + c) * kMoving * 128;
                tc::tma_load_5d(dst, &p.m1, m_full + st, 64 * c, row, h, b, pl);
                tc::tma_load_5d(dst + L::kMov, &p.m2, m_full + st, 64 * c, row, h, b, pl);
              }
          }
          if constexpr (KEYS) {
            const uint64_t at = (static_cast<uint64_t>(b) * w.heads + h) * w.q_len;
#pragma unroll
            for (int e = lane; e < kMoving; e += 32) {
              const bool in = row + e < k.end;
              const float lse = in ? __ldg(w.lse + at + row + e) : 0.f;
              const float delta = in ? __ldg(w.delta + at + row + e) : 0.f;
              if constexpr (L::kAugment) {
                uint8_t* tile = smem + L::kRows + st * L::kRowsBytes + core_row(e);
                *reinterpret_cast<uint4*>(tile) = plane_row(-lse * p.inv_scale);
                *reinterpret_cast<uint4*>(tile + 2048) = plane_row(-delta);
              } else {
                float* stats = reinterpret_cast<float*>(smem + L::kRows + st * L::kRowsBytes);
                stats[e] = -lse * kLog2e;
                stats[kMoving + e] = -delta;
              }
            }
            if (L::kAugment) tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(m_full + st);
          }
          __syncwarp();
        }
      }
      for (uint32_t i = an > L::kStats ? an - L::kStats : 0; i < an; ++i)
        wait_or_abort(a_full + i % L::kStats, i / L::kStats, abort_flag);
      for (uint32_t i = mn > ST ? mn - ST : 0; i < mn; ++i)
        wait_or_abort(m_full + i % ST, i / ST, abort_flag);
    } else if (warp == 1) {
      // -------------------------------------------------------------- product issuer
      if (tc::elect_one()) {
        const uint32_t idesc_s = tc::idesc_bf16(128, kMoving, 0, 0);
        const uint32_t idesc_o = tc::idesc_bf16(128, 16 * p.ksteps, 0, 1);
        const uint32_t a_addr = tc::smem_u32(smem + L::kA), b_addr = tc::smem_u32(smem + L::kB);
        [[maybe_unused]] const uint32_t ones = tc::smem_u32(smem + L::kOnes),
                                        stats = tc::smem_u32(smem + L::kRows);
        uint32_t an = 0, mn = 0, sums = 0;
        bool ok = true;
        // S and dP of moving tile number m; after the item's last one the stationary operands are free.
        auto scores = [&](uint32_t m, bool last) -> bool {
          const uint32_t st = m % ST, buf = tmem + (m % L::kBuffers) * L::kBuf;
          if (!wait_or_abort(m_full + st, m / ST, abort_flag)) return false;
          tc::tc_fence_after();
#pragma unroll
          for (int half = 0; half < (OUT == 2 ? 1 : 2); ++half) {
            const uint32_t a = kmajor_low(a_addr + (2 * (an % L::kStats) + half) * L::kStat),
                           b = kmajor_low(b_addr + (2 * st + half) * L::kMov);
            uint32_t acc = 0;
            if constexpr (L::kAugment) {
              tc::mma_f16(buf + half * 64, core_desc(ones),
                          core_desc(stats + st * L::kRowsBytes + half * 2048), idesc_s, 0);
              acc = 1;
            }
#pragma unroll
            for (int pr = 0; pr < kProducts<NP>; ++pr)
#pragma unroll
              for (int ks = 0; ks < DH / 16; ++ks)
                if (ks < p.ksteps) {
                  tc::mma_f16(buf + half * 64, desc(a + kmajor_step(L::kTile, plane_a<NP>(pr), kBoxes, ks)),
                              desc(b + kmajor_step(kMoving, plane_b<NP>(pr), kBoxes, ks)), idesc_s, acc);
                  acc = 1;
                }
          }
          tc::mma_commit(s_full + m % L::kBuffers);
          if (last) tc::mma_commit(a_empty + an % L::kStats);
          return true;
        };
        // The products of tile m's P and dS: queries dq += dS k (and P k); keys dk += dS^T q, dv += P^T dout.
        auto products = [&](uint32_t m, bool first, bool last) {
          const uint32_t st = m % ST, buf = tmem + (m % L::kBuffers) * L::kBuf;
          tc::tc_fence_after();
#pragma unroll
          for (int out = 0; out < static_cast<int>(L::kOuts); ++out) {
            const int operand = OUT == 2 ? 1 : out, which = operand == 0 ? L::kDsAt : 0;
            const uint32_t b = mnmajor_low(b_addr + (2 * st + (KEYS ? operand : 0)) * L::kMov, kMoving);
            uint32_t acc = NP == 1 && !first;
#pragma unroll
            for (int pr = 0; pr < kProducts<NP>; ++pr)
#pragma unroll
              for (int ks = 0; ks < kMoving / 16; ++ks) {
                tc::mma_f16_ts(tmem + L::kAcc + out * DH, buf + operand_col<KEYS>(which, plane_a<NP>(pr), ks),
                               desc(b + mnmajor_step(kMoving, plane_b<NP>(pr), kBoxes, ks)), idesc_o, acc);
                acc = 1;
              }
          }
          tc::mma_commit(m_empty + st);
          if (NP > 1 || last) tc::mma_commit(sum_full);
        };
        auto tiles_of = [&](int idx) -> int {
          Item q;
          KeyItem k;
          return idx < p.items ? jobs_of(idx, q, k) : -1;
        };
        if constexpr (NP == 1 || L::kBuffers == 1) {
          for (uint32_t tn = 0; ok && !*abort_flag.cta; ++tn) {
            int idx;
            if (!(ok = take(tn, idx))) break;
            tc::mbar_arrive(item_empty + (tn & 3));
            const int n = tiles_of(idx);
            if (n < 0) break;
            if (!n) continue;
            if (!(ok = wait_or_abort(a_full + an % L::kStats, an / L::kStats, abort_flag))) break;
            constexpr int kAhead = L::kBuffers > 1 ? L::kBuffers - 1 : 1;
            for (int i = 0; i < kAhead && i < n && ok; ++i) ok = scores(mn + i, i + 1 == n);
            for (int i = 0; i < n && ok; ++i) {
              const uint32_t m = mn + i;
              // The buffer of tile i + kAhead was last read by the products of tile i - 1, issued before.
              if (L::kBuffers > 1 && i + kAhead < n && !(ok = scores(m + kAhead, i + kAhead + 1 == n))) break;
              if (!(ok = wait_or_abort(pd_full + m % L::kBuffers, m / L::kBuffers, abort_flag))) break;
              // Sums start afresh with an item; the softmax warps have read the ones before.
              if (i == 0 && !(ok = wait_or_abort(sum_empty, sums + 1, abort_flag))) break;
              products(m, i == 0, i + 1 == n);
              if (L::kBuffers == 1 && i + 1 < n) ok = scores(m + 1, i + 2 == n);
            }
            mn += n;
            ++sums;
            ++an;
          }
        } else {
          // fp32: scores run ahead of the products over both buffers, also into the next item, whichever is
          // ready first, so that an item's end, its results and the next one's operands cost the tensor
          // cores less (16 x 1024 x 16 x 64, all keys: 980 -> 894 us). Nothing here waits for one while the
          // other could go on. (bf16, with six times fewer products, is bound by this thread's and the
          // softmax's instructions: there it was slower, 137 -> 145 us of 2 x 4096 x 16/4 x 64.)
          uint32_t tn = 0, done = 0;
          uint32_t firsts = 0, lasts = 0;  // bit m & 3: tile m is its item's first or last
          int n = 0, i = 0;                // the item whose scores are under way
          bool more = true;
          uint32_t idle = 0;
          uint64_t since = 0;
          while (ok && (more || done != mn)) {  // tiles whose products, and whose scores, are issued
            bool moved = false;
            if (more && mn - done < static_cast<uint32_t>(L::kBuffers)) {
              if (i >= n) {
                if ((moved = tc::mbar_test(item_full + (tn & 3), tn / 4 & 1))) {
                  const int idx = items[tn & 3];
                  tc::mbar_arrive(item_empty + (tn & 3));
                  ++tn;
                  i = 0;
                  n = tiles_of(idx);
                  more = n >= 0;
                }
              } else if ((i || tc::mbar_test(a_full + an % L::kStats, an / L::kStats & 1)) &&
                         tc::mbar_test(m_full + mn % ST, mn / ST & 1)) {
                const uint32_t bit = 1u << (mn & 3);
                firsts = i ? firsts & ~bit : firsts | bit;
                lasts = i + 1 < n ? lasts & ~bit : lasts | bit;
                ok = scores(mn, i + 1 == n);
                if (++i == n) ++an;
                ++mn;
                moved = true;
              }
            }
            if (done != mn && tc::mbar_test(pd_full + done % L::kBuffers, done / L::kBuffers & 1)) {
              const bool first = firsts >> (done & 3) & 1;
              // (sum_empty as above)
              if (!first || tc::mbar_test(sum_empty, (sums + 1) & 1)) {
                if (first) ++sums;
                products(done, first, lasts >> (done & 3) & 1);
                ++done;
                moved = true;
              }
            }
            if (moved) {
              idle = 0;
            } else if ((++idle & 1023) == 0) {  // the bound on all of these waits
              const uint64_t now = tc::global_timer_ns();
              if (idle == 1024) since = now;
              if (*abort_flag.cta || now - since > tc::kWaitLimitNs) {
                atomicExch(abort_flag.device, 1);
                *abort_flag.cta = 1;
                ok = false;
              }
            }
          }
        }
        tc::mma_commit(drain);
        wait_or_abort(drain, 0, abort_flag);
      }
      __syncwarp();
    }
  } else {
    // -------------------------------------------------------------- softmax and results
    registers_up<208>();
    // bf16: the two groups take the tiles in turn, all 64 columns each (in two halves, as registers
    // allow): while one waits the other works. Half of every tile each took 1460 cycles a tile of
    // 64, most of it in waits and in the latency of two warps a scheduler that did the same.
    // fp32, whose three planes leave fewer buffers than it has groups and tiles in turn: half of every
    // tile each.
    constexpr bool kTurns = NP == 1;
    const int g = (warp - 4) >> 2;
    const uint32_t quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lanes = tmem + ((quarter * 32) << 16);
    const Box box = {smem + L::kOut + (warp - 4) * 4096};
    const uint64_t scale = both(p.scale_log2, p.scale_log2);
    uint32_t mn = 0, sums = 0;
    [[maybe_unused]] uint32_t corrected = 0;
    bool ok = true;
    // NP = 3: the sums over tiles of this thread's row, the groups share the columns; add_sums adds the
    // last tile's products.
    constexpr int kSums = NP > 1 ? L::kOuts * DH / 2 : 32;
    [[maybe_unused]] float tile_sums[kSums];
    auto add_sums = [&](bool first) {
#pragma unroll
      for (int c = 0; c < kSums; c += 32) {
        uint32_t o[32];
        tc::tmem_load_32x32(lanes + L::kAcc + g * kSums + c, o);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          tile_sums[c + e] = first ? __uint_as_float(o[e]) : tile_sums[c + e] + __uint_as_float(o[e]);
      }
    };
    for (uint32_t tn = 0; ok; ++tn) {
      int idx;
      if (!(ok = take(tn, idx))) break;
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(item_empty + (tn & 3));
      if (idx >= p.items) break;
      Item q;
      KeyItem k;
      const int n = jobs_of(idx, q, k);
      const int b = KEYS ? k.b : q.b;
      const Sequence s = KEYS ? k.s : q.s;
      // queries: this row's position and statistics; keys: this row's key
      const int row = (KEYS ? k.key : q.row[0]) + r;
      const int pos = KEYS ? row : s.p0 + row;
      const int first_pos = pos - lane;  // of this warp
      // (keys: older than the first row's window, and no first token, is seen by no row)
      const int oldest = KEYS ? max(s.p0, 0) - w.window + 1 : 0;
      const bool valid = r < L::kTile && (KEYS ? row < s.n && (row >= oldest || row < w.sinks)
                                               : row < w.q_len && pos >= 0 && pos < s.n);
      const bool rows_in = r - lane >= L::kTile ? false
                           : KEYS               ? first_pos + 31 < s.n && first_pos >= oldest
                                : first_pos >= 0 && first_pos + 31 < s.n && row - lane + 31 < w.q_len;
      uint64_t minus_lse = 0, minus_delta = 0;
      [[maybe_unused]] uint64_t ds_sums[2] = {0, 0};
      if (!KEYS && valid && n) {
        const uint64_t at = (static_cast<uint64_t>(b) * w.heads + q.h[0]) * w.q_len + row;
        const float lse2 = __ldg(w.lse + at) * kLog2e, delta = w.delta[at];
        minus_lse = both(-lse2, -lse2);
        minus_delta = both(-delta, -delta);
      }
      for (int i = 0; i < n && ok; ++i) {
        const uint32_t m = mn + i, st = m % ST;
        if (kTurns && (m & 1) != static_cast<uint32_t>(g)) continue;
        const uint32_t buf = lanes + (m % L::kBuffers) * L::kBuf;
        // Columns lo .. hi of the tile are seen, but for the query side's columns before `near`
        // that are not below `kept`. `clear`: moving rows from here on may hold anything.
        int lo = 0, hi, near = 0, kept = 0, clear, key = 0, base = 0, upto = 0;
        if constexpr (KEYS) {
          const int head = i / k.jobs_per_head;
          const int at = k.row + (i - head * k.jobs_per_head) * kMoving;  // first moving row
          base = s.p0 + at;                                               // its position
          upto = k.end - at;
          clear = min(s.n - base, kMoving);
          lo = pos - base;
          hi = min(upto - 1, pos < w.sinks ? kMoving : pos - base + w.window - 1);
        } else {
          key = key_of<kMoving>(q, i);
          clear = min(min(s.n, i < q.ns ? w.sinks : w.kv_len) - key, kMoving);
          hi = min(pos, s.n - 1) - key;
          if (i < q.ns) hi = min(hi, w.sinks - 1 - key);
          near = pos - w.window + 1 - key;
          kept = w.sinks - key;
        }
        if (!valid) hi = -1;
        const bool behind = clear < kMoving && (KEYS ? s.n < s.p0 + w.q_len : key + clear < w.kv_len);
        if (!(ok = wait_or_abort(s_full + m % L::kBuffers, m / L::kBuffers, abort_flag))) break;
        tc::tc_fence_after();
        const float* stats = reinterpret_cast<const float*>(smem + L::kRows + st * L::kRowsBytes);
        if (KEYS && !L::kAugment && !(ok = wait_or_abort(m_full + st, m / ST, abort_flag))) break;
        auto seen_of = [&](int c0) {  // bits of columns c0 .. c0 + 31
          uint32_t seen = below(hi + 1 - c0) & ~below(lo - c0);
          if (!KEYS) seen &= ~below(near - c0) | below(kept - c0);
          return seen;
        };
        // Where the tile or its rows reach behind the sequence they may hold anything, and 0 times NaN is
        // NaN: hidden dP become zero. (Here and not beside the hidden scores: few tiles need it, and in
        // the loop below it cost all of them 3 %.)
        if ((behind || !rows_in) && r - lane < L::kTile) {
#pragma unroll 1
          for (int half = kTurns ? 0 : g; half < (kTurns ? 2 : g + 1); ++half) {
            const uint32_t seen = seen_of(half * 32);
            uint32_t v[32];
            tc::tmem_load_32x32(buf + 64 + half * 32, v);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = seen & (1u << e) ? v[e] : 0u;
            tc::tmem_store_32x32(buf + 64 + half * 32, v);
          }
        }
#pragma unroll
        for (int half = kTurns ? 0 : g; half < (kTurns ? 2 : g + 1); ++half) {
          const int c0 = half * 32;
          uint32_t sv[32], dv[32];
          tc::tmem_load_2x32(buf + c0, buf + 64 + c0, sv, dv);
          bool all_seen = rows_in;
          if constexpr (KEYS)
            all_seen = all_seen && first_pos + 31 <= base + c0 && c0 + 32 <= upto &&
                       (base + c0 + 31 < first_pos + w.window || first_pos + 32 <= w.sinks);
          else
            all_seen = all_seen && key + c0 + 31 <= first_pos &&
                       (i < q.ns ? key + c0 + 32 <= w.sinks
                                 : key + c0 > first_pos + 31 - w.window || key + c0 + 32 <= w.sinks);
          if (!all_seen) hide32(sv, seen_of(c0));  // P and dS of zero
          uint64_t pr[16], ds[16];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            const uint64_t s0 = both(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])),
                           s1 = both(__uint_as_float(sv[2 * e + 2]), __uint_as_float(sv[2 * e + 3]));
            uint64_t g0 = both(__uint_as_float(dv[2 * e]), __uint_as_float(dv[2 * e + 1])),
                     g1 = both(__uint_as_float(dv[2 * e + 2]), __uint_as_float(dv[2 * e + 3]));
            uint64_t x0, x1;
            if constexpr (L::kAugment) {
              x0 = mul2(s0, scale), x1 = mul2(s1, scale);
            } else {
              uint64_t l0 = minus_lse, l1 = minus_lse, d0 = minus_delta, d1 = minus_delta;
              if constexpr (KEYS) {
                const float4 l = *reinterpret_cast<const float4*>(stats + c0 + 2 * e);
                const float4 d = *reinterpret_cast<const float4*>(stats + kMoving + c0 + 2 * e);
                l0 = both(l.x, l.y), l1 = both(l.z, l.w), d0 = both(d.x, d.y), d1 = both(d.z, d.w);
              }
              x0 = fma2(s0, scale, l0), x1 = fma2(s1, scale, l1);
              g0 = add2(g0, d0), g1 = add2(g1, d1);
            }
            const float2 t0 = halves(x0), t1 = halves(x1);
            pr[e] = both(ex2(t0.x), ex2(t0.y));
            pr[e + 1] = both(ex2(t1.x), ex2(t1.y));
            ds[e] = mul2(pr[e], g0);
            ds[e + 1] = mul2(pr[e + 1], g1);
            if constexpr (L::kCorrect) {
              ds_sums[0] = add2(ds_sums[0], ds[e]);
              ds_sums[1] = add2(ds_sums[1], ds[e + 1]);
            }
          }
          // Operands over the columns just read: plane pl of both K steps is 16 columns.
#pragma unroll
          for (int pl = 0; pl < NP; ++pl) {
            uint32_t u[16];
            auto pack = [&](uint64_t& v) -> uint32_t {
              float2 t = halves(v);
              if constexpr (NP == 1) return pack_bf16(t.x, t.y);
              const uint32_t upper = take_upper(t.x, t.y);
              v = both(t.x, t.y);
              return upper;
            };
            if constexpr (L::kP) {
#pragma unroll
              for (int e = 0; e < 16; ++e) u[e] = pack(pr[e]);
              tc::tmem_store_32x16_async(
                  buf + operand_col<KEYS>(0, pl, 0) + (pl < 2 ? half * 32 : half * 16), u);
            }
            if constexpr (L::kDs) {
#pragma unroll
              for (int e = 0; e < 16; ++e) u[e] = pack(ds[e]);
              tc::tmem_store_32x16_async(
                  buf + operand_col<KEYS>(L::kDsAt, pl, 0) + (pl < 2 || !KEYS ? half * 32 : half * 16), u);
            }
          }
        }
        // Moving rows behind the sequence may hold anything, and 0 times NaN is NaN: clear them (and the
        // keys behind the first tokens in their tiles, which every row visits).
        if (behind) {
          if (!KEYS && !(ok = wait_or_abort(m_full + st, m / ST, abort_flag))) break;
          uint8_t* mt = smem + L::kB + st * 2 * L::kMov;
          for (int c = max(clear, 0) * 8 + (kTurns ? r : g * 128 + r); c < kMoving * 8; c += kTurns ? 128 : 256)
            for (int op = 0; op < (KEYS ? 2 : 1) * NP * kBoxes; ++op)
              *reinterpret_cast<uint4*>(mt + op * kMoving * 128 + c * 16) = make_uint4(0, 0, 0, 0);
          tc::fence_proxy_async_smem();
        }
        if constexpr (NP > 1) {
          if (i > 0) {
            if (!(ok = wait_or_abort(sum_full, sums, abort_flag))) break;
            ++sums;
            tc::tc_fence_after();
            add_sums(i == 1);
          }
        }
        tc::tmem_store_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(pd_full + m % L::kBuffers);
      }
      if (!ok) break;
      mn += n;
      if (n) {
        if (!(ok = wait_or_abort(sum_full, sums, abort_flag))) break;
        ++sums;
        tc::tc_fence_after();
        if constexpr (NP > 1) add_sums(n == 1);
      }
      // D - D' of this row: the two groups' tiles, in the order of the groups.
      [[maybe_unused]] float correction = 0.f;
      if constexpr (L::kCorrect) {
        if (n) {
          float* shared_sums = reinterpret_cast<float*>(smem + L::kRows);  // [2][128]
          const float2 t = halves(add2(ds_sums[0], ds_sums[1]));
          shared_sums[g * 128 + r] = t.x + t.y;
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(row_sums);
          if (!(ok = wait_or_abort(row_sums, corrected, abort_flag))) break;
          ++corrected;
          correction = shared_sums[r] + shared_sums[128 + r];
          if (g == 0 && valid)
            w.delta[(static_cast<uint64_t>(b) * w.heads + q.h[0]) * w.q_len + row] =
                correction - halves(minus_delta).x;
        }
      }
      // One result: both groups store half of its columns (bf16 heads of 64: group 0 stores all, as 64
      // columns are one box); both of the key side's: group 0 stores dk, group 1 dv.
      constexpr bool kBoth = KEYS && OUT == 0;
      constexpr int cols = NP == 1 && L::kResults * DH == 64 ? 64 : L::kResults * DH / 2;
      const int out = kBoth ? g : OUT == 2;
      const uint32_t from = lanes + L::kAcc + g * cols;
      const float factor = KEYS && out ? 1.f : w.scale;
      const int warp_row = row - lane;
#pragma unroll(NP > 1 ? cols / 32 : 1)
      for (int c = 0; c < cols; c += 32) {
        if (g * cols >= static_cast<int>(L::kResults) * DH) break;
        float o[32];
        if constexpr (NP > 1) {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = n ? tile_sums[c + e] * factor : 0.f;
        } else {
          uint32_t u[32];
          if constexpr (L::kCorrect) {
            uint32_t pk[32];
            if (n) tc::tmem_load_2x32(from + c, from + DH + c, u, pk);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              u[e] = __float_as_uint(fmaf(-correction, __uint_as_float(pk[e]), __uint_as_float(u[e])));
          } else {
            if (n) tc::tmem_load_32x32(from + c, u);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = n ? __uint_as_float(u[e]) * factor : 0.f;
        }
        const int col = kBoth ? c : g * cols + c;
        if (r - lane >= L::kTile) continue;
        if (KEYS && k.slot >= 0) {
          float* dst = p.partial + ((k.slot * 2 + out) * p.tile + r) * w.head_dim + col;
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (col + e < w.head_dim)
              *reinterpret_cast<float4*>(dst + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        } else if (warp_row < (KEYS ? w.kv_len : w.q_len)) {
          box.put<NP>(out ? &p.out2 : &p.out1, o, col, warp_row, KEYS ? k.kh : q.h[0], b);
        }
      }
      if (n) {
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(sum_empty);
      }
    }
    if (lane == 0) tc::bulk_wait_all();
    __syncwarp();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 1) tc::tmem_dealloc(tmem, kTmemCols);
}

// dk, dv of the key tiles that were cut: the sum of their partials in order.
template <typename T>
__global__ void __launch_bounds__(256) window_partials_kernel(const __grid_constant__ BackwardParams p) {
  pdl_begin();
  const WindowParams& w = p.w;
  const int bk = w.batch * w.kv_heads, d4 = w.head_dim / 4;
  const uint64_t i = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int e = static_cast<int>(i % d4) * 4;
  uint64_t rest = i / d4;
  const int r = static_cast<int>(rest % p.tile);
  rest /= p.tile;
  const int out = static_cast<int>(rest & 1);
  rest >>= 1;
  const int which = static_cast<int>(rest % bk);
  const int tile = static_cast<int>(rest / bk), row = tile * p.tile + r;
  if (tile >= (p.head_parts > 1 ? p.tiles : p.first_tiles) || row >= w.kv_len) return;
  const int parts_first = p.chunks * p.head_parts;
  const bool is_first = tile < p.first_tiles;
  const int parts = is_first ? parts_first : p.head_parts;
  const uint64_t slot =
      is_first ? (static_cast<uint64_t>(tile) * bk + which) * parts_first
               : static_cast<uint64_t>(p.first_tiles) * bk * parts_first +
                     (static_cast<uint64_t>(tile - p.first_tiles) * bk + which) * p.head_parts;
  const float* src = p.partial + ((slot * 2 + out) * p.tile + r) * w.head_dim + e;
  const uint64_t step = 2ull * p.tile * w.head_dim;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < parts; ++k) {
    const float4 v = *reinterpret_cast<const float4*>(src + k * step);
    a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
  }
  const int b = which / w.kv_heads, kh = which - b * w.kv_heads;
  T* dst = row_out<T>(out ? w.dv : w.dk, b, row, kh) + e;
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w));
  else
    *reinterpret_cast<float4*>(dst) = a;
}

// D = rowsum(dout o out), `lanes` threads per (token, head) row, eight elements each; and the item
// counters of the launches that follow, to zero.
template <typename T>
__global__ void __launch_bounds__(256) window_delta_kernel(const __grid_constant__ WindowParams w,
                                                           int lanes, int* tickets, int count) {
  pdl_begin();
  if (blockIdx.x == 0 && threadIdx.x < static_cast<unsigned>(count)) tickets[threadIdx.x] = 0;
  const uint64_t unit = (static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x) / lanes;
  const int l = threadIdx.x & (lanes - 1);
  const bool live = unit < static_cast<uint64_t>(w.batch) * w.q_len * w.heads;
  const int h = live ? static_cast<int>(unit % w.heads) : 0;
  const uint64_t bt = live ? unit / w.heads : 0;
  const int i = static_cast<int>(bt % w.q_len), b = static_cast<int>(bt / w.q_len);
  float s = 0.f;
  if (live && l * 8 < w.head_dim) {
    const T* g = row_ptr<T>(w.dout, b, i, h) + l * 8;
    const T* o = row_ptr<T>(w.out, b, i, h) + l * 8;
    constexpr int n = 16 / sizeof(T);
#pragma unroll
    for (int v = 0; v < 8; v += n) {
      alignas(16) T x[n];
      alignas(16) T y[n];
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(g + v);
      *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(o + v);
#pragma unroll
      for (int e = 0; e < n; ++e) s += as_float(x[e]) * as_float(y[e]);
    }
  }
  for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (live && l == 0) w.delta[(static_cast<uint64_t>(b) * w.heads + h) * w.q_len + i] = s;
}

// The three bf16 planes of an fp32 view, [plane][batch][head][token][dim], in units of four elements.
struct SplitParams {
  View src[4];
  uint16_t* dst[4];
  uint64_t plane[4];  // elements of one plane
  uint64_t units[4];  // running totals of groups of four elements
  int tokens[4], heads[4];
  int dim4;
};
__global__ void __launch_bounds__(256) split_planes_kernel(const __grid_constant__ SplitParams p) {
  pdl_begin();
  const uint64_t u = static_cast<uint64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  int s = 0;
  while (s < 4 && u >= p.units[s]) ++s;
  if (s == 4) return;
  const uint64_t i = u - (s ? p.units[s - 1] : 0);
  const int e = static_cast<int>(i % p.dim4);
  uint64_t row = i / p.dim4;
  const int t = static_cast<int>(row % p.tokens[s]);
  row /= p.tokens[s];
  const int h = static_cast<int>(row % p.heads[s]), b = static_cast<int>(row / p.heads[s]);
  float4 v = *reinterpret_cast<const float4*>(row_ptr<float>(p.src[s], b, t, h) + 4 * e);
#pragma unroll
  for (int pl = 0; pl < 3; ++pl) {
    const uint32_t lo = take_upper(v.x, v.y), hi = take_upper(v.z, v.w);
    *reinterpret_cast<uint2*>(p.dst[s] + pl * p.plane[s] + 4 * i) = make_uint2(lo, hi);
  }
}

// ------------------------------------------------------------------------------- host side
// bf16 (or fp32) view as a 5-D map (element, token, head, batch, plane), boxes of 128 bytes x `rows`.
bool make_view_map(CUtensorMap* map, const void* base, const uint64_t (&dims)[5],
                   const uint64_t (&strides)[4], uint32_t rows, bool f32 = false) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t d[5], s[4];
  for (int i = 0; i < 5; ++i) d[i] = dims[i];
  for (int i = 0; i < 4; ++i) s[i] = dims[i + 1] > 1 ? strides[i] * (f32 ? 4 : 2) : 16;
  cuuint32_t box[5] = {f32 ? 32u : 64u, rows, 1, 1, 1}, unit[5] = {1, 1, 1, 1, 1};
  return fn(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5,
            const_cast<void*>(base), d, s, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

uint64_t round256(uint64_t v) { return (v + 255) & ~255ull; }

// A bf16 view in place, or the planes of an fp32 one.
struct Operand {
  const View* view;
  uint64_t tokens, heads;
  uint16_t* planes;
};
bool operand_map(CUtensorMap* map, const WindowParams& w, const Operand& o, uint32_t rows) {
  const uint64_t d = w.head_dim, b = w.batch;
  if (w.dtype == SPAR_B200_BFLOAT16)
    return make_view_map(map, o.view->data, {d, o.tokens, o.heads, b, 1},
                         {o.view->token, o.view->head, o.view->batch, 8}, rows);
  return make_view_map(map, o.planes, {d, o.tokens, o.heads, b, 3},
                       {d, d * o.tokens, d * o.tokens * o.heads, d * o.tokens * o.heads * b}, rows);
}
// Results in place, in boxes of 32 rows.
bool result_map(CUtensorMap* map, const WindowParams& w, const View& v, uint64_t tokens, uint64_t heads) {
  return make_view_map(map, v.data,
                       {static_cast<uint64_t>(w.head_dim), tokens, heads, static_cast<uint64_t>(w.batch), 1},
                       {v.token, v.head, v.batch, 8}, 32, w.dtype == SPAR_B200_FLOAT32);
}
uint64_t planes_bytes(const WindowParams& w, uint64_t tokens, uint64_t heads) {
  return w.dtype == SPAR_B200_BFLOAT16
             ? 0
             : round256(6ull * w.batch * tokens * heads * static_cast<uint64_t>(w.head_dim));
}

cudaError_t split(const WindowParams& w, const Operand* o, int n, cudaStream_t stream) {
  SplitParams p = {};
  p.dim4 = w.head_dim / 4;
  uint64_t total = 0;
  for (int i = 0; i < 4; ++i) {
    if (i < n) {
      p.src[i] = *o[i].view;
      p.dst[i] = o[i].planes;
      p.tokens[i] = static_cast<int>(o[i].tokens);
      p.heads[i] = static_cast<int>(o[i].heads);
      const uint64_t elements = w.batch * o[i].tokens * o[i].heads * static_cast<uint64_t>(w.head_dim);
      p.plane[i] = elements;
      total += elements / 4;
    }
    p.units[i] = total;
  }
  return launch(split_planes_kernel, dim3(static_cast<unsigned>((total + 255) / 256)), dim3(256), 0,
                stream, p);
}

template <int DH, int NP, int QT, int BN, int KS, int VS>
cudaError_t launch_forward(TcParams& p, int device, cudaStream_t stream) {
  using L = Fwd<DH, NP, QT, BN, KS, VS>;
  auto kernel = window_forward_kernel<DH, NP, QT, BN, KS, VS>;
  const cudaError_t e = raise_dynamic_smem(reinterpret_cast<const void*>(kernel), device, L::kSmem);
  if (e != cudaSuccess) return e;
  const WindowParams& w = p.w;
  p.tiles = (w.q_len + 127) / 128;
  p.pair_heads = QT == 2 && w.group % 2 == 0;
  const int64_t per = p.pair_heads ? w.heads / 2 : w.heads;
  p.items = static_cast<int>(w.batch * per * (p.pair_heads ? p.tiles : (p.tiles + QT - 1) / QT));
  const unsigned grid = static_cast<unsigned>(std::min(p.items, sm_count(device)));
  return launch(kernel, dim3(grid), dim3(128 + 128 * QT), L::kSmem, stream, p);
}

struct BackwardPlan {
  int tile, tiles, first_tiles, chunks, chunk, head_parts;
  uint64_t slots;  // partials
};
// Chunks of the first tokens' tiles cost about half of what another key tile does (window + 127 rows;
// at least 256 so that a short window does not make hundreds) and come last: they even out what the
// whole tiles leave. Query heads of a group are split over items where there would be fewer than two
// items per SM.
BackwardPlan backward_plan(const WindowParams& w, int device) {
  BackwardPlan b;
  b.tile = w.dtype == SPAR_B200_FLOAT32 && w.head_dim > 64 ? 64 : 128;  // Bwd::kTile
  b.tiles = (w.kv_len + b.tile - 1) / b.tile;
  b.first_tiles = (std::min(w.sinks, w.kv_len) + b.tile - 1) / b.tile;
  const int64_t bk = static_cast<int64_t>(w.batch) * w.kv_heads, items = bk * b.tiles;
  b.head_parts = static_cast<int>(
      std::min<int64_t>(w.group, std::max<int64_t>(1, 2 * sm_count(device) / std::max<int64_t>(1, items))));
  // About 1024 items at most come from cutting (first tokens may be many: whole tiles then suffice).
  const int64_t most =
      std::max<int64_t>(1, 1024 / std::max<int64_t>(1, bk * b.first_tiles * b.head_parts));
  const int64_t rows = std::max<int64_t>(
      {256, (static_cast<int64_t>(w.window) / 2 + 127) / 64 * 64, (w.q_len + most - 1) / most});
  b.chunk = static_cast<int>(std::min<int64_t>(rows, std::max(1, w.q_len)));
  b.chunks = (w.q_len + b.chunk - 1) / b.chunk;
  b.slots = 0;
  const uint64_t first_parts = static_cast<uint64_t>(b.chunks) * b.head_parts;
  if (first_parts > 1) b.slots += bk * b.first_tiles * first_parts;
  if (b.head_parts > 1) b.slots += bk * (b.tiles - b.first_tiles) * b.head_parts;
  return b;
}
uint64_t partial_bytes(const WindowParams& w, const BackwardPlan& b) {
  return round256(b.slots * 2 * b.tile * w.head_dim * sizeof(float));
}

template <bool KEYS, int DH, int NP, int ST, int OUT = 0>
cudaError_t launch_backward(const BackwardParams& p, int device, cudaStream_t stream) {
  using L = Bwd<KEYS, DH, NP, ST, OUT>;
  auto kernel = window_backward_kernel<KEYS, DH, NP, ST, OUT>;
  const cudaError_t e = raise_dynamic_smem(reinterpret_cast<const void*>(kernel), device, L::kSmem);
  if (e != cudaSuccess) return e;
  const unsigned grid = static_cast<unsigned>(std::min(p.items, sm_count(device)));
  return launch(kernel, dim3(grid), dim3(384), L::kSmem, stream, p);
}

}  // namespace

bool tc_supported(const WindowParams& w, bool backward) {
  if (w.head_dim % 8 || w.head_dim > 128) return false;
  const int size = w.dtype == SPAR_B200_FLOAT32 ? 4 : 2;
  if (backward) {
    if (w.q_len == 0 || !tiled_view(w.dout, size, w.batch, w.q_len, w.heads) ||
        !tiled_view(w.dq, size, w.batch, w.q_len, w.heads) ||
        !tiled_view(w.dk, size, w.batch, w.kv_len, w.kv_heads) ||
        !tiled_view(w.dv, size, w.batch, w.kv_len, w.kv_heads))
      return false;
  }
  return w.kv_len > 0 && tiled_view(w.q, size, w.batch, w.q_len, w.heads) &&
         tiled_view(w.k, size, w.batch, w.kv_len, w.kv_heads) &&
         tiled_view(w.v, size, w.batch, w.kv_len, w.kv_heads) &&
         tiled_view(w.out, size, w.batch, w.q_len, w.heads);
}

uint64_t tc_scratch_bytes(const WindowParams& w, bool backward, int device) {
  const uint64_t operands = (backward ? 2 : 1) * planes_bytes(w, w.q_len, w.heads) +
                            2 * planes_bytes(w, w.kv_len, w.kv_heads);
  return backward ? operands + partial_bytes(w, backward_plan(w, device)) + 256 : operands;
}

cudaError_t tc_forward(const WindowParams& w, void* scratch, int device, cudaStream_t stream) {
  TcParams p;
  memset(&p, 0, sizeof(p));
  p.w = w;
  p.wait_flag = attention_wait_flag(device);
  if (!p.wait_flag) return cudaErrorInvalidDevice;
  p.ksteps = (w.head_dim + 15) / 16;
  p.scale_log2 = w.scale * kLog2e;
  char* at = static_cast<char*>(scratch);
  Operand o[3] = {{&w.q, static_cast<uint64_t>(w.q_len), static_cast<uint64_t>(w.heads), nullptr},
                  {&w.k, static_cast<uint64_t>(w.kv_len), static_cast<uint64_t>(w.kv_heads), nullptr},
                  {&w.v, static_cast<uint64_t>(w.kv_len), static_cast<uint64_t>(w.kv_heads), nullptr}};
  for (Operand& x : o) {
    x.planes = reinterpret_cast<uint16_t*>(at);
    at += planes_bytes(w, x.tokens, x.heads);
  }
  const bool wide = w.head_dim > 64, f32 = w.dtype == SPAR_B200_FLOAT32;
  const uint32_t rows = f32 ? 64 : 128;
  if (!operand_map(&p.q, w, o[0], 128) || !operand_map(&p.k, w, o[1], rows) ||
      !operand_map(&p.v, w, o[2], rows) || !result_map(&p.out, w, w.out, w.q_len, w.heads))
    return cudaErrorInvalidValue;
  if (f32) {
    const cudaError_t e = split(w, o, 3, stream);
    if (e != cudaSuccess) return e;
    return wide ? launch_forward<128, 3, 1, 64, 1, 1>(p, device, stream)
                : launch_forward<64, 3, 2, 64, 2, 2>(p, device, stream);
  }
  return wide ? launch_forward<128, 1, 2, 128, 2, 2>(p, device, stream)
              : launch_forward<64, 1, 2, 128, 3, 3>(p, device, stream);
}

cudaError_t tc_backward(const WindowParams& w, void* scratch, int device, cudaStream_t stream) {
  const uint64_t ql = w.q_len, kl = w.kv_len, h = w.heads, kh = w.kv_heads;
  const BackwardPlan plan = backward_plan(w, device);
  char* at = static_cast<char*>(scratch);
  Operand o[4] = {{&w.q, ql, h, nullptr}, {&w.k, kl, kh, nullptr}, {&w.v, kl, kh, nullptr},
                  {&w.dout, ql, h, nullptr}};
  for (Operand& x : o) {
    x.planes = reinterpret_cast<uint16_t*>(at);
    at += planes_bytes(w, x.tokens, x.heads);
  }
  BackwardParams p;
  memset(&p, 0, sizeof(p));
  p.w = w;
  p.partial = reinterpret_cast<float*>(at);
  int* tickets = reinterpret_cast<int*>(at + partial_bytes(w, plan));
  p.wait_flag = attention_wait_flag(device);
  if (!p.wait_flag) return cudaErrorInvalidDevice;
  p.ksteps = (w.head_dim + 15) / 16;
  p.scale_log2 = w.scale * kLog2e;
  p.inv_scale = 1.f / w.scale;
  p.tile = plan.tile;
  p.tiles = plan.tiles;
  p.first_tiles = plan.first_tiles;
  p.chunks = plan.chunks;
  p.chunk = plan.chunk;
  p.head_parts = plan.head_parts;
  const bool f32 = w.dtype == SPAR_B200_FLOAT32, wide = w.head_dim > 64;
  cudaError_t e = cudaSuccess;
  if (f32 && (e = split(w, o, 4, stream)) != cudaSuccess) return e;

  int lanes = 1;
  while (lanes * 8 < w.head_dim) lanes *= 2;
  const uint64_t threads = static_cast<uint64_t>(w.batch) * ql * h * lanes;
  auto delta = f32 ? window_delta_kernel<float> : window_delta_kernel<__nv_bfloat16>;
  e = launch(delta, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, stream, w, lanes,
             tickets, 4);
  if (e != cudaSuccess) return e;

  if (!operand_map(&p.s1, w, o[0], p.tile) || !operand_map(&p.s2, w, o[3], p.tile) ||
      !operand_map(&p.m1, w, o[1], kMoving) || !operand_map(&p.m2, w, o[2], kMoving) ||
      !result_map(&p.out1, w, w.dq, ql, h))
    return cudaErrorInvalidValue;
  p.items = static_cast<int>(w.batch * h * ((ql + p.tile - 1) / p.tile));
  p.ticket = tickets;
  e = f32    ? (wide ? launch_backward<false, 128, 3, 1>(p, device, stream)
                     : launch_backward<false, 64, 3, 2>(p, device, stream))
      : wide ? launch_backward<false, 128, 1, 4>(p, device, stream)
             : launch_backward<false, 64, 1, 6>(p, device, stream);
  if (e != cudaSuccess) return e;

  if (!operand_map(&p.s1, w, o[1], p.tile) || !operand_map(&p.s2, w, o[2], p.tile) ||
      !operand_map(&p.m1, w, o[0], kMoving) || !operand_map(&p.m2, w, o[3], kMoving) ||
      !result_map(&p.out1, w, w.dk, kl, kh) || !result_map(&p.out2, w, w.dv, kl, kh))
    return cudaErrorInvalidValue;
  p.items = static_cast<int>(w.batch * kh * p.head_parts *
                             (p.first_tiles * static_cast<uint64_t>(p.chunks) + p.tiles - p.first_tiles));
  p.ticket = tickets + 1;
  // (the sums of dk and dv and their tiles' products, 512 columns, leave TMEM no room for the scores of
  // fp32 heads above 64: a launch each)
  if (f32 && wide && (e = launch_backward<true, 128, 3, 1, 2>(p, device, stream)) != cudaSuccess) return e;
  if (f32 && wide) p.ticket = tickets + 2;
  e = f32    ? (wide ? launch_backward<true, 128, 3, 1, 1>(p, device, stream)
                     : launch_backward<true, 64, 3, 2>(p, device, stream))
      : wide ? launch_backward<true, 128, 1, 3>(p, device, stream)
             : launch_backward<true, 64, 1, 6>(p, device, stream);
  if (e != cudaSuccess || !plan.slots) return e;

  const uint64_t cut = p.head_parts > 1 ? p.tiles : p.first_tiles;
  const uint64_t units = w.batch * kh * cut * 2 * p.tile * (w.head_dim / 4);
  auto sum = f32 ? window_partials_kernel<float> : window_partials_kernel<__nv_bfloat16>;
  return launch(sum, dim3(static_cast<unsigned>((units + 255) / 256)), dim3(256), 0, stream, p);
}

}  // namespace window
}  // namespace spar_b200
