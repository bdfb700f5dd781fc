// Weight-only NVFP4 (w4a16.cuh): the packing of a checkpoint's weights, the linear layer of few tokens, and the mixture-of-experts layer.
//
// One kernel, three uses.  A warp multiplies units of 32 packed rows with up to 8 * kCols columns of activations: codes become the
// 16-bit A operand in registers, the activations of a lane are the B operand as they lie in memory, sums are f32.
//   linear   columns are tokens
//   gate/up  columns are the (token, expert) pairs of one expert; a tile's rows are eight gate rows and the same eight up rows, so that a
//            lane holds both halves of its values and applies SiLU(gate) * up to them
//   down     the value between the projections as two f16, upper and lower part, in two columns: their sum has f32's precision
// Work items are (strip of 32 rows, slot); a slot is a run of one expert's pairs that fits the columns.  A block has a contiguous range of them,
// groups of warps take items in turn and split k among themselves.
// The layer is two launches without anything that has to outlast them: both find the slots from the routing by themselves, the first sets the
// counters of the second, in which the block that finishes a strip's last item adds up its pairs in their order.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "sm100_ptx.cuh"
#include "w4a16.cuh"
#include "w4a16_linear.cuh"

namespace b200fp4 {
namespace {

using namespace w4;

// ------------------------------------------------------------------------------------------ packing

struct PackParams {
  const uint8_t* codes;       // [E, N, K/2]
  const uint8_t* scales;      // [E, N, K/16]
  uint8_t* packed;
  uint32_t* tails;            // [E], gated [E][gate, up]: behind the units, zeroed before
  int64_t strips, units;
  int N, K, gated;
};

// one warp per tile of a unit
__global__ void __launch_bounds__(256) w4a16_pack_kernel(const PackParams p, int64_t n_tiles) {
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= n_tiles) return;
  const int lane = threadIdx.x & 31, tile = (int)(at & 1);
  const int64_t unit = at >> 1, u = unit % p.units, strip = unit / p.units % p.strips, e = unit / p.units / p.strips;
  int step;
  uint8_t* const dst = p.packed + (e * p.strips * p.units + strip_at(strip, p.strips, p.units, u, step)) * kUnitBytes;
  const int64_t row0 = (strip * 2 + tile) * (p.gated ? 8 : 16) + (lane >> 2), apart = p.gated ? p.N / 2 : 8, rows = p.gated ? p.N / 2 : p.N;
  uint32_t sc = 0;
  float peak[2] = {0.f, 0.f};
  for (int half = 0; half < 2; ++half) {
    const int64_t k = u * kUnitK + half * 64 + (lane & 3) * 16;
    uint2 word[2];
    for (int r = 0; r < 2; ++r) {
      uint32_t scale = 0;
      uint2 c = make_uint2(0, 0);
      if ((p.gated ? row0 : row0 + r * 8) < rows && k < p.K) {
        const int64_t row = e * p.N + row0 + r * apart;
        c = *reinterpret_cast<const uint2*>(p.codes + row * (p.K / 2) + k / 2);
        scale = p.scales[row * (p.K / 16) + k / 16];
        if (scale & 0x80) {
          c.x ^= 0x88888888u;
          c.y ^= 0x88888888u;
        }
      }
      scale &= 0x7F;
      if (scale == 0x7F) scale = 0x7E;             // NaN, which the caller has refused
      sc |= scale << (8 * (half * 2 + r));
      word[r] = c;
      uint32_t code = 0;
      for (int i = 0; i < 16; ++i) code = max(code, ((i < 8 ? c.x : c.y) >> (4 * (i & 7))) & 7);
      const float value = (code < 2 ? 0.5f * code : (1.f + 0.5f * (code & 1)) * (float)(1 << (code >> 1)) * 0.5f) * e4m3_to_f32((uint8_t)scale);
      peak[p.gated ? r : 0] = fmaxf(peak[p.gated ? r : 0], value);
    }
    *reinterpret_cast<uint4*>(dst + (tile * 2 + half) * 512 + chunk_at(lane >> 2, lane & 3)) = make_uint4(word[0].x, word[0].y, word[1].x, word[1].y);
  }
  *reinterpret_cast<uint32_t*>(dst + kUnitScales + lane * 8 + tile * 4) = sc;
  // magnitudes are not negative: their bits order as they do, above a tag that is the same for all
  for (int r = 0; r <= p.gated; ++r) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(peak[r]));
    if (lane == 0) atomicMax(p.tails + e * (p.gated + 1) + r, top | size_tag(p.N, p.K, p.gated));
  }
}

// ------------------------------------------------------------------------------------------ products

constexpr int kWarps = 16, kThreads = 32 * kWarps;
constexpr uint32_t kSmemMost = 227 * 1024;
// Units of a warp's ring: three, two where partial sums and rows for more columns need the room.  Two keep as much of HBM busy, but bear less
// unevenness.
__host__ __device__ __forceinline__ constexpr int stages_of(int cols) { return cols == 1 ? 3 : 2; }
__host__ __device__ __forceinline__ constexpr uint32_t ring_bytes(int cols) { return kWarps * stages_of(cols) * kUnitBytes; }
__host__ __device__ __forceinline__ constexpr uint32_t bar_bytes(int cols) { return kWarps * stages_of(cols) * 8; }

__host__ __device__ __forceinline__ uint32_t pad16(uint32_t v) { return (v + 15) / 16 * 16; }
__host__ __device__ __forceinline__ constexpr uint32_t red_bytes(int cols) { return kWarps * 2 * cols * 4 * 32 * 4; }

__device__ __forceinline__ uint4 ld_u4(const void* p) { return *static_cast<const uint4*>(p); }

// A warp's ring of units: one lane asks for them, all wait for them.  Every unit that was asked for is waited for.
template <int kStages>
struct Ring {
  uint32_t units, bars, stage, phase, fill;
  bool ok;
  __device__ __forceinline__ void init(uint32_t base, uint32_t bars_at, int warp, int lane) {
    units = base + warp * (kStages * kUnitBytes);
    bars = bars_at + warp * (kStages * 8);
    stage = phase = fill = 0;
    ok = true;
    if (lane < kStages) mbar_init(bars + lane * 8, 1);
    fence_proxy_async_smem();
    __syncwarp();
  }
  __device__ __forceinline__ void ask(const uint8_t* src, int lane) {
    if (lane == 0) {
      mbar_expect_tx(bars + fill * 8, kUnitBytes);
      bulk_load_1d(units + fill * kUnitBytes, src, kUnitBytes, bars + fill * 8);
    }
    if (++fill == kStages) fill = 0;
  }
  __device__ __forceinline__ uint32_t wait(int* status) {
    if (ok) ok = mbar_wait(bars + stage * 8, phase, status, 61);
    return units + stage * kUnitBytes;
  }
  __device__ __forceinline__ void advance() {      // every lane has read the unit
    if (++stage == kStages) {
      stage = 0;
      phase ^= 1;
    }
    __syncwarp();
  }
  // after a wait that ran out: copies that were asked for land before the block's memory goes
  __device__ __forceinline__ void drain() {
    if (ok) return;
    const long long t0 = clock64();
    while (clock64() - t0 < kWaitCycles / 64) {
    }
  }
};

// a unit's 32 rows times kCols columns of eight; b: the columns' operands, [half][column][8]
template <int kCols>
__device__ __forceinline__ void multiply_unit(uint32_t unit, int lane, uint32_t chunk, const uint32_t (&b)[2][kCols][8], float (&acc)[2][kCols][4]) {
  const uint2 sc = lds64(unit + kUnitScales + lane * 8);
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint4 w = lds128(unit + (t * 2 + half) * 512 + chunk);
      const __half2 s = scales_of(t ? sc.y : sc.x, half), s_lo = __low2half2(s), s_hi = __high2half2(s);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t lo[4], hi[4];
        codes_to_pairs(q ? w.y : w.x, lo);
        codes_to_pairs(q ? w.w : w.z, hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo[j] = as_u32(__hmul2(as_half2(lo[j]), s_lo));
          hi[j] = as_u32(__hmul2(as_half2(hi[j]), s_hi));
        }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          mma_16x8x16(acc[t][c], lo[0], hi[0], lo[1], hi[1], b[half][c][q * 4], b[half][c][q * 4 + 1]);
          mma_16x8x16(acc[t][c], lo[2], hi[2], lo[3], hi[3], b[half][c][q * 4 + 2], b[half][c][q * 4 + 3]);
        }
      }
    }
}

// The same for one or two tokens, without a multiplication by a scale for every pair of values: a column holds one block of 16 of a token's k and
// zeros elsewhere, so that a matrix instruction's sums stay apart by block (kTokens = 1: the eight blocks of the unit; 2: the four of a half, for
// each token), and a scale goes with the block's sum.  268 instructions a unit become 200.  Lane l has columns 2 (l % 4) and the next one:
// part[tile][row l / 4, l / 4 + 8] gets their sum.
template <int kTokens>
__device__ __forceinline__ void multiply_unit_by_block(uint32_t unit, int lane, uint32_t chunk, const uint32_t (&b)[2][8], float (&part)[2][2]) {
  const int row8 = lane >> 2, quad = lane & 3;
  const uint32_t scales = unit + kUnitScales + row8 * 32;
  float d[2][4];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (half == 0 || kTokens == 2)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) d[t][j] = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint4 w = lds128(unit + (t * 2 + half) * 512 + chunk);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t lo[4], hi[4];
        codes_to_pairs(q ? w.y : w.x, lo);
        codes_to_pairs(q ? w.w : w.z, hi);
        mma_16x8x16(d[t], lo[0], hi[0], lo[1], hi[1], b[half][q * 4], b[half][q * 4 + 1]);
        mma_16x8x16(d[t], lo[2], hi[2], lo[3], hi[3], b[half][q * 4 + 2], b[half][q * 4 + 3]);
      }
    }
    if (half == 0 && kTokens == 1) continue;
    // scales of this lane's two blocks: [tile][half: row l / 4, row l / 4 + 8]
    const int first = (quad & 1) * 2;
    const uint2 s0 = lds64(scales + first * 8), s1 = lds64(scales + first * 8 + 8);
    const bool upper = kTokens == 1 ? quad >= 2 : half == 1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t w0 = t ? s0.y : s0.x, w1 = t ? s1.y : s1.x;
      const float2 f0 = __half22float2(e4m3_pair(upper ? w0 >> 16 : w0)), f1 = __half22float2(e4m3_pair(upper ? w1 >> 16 : w1));
      part[t][0] += d[t][0] * f0.x + d[t][1] * f1.x;
      part[t][1] += d[t][2] * f0.y + d[t][3] * f1.y;
    }
  }
}

// columns that are rows in shared memory (f16): lane l's are blocks l % 4 of the unit's two halves
template <int kCols>
__device__ __forceinline__ void staged_columns(const uint32_t (&col)[kCols], uint32_t at, uint32_t (&b)[2][kCols][8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const uint4 lo = lds128(col[c] + at + half * 128), hi = lds128(col[c] + at + half * 128 + 16);
      b[half][c][0] = lo.x, b[half][c][1] = lo.y, b[half][c][2] = lo.z, b[half][c][3] = lo.w;
      b[half][c][4] = hi.x, b[half][c][5] = hi.y, b[half][c][6] = hi.z, b[half][c][7] = hi.w;
    }
}

// Warps that share the units of an item, as a power of two, given the block's items and the units of one.  A unit takes a warp 750 cycles, and 350 of
// its scheduler (an SM has four, warp w is with scheduler w % 4); an item's ending a third of a unit where a warp has the item for itself, else
// nearly one.
inline float share_cost(int items, int units, int log_share) {
  const int share = 1 << log_share, full = (items << log_share) / kWarps, rest = (items << log_share) % kWarps;
  const float item = (float)((units + share - 1) / share) + (log_share == 0 ? 0.33f : 0.9f);
  return item * (float)(full * 1400 + (rest > 0 ? std::max(750, (rest + 3) / 4 * 350) : 0));
}
inline int share_of(int items, int units, int least) {
  int log_share = least;
  for (int s = least + 1; s < 5 && (1 << s) <= units; ++s)
    if (share_cost(items, units, s) < share_cost(items, units, log_share)) log_share = s;
  return log_share;
}
// The least of it where the result is f32: so many warps that each has a chain of the item's k
inline int least_share(int out_dtype, int units) {
  int share = 0;
  while (out_dtype == B200FP4_DTYPE_F32 && share < 4 && (kWarpChain << share) < units) ++share;
  return share;
}

// A run of items is done in phases: rounds of an item a warp, then the rest by groups of warps, so that no warp is without work for more than a part
// of an item.  Against one size of group for all, when they came: 29 tokens, eight experts of 4096, H = 4096, 78 us / 84; one token, ten experts of
// 512, H = 2048, 0.3 us more of its 14, for the longer way to a warp's first weights.
// share: log2 of the warps of a group.  The plan has that of each number of items under a round, four bits each.
struct Phase {
  int count, share;
};
__device__ __forceinline__ Phase next_phase(int rest, uint64_t plan) {
  if (rest >= kWarps) return {rest & -kWarps, 0};
  const int share = (int)(plan >> (rest * 4)) & 15, most = kWarps >> share;
  return {rest < most ? rest : most, share};
}
inline uint64_t phase_plan(int units) {
  static_assert(kWarps == 16, "a plan has 16 numbers of four bits");
  uint64_t plan = 0;
  float cost[kWarps] = {};
  for (int rest = 1; rest < kWarps; ++rest) {
    int best = 0;
    cost[rest] = 1e30f;
    for (int s = 0; s < 5 && (1 << s) <= units; ++s) {
      const int count = std::min(rest, kWarps >> s);
      const float all = share_cost(count, units, s) + cost[rest - count] + 400.f;
      if (all < cost[rest]) cost[rest] = all, best = s;
    }
    plan |= (uint64_t)best << (rest * 4);
  }
  return plan;
}

// An f32 result's chains (kWarpChain): the sums of one to those of the chains before it, in the room where warps exchange theirs, and all of them back.
template <int kCols>
__device__ __forceinline__ void put_aside(float* own, bool first, float (&acc)[2][kCols][4]) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float& sum = own[((t * kCols + c) * 4 + j) * 32];
        sum = first ? acc[t][c][j] : sum + acc[t][c][j];
        acc[t][c][j] = 0.f;
      }
}
template <int kCols>
__device__ __forceinline__ void take_back(const float* own, float (&acc)[2][kCols][4]) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[t][c][j] += own[((t * kCols + c) * 4 + j) * 32];
}

// Sums of the warps that share an item, [warp][tile][column of eight][j][lane]: each warp adds up some of them, in the order of k, and finishes them.
// A lane's sums j are row l / 4 (0, 1) or l / 4 + 8 (2, 3) of a tile and columns 2 (l % 4) and the next one; finish gets those of j = kFirst[i] and
// kSecond[i].  Both barriers are the group's, whichever others there are at the time.
// finish(t, c, i, a, b, std::false_type) may say, with the whole warp, that it wants these sums a second time, with std::true_type: what is rarely
// needed stays out of what always is.
template <int kCols, bool kAcross, typename F>
__device__ __forceinline__ void finish_item(float* red, int log_share, int in_group, int group, int lane, const float (&acc)[2][kCols][4], F&& finish) {
  const int share = 1 << log_share;
  // kAcross: the pair is the two columns of one row (j, j + 1), otherwise the two rows of one column (j, j + 2)
  constexpr int kSums = 2 * kCols * 4 * 32;
  if (share == 1) {
    auto all = [&](auto again) {
      bool done = true;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) done &= finish(t, c, i, acc[t][c][kAcross ? 2 * i : i], acc[t][c][kAcross ? 2 * i + 1 : i + 2], again);
      return done;
    };
    if (!all(std::false_type{})) all(std::true_type{});
    return;
  }
  float* const own = red + group * share * kSums + lane;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int j = 0; j < 4; ++j) own[in_group * kSums + ((t * kCols + c) * 4 + j) * 32] = acc[t][c][j];
  asm volatile("bar.sync %0, %1;" ::"r"((kWarps >> log_share) + group), "r"(share * 32) : "memory");
  for (int u = in_group; u < 4 * kCols; u += share) {
    const int i = u & 1, tc = u >> 1;
    const float *a = own + (tc * 4 + (kAcross ? 2 * i : i)) * 32, *b = a + (kAcross ? 32 : 64);
    float va = 0.f, vb = 0.f;
#pragma unroll 4
    for (int w = 0; w < share; ++w) {
      va += a[w * kSums];
      vb += b[w * kSums];
    }
    const int t = kCols == 1 ? tc : tc / kCols, c = kCols == 1 ? 0 : tc % kCols;
    if (!finish(t, c, i, va, vb, std::false_type{})) finish(t, c, i, va, vb, std::true_type{});
  }
  asm volatile("bar.sync %0, %1;" ::"r"((kWarps >> log_share) + group), "r"(share * 32) : "memory");
}

// ---- powers of two that bring values into f16's range

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float v) { return (int)(__float_as_uint(v) >> 23) - 127; }     // v not negative

// The exponent that brings a row whose largest magnitude has these bf16 bits below 2^15.  Rows with infinities or NaN, which only give such
// again, take the least that no finite value overflows with.
__device__ __forceinline__ int row_exponent(uint32_t bits) { return min(141 - min((int)(bits >> 7), 254), 126); }

// Largest magnitude (as bf16 bits, two of them; bf16 only) and sum of squares (kSquares) of eight elements, added to what there is
template <typename T, bool kSquares>
__device__ __forceinline__ void look_at(const uint4& v, uint32_t& top, float& sum) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);
    if constexpr (kSquares) {
      float2 f;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) f = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
      else f = __half22float2(as_half2(w[j]));
      sum += f.x * f.x + f.y * f.y;
    }
  }
}

// Rows [0, n_rows) -> f16 in shared memory, row_bytes apart, elements [k_begin, k_end) and zeros up to k_stop; all threads.  row_at(r): the row's
// elements; seen(r, factor's reciprocal, sum of squares): called once a row.  Few rows are shared by several warps.
// In two steps: what ask() loads is on its way before a block asks for its weights, behind which it would wait for some 2 us.
template <typename T, bool kSquares>
struct StagedRows {
  static constexpr bool kConvert = std::is_same<T, __nv_bfloat16>::value;
  static constexpr int kHeld = 4;                  // pieces that a lane holds; others are read when they are needed
  int n_rows, k_begin, k_end, log_parts;
  uint4 held[kHeld];

  __device__ __forceinline__ void range(int part, int& k0, int& k1) const {
    const int octets = (k_end - k_begin) >> 3;
    k0 = k_begin + ((octets * part) >> log_parts) * 8 + (threadIdx.x & 31) * 8;
    k1 = k_begin + ((octets * (part + 1)) >> log_parts) * 8;
  }
  __device__ __forceinline__ void hold(const T* row, int k0, int k1) {
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
      if (k0 + h * 256 < k1) held[h] = ld_u4(row + k0 + h * 256);
  }
  template <typename RowAt>
  __device__ __forceinline__ void ask(int rows, int begin, int end, RowAt&& row_at) {
    n_rows = rows;
    k_begin = begin;
    k_end = end;
    log_parts = 4;
    while (log_parts > 0 && (n_rows << log_parts) > kWarps) --log_parts;
    const int warp = threadIdx.x >> 5, r = warp >> log_parts;
    int k0, k1;
    range(warp & ((1 << log_parts) - 1), k0, k1);
    if (r < n_rows) hold(row_at(r), k0, k1);
  }
  template <typename RowAt, typename Seen>
  __device__ __forceinline__ void finish(int k_stop, unsigned char* rows, uint32_t row_bytes, float2* parts, RowAt&& row_at, Seen&& seen) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_parts = 1 << log_parts;
#pragma unroll 1
    for (int i0 = 0; i0 < n_rows << log_parts; i0 += kWarps) {
      const int r = (i0 + warp) >> log_parts, part = (i0 + warp) & (n_parts - 1);
      const bool work = r < n_rows;
      int k0, k1;
      range(part, k0, k1);
      if (!work) k1 = 0;
      const T* const row = work ? row_at(r) : nullptr;
      if (i0 > 0) hold(row, k0, k1);
      uint32_t factor = 0;
      float inv = 1.f, squares = 0.f;
      if constexpr (kConvert || kSquares) {
        uint32_t top = 0;
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
          if (k0 + h * 256 < k1) look_at<T, kSquares>(held[h], top, squares);
#pragma unroll 2
        for (int k = k0 + kHeld * 256; k < k1; k += 256) look_at<T, kSquares>(ld_u4(row + k), top, squares);
        top = __reduce_max_sync(0xffffffffu, max(top & 0xFFFFu, top >> 16));
        if constexpr (kSquares)
#pragma unroll
          for (int d = 16; d > 0; d /= 2) squares += __shfl_xor_sync(0xffffffffu, squares, d);
        if (n_parts > 1) {                         // one round then
          if (lane == 0) parts[warp] = make_float2(__uint_as_float(top), squares);
          __syncthreads();
          // one part a lane, and sums in the same order for every warp of the row
          const float2 u = lane < n_parts ? parts[warp - part + lane] : make_float2(0.f, 0.f);
          top = __reduce_max_sync(0xffffffffu, __float_as_uint(u.x));
          squares = u.y;
          if constexpr (kSquares)
#pragma unroll
            for (int d = kWarps / 2; d > 0; d /= 2) squares += __shfl_xor_sync(0xffffffffu, squares, d);
        }
        const int e = kConvert ? row_exponent(top) : 0;
        factor = (uint32_t)(e + 127) * 0x00800080u;
        inv = pow2(-e);
      }
      if (!work) continue;
      unsigned char* const to = rows + r * row_bytes - k_begin * 2;
      auto put = [&](int k, uint4 v) {
        if constexpr (kConvert)
          v = make_uint4(bf16_to_f16_pair(v.x, factor), bf16_to_f16_pair(v.y, factor), bf16_to_f16_pair(v.z, factor), bf16_to_f16_pair(v.w, factor));
        *reinterpret_cast<uint4*>(to + k * 2) = v;
      };
#pragma unroll
      for (int h = 0; h < kHeld; ++h)
        if (k0 + h * 256 < k1) put(k0 + h * 256, held[h]);
#pragma unroll 2
      for (int k = k0 + kHeld * 256; k < k1; k += 256) put(k, ld_u4(row + k));
      if (part == n_parts - 1)
        for (int k = k_end + lane * 8; k < k_stop; k += 256) *reinterpret_cast<uint4*>(to + k * 2) = make_uint4(0, 0, 0, 0);
      if constexpr (kConvert || kSquares)
        if (part == 0 && lane == 0) seen(r, inv, squares);
    }
  }
};

// ------------------------------------------------------------------------------------------ linear layer of few tokens

constexpr int kMaxSplit = 8;

struct LinearParams {
  const void* x;              // [M, K], rows ldx apart
  int64_t ldx;
  const uint8_t* packed;
  const uint32_t* tail;
  const float* g;
  void* out;                  // [M, N]
  const void* bias;           // [N] or null
  int out_dtype, bias_dtype;
  int M, N, K;
  int strips, units;
  int split;                  // blocks of a cluster, which share the units of an item
  int cap;                    // columns of an item
  int per, more;              // items of a cluster: `per`, and one more for the first `more` clusters
  int log_share;
  uint32_t tag;
  int* status;
};

// Shared memory behind the rings and barriers: partial sums of warps | factors' reciprocals | parts of the rows' statistics | rows in f16 | sums of a
// cluster's items, [source block][value], of this block's share of the values
struct LinearLayout {
  uint32_t red, inv, parts, rows, sums, bytes;
};
__host__ __device__ __forceinline__ LinearLayout linear_layout(int cols, int cap, uint32_t row_bytes, int split, int items) {
  LinearLayout l;
  l.red = pad16(ring_bytes(cols) + bar_bytes(cols));
  l.inv = l.red + red_bytes(cols);
  l.parts = pad16(l.inv + (uint32_t)cap * 4);
  l.rows = l.parts + kWarps * 8;
  l.sums = l.rows + (uint32_t)cap * row_bytes;
  // strips of an item are 32 rows: each block of the cluster finishes 32 / split of them
  l.bytes = l.sums + (split > 1 ? (uint32_t)items * cap * 32 * 4 : 0);
  return l;
}

// The linear layer of few tokens: bound by the copies of the weight, then by decoding it.  An SM's 16 warps decode and multiply a unit in 87 cycles
// with one column of eight (131 with two), and its share of HBM brings one in 98: N=14336 K=4096, 33 MB, takes 9.2 us for one token and 10.8 for
// eight, of which 2 are the launch and the row, 1.5 the first units' way and 5.1 the floor; N=K=2048 4.4, most of it launch.  Large layers stay below
// the copy rate, since a block or a cluster has whole strips: 448 of them are three or four a block, and 256 one or two, a sixth more than the mean:
// four tokens, N=8192 K=14336, 66 MB, 18.2 us, 56 % of the copy rate.
// XT: type of the activations; kCols: columns of eight; kTokens: 1 or 2 where there are no more, else 0
template <typename XT, int kCols, int kTokens>
__global__ void __launch_bounds__(kThreads, 1) w4a16_linear_kernel(const LinearParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr bool kConvert = std::is_same<XT, __nv_bfloat16>::value;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row8 = lane >> 2, quad = lane & 3;
  const uint32_t base = smem_u32(smem), chunk = chunk_at(row8, quad);
  Ring<stages_of(kCols)> ring;
  ring.init(base, base + ring_bytes(kCols), warp, lane);
  const int split = p.split, rank = (int)blockIdx.x & (split - 1), cluster = (int)blockIdx.x / split;      // split: a power of two
  const int unit_first = p.units * rank / split, own_units = p.units * (rank + 1) / split - unit_first;
  const int share = 1 << p.log_share, group = warp >> p.log_share, in_group = warp & (share - 1), n_groups = kWarps >> p.log_share;
  const int k_first = (own_units * in_group) >> p.log_share, n_units = ((own_units * (in_group + 1)) >> p.log_share) - k_first;
  const int first = cluster * p.per + min(cluster, p.more), last = first + p.per + (cluster < p.more ? 1 : 0);
  // Strips of a slot of tokens are neighbours
  int ahead = first + group, ahead_left = 0, src_step = 0;
  const uint8_t* src = nullptr;
  auto fetch = [&]() {
    if (ahead_left == 0) {
      if (ahead >= last) return;
      src = p.packed + (size_t)strip_at(ahead % p.strips, p.strips, p.units, unit_first + k_first, src_step) * kUnitBytes;
      ahead_left = n_units;
      ahead += n_groups;
    }
    ring.ask(src, lane);
    src += src_step * kUnitBytes;
    --ahead_left;
  };
  const int k_begin = unit_first * kUnitK, k_stop = (unit_first + own_units) * kUnitK, k_end = min(p.K, k_stop);
  StagedRows<XT, false> staged;
  const int first_slot = first / p.strips;
  int m0 = first_slot * p.cap;
  auto row_at = [&](int r) { return static_cast<const XT*>(p.x) + (m0 + r) * p.ldx; };
  pdl_wait();
  staged.ask(min(p.cap, p.M - m0), k_begin, k_end, row_at);
#pragma unroll 1
  for (int i = 0; i < stages_of(kCols); ++i) fetch();
  pdl_launch_dependents();
  const bool reports = blockIdx.x == gridDim.x - split && threadIdx.x == 0;       // this block has the last item of all
  if (reports) *p.status = 0;
  if (split > 1) cluster_arrive_relaxed();         // the other blocks run before anything is sent to them
  // rows are shifted by 16 bytes against each other: no two lanes of a load meet
  const uint32_t row_bytes = (uint32_t)((p.units + split - 1) / split) * (kUnitK * 2) + 16;
  const LinearLayout l = linear_layout(kCols, p.cap, row_bytes, split, p.per + (p.more > 0));
  float* const inv = reinterpret_cast<float*>(smem + l.inv);
  const float g = *p.g;
  // The word behind the units is read by the blocks that read the last strip, next to it: as a page of its own for all of them it cost a tenth of one
  // token's time.  It is looked at when the strip is done.
  const uint32_t tail = last >= (first_slot + 1) * p.strips ? *p.tail : p.tag;
  auto factor = [&](int strip) {
    if (strip != p.strips - 1) return g;
    uint32_t word = tail;
    asm volatile("" : "+r"(word));
    return packed_for(word, p.tag) ? g : __int_as_float(0x7FC00000);
  };
  bool arrived = split == 1;
  int item = first + group;
  for (int done = first; done < last;) {
    // one slot of tokens at a time
    const int slot = done / p.strips, end = min(last, (slot + 1) * p.strips);
    m0 = slot * p.cap;
    const int n = min(p.cap, p.M - m0);
    if (done > first) {
      __syncthreads();                             // nobody reads the rows before these any more
      staged.ask(n, k_begin, k_end, row_at);
    }
    staged.finish(k_stop, smem + l.rows, row_bytes, reinterpret_cast<float2*>(smem + l.parts), row_at, [&](int r, float v, float) { inv[r] = v; });
    __syncthreads();
    uint32_t col[kCols];
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      const int i = c * 8 + row8;                  // columns past the tokens read the first one's row: nobody reads their sums
      col[c] = base + l.rows + (i < n ? i : 0) * row_bytes + quad * 32;
    }
    for (; item < end; item += n_groups) {
      float acc[2][kCols][4] = {};
      if constexpr (kTokens > 0) {
        // this lane's column: block (l / 4) % 4 of a half, of the first half and then the second or of token l / 16
        const int token = kTokens == 2 ? row8 >> 2 : 0;
        const bool mine0 = kTokens == 2 ? (row8 & 3) == quad : row8 == quad, mine1 = kTokens == 2 ? mine0 : row8 == quad + 4;
        const uint32_t row = base + l.rows + (token < n ? token : 0) * row_bytes + quad * 32;
        float part[2][2] = {};
        uint32_t b[2][8] = {};
#pragma unroll 1
        for (int k = k_first; k < k_first + n_units; ++k) {
#pragma unroll
          for (int half = 0; half < 2; ++half)
            if (half ? mine1 : mine0) {
              const uint4 lo = lds128(row + k * (kUnitK * 2) + half * 128), hi = lds128(row + k * (kUnitK * 2) + half * 128 + 16);
              b[half][0] = lo.x, b[half][1] = lo.y, b[half][2] = lo.z, b[half][3] = lo.w;
              b[half][4] = hi.x, b[half][5] = hi.y, b[half][6] = hi.z, b[half][7] = hi.w;
            }
          multiply_unit_by_block<kTokens>(ring.wait(p.status), lane, chunk, b, part);
          ring.advance();
          if (ring.ok) fetch();
        }
        // a token's blocks: four lanes, or two; the second token's sums to where columns 0 and 1 are
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float v = part[t][r] + __shfl_xor_sync(0xffffffffu, part[t][r], 1);
            const float other = __shfl_xor_sync(0xffffffffu, v, 2);
            acc[t][0][r * 2] = kTokens == 1 ? v + other : v;
            if (kTokens == 2) acc[t][0][r * 2 + 1] = other;
          }
      } else {
#pragma unroll 1
        for (int k = k_first; k < k_first + n_units; ++k) {
          uint32_t b[2][kCols][8];
          staged_columns<kCols>(col, k * (kUnitK * 2), b);
          multiply_unit<kCols>(ring.wait(p.status), lane, chunk, b, acc);
          ring.advance();
          if (ring.ok) fetch();
        }
      }
      if (!arrived) {
        cluster_wait();
        arrived = true;
      }
      const int strip = item - slot * p.strips;
      finish_item<kCols, false>(reinterpret_cast<float*>(smem + l.red), p.log_share, in_group, group, lane, acc, [&](int t, int c, int i, float va, float vb, auto) {
        const int column = c * 8 + quad * 2 + i, row = t * 16 + row8;
        if (column >= n) return true;
        const float f = kConvert ? inv[column] : 1.f;
        if (split > 1) {
          // value [row of the strip] is finished by block row / (32 / split): [source][item][column][its rows]
          const int rows = 32 / split;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = row + h * 8, owner = at / rows;
            const uint32_t to = base + l.sums + (((uint32_t)(rank * (p.per + (p.more > 0)) + item - first) * p.cap + column) * rows + at - owner * rows) * 4;
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(to, owner)), "f"((h ? vb : va) * f) : "memory");
          }
        } else {
          const float gf = factor(strip);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int at = strip * 32 + row + h * 8;
            if (at < p.N) {
              float v = (h ? vb : va) * f * gf;
              if (p.bias != nullptr) v += load_value(p.bias, p.bias_dtype, at);
              store_value(p.out, p.out_dtype, (size_t)(m0 + column) * p.N + at, v);
            }
          }
        }
        return true;
      });
    }
    done = end;
  }
  ring.drain();
  if (reports && !packed_for(tail, p.tag)) *p.status = kOtherSizes;
  if (split > 1) {
    if (!arrived) cluster_wait();
    cluster_sync_any();                            // the parts of k have arrived; they are added in their order
    const int rows = 32 / split, items = p.per + (p.more > 0), count = (last - first) * p.cap * rows;
    const float* const sums = reinterpret_cast<const float*>(smem + l.sums);
    for (int i = threadIdx.x; i < count; i += kThreads) {
      const int r = i & (rows - 1), ic = i / rows, it = first + ic / p.cap, column = ic % p.cap;
      const int slot = it / p.strips, row = (it - slot * p.strips) * 32 + rank * rows + r, m = slot * p.cap + column;
      if (m >= p.M || row >= p.N) continue;
      float v = 0.f;
      for (int s = 0; s < split; ++s) v += sums[s * items * p.cap * rows + i];
      v *= factor(it - slot * p.strips);
      if (p.bias != nullptr) v += load_value(p.bias, p.bias_dtype, row);
      store_value(p.out, p.out_dtype, (size_t)m * p.N + row, v);
    }
  }
}

template <typename Kernel>
bool allow_smem(Kernel kernel, std::once_flag (&once)[64], bool (&ready)[64]) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  std::call_once(once[dev], [&] {
    ready[dev] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMost) == cudaSuccess;
    cudaGetLastError();
  });
  return ready[dev];
}

template <typename XT, int kCols, int kTokens>
int launch_linear_of(LinearParams p, cudaStream_t st) {
  static std::once_flag once[64];
  static bool ready[64];
  static ResidentClusters counts[kMaxSplit + 1][64];
  if (!allow_smem(w4a16_linear_kernel<XT, kCols, kTokens>, once, ready)) return B200FP4_STATUS_EXECUTION_FAILED;
  // Blocks that share the k of an item in a cluster: a shorter k leaves room for more rows, and few strips reach all SMs
  float best = 1e30f;
  unsigned grid = 0;
  uint32_t smem = 0;
  LinearParams chosen = p;
  for (int split = 1; split <= kMaxSplit && split <= p.units; split *= 2) {
    const int clusters = split == 1 ? sm_count() : resident_clusters_of(counts[split], w4a16_linear_kernel<XT, kCols, kTokens>, split, kThreads, kSmemMost);
    if (clusters < 1) break;
    const int own = (p.units + split - 1) / split;
    const uint32_t row_bytes = (uint32_t)own * (kUnitK * 2) + 16;
    // Rows of fewer tokens where there is no room for all; tokens of a block of k a column are there together or not at all.
    for (int cap = std::min(8 * kCols, p.M); cap >= std::max(1, kTokens); cap /= 2) {
      const int64_t items = (int64_t)((p.M + cap - 1) / cap) * p.strips;
      if (items > 0x3FFFFFFF) break;
      const int used = (int)std::min<int64_t>(clusters, items), most = (int)((items + used - 1) / used);
      const uint64_t bytes = (uint64_t)linear_layout(kCols, cap, row_bytes, 1, 0).bytes + (split > 1 ? (uint64_t)most * cap * 128 : 0);
      if ((uint64_t)own * 256 > kSmemMost || bytes > kSmemMost) continue;
      if (kTokens == 0 && p.out_dtype == B200FP4_DTYPE_F32 && own > kWarpChain * kWarps) continue;       // too long a chain for an f32 result
      // The busiest block's units; a cluster's exchange costs some 1500 cycles.  Shared / not shared, us: M=1 N=512 K=16384 6.2 / 8.9, M=8 N=512
      // K=4096 4.7 / 6.1; by this rule not shared: M=1 N=K=4096 5.2, N=14336 K=4096 9.2.
      const int log_share = share_of(most, p.units / split, kTokens > 0 ? 0 : least_share(p.out_dtype, own));
      const float cost = share_cost(most, own, log_share) + (split > 1 ? 1500.f : 0.f);
      if (cost < best) {
        best = cost;
        chosen.split = split;
        chosen.cap = cap;
        chosen.per = (int)(items / used);
        chosen.more = (int)(items % used);
        chosen.log_share = log_share;
        grid = (unsigned)(used * split);
        smem = (uint32_t)bytes;
      }
      break;
    }
  }
  if (grid == 0) return B200FP4_STATUS_NOT_SUPPORTED;
  if (launch_pdl_cluster(chosen.split, w4a16_linear_kernel<XT, kCols, kTokens>, dim3(grid), dim3(kThreads), smem, st, chosen) != cudaSuccess) {
    cudaGetLastError();
    return B200FP4_STATUS_EXECUTION_FAILED;
  }
  return finish_launch(1);
}

// Up to eight tokens fill the columns of one instruction; with up to sixteen, two of them, the tcgen05 kernel is the faster one but for the smallest
// weights: M=16, us from Python, this / that: N=K=2048 5.7 / 5.9, N=3001 K=4144 9.7 / 7.9, N=K=4096 10.1 / 8.1, N=14336 K=4096 19.7 / 15.1.
bool few_tokens(const LinearCall& c) { return c.M <= 8 || (c.M <= 16 && strips_of(c.N) * units_of(c.K) <= 1536); }

template <typename T>
int launch_linear(const LinearCall& c, cudaStream_t st) {
  LinearParams p = {};
  p.x = c.x;
  p.ldx = c.ldx;
  p.packed = c.packed;
  p.tail = c.tail;
  p.tag = size_tag(c.N, c.K, 0);
  p.g = c.g;
  p.out = c.out;
  p.out_dtype = c.out_dtype;
  p.bias = c.bias;
  p.bias_dtype = c.bias_dtype;
  p.M = (int)c.M;
  p.N = (int)c.N;
  p.K = (int)c.K;
  p.strips = (int)strips_of(c.N);
  p.units = (int)units_of(c.K);
  p.status = c.status;
  // One or two tokens, a block of k a column / a token a column, us: N=14336 K=4096 9.2 / 10.0 for one and 9.8 / 10.0 for two, N=K=2048 the same.
  if (p.M == 1) return launch_linear_of<T, 1, 1>(p, st);
  if (p.M == 2) return launch_linear_of<T, 1, 2>(p, st);
  return p.M <= 8 ? launch_linear_of<T, 1, 0>(p, st) : launch_linear_of<T, 2, 0>(p, st);
}

// ------------------------------------------------------------------------------------------ mixture of experts

constexpr int kMaxPairs = 2048;                // pairs whose slots a block finds in its shared memory; more are done in turns
constexpr int kMaxExperts = 4096;

struct MoeParams {
  const void* x;              // gate/up [M, K], rows ldx apart; down: the rows of act
  int64_t ldx;
  const uint8_t* packed;
  const float* g;             // [E]; gate/up [E][gate, up]
  const uint2* peaks;         // gate/up: [E][gate, up]
  const uint32_t *tail13, *tail2;        // behind the units of both projections
  uint32_t tag13, tag2;
  int M, N, K;
  int strips, units;
  int cap, rows;              // columns of a slot; rows that there is room for
  uint64_t phases;
  int split;                  // whole strips: blocks of a cluster, which share the slots of a strip
  float rcp_topk, rcp_grid, rcp_strips;
  const int32_t* ids;         // [M, topk]
  const float* weights;       // [M, topk]
  const int32_t* map;         // [global_E] or null
  int64_t global_E;
  int topk, E, weight_on_input;
  __half* act;                // gate/up out: for each pair, rows act_row(I) apart, [part][I] and the levels of its runs (run_at)
  float* act_inv;             // [pair]: the reciprocal of the factor that brought its row of act into f16's range
  float* y;                   // down: [pair][N]
  uint32_t* said;             // by gate/up: `call` of the last call with a run above level 0 | whether the weights have the call's sizes
  uint32_t call;
  int* counters;              // [strips of down]
  int n_counters;
  void* out;                  // down [M, N]
  int out_dtype;
  int* status;
  int clear_status;
};

// ---- the value between the projections
//
// SiLU(gate) * up of a pair is brought below 2^15 by a power of two that goes by a bound, known before any of its values is.  Then it is two f16, v =
// upper + lower * 2^-12: the rest of the upper part is at most 2^-12 of it, so that the lower part uses f16's range too, and a value is off by the
// larger of 2^-37 and 2^-23 of itself. A bound may be far from the values (gates of -30: SiLU is 2^-38 of them).  So each run of eight has a level:
// 2^(28 k) more, with the least k that brings its largest value to 2^-13 or above, where it is off by 2^-24 of that at most.  A level is kept as a
// bit, 1 << k, none for a run of zeros.  Ordinary layers have no run above level 0; a word says whether a call has one, and only then the second
// projection looks at the levels: runs of the level above a pair's lowest are brought down to that and split anew, higher ones are less than 2^-28 of
// the pair's largest value and left out.
// One f16 of eleven bits instead (bf16 results are then off by 8e-4 of their norm more): 32 tokens, ten of 512 experts, H=2048 I=512, 94 us against
// 99; 128 tokens 187 / 200; one 14.1 / 14.9.  With the same inputs in every call 32 tokens take 90.2; with a power of two of its own for each run,
// applied to every operand, 93.8; where the loops that do without levels look at them 94.3.
constexpr int kLevel = 28, kLevels = 8;
constexpr float kLeast = 0x1p-13f, kLower = 4096.f;
__host__ __device__ __forceinline__ int64_t act_row(int64_t I) { return 2 * I + units_of(I) * 8; }      // halves of a pair: two parts, and 16 bytes for each 128 values
// Where the level of run n (values 8 n to 8 n + 7) is: lane l of the second projection has its four of a unit in a word, [block l % 4][half of the
// unit][eight of the block]
__device__ __forceinline__ int run_at(int n) { return (n >> 4) * 16 + ((n >> 1) & 3) * 4 + ((n >> 3) & 1) * 2 + (n & 1); }

// A lane's eight values of a run, the upper parts or (odd) the lower ones, from one level to the one below it: times 2^-28.  Lanes apart by four have
// the two parts.
__device__ __forceinline__ void level_down(uint32_t* b, bool odd, int levels) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, b[j], 4);
    const float2 hi = __half22float2(as_half2(odd ? other : b[j])), lo = __half22float2(as_half2(odd ? b[j] : other));
    const float2 v = make_float2((hi.x + lo.x * (1.f / kLower)) * 0x1p-28f, (hi.y + lo.y * (1.f / kLower)) * 0x1p-28f);
    const __half2 upper = __floats2half2_rn(v.x, v.y);
    const float2 f = __half22float2(upper);
    const uint32_t next = odd ? as_u32(__floats2half2_rn((v.x - f.x) * kLower, (v.y - f.y) * kLower)) : as_u32(upper);
    if (levels > 0) b[j] = levels == 1 ? next : 0u;
  }
}

struct RowStat {
  float inv, act;             // the reciprocal of the row's factor; what brings the pair's row of act into f16's range
};
// Shared memory behind the rings and barriers: partial sums of warps | expert of a pair | pairs by expert, and as they came | first place of an
// expert | slots | scan | routing weights (down) | statistics of the staged rows | parts of those | the rows in f16, and before them an expert's
// pairs | products of whole strips
struct MoeLayout {
  uint32_t red, expert, list, came, start, slots, scan, weights, stats, parts, rows, y, bytes;
};
__host__ __device__ __forceinline__ MoeLayout moe_layout(int cols, int pairs, int E, int cap, int rows, uint32_t row_bytes, int whole_strips) {
  MoeLayout l;
  l.red = pad16(ring_bytes(cols) + bar_bytes(cols));
  l.expert = l.red + red_bytes(cols);
  l.list = pad16(l.expert + (uint32_t)pairs * 2);
  l.came = pad16(l.list + (uint32_t)pairs * 2);
  l.start = pad16(l.came + (uint32_t)pairs * 2);
  l.slots = pad16(l.start + (uint32_t)E * 2);
  l.scan = pad16(l.slots + (uint32_t)((pairs < E ? pairs : E) + pairs / cap) * 8);
  l.weights = l.scan + 36 * 4;
  l.stats = pad16(l.weights + (rows > 0 ? 0 : (uint32_t)pairs * 4));
  l.parts = pad16(l.stats + (uint32_t)rows * sizeof(RowStat));
  l.rows = l.parts + kWarps * 8;
  const uint32_t counts = pad16((uint32_t)E * 4), staged = (uint32_t)rows * row_bytes;
  l.y = l.rows + (counts > staged ? counts : staged);
  l.bytes = l.y + (uint32_t)whole_strips * pairs * 128;
  return l;
}

// n / d for 0 <= n, given 1 / d: a float's product is off by less than one for n below 2^22
__device__ __forceinline__ int quotient(int n, int d, float rcp) {
  if (n >= 1 << 22) return n / d;
  int q = __float2int_rz(__int2float_rn(n) * rcp);
  const int r = n - q * d;
  q += r >= d ? 1 : 0;
  q -= r < 0 ? 1 : 0;
  return q;
}

// Items of a block of the down projection, of the pairs' slots and the strips of the result: a run of all of them, strip by strip; or a cluster has
// whole strips and each of its blocks some of the slots.
struct DownItems {
  int first, last, fast;      // items; slots of a strip
  int strip0, strip_step, slot0;
  __device__ __forceinline__ void of(int block, int grid, float rcp_grid, int n_slots, int strips, int split, bool whole) {
    strip0 = slot0 = 0;
    strip_step = 1;
    fast = n_slots;
    if (whole) {
      const int cluster = block / split, clusters = grid / split, rank = block & (split - 1);
      slot0 = n_slots * rank / split;
      fast = n_slots * (rank + 1) / split - slot0;
      strip0 = cluster;
      strip_step = clusters;
      first = 0;
      last = cluster < strips ? (strips - cluster + clusters - 1) / clusters * fast : 0;
    } else {
      const int n = n_slots * strips, per = quotient(n, grid, rcp_grid), more = n - per * grid;
      first = block * per + min(block, more);
      last = first + per + (block < more ? 1 : 0);
    }
  }
};

__device__ __forceinline__ int local_expert(const MoeParams& p, int pair) {
  int64_t e = p.ids[pair];
  if (p.map != nullptr) e = e >= 0 && e < p.global_E ? p.map[e] : -1;
  return e >= 0 && e < p.E ? (int)e : -1;
}

// An expert's pairs to zero; needs nothing of the call's inputs
__device__ __forceinline__ void clear_counts(const MoeParams& p, unsigned char* smem, const MoeLayout& l) {
  if (p.M * p.topk <= 32) return;                  // found without
  for (int i = threadIdx.x; i < p.E; i += kThreads) reinterpret_cast<int*>(smem + l.rows)[i] = 0;
}

// Slots (expert | pairs << 16, first place in the list): runs of at most `cap` pairs of one expert, experts in order and pairs in theirs.  Every
// block finds the same ones, whatever the order in which its threads run: pairs are counted and gathered by expert as they come, and then each takes
// the place that the number of smaller ones in its expert's run gives it.  Returns the number of slots.
__device__ __forceinline__ int find_slots(const MoeParams& p, unsigned char* smem, const MoeLayout& l) {
  constexpr int kMost = kMaxPairs / kThreads;
  const int cap = p.cap, P = p.M * p.topk, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint16_t* const expert = reinterpret_cast<uint16_t*>(smem + l.expert);
  uint16_t* const list = reinterpret_cast<uint16_t*>(smem + l.list);
  uint16_t* const came = reinterpret_cast<uint16_t*>(smem + l.came);
  uint16_t* const start = reinterpret_cast<uint16_t*>(smem + l.start);
  int2* const slots = reinterpret_cast<int2*>(smem + l.slots);
  uint32_t* const scan = reinterpret_cast<uint32_t*>(smem + l.scan);
  int* const count = reinterpret_cast<int*>(smem + l.rows);
  if (P <= 32) {
    // Every warp finds all of them and writes the same; slots in the order of their first pairs.
    const int e = lane < P ? local_expert(p, lane) : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1)), chunk = before / cap, place = before - chunk * cap;
    const bool leads = e >= 0 && place == 0;
    const int size = leads ? min(cap, __popc(same) - before) : 0;
    const uint32_t leaders = __ballot_sync(0xffffffffu, leads);
    int first = size;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int a = __shfl_up_sync(0xffffffffu, first, d);
      if (lane >= d) first += a;
    }
    first -= size;
    uint32_t rest = same;
    for (int c = 0; c < before - place; ++c) rest &= rest - 1;
    const int at = __shfl_sync(0xffffffffu, first, e >= 0 ? __ffs((int)rest) - 1 : 0) + place;
    if (lane < P) expert[lane] = (uint16_t)e;
    if (leads) slots[__popc(leaders & ((1u << lane) - 1))] = make_int2(e | (size << 16), first);
    if (e >= 0) list[at] = (uint16_t)lane;
    __syncwarp();
    return __popc(leaders);
  }
  int e[kMost], at[kMost];
#pragma unroll
  for (int q = 0; q < kMost; ++q) {
    const int i = q * kThreads + threadIdx.x;
    e[q] = i < P ? local_expert(p, i) : -1;
  }
  __syncthreads();                                 // the counts are clear
#pragma unroll
  for (int q = 0; q < kMost; ++q) {
    const int i = q * kThreads + threadIdx.x;
    if (i < P) expert[i] = (uint16_t)e[q];
    at[q] = e[q] >= 0 ? atomicAdd(&count[e[q]], 1) : 0;
  }
  __syncthreads();
  // a run of experts a thread; their pairs | slots << 16, and an exclusive scan of those over the threads
  const int per = (p.E + kThreads - 1) / kThreads, e0 = min(p.E, (int)threadIdx.x * per), e1 = min(p.E, e0 + per);
  uint32_t mine = 0;
  for (int x = e0; x < e1; ++x) mine += (uint32_t)count[x] | ((uint32_t)(count[x] + cap - 1) / cap << 16);
  uint32_t sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += a;
  }
  if (lane == 31) scan[warp] = sum;
  __syncthreads();
  uint32_t warps = lane < kWarps ? scan[lane] : 0;
#pragma unroll
  for (int d = 1; d < kWarps; d *= 2) {
    const uint32_t a = __shfl_up_sync(0xffffffffu, warps, d);
    if (lane >= d) warps += a;
  }
  const uint32_t others = __shfl_sync(0xffffffffu, warps, warp > 0 ? warp - 1 : 0);
  const int total = (int)(__shfl_sync(0xffffffffu, warps, kWarps - 1) >> 16);
  uint32_t next = sum - mine + (warp > 0 ? others : 0);
  for (int x = e0; x < e1; ++x) {
    const int pairs = count[x], first = next & 0xFFFF;
    int slot = next >> 16;
    start[x] = (uint16_t)first;
    for (int c = 0; c < pairs; c += cap) slots[slot++] = make_int2(x | (min(cap, pairs - c) << 16), first + c);
    next = (next & 0xFFFF0000u) + ((uint32_t)(slot - (int)(next >> 16)) << 16) + first + pairs;
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kMost; ++q)
    if (e[q] >= 0) came[start[e[q]] + at[q]] = (uint16_t)(q * kThreads + threadIdx.x);
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kMost; ++q) {
    if (e[q] < 0) continue;
    const int i = q * kThreads + threadIdx.x, first = start[e[q]], n = count[e[q]];
    int place = first;
    for (int j = first; j < first + n; ++j) place += came[j] < i;
    list[place] = (uint16_t)i;
  }
  __syncthreads();
  return total;
}

enum Projection { kGateUp, kDownItems, kDownStrips };       // kDownStrips: whole strips

// Bound by the copies of the experts that the routing reaches: 32 tokens, ten of 512 experts, H=2048 I=512, take 99 us with inputs that change from
// call to call, of which their 420 MB would take 66 at the copy rate; finding the slots takes 2, rows and first units 3, the down projection's start 3
// and the strips' last sums 4.  Alone and cold gate/up takes 57 us and down 44.  128 tokens 200.  The kernels over items are at the limit of 128
// registers and spill (12 bytes stored, 28 loaded).
// A prompt goes through in turns of kMaxPairs pairs, each of which reads the experts again: 8192 tokens 9.7 ms.
// Two launches: every value of the first projection is needed by the second, which finds its slots and asks for its first weights while the first one
// ends.
// XT: type of the activations (gate/up); kCols: columns of eight; kChains: sums of more than a chain, for an f32 result (as a choice at run time it
// cost the others 5 to 9 %)
template <typename XT, int kMode, int kCols, bool kChains>
__global__ void __launch_bounds__(kThreads, 1) w4a16_moe_kernel(const MoeParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr bool kDown = kMode != kGateUp, kWhole = kMode == kDownStrips;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row8 = lane >> 2, quad = lane & 3;
  const uint32_t base = smem_u32(smem), chunk = chunk_at(row8, quad);
  const uint32_t row_bytes = (uint32_t)p.units * (kUnitK * 2) + 16;      // rows are shifted by 16 bytes against each other: no two lanes of a load meet
  const MoeLayout l = moe_layout(kCols, p.M * p.topk, p.E, p.cap, p.rows, row_bytes, 0);
  const uint16_t* const expert = reinterpret_cast<const uint16_t*>(smem + l.expert);
  const int2* const slots = reinterpret_cast<const int2*>(smem + l.slots);
  const uint16_t* const list = reinterpret_cast<const uint16_t*>(smem + l.list);
  Ring<stages_of(kCols)> ring;
  ring.init(base, base + ring_bytes(kCols), warp, lane);
  if (kWhole && p.split > 1) cluster_arrive_relaxed();     // the other blocks run before anything is sent to them
  // The routing is not the first projection's work, and its kernel lets this one start only once what came before it is complete: the second
  // projection finds its slots and asks for its first weights while the first one ends.
  clear_counts(p, smem, l);
  if (!kDown) {
    pdl_wait();
    pdl_launch_dependents();
  }
  // the weights are on their way with the ids
  float weight[kDown ? kMaxPairs / kThreads : 1];
  if constexpr (kDown)
#pragma unroll
    for (int q = 0; q < kMaxPairs / kThreads; ++q) {
      const int i = q * kThreads + threadIdx.x;
      weight[q] = i < p.M * p.topk && !p.weight_on_input ? p.weights[i] : 1.f;
    }
  // one thread of gate/up compares the weights' sizes with the call's
  const bool compares = !kDown && blockIdx.x == 0 && threadIdx.x == kThreads - 1;
  const uint32_t tail13 = compares ? *p.tail13 : 0, tail2 = compares ? *p.tail2 : 0;
  const int n_slots = find_slots(p, smem, l);
  if (compares) {
    const bool fits = packed_for(tail13, p.tag13) && packed_for(tail2, p.tag2);
    p.said[1] = fits;
    if (!fits) *p.status = kOtherSizes;
    else if (p.clear_status) *p.status = 0;
  }
  if constexpr (kDown)
#pragma unroll
    for (int q = 0; q < kMaxPairs / kThreads; ++q) {
      const int i = q * kThreads + threadIdx.x;
      if (i < p.M * p.topk) reinterpret_cast<float*>(smem + l.weights)[i] = weight[q];
    }
  // Items (strip, slot) of a slot are neighbours, or (down) those of a strip
  DownItems d;
  if constexpr (kDown) {
    d.of(blockIdx.x, gridDim.x, p.rcp_grid, n_slots, p.strips, p.split, kWhole);
  } else {
    const int n = n_slots * p.strips, per = quotient(n, gridDim.x, p.rcp_grid), more = n - per * (int)gridDim.x;
    d.first = (int)blockIdx.x * per + min((int)blockIdx.x, more);
    d.last = d.first + per + ((int)blockIdx.x < more ? 1 : 0);
    d.fast = p.strips;
  }
  const int first = d.first, last = d.last, fast = d.fast;
  const float rcp_fast = kDown ? __frcp_rn((float)fast) : p.rcp_strips;
  // Gate/up: rows are staged for as many slots at a time as there is room for: a turn's items end before slot stop
  auto turn_of = [&](int slot, int& n_rows) {
    int stop = slot + 1;
    n_rows = slots[slot].x >> 16;
#pragma unroll 1
    while (stop < n_slots && stop * fast < last && n_rows + (slots[stop].x >> 16) <= p.rows) n_rows += slots[stop++].x >> 16;
    return stop;
  };
  // This warp's part of an item
  struct Part {
    int group, in_group, k_first, n_units;
  };
  auto part_of = [&](int log_share) {
    Part part;
    part.group = warp >> log_share;
    part.in_group = warp & ((1 << log_share) - 1);
    part.k_first = (p.units * part.in_group) >> log_share;
    part.n_units = ((p.units * (part.in_group + 1)) >> log_share) - part.k_first;
    return part;
  };
  // Weights are asked for ahead of the items, in the same order
  int ahead = first, ahead_share = 4, phase_end = first, turn_end = kDown ? last : first, ahead_left = 0, src_step = 0;
  const uint8_t* src = nullptr;
  auto fetch = [&]() {
    if (__builtin_expect(ahead_left == 0, 0)) {
      ahead += kWarps >> ahead_share;
#pragma unroll 1
      while (ahead >= phase_end) {
        if (phase_end >= last) return;
        if (!kDown && phase_end == turn_end) {
          int n_rows;
          turn_end = min(last, turn_of(quotient(phase_end, fast, rcp_fast), n_rows) * fast);
        }
        const Phase phase = next_phase(turn_end - phase_end, p.phases);
        ahead_share = phase.share;
        ahead = phase_end + (warp >> ahead_share);
        phase_end += phase.count;
      }
      const Part part = part_of(ahead_share);
      const int hi = quotient(ahead, fast, rcp_fast), lo = ahead - hi * fast;
      const int e = slots[kDown ? d.slot0 + lo : hi].x & 0xFFFF, strip = kDown ? d.strip0 + hi * d.strip_step : lo;
      src = p.packed + (size_t)(e * p.strips * p.units + strip_at(strip, p.strips, p.units, part.k_first, src_step)) * kUnitBytes;
      ahead_left = part.n_units;
    }
    ring.ask(src, lane);
    src += src_step * kUnitBytes;
    --ahead_left;
  };
  float* const red = reinterpret_cast<float*>(smem + l.red);
  // units(from, to): some of an item's part; their sums in acc
  auto in_chains = [&](const Part& part, float (&acc)[2][kCols][4], auto&& units) {
    if constexpr (kChains) {
      float* const own = red + warp * (2 * kCols * 4 * 32) + lane;
      for (int k = part.k_first, rest = part.n_units;;) {
        const int n = min(rest, kWarpChain);
        units(k, k + n);
        k += n;
        if ((rest -= n) == 0) break;
        put_aside<kCols>(own, k == part.k_first + kWarpChain, acc);
      }
      if (part.n_units > kWarpChain) take_back<kCols>(own, acc);
    } else {
      units(part.k_first, part.k_first + part.n_units);
    }
  };

  if constexpr (!kDown) {
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; i < p.n_counters; i += kThreads) p.counters[i] = 0;
    }
    RowStat* const stats = reinterpret_cast<RowStat*>(smem + l.stats);
    // slots [slot, stop) of a turn, the pairs in places [row0, row0 + n_rows) of the list
    StagedRows<XT, true> staged;
    int slot = last > first ? quotient(first, fast, rcp_fast) : 0;
    for (int end = first; end < last;) {
      int n_rows, done = end;
      const int row0 = slots[slot].y, stop = turn_of(slot, n_rows);
      if (end > first) __syncthreads();            // nobody reads the rows before these any more
      auto row_at = [&](int r) { return static_cast<const XT*>(p.x) + (int64_t)quotient(list[row0 + r], p.topk, p.rcp_topk) * p.ldx; };
      staged.ask(n_rows, 0, p.K, row_at);
      float2 g = {0.f, 0.f}, peak = {0.f, 0.f};
      float w = 1.f;
      const int own = (int)threadIdx.x < n_rows ? list[row0 + threadIdx.x] : -1;
      if (own >= 0) {
        g = reinterpret_cast<const float2*>(p.g)[expert[own]];
        const uint2 words = p.peaks[expert[own]];
        peak = make_float2(peak_of(words.x), peak_of(words.y));
        if (p.weight_on_input) w = p.weights[own];
      }
      if (end == first)
#pragma unroll 1
        for (int i = 0; i < stages_of(kCols); ++i) fetch();
      end = min(last, stop * fast);
      slot = stop;
      staged.finish(p.units * kUnitK, smem + l.rows, row_bytes, reinterpret_cast<float2*>(smem + l.parts), row_at,
                    [&](int r, float inv, float squares) { stats[r] = {inv, squares}; });
      __syncthreads();
      if (own >= 0) {
        // |gate|, |up| <= |x| * sqrt(K) * the matrix's largest magnitude, and |SiLU(gate)| <= |gate|.  The product is brought below 2^15; that the
        // bound is far above the values costs little: f16 reaches 40 binades down.
        // Where the squares have left f32's range, |x| <= 2^16 inv sqrt(K) is the bound that is left.
        const float squares = stats[threadIdx.x].act, root = sqrtf((float)p.K);
        const float norm = (squares > 1e-30f && squares < 1e30f ? sqrtf(squares) : 65536.f * stats[threadIdx.x].inv * root) * root * w;
        const float bound = fabsf(norm * (g.x * peak.x)) * fabsf(norm * (g.y * peak.y));
        const int up = min(14 - ((int)(__float_as_uint(bound) >> 23) - 126), 100);        // from -115, an infinite bound
        stats[threadIdx.x].act = pow2(up);
        p.act_inv[own] = pow2(-up);
      }
      __syncthreads();
      while (done < end) {
        const Phase phase = next_phase(end - done, p.phases);
        const Part part = part_of(phase.share);
        for (int item = done + part.group; item < done + phase.count; item += kWarps >> phase.share) {
          const int hi = quotient(item, fast, rcp_fast), strip = item - hi * fast;
          const int2 s = slots[hi];
          const int n = s.x >> 16, e = s.x & 0xFFFF;
          uint32_t col[kCols];
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            const int i = c * 8 + row8;              // columns past the slot's pairs read the first one's row: nobody reads their sums
            col[c] = base + l.rows + (s.y - row0 + (i < n ? i : 0)) * row_bytes + quad * 32;
          }
          float acc[2][kCols][4] = {};
          in_chains(part, acc, [&](int k, int end) {
#pragma unroll 1
            for (; k < end; ++k) {
              uint32_t b[2][kCols][8];
              staged_columns<kCols>(col, k * (kUnitK * 2), b);
              multiply_unit<kCols>(ring.wait(p.status), lane, chunk, b, acc);
              ring.advance();
              if (ring.ok) fetch();
            }
          });
          const float g_gate = p.g[2 * e], g_up = p.g[2 * e + 1];
          finish_item<kCols, false>(red, phase.share, part.in_group, part.group, lane, acc, [&](int t, int c, int i, float gate, float up, auto again) {
            // a run: eight rows of a tile, a column; I is a multiple of 16, so that it is whole
            const int column = c * 8 + quad * 2 + i, I = p.N / 2, run = strip * 2 + t;
            const bool here = column < n && run * 8 < I;
            float v = 0.f, scale = 1.f;
            int pair = 0;
            if (here) {
              pair = list[s.y + column];
              const RowStat st = stats[s.y - row0 + column];
              const float f = p.weight_on_input ? p.weights[pair] * st.inv : st.inv;
              v = silu_f32(gate * f * g_gate) * (up * f * g_up);
              scale = st.act;
            }
            uint32_t level = 1, large = 15;
            if constexpr (again.value) {
              uint32_t top = __float_as_uint(v) & 0x7FFFFFFFu;
#pragma unroll
              for (int d = 4; d < 32; d *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
              const int power = exponent_of(scale), under = exponent_of(kLeast) - (exponent_of(__uint_as_float(top)) + power);
              const int k = min(max(under + kLevel - 1, 0) / kLevel, min(kLevels - 1, (126 - power) / kLevel));
              scale = pow2(power + k * kLevel);
              level = top != 0 ? 1u << k : 0u;
              if (level > 1 && here) p.said[0] = p.call;
            } else {
              // four runs a warp: level 0 where one of a run's values is large enough
              large = __ballot_sync(0xffffffffu, !here || !(fabsf(v) * scale < kLeast));
              large |= large >> 16;
              large |= large >> 8;
              large |= large >> 4;
            }
            if (here) {
              v *= scale;
              const __half hi = __float2half_rn(v);
              const float rest = (v - __half2float(hi)) * kLower;
              __half* const to = p.act + pair * act_row(I);
              to[run * 8 + row8] = hi;
              to[I + run * 8 + row8] = __float2half_rn(isfinite(rest) ? rest : 0.f);        // an infinite or NaN value is the upper part's alone
              if (row8 == 0) reinterpret_cast<uint8_t*>(to + 2 * I)[run_at(strip * 2) + t] = (uint8_t)level;
            }
            return (large & 15) == 15;
          });
        }
        done += phase.count;
      }
    }
    ring.drain();
  } else {
#pragma unroll 1
    for (int i = 0; i < stages_of(kCols); ++i) fetch();
    pdl_wait();
    pdl_launch_dependents();
    if (kWhole && p.split > 1) cluster_wait();
    const uint2 said = *reinterpret_cast<const uint2*>(p.said);
    const bool leveled = said.x == p.call;           // otherwise every run of every pair is at level 0, and nobody looks
    if (__builtin_expect(said.y == 0, 0))
      for (int i = threadIdx.x; i < p.M * p.topk; i += kThreads) reinterpret_cast<float*>(smem + l.weights)[i] = __int_as_float(0x7FC00000);
    if (n_slots == 0) {
      for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < (size_t)p.M * p.N; i += (size_t)gridDim.x * kThreads)
        store_value(p.out, p.out_dtype, i, 0.f);
      return;
    }
    for (int done = first; done < last;) {
      const Phase phase = next_phase(last - done, p.phases);
      const Part part = part_of(phase.share);
      for (int item = done + part.group; item < done + phase.count; item += kWarps >> phase.share) {
        const int strip_nth = quotient(item, fast, rcp_fast);
        const int2 s = slots[d.slot0 + item - strip_nth * fast];
        const int n = s.x >> 16, e = s.x & 0xFFFF, strip = d.strip0 + strip_nth * d.strip_step;
        const __half* act[kCols];
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int i = (c * 8 + row8) / 2;          // a pair's columns are its parts
          act[c] = static_cast<const __half*>(p.x) + list[s.y + (i < n ? i : 0)] * p.ldx + (row8 & 1) * p.K + quad * 16;
        }
        float acc[2][kCols][4] = {};
        uint32_t b[2][kCols][8];
        auto load_columns = [&](int k, uint32_t(&to)[2][kCols][8]) {
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              const int x = k * kUnitK + half * 64;
              uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
              if (x + quad * 16 < p.K) {
                lo = ld_u4(act[c] + x);
                hi = ld_u4(act[c] + x + 8);
              }
              to[half][c][0] = lo.x, to[half][c][1] = lo.y, to[half][c][2] = lo.z, to[half][c][3] = lo.w;
              to[half][c][4] = hi.x, to[half][c][5] = hi.y, to[half][c][6] = hi.z, to[half][c][7] = hi.w;
            }
        };
        auto multiply = [&]() {
          multiply_unit<kCols>(ring.wait(p.status), lane, chunk, b, acc);
          ring.advance();
          if (ring.ok) fetch();
        };
        // Back to the values' own size: this lane's sums are those of pair c * 4 + quad, lowest_of(c) the level that it was brought to.
        auto scale_sums = [&](auto&& lowest_of) {
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            const int column = c * 4 + quad;
            const float inv = p.act_inv[list[s.y + (column < n ? column : 0)]], f = pow2(exponent_of(inv) - lowest_of(c) * kLevel);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int j = 0; j < 4; ++j) acc[t][c][j] *= j & 1 ? f * (1.f / kLower) : f;
          }
        };
        if (__builtin_expect(leveled, 0)) {
          // four lanes have a pair, each its own words of the levels
          const bool odd = row8 & 1;
          auto levels_at = [&](int k, int c) { return reinterpret_cast<const uint32_t*>(act[c] + (odd ? 1 : 2) * p.K - quad * 16 + k * 8)[quad]; };
          uint32_t levels[kCols];
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            uint32_t set = 0;
            for (int k = part.k_first; k < part.k_first + part.n_units; ++k) {
              const int x = k * kUnitK + quad * 16;
              const uint32_t w = x < p.K ? levels_at(k, c) : 0u;
              set |= x + 64 < p.K ? w : w & 0xFFFFu;
            }
            set |= set >> 16;
            set = (set | set >> 8) & 0xFFu;
            set |= __shfl_xor_sync(0xffffffffu, set, 1);
            levels[c] = set | __shfl_xor_sync(0xffffffffu, set, 2);
          }
          in_chains(part, acc, [&](int k, int end) {
#pragma unroll 1
            for (; k < end; ++k) {
              load_columns(k, b);
#pragma unroll
              for (int c = 0; c < kCols; ++c) {
                const uint32_t w = levels_at(k, c);
#pragma unroll
                for (int run = 0; run < 4; ++run)    // levels above the pair's lowest; values that are zeros stay so
                  level_down(&b[run >> 1][c][(run & 1) * 4], odd, __ffs((int)((w >> (8 * run)) & 0xFFu)) - __ffs((int)levels[c]));
              }
              multiply();
            }
          });
          scale_sums([&](int c) { return max(__ffs((int)__shfl_sync(0xffffffffu, levels[c], quad * 8)) - 1, 0); });
        } else {
          if constexpr (kCols == 1) load_columns(part.k_first, b);       // a unit ahead, as far as there are registers
          in_chains(part, acc, [&](int k, int end) {
#pragma unroll 1
            for (; k < end; ++k) {
              if constexpr (kCols == 1) {
                uint32_t after[2][kCols][8];
                load_columns(k + 1, after);
                multiply();
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                  for (int j = 0; j < 8; ++j) b[half][0][j] = after[half][0][j];
              } else {
                load_columns(k, b);
                multiply();
              }
            }
          });
          scale_sums([](int) { return 0; });
        }
        finish_item<kCols, true>(red, phase.share, part.in_group, part.group, lane, acc, [&](int t, int c, int i, float va, float vb, auto) {
          // the two columns of a pair in one row
          const int column = c * 4 + quad, in_strip = t * 16 + row8 + i * 8;
          if (column >= n) return true;
          const int pair = list[s.y + column];
          const float v = (va + vb) * p.g[e];
          if constexpr (kWhole) {
            // [strip of the cluster][pair][32 rows], in its first block
            const uint32_t to = base + l.y + (uint32_t)((strip_nth * p.M * p.topk + pair) * 32 + in_strip) * 4;
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(p.split > 1 ? map_to_cta(to, 0) : to), "f"(v) : "memory");
          } else if (strip * 32 + in_strip < p.N) {
            p.y[(size_t)pair * p.N + strip * 32 + in_strip] = v;
          }
          return true;
        });
      }
      done += phase.count;
    }
    ring.drain();
    const float* const weights = reinterpret_cast<const float*>(smem + l.weights);
    if constexpr (kWhole) {
      // every token's pairs are added up in the order of the routing
      if (p.split > 1) cluster_sync_any();
      else __syncthreads();
      if ((int)blockIdx.x % p.split != 0 || d.strip0 >= p.strips) return;
      // a warp a token of a strip: its lanes read the routing, then each has a row
      const int P = p.M * p.topk, count = ((p.strips - d.strip0 + d.strip_step - 1) / d.strip_step) * p.M;
      for (int i = warp; i < count; i += kWarps) {
        const int hi = i / p.M, m = i - hi * p.M, row = (d.strip0 + hi * d.strip_step) * 32 + lane;
        const float* const y = reinterpret_cast<const float*>(smem + l.y) + (hi * P + m * p.topk) * 32 + lane;
        float sum = 0.f;
        for (int s0 = 0; s0 < p.topk; s0 += 32) {
          const bool here = s0 + lane < p.topk && expert[m * p.topk + s0 + lane] != 0xFFFF;
          const float own = here ? weights[m * p.topk + s0 + lane] : 0.f;
          for (uint32_t left = __ballot_sync(0xffffffffu, here); left != 0;) {
            float v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {          // four loads before the first is needed
              const int s = left != 0 ? __ffs(left) - 1 : 0;
              const float product = __shfl_sync(0xffffffffu, own, s) * y[(s0 + s) * 32];
              v[u] = left != 0 ? product : 0.f;
              left &= left - 1;
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) sum += v[u];
          }
        }
        if (row < p.N) store_value(p.out, p.out_dtype, (size_t)m * p.N + row, sum);
      }
      return;
    }
    // The block that completes a strip adds up every token's pairs, in the order of the routing.
    int* const done_strips = reinterpret_cast<int*>(smem + l.scan);
    int& n_done = done_strips[32];
    __threadfence();
    __syncthreads();
    if (last == first) return;
    const int strip_first = first / n_slots, strip_end = (last - 1) / n_slots + 1;
    for (int strip0 = strip_first; strip0 < strip_end; strip0 += 32) {
      if (strip0 > strip_first) __syncthreads();
      if (warp == 0) {
        const int strip = strip0 + lane;
        bool mine = false;
        if (strip < strip_end) {
          const int done = min(last, (strip + 1) * n_slots) - max(first, strip * n_slots);
          mine = atomicAdd(&p.counters[strip], done) + done == n_slots;
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, mine);
        __threadfence();
        if (mine) done_strips[__popc(mask & ((1u << lane) - 1))] = strip;
        if (lane == 0) n_done = __popc(mask);
      }
      __syncthreads();
      const int per_strip = p.M * 8, count = n_done * per_strip;
      // four outputs of a token each, two of them and eight of their pairs at a time: all that is asked for is on its way before the first is needed
      for (int i0 = threadIdx.x; i0 < count; i0 += 2 * kThreads) {
        int m[2], row[2];
        bool inside[2];
        float4 sum[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = i0 + h * kThreads, nth = i / per_strip;
          m[h] = (i - nth * per_strip) >> 3;
          row[h] = i < count ? done_strips[nth] * 32 + (i & 7) * 4 : p.N;
          inside[h] = row[h] < p.N;
          sum[h] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        for (int s0 = 0; s0 < p.topk; s0 += 8) {
          float4 v[2][8];
          float w[2][8];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const int pair = m[h] * p.topk + s0 + u;
              v[h][u] = make_float4(0.f, 0.f, 0.f, 0.f);
              w[h][u] = 0.f;
              if (inside[h] && s0 + u < p.topk && expert[pair] != 0xFFFF) {
                v[h][u] = __ldcg(reinterpret_cast<const float4*>(p.y + (size_t)pair * p.N + row[h]));
                w[h][u] = weights[pair];
              }
            }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              sum[h].x += w[h][u] * v[h][u].x;
              sum[h].y += w[h][u] * v[h][u].y;
              sum[h].z += w[h][u] * v[h][u].z;
              sum[h].w += w[h][u] * v[h][u].w;
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!inside[h]) continue;
          const size_t to = (size_t)m[h] * p.N + row[h];
          store_value(p.out, p.out_dtype, to, sum[h].x);
          store_value(p.out, p.out_dtype, to + 1, sum[h].y);
          store_value(p.out, p.out_dtype, to + 2, sum[h].z);
          store_value(p.out, p.out_dtype, to + 3, sum[h].w);
        }
      }
    }
  }
}

struct MoePlan {
  MoeParams p;
  uint32_t smem;
  unsigned grid;
  double items;               // of the busiest block, if the slots are as many as foretold
};

// Slots of a call as far as they can be foretold: what a router without favourites would give
double slots_of(const MoeParams& p, int cap) {
  const double pairs = (double)p.M * p.topk, local = pairs * p.E / (double)(p.map != nullptr ? std::max<int64_t>(p.global_E, p.E) : p.E);
  const double each = std::min(1.0, local / ((double)p.M * p.E)), reached = p.E * (1.0 - std::pow(1.0 - each, p.M));
  return std::max(1.0, std::max(reached, local / cap));
}

// What a launch would be, without launching; a status other than success where there is no room for it
template <typename XT, int kMode, int kCols, bool kChains>
int plan_moe(const MoeParams& given, MoePlan& plan) {
  static std::once_flag once[64];
  static bool ready[64];
  static ResidentClusters counts[kMaxSplit + 1][64];
  constexpr auto kernel = w4a16_moe_kernel<XT, kMode, kCols, kChains>;
  if (!allow_smem(kernel, once, ready)) return B200FP4_STATUS_EXECUTION_FAILED;
  MoeParams p = given;
  const int pairs = p.M * p.topk, sms = sm_count();
  const uint32_t row_bytes = (uint32_t)p.units * (kUnitK * 2) + 16;
  p.cap = kMode == kGateUp ? 8 * kCols : 4 * kCols;
  p.rows = 0;
  p.split = 1;
  while (kMode == kGateUp) {
    // rows that there is room for; a slot has no more columns than that
    const uint32_t rest = moe_layout(kCols, pairs, p.E, p.cap, 0, 0, 0).rows + 16;      // the counts lie where the rows come
    p.rows = rest < kSmemMost ? (int)std::min<uint32_t>((uint32_t)std::min(pairs, kThreads), (kSmemMost - rest) / (row_bytes + (uint32_t)sizeof(RowStat))) : 0;
    if (p.rows < 1) return B200FP4_STATUS_NOT_SUPPORTED;
    if (p.rows >= std::min(p.cap, pairs)) break;
    p.cap = p.rows;
  }
  if ((int64_t)(std::min(pairs, p.E) + pairs / p.cap) * p.strips > 0x3FFFFFFF) return B200FP4_STATUS_NOT_SUPPORTED;
  const double slots = slots_of(p, p.cap);
  int strips = 0;
  double items = slots * p.strips / sms;
  plan.grid = (unsigned)sms;
  if (kMode == kDownStrips) {
    // blocks of a cluster: the fewest items of a block
    items = 1e30;
    for (int split = 1; split <= kMaxSplit; split *= 2) {
      const int clusters = std::min(p.strips, split == 1 ? sms : resident_clusters_of(counts[split], kernel, split, kThreads, kSmemMost));
      if (clusters < 1) break;
      const int own = (p.strips + clusters - 1) / clusters;
      const double most = own * std::ceil(slots / split);
      if (most < items) {
        items = most;
        strips = own;
        p.split = split;
        plan.grid = (unsigned)(clusters * split);
      }
    }
    if (strips == 0) return B200FP4_STATUS_NOT_SUPPORTED;
  }
  plan.smem = moe_layout(kCols, pairs, p.E, p.cap, p.rows, row_bytes, strips).bytes;
  if (plan.smem > kSmemMost) return B200FP4_STATUS_NOT_SUPPORTED;
  plan.items = items;
  p.phases = phase_plan(p.units);
  p.rcp_topk = 1.f / (float)p.topk;
  p.rcp_grid = 1.f / (float)plan.grid;
  p.rcp_strips = 1.f / (float)p.strips;
  plan.p = p;
  return B200FP4_STATUS_SUCCESS;
}

template <typename XT, int kMode, int kCols, bool kChains>
int launch_moe(const MoePlan& plan, cudaStream_t st) {
  if (launch_pdl_cluster(plan.p.split, w4a16_moe_kernel<XT, kMode, kCols, kChains>, dim3(plan.grid), dim3(kThreads), plan.smem, st, plan.p) != cudaSuccess) {
    cudaGetLastError();
    return B200FP4_STATUS_EXECUTION_FAILED;
  }
  return finish_launch(1);
}

// Both projections are planned before the first is launched.
template <typename T, int kUpCols, int kMode, int kDownCols, bool kChains>
int launch_both(const MoeParams& up, const MoeParams& down, cudaStream_t st) {
  MoePlan u, d;
  int rc = plan_moe<T, kGateUp, kUpCols, kChains>(up, u);
  if (rc == B200FP4_STATUS_SUCCESS) rc = plan_moe<__half, kMode, kDownCols, kChains>(down, d);
  if (rc != B200FP4_STATUS_SUCCESS) return rc;
  rc = launch_moe<T, kGateUp, kUpCols, kChains>(u, st);
  return rc == B200FP4_STATUS_SUCCESS ? launch_moe<__half, kMode, kDownCols, kChains>(d, st) : rc;
}

template <typename T, bool kChains>
int launch_layer_of(const MoeParams& up, const MoeParams& down, cudaStream_t st) {
  // Columns of eight, one or two: with two a unit takes half as long again, with one an expert of more pairs than fit (eight; four in the down
  // projection, where a pair has two columns) is read again, mostly from L2.  Columns of gate/up and of down, us, by pairs an expert, bf16; eight
  // experts of 4096, H = 4096: 7.25 pairs 1/1 83.4, 1/2 86.9, 2/1 86.4, 2/2 90.2; 8.5 89.0 / 90.8 / 89.4 / 91.3; 9 94.1 / 96.1 / 93.6 / 95.5; 10 96.3
  // / 96.5 / 95.7 / 96.1; 11 106 / 104 / 100.6 / 99.8.  64 experts of 768, H = 2048: four 51.4 / 56.2 / 60.8 / 69.9; 8.5 74.3 / 75.5 / 75.3 / 81.1; 9
  // 78.3 / 78.0 / 76.6 / 81.3; 10 83.9 / 84.8 / 79.8 / 82.7; 12 93.6 / 92.0 / 90.8 / 90.1.
  const double each = (double)up.M * up.topk / (double)(up.map != nullptr ? std::max<int64_t>(up.global_E, up.E) : up.E);
  if (each > 10.5) return launch_both<T, 2, kDownItems, 2, kChains>(up, down, st);
  if (each > 8.75) return launch_both<T, 2, kDownItems, 1, kChains>(up, down, st);
  // Whole strips: nothing goes through memory and no block waits for a counter, 1.6 us less for one token (H = 2048, ten experts of 512: 14.9 against
  // 16.5), but the blocks' shares are less even.  Items / whole strips, us, by the units that the busiest block has more than its share, eight
  // experts of 4096, H = 4096: 32 units (3 tokens) 38.7 / 37.6, 41 (4) 46.9 / 44.4, 42 (12) 56.2 / 56.3, 43 (20) 65.5 / 66.4, 52 (24) 70.8 / 71.4, 79
  // (29) 83.2 / 84.9; eight of 8192, H = 5120, 6 tokens, 185: 90.0 / 97.9.
  MoePlan strips;
  if (plan_moe<__half, kDownStrips, 1, kChains>(down, strips) == B200FP4_STATUS_SUCCESS &&
      (strips.items - slots_of(down, strips.p.cap) * down.strips / sm_count()) * down.units < 43)
    return launch_both<T, 1, kDownStrips, 1, kChains>(up, down, st);
  return launch_both<T, 1, kDownItems, 1, kChains>(up, down, st);
}
template <typename T>
int launch_layer(const MoeParams& up, const MoeParams& down, cudaStream_t st) {
  const bool chains = down.out_dtype == B200FP4_DTYPE_F32 && std::max(up.units, down.units) > kWarpChain;
  const int rc = chains ? launch_layer_of<T, true>(up, down, st) : launch_layer_of<T, false>(up, down, st);
  if (rc != B200FP4_STATUS_NOT_SUPPORTED) return rc;
  // Long rows: rings and sums for two columns leave more room than those for one.  So a last turn of few pairs is never refused where the full ones
  // before it were not.
  return chains ? launch_both<T, 2, kDownItems, 2, true>(up, down, st) : launch_both<T, 2, kDownItems, 2, false>(up, down, st);
}

bool fits_int(int64_t v) { return v >= 0 && v <= 0x7FFFFFFF; }
bool is_16bit(int dtype) { return dtype == B200FP4_DTYPE_F16 || dtype == B200FP4_DTYPE_BF16; }
bool is_dtype(int dtype) { return is_16bit(dtype) || dtype == B200FP4_DTYPE_F32; }
size_t pad256(size_t v) { return (v + 255) / 256 * 256; }


int64_t packed_strips(int64_t N, int gated) { return gated ? (N / 2 + 15) / 16 : strips_of(N); }
size_t unit_bytes(int64_t E, int64_t N, int64_t K, int gated) {
  return (size_t)E * packed_strips(N, gated) * units_of(K) * kUnitBytes;
}

// tokens of a layer whose pairs fit one turn
int64_t turn_of(int64_t M, int64_t topk) { return std::min(M, std::max<int64_t>(1, kMaxPairs / topk)); }

struct MoeScratch {
  size_t act, act_inv, y, counters, said, bytes;
};
MoeScratch moe_scratch(int64_t M, int64_t topk, int64_t H, int64_t I) {
  MoeScratch s;
  const size_t pairs = (size_t)turn_of(M, topk) * topk;
  s.act = 0;
  s.act_inv = s.act + pad256(pairs * act_row(I) * 2);
  s.y = s.act_inv + pad256(pairs * 4);
  s.counters = s.y + pad256(pairs * H * 4);
  s.said = s.counters + pad256((size_t)strips_of(H) * 4);
  s.bytes = s.said + 256;
  return s;
}

}  // namespace
}  // namespace b200fp4

using namespace b200fp4;

extern "C" size_t b200fp4_w4a16_packed_bytes(int64_t E, int64_t N, int64_t K, int gated) {
  if (E < 1 || N < 1 || K < 16 || K % 16 != 0 || (gated && N % 2 != 0)) return 0;
  return unit_bytes(E, N, K, gated) + (size_t)E * (gated ? 2 : 1) * 4;
}

extern "C" int b200fp4_w4a16_pack(const uint8_t* codes, const uint8_t* scales, int64_t E, int64_t N, int64_t K, int gated, uint8_t* packed,
                                  void* stream) {
  if (b200fp4_w4a16_packed_bytes(E, N, K, gated) == 0 || !fits_int(N) || !fits_int(K)) return B200FP4_STATUS_INVALID_VALUE;
  if (codes == nullptr || scales == nullptr || packed == nullptr || !aligned(codes, 8) || !aligned(packed, 16)) return B200FP4_STATUS_INVALID_VALUE;
  PackParams p = {};
  p.codes = codes;
  p.scales = scales;
  p.packed = packed;
  p.strips = packed_strips(N, gated);
  p.units = w4::units_of(K);
  p.N = (int)N;
  p.K = (int)K;
  p.gated = gated != 0;
  const int64_t n = E * p.strips * p.units * 2;
  if ((n + 7) / 8 > 0x7FFFFFFF) return B200FP4_STATUS_NOT_SUPPORTED;
  p.tails = reinterpret_cast<uint32_t*>(packed + unit_bytes(E, N, K, gated));
  if (cudaMemsetAsync(p.tails, 0, (size_t)E * (gated ? 2 : 1) * 4, static_cast<cudaStream_t>(stream)) != cudaSuccess) {
    cudaGetLastError();
    return B200FP4_STATUS_EXECUTION_FAILED;
  }
  w4a16_pack_kernel<<<(unsigned)((n + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(p, n);
  return finish_launch(1);
}

extern "C" int b200fp4_w4a16_linear(const void* x, int x_dtype, int64_t ldx, const uint8_t* packed, const float* g_scale, const void* bias,
                                    int bias_dtype, void* out, int out_dtype, int64_t M, int64_t N, int64_t K, int32_t* status,
                                    void* stream) {
  if (M < 0 || N < 1 || K < 16 || K % 16 != 0) return B200FP4_STATUS_INVALID_VALUE;
  if (!is_16bit(x_dtype) || !is_dtype(out_dtype) || (bias != nullptr && !is_dtype(bias_dtype))) return B200FP4_STATUS_INVALID_VALUE;
  if (M == 0) return B200FP4_STATUS_SUCCESS;
  if (x == nullptr || packed == nullptr || g_scale == nullptr || out == nullptr || status == nullptr) return B200FP4_STATUS_INVALID_VALUE;
  if (!aligned(x, 16) || !aligned(packed, 16) || !aligned(out, 16) || ldx % 8 != 0 || (M > 1 && ldx < K)) return B200FP4_STATUS_INVALID_VALUE;
  if (!fits_int(M) || !fits_int(N + 64) || !fits_int(K + 128)) return B200FP4_STATUS_NOT_SUPPORTED;
  const LinearCall c = {x, x_dtype, ldx, packed, reinterpret_cast<const uint32_t*>(packed + unit_bytes(1, N, K, 0)), g_scale, bias, bias_dtype, out, out_dtype, M, N, K, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (few_tokens(c)) {
    const int rc = x_dtype == B200FP4_DTYPE_BF16 ? launch_linear<__nv_bfloat16>(c, st) : launch_linear<__half>(c, st);
    if (rc != B200FP4_STATUS_NOT_SUPPORTED) return rc;        // rows too long for shared memory (K above some 400,000) are not for this kernel
  }
  return launch_w4a16_gemm(c, st);
}

extern "C" size_t b200fp4_w4a16_moe_workspace_bytes(int64_t M, int64_t topk, int64_t H, int64_t I) {
  if (M < 1 || topk < 1 || H < 1 || I < 1) return 0;
  return moe_scratch(M, topk, H, I).bytes;
}

extern "C" int b200fp4_w4a16_moe(const void* hidden, int h_dtype, const float* topk_weights, const int32_t* topk_ids, const int32_t* expert_map,
                                 int64_t global_E, const uint8_t* w13_packed, const float* w13_g, const uint8_t* w2_packed, const float* w2_g,
                                 void* out, int out_dtype, int64_t M, int64_t topk, int64_t H, int64_t I, int64_t E, int flags, int32_t* status,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || topk < 1 || E < 1 || H < 16 || H % 16 != 0 || I < 16 || I % 16 != 0) return B200FP4_STATUS_INVALID_VALUE;
  if (!is_16bit(h_dtype) || !is_dtype(out_dtype) || (flags & ~B200FP4_MOE_ROUTER_WEIGHT_ON_INPUT) != 0) return B200FP4_STATUS_INVALID_VALUE;
  if (M == 0) return B200FP4_STATUS_SUCCESS;
  if (hidden == nullptr || topk_weights == nullptr || topk_ids == nullptr || w13_packed == nullptr || w13_g == nullptr || w2_packed == nullptr ||
      w2_g == nullptr || out == nullptr || status == nullptr || (expert_map != nullptr && global_E < 1))
    return B200FP4_STATUS_INVALID_VALUE;
  if (!aligned(hidden, 16) || !aligned(w13_packed, 16) || !aligned(w13_g, 8) || !aligned(w2_packed, 16) || !aligned(out, 16)) return B200FP4_STATUS_INVALID_VALUE;
  if (E > kMaxExperts || topk > kMaxPairs || !fits_int(M * topk) || !fits_int(H + 128) || !fits_int(2 * I + 128) || !fits_int(E * (2 * I / 32 + 1) * (H / 128 + 1)) ||
      !fits_int(E * (H / 32 + 1) * (I / 128 + 1)))
    return B200FP4_STATUS_NOT_SUPPORTED;
  if (workspace == nullptr || !aligned(workspace, 256) || workspace_bytes < b200fp4_w4a16_moe_workspace_bytes(M, topk, H, I))
    return B200FP4_STATUS_ALLOC_FAILED;
  const MoeScratch s = moe_scratch(M, topk, H, I);
  unsigned char* const ws = static_cast<unsigned char*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t turn = turn_of(M, topk);
  for (int64_t m = 0; m < M; m += turn) {
    MoeParams p = {};
    p.M = (int)std::min(turn, M - m);
    p.status = status;
    p.clear_status = m == 0;
    p.ids = topk_ids + m * topk;
    p.weights = topk_weights + m * topk;
    p.map = expert_map;
    p.global_E = global_E;
    p.topk = (int)topk;
    p.E = (int)E;
    p.weight_on_input = flags & B200FP4_MOE_ROUTER_WEIGHT_ON_INPUT ? 1 : 0;
    p.act = reinterpret_cast<__half*>(ws + s.act);
    p.act_inv = reinterpret_cast<float*>(ws + s.act_inv);
    p.peaks = reinterpret_cast<const uint2*>(w13_packed + unit_bytes(E, 2 * I, H, 1));
    p.tail13 = reinterpret_cast<const uint32_t*>(p.peaks);
    p.tail2 = reinterpret_cast<const uint32_t*>(w2_packed + unit_bytes(E, H, I, 0));
    p.tag13 = size_tag(2 * I, H, 1);
    p.tag2 = size_tag(H, I, 0);
    p.y = reinterpret_cast<float*>(ws + s.y);
    p.counters = reinterpret_cast<int*>(ws + s.counters);
    p.n_counters = (int)w4::strips_of(H);
    p.said = reinterpret_cast<uint32_t*>(ws + s.said);
    static std::atomic<uint32_t> calls{0};
    p.call = calls.fetch_add(1, std::memory_order_relaxed);
    MoeParams d = p;
    p.x = static_cast<const unsigned char*>(hidden) + (size_t)m * H * 2;
    p.ldx = H;
    p.packed = w13_packed;
    p.g = w13_g;
    p.N = (int)(2 * I);
    p.K = (int)H;
    p.out_dtype = out_dtype;
    p.strips = (int)((I + 15) / 16);
    p.units = (int)w4::units_of(H);
    d.x = p.act;
    d.ldx = act_row(I);
    d.packed = w2_packed;
    d.g = w2_g;
    d.out = static_cast<unsigned char*>(out) + (size_t)m * H * (out_dtype == B200FP4_DTYPE_F32 ? 4 : 2);
    d.out_dtype = out_dtype;
    d.N = (int)H;
    d.K = (int)I;
    d.strips = (int)w4::strips_of(H);
    d.units = (int)w4::units_of(I);
    const int rc = h_dtype == B200FP4_DTYPE_BF16 ? launch_layer<__nv_bfloat16>(p, d, st) : launch_layer<__half>(p, d, st);
    if (rc != B200FP4_STATUS_SUCCESS) return rc;
  }
  return B200FP4_STATUS_SUCCESS;
}
