// Weight-only NVFP4 (w4a16.cuh): the packing of a checkpoint's weights, the linear layer of few tokens, and the mixture-of-experts layer.
//
// One kernel, three uses.  A warp multiplies units of 32 packed rows with up to 8 * kCols columns of activations: codes become the
// 16-bit A operand in registers, the activations of a lane are the B operand as they lie in memory, sums are f32.
//   linear   columns are tokens
//   gate/up  columns are the (token, expert) pairs of one expert; a tile's rows are eight gate rows and the same eight up rows, so that a
//            lane holds both halves of its values and applies SiLU(gate) * up to them
//   down     two columns a pair, the activation's upper and lower part in f16: their sum has 22 bits, so that the value between the projections is
//            not what limits the result
// Work items are (strip of 32 rows, slot); a slot is a run of one expert's pairs that fits the columns.  A block has a contiguous range of them, groups of
// warps take items in turn and split k among themselves.
// The layer is two launches without anything that has to outlast them: both find the slots from the routing by themselves, the first sets the
// counters of the second, in which the block that finishes a strip's last item adds up its pairs in their order.
#include <algorithm>
#include <type_traits>

#include "sm100_ptx.cuh"
#include "w4a16.cuh"

namespace b200fp4 {
namespace {

using namespace w4;

// ------------------------------------------------------------------------------------------ packing

struct PackParams {
  const uint8_t* codes;       // [E, N, K/2]
  const uint8_t* scales;      // [E, N, K/16]
  uint8_t* packed;
  uint32_t* peaks;            // [E], gated [E][gate, up]: behind the units, zeroed before
  int64_t strips, units;
  int N, K, gated;
};

// one warp per tile of a unit
__global__ void __launch_bounds__(256) w4a16_pack_kernel(const PackParams p, int64_t n_tiles) {
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= n_tiles) return;
  const int lane = threadIdx.x & 31, tile = (int)(at & 1);
  const int64_t unit = at >> 1, u = unit % p.units, strip = unit / p.units % p.strips, e = unit / p.units / p.strips;
  uint8_t* const dst = p.packed + unit * kUnitBytes;
  const int64_t row0 = (strip * 2 + tile) * (p.gated ? 8 : 16) + (lane >> 2), step = p.gated ? p.N / 2 : 8, rows = p.gated ? p.N / 2 : p.N;
  uint32_t sc = 0;
  float peak[2] = {0.f, 0.f};
  for (int half = 0; half < 2; ++half) {
    const int64_t k = u * kUnitK + half * 64 + (lane & 3) * 16;
    uint2 word[2];
    for (int r = 0; r < 2; ++r) {
      uint32_t scale = 0;
      uint2 c = make_uint2(0, 0);
      if ((p.gated ? row0 : row0 + r * 8) < rows && k < p.K) {
        const int64_t row = e * p.N + row0 + r * step;
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
    *reinterpret_cast<uint4*>(dst + (tile * 2 + half) * 512 + lane * 16) = make_uint4(word[0].x, word[0].y, word[1].x, word[1].y);
  }
  *reinterpret_cast<uint32_t*>(dst + kUnitScales + lane * 8 + tile * 4) = sc;
  // magnitudes are not negative: their bits order as they do
  for (int r = 0; r <= p.gated; ++r) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(peak[r]));
    if (lane == 0) atomicMax(p.peaks + e * (p.gated + 1) + r, top);
  }
}

// ------------------------------------------------------------------------------------------ products

enum Mode { kLinear, kGateUp, kDown };

constexpr int kWarps = 16, kThreads = 32 * kWarps;
constexpr int kMaxPairs = 2048;                // pairs whose slots a block finds in its shared memory; more are done in turns
constexpr int kMaxExperts = 4096;

struct RowsParams {
  const void* x;              // [M, K], rows ldx apart; down: [pair][upper, lower][K] f16
  int64_t ldx;
  const uint8_t* packed;
  const float* g;             // [E]; gate/up [E][gate, up]
  void* out;                  // linear [M, N]; down [M, N]
  const void* bias;           // [N] or null
  int out_dtype, bias_dtype;
  int M, N, K;
  int strips, units;
  int split;                  // linear: blocks of a cluster, which share the units of an item
  int cap, rows;              // columns of a slot; rows that there is room for
  int* status;
  int clear_status;
  // layer
  const int32_t* ids;         // [M, topk]
  const float* weights;       // [M, topk]
  const int32_t* map;         // [global_E] or null
  int64_t global_E;
  int topk, E, weight_on_input;
  const float* peaks;         // gate/up [E][gate, up]
  __half* act;                // gate/up out
  float* act_inv;             // [pair]: the reciprocal of the factor that brought its row of act into f16's range
  float* y;                   // down: [pair][N]
  int* counters;              // [strips of down]
  int n_counters;
};

// Shared memory of a block.  Rings of weight units, a warp's its own | their barriers | partial sums, two of them in turn | and for the layer: pairs
// an expert has, then where they begin | expert of a pair | its place among that expert's | pairs by expert | slots | scan | and where rows are
// staged: their statistics | parts of those | the rows in f16 | (linear, split) sums of the block's items
struct Layout {
  uint32_t bars, red, count, expert, rank, list, slots, scan, stats, parts, rows, sums, bytes;
};
struct RowStat {
  float inv, act;             // the reciprocal of the row's factor; what brings the pair's row of act into f16's range
};
constexpr uint32_t kSmemMost = 227 * 1024;

__host__ __device__ __forceinline__ uint32_t pad16(uint32_t v) { return (v + 15) / 16 * 16; }
// pairs, E: 0 for a linear layer; rows: staged rows of row_bytes each
__host__ __device__ __forceinline__ Layout layout_of(uint32_t ring, uint32_t bars, uint32_t red, int pairs, int E, int cap, int rows, uint32_t row_bytes,
                                                      uint32_t sums) {
  Layout l;
  l.bars = ring;
  l.red = pad16(l.bars + bars);
  l.count = l.red + red;
  l.expert = l.count + (uint32_t)E * 4;
  l.rank = pad16(l.expert + (uint32_t)pairs * 2);
  l.list = pad16(l.rank + (uint32_t)pairs * 2);
  l.slots = pad16(l.list + (uint32_t)pairs * 2);
  l.scan = l.slots + (pairs > 0 ? (uint32_t)((pairs < E ? pairs : E) + pairs / cap) * 8 : 0);
  l.stats = pad16(l.scan + (pairs > 0 ? 2 * kWarps * 4 + 16 : 0));
  l.parts = l.stats + (uint32_t)rows * sizeof(RowStat);
  l.rows = pad16(l.parts + (rows > 0 ? kWarps * kWarps * 8 : 0));
  l.sums = l.rows + (uint32_t)rows * row_bytes;
  l.bytes = l.sums + sums;
  return l;
}

__device__ __forceinline__ int local_expert(const RowsParams& p, int pair) {
  int64_t e = p.ids[pair];
  if (p.map != nullptr) e = e >= 0 && e < p.global_E ? p.map[e] : -1;
  return e >= 0 && e < p.E ? (int)e : -1;
}

// Slots of at most `cap` pairs of one expert, experts in order and pairs in theirs, so that every block finds the same; returns their number.
// One warp counts, 32 pairs at a time: a few steps for a decode batch, and no order of atomics to depend on.
__device__ int find_slots(const RowsParams& p, unsigned char* smem, const Layout& l, int cap) {
  int* const count = reinterpret_cast<int*>(smem + l.count);
  uint16_t* const expert = reinterpret_cast<uint16_t*>(smem + l.expert);
  uint16_t* const rank = reinterpret_cast<uint16_t*>(smem + l.rank);
  uint16_t* const list = reinterpret_cast<uint16_t*>(smem + l.list);
  int2* const slots = reinterpret_cast<int2*>(smem + l.slots);
  int* const scan = reinterpret_cast<int*>(smem + l.scan);
  const int P = p.M * p.topk, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < p.E; e += kThreads) count[e] = 0;
  for (int i = threadIdx.x; i < P; i += kThreads) {
    const int e = local_expert(p, i);
    expert[i] = (uint16_t)(e < 0 ? 0xFFFF : e);
  }
  __syncthreads();
  if (warp == 0) {
    for (int i = lane; i - lane < P; i += 32) {
      const int e = i < P ? expert[i] : 0xFFFF;
      const uint32_t same = __match_any_sync(0xffffffffu, e), before = same & ((1u << lane) - 1);
      const int seen = e != 0xFFFF ? count[e] : 0;
      __syncwarp();
      if (e != 0xFFFF) {
        rank[i] = (uint16_t)(seen + __popc(before));
        if (before == 0) count[e] = seen + __popc(same);
      }
      __syncwarp();
    }
  }
  __syncthreads();
  // a run of experts a thread: sums, an exclusive scan over the threads, then slots and first places
  const int per = (p.E + kThreads - 1) / kThreads, e0 = min(p.E, (int)threadIdx.x * per), e1 = min(p.E, e0 + per);
  int pairs = 0, n = 0;
  for (int e = e0; e < e1; ++e) {
    pairs += count[e];
    n += (count[e] + cap - 1) / cap;
  }
  int ip = pairs, in = n;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int a = __shfl_up_sync(0xffffffffu, ip, d), b = __shfl_up_sync(0xffffffffu, in, d);
    if (lane >= d) {
      ip += a;
      in += b;
    }
  }
  if (lane == 31) {
    scan[warp] = ip;
    scan[kWarps + warp] = in;
  }
  __syncthreads();
  int total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      ip += scan[w];
      in += scan[kWarps + w];
    }
    total += scan[kWarps + w];
  }
  int at = ip - pairs, slot = in - n;
  for (int e = e0; e < e1; ++e) {
    const int c = count[e];
    for (int i = 0; i < c; i += cap) slots[slot++] = make_int2(e | (min(cap, c - i) << 16), at + i);
    count[e] = at;
    at += c;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < P; i += kThreads)
    if (expert[i] != 0xFFFF) list[count[expert[i]] + rank[i]] = (uint16_t)i;
  __syncthreads();
  return total;
}

__device__ __forceinline__ uint32_t ldg_stream_u32(const void* p) {
  uint32_t v;
  asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ uint4 ld_u4(const void* p) {      // through L1: the warps of a block share activations
  return *static_cast<const uint4*>(p);
}

__device__ __forceinline__ void store_value(void* out, int dtype, size_t at, float v) {
  if (dtype == B200FP4_DTYPE_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else if (dtype == B200FP4_DTYPE_F16) static_cast<__half*>(out)[at] = __float2half_rn(v);
  else static_cast<float*>(out)[at] = v;
}
__device__ __forceinline__ float load_value(const void* p, int dtype, size_t at) {
  if (dtype == B200FP4_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
  if (dtype == B200FP4_DTYPE_F16) return __half2float(static_cast<const __half*>(p)[at]);
  return static_cast<const float*>(p)[at];
}

// ---- powers of two that bring values into f16's range

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127

// The exponent that brings a row whose largest magnitude has these bf16 bits below 2^15.  Rows with infinities or NaN, which only give such
// again, take the least that no finite value overflows with.
__device__ __forceinline__ int row_exponent(uint32_t bits) { return min(141 - min((int)(bits >> 7), 254), 126); }

// Largest magnitude (bf16 bits; bf16 only) and sum of squares (layer only) of elements [k0, k1) of a row, all lanes; k0 and k1 multiples of 8
template <typename T, bool kSquares>
__device__ __forceinline__ float2 row_part(const T* row, int k0, int k1) {
  uint32_t top = 0;
  float sum = 0.f;
  for (int k = k0 + (threadIdx.x & 31) * 8; k < k1; k += 256) {
    const uint4 v = ld_u4(row + k);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) top = __vmaxu2(top, w[j] & 0x7FFF7FFFu);
      if constexpr (kSquares) {
        float2 f;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) f = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
        else f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        sum += f.x * f.x + f.y * f.y;
      }
    }
  }
  top = __reduce_max_sync(0xffffffffu, max(top & 0xFFFFu, top >> 16));
  if constexpr (kSquares)
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  return make_float2(__uint_as_float(top), sum);
}

template <int kCols>
struct Shape {
  static constexpr int kStages = 3;                            // of a warp's ring
  static constexpr uint32_t kRing = kWarps * kStages * kUnitBytes;
  static constexpr uint32_t kBars = kWarps * kStages * 8;
  static constexpr int kSums = 2 * kCols * 4 * 32;             // of a warp
  static constexpr uint32_t kRed = kWarps * kSums * 4;
};

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// a unit's 32 rows times kCols columns of eight; b: the columns' operands, [half][column][8]
template <int kCols>
__device__ __forceinline__ void multiply_unit(uint32_t unit, int lane, const uint32_t (&b)[2][kCols][8], float (&acc)[2][kCols][4]) {
  const uint2 sc = lds64(unit + kUnitScales + lane * 8);
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint4 w = lds128(unit + (t * 2 + half) * 512 + lane * 16);
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

// XT: type of the activations; kCols: columns of eight
template <typename XT, int kMode, int kCols>
__global__ void __launch_bounds__(kThreads, 1) w4a16_rows_kernel(const RowsParams p) {
  extern __shared__ __align__(128) unsigned char smem[];
  using S = Shape<kCols>;
  constexpr bool kConvert = std::is_same<XT, __nv_bfloat16>::value;
  constexpr bool kStaged = kMode != kDown;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row8 = lane >> 2, quad = lane & 3;
  const int cap = p.cap, split = kMode == kLinear ? p.split : 1;
  const int rank = kMode == kLinear ? (int)(blockIdx.x % (unsigned)split) : 0;
  const int unit_first = p.units * rank / split, unit_last = p.units * (rank + 1) / split, own_units = unit_last - unit_first;
  // rows are shifted by 16 bytes against each other: no two lanes of a load meet
  const uint32_t row_bytes = (uint32_t)((p.units + split - 1) / split) * (kUnitK * 2) + 16;
  const Layout l = layout_of(S::kRing, S::kBars, S::kRed, kMode == kLinear ? 0 : p.M * p.topk, kMode == kLinear ? 0 : p.E, cap, p.rows, row_bytes, 0);
  const uint32_t base = smem_u32(smem);
  const int2* const slots = reinterpret_cast<const int2*>(smem + l.slots);
  const uint16_t* const list = reinterpret_cast<const uint16_t*>(smem + l.list);
  const uint32_t ring = base + warp * (S::kStages * kUnitBytes), bars = base + l.bars + warp * (S::kStages * 8);
  if (lane < S::kStages) mbar_init(bars + lane * 8, 1);
  fence_proxy_async_smem();
  __syncwarp();
  pdl_wait();
  pdl_launch_dependents();
  int n_slots;
  if constexpr (kMode == kLinear) {
    n_slots = (p.M + cap - 1) / cap;
    if (p.clear_status && blockIdx.x == 0 && threadIdx.x == 0) *p.status = 0;
  } else {
    n_slots = find_slots(p, smem, l, cap);
    if (kMode == kGateUp && blockIdx.x == 0) {
      if (p.clear_status && threadIdx.x == 0) *p.status = 0;
      for (int i = threadIdx.x; i < p.n_counters; i += kThreads) p.counters[i] = 0;
    }
    if (kMode == kDown && n_slots == 0) {
      for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < (size_t)p.M * p.N; i += (size_t)gridDim.x * kThreads)
        store_value(p.out, p.out_dtype, i, 0.f);
      return;
    }
  }
  // Items of a slot are neighbours, or (down) those of a strip
  const int fast = kMode == kDown ? n_slots : p.strips;
  const int64_t n_items = (int64_t)n_slots * p.strips;
  const unsigned cluster = blockIdx.x / (unsigned)split, clusters = gridDim.x / (unsigned)split;
  const int first = (int)(n_items * cluster / clusters), last = (int)(n_items * (cluster + 1) / clusters);
  const int n_block = last - first;

  // Warps that share an item.  Busy warps take a unit in about 110 cycles of the SM, a warp alone in 350; an item's ending costs a warp that shares it
  // about half a unit.
  int share = 1, best = 0x7FFFFFFF;
  for (int s = 1; s <= kWarps && s <= own_units; s *= 2) {
    const int busy = n_block * (2 * own_units + s), alone = (n_block * s + kWarps - 1) / kWarps * ((own_units + s - 1) / s + 1) * 7;
    const int cost = busy > alone ? busy : alone;
    if (cost < best) {
      best = cost;
      share = s;
    }
  }
  const int group = warp / share, in_group = warp - group * share, n_groups = kWarps / share;
  const int k_first = unit_first + own_units * in_group / share, k_last = unit_first + own_units * (in_group + 1) / share;

  struct Cursor {
    int item, hi, lo;         // hi * fast + lo
  };
  auto start = [&](Cursor& c) {
    c.item = first + group;
    c.hi = c.item / fast;
    c.lo = c.item - c.hi * fast;
  };
  auto next = [&](Cursor& c) {
    c.item += n_groups;
    c.lo += n_groups;
    while (c.lo >= fast) {
      c.lo -= fast;
      ++c.hi;
    }
  };
  auto slot_of = [&](const Cursor& c) { return kMode == kDown ? c.lo : c.hi; };
  auto strip_of = [&](const Cursor& c) { return kMode == kDown ? c.hi : c.lo; };

  // ---- the ring: one lane asks for the units, all wait for them
  Cursor ahead;
  start(ahead);
  int ahead_left = 0;
  uint32_t fill = 0;
  const uint8_t* src = nullptr;
  auto fetch = [&]() {
    if (ahead_left == 0) {
      if (ahead.item >= last) return;
      const size_t e = kMode == kLinear ? 0 : slots[slot_of(ahead)].x & 0xFFFF;
      src = p.packed + ((e * p.strips + strip_of(ahead)) * p.units + k_first) * kUnitBytes;
      ahead_left = k_last - k_first;
      next(ahead);
    }
    if (lane == 0) {
      mbar_expect_tx(bars + fill * 8, kUnitBytes);
      bulk_load_1d(ring + fill * kUnitBytes, src, kUnitBytes, bars + fill * 8);
    }
    src += kUnitBytes;
    --ahead_left;
    if (++fill == S::kStages) fill = 0;
  };
  for (int i = 0; i < S::kStages; ++i) fetch();

  Cursor at;
  start(at);
  uint32_t stage = 0, phase = 0;
  bool ok = true;
  // Rows are staged for as many slots at a time as there is room for
  int slot = kStaged && n_block > 0 ? first / fast : 0;
  for (int end = first; end < last;) {
    int row0 = 0;
    if constexpr (!kStaged) {
      end = last;
    } else {
      // slots [slot, stop), rows [row0, row0 + n_rows) of the tokens or of the pairs by expert
      const int slots_end = (last - 1) / fast + 1;
      int stop = slot + 1, n_rows;
      if constexpr (kMode == kLinear) {
        row0 = slot * cap;
        n_rows = min(cap, p.M - row0);
      } else {
        row0 = slots[slot].y;
        n_rows = slots[slot].x >> 16;
        while (stop < slots_end && n_rows + (slots[stop].x >> 16) <= p.rows) n_rows += slots[stop++].x >> 16;
      }
      end = min(last, stop * fast);
      slot = stop;
      auto row_at = [&](int r) {
        const int64_t row = kMode == kLinear ? row0 + r : list[row0 + r] / p.topk;
        return static_cast<const XT*>(p.x) + row * p.ldx;
      };
      RowStat* const stats = reinterpret_cast<RowStat*>(smem + l.stats);
      float2* const parts = reinterpret_cast<float2*>(smem + l.parts);
      // few rows: several warps a row
      int n_parts = kWarps;
      while (n_parts > 1 && n_parts * n_rows > kWarps) n_parts /= 2;
      const int k_begin = unit_first * kUnitK, k_end = min(p.K, unit_last * kUnitK), octets = (k_end - k_begin) / 8;
      __syncthreads();                             // nobody reads the rows before these any more
      for (int i0 = 0; i0 < n_rows * n_parts; i0 += kWarps) {
        const int i = i0 + warp, r = i / n_parts, part = i - r * n_parts;
        const int k0 = k_begin + octets * part / n_parts * 8, k1 = k_begin + octets * (part + 1) / n_parts * 8;
        const bool work = r < n_rows;
        uint32_t factor = 0;
        if constexpr (kConvert || kMode == kGateUp) {
          float2 v = make_float2(0.f, 0.f);
          if (work) v = row_part<XT, kMode == kGateUp>(row_at(r), k0, k1);
          if (n_parts > 1) {
            if (work && lane == 0) parts[r * n_parts + part] = v;
            __syncthreads();
            if (work) {
              v = make_float2(0.f, 0.f);
              for (int j = 0; j < n_parts; ++j) {
                const float2 u = parts[r * n_parts + j];
                v.x = __uint_as_float(max(__float_as_uint(v.x), __float_as_uint(u.x)));
                v.y += u.y;
              }
            }
          }
          if (work) {
            const int e = kConvert ? row_exponent(__float_as_uint(v.x)) : 0;
            factor = (uint32_t)(e + 127) * 0x00800080u;
            if (part == 0 && lane == 0) {
              RowStat st = {pow2(-e), 0.f};
              if constexpr (kMode == kGateUp) {
                // |gate|, |up| <= |x| * sqrt(K) * the matrix's largest magnitude, and |SiLU(gate)| <= |gate|.  The product is brought below 2^15; that the
                // bound is far above the values costs nothing while act's two parts reach 40 binades down.
                const int pair = list[row0 + r], x = reinterpret_cast<const uint16_t*>(smem + l.expert)[pair];
                const float w = p.weight_on_input ? p.weights[pair] : 1.f;
                const float norm = sqrtf(v.y * (float)p.K) * w;
                const float bound = fabsf(norm * p.g[2 * x] * p.peaks[2 * x]) * fabsf(norm * p.g[2 * x + 1] * p.peaks[2 * x + 1]);
                const int up = min(max(14 - ((int)(__float_as_uint(bound) >> 23) - 126), -100), 100);
                st.act = pow2(up);
                p.act_inv[pair] = pow2(-up);
              }
              stats[r] = st;
            }
          }
        }
        if (work) {
          const XT* const row = row_at(r);
          unsigned char* const to = smem + l.rows + r * row_bytes;
          for (int k = k0 + lane * 8; k < k1; k += 256) {
            uint4 v = ld_u4(row + k);
            if constexpr (kConvert)
              v = make_uint4(bf16_to_f16_pair(v.x, factor), bf16_to_f16_pair(v.y, factor), bf16_to_f16_pair(v.z, factor), bf16_to_f16_pair(v.w, factor));
            *reinterpret_cast<uint4*>(to + (k - k_begin) * 2) = v;
          }
          if (part == n_parts - 1)                 // a unit's k past the row's end
            for (int k = k_end + lane * 8; k < unit_last * kUnitK; k += 256) *reinterpret_cast<uint4*>(to + (k - k_begin) * 2) = make_uint4(0, 0, 0, 0);
        }
      }
      __syncthreads();
    }

    for (; at.item < end; next(at)) {
      const int slot_at = slot_of(at), strip = strip_of(at);
      const int2 s = kMode == kLinear ? make_int2(min(cap, p.M - slot_at * cap) << 16, slot_at * cap) : slots[slot_at];
      const int n = s.x >> 16;                     // columns in use; the others read the first one's row, and nobody reads their sums
      float acc[2][kCols][4];
      uint32_t b[2][kCols][8];
      uint32_t col[kCols];
      const __half* act[kCols];
#pragma unroll
      for (int c = 0; c < kCols; ++c) {
        const int i = c * 8 + row8;
        if constexpr (kStaged) col[c] = base + l.rows + (uint32_t)(s.y - row0 + (i < n ? i : 0)) * row_bytes + (k_first - unit_first) * (kUnitK * 2) + quad * 32;
        else act[c] = static_cast<const __half*>(p.x) + ((int64_t)list[s.y + (i / 2 < n ? i / 2 : 0)] * 2 + (i & 1)) * p.ldx + k_first * kUnitK + quad * 16;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[t][c][j] = 0.f;
      }
      auto load_columns = [&](int k) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
            if constexpr (kStaged) {
              lo = lds128(col[c] + half * 128);
              hi = lds128(col[c] + half * 128 + 16);
            } else if (k * kUnitK + half * 64 + quad * 16 < p.K) {
              lo = ld_u4(act[c] + half * 64);
              hi = ld_u4(act[c] + half * 64 + 8);
            }
            b[half][c][0] = lo.x, b[half][c][1] = lo.y, b[half][c][2] = lo.z, b[half][c][3] = lo.w;
            b[half][c][4] = hi.x, b[half][c][5] = hi.y, b[half][c][6] = hi.z, b[half][c][7] = hi.w;
          }
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          if constexpr (kStaged) col[c] += kUnitK * 2;
          else act[c] += kUnitK;
        }
      };
      for (int k = k_first; k < k_last; ++k) {
        load_columns(k);
        if (ok) ok = mbar_wait(bars + stage * 8, phase, p.status, 61);
        multiply_unit<kCols>(ring + stage * kUnitBytes, lane, b, acc);
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1;
        }
        __syncwarp();                              // every lane has read the stage
        if (ok) fetch();
      }

      // ---- the item's end.  A lane's sums j are row l / 4 (0, 1) or l / 4 + 8 (2, 3) of a tile and columns 2 (l % 4) and the next one.
      const int e = kMode == kLinear ? 0 : s.x & 0xFFFF;
      auto finish = [&](int t, int c, int j, float va, float vb) {
        // va, vb: sums j and j + 2 (gate and up, or rows eight apart); down: the two parts' sums of row j * 8
        const int column = c * 8 + quad * 2;
        if constexpr (kMode == kDown) {
          const int row = strip * 32 + t * 16 + j * 8 + row8;
          if (column / 2 < n && row < p.N) {
            const int pair = list[s.y + column / 2];
            p.y[(size_t)pair * p.N + row] = (va + vb) * (p.act_inv[pair] * p.g[e]);
          }
        } else if (column + j < n) {
          const RowStat st = reinterpret_cast<const RowStat*>(smem + l.stats)[s.y - row0 + column + j];
          if constexpr (kMode == kGateUp) {
            const int pair = list[s.y + column + j], I = p.N / 2, i_at = strip * 16 + t * 8 + row8;
            if (i_at < I) {
              const float f = p.weight_on_input ? p.weights[pair] * st.inv : st.inv;
              const float v = silu_f32(va * f * p.g[2 * e]) * (vb * f * p.g[2 * e + 1]) * st.act;
              const __half hi = __float2half_rn(v);
              const float rest = v - __half2float(hi);
              __half* const to = p.act + (size_t)pair * 2 * I + i_at;
              to[0] = hi;
              to[I] = __float2half_rn(isfinite(rest) ? rest : 0.f);        // an infinite or NaN value is the upper part's alone
            }
          } else {
            const int row = strip * 32 + t * 16 + row8;
            const float f = kConvert ? st.inv : 1.f;
            if (split > 1) {
              float* const to = reinterpret_cast<float*>(smem + l.sums) + ((at.item - first) * cap + column + j) * 32 + t * 16 + row8;
              to[0] = va * f;
              to[8] = vb * f;
            } else {
              const int m = s.y + column + j;
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (row + h * 8 < p.N) {
                  float v = (h ? vb : va) * f * p.g[0];
                  if (p.bias != nullptr) v += load_value(p.bias, p.bias_dtype, row + h * 8);
                  store_value(p.out, p.out_dtype, (size_t)m * p.N + row + h * 8, v);
                }
            }
          }
        }
      };
      if (share == 1) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int j = 0; j < 2; ++j) finish(t, c, j, acc[t][c][kMode == kDown ? 2 * j : j], acc[t][c][kMode == kDown ? 2 * j + 1 : j + 2]);
      } else {
        // [warp][tile][column of eight][j][lane]; each warp adds up and finishes its part
        float* const red = reinterpret_cast<float*>(smem + l.red) + group * share * S::kSums + lane;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) red[in_group * S::kSums + ((t * kCols + c) * 4 + j) * 32] = acc[t][c][j];
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(share * 32) : "memory");
        for (int i = in_group; i < 4 * kCols; i += share) {
          const int j = i & 1, tc = i >> 1;
          const float *a_from = red + (tc * 4 + (kMode == kDown ? 2 * j : j)) * 32, *b_from = a_from + (kMode == kDown ? 32 : 64);
          float va = 0.f, vb = 0.f;
          for (int w = 0; w < share; ++w) {
            va += a_from[w * S::kSums];
            vb += b_from[w * S::kSums];
          }
          finish(tc / kCols, tc % kCols, j, va, vb);
        }
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(share * 32) : "memory");
      }
    }
  }

  if (!ok) {                                       // copies that were asked for land before the block's memory goes
    const long long t0 = clock64();
    while (clock64() - t0 < kWaitCycles / 64) {
    }
  }
  if constexpr (kMode == kLinear) {
    if (split > 1) {
      // the parts of k are added in their order, each block of the cluster some of the items' values
      cluster_sync_any();
      const int count = n_block * cap * 32;
      for (int i = rank * kThreads + threadIdx.x; i < count; i += split * kThreads) {
        const int item = first + i / (cap * 32), column = i / 32 % cap, slot_at = item / fast;
        const int row = (item - slot_at * fast) * 32 + (i & 31), m = slot_at * cap + column;
        if (m >= p.M || row >= p.N) continue;
        float v = 0.f;
        for (int r = 0; r < split; ++r) {
          float u;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u) : "r"(map_to_cta(base + l.sums + i * 4, r)) : "memory");
          v += u;
        }
        v *= p.g[0];
        if (p.bias != nullptr) v += load_value(p.bias, p.bias_dtype, row);
        store_value(p.out, p.out_dtype, (size_t)m * p.N + row, v);
      }
      cluster_sync_any();                          // nobody leaves while its sums are read
    }
  }
  if constexpr (kMode == kDown) {
    // The block that completes a strip adds up every token's pairs, in the order of the routing.
    const uint16_t* const expert = reinterpret_cast<const uint16_t*>(smem + l.expert);
    int* const flag = reinterpret_cast<int*>(smem + l.scan);
    __threadfence();
    __syncthreads();
    if (n_block == 0) return;
    for (int strip = first / n_slots; strip <= (last - 1) / n_slots; ++strip) {
      if (threadIdx.x == 0) {
        const int done = min(last, (strip + 1) * n_slots) - max(first, strip * n_slots);
        *flag = atomicAdd(&p.counters[strip], done) + done == n_slots;
        __threadfence();
      }
      __syncthreads();
      const bool mine = *flag != 0;
      __syncthreads();
      if (!mine) continue;
      const int row0 = strip * 32, quads = (min(32, p.N - row0)) / 4;
      for (int i = threadIdx.x; i < p.M * quads; i += kThreads) {
        const int m = i / quads, row = row0 + (i - m * quads) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < p.topk; ++s) {
          const int pair = m * p.topk + s;
          if (expert[pair] == 0xFFFF) continue;
          const float w = p.weight_on_input ? 1.f : p.weights[pair];
          const float4 v = __ldcg(reinterpret_cast<const float4*>(p.y + (size_t)pair * p.N + row));
          sum.x += w * v.x;
          sum.y += w * v.y;
          sum.z += w * v.z;
          sum.w += w * v.w;
        }
        const size_t to = (size_t)m * p.N + row;
        store_value(p.out, p.out_dtype, to, sum.x);
        store_value(p.out, p.out_dtype, to + 1, sum.y);
        store_value(p.out, p.out_dtype, to + 2, sum.z);
        store_value(p.out, p.out_dtype, to + 3, sum.w);
      }
    }
  }
}

constexpr int kMaxSplit = 8;

template <typename XT, int kMode, int kCols>
int launch_rows(RowsParams p, cudaStream_t st) {
  using S = Shape<kCols>;
  static std::once_flag once[64];
  static bool ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return B200FP4_STATUS_NOT_SUPPORTED;
  std::call_once(once[dev], [&] {
    ready[dev] = cudaFuncSetAttribute(w4a16_rows_kernel<XT, kMode, kCols>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMost) == cudaSuccess;
    cudaGetLastError();
  });
  if (!ready[dev]) return B200FP4_STATUS_EXECUTION_FAILED;
  const int pairs = kMode == kLinear ? 0 : p.M * p.topk, E = kMode == kLinear ? 0 : p.E;
  unsigned grid = 0;
  uint32_t smem = 0;
  int64_t best = INT64_MAX;
  RowsParams chosen = p;
  // Blocks that share the k of an item in a cluster (linear): a shorter k leaves room for more rows and spreads few strips over all SMs
  for (int split = 1; split <= (kMode == kLinear ? kMaxSplit : 1) && split <= p.units; split *= 2) {
    static ResidentClusters counts[kMaxSplit + 1][64];
    const int clusters = split == 1 ? sm_count() : resident_clusters_of(counts[split], w4a16_rows_kernel<XT, kMode, kCols>, split, kThreads, kSmemMost);
    if (clusters < 1) break;
    RowsParams q = p;
    const uint32_t own = (uint32_t)((p.units + split - 1) / split), row_bytes = own * (kUnitK * 2) + 16;
    const int64_t most = kMode == kLinear ? p.M : pairs;
    q.split = split;
    q.cap = (kMode == kDown ? 4 : 8) * kCols;
    q.rows = 0;
    uint32_t sums = 0;
    while (kMode != kDown) {
      // rows that there is room for; a slot has no more columns than that
      if (kMode == kLinear) q.cap = (int)std::min<int64_t>(q.cap, most);
      const int64_t items = kMode == kLinear ? (most + q.cap - 1) / q.cap * p.strips : 0;
      sums = split > 1 ? (uint32_t)std::min<int64_t>((items + clusters - 1) / clusters, 1 << 16) * q.cap * 128 : 0;
      const uint32_t rest = layout_of(S::kRing, S::kBars, S::kRed, pairs, E, q.cap, 1, 0, sums).bytes;
      q.rows = (int)std::min<int64_t>(kMode == kLinear ? q.cap : most, rest < kSmemMost ? (kSmemMost - rest) / (row_bytes + (uint32_t)sizeof(RowStat)) : 0);
      if (q.rows < 1 || q.rows >= q.cap || q.rows == most) break;
      q.cap = q.rows;
    }
    if (kMode != kDown && q.rows < 1) continue;
    const uint32_t bytes = layout_of(S::kRing, S::kBars, S::kRed, pairs, E, q.cap, q.rows, row_bytes, sums).bytes;
    if (bytes > kSmemMost) continue;
    const int64_t slots = kMode == kLinear ? (most + q.cap - 1) / q.cap : std::min(pairs, E) + pairs / q.cap;
    if (slots * p.strips > 0x3FFFFFFF) continue;
    // units of the block with the most of them; a cluster costs its synchronisation
    const int64_t cost = kMode == kLinear ? ((slots * p.strips + clusters - 1) / clusters * own + (split > 1 ? 4 : 0)) : 0;
    if (cost < best) {
      best = cost;
      chosen = q;
      grid = (unsigned)(kMode == kLinear ? std::min<int64_t>(clusters, slots * p.strips) * split : clusters);
      smem = bytes;
    }
  }
  if (grid == 0) return B200FP4_STATUS_NOT_SUPPORTED;
  if (launch_pdl_cluster(chosen.split, w4a16_rows_kernel<XT, kMode, kCols>, dim3(grid), dim3(kThreads), smem, st, chosen) != cudaSuccess) {
    cudaGetLastError();
    return B200FP4_STATUS_EXECUTION_FAILED;
  }
  return finish_launch(1);
}

template <typename T>
int launch_linear(const RowsParams& p, cudaStream_t st) {
  return p.M <= 8 ? launch_rows<T, kLinear, 1>(p, st) : launch_rows<T, kLinear, 2>(p, st);
}
template <typename T>
int launch_gate_up(const RowsParams& p, cudaStream_t st) {
  return (int64_t)p.M * p.topk <= 4 * (int64_t)p.E ? launch_rows<T, kGateUp, 1>(p, st) : launch_rows<T, kGateUp, 2>(p, st);
}
int launch_down(const RowsParams& p, cudaStream_t st) {
  return (int64_t)p.M * p.topk <= 2 * (int64_t)p.E ? launch_rows<__half, kDown, 1>(p, st) : launch_rows<__half, kDown, 2>(p, st);
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
  size_t act, act_inv, y, counters, bytes;
};
MoeScratch moe_scratch(int64_t M, int64_t topk, int64_t H, int64_t I) {
  MoeScratch s;
  const size_t pairs = (size_t)turn_of(M, topk) * topk;
  s.act = 0;
  s.act_inv = s.act + pad256(pairs * 2 * I * 2);
  s.y = s.act_inv + pad256(pairs * 4);
  s.counters = s.y + pad256(pairs * H * 4);
  s.bytes = s.counters + pad256((size_t)strips_of(H) * 4);
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
  p.peaks = reinterpret_cast<uint32_t*>(packed + unit_bytes(E, N, K, gated));
  if (cudaMemsetAsync(p.peaks, 0, (size_t)E * (gated ? 2 : 1) * 4, static_cast<cudaStream_t>(stream)) != cudaSuccess) {
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
  RowsParams p = {};
  p.x = x;
  p.ldx = ldx;
  p.packed = packed;
  p.g = g_scale;
  p.out = out;
  p.out_dtype = out_dtype;
  p.bias = bias;
  p.bias_dtype = bias_dtype;
  p.M = (int)M;
  p.N = (int)N;
  p.K = (int)K;
  p.strips = (int)w4::strips_of(N);
  p.units = (int)w4::units_of(K);
  p.status = status;
  p.clear_status = 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return x_dtype == B200FP4_DTYPE_BF16 ? launch_linear<__nv_bfloat16>(p, st) : launch_linear<__half>(p, st);
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
  if (!aligned(hidden, 16) || !aligned(w13_packed, 16) || !aligned(w2_packed, 16) || !aligned(out, 16)) return B200FP4_STATUS_INVALID_VALUE;
  if (E > kMaxExperts || topk > kMaxPairs || !fits_int(M * topk) || !fits_int(H + 128) || !fits_int(2 * I + 128)) return B200FP4_STATUS_NOT_SUPPORTED;
  if (workspace == nullptr || !aligned(workspace, 256) || workspace_bytes < b200fp4_w4a16_moe_workspace_bytes(M, topk, H, I))
    return B200FP4_STATUS_ALLOC_FAILED;
  const MoeScratch s = moe_scratch(M, topk, H, I);
  unsigned char* const ws = static_cast<unsigned char*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t turn = turn_of(M, topk);
  for (int64_t m = 0; m < M; m += turn) {
    RowsParams p = {};
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
    p.peaks = reinterpret_cast<const float*>(w13_packed + unit_bytes(E, 2 * I, H, 1));
    p.y = reinterpret_cast<float*>(ws + s.y);
    p.counters = reinterpret_cast<int*>(ws + s.counters);
    p.n_counters = (int)w4::strips_of(H);
    RowsParams d = p;
    p.x = static_cast<const unsigned char*>(hidden) + (size_t)m * H * 2;
    p.ldx = H;
    p.packed = w13_packed;
    p.g = w13_g;
    p.N = (int)(2 * I);
    p.K = (int)H;
    p.strips = (int)((I + 15) / 16);
    p.units = (int)w4::units_of(H);
    d.x = p.act;
    d.ldx = I;
    d.packed = w2_packed;
    d.g = w2_g;
    d.out = static_cast<unsigned char*>(out) + (size_t)m * H * (out_dtype == B200FP4_DTYPE_F32 ? 4 : 2);
    d.out_dtype = out_dtype;
    d.N = (int)H;
    d.K = (int)I;
    d.strips = (int)w4::strips_of(H);
    d.units = (int)w4::units_of(I);
    int rc = h_dtype == B200FP4_DTYPE_BF16 ? launch_gate_up<__nv_bfloat16>(p, st) : launch_gate_up<__half>(p, st);
    if (rc == B200FP4_STATUS_SUCCESS) rc = launch_down(d, st);
    if (rc != B200FP4_STATUS_SUCCESS) return rc;
  }
  return B200FP4_STATUS_SUCCESS;
}
