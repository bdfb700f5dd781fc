// Weight-only NVFP4 (w4a16.cuh): the packing of a checkpoint's weights, the linear layer of few tokens, and the mixture-of-experts layer.
//
// One kernel, three uses.  A warp multiplies a tile of 16 packed rows with up to 8 * kCols columns of activations: codes become the
// 16-bit A operand in registers, the activations of a lane are the B operand as they lie in memory, sums are f32.
//   linear   columns are tokens
//   gate/up  columns are the (token, expert) pairs of one expert; a tile's rows are eight gate rows and the same eight up rows, so that a
//            lane holds both halves of its values and applies SiLU(gate) * up to them
//   down     two columns a pair, the activation's upper and lower 16 bits: bf16 holds eight significant bits, the sum of two holds
//            sixteen, at any magnitude that f32 has, so that the value between the projections is not what limits the result
// Work items are (tile, slot); a slot is a run of one expert's pairs that fits the columns.  A block has a contiguous range of them, groups of
// warps take items in turn and split k among themselves.
// The layer is two launches without anything that has to outlast them: both find the slots from the routing by themselves, the first sets the
// counters of the second, in which the block that finishes a tile's last item adds up its pairs in their order.
#include <algorithm>

#include "w4a16.cuh"

namespace b200fp4 {
namespace {

using namespace w4;

// ------------------------------------------------------------------------------------------ packing

struct PackParams {
  const uint8_t* codes;       // [E, N, K/2]
  const uint8_t* scales;      // [E, N, K/16]
  uint8_t* packed;
  int64_t tiles, units;
  int N, K, gated;
};

// one warp per unit
__global__ void __launch_bounds__(256) w4a16_pack_kernel(const PackParams p, int64_t n_units) {
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= n_units) return;
  const int lane = threadIdx.x & 31;
  const int64_t u = unit % p.units, tile = unit / p.units % p.tiles, e = unit / p.units / p.tiles;
  uint8_t* const dst = p.packed + unit * kUnitBytes;
  uint32_t sc = 0;
  for (int half = 0; half < 2; ++half) {
    const int64_t k = u * kUnitK + half * 64 + (lane & 3) * 16;
    uint32_t word[4];
    for (int r = 0; r < 2; ++r) {
      // rows of a tile: 16 neighbours, or eight of the gate and the same eight of the up half
      const int64_t row = p.gated ? (tile * 8 + (lane >> 2) < p.N / 2 ? r * (int64_t)(p.N / 2) + tile * 8 + (lane >> 2) : p.N)
                                  : tile * 16 + r * 8 + (lane >> 2);
      uint32_t scale = 0;
      uint2 c = make_uint2(0, 0);
      if (row < p.N && k < p.K) {
        const int64_t at = e * p.N + row;
        c = *reinterpret_cast<const uint2*>(p.codes + at * (p.K / 2) + k / 2);
        scale = p.scales[at * (p.K / 16) + k / 16];
        if (scale & 0x80) {
          c.x ^= 0x88888888u;
          c.y ^= 0x88888888u;
        }
      }
      sc |= (scale & 0x7F) << (8 * (half * 2 + r));
      for (int q = 0; q < 2; ++q) {
        const uint32_t w = q ? c.y : c.x;
        uint32_t out = 0;
        for (int i = 0; i < 8; ++i) {
          constexpr int kSign[4] = {15, 12, 13, 14}, kMag[4] = {6, 3, 0, 9};
          const uint32_t code = (w >> (4 * i)) & 15;
          out |= (((code >> 3) << kSign[i >> 1]) | ((code & 7) << kMag[i >> 1])) << (16 * (i & 1));
        }
        word[r * 2 + q] = out;
      }
    }
    *reinterpret_cast<uint4*>(dst + half * 512 + lane * 16) = make_uint4(word[0], word[1], word[2], word[3]);
  }
  *reinterpret_cast<uint32_t*>(dst + kUnitScales + lane * 4) = sc;
}

// ------------------------------------------------------------------------------------------ products

enum Mode { kLinear, kGateUp, kDown };

constexpr int kWarps = 16, kThreads = 32 * kWarps;
constexpr int kMaxPairs = 4096;                // pairs whose slots a block finds in its shared memory; more are done in turns
constexpr int kMaxExperts = 4096;

struct RowsParams {
  const void* x;              // [M, K], rows ldx apart; down: [pair][upper, lower][K] bf16
  int64_t ldx;
  const uint8_t* packed;
  const float* g;             // [E]; gate/up [E][gate, up]
  void* out;                  // linear [M, N]; down [M, N]
  const void* bias;           // [N] or null
  int out_dtype, bias_dtype;
  int M, N, K;
  int tiles, units;
  // layer
  const int32_t* ids;         // [M, topk]
  const float* weights;       // [M, topk]
  const int32_t* map;         // [global_E] or null
  int64_t global_E;
  int topk, E, weight_on_input;
  __nv_bfloat16* act;         // gate/up out
  float* y;                   // down: [pair][N]
  int* counters;              // [tile groups of down]
  int n_counters;
};

struct SlotLayout {
  uint32_t count, expert, rank, list, slots, scan, red, bytes;
};
// Shared memory: pairs an expert has, then where they begin | expert of a pair | its place among that expert's | pairs by expert | slots | scan |
// partial sums
__host__ __device__ __forceinline__ SlotLayout slot_layout(int pairs, int E, int cap, uint32_t red_bytes) {
  SlotLayout l;
  l.count = 0;
  l.expert = l.count + (uint32_t)E * 4;
  l.rank = l.expert + ((uint32_t)pairs * 2 + 3) / 4 * 4;
  l.list = l.rank + ((uint32_t)pairs * 2 + 3) / 4 * 4;
  l.slots = (l.list + (uint32_t)pairs * 2 + 15) / 16 * 16;
  const int most = (pairs < E ? pairs : E) + pairs / cap;
  l.scan = l.slots + (uint32_t)most * 8;
  l.red = (l.scan + (pairs > 0 ? 2 * kWarps * 4 + 16 : 0) + 15) / 16 * 16;
  l.bytes = l.red + red_bytes;
  return l;
}

__device__ __forceinline__ int local_expert(const RowsParams& p, int pair) {
  int64_t e = p.ids[pair];
  if (p.map != nullptr) e = e >= 0 && e < p.global_E ? p.map[e] : -1;
  return e >= 0 && e < p.E ? (int)e : -1;
}

// Slots of at most `cap` pairs of one expert, experts in order and pairs in theirs, so that every block finds the same; returns their number.
// One warp counts, 32 pairs at a time: a few steps for a decode batch, and no order of atomics to depend on.
__device__ int find_slots(const RowsParams& p, unsigned char* smem, const SlotLayout& l, int cap) {
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

// T: type of the operand; kCols: columns of eight; kTiles: row tiles a warp does at once
template <typename T, int kMode, int kCols, int kTiles>
__global__ void __launch_bounds__(kThreads, 1) w4a16_rows_kernel(const RowsParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  constexpr int kCap = (kMode == kDown ? 4 : 8) * kCols;
  constexpr int kAhead = kTiles == 1 ? 4 : 2;
  constexpr int kRedFloats = kTiles * kCols * 4 * 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row8 = lane >> 2, quad = lane & 3;
  const SlotLayout l = slot_layout(kMode == kLinear ? 0 : p.M * p.topk, kMode == kLinear ? 0 : p.E, kCap, kWarps * kRedFloats * 4);
  const int2* const slots = reinterpret_cast<const int2*>(smem + l.slots);
  const uint16_t* const list = reinterpret_cast<const uint16_t*>(smem + l.list);
  pdl_wait();
  pdl_launch_dependents();
  int n_slots;
  if constexpr (kMode == kLinear) {
    n_slots = (p.M + kCap - 1) / kCap;
  } else {
    n_slots = find_slots(p, smem, l, kCap);
    if (kMode == kGateUp && blockIdx.x == 0)
      for (int i = threadIdx.x; i < p.n_counters; i += kThreads) p.counters[i] = 0;
    if (kMode == kDown && n_slots == 0) {
      for (size_t i = (size_t)blockIdx.x * kThreads + threadIdx.x; i < (size_t)p.M * p.N; i += (size_t)gridDim.x * kThreads)
        store_value(p.out, p.out_dtype, i, 0.f);
      return;
    }
  }
  const int groups_of_tiles = (p.tiles + kTiles - 1) / kTiles;
  const int64_t n_items = (int64_t)n_slots * groups_of_tiles;
  const int64_t first = n_items * blockIdx.x / gridDim.x, last = n_items * (blockIdx.x + 1) / gridDim.x;
  const int n_block = (int)(last - first);

  // Warps that share an item: as few rounds as possible, an item's ending counted as one more unit
  int share = 1, best = 1 << 30;
  for (int s = 1; s <= kWarps && s <= p.units; s *= 2) {
    const int cost = (n_block * s + kWarps - 1) / kWarps * ((p.units + s - 1) / s + 1);
    if (cost < best) {
      best = cost;
      share = s;
    }
  }
  const int group = warp / share, in_group = warp - group * share, n_groups = kWarps / share;
  const int k_first = p.units * in_group / share, k_last = p.units * (in_group + 1) / share, n_units = k_last - k_first;
  const int n_mine = n_block > group ? (n_block - group + n_groups - 1) / n_groups : 0;
  const int total = n_mine * n_units;

  auto slot_of = [&](int64_t item) { return kMode == kGateUp ? (int)(item / groups_of_tiles) : (int)(item % n_slots); };
  auto tile_of = [&](int64_t item) { return (kMode == kGateUp ? (int)(item % groups_of_tiles) : (int)(item / n_slots)) * kTiles; };

  struct Unit {
    uint4 codes[kTiles][2];
    uint32_t scales[kTiles];
  } ring[kAhead];
  // what is loaded next
  int64_t load_item = first + group;
  int load_k = k_first;
  const uint8_t* src[kTiles];
  auto load = [&](Unit& u) {
    if (load_k == k_first) {
      const int tile = tile_of(load_item);
      const size_t e = kMode == kLinear ? 0 : slots[slot_of(load_item)].x & 0xFFFF;
#pragma unroll
      for (int r = 0; r < kTiles; ++r)
        src[r] = p.packed + ((e * p.tiles + min(tile + r, p.tiles - 1)) * p.units + k_first) * kUnitBytes;
    }
#pragma unroll
    for (int r = 0; r < kTiles; ++r) {
      u.codes[r][0] = ldg_stream_u4(src[r] + lane * 16);
      u.codes[r][1] = ldg_stream_u4(src[r] + 512 + lane * 16);
      u.scales[r] = ldg_stream_u32(src[r] + kUnitScales + lane * 4);
      src[r] += kUnitBytes;
    }
    if (++load_k == k_last) {
      load_k = k_first;
      load_item += n_groups;
    }
  };
#pragma unroll
  for (int a = 0; a < kAhead; ++a)
    if (a < total) load(ring[a]);

  int64_t item = first + group;
  int k = k_first;
  float acc[kTiles][kCols][4];
  const T* col[kCols];
  for (int i = 0; i < total; i += kAhead) {
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (i + a >= total) break;
      if (k == k_first) {
        const int slot = slot_of(item);
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int at = c * 8 + row8;
          int64_t row = -1;
          if constexpr (kMode == kLinear) {
            if (slot * kCap + at < p.M) row = slot * kCap + at;
          } else {
            const int2 s = slots[slot];
            const int n = s.x >> 16;
            if constexpr (kMode == kGateUp) {
              if (at < n) row = list[s.y + at] / p.topk;
            } else {
              if (at / 2 < n) row = (int64_t)list[s.y + at / 2] * 2 + (at & 1);
            }
          }
          col[c] = row >= 0 ? static_cast<const T*>(p.x) + row * p.ldx + quad * 16 : nullptr;
#pragma unroll
          for (int r = 0; r < kTiles; ++r)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[r][c][j] = 0.f;
        }
      }
      // ---- one unit
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int at = k * kUnitK + half * 64;
        const bool inside = at + quad * 16 < p.K;
        uint32_t b[kCols][8];
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
          if (inside && col[c] != nullptr) {
            lo = ld_u4(col[c] + at);
            hi = ld_u4(col[c] + at + 8);
          }
          b[c][0] = lo.x, b[c][1] = lo.y, b[c][2] = lo.z, b[c][3] = lo.w;
          b[c][4] = hi.x, b[c][5] = hi.y, b[c][6] = hi.z, b[c][7] = hi.w;
        }
#pragma unroll
        for (int r = 0; r < kTiles; ++r) {
          uint32_t s_lo, s_hi;
          scales_of<T>(ring[a].scales[r], half, s_lo, s_hi);
          const uint4 w = ring[a].codes[r][half];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t lo[4], hi[4];
            codes_to_pairs<T>(q ? w.y : w.x, lo);
            codes_to_pairs<T>(q ? w.w : w.z, hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              lo[j] = mul2<T>(lo[j], s_lo);
              hi[j] = mul2<T>(hi[j], s_hi);
            }
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
              mma_16x8x16<T>(acc[r][c], lo[0], hi[0], lo[1], hi[1], b[c][q * 4], b[c][q * 4 + 1]);
              mma_16x8x16<T>(acc[r][c], lo[2], hi[2], lo[3], hi[3], b[c][q * 4 + 2], b[c][q * 4 + 3]);
            }
          }
        }
      }
      if (i + a + kAhead < total) load(ring[a]);
      if (++k < k_last) continue;
      // ---- an item's end
      k = k_first;
      float* const red = reinterpret_cast<float*>(smem + l.red) + group * share * kRedFloats + lane;
      if (share > 1) {
        if (in_group > 0) {
#pragma unroll
          for (int r = 0; r < kTiles; ++r)
#pragma unroll
            for (int c = 0; c < kCols; ++c)
#pragma unroll
              for (int j = 0; j < 4; ++j) red[in_group * kRedFloats + ((r * kCols + c) * 4 + j) * 32] = acc[r][c][j];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(share * 32) : "memory");
        if (in_group == 0) {
          for (int s = 1; s < share; ++s)
#pragma unroll
            for (int r = 0; r < kTiles; ++r)
#pragma unroll
              for (int c = 0; c < kCols; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[r][c][j] += red[s * kRedFloats + ((r * kCols + c) * 4 + j) * 32];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(share * 32) : "memory");
      }
      if (in_group == 0) {
        const int slot = slot_of(item), tile = tile_of(item);
        const int2 s = kMode == kLinear ? make_int2(0, 0) : slots[slot];
        const int e = kMode == kLinear ? 0 : s.x & 0xFFFF;
        const float scale = p.g[kMode == kGateUp ? 2 * e : e] * kOutScale, up_scale = kMode == kGateUp ? p.g[2 * e + 1] * kOutScale : 0.f;
#pragma unroll
        for (int r = 0; r < kTiles; ++r) {
          if (tile + r >= p.tiles) break;
#pragma unroll
          for (int c = 0; c < kCols; ++c) {
            const int at = c * 8 + quad * 2;       // this lane's two columns
            if constexpr (kMode == kLinear) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int m = slot * kCap + at + (j & 1), n = (tile + r) * 16 + row8 + (j >> 1) * 8;
                if (m < p.M && n < p.N) {
                  float v = acc[r][c][j] * scale;
                  if (p.bias != nullptr) v += load_value(p.bias, p.bias_dtype, n);
                  store_value(p.out, p.out_dtype, (size_t)m * p.N + n, v);
                }
              }
            } else if constexpr (kMode == kGateUp) {
              const int i_at = (tile + r) * 8 + row8, I = p.N / 2;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                if (at + j < (s.x >> 16) && i_at < I) {
                  const int pair = list[s.y + at + j];
                  const float f = p.weight_on_input ? p.weights[pair] : 1.f;
                  const float v = silu_f32(acc[r][c][j] * scale * f) * (acc[r][c][2 + j] * up_scale * f);
                  const __nv_bfloat16 hi = __float2bfloat16_rn(v);
                  const float rest = v - __bfloat162float(hi);
                  __nv_bfloat16* const to = p.act + (size_t)pair * 2 * I + i_at;
                  to[0] = hi;
                  to[I] = __float2bfloat16_rn(isfinite(rest) ? rest : 0.f);      // an infinite or NaN value is the upper part's alone
                }
              }
            } else {
              if (at / 2 < (s.x >> 16)) {
                float* const to = p.y + (size_t)list[s.y + at / 2] * p.N + (tile + r) * 16 + row8;
                to[0] = (acc[r][c][0] + acc[r][c][1]) * scale;
                to[8] = (acc[r][c][2] + acc[r][c][3]) * scale;
              }
            }
          }
        }
      }
      item += n_groups;
    }
  }

  if constexpr (kMode == kDown) {
    // The block that completes a group of tiles adds up every token's pairs, in the order of the routing.
    const uint16_t* const expert = reinterpret_cast<const uint16_t*>(smem + l.expert);
    int* const flag = reinterpret_cast<int*>(smem + l.scan);
    __threadfence();
    __syncthreads();
    if (n_block == 0) return;
    for (int tg = (int)(first / n_slots); tg <= (int)((last - 1) / n_slots); ++tg) {
      if (threadIdx.x == 0) {
        const int64_t from = max(first, (int64_t)tg * n_slots), to = min(last, (int64_t)(tg + 1) * n_slots);
        const int done = (int)(to - from);
        *flag = atomicAdd(&p.counters[tg], done) + done == n_slots;
        __threadfence();
      }
      __syncthreads();
      const bool mine = *flag != 0;
      __syncthreads();
      if (!mine) continue;
      const int row0 = tg * kTiles * 16, quads = (min(kTiles * 16, p.N - row0)) / 4;
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
        const size_t at = (size_t)m * p.N + row;
        store_value(p.out, p.out_dtype, at, sum.x);
        store_value(p.out, p.out_dtype, at + 1, sum.y);
        store_value(p.out, p.out_dtype, at + 2, sum.z);
        store_value(p.out, p.out_dtype, at + 3, sum.w);
      }
    }
  }
}

template <typename T, int kMode, int kCols, int kTiles>
int launch_rows(const RowsParams& p, cudaStream_t st) {
  constexpr uint32_t kRed = kWarps * kTiles * kCols * 4 * 32 * 4;
  constexpr int kCap = (kMode == kDown ? 4 : 8) * kCols;
  static std::once_flag once[64];
  static bool ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return B200FP4_STATUS_NOT_SUPPORTED;
  std::call_once(once[dev], [&] {
    ready[dev] = cudaFuncSetAttribute(w4a16_rows_kernel<T, kMode, kCols, kTiles>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)slot_layout(kMode == kLinear ? 0 : kMaxPairs, kMode == kLinear ? 0 : kMaxExperts, kCap, kRed).bytes) == cudaSuccess;
    cudaGetLastError();
  });
  if (!ready[dev]) return B200FP4_STATUS_EXECUTION_FAILED;
  const uint32_t smem = slot_layout(kMode == kLinear ? 0 : p.M * p.topk, kMode == kLinear ? 0 : p.E, kCap, kRed).bytes;
  if (launch_pdl(w4a16_rows_kernel<T, kMode, kCols, kTiles>, dim3(sm_count()), dim3(kThreads), smem, st, p) != cudaSuccess) {
    cudaGetLastError();
    return B200FP4_STATUS_EXECUTION_FAILED;
  }
  return finish_launch(1);
}

template <typename T>
int launch_linear(const RowsParams& p, cudaStream_t st) {
  if (p.M <= 8) return launch_rows<T, kLinear, 1, 1>(p, st);
  if (p.M <= 16) return launch_rows<T, kLinear, 2, 2>(p, st);
  return launch_rows<T, kLinear, 4, 2>(p, st);
}
template <typename T>
int launch_gate_up(const RowsParams& p, cudaStream_t st) {
  if ((int64_t)p.M * p.topk <= 4 * (int64_t)p.E) return launch_rows<T, kGateUp, 1, 1>(p, st);
  return launch_rows<T, kGateUp, 2, 2>(p, st);
}
int launch_down(const RowsParams& p, cudaStream_t st) {
  if ((int64_t)p.M * p.topk <= 2 * (int64_t)p.E) return launch_rows<__nv_bfloat16, kDown, 1, 1>(p, st);
  return launch_rows<__nv_bfloat16, kDown, 2, 2>(p, st);
}

bool fits_int(int64_t v) { return v >= 0 && v <= 0x7FFFFFFF; }
bool is_16bit(int dtype) { return dtype == B200FP4_DTYPE_F16 || dtype == B200FP4_DTYPE_BF16; }
bool is_dtype(int dtype) { return is_16bit(dtype) || dtype == B200FP4_DTYPE_F32; }
size_t pad256(size_t v) { return (v + 255) / 256 * 256; }

constexpr size_t kStatusBytes = 256;

// tokens of a layer whose pairs fit one turn
int64_t turn_of(int64_t M, int64_t topk) { return std::min(M, std::max<int64_t>(1, kMaxPairs / topk)); }

struct MoeScratch {
  size_t act, y, counters, bytes;
};
MoeScratch moe_scratch(int64_t M, int64_t topk, int64_t H, int64_t I) {
  MoeScratch s;
  const size_t pairs = (size_t)turn_of(M, topk) * topk;
  s.act = kStatusBytes;
  s.y = s.act + pad256(pairs * 2 * I * 2);
  s.counters = s.y + pad256(pairs * H * 4);
  s.bytes = s.counters + pad256((size_t)tiles_of(H) * 4);
  return s;
}

}  // namespace
}  // namespace b200fp4

using namespace b200fp4;

extern "C" size_t b200fp4_w4a16_packed_bytes(int64_t E, int64_t N, int64_t K, int gated) {
  if (E < 1 || N < 1 || K < 16 || K % 16 != 0 || (gated && N % 2 != 0)) return 0;
  return (size_t)E * (gated ? (N / 2 + 7) / 8 : w4::tiles_of(N)) * w4::units_of(K) * w4::kUnitBytes;
}

extern "C" int b200fp4_w4a16_pack(const uint8_t* codes, const uint8_t* scales, int64_t E, int64_t N, int64_t K, int gated, uint8_t* packed,
                                  void* stream) {
  if (b200fp4_w4a16_packed_bytes(E, N, K, gated) == 0 || !fits_int(N) || !fits_int(K)) return B200FP4_STATUS_INVALID_VALUE;
  if (codes == nullptr || scales == nullptr || packed == nullptr || !aligned(codes, 8) || !aligned(packed, 16)) return B200FP4_STATUS_INVALID_VALUE;
  PackParams p = {};
  p.codes = codes;
  p.scales = scales;
  p.packed = packed;
  p.tiles = gated ? (N / 2 + 7) / 8 : w4::tiles_of(N);
  p.units = w4::units_of(K);
  p.N = (int)N;
  p.K = (int)K;
  p.gated = gated != 0;
  const int64_t n = E * p.tiles * p.units;
  if ((n + 7) / 8 > 0x7FFFFFFF) return B200FP4_STATUS_NOT_SUPPORTED;
  w4a16_pack_kernel<<<(unsigned)((n + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(p, n);
  return finish_launch(1);
}

extern "C" size_t b200fp4_w4a16_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  (void)M, (void)N, (void)K;
  return kStatusBytes;
}

extern "C" int b200fp4_w4a16_linear(const void* x, int x_dtype, int64_t ldx, const uint8_t* packed, const float* g_scale, const void* bias,
                                    int bias_dtype, void* out, int out_dtype, int64_t M, int64_t N, int64_t K, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (M < 0 || N < 1 || K < 16 || K % 16 != 0) return B200FP4_STATUS_INVALID_VALUE;
  if (!is_16bit(x_dtype) || !is_dtype(out_dtype) || (bias != nullptr && !is_dtype(bias_dtype))) return B200FP4_STATUS_INVALID_VALUE;
  if (M == 0) return B200FP4_STATUS_SUCCESS;
  if (x == nullptr || packed == nullptr || g_scale == nullptr || out == nullptr) return B200FP4_STATUS_INVALID_VALUE;
  if (!aligned(x, 16) || !aligned(packed, 16) || !aligned(out, 16) || ldx % 8 != 0 || (M > 1 && ldx < K)) return B200FP4_STATUS_INVALID_VALUE;
  if (workspace == nullptr || !aligned(workspace, 256) || workspace_bytes < b200fp4_w4a16_linear_workspace_bytes(M, N, K))
    return B200FP4_STATUS_ALLOC_FAILED;
  if (!fits_int(M) || !fits_int(N + 16) || !fits_int(K + 128)) return B200FP4_STATUS_NOT_SUPPORTED;
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
  p.tiles = (int)w4::tiles_of(N);
  p.units = (int)w4::units_of(K);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return x_dtype == B200FP4_DTYPE_BF16 ? launch_linear<__nv_bfloat16>(p, st) : launch_linear<__half>(p, st);
}

extern "C" size_t b200fp4_w4a16_moe_workspace_bytes(int64_t M, int64_t topk, int64_t H, int64_t I) {
  if (M < 1 || topk < 1 || H < 1 || I < 1) return kStatusBytes;
  return moe_scratch(M, topk, H, I).bytes;
}

extern "C" int b200fp4_w4a16_moe(const void* hidden, int h_dtype, const float* topk_weights, const int32_t* topk_ids, const int32_t* expert_map,
                                 int64_t global_E, const uint8_t* w13_packed, const float* w13_g, const uint8_t* w2_packed, const float* w2_g,
                                 void* out, int out_dtype, int64_t M, int64_t topk, int64_t H, int64_t I, int64_t E, int flags, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (M < 0 || topk < 1 || E < 1 || H < 16 || H % 16 != 0 || I < 16 || I % 16 != 0) return B200FP4_STATUS_INVALID_VALUE;
  if (!is_16bit(h_dtype) || !is_dtype(out_dtype) || (flags & ~B200FP4_MOE_ROUTER_WEIGHT_ON_INPUT) != 0) return B200FP4_STATUS_INVALID_VALUE;
  if (M == 0) return B200FP4_STATUS_SUCCESS;
  if (hidden == nullptr || topk_weights == nullptr || topk_ids == nullptr || w13_packed == nullptr || w13_g == nullptr || w2_packed == nullptr ||
      w2_g == nullptr || out == nullptr || (expert_map != nullptr && global_E < 1))
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
    p.ids = topk_ids + m * topk;
    p.weights = topk_weights + m * topk;
    p.map = expert_map;
    p.global_E = global_E;
    p.topk = (int)topk;
    p.E = (int)E;
    p.weight_on_input = flags & B200FP4_MOE_ROUTER_WEIGHT_ON_INPUT ? 1 : 0;
    p.act = reinterpret_cast<__nv_bfloat16*>(ws + s.act);
    p.y = reinterpret_cast<float*>(ws + s.y);
    p.counters = reinterpret_cast<int*>(ws + s.counters);
    p.n_counters = (int)w4::tiles_of(H);
    RowsParams d = p;
    p.x = static_cast<const unsigned char*>(hidden) + (size_t)m * H * 2;
    p.ldx = H;
    p.packed = w13_packed;
    p.g = w13_g;
    p.N = (int)(2 * I);
    p.K = (int)H;
    p.tiles = (int)((I + 7) / 8);
    p.units = (int)w4::units_of(H);
    d.x = p.act;
    d.ldx = I;
    d.packed = w2_packed;
    d.g = w2_g;
    d.out = static_cast<unsigned char*>(out) + (size_t)m * H * (out_dtype == B200FP4_DTYPE_F32 ? 4 : 2);
    d.out_dtype = out_dtype;
    d.N = (int)H;
    d.K = (int)I;
    d.tiles = (int)w4::tiles_of(H);
    d.units = (int)w4::units_of(I);
    int rc = h_dtype == B200FP4_DTYPE_BF16 ? launch_gate_up<__nv_bfloat16>(p, st) : launch_gate_up<__half>(p, st);
    if (rc == B200FP4_STATUS_SUCCESS) rc = launch_down(d, st);
    if (rc != B200FP4_STATUS_SUCCESS) return rc;
  }
  return B200FP4_STATUS_SUCCESS;
}
