// Weight-only NVFP4 linear of many tokens: out[M,N] = x . W^T * g (+ bias) on the tcgen05 tensor cores.
//
// The 128 rows of an MMA are rows of the weight, the tokens are its columns.  Decoding warps turn packed units (w4a16.cuh) into 16-bit values and write
// them straight into tensor memory, from where the MMA takes its A operand: a decoded weight never is in shared memory, and it is decoded once for
// up to 192 tokens.  The activations are the B operand as they lie in memory, brought in by TMA, in the type they have: products are exact in bf16
// and in f16 alike.
// Roles (23 warps): 0 copies of the weight, 22 of the tokens, 1 MMAs and tensor memory, 2-5 (in the end 2-21) epilogue, 6-21 decoding (four sets of
// four, a warp 32 rows of the tile and every fourth 128 of k).  One warp that brought in weight and tokens, four copies for 128 rows, took 1040
// cycles for 128 of k and was what all waited for. Tensor memory: accumulators, and the rest for A stages of 64 columns (128 rows x 128 of k): the
// MMA warp's waits, MMAs and commits take 300 cycles a stage however few the tokens are.  Persistent blocks, one to an SM; where there are too few
// tiles for them, a cluster shares the k of one and adds up its parts through distributed shared memory, each block some of the tokens. Every wait is
// bounded (status word), tensor memory is always freed.
// Bound: with many tokens by the tensor cores, M=4096 N=14336 K=4096 400 us, 1.20 PFLOP/s under the power cap (73 % of the measured burst rate, 88 %
// of the sustained one), the tensor pipe busy 73 % of active cycles; with few by decoding and the MMA warp's turn, some 450 cycles for 128 of k where
// HBM brings them in 390: M=32 N=4096 K=14336 15.1 us (33 MB, floor 5.3), M=333 N=K=4096 15.9 (0.70 PFLOP/s).
#include <algorithm>
#include <type_traits>

#include "sm100_ptx.cuh"
#include "w4a16_linear.cuh"
#include "w4a16.cuh"

namespace b200fp4 {
namespace {

using namespace w4;

constexpr int kMmaRows = 128, kMostTokens = 192;
constexpr int kDecodeSets = 4, kFirstDecode = 6, kTokenWarp = kFirstDecode + 4 * kDecodeSets;
constexpr int kThreads = 32 * (kTokenWarp + 1);
// Stages at most; how many there are goes by the tokens of a tile.  Of the MMA's operands: 128 rows x 128 of k in tensor memory, beside the
// accumulators, and tokens x 128 of k in shared memory, two boxes of 64; of packed units of 128 rows x 128 of k.
constexpr int kMost = 6, kWMost = 12;
constexpr uint32_t kWStageBytes = 4 * kUnitBytes, kRingBytes = 212 * 1024;
constexpr uint32_t kSmemBytes = 1024 + kRingBytes + 1024;
constexpr int kMaxSplit = 8;

struct GemmParams {
  const uint8_t* packed;
  const uint32_t* tail;
  const float* g;
  const void* bias;
  void* out;
  int bias_dtype, out_dtype;
  int M, N, K;
  int strips, units;
  int tokens;                 // columns of a tile, a multiple of 16
  int row_tiles, tiles;       // tiles: row tiles x token tiles, row tiles first
  int split;                  // blocks of a cluster, which share the units of a tile (then each block has one)
  int stages, w_stages;
  int sets;                   // decoding sets at work: no more than stages of either kind, since a set that is further ahead would take a stage's round for the one before
  uint32_t acc_cols;          // columns of an accumulator
  int accs;                   // accumulators in turn: two where a block does several tiles, or one in several chains
  int chain, chains;          // units that are summed in one accumulator; one tile: accumulators next to each other, whose sum is the result
  uint32_t tag;
  int last_block;             // which has the last tile of all
  uint32_t sums_at;           // split: where the cluster's sums go; 0: where the token stages were
  int* status;
};

// A pair of codes' f16 values times a block's scale, in the operand's type; both products are exact.  To bf16 by way of two f32, which a
// mixed-precision multiplication gives at once: 54 cycles of an SM for 32 rows x 64 of k, against 75 where the bits are moved and multiplied in bf16,
// and 34 in f16.
template <typename T>
__device__ __forceinline__ uint32_t scaled(uint32_t pair, uint32_t scale);
template <>
__device__ __forceinline__ uint32_t scaled<__half>(uint32_t pair, uint32_t scale) {
  return as_u32(__hmul2(as_half2(pair), as_half2(scale)));
}
template <>
__device__ __forceinline__ uint32_t scaled<__nv_bfloat16>(uint32_t pair, uint32_t scale) {
  uint32_t r;
  asm("{\n"
      ".reg .b16 lo, hi, s, unused;\n"
      ".reg .f32 a, b;\n"
      "mov.b32 {lo, hi}, %1;\n"
      "mov.b32 {s, unused}, %2;\n"
      "fma.rn.f32.f16 a, lo, s, 0f80000000;\n"
      "fma.rn.f32.f16 b, hi, s, 0f80000000;\n"
      "cvt.rn.bf16x2.f32 %0, b, a;\n"
      "}\n"
      : "=r"(r)
      : "r"(pair), "r"(scale));
  return r;
}
// E4M3 byte -> the scale twice in a register, f16
__device__ __forceinline__ uint32_t scale_pair(uint32_t byte) {
  return as_u32(__hmul2(as_half2(byte * 0x00800080u), as_half2(0x5C005C00u)));      // fields in place: times 2^-8
}

__device__ __forceinline__ void tcgen05_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// D += A . B^T, A in tensor memory; by the lane whose `issue` is set.  Predicates instead of a branch: in a branch of one lane every operand is moved
// to the uniform registers that the instruction wants.
__device__ __forceinline__ void tcgen05_mma_ts(uint32_t issue, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_desc_lo, uint32_t b_desc_hi, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      ".reg .b64 b;\n"
      "mov.b64 b, {%2, %3};\n"
      "setp.ne.b32 p, %5, 0;\n"
      "setp.ne.b32 q, %6, 0;\n"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n"
      "}\n" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_desc_lo), "r"(b_desc_hi), "r"(idesc), "r"(accumulate), "r"(issue)
      : "memory");
}
__device__ __forceinline__ bool mbar_test_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void tcgen05_commit_if(uint32_t issue, uint32_t bar) {
  asm volatile(
      "{\n"
      ".reg .pred q;\n"
      "setp.ne.b32 q, %1, 0;\n"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
      "}\n" ::"r"(bar),
      "r"(issue)
      : "memory");
}
// a position in a ring of `size` stages
struct Slot {
  uint32_t at = 0, phase = 0;
  __device__ __forceinline__ void next(uint32_t size) {
    if (++at == size) {
      at = 0;
      phase ^= 1;
    }
  }
};

// kChains: an f32 result of more units than a chain has; the others' loops are the shorter for it (M=32 N=4096 K=14336 bf16 14.8 us, 15.7 with the
// chains' counting)
template <typename T, bool kChains>
__global__ void __launch_bounds__(kThreads, 1) w4a16_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const GemmParams p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* const smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = smem_u32(smem), bars = base + kRingBytes;
  const uint32_t full = bars, empty = full + 8 * kMost, w_full = empty + 8 * kMost, w_empty = w_full + 8 * kWMost;
  const uint32_t acc_full = w_empty + 8 * kWMost, acc_empty = acc_full + 16, tmem_ptr = acc_empty + 16;
  const int tokens = p.tokens, split = p.split;
  const uint32_t stages = p.stages, w_stages = p.w_stages, acc_cols = p.acc_cols, a_col = acc_cols * (kChains ? max(p.accs, p.chains) : p.accs);
  const uint32_t b_half = (uint32_t)tokens * 128, b_bytes = 2 * b_half, w_ring = base + stages * b_bytes;
  const int rank = split > 1 ? (int)blockIdx.x & (split - 1) : 0;
  const int first_tile = (int)blockIdx.x / split, step = (int)gridDim.x / split;
  const int unit_first = p.units * rank / split, n_units = p.units * (rank + 1) / split - unit_first;
  int* const status = p.status;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMost; ++i) {
      mbar_init(full + 8 * i, 5);                  // the tokens, and each of a set's four warps
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < kWMost; ++i) {
      mbar_init(w_full + 8 * i, 1);
      mbar_init(w_empty + 8 * i, 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async_smem();
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_ptr), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = lds32(tmem_ptr);
  pdl_wait();
  pdl_launch_dependents();
  const bool reports = (int)blockIdx.x == p.last_block && threadIdx.x == 0;
  if (reports) *status = 0;
  if (split > 1) cluster_arrive_relaxed();         // the other blocks run before anything is sent to them

  if (warp == 0) {
    // ------------------------------------------------------------------ copies of the weight
    const bool leader = elect_one();
    Slot w;
    bool ok = true;
    w.phase = 1;
    for (int tile = first_tile; tile < p.tiles && ok; tile += step) {
      const int strip0 = tile % p.row_tiles * 4;
      int strips;
      const uint8_t* src = p.packed + (size_t)strip_at(strip0, p.strips, p.units, unit_first, strips) * kUnitBytes;
      const uint32_t bytes = (uint32_t)strips * kUnitBytes;
      for (int u = 0; u < n_units; ++u, src += bytes) {
        ok = mbar_wait_warp(w_empty + 8 * w.at, w.phase, status, 71);
        if (!ok) break;
        if (leader) {
          mbar_expect_tx(w_full + 8 * w.at, bytes);
          bulk_load_1d(w_ring + w.at * kWStageBytes, src, bytes, w_full + 8 * w.at);
        }
        __syncwarp();
        w.next(w_stages);
      }
    }
  } else if (warp == kTokenWarp) {
    // ------------------------------------------------------------------ copies of the tokens
    const bool leader = elect_one();
    Slot b;
    bool ok = true;
    b.phase = 1;
    for (int tile = first_tile; tile < p.tiles && ok; tile += step) {
      const int token0 = tile / p.row_tiles * tokens;
      for (int u = 0; u < n_units; ++u) {
        ok = mbar_wait_warp(empty + 8 * b.at, b.phase, status, 72);
        if (!ok) break;
        if (leader) {
          const uint32_t bar = full + 8 * b.at, to = base + b.at * b_bytes;
          mbar_expect_tx(bar, b_bytes);
          tma_load_2d(to, &map_x, (unit_first + u) * 256, token0, bar);
          tma_load_2d(to + b_half, &map_x, (unit_first + u) * 256 + 128, token0, bar);
        }
        __syncwarp();
        b.next(stages);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMAs
    const bool leader = elect_one();
    // f32 accumulators, A and B both f16 or both bf16, K-major, M = 128, N = tokens
    constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    const uint32_t idesc = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(tokens >> 3) << 17) | ((uint32_t)(kMmaRows >> 4) << 24);
    const uint64_t b0 = desc_kmajor<128>(base);
    const uint32_t b0_lo = (uint32_t)b0, b0_hi = (uint32_t)(b0 >> 32);      // a stage's address does not reach the upper half
    bool ready = false;
    Slot op, acc;
    bool ok = true;
    acc.phase = 1;
    uint32_t d = tmem;
    for (int tile = first_tile; tile < p.tiles && ok; tile += step) {
      int chained = 0;                             // units of this chain
      for (int u = 0; u < n_units; ++u) {
        if (u == 0 || (kChains && chained == 0 && p.accs > 1)) {
          ok = mbar_wait_warp(acc_empty + 8 * acc.at, acc.phase, status, 73);
          if (!ok) break;
          tcgen05_fence_after();
          d = tmem + acc.at * acc_cols;
        }
        // One wait and one commit for 128 of k: with barriers of their own for the two operands the loop took 650 cycles for few tokens.  The next
        // stage is looked at while this one's MMAs are issued.
        if (!ready) ok = mbar_wait_warp(full + 8 * op.at, op.phase, status, 74);
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t desc = b0_lo + ((op.at * b_bytes) >> 4), from = tmem + a_col + op.at * 64, done = empty + 8 * op.at;
        op.next(stages);
        const bool next = mbar_test_wait(full + 8 * op.at, op.phase);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          tcgen05_mma_ts(leader, d, from + i * 8, desc + (i & 3) * 2 + (i >> 2) * (b_half >> 4), b0_hi, idesc, ((kChains ? chained : u) > 0 || i > 0) ? 1u : 0u);
        tcgen05_commit_if(leader, done);
        if (u == n_units - 1) tcgen05_commit_if(leader, acc_full + 8 * acc.at);
        if (kChains && ++chained == p.chain) {
          chained = 0;
          if (p.accs == 1) {
            d += acc_cols;
          } else if (u < n_units - 1) {
            tcgen05_commit_if(leader, acc_full + 8 * acc.at);
            acc.next(p.accs);
          }
        }
        ready = __all_sync(0xffffffffu, next);
      }
      acc.next(p.accs);
    }
  } else if (warp >= kFirstDecode) {
    // ------------------------------------------------------------------ decoding: a lane is a row
    const int set = (warp - kFirstDecode) >> 2, quarter = warp & 3, r8 = lane & 7, upper = (lane >> 3) & 1, tile16 = lane >> 4;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    uint32_t code_at[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) code_at[t] = quarter * kUnitBytes + tile16 * 1024 + chunk_at(r8, t) + upper * 8;
    const uint32_t scale_at = quarter * kUnitBytes + kUnitScales + r8 * 32 + tile16 * 4, scale_shift = upper * 8;
    bool ok = true;
    // each set every `sets`th unit of all that the block does
    int tiles = 0;
    for (int tile = first_tile; tile < p.tiles; tile += step) ++tiles;
    const int turns = set < p.sets ? tiles * n_units : 0;
    Slot w, a;
    a.phase = 1;                                   // the first round finds its stages free
    for (int i = 0; i < set; ++i) {
      w.next(w_stages);
      a.next(stages);
    }
    for (int turn = set; turn < turns; turn += p.sets) {
      ok = mbar_wait_warp(w_full + 8 * w.at, w.phase, status, 76);
      if (!ok) break;
      const uint32_t unit = w_ring + w.at * kWStageBytes;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t v[32];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const uint2 code = lds64(unit + code_at[t] + half * 512);
          uint32_t pair[8];
          codes_to_pairs(code.x, *reinterpret_cast<uint32_t(*)[4]>(&pair[0]));
          codes_to_pairs(code.y, *reinterpret_cast<uint32_t(*)[4]>(&pair[4]));
          const uint32_t s = scale_pair((lds32(unit + scale_at + t * 8) >> (scale_shift + half * 16)) & 0x7Fu);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[t * 8 + i] = scaled<T>(pair[i], s);
        }
        if (half == 0) {
          ok = mbar_wait_warp(empty + 8 * a.at, a.phase, status, 77);
          if (!ok) break;
          tcgen05_fence_after();
        } else {
          __syncwarp();
          if (lane == 0) mbar_arrive(w_empty + 8 * w.at);
        }
        tcgen05_st_32x32(tmem + a_col + lanes + a.at * 64 + half * 32, v);
      }
      if (!ok) break;
      tcgen05_wait_st();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(full + 8 * a.at);
      for (int i = 0; i < p.sets; ++i) {
        w.next(w_stages);
        a.next(stages);
      }
    }
  }
  __syncwarp();
  // ---------------------------------------------------------------------- epilogue: a lane is a row of the weight, a column a token
  const int quarter = warp & 3;
  const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
  auto factor = [&](int row_tile) { return row_tile < p.row_tiles - 1 || packed_for(*p.tail, p.tag) ? *p.g : __int_as_float(0x7FC00000); };      // read next to the last rows' units
  // columns from, from + by, ... of a tile of n tokens, 32 at a time
  auto write_columns = [&](uint32_t acc, int row, int token0, int n, int from, int by, float g, bool more) {
    const float bias = p.bias != nullptr && row < p.N ? load_value(p.bias, p.bias_dtype, row) : 0.f;
    for (int c = from; c < n; c += by) {
      uint32_t r[32];
      tcgen05_ld_32x32(tmem + lanes + acc + c, r);
      tcgen05_wait_ld();
      if (row >= p.N) continue;
      const size_t at = (size_t)(token0 + c) * p.N + row;
      const int most = n - c;
      if (p.out_dtype == B200FP4_DTYPE_BF16) {
        __nv_bfloat16* const to = static_cast<__nv_bfloat16*>(p.out) + at;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < most) to[(size_t)i * p.N] = __float2bfloat16_rn(__uint_as_float(r[i]) * g + bias);
      } else if (p.out_dtype == B200FP4_DTYPE_F16) {
        __half* const to = static_cast<__half*>(p.out) + at;
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (i < most) to[(size_t)i * p.N] = __float2half_rn(__uint_as_float(r[i]) * g + bias);
      } else {
        float* const to = static_cast<float*>(p.out) + at;
        if (kChains && more) {
          // to the sum of the chains before this one: the same lane's, so that the order is the program's
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i < most) asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(to + (size_t)i * p.N), "f"(__uint_as_float(r[i]) * g) : "memory");
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i < most) to[(size_t)i * p.N] = __uint_as_float(r[i]) * g + bias;
        }
      }
    }
  };
  if (reports && !packed_for(*p.tail, p.tag)) *status = kOtherSizes;
  if (p.accs > 1) {
    // several tiles: four warps, while the others go on
    if (warp >= 2 && warp < kFirstDecode) {
      Slot acc;
      for (int tile = first_tile; tile < p.tiles; tile += step) {
        const int token0 = tile / p.row_tiles * tokens;
        const float g = factor(tile % p.row_tiles);
        bool ok = true;
        for (int u = 0; u < n_units; u += kChains ? p.chain : n_units) {
          ok = mbar_wait_warp(acc_full + 8 * acc.at, acc.phase, status, 78);
          if (!ok) break;
          tcgen05_fence_after();
          write_columns(acc.at * acc_cols, tile % p.row_tiles * kMmaRows + quarter * 32 + lane, token0, min(tokens, p.M - token0), 0, 32, g, u > 0);
          tcgen05_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty + 8 * acc.at);
          acc.next(2);
        }
        if (!ok) break;
      }
    }
  } else {
    // one tile: all warps that are left, five to a quarter of tensor memory
    const bool work = warp >= 2 && warp < kTokenWarp;
    const int nth = (warp - 2) >> 2, row_tile = first_tile % p.row_tiles, token0 = first_tile / p.row_tiles * tokens;
    bool ok = true;
    if (work) ok = mbar_wait_warp(acc_full, 0, status, 79);
    tcgen05_fence_after();
    const float g = factor(row_tile);
    if (split == 1) {
      if (work && ok) write_columns(0, row_tile * kMmaRows + quarter * 32 + lane, token0, min(tokens, p.M - token0), nth * 32, 5 * 32, g, false);
    } else {
      // Token t of the tile is finished by block t / (tokens / split): [source][its tokens][128 rows] of f32
      cluster_wait();
      if (p.sums_at == 0) cluster_sync_any();      // all MMAs of the cluster have read their token stages
      const int own = tokens / split;
      const uint32_t sums_base = base + p.sums_at;
      if (work)
        for (int c = nth * 16; c < tokens; c += 5 * 16) {
          uint32_t r[16];
          tcgen05_ld_32x16(tmem + lanes + c, r);
          tcgen05_wait_ld();
          for (int u = p.chain, at = acc_cols; kChains && u < n_units; u += p.chain, at += acc_cols) {
            uint32_t other[16];
            tcgen05_ld_32x16(tmem + lanes + at + c, other);
            tcgen05_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(other[i]));
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int t = c + i, owner = t / own;
            const uint32_t to = sums_base + ((uint32_t)(rank * own + t - owner * own) * kMmaRows + quarter * 32 + lane) * 4;
            asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(map_to_cta(to, owner)), "r"(r[i]) : "memory");
          }
        }
      cluster_sync_any();
      const int row0 = row_tile * kMmaRows, first = token0 + rank * own;
      const float* const sums = reinterpret_cast<const float*>(smem + p.sums_at);
      for (int i = threadIdx.x; i < own * kMmaRows; i += kThreads) {
        const int m = first + i / kMmaRows, row = row0 + i % kMmaRows;
        if (m >= p.M || row >= p.N) continue;
        float v = 0.f;
        for (int s = 0; s < split; ++s) v += sums[s * own * kMmaRows + i];
        v *= g;
        if (p.bias != nullptr) v += load_value(p.bias, p.bias_dtype, row);
        store_value(p.out, p.out_dtype, (size_t)m * p.N + row, v);
      }
    }
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <typename T, bool kChains>
int launch_gemm(const LinearCall& c, cudaStream_t st) {
  static std::once_flag once[64];
  static bool ready[64];
  static ResidentClusters counts[kMaxSplit + 1][64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return B200FP4_STATUS_NOT_SUPPORTED;
  std::call_once(once[dev], [&] {
    ready[dev] = cudaFuncSetAttribute(w4a16_gemm_kernel<T, kChains>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBytes) == cudaSuccess;
    cudaGetLastError();
  });
  if (!ready[dev]) return B200FP4_STATUS_EXECUTION_FAILED;
  GemmParams p = {};
  p.packed = c.packed;
  p.tail = c.tail;
  p.tag = size_tag(c.N, c.K, 0);
  p.g = c.g;
  p.bias = c.bias;
  p.bias_dtype = c.bias_dtype;
  p.out = c.out;
  p.out_dtype = c.out_dtype;
  p.M = (int)c.M;
  p.N = (int)c.N;
  p.K = (int)c.K;
  p.strips = (int)strips_of(c.N);
  p.units = (int)units_of(c.K);
  p.row_tiles = (int)((c.N + kMmaRows - 1) / kMmaRows);
  p.status = c.status;
  const int sms = sm_count();
  // Tokens of a tile and blocks that share one: the least time of the busiest block, in cycles.  128 of k take the MMAs four cycles a token, the
  // copies one for each 57 bytes, and decoding and issue 450.  Shared by this rule / one block a tile, us: M=32 N=4096 K=14336 14.8 / 40.3, M=64
  // N=K=4096 8.8 / 14.1, M=128 12.1 / 14.4; by it not shared: M=333 N=K=4096 15.7.
  double best = 1e30;
  unsigned grid = 0;
  const int64_t least = (c.M + kMostTokens - 1) / kMostTokens;
  for (int64_t tt = least; tt <= least + 3; ++tt) {
    const int tokens = (int)(((c.M + tt - 1) / tt + 15) / 16 * 16);
    const int64_t token_tiles = (c.M + tokens - 1) / tokens, tiles = token_tiles * p.row_tiles;
    if (tiles > 0x3FFFFFFF) continue;
    for (int split = 1; split <= kMaxSplit && split <= p.units; split *= 2) {
      const int clusters = split == 1 ? sms : resident_clusters_of(counts[split], w4a16_gemm_kernel<T, kChains>, split, kThreads, kSmemBytes);
      if (clusters < 1) break;
      if (split > 1 && tiles > clusters) break;    // a cluster does one tile
      // An f32 result: chains of all of a block's units (kChain), unless blocks of a cluster, whose chains are all in tensor memory, would need
      // longer ones
      const int own_units = (p.units + split - 1) / split, wanted = kChains ? (own_units + kChain - 1) / kChain : 1;
      const int acc_cols = (tokens + 31) / 32 * 32, chains = split == 1 ? 1 : std::min(wanted, (512 - 2 * 64) / acc_cols);
      if (wanted > 1 && split > 1 && (own_units + chains - 1) / chains > kChain + 1) continue;
      const double unit = std::max(std::max(4.0 * tokens, 450.0), (2.0 * tokens * 128 + 4.0 * kUnitBytes) / 57.0);
      const double waves = (double)((tiles + clusters - 1) / clusters);
      const double cost = waves * ((p.units + split - 1) / split * unit) + 2000.0 + tokens * 20.0 + (split > 1 ? 2000.0 + tokens * 20.0 : 0.0);
      if (cost < best) {
        best = cost;
        p.tokens = tokens;
        p.tiles = (int)tiles;
        p.split = split;
        // Tensor memory: accumulators (two where a block has several tiles), the rest for the weight.  Shared memory: 144 KB of tokens at most, the
        // rest for packed units, whose copies take longest.
        p.acc_cols = (uint32_t)acc_cols;
        p.accs = tiles > clusters || (split == 1 && wanted > 1) ? 2 : 1;
        p.chains = chains;
        p.chain = split == 1 && wanted > 1 ? kChain : (own_units + chains - 1) / chains;
        p.stages = (int)std::min<uint32_t>(kMost, std::min<uint32_t>((512 - std::max(p.accs, p.chains) * p.acc_cols) / 64, 144 * 1024 / ((uint32_t)tokens * 256)));
        // A cluster's sums have room of their own where they are small: nobody waits for the others' MMAs then (M=32 N=4096 K=14336 15.1 us / 15.7,
        // M=64 N=K=4096 9.2 / 9.7).
        const uint32_t sums = split > 1 && tokens <= 64 ? (uint32_t)tokens * kMmaRows * 4 : 0;
        p.sums_at = sums > 0 ? kRingBytes - sums : 0;
        p.w_stages = (int)std::min<uint32_t>(kWMost, (kRingBytes - sums - (uint32_t)p.stages * tokens * 256) / kWStageBytes);
        p.sets = std::min(kDecodeSets, std::min(p.stages, p.w_stages));
        grid = (unsigned)(std::min<int64_t>(clusters, tiles) * split);
        p.last_block = (int)((tiles - 1) % std::min<int64_t>(clusters, tiles)) * split;
      }
    }
  }
  if (grid == 0) return B200FP4_STATUS_NOT_SUPPORTED;
  CUtensorMap map;
  if (!make_rows_map(&map, c.x, (uint64_t)c.M, (uint64_t)c.K * 2, (uint64_t)(c.M > 1 ? c.ldx : c.K) * 2, (uint32_t)p.tokens, 128)) return B200FP4_STATUS_INTERNAL_ERROR;
  if (launch_pdl_cluster(p.split, w4a16_gemm_kernel<T, kChains>, dim3(grid), dim3(kThreads), kSmemBytes, st, map, p) != cudaSuccess) {
    cudaGetLastError();
    return B200FP4_STATUS_EXECUTION_FAILED;
  }
  return finish_launch(1);
}

}  // namespace

int launch_w4a16_gemm(const LinearCall& c, cudaStream_t st) {
  const bool chains = c.out_dtype == B200FP4_DTYPE_F32 && units_of(c.K) > kChain;
  if (c.x_dtype == B200FP4_DTYPE_BF16) return chains ? launch_gemm<__nv_bfloat16, true>(c, st) : launch_gemm<__nv_bfloat16, false>(c, st);
  return chains ? launch_gemm<__half, true>(c, st) : launch_gemm<__half, false>(c, st);
}

}  // namespace b200fp4
