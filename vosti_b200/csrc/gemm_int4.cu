// Product with weights in 4 bits and a scale for each group along k:
//   Y[t, f] = sum_k X[t, k] * c[f, k] * s[f, k / group]       c in -8 .. 7, X and s bfloat16, sums float32
// Layout (what a reader wants next to one another lies next to one another):
//   codes   [features / 16][k / 128][16 rows][4 j][4 i][4 bytes]     a row's 128 codes in 64 bytes; the 32-bit word (j, i) holds k = 32 i +
//                                                                    8 j .. + 7, nibble p the code c + 8 of k offset 2 p (p < 4) or 2 p - 7
//   scales  [features / 16][k / 128][16 rows][128 / group]           bfloat16, group 32, 64 or 128
// A word shifted by 4 p and masked holds the codes of neighbouring k in its halves; with the exponent of 128 or'ed in they are 128 + c + 8 in
// bfloat16, exactly, and minus 136 the codes.
// (The published way of making small integers floating point without a conversion: Kim, Henry, Fahim and Awadalla, "Who Says Elephants Can't Run:
// Bringing Large Scale MoE Models into Cloud Scale Production", 2022, there for float16.)
//
// Gated: tiles of 16 features are taken in pairs, a gate and what it is for, and Y[t, 16 p + i] = silu(gate) * up of pair p, in float32 (24,576 x 4,096,
// us without and with it, and with a kernel of its own behind: 8 tokens 14.5, 14.5, 19.1, 64 25.8, 26.2, 33.8, 2,048 371, 378, 446 under the power cap at
// 1,520 to 1,660 MHz, 316, 322, 385 after a rest at 1,965).
//
// Up to 16 tokens: mma.sync, weights as the 16 rows (int4_few_kernel). What bounds it is the weights' bytes. More tokens: tcgen05
// (int4_tiles_kernel), weights made bfloat16 in tensor memory.
#include "common.cuh"
#include "mma_util.cuh"
#include "tcgen05.cuh"
#include "tensor_map.cuh"

namespace {

constexpr int KB = 128;                    // k of a block of codes: 64 bytes a row
constexpr int TILE_BYTES = 16 * KB / 2;    // codes of 16 rows

// Codes of k offsets 2 P and 2 P + 1 of a word, in bfloat16. The constants are handed over in registers: mask and or are then one
// instruction (with constants in place they were two, and the integer pipe, at half the issue rate, bounded the product).
struct Int4Masks { uint32_t low, base, minus; };
__device__ __forceinline__ Int4Masks int4_masks() {
  Int4Masks m;
  asm volatile("mov.b32 %0, 0x000f000f;" : "=r"(m.low));
  asm volatile("mov.b32 %0, 0x43004300;" : "=r"(m.base));
  asm volatile("mov.b32 %0, 0xc308c308;" : "=r"(m.minus));
  return m;
}
template <int P>
__device__ __forceinline__ uint32_t int4_codes(uint32_t w, const Int4Masks& m) {
  uint32_t t, r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(t) : "r"(w >> (4 * P)), "r"(m.low), "r"(m.base));
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(t), "r"(m.minus));
  return r;
}
__device__ __forceinline__ uint32_t int4_word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint4 load_codes(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// A row's scales of a block of 128 k (N = 1, 2 or 4), two to a word, of which `left` k are the matrix's: what stands for groups beyond
// them (k < 128 in the last block) may be no number and becomes zero.
template <int N>
__device__ __forceinline__ void load_scales(const bf16* p, int left, uint32_t (&s)[(N + 1) / 2]) {
  if constexpr (N == 1) {
    s[0] = *reinterpret_cast<const unsigned short*>(p);
  } else if constexpr (N == 2) {
    s[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    s[0] = v.x;
    s[1] = v.y;
  }
  if (N > 1 && left < KB) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i * (KB / N) >= left) s[i / 2] &= (i & 1) ? 0x0000ffffu : 0xffff0000u;
  }
}
// (the quick division: a divisor beyond 2^126 gives 0, where silu is below 1e-36)
__device__ __forceinline__ float int4_gated(float gate, float up) { return __fdividef(gate, 1.f + __expf(-gate)) * up; }
__device__ __forceinline__ float scale_of(uint32_t word, int i) { return __uint_as_float((i & 1) ? word & 0xffff0000u : word << 16); }

// ---------------------------------------------------------------------------------------------- up to 16 tokens
// A CTA takes FT tiles of 16 features over all of k, each of its eight warps a run of the blocks of 128 k, which comes by bulk copies (a
// tile's codes of neighbouring blocks are contiguous, and so are its scales) into two buffers of 4 KB of the warp's own: with three CTAs an
// SM some 190 KB are on their way from the start. The order of k inside an instruction is free: lane j of a row takes offsets 8 j .. 8 j + 7
// of every 32 k, so that four of them are a word's half and the tokens' 8 are one 16-byte load. An instruction never mixes groups: a group's codes
// are summed exactly, then multiplied by its scale in float32. The warps' sums meet in shared memory, in warp order.
// What bounds it: with many tiles the integer pipe (seven operations at half rate for a word of eight codes: 8 tokens, 151,936 x 4,096 in 74 us, 66% of
// its bytes' rate); with few the chain from launch to the last sum (4,096 x 4,096 5.2, 4,096 x 12,288 11.5 us; 13.3 when a block's addresses and the
// tokens' bounds were worked out block by block).
constexpr int FEW_WARPS = 8, FEW_THREADS = FEW_WARPS * 32;
constexpr int STAGE_CODES = 4096, FEW_STAGES = 2;
template <int GROUPS> __host__ __device__ constexpr int stage_bytes() { return STAGE_CODES + 4 * 32 * GROUPS; }

// 16 bytes of a token's row from element kk on; rows that do not start on whole words are read element by element, zeros beyond k.
template <bool WORDS>
__device__ __forceinline__ uint4 load_tokens(const bf16* row, int kk, int k) {
  if constexpr (WORDS) {
    return kk < k ? *reinterpret_cast<const uint4*>(row + kk) : make_uint4(0, 0, 0, 0);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = kk + 2 * i < k ? reinterpret_cast<const unsigned short*>(row)[kk + 2 * i] : 0;
      const uint32_t hi = kk + 2 * i + 1 < k ? reinterpret_cast<const unsigned short*>(row)[kk + 2 * i + 1] : 0;
      w[i] = lo | hi << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int FT, int NT, int GROUPS, bool WORDS, bool GATED>
__global__ void __launch_bounds__(FEW_THREADS, NT == 1 ? 3 : 2)
int4_few_kernel(const bf16* __restrict__ x, const uint8_t* __restrict__ codes, const bf16* __restrict__ scales, void* __restrict__ y, int y_is_f32,
                int rows, int n, int k, int tiles, int deep, unsigned* status) {
  constexpr int SW = (GROUPS + 1) / 2, DEEP = 4 / FT, SCALES = 32 * GROUPS;       // blocks of k a buffer, bytes of a tile's scales a block
  constexpr int STAGE = stage_bytes<GROUPS>();
  extern __shared__ __align__(128) uint8_t ring[];             // [warp][buffer]: codes [FT][DEEP][1,024], then scales [FT][DEEP][SCALES]
  __shared__ __align__(8) uint64_t full[FEW_WARPS][FEW_STAGES];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r8 = lane >> 2, j = lane & 3;
  const int tile0 = blockIdx.x * FT;
  const Int4Masks masks = int4_masks();
  const int kb_begin = deep * warp / FEW_WARPS, blocks = deep * (warp + 1) / FEW_WARPS - kb_begin, stages = (blocks + DEEP - 1) / DEEP;
  uint8_t* const mine = ring + warp * (FEW_STAGES * STAGE);
  if (lane == 0) {
    for (int i = 0; i < FEW_STAGES; ++i) mb_init(smem_addr(&full[warp][i]), 1);
    mb_fence_init();
  }
  __syncwarp();
  auto request = [&](int st) {                                   // lanes 0 .. FT - 1: a tile's codes and scales
    const int count = min(DEEP, blocks - st * DEEP);
    const uint32_t bar = smem_addr(&full[warp][st % FEW_STAGES]);
    if (lane == 0) mb_expect_tx(bar, (uint32_t)(FT * count * (TILE_BYTES + SCALES)));
    __syncwarp();
    if (lane < FT) {
      uint8_t* const to = mine + st % FEW_STAGES * STAGE;
      const int64_t from = (int64_t)min(tile0 + lane, tiles - 1) * deep + kb_begin + st * DEEP;
      bulk_copy_g2s(smem_addr(to + lane * DEEP * TILE_BYTES), codes + from * TILE_BYTES, (uint32_t)(count * TILE_BYTES), bar);
      bulk_copy_g2s(smem_addr(to + STAGE_CODES + lane * DEEP * SCALES), reinterpret_cast<const uint8_t*>(scales) + from * SCALES, (uint32_t)(count * SCALES), bar);
    }
  };
  // the weights do not depend on the kernel before this one
  for (int st = 0; st < min(stages, FEW_STAGES); ++st) request(st);
  pdl_wait();
  pdl_launch_dependents();
  uint4 b[NT][4];                                                // [8 tokens][32 k] of a block; beyond the last token it again (its column is not stored)
  const bf16* row[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) row[t] = x + (int64_t)min(t * 8 + r8, rows - 1) * k;
  const bool whole = WORDS && k % KB == 0;
  auto load_block = [&](int kb) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if (whole) {
        const uint4* const from = reinterpret_cast<const uint4*>(row[t] + kb * KB + 8 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) b[t][i] = from[4 * i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) b[t][i] = load_tokens<WORDS>(row[t], kb * KB + 32 * i + 8 * j, k);
      }
    }
  };
  if (blocks > 0) load_block(kb_begin);
  float acc[FT][NT][4];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[f][t][0] = acc[f][t][1] = acc[f][t][2] = acc[f][t][3] = 0.f;
  for (int st = 0; st < stages; ++st) {
    const uint32_t bar = smem_addr(&full[warp][st % FEW_STAGES]);
    if (!__all_sync(0xffffffffu, mb_try_wait(bar, (uint32_t)(st / FEW_STAGES) & 1) || mb_wait(bar, (uint32_t)(st / FEW_STAGES) & 1, status))) {
      // reported; once more, so that none of the warp's copies is in flight when it ends
      (void)mb_wait(bar, (uint32_t)(st / FEW_STAGES) & 1, status);
      if (st + 1 < stages) (void)mb_wait(smem_addr(&full[warp][(st + 1) % FEW_STAGES]), (uint32_t)((st + 1) / FEW_STAGES) & 1, status);
      break;
    }
#pragma unroll
    for (int inside = 0; inside < DEEP; ++inside) {
      const int at = st * DEEP + inside;
      if (inside > 0 && at >= blocks) break;
      uint4 now[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) now[t][i] = b[t][i];
      if (at + 1 < blocks) load_block(kb_begin + at + 1);
      const uint8_t* const stage = mine + st % FEW_STAGES * STAGE + inside * TILE_BYTES;
      const bf16* const stage_scales = reinterpret_cast<const bf16*>(mine + st % FEW_STAGES * STAGE + STAGE_CODES + inside * SCALES);
#pragma unroll
      for (int f = 0; f < FT; ++f) {
        uint4 c[2];
        uint32_t s[2][SW];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          c[h] = *reinterpret_cast<const uint4*>(stage + f * DEEP * TILE_BYTES + (r8 + 8 * h) * (KB / 2) + 16 * j);
          load_scales<GROUPS>(stage_scales + f * DEEP * (SCALES / 2) + (r8 + 8 * h) * GROUPS, k - (kb_begin + at) * KB, s[h]);
        }
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          float part[NT][4];
#pragma unroll
          for (int t = 0; t < NT; ++t) part[t][0] = part[t][1] = part[t][2] = part[t][3] = 0.f;
#pragma unroll
          for (int i = g * 4 / GROUPS; i < (g + 1) * 4 / GROUPS; ++i) {
            const uint32_t lo = int4_word(c[0], i), hi = int4_word(c[1], i);
            const uint32_t first[4] = {int4_codes<0>(lo, masks), int4_codes<0>(hi, masks), int4_codes<1>(lo, masks), int4_codes<1>(hi, masks)};
            const uint32_t second[4] = {int4_codes<2>(lo, masks), int4_codes<2>(hi, masks), int4_codes<3>(lo, masks), int4_codes<3>(hi, masks)};
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              mma_bf16(part[t], first, now[t][i].x, now[t][i].y);
              mma_bf16(part[t], second, now[t][i].z, now[t][i].w);
            }
          }
          const float s0 = scale_of(s[0][g / 2], g), s1 = scale_of(s[1][g / 2], g);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            acc[f][t][0] = fmaf(part[t][0], s0, acc[f][t][0]);
            acc[f][t][1] = fmaf(part[t][1], s0, acc[f][t][1]);
            acc[f][t][2] = fmaf(part[t][2], s1, acc[f][t][2]);
            acc[f][t][3] = fmaf(part[t][3], s1, acc[f][t][3]);
          }
        }
      }
    }
    if (st + FEW_STAGES < stages) {
      __syncwarp();                                              // every lane has read the buffer
      request(st + FEW_STAGES);
    }
  }
  __syncthreads();                                               // the buffers' place takes the sums
  constexpr int PITCH = FT * 16 + 4;
  float* const sums = reinterpret_cast<float*>(ring);            // [warp][token][feature]
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[(warp * NT * 8 + t * 8 + 2 * j + (e & 1)) * PITCH + f * 16 + r8 + 8 * (e >> 1)] = acc[f][t][e];
  __syncthreads();
  auto total = [&](int t, int f) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < FEW_WARPS; ++w) v += sums[(w * NT * 8 + t) * PITCH + f];
    return v;
  };
  auto store = [&](int64_t at, float v) {
    if (y_is_f32) reinterpret_cast<float*>(y)[at] = v;
    else reinterpret_cast<bf16*>(y)[at] = __float2bfloat16_rn(v);
  };
  int mine_at;                                                   // (read again here: worked out ahead, places spill registers in the main loop)
  asm volatile("mov.u32 %0, %%tid.x;" : "=r"(mine_at));
  if constexpr (GATED) {
    for (int i = mine_at; i < rows * FT * 8; i += FEW_THREADS) {
      const int t = i / (FT * 8), f = i % (FT * 8), gate = f / 16 * 32 + f % 16;
      if (tile0 * 8 + f < n / 2) store((int64_t)t * (n / 2) + tile0 * 8 + f, int4_gated(total(t, gate), total(t, gate + 16)));
    }
  } else {
    for (int i = mine_at; i < rows * FT * 16; i += FEW_THREADS) {
      const int t = i / (FT * 16), f = i % (FT * 16);
      if (tile0 * 16 + f < n) store((int64_t)t * n + tile0 * 16 + f, total(t, f));
    }
  }
}

// ---------------------------------------------------------------------------------------------- more tokens
// Features on M = 128, TOK tokens on N; k in `segments`, one CTA of a cluster each, summed in their order through distributed shared
// memory. Eight warps read the codes into registers DEPTH blocks ahead (a thread: half a feature's block, one 32-byte sector), make them
// bfloat16 times their scale (rounded once: codes of 1, 2, 4 and 8 are exact) and store them to one of two stages in tensor memory; a
// ninth warp issues the MMAs, a tenth brings the tokens by TMA.
constexpr int FEATURES = 128;
constexpr int A_COLS = KB / 2;

constexpr int MAX_SEGMENTS = 8;

template <int TOK>
struct Int4Tile {
  // Eight warps fill the stages' weights, DEPTH blocks asked for ahead; up to 128 tokens two CTAs share an SM, above two groups of eight
  // warps take a CTA's stages in turn (one CTA with two groups for 24,576 x 4,096 of 128 tokens: 38 us, two with one 32).
  static constexpr int GROUPS = TOK > 128 ? 2 : 1, DEPTH = 4, WORKERS = 256 * GROUPS, THREADS = WORKERS + 64;
  static constexpr int X_STAGE = TOK * KB * 2, STAGES = TOK > 128 ? 3 : TOK > 64 ? 2 : 3;
  // A stage's MMAs are reported on a barrier that goes by the block, and whoever refills a stage waits for the block that held it. With as many
  // barriers as stages and groups have a common multiple of, (1) a waiter's blocks meet a barrier's phases one after another, so that a parity
  // never stands for an earlier phase, and (2) the phase after the awaited one takes the MMAs of a block behind the one that the waiter is about to
  // fill, so that it never stands for a later one, however late the waiter looks.
  static constexpr int REPORTS = STAGES % GROUPS == 0 ? STAGES : STAGES * GROUPS;
  static __host__ __device__ constexpr int report(int block) { return block % REPORTS; }
  static __host__ __device__ constexpr uint32_t report_parity(int block) { return (uint32_t)(block / REPORTS) & 1; }
  static constexpr int COLS = TOK + STAGES * A_COLS <= 256 ? 256 : 512;
  static constexpr int RING = STAGES * X_STAGE, SUMS = TOK * FEATURES * 4;
  // no more CTAs an SM than tensor memory has columns for: shared memory (228 KB, 1 KB of it with every CTA) is padded until that many fit
  static constexpr int FEWEST = 228 * 1024 / (512 / COLS + 1);
  static constexpr int NEEDED = (RING > SUMS ? RING : SUMS) + 1024;
  static constexpr int SMEM = NEEDED > FEWEST ? NEEDED : FEWEST;
  static constexpr int CTAS = 512 / COLS;
};

__device__ __forceinline__ void int4_tmem_store8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ uint32_t int4_times(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float4 int4_load_rank(uint32_t smem_at, uint32_t rank) {
  uint32_t remote;
  float4 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_at), "r"(rank));
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(remote) : "memory");
  return v;
}
// A wait of every lane: 50 cycles where the phase is complete already, as it should be (with the clock read first 105, one lane asking for all 290).
__device__ __forceinline__ bool int4_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, unsigned* status) {
  return mbar_try_wait(bar, parity) || mbar_wait(bar, parity, abort_flag, status);
}
template <int WORKERS>
__device__ __forceinline__ void int4_workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(WORKERS) : "memory"); }

template <int TOK, int GROUPS, bool GATED>
__global__ void __launch_bounds__(Int4Tile<TOK>::THREADS, Int4Tile<TOK>::CTAS)
int4_tiles_kernel(const __grid_constant__ CUtensorMap map_x, const uint8_t* __restrict__ codes, const bf16* __restrict__ scales, void* __restrict__ y,
                  int y_is_f32, int rows, int n, int k, int tiles, int deep, int token_tiles, int segments, unsigned* status) {
  using Tile = Int4Tile<TOK>;
  constexpr int SW = (GROUPS + 1) / 2, WORKERS = Tile::WORKERS, STAGES = Tile::STAGES, DEPTH = Tile::DEPTH, TURNS = Tile::GROUPS;
  constexpr int COLS = TOK / (WORKERS / 128);                    // token columns of a warp at the end
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  // a stage: the tokens have arrived and eight warps have stored the weights; a block's MMAs are complete; all MMAs are
  __shared__ __align__(8) uint64_t full[STAGES], empty[Tile::REPORTS], done;
  __shared__ uint32_t tmem_base_holder;
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int segment = blockIdx.x % segments;
  const int t0 = (blockIdx.x / segments) % token_tiles * TOK, f0 = blockIdx.x / (segments * token_tiles) * FEATURES;
  const int kb_begin = (int)((int64_t)deep * segment / segments), blocks = (int)((int64_t)deep * (segment + 1) / segments) - kb_begin;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) mbar_init(smem_u32(&full[s]), 9);
    for (int r = 0; r < Tile::REPORTS; ++r) mbar_init(smem_u32(&empty[r]), 1);
    mbar_init(smem_u32(&done), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc(smem_u32(&tmem_base_holder), Tile::COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();               // (after this CTA's tensor memory is its own)
  const uint32_t tmem_sum = tmem_base_holder, tmem_a = tmem_sum + TOK;

  if (warp == WORKERS / 32 + 1) {
    if (lane == 0) {
      pdl_wait();
      for (int b = 0; b < blocks; ++b) {
        const int s = b % STAGES;
        if (b >= STAGES && !int4_wait(smem_u32(&empty[Tile::report(b - STAGES)]), Tile::report_parity(b - STAGES), &abort_flag, status)) break;
        mbar_expect_tx(smem_u32(&full[s]), (uint32_t)Tile::X_STAGE);
        for (int h = 0; h < 2; ++h)
          tma_load_2d(smem_u32(smem + s * Tile::X_STAGE + h * (TOK * 128)), &map_x, (kb_begin + b) * KB + h * 64, t0, smem_u32(&full[s]));
      }
    }
    return;
  }
  if (warp == WORKERS / 32) {
    constexpr uint32_t idesc = umma_instr_desc(FEATURES, TOK, false);
    bool ok = true;
    for (int b = 0; b < blocks && ok; ++b) {
      const int s = b % STAGES;
      ok = __all_sync(0xffffffffu, int4_wait(smem_u32(&full[s]), (b / STAGES) & 1, &abort_flag, status)) != 0;
      if (!ok) break;
      tc_fence_after();
      const uint64_t desc = smem_desc_sw128(smem_u32(smem + s * Tile::X_STAGE));
      if (elect_one()) {
#pragma unroll
        for (int q = 0; q < KB / 16; ++q)
          umma_bf16_ts(tmem_sum, tmem_a + s * A_COLS + 8 * q, desc + (uint64_t)(((q >> 2) * (TOK * 128) + (q & 3) * 32) >> 4), idesc, b > 0 || q > 0);
        umma_commit(smem_u32(&empty[Tile::report(b)]));
        if (b + 1 == blocks) umma_commit(smem_u32(&done));
      }
      __syncwarp();
    }
    return;
  }

  // -------------------------------------------------------------- workers
  const int quarter = warp & 3, half = (warp >> 2) & 1, turn = warp >> 3, feature = quarter * 32 + lane;
  const int tile = min(f0 / 16 + feature / 16, tiles - 1);       // (rows beyond the matrix are never stored)
  const int64_t row = ((int64_t)tile * deep + kb_begin) * 16 + feature % 16;
  const uint8_t* const my_codes = codes + row * (KB / 2) + 32 * half;
  const bf16* const my_scales = scales + row * GROUPS;
  const uint32_t my_a = tmem_a + ((uint32_t)(quarter * 32) << 16) + 8 * half;
  const Int4Masks masks = int4_masks();
  uint4 c[DEPTH][2];
  uint32_t sc[DEPTH][SW];
  auto load = [&](int b, int d) {
    const uint8_t* const at = my_codes + (int64_t)b * TILE_BYTES;
    c[d][0] = load_codes(at);
    c[d][1] = load_codes(at + 16);
    load_scales<GROUPS>(my_scales + (int64_t)b * 16 * GROUPS, k - (kb_begin + b) * KB, sc[d]);
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (turn + d * TURNS < blocks) load(turn + d * TURNS, d);
  bool ok = true;
  for (int b0 = turn; b0 < blocks && ok; b0 += DEPTH * TURNS) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int b = b0 + d * TURNS, s = b % STAGES;
      if (b >= blocks || !ok) break;
      if (b >= STAGES) {
        ok = __all_sync(0xffffffffu, int4_wait(smem_u32(&empty[Tile::report(b - STAGES)]), Tile::report_parity(b - STAGES), &abort_flag, status)) != 0;
        if (!ok) break;
        tc_fence_after();                                        // (the MMAs that read the stage)
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int g = i * GROUPS / 4;
        const uint32_t two = __byte_perm(sc[d][g / 2], 0, (g & 1) ? 0x3232 : 0x1010);
        const uint32_t lo = int4_word(c[d][0], i), hi = int4_word(c[d][1], i);
        const uint32_t r[8] = {int4_times(int4_codes<0>(lo, masks), two), int4_times(int4_codes<1>(lo, masks), two), int4_times(int4_codes<2>(lo, masks), two),
                               int4_times(int4_codes<3>(lo, masks), two), int4_times(int4_codes<0>(hi, masks), two), int4_times(int4_codes<1>(hi, masks), two),
                               int4_times(int4_codes<2>(hi, masks), two), int4_times(int4_codes<3>(hi, masks), two)};
        int4_tmem_store8(my_a + s * A_COLS + 16 * i, r);
      }
      if (b + DEPTH * TURNS < blocks) load(b + DEPTH * TURNS, d);
      tmem_wait_stores();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&full[s]));
    }
  }
  // (a barrier of its own: a group of warps that never waited for a stage's earlier phase could take it for the last)
  if (ok && blocks > 0) ok = __all_sync(0xffffffffu, int4_wait(smem_u32(&done), 0, &abort_flag, status)) != 0;
  tc_fence_after();
  pdl_wait();                                                    // (what this kernel writes may still be read before that)

  const uint32_t my_sums = tmem_sum + ((uint32_t)(quarter * 32) << 16) + (warp >> 2) * COLS;
  float* const part = reinterpret_cast<float*>(smem);            // [TOK][128] sums (every MMA that read the ring is complete)
  constexpr int STEP = COLS < 32 ? COLS : 32;
  for (int c0 = 0; c0 < COLS && blocks > 0; c0 += STEP) {
    uint32_t r[32];
    if constexpr (STEP == 32) {
      tmem_load32(my_sums + c0, r);
    } else {
      asm volatile(
          "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
          : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
            "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
          : "r"(my_sums + c0));
      tmem_wait_loads();
    }
#pragma unroll
    for (int i = 0; i < STEP; ++i) part[((warp >> 2) * COLS + c0 + i) * FEATURES + feature] = __uint_as_float(r[i]);
  }
  tc_fence_before();
  // Four neighbouring features of a token at a time, so that a warp writes whole rows (each warp its 32 features: 64 bytes a store).
  constexpr int WORDS = GATED ? FEATURES / 8 : FEATURES / 4;
  const int wide = GATED ? n / 2 : n, first = GATED ? f0 / 2 : f0;
  const bool quads = wide % 4 == 0 && (uintptr_t)y % 16 == 0;
  auto store = [&](int t, int f, const float4& v) {
    if (first + f >= wide) return;
    const int64_t at = (int64_t)(t0 + t) * wide + first + f;
    if (quads) {
      if (y_is_f32) store_four(reinterpret_cast<float*>(y) + at, v);
      else store_four(reinterpret_cast<bf16*>(y) + at, v);
      return;
    }
    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (first + f + i >= wide) return;
      if (y_is_f32) reinterpret_cast<float*>(y)[at + i] = e[i];
      else reinterpret_cast<bf16*>(y)[at + i] = __float2bfloat16_rn(e[i]);
    }
  };
  // (`total` sums four features of a token)
  auto finish = [&](int t, int word, auto total) {
    const int f = word * 4;
    if constexpr (GATED) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f), gate = v;
#pragma unroll 1                                                 // (both at once do not fit the registers)
      for (int side = 0; side < 2; ++side) {
        gate = v;
        v = total(t, f / 16 * 32 + f % 16 + 16 * side);
      }
      store(t, f, make_float4(int4_gated(gate.x, v.x), int4_gated(gate.y, v.y), int4_gated(gate.z, v.z), int4_gated(gate.w, v.w)));
    } else {
      store(t, f, total(t, f));
    }
  };
  if (segments == 1) {
    int4_workers_sync<WORKERS>();
    const int count = min(TOK, rows - t0);
    for (int word = threadIdx.x; word < count * WORDS; word += WORKERS)
      finish(word / WORDS, word % WORDS, [&](int t, int f) { return *reinterpret_cast<const float4*>(part + t * FEATURES + f); });
  } else {
    // the segments' sums in their order, each CTA a share of the tokens (the roles that bring and issue have ended: every thread of the cluster
    // that is left takes part)
    cluster_sync_all();
    const int lo = TOK * segment / segments, hi = min(TOK * (segment + 1) / segments, rows - t0);
    for (int word = threadIdx.x; word < (hi - lo) * WORDS; word += WORKERS)
      finish(lo + word / WORDS, word % WORDS, [&](int t, int f) {
        const uint32_t at = smem_u32(&part[t * FEATURES + f]);
        // (all of them on their way at once: one after the other, eight took 4 us)
        float4 u[MAX_SEGMENTS];
#pragma unroll
        for (int r = 0; r < MAX_SEGMENTS; ++r)
          if (r < segments) u[r] = int4_load_rank(at, r);
        float4 v = u[0];
#pragma unroll
        for (int r = 1; r < MAX_SEGMENTS; ++r)
          if (r < segments) {
            v.x += u[r].x;
            v.y += u[r].y;
            v.z += u[r].z;
            v.w += u[r].w;
          }
        return v;
      });
    cluster_sync_all();                                          // nobody reads this CTA's sums after this
  }
  int4_workers_sync<WORKERS>();
  if (abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
    int4_workers_sync<WORKERS>();
  }
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem_sum, Tile::COLS);
  }
}

// Segments of k: as many as still find an SM at once, each of eight blocks at least, of four where few CTAs are at work. us at 1, 2, 4 and 8: 64
// tokens, 4,096 x 4,096 16.9, 12.4, 10.2 and 11.5, 4,096 x 12,288 42, 25, 19.6 and 16.7, 24,576 x 4,096 28, 31, 37 and 61, 128 x 4,096 15.9, 11.5, 8.0 and 6.9.
int int4_segments(int64_t ctas, int deep, int at_once) {
  int s = 1;
  while (s < MAX_SEGMENTS && ctas * s * 2 <= at_once && deep >= (ctas * s * 2 <= 64 ? 8 : 16) * s) s *= 2;
  return s;
}

struct Int4Args {
  const bf16* x;
  const uint8_t* codes;
  const bf16* scales;
  void* y;
  int y_is_f32, gated, rows, n, k, tiles, deep;
  unsigned* status;
  cudaStream_t stream;
};

template <int FT, int NT, int GROUPS, bool WORDS, bool GATED = false>
cudaError_t launch_few(const Int4Args& a) {
  auto kernel = int4_few_kernel<FT, NT, GROUPS, WORDS, GATED>;
  constexpr int SMEM = FEW_WARPS * FEW_STAGES * stage_bytes<GROUPS>();
  static_assert(FEW_WARPS * NT * 8 * (FT * 16 + 4) * 4 <= SMEM, "the sums take the buffers' place");
  const cudaError_t raised = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (raised != cudaSuccess) return raised;
  return vosti_launch(kernel, dim3((a.tiles + FT - 1) / FT), dim3(FEW_THREADS), SMEM, a.stream, a.x, a.codes, a.scales, a.y, a.y_is_f32, a.rows, a.n, a.k,
                      a.tiles, a.deep, a.status);
}
// Tiles of 16 features a CTA: as many as leave two CTAs an SM. us, 8 tokens, two and four of them: 24,576 x 4,096 18.7 and 14.8, 151,936 x 4,096 89 and 74.
template <int GROUPS, int NT>
cudaError_t launch_few_as(const Int4Args& a, bool words) {
  if (a.gated) return a.tiles >= 4 * 296 ? launch_few<4, NT, GROUPS, true, true>(a) : launch_few<2, NT, GROUPS, true, true>(a);      // (tiles in pairs)
  if (!words) return launch_few<1, NT, GROUPS, false>(a);
  if (a.tiles >= 4 * 296) return launch_few<4, NT, GROUPS, true>(a);
  return a.tiles >= 2 * 296 ? launch_few<2, NT, GROUPS, true>(a) : launch_few<1, NT, GROUPS, true>(a);
}
template <int GROUPS>
cudaError_t launch_few_groups(const Int4Args& a, bool words) {
  return a.rows <= 8 ? launch_few_as<GROUPS, 1>(a, words) : launch_few_as<GROUPS, 2>(a, words);
}

template <int TOK, int GROUPS>
int launch_tiles(const Int4Args& a) {
  auto kernel = a.gated ? int4_tiles_kernel<TOK, GROUPS, true> : int4_tiles_kernel<TOK, GROUPS, false>;
  constexpr int SMEM = Int4Tile<TOK>::SMEM;
  const cudaError_t raised = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  VOSTI_REQUIRE(raised == cudaSuccess, "gemm_int4: %s", cudaGetErrorString(raised));
  CUtensorMap map;
  VOSTI_REQUIRE(encode_tensor_map_2d(&map, a.x, a.rows, a.k, TOK, 64), "gemm_int4: cuTensorMapEncodeTiled failed");
  const int token_tiles = (a.rows + TOK - 1) / TOK;
  const int64_t whole = (int64_t)((a.n + FEATURES - 1) / FEATURES) * token_tiles;
  const int segments = int4_segments(whole, a.deep, 140 * Int4Tile<TOK>::CTAS);
  VOSTI_REQUIRE(whole * segments <= 0x7fffffff, "gemm_int4: too many tiles for one launch");
  const cudaError_t e = vosti_launch_clusters(kernel, dim3((unsigned)(whole * segments)), dim3(Int4Tile<TOK>::THREADS), (unsigned)segments, SMEM, a.stream, map,
                                              a.codes, a.scales, a.y, a.y_is_f32, a.rows, a.n, a.k, a.tiles, a.deep, token_tiles, segments, a.status);
  VOSTI_REQUIRE(e == cudaSuccess, "gemm_int4: %s", cudaGetErrorString(e));
  return VOSTI_OK;
}
template <int GROUPS>
int launch_tiles_as(const Int4Args& a) {
  if (a.rows <= 32) return launch_tiles<32, GROUPS>(a);
  if (a.rows <= 64) return launch_tiles<64, GROUPS>(a);
  if (a.rows <= 128) return launch_tiles<128, GROUPS>(a);
  return launch_tiles<256, GROUPS>(a);
}

}  // namespace

// Tensor memory columns that the CTAs of a token tile (0 .. 3, -1 beyond) may ask for on one SM.
VOSTI_API int vosti_gemm_int4_columns_an_sm(int tile) {
  auto of = [](int smem, int cols) { return 228 * 1024 / (smem + 1024) * cols; };
  switch (tile) {
    case 0: return of(Int4Tile<32>::SMEM, Int4Tile<32>::COLS);
    case 1: return of(Int4Tile<64>::SMEM, Int4Tile<64>::COLS);
    case 2: return of(Int4Tile<128>::SMEM, Int4Tile<128>::COLS);
    case 3: return of(Int4Tile<256>::SMEM, Int4Tile<256>::COLS);
  }
  return -1;
}

// What the roles of a token tile (0 .. 3) do about block `block`: out = {stages, groups of warps, barrier that reports its MMAs, barrier and parity
// waited for before its stage is filled (barrier -1: none)}.
VOSTI_API int vosti_gemm_int4_schedule(int tile, int block, int* out) {
  auto of = [&](auto kind) {
    using Tile = decltype(kind);
    const int held = block - Tile::STAGES;
    out[0] = Tile::STAGES;
    out[1] = Tile::GROUPS;
    out[2] = Tile::report(block);
    out[3] = held >= 0 ? Tile::report(held) : -1;
    out[4] = held >= 0 ? (int)Tile::report_parity(held) : 0;
    return VOSTI_OK;
  };
  VOSTI_REQUIRE(block >= 0 && out != nullptr && tile >= 0 && tile <= 3, "gemm_int4: no such tile or block");
  return tile == 0 ? of(Int4Tile<32>()) : tile == 1 ? of(Int4Tile<64>()) : tile == 2 ? of(Int4Tile<128>()) : of(Int4Tile<256>());
}

// x: bfloat16 [rows, k]; codes, scales: as at the top of this file, for n features and k, group 32, 64 or 128; y: [rows, n] bfloat16, or
// float32 with y_is_f32. `gated`: y [rows, n / 2], n a multiple of 32, k one of 8 and x on 16 bytes.
VOSTI_API int vosti_gemm_int4(const void* x, const void* codes, const void* scales, void* y, int y_is_f32, int gated, int rows, int n, int k, int group,
                              unsigned* status, cudaStream_t stream) {
  VOSTI_REQUIRE(rows >= 0 && n > 0 && k > 0, "gemm_int4: bad sizes rows=%d n=%d k=%d", rows, n, k);
  VOSTI_REQUIRE(group == 32 || group == 64 || group == 128, "gemm_int4: the group is 32, 64 or 128, not %d", group);
  VOSTI_REQUIRE((((uintptr_t)codes | (uintptr_t)scales) & 15) == 0, "gemm_int4: the weights must start on 16 bytes");
  if (rows == 0) return VOSTI_OK;
  Int4Args a = {(const bf16*)x, (const uint8_t*)codes, (const bf16*)scales, y, y_is_f32, gated != 0, rows, n, k, (n + 15) / 16, (k + KB - 1) / KB, status, stream};
  // whole words of eight tokens' elements: every row starts on 16 bytes
  const bool words = k % 8 == 0 && ((uintptr_t)x & 15) == 0;
  VOSTI_REQUIRE(!gated || (n % 32 == 0 && words), "gemm_int4: a gated product takes 32 features at a time and rows that start on 16 bytes");
  if (rows > 16 && words) {
    const int code = group == 32 ? launch_tiles_as<4>(a) : group == 64 ? launch_tiles_as<2>(a) : launch_tiles_as<1>(a);
    if (code != VOSTI_OK) return code;
    VOSTI_LAUNCH_CHECK();
  }
  for (int t = 0; t < rows; t += 16) {                           // (more than one turn only where rows do not start on whole words)
    a.x = (const bf16*)x + (int64_t)t * k;
    a.y = (uint8_t*)y + (int64_t)t * n * (y_is_f32 ? 4 : 2);
    a.rows = rows - t < 16 ? rows - t : 16;
    const cudaError_t e = group == 32 ? launch_few_groups<4>(a, words) : group == 64 ? launch_few_groups<2>(a, words) : launch_few_groups<1>(a, words);
    if (e != cudaSuccess) {
      vosti_set_error("gemm_int4: %s", cudaGetErrorString(e));
      return (int)e;
    }
  }
  VOSTI_LAUNCH_CHECK();
}
