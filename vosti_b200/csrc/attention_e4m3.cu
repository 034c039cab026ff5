// Attention of single tokens over the paged cache of 8 bits (e4m3.cuh):
//   out[t, h] = sum_j softmax_j(scale q[t, h] . k_j) v_j      over the request's keys j <= position (the last `window` of them)
// with k_j = payload * 2^(scale - 127), float32 scores, statistics and sums; 0 where nothing is visible. The semantics are
// attention_decode.cu's (kernels/triton_kernels/fattn_paged.py:176-252).
//
// Two kernels: one on the tensor cores for bfloat16 and head sizes 64 and 128, one on the CUDA cores for the rest.
#include <mutex>
#include <unordered_map>

#include "common.cuh"
#include "e4m3.cuh"
#include "mma_util.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct CacheArgs {
  const uint8_t *k, *v, *k_scale, *v_scale;
  const int* block_table;        // [requests, max_pages]
  int max_pages, page_size, num_pages;
};

// ---------------------------------------------------------------------------------------------- tensor cores
// One CTA for (token, kv head, up to 8 of its query heads, segment of the visible keys); the segments of a token and kv head form a cluster.
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that the 16 rows of an m16n8k16 instruction are keys and
// features, all of them needed, and the 8 columns query heads. A warp takes 64 keys at a time, by bulk copies (a block's keys, or
// values, are contiguous) into a buffer of its own for each, refilled as soon as it has been read: what is in flight costs no registers, so an
// SM holds twelve warps instead of eight and ends of CTAs overlap others' middles (us, straight into registers / so, 8 kv heads: 48 tokens at 512
// keys 18.8 / 12.3, at 2,048 52 / 37, 96 at 600 to 3,500 80 / 65, eight at 16,384 51 / 48).
//   * the order of the summed index is free as long as both operands share it. A lane's 16 bytes of a key row are features
//     64 c + 16 j .. + 15 (j = lane % 4): four k-steps of four features. Rows of S^T are chosen so that the weights come out
//     where the second product wants them: row r of step s is token 4 s + r % 2 (+ 2 for rows 8 to 15) of block r % 8 / 2.
//   * a lane's 16 bytes of a value row are one feature's 16 tokens of block j: four k-steps of four tokens.
//   * the weights turn from (key, head) into (head, key) by movmatrix on pairs rounded to float16.
// Payloads become float16, exactly, by one conversion for two of them; scales never touch them. A lane's scores are all of one block, so the
// keys' scale is a factor of the scores, and the values' one joins the weights in the exponent: the products sum
// 2^(s_j + log2 scale_j - M + 15) payload_j with a running maximum M of s_j + log2 scale_j of their own, so that a weight is 2^15 at
// most whatever the scales are, and full float16 precision reaches 2^-29 of the largest (2^-39 of it is the smallest), while the denominator sums
// 2^(s_j - m) under the scores' own maximum. Queries become float16 too, a row times the power of two that brings
// its largest to 2^14 .. 2^15: exact down to 2^-28 of it.
// What bounds it is the cache's bytes. (Payloads made bfloat16 by moving their bits, four integer instructions and a multiplication for two, kept
// the integer pipe busy: 96 us for 64 tokens at 600 to 3,500 keys, 75 for eight at 16,384.)
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int RESIDENT = 3;                // CTAs an SM holds of the kernel's registers and buffers
constexpr int TILE = 64;                   // keys of a warp's step: four blocks
constexpr int HEADS = 8;                   // query heads of a CTA
constexpr int MAX_SEGMENTS = 16;
constexpr int MAX_ORDERED = 256;           // tokens of a launch that starts with the longest

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Payload bytes 0 and 1 (2 and 3) of a word in float16.
__device__ __forceinline__ uint32_t lower_f16(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t upper_f16(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank_of() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_at_rank(float* p, uint32_t rank, float v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}

template <int D>
__global__ void __launch_bounds__(THREADS, RESIDENT)
attention_e4m3_kernel(const bf16* __restrict__ q, bf16* __restrict__ out, const CacheArgs c, const int* __restrict__ token_list,
                      const int* __restrict__ positions, const int* __restrict__ request_of, int nq, int nkv, float scale_log2, int window,
                      int segments, int ordered, int beside, int appended, unsigned* status) {
  constexpr int CHUNKS = D / 64, FT = D / 16;
  constexpr int RAISED = 15;
  // a warp's buffers: four blocks of keys, and four of values whose starts lie 32 bytes apart in the banks (lanes read all four at once)
  constexpr int BLOCK_BYTES = E4M3_BLOCK * D, V_STRIDE = BLOCK_BYTES + 32, WARP_BYTES = 4 * (BLOCK_BYTES + V_STRIDE);
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[WARPS][2];             // a warp's keys, its values
  float (*const part)[HEADS][D + 4] = reinterpret_cast<float (*)[HEADS][D + 4]>(ring);      // at the end: the warps' products, under the CTA's maximum
  __shared__ float stats[WARPS][HEADS][3];                     // m, sum, M
  __shared__ float inbox[HEADS * D + MAX_SEGMENTS];            // of each segment, its products of this CTA's share of the row
  __shared__ float inbox_stats[MAX_SEGMENTS][HEADS][3];
  if (segments > 1) cluster_arrive();                          // (waited for before the first store to another CTA)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = lane & 3, r8 = lane >> 2;
  const int group = nq / nkv, halves = (group + HEADS - 1) / HEADS;
  const int seg = segments > 1 ? (int)cluster_rank_of() : 0;
  int item = blockIdx.x / segments;
  const int part_of_group = item % halves;
  item /= halves;
  const int g = item % nkv;
  item /= nkv;
  if (ordered > 0) {
    // CTAs that start later than others take the tokens with fewer keys: the item's place is a rank among all tokens
    __shared__ __align__(16) int keys_of[MAX_ORDERED];
    __shared__ int chosen;
    for (int i = threadIdx.x; i < (ordered + 3) / 4 * 4; i += THREADS) {
      const int p = i < ordered ? positions[token_list ? token_list[i] : i] : -1;
      keys_of[i] = i < ordered ? p - first_visible_key(p, window) : -0x7fffffff;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ordered; i += THREADS) {
      const int mine = keys_of[i];
      int rank = 0;
      for (int k = 0; k < ordered; k += 4) {
        const int4 v = *reinterpret_cast<const int4*>(keys_of + k);
        rank += (v.x > mine || (v.x == mine && k < i)) + (v.y > mine || (v.y == mine && k + 1 < i)) + (v.z > mine || (v.z == mine && k + 2 < i)) +
                (v.w > mine || (v.w == mine && k + 3 < i));
      }
      if (rank == item) chosen = i;
    }
    __syncthreads();
    item = chosen;
  }
  const int t = token_list ? token_list[item] : item;
  const int heads = min(HEADS, group - part_of_group * HEADS);
  const int64_t q_at = ((int64_t)t * nq + g * group + part_of_group * HEADS) * D;
  const int pos = positions[t], req = request_of[t];
  const int kstart = first_visible_key(pos, window);
  // this CTA's tiles: the visible ones in `segments` nearly equal runs; the warps take them in turn
  const int first = kstart / TILE, count = pos >= 0 ? pos / TILE - first + 1 : 0;
  const int begin = first + (int)((int64_t)count * seg / segments), end = first + (int)((int64_t)count * (seg + 1) / segments);
  const int blocks_a_page = c.page_size / E4M3_BLOCK;
  const int* const table = c.block_table + (int64_t)req * c.max_pages;

  // index of block `lane % 4` of a tile among the cache's blocks, -1 where nothing of it is visible
  auto block_of = [&](int tile) {
    const int key0 = tile * TILE + j * E4M3_BLOCK;
    if (tile >= end || key0 > pos || key0 + E4M3_BLOCK <= kstart) return (int64_t)-1;
    const int index = key0 / c.page_size;
    int page = index < c.max_pages ? table[index] : -1;
    if (page < 0 || page >= c.num_pages) {
      raise_fault(status, VOSTI_FAULT_PAGE_RANGE);
      page = 0;
    }
    return ((int64_t)page * nkv + g) * blocks_a_page + (key0 - index * c.page_size) / E4M3_BLOCK;
  };

  uint8_t* const keys_s = ring + warp * WARP_BYTES;
  uint8_t* const values_s = keys_s + 4 * BLOCK_BYTES;
  const uint32_t bar[2] = {smem_addr(&full[warp][0]), smem_addr(&full[warp][1])};
  if (lane == 0) {
    mb_init(bar[0], 1);
    mb_init(bar[1], 1);
    mb_fence_init();
  }
  __syncwarp();
  // the visible blocks of a tile (lane j < 4 names block j) into the keys' or the values' buffer
  auto request = [&](int side, int64_t block) {
    const unsigned some = __ballot_sync(0xffffffffu, lane < 4 && block >= 0);
    if (lane == 0) mb_expect_tx(bar[side], (uint32_t)(__popc(some) * BLOCK_BYTES));
    __syncwarp();
    if (lane < 4 && block >= 0)
      bulk_copy_g2s(smem_addr(side == 0 ? keys_s + lane * BLOCK_BYTES : values_s + lane * V_STRIDE), (side == 0 ? c.k : c.v) + block * BLOCK_BYTES,
                    BLOCK_BYTES, bar[side]);
  };
  int k_exp = 0, v_exp = 0;                                    // scales of block lane / 8, the block of this lane's scores
  auto load_scales = [&](int64_t block) {
    const int64_t mine = __shfl_sync(0xffffffffu, block, lane >> 3);
    k_exp = mine >= 0 ? c.k_scale[mine] : 0;
    v_exp = mine >= 0 ? c.v_scale[mine] : 0;
  };
  // A wait that runs out is reported, and the warp stops; before, it waits once more for what it has in flight (`other`: the other side too).
  auto arrived = [&](int side, uint32_t parity, bool other, uint32_t other_parity) {
    const bool ok = mb_try_wait(bar[side], parity) || mb_wait(bar[side], parity, status);    // (asked once before the clock is read)
    if (__all_sync(0xffffffffu, ok)) return true;
    (void)mb_wait(bar[side], parity, status);
    if (other) (void)mb_wait(bar[side ^ 1], other_parity, status);
    return false;
  };

  // `beside`: the kernel before this one is the same step's attention of portions, which neither writes what this one reads nor reads what it
  // writes, and waited for everything before it in all of its CTAs before it let this one start. The last CTA alone waits for it, at its end:
  // this kernel then ends after it (the chain of completed kernels stays unbroken), while CTAs that are done leave their place to others.
  int64_t next = block_of(begin + warp);
  auto start = [&] {
    request(0, next);
    request(1, next);
    load_scales(next);
  };
  // `appended` > 0: the kernel before this one writes, of what is read here, the blocks of the requests' newest `appended` tokens and nothing
  // else; a first tile before them is asked for at once (it is aligned to blocks).
  const bool early = appended > 0 && begin + warp < end && (begin + warp + 1) * TILE <= pos - appended + 1;
  if (early) start();
  if (!beside) pdl_wait();
  pdl_launch_dependents();
  if (!early && begin + warp < end) start();
  uint32_t qb[CHUNKS][4][2];                                   // Q^T: [chunk][k-step][features 4 w, + 2]
  float q_scale[2];                                            // what heads 2 j and 2 j + 1 were divided by, times scale_log2
  {
    uint4 raw[CHUNKS][2];
    uint32_t top = 0;                                          // largest size of the row, as bits of a bfloat16
#pragma unroll
    for (int ch = 0; ch < CHUNKS; ++ch) {
      raw[ch][0] = raw[ch][1] = make_uint4(0, 0, 0, 0);
      if (r8 < heads) {
        const uint4* const at = reinterpret_cast<const uint4*>(q + q_at + (int64_t)r8 * D + 64 * ch + 16 * j);
        raw[ch][0] = at[0];
        raw[ch][1] = at[1];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = word_of(raw[ch][i >> 2], i & 3) & 0x7fff7fffu;
        top = max(top, max(w & 0xffffu, w >> 16));
      }
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^(14 - exponent) as exponent bits, and its inverse
    const int biased = min(max((int)(top >> 7), 15), 254);
    const float up = __uint_as_float((uint32_t)(268 - biased) << 23), down = __uint_as_float((uint32_t)(biased - 14) << 23);
#pragma unroll
    for (int ch = 0; ch < CHUNKS; ++ch)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = word_of(raw[ch][i >> 2], i & 3);
        qb[ch][i >> 1][i & 1] = pack_f16(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) q_scale[h] = __shfl_sync(0xffffffffu, down, (2 * j + h) * 4) * scale_log2;
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};      // of heads 2 j and 2 j + 1
  float mv[2] = {-INFINITY, -INFINITY};                        // the products' M
  float o[FT][4];
#pragma unroll
  for (int i = 0; i < FT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  uint32_t parity = 0;
  for (int tile = begin + warp; tile < end; tile += WARPS, parity ^= 1) {
    next = block_of(tile + WARPS);
    if (!arrived(0, parity, true, parity)) break;

    // ---- S^T = K Q^T
    float s[4][4];
    const float k_times = e4m3_scale(k_exp);
    const float v_log = v_exp == E4M3_NAN_SCALE ? __uint_as_float(0x7fffffffu) : (float)(v_exp - 127);
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      s[st][0] = s[st][1] = s[st][2] = s[st][3] = 0.f;
#pragma unroll
      for (int ch = 0; ch < CHUNKS; ++ch) {
        const uint8_t* const at = keys_s + (lane >> 3) * BLOCK_BYTES + (4 * st + (r8 & 1)) * D + 64 * ch + 16 * j;
        const uint4 rows[2] = {*reinterpret_cast<const uint4*>(at), *reinterpret_cast<const uint4*>(at + 2 * D)};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t lo = word_of(rows[0], w), hi = word_of(rows[1], w);
          const uint32_t a[4] = {lower_f16(lo), lower_f16(hi), upper_f16(lo), upper_f16(hi)};
          mma_f16(s[st], a, qb[ch][w][0], qb[ch][w][1]);
        }
      }
    }
    __syncwarp();                                              // every lane has read the keys
    if (tile + WARPS < end) {
      request(0, next);
      load_scales(next);
    }

    // ---- online softmax of the lane's two heads over the warp's 64 keys
    const int key_lane = tile * TILE + (lane >> 3) * E4M3_BLOCK + (r8 & 1);        // + 4 st (+ 2)
    const bool edge = tile * TILE < kstart || tile * TILE + TILE - 1 > pos;
    const float factor[2] = {q_scale[0] * k_times, q_scale[1] * k_times};
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[st][e] *= factor[e & 1];
        if (edge) {
          const int key = key_lane + 4 * st + (e >> 1) * 2;
          if (key < kstart || key > pos) s[st][e] = -INFINITY;
        }
        top[e & 1] = fmaxf(top[e & 1], s[st][e]);
      }
    float alpha[2];
    uint32_t p[4][2];                                          // P^T: [step][tokens 4 s, + 2]
    {
      float w[4][4];                                           // the products' weights
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top_v = top[h] + v_log;
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) {
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], x));
          top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, x));
        }
        const float m_new = fmaxf(m[h], top[h]), safe = m_new == -INFINITY ? 0.f : m_new;
        const float mv_new = fmaxf(mv[h], top_v), less = v_log + RAISED - (mv_new == -INFINITY ? 0.f : mv_new);
        const float keep = fast_exp2(m[h] - safe);
        alpha[h] = mv_new == mv[h] ? 1.f : fast_exp2(mv[h] - mv_new);
        m[h] = m_new;
        mv[h] = mv_new;
        float sum = 0.f;
#pragma unroll
        for (int st = 0; st < 4; ++st)
#pragma unroll
          for (int e = h; e < 4; e += 2) {
            sum += fast_exp2(s[st][e] - safe);
            w[st][e] = fast_exp2(s[st][e] + less);
            if (edge && s[st][e] == -INFINITY) w[st][e] = 0.f;  // (a scale that is no number)
          }
        l[h] = l[h] * keep + sum;                              // the lane's share; added up at the end
      }
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        p[st][0] = turn8x8(pack_f16(w[st][0], w[st][1]));
        p[st][1] = turn8x8(pack_f16(w[st][2], w[st][3]));
      }
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < FT; ++i) {
        o[i][0] *= alpha[0];
        o[i][1] *= alpha[1];
        o[i][2] *= alpha[0];
        o[i][3] *= alpha[1];
      }
    }

    // ---- O^T += V^T P^T
    // (bytes of tokens that are not visible become zeros: whatever they hold must not meet a weight of zero)
    const int key0 = tile * TILE + j * E4M3_BLOCK;
    uint32_t seen[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
    if (edge) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        seen[w] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (key0 + 4 * w + b >= kstart && key0 + 4 * w + b <= pos) seen[w] |= 0xffu << (8 * b);
      }
    }
    if (!arrived(1, parity, tile + WARPS < end, parity ^ 1)) break;
    auto product = [&](bool masked) {
#pragma unroll
      for (int i = 0; i < FT; ++i) {
        const uint8_t* const at = values_s + j * V_STRIDE + (16 * i + r8) * E4M3_BLOCK;
        const uint4 rows[2] = {*reinterpret_cast<const uint4*>(at), *reinterpret_cast<const uint4*>(at + 8 * E4M3_BLOCK)};
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          uint32_t lo = word_of(rows[0], st), hi = word_of(rows[1], st);
          if (masked) {
            lo &= seen[st];
            hi &= seen[st];
          }
          const uint32_t a[4] = {lower_f16(lo), lower_f16(hi), upper_f16(lo), upper_f16(hi)};
          mma_f16(o[i], a, p[st][0], p[st][1]);
        }
      }
    };
    if (edge) product(true);
    else product(false);
    __syncwarp();                                              // every lane has read the values
    if (tile + WARPS < end) request(1, next);
  }

  // ---- the warps' sums into one, in warp order
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int x = 4; x <= 16; x <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], x);
    if (r8 == 0) {
      stats[warp][2 * j + h][0] = m[h];
      stats[warp][2 * j + h][1] = l[h];
      stats[warp][2 * j + h][2] = mv[h];
    }
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, stats[w][2 * j + h][2]);
    const float weight = fast_exp2(mv[h] - (top == -INFINITY ? 0.f : top));
    float* const to = part[warp][2 * j + h];
#pragma unroll
    for (int i = 0; i < FT; ++i) {
      to[16 * i + r8] = o[i][h] * weight;
      to[16 * i + 8 + r8] = o[i][h + 2] * weight;
    }
  }
  __syncthreads();
  // (m, sum, M) of a head over all records of `from`
  struct Stats { float m, sum, mv; };
  auto joined = [](const float (*from)[HEADS][3], int count, int h) {
    Stats r = {-INFINITY, 0.f, -INFINITY};
    for (int w = 0; w < count; ++w) {
      r.m = fmaxf(r.m, from[w][h][0]);
      r.mv = fmaxf(r.mv, from[w][h][2]);
    }
    const float safe = r.m == -INFINITY ? 0.f : r.m;
    for (int w = 0; w < count; ++w) r.sum += from[w][h][1] * fast_exp2(from[w][h][0] - safe);
    return r;
  };
  // products / 2^RAISED, divided by the sum, their maximum against the scores'
  auto finish = [](float v, const Stats& r) {
    const float safe = r.m == -INFINITY ? 0.f : r.m, safe_v = r.mv == -INFINITY ? 0.f : r.mv;
    return __float2bfloat16_rn(r.sum == 0.f ? 0.f : v * (1.f / (1 << RAISED)) / r.sum * exp2f(safe_v - safe));
  };
  const int total = heads * D;
  if (segments == 1) {
    for (int i = threadIdx.x; i < total; i += THREADS) {
      const int h = i / D, f = i % D;
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) v += part[w][h][f];
      out[q_at + i] = finish(v, joined(stats, WARPS, h));
    }
    if (beside && blockIdx.x == gridDim.x - 1) pdl_wait();
    return;
  }
  // ---- the segments' sums into one, in their order: each CTA of the cluster is sent its share of the row by all of them
  const int share = (total + segments - 1) / segments;
  cluster_wait();
  for (int i = threadIdx.x; i < total; i += THREADS) {
    const int h = i / D, f = i % D;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += part[w][h][f];
    store_at_rank(&inbox[seg * share + i % share], i / share, v);
  }
  for (int i = threadIdx.x; i < heads * segments; i += THREADS) {
    const int h = i / segments;
    const Stats r = joined(stats, WARPS, h);
    store_at_rank(&inbox_stats[seg][h][0], i % segments, r.m);
    store_at_rank(&inbox_stats[seg][h][1], i % segments, r.sum);
    store_at_rank(&inbox_stats[seg][h][2], i % segments, r.mv);
  }
  cluster_arrive();
  cluster_wait();                                              // all of it has arrived; nobody stores to this CTA after this
  for (int i = threadIdx.x; i < share && seg * share + i < total; i += THREADS) {
    const int h = (seg * share + i) / D;
    const Stats r = joined(inbox_stats, segments, h);
    const float safe_v = r.mv == -INFINITY ? 0.f : r.mv;
    float v = 0.f;
    for (int s = 0; s < segments; ++s) v += inbox[s * share + i] * fast_exp2(inbox_stats[s][h][2] - safe_v);
    out[q_at + seg * share + i] = finish(v, r);
  }
  if (beside && blockIdx.x == gridDim.x - 1) pdl_wait();
}

// ---------------------------------------------------------------------------------------------- CUDA cores
constexpr int SIMT_WARPS = 4, SIMT_THREADS = SIMT_WARPS * 32;
// One CTA for (token, query head), four warps that take 32 keys in turn: a lane multiplies a whole key (its row is contiguous),
// then takes features, whose 16 values of a block are contiguous. All of it float32.
template <typename T>
__global__ void __launch_bounds__(SIMT_THREADS)
attention_e4m3_simt_kernel(const T* __restrict__ q, T* __restrict__ out, const CacheArgs c, const int* __restrict__ positions,
                           const int* __restrict__ request_of, int nq, int nkv, int d, float scale_log2, int window, unsigned* status) {
  constexpr int STEP = 2 * E4M3_BLOCK, MAX_D = 256;
  __shared__ __align__(16) float q_s[MAX_D];
  __shared__ __align__(16) float p_s[SIMT_WARPS][STEP];
  __shared__ float rec[SIMT_WARPS][MAX_D + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x, head = blockIdx.y, g = head / (nq / nkv);
  pdl_wait();
  pdl_launch_dependents();
  const int64_t at = ((int64_t)t * nq + head) * d;
  for (int i = threadIdx.x; i < d; i += SIMT_THREADS) q_s[i] = to_f32(q[at + i]);
  __syncthreads();
  const int pos = positions[t], req = request_of[t], kstart = first_visible_key(pos, window);
  const int blocks_a_page = c.page_size / E4M3_BLOCK;
  float m = -INFINITY, l = 0.f, o[MAX_D / 32];
#pragma unroll
  for (int i = 0; i < MAX_D / 32; ++i) o[i] = 0.f;
  for (int key0 = kstart / STEP * STEP + warp * STEP; key0 <= pos; key0 += SIMT_WARPS * STEP) {
    // lane < 16: the first block of the two, else the second
    int64_t block = -1;
    {
      const int b0 = key0 + (lane >> 4) * E4M3_BLOCK;
      if (b0 <= pos && b0 + E4M3_BLOCK > kstart) {
        const int index = b0 / c.page_size;
        const int page = index < c.max_pages ? c.block_table[(int64_t)req * c.max_pages + index] : -1;
        if (page >= 0 && page < c.num_pages) block = ((int64_t)page * nkv + g) * blocks_a_page + (b0 - index * c.page_size) / E4M3_BLOCK;
        else raise_fault(status, VOSTI_FAULT_PAGE_RANGE);
      }
    }
    const int key = key0 + lane;
    float score = -INFINITY;
    if (block >= 0 && key >= kstart && key <= pos) {
      const uint8_t* const row = c.k + (block * E4M3_BLOCK + (lane & 15)) * d;
      float sum = 0.f;
      for (int i = 0; i < d; i += 16) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + i);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float4 u = *reinterpret_cast<const float4*>(q_s + i + 4 * x);
          const float2 lo = e4m3_unpack((uint16_t)word_of(w, x)), hi = e4m3_unpack((uint16_t)(word_of(w, x) >> 16));
          sum = fmaf(u.x, lo.x, sum);
          sum = fmaf(u.y, lo.y, sum);
          sum = fmaf(u.z, hi.x, sum);
          sum = fmaf(u.w, hi.y, sum);
        }
      }
      score = sum * e4m3_scale(c.k_scale[block]) * scale_log2;
    }
    const float m_new = fmaxf(m, warp_max(score)), safe = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - safe), p = exp2f(score - safe);
    m = m_new;
    l = l * alpha + warp_sum(p);
    p_s[warp][lane] = p;
    __syncwarp();
    float part[MAX_D / 32];
#pragma unroll
    for (int i = 0; i < MAX_D / 32; ++i) part[i] = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int64_t b = __shfl_sync(0xffffffffu, block, half * 16);
      if (b < 0) continue;
      const float factor = e4m3_scale(c.v_scale[b]);
      const int b0 = key0 + half * E4M3_BLOCK;
#pragma unroll
      for (int i = 0; i < MAX_D / 32; ++i) {
        const int feature = lane + 32 * i;
        if (feature >= d) continue;
        const uint4 w = *reinterpret_cast<const uint4*>(c.v + (b * d + feature) * E4M3_BLOCK);
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float4 u = *reinterpret_cast<const float4*>(p_s[warp] + half * E4M3_BLOCK + 4 * x);
          const float2 lo = e4m3_unpack((uint16_t)word_of(w, x)), hi = e4m3_unpack((uint16_t)(word_of(w, x) >> 16));
          // (what a token that is not visible holds must not meet its weight of zero)
          auto seen = [&](int b) { return b0 + 4 * x + b >= kstart && b0 + 4 * x + b <= pos; };
          if (seen(0)) sum = fmaf(u.x, lo.x, sum);
          if (seen(1)) sum = fmaf(u.y, lo.y, sum);
          if (seen(2)) sum = fmaf(u.z, hi.x, sum);
          if (seen(3)) sum = fmaf(u.w, hi.y, sum);
        }
        part[i] += sum * factor;
      }
    }
#pragma unroll
    for (int i = 0; i < MAX_D / 32; ++i) o[i] = o[i] * alpha + part[i];
    __syncwarp();
  }
  if (lane == 0) {
    rec[warp][0] = m;
    rec[warp][1] = l;
  }
#pragma unroll
  for (int i = 0; i < MAX_D / 32; ++i)
    if (lane + 32 * i < d) rec[warp][2 + lane + 32 * i] = o[i];
  __syncthreads();
  for (int f = threadIdx.x; f < d; f += SIMT_THREADS) {
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < SIMT_WARPS; ++w) top = fmaxf(top, rec[w][0]);
    const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < SIMT_WARPS; ++w) {
      const float weight = exp2f(rec[w][0] - safe);
      sum += rec[w][1] * weight;
      v += rec[w][2 + f] * weight;
    }
    out[at + f] = from_f32<T>(sum == 0.f ? 0.f : v / sum);
  }
}

// Segments of a token's keys: as many as find an SM at once, each of a tile a warp at least, eight at most (what a cluster always may have); sixteen
// where they are few and long. us at 1, 4, 8 and 16 segments: 8 kv heads, one token at 2,048 keys 18.7, 7.8, 6.1 and 7.2, at 8,192 67, 20, 12.3 and
// 10.5; four at 8,192 72, 24, 18.8 and 25; eight at 8,192 with 4, 6 and 8 31, 28 and 37; sixteen at 2,048 with 1, 3 and 4 21.7, 17.6 and 23.8.
// A window is left out of it: what it leaves is read sooner by more CTAs than have a tile for every warp (one token, a window of 512 behind 16,384 keys: 16
// segments 6.3, the two of nine tiles 7.3; a window of 4,096 7.9 and, in eight, 9.0; eight tokens, 512: six segments 7.3, two 8.3).
int segments_of(int64_t items, int max_kv_len) {
  const int64_t room = 148 * RESIDENT / items, work = (max_kv_len + TILE - 1) / TILE / WARPS;
  if (items * MAX_SEGMENTS <= 2 * 148 && work >= 2 * MAX_SEGMENTS) return MAX_SEGMENTS;
  int64_t most = room < work ? room : work;
  most = most < 8 ? most : 8;
  return most < 1 ? 1 : (int)most;
}

// Whether clusters of `size` CTAs can run at all; asked once per device, kernel (by its head size) and size.
template <int D>
bool cluster_runs(int smem, int size) {
  auto kernel = attention_e4m3_kernel<D>;
  static std::unordered_map<uint64_t, bool> known;
  static std::mutex mutex;
  std::lock_guard<std::mutex> lock(mutex);
  int device = 0;
  (void)cudaGetDevice(&device);
  const uint64_t key = (uint64_t)device << 8 | (uint64_t)size;
  auto it = known.find(key);
  if (it != known.end()) return it->second;
  cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)size);
  config.blockDim = dim3((unsigned)THREADS);
  config.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = (unsigned)size;
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess) {
    (void)cudaGetLastError();
    clusters = 0;
  }
  known.emplace(key, clusters > 0);
  return clusters > 0;
}

struct Launch {
  const bf16* q;
  bf16* out;
  CacheArgs c;
  const int *token_list, *positions, *request_of;
  int64_t items;
  int nq, nkv, window, segments, ordered, beside, appended;
  float scale_log2;
  unsigned* status;
  cudaStream_t stream;
};

template <int D>
cudaError_t launch_e4m3(const Launch& a) {
  auto kernel = attention_e4m3_kernel<D>;
  constexpr int SMEM = WARPS * 4 * (2 * E4M3_BLOCK * D + 32);
  const cudaError_t raised = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
  if (raised != cudaSuccess) return raised;
  int segments = a.segments;
  while (segments > 1 && !cluster_runs<D>(SMEM, segments)) --segments;
  const dim3 grid((unsigned)(a.items * segments));
  if (segments == 1)
    return vosti_launch(kernel, grid, dim3(THREADS), SMEM, a.stream, a.q, a.out, a.c, a.token_list, a.positions, a.request_of, a.nq, a.nkv, a.scale_log2,
                        a.window, 1, a.ordered, a.beside, a.appended, a.status);
  return vosti_launch_clusters(kernel, grid, dim3(THREADS), (unsigned)segments, SMEM, a.stream, a.q, a.out, a.c, a.token_list, a.positions, a.request_of,
                               a.nq, a.nkv, a.scale_log2, a.window, segments, a.ordered, a.beside, a.appended, a.status);
}
int check_cache(const void* k, const void* v, const void* k_scale, const void* v_scale, const int* block_table, int max_pages, int page_size,
                int num_pages, int nq, int nkv, float scale, int window) {
  VOSTI_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "attention_e4m3: bad head counts nq=%d nkv=%d", nq, nkv);
  VOSTI_REQUIRE(page_size > 0 && page_size % E4M3_BLOCK == 0, "attention_e4m3: page_size %d must be a multiple of 16", page_size);
  VOSTI_REQUIRE(max_pages > 0 && num_pages > 0 && block_table != nullptr, "attention_e4m3: bad geometry");
  VOSTI_REQUIRE(k != nullptr && v != nullptr && k_scale != nullptr && v_scale != nullptr && (((uintptr_t)k | (uintptr_t)v) & 15) == 0,
                "attention_e4m3: the cache is missing or does not start on 16 bytes");
  VOSTI_REQUIRE(scale > 0.f && window >= 0, "attention_e4m3: the score scale must be positive and the window not negative");
  return VOSTI_OK;
}

}  // namespace

// q, out: bfloat16 [tokens, nq * d]; the cache as in e4m3.cuh. `token_list` (or null: 0 .. count - 1) names the tokens; d is 64 or 128. `beside`: the
// launch right before this one on the stream is vosti_attention_prefill_tc_e4m3 for other rows of the same q, out and cache. `appended`
// > 0: the launch before (before the one it is beside) is the step's store of keys and values, which wrote at most that many of each request's newest tokens;
// 0: nothing is known of it.
VOSTI_API int vosti_attention_e4m3(const void* q, const void* k, const void* v, const void* k_scale, const void* v_scale, void* out,
                                   const int* token_list, int count, const int* positions, const int* request_of, const int* block_table,
                                   int max_pages, int page_size, int num_pages, int nq, int nkv, int d, int max_kv_len, float scale, int window,
                                   int beside, int appended, unsigned* status, cudaStream_t stream) {
  if (int bad = check_cache(k, v, k_scale, v_scale, block_table, max_pages, page_size, num_pages, nq, nkv, scale, window)) return bad;
  VOSTI_REQUIRE(d == 64 || d == 128, "attention_e4m3: head_dim %d must be 64 or 128", d);
  VOSTI_REQUIRE((((uintptr_t)q | (uintptr_t)out) & 15) == 0, "attention_e4m3: queries must start on 16 bytes");
  VOSTI_REQUIRE(appended >= 0, "attention_e4m3: bad count of appended tokens");
  VOSTI_REQUIRE(count >= 0 && (int64_t)count * nq * MAX_SEGMENTS <= 0x7fffffff, "attention_e4m3: bad token count %d", count);
  if (count == 0) return VOSTI_OK;
  const CacheArgs c = {(const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)k_scale, (const uint8_t*)v_scale, block_table, max_pages, page_size, num_pages};
  const int64_t items = (int64_t)count * nkv * ((nq / nkv + HEADS - 1) / HEADS);
  // more CTAs than run at once: those of the tokens with most keys first
  const bool ordered = items > 148 * RESIDENT && count > 1 && count <= MAX_ORDERED;
  const Launch launch = {(const bf16*)q, (bf16*)out, c, token_list, positions, request_of, items, nq, nkv, window, segments_of(items, max_kv_len),
                         ordered ? count : 0, beside, appended, scale * LOG2E, status, stream};
  const cudaError_t e = d == 64 ? launch_e4m3<64>(launch) : launch_e4m3<128>(launch);
  if (e != cudaSuccess) {
    vosti_set_error("attention_e4m3: %s", cudaGetErrorString(e));
    return (int)e;
  }
  VOSTI_LAUNCH_CHECK();
}

// The same on the CUDA cores for every token of q (float32 or bfloat16), d a multiple of 16 up to 256.
VOSTI_API int vosti_attention_e4m3_simt(const void* q, const void* k, const void* v, const void* k_scale, const void* v_scale, void* out, int tokens,
                                        const int* positions, const int* request_of, const int* block_table, int max_pages, int page_size,
                                        int num_pages, int nq, int nkv, int d, float scale, int window, int is_f32, unsigned* status,
                                        cudaStream_t stream) {
  VOSTI_REQUIRE(tokens >= 0 && nq <= 65535, "attention_e4m3: bad sizes");
  VOSTI_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "attention_e4m3: head_dim %d must be a multiple of 16, at most 256", d);
  if (tokens == 0) return VOSTI_OK;                              // (arrays of nothing are null)
  if (int bad = check_cache(k, v, k_scale, v_scale, block_table, max_pages, page_size, num_pages, nq, nkv, scale, window)) return bad;
  const CacheArgs c = {(const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)k_scale, (const uint8_t*)v_scale, block_table, max_pages, page_size, num_pages};
  const dim3 grid(tokens, nq);
  const cudaError_t e = is_f32 ? vosti_launch(attention_e4m3_simt_kernel<float>, grid, dim3(SIMT_THREADS), 0, stream, (const float*)q, (float*)out, c, positions,
                                              request_of, nq, nkv, d, scale * LOG2E, window, status)
                               : vosti_launch(attention_e4m3_simt_kernel<bf16>, grid, dim3(SIMT_THREADS), 0, stream, (const bf16*)q, (bf16*)out, c, positions,
                                              request_of, nq, nkv, d, scale * LOG2E, window, status);
  if (e != cudaSuccess) {
    vosti_set_error("attention_e4m3: %s", cudaGetErrorString(e));
    return (int)e;
  }
  VOSTI_LAUNCH_CHECK();
}
