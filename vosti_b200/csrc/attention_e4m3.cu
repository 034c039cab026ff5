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
// features, all of them needed, and the 8 columns query heads. A warp takes 64 keys at a time, straight from memory into registers, no staging:
//   * the order of the summed index is free as long as both operands share it. A lane's 16 bytes of a key row are features
//     64 c + 16 j .. + 15 (j = lane % 4): four k-steps of four features. Rows of S^T are chosen so that the weights come out
//     where the second product wants them: row r of step s is token 4 s + r % 2 (+ 2 for rows 8 to 15) of block r % 8 / 2.
//   * a lane's 16 bytes of a value row are one feature's 16 tokens of block j: four k-steps of four tokens.
//   * the weights turn from (key, head) into (head, key) by movmatrix on pairs rounded to bfloat16.
// Payloads become bfloat16 by moving their bits and one multiplication by the block's scale, which is exact.
// What bounds it is the cache's bytes; the conversion is some five instructions for two values.
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int TILE = 64;                   // keys of a warp's step: four blocks
constexpr int HEADS = 8;                   // query heads of a CTA
constexpr int MAX_SEGMENTS = 16;

__device__ __forceinline__ uint4 load_line(const uint8_t* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

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
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float load_of_rank(const float* p, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

template <int D>
__global__ void __launch_bounds__(THREADS, 2)
attention_e4m3_kernel(const bf16* __restrict__ q, bf16* __restrict__ out, const CacheArgs c, const int* __restrict__ token_list,
                      const int* __restrict__ positions, const int* __restrict__ request_of, int nq, int nkv, float scale_log2, int window,
                      int segments, unsigned* status) {
  constexpr int CHUNKS = D / 64, FT = D / 16;
  constexpr int REC = D + 2;                                   // a head's record: largest score, sum, products
  __shared__ float part[WARPS][HEADS][REC];
  __shared__ float whole[HEADS][REC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int j = lane & 3, r8 = lane >> 2;
  const int group = nq / nkv, halves = (group + HEADS - 1) / HEADS;
  const int seg = segments > 1 ? (int)cluster_rank_of() : 0;
  int item = blockIdx.x / segments;
  const int part_of_group = item % halves;
  item /= halves;
  const int g = item % nkv, t = token_list ? token_list[item / nkv] : item / nkv;
  const int heads = min(HEADS, group - part_of_group * HEADS);
  const int64_t q_at = ((int64_t)t * nq + g * group + part_of_group * HEADS) * D;
  const int pos = positions[t], req = request_of[t];
  const int kstart = first_visible_key(pos, window);
  // this CTA's tiles: the visible ones in `segments` nearly equal runs; the warps take them in turn
  const int first = kstart / TILE, count = pos >= 0 ? pos / TILE - first + 1 : 0;
  const int begin = first + (int)((int64_t)count * seg / segments), end = first + (int)((int64_t)count * (seg + 1) / segments);
  const int blocks_a_page = c.page_size / E4M3_BLOCK;
  const int* const table = c.block_table + (int64_t)req * c.max_pages;

  // index of block `lane % 4` of a tile among the cache's blocks of this kv head, 0 where nothing of it is visible
  auto block_of = [&](int tile) {
    const int key0 = tile * TILE + j * E4M3_BLOCK;
    if (tile >= end || key0 > pos || key0 + E4M3_BLOCK <= kstart) return (int64_t)g * blocks_a_page;
    const int index = key0 / c.page_size;
    int page = index < c.max_pages ? table[index] : -1;
    if (page < 0 || page >= c.num_pages) {
      raise_fault(status, VOSTI_FAULT_PAGE_RANGE);
      page = 0;
    }
    return ((int64_t)page * nkv + g) * blocks_a_page + (key0 - index * c.page_size) / E4M3_BLOCK;
  };

  uint4 kk[4][2][CHUNKS];                                      // [step][rows 0-7, 8-15][chunk]
  int k_exp = 0, v_exp = 0;
  auto load_keys = [&](int64_t block) {
    const int64_t mine = __shfl_sync(0xffffffffu, block, lane >> 3);
    const uint8_t* const at = c.k + mine * (E4M3_BLOCK * D) + (r8 & 1) * D + 16 * j;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int ch = 0; ch < CHUNKS; ++ch) kk[s][h][ch] = load_line(at + (4 * s + 2 * h) * D + 64 * ch);
    k_exp = c.k_scale[mine];
  };

  int64_t block = begin + warp < end ? block_of(begin + warp) : 0;
  pdl_wait();
  pdl_launch_dependents();
  uint32_t qb[CHUNKS][4][2];                                   // Q^T: [chunk][k-step][features 4 w, + 2]
#pragma unroll
  for (int ch = 0; ch < CHUNKS; ++ch) {
    uint4 u = make_uint4(0, 0, 0, 0), v = u;
    if (r8 < heads) {
      const uint4* const at = reinterpret_cast<const uint4*>(q + q_at + (int64_t)r8 * D + 64 * ch + 16 * j);
      u = at[0];
      v = at[1];
    }
    qb[ch][0][0] = u.x, qb[ch][0][1] = u.y, qb[ch][1][0] = u.z, qb[ch][1][1] = u.w;
    qb[ch][2][0] = v.x, qb[ch][2][1] = v.y, qb[ch][3][0] = v.z, qb[ch][3][1] = v.w;
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};      // of heads 2 j and 2 j + 1
  float o[FT][4];
#pragma unroll
  for (int i = 0; i < FT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

  if (begin + warp < end) load_keys(block);
  for (int tile = begin + warp; tile < end; tile += WARPS) {
    // this tile's values, and where the next one lies
    uint4 vv[FT][2];                                           // [16 features][rows 0-7, 8-15]
    const uint8_t* const v_at = c.v + block * (E4M3_BLOCK * D) + r8 * E4M3_BLOCK;
#pragma unroll
    for (int i = 0; i < FT; ++i) {
      vv[i][0] = load_line(v_at + i * 16 * E4M3_BLOCK);
      vv[i][1] = load_line(v_at + i * 16 * E4M3_BLOCK + 8 * E4M3_BLOCK);
    }
    v_exp = c.v_scale[block];
    const int64_t next = block_of(tile + WARPS);

    // ---- S^T = K Q^T
    float s[4][4];
    {
      const E4m3Factor f = e4m3_factor(k_exp);
      const bool twice = __any_sync(0xffffffffu, f.second != E4M3_ONE);
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        s[st][0] = s[st][1] = s[st][2] = s[st][3] = 0.f;
#pragma unroll
        for (int ch = 0; ch < CHUNKS; ++ch)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t lo = word_of(kk[st][0][ch], w), hi = word_of(kk[st][1][ch], w);
            uint32_t a[4] = {e4m3_widen<0>(lo, f), e4m3_widen<0>(hi, f), e4m3_widen<1>(lo, f), e4m3_widen<1>(hi, f)};
            if (twice)
#pragma unroll
              for (int i = 0; i < 4; ++i) a[i] = bf16x2_times(a[i], f.second);
            mma_bf16(s[st], a, qb[ch][w][0], qb[ch][w][1]);
          }
      }
    }
    if (tile + WARPS < end) load_keys(next);

    // ---- online softmax of the lane's two heads over the warp's 64 keys
    const int key_lane = tile * TILE + (lane >> 3) * E4M3_BLOCK + (r8 & 1);        // + 4 st (+ 2)
    const bool edge = tile * TILE < kstart || tile * TILE + TILE - 1 > pos;
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[st][e] *= scale_log2;
        if (edge) {
          const int key = key_lane + 4 * st + (e >> 1) * 2;
          if (key < kstart || key > pos) s[st][e] = -INFINITY;
        }
        top[e & 1] = fmaxf(top[e & 1], s[st][e]);
      }
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int x = 4; x <= 16; x <<= 1) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], x));
      const float m_new = fmaxf(m[h], top[h]), safe = m_new == -INFINITY ? 0.f : m_new;
      alpha[h] = fast_exp2(m[h] - safe);
      m[h] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int st = 0; st < 4; ++st) {
        s[st][h] = fast_exp2(s[st][h] - safe);
        s[st][h + 2] = fast_exp2(s[st][h + 2] - safe);
        sum += s[st][h] + s[st][h + 2];
      }
      l[h] = l[h] * alpha[h] + sum;                            // the lane's share; added up at the end
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
    uint32_t p[4][2];                                          // P^T: [step][tokens 4 s, + 2]
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      p[st][0] = turn8x8(pack_bf16(s[st][0], s[st][1]));
      p[st][1] = turn8x8(pack_bf16(s[st][2], s[st][3]));
    }

    // ---- O^T += V^T P^T
    if (edge) {
      // bytes of tokens that are not visible become zeros: whatever they hold must not meet a weight of zero
      const int key0 = tile * TILE + j * E4M3_BLOCK;
      uint32_t keep[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        keep[w] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (key0 + 4 * w + b >= kstart && key0 + 4 * w + b <= pos) keep[w] |= 0xffu << (8 * b);
      }
      if ((keep[0] | keep[1] | keep[2] | keep[3]) == 0) v_exp = 0;
#pragma unroll
      for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          vv[i][h].x &= keep[0];
          vv[i][h].y &= keep[1];
          vv[i][h].z &= keep[2];
          vv[i][h].w &= keep[3];
        }
    }
    {
      const E4m3Factor f = e4m3_factor(v_exp);
      const bool twice = __any_sync(0xffffffffu, f.second != E4M3_ONE);
#pragma unroll
      for (int i = 0; i < FT; ++i)
#pragma unroll
        for (int st = 0; st < 4; ++st) {
          const uint32_t lo = word_of(vv[i][0], st), hi = word_of(vv[i][1], st);
          uint32_t a[4] = {e4m3_widen<0>(lo, f), e4m3_widen<0>(hi, f), e4m3_widen<1>(lo, f), e4m3_widen<1>(hi, f)};
          if (twice)
#pragma unroll
            for (int x = 0; x < 4; ++x) a[x] = bf16x2_times(a[x], f.second);
          mma_bf16(o[i], a, p[st][0], p[st][1]);
        }
    }
    block = next;
  }

  // ---- the four warps' records into one, in warp order
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int x = 4; x <= 16; x <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], x);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float* const rec = part[warp][2 * j + h];
    if (r8 == 0) {
      rec[0] = m[h];
      rec[1] = l[h];
    }
#pragma unroll
    for (int i = 0; i < FT; ++i) {
      rec[2 + 16 * i + r8] = o[i][h];
      rec[2 + 16 * i + 8 + r8] = o[i][h + 2];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += THREADS) {
    const int h = i / D, f = i % D;
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, part[w][h][0]);
    const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float weight = fast_exp2(part[w][h][0] - safe);
      sum += part[w][h][1] * weight;
      v += part[w][h][2 + f] * weight;
    }
    if (segments == 1) {
      out[q_at + i] = __float2bfloat16_rn(sum == 0.f ? 0.f : v / sum);
    } else {
      whole[h][2 + f] = v;
      if (f == 0) {
        whole[h][0] = top;
        whole[h][1] = sum;
      }
    }
  }
  if (segments == 1) return;
  // ---- the segments' records, in their order; each CTA of the cluster takes a share of the row
  cluster_sync();
  for (int i = seg * THREADS + threadIdx.x; i < heads * D; i += segments * THREADS) {
    const int h = i / D, f = i % D;
    float top = -INFINITY, sum = 0.f, v = 0.f;
    for (int s = 0; s < segments; ++s) top = fmaxf(top, load_of_rank(&whole[h][0], s));
    const float safe = top == -INFINITY ? 0.f : top;
    for (int s = 0; s < segments; ++s) {
      const float weight = fast_exp2(load_of_rank(&whole[h][0], s) - safe);
      sum += load_of_rank(&whole[h][1], s) * weight;
      v += load_of_rank(&whole[h][2 + f], s) * weight;
    }
    out[q_at + i] = __float2bfloat16_rn(sum == 0.f ? 0.f : v / sum);
  }
  cluster_sync();                                              // nobody reads this CTA's record after this
}

// ---------------------------------------------------------------------------------------------- CUDA cores
// One CTA for (token, query head), four warps that take 32 keys in turn: a lane multiplies a whole key (its row is contiguous),
// then takes features, whose 16 values of a block are contiguous. All of it float32.
template <typename T>
__global__ void __launch_bounds__(THREADS)
attention_e4m3_simt_kernel(const T* __restrict__ q, T* __restrict__ out, const CacheArgs c, const int* __restrict__ positions,
                           const int* __restrict__ request_of, int nq, int nkv, int d, float scale_log2, int window, unsigned* status) {
  constexpr int STEP = 2 * E4M3_BLOCK, MAX_D = 256;
  __shared__ __align__(16) float q_s[MAX_D];
  __shared__ __align__(16) float p_s[WARPS][STEP];
  __shared__ float rec[WARPS][MAX_D + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = blockIdx.x, head = blockIdx.y, g = head / (nq / nkv);
  pdl_wait();
  pdl_launch_dependents();
  const int64_t at = ((int64_t)t * nq + head) * d;
  for (int i = threadIdx.x; i < d; i += THREADS) q_s[i] = to_f32(q[at + i]);
  __syncthreads();
  const int pos = positions[t], req = request_of[t], kstart = first_visible_key(pos, window);
  const int blocks_a_page = c.page_size / E4M3_BLOCK;
  float m = -INFINITY, l = 0.f, o[MAX_D / 32];
#pragma unroll
  for (int i = 0; i < MAX_D / 32; ++i) o[i] = 0.f;
  for (int key0 = kstart / STEP * STEP + warp * STEP; key0 <= pos; key0 += WARPS * STEP) {
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
  for (int f = threadIdx.x; f < d; f += THREADS) {
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, rec[w][0]);
    const float safe = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float weight = exp2f(rec[w][0] - safe);
      sum += rec[w][1] * weight;
      v += rec[w][2 + f] * weight;
    }
    out[at + f] = from_f32<T>(sum == 0.f ? 0.f : v / sum);
  }
}

// Whether clusters of `size` CTAs can run at all; asked once per device, kernel and size.
template <typename Kernel>
bool cluster_runs(Kernel kernel, int size) {
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
  config.blockDim = dim3(THREADS);
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

template <int D>
cudaError_t launch_e4m3(const bf16* q, bf16* out, const CacheArgs& c, const int* token_list, int count, const int* positions, const int* request_of,
                        int nq, int nkv, float scale_log2, int window, int segments, unsigned* status, cudaStream_t stream) {
  auto kernel = attention_e4m3_kernel<D>;
  while (segments > 1 && !cluster_runs(kernel, segments)) segments /= 2;
  const int halves = (nq / nkv + HEADS - 1) / HEADS;
  const dim3 grid((unsigned)((int64_t)count * nkv * halves * segments));
  if (segments == 1)
    return vosti_launch(kernel, grid, dim3(THREADS), 0, stream, q, out, c, token_list, positions, request_of, nq, nkv, scale_log2, window, 1, status);
  return vosti_launch_clusters(kernel, grid, dim3(THREADS), (unsigned)segments, 0, stream, q, out, c, token_list, positions, request_of, nq, nkv,
                               scale_log2, window, segments, status);
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

// How many segments the visible keys of a token are cut into: `count` tokens, the longest of them with max_kv_len keys.
VOSTI_API int vosti_attention_e4m3_segments(int count, int nq, int nkv, int max_kv_len) {
  const int64_t items = (int64_t)count * nkv * ((nq / nkv + HEADS - 1) / HEADS);
  const int tiles = (max_kv_len + TILE - 1) / TILE;
  int segments = 1;
  while (segments < MAX_SEGMENTS && items * segments * 2 <= 296 && tiles >= segments * 2 * WARPS) segments *= 2;
  return segments;
}

// q, out: bfloat16 [tokens, nq * d]; the cache as in e4m3.cuh. `token_list` (or null: 0 .. count - 1) names the tokens; d is 64 or 128.
VOSTI_API int vosti_attention_e4m3(const void* q, const void* k, const void* v, const void* k_scale, const void* v_scale, void* out,
                                   const int* token_list, int count, const int* positions, const int* request_of, const int* block_table,
                                   int max_pages, int page_size, int num_pages, int nq, int nkv, int d, int max_kv_len, float scale, int window,
                                   unsigned* status, cudaStream_t stream) {
  if (int bad = check_cache(k, v, k_scale, v_scale, block_table, max_pages, page_size, num_pages, nq, nkv, scale, window)) return bad;
  VOSTI_REQUIRE(d == 64 || d == 128, "attention_e4m3: head_dim %d must be 64 or 128", d);
  VOSTI_REQUIRE((((uintptr_t)q | (uintptr_t)out) & 15) == 0, "attention_e4m3: queries must start on 16 bytes");
  VOSTI_REQUIRE(count >= 0 && (int64_t)count * nq * MAX_SEGMENTS <= 0x7fffffff, "attention_e4m3: bad token count %d", count);
  if (count == 0) return VOSTI_OK;
  const CacheArgs c = {(const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)k_scale, (const uint8_t*)v_scale, block_table, max_pages, page_size, num_pages};
  const int segments = vosti_attention_e4m3_segments(count, nq, nkv, max_kv_len);
  const cudaError_t e = d == 64 ? launch_e4m3<64>((const bf16*)q, (bf16*)out, c, token_list, count, positions, request_of, nq, nkv, scale * LOG2E, window,
                                                  segments, status, stream)
                                : launch_e4m3<128>((const bf16*)q, (bf16*)out, c, token_list, count, positions, request_of, nq, nkv, scale * LOG2E,
                                                   window, segments, status, stream);
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
  if (int bad = check_cache(k, v, k_scale, v_scale, block_table, max_pages, page_size, num_pages, nq, nkv, scale, window)) return bad;
  VOSTI_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "attention_e4m3: head_dim %d must be a multiple of 16, at most 256", d);
  VOSTI_REQUIRE(tokens >= 0 && nq <= 65535, "attention_e4m3: bad sizes");
  if (tokens == 0) return VOSTI_OK;
  const CacheArgs c = {(const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)k_scale, (const uint8_t*)v_scale, block_table, max_pages, page_size, num_pages};
  const dim3 grid(tokens, nq);
  const cudaError_t e = is_f32 ? vosti_launch(attention_e4m3_simt_kernel<float>, grid, dim3(THREADS), 0, stream, (const float*)q, (float*)out, c, positions,
                                              request_of, nq, nkv, d, scale * LOG2E, window, status)
                               : vosti_launch(attention_e4m3_simt_kernel<bf16>, grid, dim3(THREADS), 0, stream, (const bf16*)q, (bf16*)out, c, positions,
                                              request_of, nq, nkv, d, scale * LOG2E, window, status);
  if (e != cudaSuccess) {
    vosti_set_error("attention_e4m3: %s", cudaGetErrorString(e));
    return (int)e;
  }
  VOSTI_LAUNCH_CHECK();
}
