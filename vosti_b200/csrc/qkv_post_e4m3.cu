// After the fused QKV projection, for a cache of 8 bits (e4m3.cuh), in one pass over each token's heads:
//   q heads: per-head RMSNorm (optional) -> rotation (optional) -> q_out
//   k heads: the same -> rounded to e4m3 under their block's scale -> key cache
//   v heads: rounded to e4m3 under their block's scale -> value cache, feature-major inside the block
// Norm and rotation are qkv_post.cu's (kernels/triton_kernels/qk_norm.py:40-95, rope.py:78-101); everything is float32 up to
// the one rounding at the store.
//
// A scale belongs to a block, so the unit of work for keys and values is a run: the step's tokens of one block and kv head, which stand
// next to one another in the batch and in the block. One CTA takes a run: it holds the run's keys and values in
// registers, finds their largest size, takes the larger of what they need and (a block that holds earlier tokens) the
// scale that is there, rounds the earlier tokens again where the scale grew, and stores. Nothing of another CTA's is read.
// A value that is not finite, or not below 2^96, makes its block's scale 255: the block is no number from then on.
#include "common.cuh"
#include "e4m3.cuh"

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int PER_WARP = E4M3_BLOCK / WARPS;   // tokens of a run, or q heads, that a warp holds
constexpr int V_PITCH = 20;                    // bytes between a feature's rows of values in shared memory (banks apart)
constexpr int FEW = 64;                        // up to so many tokens: one a CTA
constexpr int Q_TOKENS = 2;                    // of a CTA of query heads, with more

struct PostArgs {
  const void* qkv;               // [tokens, (nq + 2 nkv) d], or null with
  const float* partial;          // [splits, tokens, (nq + 2 nkv) d]
  int splits;
  int64_t plane;
  void* q_out;                   // [tokens, nq d]
  uint8_t *k, *v, *k_scale, *v_scale;
  const void *q_norm_w, *k_norm_w;
  int norm_w_is_f32;
  float eps;
  const float *cos_table, *sin_table;
  int max_positions;
  const int *positions, *slot_mapping;
  int64_t num_slots;
  int page_size, tokens, nq, nkv, d, rotary_dim, interleaved, tile;
  unsigned* status;
};

// A lane holds PAIRS pairs of a head's elements; those of a rotation turn with one another. FAST (the whole head turns in pairs
// (i, i + d/2), or nothing turns; d a multiple of 64, of 128 above one pair): neighbouring pairs in neighbouring words.
template <int PAIRS, bool FAST>
__device__ __forceinline__ int pair_index(int lane, int j) {
  return FAST && PAIRS > 1 ? 2 * lane + (j & 1) + 64 * (j >> 1) : lane + 32 * j;
}
// Elements of pair p: the first `rotary_dim` turn, the rest pair up with their neighbours.
template <bool FAST>
__device__ __forceinline__ void pair_elements(int p, const PostArgs& a, int& ia, int& ib) {
  if (FAST) {
    ia = p;
    ib = p + (a.d >> 1);
    return;
  }
  const int turning = a.rotary_dim >> 1;
  if (p < turning) {
    ia = a.interleaved ? 2 * p : p;
    ib = a.interleaved ? 2 * p + 1 : p + turning;
  } else {
    ia = 2 * p;
    ib = 2 * p + 1;
  }
}

template <typename T, int PAIRS, bool FAST>
__device__ __forceinline__ void load_head(const PostArgs& a, int64_t at, int lane, float (&x)[PAIRS], float (&y)[PAIRS]) {
  const int half = a.d >> 1;
  if constexpr (FAST && PAIRS > 1) {
#pragma unroll
    for (int j = 0; j < PAIRS; j += 2) {
      const int64_t i = at + 2 * lane + 32 * j;
      if (a.partial != nullptr) {
        float2 u = make_float2(0.f, 0.f), v = u;
#pragma unroll 4
        for (int s = 0; s < a.splits; ++s) {
          const float2 p = *reinterpret_cast<const float2*>(a.partial + s * a.plane + i);
          const float2 r = *reinterpret_cast<const float2*>(a.partial + s * a.plane + i + half);
          u.x += p.x, u.y += p.y, v.x += r.x, v.y += r.y;
        }
        x[j] = u.x, x[j + 1] = u.y, y[j] = v.x, y[j + 1] = v.y;
      } else if (sizeof(T) == 4) {
        const float2 u = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(a.qkv) + i);
        const float2 v = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(a.qkv) + i + half);
        x[j] = u.x, x[j + 1] = u.y, y[j] = v.x, y[j + 1] = v.y;
      } else {
        const float2 u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(reinterpret_cast<const bf16*>(a.qkv) + i));
        const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(reinterpret_cast<const bf16*>(a.qkv) + i + half));
        x[j] = u.x, x[j + 1] = u.y, y[j] = v.x, y[j + 1] = v.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      const int p = pair_index<PAIRS, FAST>(lane, j);
      x[j] = y[j] = 0.f;
      if (p >= half) continue;
      int ia, ib;
      pair_elements<FAST>(p, a, ia, ib);
      if (a.partial != nullptr) {
#pragma unroll 4
        for (int s = 0; s < a.splits; ++s) {
          x[j] += a.partial[s * a.plane + at + ia];
          y[j] += a.partial[s * a.plane + at + ib];
        }
      } else {
        x[j] = to_f32(reinterpret_cast<const T*>(a.qkv)[at + ia]);
        y[j] = to_f32(reinterpret_cast<const T*>(a.qkv)[at + ib]);
      }
    }
  }
}

// Norm weights of this lane's elements (ones without a norm).
template <int PAIRS, bool FAST>
__device__ __forceinline__ void load_norm(const PostArgs& a, const void* w, int lane, float (&wx)[PAIRS], float (&wy)[PAIRS]) {
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) {
    const int p = pair_index<PAIRS, FAST>(lane, j);
    wx[j] = wy[j] = 1.f;
    if (w == nullptr || p >= (a.d >> 1)) continue;
    int ia, ib;
    pair_elements<FAST>(p, a, ia, ib);
    wx[j] = load_flex(w, a.norm_w_is_f32, ia);
    wy[j] = load_flex(w, a.norm_w_is_f32, ib);
  }
}

// Cosines and sines of this lane's pairs at a position (no turn: 1 and 0).
template <int PAIRS, bool FAST>
__device__ __forceinline__ void load_turn(const PostArgs& a, int pos, int lane, float (&c)[PAIRS], float (&s)[PAIRS]) {
  const int turning = a.cos_table != nullptr ? a.rotary_dim >> 1 : 0;
  const int64_t at = (int64_t)pos * turning;
  if (FAST && PAIRS > 1 && turning > 0) {
#pragma unroll
    for (int j = 0; j < PAIRS; j += 2) {
      const float2 u = *reinterpret_cast<const float2*>(a.cos_table + at + 2 * lane + 32 * j);
      const float2 v = *reinterpret_cast<const float2*>(a.sin_table + at + 2 * lane + 32 * j);
      c[j] = u.x, c[j + 1] = u.y, s[j] = v.x, s[j + 1] = v.y;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) {
    const int p = pair_index<PAIRS, FAST>(lane, j);
    c[j] = 1.f;
    s[j] = 0.f;
    if (p < turning) {
      c[j] = a.cos_table[at + p];
      s[j] = a.sin_table[at + p];
    }
  }
}

template <int PAIRS>
__device__ __forceinline__ void norm_and_turn(const PostArgs& a, bool normed, float (&x)[PAIRS], float (&y)[PAIRS], const float (&wx)[PAIRS],
                                              const float (&wy)[PAIRS], const float (&c)[PAIRS], const float (&s)[PAIRS]) {
  float r = 1.f;
  if (normed) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) ss += x[j] * x[j] + y[j] * y[j];
    r = rsqrtf(warp_sum(ss) / (float)a.d + a.eps);
  }
#pragma unroll
  for (int j = 0; j < PAIRS; ++j) {
    const float u = x[j] * r * wx[j], v = y[j] * r * wy[j];
    x[j] = u * c[j] - v * s[j];
    y[j] = v * c[j] + u * s[j];
  }
}

template <typename T, int PAIRS, bool FAST>
__device__ __forceinline__ void store_head(const PostArgs& a, T* dst, int lane, const float (&x)[PAIRS], const float (&y)[PAIRS]) {
  const int half = a.d >> 1;
  if constexpr (FAST && PAIRS > 1) {
#pragma unroll
    for (int j = 0; j < PAIRS; j += 2) {
      const int p = pair_index<PAIRS, FAST>(lane, j);
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float2*>(dst + p) = make_float2(x[j], x[j + 1]);
        *reinterpret_cast<float2*>(dst + p + half) = make_float2(y[j], y[j + 1]);
      } else {
        *reinterpret_cast<__nv_bfloat162*>(dst + p) = __floats2bfloat162_rn(x[j], x[j + 1]);
        *reinterpret_cast<__nv_bfloat162*>(dst + p + half) = __floats2bfloat162_rn(y[j], y[j + 1]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      const int p = pair_index<PAIRS, FAST>(lane, j);
      if (p >= half) continue;
      int ia, ib;
      pair_elements<FAST>(p, a, ia, ib);
      dst[ia] = from_f32<T>(x[j]);
      dst[ib] = from_f32<T>(y[j]);
    }
  }
}

__device__ __forceinline__ int position_of(const PostArgs& a, int t) {
  if (a.cos_table == nullptr) return 0;
  const int pos = a.positions[t];
  if (pos >= 0 && pos < a.max_positions) return pos;
  if ((threadIdx.x & 31) == 0) raise_fault(a.status, VOSTI_FAULT_POSITION_RANGE);
  return 0;
}

// Blocks: `tile` neighbouring tokens' keys and values of a kv head, then 16 query heads of one or two tokens (what is in flight is what
// counts for a prompt: a warp has four heads of two tokens, or keys and values of four, on their way, 32 warps an SM).
template <typename T, int PAIRS, bool FAST>
__global__ void __launch_bounds__(THREADS, PAIRS >= 4 ? 4 : 8) qkv_post_e4m3_kernel(const PostArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int heads = a.nq + 2 * a.nkv, half = a.d >> 1;
  const int kv_blocks = (a.tokens + a.tile - 1) / a.tile * a.nkv;

  if ((int)blockIdx.x >= kv_blocks) {
    // ------------------------------------------------------------ queries: a warp takes four heads
    const int groups = (a.nq + E4M3_BLOCK - 1) / E4M3_BLOCK, block = (int)blockIdx.x - kv_blocks;
    const int h0 = block % groups * E4M3_BLOCK + warp * PER_WARP;
    const int step = a.tokens <= FEW ? 1 : Q_TOKENS, t0 = block / groups * step, count = min(step, a.tokens - t0);
    float wx[PAIRS], wy[PAIRS];
    load_norm<PAIRS, FAST>(a, a.q_norm_w, lane, wx, wy);
    pdl_wait();
    pdl_launch_dependents();
    if (h0 >= a.nq) return;
    float x[Q_TOKENS][PER_WARP][PAIRS], y[Q_TOKENS][PER_WARP][PAIRS];
#pragma unroll
    for (int n = 0; n < Q_TOKENS; ++n)
#pragma unroll
      for (int i = 0; i < PER_WARP; ++i)
        if (n < count && h0 + i < a.nq) load_head<T, PAIRS, FAST>(a, ((int64_t)(t0 + n) * heads + h0 + i) * a.d, lane, x[n][i], y[n][i]);
#pragma unroll
    for (int n = 0; n < Q_TOKENS; ++n) {
      if (n >= count) break;
      float c[PAIRS], s[PAIRS];
      load_turn<PAIRS, FAST>(a, position_of(a, t0 + n), lane, c, s);
      T* out = reinterpret_cast<T*>(a.q_out) + ((int64_t)(t0 + n) * a.nq + h0) * a.d;
#pragma unroll
      for (int i = 0; i < PER_WARP; ++i) {
        if (h0 + i >= a.nq) break;
        norm_and_turn<PAIRS>(a, a.q_norm_w != nullptr, x[n][i], y[n][i], wx, wy, c, s);
        store_head<T, PAIRS, FAST>(a, out + (int64_t)i * a.d, lane, x[n][i], y[n][i]);
      }
    }
    return;
  }

  // -------------------------------------------------------------- keys and values of one kv head, run by run
  extern __shared__ __align__(16) uint8_t v_rows[];             // [d][V_PITCH]: the run's values, feature-major, at their places in the block
  __shared__ float most[2][WARPS];
  __shared__ int broken[2][WARPS];
  const int g = (int)blockIdx.x % a.nkv, t_begin = (int)blockIdx.x / a.nkv * a.tile, t_end = min(a.tokens, t_begin + a.tile);
  float wx[PAIRS], wy[PAIRS];
  load_norm<PAIRS, FAST>(a, a.k_norm_w, lane, wx, wy);
  // slots were written before the step began
  const int my_t = t_begin + lane;
  auto slot_at = [&](int t) { return t >= 0 && t < a.tokens ? a.slot_mapping[t] : -1; };
  // which of the tile's tokens begin a run (lane i: token t_begin + i)
  bool begins = false;
  if (my_t < t_end) {
    const int slot = slot_at(my_t), before = slot_at(my_t - 1);
    if (slot < -1 || slot >= a.num_slots) {
      if (warp == 0 && g == 0) raise_fault(a.status, VOSTI_FAULT_SLOT_RANGE);
    } else if (slot >= 0) {
      const bool same = before >= 0 && before / E4M3_BLOCK == slot / E4M3_BLOCK;
      begins = !same;
      // a block's tokens of a step stand next to one another in its order; others are left out
      if (same && before != slot - 1 && warp == 0 && g == 0) raise_fault(a.status, VOSTI_FAULT_SLOT_RANGE);
    }
  }
  unsigned runs = __ballot_sync(0xffffffffu, begins);
  pdl_wait();
  pdl_launch_dependents();

  for (; runs != 0; runs &= runs - 1) {                          // (the same in all warps)
    const int t0 = t_begin + __ffs(runs) - 1;
    const int slot = slot_at(t0), offset = slot % E4M3_BLOCK;
    // the run's tokens: the neighbours that continue it
    const int next = slot_at(t0 + lane);
    const unsigned gone = ~__ballot_sync(0xffffffffu, offset + lane < E4M3_BLOCK && next == slot + lane);
    const int n = __ffs(gone) - 1;                               // (lane 16 never continues it)
    const int64_t page = slot / a.page_size, in_page = slot % a.page_size;
    const int64_t block = (page * a.nkv + g) * (a.page_size / E4M3_BLOCK) + in_page / E4M3_BLOCK;

    float kx[PER_WARP][PAIRS], ky[PER_WARP][PAIRS], vx[PER_WARP][PAIRS], vy[PER_WARP][PAIRS];
    float k_most = 0.f, v_most = 0.f;
    bool k_fine = true, v_fine = true;
#pragma unroll
    for (int i = 0; i < PER_WARP; ++i) {
      const int r = warp + i * WARPS;
      if (r >= n) break;
      const int64_t at = ((int64_t)(t0 + r) * heads + a.nq + g) * a.d;
      load_head<T, PAIRS, FAST>(a, at, lane, kx[i], ky[i]);
      load_head<T, PAIRS, FAST>(a, at + (int64_t)a.nkv * a.d, lane, vx[i], vy[i]);
    }
    const int k_old = offset > 0 ? a.k_scale[block] : 0, v_old = offset > 0 ? a.v_scale[block] : 0;
#pragma unroll
    for (int i = 0; i < PER_WARP; ++i) {
      const int r = warp + i * WARPS;
      if (r >= n) break;
      float c[PAIRS], s[PAIRS];
      load_turn<PAIRS, FAST>(a, position_of(a, t0 + r), lane, c, s);
      norm_and_turn<PAIRS>(a, a.k_norm_w != nullptr, kx[i], ky[i], wx, wy, c, s);
      auto look = [](float v, float& top, bool& fine) {
        const float size = fabsf(v);
        const bool ok = size < E4M3_LIMIT;
        fine = fine && ok;
        if (ok) top = fmaxf(top, size);
      };
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        look(kx[i][j], k_most, k_fine);
        look(ky[i][j], k_most, k_fine);
        look(vx[i][j], v_most, v_fine);
        look(vy[i][j], v_most, v_fine);
      }
    }
    k_most = warp_max(k_most);
    v_most = warp_max(v_most);
    const bool k_bad = __any_sync(0xffffffffu, !k_fine), v_bad = __any_sync(0xffffffffu, !v_fine);
    if (lane == 0) {
      most[0][warp] = k_most;
      most[1][warp] = v_most;
      broken[0][warp] = k_bad;
      broken[1][warp] = v_bad;
    }
    __syncthreads();
    int k_new, v_new;
    {
      float top[2] = {0.f, 0.f};
      int bad[2] = {0, 0};
#pragma unroll
      for (int w = 0; w < WARPS; ++w)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[i] = fmaxf(top[i], most[i][w]);
          bad[i] |= broken[i][w];
        }
      k_new = bad[0] ? E4M3_NAN_SCALE : max(e4m3_scale_for(top[0]), k_old);
      v_new = bad[1] ? E4M3_NAN_SCALE : max(e4m3_scale_for(top[1]), v_old);
    }
    // 2^-(scale - 127): the bits 254 - scale as an exponent (a scale that is no number: any payload will do)
    const float k_times = __uint_as_float((uint32_t)max(254 - k_new, 1) << 23), v_times = __uint_as_float((uint32_t)max(254 - v_new, 1) << 23);
    uint8_t* const k_rows = a.k + block * E4M3_BLOCK * a.d;
    uint8_t* const v_block = a.v + block * E4M3_BLOCK * a.d;
    // earlier keys under a larger scale: whole words, 2 tokens or more apart from the run's own rows
    if (offset > 0 && k_new > k_old && k_new != E4M3_NAN_SCALE) {
      const float f = e4m3_scale(max(127 + k_old - k_new, 0));   // (beyond 2^-127: everything is zero anyway)
      for (int i = threadIdx.x; i < offset * a.d / 4; i += THREADS) {
        uint32_t* const word = reinterpret_cast<uint32_t*>(k_rows) + i;
        const uint32_t w = *word;
        const float2 lo = e4m3_unpack((uint16_t)w), hi = e4m3_unpack((uint16_t)(w >> 16));
        *word = (uint32_t)e4m3_pack(lo.x * f, lo.y * f) | (uint32_t)e4m3_pack(hi.x * f, hi.y * f) << 16;
      }
    }
#pragma unroll
    for (int i = 0; i < PER_WARP; ++i) {
      const int r = warp + i * WARPS;
      if (r >= n) break;
      uint8_t* const key = k_rows + (offset + r) * a.d;
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) {
        const int p = pair_index<PAIRS, FAST>(lane, j);
        if (p >= half) continue;
        int ia, ib;
        pair_elements<FAST>(p, a, ia, ib);
        const uint16_t vv = e4m3_pack(vx[i][j] * v_times, vy[i][j] * v_times);
        v_rows[ia * V_PITCH + offset + r] = (uint8_t)vv;
        v_rows[ib * V_PITCH + offset + r] = (uint8_t)(vv >> 8);
        if (FAST && PAIRS > 1) {
          if (j & 1) continue;
          *reinterpret_cast<uint16_t*>(key + p) = e4m3_pack(kx[i][j] * k_times, kx[i][(j + 1) % PAIRS] * k_times);
          *reinterpret_cast<uint16_t*>(key + p + half) = e4m3_pack(ky[i][j] * k_times, ky[i][(j + 1) % PAIRS] * k_times);
          continue;
        }
        const uint16_t kk = e4m3_pack(kx[i][j] * k_times, ky[i][j] * k_times);
        key[ia] = (uint8_t)kk;
        key[ib] = (uint8_t)(kk >> 8);
      }
    }
    __syncthreads();
    // values: a thread takes a feature's 16 tokens, a word of four at a time
    const bool regrow = offset > 0 && v_new > v_old && v_new != E4M3_NAN_SCALE;
    const float f = regrow ? e4m3_scale(max(127 + v_old - v_new, 0)) : 1.f;
    for (int i = threadIdx.x; i < a.d * 4; i += THREADS) {
      const int feature = i >> 2, w0 = (i & 3) * 4;              // tokens w0 .. w0 + 3 of the block
      if (w0 >= offset + n || (w0 + 4 <= offset && !regrow)) continue;
      uint32_t* const word = reinterpret_cast<uint32_t*>(v_block + feature * E4M3_BLOCK) + (i & 3);
      const uint32_t old_bytes = e4m3_first_bytes(offset - w0), new_bytes = e4m3_first_bytes(offset + n - w0) & ~old_bytes;
      uint32_t w = *reinterpret_cast<const uint32_t*>(v_rows + feature * V_PITCH + w0) & new_bytes;
      if (new_bytes != 0xffffffffu) {
        uint32_t there = *word;
        if (regrow) {
          const float2 lo = e4m3_unpack((uint16_t)there), hi = e4m3_unpack((uint16_t)(there >> 16));
          const uint32_t again = (uint32_t)e4m3_pack(lo.x * f, lo.y * f) | (uint32_t)e4m3_pack(hi.x * f, hi.y * f) << 16;
          there = (there & ~old_bytes) | (again & old_bytes);
        }
        w |= there & ~new_bytes;
      }
      *word = w;
    }
    if (threadIdx.x == 0) {
      a.k_scale[block] = (uint8_t)k_new;
      a.v_scale[block] = (uint8_t)v_new;
    }
    __syncthreads();                                             // the next run takes the shared memory
  }
}

template <typename T, int PAIRS, bool FAST>
cudaError_t launch_post(const PostArgs& a, cudaStream_t stream) {
  const int64_t q_steps = a.tokens <= FEW ? a.tokens : (a.tokens + Q_TOKENS - 1) / Q_TOKENS;
  const dim3 grid((unsigned)((int64_t)((a.tokens + a.tile - 1) / a.tile) * a.nkv + q_steps * ((a.nq + E4M3_BLOCK - 1) / E4M3_BLOCK)));
  return vosti_launch(qkv_post_e4m3_kernel<T, PAIRS, FAST>, grid, dim3(THREADS), (size_t)a.d * V_PITCH, stream, a);
}
template <typename T>
cudaError_t launch_post_as(const PostArgs& a, cudaStream_t stream) {
  // whole words: two elements of every operand
  const uintptr_t words = (uintptr_t)a.partial | (uintptr_t)a.cos_table | (uintptr_t)a.sin_table, rows = (uintptr_t)a.qkv | (uintptr_t)a.q_out;
  const bool whole = (a.cos_table == nullptr || (a.rotary_dim == a.d && !a.interleaved)) && (a.d == 64 || a.d == 128 || a.d == 256) &&
                     words % 8 == 0 && rows % (2 * sizeof(T)) == 0;
  if (whole) return a.d == 64 ? launch_post<T, 1, true>(a, stream) : a.d == 128 ? launch_post<T, 2, true>(a, stream) : launch_post<T, 4, true>(a, stream);
  return a.d <= 64 ? launch_post<T, 1, false>(a, stream) : a.d <= 128 ? launch_post<T, 2, false>(a, stream) : launch_post<T, 4, false>(a, stream);
}

}  // namespace

// qkv: [tokens, (nq + 2 nkv) d], or null with `partial`: float32 [splits, tokens, (nq + 2 nkv) d], summed here in split order. q_out:
// [tokens, nq d]. k, v, k_scale, v_scale: the cache (e4m3.cuh), num_slots = pages * page_size; token t goes to slot
// slot_mapping[t] (-1: nowhere). The tokens of a step that share a block stand next to one another, in the block's order, and hold
// all its tokens from the first of them on; no block is another request's too. q_norm_w / k_norm_w null: no head norm. cos / sin null: no
// rotation; else float32 [max_positions, rotary_dim / 2], pairs as in vosti_qkv_post.
VOSTI_API int vosti_qkv_post_e4m3(const void* qkv, const float* partial, int splits, void* q_out, void* k, void* v, void* k_scale, void* v_scale,
                                  const void* q_norm_w, const void* k_norm_w, int norm_w_is_f32, float eps, const float* cos_table,
                                  const float* sin_table, int max_positions, const int* positions, const int* slot_mapping, int64_t num_slots,
                                  int page_size, int tokens, int nq, int nkv, int d, int rotary_dim, int interleaved, int is_f32,
                                  unsigned* status, cudaStream_t stream) {
  VOSTI_REQUIRE(tokens >= 0 && nq > 0 && nkv > 0, "qkv_post_e4m3: bad sizes");
  VOSTI_REQUIRE(d >= 16 && d <= 256 && d % 16 == 0, "qkv_post_e4m3: head_dim %d must be a multiple of 16, at most 256", d);
  VOSTI_REQUIRE(page_size > 0 && page_size % E4M3_BLOCK == 0, "qkv_post_e4m3: page_size %d must be a multiple of 16", page_size);
  VOSTI_REQUIRE((qkv != nullptr) != (partial != nullptr), "qkv_post_e4m3: give the projection or its partial sums");
  VOSTI_REQUIRE(partial == nullptr || splits >= 1, "qkv_post_e4m3: bad split count");
  VOSTI_REQUIRE(num_slots >= 0 && num_slots <= 0x7fffffff, "qkv_post_e4m3: a cache of %lld slots is too large", (long long)num_slots);
  VOSTI_REQUIRE((cos_table == nullptr) == (sin_table == nullptr), "qkv_post_e4m3: cos and sin go together");
  VOSTI_REQUIRE(cos_table == nullptr || positions != nullptr, "qkv_post_e4m3: rotation needs positions");
  VOSTI_REQUIRE(cos_table == nullptr || (rotary_dim > 0 && rotary_dim <= d && rotary_dim % 2 == 0),
                "qkv_post_e4m3: rotary_dim %d must be even and between 2 and head_dim %d", rotary_dim, d);
  VOSTI_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "qkv_post_e4m3: the cache must start on 16 bytes");
  VOSTI_REQUIRE(slot_mapping != nullptr && k != nullptr && v != nullptr && k_scale != nullptr && v_scale != nullptr, "qkv_post_e4m3: the cache is missing");
  if (tokens == 0) return VOSTI_OK;
  VOSTI_REQUIRE((int64_t)tokens * (nkv + (nq + E4M3_BLOCK - 1) / E4M3_BLOCK) <= 0x7fffffff, "qkv_post_e4m3: too many tokens and heads for one launch");
  // few tokens: a CTA for each, so that none waits for another's run; many (prompts): a CTA for 16, one or two runs
  const int tile = tokens <= FEW ? 1 : E4M3_BLOCK;
  const PostArgs a = {qkv, partial, splits, (int64_t)tokens * (nq + 2 * nkv) * d, q_out, (uint8_t*)k, (uint8_t*)v, (uint8_t*)k_scale,
                      (uint8_t*)v_scale, q_norm_w, k_norm_w, norm_w_is_f32, eps, cos_table, sin_table, max_positions, positions, slot_mapping,
                      num_slots, page_size, tokens, nq, nkv, d, cos_table != nullptr ? rotary_dim : d, interleaved, tile, status};
  const cudaError_t e = is_f32 ? launch_post_as<float>(a, stream) : launch_post_as<bf16>(a, stream);
  if (e != cudaSuccess) {
    vosti_set_error("qkv_post_e4m3: %s", cudaGetErrorString(e));
    return (int)e;
  }
  VOSTI_LAUNCH_CHECK();
}
