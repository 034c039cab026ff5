// After the fused QKV projection, for a cache of 8 bits (e4m3.cuh), in one pass over each token's heads:
//   q heads: per-head RMSNorm (optional) -> rotation (optional) -> q_out
//   k heads: the same -> rounded to e4m3 under their block's scale -> key cache
//   v heads: rounded to e4m3 under their block's scale -> value cache, feature-major inside the block
// Norm and rotation are qkv_post.cu's (kernels/triton_kernels/qk_norm.py:40-95, rope.py:78-101); everything is float32 up to
// the one rounding at the store.
//
// A scale belongs to a block, so the unit of work for keys, and for values, is a run: the step's tokens of one block and kv head, which stand
// next to one another in the batch and in the block. A CTA (runs of more than four tokens) or a warp (shorter ones) takes a run's keys, another its
// values: it holds them in registers, finds their largest size, takes the larger of what they need and (a block that holds earlier
// tokens) the scale that is there, rounds the earlier tokens again where the scale grew, and stores. Nothing of another run's is read.
// A value that is not finite, or not below 2^96, makes its block's scale 255: the block is no number from then on.
//
// A head of 64, 128 or 256 that turns as a whole in pairs (i, i + d/2), or not at all, is d / 8 lanes with four neighbouring elements of each half;
// any other is a warp with an element pair every 32. A prompt of 2,048 tokens of the 8B sizes takes 19 us, 38% of the rate its bytes could move
// at: blocks are short, and the latencies of their loads in a row are not hidden by the 24 warps an SM holds of their registers (20 warps with more
// registers, blocks that walked on over query heads, and a head on a whole warp were slower). Eight tokens take 3 us; a CTA that took a run's keys and
// values both needed 5.3. Between a model's other kernels, which leave neither the cache nor the turns in L2, they take 4.5 us behind the projection;
// without the turns' loads and the blocks' prefetch before its end 6.3, with a grown block's words read one after another 7.4.
#include "common.cuh"
#include "e4m3.cuh"

namespace {

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int SHORT = 4;                       // tokens of a run that one warp takes
constexpr int ROWS = 4;                        // words of 16 bytes of a block that a lane asks for at a time
constexpr int V_PITCH = 20;                    // bytes between a feature's rows of values in shared memory (banks apart)
constexpr int FEW = 32, MANY = 256;
constexpr int Q_MANY = 4;                      // query heads that a lane holds at a time with more than FEW tokens (up to that, one)

struct PostArgs {
  const void* qkv;               // [tokens, (nq + 2 nkv) d], or null with
  const float* partial;          // [splits, tokens, (nq + 2 nkv) d]
  int splits;
  int64_t plane;
  void* q_out;                   // [tokens, nq d]
  uint8_t *k, *v, *k_scale, *v_scale;
  const void *q_norm_w, *k_norm_w;
  int norm_w_is_f32;
  float eps, inverse_d;
  const float *cos_table, *sin_table;
  int max_positions;
  const int *positions, *slot_mapping;
  int64_t num_slots;
  int page_size, tokens, nq, nkv, d, rotary_dim, interleaved, tile;
  unsigned* status;
};

// How a head lies on lanes: `LANES` of them with `PAIRS` pairs each; those of a rotation turn with one another.
template <int LANES_, int PAIRS_, bool FAST_>
struct Lay {
  static constexpr int LANES = LANES_, PAIRS = PAIRS_, HEADS = 32 / LANES_;
  static constexpr bool FAST = FAST_;
  static __device__ __forceinline__ int pair(int sub, int j) { return FAST ? 4 * sub + j : sub + 32 * j; }
  // Elements of pair p: the first `rotary_dim` turn, the rest pair up with their neighbours.
  static __device__ __forceinline__ void elements(int p, const PostArgs& a, int& ia, int& ib) {
    if (FAST) {
      ia = p;
      ib = p + (a.d >> 1);
      return;
    }
    const int turning = a.rotary_dim >> 1;
    const bool turns = p < turning;
    ia = turns && !a.interleaved ? p : 2 * p;
    ib = turns && !a.interleaved ? p + turning : 2 * p + 1;
  }
};

template <typename T>
__device__ __forceinline__ void load_words(const T* p, float (&x)[4]) {
  const float4 v = load_four(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}

// N heads of the projection that begin at elements at[i], or the sums of their partial sums in split order; those without `live` are zeros. The loads
// of all of them, and of FLIGHT splits, are on their way together.
template <typename T, typename L, int N>
__device__ __forceinline__ void load_heads(const PostArgs& a, const int64_t (&at)[N], const bool (&live)[N], int sub, float (&x)[N][L::PAIRS],
                                           float (&y)[N][L::PAIRS]) {
  const int half = a.d >> 1;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < L::PAIRS; ++j) x[i][j] = y[i][j] = 0.f;
  if (a.partial == nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!live[i]) continue;
      const T* const from = reinterpret_cast<const T*>(a.qkv) + at[i];
      if constexpr (L::FAST) {
        load_words(from + 4 * sub, x[i]);
        load_words(from + 4 * sub + half, y[i]);
      } else {
#pragma unroll
        for (int j = 0; j < L::PAIRS; ++j) {
          const int p = L::pair(sub, j);
          if (p >= half) continue;
          int ia, ib;
          L::elements(p, a, ia, ib);
          x[i][j] = to_f32(from[ia]);
          y[i][j] = to_f32(from[ib]);
        }
      }
    }
    return;
  }
  constexpr int FLIGHT = !L::FAST || N > 2 ? 1 : N == 2 ? 4 : 8;
  for (int s0 = 0; s0 < a.splits; s0 += FLIGHT) {
    float u[FLIGHT][N][L::PAIRS], v[FLIGHT][N][L::PAIRS];
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool here = live[i] && s0 + f < a.splits;
        const float* const from = a.partial + (s0 + f) * a.plane + at[i];
        if constexpr (L::FAST) {
          if (here) {
            load_words(from + 4 * sub, u[f][i]);
            load_words(from + 4 * sub + half, v[f][i]);
          } else {
#pragma unroll
            for (int j = 0; j < L::PAIRS; ++j) u[f][i][j] = v[f][i][j] = 0.f;
          }
        } else {
#pragma unroll
          for (int j = 0; j < L::PAIRS; ++j) {
            const int p = L::pair(sub, j);
            int ia, ib;
            L::elements(p, a, ia, ib);
            u[f][i][j] = here && p < half ? from[ia] : 0.f;
            v[f][i][j] = here && p < half ? from[ib] : 0.f;
          }
        }
      }
#pragma unroll
    for (int f = 0; f < FLIGHT; ++f)
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < L::PAIRS; ++j) {
          x[i][j] += u[f][i][j];
          y[i][j] += v[f][i][j];
        }
  }
}

// Norm weights of this lane's elements (ones without a norm).
template <typename L>
__device__ __forceinline__ void load_norm(const PostArgs& a, const void* w, int sub, float (&wx)[L::PAIRS], float (&wy)[L::PAIRS]) {
  if constexpr (L::FAST) {
    if (w != nullptr) {
      if (a.norm_w_is_f32) {
        load_words(reinterpret_cast<const float*>(w) + 4 * sub, wx);
        load_words(reinterpret_cast<const float*>(w) + 4 * sub + (a.d >> 1), wy);
      } else {
        load_words(reinterpret_cast<const bf16*>(w) + 4 * sub, wx);
        load_words(reinterpret_cast<const bf16*>(w) + 4 * sub + (a.d >> 1), wy);
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < L::PAIRS; ++j) {
    const int p = L::pair(sub, j);
    wx[j] = wy[j] = 1.f;
    if (w == nullptr || p >= (a.d >> 1)) continue;
    int ia, ib;
    L::elements(p, a, ia, ib);
    wx[j] = load_flex(w, a.norm_w_is_f32, ia);
    wy[j] = load_flex(w, a.norm_w_is_f32, ib);
  }
}

// A token's position (0 without a rotation); positions were written before the step began.
__device__ __forceinline__ int position_of(const PostArgs& a, int t) {
  if (a.cos_table == nullptr) return 0;
  const int pos = a.positions[t];
  if (pos >= 0 && pos < a.max_positions) return pos;
  raise_fault(a.status, VOSTI_FAULT_POSITION_RANGE);
  return 0;
}

// Cosines and sines of this lane's pairs (no turn: 1 and 0).
template <typename L>
__device__ __forceinline__ void load_turn(const PostArgs& a, int pos, int sub, float (&c)[L::PAIRS], float (&s)[L::PAIRS]) {
#pragma unroll
  for (int j = 0; j < L::PAIRS; ++j) {
    c[j] = 1.f;
    s[j] = 0.f;
  }
  if (a.cos_table == nullptr) return;
  const int turning = a.rotary_dim >> 1;
  const int64_t at = (int64_t)pos * turning;
  if constexpr (L::FAST) {
    load_words(a.cos_table + at + 4 * sub, c);
    load_words(a.sin_table + at + 4 * sub, s);
  } else {
#pragma unroll
    for (int j = 0; j < L::PAIRS; ++j) {
      const int p = L::pair(sub, j);
      if (p >= turning) continue;
      c[j] = a.cos_table[at + p];
      s[j] = a.sin_table[at + p];
    }
  }
}

// All lanes of the warp take part: a head's sum of squares runs over its lanes. Lanes without `live` hold zeros and keep them (a norm without an
// eps would make them no numbers, and with them the largest size of the run).
template <typename L>
__device__ __forceinline__ void norm_and_turn(const PostArgs& a, bool normed, bool live, float (&x)[L::PAIRS], float (&y)[L::PAIRS], const float (&wx)[L::PAIRS],
                                              const float (&wy)[L::PAIRS], const float (&c)[L::PAIRS], const float (&s)[L::PAIRS]) {
  if (normed) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < L::PAIRS; ++j) ss = fmaf(x[j], x[j], fmaf(y[j], y[j], ss));
#pragma unroll
    for (int o = 1; o < L::LANES; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = live ? rsqrtf(fmaf(ss, a.inverse_d, a.eps)) : 0.f;
#pragma unroll
    for (int j = 0; j < L::PAIRS; ++j) {
      x[j] *= r * wx[j];
      y[j] *= r * wy[j];
    }
  }
  if (a.cos_table == nullptr) return;
#pragma unroll
  for (int j = 0; j < L::PAIRS; ++j) {
    const float u = x[j], v = y[j];
    if (!L::FAST && c[j] == 1.f && s[j] == 0.f) continue;        // (not turned: whatever its neighbour is)
    x[j] = u * c[j] - v * s[j];
    y[j] = v * c[j] + u * s[j];
  }
}

template <typename T, typename L>
__device__ __forceinline__ void store_head(const PostArgs& a, T* dst, int sub, const float (&x)[L::PAIRS], const float (&y)[L::PAIRS]) {
  if constexpr (L::FAST) {
    store_four(dst + 4 * sub, make_float4(x[0], x[1], x[2], x[3]));
    store_four(dst + 4 * sub + (a.d >> 1), make_float4(y[0], y[1], y[2], y[3]));
  } else {
#pragma unroll
    for (int j = 0; j < L::PAIRS; ++j) {
      const int p = L::pair(sub, j);
      if (p >= (a.d >> 1)) continue;
      int ia, ib;
      L::elements(p, a, ia, ib);
      dst[ia] = from_f32<T>(x[j]);
      dst[ib] = from_f32<T>(y[j]);
    }
  }
}

__device__ __forceinline__ uint32_t e4m3_pack4(float v0, float v1, float v2, float v3) {
  return (uint32_t)e4m3_pack(v0, v1) | (uint32_t)e4m3_pack(v2, v3) << 16;
}
// A word's four payloads under a scale 2^-(shift) times larger.
__device__ __forceinline__ uint32_t e4m3_again(uint32_t w, float f) {
  const float2 lo = e4m3_unpack((uint16_t)w), hi = e4m3_unpack((uint16_t)(w >> 16));
  return e4m3_pack4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
}

__device__ __forceinline__ int slot_at(const PostArgs& a, int t) { return t >= 0 && t < a.tokens ? a.slot_mapping[t] : -1; }

// The larger size; no number if either is none.
__device__ __forceinline__ float larger(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}
// Masks of the first n bytes of 16.
__device__ __forceinline__ uint4 first_bytes(int n) {
  return make_uint4(e4m3_first_bytes(n), e4m3_first_bytes(n - 4), e4m3_first_bytes(n - 8), e4m3_first_bytes(n - 12));
}
// Four values' payloads: earlier ones again under the larger scale, new ones, and what else there is.
__device__ __forceinline__ uint32_t merged(uint32_t there, uint32_t given, uint32_t old_bytes, uint32_t new_bytes, float f) {
  if (old_bytes != 0) there = (there & ~old_bytes) | (e4m3_again(there, f) & old_bytes);
  return (there & ~new_bytes) | (given & new_bytes);
}

// One run's keys (or VALUES): the tokens from t0 on of kv head g, by the whole CTA or by one warp. `rows`: [d][V_PITCH] of its own,
// `most_of`: a CTA's warps' largest sizes.
template <typename T, typename L, bool WHOLE, bool VALUES>
__device__ __forceinline__ void store_run(const PostArgs& a, int t0, int g, uint8_t* rows, float* most_of, const float (&wx)[L::PAIRS], const float (&wy)[L::PAIRS]) {
  constexpr int STEP = (WHOLE ? WARPS : 1) * L::HEADS, ROUNDS = ((WHOLE ? E4M3_BLOCK : SHORT) + STEP - 1) / STEP;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L::LANES;
  const int me = (WHOLE ? warp * L::HEADS : 0) + lane / L::LANES, thread = WHOLE ? threadIdx.x : lane, threads = WHOLE ? THREADS : 32;
  const int heads = a.nq + 2 * a.nkv, half = a.d >> 1;
  const int slot = slot_at(a, t0), offset = slot % E4M3_BLOCK;
  // the neighbours that continue the run (lane 16 never does)
  const unsigned gone = ~__ballot_sync(0xffffffffu, offset + lane < E4M3_BLOCK && slot_at(a, t0 + lane) == slot + lane);
  const int n = __ffs(gone) - 1;
  const int64_t page = slot / a.page_size, in_page = slot % a.page_size;
  const int64_t block = (page * a.nkv + g) * (a.page_size / E4M3_BLOCK) + in_page / E4M3_BLOCK;

  float c[VALUES ? 1 : ROUNDS][L::PAIRS], s[VALUES ? 1 : ROUNDS][L::PAIRS];
  if constexpr (!VALUES) {
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) load_turn<L>(a, position_of(a, t0 + min(me + i * STEP, n - 1)), sub, c[i], s[i]);
  }
  float x[ROUNDS][L::PAIRS], y[ROUNDS][L::PAIRS];
  int64_t at[ROUNDS];
  bool live[ROUNDS];
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    const int r = me + i * STEP;
    live[i] = r < n;
    at[i] = ((int64_t)(t0 + r) * heads + a.nq + (VALUES ? a.nkv : 0) + g) * a.d;
  }
  uint8_t* const scale = (VALUES ? a.v_scale : a.k_scale) + block;
  pdl_wait();                                                    // (nothing before this is of an earlier kernel's making)
  pdl_launch_dependents();
  const int old = offset > 0 ? *scale : 0;
  load_heads<T, L, ROUNDS>(a, at, live, sub, x, y);              // (zeros beyond the run)
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < ROUNDS; ++i) {
    if (i * STEP >= n) break;                                    // (the same in all lanes)
    if (!VALUES) {
      norm_and_turn<L>(a, a.k_norm_w != nullptr, live[i], x[i], y[i], wx, wy, c[i], s[i]);
    }
#pragma unroll
    for (int j = 0; j < L::PAIRS; ++j) most = larger(larger(most, x[i][j]), y[i][j]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = larger(most, __shfl_xor_sync(0xffffffffu, most, o));
  if constexpr (WHOLE) {
    if (lane == 0) most_of[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) most = larger(most, most_of[w]);
  }
  const int now = !(most < E4M3_LIMIT) ? E4M3_NAN_SCALE : max(e4m3_scale_for(most), old);
  // 2^-(scale - 127): the bits 254 - scale as an exponent (a scale that is no number: any payload will do)
  const float times = __uint_as_float((uint32_t)max(254 - now, 1) << 23);
  uint8_t* const payloads = (VALUES ? a.v : a.k) + block * E4M3_BLOCK * a.d;
  // earlier tokens under a larger scale (beyond 2^-127 everything is zero)
  const bool regrow = offset > 0 && now > old && now != E4M3_NAN_SCALE;
  const float f = regrow ? e4m3_scale(max(127 + old - now, 0)) : 1.f;

  if constexpr (!VALUES) {
    if (regrow) {
      uint4* const words = reinterpret_cast<uint4*>(payloads);
      for (int i0 = thread; i0 < offset * a.d / 16; i0 += ROWS * threads) {
        uint4 there[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) there[r] = i0 + r * threads < offset * a.d / 16 ? words[i0 + r * threads] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
          if (i0 + r * threads < offset * a.d / 16)
            words[i0 + r * threads] = make_uint4(e4m3_again(there[r].x, f), e4m3_again(there[r].y, f), e4m3_again(there[r].z, f), e4m3_again(there[r].w, f));
      }
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      if (!live[i]) continue;
      uint8_t* const key = payloads + (offset + me + i * STEP) * a.d;
      if constexpr (L::FAST) {
        *reinterpret_cast<uint32_t*>(key + 4 * sub) = e4m3_pack4(x[i][0] * times, x[i][1] * times, x[i][2] * times, x[i][3] * times);
        *reinterpret_cast<uint32_t*>(key + 4 * sub + half) = e4m3_pack4(y[i][0] * times, y[i][1] * times, y[i][2] * times, y[i][3] * times);
      } else {
#pragma unroll
        for (int j = 0; j < L::PAIRS; ++j) {
          const int p = L::pair(sub, j);
          if (p >= half) continue;
          int ia, ib;
          L::elements(p, a, ia, ib);
          const uint16_t both = e4m3_pack(x[i][j] * times, y[i][j] * times);
          key[ia] = (uint8_t)both;
          key[ib] = (uint8_t)(both >> 8);
        }
      }
    }
  } else {
    // A short run goes to its places byte by byte, without waiting for what is there; others, and runs that round earlier tokens again, through
    // shared memory, a feature's 16 tokens at a time.
    const bool direct = !WHOLE && !regrow;
    uint8_t* const column = direct ? payloads + offset + me : rows + offset + me;
    const int pitch = direct ? E4M3_BLOCK : V_PITCH;
#pragma unroll
    for (int i = 0; i < ROUNDS; ++i) {
      if (!live[i]) continue;
#pragma unroll
      for (int j = 0; j < L::PAIRS; ++j) {
        const int p = L::pair(sub, j);
        if (p >= half) continue;
        int ia, ib;
        L::elements(p, a, ia, ib);
        const uint16_t both = e4m3_pack(x[i][j] * times, y[i][j] * times);
        column[ia * pitch + i * STEP] = (uint8_t)both;
        column[ib * pitch + i * STEP] = (uint8_t)(both >> 8);
      }
    }
    if (!direct) {
      if constexpr (WHOLE) __syncthreads();
      else __syncwarp();
      const uint4 old_bytes = first_bytes(regrow ? offset : 0);
      const uint4 mine = first_bytes(offset + n), before = first_bytes(offset);
      for (int f0 = thread; f0 < a.d; f0 += ROWS * threads) {
        uint4 there[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const bool read = n < E4M3_BLOCK && f0 + r * threads < a.d;
          there[r] = read ? reinterpret_cast<const uint4*>(payloads)[f0 + r * threads] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const int feature = f0 + r * threads;
          if (feature >= a.d) break;
          const uint32_t* const row = reinterpret_cast<const uint32_t*>(rows + feature * V_PITCH);
          reinterpret_cast<uint4*>(payloads)[feature] =
              make_uint4(merged(there[r].x, row[0], old_bytes.x, mine.x & ~before.x, f), merged(there[r].y, row[1], old_bytes.y, mine.y & ~before.y, f),
                         merged(there[r].z, row[2], old_bytes.z, mine.z & ~before.z, f), merged(there[r].w, row[3], old_bytes.w, mine.w & ~before.w, f));
        }
      }
    }
  }
  if (thread == 0) *scale = (uint8_t)now;
  if constexpr (WHOLE) __syncthreads();                          // the next run takes the shared memory
  else __syncwarp();
}

// Blocks: `tile` neighbouring tokens' keys, or values, of a kv head, then query heads, WARPS * HEADS * Q_ITEMS of them.
template <typename T, typename L, int Q_ITEMS>
__global__ void __launch_bounds__(THREADS, Q_ITEMS > 1 && L::LANES * L::PAIRS <= 64 ? 6 : 4) qkv_post_e4m3_kernel(const PostArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % L::LANES;
  const int kv_blocks = (a.tokens + a.tile - 1) / a.tile * a.nkv * 2;

  if ((int)blockIdx.x >= kv_blocks) {
    // ------------------------------------------------------------ queries: (token, head) pairs in their order
    float wx[L::PAIRS], wy[L::PAIRS];
    load_norm<L>(a, a.q_norm_w, sub, wx, wy);
    constexpr int CHUNK = L::HEADS * Q_ITEMS;                    // heads of a token that a warp takes
    const int of_token = (a.nq + CHUNK - 1) / CHUNK, chunk = ((int)blockIdx.x - kv_blocks) * WARPS + warp;
    const int t = min(chunk / of_token, a.tokens - 1), h0 = chunk % of_token * CHUNK + lane / L::LANES;
    const int pos = position_of(a, t);
    pdl_wait();
    pdl_launch_dependents();
    if (chunk >= a.tokens * of_token) return;
    float x[Q_ITEMS][L::PAIRS], y[Q_ITEMS][L::PAIRS], c[L::PAIRS], s[L::PAIRS];
    const int64_t in = (int64_t)t * (a.nq + 2 * a.nkv) * a.d, out = (int64_t)t * a.nq * a.d;
    int64_t at[Q_ITEMS];
    bool live[Q_ITEMS];
#pragma unroll
    for (int i = 0; i < Q_ITEMS; ++i) {
      live[i] = h0 + i * L::HEADS < a.nq;
      at[i] = in + (int64_t)(h0 + i * L::HEADS) * a.d;
    }
    load_heads<T, L, Q_ITEMS>(a, at, live, sub, x, y);
    load_turn<L>(a, pos, sub, c, s);                             // (behind the heads: the position has arrived by now)
#pragma unroll
    for (int i = 0; i < Q_ITEMS; ++i) norm_and_turn<L>(a, a.q_norm_w != nullptr, true, x[i], y[i], wx, wy, c, s);
#pragma unroll
    for (int i = 0; i < Q_ITEMS; ++i)
      if (live[i]) store_head<T, L>(a, reinterpret_cast<T*>(a.q_out) + out + (int64_t)(h0 + i * L::HEADS) * a.d, sub, x[i], y[i]);
    return;
  }

  // -------------------------------------------------------------- keys or values of one kv head
  extern __shared__ __align__(16) uint8_t rows_of_values[];     // [WARPS][d][V_PITCH]
  __shared__ float most_of[WARPS];
  const int item = (int)blockIdx.x >> 1, g = item % a.nkv, t_begin = item / a.nkv * a.tile, t_end = min(a.tokens, t_begin + a.tile);
  const bool values = blockIdx.x & 1;
  float wx[L::PAIRS], wy[L::PAIRS];
  load_norm<L>(a, values ? nullptr : a.k_norm_w, sub, wx, wy);
  // which of the tile's tokens begin a run, and which runs are short (lane i: token t_begin + i; slots were written before the step)
  const int my_t = t_begin + lane;
  bool begins = false, is_short = false;
  if (my_t < t_end) {
    const int slot = slot_at(a, my_t), before = slot_at(a, my_t - 1);
    if (slot < -1 || slot >= a.num_slots) {
      if (warp == 0 && blockIdx.x % (2 * a.nkv) == 0) raise_fault(a.status, VOSTI_FAULT_SLOT_RANGE);
    } else if (slot >= 0) {
      const bool same = before >= 0 && before / E4M3_BLOCK == slot / E4M3_BLOCK;
      begins = !same;
      // a block's tokens of a step stand next to one another in its order; others are left out
      if (same && before != slot - 1 && warp == 0 && blockIdx.x % (2 * a.nkv) == 0) raise_fault(a.status, VOSTI_FAULT_SLOT_RANGE);
      is_short = begins && !(slot % E4M3_BLOCK + SHORT < E4M3_BLOCK && slot_at(a, my_t + SHORT) == slot + SHORT);
    }
  }
  unsigned long_runs = __ballot_sync(0xffffffffu, begins && !is_short), short_runs = __ballot_sync(0xffffffffu, is_short);
  // Blocks that hold earlier tokens: on their way to L2 before the projection ends.
  for (unsigned todo = long_runs | short_runs; todo != 0; todo &= todo - 1) {
    const int slot = slot_at(a, t_begin + __ffs(todo) - 1), line = (int)threadIdx.x * 128;
    if (slot % E4M3_BLOCK == 0 || line >= E4M3_BLOCK * a.d + 128) continue;
    const int64_t block = ((int64_t)(slot / a.page_size) * a.nkv + g) * (a.page_size / E4M3_BLOCK) + slot % a.page_size / E4M3_BLOCK;
    const uint8_t* const from = threadIdx.x == 0 ? (values ? a.v_scale : a.k_scale) + block : (values ? a.v : a.k) + block * E4M3_BLOCK * a.d + line - 128;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(from));
  }
  uint8_t* const mine = rows_of_values + warp * a.d * V_PITCH;
  for (; long_runs != 0; long_runs &= long_runs - 1) {           // (the same in all warps)
    const int t0 = t_begin + __ffs(long_runs) - 1;
    if (values) store_run<T, L, true, true>(a, t0, g, rows_of_values, most_of, wx, wy);
    else store_run<T, L, true, false>(a, t0, g, rows_of_values, most_of, wx, wy);
  }
  for (int i = 0; short_runs != 0; short_runs &= short_runs - 1, ++i) {
    const int t0 = t_begin + __ffs(short_runs) - 1;
    if (i % WARPS != warp) continue;
    if (values) store_run<T, L, false, true>(a, t0, g, mine, nullptr, wx, wy);
    else store_run<T, L, false, false>(a, t0, g, mine, nullptr, wx, wy);
  }
  pdl_wait();                                                    // (warps that stored nothing)
}

template <typename T, typename L, int Q_ITEMS>
cudaError_t launch_post_items(const PostArgs& a, cudaStream_t stream) {
  constexpr int CHUNK = L::HEADS * Q_ITEMS;
  const int64_t q_blocks = ((int64_t)a.tokens * ((a.nq + CHUNK - 1) / CHUNK) + WARPS - 1) / WARPS;
  const int64_t blocks = (int64_t)((a.tokens + a.tile - 1) / a.tile) * a.nkv * 2 + q_blocks;
  return vosti_launch(qkv_post_e4m3_kernel<T, L, Q_ITEMS>, dim3((unsigned)blocks), dim3(THREADS), (size_t)WARPS * a.d * V_PITCH, stream, a);
}
template <typename T, typename L>
cudaError_t launch_post(const PostArgs& a, cudaStream_t stream) {
  return a.tokens <= FEW ? launch_post_items<T, L, 1>(a, stream) : launch_post_items<T, L, Q_MANY>(a, stream);
}
template <typename T>
cudaError_t launch_post_as(const PostArgs& a, cudaStream_t stream) {
  // whole words: four elements of every operand
  const uintptr_t words = (uintptr_t)a.partial | (uintptr_t)a.cos_table | (uintptr_t)a.sin_table | (uintptr_t)a.q_norm_w | (uintptr_t)a.k_norm_w, rows = (uintptr_t)a.qkv | (uintptr_t)a.q_out;
  if ((a.cos_table == nullptr || (a.rotary_dim == a.d && !a.interleaved)) && words % 16 == 0 && rows % (4 * sizeof(T)) == 0) {
    if (a.d == 64) return launch_post<T, Lay<8, 4, true>>(a, stream);
    if (a.d == 128) return launch_post<T, Lay<16, 4, true>>(a, stream);
    if (a.d == 256) return launch_post<T, Lay<32, 4, true>>(a, stream);
  }
  if (a.d <= 64) return launch_post<T, Lay<32, 1, false>>(a, stream);
  return a.d <= 128 ? launch_post<T, Lay<32, 2, false>>(a, stream) : launch_post<T, Lay<32, 4, false>>(a, stream);
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
  if (tokens == 0) return VOSTI_OK;                              // (arrays of nothing are null)
  VOSTI_REQUIRE((qkv != nullptr) != (partial != nullptr), "qkv_post_e4m3: give the projection or its partial sums");
  VOSTI_REQUIRE(partial == nullptr || splits >= 1, "qkv_post_e4m3: bad split count");
  VOSTI_REQUIRE(num_slots >= 0 && num_slots <= 0x7fffffff, "qkv_post_e4m3: a cache of %lld slots is too large", (long long)num_slots);
  VOSTI_REQUIRE((cos_table == nullptr) == (sin_table == nullptr), "qkv_post_e4m3: cos and sin go together");
  VOSTI_REQUIRE(cos_table == nullptr || positions != nullptr, "qkv_post_e4m3: rotation needs positions");
  VOSTI_REQUIRE(cos_table == nullptr || (rotary_dim > 0 && rotary_dim <= d && rotary_dim % 2 == 0),
                "qkv_post_e4m3: rotary_dim %d must be even and between 2 and head_dim %d", rotary_dim, d);
  VOSTI_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0, "qkv_post_e4m3: the cache must start on 16 bytes");
  VOSTI_REQUIRE(slot_mapping != nullptr && k != nullptr && v != nullptr && k_scale != nullptr && v_scale != nullptr, "qkv_post_e4m3: the cache is missing");
  VOSTI_REQUIRE((int64_t)tokens * (nq + 2 * nkv) <= 0x7fffffff - 4096, "qkv_post_e4m3: too many tokens and heads for one launch");
  // Neighbouring tokens whose runs a CTA takes: few tokens one, so that none waits for another's run; more of them four, a run a warp in a batch of
  // single tokens; many, as prompts bring them, eight or sixteen, which hold a run or two. us with tiles of 1, 4, 8, 16 (8B sizes): 8 single tokens 3.0, 3.1, 4.2,
  // 4.2; 64 5.4, 3.7, 5.0, 8.6; 256 12.3, 9.0, 8.8, 13.0; a prompt of 512 13.3, 6.6, 5.8, 5.4; of 2,048 53, 25.9, 21.0, 18.6; of 4,096 105, 52, 42, 37.5.
  const int tile = tokens <= FEW ? 1 : tokens <= MANY ? 4 : tokens <= 4 * MANY ? 8 : 16;
  const PostArgs a = {qkv, partial, splits, (int64_t)tokens * (nq + 2 * nkv) * d, q_out, (uint8_t*)k, (uint8_t*)v, (uint8_t*)k_scale,
                      (uint8_t*)v_scale, q_norm_w, k_norm_w, norm_w_is_f32, eps, 1.f / (float)d, cos_table, sin_table, max_positions, positions, slot_mapping,
                      num_slots, page_size, tokens, nq, nkv, d, cos_table != nullptr ? rotary_dim : d, interleaved, tile, status};
  const cudaError_t e = is_f32 ? launch_post_as<float>(a, stream) : launch_post_as<bf16>(a, stream);
  if (e != cudaSuccess) {
    vosti_set_error("qkv_post_e4m3: %s", cudaGetErrorString(e));
    return (int)e;
  }
  VOSTI_LAUNCH_CHECK();
}
