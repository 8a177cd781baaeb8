// Rotary positions over several axes (gfx950): each channel pair (a, b) of a head turns by
// t = pos[axis] * freq, (a cos t - b sin t, a sin t + b cos t).
#include "lic_common.h"

namespace lic {

struct RotaryPair {
  uint64_t freq;   // angle at position 1, in 2^-64 turns
  int32_t axis, zero;
};

// cos / sin of pos * freq.  The angle lives in 64-bit fixed-point turns, where the product wraps modulo one
// turn by itself: exact for any 32-bit position, no range reduction.  Nearest quarter turn off the top, the
// rest (|r| <= 1/8 turn, 2^-32 turn steps: 1.5e-9 rad) through the Taylor series of sin and cos to x^9 / x^10
// (first terms left out: 1.8e-9, 1.2e-10 at pi/4).
__device__ __forceinline__ void rotary_angle(uint64_t freq, int32_t pos, float& c, float& s) {
  const uint64_t turns = freq * (uint64_t)(int64_t)pos;
  const uint32_t hi = (uint32_t)(turns >> 32);
  const uint32_t quad = (hi + 0x20000000u) >> 30;
  const float r = (float)(int32_t)(hi - (quad << 30)) * 1.4629180792671596e-9f;   // 2 pi / 2^32
  const float r2 = r * r;
  const float sn = r + r * r2 * (-1.66666667e-1f + r2 * (8.33333333e-3f + r2 * (-1.98412698e-4f + r2 * 2.75573192e-6f)));
  const float cs = 1.f + r2 * (-0.5f + r2 * (4.16666667e-2f + r2 * (-1.38888889e-3f + r2 * (2.48015873e-5f - r2 * 2.75573192e-7f))));
  const float a = (quad & 1) ? sn : cs, b = (quad & 1) ? cs : sn;
  c = (quad == 1 || quad == 2) ? -a : a;
  s = (quad & 2) ? -b : b;
}

struct RotaryArgs {
  const void* x;
  void* y;
  const RotaryPair* table;
  const int32_t* pos;
  int32_t tokens, ldx, ldy, h, w, heads, head_dim, pairs, naxes, pos_per_image, inverse;
  int32_t c, per_block;        // channels of the view, tokens of a block
  int32_t vecs, head_vecs;     // work items of a token, and of one of its heads
  uint32_t inv_vecs, inv_head_vecs, inv_pairs;   // rotary_inverse of the divisors
};

// q = i / d as the high word of i * (floor(2^32 / d) + 1): too large by less than i / 2^32, so exact where i d < 2^32.
// The sizes keep to that: angles i < 8192, d <= 4096; vectors of several tokens i < 4096, d <= 1024 (of one token: q = 0);
// vectors of a head i <= 2^18, d <= 2^13.
static uint32_t rotary_inverse(int d) { return d > 1 ? (uint32_t)((1ull << 32) / d + 1) : 0; }
__device__ __forceinline__ int rotary_div(int i, uint32_t inv) { return inv ? (int)__umulhi((uint32_t)i, inv) : i; }

__device__ __forceinline__ int32_t rotary_pos(const RotaryArgs& a, uint32_t token, int axis) {
  const uint32_t hw = (uint32_t)a.h * a.w;
  if (a.pos) return a.pos_per_image ? a.pos[(int64_t)axis * a.tokens + token] : a.pos[(int64_t)axis * hw + token % hw];
  if (a.naxes == 1) return (int32_t)(token % hw);
  const int k = axis + 3 - a.naxes;   // 0: image, 1: row, 2: column
  return (int32_t)(k == 0 ? token / hw : k == 1 ? token / a.w % a.h : token % a.w);
}

constexpr int ROTARY_UNROLL = 4;

// How a vector of V elements meets its pairs' other members:
//   PARTNER  every vector of the token is read, turned or passed through, and written; the members that its own ones
//            are paired with are read a second time (from the cache).  Loads and stores run over the token without a
//            gap: 111 us for 61440 tokens x 2560 bf16 channels, 96 of 128 rotated (5.7 TB/s; 151 us in the form below).
//   INSIDE   the pairs lie inside the vector.
//   BOTH     in place, where nobody may read what another thread writes: a thread takes both members of its pairs,
//            and touches nothing else.  The q | k window of a 576-channel qkv map, 32 x 64 x 64 fp16: 35 us (5.7 TB/s).
enum RotaryForm { PARTNER, INSIDE, BOTH };

// A block takes a few whole tokens: each angle's cos / sin once into LDS (all heads of the token share it), then the
// tokens' vectors stream through, consecutive threads on consecutive vectors, ROTARY_UNROLL of them in flight a thread.
// Bound by the bytes of x and y: 32 x 64 x 64 tokens of 384 fp16 channels 35 us (5.7 TB/s), 8 x 64 x 64 of 576 bf16 channels
// with neighbouring pairs 13.9 us (5.4 TB/s); two tokens 2.8 us.
template <typename T, int V, bool HALF, RotaryForm FORM>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 turn[];   // [tokens of the block][pairs]
  typedef T Vec __attribute__((ext_vector_type(V)));
  const int64_t first = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.per_block;
  if (first >= a.tokens) return;
  const int t0 = (int)first;
  const int nt = min(a.per_block, a.tokens - t0);
  for (int i = threadIdx.x; i < nt * a.pairs; i += 256) {
    const int t = rotary_div(i, a.inv_pairs), p = i - t * a.pairs;
    const RotaryPair rp = a.table[p];
    float2 cs;
    rotary_angle(rp.freq, rotary_pos(a, (uint32_t)(t0 + t), rp.axis), cs.x, cs.y);
    if (a.inverse) cs.y = -cs.y;
    turn[i] = cs;
  }
  __syncthreads();
  const T* x = (const T*)a.x + (int64_t)t0 * a.ldx;
  T* y = (T*)a.y + (int64_t)t0 * a.ldy;
  const int n = nt * a.vecs, in_heads = a.heads * a.head_vecs;
  const int step = HALF ? a.pairs : 1;   // from a pair's first member to its second (INSIDE: both in one vector)
  for (int i0 = threadIdx.x; i0 < n; i0 += 256 * ROTARY_UNROLL) {
    Vec u[ROTARY_UNROLL], v[ROTARY_UNROLL];
    int at[ROTARY_UNROLL], tok[ROTARY_UNROLL], pair[ROTARY_UNROLL];
    bool turns[ROTARY_UNROLL], second[ROTARY_UNROLL];
#pragma unroll
    for (int k = 0; k < ROTARY_UNROLL; ++k) {
      const int i = i0 + 256 * k;
      const int t = rotary_div(i, a.inv_vecs), r = i - t * a.vecs;
      const int j = rotary_div(r, a.inv_head_vecs), q = (r - j * a.head_vecs) * V;
      int d = q;   // channel in the head
      turns[k] = r < in_heads && i < n;
      second[k] = false;
      tok[k] = t;
      if constexpr (FORM == BOTH) {
        d = HALF ? q : 2 * q;
        pair[k] = t * a.pairs + q;
      } else if constexpr (FORM == INSIDE) {
        turns[k] = turns[k] && q < 2 * a.pairs;
        pair[k] = t * a.pairs + q / 2;
      } else {
        turns[k] = turns[k] && q < 2 * a.pairs;
        second[k] = HALF ? q >= a.pairs : q & 1;
        pair[k] = t * a.pairs + (HALF ? (second[k] ? q - a.pairs : q) : q / 2);
      }
      at[k] = r < in_heads ? j * a.head_dim + d : a.heads * a.head_dim + (r - in_heads) * V;
      if (i < n) {
        const T* px = x + (int64_t)t * a.ldx + at[k];
        u[k] = *(const Vec*)px;
        if constexpr (FORM != INSIDE)
          if (turns[k]) v[k] = *(const Vec*)(second[k] ? px - step : px + step);
      }
    }
#pragma unroll
    for (int k = 0; k < ROTARY_UNROLL; ++k) {
      if (i0 + 256 * k < n) {
        if (turns[k]) {
          if constexpr (FORM == INSIDE) {
#pragma unroll
            for (int e = 0; e + 1 < V; e += 2) {
              const float2 cs = turn[pair[k] + e / 2];
              const float p = to_f(u[k][e]), q = to_f(u[k][e + 1]);
              u[k][e] = from_f<T>(p * cs.x - q * cs.y);
              u[k][e + 1] = from_f<T>(p * cs.y + q * cs.x);
            }
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float2 cs = turn[pair[k] + e];
              const float p = to_f(u[k][e]), q = to_f(v[k][e]);
              if constexpr (FORM == BOTH) v[k][e] = from_f<T>(p * cs.y + q * cs.x);
              u[k][e] = from_f<T>(second[k] ? q * cs.y + p * cs.x : p * cs.x - q * cs.y);
            }
          }
        }
        T* py = y + (int64_t)tok[k] * a.ldy + at[k];
        *(Vec*)py = u[k];
        if constexpr (FORM == BOTH) *(Vec*)(py + step) = v[k];
      }
    }
  }
}

template <typename T, int V, bool HALF, RotaryForm FORM>
static int rotary_launch(RotaryArgs a, hipStream_t s) {
  // INSIDE in place: the rotated channels only
  a.head_vecs = (FORM == BOTH ? a.pairs : a.x == a.y ? 2 * a.pairs : a.head_dim) / V;
  a.vecs = a.heads * a.head_vecs + (a.x == a.y ? 0 : (a.c - a.heads * a.head_dim) / V);
  // tokens of a block: vectors for every thread's ROTARY_UNROLL, at most 16 KB of angles (one token's at least),
  // fewer where the grid would leave compute units idle
  int tk = (ROTARY_UNROLL * 256 + a.vecs - 1) / a.vecs;
  tk = tk < 2048 / a.pairs ? tk : 2048 / a.pairs;
  tk = tk < a.tokens / 1024 ? tk : a.tokens / 1024;
  a.per_block = tk > 1 ? tk : 1;
  a.inv_vecs = a.per_block > 1 ? rotary_inverse(a.vecs) : 1;
  a.inv_head_vecs = rotary_inverse(a.head_vecs);
  a.inv_pairs = rotary_inverse(a.pairs);
  // a dimension of a launch has less than 2^32 threads
  const unsigned blocks = (unsigned)(((int64_t)a.tokens + a.per_block - 1) / a.per_block);
  const unsigned bx = blocks < 1u << 22 ? blocks : 1u << 22;
  const unsigned lds = (unsigned)(a.per_block * a.pairs * sizeof(float2));
  hipLaunchKernelGGL((rotary_kernel<T, V, HALF, FORM>), dim3(bx, (blocks + bx - 1) / bx), dim3(256), lds, s, a);
  LIC_CHECK_LAUNCH();
  return 0;
}

template <typename T, int V>
static int rotary_run(const RotaryArgs& a, bool half, hipStream_t s) {
  if (half) return a.x == a.y ? rotary_launch<T, V, true, BOTH>(a, s) : rotary_launch<T, V, true, PARTNER>(a, s);
  if constexpr (V > 1) return rotary_launch<T, V, false, INSIDE>(a, s);
  else return a.x == a.y ? rotary_launch<T, V, false, BOTH>(a, s) : rotary_launch<T, V, false, PARTNER>(a, s);
}

// The widest vectors (up to 16 bytes) that every offset is a multiple of.
template <typename T>
static int rotary_any(const RotaryArgs& a, bool half, hipStream_t s) {
  const uintptr_t p = (uintptr_t)a.x | (uintptr_t)a.y;
  const int64_t units = (int64_t)a.ldx | a.ldy | a.head_dim | a.c | (half ? a.pairs : 2 * a.pairs);
  auto fits = [&](int v) { return p % (v * sizeof(T)) == 0 && units % v == 0; };
  if constexpr (sizeof(T) == 2)
    if (fits(8)) return rotary_run<T, 8>(a, half, s);
  if (fits(4)) return rotary_run<T, 4>(a, half, s);
  if (fits(2)) return rotary_run<T, 2>(a, half, s);
  return rotary_run<T, 1>(a, half, s);
}

}  // namespace lic

extern "C" int lic_rotary(int32_t dtype, const void* x, int32_t ldx, int32_t n, int32_t h, int32_t w, int32_t c,
                          int32_t heads, int32_t head_dim, int32_t pairs, int32_t layout, const void* table,
                          int32_t naxes, const int32_t* pos, int32_t pos_per_image, int32_t inverse, void* y,
                          int32_t ldy, lic_stream_t stream) {
  using namespace lic;
  if (dtype != LIC_F32 && dtype != LIC_F16 && dtype != LIC_BF16) return fail("rotary: bad dtype");
  if (n < 0 || h < 0 || w < 0) return fail("rotary: negative size");
  if (heads < 1 || head_dim < 2 || pairs < 1 || pairs > head_dim / 2 || c < 1 ||
      (int64_t)heads * head_dim > c || ldx < c || ldy < c)
    return fail("rotary: heads x head_dim channels with 2 x pairs rotated have to fit the view");
  if (layout != LIC_ROTARY_HALF && layout != LIC_ROTARY_PAIRS) return fail("rotary: bad layout");
  if (naxes < 1 || naxes > LIC_ROTARY_MAX_AXES || (!pos && naxes > 3)) return fail("rotary: naxes out of range");
  if ((int64_t)n * h * w == 0) return 0;
  if ((double)n * h * w >= 2147483648.0 || head_dim > 8192 || c > (1 << 18))
    return fail("rotary: up to 2^31 tokens, 8192 channels a head, 2^18 channels a token");
  if (!x || !y || !table) return fail("rotary: null pointer");
  if (x == y && ldx != ldy) return fail("rotary: in place needs ldx == ldy");
  RotaryArgs a{x, y, (const RotaryPair*)table, pos, n * h * w, ldx, ldy, h, w, heads, head_dim, pairs, naxes,
               pos_per_image, inverse, c};
  hipStream_t s = (hipStream_t)stream;
  const bool half = layout == LIC_ROTARY_HALF;
  if (dtype == LIC_F32) return rotary_any<float>(a, half, s);
  if (dtype == LIC_F16) return rotary_any<half_t>(a, half, s);
  return rotary_any<bf16_t>(a, half, s);
}
