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
  int64_t tokens;
  int32_t ldx, ldy, n, h, w, c, heads, head_dim, pairs, layout, naxes, pos_per_image, inverse;
};

__device__ __forceinline__ int32_t rotary_pos(const RotaryArgs& a, int64_t token, int axis) {
  const int64_t hw = (int64_t)a.h * a.w;
  if (a.pos) {
    const int64_t per_axis = a.pos_per_image ? a.tokens : hw;
    return a.pos[axis * per_axis + (a.pos_per_image ? token : token % hw)];
  }
  if (a.naxes == 1) return (int32_t)(token % hw);
  const int k = axis + 3 - a.naxes;   // 0: image, 1: row, 2: column
  return (int32_t)(k == 0 ? token / hw : k == 1 ? token / a.w % a.h : token % a.w);
}

// One thread per (token, pair of the head, or channel that passes through).
template <typename T>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const int rest = a.head_dim - 2 * a.pairs, tail = a.c - a.heads * a.head_dim;
  const int items = a.pairs + rest + tail;
  const int64_t total = a.tokens * items;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < total; id += (int64_t)gridDim.x * 256) {
    const int64_t token = id / items;
    const int it = (int)(id % items);
    const T* x = (const T*)a.x + token * a.ldx;
    T* y = (T*)a.y + token * a.ldy;
    if (it < a.pairs) {
      const RotaryPair rp = a.table[it];
      float cs, sn;
      rotary_angle(rp.freq, rotary_pos(a, token, rp.axis), cs, sn);
      if (a.inverse) sn = -sn;
      const int i0 = a.layout == LIC_ROTARY_HALF ? it : 2 * it;
      const int i1 = a.layout == LIC_ROTARY_HALF ? it + a.pairs : 2 * it + 1;
      for (int j = 0; j < a.heads; ++j) {
        const float p = to_f(x[j * a.head_dim + i0]), q = to_f(x[j * a.head_dim + i1]);
        y[j * a.head_dim + i0] = from_f<T>(p * cs - q * sn);
        y[j * a.head_dim + i1] = from_f<T>(p * sn + q * cs);
      }
    } else if (a.x != a.y) {
      if (it < a.pairs + rest) {
        for (int j = 0; j < a.heads; ++j) y[j * a.head_dim + it + a.pairs] = x[j * a.head_dim + it + a.pairs];
      } else {
        const int ch = a.heads * a.head_dim + it - a.pairs - rest;
        y[ch] = x[ch];
      }
    }
  }
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
  if ((double)n * h * w >= 2147483648.0 * 64) return fail("rotary: too many tokens");
  if (!x || !y || !table) return fail("rotary: null pointer");
  if (x == y && ldx != ldy) return fail("rotary: in place needs ldx == ldy");
  RotaryArgs a{x, y, (const RotaryPair*)table, pos, (int64_t)n * h * w, ldx, ldy, n, h, w, c, heads, head_dim, pairs,
               layout, naxes, pos_per_image, inverse};
  const int64_t items = a.tokens * (head_dim - pairs + c - heads * head_dim);
  const int64_t need = (items + 255) / 256;
  const unsigned blocks = (unsigned)(need < 65536 ? need : 65536);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == LIC_F32) hipLaunchKernelGGL(rotary_kernel<float>, dim3(blocks), dim3(256), 0, s, a);
  else if (dtype == LIC_F16) hipLaunchKernelGGL(rotary_kernel<half_t>, dim3(blocks), dim3(256), 0, s, a);
  else hipLaunchKernelGGL(rotary_kernel<bf16_t>, dim3(blocks), dim3(256), 0, s, a);
  LIC_CHECK_LAUNCH();
  return 0;
}
