// Products in 8-bit integers with a scale for each token and output channel (gfx950).
#include "lic_common.h"

namespace lic {

// code = rint(127 x / amax), half to even, exactly.  x and amax are first scaled by one power of two (amax to
// [1, 2)), so nothing overflows; the fp32 quotient is exact enough except next to a border k + 1/2, which is
// decided in 64 bits, where 254 x and (2k + 1) amax are exact.
__device__ __forceinline__ int quant_code(float x, float amax) {
  const float t = x * 127.f / amax;
  float q = rintf(t);
  const float d = t - q;
  if (fabsf(fabsf(d) - 0.5f) < 1e-4f) {
    const double lo = floor((double)t);   // t is within 1e-4 of lo + 1/2
    const double diff = 254.0 * (double)x - (2.0 * lo + 1.0) * (double)amax;
    q = (float)(diff > 0 ? lo + 1 : diff < 0 ? lo : 2.0 * rint(lo * 0.5 + 0.25));
  }
  return (int)q;
}

// Largest magnitude of a row; NaN if the row holds a NaN or an infinity.
__device__ __forceinline__ float quant_absmax(float m, float v) {
  const float a = fabsf(v);
  return a <= m ? m : (a < INFINITY ? (m == m ? a : m) : NAN);
}

// One wave per row.
template <typename T>
__global__ __launch_bounds__(256) void quantize_int8_kernel(const T* __restrict__ x, int64_t ldx, int m, int k,
                                                            int8_t* __restrict__ codes, int kpad,
                                                            float* __restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= m) return;
  const T* xr = x + row * ldx;
  float top = 0.f;
  for (int j = lane; j < k; j += 64) top = quant_absmax(top, to_f(xr[j]));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float other = __shfl_xor(top, o);
    top = other != other ? other : (other > top ? other : top);
  }
  if (lane == 0) scale[row] = top / 127.f;
  const bool live = top > 0.f;   // false for zero rows and NaN
  int e = 0;
  if (live) (void)frexpf(top, &e);
  const float amax = live ? ldexpf(top, 1 - e) : 1.f;
  int8_t* cr = codes + row * kpad;
  for (int j = lane; j < kpad; j += 64)
    cr[j] = (live && j < k) ? (int8_t)quant_code(ldexpf(to_f(xr[j]), 1 - e), amax) : (int8_t)0;
}

struct Int8Args {
  const int8_t* xc;
  const float* xs;
  const int8_t* w;
  const float* ws;
  const float* bias;
  const void* r1;
  void* y;
  int64_t ldr1, ldy;
  int32_t m, n, kpad, act;
  float slope;
};

template <typename T>
__device__ __forceinline__ void int8_store(const Int8Args& a, int64_t row, int col, int acc, float xs) {
  float v = (float)acc * (xs * a.ws[col]) + (a.bias ? a.bias[col] : 0.f);
  v = apply_act(v, a.act, a.slope);
  if (a.r1) v += to_f(((const T*)a.r1)[row * a.ldr1 + col]);
  ((T*)a.y)[row * a.ldy + col] = from_f<T>(v);
}

// One output per thread, four products an instruction.
template <typename T>
__global__ __launch_bounds__(256) void linear_int8_kernel(Int8Args a) {
  const int col = blockIdx.x * 16 + (threadIdx.x & 15);
  const int64_t row = (int64_t)blockIdx.y * 16 + (threadIdx.x >> 4);
  if (row >= a.m || col >= a.n) return;
  const int* p = (const int*)(a.xc + row * a.kpad);
  const int* q = (const int*)(a.w + (int64_t)col * a.kpad);
  int acc = 0;
  for (int j = 0; j < a.kpad / 4; ++j) acc = __builtin_amdgcn_sdot4(p[j], q[j], acc, false);
  int8_store<T>(a, row, col, acc, a.xs[row]);
}

template <typename T>
static int quantize_run(const void* x, int64_t ldx, int m, int k, int8_t* codes, int kpad, float* scale,
                        hipStream_t s) {
  hipLaunchKernelGGL(quantize_int8_kernel<T>, dim3((unsigned)((m + 3) / 4)), dim3(256), 0, s, (const T*)x, ldx, m, k,
                     codes, kpad, scale);
  LIC_CHECK_LAUNCH();
  return 0;
}

static int quantize_any(int32_t dtype, const void* x, int64_t ldx, int m, int k, int8_t* codes, int kpad, float* scale,
                        hipStream_t s) {
  if (dtype == LIC_F32) return quantize_run<float>(x, ldx, m, k, codes, kpad, scale, s);
  if (dtype == LIC_F16) return quantize_run<half_t>(x, ldx, m, k, codes, kpad, scale, s);
  return quantize_run<bf16_t>(x, ldx, m, k, codes, kpad, scale, s);
}

template <typename T>
static int linear_run(const Int8Args& a, hipStream_t s) {
  if ((a.m + 15) / 16 > 65535) {   // the grid's second dimension
    Int8Args b = a;
    const int rows = 65535 * 16;
    for (int64_t r = 0; r < a.m; r += rows) {
      b.xc = a.xc + r * a.kpad;
      b.xs = a.xs + r;
      b.y = (T*)a.y + r * a.ldy;
      b.r1 = a.r1 ? (const T*)a.r1 + r * a.ldr1 : nullptr;
      b.m = (int)(a.m - r < rows ? a.m - r : rows);
      if (linear_run<T>(b, s)) return 1;
    }
    return 0;
  }
  hipLaunchKernelGGL(linear_int8_kernel<T>, dim3((unsigned)((a.n + 15) / 16), (unsigned)((a.m + 15) / 16)), dim3(256),
                     0, s, a);
  LIC_CHECK_LAUNCH();
  return 0;
}

static int check_sizes(const char* who, int32_t dtype, int32_t m, int32_t k, int32_t kpad) {
  if (dtype != LIC_F32 && dtype != LIC_F16 && dtype != LIC_BF16) return fail(std::string(who) + ": bad dtype");
  if (m < 0 || k < 1 || k > LIC_INT8_MAX_K || kpad < k || kpad % 64 || kpad > LIC_INT8_MAX_K)
    return fail(std::string(who) + ": sizes out of range (k up to 131072, kpad a multiple of 64)");
  return 0;
}

}  // namespace lic

extern "C" int lic_quantize_int8(int32_t dtype, const void* x, int64_t ldx, int32_t m, int32_t k, int8_t* codes,
                                 int32_t kpad, float* scale, lic_stream_t stream) {
  using namespace lic;
  if (check_sizes("quantize_int8", dtype, m, k, kpad)) return 1;
  if (m == 0) return 0;
  if (!x || !codes || !scale || ldx < k) return fail("quantize_int8: null pointer or row stride below k");
  if ((uintptr_t)codes % 16) return fail("quantize_int8: codes have to be 16-byte aligned");
  return quantize_any(dtype, x, ldx, m, k, codes, kpad, scale, (hipStream_t)stream);
}

extern "C" int64_t lic_linear_int8_workspace(int32_t m, int32_t kpad) {
  if (m < 0 || kpad < 1 || kpad > LIC_INT8_MAX_K) return -1;
  const int64_t codes = (int64_t)m * kpad;
  return (codes + 15) / 16 * 16 + 4 * (int64_t)m;
}

extern "C" int lic_linear_int8(int32_t dtype, const void* x, int64_t ldx, const int8_t* xcodes, const float* xscale,
                               int32_t m, int32_t k, const int8_t* w, int32_t kpad, const float* wscale,
                               const float* bias, int32_t n, int32_t act, float slope, const void* r1, int64_t ldr1,
                               void* y, int64_t ldy, void* ws, int64_t ws_bytes, lic_stream_t stream) {
  using namespace lic;
  if (check_sizes("linear_int8", dtype, m, k, kpad)) return 1;
  if (n < 1) return fail("linear_int8: n out of range");
  if (act < LIC_ACT_NONE || act > LIC_ACT_GELU) return fail("linear_int8: act has to be none, relu, lrelu or gelu");
  if (m == 0) return 0;
  if (!w || !wscale || !y || ldy < n || (r1 && ldr1 < n)) return fail("linear_int8: null pointer or row stride below n");
  if ((x == nullptr) == (xcodes == nullptr) || (xcodes && !xscale)) return fail("linear_int8: give x or xcodes with xscale");
  if ((uintptr_t)w % 16 || (uintptr_t)xcodes % 16) return fail("linear_int8: codes have to be 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  if (x) {
    if (ldx < k) return fail("linear_int8: row stride below k");
    if (!ws || (uintptr_t)ws % 16 || ws_bytes < lic_linear_int8_workspace(m, kpad))
      return fail("linear_int8: workspace missing, misaligned or too small");
    int8_t* codes = (int8_t*)ws;
    float* scale = (float*)((char*)ws + ((int64_t)m * kpad + 15) / 16 * 16);
    if (quantize_any(dtype, x, ldx, m, k, codes, kpad, scale, s)) return 1;
    xcodes = codes;
    xscale = scale;
  }
  Int8Args a{xcodes, xscale, w, wscale, bias, r1, y, ldr1, ldy, m, n, kpad, act, slope};
  if (dtype == LIC_F32) return linear_run<float>(a, s);
  if (dtype == LIC_F16) return linear_run<half_t>(a, s);
  return linear_run<bf16_t>(a, s);
}
