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

// The largest magnitude of two running ones (NaN wins).
__device__ __forceinline__ float quant_max2(float a, float b) { return b != b ? b : (b > a ? b : a); }

// A row's power-of-two scaling and the scaled maximum; `live` is false for zero rows and NaN (codes 0).
struct QuantRow {
  float amax;
  int shift;
  bool live;
};
__device__ __forceinline__ QuantRow quant_row(float top) {
  QuantRow q{1.f, 0, top > 0.f};
  if (q.live) {
    int e;
    (void)frexpf(top, &e);
    q.shift = 1 - e;
    q.amax = ldexpf(top, q.shift);
  }
  return q;
}
__device__ __forceinline__ int quant_code(float x, const QuantRow& q) {
  return q.live ? quant_code(ldexpf(x, q.shift), q.amax) : 0;
}

template <typename T, int V> using QuantVec = T __attribute__((ext_vector_type(V)));

// G lanes a row, V elements a load; a lane keeps its part of the row in registers (NV vectors of it; longer rows are read
// a second time).  Bound by the bytes of x and codes.
template <typename T, int V, int G>
__global__ __launch_bounds__(256) void quantize_int8_kernel(const T* __restrict__ x, int64_t ldx, int m, int k,
                                                            int8_t* __restrict__ codes, int kpad,
                                                            float* __restrict__ scale) {
  constexpr int NV = V == 1 ? 8 : 4;
  typedef QuantVec<T, V> Vec;
  const int lane = threadIdx.x & (G - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (row >= m) return;
  const T* xr = x + row * ldx;
  Vec v[NV];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((lane + i * G) * V < k) v[i] = *(const Vec*)(xr + (lane + i * G) * V);
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((lane + i * G) * V < k)
#pragma unroll
      for (int e = 0; e < V; ++e) top = quant_absmax(top, to_f(v[i][e]));
  for (int j = (lane + NV * G) * V; j < k; j += G * V) {
    const Vec u = *(const Vec*)(xr + j);
#pragma unroll
    for (int e = 0; e < V; ++e) top = quant_absmax(top, to_f(u[e]));
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) top = quant_max2(top, __shfl_xor(top, o));
  if (lane == 0) scale[row] = top / 127.f;
  const QuantRow q = quant_row(top);
  typedef QuantVec<int8_t, V> Codes;
  Codes* cr = (Codes*)(codes + row * kpad);
  auto put = [&](const Vec& u, int j) {
    Codes c;
#pragma unroll
    for (int e = 0; e < V; ++e) c[e] = j < k ? (int8_t)quant_code(to_f(u[e]), q) : (int8_t)0;
    cr[j / V] = c;
  };
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((lane + i * G) * V < kpad) put(v[i], (lane + i * G) * V);
  for (int j = (lane + NV * G) * V; j < kpad; j += G * V) {
    Vec u{};
    if (j < k) u = *(const Vec*)(xr + j);
    put(u, j);
  }
}

typedef int int32x4 __attribute__((ext_vector_type(4)));
typedef int int32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void int8_lds_void;

struct Int8Args {
  const int8_t* xc;
  const float* xs;
  const int8_t* w;
  const float* ws;
  const float* bias;
  const void* r1;
  void* y;
  const void* x;
  int64_t ldr1, ldy, ldx;
  int32_t m, n, k, kpad, act;
  float slope;
  int32_t wide;   // y and r1 take 16-byte accesses at multiples of 16 columns, and the activation is not GELU
};

template <typename T>
__device__ __forceinline__ void int8_finish_one(const Int8Args& a, int64_t row, int col, float xs, int acc) {
  if (row >= a.m || col >= a.n) return;
  float u = (float)acc * (xs * a.ws[col]) + (a.bias ? a.bias[col] : 0.f);
  u = apply_act(u, a.act, a.slope);
  if (a.r1) u += to_f(((const T*)a.r1)[row * a.ldr1 + col]);
  ((T*)a.y)[row * a.ldy + col] = from_f<T>(u);
}

// N consecutive columns of one row, all inside y, aligned; not GELU.
template <typename T, int N>
__device__ __forceinline__ void int8_finish(const Int8Args& a, int64_t row, int col, float xs, const int* acc) {
  if (row >= a.m) return;
  constexpr int E = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  typedef QuantVec<T, E> Vec;
  T* y = (T*)a.y + row * a.ldy + col;
  const T* r = (const T*)a.r1 + row * a.ldr1 + col;
#pragma unroll
  for (int e = 0; e < N; e += E) {
    float v[E];
#pragma unroll
    for (int f = 0; f < E; ++f) v[f] = (float)acc[e + f] * (xs * a.ws[col + e + f]);
    if (a.bias)
#pragma unroll
      for (int f = 0; f < E; ++f) v[f] += a.bias[col + e + f];
    if (a.act == LIC_ACT_RELU) {
#pragma unroll
      for (int f = 0; f < E; ++f) v[f] = v[f] > 0.f ? v[f] : 0.f;
    } else if (a.act == LIC_ACT_LRELU) {
#pragma unroll
      for (int f = 0; f < E; ++f) v[f] = v[f] > 0.f ? v[f] : v[f] * a.slope;
    }
    if (a.r1) {
      const Vec u = *(const Vec*)(r + e);
#pragma unroll
      for (int f = 0; f < E; ++f) v[f] += to_f(u[f]);
    }
    Vec o;
#pragma unroll
    for (int f = 0; f < E; ++f) o[f] = from_f<T>(v[f]);
    *(Vec*)(y + e) = o;
  }
}

// A wave's 32 x 32 tile (lane: token lane & 31, channels 16 (lane / 32) ..): wide stores where the tile lies inside y, else
// one element at a time through the wave's 4 KB of LDS.
template <typename T>
__device__ __forceinline__ void int8_tile_out(const Int8Args& a, int64_t token, int n0, float xs, const int32x16& acc,
                                              int* stage, int lane) {
  if (a.wide && n0 + 32 <= a.n) {
    int v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = acc[e];
    int8_finish<T, 16>(a, token, n0 + 16 * (lane >> 5), xs, v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) stage[e * 64 + lane] = acc[e];
#pragma nounroll
  for (int e = 0; e < 16; ++e) int8_finish_one<T>(a, token, n0 + 16 * (lane >> 5) + e, xs, stage[e * 64 + lane]);
}

// A 32 x 32 tile of v_mfma_i32_32x32x32_i8 with weights as the first operand: lane l holds token l & 31 and result rows
// 8 (i / 4) + 4 (l / 32) + i % 4, i < 16.  Weights are placed so that these are 16 consecutive channels: operand row r is
// channel 16 ((r / 4) % 2) + 4 (r / 8) + r % 4 of the tile.
__device__ __forceinline__ int int8_channel(int r) {
  return (r & ~31) | (((r >> 2) & 1) << 4) | (((r >> 3) & 3) << 2) | (r & 3);
}

// Tiled product: BM tokens x BN channels a workgroup of WM x WN waves, 64 bytes of k a step, four steps of both operands
// in LDS, three of them in flight by LDS-DMA while one is multiplied (one barrier a step).  A row's four 16-byte chunks sit
// at chunk ^ (row / 2) % 4: eight neighbouring lanes of a fragment read cover all 64 banks.
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void int8_tile_kernel(Int8Args a, int mt, int nt) {
  constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, BK = 64, STAGES = 4;
  constexpr int ROWS = BM + BN, LOADS = ROWS / 16 / NW;   // a wave's load: 16 rows of 64 bytes
  static_assert(ROWS % (16 * NW) == 0, "rows");
  extern __shared__ __attribute__((aligned(1024))) int8_t smem[];   // [STAGES][BN weights, BM tokens][BK]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // workgroups go round the 8 XCDs: each gets a run of tiles, in groups of 8 token tiles that share their weights
  const int total = mt * nt, xcd = blockIdx.x & 7, per = total / 8, more = total & 7;
  const int id = xcd * per + min(xcd, more) + (int)(blockIdx.x >> 3);
  const int group = id / (8 * nt), in_group = id - group * 8 * nt, gm = min(8, mt - group * 8);
  const int tm = group * 8 + in_group % gm, tn = in_group / gm;
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;

  const int8_t* src[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int r = (wave * LOADS + j) * 16 + (lane >> 2);
    const int chunk = (lane & 3) ^ ((r >> 1) & 3);
    if (r < BN) src[j] = a.w + (int64_t)min(n0 + int8_channel(r), a.n - 1) * a.kpad + 16 * chunk;
    else src[j] = a.xc + min(m0 + r - BN, (int64_t)a.m - 1) * a.kpad + 16 * chunk;
  }
  auto load = [&](int s) {
    int8_t* dst = smem + (s % STAGES) * ROWS * BK + wave * LOADS * 1024;
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[j] + s * BK),
                                       (int8_lds_void*)(dst + j * 1024), 16, 0, 0);
  };
  const int wm = wave % WM, wn = wave / WM;
  const int steps = a.kpad / BK;
  int32x16 acc[TN][TM] = {};
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < steps) load(s);
  const int row = lane & 31, sw = (lane >> 1) & 3, half = lane >> 5;
  const int8_t* wbase = smem + (wn * TN * 32 + row) * BK;
  const int8_t* xbase = smem + (BN + wm * TM * 32 + row) * BK;
  for (int s = 0; s < steps; ++s) {
    // step s has landed: at most the loads of the two steps behind it are under way
    if (s + 2 < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LOADS) : "memory");
    else if (s + 1 < steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + STAGES - 1 < steps) load(s + STAGES - 1);   // over step s - 1, which every wave has left
    const int off = (s % STAGES) * ROWS * BK;
    int32x4 fw[2][TN], fx[2][TM];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int c = ((2 * kk + half) ^ sw) << 4;
#pragma unroll
      for (int i = 0; i < TN; ++i) fw[kk][i] = *(const int32x4*)(wbase + off + i * 32 * BK + c);
#pragma unroll
      for (int j = 0; j < TM; ++j) fx[kk][j] = *(const int32x4*)(xbase + off + j * 32 * BK + c);
    }
    __builtin_amdgcn_sched_barrier(0);   // all reads first: the second half's arrive under the first half's products
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int j = 0; j < TM; ++j)
#pragma unroll
        for (int i = 0; i < TN; ++i)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[kk][i], fx[kk][j], acc[i][j], 0, 0, 0);
  }
  __syncthreads();   // the steps' buffers become the waves' staging
  int* stage = (int*)smem + wave * 1024;
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int64_t token = m0 + (wm * TM + j) * 32 + row;
    const float xs = token < a.m ? a.xs[token] : 0.f;
#pragma unroll
    for (int i = 0; i < TN; ++i)
      int8_tile_out<T>(a, token, n0 + (wn * TN + i) * 32, xs, acc[i][j], stage, lane);
  }
}

// Few tokens: 16 channels x 16 TT tokens a workgroup, its 8 waves on an eighth of k each (fragments straight from memory),
// joined in LDS.  Bound by the weights' bytes, or by latency.
template <typename T, int TT>
__global__ __launch_bounds__(512) void int8_few_kernel(Int8Args a) {
  __shared__ int part[8][TT][256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * 16 * TT;
  const int steps = a.kpad / 64, s0 = steps * wave / 8, s1 = steps * (wave + 1) / 8;
  const int8_t* w = a.w + (int64_t)min(n0 + row, a.n - 1) * a.kpad + 16 * q;
  const int8_t* x[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) x[t] = a.xc + min(m0 + 16 * t + row, (int64_t)a.m - 1) * a.kpad + 16 * q;
  int32x4 acc[TT] = {};
#pragma unroll 4
  for (int s = s0; s < s1; ++s) {
    const int32x4 fw = *(const int32x4*)(w + 64 * s);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int32x4 fx = *(const int32x4*)(x[t] + 64 * s);
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw, fx, acc[t], 0, 0, 0);
    }
  }
  // lane: token row, channels 4 q .. 4 q + 3
#pragma unroll
  for (int t = 0; t < TT; ++t) *(int32x4*)&part[wave][t][row * 16 + 4 * q] = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < TT * 64; i += 512) {
    const int t = i >> 6, l = i & 63;
    int32x4 v{};
#pragma unroll
    for (int k = 0; k < 8; ++k) v += *(const int32x4*)&part[k][t][l * 4];
    const int64_t token = m0 + 16 * t + l / 4;
    const float xs = token < a.m ? a.xs[token] : 0.f;
    const int u[4] = {v[0], v[1], v[2], v[3]};
    if (a.wide && n0 + 16 <= a.n) int8_finish<T, 4>(a, token, n0 + 4 * (l & 3), xs, u);
    else
#pragma unroll
      for (int e = 0; e < 4; ++e) int8_finish_one<T>(a, token, n0 + 4 * (l & 3) + e, xs, u[e]);
  }
}

template <typename T, int V>
static void quantize_launch(const void* x, int64_t ldx, int m, int k, int8_t* codes, int kpad, float* scale,
                            hipStream_t s) {
  const int vecs = kpad / V;
  // lanes of a row: up to four vectors each, a whole wave from there on
  if (vecs <= 32) hipLaunchKernelGGL((quantize_int8_kernel<T, V, 8>), dim3((m + 31) / 32), dim3(256), 0, s, (const T*)x, ldx, m, k, codes, kpad, scale);
  else if (vecs <= 64) hipLaunchKernelGGL((quantize_int8_kernel<T, V, 16>), dim3((m + 15) / 16), dim3(256), 0, s, (const T*)x, ldx, m, k, codes, kpad, scale);
  else if (vecs <= 1024) hipLaunchKernelGGL((quantize_int8_kernel<T, V, 64>), dim3((m + 3) / 4), dim3(256), 0, s, (const T*)x, ldx, m, k, codes, kpad, scale);
  else hipLaunchKernelGGL((quantize_int8_kernel<T, V, 64>), dim3((m + 3) / 4), dim3(256), 0, s, (const T*)x, ldx, m, k, codes, kpad, scale);
}

template <typename T>
static int quantize_run(const void* x, int64_t ldx, int m, int k, int8_t* codes, int kpad, float* scale,
                        hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  auto fits = [&](int v) { return (uintptr_t)x % (v * sizeof(T)) == 0 && ldx % v == 0 && k % v == 0; };
  if (fits(V)) quantize_launch<T, V>(x, ldx, m, k, codes, kpad, scale, s);
  else if (fits(2)) quantize_launch<T, 2>(x, ldx, m, k, codes, kpad, scale, s);
  else quantize_launch<T, 1>(x, ldx, m, k, codes, kpad, scale, s);
  LIC_CHECK_LAUNCH();
  return 0;
}

static int quantize_any(int32_t dtype, const void* x, int64_t ldx, int m, int k, int8_t* codes, int kpad, float* scale,
                        hipStream_t s) {
  if (dtype == LIC_F32) return quantize_run<float>(x, ldx, m, k, codes, kpad, scale, s);
  if (dtype == LIC_F16) return quantize_run<half_t>(x, ldx, m, k, codes, kpad, scale, s);
  return quantize_run<bf16_t>(x, ldx, m, k, codes, kpad, scale, s);
}

template <typename T, int BM, int BN, int WM, int WN>
static int tile_launch(const Int8Args& a, hipStream_t s) {
  const int mt = (int)(((int64_t)a.m + BM - 1) / BM), nt = (a.n + BN - 1) / BN;
  if ((int64_t)mt * nt > INT32_MAX / 8) return fail("linear_int8: m x n out of range");
  constexpr int LDS = 4 * (BM + BN) * 64;
  const void* k = (const void*)int8_tile_kernel<T, BM, BN, WM, WN>;
  if (ensure_dyn_lds(k, LDS) != hipSuccess) return fail("linear_int8: LDS limit");
  hipLaunchKernelGGL((int8_tile_kernel<T, BM, BN, WM, WN>), dim3((unsigned)mt * nt), dim3(64 * WM * WN), LDS, s, a, mt,
                     nt);
  LIC_CHECK_LAUNCH();
  return 0;
}

template <typename T, int TT>
static int few_launch(const Int8Args& a, hipStream_t s) {
  hipLaunchKernelGGL((int8_few_kernel<T, TT>), dim3((a.n + 15) / 16, (a.m + 16 * TT - 1) / (16 * TT)), dim3(512), 0, s,
                     a);
  LIC_CHECK_LAUNCH();
  return 0;
}

template <typename T>
static int linear_run(Int8Args a, hipStream_t s) {
  const uintptr_t p = (uintptr_t)a.y | (uintptr_t)a.r1;
  constexpr int E = 16 / sizeof(T);
  a.wide = a.act != LIC_ACT_GELU && p % 16 == 0 && a.ldy % E == 0 && (!a.r1 || a.ldr1 % E == 0);
  if (a.m <= 16) return few_launch<T, 1>(a, s);
  if (a.m <= 64) return few_launch<T, 4>(a, s);
  const int64_t big = ((int64_t)a.m + 255) / 256 * ((a.n + 255) / 256);
  const int64_t mid = ((int64_t)a.m + 127) / 128 * ((a.n + 127) / 128);
  if (big >= 256) return tile_launch<T, 256, 256, 2, 4>(a, s);
  if (mid >= 256) return tile_launch<T, 128, 128, 2, 2>(a, s);
  return tile_launch<T, 64, 64, 2, 2>(a, s);
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
  Int8Args a{xcodes, xscale, w, wscale, bias, r1, y, x, ldr1, ldy, ldx, m, n, k, kpad, act, slope, 0};
  if (dtype == LIC_F32) return linear_run<float>(a, s);
  if (dtype == LIC_F16) return linear_run<half_t>(a, s);
  return linear_run<bf16_t>(a, s);
}
