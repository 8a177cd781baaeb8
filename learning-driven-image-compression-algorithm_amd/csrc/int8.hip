// Products in 8-bit integers with a scale for each token and output channel (gfx950):
//   y = act(xs[i] ws[o] sum_j X[i][j] W[o][j] + bias[o]) + r1,  X[i][j] = rint(127 x[i][j] / max_j |x[i][j]|), xs = max / 127.
// The sum is an integer of 32 bits (exact, so no form or order of it shows in a result), the rest is fp32 and is rounded
// once, to y's type.  The codes' 8 bits are the operator's definition.
#include "lic_common.h"
#include <algorithm>
#include <type_traits>

namespace lic {

template <typename T, int V> using QuantVec = T __attribute__((ext_vector_type(V)));
// at any address: wide accesses need no alignment, those that cross a line cost two (4096 x 64 -> 4097 bf16, one element at a
// time / 16 bytes: 61 / 46 us; -> 4098: 62 / 30)
template <typename T, int V> using QuantLoose = T __attribute__((ext_vector_type(V), aligned(sizeof(T))));

// A row's codes: rint(127 x / top), half to even, exactly.  The fp32 product t = x * (127 / top) is within |t| 2^-22.4 of the
// quotient.  16-bit x: a quotient that is no border k + 1/2 is at least |t| 2^-19 away from one (254 X - (2k + 1) T is a whole
// number in units of x's last place, X < 2^11), so only exact borders can be missed, and a t that near to a border is one.
// fp32 x: next to a border 254 x is compared with (2k + 1) top in two floats each, exactly.  Rows outside 2^-100 .. 2^100
// are scaled by a power of two, so nothing overflows or loses bits.
struct QuantRow {
  float top, scale, inv;   // scaled maximum, the scaling, 127 / top; inv 0: a zero row or one with a NaN or an infinity
};
__device__ __forceinline__ QuantRow quant_row(float top) {
  const float scale = top < 7.9e-31f ? 18446744073709551616.f : top > 1.2e30f ? 5.421010862427522e-20f : 1.f;
  QuantRow q{top * scale, scale, 0.f};
  if (top > 0.f) q.inv = 127.f / q.top;
  return q;
}
constexpr float QUANT_ROUND = 12582912.f;   // 1.5 * 2^23: adding it rounds, and leaves the integer in the low bits
// N codes packed four to a word (the last word's missing ones 0)
template <typename T, int N>
__device__ __forceinline__ void quant_codes(const float* x, const QuantRow& q, uint32_t* out) {
#pragma clang fp contract(off)   // every product below is a rounded one
  float t[N], r[N];
  if (q.scale == 1.f) {
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = x[e] * q.inv;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = x[e] * q.scale * q.inv;
  }
  float far = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    r[e] = t[e] + QUANT_ROUND;
    far = fmaxf(far, fabsf(t[e] - (r[e] - QUANT_ROUND)));
  }
  if (far > 0.5f - 4e-5f) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float n = r[e] - QUANT_ROUND, d = t[e] - n;
      if (fabsf(d) > 0.5f - fabsf(t[e]) * 3e-7f) {
        const float even = 2.f * rintf(0.5f * t[e]);
        if constexpr (sizeof(T) == 2) {
          r[e] = even + QUANT_ROUND;
        } else {
          const float b2 = 2.f * n + (d > 0.f ? 1.f : -1.f), xs = x[e] * q.scale;   // the border, doubled
          const float h0 = 254.f * xs, h1 = b2 * q.top;
          const float l0 = fmaf(254.f, xs, -h0), l1 = fmaf(b2, q.top, -h1);
          const float diff = (h0 - h1) + (l0 - l1);
          r[e] = (diff > 0.f ? 0.5f * (b2 + 1.f) : diff < 0.f ? 0.5f * (b2 - 1.f) : even) + QUANT_ROUND;
        }
      }
    }
  }
#pragma unroll
  for (int w = 0; w < (N + 3) / 4; ++w) {
    uint32_t b[4] = {};
#pragma unroll
    for (int e = 0; e < 4 && 4 * w + e < N; ++e) b[e] = __float_as_uint(r[4 * w + e]);
    // the low bytes of four words
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    out[w] = lo | hi;
  }
}

// Magnitudes are compared as bit patterns, where infinities and NaN are the largest (16-bit types two at a time).
template <typename T> struct QuantMax {
  typedef unsigned short Two __attribute__((ext_vector_type(2)));
  Two m{};
  template <typename Vec> __device__ __forceinline__ void add(const Vec& v) {
    constexpr int V = sizeof(Vec) / 2;
    if constexpr (V == 1) {
      const unsigned short b = __builtin_bit_cast(unsigned short, v[0]) & 0x7fff;
      m[0] = b > m[0] ? b : m[0];
    } else {
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const T two[2] = {v[e], v[e + 1]};
        m = __builtin_elementwise_max(m, __builtin_bit_cast(Two, __builtin_bit_cast(uint32_t, two) & 0x7fff7fffu));
      }
    }
  }
  __device__ __forceinline__ uint32_t bits() const { return m[0] > m[1] ? m[0] : m[1]; }
  // the magnitude; NaN for an infinity or a NaN (then also the row's scale, and its results)
  static __device__ __forceinline__ float value(uint32_t b) {
    const float f = to_f(__builtin_bit_cast(T, (unsigned short)b));
    return f < INFINITY ? f : NAN;
  }
};
template <> struct QuantMax<float> {
  uint32_t m = 0;
  template <typename Vec> __device__ __forceinline__ void add(const Vec& v) {
#pragma unroll
    for (int e = 0; e < (int)(sizeof(Vec) / 4); ++e) {
      const uint32_t b = __float_as_uint(v[e]) & 0x7fffffffu;
      m = b > m ? b : m;
    }
  }
  __device__ __forceinline__ uint32_t bits() const { return m; }
  static __device__ __forceinline__ float value(uint32_t b) { return b < 0x7f800000u ? __uint_as_float(b) : NAN; }
};

// Elements [j, j + V) of a row, V those of 16 bytes: the vector that would pass the row's end is read where it ends, and its
// codes are moved down by what it reads twice, which also leaves zeros behind k.  A row of less than one vector is gathered.
template <typename T> constexpr int QUANT_V = 16 / sizeof(T);
template <typename T>
__device__ __forceinline__ QuantVec<T, QUANT_V<T>> quant_load(const T* x, int j, int k) {
  constexpr int V = QUANT_V<T>;
  typedef QuantVec<T, V> Vec;
  if (j >= k) return Vec{};
  if (k >= V) return *(const QuantLoose<T, V>*)(x + (j + V <= k ? j : k - V));
  typedef std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t> Bits;
  unsigned __int128 w = 0;
#pragma nounroll
  for (int e = k - 1; e >= 0; --e) w = w << 8 * sizeof(T) | __builtin_bit_cast(Bits, x[e]);
  return __builtin_bit_cast(Vec, w);
}
template <typename T>
__device__ __forceinline__ void quant_put(int8_t* to, const QuantVec<T, QUANT_V<T>>& u, int j, int k, const QuantRow& q) {
  constexpr int V = QUANT_V<T>;
  float f[V];
  uint32_t w[V / 4] = {};
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = to_f(u[e]);
  if (q.inv != 0.f) quant_codes<T, V>(f, q, w);
  const int twice = k >= V && j < k && j + V > k ? 8 * (j + V - k) : 0;
  if constexpr (V == 8) *(uint64_t*)to = (w[0] | (uint64_t)w[1] << 32) >> twice;
  else *(uint32_t*)to = w[0] >> twice;
}

// G lanes a row; a lane keeps its part of the row in registers (NV vectors of it; longer rows are read
// a second time).  Bound by the bytes of x and codes: 8192 x 4096 bf16 21.5 us, 4.7 TB/s; 8192 x 4095
// 22.6 (elements one by one: 49); 1037 x 333 fp32 2.9 us.
template <typename T, int G>
__global__ __launch_bounds__(256) void quantize_int8_kernel(const T* __restrict__ x, int64_t ldx, int m, int k,
                                                            int8_t* __restrict__ codes, int kpad,
                                                            float* __restrict__ scale) {
  constexpr int V = QUANT_V<T>;
  constexpr int NV = 4;
  const int lane = threadIdx.x & (G - 1);
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * (256 / G) + threadIdx.x / G;
  if (row >= m) return;
  const T* xr = x + row * ldx;
  QuantVec<T, V> v[NV];
  QuantMax<T> most;
#pragma unroll
  for (int i = 0; i < NV; ++i) v[i] = quant_load<T>(xr, (lane + i * G) * V, k);
#pragma unroll
  for (int i = 0; i < NV; ++i) most.add(v[i]);
  for (int j = (lane + NV * G) * V; j < k; j += G * V) most.add(quant_load<T>(xr, j, k));
  uint32_t bits = most.bits();
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor(bits, o);
    bits = other > bits ? other : bits;
  }
  const float top = QuantMax<T>::value(bits);
  if (lane == 0) scale[row] = top / 127.f;
  const QuantRow q = quant_row(top);
  int8_t* cr = codes + row * kpad;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = (lane + i * G) * V;
    if (j < kpad) quant_put<T>(cr + j, v[i], j, k, q);   // columns behind k: zeros
  }
  for (int j = (lane + NV * G) * V; j < kpad; j += G * V) quant_put<T>(cr + j, quant_load<T>(xr, j, k), j, k, q);
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
  int32_t wide;   // not GELU, whose many instructions would stand at every store
};

template <typename T>
__device__ __forceinline__ void int8_finish_one(const Int8Args& a, int64_t row, int col, float xs, int acc) {
  if (row >= a.m || col >= a.n) return;
  float u = (float)acc * (xs * a.ws[col]) + (a.bias ? a.bias[col] : 0.f);
  u = apply_act(u, a.act, a.slope);
  if (a.r1) u += to_f(((const T*)a.r1)[row * a.ldr1 + col]);
  ((T*)a.y)[row * a.ldy + col] = from_f<T>(u);
}

// N consecutive columns of one row, all inside y (at any alignment); not GELU.  ws, bias (or nullptr): those columns' own.
template <typename T, int N>
struct Int8Out {
  static constexpr int E = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  typedef QuantVec<T, E> Vec;
  typedef QuantLoose<T, E> Loose;
  Vec o[N / E];
  __device__ __forceinline__ void compute(const Int8Args& a, int64_t row, int col, float xs, const int* acc,
                                          const float* ws, const float* bias) {
    float v[N];
    floatx4 b[N / 4] = {};
    if (bias)
#pragma unroll
      for (int e = 0; e < N / 4; ++e) b[e] = *(const QuantLoose<float, 4>*)(bias + 4 * e);
#pragma unroll
    for (int e = 0; e < N / 4; ++e) {
      const floatx4 w = *(const QuantLoose<float, 4>*)(ws + 4 * e);
#pragma unroll
      for (int f = 0; f < 4; ++f) v[4 * e + f] = (float)acc[4 * e + f] * (xs * w[f]) + b[e][f];
    }
    if (a.act != LIC_ACT_NONE) {
      const bool relu = a.act == LIC_ACT_RELU;
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = v[e] > 0.f ? v[e] : (relu ? 0.f : v[e] * a.slope);
    }
    if (a.r1) {
      const Loose* r = (const Loose*)((const T*)a.r1 + (row < a.m ? row : 0) * a.ldr1 + col);
#pragma unroll
      for (int e = 0; e < N / E; ++e) {
        const Vec u = r[e];
#pragma unroll
        for (int f = 0; f < E; ++f) v[E * e + f] += to_f(u[f]);
      }
    }
#pragma unroll
    for (int e = 0; e < N / E; ++e) o[e] = __builtin_convertvector(*(QuantVec<float, E>*)(v + E * e), Vec);
  }
  __device__ __forceinline__ void store(const Int8Args& a, int64_t row, int col) const {
    if (row >= a.m) return;
    T* y = (T*)a.y + row * a.ldy + col;
#pragma unroll
    for (int e = 0; e < N / E; ++e) *(Loose*)(y + e * E) = o[e];
  }
};

// A wave's 32 x 32 tile (lane: token m0 + lane % 32 with scale xs, channels n0 + 16 (lane / 32) ..): wide stores, one by one
// where y's columns end inside a lane's; GELU is turned in the wave's LDS (INT8_STAGE words), so that its code stands once and
// 32 lanes meet consecutive channels (so turned, the last columns cost 1 to 2 us more: 64 x 256 -> 1000 7.2 us for 6.1).
constexpr int INT8_STAGE = 32 * 33;
template <typename T>
__device__ __forceinline__ void int8_tile_out(const Int8Args& a, int64_t m0, int n0, float xs, const int32x16& acc,
                                              int* stage, int lane) {
  const int row = lane & 31, half = lane >> 5;
  if (m0 >= a.m || n0 >= a.n) return;
  if (a.wide) {
    const int col = n0 + 16 * half;
    const int64_t token = m0 + row;
    if (col + 16 <= a.n) {
      int v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = acc[e];
      Int8Out<T, 16> out;
      out.compute(a, token, col, xs, v, a.ws + col, a.bias ? a.bias + col : nullptr);
      out.store(a, token, col);
    } else {
      const T* r1 = (const T*)a.r1 + (token < a.m ? token : 0) * a.ldr1;
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int at = min(col + e, a.n - 1);
        v[e] = (float)acc[e] * (xs * a.ws[at]) + (a.bias ? a.bias[at] : 0.f);
        if (a.act != LIC_ACT_NONE) v[e] = v[e] > 0.f ? v[e] : (a.act == LIC_ACT_RELU ? 0.f : v[e] * a.slope);
        if (a.r1) v[e] += to_f(r1[at]);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (token < a.m && col + e < a.n) ((T*)a.y)[token * a.ldy + col + e] = from_f<T>(v[e]);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) stage[row * 33 + 16 * half + e] = acc[e];
  wave_lds_sync();
  const int col = n0 + row, at = min(col, a.n - 1);
  const float ws = a.ws[at], bias = a.bias ? a.bias[at] : 0.f;
#pragma unroll 2
  for (int e = 0; e < 32; e += 2) {
    const int64_t token = m0 + e + half;
    const float s = __shfl(xs, e + half);
    if (token < a.m && col < a.n) {
      float u = (float)stage[(e + half) * 33 + row] * (s * ws) + bias;
      u = apply_act(u, a.act, a.slope);
      if (a.r1) u += to_f(((const T*)a.r1)[token * a.ldr1 + col]);
      ((T*)a.y)[token * a.ldy + col] = from_f<T>(u);
    }
  }
  wave_lds_sync();
}

// A 32 x 32 tile of v_mfma_i32_32x32x32_i8 with weights as the first operand: lane l holds token l & 31 and result rows
// 8 (i / 4) + 4 (l / 32) + i % 4, i < 16.  Weights are placed so that these are 16 consecutive channels: operand row r is
// channel 16 ((r / 4) % 2) + 4 (r / 8) + r % 4 of the tile.
__device__ __forceinline__ int int8_channel(int r) {
  return (r & ~31) | (((r >> 2) & 1) << 4) | (((r >> 3) & 3) << 2) | (r & 3);
}

// Tiled product: BM tokens x BN channels a workgroup of WM x WN waves, 64 bytes of k a step, four steps of both operands
// in LDS, three of them in flight by LDS-DMA while one is multiplied (one barrier a step).  A row's four 16-byte chunks sit
// at chunk ^ (row / 2) % 4: eight neighbouring lanes of a fragment read cover all 64 banks.  Bound by the matrix
// instructions: 8192 x 4096 -> 8192 282 us, 1.95 POP/s, on the same operands again and again, 300 to 318 on new ones (a large
// library product reaches 2.06); small ones by the latency of their k steps, which KG groups of waves take a part of each and
// join in LDS: 128 x 4096 -> 4096 12.9 us with one, 9.9 with two; 1037 x 333 -> 517 fp32 5.3 us.  More than four steps in flight
// gain nothing (128 x 4096 -> 4096 13.5 us with eight).
template <typename T, int BM, int BN, int WM, int WN, int KG>
__global__ __launch_bounds__(64 * WM * WN * KG) void int8_tile_kernel(Int8Args a, int mt, int nt) {
  constexpr int NW = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32, BK = 64, STAGES = 4;
  static_assert(KG == 1 || TM * TN == 1, "groups join one tile a wave");
  constexpr int ROWS = BM + BN, LOADS = ROWS / 16 / NW;   // a wave's load: 16 rows of 64 bytes
  static_assert(ROWS % (16 * NW) == 0, "rows");
  extern __shared__ __attribute__((aligned(1024))) int8_t lds[];   // [KG][STAGES][BN weights, BM tokens][BK]
  const int lane = threadIdx.x & 63, id8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = id8 % NW, kg = id8 / NW;
  int8_t* smem = lds + kg * STAGES * ROWS * BK;
  // workgroups go round the 8 XCDs: each gets a run of tiles, in groups of 8 token tiles that share their weights
  const int total = mt * nt, xcd = blockIdx.x & 7, per = total / 8, more = total & 7;
  const int id = xcd * per + min(xcd, more) + (int)(blockIdx.x >> 3);
  const int group = id / (8 * nt), in_group = id - group * 8 * nt, gm = min(8, mt - group * 8);
  const int tm = group * 8 + in_group % gm, tn = in_group / gm;
  const int64_t m0 = (int64_t)tm * BM;
  const int n0 = tn * BN;

  // a group's steps of k; all of them meet at `most` barriers
  const int whole = a.kpad / BK, s0 = whole * kg / KG, steps = whole * (kg + 1) / KG - s0, most = (whole + KG - 1) / KG;
  const int8_t* src[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int r = (wave * LOADS + j) * 16 + (lane >> 2);
    const int chunk = (lane & 3) ^ ((r >> 1) & 3);
    if (r < BN) src[j] = a.w + (int64_t)min(n0 + int8_channel(r), a.n - 1) * a.kpad + 16 * chunk + s0 * BK;
    else src[j] = a.xc + min(m0 + r - BN, (int64_t)a.m - 1) * a.kpad + 16 * chunk + s0 * BK;
  }
  auto load = [&](int s) {
    int8_t* dst = smem + (s % STAGES) * ROWS * BK + wave * LOADS * 1024;
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src[j] + s * BK),
                                       (int8_lds_void*)(dst + j * 1024), 16, 0, 0);
  };
  const int wm = wave % WM, wn = wave / WM;
  int32x16 acc[TN][TM] = {};
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s)
    if (s < steps) load(s);
  const int row = lane & 31, sw = (lane >> 1) & 3, half = lane >> 5;
  const int8_t* wbase = smem + (wn * TN * 32 + row) * BK;
  const int8_t* xbase = smem + (BN + wm * TM * 32 + row) * BK;
  int32x4 fw[2][TN], fx[2][TM];   // the fragments of a step's two halves
  auto read = [&](int s, int kk) {
    const int off = (s % STAGES) * ROWS * BK, c = ((2 * kk + half) ^ sw) << 4;
#pragma unroll
    for (int i = 0; i < TN; ++i) fw[kk][i] = *(const int32x4*)(wbase + off + i * 32 * BK + c);
#pragma unroll
    for (int j = 0; j < TM; ++j) fx[kk][j] = *(const int32x4*)(xbase + off + j * 32 * BK + c);
  };
  auto multiply = [&](int kk, int j0, int j1) {
#pragma unroll
    for (int j = j0; j < j1; ++j)
#pragma unroll
      for (int i = 0; i < TN; ++i)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[kk][i], fx[kk][j], acc[i][j], 0, 0, 0);
  };
  // waits until step s has landed for every wave (behind it at most the loads of two more steps are under way), and until
  // every wave has what it read so far, so that the step before may be overwritten
  auto landed = [&](int s) {
    if (s + 2 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * LOADS) : "memory");
    else if (s + 1 < steps) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  landed(0);
  if (STAGES - 1 < steps) load(STAGES - 1);
  read(0, 0);
  for (int s = 0; s < steps; ++s) {
    // each half's fragments are read under the other half's products (after the first of them, whose wait for its own
    // fragments would else be one for both); the barrier stands between the halves
    multiply(0, 0, 1);
    __builtin_amdgcn_sched_barrier(0);
    read(s, 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(0, 1, TM);
    __builtin_amdgcn_sched_barrier(0);
    if (s + 1 < most) {
      landed(s + 1);
      if (s + STAGES < steps) load(s + STAGES);
      if (KG == 1 || s + 1 < steps) read(s + 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    multiply(1, 0, TM);
    __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();   // the steps' buffers become the waves' staging
  int* stage = (int*)lds + wave * INT8_STAGE;
  if constexpr (KG > 1) {
    int* join = (int*)lds + NW * INT8_STAGE + wave * 1024 + lane;   // [KG - 1][NW][16][64]
    if (kg) {
#pragma unroll
      for (int e = 0; e < 16; ++e) join[(kg - 1) * NW * 1024 + e * 64] = acc[0][0][e];
    }
    __syncthreads();
    if (kg) return;
#pragma unroll
    for (int g = 0; g < KG - 1; ++g)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[0][0][e] += join[g * NW * 1024 + e * 64];
  }
#pragma unroll
  for (int j = 0; j < TM; ++j) {
    const int64_t token = m0 + (wm * TM + j) * 32 + row;
    const float xs = token < a.m ? a.xs[token] : 0.f;
#pragma unroll
    for (int i = 0; i < TN; ++i)
      int8_tile_out<T>(a, m0 + (wm * TM + j) * 32, n0 + (wn * TN + i) * 32, xs, acc[i][j], stage, lane);
  }
}

// Joins the eighths of k that the waves of the two kernels below computed (lane: token lane % 16, channels 4 (lane / 16) ..)
// and writes 16 channels x 16 TT tokens.
template <typename T, int TT>
__device__ __forceinline__ void int8_join(const Int8Args& a, int (*part)[TT][256], const int32x4* acc, int n0, int64_t m0,
                                          const float* xscale) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int t = 0; t < TT; ++t) *(int32x4*)&part[wave][t][(lane & 15) * 16 + 4 * (lane >> 4)] = acc[t];
  __syncthreads();
  for (int i = threadIdx.x; i < TT * 64; i += 512) {
    const int t = i >> 6, l = i & 63;
    int32x4 v{};
#pragma unroll
    for (int k = 0; k < 8; ++k) v += *(const int32x4*)&part[k][t][l * 4];
    const int64_t token = m0 + 16 * t + l / 4;
    if (token >= a.m) continue;
    const float xs = xscale[token];
    const int u[4] = {v[0], v[1], v[2], v[3]};
    const int col = n0 + 4 * (l & 3);
    if (a.wide && n0 + 16 <= a.n) {
      Int8Out<T, 4> out;
      out.compute(a, token, col, xs, u, a.ws + col, a.bias ? a.bias + col : nullptr);
      out.store(a, token, col);
    } else {
#pragma nounroll
      for (int e = 0; e < 4; ++e) int8_finish_one<T>(a, token, col + e, xs, v[e]);
    }
  }
}

// Few tokens: 16 channels x 16 TT tokens a workgroup, its 8 waves on an eighth of k each, fragments straight from memory.
// Bound by the weights' bytes, or by latency: 16 x 4096 -> 4096 6.5 us (2.6 TB/s), 16 x 192 -> 576 5.4 us.
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
  int s = s0;
  for (; s + 4 <= s1; s += 4) {   // four steps' loads under way at once
    int32x4 fw[4], fx[4][TT];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      fw[u] = *(const int32x4*)(w + 64 * (s + u));
#pragma unroll
      for (int t = 0; t < TT; ++t) fx[u][t] = *(const int32x4*)(x[t] + 64 * (s + u));
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u], fx[u][t], acc[t], 0, 0, 0);
  }
  for (; s < s1; ++s) {
    const int32x4 fw = *(const int32x4*)(w + 64 * s);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const int32x4 fx = *(const int32x4*)(x[t] + 64 * s);
      acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw, fx, acc[t], 0, 0, 0);
    }
  }
  int8_join<T, TT>(a, part, acc, n0, m0, a.xs);
}

// One to ONE_TOKENS tokens of up to ONE_K channels in one launch: every workgroup quantises them into LDS, its first weights
// already under way.  Bound by latency, then the weights' bytes: 1 x 4096 -> 4096 7.5 to 8 us (quantised apart: 5.6 + 5.4).
constexpr int ONE_TOKENS = 4, ONE_K = 4096;
template <typename T>
__global__ __launch_bounds__(512) void int8_one_kernel(Int8Args a) {
  constexpr int V = QUANT_V<T>, VECS = ONE_K / 512 / V;   // a thread's part of a row
  __shared__ int part[8][1][256];
  __shared__ uint32_t most[ONE_TOKENS][8];
  __shared__ float scale[ONE_TOKENS];
  extern __shared__ __attribute__((aligned(16))) int8_t codes[];   // [m][kpad]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int steps = a.kpad / 64, s0 = steps * wave / 8, s1 = steps * (wave + 1) / 8;
  const int8_t* w = a.w + (int64_t)min(n0 + row, a.n - 1) * a.kpad + 16 * q;
  static_assert(ONE_K <= 8 * 8 * 64, "a wave's steps of k are held at once");
  int32x4 fw[8];
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (s0 + u < s1) fw[u] = *(const int32x4*)(w + 64 * (s0 + u));
  QuantVec<T, V> v[ONE_TOKENS][VECS];
#pragma unroll
  for (int r = 0; r < ONE_TOKENS; ++r) {
    if (r >= a.m) break;
    QuantMax<T> top;
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      v[r][i] = quant_load<T>((const T*)a.x + r * a.ldx, (threadIdx.x + 512 * i) * V, a.k);
      top.add(v[r][i]);
    }
    uint32_t bits = top.bits();
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint32_t other = __shfl_xor(bits, o);
      bits = other > bits ? other : bits;
    }
    if (lane == 0) most[r][wave] = bits;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ONE_TOKENS; ++r) {
    if (r >= a.m) break;
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) bits = most[r][i] > bits ? most[r][i] : bits;
    const float top = QuantMax<T>::value(bits);
    if (threadIdx.x == 0) scale[r] = top / 127.f;
    const QuantRow qr = quant_row(top);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int j = (threadIdx.x + 512 * i) * V;
      if (j < a.kpad) quant_put<T>(codes + r * a.kpad + j, v[r][i], j, a.k, qr);
    }
  }
  __syncthreads();
  const int8_t* x = codes + min(row, a.m - 1) * a.kpad + 16 * q;
  int32x4 acc[1] = {};
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (s0 + u < s1)
      acc[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u], *(const int32x4*)(x + 64 * (s0 + u)), acc[0], 0, 0, 0);
  int8_join<T, 1>(a, part, acc, n0, 0, scale);
}

// Few tiles of up to FUSED_K channels in one launch: 32 tokens x 128 channels a workgroup.  Its weights are all asked for at
// once (LDS-DMA), and while they come its tokens are quantised into LDS, sixteen lanes a token; then its 8 waves multiply, four
// tiles of 32 x 32 in two halves of k that are joined in LDS.  Each of a token's tiles quantises it again.  us (two launches):
// 64 x 192 -> 576 fp16 4.6 (5.5), 1037 x 333 -> 517 fp32 8.1 (8.4; 9.2 with an activation and a shortcut), 2500 x 192 -> 576 (395
// tiles) 6.3 (7.8), fp32 8.0 (9.3), 2000 x 384 -> 1000 fp32 (504) 12.7 (11.8), 4096 x 192 -> 576 (640) 7.9 (8.4), fp32 10.5
// (10.8); and a call, a workspace less.
constexpr int FUSED_K = 384, FUSED_M = 32, FUSED_N = 128, FUSED_TILES = 512;
constexpr int FUSED_SUMS = 4 * (4096 + 4 * INT8_STAGE);   // four tiles of sums, then four waves' staging
template <typename T>
__global__ __launch_bounds__(512) void int8_fused_kernel(Int8Args a) {
  constexpr int V = QUANT_V<T>, VECS = FUSED_K / 16 / V;
  __shared__ float scale[FUSED_M];
  extern __shared__ __attribute__((aligned(1024))) int8_t smem[];   // [FUSED_N weights, FUSED_M tokens][kpad], then the sums
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m0 = (int64_t)blockIdx.y * FUSED_M;
  const int n0 = blockIdx.x * FUSED_N, chunks = a.kpad / 16, ks = a.kpad / 64;
  // where a row's 16-byte chunks are placed: a fragment read meets every bank once (rows advance by 16 ks of the 64 words)
  const int shift = ks % 4 == 0 ? 0 : ks % 2 == 0 ? 1 : 2, mask = ks % 4 == 0 ? 15 : ks % 2 == 0 ? 7 : 3;
  auto place = [&](int r, int c) { return c ^ ((r >> shift) & mask); };
  const uint32_t inv = (1u << 22) / chunks + 1;   // g / chunks = g inv >> 22 for g < 4096, chunks from 4 to 64
  for (int i = wave; i < FUSED_N / 64 * chunks; i += 8) {
    const int g = i * 64 + lane, r = (int)((uint32_t)g * inv >> 22), p = g - r * chunks;
    const int64_t ch = min(n0 + int8_channel(r), a.n - 1);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(a.w + ch * a.kpad + 16 * place(r, p)),
                                     (int8_lds_void*)(smem + i * 1024), 16, 0, 0);
  }
  const int r = threadIdx.x >> 4, l = threadIdx.x & 15;
  const T* x = (const T*)a.x + min(m0 + r, (int64_t)a.m - 1) * a.ldx;
  QuantVec<T, V> v[VECS];
  QuantMax<T> most;
#pragma unroll
  for (int i = 0; i < VECS; ++i) v[i] = quant_load<T>(x, (l + 16 * i) * V, a.k);
#pragma unroll
  for (int i = 0; i < VECS; ++i) most.add(v[i]);
  uint32_t bits = most.bits();
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor(bits, o);
    bits = other > bits ? other : bits;
  }
  const float top = QuantMax<T>::value(bits);
  if (l == 0) scale[r] = top / 127.f;
  const QuantRow q = quant_row(top);
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int j = (l + 16 * i) * V;
    if (j < a.kpad) quant_put<T>(smem + (FUSED_N + r) * a.kpad + 16 * place(r, j / 16) + j % 16, v[i], j, a.k, q);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  const int row = lane & 31, half = lane >> 5, wn = wave & 3, part = wave >> 2;
  const int8_t *wrow = smem + (wn * 32 + row) * a.kpad, *xrow = smem + (FUSED_N + row) * a.kpad;
  int32x16 acc{};
  for (int s = part; s < 2 * ks; s += 2) {
    const int c = 16 * place(row, 2 * s + half);   // the same for rows 32 apart
    acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*(const int32x4*)(wrow + c), *(const int32x4*)(xrow + c), acc, 0, 0, 0);
  }
  __syncthreads();   // the operands become sums and staging
  int* join = (int*)smem + (wave & 3) * 1024 + lane;
  if (part) {
#pragma unroll
    for (int e = 0; e < 16; ++e) join[e * 64] = acc[e];
  }
  __syncthreads();
  if (part) return;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] += join[e * 64];
  int8_tile_out<T>(a, m0, n0 + wn * 32, scale[row], acc, (int*)smem + 4096 + wave * INT8_STAGE, lane);
}

// Many tokens of few channels (kpad = 64 KS; whole tiles of y only: n a multiple of 32, aligned): 32 tokens a wave, quantised
// straight into matrix operands that stay in registers; the weights pass through LDS, 64 channels at a time, the next under
// way.  x is read once and y written once, the codes never reach memory.  Bound by the bytes of y: 131072 x 192 -> 576 fp16
// 42 to 48 us alone, 55 with the call (201 MB; 35 without its stores).  A weight row's 16-byte chunks are placed so that a fragment
// read meets every bank once: rows advance by 16 KS of the 64 words, so chunk ^ swizzle(row) within 4, 8 or 16 chunks spreads
// those that coincide.
template <int KS>
__device__ __forceinline__ int int8_rows_swizzle(int r) {
  return KS % 4 == 0 ? r & 15 : KS % 2 == 0 ? (r >> 1) & 7 : (r >> 2) & 3;
}

// waves a SIMD that the registers and the LDS of a form allow
template <typename T, int KS> constexpr int ROWS_WAVES = sizeof(T) == 2 ? (KS <= 3 ? 4 : 3) : (KS == 1 ? 4 : KS <= 3 ? 3 : 2);
template <typename T, int KS>
__global__ __launch_bounds__(256, (ROWS_WAVES<T, KS>)) void int8_rows_kernel(Int8Args a) {
  constexpr int CK = 2 * KS, KP = 64 * KS, V = 16 / sizeof(T), L = 16 / V;   // products of 32 k; loads of 16 elements
  constexpr bool HOLD = CK * 16 * sizeof(T) <= 256;                          // a lane's half row fits 64 registers
  typedef QuantVec<T, V> Vec;
  __shared__ __attribute__((aligned(1024))) int8_t smem[2][64 * KP];
  __shared__ __attribute__((aligned(16))) float cols[2][2][64];   // the chunk's scales and biases
  constexpr int LINE = 64 * sizeof(T) + 16;                       // a token's results of a chunk (fp32)
  __shared__ __attribute__((aligned(16))) char stage[4][sizeof(T) == 2 ? 16 : 32 * LINE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 31, half = lane >> 5;
  const int64_t token = (int64_t)blockIdx.x * 128 + wave * 32 + row;
  // the workgroup's share of the 64-channel chunks
  const int all = (a.n + 63) / 64, first = all * blockIdx.y / gridDim.y, chunks = all * (blockIdx.y + 1) / gridDim.y;

  auto load = [&](int c) {
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      const int g = (wave * KS + j) * 64 + lane, r = g / (4 * KS), p = g % (4 * KS);
      const int64_t ch = min(64 * c + int8_channel(r), a.n - 1);
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void*)(a.w + ch * KP + 16 * (p ^ int8_rows_swizzle<KS>(r))),
          (int8_lds_void*)(smem[c & 1] + (wave * KS + j) * 1024), 16, 0, 0);
    }
    const float* col = wave == 0 ? a.ws : wave == 1 ? a.bias : nullptr;
    if (col)
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(col + min(64 * c + lane, a.n - 1)),
                                       (int8_lds_void*)cols[c & 1][wave], 4, 0, 0);
  };
  load(first);
  if (!a.bias && threadIdx.x < 128) cols[threadIdx.x >> 6][1][lane] = 0.f;

  const T* x = (const T*)a.x + min(token, (int64_t)a.m - 1) * a.ldx + 16 * half;
  Vec raw[HOLD ? CK : 1][L];
  QuantMax<T> most;
  auto fetch = [&](int ks, Vec* u) {
#pragma unroll
    for (int l = 0; l < L; ++l) {
      u[l] = Vec{};
      if (32 * ks + 16 * half + V * l < a.k) u[l] = *(const Vec*)(x + 32 * ks + V * l);
    }
  };
  if constexpr (HOLD) {
#pragma unroll
    for (int ks = 0; ks < CK; ++ks) fetch(ks, raw[ks]);
  }
#pragma unroll
  for (int ks = 0; ks < CK; ++ks) {
    Vec* u = raw[HOLD ? ks : 0];
    if constexpr (!HOLD) fetch(ks, u);
#pragma unroll
    for (int l = 0; l < L; ++l) most.add(u[l]);
  }
  const uint32_t bits = most.bits(), other = __shfl_xor(bits, 32);
  const float top = QuantMax<T>::value(other > bits ? other : bits);
  const float xs = top / 127.f;
  const QuantRow q = quant_row(top);
  int32x4 fx[CK];
#pragma unroll
  for (int ks = 0; ks < CK; ++ks) {
    Vec* u = raw[HOLD ? ks : 0];
    if constexpr (!HOLD) fetch(ks, u);
    float f[16];
    uint32_t w[4] = {};
#pragma unroll
    for (int e = 0; e < 16; ++e) f[e] = to_f(u[e / V][e % V]);
    if (q.inv != 0.f) quant_codes<T, 16>(f, q, w);
    fx[ks] = int32x4{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
  }

  const int sw = int8_rows_swizzle<KS>(row);   // the same for both tiles: 32 rows apart
  auto landed = [] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  landed();
  if (first + 1 < chunks) load(first + 1);
  for (int c = first; c < chunks; ++c) {
    Int8Out<T, 16> out[2] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int32x16 acc{};
#pragma unroll
      for (int ks = 0; ks < CK; ++ks) {
        const int32x4 fw = *(const int32x4*)(smem[c & 1] + (32 * i + row) * KP + 16 * ((2 * ks + half) ^ sw));
        acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw, fx[ks], acc, 0, 0, 0);
      }
      const int at = 32 * i + 16 * half;
      int v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = acc[e];
      if (64 * c + 32 * i < a.n) out[i].compute(a, token, 64 * c + at, xs, v, cols[c & 1][0] + at, cols[c & 1][1] + at);
    }
    // chunk c + 1 has landed and chunk c been read by every wave; this chunk's stores come after the wait, so that they
    // have a whole chunk's time until the next
    landed();
    if (c + 2 < chunks) load(c + 2);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (64 * c + 32 * i < a.n) out[i].store(a, token, 64 * c + 32 * i + 16 * half);
    } else {
      // 64 bytes a lane would be four stores of a line's eighth each: through the wave's LDS, a store covers two lines of
      // each of its tokens (131072 x 192 -> 576: 134.8 -> 94.9 us; 16-bit results gain nothing by it, 54.4 / 56.1)
      char* st = stage[wave];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 16 / V; ++e) *(Vec*)(st + row * LINE + (32 * i + 16 * half + V * e) * sizeof(T)) = out[i].o[e];
      wave_lds_sync();
      Vec u[32 / V];
#pragma unroll
      for (int e = 0; e < 32 / V; ++e)
        u[e] = *(const Vec*)(st + (e * 64 + lane) / (64 / V) * LINE + (e * 64 + lane) % (64 / V) * 16);
#pragma unroll
      for (int e = 0; e < 32 / V; ++e) {
        const int col = (e * 64 + lane) % (64 / V) * V;
        const int64_t to = token - row + (e * 64 + lane) / (64 / V);
        if (to < a.m && 64 * c + col < a.n) *(Vec*)((T*)a.y + to * a.ldy + 64 * c + col) = u[e];
      }
    }
  }
}

constexpr int ROWS_FILL = 512;   // workgroups; 32768 x 192 -> 576 fp16: 28.0 us with 256, 23.5 with 512, 24.8 with 1024
template <typename T, int KS>
static int rows_launch(const Int8Args& a, hipStream_t s) {
  // channels are shared out where the token blocks alone would not fill the chip (each share quantises its tokens again)
  const int blocks = (int)(((int64_t)a.m + 127) / 128), chunks = (a.n + 63) / 64;
  const int fill = (ROWS_FILL + blocks - 1) / blocks, shares = fill < chunks ? fill : chunks;
  hipLaunchKernelGGL((int8_rows_kernel<T, KS>), dim3((unsigned)blocks, (unsigned)shares), dim3(256), 0, s, a);
  LIC_CHECK_LAUNCH();
  return 0;
}

template <typename T>
static int rows_run(const Int8Args& a, hipStream_t s) {
  switch (a.kpad / 64) {
    case 1: return rows_launch<T, 1>(a, s);
    case 2: return rows_launch<T, 2>(a, s);
    case 3: return rows_launch<T, 3>(a, s);
    case 4: return rows_launch<T, 4>(a, s);
    case 5: return rows_launch<T, 5>(a, s);
    case 6: return rows_launch<T, 6>(a, s);
    default: return fail("linear_int8: rows kernel sizes");
  }
}

// Rows of few vectors share a wave only where there are many: 1000 x 500 bf16 2.7 us with a wave a row, 3.5 with four rows a
// wave; 131072 x 192 14.7 us with eight.
constexpr int QUANT_FEW = 2048;
template <typename T>
static int quantize_run(const void* x, int64_t ldx, int m, int k, int8_t* codes, int kpad, float* scale,
                        hipStream_t s) {
  const int vecs = kpad / QUANT_V<T>;
  auto launch = [&](auto kernel, int rows) {
    // a dimension of a launch has less than 2^32 threads
    const int64_t blocks = ((int64_t)m + rows - 1) / rows, bx = std::min<int64_t>(blocks, 1 << 22);
    hipLaunchKernelGGL(kernel, dim3((unsigned)bx, (unsigned)((blocks + bx - 1) / bx)), dim3(256), 0, s, (const T*)x, ldx, m,
                       k, codes, kpad, scale);
  };
  if (vecs <= 32 && m > QUANT_FEW) launch(quantize_int8_kernel<T, 8>, 32);
  else if (vecs <= 64 && m > QUANT_FEW) launch(quantize_int8_kernel<T, 16>, 16);
  else launch(quantize_int8_kernel<T, 64>, 4);
  LIC_CHECK_LAUNCH();
  return 0;
}

static int quantize_any(int32_t dtype, const void* x, int64_t ldx, int m, int k, int8_t* codes, int kpad, float* scale,
                        hipStream_t s) {
  if (dtype == LIC_F32) return quantize_run<float>(x, ldx, m, k, codes, kpad, scale, s);
  if (dtype == LIC_F16) return quantize_run<half_t>(x, ldx, m, k, codes, kpad, scale, s);
  return quantize_run<bf16_t>(x, ldx, m, k, codes, kpad, scale, s);
}

template <typename T, int BM, int BN, int WM, int WN, int KG>
static int tile_launch(const Int8Args& a, hipStream_t s) {
  const int mt = (int)(((int64_t)a.m + BM - 1) / BM), nt = (a.n + BN - 1) / BN;
  constexpr int LDS = KG * 4 * (BM + BN) * 64;
  const void* k = (const void*)int8_tile_kernel<T, BM, BN, WM, WN, KG>;
  if (ensure_dyn_lds(k, LDS) != hipSuccess) return fail("linear_int8: LDS limit");
  hipLaunchKernelGGL((int8_tile_kernel<T, BM, BN, WM, WN, KG>), dim3((unsigned)mt * nt), dim3(64 * WM * WN * KG), LDS, s, a, mt,
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

static bool int8_fused(int64_t m, int32_t kpad, int64_t n) {
  return kpad <= FUSED_K && (m + FUSED_M - 1) / FUSED_M * ((n + FUSED_N - 1) / FUSED_N) <= FUSED_TILES;
}
template <typename T>
static int fused_launch(const Int8Args& a, hipStream_t s) {
  const int lds = std::max((FUSED_M + FUSED_N) * a.kpad, FUSED_SUMS);   // below 64 KB
  const dim3 tiles((a.n + FUSED_N - 1) / FUSED_N, (a.m + FUSED_M - 1) / FUSED_M);
  hipLaunchKernelGGL(int8_fused_kernel<T>, tiles, dim3(512), lds, s, a);
  LIC_CHECK_LAUNCH();
  return 0;
}

template <typename T>
static int one_launch(const Int8Args& a, hipStream_t s) {
  hipLaunchKernelGGL(int8_one_kernel<T>, dim3((a.n + 15) / 16), dim3(512), a.m * a.kpad, s, a);
  LIC_CHECK_LAUNCH();
  return 0;
}

template <typename T>
static int linear_run(Int8Args a, int8_t* codes, float* scale, hipStream_t s) {
  const uintptr_t p = (uintptr_t)a.y | (uintptr_t)a.r1 | (uintptr_t)a.ws | (uintptr_t)a.bias;
  constexpr int E = 16 / sizeof(T);
  a.wide = a.act != LIC_ACT_GELU;
  const bool lines = a.wide && p % 16 == 0 && a.ldy % E == 0 && (!a.r1 || a.ldr1 % E == 0);
  if (a.x) {
    const bool aligned = (uintptr_t)a.x % 16 == 0 && a.ldx % E == 0 && a.k % E == 0;
    if (a.m <= ONE_TOKENS && a.kpad <= ONE_K) return one_launch<T>(a, s);
    // us, 192 -> 576 fp16 (quantised apart, tiles): 131072 tokens 54.4 (97), 16384: 16.0 (20.1), 8192: 13.4 (14.5), 4096: 12
    // (10); 384 -> 384: 79.5 (94); from kpad 448 on the operands spill; fp32, 192 -> 576: 32768 tokens 34 (45), 8192: 21 (17.5)
    if (aligned && a.m >= (sizeof(T) == 2 ? 8192 : 16384) && a.kpad <= 384 && lines && a.n % 32 == 0) return rows_run<T>(a, s);
    if (int8_fused(a.m, a.kpad, a.n)) return fused_launch<T>(a, s);
    if (quantize_run<T>(a.x, a.ldx, a.m, a.k, codes, a.kpad, scale, s)) return 1;
    a.xc = codes;
    a.xs = scale;
  }
  // us, 4096 -> 4096 bf16, 16 / 64 tokens a workgroup / 64 x 64 tiles: 16 tokens 6.5 / 8.8 / -, 17: - / 8.5 / 9.5, 32: - /
  // 9.6 / 9.6, 64: - / 12.2 / 9.8; 64 x 1024 -> 1024: - / 4.6 / 4.8
  if (a.m <= 16) return few_launch<T, 1>(a, s);
  if (a.m <= 32 || (a.m <= 64 && a.kpad <= 1024)) return few_launch<T, 4>(a, s);
  // Rounds of workgroups over 256 compute units: one with 256 x 256 tiles takes as long as 1 / 0.28 with 128 x 128 ones (two
  // of which share a unit).  us, 256 x 256 / 128 x 128 / 64 x 64: 4096 x 2048 -> 4096 (256 of the largest) 44.7 / 51.9 / -,
  // -> 4097 (272) 94.2 / 69.8 / -, -> 2048 (128) 37.5 / 27.7 / -; 2048 x 2048 -> 2048 (256 of the middle) - / 16.5 / 20.3,
  // -> 1024 (128) - / 14.6 / 10.7
  const int64_t big = ((int64_t)a.m + 255) / 256 * (((int64_t)a.n + 255) / 256);
  const int64_t mid = ((int64_t)a.m + 127) / 128 * (((int64_t)a.n + 127) / 128);
  if (big >= 256 && 100 * ((big + 255) / 256) <= 28 * ((mid + 255) / 256)) return tile_launch<T, 256, 256, 2, 4, 1>(a, s);
  if (mid >= 256) return tile_launch<T, 128, 128, 2, 2, 1>(a, s);
  // few tiles of a long k, 1 / 2 groups of waves: 128 x 4096 -> 4096 12.9 / 9.9 us, 1024 x 1024 -> 1024 5.8 / 5.3, 200 x 500 ->
  // 1000 6.8 / 6.7; 2048 x 2048 -> 1024, of 512 tiles: 10.1 / 11.3
  const int64_t small = ((int64_t)a.m + 63) / 64 * (((int64_t)a.n + 63) / 64);
  return small <= 256 && a.kpad >= 1024 ? tile_launch<T, 64, 64, 2, 2, 2>(a, s) : tile_launch<T, 64, 64, 2, 2, 1>(a, s);
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

extern "C" int64_t lic_linear_int8_workspace(int32_t m, int32_t kpad, int32_t n) {
  if (m < 0 || n < 1 || kpad < 1 || kpad > LIC_INT8_MAX_K) return -1;
  if ((m <= lic::ONE_TOKENS && kpad <= lic::ONE_K) || lic::int8_fused(m, kpad, n)) return 0;   // quantised in LDS
  const int64_t codes = (int64_t)m * kpad;
  return (codes + 15) / 16 * 16 + 4 * (int64_t)m;
}

extern "C" int lic_linear_int8(int32_t dtype, const void* x, int64_t ldx, const int8_t* xcodes, const float* xscale,
                               int32_t m, int32_t k, const int8_t* w, int32_t kpad, const float* wscale,
                               const float* bias, int32_t n, int32_t act, float slope, const void* r1, int64_t ldr1,
                               void* y, int64_t ldy, void* ws, int64_t ws_bytes, lic_stream_t stream) {
  using namespace lic;
  if (check_sizes("linear_int8", dtype, m, k, kpad)) return 1;
  // a launch has less than 2^32 threads: 256 for a tile of 128 x 128 or 128 tokens, 512 for one of 256 x 256 or 16 channels
  if (m > INT32_MAX - 255) return fail("linear_int8: m out of range");
  if (n < 1 || n > (1 << 27) - 16) return fail("linear_int8: n out of range");
  if (((int64_t)m + 127) / 128 * (((int64_t)n + 127) / 128) >= 1 << 24) return fail("linear_int8: m x n out of range");
  if (act < LIC_ACT_NONE || act > LIC_ACT_GELU) return fail("linear_int8: act has to be none, relu, lrelu or gelu");
  if (m == 0) return 0;
  if (!w || !wscale || !y || ldy < n || (r1 && ldr1 < n)) return fail("linear_int8: null pointer or row stride below n");
  if ((x == nullptr) == (xcodes == nullptr) || (xcodes && !xscale)) return fail("linear_int8: give x or xcodes with xscale");
  if ((uintptr_t)w % 16 || (uintptr_t)xcodes % 16) return fail("linear_int8: codes have to be 16-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  if (x) {
    if (ldx < k) return fail("linear_int8: row stride below k");
    const int64_t need = lic_linear_int8_workspace(m, kpad, n);
    if (need && (!ws || (uintptr_t)ws % 16 || ws_bytes < need))
      return fail("linear_int8: workspace missing, misaligned or too small");
  }
  Int8Args a{xcodes, xscale, w, wscale, bias, r1, y, x, ldr1, ldy, ldx, m, n, k, kpad, act, slope, 0};
  int8_t* codes = (int8_t*)ws;
  float* scale = (float*)((char*)ws + ((int64_t)m * kpad + 15) / 16 * 16);
  if (dtype == LIC_F32) return linear_run<float>(a, codes, scale, s);
  if (dtype == LIC_F16) return linear_run<half_t>(a, codes, scale, s);
  return linear_run<bf16_t>(a, codes, scale, s);
}
