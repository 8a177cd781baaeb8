// Newton-Schulz orthogonalisation of many matrices at once (gfx950):
//   X = G / (|G|_F + eps);  `steps` times: A = X X^T, X = (a I + b A + c A A) X
// on r x c matrices with r <= c (G^T where G has more rows than columns).
#include "lic_common.h"

namespace lic {

struct OrthoDesc {
  const void* g;
  void* out;
  int64_t rs, cs;       // strides of G's (or G^T's) rows and columns
  int64_t x0, x1;       // the two copies of X, floats from the workspace's float area
  int64_t a, q;         // A and Q = a I + b A + c A A
  int32_t r, c, flip;   // flip: out is the transpose of X
  int32_t norm0;        // first partial sum of |G|^2
  int32_t gram0, upd0;  // first block of the r x r and of the r x c tiles
};

constexpr int ORTHO_BATCH = 32;   // descriptors a launch carries to the device in its arguments
struct OrthoBatch { OrthoDesc d[ORTHO_BATCH]; };

__global__ void ortho_desc_kernel(OrthoBatch b, int first, int count, OrthoDesc* dst) {
  if ((int)threadIdx.x < count) dst[first + threadIdx.x] = b.d[threadIdx.x];
}

template <int OrthoDesc::* FIRST>
__device__ __forceinline__ int ortho_find(const OrthoDesc* d, int count, int block) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (d[mid].*FIRST <= block) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

constexpr int ORTHO_NORM = 4096;   // elements of one partial sum

// Partial sums of squares in 64 bits: small gradients square to below fp32's range.
template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(const OrthoDesc* desc, int count, double* parts) {
  __shared__ double red[4];
  const int i = ortho_find<&OrthoDesc::norm0>(desc, count, blockIdx.x);
  const OrthoDesc d = desc[i];
  const int64_t first = (int64_t)((int)blockIdx.x - d.norm0) * ORTHO_NORM, total = (int64_t)d.r * d.c;
  double s = 0;
  for (int64_t e = first + threadIdx.x; e < first + ORTHO_NORM && e < total; e += 256) {
    const double v = (double)to_f(((const T*)d.g)[e / d.c * d.rs + e % d.c * d.cs]);
    s += v * v;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) parts[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

template <typename T>
__global__ __launch_bounds__(256) void ortho_scale_kernel(const OrthoDesc* desc, int count, const double* parts,
                                                          float eps, float* f) {
  const int i = ortho_find<&OrthoDesc::norm0>(desc, count, blockIdx.x);
  const OrthoDesc d = desc[i];
  const int64_t first = (int64_t)((int)blockIdx.x - d.norm0) * ORTHO_NORM, total = (int64_t)d.r * d.c;
  double s = 0;
  for (int64_t p = 0; p * ORTHO_NORM < total; ++p) s += parts[d.norm0 + p];
  const double inv = 1.0 / (sqrt(s) + (double)eps);
  for (int64_t e = first + threadIdx.x; e < first + ORTHO_NORM && e < total; e += 256)
    f[d.x0 + e] = (float)((double)to_f(((const T*)d.g)[e / d.c * d.rs + e % d.c * d.cs]) * inv);
}

// One 32 x 32 tile of P R (or P R^T) in fp32, four outputs a thread.
template <bool TRANS>
__device__ __forceinline__ void ortho_tile(const float* p, int ldp, const float* rr, int ldr, int rows, int cols,
                                           int kk, int i0, int j0, float* acc) {
  __shared__ float sp[32][33], sr[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  for (int k0 = 0; k0 < kk; k0 += 32) {
    for (int q = ty; q < 32; q += 8) {
      sp[q][tx] = (i0 + q < rows && k0 + tx < kk) ? p[(int64_t)(i0 + q) * ldp + k0 + tx] : 0.f;
      if (TRANS) sr[tx][q] = (j0 + q < cols && k0 + tx < kk) ? rr[(int64_t)(j0 + q) * ldr + k0 + tx] : 0.f;
      else sr[q][tx] = (k0 + q < kk && j0 + tx < cols) ? rr[(int64_t)(k0 + q) * ldr + j0 + tx] : 0.f;
    }
    __syncthreads();
    float part[4] = {0, 0, 0, 0};   // sums of sums: a long row's rounding errors do not pile up
    for (int k = 0; k < 32; ++k)
#pragma unroll
      for (int q = 0; q < 4; ++q) part[q] += sp[ty + 8 * q][k] * sr[k][tx];
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[q] += part[q];
    __syncthreads();
  }
}

// stage 0: A = X X^T;  1: Q = a I + b A + c A A
__global__ __launch_bounds__(256) void ortho_gram_kernel(const OrthoDesc* desc, int count, float* f, int odd, int stage,
                                                         float ca, float cb, float cc) {
  const OrthoDesc d = desc[ortho_find<&OrthoDesc::gram0>(desc, count, blockIdx.x)];
  const int nt = (d.r + 31) / 32, t = blockIdx.x - d.gram0;
  const int i0 = t / nt * 32, j0 = t % nt * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float acc[4] = {0, 0, 0, 0};
  const float* x = f + (odd ? d.x1 : d.x0);
  if (stage == 0) ortho_tile<true>(x, d.c, x, d.c, d.r, d.r, d.c, i0, j0, acc);
  else ortho_tile<true>(f + d.a, d.r, f + d.a, d.r, d.r, d.r, d.r, i0, j0, acc);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = i0 + ty + 8 * q, j = j0 + tx;
    if (i >= d.r || j >= d.r) continue;
    const int64_t at = (int64_t)i * d.r + j;
    if (stage == 0) f[d.a + at] = acc[q];
    else f[d.q + at] = (i == j ? ca : 0.f) + cb * f[d.a + at] + cc * acc[q];
  }
}

// X <- Q X; the last step writes the result
template <typename T>
__global__ __launch_bounds__(256) void ortho_update_kernel(const OrthoDesc* desc, int count, float* f, int odd,
                                                           int last) {
  const OrthoDesc d = desc[ortho_find<&OrthoDesc::upd0>(desc, count, blockIdx.x)];
  const int nt = (d.c + 31) / 32, t = blockIdx.x - d.upd0;
  const int i0 = t / nt * 32, j0 = t % nt * 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  float acc[4] = {0, 0, 0, 0};
  ortho_tile<false>(f + d.q, d.r, f + (odd ? d.x1 : d.x0), d.c, d.r, d.c, d.r, i0, j0, acc);
  float* xn = f + (odd ? d.x0 : d.x1);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int i = i0 + ty + 8 * q, j = j0 + tx;
    if (i >= d.r || j >= d.c) continue;
    if (last) ((T*)d.out)[d.flip ? (int64_t)j * d.r + i : (int64_t)i * d.c + j] = from_f<T>(acc[q]);
    else xn[(int64_t)i * d.c + j] = acc[q];
  }
}

struct OrthoPlan {
  int64_t desc_bytes = 0, parts_bytes = 0, floats = 0;
  int64_t norm = 0, gram = 0, upd = 0;
  int64_t bytes() const { return desc_bytes + parts_bytes + 4 * floats; }
};

static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Offsets and block counts of every matrix; false: sizes out of range.
static bool ortho_plan(int count, const lic_ortho_mat* mats, OrthoPlan& p, OrthoDesc* d) {
  for (int i = 0; i < count; ++i) {
    const lic_ortho_mat& m = mats[i];
    if (m.rows < 1 || m.cols < 1 || m.rows > 65536 || m.cols > (1 << 24)) return false;
    const bool flip = m.rows > m.cols;
    const int64_t r = flip ? m.cols : m.rows, c = flip ? m.rows : m.cols;
    OrthoDesc o{m.g, m.out, flip ? m.cs : m.rs, flip ? m.rs : m.cs};
    o.r = (int32_t)r;
    o.c = (int32_t)c;
    o.flip = flip;
    o.x0 = p.floats;
    o.x1 = o.x0 + up(r * c, 64);
    o.a = o.x1 + up(r * c, 64);
    o.q = o.a + up(r * r, 64);
    p.floats = o.q + up(r * r, 64);
    o.norm0 = (int32_t)p.norm;
    o.gram0 = (int32_t)p.gram;
    o.upd0 = (int32_t)p.upd;
    p.norm += (r * c + ORTHO_NORM - 1) / ORTHO_NORM;
    p.gram += up(r, 32) / 32 * (up(r, 32) / 32);
    p.upd += up(r, 32) / 32 * (up(c, 32) / 32);
    if (p.norm > (1 << 30) || p.gram > (1 << 30) || p.upd > (1 << 30)) return false;
    if (d) d[i] = o;
  }
  p.desc_bytes = up((int64_t)count * sizeof(OrthoDesc), 256);
  p.parts_bytes = up(p.norm * 8, 256);
  return true;
}

template <typename T>
static int ortho_run(const OrthoPlan& p, int count, const lic_ortho_mat* mats, int steps, const float* co, float eps,
                     char* ws, hipStream_t s) {
  OrthoDesc* desc = (OrthoDesc*)ws;
  double* parts = (double*)(ws + p.desc_bytes);
  float* f = (float*)(ws + p.desc_bytes + p.parts_bytes);
  OrthoPlan q;
  OrthoBatch b;
  // the offsets are those of the whole list: planned again in batches of descriptors
  for (int i = 0; i < count; i += ORTHO_BATCH) {
    const int k = count - i < ORTHO_BATCH ? count - i : ORTHO_BATCH;
    if (!ortho_plan(k, mats + i, q, b.d)) return fail("orthogonalize: sizes out of range");
    hipLaunchKernelGGL(ortho_desc_kernel, dim3(1), dim3(64), 0, s, b, i, k, desc);
    LIC_CHECK_LAUNCH();
  }
  hipLaunchKernelGGL(ortho_norm_kernel<T>, dim3((unsigned)p.norm), dim3(256), 0, s, desc, count, parts);
  hipLaunchKernelGGL(ortho_scale_kernel<T>, dim3((unsigned)p.norm), dim3(256), 0, s, desc, count, parts, eps, f);
  for (int k = 0; k < steps; ++k) {
    for (int stage = 0; stage < 2; ++stage)
      hipLaunchKernelGGL(ortho_gram_kernel, dim3((unsigned)p.gram), dim3(256), 0, s, desc, count, f, k & 1, stage, co[0],
                         co[1], co[2]);
    hipLaunchKernelGGL(ortho_update_kernel<T>, dim3((unsigned)p.upd), dim3(256), 0, s, desc, count, f, k & 1,
                       k == steps - 1);
  }
  LIC_CHECK_LAUNCH();
  return 0;
}

}  // namespace lic

extern "C" int64_t lic_orthogonalize_workspace(int32_t dtype, int32_t count, const lic_ortho_mat* mats) {
  using namespace lic;
  OrthoPlan p;
  if (count < 0 || (count && !mats) || !ortho_plan(count, mats, p, nullptr)) return -1;
  return p.bytes();
}

extern "C" int lic_orthogonalize(int32_t dtype, int32_t count, const lic_ortho_mat* mats, int32_t steps,
                                 const float* coeffs, float eps, void* ws, int64_t ws_bytes, lic_stream_t stream) {
  using namespace lic;
  if (dtype != LIC_F32 && dtype != LIC_F16 && dtype != LIC_BF16) return fail("orthogonalize: bad dtype");
  if (count < 0 || (count && !mats) || !coeffs) return fail("orthogonalize: null pointer");
  if (steps < 1 || steps > 64) return fail("orthogonalize: steps out of range");
  if (!(eps >= 0.f)) return fail("orthogonalize: eps has to be >= 0");
  if (count == 0) return 0;
  OrthoPlan p;
  if (!ortho_plan(count, mats, p, nullptr)) return fail("orthogonalize: sizes out of range");
  for (int i = 0; i < count; ++i)
    if (!mats[i].g || !mats[i].out) return fail("orthogonalize: null matrix");
  if (!ws || (uintptr_t)ws % 256 || ws_bytes < p.bytes()) return fail("orthogonalize: workspace missing, misaligned or too small");
  hipStream_t s = (hipStream_t)stream;
  if (dtype == LIC_F32) return ortho_run<float>(p, count, mats, steps, coeffs, eps, (char*)ws, s);
  if (dtype == LIC_F16) return ortho_run<half_t>(p, count, mats, steps, coeffs, eps, (char*)ws, s);
  return ortho_run<bf16_t>(p, count, mats, steps, coeffs, eps, (char*)ws, s);
}
