// Newton-Schulz orthogonalisation of many matrices at once (gfx950):
//   X = G / (|G|_F + eps);  `steps` times: A = X X^T, X = (a I + b A + c A A) X
// on r x c matrices with r <= c (G^T where G has more rows than columns).
//
// Every product runs on fp16 matrix instructions with operands of two parts, value = hi + lo, as hi hi' + hi lo' + lo hi' with
// fp32 sums.  So X, A and Q have 22 bits between the products, two less than fp32's: taken for its cost, three eighths of fp32
// matrix instructions' (one part alone would leave 4e-4 .. 3e-3 of the result).  Error against 64 bits, over that of the same
// iteration in fp32 products, in the Frobenius norm: 16 x 144 0.74, 64 x 64 1.01, 66 x 66 1.22, 128 x 128 1.15, 128 x 576
// 1.12, 192 x 1728 1.03, 512 x 2304 0.79, 2048 x 2048 0.53 (3.0e-6 of the result for 5.6e-6).  More of it than of fp32's lies
// along few directions: in the 2-norm 66 x 66 1.22, 192 x 1728 1.37, 512 x 2304 1.98, 2048 x 2048 2.11 (1.7e-5 for 8.1e-6).
// X is held divided by a power of two above its norm (from |G| and the polynomial's bounds), so the parts never leave fp16's
// range.
//
// Operands lie in fragment order: [row / 32][k / 16][hi, lo][64 lanes][8], one contiguous KB a fragment, loaded straight into
// registers; place p of a 32-row tile is row 16 ((p / 4) % 2) + 4 (p / 8) + p % 4 of it.  With that order on both operands a
// lane's 16 results (rows 8 (i / 4) + 4 (lane / 32) + i % 4 of the instruction) are 16 consecutive rows, a whole k step of the
// transposed operand.  X is kept in both orders: rows along r for A = X X^T, rows along c (X^T) for Q X.
#include "lic_common.h"
#include <algorithm>
#include <cmath>
#include <vector>

namespace lic {

constexpr int ORTHO_MAX_STEPS = 64;

struct OrthoDesc {
  const void* g;
  void* out;
  int64_t rs, cs;       // strides of G's (or G^T's) rows and columns
  int64_t x, xt;        // the two copies of X in both orders, halves from the workspace's operand area; the second of
  int64_t a, q;         // each follows at + step.  A and Q = a I + b A + c A A
  int64_t step;
  int32_t r, c, flip;   // flip: out is the transpose of X
  int32_t parts0;       // first of its 64 x 64 tiles' partial sums of |G|^2
  int32_t gram0, upd0;  // first workgroup of A's lower triangle, and of X
  int32_t slices;       // workgroups that share a tile of A = X X^T
  int32_t slice0, sum0; // first of them, and of the tiles that are summed up from more than one
  int32_t partial0;     // first of the slices' sums
  int64_t rest;         // both copies' third parts of X^T (fine matrices only, else -1)
};

// The workgroups of a stage in matrix order.
struct OrthoTile { int32_t mat, at; };

constexpr int ORTHO_BATCH = 24;   // descriptors that a launch carries to the device in its arguments
struct OrthoBatch { OrthoDesc d[ORTHO_BATCH]; };

struct OrthoWork {
  OrthoDesc* desc;
  OrthoTile *tiles, *gram, *upd;   // 64 x 64 tiles of G, lower tiles of A, 64 x 256 tiles of X
  OrthoTile *slices, *sums;        // slices of lower tiles, tiles of several slices
  float* partial;                  // [slice of a tile that has several][4096]
  double* parts;
  int32_t* exps;                   // [count][ORTHO_MAX_STEPS + 1] exponents of X's scale
  half_t* ops;
};

// What the polynomial alone says: bounds of |X| after k steps for |X| <= 1, of |X'| / |X|, exponents of Q's scale.
struct OrthoBounds {
  float most[ORTHO_MAX_STEPS + 1], gain;
  int32_t qexp[ORTHO_MAX_STEPS];
};

__device__ __forceinline__ int ortho_tiles(int n) { return (n + 63) / 64; }

// The tables' entries of one matrix, for the kernels that follow.
__device__ __forceinline__ void ortho_setup(const OrthoDesc& d, int mat, const OrthoWork& w) {
  const int nr = ortho_tiles(d.r), nc = ortho_tiles(d.c), nu = (d.c + 255) / 256;
  if (threadIdx.x == 0) w.desc[mat] = d;
  for (int i = threadIdx.x; i < nr * nc; i += 256) w.tiles[d.parts0 + i] = {mat, i};
  // workgroups of one group of columns follow each other (in groups of 8 tiles of rows): they share X's fragments in the L2
  for (int i = threadIdx.x; i < nr * nu; i += 256) {
    const int group = i / (8 * nu), rest = i - group * 8 * nu, rows = min(8, nr - group * 8);
    w.upd[d.upd0 + i] = {mat, (group * 8 + rest % rows) << 16 | rest / rows};
  }
  for (int i = threadIdx.x; i < nr; i += 256)
    for (int j = 0; j <= i; ++j) {
      const int at = i * (i + 1) / 2 + j;
      w.gram[d.gram0 + at] = {mat, i << 16 | j};
      for (int k = 0; k < d.slices; ++k) w.slices[d.slice0 + at * d.slices + k] = {mat, i << 16 | j};
      if (d.slices > 1) w.sums[d.sum0 + at] = {mat, i << 16 | j};
    }
}

// Workgroups go round the 8 XCDs: ORTHO_RUN neighbouring tiles, which share operands in an L2, for each in turn (longer runs
// would give one XCD all the tiles of the longest matrices).
constexpr int ORTHO_RUN = 16;   // codec-sized lists: 432 us; 1: 504, 4: 447, 8: 440
__device__ __forceinline__ int ortho_id() {
  const int b = blockIdx.x, round = 8 * ORTHO_RUN;
  if (b >= (int)gridDim.x / round * round) return b;
  const int xcd = b & 7, slot = b >> 3;
  return slot / ORTHO_RUN * round + xcd * ORTHO_RUN + slot % ORTHO_RUN;
}

__device__ __forceinline__ int ortho_place(int p) { return (((p >> 2) & 1) << 4) | (((p >> 3) & 3) << 2) | (p & 3); }

// G and the result come as addresses from a table: said to be global, so that their accesses are not flat ones.
template <typename T> using OrthoGlobal = __attribute__((address_space(1))) T*;

// A 64 x 64 tile of G, element (i, j) of it to thread (of 256) and slot (of 16) so that either order of G reads in lines.
template <typename T, typename F>
__device__ __forceinline__ void ortho_read(const OrthoDesc& d, int i0, int j0, F f) {
  const bool along = d.cs <= d.rs;   // columns are the nearer ones
  const int fast = threadIdx.x & 63, slow = threadIdx.x >> 6;
#pragma unroll
  for (int s = 0; s < 16; ++s) {
    const int i = along ? slow * 16 + s : fast, j = along ? fast : slow * 16 + s;
    const bool in = i0 + i < d.r && j0 + j < d.c;
    f(i, j, in ? to_f(((OrthoGlobal<const T>)d.g)[(i0 + i) * d.rs + (j0 + j) * d.cs]) : 0.f);
  }
}

// Sums of squares in 64 bits: the squares of small gradients are below fp32's range.  A matrix without gaps is read as a
// line, 4096 elements a workgroup.  Bound by G's bytes: 42 matrices of a codec's layers (42 MB)
// 19 us in two launches, tables included (12 without them), 2048 x 2048 7.8 us (5.3).
// The descriptors come in the launch's arguments, a batch of them at a time; a matrix's first workgroup also writes its
// entries of the tables (128 x 576: 108.8 -> 107.6 us without a launch for them).
template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(OrthoBatch b, int count, int first, OrthoWork w) {
  __shared__ double red[4];
  const int id = b.d[0].parts0 + (int)blockIdx.x;
  int m = 0;
#pragma unroll
  for (int i = 1; i < ORTHO_BATCH; ++i) m += i < count && b.d[i].parts0 <= id;
  const OrthoDesc d = b.d[m];
  const OrthoTile t{first + m, id - d.parts0};
  if (t.at == 0) ortho_setup(d, t.mat, w);
  const int nc = ortho_tiles(d.c);
  double s = 0;
  if ((d.cs == 1 && d.rs == d.c) || (d.rs == 1 && d.cs == d.r)) {
    constexpr int V = 16 / sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(V)));
    const OrthoGlobal<const T> g = (OrthoGlobal<const T>)d.g;
    const int64_t total = (int64_t)d.r * d.c, first = (int64_t)t.at * 4096;
    if ((uintptr_t)d.g % 16 == 0 && first + 4096 <= total) {
      Vec v[16 / V];
#pragma unroll
      for (int i = 0; i < 16 / V; ++i) v[i] = ((OrthoGlobal<const Vec>)(g + first))[i * 256 + threadIdx.x];
#pragma unroll
      for (int i = 0; i < 16 / V; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) s += (double)to_f(v[i][e]) * (double)to_f(v[i][e]);
    } else {
      for (int64_t e = first + threadIdx.x; e < first + 4096 && e < total; e += 256)
        s += (double)to_f(g[e]) * (double)to_f(g[e]);
    }
  } else {
    ortho_read<T>(d, t.at / nc * 64, t.at % nc * 64, [&](int, int, float v) { s += (double)v * (double)v; });
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) w.parts[id] = red[0] + red[1] + red[2] + red[3];
}

// value * 2^14 in two fp16 parts (|value| <= 1)
struct OrthoParts { half8 hi, lo, rest; };
__device__ __forceinline__ void ortho_split(OrthoParts& p, int e, float scaled) {
  const half_t h = (half_t)scaled;
  p.hi[e] = h;
  p.lo[e] = (half_t)(scaled - (float)h);
  p.rest[e] = (half_t)(scaled - (float)h - (float)p.lo[e]);   // fine matrices'
}

// The fragments of a 64 x 64 tile in LDS (t[row][col], `flip`: its transpose): thread (of 512) -> 8 values of k.
constexpr int ORTHO_LD = 65;
template <bool FLIP>
__device__ __forceinline__ OrthoParts ortho_gather(const float* t, int rowtile, int ks, int lane, float scale) {
  const int row = 32 * rowtile + ortho_place(lane & 31), k = 16 * ks + 8 * (lane >> 5);
  OrthoParts p;
#pragma unroll
  for (int e = 0; e < 8; ++e) ortho_split(p, e, scale * (FLIP ? t[(k + e) * ORTHO_LD + row] : t[row * ORTHO_LD + k + e]));
  return p;
}
__device__ __forceinline__ half_t* ortho_fragment(half_t* m, int ksteps, int rowtile, int ks) {
  return m + ((int64_t)rowtile * ksteps + ks) * 1024;
}
__device__ __forceinline__ half_t* ortho_third(half_t* m, int ksteps, int rowtile, int ks, int lane) {
  return m + ((int64_t)rowtile * ksteps + ks) * 512 + lane * 8;
}
__device__ __forceinline__ void ortho_put(half_t* frag, int lane, const OrthoParts& p) {
  *(half8*)(frag + lane * 8) = p.hi;
  *(half8*)(frag + 512 + lane * 8) = p.lo;
}

// X = G / (|G| + eps) in both orders; the exponents of all steps' scales.  Bound by the bytes of G and of both copies (12 a
// fp32 element): 2048 x 2048 16.3 us (3.1 TB/s), the 42 matrices 28 us (4.4 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void ortho_scale_kernel(OrthoWork w, OrthoBounds b, int steps, float eps) {
  __shared__ double red[4];
  __shared__ float tile[64 * ORTHO_LD];
  const OrthoTile t = w.tiles[blockIdx.x];
  const OrthoDesc d = w.desc[t.mat];
  const int nr = ortho_tiles(d.r), nc = ortho_tiles(d.c), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double s = 0;
  for (int i = threadIdx.x; i < nr * nc; i += 256) s += w.parts[d.parts0 + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  const double norm = sqrt(red[0] + red[1] + red[2] + red[3]);
  const double size = norm + (double)eps, ratio = size > 0 ? norm / size : 0.0;   // |X|
  auto exponent = [](double v) {   // 2^e > v; bounded: below it X is zero in fp32
    int e = 0;
    if (v > 0 && v < 1e30) (void)frexp(v, &e);
    return v > 0 ? (e > -140 ? e : -140) : -140;
  };
  const int e0 = norm == norm ? exponent(ratio) : 0;
  if (t.at == 0 && threadIdx.x == 0) {
    double most = ratio;
    for (int k = 0; k <= steps; ++k) {
      w.exps[t.mat * (ORTHO_MAX_STEPS + 1) + k] = norm == norm ? exponent(most) : 0;
      most = fmin(most * (double)b.gain, (double)b.most[k < steps ? k + 1 : k]);
    }
  }
  const double inv = size > 0 ? ldexp(1.0 / size, 14 - e0) : 0.0;
  const int i0 = t.at / nc, j0 = t.at % nc;
  ortho_read<T>(d, i0 * 64, j0 * 64, [&](int i, int j, float v) { tile[i * ORTHO_LD + j] = (float)((double)v * inv); });
  __syncthreads();
  half_t *x = w.ops + d.x, *xt = w.ops + d.xt;
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int f = wave * 2 + u, rt = f >> 2, ks = f & 3;
    ortho_put(ortho_fragment(x, nc * 4, i0 * 2 + rt, j0 * 4 + ks), lane, ortho_gather<false>(tile, rt, ks, lane, 1.f));
    const OrthoParts pt = ortho_gather<true>(tile, rt, ks, lane, 1.f);
    ortho_put(ortho_fragment(xt, nr * 4, j0 * 2 + rt, i0 * 4 + ks), lane, pt);
    if (d.rest >= 0) *(half8*)ortho_third(w.ops + d.rest, nr * 4, j0 * 2 + rt, i0 * 4 + ks, lane) = pt.rest;
  }
}

// 64 x 64 results of P R^T over k steps [s0, s1), operands in fragment order (two row tiles each): acc[i][j] is P's tile i
// against R's tile j.
// Steps that the matrix instructions sum up before the rounded fp32 addition to the total: their own additions of a long chain
// lose more.  Error of the result (Frobenius) at 2048 x 2048: one chain 8.9e-6, chains of 16 steps 4.0e-6, of 8 3.3e-6, of 4 3.0e-6 (fp32
// products: 5.6e-6); 128 x 576: 2.9e-6, .., 2.4e-6 (2.2e-6).  4 costs 1 to 3 % of the time.
constexpr int ORTHO_CHAIN = 4;
struct OrthoFrags { half8 p[2][2], r[2][2]; };
__device__ __forceinline__ void ortho_load(OrthoFrags& f, const half_t* p, const half_t* r, int64_t ptile, int64_t rtile,
                                           int s) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f.p[i][h] = *(const half8*)(p + i * ptile + (int64_t)s * 1024 + h * 512);
      f.r[i][h] = *(const half8*)(r + i * rtile + (int64_t)s * 1024 + h * 512);
    }
}
// The small products first, while the sums that they are added to are small.  FIRST: of a chain, which starts from zero.
template <bool FIRST>
__device__ __forceinline__ void ortho_multiply(floatx16 (&acc)[2][2], const OrthoFrags& f) {
#pragma unroll
  for (int q = 2; q >= 0; --q)   // lo hi, hi lo, hi hi
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.p[i][q == 2], f.r[j][q == 1],
                                                           FIRST && q == 2 ? floatx16{} : acc[i][j], 0, 0, 0);
}
__device__ __forceinline__ void ortho_sum(floatx16 (&sum)[2][2], const floatx16 (&acc)[2][2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[i][j][e] += acc[i][j][e];
}
__device__ __forceinline__ void ortho_product(floatx16 (&sum)[2][2], const half_t* p, const half_t* r, int64_t ptile,
                                              int64_t rtile, int s0, int s1) {
  if (s0 >= s1) return;
  OrthoFrags f0, f1;   // one step is multiplied while the next one is under way
  floatx16 acc[2][2];
  auto load = [&](OrthoFrags& f, int s) {
    ortho_load(f, p, r, ptile, rtile, s < s1 ? s : s1 - 1);
    __builtin_amdgcn_sched_barrier(0);
  };
  load(f0, s0);
  int s = s0;
  for (; s + ORTHO_CHAIN <= s1; s += ORTHO_CHAIN) {
#pragma unroll
    for (int c = 0; c < ORTHO_CHAIN; c += 2) {
      load(f1, s + c + 1);
      if (c == 0) ortho_multiply<true>(acc, f0);
      else ortho_multiply<false>(acc, f0);
      load(f0, s + c + 2);
      ortho_multiply<false>(acc, f1);
    }
    ortho_sum(sum, acc);
  }
  if (s < s1) {   // up to three steps
    load(f1, s + 1);
    ortho_multiply<true>(acc, f0);
    if (s + 1 < s1) {
      load(f0, s + 2);
      ortho_multiply<false>(acc, f1);
      if (s + 2 < s1) ortho_multiply<false>(acc, f0);
    }
    ortho_sum(sum, acc);
  }
}

// What two parts leave out of Q X, for matrices whose short sums would show it: Q's low part with X's, Q's high part with X's
// third, which is what fp32 holds of X beyond 22 bits.  The error against 64 bits is mostly that of X between the steps;
// Frobenius norm against that of fp32 products: 16 x 144 1.20 -> 0.81 of it, 64 x 64 1.25 -> 1.02; 66 x 66, without, 1.24, 128 x 128 1.13,
// 192 x 192 1.01, where the sums' own rounding is as large.  64 x 576 91.9 -> 103.3 us; up to 128 rows 128 x 576 would be 135.
constexpr int ORTHO_FINE = 64;
__device__ __forceinline__ void ortho_finer(floatx16 (&sum)[2][2], const half_t* x, const half_t* rest, const half_t* q,
                                            int64_t tile) {
  floatx16 acc[2][2] = {};
#pragma unroll
  for (int s = 0; s < ORTHO_FINE / 16; ++s) {   // all of the sum
    half8 lo[2], third[2], qh[2], ql[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      lo[i] = *(const half8*)(x + i * tile + (int64_t)s * 1024 + 512);
      third[i] = *(const half8*)(rest + i * tile / 2 + (int64_t)s * 512);
      qh[i] = *(const half8*)(q + i * tile + (int64_t)s * 1024);
      ql[i] = *(const half8*)(q + i * tile + (int64_t)s * 1024 + 512);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(lo[i], ql[j], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(third[i], qh[j], acc[i][j], 0, 0, 0);
      }
  }
  ortho_sum(sum, acc);
}

// A 64 x 64 tile of the lower triangle of A = X X^T (STAGE 0) or Q = a I + b A + c A A (STAGE 1), and its mirror image, from
// the sums in LDS (which carry 2^28): 8 fragments among the waves.
template <int STAGE>
__device__ __forceinline__ void ortho_lower(const OrthoWork& w, const OrthoDesc& d, int mat, int at, const float* out, int k,
                                            float ca, float cb, float cc, int qexp) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ti = at >> 16, tj = at & 0xffff, nr = ortho_tiles(d.r);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int m = g / 2, f8 = g % 2 * 4 + wave, rt = f8 >> 2, ks = f8 & 3;
    if (m == 1 && ti == tj) break;
    const int I = m ? tj : ti, J = m ? ti : tj;
    OrthoParts p;
    if constexpr (STAGE == 0) {
      p = m ? ortho_gather<true>(out, rt, ks, lane, 0x1p-14f) : ortho_gather<false>(out, rt, ks, lane, 0x1p-14f);
      ortho_put(ortho_fragment(w.ops + d.a, nr * 4, I * 2 + rt, J * 4 + ks), lane, p);
    } else {
      const half_t* f = ortho_fragment(w.ops + d.a, nr * 4, I * 2 + rt, J * 4 + ks);
      const half8 hi = *(const half8*)(f + lane * 8), lo = *(const half8*)(f + 512 + lane * 8);
      const int e2 = 2 * w.exps[mat * (ORTHO_MAX_STEPS + 1) + k];
      const float s1 = ldexpf(cb, e2 - 14), s2 = ldexpf(cc, 2 * e2 - 28), down = ldexpf(1.f, 14 - qexp);
      const int row = 32 * rt + ortho_place(lane & 31), col = 16 * ks + 8 * (lane >> 5);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float aa = m ? out[(col + e) * ORTHO_LD + row] : out[row * ORTHO_LD + col + e];
        float v = s1 * ((float)hi[e] + (float)lo[e]) + s2 * aa;
        if (I * 64 + row == J * 64 + col + e) v += ca;
        ortho_split(p, e, down * v);
      }
      ortho_put(ortho_fragment(w.ops + d.q, nr * 4, I * 2 + rt, J * 4 + ks), lane, p);
    }
  }
}

// A thread's sums of a tile (place e * 256 + thread of the joined order) to LDS, [64][ORTHO_LD].
__device__ __forceinline__ void ortho_spread(float* out, const float* v) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int at = e * 256 + threadIdx.x, l = at & 63, f = at >> 6, i = f & 15, b = (f >> 4) & 1, a = f >> 5;
    out[(32 * a + 16 * (l >> 5) + i) * ORTHO_LD + 32 * b + ortho_place(l & 31)] = v[e];
  }
}

// A tile of the lower triangle a workgroup.  Its four waves take a quarter of k each and are joined in LDS in a fixed order:
// a single long matrix has few tiles.  STAGE 0: of a slice of k where there are several; their sums go on to
// ortho_sum_kernel.  Half of the products of a symmetric result are left out: 2048 x 2048 47 us, 565 TFLOP/s of fp16 products
// (528 tiles on the 512 places of the chip: the last 16 cost a third of it); 128 x 576 6.6 us, the latency of nine k steps a
// wave; tiles of 128 x 128 would be 36 at a shorter side of 1024, for 256 compute units.
template <int STAGE>
__global__ __launch_bounds__(256, 2) void ortho_gram_kernel(OrthoWork w, int k, float ca, float cb, float cc, int qexp) {
  __shared__ float join[2][4096];   // [wave][tile of 32 x 32][result][lane]; then the tile, [64][ORTHO_LD]
  const int id = ortho_id();
  const OrthoTile t = STAGE == 0 ? w.slices[id] : w.gram[id];
  const OrthoDesc d = w.desc[t.mat];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ti = t.at >> 16, tj = t.at & 0xffff, nr = ortho_tiles(d.r), nc = ortho_tiles(d.c);
  const half_t* op = w.ops + (STAGE == 0 ? d.x + (k & 1) * d.step : d.a);
  const int ksteps = (STAGE == 0 ? nc : nr) * 4;
  const int64_t tile = (int64_t)ksteps * 1024;
  const int shares = STAGE == 0 ? 4 * d.slices : 4, share = STAGE == 0 ? (id - d.slice0) % d.slices * 4 + wave : wave;
  floatx16 acc[2][2] = {};
  ortho_product(acc, op + ti * 2 * tile + lane * 8, op + tj * 2 * tile + lane * 8, tile, tile,
                (int)((int64_t)ksteps * share / shares), (int)((int64_t)ksteps * (share + 1) / shares));
  if (wave >= 2) {
#pragma unroll
    for (int e = 0; e < 64; ++e) join[wave - 2][e * 64 + lane] = acc[e >> 5][(e >> 4) & 1][e & 15];
  }
  __syncthreads();
  if (wave < 2) {
#pragma unroll
    for (int e = 0; e < 64; ++e) join[wave][e * 64 + lane] += acc[e >> 5][(e >> 4) & 1][e & 15];
  }
  __syncthreads();
  float v[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = join[0][e * 256 + threadIdx.x] + join[1][e * 256 + threadIdx.x];
  if (STAGE == 0 && d.slices > 1) {
    float* part = w.partial + (int64_t)(id - d.slice0 + d.partial0) * 4096;
#pragma unroll
    for (int e = 0; e < 16; ++e) part[e * 256 + threadIdx.x] = v[e];
    return;
  }
  __syncthreads();
  ortho_spread(&join[0][0], v);
  __syncthreads();
  ortho_lower<STAGE>(w, d, t.mat, t.at, &join[0][0], k, ca, cb, cc, qexp);
}

// A from the slices' sums, in their order.
__global__ __launch_bounds__(256) void ortho_sum_kernel(OrthoWork w) {
  __shared__ float out[64 * ORTHO_LD];
  const OrthoTile t = w.sums[blockIdx.x];
  const OrthoDesc d = w.desc[t.mat];
  const float* from = w.partial + (d.partial0 + (int64_t)((int)blockIdx.x - d.sum0) * d.slices) * 4096;
  float v[16] = {};
#pragma unroll 3   // 192 x 4800: 167.6 -> 161.8 us
  for (int s = 0; s < d.slices; ++s)
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] += from[s * 4096 + e * 256 + threadIdx.x];
  ortho_spread(out, v);
  __syncthreads();
  ortho_lower<0>(w, d, t.mat, t.at, out, 0, 0.f, 0.f, 0.f, 0);
}

template <typename T, int N>
__device__ __forceinline__ void ortho_out(OrthoGlobal<T> out, int count, bool wide, const float* v) {
  if (wide && count >= N) {
    constexpr int E = 16 / sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(E)));
#pragma unroll
    for (int e = 0; e < N; e += E) {
      Vec o;
#pragma unroll
      for (int f = 0; f < E; ++f) o[f] = from_f<T>(v[e + f]);
      *(OrthoGlobal<Vec>)(out + e) = o;
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < count) out[e] = from_f<T>(v[e]);
  }
}

// X <- Q X: 64 rows x 64 columns a wave, 64 x 256 a workgroup (Q's fragments are shared through the L1).  The last step
// writes the result instead.  Bound by the matrix instructions and the 8 bytes an element of both copies: 2048 x 2048 59 us,
// 873 TFLOP/s of fp16 products (the library's large fp16 product: 1160; operands through LDS in 128 x 128 tiles: 68 us;
// 128 x 256 a workgroup: 93); the 42 matrices, whose sums are 1 to 32 k steps long, 35 us for 123 MB.
template <typename T>
__global__ __launch_bounds__(256, 2) void ortho_update_kernel(OrthoWork w, int k, int last, int qexp) {
  __shared__ float turn[4][32 * 33];
  const OrthoTile t = w.upd[ortho_id()];
  const OrthoDesc d = w.desc[t.mat];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nr = ortho_tiles(d.r), nc = ortho_tiles(d.c);
  const int ti = t.at >> 16, tj = (t.at & 0xffff) * 4 + wave;
  if (tj >= nc) return;
  const int64_t now = (k & 1) * d.step, next = d.step - now, tile = (int64_t)nr * 4 * 1024;
  floatx16 acc[2][2] = {};   // [tile of columns][tile of rows]
  ortho_product(acc, w.ops + d.xt + now + tj * 2 * tile + lane * 8, w.ops + d.q + ti * 2 * tile + lane * 8, tile, tile, 0,
                nr * 4);
  if (d.rest >= 0)
    ortho_finer(acc, w.ops + d.xt + now + tj * 2 * tile + lane * 8,
                ortho_third(w.ops + d.rest + (k & 1) * (int64_t)nr * nc * 4096, nr * 4, tj * 2, 0, lane),
                w.ops + d.q + ti * 2 * tile + lane * 8, tile);
  const int32_t* ex = w.exps + t.mat * (ORTHO_MAX_STEPS + 1) + k;
  const int half = lane >> 5, place = ortho_place(lane & 31);
  // the sum carries 2^28, Q's and X's scales
  const float scale = last ? ldexpf(1.f, qexp + ex[0] - 28) : ldexpf(1.f, qexp + ex[0] - ex[1] - 14);
  float* tt = turn[wave];
#pragma unroll
  for (int i = 0; i < 2; ++i)     // rows
#pragma unroll
    for (int j = 0; j < 2; ++j) { // columns
      // this lane: row 32 i + place, columns 32 j + 16 half ..
      float v[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = acc[j][i][e] * scale;
      const bool turned = !last || d.flip;
      if (turned) {
#pragma unroll
        for (int e = 0; e < 16; ++e) tt[place * 33 + 16 * half + e] = v[e];
        wave_lds_sync();
      }
      float u[16];                // column 32 j + place, rows 32 i + 16 half ..
      if (turned) {
#pragma unroll
        for (int e = 0; e < 16; ++e) u[e] = tt[(16 * half + e) * 33 + place];
        wave_lds_sync();
      }
      if (last) {
        const int row = ti * 64 + 32 * i, col = tj * 64 + 32 * j;
        if (d.flip) {
          if (col + place < d.c)
            ortho_out<T, 16>((OrthoGlobal<T>)d.out + (int64_t)(col + place) * d.r + row + 16 * half, d.r - row - 16 * half,
                             d.r % 8 == 0 && (uintptr_t)d.out % 16 == 0, u);
        } else if (row + place < d.r) {
          ortho_out<T, 16>((OrthoGlobal<T>)d.out + (int64_t)(row + place) * d.c + col + 16 * half, d.c - col - 16 * half,
                           d.c % 8 == 0 && (uintptr_t)d.out % 16 == 0, v);
        }
      } else {
        // 16 consecutive k: both halves of one step's fragment
        half_t* fx = ortho_fragment(w.ops + d.x + next, nc * 4, ti * 2 + i, tj * 4 + j * 2 + half);
        half_t* ft = ortho_fragment(w.ops + d.xt + next, nr * 4, tj * 2 + j, ti * 4 + i * 2 + half);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          OrthoParts px, pt;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            ortho_split(px, e, v[8 * h + e]);
            ortho_split(pt, e, u[8 * h + e]);
          }
          ortho_put(fx, (lane & 31) + 32 * h, px);
          ortho_put(ft, (lane & 31) + 32 * h, pt);
          if (d.rest >= 0)
            *(half8*)ortho_third(w.ops + d.rest + (1 - (k & 1)) * (int64_t)nr * nc * 4096, nr * 4, tj * 2 + j,
                                 ti * 4 + i * 2 + half, (lane & 31) + 32 * h) = pt.rest;
        }
      }
    }
}

struct OrthoPlan {
  int64_t halves = 0, parts = 0, gram = 0, upd = 0, slices = 0, partials = 0, sums = 0, count = 0;
  int64_t o_tiles, o_gram, o_upd, o_slices, o_sums, o_parts, o_exps, o_partial, o_ops, bytes;
};

// A tile's k is shared out among workgroups in slices of at least ORTHO_SLICE steps of 16 while a matrix has fewer than
// ORTHO_FILL of them (one slice / 20 / 32 steps: 192 x 4800: 259 / 172 / 165 us; the codec's list 428 / 439 / 410).  Both
// are rules of the matrix alone, and so is the four waves' part: its result is the same in any list (eight waves:
// 128 x 576 108.6 us, with four 110.8; 2048 x 2048 810 us, with four 739).
constexpr int ORTHO_SLICE = 32, ORTHO_FILL = 256;

static int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Offsets and workgroups of every matrix (the totals do not depend on the matrices' order); false: sizes out of range.
static bool ortho_plan(int count, const lic_ortho_mat* mats, OrthoPlan& p, OrthoDesc* d) {
  for (int i = 0; i < count; ++i) {
    const lic_ortho_mat& m = mats[i];
    const bool flip = m.rows > m.cols;
    const int64_t r = flip ? m.cols : m.rows, c = flip ? m.rows : m.cols;
    if (r < 1 || r > 65536 || c > (1 << 24)) return false;
    const int64_t nr = up(r, 64) / 64, nc = up(c, 64) / 64, x = nr * nc * 8192, a = nr * nr * 8192;   // halves, both parts
    OrthoDesc o{m.g, m.out, flip ? m.cs : m.rs, flip ? m.rs : m.cs};
    o.r = (int32_t)r;
    o.c = (int32_t)c;
    o.flip = flip;
    o.step = 2 * x;
    o.x = p.halves;
    o.xt = o.x + x;
    o.a = o.x + 4 * x;
    o.q = o.a + a;
    p.halves = o.q + a;
    o.rest = r <= ORTHO_FINE ? p.halves : -1;
    if (r <= ORTHO_FINE) p.halves += x;   // two copies of half as much as X's two parts
    o.parts0 = (int32_t)p.parts;
    o.gram0 = (int32_t)p.gram;
    o.upd0 = (int32_t)p.upd;
    // slices of k of at least ORTHO_SLICE steps where the tiles of A are few
    const int64_t lower = nr * (nr + 1) / 2, most = ORTHO_FILL / lower;
    o.slices = (int32_t)std::max<int64_t>(1, std::min(nc * 4 / ORTHO_SLICE, most));
    o.slice0 = (int32_t)p.slices;
    o.sum0 = (int32_t)p.sums;
    o.partial0 = (int32_t)p.partials;
    p.slices += lower * o.slices;
    if (o.slices > 1) {
      p.sums += lower;
      p.partials += lower * o.slices;
    }
    p.parts += nr * nc;
    p.gram += lower;
    p.upd += nr * ((nc + 3) / 4);
    // a launch of workgroups of 256 has less than 2^32 threads
    if (p.parts >= 1 << 24 || p.slices >= 1 << 24 || p.upd >= 1 << 24) return false;
    if (d) d[i] = o;
  }
  p.count += count;
  p.o_tiles = up(p.count * (int64_t)sizeof(OrthoDesc), 256);
  p.o_gram = p.o_tiles + up(p.parts * 8, 256);
  p.o_upd = p.o_gram + up(p.gram * 8, 256);
  p.o_slices = p.o_upd + up(p.upd * 8, 256);
  p.o_sums = p.o_slices + up(p.slices * 8, 256);
  p.o_parts = p.o_sums + up(p.sums * 8, 256);
  p.o_exps = p.o_parts + up(p.parts * 8, 256);
  p.o_partial = p.o_exps + up(p.count * 4 * (ORTHO_MAX_STEPS + 1), 256);
  p.o_ops = p.o_partial + p.partials * 4096 * 4;
  p.bytes = p.o_ops + 2 * p.halves;
  return true;
}

// Bounds of a x + b x^3 + c x^5 on [0, most] and of a + b l + c l^2 on [0, most^2]; false where they run away.
static bool ortho_bounds(int steps, const float* co, OrthoBounds& o) {
  const double a = co[0], b = co[1], c = co[2];
  auto at = [&](double x) { return std::fabs(x * (a + x * x * (b + x * x * c))); };
  auto q = [&](double l) { return std::fabs(a + l * (b + l * c)); };
  double most = 1.0, gain = 0.0;
  o.most[0] = 1.0f;
  for (int k = 0; k < steps; ++k) {
    const double l = most * most;
    double qm = std::fmax(q(0), q(l));
    if (c != 0 && -b / (2 * c) > 0 && -b / (2 * c) < l) qm = std::fmax(qm, q(-b / (2 * c)));
    gain = std::fmax(gain, qm);
    int e;
    (void)std::frexp(qm * 1.01, &e);
    o.qexp[k] = qm > 0 ? e : 0;
    double pm = at(most);
    // extrema: a + 3 b u + 5 c u^2 = 0, u = x^2
    const double disc = 9 * b * b - 20 * a * c;
    double u[2] = {-1, -1};
    if (c != 0 && disc >= 0) {
      u[0] = (-3 * b + std::sqrt(disc)) / (10 * c);
      u[1] = (-3 * b - std::sqrt(disc)) / (10 * c);
    } else if (c == 0 && b != 0) {
      u[0] = -a / (3 * b);
    }
    for (double v : u)
      if (v > 0 && v < l) pm = std::fmax(pm, at(std::sqrt(v)));
    most = pm * 1.01;   // rounding errors on top
    if (!(most < 1e9)) return false;
    o.most[k + 1] = (float)most;
  }
  o.gain = (float)(gain * 1.01);
  return true;
}

template <typename T>
static int ortho_run(const OrthoPlan& p, int count, const lic_ortho_mat* mats, int steps, const float* co,
                     const OrthoBounds& bounds, float eps, char* ws, hipStream_t s) {
  OrthoWork w{(OrthoDesc*)ws, (OrthoTile*)(ws + p.o_tiles), (OrthoTile*)(ws + p.o_gram), (OrthoTile*)(ws + p.o_upd),
              (OrthoTile*)(ws + p.o_slices), (OrthoTile*)(ws + p.o_sums), (float*)(ws + p.o_partial),
              (double*)(ws + p.o_parts), (int32_t*)(ws + p.o_exps), (half_t*)(ws + p.o_ops)};
  OrthoPlan q;
  OrthoBatch b;
  std::vector<lic_ortho_mat> sorted(mats, mats + count);   // the longest products start first
  auto shorter = [](const lic_ortho_mat& m) { return std::min(m.rows, m.cols); };
  std::stable_sort(sorted.begin(), sorted.end(),
                   [&](const lic_ortho_mat& x, const lic_ortho_mat& y) { return shorter(x) > shorter(y); });
  mats = sorted.data();
  for (int i = 0; i < count; i += ORTHO_BATCH) {   // offsets run on from batch to batch
    const int n = count - i < ORTHO_BATCH ? count - i : ORTHO_BATCH;
    if (!ortho_plan(n, mats + i, q, b.d)) return fail("orthogonalize: sizes out of range");
    hipLaunchKernelGGL(ortho_norm_kernel<T>, dim3((unsigned)(q.parts - b.d[0].parts0)), dim3(256), 0, s, b, n, i, w);
  }
  hipLaunchKernelGGL(ortho_scale_kernel<T>, dim3((unsigned)p.parts), dim3(256), 0, s, w, bounds, steps, eps);
  for (int k = 0; k < steps; ++k) {
    hipLaunchKernelGGL(ortho_gram_kernel<0>, dim3((unsigned)p.slices), dim3(256), 0, s, w, k, 0.f, 0.f, 0.f, 0);
    if (p.sums) hipLaunchKernelGGL(ortho_sum_kernel, dim3((unsigned)p.sums), dim3(256), 0, s, w);
    hipLaunchKernelGGL(ortho_gram_kernel<1>, dim3((unsigned)p.gram), dim3(256), 0, s, w, k, co[0], co[1], co[2],
                       bounds.qexp[k]);
    hipLaunchKernelGGL(ortho_update_kernel<T>, dim3((unsigned)p.upd), dim3(256), 0, s, w, k, k == steps - 1,
                       bounds.qexp[k]);
  }
  LIC_CHECK_LAUNCH();
  return 0;
}

}  // namespace lic

extern "C" int64_t lic_orthogonalize_workspace(int32_t dtype, int32_t count, const lic_ortho_mat* mats) {
  using namespace lic;
  OrthoPlan p;
  if (count < 0 || (count && !mats) || !ortho_plan(count, mats, p, nullptr)) return -1;
  return p.bytes;
}

extern "C" int lic_orthogonalize(int32_t dtype, int32_t count, const lic_ortho_mat* mats, int32_t steps,
                                 const float* coeffs, float eps, void* ws, int64_t ws_bytes, lic_stream_t stream) {
  using namespace lic;
  if (dtype != LIC_F32 && dtype != LIC_F16 && dtype != LIC_BF16) return fail("orthogonalize: bad dtype");
  if (count < 0 || (count && !mats) || !coeffs) return fail("orthogonalize: null pointer");
  if (steps < 1 || steps > ORTHO_MAX_STEPS) return fail("orthogonalize: steps out of range");
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail("orthogonalize: eps has to be >= 0");
  if (count == 0) return 0;
  OrthoPlan p;
  if (!ortho_plan(count, mats, p, nullptr)) return fail("orthogonalize: sizes out of range");
  for (int i = 0; i < count; ++i)
    if (!mats[i].g || !mats[i].out) return fail("orthogonalize: null matrix");
  OrthoBounds bounds;
  if (!ortho_bounds(steps, coeffs, bounds)) return fail("orthogonalize: the coefficients let the matrices run away");
  if (!ws || (uintptr_t)ws % 256 || ws_bytes < p.bytes)
    return fail("orthogonalize: workspace missing, misaligned or too small");
  hipStream_t s = (hipStream_t)stream;
  if (dtype == LIC_F32) return ortho_run<float>(p, count, mats, steps, coeffs, bounds, eps, (char*)ws, s);
  if (dtype == LIC_F16) return ortho_run<half_t>(p, count, mats, steps, coeffs, bounds, eps, (char*)ws, s);
  return ortho_run<bf16_t>(p, count, mats, steps, coeffs, bounds, eps, (char*)ws, s);
}
