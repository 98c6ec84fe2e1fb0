// Group normalisation with a LeakyReLU on channels-last maps, forward and backward.
//
//   mean, var over one image's pixels and the C / G channels of a group;  rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd;  z = weight xh + bias;  y = z > 0 ? z : slope z
//   dz = dy (z > 0 ? 1 : slope);  dbias = sum dz;  dweight = sum dz xh           (over images and pixels)
//   dx = rstd (weight dz - m1 - xh m2),  m1 / m2 = group means of weight dz / weight dz xh
//
// An image is a flat run of E = pixels * C values.  The kernels walk it in rows of L = lcm(C, 16 bytes) values, so that a
// lane's 16-byte piece holds the same channels in every row whatever C is (position q of a row is channel q mod C); only
// the last piece of an image can be partial.
//
// Statistics are summed in 64 bits.  That is what makes the backward pass' choice of side (z > 0) safe: it is taken from
// the 32-bit z unless |z| is within that value's rounding of zero, and then from z in 64 bits.
#include <hip/hip_runtime.h>
#include <algorithm>
#include "sg2im_hip.h"
#include "launch_count.h"
#include "vecio.h"
#include "ckpt8.h"

namespace sg2im {
namespace gn {

constexpr int THREADS = 256;

struct Params {
  const void* x;
  const signed char* codes;          // instead of x in the backward pass (and written by the forward pass)
  const unsigned char* exps;
  signed char* codes_out;
  unsigned char* exps_out;
  const void* dy;
  const void* gamma;
  const void* beta;
  int param_bf16;
  float slope, eps;
  void* out;                         // y, or dx
  double* stats;                     // [N][G][2] mean, rstd
  void* part;                        // [N][chunks][2][L]: double sums of x, x^2 / float sums of dz, dz xh
  double* chan;                      // [N][C][2] sums of dz, dz xh over the pixels
  float* coef;                       // [N][G][2] m1, m2
  void* dgamma;
  void* dbeta;
  int grad_bf16, accumulate;
  long long E;
  int N, C, G, D, L, rows, chunks, rows_per_chunk, slabs, TV, TP, nblk;
};

// the lane's place: position q0 of its piece in a row, the pixel lane, and this workgroup's image / rows
struct Place { int q0, pl, n, row0, row1; bool on; };
__device__ __forceinline__ Place place_of(const Params& p, int NV, long long block) {
  Place w;
  const int slab = (int)(block % p.slabs);
  long long b = block / p.slabs;
  const int chunk = (int)(b % p.chunks);
  w.n = (int)(b / p.chunks);
  const int v = slab * p.TV + (int)threadIdx.x % p.TV;
  w.pl = (int)threadIdx.x / p.TV;
  w.q0 = v * NV;
  w.on = w.q0 < p.L && w.pl < p.TP;
  w.row0 = chunk * p.rows_per_chunk;
  w.row1 = min(p.rows, w.row0 + p.rows_per_chunk);
  return w;
}

// values of one piece; f(j) only for those of the image (all of them but in its last piece)
template <typename T, int NV>
__device__ __forceinline__ int load_piece(const T* base, long long at, long long E, float (&v)[NV]) {
  if (at + NV <= E) { load_vec<T, NV>(base + at, v); return NV; }
  const int have = at < E ? (int)(E - at) : 0;
  #pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = j < have ? load1(base + at + j) : 0.f;
  return have;
}
template <typename T, int NV>
__device__ __forceinline__ void store_piece(T* base, long long at, int have, const float (&v)[NV]) {
  if (have == NV) { store_vec<T, NV>(base + at, v); return; }
  #pragma unroll
  for (int j = 0; j < NV; ++j) if (j < have) store1(base + at + j, v[j]);
}

// NV decoded values of the 8-bit form; aligned (C % 32 == 0 or C % NV == 0): the piece lies in one block of one pixel
template <int NV>
__device__ __forceinline__ int load_codes(const Params& p, int n, long long at, bool one_block, float (&v)[NV]) {
  const signed char* c = p.codes + (long long)n * p.E;
  const long long pix0 = (long long)n * (p.E / p.C);
  if (one_block && at + NV <= p.E) {
    signed char q[NV];
    __builtin_memcpy(q, c + at, NV);
    const long long pix = at / p.C;
    const float s = c8_scale(p.exps[(pix0 + pix) * p.nblk + (int)(at - pix * p.C) / C8_BLOCK]);
    #pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = c8_decode(q[j], s);
    return NV;
  }
  const int have = at + NV <= p.E ? NV : at < p.E ? (int)(p.E - at) : 0;
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    v[j] = 0.f;
    if (j < have) {
      const long long pix = (at + j) / p.C;
      v[j] = c8_decode(c[at + j], c8_scale(p.exps[(pix0 + pix) * p.nblk + (int)(at + j - pix * p.C) / C8_BLOCK]));
    }
  }
  return have;
}

// ---- forward ------------------------------------------------------------------------------------------------------

// sums of x and x^2 of every position over a chunk of rows
template <typename TX>
__global__ __launch_bounds__(THREADS) void fwd_partial_kernel(const Params p) {
  constexpr int NV = VecOf<TX>::n;
  __shared__ double red[THREADS * NV];
  const Place w = place_of(p, NV, blockIdx.x);
  const TX* x = reinterpret_cast<const TX*>(p.x) + (long long)w.n * p.E;
  double s[NV], q[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) s[j] = q[j] = 0.0;
  if (w.on) {
    #pragma unroll 4
    for (int r = w.row0 + w.pl; r < w.row1; r += p.TP) {
      float v[NV];
      load_piece<TX, NV>(x, (long long)r * p.L + w.q0, p.E, v);      // (what is behind the image reads as 0)
      #pragma unroll
      for (int j = 0; j < NV; ++j) { const double d = v[j]; s[j] += d; q[j] = fma(d, d, q[j]); }
    }
  }
  double* out = reinterpret_cast<double*>(p.part) + ((long long)w.n * p.chunks + w.row0 / p.rows_per_chunk) * 2 * p.L;
  for (int k = 0; k < 2; ++k) {
    if (k) __syncthreads();
    if (w.pl < p.TP) {
      #pragma unroll
      for (int j = 0; j < NV; ++j) red[threadIdx.x * NV + j] = k ? q[j] : s[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.TV * NV; i += THREADS) {
      const int pos = (w.q0 - (int)(threadIdx.x % p.TV) * NV) + i;
      if (pos < p.L) {
        double a = 0.0;
        for (int t = 0; t < p.TP; ++t) a += red[t * p.TV * NV + i];
        out[(long long)k * p.L + pos] = a;
      }
    }
  }
}

__device__ __forceinline__ void block_sum2(double& a, double& b, double (*red)[2]) {
  #pragma unroll
  for (int o = 32; o; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
  const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) { red[wave][0] = a; red[wave][1] = b; }
  __syncthreads();
  a = b = 0.0;
  for (int i = 0; i < waves; ++i) { a += red[i][0]; b += red[i][1]; }
}

// one workgroup per (image, group): the chunks' sums joined in a fixed order
__global__ __launch_bounds__(1024) void fwd_finish_kernel(const Params p) {
  __shared__ double red[16][2];
  const long long b = blockIdx.x;
  const int g = (int)(b % p.G);
  const long long n = b / p.G;
  const int reps = p.L / p.C, per = reps * p.D;
  const double* part = reinterpret_cast<const double*>(p.part) + n * p.chunks * 2 * p.L;
  double s = 0.0, q = 0.0;
  for (long long i = threadIdx.x; i < (long long)p.chunks * per; i += blockDim.x) {
    const long long chunk = i / per;
    const int k = (int)(i - chunk * per), rep = k / p.D;
    const long long at = chunk * 2 * p.L + rep * p.C + g * p.D + (k - rep * p.D);
    s += part[at];
    q += part[at + p.L];
  }
  block_sum2(s, q, red);
  if (threadIdx.x == 0) {
    const double cnt = (double)(p.E / p.C) * p.D, mean = s / cnt;
    double var = q / cnt - mean * mean;
    if (var < 0.0) var = 0.0;                                        // (a NaN stays one)
    p.stats[b * 2] = mean;
    p.stats[b * 2 + 1] = 1.0 / sqrt(var + (double)p.eps);
  }
}

// a position's affine: z = fma(x - m, a, b) with m = float(mean), the difference of the two means in b
struct Affine { float m, a, b; };
__device__ __forceinline__ Affine affine_of(const Params& p, int n, int pos) {
  const int c = pos % p.C;
  const double* st = p.stats + ((long long)n * p.G + c / p.D) * 2;
  const double mean = st[0], rstd = st[1];
  const double ga = p.gamma ? load_param(p.gamma, p.param_bf16, c) : 1.0;
  const double be = p.beta ? load_param(p.beta, p.param_bf16, c) : 0.0;
  Affine f;
  f.m = (float)mean;
  f.a = (float)(ga * rstd);
  f.b = (float)(be + ((double)f.m - mean) * ga * rstd);
  return f;
}

template <typename TX, typename TY>
__global__ __launch_bounds__(THREADS) void fwd_apply_kernel(const Params p) {
  constexpr int NV = VecOf<TX>::n;
  const Place w = place_of(p, NV, blockIdx.x);
  if (!w.on) return;
  const TX* x = reinterpret_cast<const TX*>(p.x) + (long long)w.n * p.E;
  TY* y = reinterpret_cast<TY*>(p.out) + (long long)w.n * p.E;
  Affine f[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) f[j] = affine_of(p, w.n, w.q0 + j);
  #pragma unroll 4
  for (int r = w.row0 + w.pl; r < w.row1; r += p.TP) {
    const long long at = (long long)r * p.L + w.q0;
    float v[NV];
    const int have = load_piece<TX, NV>(x, at, p.E, v);
    #pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float z = fmaf(v[j] - f[j].m, f[j].a, f[j].b);
      v[j] = z > 0.f ? z : z * p.slope;
    }
    store_piece<TY, NV>(y, at, have, v);
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------

// SRC: the type x is read in - float, bf16_s, or signed char for its 8-bit form
template <typename SRC, int NV>
__device__ __forceinline__ int load_x(const Params& p, int n, long long at, bool one_block, float (&v)[NV]) {
  if constexpr (sizeof(SRC) == 1) return load_codes<NV>(p, n, at, one_block, v);
  else return load_piece<SRC, NV>(reinterpret_cast<const SRC*>(p.x) + (long long)n * p.E, at, p.E, v);
}

struct Back { float m, rs, k, a, b, tol; };      // xh = fma(x - m, rs, k);  z = fma(x - m, a, b)
__device__ __forceinline__ Back back_of(const Params& p, int n, int pos) {
  const double* st = p.stats + ((long long)n * p.G + pos % p.C / p.D) * 2;
  const Affine f = affine_of(p, n, pos);
  Back q;
  q.m = f.m; q.a = f.a; q.b = f.b;
  q.rs = (float)st[1];
  q.k = (float)(((double)f.m - st[0]) * st[1]);
  // |z| below this: the rounding of the two products (2^-24 each, of terms as large as b where z is near 0) may decide
  q.tol = p.slope == 1.f ? -1.f : 1e-6f * fabsf(f.b);
  return q;
}
__device__ __forceinline__ bool above_zero(const Params& p, const Back& f, int n, int pos, float x, float z) {
  if (fabsf(z) > f.tol) return z > 0.f;
  const int c = pos % p.C;
  const double* st = p.stats + ((long long)n * p.G + c / p.D) * 2;
  const double ga = p.gamma ? load_param(p.gamma, p.param_bf16, c) : 1.0;
  const double be = p.beta ? load_param(p.beta, p.param_bf16, c) : 0.0;
  return fma((double)x - st[0], ga * st[1], be) > 0.0;
}

// sums of dz and dz xh of every position over a chunk of rows
template <typename SRC, typename TX, typename TY>
__global__ __launch_bounds__(THREADS) void bwd_partial_kernel(const Params p) {
  constexpr int NV = VecOf<TX>::n;
  __shared__ float red[THREADS * NV];
  const Place w = place_of(p, NV, blockIdx.x);
  const TY* dy = reinterpret_cast<const TY*>(p.dy) + (long long)w.n * p.E;
  const bool one_block = p.C % NV == 0;
  float s[NV], q[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) s[j] = q[j] = 0.f;
  if (w.on) {
    Back f[NV];
    #pragma unroll
    for (int j = 0; j < NV; ++j) f[j] = back_of(p, w.n, w.q0 + j);
    #pragma unroll 2
    for (int r = w.row0 + w.pl; r < w.row1; r += p.TP) {
      const long long at = (long long)r * p.L + w.q0;
      float v[NV], g[NV];
      const int have = load_x<SRC, NV>(p, w.n, at, one_block, v);
      load_piece<TY, NV>(dy, at, p.E, g);
      #pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (j >= have) break;
        const float d = v[j] - f[j].m, z = fmaf(d, f[j].a, f[j].b);
        const float dz = above_zero(p, f[j], w.n, w.q0 + j, v[j], z) ? g[j] : g[j] * p.slope;
        s[j] += dz;
        q[j] = fmaf(dz, fmaf(d, f[j].rs, f[j].k), q[j]);
      }
    }
  }
  float* out = reinterpret_cast<float*>(p.part) + ((long long)w.n * p.chunks + w.row0 / p.rows_per_chunk) * 2 * p.L;
  for (int k = 0; k < 2; ++k) {
    if (k) __syncthreads();
    if (w.pl < p.TP) {
      #pragma unroll
      for (int j = 0; j < NV; ++j) red[threadIdx.x * NV + j] = k ? q[j] : s[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.TV * NV; i += THREADS) {
      const int pos = (w.q0 - (int)(threadIdx.x % p.TV) * NV) + i;
      if (pos < p.L) {
        double a = 0.0;
        for (int t = 0; t < p.TP; ++t) a += red[t * p.TV * NV + i];
        out[(long long)k * p.L + pos] = (float)a;
      }
    }
  }
}

// one workgroup per (image, run of whole groups of at least 64 channels or one group): 64 channel lanes x 16 chunk lanes
constexpr int FIN_CH = 64, FIN_LANES = 16;
__global__ __launch_bounds__(FIN_CH * FIN_LANES) void bwd_finish_kernel(const Params p, int groups_per_block) {
  __shared__ double red[FIN_LANES][FIN_CH][2];
  __shared__ double sums[FIN_CH][2];
  const int nb = (p.G + groups_per_block - 1) / groups_per_block;
  const long long n = blockIdx.x / nb;
  const int g0 = (int)(blockIdx.x % nb) * groups_per_block, g1 = min(p.G, g0 + groups_per_block);
  const int c0 = g0 * p.D, c1 = g1 * p.D, cl = threadIdx.x & 63, lane = threadIdx.x >> 6;
  const int reps = p.L / p.C;
  const float* part = reinterpret_cast<const float*>(p.part) + n * p.chunks * 2 * p.L;
  const double inv = 1.0 / ((double)(p.E / p.C) * p.D);
  double t1 = 0.0, t2 = 0.0;                             // (thread cl of lane 0, groups of more than 64 channels)
  for (int cb = c0; cb < c1; cb += FIN_CH) {
    const int c = cb + cl;
    double s = 0.0, q = 0.0;
    if (c < c1)
      for (int i = lane; i < p.chunks * reps; i += FIN_LANES) {
        const int chunk = i / reps;
        const long long at = (long long)chunk * 2 * p.L + (i - chunk * reps) * p.C + c;
        s += part[at];
        q += part[at + p.L];
      }
    red[lane][cl][0] = s; red[lane][cl][1] = q;
    __syncthreads();
    if (lane == 0) {
      s = q = 0.0;
      for (int i = 0; i < FIN_LANES; ++i) { s += red[i][cl][0]; q += red[i][cl][1]; }
      if (c < c1) { p.chan[(n * p.C + c) * 2] = s; p.chan[(n * p.C + c) * 2 + 1] = q; }
      const double ga = c < c1 ? (p.gamma ? load_param(p.gamma, p.param_bf16, c) : 1.0) : 0.0;
      sums[cl][0] = ga * s; sums[cl][1] = ga * q;
      if (c >= c1) sums[cl][0] = sums[cl][1] = 0.0;
    }
    __syncthreads();
    if (p.D <= FIN_CH) {                                 // whole groups in this (only) block of channels
      const int g = g0 + threadIdx.x;
      if (threadIdx.x < FIN_CH && g < g1) {
        double m1 = 0.0, m2 = 0.0;
        for (int d = 0; d < p.D; ++d) { m1 += sums[threadIdx.x * p.D + d][0]; m2 += sums[threadIdx.x * p.D + d][1]; }
        p.coef[(n * p.G + g) * 2] = (float)(m1 * inv);
        p.coef[(n * p.G + g) * 2 + 1] = (float)(m2 * inv);
      }
    } else if (lane == 0) { t1 += sums[cl][0]; t2 += sums[cl][1]; }
    __syncthreads();
  }
  if (p.D > FIN_CH && lane == 0) {
    #pragma unroll
    for (int o = 32; o; o >>= 1) { t1 += __shfl_xor(t1, o); t2 += __shfl_xor(t2, o); }
    if (cl == 0) { p.coef[(n * p.G + g0) * 2] = (float)(t1 * inv); p.coef[(n * p.G + g0) * 2 + 1] = (float)(t2 * inv); }
  }
}

// the parameters' gradients: sums over the images, 32 channels x 8 image lanes per workgroup
__device__ __forceinline__ void param_grads(const Params& p, int block) {
  __shared__ double red[8][32][2];
  const int cl = threadIdx.x & 31, lane = threadIdx.x >> 5, c = block * 32 + cl;
  double s = 0.0, q = 0.0;
  if (c < p.C)
    for (long long n = lane; n < p.N; n += 8) { s += p.chan[(n * p.C + c) * 2]; q += p.chan[(n * p.C + c) * 2 + 1]; }
  red[lane][cl][0] = s; red[lane][cl][1] = q;
  __syncthreads();
  if (lane == 0 && c < p.C) {
    s = q = 0.0;
    for (int i = 0; i < 8; ++i) { s += red[i][cl][0]; q += red[i][cl][1]; }
    if (p.dbeta) store_param(p.dbeta, p.grad_bf16, c, (float)s, p.accumulate);
    if (p.dgamma) store_param(p.dgamma, p.grad_bf16, c, (float)q, p.accumulate);
  }
}

__global__ __launch_bounds__(THREADS) void param_grads_kernel(const Params p) { param_grads(p, blockIdx.x); }

template <typename SRC, typename TX, typename TY>
__global__ __launch_bounds__(THREADS) void bwd_apply_kernel(const Params p, long long main_blocks) {
  constexpr int NV = VecOf<TX>::n;
  if ((long long)blockIdx.x >= main_blocks) { param_grads(p, (int)(blockIdx.x - main_blocks)); return; }
  const Place w = place_of(p, NV, blockIdx.x);
  if (!w.on) return;
  const TY* dy = reinterpret_cast<const TY*>(p.dy) + (long long)w.n * p.E;
  TX* dx = reinterpret_cast<TX*>(p.out) + (long long)w.n * p.E;
  const bool one_block = p.C % NV == 0;
  Back f[NV];
  float ga[NV], m1[NV], m2[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (w.q0 + j) % p.C;
    f[j] = back_of(p, w.n, w.q0 + j);
    ga[j] = p.gamma ? load_param(p.gamma, p.param_bf16, c) : 1.f;
    m1[j] = p.coef[((long long)w.n * p.G + c / p.D) * 2];
    m2[j] = p.coef[((long long)w.n * p.G + c / p.D) * 2 + 1];
  }
  #pragma unroll 2
  for (int r = w.row0 + w.pl; r < w.row1; r += p.TP) {
    const long long at = (long long)r * p.L + w.q0;
    float v[NV], g[NV];
    const int have = load_x<SRC, NV>(p, w.n, at, one_block, v);
    load_piece<TY, NV>(dy, at, p.E, g);
    #pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float d = v[j] - f[j].m, z = fmaf(d, f[j].a, f[j].b), xh = fmaf(d, f[j].rs, f[j].k);
      const float dz = above_zero(p, f[j], w.n, w.q0 + j, v[j], z) ? g[j] : g[j] * p.slope;
      v[j] = f[j].rs * (fmaf(dz, ga[j], -m1[j]) - xh * m2[j]);
    }
    store_piece<TX, NV>(dx, at, have, v);
  }
}

// ---- the 8-bit form on its own ------------------------------------------------------------------------------------

// 8 lanes per block of 32 channels, 4 elements each
template <typename T>
__global__ __launch_bounds__(THREADS) void pack8_kernel(const T* __restrict__ x, long long rows, int C, int nblk, long long ld,
                                                        signed char* __restrict__ codes, unsigned char* __restrict__ exps) {
  const long long blocks = rows * nblk, per = (long long)gridDim.x * (THREADS / 8);
  const int sub = threadIdx.x & 7;
  for (long long b0 = (long long)blockIdx.x * (THREADS / 8); b0 < blocks; b0 += per) {
    const long long b = b0 + (threadIdx.x >> 3);
    const bool on = b < blocks;
    const long long row = on ? b / nblk : 0;
    const int blk = (int)(b - row * nblk), c = blk * C8_BLOCK + sub * 4;
    const int have = on ? min(4, max(0, C - c)) : 0;
    float v[4];
    const T* src = x + row * ld + c;
    if (have == 4) load_vec<T, 4>(src, v);
    else {
      #pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = j < have ? load1(src + j) : 0.f;
    }
    float top = fmaxf(fmaxf(c8_magnitude(v[0]), c8_magnitude(v[1])), fmaxf(c8_magnitude(v[2]), c8_magnitude(v[3])));
    #pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    const int e = c8_exponent(top);
    const float inv = c8_inverse(e);
    signed char q[4];
    #pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = c8_encode(v[j], inv);
    signed char* dst = codes + row * C + c;
    if (have == 4) __builtin_memcpy(dst, q, 4);
    else {
      #pragma unroll
      for (int j = 0; j < 4; ++j) if (j < have) dst[j] = q[j];
    }
    if (on && sub == 0) exps[b] = (unsigned char)e;
  }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void unpack8_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                          long long rows, int C, int nblk, T* __restrict__ out, long long ld) {
  const int pieces = nblk * 8;
  const long long total = rows * pieces;
  for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < total; i += (long long)gridDim.x * THREADS) {
    const long long row = i / pieces;
    const int piece = (int)(i - row * pieces), c = piece * 4, have = min(4, C - c);
    if (have <= 0) continue;
    const float s = c8_scale(exps[row * nblk + (piece >> 3)]);
    const signed char* src = codes + row * C + c;
    T* dst = out + row * ld + c;
    if (have == 4) {
      signed char q[4];
      __builtin_memcpy(q, src, 4);
      float v[4];
      #pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = c8_decode(q[j], s);
      store_vec<T, 4>(dst, v);
    } else {
      for (int j = 0; j < have; ++j) store1(dst + j, c8_decode(src[j], s));
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// How an image is cut: slabs of at most 64 pieces across a row, and chunks of rows so that there are about 2 048
// workgroups (8 per CU) - but never less than four rows per lane, where a workgroup would be all set-up.
bool cut(Params& p, int N, long long hw, int C, int G, int x_bf16) {
  const int nv = x_bf16 ? 8 : 4;
  if ((long long)C * nv > 0x7fffffffLL || hw > 0x7fffffffLL / 2) return false;
  p.N = N; p.C = C; p.G = G; p.D = C / G;
  p.L = nv / gcd(nv, C) * C;
  p.E = hw * C;
  p.nblk = (C + C8_BLOCK - 1) / C8_BLOCK;
  const long long rows = (p.E + p.L - 1) / p.L;
  p.rows = (int)rows;
  const int pieces = p.L / nv;
  p.slabs = (pieces + 63) / 64;
  p.TV = (pieces + p.slabs - 1) / p.slabs;
  if (C % C8_BLOCK == 0) p.TV = (p.TV + 7) / 8 * 8;        // (a block of 32 channels stays inside one wave)
  p.slabs = (pieces + p.TV - 1) / p.TV;
  p.TP = THREADS / p.TV;
  const long long want = std::max(1LL, 2048 / std::max(1LL, (long long)N * p.slabs));
  long long rpc = std::max((rows + want - 1) / want, (long long)p.TP * 4);
  rpc = std::min(rpc, std::max(1LL, rows));
  p.rows_per_chunk = (int)rpc;
  p.chunks = (int)((rows + rpc - 1) / rpc);
  return (long long)N * p.chunks * p.slabs + (C + 31) / 32 <= 0x7fffffffLL && (long long)N * G <= 0x7fffffffLL;
}

size_t part_bytes(const Params& p, bool backward) {
  return (size_t)p.N * p.chunks * 2 * p.L * (backward ? 4 : 8);
}
size_t align16(size_t b) { return (b + 15) / 16 * 16; }
size_t need_bytes(const Params& p, bool backward) {
  if (!backward) return part_bytes(p, false);
  return align16(part_bytes(p, true)) + (size_t)p.N * p.C * 16 + (size_t)p.N * p.G * 8;
}

int status() { return hipGetLastError() == hipSuccess ? SG2IM_OK : SG2IM_ERR_HIP; }
bool type_ok(int t) { return t == 0 || t == 1; }

template <typename TX>
int pack(const void* x, long long rows, int C, int nblk, long long ld, signed char* codes, unsigned char* exps, hipStream_t stream) {
  const long long blocks = (rows * nblk + 31) / 32;
  SG2IM_LAUNCH(pack8_kernel<TX>, dim3((unsigned)std::min(blocks, 1LL << 20)), dim3(THREADS), 0, stream,
               reinterpret_cast<const TX*>(x), rows, C, nblk, ld, codes, exps);
  return status();
}

template <typename TX, typename TY>
void launch_forward(const Params& p, hipStream_t stream) {
  const unsigned blocks = (unsigned)((long long)p.N * p.chunks * p.slabs);
  SG2IM_LAUNCH(fwd_partial_kernel<TX>, dim3(blocks), dim3(THREADS), 0, stream, p);
  const long long per = (long long)p.chunks * (p.L / p.C) * p.D;
  const int threads = per <= 256 ? 64 : per <= 4096 ? 256 : 1024;
  SG2IM_LAUNCH(fwd_finish_kernel, dim3((unsigned)((long long)p.N * p.G)), dim3(threads), 0, stream, p);
  SG2IM_LAUNCH((fwd_apply_kernel<TX, TY>), dim3(blocks), dim3(THREADS), 0, stream, p);
}

template <typename SRC, typename TX, typename TY>
void launch_backward(const Params& p, bool need_dx, bool need_params, hipStream_t stream) {
  const long long blocks = (long long)p.N * p.chunks * p.slabs;
  SG2IM_LAUNCH((bwd_partial_kernel<SRC, TX, TY>), dim3((unsigned)blocks), dim3(THREADS), 0, stream, p);
  const int gpb = p.D >= FIN_CH ? 1 : FIN_CH / p.D;
  SG2IM_LAUNCH(bwd_finish_kernel, dim3((unsigned)((long long)p.N * ((p.G + gpb - 1) / gpb))), dim3(FIN_CH * FIN_LANES), 0,
               stream, p, gpb);
  const int tail = need_params ? (p.C + 31) / 32 : 0;
  if (need_dx)
    SG2IM_LAUNCH((bwd_apply_kernel<SRC, TX, TY>), dim3((unsigned)(blocks + tail)), dim3(THREADS), 0, stream, p, blocks);
  else if (tail)
    SG2IM_LAUNCH(param_grads_kernel, dim3(tail), dim3(THREADS), 0, stream, p);
}

}  // namespace gn
}  // namespace sg2im

using namespace sg2im;
using namespace sg2im::gn;

extern "C" {

size_t sg2im_groupnorm_workspace(int batch, long long hw, int channels, int groups, int x_dtype, int backward) {
  Params p = {};
  if (batch < 0 || hw < 1 || channels < 1 || groups < 1 || channels % groups || !type_ok(x_dtype) ||
      !cut(p, batch, hw, channels, groups, x_dtype)) return 0;
  return std::max((size_t)16, need_bytes(p, backward != 0));
}

int sg2im_groupnorm_act_forward(const void* x, int x_dtype, int batch, long long hw, int channels, int groups, const void* gamma,
                                const void* beta, int param_dtype, float slope, float eps, void* out, int out_dtype,
                                double* stats, signed char* codes, unsigned char* exps, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
  Params p = {};
  if (batch < 0 || hw < 1 || channels < 1 || groups < 1 || channels % groups || !(eps >= 0.f) || !type_ok(x_dtype) ||
      !type_ok(out_dtype) || !type_ok(param_dtype) || (x_dtype == 1 && out_dtype == 0) || !codes != !exps ||
      !cut(p, batch, hw, channels, groups, x_dtype)) return SG2IM_ERR_ARG;
  if (batch == 0) return SG2IM_OK;
  if (!x || !out || !stats || !workspace || workspace_bytes < need_bytes(p, false)) return SG2IM_ERR_ARG;
  p.x = x; p.gamma = gamma; p.beta = beta; p.param_bf16 = param_dtype; p.slope = slope; p.eps = eps; p.out = out;
  p.stats = stats; p.part = workspace;
  if (x_dtype == 0 && out_dtype == 0) launch_forward<float, float>(p, stream);
  else if (x_dtype == 0) launch_forward<float, bf16_s>(p, stream);
  else launch_forward<bf16_s, bf16_s>(p, stream);
  if (status() != SG2IM_OK) return SG2IM_ERR_HIP;
  if (codes) {
    const long long rows = (long long)batch * hw;
    return x_dtype ? pack<bf16_s>(x, rows, channels, p.nblk, channels, codes, exps, stream)
                   : pack<float>(x, rows, channels, p.nblk, channels, codes, exps, stream);
  }
  return SG2IM_OK;
}

int sg2im_groupnorm_act_backward(const void* dy, int dy_dtype, const void* x, int x_dtype, const signed char* codes,
                                 const unsigned char* exps, int batch, long long hw, int channels, int groups,
                                 const void* gamma, const void* beta, int param_dtype, float slope, const double* stats,
                                 void* dx, void* dgamma, void* dbeta, int grad_dtype, int accumulate, void* workspace,
                                 size_t workspace_bytes, hipStream_t stream) {
  Params p = {};
  if (batch < 0 || hw < 1 || channels < 1 || groups < 1 || channels % groups || !type_ok(x_dtype) || !type_ok(dy_dtype) ||
      !type_ok(param_dtype) || !type_ok(grad_dtype) || (x_dtype == 1 && dy_dtype == 0) || !codes != !exps ||
      !cut(p, batch, hw, channels, groups, x_dtype)) return SG2IM_ERR_ARG;
  if (batch > 0 && (!dy || (!x && !codes) || !stats || !workspace || workspace_bytes < need_bytes(p, true))) return SG2IM_ERR_ARG;
  p.dy = dy; p.x = x; p.codes = codes; p.exps = exps; p.gamma = gamma; p.beta = beta; p.param_bf16 = param_dtype;
  p.slope = slope; p.stats = const_cast<double*>(stats); p.out = dx; p.dgamma = dgamma; p.dbeta = dbeta;
  p.grad_bf16 = grad_dtype; p.accumulate = accumulate;
  p.part = workspace;
  p.chan = reinterpret_cast<double*>(reinterpret_cast<char*>(workspace) + align16(part_bytes(p, true)));
  p.coef = reinterpret_cast<float*>(p.chan + (size_t)batch * channels * 2);
  const bool need_params = dgamma || dbeta;
  if (batch == 0) {                                       // no image: the sums are empty (and nothing else is written)
    if (need_params) SG2IM_LAUNCH(param_grads_kernel, dim3((channels + 31) / 32), dim3(THREADS), 0, stream, p);
    return status();
  }
  #define SG2IM_GN_BWD(SRC)                                                                                       \
    if (x_dtype == 0 && dy_dtype == 0) launch_backward<SRC(float), float, float>(p, dx != nullptr, need_params, stream);      \
    else if (x_dtype == 0) launch_backward<SRC(float), float, bf16_s>(p, dx != nullptr, need_params, stream);                 \
    else launch_backward<SRC(bf16_s), bf16_s, bf16_s>(p, dx != nullptr, need_params, stream)
  #define SG2IM_GN_SAME(T) T
  #define SG2IM_GN_CODES(T) signed char
  if (codes) { SG2IM_GN_BWD(SG2IM_GN_CODES); } else { SG2IM_GN_BWD(SG2IM_GN_SAME); }
  #undef SG2IM_GN_BWD
  #undef SG2IM_GN_SAME
  #undef SG2IM_GN_CODES
  return status();
}

int sg2im_pack8(const void* x, int dtype, long long rows, int channels, long long ld, signed char* codes, unsigned char* exps,
                hipStream_t stream) {
  if (rows < 0 || channels < 1 || ld < channels || !type_ok(dtype)) return SG2IM_ERR_ARG;
  if (rows == 0) return SG2IM_OK;
  if (!x || !codes || !exps) return SG2IM_ERR_ARG;
  const int nblk = (channels + C8_BLOCK - 1) / C8_BLOCK;
  return dtype ? pack<bf16_s>(x, rows, channels, nblk, ld, codes, exps, stream)
               : pack<float>(x, rows, channels, nblk, ld, codes, exps, stream);
}

int sg2im_unpack8(const signed char* codes, const unsigned char* exps, long long rows, int channels, void* out, int dtype,
                  long long ld, hipStream_t stream) {
  if (rows < 0 || channels < 1 || ld < channels || !type_ok(dtype)) return SG2IM_ERR_ARG;
  if (rows == 0) return SG2IM_OK;
  if (!out || !codes || !exps) return SG2IM_ERR_ARG;
  const int nblk = (channels + C8_BLOCK - 1) / C8_BLOCK;
  const long long blocks = (rows * nblk * 8 + THREADS - 1) / THREADS;
  const dim3 grid((unsigned)std::min(blocks, 1LL << 20));
  if (dtype) SG2IM_LAUNCH(unpack8_kernel<bf16_s>, grid, dim3(THREADS), 0, stream, codes, exps, rows, channels, nblk, reinterpret_cast<bf16_s*>(out), ld);
  else SG2IM_LAUNCH(unpack8_kernel<float>, grid, dim3(THREADS), 0, stream, codes, exps, rows, channels, nblk, reinterpret_cast<float*>(out), ld);
  return status();
}

}  // extern "C"
