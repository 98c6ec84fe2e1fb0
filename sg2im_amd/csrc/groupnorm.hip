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
//
// From the 8-bit form the backward pass evaluates the same formula with xh and z of the rounded x, but mean and rstd of x: an
// approximation (a step of at most 1/127 of the block's largest value), whose sides are the rounded values' own.  Keeping the forward
// pass' sides would take another 1/8 byte an element.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <type_traits>
#include "sg2im_hip.h"
#include "launch_count.h"
#include "vecio.h"
#include "ckpt8.h"

namespace sg2im {
namespace gn {

// The chunked kernels and the 8-bit form's write past the caches (store_vec_nt).  Alone that is what lets them reach the
// memory's rate (unpack of 134 M values 110 -> 60 us, 32 x 256 x 256 x 64 bfloat16 forward 176 -> 140), and with a reader right
// behind them the two together lose nothing at any size (4 MB 15.5 / 15.5 us, 17 MB 31.6 / 30.6, 134 MB 130 / 126,
// 268 MB 259 / 252): what stays in cache without it is the input, not the output.

constexpr int THREADS = 256;

// (Times beside the kernels: medians of a profile, MI355X.)
struct Params {
  const void* x;
  const signed char* codes;          // instead of x in the backward pass
  const unsigned char* exps;
  signed char* codes_out;            // written by the forward pass
  unsigned char* exps_out;
  const void* dy;
  const void* gamma;
  const void* beta;
  int param_bf16;
  float slope, eps;
  void* out;                         // y, or dx
  double* stats;                     // [N][G][2] mean, rstd
  void* part;                        // [N][chunks][2][L]: double sums of x, x^2 / float sums of dz, dz (x - m)
  double* chan;                      // [N][C][2] sums of dz, dz xh over the pixels
  float* coef;                       // [N][G][2] m1, m2
  void* dgamma;
  void* dbeta;
  int grad_bf16, accumulate;
  long long E;
  int N, C, G, D, L, rows, full_rows, chunks, rows_per_chunk, slabs, TV, TP, nblk;
  int S;                             // slab kernels: positions per workgroup
  int merged;                        // the normalising pass joins the chunks' sums itself
  int span;                          // of the channels of the groups that a slab touches, the most
  int bypass;                        // the backward statistics read dy past the caches
};

template <bool V> struct Flag { static constexpr bool value = V; };

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

// the first `have` elements of a piece, zeros behind them
template <typename T, int NV> __device__ __forceinline__ RawVec<T, NV> load_some(const T* p, int have) {
  if (have >= NV) return load_raw<T, NV>(p);
  RawVec<T, NV> r;
  #pragma unroll
  for (int j = 0; j < NV; ++j) r.h[j] = 0;
  #pragma unroll
  for (int j = 0; j < NV; ++j) if (j < have) __builtin_memcpy(&r.h[j], p + j, sizeof(T));
  return r;
}
template <typename T, int NV> __device__ __forceinline__ void store_some(T* p, int have, const float (&v)[NV]) {
  if (have >= NV) { store_vec<T, NV>(p, v); return; }
  #pragma unroll
  for (int j = 0; j < NV; ++j) if (j < have) store1(p + j, v[j]);
}

// ---- where x comes from: itself, or its 8-bit form ------------------------------------------------------------------
// A source hands out raw pieces (so that several loads are in flight) and turns them into floats.  EVEN: C is a multiple of
// the piece, so a row is a pixel and a piece lies in one block of 32 channels.
template <typename T, int NV, bool EVEN> struct Source {
  typedef RawVec<T, NV> Raw;
  const T* x;
  int q0, L;
  __device__ __forceinline__ Source(const Params& p, int n, int q0_) : x(reinterpret_cast<const T*>(p.x) + (long long)n * p.E + q0_), q0(q0_), L(p.L) {}
  __device__ __forceinline__ Raw load(const Params&, int row) const { return load_raw<T, NV>(x + (long long)row * L); }
  __device__ __forceinline__ Raw load_tail(const Params&, int row, int have) const { return load_some<T, NV>(x + (long long)row * L, have); }
  static __device__ __forceinline__ void values(const Raw& r, float (&v)[NV]) { widen(r, v); }
};
template <int NV> struct RawCodes { signed char q[NV]; unsigned char e[NV]; };
template <int NV> struct RawCodes1 { signed char q[NV]; unsigned char e; };
template <int NV> struct Source<signed char, NV, true> {
  typedef RawCodes1<NV> Raw;
  const signed char* c;
  const unsigned char* e;
  int L;
  __device__ __forceinline__ Source(const Params& p, int n, int q0)
    : c(p.codes + (long long)n * p.E + q0), e(p.exps + (long long)n * (p.E / p.C) * p.nblk + q0 / C8_BLOCK), L(p.L) {}
  __device__ __forceinline__ Raw load(const Params& p, int row) const {
    Raw r;
    __builtin_memcpy(r.q, c + (long long)row * L, NV);
    r.e = e[(long long)row * p.nblk];
    return r;
  }
  __device__ __forceinline__ Raw load_tail(const Params& p, int row, int) const { return load(p, row); }    // (no partial piece)
  static __device__ __forceinline__ void values(const Raw& r, float (&v)[NV]) {
    const float s = c8_scale(r.e);
    #pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = c8_decode(r.q[j], s);
  }
};
template <int NV> struct Source<signed char, NV, false> {
  typedef RawCodes<NV> Raw;
  const signed char* c;
  const unsigned char* e;
  int L, per;                          // pixels per row
  int at[NV];                          // exponent of position j, from the row's first pixel
  __device__ __forceinline__ Source(const Params& p, int n, int q0)
    : c(p.codes + (long long)n * p.E + q0), e(p.exps + (long long)n * (p.E / p.C) * p.nblk), L(p.L), per(p.L / p.C) {
    #pragma unroll
    for (int j = 0; j < NV; ++j) { const int pix = (q0 + j) / p.C; at[j] = pix * p.nblk + (q0 + j - pix * p.C) / C8_BLOCK; }
  }
  __device__ __forceinline__ Raw load(const Params& p, int row) const {
    Raw r;
    __builtin_memcpy(r.q, c + (long long)row * L, NV);
    const unsigned char* er = e + (long long)row * per * p.nblk;
    #pragma unroll
    for (int j = 0; j < NV; ++j) r.e[j] = er[at[j]];
    return r;
  }
  __device__ __forceinline__ Raw load_tail(const Params& p, int row, int have) const {
    if (have >= NV) return load(p, row);
    Raw r;
    const unsigned char* er = e + (long long)row * per * p.nblk;
    #pragma unroll
    for (int j = 0; j < NV; ++j) { r.q[j] = 0; r.e[j] = 127; }
    #pragma unroll
    for (int j = 0; j < NV; ++j) if (j < have) { r.q[j] = c[(long long)row * L + j]; r.e[j] = er[at[j]]; }
    return r;
  }
  static __device__ __forceinline__ void values(const Raw& r, float (&v)[NV]) {
    #pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = c8_decode(r.q[j], c8_scale(r.e[j]));
  }
};

// f over this lane's rows: U at a time where the image has all of a piece, the rest one by one (a partial piece only in the
// image's last row)
template <int U, typename F, typename H>
__device__ __forceinline__ void each_row(const Params& p, const Place& w, int NV, F batch, H tail) {
  const int end = min(w.row1, p.full_rows);
  int r = w.row0 + w.pl;
  for (; r + (U - 1) * p.TP < end; r += U * p.TP) batch(r);
  for (; r < w.row1; r += p.TP) {
    const long long left = p.E - (long long)r * p.L - w.q0;
    if (left > 0) tail(r, left < NV ? (int)left : NV);
  }
}

// ---- forward ------------------------------------------------------------------------------------------------------

// sums over the pixel lanes of two times NV values per thread: out(which, position of the slab, sum); buf: 2 * THREADS * NV
// values.  (One thread per sum: spreading a sum over idle threads, as the slab kernels do, measured 0.5 - 1 us slower here.)
template <typename V, int NV, typename F>
__device__ __forceinline__ void sum_pixel_lanes(const V (&s)[NV], const V (&q)[NV], V* buf, int TV, int TP, int pl, F out) {
  constexpr int HALF = THREADS * NV;
  if (pl < TP) {
    #pragma unroll
    for (int j = 0; j < NV; ++j) {
      buf[threadIdx.x * NV + j] = s[j];
      buf[HALF + threadIdx.x * NV + j] = q[j];
    }
  }
  __syncthreads();
  const int S = TV * NV;
  for (int i = threadIdx.x; i < 2 * S; i += THREADS) {
    const int which = i >= S, at = which * (HALF - S) + i;
    double a = 0.0;
    for (int t = 0; t < TP; ++t) a += buf[t * S + at];
    out(which, i - which * S, a);
  }
}

// sums of x and x^2 of every position over a chunk of rows.  Bound by memory: 32 x 256 x 256 x 64 bfloat16 47 us, 5.7 TB/s (the part
// of x that a producer left in cache comes faster); 32 x 64 x 64 x 64 6.4 us.
template <typename TX>
__global__ __launch_bounds__(THREADS) void fwd_partial_kernel(const Params p) {
  constexpr int NV = VecOf<TX>::n, U = 4;
  __shared__ double buf[2 * THREADS * NV];
  const Place w = place_of(p, NV, blockIdx.x);
  double s[NV], q[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) s[j] = q[j] = 0.0;
  if (w.on) {
    const Source<TX, NV, true> src(p, w.n, w.q0);
    auto add = [&](const RawVec<TX, NV>& raw) {
      float v[NV];
      widen(raw, v);
      #pragma unroll
      for (int j = 0; j < NV; ++j) { const double d = v[j]; s[j] += d; q[j] = fma(d, d, q[j]); }
    };
    each_row<U>(p, w, NV,
      [&](int r) {
        RawVec<TX, NV> raw[U];
        #pragma unroll
        for (int k = 0; k < U; ++k) raw[k] = src.load(p, r + k * p.TP);
        #pragma unroll
        for (int k = 0; k < U; ++k) add(raw[k]);
      },
      [&](int r, int have) { add(src.load_tail(p, r, have)); });          // (what is behind the image reads as 0)
  }
  double* out = reinterpret_cast<double*>(p.part) + ((long long)w.n * p.chunks + w.row0 / p.rows_per_chunk) * 2 * p.L;
  const int base = w.q0 - (int)(threadIdx.x % p.TV) * NV;
  sum_pixel_lanes<double, NV>(s, q, buf, p.TV, p.TP, w.pl, [&](int k, int i, double a) { if (base + i < p.L) out[k * p.L + base + i] = a; });
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

__device__ __forceinline__ void stats_of(const Params& p, double s, double q, double& mean, double& rstd) {
  const double cnt = (double)(p.E / p.C) * p.D;
  mean = s / cnt;
  double var = q / cnt - mean * mean;
  if (var < 0.0) var = 0.0;                                        // (a NaN stays one)
  rstd = 1.0 / sqrt(var + (double)p.eps);
}
__device__ __forceinline__ void write_stats(const Params& p, long long group, double s, double q, double& mean, double& rstd) {
  stats_of(p, s, q, mean, rstd);
  p.stats[group * 2] = mean;
  p.stats[group * 2 + 1] = rstd;
}

// one workgroup per (image, group): the chunks' sums joined in a fixed order.  A launch's latency, 5 us.
__global__ __launch_bounds__(1024) void fwd_finish_kernel(const Params p) {
  __shared__ double red[16][2];
  const long long b = blockIdx.x;
  const int g = (int)(b % p.G);
  const long long n = b / p.G;
  const int reps = p.L / p.C, per = reps * p.D;
  const double* part = reinterpret_cast<const double*>(p.part) + n * p.chunks * 2 * p.L;
  double s = 0.0, q = 0.0;
  for (int i = threadIdx.x; i < p.chunks * per; i += blockDim.x) {
    const int chunk = i / per, k = i - chunk * per, rep = k / p.D;
    const long long at = (long long)chunk * 2 * p.L + rep * p.C + g * p.D + (k - rep * p.D);
    s += part[at];
    q += part[at + p.L];
  }
  block_sum2(s, q, red);
  if (threadIdx.x == 0) { double mean, rstd; write_stats(p, b, s, q, mean, rstd); }
}

// a position's affine: z = fma(x - m, a, b) with m = float(mean), the difference of the two means in b
struct Affine { float m, a, b; };
__device__ __forceinline__ Affine affine_of(const Params& p, int c, double mean, double rstd) {
  const double ga = p.gamma ? load_param(p.gamma, p.param_bf16, c) : 1.0;
  const double be = p.beta ? load_param(p.beta, p.param_bf16, c) : 0.0;
  Affine f;
  f.m = (float)mean;
  f.a = (float)(ga * rstd);
  f.b = (float)(be + ((double)f.m - mean) * ga * rstd);
  return f;
}
__device__ __forceinline__ Affine affine_at(const Params& p, int n, int pos) {
  const int c = pos % p.C;
  const double* st = p.stats + ((long long)n * p.G + c / p.D) * 2;
  return affine_of(p, c, st[0], st[1]);
}

template <int NV>
__device__ __forceinline__ void forward_values(float (&v)[NV], const Affine (&f)[NV], float slope) {
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    const float z = fmaf(v[j] - f[j].m, f[j].a, f[j].b);
    v[j] = z > 0.f ? z : z * slope;
  }
}

// the 8-bit form of a piece (C % 32 == 0: a block is 32 / NV neighbouring lanes of one wave, all of them active)
template <int NV>
__device__ __forceinline__ void write_codes(const Params& p, int n, int row, int q0, const float (&v)[NV]) {
  float top = 0.f;
  #pragma unroll
  for (int j = 0; j < NV; ++j) top = fmaxf(top, c8_magnitude(v[j]));
  #pragma unroll
  for (int o = 1; o < C8_BLOCK / NV; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  const int e = c8_exponent(top);
  const float inv = c8_inverse(e);
  signed char c[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) c[j] = c8_encode(v[j], inv);
  const long long pix = (long long)n * p.rows + row;
  store_bytes_nt<NV>(p.codes_out + pix * p.C + q0, c);
  if (q0 % C8_BLOCK == 0) p.exps_out[pix * p.nblk + q0 / C8_BLOCK] = (unsigned char)e;
}

// Statistics of the groups that the slab's channels [c0, c0 + width) belong to, from the chunks' sums, into st[group][2];
// returns the first group.  Every workgroup of an image does it over again: a few KB from the L2 against a launch of its own
// between the two passes (figures where it is chosen).  A group that reaches over a slab's border is joined by both slabs - in
// the same order, since how many threads share a sum goes by the widest slab - and written by the one that holds its first channel.
constexpr int MERGE_SPAN = 512;
__device__ __forceinline__ int merged_stats(const Params& p, const Place& w, int c0, int width, double* st) {
  __shared__ double red[2 * MERGE_SPAN];
  const int g0 = c0 / p.D, g1 = (min(p.C, c0 + width) - 1) / p.D + 1, span = (g1 - g0) * p.D, parts = max(1, THREADS / p.span);
  const double* part = reinterpret_cast<const double*>(p.part) + (long long)w.n * p.chunks * 2 * p.L + g0 * p.D;
  for (int i = threadIdx.x; i < span * parts; i += THREADS) {
    const int c = i % span;
    double s = 0.0, q = 0.0;
    #pragma unroll 4
    for (int k = i / span; k < p.chunks; k += parts) { s += part[(long long)k * 2 * p.L + c]; q += part[(long long)k * 2 * p.L + p.L + c]; }
    red[2 * i] = s;
    red[2 * i + 1] = q;
  }
  __syncthreads();
  // lanes per group: as many of 1, 4, 16, 64 as its sums keep busy
  const int items = p.D * parts, lanes = items <= 16 ? 1 : items <= 64 ? 4 : items <= 256 ? 16 : 64;
  for (int g = threadIdx.x / lanes; g < g1 - g0; g += THREADS / lanes) {
    double s = 0.0, q = 0.0;
    for (int i = threadIdx.x % lanes; i < items; i += lanes) {
      const int at = i / p.D * span + g * p.D + i % p.D;
      s += red[2 * at];
      q += red[2 * at + 1];
    }
    for (int o = 1; o < lanes; o <<= 1) { s += __shfl_xor(s, o); q += __shfl_xor(q, o); }
    if (threadIdx.x % lanes == 0) stats_of(p, s, q, st[2 * g], st[2 * g + 1]);
  }
  __syncthreads();
  if (w.row0 == 0)
    for (int i = threadIdx.x; i < 2 * (g1 - g0); i += THREADS)
      if ((g0 + i / 2) * p.D >= c0) p.stats[((long long)w.n * p.G + g0) * 2 + i] = st[i];
  return g0;
}

// the normalised, activated map (and x in 8 bits on the way).  Bound by memory: 32 x 128 x 128 x 64 float 44 us, 6.1 TB/s;
// 32 x 256 x 256 x 64 bfloat16 with its codes 150 us, 4.5 TB/s.
template <typename TX, typename TY, bool PACK>
__global__ __launch_bounds__(THREADS) void fwd_apply_kernel(const Params p) {
  constexpr int NV = VecOf<TX>::n, U = 4;
  const Place w = place_of(p, NV, blockIdx.x);
  __shared__ double st[2 * MERGE_SPAN];
  int first = 0;
  if (p.merged) first = merged_stats(p, w, w.q0 - (int)(threadIdx.x % p.TV) * NV, p.TV * NV, st);
  if (!w.on) return;
  const Source<TX, NV, true> src(p, w.n, w.q0);
  TY* y = reinterpret_cast<TY*>(p.out) + (long long)w.n * p.E + w.q0;
  Affine f[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = w.q0 + j, g = c / p.D - first;
    f[j] = p.merged ? affine_of(p, c, st[2 * g], st[2 * g + 1]) : affine_at(p, w.n, c);
  }
  each_row<U>(p, w, NV,
    [&](int r) {
      RawVec<TX, NV> raw[U];
      #pragma unroll
      for (int k = 0; k < U; ++k) raw[k] = src.load(p, r + k * p.TP);
      #pragma unroll
      for (int k = 0; k < U; ++k) {
        float v[NV];
        widen(raw[k], v);
        if constexpr (PACK) write_codes<NV>(p, w.n, r + k * p.TP, w.q0, v);
        forward_values<NV>(v, f, p.slope);
        store_vec_nt<TY, NV>(y + (long long)(r + k * p.TP) * p.L, v);
      }
    },
    [&](int r, int have) {
      float v[NV];
      widen(src.load_tail(p, r, have), v);
      if constexpr (PACK) write_codes<NV>(p, w.n, r, w.q0, v);
      forward_values<NV>(v, f, p.slope);
      store_some<TY, NV>(y + (long long)r * p.L, have, v);
    });
}

// ---- backward -----------------------------------------------------------------------------------------------------

// Which side of the kink: z > 0 with z = fma(x - m, a, b) where |z| is above `tol`, else decided in 64 bits.  Near zero the
// product is as large as b, so 1e-6 |b| covers its three roundings (2^-24 each); a lane uses the largest of its b.
template <int NV>
__device__ __forceinline__ float kink_tolerance(const Affine (&f)[NV], float slope) {
  float t = 0.f;
  #pragma unroll
  for (int j = 0; j < NV; ++j) t = fmaxf(t, fabsf(f[j].b));
  return slope == 1.f ? -1.f : 1e-6f * t;
}
__device__ __forceinline__ bool above_zero_64(const Params& p, int n, int pos, float x) {
  const int c = pos % p.C;
  const double* st = p.stats + ((long long)n * p.G + c / p.D) * 2;
  const double ga = p.gamma ? load_param(p.gamma, p.param_bf16, c) : 1.0;
  const double be = p.beta ? load_param(p.beta, p.param_bf16, c) : 0.0;
  return fma((double)x - st[0], ga * st[1], be) > 0.0;
}
// g: dy -> dz, v: x -> x - m
template <int NV>
__device__ __forceinline__ void back_values(const Params& p, int n, int q0, float (&v)[NV], float (&g)[NV], const Affine (&f)[NV], float tol) {
  float z[NV], low = 3.4e38f;
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    z[j] = fmaf(v[j] - f[j].m, f[j].a, f[j].b);
    low = fminf(low, fabsf(z[j]));
  }
  if (low <= tol) {
    int pos = q0;
    asm volatile("" : "+v"(pos));          // (keeps what only this rare branch reads from being held through the loop)
    #pragma unroll
    for (int j = 0; j < NV; ++j) if (fabsf(z[j]) <= tol) z[j] = above_zero_64(p, n, pos + j, v[j]) ? 1.f : -1.f;
  }
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    g[j] = z[j] > 0.f ? g[j] : g[j] * p.slope;
    v[j] -= f[j].m;
  }
}

// sums of dz and dz (x - m) of every position over a chunk of rows.  Bound by memory: 32 x 256 x 256 x 64 bfloat16 from the 8-bit
// form 80 us, 5.1 TB/s.
template <typename SRC, typename TX, typename TY, bool EVEN>
__global__ __launch_bounds__(THREADS) void bwd_partial_kernel(const Params p) {
  constexpr int NV = VecOf<TX>::n, U = 2;
  __shared__ float buf[2 * THREADS * NV];
  const Place w = place_of(p, NV, blockIdx.x);
  float s[NV], q[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) s[j] = q[j] = 0.f;
  if (w.on) {
    typedef Source<SRC, NV, EVEN> X;
    const X src(p, w.n, w.q0);
    const TY* dy = reinterpret_cast<const TY*>(p.dy) + (long long)w.n * p.E + w.q0;
    Affine f[NV];
    #pragma unroll
    for (int j = 0; j < NV; ++j) f[j] = affine_at(p, w.n, w.q0 + j);
    const float tol = kink_tolerance<NV>(f, p.slope);
    auto add = [&](const typename X::Raw& rx, const RawVec<TY, NV>& rg) {
      float v[NV], g[NV];
      X::values(rx, v);
      widen(rg, g);
      back_values<NV>(p, w.n, w.q0, v, g, f, tol);
      #pragma unroll
      for (int j = 0; j < NV; ++j) { s[j] += g[j]; q[j] = fmaf(g[j], v[j], q[j]); }
    };
    auto rows = [&](auto bypass) {
      each_row<U>(p, w, NV,
        [&](int r) {
          typename X::Raw rx[U];
          RawVec<TY, NV> rg[U];
          #pragma unroll
          for (int k = 0; k < U; ++k) {
            const TY* at = dy + (long long)(r + k * p.TP) * p.L;
            rx[k] = src.load(p, r + k * p.TP);
            if constexpr (bypass.value) load_bytes_nt<sizeof(rg[k])>(&rg[k], at); else rg[k] = load_raw<TY, NV>(at);
          }
          #pragma unroll
          for (int k = 0; k < U; ++k) add(rx[k], rg[k]);
        },
        // (behind the image dy reads as 0, and 0 times a finite x - m adds nothing)
        [&](int r, int have) { add(src.load_tail(p, r, have), load_some<TY, NV>(dy + (long long)r * p.L, have)); });
    };
    if (p.bypass) rows(Flag<true>()); else rows(Flag<false>());
  }
  float* out = reinterpret_cast<float*>(p.part) + ((long long)w.n * p.chunks + w.row0 / p.rows_per_chunk) * 2 * p.L;
  const int base = w.q0 - (int)(threadIdx.x % p.TV) * NV;
  sum_pixel_lanes<float, NV>(s, q, buf, p.TV, p.TP, w.pl, [&](int k, int i, double a) { if (base + i < p.L) out[k * p.L + base + i] = (float)a; });
}

// a channel's sum of dz xh from those of dz (x - m) and dz:  xh = (x - m) rstd + (m - mean) rstd
__device__ __forceinline__ double sum_xh(const double* st, double s, double q) {
  return st[1] * (q + ((double)(float)st[0] - st[0]) * s);
}

// one workgroup per (image, run of whole groups of at least 64 channels or one group): 64 channel lanes x 16 chunk lanes.
// A launch's latency, 5 us.
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
      double ga = 0.0;
      if (c < c1) {
        q = sum_xh(p.stats + (n * p.G + c / p.D) * 2, s, q);
        p.chan[(n * p.C + c) * 2] = s;
        p.chan[(n * p.C + c) * 2 + 1] = q;
        ga = p.gamma ? load_param(p.gamma, p.param_bf16, c) : 1.0;
        sums[cl][0] = ga * s; sums[cl][1] = ga * q;
      } else sums[cl][0] = sums[cl][1] = 0.0;
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

// dx = rstd (weight dz - m1 - xh m2) = a dz - c0 - c1 (x - m) with c1 = rstd^2 m2, c0 = rstd m1 + (m - mean) c1
struct DxCoef { float c0, c1; };
__device__ __forceinline__ DxCoef dx_coef(double mean, double rstd, double m1, double m2) {
  DxCoef k;
  const double c1 = rstd * rstd * m2;
  k.c1 = (float)c1;
  k.c0 = (float)(rstd * m1 + ((double)(float)mean - mean) * c1);
  return k;
}

// dx; the workgroups behind the map's add up the parameters' gradients over the images (a launch less).  Bound by memory:
// 32 x 256 x 256 x 64 bfloat16 from the 8-bit form 117 us, 5.8 TB/s.
template <typename SRC, typename TX, typename TY, bool EVEN>
__global__ __launch_bounds__(THREADS) void bwd_apply_kernel(const Params p, long long main_blocks) {
  constexpr int NV = VecOf<TX>::n, U = 2;
  if ((long long)blockIdx.x >= main_blocks) { param_grads(p, (int)(blockIdx.x - main_blocks)); return; }
  const Place w = place_of(p, NV, blockIdx.x);
  if (!w.on) return;
  typedef Source<SRC, NV, EVEN> X;
  const X src(p, w.n, w.q0);
  const TY* dy = reinterpret_cast<const TY*>(p.dy) + (long long)w.n * p.E + w.q0;
  TX* dx = reinterpret_cast<TX*>(p.out) + (long long)w.n * p.E + w.q0;
  Affine f[NV];
  DxCoef k[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    const long long g = (long long)w.n * p.G + (w.q0 + j) % p.C / p.D;
    f[j] = affine_at(p, w.n, w.q0 + j);
    k[j] = dx_coef(p.stats[g * 2], p.stats[g * 2 + 1], p.coef[g * 2], p.coef[g * 2 + 1]);
  }
  const float tol = kink_tolerance<NV>(f, p.slope);
  auto one = [&](const typename X::Raw& rx, const RawVec<TY, NV>& rg, float (&v)[NV]) {
    float g[NV];
    X::values(rx, v);
    widen(rg, g);
    back_values<NV>(p, w.n, w.q0, v, g, f, tol);
    #pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = fmaf(g[j], f[j].a, -fmaf(v[j], k[j].c1, k[j].c0));
  };
  each_row<U>(p, w, NV,
    [&](int r) {
      typename X::Raw rx[U];
      RawVec<TY, NV> rg[U];
      #pragma unroll
      for (int u = 0; u < U; ++u) { rx[u] = src.load(p, r + u * p.TP); load_bytes_nt<sizeof(rg[u])>(&rg[u], dy + (long long)(r + u * p.TP) * p.L); }
      #pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[NV];
        one(rx[u], rg[u], v);
        store_vec_nt<TX, NV>(dx + (long long)(r + u * p.TP) * p.L, v);
      }
    },
    [&](int r, int have) {
      float v[NV];
      one(src.load_tail(p, r, have), load_some<TY, NV>(dy + (long long)r * p.L, have), v);
      store_some<TX, NV>(dx + (long long)r * p.L, have, v);
    });
}

// ---- small maps: one workgroup keeps a slab of an image ------------------------------------------------------------------
// A slab is S positions of a row that hold whole groups, over all rows of one image.  Its pieces stay in registers (up to
// ITER per thread) between the statistics and their use: x is read once and one launch does the forward pass, one (and one
// for the parameters' sums over the images) the backward pass.  Bound by latency - load, join, join, store: 32 x 4 x 4 x 1024
// float 6.2 us forward, 9.0 + 3.8 backward.

struct Slab { int q0, pl, n, base, TV, TP; bool on; };
__device__ __forceinline__ Slab slab_of(const Params& p, int NV) {
  Slab w;
  w.n = (int)(blockIdx.x / p.slabs);
  w.base = (int)(blockIdx.x % p.slabs) * p.S;
  w.TV = p.S / NV;
  w.TP = blockDim.x / w.TV;
  w.q0 = w.base + (int)(threadIdx.x % w.TV) * NV;
  w.pl = threadIdx.x / w.TV;
  w.on = w.pl < w.TP && w.q0 < p.L;
  return w;
}
__device__ __forceinline__ int piece_length(const Params& p, const Slab& w, int NV, int row) {
  const long long left = w.on && row < p.rows ? p.E - (long long)row * p.L - w.q0 : 0;
  return left >= NV ? NV : left > 0 ? (int)left : 0;
}

// sums of NV values per thread over the pixel lanes, into sums[0 .. S); a thread's values are those of position
// threadIdx % (S / NV) * NV on.  buf: blockDim * NV values of V
template <typename V, int NV>
__device__ __forceinline__ void pixel_sums(const V (&s)[NV], V* buf, double* sums, int pl, int TP, int S) {
  if (pl < TP) {
    #pragma unroll
    for (int j = 0; j < NV; ++j) buf[threadIdx.x * NV + j] = s[j];
  }
  __syncthreads();
  const int B = blockDim.x;
  if (S >= B) {
    for (int i = threadIdx.x; i < S; i += B) {
      double a = 0.0;
      for (int t = 0; t < TP; ++t) a += buf[t * S + i];
      sums[i] = a;
    }
    __syncthreads();
    return;
  }
  // more threads than positions: `parts` threads per position, then one
  const int parts = B / S, i = threadIdx.x % S, part = threadIdx.x / S;
  double a = 0.0;
  if (part < parts) for (int t = part; t < TP; t += parts) a += buf[t * S + i];
  __syncthreads();
  double* mid = reinterpret_cast<double*>(buf);              // (B doubles; buf holds at least that: NV * sizeof(V) >= 8)
  if (part < parts) mid[part * S + i] = a;
  __syncthreads();
  if ((int)threadIdx.x < S) {
    a = 0.0;
    for (int t = 0; t < parts; ++t) a += mid[t * S + threadIdx.x];
    sums[threadIdx.x] = a;
  }
  __syncthreads();
}

// positions of the slab -> groups: f(group, its sums of two arrays); a wave per group
template <typename F>
__device__ __forceinline__ void slab_groups(const Params& p, const Slab& w, const double* s0, const double* s1, F f) {
  const int reps = p.L / p.C, span = min(p.S, p.L - w.base);          // (reps > 1: the slab is the whole row)
  const int g0 = reps > 1 ? 0 : w.base / p.D, ng = reps > 1 ? p.G : span / p.D;
  const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
  for (int g = threadIdx.x >> 6; g < ng; g += waves) {
    double a = 0.0, b = 0.0;
    for (int i = lane; i < p.D * reps; i += 64) {
      const int at = reps > 1 ? (i / p.D) * p.C + g * p.D + i % p.D : g * p.D + i;
      a += s0[at];
      b += s1[at];
    }
    #pragma unroll
    for (int o = 32; o; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
    if (lane == 0) f(g0 + g, a, b);
  }
}

constexpr int SLAB_MAX = 2048;              // positions of a slab (two double arrays in LDS)

// (a piece's second use widens it again: without this its floats would be held from the first one on, at twice the registers)
template <typename R> __device__ __forceinline__ void forget(R& raw) {
  unsigned w[(sizeof(R) + 3) / 4] = {};
  __builtin_memcpy(w, &raw, sizeof(R));
  #pragma unroll
  for (unsigned i = 0; i < sizeof(w) / 4; ++i) asm volatile("" : "+v"(w[i]));
  __builtin_memcpy(&raw, w, sizeof(R));
}

template <typename TX, typename TY, bool PACK, int B, int ITER>
__global__ __launch_bounds__(B) void fwd_slab_kernel(const Params p) {
  constexpr int NV = VecOf<TX>::n;
  __shared__ __attribute__((aligned(16))) double buf[B * NV];
  __shared__ double s0[SLAB_MAX], s1[SLAB_MAX];
  const Slab w = slab_of(p, NV);
  const TX* x = reinterpret_cast<const TX*>(p.x) + (long long)w.n * p.E + w.q0;
  RawVec<TX, NV> raw[ITER];
  #pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int row = w.pl + k * w.TP;
    raw[k] = load_some<TX, NV>(x + (long long)row * p.L, piece_length(p, w, NV, row));
  }
  double s[NV], q[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) s[j] = q[j] = 0.0;
  #pragma unroll
  for (int k = 0; k < ITER; ++k) {
    float v[NV];
    widen(raw[k], v);
    #pragma unroll
    for (int j = 0; j < NV; ++j) { const double d = v[j]; s[j] += d; q[j] = fma(d, d, q[j]); }
    forget(raw[k]);
  }
  const int first = p.L > p.C ? 0 : w.base / p.D;
  if (p.L == p.C && p.D % NV == 0) {
    // a piece lies in one group: a thread has one sum, and a wave joins a group's (32 x 8 x 8 x 512 bfloat16 8.5 us; by
    // positions first, as below, 10.7)
    double a = 0.0, b = 0.0;
    #pragma unroll
    for (int j = 0; j < NV; ++j) { a += s[j]; b += q[j]; }
    buf[threadIdx.x] = a;
    buf[B + threadIdx.x] = b;
    __syncthreads();
    const int lane = threadIdx.x & 63, per = p.D / NV, entries = w.TP * per, ng = min(p.S, p.L - w.base) / p.D;
    for (int g = threadIdx.x >> 6; g < ng; g += B / 64) {
      a = b = 0.0;
      for (int i = lane; i < entries; i += 64) {
        const int t = i / per * w.TV + g * per + i % per;
        a += buf[t];
        b += buf[B + t];
      }
      #pragma unroll
      for (int o = 32; o; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
      if (lane == 0) {
        double mean, rstd;
        write_stats(p, (long long)w.n * p.G + first + g, a, b, mean, rstd);
        s0[g * p.D] = mean;
        s1[g * p.D] = rstd;
      }
    }
  } else {
    pixel_sums<double, NV>(s, buf, s0, w.pl, w.TP, p.S);
    pixel_sums<double, NV>(q, buf, s1, w.pl, w.TP, p.S);
    // (a group's results take the place of its first position, which only its own wave has read)
    slab_groups(p, w, s0, s1, [&](int g, double a, double b) {
      double mean, rstd;
      write_stats(p, (long long)w.n * p.G + g, a, b, mean, rstd);
      s0[(g - first) * p.D] = mean;
      s1[(g - first) * p.D] = rstd;
    });
  }
  __syncthreads();
  if (!w.on) return;
  Affine f[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (w.q0 + j) % p.C, l = (c / p.D - first) * p.D;
    f[j] = affine_of(p, c, s0[l], s1[l]);
  }
  TY* y = reinterpret_cast<TY*>(p.out) + (long long)w.n * p.E + w.q0;
  #pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int row = w.pl + k * w.TP, have = piece_length(p, w, NV, row);
    if (have > 0) {
      float v[NV];
      widen(raw[k], v);
      if constexpr (PACK) write_codes<NV>(p, w.n, row, w.q0, v);
      forward_values<NV>(v, f, p.slope);
      store_some<TY, NV>(y + (long long)row * p.L, have, v);
    }
  }
}

template <typename SRC, typename TX, typename TY, bool EVEN, int B, int ITER>
__global__ __launch_bounds__(B) void bwd_slab_kernel(const Params p) {
  constexpr int NV = VecOf<TX>::n;
  __shared__ __attribute__((aligned(16))) float buf[B * NV];
  __shared__ double s0[SLAB_MAX], s1[SLAB_MAX];
  typedef Source<SRC, NV, EVEN> X;
  const Slab w = slab_of(p, NV);
  const int q0 = w.on ? w.q0 : 0;
  const X src(p, w.n, q0);
  const TY* dy = reinterpret_cast<const TY*>(p.dy) + (long long)w.n * p.E + q0;
  typename X::Raw rx[ITER];
  RawVec<TY, NV> rg[ITER];
  #pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int row = w.pl + k * w.TP, have = piece_length(p, w, NV, row);
    rg[k] = load_some<TY, NV>(dy + (long long)row * p.L, have);
    if (have > 0) rx[k] = src.load_tail(p, row, have);
  }
  Affine f[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) f[j] = affine_at(p, w.n, q0 + j);
  const float tol = kink_tolerance<NV>(f, p.slope);
  float s[NV], q[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) s[j] = q[j] = 0.f;
  #pragma unroll
  for (int k = 0; k < ITER; ++k) {
    if (piece_length(p, w, NV, w.pl + k * w.TP) > 0) {
      float v[NV], g[NV];
      X::values(rx[k], v);
      widen(rg[k], g);
      back_values<NV>(p, w.n, q0, v, g, f, tol);
      #pragma unroll
      for (int j = 0; j < NV; ++j) { s[j] += g[j]; q[j] = fmaf(g[j], v[j], q[j]); }
    }
    forget(rx[k]);
    forget(rg[k]);
  }
  pixel_sums<float, NV>(s, buf, s0, w.pl, w.TP, p.S);
  pixel_sums<float, NV>(q, buf, s1, w.pl, w.TP, p.S);
  // positions -> channels (dz, dz xh) for the parameters; then weighted, for the groups
  const int reps = p.L / p.C, span = min(p.S, p.L - w.base);
  for (int i = threadIdx.x; i < (reps > 1 ? p.C : span); i += B) {
    const int c = reps > 1 ? i : w.base + i;
    const double* st = p.stats + ((long long)w.n * p.G + c / p.D) * 2;
    double a = 0.0, b = 0.0;
    for (int r = 0; r < reps; ++r) { a += s0[r * p.C + i]; b += s1[r * p.C + i]; }
    b = sum_xh(st, a, b);
    const double ga = p.gamma ? load_param(p.gamma, p.param_bf16, c) : 1.0;
    s0[i] = ga * a;
    s1[i] = ga * b;
    for (int r = 1; r < reps; ++r) s0[r * p.C + i] = s1[r * p.C + i] = 0.0;
    if (p.N > 1) {
      p.chan[((long long)w.n * p.C + c) * 2] = a;
      p.chan[((long long)w.n * p.C + c) * 2 + 1] = b;
    } else {
      if (p.dbeta) store_param(p.dbeta, p.grad_bf16, c, (float)a, p.accumulate);
      if (p.dgamma) store_param(p.dgamma, p.grad_bf16, c, (float)b, p.accumulate);
    }
  }
  if (!p.out) return;
  __syncthreads();
  const int first = reps > 1 ? 0 : w.base / p.D;
  const double inv = 1.0 / ((double)(p.E / p.C) * p.D);
  slab_groups(p, w, s0, s1, [&](int g, double a, double b) {
    const double* st = p.stats + ((long long)w.n * p.G + g) * 2;
    const DxCoef d = dx_coef(st[0], st[1], a * inv, b * inv);
    s0[(g - first) * p.D] = d.c0;
    s1[(g - first) * p.D] = d.c1;
  });
  __syncthreads();
  if (!w.on) return;
  DxCoef kc[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int l = ((w.q0 + j) % p.C / p.D - first) * p.D;
    kc[j].c0 = (float)s0[l];
    kc[j].c1 = (float)s1[l];
  }
  TX* dx = reinterpret_cast<TX*>(p.out) + (long long)w.n * p.E + w.q0;
  #pragma unroll
  for (int k = 0; k < ITER; ++k) {
    const int row = w.pl + k * w.TP, have = piece_length(p, w, NV, row);
    if (have > 0) {
      float v[NV], g[NV];
      X::values(rx[k], v);
      widen(rg[k], g);
      back_values<NV>(p, w.n, w.q0, v, g, f, tol);
      #pragma unroll
      for (int j = 0; j < NV; ++j) v[j] = fmaf(g[j], f[j].a, -fmaf(v[j], kc[j].c1, kc[j].c0));
      store_some<TX, NV>(dx + (long long)row * p.L, have, v);
    }
  }
}

// ---- the 8-bit form on its own ------------------------------------------------------------------------------------

// A lane takes one 16-byte piece of x; 4 (bfloat16) or 8 (float) neighbouring lanes make a block of 32 channels.  Pieces are
// numbered along the rows; a workgroup takes a run of U * 256 of them, U in flight per lane.  2097152 x 64 bfloat16: pack 83 us,
// unpack 64 us (4.9 and 6.4 TB/s; with the grid's stride between a lane's pieces and cached stores 98 and 123).
template <typename T>
__global__ __launch_bounds__(THREADS) void pack8_kernel(const T* __restrict__ x, long long rows, int C, int nblk, long long ld,
                                                        signed char* __restrict__ codes, unsigned char* __restrict__ exps) {
  constexpr int NV = VecOf<T>::n, LANES = C8_BLOCK / NV, U = 2;
  const int per_row = nblk * LANES;
  const long long pieces = rows * per_row, step = THREADS;
  for (long long i0 = (long long)blockIdx.x * THREADS * U + threadIdx.x; i0 - threadIdx.x < pieces; i0 += (long long)U * gridDim.x * THREADS) {
    RawVec<T, NV> raw[U];
    long long row[U];
    int c[U];
    #pragma unroll
    for (int k = 0; k < U; ++k) {
      const long long i = i0 + k * step;
      const bool on = i < pieces;
      row[k] = !on ? 0 : pieces <= 0x7fffffffLL ? (long long)((unsigned)i / (unsigned)per_row) : i / per_row;
      c[k] = on ? (int)(i - row[k] * per_row) * NV : C;
      if (C - c[k] >= NV) load_bytes_nt<16>(&raw[k], x + row[k] * ld + c[k]); else raw[k] = load_some<T, NV>(x + row[k] * ld + c[k], C - c[k]);
    }
    #pragma unroll
    for (int k = 0; k < U; ++k) {
      float v[NV], top = 0.f;
      widen(raw[k], v);
      #pragma unroll
      for (int j = 0; j < NV; ++j) top = fmaxf(top, c8_magnitude(v[j]));
      #pragma unroll
      for (int o = 1; o < LANES; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
      const int e = c8_exponent(top), have = C - c[k];
      const float inv = c8_inverse(e);
      signed char q[NV];
      #pragma unroll
      for (int j = 0; j < NV; ++j) q[j] = c8_encode(v[j], inv);
      signed char* dst = codes + row[k] * C + c[k];
      if (have >= NV) store_bytes_nt<NV>(dst, q);
      else {
        #pragma unroll
        for (int j = 0; j < NV; ++j) if (j < have) dst[j] = q[j];
      }
      if (i0 + k * step < pieces && c[k] % C8_BLOCK == 0) exps[row[k] * nblk + c[k] / C8_BLOCK] = (unsigned char)e;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(THREADS) void unpack8_kernel(const signed char* __restrict__ codes, const unsigned char* __restrict__ exps,
                                                          long long rows, int C, int nblk, T* __restrict__ out, long long ld) {
  constexpr int NV = VecOf<T>::n, U = 2;
  const int per_row = (C + NV - 1) / NV;
  const long long pieces = rows * per_row, step = THREADS;
  for (long long i0 = (long long)blockIdx.x * THREADS * U + threadIdx.x; i0 < pieces; i0 += (long long)U * gridDim.x * THREADS) {
    signed char q[U][NV];
    unsigned char e[U];
    long long row[U];
    int c[U];
    #pragma unroll
    for (int k = 0; k < U; ++k) {
      const long long i = i0 + k * step < pieces ? i0 + k * step : i0;      // (behind the end: the first piece once more)
      row[k] = pieces <= 0x7fffffffLL ? (long long)((unsigned)i / (unsigned)per_row) : i / per_row;
      c[k] = (int)(i - row[k] * per_row) * NV;
      const signed char* src = codes + row[k] * C + c[k];
      if (C - c[k] >= NV) __builtin_memcpy(q[k], src, NV);
      else {
        #pragma unroll
        for (int j = 0; j < NV; ++j) q[k][j] = j < C - c[k] ? src[j] : 0;
      }
      e[k] = exps[row[k] * nblk + c[k] / C8_BLOCK];
    }
    #pragma unroll
    for (int k = 0; k < U; ++k) {
      const float s = c8_scale(e[k]);
      float v[NV];
      #pragma unroll
      for (int j = 0; j < NV; ++j) v[j] = c8_decode(q[k][j], s);
      if (C - c[k] >= NV) store_vec_nt<T, NV>(out + row[k] * ld + c[k], v); else store_some<T, NV>(out + row[k] * ld + c[k], C - c[k], v);
    }
  }
}

// workgroups of the two kernels above: U pieces per lane
unsigned piece_blocks(long long pieces) { return (unsigned)std::max(1LL, std::min((pieces + 2 * THREADS - 1) / (2 * THREADS), 1LL << 20)); }

// ---- host ---------------------------------------------------------------------------------------------------------

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

constexpr long long LAUNCH_THREADS = 0xffffffffLL;

// the finish launches: threads of a workgroup per (image, group) forward, workgroups per image backward
int finish_threads(const Params& p) {
  const long long per = (long long)p.chunks * (p.L / p.C) * p.D;
  return per <= 256 ? 64 : per <= 4096 ? 256 : 1024;
}
int groups_per_block(const Params& p) { return p.D >= FIN_CH ? 1 : FIN_CH / p.D; }
int finish_blocks(const Params& p) { return (p.G + groups_per_block(p) - 1) / groups_per_block(p); }

// How an image is cut: slabs of at most 64 pieces across a row, and chunks of rows so that there are about 1 024
// workgroups (4 per CU; 2 048 and more cost 3 % and up on the largest map, in partial sums) - but never less than four rows per lane, where a workgroup would be all set-up.
bool cut(Params& p, int N, long long hw, int C, int G, int x_bf16) {
  const int nv = x_bf16 ? 8 : 4;
  if ((long long)C * nv > 0x7fffffffLL || hw > 0x7fffffffLL / 2) return false;
  p.N = N; p.C = C; p.G = G; p.D = C / G;
  p.L = nv / gcd(nv, C) * C;
  p.E = hw * C;
  p.nblk = (C + C8_BLOCK - 1) / C8_BLOCK;
  const long long rows = (p.E + p.L - 1) / p.L;
  p.rows = (int)rows;
  p.full_rows = (int)(p.E / p.L);
  const int pieces = p.L / nv;
  p.slabs = (pieces + 63) / 64;
  p.TV = (pieces + p.slabs - 1) / p.slabs;
  if (C % C8_BLOCK == 0) p.TV = (p.TV + 7) / 8 * 8;        // (a block of 32 channels stays inside one wave)
  p.slabs = (pieces + p.TV - 1) / p.TV;
  p.TP = THREADS / p.TV;
  const long long want = std::max(1LL, 1024 / std::max(1LL, (long long)N * p.slabs));
  long long rpc = std::max((rows + want - 1) / want, (long long)p.TP * 4);
  rpc = std::min(rpc, std::max(1LL, rows));
  p.rows_per_chunk = (int)rpc;
  p.chunks = (int)((rows + rpc - 1) / rpc);
  // (each launch of one image)
  return ((long long)p.chunks * p.slabs + (C + 31) / 32) * THREADS <= LAUNCH_THREADS && (long long)G * finish_threads(p) <= LAUNCH_THREADS &&
         (long long)finish_blocks(p) * FIN_CH * FIN_LANES <= LAUNCH_THREADS;
}

// A launch has fewer than 2^32 threads, so a batch of many small images takes several: launch(parameters of the images from
// n on, how many, whether they are all).  TX, TY, TP: x; dy; the chunks' sums, OUT: y or dx.
template <typename TX, typename TY, typename OUT, typename TP, typename F>
void over_images(const Params& p, long long blocks_per_image, int threads, F launch) {
  const long long most = std::max(1LL, LAUNCH_THREADS / (blocks_per_image * threads));
  for (long long n = 0; n < p.N; n += most) {
    Params q = p;
    auto move = [](auto*& at, long long bytes) { if (at) at = reinterpret_cast<std::remove_reference_t<decltype(at)>>((unsigned long long)at + bytes); };
    move(q.x, n * p.E * (int)sizeof(TX));
    move(q.codes, n * p.E);
    move(q.exps, n * (p.E / p.C) * p.nblk);
    move(q.codes_out, n * p.E);
    move(q.exps_out, n * (p.E / p.C) * p.nblk);
    move(q.dy, n * p.E * (int)sizeof(TY));
    move(q.out, n * p.E * (int)sizeof(OUT));
    move(q.stats, n * p.G * 2 * 8);
    move(q.part, n * p.chunks * 2 * p.L * (int)sizeof(TP));
    move(q.chan, n * p.C * 2 * 8);
    move(q.coef, n * p.G * 2 * 4);
    const long long count = std::min(most, p.N - n);
    launch(q, count, count == p.N);
  }
}

// The slab kernels' cut: the fewest positions that hold whole groups, whole pieces (`unit`) and 32 channels, more of them where
// a thread would not have its first piece yet and there are workgroups to spare.  False: an image does not fit
// the registers of a workgroup, and the chunked kernels take it.  Slab / chunks, microseconds: few images of small maps gain (float
// forward 32 x 4 x 4 x 512 5.5 / 9.8, 32 x 16 x 16 x 256 9.4 / 14.0; bfloat16 32 x 16 x 16 x 512 11.3 / 18.9; backward 32 x 4 x 4 x 512 float
// 10.5 / 13.3), many images and groups of one or two channels lose (float forward 32 x 8 x 8 x 32 14.7 / 9.3, 2048 x 4 x 4 x 256 51 / 24;
// backward 256 x 16 x 16 x 256 99 / 73); over 214 maps the geometric mean is 2 % apart forward, 1 % backward.
struct SlabPlan { int S, slabs, threads, iter; };
bool slab_plan(const Params& p, int nv, int most, SlabPlan& q) {
  int unit = p.L > p.C ? p.L : p.D / gcd(p.D, nv) * nv;
  if (p.codes_out) unit = unit / gcd(unit, C8_BLOCK) * C8_BLOCK;
  if (unit > SLAB_MAX) return false;
  int S = std::min(p.L, (C8_BLOCK + unit - 1) / unit * unit);
  while (2 * S <= p.L && 2 * S <= SLAB_MAX && (long long)(2 * S / nv) * p.rows <= 256 && (long long)p.N * ((p.L + 2 * S - 1) / (2 * S)) >= 256) S *= 2;
  if (S > SLAB_MAX) return false;
  q.S = S;
  q.slabs = (p.L + S - 1) / S;
  static const int forms[4][2] = {{256, 1}, {256, 4}, {512, 8}, {1024, 4}};      // (as many pieces in registers as spill nothing)
  for (int k = 0; k < 4; ++k) {
    const int tp = forms[k][0] / (S / nv);
    if (k >= 2 && k != most) continue;
    if (tp > 0 && (long long)tp * forms[k][1] >= p.rows) { q.threads = forms[k][0]; q.iter = forms[k][1]; return true; }
  }
  return false;
}

// channels of the groups that a slab of `width` channels touches, the most over the slabs
int slab_span(const Params& p, int width) {
  int most = 0;
  for (int c0 = 0; c0 < p.C; c0 += width) most = std::max(most, ((std::min(p.C, c0 + width) - 1) / p.D + 1 - c0 / p.D) * p.D);
  return most;
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
  SG2IM_LAUNCH(pack8_kernel<TX>, dim3(piece_blocks(rows * nblk * (C8_BLOCK / VecOf<TX>::n))), dim3(THREADS), 0, stream,
               reinterpret_cast<const TX*>(x), rows, C, nblk, ld, codes, exps);
  return status();
}

template <typename TX, typename TY, int B, int ITER>
void forward_slabs(const Params& p0, hipStream_t stream) {
  over_images<TX, char, TY, double>(p0, p0.slabs, B, [&](const Params& p, long long images, bool) {
    const dim3 grid((unsigned)(images * p.slabs));
    if (p.codes_out) SG2IM_LAUNCH((fwd_slab_kernel<TX, TY, true, B, ITER>), grid, dim3(B), 0, stream, p);
    else SG2IM_LAUNCH((fwd_slab_kernel<TX, TY, false, B, ITER>), grid, dim3(B), 0, stream, p);
  });
}
template <typename SRC, typename TX, typename TY, bool EVEN, int B, int ITER>
void backward_slabs(const Params& p0, hipStream_t stream) {
  over_images<TX, TY, TX, float>(p0, p0.slabs, B, [&](const Params& p, long long images, bool) {
    SG2IM_LAUNCH((bwd_slab_kernel<SRC, TX, TY, EVEN, B, ITER>), dim3((unsigned)(images * p.slabs)), dim3(B), 0, stream, p);
  });
}

template <typename TX, typename TY>
void launch_forward(const Params& p0, hipStream_t stream) {
  Params p = p0;
  SlabPlan q;
  if (slab_plan(p, VecOf<TX>::n, 3, q)) {
    p.S = q.S; p.slabs = q.slabs;
    if (q.iter == 1) forward_slabs<TX, TY, 256, 1>(p, stream);
    else if (q.threads == 256) forward_slabs<TX, TY, 256, 4>(p, stream);
    else forward_slabs<TX, TY, 1024, 4>(p, stream);
    return;
  }
  const long long per_image = (long long)p.chunks * p.slabs;
  over_images<TX, char, TY, double>(p, per_image, THREADS, [&](const Params& s, long long images, bool) {
    SG2IM_LAUNCH(fwd_partial_kernel<TX>, dim3((unsigned)(images * per_image)), dim3(THREADS), 0, stream, s);
  });
  // A finish launch, or its work in every workgroup of the normalising pass: by the sums that such a workgroup would join (a
  // slab's groups reach over it by less than a group on either side).  Forward, microseconds, with the launch / without, groups in
  // 32: 544 sums 64 x 64 x 64 x 32 float 20.6 / 18.2; 1088 64 x 32 x 32 x 64 float 15.6 / 12.6; 2176 32 x 64 x 64 x 64 float 21.4 / 19.6,
  // bfloat16 17.9 / 15.9; 4352 (14 maps: 0.91 - 1.09, 0.99 on average) 16 x 128 x 128 x 64 bfloat16 23.7 / 22.6, 32 x 32 x 32 x 128 float
  // 15.8 / 17.3; 8704 32 x 32 x 32 x 256 float 22.7 / 25.6, 16 x 64 x 64 x 128 bfloat16 19.4 / 23.5; 17408 16 x 32 x 32 x 256 float 17.3 / 29.4.
  // (Where the host issues slower than the card works, the launch costs another 2 - 3.)
  p.merged = p.L == p.C && p.chunks <= 64 && p.TV * VecOf<TX>::n + 2 * (p.D - 1) <= MERGE_SPAN && (p.TV * VecOf<TX>::n + 2 * p.D) * p.chunks <= 4608;
  if (p.merged) p.span = slab_span(p, p.TV * VecOf<TX>::n);
  const int threads = finish_threads(p);
  if (!p.merged)
    over_images<TX, char, TY, double>(p, p.G, threads, [&](const Params& s, long long images, bool) {
      SG2IM_LAUNCH(fwd_finish_kernel, dim3((unsigned)(images * s.G)), dim3(threads), 0, stream, s);
    });
  over_images<TX, char, TY, double>(p, per_image, THREADS, [&](const Params& s, long long images, bool) {
    const dim3 blocks((unsigned)(images * per_image));
    if (s.codes_out) SG2IM_LAUNCH((fwd_apply_kernel<TX, TY, true>), blocks, dim3(THREADS), 0, stream, s);
    else SG2IM_LAUNCH((fwd_apply_kernel<TX, TY, false>), blocks, dim3(THREADS), 0, stream, s);
  });
}

template <typename SRC, typename TX, typename TY, bool EVEN>
void launch_backward(const Params& p0, bool need_dx, bool need_params, hipStream_t stream) {
  Params p = p0;
  SlabPlan q;
  constexpr int LARGE = sizeof(TX) == 4 ? 3 : EVEN ? 2 : 0;
  if (slab_plan(p, VecOf<TX>::n, LARGE, q)) {
    p.S = q.S; p.slabs = q.slabs;
    if (q.iter == 1) backward_slabs<SRC, TX, TY, EVEN, 256, 1>(p, stream);
    else if (q.threads == 256) backward_slabs<SRC, TX, TY, EVEN, 256, 4>(p, stream);
    else if constexpr (LARGE == 2) backward_slabs<SRC, TX, TY, EVEN, 512, 8>(p, stream);
    else if constexpr (LARGE == 3) backward_slabs<SRC, TX, TY, EVEN, 1024, 4>(p, stream);
    if (p.N > 1 && need_params) SG2IM_LAUNCH(param_grads_kernel, dim3((p.C + 31) / 32), dim3(THREADS), 0, stream, p);
    return;
  }
  const long long per_image = (long long)p.chunks * p.slabs;
  // Where x and dy together are far beyond the 256 MB cache, one of them can stay in it between the two passes if the other
  // goes past: 32 x 256 x 256 x 64 bfloat16 263 -> 217 us.  Where most of both stays anyway that costs (268 MB: 111 -> 114).
  p.bypass = (double)p.N * p.E * (sizeof(SRC) + sizeof(TY)) > 384e6;
  over_images<TX, TY, TX, float>(p, per_image, THREADS, [&](const Params& s, long long images, bool) {
    SG2IM_LAUNCH((bwd_partial_kernel<SRC, TX, TY, EVEN>), dim3((unsigned)(images * per_image)), dim3(THREADS), 0, stream, s);
  });
  const int gpb = groups_per_block(p), fin = finish_blocks(p);
  over_images<TX, TY, TX, float>(p, fin, FIN_CH * FIN_LANES, [&](const Params& s, long long images, bool) {
    SG2IM_LAUNCH(bwd_finish_kernel, dim3((unsigned)(images * fin)), dim3(FIN_CH * FIN_LANES), 0, stream, s, gpb);
  });
  // (the parameters' sums run over all images: behind the map of a launch that has them all, or in one of their own)
  const int tail = need_params ? (p.C + 31) / 32 : 0;
  bool summed = false;
  if (need_dx)
    over_images<TX, TY, TX, float>(p, per_image + tail, THREADS, [&](const Params& s, long long images, bool all) {
      const long long blocks = images * per_image;
      summed = all;
      SG2IM_LAUNCH((bwd_apply_kernel<SRC, TX, TY, EVEN>), dim3((unsigned)(blocks + (all ? tail : 0))), dim3(THREADS), 0, stream, s, blocks);
    });
  if (tail && !summed) SG2IM_LAUNCH(param_grads_kernel, dim3(tail), dim3(THREADS), 0, stream, p);
}
template <typename TX, typename TY>
void launch_backward(const Params& p, bool need_dx, bool need_params, hipStream_t stream) {
  if (!p.codes) launch_backward<TX, TX, TY, true>(p, need_dx, need_params, stream);        // (the flag is the 8-bit form's alone)
  else if (p.C % VecOf<TX>::n == 0) launch_backward<signed char, TX, TY, true>(p, need_dx, need_params, stream);
  else launch_backward<signed char, TX, TY, false>(p, need_dx, need_params, stream);
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
  const bool fused = codes && channels % C8_BLOCK == 0;     // the 8-bit form on the way, or in a launch of its own
  if (fused) { p.codes_out = codes; p.exps_out = exps; }
  if (x_dtype == 0 && out_dtype == 0) launch_forward<float, float>(p, stream);
  else if (x_dtype == 0) launch_forward<float, bf16_s>(p, stream);
  else launch_forward<bf16_s, bf16_s>(p, stream);
  if (status() != SG2IM_OK) return SG2IM_ERR_HIP;
  if (codes && !fused) {
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
  if (x_dtype == 0 && dy_dtype == 0) launch_backward<float, float>(p, dx != nullptr, need_params, stream);
  else if (x_dtype == 0) launch_backward<float, bf16_s>(p, dx != nullptr, need_params, stream);
  else launch_backward<bf16_s, bf16_s>(p, dx != nullptr, need_params, stream);
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
  const int nv = dtype ? 8 : 4;
  const dim3 grid(piece_blocks(rows * ((channels + nv - 1) / nv)));
  if (dtype) SG2IM_LAUNCH(unpack8_kernel<bf16_s>, grid, dim3(THREADS), 0, stream, codes, exps, rows, channels, nblk, reinterpret_cast<bf16_s*>(out), ld);
  else SG2IM_LAUNCH(unpack8_kernel<float>, grid, dim3(THREADS), 0, stream, codes, exps, rows, channels, nblk, reinterpret_cast<float*>(out), ld);
  return status();
}

}  // extern "C"
