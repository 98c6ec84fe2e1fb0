// Linear layer with bias, LeakyReLU and a residual in its epilogue, and its backward pass, on the matrix cores:
//
//   z = x W^T + b,   y = (z > 0 ? z : slope z) + residual                      x (M, K), W (N, K)
//   dz = dy (z > 0 ? 1 : slope),  dresidual = dy,  db = sum_m dz
//   dx = dz W,   dW = dz^T x        (x, or its 8-bit form)
//
// The forward pass keeps one bit per element, z > 0, for the backward pass.  Next to a bfloat16 x the backward products take dz in
// bfloat16 (a matrix operand is; linear.h at the gate says what that costs), db sums it unrounded.
//
// The products are linear.h's.
#define SG2IM_GEMM_TU 1
#include "linear.h"

namespace sg2im {
namespace lin {

// ---- small forward products ------------------------------------------------------------------------------------------
// Few tiles and a long reduction is a chain of waits: a workgroup takes 16 x 16 outputs and its NW waves split the reduction;
// operands go from memory straight into the matrix instructions' registers (r contiguous: a lane's 16 bytes are its operand
// of v_mfma_f32_16x16x32_bf16, or of four v_mfma_f32_16x16x4_f32), U pieces of each in flight, and the waves' sums meet in
// LDS.  One launch instead of a split product and its join.  (32 x 32 outputs per workgroup were slower: a CU is then
// busy with the products themselves, and few CUs are used.)
typedef float f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 multiply16(const bf16x8& a, const bf16x8& b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 multiply16(const float4& a, const float4& b, f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.x, b.x, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.y, b.y, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.z, b.z, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a.w, b.w, c, 0, 0, 0);
}

// 16 bytes at p.  HALF: p may lie in the middle of a word; the five words that hold them are loaded and moved (a 16-byte load at
// such an address takes several times as long: 16 x 128 x 2001 bfloat16 12.2 us with it, 7.3 so)
template <bool HALF, typename T> __device__ __forceinline__ uint4 piece_at(const T* p) {
  uint4 w;
  if constexpr (!HALF) __builtin_memcpy(&w, p, 16);
  else {
    const unsigned long long at = reinterpret_cast<unsigned long long>(p);
    const unsigned by = (unsigned)at & 2;
    const unsigned* word = reinterpret_cast<const unsigned*>(at - by);
    const unsigned w4 = word[by ? 4 : 3];                            // (a word that holds some of the 16 bytes)
    __builtin_memcpy(&w, word, 16);
    w = make_uint4(__builtin_amdgcn_alignbyte(w.y, w.x, by), __builtin_amdgcn_alignbyte(w.z, w.y, by),
                   __builtin_amdgcn_alignbyte(w.w, w.z, by), __builtin_amdgcn_alignbyte(w4, w.w, by));
  }
  return w;
}

template <typename T, int NW, bool HALF>
__global__ __launch_bounds__(NW * 64) void short_kernel(const Product p) {
  constexpr int NV = Geo<T>::NV, RS = 4 * NV, U = 4, LD = 20;
  __shared__ __attribute__((aligned(16))) float red[NW * 16 * LD];
  const int tiles_j = (p.J + 15) / 16, i0 = (int)(blockIdx.x / tiles_j) * 16, j0 = (int)(blockIdx.x % tiles_j) * 16;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, h = (lane >> 4) * NV;
  const T* a = reinterpret_cast<const T*>(p.a) + (long long)min(i0 + (lane & 15), p.I - 1) * p.lda + h;
  const T* b = reinterpret_cast<const T*>(p.b) + (long long)min(j0 + (lane & 15), p.J - 1) * p.ldb + h;
  const int steps = (p.R + RS - 1) / RS, per = (steps + NW - 1) / NW, s1 = min(steps, (wave + 1) * per), full = min(s1, p.R / RS);
  typedef decltype(operand<32, RC>((const T*)nullptr, 0, 0, 0)) Op;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  int s = wave * per;
  for (; s + U <= full; s += U) {
    Op oa[U], ob[U];
    #pragma unroll
    for (int k = 0; k < U; ++k) {
      oa[k] = __builtin_bit_cast(Op, piece_at<HALF>(a + (long long)(s + k) * RS));
      ob[k] = __builtin_bit_cast(Op, piece_at<HALF>(b + (long long)(s + k) * RS));
    }
    #pragma unroll
    for (int k = 0; k < U; ++k) acc = multiply16(ob[k], oa[k], acc);
  }
  for (; s < s1; ++s) {
    // (a piece over the end: from where it fits, moved into place, as in Feeder)
    const int over = max(0, s * RS + h + NV - p.R);
    const uint4 wa = moved(piece_at<HALF>(a + (long long)s * RS - over), over * (int)sizeof(T) * 8);
    const uint4 wb = moved(piece_at<HALF>(b + (long long)s * RS - over), over * (int)sizeof(T) * 8);
    acc = multiply16(__builtin_bit_cast(Op, wb), __builtin_bit_cast(Op, wa), acc);
  }
  *reinterpret_cast<float4*>(red + (wave * 16 + (lane & 15)) * LD + 4 * (lane >> 4)) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (wave) return;
  const int row = lane >> 2, col = (lane & 3) * 4, i = i0 + row, j = j0 + col;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  #pragma unroll
  for (int w = 0; w < NW; ++w) {
    const float4 u = *reinterpret_cast<const float4*>(red + (w * 16 + row) * LD + col);
    v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w;
  }
  unsigned bits = 0;
  if (i < p.I && j + 4 <= p.J) bits = finish<4>(p, i, j, v);
  else if (i < p.I) {
    if (j < p.J) bits = finish_one(p, i, j, v[0]);
    if (j + 1 < p.J) bits |= finish_one(p, i, j + 1, v[1]) << 1;
    if (j + 2 < p.J) bits |= finish_one(p, i, j + 2, v[2]) << 2;
  }
  if (p.signs) {                                     // (half a word; the upper half of a row's last one may have no columns)
    bits <<= col;
    bits |= __shfl_xor(bits, 1);
    bits |= __shfl_xor(bits, 2);
    unsigned short* half = reinterpret_cast<unsigned short*>(p.signs) + (long long)i * p.sign_words * 2 + j0 / 16;
    if (col == 0 && i < p.I) {
      half[0] = (unsigned short)bits;
      if (j0 + 16 >= p.J && (j0 / 16 & 1) == 0) half[1] = 0;
    }
  }
}

template <typename T, bool HALF>
static int run_short_as(const Product& p, hipStream_t stream) {
  const dim3 grid((unsigned)(((long long)p.I + 15) / 16 * ((p.J + 15) / 16)));
  if (p.R <= 16 * 4 * Geo<T>::NV) SG2IM_LAUNCH((short_kernel<T, 4, HALF>), grid, dim3(256), 0, stream, p);
  else SG2IM_LAUNCH((short_kernel<T, 8, HALF>), grid, dim3(512), 0, stream, p);
  return status();
}
template <typename T>
static int run_short(const Product& p, hipStream_t stream) {
  const auto odd = [](const void* at, long long ld) { return (reinterpret_cast<unsigned long long>(at) & 2) || (ld & 1); };
  if constexpr (sizeof(T) == 2) if (odd(p.a, p.lda) || odd(p.b, p.ldb) || p.R % 2) return run_short_as<T, true>(p, stream);
  return run_short_as<T, false>(p, stream);
}

// ---- dz and the bias gradient -------------------------------------------------------------------------------------

struct ActParams {
  const void* dy; long long ld_dy;
  const unsigned* signs; int sign_words;
  float slope;
  void* dz;                                      // dense, or null: dz is dy
  float* part;                                   // [chunks][N], or null: no bias gradient
  void* db; int db_bf16, accumulate;
  long long M;
  int N, TV, TP, slabs, chunks;
  long long rows_per_chunk;
};

// dz and a chunk of rows' column sums of it in one pass: 32768 x 1024 bfloat16 31 us, 4.5 TB/s, and 4 - 5 us to join the chunks
template <typename TY, typename TZ>
__global__ __launch_bounds__(THREADS) void act_backward_kernel(const ActParams p) {
  constexpr int NV = 8;
  __shared__ float red[THREADS * NV];
  const int slab = blockIdx.x % p.slabs;
  const long long chunk = blockIdx.x / p.slabs;
  const int v = threadIdx.x % p.TV, pl = threadIdx.x / p.TV, c0 = (slab * p.TV + v) * NV;
  const int have = min(NV, p.N - c0);
  const long long m0 = chunk * p.rows_per_chunk, m1 = min(p.M, m0 + p.rows_per_chunk);
  float sum[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) sum[j] = 0.f;
  if (pl < p.TP && have > 0) {
    #pragma unroll 4
    for (long long m = m0 + pl; m < m1; m += p.TP) {
      const TY* src = reinterpret_cast<const TY*>(p.dy) + m * p.ld_dy + c0;
      float g[NV];
      if (have == NV) load_vec<TY, NV>(src, g);
      else {
        #pragma unroll
        for (int j = 0; j < NV; ++j) g[j] = j < have ? load1(src + j) : 0.f;
      }
      if (p.signs) {
        const unsigned bits = p.signs[m * p.sign_words + c0 / 32] >> (c0 % 32);
        #pragma unroll
        for (int j = 0; j < NV; ++j) if (!(bits >> j & 1)) g[j] *= p.slope;
      }
      #pragma unroll
      for (int j = 0; j < NV; ++j) sum[j] += g[j];
      if (p.dz) {
        TZ* dst = reinterpret_cast<TZ*>(p.dz) + m * p.N + c0;
        if (have == NV) store_vec<TZ, NV>(dst, g);
        else {
          #pragma unroll
          for (int j = 0; j < NV; ++j) if (j < have) store1(dst + j, g[j]);
        }
      }
    }
  }
  if (!p.part) return;
  if (pl < p.TP) {
    #pragma unroll
    for (int j = 0; j < NV; ++j) red[threadIdx.x * NV + j] = sum[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.TV * NV; i += THREADS) {
    const int c = slab * p.TV * NV + i;
    if (c < p.N) {
      float a = 0.f;
      for (int t = 0; t < p.TP; ++t) a += red[t * p.TV * NV + i];
      p.part[chunk * p.N + c] = a;
    }
  }
}

// the chunks' sums joined: 32 columns x 32 chunk lanes
__global__ __launch_bounds__(1024) void bias_finish_kernel(const ActParams p) {
  __shared__ double red[32][33];
  const int cl = threadIdx.x & 31, lane = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  double s = 0.0;
  if (c < p.N) {
    #pragma unroll 8
    for (int k = lane; k < p.chunks; k += 32) s += p.part[(long long)k * p.N + c];
  }
  red[lane][cl] = s;
  __syncthreads();
  if (lane == 0 && c < p.N) {
    s = 0.0;
    #pragma unroll
    for (int i = 0; i < 32; ++i) s += red[i][cl];
    store_param(p.db, p.db_bf16, c, (float)s, p.accumulate);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------

constexpr int LD_MAX = 1 << 22;      // (a tile's 256 rows stay within 32-bit byte offsets)
bool ld_ok(long long ld, int cols) { return ld >= cols && ld <= LD_MAX; }
bool sizes_ok(long long rows, int k, int n) { return rows >= 0 && rows <= 0x7fffffffLL - 256 && k >= 1 && n >= 1 && k <= LD_MAX && n <= LD_MAX; }

// The whole reduction in one workgroup's waves, where that is estimated faster than the tiles (whose estimate leaves the
// launch out).  Fitted to 24 shapes; microseconds, tiles / short, rows x n x k:
//   float     342 x 384 x 512 11.8 / 8.5, 1 x 4096 x 4096 27.7 / 14.0, 1000 x 300 x 300 12.6 / 9.6; 342 x 512 x 1152 14.4 / 16.6
//   bfloat16  29 x 23 x 1823 7.0 / 5.0, 1 x 4096 x 4096 11.5 / 8.8, 64 x 2048 x 512 9.2 / 7.6; 512 x 1024 x 1024 9.2 / 18.8
bool short_form(long long I, long long J, long long R, int bf16, const Plan& q) {
  const double tiles = (double)((I + 15) / 16) * (double)((J + 15) / 16), chunks = (double)R / (bf16 ? 64 : 32);
  const double us = 4.5 + tiles / 256 * (0.3 + chunks * (bf16 ? 0.12 : 0.11));
  return R >= (bf16 ? 8 : 4) && us < q.us + (bf16 ? 3.0 : 3.5) && tiles < 65536;   // (a lane's 16 bytes have to fit in a row)
}

// which: 0 forward, 1 dx, 2 dW, as in the workspace query; gated, summed: Product's fields
Plan plan_of(int which, long long rows, int k, int n, int dtype, bool gated, bool summed) {
  if (which == 0) return plan(0, rows, n, k, dtype);
  if (which == 1) return plan(1, rows, k, n, dtype, gated ? GATED[dtype] : 0.0);
  return plan(2, n, k, std::max(1LL, rows), dtype, gated ? GATED[dtype] : summed ? SUMMED[dtype] : 0.0);      // (no row: one empty sum, zeros or what was there)
}

ActParams act_plan(long long rows, int n) {
  ActParams p = {};
  p.M = rows; p.N = n;
  const int pieces = (n + 7) / 8;
  p.slabs = (pieces + 63) / 64;
  p.TV = (pieces + p.slabs - 1) / p.slabs;
  p.TP = THREADS / p.TV;
  const long long want = std::max(1LL, 1024LL / p.slabs);
  p.rows_per_chunk = std::max((rows + want - 1) / want, (long long)p.TP * 4);
  p.chunks = (int)((rows + p.rows_per_chunk - 1) / p.rows_per_chunk);
  return p;
}

}  // namespace lin
}  // namespace sg2im

using namespace sg2im;
using namespace sg2im::lin;

extern "C" {

size_t sg2im_linear_workspace(long long rows, int k, int n, int dtype, int which) {
  if (!sizes_ok(rows, k, n) || !type_ok(dtype) || rows == 0) return 16;
  if (which == 3) return std::max((size_t)16, (size_t)act_plan(rows, n).chunks * n * 4);
  const auto form = [&](bool gated, bool summed) { return plan_of(which, rows, k, n, dtype, gated, summed); };
  if (which == 0) return plan_bytes(form(false, false), rows, n, false);
  if (which == 1) return std::max(plan_bytes(form(false, false), rows, k, false), plan_bytes(form(true, false), rows, k, false));
  return std::max({plan_bytes(form(false, false), n, k, false), plan_bytes(form(true, true), n, k, true), plan_bytes(form(false, true), n, k, true)});
}

int sg2im_linear_backward_act_first(long long rows, int k, int n, int dtype, int gated, int bias, int need_dx, int need_dw) {
  if (!sizes_ok(rows, k, n) || !type_ok(dtype) || (!need_dx && !need_dw) || rows == 0) return 0;
  if (!gated && !(bias && need_dw)) return 0;
  // one pass over dy (and dz to memory) at 4.5 TB/s and its last sum, then plain products; or products that do it themselves
  const double es = dtype ? 2 : 4;
  double first = 8.0 + es * rows * n * (gated ? 2 : 1) / 4.5e6, itself = 0.0;
  const auto us = [&](int which, bool by_itself) { return plan_of(which, rows, k, n, dtype, by_itself && gated, by_itself).us; };
  if (need_dx && gated) { first += us(1, false); itself += us(1, true); }
  if (need_dw) { first += us(2, false); itself += us(2, true); }
  return first < itself;
}

int sg2im_linear_plan(long long rows, int k, int n, int dtype, int which, int gated, int bias, int* tile, int* splits) {
  if (!sizes_ok(rows, k, n) || rows == 0 || !type_ok(dtype) || which < 0 || which > 2 || !tile || !splits) return SG2IM_ERR_ARG;
  const Plan q = plan_of(which, rows, k, n, dtype, gated != 0, bias != 0);
  const bool small = which == 0 && short_form(rows, n, k, dtype, q);
  *tile = small ? 16 : q.tile;
  *splits = small ? 1 : q.splits;
  return SG2IM_OK;
}

int sg2im_linear_forward(const void* x, int dtype, long long ld_x, const void* weight, const void* bias, int bias_dtype,
                         const void* residual, long long ld_res, float slope, void* out, int out_dtype, long long ld_out,
                         unsigned* signs, long long rows, int k, int n, void* workspace, size_t workspace_bytes,
                         hipStream_t stream) {
  if (!sizes_ok(rows, k, n) || !type_ok(dtype) || !type_ok(out_dtype) || !type_ok(bias_dtype) || (dtype == 0 && out_dtype == 1) ||
      !ld_ok(ld_x, k) || ld_out < n || (residual && ld_res < n)) return SG2IM_ERR_ARG;
  if (rows == 0) return SG2IM_OK;
  if (!x || !weight || !out) return SG2IM_ERR_ARG;
  Product p = {};
  p.a = x; p.lda = ld_x; p.b = weight; p.ldb = k; p.I = (int)rows; p.J = n; p.R = k;
  p.bias = bias; p.bias_bf16 = bias_dtype; p.residual = residual; p.ld_res = ld_res; p.slope = slope;
  p.signs = signs; p.sign_words = (n + 31) / 32; p.out = out; p.out_bf16 = out_dtype; p.ld_out = ld_out;
  const Plan q = plan_of(0, rows, k, n, dtype, false, false);
  if (short_form(rows, n, k, dtype, q)) return dtype == 0 ? run_short<float>(p, stream) : run_short<bf16_s>(p, stream);
  return dtype == 0 ? run<float, RC, RC, false, false>(p, q, workspace, workspace_bytes, stream)
                    : run<bf16_s, RC, RC, false, false>(p, q, workspace, workspace_bytes, stream);
}

int sg2im_linear_backward_act(const void* dy, int dy_dtype, long long ld_dy, const unsigned* signs, float slope, void* dz,
                              int dz_dtype, void* dbias, int bias_dtype, int accumulate, long long rows, int n, void* workspace,
                              size_t workspace_bytes, hipStream_t stream) {
  if (!sizes_ok(rows, 1, n) || !type_ok(dy_dtype) || !type_ok(dz_dtype) || !type_ok(bias_dtype) || ld_dy < n ||
      (dy_dtype == 1 && dz_dtype == 0)) return SG2IM_ERR_ARG;
  ActParams p = act_plan(rows, n);
  if (rows > 0 && (!dy || (dbias && (!workspace || workspace_bytes < (size_t)p.chunks * n * 4)))) return SG2IM_ERR_ARG;
  p.dy = dy; p.ld_dy = ld_dy; p.signs = signs; p.sign_words = (n + 31) / 32; p.slope = slope; p.dz = dz;
  p.part = dbias ? reinterpret_cast<float*>(workspace) : nullptr;
  p.db = dbias; p.db_bf16 = bias_dtype; p.accumulate = accumulate;
  const long long blocks = (long long)p.chunks * p.slabs;
  if (blocks * THREADS > 0xffffffffLL) return SG2IM_ERR_ARG;
  if (rows > 0 && (dz || dbias)) {
    const dim3 grid((unsigned)blocks);
    if (dy_dtype == 0 && dz_dtype == 0) SG2IM_LAUNCH((act_backward_kernel<float, float>), grid, dim3(THREADS), 0, stream, p);
    else if (dy_dtype == 0) SG2IM_LAUNCH((act_backward_kernel<float, bf16_s>), grid, dim3(THREADS), 0, stream, p);
    else SG2IM_LAUNCH((act_backward_kernel<bf16_s, bf16_s>), grid, dim3(THREADS), 0, stream, p);
  }
  if (dbias) SG2IM_LAUNCH(bias_finish_kernel, dim3((n + 31) / 32), dim3(1024), 0, stream, p);
  return status();
}

int sg2im_linear_backward_data(const void* dz, int dtype, long long ld_dz, const unsigned* signs, float slope, const void* weight,
                               void* dx, long long ld_dx, long long rows, int k, int n, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
  if (!sizes_ok(rows, k, n) || !type_ok(dtype) || !ld_ok(ld_dz, n) || ld_dx < k) return SG2IM_ERR_ARG;
  if (rows == 0) return SG2IM_OK;
  if (!dz || !weight || !dx) return SG2IM_ERR_ARG;
  Product p = {};
  p.a = dz; p.lda = ld_dz; p.b = weight; p.ldb = k; p.I = (int)rows; p.J = k; p.R = n;
  p.slope = 1.f; p.out = dx; p.out_bf16 = dtype; p.ld_out = ld_dx;
  p.gate = reinterpret_cast<const unsigned char*>(signs); p.gate_ld = (n + 31) / 32 * 4LL; p.gate_slope = slope;
  const Plan q = plan_of(1, rows, k, n, dtype, signs != nullptr, false);
  if (signs) return dtype == 0 ? run<float, RC, RM, true, false>(p, q, workspace, workspace_bytes, stream)
                               : run<bf16_s, RC, RM, true, false>(p, q, workspace, workspace_bytes, stream);
  return dtype == 0 ? run<float, RC, RM, false, false>(p, q, workspace, workspace_bytes, stream)
                    : run<bf16_s, RC, RM, false, false>(p, q, workspace, workspace_bytes, stream);
}

int sg2im_linear_backward_weight(const void* dz, int dtype, long long ld_dz, const unsigned* signs, float slope, const void* x,
                                 long long ld_x, const signed char* codes, const unsigned char* exps, void* dweight,
                                 int dweight_dtype, int accumulate, void* dbias, int bias_dtype, int bias_accumulate, long long rows,
                                 int k, int n, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (!sizes_ok(rows, k, n) || !type_ok(dtype) || !type_ok(dweight_dtype) || !type_ok(bias_dtype) || (dtype == 0 && dweight_dtype == 1) ||
      !ld_ok(ld_dz, n) || !codes != !exps || (!codes && !ld_ok(ld_x, k)) || !dweight) return SG2IM_ERR_ARG;
  if (rows > 0 && (!dz || (!x && !codes))) return SG2IM_ERR_ARG;
  Product p = {};
  p.a = dz; p.lda = ld_dz; p.I = n; p.J = k; p.R = (int)rows;
  p.slope = 1.f; p.out = dweight; p.out_bf16 = dweight_dtype; p.ld_out = k; p.accumulate = accumulate;
  p.gate = reinterpret_cast<const unsigned char*>(signs); p.gate_ld = (n + 31) / 32 * 4LL; p.gate_slope = slope;
  p.sum = dbias; p.sum_bf16 = bias_dtype; p.sum_accumulate = bias_accumulate;
  if (codes) { p.b = codes; p.ldb = k; p.b_exps = exps; p.b_nblk = (k + C8_BLOCK - 1) / C8_BLOCK; }
  else { p.b = x; p.ldb = ld_x; }
  const Plan q = plan_of(2, rows, k, n, dtype, signs != nullptr, dbias != nullptr);
  return run_weight(p, dtype, codes != nullptr, q, workspace, workspace_bytes, stream);
}

}  // extern "C"
