// Linear layer with bias, LeakyReLU and a residual in its epilogue, and its backward pass, on the matrix cores:
//
//   z = x W^T + b,   y = (z > 0 ? z : slope z) + residual                      x (M, K), W (N, K)
//   dz = dy (z > 0 ? 1 : slope),  dresidual = dy,  db = sum_m dz
//   dx = dz W,   dW = dz^T x        (x, or its 8-bit form)
//
// The forward pass keeps one bit per element, z > 0, for the backward pass.
//
// The products are linear.h's.
#define SG2IM_GEMM_TU 1
#include "linear.h"

namespace sg2im {
namespace lin {

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
  if (which == 0) return plan_bytes(plan(0, rows, n, k, dtype), rows, n, false);
  if (which == 1) return std::max(plan_bytes(plan(1, rows, k, n, dtype), rows, k, false), plan_bytes(plan(1, rows, k, n, dtype, GATED[dtype]), rows, k, false));
  return std::max({plan_bytes(plan(2, n, k, rows, dtype), n, k, false), plan_bytes(plan(2, n, k, rows, dtype, GATED[dtype]), n, k, true),
                   plan_bytes(plan(2, n, k, rows, dtype, SUMMED[dtype]), n, k, true)});
}

int sg2im_linear_backward_act_first(long long rows, int k, int n, int dtype, int gated, int bias, int need_dx, int need_dw) {
  if (!sizes_ok(rows, k, n) || !type_ok(dtype) || (!need_dx && !need_dw) || rows == 0) return 0;
  if (!gated && !(bias && need_dw)) return 0;
  // one pass over dy (and dz to memory) at 4.5 TB/s and its last sum, then plain products; or products that do it themselves
  const double es = dtype ? 2 : 4;
  double first = 8.0 + es * rows * n * (gated ? 2 : 1) / 4.5e6, itself = 0.0;
  if (need_dx && gated) { first += plan(1, rows, k, n, dtype).us; itself += plan(1, rows, k, n, dtype, GATED[dtype]).us; }
  if (need_dw) {
    first += plan(2, n, k, rows, dtype).us;
    itself += plan(2, n, k, rows, dtype, gated ? GATED[dtype] : SUMMED[dtype]).us;
  }
  return first < itself;
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
  const Plan q = plan(0, rows, n, k, dtype);
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
  const Plan q = plan(1, rows, k, n, dtype, signs ? GATED[dtype] : 0.0);
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
  const Plan q = plan(2, n, k, std::max(1LL, rows), dtype, signs ? GATED[dtype] : dbias ? SUMMED[dtype] : 0.0);   // (no row: one empty sum, zeros or what was there)
  return run_weight(p, dtype, codes != nullptr, q, workspace, workspace_bytes, stream);
}

}  // extern "C"
