// Linear layer with bias, LeakyReLU and a residual in its epilogue, and its backward pass, on the matrix cores:
//
//   z = x W^T + b,   y = (z > 0 ? z : slope z) + residual                      x (M, K), W (N, K)
//   dz = dy (z > 0 ? 1 : slope),  dresidual = dy,  db = sum_m dz
//   dx = dz W,   dW = dz^T x        (x, or its 8-bit form)
//
// The forward pass keeps one bit per element, z > 0, for the backward pass.
//
// All three products are C[i][j] = sum_r A(i, r) B(j, r); an operand lies in memory either with r contiguous (x and W of
// the forward product, dz of dx) or with i / j contiguous (W of dx, both of dW).  A tile goes from memory through registers
// into LDS in the order it lies in; the operands of v_mfma_f32_32x32x16_bf16 (8 consecutive r of one row per lane) are read
// with ds_read_b128 from the first kind and with the transposing ds_read_b64_tr_b16 from the second.  float32 uses
// v_mfma_f32_32x32x2_f32 on the same tiles.  The operands are swapped (B's tile in the instruction's rows), so that a lane
// ends with four consecutive columns of one output row.
#include <hip/hip_runtime.h>
#include <algorithm>
#include "sg2im_hip.h"
#define SG2IM_GEMM_TU 1
#include "launch_count.h"
#include "vecio.h"
#include "ckpt8.h"

namespace sg2im {
namespace lin {

constexpr int THREADS = 256;
enum { RC = 0, RM = 1, RM8 = 2 };        // r contiguous; i / j contiguous; the same in 8 bits

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Product {
  const void* a; const void* b;
  const unsigned char* b_exps; int b_nblk;       // RM8
  long long lda, ldb;
  int I, J, R;                                   // rows, columns, reduction
  int tiles_j, splits, r_per_split;
  float* part;                                   // [splits][I][J], splits > 1
  // epilogue
  const void* bias; int bias_bf16;
  const void* residual; long long ld_res;
  float slope;
  unsigned* signs; int sign_words;               // [I][sign_words]
  void* out; long long ld_out;
  int accumulate;
};

template <typename T> struct Geo;
template <> struct Geo<bf16_s> { static constexpr int BK = 64, NV = 8; };
template <> struct Geo<float> { static constexpr int BK = 32, NV = 4; };

template <typename T, int ROWS, int MODE> struct Tile {
  static constexpr int BK = Geo<T>::BK, NV = Geo<T>::NV;
  static constexpr int LD = MODE == RC ? BK + NV : ROWS + (sizeof(T) == 2 ? 32 : 8);
  static constexpr int ELEMS = MODE == RC ? ROWS * LD : BK * LD;
  static constexpr int PIECES = ROWS / 32;       // 16-byte pieces per thread
};

struct Piece { unsigned w[4]; };

// one 16-byte piece of `have` valid elements
template <typename T> __device__ __forceinline__ Piece load_piece(const T* p, int have) {
  Piece r;
  if (have >= Geo<T>::NV) { __builtin_memcpy(&r, p, 16); return r; }
  r.w[0] = r.w[1] = r.w[2] = r.w[3] = 0;
  if constexpr (sizeof(T) == 4) {
    for (int j = 0; j < 4; ++j) if (j < have) r.w[j] = reinterpret_cast<const unsigned*>(p)[j];
  } else {
    for (int j = 0; j < 8; ++j) if (j < have) r.w[j >> 1] |= (unsigned)reinterpret_cast<const unsigned short*>(p)[j] << (16 * (j & 1));
  }
  return r;
}
template <typename T> __device__ __forceinline__ Piece load_piece8(const signed char* c, const unsigned char* e, int col, int have) {
  constexpr int NV = Geo<T>::NV;
  Piece r;
  r.w[0] = r.w[1] = r.w[2] = r.w[3] = 0;
  if (have <= 0) return r;
  const float s = c8_scale(e[col / C8_BLOCK]);   // (a piece starts at a multiple of its length: inside one block)
  signed char q[NV];
  if (have >= NV) __builtin_memcpy(q, c + col, NV);
  else for (int j = 0; j < NV; ++j) q[j] = j < have ? c[col + j] : 0;
  float v[NV];
  #pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = c8_decode(q[j], s);
  if constexpr (sizeof(T) == 4) { for (int j = 0; j < 4; ++j) r.w[j] = __float_as_uint(v[j]); }
  else { for (int j = 0; j < 4; ++j) r.w[j] = f32_to_bf16_bits(v[2 * j]) | (unsigned)f32_to_bf16_bits(v[2 * j + 1]) << 16; }
  return r;
}

// memory -> registers: rows [row0, row0 + ROWS) of an operand with `rows` rows, r in [r0, r0 + BK) below r_end
template <typename T, int ROWS, int MODE>
__device__ __forceinline__ void fetch(Piece (&out)[ROWS / 32], const void* src, long long ld, const unsigned char* exps, int nblk,
                                      int row0, int rows, int r0, int r_end) {
  typedef Tile<T, ROWS, MODE> G;
  constexpr int NV = G::NV;
  const int tid = threadIdx.x;
  #pragma unroll
  for (int i = 0; i < G::PIECES; ++i) {
    if constexpr (MODE == RC) {
      const int row = row0 + (tid >> 3) + 32 * i, r = r0 + (tid & 7) * NV;
      out[i] = load_piece<T>(reinterpret_cast<const T*>(src) + (long long)row * ld + r, row < rows ? r_end - r : 0);
    } else {
      constexpr int PR = ROWS / NV;              // pieces per r
      const int r = r0 + tid / PR + (THREADS / PR) * i, col = row0 + tid % PR * NV;
      const int have = r < r_end ? rows - col : 0;
      if constexpr (MODE == RM) out[i] = load_piece<T>(reinterpret_cast<const T*>(src) + (long long)r * ld + col, have);
      else out[i] = load_piece8<T>(reinterpret_cast<const signed char*>(src) + (long long)r * ld, exps + (long long)r * nblk, col, have);
    }
  }
}

template <typename T, int ROWS, int MODE>
__device__ __forceinline__ void stage(T* lds, const Piece (&in)[ROWS / 32]) {
  typedef Tile<T, ROWS, MODE> G;
  const int tid = threadIdx.x;
  #pragma unroll
  for (int i = 0; i < G::PIECES; ++i) {
    T* p;
    if constexpr (MODE == RC) p = lds + ((tid >> 3) + 32 * i) * G::LD + (tid & 7) * G::NV;
    else { constexpr int PR = ROWS / G::NV; p = lds + (tid / PR + (THREADS / PR) * i) * G::LD + tid % PR * G::NV; }
    *reinterpret_cast<uint4*>(p) = make_uint4(in[i].w[0], in[i].w[1], in[i].w[2], in[i].w[3]);
  }
}

// 8 consecutive r (16 step + 8 (lane / 32) ..) of row row0 + lane % 32
template <int ROWS, int MODE>
__device__ __forceinline__ bf16x8 operand(const bf16_s* lds, int row0, int step, int lane) {
  typedef Tile<bf16_s, ROWS, MODE> G;
  if constexpr (MODE == RC) {
    return *reinterpret_cast<const bf16x8*>(lds + (row0 + (lane & 31)) * G::LD + 16 * step + 8 * (lane >> 5));
  } else {
    // the 16 lanes of a group pass 4 rows x 4 pieces of 4 and receive 4 consecutive r of one column each
    typedef __attribute__((address_space(3))) bf16x4* LdsPtr;
    const int p = lane & 15, g = lane >> 4;
    const bf16_s* at = lds + (16 * step + 8 * (g >> 1) + (p >> 2)) * G::LD + row0 + 16 * (g & 1) + 4 * (p & 3);
    const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LdsPtr)at);
    const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LdsPtr)(at + 4 * G::LD));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
// float32: r = 8 step + 4 (lane / 32) .. + 3 of row row0 + lane % 32, one per matrix instruction
template <int ROWS, int MODE>
__device__ __forceinline__ float4 operand(const float* lds, int row0, int step, int lane) {
  typedef Tile<float, ROWS, MODE> G;
  const int r = 8 * step + 4 * (lane >> 5);
  if constexpr (MODE == RC) return *reinterpret_cast<const float4*>(lds + (row0 + (lane & 31)) * G::LD + r);
  else {
    const float* p = lds + r * G::LD + row0 + (lane & 31);
    return make_float4(p[0], p[G::LD], p[2 * G::LD], p[3 * G::LD]);
  }
}
__device__ __forceinline__ f32x16 multiply(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 multiply(const float4& a, const float4& b, f32x16 c) {
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.x, b.x, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.y, b.y, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.z, b.z, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a.w, b.w, c, 0, 0, 0);
}

// four consecutive columns of output row i; returns their z > 0 bits
template <typename TO>
__device__ __forceinline__ unsigned finish4(const Product& p, int i, int j, float (&v)[4]) {
  unsigned bits = 0;
  const int have = min(4, p.J - j);
  if (i >= p.I || have <= 0) return 0;
  #pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (p.bias && t < have) v[t] += load_param(p.bias, p.bias_bf16, j + t);
    if (v[t] > 0.f && t < have) bits |= 1u << t;
    v[t] = v[t] > 0.f ? v[t] : v[t] * p.slope;
  }
  TO* out = reinterpret_cast<TO*>(p.out) + (long long)i * p.ld_out + j;
  const TO* res = p.residual ? reinterpret_cast<const TO*>(p.residual) + (long long)i * p.ld_res + j : p.accumulate ? out : nullptr;
  if (have == 4) {
    if (res) {
      float r[4];
      load_vec<TO, 4>(res, r);
      #pragma unroll
      for (int t = 0; t < 4; ++t) v[t] += r[t];
    }
    store_vec<TO, 4>(out, v);
  } else {
    for (int t = 0; t < have; ++t) store1(out + t, res ? v[t] + load1(res + t) : v[t]);
  }
  return bits;
}

template <typename T, typename TO, int BM, int BN, int AMODE, int BMODE>
__global__ __launch_bounds__(THREADS) void product_kernel(const Product p) {
  typedef Tile<T, BM, AMODE> GA;
  typedef Tile<T, BN, BMODE> GB;
  constexpr int BK = GA::BK, TI = BM / 64, TJ = BN / 64, STEPS = sizeof(T) == 2 ? BK / 16 : BK / 8;
  __shared__ __attribute__((aligned(16))) T lds_a[GA::ELEMS], lds_b[GB::ELEMS];
  const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
  const int i0 = tile / p.tiles_j * BM, j0 = tile % p.tiles_j * BN;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wi = (wave >> 1) * (BM / 2), wj = (wave & 1) * (BN / 2);
  const int r_begin = split * p.r_per_split, r_end = min(p.R, r_begin + p.r_per_split);
  f32x16 acc[TI][TJ];
  #pragma unroll
  for (int a = 0; a < TI; ++a)
    #pragma unroll
    for (int b = 0; b < TJ; ++b)
      #pragma unroll
      for (int v = 0; v < 16; ++v) acc[a][b][v] = 0.f;
  Piece pa[GA::PIECES], pb[GB::PIECES];
  fetch<T, BM, AMODE>(pa, p.a, p.lda, nullptr, 0, i0, p.I, r_begin, r_end);
  fetch<T, BN, BMODE>(pb, p.b, p.ldb, p.b_exps, p.b_nblk, j0, p.J, r_begin, r_end);
  for (int r = r_begin; r < r_end; r += BK) {
    __syncthreads();
    stage<T, BM, AMODE>(lds_a, pa);
    stage<T, BN, BMODE>(lds_b, pb);
    __syncthreads();
    if (r + BK < r_end) {
      fetch<T, BM, AMODE>(pa, p.a, p.lda, nullptr, 0, i0, p.I, r + BK, r_end);
      fetch<T, BN, BMODE>(pb, p.b, p.ldb, p.b_exps, p.b_nblk, j0, p.J, r + BK, r_end);
    }
    #pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      decltype(operand<BM, AMODE>(lds_a, 0, 0, 0)) fa[TI], fb[TJ];
      #pragma unroll
      for (int a = 0; a < TI; ++a) fa[a] = operand<BM, AMODE>(lds_a, wi + 32 * a, s, lane);
      #pragma unroll
      for (int b = 0; b < TJ; ++b) fb[b] = operand<BN, BMODE>(lds_b, wj + 32 * b, s, lane);
      #pragma unroll
      for (int a = 0; a < TI; ++a)
        #pragma unroll
        for (int b = 0; b < TJ; ++b) acc[a][b] = multiply(fb[b], fa[a], acc[a][b]);
    }
  }
  #pragma unroll
  for (int a = 0; a < TI; ++a) {
    const int i = i0 + wi + 32 * a + (lane & 31);
    #pragma unroll
    for (int b = 0; b < TJ; ++b) {
      const int jb = j0 + wj + 32 * b;
      unsigned bits = 0;
      #pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int j = jb + 8 * q + 4 * (lane >> 5);
        float v[4] = {acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]};
        if (p.splits > 1) {
          if (i < p.I) {
            float* out = p.part + ((long long)split * p.I + i) * p.J + j;
            if (j + 4 <= p.J) store_vec<float, 4>(out, v);
            else for (int t = 0; t < 4; ++t) if (j + t < p.J) out[t] = v[t];
          }
        } else {
          bits |= finish4<TO>(p, i, j, v) << (8 * q + 4 * (lane >> 5));
        }
      }
      if (p.splits == 1 && p.signs) {
        bits |= __shfl_xor(bits, 32);
        if (lane < 32 && i < p.I && jb < p.J) p.signs[(long long)i * p.sign_words + jb / 32] = bits;
      }
    }
  }
}

// the splits' sums joined in a fixed order: 8 lanes of 4 columns make a word of signs
template <typename TO>
__global__ __launch_bounds__(THREADS) void join_kernel(const Product p) {
  const int words = (p.J + 31) / 32;
  const long long pieces = (long long)p.I * words * 8, plane = (long long)p.I * p.J;
  for (long long b0 = (long long)blockIdx.x * THREADS; b0 < pieces; b0 += (long long)gridDim.x * THREADS) {
    const long long at = b0 + threadIdx.x;
    const long long word = at >> 3;
    const int i = (int)(word / words), w = (int)(word - (long long)i * words), j = w * 32 + (int)(at & 7) * 4;
    unsigned bits = 0;
    if (at < pieces && j < p.J) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      const float* src = p.part + (long long)i * p.J + j;
      for (int s = 0; s < p.splits; ++s, src += plane) {
        float u[4] = {0.f, 0.f, 0.f, 0.f};
        if (j + 4 <= p.J) load_vec<float, 4>(src, u);
        else for (int t = 0; t < 4; ++t) if (j + t < p.J) u[t] = src[t];
        #pragma unroll
        for (int t = 0; t < 4; ++t) v[t] += u[t];
      }
      bits = finish4<TO>(p, i, j, v) << (4 * (int)(at & 7));
    }
    if (p.signs) {
      #pragma unroll
      for (int o = 1; o < 8; o <<= 1) bits |= __shfl_xor(bits, o);
      if (at < pieces && (at & 7) == 0) p.signs[(long long)i * p.sign_words + w] = bits;
    }
  }
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
        else for (int j = 0; j < have; ++j) store1(dst + j, g[j]);
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

__global__ __launch_bounds__(THREADS) void bias_finish_kernel(const ActParams p) {
  __shared__ double red[8][32];
  const int cl = threadIdx.x & 31, lane = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  double s = 0.0;
  if (c < p.N) for (int k = lane; k < p.chunks; k += 8) s += p.part[(long long)k * p.N + c];
  red[lane][cl] = s;
  __syncthreads();
  if (lane == 0 && c < p.N) {
    s = 0.0;
    for (int i = 0; i < 8; ++i) s += red[i][cl];
    store_param(p.db, p.db_bf16, c, (float)s, p.accumulate);
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------

int status() { return hipGetLastError() == hipSuccess ? SG2IM_OK : SG2IM_ERR_HIP; }
bool type_ok(int t) { return t == 0 || t == 1; }

struct Plan { int tile, splits, r_per_split; };

// 128 x 128 tiles where they fill the card, 64 x 64 below; the reduction is split where even those leave CUs idle.
Plan plan(long long I, long long J, long long R, int bf16) {
  const int bk = bf16 ? 64 : 32;
  auto tiles = [&](int t) { return ((I + t - 1) / t) * ((J + t - 1) / t); };
  Plan q;
  q.tile = tiles(128) >= 256 ? 128 : 64;
  const long long steps = (R + bk - 1) / bk, n = std::max(1LL, tiles(q.tile));
  long long splits = std::max(1LL, std::min(std::min(512 / n, steps / 4), 64LL));
  const long long per = (steps + splits - 1) / splits;
  q.splits = (int)((steps + per - 1) / per);
  q.r_per_split = (int)(per * bk);
  return q;
}

template <typename T, typename TO, int AMODE, int BMODE>
int run(Product& p, const Plan& q, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  p.splits = q.splits; p.r_per_split = q.r_per_split;
  p.part = reinterpret_cast<float*>(workspace);
  if (q.splits > 1 && (!workspace || workspace_bytes < (size_t)q.splits * p.I * p.J * 4)) return SG2IM_ERR_ARG;
  p.tiles_j = (p.J + q.tile - 1) / q.tile;
  const long long blocks = (long long)p.tiles_j * ((p.I + q.tile - 1) / q.tile) * q.splits;
  if (blocks > 0x7fffffffLL) return SG2IM_ERR_ARG;
  if (q.tile == 128) SG2IM_LAUNCH((product_kernel<T, TO, 128, 128, AMODE, BMODE>), dim3((unsigned)blocks), dim3(THREADS), 0, stream, p);
  else SG2IM_LAUNCH((product_kernel<T, TO, 64, 64, AMODE, BMODE>), dim3((unsigned)blocks), dim3(THREADS), 0, stream, p);
  if (q.splits > 1) {
    const long long pieces = (long long)p.I * ((p.J + 31) / 32) * 8;
    SG2IM_LAUNCH(join_kernel<TO>, dim3((unsigned)std::min((pieces + THREADS - 1) / THREADS, 1LL << 20)), dim3(THREADS), 0, stream, p);
  }
  return status();
}

bool sizes_ok(long long rows, int k, int n) { return rows >= 0 && rows <= 0x7fffffffLL - 256 && k >= 1 && n >= 1 && k <= (1 << 24) && n <= (1 << 24); }

ActParams act_plan(long long rows, int n) {
  ActParams p = {};
  p.M = rows; p.N = n;
  const int pieces = (n + 7) / 8;
  p.slabs = (pieces + 63) / 64;
  p.TV = (pieces + p.slabs - 1) / p.slabs;
  p.TP = THREADS / p.TV;
  const long long want = std::max(1LL, 2048LL / p.slabs);
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
  const Plan q = which == 0 ? plan(rows, n, k, dtype) : which == 1 ? plan(rows, k, n, dtype) : plan(n, k, rows, dtype);
  const size_t elems = which == 0 ? (size_t)rows * n : which == 1 ? (size_t)rows * k : (size_t)n * k;
  return q.splits > 1 ? q.splits * elems * 4 : 16;
}

int sg2im_linear_forward(const void* x, int dtype, long long ld_x, const void* weight, const void* bias, int bias_dtype,
                         const void* residual, long long ld_res, float slope, void* out, int out_dtype, long long ld_out,
                         unsigned* signs, long long rows, int k, int n, void* workspace, size_t workspace_bytes,
                         hipStream_t stream) {
  if (!sizes_ok(rows, k, n) || !type_ok(dtype) || !type_ok(out_dtype) || !type_ok(bias_dtype) || (dtype == 0 && out_dtype == 1) ||
      ld_x < k || ld_out < n || (residual && ld_res < n)) return SG2IM_ERR_ARG;
  if (rows == 0) return SG2IM_OK;
  if (!x || !weight || !out) return SG2IM_ERR_ARG;
  Product p = {};
  p.a = x; p.lda = ld_x; p.b = weight; p.ldb = k; p.I = (int)rows; p.J = n; p.R = k;
  p.bias = bias; p.bias_bf16 = bias_dtype; p.residual = residual; p.ld_res = ld_res; p.slope = slope;
  p.signs = signs; p.sign_words = (n + 31) / 32; p.out = out; p.ld_out = ld_out;
  const Plan q = plan(rows, n, k, dtype);
  if (dtype == 0) return run<float, float, RC, RC>(p, q, workspace, workspace_bytes, stream);
  if (out_dtype == 0) return run<bf16_s, float, RC, RC>(p, q, workspace, workspace_bytes, stream);
  return run<bf16_s, bf16_s, RC, RC>(p, q, workspace, workspace_bytes, stream);
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
  if (blocks > 0x7fffffffLL) return SG2IM_ERR_ARG;
  if (rows > 0 && (dz || dbias)) {
    const dim3 grid((unsigned)blocks);
    if (dy_dtype == 0 && dz_dtype == 0) SG2IM_LAUNCH((act_backward_kernel<float, float>), grid, dim3(THREADS), 0, stream, p);
    else if (dy_dtype == 0) SG2IM_LAUNCH((act_backward_kernel<float, bf16_s>), grid, dim3(THREADS), 0, stream, p);
    else SG2IM_LAUNCH((act_backward_kernel<bf16_s, bf16_s>), grid, dim3(THREADS), 0, stream, p);
  }
  if (dbias) SG2IM_LAUNCH(bias_finish_kernel, dim3((n + 31) / 32), dim3(THREADS), 0, stream, p);
  return status();
}

int sg2im_linear_backward_data(const void* dz, int dtype, long long ld_dz, const void* weight, void* dx, long long ld_dx,
                               long long rows, int k, int n, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (!sizes_ok(rows, k, n) || !type_ok(dtype) || ld_dz < n || ld_dx < k) return SG2IM_ERR_ARG;
  if (rows == 0) return SG2IM_OK;
  if (!dz || !weight || !dx) return SG2IM_ERR_ARG;
  Product p = {};
  p.a = dz; p.lda = ld_dz; p.b = weight; p.ldb = k; p.I = (int)rows; p.J = k; p.R = n;
  p.slope = 1.f; p.out = dx; p.ld_out = ld_dx;
  const Plan q = plan(rows, k, n, dtype);
  return dtype == 0 ? run<float, float, RC, RM>(p, q, workspace, workspace_bytes, stream)
                    : run<bf16_s, bf16_s, RC, RM>(p, q, workspace, workspace_bytes, stream);
}

int sg2im_linear_backward_weight(const void* dz, int dtype, long long ld_dz, const void* x, long long ld_x,
                                 const signed char* codes, const unsigned char* exps, void* dweight, int dweight_dtype,
                                 int accumulate, long long rows, int k, int n, void* workspace, size_t workspace_bytes,
                                 hipStream_t stream) {
  if (!sizes_ok(rows, k, n) || !type_ok(dtype) || !type_ok(dweight_dtype) || (dtype == 0 && dweight_dtype == 1) || ld_dz < n ||
      !codes != !exps || (!codes && ld_x < k) || !dweight) return SG2IM_ERR_ARG;
  if (rows > 0 && (!dz || (!x && !codes))) return SG2IM_ERR_ARG;
  Product p = {};
  p.a = dz; p.lda = ld_dz; p.I = n; p.J = k; p.R = (int)rows;
  p.slope = 1.f; p.out = dweight; p.ld_out = k; p.accumulate = accumulate;
  const Plan q = plan(n, k, std::max(1LL, rows), dtype);   // (no row: one empty sum, zeros or what was there)
  if (codes) {
    p.b = codes; p.ldb = k; p.b_exps = exps; p.b_nblk = (k + C8_BLOCK - 1) / C8_BLOCK;
    if (dtype == 0) return run<float, float, RM, RM8>(p, q, workspace, workspace_bytes, stream);
    if (dweight_dtype == 0) return run<bf16_s, float, RM, RM8>(p, q, workspace, workspace_bytes, stream);
    return run<bf16_s, bf16_s, RM, RM8>(p, q, workspace, workspace_bytes, stream);
  }
  p.b = x; p.ldb = ld_x;
  if (dtype == 0) return run<float, float, RM, RM>(p, q, workspace, workspace_bytes, stream);
  if (dweight_dtype == 0) return run<bf16_s, float, RM, RM>(p, q, workspace, workspace_bytes, stream);
  return run<bf16_s, bf16_s, RM, RM>(p, q, workspace, workspace_bytes, stream);
}

}  // extern "C"
