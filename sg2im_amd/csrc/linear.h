// The product kernel of the linear layers (linear.hip, linear_dw.hip): tiles, loaders, schedule, epilogue, choice of the tile.
//
// All three products are C[i][j] = sum_r A(i, r) B(j, r); an operand lies in memory either with r contiguous (x and W of
// the forward product, dz of dx) or with i / j contiguous (W of dx, both of dW).  A tile goes from memory through registers
// into LDS in the order it lies in (so any alignment, any width and the 8-bit form are only a matter of the load); the
// operands of v_mfma_f32_32x32x16_bf16 (8 consecutive r of one row per lane) are read with ds_read_b128 from the first kind
// and with the transposing ds_read_b64_tr_b16 from the second.  float32 uses v_mfma_f32_32x32x2_f32 on the same tiles.
//
// Four waves share a tile of BM x BN (eight the largest).  The reduction advances in chunks of 128 bytes of r, with
// two LDS images of each operand: while the matrix cores work on chunk c, chunk c + 1 is written to the other image and
// chunk c + 2 is on its way from memory; operands of the next step are read during the current one, also across the one
// barrier per chunk.
//
// Bound by the matrix cores where there is enough to do: bfloat16 8192^3 1.23 PFLOP/s (a library's product 1.5: its matrix cores
// are busy 88 % of the time, these 71 %), 32768 x 4096 x 1024 with bias and activation 272 us in a stream of
// such passes (299 - 315 in profiles of ten); float 3200 x 1152 x 512 44 us, of which 1.79 us per 32 of r at 1.71 of matrix
// instructions.  Narrow reductions are bound by their first loads and the epilogue.
#pragma once
#include <hip/hip_runtime.h>
#include <algorithm>
#include "sg2im_hip.h"
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
#define SG2IM_FENCE() __builtin_amdgcn_sched_barrier(0)

struct Product {
  const void* a; const void* b;
  const unsigned char* b_exps; int b_nblk;       // RM8
  long long lda, ldb;
  int I, J, R;                                   // rows, columns, reduction
  int tiles_i, tiles_j, splits, r_per_split;
  float* part;                                   // [splits][I][J], splits > 1
  // what happens to A on its way into LDS: A *= (bit of gate ? 1 : gate_slope), and its sums over r
  const unsigned char* gate; long long gate_ld;  // the signs of the forward pass as bytes, bytes per row
  float gate_slope;
  void* sum; int sum_bf16, sum_accumulate;       // [I]
  float* sum_part;                               // [splits][I], splits > 1
  // epilogue
  const void* bias; int bias_bf16;
  const void* residual; long long ld_res;
  float slope;
  unsigned* signs; int sign_words;               // [I][sign_words]
  void* out; int out_bf16; long long ld_out;
  int accumulate;
};

template <typename T> struct Geo;
template <> struct Geo<bf16_s> { static constexpr int BK = 64, NV = 8; };
template <> struct Geo<float> { static constexpr int BK = 32, NV = 4; };
constexpr int STEPS = 4;                         // per chunk: 16 r of bfloat16, 8 of float

// the LDS image of ROWS rows of an operand by one chunk.  Strides: 144 bytes (36 banks: the 16 rows of a b128 phase start on
// 16 different bank quads); columns + 64 bytes (the 4 rows of a transposing read lie on different quarters of the banks) or,
// for float32, + 32 bytes (rows 4 apart lie on different halves)
template <typename T, int ROWS, int MODE> struct Tile {
  static constexpr int BK = Geo<T>::BK, NV = Geo<T>::NV;
  static constexpr int LD = MODE == RC ? BK + NV : ROWS + (sizeof(T) == 2 ? 32 : 8);
  static constexpr int ELEMS = MODE == RC ? ROWS * LD : BK * LD;
};

struct Piece { unsigned w[4]; };
template <int MODE, int N> struct Staged { Piece v[N]; unsigned char g[N]; };        // (g: the gate's bits of a piece)
template <int N> struct Staged<RM8, N> { unsigned q[N][2]; unsigned char e[N], g[1]; };      // codes (float: the first word) and exponent

// the first `have` elements of a piece, zeros behind them
template <typename T> __device__ __forceinline__ Piece load_part(const T* p, int have) {
  Piece r = {{0, 0, 0, 0}};
  if (have >= Geo<T>::NV) {
    __builtin_memcpy(&r.w[0], p, 16);
  } else if (have > 0) {
    // (an element behind the end reads the last one instead and is dropped: no branch per element)
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        const unsigned w = reinterpret_cast<const unsigned*>(p)[min(j, have - 1)];
        r.w[j] = j < have ? w : 0;
      } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
        const unsigned lo = h[min(2 * j, have - 1)], hi = h[min(2 * j + 1, have - 1)];
        r.w[j] = (2 * j < have ? lo : 0) | (2 * j + 1 < have ? hi << 16 : 0);
      }
    }
  }
  return r;
}

// 128 bits moved down by n, zeros from above
__device__ __forceinline__ uint4 moved(const uint4& w, int n) {
  typedef unsigned long long u64;
  const u64 lo = w.x | (u64)w.y << 32, hi = w.z | (u64)w.w << 32;
  const int k = n & 63;
  const u64 l = n >= 64 ? hi : lo, h = n >= 64 ? 0 : hi;
  const u64 a = (l >> k) | ((h << 1) << (63 - k)), b = h >> k;
  const bool none = n >= 128;
  return make_uint4(none ? 0 : (unsigned)a, none ? 0 : (unsigned)(a >> 32), none ? 0 : (unsigned)b, none ? 0 : (unsigned)(b >> 32));
}

enum { WHOLE = 0, EDGE = 1, NARROW = 2 };
template <int V> struct Int { static constexpr int value = V; };

// One operand's way from memory to LDS: ROWS rows from row0, chunk by chunk.
//   whole: every piece of every full chunk lies inside the operand (the rows of an r-contiguous one are clamped: what a row
//   behind the last one computes is not stored), so that loads need no check
//   GATE / SUM: the two fields of Product; a thread's pieces of an i-contiguous operand always hold the same NV rows i
template <typename T, int ROWS, int MODE, int NT, bool GATE, bool SUM> struct Feeder {
  typedef Tile<T, ROWS, MODE> G;
  static constexpr int NV = G::NV, P = ROWS * 8 / NT;     // 16-byte pieces per thread
  static constexpr int PR = ROWS / NV;                     // pieces per r (i / j contiguous)
  const char* base;                                        // this chunk
  const unsigned char* exps;                               // RM8: this chunk's row of exponents
  unsigned off[MODE == RC ? P : 1];                        // bytes from base
  const unsigned char* gate;                               // this chunk's byte of the first piece's row
  unsigned gate_off[GATE ? P : 1];
  float sum[SUM ? NV : 1], gate_slope;
  long long ld, gate_ld;
  int rows, row0, nblk;
  __device__ __forceinline__ Feeder(const Product& p, const void* src, long long ld_, const unsigned char* e, int nblk_, int row0_, int rows_, int r0)
    : ld(ld_), rows(rows_), row0(row0_), nblk(nblk_) {
    const int tid = threadIdx.x;
    if constexpr (SUM) {
      #pragma unroll
      for (int j = 0; j < NV; ++j) sum[j] = 0.f;
    }
    if constexpr (GATE) {
      gate_slope = p.gate_slope;
      gate_ld = p.gate_ld;
      gate = p.gate + (MODE == RC ? row0 * gate_ld + r0 / 8 : r0 * gate_ld + row0 / 8);
      #pragma unroll
      for (int i = 0; i < P; ++i) {
        if constexpr (MODE == RC) gate_off[i] = (unsigned)min((tid >> 3) + NT / 8 * i, rows - 1 - row0) * (unsigned)gate_ld + (tid & 7) * NV / 8;
        else gate_off[i] = (unsigned)(tid / PR + NT / PR * i) * (unsigned)gate_ld + tid % PR * NV / 8;
      }
    }
    if constexpr (MODE == RC) {
      base = reinterpret_cast<const char*>(src) + ((long long)row0 * ld + r0) * (int)sizeof(T);
      #pragma unroll
      for (int i = 0; i < P; ++i) {
        const int row = min((tid >> 3) + NT / 8 * i, rows - 1 - row0);
        off[i] = (unsigned)(row * (unsigned)ld + (tid & 7) * NV) * (unsigned)sizeof(T);
      }
    } else {
      const int size = MODE == RM8 ? 1 : (int)sizeof(T);
      base = reinterpret_cast<const char*>(src) + ((long long)r0 * ld + row0) * size;
      off[0] = (unsigned)((tid / PR) * (unsigned)ld + tid % PR * NV) * (unsigned)size;
      exps = e + (long long)r0 * nblk;
    }
  }
  __device__ __forceinline__ bool whole() const { return MODE == RC || row0 + ROWS <= rows; }
  __device__ __forceinline__ void next() {
    if constexpr (GATE) gate += MODE == RC ? G::BK / 8 : G::BK * gate_ld;
    if constexpr (MODE == RC) base += 128;
    else {
      base += G::BK * ld * (MODE == RM8 ? 1 : (int)sizeof(T));
      if constexpr (MODE == RM8) exps += (long long)G::BK * nblk;
    }
  }
  // a full chunk of a whole tile
  __device__ __forceinline__ void load(Staged<MODE, P>& s) const {
    #pragma unroll
    for (int i = 0; i < P; ++i) {
      if constexpr (GATE) s.g[i] = gate[gate_off[i]];
      if constexpr (MODE == RC) __builtin_memcpy(&s.v[i], base + off[i], 16);
      else {
        const char* at = base + (long long)(NT / PR * i) * ld * (MODE == RM8 ? 1 : (int)sizeof(T)) + off[0];
        if constexpr (MODE == RM) __builtin_memcpy(&s.v[i], at, 16);
        else {
          __builtin_memcpy(s.q[i], at, NV);
          s.e[i] = exps[(long long)(threadIdx.x / PR + NT / PR * i) * nblk + (row0 + (int)(threadIdx.x % PR) * NV) / C8_BLOCK];
        }
      }
    }
  }
  // A chunk of `left` r, or of a tile that reaches over the operand's columns.  A piece over the end is read from where it
  // just fits and moved into place when it is stored (take), so that the loads stay free of branches; what lies behind the
  // end becomes zero.  (An operand narrower than a piece goes element by element.)
  __device__ __forceinline__ bool narrow(int R) const { return (MODE == RC ? R : rows) < NV; }
  __device__ __forceinline__ int over(int left) const {                    // elements that a piece starts too late for
    const int tid = threadIdx.x;
    return MODE == RC ? max(0, (tid & 7) * NV - (left - NV)) : max(0, row0 + tid % PR * NV - (rows - NV));
  }
  __device__ __forceinline__ void load_edge(Staged<MODE, P>& s, int left) const {
    const int tid = threadIdx.x, d = over(left);
    #pragma unroll
    for (int i = 0; i < P; ++i) {
      if constexpr (MODE == RC) {
        __builtin_memcpy(&s.v[i], base + off[i] - d * (int)sizeof(T), 16);
        if constexpr (GATE) s.g[i] = gate[gate_off[i] - (tid & 7) * NV / 8 + min((tid & 7) * NV, left - 1) / 8];
      } else {
        constexpr int size = MODE == RM8 ? 1 : (int)sizeof(T);
        const int r = min(tid / PR + NT / PR * i, left - 1), c = tid % PR * NV;
        const char* at = base + (r * ld + c - d) * size;
        if constexpr (GATE) s.g[i] = gate[r * gate_ld + min(c, rows - 1 - row0) / 8];
        if constexpr (MODE == RM) __builtin_memcpy(&s.v[i], at, 16);
        else {
          __builtin_memcpy(s.q[i], at, NV);
          s.e[i] = exps[(long long)r * nblk + min(row0 + c, rows - 1) / C8_BLOCK];
        }
      }
    }
  }
  __device__ __forceinline__ void load_narrow(Staged<MODE, P>& s, int left) const {
    const int tid = threadIdx.x;
    #pragma unroll
    for (int i = 0; i < P; ++i) {
      if constexpr (MODE == RC) {
        const int have = row0 + (tid >> 3) + NT / 8 * i < rows ? left - (tid & 7) * NV : 0;
        s.v[i] = load_part<T>(reinterpret_cast<const T*>(base + off[i]), have);
        if constexpr (GATE) s.g[i] = have > 0 ? gate[gate_off[i]] : 0;
      } else {
        const int r = tid / PR + NT / PR * i, col = row0 + tid % PR * NV, have = r < left ? rows - col : 0;
        const char* at = base + (long long)(NT / PR * i) * ld * (MODE == RM8 ? 1 : (int)sizeof(T)) + off[0];
        if constexpr (GATE) s.g[i] = have > 0 ? gate[gate_off[i]] : 0;
        if constexpr (MODE == RM) s.v[i] = load_part<T>(reinterpret_cast<const T*>(at), have);
        else {
          s.q[i][0] = s.q[i][1] = 0;
          s.e[i] = 127;
          if (have > 0) {
            #pragma unroll
            for (int j = 0; j < NV; ++j) {
              const unsigned q = (unsigned char)at[min(j, have - 1)];
              s.q[i][j >> 2] |= (j < have ? q : 0) << (8 * (j & 3));
            }
            s.e[i] = exps[(long long)r * nblk + col / C8_BLOCK];
          }
        }
      }
    }
  }
  // how: WHOLE, EDGE (load_edge's pieces are moved into place) or NARROW
  template <int HOW> __device__ __forceinline__ void store(T* lds, const Staged<MODE, P>& s, int left) {
    const int tid = threadIdx.x, d = HOW == EDGE ? over(left) : 0;
    #pragma unroll
    for (int i = 0; i < P; ++i) {
      const bool gone = HOW == EDGE && MODE != RC && tid / PR + NT / PR * i >= left;       // (this r is behind the end)
      T* p;
      if constexpr (MODE == RC) p = lds + ((tid >> 3) + NT / 8 * i) * G::LD + (tid & 7) * NV;
      else p = lds + (tid / PR + NT / PR * i) * G::LD + tid % PR * NV;
      uint4 w;
      if constexpr (MODE == RM8) {
        const float scale = c8_scale(s.e[i]);              // (a piece starts at a multiple of its length: one block)
        unsigned long long q = s.q[i][0] | (NV == 8 ? (unsigned long long)s.q[i][1] << 32 : 0);
        if constexpr (HOW == EDGE) q = gone || d >= NV ? 0 : (NV == 8 ? q : q & 0xffffffffu) >> (8 * d);
        float v[NV];
        #pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = c8_decode((signed char)(q >> (8 * j)), scale);
        if constexpr (sizeof(T) == 4) w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        else {
          auto two = [&](int j) { return f32_to_bf16_bits(v[j]) | (unsigned)f32_to_bf16_bits(v[j + 1]) << 16; };
          w = make_uint4(two(0), two(2), two(4), two(6));
        }
      } else {
        w = make_uint4(s.v[i].w[0], s.v[i].w[1], s.v[i].w[2], s.v[i].w[3]);
        if constexpr (HOW == EDGE) w = moved(w, gone ? 128 : d * (int)sizeof(T) * 8);
        if constexpr (GATE || SUM) {
          RawVec<T, NV> raw;
          __builtin_memcpy(&raw, &w, 16);
          float v[NV];
          widen(raw, v);
          if constexpr (GATE) {
            // (a float's piece is half of its byte: pieces start at multiples of 4)
            // bfloat16: dy * slope is rounded to the matrix operand's type, half a step (2^-8 relative) an element - none for
            // slopes 0, 1 and powers of two.  The other way, dz as two bfloat16 terms, is twice the matrix instructions; the outputs are
            // rounded by as much (dx, dW at slope 0.2 against 64 bits: 0.00165 with dz in float, 0.00168 so).
            const unsigned bits = sizeof(T) == 2 ? s.g[i] : s.g[i] >> (MODE == RC ? tid & 1 : tid % PR & 1) * 4;
            #pragma unroll
            for (int j = 0; j < NV; ++j) v[j] = bits >> j & 1 ? v[j] : v[j] * gate_slope;
          }
          if constexpr (SUM) {
            #pragma unroll
            for (int j = 0; j < NV; ++j) sum[j] += v[j];
          }
          if constexpr (GATE) {
            if constexpr (sizeof(T) == 4) w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            else {
              auto two = [&](int j) { return f32_to_bf16_bits(v[j]) | (unsigned)f32_to_bf16_bits(v[j + 1]) << 16; };
              w = make_uint4(two(0), two(2), two(4), two(6));
            }
          }
        }
      }
      *reinterpret_cast<uint4*>(p) = w;
    }
  }
};

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

// NC consecutive columns of output row i from j on, all of them inside; returns their z > 0 bits
template <typename TO, int NC>
__device__ __forceinline__ void finish_as(const Product& p, int i, int j, float (&v)[NC]) {
  TO* out = reinterpret_cast<TO*>(p.out) + (long long)i * p.ld_out + j;
  const TO* res = p.residual ? reinterpret_cast<const TO*>(p.residual) + (long long)i * p.ld_res + j : p.accumulate ? out : nullptr;
  if (res) {
    float r[NC];
    load_vec<TO, NC>(res, r);
    #pragma unroll
    for (int t = 0; t < NC; ++t) v[t] += r[t];
  }
  // (past the caches: 32768 x 1024 x 4096 bfloat16 311 -> 288 us, 131072 x 64 x 256 28 -> 23, and a reader right behind loses
  // nothing - 386 -> 372 and 48 -> 47 us for the two)
  if constexpr (sizeof(TO) * NC == 32) {
    float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
    store_vec_nt<TO, 4>(out, a);
    store_vec_nt<TO, 4>(out + 4, b);
  } else store_vec_nt<TO, NC>(out, v);
}
template <int NC>
__device__ __forceinline__ unsigned finish(const Product& p, int i, int j, float (&v)[NC]) {
  unsigned bits = 0;
  if (p.bias) {
    float b[NC];
    if (p.bias_bf16) load_vec<bf16_s, NC>(reinterpret_cast<const bf16_s*>(p.bias) + j, b);
    else load_vec<float, NC>(reinterpret_cast<const float*>(p.bias) + j, b);
    #pragma unroll
    for (int t = 0; t < NC; ++t) v[t] += b[t];
  }
  #pragma unroll
  for (int t = 0; t < NC; ++t) {
    if (v[t] > 0.f) bits |= 1u << t;
    v[t] = v[t] > 0.f ? v[t] : v[t] * p.slope;
  }
  if (p.out_bf16) finish_as<bf16_s, NC>(p, i, j, v); else finish_as<float, NC>(p, i, j, v);
  return bits;
}
template <typename TO> __device__ __forceinline__ void finish_one_as(const Product& p, int i, int j, float v) {
  TO* out = reinterpret_cast<TO*>(p.out) + (long long)i * p.ld_out + j;
  if (p.residual) v += load1(reinterpret_cast<const TO*>(p.residual) + (long long)i * p.ld_res + j);
  else if (p.accumulate) v += load1(out);
  store1(out, v);
}
__device__ __forceinline__ unsigned finish_one(const Product& p, int i, int j, float v) {
  if (p.bias) v += load_param(p.bias, p.bias_bf16, j);
  const unsigned bit = v > 0.f;
  if (!bit) v *= p.slope;
  if (p.out_bf16) finish_one_as<bf16_s>(p, i, j, v); else finish_one_as<float>(p, i, j, v);
  return bit;
}

// the schedule of a step: P products with the LDS reads, LDS writes and memory loads spread evenly between them
template <int P, int READS, int WRITES, int LOADS, int K = 0>
__device__ __forceinline__ void interleave() {
  if constexpr (K < P) {
    constexpr int r = (K + 1) * READS / P - K * READS / P, w = (K + 1) * WRITES / P - K * WRITES / P, l = (K + 1) * LOADS / P - K * LOADS / P;
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (r > 0) __builtin_amdgcn_sched_group_barrier(0x100, r, 0);
    if constexpr (w > 0) __builtin_amdgcn_sched_group_barrier(0x200, w, 0);
    if constexpr (l > 0) __builtin_amdgcn_sched_group_barrier(0x020, l, 0);
    interleave<P, READS, WRITES, LOADS, K + 1>();
  }
}
// LDS reads of an operand, matrix instructions of a product
template <typename T, int MODE> constexpr int READS_OF = MODE == RC ? 1 : sizeof(T) == 2 ? 2 : 4;
template <typename T> constexpr int MFMAS_OF = sizeof(T) == 2 ? 1 : 4;

// EDGES: there are partial chunks or tiles over the end of an i / j contiguous operand
template <typename T, int BM, int BN, int NT, int AMODE, int BMODE, bool GATE, bool SUM, bool EDGES>
__global__ __launch_bounds__(NT, 2) void product_kernel(const Product p) {
  typedef Feeder<T, BM, AMODE, NT, GATE, SUM> FA;
  typedef Feeder<T, BN, BMODE, NT, false, false> FB;
  typedef Tile<T, BM, AMODE> GA;
  typedef Tile<T, BN, BMODE> GB;
  constexpr int WJ = NT / 128, WM = BM / 2, WN = BN / WJ;          // 2 x WJ waves of WM x WN
  constexpr int BK = GA::BK, TI = WM / 32, TJ = WN / 32;
  constexpr int NP = TI * TJ * MFMAS_OF<T>, NR = TI * READS_OF<T, AMODE> + TJ * READS_OF<T, BMODE>, NL = FA::P + FB::P;
  constexpr int EP = WN + 4;                                   // floats of an epilogue row (4 banks apart, 32 rows per wave)
  constexpr int BYTES = 2 * (GA::ELEMS + GB::ELEMS) * (int)sizeof(T), EP_BYTES = NT / 64 * 32 * EP * 4;
  __shared__ __attribute__((aligned(16))) char lds[BYTES > EP_BYTES ? BYTES : EP_BYTES];
  T* lds_a = reinterpret_cast<T*>(lds);
  T* lds_b = lds_a + 2 * GA::ELEMS;
  // Workgroups go round robin over the 8 XCDs: a contiguous run of tiles each, four rows of tiles at a time, so that the
  // workgroups that share an L2 share operands
  const int tiles = p.tiles_i * p.tiles_j, blocks = tiles * p.splits;
  int id = blockIdx.x;
  if (blocks % 8 == 0) id = id % 8 * (blocks / 8) + id / 8;
  const int split = id / tiles, tile = id - split * tiles;
  const int group = tile / (4 * p.tiles_j), in = tile - group * 4 * p.tiles_j, gi = min(4, p.tiles_i - 4 * group);
  const int i0 = (4 * group + in % gi) * BM, j0 = in / gi * BN;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wi = wave / WJ * WM, wj = wave % WJ * WN;
  const int r_begin = split * p.r_per_split, length = min(p.R - r_begin, p.r_per_split);
  const int chunks = (length + BK - 1) / BK, full = length / BK;

  f32x16 acc[TI][TJ];
  #pragma unroll
  for (int a = 0; a < TI; ++a)
    #pragma unroll
    for (int b = 0; b < TJ; ++b)
      #pragma unroll
      for (int v = 0; v < 16; ++v) acc[a][b][v] = 0.f;

  FA fa(p, p.a, p.lda, nullptr, 0, i0, p.I, r_begin);
  FB fb(p, p.b, p.ldb, p.b_exps, p.b_nblk, j0, p.J, r_begin);
  Staged<AMODE, FA::P> sa;
  Staged<BMODE, FB::P> sb;
  const bool whole = fa.whole() && fb.whole(), narrow = fa.narrow(p.R) || fb.narrow(p.R);
  int fetched = 0, staged = 0;                                     // chunks on their way so far; how many r the last one has
  auto fetch = [&](auto how) {
    staged = length - fetched * BK;
    if constexpr (how.value == WHOLE) { fa.load(sa); fb.load(sb); }
    else if constexpr (how.value == EDGE) { fa.load_edge(sa, staged); fb.load_edge(sb, staged); }
    else { fa.load_narrow(sa, staged); fb.load_narrow(sb, staged); }
    fa.next(); fb.next();
    ++fetched;
  };
  auto put = [&](auto how, int image) {
    fa.template store<how.value>(lds_a + image * GA::ELEMS, sa, staged);
    fb.template store<how.value>(lds_b + image * GB::ELEMS, sb, staged);
  };
  typedef decltype(operand<BM, AMODE>(lds_a, 0, 0, 0)) Op;
  Op oa[2][TI], ob[2][TJ];
  auto read = [&](int into, int image, int step) {
    #pragma unroll
    for (int a = 0; a < TI; ++a) oa[into][a] = operand<BM, AMODE>(lds_a + image * GA::ELEMS, wi + 32 * a, step, lane);
    #pragma unroll
    for (int b = 0; b < TJ; ++b) ob[into][b] = operand<BN, BMODE>(lds_b + image * GB::ELEMS, wj + 32 * b, step, lane);
  };
  auto compute = [&](int from) {
    #pragma unroll
    for (int a = 0; a < TI; ++a)
      #pragma unroll
      for (int b = 0; b < TJ; ++b) acc[a][b] = multiply(ob[from][b], oa[from][a], acc[a][b]);
  };

  // the products of chunks [c, end), with chunk c + 1 put and c + 2 fetched next to those of chunk c
  int c = 0;
  auto run_to = [&](auto how, int end) {
    for (; c < end; ++c) {
      const int image = c & 1;
      // The order inside a step: the LDS and memory traffic spread between the products (left to itself the compiler moves
      // each access next to its use, and the matrix cores wait for it)
      read(1, image, 1);
      put(how, image ^ 1);
      compute(0);
      interleave<NP, NR, NL, 0>();
      SG2IM_FENCE();
      read(0, image, 2);
      fetch(how);
      compute(1);
      interleave<NP, NR, 0, NL>();
      SG2IM_FENCE();
      read(1, image, 3);
      compute(0);
      interleave<NP, NR, 0, 0>();
      __syncthreads();
      SG2IM_FENCE();
      read(0, image ^ 1, 0);
      compute(1);
      interleave<NP, NR, 0, 0>();
      SG2IM_FENCE();
    }
  };
  // One that has all its pieces is loaded without checks, and so is each of its full chunks
  auto with_form = [&](int chunk, auto f) {
    if constexpr (!EDGES) f(Int<WHOLE>());
    else if (narrow) f(Int<NARROW>());
    else if (whole && chunk < full) f(Int<WHOLE>());
    else f(Int<EDGE>());
  };
  if (chunks > 0) {
    with_form(0, [&](auto how) { fetch(how); put(how, 0); });
    if (chunks > 1) with_form(1, fetch);
    __syncthreads();
    read(0, 0, 0);
    if (!EDGES || (whole && !narrow)) run_to(Int<WHOLE>(), full - 2);
    if constexpr (EDGES) if (!whole && !narrow) run_to(Int<EDGE>(), chunks - 2);
    for (; c < chunks; ++c) {
      const int image = c & 1;
      read(1, image, 1);
      if (c + 1 < chunks) with_form(c + 1, [&](auto how) { put(how, image ^ 1); });
      compute(0);
      read(0, image, 2);
      if (c + 2 < chunks) with_form(c + 2, fetch);
      compute(1);
      read(1, image, 3);
      compute(0);
      __syncthreads();
      if (c + 1 < chunks) read(0, image ^ 1, 0);
      compute(1);
    }
  }

  if constexpr (SUM) {
    // every column of tiles has A's sums; the first one's are kept
    if (j0 == 0 && p.sum) {
      constexpr int PR = FA::PR, LANES = NT / PR;
      float* sums = reinterpret_cast<float*>(lds);                 // [LANES][BM]
      __syncthreads();
      #pragma unroll
      for (int j = 0; j < FA::NV; ++j) sums[threadIdx.x / PR * BM + threadIdx.x % PR * FA::NV + j] = fa.sum[j];
      __syncthreads();
      for (int i = threadIdx.x; i < BM && i0 + i < p.I; i += NT) {
        float t = 0.f;
        #pragma unroll
        for (int k = 0; k < LANES; ++k) t += sums[k * BM + i];
        if (p.splits > 1) p.sum_part[(long long)split * p.I + i0 + i] = t;
        else store_param(p.sum, p.sum_bf16, i0 + i, t, p.sum_accumulate);
      }
    }
  }
  if (p.splits > 1) {
    #pragma unroll
    for (int a = 0; a < TI; ++a) {
      const int i = i0 + wi + 32 * a + (lane & 31);
      #pragma unroll
      for (int b = 0; b < TJ; ++b)
        #pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int j = j0 + wj + 32 * b + 8 * q + 4 * (lane >> 5);
          float v[4] = {acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]};
          if (i < p.I) {
            float* out = p.part + ((long long)split * p.I + i) * p.J + j;
            if (j + 4 <= p.J) store_vec<float, 4>(out, v);
            else {
              #pragma unroll
              for (int t = 0; t < 4; ++t) if (j + t < p.J) out[t] = v[t];
            }
          }
        }
    }
    return;
  }
  // A lane holds scattered fours of one row; 32 rows at a time go through the wave's own part of LDS, so that 8 (4) lanes
  // then hold whole runs of a row and bias, residual and output are read and written in 16-byte pieces
  constexpr int NC = 8, LANES = WN / NC;                       // lanes per row
  __syncthreads();
  float* mine = reinterpret_cast<float*>(lds) + wave * 32 * EP;
  #pragma unroll
  for (int a = 0; a < TI; ++a) {
    #pragma unroll
    for (int b = 0; b < TJ; ++b)
      #pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4*>(mine + (lane & 31) * EP + 32 * b + 8 * q + 4 * (lane >> 5)) =
            make_float4(acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2], acc[a][b][4 * q + 3]);
    __builtin_amdgcn_wave_barrier();
    #pragma unroll
    for (int k = 0; k < 32 * LANES / 64; ++k) {
      const int row = k * (64 / LANES) + lane / LANES, col = lane % LANES * NC;
      const float* from = mine + row * EP + col;
      const int i = i0 + wi + 32 * a + row, j = j0 + wj + col;
      unsigned bits = 0;
      if (i < p.I && j + NC <= p.J) {
        const float4 lo = *reinterpret_cast<const float4*>(from), hi = *reinterpret_cast<const float4*>(from + 4);
        float v[NC] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        bits = finish<NC>(p, i, j, v);
      } else if (i < p.I) {
        for (int t = 0; j + t < p.J; ++t) bits |= finish_one(p, i, j + t, from[t]) << t;
      }
      bits <<= 8 * (lane & 3);
      if (p.signs) {
        bits |= __shfl_xor(bits, 1);
        bits |= __shfl_xor(bits, 2);
        if ((lane & 3) == 0 && i < p.I && j < p.J) p.signs[(long long)i * p.sign_words + j / 32] = bits;
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The splits' sums joined in a fixed order: SL threads share a piece of 4 columns (a small output has few pieces, and one
// thread's walk over 64 splits took 18 us), and 8 pieces make a word of signs.  256 x 1024 of 16 splits 7.7 us.
template <int SL>
__global__ __launch_bounds__(THREADS) static void join_kernel(const Product p) {
  constexpr int NPIECE = THREADS / SL;
  __shared__ float4 red[SL > 1 ? THREADS : 1];
  __shared__ float red_sum[SL > 1 ? THREADS : 1];
  const int words = (p.J + 31) / 32, sl = threadIdx.x / NPIECE, pc = threadIdx.x % NPIECE;
  const long long pieces = (long long)p.I * words * 8, plane = (long long)p.I * p.J;
  for (long long b0 = (long long)blockIdx.x * NPIECE; b0 < pieces; b0 += (long long)gridDim.x * NPIECE) {
    const long long at = b0 + pc, word = at >> 3;
    const int i = (int)(word / words), w = (int)(word - (long long)i * words), j = w * 32 + (int)(at & 7) * 4;
    const int have = at < pieces ? min(4, p.J - j) : 0;
    const float* src = p.part + (long long)i * p.J + j;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (have == 4) {
      #pragma unroll 8
      for (int s = sl; s < p.splits; s += SL) {
        float u[4];
        load_vec<float, 4>(src + s * plane, u);
        #pragma unroll
        for (int t = 0; t < 4; ++t) v[t] += u[t];
      }
    } else if (have > 0) {
      for (int s = sl; s < p.splits; s += SL) {
        v[0] += src[s * plane];
        if (have > 1) v[1] += src[s * plane + 1];
        if (have > 2) v[2] += src[s * plane + 2];
      }
    }
    // A's sums over r: the row's first piece joins them too
    const bool sums = p.sum_part && j == 0 && at < pieces;
    float sum = 0.f;
    if (sums) {
      #pragma unroll 8
      for (int s = sl; s < p.splits; s += SL) sum += p.sum_part[(long long)s * p.I + i];
    }
    if constexpr (SL > 1) {
      red_sum[threadIdx.x] = sum;
      red[threadIdx.x] = make_float4(v[0], v[1], v[2], v[3]);
      __syncthreads();
      if (sl == 0) {
        #pragma unroll
        for (int k = 1; k < SL; ++k) {
          const float4 u = red[k * NPIECE + pc];
          v[0] += u.x; v[1] += u.y; v[2] += u.z; v[3] += u.w;
          sum += red_sum[k * NPIECE + pc];
        }
      }
      __syncthreads();
    }
    unsigned bits = 0;
    if (sl == 0) {
      if (sums) store_param(p.sum, p.sum_bf16, i, sum, p.sum_accumulate);
      if (have == 4) bits = finish<4>(p, i, j, v);
      else if (have > 0) {
        bits = finish_one(p, i, j, v[0]);
        if (have > 1) bits |= finish_one(p, i, j + 1, v[1]) << 1;
        if (have > 2) bits |= finish_one(p, i, j + 2, v[2]) << 2;
      }
    }
    if (p.signs) {
      bits <<= 4 * (int)(at & 7);
      #pragma unroll
      for (int o = 1; o < 8; o <<= 1) bits |= __shfl_xor(bits, o);
      if (sl == 0 && at < pieces && (at & 7) == 0) p.signs[(long long)i * p.sign_words + w] = bits;
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------

inline int status() { return hipGetLastError() == hipSuccess ? SG2IM_OK : SG2IM_ERR_HIP; }
inline bool type_ok(int t) { return t == 0 || t == 1; }

struct Plan { int tile, splits, r_per_split; double us; };

// The tile and the number of splits with the least estimated time.  A CU holds 3 / 2 / 1 workgroups of the 64 / 128 / 256
// tile; a round of o of them takes the tile's fixed part and, per chunk, the larger of its latency and o times its share of
// the matrix cores; splitting costs a second launch and the partial sums' way to memory and back at 3.5 TB/s.  The figures
// (microseconds) are fitted to 13 shapes x 3 products x all tiles and splits, 0.2 to 340 us; the estimate is within 20 %, and
// the tile it picks within 10 % of the best.  E.g. (bfloat16, I x J x R): 32768 x 4096 x 1024 256-tile 272, 128 327, 64 473;
// 32768 x 256 x 1024 33, 27, 33; 131072 x 64 x 256 38, 28, 19; 256 x 1024 x 32768 with 16 splits of the 128-tile 40, none
// split faster than 44; 2048 x 2048 x 512 12.4 with one, 30 with two.
// work: what the gate (GATED) or the sums (SUMMED) add to the 128 tile's chunk (bfloat16, 2048 x 512 x 2048: dx 13.6 -> 21.7 us
// gated, 32768 x 512 x 512 29 -> 42; dW with its sums 14.4 -> 17.2); their kernels have no 256 tile, nor
// have products with edges (which: 0 forward, 1 dx, 2 dW): the registers of two waves per SIMD do not hold more.
constexpr double GATED[2] = {0.20, 0.35}, SUMMED[2] = {0.05, 0.12};
struct TileCost { int tile, per_cu; double fixed, latency, share; };
constexpr TileCost COSTS[2][3] = {{{64, 3, 2.0, 0.55, 0.50}, {128, 2, 3.0, 1.9, 1.85}, {256, 1, 6.0, 7.5, 7.5}},        // float
                                  {{64, 3, 2.0, 0.33, 0.23}, {128, 2, 3.0, 0.65, 0.62}, {256, 1, 6.0, 1.75, 1.75}}};    // bfloat16
inline Plan plan(int which, long long I, long long J, long long R, int bf16, double work = 0.0) {
  static const int ways[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64, 96, 128};
  const int bk = bf16 ? 64 : 32;
  const long long steps = std::max(1LL, (R + bk - 1) / bk);
  Plan best = {64, 1, (int)(steps * bk), 1e30};
  for (const TileCost& t : COSTS[bf16]) {
    if (t.tile == 256 && (work > 0.0 || R % bk || (which >= 1 && J % 256) || (which == 2 && I % 256))) break;
    const long long tiles = ((I + t.tile - 1) / t.tile) * ((J + t.tile - 1) / t.tile);
    for (int w : ways) {
      if (w > steps || (w > 1 && tiles * w > 1024)) break;
      const long long per = (steps + w - 1) / w, splits = (steps + per - 1) / per, q = (tiles * splits + 255) / 256;
      const long long rounds = (q + t.per_cu - 1) / t.per_cu, last = q - (rounds - 1) * t.per_cu;
      auto round = [&](long long o) { return t.fixed + per * std::max(t.latency + work * t.tile / 128, o * (t.share + work * t.tile / 128)); };
      double us = (rounds - 1) * round(t.per_cu) + round(last);
      if (splits > 1) us += 3.5 + 8.0 * splits * I * J / 3.5e6;
      if (us < best.us) best = {t.tile, (int)splits, (int)(per * bk), us};
    }
  }
  return best;
}

inline size_t plan_bytes(const Plan& q, size_t I, size_t J, bool sums) { return q.splits > 1 ? q.splits * (I * J + (sums ? I : 0)) * 4 : 16; }

template <typename T, int AMODE, int BMODE, bool GATE, bool SUM>
int run(Product& p, const Plan& q, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  p.splits = q.splits; p.r_per_split = q.r_per_split;
  if (q.splits > 1) {
    if (!workspace || workspace_bytes < plan_bytes(q, p.I, p.J, SUM)) return SG2IM_ERR_ARG;
    p.part = reinterpret_cast<float*>(workspace);
    if (SUM && p.sum) p.sum_part = p.part + (size_t)q.splits * p.I * p.J;
  }
  p.tiles_i = (p.I + q.tile - 1) / q.tile;
  p.tiles_j = (p.J + q.tile - 1) / q.tile;
  const long long blocks = (long long)p.tiles_j * p.tiles_i * q.splits;
  if (blocks * (q.tile == 256 ? 512 : 256) > 0xffffffffLL) return SG2IM_ERR_ARG;      // (a launch has fewer than 2^32 threads)
  const dim3 grid((unsigned)blocks);
  if constexpr (!GATE && !SUM) if (q.tile == 256) SG2IM_LAUNCH((product_kernel<T, 256, 256, 512, AMODE, BMODE, GATE, SUM, false>), grid, dim3(512), 0, stream, p);
  if (q.tile == 128) SG2IM_LAUNCH((product_kernel<T, 128, 128, 256, AMODE, BMODE, GATE, SUM, true>), grid, dim3(256), 0, stream, p);
  if (q.tile == 64) SG2IM_LAUNCH((product_kernel<T, 64, 64, 256, AMODE, BMODE, GATE, SUM, true>), grid, dim3(256), 0, stream, p);
  if (q.splits > 1) {
    const long long pieces = (long long)p.I * ((p.J + 31) / 32) * 8;
    // Eight threads to a piece where there are splits for each of them and too few pieces to fill the card.  dW with its join, microseconds,
    // one thread / eight: 128 splits of 1024 pieces (65536 x 64 -> 64 bfloat16) 44.1 / 13.1, 128 of 4096 49.8 / 23.2, 32 of 16384 24.4 / 17.9,
    // 8 of 24720 15.7 / 12.4; 16 of 65536 39.3 / 38.7; 4 of 262144 92 / 98, 3 of 147456 (float) 47.8 / 50.5.
    if (q.splits >= 8 && pieces < 1 << 16) SG2IM_LAUNCH(join_kernel<8>, dim3((unsigned)((pieces + 31) / 32)), dim3(THREADS), 0, stream, p);
    else SG2IM_LAUNCH(join_kernel<1>, dim3((unsigned)std::min((pieces + THREADS - 1) / THREADS, 1LL << 20)), dim3(THREADS), 0, stream, p);
  }
  return status();
}

// the weight gradient's products (linear_dw.hip): x (or codes) as B; gate, sum: Product's fields
int run_weight(Product& p, int dtype, bool codes, const Plan& q, void* workspace, size_t workspace_bytes, hipStream_t stream);

}  // namespace lin
}  // namespace sg2im
