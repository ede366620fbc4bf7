// 8-bit block-scaled operands (e4m3, one fp32 scale for each 128 values of a
// row or each 128 x 128 block of a weight) and the launchers of fp8.hip and
// fp8_gemm.hip.  Shapes and pointers are checked by ops_api.hip before any of
// these is called.
//
// A block with a = max |v| (at least 2^-100, so that both factors below are
// normal fp32 numbers) is held as q = e4m3(v · fp32(448 / a)), rounded to
// nearest even, and stands for q · fp32(a / 448).  A block with a NaN or an
// infinity gives NaN wherever it is multiplied.
//
// Layouts (R rows, K values a row, Kb = ceil(K / 128), Kp = 128·Kb):
//   q       (R, Kp) bytes, zero from K on
//   scales  ROWS:  (Kb, R): the scales of one slice of K next to each other,
//                  as a tile of the product reads them
//           TILES: (ceil(R / 128), Kb), the layout of checkpoints
#pragma once

#include "common.h"
#include "internal.h"

namespace rwkvmoe {

constexpr int kFp8Block = 128;
constexpr float kE4m3Max = 448.f;
constexpr float kFp8Least = 0x1p-100f;

inline int fp8_blocks(int n) { return (n + kFp8Block - 1) / kFp8Block; }
inline size_t fp8_pad(int n) { return (size_t)fp8_blocks(n) * kFp8Block; }

enum { FP8_ROWS = 0, FP8_TILES = 1 };

struct Fp8Quant {
  const void* x;          // (groups, rows, cols), row stride ld elements
  int dtype;
  int groups, rows, cols;
  long long ld;           // groups follow each other at rows·ld
  unsigned char* q;       // or null
  float* s;
  unsigned char* qt;      // the transpose (groups, cols, pad(rows)), or null
  float* st;
};
// ROWS: q with blocks along a row, qt with blocks along a column (one group).
hipError_t launch_fp8_quant_rows(const Fp8Quant& p, hipStream_t s);
// TILES: q and qt share their blocks.
hipError_t launch_fp8_quant_tiles(const Fp8Quant& p, hipStream_t s);
// q (groups, rows, pad(cols)) and its scales from a checkpoint's e4m3 values
// (groups, rows, cols) and tile scales, and their transpose when qt is given.
hipError_t launch_fp8_layout(const unsigned char* src, const float* src_s, const Fp8Quant& p, hipStream_t s);

// What the product writes: out in fp32 / fp16 / bf16, or relu(.)² rounded to
// e4m3 again (the hidden rows of an expert layer).
enum { FP8_OUT_F32 = 0, FP8_OUT_F16 = 1, FP8_OUT_BF16 = 2, FP8_OUT_RELU2Q = 3 };

struct Fp8Gemm {
  const unsigned char* a;  // (m, pad(k))
  const float* sa;         // (Kb, m)
  const unsigned char* b;  // (groups or 1, n, pad(k))
  const float* sb;         // TILES (.., ceil(n / 128), Kb) or ROWS (Kb, n)
  const int* off;          // (groups + 1) row ranges, or null: one weight
  int groups;
  int m, n, k;
  int b_kind;              // FP8_ROWS / FP8_TILES
  bool exact;              // products summed in fp32 throughout (OUT_F32, OUT_RELU2Q; always with few rows)
  int out_kind;
  void* out;               // (m, n), or q (m, pad(n)) with FP8_OUT_RELU2Q
  float* out_s;            // (ceil(n / 128), m) with FP8_OUT_RELU2Q
  // few rows (fp8_few): the rows as they are, (m, k) in the type of out with row stride ldx, instead of a and sa
  const void* x;
  long long ldx;
};
// At most this many rows: the weight's bytes bound the product.
constexpr int kFp8FewRows = 64;
inline bool fp8_few(int m) { return m <= kFp8FewRows; }
hipError_t launch_fp8_gemm(const Fp8Gemm& p, hipStream_t s);

// xk_j = x[t] + (shift(x)[t] - x[t]) · x_k[e] for row j of the dispatch's
// order (t = perm[j] / k, e = inds[perm[j]]), rounded to e4m3 in rows.
hipError_t launch_fp8_mix(int dtype, const void* x, const void* xprev, const void* mu, const int* perm,
                          const int* inds, const int* off, int N, int T, int C, int E, int k, unsigned char* q,
                          float* s, hipStream_t st);
// out[t] = Σ_slots gates[t,slot] · rows[inv[t·k + slot]] (+ resid[t]), fp32 sums.
hipError_t launch_fp8_combine(int dtype, const float* rows, const float* gates, const int* inv, const void* resid,
                              void* out, int N, int C, int k, hipStream_t st);

// ---- device pieces ----

struct Fp8Factors {
  float up, down;  // 448 / a, a / 448
};
// amax_bits: the largest |v| of the block as its bits, which order like the
// values and put infinities and NaNs above all of them.
RWKV_DEV Fp8Factors fp8_factors(unsigned amax_bits) {
  const float a = __builtin_bit_cast(float, amax_bits > __builtin_bit_cast(unsigned, kFp8Least)
                                                ? amax_bits
                                                : __builtin_bit_cast(unsigned, kFp8Least));
  return {kE4m3Max / a, a / kE4m3Max};
}
RWKV_DEV unsigned abs_bits(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }
RWKV_DEV unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }

// Four values (already times `up`) as e4m3 bytes, v0 lowest.
RWKV_DEV unsigned fp8_pack4(float v0, float v1, float v2, float v3) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v0, v1, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v2, v3, w, true);
  return (unsigned)w;
}

// Eight consecutive values of a row from column c (zero from `cols` on).  VEC:
// rows are 16-byte aligned and cols is a multiple of 8.
template <typename T, bool VEC>
RWKV_DEV void load8(const T* row, int c, int cols, float (&v)[8]) {
  if constexpr (VEC) {
    if (c < cols) {
      if constexpr (sizeof(T) == 2) {
        Chunk<T> ch;
        ch.raw = *(const u32x4*)(row + c);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f(ch.e[i]);
      } else {
        const f32x4 a = *(const f32x4*)(row + c), b = *(const f32x4*)(row + c + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = a[i];
          v[4 + i] = b[i];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? to_f(row[c + i]) : 0.f;
  }
}

RWKV_DEV unsigned amax8(const float (&v)[8]) {
  unsigned a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = umax(a, abs_bits(v[i]));
  return a;
}
RWKV_DEV unsigned long long pack8(const float (&v)[8], float up) {
  const unsigned lo = fp8_pack4(v[0] * up, v[1] * up, v[2] * up, v[3] * up);
  const unsigned hi = fp8_pack4(v[4] * up, v[5] * up, v[6] * up, v[7] * up);
  return (unsigned long long)hi << 32 | lo;
}

}  // namespace rwkvmoe
