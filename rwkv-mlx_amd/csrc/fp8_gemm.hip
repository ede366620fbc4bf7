// Products of e4m3 operands with a scale for each 128 values (fp8.h):
//   out[m, n] = Σ_kb sa[m, kb] · sb[n / 128, kb] · Σ_{k in block kb} qa[m, k] · qb[n, k]
// The inner sum is one v_mfma_f32_16x16x128_f8f6f4 with a zero accumulator, a
// whole block of K; its four results a lane are then scaled into the fp32
// accumulators by one fma each.  That instruction (as the 16x16x32 e4m3 one)
// does not add products in fp32 from the start: it aligns every 8 consecutive
// k to their largest product and drops what lies 2^-13 below it (measured:
// 2^16 - 2^16 + 2^e is exact down to e = 3 within such a group and to e = -8
// or lower across groups).  On N(0, 1) operands that is about 2^-13.5 of a
// result, which a 16-bit result's rounding (2^-8, 2^-11) covers.  EX forms
// convert both operands to fp16 (exact) and use the fp16 instruction, whose
// sums are fp32's: for fp32 results, and where few rows leave the weight's
// bytes to bound the product anyway.  Blocks are computed transposed (the MFMA's A
// operand is rows of b), so that a lane's results lie in one row of out: the
// scale of its row is one register, the weight's scale a scalar.
#include "fp8.h"
#include "gemm_tile.h"

#include <algorithm>

namespace rwkvmoe {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// 16-byte chunk swizzle of a 128-byte LDS row (a function of row % 16): the 16
// rows of a fragment read hit distinct 16-byte bank groups.
RWKV_DEV int swz(int row) { return (row & 7) ^ ((row >> 3) & 1); }

RWKV_DEV i32x8 join(u32x4 lo, u32x4 hi) {
  i32x8 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = (int)lo[i];
    r[4 + i] = (int)hi[i];
  }
  return r;
}

// D = A · Bᵀ over one block of 128: lane l feeds row l % 16 of either operand
// with the chunks l / 16 and l / 16 + 4 of its 128 bytes (any order of k does,
// as long as both operands take the same).
RWKV_DEV f32x4 mma128(i32x8 a, i32x8 b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// The same in four steps of fp16: piece p is the p-th 8 bytes of a lane's 32.
struct Wide {
  f16x8 p[4];
};
RWKV_DEV Wide widen(i32x8 v) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  Wide w;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const h2 lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[i], 1.f, false);
    const h2 hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[i], 1.f, true);
    w.p[i >> 1][(i & 1) * 4 + 0] = lo[0];
    w.p[i >> 1][(i & 1) * 4 + 1] = lo[1];
    w.p[i >> 1][(i & 1) * 4 + 2] = hi[0];
    w.p[i >> 1][(i & 1) * 4 + 3] = hi[1];
  }
  return w;
}
RWKV_DEV f32x4 mma128(const Wide& a, const Wide& b) {
  f32x4 t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) t = Mma16<f16>::run(a.p[i], b.p[i], t);
  return t;
}
template <bool EX> struct Operand {
  typedef i32x8 type;
  static RWKV_DEV i32x8 of(i32x8 v) { return v; }
};
template <> struct Operand<true> {
  typedef Wide type;
  static RWKV_DEV Wide of(i32x8 v) { return widen(v); }
};

// Asynchronous 16 or 4 bytes a lane into LDS.
RWKV_DEV void load_lds16(__amdgpu_buffer_rsrc_t r, unsigned char* dst, unsigned voff, unsigned soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 16, voff, soff, 0, 0);
}
RWKV_DEV void load_lds4(__amdgpu_buffer_rsrc_t r, unsigned char* dst, unsigned voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr_t)dst, 4, voff, 0, 0, 0);
}

// The row range [lo, hi) of tile row mt and its group; group == p.groups: the
// rows after the last range.  False: past every tile row.
struct Range {
  int lo, hi, g;
};
template <int BM>
RWKV_DEV bool find_range(const Fp8Gemm& p, int mt, Range* r) {
  const int lane = threadIdx.x & 63;
  int before = 0, edge = 0;  // tiles and rows of the 64s of groups before
  for (int g0 = 0; g0 <= p.groups; g0 += 64) {
    const int g = g0 + lane;
    // ranges are clamped to the rows, and do not overlap, whatever the offsets hold
    int hi = g < p.groups ? min(max(p.off[g + 1], 0), p.m) : g == p.groups ? p.m : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(hi, d);
      if (lane >= d) hi = max(hi, v);
    }
    hi = max(hi, edge);
    int lo = __shfl_up(hi, 1);
    if (lane == 0) lo = edge;
    edge = __builtin_amdgcn_readlane(hi, 63);
    int sum = (hi - lo + BM - 1) / BM;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    const int found = __popcll(__ballot(before + sum <= mt));
    if (found < 64) {
      const int f = __builtin_amdgcn_readfirstlane(found);
      const int prev = f > 0 ? __builtin_amdgcn_readlane(sum, f - 1) : 0;
      r->g = g0 + f;
      r->lo = __builtin_amdgcn_readlane(lo, f) + (mt - before - prev) * BM;
      r->hi = __builtin_amdgcn_readlane(hi, f);
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

template <typename T>
RWKV_DEV void store4(T* row, int c, int n, bool vec, const float (&v)[4]) {
  if (vec && c + 4 <= n) {
    union { T e[4]; unsigned long long u[sizeof(T) / 2]; } w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w.e[i] = from_f<T>(v[i]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((unsigned long long*)(row + c))[i] = w.u[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < n) row[c + i] = from_f<T>(v[i]);
  }
}

template <int OUT> struct OutType { typedef float type; };
template <> struct OutType<FP8_OUT_F16> { typedef f16 type; };
template <> struct OutType<FP8_OUT_BF16> { typedef bf16 type; };

// ---- tiles --------------------------------------------------------------------

// A BM x BN tile, WGM x WGN waves.  Slices of one block of K (128 bytes a row)
// go straight from memory into a ring of ST LDS stages; slice kb + ST - 1 is
// requested as slice kb is multiplied, one barrier a slice.
template <int BM, int BN, int WGM, int WGN, int ST, int BKIND, int OUT, bool GRP, bool EX>
__global__ __launch_bounds__(WGM * WGN * 64) void fp8_tile_kernel(Fp8Gemm p, int tiles_m, int tiles_n, int group_m) {
  constexpr int NW = WGM * WGN;
  constexpr int WM = BM / WGM, WN = BN / WGN, MI = WM / 16, NI = WN / 16;
  constexpr int DA = BM / 8 / NW, DB = BN / 8 / NW;  // 1 KB requests of a wave a slice
  static_assert(DA * 8 * NW == BM && DB * 8 * NW == BN, "requests");
  static_assert(BM / 64 + BN / 64 <= NW, "one scale request a wave");
  static_assert(128 % WN == 0 || WN == 128, "a wave's columns share one weight block");
  static_assert(OUT != FP8_OUT_RELU2Q || WN == 128, "a wave holds whole blocks of its rows");
  constexpr int UA = BM * 128, UB = BN * 128, US = (BM + BN) * 4;
  constexpr int STAGE = UA + UB + US;
  static_assert(ST * STAGE <= 163840, "LDS");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[ST * STAGE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const int Kb = (p.k + 127) / 128, Kp = Kb * 128;

  // XCD w % 8 takes a contiguous run of the tiles, group_m tile rows at a time
  const int total = tiles_m * tiles_n, w = blockIdx.x, xcd = w & 7;
  const int l = xcd * (total / 8) + min(xcd, total % 8) + (w >> 3);
  const int in_group = group_m * tiles_n, first = (l / in_group) * group_m;
  const int gsize = min(tiles_m - first, group_m);
  const int mt = first + (l % in_group) % gsize, n0 = ((l % in_group) / gsize) * BN;
  Range r{mt * BM, p.m, 0};
  if constexpr (GRP) {
    if (!find_range<BM>(p, mt, &r)) return;
    if (r.g == p.groups) {  // rows of no range
      if constexpr (OUT != FP8_OUT_RELU2Q) {
        typedef typename OutType<OUT>::type T;
        for (int i = tid; i < BM * BN; i += NW * 64) {
          const int row = r.lo + i / BN, c = n0 + i % BN;
          if (row < r.hi && c < p.n) ((T*)p.out)[(size_t)row * p.n + c] = from_f<T>(0.f);
        }
      }
      return;
    }
  }
  const int m0 = r.lo, mlim = min(r.hi, m0 + BM);

  const __amdgpu_buffer_rsrc_t ra = buf_rsrc(p.a + (size_t)m0 * Kp, 0xFFFFFFF0u);
  const __amdgpu_buffer_rsrc_t rb = buf_rsrc(p.b + ((size_t)r.g * p.n + n0) * Kp, 0xFFFFFFF0u);
  unsigned va[DA], vb[DB];
#pragma unroll
  for (int i = 0; i < DA; ++i) {
    const int row = (wave * DA + i) * 8 + (lane >> 3);
    // rows past the end read the last one
    va[i] = (unsigned)(min(m0 + row, mlim - 1) - m0) * (unsigned)Kp + ((lane & 7) ^ swz(row)) * 16;
  }
#pragma unroll
  for (int i = 0; i < DB; ++i) {
    const int row = (wave * DB + i) * 8 + (lane >> 3);
    vb[i] = (unsigned)(min(n0 + row, p.n - 1) - n0) * (unsigned)Kp + ((lane & 7) ^ swz(row)) * 16;
  }
  // every wave makes one request of 64 scales: of a's rows, or of b's; with
  // one scale a block of b the waves behind a's repeat them
  const bool sb_wave = BKIND == FP8_ROWS && NW - 1 - wave < BN / 64;
  const int sw = sb_wave ? NW - 1 - wave : wave % (BM / 64);
  auto request = [&](int kb, int slot) {
    unsigned char* st = lds + slot * STAGE;
    const unsigned so = (unsigned)kb * 128u;
#pragma unroll
    for (int i = 0; i < DA; ++i)
      load_lds16(ra, st + (wave * DA + i) * 1024, va[i], so);
#pragma unroll
    for (int i = 0; i < DB; ++i)
      load_lds16(rb, st + UA + (wave * DB + i) * 1024, vb[i], so);
    const float* sp = sb_wave ? p.sb + (size_t)kb * p.n + n0 : p.sa + (size_t)kb * p.m + m0;
    const __amdgpu_buffer_rsrc_t rs = buf_rsrc(sp, (unsigned)(sb_wave ? min(BN, p.n - n0) : mlim - m0) * 4u);
    load_lds4(rs, st + UA + UB + (sb_wave ? BM * 4 : 0) + sw * 256, (sw * 64 + lane) * 4);
  };

  // the weight block's scales along K
  const int nb = (n0 + wn * WN) / 128;
  const float* sbp = BKIND == FP8_TILES
                         ? p.sb + ((size_t)r.g * ((p.n + 127) / 128) + min(nb, (p.n + 127) / 128 - 1)) * Kb
                         : nullptr;
  float sb_next = BKIND == FP8_TILES ? sbp[0] : 1.f;

  const int fsw = swz(lane & 15), fch = lane >> 4;
  const int ao = (wm * WM + (lane & 15)) * 128 + ((fch ^ fsw) << 4);
  const int bo = UA + (wn * WN + (lane & 15)) * 128 + ((fch ^ fsw) << 4);
  f32x4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int s = 0; s < ST - 1; ++s) request(min(s, Kb - 1), s);
  int slot = 0;
  for (int kb = 0; kb < Kb; ++kb) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((ST - 2) * (DA + DB + 1)) : "memory");
    const int free_slot = slot == 0 ? ST - 1 : slot - 1;
    request(min(kb + ST - 1, Kb - 1), free_slot);  // (past the end: the last slice again, into a stage of no reader)
    const float sb = sb_next;
    if constexpr (BKIND == FP8_TILES) sb_next = sbp[min(kb + 1, Kb - 1)];
    const unsigned char* st = lds + slot * STAGE;
    typename Operand<EX>::type fa[MI];
    float f[MI];
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      fa[i] = Operand<EX>::of(join(*(const u32x4*)(st + ao + i * 2048), *(const u32x4*)(st + (ao ^ 64) + i * 2048)));
      f[i] = *(const float*)(st + UA + UB + (wm * WM + i * 16 + (lane & 15)) * 4) * sb;
    }
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const auto fb =
          Operand<EX>::of(join(*(const u32x4*)(st + bo + j * 2048), *(const u32x4*)(st + (bo ^ 64) + j * 2048)));
      f32x4 cs{1.f, 1.f, 1.f, 1.f};
      if constexpr (BKIND == FP8_ROWS)
        cs = *(const f32x4*)(st + UA + UB + BM * 4 + (wn * WN + j * 16 + (lane >> 4) * 4) * 4);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const f32x4 t = mma128(fb, fa[i]);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[i][j][q] = __builtin_fmaf(BKIND == FP8_ROWS ? t[q] * cs[q] : t[q], f[i], acc[i][j][q]);
      }
    }
    slot = slot + 1 == ST ? 0 : slot + 1;
  }

  // ---- epilogue ----
  if constexpr (OUT == FP8_OUT_RELU2Q) {
    const int col0 = n0 + wn * WN;
    const int Np = (p.n + 127) / 128 * 128;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int row = m0 + wm * WM + i * 16 + (lane & 15);
      unsigned am = 0;
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float v = acc[i][j][q], z = v < 0.f ? 0.f : v;  // (a NaN stays one)
          acc[i][j][q] = col0 + j * 16 + (lane >> 4) * 4 + q < p.n ? z * z : 0.f;
          am = umax(am, abs_bits(acc[i][j][q]));
        }
      am = umax(am, (unsigned)__shfl_xor((int)am, 16));
      am = umax(am, (unsigned)__shfl_xor((int)am, 32));
      const Fp8Factors fc = fp8_factors(am);
      if (row < mlim && col0 < p.n) {
        unsigned char* q = (unsigned char*)p.out + (size_t)row * Np + col0 + (lane >> 4) * 4;
#pragma unroll
        for (int j = 0; j < NI; ++j)
          *(unsigned*)(q + j * 16) = fp8_pack4(acc[i][j][0] * fc.up, acc[i][j][1] * fc.up, acc[i][j][2] * fc.up,
                                               acc[i][j][3] * fc.up);
        if (lane < 16) p.out_s[(size_t)(col0 / 128) * p.m + row] = fc.down;
      }
    }
  } else {
    typedef typename OutType<OUT>::type T;
    const bool vec = p.n % (8 / sizeof(T) * (sizeof(T) / 2)) == 0 && p.n % 4 == 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int row = m0 + wm * WM + i * 16 + (lane & 15);
      if (row >= mlim) continue;
      T* o = (T*)p.out + (size_t)row * p.n;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        store4<T>(o, n0 + wn * WN + j * 16 + (lane >> 4) * 4, p.n, vec, v);
      }
    }
  }
  // requests into LDS land before the workgroup ends
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ---- few rows -------------------------------------------------------------------

// At most a few rows to a weight: the weight's bytes are what counts, each is
// read once from memory straight into registers.  Eight waves: NT blocks of 16
// columns, each of them shared by 8 / NT waves that take every (8 / NT)-th
// slice of K and are summed through LDS.
template <int NT, int BKIND, int OUT, bool GRP>
__global__ __launch_bounds__(512) void fp8_few_kernel(Fp8Gemm p) {
  constexpr int KS = 8 / NT;
  static_assert(OUT != FP8_OUT_RELU2Q || NT == 8, "whole blocks of 128 columns");
  __shared__ __attribute__((aligned(16))) f32x4 part[KS > 1 ? 8 * 64 : 1];
  __shared__ unsigned amax[8][16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = wave % NT, ks = wave / NT;
  const int Kb = (p.k + 127) / 128, Kp = Kb * 128;
  const int c0 = blockIdx.x * NT * 16 + nt * 16, g = blockIdx.y;
  int lo = 0, hi = p.m;
  if constexpr (GRP) {
    // as find_range: from the largest offset before
    for (int i = lane; i <= g; i += 64) lo = max(lo, i > 0 ? p.off[i] : 0);
    hi = g == p.groups ? p.m : p.off[g + 1];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) lo = max(lo, __shfl_xor(lo, d));
    lo = __builtin_amdgcn_readfirstlane(min(lo, p.m));
    hi = min(max(hi, lo), p.m);
    if (g == p.groups) {  // rows of no range
      if constexpr (OUT != FP8_OUT_RELU2Q) {
        typedef typename OutType<OUT>::type T;
        for (int i = tid; i < (hi - lo) * NT * 16; i += 512) {
          const int row = lo + i / (NT * 16), c = blockIdx.x * NT * 16 + i % (NT * 16);
          if (c < p.n) ((T*)p.out)[(size_t)row * p.n + c] = from_f<T>(0.f);
        }
      }
      return;
    }
  }
  const unsigned char* brow = p.b + ((size_t)g * p.n + min(c0 + (lane & 15), p.n - 1)) * Kp + (lane >> 4) * 16;
  const float* sbp = BKIND == FP8_TILES
                         ? p.sb + ((size_t)g * ((p.n + 127) / 128) + min(c0 / 128, (p.n + 127) / 128 - 1)) * Kb
                         : p.sb;
  for (int m0 = lo; m0 < hi; m0 += 16) {
    const int row = m0 + (lane & 15), arow = min(row, hi - 1);
    const unsigned char* ar = p.a + (size_t)arow * Kp + (lane >> 4) * 16;
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int kb = ks; kb < Kb; kb += KS) {
      const i32x8 fb = join(*(const u32x4*)(brow + kb * 128), *(const u32x4*)(brow + kb * 128 + 64));
      const i32x8 fa = join(*(const u32x4*)(ar + kb * 128), *(const u32x4*)(ar + kb * 128 + 64));
      const float sa = p.sa[(size_t)kb * p.m + arow];
      const f32x4 t = mma128(widen(fb), widen(fa));
      if constexpr (BKIND == FP8_TILES) {
        const float f = sa * sbp[kb];
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[q] = __builtin_fmaf(t[q], f, acc[q]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[q] = __builtin_fmaf(t[q] * sbp[(size_t)kb * p.n + min(c0 + (lane >> 4) * 4 + q, p.n - 1)], sa, acc[q]);
      }
    }
    if constexpr (KS > 1) {
      part[wave * 64 + lane] = acc;
      __syncthreads();
      if (ks == 0) {
#pragma unroll
        for (int s = 1; s < KS; ++s) {
          const f32x4 v = part[(s * NT + nt) * 64 + lane];
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[q] += v[q];
        }
      }
      __syncthreads();
      if (ks != 0) continue;
    }
    const int c = c0 + (lane >> 4) * 4;
    if constexpr (OUT == FP8_OUT_RELU2Q) {
      unsigned am = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float z = acc[q] < 0.f ? 0.f : acc[q];
        acc[q] = c + q < p.n ? z * z : 0.f;
        am = umax(am, abs_bits(acc[q]));
      }
      am = umax(am, (unsigned)__shfl_xor((int)am, 16));
      am = umax(am, (unsigned)__shfl_xor((int)am, 32));
      if (lane < 16) amax[wave][lane] = am;
      __syncthreads();
#pragma unroll
      for (int s = 0; s < 8; ++s) am = umax(am, amax[s][lane & 15]);
      __syncthreads();
      const Fp8Factors fc = fp8_factors(am);
      const int Np = (p.n + 127) / 128 * 128;
      if (row < hi) {
        *(unsigned*)((unsigned char*)p.out + (size_t)row * Np + c) =
            fp8_pack4(acc[0] * fc.up, acc[1] * fc.up, acc[2] * fc.up, acc[3] * fc.up);
        if (wave == 0 && lane < 16) p.out_s[(size_t)blockIdx.x * p.m + row] = fc.down;
      }
    } else {
      typedef typename OutType<OUT>::type T;
      const float v[4] = {acc[0], acc[1], acc[2], acc[3]};
      if (row < hi) store4<T>((T*)p.out + (size_t)row * p.n, c, p.n, p.n % 4 == 0, v);
    }
  }
}

template <int BM, int BN, int WGM, int WGN, int ST, int BKIND, int OUT, bool GRP, bool EX>
hipError_t run_tile(const Fp8Gemm& p, hipStream_t s) {
  const int tiles_n = (p.n + BN - 1) / BN;
  const int tiles_m = (p.m + BM - 1) / BM + (GRP ? p.groups : 0);
  launch_kernel((fp8_tile_kernel<BM, BN, WGM, WGN, ST, BKIND, OUT, GRP, EX>), dim3(tiles_m * tiles_n),
                dim3(WGM * WGN * 64), 0, s, p, tiles_m, tiles_n, walk_group_m(tiles_m, tiles_n, BM, BN));
  return hipGetLastError();
}

template <int NT, int BKIND, int OUT, bool GRP>
hipError_t run_few(const Fp8Gemm& p, hipStream_t s) {
  launch_kernel((fp8_few_kernel<NT, BKIND, OUT, GRP>), dim3((p.n + NT * 16 - 1) / (NT * 16), GRP ? p.groups + 1 : 1),
                dim3(512), 0, s, p);
  return hipGetLastError();
}

template <int BKIND, int OUT, bool GRP, bool EX>
hipError_t run_tiles(const Fp8Gemm& p, hipStream_t s) {
  const long long big = (long long)((p.m + 255) / 256) * ((p.n + 255) / 256);
  if (big >= num_cus() * 3 / 4) return run_tile<256, 256, 4, 2, 2, BKIND, OUT, GRP, EX>(p, s);
  return run_tile<128, 128, 4, 1, 2, BKIND, OUT, GRP, EX>(p, s);
}

template <int BKIND, int OUT, bool GRP>
hipError_t run(const Fp8Gemm& p, hipStream_t s) {
  if (p.m <= 64) return run_few<OUT == FP8_OUT_RELU2Q ? 8 : 1, BKIND, OUT, GRP>(p, s);
  if constexpr (OUT == FP8_OUT_F32 || OUT == FP8_OUT_RELU2Q) {
    if (p.exact) return run_tiles<BKIND, OUT, GRP, true>(p, s);
  }
  return run_tiles<BKIND, OUT, GRP, false>(p, s);
}
template <int BKIND, bool GRP>
hipError_t run_out(const Fp8Gemm& p, hipStream_t s) {
  switch (p.out_kind) {
    case FP8_OUT_F32: return run<BKIND, FP8_OUT_F32, GRP>(p, s);
    case FP8_OUT_F16: return run<BKIND, FP8_OUT_F16, GRP>(p, s);
    case FP8_OUT_BF16: return run<BKIND, FP8_OUT_BF16, GRP>(p, s);
    case FP8_OUT_RELU2Q:
      if constexpr (BKIND == FP8_TILES && GRP) return run<BKIND, FP8_OUT_RELU2Q, GRP>(p, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_fp8_gemm(const Fp8Gemm& p, hipStream_t s) {
  hipError_t e = hipErrorInvalidValue;
  if (p.b_kind == FP8_TILES) e = p.off ? run_out<FP8_TILES, true>(p, s) : run_out<FP8_TILES, false>(p, s);
  else if (!p.off) e = run_out<FP8_ROWS, false>(p, s);
  return mark(e, "fp8_gemm", s);
}

}  // namespace rwkvmoe
