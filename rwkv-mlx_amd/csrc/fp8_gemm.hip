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

// The same with the operands in accumulation registers and the result in
// ordinary ones, which the fmas read: with more than 256 registers the compiler
// itself would put the result the other way round and copy it.  The result is
// there after 8 passes: two more of these have to be issued before it is read.
RWKV_DEV void mma128_to(f32x4& d, i32x8 a, i32x8 b) {
  asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, %1, %2, 0" : "=v"(d) : "a"(a), "a"(b));
}
RWKV_DEV void pin(f32x4& v) { asm volatile("" : "+v"(v)); }

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

// Four values at any multiple of their size: one store.
template <typename T> struct Four {
  T e[4];
};

template <int OUT> struct OutType { typedef float type; };
template <> struct OutType<FP8_OUT_F16> { typedef f16 type; };
template <> struct OutType<FP8_OUT_BF16> { typedef bf16 type; };

// ---- tiles --------------------------------------------------------------------

// The rows a tile row covers: [lo, hi) of group g (p.groups: the rows after the
// last range, which become 0).
struct Range {
  int lo, hi, g;
};

// Tile rows of BM rows of every group, for the whole launch: lane l keeps group
// l's range and the tile rows up to its end (up to 63 groups), else they are
// summed again for every tile.  Ranges are clamped to the rows and do not
// overlap, whatever the offsets hold.
template <int BM> struct Ranges {
  int lo, hi, sum, total;
  bool kept;

  // Groups g0 .. g0 + 63; edge: the row they start from.
  static RWKV_DEV void scan(const Fp8Gemm& p, int g0, int edge, int* lo, int* hi, int* sum) {
    const int lane = threadIdx.x & 63, g = g0 + lane;
    int h = g < p.groups ? min(max(p.off[g + 1], 0), p.m) : g == p.groups ? p.m : 0;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(h, d);
      if (lane >= d) h = max(h, v);
    }
    h = max(h, edge);
    int l = __shfl_up(h, 1);
    if (lane == 0) l = edge;
    int n = (h - l + BM - 1) / BM;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(n, d);
      if (lane >= d) n += v;
    }
    *lo = l;
    *hi = h;
    *sum = n;
  }
  RWKV_DEV void init(const Fp8Gemm& p) {
    kept = p.groups < 64;
    total = 0;
    int edge = 0;
    for (int g0 = 0; g0 <= p.groups; g0 += 64) {
      scan(p, g0, edge, &lo, &hi, &sum);
      edge = __builtin_amdgcn_readlane(hi, 63);
      total += __builtin_amdgcn_readlane(sum, 63);
    }
  }
  RWKV_DEV Range find(const Fp8Gemm& p, int mt) {
    int g0 = 0, before = 0;
    if (!kept) {
      int edge = 0;
      for (;; g0 += 64) {
        scan(p, g0, edge, &lo, &hi, &sum);
        const int n = __builtin_amdgcn_readlane(sum, 63);
        if (mt < before + n) break;
        before += n;
        edge = __builtin_amdgcn_readlane(hi, 63);
      }
    }
    const int f = __builtin_amdgcn_readfirstlane(__popcll(__ballot(before + sum <= mt)));
    const int prev = f > 0 ? __builtin_amdgcn_readlane(sum, f - 1) : 0;
    return {__builtin_amdgcn_readlane(lo, f) + (mt - before - prev) * BM, __builtin_amdgcn_readlane(hi, f), g0 + f};
  }
};

template <int N> struct Int { static constexpr int value = N; };

// A BM x BN tile, WGM x WGN waves, one wave a SIMD: the registers of two hold
// a bigger tile and the fragments ahead.  K is walked in slices of one block
// (128 bytes a row), which go straight from memory into LDS rings.
//   * A slice is MI x NI steps: one MFMA, and the four fmas that scale the
//     result of two steps before.  Rows of b (fragments j) stream through four
//     registers sets, three ahead; the rows of a stay for the slice, and the
//     next slice's are read into a second set.
//   * One barrier a slice, three fragments of b before its end: every fragment
//     of the slice has been read then, so its stage takes the requests of the
//     slice after next, and the next slice has to have landed.
//   * Workgroups are persistent and the slices run on across tiles.
// 16384 x 8192 x 2048 bf16: 278-329 us with the card's clock, 1.7-2.0 PFLOP/s
// (a library product of plain e4m3 operands, one scale a matrix: 251).  With
// K = 16384 the loop reaches 2.34 PFLOP/s, and 3.5 with its loads left out: the
// bytes from the L2s into LDS (about 11 TB/s) bound it, and 4 us a tile are the
// stores and the change to the next.
template <int BM, int BN, int WGM, int WGN, int PER_CU, int NB, int BKIND, int OUT, bool GRP, bool EX>
__global__ __launch_bounds__(WGM * WGN * 64, (PER_CU * WGM * WGN + 3) / 4) void fp8_tile_kernel(Fp8Gemm p, int tiles_m,
                                                                                     int tiles_n, int group_m) {
  constexpr int NW = WGM * WGN;
  constexpr int WM = BM / WGM, WN = BN / WGN, MI = WM / 16, NI = WN / 16;
  constexpr int DA = BM / 8 / NW, DB = BN / 8 / NW;  // 1 KB requests of a wave a slice
  static_assert(DA * 8 * NW == BM && DB * 8 * NW == BN, "requests");
  // 256 B requests of scales: with a its rows' and the weight blocks', with b its columns'
  constexpr bool ROWS = BKIND == FP8_ROWS;
  constexpr int SA = BM / 64, SB = BN / 64;
  static_assert(SA + 1 <= NW && SB <= NW, "one request of scales a wave");
  constexpr int DAS = DA + 1, DBS = DB + (ROWS ? 1 : 0);
  static_assert(128 % WN == 0 || WN == 128, "a wave's columns share one weight block");
  static_assert(OUT != FP8_OUT_RELU2Q || WN == 128, "a wave holds whole blocks of its rows");
  constexpr int UA = BM * 128, UB = BN * 128 + (ROWS ? NW * 256 : 0), US = NW * 256;
  constexpr int STA = UA + US, B0 = 2 * STA;         // a's stages, then b's
  constexpr int LDS_BYTES = B0 + NB * UB;
  static_assert(PER_CU * LDS_BYTES <= 163840, "LDS");
  constexpr bool ONE = NW * PER_CU == 4;             // one wave a SIMD
  static_assert(!(ONE && EX), "the fp16 form is the compiler's");
  constexpr int JB = NI - 3;                         // the barrier is in front of fragment JB of b
  static_assert(NI % 4 == 0, "four fragments of b in turn");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[LDS_BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WGN, wn = wave % WGN;
  const int Kb = (p.k + 127) / 128, Kp = Kb * 128, Nb = (p.n + 127) / 128;

  // XCD w % 8 takes a contiguous run of the tiles, group_m tile rows at a time
  Ranges<BM> ranges;
  if constexpr (GRP) {
    ranges.init(p);
    tiles_m = ranges.total;
  }
  const int total = tiles_m * tiles_n, G = gridDim.x, w = blockIdx.x, xcd = w & 7;
  const int step = (G - xcd + 7) >> 3, run = total / 8 + (xcd < total % 8 ? 1 : 0);
  const int base = xcd * (total / 8) + min(xcd, total % 8) + (w >> 3);
  const int count = (w >> 3) < run ? (run - (w >> 3) + step - 1) / step : 0;
  if (count == 0) return;
  struct Tile {
    int m0, mlim, n0, g;
  };
  auto tile_of = [&](int i) __attribute__((always_inline)) -> Tile {
    const int l = base + i * step, in_group = group_m * tiles_n, first = (l / in_group) * group_m;
    const int gsize = min(tiles_m - first, group_m), mt = first + (l % in_group) % gsize;
    Range r{mt * BM, p.m, 0};
    if constexpr (GRP) r = ranges.find(p, mt);
    return {r.lo, min(r.hi, r.lo + BM), ((l % in_group) / gsize) * BN, r.g};
  };

  // ---- requests: slice kb of tile i of a (with the scales), and of b further on ----
  struct Ahead {
    int i, kb;
  };
  Ahead da{0, 0}, db{0, 0};
  __amdgpu_buffer_rsrc_t ra, rb;
  unsigned va[DA], vb[DB];
  // this wave's 64 scales of the present slice of a: of its rows (wave w < SA: rows 64·w on, further waves the last
  // ones again), or of the tile's weight blocks; and of the present slice of b, of its columns
  const bool blocks = !ROWS && wave >= SA;
  const float *sap = nullptr, *sbp = nullptr;
  unsigned sa_bytes = 0, sb_bytes = 0, sa_at = 0;
  auto open_a = [&]() __attribute__((always_inline)) {
    const Tile t = tile_of(da.i);
    int sl = lane;  // (opaque: addresses that depend on the lane alone would be kept in registers)
    asm volatile("" : "+v"(sl));
    ra = buf_rsrc(p.a + (size_t)t.m0 * Kp, 0xFFFFFFF0u);
#pragma unroll
    for (int i = 0; i < DA; ++i) {
      const int row = (wave * DA + i) * 8 + (sl >> 3);
      // rows past the end read the last one
      va[i] = (unsigned)(min(t.m0 + row, t.mlim - 1) - t.m0) * (unsigned)Kp + ((sl & 7) ^ swz(row)) * 16;
    }
    if (blocks) {
      const int nb = t.n0 / 128;
      sap = p.sb + ((size_t)(GRP ? min(t.g, p.groups - 1) : 0) * Nb + nb) * Kb;
      sa_at = BN / 128 > 1 && nb + 1 < Nb ? (sl & 1) * Kb * 4 : 0;
      sa_bytes = 0xFFFFFFF0u;
    } else {
      sap = p.sa + t.m0;
      sa_at = (min(wave, SA - 1) * 64 + sl) * 4;
      sa_bytes = (t.mlim - t.m0) * 4;
    }
  };
  auto open_b = [&]() __attribute__((always_inline)) {
    const Tile t = tile_of(db.i);
    int sl = lane;
    asm volatile("" : "+v"(sl));
    const int g = GRP ? min(t.g, p.groups - 1) : 0;  // (tiles of no range multiply anything)
    rb = buf_rsrc(p.b + ((size_t)g * p.n + t.n0) * Kp, 0xFFFFFFF0u);
#pragma unroll
    for (int i = 0; i < DB; ++i) {
      const int row = (wave * DB + i) * 8 + (sl >> 3);
      vb[i] = (unsigned)(min(t.n0 + row, p.n - 1) - t.n0) * (unsigned)Kp + ((sl & 7) ^ swz(row)) * 16;
    }
    if constexpr (ROWS) {
      sbp = p.sb + t.n0;
      sb_bytes = min(BN, p.n - t.n0) * 4;
    }
  };
  // (past the last slice it is requested again, into a stage that nothing reads any more)
  auto advance_a = [&]() __attribute__((always_inline)) {
    if (da.kb + 1 < Kb) {
      ++da.kb;
      sap += blocks ? 1 : p.m;
    } else if (da.i + 1 < count) {
      ++da.i;
      da.kb = 0;
      open_a();
    }
  };
  auto advance_b = [&]() __attribute__((always_inline)) {
    if (db.kb + 1 < Kb) {
      ++db.kb;
      if constexpr (ROWS) sbp += p.n;
    } else if (db.i + 1 < count) {
      ++db.i;
      db.kb = 0;
      open_b();
    }
  };
  auto request_a = [&](int stage, int q) __attribute__((always_inline)) {
    unsigned char* st = lds + stage;
    if (q < DA) load_lds16(ra, st + (wave * DA + q) * 1024, va[q], (unsigned)da.kb * 128u);
    else load_lds4(buf_rsrc(sap, sa_bytes), st + UA + wave * 256, sa_at);
  };
  auto request_b = [&](int stage, int q) __attribute__((always_inline)) {
    unsigned char* st = lds + stage;
    if (q < DB) load_lds16(rb, st + (wave * DB + q) * 1024, vb[q], (unsigned)db.kb * 128u);
    else load_lds4(buf_rsrc(sbp, sb_bytes), st + BN * 128 + wave * 256, (min(wave, SB - 1) * 64 + lane) * 4);
  };

  // ---- fragments ----
  const int fsw = swz(lane & 15), fch = lane >> 4;
  const int ao = (wm * WM + (lane & 15)) * 128 + ((fch ^ fsw) << 4);
  const int bo = B0 + (wn * WN + (lane & 15)) * 128 + ((fch ^ fsw) << 4);
  const int so = UA + (wm * WM + (lane & 15)) * 4;
  // b's scales of this wave's columns: by column, or one for all
  const int co = ROWS ? B0 + BN * 128 + (wn * WN + (lane >> 4) * 4) * 4 : UA + SA * 256 + wn * WN / 128 * 4;
  const int a1 = ao ^ 64, b1 = bo ^ 64;  // the second chunk
  auto frag = [&](int at, int at1) __attribute__((always_inline)) {
    return join(*(const u32x4*)(lds + at), *(const u32x4*)(lds + at1));
  };

  f32x4 acc[MI][NI];
  auto zero_acc = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  i32x8 fa[MI], ga[MI], fb[4];
  f32x4 cs[BKIND == FP8_ROWS ? 4 : 1];
  float f[MI], sa[MI], sb = 1.f;

  // stores of whole 16 bytes, NST of them a tile, which may be in flight through the next tile's first slice
  constexpr int NST = OUT == FP8_OUT_F32 ? MI * NI : OUT == FP8_OUT_RELU2Q ? MI * (NI / 4 + 1) : MI * NI / 2;
  constexpr int WV = DAS + (NB - 2) * DBS;  // requests behind the slice that has to have landed
  static_assert(WV + NST < 64, "vmcnt range");
  const bool whole = OUT == FP8_OUT_RELU2Q || p.n % (OUT == FP8_OUT_F32 ? 4 : 8) == 0;
  bool stores = false;
  auto epilogue = [&](const Tile& it) __attribute__((always_inline)) {
    int el = lane;
    asm volatile("" : "+v"(el));
    if constexpr (OUT == FP8_OUT_RELU2Q) {
      const int col0 = it.n0 + wn * WN, Np = Nb * 128;
      const int rows = GRP && it.g == p.groups ? 0 : it.mlim - it.m0;  // (rows of no range are not read)
      const __amdgpu_buffer_rsrc_t ro =
          buf_rsrc((unsigned char*)p.out + (size_t)it.m0 * Np, (unsigned)rows * (unsigned)Np);
      const __amdgpu_buffer_rsrc_t rs =
          buf_rsrc(p.out_s + (size_t)(col0 / 128) * p.m + it.m0, (unsigned)rows * 4u);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int row = it.m0 + wm * WM + i * 16 + (el & 15);
        unsigned am = 0;
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float v = acc[i][j][q], z = v < 0.f ? 0.f : v;  // (a NaN stays one)
            acc[i][j][q] = col0 + j * 16 + (el >> 4) * 4 + q < p.n ? z * z : 0.f;
            am = umax(am, abs_bits(acc[i][j][q]));
          }
        am = umax(am, (unsigned)__shfl_xor((int)am, 16));
        am = umax(am, (unsigned)__shfl_xor((int)am, 32));
        const Fp8Factors fc = fp8_factors(am);
        // four blocks of 16 columns, exchanged so that a lane of 16-lane row r holds block r's 16 bytes: a store
        // covers 64 consecutive bytes of 16 rows
#pragma unroll
        for (int j = 0; j < NI; j += 4) {
          unsigned w[4];
#pragma unroll
          for (int h = 0; h < 4; ++h)
            w[h] = fp8_pack4(acc[i][j + h][0] * fc.up, acc[i][j + h][1] * fc.up, acc[i][j + h][2] * fc.up,
                             acc[i][j + h][3] * fc.up);
          // w[h], row r: block h's bytes 4r.. -> x[..] of blocks {0, 1} and {2, 3}, then of all four
          const auto x = __builtin_amdgcn_permlane16_swap(w[0], w[1], false, false);
          const auto y = __builtin_amdgcn_permlane16_swap(w[2], w[3], false, false);
          const auto lo = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
          const auto hi = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
          const unsigned off = row < it.mlim && col0 < p.n
                                   ? (unsigned)(row - it.m0) * (unsigned)Np + col0 + (j + (el >> 4)) * 16
                                   : kOOB;
          __builtin_amdgcn_raw_buffer_store_b128(u32x4{lo[0], hi[0], lo[1], hi[1]}, ro, off, 0, 0);
        }
        const unsigned soff = el < 16 && row < it.mlim && col0 < p.n ? (unsigned)(row - it.m0) * 4u : kOOB;
        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, fc.down), rs, soff, 0, 0);
      }
    } else {
      typedef typename OutType<OUT>::type T;
      const bool none = GRP && it.g == p.groups;
      const int rows = it.mlim - it.m0, col0 = it.n0 + wn * WN;
      if (whole) {
        // 16 bytes a lane.  16-bit results: of two blocks of 16 columns, exchanged between the 16-lane rows so that
        // lanes 0-15 and 32-47 hold the first one's two halves, the others the second one's; a store covers 64
        // consecutive bytes of 16 rows.  Offsets past the rows or columns are dropped by the buffer's bound.
        const __amdgpu_buffer_rsrc_t ro =
            buf_rsrc((T*)p.out + (size_t)it.m0 * p.n, (unsigned)rows * (unsigned)p.n * (unsigned)sizeof(T));
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const int row = wm * WM + i * 16 + (el & 15);
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < NI; j += 2) {
              unsigned v[2][2];
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  union { T e[2]; unsigned u; } w;
                  w.e[0] = from_f<T>(none ? 0.f : acc[i][j + h][q * 2]);
                  w.e[1] = from_f<T>(none ? 0.f : acc[i][j + h][q * 2 + 1]);
                  v[h][q] = w.u;
                }
              const auto x = __builtin_amdgcn_permlane16_swap(v[0][0], v[1][0], false, false);
              const auto y = __builtin_amdgcn_permlane16_swap(v[0][1], v[1][1], false, false);
              const int c = col0 + (j + ((el >> 4) & 1)) * 16 + (el >> 5) * 8;
              const unsigned off = c < p.n ? ((unsigned)row * (unsigned)p.n + c) * 2u : kOOB;
              __builtin_amdgcn_raw_buffer_store_b128(u32x4{x[0], y[0], x[1], y[1]}, ro, off, 0, 0);
            }
          } else {
#pragma unroll
            for (int j = 0; j < NI; ++j) {
              const int c = col0 + j * 16 + (el >> 4) * 4;
              const unsigned off = c < p.n ? ((unsigned)row * (unsigned)p.n + c) * 4u : kOOB;
              f32x4 v = acc[i][j];
              if (none) v = f32x4{0.f, 0.f, 0.f, 0.f};
              __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), ro, off, 0, 0);
            }
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const int row = wm * WM + i * 16 + (el & 15);
          if (row < rows) {
            T* o = (T*)p.out + (size_t)(it.m0 + row) * p.n;
#pragma unroll
            for (int j = 0; j < NI; ++j) {
              const int c = col0 + j * 16 + (el >> 4) * 4;
              Four<T> w;
#pragma unroll
              for (int q = 0; q < 4; ++q) w.e[q] = from_f<T>(none ? 0.f : acc[i][j][q]);
              if (c + 4 <= p.n) {
                *(Four<T>*)(o + c) = w;
              } else {
#pragma unroll
                for (int q = 0; q < 3; ++q)
                  if (c + q < p.n) o[c + q] = w.e[q];
              }
            }
          }
        }
      }
    }
  };

  // One slice: a's rows in xa, its stage `cur`; the next slice's (stage nxt)
  // into ya.  b_cur, b_nxt: b's stages.  The fmas of a slice's last two steps
  // follow the next slice's first two, with the factors g.
  int b_cur = 0, b_nxt = UB;
  f32x4 t[4];
  f32x4 tc[ROWS ? 2 : 1];  // b's column scales of those steps
  float g[2];
  constexpr int NS = MI * NI;
  static_assert(MI >= 2 && NS % 4 == 0, "four results in turn");
  auto scale = [&](int s, float fs, const f32x4& c) __attribute__((always_inline)) {
    const int i = s % MI, j = s / MI;
    const f32x4 v = t[s % 4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      acc[i][j][q] = __builtin_fmaf(ROWS ? v[q] * c[q] : v[q], fs, acc[i][j][q]);
    pin(acc[i][j]);  // (not later than here)
  };
  auto nothing_pending = [&]() __attribute__((always_inline)) {
    t[2] = t[3] = f32x4{0.f, 0.f, 0.f, 0.f};
    g[0] = g[1] = 0.f;
    if constexpr (ROWS) tc[0] = tc[1] = t[2];
  };
  // the fmas that a slice leaves to the next
  auto flush = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (ONE) asm volatile("s_nop 15" ::: "memory");
    pin(t[2]);
    pin(t[3]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int h = 0; h < 2; ++h) scale(NS - 2 + h, g[h], tc[ROWS ? h : 0]);
  };
  auto slice = [&](i32x8 (&xa)[MI], i32x8 (&ya)[MI], int cur, int nxt) __attribute__((always_inline)) {
    const int vb0 = bo + b_cur, vb1 = b1 + b_cur, wb0 = bo + b_nxt, wb1 = b1 + b_nxt;
#pragma unroll
    for (int i = 0; i < MI; ++i) f[i] = sa[i] * sb;
    f32x4 cj{1.f, 1.f, 1.f, 1.f}, cl = cj;  // b's column scales of this fragment, and of the one before
    auto steps = [&](auto from, auto to) __attribute__((always_inline)) {
#pragma unroll
      for (int s = decltype(from)::value; s < decltype(to)::value; ++s) {
        const int j = s / MI, i = s % MI;
        const auto w = Operand<EX>::of(fb[j & 3]);
        if constexpr (ONE) mma128_to(t[s % 4], w, xa[i]);
        else t[s % 4] = mma128(w, Operand<EX>::of(xa[i]));
        // (the fmas of two steps before: not before this point)
        pin(t[(s + 2) % 4]);
        __builtin_amdgcn_sched_barrier(0);
        if (i == 0) {  // fragment j + 3 of b, from NI on the next slice's
          const int e = j + 3;
          fb[e & 3] = e < NI ? frag(vb0 + e * 2048, vb1 + e * 2048) : frag(wb0 + (e - NI) * 2048, wb1 + (e - NI) * 2048);
          if constexpr (ROWS) {
            cl = cj;
            cj = cs[j & 3];
            cs[e & 3] = *(const f32x4*)(lds + (e < NI ? b_cur : b_nxt) + co + (e % NI) * 64);
          }
        }
        if (j >= 1 && j < JB) {
#pragma unroll
          for (int q = 0; q < DAS; ++q)
            if (q * (JB - 1) * MI / DAS == s - MI) request_a(cur, q);
        }
        if (j >= JB) {
          const int u = s - JB * MI;  // of 3 · MI
          if (u % 3 == 1) {
            ya[u / 3] = frag(nxt + ao + (u / 3) * 2048, nxt + a1 + (u / 3) * 2048);
            sa[u / 3] = *(const float*)(lds + nxt + so + (u / 3) * 64);
            if (!ROWS && u == 1) sb = *(const float*)(lds + nxt + co);
          }
#pragma unroll
          for (int q = 0; q < DBS; ++q)
            if (q * 3 * MI / DBS == u) request_b(B0 + b_cur, q);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (s < 2) scale(NS - 2 + s, g[s], tc[ROWS ? s : 0]);
        else scale(s - 2, f[(s - 2) % MI], i < 2 ? cl : cj);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    steps(Int<0>{}, Int<MI>{});
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    advance_a();
    steps(Int<MI>{}, Int<JB * MI>{});
    if (stores) {  // (behind them: this slice's requests of a)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(WV + NST) : "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(WV) : "memory");
    }
    stores = false;
    __builtin_amdgcn_sched_barrier(0);
    advance_b();
    steps(Int<JB * MI>{}, Int<NS>{});
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      g[h] = f[MI - 2 + h];
      if constexpr (ROWS) tc[h] = cj;
    }
    b_cur = b_nxt;
    b_nxt = b_nxt == (NB - 1) * UB ? 0 : b_nxt + UB;
  };

  // ---- the first slices: two of a, NB of b ----
  open_a();
  open_b();
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    if (n < 2) {
      if (n > 0) advance_a();
#pragma unroll
      for (int q = 0; q < DAS; ++q) request_a(n * STA, q);
    }
    if (n > 0) advance_b();
#pragma unroll
    for (int q = 0; q < DBS; ++q) request_b(B0 + n * UB, q);
  }
  zero_acc();
  nothing_pending();
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(DAS + (NB - 1) * DBS) : "memory");
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    fa[i] = frag(ao + i * 2048, a1 + i * 2048);
    sa[i] = *(const float*)(lds + so + i * 64);
  }
  if constexpr (BKIND == FP8_TILES) sb = *(const float*)(lds + co);
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    fb[j] = frag(bo + j * 2048, b1 + j * 2048);
    if constexpr (BKIND == FP8_ROWS) cs[j] = *(const f32x4*)(lds + co + j * 64);
  }

  if constexpr (ONE) {
#pragma unroll
    for (int i = 0; i < MI; ++i) asm volatile("" : "+a"(fa[i]));
#pragma unroll
    for (int j = 0; j < 3; ++j) asm volatile("" : "+a"(fb[j]));
  }
  int ci = 0, kb = 0;
  // true after the last slice of the last tile
  auto next = [&]() __attribute__((always_inline)) {
    if (++kb < Kb) return false;
    flush();
    nothing_pending();
    epilogue(tile_of(ci));
    stores = whole;
    if (++ci == count) return true;
    zero_acc();
    kb = 0;
    return false;
  };
  for (;;) {
    slice(fa, ga, 0, STA);
    if (next()) break;
    slice(ga, fa, STA, 0);
    if (next()) break;
    if constexpr (ONE) {  // whole registers go round the loop (halves would be put together again)
#pragma unroll
      for (int i = 0; i < MI; ++i) asm volatile("" : "+a"(fa[i]));
#pragma unroll
      for (int j = 0; j < 3; ++j) asm volatile("" : "+a"(fb[j]));
    }
  }
  // requests into LDS land before the workgroup ends
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ---- few rows -------------------------------------------------------------------

// At most a few rows to a weight: the weight's bytes are what counts, each is
// read once from memory straight into registers.  Eight waves, each with CT
// blocks of 16 columns; NT waves side by side, and 8 / NT share their columns,
// take every (8 / NT)-th slice of K and are summed through LDS.
// RAW: the rows come unrounded, and every wave rounds the blocks it multiplies
// itself, which saves a launch (one bf16 row by 8192 x 2048: kernels of 2.6 and
// 5.4 us against one of 8.2, but a pass from the host 12.9 against 8.6); what
// that costs in every workgroup is shared by its CT blocks.  VEC: their loads
// are 16 bytes.  D: slices whose loads are under way together (past the end: the
// last slice again).  One row by 8192 x 2048: 8.5 us, 17 MB at 2.0 TB/s, of
// which the launch and the chain row - scale - product are the larger part.
template <int NT, int CT, int D, int BKIND, int OUT, bool GRP, bool RAW, bool VEC>
__global__ __launch_bounds__(512) void fp8_few_kernel(Fp8Gemm p) {
  constexpr int KS = 8 / NT, COLS = NT * CT * 16;
  static_assert(OUT != FP8_OUT_RELU2Q || (NT == 8 && CT == 1), "whole blocks of 128 columns");
  __shared__ __attribute__((aligned(16))) f32x4 part[KS > 1 ? CT * 8 * 64 : 1];
  __shared__ unsigned amax[8][16];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = wave % NT, ks = wave / NT;
  const int Kb = (p.k + 127) / 128, Kp = Kb * 128, Nb = (p.n + 127) / 128;
  const int c0 = blockIdx.x * COLS + nt * CT * 16, g = blockIdx.y;
  int lo = 0, hi = p.m;
  if constexpr (GRP) {
    // as Ranges: from the largest offset before
    for (int i = lane; i <= g; i += 64) lo = max(lo, i > 0 ? p.off[i] : 0);
    hi = g == p.groups ? p.m : p.off[g + 1];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) lo = max(lo, __shfl_xor(lo, d));
    lo = __builtin_amdgcn_readfirstlane(min(lo, p.m));
    hi = min(max(hi, lo), p.m);
    if (g == p.groups) {  // rows of no range
      if constexpr (OUT != FP8_OUT_RELU2Q) {
        typedef typename OutType<OUT>::type T;
        for (int i = tid; i < (hi - lo) * COLS; i += 512) {
          const int row = lo + i / COLS, c = blockIdx.x * COLS + i % COLS;
          if (c < p.n) ((T*)p.out)[(size_t)row * p.n + c] = from_f<T>(0.f);
        }
      }
      return;
    }
  }
  const unsigned char* brow[CT];
  const float* sbp[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int c = c0 + ct * 16;
    brow[ct] = p.b + ((size_t)g * p.n + min(c + (lane & 15), p.n - 1)) * Kp + (lane >> 4) * 16;
    sbp[ct] = BKIND == FP8_TILES ? p.sb + ((size_t)g * Nb + min(c / 128, Nb - 1)) * Kb : p.sb;
  }
  for (int m0 = lo; m0 < hi; m0 += 16) {
    const int row = m0 + (lane & 15), arow = min(row, hi - 1);
    f32x4 acc[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) acc[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int k0 = ks; k0 < Kb; k0 += KS * D) {
      u32x4 w[D][CT][2];
#pragma unroll
      for (int d = 0; d < D; ++d)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const unsigned char* bp = brow[ct] + min(k0 + d * KS, Kb - 1) * 128;
          w[d][ct][0] = *(const u32x4*)bp;
          w[d][ct][1] = *(const u32x4*)(bp + 64);
        }
      i32x8 fa[D];
      float sa[D];
      if constexpr (RAW) {
        // this lane's 16 values of either chunk; the block's others lie in the lanes 16, 32 and 48 further on
        typedef typename OutType<OUT>::type T;
        const T* xr = (const T*)p.x + (size_t)arow * p.ldx;
        float v[D][4][8];
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
          for (int h = 0; h < 4; ++h)
            load8<T, VEC>(xr, min(k0 + d * KS, Kb - 1) * 128 + (lane >> 4) * 16 + (h >> 1) * 64 + (h & 1) * 8, p.k,
                          v[d][h]);
#pragma unroll
        for (int d = 0; d < D; ++d) {
          unsigned am = 0;
#pragma unroll
          for (int h = 0; h < 4; ++h) am = umax(am, amax8(v[d][h]));
          am = umax(am, (unsigned)__shfl_xor((int)am, 16));
          am = umax(am, (unsigned)__shfl_xor((int)am, 32));
          const Fp8Factors fx = fp8_factors(am);
          sa[d] = fx.down;
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const unsigned long long q = pack8(v[d][h], fx.up);
            fa[d][h * 2] = (int)(unsigned)q;
            fa[d][h * 2 + 1] = (int)(unsigned)(q >> 32);
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < D; ++d) {
          const int kb = min(k0 + d * KS, Kb - 1);
          const unsigned char* ar = p.a + (size_t)arow * Kp + kb * 128 + (lane >> 4) * 16;
          fa[d] = join(*(const u32x4*)ar, *(const u32x4*)(ar + 64));
          sa[d] = p.sa[(size_t)kb * p.m + arow];
        }
      }
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const int kb = k0 + d * KS;
        if (kb >= Kb) break;
        const Wide wa = widen(fa[d]);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const f32x4 t = mma128(widen(join(w[d][ct][0], w[d][ct][1])), wa);
          if constexpr (BKIND == FP8_TILES) {
            const float f = sa[d] * sbp[ct][kb];
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[ct][q] = __builtin_fmaf(t[q], f, acc[ct][q]);
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              acc[ct][q] = __builtin_fmaf(
                  t[q] * sbp[ct][(size_t)kb * p.n + min(c0 + ct * 16 + (lane >> 4) * 4 + q, p.n - 1)], sa[d],
                  acc[ct][q]);
          }
        }
      }
    }
    if constexpr (KS > 1) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) part[(ct * 8 + wave) * 64 + lane] = acc[ct];
      __syncthreads();
      if (ks == 0) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int s = 1; s < KS; ++s) {
            const f32x4 v = part[(ct * 8 + s * NT + nt) * 64 + lane];
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[ct][q] += v[q];
          }
      }
      __syncthreads();
      if (ks != 0) continue;
    }
    if constexpr (OUT == FP8_OUT_RELU2Q) {
      const int c = c0 + (lane >> 4) * 4;
      unsigned am = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float z = acc[0][q] < 0.f ? 0.f : acc[0][q];  // (a NaN stays one)
        acc[0][q] = c + q < p.n ? z * z : 0.f;
        am = umax(am, abs_bits(acc[0][q]));
      }
      am = umax(am, (unsigned)__shfl_xor((int)am, 16));
      am = umax(am, (unsigned)__shfl_xor((int)am, 32));
      if (lane < 16) amax[wave][lane] = am;
      __syncthreads();
#pragma unroll
      for (int s = 0; s < 8; ++s) am = umax(am, amax[s][lane & 15]);
      __syncthreads();
      const Fp8Factors fc = fp8_factors(am);
      if (row < hi) {
        *(unsigned*)((unsigned char*)p.out + (size_t)row * Nb * 128 + c) =
            fp8_pack4(acc[0][0] * fc.up, acc[0][1] * fc.up, acc[0][2] * fc.up, acc[0][3] * fc.up);
        if (wave == 0 && lane < 16) p.out_s[(size_t)blockIdx.x * p.m + row] = fc.down;
      }
    } else {
      typedef typename OutType<OUT>::type T;
      if (row < hi) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const float v[4] = {acc[ct][0], acc[ct][1], acc[ct][2], acc[ct][3]};
          store4<T>((T*)p.out + (size_t)row * p.n, c0 + ct * 16 + (lane >> 4) * 4, p.n, p.n % 4 == 0, v);
        }
      }
    }
  }
}

template <int BM, int BN, int WGM, int WGN, int PER_CU, int NB, int BKIND, int OUT, bool GRP, bool EX>
hipError_t run_tile(const Fp8Gemm& p, hipStream_t s) {
  const int tiles_n = (p.n + BN - 1) / BN;
  const int tiles_m = (p.m + BM - 1) / BM + (GRP ? p.groups : 0);
  launch_kernel((fp8_tile_kernel<BM, BN, WGM, WGN, PER_CU, NB, BKIND, OUT, GRP, EX>),
                dim3(std::min(tiles_m * tiles_n, num_cus() * PER_CU)), dim3(WGM * WGN * 64), 0, s, p, tiles_m, tiles_n,
                walk_group_m(tiles_m, tiles_n, BM, BN));
  return hipGetLastError();
}

template <int NT, int CT, int D, int BKIND, int OUT, bool GRP>
hipError_t run_few(const Fp8Gemm& p, hipStream_t s) {
  const dim3 grid((p.n + NT * CT * 16 - 1) / (NT * CT * 16), GRP ? p.groups + 1 : 1), block(512);
  if constexpr (OUT != FP8_OUT_RELU2Q && BKIND == FP8_TILES) {
    if (p.x) {
      typedef typename OutType<OUT>::type T;
      const bool vec = p.k % 8 == 0 && (uintptr_t)p.x % 16 == 0 && (p.ldx * sizeof(T)) % 16 == 0;
      if (vec) launch_kernel((fp8_few_kernel<NT, CT, D, BKIND, OUT, GRP, true, true>), grid, block, 0, s, p);
      else launch_kernel((fp8_few_kernel<NT, CT, D, BKIND, OUT, GRP, true, false>), grid, block, 0, s, p);
      return hipGetLastError();
    }
  }
  launch_kernel((fp8_few_kernel<NT, CT, D, BKIND, OUT, GRP, false, true>), grid, block, 0, s, p);
  return hipGetLastError();
}

template <int BKIND, int OUT, bool GRP>
hipError_t run_few_rows(const Fp8Gemm& p, hipStream_t s) {
  if constexpr (OUT == FP8_OUT_RELU2Q) {
    return run_few<8, 1, 2, BKIND, OUT, GRP>(p, s);
  } else {
    // workgroups of 64 columns where they fill the card, so that a row's block is rounded once for four blocks of
    // columns (16 weights of 4096 x 1024, 24 bf16 rows: 19 us against 42); slices of K a wave: one or more
    const long long groups = GRP ? std::min(p.groups, p.m) : 1;
    const bool wide = (p.n + 63) / 64 * groups >= 2 * num_cus();
    const bool deep = p.k > 8 * 128;
    if (wide) return deep ? run_few<1, 4, 2, BKIND, OUT, GRP>(p, s) : run_few<1, 4, 1, BKIND, OUT, GRP>(p, s);
    return deep ? run_few<1, 1, 2, BKIND, OUT, GRP>(p, s) : run_few<1, 1, 1, BKIND, OUT, GRP>(p, s);
  }
}

template <int BKIND, int OUT, bool GRP, bool EX>
hipError_t run_tiles(const Fp8Gemm& p, hipStream_t s) {
  // The wide tile reads 0.73 of the 128 x 128 tile's bytes a product, but only
  // one fits a CU: nothing runs beside a tile's first and last slices, and a
  // round of tiles that fills few CUs costs a whole one.  Measured (us, 128 x
  // 128 against 192 x 256): 16384 x 8192 x 2048 311, 288; 3000 x 4096 x 8192
  // 117, 105; 8192 x 8192 x 1024 94, 101; 4096 x 1024 x 4096 (96 wide tiles) 27, 44.
  // Hidden rows are half the bytes of 16-bit results, so their epilogue pays for
  // itself sooner: 32496 rows of 32 experts x 4096 x 1024 285, 249.
  // Where 128 x 128 tiles leave half of the CUs idle, or are a quarter more than
  // there are CUs at most, so that few CUs take two, 64 x 128 ones read more but
  // are sooner done (us, 128 x 128 against 64 x 128; in brackets the tiles a CU):
  // 200 x 4096 x 1024 (1/4) 9.4, 8.1; 1024 x 2048 x 1024 (1/2) 9.4, 8.6;
  // 300 x 8192 x 8192 (3/4) 45.8, 51.8; 2048 x 2048 x 1024 (1) 10.4, 11.6;
  // 300 x 12288 x 2048 (1.1) 20.9, 18.3; 2560 x 2048 x 4096 (1.25) 37.7, 36.4;
  // 2048 x 3584 x 1024 (1.75) 15.1, 17.8.
  if constexpr (BKIND == FP8_TILES) {
    const long long cus = num_cus();
    auto tiles = [&](int bm, int bn) {
      return ((p.m + bm - 1) / bm + (GRP ? p.groups / 2 : 0)) * (long long)((p.n + bn - 1) / bn);
    };
    if constexpr (!EX) {
      const long long wide = tiles(192, 256);
      if (p.k > (OUT == FP8_OUT_RELU2Q ? 7 : 11) * 128 && wide * 5 >= (wide + cus - 1) / cus * cus * 4)
        return run_tile<192, 256, 2, 2, 1, 3, BKIND, OUT, GRP, EX>(p, s);
    }
    const long long t = tiles(128, 128);
    if (t * 2 <= cus || (t > cus && t * 4 <= cus * 5))
      return run_tile<64, 128, 2, 1, 3, 2, BKIND, OUT, GRP, EX>(p, s);
  }
  return run_tile<128, 128, 4, 1, 2, 2, BKIND, OUT, GRP, EX>(p, s);
}

template <int BKIND, int OUT, bool GRP>
hipError_t run(const Fp8Gemm& p, hipStream_t s) {
  if (fp8_few(p.m)) return run_few_rows<BKIND, OUT, GRP>(p, s);
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
