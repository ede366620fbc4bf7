// Rounding of matrices to e4m3 blocks (fp8.h): activations in rows of 128
// values, weights in 128 x 128 blocks, each also transposed for the products
// of a backward pass.  All of these move bytes: a pass over x (and its 8-bit
// copy) is what bounds them.
#include "fp8.h"

namespace rwkvmoe {
namespace {

// over the 16 lanes that share a block (a DPP row)
RWKV_DEV unsigned amax16(unsigned a) {
  a = umax(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x128, 0xf, 0xf, false));  // row_ror:8
  a = umax(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x124, 0xf, 0xf, false));
  a = umax(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x122, 0xf, 0xf, false));
  return umax(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x121, 0xf, 0xf, false));
}
// Rows: 16 lanes a block of 128 values, a workgroup 16 rows of one slice of K;
// the scales (kb, row) of the 16 rows are 64 consecutive bytes.  Workgroups run
// along K first, so that those under way together read whole rows.  16384 x
// 2048 bf16: 23.6 us, 101 MB at 4.3 TB/s (four slices a thread: 31 against 28).
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void fp8_quant_rows_kernel(const T* __restrict__ x, int rows, int cols, long long ld,
                                                             unsigned char* __restrict__ q, float* __restrict__ s) {
  const int Kb = (cols + kFp8Block - 1) / kFp8Block;
  const int row = blockIdx.x / Kb * 16 + (threadIdx.x >> 4), kb = blockIdx.x % Kb;
  if (row >= rows) return;  // (whole 16-lane blocks)
  const int c = kb * kFp8Block + (threadIdx.x & 15) * 8;
  float v[8];
  load8<T, VEC>(x + (size_t)row * ld, c, cols, v);
  const Fp8Factors f = fp8_factors(amax16(amax8(v)));
  *(unsigned long long*)(q + (size_t)row * Kb * kFp8Block + c) = pack8(v, f.up);
  if ((threadIdx.x & 15) == 0) s[(size_t)kb * rows + row] = f.down;
}

// A 128 x 128 block of x by 512 threads, thread (g, c8) rows 4g.. and columns
// 8·c8..; its maxima by row, by column or over all, the transposed bytes through
// LDS so that they leave in whole lines.
//   ROWS   q in rows (row maxima), qt in columns (column maxima)
//   TILES  q and qt with the block's maximum
// 4096 x 4096 bf16 in rows and columns: 16.8 us, 67 MB at 4.0 TB/s.
template <typename T, bool VEC, bool TILES>
__global__ __launch_bounds__(512) void fp8_quant_block_kernel(const T* __restrict__ x, int rows, int cols,
                                                              long long ld, unsigned char* __restrict__ q,
                                                              float* __restrict__ s, unsigned char* __restrict__ qt,
                                                              float* __restrict__ st) {
  constexpr int R = 4, P = 33;  // rows of a thread; dwords between columns of the transposed bytes
  __shared__ unsigned tile[128 * P];
  __shared__ unsigned cmax[8][128];
  __shared__ float cup[128];
  const int tid = threadIdx.x, c8 = tid & 15, g = tid >> 4, wave = tid >> 6;
  const int rb = blockIdx.y, kb = blockIdx.x, grp = blockIdx.z;
  const int Kb = gridDim.x, Rb = gridDim.y;
  const int r0 = rb * kFp8Block + g * R, c0 = kb * kFp8Block + c8 * 8;
  const T* xg = x + (size_t)grp * rows * ld;
  float v[R][8];
#pragma unroll
  for (int i = 0; i < R; ++i)
    load8<T, VEC>(xg + (size_t)min(r0 + i, rows - 1) * ld, c0, r0 + i < rows ? cols : 0, v[i]);
  float up[R];
  if constexpr (TILES) {
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) a = umax(a, amax8(v[i]));
    a = amax16(a);
    a = umax(a, (unsigned)__shfl_xor((int)a, 16));
    a = umax(a, (unsigned)__shfl_xor((int)a, 32));
    if ((tid & 63) == 0) cmax[0][wave] = a;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) a = umax(a, cmax[0][w]);
    const Fp8Factors f = fp8_factors(a);
#pragma unroll
    for (int i = 0; i < R; ++i) up[i] = f.up;
    if (tid == 0) {
      if (q) s[((size_t)grp * Rb + rb) * Kb + kb] = f.down;
      if (qt) st[((size_t)grp * Kb + kb) * Rb + rb] = f.down;
    }
  } else {
    if (q) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const Fp8Factors f = fp8_factors(amax16(amax8(v[i])));
        up[i] = f.up;
        if (c8 == 0 && r0 + i < rows) s[(size_t)kb * rows + r0 + i] = f.down;
      }
    }
    if (qt) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        unsigned a = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) a = umax(a, abs_bits(v[i][j]));
        a = umax(a, (unsigned)__shfl_xor((int)a, 16));
        a = umax(a, (unsigned)__shfl_xor((int)a, 32));
        if ((tid & 63) < 16) cmax[wave][c8 * 8 + j] = a;
      }
      __syncthreads();
      if (tid < 128) {
        unsigned a = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) a = umax(a, cmax[w][tid]);
        const Fp8Factors f = fp8_factors(a);
        cup[tid] = f.up;
        if (kb * kFp8Block + tid < cols) st[(size_t)rb * cols + kb * kFp8Block + tid] = f.down;
      }
      __syncthreads();
    }
  }
  if (q) {
    unsigned char* qg = q + (size_t)grp * rows * Kb * kFp8Block;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (r0 + i < rows)
        *(unsigned long long*)(qg + ((size_t)(r0 + i) * Kb + kb) * kFp8Block + c8 * 8) = pack8(v[i], up[i]);
  }
  if (qt) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float u = TILES ? up[0] : cup[c8 * 8 + j];
      tile[(c8 * 8 + j) * P + g] = fp8_pack4(v[0][j] * u, v[1][j] * u, v[2][j] * u, v[3][j] * u);
    }
    __syncthreads();
    unsigned char* tg = qt + (size_t)grp * cols * Rb * kFp8Block;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = i * 16 + (tid >> 5), d = tid & 31;
      if (kb * kFp8Block + c < cols)
        *(unsigned*)(tg + ((size_t)(kb * kFp8Block + c) * Rb + rb) * kFp8Block + d * 4) = tile[c * P + d];
    }
  }
}

// A checkpoint's e4m3 values (rows, cols) into padded rows and, with qt, their
// transpose; the block scales are copied and transposed.
__global__ __launch_bounds__(256) void fp8_layout_kernel(const unsigned char* __restrict__ src,
                                                         const float* __restrict__ ss, int rows, int cols,
                                                         unsigned char* __restrict__ q, float* __restrict__ s,
                                                         unsigned char* __restrict__ qt, float* __restrict__ st) {
  __shared__ unsigned char tile[128][136];
  const int rb = blockIdx.y, kb = blockIdx.x, grp = blockIdx.z, Kb = gridDim.x, Rb = gridDim.y;
  const unsigned char* sg = src + (size_t)grp * rows * cols;
  for (int i = threadIdx.x; i < 128 * 128; i += 256) {
    const int r = i >> 7, c = i & 127, gr = rb * 128 + r, gc = kb * 128 + c;
    tile[r][c] = gr < rows && gc < cols ? sg[(size_t)gr * cols + gc] : 0;
  }
  if (threadIdx.x == 0) {
    const float v = ss[((size_t)grp * Rb + rb) * Kb + kb];
    s[((size_t)grp * Rb + rb) * Kb + kb] = v;
    if (qt) st[((size_t)grp * Kb + kb) * Rb + rb] = v;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 128 * 16; i += 256) {
    const int r = i >> 4, c = (i & 15) * 8;
    if (rb * 128 + r < rows)
      *(unsigned long long*)(q + (((size_t)grp * rows + rb * 128 + r) * Kb + kb) * 128 + c) =
          *(const unsigned long long*)&tile[r][c];
  }
  if (!qt) return;
  for (int i = threadIdx.x; i < 128 * 16; i += 256) {
    const int c = i >> 4, r = (i & 15) * 8;
    if (kb * 128 + c >= cols) continue;
    union { unsigned char b[8]; unsigned long long u; } w;
#pragma unroll
    for (int j = 0; j < 8; ++j) w.b[j] = tile[r + j][c];
    *(unsigned long long*)(qt + (((size_t)grp * cols + kb * 128 + c) * Rb + rb) * 128 + r) = w.u;
  }
}

template <typename T>
bool vec_rows(const Fp8Quant& p) {
  return p.cols % 8 == 0 && (uintptr_t)p.x % 16 == 0 && (p.ld * sizeof(T)) % 16 == 0;
}

// Token t's mixed row for expert e in fp32 (one rounding, to e4m3, follows); as
// the rows kernel, one slice of K a workgroup.  The order's three dependent
// loads stand before the row's: 32496 rows of 1024 bf16 28-30 us, of which
// about 10 are the bytes (two slices a thread 28, four 36).
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void fp8_mix_kernel(const T* __restrict__ x, const T* __restrict__ xprev,
                                                      const T* __restrict__ mu, const int* __restrict__ perm,
                                                      const int* __restrict__ inds, const int* __restrict__ off,
                                                      int nk, int T_, int C, int E, int k,
                                                      unsigned char* __restrict__ q, float* __restrict__ s) {
  const int Kb = (C + kFp8Block - 1) / kFp8Block;
  const int j = blockIdx.x / Kb * 16 + (threadIdx.x >> 4), kb = blockIdx.x % Kb;
  if (j >= off[E]) return;  // (assignments of no expert are not in perm)
  const int a = perm[j], t = a / k, e = inds[a];
  const int c = kb * kFp8Block + (threadIdx.x & 15) * 8;
  const T* prev = t % T_ > 0 ? x + (size_t)(t - 1) * C : xprev ? xprev + (size_t)(t / T_) * C : nullptr;
  float v[8], pv[8], m[8];
  load8<T, VEC>(x + (size_t)t * C, c, C, v);
  load8<T, VEC>(prev ? prev : x, c, prev ? C : 0, pv);
  load8<T, VEC>(mu + (size_t)e * C, c, C, m);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = v[i] + (pv[i] - v[i]) * m[i];
  const Fp8Factors f = fp8_factors(amax16(amax8(v)));
  *(unsigned long long*)(q + (size_t)j * Kb * kFp8Block + c) = pack8(v, f.up);
  if ((threadIdx.x & 15) == 0) s[(size_t)kb * nk + j] = f.down;
}

// Four columns of a token a thread; fp32 sums in the order of the slots.  8124
// tokens of 4 rows of 1024: 31.5 us, 150 MB at 4.8 TB/s, which is what bounds it.
template <typename T>
__global__ __launch_bounds__(256) void fp8_combine_kernel(const float* __restrict__ rows,
                                                          const float* __restrict__ gates,
                                                          const int* __restrict__ inv, const T* __restrict__ resid,
                                                          T* __restrict__ out, int N, int C, int k) {
  const int cpr = C / 4;
  const size_t id = blockIdx.x * (size_t)256 + threadIdx.x;
  if (id >= (size_t)N * cpr) return;
  const size_t t = id / cpr;
  const int c = (int)(id - t * cpr) * 4;
  f32x4 sum{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < k; ++s) {
    const int j = inv[t * k + s];
    if (j < 0) continue;  // an unrouted slot
    const float g = gates[t * k + s];
    const f32x4 v = *(const f32x4*)(rows + (size_t)j * C + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(g, v[i], sum[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float r = resid ? to_f(resid[t * C + c + i]) : 0.f;
    out[t * C + c + i] = from_f<T>(resid ? r + sum[i] : sum[i]);
  }
}

}  // namespace

hipError_t launch_fp8_quant_rows(const Fp8Quant& p, hipStream_t s) {
  const int Kb = fp8_blocks(p.cols);
  RWKV_DISPATCH_DTYPE(p.dtype, T, {
    const bool v = vec_rows<T>(p);
    if (p.qt) {
      launch_kernel(v ? fp8_quant_block_kernel<T, true, false> : fp8_quant_block_kernel<T, false, false>,
                    dim3(Kb, fp8_blocks(p.rows), 1), dim3(512), 0, s, (const T*)p.x, p.rows, p.cols, p.ld, p.q, p.s,
                    p.qt, p.st);
    } else {
      launch_kernel(v ? fp8_quant_rows_kernel<T, true> : fp8_quant_rows_kernel<T, false>,
                    dim3(Kb * ((p.rows + 15) / 16)), dim3(256), 0, s, (const T*)p.x, p.rows, p.cols, p.ld, p.q, p.s);
    }
  });
  return mark(hipGetLastError(), "fp8_quant", s);
}

hipError_t launch_fp8_quant_tiles(const Fp8Quant& p, hipStream_t s) {
  RWKV_DISPATCH_DTYPE(p.dtype, T, {
    launch_kernel(vec_rows<T>(p) ? fp8_quant_block_kernel<T, true, true> : fp8_quant_block_kernel<T, false, true>,
                  dim3(fp8_blocks(p.cols), fp8_blocks(p.rows), p.groups), dim3(512), 0, s, (const T*)p.x, p.rows,
                  p.cols, p.ld, p.q, p.s, p.qt, p.st);
  });
  return mark(hipGetLastError(), "fp8_quant", s);
}

hipError_t launch_fp8_layout(const unsigned char* src, const float* src_s, const Fp8Quant& p, hipStream_t s) {
  launch_kernel(fp8_layout_kernel, dim3(fp8_blocks(p.cols), fp8_blocks(p.rows), p.groups), dim3(256), 0, s, src, src_s,
                p.rows, p.cols, p.q, p.s, p.qt, p.st);
  return mark(hipGetLastError(), "fp8_layout", s);
}

hipError_t launch_fp8_mix(int dtype, const void* x, const void* xprev, const void* mu, const int* perm,
                          const int* inds, const int* off, int N, int T_, int C, int E, int k, unsigned char* q,
                          float* s, hipStream_t st) {
  const int nk = N * k;
  RWKV_DISPATCH_DTYPE(dtype, T, {
    const bool v = C % 8 == 0 && ((uintptr_t)x | (uintptr_t)xprev | (uintptr_t)mu) % 16 == 0;
    launch_kernel(v ? fp8_mix_kernel<T, true> : fp8_mix_kernel<T, false>, dim3(fp8_blocks(C) * ((nk + 15) / 16)), dim3(256), 0, st,
                  (const T*)x, (const T*)xprev, (const T*)mu, perm, inds, off, nk, T_, C, E, k, q, s);
  });
  return mark(hipGetLastError(), "fp8_mix", st);
}

hipError_t launch_fp8_combine(int dtype, const float* rows, const float* gates, const int* inv, const void* resid,
                              void* out, int N, int C, int k, hipStream_t st) {
  const size_t total = (size_t)N * (C / 4);
  RWKV_DISPATCH_DTYPE(dtype, T, {
    launch_kernel(fp8_combine_kernel<T>, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, st, rows, gates, inv,
                  (const T*)resid, (T*)out, N, C, k);
  });
  return mark(hipGetLastError(), "fp8_combine", st);
}

}  // namespace rwkvmoe
