// 8-bit activation checkpoints (act8.h: format): packing, restoring, and GELU with its checkpoint in one pass.
//
// All of these move bytes: a lane takes 8 neighbouring columns, the chunks of a matrix are numbered row by row and dealt to the
// threads in order, so that narrow, wide and odd rows fill the chip alike.  One chunk to a thread: two or four with their loads
// together are no faster (GELU backward 46082 x 4100: 250, 264, 284 us).  Measured (MI355X, kernels alone; a copy reaches 5 TB/s):
//   pack 13826 x 1025 fp32 13 us (5.4 TB/s); restore it with gamma and beta 12 us (one load for each element of gamma: 55 us)
//   GELU forward 13826 x 4100 55 us (5.2 TB/s), 3776 x 4100 17 us; backward 46082 x 4100 246 us (5.4 TB/s), 3776 x 4100 21 us (about 36
//   issue slots an element, 8 of them exp and rcp: two thirds of the time at this size)
#include "act8.h"

// the values of 8 neighbouring codes; zeros behind the row's end
__device__ __forceinline__ void codes_load8(const uint8_t* q, const uint8_t* scale, int c, int d, float (&v)[8]) {
  u32x2 w = {0, 0};
  uint32_t byte = 127;
  if (c < d) { w = *reinterpret_cast<const u32x2*>(q + c); byte = scale[c >> 5]; }
  act8_decode(w, byte, v);
}

// 8 neighbouring columns of a row as floats, zeros behind the row's end (whole: see raw_load8)
template <bool F32>
__device__ __forceinline__ void row_load8(const void* row, int c, int d, bool whole, float (&v)[8]) {
  raw_values8<F32>(raw_load8<F32>(row, c, d, whole), v);
  if (c + 8 > d) {
#pragma unroll
    for (int r = 0; r < 8; ++r) if (c + r >= d) v[r] = 0.f;
  }
}

struct ChunkMap {      // chunk number -> (row, column) for rows of nc chunks
  int64_t rows;
  uint32_t nc;
};

#define A8_THREADS 256

// f(row, c) for this thread's chunk
template <typename F>
__device__ __forceinline__ void for_chunk(const ChunkMap M, F f) {
  const int64_t base = (int64_t)blockIdx.x * A8_THREADS;
  const int64_t row0 = base / M.nc;
  const uint32_t t = (uint32_t)(base - row0 * M.nc) + threadIdx.x;      // < nc + A8_THREADS
  const uint32_t dr = M.nc >= A8_THREADS ? (t >= M.nc ? 1u : 0u) : t / M.nc;
  const int64_t row = row0 + dr;
  if (row < M.rows) f(row, (int)(t - dr * M.nc) * 8);                    // M.nc % 4 == 0: a quad never straddles two rows
}
static bool chunk_grid(int64_t rows, int64_t cols, ChunkMap& M, dim3& grid) {
  if (rows > ((int64_t)1 << 40)) return false;
  M.rows = rows;
  M.nc = (uint32_t)((cols + ACT8_GROUP - 1) / ACT8_GROUP * (ACT8_GROUP / 8));
  const int64_t blocks = (rows * M.nc + A8_THREADS - 1) / A8_THREADS;
  grid = dim3((unsigned)blocks);
  return blocks < (int64_t)0x7fffffff;
}

template <bool F32>
__global__ __launch_bounds__(A8_THREADS) void act8_pack_kernel(const void* __restrict__ x, int64_t ldx, ChunkMap M, int d,
                                                               uint8_t* __restrict__ q, int64_t ldq, uint8_t* __restrict__ scale,
                                                               int64_t lds) {
  for_chunk(M, [&](int64_t row, int c) {
    float v[8];
    row_load8<F32>((const char*)x + row * ldx * (F32 ? 4 : 2), c, d, row + 2 < M.rows, v);
    uint32_t byte;
    const u32x2 w = act8_encode(v, byte);
    *reinterpret_cast<u32x2*>(q + row * ldq + c) = w;
    if ((c & 31) == 0) scale[row * lds + (c >> 5)] = (uint8_t)byte;
  });
}

extern "C" int vita_act8_pack(const void* x, int32_t dtype, int64_t ldx, int64_t rows, int64_t d, void* q, int64_t ldq,
                              void* scale, int64_t lds, void* stream) {
  VITA_REQUIRE(rows > 0 && d > 0 && d <= ACT8_MAX_COLS);
  VITA_REQUIRE(act8_mat_ok(x, ldx, d, dtype));
  VITA_REQUIRE(act8_codes_ok(q, ldq, scale, lds, d));
  ChunkMap M; dim3 grid;
  VITA_REQUIRE(chunk_grid(rows, d, M, grid));
  if (dtype == VITA_DT_F32)
    hipLaunchKernelGGL(act8_pack_kernel<true>, grid, dim3(A8_THREADS), 0, (hipStream_t)stream, x, ldx, M, (int)d, (uint8_t*)q, ldq,
                       (uint8_t*)scale, lds);
  else
    hipLaunchKernelGGL(act8_pack_kernel<false>, grid, dim3(A8_THREADS), 0, (hipStream_t)stream, x, ldx, M, (int)d, (uint8_t*)q, ldq,
                       (uint8_t*)scale, lds);
  VITA_CHECK_LAUNCH("vita_act8_pack");
  return VITA_OK;
}

// y = value [* gamma + beta], columns [d, ldy) zero
__global__ __launch_bounds__(A8_THREADS) void act8_unpack_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                                                                 const uint8_t* __restrict__ scale, int64_t lds, ChunkMap M, int d,
                                                                 const float* __restrict__ gamma, const float* __restrict__ beta, int al,
                                                                 void* __restrict__ y, int64_t ldy, int y_f32) {
  for_chunk(M, [&](int64_t row, int c) {
    float v[8];
    codes_load8(q + row * ldq, scale + row * lds, c, d, v);
    if (c < d) {
      if (gamma) {
        float g[8], b[8];
        vec_load8(gamma, c, d, al, 0.f, g);
        vec_load8(beta, c, d, al, 0.f, b);
#pragma unroll
        for (int r = 0; r < 8; ++r) v[r] = __builtin_fmaf(v[r], g[r], b[r]);
      }
      if (c + 8 > d) {
#pragma unroll
        for (int r = 0; r < 8; ++r) if (c + r >= d) v[r] = 0.f;
      }
    }
    store8((char*)y + row * ldy * (y_f32 ? 4 : 2), c, ldy, y_f32, v);
  });
}

extern "C" int vita_act8_unpack(const void* q, int64_t ldq, const void* scale, int64_t lds, int64_t rows, int64_t d,
                                const float* gamma, const float* beta, void* y, int32_t y_dtype, int64_t ldy, void* stream) {
  VITA_REQUIRE(rows > 0 && d > 0 && d <= ACT8_MAX_COLS && ldy <= 2 * ACT8_MAX_COLS);
  VITA_REQUIRE(act8_codes_ok(q, ldq, scale, lds, d));
  VITA_REQUIRE(act8_mat_ok(y, ldy, d, y_dtype));
  VITA_REQUIRE(gamma || !beta);
  ChunkMap M; dim3 grid;
  VITA_REQUIRE(chunk_grid(rows, ldy, M, grid));
  hipLaunchKernelGGL(act8_unpack_kernel, grid, dim3(A8_THREADS), 0, (hipStream_t)stream, (const uint8_t*)q, ldq, (const uint8_t*)scale,
                     lds, M, (int)d, gamma, beta, (((uintptr_t)gamma | (uintptr_t)beta) & 15) == 0, y, ldy, y_dtype == VITA_DT_F32);
  VITA_CHECK_LAUNCH("vita_act8_unpack");
  return VITA_OK;
}

// g = gelu(z) from the full-precision z, and z itself in 8 bits: what the backward pass needs of the pair (gelu', gelu)
template <bool F32>
__global__ __launch_bounds__(A8_THREADS) void gelu_act8_fwd_kernel(const void* __restrict__ z, int64_t ldz, ChunkMap M, int d,
                                                                   uint16_t* __restrict__ g, int64_t ldg, uint8_t* __restrict__ q,
                                                                   int64_t ldq, uint8_t* __restrict__ scale, int64_t lds) {
  for_chunk(M, [&](int64_t row, int c) {
    float v[8];
    row_load8<F32>((const char*)z + row * ldz * (F32 ? 4 : 2), c, d, row + 2 < M.rows, v);
    uint32_t byte;
    const u32x2 w = act8_encode(v, byte);
    if (c < d + 31 - (d + 31) % 32) {      // d rounded up to whole groups
      *reinterpret_cast<u32x2*>(q + row * ldq + c) = w;
      if ((c & 31) == 0) scale[row * lds + (c >> 5)] = (uint8_t)byte;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) v[r] = gelu_erf(v[r]);       // gelu(0) = 0: the pads stay zero
    store8(g + row * ldg, c, ldg, false, v);
  });
}

extern "C" int vita_gelu_act8_fwd(const void* z, int32_t z_dtype, int64_t ldz, int64_t rows, int64_t d, void* g, int64_t ldg, void* q,
                                  int64_t ldq, void* scale, int64_t lds, void* stream) {
  VITA_REQUIRE(rows > 0 && d > 0 && d <= ACT8_MAX_COLS && ldg <= 2 * ACT8_MAX_COLS);
  VITA_REQUIRE(act8_mat_ok(z, ldz, d, z_dtype));
  VITA_REQUIRE(act8_mat_ok(g, ldg, d, VITA_DT_BF16));
  VITA_REQUIRE(act8_codes_ok(q, ldq, scale, lds, d));
  ChunkMap M; dim3 grid;
  VITA_REQUIRE(chunk_grid(rows, ldg > d ? ldg : d, M, grid));
  if (z_dtype == VITA_DT_F32)
    hipLaunchKernelGGL(gelu_act8_fwd_kernel<true>, grid, dim3(A8_THREADS), 0, (hipStream_t)stream, z, ldz, M, (int)d, (uint16_t*)g, ldg,
                       (uint8_t*)q, ldq, (uint8_t*)scale, lds);
  else
    hipLaunchKernelGGL(gelu_act8_fwd_kernel<false>, grid, dim3(A8_THREADS), 0, (hipStream_t)stream, z, ldz, M, (int)d, (uint16_t*)g,
                       ldg, (uint8_t*)q, ldq, (uint8_t*)scale, lds);
  VITA_CHECK_LAUNCH("vita_gelu_act8_fwd");
  return VITA_OK;
}

// dz = dg * gelu'(value), g = gelu(value) (optional: the operand of the next product's weight gradient)
__global__ __launch_bounds__(A8_THREADS) void gelu_act8_bwd_kernel(const uint16_t* dg, int64_t lddg, const uint8_t* __restrict__ q,
                                                                   int64_t ldq, const uint8_t* __restrict__ scale, int64_t lds,
                                                                   ChunkMap M, int d, uint16_t* dz, int64_t lddz,
                                                                   uint16_t* __restrict__ g, int64_t ldg) {
  for_chunk(M, [&](int64_t row, int c) {
    float v[8], t[8], p[8];
    raw_values8<false>(raw_load8<false>(dg + row * lddg, c, d, row + 2 < M.rows), t);
    codes_load8(q + row * ldq, scale + row * lds, c, d, v);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      float der;
      gelu_erf_both(v[r], p[r], der);
      t[r] *= der;
    }
    if (c + 8 > d) {                        // codes and dg behind d are whatever the caller's buffers hold
#pragma unroll
      for (int r = 0; r < 8; ++r) if (c + r >= d) t[r] = p[r] = 0.f;
    }
    store8(dz + row * lddz, c, lddz, false, t);
    if (g) store8(g + row * ldg, c, ldg, false, p);
  });
}

extern "C" int vita_gelu_act8_bwd(const void* dg, int64_t lddg, const void* q, int64_t ldq, const void* scale, int64_t lds,
                                  int64_t rows, int64_t d, void* dz, int64_t lddz, void* g, int64_t ldg, void* stream) {
  VITA_REQUIRE(rows > 0 && d > 0 && d <= ACT8_MAX_COLS && lddz <= 2 * ACT8_MAX_COLS && ldg <= 2 * ACT8_MAX_COLS);
  VITA_REQUIRE(act8_mat_ok(dg, lddg, d, VITA_DT_BF16));
  VITA_REQUIRE(act8_codes_ok(q, ldq, scale, lds, d));
  VITA_REQUIRE(act8_mat_ok(dz, lddz, d, VITA_DT_BF16));
  if (g) VITA_REQUIRE(act8_mat_ok(g, ldg, d, VITA_DT_BF16));
  ChunkMap M; dim3 grid;
  VITA_REQUIRE(chunk_grid(rows, g && ldg > lddz ? ldg : lddz, M, grid));
  hipLaunchKernelGGL(gelu_act8_bwd_kernel, grid, dim3(A8_THREADS), 0, (hipStream_t)stream, (const uint16_t*)dg, lddg, (const uint8_t*)q,
                     ldq, (const uint8_t*)scale, lds, M, (int)d, (uint16_t*)dz, lddz, (uint16_t*)g, ldg);
  VITA_CHECK_LAUNCH("vita_gelu_act8_bwd");
  return VITA_OK;
}
