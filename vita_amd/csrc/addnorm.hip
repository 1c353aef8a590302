// Residual addition + norm (root mean square, or LayerNorm) in one pass, with an optional 8-bit output, and its backward pass
// from the 8-bit rows or from the kept sum.
//
//   s = x + r                                  (fp32; written rounded to its type when asked for)
//   mu = 0 (rms) | mean(s) (layer);  rstd = 1 / sqrt(mean((s - mu)^2) + eps)       two passes over registers, fp32
//   n = (s - mu) rstd;  y = n gamma [+ beta]   y in bf16 / fp32, and n or y in 8 bits (act8.h)
// backward, with h = dy gamma:
//   dx = dx_in + rstd (h - [mean(h)] - n mean(h n)),  dgamma = sum_rows dy n,  dbeta = sum_rows dy
// n comes from the 8-bit rows (1.03 bytes a value and rstd) or from s and (mu, rstd).
#include "act8.h"

#define AN_RMS 0
#define AN_LAYER 1
#define AN_MAX_D 8192

// sum over the W waves that share a row (W = 1: the wave itself, no barrier)
template <int W>
__device__ __forceinline__ float row_sum(float v, float* red, int wave, int lane) {
  v = wave_sum(v);
  if (W == 1) return v;
  __syncthreads();                    // the previous use of red is over
  if (lane == 0) red[wave] = v;
  __syncthreads();
  float t = red[0];
#pragma unroll
  for (int w = 1; w < W; ++w) t += red[w];
  return t;
}

template <int W, int NV, bool XF, int RT>      // RT: 0 no residual, 1 bf16, 2 fp32
__global__ __launch_bounds__(256) void addnorm_fwd_kernel(const vita_addnorm_fwd_desc D) {
  __shared__ float red[W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x;
  if (row >= D.rows) return;          // whole rows leave together: W waves of one row share the block
  const int d = (int)D.d, t0 = (W == 1 ? lane : (int)threadIdx.x) * 8;
  Raw8 xr[NV], rr[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) xr[i] = raw_load8<XF>((const char*)D.x + row * D.ldx * (XF ? 4 : 2), t0 + i * W * 512, d);
  if (RT) {
#pragma unroll
    for (int i = 0; i < NV; ++i) rr[i] = raw_load8<RT == 2>((const char*)D.res + row * D.ldr * (RT == 2 ? 4 : 2), t0 + i * W * 512, d);
  }
  float v[NV][8], s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    raw_values8<XF>(xr[i], v[i]);
    if (RT) {
      float t[8];
      raw_values8<RT == 2>(rr[i], t);
#pragma unroll
      for (int r = 0; r < 8; ++r) v[i][r] += t[r];
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) s += v[i][r];
  }
  if (RT && D.sum) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      store8((char*)D.sum + row * D.ldsum * (D.sum_dtype == VITA_DT_F32 ? 4 : 2), t0 + i * W * 512, D.ldsum, D.sum_dtype == VITA_DT_F32, v[i]);
  }
  const float inv_d = 1.f / (float)d;
  const float mu = D.kind == AN_LAYER ? row_sum<W>(s, red, wave, lane) * inv_d : 0.f;
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const bool on = t0 + i * W * 512 + r < d;
      v[i][r] = on ? v[i][r] - mu : 0.f;
      q = __builtin_fmaf(v[i][r], v[i][r], q);
    }
  const float rs = rsqrtf(row_sum<W>(q, red, wave, lane) * inv_d + D.eps);
  if (t0 == 0) {
    if (D.mean) D.mean[row] = mu;
    if (D.rstd) D.rstd[row] = rs;
  }
  const int dq = (d + 31) & ~31;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = t0 + i * W * 512;
    float y[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      v[i][r] *= rs;
      y[r] = c + r < d ? __builtin_fmaf(v[i][r], D.gamma ? D.gamma[c + r] : 1.f, D.beta ? D.beta[c + r] : 0.f) : 0.f;
    }
    if (D.q) {
      uint32_t byte;
      const u32x2 w = D.pack == VITA_PACK_OUTPUT ? act8_encode(y, byte) : act8_encode(v[i], byte);
      if (c < dq) {
        *reinterpret_cast<u32x2*>((uint8_t*)D.q + row * D.ldq + c) = w;
        if ((c & 31) == 0) ((uint8_t*)D.scale)[row * D.lds + (c >> 5)] = (uint8_t)byte;
      }
    }
    if (D.y) store8((char*)D.y + row * D.ldy * (D.y_dtype == VITA_DT_F32 ? 4 : 2), c, D.ldy, D.y_dtype == VITA_DT_F32, y);
  }
}

extern "C" int vita_addnorm_fwd(const vita_addnorm_fwd_desc* dp, void* stream) {
  if (!dp) return VITA_ERR_INVALID_ARG;
  vita_addnorm_fwd_desc D = *dp;
  VITA_REQUIRE(D.rows > 0 && D.d > 0);
  VITA_REQUIRE(D.kind == AN_RMS || D.kind == AN_LAYER);
  VITA_REQUIRE(act8_mat_ok(D.x, D.ldx, D.d, D.x_dtype));
  if (D.res) VITA_REQUIRE(act8_mat_ok(D.res, D.ldr, D.d, D.res_dtype));
  if (D.sum) VITA_REQUIRE(D.res && act8_mat_ok(D.sum, D.ldsum, D.d, D.sum_dtype));
  VITA_REQUIRE(D.y || D.q);
  VITA_REQUIRE(D.gamma || !D.beta);
  if (D.y) VITA_REQUIRE(act8_mat_ok(D.y, D.ldy, D.d, D.y_dtype));
  if (D.q) {
    VITA_REQUIRE(D.pack == VITA_PACK_NORMED || D.pack == VITA_PACK_OUTPUT);
    VITA_REQUIRE(act8_codes_ok(D.q, D.ldq, D.scale, D.lds, D.d));
  }
  int64_t width = (D.d + 31) & ~(int64_t)31;
  if (D.y && D.ldy > width) width = D.ldy;
  if (D.sum && D.ldsum > width) width = D.ldsum;
  if (width > AN_MAX_D) {
    vita_set_error("vita_addnorm_fwd: rows of more than 8192 columns (with their pads)", hipSuccess);
    return VITA_ERR_UNSUPPORTED;
  }
  VITA_REQUIRE(D.rows < (int64_t)0x7fffffff);
  const int rt = D.res ? (D.res_dtype == VITA_DT_F32 ? 2 : 1) : 0;
#define AN_LAUNCH(W, NV, XF, RT)                                                                                                     \
  hipLaunchKernelGGL((addnorm_fwd_kernel<W, NV, XF, RT>), dim3((unsigned)(W == 1 ? (D.rows + 3) / 4 : D.rows)), dim3(256), 0,        \
                     (hipStream_t)stream, D)
#define AN_TYPES(W, NV)                                                                 \
  do {                                                                                  \
    if (D.x_dtype == VITA_DT_F32) {                                                     \
      if (rt == 0) AN_LAUNCH(W, NV, true, 0); else if (rt == 1) AN_LAUNCH(W, NV, true, 1); else AN_LAUNCH(W, NV, true, 2);    \
    } else {                                                                            \
      if (rt == 0) AN_LAUNCH(W, NV, false, 0); else if (rt == 1) AN_LAUNCH(W, NV, false, 1); else AN_LAUNCH(W, NV, false, 2); \
    }                                                                                   \
  } while (0)
  if (width <= 512) AN_TYPES(1, 1);
  else if (width <= 1536) AN_TYPES(1, 3);
  else if (width <= 4096) AN_TYPES(4, 2);
  else AN_TYPES(4, 4);
#undef AN_TYPES
#undef AN_LAUNCH
  VITA_CHECK_LAUNCH("vita_addnorm_fwd");
  return VITA_OK;
}

// ---- backward: a block walks over rows; a lane's dgamma / dbeta sums stay in registers, then one partial row per block
#define AN_BWD_MAXBLK 768
template <int W, int NV, int SRC, bool DYF>      // SRC: 0 8-bit rows, 1 bf16 sum, 2 fp32 sum
__global__ __launch_bounds__(256) void addnorm_bwd_kernel(const vita_addnorm_bwd_desc D, const int nblk) {
  __shared__ float red[W == 1 ? 1 : 8];
  __shared__ float sums[W == 1 ? NV * 512 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int d = (int)D.d, t0 = (W == 1 ? lane : (int)threadIdx.x) * 8;
  const float inv_d = 1.f / (float)d;
  float ag[NV][8], ab[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int r = 0; r < 8; ++r) ag[i][r] = ab[i][r] = 0.f;
  const int64_t step = W == 1 ? (int64_t)nblk * 4 : nblk;
  for (int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + wave : (int64_t)blockIdx.x; row < D.rows; row += step) {
    Raw8 dyr[NV], sr[NV];
    uint32_t byte[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t0 + i * W * 512;
      dyr[i] = raw_load8<DYF>((const char*)D.dy + row * D.lddy * (DYF ? 4 : 2), c, d);
      if (SRC == 0) {
        sr[i].a = u32x4{0, 0, 0, 0};
        byte[i] = 0;
        if (c < d) {
          const u32x2 w = *reinterpret_cast<const u32x2*>((const uint8_t*)D.q + row * D.ldq + c);
          sr[i].a[0] = w[0]; sr[i].a[1] = w[1];
          byte[i] = ((const uint8_t*)D.scale)[row * D.lds + (c >> 5)];
        }
      } else {
        sr[i] = raw_load8<SRC == 2>((const char*)D.src + row * D.ldx * (SRC == 2 ? 4 : 2), c, d);
      }
    }
    const float rs = D.rstd[row], mu = SRC != 0 && D.mean ? D.mean[row] : 0.f;
    float n[NV][8], h[NV][8], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t0 + i * W * 512;
      float dy[8];
      raw_values8<DYF>(dyr[i], dy);
      if (SRC == 0) act8_decode(u32x2{sr[i].a[0], sr[i].a[1]}, byte[i], n[i]);
      else raw_values8<SRC == 2>(sr[i], n[i]);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (SRC != 0) n[i][r] = (n[i][r] - mu) * rs;
        if (c + r >= d) n[i][r] = 0.f;               // dy is zero there already
        h[i][r] = c + r < d ? dy[r] * (D.gamma ? D.gamma[c + r] : 1.f) : 0.f;
        ag[i][r] = __builtin_fmaf(dy[r], n[i][r], ag[i][r]);
        ab[i][r] += dy[r];
        s1 += h[i][r];
        s2 = __builtin_fmaf(h[i][r], n[i][r], s2);
      }
    }
    const float c1 = D.kind == AN_LAYER ? row_sum<W>(s1, red, wave, lane) * inv_d : 0.f;
    const float c2 = row_sum<W>(s2, red, wave, lane) * inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t0 + i * W * 512;
      float o[8];
      if (D.dx_in) {
        if (D.dx_dtype == VITA_DT_F32) raw_values8<true>(raw_load8<true>((const float*)D.dx_in + row * D.lddx_in, c, d), o);
        else raw_values8<false>(raw_load8<false>((const uint16_t*)D.dx_in + row * D.lddx_in, c, d), o);
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float t = (h[i][r] - c1 - n[i][r] * c2) * rs;
        o[r] = c + r < d ? (D.dx_in ? t + o[r] : t) : 0.f;
      }
      store8((char*)D.dx + row * D.lddx * (D.dx_dtype == VITA_DT_F32 ? 4 : 2), c, D.lddx, D.dx_dtype == VITA_DT_F32, o);
      if (D.dx_bf16) store8((uint16_t*)D.dx_bf16 + row * D.lddxb, c, D.lddxb, false, o);
    }
  }
  if (!D.partial) return;
  float* pg = D.partial + (int64_t)blockIdx.x * d;
  float* pb = D.partial + ((int64_t)nblk + blockIdx.x) * d;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k == 1 && !D.dbeta) break;
    if (W == 1) {                       // the block's four waves one after another, through LDS
      for (int w = 0; w < 4; ++w) {
        __syncthreads();
        if (wave == w) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              const float a = k ? ab[i][r] : ag[i][r];
              float* p = &sums[t0 + i * 512 + r];
              *p = w ? *p + a : a;
            }
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < d; c += 256) (k ? pb : pg)[c] = sums[c];
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int c = t0 + i * W * 512 + r;
          if (c < d) (k ? pb : pg)[c] = k ? ab[i][r] : ag[i][r];
        }
    }
  }
}

// column sums of the partial rows: grid (ceil(d / 64), 1 or 2), 16 waves over interleaved rows, fixed order
__global__ __launch_bounds__(1024) void addnorm_reduce_kernel(const float* __restrict__ partial, int nblk, int d, float* dgamma,
                                                              float* dbeta, int acc) {
  __shared__ float red[16][64];
  const int cx = threadIdx.x & 63, ry = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + cx;
  const float* p = partial + (int64_t)blockIdx.y * nblk * d + c;
  float a = 0.f;
  if (c < d)
    for (int k = ry; k < nblk; k += 16) a += p[(int64_t)k * d];
  red[ry][cx] = a;
  __syncthreads();
  float* o = blockIdx.y ? dbeta : dgamma;
  if (ry == 0 && c < d && o) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += red[w][cx];
    o[c] = acc ? o[c] + t : t;
  }
}

extern "C" int64_t vita_addnorm_bwd_nblk(int64_t rows, int64_t d) {
  const int64_t n = d <= 1536 ? (rows + 15) / 16 : (rows + 3) / 4;
  return n < AN_BWD_MAXBLK ? n : AN_BWD_MAXBLK;
}

extern "C" int vita_addnorm_bwd(const vita_addnorm_bwd_desc* dp, void* stream) {
  if (!dp) return VITA_ERR_INVALID_ARG;
  vita_addnorm_bwd_desc D = *dp;
  VITA_REQUIRE(D.rows > 0 && D.d > 0);
  VITA_REQUIRE(D.kind == AN_RMS || D.kind == AN_LAYER);
  VITA_REQUIRE(act8_mat_ok(D.dy, D.lddy, D.d, D.dy_dtype) && D.rstd);
  VITA_REQUIRE((D.src != nullptr) != (D.q != nullptr));
  if (D.q) VITA_REQUIRE(act8_codes_ok(D.q, D.ldq, D.scale, D.lds, D.d));
  else VITA_REQUIRE(act8_mat_ok(D.src, D.ldx, D.d, D.src_dtype) && (D.mean || D.kind == AN_RMS));
  VITA_REQUIRE(act8_mat_ok(D.dx, D.lddx, D.d, D.dx_dtype));
  if (D.dx_in) VITA_REQUIRE(act8_mat_ok(D.dx_in, D.lddx_in, D.d, D.dx_dtype));
  if (D.dx_bf16) VITA_REQUIRE(act8_mat_ok(D.dx_bf16, D.lddxb, D.d, VITA_DT_BF16));
  VITA_REQUIRE((D.partial != nullptr) == (D.dgamma || D.dbeta));
  if (D.kind == AN_RMS) VITA_REQUIRE(!D.dbeta);
  int64_t width = (D.d + 7) & ~(int64_t)7;
  if (D.lddx > width) width = D.lddx;
  if (D.dx_bf16 && D.lddxb > width) width = D.lddxb;
  if (width > AN_MAX_D) {
    vita_set_error("vita_addnorm_bwd: rows of more than 8192 columns (with their pads)", hipSuccess);
    return VITA_ERR_UNSUPPORTED;
  }
  const int nblk = (int)vita_addnorm_bwd_nblk(D.rows, D.d);
  const int src = D.q ? 0 : (D.src_dtype == VITA_DT_F32 ? 2 : 1);
#define AN_LAUNCH(W, NV, SRC, DYF) \
  hipLaunchKernelGGL((addnorm_bwd_kernel<W, NV, SRC, DYF>), dim3(nblk), dim3(256), 0, (hipStream_t)stream, D, nblk)
#define AN_TYPES(W, NV)                                                                                                       \
  do {                                                                                                                        \
    if (D.dy_dtype == VITA_DT_F32) {                                                                                          \
      if (src == 0) AN_LAUNCH(W, NV, 0, true); else if (src == 1) AN_LAUNCH(W, NV, 1, true); else AN_LAUNCH(W, NV, 2, true);  \
    } else {                                                                                                                  \
      if (src == 0) AN_LAUNCH(W, NV, 0, false); else if (src == 1) AN_LAUNCH(W, NV, 1, false); else AN_LAUNCH(W, NV, 2, false); \
    }                                                                                                                         \
  } while (0)
  if (width <= 512) AN_TYPES(1, 1);
  else if (width <= 1536) AN_TYPES(1, 3);
  else if (width <= 4096) AN_TYPES(4, 2);
  else AN_TYPES(4, 4);
#undef AN_TYPES
#undef AN_LAUNCH
  VITA_CHECK_LAUNCH("vita_addnorm_bwd");
  if (D.partial) {
    hipLaunchKernelGGL(addnorm_reduce_kernel, dim3((unsigned)((D.d + 63) / 64), D.dbeta ? 2 : 1), dim3(1024), 0, (hipStream_t)stream,
                       D.partial, nblk, (int)D.d, D.dgamma, D.dbeta, D.accumulate);
    VITA_CHECK_LAUNCH("vita_addnorm_bwd_reduce");
  }
  return VITA_OK;
}
