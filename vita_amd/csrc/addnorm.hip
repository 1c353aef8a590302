// Residual addition + norm (root mean square, or LayerNorm) in one pass, with an optional 8-bit output, and its backward pass
// from the 8-bit rows or from the kept sum.
//
//   s = x + r                                  (fp32; written rounded to its type when asked for)
//   mu = 0 (rms) | mean(s) (layer);  rstd = 1 / sqrt(mean((s - mu)^2) + eps)       two passes over registers, summed in 64 bits
//   n = (s - mu) rstd;  y = n gamma [+ beta]   y in bf16 / fp32, and n or y in 8 bits (act8.h)
// backward, with h = dy gamma:
//   dx = dx_in + rstd (h - [mean(h)] - n mean(h n)),  dgamma = sum_rows dy n,  dbeta = sum_rows dy
// n comes from the 8-bit rows (1.03 bytes a value and rstd) or from s and (mu, rstd).
//
// Both move bytes.  Measured (MI355X, kernels alone; a copy of that size reaches 5 TB/s):
//   forward, 46082 x 1025, bf16 + fp32 -> fp32 sum, bf16 y, 8-bit n: 130 us, 4.8 TB/s (one wave per row and a row per block of gamma
//     and beta loads: 186 us; rows dealt to resident waves with gamma in registers: 141 us; 64 columns behind the chunks one to a
//     lane: 134 us; all of it in 64 bits instead of the sums and the values next to a border: 134 us, with a LayerNorm's 8-bit output of bf16 +
//     bf16 107 instead of 95)
//   backward, 13826 x 1025, from 8 bits, bf16 dy, fp32 dx_in and dx: 37 + 4 us (sums of the partial rows), 4.5 TB/s (gamma read
//     anew for each row and dx_in after the sums: 89 + 16 us; loads together, gamma in registers: 61; 768 partial rows of 1025
//     columns added with all loads in flight: 4 instead of 16 us; last columns one to a lane, 3 blocks a CU instead of 2: 37; with
//     fp32 dy the compiler has to be held to the registers of 3 blocks: 46082 rows 118 -> 88 us)
//   backward, 4096 x 4096, from a bf16 sum: 30 + 4 us (four waves with two chunks a lane instead of eight with one: 33)
//   rows whose last chunk is not whole, loaded in one piece instead of by columns: 46082 x 777 backward 80 -> 63 us, 29000 x 1601
//     forward 162 -> 133, backward 132 -> 93
#include "act8.h"

#define AN_RMS 0
#define AN_LAYER 1
#define AN_MAX_D 8192
#define AN_FWD_MAXBLK 2048
#define AN_FEW_ROWS 1024
// how a wave holds a row: its 64 lanes; those and one column a lane more; or (16, 32) that many lanes of it
#define AN_FULL 0
#define AN_TAIL 1

// A wave's sums of doubles in all of its lanes (or its L neighbouring ones) without LDS: quads, halves and whole rows of 16 lanes by DPP
// (mirrored: the lanes that differ in lower bits hold the same sum by then), rows and halves of the wave by swaps
template <int CTRL>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b, CTRL, 0xf, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, true);
  return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int O>
__device__ __forceinline__ double swap_add(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)b, hi = (uint32_t)(b >> 32);
  const auto p = O == 16 ? __builtin_amdgcn_permlane16_swap(lo, lo, false, false) : __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
  const auto q = O == 16 ? __builtin_amdgcn_permlane16_swap(hi, hi, false, false) : __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
  return __builtin_bit_cast(double, (uint64_t)q[0] << 32 | p[0]) + __builtin_bit_cast(double, (uint64_t)q[1] << 32 | p[1]);
}
template <int L>
__device__ __forceinline__ double lane_sum(double v) {
  v = dpp_add<0xB1>(v);                 // quad_perm [1,0,3,2]
  v = dpp_add<0x4E>(v);                 // quad_perm [2,3,0,1]
  v = dpp_add<0x141>(v);                // row_half_mirror
  v = dpp_add<0x140>(v);                // row_mirror
  if (L > 16) v = swap_add<16>(v);
  if (L > 32) v = swap_add<32>(v);
  return v;
}
template <int L>
__device__ __forceinline__ void lane_sum2(double& a, double& b) { a = lane_sum<L>(a); b = lane_sum<L>(b); }
template <int L>
__device__ __forceinline__ void lane_sum2(float& a, float& b) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) { a += __shfl_xor(a, o, 64); b += __shfl_xor(b, o, 64); }
}
// sums over the W waves that share a row (W = 1: the wave itself, or its L neighbouring lanes, no barrier), two at a time
template <int W, int L, typename F>
__device__ __forceinline__ void row_sum2(F& a, F& b, F (*red)[2][W], int& turn, int wave, int lane) {
  lane_sum2<L>(a, b);
  if (W == 1) return;
  turn ^= 1;                          // two slots in turn: the barrier of the next sum lies between a slot's reads and its next writes
  if (lane == 0) { red[turn][0][wave] = a; red[turn][1][wave] = b; }
  __syncthreads();
  a = red[turn][0][0]; b = red[turn][1][0];
#pragma unroll
  for (int w = 1; w < W; ++w) { a += red[turn][0][w]; b += red[turn][1][w]; }
}
template <int W, int L>
__device__ __forceinline__ double row_sum(double a, double (*red)[2][W], int& turn, int wave, int lane) {
  a = lane_sum<L>(a);
  if (W == 1) return a;
  turn ^= 1;
  if (lane == 0) red[turn][0][wave] = a;
  __syncthreads();
  a = red[turn][0][0];
#pragma unroll
  for (int w = 1; w < W; ++w) a += red[turn][0][w];
  return a;
}

// A double as the float next to it towards zero, its last bit set where that is not exact: on the same side of every number of fewer
// bits (the borders between 8-bit codes, the maxima at which a scale changes) as the double itself
__device__ __forceinline__ float odd_float(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t rest = (uint32_t)b & 0x1fffffffu;
  const float f = (float)__builtin_bit_cast(double, b & ~(uint64_t)0x1fffffffu);
  return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, f) | (rest ? 1u : 0u));
}

// A wave (W = 1) or the four waves of a block (W = 4) walk over rows, 8 neighbouring columns to a lane and chunk, the row in
// registers from its loads to its stores; gamma and beta stay in registers.  T: up to 64 columns behind the last whole chunk go one to
// a lane instead of opening another chunk (1025 columns would fill 1 of its 64 lanes and cost every lane 8 columns of registers and
// arithmetic).  M = 16, 32: narrow rows, 4 or 2 of them to a wave.
template <int W, int NV, int M, bool XF, int RT, bool LAYER>      // RT: 0 no residual, 1 bf16, 2 fp32
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W, NV == 2 ? 4 : 1) void addnorm_fwd_kernel(const vita_addnorm_fwd_desc D, const int al) {
  constexpr bool T = M == AN_TAIL;
  constexpr int L = M > AN_TAIL ? M : 64, R = W == 1 ? 256 / L : 1;      // lanes of a wave to a row; rows of a block at a time
  __shared__ double red[2][2][W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int d = (int)D.d, t0 = (W == 1 ? lane % L : (int)threadIdx.x) * 8;
  const double inv_d = 1.0 / (double)d;
  int turn = 0;
  float gm[NV][8], bt[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    vec_load8(D.gamma, t0 + i * W * 512, d, al, 1.f, gm[i]);
    vec_load8(D.beta, t0 + i * W * 512, d, al, 0.f, bt[i]);
  }
  const int ct = NV * 512 + lane;                // the lane's column behind the chunks
  const float gt = T && ct < d && D.gamma ? D.gamma[ct] : 1.f, btt = T && ct < d && D.beta ? D.beta[ct] : 0.f;
  const int64_t step = (int64_t)gridDim.x * R;
  for (int64_t row = (int64_t)blockIdx.x * R + (L < 64 ? (int)threadIdx.x / L : W == 1 ? wave : 0); row < D.rows; row += step) {
    Raw8 xr[NV], rr[NV];
    const bool whole = row + 2 < D.rows;       // the last chunk of a row as one load, its pads cleared afterwards
#pragma unroll
    for (int i = 0; i < NV; ++i) xr[i] = raw_load8<XF>((const char*)D.x + row * D.ldx * (XF ? 4 : 2), t0 + i * W * 512, d, whole);
    if (RT) {
#pragma unroll
      for (int i = 0; i < NV; ++i) rr[i] = raw_load8<RT == 2>((const char*)D.res + row * D.ldr * (RT == 2 ? 4 : 2), t0 + i * W * 512, d, whole);
    }
    float vt = 0.f;
    if (T) {
      vt = load1<XF>((const char*)D.x + row * D.ldx * (XF ? 4 : 2), ct, d);
      if (RT) vt += load1<RT == 2>((const char*)D.res + row * D.ldr * (RT == 2 ? 4 : 2), ct, d);
    }
    float v[NV][8];
    const auto clear = [&](int i, float (&a)[8]) {       // behind the row's end
      const int c = t0 + i * W * 512;
      if (c + 8 > d) {
#pragma unroll
        for (int r = 0; r < 8; ++r) if (c + r >= d) a[r] = 0.f;
      }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      raw_values8<XF>(xr[i], v[i]);
      if (RT) {
        float t[8];
        raw_values8<RT == 2>(rr[i], t);
#pragma unroll
        for (int r = 0; r < 8; ++r) v[i][r] += t[r];
      }
      clear(i, v[i]);
    }
    if (RT && D.sum) {
      const bool f = D.sum_dtype == VITA_DT_F32;
#pragma unroll
      for (int i = 0; i < NV; ++i) store8((char*)D.sum + row * D.ldsum * (f ? 4 : 2), t0 + i * W * 512, D.ldsum, f, v[i]);
      if (T) store1((char*)D.sum + row * D.ldsum * (f ? 4 : 2), ct, D.ldsum, f, vt);
    }
    const auto forget = [&]() {         // the 64-bit form of v, or it would be held from one use to the next: 16 NV registers
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int r = 0; r < 8; ++r) asm volatile("" : "+v"(v[i][r]));
    };
    double mu = 0.0;
    if (LAYER) {
      double s = (double)vt;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int r = 0; r < 8; ++r) s += (double)v[i][r];
      mu = row_sum<W, L>(s, red, turn, wave, lane) * inv_d;
      if (D.mean && t0 == 0) D.mean[row] = (float)mu;
      forget();
    }
    double q = T && ct < d ? ((double)vt - mu) * ((double)vt - mu) : 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t0 + i * W * 512;
      double a[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) a[r] = LAYER ? (double)v[i][r] - mu : (double)v[i][r];
      if (LAYER && c + 8 > d) {
#pragma unroll
        for (int r = 0; r < 8; ++r) if (c + r >= d) a[r] = 0.0;
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) q = __builtin_fma(a[r], a[r], q);
    }
    forget();
    const double rs = 1.0 / sqrt(row_sum<W, L>(q, red, turn, wave, lane) * inv_d + (double)D.eps);
    // mu and rstd as pairs of floats: s - mu and n are each rounded as if from 64 bits, up to 3 steps of 2^-24 in all
    const float rh = (float)rs, rl = (float)(rs - (double)rh), mh = (float)mu, ml = (float)(mu - (double)mh);
    if (D.rstd && t0 == 0) D.rstd[row] = rh;
    // A rounding that carries a value across a border between two codes changes the code by a whole step of 2^-3: where one comes within
    // `near` steps of 2^-23 of a border, its chunk is computed once more in 64 bits (a wave in 120 normed ones, in 30 of outputs, whose
    // beta may cancel some bits)
    const bool out = D.pack == VITA_PACK_OUTPUT;
    const uint32_t near = out ? 32 : 8;
    const int dq = (d + 31) & ~31;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t0 + i * W * 512;
      float n[8], y[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float a = LAYER ? (v[i][r] - mh) - ml : v[i][r];
        n[r] = __builtin_fmaf(a, rh, a * rl);
        y[r] = __builtin_fmaf(n[r], gm[i][r], bt[i][r]);
      }
      clear(i, n);                             // also in a row whose rstd is NaN
      clear(i, y);
      if (D.y) store8((char*)D.y + row * D.ldy * (D.y_dtype == VITA_DT_F32 ? 4 : 2), c, D.ldy, D.y_dtype == VITA_DT_F32, y);
      if (D.q) {
        uint32_t byte, m, off = 0xffffffffu;
        float t[8];
        if (out) act8_scaled(y, t, byte, m); else act8_scaled(n, t, byte, m);
#pragma unroll
        for (int r = 0; r < 8; ++r) { const uint32_t o = act8_off_border(t[r], near); off = off < o ? off : o; }
        u32x2 w = act8_codes(t);
        if (__builtin_expect(__any(off <= 2 * near || act8_near_scale(m, near)), 0)) {
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            float a = v[i][r], b = gm[i][r], e = bt[i][r];
            asm volatile("" : "+v"(a), "+v"(b), "+v"(e));      // or their 64-bit forms would be held in registers from the row's start
            const double u = ((double)a - mu) * rs;
            t[r] = odd_float(out ? __builtin_fma(u, (double)b, (double)e) : u);
          }
          clear(i, t);
          w = act8_encode(t, byte);
        }
        if (c < dq) {
          *reinterpret_cast<u32x2*>((uint8_t*)D.q + row * D.ldq + c) = w;
          if ((c & 31) == 0) ((uint8_t*)D.scale)[row * D.lds + (c >> 5)] = (uint8_t)byte;
        }
      }
    }
    if (T) {                                   // one value: in 64 bits at once
      const double n = ((double)vt - mu) * rs;
      if (D.q) {
        uint32_t byte;
        const uint8_t w = act8_encode1(ct < d ? odd_float(out ? __builtin_fma(n, (double)gt, (double)btt) : n) : 0.f, byte);
        if (ct < dq) {
          ((uint8_t*)D.q)[row * D.ldq + ct] = w;
          if ((ct & 31) == 0) ((uint8_t*)D.scale)[row * D.lds + (ct >> 5)] = (uint8_t)byte;
        }
      }
      if (D.y) store1((char*)D.y + row * D.ldy * (D.y_dtype == VITA_DT_F32 ? 4 : 2), ct, D.ldy, D.y_dtype == VITA_DT_F32, ct < d ? __builtin_fmaf((float)n, gt, btt) : 0.f);
    }
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
  const int al = (((uintptr_t)D.gamma | (uintptr_t)D.beta) & 15) == 0;
  const auto blocks = [&](int w, int m) {
    const int64_t at_once = w > 1 ? 1 : m > AN_TAIL ? 256 / m : 4, n = (D.rows + at_once - 1) / at_once;
    return n < AN_FWD_MAXBLK ? n : AN_FWD_MAXBLK;
  };
#define AN_LAUNCH(W, NV, M, XF, RT)                                                                                                          \
  do {                                                                                                                                       \
    const dim3 g((unsigned)blocks(W, M)), b(W == 1 ? 256 : 64 * W);                                                                          \
    if (D.kind == AN_LAYER) hipLaunchKernelGGL((addnorm_fwd_kernel<W, NV, M, XF, RT, true>), g, b, 0, (hipStream_t)stream, D, al);           \
    else hipLaunchKernelGGL((addnorm_fwd_kernel<W, NV, M, XF, RT, false>), g, b, 0, (hipStream_t)stream, D, al);                             \
  } while (0)
#define AN_TYPES(W, NV, M)                                                                                                                   \
  do {                                                                                                                                       \
    if (D.x_dtype == VITA_DT_F32) {                                                                                                          \
      if (rt == 0) AN_LAUNCH(W, NV, M, true, 0); else if (rt == 1) AN_LAUNCH(W, NV, M, true, 1); else AN_LAUNCH(W, NV, M, true, 2);         \
    } else {                                                                                                                                 \
      if (rt == 0) AN_LAUNCH(W, NV, M, false, 0); else if (rt == 1) AN_LAUNCH(W, NV, M, false, 1); else AN_LAUNCH(W, NV, M, false, 2);      \
    }                                                                                                                                        \
  } while (0)
  // Few rows: four waves to a row shorten the way through one row, many rows: a wave to each saves the barriers.  One wave / four, us,
  // bf16 + fp32 residual, 600 columns: 1 row 3.7 / 3.0, 512 rows 5.3 / 4.8, 1024 5.8 / 6.0, 2048 7.0 / 8.7; 1025 columns: 3.8 / 3.2,
  // 5.6 / 5.2, 6.2 / 6.3, 8.3 / 9.7.  Above 1536 columns a wave would hold 4 chunks and more (64 registers of values): four waves, with
  // one chunk a lane as far as that goes (2000 columns, 8192 rows: 34.0 us, with two chunks, half of them empty, 36.6).  Above 4096 columns
  // eight waves with two chunks a lane, in whose registers four of them fit a SIMD (four waves with four chunks, two of which fit: 9000 x
  // 5000, fp32, 153 against 140 us; 6000 x 4106 91 against 84; 16 x 4600 the same).  Narrow rows share a wave: 46082 rows
  // of 69 columns, 16 lanes each 11.2 us, 64 lanes 24.4; of 130 columns, 32 lanes 15.9 us, 64 lanes 24.6.
  if (width <= 128) AN_TYPES(1, 1, 16);
  else if (width <= 256) AN_TYPES(1, 1, 32);
  else if (width <= 512) AN_TYPES(1, 1, AN_FULL);
  else if (width <= 2048 && (D.rows <= AN_FEW_ROWS || width > 1536)) AN_TYPES(4, 1, AN_FULL);
  else if (width <= 1024) AN_TYPES(1, 2, AN_FULL);
  else if (width <= 1088) AN_TYPES(1, 2, AN_TAIL);
  else if (width <= 1536) AN_TYPES(1, 3, AN_FULL);
  else if (width <= 4096) AN_TYPES(4, 2, AN_FULL);
  else AN_TYPES(8, 2, AN_FULL);
#undef AN_TYPES
#undef AN_LAUNCH
  VITA_CHECK_LAUNCH("vita_addnorm_fwd");
  return VITA_OK;
}

// ---- backward: rows as above; every load of a row is in flight before its first sum, the values are taken from the raw registers
// twice (to sum, to store) instead of being kept, and a lane's dgamma / dbeta sums stay in registers until one partial row per block
#define AN_BWD_MAXBLK 768
template <int W, int NV, int M, int SRC, bool DYF>      // SRC: 0 8-bit rows, 1 bf16 sum, 2 fp32 sum
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W, M == AN_TAIL ? 3 : 1) void addnorm_bwd_kernel(const vita_addnorm_bwd_desc D, const int al) {
  constexpr bool T = M == AN_TAIL;
  constexpr int L = M > AN_TAIL ? M : 64, R = W == 1 ? 256 / L : 1;      // as in the forward kernel
  __shared__ float red[2][2][W];
  __shared__ __attribute__((aligned(16))) float sums[W == 1 ? NV * 512 + 64 : 4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int d = (int)D.d, t0 = (W == 1 ? lane % L : (int)threadIdx.x) * 8, nblk = gridDim.x;
  const float inv_d = 1.f / (float)d;
  const bool dxf = D.dx_dtype == VITA_DT_F32;
  int turn = 0;
  float gm[NV][8], ag[NV][8], ab[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    vec_load8(D.gamma, t0 + i * W * 512, d, al, 1.f, gm[i]);
#pragma unroll
    for (int r = 0; r < 8; ++r) ag[i][r] = ab[i][r] = 0.f;
  }
  const int ct = NV * 512 + lane;                // the lane's column behind the chunks
  const float gt = T && ct < d && D.gamma ? D.gamma[ct] : 1.f;
  float agt = 0.f, abt = 0.f;
  const int64_t step = (int64_t)nblk * R;
  for (int64_t row = (int64_t)blockIdx.x * R + (L < 64 ? (int)threadIdx.x / L : W == 1 ? wave : 0); row < D.rows; row += step) {
    Raw8 dyr[NV], sr[NV], ir[NV];
    uint32_t byte[NV];
    const bool whole = !T && row + 2 < D.rows; // the last chunk of a row as one load (pieces cost a wait in front of the next operand's)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t0 + i * W * 512;
      dyr[i] = raw_load8<DYF>((const char*)D.dy + row * D.lddy * (DYF ? 4 : 2), c, d, whole);
      if (SRC == 0) {
        sr[i].a = u32x4{0, 0, 0, 0};
        byte[i] = 127;
        if (c < d) {
          const u32x2 w = *reinterpret_cast<const u32x2*>((const uint8_t*)D.q + row * D.ldq + c);
          sr[i].a[0] = w[0]; sr[i].a[1] = w[1];
          byte[i] = ((const uint8_t*)D.scale)[row * D.lds + (c >> 5)];
        }
      } else {
        sr[i] = raw_load8<SRC == 2>((const char*)D.src + row * D.ldx * (SRC == 2 ? 4 : 2), c, d, whole);
      }
    }
    if (D.dx_in) {
      if (dxf) {
#pragma unroll
        for (int i = 0; i < NV; ++i) ir[i] = raw_load8<true>((const float*)D.dx_in + row * D.lddx_in, t0 + i * W * 512, d, whole);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) ir[i] = raw_load8<false>((const uint16_t*)D.dx_in + row * D.lddx_in, t0 + i * W * 512, d, whole);
      }
    }
    const float rs = D.rstd[row], mu = SRC != 0 && D.mean ? D.mean[row] : 0.f;
    float dyt = 0.f, nt = 0.f, it = 0.f;
    if (T) {
      dyt = load1<DYF>((const char*)D.dy + row * D.lddy * (DYF ? 4 : 2), ct, d);
      if (SRC == 0) {
        if (ct < d) nt = act8_decode1(((const uint8_t*)D.q)[row * D.ldq + ct], ((const uint8_t*)D.scale)[row * D.lds + (ct >> 5)]);
      } else if (ct < d) {
        nt = (load1<SRC == 2>((const char*)D.src + row * D.ldx * (SRC == 2 ? 4 : 2), ct, d) - mu) * rs;
      }
      if (D.dx_in) it = dxf ? load1<true>((const float*)D.dx_in + row * D.lddx_in, ct, d) : load1<false>((const uint16_t*)D.dx_in + row * D.lddx_in, ct, d);
    }
    const auto values = [&](int i, float (&dy)[8], float (&n)[8]) {
      raw_values8<DYF>(dyr[i], dy);
      if (SRC == 0) {
        act8_decode(u32x2{sr[i].a[0], sr[i].a[1]}, byte[i], n);
      } else {
        raw_values8<SRC == 2>(sr[i], n);
#pragma unroll
        for (int r = 0; r < 8; ++r) n[r] = (n[r] - mu) * rs;
      }
      const int c = t0 + i * W * 512;
      if (c + 8 > d) {
#pragma unroll
        for (int r = 0; r < 8; ++r) if (c + r >= d) { n[r] = 0.f; if (!T) dy[r] = 0.f; }
      }
    };
    float s1 = 0.f, s2 = 0.f;
    if (T) {
      s1 = dyt * gt;
      s2 = s1 * nt;
      agt = __builtin_fmaf(dyt, nt, agt);
      abt += dyt;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float dy[8], n[8];
      values(i, dy, n);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float h = dy[r] * gm[i][r];
        ag[i][r] = __builtin_fmaf(dy[r], n[r], ag[i][r]);
        ab[i][r] += dy[r];
        s1 += h;
        s2 = __builtin_fmaf(h, n[r], s2);
      }
    }
    row_sum2<W, L>(s1, s2, red, turn, wave, lane);
    // the values once more from the raw registers (the empty asm keeps the compiler from holding them over the sum: 16 NV registers)
#pragma unroll
    for (int i = 0; i < NV; ++i) asm volatile("" : "+v"(dyr[i].a), "+v"(sr[i].a));
    const float c1 = D.kind == AN_LAYER ? s1 * inv_d : 0.f, c2 = s2 * inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t0 + i * W * 512;
      float dy[8], n[8], o[8];
      values(i, dy, n);
#pragma unroll
      for (int r = 0; r < 8; ++r) o[r] = (dy[r] * gm[i][r] - c1 - n[r] * c2) * rs;
      if (D.dx_in) {
        float t[8];
        if (dxf) raw_values8<true>(ir[i], t); else raw_values8<false>(ir[i], t);
#pragma unroll
        for (int r = 0; r < 8; ++r) o[r] += t[r];
      }
      if (c + 8 > d) {
#pragma unroll
        for (int r = 0; r < 8; ++r) if (c + r >= d) o[r] = 0.f;
      }
      store8((char*)D.dx + row * D.lddx * (dxf ? 4 : 2), c, D.lddx, dxf, o);
      if (D.dx_bf16) store8((uint16_t*)D.dx_bf16 + row * D.lddxb, c, D.lddxb, false, o);
    }
    if (T) {
      const float o = ct < d ? (dyt * gt - c1 - nt * c2) * rs + it : 0.f;
      store1((char*)D.dx + row * D.lddx * (dxf ? 4 : 2), ct, D.lddx, dxf, o);
      if (D.dx_bf16) store1((uint16_t*)D.dx_bf16 + row * D.lddxb, ct, D.lddxb, false, o);
    }
  }
  if (!D.partial) return;
  if (L < 64) {                         // the wave's rows first
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int o = L; o < 64; o <<= 1) { ag[0][r] += __shfl_xor(ag[0][r], o, 64); ab[0][r] += __shfl_xor(ab[0][r], o, 64); }
  }
  float* pg = D.partial + (int64_t)blockIdx.x * d;
  float* pb = D.partial + ((int64_t)nblk + blockIdx.x) * d;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (k == 1 && !D.dbeta) break;
    if (W == 1) {                       // the block's four waves one after another, through LDS
      for (int w = 0; w < 4; ++w) {
        __syncthreads();
        if (wave == w && lane < L) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              f32x4* p = reinterpret_cast<f32x4*>(&sums[t0 + i * 512 + 4 * h]);
              const float (&a)[8] = k ? ab[i] : ag[i];
              f32x4 t = f32x4{a[4 * h], a[4 * h + 1], a[4 * h + 2], a[4 * h + 3]};
              if (w) t += *p;
              *p = t;
            }
          if (T) sums[ct] = (w ? sums[ct] : 0.f) + (k ? abt : agt);
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

// column sums of the partial rows: grid (ceil(d / 32), 1 or 2), 32 rows of threads over interleaved rows, all of a thread's loads in
// flight at once, fixed order
#define AN_RED_U ((AN_BWD_MAXBLK + 31) / 32)
__global__ __launch_bounds__(1024) void addnorm_reduce_kernel(const float* __restrict__ partial, int nblk, int d, float* dgamma,
                                                              float* dbeta, int acc) {
  __shared__ float red[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cx;
  const float* p = partial + (int64_t)blockIdx.y * nblk * d + c;
  float a[AN_RED_U], t = 0.f;
#pragma unroll
  for (int u = 0; u < AN_RED_U; ++u) {
    const int k = ry + 32 * u;
    a[u] = c < d && k < nblk ? p[(int64_t)k * d] : 0.f;
  }
#pragma unroll
  for (int u = 0; u < AN_RED_U; ++u) t += a[u];
  red[ry][cx] = t;
  __syncthreads();
  float* o = blockIdx.y ? dbeta : dgamma;
  if (ry == 0 && c < d && o) {
    t = 0.f;
#pragma unroll
    for (int w = 0; w < 32; ++w) t += red[w][cx];
    o[c] = acc ? o[c] + t : t;
  }
}

extern "C" int64_t vita_addnorm_bwd_nblk(int64_t rows, int64_t d) {
  // two rows at least for a wave (for a block of several waves to a row), and no more blocks than are resident: 1 to 3 a CU
  const int64_t n = d <= 128 ? (rows + 31) / 32 : d <= 256 ? (rows + 15) / 16 : d <= 1536 ? (rows + 7) / 8 : (rows + 1) / 2;
  const int64_t most = d > 4096 ? AN_BWD_MAXBLK / 3 : d > 2048 || (d > 1088 && d <= 1536) ? AN_BWD_MAXBLK * 2 / 3 : AN_BWD_MAXBLK;
  return n < most ? n : most;
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
  if (D.kind == AN_RMS) {
    VITA_REQUIRE(!D.dbeta);
    D.mean = nullptr;                   // mu = 0
  }
  int64_t width = (D.d + 7) & ~(int64_t)7;
  if (D.lddx > width) width = D.lddx;
  if (D.dx_bf16 && D.lddxb > width) width = D.lddxb;
  if (width > AN_MAX_D) {
    vita_set_error("vita_addnorm_bwd: rows of more than 8192 columns (with their pads)", hipSuccess);
    return VITA_ERR_UNSUPPORTED;
  }
  const int nblk = (int)vita_addnorm_bwd_nblk(D.rows, D.d);
  const int al = ((uintptr_t)D.gamma & 15) == 0;
  const int src = D.q ? 0 : (D.src_dtype == VITA_DT_F32 ? 2 : 1);
#define AN_LAUNCH(W, NV, M, SRC, DYF) \
  hipLaunchKernelGGL((addnorm_bwd_kernel<W, NV, M, SRC, DYF>), dim3(nblk), dim3(W == 1 ? 256 : 64 * W), 0, (hipStream_t)stream, D, al)
#define AN_TYPES(W, NV, M)                                                                                                                   \
  do {                                                                                                                                       \
    if (D.dy_dtype == VITA_DT_F32) {                                                                                                         \
      if (src == 0) AN_LAUNCH(W, NV, M, 0, true); else if (src == 1) AN_LAUNCH(W, NV, M, 1, true); else AN_LAUNCH(W, NV, M, 2, true);       \
    } else {                                                                                                                                 \
      if (src == 0) AN_LAUNCH(W, NV, M, 0, false); else if (src == 1) AN_LAUNCH(W, NV, M, 1, false); else AN_LAUNCH(W, NV, M, 2, false);    \
    }                                                                                                                                        \
  } while (0)
  // One wave a row up to 1536 columns (30000 x 1025 from 8 bits, fp32 dx_in and dx: 70 us, with four waves 121), beyond as many waves as
  // hold the row with one chunk a lane, since a chunk costs some 50 registers here: 20000 x 2000 140 us with four waves, 158 with two chunks
  // a lane; fp32 dy, bf16 dx_in and dx: 17918 x 2636 102 with six, 135 with eight and 205 with four of two chunks; 9000 x 5000 96
  // with twelve, 115 with sixteen, 209 with four of four.  Narrow rows as in the forward pass: 46082 x 69 11.4 against 26.4 us.
  if (width <= 128) AN_TYPES(1, 1, 16);
  else if (width <= 256) AN_TYPES(1, 1, 32);
  else if (width <= 512) AN_TYPES(1, 1, AN_FULL);
  else if (width <= 1024) AN_TYPES(1, 2, AN_FULL);
  else if (width <= 1088) AN_TYPES(1, 2, AN_TAIL);
  else if (width <= 1536) AN_TYPES(1, 3, AN_FULL);
  else if (width <= 2048) AN_TYPES(4, 1, AN_FULL);
  else if (width <= 6 * 512) AN_TYPES(6, 1, AN_FULL);
  else if (width <= 4096) AN_TYPES(8, 1, AN_FULL);
  else if (width <= 6144) AN_TYPES(12, 1, AN_FULL);
  else AN_TYPES(16, 1, AN_FULL);
#undef AN_TYPES
#undef AN_LAUNCH
  VITA_CHECK_LAUNCH("vita_addnorm_bwd");
  if (D.partial) {
    hipLaunchKernelGGL(addnorm_reduce_kernel, dim3((unsigned)((D.d + 31) / 32), D.dbeta ? 2 : 1), dim3(1024), 0, (hipStream_t)stream,
                       D.partial, nblk, (int)D.d, D.dgamma, D.dbeta, D.accumulate);
    VITA_CHECK_LAUNCH("vita_addnorm_bwd_reduce");
  }
  return VITA_OK;
}
