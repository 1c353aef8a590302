// Weight gradient from an 8-bit checkpoint: dw[i][j] = sum_k dy[k][i] * value[k][j], fp32.
//
// value = code * 2^e is exact in bf16 (act8.h), so the codes are turned into bf16 on their way into LDS and the products run on
// v_mfma_f32_16x16x32_bf16 with no rounding beyond fp32 accumulation: nothing of the restored matrix ever reaches HBM.
//
//   * 256 x (16 NF) x 64 tiles, 8 waves (4 x 2), the pipeline of gemm256.hip: dy goes HBM -> LDS by LDS-DMA, fragments are read
//     with ds_read_b64_tr_b16 under the MFMAs, one barrier per K-tile.  A code tile takes the same road through registers: 16 codes
//     and their scale byte per load, fetched a whole K-tile before they are needed, converted (16 conversions, 4 ds_write_b128 per
//     thread and K-tile) right behind the barrier that frees their stage - before the dy DMA is issued, so that the compiler has
//     no LDS-DMA in flight to order the writes against.
//   * the work is one line of tiles x K-tiles, cut into as many equal pieces as there are workgroups, wherever that falls.  A
//     weight matrix gives few tiles (1025 x 4100: 85) and a token count long sums: a cut at whole tiles leaves up to half of
//     the chip idle in the last round.  A piece that is not a whole tile goes to the workspace as fp32; a second kernel adds a
//     tile's pieces in their order.  One writer per element, no atomics: the same bits on every call.
#include "act8.h"
#include "gemm256.h"

struct Wgrad8Params {
  const uint16_t* dy;
  const uint8_t* q;
  const uint8_t* scale;
  float* dw;
  float* ws;
  int64_t lddy, ldq, lds, lddw;
  int64_t m, n, k;
  int tiles_m, tiles_n, kt;      // kt = K-tiles of one tile
  int pieces;                    // workgroups
  int per_tile;                  // pieces per tile, rounded: workgroups that far apart walk over the same tokens
  int accumulate;
};

// first iteration (tile * kt + K-tile) of piece w
__device__ __host__ __forceinline__ int64_t w8_begin(const Wgrad8Params& P, int w) {
  return (int64_t)P.tiles_m * P.tiles_n * P.kt * w / P.pieces;
}
// workspace slot of the part of a tile that piece w holds: a piece has at most one that starts inside a tile (slot 0) and one
// that starts with a tile and ends inside it (slot 1)
__device__ __forceinline__ int64_t w8_slot(int w, bool from_start) { return 2 * (int64_t)w + (from_start ? 1 : 0); }

__device__ __forceinline__ uint64_t w8_uniform(uint64_t v) { return ((uint64_t)g2_sgpr((uint32_t)(v >> 32)) << 32) | g2_sgpr((uint32_t)v); }
// descriptor of the bytes [adv, bytes) behind base, all in scalar registers
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w8_rsrc(uint64_t base, uint32_t adv, uint32_t bytes) {
  return g2_rsrc((const void*)(base + adv), g2_sgpr(adv < bytes ? bytes - adv : 0u));
}

template <int NF>
__global__ __launch_bounds__(G2_THREADS, 2) void act8_wgrad_kernel(const Wgrad8Params P) {
  constexpr int NFW = (NF + 1) / 2, BM = 256;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 3, wn = wave >> 2;
  const int nfw = wn == 0 ? NFW : NF - NFW;

  // workgroup -> piece.  Workgroups of one XCD (blockIdx % 8) get pieces per_tile apart: neighbouring tiles over the same tokens,
  // whose rows of dy and codes they share in that XCD's L2.
  int w;
  {
    const int nwg = P.pieces, qd = nwg >> 3, r = nwg & 7, xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
    const int l = (xcd < r ? xcd * (qd + 1) : r * (qd + 1) + (xcd - r) * qd) + idx;
    const int per = nwg / P.per_tile;
    w = l < per * P.per_tile ? (l % per) * P.per_tile + l / per : l;
  }
  const int64_t it_end = w8_begin(P, w + 1);
  int64_t it = w8_begin(P, w);

  typedef G2Loader<1, BM, 8> LoaderA;
  constexpr int BOFF = LoaderA::BYTES, STAGE = BOFF + 32768;
  constexpr int PA = LoaderA::PPW;
  // code chunks of this thread: k-rows tid / 16 and 32 below, columns 16 (tid % 16); 16 codes = one 32-byte chunk of the bf16 image
  // (the swizzle g2_f does not see bit 5 of the row: the second chunk lies 32 rows of 512 bytes behind the first)
  const int bcol = tid & 15, brow = tid >> 4;
  const uint32_t boff = BOFF + brow * 512 + ((bcol ^ (int)g2_f(brow)) << 5);
  const int64_t ncodes = (P.n + ACT8_GROUP - 1) / ACT8_GROUP * ACT8_GROUP;

  while (it < it_end) {
    const int tile = (int)g2_sgpr((uint32_t)(it / P.kt));
    const int kt0 = (int)g2_sgpr((uint32_t)(it - (int64_t)tile * P.kt));
    int nkt = P.kt - kt0;
    if (nkt > it_end - it) nkt = (int)(it_end - it);
    const int tm = tile / P.tiles_n, tn = tile - tm * P.tiles_n;
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * (NF * 16), k0 = (int64_t)kt0 * G2_BK;
    const int64_t krows = P.k - k0 < (int64_t)nkt * G2_BK ? P.k - k0 : (int64_t)nkt * G2_BK;      // tokens of this part

    LoaderA la;
    la.init(P.dy + k0 * P.lddy, m0, P.m, krows, P.lddy, wave, lane);
    G2Frags<1, 4> fa;
    G2Frags<1, NFW> fb;
    fa.init(wm * 4, 0, lane);
    fb.init(wn * NFW, BOFF, lane);

    // bounds-checked loads: tokens past the part and columns past the codes arrive as zeros
    const uint32_t col_on = bcol < NF && n0 + bcol * 16 < ncodes;
    const uint32_t qoff = col_on ? (uint32_t)(brow * P.ldq) + bcol * 16 : G2_OOB;
    const uint32_t soff = col_on ? (uint32_t)(brow * P.lds) + (((uint32_t)(n0 & 31) + bcol * 16) >> 5) : G2_OOB;
    const uint64_t qbase = w8_uniform((uint64_t)(P.q + k0 * P.ldq + n0)), sbase = w8_uniform((uint64_t)(P.scale + k0 * P.lds + (n0 >> 5)));
    const uint32_t qbytes = g2_sgpr((uint32_t)((krows - 1) * P.ldq + (ncodes - n0)));
    const uint32_t sbytes = g2_sgpr((uint32_t)((krows - 1) * P.lds + ((ncodes >> 5) - (n0 >> 5))));
    u32x4 qv[2];
    uint32_t sv[2];
    auto b_load = [&](int t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t r = (uint32_t)t * G2_BK + 32 * i;
        const uint32_t qa = g2_sgpr(r * (uint32_t)P.ldq), sa = g2_sgpr(r * (uint32_t)P.lds);
        qv[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(w8_rsrc(qbase, qa, qbytes), qoff, 0, 0));
        sv[i] = __builtin_amdgcn_raw_buffer_load_b8(w8_rsrc(sbase, sa, sbytes), soff, 0, 0);
      }
    };
    auto b_write = [&](int stage) {
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float s = act8_scale(sv[i]);
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[2 * j] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)qv[i][j], s, false));
          o[2 * j + 1] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)qv[i][j], s, true));
        }
        char* p = smem + stage * STAGE + boff + i * 16384;
        *reinterpret_cast<u32x4*>(p) = u32x4{o[0], o[1], o[2], o[3]};
        *reinterpret_cast<u32x4*>(p + 16) = u32x4{o[4], o[5], o[6], o[7]};
      }
    };

    f32x4 acc[4][NFW];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NFW; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    bf16x8 a0[4], b0[NFW], a1[4], b1[NFW];
    // operands swapped: a lane ends up with 4 neighbouring columns of one row
#define W8_MFMA_GROUP(J, AF, BF)                                                                       \
  if (NF % 2 == 0 || (J) < NFW - 1 || wn == 0) {                                                       \
    _Pragma("unroll") for (int i = 0; i < 4; ++i)                                                      \
      acc[i][J] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(BF[J], AF[i], acc[i][J], 0, 0, 0);           \
  }
#define W8_READ_B(KS, BF, LO, HI) fb.template read_range<KS, true, LO, HI, NFW>(smem, BF)
#define W8_READ_A(KS, AF) fa.template read_range<KS, true, 0, 4, 4>(smem, AF)
    // every fragment read issued so far has landed (the compiler cannot see those reads)
#define W8_WAIT_FRAGS() do { __builtin_amdgcn_s_waitcnt(0xc07f); __builtin_amdgcn_sched_barrier(0); } while (0)
#define W8_PHASE1()                                                  \
  W8_WAIT_FRAGS();                                                   \
  _Pragma("unroll") for (int j = 0; j < NFW; ++j) {                  \
    if (j == 0) { W8_READ_A(1, a1); W8_READ_B(1, b1, 0, 1); }        \
    if (j == 1) { W8_READ_B(1, b1, 1, 4); }                          \
    if (j == 2) { W8_READ_B(1, b1, 4, NFW); }                        \
    W8_MFMA_GROUP(j, a0, b0);                                        \
    __builtin_amdgcn_sched_barrier(0);                               \
  }
    // K-tiles 0 and 1 (one past the end: dy arrives as zeros, the codes are taken as zeros)
    b_load(0);
    b_write(0);
    b_load(1);
    {
      const __amdgpu_buffer_rsrc_t ra = la.rsrc(0);
#pragma unroll
      for (int i = 0; i < PA; ++i) la.issue(ra, true, i, smem, wave);
    }
    g2_sync_all();
    b_write(1);
    b_load(2);
    {
      const __amdgpu_buffer_rsrc_t ra = la.rsrc(1);
#pragma unroll
      for (int i = 0; i < PA; ++i) la.issue(ra, true, i, smem + STAGE, wave);
    }
    W8_READ_A(0, a0); W8_READ_B(0, b0, 0, NFW);
    for (int t = 0; t + 1 < nkt; ++t) {
      W8_PHASE1();
      // K-tile t+1 is complete in LDS for every wave, and every wave has read K-tile t: its stage is free for K-tile t+2
      g2_sync_all();
      fa.toggle((t & 1) ? -STAGE : STAGE); fb.toggle((t & 1) ? -STAGE : STAGE);
      b_write(t & 1);
      b_load(t + 3);
      const __amdgpu_buffer_rsrc_t ra = la.rsrc(t + 2);
      char* st = smem + (t & 1) * STAGE;
#pragma unroll
      for (int j = 0; j < NFW; ++j) {
#pragma unroll
        for (int i = 0; i < PA; ++i)
          if (i == j) la.issue(ra, true, i, st, wave);
        if (j == 0) { W8_READ_A(0, a0); }
        if (j == 1) { W8_READ_B(0, b0, 0, 3); }
        if (j == 2) { W8_READ_B(0, b0, 3, NFW); }
        W8_MFMA_GROUP(j, a1, b1);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    W8_PHASE1();
    W8_WAIT_FRAGS();
#pragma unroll
    for (int j = 0; j < NFW; ++j) { W8_MFMA_GROUP(j, a1, b1); }
#undef W8_PHASE1
#undef W8_WAIT_FRAGS
#undef W8_MFMA_GROUP
#undef W8_READ_A
#undef W8_READ_B
    __builtin_amdgcn_s_waitcnt(0x0070);      // no LDS-DMA (of the K-tile past the end) outlives its part, or the workgroup

    // lane: row lane & 15, columns 4 (lane >> 4) .. + 3 of each 16 x 16 fragment
    const int cl = wn * NFW * 16 + 4 * (lane >> 4), rl = wm * 64 + (lane & 15);
    if (nkt == P.kt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t row = m0 + rl + 16 * i;
        if (row >= P.m) continue;
        float* o = P.dw + row * P.lddw;
#pragma unroll
        for (int j = 0; j < NFW; ++j) {
          if (j >= nfw) continue;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int64_t col = n0 + cl + 16 * j + r;
            if (col < P.n) o[col] = P.accumulate ? o[col] + acc[i][j][r] : acc[i][j][r];
          }
        }
      }
    } else {
      float* o = P.ws + w8_slot(w, kt0 == 0) * (BM * NF * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NFW; ++j)
          if (j < nfw) *reinterpret_cast<f32x4*>(o + (rl + 16 * i) * (NF * 16) + cl + 16 * j) = acc[i][j];
    }
    it += nkt;
    if (it < it_end) g2_sync_all();          // every wave has read the last K-tile: the stages are free
  }
}

// adds the parts of each cut tile, in their order.  A thread owns 4 neighbouring columns of a row.
__global__ __launch_bounds__(256) void act8_wgrad_join_kernel(const Wgrad8Params P, const int width) {
  const int tile = blockIdx.x;
  const int64_t t0 = (int64_t)tile * P.kt, t1 = t0 + P.kt;
  const int64_t total = (int64_t)P.tiles_m * P.tiles_n * P.kt;
  int w0 = (int)(t0 * P.pieces / total);                 // the piece that holds iteration t0
  while (w0 + 1 < P.pieces && w8_begin(P, w0 + 1) <= t0) ++w0;
  while (w0 > 0 && w8_begin(P, w0) > t0) --w0;
  if (w8_begin(P, w0 + 1) >= t1) return;                 // one piece holds all of the tile: written already
  const int quad = blockIdx.y * 256 + threadIdx.x;       // 4 columns each
  const int per_row = width / 4;
  const int rl = quad / per_row, cl = (quad - rl * per_row) * 4;
  if (rl >= 256) return;
  const int tm = tile / P.tiles_n, tn = tile - tm * P.tiles_n;
  const int64_t row = (int64_t)tm * 256 + rl, col = (int64_t)tn * width + cl;
  if (row >= P.m || col >= P.n) return;
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int w = w0; w < P.pieces && w8_begin(P, w) < t1; ++w)
    s += *reinterpret_cast<const f32x4*>(P.ws + w8_slot(w, w8_begin(P, w) <= t0) * (256 * (int64_t)width) + (int64_t)rl * width + cl);
  float* o = P.dw + row * P.lddw + col;
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (col + r < P.n) o[r] = P.accumulate ? o[r] + s[r] : s[r];
}

// ---- host
struct Wgrad8Plan { int nf, pieces; };
// Tile width and number of workgroups: the longest piece in K-tiles (plus 3 of start and end) times the cost of one (its width plus
// what a narrow tile loses), plus the parts' way through the workspace.
static Wgrad8Plan w8_plan(int64_t m, int64_t n, int64_t k) {
  const int64_t tm = (m + 255) / 256, kt = (k + G2_BK - 1) / G2_BK;
  Wgrad8Plan best = {13, 1};
  double cost = -1;
  const int cand[3] = {8, 13, 16};
  for (int c = 0; c < 3; ++c) {
    const int nf = cand[c];
    const int64_t tiles = tm * ((n + nf * 16 - 1) / (nf * 16)), total = tiles * kt;
    int64_t pieces = total < 256 ? total : 256;
    const int64_t few = (total + 3) / 4;                  // at least 4 K-tiles to a piece
    if (pieces > few) pieces = few;
    const double x = (double)((total + pieces - 1) / pieces + 3) * (nf + 3);
    if (cost < 0 || x < cost) { cost = x; best = {nf, (int)pieces}; }
  }
  return best;
}
extern "C" int64_t vita_act8_wgrad_ws_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const Wgrad8Plan p = w8_plan(m, n, k);
  return 2 * (int64_t)p.pieces * 256 * p.nf * 16 * 4;
}

template <int NF>
static int w8_launch(const Wgrad8Params& P, hipStream_t s) {
  constexpr int lds = 2 * (32768 + 32768);
  static VitaPerDeviceOnce once;
  vita_set_max_lds_once(once, (const void*)act8_wgrad_kernel<NF>, lds);
  hipLaunchKernelGGL(act8_wgrad_kernel<NF>, dim3((unsigned)P.pieces), dim3(G2_THREADS), lds, s, P);
  VITA_CHECK_LAUNCH("vita_act8_wgrad");
  if (P.pieces % (P.tiles_m * P.tiles_n) == 0 ? P.pieces > P.tiles_m * P.tiles_n : true) {
    hipLaunchKernelGGL(act8_wgrad_join_kernel, dim3((unsigned)(P.tiles_m * P.tiles_n), 256 * NF * 4 / 256), dim3(256), 0, s, P, NF * 16);
    VITA_CHECK_LAUNCH("vita_act8_wgrad_join");
  }
  return VITA_OK;
}

extern "C" int vita_act8_wgrad(const void* dy, int64_t lddy, const void* q, int64_t ldq, const void* scale, int64_t lds, float* dw,
                               int64_t lddw, int64_t m, int64_t n, int64_t k, int32_t accumulate, void* ws, int64_t ws_bytes, void* stream) {
  VITA_REQUIRE(m > 0 && n > 0 && k > 0 && n <= ACT8_MAX_COLS && m <= ACT8_MAX_COLS && k <= ((int64_t)1 << 31));
  VITA_REQUIRE(act8_mat_ok(dy, lddy, m, VITA_DT_BF16) && dw && lddw >= n);
  VITA_REQUIRE(act8_codes_ok(q, ldq, scale, lds, n));
  VITA_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= vita_act8_wgrad_ws_bytes(m, n, k));
  const Wgrad8Plan plan = w8_plan(m, n, k);
  Wgrad8Params P;
  P.dy = (const uint16_t*)dy; P.q = (const uint8_t*)q; P.scale = (const uint8_t*)scale; P.dw = dw; P.ws = (float*)ws;
  P.lddy = lddy; P.ldq = ldq; P.lds = lds; P.lddw = lddw;
  P.m = m; P.n = n; P.k = k;
  const int64_t tiles_m = (m + 255) / 256, tiles_n = (n + plan.nf * 16 - 1) / (plan.nf * 16), kt = (k + G2_BK - 1) / G2_BK;
  VITA_REQUIRE(tiles_m * tiles_n < ((int64_t)1 << 30));
  P.tiles_m = (int)tiles_m; P.tiles_n = (int)tiles_n; P.kt = (int)kt;
  P.pieces = plan.pieces;
  P.accumulate = accumulate;
  // 32-bit offsets inside a part's tokens (a part is at most kt K-tiles long, and is read up to 3 K-tiles past its end)
  const int64_t longest = (tiles_m * tiles_n * kt + P.pieces - 1) / P.pieces;
  const int64_t part = ((longest < kt ? longest : kt) + 4) * G2_BK;
  if (part * lddy * 2 >= (int64_t)0x7fffff00ll || part * ldq >= (int64_t)0x7fffff00ll || part * lds >= (int64_t)0x7fffff00ll) {
    vita_set_error("vita_act8_wgrad: 2 GiB or more of dy or of codes in one part of the sum", hipSuccess);
    return VITA_ERR_UNSUPPORTED;
  }
  const int64_t per = (P.pieces + tiles_m * tiles_n / 2) / (tiles_m * tiles_n);
  P.per_tile = per < 1 ? 1 : (int)per;
  switch (plan.nf) {
    case 8: return w8_launch<8>(P, (hipStream_t)stream);
    case 13: return w8_launch<13>(P, (hipStream_t)stream);
    default: return w8_launch<16>(P, (hipStream_t)stream);
  }
}
template __global__ void act8_wgrad_kernel<8>(const Wgrad8Params);
template __global__ void act8_wgrad_kernel<13>(const Wgrad8Params);
template __global__ void act8_wgrad_kernel<16>(const Wgrad8Params);
