// Weight gradient from an 8-bit checkpoint: dw[i][j] = sum_k dy[k][i] * value[k][j], fp32.
//
// value = code * 2^e is exact in bf16 (act8.h), so the codes are turned into bf16 on their way into LDS and the products run on
// v_mfma_f32_16x16x32_bf16 with no rounding beyond fp32 accumulation: nothing of the restored matrix ever reaches HBM.
//
//   * 256 x (16 NF) x 64 tiles, 8 waves (4 x 2), LDS images and fragments of gemm256.hip: dy goes HBM -> LDS by LDS-DMA, fragments are
//     read with ds_read_b64_tr_b16.  A code tile goes through registers: 16 codes and their scale byte per load, fetched a whole
//     K-tile before they are needed, converted and written (16 conversions, 4 ds_write_b128 per thread and K-tile) between the
//     matrix instructions.  The two waves of a SIMD take turns at the matrix pipe (schedule at the loop).
//   * a weight matrix gives few tiles (1025 x 4100: 85) and a token count long sums, so tiles are cut along the tokens (w8_plan):
//     whole rounds of 256 tiles stay whole, of the others as many as fit are cut into `cut` equal parts, one per workgroup, and
//     what is left over is dealt out in short pieces behind those.  Equal cuts keep the workgroups of an XCD (blockIdx % 8) on the
//     same tokens of neighbouring tiles, whose rows of dy and codes they then share in that XCD's L2: one line of tiles x K-tiles
//     cut into 256 equal pieces balances better by a tenth, but the pieces drift apart and 70 % of the L2 requests missed (6 TB/s
//     from behind it; 13826 tokens, 1025 x 3075: 114 us).
//   * a part of a tile goes to the workspace as fp32; a second kernel adds a tile's parts in their order.  One writer per
//     element, no atomics: the same bits on every call.
//
// Measured (MI355X): 3776 tokens, 1025 x 4100: 42 + 13 us (join), 750 TFLOP/s without the join; 13826 tokens, 1025 x 3075: 100 to 109 + 13
// us, 800 to 870 TFLOP/s; the bf16 kernel of gemm256.hip with atomics takes 85 and 131 us for the same shapes, without the pass that restores its
// operand.  Bound by what one wave after another can issue: without the conversions 98 us of the 109 are left, without the DMA of dy
// 96, without either 85 (matrix instructions, fragment reads, barriers); without the loads of the codes 109.  With all waves in step and
// the conversions in one piece behind the barrier the two shapes take 43 and 114 to 122 us; with four waves of twice the rows 124; when
// in the K-tile the DMA is issued makes no difference.  8 of the 42 us are the writing of the parts (in fragment order or not alike,
// non-temporal 12); 15 us the join with single floats stored.
#include "act8.h"
#include "gemm256.h"
#include <type_traits>

#define W8_WGS 256               // workgroups of a full round: one per CU

struct Wgrad8Params {
  const uint16_t* dy;
  const uint8_t* q;
  const uint8_t* scale;
  float* dw;
  float* ws;
  int64_t lddy, ldq, lds, lddw;
  int64_t m, n, k;
  int tiles_m, tiles_n, kt;      // kt = K-tiles of one tile
  int whole;                     // tiles [0, whole) are never cut: whole / W8_WGS per workgroup
  int cut, cut_tiles;            // tiles [whole, whole + cut_tiles) in `cut` parts each, cut_tiles * cut <= W8_WGS
  int cut_kt, cut_more;          // K-tiles of a part; one more in the first cut_more of them
  int piece, pieces;             // the K-tiles of the other tiles, in one line, dealt out in pieces of `piece`
  int accumulate;
};

// tile number -> (tile row, tile column): neighbours along the shorter side, so that 32 workgroups in a row touch few panels
__device__ __forceinline__ void w8_tile(const Wgrad8Params& P, int tile, int& tm, int& tn) {
  if (P.tiles_n <= P.tiles_m) { tm = tile / P.tiles_n; tn = tile - tm * P.tiles_n; }
  else { tn = tile / P.tiles_m; tm = tile - tn * P.tiles_m; }
}
// workspace slots: one for each part of a cut tile, then two for each piece (it may hold the end of one tile and the start of the next)
__device__ __forceinline__ int64_t w8_cut_slot(const Wgrad8Params& P, int tile, int part) { return (int64_t)(tile - P.whole) * P.cut + part; }
__device__ __forceinline__ int64_t w8_piece_slot(const Wgrad8Params& P, int piece, int second) {
  return (int64_t)P.cut_tiles * P.cut + 2 * piece + second;
}
__device__ __forceinline__ int w8_cut_begin(const Wgrad8Params& P, int part) { return part * P.cut_kt + (part < P.cut_more ? part : P.cut_more); }

// 4 neighbouring columns of a row of dw, `left` of them inside; rows start on any 4-byte boundary, which 16-byte stores take too
__device__ __forceinline__ void w8_put(const Wgrad8Params& P, float* o, f32x4 v, int64_t left) {
  typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
  if (left >= 4) {
    if (P.accumulate) v += *reinterpret_cast<const f32x4_any*>(o);
    *reinterpret_cast<f32x4_any*>(o) = v;
  } else {
#pragma unroll
    for (int r = 0; r < 3; ++r)
      if (r < left) o[r] = P.accumulate ? o[r] + v[r] : v[r];
  }
}

__device__ __forceinline__ uint64_t w8_uniform(uint64_t v) { return ((uint64_t)g2_sgpr((uint32_t)(v >> 32)) << 32) | g2_sgpr((uint32_t)v); }
// descriptor of the bytes [adv, bytes) behind base; operands uniform and below 2^31 (the host checks them).  The maximum is a signed one
// because that stays on the scalar unit: a compare and select went to vector registers, and the loads into loops over lanes.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t w8_rsrc(uint64_t base, uint32_t adv, uint32_t bytes) {
  const int rem = (int)bytes - (int)adv;
  return g2_rsrc((const void*)(base + adv), (uint32_t)(rem > 0 ? rem : 0));
}

template <int NF>
__global__ __launch_bounds__(G2_THREADS, 2) void act8_wgrad_kernel(const Wgrad8Params P) {
  constexpr int NFW = (NF + 1) / 2, BM = 256;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 3, wn = wave >> 2;
  const int nfw = wn == 0 ? NFW : NF - NFW;

  // position in the order of XCDs: neighbours share an L2
  int l;
  {
    const int nwg = gridDim.x, qd = nwg >> 3, r = nwg & 7, xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
    l = (xcd < r ? xcd * (qd + 1) : r * (qd + 1) + (xcd - r) * qd) + idx;
  }
  // this workgroup's parts, one after another: its whole tiles, its part of a cut tile, its piece (in two parts where it straddles
  // two tiles).  step counts them.
  const int n_whole = P.whole / W8_WGS;
  const int first_piece = (int)gridDim.x - 1 - l;      // from the far end: the workgroups without a cut part come first
  int step = 0;

  typedef G2Loader<1, BM, 8> LoaderA;
  constexpr int BOFF = LoaderA::BYTES, STAGE = BOFF + 32768;
  constexpr int PA = LoaderA::PPW;
  // code chunks of this thread: k-rows tid / 16 and 32 below, columns 16 (tid % 16); 16 codes = one 32-byte chunk of the bf16 image
  // (the swizzle g2_f does not see bit 5 of the row: the second chunk lies 32 rows of 512 bytes behind the first)
  const int bcol = tid & 15, brow = tid >> 4;
  const uint32_t boff = BOFF + brow * 512 + ((bcol ^ (int)g2_f(brow)) << 5);
  const int64_t ncodes = (P.n + ACT8_GROUP - 1) / ACT8_GROUP * ACT8_GROUP;

  for (;; ++step) {
    int tile, kt0, nkt;
    int64_t slot = -1;
    if (step < n_whole) {
      tile = step * W8_WGS + l; kt0 = 0; nkt = P.kt;
    } else if (step == n_whole) {
      if (l >= P.cut_tiles * P.cut) continue;
      const int part = l / P.cut_tiles;
      tile = P.whole + (l - part * P.cut_tiles);
      kt0 = w8_cut_begin(P, part);
      nkt = w8_cut_begin(P, part + 1) - kt0;
      if (P.cut > 1) slot = w8_cut_slot(P, tile, part);
    } else {
      const int second = step - n_whole - 1;
      if (second > 1 || first_piece >= P.pieces) break;
      const int rest = P.whole + P.cut_tiles;          // first tile of the line
      const int64_t line = (int64_t)(P.tiles_m * P.tiles_n - rest) * P.kt;
      int64_t a = (int64_t)first_piece * P.piece, e = a + P.piece;
      if (e > line) e = line;
      const int64_t border = (a / P.kt + 1) * P.kt;    // end of the tile that the piece starts in
      if (second) a = border; else if (e > border) e = border;
      if (a >= e) break;
      tile = rest + (int)(a / P.kt);
      kt0 = (int)(a % P.kt);
      nkt = (int)(e - a);
      slot = w8_piece_slot(P, first_piece, second);
    }
    tile = (int)g2_sgpr((uint32_t)tile); kt0 = (int)g2_sgpr((uint32_t)kt0); nkt = (int)g2_sgpr((uint32_t)nkt);
    int tm, tn;
    w8_tile(P, tile, tm, tn);
    if (step > 0) g2_sync_all();               // every wave has read the previous part's last K-tile: the stages are free
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * (NF * 16), k0 = (int64_t)kt0 * G2_BK;
    const int64_t krows = P.k - k0 < (int64_t)nkt * G2_BK ? P.k - k0 : (int64_t)nkt * G2_BK;      // tokens of this part

    LoaderA la;
    la.init(P.dy + k0 * P.lddy, m0, P.m, krows, P.lddy, wave, lane);
    // 16-byte pieces: the last one of the last token may reach behind the matrix' last element.  It is left out then (arrives as zeros)
    // and its up to 7 columns of dy are added after the products.
    if ((P.m & 7) && kt0 + nkt == P.kt) la.bytes -= 16;
    // bounds-checked loads: tokens past the part and columns past the codes arrive as zeros
    const uint32_t col_on = bcol < NF && n0 + bcol * 16 < ncodes;
    uint32_t qoff[2], soff[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      qoff[i] = col_on ? (uint32_t)((brow + 32 * i) * P.ldq) + bcol * 16 : G2_OOB;
      soff[i] = col_on ? (uint32_t)((brow + 32 * i) * P.lds) + (((uint32_t)(n0 & 31) + bcol * 16) >> 5) : G2_OOB;
    }
    const uint64_t abase = w8_uniform((uint64_t)(P.dy + k0 * P.lddy + m0));
    const uint64_t qbase = w8_uniform((uint64_t)(P.q + k0 * P.ldq + n0)), sbase = w8_uniform((uint64_t)(P.scale + k0 * P.lds + (n0 >> 5)));
    const uint32_t qbytes = g2_sgpr((uint32_t)((krows - 1) * P.ldq + (ncodes - n0)));
    const uint32_t sbytes = g2_sgpr((uint32_t)((krows - 1) * P.lds + ((ncodes >> 5) - (n0 >> 5))));
    const uint32_t qstep = g2_sgpr((uint32_t)(G2_BK * P.ldq)), sstep = g2_sgpr((uint32_t)(G2_BK * P.lds));
    auto a_rsrc = [&](int t) { return w8_rsrc(abase, (uint32_t)t * la.kstep, la.bytes); };
    auto q_rsrc = [&](int t) { return w8_rsrc(qbase, (uint32_t)t * qstep, qbytes); };
    auto s_rsrc = [&](int t) { return w8_rsrc(sbase, (uint32_t)t * sstep, sbytes); };
    u32x4 qv[2];
    uint32_t sv[2];
    auto b_load = [&](__amdgpu_buffer_rsrc_t rq, __amdgpu_buffer_rsrc_t rs, int i) {
      qv[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rq, qoff[i], 0, 0));
      sv[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, soff[i], 0, 0);
    };
    // 16 codes -> 16 bf16 -> LDS in six steps: four codes each, then the two halves written.  The writes are inline asm: the compiler
    // would wait for every LDS-DMA in flight before a write of its own.  They are waited for with the fragment reads (lgkmcnt(0)).
    u32x4 bo[2];
    auto b_step = [&](int stage, int i, int step) {
      typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
      if (step < 4) {
        const float sc = act8_scale(sv[i]);
        bo[step >> 1][2 * (step & 1)] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)qv[i][step], sc, false));
        bo[step >> 1][2 * (step & 1) + 1] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)qv[i][step], sc, true));
      } else {
        const uint32_t at = boff + stage * STAGE + i * 16384;
        if (step == 4) asm volatile("ds_write_b128 %0, %1" :: "v"(at), "v"(bo[0]) : "memory");
        else asm volatile("ds_write_b128 %0, %1 offset:16" :: "v"(at), "v"(bo[1]) : "memory");
      }
    };

    f32x4 acc[4][NFW];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NFW; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // K-tile 0, and the codes of K-tile 1 on their way (past the end: dy arrives as zeros, the codes are taken as zeros)
    {
      const __amdgpu_buffer_rsrc_t ra = a_rsrc(0), rq = q_rsrc(0), rs = s_rsrc(0), rq1 = q_rsrc(1), rs1 = s_rsrc(1);
#pragma unroll
      for (int i = 0; i < PA; ++i) la.issue(ra, true, i, smem, wave);
      b_load(rq, rs, 0); b_load(rq, rs, 1);
      __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt(0): this wave's pieces of dy are in LDS
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int k = 0; k < 6; ++k) b_step(0, i, k);
        b_load(rq1, rs1, i);
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);        // lgkmcnt(0): the codes too
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);

    // The two waves of a SIMD take turns.  Time goes in slots between barriers; in a K-tile a wave has four: it reads the fragments of
    // the first half (M0), multiplies them (C0), reads (M1) and multiplies (C1) the second half, and the second half of the workgroup
    // does the same one slot later, so that the matrix pipe of a SIMD always has one wave that feeds it.  A wave issues in order: what
    // else it does in C0 and C1 stands between its matrix instructions, two or three instructions at a time.  With slots counted from
    // the first group's M0 of K-tile t, its own slots are 0 1 2 3, the second group's 1 2 3 4:
    //   dy of K-tile t+1 (its stage was last read in slot -1): first group from its M0 (slot 0), second from its previous C1 (slot 0);
    //     waited for before the end of slot 3 (first group's C1, second group's M1), read from slot 4 on
    //   codes of K-tile t+1: converted and written in C0 (slots 1 and 2), waited for in M1; the codes of K-tile t+2 are loaded then
    // (K-tiles past the end are written into a stage that nothing reads any more).
    // A wave's vector-memory instructions retire in order and every C0 issues four loads behind the dy of its K-tile, so vmcnt(4)
    // waits for dy and leaves the codes in flight.
    auto half = [&](auto second_tag) {
      constexpr bool SECOND = decltype(second_tag)::value;
      constexpr int NB = SECOND ? NF - NFW : NFW;
      G2Frags<1, 4> fa;
      G2Frags<1, NB> fb;
      fa.init(wm * 4, 0, lane);
      fb.init(SECOND ? NFW : 0, BOFF, lane);
      bf16x8 af[4], bf[NB];
      auto dma = [&](__amdgpu_buffer_rsrc_t rs, int t, int i) { la.issue(rs, true, i, smem + (t & 1) * STAGE, wave); };      // piece i
#define W8_SLOT_END() do { __builtin_amdgcn_sched_barrier(0); __builtin_amdgcn_s_barrier(); __builtin_amdgcn_sched_barrier(0); } while (0)
#define W8_READ(KS)                                              \
  fa.template read_range<KS, true, 0, 4, 4>(smem, af);           \
  fb.template read_range<KS, true, 0, NB, NB>(smem, bf);
      if (SECOND) {
        const __amdgpu_buffer_rsrc_t rs = a_rsrc(1);
#pragma unroll
        for (int i = 0; i < PA; ++i) dma(rs, 1, i);
        W8_SLOT_END();
      }
      for (int t = 0; t < nkt; ++t) {
        // M0
        W8_READ(0);
        if (!SECOND) {
          const __amdgpu_buffer_rsrc_t ra = a_rsrc(t + 1);
#pragma unroll
          for (int i = 0; i < PA; ++i) dma(ra, t + 1, i);
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);    // lgkmcnt(0): the fragments (the compiler cannot see those reads)
        W8_SLOT_END();
        // C0; operands swapped: a lane ends up with 4 neighbouring columns of one row
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < 4 * NB; ++x) {
          acc[x & 3][x >> 2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[x >> 2], af[x & 3], acc[x & 3][x >> 2], 0, 0, 0);
          __builtin_amdgcn_sched_barrier(0);
          if (x < 6) b_step((t + 1) & 1, 0, x);
          if (x == 6) b_load(q_rsrc(t + 2), s_rsrc(t + 2), 0);
          if (x >= 7 && x < 13) b_step((t + 1) & 1, 1, x - 7);
          if (x == 13) b_load(q_rsrc(t + 2), s_rsrc(t + 2), 1);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        W8_SLOT_END();
        // M1
        W8_READ(1);
        __builtin_amdgcn_s_waitcnt(SECOND ? 0x0074 : 0xc07f);      // lgkmcnt(0); second group: and dy of K-tile t+1, vmcnt(4)
        W8_SLOT_END();
        // C1
        const __amdgpu_buffer_rsrc_t ra = a_rsrc(t + 2);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < 4 * NB; ++x) {
          acc[x & 3][x >> 2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[x >> 2], af[x & 3], acc[x & 3][x >> 2], 0, 0, 0);
          if (SECOND && (x & 3) == 1 && (x >> 2) < PA) { __builtin_amdgcn_sched_barrier(0); dma(ra, t + 2, x >> 2); __builtin_amdgcn_sched_barrier(0); }
        }
        __builtin_amdgcn_s_setprio(0);
        if (!SECOND) __builtin_amdgcn_s_waitcnt(0x0f74);           // dy of K-tile t+1
        W8_SLOT_END();
        fa.toggle((t & 1) ? -STAGE : STAGE); fb.toggle((t & 1) ? -STAGE : STAGE);
      }
      if (!SECOND) W8_SLOT_END();
#undef W8_SLOT_END
#undef W8_READ
    };
    if (wn == 0) half(std::false_type{}); else half(std::true_type{});
    __builtin_amdgcn_s_waitcnt(0x0070);      // no LDS-DMA (of the K-tile past the end) outlives its part, or the workgroup

    // lane: row lane & 15, columns 4 (lane >> 4) .. + 3 of each 16 x 16 fragment
    const int cl = wn * NFW * 16 + 4 * (lane >> 4), rl = wm * 64 + (lane & 15);
    if ((P.m & 7) && kt0 + nkt == P.kt && P.m <= m0 + BM) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t row = m0 + rl + 16 * i;
        if (row < (P.m & ~(int64_t)7) || row >= P.m) continue;
        const float v = bf16_bits_to_f32(P.dy[(P.k - 1) * P.lddy + row]);
#pragma unroll
        for (int j = 0; j < NFW; ++j) {
          const int64_t col = n0 + cl + 16 * j;
          if (j >= nfw || col >= P.n) continue;
          const int w = *reinterpret_cast<const int*>(P.q + (P.k - 1) * P.ldq + col);
          const float s = v * act8_scale(P.scale[(P.k - 1) * P.lds + (col >> 5)]);       // an exact product, a power of two
          acc[i][j] += f32x4{__builtin_amdgcn_cvt_f32_fp8(w, 0) * s, __builtin_amdgcn_cvt_f32_fp8(w, 1) * s, __builtin_amdgcn_cvt_f32_fp8(w, 2) * s,
                             __builtin_amdgcn_cvt_f32_fp8(w, 3) * s};
        }
      }
    }
    if (slot < 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t row = m0 + rl + 16 * i;
        if (row >= P.m) continue;
        float* o = P.dw + row * P.lddw;
#pragma unroll
        for (int j = 0; j < NFW; ++j) {
          if (j >= nfw) continue;
          const int64_t col = n0 + cl + 16 * j;
          w8_put(P, o + col, acc[i][j], P.n - col);
        }
      }
    } else {
      float* o = P.ws + slot * (BM * NF * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NFW; ++j)          // fragments that hold something of dw
          if (j < nfw && m0 + wm * 64 + 16 * i < P.m && n0 + (wn * NFW + j) * 16 < P.n) *reinterpret_cast<f32x4*>(o + (rl + 16 * i) * (NF * 16) + cl + 16 * j) = acc[i][j];
    }
  }
}

// p[sub] + p[sub + S] + ... of n parts `step` floats apart, eight loads in flight; then over the S neighbouring lanes (sub = 0 .. S - 1)
template <int S>
__device__ __forceinline__ f32x4 w8_sum_parts(const float* p, int n, int64_t step, int sub) {
  f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int i = sub; i < n; i += 8 * S) {
    f32x4 t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u * S < n) t[u] = *reinterpret_cast<const f32x4*>(p + (i + u * S) * step);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i + u * S < n) s += t[u];
  }
#pragma unroll
  for (int o = 1; o < S; o <<= 1)
#pragma unroll
    for (int r = 0; r < 4; ++r) s[r] += __shfl_xor(s[r], o, 64);
  return s;
}
// adds the parts of each tile that was cut, always in the same order: grid (tiles behind the whole ones, quads of a tile * S / 256); S
// neighbouring lanes own 4 neighbouring columns of a row
template <int S>
__global__ __launch_bounds__(256) void act8_wgrad_join_kernel(const Wgrad8Params P, const int width) {
  const int tile = P.whole + blockIdx.x;
  const int at = blockIdx.y * 256 + threadIdx.x, quad = at / S, sub = at % S;
  const int per_row = width / 4;
  const int rl = quad / per_row, cl = (quad - rl * per_row) * 4;
  int tm, tn;
  w8_tile(P, tile, tm, tn);
  const int64_t row = (int64_t)tm * 256 + rl, col = (int64_t)tn * width + cl;
  if (rl >= 256 || row >= P.m || col >= P.n) return;
  const int64_t slot_floats = 256 * (int64_t)width;
  const float* p = P.ws + (int64_t)rl * width + cl;
  f32x4 s;
  if (blockIdx.x < (unsigned)P.cut_tiles) {
    if (P.cut == 1) return;                              // written already
    s = w8_sum_parts<S>(p + w8_cut_slot(P, tile, 0) * slot_floats, P.cut, slot_floats, sub);
  } else {
    const int64_t t0 = (int64_t)(blockIdx.x - P.cut_tiles) * P.kt, t1 = t0 + P.kt;
    const int w0 = (int)(t0 / P.piece), w1 = (int)((t1 + P.piece - 1) / P.piece);
    // the first part may be the second half of its piece
    const f32x4 first = *reinterpret_cast<const f32x4*>(p + w8_piece_slot(P, w0, (int64_t)w0 * P.piece < t0) * slot_floats);
    s = first + w8_sum_parts<S>(p + w8_piece_slot(P, w0 + 1, 0) * slot_floats, w1 - w0 - 1, 2 * slot_floats, sub);
  }
  if (sub == 0) w8_put(P, P.dw + row * P.lddw + col, s, P.n - col);
}

// ---- host
struct Wgrad8Plan { int nf, grid, whole, cut, cut_tiles, piece, pieces; int64_t slots; };
// Many parts and few elements: eight lanes share the parts of an element.  One lane / eight, us: 46082 tokens, 20 x 20 in 128 parts 14.0 /
// 4.0, 200 x 300 9.6 / 6.0, 64 x 1025 7.3 / 5.8, 300 x 300 9.0 / 9.6 (shorter runs of memory to a load), 600 x 600 8.6 / 11.0.
static bool w8_deep(int64_t elements, int64_t cut, int64_t line_depth) { return elements <= 80000 && (cut > 16 || line_depth > 16); }
// The cheapest of the tile widths and cuts, in microseconds of the longest workgroup: K-tiles (measured 1.30 us at 128 columns, 1.38
// at 208, 1.53 at 256), start and end of each part, and the parts' way to the workspace and back over the whole chip
// (256 x 16 nf floats written and read at 5 TB/s) with the join's launch and the depth of its sums.
static Wgrad8Plan w8_plan(int64_t m, int64_t n, int64_t k) {
  const int64_t tm = (m + 255) / 256, kt = (k + G2_BK - 1) / G2_BK;
  Wgrad8Plan best = {};
  double cost = -1;
  const double filled = (double)m / (tm * 256);          // rows of the tiles that are written
  const int cand[3] = {8, 13, 16};
  for (int c = 0; c < 3; ++c) {
    const int nf = cand[c];
    const int64_t tiles = tm * ((n + nf * 16 - 1) / (nf * 16));
    const int64_t whole = tiles / W8_WGS * W8_WGS, left = tiles - whole;
    const int64_t most = left ? (W8_WGS + left - 1) / left : 1;      // more parts than that leave tiles for the line
    for (int64_t cut = 1; cut <= most && (cut == 1 || kt / cut >= 4); cut = cut < 8 || cut + 1 >= most - 1 ? cut + 1 : cut * 2 < most - 1 ? cut * 2 : most - 1) {
      int64_t ct = W8_WGS / cut; if (ct > left) ct = left;
      const int64_t line = (left - ct) * kt;
      int64_t piece = (line + W8_WGS - 1) / W8_WGS;
      if (piece < 4) piece = kt < 4 ? kt : 4;            // <= kt always: a piece lies in two tiles at most
      const int64_t pieces = (line + piece - 1) / piece;
      const int64_t slots = (cut > 1 ? ct * cut : 0) + (line ? pieces + (left - ct) : 0);
      const double kt_us = nf == 8 ? 1.30 : nf == 13 ? 1.38 : 1.53;
      const double longest = (double)(whole / W8_WGS) * (kt * kt_us + 5) + (left ? (kt + cut - 1) / cut * kt_us + 5 : 0) +
                             (line ? piece * kt_us + 5 : 0);
      double depth = line ? (double)kt / piece : (double)cut;
      if (w8_deep(m * n, cut, line ? kt / piece : 0)) depth /= 8;
      const double x = longest + (slots ? 0.0065 * nf * slots * filled + 4 + 0.1 * depth : 0);
      if (cost < 0 || x < cost) {
        cost = x;
        const int64_t busy = whole ? W8_WGS : (ct * cut > pieces ? ct * cut : pieces);
        best = {nf, (int)busy, (int)whole, (int)cut, (int)ct, (int)piece, (int)(line ? pieces : 0), ct * cut + 2 * pieces};
        if (!line) best.slots = cut > 1 ? ct * cut : 0;
      }
    }
  }
  return best;
}
extern "C" int64_t vita_act8_wgrad_ws_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || m > ACT8_MAX_COLS || n > ACT8_MAX_COLS || k > ((int64_t)1 << 31)) return 0;
  const Wgrad8Plan p = w8_plan(m, n, k);
  return p.slots * 256 * p.nf * 16 * 4;
}

template <int NF>
static int w8_launch(const Wgrad8Params& P, int grid, bool join, hipStream_t s) {
  constexpr int lds = 2 * (32768 + 32768);
  static VitaPerDeviceOnce once;
  vita_set_max_lds_once(once, (const void*)act8_wgrad_kernel<NF>, lds);
  hipLaunchKernelGGL(act8_wgrad_kernel<NF>, dim3((unsigned)grid), dim3(G2_THREADS), lds, s, P);
  VITA_CHECK_LAUNCH("vita_act8_wgrad");
  if (join) {
    const unsigned tiles = (unsigned)(P.tiles_m * P.tiles_n - P.whole);
    if (w8_deep(P.m * P.n, P.cut, P.pieces ? P.kt / P.piece : 0))
      hipLaunchKernelGGL(act8_wgrad_join_kernel<8>, dim3(tiles, 32 * NF), dim3(256), 0, s, P, NF * 16);
    else
      hipLaunchKernelGGL(act8_wgrad_join_kernel<1>, dim3(tiles, 4 * NF), dim3(256), 0, s, P, NF * 16);
    VITA_CHECK_LAUNCH("vita_act8_wgrad_join");
  }
  return VITA_OK;
}

extern "C" int vita_act8_wgrad(const void* dy, int64_t lddy, const void* q, int64_t ldq, const void* scale, int64_t lds, float* dw,
                               int64_t lddw, int64_t m, int64_t n, int64_t k, int32_t accumulate, void* ws, int64_t ws_bytes, void* stream) {
  VITA_REQUIRE(m > 0 && n > 0 && k > 0 && n <= ACT8_MAX_COLS && m <= ACT8_MAX_COLS && k <= ((int64_t)1 << 31));
  VITA_REQUIRE(act8_mat_ok(dy, lddy, m, VITA_DT_BF16) && dw && lddw >= n);
  VITA_REQUIRE(act8_codes_ok(q, ldq, scale, lds, n));
  const int64_t need = vita_act8_wgrad_ws_bytes(m, n, k);
  VITA_REQUIRE(need == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= need));
  const Wgrad8Plan plan = w8_plan(m, n, k);
  Wgrad8Params P;
  P.dy = (const uint16_t*)dy; P.q = (const uint8_t*)q; P.scale = (const uint8_t*)scale; P.dw = dw; P.ws = (float*)ws;
  P.lddy = lddy; P.ldq = ldq; P.lds = lds; P.lddw = lddw;
  P.m = m; P.n = n; P.k = k;
  const int64_t tiles_m = (m + 255) / 256, tiles_n = (n + plan.nf * 16 - 1) / (plan.nf * 16), kt = (k + G2_BK - 1) / G2_BK;
  VITA_REQUIRE(tiles_m * tiles_n < ((int64_t)1 << 30));
  P.tiles_m = (int)tiles_m; P.tiles_n = (int)tiles_n; P.kt = (int)kt;
  P.cut_kt = P.kt / plan.cut; P.cut_more = P.kt % plan.cut;
  P.whole = plan.whole; P.cut = plan.cut; P.cut_tiles = plan.cut_tiles; P.piece = plan.piece; P.pieces = plan.pieces;
  P.accumulate = accumulate;
  // 32-bit offsets inside a part's tokens (a part is at most kt K-tiles long, and is read up to 3 K-tiles past its end)
  const int64_t part = ((plan.whole || plan.cut == 1 ? kt : (kt + plan.cut - 1) / plan.cut) + 4) * G2_BK;
  if (part * lddy * 2 >= (int64_t)0x7fffff00ll || part * ldq >= (int64_t)0x7fffff00ll || part * lds >= (int64_t)0x7fffff00ll) {
    vita_set_error("vita_act8_wgrad: 2 GiB or more of dy or of codes in one part of the sum", hipSuccess);
    return VITA_ERR_UNSUPPORTED;
  }
  const bool join = plan.slots > 0;
  switch (plan.nf) {
    case 8: return w8_launch<8>(P, plan.grid, join, (hipStream_t)stream);
    case 13: return w8_launch<13>(P, plan.grid, join, (hipStream_t)stream);
    default: return w8_launch<16>(P, plan.grid, join, (hipStream_t)stream);
  }
}
template __global__ void act8_wgrad_kernel<8>(const Wgrad8Params);
template __global__ void act8_wgrad_kernel<13>(const Wgrad8Params);
template __global__ void act8_wgrad_kernel<16>(const Wgrad8Params);
