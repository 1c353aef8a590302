// Building blocks of the 256-row matrix kernels (gemm256.hip, act8_wgrad.hip): the LDS-DMA loader of an operand's K-tile, the
// readers of its fragments and the barrier between K-tiles.  The LDS images are described in gemm256.hip.
#pragma once
#include "common.h"

#ifndef G2_DBG
#define G2_DBG 0
#endif
#define G2_BM 256
#define G2_BK 64
#define G2_STAGE 65536
#define G2_BOFF 32768
#define G2_THREADS 512
#define G2_OOB 0x7ffffff0u

typedef __attribute__((address_space(3))) void lds_void_t;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t g2_rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
__device__ __forceinline__ uint32_t g2_f(int r) { return (r & 3) | (((r >> 3) & 1) << 2); }

// ---- LDS-DMA loader of one operand's K-tile image -------------------------------------------------
// FREE = free extent of the tile (256 for A, NF*16 for B).  Every wave issues PPW = 4 pieces of 1 KiB per
// K-tile; pieces past the image write zeros into the unused tail of the 32 KiB region.
__device__ __forceinline__ uint32_t g2_sgpr(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

template <int LAYOUT, int FREE, int NWAVE = 8>
struct G2Loader {
  static constexpr int NPIECE = LAYOUT == 0 ? FREE / 8 : 32;
  static constexpr int PPW = (NPIECE + NWAVE - 1) / NWAVE;     // 4 with 8 waves; the region holds PPW * NWAVE KiB
  static constexpr int BYTES = PPW * NWAVE * 1024;
  uint32_t voff[PPW];
  uint32_t base_lo, base_hi, bytes, kstep;   // wave-uniform (SGPRs)
  int kchunk;   // LAYOUT 0: k element offset of this lane's 16-B chunk inside a K-tile
  int K;

  __device__ __forceinline__ void init(const uint16_t* op, int64_t free0, int64_t nfree, int64_t Ktot, int64_t ld,
                                       int wave, int lane) {
    K = (int)Ktot;
    uint64_t bp;
    if (LAYOUT == 0) {
      int64_t rows = nfree - free0; if (rows > FREE) rows = FREE;
      bp = (uint64_t)(op + free0 * ld);
      bytes = g2_sgpr((uint32_t)(rows * ld * 2));
      kstep = G2_BK * 2;
      const int clog = (lane & 7) ^ (lane >> 3);
      kchunk = clog * 8;
#pragma unroll
      for (int i = 0; i < PPW; ++i) {
        const int p = wave + NWAVE * i;
        const int row = p * 8 + (lane >> 3);
        voff[i] = p < NPIECE ? (uint32_t)(row * ld * 2 + clog * 16) : G2_OOB;
      }
    } else {
      int64_t nfree8 = (nfree + 7) & ~(int64_t)7; if (nfree8 > ld) nfree8 = ld;
      bp = (uint64_t)(op + free0);
      bytes = g2_sgpr((uint32_t)(((Ktot - 1) * ld + (nfree8 - free0)) * 2));
      kstep = g2_sgpr((uint32_t)(G2_BK * ld * 2));
      kchunk = 0;
#pragma unroll
      for (int i = 0; i < PPW; ++i) {
        const int p = wave + NWAVE * i;
        const int krow = 2 * p + (lane >> 5);
        const int pc = (lane & 31) >> 1, half = lane & 1;
        const int lc = pc ^ (int)g2_f(krow);
        const int col = lc * 16 + half * 8;
        const bool ok = col < FREE && free0 + col < nfree8;
        voff[i] = ok ? (uint32_t)((int64_t)krow * ld * 2 + col * 2) : G2_OOB;
      }
    }
    base_lo = g2_sgpr((uint32_t)bp); base_hi = g2_sgpr((uint32_t)(bp >> 32));
  }
  // resource descriptor of K-tile kt (absolute index): base advanced, extent shrunk, all in SGPRs
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(int kt) const {
    const uint32_t adv = g2_sgpr((uint32_t)kt * kstep);
    const uint64_t bp = (((uint64_t)base_hi << 32) | base_lo) + adv;
    const uint32_t rem = g2_sgpr(adv < bytes ? bytes - adv : 0u);
    return g2_rsrc((const void*)bp, rem);
  }
  __device__ __forceinline__ bool keep(int kt) const { return LAYOUT != 0 || (kt * G2_BK + kchunk < K); }
  // piece i (0..3) of this wave; img = LDS address of this operand's 32 KiB region in the target stage
  __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t rs, bool kp, int i, char* img, int wave, bool in_loop = false) const {
    if ((G2_DBG & 8) && in_loop) return;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(img + (wave + NWAVE * i) * 1024), 16, kp ? voff[i] : G2_OOB, 0, 0, 0);
  }
};

// ---- fragment readers -------------------------------------------------------------------------------
// NFR fragments (16 free indices each) starting at tile-local fragment index f_first.
template <int LAYOUT, int NFR>
struct G2Frags {
  // LAYOUT 0: b[ks] ; LAYOUT 1: b[j]
  uint32_t b[LAYOUT == 0 ? 2 : NFR];
  __device__ __forceinline__ void init(int f_first, uint32_t img_off, int lane) {
    if (LAYOUT == 0) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        b[ks] = img_off + (f_first * 16 + (lane & 15)) * 128 + ((((ks * 4 + (lane >> 4)) ^ (lane & 7))) << 4);
    } else {
      const int g = lane >> 4, t = lane & 15, q = t >> 2, p = t & 3;
      const int fl = q | ((g & 1) << 2);
#pragma unroll
      for (int j = 0; j < NFR; ++j) {
        const int fi = f_first + j;
        b[j] = img_off + (8 * g + q) * 512 + ((fi ^ fl) << 5) + p * 8;
      }
    }
  }
  // delta = +stage bytes when moving from stage 0 to stage 1, -stage bytes back
  __device__ __forceinline__ void toggle(int delta) {
#pragma unroll
    for (int j = 0; j < (LAYOUT == 0 ? 2 : NFR); ++j) b[j] += delta;
  }
  // ASM: issue the LDS reads as inline asm.  hipcc puts s_waitcnt vmcnt(0) in front of every
  // ds_read_b64_tr_b16 builtin while an LDS-DMA is in flight (it cannot tell the DMA's LDS write from the
  // read), which would serialise the pipeline; the asm form is invisible to that pass, so kernels that use
  // it wait for their fragments with an explicit lgkmcnt(0) before the MFMAs that consume them.
  template <int KS, bool ASM, int J>
  __device__ __forceinline__ bf16x8 read(const char* smem) const {
    typedef int v2i __attribute__((ext_vector_type(2)));
    typedef int v4i __attribute__((ext_vector_type(4)));
    if constexpr (LAYOUT == 0) {
      if constexpr (!ASM) {
        return *reinterpret_cast<const bf16x8*>(smem + b[KS] + J * 2048);
      } else {
        v4i v;
        asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v) : "v"(b[KS]), "n"(J * 2048) : "memory");
        return __builtin_bit_cast(bf16x8, v);
      }
    } else {
      v2i lo, hi;
      asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(lo) : "v"(b[J]), "n"(KS * 16384) : "memory");
      asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(hi) : "v"(b[J]), "n"(KS * 16384 + 2048) : "memory");
      v4i v = {lo[0], lo[1], hi[0], hi[1]};
      return __builtin_bit_cast(bf16x8, v);
    }
  }
  // fragments [LO, HI) of k-step KS into dst
  template <int KS, bool ASM, int LO, int HI, int N>
  __device__ __forceinline__ void read_range(const char* smem, bf16x8 (&dst)[N]) const {
    if constexpr (LO < HI && LO < N) {
      dst[LO] = read<KS, ASM, LO>(smem);
      read_range<KS, ASM, LO + 1, HI, N>(smem, dst);
    }
  }
};

// s_waitcnt vmcnt(0) lgkmcnt(0) as a builtin (the compiler's own counters stay in step), then a raw
// barrier: a __syncthreads() would be the same here, but this keeps the intent explicit
__device__ __forceinline__ void g2_sync_all() {
  __builtin_amdgcn_s_waitcnt(0x0070);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);   // nothing (e.g. a register-only MFMA fed by asm reads) moves above the wait
}
