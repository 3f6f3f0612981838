// What the GEMM kernels share: operand tiles copied from memory to LDS by DMA,
// and the order in which a grid's workgroups take output tiles.
#pragma once

#include "common.hpp"

namespace dlm {

typedef int i32x4 __attribute__((ext_vector_type(4)));
#define DLM_LDS __attribute__((address_space(3)))

// 128-bit raw-buffer descriptor in SGPRs: base, no stride, byte size
// (offsets at or past it read 0).
__device__ __forceinline__ i32x4 dma_rsrc(const void* p, unsigned bytes) {
  const uint64_t a = (uint64_t)p;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff));
  r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
  r[3] = 0x00020000;
  return r;
}

// One wave-wide global -> LDS copy: lane l reads 16 bytes at byte offset voff
// of the buffer and the hardware writes them to LDS at dst + 16 l (dst goes
// through M0).  Issued as inline asm so the compiler neither tracks nor
// drains it: the kernel orders it with explicit vmcnt waits and barriers.
// Nothing else in the kernels that use it uses M0, so clobbering it is safe although the
// compiler warns that it treats M0 as reserved.
__device__ __forceinline__ void dma16(const i32x4& r, const unsigned char DLM_LDS* dst, int voff, int soff) {
  const unsigned lds = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)dst);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds),
               "v"(voff), "s"(r), "s"(soff)
               : "memory", "m0");
}

// s_waitcnt vmcnt(n), other counters untouched (gfx9 encoding: vmcnt in bits
// [3:0] and [15:14], expcnt [6:4], lgkmcnt [11:8]).
#define DLM_WAIT_VM(n) \
  __builtin_amdgcn_s_waitcnt((((n)&15) | (((n) >> 4) << 14)) | (0x7 << 4) | (0xF << 8))

// Lane -> (row, chunk) map of DMA instruction i of wave w (NW waves): row
// group g = i*NW + w of 8 rows x 128 B; lane l covers row 8g + l/8, physical
// chunk l%8, which holds the logical K chunk (l%8) ^ ((row >> 1) & 7).  A
// tile whose row-group count is not a multiple of NW leaves the last
// instruction to the first (groups % NW) waves.
__device__ __forceinline__ int dma_row(int nw, int i, int wave, int lane) {
  return (i * nw + wave) * 8 + (lane >> 3);
}
__device__ __forceinline__ int dma_chunk(int row, int lane) { return (lane & 7) ^ ((row >> 1) & 7); }

// ---------------------------------------------------------------------------
// Tile scheduling: spread consecutive logical tiles over one XCD (the
// hardware deals workgroup i to XCD i % 8, each XCD has its own L2), then
// walk logical tiles in groups of 8 M-tiles so co-resident tiles share both
// operand panels.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void tile_coords(int bid, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int total = tiles_m * tiles_n;
  const int q = total >> 3, r = total & 7;
  const int x = bid & 7, slot = bid >> 3;
  const int logical = x * q + (x < r ? x : r) + slot;
  constexpr int GM = 8;
  const int per_group = GM * tiles_n;
  const int g = logical / per_group;
  const int first_m = g * GM;
  const int gsz = min(tiles_m - first_m, GM);
  const int rem = logical - g * per_group;
  tm = first_m + rem % gsz;
  tn = rem / gsz;
}

}  // namespace dlm
