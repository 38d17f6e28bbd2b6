// lds_dma.hpp -- 16-bit tiles from memory to LDS without a detour through registers, and the two
// ways the matrix instructions read them (cross_attention.hip, linear.hip).
//
// A DMA instruction (buffer load with the lds flag) fills 64 consecutive 16-byte units of LDS, one
// per lane, from the lanes' own addresses, so the rows of a tile cannot be padded apart.  Instead
// unit u of row r lies at u ^ swz(r), chosen so that neither way of reading meets a bank twice in a
// cycle (256 bytes): 16 rows at one unit fall on 16 different units of the 64 banks, and so do the
// four rows x 64 bytes that 32 lanes of a transpose read touch.  An offset of kFar is beyond the
// descriptor's bound: that lane's unit is filled with zeros.
#pragma once
#include "decoder_ops.hpp"

namespace btr {

typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t *lds_s16x4;
constexpr int kFar = 0x7ffffff0;

// tile of rows of D elements
template <int D>
struct Dma {
  static constexpr int UNITS = D / 8, PITCH = D * 2;
  static_assert(D == 32 || D == 64 || D == 128, "a row is a power of two of units");
  __device__ static __forceinline__ int swz(int row) {   // (D = 32: row reads only)
    return (D == 128 ? (row & 3) << 2 : D == 64 ? (row & 2) << 1 : 0) | ((row >> 2) & 3);
  }
  // fragment j of tile row l31 (+ 32 per subtile as an immediate): base ^ (j << 5)
  __device__ static __forceinline__ int row_base(int l31, int hh) {
    return l31 * PITCH + ((hh ^ swz(l31)) << 4);
  }
  // transpose read of columns 32 nt .. + 31: base ^ (nt << 6); the eight rows further on: one bit of
  // the swizzle flips, + 8 rows
  __device__ static __forceinline__ int tr_base(int lane) {
    const int p = lane & 15, half = (lane >> 4) & 1, hh = lane >> 5, row = 4 * hh + (p >> 2);
    return row * PITCH + (((2 * half + ((p & 3) >> 1)) ^ swz(row)) << 4) + (p & 1) * 8;
  }
  static constexpr int kTrHi = 32;
  // the same in natural order of the reduction: rows 8 hh .. + 3, and with ^ kNatHi rows four on
  __device__ static __forceinline__ int nat_base(int lane) {
    const int p = lane & 15, half = (lane >> 4) & 1, hh = lane >> 5, row = 8 * hh + (p >> 2);
    return row * PITCH + (((2 * half + ((p & 3) >> 1)) ^ swz(row)) << 4) + (p & 1) * 8;
  }
  static constexpr int kNatHi = 16;
};

__device__ __forceinline__ i32x4_t dma_rsrc(const char *base, int bytes) {
  // raw buffer descriptor: 48-bit base, bytes, 32-bit data
  const unsigned long long at = (unsigned long long)base;
  return i32x4_t{__builtin_amdgcn_readfirstlane((int)at),
                 __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff),
                 __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
// 64 lanes x 16 (4) bytes at their offsets -> 64 consecutive units from lds (the same in all lanes).
// In assembly: the compiler would wait for every DMA in flight before any transpose read; the
// kernels wait for a tile themselves, dma_wait, before the barrier in front of its first read.  (It
// does not see the instruction either: five wait states between a VALU write of a scalar register --
// readfirstlane -- and a vector memory instruction that reads it are the assembly's to keep.)
__device__ __forceinline__ unsigned lds_at(const char *lds) {
  return __builtin_amdgcn_readfirstlane(
      (unsigned)(unsigned long long)(__attribute__((address_space(3))) const char *)lds);
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // (m0 is reserved: it warns, and honours it)
__device__ __forceinline__ void dma16(i32x4_t rsrc, int off, const char *lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds_at(lds)), "v"(off), "s"(rsrc)
               : "memory", "m0");
}
__device__ __forceinline__ void dma4(i32x4_t rsrc, int off, const char *lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :
               : "s"(lds_at(lds)), "v"(off), "s"(rsrc)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// The DMA instructions are the compiler's to count only through this: what it has loaded itself must
// have arrived before the first of them, or it waits for everything in flight at the first use.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }   // vmcnt(0)
template <int LEFT = 0>   // all but the newest LEFT of this wave's instructions have arrived
__device__ __forceinline__ void dma_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}

}  // namespace btr
