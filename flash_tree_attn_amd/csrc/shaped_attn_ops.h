// The gfx950 instructions that the shaped-attention kernel names itself beyond gfx950_ops.h.
#ifndef FTA_SHAPED_ATTN_OPS_H
#define FTA_SHAPED_ATTN_OPS_H
#include "gfx950_ops.h"

namespace fta {
namespace {

// D = A B + C of 32 x 2 by 2 x 32 floats: lane (i, h) supplies A[i][h] and B[h][i], accumulator layout as the
// 32x32x16 products'.
__device__ __forceinline__ f32x16 mma_f32(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }

// Explicit LDS reads with explicit waits, as in gfx950_ops.h.
template <int OFF>
__device__ __forceinline__ float lds_read_b32(uint32_t addr) {
  float v;
  asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "n"(OFF));
  return v;
}
template <int N>
__device__ __forceinline__ void wait_lgkm(float (&v)[4]) {
  asm volatile("s_waitcnt lgkmcnt(%4)" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]) : "n"(N));
}

// A 32-bit value at a wave-uniform address of memory that nothing writes while the kernel runs: a scalar load that
// the compiler tracks by itself.
__device__ __forceinline__ int load_uniform(const int32_t* at) {
  return *(const __attribute__((address_space(4))) int32_t*)(uniform_ptr(reinterpret_cast<const char*>(at)));
}

// The kernel's parameters, read again from where they were passed: what only the edges of a pair need does not stay
// in scalar registers (of which the loop has none to spare) from one use to the next.
template <typename P>
__device__ __forceinline__ const __attribute__((address_space(4))) P* parameters_again(const P&) {
  auto* at = (const __attribute__((address_space(4))) P*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  return at;
}

// Pins a value to this place: arithmetic on it stays behind, where the compiler would otherwise do the cheap first
// operation of one branch ahead of the branch, for the other one in vain.
__device__ __forceinline__ void pin(float& x) { asm volatile("" : "+v"(x)); }

// A wave in its matrix products goes ahead of one in its vector arithmetic, which then runs between the products.
__device__ __forceinline__ void matrix_phase(bool on) {
  if (on) __builtin_amdgcn_s_setprio(1); else __builtin_amdgcn_s_setprio(0);
}

__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

}  // namespace
}  // namespace fta
#endif
