// Host stand-ins for flash_tree_attn_amd/csrc/shaped_attn_ops.h (whose include guard this claims), on top of
// gfx950_ops_host.h. TEST INFRASTRUCTURE ONLY.
#pragma once
#define FTA_SHAPED_ATTN_OPS_H
#include "gfx950_ops_host.h"
#include "step_ops_host.h"

inline uint32_t atomicOr(uint32_t* at, uint32_t v) { return std::atomic_ref<uint32_t>(*at).fetch_or(v); }
inline int __shfl_up(int v, unsigned by, int /*width*/) {
  host_block::Block& b = *host_block::current();
  const unsigned t = threadIdx.x, w = t / 64, lane = t & 63;
  std::memcpy(&b.slot[t], &v, 4);
  b.wave[w]->arrive_and_wait();
  int r;
  std::memcpy(&r, &b.slot[lane >= by ? t - by : t], 4);
  b.wave[w]->arrive_and_wait();
  return r;
}

namespace fta {
namespace {

// v_mfma_f32_32x32x2: D[m][n] = C[m][n] + sum_k A[m][k] B[k][n], k = 0, 1. Lane (i, h) supplies A[i][h] and B[h][i].
inline f32x16 mma_f32(float a, float b, f32x16 c) {
  host_block::WaveExchange& x = host_block::my_exchange();
  const unsigned lane = host_block::lane_id(), i = lane & 31, h = lane >> 5;
  float* mine = reinterpret_cast<float*>(x.bytes[lane]);
  mine[0] = a;
  mine[1] = b;
  host_wave_barrier();
  f32x16 d = c;
  for (int r = 0; r < 16; ++r) {
    const unsigned m = 8 * (r / 4) + 4 * h + r % 4;
    for (unsigned k = 0; k < 2; ++k) d[r] += reinterpret_cast<const float*>(x.bytes[m + 32 * k])[0] * reinterpret_cast<const float*>(x.bytes[i + 32 * k])[1];
  }
  host_wave_barrier();
  return d;
}
template <int OFF>
inline float lds_read_b32(uint32_t addr) {
  return lds_reads::issue<float>(host_block::lds_at(addr + OFF, 4));
}
template <int N>
inline void wait_lgkm(float (&v)[4]) {
  lds_reads::expect_landing(N, 4);
  for (float& x : v) lds_reads::land_into(x);
}
inline int load_uniform(const int32_t* at) { return *reinterpret_cast<const int32_t*>(uniform_ptr(reinterpret_cast<const char*>(at))); }
template <typename P>
inline const P* parameters_again(const P& p) { return &p; }
inline void pin(float&) {}
inline void matrix_phase(bool) {}
inline float fast_rcp(float x) { return 1.f / x; }

}  // namespace
}  // namespace fta
