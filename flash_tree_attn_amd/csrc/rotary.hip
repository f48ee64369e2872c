// Rotary positions (fta_rotary, include/fta.h): the rows of q and k that enter a tree-attention call are
// turned in pairs by pos * inv_freq, pos = positions[b, i] (+ kv_seq_len[b]).
//
// One pass over the rows: a thread owns one unit of a row (half layout: 16 bytes of first and 16 bytes of
// second pair members; interleaved: 16 bytes of whole pairs), takes the sines of its pairs once and walks over
// `heads_per_thread` heads with them, so that the 64-bit angles and the sines (about 60 instructions a pair)
// are shared between heads. Units behind rotary_dim copy. Rotary dims that do not fill 16-byte units take one
// pair per thread. What bounds it: every row read and written once (336 MB in 73 us, 4.6 TB/s of a copy's 5.1; 66 us
// where the inputs' 168 MB are still in the memory-side cache); calls of a few rows are launch-bound (3.3 us). Pair by
// pair, in accesses of 2 or 4 bytes, rotary dims of 22 or 40 take 113 to 124 us for the same rows in 16 bits.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "fta_device.h"

namespace fta {
namespace {

struct RotaryParams {
  const char* in[2];          // q, k
  char* out[2];
  const void* positions;
  const void* lens;
  const void* freq;
  int32_t heads[2], chunks[2];   // chunks: groups of heads_per_thread heads
  int32_t heads_per_thread;
  int32_t q_len, half, rotary_dim;   // half = pairs per head
  int32_t units, turning;     // units per row; the first `turning` of them hold pairs
  int32_t copy_second;        // bytes between the two accesses of a copying unit; -1: copying units are single accesses apart
  int32_t pos_is_i64, len_is_i64, freq_is_f64, inverse;
  float factor;
  int64_t items;              // bsz * q_len * units
  int64_t in_stride[2][3], out_stride[2][3];   // bytes
  int64_t pos_stride[2];
};

// Cosine and sine of pos * freq, times the factor. The angle is formed and reduced in 64 bits, in half turns,
// where the reduction is exact: 32 bits would be 0.06 radians off at position 10^6. The sine runs in 32 bits.
__device__ __forceinline__ void turn_of(const RotaryParams& p, double pos, int pair, float* c, float* s) {
  const double f = p.freq_is_f64 ? static_cast<const double*>(p.freq)[pair] : static_cast<double>(static_cast<const float*>(p.freq)[pair]);
  constexpr double kHalfTurnsPerRadian = 0.31830988618379067153776752674503;   // 1 / pi
  double t = pos * f * kHalfTurnsPerRadian;
  t -= 2.0 * rint(0.5 * t);
  float sn, cs;
  sincospif(static_cast<float>(t), &sn, &cs);
  *c = cs * p.factor;
  *s = (p.inverse ? -sn : sn) * p.factor;
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Unit {
  T v[N];
};

template <bool PAST_L2, typename U>
__device__ __forceinline__ void store(char* at, const U& u) {
  if constexpr (PAST_L2) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, u), reinterpret_cast<u32x4*>(at));
  else *reinterpret_cast<U*>(at) = u;
}

constexpr int kHalves = 0, kInterleaved = 1, kHalvesByPair = 2, kInterleavedByPair = 3;

// PAST_L2: results do not go into the L2.
template <typename T, int LAYOUT, bool PAST_L2 = false>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryParams p) {
  constexpr bool kWide = LAYOUT < kHalvesByPair;
  constexpr int kVec = kWide ? 16 / static_cast<int>(sizeof(T)) : LAYOUT == kInterleavedByPair ? 2 : 1;   // values per access
  constexpr bool kTwo = LAYOUT == kHalves || LAYOUT == kHalvesByPair;   // a unit is two accesses, one per pair member
  constexpr int kPairs = kTwo ? kVec : kVec / 2;
  constexpr int kGroup = 4;   // heads whose loads are in flight together
  using U = Unit<T, kVec>;
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  // consecutive threads: the units of a row, then the rows, then the groups of heads
  const int64_t chunk64 = gid / p.items;
  if (chunk64 >= p.chunks[0] + p.chunks[1]) return;
  const int chunk = static_cast<int>(chunk64);
  const int64_t item = gid - chunk64 * p.items;
  const int64_t row = item / p.units;
  const int unit = static_cast<int>(item - row * p.units);
  const int b = static_cast<int>(row / p.q_len), i = static_cast<int>(row - static_cast<int64_t>(b) * p.q_len);
  const int is_k = chunk >= p.chunks[0];
  const int head0 = (chunk - (is_k ? p.chunks[0] : 0)) * p.heads_per_thread;
  const int head1 = min(head0 + p.heads_per_thread, p.heads[is_k]);
  const char* in = p.in[is_k] + b * p.in_stride[is_k][0] + i * p.in_stride[is_k][2];
  char* out = p.out[is_k] + b * p.out_stride[is_k][0] + i * p.out_stride[is_k][2];
  const int64_t in_head = p.in_stride[is_k][1], out_head = p.out_stride[is_k][1];

  const bool turns = unit < p.turning;
  if (!turns && p.copy_second < 0) {   // behind rotary_dim: copied, unless it is there already
    if (in == out) return;
    const int64_t at = static_cast<int64_t>(sizeof(T)) * (p.rotary_dim + (unit - p.turning) * kVec);
    for (int h = head0; h < head1; h += kGroup) {
      U x[kGroup];
#pragma unroll
      for (int g = 0; g < kGroup; ++g)
        if (h + g < head1) x[g] = *reinterpret_cast<const U*>(in + (h + g) * in_head + at);
#pragma unroll
      for (int g = 0; g < kGroup; ++g)
        if (h + g < head1) *reinterpret_cast<U*>(out + (h + g) * out_head + at) = x[g];
    }
    return;
  }

  const int64_t where = b * p.pos_stride[0] + i * p.pos_stride[1];
  int64_t pos = p.pos_is_i64 ? static_cast<const int64_t*>(p.positions)[where] : static_cast<const int32_t*>(p.positions)[where];
  if (p.lens) pos += load_len(p.lens, p.len_is_i64, b);
  float c[kPairs], s[kPairs];
#pragma unroll
  for (int e = 0; e < kPairs; ++e) turn_of(p, static_cast<double>(pos), min(unit, p.turning - 1) * kPairs + e, &c[e], &s[e]);

  const int64_t at = static_cast<int64_t>(sizeof(T)) * (turns ? unit * kVec : p.rotary_dim + (unit - p.turning) * kVec);
  const int64_t second = turns ? static_cast<int64_t>(sizeof(T)) * p.half : p.copy_second;
  for (int h = head0; h < head1; h += kGroup) {
    U x[kGroup], y[kGroup];
#pragma unroll
    for (int g = 0; g < kGroup; ++g) {
      if (h + g >= head1) continue;
      const char* src = in + (h + g) * in_head + at;
      x[g] = *reinterpret_cast<const U*>(src);
      if constexpr (kTwo) y[g] = *reinterpret_cast<const U*>(src + second);
    }
#pragma unroll
    for (int g = 0; g < kGroup; ++g) {
      if (h + g >= head1) continue;
      U u, v;
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        const float a = to_f32(x[g].v[kTwo ? e : 2 * e]), bb = to_f32(kTwo ? y[g].v[e] : x[g].v[2 * e + 1]);
        const float first = a * c[e] - bb * s[e], other = bb * c[e] + a * s[e];   // one rounding to T each, below
        if constexpr (kTwo) {
          u.v[e] = static_cast<T>(first);
          v.v[e] = static_cast<T>(other);
        } else {
          u.v[2 * e] = static_cast<T>(first);
          u.v[2 * e + 1] = static_cast<T>(other);
        }
      }
      if (!turns) {   // behind rotary_dim: as they are, also where they are not numbers
        u = x[g];
        v = y[g];
      }
      char* dst = out + (h + g) * out_head + at;
      store<PAST_L2>(dst, u);
      if constexpr (kTwo) store<PAST_L2>(dst + second, v);
    }
  }
}

int validate(const fta_rotary_args& a) {
  if (!a.q || !a.out_q || !a.positions || !a.inv_freq) return FTA_ERR_NULL_POINTER;
  if ((a.k == nullptr) != (a.out_k == nullptr)) return FTA_ERR_NULL_POINTER;
  if (a.dtype != FTA_F32 && a.dtype != FTA_F16 && a.dtype != FTA_BF16) return FTA_ERR_DTYPE;
  if ((a.pos_dtype != FTA_I32 && a.pos_dtype != FTA_I64) || (a.len_dtype != FTA_I32 && a.len_dtype != FTA_I64)) return FTA_ERR_DTYPE;
  if (a.head_dim != 32 && a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return FTA_ERR_HEAD_DIM;
  if (a.bsz <= 0 || a.num_q_heads <= 0 || a.q_len <= 0 || a.rotary_dim < 2 || a.rotary_dim > a.head_dim || a.rotary_dim % 2) return FTA_ERR_SHAPE;
  if (a.k ? a.num_kv_heads <= 0 : a.num_kv_heads != 0) return FTA_ERR_SHAPE;
  if (!std::isfinite(a.attention_factor)) return FTA_ERR_UNSUPPORTED;   // (also a double that left 32 bits on its way here)
  const int vec = a.dtype == FTA_F32 ? 4 : 8;
  const int64_t* strides[] = {a.q_stride, a.out_q_stride, a.k_stride, a.out_k_stride};
  const void* ptrs[] = {a.q, a.out_q, a.k, a.out_k};
  for (int t = 0; t < (a.k ? 4 : 2); ++t) {
    for (int d = 0; d < 3; ++d)
      if (strides[t][d] < 0 || strides[t][d] % vec) return FTA_ERR_STRIDE;
    if (reinterpret_cast<uintptr_t>(ptrs[t]) % 16) return FTA_ERR_STRIDE;
  }
  if (a.pos_stride[0] < 0 || a.pos_stride[1] < 0) return FTA_ERR_STRIDE;
  if (reinterpret_cast<uintptr_t>(a.inv_freq) % (a.freq_is_f64 ? 8 : 4)) return FTA_ERR_STRIDE;
  return FTA_OK;
}

template <typename T>
int launch(const RotaryParams& p, int layout, bool past_l2, int64_t grid, hipStream_t stream) {
  const dim3 g(static_cast<unsigned>(grid)), block(256);
  switch (layout) {
    case kHalves:
      if (past_l2) return launch_checked(rotary_kernel<T, kHalves, true>, g, block, 0, stream, p);
      return launch_checked(rotary_kernel<T, kHalves>, g, block, 0, stream, p);
    case kInterleaved:
      if (past_l2) return launch_checked(rotary_kernel<T, kInterleaved, true>, g, block, 0, stream, p);
      return launch_checked(rotary_kernel<T, kInterleaved>, g, block, 0, stream, p);
    case kHalvesByPair: return launch_checked(rotary_kernel<T, kHalvesByPair>, g, block, 0, stream, p);
    default: return launch_checked(rotary_kernel<T, kInterleavedByPair>, g, block, 0, stream, p);
  }
}

}  // namespace
}  // namespace fta

extern "C" int fta_rotary(const fta_rotary_args* args, void* hip_stream) {
  using namespace fta;
  if (!args) return FTA_ERR_NULL_POINTER;
  const fta_rotary_args& a = *args;
  if (int st = validate(a)) return st;
  const int es = a.dtype == FTA_F32 ? 4 : 2, vec = 16 / es;

  RotaryParams p{};
  p.in[0] = static_cast<const char*>(a.q);
  p.in[1] = static_cast<const char*>(a.k);
  p.out[0] = static_cast<char*>(a.out_q);
  p.out[1] = static_cast<char*>(a.out_k);
  p.positions = a.positions;
  p.lens = a.kv_seq_len;
  p.freq = a.inv_freq;
  p.heads[0] = a.num_q_heads;
  p.heads[1] = a.num_kv_heads;
  p.q_len = a.q_len;
  p.half = a.rotary_dim / 2;
  p.rotary_dim = a.rotary_dim;
  p.pos_is_i64 = a.pos_dtype == FTA_I64;
  p.len_is_i64 = a.len_dtype == FTA_I64;
  p.freq_is_f64 = a.freq_is_f64 != 0;
  p.inverse = a.inverse != 0;
  p.factor = a.attention_factor;
  for (int d = 0; d < 3; ++d) {
    p.in_stride[0][d] = a.q_stride[d] * es;
    p.out_stride[0][d] = a.out_q_stride[d] * es;
    p.in_stride[1][d] = a.k_stride[d] * es;
    p.out_stride[1][d] = a.out_k_stride[d] * es;
  }
  p.pos_stride[0] = a.pos_stride[0];
  p.pos_stride[1] = a.pos_stride[1];

  // 16-byte units where the halves (or the interleaved part) are whole units, else one pair per thread
  const bool wide = a.interleaved ? a.rotary_dim % vec == 0 : p.half % vec == 0;
  const int layout = a.interleaved ? (wide ? kInterleaved : kInterleavedByPair) : (wide ? kHalves : kHalvesByPair);
  const int access = wide ? vec : a.interleaved ? 2 : 1;           // values per access
  p.turning = p.half / (a.interleaved ? access / 2 : access);
  p.units = p.turning + (a.head_dim - a.rotary_dim) / access;
  p.copy_second = -1;
  if (wide) {
    // copying units of the turning ones' form: no lane of a wave waits while the others copy. (head_dim and a wide
    // rotary_dim are both whole numbers of units.)
    if (!a.interleaved) p.units = p.turning + (a.head_dim - a.rotary_dim) / (2 * vec);
    p.copy_second = (a.head_dim - a.rotary_dim) / 2 * es;
  }
  p.items = static_cast<int64_t>(a.bsz) * a.q_len * p.units;
  // Heads that share one thread's sines: as many as leave 2^18 threads (256 CUs x 1024), so that large calls
  // take the sines rarely and small ones spread over the machine.
  p.heads_per_thread = 1;
  while (p.heads_per_thread < 16 && p.items * (a.num_q_heads + a.num_kv_heads) >= (int64_t{1} << 18) * 2 * p.heads_per_thread) p.heads_per_thread *= 2;
  for (int t = 0; t < 2; ++t) p.chunks[t] = (p.heads[t] + p.heads_per_thread - 1) / p.heads_per_thread;

  // Results that the L2s (32 MiB) cannot hold until they are read would only push the inputs out: 84 us became 78 by the
  // alike units and 66 by these stores for 8 x 2048 rows, 32 + 8 heads of 128 values, one set of inputs again and again (its
  // 168 MB stay in the memory-side cache; from sets in turn 73).
  const bool past_l2 = static_cast<int64_t>(a.bsz) * a.q_len * (a.num_q_heads + a.num_kv_heads) * a.head_dim * es > (int64_t{32} << 20);

  const int64_t threads = p.items * (p.chunks[0] + p.chunks[1]);
  const int64_t grid = (threads + 255) / 256;
  if (grid > 0x7fffffffLL) return FTA_ERR_SHAPE;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return FTA_ERR_NO_DEVICE;
  hipStream_t stream = static_cast<hipStream_t>(hip_stream);
  if (a.dtype == FTA_F32) return launch<float>(p, layout, past_l2, grid, stream);
  if (a.dtype == FTA_F16) return launch<_Float16>(p, layout, past_l2, grid, stream);
  return launch<__bf16>(p, layout, past_l2, grid, stream);
}
