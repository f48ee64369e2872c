// Log probabilities, entropy and the largest alternatives from rows of logits (fta_logprobs, include/fta.h).
//
// One read of the logits: a workgroup takes a row, or a chunk of one, into registers as it comes from memory
// (16-byte loads, all in flight together) and works on the registers from there:
//     m = max x,  l = sum e,  t = sum e d   with d = (x - m) / T log2(e), e = 2^d
//     lse = m / T + ln l,  entropy = ln l - ln2 t / l
// (d is relative to the row's maximum, so nothing cancels), and for the alternatives a threshold: of the maxima
// of 64 (or 256) groups of threads the k-th largest is a lower bound of the k-th largest logit, since k different
// logits reach it. What reaches the threshold (about k + k / 4 logits of random rows) goes to LDS as
// (order-preserving key of the value, ~index) and is ranked by counting: equal values by ascending index, the
// same result whatever order the candidates arrive in. Rows with more candidates than LDS slots (many equal
// logits) extract the k largest one by one instead.
// Rows cut into chunks leave (m, l, t, k keys) per chunk in the workspace and a second launch joins them.
//
// What bounds it: the read of the logits, with about 35 vector instructions per 64 logits next to it: 512 rows of 131072
// take 42 us in bf16 (3.2 TB/s; 32 us without alternatives, 4.2 TB/s) and 54 us in fp32 (4.9 TB/s), the large copy's rate
// being 5.1. Rows that one workgroup does not hold are two launches: 5.1 + 4.3 us for one of 32000 fp32, 9.3 + 4.6 for 104
// of 50001 fp16.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "fta_device.h"

namespace fta {
namespace {

constexpr int kMaxTop = 128;
constexpr int kThreads = 512;   // of a workgroup of the first launch

// Ends what the compiler knows of a register's value: without it, it converts all logits to 32 bits once and keeps
// the results from phase to phase, twice the registers of the 16-bit values and far more than there are.
#ifndef FTA_FORGET
#define FTA_FORGET(x) asm volatile("" : "+v"(x))
#endif

struct LogprobParams {
  const void* logits;
  const void* ids;
  float* logprobs;
  float* entropy;
  float* lse;
  float* top_logprobs;
  int64_t* top_ids;
  char* workspace;
  int64_t rows, logits_stride, id_stride[2];
  int32_t vocab, num_ids, top_k, id_is_i64, chunks;
  float inv_temp;
};

template <typename T> constexpr bool kIsF16 = false;
template <> constexpr bool kIsF16<_Float16> = true;

struct ChunkStats {
  float m, l, t, unused;
};
// Workspace of one chunk: its statistics, then top_k keys.
__host__ __device__ inline int64_t chunk_bytes(int top_k) { return static_cast<int64_t>(sizeof(ChunkStats)) + 8 * ((top_k + 1) / 2 * 2); }

// Order-preserving map of a float to 32 bits: NaN 1, -inf above it, -0 = +0. 0 stands for "no logit".
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 1;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);   // -0 + 0 = +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key <= 1) return __builtin_nanf("");
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ uint64_t entry_of(float x, int index) {
  return static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ int index_of(uint64_t entry) { return static_cast<int>(~static_cast<uint32_t>(entry)); }

__device__ __forceinline__ float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }   // NaN if either is

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t hi = __shfl_xor(static_cast<uint32_t>(x >> 32), o, 64), lo = __shfl_xor(static_cast<uint32_t>(x), o, 64);
    const uint64_t y = static_cast<uint64_t>(hi) << 32 | lo;
    x = x > y ? x : y;
  }
  return x;
}

// The logit of the row's token j: requested at the start of a kernel, so that the two round trips (the id, then its
// logit) pass under everything else. -inf outside the vocabulary.
template <typename T>
__device__ __forceinline__ float logit_of_id(const LogprobParams& p, int64_t row, int j) {
  const int64_t at = row * p.id_stride[0] + j * p.id_stride[1];
  const int64_t id = p.id_is_i64 ? static_cast<const int64_t*>(p.ids)[at] : static_cast<int64_t>(static_cast<const int32_t*>(p.ids)[at]);
  return id >= 0 && id < p.vocab ? to_f32(static_cast<const T*>(p.logits)[row * p.logits_stride + id]) : neg_inf();
}

// Results of one row, by all threads of the block: statistics (m, l, t), the logit of token threadIdx.x, and the k
// largest entries in `top` (LDS, descending; 0 where the row has none left).
template <typename T>
__device__ __forceinline__ void write_row(const LogprobParams& p, int64_t row, float m, float l, float t, float token_logit, const uint64_t* top) {
  const bool empty = l == 0.f;                      // every logit is -inf
  const float log_l = empty ? 0.f : logf(l);
  auto logprob = [&](float x) { return empty ? neg_inf() : (x - m) * p.inv_temp - log_l; };
  if (threadIdx.x == 0) {
    p.lse[row] = empty ? neg_inf() : m * p.inv_temp + log_l;
    p.entropy[row] = empty ? 0.f : log_l - kLn2 * (t / l);
  }
  for (int j = threadIdx.x; j < p.num_ids; j += blockDim.x)
    p.logprobs[row * p.num_ids + j] = logprob(j < static_cast<int>(blockDim.x) ? token_logit : logit_of_id<T>(p, row, j));
  for (int j = threadIdx.x; j < p.top_k; j += blockDim.x) {
    p.top_logprobs[row * p.top_k + j] = logprob(value_of(static_cast<uint32_t>(top[j] >> 32)));
    p.top_ids[row * p.top_k + j] = index_of(top[j]);
  }
}

// How many of the first n entries are larger than `mine`. LDS answers after about 100 cycles, so four are read at a
// time (more cost registers, and with them resident workgroups); `entry` holds a multiple of 4.
__device__ __forceinline__ int larger(const uint64_t* entry, int n, uint64_t mine) {
  int rank = 0;
#pragma unroll 1
  for (int j0 = 0; j0 < n; j0 += 4) {
    uint64_t other[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) other[j] = entry[j0 + j];
#pragma unroll
    for (int j = 0; j < 4; ++j) rank += (j0 + j < n) & (other[j] > mine);
  }
  return rank;
}

// Ranks the n entries in `entry` (all different) and leaves the k largest in `top`, descending, 0 behind them.
__device__ __forceinline__ void rank_entries(const uint64_t* entry, int n, int k, uint64_t* top) {
  for (int i = threadIdx.x; i < k; i += blockDim.x)
    if (i >= n) top[i] = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const uint64_t mine = entry[i];
    const int rank = larger(entry, n, mine);
    if (rank < k) top[rank] = mine;
  }
}

template <typename T, int LOADS>
__global__ void __launch_bounds__(kThreads) logprob_kernel(const LogprobParams p) {
  constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  constexpr int kWaves = kThreads / 64;
  constexpr int kSlots = kThreads;   // candidates that LDS holds
  struct alignas(16) Granule { T v[kVec]; };
  __shared__ float s_m[kWaves], s_l[kWaves], s_t[kWaves];
  __shared__ uint32_t s_key[kThreads];
  alignas(16) __shared__ uint64_t s_entry[kSlots];
  __shared__ uint64_t s_top[kMaxTop];
  __shared__ uint64_t s_best[kWaves];
  __shared__ uint32_t s_threshold;
  __shared__ int s_count;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / p.chunks;
  const int chunk = static_cast<int>(blockIdx.x - row * p.chunks);
  const T* x = static_cast<const T*>(p.logits) + row * p.logits_stride;
  // Logits are taken in granules of 16 aligned bytes, counted from the granule that holds the row's first one:
  // `lead` values of that granule lie in front of the row. Only granules that lie in the row as a whole are
  // loaded as such. The up to kVec - 1 logits in front of the first and behind the last of them are strays, one
  // per thread: of the first chunk's threads 0 .. kVec - 1, and of the last one's threads kVec .. 2 kVec - 1.
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  const int first = (chunk * kThreads * LOADS + tid) * kVec - lead;   // index of this thread's first granule's first logit (vocab <= 2^30)
  const int head_end = min((kVec - lead) % kVec, p.vocab);      // strays: [0, head_end) and [tail, vocab)
  const int tail = max(head_end, (p.vocab + lead) / kVec * kVec - lead);
  int stray_at = -1;
  if (chunk == 0 && tid < head_end) stray_at = tid;
  if (chunk == p.chunks - 1 && tid >= kVec && tid - kVec < p.vocab - tail) stray_at = tail + tid - kVec;
  constexpr uint32_t kInf = sizeof(T) == 4 ? 0xff800000u : kIsF16<T> ? 0xfc00fc00u : 0xff80ff80u;   // -inf in every value
  u32x4 raw[LOADS];
  bool any = stray_at >= 0;
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const int e0 = first + j * kThreads * kVec;
    raw[j] = u32x4{kInf, kInf, kInf, kInf};
    if (e0 >= 0 && e0 + kVec <= p.vocab) {
      raw[j] = *reinterpret_cast<const u32x4*>(x + e0);
      any = true;
    }
  }
  const float stray = stray_at >= 0 ? to_f32(x[stray_at]) : neg_inf();
  const float token_logit = p.chunks == 1 && tid < p.num_ids ? logit_of_id<T>(p, row, tid) : neg_inf();

  float mine = stray, mine_number = stray;   // the largest, NaN if there is one; the largest number
#pragma unroll
  for (int j = 0; j < LOADS; ++j) {
    const Granule g = __builtin_bit_cast(Granule, raw[j]);
#pragma unroll
    for (int e = 0; e < kVec; ++e) mine = max_or_nan(mine, to_f32(g.v[e]));
  }
  if (mine != mine) mine_number = __builtin_huge_valf(); else mine_number = mine;   // (with a NaN: look at all of them)
  float m = mine;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = max_or_nan(m, __shfl_xor(m, o, 64));
  if (lane == 0) s_m[wave] = m;
  s_key[tid] = any ? key_of(mine) : 0;
  if (tid == 0) s_count = 0;
  __syncthreads();
  m = s_m[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = max_or_nan(m, s_m[w]);
  m = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, m)));   // (the same in all: a scalar register)

  // wave 0 searches the threshold while the others sum
  if (p.top_k > 0 && wave == 0) {
    // the maxima of 64 groups of threads for k up to 32, of 256 for k up to 128
    uint32_t key[4] = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) key[w % 4] = max(key[w % 4], s_key[w * 64 + lane]);
    auto search = [&](auto groups_c) __attribute__((always_inline)) {
      uint32_t found = 0;
      for (int bit = 31; bit >= 12; --bit) {   // the low bits stay zero: a slightly lower threshold, a few more candidates
        const uint32_t trial = found | 1u << bit;
        int reach = 0;
#pragma unroll
        for (int r = 0; r < decltype(groups_c)::value; ++r) reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[r] >= trial));
        if (reach >= p.top_k) found = trial;
      }
      return found;
    };
    uint32_t threshold;
    if (p.top_k <= 32) {
      key[0] = max(max(key[0], key[1]), max(key[2], key[3]));
      threshold = search(std::integral_constant<int, 1>{});
    } else {
      threshold = search(std::integral_constant<int, 4>{});
    }
    if (lane == 0) s_threshold = threshold;
  }

  // d as one multiply-add against m scale, which is rounded: every exponent is then off by the same half a step of it, taken
  // out of the sums below. Where that is more than half a unit (a temperature near 0, or nothing but tokens banned with
  // the type's lowest value) the difference comes first instead, which is exact near the maximum; as rare, from memory
  // again (unrolled over the registers it cost the common path 20 of them: 61 instead of 51 us for 512 fp32 rows of
  // 131072).
  const float scale = p.inv_temp * kLog2e, m_finite = m == neg_inf() ? 0.f : m;
  const bool near = __builtin_fabsf(m_finite * scale) <= 16777216.f;
  const float m_scaled = m_finite * scale;
  float l = 0.f, t = 0.f;
  auto add = [&](float exponent) __attribute__((always_inline)) {
    const float d = max_or_nan(exponent, -256.f);   // 2^-256 is 0 in 32 bits; keeps 0 * inf out of t
    const float w = fast_exp2(d);
    l += w;
    t = __builtin_fmaf(w, d, t);
  };
  if (near) {
    add(__builtin_fmaf(stray, scale, -m_scaled));
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      FTA_FORGET(raw[j]);
      const Granule g = __builtin_bit_cast(Granule, raw[j]);
#pragma unroll
      for (int e = 0; e < kVec; ++e) add(__builtin_fmaf(to_f32(g.v[e]), scale, -m_scaled));
    }
  } else {
    add((stray - m_finite) * scale);
#pragma unroll 1
    for (int j = 0; j < LOADS; ++j) {
      const int e0 = first + j * kThreads * kVec;
      if (e0 < 0 || e0 + kVec > p.vocab) continue;
      const Granule g = *reinterpret_cast<const Granule*>(x + e0);
#pragma unroll
      for (int e = 0; e < kVec; ++e) add((to_f32(g.v[e]) - m_finite) * scale);
    }
  }
  l = wave_sum(l);
  t = wave_sum(t);
  if (lane == 0) {
    s_l[wave] = l;
    s_t[wave] = t;
  }
  __syncthreads();
  l = s_l[0];
  t = s_t[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    l += s_l[w];
    t += s_t[w];
  }
  if (near) {
    const float off = __builtin_fmaf(m_finite, scale, -m_scaled), back = exp2f(-off);   // the exponents' common rounding
    t = back * __builtin_fmaf(-off, l, t);
    l *= back;
  }

  if (p.top_k > 0) {
    // Where fewer than k groups of threads hold a finite logit, every finite one is a candidate, and of a small vocabulary
    // every number; what is short of k even so (-inf and NaN fill up) is extracted one by one.
    const bool few = s_threshold < key_of(neg_inf());
    const float least = !few ? value_of(s_threshold) : p.vocab <= kSlots ? neg_inf() : -__FLT_MAX__;
    if (mine_number >= least) {
      auto collect = [&](float v, int at) __attribute__((always_inline)) {
        if (!(v >= least)) return;
        const int slot = atomicAdd(&s_count, 1);
        if (slot < kSlots) s_entry[slot] = entry_of(v, at);
      };
      if (stray_at >= 0) collect(stray, stray_at);
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        FTA_FORGET(raw[j]);
        const Granule g = __builtin_bit_cast(Granule, raw[j]);
        const int e0 = first + j * kThreads * kVec;
        float best = to_f32(g.v[0]);
#pragma unroll
        for (int e = 1; e < kVec; ++e) best = fmaxf(best, to_f32(g.v[e]));
        if (!(best >= least) || e0 < 0 || e0 + kVec > p.vocab) continue;   // most granules, for all lanes of a wave
#pragma unroll
        for (int e = 0; e < kVec; ++e) collect(to_f32(g.v[e]), e0 + e);
      }
    }
    __syncthreads();
    const int n = s_count;
    if (n <= kSlots && (!few || n >= p.top_k)) {
      rank_entries(s_entry, n, p.top_k, s_top);
    } else {
      uint64_t last = ~0ull;
      for (int k = 0; k < p.top_k; ++k) {
        uint64_t best = 0;
        auto look = [&](float v, int at) __attribute__((always_inline)) {
          const uint64_t c = entry_of(v, at);
          if (c < last && c > best) best = c;
        };
        if (stray_at >= 0) look(stray, stray_at);
        // from memory again: rare, and a second unrolled walk over the registers would cost the common path its own
#pragma unroll 1
        for (int j = 0; j < LOADS; ++j) {
          const int e0 = first + j * kThreads * kVec;
          if (e0 < 0 || e0 + kVec > p.vocab) continue;
          const Granule g = *reinterpret_cast<const Granule*>(x + e0);
#pragma unroll
          for (int e = 0; e < kVec; ++e) look(to_f32(g.v[e]), e0 + e);
        }
        best = wave_max_u64(best);
        if (lane == 0) s_best[wave] = best;
        __syncthreads();
        best = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) best = s_best[w] > best ? s_best[w] : best;
        if (tid == 0) s_top[k] = best;
        last = best;
        __syncthreads();   // s_best is free again
        if (best == 0) {   // none left
          for (int i = k + tid; i < p.top_k; i += kThreads) s_top[i] = 0;
          break;
        }
      }
    }
    __syncthreads();
  }

  if (p.chunks == 1) {
    write_row<T>(p, row, m, l, t, token_logit, s_top);
    return;
  }
  char* out = p.workspace + (row * p.chunks + chunk) * chunk_bytes(p.top_k);
  if (tid == 0) *reinterpret_cast<ChunkStats*>(out) = ChunkStats{m, l, t, 0.f};
  uint64_t* keys = reinterpret_cast<uint64_t*>(out + sizeof(ChunkStats));
  for (int k = tid; k < p.top_k; k += kThreads) keys[k] = s_top[k];
}

// Joins the chunks of a row. One workgroup per row.
template <typename T>
__global__ void __launch_bounds__(256) logprob_join_kernel(const LogprobParams p) {
  constexpr int kSlots = 1024;
  alignas(16) __shared__ uint64_t s_entry[kSlots];
  alignas(16) __shared__ uint64_t s_reach[kSlots];
  __shared__ uint64_t s_top[kMaxTop];
  __shared__ int s_count;
  const int64_t row = blockIdx.x;
  const char* ws = p.workspace + row * p.chunks * chunk_bytes(p.top_k);
  const float token_logit = static_cast<int>(threadIdx.x) < p.num_ids ? logit_of_id<T>(p, row, threadIdx.x) : neg_inf();
  // every wave joins the chunks, one per lane
  const int lane = threadIdx.x & 63;
  const float scale = p.inv_temp * kLog2e;
  float m = neg_inf(), l = 0.f, t = 0.f;
  for (int c0 = 0; c0 < p.chunks; c0 += 64) {
    ChunkStats s{neg_inf(), 0.f, 0.f, 0.f};
    if (c0 + lane < p.chunks) s = *reinterpret_cast<const ChunkStats*>(ws + (c0 + lane) * chunk_bytes(p.top_k));
    float top = s.m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max_or_nan(top, __shfl_xor(top, o, 64));
    top = max_or_nan(top, m);
    auto moved = [&](float from, float sum, float weighted, float* to_sum, float* to_weighted) {
      *to_sum = *to_weighted = 0.f;
      if (from == neg_inf()) return;
      const float shift = (from - top) * scale;          // NaN where the maximum is NaN or +inf, and so are l and t then
      const float w = exp2f(shift);
      *to_sum = w * sum;
      if (w != 0.f) *to_weighted = w * (weighted + shift * sum);   // (a NaN weight is not 0)
    };
    float sum, weighted, sum_before, weighted_before;
    moved(s.m, s.l, s.t, &sum, &weighted);
    moved(m, l, t, &sum_before, &weighted_before);
    l = wave_sum(sum) + sum_before;
    t = wave_sum(weighted) + weighted_before;
    m = top;
  }
  if (p.top_k > 0) {
    // As many chunks' keys at a time as fit next to the best so far. Ranking them all by counting takes n^2 steps (20 us
    // for 320 keys), so the k-th largest value is searched first, bit by bit, and what reaches it is ranked.
    const int step = (kSlots - p.top_k) / p.top_k;
    int kept = 0;
    for (int c0 = 0; c0 < p.chunks; c0 += step) {
      const int n = kept + min(step, p.chunks - c0) * p.top_k;
      for (int i = kept + threadIdx.x; i < n; i += 256) {
        const int j = i - kept;
        s_entry[i] = reinterpret_cast<const uint64_t*>(ws + (c0 + j / p.top_k) * chunk_bytes(p.top_k) + sizeof(ChunkStats))[j % p.top_k];
      }
      if (threadIdx.x == 0) s_count = 0;
      __syncthreads();
      auto search = [&](auto groups_c) __attribute__((always_inline)) {   // by every wave for itself
        constexpr int kGroups = decltype(groups_c)::value;
        uint32_t key[kGroups];
#pragma unroll
        for (int r = 0; r < kGroups; ++r) key[r] = r * 64 + lane < n ? static_cast<uint32_t>(s_entry[r * 64 + lane] >> 32) : 0;
        uint32_t found = 0;
        for (int bit = 31; bit >= 0; --bit) {
          const uint32_t trial = found | 1u << bit;
          int reach = 0;
#pragma unroll
          for (int r = 0; r < kGroups; ++r) reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[r] >= trial));
          if (reach >= p.top_k) found = trial;
        }
        return found;
      };
      const uint32_t found = n <= 64 ? search(std::integral_constant<int, 1>{}) : n <= 256 ? search(std::integral_constant<int, 4>{})
                                                                                           : search(std::integral_constant<int, kSlots / 64>{});
      for (int i = threadIdx.x; i < n; i += 256) {
        const uint64_t mine = s_entry[i];
        if (mine != 0 && static_cast<uint32_t>(mine >> 32) >= found) s_reach[atomicAdd(&s_count, 1)] = mine;
      }
      __syncthreads();
      rank_entries(s_reach, s_count, p.top_k, s_top);
      __syncthreads();
      if (c0 + step < p.chunks) {
        for (int i = threadIdx.x; i < p.top_k; i += 256) s_entry[i] = s_top[i];
        kept = p.top_k;
        __syncthreads();
      }
    }
  }
  write_row<T>(p, row, m, l, t, token_logit, s_top);
}

// How a call is cut. A workgroup of 512 threads holds 8 granules of 16 bytes per thread in registers; a CU holds four
// such workgroups, so that the loads of some overlap the arithmetic of others. A row that fits one takes one launch. Where
// a row is cut anyway and the pieces would leave CUs idle, a thread takes half as much: 8 rows of 50001 fp16 10.5 instead
// of 12.1 us, one of 131072 bf16 12.4 instead of 14.9 (a quarter: 16.8, the join has more to rank). Whole rows of up to
// 131072 in a workgroup of 1024 threads saved the second launch and lost by the longer chain: 15.8 instead of 12.6 us
// for 104 rows of 50001.
struct Cut {
  bool small;
  int chunks;
};
// `aligned`: every row starts 16-byte aligned, which is only known with the pointer; the workspace is sized without.
Cut cut_of(const fta_logprob_args& a, bool aligned) {
  const int vec = a.dtype == FTA_F32 ? 4 : 8;
  const int64_t span = static_cast<int64_t>(a.vocab) + (aligned ? 0 : vec - 1);   // with the largest possible lead
  const auto chunks = [vec](int64_t values, int loads) { return (values + kThreads * loads * vec - 1) / (kThreads * loads * vec); };
  Cut c;
  c.small = chunks(a.vocab, 8) > 1 && a.rows * chunks(a.vocab, 4) <= 256;
  c.chunks = static_cast<int>(chunks(span, c.small ? 4 : 8));
  return c;
}

int validate_sizes(const fta_logprob_args& a) {
  if (a.dtype != FTA_F32 && a.dtype != FTA_F16 && a.dtype != FTA_BF16) return FTA_ERR_DTYPE;
  if (a.id_dtype != FTA_I32 && a.id_dtype != FTA_I64) return FTA_ERR_DTYPE;
  if (a.rows <= 0 || a.vocab <= 0 || a.num_ids < 0 || a.top_k < 0 || a.top_k > a.vocab) return FTA_ERR_SHAPE;
  if (a.top_k > kMaxTop || a.vocab > 1 << 30) return FTA_ERR_UNSUPPORTED;
  if (!(a.inv_temperature > 0.f) || !std::isfinite(kLog2e * a.inv_temperature)) return FTA_ERR_UNSUPPORTED;   // the exponents' scale
  return FTA_OK;
}

int64_t workspace_bytes(const fta_logprob_args& a) {
  const Cut c = cut_of(a, false);
  return c.chunks == 1 ? 0 : a.rows * c.chunks * chunk_bytes(a.top_k);
}

template <typename T>
int launch(const LogprobParams& p, const Cut& cut, hipStream_t stream) {
  const int64_t grid = p.rows * p.chunks;
  if (grid > 0x7fffffffLL) return FTA_ERR_SHAPE;
  const dim3 g(static_cast<unsigned>(grid));
  if (int st = cut.small ? launch_checked(logprob_kernel<T, 4>, g, dim3(kThreads), 0, stream, p)
                         : launch_checked(logprob_kernel<T, 8>, g, dim3(kThreads), 0, stream, p))
    return st;
  if (cut.chunks == 1) return FTA_OK;
  return launch_checked(logprob_join_kernel<T>, dim3(static_cast<unsigned>(p.rows)), dim3(256), 0, stream, p);
}

}  // namespace
}  // namespace fta

extern "C" {

int fta_logprobs_workspace(const fta_logprob_args* args, int64_t* bytes) {
  if (!args || !bytes) return FTA_ERR_NULL_POINTER;
  if (int st = fta::validate_sizes(*args)) return st;
  *bytes = fta::workspace_bytes(*args);
  return FTA_OK;
}

int fta_logprobs(const fta_logprob_args* args, void* hip_stream) {
  using namespace fta;
  if (!args) return FTA_ERR_NULL_POINTER;
  const fta_logprob_args& a = *args;
  if (int st = validate_sizes(a)) return st;
  if (!a.logits || !a.entropy || !a.lse) return FTA_ERR_NULL_POINTER;
  if (a.num_ids > 0 && (!a.token_ids || !a.logprobs)) return FTA_ERR_NULL_POINTER;
  if (a.top_k > 0 && (!a.top_logprobs || !a.top_ids)) return FTA_ERR_NULL_POINTER;
  if (a.logits_stride < 0 || a.id_stride[0] < 0 || a.id_stride[1] < 0) return FTA_ERR_STRIDE;
  if (reinterpret_cast<uintptr_t>(a.logits) % (a.dtype == FTA_F32 ? 4 : 2)) return FTA_ERR_STRIDE;
  const int64_t need = workspace_bytes(a);
  if (need > 0) {
    if (!a.workspace) return FTA_ERR_NULL_POINTER;
    if (a.workspace_bytes < need) return FTA_ERR_SCRATCH_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(a.workspace) % 16) return FTA_ERR_STRIDE;
  }
  const int es = a.dtype == FTA_F32 ? 4 : 2;
  const Cut cut = cut_of(a, reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (a.rows == 1 || a.logits_stride * es % 16 == 0));
  LogprobParams p{};
  p.logits = a.logits; p.ids = a.token_ids; p.logprobs = a.logprobs; p.entropy = a.entropy; p.lse = a.lse;
  p.top_logprobs = a.top_logprobs; p.top_ids = a.top_ids; p.workspace = static_cast<char*>(a.workspace);
  p.rows = a.rows; p.logits_stride = a.logits_stride;
  p.id_stride[0] = a.id_stride[0]; p.id_stride[1] = a.id_stride[1];
  p.vocab = a.vocab; p.num_ids = a.num_ids; p.top_k = a.top_k; p.id_is_i64 = a.id_dtype == FTA_I64;
  p.chunks = cut.chunks;
  p.inv_temp = a.inv_temperature;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return FTA_ERR_NO_DEVICE;
  hipStream_t stream = static_cast<hipStream_t>(hip_stream);
  if (a.dtype == FTA_F32) return launch<float>(p, cut, stream);
  if (a.dtype == FTA_F16) return launch<_Float16>(p, cut, stream);
  return launch<__bf16>(p, cut, stream);
}

}  // extern "C"
