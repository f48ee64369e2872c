// Tree attention with shaped scores (fta_shaped_decode, include/fta.h): scores capped by a tanh, a bias that
// falls with distance, a sliding window, a document start per sequence; f16 / bf16 / f32, head_dim 32 .. 256.
//
// One pass over the keys with a running maximum and sum. Query heads that share a cache head form a unit, their
// rows share one K/V stream; a workgroup of four waves holds 128 rows of a unit (or 64, with two waves per 32 rows
// that take half of the keys each) and walks over tiles of 64 keys (f32: 32) that go from memory straight into
// LDS (global_load_lds, two stages; f32 units of up to 64 rows: two or four waves per 32 rows, 64 or 128 keys a tile). Per tile a wave computes
//     S^T = K Q^T     (32x32x16 products, lane = query row; Q stays in registers)
//     z = shape(S), p = 2^(z - m)        (everything in units of log2 e)
//     O^T += V^T P^T  (V^T by transposing LDS reads, P^T straight from the accumulator registers)
//
// What bounds it: the stream of K and V for calls of few rows; else the vector unit. Per 32x32 scores the two
// products take 512 cycles of the matrix unit (head_dim 128), the plain softmax about 290 cycles of the vector
// unit and the capped one about 670 (three transcendentals a score), so two workgroups share a CU and one's
// products run under the other's softmax. 64 sequences of up to 32768 keys, 64 heads on 8, 16 nodes, capped and biased
// scores: 3.85 GB in 804 us (4.8 TB/s of a copy's 5.1); 8 sequences of 8192 keys, 32 heads on 8, 64 nodes, capped
// scores: 124 to 127 us (558 TFLOP/s of a large product's 1135), with a bias too about as long (119 to 126, in turn with the
// former's 120 to 127), 107 to 112 us with plain scores; one token of 8 sequences, 84 MB: 28 us.
//
// The work is cut evenly whatever the lengths: the (sequence, unit) pairs' tiles are laid out as one line, every
// workgroup takes an equal stretch of it, computed by each workgroup from the lengths on the device. A pair that
// lies in one stretch is written to `out`; one that is cut leaves fp32 partials (O, m, l), at most two per
// workgroup, and a second kernel joins them. Short calls give every pair a workgroup and skip the second kernel.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "fta_device.h"
#include "shaped_attn_ops.h"

namespace fta {
namespace {

struct ShapedParams {
  const void* q;
  const void* k;
  const void* v;
  const void* ck;
  const void* cv;
  const void* mask;
  const void* lens;
  void* out;
  const int32_t* table;
  const float* slopes;
  const int32_t* first;
  const int32_t* depths;
  float* partial;
  int32_t bsz, num_q_heads, q_len, cache_len, heads_per_unit, units, kv_group, cur_group;
  int32_t rows, row_blocks, groups, tree_tiles;   // groups: stretches per row block
  int32_t whole;          // every (sequence, unit) pair is a stretch of its own
  int32_t rows_cap;       // rows per partial
  int32_t lead_groups, lead_share;   // the first lead_groups stretches hold lead_share / 1024 of the line; 0: all alike
  int32_t len_is_i64, mask_packed, page_shift, window;
  float scale, softcap;
  int64_t partial_floats; // per partial
  int64_t q_stride[3], k_stride[3], v_stride[3], ck_stride[3], cv_stride[3], mask_stride[3], out_stride[3];
  int64_t table_stride, depth_stride;
};

// A tree tile is a masked step of its own and comes after a drained cache stream: it is counted as this many cache
// tiles when the line is cut.
constexpr int kTreeWeight = 3;
// Stretches are at least this many tiles long: below, the prologue and the partials cost more than they spread.
constexpr int kMinStretch = 4;

// 2^z is 0 in 32 bits for z up to here (the smallest positive value is 2^-149).
constexpr float kNoWeight = -150.f;
// Scores are formed relative to a row's running maximum, which rounds them to 2^-24 of its size. Keys that a finite mask
// (-10^4, the type's lowest value) puts out of reach may come before those that count, and a maximum of theirs would
// swallow the scores behind it: one below this bound is not subtracted until the tile's own maximum is known. That matters
// up to the second cache tile behind the tree's: of the nearest one some waves may hold only keys behind the length, and
// who sees no key of the second sees none of those in front of it. (In every tile it costs a rescaling each where the
// nearest keys are far off: 396 instead of 355 us for 8 sequences of 32768 keys, 32 heads on 8, 64 nodes, cap and bias.)
constexpr float kLowMaximum = -128.f;

// One 1 KiB block of LDS per wave-wide load: 1024 / ROW_BYTES rows, their 16-byte chunks interleaved, blocks 1024 +
// one chunk column apart, so that both operand reads fall on distinct banks and every fragment address is a lane
// base plus a constant (the layout of the stage-1 kernel's tiles, for any row size).
template <int ROW_BYTES, int KEYS>
struct RowTile {
  static constexpr int kRowsPerBlock = 1024 / ROW_BYTES;
  static constexpr int kChunkStride = 16 * kRowsPerBlock;
  static constexpr int kBlockPitch = 1024 + kChunkStride;
  static constexpr int kBlocks = KEYS / kRowsPerBlock;
  static constexpr int kBytes = kBlocks * kBlockPitch;
  static __host__ __device__ constexpr int at(int r, int c) {
    return (r / kRowsPerBlock) * kBlockPitch + c * kChunkStride + (r % kRowsPerBlock) * 16;
  }
};

template <int I, int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unrolled<I + 1, N>(f);
  }
}

template <typename T> constexpr bool kIs32 = sizeof(T) == 4;
// Weights are taken against a reference this far below the running maximum, in units of log2. fp16 ends at 2^-24 and
// 2^16: with 2^7 for the largest key (up to 2^15 until the maximum moves) what is lost of 131072 keys far below it is less
// than 2^-15 of the sum; against the maximum itself it was up to 2^-8. The other types have the range of 32 bits.
template <typename T> constexpr float kHeadroom = 0.f;
template <> constexpr float kHeadroom<_Float16> = 7.f;
// Keys of a tile; WK waves of the same 32 rows share them.
template <typename T, int WK> constexpr int kTileKeys = kIs32<T> ? 32 * WK : 64;
template <typename T, int D, int WK> constexpr int kLdsBytes = 4 * RowTile<D * static_cast<int>(sizeof(T)), kTileKeys<T, WK>>::kBytes;

// S^T block += K fragment x Q fragment, 16 bytes of a row each: one product for 16-bit types, four for f32.
template <typename T>
__device__ __forceinline__ f32x16 mma_chunk(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (kIs32<T>) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = mma_f32(x[e], y[e], c);
    return c;
  } else {
    return Mfma<T>::mma(__builtin_bit_cast(typename Mfma<T>::Vec8, a), __builtin_bit_cast(typename Mfma<T>::Vec8, b), c);
  }
}

// tanh(y) where the form 1 - 2 / (1 + e^(2 y)) alone would show: its error is about 2^-23 absolute and a cap multiplies it.
// f32 calls take this one, 16-bit calls under a cap above kShortCap, where that error passes 2^-13, a quarter of fp16's
// half step (a cap of 10^6 was off by 0.02 in the output, one of 10^8 averaged all values). Below 0.45 the series of tanh through y^13 (the next term is 2^-25 of the value), above it that form,
// there off by at most 3.1e-7 of the value. The library's tanhf took half as long again per score.
constexpr float kShortCap = 256.f;
__device__ __forceinline__ float tanh_of(float y) {
  const float q = y * y;
  float series = __builtin_fmaf(q, 21844.f / 6081075.f, -1382.f / 155925.f);
  series = __builtin_fmaf(q, series, 62.f / 2835.f);
  series = __builtin_fmaf(q, series, -17.f / 315.f);
  series = __builtin_fmaf(q, series, 2.f / 15.f);
  series = __builtin_fmaf(q, series, -1.f / 3.f);
  series = __builtin_fmaf(y * q, series, y);
  const float far = __builtin_fmaf(-2.f, fast_rcp(1.f + fast_exp2(2.f * kLog2e * y)), 1.f);
  return q < 0.2025f ? series : far;
}

// What a sequence contributes to the line, per unit.
struct Sequence {
  int length;   // T, clamped to the cache
  int first;    // first key of the document
  int lo;       // first key any row may see (depths are >= 0)
  int tile0;    // its tile
  int n_cache;  // cache tiles
  int n;        // stretch of the line: cache tiles, then kTreeWeight per tree tile
};
template <int KEYS>
__device__ __forceinline__ Sequence sequence_of(const ShapedParams& p, int b) {
  Sequence s;
  const int64_t len = load_len(p.lens, p.len_is_i64, b);
  s.length = static_cast<int>(len < 0 ? 0 : len > p.cache_len ? p.cache_len : len);
  s.first = p.first ? min(max(p.first[b], 0), s.length) : 0;
  s.lo = p.window > 0 ? max(s.first, s.length - p.window + 1) : s.first;
  s.lo = min(max(s.lo, 0), s.length);
  s.tile0 = s.lo / KEYS;
  s.n_cache = s.length > s.lo ? (s.length + KEYS - 1) / KEYS - s.tile0 : 0;
  s.n = s.n_cache + kTreeWeight * p.tree_tiles;
  return s;
}
// The line: every sequence's units, one after the other. Each lane of a wave looks at one sequence of a batch of up to
// 64; larger batches in rounds.
struct Place {
  int b;       // sequence
  int begin;   // where its first unit begins
  int total;   // length of the whole line
  Sequence seq;
};
// The place of x = at(total) on the line, for the kernel, or (with by_sequence) of sequence `at` itself, for the join.
// Every lane of the wave must call it.
template <int KEYS, typename At>
__device__ __forceinline__ Place place_of(const ShapedParams& p, bool by_sequence, At&& at) {
  const int lane = threadIdx.x & 63;
  Place r{-1, 0, 0, {}};
  Sequence mine{};
  int n = 0, upto = 0;   // of this lane's sequence: its length on the line, and that of all up to it in this round
  auto look = [&](int c) __attribute__((always_inline)) {
    mine = sequence_of<KEYS>(p, min(c + lane, p.bsz - 1));
    n = c + lane < p.bsz ? mine.n * p.units : 0;
    upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(upto, o, 64);
      upto += lane >= o ? y : 0;
    }
    return __builtin_amdgcn_readlane(upto, 63);
  };
  for (int c = 0; c < p.bsz; c += 64) r.total += look(c);
  const int x = at(r.total);
  int base = 0;
  for (int c = 0; c < p.bsz; c += 64) {
    const int round = p.bsz > 64 ? look(c) : r.total;
    const uint64_t holds = __builtin_amdgcn_ballot_w64(by_sequence ? c + lane == x : n > 0 && x < base + upto);
    if (holds) {
      const int l = __builtin_ctzll(holds);
      r.b = c + l;
      r.begin = base + __builtin_amdgcn_readlane(upto - n, l);
      r.seq.length = __builtin_amdgcn_readlane(mine.length, l);
      r.seq.first = __builtin_amdgcn_readlane(mine.first, l);
      r.seq.lo = __builtin_amdgcn_readlane(mine.lo, l);
      r.seq.tile0 = __builtin_amdgcn_readlane(mine.tile0, l);
      r.seq.n_cache = __builtin_amdgcn_readlane(mine.n_cache, l);
      r.seq.n = __builtin_amdgcn_readlane(mine.n, l);
      return r;
    }
    base += round;
  }
  return r;
}

// How the line is cut: into stretches whose bounds are rounded multiples of an unrounded length, so that equally long
// pairs are cut alike (multiples of a rounded length drift and leave pieces of a tile or two, each a prologue and a
// partial: 240 against 222 us for 16 sequences of 16384 keys, 64 heads on 8, 16 nodes). `heads` of them share the line up
// to `middle`, the rest what is behind it. In 32-bit floats, a division each: any bounds do that both kernels agree on, so
// the one product with a sum behind it is written as a fused one, and no compilation rounds it differently.
struct Stretches {
  int total, groups, heads, middle;
  float lead, tail;   // lengths
  __device__ __forceinline__ int start(int g) const {
    const float nth = static_cast<float>(g < heads ? g : g - heads), length = g < heads ? lead : tail;
    const int x = static_cast<int>(__builtin_fmaf(nth, length, 0.03125f));   // (a length of 43 2/3 times 3 is 131, not 130)
    return g >= groups ? total : g < heads ? min(x, middle) : min(middle + x, total);
  }
  __device__ __forceinline__ int holder(int x) const {
    int g = x < middle ? static_cast<int>(static_cast<float>(x) * fast_rcp(lead)) : heads + static_cast<int>(static_cast<float>(x - middle) * fast_rcp(tail));
    g = min(g, groups - 1);   // (about right)
    while (start(g) > x) --g;
    while (start(g + 1) <= x) ++g;
    return g;
  }
};
__device__ __forceinline__ Stretches cut_line(const ShapedParams& p, int total) {
  Stretches s;
  s.total = total;
  s.groups = max(min(p.groups, total / kMinStretch), 1);
  s.heads = total / (2 * kMinStretch) > p.groups ? p.lead_groups : 0;
  s.middle = s.heads > 0 ? (total >> 10) * p.lead_share + ((total & 1023) * p.lead_share >> 10) : 0;
  s.lead = s.heads > 0 ? static_cast<float>(s.middle) * fast_rcp(static_cast<float>(s.heads)) : 1.f;
  s.tail = static_cast<float>(total - s.middle) * fast_rcp(static_cast<float>(s.groups - s.heads));
  return s;
}

// SERIES: a cap's tanh is tanh_of. A kernel of its own for 16-bit types: in one with the short form the series, unused,
// took 7 % of plain calls (362 against 338 us for 8 sequences of 32768 keys, 32 heads on 8, 64 nodes).
template <typename T, int D, int WK, bool PAGED, bool SERIES = kIs32<T>>
__global__ void __launch_bounds__(256)
FTA_WAVES_PER_EU((D <= 128 ? 2 : 1))   // head_dim 256 needs the whole register file
shaped_kernel(const ShapedParams p) {
  constexpr int kKeys = kTileKeys<T, WK>;
  constexpr int ES = sizeof(T);
  using Tile = RowTile<D * ES, kKeys>;
  constexpr int kStages = 2;
  constexpr int KS = D * ES / 32;            // 32-byte steps of a row in the first product
  constexpr int DB = D / 32;                 // 32-column blocks of O
  constexpr int NB = kKeys / 32 / WK;        // 32-key blocks of a tile per wave
  constexpr int RPB = Tile::kRowsPerBlock;
  constexpr int kLoads = Tile::kBlocks / 4;  // wave-wide loads per wave, tile and tensor
  constexpr int kRowsPerWg = 128 / WK;
  constexpr int kVRing = kStages * Tile::kBytes;
  static_assert(NB >= 1 && Tile::kBlocks % 4 == 0, "tile shape");

  FTA_DYNAMIC_LDS(smem);
  __shared__ uint32_t s_seen[kKeys / 32];   // keys of a tree tile that a row of the workgroup sees
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 31, lh = lane >> 5;
  const int L = p.q_len;

  // Workgroup ids go round-robin to the 8 XCDs: the row blocks of one stretch read the same keys and get ids that
  // differ by a multiple of 8, so that the second one's reads hit the XCD's L2.
  int group, row_block;
  {
    const int id = blockIdx.x, rbs = p.row_blocks, even = p.groups - p.groups % 8;
    if (id < even * rbs) {
      row_block = id / 8 % rbs;
      group = id / 8 / rbs * 8 + id % 8;
    } else {
      row_block = (id - even * rbs) % rbs;
      group = even + (id - even * rbs) / rbs;
    }
  }

  // ---- this workgroup's stretch [x0, x1) of the line; x walks over it pair by pair
  int b, unit, begin, x, x0, x1;   // begin: where the current pair starts
  Sequence seq;
  if (p.whole) {
    b = group / p.units;
    unit = group % p.units;
    seq = sequence_of<kKeys>(p, b);
    begin = x0 = x = 0;
    x1 = seq.n;
  } else {
    bool none = false;
    const Place here = place_of<kKeys>(p, false, [&](int total) __attribute__((always_inline)) {
      const Stretches cut = cut_line(p, total);
      x0 = cut.start(group);
      x1 = cut.start(group + 1);
      none = x0 >= total;
      return min(x0, total - 1);
    });
    if (none) return;
    x = x0;
    b = here.b;
    seq = here.seq;
    unit = (x0 - here.begin) / seq.n;
    begin = here.begin + unit * seq.n;
  }

  // ---- lane constants of the loads and of the operand reads
  const int ld_row = lane % RPB, ld_chunk = lane / RPB;   // lane i fetches chunk i / RPB of row i % RPB of a block
  const int64_t k_row = p.k_stride[2] * ES, v_row = p.v_stride[2] * ES;
  // bytes from a tile's first row to this lane's piece of its block (of its wave's first block, for contiguous caches)
  const int64_t k_lane = ((PAGED ? 0 : wave * RPB) + ld_row) * k_row + ld_chunk * 16, v_lane = ((PAGED ? 0 : wave * RPB) + ld_row) * v_row + ld_chunk * 16;
  const int64_t k_step = 4 * RPB * k_row, v_step = 4 * RPB * v_row;   // to the wave's next block
  const uint32_t lds0 = lds_address(smem);
  const int kb0 = wave % WK * NB;          // first key block of this wave
  const uint32_t k_rd = lds0 + Tile::at(li, lh) + kb0 * Tile::at(32, 0);
  // 16-bit V^T: 16-lane group g covers columns 16 (g % 2) .. + 15 of a 32-column block, lane s of it addresses key
  // s / 4, columns 4 (s % 4) .. + 3. f32 V: lane (i, h) reads column i of the keys 4 h + r % 4 + 8 (r / 4).
  const uint32_t v_rd = lds0 + kVRing + kb0 * Tile::at(32, 0) +
      (kIs32<T> ? Tile::at(4 * lh, li / 4) + li % 4 * 4
                : Tile::at(4 * lh + (lane & 15) / 4, 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) + (lane & 1) * 8);
  const int page_mask = (1 << p.page_shift) - 1;
  const int64_t k_page = p.k_stride[0] * ES, v_page = p.v_stride[0] * ES;

  // Scores in units of log2 e: without a cap z = c s; with one cap2 tanh(x / cap), the tanh written out as
  // 1 - 2 / (1 + 2^(ex s)), or tanh_of(ex s).
  const bool capped = p.softcap > 0.f, sloped = p.slopes != nullptr;
  const float c = p.scale * kLog2e;
  const float cap2 = p.softcap * kLog2e;
  const float ex = capped ? (SERIES ? 1.f : 2.f * kLog2e) * p.scale / p.softcap : 0.f;

  for (;;) {
    // ---- one pair: places [from, to) of its stretch
    const int from = x - begin, to = min(seq.n, x1 - begin);
    const bool complete = from == 0 && to == seq.n;
    const int cache_from = min(from, seq.n_cache), cache_tiles = min(to, seq.n_cache) - cache_from;
    const int u0 = (max(from - seq.n_cache, 0) + kTreeWeight - 1) / kTreeWeight;   // tree tiles whose first place is in [from, to)
    const int u1 = to > seq.n_cache ? (to - seq.n_cache + kTreeWeight - 1) / kTreeWeight : 0;
    // Nearest keys first: the tree's tiles, then the cache's from the last one back, so that with a bias the running
    // maximum is there at once and what follows only falls.
    const int trees = max(u1 - u0, 0), tiles = trees + cache_tiles;
    const int last_tile = seq.tile0 + cache_from + cache_tiles - 1;
    const int T_b = seq.length;

    const int head0 = unit * p.heads_per_unit;
    const int cache_head = head0 / p.kv_group;
    const char* kbase = static_cast<const char*>(p.k) + ((PAGED ? 0 : b * p.k_stride[0]) + cache_head * p.k_stride[1]) * ES;
    const char* vbase = static_cast<const char*>(p.v) + ((PAGED ? 0 : b * p.v_stride[0]) + cache_head * p.v_stride[1]) * ES;
    const int32_t* table = PAGED ? p.table + b * p.table_stride : nullptr;

    // pages of the blocks of the next cache tile, requested when the one ahead of it goes out
    int page_of[kLoads], at0 = 0;
    auto look_up = [&](int tile) __attribute__((always_inline)) {
      if constexpr (PAGED) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int key = min(max(tile, 0) * kKeys + (i * 4 + wave) * RPB, p.cache_len - 1);
          page_of[i] = load_uniform(table + (key >> p.page_shift));
        }
      }
    };
    // Tile t of this pair goes out into stage t % 2. Cache tiles that lie in [lo, T) as a whole come in blocks; of
    // others every row is clamped to that range (or to the tree): data of keys that are left out below, and
    // nothing is read that no row may see.
    auto request_rows = [&](auto tree_c, int t, int key0, const char* kb_, const char* vb_, int64_t krow, int64_t vrow, int low, int last) __attribute__((always_inline)) {
      char* kst = smem + (t % kStages) * Tile::kBytes;
      char* vst = kst + kVRing;
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int blk = i * 4 + wave;
        const int j = min(max(key0 + blk * RPB + ld_row, low), last);
        int64_t koff = j * krow, voff = j * vrow;
        if constexpr (PAGED && !decltype(tree_c)::value) {
          const int64_t page = table[j >> p.page_shift];
          koff = page * k_page + (j & page_mask) * krow;
          voff = page * v_page + (j & page_mask) * vrow;
        }
        FTA_LOAD_BLOCK_TO_LDS(kb_ + koff + ld_chunk * 16, kst + blk * Tile::kBlockPitch);
        FTA_LOAD_BLOCK_TO_LDS(vb_ + voff + ld_chunk * 16, vst + blk * Tile::kBlockPitch);
      }
    };
    auto request_tree = [&](int t) __attribute__((always_inline)) {
      const auto* c = parameters_again(p);
      const int cur_head = unit * c->heads_per_unit / c->cur_group;
      request_rows(std::true_type{}, t, (u0 + t) * kKeys, static_cast<const char*>(c->ck) + (b * c->ck_stride[0] + cur_head * c->ck_stride[1]) * ES,
                   static_cast<const char*>(c->cv) + (b * c->cv_stride[0] + cur_head * c->cv_stride[1]) * ES, c->ck_stride[2] * ES, c->cv_stride[2] * ES, 0, L - 1);
    };
    // Where tile t's blocks come from and go to, if it is a cache tile that lies in [lo, T) as a whole.
    const char* ksrc;
    const char* vsrc;
    char* kst;
    auto blocks_of = [&](int t) __attribute__((always_inline)) {
      const int key0 = (last_tile - (t - trees)) * kKeys;
      const bool whole = t >= trees && t < tiles && key0 >= seq.lo && key0 + kKeys <= T_b;
      kst = smem + (t % kStages) * Tile::kBytes + wave * Tile::kBlockPitch;
      ksrc = kbase + k_lane;
      vsrc = vbase + v_lane;
      if constexpr (PAGED) {
        at0 = key0 + wave * RPB;
      } else if (whole) {
        ksrc += key0 * k_row;
        vsrc += key0 * v_row;
      }
      return whole;
    };
    // Load q of 2 * kLoads of them: K and V of this wave's blocks in turn.
    auto load_block = [&](auto q_c) __attribute__((always_inline)) {
      constexpr int Q = decltype(q_c)::value, i = Q / 2;
      constexpr bool is_v = Q % 2 != 0;
      const char* src = is_v ? vsrc : ksrc;
      if constexpr (PAGED) {
        const int at = (at0 + i * 4 * RPB) & page_mask;
        src += is_v ? page_of[i] * v_page + at * v_row : page_of[i] * k_page + at * k_row;
      } else {
        src += i * (is_v ? v_step : k_step);
      }
      FTA_LOAD_BLOCK_TO_LDS(src, kst + (is_v ? kVRing : 0) + i * 4 * Tile::kBlockPitch);
    };
    // Tile t in one go: the first of a pair, edges, tree tiles, and where the wave has no products to spread the loads over.
    auto request = [&](int t) __attribute__((always_inline)) {
      if (t < trees) {
        request_tree(t);
        return;
      }
      const int tile = last_tile - (t - trees);
      if (blocks_of(t)) unrolled<0, 2 * kLoads>(load_block);
      else request_rows(std::false_type{}, t, tile * kKeys, kbase, vbase, k_row, v_row, seq.lo, T_b - 1);
      look_up(tile - 1);
    };
    if (cache_tiles > 0) look_up(last_tile);
    if (tiles > 0) request(0);

    // ---- this lane's query row
    const int wave_row = row_block * kRowsPerWg + wave / WK * 32;
    const bool wave_active = wave_row < p.rows;
    const int row = wave_row + li;
    const bool row_ok = row < p.rows;
    const int head = head0 + (row_ok ? row / L : 0), qi = row_ok ? row % L : 0;
    u32x4 qf[KS];
    int depth = qi;
    float slope = 0.f;
    {
      const auto* c = parameters_again(p);
      if (c->depths) depth = max(c->depths[b * c->depth_stride + qi], 0);
      if (c->slopes) slope = c->slopes[head] * kLog2e;
      const char* qrow = static_cast<const char*>(c->q) + (b * c->q_stride[0] + head * c->q_stride[1] + qi * c->q_stride[2]) * ES + 16 * lh;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 raw = *reinterpret_cast<const u32x4*>(qrow + 32 * ks), zero = {0, 0, 0, 0};
        qf[ks] = row_ok ? raw : zero;
      }
    }
    const int pos = T_b + depth;
    const int row_lo = max(seq.first, p.window > 0 ? pos - p.window + 1 : 0);   // cache keys this row sees start here
    int wave_lo = row_lo;                                                          // the latest start of the wave's rows
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) wave_lo = max(wave_lo, __shfl_xor(wave_lo, o, 64));
    wave_lo = __builtin_amdgcn_readfirstlane(wave_lo);

    // Register r of block nb holds the score of key key0 + lane_key0 + key_of(nb, r), the last a constant (and not the
    // sum: the compiler would keep all of them in registers, being the same for every tile but for key0).
    const int lane_key0 = 32 * kb0 + 4 * lh;
    auto key_of = [](int nb, int r) __attribute__((always_inline)) { return 32 * nb + 8 * (r / 4) + r % 4; };

    // A tree tile's scores: the bias between the nodes, the mask, -inf for what the row does not see.
    auto tree_scores = [&](float (&s)[NB][16], int key0, int lane_key) __attribute__((always_inline)) {
      const auto* c = parameters_again(p);
      const int64_t mrow = b * c->mask_stride[0] + head * c->mask_stride[1] + qi * c->mask_stride[2];
      if (c->mask_packed) {   // a wave's keys of a tile lie in one word
        const uint64_t word = static_cast<const uint64_t*>(c->mask)[mrow + (min(lane_key, L - 1) >> 6)] >> (lane_key & 63);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[nb][r] = word >> key_of(nb, r) & 1 ? s[nb][r] : neg_inf();
      } else {
        const float* mrow_at = static_cast<const float*>(c->mask) + mrow;
        float mv[NB][16];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) mv[nb][r] = mrow_at[min(lane_key + key_of(nb, r), L - 1)];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            // finite mask values stay finite in units of log2 e: a row of nothing but the type's lowest value sees all
            // of its keys alike
            const float z = s[nb][r] + fmaxf(mv[nb][r] * kLog2e, -__FLT_MAX__);
            s[nb][r] = mv[nb][r] == neg_inf() ? neg_inf() : z;
          }
      }
      if (c->slopes || c->window > 0) {
        int key_depth = min(key0 + 32 * kb0 + lane % (32 * NB), L - 1);   // depths of the wave's keys, one per lane, handed round
        if (c->depths) key_depth = max(c->depths[b * c->depth_stride + key_depth], 0);
        const int window = c->window > 0 ? c->window : 0x7fffffff;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int d0 = __builtin_amdgcn_readlane(key_depth, key_of(nb, r)), d1 = __builtin_amdgcn_readlane(key_depth, key_of(nb, r) + 4);
            const int away = depth - (lh ? d1 : d0);
            const float z = __builtin_fmaf(-slope, static_cast<float>(away), s[nb][r]);
            s[nb][r] = away >= window ? neg_inf() : z;
          }
      }
      const int keys_left = L - lane_key;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[nb][r] = key_of(nb, r) < keys_left ? s[nb][r] : neg_inf();
    };
    // Value rows of a tree tile that no row of the workgroup sees (padding nodes) are zeroed in LDS: their weights
    // are 0, but 0 times an infinity or a NaN in them would not be. All waves must call it.
    auto clear_unseen = [&](const float (&s)[NB][16], char* vst) __attribute__((always_inline)) {
      if (tid < kKeys / 32) s_seen[tid] = 0;
      __syncthreads();
      if (wave_active) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          uint32_t bits = 0;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const uint64_t any = __builtin_amdgcn_ballot_w64(row_ok && s[nb][r] != neg_inf());
            bits |= (static_cast<uint32_t>(any) ? 1u << key_of(0, r) : 0u) | (any >> 32 ? 16u << key_of(0, r) : 0u);
          }
          if (lane == 0) atomicOr(&s_seen[kb0 + nb], bits);
        }
      }
      __syncthreads();
      constexpr int kChunks = D * ES / 16;
      for (int i = tid; i < kKeys * kChunks; i += 256) {
        const int key = i / kChunks;
        if (!(s_seen[key / 32] >> (key % 32) & 1)) *reinterpret_cast<u32x4*>(vst + Tile::at(key, i % kChunks)) = u32x4{0, 0, 0, 0};
      }
      __syncthreads();
    };

    f32x16 o[DB];
    float m_run = neg_inf(), l_run = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[db][r] = 0.f;

    for (int t = 0; t < tiles; ++t) {
      wait_vmcnt<0>();          // this wave's part of tile t has landed ...
      workgroup_barrier();      // ... and everybody's, and everybody is done with tile t - 1, whose stage tile t + 1 takes
      const bool tree = t < trees;
      const uint32_t stage = (t % kStages) * Tile::kBytes;
      const int key0 = (tree ? u0 + t : last_tile - (t - trees)) * kKeys;
      const int lane_key = key0 + lane_key0;
      bool idle = !wave_active && !tree;
      // A tile whose capped scores, lowered by their distance, are all more than 2^150 below the row's maximum has
      // weights of exactly 0 in 32 bits: nothing of it would be added.
      if (capped && sloped && !tree) {
        const float nearest = static_cast<float>(pos - key0 - (kKeys - 1)), farthest = static_cast<float>(pos - key0);
        idle = idle || !wave_any(row_ok && !(cap2 - fminf(slope * nearest, slope * farthest) < m_run + kNoWeight));
      }
      // The next tile's loads go out between the products: in one go they hold the wave for 900 to 1500 cycles a tile
      // (the CU takes a wave-wide load every 16), a third of its time; spread, they cost their issue.
      const bool spread = !idle && blocks_of(t + 1);
      if (!spread && t + 1 < tiles) request(t + 1);
      if (idle) continue;

      // ---- S^T = K Q^T, fragments requested a few products ahead
      float s[NB][16];
      {
        f32x16 acc[NB];
        constexpr int kFrags = KS * NB, kAhead = kFrags < 4 ? kFrags : 4;
        const uint32_t ka = k_rd + stage;
        u32x4 kf[kFrags];
        auto ask = [&](auto f) __attribute__((always_inline)) {
          constexpr int F = decltype(f)::value;
          kf[F] = lds_read_b128<(F % NB) * Tile::at(32, 0) + (F / NB) * 2 * Tile::kChunkStride>(ka);
        };
        matrix_phase(true);
        unrolled<0, kAhead>(ask);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[nb][r] = 0.f;
        unrolled<0, kFrags>([&](auto f) __attribute__((always_inline)) {
          constexpr int F = decltype(f)::value;
          wait_lgkm<(kFrags - 1 - F < kAhead - 1 ? kFrags - 1 - F : kAhead - 1)>(kf[F]);
          acc[F % NB] = mma_chunk<T>(kf[F], qf[F / NB], acc[F % NB]);
          if constexpr (F + kAhead < kFrags) ask(std::integral_constant<int, F + kAhead>{});
          constexpr int kFrom = F * 2 * kLoads / kFrags, kTo = (F + 1) * 2 * kLoads / kFrags;
          if constexpr (kTo > kFrom) {
            if (spread) unrolled<kFrom, kTo>(load_block);
            schedule_fence();
          }
        });
        if (spread) look_up(last_tile - (t + 1 - trees) - 1);
        matrix_phase(false);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[nb][r] = acc[nb][r];
      }

      // ---- z, relative to the running maximum: one multiply-add away from the products (or from the tanh), so that
      // 2^z needs no subtraction. A cache key's bias is linear in the constant part of its index.
      const bool whole_tile = !tree && key0 >= wave_lo && key0 + kKeys <= T_b;   // seen by every row of the wave
      const bool low = m_run < (t <= trees + 1 ? kLowMaximum : -__FLT_MAX__);   // (also where there is none yet)
      const float m_use = low ? 0.f : m_run;
      const float away = static_cast<float>(pos - lane_key);
      const float base = (capped && !SERIES ? cap2 : 0.f) - m_use - (tree ? 0.f : slope * away);
      auto shape = [&](auto capped_c, auto sloped_c) __attribute__((always_inline)) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            pin(s[nb][r]);
            float z;
            if constexpr (!decltype(capped_c)::value) z = __builtin_fmaf(c, s[nb][r], base);
            else if constexpr (SERIES) z = __builtin_fmaf(cap2, tanh_of(ex * s[nb][r]), base);
            else z = __builtin_fmaf(-2.f * cap2, fast_rcp(1.f + fast_exp2(ex * s[nb][r])), base);
            if constexpr (decltype(sloped_c)::value) z = __builtin_fmaf(slope, static_cast<float>(key_of(nb, r)), z);
            s[nb][r] = z;
          }
      };
      if (capped) {
        if (sloped && !tree) shape(std::true_type{}, std::true_type{}); else shape(std::true_type{}, std::false_type{});
      } else {
        if (sloped && !tree) shape(std::false_type{}, std::true_type{}); else shape(std::false_type{}, std::false_type{});
      }
      if (tree) {
        tree_scores(s, key0, lane_key);
        clear_unseen(s, smem + kVRing + stage);
        if (!wave_active) continue;
      } else if (!whole_tile) {
        const int from_key = row_lo - lane_key, keys_left = T_b - lane_key;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[nb][r] = key_of(nb, r) >= from_key && key_of(nb, r) < keys_left ? s[nb][r] : neg_inf();
      }
      float top = s[0][0];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[nb][r]);
      // The maximum (less the headroom) only has to keep the weights in range: it moves, and O and l are rescaled, when a
      // row has none yet or a low one, or its scores pass it by more than 8 (weights up to 2^8 times the headroom's).
      if (wave_any(top > (low ? neg_inf() : 8.f + kHeadroom<T>))) {
        const float m_new = fmaxf(m_run, m_use + half_swap_max(top, lh) - kHeadroom<T>);
        const float shift = m_new == neg_inf() ? 0.f : m_new - m_use;
        const float a = m_run == neg_inf() ? 1.f : fast_exp2(m_run - m_new);   // (l and O are 0 where there was no maximum)
        m_run = m_new;
        l_run *= a;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] *= a;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[nb][r] -= shift;
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[nb][r] = fast_exp2(s[nb][r]);

      // ---- O^T += V^T P^T
      const uint32_t va = v_rd + stage;
      if constexpr (kIs32<T>) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < 16; ++r) l_run += s[nb][r];
        constexpr int kSteps = NB * DB * 4;   // four keys of this half a step
        float vf[kSteps][4];
        auto ask = [&](auto g) __attribute__((always_inline)) {
          constexpr int G = decltype(g)::value, nb = G / (DB * 4), db = G / 4 % DB, rq = G % 4;
          constexpr int kOff = Tile::at(32 * nb + 8 * rq, 0) + db * 8 * Tile::kChunkStride;
          unrolled<0, 4>([&](auto e) __attribute__((always_inline)) {
            constexpr int E = decltype(e)::value;
            vf[G][E] = lds_read_b32<kOff + (Tile::at(E, 0))>(va);
          });
        };
        constexpr int kAhead = 2;
        unrolled<0, kAhead>(ask);
        unrolled<0, kSteps>([&](auto g) __attribute__((always_inline)) {
          constexpr int G = decltype(g)::value, nb = G / (DB * 4), db = G / 4 % DB, rq = G % 4;
          wait_lgkm<4 * (kSteps - 1 - G < kAhead - 1 ? kSteps - 1 - G : kAhead - 1)>(vf[G]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            o[db] = mma_f32(vf[G][e], s[nb][4 * rq + e], o[db]);
          }
          if constexpr (G + kAhead < kSteps) ask(std::integral_constant<int, G + kAhead>{});
        });
      } else {
        using M = Mfma<T>;
        typename M::Vec8 pf[2 * NB];
#pragma unroll
        for (int kk = 0; kk < 2 * NB; ++kk)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const f32x2 pair = {s[kk / 2][kk % 2 * 8 + e], s[kk / 2][kk % 2 * 8 + e + 1]};
            const auto rounded = __builtin_convertvector(pair, typename M::Vec2);
            // The weights enter the product in the type, as the values do: half a step each, which with l summing the
            // rounded ones moves the result by about as much as its own rounding does (0.0023 from the 64-bit result in
            // bf16, relative to its size, where rounding that result once is 0.0017). A second product of what they lose
            // would double the matrix unit's share of this half.
            l_run = M::add_pair(rounded, l_run);
            pf[kk][e] = rounded[0];
            pf[kk][e + 1] = rounded[1];
          }
        constexpr int kFrags = 2 * NB * DB, kAhead = kFrags < 4 ? kFrags : 4;
        constexpr int kRows8 = Tile::at(8, 0), kRows16 = Tile::at(16, 0);
        u32x2 vlo[kFrags], vhi[kFrags];
        auto ask = [&](auto g) __attribute__((always_inline)) {
          constexpr int G = decltype(g)::value, kOff = (G / DB) * kRows16 + (G % DB) * 4 * Tile::kChunkStride;
          vlo[G] = lds_read_tr16_b64<kOff>(va);
          vhi[G] = lds_read_tr16_b64<kOff + kRows8>(va);
        };
        matrix_phase(true);
        unrolled<0, kAhead>(ask);
        unrolled<0, kFrags>([&](auto g) __attribute__((always_inline)) {
          constexpr int G = decltype(g)::value;
          wait_lgkm<2 * (kFrags - 1 - G < kAhead - 1 ? kFrags - 1 - G : kAhead - 1)>(vlo[G], vhi[G]);
          const u32x4 raw_v = {vlo[G][0], vlo[G][1], vhi[G][0], vhi[G][1]};
          o[G % DB] = M::mma(__builtin_bit_cast(typename M::Vec8, raw_v), pf[G / DB], o[G % DB]);
          if constexpr (G + kAhead < kFrags) ask(std::integral_constant<int, G + kAhead>{});
        });
        matrix_phase(false);
      }
    }

    // ---- waves of the same rows: those behind the first park their states, the first takes them in
    bool writes = wave_active;
    if constexpr (WK > 1) {
      constexpr int kWords = 2 + 16 * DB;
      static_assert(4 * kWords * 64 * 4 <= 2 * kStages * Tile::kBytes, "the parked states fit the rings");
      float* park = reinterpret_cast<float*>(smem) + wave * kWords * 64 + lane;
      workgroup_barrier();   // the stages are done with
      if (wave % WK != 0 && wave_active) {
        park[0] = m_run;
        park[64] = l_run;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) park[(2 + db * 16 + r) * 64] = o[db][r];
      }
      __syncthreads();
      writes = wave_active && wave % WK == 0;
      if (writes) {
#pragma unroll
        for (int w = 1; w < WK; ++w) {
          const float* other = park + w * kWords * 64;
          const float m_other = other[0], m_both = fmaxf(m_run, m_other), m_use = m_both == neg_inf() ? 0.f : m_both;
          const float mine = fast_exp2(m_run - m_use), theirs = fast_exp2(m_other - m_use);
          l_run = l_run * mine + other[64] * theirs;
          m_run = m_both;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[db][r] = o[db][r] * mine + other[(2 + db * 16 + r) * 64] * theirs;
        }
      }
    }

    // ---- the result, or a partial
    if (writes) {
      const auto* c = parameters_again(p);
      const float l_all = half_swap_sum(l_run, lh);
      if (row_ok && complete) {
        const float inv = l_all > 0.f ? 1.f / l_all : 0.f;
        T* dst = static_cast<T*>(c->out) + b * c->out_stride[0] + head * c->out_stride[1] + qi * c->out_stride[2];
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int rg = 0; rg < 4; ++rg) {
            typedef __attribute__((ext_vector_type(4))) T Vec4;
            Vec4 v4;
#pragma unroll
            for (int e = 0; e < 4; ++e) v4[e] = static_cast<T>(o[db][rg * 4 + e] * inv);
            *reinterpret_cast<Vec4*>(dst + db * 32 + rg * 8 + 4 * lh) = v4;
          }
      } else if (row_ok) {
        const int slot = begin < x0 ? 0 : 1;
        float* part = c->partial + ((static_cast<int64_t>(row_block) * c->groups + group) * 2 + slot) * c->partial_floats;
        const int local = row - row_block * kRowsPerWg;
        float* dst = part + static_cast<int64_t>(local) * D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int rg = 0; rg < 4; ++rg) {
            const f32x4 v4 = {o[db][rg * 4], o[db][rg * 4 + 1], o[db][rg * 4 + 2], o[db][rg * 4 + 3]};
            *reinterpret_cast<f32x4*>(dst + db * 32 + rg * 8 + 4 * lh) = v4;
          }
        if (lh == 0) {
          part[c->rows_cap * D + 2 * local] = m_run;
          part[c->rows_cap * D + 2 * local + 1] = l_all;
        }
      }
    }

    // ---- the next pair of the stretch
    x = begin + to;
    if (x >= x1) break;
    begin += seq.n;
    if (++unit == p.units) {
      unit = 0;
      ++b;
      seq = sequence_of<kKeys>(p, b);
    }
    __syncthreads();   // the stages (and the parked states) are free
  }
}

// Joins the partials of the pairs that were cut. One workgroup per few rows of a pair, four columns a thread; the
// partials of up to kTogether stretches are in flight together (they come from other XCDs' workgroups, so every
// one is a round trip to memory).
template <typename T, int D, int WK>
__global__ void __launch_bounds__(256) shaped_join_kernel(const ShapedParams p) {
  constexpr int kKeys = kTileKeys<T, WK>, kRowsPerWg = 128 / WK, kRowsPerBlock = 256 / (D / 4), kTogether = 8;
  const int per_pair = (p.rows + kRowsPerBlock - 1) / kRowsPerBlock;
  const int pair = blockIdx.x / per_pair;
  const int unit = pair % p.units;
  const int row = (blockIdx.x % per_pair) * kRowsPerBlock + threadIdx.x / (D / 4), d = threadIdx.x % (D / 4) * 4;
  const Place here = place_of<kKeys>(p, true, [&](int) { return pair / p.units; });
  const Stretches cut = cut_line(p, here.total);
  const int begin = here.begin + unit * here.seq.n;
  const int g0 = cut.holder(begin), g1 = cut.holder(begin + here.seq.n - 1);
  if (g0 == g1 || row >= p.rows) return;
  const int row_block = row / kRowsPerWg, local = row % kRowsPerWg;
  const int64_t stats = static_cast<int64_t>(p.rows_cap) * D + 2 * local, values = static_cast<int64_t>(local) * D + d;
  float m = neg_inf(), l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int g = g0; g <= g1; g += kTogether) {
    f32x2 ml[kTogether];
    f32x4 o[kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      if (g + i > g1) continue;
      const float* part = p.partial + ((static_cast<int64_t>(row_block) * p.groups + g + i) * 2 + (begin < cut.start(g + i) ? 0 : 1)) * p.partial_floats;
      ml[i] = *reinterpret_cast<const f32x2*>(part + stats);
      o[i] = *reinterpret_cast<const f32x4*>(part + values);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kTogether; ++i)
      if (g + i <= g1) top = fmaxf(top, ml[i][0]);
    if (top == neg_inf()) continue;
    const float keep = fast_exp2(m - top);
    m = top;
    l *= keep;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= keep;
#pragma unroll
    for (int i = 0; i < kTogether; ++i) {
      if (g + i > g1) continue;
      const float w = fast_exp2(ml[i][0] - top);
      l += w * ml[i][1];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += w * o[i][e];
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int head = unit * p.heads_per_unit + row / p.q_len, i = row % p.q_len;
  typedef __attribute__((ext_vector_type(4))) T Vec4;
  Vec4 v4;
#pragma unroll
  for (int e = 0; e < 4; ++e) v4[e] = static_cast<T>(acc[e] * inv);
  *reinterpret_cast<Vec4*>(static_cast<T*>(p.out) + here.b * p.out_stride[0] + head * p.out_stride[1] + i * p.out_stride[2] + d) = v4;
}

// ---------------------------------------------------------------------------------------------- host
struct Cut {
  int key_waves, rows_per_wg, row_blocks, heads_per_unit, units, rows, groups, whole, rows_cap, tree_tiles, lead_groups, lead_share;
  int64_t partial_floats, bytes;
};

int cut_of(const fta_shaped_args& a, int num_cus, Cut* out) {
  if (num_cus <= 0) num_cus = kDefaultCUs;
  Cut c{};
  const bool is32 = a.dtype == FTA_F32;
  c.heads_per_unit = a.cur_heads == a.num_kv_heads ? a.num_q_heads / a.num_kv_heads : 1;
  c.units = a.num_q_heads / c.heads_per_unit;
  const int64_t rows = static_cast<int64_t>(c.heads_per_unit) * a.q_len;
  if (rows > 1 << 24) return FTA_ERR_SHAPE;
  c.rows = static_cast<int>(rows);
  // Units of up to 64 rows: two waves per 32 rows, so that all four compute. f32 tiles take four times the memory and
  // eight times the matrix unit's cycles a key, and few rows leave most of the waves idle: up to 32 rows take four
  // waves where the stages fit LDS.
  c.key_waves = c.rows > 64 || (is32 && a.head_dim > 128) ? 1 : is32 && c.rows <= 32 && a.head_dim <= 64 ? 4 : 2;
  const int keys = is32 ? 32 * c.key_waves : 64;
  c.rows_per_wg = 128 / c.key_waves;
  c.row_blocks = (c.rows + c.rows_per_wg - 1) / c.rows_per_wg;
  c.tree_tiles = (a.q_len + keys - 1) / keys;
  const int64_t cap = a.max_seq_len_hint > 0 ? std::min(a.max_seq_len_hint, a.cache_len) : a.cache_len;
  int64_t cap_tiles = (cap + keys - 1) / keys;
  if (a.window > 0) cap_tiles = std::min<int64_t>(cap_tiles, a.window / keys + 2);
  const int64_t pairs = static_cast<int64_t>(a.bsz) * c.units;
  const int64_t line = pairs * ((a.cache_len + keys - 1) / keys + 1 + static_cast<int64_t>(kTreeWeight) * c.tree_tiles);
  if (line > 0x3fffffff || pairs * c.row_blocks > 0x3fffffff) return FTA_ERR_SHAPE;
  // (an f32 tile of more than 16 KiB leaves room for one workgroup)
  const int per_cu = a.head_dim > 128 || (is32 && keys * a.head_dim > 4096) ? 1 : 2;
  c.whole = cap_tiles <= 2 * kMinStretch;
  c.groups = c.whole ? static_cast<int>(pairs) : std::max(1, num_cus * per_cu / c.row_blocks);
  c.rows_cap = std::min(c.rows, c.rows_per_wg);
  // Where a CU holds two workgroups, the one that came first has the older waves, which the scheduler serves first:
  // with a cap and a bias it takes 2.7 us a tile, the other one 3.3, and equal stretches leave the CU half empty at
  // the end. The first half of the stretches gets 57 % of the line: 64 sequences up to 32768 keys, 64 heads on 8,
  // 16 nodes 820 us against 851, 8 x 32768, 32 on 8, 64 nodes 371 against 395, head_dim 64 169 against 176. With a
  // cap or a bias alone it is even (268 against 265) or loses (258 against 244), and is not done.
  c.lead_groups = c.lead_share = 0;
  if (!c.whole && per_cu == 2 && !is32 && c.key_waves == 1 && a.softcap > 0.f && a.slopes && c.groups >= 2) {
    c.lead_groups = c.groups / 2;
    c.lead_share = 584;
  }
  c.partial_floats = (static_cast<int64_t>(c.rows_cap) * (a.head_dim + 2) + 3) / 4 * 4;
  c.bytes = c.whole ? 0 : static_cast<int64_t>(c.row_blocks) * c.groups * 2 * c.partial_floats * 4;
  *out = c;
  return FTA_OK;
}

int validate_sizes(const fta_shaped_args& a) {
  if (a.dtype != FTA_F32 && a.dtype != FTA_F16 && a.dtype != FTA_BF16) return FTA_ERR_DTYPE;
  if (a.len_dtype != FTA_I32 && a.len_dtype != FTA_I64) return FTA_ERR_DTYPE;
  if (a.mask_kind != FTA_MASK_ADDITIVE_F32 && a.mask_kind != FTA_MASK_PACKED_U64) return FTA_ERR_DTYPE;
  if (a.head_dim != 32 && a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return FTA_ERR_HEAD_DIM;
  if (a.bsz <= 0 || a.num_q_heads <= 0 || a.num_kv_heads <= 0 || a.q_len <= 0 || a.cache_len < 0 || a.max_seq_len_hint < 0 || a.window < 0)
    return FTA_ERR_SHAPE;
  if (a.num_q_heads % a.num_kv_heads != 0) return FTA_ERR_SHAPE;
  if (a.cur_heads != a.num_kv_heads && a.cur_heads != a.num_q_heads) return FTA_ERR_SHAPE;
  if (!(a.softcap >= 0.f) || !std::isfinite(kLog2e * a.softcap) || !std::isfinite(kLog2e * a.sm_scale)) return FTA_ERR_UNSUPPORTED;
  if (a.softcap > 0.f && !std::isfinite(2.f * kLog2e * a.sm_scale / a.softcap)) return FTA_ERR_UNSUPPORTED;   // the tanh's argument
  return FTA_OK;
}

int validate(const fta_shaped_args& a) {
  if (int st = validate_sizes(a)) return st;
  if (!a.q || !a.k_cache || !a.v_cache || !a.cur_k || !a.cur_v || !a.mask || !a.kv_seq_len || !a.out) return FTA_ERR_NULL_POINTER;
  if (a.block_table) {
    if (a.page_size != 16 && a.page_size != 32 && a.page_size != 64 && a.page_size != 128) return FTA_ERR_BLOCK_SIZE;
    if (a.block_table_stride < 0 || a.cache_len == 0 || a.block_table_stride * a.page_size < a.cache_len) return FTA_ERR_SHAPE;
  }
  const int es = a.dtype == FTA_F32 ? 4 : 2, vec = 16 / es;
  const int64_t* strides[] = {a.q_stride, a.k_stride, a.v_stride, a.ck_stride, a.cv_stride, a.out_stride};
  for (const int64_t* s : strides)
    for (int i = 0; i < 3; ++i)
      if (s[i] < 0 || s[i] % vec) return FTA_ERR_STRIDE;
  for (const void* ptr : {a.q, a.k_cache, a.v_cache, a.cur_k, a.cur_v, static_cast<const void*>(a.out)})
    if (reinterpret_cast<uintptr_t>(ptr) % 16) return FTA_ERR_STRIDE;
  for (int i = 0; i < 3; ++i)
    if (a.mask_stride[i] < 0) return FTA_ERR_STRIDE;
  if (a.depth_stride < 0) return FTA_ERR_STRIDE;
  if (reinterpret_cast<uintptr_t>(a.mask) % (a.mask_kind == FTA_MASK_PACKED_U64 ? 8 : 4)) return FTA_ERR_STRIDE;
  // a block's rows are addressed with 32-bit lane offsets
  if (a.k_stride[2] * es * 16 > 0x7fffffffLL || a.v_stride[2] * es * 16 > 0x7fffffffLL) return FTA_ERR_UNSUPPORTED;
  return FTA_OK;
}

template <typename T, int D, int WK, bool PAGED, bool SERIES>
int launch_form(const ShapedParams& p, hipStream_t stream) {
  constexpr int kSmem = kLdsBytes<T, D, WK>;
  static_assert(kSmem <= 160 * 1024 / (D <= 128 && D * kTileKeys<T, WK> * sizeof(T) <= 16384 ? 2 : 1), "LDS budget");
  auto kern = shaped_kernel<T, D, WK, PAGED, SERIES>;
  if (kSmem > 64 * 1024) {   // once per kernel and device
    static thread_local int configured_device = -1;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return FTA_ERR_NO_DEVICE;
    if (configured_device != dev) {
      if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, kSmem) != hipSuccess) return FTA_ERR_LAUNCH;
      configured_device = dev;
    }
  }
  if (int st = launch_checked(kern, dim3(static_cast<unsigned>(p.groups * p.row_blocks)), dim3(256), kSmem, stream, p)) return st;
  if (p.whole) return FTA_OK;
  constexpr int kRowsPerBlock = 256 / (D / 4);
  const int64_t grid = static_cast<int64_t>(p.bsz) * p.units * ((p.rows + kRowsPerBlock - 1) / kRowsPerBlock);
  if (grid > 0x7fffffffLL) return FTA_ERR_SHAPE;
  return launch_checked(shaped_join_kernel<T, D, WK>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, p);
}

template <typename T, int D, int WK, bool PAGED>
int launch(const ShapedParams& p, hipStream_t stream) {
  if constexpr (!kIs32<T>) {
    if (p.softcap <= kShortCap) return launch_form<T, D, WK, PAGED, false>(p, stream);
  }
  return launch_form<T, D, WK, PAGED, true>(p, stream);
}

template <typename T, int D>
int launch_d(const ShapedParams& p, const Cut& c, hipStream_t stream) {
  if constexpr (kIs32<T> && D <= 64) {
    if (c.key_waves == 4) return p.table ? launch<T, D, 4, true>(p, stream) : launch<T, D, 4, false>(p, stream);
  }
  if constexpr (!kIs32<T> || D <= 128) {
    if (c.key_waves == 2) return p.table ? launch<T, D, 2, true>(p, stream) : launch<T, D, 2, false>(p, stream);
  }
  return p.table ? launch<T, D, 1, true>(p, stream) : launch<T, D, 1, false>(p, stream);
}

template <typename T>
int launch_t(const ShapedParams& p, int head_dim, const Cut& c, hipStream_t stream) {
  switch (head_dim) {
    case 32: return launch_d<T, 32>(p, c, stream);
    case 64: return launch_d<T, 64>(p, c, stream);
    case 128: return launch_d<T, 128>(p, c, stream);
    default: return launch_d<T, 256>(p, c, stream);
  }
}

}  // namespace
}  // namespace fta

extern "C" {

int fta_shaped_workspace(const fta_shaped_args* args, int num_cus, int64_t* bytes) {
  if (!args || !bytes) return FTA_ERR_NULL_POINTER;
  if (int st = fta::validate_sizes(*args)) return st;
  fta::Cut c;
  if (int st = fta::cut_of(*args, num_cus, &c)) return st;
  *bytes = c.bytes;
  return FTA_OK;
}

int fta_shaped_decode(const fta_shaped_args* args, void* hip_stream) {
  using namespace fta;
  if (!args) return FTA_ERR_NULL_POINTER;
  const fta_shaped_args& a = *args;
  if (int st = validate(a)) return st;
  static thread_local int cached_device = -1, cached_cus = 0;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return FTA_ERR_NO_DEVICE;
  if (dev != cached_device) {
    if (hipDeviceGetAttribute(&cached_cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return FTA_ERR_NO_DEVICE;
    cached_device = dev;
  }
  Cut c;
  if (int st = cut_of(a, cached_cus, &c)) return st;
  if (c.bytes > 0) {
    if (!a.workspace) return FTA_ERR_NULL_POINTER;
    if (a.workspace_bytes < c.bytes) return FTA_ERR_SCRATCH_TOO_SMALL;
    if (reinterpret_cast<uintptr_t>(a.workspace) % 16) return FTA_ERR_STRIDE;
  }
  ShapedParams p{};
  p.q = a.q; p.k = a.k_cache; p.v = a.v_cache; p.ck = a.cur_k; p.cv = a.cur_v; p.mask = a.mask; p.lens = a.kv_seq_len; p.out = a.out;
  p.table = a.block_table; p.slopes = a.slopes; p.first = a.first_key; p.depths = a.depths;
  p.partial = static_cast<float*>(a.workspace);
  p.bsz = a.bsz; p.num_q_heads = a.num_q_heads; p.q_len = a.q_len; p.cache_len = a.cache_len;
  p.heads_per_unit = c.heads_per_unit; p.units = c.units;
  p.kv_group = a.num_q_heads / a.num_kv_heads; p.cur_group = a.num_q_heads / a.cur_heads;
  p.rows = c.rows; p.row_blocks = c.row_blocks; p.groups = c.groups; p.tree_tiles = c.tree_tiles; p.whole = c.whole; p.rows_cap = c.rows_cap;
  p.lead_groups = c.lead_groups; p.lead_share = c.lead_share;
  p.len_is_i64 = a.len_dtype == FTA_I64; p.mask_packed = a.mask_kind == FTA_MASK_PACKED_U64;
  p.page_shift = a.page_size == 16 ? 4 : a.page_size == 32 ? 5 : a.page_size == 64 ? 6 : 7;
  p.window = a.window; p.scale = a.sm_scale; p.softcap = a.softcap;
  p.partial_floats = c.partial_floats;
  for (int i = 0; i < 3; ++i) {
    p.q_stride[i] = a.q_stride[i]; p.k_stride[i] = a.k_stride[i]; p.v_stride[i] = a.v_stride[i]; p.ck_stride[i] = a.ck_stride[i];
    p.cv_stride[i] = a.cv_stride[i]; p.mask_stride[i] = a.mask_stride[i]; p.out_stride[i] = a.out_stride[i];
  }
  p.table_stride = a.block_table_stride; p.depth_stride = a.depth_stride;
  hipStream_t stream = static_cast<hipStream_t>(hip_stream);
  if (a.dtype == FTA_F32) return launch_t<float>(p, a.head_dim, c, stream);
  if (a.dtype == FTA_F16) return launch_t<_Float16>(p, a.head_dim, c, stream);
  return launch_t<__bf16>(p, a.head_dim, c, stream);
}

}  // extern "C"
