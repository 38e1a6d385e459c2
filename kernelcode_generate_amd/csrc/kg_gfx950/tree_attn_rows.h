// Attention over a paged cache (tree_attn.h) for few rows per request and key head: decoding steps and small
// trees. A row is a (token, query head) of the key head's group, so a step of four query heads per key
// head fills a quarter of a 16-row matrix block and reads each key once for all four.
//
// Such a call is bound by reading keys and values. As in flash_attn_decode.h each of a workgroup's four waves
// walks its own steps of 32 or 64 keys with its own running maximum and sums: S^T = K Q^T (v_mfma_f32_16x16x32, operand A
// 16 keys x 32 d from K's rows, operand B the 16 rows), P in registers straight to O^T += V^T P^T, no LDS until the end.
// (A second block of rows per wave took twice the registers: more rows go through shared tiles, tree_attn_tiles.h.)
//
// Work is shared out in rounds (one step of each wave) of all requests, heads and blocks of rows in one line, an
// equal range of it to each workgroup whatever the requests' lengths, which only the device knows: each
// workgroup sums the requests' rounds by itself. A range that covers an item (request, head, block of rows) writes
// its rows; others leave O, maximum and sum in 32 bits, and tree_attn_join_kernel joins them in
// the order of the ranges.
//
// 8-bit caches: codes are widened to 16 bits (exact for both types) for the products; a key's scale multiplies
// its scores, a value's its weights. Weights are rounded to 16 bits with that scale in them, so the running
// maximum is of s + log2(value's scale): weights of at most 2^8, whatever the scales' sizes. The sum of weights, which has no scales
// in it, stays in 32 bits, so the scale that counts there lies within 2^-80..2^80 (ValueScale).
//
// Weights of 16-bit caches are rounded to 16 bits, as in the flash attention kernels, and summed as rounded. The matrix instructions
// take them in the values' type: a second product with what rounding leaves would double that half of the work, for an error
// of half a step a weight, which the output's own rounding has too.
#pragma once

#include <type_traits>

#include "common.h"
#include "flash_attn_mfma.h"
#include "kv_cache.h"
#include "tree_attn.h"

namespace kg_gfx950 {

namespace treer {
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr float kMinMax = -3.0e38f;  // the lowest running maximum: scores of -inf weigh nothing beside it
// The running maximum (log2 units) is raised by scores beyond it by more than this: weights are at most 2^8, and sums
// are rescaled a few times and not at every other tile. Weights and their sum have the same maximum, so the result does not depend on it.
constexpr float kSlack = 8.f;
// keys of a wave's step: 16 KiB of K and V rows, or what the registers hold (8 KiB of 8-bit heads of 64;
// 32 KiB of 16-bit heads of 256)
template <typename C, int D>
constexpr int step_keys() { return (sizeof(C) == 2 && D >= 128) || D == 256 ? 32 : 64; }

// A 16-bit pair of two 8-bit codes.
template <typename Tag, typename C>
struct Widen;
template <>
struct Widen<Bf16Tag, E4m3> {
  template <bool kHigh>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, float ratio = 1.f) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, ratio, kHigh));
  }
};
template <>
struct Widen<F16Tag, E4m3> {
  template <bool kHigh>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, float ratio = 1.f) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, ratio, kHigh));
  }
};
template <typename Tag>
struct Widen<Tag, int8_t> {
  template <bool kHigh>
  static __device__ __forceinline__ uint32_t pair(uint32_t w, float ratio = 1.f) {
    const int a = (int)(w << (kHigh ? 8 : 24)) >> 24, b = (int)(w << (kHigh ? 0 : 16)) >> 24;
    return Half16<Tag>::pack2((float)a * ratio, (float)b * ratio);
  }
};
// 8 codes to 8 16-bit elements, times a ValueScale's ratio
template <typename Tag, typename C>
__device__ __forceinline__ u32x4 widen8(uint32_t lo, uint32_t hi, float ratio = 1.f) {
  using W = Widen<Tag, C>;
  if constexpr (std::is_same<C, E4m3>::value) {  // (the conversion takes the power of two)
    const uint32_t sign = (uint32_t)((int)__builtin_bit_cast(uint32_t, ratio) >> 31) & 0x80808080u;
    lo ^= sign, hi ^= sign;
    ratio = __builtin_fabsf(ratio);
  }
  return u32x4{W::template pair<false>(lo, ratio), W::template pair<true>(lo, ratio), W::template pair<false>(hi, ratio),
               W::template pair<true>(hi, ratio)};
}

// a lane's columns of a V row
template <int kDwords, typename C>
__device__ __forceinline__ void load_v(uint32_t (&v)[kDwords], const C* p) {
  if constexpr (kDwords == 1) {
    v[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (kDwords == 2) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(p);
    v[0] = x[0], v[1] = x[1];
  } else {
#pragma unroll
    for (int q = 0; q < kDwords; q += 4) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(p) + 4 * q);
      v[q] = x[0], v[q + 1] = x[1], v[q + 2] = x[2], v[q + 3] = x[3];
    }
  }
}

// A value's scale, of any sign and size. What counts for the running maximum is its magnitude with an exponent within -79..80 (`log`
// its logarithm): a sum of weights is then 2^-80..2^88 for each of up to 2^31 keys, with 46 bits or more below it that 32 bits hold.
// What is left goes to the value or its weight in 16 bits, without loss: `ratio`, the sign and a power of two, 1 of scales that are
// not odd, 0 of a scale of 0, and within 2^-69..2^48, which bf16 holds. In fp16 a ratio ends at 2^7, so that what it multiplies
// stays finite: the result is infinite with it as without, unless that key's weight is below some 2^-70.
template <typename Tag>
struct ValueScale {
  float log, ratio;
  static __device__ __forceinline__ bool odd(float scale) { return !(scale >= 0x1p-80f && scale <= 0x1p79f); }
  explicit __device__ __forceinline__ ValueScale(float scale) {
    const int exponent = scale == 0.f ? -126 : __builtin_amdgcn_frexp_expf(scale), within = max(min(exponent, 80), -79), left = exponent - within;
    // a mantissa within 0.5..1, also of 0; an infinity or NaN passes: the rows that see the value are NaN
    const float mantissa = nan_max(__builtin_fabsf(__builtin_amdgcn_frexp_mantf(scale)), 0.5f);
    log = __builtin_amdgcn_logf(__builtin_ldexpf(mantissa, within));
    ratio = __builtin_ldexpf(scale == 0.f ? 0.f : __builtin_copysignf(1.f, scale), std::is_same<Tag, F16Tag>::value ? min(left, 7) : left);
  }
};

template <typename C>
constexpr bool kScaled = CacheElem<C>::kScaled;
template <>
inline constexpr bool kScaled<uint16_t> = false;
}  // namespace treer

// A workgroup's share of the work: `units` of request b are its items times their rounds.
struct TreeShare {
  int w;            // the workgroup's place among those that have work
  int first, last;  // [first, last) of all units
  int b, base;      // the request that `first` lies in, and the units before it
  int total;
};
constexpr int kTreePad = 4;  // of a record's rows: maximum and sum, on 16-byte rows
struct TreeSplit {
  int grid;       // workgroups the units are shared among
  int block;      // rows of an item
  int round;      // keys of a round; 0: items are not split, a unit is an item
  float* partial; // 2 grid records of `block` rows x (width + kTreePad): O, maximum (log2 units), sum
  int width;
};
__device__ __forceinline__ int tree_rounds(const TreeRequest& r, int round) {
  return round == 0 ? 1 : max((r.keys + round - 1) / round, 1);
}
__device__ __forceinline__ int tree_blocks(const TreeRequest& r, int group, int block) {
  return (r.count * group + block - 1) / block;
}
__device__ __forceinline__ int tree_units(const TreeArgs& a, const TreeSplit& s, int b) {
  if (b >= a.batch) return 0;
  const TreeRequest r = tree_request(a, b);
  return r.count == 0 ? 0 : a.heads * tree_blocks(r, a.group, s.block) * tree_rounds(r, s.round);
}
// Sums of units, up to the most there are where `starts` ascend: others than that may repeat the tokens, and their requests
// past the limit have no units (a request's own are below it by the host's checks).
constexpr int kTreeMostUnits = 1 << 30;
__device__ __forceinline__ int tree_sum(int a, int b) { return (int)min((uint32_t)a + (uint32_t)b, (uint32_t)kTreeMostUnits); }
__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(v, o, 64);
    if (lane >= o) v = tree_sum(v, x);
  }
  return v;
}
// Workgroup w of those that have work takes the units from bound(w) up to bound(w + 1), at least one.
__device__ __forceinline__ int share_bound(int w, const TreeSplit& s, int total) {
  const int grid = min(s.grid, total);
  if (w >= grid) return total;
  if (total <= 1 << 22) return (int)((uint32_t)w * (uint32_t)total / (uint32_t)grid);  // (grids have at most 512)
  return (int)((long long)w * total / grid);
}
// The workgroup whose range holds unit u.
__device__ __forceinline__ int share_of(int u, const TreeSplit& s, int total) {
  const int grid = min(s.grid, total);
  if (total <= 1 << 22) return (int)((((uint32_t)u + 1) * (uint32_t)grid - 1) / (uint32_t)total);
  return (int)((((long long)u + 1) * grid - 1) / total);
}

// Workgroups go to the 8 XCDs in turn; neighbouring shares to the same XCD, whose L2 has the keys that they read for other rows or
// one request (e4m3, 16 requests behind 4096: 38.5 -> 36 us; 2 x 512 rows: no change).
__device__ __forceinline__ TreeShare tree_share(const TreeArgs& a, const TreeSplit& s, int id) {
  const int lane = threadIdx.x & 63;
  TreeShare t;
  t.total = 0;
  const int mine = tree_units(a, s, lane);
  const int upto = wave_scan(mine, lane);
  t.total = __builtin_amdgcn_readlane(upto, 63);
  for (int b0 = 64; b0 < a.batch; b0 += 64)
    t.total = tree_sum(t.total, __builtin_amdgcn_readlane(wave_scan(tree_units(a, s, b0 + lane), lane), 63));
  const int eighth = min(s.grid, t.total) >> 3;
  t.w = id < 8 * eighth ? (id & 7) * eighth + (id >> 3) : id;
  t.first = share_bound(t.w, s, t.total);
  t.last = share_bound(t.w + 1, s, t.total);
  // the first request that ends behind `first`
  t.b = a.batch;
  t.base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int own = b0 == 0 ? mine : tree_units(a, s, b0 + lane);
    const int end = tree_sum(t.base, b0 == 0 ? upto : wave_scan(own, lane));
    const unsigned long long behind = __builtin_amdgcn_ballot_w64(end > t.first);
    if (behind != 0) {
      const int x = __builtin_ctzll(behind);
      t.b = b0 + x;
      t.base = __builtin_amdgcn_readlane(end, x) - __builtin_amdgcn_readlane(own, x);
      break;
    }
    t.base = __builtin_amdgcn_readlane(end, 63);
  }
  return t;
}

// Keys key + 0..63 that a row sees of those there are (bit n: key + n), its token j of the request, whose mask begins with
// `first`. At once for a tile: a loop over the keys took 18 us of 176 at 2 x 512 tokens behind 4096.
__device__ __forceinline__ unsigned long long tree_visible(const TreeArgs& a, const TreeRequest& r, bool row, int j,
                                                           unsigned long long first, int key) {
  const int before = r.context - key;  // the first of them are the context's
  if (before >= 64) return ~0ull;
  const int draft = max(-before, 0);  // the next one's number
  unsigned long long seen = 0;
  if (a.words < 0) {
    const int n = j + 1 - draft;
    if (n > 0) seen = n >= 64 ? ~0ull : (1ull << n) - 1;
  } else {
    const int w = draft >> 6, shift = draft & 63;
    auto word = [&](int i) __attribute__((always_inline)) {
      if (i == 0) return first;
      return row && i < a.words ? (unsigned long long)a.mask[(r.first + j) * a.mask_0 + i * a.mask_1] : 0ull;
    };
    seen = word(w) >> shift;
    if (shift != 0) seen |= word(w + 1) << (64 - shift);
  }
  return before <= 0 ? seen : seen << before | ((1ull << before) - 1);
}
// Of those the ones that exist and lie with this lane: bit 4 kb + i is key 16 kb + 4 lr + i.
template <int NKB>
__device__ __forceinline__ uint32_t tree_lane_keys(unsigned long long keys, int lr) {
  uint32_t bits = 0;
#pragma unroll
  for (int kb = 0; kb < NKB; ++kb) bits |= ((uint32_t)(keys >> (16 * kb) >> (4 * lr)) & 0xfu) << (4 * kb);
  return bits;
}

// A weight of 0 does not take an infinity or NaN out of a sum, and only some rows see a drafted token: where values are
// not finite, the products run on zeros in their place and this adds them to the rows that see them (times a
// weight they would be the same). One key of a step after another, from memory: row l16's elements d_of(e, i).
// seen: bit 4 (n / 16) + n % 4 of the lane of row l16 and keys 4 (l / 16) + 0..3 is key n's.
template <typename Tag, typename C, int kKeys, int NE, typename DOf>
__device__ __forceinline__ void tree_add_nonfinite(const TreeArgs& a, f32x4 (&o)[NE], uint32_t seen, int page, int offset, int h,
                                                   int lane, DOf d_of) {
#pragma unroll 1
  for (int n = 0; n < kKeys; ++n) {
    const int at_page = __shfl(page, n, 64), at_offset = __shfl(offset, n, 64);
    const uint32_t bits = (uint32_t)__shfl((int)seen, 16 * ((n & 15) >> 2) + (lane & 15), 64);
    if (at_page < 0 || !(bits >> (4 * (n >> 4) + (n & 3)) & 1u)) continue;
    const C* v = static_cast<const C*>(a.v) + at_page * a.v_page + h * a.v_head + at_offset * a.v_row;
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = d_of(e, i);
        if (d >= a.d) continue;
        float x;
        if constexpr (sizeof(C) == 1) x = CacheElem<C>::load(v + d);
        else x = Half16<Tag>::to_float(v[d]);
        if (!__builtin_isfinite(x)) o[e][i] += x;
      }
  }
}

// C: uint16_t (elements of Tag), E4m3 or int8_t. D: 64, 128 or 256, heads of d <= D elements, d % 16 == 0. Pages of a
// multiple of 16 tokens, so that 16 keys share one.
template <typename Tag, typename C, int D>
__global__ __launch_bounds__(treer::kThreads, D == 256 ? 1 : 2) void tree_attn_rows_kernel(TreeArgs a, TreeSplit split) {
  using namespace treer;
  using H = Half16<Tag>;
  constexpr bool kS = kScaled<C>;
  constexpr int kES = sizeof(C);
  constexpr int kStep = step_keys<C, D>();
  constexpr int NC = kStep / 32, NKB = kStep / 16;  // chunks of 32, blocks of 16 keys
  constexpr int NDS = D / 32;                       // 32-deep steps of S^T
  constexpr int NE = D / 16;                        // columns of V per lane, blocks of O^T
  constexpr int kRows = 16;
  constexpr int NKW = kS ? D / 64 : NDS;            // 16-byte pieces of a K row per lane
  constexpr int NVW = NE * kES / 4;                 // dwords of a V row per lane
  __shared__ float o_lds[kWaves][kRows][D];
  __shared__ float ml_lds[kWaves][kRows][2];
  __shared__ __attribute__((aligned(16))) float sc_lds[kS ? kWaves : 1][3][kStep];

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lr = lane >> 4;

  TreeShare share = tree_share(a, split, blockIdx.x);
  const int own_first = share.first;

  while (share.first < share.last && share.b < a.batch) {
    const TreeRequest r = tree_request(a, share.b);
    const int rounds = tree_rounds(r, split.round), blocks = tree_blocks(r, a.group, kRows);
    const int units = r.count == 0 ? 0 : a.heads * blocks * rounds;
    const int local = share.first - share.base;
    if (local >= units) {
      share.base = tree_sum(share.base, units);
      ++share.b;
      continue;
    }
    const int item = local / rounds, round0 = local - item * rounds;
    const int round1 = min(rounds, round0 + share.last - share.first);
    const int h = item / blocks, row0 = (item - h * blocks) * kRows;
    const bool whole_item = round0 == 0 && round1 == rounds;
    const int item_rows = min(r.count * a.group - row0, kRows);
    const bool starts_here = share.first == own_first;
    share.first += round1 - round0;

    // keys of this range; of a chain only those that its last token sees
    constexpr int kRound = kStep * kWaves;
    int key_lo = split.round == 0 ? 0 : round0 * kRound;
    int key_hi = split.round == 0 ? r.keys : min(r.keys, round1 * kRound);
    if (a.words < 0) key_hi = (int)min((long long)key_hi, (long long)r.context + (row0 + item_rows - 1) / a.group + 1);
    key_lo = __builtin_amdgcn_readfirstlane(key_lo);
    key_hi = __builtin_amdgcn_readfirstlane(key_hi);

    // this lane's rows: token of the request and query head
    u32x4 qf[NDS];
    const int row = row0 + l16, tok = row / a.group;
    const bool real = l16 < item_rows;
    const unsigned long long first_word =  // of the token's mask
        real && a.words > 0 ? (unsigned long long)a.mask[(long long)(r.first + tok) * a.mask_0] : 0ull;
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (real ? r.first + tok : 0) * a.q_token +
                        ((long long)h * a.group + (row - tok * a.group)) * a.q_head;
#pragma unroll
    for (int s = 0; s < NDS; ++s) {
      // 8-bit rows: 16 bytes of a lane are the 8 d of two steps
      const int d = kS ? 64 * (s >> 1) + 16 * lr + 8 * (s & 1) : 32 * s + 8 * lr;
      qf[s] = real && d < a.d ? ld16(q + d) : u32x4{0, 0, 0, 0};
    }
    const C* kc = static_cast<const C*>(a.k) + h * a.k_head;
    const C* vc = static_cast<const C*>(a.v) + h * a.v_head;
    const float* k_scale = kS ? a.k_scale + h * a.ks_head : nullptr;
    const float* v_scale = kS ? a.v_scale + h * a.vs_head : nullptr;
    const int* table = a.table + share.b * a.table_0;

    // Page of key `lane` of a step (-1: none, or a key past the range) and its offset there.
    struct Place {
      int page, offset;
    };
    auto place = [&](int key0) __attribute__((always_inline)) {
      const int key = key0 + (lane & (kStep - 1));
      Place p = {-1, 0};
      if (key < key_hi) {
        const int n = div_page(key, a.div);
        p.page = table[n * a.table_1];
        p.offset = key - n * a.page_size;
      }
      return p;
    };
    auto checked = [&](Place p) __attribute__((always_inline)) {
      const bool there = p.page >= 0 && p.page < a.pages;
      return Place{there ? p.page : -1, there ? p.offset : 0};
    };

    // Rows of a step. What is not there is read from page 0 instead, whose rows exist, and dropped later.
    u32x4 k[NKB][NKW];
    uint32_t v[NC][8][NVW];
    float ks = 0.f, vs = 0.f;  // of key `lane` of the step
    auto load_k = [&](const Place& p) __attribute__((always_inline)) {
      if constexpr (kS) {
        ks = k_scale[tree_row(max(p.page, 0), p.offset, a.ks_page, a.ks_row)];
        vs = v_scale[tree_row(max(p.page, 0), p.offset, a.vs_page, a.vs_row)];
      }
      // (a lane's d past the head's end: its first ones)
      auto piece = [&](const C* row, int kb, int s) __attribute__((always_inline)) {
        const int d = (kS ? 16 : 8) * lr + (kS ? 64 : 32) * s;
        k[kb][s] = ld16(row + (d < a.d ? d : 0));
      };
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {  // 16 keys on one page
        const int page = __builtin_amdgcn_readlane(p.page, 16 * kb), offset = __builtin_amdgcn_readlane(p.offset, 16 * kb);
        const C* row = kc + ((long long)max(page, 0) * a.k_page + (long long)offset * a.k_row);
#pragma unroll
        for (int s = 0; s < NKW; ++s) piece(row + (uint32_t)(l16 * (int)a.k_row), kb, s);
      }
    };
    const int v_col = NE * l16 < a.d ? NE * l16 : 0;
    auto load_v_rows = [&](const Place& p) __attribute__((always_inline)) {
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        const int page = __builtin_amdgcn_readlane(p.page, 16 * kb), offset = __builtin_amdgcn_readlane(p.offset, 16 * kb);
        const C* row = vc + ((long long)max(page, 0) * a.v_page + (long long)offset * a.v_row);
#pragma unroll
        for (int x = 0; x < 4; ++x) load_v(v[kb >> 1][(kb & 1) * 4 + x], row + (uint32_t)((4 * lr + x) * (int)a.v_row + v_col));
      }
    };

    f32x4 o[NE];
    f32x4 l_run = {0.f, 0.f, 0.f, 0.f};  // scaled caches: element 0, this lane's keys alone
    float m_run = kMinMax;
#pragma unroll
    for (int e = 0; e < NE; ++e) o[e] = f32x4{0.f, 0.f, 0.f, 0.f};
    const u32x4 ones = {H::kOnePair, H::kOnePair, H::kOnePair, H::kOnePair};

    // This wave's steps: key_lo + kStep (wave + 4 i). A step reads its rows and waits for them; eight to twelve waves of a CU
    // keep it reading (kept across steps, the rows took twice the registers in copies). The next step's pages are
    // looked up ahead of the rows, since loads return in order.
    constexpr int kStride = kStep * kWaves;
    int key = key_lo + kStep * wave;
    Place p = checked(place(key));
#pragma unroll 1
    for (; key < key_hi; key += kStride) {
      const Place next = place(key + kStride);
      load_k(p);
      load_v_rows(p);
      // plain: a step of the context, every key of it there; `there`: bits of those that are
      const unsigned long long there = __builtin_amdgcn_ballot_w64(p.page >= 0);
      const bool plain = ~there == 0 && key + kStep <= r.context;
      // ---- scores in log2 units; lane: row l16, keys 16 kb + 4 lr + i ----
      if (a.d != D) {
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int s = 0; s < NKW; ++s)
            if ((kS ? 16 : 8) * lr + (kS ? 64 : 32) * s >= a.d) k[kb][s] = u32x4{0, 0, 0, 0};
      }
      f32x4 sc[NKB], y[NKB];  // y: with the values' scales
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        sc[kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NDS; ++s) {
          u32x4 kf;
          if constexpr (kS) kf = widen8<Tag, C>(k[kb][s >> 1][(s & 1) * 2], k[kb][s >> 1][(s & 1) * 2 + 1]);
          else kf = k[kb][s];
          sc[kb] = H::mfma16(kf, qf[s], sc[kb]);
        }
      }
      bool odd = false;  // whether there are values with a ratio
      if constexpr (kS) {
        sc_lds[wave][0][lane & (kStep - 1)] = ks * a.scale_log2;
        sc_lds[wave][1][lane & (kStep - 1)] = __builtin_amdgcn_logf(vs);
        odd = __builtin_amdgcn_ballot_w64(ValueScale<Tag>::odd(vs)) != 0;
        if (odd) {
          const ValueScale<Tag> scale(vs);
          sc_lds[wave][1][lane & (kStep - 1)] = scale.log;
          sc_lds[wave][2][lane & (kStep - 1)] = scale.ratio;
        }
      }
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        f32x4 f = {a.scale_log2, a.scale_log2, a.scale_log2, a.scale_log2}, lv;
        if constexpr (kS) {
          f = *reinterpret_cast<const f32x4*>(&sc_lds[wave][0][16 * kb + 4 * lr]);
          lv = *reinterpret_cast<const f32x4*>(&sc_lds[wave][1][16 * kb + 4 * lr]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[kb][i] *= f[i];
          if constexpr (kS) y[kb][i] = sc[kb][i] + lv[i];
        }
      }
      // ---- what is not seen ----
      uint32_t seen, found = 0;  // bit 4 kb + i: this lane's row sees its key
      if (!plain) {
        const uint32_t there_lo = (uint32_t)(there >> (4 * lr)), there_hi = (uint32_t)(there >> 32 >> (4 * lr));
        seen = tree_lane_keys<NKB>(there & tree_visible(a, r, l16 < item_rows, tok, first_word, key), lr);
#pragma unroll
        for (int n = 0; n < 4 * NKB; ++n)
          if (!(seen >> n & 1u)) {
            sc[n >> 2][n & 3] = -INFINITY;
            if constexpr (kS) y[n >> 2][n & 3] = -INFINITY;
          }
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int n = 0; n < 8; ++n) {
            const int in_step = 32 * c + (n < 4 ? n : 12 + n);
            const bool here = ((in_step < 32 ? there_lo : there_hi) >> (in_step & 31) & 1u) != 0;
#pragma unroll
            for (int q = 0; q < NVW; ++q) {
              uint32_t w = here ? v[c][n][q] : 0;
              if constexpr (!kS) {
                w = finite_pair<H>(w, found);
              } else if constexpr (std::is_same<C, E4m3>::value) {  // NaN: all ones below the sign
                const uint32_t bad = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                found |= bad;
                w &= ~((bad >> 7) * 0xffu);
              }
              v[c][n][q] = w;
            }
          }
      }
      // ---- weights: keys 32 c + 4 lr + 0..3, then + 16 ----
      u32x4 pp[NC];
      auto weighed = [&](int n) __attribute__((always_inline)) {
        if constexpr (kS) return (float)y[n >> 2][n & 3];
        else return (float)sc[n >> 2][n & 3];
      };
      float mx = weighed(0);
#pragma unroll
      for (int n = 1; n < 4 * NKB; ++n) mx = nan_max(mx, weighed(n));
      float mx2 = mx;
      fa::rows4_combine<true>(mx, mx2);
      const bool raise = !(mx <= m_run + kSlack);  // (a NaN too)
      if (__builtin_amdgcn_ballot_w64(raise)) {
        const float alpha = raise ? __builtin_amdgcn_exp2f(m_run - mx) : 1.f;
        m_run = raise ? mx : m_run;
        l_run *= alpha;
#pragma unroll
        for (int e = 0; e < NE; ++e) o[e] *= alpha;
      }
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = __builtin_amdgcn_exp2f(weighed(4 * kb + i) - m_run);
          if constexpr (kS) l_run[0] += __builtin_amdgcn_exp2f((float)sc[kb][i] - m_run);
        }
        pp[kb >> 1][(kb & 1) * 2] = H::pack2(w[0], w[1]);
        pp[kb >> 1][(kb & 1) * 2 + 1] = H::pack2(w[2], w[3]);
      }
      if constexpr (!kS) {
#pragma unroll
        for (int c = 0; c < NC; ++c) l_run = H::mfma16(ones, pp[c], l_run);
      }
      if constexpr (kS) {
        if (odd) {
#pragma unroll
          for (int kb = 0; kb < NKB; ++kb) {
            const f32x4 ratio = *reinterpret_cast<const f32x4*>(&sc_lds[wave][2][16 * kb + 4 * lr]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t p2 = pp[kb >> 1][(kb & 1) * 2 + i];
              pp[kb >> 1][(kb & 1) * 2 + i] =
                  H::pack2(H::to_float(p2 & 0xffffu) * ratio[2 * i], H::to_float(p2 >> 16) * ratio[2 * i + 1]);
            }
          }
        }
      }
      // ---- O^T += V^T P^T ----
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint32_t row16[8][NE / 2];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
          for (int q = 0; q < NE / 2; ++q) {
            if constexpr (kS)
              row16[n][q] = (q & 1) ? Widen<Tag, C>::template pair<true>(v[c][n][q >> 1])
                                    : Widen<Tag, C>::template pair<false>(v[c][n][q >> 1]);
            else row16[n][q] = v[c][n][q];
          }
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          u32x4 vt;  // column e of this lane's 8 rows
#pragma unroll
          for (int q = 0; q < 4; ++q)
            vt[q] = (e & 1) ? hi_halves(row16[2 * q][e >> 1], row16[2 * q + 1][e >> 1])
                            : lo_halves(row16[2 * q][e >> 1], row16[2 * q + 1][e >> 1]);
          o[e] = H::mfma16(vt, pp[c], o[e]);
        }
      }
      if (!plain && __builtin_amdgcn_ballot_w64(found != 0) != 0)
        tree_add_nonfinite<Tag, C, kStep>(a, o, seen, p.page, p.offset, h, lane, [&](int e, int i) { return NE * (4 * lr + i) + e; });
      p = checked(next);
    }

    // ---- join the waves ----
    if constexpr (kS) {
      float l0 = l_run[0], l1 = l0;
      fa::rows4_combine<false>(l0, l1);
      l_run[0] = l0;
    }
#pragma unroll
    for (int e = 0; e < NE; ++e)
#pragma unroll
      for (int i = 0; i < 4; ++i) o_lds[wave][l16][NE * (4 * lr + i) + e] = o[e][i];
    if (lr == 0) {
      ml_lds[wave][l16][0] = m_run;
      ml_lds[wave][l16][1] = l_run[0];
    }
    __syncthreads();
    float* record = split.partial + ((long long)2 * share.w + (starts_here ? 0 : 1)) * kRows * (D + kTreePad);
    for (int y = tid; y < item_rows * (D / 2); y += kThreads) {
      const int n = y / (D / 2), d = 2 * (y - n * (D / 2));
      if (d >= a.d) continue;
      float m = ml_lds[0][n][0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) m = nan_max(m, ml_lds[w][n][0]);
      float l = 0.f, v0 = 0.f, v1 = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(ml_lds[w][n][0] - m);
        l += f * ml_lds[w][n][1];
        v0 += f * o_lds[w][n][d];
        v1 += f * o_lds[w][n][d + 1];
      }
      if (whole_item) {
        const int row = row0 + n, token = row / a.group;
        const float inv = l != 0.f ? 1.f / l : 0.f;
        uint16_t* out = static_cast<uint16_t*>(a.out) + (r.first + token) * a.o_token +
                        ((long long)h * a.group + (row - token * a.group)) * a.o_head + d;
        *reinterpret_cast<uint32_t*>(out) = H::pack2(l != 0.f ? v0 * inv : 0.f, l != 0.f ? v1 * inv : 0.f);
      } else {
        float* p = record + (long long)n * (D + kTreePad);
        *reinterpret_cast<f32x2*>(p + d) = f32x2{v0, v1};
        if (d == 0) *reinterpret_cast<f32x2*>(p + D) = f32x2{m, l};
      }
    }
    __syncthreads();
  }
}

// The records of the items that several ranges share, joined: a wave takes four consecutive rows of an item, a lane four
// columns. (A wave per row spent most of its time on finding its item: 14 us for 3104 rows of 8 records each, 8 now.)
// kWaves: more where few rows have many records, which take every kWaves-th record of the same rows (32 rows of 64 records: 34 us
// with one wave each, 13 with four, 9 with 16; 512 rows of 4: 6.2, 4.7 with four; 4096 rows of 8: 8.2, 6.5; 34816 rows of 2: 11 with one).
constexpr int kTreeJoinRows = 4;
__host__ __device__ constexpr int tree_join_waves(int waves) { return waves > 4 ? waves : 4; }  // of a workgroup
template <typename Tag, int D, int kWaves>
__global__ __launch_bounds__(64 * tree_join_waves(kWaves)) void tree_attn_join_kernel(TreeArgs a, TreeSplit split) {
  constexpr int kLanes = D / 4, kAtOnce = 64 / kLanes;                    // lanes of a row, rows of a load
  constexpr int kLoads = kTreeJoinRows / kAtOnce < 1 ? 1 : kTreeJoinRows / kAtOnce;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int turn = wave % kWaves;
  constexpr int kAll = tree_join_waves(kWaves);
  const long long id = (long long)blockIdx.x * (kAll / kWaves) + wave / kWaves;
  const int parts = split.block / kTreeJoinRows;
  const int item = (int)(id / parts), part = (int)(id - (long long)item * parts);
  // the request of this item, the items and units before it, and all units
  int owner = -1, items = 0, base = 0, total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int b = b0 + lane;
    int own_items = 0, own_units = 0;
    if (b < a.batch) {
      const TreeRequest r = tree_request(a, b);
      own_items = r.count == 0 ? 0 : a.heads * tree_blocks(r, a.group, split.block);
      own_units = own_items * tree_rounds(r, split.round);
    }
    const int upto_items = wave_scan(own_items, lane), upto = wave_scan(own_units, lane);
    if (owner < 0) {
      const unsigned long long behind = __builtin_amdgcn_ballot_w64(tree_sum(items, upto_items) > item);
      if (behind != 0) {
        const int x = __builtin_ctzll(behind);
        owner = b0 + x;
        items = tree_sum(items, __builtin_amdgcn_readlane(upto_items, x)) - __builtin_amdgcn_readlane(own_items, x);
        base = tree_sum(total, __builtin_amdgcn_readlane(upto, x)) - __builtin_amdgcn_readlane(own_units, x);
      } else {
        items = tree_sum(items, __builtin_amdgcn_readlane(upto_items, 63));
      }
    }
    total = tree_sum(total, __builtin_amdgcn_readlane(upto, 63));
  }
  if (owner < 0) return;
  const TreeRequest r = tree_request(a, owner);
  const int rounds = tree_rounds(r, split.round), blocks = tree_blocks(r, a.group, split.block);
  const int begin = base + (item - items) * rounds;
  const int w0 = share_of(begin, split, total), w1 = share_of(begin + rounds - 1, split, total);
  if (w0 >= w1) return;  // one range: its rows are written
  const int h = (item - items) / blocks, row0 = ((item - items) - h * blocks) * split.block + part * kTreeJoinRows;
  const int item_rows = r.count * a.group - row0;  // from this wave's first row on
  if (item_rows <= 0) return;
  // an item that begins inside a workgroup's range is that workgroup's second record
  const int first_slot = 2 * w0 + (share_bound(w0, split, total) >= begin ? 0 : 1);
  const long long pitch = (long long)split.block * (D + kTreePad);
  const int sub = lane / kLanes, col = 4 * (lane % kLanes);
  const float* rows = split.partial + (long long)(part * kTreeJoinRows + sub) * (D + kTreePad);
  float m[kLoads], l[kLoads];
  f32x4 o[kLoads];
#pragma unroll
  for (int x = 0; x < kLoads; ++x) {
    m[x] = treer::kMinMax;
    l[x] = 0.f;
    o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  constexpr int kAhead = kWaves == 4 ? 8 : 4;
  for (int v0 = w0 + turn; v0 <= w1; v0 += kWaves * kAhead) {
    f32x4 ov[kAhead][kLoads];
    f32x2 ml[kAhead][kLoads];
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      const int w = min(v0 + kWaves * y, w1);
      const float* rec = rows + (w == w0 ? first_slot : 2 * w) * pitch;
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {  // (rows past the item's are in the record's bounds)
        ov[y][x] = *reinterpret_cast<const f32x4*>(rec + x * kAtOnce * (D + kTreePad) + col);
        ml[y][x] = *reinterpret_cast<const f32x2*>(rec + x * kAtOnce * (D + kTreePad) + D);
      }
    }
#pragma unroll
    for (int y = 0; y < kAhead; ++y) {
      if (v0 + kWaves * y > w1) break;
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        const float m_new = nan_max(m[x], ml[y][x][0]);
        const float f = __builtin_amdgcn_exp2f(m[x] - m_new), g = __builtin_amdgcn_exp2f(ml[y][x][0] - m_new);
        m[x] = m_new;
        l[x] = l[x] * f + ml[y][x][1] * g;
        o[x] = o[x] * f + ov[y][x] * g;
      }
    }
  }
  if constexpr (kWaves > 1) {  // (all waves of a group are here: what they returned on is the same for them)
    __shared__ f32x4 o_lds[kAll][kLoads][64];
    __shared__ f32x2 ml_lds[kAll][kLoads][64];
#pragma unroll
    for (int x = 0; x < kLoads; ++x) o_lds[wave][x][lane] = o[x], ml_lds[wave][x][lane] = f32x2{m[x], l[x]};
    __syncthreads();
    if (turn != 0) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
#pragma unroll
      for (int x = 0; x < kLoads; ++x) {
        const f32x2 ml = ml_lds[wave + w][x][lane];
        const float m_new = nan_max(m[x], ml[0]);
        const float f = __builtin_amdgcn_exp2f(m[x] - m_new), g = __builtin_amdgcn_exp2f(ml[0] - m_new);
        m[x] = m_new;
        l[x] = l[x] * f + ml[1] * g;
        o[x] = o[x] * f + o_lds[wave + w][x][lane] * g;
      }
  }
#pragma unroll
  for (int x = 0; x < kLoads; ++x) {
    const int n = x * kAtOnce + sub;
    if (n >= item_rows || n >= kTreeJoinRows || col >= a.d) continue;
    const int row = row0 + n, token = row / a.group;
    const float inv = l[x] != 0.f ? 1.f / l[x] : 0.f;
    uint16_t* out = static_cast<uint16_t*>(a.out) + (r.first + token) * a.o_token +
                    ((long long)h * a.group + (row - token * a.group)) * a.o_head + col;
    u32x2 w = {0, 0};
    if (l[x] != 0.f)
      w = u32x2{Half16<Tag>::pack2(o[x][0] * inv, o[x][1] * inv), Half16<Tag>::pack2(o[x][2] * inv, o[x][3] * inv)};
    *reinterpret_cast<uint32_t*>(out) = w[0];
    *reinterpret_cast<uint32_t*>(out + 2) = w[1];
  }
}

}  // namespace kg_gfx950
