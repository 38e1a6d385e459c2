// Attention over a paged cache (tree_attn.h) for many rows per request and key head: trees of drafted tokens,
// pieces of prompts; and for pages of no multiple of 16 tokens.
//
// Sharing of the work, weights, scales and joining are those of tree_attn_rows.h. Here the four waves of a workgroup take
// different rows (16 or 32 each) and the same keys: tiles of 64 (32 for heads of 256) in one of two LDS stages as 16-bit
// [key][d], the next one on its way under the current one's products, with one barrier per tile. 16-bit rows are copied there by the
// loads; 8-bit codes go through registers, where they are widened once for all rows. K fragments are one ds_read_b128 per 16 keys x 32 d
// (16-byte chunk c of row r at c ^ (r % 16): 16 rows hit distinct banks), V^T fragments two ds_read_b64_tr_b16 per 16 d x 32
// keys in the key order that P's lanes hold (chunk pairs at pair ^ (r % 8): the 8 rows of half a wave do).
//
// Measured, heads of 128 in 8 groups of 4: 2 x 512 rows behind 4096 in bf16 127 us a call with the join, 575 TFLOP/s (740
// behind 16384); with rows through registers, which spilled, and a loop over the keys of tiles with drafts, 185. Two waves a SIMD
// issue vector instructions for 3000 of the 6500 cycles that two tiles of 128 rows take, MFMAs fill 2200, reads of LDS 2000: a
// tile's scores taken under the exponentials of the one before (33 registers more, spilled) took 151. 8 x 16 rows behind
// 16384: bf16 115 us, 4.7 TB/s of rows; e4m3 94-98 us, bound by each wave's chain of widening, products and softmax, not by bytes (two
// tiles in flight: 6 % longer; eight waves with half the keys each, in 128 registers: 56 %).
#pragma once

#include "common.h"
#include "flash_attn_mfma.h"
#include "kv_cache.h"
#include "lds_dma.h"
#include "tree_attn.h"
#include "tree_attn_rows.h"

namespace kg_gfx950 {

namespace treet {
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
template <int D>
constexpr int tile_keys() { return D == 256 ? 32 : 64; }
// byte address of 16-byte chunk c of row r within a [rows][D] 16-bit tile
template <int D>
__device__ __forceinline__ uint32_t k_at(int r, int c) {
  return r * D * 2 + 16 * (D == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & 15));
}
template <int D>
__device__ __forceinline__ uint32_t v_at(int r, int c) {
  return r * D * 2 + 16 * (D == 64 ? c ^ (2 * ((r >> 1) & 3)) : c ^ (2 * (r & 7)));
}
// A query pair for scores that are multiplied by |scale|, or 1 where scale is 0: their products are -1 or 0 times
// those of the pair (0 times what is not finite: NaN). A positive factor leaves the largest score the largest.
template <typename H>
__device__ __forceinline__ uint32_t with_sign(uint32_t w, float scale) {
  uint32_t bad = 0;
  if (scale == 0.f) {
    const uint32_t finite = finite_pair<H>(w, bad);
    return (w ^ finite) | (bad >> 15);
  }
  return scale < 0.f ? w ^ 0x80008000u : w;
}
__device__ const char kZeros[512] = {};  // the row of a key that is not there
}  // namespace treet

template <typename Tag, typename C, int D, int kNQ>
__global__ __launch_bounds__(treet::kThreads, 2) void tree_attn_tiles_kernel(TreeArgs a, TreeSplit split) {
  using namespace treet;
  using treer::kMinMax;
  using treer::kSlack;
  using Scale = treer::ValueScale<Tag>;
  using H = Half16<Tag>;
  constexpr bool kS = treer::kScaled<C>;
  constexpr int kES = sizeof(C);
  constexpr int kTile = tile_keys<D>();
  constexpr int NC = kTile / 32, NKB = kTile / 16;
  constexpr int NDS = D / 32, NE = D / 16;
  constexpr int kWaveRows = 16 * kNQ, kRows = kWaves * kWaveRows;
  constexpr int kPerRow = D * kES / 16;              // 16-byte pieces of a row
  constexpr int kPieces = kTile * kPerRow / kThreads;  // of a thread, K and V each
  constexpr int kRowStep = kThreads / kPerRow;       // rows between a thread's pieces
  constexpr int kStage = kTile * D * 2;              // bytes of one tile
  __shared__ __attribute__((aligned(1024))) char lds[4 * kStage];  // K, V of stage 0, K, V of stage 1
  __shared__ __attribute__((aligned(16))) float sc_lds[kS ? 2 : 1][2][kTile];
  __shared__ int found_lds[3];  // whether tile t has values that are not finite, at t % 3

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lr = lane >> 4;
  const uint32_t lds0 = lds_addr(lds);
  const int piece_row = tid / kPerRow, piece = tid % kPerRow;
  const bool piece_in = piece * 16 / kES < a.d;

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

    int key_lo = split.round == 0 ? 0 : round0 * kTile;
    int key_hi = split.round == 0 ? r.keys : min(r.keys, round1 * kTile);
    if (a.words < 0) key_hi = (int)min((long long)key_hi, (long long)r.context + (row0 + item_rows - 1) / a.group + 1);
    key_lo = __builtin_amdgcn_readfirstlane(key_lo);
    key_hi = __builtin_amdgcn_readfirstlane(key_hi);

    // this wave's rows: lane l16 of block x
    const int wave_rows = min(item_rows - wave * kWaveRows, kWaveRows);  // (may be none)
    int tok[kNQ];
    unsigned long long first_word[kNQ];
    u32x4 qf[kNQ][NDS];
#pragma unroll
    for (int x = 0; x < kNQ; ++x) {
      const bool real = 16 * x + l16 < wave_rows;
      const int row = row0 + wave * kWaveRows + 16 * x + l16;
      tok[x] = row / a.group;
      first_word[x] = real && a.words > 0 ? (unsigned long long)a.mask[(long long)(r.first + tok[x]) * a.mask_0] : 0ull;
      const uint16_t* q = static_cast<const uint16_t*>(a.q) + (real ? r.first + tok[x] : 0) * a.q_token +
                          ((long long)h * a.group + (row - tok[x] * a.group)) * a.q_head;
#pragma unroll
      for (int s = 0; s < NDS; ++s) qf[x][s] = real && 32 * s + 8 * lr < a.d ? ld16(q + 32 * s + 8 * lr) : u32x4{0, 0, 0, 0};
      if constexpr (!kS)
#pragma unroll
        for (int s = 0; s < NDS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) qf[x][s][i] = treet::with_sign<H>(qf[x][s][i], a.scale_log2);
    }
    const float scale = a.scale_log2 == 0.f ? 1.f : __builtin_fabsf(a.scale_log2);
    const C* kc = static_cast<const C*>(a.k) + h * a.k_head;
    const C* vc = static_cast<const C*>(a.v) + h * a.v_head;
    const float* k_scale = kS ? a.k_scale + h * a.ks_head : nullptr;
    const float* v_scale = kS ? a.v_scale + h * a.vs_head : nullptr;
    const int* table = a.table + share.b * a.table_0;

    // Page of key `lane` of a tile (-1: none, or a key past the range), its offset there, and its rows: a lane's 64-bit
    // products for its key and not for each piece it copies (158 -> 146 us at 2 x 512 rows behind 4096).
    struct Place {
      int page, offset;
      unsigned long long k, v;
    };
    auto place = [&](int first) __attribute__((always_inline)) {
      const int key = first + (lane & (kTile - 1)), n = div_page(max(min(key, key_hi - 1), 0), a.div);
      Place p = {table[n * a.table_1], key - n * a.page_size, 0, 0};
      if (key >= key_hi) p.page = -1;
      return p;
    };
    auto checked = [&](Place p) __attribute__((always_inline)) {
      const bool there = p.page >= 0 && p.page < a.pages;
      const unsigned long long k = (unsigned long long)(kc + tree_row(p.page, p.offset, a.k_page, a.k_row));
      const unsigned long long v = (unsigned long long)(vc + tree_row(p.page, p.offset, a.v_page, a.v_row));
      const unsigned long long zeros = (unsigned long long)&kZeros;
      return Place{there ? p.page : -1, there ? p.offset : 0, there ? k : zeros, there ? v : zeros};
    };
    auto row_of = [&](unsigned long long p, int n) __attribute__((always_inline)) {  // key n's
      return (unsigned long long)(uint32_t)__shfl((int)(p >> 32), n, 64) << 32 | (uint32_t)__shfl((int)p, n, 64);
    };

    // 16-bit rows: copied to LDS by the load itself, a wave's 1 KiB at a time; d past the head's end comes from kZeros.
    // Lane l's 16 bytes land at 16 l, so it takes the chunk that the swizzle puts there.
    auto copy = [&](int stage, const Place& p) __attribute__((always_inline)) {
      const uint32_t kb = lds0 + stage * 2 * kStage + wave * 1024, vb = kb + kStage;
      auto pieces = [&](auto padded) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int n = piece_row + kRowStep * i;
          const uint32_t ck = k_at<D>(n, piece) - n * D * 2, cv = v_at<D>(n, piece) - n * D * 2;  // bytes in the row
          unsigned long long k = row_of(p.k, n), v = row_of(p.v, n);
          if constexpr (decltype(padded)::value != 0) {
            const unsigned long long zeros = (unsigned long long)&kZeros;
            k = (int)ck < 2 * a.d ? k : zeros;
            v = (int)cv < 2 * a.d ? v : zeros;
          }
          g2lds16_m(reinterpret_cast<const char*>(k + ck), kb + i * kThreads * 16);
          g2lds16_m(reinterpret_cast<const char*>(v + cv), vb + i * kThreads * 16);
        }
      };
      if (a.d == D) pieces(Int<0>{});
      else pieces(Int<1>{});
    };
    // A tile that not every row sees in full: values that are not finite are left out of the products (tree_add_nonfinite).
    auto sift = [&](int stage, int at) __attribute__((always_inline)) {
      uint32_t found = 0;
#pragma unroll
      for (int i = 0; i < kStage / (kThreads * 16); ++i) {
        const auto to = (__attribute__((address_space(3))) u32x4*)(uintptr_t)(lds0 + (2 * stage + 1) * kStage + (i * kThreads + tid) * 16);
        u32x4 x = *to;
#pragma unroll
        for (int q = 0; q < 4; ++q) x[q] = finite_pair<H>(x[q], found);
        *to = x;
      }
      if (found != 0) found_lds[at] = 1;
    };

    // 8-bit rows: through registers, where they are widened. What is not there is read from a row that is, and written as
    // zeros.
    u32x4 kr[kPieces], vr[kPieces];
    uint32_t row_there = 0;
    float ks = 0.f, vs = 0.f;
    auto load = [&](const Place& p) __attribute__((always_inline)) {
      row_there = 0;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int n = piece_row + kRowStep * i;
        const int page = __shfl(p.page, n, 64), offset = __shfl(p.offset, n, 64);
        row_there |= (page >= 0 ? 1u : 0u) << i;
        const int d = piece_in ? piece * 16 : 0;
        kr[i] = ld16(kc + tree_row(max(page, 0), offset, a.k_page, a.k_row) + d);
        vr[i] = ld16(vc + tree_row(max(page, 0), offset, a.v_page, a.v_row) + d);
      }
      if constexpr (kS) {
        ks = k_scale[tree_row(max(p.page, 0), p.offset, a.ks_page, a.ks_row)];
        vs = v_scale[tree_row(max(p.page, 0), p.offset, a.vs_page, a.vs_row)];
      }
    };
    auto put = [&](uint32_t at, u32x4 x) __attribute__((always_inline)) {
      *(__attribute__((address_space(3))) u32x4*)(uintptr_t)at = x;
    };
    auto store = [&](int stage, const Place& p) __attribute__((always_inline)) {
      const uint32_t kb = lds0 + stage * 2 * kStage, vb = kb + kStage;
      // heed: there are scales that are odd, whose ratio goes to the values. Two copies of the stores, since what the ratio takes in one
      // costs every tile (2 x 512 rows over e4m3 behind 4096: 156 us as without it, 163 in one copy, 193 on the weights; 8 x 16 rows
      // behind 16384: 94, 96, 94, without 90).
      auto pieces = [&](auto heed) __attribute__((always_inline)) {
        constexpr bool kHeed = decltype(heed)::value != 0;
        const float ratio = kHeed ? Scale(vs).ratio : 1.f;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int n = piece_row + kRowStep * i;
          const bool there = piece_in && (row_there >> i & 1u);
          const u32x4 k = there ? kr[i] : u32x4{0, 0, 0, 0}, v = there ? vr[i] : u32x4{0, 0, 0, 0};
          if constexpr (kS) {
            put(kb + k_at<D>(n, 2 * piece), treer::widen8<Tag, C>(k[0], k[1]));
            put(kb + k_at<D>(n, 2 * piece + 1), treer::widen8<Tag, C>(k[2], k[3]));
            const float to = kHeed ? __shfl(ratio, n, 64) : 1.f;  // (a wave has the scales of all keys)
            put(vb + v_at<D>(n, 2 * piece), treer::widen8<Tag, C>(v[0], v[1], to));
            put(vb + v_at<D>(n, 2 * piece + 1), treer::widen8<Tag, C>(v[2], v[3], to));
          }
        }
        if (tid < kTile) {
          sc_lds[stage][0][tid] = p.page >= 0 ? ks * a.scale_log2 : 0.f;
          sc_lds[stage][1][tid] = p.page >= 0 ? (kHeed ? Scale(vs).log : __builtin_amdgcn_logf(vs)) : 0.f;
        }
      };
      if (__builtin_amdgcn_ballot_w64(p.page >= 0 && Scale::odd(vs)) == 0) pieces(Int<0>{});
      else pieces(Int<1>{});
    };

    f32x4 o[kNQ][NE];
    f32x4 l_run[kNQ];
    float m_run[kNQ];
#pragma unroll
    for (int x = 0; x < kNQ; ++x) {
#pragma unroll
      for (int e = 0; e < NE; ++e) o[x][e] = f32x4{0.f, 0.f, 0.f, 0.f};
      l_run[x] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_run[x] = kMinMax;
    }
    const u32x4 ones = {H::kOnePair, H::kOnePair, H::kOnePair, H::kOnePair};

    // V^T of block e, keys 32 c + 4 lr + 0..3 and + 16, of column d = 16 e + l16
    auto v_frag = [&](int stage, int c, int e) __attribute__((always_inline)) {
      const uint32_t vb = lds0 + stage * 2 * kStage + kStage;
      const int n = 32 * c + 4 * lr + (l16 >> 2), d = 16 * e + 4 * (l16 & 3);
      const uint32_t at = vb + v_at<D>(n, d >> 3) + (d & 7) * 2;  // row n + 16: the same swizzle
      const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)at);
      const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(uintptr_t)(at + 16 * D * 2));
      const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
      return u32x4{w0[0], w0[1], w1[0], w1[1]};
    };
    // plain: a tile of the context, every key of it there; `there`: bits of those that are; found: the
    // tile had values that are not finite
    auto compute = [&](int stage, int key, unsigned long long there, bool found) __attribute__((always_inline)) {
      const bool plain = ~there == 0 && key + kTile <= r.context;
      const uint32_t kbase = lds0 + stage * 2 * kStage;
      f32x4 sc[kNQ][NKB], y[kS ? kNQ : 1][NKB];  // y: with the values' scales
      // a block's fragments are read under the products of the block before
      u32x4 kf[2][NDS];
      auto read_k = [&](int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < NDS; ++s)
          kf[kb & 1][s] = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(kbase + k_at<D>(16 * kb + l16, 4 * s + lr));
      };
      read_k(0);
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        if (kb + 1 < NKB) read_k(kb + 1);
#pragma unroll
        for (int x = 0; x < kNQ; ++x) sc[x][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NDS; ++s)
#pragma unroll
          for (int x = 0; x < kNQ; ++x) sc[x][kb] = H::mfma16(kf[kb & 1][s], qf[x][s], sc[x][kb]);
      }
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
        if constexpr (kS) {
          const f32x4 f = *reinterpret_cast<const f32x4*>(&sc_lds[stage][0][16 * kb + 4 * lr]);
          const f32x4 lv = *reinterpret_cast<const f32x4*>(&sc_lds[stage][1][16 * kb + 4 * lr]);
#pragma unroll
          for (int x = 0; x < kNQ; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              sc[x][kb][i] *= f[i];
              y[x][kb][i] = sc[x][kb][i] + lv[i];
            }
        }
      uint32_t seen[kNQ];  // bit 4 kb + i: this lane's row sees its key
      if (!plain) {
#pragma unroll
        for (int x = 0; x < kNQ; ++x) {
          seen[x] = tree_lane_keys<NKB>(there & tree_visible(a, r, 16 * x + l16 < wave_rows, tok[x], first_word[x], key), lr);
#pragma unroll
          for (int n = 0; n < 4 * NKB; ++n)
            if (!(seen[x] >> n & 1u)) {
              sc[x][n >> 2][n & 3] = -INFINITY;
              if constexpr (kS) y[x][n >> 2][n & 3] = -INFINITY;
            }
        }
      }
      u32x4 vf[2][4];
      auto read_v = [&](int g) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 4; ++u) vf[g & 1][u] = v_frag(stage, (4 * g + u) / NE, (4 * g + u) % NE);
      };
      read_v(0);
      auto weighed = [&](int x, int n) __attribute__((always_inline)) {
        if constexpr (kS) return (float)y[x][n >> 2][n & 3];
        else return (float)sc[x][n >> 2][n & 3];
      };
#pragma unroll
      for (int x = 0; x < kNQ; ++x) {
        float mx = weighed(x, 0);
#pragma unroll
        for (int n = 1; n < 4 * NKB; ++n) mx = nan_max(mx, weighed(x, n));
        if constexpr (!kS) mx *= scale;
        float mx2 = mx;
        fa::rows4_combine<true>(mx, mx2);
        const bool raise = !(mx <= m_run[x] + kSlack);  // (a NaN too)
        if (__builtin_amdgcn_ballot_w64(raise)) {
          const float alpha = raise ? __builtin_amdgcn_exp2f(m_run[x] - mx) : 1.f;
          m_run[x] = raise ? mx : m_run[x];
          l_run[x] *= alpha;
#pragma unroll
          for (int e = 0; e < NE; ++e) o[x][e] *= alpha;
        }
      }
      u32x4 pp[kNQ][NC];
#pragma unroll
      for (int x = 0; x < kNQ; ++x) {
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (kS) w[i] = __builtin_amdgcn_exp2f(weighed(x, 4 * kb + i) - m_run[x]);
            else w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(weighed(x, 4 * kb + i), scale, -m_run[x]));
            if constexpr (kS) l_run[x][0] += __builtin_amdgcn_exp2f((float)sc[x][kb][i] - m_run[x]);
          }
          pp[x][kb >> 1][(kb & 1) * 2] = H::pack2(w[0], w[1]);
          pp[x][kb >> 1][(kb & 1) * 2 + 1] = H::pack2(w[2], w[3]);
        }
        if constexpr (!kS) {
#pragma unroll
          for (int c = 0; c < NC; ++c) l_run[x] = H::mfma16(ones, pp[x][c], l_run[x]);
        }
      }
      // groups of four V fragments, read under the products of the group before (the first under the softmax)
      constexpr int kGroups = NC * NE / 4;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        if (g + 1 < kGroups) read_v(g + 1);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int c = (4 * g + u) / NE, e = (4 * g + u) % NE;
#pragma unroll
          for (int x = 0; x < kNQ; ++x) o[x][e] = H::mfma16(vf[g & 1][u], pp[x][c], o[x][e]);
        }
      }
      if (!plain && found) {
        const Place p = checked(place(key));
#pragma unroll
        for (int x = 0; x < kNQ; ++x)
          tree_add_nonfinite<Tag, C, kTile>(a, o[x], seen[x], p.page, p.offset, h, lane, [&](int e, int i) { return 16 * e + 4 * lr + i; });
      }
    };

    // ---- the tiles ----
    auto drafts = [&](int key) __attribute__((always_inline)) { return key + kTile > r.context; };
    // the copies or stores of a tile are done, in every wave
    auto landed = [&](int stage, int key, int at) __attribute__((always_inline)) {
      if constexpr (kS) __syncthreads();
      else wait_and_barrier<0>();
      if constexpr (!std::is_same_v<C, int8_t>) {
        if (key < key_hi && drafts(key)) {
          sift(stage, at);
          __syncthreads();
        }
      }
    };
    if (tid < 3) found_lds[tid] = 0;
    Place p = checked(place(key_lo)), p1 = place(key_lo + kTile);
    unsigned long long there = __builtin_amdgcn_ballot_w64(p.page >= 0);
    if constexpr (kS) load(p);
    __syncthreads();
    if constexpr (kS) store(0, p);
    else copy(0, p);
    landed(0, key_lo, 0);
    int stage = 0, at = 0;  // at: the tile's number % 3
#pragma unroll 1
    for (int key = key_lo; key < key_hi; key += kTile) {
      const bool more = key + kTile < key_hi;
      const Place p2 = place(key + 2 * kTile);  // (before the rows: loads return in order)
      p1 = checked(p1);
      if constexpr (kS) load(p1);  // (also past the last: the wait for p2 behind a branch would be for every load)
      else if (more) copy(stage ^ 1, p1);
      const int at1 = at == 2 ? 0 : at + 1;
      if (tid == 0) found_lds[at1 == 2 ? 0 : at1 + 1] = 0;  // read a tile ago, written in the next turn
      if (wave_rows > 0)
        compute(stage, key, there, drafts(key) && found_lds[at] != 0);
      stage ^= 1;
      at = at1;
      if constexpr (kS) {
        if (more) store(stage, p1);
      }
      landed(stage, key + kTile, at);
      there = __builtin_amdgcn_ballot_w64(p1.page >= 0);
      p1 = p2;
    }

    // ---- this wave's rows: lane l16 holds row l16 of block x, d = 16 e + 4 lr + 0..3 ----
    float* record = split.partial + ((long long)2 * share.w + (starts_here ? 0 : 1)) * kRows * (D + kTreePad);
#pragma unroll
    for (int x = 0; x < kNQ; ++x) {
      float l = l_run[x][0];
      if constexpr (kS) {
        float l1 = l;
        fa::rows4_combine<false>(l, l1);
      }
      if (16 * x + l16 >= wave_rows) continue;
      const int n = wave * kWaveRows + 16 * x + l16;
      if (whole_item) {
        const float inv = l != 0.f ? 1.f / l : 0.f;
        uint16_t* out = static_cast<uint16_t*>(a.out) + (r.first + tok[x]) * a.o_token +
                        ((long long)h * a.group + (row0 + n - tok[x] * a.group)) * a.o_head;
#pragma unroll
        for (int e = 0; e < NE; ++e) {
          const int d = 16 * e + 4 * lr;
          if (d >= a.d) continue;
          u32x2 w = {0, 0};
          if (l != 0.f) w = u32x2{H::pack2(o[x][e][0] * inv, o[x][e][1] * inv), H::pack2(o[x][e][2] * inv, o[x][e][3] * inv)};
          *reinterpret_cast<uint32_t*>(out + d) = w[0];
          *reinterpret_cast<uint32_t*>(out + d + 2) = w[1];
        }
      } else {
        float* rec = record + (long long)n * (D + kTreePad);
#pragma unroll
        for (int e = 0; e < NE; ++e)
          if (16 * e + 4 * lr < a.d) *reinterpret_cast<f32x4*>(rec + 16 * e + 4 * lr) = o[x][e];
        if (lr == 0) *reinterpret_cast<f32x2*>(rec + D) = f32x2{m_run[x], l};
      }
    }
  }
}

}  // namespace kg_gfx950
