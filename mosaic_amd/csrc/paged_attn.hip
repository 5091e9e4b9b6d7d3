// Attention over the paged 8-bit cache (layout: paged_kv.hip): each query row of
// a ragged batch sees its request's tokens up to its own position, optionally
// only the last `window` of them, with an optional sink logit for each head.
//
//   s = scale q . k in fp32 (k = code 2^(e - 127) in bf16: exact from 2^-126 on,
//   rounded to its step of 2^-133 below, infinite from 2^128 on), running
//   maximum and sum of exp(s - m) in fp32, o = sum p v / (sum p + exp(sink - m)).
//   p is rounded to bf16 for the matrix unit's value product: at most 2^-8 of a
//   term, of either sign, as much as the bf16 output's own rounding.  Sums are
//   fp32: of the unrounded p where rows are few, of the rounded (which makes the
//   rounding's common part cancel) where they are many.  m begins at fp32's lowest
//   number: a score of -inf, masked or overflowed, weighs 0 against it.
//
// Rows of one key head (tokens x query heads of its group) are tiled by 16.  A
// work unit is a (request, key head, row tile, block of 64 tokens), and a tile's
// first block is preceded by kStart empty ones; the units of all requests are
// numbered through and each workgroup takes an equal run of them, so the lengths
// may be as unequal as they like.  A run's piece of one tile
// is a segment: the waves take its blocks in turn, keep (m, l, O) in registers
// and meet in LDS at its end.  A tile in one segment is finished there; one that
// is cut at a run's border leaves partial sums that paged_attn_join_kernel adds up.
//
// Scores are computed transposed, S^T = K Q^T (16 tokens x 16 rows a tile): lane
// (q, c) then holds four tokens of row c, which are its own operand of
// O^T = V^T P^T; the cache stores the values in that order, so neither keys,
// values nor probabilities pass through LDS or between lanes.
#include <limits.h>

#include <cmath>
#include <type_traits>
#include <utility>

#include "common.h"
#include "../../include/mosaic_amd.h"

namespace mosaic {
namespace {

constexpr int kBlock = 64;
constexpr int kRows = 16;           // rows of a tile
// Workgroups of the few-row kernel: one a CU (eight waves; four beside the many-row
// kernel's), so that none begins late.  A context of 131000 tokens, 64 heads on 8 of 128: 58.5 us,
// with 512 62.6, with 1024 69.7; 64 requests of up to 32768: 386, 389 and 395 us.
constexpr int kGroups = 256;
// What a tile's first piece costs beside its blocks, in blocks (its queries, the chain of page, codes
// and scores, the meeting of the waves): a run of many short tiles gets as much less.  64 requests
// of up to 2000 tokens, 64 heads on 8 of 128: 61.0 us without, 41.5 with 4, 34.6 with 8, 33.0 with
// 14; 64 of up to 32768: 387, 376, 368, 368; 8 pieces beside them 46.4, 44.9, 45.7, 47.2.
constexpr int kStart = 8;
// Blocks of a table up to which tiles are not cut, which saves the join: a tile is then the run's
// that holds its first unit.  Tables of 30 blocks, 64 heads on 8 of 128, cut and whole: 1 request 13.4 and
// 12.6 us, 16 17.3 and 13.9, 64 31.2 and 28.4, 200 90.1 and 87.2; of 50: 12.8 and 17.8, 19.8 and 20.5, 50.7 and 55.6.
constexpr int kWhole = 32;
// Up to this, where there are more tiles than workgroups, a tile is four waves' and a CU has two
// workgroups, whose chains overlap.  64 heads on 8 of 128, eight and four waves: 256 requests of up to 500
// tokens 56.5 and 42.2 us, 64 of up to 800 20.4 and 19.8, but 64 of up to 1700 28.4 and 29.1; with fewer
// tiles, 16 of up to 800, 10.9 and 13.2.
constexpr int kNarrow = 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;  // fp32's: a maximum of nothing
// Each block that a row sees a key of adds so much to its sum (1 and more where there is a
// weight, which that does not round), so that a row of nothing but scores of -inf is told from one without keys
constexpr float kSeen = 0x1p-100f, kWeightless = 0x1p-60f;

struct AttnArgs {
  const uint16_t* q;
  const uint8_t *codes, *scales;
  const int32_t *table, *starts, *seq;
  const float* sink;
  uint16_t* out;
  float* part_o;   // [2 kGroups][16][D], unnormalized
  float* part_ml;  // [2 kGroups][2][16]
  int32_t* info;   // [0]: tiles; from [8]: [tiles][Hkv][8]: first row, rows, pieces, slots of the first and second
                   // piece, from one piece's slot to the next's (a slot: partial sums of 16 rows)
  float *tile_o, *tile_ml;  // the same of the many-row kernel, where it cuts tiles
  int32_t* tile_info;
  int64_t q_tok, q_head, stride;
  int r, tokens, hq, hkv, group, width, pages, nb, window;
  bool whole;      // few-row tiles are not cut (no join)
  int rows_max;    // requests of more rows are the many-row kernel's
  uint32_t few_cap, many_cap;  // row tiles that the workspace and grid hold: ascending starts have no more
  bool zero_rows;  // the many-row kernel clears what lies behind the last request
  float scale;     // |softmax scale| log2(e)
  float sign;      // of the softmax scale
};

struct Request {
  int s0, n, held, first, blocks, rows;  // first: the first block that any row sees
};

__device__ __forceinline__ Request request_of(const AttnArgs& a, int r) {
  Request x{0, 0, 0, 0, 0, 0};
  if (r < a.r) {
    x.s0 = min(max(a.starts[r], 0), a.tokens);
    x.n = min(max(a.starts[r + 1], x.s0), a.tokens) - x.s0;
    const int seq = min(max(a.seq[r], 0), a.width * a.nb * kBlock);
    x.held = seq - x.n;
    x.first = a.window && x.held + 1 > a.window ? (x.held + 1 - a.window) / kBlock : 0;
    x.blocks = max((seq + kBlock - 1) / kBlock - x.first, 1);  // a tile without tokens still writes its zeros
    x.rows = x.n * a.group;
  }
  return x;
}
// row tiles of 16 of a request that is not left to the many-row kernel
__device__ __forceinline__ int few_tiles(const AttnArgs& a, const Request& x) {
  return x.rows > a.rows_max ? 0 : (x.rows + kRows - 1) / kRows;
}
__device__ __forceinline__ bool many_rows(const AttnArgs& a, const Request& x) { return x.rows > a.rows_max; }

// 1 / (l + exp2(sink - m)): what a row's sums are multiplied by.  Without weights they
// are zeros, and so is the output: 0 / exp(sink), or by convention where the row sees
// no key at all; but 0 / 0, not a number, where it sees some and has no sink.
__device__ __forceinline__ float row_factor(const AttnArgs& a, int head, float m, float l) {
  const float s = a.sink ? a.sink[head] * kLog2e : -INFINITY;
  if (l < kWeightless) return l > 0.f && s == -INFINITY ? NAN : 0.f;
  return 1.f / (l + __builtin_amdgcn_exp2f(s - m));
}

__device__ __forceinline__ float lane4_max(float x) {  // over the four lanes of a column
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = fmaxf(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return fmaxf(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
}
__device__ __forceinline__ float lane4_sum(float x) {
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = __uint_as_float(r16[0]) + __uint_as_float(r16[1]);
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return __uint_as_float(r32[0]) + __uint_as_float(r32[1]);
}

// Eight codes (two words) times a scale byte's 2^(e - 127) in bf16, by the exponent of
// `scale`: 2^-127 for byte 0, though that is 0 as a float.
__device__ __forceinline__ bf16x8_t to_bf16(uint32_t w0, uint32_t w1, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// The least code that is no finite number at scale byte e: NaN's, 0x7F; from byte 247 on the
// one of 2^(255 - e), which times 2^(e - 127) is 2^128 (zero times that is no number either); at
// 255 any.  As what is to be added to a byte's magnitude for its high bit, in every byte.
constexpr uint32_t kOverflow = 247;  // the least scale byte at which codes pass the range
__device__ __forceinline__ uint32_t bad_from(uint32_t e) {
  return (e < kOverflow ? 1u : e == 255u ? 0x80u : 0x80u - 8u * (262u - e)) * 0x01010101u;
}
// 0xFF in every byte of w that is such a code
__device__ __forceinline__ uint32_t bad_bytes(uint32_t w, uint32_t from) {
  const uint32_t x = ((w & 0x7F7F7F7Fu) + from) & 0x80808080u;
  return x | (x - (x >> 7));
}
constexpr uint32_t kNan = 0x01010101u;  // bad_from of the ordinary scales

// The units of all requests are numbered through, `units(request)` of each, and so
// are their row tiles, `tiles(request)`.  Finds the request that holds unit
// pick(total), with its first unit and tile; none where pick gives total or more.
// Every workgroup does this by itself: one round trip to L2 for up to 64 NW requests.
struct Place {
  Request x;
  int r, tile0;
  uint32_t unit0, unit, total, tiles;
};
template <int NW, typename Units, typename Tiles, typename Pick>
__device__ __forceinline__ Place place(const AttnArgs& a, Units units, Tiles tiles, Pick pick) {
  __shared__ uint32_t sums[NW][2];
  __shared__ int found[10];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  Place p{};
  uint32_t n = 0, t = 0, at = 0, t_at = 0;
  auto count = [&](int base) {  // this thread's request, and what lies before it
    p.x = request_of(a, base + tid);
    n = units(p.x);
    t = tiles(p.x);
    const uint32_t incl = wave_incl_scan_u32(n), tinc = wave_incl_scan_u32(t);
    if (lane == 63) {
      sums[wave][0] = incl;
      sums[wave][1] = tinc;
    }
    __syncthreads();
    at = p.total + incl - n;
    t_at = p.tiles + tinc - t;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      at += w < wave ? sums[w][0] : 0u;
      t_at += w < wave ? sums[w][1] : 0u;
      p.total += sums[w][0];
      p.tiles += sums[w][1];
    }
    __syncthreads();
  };
  for (int base = 0; base < a.r; base += 64 * NW) count(base);
  const uint32_t total = __builtin_amdgcn_readfirstlane(p.total), all = __builtin_amdgcn_readfirstlane(p.tiles);
  p.unit = pick(total);
  if (p.unit >= total) return Place{Request{}, 0, 0, 0u, p.unit, total, all};  // nothing of a lane's own in the answer
  auto note = [&](int base) {
    if (p.unit >= at && p.unit - at < n) {
      const int v[10] = {p.x.s0, p.x.n, p.x.held, p.x.first, p.x.blocks, p.x.rows, base + tid, (int)t_at, (int)at, 0};
#pragma unroll
      for (int i = 0; i < 9; ++i) found[i] = v[i];
    }
    __syncthreads();
  };
  if (a.r <= 64 * NW) {
    note(0);
  } else {
    p.total = p.tiles = 0;
    for (int base = 0; base < a.r && (uint32_t)__builtin_amdgcn_readfirstlane(p.total) <= p.unit; base += 64 * NW) {
      count(base);
      note(base);
    }
  }
  auto get = [&](int i) { return __builtin_amdgcn_readfirstlane(found[i]); };
  p.x = Request{get(0), get(1), get(2), get(3), get(4), get(5)};
  p.r = get(6);
  p.tile0 = get(7);
  p.unit0 = (uint32_t)get(8);
  p.total = total;
  p.tiles = all;
  return p;
}

// rows behind the last request are zero
template <int D>
__device__ __forceinline__ void clear_rest(const AttnArgs& a, int64_t thread, int64_t threads) {
  const int64_t from = a.r ? min(max(a.starts[a.r], 0), a.tokens) : 0, per = (int64_t)a.hq * D;
  for (int64_t i = from * per + 8 * thread; i < a.tokens * per; i += 8 * threads)
    *reinterpret_cast<u32x4_t*>(a.out + i) = u32x4_t{0u, 0u, 0u, 0u};
}

template <int D, int NW>
constexpr int kRowsLds = NW / 2 * D * 16 * 4;  // the halves' sums meet in fp32
template <int D, int NW>
__device__ __forceinline__ void rows_body(const AttnArgs& a, uint8_t* lds, uint32_t groups) {
  constexpr int DG = D / 64, DT = D / 16;
  auto so = reinterpret_cast<f32x4_t(*)[DT * 4 * 16]>(lds);  // [NW / 2]
  __shared__ float sm[NW][16], sl[NW][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, c = lane & 15;
  const float scale = a.scale * a.sign;

  // units of a tile and head: what it costs.  Where tiles are whole, they are their first unit's run's.
  auto per_tile = [&](const Request& x) { return (uint32_t)(kStart + x.blocks); };
  uint32_t share = 0;
  const Place at = place<NW>(
      a, [&](const Request& x) { return (uint32_t)few_tiles(a, x) * (uint32_t)a.hkv * per_tile(x); },
      [&](const Request& x) { return (uint32_t)few_tiles(a, x); },
      [&](uint32_t total) {
        share = (total + groups - 1) / groups;
        if (!a.whole) share = max(share, (uint32_t)NW / 2);
        return min(blockIdx.x * (uint64_t)share, (uint64_t)total);
      });
  clear_rest<D>(a, (int64_t)blockIdx.x * 64 * NW + tid, (int64_t)groups * 64 * NW);
  if (!a.whole && blockIdx.x == 0 && tid == 0) a.info[0] = (int32_t)at.tiles;
  const uint32_t u0 = at.unit, u1 = min(u0 + share, at.total);
  if (u0 >= at.total) return;
  Request x = at.x, after = request_of(a, at.r + 1);
  int r = at.r, tile0 = at.tile0;
  uint32_t req0 = at.unit0, tiles = (uint32_t)few_tiles(a, x), per = per_tile(x);
  for (uint32_t u = u0; u < u1;) {
    while (u - req0 >= tiles * (uint32_t)a.hkv * per) {
      req0 += tiles * (uint32_t)a.hkv * per;
      tile0 += (int)tiles;
      x = after;
      after = request_of(a, ++r + 1);  // read ahead: the next segment does not wait for it
      tiles = (uint32_t)few_tiles(a, x);
      per = per_tile(x);
      if (r >= a.r) return;  // only where starts that do not ascend number more units than 32 bits hold
    }
    // unit -> (head, tile, block), blocks fastest
    const uint32_t in = u - req0, ht = in / per;
    const int begin = (int)(in % per), units = (int)(a.whole ? per - begin : min(per - begin, u1 - u));
    const int b_from = a.whole ? 0 : max(begin - kStart, 0), b_to = begin + units - kStart;
    const int h = (int)(ht / tiles), tile = (int)(ht % tiles);
    const uint32_t tile_u0 = u - begin;
    u += units;
    if (a.whole ? begin > 0 : b_to <= 0) continue;  // an earlier run's; the run ends before the tile's first block
    const int row0 = tile * kRows, rows = min(kRows, x.rows - row0);
    const int row = row0 + min(c, rows - 1);
    const int tok = row / a.group, head = h * a.group + row % a.group;
    const int pos = x.held + tok;
    const int row_hi = min(max(pos + 1, 0), a.width * a.nb * kBlock), row_lo = a.window ? max(pos + 1 - a.window, 0) : 0;
    // over the tile's rows: the tokens that all of them see, and that any sees
    const int tok_a = row0 / a.group, tok_b = (row0 + rows - 1) / a.group;
    const int any_hi = max(x.held + tok_b + 1, 0), all_hi = max(x.held + tok_a + 1, 0);
    const int any_lo = a.window ? max(x.held + tok_a + 1 - a.window, 0) : 0;
    const int all_lo = a.window ? max(x.held + tok_b + 1 - a.window, 0) : 0;
    bf16x8_t qf[DG][2];
    const uint16_t* qrow = a.q + (int64_t)(x.s0 + tok) * a.q_tok + (int64_t)head * a.q_head;
#pragma unroll
    for (int g = 0; g < DG; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) qf[g][i] = *reinterpret_cast<const bf16x8_t*>(qrow + 64 * g + 16 * q + 8 * i);
    float m = kLowest, l = 0.f;
    f32x4_t o[DT];
#pragma unroll
    for (int j = 0; j < DT; ++j) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const int32_t* trow = a.table + (int64_t)r * a.stride;
    for (int b = b_from + wave; b < b_to; b += NW) {
      const int blk = x.first + b, t0 = blk * kBlock;
      if (t0 >= any_hi || t0 + kBlock <= any_lo) continue;
      const int page = trow[blk / a.nb];
      const bool good = page >= 0 && page < a.pages;
      const int64_t unit = ((int64_t)(good ? page : 0) * a.nb + blk % a.nb) * a.hkv + h;
      const u32x4_t* kc = reinterpret_cast<const u32x4_t*>(a.codes + unit * (2 * kBlock * D)) + lane;
      const u32x4_t* vc = kc + 4 * D;  // 64 D bytes on
      const uint32_t se = *reinterpret_cast<const uint16_t*>(a.scales + unit * 2);
      const uint32_t ke = se & 0xFFu, ve = se >> 8;
      u32x4_t kw[4][DG], vw[DT];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int g = 0; g < DG; ++g) kw[t][g] = kc[(t * DG + g) * 64];
#pragma unroll
      for (int j = 0; j < DT; ++j) vw[j] = vc[j * 64];
      const float ks = e8m0_f32(ke), vs = e8m0_f32(ve);
      f32x4_t s[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        s[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < DG; ++g)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(kw[t][g][2 * i], kw[t][g][2 * i + 1], ks), qf[g][i],
                                                           s[t], 0, 0, 0);
      }
      // a block that some row does not see whole, one without a page, or whose scale makes no numbers
      const bool edge = t0 + kBlock > all_hi || t0 < all_lo || !good || ke == 255u || ve >= kOverflow;
      const int hi = good ? row_hi : 0;
      float bm = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = s[t][i] * scale;
          if (edge) {
            const int p = t0 + 16 * t + 4 * q + i;
            v = ke == 255u ? NAN : v;
            v = p < hi && p >= row_lo ? v : -INFINITY;
          }
          s[t][i] = v;
          bm = fmaxf(bm, v);
        }
      bm = lane4_max(bm);
      const float ref = fmaxf(m, bm);
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
      m = ref;
      bf16x8_t p[2];
      float sum = !edge || min(hi, t0 + kBlock) > max(row_lo, t0) ? kSeen : 0.f;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(s[t][i] - ref);
          sum += e[i];
        }
        const bf16x2_t lo = __builtin_convertvector(f32x2_t{e[0], e[1]}, bf16x2_t);
        const bf16x2_t up = __builtin_convertvector(f32x2_t{e[2], e[3]}, bf16x2_t);
        p[t >> 1][4 * (t & 1)] = lo[0];
        p[t >> 1][4 * (t & 1) + 1] = lo[1];
        p[t >> 1][4 * (t & 1) + 2] = up[0];
        p[t >> 1][4 * (t & 1) + 3] = up[1];
      }
      l = l * alpha + sum;
#pragma unroll
      for (int j = 0; j < DT; ++j) o[j] *= alpha;
      if (edge) {
        // A code that is not a finite number reaches only the rows that see its token: it
        // is taken out of the product (zero times it would reach all), and where a
        // count of the seen ones is not zero, the result is not a number.
        if (ve >= kOverflow)  // seldom: NaN codes for all of them
#pragma unroll
          for (int j = 0; j < DT; ++j)
#pragma unroll
            for (int w = 0; w < 4; ++w) vw[j][w] |= bad_bytes(vw[j][w], bad_from(ve));
        uint32_t any = 0u;
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
          for (int w = 0; w < 4; ++w) any |= bad_bytes(vw[j][w], kNan);
        if (__ballot(any != 0u)) {
          bf16x8_t see[2];
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int tk = t0 + 16 * t + 4 * q + i;
              see[t >> 1][4 * (t & 1) + i] = (__bf16)(tk < hi && tk >= row_lo ? 1.f : 0.f);
            }
#pragma unroll
          for (int j = 0; j < DT; ++j) {
            uint32_t bad[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              bad[w] = bad_bytes(vw[j][w], kNan);
              vw[j][w] &= ~bad[w];
              bad[w] &= 0x38383838u;  // the code of 1
            }
            f32x4_t n = f32x4_t{0.f, 0.f, 0.f, 0.f};
            n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(bad[0], bad[1], 1.f), see[0], n, 0, 0, 0);
            n = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(bad[2], bad[3], 1.f), see[1], n, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = n[i] > 0.f ? NAN : o[j][i];
          }
        }
      }
      const float vscale = ve == 255u ? 1.f : vs;
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16(vw[j][2 * i], vw[j][2 * i + 1], vscale), p[i], o[j], 0, 0, 0);
    }
    // the waves meet: a common maximum, then sums by halves
    l = lane4_sum(l);
    if (q == 0) {
      sm[wave][c] = m;
      sl[wave][c] = l;
    }
    __syncthreads();
    float M = kLowest, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w][c]);
#pragma unroll
    for (int w = 0; w < NW; ++w) L += sl[w][c] * __builtin_amdgcn_exp2f(sm[w][c] - M);
    const float f = __builtin_amdgcn_exp2f(m - M);
#pragma unroll
    for (int j = 0; j < DT; ++j) o[j] *= f;
    if (wave >= NW / 2)
#pragma unroll
      for (int j = 0; j < DT; ++j) so[wave - NW / 2][(4 * j + q) * 16 + c] = o[j];
    __syncthreads();
    if (wave < NW / 2)
#pragma unroll
      for (int j = 0; j < DT; ++j) so[wave][(4 * j + q) * 16 + c] += o[j];
    __syncthreads();
    const bool whole = b_from == 0 && b_to == x.blocks;
    // a piece that begins inside its tile is its run's first, one that only ends inside is its last
    const int slot = 2 * (int)blockIdx.x + (b_from == 0 ? 1 : 0);
    // the join's list: this tile's rows and the runs that hold it
    if (!a.whole && b_from == 0 && (uint32_t)(tile0 + tile) < a.few_cap && tid == 0) {
      int32_t* t = a.info + 8 + ((int64_t)(tile0 + tile) * a.hkv + h) * 8;
      t[0] = (x.s0 + row0 / a.group) * a.group + row0 % a.group;
      t[1] = rows;
      t[2] = (int)((tile_u0 + per - 1) / share - blockIdx.x) + 1;
      t[3] = slot;
      t[4] = slot + 1;
      t[5] = 2;
    }
    // thread -> (4 dims, row c): c stays tid's
    const float inv = whole ? row_factor(a, head, M, L) : 0.f;
    for (int i = tid; i < DT * 4 * 16; i += 64 * NW) {
      f32x4_t v = so[0][i];
#pragma unroll
      for (int w = 1; w < NW / 2; ++w) v += so[w][i];
      const int quad = i >> 4;
      if (whole) {
        if (c < rows) {
          uint2 pk;
          pk.x = (uint32_t)f32_bf16(v[0] * inv) | ((uint32_t)f32_bf16(v[1] * inv) << 16);
          pk.y = (uint32_t)f32_bf16(v[2] * inv) | ((uint32_t)f32_bf16(v[3] * inv) << 16);
          *reinterpret_cast<uint2*>(a.out + ((int64_t)(x.s0 + tok) * a.hq + head) * D + 4 * quad) = pk;
        }
      } else {
        *reinterpret_cast<f32x4_t*>(a.part_o + ((int64_t)slot * 16 + c) * D + 4 * quad) = v;
      }
    }
    if (!whole && tid < 16) {
      a.part_ml[(int64_t)slot * 32 + c] = M;
      a.part_ml[(int64_t)slot * 32 + 16 + c] = L;
    }
    __syncthreads();  // so, sm and sl are used again
  }
}

template <int D, int NW>
__global__ void __launch_bounds__(64 * NW, D == 256 ? 1 : 2) paged_attn_rows_kernel(const AttnArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[kRowsLds<D, NW>];
  rows_body<D, NW>(a, lds, gridDim.x);
}

// Adds up the pieces of a tile that was cut.  256 threads, in groups of D / 4 lanes
// (four dims each).  Up to 16 pieces: a group a row, one piece after the other.
// More (few rows over a long axis): the groups share a row's pieces and meet in LDS.
template <int D>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(const AttnArgs a, const int32_t* __restrict__ info) {
  constexpr int LANES = D / 4, SG = 256 / LANES;
  __shared__ f32x4_t so[SG][LANES];
  __shared__ float red[4], ls[SG];
  const int tile = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, g = tid / LANES, d = tid % LANES;
  if (tile >= info[0]) return;
  const int32_t* t = info + 8 + ((int64_t)tile * a.hkv + h) * 8;
  const int n = t[2];
  if (n == 1) return;
  const int step = t[5];
  auto finish = [&](int row, float m, float l, f32x4_t o) {
    const int head = h * a.group + row % a.group;
    const float inv = row_factor(a, head, m, l);
    uint2 pk;
    pk.x = (uint32_t)f32_bf16(o[0] * inv) | ((uint32_t)f32_bf16(o[1] * inv) << 16);
    pk.y = (uint32_t)f32_bf16(o[2] * inv) | ((uint32_t)f32_bf16(o[3] * inv) << 16);
    *reinterpret_cast<uint2*>(a.out + ((int64_t)(row / a.group) * a.hq + head) * D + 4 * d) = pk;
  };
  if (n <= 16) {
    for (int i = blockIdx.z * SG + g; i < t[1]; i += gridDim.z * SG) {
      const int64_t first = t[3] + i / 16, second = t[4] + i / 16;
      const int c = i % 16;
      float m = kLowest;
#pragma unroll 4
      for (int p = 0; p < n; ++p) m = fmaxf(m, a.part_ml[(p ? second + (int64_t)step * (p - 1) : first) * 32 + c]);
      f32x4_t o = {0.f, 0.f, 0.f, 0.f};
      float l = 0.f;
#pragma unroll 4
      for (int p = 0; p < n; ++p) {
        const int64_t slot = p ? second + (int64_t)step * (p - 1) : first;
        const float f = __builtin_amdgcn_exp2f(a.part_ml[slot * 32 + c] - m);
        l += f * a.part_ml[slot * 32 + 16 + c];
        o += *reinterpret_cast<const f32x4_t*>(a.part_o + (slot * 16 + c) * D + 4 * d) * f;
      }
      finish(t[0] + i, m, l, o);
    }
    return;
  }
  for (int i = blockIdx.z; i < t[1]; i += gridDim.z) {
    const int64_t first = t[3] + i / 16, second = t[4] + i / 16;
    const int c = i % 16;
    float m = kLowest;
    for (int p = tid; p < n; p += 256) m = fmaxf(m, a.part_ml[(p ? second + (int64_t)step * (p - 1) : first) * 32 + c]);
    m = wave_max_f32(m);
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
#pragma unroll 8
    for (int p = g; p < n; p += SG) {
      const int64_t slot = p ? second + (int64_t)step * (p - 1) : first;
      const float f = __builtin_amdgcn_exp2f(a.part_ml[slot * 32 + c] - m);
      l += f * a.part_ml[slot * 32 + 16 + c];
      o += *reinterpret_cast<const f32x4_t*>(a.part_o + (slot * 16 + c) * D + 4 * d) * f;
    }
    so[g][d] = o;
    if (d == 0) ls[g] = l;
    __syncthreads();
    if (g == 0) {
#pragma unroll
      for (int p = 1; p < SG; ++p) {
        o += so[p][d];
        l += ls[p];
      }
      finish(t[0] + i, m, l, o);
    }
    __syncthreads();  // so, ls and red are used again
  }
}

// ---------------------------------------------------------- many rows ----
// Requests of many rows (prompts and their pieces): a workgroup owns 32 NW rows of
// a key head, 32 a wave, and its waves share the blocks, which are copied
// straight into LDS, three ahead.
//
//   scores   S^T = K Q^T in bf16 (32 x 32 x 16), codes converted with their scale as
//            they come out of LDS.  (Codes as they are, against q in two e4m3 parts on
//            the fp8 unit, were slower: a prompt of 4096 tokens, 64 heads of 128, 376
//            against 323 us; and its sums are not as exact as fp32.)
//   values   O^T = V^T P^T in bf16 (32 x 32 x 16), codes converted with their
//            scale as they come out of LDS; lane (h, c) holds tokens
//            8 i + 4 h + .. of row c, which are its operand.
// The reference of a row's exponentials follows its maximum only when one of them
// would be larger than 2^8: up to there the relative rounding is the same, O is
// seldom scaled, and the exponentials need not wait for a maximum (they find out
// themselves).

typedef __attribute__((ext_vector_type(16))) float f32x16_t;

constexpr float kLazy = 256.f;

__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// run I of 1 KB, 16 bytes a lane, of those from g (one address for the wave) to LDS;
// the immediate offset counts on both sides.  s_nop: a load that takes m0 needs one
// wait state behind its write, which nothing adds inside an asm text
template <int I>
__device__ __forceinline__ void lds_copy(const uint8_t* g, uint32_t lane16, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3" ::"s"(lds + I / 4 * 4096),
               "v"(lane16), "s"(g + I / 4 * 4096), "n"(I % 4 * 1024)
               : "memory", "m0");
}
// f(std::integral_constant<int, 0>) .. f(<N - 1>)
template <typename F, int... I>
__device__ __forceinline__ void unrolled(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  unrolled(f, std::make_integer_sequence<int, N>{});
}
template <int N>
__device__ __forceinline__ void lds_copies(const uint8_t* g, uint32_t lane16, uint32_t lds) {
  unrolled<N>([&](auto i) __attribute__((always_inline)) { lds_copy<decltype(i)::value>(g, lane16, lds); });
}
// own copies but the last N are in LDS, own LDS reads are done, and so are the other waves'
template <int N>
__device__ __forceinline__ void stage_ready() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int D>
constexpr int kTileLds = 4 * 2 * kBlock * D;  // four stages
// `group`: this workgroup's number among those of its kind, of `groups`
template <int D, int NW>
__device__ __forceinline__ void tile_body(const AttnArgs& a, uint8_t* buf, int group, int groups) {
  constexpr int DG = D / 64, DQ = D / 32, ROWS = 32 * NW, STAGE = 2 * kBlock * D;
  constexpr int STAGES = 4, CPW = STAGE / 1024 / NW;  // copies of 1 KB a wave and block
  static_assert(CPW >= 1, "every wave copies");
  static_assert(kTileLds<D> == STAGES * STAGE, "the ring");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, c = lane & 31, c16 = lane & 15, up = (lane >> 4) & 1;

  if (a.zero_rows && blockIdx.y == 0) clear_rest<D>(a, (int64_t)group * 64 * NW + tid, (int64_t)groups * 64 * NW);
  // the request and tile: key heads fastest (a head's workgroups meet in one XCD's
  // L2 where there are eight), the last tiles, which see most, first
  const int h = group % a.hkv;
  const uint32_t idx = group / a.hkv;
  auto count = [&](const Request& x) { return many_rows(a, x) ? (uint32_t)((x.rows + ROWS - 1) / ROWS) : 0u; };
  const Place found = place<NW>(a, count, [](const Request&) { return 0u; },
                                [&](uint32_t total) {
                                  const uint32_t last = min(total, a.many_cap);
                                  return idx < last ? last - 1 - idx : total;
                                });
  if (gridDim.y > 1 && group == 0 && blockIdx.y == 0 && tid == 0) a.tile_info[0] = (int32_t)found.total;
  if (found.unit >= found.total) return;
  const uint32_t want = found.unit;
  const int r = found.r, tile = (int)(want - found.unit0);
  const Request x = found.x;
  const int row0 = tile * ROWS, rows = min(ROWS, x.rows - row0);
  const int limit = a.width * a.nb * kBlock;
  // blocks that the tile sees, and this workgroup's share of them
  const int tile_hi = min(max(x.held + (row0 + rows - 1) / a.group + 1, 0), limit);
  const int tile_lo = a.window ? max(x.held + row0 / a.group + 1 - a.window, 0) : 0;
  const int first = tile_lo / kBlock, all_blocks = max((tile_hi + kBlock - 1) / kBlock - first, 0);
  const int b0 = __builtin_amdgcn_readfirstlane(first + (int)((int64_t)all_blocks * blockIdx.y / gridDim.y));
  const int nblk = __builtin_amdgcn_readfirstlane(first + (int)((int64_t)all_blocks * (blockIdx.y + 1) / gridDim.y)) - b0;

  // Every NW-th row is a wave's: the waves meet the blocks that some row does not
  // see together, instead of one after the other at every barrier.
  const bool has_rows = wave < rows;
  const int in_tile = min(NW * c + wave, rows - 1), row = row0 + in_tile;
  const bool own_row = NW * c + wave < rows;
  const int tok = row / a.group, head = h * a.group + row % a.group, pos = x.held + tok;
  const int row_hi = min(max(pos + 1, 0), limit), row_lo = a.window ? max(pos + 1 - a.window, 0) : 0;
  // over the tile's rows: the tokens that any and that all of them see
  const int tok_a = row0 / a.group, tok_b = (row0 + rows - 1) / a.group;
  const int any_hi = has_rows ? max(x.held + tok_b + 1, 0) : 0, all_hi = max(x.held + tok_a + 1, 0);
  const int any_lo = a.window ? max(x.held + tok_a + 1 - a.window, 0) : 0;
  const int all_lo = a.window ? max(x.held + tok_b + 1 - a.window, 0) : 0;

  // q: 32 dims of a row for each 64, in the order of the keys' bytes
  bf16x8_t qf[DG][4];
  {
    const uint16_t* qrow = a.q + (int64_t)(x.s0 + tok) * a.q_tok + (int64_t)head * a.q_head + 32 * hl;
    const uint32_t flip = a.sign < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int g = 0; g < DG; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u32x4_t w = *reinterpret_cast<const u32x4_t*>(qrow + 64 * g + 8 * i);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] ^= flip;
        qf[g][i] = __builtin_bit_cast(bf16x8_t, w);
      }
  }

  // where the 64 blocks from `meta` on lie and their scales (~0: no page), one a lane
  const int32_t* trow = a.table + (int64_t)r * a.stride;
  int meta = 0;
  uint32_t at_lo = 0u, at_hi = 0u, scales_ = ~0u, sc_in = 0u;
  auto load_meta = [&](int from) {
    meta = from;
    at_lo = at_hi = 0u;
    scales_ = ~0u;
    if (from + lane < nblk) {
      const int blk = b0 + from + lane, page = trow[blk / a.nb];
      const bool good = page >= 0 && page < a.pages;
      const int64_t unit = ((int64_t)(good ? page : 0) * a.nb + blk % a.nb) * a.hkv + h;
      const uint32_t sc = *reinterpret_cast<const uint16_t*>(a.scales + unit * 2);
      scales_ = good ? sc : ~0u;
      at_lo = (uint32_t)(unit * STAGE);
      at_hi = (uint32_t)((unit * STAGE) >> 32);
    }
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)buf + wave * CPW * 1024;
  const uint32_t lane16 = lane * 16;
  // block j, or the last one again: every turn copies as much, so the waits are constant
  auto locate = [&](int j) -> const uint8_t* {
    j = min(j, nblk - 1);
    if (j - meta >= 64) load_meta(j);
    const uint64_t at = (uint32_t)__builtin_amdgcn_readlane((int)at_lo, j - meta) |
                        (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)at_hi, j - meta) << 32;
    sc_in = (uint32_t)__builtin_amdgcn_readlane((int)scales_, j - meta);
    return a.codes + wave * CPW * 1024 + at;
  };

  float ref = kLowest, l = 0.f;  // ref: what a row's exponents are taken against
  f32x16_t o[DQ];
  const f32x16_t zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < DQ; ++j) o[j] = zero;

  u32x4_t k0[2][2], vw[DQ][2];  // k0: the keys' first 64 dims
  f32x16_t s[2];
  const uint8_t* src = nullptr;  // the block being copied this turn, and to where
  uint32_t dst = lds0;
  auto load_keys = [&](const uint8_t* kb, int g, u32x4_t (&w)[2][2]) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const u32x4_t* p = reinterpret_cast<const u32x4_t*>(kb + (((2 * t + up) * DG + g) * 64 + 2 * hl * 16 + c16) * 16);
      w[t][0] = p[0];
      w[t][1] = p[16];
    }
  };
  auto load_values = [&](const uint8_t* kb) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < DQ; ++j) {
      const u32x4_t* p = reinterpret_cast<const u32x4_t*>(kb + kBlock * D + ((2 * j + up) * 64 + hl * 16 + c16) * 16);
      vw[j][0] = p[0];
      vw[j][1] = p[32];
    }
  };
  // Scores of a block whose keys' first 64 dims are in k0; the others' reads go out
  // 64 dims ahead.  COPY: this turn's copies between the products.
  auto scores = [&](auto copy, const uint8_t* kb, float ks) __attribute__((always_inline)) {
    constexpr bool COPY = decltype(copy)::value;
    u32x4_t kw[2][2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) kw[0][t][i] = k0[t][i];
    auto step = [&](auto n) __attribute__((always_inline)) {
      constexpr int N = decltype(n)::value, g = N / 4, i = N % 4;
      if constexpr (i == 0 && g + 1 < DG) {
        load_keys(kb, g + 1, kw[(g + 1) % 2]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4_t w = kw[g % 2][t][i >> 1];
        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(to_bf16(w[2 * (i & 1)], w[2 * (i & 1) + 1], ks), qf[g][i],
                                                       N ? s[t] : zero, 0, 0, 0);
      }
      if constexpr (COPY && N % 2 == 1 && N / 2 < CPW) {
        __builtin_amdgcn_sched_barrier(0);
        lds_copy<N / 2>(src, lane16, dst);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    unrolled<4 * DG>(step);
  };
  static_assert(CPW <= 2 * DG, "a copy for every second step");
  auto largest = [&]() __attribute__((always_inline)) -> float {
    float bm = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) bm = fmaxf(fmaxf(bm, s[0][i]), s[1][i]);
    return half_max(bm);
  };
  // The reference of every row moves to its maximum with these scores.  A row that has
  // none yet (fp32's lowest number) makes its next exponential infinite, which calls for
  // this; one of a score of -inf is 0, and does not.
  auto move = [&]() __attribute__((always_inline)) {
    const float top = largest() * a.scale;
    const bool go = top > ref;
    const float alpha = go ? __builtin_amdgcn_exp2f(ref - top) : 1.f;
    ref = go ? top : ref;
    l *= alpha;
#pragma unroll
    for (int j = 0; j < DQ; ++j) o[j] *= alpha;
  };
  bf16x8_t p[4];
  // -> the lane's largest; their sum is added to l by the caller
  float sum;
  auto exponentials = [&](auto fused, float to, float seen) __attribute__((always_inline)) -> float {
    // one rounding, or two: with those, the maximum's exponent is 0 however large the scores are
    auto power = [&](float x) __attribute__((always_inline)) {
      return __builtin_amdgcn_exp2f(decltype(fused)::value ? __builtin_fmaf(x, a.scale, -to) : x * a.scale - to);
    };
    float big = 0.f;
    sum = seen;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e0 = power(s[t][8 * u + 2 * i]);
          const float e1 = power(s[t][8 * u + 2 * i + 1]);
          big = fmaxf(fmaxf(big, e0), e1);
          const bf16x2_t v = __builtin_convertvector(f32x2_t{e0, e1}, bf16x2_t);
          sum = __builtin_amdgcn_fdot2_f32_bf16(v, bf16x2_t{(__bf16)1.f, (__bf16)1.f}, sum, false);
          p[2 * t + u][2 * i] = v[0];
          p[2 * t + u][2 * i + 1] = v[1];
        }
    return big;
  };
  auto products = [&](float vs) __attribute__((always_inline)) {
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int j = 0; j < DQ; ++j)
        o[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(to_bf16(vw[j][0][w], vw[j][1][w], vs), p[w], o[j], 0, 0, 0);
  };
  // A block that every row sees whole, its first keys in registers.  The values' and the
  // next block's keys' reads go out before the exponentials, so that no product
  // waits for LDS.  False, and nothing done, where a reference has to move.
  auto whole_block = [&](const uint8_t* kb, const uint8_t* next, uint32_t ke, uint32_t ve) __attribute__((always_inline)) -> bool {
    scores(std::true_type{}, kb, e8m0_f32(ke));
    __builtin_amdgcn_sched_barrier(0);
    load_values(kb);
    load_keys(next, 0, k0);
    __builtin_amdgcn_sched_barrier(0);
    if (__ballot(exponentials(std::true_type{}, ref, kSeen) > kLazy)) return false;
    l += sum;
    __builtin_amdgcn_sched_barrier(0);
    products(e8m0_f32(ve));
    return true;
  };
  // any other: one that some row does not see whole, without a page, or whose scale makes no numbers
  auto edge_block = [&](const uint8_t* kb, int t0, bool good, uint32_t ke, uint32_t ve) __attribute__((always_inline)) {
    load_keys(kb, 0, k0);
    scores(std::false_type{}, kb, e8m0_f32(ke));
    // of the lane's tokens, counted from t0 + 4 hl: those before see_hi, from see_lo on
    const int see_hi = (good ? row_hi : 0) - t0 - 4 * hl, see_lo = row_lo - t0 - 4 * hl;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = 32 * t + 8 * (i >> 2) + (i & 3);
        s[t][i] = at < see_hi && at >= see_lo ? (ke == 255u ? NAN : s[t][i]) : -INFINITY;
      }
    move();
    exponentials(std::false_type{}, ref, min(good ? row_hi : 0, t0 + kBlock) > max(row_lo, t0) ? kSeen : 0.f);
    l += sum;
    __builtin_amdgcn_sched_barrier(0);
    load_values(kb);
    // A code that is not a finite number reaches only the rows that see its token (see
    // the kernel above): it is taken out, and where a count of the seen ones is not
    // zero, the result is not a number.
    const uint32_t from = bad_from(ve);
    uint32_t any = 0u;
#pragma unroll
    for (int j = 0; j < DQ; ++j)
#pragma unroll
      for (int w = 0; w < 8; ++w) any |= (vw[j][w >> 2][w & 3] & 0x7F7F7F7Fu) + from;
    if (__ballot((any & 0x80808080u) != 0u)) {
      bf16x8_t see[4];
#pragma unroll
      for (int w = 0; w < 4; ++w)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int at = 16 * w + 8 * (i >> 2) + (i & 3);
          see[w][i] = (__bf16)(at < see_hi && at >= see_lo ? 1.f : 0.f);
        }
#pragma unroll
      for (int j = 0; j < DQ; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        f32x16_t n = zero;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t ba = bad_bytes(vw[j][0][w], from), bb = bad_bytes(vw[j][1][w], from);
          n = __builtin_amdgcn_mfma_f32_32x32x16_bf16(to_bf16(ba & 0x38383838u, bb & 0x38383838u, 1.f), see[w], n, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) o[j][i] = n[i] > 0.f ? NAN : o[j][i];
      }
      __builtin_amdgcn_sched_barrier(0);
      load_values(kb);
#pragma unroll
      for (int j = 0; j < DQ; ++j)
#pragma unroll
        for (int w = 0; w < 8; ++w) vw[j][w >> 2][w & 3] &= ~bad_bytes(vw[j][w >> 2][w & 3], from);
    }
    products(ve == 255u ? 1.f : e8m0_f32(ve));
  };

  if (nblk > 0) {
    // Turn b begins when blocks b and b + 1 are in LDS (the keys of b + 1 are read
    // in it) and everyone is done with b - 1, whose stage takes block b + 3.
    // Whole blocks run in a loop of their own, in which O stays where it is in
    // registers; the others leave it for one turn.
    load_meta(0);
    uint32_t sc = 0u, sc1, sc2;
    src = locate(0);
    sc1 = sc_in;
    lds_copies<CPW>(src, lane16, lds0);
    src = locate(1);
    sc2 = sc_in;
    lds_copies<CPW>(src, lane16, lds0 + STAGE);
    src = locate(2);
    lds_copies<CPW>(src, lane16, lds0 + 2 * STAGE);
    dst = lds0 + 2 * STAGE;
    stage_ready<2 * CPW>();
    load_keys(buf, 0, k0);
    const uint8_t *kb = buf, *next = buf + STAGE;
    int b = 0, t0 = 0;
    auto arrive = [&]() __attribute__((always_inline)) {
      stage_ready<CPW>();
      sc = sc1;
      sc1 = sc2;
      sc2 = sc_in;
      src = locate(b + 3);
      dst = dst == lds0 + (STAGES - 1) * STAGE ? lds0 : dst + STAGE;
      t0 = (b0 + b) * kBlock;
    };
    auto leave = [&]() __attribute__((always_inline)) {
      ++b;
      kb = next;
      next = next == buf + (STAGES - 1) * STAGE ? buf : next + STAGE;
    };
    bool again = false;
    while (b < nblk) {
      bool edge = false;
      for (; b < nblk; leave()) {
        if (!again) arrive();
        edge = t0 + kBlock > all_hi || t0 < all_lo || sc >= kOverflow << 8 || (sc & 0xFFu) == 255u;
        if (edge) break;
        const bool done = whole_block(kb, next, sc & 0xFFu, sc >> 8);
        edge = !done && again;  // scores so large that a rounding of them is more than 8: two roundings
        again = !done && !again;
        if (!done) break;
      }
      if (again) {  // move the references, then the block once more (its copies too, to the same place)
        load_keys(kb, 0, k0);
        scores(std::false_type{}, kb, e8m0_f32(sc & 0xFFu));
        move();
        load_keys(kb, 0, k0);
      } else if (edge) {
        lds_copies<CPW>(src, lane16, dst);
        const bool good = sc != ~0u;
        if (t0 < any_hi && t0 + kBlock > any_lo)
          edge_block(kb, t0, good, good ? sc & 0xFFu : 127u, good ? sc >> 8 : 127u);
        load_keys(next, 0, k0);
        leave();
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy outlives the workgroup
  }
  l = half_sum(l);
  if (gridDim.y == 1) {
    if (own_row) {
      const float inv = row_factor(a, head, ref, l);
      uint16_t* orow = a.out + ((int64_t)(x.s0 + tok) * a.hq + head) * D;
#pragma unroll
      for (int j = 0; j < DQ; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // dims 8 (2 i + hl) .. + 7 of 32: four of them are the other half's
          uint32_t w[2][2];
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int n = 0; n < 2; ++n)
              w[k][n] = (uint32_t)f32_bf16(o[j][4 * (2 * i + k) + 2 * n] * inv) |
                        ((uint32_t)f32_bf16(o[j][4 * (2 * i + k) + 2 * n + 1] * inv) << 16);
          const auto r0 = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
          const auto r1 = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
          *reinterpret_cast<u32x4_t*>(orow + 32 * j + 8 * (2 * i + hl)) = u32x4_t{r0[0], r1[0], r0[1], r1[1]};
        }
    }
    return;
  }
  const int64_t base = ((int64_t)(want * a.hkv + h) * gridDim.y + blockIdx.y) * (ROWS / 16);
  if (own_row) {
    const int64_t slot = base + in_tile / 16, at = in_tile % 16;
#pragma unroll
    for (int j = 0; j < DQ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4_t*>(a.tile_o + (slot * 16 + at) * D + 32 * j + 8 * i + 4 * hl) =
            f32x4_t{o[j][4 * i], o[j][4 * i + 1], o[j][4 * i + 2], o[j][4 * i + 3]};
    if (hl == 0) {
      a.tile_ml[slot * 32 + at] = ref;
      a.tile_ml[slot * 32 + 16 + at] = l;
    }
  }
  if (blockIdx.y == 0 && tid == 0) {
    int32_t* t = a.tile_info + 8 + ((int64_t)want * a.hkv + h) * 8;
    t[0] = (x.s0 + row0 / a.group) * a.group + row0 % a.group;
    t[1] = rows;
    t[2] = gridDim.y;
    t[3] = (int)base;
    t[4] = (int)base + ROWS / 16;
    t[5] = ROWS / 16;
  }
}

// A prompt of 4096 tokens, 64 heads on 8 of 128: 293 us, 937 TFLOP/s (matrix units busy 44% of the
// cycles).  At a head dim of 128 two waves a SIMD leave 52 registers spilled, at 256 one wave
// 103, in the paths of edge blocks and of those done again.
template <int D, int NW>
__global__ void __launch_bounds__(64 * NW, D == 256 ? 1 : 2) paged_attn_tile_kernel(const AttnArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[kTileLds<D>];
  tile_body<D, NW>(a, lds, blockIdx.x, gridDim.x);
}
// Both kinds in one launch, the few-row workgroups first: a stream of the cache
// beside products.
template <int D, int NW>
__global__ void __launch_bounds__(64 * NW, D == 256 ? 1 : 2) paged_attn_both_kernel(const AttnArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[kTileLds<D> > kRowsLds<D, NW> ? kTileLds<D> : kRowsLds<D, NW>];
  if (blockIdx.x >= kGroups)
    tile_body<D, NW>(a, lds, blockIdx.x - kGroups, gridDim.x - kGroups);
  else if (blockIdx.y == 0)
    rows_body<D, NW>(a, lds, kGroups);
}

constexpr int kTileWaves = 4, kTileRows = 32 * kTileWaves;
// Tiles of many rows are cut where there are clearly fewer than this many (as many workgroups as are
// resident; half of it for a head dim of 256), and into pieces of no fewer
// blocks, by what the tables and the window let a tile see.  A prompt of 2000 tokens, 8 heads on 8 of
// 128, with 32, 16 and 8: 48.4, 40.8 and 42.9 us; two of up to 1190, 7 heads on one: 32.8, 30.2 and 37.0.
constexpr int kSplitGroups = 512, kSplitBlocks = 16;

// How a call is carried out, by its sizes alone (the lengths are on the GPU).
struct Plan {
  bool few, many;      // which kernels run
  bool whole, narrow;  // few-row tiles are not cut; two workgroups a CU share the work
  int rows_max;        // requests of up to so many rows are the few-row kernel's
  int64_t few_tiles, many_tiles, splits;  // bounds of the tiles a head; splits: workgroups a many-row tile
  int64_t o, ml, info, tile_o, tile_ml, tile_info, total;  // workspace
};

Plan plan_of(int64_t tokens, int64_t requests, int64_t hq, int64_t hkv, int64_t d, int64_t width_blocks,
             int64_t max_new, int64_t window) {
  Plan p{};
  const int64_t group = hq / hkv, most = (max_new && max_new < tokens ? max_new : tokens) * group;
  const int64_t some = requests < tokens ? requests : tokens;  // requests with rows
  p.many = some > 0 && most > kRows;
  p.few = !p.many || requests > 1;
  p.rows_max = !p.many ? INT_MAX : p.few ? kRows : 0;
  p.whole = width_blocks <= kWhole;
  p.few_tiles = p.few ? (p.many ? some : tokens * group / kRows + some) : 0;
  p.many_tiles = p.many ? tokens * group / kTileRows + some : 0;
  p.splits = 1;
  if (p.many) {
    const int64_t groups = p.many_tiles * hkv;
    const int64_t resident = d == 256 ? kSplitGroups / 2 : kSplitGroups;
    p.splits = (resident + groups / 2) / groups;
    // a tile's last row sees `window` tokens, its first as many from up to a tile's rows before
    const int64_t seen = window ? (window + kTileRows / group) / kBlock + 2 : width_blocks;
    const int64_t blocks = seen < width_blocks ? seen : width_blocks;
    if (p.splits > blocks / kSplitBlocks) p.splits = blocks / kSplitBlocks;
    if (p.splits > 16) p.splits = 16;
    if (p.splits < 1) p.splits = 1;
  }
  p.narrow = p.few && !p.many && width_blocks <= kNarrow && p.few_tiles * hkv > kGroups;
  const int64_t slots = p.few && !p.whole ? 2 * kGroups : 0;
  const int64_t tile_slots = p.splits > 1 ? p.many_tiles * hkv * p.splits * (kTileRows / kRows) : 0;
  p.o = 0;
  p.ml = p.o + slots * kRows * d * 4;
  p.info = p.ml + slots * 2 * kRows * 4;
  p.tile_o = p.info + (p.few && !p.whole ? 32 + p.few_tiles * hkv * 32 : 0);
  p.tile_ml = p.tile_o + tile_slots * kRows * d * 4;
  p.tile_info = p.tile_ml + tile_slots * 2 * kRows * 4;
  p.total = p.tile_info + (p.splits > 1 ? 32 + p.many_tiles * hkv * 32 : 0);
  return p;
}

template <int D, int NW>
int launch(const AttnArgs& a, const Plan& p, int few_rows, hipStream_t st) {
  const unsigned tiles = (unsigned)(p.many_tiles * a.hkv), splits = (unsigned)p.splits;
  if (p.few && p.many)
    MOSAIC_LAUNCH((paged_attn_both_kernel<D, kTileWaves>), dim3(kGroups + tiles, splits), dim3(64 * kTileWaves), 0, st, a);
  else if (p.few && p.narrow)
    MOSAIC_LAUNCH((paged_attn_rows_kernel<D, 4>), dim3(NW / 4 * kGroups), dim3(256), 0, st, a);
  else if (p.few)
    MOSAIC_LAUNCH((paged_attn_rows_kernel<D, NW>), dim3(kGroups), dim3(64 * NW), 0, st, a);
  else
    MOSAIC_LAUNCH((paged_attn_tile_kernel<D, kTileWaves>), dim3(tiles, splits), dim3(64 * kTileWaves), 0, st, a);
  MOSAIC_LAUNCH_CHECK("paged_attention");
  if (p.few && !p.whole) {
    // few tiles are cut into many pieces: a workgroup for each row of theirs
    const int z = p.few_tiles * a.hkv <= 64 ? few_rows : (few_rows * D + 1023) / 1024;
    MOSAIC_LAUNCH(paged_attn_join_kernel<D>, dim3((unsigned)p.few_tiles, (unsigned)a.hkv, (unsigned)z), dim3(256), 0, st,
                  a, (const int32_t*)a.info);
    MOSAIC_LAUNCH_CHECK("paged_attention");
  }
  if (p.splits > 1) {
    AttnArgs t = a;
    t.part_o = a.tile_o;
    t.part_ml = a.tile_ml;
    MOSAIC_LAUNCH(paged_attn_join_kernel<D>, dim3((unsigned)p.many_tiles, (unsigned)a.hkv, kTileRows * D / 1024),
                  dim3(256), 0, st, t, (const int32_t*)a.tile_info);
    MOSAIC_LAUNCH_CHECK("paged_attention");
  }
  return kOk;
}

bool valid(int64_t tokens, int64_t requests, int64_t hq, int64_t hkv, int64_t d) {
  return tokens >= 0 && tokens < (1 << 21) && requests >= 0 && requests <= (1 << 20) && hkv >= 1 && hkv <= 65535 &&
         hq >= hkv && hq <= 65535 && hq % hkv == 0 && tokens * (hq / hkv) < (1ll << 31) && (d == 64 || d == 128 || d == 256);
}

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" size_t mosaic_paged_attention_workspace_bytes(int64_t tokens, int64_t requests, int64_t q_heads,
                                                         int64_t kv_heads, int64_t head_dim, int64_t blocks,
                                                         int64_t width, int64_t max_new) {
  if (!valid(tokens, requests, q_heads, kv_heads, head_dim) || blocks < 1 || width < 1 || max_new < 0) return 0;
  return (size_t)plan_of(tokens, requests, q_heads, kv_heads, head_dim, width * blocks, max_new, 0).total;
}

extern "C" int mosaic_paged_attention(const uint16_t* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                                      int64_t q_heads, const uint8_t* codes, const uint8_t* scales, int64_t pages,
                                      int64_t blocks, int64_t kv_heads, int64_t head_dim, const int32_t* block_table,
                                      int64_t table_stride, int64_t width, const int32_t* starts,
                                      const int32_t* seq_lens, int64_t requests, const float* sink, int64_t window,
                                      int64_t max_new, float softmax_scale, uint16_t* out, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  MOSAIC_CHECK_ARG(valid(tokens, requests, q_heads, kv_heads, head_dim),
                   "paged_attention: %lld query heads on %lld key heads of %lld (64, 128 or 256), %lld tokens (below "
                   "2^21) of %lld requests",
                   (long long)q_heads, (long long)kv_heads, (long long)head_dim, (long long)tokens, (long long)requests);
  MOSAIC_CHECK_ARG(pages >= 1 && pages < (1ll << 31) && blocks >= 1 && blocks <= 64,
                   "paged_attention: %lld pages of %lld blocks", (long long)pages, (long long)blocks);
  MOSAIC_CHECK_ARG(width >= 1 && width * blocks * kBlock < (1ll << 30) && table_stride >= width,
                   "paged_attention: tables of %lld pages", (long long)width);
  MOSAIC_CHECK_ARG(window >= 0 && window < (1ll << 31), "paged_attention: window %lld", (long long)window);
  MOSAIC_CHECK_ARG(max_new >= 0, "paged_attention: max_new %lld", (long long)max_new);
  MOSAIC_CHECK_ARG(std::isfinite(softmax_scale), "paged_attention: the softmax scale is not finite");
  if (tokens == 0) return kOk;
  MOSAIC_CHECK_ARG(q && out && starts && (requests == 0 || (block_table && seq_lens)) && codes && scales,
                   "paged_attention: null pointer");
  MOSAIC_CHECK_ARG(((uintptr_t)q | (uintptr_t)out | (uintptr_t)codes | (uintptr_t)workspace) % 16 == 0 &&
                       (uintptr_t)scales % 2 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0,
                   "paged_attention: q, out, codes and the workspace are read and written 16 bytes at a time");
  const Plan p = plan_of(tokens, requests, q_heads, kv_heads, head_dim, width * blocks, max_new, window);
  MOSAIC_CHECK_ARG(p.total == 0 || (workspace && workspace_bytes >= (size_t)p.total),
                   "paged_attention: workspace of %lld bytes, %lld needed",
                   (long long)workspace_bytes, (long long)p.total);
  // the few-row kernel numbers its (tile, head, block) units in 32 bits, a launch its threads
  MOSAIC_CHECK_ARG(p.few_tiles * kv_heads < (1ll << 31) / (kStart + width * blocks) &&
                       (p.many_tiles * kv_heads + kGroups) * 64 * kTileWaves < (1ll << 32),
                   "paged_attention: %lld row tiles over tables of %lld blocks are too many for one call",
                   (long long)((p.few_tiles + p.many_tiles) * kv_heads), (long long)(width * blocks));
  const uint16_t* q_end = q + (tokens - 1) * q_token_stride + (q_heads - 1) * q_head_stride + head_dim;
  MOSAIC_CHECK_ARG(q_end <= out || out + tokens * q_heads * head_dim <= q, "paged_attention: out overlaps q");
  AttnArgs a{};
  a.q = q;
  a.codes = codes;
  a.scales = scales;
  a.table = block_table;
  a.starts = starts;
  a.seq = seq_lens;
  a.sink = sink;
  a.out = out;
  char* ws = (char*)workspace;
  a.part_o = (float*)(ws + p.o);
  a.part_ml = (float*)(ws + p.ml);
  a.info = (int32_t*)(ws + p.info);
  a.tile_o = (float*)(ws + p.tile_o);
  a.tile_ml = (float*)(ws + p.tile_ml);
  a.tile_info = (int32_t*)(ws + p.tile_info);
  a.rows_max = p.rows_max;
  a.few_cap = (uint32_t)p.few_tiles;
  a.many_cap = (uint32_t)p.many_tiles;
  a.whole = p.whole;
  a.zero_rows = !p.few;
  a.q_tok = q_token_stride;
  a.q_head = q_head_stride;
  a.stride = table_stride;
  a.r = (int)requests;
  a.tokens = (int)tokens;
  a.hq = (int)q_heads;
  a.hkv = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.width = (int)width;
  a.pages = (int)pages;
  a.nb = (int)blocks;
  a.window = window >= (1 << 30) ? 0 : (int)window;  // longer than any context: none
  // Finite and not zero, or a score of 0, or a masked one, would be no number: a scale of zero is fp32's
  // least number, which brings no product of fp32's range to more than 2^-21.
  a.scale = fminf(fmaxf(fabsf(softmax_scale) * kLog2e, 0x1p-149f), -kLowest);
  a.sign = softmax_scale < 0.f ? -1.f : 1.f;
  const int64_t rows = (max_new && max_new < tokens ? max_new : tokens) * a.group;
  const int few_rows = (int)(rows < kRows ? rows : kRows);
  switch (head_dim) {
    case 64: return launch<64, 8>(a, p, few_rows, (hipStream_t)stream);
    case 128: return launch<128, 8>(a, p, few_rows, (hipStream_t)stream);
    default: return launch<256, 4>(a, p, few_rows, (hipStream_t)stream);
  }
}
