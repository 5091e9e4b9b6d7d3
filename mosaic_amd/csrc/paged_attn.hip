// Attention over the paged 8-bit cache (layout: paged_kv.hip): each query row of
// a ragged batch sees its request's tokens up to its own position, optionally
// only the last `window` of them, with an optional sink logit for each head.
//
//   s = scale q . k in fp32 (k = code 2^(e - 127), exact in bf16), running
//   maximum and sum of exp(s - m) in fp32, o = sum p v / (sum p + exp(sink - m)).
//   p is rounded to bf16 for the matrix unit's value product (its sum is not):
//   an error of at most 2^-9 a term, of either sign, against the 2^-9 of the
//   bf16 output itself.
//
// Rows of one key head (tokens x query heads of its group) are tiled by 16.  A
// work unit is a (request, key head, row tile, block of 64 tokens); the units of
// all requests are numbered through and each workgroup takes an equal run of
// them, so the lengths may be as unequal as they like.  A run's piece of one tile
// is a segment: eight waves take its blocks in turn, keep (m, l, O) in registers
// and meet in LDS at its end.  A tile in one segment is finished there; one that
// is cut at a run's border leaves partial sums that paged_attn_join_kernel adds up.
//
// Scores are computed transposed, S^T = K Q^T (16 tokens x 16 rows a tile): lane
// (q, c) then holds four tokens of row c, which are its own operand of
// O^T = V^T P^T; the cache stores the values in that order, so neither keys,
// values nor probabilities pass through LDS or between lanes.
#include <cmath>

#include "common.h"
#include "../../include/mosaic_amd.h"

namespace mosaic {
namespace {

constexpr int kBlock = 64;
constexpr int kRows = 16;           // rows of a tile
constexpr int kGroups = 512;        // workgroups of a launch (two a CU)
constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  const uint16_t* q;
  const uint8_t *codes, *scales;
  const int32_t *table, *starts, *seq;
  const float* sink;
  uint16_t* out;
  float* part_o;   // [2 kGroups][16][D], unnormalized
  float* part_ml;  // [2 kGroups][2][16]
  int32_t* info;   // [0]: tiles; from [4]: [tiles][Hkv][4]: first row, rows, the runs of its first and last piece
  int64_t q_tok, q_head, stride;
  int r, tokens, hq, hkv, group, width, pages, nb, window, tiles;
  float scale;  // softmax scale times log2(e)
};

struct Request {
  int s0, n, held, first, blocks, tiles;  // first: the first block that any row sees
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
    x.tiles = (x.n * a.group + kRows - 1) / kRows;
  }
  return x;
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

// eight codes (two words) times 2^n, exact in bf16
__device__ __forceinline__ bf16x8_t to_bf16(uint32_t w0, uint32_t w1, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 0xFF in every byte of w that is a NaN code (0x7F or 0xFF)
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t x = (w & 0x7F7F7F7Fu) + 0x01010101u;  // the high bit of a byte: it was 0x7F
  return ((x & 0x80808080u) >> 7) * 0xFFu;
}

template <int D, int NW>
__global__ void __launch_bounds__(64 * NW) paged_attn_rows_kernel(const AttnArgs a) {
  constexpr int DG = D / 64, DT = D / 16;
  __shared__ __attribute__((aligned(16))) f32x4_t so[NW / 2][DT * 4 * 16];
  __shared__ float sm[NW][16], sl[NW][16];
  __shared__ uint32_t sums[NW], sums_t[NW], s_unit;
  __shared__ int s_req, s_tile;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, c = lane & 15;

  // every workgroup counts the units of all requests; then the one that holds its run's first unit
  uint32_t total = 0, tiles_all = 0;
  for (int base = 0; base < a.r; base += 64 * NW) {
    const Request x = request_of(a, base + tid);
    const uint32_t n = (uint32_t)(x.tiles * a.hkv) * (uint32_t)x.blocks;
    const uint32_t incl = wave_incl_scan_u32(n), tinc = wave_incl_scan_u32((uint32_t)x.tiles);
    if (lane == 63) {
      sums[wave] = incl;
      sums_t[wave] = tinc;
    }
    __syncthreads();
    for (int w = 0; w < NW; ++w) {
      total += sums[w];
      tiles_all += sums_t[w];
    }
    __syncthreads();
  }
  const uint32_t share = max((total + kGroups - 1) / kGroups, (uint32_t)NW / 2);
  const uint32_t u0 = blockIdx.x * share, u1 = min(u0 + share, total);
  if (blockIdx.x == 0) {  // rows behind the last request are zero
    if (tid == 0) a.info[0] = (int32_t)tiles_all;
    const int64_t from = a.r ? min(max(a.starts[a.r], 0), a.tokens) : 0;
    const int64_t per = (int64_t)a.hq * D;
    for (int64_t i = from * per + 8 * tid; i < a.tokens * per; i += 8 * 64 * NW)
      *reinterpret_cast<u32x4_t*>(a.out + i) = u32x4_t{0u, 0u, 0u, 0u};
  }
  if (u0 >= total) return;
  {
    uint32_t seen = 0;
    uint32_t tiles = 0;
    for (int base = 0; base < a.r; base += 64 * NW) {
      const Request x = request_of(a, base + tid);
      const uint32_t n = (uint32_t)(x.tiles * a.hkv) * (uint32_t)x.blocks;
      const uint32_t incl = wave_incl_scan_u32(n), tinc = wave_incl_scan_u32((uint32_t)x.tiles);
      if (lane == 63) {
        sums[wave] = incl;
        sums_t[wave] = tinc;
      }
      __syncthreads();
      uint32_t at = seen, t_at = tiles;
      for (int w = 0; w < NW; ++w) {
        if (w < wave) {
          at += sums[w];
          t_at += sums_t[w];
        }
        seen += sums[w];
        tiles += sums_t[w];
      }
      at += incl - n;
      if (u0 >= at && u0 - at < n) {
        s_req = base + tid;
        s_unit = at;
        s_tile = (int)(t_at + tinc) - x.tiles;
      }
      __syncthreads();
      if (seen > u0) break;
    }
  }
  __syncthreads();
  int r = s_req, tile0 = s_tile;
  uint32_t req0 = s_unit;
  Request x = request_of(a, r);
    for (uint32_t u = u0; u < u1;) {
    while (u - req0 >= (uint32_t)(x.tiles * a.hkv) * (uint32_t)x.blocks) {
      req0 += (uint32_t)(x.tiles * a.hkv) * (uint32_t)x.blocks;
      tile0 += x.tiles;
      x = request_of(a, ++r);
    }
    // unit -> (head, tile, block), blocks fastest
    const uint32_t in = u - req0, ht = in / (uint32_t)x.blocks;
    const int b_from = (int)(in % (uint32_t)x.blocks), b_to = (int)min((uint32_t)x.blocks, (uint32_t)b_from + (u1 - u));
    const int h = (int)(ht / (uint32_t)x.tiles), tile = (int)(ht % (uint32_t)x.tiles);
    const uint32_t tile_u0 = u - b_from;
    u += b_to - b_from;
    const int row0 = tile * kRows, rows = min(kRows, x.n * a.group - row0);
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
    float m = -INFINITY, l = 0.f;
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
      // a block that some row does not see whole, one without a page, or of a NaN scale
      const bool edge = t0 + kBlock > all_hi || t0 < all_lo || !good || ke == 255u || ve == 255u;
      const int hi = good ? row_hi : 0;
      float bm = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = s[t][i] * a.scale;
          if (edge) {
            const int p = t0 + 16 * t + 4 * q + i;
            v = ke == 255u ? NAN : v;
            v = p < hi && p >= row_lo ? v : -INFINITY;
          }
          s[t][i] = v;
          bm = fmaxf(bm, v);
        }
      bm = lane4_max(bm);
      const float mn = fmaxf(m, bm);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float alpha = __builtin_amdgcn_exp2f(m - ref);
      m = mn;
      bf16x8_t p[2];
      float sum = 0.f;
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
        // A code that is not a number reaches only the rows that see its token: it is
        // taken out of the product (zero times it would reach all), and where a
        // count of the seen ones is not zero, the result is not a number.
        uint32_t any = 0u;
#pragma unroll
        for (int j = 0; j < DT; ++j)
#pragma unroll
          for (int w = 0; w < 4; ++w) any |= nan_bytes(vw[j][w]);
        if (__ballot(any != 0u || ve == 255u)) {
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
              bad[w] = ve == 255u ? 0xFFFFFFFFu : nan_bytes(vw[j][w]);
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
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w][c]);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int w = 0; w < NW; ++w) L += sl[w][c] * __builtin_amdgcn_exp2f(sm[w][c] - ref);
    const float f = __builtin_amdgcn_exp2f(m - ref);
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
    if (b_from == 0 && tid == 0) {  // the join's list: this tile's rows and the runs that hold it
      int32_t* t = a.info + 4 + ((int64_t)(tile0 + tile) * a.hkv + h) * 4;
      t[0] = (x.s0 + row0 / a.group) * a.group + row0 % a.group;
      t[1] = rows;
      t[2] = (int)blockIdx.x;
      t[3] = (int)((tile_u0 + x.blocks - 1) / share);
    }
    float inv = 0.f;
    if (whole) {
      // thread -> (4 dims, row c): c stays tid's
      const float s_ = a.sink ? a.sink[head] * kLog2e : -INFINITY;
      // a row without keys is zero, whatever its sink
      const float den = L + __builtin_amdgcn_exp2f(s_ - ref);
      inv = M == -INFINITY ? L : 1.f / den;  // L is 0 there, or not a number where every score is not
    }
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

// Adds up the pieces of a tile that was cut: one workgroup a row, its 256
// threads as groups of D / 4 lanes (four dims each) that take the pieces in turn.
template <int D>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(const AttnArgs a) {
  constexpr int LANES = D / 4, SG = 256 / LANES;
  __shared__ f32x4_t so[SG][LANES];
  __shared__ float red[4][2];
  const int tile = blockIdx.x, h = blockIdx.y, c = blockIdx.z, tid = threadIdx.x;
  if (tile >= a.info[0]) return;
  const int32_t* t = a.info + 4 + ((int64_t)tile * a.hkv + h) * 4;
  const int w0 = t[2], w1 = t[3];
  if (w0 == w1 || c >= t[1]) return;
  const int row = t[0] + c, head = h * a.group + row % a.group;
  auto slot = [&](int i) { return (int64_t)(i == 0 ? 2 * w0 + 1 : 2 * (w0 + i)); };
  const int n = w1 - w0 + 1;
  float m = -INFINITY;
  for (int i = tid; i < n; i += 256) m = fmaxf(m, a.part_ml[slot(i) * 32 + c]);
  m = wave_max_f32(m);
  if ((tid & 63) == 0) red[tid >> 6][0] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
  const float ref = m == -INFINITY ? 0.f : m;
  const int g = tid / LANES, d = tid % LANES;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 8
  for (int i = g; i < n; i += SG) {
    const float f = __builtin_amdgcn_exp2f(a.part_ml[slot(i) * 32 + c] - ref);
    l += f * a.part_ml[slot(i) * 32 + 16 + c];
    o += *reinterpret_cast<const f32x4_t*>(a.part_o + (slot(i) * 16 + c) * D + 4 * d) * f;
  }
  __shared__ float ls[SG];
  so[g][d] = o;
  if (d == 0) ls[g] = l;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int i = 1; i < SG; ++i) {
    o += so[i][d];
    l += ls[i];
  }
  const float s_ = a.sink ? a.sink[head] * kLog2e : -INFINITY;
  const float inv = m == -INFINITY ? l : 1.f / (l + __builtin_amdgcn_exp2f(s_ - ref));
  uint2 pk;
  pk.x = (uint32_t)f32_bf16(o[0] * inv) | ((uint32_t)f32_bf16(o[1] * inv) << 16);
  pk.y = (uint32_t)f32_bf16(o[2] * inv) | ((uint32_t)f32_bf16(o[3] * inv) << 16);
  *reinterpret_cast<uint2*>(a.out + ((int64_t)(row / a.group) * a.hq + head) * D + 4 * d) = pk;
}

struct Sizes {
  int64_t tiles, info, part_o, part_ml, total;
};

Sizes sizes(int64_t tokens, int64_t requests, int64_t hq, int64_t hkv, int64_t d) {
  Sizes s;
  s.tiles = tokens * (hq / hkv) / kRows + (requests < tokens ? requests : tokens);
  s.part_o = (int64_t)2 * kGroups * kRows * d * 4;
  s.part_ml = (int64_t)2 * kGroups * 2 * kRows * 4;
  s.info = 16 + s.tiles * hkv * 16;
  s.total = s.part_o + s.part_ml + s.info;
  return s;
}

template <int D, int NW>
int launch(const AttnArgs& a, int rows, hipStream_t st) {
  MOSAIC_LAUNCH((paged_attn_rows_kernel<D, NW>), dim3(kGroups), dim3(64 * NW), 0, st, a);
  MOSAIC_LAUNCH_CHECK("paged_attention");
  MOSAIC_LAUNCH(paged_attn_join_kernel<D>, dim3((unsigned)a.tiles, (unsigned)a.hkv, (unsigned)rows), dim3(256), 0, st, a);
  MOSAIC_RETURN_LAUNCH("paged_attention");
}

bool valid(int64_t tokens, int64_t requests, int64_t hq, int64_t hkv, int64_t d) {
  return tokens >= 0 && tokens < (1 << 21) && requests >= 0 && requests <= (1 << 20) && hkv >= 1 && hkv <= 65535 &&
         hq >= hkv && hq <= 65535 && hq % hkv == 0 && (d == 64 || d == 128 || d == 256);
}

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" size_t mosaic_paged_attention_workspace_bytes(int64_t tokens, int64_t requests, int64_t q_heads,
                                                         int64_t kv_heads, int64_t head_dim) {
  if (!valid(tokens, requests, q_heads, kv_heads, head_dim)) return 0;
  return (size_t)sizes(tokens, requests, q_heads, kv_heads, head_dim).total;
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
  MOSAIC_CHECK_ARG(pages >= 0 && pages < (1ll << 31) && blocks >= 1 && blocks <= 64,
                   "paged_attention: %lld pages of %lld blocks", (long long)pages, (long long)blocks);
  MOSAIC_CHECK_ARG(width >= 1 && width * blocks * kBlock < (1ll << 30) && table_stride >= width,
                   "paged_attention: tables of %lld pages", (long long)width);
  MOSAIC_CHECK_ARG(window >= 0 && window < (1ll << 31), "paged_attention: window %lld", (long long)window);
  MOSAIC_CHECK_ARG(max_new >= 0, "paged_attention: max_new %lld", (long long)max_new);
  MOSAIC_CHECK_ARG(std::isfinite(softmax_scale), "paged_attention: the softmax scale is not finite");
  if (tokens == 0) return kOk;
  MOSAIC_CHECK_ARG(q && out && starts && workspace && (requests == 0 || (block_table && seq_lens)) &&
                       (pages == 0 || (codes && scales)),
                   "paged_attention: null pointer");
  MOSAIC_CHECK_ARG(((uintptr_t)q | (uintptr_t)out | (uintptr_t)codes | (uintptr_t)workspace) % 16 == 0 &&
                       (uintptr_t)scales % 2 == 0 && q_token_stride % 8 == 0 && q_head_stride % 8 == 0,
                   "paged_attention: q, out, codes and the workspace are read and written 16 bytes at a time");
  const Sizes s = sizes(tokens, requests, q_heads, kv_heads, head_dim);
  MOSAIC_CHECK_ARG(workspace_bytes >= (size_t)s.total, "paged_attention: workspace of %lld bytes, %lld needed",
                   (long long)workspace_bytes, (long long)s.total);
  MOSAIC_CHECK_ARG(s.tiles * kv_heads < (1ll << 31) / (width * blocks),
                   "paged_attention: %lld row tiles over tables of %lld blocks are too many for one call",
                   (long long)(s.tiles * kv_heads), (long long)(width * blocks));
  AttnArgs a{};
  a.q = q;
  a.codes = codes;
  a.scales = scales;
  a.table = block_table;
  a.starts = starts;
  a.seq = seq_lens;
  a.sink = sink;
  a.out = out;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + s.part_o / 4;
  a.info = (int32_t*)(a.part_ml + s.part_ml / 4);
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
  a.window = (int)window;
  a.tiles = (int)s.tiles;
  a.scale = softmax_scale * kLog2e;
  const int64_t rows = (max_new && max_new < tokens ? max_new : tokens) * a.group;
  const int z = (int)(rows < kRows ? rows : kRows);
  switch (head_dim) {
    case 64: return launch<64, 8>(a, z, (hipStream_t)stream);
    case 128: return launch<128, 8>(a, z, (hipStream_t)stream);
    default: return launch<256, 4>(a, z, (hipStream_t)stream);
  }
}
