// A paged KV cache in 8 bits: block tables and slot maps from request lengths,
// the release of pages, and the writer of new keys and values.
//
// Cache: codes [P, NB, Hkv, 2, 64 D] e4m3 and scales [P, NB, Hkv, 2] e8m0 (value
// 2^(byte - 127)).  A page is NB blocks of 64 tokens; a block and head has one
// scale for its keys and one for its values.  The 64 D bytes of a block are in
// the order in which the attention's matrix operands take them, so that a wave
// loads whole runs of 1 KB (16 bytes a lane) straight into registers:
//   keys    [4 tg][D/64 dg][4 q][16 c][16 j]: token 16 tg + c, dim 64 dg + 16 q + j
//   values  [D/16 dt][4 q][16 c][4 w][4 j]:   token 16 w + 4 q + j, dim 16 dt + c
// Values are stored transposed, four consecutive tokens a word: these are the
// tokens whose probabilities a lane of the score tile holds.
#include <type_traits>

#include "common.h"
#include "../../include/mosaic_amd.h"

namespace mosaic {
namespace {

constexpr int kBlock = 64;   // tokens of a scale
constexpr int kRows = 1024;  // token rows a workgroup of the step

// Exclusive prefix of v over the workgroup's 256 threads; `sums`: four words of
// LDS.  total: the sum over all of them.  Two barriers.
__device__ __forceinline__ uint32_t block_excl_scan(uint32_t v, uint32_t* sums, uint32_t& total) {
  const uint32_t incl = wave_incl_scan_u32(v);
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 63) sums[wave] = incl;
  __syncthreads();
  const uint32_t s0 = sums[0], s1 = sums[1], s2 = sums[2], s3 = sums[3];
  total = s0 + s1 + s2 + s3;
  const uint32_t base = wave == 0 ? 0 : wave == 1 ? s0 : wave == 2 ? s0 + s1 : s0 + s1 + s2;
  __syncthreads();
  return base + incl - v;
}

// The first of TILE (a power of two) ascending values that is greater than x, for N
// x's at once (the steps' LDS latencies overlap); the last if none is.
template <int TILE, int N>
__device__ __forceinline__ void first_above(const uint32_t* a, const uint32_t (&x)[N], int (&at)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) at[i] = 0;
#pragma unroll
  for (int half = TILE / 2; half; half >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) at[i] += a[at[i] + half - 1] <= x[i] ? half : 0;
}

struct StepArgs {
  const int32_t *lengths, *add, *free_pages, *free_count;
  int32_t *table, *starts, *lengths_out, *seq, *positions, *slots, *count_out;
  int64_t stride;
  int r, pages;
  uint32_t ids;  // page ids from here on, and below 0, have no slot: it would not fit
  uint32_t width, page, tokens;
};

// Two prefix sums over the requests (token rows, then pages), and from them every
// output.  Latency-bound: kilobytes of reads and writes.  One launch: each
// workgroup scans all requests by itself (the reads come from L2) and then
// writes its own 1024 token rows, four a thread, and its share of the popped pages, so no
// workgroup waits for another; the outputs may not overlap the inputs for that.
template <int EACH>
__global__ void __launch_bounds__(256) paged_step_kernel(const StepArgs a) {
  constexpr int TILE = 256 * EACH;  // requests of a scan, EACH consecutive ones a thread
  __shared__ uint32_t s_end[TILE], s_take[TILE], s_len[TILE], s_before[TILE], sums[4];
  const int tid = threadIdx.x;
  const uint32_t t0 = blockIdx.x * (uint32_t)kRows, t1 = min(t0 + kRows, a.tokens);
  const uint32_t most = a.width * a.page;
  const uint32_t free = a.free_pages ? (uint32_t)min(max(*a.free_count, 0), a.pages) : 0u;
  uint32_t tok = 0, taken = 0, used = 0;
  for (int base = 0, tile = 0; base < a.r; base += TILE, ++tile) {
    const int r0 = base + EACH * tid;
    uint32_t len[EACH], n[EACH], sum_n = 0, sum_need = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const bool in = r0 + i < a.r;
      len[i] = in ? (uint32_t)max(a.lengths[r0 + i], 0) : 0u;
      // a count past the token rows is as good as one more than they are, and so is a
      // thread's sum: 256 of them stay in 32 bits
      n[i] = in ? min((uint32_t)max(a.add[r0 + i], 0), a.tokens + 1) : 0u;
      sum_n = min(sum_n + n[i], a.tokens + 1);
    }
    uint32_t total, end[EACH], need[EACH], before[EACH];
    uint32_t sum = tok + block_excl_scan(sum_n, sums, total);
    const uint32_t tok_end = min(tok + total, a.tokens + 1);
    bool fits[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      sum += n[i];
      end[i] = sum;
      fits[i] = sum <= a.tokens && len[i] + n[i] <= most;
      before[i] = (len[i] + a.page - 1) / a.page;
      need[i] = fits[i] ? (len[i] + n[i] + a.page - 1) / a.page - before[i] : 0u;
      sum_need += need[i];
    }
    uint32_t pop = taken + block_excl_scan(sum_need, sums, total);
    const uint32_t taken_end = taken + total;
    const bool mine = blockIdx.x == (uint32_t)tile % gridDim.x;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      pop += need[i];
      const bool placed = fits[i] && (!a.free_pages || need[i] == 0 || pop <= free);
      if (placed && need[i] && a.free_pages) used = max(used, pop);
      s_end[EACH * tid + i] = end[i];
      s_take[EACH * tid + i] = pop;
      s_len[EACH * tid + i] = len[i];
      s_before[EACH * tid + i] = before[i] | (placed ? 0x80000000u : 0u);
      if (mine && r0 + i < a.r) {
        a.starts[r0 + i + 1] = (int32_t)min(end[i], a.tokens);
        a.lengths_out[r0 + i] = (int32_t)(placed ? len[i] + n[i] : len[i]);
        a.seq[r0 + i] = (int32_t)(placed ? len[i] + n[i] : 0u);
      }
    }
    __syncthreads();
    if (max(t0, tok) < min(t1, tok_end)) {  // the workgroup has rows of this tile: four a thread
      constexpr int N = kRows / 256;
      uint32_t row[N], slot[N];
      int at[N];
#pragma unroll
      for (int i = 0; i < N; ++i) row[i] = t0 + tid + 256 * i;
      first_above<TILE, N>(s_end, row, at);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t t = row[i], old_pages = s_before[at[i]] & 0x7FFFFFFFu;
        const bool here = t >= tok && t < min(t1, tok_end), placed = here && (s_before[at[i]] >> 31);
        const uint32_t p = s_len[at[i]] + t - (at[i] ? s_end[at[i] - 1] : tok), page = p / a.page;
        int32_t id = 0;
        if (placed) {
          if (page < old_pages || !a.free_pages)
            id = a.table[(int64_t)(base + at[i]) * a.stride + page];
          else
            id = a.free_pages[free - 1 - ((at[i] ? s_take[at[i] - 1] : taken) + page - old_pages)];
        }
        slot[i] = placed && (uint32_t)id < a.ids ? (uint32_t)id * a.page + p % a.page : ~0u;
        if (here) a.positions[t] = placed ? (int32_t)p : -1;
      }
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (row[i] >= tok && row[i] < min(t1, tok_end)) a.slots[row[i]] = (int32_t)slot[i];
    }
    if (a.free_pages)
      for (uint32_t k = taken + blockIdx.x * 256 + tid; k < min(taken_end, free); k += gridDim.x * 256) {
        const uint32_t ks[1] = {k};
        int at[1];
        first_above<TILE, 1>(s_take, ks, at);
        const int i = at[0];
        if (s_before[i] >> 31)
          a.table[(int64_t)(base + i) * a.stride + (s_before[i] & 0x7FFFFFFFu) + k - (i ? s_take[i - 1] : taken)] =
              a.free_pages[free - 1 - k];
      }
    __syncthreads();
    tok = tok_end;
    taken = taken_end;
  }
  for (uint32_t t = max(t0, tok) + tid; t < t1; t += 256) a.positions[t] = a.slots[t] = -1;
  if (blockIdx.x == 0) {
    used = wave_max_u32(used);
    if ((tid & 63) == 0) sums[tid >> 6] = used;
    __syncthreads();
    if (tid == 0) {
      a.starts[0] = 0;
      *a.count_out = (int32_t)(free - max(max(sums[0], sums[1]), max(sums[2], sums[3])));
    }
  }
}

struct TrimArgs {
  const int32_t *lengths, *keep, *table, *free_count;
  int32_t *free_pages, *lengths_out, *count_out;
  int64_t stride;
  int r, pages;
  uint32_t width, page;
};

// The inverse of popping: requests are walked from the last to the first and
// their pages from the last to the first, so that a step taken back leaves the
// stack as it was.  Every workgroup scans all requests, as in the step.
template <int EACH>
__global__ void __launch_bounds__(256) paged_trim_kernel(const TrimArgs a) {
  constexpr int TILE = 256 * EACH;  // requests of a scan, EACH consecutive ones a thread
  __shared__ uint32_t s_take[TILE], s_last[TILE], sums[4];
  const int tid = threadIdx.x;
  const uint32_t most = a.width * a.page;
  const uint32_t free = (uint32_t)min(max(*a.free_count, 0), a.pages);
  uint32_t taken = 0;
  for (int base = 0, tile = 0; base < a.r; base += TILE, ++tile) {
    uint32_t back[EACH], last[EACH], keep[EACH], sum_back = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int r = a.r - 1 - (base + EACH * tid + i);
      const uint32_t held = r >= 0 ? min((uint32_t)max(a.lengths[r], 0), most) : 0u;
      keep[i] = r >= 0 ? min((uint32_t)max(a.keep[r], 0), held) : 0u;
      last[i] = (held + a.page - 1) / a.page;
      back[i] = last[i] - (keep[i] + a.page - 1) / a.page;
      sum_back += back[i];
    }
    uint32_t total;
    uint32_t sum = taken + block_excl_scan(sum_back, sums, total);
    const bool mine = blockIdx.x == (uint32_t)tile % gridDim.x;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      sum += back[i];
      s_take[EACH * tid + i] = sum;
      s_last[EACH * tid + i] = last[i];
      const int r = a.r - 1 - (base + EACH * tid + i);
      if (mine && r >= 0) a.lengths_out[r] = (int32_t)keep[i];
    }
    __syncthreads();
    // four pages a thread and turn
    for (uint32_t k0 = taken + blockIdx.x * 1024 + tid; k0 < taken + total; k0 += gridDim.x * 1024) {
      const uint32_t k[4] = {k0, k0 + 256, k0 + 512, k0 + 768};
      int i[4];
      first_above<TILE, 4>(s_take, k, i);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k[j] < taken + total && free + k[j] < (uint32_t)a.pages)
          a.free_pages[free + k[j]] =
              a.table[(int64_t)(a.r - 1 - (base + i[j])) * a.stride + s_last[i[j]] - 1 - (k[j] - (i[j] ? s_take[i[j] - 1] : taken))];
    }
    __syncthreads();
    taken += total;
  }
  if (blockIdx.x == 0 && tid == 0) *a.count_out = (int32_t)min(free + taken, (uint32_t)a.pages);
}

struct WriteArgs {
  const uint16_t *k, *v;
  uint8_t *codes, *scales;
  const int32_t *table, *starts, *seq;
  int64_t k_tok, k_head, v_tok, v_head, stride;
  int r, tokens, width, pages, nb, heads;
};

// The least e >= -126 with amax <= 448 2^e, by amax's bits (finite, >= 0): 448 is 1.75 2^8
__device__ __forceinline__ int scale_exp(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return max(e, -126);
}
__device__ __forceinline__ float pow2f(int e) {  // -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// The largest code that is finite times 2^e: 448, and 240 for e = 120 (1.875 2^127; 256 would be 2^128)
__device__ __forceinline__ float largest_code(int e) { return fminf(1.875f * pow2f(127 - max(e, 1)), 448.f); }
// four values as e4m3 bytes, nearest even.  ODD: what is larger goes to +-top, infinities
// too, and NaN stays NaN; without it |x| is at most 448, and top too.
template <bool ODD>
__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d, float top) {
  if constexpr (ODD) {
    auto fit = [=](float x) { return x == x ? fminf(fmaxf(x, -top), top) : x; };
    a = fit(a);
    b = fit(b);
    c = fit(c);
    d = fit(d);
  }
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
}
// four codes times 2^(-down), down >= 0, each rounded to the nearest even
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float f) {
  const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  int o = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * f, lo[1] * f, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * f, hi[1] * f, o, true);
}

// One workgroup of 256 threads a touched block of 64 tokens and head; bound by
// memory (2 bytes read and 1 written a value).  The new keys and values of the
// block are read once and stay in registers while the block's largest is found;
// keys go out 16 bytes a lane, values through LDS into their transposed order.
// In a block that held tokens before, the scale only grows; where it does, the
// old codes are moved to it (one more rounding, to e4m3, only where the
// difference of the exponents drives a code into the subnormals).
template <int D>
__global__ void __launch_bounds__(256) paged_kv_write_kernel(const WriteArgs a) {
  constexpr int G = D / 64;     // 16-value granules a thread, keys and values each
  constexpr int PITCH = D + 4;  // bytes a token of the staged values
  __shared__ __attribute__((aligned(16))) uint8_t stage[kBlock * PITCH];
  __shared__ uint32_t sums[4], peak[2][4];
  __shared__ int where[5];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, c = lane & 15, h = blockIdx.y;
  // which request, and which of its blocks
  uint32_t seen = 0;
  if (tid == 0) where[0] = -1;
  for (int base = 0; base < a.r; base += 256) {
    const int r = base + tid;
    uint32_t n = 0;
    int s0 = 0, s1 = 0, seq = 0;
    if (r < a.r) {
      s0 = min(max(a.starts[r], 0), a.tokens);
      s1 = min(max(a.starts[r + 1], s0), a.tokens);
      seq = a.seq[r];
      if (s1 > s0 && seq >= s1 - s0) n = (uint32_t)((seq - 1) / kBlock - (seq - (s1 - s0)) / kBlock + 1);
    }
    uint32_t total;
    const uint32_t at = seen + block_excl_scan(n, sums, total);
    if (blockIdx.x >= at && blockIdx.x - at < n) {
      where[0] = r;
      where[1] = (seq - (s1 - s0)) / kBlock + (int)(blockIdx.x - at);
      where[2] = s0;
      where[3] = s1 - s0;
      where[4] = seq - (s1 - s0);
    }
    seen += total;
    if (seen > blockIdx.x) break;
  }
  __syncthreads();
  const int r = where[0], block = where[1], s0 = where[2], n = where[3], held = where[4];
  if (r < 0 || block / a.nb >= a.width) return;
  const int page = a.table[(int64_t)r * a.stride + block / a.nb];
  const int lo = max(held - kBlock * block, 0), hi = min(held + n - kBlock * block, kBlock);  // the new tokens
  const int row0 = s0 + kBlock * block - held;                                                // token row of token 0
  // the new values are under way while the page is looked up
  u32x4_t x[2][G][2];
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const uint16_t* src = part ? a.v + (int64_t)h * a.v_head : a.k + (int64_t)h * a.k_head;
    const int64_t st = part ? a.v_tok : a.k_tok;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int chunk = wave + 4 * i, tok = 16 * (chunk / G) + c, dim = 64 * (chunk % G) + 16 * q;
      x[part][i][0] = x[part][i][1] = u32x4_t{0u, 0u, 0u, 0u};
      if (tok >= lo && tok < hi) {
        const u32x4_t* p = reinterpret_cast<const u32x4_t*>(src + (int64_t)(row0 + tok) * st + dim);
        x[part][i][0] = p[0];
        x[part][i][1] = p[1];
      }
    }
  }
  if (page < 0 || page >= a.pages) return;
  const int64_t unit = ((int64_t)page * a.nb + block % a.nb) * a.heads + h;
  uint8_t* kc = a.codes + unit * (2 * kBlock * D);
  uint8_t* vc = kc + kBlock * D;
  uint8_t* sc = a.scales + unit * 2;
  const bool had = lo > 0;
  const int was[2] = {had ? (int)sc[0] - 127 : -126, had ? (int)sc[1] - 127 : -126};
  u32x4_t held_v[G];  // the values that the block held, for the granules that take new ones or move
  if (had)
#pragma unroll
    for (int i = 0; i < G; ++i) held_v[i] = *reinterpret_cast<const u32x4_t*>(vc + ((wave + 4 * i) * 64 + lane) * 16);
  // the largest magnitude, by its bits; infinities and NaN, where there are some, do not count
  uint32_t big[2] = {0u, 0u};
  bool odd = false;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t w = x[part][i][j >> 2][j & 3];
        big[part] = max(max(big[part], (w << 16) & 0x7FFF0000u), w & 0x7FFF0000u);
      }
    big[part] = wave_max_u32(big[part]);
    if (big[part] >= 0x7F800000u) {
      odd = true;
      big[part] = 0u;
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t w = x[part][i][j >> 2][j & 3], a0 = (w << 16) & 0x7FFF0000u, a1 = w & 0x7FFF0000u;
          big[part] = max(big[part], max(a0 < 0x7F800000u ? a0 : 0u, a1 < 0x7F800000u ? a1 : 0u));
        }
      big[part] = wave_max_u32(big[part]);
    }
    if (lane == 0) peak[part][wave] = big[part];
  }
  __syncthreads();
  int e[2];
#pragma unroll
  for (int part = 0; part < 2; ++part)
    e[part] = max(scale_exp(max(max(peak[part][0], peak[part][1]), max(peak[part][2], peak[part][3]))), was[part]);
  uint32_t code[2][G][4];
  auto encode = [&](auto odd_) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      // 2^-e by halves: e = 128 (a NaN scale that was written by someone else) has no normal inverse
      const float i0 = pow2f(-(e[part] / 2)), i1 = pow2f(-(e[part] - e[part] / 2)), top = largest_code(e[part]);
#pragma unroll
      for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w0 = x[part][i][j >> 1][2 * (j & 1)], w1 = x[part][i][j >> 1][2 * (j & 1) + 1];
          code[part][i][j] = to_e4m3<decltype(odd_)::value>(
              __uint_as_float(w0 << 16) * i0 * i1, __uint_as_float(w0 & 0xFFFF0000u) * i0 * i1,
              __uint_as_float(w1 << 16) * i0 * i1, __uint_as_float(w1 & 0xFFFF0000u) * i0 * i1, top);
        }
    }
  };
  if (odd || max(e[0], e[1]) >= 120)
    encode(std::true_type{});
  else
    encode(std::false_type{});
  const bool grow[2] = {had && e[0] > was[0], had && e[1] > was[1]};
  const float down[2] = {grow[0] ? pow2f(max(was[0] - e[0], -126)) : 1.f, grow[1] ? pow2f(max(was[1] - e[1], -126)) : 1.f};
  // keys: a granule is 16 dims of one token
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int chunk = wave + 4 * i, tok = 16 * (chunk / G) + c;
    u32x4_t* dst = reinterpret_cast<u32x4_t*>(kc + (chunk * 64 + lane) * 16);
    if ((tok >= lo && tok < hi) || (!had && tok >= hi)) {
      *dst = u32x4_t{code[0][i][0], code[0][i][1], code[0][i][2], code[0][i][3]};
    } else if (tok < lo && grow[0]) {
      const u32x4_t o = *dst;
      *dst = u32x4_t{rescale4(o[0], down[0]), rescale4(o[1], down[0]), rescale4(o[2], down[0]), rescale4(o[3], down[0])};
    }
  }
  // values: a granule is 16 tokens of one dim
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int chunk = wave + 4 * i;
    uint32_t* dst = reinterpret_cast<uint32_t*>(stage + (16 * (chunk / G) + c) * PITCH + 64 * (chunk % G) + 16 * q);
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[j] = code[1][i][j];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const int dt = wave + 4 * i;
    u32x4_t* dst = reinterpret_cast<u32x4_t*>(vc + (dt * 64 + lane) * 16);
    uint32_t fresh[4], take[4];  // new codes, and the bytes that they replace
    bool any = false;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      fresh[w] = take[w] = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = 16 * w + 4 * q + j;
        fresh[w] |= (uint32_t)stage[tok * PITCH + 16 * dt + c] << (8 * j);
        take[w] |= (tok >= lo && (tok < hi || !had)) ? 0xFFu << (8 * j) : 0u;
      }
      any |= take[w] != 0u;
    }
    if (!had) {
      *dst = u32x4_t{fresh[0], fresh[1], fresh[2], fresh[3]};
    } else if (any || grow[1]) {
      u32x4_t o = held_v[i];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t old = 0u;  // bytes of tokens held before
#pragma unroll
        for (int j = 0; j < 4; ++j) old |= 16 * w + 4 * q + j < lo ? 0xFFu << (8 * j) : 0u;
        const uint32_t moved = grow[1] ? rescale4(o[w], down[1]) : o[w];
        o[w] = (fresh[w] & take[w]) | (moved & old) | (o[w] & ~(take[w] | old));
      }
      *dst = o;
    }
  }
  if (tid < 2) sc[tid] = (uint8_t)(e[tid] + 127);
}

bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const char *x = (const char*)a, *y = (const char*)b;
  return x && y && na && nb && x < y + nb && y < x + na;
}
// the rows of a table, not what lies between them
bool overlap(const int32_t* table, int64_t rows, int64_t width, int64_t stride, const int32_t* b, int64_t n) {
  const int64_t at = ((intptr_t)b - (intptr_t)table) / 4;  // the last row that begins in front of b, or the first
  const int64_t row = at <= 0 || rows == 0 ? 0 : at / stride < rows ? at / stride : rows - 1;
  return table && rows && (overlap(table + row * stride, 4 * width, b, 4 * n) ||
                           (row + 1 < rows && overlap(table + (row + 1) * stride, 4 * width, b, 4 * n)));
}

}  // namespace
}  // namespace mosaic

using namespace mosaic;

extern "C" int mosaic_paged_step(const int32_t* lengths, const int32_t* add, int32_t* block_table, int64_t table_stride,
                                 const int32_t* free_pages, const int32_t* free_count, int64_t requests, int64_t width,
                                 int64_t pages, int64_t tokens, int64_t page_size, int32_t* starts,
                                 int32_t* lengths_out, int32_t* seq_lens, int32_t* positions, int32_t* slots,
                                 int32_t* count_out, void* stream) {
  MOSAIC_CHECK_ARG(requests >= 0 && requests <= (1 << 20) && tokens >= 0 && tokens < (1 << 21),
                   "paged_step: %lld requests (up to 2^20), %lld token rows (below 2^21)", (long long)requests,
                   (long long)tokens);
  MOSAIC_CHECK_ARG(page_size >= kBlock && page_size % kBlock == 0 && page_size <= 4096,
                   "paged_step: page size %lld (a multiple of 64, at most 4096)", (long long)page_size);
  MOSAIC_CHECK_ARG(width >= 1 && width * page_size < (1ll << 30) && table_stride >= width,
                   "paged_step: tables of %lld pages (rows hold fewer than 2^30 tokens)", (long long)width);
  MOSAIC_CHECK_ARG(starts && count_out && (requests == 0 || (lengths && add && block_table && lengths_out && seq_lens)) &&
                       (tokens == 0 || (positions && slots)),
                   "paged_step: null pointer");
  MOSAIC_CHECK_ARG((free_pages != nullptr) == (free_count != nullptr), "paged_step: free_pages goes with free_count");
  MOSAIC_CHECK_ARG(!free_pages || (pages >= 0 && pages * page_size < (1ll << 31)),
                   "paged_step: %lld pages (slots are below 2^31)", (long long)pages);
  const int32_t* in[4] = {lengths, add, free_pages, free_count};
  const int64_t in_n[4] = {requests, requests, pages, 1};
  int32_t* out[6] = {starts, lengths_out, seq_lens, positions, slots, count_out};
  const int64_t out_n[6] = {requests + 1, requests, requests, tokens, tokens, 1};
  for (int i = 0; i < 4; ++i)
    for (int o = 0; o < 6; ++o)
      MOSAIC_CHECK_ARG(!overlap(in[i], 4 * in_n[i], out[o], 4 * out_n[o]), "paged_step: an output overlaps an input");
  for (int o = 0; o < 6; ++o) {
    for (int i = 0; i < o; ++i)
      MOSAIC_CHECK_ARG(!overlap(out[i], 4 * out_n[i], out[o], 4 * out_n[o]), "paged_step: an output overlaps another");
    MOSAIC_CHECK_ARG(!overlap(block_table, requests, width, table_stride, out[o], out_n[o]),
                     "paged_step: an output overlaps the tables");
  }
  for (int i = 0; free_pages && i < 4; ++i)
    MOSAIC_CHECK_ARG(!overlap(block_table, requests, width, table_stride, in[i], in_n[i]),
                     "paged_step: the tables overlap an input");
  StepArgs a{lengths, add, free_pages, free_count, block_table, starts, lengths_out, seq_lens, positions, slots,
             count_out, table_stride, (int)requests, (int)(free_pages ? pages : 0),
             (uint32_t)((1ll << 31) / page_size), (uint32_t)width, (uint32_t)page_size, (uint32_t)tokens};
  const unsigned grid = (unsigned)(tokens > kRows ? (tokens + kRows - 1) / kRows : 1);
  // one request a thread is read at once (16 requests: 4.4 us, with eight 6.5), eight
  // need one scan for 2048 of them (in two of 1024: 11.4 us, so 9.3)
  if (requests <= 256)
    MOSAIC_LAUNCH(paged_step_kernel<1>, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
  else
    MOSAIC_LAUNCH(paged_step_kernel<8>, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
  MOSAIC_RETURN_LAUNCH("paged_step");
}

extern "C" int mosaic_paged_trim(const int32_t* lengths, const int32_t* keep, const int32_t* block_table,
                                 int64_t table_stride, int32_t* free_pages, const int32_t* free_count,
                                 int64_t requests, int64_t width, int64_t pages, int64_t page_size,
                                 int32_t* lengths_out, int32_t* count_out, void* stream) {
  MOSAIC_CHECK_ARG(requests >= 0 && requests <= (1 << 20), "paged_trim: %lld requests (up to 2^20)",
                   (long long)requests);
  MOSAIC_CHECK_ARG(page_size >= kBlock && page_size % kBlock == 0 && page_size <= 4096,
                   "paged_trim: page size %lld (a multiple of 64, at most 4096)", (long long)page_size);
  MOSAIC_CHECK_ARG(width >= 1 && width * page_size < (1ll << 30) && table_stride >= width,
                   "paged_trim: tables of %lld pages (rows hold fewer than 2^30 tokens)", (long long)width);
  MOSAIC_CHECK_ARG(pages >= 0 && pages * page_size < (1ll << 31), "paged_trim: %lld pages", (long long)pages);
  // what lengths may say to hold in all is counted in 32 bits, and columns are found by that count
  MOSAIC_CHECK_ARG(requests * width < (1ll << 31), "paged_trim: tables of %lld entries (below 2^31)",
                   (long long)(requests * width));
  MOSAIC_CHECK_ARG(free_count && count_out && (pages == 0 || free_pages) &&
                       (requests == 0 || (lengths && keep && block_table && lengths_out)),
                   "paged_trim: null pointer");
  const int32_t* in[3] = {lengths, keep, free_count};
  const int64_t in_n[3] = {requests, requests, 1};
  int32_t* out[3] = {lengths_out, count_out, free_pages};
  const int64_t out_n[3] = {requests, 1, pages};
  for (int i = 0; i < 3; ++i)
    for (int o = 0; o < 3; ++o)
      MOSAIC_CHECK_ARG(!overlap(in[i], 4 * in_n[i], out[o], 4 * out_n[o]), "paged_trim: an output overlaps an input");
  for (int o = 0; o < 3; ++o) {
    for (int i = 0; i < o; ++i)
      MOSAIC_CHECK_ARG(!overlap(out[i], 4 * out_n[i], out[o], 4 * out_n[o]), "paged_trim: an output overlaps another");
    MOSAIC_CHECK_ARG(!overlap(block_table, requests, width, table_stride, out[o], out_n[o]),
                     "paged_trim: an output overlaps the tables");
  }
  TrimArgs a{lengths, keep, block_table, free_count, free_pages, lengths_out, count_out, table_stride,
             (int)requests, (int)pages, (uint32_t)width, (uint32_t)page_size};
  const int64_t most = (pages < requests * width ? pages : requests * width) / 1024;
  const unsigned grid = (unsigned)(most < 1 ? 1 : most > 128 ? 128 : most);
  if (requests <= 256)
    MOSAIC_LAUNCH(paged_trim_kernel<1>, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
  else
    MOSAIC_LAUNCH(paged_trim_kernel<8>, dim3(grid), dim3(256), 0, (hipStream_t)stream, a);
  MOSAIC_RETURN_LAUNCH("paged_trim");
}

extern "C" int mosaic_paged_kv_write(const uint16_t* k, const uint16_t* v, int64_t k_token_stride,
                                     int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                     int64_t tokens, uint8_t* codes, uint8_t* scales, int64_t pages, int64_t blocks,
                                     int64_t kv_heads, int64_t head_dim, const int32_t* block_table,
                                     int64_t table_stride, int64_t width, const int32_t* starts,
                                     const int32_t* seq_lens, int64_t requests, void* stream) {
  MOSAIC_CHECK_ARG(head_dim == 64 || head_dim == 128 || head_dim == 256, "paged_kv_write: head dim %lld (64, 128 or 256)",
                   (long long)head_dim);
  MOSAIC_CHECK_ARG(kv_heads >= 1 && kv_heads <= 65535, "paged_kv_write: %lld heads", (long long)kv_heads);
  MOSAIC_CHECK_ARG(pages >= 0 && pages < (1ll << 31) && blocks >= 1 && blocks <= 64,
                   "paged_kv_write: %lld pages of %lld blocks", (long long)pages, (long long)blocks);
  MOSAIC_CHECK_ARG(tokens >= 0 && tokens < (1 << 21) && requests >= 0 && requests <= (1 << 20),
                   "paged_kv_write: %lld tokens of %lld requests", (long long)tokens, (long long)requests);
  MOSAIC_CHECK_ARG(width >= 1 && width * blocks * kBlock < (1ll << 30) && table_stride >= width,
                   "paged_kv_write: tables of %lld pages", (long long)width);
  if (tokens == 0 || requests == 0 || pages == 0) return kOk;
  MOSAIC_CHECK_ARG(k && v && codes && scales && block_table && starts && seq_lens, "paged_kv_write: null pointer");
  MOSAIC_CHECK_ARG(((uintptr_t)k | (uintptr_t)v | (uintptr_t)codes) % 16 == 0 && k_token_stride % 8 == 0 &&
                       k_head_stride % 8 == 0 && v_token_stride % 8 == 0 && v_head_stride % 8 == 0,
                   "paged_kv_write: k, v and codes are read and written 16 bytes at a time");
  WriteArgs a{k, v, codes, scales, block_table, starts, seq_lens, k_token_stride, k_head_stride, v_token_stride,
              v_head_stride, table_stride, (int)requests, (int)tokens, (int)width, (int)pages, (int)blocks,
              (int)kv_heads};
  // n consecutive tokens touch at most n blocks, and at most (n - 2) / 64 + 2
  const int64_t most = tokens / kBlock + 2 * requests;
  const dim3 grid((unsigned)(most < tokens ? most : tokens), (unsigned)kv_heads);
  if (head_dim == 64)
    MOSAIC_LAUNCH(paged_kv_write_kernel<64>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else if (head_dim == 128)
    MOSAIC_LAUNCH(paged_kv_write_kernel<128>, grid, dim3(256), 0, (hipStream_t)stream, a);
  else
    MOSAIC_LAUNCH(paged_kv_write_kernel<256>, grid, dim3(256), 0, (hipStream_t)stream, a);
  MOSAIC_RETURN_LAUNCH("paged_kv_write");
}
