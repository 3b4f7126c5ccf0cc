// Bounds of the 4-bit cache's keys by blocks of 32 tokens, and the blocks that
// each query attends to.
//
// With lo_c <= k_c <= hi_c for the keys of a block, the sum of a KV head's query
// heads' products with any of them is at most
//   sum_g sum_c max(q_gc lo_c, q_gc hi_c) = sum_c (P_c hi_c - N_c lo_c),
// P and N the sums over the heads of the positive and of the negated negative
// channels: one product of 2 D channels a block, however many heads there are.
// It is computed in whole numbers (P, N of 7 bits, bounds of 7 bits and a sign in
// units of a power of two), so it has one value whatever the order of its sums,
// and a selection has one right answer.  The sums are below 2^22 and exact as
// floats; times the power of two they rank the blocks.

#include <algorithm>

#include "kv4_attend.h"
#include "launch.h"

namespace sfx {

namespace {

constexpr int kNanUnit = 127;
constexpr int kNoPage = -128;

struct BoundsArgs {
  KvView c;
  int64_t tokens;
  const void* start;
  const void* count;
  int start64, count64;
  int8_t* range;
  int8_t* unit;
};

typedef float F2 __attribute__((ext_vector_type(2)));

// A wave per block of 32 positions, KV head and row: a lane has eight channels of
// every 512 / D-th token.
template <int D>
__global__ __launch_bounds__(kWave) void k_kv4_bounds(BoundsArgs a) {
  using L = KvLayout<D>;
  constexpr int kWords = D / 8;             // of a token's keys
  constexpr int kAtOnce = kWave / kWords;   // tokens
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  int64_t n = a.count ? load_count(a.count, a.count64, b) : a.tokens;
  n = n < a.tokens ? n : a.tokens;
  const int64_t s0 = load_count(a.start, a.start64, b);
  if (n <= 0 || s0 < 0 || s0 >= a.c.positions) return;
  if (n > a.c.positions - s0) n = a.c.positions - s0;
  const int64_t blk = s0 / kKvBlock + blockIdx.x;
  if (blk * kKvBlock >= s0 + n) return;
  const int64_t at = kv_place(a.c, b, h, blk);
  if (at < 0) return;
  const char* base = a.c.pages + at * (int64_t)L::kBytes;
  const int64_t end64 = s0 + n - blk * kKvBlock;
  const int end = end64 < kKvBlock ? (int)end64 : kKvBlock;  // tokens held
  const int word = lane_id() % kWords, sub = lane_id() / kWords;
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo[e] = __builtin_inff();
    hi[e] = kNegInf;
  }
  bool bad = false;
  constexpr int kSteps = kKvBlock / kAtOnce;
  uint32_t w[kSteps];
  uint32_t sb[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int t = i * kAtOnce + sub;
    w[i] = ((const uint32_t*)base)[t * kWords + word];
    sb[i] = ((const uint8_t*)(base + L::kScale))[t * (D / 32) + word / 4];
  }
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    if (i * kAtOnce + sub >= end) continue;
    bad |= sb[i] == 255u;
    const float sc = __uint_as_float(sb[i] << 23);
    F2 x[4];
    x[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sc, 0);
    x[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sc, 1);
    x[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sc, 2);
    x[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], sc, 3);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = fminf(lo[e], x[e / 2][e % 2]);
      hi[e] = fmaxf(hi[e], x[e / 2][e % 2]);
    }
  }
#pragma unroll
  for (int o = kWords; o < kWave; o <<= 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = fminf(lo[e], __shfl_xor(lo[e], o));
      hi[e] = fmaxf(hi[e], __shfl_xor(hi[e], o));
    }
  bad = __any(bad);
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    top = fmaxf(top, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
#pragma unroll
  for (int o = 1; o < kWords; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  int u = (int)(__float_as_uint(top) >> 23) - 127 - 6;
  u = u < -100 ? -100 : (u > 100 ? 100 : u);
  const float inv = __uint_as_float((uint32_t)(127 - u) << 23);
  if (sub == 0) {
    uint32_t l[2] = {0, 0}, g[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int x = (int)fminf(fmaxf(floorf(lo[e] * inv), -127.0f), 127.0f);
      const int y = (int)fminf(fmaxf(ceilf(hi[e] * inv), -127.0f), 127.0f);
      l[e / 4] |= (uint32_t)(bad ? 0 : x & 255) << (8 * (e % 4));
      g[e / 4] |= (uint32_t)(bad ? 0 : y & 255) << (8 * (e % 4));
    }
    int8_t* r = a.range + at * (2 * D) + 8 * word;
    *(uint2*)r = uint2{l[0], l[1]};
    *(uint2*)(r + D) = uint2{g[0], g[1]};
    if (word == 0) a.unit[at] = (int8_t)(bad ? kNanUnit : u);
  }
}

typedef int32_t I4 __attribute__((ext_vector_type(4)));

struct SelectArgs : AttendArgs {
  const int8_t* range;
  const int8_t* unit;
  int want, sinks, recent;  // blocks: in all, first, last
  int span;      // query tokens of a tile
  int tiles;
  int chunks;    // of kScoreChunk blocks
  int64_t pitch; // of a query's keys
  uint32_t* keys;     // [batch, tokens, heads, pitch]
  int32_t* selected;  // [batch, tokens, heads, want]
};

// Positions that query token t of row b sees.
__device__ __forceinline__ int token_sees(const SelectArgs& a, int64_t len,
                                          int64_t nq, int64_t t) {
  if (t >= a.tokens || t >= nq) return 0;
  const int64_t v = len - nq + t + 1;
  return v > a.c.positions ? (int)a.c.positions : (v > 0 ? (int)v : 0);
}

// P and -N of a query token and KV head, in 7 bits, by a wave: [0, D) against the
// least keys, [D, 2 D) against the largest.
template <int D, bool kHalf>
__device__ __forceinline__ void pack_query(const SelectArgs& a, int64_t b,
                                           int h, int64_t t, int8_t* out) {
  constexpr int C = D / kWave;  // channels of a lane
  constexpr int kHold = 8;      // query heads kept; of more all are read twice
  const int lane = lane_id();
  const uint16_t* q = (const uint16_t*)a.q.data + b * a.q.stride_b +
                      t * a.q.stride_t + (int64_t)h * a.group * a.q.stride_h +
                      lane * C;
  struct Head {
    uint16_t x[C];
  };
  auto read = [&](int g) {
    Head r;
    const uint16_t* p = q + (int64_t)g * a.q.stride_h;
    if (C == 1) {
      r.x[0] = p[0];
    } else if (a.vec) {
      typedef uint32_t W __attribute__((ext_vector_type(C > 1 ? C / 2 : 1)));
      const W w = *(const W*)p;
      __builtin_memcpy(r.x, &w, 2 * C);
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) r.x[c] = p[c];
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
      if ((r.x[c] & 0x7fffu) >= (kHalf ? 0x7c00u : 0x7f80u)) r.x[c] = 0;
    return r;
  };
  Head held[kHold] = {};
#pragma unroll
  for (int g = 0; g < kHold; ++g)
    if (g < a.group) held[g] = read(g);
  uint32_t top = 0;
  auto most_of = [&](const Head& x) {
#pragma unroll
    for (int c = 0; c < C; ++c) top = max(top, x.x[c] & 0x7fffu);
  };
#pragma unroll
  for (int g = 0; g < kHold; ++g) most_of(held[g]);
  for (int g = kHold; g < a.group; ++g) most_of(read(g));
  top = wave_all_max(top);
  // 2^e is the power of two above the largest
  const int e = __builtin_amdgcn_frexp_expf(to_float16b<kHalf>(top));
  uint32_t p[C], n[C];
#pragma unroll
  for (int c = 0; c < C; ++c) p[c] = n[c] = 0;
  auto add = [&](const Head& x) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int z = (int)rintf(
          __builtin_amdgcn_ldexpf(to_float16b<kHalf>(x.x[c]), 15 - e));
      p[c] += (uint32_t)max(z, 0);
      n[c] += (uint32_t)max(-z, 0);
    }
  };
#pragma unroll
  for (int g = 0; g < kHold; ++g)
    if (g < a.group) add(held[g]);
  for (int g = kHold; g < a.group; ++g) add(read(g));
  uint32_t most = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) most = max(most, max(p[c], n[c]));
  most = wave_all_max(most);
  const int shift = most ? max(0, 32 - __builtin_clz(most) - 7) : 0;
  const uint32_t half = shift ? 1u << (shift - 1) : 0u;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    out[lane * C + c] = (int8_t)-(int)min((n[c] + half) >> shift, 127u);
    out[D + lane * C + c] = (int8_t)min((p[c] + half) >> shift, 127u);
  }
}

// Order of scores as whole numbers; 0 is no score's.
__device__ __forceinline__ uint32_t score_key(int32_t dot, int unit) {
  if (unit == kNoPage) return 0;
  const float f = unit == kNanUnit
                      ? __builtin_inff()
                      : (float)dot * __uint_as_float((uint32_t)(unit + 127)
                                                     << 23);
  const uint32_t x = __float_as_uint(f);
  return x >> 31 ? ~x : x | 0x80000000u;
}

constexpr int kScoreThreads = 256;
constexpr int kScoreTiles = 2;  // of 16 blocks, per wave
constexpr int kScoreChunk = kScoreThreads / kWave * kScoreTiles * 16;

// Scores of 128 blocks for up to 16 query tokens of a row and KV head.
template <int D, bool kHalf>
__global__ __launch_bounds__(kScoreThreads) void k_kv4_scores(SelectArgs a) {
  constexpr int kStep = 2 * D / 64;  // matrix instructions a tile
  constexpr int kPitch = 2 * D + 16;
  __shared__ __align__(16) int8_t sq[16][kPitch];
  const int id = (int)blockIdx.x;
  // tiles of one piece of the cache follow each other on one XCD
  const int k = id >> 3;
  const int tile = k % a.tiles;
  const int64_t item = (int64_t)(k / a.tiles) * 8 + (id & 7);
  const int64_t rows = a.batch * a.c.heads;
  const int64_t bh = item % rows;
  const int64_t chunk = item / rows;
  if (chunk >= a.chunks) return;
  const int64_t b = bh / a.c.heads;
  const int h = (int)(bh % a.c.heads);
  const int64_t len = kv_len_of(a, b), nq = q_len_of(a, b);
  const int64_t t0 = (int64_t)tile * 16;  // (the span)
  const int64_t last = std::min(std::min(nq, a.tokens), t0 + 16) - 1;
  const int64_t blk0 = chunk * kScoreChunk;
  if (last < t0 || blk0 * kKvBlock >= token_sees(a, len, nq, last)) return;
  const int lane = lane_id(), wave = threadIdx.x / kWave;
  const int i16 = lane % 16, quad = lane / 16;

  // the bounds of the wave's blocks
  I4 r[kScoreTiles][kStep];
  int unit[kScoreTiles];
#pragma unroll
  for (int t = 0; t < kScoreTiles; ++t) {
    const int64_t blk = blk0 + (wave * kScoreTiles + t) * 16 + i16;
    const int64_t at = kv_place(a.c, b, h, blk);
    unit[t] = at < 0 ? kNoPage : a.unit[at];
    const I4* p = (const I4*)(a.range + (at < 0 ? 0 : at) * (2 * D)) + quad;
#pragma unroll
    for (int i = 0; i < kStep; ++i) r[t][i] = at < 0 ? I4{0, 0, 0, 0} : p[4 * i];
  }
  for (int i = wave; i < 16; i += kScoreThreads / kWave) {
    if (t0 + i <= last) {
      pack_query<D, kHalf>(a, b, h, t0 + i, sq[i]);
    } else {
      for (int c = lane; c < 2 * D; c += kWave) sq[i][c] = 0;
    }
  }
  __syncthreads();
  const int64_t t = t0 + i16;
  uint32_t* out = a.keys + ((b * a.tokens + t) * a.c.heads + h) * a.pitch;
#pragma unroll
  for (int w = 0; w < kScoreTiles; ++w) {
    I4 s = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kStep; ++i)
      s = __builtin_amdgcn_mfma_i32_16x16x64_i8(
          r[w][i], *(const I4*)&sq[i16][i * 64 + quad * 16], s, 0, 0, 0);
    uint32_t key[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      key[e] = score_key(s[e], __shfl(unit[w], quad * 4 + e));
    const int64_t blk = blk0 + (wave * kScoreTiles + w) * 16 + quad * 4;
    if (t <= last && blk < a.pitch)
      *(uint4*)(out + blk) = uint4{key[0], key[1], key[2], key[3]};
  }
}

// Whether a query whose last block is `last` takes block j whatever its score.
__device__ __forceinline__ bool always(const SelectArgs& a, int j, int last) {
  return j < a.sinks || j > last - a.recent;
}

// The blocks of a query with the keys key[0 .. last] in LDS, by a wave that keeps
// kRegs of them in each lane: the least key that is taken, bit by bit, below the
// bits that all have and until as many as are wanted lie past it; then the blocks
// past it, and those at it while there is room.
template <int kRegs>
__device__ __forceinline__ void pick_blocks(int sinks, int recent, int all,
                                            int last, const uint32_t* key,
                                            int32_t* out) {
  const int lane = lane_id();
  uint32_t k[kRegs];
  uint32_t sure = 0;  // a bit for each register
  uint32_t hi = 0, lo = 0;
  int want = all;
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int j = i * kWave + lane;
    k[i] = j <= last ? key[j] : 0;
    const bool is = k[i] && (j < sinks || j > last - recent);
    want -= popc(ballot(is));
    if (is) {
      sure |= 1u << i;
      k[i] = 0;
    }
    hi = max(hi, k[i]);
    lo = max(lo, 0u - k[i]);  // (none is the least)
  }
  auto at_least = [&](uint32_t x) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) n += popc(ballot(k[i] >= x));
    return n;
  };
  // line: keys past it are taken, and `room` of those at it
  uint32_t line = 0;
  int room = 0;
  if (want <= 0) {
    line = 0xffffffffu;
  } else if (at_least(1) > want) {
    hi = wave_all_max(hi);
    lo = 0u - wave_all_max(lo);
    int bit = 31 - __builtin_clz((hi ^ lo) | 1u);
    line = hi >> bit >> 1 << bit << 1;
    for (; bit >= 0; --bit) {
      const uint32_t x = line | 1u << bit;
      const int n = at_least(x);
      if (n >= want) line = x;
      if (n == want) break;
    }
    if (bit >= 0)
      --line;  // those past it now are the wanted ones
    else
      room = want - at_least(line + 1);
  }
  int n = 0;
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    bool in = k[i] > line || (sure >> i & 1);
    if (room > 0) {
      const uint64_t eq = ballot(k[i] == line);
      in = in || (k[i] == line && rank_lt(eq) < room);
      room -= popc(eq);
    }
    const uint64_t m = ballot(in);
    if (in) out[n + rank_lt(m)] = i * kWave + lane;
    n += popc(m);
  }
  for (int i = n + lane; i < all; i += kWave) out[i] = -1;
}

// Scores and choice at once, where a workgroup holds the keys of its tokens: rows
// of up to 1,024 blocks.
constexpr int kSelectThreads = 512;
constexpr int kSelectTokens = 32;

template <int D, bool kHalf>
__global__ __launch_bounds__(kSelectThreads) void k_kv4_select(SelectArgs a) {
  constexpr int kStep = 2 * D / 64;  // matrix instructions a tile
  constexpr int kPitch = 2 * D + 16;
  constexpr int kSelectWaves = kSelectThreads / kWave;
  extern __shared__ __align__(16) char lds[];
  const int id = (int)blockIdx.x;
  // tiles of one row and KV head follow each other on one XCD
  const int k = id >> 3;
  const int tile = k % a.tiles;
  const int64_t bh = (int64_t)(k / a.tiles) * 8 + (id & 7);
  if (bh >= a.batch * a.c.heads) return;
  const int64_t b = bh / a.c.heads;
  const int h = (int)(bh % a.c.heads);
  const int64_t len = kv_len_of(a, b), nq = q_len_of(a, b);
  const int64_t t0 = (int64_t)tile * a.span;
  const int tokens = (int)std::min<int64_t>(a.span, a.tokens - t0);
  const int queries = (int)std::max<int64_t>(
      0, std::min<int64_t>(tokens, nq - t0));
  auto sq = (int8_t(*)[kPitch])lds;
  // (rows 4 banks apart)
  const int pitch = (int)a.pitch + 4;
  uint32_t* keys = (uint32_t*)(lds + (a.span + 15) / 16 * 16 * kPitch);
  const int blocks =
      queries ? (token_sees(a, len, nq, t0 + queries - 1) + kKvBlock - 1) /
                    kKvBlock
              : 0;
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int i16 = lane % 16, quad = lane / 16;

  // bounds of 16 blocks; the next ones are on their way while these are used
  I4 r[kStep];
  int unit;
  auto load = [&](int blk0) {
    const int64_t at = blk0 < blocks ? kv_place(a.c, b, h, blk0 + i16) : -1;
    unit = at < 0 ? kNoPage : a.unit[at];
    const I4* p = (const I4*)(a.range + (at < 0 ? 0 : at) * (2 * D)) + quad;
#pragma unroll
    for (int i = 0; i < kStep; ++i) r[i] = at < 0 ? I4{0, 0, 0, 0} : p[4 * i];
  };
  load(wave * 16);
  const int rows = (tokens + 15) / 16 * 16;
  for (int i = wave; i < rows; i += kSelectWaves) {
    if (i < queries) {
      pack_query<D, kHalf>(a, b, h, t0 + i, sq[i]);
    } else {
      for (int c = lane; c < D / 2; c += kWave) ((uint32_t*)sq[i])[c] = 0;
    }
  }
  __syncthreads();
  for (int blk0 = wave * 16; blk0 < blocks; blk0 += kSelectWaves * 16) {
    I4 now[kStep];
#pragma unroll
    for (int i = 0; i < kStep; ++i) now[i] = r[i];
    const int u = unit;
    load(blk0 + kSelectWaves * 16);
    int us[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) us[e] = __shfl(u, quad * 4 + e);
    for (int q0 = 0; q0 < queries; q0 += 16) {
      I4 s = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kStep; ++i)
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(
            now[i], *(const I4*)&sq[q0 + i16][i * 64 + quad * 16], s, 0, 0, 0);
      if (q0 + i16 < queries)
        *(uint4*)(keys + (q0 + i16) * pitch + blk0 + quad * 4) =
            uint4{score_key(s[0], us[0]), score_key(s[1], us[1]),
                  score_key(s[2], us[2]), score_key(s[3], us[3])};
    }
  }
  __syncthreads();
  for (int i = wave; i < tokens; i += kSelectWaves) {
    const int last = __builtin_amdgcn_readfirstlane(
        (token_sees(a, len, nq, t0 + i) + kKvBlock - 1) / kKvBlock - 1);
    const uint32_t* own = keys + i * pitch;
    int32_t* out =
        a.selected + ((b * a.tokens + t0 + i) * a.c.heads + h) * a.want;
    if (last < 4 * kWave)
      pick_blocks<4>(a.sinks, a.recent, a.want, last, own, out);
    else if (last < 8 * kWave)
      pick_blocks<8>(a.sinks, a.recent, a.want, last, own, out);
    else
      pick_blocks<16>(a.sinks, a.recent, a.want, last, own, out);
  }
}

// The key of block j for what follows: first and recent blocks above all others.
__device__ __forceinline__ uint32_t ranked(const SelectArgs& a, uint32_t key,
                                           int j, int last) {
  if (j > last || key == 0) return 0;
  return always(a, j, last) ? 0xffffffffu : key;
}

// The choice by a workgroup, for tables of more blocks than a wave keeps: the keys
// are in memory, and four passes narrow the threshold down by 8 bits each.
constexpr int kWideThreads = 1024;

__global__ __launch_bounds__(kWideThreads) void k_kv4_pick_wide(SelectArgs a) {
  constexpr int kWideWaves = kWideThreads / kWave;
  __shared__ int hist[256];
  __shared__ int sums[kWideWaves];
  __shared__ int found[2];
  const int64_t list = blockIdx.x;
  const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWave;
  const int64_t b = list / (a.tokens * a.c.heads);
  const int64_t t = list / a.c.heads % a.tokens;
  const int sees = token_sees(a, kv_len_of(a, b), q_len_of(a, b), t);
  const int last = (sees + kKvBlock - 1) / kKvBlock - 1;
  const uint32_t* keys = a.keys + list * a.pitch;
  int32_t* out = a.selected + list * a.want;
  uint32_t line = 0, mask = 0;
  int want = a.want;  // of the keys that agree with the line so far
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int j = tid; j <= last; j += kWideThreads) {
      const uint32_t k = ranked(a, keys[j], j, last);
      if (k && (k & mask) == line) atomicAdd(&hist[k >> shift & 255], 1);
    }
    __syncthreads();
    if (wave == 0) {
      // bins from the top: lane l has 255 - 4 l and the three below
      int n[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum += n[e] = hist[255 - 4 * lane - e];
      const int upto = (int)wave_incl_scan((uint32_t)sum);
      const uint64_t m = ballot(upto >= want);
      if (m == 0) {
        if (lane == 0) found[0] = -1;  // fewer than that
      } else if (lane == __builtin_ctzll(m)) {
        int left = want - (upto - sum), e = 0;
        while (n[e] < left) left -= n[e++];
        found[0] = 255 - 4 * lane - e;
        found[1] = left;
      }
    }
    __syncthreads();
    if (found[0] < 0) break;  // (in the first pass only)
    line |= (uint32_t)found[0] << shift;
    mask |= 255u << shift;
    want = found[1];
    __syncthreads();
  }
  // `want` of the keys at the line, in order; without a line all
  int n = 0, room = mask ? want : 0;
  if (!mask) line = 0;
  for (int j0 = 0; j0 <= last; j0 += kWideThreads) {
    const int j = j0 + tid;
    const uint32_t k = j <= last ? ranked(a, keys[j], j, last) : 0;
    const bool eq = mask && k == line;
    // both counts in one scan
    const uint32_t mine = (uint32_t)(k > line) | (uint32_t)eq << 16;
    const uint32_t to = wave_incl_scan(mine);
    __syncthreads();
    if (lane == kWave - 1) sums[wave] = (int)to;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < kWideWaves; ++w) {
      if (w < wave) before += (uint32_t)sums[w];
      all += (uint32_t)sums[w];
    }
    const uint32_t ex = before + to - mine;
    const int gt = (int)(ex & 0xffffu), eqs = (int)(ex >> 16);
    if (k > line || (eq && eqs < room))
      out[n + gt + min(eqs, room)] = j;
    const int all_eq = min((int)(all >> 16), room);
    n += (int)(all & 0xffffu) + all_eq;
    room -= all_eq;
  }
  for (int i = n + tid; i < a.want; i += kWideThreads) out[i] = -1;
}

struct LaunchBounds {
  BoundsArgs a;
  dim3 grid;
  hipStream_t stream;
  template <int D>
  int run() {
    hipLaunchKernelGGL(k_kv4_bounds<D>, grid, dim3(kWave), 0, stream, a);
    return (int)hipGetLastError();
  }
};

int64_t pitch_of(const sfx_kv4* c) {
  const int64_t blocks = c->table_width * c->page_size / kKvBlock;
  return (blocks + 15) / 16 * 16;
}

bool select_ok(const sfx_kv4* c, int64_t batch, int64_t tokens) {
  KvView v;
  // the keys' number in 62 bits, lists in a grid's
  return kv_view(c, &v) && batch >= 0 && batch <= 65535 && tokens >= 0 &&
         tokens <= (int64_t(1) << 24) &&
         batch * tokens <= ((int64_t(1) << 22) - 1) / c->heads;
}

bool held_in_lds(const sfx_kv4* c) {
  return pitch_of(c) <= 16 * kWave;
}

template <int D, bool kHalf>
int launch_held(SelectArgs a, hipStream_t stream) {
  // As many tokens as a workgroup's 64 KB hold keys of; past kSelectTokens in
  // tiles of 16.
  const int64_t row = 4 * (a.pitch + 4), packed = 2 * D + 16;
  const int64_t room = 65536 - kSelectTokens * packed;
  a.span = (int)std::min<int64_t>(a.tokens <= kSelectTokens ? a.tokens : 16,
                                  room / row);
  a.tiles = (int)((a.tokens + a.span - 1) / a.span);
  const size_t lds = (a.span + 15) / 16 * 16 * packed + a.span * row;
  const int64_t items = (a.batch * a.c.heads + 7) / 8 * 8;
  if (items * a.tiles >= (int64_t(1) << 32) / kSelectThreads)
    return SFX_EINVAL;
  hipLaunchKernelGGL((k_kv4_select<D, kHalf>),
                     dim3((unsigned)(items * a.tiles)), dim3(kSelectThreads),
                     lds, stream, a);
  return (int)hipGetLastError();
}

template <int D, bool kHalf>
int launch_wide(SelectArgs a, hipStream_t stream) {
  a.span = 16;
  a.tiles = (int)((a.tokens + 15) / 16);
  const int64_t lists = a.batch * a.tokens * a.c.heads;
  const int64_t items = (a.batch * a.c.heads * a.chunks + 7) / 8 * 8;
  if (items * a.tiles >= (int64_t(1) << 32) / kScoreThreads) return SFX_EINVAL;
  hipLaunchKernelGGL((k_kv4_scores<D, kHalf>),
                     dim3((unsigned)(items * a.tiles)), dim3(kScoreThreads), 0,
                     stream, a);
  hipLaunchKernelGGL(k_kv4_pick_wide, dim3((unsigned)lists),
                     dim3(kWideThreads), 0, stream, a);
  return (int)hipGetLastError();
}

template <int D, bool kHalf>
int launch(const SelectArgs& a, const sfx_kv4* cache, hipStream_t stream) {
  return held_in_lds(cache) ? launch_held<D, kHalf>(a, stream)
                            : launch_wide<D, kHalf>(a, stream);
}

constexpr int64_t kMaxTokens = int64_t(1) << 28;  // the grid's limit

bool bounds_ok(const sfx_kv4* c, const sfx_kv4_bounds* b) {
  return b && (c->num_pages == 0 ||
               (b->range && !((uintptr_t)b->range & 15) && b->unit));
}

}  // namespace

}  // namespace sfx

using namespace sfx;

extern "C" int sfx_kv4_bounds_update(const sfx_kv4* cache,
                                     const sfx_kv4_bounds* bounds,
                                     int64_t batch, int64_t tokens,
                                     const void* start, int32_t start_is64,
                                     const void* count, int32_t count_is64,
                                     hipStream_t stream) {
  LaunchBounds l;
  if (!kv_view(cache, &l.a.c) || !bounds_ok(cache, bounds) || batch < 0 ||
      batch > 65535 || tokens < 0 || tokens > kMaxTokens)
    return SFX_EINVAL;
  if (batch == 0 || tokens == 0) return 0;
  if (!start) return SFX_EINVAL;
  l.a.tokens = tokens;
  l.a.start = start;
  l.a.start64 = start_is64;
  l.a.count = count;
  l.a.count64 = count_is64;
  l.a.range = bounds->range;
  l.a.unit = bounds->unit;
  // a stretch of `tokens` positions touches at most this many blocks, and no
  // more than a row has
  const int64_t blocks = std::min<int64_t>(
      (tokens + kKvBlock - 2) / kKvBlock + 1,
      cache->table_width * cache->page_size / kKvBlock);
  if (blocks == 0) return 0;
  l.grid = dim3((unsigned)blocks, (unsigned)cache->heads, (unsigned)batch);
  l.stream = stream;
  switch (cache->head_dim) {
    case 64: return l.run<64>();
    case 128: return l.run<128>();
    default: return l.run<256>();
  }
}

extern "C" size_t sfx_kv4_select_workspace_size(const sfx_kv4* cache,
                                                int64_t batch,
                                                int64_t tokens) {
  if (!select_ok(cache, batch, tokens) || held_in_lds(cache)) return 0;
  return (size_t)(batch * tokens * cache->heads) * (size_t)pitch_of(cache) * 4;
}

extern "C" int sfx_kv4_select(const sfx_kv4* cache,
                              const sfx_kv4_bounds* bounds, const sfx_heads* q,
                              int64_t batch, int64_t tokens, int64_t q_heads,
                              const void* kv_len, int32_t kv_len_is64,
                              const void* q_len, int32_t q_len_is64,
                              int64_t blocks, int64_t first, int64_t recent,
                              int32_t* selected, void* workspace,
                              size_t workspace_bytes, hipStream_t stream) {
  if (!select_ok(cache, batch, tokens) || !bounds_ok(cache, bounds) || !q ||
      q_heads <= 0 || q_heads % cache->heads || q_heads > 65535 || first < 0 ||
      recent < 1 || blocks > 32768 || first > blocks - recent)
    return SFX_EINVAL;
  if (batch == 0 || tokens == 0) return 0;
  if (!q->data || !kv_len || !selected) return SFX_EINVAL;
  const size_t need = sfx_kv4_select_workspace_size(cache, batch, tokens);
  if (workspace_bytes < need ||
      (need && (!workspace || ((uintptr_t)workspace & 15))))
    return SFX_EINVAL;
  SelectArgs a;
  kv_view(cache, &a.c);
  a.q = *q;
  a.tokens = tokens;
  a.q_heads = (int)q_heads;
  a.group = (int)(q_heads / cache->heads);
  a.batch = batch;
  a.kv_len = kv_len;
  a.kv64 = kv_len_is64;
  a.q_len = q_len;
  a.q64 = q_len_is64;
  a.vec = (((uintptr_t)q->data & 15) |
           ((q->stride_b | q->stride_t | q->stride_h) & 7)) == 0;
  a.range = bounds->range;
  a.unit = bounds->unit;
  a.want = (int)blocks;
  a.sinks = (int)first;
  a.recent = (int)recent;
  a.pitch = pitch_of(cache);
  a.chunks = (int)((a.pitch + kScoreChunk - 1) / kScoreChunk);
  a.keys = (uint32_t*)workspace;
  a.selected = selected;
  const bool half = cache->dtype == SFX_F16;
  switch (cache->head_dim) {
    case 64:
      return half ? launch<64, true>(a, cache, stream) : launch<64, false>(a, cache, stream);
    case 128:
      return half ? launch<128, true>(a, cache, stream)
                  : launch<128, false>(a, cache, stream);
    default:
      return half ? launch<256, true>(a, cache, stream)
                  : launch<256, false>(a, cache, stream);
  }
}
