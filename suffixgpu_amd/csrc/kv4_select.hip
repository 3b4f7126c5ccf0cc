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
// and a selection has one right answer.  The sums are below 2^23 and exact as
// floats; times the power of two they rank the blocks.
//
// What bounds it are the steps that follow each other in a workgroup, most of which
// run at once: packing the query, the scores, the choice (vector instructions issue in
// half of the cycles); of many long rows, the memory (64 x 1 tokens over 32,768 each
// 30.6 us, 135 MB, 4.4 TB/s; over 16,384 to 32,768 26 us, 110 MB).  The choice is made
// where the scores are: in LDS and a wave's or a workgroup's registers for rows of up to
// 1,024 blocks (the 26 us, with the scores in memory and a second launch 33; 64 x 17 over
// up to 8,192 16 and 85; a prompt's 2,048 over 16,384 38 and 192), in the registers of a
// workgroup of a second launch past that (one token over 131,072 11 us, 4 x 9 with heads
// of 256 24), and in memory past 16,384 blocks (one token over 1,048,576 87 us, eight of
// them 189, 539 MB).

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
// every 512 / D-th token.  A step's new tokens: 4 to 5 us, a launch's latency; a
// prompt's 14,336 tokens 9 MB (every block's keys once).
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
  int piece;     // blocks of a workgroup of k_kv4_scores
  int pieces;
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
// least keys, [D, 2 D) against the largest.  Made in two steps, so that one
// query's heads can be on their way while another's are packed.
template <int D, bool kHalf>
struct PackQuery {
  static constexpr int C = D / kWave;  // channels of a lane
  static constexpr int kHold = 8;  // query heads kept; of more all are read twice
  struct Head {
    uint16_t x[C];
  };
  const uint16_t* q;
  Head held[kHold];

  __device__ __forceinline__ Head read(const SelectArgs& a, int g) const {
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
    return r;
  }
  __device__ __forceinline__ PackQuery() {}
  __device__ __forceinline__ PackQuery(const SelectArgs& a, int64_t b, int h,
                                       int64_t t) {
    q = (const uint16_t*)a.q.data + b * a.q.stride_b + t * a.q.stride_t +
        (int64_t)h * a.group * a.q.stride_h + lane_id() * C;
#pragma unroll
    for (int g = 0; g < kHold; ++g)
      if (g < a.group) held[g] = read(a, g);
  }
  __device__ __forceinline__ void put(const SelectArgs& a, int8_t* out) const {
    const int lane = lane_id();
    constexpr uint32_t kInf = kHalf ? 0x7c00u : 0x7f80u;
    uint32_t top = 0;
    auto most_of = [&](const Head& x) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint32_t m = x.x[c] & 0x7fffu;
        top = max(top, m < kInf ? m : 0u);
      }
    };
#pragma unroll
    for (int g = 0; g < kHold; ++g)
      if (g < a.group) most_of(held[g]);
    for (int g = kHold; g < a.group; ++g) most_of(read(a, g));
    top = wave_all_max(top);
    // 2^e is the power of two above the largest
    const int e = __builtin_amdgcn_frexp_expf(to_float16b<kHalf>(top));
    uint32_t p[C], n[C];
#pragma unroll
    for (int c = 0; c < C; ++c) p[c] = n[c] = 0;
    auto add = [&](const Head& x) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const uint32_t u = (x.x[c] & 0x7fffu) < kInf ? x.x[c] : 0u;
        const int z =
            (int)rintf(__builtin_amdgcn_ldexpf(to_float16b<kHalf>(u), 15 - e));
        p[c] += (uint32_t)max(z, 0);
        n[c] += (uint32_t)max(-z, 0);
      }
    };
#pragma unroll
    for (int g = 0; g < kHold; ++g)
      if (g < a.group) add(held[g]);
    for (int g = kHold; g < a.group; ++g) add(read(a, g));
    uint32_t most = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) most = max(most, max(p[c], n[c]));
    most = wave_all_max(most);
    const int shift = most ? max(0, 32 - __builtin_clz(most) - 7) : 0;
    const uint32_t half = shift ? 1u << (shift - 1) : 0u;
    uint32_t lo = 0, hi = 0;  // bytes, of up to four channels
#pragma unroll
    for (int c = 0; c < C; ++c) {
      lo |= (-min((n[c] + half) >> shift, 127u) & 255u) << (8 * c);
      hi |= min((p[c] + half) >> shift, 127u) << (8 * c);
    }
    if (C == 1) {
      out[lane] = (int8_t)lo;
      out[D + lane] = (int8_t)hi;
    } else if (C == 2) {
      ((uint16_t*)out)[lane] = (uint16_t)lo;
      ((uint16_t*)(out + D))[lane] = (uint16_t)hi;
    } else {
      ((uint32_t*)out)[lane] = lo;
      ((uint32_t*)(out + D))[lane] = hi;
    }
  }
};

// Order of scores as whole numbers; 0 is no score's.  A sum of 2 D products of up to
// 127^2 has 23 bits, so the last of a float's 24 is nothing but zero: without it all
// of these are below 2^31, and no line that the choice tries passes 2^32 (a NaN's key is
// 2^23 below that otherwise, less than the parts of the range that it looks through).
template <int D>
__device__ __forceinline__ uint32_t score_key(int32_t dot, int unit) {
  static_assert(2 * D * 127 * 127 < 1 << 23, "");
  if (unit == kNoPage) return 0;
  const float f = unit == kNanUnit
                      ? __builtin_inff()
                      : (float)dot * __uint_as_float((uint32_t)(unit + 127)
                                                     << 23);
  const uint32_t x = __float_as_uint(f);
  return (x >> 31 ? ~x : x | 0x80000000u) >> 1;
}

// Scores of blocks [blk0, end) of row b and KV head h for its query tokens t0 ..
// t0 + queries - 1 (packed into sq here, with zeros up to `rows`, a multiple of
// 16), by a workgroup: put(query, block, keys) of four blocks each.  A wave takes
// 16 blocks at a time, at most 8 times; the next ones are on their way while these
// are used.  (Two and three ahead give nothing: 64 x 1 tokens 29 us, a prompt 42 and 44
// instead of 38, as the registers leave fewer waves.  Places read one ahead, instead
// of all at first, wait for the bounds before them: one token over 32,768 18.0 us, now
// 16.1.)
constexpr int kSelectThreads = 512;

template <int D, bool kHalf, class Put>
__device__ __forceinline__ void score_blocks(
    const SelectArgs& a, int64_t b, int h, int64_t t0, int queries, int rows,
    int blk0, int end, int8_t (*sq)[2 * D + 16], Put put) {
  constexpr int kStep = 2 * D / 64;  // matrix instructions of 16 blocks
  constexpr int kSelectWaves = kSelectThreads / kWave;
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int i16 = lane % 16, quad = lane / 16;
  // Places and units of all the wave's blocks, 16 i + j of them in lane 16 (i % 4) +
  // j: their loads wait for each other once.  (In 32 bits: a pool of 2^31 blocks would
  // be 4 TB.)
  constexpr int kAll = kSelectWaves * 16;
  int at[2], unit[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int blk = blk0 + (wave + (4 * i + quad) * kSelectWaves) * 16 + i16;
    at[i] = blk < end ? (int)kv_place(a.c, b, h, blk) : -1;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) unit[i] = at[i] < 0 ? kNoPage : a.unit[at[i]];
  auto of_turn = [&](const int (&x)[2], int turn, int j) {
    return __shfl(turn < 4 ? x[0] : x[1], turn % 4 * 16 + j);
  };
  I4 r[2][kStep];
  auto load = [&](int set, int turn) {
    const int from = turn < 8 ? of_turn(at, turn, i16) : -1;
    const I4* p =
        (const I4*)(a.range + (int64_t)(from < 0 ? 0 : from) * (2 * D)) + quad;
#pragma unroll
    for (int i = 0; i < kStep; ++i)
      r[set][i] = from < 0 ? I4{0, 0, 0, 0} : p[4 * i];
  };
  load(0, 0);
  {
    typedef PackQuery<D, kHalf> Pack;
    Pack now;
    if (wave < queries) now = Pack(a, b, h, t0 + wave);
    for (int i = wave; i < rows; i += kSelectWaves) {
      if (i < queries) {
        Pack then;
        if (i + kSelectWaves < queries)
          then = Pack(a, b, h, t0 + i + kSelectWaves);
        now.put(a, sq[i]);
        now = then;
      } else {
        for (int c = lane; c < D / 2; c += kWave) ((uint32_t*)sq[i])[c] = 0;
      }
    }
  }
  __syncthreads();
  int turn = 0, blk = blk0 + wave * 16;
  auto step = [&](int set) {
    load(1 - set, turn + 1);
    int us[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) us[e] = of_turn(unit, turn, quad * 4 + e);
    for (int q0 = 0; q0 < queries; q0 += 16) {
      I4 s = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kStep; ++i)
        s = __builtin_amdgcn_mfma_i32_16x16x64_i8(
            r[set][i], *(const I4*)&sq[q0 + i16][i * 64 + quad * 16], s, 0, 0,
            0);
      if (q0 + i16 < queries)
        put(q0 + i16, blk + quad * 4,
            uint4{score_key<D>(s[0], us[0]), score_key<D>(s[1], us[1]),
                  score_key<D>(s[2], us[2]), score_key<D>(s[3], us[3])});
    }
    blk += kAll;
    ++turn;
  };
  while (blk < end) {
#pragma unroll
    for (int set = 0; set < 2; ++set)
      if (blk < end) step(set);
  }
}

// The scores of a piece of a row's blocks, into memory: for rows whose keys a
// workgroup does not hold.
constexpr int kScorePiece = 128;  // blocks: pieces are multiples of it

template <int D, bool kHalf>
__global__ __launch_bounds__(kSelectThreads) void k_kv4_scores(SelectArgs a) {
  __shared__ __align__(16) int8_t sq[16][2 * D + 16];
  // tiles of one piece follow each other on one XCD (32 bits hold all of these)
  const uint32_t k = blockIdx.x / 8;
  const int tile = (int)(k % (uint32_t)a.tiles);
  const uint32_t item = k / (uint32_t)a.tiles * 8 + blockIdx.x % 8;
  const uint32_t rows = (uint32_t)a.batch * (uint32_t)a.c.heads;
  const uint32_t bh = item % rows;
  const int piece = (int)(item / rows);
  if (piece >= a.pieces) return;
  const int64_t b = bh / (uint32_t)a.c.heads;
  const int h = (int)(bh % (uint32_t)a.c.heads);
  const int64_t len = kv_len_of(a, b), nq = q_len_of(a, b);
  const int64_t t0 = (int64_t)tile * 16;
  const int queries = (int)std::max<int64_t>(
      0, std::min<int64_t>(std::min<int64_t>(a.tokens, nq) - t0, 16));
  const int blk0 = piece * a.piece;
  if (queries == 0) return;
  const int end = std::min(
      blk0 + a.piece,
      (token_sees(a, len, nq, t0 + queries - 1) + kKvBlock - 1) / kKvBlock);
  if (blk0 >= end) return;
  uint32_t* keys = a.keys + ((b * a.tokens + t0) * a.c.heads + h) * a.pitch;
  score_blocks<D, kHalf>(
      a, b, h, t0, queries, 16, blk0, end, sq, [&](int q, int blk, uint4 key) {
        *(uint4*)(keys + (int64_t)q * a.c.heads * a.pitch + blk) = key;
      });
}

// The blocks of a query with the keys key[0 .. last] in LDS, by a wave that keeps
// kRegs of them in each lane: the least key that is taken, from counts of 64 equal
// parts of the keys' range and then bit by bit, until as many as are wanted lie past
// it; then the blocks past it, and those at it while there is room.
// bins: 64 words of the wave's own.  Bit by bit from the start 64 x 17 tokens take 18.4
// us, 2,048 of a prompt 44, with the counts first 16.2 and 40; the keys of one part a
// lane's each, as pick_together has them, changed neither.
template <int kRegs>
__device__ __forceinline__ void pick_blocks(int sinks, int recent, int all,
                                            int last, const uint32_t* key,
                                            uint32_t* bins, int32_t* out) {
  const int lane = lane_id();
  uint32_t k[kRegs];
  uint32_t sure = 0;  // a bit for each register
  uint32_t hi = 0, lo = 0;
  int want = all;
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int j = i * kWave + lane;
    k[i] = j <= last ? key[j] : 0;
    if (i * kWave < sinks || (i + 1) * kWave > last - recent) {
      const bool is = k[i] && (j < sinks || j > last - recent);
      want -= popc(ballot(is));
      if (is) {
        sure |= 1u << i;
        k[i] = 0;
      }
    }
    hi = max(hi, k[i]);
    lo = max(lo, 0u - k[i]);  // (none is the least)
  }
  // line: keys past it are taken, and `room` of those at it
  uint32_t line = 0xffffffffu;
  int room = 0;
  if (want > 0) {
    hi = wave_all_max(hi);
    lo = 0u - wave_all_max(lo);
    const int shift = max(0, 26 - __builtin_clz((hi - lo) | 1u));
    bins[lane] = 0;
    wave_lds_sync();
#pragma unroll
    for (int i = 0; i < kRegs; ++i)
      if (k[i]) atomicAdd(&bins[(k[i] - lo) >> shift], 1u);
    wave_lds_sync();
    const int upto = (int)wave_incl_scan(bins[kWave - 1 - lane]);
    const uint64_t enough = ballot(upto >= want);
    line = 0;
    if (enough && __builtin_amdgcn_readlane(upto, kWave - 1) > want) {
      const int f = __builtin_ctzll(enough);
      line = lo + ((uint32_t)(kWave - 1 - f) << shift);
      int n = __builtin_amdgcn_readlane(upto, f);
      auto at_least = [&](uint32_t x) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < kRegs; ++i) c += popc(ballot(k[i] >= x));
        return c;
      };
      for (int bit = shift - 1; bit >= 0 && n != want; --bit) {
        const int c = at_least(line + (1u << bit));
        if (c >= want) {
          line += 1u << bit;
          n = c;
        }
      }
      if (n == want)
        --line;  // those past it now are the wanted ones
      else
        room = want - at_least(line + 1);
    }
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

// As pick_blocks, by a workgroup with the keys of up to 64 kRegs kPickWaves blocks in
// its registers.  Among 1,024 equal parts of the keys' range it looks for the one that
// the line lies in, and the keys of that part, if they are no more than 64, are a
// lane's each in every wave.  Two bits of the line at a time, a barrier each, one token
// over 131,072 took 14.7 us and 4 x 9 29.7, now 11.2 and 23.9.
constexpr int kParts = 1024;

template <int kRegs, int kPickWaves>
struct PickRoom {
  uint32_t of_wave[3][4][16];
  uint32_t at[kRegs * kPickWaves];  // past the line, and on it << 16
  __align__(16) uint32_t bins[kParts];
  uint32_t line_bin[3], cand[kWave], cands;
};

template <int kRegs, int kPickWaves>
__device__ __forceinline__ void pick_together(
    int sinks, int recent, int all, int last, const uint32_t* keys,
    PickRoom<kRegs, kPickWaves>& lds, int32_t* out) {
  // (a row of a wave's lanes sums up one number of each wave)
  static_assert(kPickWaves <= 16, "");
  constexpr int kThreads = kPickWaves * kWave;
  const int tid = threadIdx.x, lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  uint32_t k[kRegs], sure = 0, hi = 0, lo = 0;
  uint32_t n_sure = 0, n_some = 0;
#pragma unroll
  for (int i = tid; i < kParts; i += kThreads) lds.bins[i] = 0;
  if (tid == 0) lds.cands = 0;
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int j = i * kThreads + tid;
    k[i] = j <= last ? keys[j] : 0;
  }
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const int j = i * kThreads + tid;
    const bool is = k[i] && (j < sinks || j > last - recent);
    n_sure += (uint32_t)popc(ballot(is));
    if (is) {
      sure |= 1u << i;
      k[i] = 0;
    }
    n_some += (uint32_t)popc(ballot(k[i] > 0));
    hi = max(hi, k[i]);
    lo = max(lo, 0u - k[i]);  // (none is the least)
  }
  hi = wave_all_max(hi);
  lo = wave_all_max(lo);
  if (lane == 0) {
    lds.of_wave[2][0][wave] = n_sure;
    lds.of_wave[2][1][wave] = n_some;
    lds.of_wave[2][2][wave] = hi;
    lds.of_wave[2][3][wave] = lo;
  }
  __syncthreads();
  auto row_sums = [&](int turn) {
    return row16_incl_scan(lane % 16 < kPickWaves
                               ? lds.of_wave[turn][lane / 16][lane % 16]
                               : 0);
  };
  auto of_row = [](uint32_t x, int row) {
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 16 * row + 15);
  };
  const uint32_t sums = row_sums(2);
  const int want = all - (int)of_row(sums, 0);
  const int some = (int)of_row(sums, 1);
  hi = wave_all_max(lane < kPickWaves ? lds.of_wave[2][2][lane] : 0);
  lo = 0u - wave_all_max(lane < kPickWaves ? lds.of_wave[2][3][lane] : 0);
  int turn = 0;
  // keys of at least x, x + step, x + 2 step
  auto at_least = [&](uint32_t x, uint32_t step, int (&n)[3]) {
#pragma unroll
    for (int s = 0; s < 3; ++s) {
      n[s] = 0;
#pragma unroll
      for (int i = 0; i < kRegs; ++i)
        n[s] += popc(ballot(k[i] >= x + s * step));
      if (lane == 0) lds.of_wave[turn][s][wave] = (uint32_t)n[s];
    }
    __syncthreads();
    const uint32_t sums = row_sums(turn);
#pragma unroll
    for (int s = 0; s < 3; ++s) n[s] = (int)of_row(sums, s);
    turn ^= 1;
  };
  uint32_t line = 0;
  int room = 0;
  if (want <= 0) {
    line = 0xffffffffu;
  } else if (some > want) {
    const int shift = max(0, 22 - __builtin_clz((hi - lo) | 1u));
#pragma unroll
    for (int i = 0; i < kRegs; ++i)
      if (k[i]) atomicAdd(&lds.bins[(k[i] - lo) >> shift], 1u);
    __syncthreads();
    if (wave == 0) {
      // a lane's 16 parts, the largest keys first
      uint32_t x[16], n = 0;
      const uint4* p = (const uint4*)lds.bins + (kWave - 1 - lane) * 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 v = p[3 - i];
        x[4 * i] = v.w;
        x[4 * i + 1] = v.z;
        x[4 * i + 2] = v.y;
        x[4 * i + 3] = v.x;
        n += v.x + v.y + v.z + v.w;
      }
      int upto = (int)(wave_incl_scan(n) - n);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int next = upto + (int)x[i];
        if (upto < want && next >= want) {
          lds.line_bin[0] = (uint32_t)(kParts - 1 - lane * 16 - i);
          lds.line_bin[1] = (uint32_t)upto;
          lds.line_bin[2] = (uint32_t)next;
        }
        upto = next;
      }
    }
    __syncthreads();
    const uint32_t bin = lds.line_bin[0];
    const int past = (int)lds.line_bin[1], upto = (int)lds.line_bin[2];
    line = lo + (bin << shift);
    bool exact = upto == want;
    if (!exact && upto - past <= kWave) {
      // a wave's lanes hold what lies in that part
#pragma unroll
      for (int i = 0; i < kRegs; ++i)
        if (k[i] && (k[i] - lo) >> shift == bin)
          lds.cand[atomicAdd(&lds.cands, 1u)] = k[i];
      __syncthreads();
      const uint32_t x = lane < upto - past ? lds.cand[lane] : 0;
      int n = upto;
      for (int bit = shift - 1; bit >= 0 && n != want; --bit) {
        const uint32_t y = line + (1u << bit);
        const int c = past + popc(ballot(x >= y));
        if (c >= want) {
          line = y;
          n = c;
        }
      }
      exact = n == want;
      room = want - past - popc(ballot(x > line));
    } else if (!exact) {
      // many equal or nearly equal keys; (an even number of bits is left)
      for (int bit = (shift - 1) & ~1; bit >= 0 && !exact; bit -= 2) {
        const uint32_t step = 1u << bit;
        int n[3];
        at_least(line + step, step, n);
        uint32_t more = 0;
#pragma unroll
        for (int s = 0; s < 3; ++s) {
          if (n[s] >= want) more = (uint32_t)(s + 1) * step;
          exact = exact || n[s] == want;
        }
        line += more;
      }
      if (!exact) {
        int n[3];
        at_least(line + 1, 0, n);
        room = want - n[0];
      }
    }
    if (exact) {
      --line;  // those past it now are the wanted ones
      room = 0;
    }
  }
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const uint64_t gt = ballot(k[i] > line || (sure >> i & 1));
    const uint64_t eq = ballot(room > 0 && k[i] == line);
    if (lane == 0)
      lds.at[i * kPickWaves + wave] = (uint32_t)(popc(gt) | popc(eq) << 16);
  }
  __syncthreads();
  // what comes before each 64, and in all; no sum passes 16 bits
  uint32_t sum = 0;
  if (wave == 0) {
    for (int i0 = 0; i0 < kRegs * kPickWaves; i0 += kWave) {
      const bool is = i0 + lane < kRegs * kPickWaves;
      const uint32_t x = is ? lds.at[i0 + lane] : 0;
      const uint32_t to = wave_incl_scan(x);
      if (is) lds.at[i0 + lane] = sum + to - x;
      sum += (uint32_t)__builtin_amdgcn_readlane((int)to, kWave - 1);
    }
    const int n = (int)(sum & 0xffffu) + min((int)(sum >> 16), room);
    for (int i = n + lane; i < all; i += kWave) out[i] = -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRegs; ++i) {
    const uint32_t before = lds.at[i * kPickWaves + wave];
    const bool over = k[i] > line || (sure >> i & 1);
    const bool on = room > 0 && k[i] == line;
    const int gt = (int)(before & 0xffffu) + rank_lt(ballot(over));
    const int eq = (int)(before >> 16) + rank_lt(ballot(on));
    if (over || (on && eq < room))
      out[gt + min(eq, room)] = i * kThreads + tid;
  }
}

// Scores and choice at once, where a workgroup holds the keys of its tokens: rows
// of up to 1,024 blocks.
constexpr int kSelectTokens = 32;
constexpr int kSelectBlocks = 1024;
constexpr int kSelectRegs = kSelectBlocks / kSelectThreads;
typedef PickRoom<kSelectRegs, kSelectThreads / kWave> SelectRoom;

// kFew: all waves choose for one token after the other, rather than each for its own
// (64 x 1 tokens over up to 32,768 28.6 and 26.3 us).  A kernel of its own: with both in
// one the registers leave five waves a SIMD of seven, and a prompt takes 44 us
// instead of 38.
template <int D, bool kHalf, bool kFew>
__global__ __launch_bounds__(kSelectThreads) void k_kv4_select(SelectArgs a) {
  constexpr int kPitch = 2 * D + 16;
  constexpr int kSelectWaves = kSelectThreads / kWave;
  extern __shared__ __align__(16) char lds[];
  // tiles of one row and KV head follow each other on one XCD (32 bits hold all
  // of these)
  const uint32_t k = blockIdx.x / 8;
  const int tile = (int)(k % (uint32_t)a.tiles);
  const uint32_t bh = k / (uint32_t)a.tiles * 8 + blockIdx.x % 8;
  if (bh >= (uint32_t)a.batch * (uint32_t)a.c.heads) return;
  const int64_t b = bh / (uint32_t)a.c.heads;
  const int h = (int)(bh % (uint32_t)a.c.heads);
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
  score_blocks<D, kHalf>(a, b, h, t0, queries, (tokens + 15) / 16 * 16, 0,
                         blocks, sq, [&](int q, int blk, uint4 key) {
                           *(uint4*)(keys + q * pitch + blk) = key;
                         });
  __syncthreads();
  auto last_of = [&](int i) {
    return __builtin_amdgcn_readfirstlane(
        (token_sees(a, len, nq, t0 + i) + kKvBlock - 1) / kKvBlock - 1);
  };
  auto out_of = [&](int i) {
    return a.selected + ((b * a.tokens + t0 + i) * a.c.heads + h) * a.want;
  };
  if constexpr (kFew) {
    __shared__ SelectRoom room;
    for (int i = 0; i < tokens; ++i) {
      if (i) __syncthreads();
      pick_together<kSelectRegs, kSelectWaves>(a.sinks, a.recent, a.want,
                                               last_of(i), keys + i * pitch,
                                               room, out_of(i));
    }
  } else {
    __shared__ uint32_t bins[kSelectWaves][kWave];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    for (int i = wave; i < tokens; i += kSelectWaves) {
      const int last = last_of(i);
      const uint32_t* own = keys + i * pitch;
      int32_t* out = out_of(i);
      if (last < 4 * kWave)
        pick_blocks<4>(a.sinks, a.recent, a.want, last, own, bins[wave], out);
      else if (last < 8 * kWave)
        pick_blocks<8>(a.sinks, a.recent, a.want, last, own, bins[wave], out);
      else
        pick_blocks<16>(a.sinks, a.recent, a.want, last, own, bins[wave], out);
    }
  }
}

// The choice by a workgroup of 1,024 threads, for rows whose keys are in memory.
constexpr int kWideThreads = 1024;
constexpr int kWideWaves = kWideThreads / kWave;

struct WideList {
  int last;
  const uint32_t* keys;
  int32_t* out;
  __device__ __forceinline__ WideList(const SelectArgs& a) {
    const uint32_t list = blockIdx.x, token = list / (uint32_t)a.c.heads;
    const uint32_t b = token / (uint32_t)a.tokens;
    const uint32_t t = token % (uint32_t)a.tokens;
    const int sees = token_sees(a, kv_len_of(a, b), q_len_of(a, b), t);
    last = (sees + kKvBlock - 1) / kKvBlock - 1;
    keys = a.keys + list * a.pitch;
    out = a.selected + (int64_t)list * a.want;
  }
};

template <int kRegs>
__global__ __launch_bounds__(kWideThreads) void k_kv4_pick_wide(SelectArgs a) {
  __shared__ PickRoom<kRegs, kWideWaves> room;
  const WideList l(a);
  pick_together<kRegs, kWideWaves>(a.sinks, a.recent, a.want, l.last, l.keys,
                                   room, l.out);
}

// The key of block j for what follows: first and recent blocks above all others.
__device__ __forceinline__ uint32_t ranked(const SelectArgs& a, uint32_t key,
                                           int j, int last) {
  if (j > last || key == 0) return 0;
  return j < a.sinks || j > last - a.recent ? 0xffffffffu : key;
}

// Rows of any length: the keys stay in memory, and four passes narrow the line
// down by 8 bits each.  (71 us for a list of 32,768 blocks: a workgroup's loads, of
// which few are under way at a time.)
__global__ __launch_bounds__(kWideThreads) void k_kv4_pick_far(SelectArgs a) {
  __shared__ int hist[256];
  __shared__ int sums[kWideWaves];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWave;
  const WideList l(a);
  const int last = l.last;
  const uint32_t* keys = l.keys;
  int32_t* out = l.out;
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

// Whether one launch serves.  With the rows' scores cut into pieces and a second
// launch for the choice few lists of long rows are chosen sooner: of 1,024 blocks each
// for one token of one row 14.4 us in one launch, 10.3 in two, of 16 rows 16.9 and
// 16.8, five tokens of four rows 19.7 and 11.9, 17 of 16 rows 26 and 36; of 512 blocks
// 10.5 and 10.4, 11.0 and 13.0.
bool held_in_lds(const sfx_kv4* c, int64_t batch, int64_t tokens) {
  const int64_t blocks = pitch_of(c);
  return blocks <= kSelectBlocks / 2 ||
         (blocks <= kSelectBlocks && batch * tokens * c->heads > 256);
}

// In one launch, the tokens of a workgroup: as many as its 64 KB hold keys of; past
// kSelectTokens in tiles of 16.
int64_t held_span(const sfx_kv4* c, int64_t tokens) {
  const int64_t row = 4 * (pitch_of(c) + 4), packed = 2 * c->head_dim + 16;
  const int64_t room = 65536 - kSelectThreads * 4 - kSelectTokens * packed;
  return std::min<int64_t>(tokens <= kSelectTokens ? tokens : 16, room / row);
}

bool select_ok(const sfx_kv4* c, int64_t batch, int64_t tokens) {
  KvView v;
  if (!kv_view(c, &v) || batch < 0 || batch > 65535 || tokens < 0 ||
      tokens > (int64_t(1) << 24))
    return false;
  if (batch == 0 || tokens == 0) return true;
  // a grid's threads: of a workgroup for each tile, or for each list
  if (!held_in_lds(c, batch, tokens))
    return batch * tokens <= ((int64_t(1) << 22) - 1) / c->heads;
  const int64_t span = held_span(c, tokens);
  return (batch * c->heads + 7) / 8 * 8 * ((tokens + span - 1) / span) <
         (int64_t(1) << 32) / kSelectThreads;
}

template <int D, bool kHalf>
int launch_held(SelectArgs a, const sfx_kv4* cache, hipStream_t stream) {
  a.span = (int)held_span(cache, a.tokens);
  a.tiles = (int)((a.tokens + a.span - 1) / a.span);
  const size_t lds =
      (a.span + 15) / 16 * 16 * (2 * D + 16) + a.span * 4 * (a.pitch + 4);
  const int64_t items = (a.batch * a.c.heads + 7) / 8 * 8;
  const dim3 grid((unsigned)(items * a.tiles)), block(kSelectThreads);
  // one token, of up to 1,024 blocks, by a wave 18 us, by all of them 14; of up to 256
  // 7.8 and 8.6
  if (a.span <= 2 && a.pitch > kSelectBlocks / 4)
    hipLaunchKernelGGL((k_kv4_select<D, kHalf, true>), grid, block, lds, stream,
                       a);
  else
    hipLaunchKernelGGL((k_kv4_select<D, kHalf, false>), grid, block, lds,
                       stream, a);
  return (int)hipGetLastError();
}

template <int D, bool kHalf>
int launch_wide(SelectArgs a, hipStream_t stream) {
  a.span = 16;
  a.tiles = (int)((a.tokens + 15) / 16);
  const int64_t lists = a.batch * a.tokens * a.c.heads;
  // two workgroups a CU where the rows are few, long pieces where they are many
  const int64_t whole = a.batch * a.c.heads * a.tiles;
  const int64_t piece = std::min<int64_t>(whole * a.pitch / 512, 1024);
  a.piece = (int)std::max<int64_t>(piece / kScorePiece, 1) * kScorePiece;
  a.pieces = (int)((a.pitch + a.piece - 1) / a.piece);
  const int64_t items = (a.batch * a.c.heads * a.pieces + 7) / 8 * 8;
  if (items * a.tiles >= (int64_t(1) << 32) / kSelectThreads)
    return SFX_EINVAL;
  hipLaunchKernelGGL((k_kv4_scores<D, kHalf>),
                     dim3((unsigned)(items * a.tiles)), dim3(kSelectThreads), 0,
                     stream, a);
  const dim3 grid((unsigned)lists), block(kWideThreads);
  const int64_t blocks = a.c.positions / kKvBlock;
  if (blocks <= 4 * kWideThreads)
    hipLaunchKernelGGL(k_kv4_pick_wide<4>, grid, block, 0, stream, a);
  else if (blocks <= 16 * kWideThreads)
    hipLaunchKernelGGL(k_kv4_pick_wide<16>, grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL(k_kv4_pick_far, grid, block, 0, stream, a);
  return (int)hipGetLastError();
}

template <int D, bool kHalf>
int launch(const SelectArgs& a, const sfx_kv4* cache, hipStream_t stream) {
  return held_in_lds(cache, a.batch, a.tokens)
             ? launch_held<D, kHalf>(a, cache, stream)
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
  if (!select_ok(cache, batch, tokens) || held_in_lds(cache, batch, tokens))
    return 0;
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
