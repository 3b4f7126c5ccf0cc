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
  int tiles;     // of 16 query tokens
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
  const int lane = lane_id();
  const uint16_t* q = (const uint16_t*)a.q.data + b * a.q.stride_b +
                      t * a.q.stride_t + (int64_t)h * a.group * a.q.stride_h +
                      lane * C;
  auto bits = [&](int g, int c) {
    const uint32_t x = q[g * a.q.stride_h + c];
    return (x & 0x7fffu) >= (kHalf ? 0x7c00u : 0x7f80u) ? 0u : x;
  };
  int top = 0;
  for (int g = 0; g < a.group; ++g)
#pragma unroll
    for (int c = 0; c < C; ++c) top = max(top, (int)(bits(g, c) & 0x7fffu));
  top = wave_max_i32(top);
  // 2^e is the power of two above the largest
  const int e =
      __builtin_amdgcn_frexp_expf(to_float16b<kHalf>((uint32_t)top));
  uint32_t p[C], n[C];
  uint32_t most = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) p[c] = n[c] = 0;
  for (int g = 0; g < a.group; ++g)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int z = (int)rintf(
          __builtin_amdgcn_ldexpf(to_float16b<kHalf>(bits(g, c)), 15 - e));
      p[c] += (uint32_t)max(z, 0);
      n[c] += (uint32_t)max(-z, 0);
    }
#pragma unroll
  for (int c = 0; c < C; ++c) most = max(most, max(p[c], n[c]));
  most = (uint32_t)wave_max_i32((int)most);
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
  const int64_t t0 = (int64_t)tile * 16;
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

// The key of block j of a query whose last block is `last`, first and recent
// blocks above all others.
__device__ __forceinline__ uint32_t ranked(const SelectArgs& a, uint32_t key,
                                           int j, int last) {
  if (j > last || key == 0) return 0;
  return j < a.sinks || j > last - a.recent ? 0xffffffffu : key;
}

// A wave per query token and KV head, whose keys it keeps: the threshold bit by
// bit, then the blocks past it, and those at it while there is room.
constexpr int kPickRegs = 16;

__global__ __launch_bounds__(256) void k_kv4_pick(SelectArgs a) {
  const int64_t list = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
  if (list >= a.batch * a.tokens * a.c.heads) return;
  const int lane = lane_id();
  const int64_t b = list / (a.tokens * a.c.heads);
  const int64_t t = list / a.c.heads % a.tokens;
  const int sees = token_sees(a, kv_len_of(a, b), q_len_of(a, b), t);
  const int last = __builtin_amdgcn_readfirstlane((sees + kKvBlock - 1) /
                                                  kKvBlock) - 1;
  const uint32_t* keys = a.keys + list * a.pitch;
  int32_t* out = a.selected + list * a.want;
  const int regs = last / kWave + 1;
  uint32_t k[kPickRegs];
#pragma unroll
  for (int i = 0; i < kPickRegs; ++i) {
    const int j = i * kWave + lane;
    k[i] = 0;
    if (i < regs && j <= last) k[i] = ranked(a, keys[j], j, last);
  }
  auto at_least = [&](uint32_t x) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kPickRegs; ++i)
      if (i < regs) n += popc(ballot(k[i] >= x));
    return n;
  };
  uint32_t line = 1;
  if (at_least(1) > a.want) {
    line = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t x = line | 1u << bit;
      if (at_least(x) >= a.want) line = x;
    }
  }
  int above = 0;
#pragma unroll
  for (int i = 0; i < kPickRegs; ++i)
    if (i < regs) above += popc(ballot(k[i] > line));
  int room = a.want - above, n = 0;  // room: for those at the line
#pragma unroll
  for (int i = 0; i < kPickRegs; ++i) {
    if (i >= regs) continue;
    const uint64_t eq = ballot(k[i] == line && line > 0);
    const bool in = k[i] > line || (k[i] == line && rank_lt(eq) < room);
    const uint64_t m = ballot(in);
    if (in) out[n + rank_lt(m)] = i * kWave + lane;
    n += popc(m);
    room -= popc(eq);
    if (room < 0) room = 0;
  }
  for (int i = n + lane; i < a.want; i += kWave) out[i] = -1;
}

// The same by a workgroup, for tables of more blocks than a wave keeps: the keys
// stay in memory, and four passes narrow the threshold down by 8 bits each.
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

template <int D, bool kHalf>
int launch(const SelectArgs& a, hipStream_t stream) {
  const int64_t lists = a.batch * a.tokens * a.c.heads;
  const int64_t items = (a.batch * a.c.heads * a.chunks + 7) / 8 * 8;
  if (items * a.tiles >= (int64_t(1) << 32) / kScoreThreads) return SFX_EINVAL;
  hipLaunchKernelGGL((k_kv4_scores<D, kHalf>),
                     dim3((unsigned)(items * a.tiles)), dim3(kScoreThreads), 0,
                     stream, a);
  if (a.c.positions / kKvBlock <= kPickRegs * kWave)
    hipLaunchKernelGGL(k_kv4_pick, dim3((unsigned)((lists + 3) / 4)), dim3(256),
                       0, stream, a);
  else
    hipLaunchKernelGGL(k_kv4_pick_wide, dim3((unsigned)lists),
                       dim3(kWideThreads), 0, stream, a);
  return (int)hipGetLastError();
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
  if (!select_ok(cache, batch, tokens)) return 0;
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
  a.range = bounds->range;
  a.unit = bounds->unit;
  a.want = (int)blocks;
  a.sinks = (int)first;
  a.recent = (int)recent;
  a.tiles = (int)((tokens + 15) / 16);
  a.pitch = pitch_of(cache);
  a.chunks = (int)((a.pitch + kScoreChunk - 1) / kScoreChunk);
  a.keys = (uint32_t*)workspace;
  a.selected = selected;
  const bool half = cache->dtype == SFX_F16;
  switch (cache->head_dim) {
    case 64:
      return half ? launch<64, true>(a, stream) : launch<64, false>(a, stream);
    case 128:
      return half ? launch<128, true>(a, stream)
                  : launch<128, false>(a, stream);
    default:
      return half ? launch<256, true>(a, stream)
                  : launch<256, false>(a, stream);
  }
}
