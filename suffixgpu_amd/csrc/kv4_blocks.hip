// Attention over selected blocks of the 4-bit cache.  The mathematics is in
// kv4_attend.h: a workgroup takes the query heads of one KV head of as many tokens
// as give 16 rows, over the blocks that any of these tokens selected (or a part of
// them); a row passes over the blocks of the others.  Neighbouring tokens select
// much the same blocks, each of which is then loaded and converted once.
//
// 2,048 tokens of a prompt with 64 blocks each of 512: 143 us and 8 for the unions,
// which have 84 blocks on average; vector instructions issue in 83% of the cycles,
// matrix instructions in 30%.  64 x 17 tokens with 32 of 256 36 and 7.  Single tokens
// are bound by memory: 64 with 64 of 1,024 27 us, 145 MB, 5.4 TB/s.
// Tiles of 32 rows, whose unions are larger (97 blocks), gave 170 us instead of 177 for
// the prompt, 53 instead of 50 for 64 x 17.  Keys as their 4 bits stand, in products
// with 8-bit parts of the queries, gave 143 instead of 156 in all, but the instruction
// adds 32 channels to fewer than 24 bits.

#include <algorithm>

#include "kv4_attend.h"
#include "launch.h"

namespace sfx {

namespace {

struct ListArgs : AttendArgs {
  const int32_t* selected;  // [batch, tokens, heads, width]
  int width;
  int span;   // query tokens of a tile
  int tiles;  // of 16 query heads, of a token with more than that
  // with a span of more than one: the blocks of each tile [batch, heads, tiles of
  // the query, span * width] and their number
  int2* entry;
  int32_t* entries;
};

// The first query row of tile qt, and the row behind its last.
__device__ __forceinline__ int first_row(const ListArgs& a, int qt) {
  return a.tiles > 1 ? qt / a.tiles * a.group + qt % a.tiles * 16
                     : qt * a.span * a.group;
}
__device__ __forceinline__ int end_row(const ListArgs& a, int qt) {
  const int t = a.tiles > 1 ? qt / a.tiles + 1 : (qt + 1) * a.span;
  return (int)min((int64_t)t, a.tokens) * a.group;
}

// The blocks that any token of a tile has in its list, in order, with the rows of
// the tokens that take them (a bit each), by a workgroup: a window of the row's
// blocks at a time, of which each token has a bit for each, so that a block named
// twice is one.
// 1,024 threads for rows that a window of 256 does not span: 32 tiles of eight tokens
// with 96 blocks each of up to 4,096 take 7.5 us, by 256 threads 9.  64 where there
// are many tiles and a window of 64 spans the rows: 4,096 of four tokens with 64 blocks
// each of 512 take 8 us, by 256 threads 12, but 384 of two tokens with 48 each 0.7 more.
template <int kUnionThreads>
__global__ __launch_bounds__(kUnionThreads) void k_kv4_union(ListArgs a) {
  constexpr int kWindow = 8 * kUnionThreads;  // eight blocks a thread
  constexpr int kWords = kWindow / 32;
  constexpr int kUnionWaves = kUnionThreads / kWave;
  __shared__ uint32_t bits[16][kWords];
  __shared__ int sums[kUnionWaves];
  const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWave;
  const uint32_t tile = blockIdx.x;  // [batch, heads, q_tiles]
  const int qt = (int)(tile % (uint32_t)a.q_tiles);
  const uint32_t bh = tile / (uint32_t)a.q_tiles;
  const int h = (int)(bh % (uint32_t)a.c.heads);
  const int64_t b = bh / (uint32_t)a.c.heads;
  const int64_t len = kv_len_of(a, b), nq = q_len_of(a, b);
  const int t0 = qt * a.span;
  const int32_t* lists =
      a.selected + ((b * a.tokens + t0) * a.c.heads + h) * a.width;
  const int64_t next = (int64_t)a.c.heads * a.width;
  int2* out = a.entry + (int64_t)tile * a.span * a.width;
  // a later token sees no less
  int limit = 0;
  for (int k = 0; k < a.span; ++k)
    limit = max(limit, (visible(a, len, nq, (t0 + k) * a.group) + kKvBlock - 1) /
                           kKvBlock);
  const uint32_t rows = (1u << a.group) - 1;  // of a token (several: at most 8)
  int count = 0;
  for (int w0 = 0; w0 < limit; w0 += kWindow) {
    for (int i = tid; i < a.span * kWords; i += kUnionThreads)
      bits[i / kWords][i % kWords] = 0;
    __syncthreads();
    for (int k = wave; k < a.span; k += kUnionWaves) {
      // none where the token is none
      const int sees = visible(a, len, nq, (t0 + k) * a.group);
      const int n = min((sees + kKvBlock - 1) / kKvBlock - w0, kWindow);
      if (n <= 0) continue;
      for (int e = lane; e < a.width; e += kWave) {
        const int64_t r = (int64_t)lists[k * next + e] - w0;
        if (r >= 0 && r < n) atomicOr(&bits[k][r / 32], 1u << (r % 32));
      }
    }
    __syncthreads();
    const int word = tid / 4, at = tid % 4 * 8;
    uint32_t any = 0;
    for (int k = 0; k < a.span; ++k) any |= bits[k][word] >> at;
    any &= 255u;
    const uint32_t n = (uint32_t)__builtin_popcount(any);
    const uint32_t to = wave_incl_scan(n);
    if (lane == kWave - 1) sums[wave] = (int)to;
    __syncthreads();
    int pos = count + (int)(to - n);
#pragma unroll
    for (int w = 0; w < kUnionWaves; ++w) {
      if (w < wave) pos += sums[w];
      count += sums[w];
    }
    while (any) {
      const int bit = at + __builtin_ctz(any);
      any &= any - 1;
      uint32_t m = 0;
      for (int k = 0; k < a.span; ++k)
        m |= (bits[k][word] >> bit & 1) * rows << k * a.group;
      out[pos++] = int2{w0 + word * 32 + bit, (int)m};
    }
    __syncthreads();
  }
  if (tid == 0) a.entries[tile] = count;
}

typedef const __attribute__((address_space(4))) int32_t* Scalars;

// threadIdx.x for what is worked out again in a loop rather than kept in a
// register, of which the attention has none to spare.
__device__ __forceinline__ int fresh_thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  return t;
}

// A block of a list, negative where there is none, and the rows that take it.
struct Entry {
  int blk;
  uint32_t rows;
};

// As each_block, over entries first, first + step, ... below last.  An entry is read
// (as a scalar) a block ahead of its page id, and that a block ahead of the loads.
template <class B, class Read, class F>
__device__ __forceinline__ void each_entry(const KvView& c, int64_t b, int h,
                                           int bytes, int first, int step,
                                           int last, Read read, F body) {
  if (first >= last || c.num_pages == 0) return;
  const Scalars ids = (Scalars)(uintptr_t)(c.table + b * c.table_stride);
  const int in_page = (1 << c.page_shift) - 1;
  const uint32_t pages = (uint32_t)min(c.num_pages, int64_t(1) << 31);
  auto page = [&](Entry e) {
    return e.blk < 0 ? -1 : ids[e.blk >> c.page_shift];
  };
  auto good = [&](int32_t id) { return (uint32_t)id < pages; };
  // past the last block, and without a page: memory that is there
  auto at = [&](int32_t id, Entry e) {
    return good(id) ? c.pages + ((((int64_t)id * c.heads + h) << c.page_shift) +
                                 (e.blk & in_page)) * bytes
                    : c.pages;
  };
  auto entry = [&](int i) { return read(min(i, last - 1)); };
  B x;
  Entry e = entry(first), e1 = entry(first + step), e2 = entry(first + 2 * step);
  int32_t id = page(e), id1 = page(e1);
  x.load_k(at(id, e));
  x.load_v(at(id, e));
  for (int i = first; i < last; i += step) {
    const char* next = at(id1, e1);
    const int32_t id2 = page(e2);
    const Entry e3 = entry(i + 3 * step);
    if (good(id)) {
      body(x, e, [&]() { x.load_k(next); }, [&]() { x.load_v(next); });
    } else {
      x.load_k(next);
      x.load_v(next);
    }
    e = e1;
    e1 = e2;
    e2 = e3;
    id = id1;
    id1 = id2;
  }
}

// The list of a single token.  It ascends, as select_blocks gives it, or each of
// its entries is looked for among those before it.
struct OneList {
  int splits, first, step, last, limit;
  bool ascends;
  Scalars list;
  __device__ __forceinline__ OneList(const ListArgs& a, const Work& wk, int64_t,
                                     int most, int wave) {
    splits = a.splits;
    first = wk.split * kWaves + wave;
    step = splits * kWaves;
    last = a.width;
    limit = (most + kKvBlock - 1) / kKvBlock;
    const int32_t* p =
        a.selected +
        ((wk.b * a.tokens + wk.qt / a.tiles) * a.c.heads + wk.h) * a.width;
    bool bad = false;
    for (int e = lane_id(); e < last; e += kWave) {
      const int x = p[e], y = e ? p[e - 1] : -1;
      bad |= x >= 0 && x < limit && e > 0 && (y < 0 || y >= x);
    }
    ascends = !__any(bad);
    list = (Scalars)(uintptr_t)p;
  }
  __device__ __forceinline__ bool seen(int vis) const {
    return vis > 0 && first < last;
  }
  template <class B, class F>
  __device__ __forceinline__ void each(const ListArgs& a, const Work& wk,
                                       int bytes, F body) const {
    auto read = [&](int e) {
      const int x = list[e];
      if (x < 0 || x >= limit) return Entry{-1, 0};
      if (!ascends) {
        const int32_t* p = (const int32_t*)(uintptr_t)list;
        bool twice = false;
        for (int i = fresh_thread() % kWave; i < e; i += kWave)
          twice |= p[i] == x;
        if (__any(twice)) return Entry{-1, 0};
      }
      return Entry{x, 0};
    };
    each_entry<B>(a.c, wk.b, wk.h, bytes, first, step, last, read,
                  [&](B& x, Entry e, auto kdone, auto vdone) {
                    body(x, e.blk, AllRows(), kdone, vdone);
                  });
  }
};

// The rows of a tile that take a block, as bits of the wave's lanes (scalars: no
// vector instruction goes into them).
struct SomeRows {
  uint64_t mask;
  bool all;
  __device__ __forceinline__ bool whole() const { return all; }
  __device__ __forceinline__ bool lanes() const {
    return __builtin_amdgcn_inverse_ballot_w64(mask);
  }
};

// The blocks of a tile of several tokens, from k_kv4_union.
struct TileList {
  int splits, first, step, last;
  uint32_t full;
  Scalars entry;
  uint64_t saw = 0;
  __device__ __forceinline__ TileList(const ListArgs& a, const Work& wk,
                                      int64_t, int, int wave) {
    splits = a.splits;
    first = wk.split * kWaves + wave;
    step = splits * kWaves;
    const int64_t tile = (wk.b * a.c.heads + wk.h) * a.q_tiles + wk.qt;
    last = ((Scalars)(uintptr_t)a.entries)[tile];
    entry = (Scalars)(uintptr_t)(a.entry + tile * a.span * a.width);
    full = (1u << a.span * a.group) - 1;
  }
  __device__ __forceinline__ bool seen(int vis) const {
    return vis > 0 && __builtin_amdgcn_inverse_ballot_w64(saw);
  }
  template <class B, class F>
  __device__ __forceinline__ void each(const ListArgs& a, const Work& wk,
                                       int bytes, F body) {
    each_entry<B>(a.c, wk.b, wk.h, bytes, first, step, last,
                  [&](int e) {
                    return Entry{entry[2 * e], (uint32_t)entry[2 * e + 1]};
                  },
                  [&](B& x, Entry e, auto kdone, auto vdone) {
                    uint64_t mask = e.rows | e.rows << 16;
                    mask |= mask << 32;
                    saw |= mask;
                    body(x, e.blk, SomeRows{mask, e.rows == full}, kdone, vdone);
                  });
  }
};

template <int D, bool kHalf, class List>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 2 : 4)
void k_kv4_attend_blocks(ListArgs a) {
  __shared__ Lds<kLds16<D>> lds;
  const Work wk = work_of(a);
  if (!wk.any) return;
  const int64_t len = kv_len_of(a, wk.b), nq = q_len_of(a, wk.b);
  const int row0 = first_row(a, wk.qt), end = end_row(a, wk.qt);
  // the last token sees the most
  const int live = (int)min(nq, a.tokens) * a.group;
  if (live <= row0 || visible(a, len, nq, min(end, live) - 1) == 0) {
    // no queries: what is split is the join's
    if (a.splits == 1) {
      const int n = min(16, end - row0);
      for (int i = threadIdx.x; i < n * (D / 8); i += 64 * kWaves) {
        const int r = row0 + i / (D / 8);
        ((uint4*)(a.out + ((wk.b * a.tokens + r / a.group) * a.q_heads +
                           wk.h * a.group + r % a.group) * D))[i % (D / 8)] =
            uint4{0, 0, 0, 0};
      }
    }
    return;
  }
  attend16<D, kHalf, 16, List>(a, wk, len, nq, row0, end, lds);
}

template <int D, bool kHalf>
__global__ __launch_bounds__(256) void k_kv4_join_blocks(ListArgs a) {
  const int r = blockIdx.x * 4 + (int)(threadIdx.x / kWave);
  if (r >= a.rows) return;
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y, t = r / a.group, g = r % a.group;
  if (visible(a, kv_len_of(a, b), q_len_of(a, b), r) == 0) {
    for (int c = lane_id(); c < D; c += kWave)
      a.out[((b * a.tokens + t) * a.q_heads + h * a.group + g) * D + c] = 0;
    return;
  }
  const int tile = a.tiles > 1 ? t * a.tiles + g / 16 : t / a.span;
  join_splits<D, kHalf>(a, b, h, r, tile, r - first_row(a, tile), 16, a.splits);
}

struct Plan {
  int span, tiles, splits;
  int64_t q_tiles;
  size_t part, entry, bytes;  // of the splits' parts, of the tiles' entries, all
};

size_t round_up(size_t x) { return (x + 255) & ~(size_t)255; }

// Lists are split where there are too few of them for the chip.  With 256 / 512 /
// 1,024 / 2,048 workgroups wanted: 64 x 1 tokens, 64 blocks each, 28 / 27 / 32 / 34 us;
// 4 x 9 with 96 blocks and heads of 256 38 / 32 / 41 / 53; one token with 128 the
// same.  At least 8 / 16 / 32 entries: the one token 12.3 / 12.5 / 14.6, 8 x 1 with 128
// blocks 17.4 / 15.8 / 16.2.
constexpr int64_t kWant = 512;  // workgroups
constexpr int64_t kLeast = 16;   // entries of one

Plan plan_for(const sfx_kv4* c, int64_t batch, int64_t tokens, int64_t q_heads,
              int64_t width) {
  Plan p;
  const int64_t group = q_heads / c->heads;
  p.tiles = (int)((group + 15) / 16);
  p.span = (int)std::min<int64_t>(std::max<int64_t>(1, 16 / group), tokens);
  p.q_tiles = p.tiles > 1 ? tokens * p.tiles : (tokens + p.span - 1) / p.span;
  const int64_t wgs = batch * c->heads * p.q_tiles;
  p.splits = (int)std::max<int64_t>(
      1, std::min<int64_t>({kWant / wgs, p.span * width / kLeast, kMaxSplits}));
  p.part = p.splits == 1 ? 0
                         : round_up((size_t)wgs * p.splits * 16 *
                                    (c->head_dim + kPart) * 4);
  p.entry = p.span == 1 ? 0 : round_up((size_t)wgs * p.span * width * 8);
  p.bytes = p.part + p.entry + (p.span == 1 ? 0 : (size_t)wgs * 4);
  return p;
}

bool shapes_ok(const sfx_kv4* c, int64_t batch, int64_t tokens,
               int64_t q_heads, int64_t width) {
  KvView v;
  return kv_view(c, &v) && batch >= 0 && batch <= 65535 && tokens >= 0 &&
         q_heads > 0 && q_heads % c->heads == 0 && q_heads <= 65535 &&
         tokens <= (int64_t(1) << 24) / (q_heads / c->heads) && width >= 1 &&
         width <= 32768;
}

template <int D, bool kHalf>
int launch(const ListArgs& a, hipStream_t stream) {
  const int64_t items = (a.batch * a.c.heads * a.splits + 7) / 8 * 8;
  // more threads than a grid takes, also of 1,024 a tile
  if (items * a.q_tiles >= (int64_t(1) << 32) / 1024) return SFX_EINVAL;
  const dim3 grid((unsigned)(items * a.q_tiles)), block(64 * kWaves);
  if (a.span == 1) {
    hipLaunchKernelGGL((k_kv4_attend_blocks<D, kHalf, OneList>), grid, block, 0,
                       stream, a);
  } else {
    const dim3 tiles((unsigned)(a.batch * a.c.heads * a.q_tiles));
    const int64_t blocks = a.c.positions / kKvBlock;
    if (blocks <= 512 && tiles.x >= 2048)
      hipLaunchKernelGGL(k_kv4_union<64>, tiles, dim3(64), 0, stream, a);
    else if (blocks <= 2048)
      hipLaunchKernelGGL(k_kv4_union<256>, tiles, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL(k_kv4_union<1024>, tiles, dim3(1024), 0, stream, a);
    hipLaunchKernelGGL((k_kv4_attend_blocks<D, kHalf, TileList>), grid, block,
                       0, stream, a);
  }
  if (a.splits > 1)
    hipLaunchKernelGGL((k_kv4_join_blocks<D, kHalf>),
                       dim3((unsigned)(a.rows + 3) / 4, (unsigned)a.c.heads,
                            (unsigned)a.batch),
                       dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

}  // namespace

}  // namespace sfx

using namespace sfx;

extern "C" size_t sfx_kv4_attend_blocks_workspace_size(
    const sfx_kv4* cache, int64_t batch, int64_t tokens, int64_t q_heads,
    int64_t blocks) {
  if (!shapes_ok(cache, batch, tokens, q_heads, blocks) || batch == 0 ||
      tokens == 0)
    return 0;
  return plan_for(cache, batch, tokens, q_heads, blocks).bytes;
}

extern "C" int sfx_kv4_attend_blocks(
    const sfx_kv4* cache, const sfx_heads* q, int64_t batch, int64_t tokens,
    int64_t q_heads, const int32_t* selected, int64_t blocks,
    const void* kv_len, int32_t kv_len_is64, const void* q_len,
    int32_t q_len_is64, float scale, void* out, void* workspace,
    size_t workspace_bytes, hipStream_t stream) {
  if (!shapes_ok(cache, batch, tokens, q_heads, blocks) || !q)
    return SFX_EINVAL;
  if (batch == 0 || tokens == 0) return 0;
  if (!q->data || !selected || !kv_len || !out || ((uintptr_t)out & 15))
    return SFX_EINVAL;
  const Plan p = plan_for(cache, batch, tokens, q_heads, blocks);
  if (p.bytes > workspace_bytes ||
      (p.bytes && (!workspace || ((uintptr_t)workspace & 15))))
    return SFX_EINVAL;
  ListArgs a;
  kv_view(cache, &a.c);
  a.q = *q;
  a.tokens = tokens;
  a.q_heads = (int)q_heads;
  a.group = (int)(q_heads / cache->heads);
  a.rows = (int)(tokens * a.group);
  a.q_tiles = (int)p.q_tiles;
  a.splits = p.splits;
  a.span = p.span;
  a.tiles = p.tiles;
  a.chunk = 1;
  a.vec = (((uintptr_t)q->data & 15) |
           ((q->stride_b | q->stride_t | q->stride_h) & 7)) == 0;
  a.kv_len = kv_len;
  a.kv64 = kv_len_is64;
  a.q_len = q_len;
  a.q64 = q_len_is64;
  a.scale = scale * 1.44269504088896340736f;
  a.out = (uint16_t*)out;
  a.part = (float*)workspace;
  a.entry = (int2*)((char*)workspace + p.part);
  a.entries = (int32_t*)((char*)workspace + p.part + p.entry);
  a.batch = batch;
  a.selected = selected;
  a.width = (int)blocks;
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
