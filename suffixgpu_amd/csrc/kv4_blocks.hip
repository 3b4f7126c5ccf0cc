// Attention over selected blocks of the 4-bit cache.  The mathematics is in
// kv4_attend.h: a workgroup takes a query token's heads of one KV head (16 rows of
// the matrix instruction, of which the group's are queries) over its list of
// blocks, or over a part of the list.

#include <algorithm>

#include "kv4_attend.h"
#include "launch.h"

namespace sfx {

namespace {

struct ListArgs : AttendArgs {
  const int32_t* selected;  // [batch, tokens, heads, width]
  int width;
  int per;    // entries of a split
  int tiles;  // of 16 query heads
};

// Entries wave, wave + kWaves, ... of a split.
struct ListBlocks {
  int splits, first, last, limit;
  const int32_t* list;
  __device__ __forceinline__ ListBlocks(const ListArgs& a, const Work& wk,
                                        int64_t, int most, int wave) {
    splits = a.splits;
    first = wk.split * a.per + wave;
    last = min(wk.split * a.per + a.per, a.width);
    limit = (most + kKvBlock - 1) / kKvBlock;
    list = a.selected +
           ((wk.b * a.tokens + wk.qt / a.tiles) * a.c.heads + wk.h) * a.width;
  }
  __device__ __forceinline__ bool seen(int vis) const {
    return vis > 0 && first < last;
  }
  // As each_block, with 64 entries at a time in the wave's lanes: their places in
  // the pool are looked up at once, entries without a block left out.
  template <class B, class F>
  __device__ __forceinline__ void each(const ListArgs& a, const Work& wk,
                                       int bytes, F body) const {
    for (int e0 = first; e0 < last; e0 += kWaves * kWave) {
      const int e = e0 + lane_id() * kWaves;
      const int blk = e < last ? list[e] : -1;
      int64_t at64 = -1;
      if (blk >= 0 && blk < limit) at64 = kv_place(a.c, wk.b, wk.h, blk);
      uint64_t todo = ballot(at64 >= 0);
      if (!todo) continue;
      // in 32 bits: a pool of 2^32 blocks would be 9 TB
      const uint32_t at = (uint32_t)at64;
      auto place = [&](int i) {
        return a.c.pages +
               (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at, i) * bytes;
      };
      B x;
      int i = __builtin_ctzll(todo);
      x.load_k(place(i));
      x.load_v(place(i));
      while (true) {
        todo &= todo - 1;
        // (after the last one: itself again)
        const int j = todo ? __builtin_ctzll(todo) : i;
        const char* next = place(j);
        body(x, __builtin_amdgcn_readlane(blk, i), [&]() { x.load_k(next); },
             [&]() { x.load_v(next); });
        if (!todo) break;
        i = j;
      }
    }
  }
};

template <int D, bool kHalf>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 2 : 4)
void k_kv4_attend_blocks(ListArgs a) {
  __shared__ Lds<kLds16<D>> lds;
  const Work wk = work_of(a);
  if (!wk.any) return;
  const int64_t len = kv_len_of(a, wk.b), nq = q_len_of(a, wk.b);
  const int t = wk.qt / a.tiles;
  const int row0 = t * a.group + wk.qt % a.tiles * 16, end = (t + 1) * a.group;
  if (visible(a, len, nq, row0) == 0) {
    // no query: what is split is the join's
    if (a.splits == 1) {
      uint4* out = (uint4*)(a.out + ((wk.b * a.tokens + t) * a.q_heads +
                                     wk.h * a.group + row0 - t * a.group) * D);
      const int n = min(16, end - row0) * (D / 8);
      for (int i = threadIdx.x; i < n; i += 64 * kWaves)
        out[i] = uint4{0, 0, 0, 0};
    }
    return;
  }
  attend16<D, kHalf, 16, ListBlocks>(a, wk, len, nq, row0, end, lds);
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
  join_splits<D, kHalf>(a, b, h, r, t * a.tiles + g / 16, g % 16, 16, a.splits);
}

struct Plan {
  int tiles, per, splits;
  int64_t q_tiles;
  size_t bytes;
};

// A list is split where there are too few of them for the chip.
constexpr int64_t kWant = 1024;  // workgroups
constexpr int64_t kLeast = 16;   // entries of one

Plan plan_for(const sfx_kv4* c, int64_t batch, int64_t tokens, int64_t q_heads,
              int64_t width) {
  Plan p;
  p.tiles = (int)((q_heads / c->heads + 15) / 16);
  p.q_tiles = tokens * p.tiles;
  const int64_t wgs = batch * c->heads * p.q_tiles;
  const int64_t per =
      std::max<int64_t>({kLeast, (wgs * width + kWant - 1) / kWant,
                         (width + kMaxSplits - 1) / kMaxSplits});
  p.per = (int)std::min(per, width);
  p.splits = (int)((width + p.per - 1) / p.per);
  p.bytes = p.splits == 1 ? 0
                          : (size_t)wgs * p.splits * 16 *
                                (c->head_dim + kPart) * 4;
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
  if (items * a.q_tiles >= (int64_t(1) << 32) / (64 * kWaves))
    return SFX_EINVAL;  // more threads than a grid takes
  hipLaunchKernelGGL((k_kv4_attend_blocks<D, kHalf>),
                     dim3((unsigned)(items * a.q_tiles)), dim3(64 * kWaves), 0,
                     stream, a);
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
  a.per = p.per;
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
