// Attention of a few new tokens, or of a prompt's chunk, over the 4-bit cache:
// every position that a query sees.  The mathematics is in kv4_attend.h.

#include <algorithm>

#include "kv4_attend.h"
#include "launch.h"

namespace sfx {

namespace {

// 32 query rows from row0 on.  They lie in LDS in the order of the matrix
// instruction's operand; every wave holds O of all of them.
template <int D, bool kHalf, class S>
__device__ __forceinline__ void attend32(const AttendArgs& a, const Work& wk,
                                         int64_t len, int64_t nq, int row0,
                                         S& lds) {
  constexpr int kRows = 32;
  constexpr int kStep = D / 16;
  constexpr int kDt = D / 32;
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane % 32, h2 = lane / 32;
  static_assert(sizeof(lds.pool) >= kLds32<D>, "LDS");
  U4* sq = (U4*)lds.pool;
  auto& sm = lds.m;
  auto& sl = lds.l;
  auto& sc = lds.scales;
  for (int e = threadIdx.x; e < kRows * (D / 8); e += 64 * kWaves) {
    // operand (step, lane): channels (lane / 32) D / 2 + 8 step
    const int i = e / 64, ln = e % 64;
    const int r = row0 + ln % 32;
    const bool live = visible(a, len, nq, r) > 0;
    sq[e] = load_q8(q_row(a, wk.b, wk.h, live ? r : 0) + ln / 32 * (D / 2) +
                        8 * i,
                    a.vec, live);
  }
  const int vis = visible(a, len, nq, row0 + col);
  int most = vis, least = vis ? vis : 0x7fffffff;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    most = max(most, __shfl_xor(most, o));
    least = min(least, __shfl_xor(least, o));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);
  const Range rg = range_of(a, len, most, wk.split);
  const int first = rg.first + wave, last = rg.last;
  __syncthreads();

  float m = kNegInf, l = 0.0f, inv = 0.0f;
  F16 o[kDt];
#pragma unroll
  for (int d = 0; d < kDt; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;

  each_block<Block<D, 32>>(a.c, wk.b, wk.h, KvLayout<D>::kBytes, first, last,
                           [&](Block<D, 32>& kb, int blk, auto kdone,
                               auto vdone) {
    share_scales(kb.vs, most - blk * kKvBlock, sc[wave], &inv);
    const int p0 = blk * kKvBlock + 4 * h2;
    const bool edge = blk * kKvBlock + kKvBlock > least;
    F16 s;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.0f;
    // The queries' operands come from LDS kAhead steps before they are used:
    // the matrix instructions would wait for each.
    constexpr int kAhead = 4;
    U4 qf[kAhead];
    F4 ls[4], rs[4];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) qf[i] = sq[i * 64 + lane];
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      s = mma32<kHalf>(widen<kHalf>(kb.k[i], kb.scale(i)), qf[i % kAhead], s);
      if (i + kAhead < kStep) qf[i % kAhead] = sq[(i + kAhead) * 64 + lane];
      if (i == kStep - 2) {
#pragma unroll
        for (int g = 0; g < 4; ++g)
          ls[g] = *(const F4*)&sc[wave][8 * g + 4 * h2];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = 0; g < 4; ++g)
      rs[g] = *(const F4*)&sc[wave][32 + 8 * g + 4 * h2];
    kdone();
    float top = kNegInf;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      s[r] = __builtin_fmaf(s[r], a.scale, ls[r / 4][r % 4]);
    if (edge) {
      asm volatile("");  // a branch: most blocks have no edge
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (p0 + r / 4 * 8 + r % 4 >= vis) s[r] = kNegInf;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
    if (__any(top > m + kSlack)) {
      const float f = follow<32>(top, &m);
      l = l * f * f;
#pragma unroll
      for (int d = 0; d < kDt; ++d) o[d] *= f * f;
    }
    const float mu = m == kNegInf ? 0.0f : m;
    U4 pf[2];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        w[r] = __builtin_amdgcn_exp2f(s[4 * g + r] - mu);
        l = __builtin_fmaf(w[r], rs[g][r], l);
      }
      pf[g / 2][g % 2 * 2] = pack_half(w[0], w[1]);
      pf[g / 2][g % 2 * 2 + 1] = pack_half(w[2], w[3]);
    }
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int d = 0; d < kDt; ++d)
        o[d] = mma32<true>(widen<true>(kb.v[s2][d], 1.0f), pf[s2], o[d]);
    vdone();
  });

  // The lanes of a row have their own sums until here.
  auto row_sum = [](float x) {
    return x + __shfl_xor(x, 32);
  };
  l = row_sum(l);
  float ml = m - kUnitLog2;
  if (short_of(l, vis > first * kKvBlock, inv)) {
    float lx = 0.0f;
    ml = kNegInf;
    each_block<Block<D, 32>>(a.c, wk.b, wk.h, KvLayout<D>::kBytes, first, last,
                             [&](Block<D, 32>& kb, int blk, auto kdone, auto) {
      const int p0 = blk * kKvBlock + 4 * h2;
      F16 s;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        s = mma32<kHalf>(widen<kHalf>(kb.k[i], kb.scale(i)), sq[i * 64 + lane],
                         s);
      }
      kdone();
      sum_apart<32, 16>([&](int r, float less) {
        return p0 + r / 4 * 8 + r % 4 < vis
                   ? __builtin_fmaf(s[r], a.scale, -less)
                   : kNegInf;
      }, &ml, &lx);
    });
    lx = row_sum(lx);
    l = l == l ? lx : l;  // a value's NaN stays
  }

  // Join the waves in LDS, 64 channels at a time: 8 threads a row.
  auto so = (float(*)[32][64 + 4])lds.pool;
  const int row = threadIdx.x / 8, c0 = threadIdx.x % 8 * 8;
  const bool queried = visible(a, len, nq, row0 + row) > 0;
  float f[kWaves];
  Sums sums;
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        // result rows 8 r + 4 h2 ..: channel tile 2 (r / 2) + t of the 64
        *(F4*)&so[wave][col][(2 * (r / 2) + t) * 16 + r % 2 * 8 + 4 * h2] =
            F4{o[2 * g + t][4 * r], o[2 * g + t][4 * r + 1],
               o[2 * g + t][4 * r + 2], o[2 * g + t][4 * r + 3]};
    if (g == 0 && h2 == 0) {
      sm[wave][col] = m;
      sl[wave][col] = l;
      lds.ml[wave][col] = ml;
    }
    __syncthreads();
    if (g == 0) sums = join_waves(lds, row, f);
    float x[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      x[c] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        x[c] = __builtin_fmaf(f[w], so[w][row][c0 + c], x[c]);
    }
    put_row<kHalf>(a, wk, D, kRows, row, row0 + row,
                   queried && sums.l != 0.0f, sums, 64 * g + c0, x, rg.splits);
  }
}

// Up to 16 query rows a workgroup: single tokens, and small groups of drafts.
// The memory bounds it: 64 single tokens over up to 8,192, 32 query heads on 8 KV
// heads of 128, take 87 us for 422 MB, 4.9 TB/s (as a large copy moves).  Four
// waves a SIMD, 128 registers; and 36 KB of LDS.
template <int D, bool kHalf>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 2 : 4)
void k_kv4_attend16(AttendArgs a) {
  __shared__ Lds<kLds16<D>> lds;
  const Work wk = work_of(a);
  if (!wk.any) return;
  const int64_t len = kv_len_of(a, wk.b);
  if (splits_of(a, len) <= wk.split) return;
  attend16<D, kHalf, 16, SplitBlocks>(a, wk, len, q_len_of(a, wk.b), wk.qt * 16,
                                      a.rows, lds);
}

// 32 query rows a workgroup: verification steps and prompts.  Up to some tens of
// rows the memory bounds it as above (4 x 9 tokens, 16 query heads on 8 KV heads
// of 256, over up to 131,072: 211 us for 1.07 GB, 5.1 TB/s), past that the vector
// instructions: conversions from 4 bits, exponentials and the sums beside them
// issue in 80% of a prompt's cycles, matrix instructions in 48% (2,048 tokens
// after 14,336 others: 582 us, 886 TFLOP/s of the 1,210 that a large matrix
// product reaches).  64 x 17 tokens over up to 8,192 lie between: 148 us for 440
// MB, as three tiles convert each block of a full row anew.  Three waves a SIMD;
// four spill (64 x 17 199 us then).
//
// A tile of at most 16 queries (of 17 tokens with four heads to a KV head, the
// last four rows) takes the narrower instruction, which leaves half as many
// columns idle (64 x 17 145 us, without 157; a prompt 552 and 566); its sums do
// not fit this kernel's LDS for heads of 256.
template <int D, bool kHalf>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? 2 : 3)
void k_kv4_attend32(AttendArgs a) {
  __shared__ Lds<kLds32<D>> lds;
  const Work wk = work_of(a);
  if (!wk.any) return;
  const int64_t len = kv_len_of(a, wk.b);
  if (splits_of(a, len) <= wk.split) return;
  const int64_t nq = q_len_of(a, wk.b);
  const int row0 = wk.qt * 32;
  const int64_t queries = nq < a.tokens ? nq : a.tokens;
  if (D <= 128 && queries * a.group - row0 <= 16)
    attend16<D <= 128 ? D : 128, kHalf, 32, SplitBlocks>(a, wk, len, nq, row0,
                                                         a.rows, lds);
  else
    attend32<D, kHalf>(a, wk, len, nq, row0, lds);
}

// Joins the splits of query rows: a wave per row and KV head.
template <int D, bool kHalf>
__global__ __launch_bounds__(256) void k_kv4_join(AttendArgs a,
                                                  int rows_tile) {
  const int64_t b = blockIdx.z;
  const int r = blockIdx.x * 4 + (int)(threadIdx.x / kWave);
  const int splits = splits_of(a, kv_len_of(a, b));
  if (splits == 1 || r >= a.rows) return;
  join_splits<D, kHalf>(a, b, blockIdx.y, r, r / rows_tile, r % rows_tile,
                        rows_tile, splits);
}

struct Plan {
  int rows_tile;  // query rows of a workgroup
  int q_tiles, splits, chunk;
  size_t bytes;
};

// Query rows by 16 where a KV head has no more than that, else by 32.  Measured
// over up to 8,192 tokens, 64 rows, 8 KV heads of 128, four query heads each:
// single tokens (4 rows a head) and 4 tokens (16) the same either way, 92 and 97
// us, by the smaller kernel; 5 tokens (20) 107 us by 16 and 100 by 32, 17 tokens
// (68) 160 and 149; a prompt's 2,048 tokens after 14,336 others 682 and 570.
//
// Splits: so many that with every row full the launch has about `want`
// workgroups.  More even out rows of different lengths, fewer have less to join.
// By 16, of which four workgroups fit a CU, with 512 / 1,024 / 1,536 / 2,048: the
// 64 x 1 above 91 / 93 / 101 / 94 us, 100 rows of up to 6,000 tokens and four KV
// heads 62 / 56 / 60 / 58.  By 32, of which three fit: 64 x 17 159 / 157 / 149 /
// 150, 16 x 17 over up to 32,768 221 / 167 / 170 / 166.  Heads of 256, two: 4 x 9
// over up to 131,072 198 / 203 / 205 / 215, 30 x 9 over up to 8,192 97 / 101 / 109
// / 113.
// Both of these are for tables about as wide as the rows.  What the rows hold is
// known on the device alone, so the plan takes every row as full: in a table many
// times wider than the rows, they have fewer splits than these figures stand for.
// At least kLeast blocks each: one token over 2,050 10.2 us, with 8 10.7, with 4
// 13.2.
constexpr int64_t kLeast = 16;

Plan plan_for(const sfx_kv4* c, int64_t batch, int64_t tokens,
              int64_t q_heads) {
  Plan p;
  const int64_t rows = tokens * (q_heads / c->heads);
  p.rows_tile = rows <= 16 ? 16 : 32;
  p.q_tiles = (int)((rows + p.rows_tile - 1) / p.rows_tile);
  const int64_t wgs = batch * c->heads * p.q_tiles;
  const int64_t blocks =
      std::max<int64_t>(1, c->table_width * c->page_size / kKvBlock);
  const int64_t want =
      p.rows_tile == 16 || c->head_dim == 256 ? 1024 : 1536;
  const int64_t chunk =
      std::max<int64_t>({kLeast, (wgs * blocks + want - 1) / want,
                         (blocks + kMaxSplits - 1) / kMaxSplits});
  p.chunk = (int)std::min(chunk, blocks);
  p.splits = (int)((blocks + p.chunk - 1) / p.chunk);
  p.bytes = p.splits == 1 ? 0
                          : (size_t)wgs * p.splits * p.rows_tile *
                                (c->head_dim + kPart) * 4;
  return p;
}

template <int D, bool kHalf>
int launch(AttendArgs& a, int rows_tile, hipStream_t stream) {
  const int64_t items = (a.batch * a.c.heads * a.splits + 7) / 8 * 8;
  if (items * a.q_tiles >= (int64_t(1) << 32) / (64 * kWaves))
    return SFX_EINVAL;  // more threads than a grid takes
  const dim3 grid((unsigned)(items * a.q_tiles));
  const dim3 block(64 * kWaves);
  if (rows_tile == 16)
    hipLaunchKernelGGL((k_kv4_attend16<D, kHalf>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((k_kv4_attend32<D, kHalf>), grid, block, 0, stream, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((k_kv4_join<D, kHalf>),
                       dim3((unsigned)(a.rows + 3) / 4, (unsigned)a.c.heads,
                            (unsigned)a.batch),
                       dim3(256), 0, stream, a, rows_tile);
  return (int)hipGetLastError();
}

bool shapes_ok(const sfx_kv4* c, int64_t batch, int64_t tokens,
               int64_t q_heads) {
  KvView v;
  return kv_view(c, &v) && batch >= 0 && batch <= 65535 && tokens >= 0 &&
         q_heads > 0 && q_heads % c->heads == 0 && q_heads <= 65535 &&
         tokens <= (int64_t(1) << 24) / (q_heads / c->heads);
}

}  // namespace

}  // namespace sfx

using namespace sfx;

extern "C" size_t sfx_kv4_attend_workspace_size(const sfx_kv4* cache,
                                                int64_t batch, int64_t tokens,
                                                int64_t q_heads) {
  if (!shapes_ok(cache, batch, tokens, q_heads) || batch == 0 || tokens == 0)
    return 0;
  return plan_for(cache, batch, tokens, q_heads).bytes;
}

extern "C" int sfx_kv4_attend(const sfx_kv4* cache, const sfx_heads* q,
                              int64_t batch, int64_t tokens, int64_t q_heads,
                              const void* kv_len, int32_t kv_len_is64,
                              const void* q_len, int32_t q_len_is64,
                              float scale, void* out, void* workspace,
                              size_t workspace_bytes, hipStream_t stream) {
  if (!shapes_ok(cache, batch, tokens, q_heads) || !q) return SFX_EINVAL;
  if (batch == 0 || tokens == 0) return 0;
  if (!q->data || !kv_len || !out || ((uintptr_t)out & 15)) return SFX_EINVAL;
  const Plan p = plan_for(cache, batch, tokens, q_heads);
  if (p.bytes > workspace_bytes ||
      (p.bytes && (!workspace || ((uintptr_t)workspace & 15))))
    return SFX_EINVAL;
  AttendArgs a;
  kv_view(cache, &a.c);
  a.q = *q;
  a.tokens = tokens;
  a.q_heads = (int)q_heads;
  a.group = (int)(q_heads / cache->heads);
  a.rows = (int)(tokens * a.group);
  a.q_tiles = p.q_tiles;
  a.splits = p.splits;
  a.chunk = p.chunk;
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
  const bool half = cache->dtype == SFX_F16;
  switch (cache->head_dim) {
    case 64:
      return half ? launch<64, true>(a, p.rows_tile, stream)
                  : launch<64, false>(a, p.rows_tile, stream);
    case 128:
      return half ? launch<128, true>(a, p.rows_tile, stream)
                  : launch<128, false>(a, p.rows_tile, stream);
    default:
      return half ? launch<256, true>(a, p.rows_tile, stream)
                  : launch<256, false>(a, p.rows_tile, stream);
  }
}
