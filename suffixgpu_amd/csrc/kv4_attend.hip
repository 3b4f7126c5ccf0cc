// Attention of a few new tokens, or of a prompt's chunk, over the 4-bit cache.
//
// Rows of a KV head's queries r = token * group + head are the columns of
// S^T = K Q^T (16 rows a tile) and of O^T = V^T P^T.  A wave takes blocks of 32
// tokens: keys become 16-bit operands by the conversion that applies their
// scale, the product leaves 8 scores of one row in each lane, and those lanes'
// exponentials are at once the operand of the second product (kv4.h).
//
// With s_t the scale of token t's values, x_t its score in base 2 and
// y_t = x_t + log2 s_t, a wave keeps an M near max y_t and sums
//   O = sum 2^(y_t - M) v_t (v_t as the 4 bits stand),  l = sum 2^(y_t - M) / s_t
// so the weights stay within 16-bit range whatever the scales are, and O / l is
// the result.  M is the maximum less kLift and only follows it when that has
// grown by more than 8, so most blocks rescale nothing and no maximum crosses
// lanes (followed at once, 64 x 17 tokens over up to 8,192 take 168 us instead of
// 156, a prompt's 2,048 after 14,336 others 644 instead of 604; with single tokens
// it is the same).  The largest weight is then between 2^7 and 2^15, of float16's
// 2^16, and what is rounded to steps of 2^-24 is below 2^-21 of it: however many
// tokens weigh little beside a heavy one, O has what l counts.
// A term of l is 2^(x_t - M), and where s_t is far below the scale that M comes
// from, 2^(y_t - M) vanishes before 1 / s_t can bring it back: a token of zeros
// beside one of large values would not count.  What vanishes is less than
// 2^-126 / s_t a token.  A wave one of whose l is not 2^28 times the largest of
// that (or so small that it is not a normal number) goes through its keys once
// more, for l alone, relative to the maximum of x_t (ml); O is what it is.
// Values of zero beside others of up to 2^7 do not come to that.
// Weights are rounded to float16 (11 bits, the finer of the 16-bit types, also
// where the cache is bfloat16): the products accumulate in 32 bits, l is summed
// from the unrounded weights.

#include <algorithm>

#include "kv4.h"
#include "launch.h"

namespace sfx {

namespace {

typedef float F4 __attribute__((ext_vector_type(4)));
typedef float F16 __attribute__((ext_vector_type(16)));
typedef _Float16 H2 __attribute__((ext_vector_type(2)));
typedef _Float16 H8 __attribute__((ext_vector_type(8)));
typedef __bf16 B2 __attribute__((ext_vector_type(2)));
typedef __bf16 B8 __attribute__((ext_vector_type(8)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();
constexpr float kLift = 7.0f;   // the largest weight is at least 2^kLift
constexpr float kSlack = 15.0f;  // and at most 2^kSlack
constexpr int kWaves = 4;
constexpr int kPart = 4;  // floats before the channels of a split's part

struct AttendArgs {
  KvView c;
  sfx_heads q;
  int64_t tokens;
  int group;       // query heads per KV head
  int q_heads;
  int rows;        // tokens * group
  int q_tiles;     // row groups of a workgroup
  int splits;      // of the longest row that the table can hold
  int chunk;       // blocks of a split
  int64_t batch;
  int vec;
  const void* kv_len;
  const void* q_len;
  int kv64, q64;
  float scale;     // times log2(e)
  uint16_t* out;
  float* part;     // [batch, heads, q_tiles, splits, rows of a group,
                   //  kPart + D]: M, l, what l is relative to, and O
};

// Eight 4-bit values of a word as 16-bit ones, times `scale` (a power of two,
// of which the conversion takes the exponent).
template <bool kHalf>
__device__ __forceinline__ U4 widen(uint32_t w, float scale) {
  U4 r;
  if (kHalf) {
    r.x = __builtin_bit_cast(uint32_t,
                             __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0));
    r.y = __builtin_bit_cast(uint32_t,
                             __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1));
    r.z = __builtin_bit_cast(uint32_t,
                             __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2));
    r.w = __builtin_bit_cast(uint32_t,
                             __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3));
  } else {
    r.x = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r.y = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    r.z = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    r.w = __builtin_bit_cast(
        uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
  }
  return r;
}

template <bool kHalf>
__device__ __forceinline__ F16 mma32(U4 a, U4 b, F16 c) {
  if (kHalf)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(
        __builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
      __builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0);
}

template <bool kHalf>
__device__ __forceinline__ F4 mma16(U4 a, U4 b, F4 c) {
  if (kHalf)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(
        __builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(B8, a), __builtin_bit_cast(B8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  H2 h;
  h[0] = (_Float16)a;
  h[1] = (_Float16)b;
  return __builtin_bit_cast(uint32_t, h);
}

// Both forms of the kernel keep, per query row (a lane's column), M, l and O,
// and take a block in the same steps; they differ in the matrix instruction.
// kTile = 16: 16x16x32, a lane holds 8 tokens' scores of a row, four lanes
// share it.  kTile = 32: 32x32x16, 16 tokens' scores, two lanes share a row.

// A block of the cache as a lane holds it.
// kTile = 16: row i = lane % 16 of score tile a is token 16 (i / 8) + 8 a +
// i % 8, which makes result row 4 quad + r of tile a the (4 a + r)-th token of
// the lane's words of values.
// kTile = 32: row lane % 32 is that token; result row 8 (r / 4) + 4 (lane / 32)
// + r % 4 is token r % 8 of the lane's word of step r / 8.
template <int D, int kTile>
struct Block;

// A lane's place in a block is a register, what is the same for all lanes an
// immediate of the load.
template <int D>
struct Block<D, 16> {
  uint32_t k[2][D / 32];  // 8 channels a word
  uint32_t ks[2];         // scale bytes of the lane's channels
  uint32_t v[D / 16];     // a word of tokens for each 16 channels
  float vs;               // scale of token lane % 32's values
  uint32_t at_k, at_ks, at_v, at_vs;

  using L = KvLayout<D>;
  __device__ __forceinline__ Block() {
    const int lane = lane_id(), i = lane % 16, quad = lane / 16;
    const int t = 16 * (i / 8) + i % 8;
    at_k = t * (D / 2) + quad * (D / 8);
    at_ks = t * (D / 32) + (D == 256 ? 2 * quad : (D == 64 ? quad / 2 : quad));
    at_v = lane * 16;
    at_vs = lane % 32 * 4;
  }
  __device__ __forceinline__ void load_k(const char* base) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const char* p = base + at_k + 8 * a * (D / 2);
      if (D == 64) {
        const uint2 w = *(const uint2*)p;
        k[a][0] = w.x;
        k[a][1] = w.y;
      } else {
#pragma unroll
        for (int u = 0; u < D / 128; ++u) {
          const uint4 w = ((const uint4*)p)[u];
          k[a][4 * u] = w.x;
          k[a][4 * u + 1] = w.y;
          k[a][4 * u + 2] = w.z;
          k[a][4 * u + 3] = w.w;
        }
      }
      const char* s = base + at_ks + (L::kScale + 8 * a * (D / 32));
      ks[a] = D == 256 ? *(const uint16_t*)s : *(const uint8_t*)s;
    }
    vs = *(const float*)(base + at_vs + L::kVScale);
  }
  __device__ __forceinline__ void load_v(const char* base) {
#pragma unroll
    for (int g = 0; g < D / 64; ++g) {
      const uint4 w =
          *(const uint4*)(base + at_v + (L::kValue + g * 64 * 16));
      v[4 * g] = w.x;
      v[4 * g + 1] = w.y;
      v[4 * g + 2] = w.z;
      v[4 * g + 3] = w.w;
    }
  }
  // Scale of the channels of matrix step i in tile a.  The conversion takes
  // its exponent alone, all ones is a NaN.
  __device__ __forceinline__ float scale(int a, int i) const {
    uint32_t b = ks[a];
    if (D == 256) b = i < D / 64 ? b & 255u : b >> 8;
    return __uint_as_float(b << 23);
  }
};

template <int D>
struct Block<D, 32> {
  uint32_t k[D / 16];
  uint32_t ks;
  uint32_t v[2][D / 32];  // by step of 16 tokens, then 16 channels
  float vs;
  uint32_t at_k, at_ks, at_v, at_vs;

  using L = KvLayout<D>;
  __device__ __forceinline__ Block() {
    const int lane = lane_id(), t = lane % 32, h = lane / 32;
    at_k = t * (D / 2) + h * (D / 4);
    at_ks = t * (D / 32) + h * (D / 64);
    at_v = (h * 16 + lane % 16) * 16 + lane / 16 % 2 * 8;
    at_vs = t * 4;
  }
  __device__ __forceinline__ void load_k(const char* base) {
    const uint4* p = (const uint4*)(base + at_k);
#pragma unroll
    for (int u = 0; u < D / 64; ++u) {
      const uint4 w = p[u];
      k[4 * u] = w.x;
      k[4 * u + 1] = w.y;
      k[4 * u + 2] = w.z;
      k[4 * u + 3] = w.w;
    }
    const char* s = base + at_ks + L::kScale;
    ks = D == 64 ? *(const uint8_t*)s
                 : (D == 128 ? *(const uint16_t*)s : *(const uint32_t*)s);
    vs = *(const float*)(base + at_vs + L::kVScale);
  }
  __device__ __forceinline__ void load_v(const char* base) {
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
      for (int g = 0; g < D / 64; ++g) {
        const uint2 w = *(const uint2*)(base + at_v +
                                        (L::kValue + (g * 4 + 2 * s2) * 256));
        v[s2][2 * g] = w.x;
        v[s2][2 * g + 1] = w.y;
      }
  }
  __device__ __forceinline__ float scale(int i) const {
    return __uint_as_float((ks >> (8 * (i / 4)) & 255u) << 23);
  }
};

// A lane's 8 channels of a query row, as bits.
__device__ __forceinline__ U4 load_q8(const uint16_t* p, bool vec, bool live) {
  U4 r = {0, 0, 0, 0};
  if (!live) return r;
  if (vec) return *(const U4*)p;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    r[u] = (uint32_t)p[2 * u] | (uint32_t)p[2 * u + 1] << 16;
  return r;
}

// What a workgroup works on: rows [row0, row0 + rows of a group) of KV head h
// of batch row b, one split of the row's blocks.  Workgroups go round the eight
// XCDs in turn: those of the same blocks and other query rows follow each other
// on one XCD, whose L2 then holds the blocks.  Splits that only long rows have
// come last, and each split goes through the rows from another one on, so that
// what leaves at once, and rows of one length, spread over XCDs and CUs: with a
// row's splits, or its query rows, beside each other in the same order every
// time, 64 x 12 tokens over up to 8,192 took 165 us instead of 144, 64 x 16 181
// instead of 157, 100 rows of four KV heads over up to 6,000 64 instead of 56.
struct Work {
  int64_t b;
  int h, qt, split;
  bool any;
};

__device__ __forceinline__ Work work_of(const AttendArgs& a) {
  Work w;
  const int id = (int)blockIdx.x;
  const int k = id >> 3;
  const int group = k / a.q_tiles;
  w.qt = (k + group) % a.q_tiles;
  const int64_t item = (int64_t)group * 8 + (id & 7);
  const int64_t rows = a.batch * a.c.heads;
  w.split = (int)(item / rows);
  const int64_t bh = (item + w.split * (rows * 3 / 8)) % rows;
  w.h = (int)(bh % a.c.heads);
  w.b = bh / a.c.heads;
  w.any = w.split < a.splits;
  return w;
}

// Lengths as given, also past the table and past the queries: where a query
// stands is their difference.
__device__ __forceinline__ int64_t kv_len_of(const AttendArgs& a, int64_t b) {
  const int64_t n = load_count(a.kv_len, a.kv64, b);
  return n < 0 ? 0 : n;
}

__device__ __forceinline__ int64_t q_len_of(const AttendArgs& a, int64_t b) {
  if (!a.q_len) return a.tokens;
  const int64_t n = load_count(a.q_len, a.q64, b);
  return n < 0 ? 0 : n;
}

// Positions of the table that row r sees; 0: none.
__device__ __forceinline__ int visible(const AttendArgs& a, int64_t len,
                                       int64_t nq, int r) {
  const int t = r / a.group;
  if (r >= a.rows || t >= nq) return 0;
  const int64_t v = len - nq + t + 1;  // at most len
  return v > a.c.positions ? (int)a.c.positions : (v > 0 ? (int)v : 0);
}

// Blocks of the table that a row holds.
__device__ __forceinline__ int blocks_of(const AttendArgs& a, int64_t len) {
  if (len > a.c.positions) len = a.c.positions;
  return (int)((len + kKvBlock - 1) / kKvBlock);
}

// Splits of a row, and the blocks of one that rows of up to `most` visible
// positions need.  A row is split into equal parts of at most `chunk` blocks,
// which is one number for the call: from its rows, tiles and table width
// (plan_for).  So the order of a row's sums, and its last bits, follow the call's
// shape, but not what the other rows hold.
struct Range {
  int splits, first, last;
};

__device__ __forceinline__ int splits_of(const AttendArgs& a, int64_t len) {
  const int blocks = blocks_of(a, len);
  return max(1, (blocks + a.chunk - 1) / a.chunk);
}

__device__ __forceinline__ Range range_of(const AttendArgs& a, int64_t len,
                                          int most, int split) {
  const int blocks = blocks_of(a, len);
  Range r;
  r.splits = splits_of(a, len);
  const int per = (blocks + r.splits - 1) / r.splits;
  r.first = split * per;
  r.last = min((most + kKvBlock - 1) / kKvBlock, r.first + per);
  return r;
}

__device__ __forceinline__ const uint16_t* q_row(const AttendArgs& a,
                                                 int64_t b, int h, int r) {
  return (const uint16_t*)a.q.data + b * a.q.stride_b +
         (int64_t)(r / a.group) * a.q.stride_t +
         (int64_t)(h * a.group + r % a.group) * a.q.stride_h;
}

// Scale of a block's values in base 2, and kUnit over it (l is summed that much
// smaller, so that no sum overflows), of the tokens that a lane's scores belong
// to: each lane works out one token's, and they cross in the wave's own 64 floats
// of LDS, in order as its accesses are.
// kUnit / s is finite whatever the scale: a row that does not see a token (of a
// NaN, or past the end, where a block holds anything) multiplies it by zero, and
// one that sees a NaN has it from the logarithm.
// *most: the largest kUnit / s of the block's first `held` tokens.
constexpr float kUnit = 0x1p-24f;
constexpr float kUnitLog2 = -24.0f;

__device__ __forceinline__ void share_scales(float vs, int held, float* lds,
                                             float* most) {
  const int t = lane_id() % 32;
  const float inv = __builtin_amdgcn_rcpf(vs) * kUnit;
  if (t < held) *most = fmaxf(*most, inv);
  const float x = lane_id() < 32 ? __builtin_amdgcn_logf(vs)
                                 : fminf(fmaxf(inv, 0.0f), 0x1p77f);
  lds[lane_id() / 32 * 32 + t] = x;
  asm volatile("" ::: "memory");
}

// Largest of a wave's values.
template <int kCtrl, int kRows>
__device__ __forceinline__ float max_step(float v) {
  const int x = __builtin_bit_cast(int, v);
  return fmaxf(v, __builtin_bit_cast(
                      float, __builtin_amdgcn_update_dpp(x, x, kCtrl, kRows,
                                                         0xf, false)));
}
__device__ __forceinline__ float wave_most(float v) {
  v = max_step<0x111, 0xf>(v);
  v = max_step<0x112, 0xf>(v);
  v = max_step<0x114, 0xf>(v);
  v = max_step<0x118, 0xf>(v);
  v = max_step<0x142, 0xa>(v);
  v = max_step<0x143, 0xc>(v);
  return __builtin_bit_cast(
      float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Whether terms that vanished could be missing in the sum l of a row that sees
// a token of the wave; inv: the wave's share of `most` above.
__device__ __forceinline__ bool short_of(float l, bool sees, float inv) {
  const float least = fmaxf(wave_most(inv) * 0x1p-98f, 0x1p-110f);
  return __any(sees && l < least);
}

// Goes through blocks first, first + kWaves, ... below last of row b and KV head
// h, by one wave for which all of these are the same: body(block, index, kdone,
// vdone) calls kdone() when it has used the keys and vdone() when it has used
// the values, which load the next block's into the same registers.  A second
// set for the loads under way would cost a wave in three; issued this early
// they are as well hidden.  A block's page id is read (as a scalar) one block
// ahead of that.  Blocks without a page are left out.
template <class B, class F>
__device__ __forceinline__ void each_block(const KvView& c, int64_t b, int h,
                                           int bytes, int first, int last,
                                           F body) {
  if (first >= last || c.num_pages == 0) return;
  typedef const __attribute__((address_space(4))) int32_t* Ids;
  const Ids ids = (Ids)(uintptr_t)(c.table + b * c.table_stride);
  const int in_page = (1 << c.page_shift) - 1;
  auto page = [&](int blk) { return ids[min(blk, last - 1) >> c.page_shift]; };
  auto good = [&](int32_t id) { return id >= 0 && id < c.num_pages; };
  // past the last block, and without a page: memory that is there
  auto at = [&](int32_t id, int blk) {
    return good(id) ? c.pages + ((((int64_t)id * c.heads + h) << c.page_shift) +
                                 (blk & in_page)) * bytes
                    : c.pages;
  };
  B x;
  int32_t id = page(first), id1 = page(first + kWaves);
  x.load_k(at(id, first));
  x.load_v(at(id, first));
  for (int blk = first; blk < last; blk += kWaves) {
    const char* next = at(id1, blk + kWaves);
    const int32_t id2 = page(blk + 2 * kWaves);
    if (good(id)) {
      body(x, blk, [&]() { x.load_k(next); }, [&]() { x.load_v(next); });
    } else {
      x.load_k(next);
      x.load_v(next);
    }
    id = id1;
    id1 = id2;
  }
}

// Follows the maximum of a row's scores: *m becomes at least that less kLift, O
// and l shrink by the square of the factor returned, l in two steps, as it may
// be far from one.  kLanes: distance of the lanes that share a row.
template <int kLanes>
__device__ __forceinline__ float follow(float top, float* m) {
  if (kLanes == 16) top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  const float mn = fmaxf(*m, top - kLift);
  const float f = mn == *m ? 1.0f : __builtin_amdgcn_exp2f(0.5f * (*m - mn));
  *m = mn;
  return f;
}

// Adds a lane's N weights of a block to l = sum 2^(x - ml): x(j, less) is the
// j-th score in base 2 less `less`, -inf where the row does not see it.
template <int kLanes, int N, class F>
__device__ __forceinline__ void sum_apart(F x, float* ml, float* l) {
  float top = kNegInf;
#pragma unroll
  for (int j = 0; j < N; ++j) top = fmaxf(top, x(j, 0.0f));
  if (__any(top > *ml + kSlack)) {
    const float f = follow<kLanes>(top, ml);
    *l = *l * f * f;
  }
  const float less = *ml == kNegInf ? 0.0f : *ml;
#pragma unroll
  for (int j = 0; j < N; ++j) *l += __builtin_amdgcn_exp2f(x(j, less));
}

// M, l and what l is relative to.
struct Sums {
  float m, l, ml;
};

// What a result's channels are O times: 2^(M - ml) / l, by halves of the power,
// which may be larger than a float where the result is not.
struct Factor {
  float inv, half;
  __device__ __forceinline__ Factor(const Sums& s) {
    half = __builtin_amdgcn_exp2f(0.5f * (s.m - s.ml));
    inv = half / s.l;
  }
  __device__ __forceinline__ float operator()(float o) const {
    return o * inv * half;
  }
};

// Joins the waves' sums of a row; f: the factors of their O.
template <class S>
__device__ __forceinline__ Sums join_waves(const S& lds, int row,
                                           float (&f)[kWaves]) {
  Sums r = {kNegInf, 0.0f, kNegInf};
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    r.m = fmaxf(r.m, lds.m[w][row]);
    r.ml = fmaxf(r.ml, lds.ml[w][row]);
  }
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float m = lds.m[w][row], ml = lds.ml[w][row];
    f[w] = m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(m - r.m);
    const float fl = ml == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ml - r.ml);
    r.l = __builtin_fmaf(fl, lds.l[w][row], r.l);
  }
  return r;
}

// Writes a row's joined channels c0 .. c0 + N of the workgroup's waves: to the
// result, or to this split's part.  x: the sum O.
template <bool kHalf, int N>
__device__ __forceinline__ void put_row(const AttendArgs& a, const Work& w,
                                        int d, int rows_tile, int row, int r,
                                        bool see, const Sums& sums, int c0,
                                        const float (&x)[N], int splits) {
  if (r >= a.rows) return;
  if (splits == 1) {
    const Factor by(sums);
    uint32_t* out = (uint32_t*)(a.out + ((w.b * a.tokens + r / a.group) *
                                             a.q_heads +
                                         w.h * a.group + r % a.group) * d + c0);
#pragma unroll
    for (int c = 0; c < N; c += 2)
      out[c / 2] = see ? from_float16b<kHalf>(by(x[c])) |
                             from_float16b<kHalf>(by(x[c + 1])) << 16
                       : 0u;
  } else {
    float* p = a.part + ((((w.b * a.c.heads + w.h) * a.q_tiles + w.qt) *
                              a.splits + w.split) * rows_tile + row) * (d + kPart);
    // Rows that are no queries may have met a NaN that none of theirs sees: the
    // join takes an l of NaN for a query's.
    if (c0 == 0) {
      p[0] = see ? sums.m : kNegInf;
      p[1] = see ? sums.l : 0.0f;
      p[2] = see ? sums.ml : kNegInf;
    }
    if (!see) return;
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      typedef float F2 __attribute__((ext_vector_type(2)));
      *(F2*)(p + kPart + c0 + c) = F2{x[c], x[c + 1]};
    }
  }
}

// LDS of a workgroup: the waves' sums where they are joined (or, before, the
// queries), and what goes with them.
template <int kBytes>
struct Lds {
  __align__(16) char pool[kBytes];
  float m[kWaves][32], l[kWaves][32], ml[kWaves][32];
  float scales[kWaves][64];
};

template <int D>
constexpr int kLds16 = kWaves * 16 * (D + 4) * 4;
template <int D>
constexpr int kLds32 = kWaves * 32 * (64 + 4) * 4 > 32 * D * 2
                           ? kWaves * 32 * (64 + 4) * 4
                           : 32 * D * 2;

// 16 query rows from row0 on; rows 16 .. kTileRows of the workgroup's tile are
// no queries.
template <int D, bool kHalf, int kTileRows, class S>
__device__ __forceinline__ void attend16(const AttendArgs& a, const Work& wk,
                                         int64_t len, int64_t nq, int row0,
                                         S& lds) {
  constexpr int kStep = D / 32;   // matrix instructions a score tile
  constexpr int kDt = D / 16;     // channel tiles
  const int lane = lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane % 16, quad = lane / 16;
  static_assert(sizeof(lds.pool) >= kLds16<D>, "LDS");
  auto so = (float(*)[16][D + 4])lds.pool;
  auto& sm = lds.m;
  auto& sl = lds.l;
  auto& sc = lds.scales;
  const int vis = visible(a, len, nq, row0 + col);
  U4 qf[kStep];
  {
    const uint16_t* p =
        q_row(a, wk.b, wk.h, vis ? row0 + col : 0) + quad * (D / 4);
#pragma unroll
    for (int i = 0; i < kStep; ++i) qf[i] = load_q8(p + 8 * i, a.vec, vis > 0);
  }
  int most = vis, least = vis ? vis : 0x7fffffff;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    most = max(most, __shfl_xor(most, o));
    least = min(least, __shfl_xor(least, o));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);
  const Range rg = range_of(a, len, most, wk.split);
  const int first = rg.first + wave, last = rg.last;

  float m = kNegInf, l = 0.0f, inv = 0.0f;
  F4 o[kDt];
#pragma unroll
  for (int d = 0; d < kDt; ++d) o[d] = F4{0, 0, 0, 0};

  each_block<Block<D, 16>>(a.c, wk.b, wk.h, KvLayout<D>::kBytes, first, last,
                           [&](Block<D, 16>& kb, int blk, auto kdone,
                               auto vdone) {
    share_scales(kb.vs, most - blk * kKvBlock, sc[wave], &inv);
    const int p0 = blk * kKvBlock + 16 * (quad / 2) + 4 * (quad % 2);
    const bool edge = blk * kKvBlock + kKvBlock > least;
    F4 s[2] = {F4{0, 0, 0, 0}, F4{0, 0, 0, 0}};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < kStep; ++i)
        s[t] = mma16<kHalf>(widen<kHalf>(kb.k[t][i], kb.scale(t, i)), qf[i],
                            s[t]);
    kdone();
    F4 ls[2], rs[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int at = 16 * (quad / 2) + 4 * (quad % 2) + 8 * t;
      ls[t] = *(const F4*)&sc[wave][at];
      rs[t] = *(const F4*)&sc[wave][32 + at];
    }
    float y[8];
    float top = kNegInf;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      y[j] = __builtin_fmaf(s[j / 4][j % 4], a.scale, ls[j / 4][j % 4]);
    }
    if (edge) {
      asm volatile("");  // a branch: most blocks have no edge
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (p0 + 8 * (j / 4) + j % 4 >= vis) y[j] = kNegInf;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, y[j]);
    if (__any(top > m + kSlack)) {
      const float f = follow<16>(top, &m);
      l = l * f * f;
#pragma unroll
      for (int d = 0; d < kDt; ++d) o[d] *= f * f;
    }
    const float mu = m == kNegInf ? 0.0f : m;
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      w[j] = __builtin_amdgcn_exp2f(y[j] - mu);
      l = __builtin_fmaf(w[j], rs[j / 4][j % 4], l);
    }
    const U4 pf = {pack_half(w[0], w[1]), pack_half(w[2], w[3]),
                   pack_half(w[4], w[5]), pack_half(w[6], w[7])};
#pragma unroll
    for (int d = 0; d < kDt; ++d)
      o[d] = mma16<true>(widen<true>(kb.v[d], 1.0f), pf, o[d]);
    vdone();
  });

  // The lanes of a row have their own sums until here.
  auto row_sum = [](float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
  };
  l = row_sum(l);
  float ml = m - kUnitLog2;
  if (short_of(l, vis > first * kKvBlock, inv)) {
    float lx = 0.0f;
    ml = kNegInf;
    each_block<Block<D, 16>>(a.c, wk.b, wk.h, KvLayout<D>::kBytes, first, last,
                             [&](Block<D, 16>& kb, int blk, auto kdone, auto) {
      const int p0 = blk * kKvBlock + 16 * (quad / 2) + 4 * (quad % 2);
      F4 s[2] = {F4{0, 0, 0, 0}, F4{0, 0, 0, 0}};
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < kStep; ++i)
          s[t] = mma16<kHalf>(widen<kHalf>(kb.k[t][i], kb.scale(t, i)), qf[i],
                              s[t]);
      kdone();
      sum_apart<16, 8>([&](int j, float less) {
        return p0 + 8 * (j / 4) + j % 4 < vis
                   ? __builtin_fmaf(s[j / 4][j % 4], a.scale, -less)
                   : kNegInf;
      }, &ml, &lx);
    });
    lx = row_sum(lx);
    l = l == l ? lx : l;  // a value's NaN stays
  }

  // Join the waves in LDS; 16 threads a row, D / 16 channels each.
#pragma unroll
  for (int d = 0; d < kDt; ++d) *(F4*)&so[wave][col][d * 16 + quad * 4] = o[d];
  if (quad == 0) {
    sm[wave][col] = m;
    sl[wave][col] = l;
    lds.ml[wave][col] = ml;
  }
  __syncthreads();
  const int row = threadIdx.x / 16, c0 = threadIdx.x % 16 * (D / 16);
  float f[kWaves];
  const Sums sums = join_waves(lds, row, f);
  float x[D / 16];
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    x[c] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      x[c] = __builtin_fmaf(f[w], so[w][row][c0 + c], x[c]);
  }
  const bool see = visible(a, len, nq, row0 + row) > 0 && sums.l != 0.0f;
  put_row<kHalf>(a, wk, D, kTileRows, row, row0 + row, see, sums, c0, x,
                 rg.splits);
  if (kTileRows > 16)
    put_row<kHalf>(a, wk, D, kTileRows, row + 16, row0 + row + 16, false, sums,
                   c0, x, rg.splits);
}

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
  attend16<D, kHalf, 16>(a, wk, len, q_len_of(a, wk.b), wk.qt * 16, lds);
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
    attend16<D <= 128 ? D : 128, kHalf, 32>(a, wk, len, nq, row0, lds);
  else
    attend32<D, kHalf>(a, wk, len, nq, row0, lds);
}

// Joins the splits of query rows: a wave per row and KV head.  A lane holds a
// split's M and l, then D / 64 channels.
constexpr int kMaxSplits = 64;

template <int D, bool kHalf>
__global__ __launch_bounds__(256) void k_kv4_join(AttendArgs a,
                                                  int rows_tile) {
  constexpr int C = D / 64;
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  const int r = blockIdx.x * 4 + (int)(threadIdx.x / kWave);
  const int lane = lane_id();
  const int splits = splits_of(a, kv_len_of(a, b));
  if (splits == 1 || r >= a.rows) return;
  const float* p =
      a.part + (((b * a.c.heads + h) * a.q_tiles + r / rows_tile) * a.splits *
                    rows_tile + r % rows_tile) * (D + kPart);
  const int64_t next = (int64_t)rows_tile * (D + kPart);
  Sums part = {kNegInf, 0.0f, kNegInf};
  if (lane < splits)
    part = {p[lane * next], p[lane * next + 1], p[lane * next + 2]};
  Sums sums = part;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    sums.m = fmaxf(sums.m, __shfl_xor(sums.m, o));
    sums.ml = fmaxf(sums.ml, __shfl_xor(sums.ml, o));
  }
  const float f =
      part.m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(part.m - sums.m);
  // a query's split of nothing but NaN has no M, and an l that says so
  sums.l = part.l * (part.ml == kNegInf
                         ? 0.0f
                         : __builtin_amdgcn_exp2f(part.ml - sums.ml));
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sums.l += __shfl_xor(sums.l, o);
  float x[C];
#pragma unroll
  for (int c = 0; c < C; ++c) x[c] = 0.0f;
  // parts of factor 0 were not written
  uint64_t todo = ballot(f != 0.0f);
  while (todo) {
    float w[4], v[4][C];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = todo ? __builtin_ctzll(todo) : 0;
      w[u] = todo ? __shfl(f, s) : 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c)
        v[u][c] = todo ? p[s * next + kPart + lane * C + c] : 0.0f;
      todo &= todo - 1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int c = 0; c < C; ++c) x[c] = __builtin_fmaf(w[u], v[u][c], x[c]);
  }
  const int t = r / a.group;
  uint16_t* out = a.out + ((b * a.tokens + t) * a.q_heads + h * a.group +
                           r % a.group) * D + lane * C;
  const Factor by(sums);
#pragma unroll
  for (int c = 0; c < C; ++c)
    out[c] = (uint16_t)from_float16b<kHalf>(sums.l == 0.0f ? 0.0f : by(x[c]));
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
