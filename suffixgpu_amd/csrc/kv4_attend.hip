// Attention of a few new tokens, or of a prompt's chunk, over the 4-bit cache.
//
// Rows of a KV head's queries r = token * group + head are the columns of
// S^T = K Q^T (16 rows a tile) and of O^T = V^T P^T.  A wave takes blocks of 32
// tokens: keys become 16-bit operands by the conversion that applies their
// scale, the product leaves 8 scores of one row in each lane, and those lanes'
// exponentials are at once the operand of the second product (kv4.h).
//
// With s_t the scale of token t's values, x_t its score in base 2 and
// y_t = x_t + log2 s_t, a wave keeps M >= about max y_t and sums
//   O = sum 2^(y_t - M) v_t (v_t as the 4 bits stand),  l = sum 2^(y_t - M) / s_t
// so the weights stay within 16-bit range whatever the scales are, and O / l is
// the result.  M only follows the maximum when that has grown by more than
// kSlack, so most blocks rescale nothing and no maximum crosses lanes.
// Weights are rounded to float16 (11 bits, the finer of the 16-bit types, also
// where the cache is bfloat16): the products accumulate in 32 bits, l is summed
// from the unrounded weights.

#include <algorithm>

#include "kv4.h"
#include "launch.h"

namespace sfx {

namespace {

typedef float F4 __attribute__((ext_vector_type(4)));
typedef _Float16 H2 __attribute__((ext_vector_type(2)));
typedef _Float16 H8 __attribute__((ext_vector_type(8)));
typedef __bf16 B2 __attribute__((ext_vector_type(2)));
typedef __bf16 B8 __attribute__((ext_vector_type(8)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();
constexpr float kSlack = 8.0f;
constexpr int kWaves = 4;
constexpr int kTile = 16;  // query rows of a matrix instruction

struct AttendArgs {
  KvView c;
  sfx_heads q;
  int64_t tokens;
  int group;       // query heads per KV head
  int q_heads;
  int rows;        // tokens * group
  int q_tiles;     // of 16 * NQ rows
  int splits;
  int vec;
  const void* kv_len;
  const void* q_len;
  int kv64, q64;
  float scale;     // times log2(e)
  uint16_t* out;
  float* part;     // [batch, heads, q_tiles, splits, 16 NQ, D + 2]
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
__device__ __forceinline__ F4 mma(U4 a, U4 b, F4 c) {
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

// A block of the cache as a lane holds it: row i = lane % 16 of tile a is
// token 16 (i / 8) + 8 a + i % 8, which makes result row 4 quad + r of tile a
// the (4 a + r)-th token of the lane's words of values.
template <int D>
struct Block {
  uint32_t k[2][D / 32];  // 8 channels a word
  uint32_t ks[2];         // scale bytes of the lane's channels
  uint32_t v[D / 16];     // a word of tokens for each 16 channels
  float vs[8];
};

template <int D>
__device__ __forceinline__ void load_block(const char* base, Block<D>& b) {
  using L = KvLayout<D>;
  const int lane = lane_id();
  const int i = lane % 16, quad = lane / 16;
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int t = 16 * (i / 8) + 8 * a + i % 8;
    const char* p = base + t * (D / 2) + quad * (D / 8);
    if (D == 64) {
      const uint2 w = *(const uint2*)p;
      b.k[a][0] = w.x;
      b.k[a][1] = w.y;
    } else {
#pragma unroll
      for (int u = 0; u < D / 128; ++u) {
        const uint4 w = ((const uint4*)p)[u];
        b.k[a][4 * u] = w.x;
        b.k[a][4 * u + 1] = w.y;
        b.k[a][4 * u + 2] = w.z;
        b.k[a][4 * u + 3] = w.w;
      }
    }
    const uint8_t* s = (const uint8_t*)(base + L::kScale) + t * (D / 32);
    if (D == 256)
      b.ks[a] = *(const uint16_t*)(s + 2 * quad);
    else
      b.ks[a] = s[D == 64 ? quad / 2 : quad];
  }
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    const uint4 w = *(const uint4*)(base + L::kValue + (g * 64 + lane) * 16);
    b.v[4 * g] = w.x;
    b.v[4 * g + 1] = w.y;
    b.v[4 * g + 2] = w.z;
    b.v[4 * g + 3] = w.w;
  }
  const float* vs = (const float*)(base + L::kVScale) + 16 * (quad / 2) +
                    4 * (quad % 2);
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const float4 w = *(const float4*)(vs + 8 * a);
    b.vs[4 * a] = w.x;
    b.vs[4 * a + 1] = w.y;
    b.vs[4 * a + 2] = w.z;
    b.vs[4 * a + 3] = w.w;
  }
}

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

// One workgroup: a tile of 16 NQ query rows of one KV head and batch row over
// one split of the row's visible blocks, its waves taking every fourth block.
template <int D, bool kHalf, int NQ>
__global__ __launch_bounds__(64 * kWaves) void k_kv4_attend(AttendArgs a) {
  constexpr int kRows = kTile * NQ;
  constexpr int kStep = D / 32;   // matrix instructions a score tile
  constexpr int kDt = D / 16;     // channel tiles
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  const int qt = blockIdx.x / a.splits;
  const int split = blockIdx.x % a.splits;
  const int lane = lane_id();
  const int wave = threadIdx.x / kWave;
  const int col = lane % 16, quad = lane / 16;

  int64_t len = load_count(a.kv_len, a.kv64, b);
  len = len < 0 ? 0 : (len > a.c.positions ? a.c.positions : len);
  int64_t nq = a.q_len ? load_count(a.q_len, a.q64, b) : a.tokens;
  nq = nq < 0 ? 0 : (nq > a.tokens ? a.tokens : nq);

  // Positions that each of the lane's rows sees; 0: none.
  int vis[NQ];
  U4 qf[NQ][kStep];
  int most = 0, least = 0x7fffffff;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = (qt * NQ + n) * kTile + col;
    const int t = r / a.group;
    const int64_t v = len - nq + t + 1;
    vis[n] = (r < a.rows && t < nq && v > 0) ? (int)v : 0;
    const uint16_t* p =
        (const uint16_t*)a.q.data +
        (vis[n] ? b * a.q.stride_b + (int64_t)t * a.q.stride_t +
                      (int64_t)(h * a.group + r % a.group) * a.q.stride_h +
                      quad * (D / 4)
                : 0);
#pragma unroll
    for (int i = 0; i < kStep; ++i)
      qf[n][i] = load_q8(p + 8 * i, a.vec, vis[n] > 0);
    most = max(most, vis[n]);
    if (vis[n]) least = min(least, vis[n]);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    most = max(most, __shfl_xor(most, o));
    least = min(least, __shfl_xor(least, o));
  }
  most = __builtin_amdgcn_readfirstlane(most);
  least = __builtin_amdgcn_readfirstlane(least);

  // This split's blocks.
  const int blocks = (most + kKvBlock - 1) / kKvBlock;
  const int per = (blocks + a.splits - 1) / a.splits;
  const int first = split * per;
  const int last = min(blocks, first + per);

  float m[NQ], l[NQ];
  F4 o[NQ][kDt];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = kNegInf;
    l[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < kDt; ++d) o[n][d] = F4{0, 0, 0, 0};
  }

  for (int blk = first + wave; blk < last; blk += kWaves) {
    const char* base = kv_block<D>(a.c, b, h, blk);
    if (!base) continue;
    Block<D> kb;
    load_block<D>(base, kb);
    const int p0 = blk * kKvBlock + 16 * (quad / 2) + 4 * (quad % 2);
    const bool edge = blk * kKvBlock + kKvBlock > least;
    F4 s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) s[n][0] = s[n][1] = F4{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        uint32_t sb = kb.ks[t];
        if (D == 256) sb = i < kStep / 2 ? sb & 255u : sb >> 8;
        // the conversion takes the exponent alone: 255 is NaN
        const U4 kf = widen<kHalf>(kb.k[t][i], __uint_as_float(sb << 23));
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][t] = mma<kHalf>(kf, qf[n][i], s[n][t]);
      }
    }
    float ls[8], rs[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ls[j] = __builtin_amdgcn_logf(kb.vs[j]);
      // Finite whatever the scale: a row that does not see a token (of a NaN,
      // or past the end, where a block holds anything) multiplies it by zero,
      // and one that sees a NaN has it from ls.
      rs[j] = fminf(fmaxf(__builtin_amdgcn_rcpf(kb.vs[j]), 0.0f), 0x1p101f);
    }
    U4 pf[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float y[8];
      float top = kNegInf;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = __builtin_fmaf(s[n][j / 4][j % 4], a.scale, ls[j]);
        if (edge && p0 + 8 * (j / 4) + j % 4 >= vis[n]) y[j] = kNegInf;
        top = fmaxf(top, y[j]);
      }
      if (__any(top > m[n] + kSlack)) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float mn = fmaxf(m[n], top);
        const float f = mn == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - mn);
        m[n] = mn;
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < kDt; ++d) o[n][d] *= f;
      }
      const float mu = m[n] == kNegInf ? 0.0f : m[n];
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = __builtin_amdgcn_exp2f(y[j] - mu);
        l[n] = __builtin_fmaf(w[j], rs[j], l[n]);
      }
      pf[n] = U4{pack_half(w[0], w[1]), pack_half(w[2], w[3]),
                 pack_half(w[4], w[5]), pack_half(w[6], w[7])};
    }
#pragma unroll
    for (int d = 0; d < kDt; ++d) {
      const U4 vf = widen<true>(kb.v[d], 1.0f);
#pragma unroll
      for (int n = 0; n < NQ; ++n) o[n][d] = mma<true>(vf, pf[n], o[n][d]);
    }
  }

  // Join the waves in LDS, one tile of rows at a time.
  __shared__ float so[kWaves][kTile][D + 4];
  __shared__ float sm[kWaves][kTile], sl[kWaves][kTile];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] += __shfl_xor(l[n], 16);
    l[n] += __shfl_xor(l[n], 32);
    if (n) __syncthreads();
#pragma unroll
    for (int d = 0; d < kDt; ++d)
      *(F4*)&so[wave][col][d * 16 + quad * 4] = o[n][d];
    if (quad == 0) {
      sm[wave][col] = m[n];
      sl[wave][col] = l[n];
    }
    __syncthreads();
    // 16 threads a row, D / 16 channels each
    const int row = threadIdx.x / 16, c0 = threadIdx.x % 16 * (D / 16);
    const int r = (qt * NQ + n) * kTile + row;
    float mx = kNegInf;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, sm[w][row]);
    float f[kWaves], lt = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      f[w] = sm[w][row] == kNegInf
                 ? 0.0f
                 : __builtin_amdgcn_exp2f(sm[w][row] - mx);
      lt = __builtin_fmaf(f[w], sl[w][row], lt);
    }
    float x[D / 16];
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      x[c] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        x[c] = __builtin_fmaf(f[w], so[w][row][c0 + c], x[c]);
    }
    // What a row without visible positions gathered counts for nothing.
    const int t = r / a.group;
    const bool see = r < a.rows && t < nq && len - nq + t + 1 > 0 && lt != 0.0f;
    if (a.splits == 1) {
      if (r < a.rows) {
        const float inv = see ? 1.0f / lt : 0.0f;
        uint32_t* out =
            (uint32_t*)(a.out +
                        ((b * a.tokens + t) * a.q_heads + h * a.group +
                         r % a.group) * D + c0);
#pragma unroll
        for (int c = 0; c < D / 16; c += 2)
          out[c / 2] = see ? from_float16b<kHalf>(x[c] * inv) |
                                 from_float16b<kHalf>(x[c + 1] * inv) << 16
                           : 0u;
      }
    } else {
      float* p = a.part +
                 ((((b * a.c.heads + h) * a.q_tiles + qt) * a.splits + split) *
                      kRows + n * kTile + row) * (D + 2);
#pragma unroll
      for (int c = 0; c < D / 16; ++c) p[2 + c0 + c] = x[c];
      if (threadIdx.x % 16 == 0) {
        p[0] = see ? mx : kNegInf;
        p[1] = lt;
      }
    }
  }
}

// Joins the splits of one query row and head: one workgroup of D threads.
template <int D, bool kHalf, int NQ>
__global__ __launch_bounds__(D) void k_kv4_join(AttendArgs a) {
  constexpr int kRows = kTile * NQ;
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  const int r = blockIdx.x;
  const int qt = r / kRows;
  const int c = threadIdx.x;
  const float* p = a.part +
                   (((b * a.c.heads + h) * a.q_tiles + qt) * a.splits * kRows +
                    r % kRows) * (D + 2);
  constexpr int64_t kNext = (int64_t)kRows * (D + 2);
  float mx = kNegInf;
  for (int s = 0; s < a.splits; ++s) mx = fmaxf(mx, p[s * kNext]);
  float lt = 0.0f, x = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const float m = p[s * kNext];
    if (m == kNegInf) continue;
    const float f = __builtin_amdgcn_exp2f(m - mx);
    lt = __builtin_fmaf(f, p[s * kNext + 1], lt);
    x = __builtin_fmaf(f, p[s * kNext + 2 + c], x);
  }
  const int t = r / a.group;
  a.out[((b * a.tokens + t) * a.q_heads + h * a.group + r % a.group) * D + c] =
      (uint16_t)from_float16b<kHalf>(lt == 0.0f ? 0.0f : x / lt);
}

struct Plan {
  int nq, q_tiles, splits;
  size_t bytes;
};

Plan plan_for(const sfx_kv4* c, int64_t batch, int64_t tokens,
              int64_t q_heads) {
  Plan p;
  const int64_t rows = tokens * (q_heads / c->heads);
  p.nq = rows > kTile ? 2 : 1;
  p.q_tiles = (int)((rows + kTile * p.nq - 1) / (kTile * p.nq));
  const int64_t wgs = batch * c->heads * p.q_tiles;
  const int64_t blocks = c->table_width * c->page_size / kKvBlock;
  int64_t s = wgs > 0 ? 1024 / wgs : 1;
  s = std::min<int64_t>(s, (blocks + 15) / 16);
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(s, 128));
  p.bytes = p.splits == 1 ? 0
                          : (size_t)wgs * p.splits * kTile * p.nq *
                                (c->head_dim + 2) * 4;
  return p;
}

template <int D, bool kHalf, int NQ>
int launch(AttendArgs& a, int64_t batch, hipStream_t stream) {
  hipLaunchKernelGGL((k_kv4_attend<D, kHalf, NQ>),
                     dim3((unsigned)(a.splits * a.q_tiles),
                          (unsigned)a.c.heads, (unsigned)batch),
                     dim3(64 * kWaves), 0, stream, a);
  if (a.splits > 1)
    hipLaunchKernelGGL((k_kv4_join<D, kHalf, NQ>),
                       dim3((unsigned)a.rows, (unsigned)a.c.heads,
                            (unsigned)batch),
                       dim3(D), 0, stream, a);
  return (int)hipGetLastError();
}

template <int D, bool kHalf>
int launch_nq(AttendArgs& a, int nq, int64_t batch, hipStream_t stream) {
  return nq == 1 ? launch<D, kHalf, 1>(a, batch, stream)
                 : launch<D, kHalf, 2>(a, batch, stream);
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
  a.vec = (((uintptr_t)q->data & 15) |
           ((q->stride_b | q->stride_t | q->stride_h) & 7)) == 0;
  a.kv_len = kv_len;
  a.kv64 = kv_len_is64;
  a.q_len = q_len;
  a.q64 = q_len_is64;
  a.scale = scale * 1.44269504088896340736f;
  a.out = (uint16_t*)out;
  a.part = (float*)workspace;
  const bool half = cache->dtype == SFX_F16;
  switch (cache->head_dim) {
    case 64:
      return half ? launch_nq<64, true>(a, p.nq, batch, stream)
                  : launch_nq<64, false>(a, p.nq, batch, stream);
    case 128:
      return half ? launch_nq<128, true>(a, p.nq, batch, stream)
                  : launch_nq<128, false>(a, p.nq, batch, stream);
    default:
      return half ? launch_nq<256, true>(a, p.nq, batch, stream)
                  : launch_nq<256, false>(a, p.nq, batch, stream);
  }
}
