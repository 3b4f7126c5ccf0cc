// Writing and reading the 4-bit key/value cache.

#include "kv4.h"
#include "launch.h"

namespace sfx {

namespace {

struct AppendArgs {
  KvView c;
  sfx_heads k, v;
  int64_t tokens;
  const void* start;
  const void* count;
  int start64, count64, vec;
};

typedef uint16_t S2 __attribute__((ext_vector_type(2)));
typedef __bf16 B2 __attribute__((ext_vector_type(2)));
typedef _Float16 H2 __attribute__((ext_vector_type(2)));
typedef float F2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kInf = 0x7f800000u;

// Rows are eight four-bit values of one token (channels in order); afterwards
// eight of one channel, or back: two exchanges of half words and bytes, one of
// four bits.
__device__ __forceinline__ void transpose8(uint32_t (&a)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = a[i], y = a[i + 4];
    a[i] = __builtin_amdgcn_perm(y, x, 0x05040100u);
    a[i + 4] = __builtin_amdgcn_perm(y, x, 0x07060302u);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i & 2) continue;
    const uint32_t x = a[i], y = a[i + 2];
    a[i] = __builtin_amdgcn_perm(y, x, 0x06020400u);
    a[i + 2] = __builtin_amdgcn_perm(y, x, 0x07030501u);
  }
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const uint32_t x = a[i], y = a[i + 1];
    a[i] = (x & 0x0f0f0f0fu) | (y << 4 & 0xf0f0f0f0u);
    a[i + 1] = (x >> 4 & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u);
  }
}

// Token j of the octet that word row `quad` of a block holds.
__device__ __forceinline__ int token_of(int quad, int j) {
  return 16 * (quad / 2) + 8 * (j / 4) + 4 * (quad % 2) + j % 4;
}

// Task `e` of a block's values: eight tokens of row `quad`, channels c ..
// c + 7.  Four neighbours are channels 16 apart, whose words are neighbours.
__device__ __forceinline__ void task_of(int e, int* quad, int* c) {
  *c = e / 32 * 64 + e % 4 * 16 + e / 4 % 2 * 8;
  *quad = e / 8 % 4;
}

constexpr int kAppendThreads = 256;

// One workgroup per block of 32 positions, KV head and row: eight threads a
// token, D/8 channels each.  Keys go from registers to memory; the values'
// four bits cross LDS, where a thread turns eight tokens by eight channels.
// Words whose eight tokens are not all new keep the others' bits.
// 4 x 4,099 float16 tokens, 8 heads of 128: 20 us for 67 MB read and 18 MB
// written, 4.2 TB/s of the 4.9 that a large copy moves, so the memory bounds it;
// 64 x 17 tokens take 5.4 us and one token 4.0, hardly more than a launch.
//
// The instruction that rounds to 4 bits rounds to the nearest, ties to the even
// code, after a division by a power of two: the keys' rule.  For values, whose
// unit is s = top / 6, it is given z = |v| (6 / top), first rounded to 18 bits
// of mantissa: a v that lies exactly between two codes has 24 |v| = c top, c in
// {1, 3, 5, 7, 10, 14, 20}, and any other is at least 1 / (24 2^11) of itself
// away from that (11 significant bits), many times what the product and that
// rounding are off; so z is a tie where v is one and on v's side elsewhere.
template <int D, bool kHalf>
__global__ __launch_bounds__(kAppendThreads) void k_kv4_append(AppendArgs a) {
  using L = KvLayout<D>;
  constexpr int C = D / 8;  // channels per thread
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  int64_t n = a.count ? load_count(a.count, a.count64, b) : a.tokens;
  n = n < a.tokens ? n : a.tokens;
  int64_t s0 = load_count(a.start, a.start64, b);
  if (n <= 0 || s0 < 0 || s0 >= a.c.positions) return;
  if (n > a.c.positions - s0) n = a.c.positions - s0;
  const int64_t blk = s0 / kKvBlock + blockIdx.x;
  const int64_t p0 = blk * kKvBlock;
  if (p0 >= s0 + n) return;
  char* base = kv_block<D>(a.c, b, h, blk);
  if (!base) return;  // the whole workgroup: no barrier is missed

  __shared__ uint32_t vcode[kKvBlock][D / 8 + 1];  // eight channels a word
  const int t = threadIdx.x / 8;
  const int sub = threadIdx.x % 8;
  const int64_t i = p0 + t - s0;  // token of the call
  const bool live = i >= 0 && i < n;
  uint32_t kx[C / 2], vx[C / 2];  // two channels a word
  auto load = [&](const sfx_heads& src, uint32_t (&x)[C / 2]) {
    const uint16_t* p = (const uint16_t*)src.data +
                        (live ? b * src.stride_b + i * src.stride_t +
                                    h * src.stride_h + sub * C
                              : 0);
    if (a.vec) {
#pragma unroll
      for (int u = 0; u < C / 8; ++u) {
        const uint4 w = live ? ((const uint4*)p)[u] : uint4{0, 0, 0, 0};
        x[4 * u] = w.x;
        x[4 * u + 1] = w.y;
        x[4 * u + 2] = w.z;
        x[4 * u + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int u = 0; u < C / 2; ++u)
        x[u] = live ? (uint32_t)p[2 * u] | (uint32_t)p[2 * u + 1] << 16 : 0u;
    }
  };
  load(a.k, kx);
  load(a.v, vx);
  // Largest magnitude as a float's bits, infinities and NaN past every finite
  // one: the order of the 16 bits without the sign.
  auto amax = [&](const uint32_t (&x)[C / 2], int lanes) {
    S2 m = {0, 0};
#pragma unroll
    for (int u = 0; u < C / 2; ++u)
      m = __builtin_elementwise_max(
          m, __builtin_bit_cast(S2, x[u] & 0x7fff7fffu));
    uint32_t w = m.x > m.y ? m.x : m.y;
    for (int o = 1; o < lanes; o <<= 1) {
      const uint32_t q = __shfl_xor(w, o);
      w = w > q ? w : q;
    }
    return __float_as_uint(to_float16b<kHalf>(w));
  };

  // Keys: 32 channels = kPer threads share a scale.
  constexpr int kPer = 32 / C > 1 ? 32 / C : 1;
  uint32_t m = amax(kx, kPer);
  {
    // amax = f 2^e0 with f in [1, 2): amax / 2^(e0 - 2) is in [4, 8), and one
    // step coarser past 7.
    const int ex = (int)(m >> 23);
    int e = ex - 127 - 2 + ((m & 0x7fffffu) > 0x600000u);
    if (ex == 0) e = -126;
    e = e < -126 ? -126 : (e > (kHalf ? 13 : 125) ? (kHalf ? 13 : 125) : e);
    const float unit = __uint_as_float((uint32_t)(e + 127) << 23);
    uint32_t w[C / 8];
#pragma unroll
    for (int u = 0; u < C / 8; ++u) {
      uint32_t q = 0;
      if (kHalf) {
        const uint32_t* x = kx + 4 * u;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(
            q, __builtin_bit_cast(H2, x[0]), unit, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(
            q, __builtin_bit_cast(H2, x[1]), unit, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(
            q, __builtin_bit_cast(H2, x[2]), unit, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(
            q, __builtin_bit_cast(H2, x[3]), unit, 3);
      } else {
        const uint32_t* x = kx + 4 * u;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
            q, __builtin_bit_cast(B2, x[0]), unit, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
            q, __builtin_bit_cast(B2, x[1]), unit, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
            q, __builtin_bit_cast(B2, x[2]), unit, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
            q, __builtin_bit_cast(B2, x[3]), unit, 3);
      }
      w[u] = q;
    }
    if (live) {
      uint32_t* o = (uint32_t*)(base + t * (D / 2) + sub * (C / 2));
#pragma unroll
      for (int u = 0; u < C / 8; ++u) o[u] = w[u];
      if (sub % kPer == 0)
        ((uint8_t*)(base + L::kScale))[t * (D / 32) + sub * C / 32] =
            (uint8_t)(m >= kInf ? 255 : e + 127);
    }
  }

  // Values: one scale for the D channels.
  m = amax(vx, 8);
  {
    constexpr float kTiny = 6.0f * 0x1p-100f;
    float top = __uint_as_float(m);
    if (top < kTiny) top = kTiny;
    const bool odd = m >= kInf;  // the scale says NaN, the codes are finite
    if (live && sub == 0)
      ((float*)(base + L::kVScale))[t] =
          odd ? __uint_as_float(0x7fc00000u) : top / 6.0f;
    const float inv = odd ? 0.0f : 6.0f / top;
    auto z = [&](uint32_t bits) {
      const uint32_t q = __float_as_uint(to_float16b<kHalf>(bits) * inv);
      return __uint_as_float((q + 16u) & ~31u);
    };
#pragma unroll
    for (int u = 0; u < C / 8; ++u) {
      const uint32_t* x = vx + 4 * u;
      uint32_t q = 0;
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, z(x[0] & 0xffffu),
                                                   z(x[0] >> 16), 1.0f, 0);
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, z(x[1] & 0xffffu),
                                                   z(x[1] >> 16), 1.0f, 1);
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, z(x[2] & 0xffffu),
                                                   z(x[2] >> 16), 1.0f, 2);
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, z(x[3] & 0xffffu),
                                                   z(x[3] >> 16), 1.0f, 3);
      vcode[t][sub * (C / 8) + u] = q;
    }
  }
  __syncthreads();
  // Tokens of the block that are new.
  const int64_t lo64 = s0 - p0, hi64 = s0 + n - p0;
  const int lo = lo64 > 0 ? (int)lo64 : 0;
  const int hi = hi64 < kKvBlock ? (int)hi64 : kKvBlock;
  uint32_t* words = (uint32_t*)(base + L::kValue);
  for (int e = threadIdx.x; e < D / 2; e += kAppendThreads) {
    int quad, c;
    task_of(e, &quad, &c);
    uint32_t w[8], mask = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int tk = token_of(quad, j);
      w[j] = vcode[tk][c / 8];
      if (tk >= lo && tk < hi) mask |= 15u << (4 * j);
    }
    if (mask == 0) continue;
    transpose8(w);
    uint32_t* o = words + L::word(token_of(quad, 0), c);
    if (mask != 0xffffffffu) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = (w[j] & mask) | (o[4 * j] & ~mask);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) o[4 * j] = w[j];
  }
}

struct ReadArgs {
  KvView c;
  int64_t tokens;
  const void* start;
  const void* count;
  int start64, count64;
  uint16_t* k;
  uint16_t* v;
};

// One workgroup per block of 32 positions, KV head and row, the same threads
// and tasks as the append's.  4 x 4,099 tokens as there: 18 us, 4.7 TB/s.
template <int D, bool kHalf>
__global__ __launch_bounds__(256) void k_kv4_read(ReadArgs a) {
  using L = KvLayout<D>;
  constexpr int C = D / 8;
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  int64_t n = a.count ? load_count(a.count, a.count64, b) : a.tokens;
  n = n < 0 ? 0 : (n < a.tokens ? n : a.tokens);
  const int64_t s0 = load_count(a.start, a.start64, b);
  // Rows of the result that this workgroup writes: positions of its block,
  // where a row begins inside it and all of the first block is before it.
  const int64_t off = s0 >= 0 ? s0 % kKvBlock : 0;
  const int64_t i0 = (int64_t)blockIdx.x * kKvBlock - off;
  const char* base = nullptr;
  if (s0 >= 0 && i0 < n)
    base = kv_block<D>(a.c, b, h, s0 / kKvBlock + blockIdx.x);
  // results are [batch, tokens, heads, D]
  auto row = [&](int64_t i) {
    return ((b * a.tokens + i) * a.c.heads + h) * D;
  };
  {
    const int t = threadIdx.x / 8;
    const int sub = threadIdx.x % 8;
    const int64_t i = i0 + t;
    if (i >= 0 && i < a.tokens) {
      const bool there = base && i < n;
      const uint32_t* kw =
          (const uint32_t*)(base + t * (D / 2) + sub * (C / 2));
      uint32_t sb = 0;
      if (there)
        sb = ((const uint8_t*)(base + L::kScale))[t * (D / 32) + sub * C / 32];
      const float sc = __uint_as_float(sb << 23);
      uint4* o = (uint4*)(a.k + row(i) + sub * C);
#pragma unroll
      for (int u = 0; u < C / 8; ++u) {
        uint4 r = {0, 0, 0, 0};
        if (there) {
          const uint32_t w = kw[u];
          if (kHalf) {
            r.x = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 0));
            r.y = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 1));
            r.z = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 2));
            r.w = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, sc, 3));
          } else {
            r.x = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0));
            r.y = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1));
            r.z = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2));
            r.w = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3));
          }
        }
        o[u] = r;
      }
    }
  }
  for (int e = threadIdx.x; e < D / 2; e += 256) {
    int quad, c;
    task_of(e, &quad, &c);
    uint32_t w[8];
    if (base) {
      const uint32_t* p = (const uint32_t*)(base + L::kValue) +
                          L::word(token_of(quad, 0), c);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = p[4 * j];
      transpose8(w);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int tk = token_of(quad, j);
      const int64_t i = i0 + tk;
      if (i < 0 || i >= a.tokens) continue;
      uint4 r = {0, 0, 0, 0};
      if (base && i < n) {
        const float vs = ((const float*)(base + L::kVScale))[tk];
        auto two = [&](F2 x) {
          return from_float16b<kHalf>(x.x * vs) |
                 from_float16b<kHalf>(x.y * vs) << 16;
        };
        r.x = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], 1.0f, 0));
        r.y = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], 1.0f, 1));
        r.z = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], 1.0f, 2));
        r.w = two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[j], 1.0f, 3));
      }
      *(uint4*)(a.v + row(i) + c) = r;
    }
  }
}

template <class F>
int by_shape(const sfx_kv4* c, F f) {
  const bool half = c->dtype == SFX_F16;
  switch (c->head_dim) {
    case 64:
      return half ? f.template run<64, true>() : f.template run<64, false>();
    case 128:
      return half ? f.template run<128, true>() : f.template run<128, false>();
    default:
      return half ? f.template run<256, true>() : f.template run<256, false>();
  }
}

struct LaunchAppend {
  AppendArgs a;
  dim3 grid;
  hipStream_t stream;
  template <int D, bool kHalf>
  int run() {
    hipLaunchKernelGGL((k_kv4_append<D, kHalf>), grid, dim3(kAppendThreads), 0,
                       stream, a);
    return (int)hipGetLastError();
  }
};

struct LaunchRead {
  ReadArgs a;
  dim3 grid;
  hipStream_t stream;
  template <int D, bool kHalf>
  int run() {
    hipLaunchKernelGGL((k_kv4_read<D, kHalf>), grid, dim3(256), 0, stream, a);
    return (int)hipGetLastError();
  }
};

bool vec_heads(const sfx_heads& x) {
  return (((uintptr_t)x.data & 15) | ((x.stride_b | x.stride_t | x.stride_h) &
                                      7)) == 0;
}

constexpr int64_t kMaxTokens = int64_t(1) << 28;  // the grid's limit

}  // namespace

}  // namespace sfx

using namespace sfx;

extern "C" int64_t sfx_kv4_block_bytes(int64_t head_dim) {
  switch (head_dim) {
    case 64: return KvLayout<64>::kBytes;
    case 128: return KvLayout<128>::kBytes;
    case 256: return KvLayout<256>::kBytes;
    default: return 0;
  }
}

extern "C" int sfx_kv4_append(const sfx_kv4* cache, const sfx_heads* k,
                              const sfx_heads* v, int64_t batch,
                              int64_t tokens, const void* start,
                              int32_t start_is64, const void* count,
                              int32_t count_is64, hipStream_t stream) {
  LaunchAppend l;
  if (!kv_view(cache, &l.a.c) || !k || !v || batch < 0 || batch > 65535 ||
      tokens < 0 || tokens > kMaxTokens)
    return SFX_EINVAL;
  if (batch == 0 || tokens == 0) return 0;
  if (!k->data || !v->data || !start) return SFX_EINVAL;
  l.a.k = *k;
  l.a.v = *v;
  l.a.tokens = tokens;
  l.a.start = start;
  l.a.start64 = start_is64;
  l.a.count = count;
  l.a.count64 = count_is64;
  l.a.vec = vec_heads(*k) && vec_heads(*v);
  // a stretch of `tokens` positions touches at most this many blocks
  l.grid = dim3((unsigned)((tokens + kKvBlock - 2) / kKvBlock + 1),
                (unsigned)cache->heads, (unsigned)batch);
  l.stream = stream;
  return by_shape(cache, l);
}

extern "C" int sfx_kv4_read(const sfx_kv4* cache, int64_t batch,
                            int64_t tokens, const void* start,
                            int32_t start_is64, const void* count,
                            int32_t count_is64, void* k_out, void* v_out,
                            hipStream_t stream) {
  LaunchRead l;
  if (!kv_view(cache, &l.a.c) || batch < 0 || batch > 65535 || tokens < 0 ||
      tokens > kMaxTokens)
    return SFX_EINVAL;
  if (batch == 0 || tokens == 0) return 0;
  if (!start || !k_out || !v_out ||
      (((uintptr_t)k_out | (uintptr_t)v_out) & 15))
    return SFX_EINVAL;
  l.a.tokens = tokens;
  l.a.start = start;
  l.a.start64 = start_is64;
  l.a.count = count;
  l.a.count64 = count_is64;
  l.a.k = (uint16_t*)k_out;
  l.a.v = (uint16_t*)v_out;
  l.grid = dim3((unsigned)((tokens + kKvBlock - 2) / kKvBlock + 1),
                (unsigned)cache->heads, (unsigned)batch);
  l.stream = stream;
  return by_shape(cache, l);
}
