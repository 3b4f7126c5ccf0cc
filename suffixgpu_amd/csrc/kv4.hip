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

// Code of the e2m1 magnitude nearest to mag / (4 quarter): the midpoints
// between the eight are 1, 3, 5, 7, 10, 14 and 20 quarters, ties go to the even
// code.  Callers pass quarters of at most 19 significant bits or powers of two,
// so every comparison is exact (11 bits of an input, 5 of the factor).
__device__ __forceinline__ uint32_t e2m1_code(float mag, float quarter) {
  uint32_t c = mag > quarter;
  c += mag >= 3.0f * quarter;
  c += mag > 5.0f * quarter;
  c += mag >= 7.0f * quarter;
  c += mag > 10.0f * quarter;
  c += mag >= 14.0f * quarter;
  c += mag > 20.0f * quarter;
  return c;
}

constexpr int kAppendThreads = 256;

// One workgroup per block of 32 positions, KV head and row: eight threads a
// token, D/8 channels each.  Keys are written from registers; the codes of the
// values cross LDS to become words of eight tokens.  Words whose eight tokens
// are not all new keep the others' bits.
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

  __shared__ uint32_t vcode[kKvBlock][D / 4 + 1];  // a byte per channel
  const int t = threadIdx.x / 8;
  const int sub = threadIdx.x % 8;
  const int64_t i = p0 + t - s0;  // token of the call
  const bool live = i >= 0 && i < n;
  float x[C];
  auto load = [&](const sfx_heads& src) {
    const uint16_t* p = (const uint16_t*)src.data +
                        (live ? b * src.stride_b + i * src.stride_t +
                                    h * src.stride_h + sub * C
                              : 0);
    if (a.vec) {
#pragma unroll
      for (int u = 0; u < C / 8; ++u) {
        const uint4 w = live ? ((const uint4*)p)[u] : uint4{0, 0, 0, 0};
        const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[8 * u + 2 * j] = to_float16b<kHalf>(q[j] & 0xffff);
          x[8 * u + 2 * j + 1] = to_float16b<kHalf>(q[j] >> 16);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < C; ++u)
        x[u] = live ? to_float16b<kHalf>(p[u]) : 0.0f;
    }
  };
  // Largest magnitude, and whether all are finite, as one ordered integer:
  // the bits of |x| order infinities and NaN past every finite value.
  auto amax_bits = [&]() {
    uint32_t m = 0;
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const uint32_t w = __float_as_uint(x[u]) & 0x7fffffffu;
      m = m > w ? m : w;
    }
    return m;
  };
  constexpr uint32_t kInf = 0x7f800000u;

  // Keys: 32 channels = kPer threads share a scale.
  load(a.k);
  uint32_t m = amax_bits();
  constexpr int kPer = 32 / C > 1 ? 32 / C : 1;
#pragma unroll
  for (int o = 1; o < kPer; o <<= 1) {
    const uint32_t w = __shfl_xor(m, o);
    m = m > w ? m : w;
  }
  {
    // amax = f 2^e0 with f in [1, 2): amax / 2^(e0 - 2) is in [4, 8), and one
    // step coarser past 7.
    const int ex = (int)(m >> 23);
    int e = ex - 127 - 2 + ((m & 0x7fffffu) > 0x600000u);
    if (ex == 0) e = -126;
    e = e < -126 ? -126 : (e > (kHalf ? 13 : 125) ? (kHalf ? 13 : 125) : e);
    const uint32_t sb = m >= kInf ? 255u : (uint32_t)(e + 127);
    const float unit = 0.25f * __uint_as_float((uint32_t)(e + 127) << 23);
    uint32_t w[C / 8];
#pragma unroll
    for (int u = 0; u < C / 8; ++u) {
      uint32_t q = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = x[8 * u + j];
        q |= (e2m1_code(fabsf(y), unit) |
              (__float_as_uint(y) >> 31) << 3)
             << (4 * j);
      }
      w[u] = q;
    }
    if (live) {
      uint32_t* o = (uint32_t*)(base + t * (D / 2) + sub * (C / 2));
#pragma unroll
      for (int u = 0; u < C / 8; ++u) o[u] = w[u];
      if (sub % kPer == 0)
        ((uint8_t*)(base + L::kScale))[t * (D / 32) + sub * C / 32] =
            (uint8_t)sb;
    }
  }

  // Values: one scale for the D channels.
  load(a.v);
  m = amax_bits();
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    const uint32_t w = __shfl_xor(m, o);
    m = m > w ? m : w;
  }
  {
    constexpr float kTiny = 6.0f * 0x1p-100f;
    float top = __uint_as_float(m);
    if (m < kInf && top < kTiny) top = kTiny;
    if (live && sub == 0)
      ((float*)(base + L::kVScale))[t] =
          m >= kInf ? __uint_as_float(0x7fc00000u) : top / 6.0f;
    if (m >= kInf) top = 1.0f;  // the scale says NaN, the codes are finite
    // 24 |v| against multiples of the largest; both 2^-16 times where that
    // could overflow.
    const float pre = top >= 0x1p100f ? 0x1p-16f : 1.0f;
    top *= pre;
    const float mul = 24.0f * pre;
#pragma unroll
    for (int u = 0; u < C / 4; ++u) {
      uint32_t q = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = x[4 * u + j];
        q |= (e2m1_code(mul * fabsf(y), top) |
              (__float_as_uint(y) >> 31) << 3)
             << (8 * j);
      }
      vcode[t][sub * (C / 4) + u] = q;
    }
  }
  __syncthreads();
  // Tokens of the block that are new.
  const int64_t lo64 = s0 - p0, hi64 = s0 + n - p0;
  const int lo = lo64 > 0 ? (int)lo64 : 0;
  const int hi = hi64 < kKvBlock ? (int)hi64 : kKvBlock;
  uint32_t* words = (uint32_t*)(base + L::kValue);
  for (int w = threadIdx.x; w < D * 4; w += kAppendThreads) {
    // word w: channel and token octet (word() of the layout, read backwards)
    const int c = w / 256 * 64 + w % 4 * 16 + w / 4 % 16;
    const int quad = w / 64 % 4;
    uint32_t val = 0, mask = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int tk = 16 * (quad / 2) + 8 * (j / 4) + 4 * (quad % 2) + j % 4;
      if (tk >= lo && tk < hi) {
        mask |= 15u << (4 * j);
        val |= (vcode[tk][c / 4] >> (8 * (c % 4)) & 15u) << (4 * j);
      }
    }
    if (mask == 0) continue;
    if (mask != 0xffffffffu) val |= words[w] & ~mask;
    words[w] = val;
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

// Eight threads a token and KV head, D/8 channels each.
template <int D, bool kHalf>
__global__ __launch_bounds__(256) void k_kv4_read(ReadArgs a) {
  using L = KvLayout<D>;
  constexpr int C = D / 8;
  const int64_t b = blockIdx.z;
  const int h = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x / 8;
  if (i >= a.tokens) return;
  const int sub = threadIdx.x % 8;
  int64_t n = a.count ? load_count(a.count, a.count64, b) : a.tokens;
  const int64_t s0 = load_count(a.start, a.start64, b);
  const int64_t pos = s0 + i;
  const char* base = nullptr;
  if (i < n && s0 >= 0 && pos < a.c.positions)
    base = kv_block<D>(a.c, b, h, pos / kKvBlock);
  uint32_t ko[C / 2], vo[C / 2];
#pragma unroll
  for (int u = 0; u < C / 2; ++u) ko[u] = vo[u] = 0;
  if (base) {
    const int t = (int)(pos % kKvBlock);
    const uint32_t* kw = (const uint32_t*)(base + t * (D / 2) + sub * (C / 2));
    const uint32_t sb =
        ((const uint8_t*)(base + L::kScale))[t * (D / 32) + sub * C / 32];
    const float ks = sb == 255 ? __uint_as_float(0x7fc00000u)
                               : __uint_as_float(sb << 23);
    const float vs = ((const float*)(base + L::kVScale))[t];
    const uint32_t* vw = (const uint32_t*)(base + L::kValue);
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const float kf = e2m1_value(kw[u / 8] >> (4 * (u % 8)) & 15u) * ks;
      ko[u / 2] |= from_float16b<kHalf>(kf) << (16 * (u % 2));
      const float vf =
          e2m1_value(vw[L::word(t, sub * C + u)] >> L::shift(t) & 15u) * vs;
      vo[u / 2] |= from_float16b<kHalf>(vf) << (16 * (u % 2));
    }
  }
  const int64_t o = (((b * a.tokens + i) * a.c.heads + h) * D + sub * C) / 2;
#pragma unroll
  for (int u = 0; u < C / 2; u += 4) {
    *(uint4*)((uint32_t*)a.k + o + u) =
        uint4{ko[u], ko[u + 1], ko[u + 2], ko[u + 3]};
    *(uint4*)((uint32_t*)a.v + o + u) =
        uint4{vo[u], vo[u + 1], vo[u + 2], vo[u + 3]};
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
  l.grid = dim3((unsigned)((tokens + 31) / 32), (unsigned)cache->heads,
                (unsigned)batch);
  l.stream = stream;
  return by_shape(cache, l);
}
