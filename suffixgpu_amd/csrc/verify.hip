// Verification of drafted tokens against the target model's logits.
//
// A draft d at position j stays iff u q(d) < p_j(d), p_j = softmax(x / T); the
// token after the accepted ones is drawn from r = max(p_j - q, 0) (or p_j) as
// argmax_i r_i / e_i with e_i exponentially distributed: the smallest of
// exponential clocks of rates r_i rings with probability r_i / sum r.  A draw
// by clocks needs no running sum over the vocabulary, whose rounding would
// decide between neighbours, and its argmax is the same in any order.
//
// Two launches: the first takes the largest logit and the sum of exponentials
// of every drafted position, a workgroup per 8,192 logits; the second's
// workgroups each find the row's first rejected position from those, race
// their 8,192 candidates there, and the row's last one writes the result.

#include <algorithm>

#include "launch.h"
#include "sfx_common.h"

namespace sfx {

namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;  // logits per workgroup
constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMaxScale = 1e30f;

// What a workgroup found in its part of a position: largest logit, and the sum
// of 2^((x - top) c), or, of a greedy row, the first index of the largest.
struct Part {
  float top;
  union {
    float sum;
    int32_t at;
  };
};

// A workgroup's best candidate: its rate over its clock relative to 2^(shift
// c), whether it is one of r (or, with r empty, of p), and its token (-1:
// none).
struct Best {
  float key;
  float shift;
  int32_t token;
  int32_t in_r;
};

struct VerifyArgs {
  sfx_verify v;
  int chunks;
  Part* part;         // [batch, K + 1, chunks]
  Best* best;         // [batch, chunks]
  unsigned* arrived;  // [batch]
};

template <int DT>
struct Elem;
template <>
struct Elem<SFX_BF16> {
  using T = uint16_t;
  static __device__ float get(T x) { return __uint_as_float((uint32_t)x << 16); }
};
template <>
struct Elem<SFX_F16> {
  using T = uint16_t;
  static __device__ float get(T x) {
    return (float)__builtin_bit_cast(_Float16, x);
  }
};
template <>
struct Elem<SFX_F32> {
  using T = float;
  static __device__ float get(T x) { return x; }
};

// A thread's share of chunk c of a row of n elements of any alignment: per
// step u E consecutive elements, 16 bytes from an aligned address where all
// lie inside the row.
template <class T>
struct Share {
  static constexpr int E = 16 / sizeof(T);
  static constexpr int U = kChunk / (kThreads * E);
  const T* row;
  int64_t n;
  int64_t first;  // index of the thread's first element of step 0
  __device__ Share(const T* r, int64_t len, int chunk) : row(r), n(len) {
    const int off = (int)(((uintptr_t)r & 15) / sizeof(T));
    first = ((int64_t)chunk * kThreads * U + threadIdx.x) * E - off;
  }
  __device__ int64_t index(int u, int e) const {
    return first + (int64_t)u * kThreads * E + e;
  }
};

// Logits of a share as floats, -inf for NaN and outside the row.
template <int DT>
__device__ __forceinline__ void load_logits(
    const Share<typename Elem<DT>::T>& s,
    float (&x)[Share<typename Elem<DT>::T>::U]
              [Share<typename Elem<DT>::T>::E]) {
  using T = typename Elem<DT>::T;
  constexpr int E = Share<T>::E, U = Share<T>::U;
  T raw[U][E];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = s.index(u, 0);
    if (i >= 0 && i + E <= s.n) {
      const uint4 w = *(const uint4*)(s.row + i);
      __builtin_memcpy(raw[u], &w, 16);
#pragma unroll
      for (int e = 0; e < E; ++e) x[u][e] = Elem<DT>::get(raw[u][e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        x[u][e] = i + e >= 0 && i + e < s.n ? Elem<DT>::get(s.row[i + e])
                                            : kNegInf;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) x[u][e] = fmaxf(x[u][e], kNegInf);
}

// Floats as unsigned integers of the same order (-0 as 0).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Difference to the largest, where infinities may meet.
__device__ __forceinline__ float below(float x, float top) {
  return x == top ? 0.0f : x - top;
}

template <class V, class Op>
__device__ __forceinline__ V block_reduce(V v, V* lds, Op op) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < kThreads / kWave; ++w) v = op(v, lds[w]);
  return v;
}

__device__ __forceinline__ float temperature_of(const sfx_verify& v,
                                                int64_t b) {
  if (v.all_greedy) return 0.0f;
  const float t = v.temperature ? v.temperature[b] : 1.0f;
  return t > 0.0f ? t : 0.0f;
}

__device__ __forceinline__ float scale_of(float t) {
  return fminf(kLog2e / t, kMaxScale);
}

// Drafts of row b that are candidates: those before num_valid and before the
// first id that is no token.
__device__ __forceinline__ int drafts_of(const sfx_verify& v, int64_t b) {
  int64_t n = v.num_valid[b];
  n = n < 0 ? 0 : (n > v.k ? v.k : n);
  int i = 0;
  while (i < n) {
    const int32_t d = v.draft[b * v.k + i];
    if (d < 0 || d >= v.vocab) break;
    ++i;
  }
  return i;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void k_verify_scan(VerifyArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int E = Share<T>::E, U = Share<T>::U;
  const int64_t b = blockIdx.x / a.chunks;
  const int j = blockIdx.y;
  const int chunk = blockIdx.x % a.chunks;
  if (j == 0 && chunk == 0 && threadIdx.x == 0) a.arrived[b] = 0;
  const float t = temperature_of(a.v, b);
  const int n = drafts_of(a.v, b);
  // A row that draws races the position after its drafts without a sum.
  if (j > n || (j == n && t > 0.0f)) return;
  __shared__ float ldf[kThreads / kWave];
  __shared__ uint64_t ldu[kThreads / kWave];
  const Share<T> s((const T*)a.v.logits + b * a.v.stride_b + j * a.v.stride_j,
                   a.v.vocab, chunk);
  float x[U][E];
  load_logits<DT>(s, x);
  float top = kNegInf;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, x[u][e]);
  top = block_reduce(top, ldf, [](float p, float q) { return fmaxf(p, q); });
  Part r;
  r.top = top;
  if (t > 0.0f) {
    const float c = scale_of(t);
    float sum = 0.0f;
    if (top > kNegInf) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e)
          sum += __builtin_amdgcn_exp2f(below(x[u][e], top) * c);
    }
    r.sum = block_reduce(sum, ldf, [](float p, float q) { return p + q; });
  } else {
    uint64_t best = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[u][e] == top) {
          const uint64_t k = ~(uint32_t)s.index(u, e);
          best = best > k ? best : k;
        }
    best = block_reduce(best, ldu,
                        [](uint64_t p, uint64_t q) { return p > q ? p : q; });
    r.at = (int32_t)~(uint32_t)best;
  }
  if (threadIdx.x == 0) a.part[(b * (a.v.k + 1) + j) * a.chunks + chunk] = r;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void k_verify_draw(VerifyArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int E = Share<T>::E, U = Share<T>::U;
  const int per_row = a.v.all_greedy ? 1 : a.chunks;
  const int64_t b = blockIdx.x / per_row;
  const int chunk = blockIdx.x % per_row;
  const int K = (int)a.v.k;
  const float t = temperature_of(a.v, b);
  const bool greedy = !(t > 0.0f);
  const float c = greedy ? 0.0f : scale_of(t);
  const int n = drafts_of(a.v, b);
  const T* logits = (const T*)a.v.logits + b * a.v.stride_b;
  __shared__ uint64_t ldu[kThreads / kWave];
  __shared__ float ldf[kThreads / kWave];
  __shared__ int stop;           // first position that accepts nothing
  __shared__ float s_top, s_sum;
  __shared__ int s_at;
  __shared__ int lds_flag;
  if (threadIdx.x == 0) stop = n;
  __syncthreads();
  // A wave per position: the parts of one position are read at once.
  const int wave = threadIdx.x / kWave, lane = lane_id();
  for (int j = wave; j <= n; j += kThreads / kWave) {
    if (j == n && !greedy) break;
    const Part* p = a.part + (b * (K + 1) + j) * a.chunks;
    float top = kNegInf, sum = 0.0f;
    int at = 0x7fffffff;
    for (int i = lane; i < a.chunks; i += kWave) {
      const Part q = p[i];
      if (greedy) {
        if (q.top > top) {
          top = q.top;
          at = q.at;
        }
      } else if (q.top > top) {
        sum = sum * (top == kNegInf ? 0.0f
                                    : __builtin_amdgcn_exp2f(
                                          below(top, q.top) * c)) + q.sum;
        top = q.top;
      } else if (q.top > kNegInf) {
        sum += q.sum * __builtin_amdgcn_exp2f(below(q.top, top) * c);
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float qt = __shfl_xor(top, o);
      const float qs = __shfl_xor(sum, o);
      const int qa = __shfl_xor(at, o);
      if (greedy) {
        if (qt > top || (qt == top && qa < at)) {
          top = qt;
          at = qa;
        }
      } else {
        const float mx = fmaxf(top, qt);
        if (mx > kNegInf)
          sum = sum * __builtin_amdgcn_exp2f(below(top, mx) * c) +
                qs * __builtin_amdgcn_exp2f(below(qt, mx) * c);
        top = mx;
      }
    }
    bool ok = false;
    if (j < n && top > kNegInf) {
      const int d = a.v.draft[b * K + j];
      if (greedy) {
        ok = d == at;
      } else {
        const float x = fmaxf(Elem<DT>::get(logits[j * a.v.stride_j + d]),
                              kNegInf);
        const float p1 = __builtin_amdgcn_exp2f(below(x, top) * c) / sum;
        const float q1 =
            a.v.draft_probs
                ? a.v.draft_probs[(b * K + j) * a.v.vocab + d]
                : 1.0f;
        ok = a.v.uniform[b * K + j] * q1 < p1;
      }
    }
    if (!ok && lane == 0) atomicMin(&stop, j);
  }
  __syncthreads();
  const int at_pos = stop;
  // The drawn position's statistics again, by the wave that holds them.
  if (greedy || at_pos < n) {
    const Part* p = a.part + (b * (K + 1) + at_pos) * a.chunks;
    if (threadIdx.x == 0) {
      float top = kNegInf, sum = 0.0f;
      int at = -1;
      for (int i = 0; i < a.chunks; ++i)
        if (p[i].top > top) {
          top = p[i].top;
          at = p[i].at;
        }
      if (!greedy && top > kNegInf)
        for (int i = 0; i < a.chunks; ++i)
          if (p[i].top > kNegInf)
            sum += p[i].sum * __builtin_amdgcn_exp2f(below(p[i].top, top) * c);
      s_top = top;
      s_sum = sum;
      s_at = top > kNegInf ? at : -1;
    }
    __syncthreads();
  }
  int token = -1;
  if (greedy) {
    if (chunk > 0) return;
    token = s_at;
  } else {
    const Share<T> s(logits + at_pos * a.v.stride_j, a.v.vocab, chunk);
    float x[U][E];
    load_logits<DT>(s, x);
    const float* noise = a.v.noise + b * a.v.vocab;
    const bool res = at_pos < n;  // draw from what q left of p
    const int d = res ? a.v.draft[b * K + at_pos] : -1;
    const float* q = res && a.v.draft_probs
                         ? a.v.draft_probs + (b * K + at_pos) * a.v.vocab
                         : nullptr;
    float top = kNegInf;
    if (q) {
      top = s_top;
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, x[u][e]);
      top = block_reduce(top, ldf, [](float p, float r) { return fmaxf(p, r); });
    }
    // Keys: the bits of a rate over its clock, the top bit for members of r.
    uint32_t key = 0;
    uint32_t tok = 0xffffffffu;
    const float inv = q ? s_sum : 1.0f;
    if (top > kNegInf) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t i = s.index(u, e);
          if (i < 0 || i >= a.v.vocab) continue;
          const float p = __builtin_amdgcn_exp2f(below(x[u][e], top) * c) / inv;
          const float r = q ? p - q[i] : (i == d ? 0.0f : p);
          const float g = (r > 0.0f ? r : p) / noise[i];
          uint32_t kk = g > 0.0f ? __float_as_uint(g) : 0u;
          if (kk && r > 0.0f) kk |= 0x80000000u;
          if (kk > key) {
            key = kk;
            tok = (uint32_t)i;
          }
        }
    }
    uint64_t best = (uint64_t)key << 32 | (uint32_t)~tok;
    best = block_reduce(best, ldu,
                        [](uint64_t p, uint64_t r) { return p > r ? p : r; });
    if (threadIdx.x == 0) {
      const uint32_t k32 = (uint32_t)(best >> 32);
      Best* o = a.best + b * a.chunks + chunk;
      ws_store(&o->key, __uint_as_float(k32 & 0x7fffffffu));
      ws_store(&o->shift, top);
      ws_store(&o->token, k32 ? (int32_t)~(uint32_t)best : -1);
      ws_store(&o->in_r, (int32_t)(k32 >> 31));
    }
    if (!block_arrive<false>(a.arrived + b, (unsigned)a.chunks, &lds_flag))
      return;
    // The row's last workgroup: the best of all, earlier ones on ties.
    if (wave == 0) {
      float mx = kNegInf;
      for (int i = lane; i < a.chunks; i += kWave)
        mx = fmaxf(mx, ws_load(&a.best[b * a.chunks + i].shift));
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      uint64_t all = 0;
      for (int i = lane; i < a.chunks; i += kWave) {
        const Best* o = a.best + b * a.chunks + i;
        const int32_t tk = ws_load(&o->token);
        if (tk < 0) continue;
        const float g = ws_load(&o->key) *
                        __builtin_amdgcn_exp2f(
                            below(ws_load(&o->shift), mx) * c);
        const uint32_t kk =
            __float_as_uint(g) | (uint32_t)ws_load(&o->in_r) << 31;
        const uint64_t w = (uint64_t)kk << 32 | (uint32_t)~(uint32_t)tk;
        all = all > w ? all : w;
      }
      all = wave_max_u64(all);
      token = all ? (int32_t)~(uint32_t)all : -1;
    }
  }
  if (wave == 0) {
    int32_t* out = a.v.sampled + b * (K + 1);
    for (int i = lane; i <= K; i += kWave)
      out[i] = i < at_pos ? a.v.draft[b * K + i] : (i == at_pos ? token : -1);
    if (lane == 0) a.v.count[b] = at_pos + (token >= 0);
  }
}

int chunks_for(int64_t vocab) {
  // up to seven elements before an aligned address
  return (int)((vocab + 7 + kChunk - 1) / kChunk);
}

struct Layout {
  size_t part, best, arrived, bytes;
};

Layout layout_for(int64_t batch, int64_t k, int64_t vocab) {
  const size_t ch = (size_t)chunks_for(vocab);
  Layout l;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  l.part = 0;
  l.best = up((size_t)batch * (size_t)(k + 1) * ch * sizeof(Part));
  l.arrived = l.best + up((size_t)batch * ch * sizeof(Best));
  l.bytes = l.arrived + up((size_t)batch * 4);
  return l;
}

bool sizes_ok(int64_t batch, int64_t k, int64_t vocab) {
  // the grid's limit is 2^32 threads along x
  return batch >= 0 && k >= 0 && k <= 4096 && vocab >= 1 &&
         vocab <= (int64_t(1) << 28) && batch <= (1 << 23) / chunks_for(vocab);
}

template <int DT>
int launch(const VerifyArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(k_verify_scan<DT>,
                     dim3((unsigned)(a.v.batch * a.chunks),
                          (unsigned)(a.v.k + 1)),
                     dim3(kThreads), 0, stream, a);
  hipLaunchKernelGGL(k_verify_draw<DT>,
                     dim3((unsigned)(a.v.batch *
                                     (a.v.all_greedy ? 1 : a.chunks))),
                     dim3(kThreads), 0, stream, a);
  return (int)hipGetLastError();
}

}  // namespace

}  // namespace sfx

using namespace sfx;

extern "C" size_t sfx_verify_workspace_size(int64_t batch, int64_t k,
                                            int64_t vocab) {
  if (!sizes_ok(batch, k, vocab) || batch == 0) return 0;
  return layout_for(batch, k, vocab).bytes;
}

extern "C" int sfx_verify_draft(const sfx_verify* args, void* workspace,
                                size_t workspace_bytes, hipStream_t stream) {
  if (!args) return SFX_EINVAL;
  VerifyArgs a;
  a.v = *args;
  const sfx_verify& v = a.v;
  if (!sizes_ok(v.batch, v.k, v.vocab) ||
      (v.dtype != SFX_BF16 && v.dtype != SFX_F16 && v.dtype != SFX_F32))
    return SFX_EINVAL;
  if (v.batch == 0) return 0;
  if (!v.logits || !v.num_valid || !v.sampled || !v.count ||
      (v.k > 0 && !v.draft))
    return SFX_EINVAL;
  if (!v.all_greedy && (!v.noise || (v.k > 0 && !v.uniform)))
    return SFX_EINVAL;
  const Layout l = layout_for(v.batch, v.k, v.vocab);
  if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < l.bytes)
    return SFX_EINVAL;
  char* w = (char*)workspace;
  a.chunks = chunks_for(v.vocab);
  a.part = (Part*)(w + l.part);
  a.best = (Best*)(w + l.best);
  a.arrived = (unsigned*)(w + l.arrived);
  switch (v.dtype) {
    case SFX_BF16: return launch<SFX_BF16>(a, stream);
    case SFX_F16: return launch<SFX_F16>(a, stream);
    default: return launch<SFX_F32>(a, stream);
  }
}
