// Log probabilities of given tokens, the entropy of their distributions, and the
// likeliest alternatives, in one pass over the logits.
//
// With z_i = (x_i - max x) / T and R the sum of e^z over all but one of the
// largest (a token is often nearly certain: what the others add to one is then
// all of its log probability, and would be lost beside the one),
//   log p_i = z_i - log(1 + R),   H = log(1 + R) - sum z e^z / (1 + R).
//
// The first launch takes 8,192 logits a workgroup, which stay in registers: their
// largest, R and sum z e^z, and their n largest in order.  Of the maxima of
// pieces of 16 vectors (contiguous, so that the lowest index wins ties) the n
// largest hold the n largest logits: all that reach the least of those n maxima
// and lie in those pieces are ranked, a few more than n.  The second launch joins
// a position's parts.  Positions without a token leave at once.

#include <algorithm>

#include "launch.h"
#include "vocab.h"

namespace sfx {

namespace {

constexpr int kWaves = kThreads / kWave;
constexpr float kMaxScale = 0x1.fffffep127f;
constexpr float kLn2 = 0.69314718055994530942f;
// 2^kFloor is zero in 32 bits; where z may be -inf or a NaN, z e^z shall be zero.
constexpr float kFloor = -160.0f;

// What is known of some logits: the largest, R and sum z e^z in base 2 (greedy:
// in the place of R the first index of the largest).
struct Part {
  float top, rest, zsum;
  int32_t at;
};

struct Entry {
  float x;
  int32_t at;
};

struct LogArgs {
  sfx_logprobs v;
  int chunks;
  Part* part;    // [batch * positions, chunks]
  Entry* entry;  // [batch * positions, chunks, top]
};

__device__ __forceinline__ float temperature_of(const sfx_logprobs& v,
                                                int64_t b) {
  const float t = v.temperature ? v.temperature[b] : 1.0f;
  return t > 0.0f ? t : 0.0f;
}

// Half the difference to the largest, which is a float where the difference is
// too large for one; 0 where infinities meet.
__device__ __forceinline__ float half_below(float x, float top) {
  return x == top ? 0.0f : __builtin_fmaf(x, 0.5f, -0.5f * top);
}

// Base-2 scale of such a half.
__device__ __forceinline__ float scale_of(float t) {
  return fminf(2.0f * kLog2e / t, kMaxScale);
}

// Whether candidate (x, i) comes before (y, j).
__device__ __forceinline__ bool before(float x, int i, float y, int j) {
  return x > y || (x == y && i < j);
}

// Adds q to p; c: scale_of.
__device__ __forceinline__ void join(Part& p, const Part& q, float c) {
  if (q.top == kNegInf) return;
  if (p.top == kNegInf) {
    p = q;
    return;
  }
  const bool swap = q.top > p.top;
  const Part a = swap ? q : p, b = swap ? p : q;
  const float d = fmaxf(half_below(b.top, a.top) * c, kFloor);
  const float f = __builtin_amdgcn_exp2f(d);
  p.top = a.top;
  p.rest = a.rest + (1.0f + b.rest) * f;
  p.zsum = a.zsum + (b.zsum + d * (1.0f + b.rest)) * f;
  p.at = a.top == b.top ? min(a.at, b.at) : a.at;
}

constexpr int kCap = 256;  // candidates that are ranked

template <int DT, bool kTop>
__global__ __launch_bounds__(kThreads) void k_logprobs_scan(LogArgs a) {
  using S = Share<DT>;
  constexpr int E = S::E, U = S::U;
  constexpr int kSegs = U * kThreads / 16;  // pieces of 16 vectors
  static_assert(kSegs >= SFX_LOGPROBS_TOP && kCap >= SFX_LOGPROBS_TOP, "");
  const int chunk = blockIdx.x % a.chunks;
  const int64_t pos = blockIdx.x / a.chunks;
  const int64_t b = pos / a.v.positions, j = pos % a.v.positions;
  const int32_t tok = a.v.tokens[pos];
  if (tok < 0 || tok >= a.v.vocab) return;
  const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
  __shared__ Part lds[kWaves];
  __shared__ float seg[kTop ? kSegs : 1];
  __shared__ uint32_t chosen[kTop ? (kSegs + 31) / 32 : 1];
  __shared__ Entry cand[kTop ? kCap : 1];
  __shared__ int n_cand;
  __shared__ float least;
  const float t = temperature_of(a.v, b);
  const bool greedy = !(t > 0.0f);
  const float c = greedy ? 0.0f : scale_of(t);
  const typename S::T* row = (const typename S::T*)a.v.logits +
                             b * a.v.stride_b + j * a.v.stride_j;
  S s(row, a.v.vocab, chunk);
  s.load(row);
  // largest of each vector, of the thread, of the wave
  float vtop[U], top = fmaxf(s.single, kNegInf);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    vtop[u] = kNegInf;
#pragma unroll
    for (int e = 0; e < E; ++e) vtop[u] = fmaxf(vtop[u], s.get(u, e));
    top = fmaxf(top, vtop[u]);
  }
  const float mine = top;
  top = wave_max(top);
  if (kTop) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float m = vtop[u];
      m = fmaxf(m, dpp<0xb1, 0xf>(m, m));    // lane ^ 1
      m = fmaxf(m, dpp<0x4e, 0xf>(m, m));    // lane ^ 2
      m = fmaxf(m, dpp<0x141, 0xf>(m, m));   // half of a row mirrored
      m = fmaxf(m, dpp<0x140, 0xf>(m, m));   // row mirrored
      if (lane % 16 == 0) seg[u * (kThreads / 16) + tid / 16] = m;
    }
    if (tid == 0) n_cand = 0;
  }
  Part p = {top, 0.0f, 0.0f, 0x7fffffff};
  if (greedy) {
    if (mine == top && top > kNegInf) {
      int at = 0x7fffffff;
      s.again([&](float x, int i) { at = x == top ? min(at, i) : at; });
      p.at = at;
    }
    p.at = wave_min(p.at);
  } else if (top > kNegInf) {
    s.forget();
    float sum = 0.0f, zsum = 0.0f;
    int equal = 0;
    const float half = -0.5f * top;
    auto add = [&](float x) {
      const float z = fmaxf(__builtin_fmaf(x, 0.5f, half) * c, kFloor);
      const float e = __builtin_amdgcn_exp2f(z);
      sum += e;
      zsum = __builtin_fmaf(z, e, zsum);
    };
    auto add_special = [&](float x) {
      const bool is = x == top;
      equal += is;
      const float z =
          is ? kFloor : fmaxf(__builtin_fmaf(x, 0.5f, half) * c, kFloor);
      const float e = __builtin_amdgcn_exp2f(z);
      sum += e;
      zsum = __builtin_fmaf(z, e, zsum);
    };
    add_special(s.single);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // one vector in U holds the wave's largest
      if (ballot(vtop[u] == top)) {
#pragma unroll
        for (int e = 0; e < E; ++e) add_special(s.get(u, e));
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) add(s.get(u, e));
      }
    }
    p.rest = wave_sum(sum) + (wave_sum((float)equal) - 1.0f);
    p.zsum = wave_sum(zsum);
  }
  if (lane == 0) lds[wave] = p;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) join(p, lds[w], c);
    a.part[pos * a.chunks + chunk] = p;
  }
  if (!kTop) return;

  // The n pieces with the largest maxima, the lowest on ties.
  const int n = (int)a.v.top;
  if (tid < kSegs) {
    const float m = seg[tid];
    int rank = 0;
    for (int i = 0; i < kSegs; ++i) rank += before(seg[i], i, m, tid);
    const bool in = rank < n && m > kNegInf;
    const uint64_t w = ballot(in);
    if (lane == 0) {
      chosen[2 * wave] = (uint32_t)w;
      chosen[2 * wave + 1] = (uint32_t)(w >> 32);
    }
    if (rank == n - 1) least = m;
  }
  __syncthreads();
  const float floor = least;
  auto offer = [&](float x, int i) {
    if (x >= floor && x > kNegInf) {
      const int k = atomicAdd(&n_cand, 1);
      if (k < kCap) cand[k] = Entry{x, i};
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int sg = u * (kThreads / 16) + tid / 16;
    if ((chosen[sg / 32] >> (sg % 32) & 1) && vtop[u] >= floor) {
#pragma unroll
      for (int e = 0; e < E; ++e) offer(s.get(u, e), s.index(u * E + e));
    }
  }
  if (s.extra >= 0) offer(s.single, s.extra);
  __syncthreads();
  Entry* out = a.entry + (pos * a.chunks + chunk) * n;
  const int count = n_cand;
  if (count <= kCap) {
    if (tid < n && tid >= count) out[tid] = Entry{kNegInf, -1};
    if (tid < count) {
      const Entry m = cand[tid];
      int rank = 0;
      for (int i = 0; i < count; ++i)
        rank += before(cand[i].x, cand[i].at, m.x, m.at);
      if (rank < n) out[rank] = m;
    }
    return;
  }
  // Many equal logits: one after the other, the best of what comes after the
  // last.
  Entry last = {__builtin_inff(), -1};
  for (int k = 0; k < n; ++k) {
    Entry best = {kNegInf, 0x7fffffff};
    s.again([&](float x, int i) {
      if (before(last.x, last.at, x, i) && before(x, i, best.x, best.at))
        best = Entry{x, i};
    });
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const Entry q = {__shfl_xor(best.x, o), __shfl_xor(best.at, o)};
      if (before(q.x, q.at, best.x, best.at)) best = q;
    }
    __syncthreads();
    if (lane == 0) cand[wave] = best;
    __syncthreads();
    best = cand[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
      if (before(cand[w].x, cand[w].at, best.x, best.at)) best = cand[w];
    if (tid == 0) out[k] = best;
    last = best;
  }
}

// A position's parts; a workgroup each.
constexpr int kJoin = 1024;  // candidates at a time

template <int DT, bool kTop>
__global__ __launch_bounds__(kThreads) void k_logprobs_join(LogArgs a) {
  using T = typename Elem<DT>::T;
  const int64_t pos = blockIdx.x;
  const int64_t b = pos / a.v.positions, j = pos % a.v.positions;
  const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
  const int n = (int)a.v.top;
  const int32_t tok = a.v.tokens[pos];
  const bool given = tok >= 0 && tok < a.v.vocab;
  __shared__ Part lds[kWaves];
  __shared__ Entry cand[kTop ? kJoin : 1];
  if (!given) {
    if (tid == 0) {
      a.v.logprob[pos] = 0.0f;
      a.v.entropy[pos] = 0.0f;
    }
    if (kTop && tid < n) {
      a.v.top_tokens[pos * n + tid] = -1;
      a.v.top_logprobs[pos * n + tid] = kNegInf;
    }
    return;
  }
  const float t = temperature_of(a.v, b);
  const bool greedy = !(t > 0.0f);
  const float c = greedy ? 0.0f : scale_of(t);
  Part p = {kNegInf, 0.0f, 0.0f, 0x7fffffff};
  for (int i = tid; i < a.chunks; i += kThreads)
    join(p, a.part[pos * a.chunks + i], c);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const Part q = {__shfl_xor(p.top, o), __shfl_xor(p.rest, o),
                    __shfl_xor(p.zsum, o), __shfl_xor(p.at, o)};
    join(p, q, c);
  }
  if (lane == 0) lds[wave] = p;
  __syncthreads();
  p = lds[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) join(p, lds[w], c);
  const float log_sum = greedy ? 0.0f : log1pf(p.rest);
  auto log_p = [&](float x, int i) {
    if (!(x > kNegInf)) return kNegInf;
    if (greedy) return i == p.at ? 0.0f : kNegInf;
    return 2.0f * (half_below(x, p.top) / t) - log_sum;
  };
  if (tid == 0) {
    const T* row =
        (const T*)a.v.logits + b * a.v.stride_b + j * a.v.stride_j;
    a.v.logprob[pos] = log_p(Elem<DT>::get(row[tok]), tok);
    const bool some = p.top > kNegInf && !greedy;
    a.v.entropy[pos] =
        some ? log_sum - p.zsum * kLn2 / (1.0f + p.rest) : 0.0f;
  }
  if (!kTop) return;
  // The best of the parts' lists, kJoin candidates at a time behind the best of
  // those before.
  const Entry* in = a.entry + pos * a.chunks * n;
  const int all = a.chunks * n;
  int kept = 0;
  for (int i0 = 0; i0 < all;) {
    const int take = min(kJoin - kept, all - i0);
    for (int i = tid; i < take; i += kThreads) cand[kept + i] = in[i0 + i];
    __syncthreads();
    i0 += take;
    const int count = kept + take;
    Entry mine[kJoin / kThreads];
    int rank[kJoin / kThreads];
#pragma unroll
    for (int k = 0; k < kJoin / kThreads; ++k) {
      const int i = k * kThreads + tid;
      rank[k] = n;
      if (i < count) {
        mine[k] = cand[i];
        rank[k] = 0;
        for (int q = 0; q < count; ++q)
          rank[k] += before(cand[q].x, cand[q].at, mine[k].x, mine[k].at);
      }
    }
    __syncthreads();
    if (tid < n) cand[tid] = Entry{kNegInf, -1};
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kJoin / kThreads; ++k)
      if (rank[k] < n && mine[k].at >= 0) cand[rank[k]] = mine[k];
    __syncthreads();
    kept = min(n, count);
  }
  if (tid < n) {
    const Entry e = cand[tid];
    const bool there = e.at >= 0;
    a.v.top_tokens[pos * n + tid] = e.at;
    a.v.top_logprobs[pos * n + tid] = there ? log_p(e.x, e.at) : kNegInf;
  }
}

int chunks_for(int64_t vocab) {
  return (int)((vocab + kChunk - 1) / kChunk);
}

size_t round_up(size_t x) { return (x + 255) & ~(size_t)255; }

size_t part_bytes(int64_t rows, int64_t vocab) {
  return round_up((size_t)rows * chunks_for(vocab) * sizeof(Part));
}

size_t bytes_for(int64_t rows, int64_t vocab, int64_t top) {
  return part_bytes(rows, vocab) +
         (size_t)rows * chunks_for(vocab) * top * sizeof(Entry);
}

bool sizes_ok(int64_t batch, int64_t positions, int64_t vocab, int64_t top) {
  // the grid's limit is 2^32 threads
  return batch >= 0 && positions >= 0 && vocab >= 1 &&
         vocab <= (int64_t(1) << 28) && top >= 0 && top <= SFX_LOGPROBS_TOP &&
         batch <= (1 << 23) && positions <= (1 << 23) &&
         batch * positions <= (1 << 23) / chunks_for(vocab);
}

template <int DT, bool kTop>
int launch_as(const LogArgs& a, hipStream_t stream) {
  const int64_t rows = a.v.batch * a.v.positions;
  hipLaunchKernelGGL((k_logprobs_scan<DT, kTop>),
                     dim3((unsigned)(rows * a.chunks)), dim3(kThreads), 0,
                     stream, a);
  hipLaunchKernelGGL((k_logprobs_join<DT, kTop>), dim3((unsigned)rows),
                     dim3(kThreads), 0, stream, a);
  return (int)hipGetLastError();
}

template <int DT>
int launch(const LogArgs& a, hipStream_t stream) {
  return a.v.top ? launch_as<DT, true>(a, stream)
                 : launch_as<DT, false>(a, stream);
}

}  // namespace

}  // namespace sfx

using namespace sfx;

extern "C" size_t sfx_logprobs_workspace_size(int64_t batch, int64_t positions,
                                              int64_t vocab, int64_t top) {
  if (!sizes_ok(batch, positions, vocab, top) || batch * positions == 0)
    return 0;
  return bytes_for(batch * positions, vocab, top);
}

extern "C" int sfx_token_logprobs(const sfx_logprobs* args, void* workspace,
                                  size_t workspace_bytes, hipStream_t stream) {
  if (!args) return SFX_EINVAL;
  LogArgs a;
  a.v = *args;
  const sfx_logprobs& v = a.v;
  if (!sizes_ok(v.batch, v.positions, v.vocab, v.top) ||
      (v.dtype != SFX_BF16 && v.dtype != SFX_F16 && v.dtype != SFX_F32))
    return SFX_EINVAL;
  const int64_t rows = v.batch * v.positions;
  if (rows == 0) return 0;
  if (!v.logits || !v.tokens || !v.logprob || !v.entropy ||
      (v.top && (!v.top_tokens || !v.top_logprobs)))
    return SFX_EINVAL;
  if (!workspace || ((uintptr_t)workspace & 15) ||
      workspace_bytes < bytes_for(rows, v.vocab, v.top))
    return SFX_EINVAL;
  a.chunks = chunks_for(v.vocab);
  a.part = (Part*)workspace;
  a.entry = (Entry*)((char*)workspace + part_bytes(rows, v.vocab));
  switch (v.dtype) {
    case SFX_BF16: return launch<SFX_BF16>(a, stream);
    case SFX_F16: return launch<SFX_F16>(a, stream);
    default: return launch<SFX_F32>(a, stream);
  }
}
