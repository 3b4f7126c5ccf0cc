// Log probabilities of given tokens, the entropy of their distributions, and the
// likeliest alternatives, in one pass over the logits.
//
// With z_i = (x_i - max x) / T and R the sum of e^z over all but one of the
// largest (a token is often nearly certain: what the others add to one is then
// all of its log probability, and would be lost beside the one),
//   log p_i = z_i - log(1 + R),   H = log(1 + R) - sum z e^z / (1 + R).
//
// The first launch takes 8,192 logits a workgroup, which stay in registers: their
// largest, R and sum z e^z, and what reaches a number that n of the maxima of its
// 128 parts reach, and few more: the n largest, and few others.  The second launch
// joins a position's parts and ranks what is left of those.
// Positions without a token leave at once.
//
// Memory bounds it where there are no alternatives: 2,048 positions of 128,256
// bfloat16 logits take 96 to 103 us, 5.1 to 5.5 TB/s; float32 logits also with a few
// (64 x 17 positions with five 105 us, 5.3 TB/s).  With alternatives it is the
// vector instructions, 16 a logit with one (112 to 125 us) and 18 with twenty: 256
// positions 28.5 us, 66 MB at 2.3 TB/s, 19 without any.  8,192 logits a workgroup are 32 a
// lane, which is what stays in registers beside the rest with seven or eight waves a
// SIMD.  One position of 32,000 is the latency of the two launches (5.2 + 4.2 us).

#include <algorithm>

#include "launch.h"
#include "vocab.h"

namespace sfx {

namespace {

constexpr int kWaves = kThreads / kWave;
constexpr float kMaxScale = 0x1.fffffep126f;
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
  Entry* entry;  // [batch * positions, chunks, top + kSpare]
};

__device__ __forceinline__ float temperature_of(const sfx_logprobs& v,
                                                int64_t b) {
  const float t = v.temperature ? v.temperature[b] : 1.0f;
  return t > 0.0f ? t : 0.0f;
}

// A value of another lane of the row of 16.
template <int kCtrl>
__device__ __forceinline__ float lane_of(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), kCtrl, 0xf,
                                      0xf, true));
}

// Half the difference to the largest, which is a float where the difference is
// too large for one; 0 where infinities meet.
__device__ __forceinline__ float half_below(float x, float top) {
  return x == top ? 0.0f : __builtin_fmaf(x, 0.5f, -0.5f * top);
}

// Base-2 scale of a difference; twice that of a half is a float too.
__device__ __forceinline__ float scale_of(float t) {
  return fminf(kLog2e / t, kMaxScale);
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
  const float d = fmaxf(half_below(b.top, a.top) * (2.0f * c), kFloor);
  const float f = __builtin_amdgcn_exp2f(d);
  p.top = a.top;
  p.rest = a.rest + (1.0f + b.rest) * f;
  p.zsum = a.zsum + (b.zsum + d * (1.0f + b.rest)) * f;
  p.at = a.top == b.top ? min(a.at, b.at) : a.at;
}

// Order of floats as unsigned numbers.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u >> 31 ? ~u : u | 0x80000000u;
}

// Place of the lane's entry among those of lanes 0 .. count - 1.
__device__ __forceinline__ int place_of(const Entry& m, int count) {
  int r = 0;
#pragma unroll 4
  for (int i = 0; i < count; ++i) {
    const float y = __builtin_bit_cast(
        float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, m.x), i));
    r += before(y, __builtin_amdgcn_readlane(m.at, i), m.x, m.at);
  }
  return r;
}

// The next float.
__device__ __forceinline__ float next_above(float x) {
  const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
  return __uint_as_float(u >> 31 ? u - 1 : u + 1);
}

// A number that n (at most 64) of a wave's 128 numbers x, y reach, and few more: by
// halves, until no more than n + kFew do.  Of those that are the largest of groups
// of others, what reaches it is n and few more too: 45 of 8,192 random ones with n = 32
// (of 64 groups 58, and then and when more than the 64 that a wave ranks).
constexpr int kFew = 6;
constexpr int kSpare = 8;  // entries of a list beside the n, which are in no order

__device__ __forceinline__ float reached_by(float x, float y, int n) {
  const uint32_t k0 = order_of(x), k1 = order_of(y);
  const uint32_t hi = wave_all_max(max(k0, k1)), lo = ~wave_all_max(~min(k0, k1));
  int bit = 31 - __builtin_clz((hi ^ lo) | 1u);
  uint32_t line = lo >> bit >> 1 << bit << 1;
  for (; bit >= 0; --bit) {
    const uint32_t to = line | 1u << bit;
    const int count = popc(ballot(k0 >= to)) + popc(ballot(k1 >= to));
    if (count >= n) {
      line = to;
      if (count <= n + kFew) break;
    }
  }
  // (below -inf where all are taken; the line may lie between two floats)
  line = max(line, order_of(kNegInf));
  return __uint_as_float(line >> 31 ? line & 0x7fffffffu : ~line);
}

template <int DT, bool kTop>
__global__ __launch_bounds__(kThreads) void k_logprobs_scan(LogArgs a) {
  using S = Share<DT>;
  constexpr int E = S::E, U = S::U;
  static_assert(kThreads / 2 == 2 * kWave && kWave >= SFX_LOGPROBS_TOP, "");
  const int chunk = blockIdx.x % a.chunks;
  const int64_t pos = blockIdx.x / a.chunks;
  const int64_t b = pos / a.v.positions, j = pos % a.v.positions;
  const int32_t tok = a.v.tokens[pos];
  if (tok < 0 || tok >= a.v.vocab) return;
  const int tid = threadIdx.x, wave = tid / kWave, lane = lane_id();
  __shared__ Part lds[kWaves];
  __shared__ float group[kTop ? 2 * kWave : 1];  // maxima of two threads' logits
  __shared__ float lds_line;
  __shared__ Entry cand[kTop ? kWaves : 1][kWave];
  __shared__ int counts[kWaves], ties[1 + U][kWaves];
  const float t = temperature_of(a.v, b);
  const bool greedy = !(t > 0.0f);
  const float c = greedy ? 0.0f : scale_of(t);
  const typename S::T* row = (const typename S::T*)a.v.logits +
                             b * a.v.stride_b + j * a.v.stride_j;
  S s(row, a.v.vocab, chunk);
  s.load(row);
  // The logits as floats, once; the largest of each vector, of the thread, of the
  // wave.
  float x[U][E], vtop[U], top = fmaxf(s.single, kNegInf);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    vtop[u] = kNegInf;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      x[u][e] = s.get(u, e);
      vtop[u] = fmaxf(vtop[u], x[u][e]);
    }
    top = fmaxf(top, vtop[u]);
  }
  const float mine = top;
  top = wave_max(top);
  if (kTop) {
    const float m = fmaxf(mine, lane_of<0xb1>(mine));  // lane ^ 1
    if (lane % 2 == 0) group[tid / 2] = m;
  }
  Part p = {top, 0.0f, 0.0f, 0x7fffffff};
  if (greedy) {
    if (mine == top && top > kNegInf) {
      int at = 0x7fffffff;
      s.again([&](float y, int i) { at = y == top ? min(at, i) : at; });
      p.at = at;
    }
    p.at = wave_min(p.at);
  } else if (top > kNegInf) {
    // z = x c - top c in one step, with top c rounded; what that is off, the same
    // for all, is put right in the sums.
    if (kTop && DT != SFX_F32) {
      // unpacked again where they are used: kept as floats they would cost the
      // kernel that also ranks a wave in eight
      if (DT == SFX_F16) s.forget();
      const typename S::Anew anew;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = s.get(u, e, anew);
    }
    const float tc = top * c, off = __builtin_fmaf(top, c, -tc);
    float sum = 0.0f, zsum = 0.0f;
    int equal = 0;
    auto add = [&](float z) {
      z = fmaxf(z, kFloor);
      const float e = __builtin_amdgcn_exp2f(z);
      sum += e;
      zsum = __builtin_fmaf(z, e, zsum);
    };
    auto take = [&](auto z_of) {
      auto add_special = [&](float y) {
        equal += popc(ballot(y == top));
        add(y == top ? kFloor : z_of(y));
      };
      if (ballot(s.extra >= 0)) add_special(s.single);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // one vector in U holds the wave's largest
        if (ballot(vtop[u] == top)) {
#pragma unroll
          for (int e = 0; e < E; ++e) add_special(x[u][e]);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) add(z_of(x[u][e]));
        }
      }
    };
    if (fabsf(tc) < 0x1p24f && c < 0x1p60f) {  // (off is at most a half)
      take([&](float y) { return __builtin_fmaf(y, c, -tc); });
      sum = wave_sum(sum);
      zsum = wave_sum(zsum);
      const float f = __builtin_amdgcn_exp2f(-off);
      zsum = (zsum - off * sum) * f;
      sum *= f;
    } else {
      // infinities, and what grows too large: a difference first, by halves.  (From
      // |top c| = 2^32 on 2^-off can be no float, with sums of zero a NaN.)
      const float half = -0.5f * top, c2 = 2.0f * c;
      s.again([&](float y, int) {
        const bool is = y == top;
        equal += is;
        add(is ? kFloor : __builtin_fmaf(y, 0.5f, half) * c2);
      });
      sum = wave_sum(sum);
      zsum = wave_sum(zsum);
      equal = (int)wave_sum((float)equal);
    }
    p.rest = sum + ((float)equal - 1.0f);
    p.zsum = zsum;
  }
  if (lane == 0) lds[wave] = p;
  __syncthreads();
  const int n = (int)a.v.top;
  if (kTop && wave == 1) {
    // what n groups' maxima reach, so at least n logits, and few more
    const float y = reached_by(group[lane], group[lane + kWave], n);
    if (lane == 0) lds_line = y;
  }
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kWaves; ++w) join(p, lds[w], c);
    a.part[pos * a.chunks + chunk] = p;
  }
  if (!kTop) return;
  if (DT == SFX_F16) s.forget();
  const typename S::Anew anew;
  __syncthreads();
  float line = lds_line;
  int count = 0, all;
  auto offer = [&](float y, int i, bool in) {
    const bool is = in && y >= line && y > kNegInf;
    const uint64_t m = ballot(is);
    const int k = count + rank_lt(m);
    if (is && k < kWave) cand[wave][k] = Entry{y, i};
    count += popc(m);
  };
  // whether a wave can rank what was offered
  auto offered = [&]() {
    if (lane == 0) counts[wave] = count;
    __syncthreads();
    all = 0;
    bool fits = true;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      fits = fits && counts[w] <= kWave;
      all += counts[w];
    }
    return fits && all <= kWave;
  };
  if (ballot(s.extra >= 0)) offer(s.single, s.extra, s.extra >= 0);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (ballot(vtop[u] >= line)) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (ballot(s.get(u, e, anew) >= line))
          offer(s.get(u, e, anew), s.index(u * E + e), true);
    }
  }
  const int room = n + kSpare;
  Entry* out = a.entry + (pos * a.chunks + chunk) * room;
  bool fits = offered();
  if (!fits && line > kNegInf) {
    // Many are equal to the line: what lies past it, and the first of these.  (256
    // positions of one value, twenty alternatives: 81 us, one after the other 274.)
    const float tie = line;
    line = next_above(line);
    __syncthreads();
    count = 0;
    offer(s.single, s.extra, s.extra >= 0);
#pragma unroll 1
    for (int u = 0; u < U; ++u) s.again_step(u, offer);
    fits = offered();
    if (fits && all < n) {
      // in the order of their indices: single ones before the vectors (all of
      // them a wave's), the vectors of each step, wave by wave, single ones
      const bool equal = s.extra >= 0 && s.single == tie;
      const uint64_t heads = ballot(equal && s.extra < s.head);
      const uint64_t tails = ballot(equal && s.extra >= s.head);
      const int need = n - all;
      auto equals = [&](int u) {
        uint32_t c = 0;
        s.again_step(u, [&](float y, int, bool in) { c += in && y == tie; });
        return c;
      };
#pragma unroll 1
      for (int u = 0; u < U; ++u) {
        const uint32_t to = wave_incl_scan(equals(u));
        if (lane == kWave - 1) ties[1 + u][wave] = (int)to;
      }
      if (lane == 0) ties[0][wave] = popc(heads);
      __syncthreads();
      line = tie;
      int before_it = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) before_it += ties[0][w];
      offer(s.single, s.extra, (heads >> lane & 1) && rank_lt(heads) < need);
#pragma unroll 1
      for (int u = 0; u < U; ++u) {
        int k = before_it;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          if (w < wave) k += ties[1 + u][w];
          before_it += ties[1 + u][w];
        }
        if (k >= need) continue;
        const uint32_t c = equals(u);
        k += (int)(wave_incl_scan(c) - c);
        s.again_step(u, [&](float y, int i, bool in) {
          const bool is = in && y == tie;
          offer(y, i, is && k < need);
          k += is;
        });
      }
      offer(s.single, s.extra,
            (tails >> lane & 1) && before_it + rank_lt(tails) < need);
      fits = offered();
    }
  }
  if (fits) {
    if (wave > 0) return;
    int w = 0, i = lane;
#pragma unroll
    for (int v = 0; v + 1 < kWaves; ++v)
      if (w == v && i >= counts[v]) {
        i -= counts[v];
        ++w;
      }
    Entry m = {kNegInf, -1};
    if (lane < all) m = cand[w][i];
    if (all <= room) {
      if (lane < room) out[lane] = m;
      return;
    }
    const int r = place_of(m, all);
    if (lane < all && r < n) out[r] = m;
    if (lane >= n && lane < room) out[lane] = Entry{kNegInf, -1};
    return;
  }
  if (tid >= n && tid < room) out[tid] = Entry{kNegInf, -1};
  // Many logits of few groups: one after the other, the best of what comes after
  // the last.
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
    if (lane == 0) cand[wave][0] = best;
    __syncthreads();
    best = cand[0][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w)
      if (before(cand[w][0].x, cand[w][0].at, best.x, best.at))
        best = cand[w][0];
    if (tid == 0) out[k] = best;
    last = best;
  }
}

// A position's parts, by a wave.
//
// Its n largest logits are among the entries of the parts' lists.  They reach what
// n of the largest of the lanes' halves reach, and few others do.
constexpr int kHeld = 8;  // entries a lane keeps; of more all are read again

template <int DT, bool kTop>
__global__ __launch_bounds__(kThreads) void k_logprobs_join(LogArgs a) {
  using T = typename Elem<DT>::T;
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const int64_t pos = (int64_t)blockIdx.x * kWaves + wave;
  if (pos >= a.v.batch * a.v.positions) return;  // (no barriers below)
  const int64_t b = pos / a.v.positions, j = pos % a.v.positions;
  const int n = (int)a.v.top;
  const int32_t tok = a.v.tokens[pos];
  const bool given = tok >= 0 && tok < a.v.vocab;
  if (!given) {
    if (lane == 0) {
      a.v.logprob[pos] = 0.0f;
      a.v.entropy[pos] = 0.0f;
    }
    if (kTop && lane < n) {
      a.v.top_tokens[pos * n + lane] = -1;
      a.v.top_logprobs[pos * n + lane] = kNegInf;
    }
    return;
  }
  const int lists = a.chunks;
  const int all = lists * (n + kSpare);
  const Entry* in = a.entry + pos * all;
  auto entry = [&](int i) {
    return kTop && i < all ? in[i] : Entry{kNegInf, -1};
  };
  Entry held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = entry(i * kWave + lane);
  const T* row = (const T*)a.v.logits + b * a.v.stride_b + j * a.v.stride_j;
  const float x = Elem<DT>::get(row[tok]);
  const float t = temperature_of(a.v, b);
  const bool greedy = !(t > 0.0f);
  const float c = greedy ? 0.0f : scale_of(t);
  Part p = {kNegInf, 0.0f, 0.0f, 0x7fffffff};
  for (int i = lane; i < lists; i += kWave) {
    const Part part = a.part[pos * lists + i];
    if (i == lane)
      p = part;
    else
      join(p, part, c);
  }
  // One lane's largest is the position's: R is without it.
  const float top = wave_max(p.top);
  p.at = wave_min(p.top == top ? p.at : 0x7fffffff);
  const int owner = __builtin_ctzll(ballot(p.top == top));
  const float d = fmaxf(half_below(p.top, top) * (2.0f * c), kFloor);
  const float f = p.top == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(d);
  const float rest =
      wave_sum(lane == owner ? p.rest : (1.0f + p.rest) * f);
  const float zsum = wave_sum((p.zsum + d * (1.0f + p.rest)) * f);
  const float log_sum = greedy ? 0.0f : log1pf(rest);
  auto log_p = [&](float y, int i) {
    if (!(y > kNegInf)) return kNegInf;
    if (greedy) return i == p.at ? 0.0f : kNegInf;
    return 2.0f * (half_below(y, top) / t) - log_sum;
  };
  if (lane == 0) {
    a.v.logprob[pos] = log_p(x, tok);
    const bool some = top > kNegInf && !greedy;
    a.v.entropy[pos] = some ? log_sum - zsum * kLn2 / (1.0f + rest) : 0.0f;
  }
  if (!kTop) return;

  float most[2] = {held[0].x, held[1].x};
#pragma unroll
  for (int i = 2; i < kHeld; ++i) most[i % 2] = fmaxf(most[i % 2], held[i].x);
  for (int i0 = kHeld * kWave; i0 < all; i0 += 2 * kWave) {
    most[0] = fmaxf(most[0], entry(i0 + lane).x);
    most[1] = fmaxf(most[1], entry(i0 + kWave + lane).x);
  }
  const float line = reached_by(most[0], most[1], n);
  __shared__ Entry kept[kWaves][kWave];
  int count = 0;
  auto keep = [&](const Entry& y, bool in) {
    const bool is = in && y.at >= 0;
    const uint64_t m = ballot(is);
    const int at = count + rank_lt(m);
    if (is && at < kWave) kept[wave][at] = y;
    count += popc(m);
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (i * kWave < all) keep(held[i], held[i].x >= line);
  for (int i0 = kHeld * kWave; i0 < all; i0 += kWave) {
    const Entry y = entry(i0 + lane);
    keep(y, y.x >= line);
  }
  if (count > kWave && line > kNegInf) {
    // Many are equal to the line: those past it, and the first of these.
    auto each = [&](auto f) {
#pragma unroll 1
      for (int i0 = 0; i0 < all; i0 += kWave) f(entry(i0 + lane));
    };
    const float past = next_above(line);
    wave_lds_sync();
    count = 0;
    each([&](const Entry& y) { keep(y, y.x >= past); });
    if (count < n) {
      // the one with as many before it as are missing (indices are below 2^28)
      const int need = n - count;
      int last = 0;
#pragma unroll 1
      for (int bit = 27; bit >= 0; --bit) {
        int c = 0;
        each([&](const Entry& y) {
          c += popc(ballot(y.at >= 0 && y.x == line &&
                           y.at < last + (1 << bit)));
        });
        if (c < need) last += 1 << bit;
      }
      each([&](const Entry& y) { keep(y, y.x == line && y.at <= last); });
    }
  }
  wave_lds_sync();
  Entry best = {kNegInf, -1};  // lane k: the k-th
  if (count <= kWave) {
    Entry mine = {kNegInf, 0x7fffffff};
    if (lane < count) mine = kept[wave][lane];
    const int r = place_of(mine, count);
    wave_lds_sync();
    if (lane < count && r < n) kept[wave][r] = mine;
    wave_lds_sync();
    if (lane < min(n, count)) best = kept[wave][lane];
  } else {
    // Many in few of the halves: one after the other, the first behind the last.
    Entry last = {__builtin_inff(), -1};
    for (int k = 0; k < n; ++k) {
      Entry y = {kNegInf, 0x7fffffff};
      for (int i = lane; i < all; i += kWave) {
        const Entry e = in[i];
        if (e.at >= 0 && before(last.x, last.at, e.x, e.at) &&
            before(e.x, e.at, y.x, y.at))
          y = e;
      }
      last.x = wave_max(y.x);
      last.at = wave_min(y.x == last.x ? y.at : 0x7fffffff);
      if (lane == k) best = last;
    }
  }
  if (lane < n) {
    a.v.top_tokens[pos * n + lane] = best.at;
    a.v.top_logprobs[pos * n + lane] =
        best.at >= 0 ? log_p(best.x, best.at) : kNegInf;
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
         (top ? (size_t)rows * chunks_for(vocab) * (top + kSpare) * sizeof(Entry)
              : 0);
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
  hipLaunchKernelGGL((k_logprobs_join<DT, kTop>),
                     dim3((unsigned)((rows + kWaves - 1) / kWaves)),
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
