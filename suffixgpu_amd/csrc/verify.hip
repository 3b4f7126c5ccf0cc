// Verification of drafted tokens against the target model's logits.
//
// A draft d at position j stays iff u q(d) < p_j(d), p_j = softmax(x / T); the
// token after the accepted ones is drawn from r = max(p_j - q, 0) (or p_j) as
// argmax_i r_i / e_i with e_i exponentially distributed: the smallest of
// exponential clocks of rates r_i rings with probability r_i / sum r.  A draw
// by clocks needs no running sum over the vocabulary, whose rounding would
// decide between neighbours, and its argmax is the same in any order.
//
// Two launches.  k_verify_scan takes the largest logit and the sum of
// exponentials of a drafted position, a workgroup per 8,192 logits, and a
// workgroup that finds all parts of its position there decides the draft.  The
// grid runs position by position over all rows, and a workgroup whose row has
// rejected an earlier draft leaves at once: of a draft of 16 with three kept,
// most of the logits are never read.  None waits for a decision, so how much is
// read in vain depends on timing; the result does not, since every position up
// to the first rejected one is complete.
// k_verify_draw races the candidates of the position that the row stopped at, a
// workgroup per 8,192, and the row's last one writes the result.
//
// What bounds them (drafts of 16 over 128,256 bfloat16 logits, of which two are
// kept on average): 64 rows take 33 + 14 us and read 84 + 37 MB, of which 45 + 37
// were needed; 256 greedy rows 107 + 7 us and read 331 MB of 191.  At the 4.0
// TB/s at which such a stream is read that would be 30 and 83 us; the rest are
// the workgroups that leave, some 0.4 ns each by the launch's rate, and the last
// positions, of which few rows are left.  One row of 32,000 float32 logits takes
// 5.6 + 6.9 us, of loads that depend on each other.  Measured beside it and
// slower: workgroups that walk a list of what is left (51 us for 64 rows of the
// first kind, 130 for 256 greedy, against 47 and 123 at the time), that load
// the next item ahead (spills), or that take several of the later positions in
// turn (50 and 120); 16,384 logits a workgroup 51 and 115.

#include <algorithm>

#include "launch.h"
#include "sfx_common.h"

namespace sfx {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kChunk = 8192;  // logits per workgroup
constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMaxScale = 1e30f;
// Words between the stops of two rows.  Every workgroup looks at one, past the
// XCDs' caches; with those of 64 rows side by side in two lines, all of them
// waited for those lines (64 drafts of 16, rejected at once: 45 us, not 22).
constexpr int kStopPitch = 64;

// What is known of a position, or of a chunk of it: largest logit, and the sum
// of 2^((x - top) c), or, of a greedy row, one more than the first index of the
// largest.  Never all zero bits: a sum is at least 1, or top is -inf.
struct Stat {
  float top;
  union {
    float sum;
    int32_t at1;
  };
};

__device__ __forceinline__ void put(Stat* p, Stat r) {
  __hip_atomic_store((uint64_t*)p, __builtin_bit_cast(uint64_t, r),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Stat take(const Stat* p) {
  return __builtin_bit_cast(
      Stat, __hip_atomic_load((uint64_t*)p, __ATOMIC_RELAXED,
                              __HIP_MEMORY_SCOPE_AGENT));
}

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
  // zero when a call starts and when it ends
  Stat* part;         // [batch, K + 1, chunks]
  unsigned* arrived;  // [batch] workgroups of the draw
  unsigned* stop;     // [batch, kStopPitch] K + 1 - (a rejected position), 0:
                      // none yet
  // anything
  Stat* stat;         // [batch, K + 1]
  Best* best;         // [batch, chunks]
};

template <int DT>
struct Elem;
template <>
struct Elem<SFX_BF16> {
  using T = uint16_t;
  static constexpr uint32_t kMinusInf = 0xff80ff80u;
  static __device__ float get(T x) { return __uint_as_float((uint32_t)x << 16); }
};
template <>
struct Elem<SFX_F16> {
  using T = uint16_t;
  static constexpr uint32_t kMinusInf = 0xfc00fc00u;
  static __device__ float get(T x) {
    return (float)__builtin_bit_cast(_Float16, x);
  }
};
template <>
struct Elem<SFX_F32> {
  using T = float;
  static constexpr uint32_t kMinusInf = 0xff800000u;
  static __device__ float get(T x) { return x; }
};

// A thread's share of chunk c of a row of n elements of any alignment: step u
// is E elements from a 16-byte aligned address.  The up to E - 1 elements before
// the first such address, and those after the last whole vector, are one
// element each of some threads of chunk 0.
template <int DT>
struct Share {
  using T = typename Elem<DT>::T;
  static constexpr int E = 16 / sizeof(T);
  static constexpr int U = kChunk / (kThreads * E);
  const T* body;
  int head;   // elements before the body
  int vecs;   // vectors of the body
  int first;  // the thread's vector of step 0
  int extra;  // index of its single element, or -1
  // The elements as they lie in memory: half the registers of floats where
  // they have 16 bits.
  uint4 w[U];
  float single;
  __device__ Share(const T* row, int64_t len, int chunk) {
    const int n = (int)len, tid = (int)threadIdx.x;
    head = (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T);
    head = head < n ? head : n;
    body = row + head;
    vecs = (n - head) / E;
    first = chunk * kThreads * U + tid;
    const int tail = head + vecs * E;
    extra = -1;
    if (chunk == 0 && tid < 2 * E) {
      if (tid < E)
        extra = tid < head ? tid : -1;
      else
        extra = tail + tid - E < n ? tail + tid - E : -1;
    }
  }
  // Where a thread's element e of step u lies, by place = u E + e; its single
  // element comes last.  Places are constants of the unrolled loops where
  // indices would take a register each.
  static constexpr int kSingle = U * E;
  __device__ int index(int place) const {
    return place == kSingle ? extra
                            : head + (first + place / E * kThreads) * E +
                                  place % E;
  }
  __device__ int place_of(int i) const {
    if (i < 0) return -1;
    if (i == extra) return kSingle;
    const int at = i - head;
    if (at < 0 || at >= vecs * E) return -1;
    const int v = at / E - first;
    return v >= 0 && v % kThreads == 0 && v / kThreads < U
               ? v / kThreads * E + at % E
               : -1;
  }
  // Every load is issued before any is used.  Outside the row: -inf.
  __device__ void load(const T* row) {
    constexpr uint32_t kM = Elem<DT>::kMinusInf;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = uint4{kM, kM, kM, kM};
      const int v = first + u * kThreads;
      if (v < vecs) w[u] = ((const uint4*)body)[v];
    }
    single = extra >= 0 ? Elem<DT>::get(row[extra]) : kNegInf;
  }
  __device__ float get(int u, int e) const {
    const uint32_t q[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
    if (DT == SFX_F32) return __uint_as_float(q[e]);
    const uint32_t x = q[e / 2];
    if (DT == SFX_BF16)
      return __uint_as_float(e % 2 ? x & 0xffff0000u : x << 16);
    return (float)__builtin_bit_cast(_Float16,
                                     (uint16_t)(e % 2 ? x >> 16 : x));
  }
  // The compiler shall unpack the elements again where they are next used: the
  // floats of two uses would not fit beside each other.
  __device__ void forget() {
#pragma unroll
    for (int u = 0; u < U; ++u)
      asm volatile("" : "+v"(w[u].x), "+v"(w[u].y), "+v"(w[u].z), "+v"(w[u].w));
  }
  // f(x, index) over the elements once more, from memory: for what happens
  // rarely and shall cost the usual loops no registers.
  template <class F>
  __device__ void again(F f) const {
#pragma unroll 1
    for (int u = 0; u < U; ++u) {
      const int v = first + u * kThreads;
      if (v >= vecs) break;
      T x[E];
      const uint4 q = ((const uint4*)body)[v];
      __builtin_memcpy(x, &q, 16);
#pragma unroll
      for (int e = 0; e < E; ++e) f(Elem<DT>::get(x[e]), head + v * E + e);
    }
    if (extra >= 0) f(single, extra);
  }
};

// Floats at the elements of a share's step, any alignment; 1 outside the row.
typedef float F4Any __attribute__((ext_vector_type(4), aligned(4)));
template <int E>
__device__ __forceinline__ void load_floats(const float* p, bool in,
                                            float (&x)[E]) {
#pragma unroll
  for (int k = 0; k < E; k += 4) {
    F4Any w = {1.0f, 1.0f, 1.0f, 1.0f};
    if (in) w = *(const F4Any*)(p + k);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[k + e] = w[e];
  }
}

// Difference to the largest, where infinities may meet; -inf for NaN.
__device__ __forceinline__ float below(float x, float top) {
  return x == top ? 0.0f : fmaxf(x - top, kNegInf);
}

// One step of a reduction over a wave's lanes by row shifts and broadcasts;
// lanes without a source keep `old`.
template <int kCtrl, int kRows>
__device__ __forceinline__ float dpp(float old, float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old),
                                         __builtin_bit_cast(int, x), kCtrl,
                                         kRows, 0xf, false));
}

__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<0x111, 0xf>(v, v));
  v = fmaxf(v, dpp<0x112, 0xf>(v, v));
  v = fmaxf(v, dpp<0x114, 0xf>(v, v));
  v = fmaxf(v, dpp<0x118, 0xf>(v, v));
  v = fmaxf(v, dpp<0x142, 0xa>(v, v));
  v = fmaxf(v, dpp<0x143, 0xc>(v, v));
  return __builtin_bit_cast(
      float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

__device__ __forceinline__ float wave_sum(float v) {
  v += dpp<0x111, 0xf>(0.0f, v);
  v += dpp<0x112, 0xf>(0.0f, v);
  v += dpp<0x114, 0xf>(0.0f, v);
  v += dpp<0x118, 0xf>(0.0f, v);
  v += dpp<0x142, 0xa>(0.0f, v);
  v += dpp<0x143, 0xc>(0.0f, v);
  return __builtin_bit_cast(
      float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

template <int kCtrl, int kRows>
__device__ __forceinline__ int dpp_min(int v) {
  return min(v, __builtin_amdgcn_update_dpp(v, v, kCtrl, kRows, 0xf, false));
}

__device__ __forceinline__ int wave_min(int v) {
  v = dpp_min<0x111, 0xf>(v);
  v = dpp_min<0x112, 0xf>(v);
  v = dpp_min<0x114, 0xf>(v);
  v = dpp_min<0x118, 0xf>(v);
  v = dpp_min<0x142, 0xa>(v);
  v = dpp_min<0x143, 0xc>(v);
  return __builtin_amdgcn_readlane(v, 63);
}

__device__ __forceinline__ float block_max(float v, float* lds) {
  v = wave_max(v);
  __syncthreads();
  if (lane_id() == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v = fmaxf(v, lds[w]);
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
// first id that is no token.  By a whole wave, the first 64 ids loaded beside
// num_valid.
__device__ __forceinline__ int drafts_of(const sfx_verify& v, int64_t b) {
  const int K = (int)v.k;
  int32_t d = lane_id() < K ? v.draft[b * K + lane_id()] : 0;
  int n = v.num_valid[b];
  n = n < 0 ? 0 : (n > K ? K : n);
  for (int i0 = 0; i0 < n; i0 += kWave) {
    const int i = i0 + lane_id();
    if (i0) d = i < K ? v.draft[b * K + i] : 0;
    const uint64_t bad = ballot(i < n && (d < 0 || d >= v.vocab));
    if (bad) return i0 + __builtin_ctzll(bad);
  }
  return n;
}

// block_arrive (sfx_common.h) for workgroups whose only results are ws_stores
// of thread 0, which calls this.  Those write through to where every XCD reads,
// so waiting for them is all that the counter needs; the release fence in its
// place writes the XCD's L2 back, once for each of thousands of workgroups (64
// drafts of 16 over 128,256 logits: 165 us with it, 45 without).  True in the
// last workgroup, which reads by ws_load; the counter keeps its total.
__device__ __forceinline__ bool arrive(unsigned* ctr, unsigned expected) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  return __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED,
                                __HIP_MEMORY_SCOPE_AGENT) == expected - 1;
}

// Joins the chunks of a position, by one wave; false while some are missing.
__device__ __forceinline__ bool join_parts(const Stat* p, int chunks,
                                           bool greedy, float c, Stat* out) {
  const int lane = lane_id();
  Stat r;
  r.top = kNegInf;
  r.sum = 0.0f;
  int at1 = 0x7fffffff;
  for (int i0 = 0; i0 < chunks; i0 += kWave) {
    const bool in = i0 + lane < chunks;
    Stat q;
    q.top = kNegInf;
    q.sum = 0.0f;
    if (in) q = take(p + i0 + lane);
    if (ballot(in && __builtin_bit_cast(uint64_t, q) == 0)) return false;
    const float top = fmaxf(r.top, wave_max(q.top));
    if (greedy) {
      const int a = wave_min(in && q.top == top ? q.at1 : 0x7fffffff);
      at1 = r.top == top ? min(at1, a) : a;
    } else {
      r.sum = r.sum * __builtin_amdgcn_exp2f(below(r.top, top) * c) +
              wave_sum(q.sum * __builtin_amdgcn_exp2f(below(q.top, top) * c));
    }
    r.top = top;
  }
  if (greedy) r.at1 = at1;
  *out = r;
  return true;
}

template <int DT>
__global__ __launch_bounds__(kThreads, 8) void k_verify_scan(VerifyArgs a) {
  using S = Share<DT>;
  constexpr int E = S::E, U = S::U;
  const int64_t b = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x % a.chunks;
  const int K = (int)a.v.k;
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const int j = blockIdx.y;
  __shared__ float lds[2 * kWaves];
  __shared__ int lds_at;
  __shared__ unsigned lds_stop;
  unsigned known = 0;
  if (threadIdx.x == 0)
    known = __hip_atomic_load(a.stop + b * kStopPitch, __ATOMIC_RELAXED,
                              __HIP_MEMORY_SCOPE_AGENT);
  const float t = temperature_of(a.v, b);
  const bool greedy = !(t > 0.0f);
  const float c = greedy ? 0.0f : scale_of(t);
  const int n = drafts_of(a.v, b);
  // A row that draws races the position after its drafts without a sum.
  if (j > n || (j == n && !greedy)) return;
  if (threadIdx.x == 0) lds_stop = known;
  __syncthreads();
  // the same for the whole workgroup
  if (lds_stop && (int)(K + 1 - lds_stop) < j) return;
  const typename S::T* row = (const typename S::T*)a.v.logits +
                             b * a.v.stride_b + j * a.v.stride_j;
  S s(row, a.v.vocab, chunk);
  s.load(row);
  float top = fmaxf(s.single, kNegInf);
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, s.get(u, e));
  Stat* part = a.part + (b * (K + 1) + j) * a.chunks;
  Stat r;
  if (greedy) {
    const float mine = top;
    if (threadIdx.x == 0) lds_at = 0x7fffffff;
    top = block_max(top, lds);
    // few threads hold the largest
    if (mine == top && top > kNegInf) {
      int at = 0x7fffffff;
      s.again([&](float x, int i) { at = x == top ? min(at, i) : at; });
      atomicMin(&lds_at, at);
    }
    __syncthreads();
    r.top = top;
    r.at1 = lds_at + 1;
  } else {
    // Each wave sums relative to its own largest; the four are joined.
    top = wave_max(top);
    s.forget();
    float sum = 0.0f;
    if (top > kNegInf) {
      float p0 = __builtin_amdgcn_exp2f((s.single - top) * c), p1 = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          p0 += __builtin_amdgcn_exp2f((s.get(u, e) - top) * c);
          p1 += __builtin_amdgcn_exp2f((s.get(u, e + 1) - top) * c);
        }
      sum = wave_sum(p0 + p1);
      if (!(sum < 1e30f)) {  // a NaN, or infinities that met
        sum = 0.0f;
        s.again([&](float x, int) {
          sum += __builtin_amdgcn_exp2f(below(x, top) * c);
        });
        sum = wave_sum(sum);
      }
    }
    if (lane == 0) {
      lds[2 * wave] = top;
      lds[2 * wave + 1] = sum;
    }
    __syncthreads();
    r.top = lds[0];
    r.sum = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) r.top = fmaxf(r.top, lds[2 * w]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      r.sum += lds[2 * w + 1] *
               __builtin_amdgcn_exp2f(below(lds[2 * w], r.top) * c);
  }
  if (wave == 0) {
    // Once this part has reached where every XCD reads (the wait), the
    // others' are looked at: of all workgroups of a position, the one whose
    // part arrives last finds every part.  No counter, whose updates by a
    // position's workgroups queue up one behind the other, and no fence.
    if (lane == 0) put(part + chunk, r);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (join_parts(part, a.chunks, greedy, c, &r)) {
      bool ok = false;
      if (j < n && r.top > kNegInf) {
        const int d = a.v.draft[b * K + j];
        if (greedy) {
          ok = d + 1 == r.at1;
        } else {
          const float p =
              __builtin_amdgcn_exp2f(below(Elem<DT>::get(row[d]), r.top) * c) /
              r.sum;
          const float q = a.v.draft_probs
                              ? a.v.draft_probs[(b * K + j) * a.v.vocab + d]
                              : 1.0f;
          ok = a.v.uniform[b * K + j] * q < p;
        }
      }
      // two workgroups may get here for one position, with the same words
      if (lane == 0) put(a.stat + b * (K + 1) + j, r);
      if (!ok && lane == 0) atomicMax(a.stop + b * kStopPitch, (unsigned)(K + 1 - j));
    }
  }
}

// Race key of one candidate as ordered bits; nothing for NaN or none.
__device__ __forceinline__ uint32_t race_key(float rate, float clock) {
  const float g = rate * __builtin_amdgcn_rcpf(clock);
  return g > 0.0f ? __float_as_uint(g) : 0u;
}

template <int DT, bool kProbs>
__global__ __launch_bounds__(kThreads) void k_verify_draw(VerifyArgs a) {
  using S = Share<DT>;
  constexpr int E = S::E, U = S::U;
  const int per_row = a.v.all_greedy ? 1 : a.chunks;
  const int64_t b = blockIdx.x / per_row;
  const int chunk = blockIdx.x % per_row;
  const int K = (int)a.v.k;
  const float t = temperature_of(a.v, b);
  const bool greedy = !(t > 0.0f);
  if (greedy && chunk > 0) return;
  const int wave = threadIdx.x / kWave, lane = lane_id();
  __shared__ float lds[kWaves];
  __shared__ uint64_t ldu[kWaves];
  __shared__ int lds_last;
  const int64_t V = a.v.vocab;
  const typename S::T* base = (const typename S::T*)a.v.logits +
                              b * a.v.stride_b;
  const unsigned known = a.stop[b * kStopPitch];
  const int at_pos = known ? (int)(K + 1 - known) : drafts_of(a.v, b);
  // a row that stopped nowhere has all its drafts kept
  const bool res = known != 0;
  int token = -1;
  if (greedy) {
    const Stat r = a.stat[b * (K + 1) + at_pos];
    token = r.top > kNegInf ? r.at1 - 1 : -1;
  } else {
    const float c = scale_of(t);
    const typename S::T* row = base + at_pos * a.v.stride_j;
    S s(row, V, chunk);
    s.load(row);
    const float* noise = a.v.noise + b * V;
    float clock[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u)
      load_floats<E>(noise + s.index(u * E), s.first + u * kThreads < s.vecs,
                     clock[u]);
    const float clock1 = s.extra >= 0 ? noise[s.extra] : 1.0f;
    const int d = res ? a.v.draft[b * K + at_pos] : -1;
    const float* q = kProbs && res
                         ? a.v.draft_probs + (b * K + at_pos) * V
                         : nullptr;
    float top, inv = 1.0f;
    if (kProbs && q) {
      const Stat r = a.stat[b * (K + 1) + at_pos];
      top = r.top;
      inv = 1.0f / r.sum;
    } else {
      top = fmaxf(s.single, kNegInf);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, s.get(u, e));
      top = block_max(top, lds);
    }
    // Keys: the bits of a rate over its clock, the top bit for members of r.
    const int d_place = s.place_of(d);
    uint32_t key = 0;
    int place = 0;
    auto race = [&](float z, float e, float qi, int at) {
      z = z == top ? 0.0f : z - top;  // a NaN makes no key
      const float p = __builtin_amdgcn_exp2f(z * c);
      uint32_t kk;
      if (kProbs && q) {
        const float r = p * inv - qi;
        kk = race_key(r > 0.0f ? r : p * inv, e);
        if (kk && r > 0.0f) kk |= 0x80000000u;
      } else {
        kk = race_key(p, e);
        if (kk && at != d_place) kk |= 0x80000000u;
      }
      return kk;
    };
    uint32_t tok = 0xffffffffu;
    if (top > kNegInf) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float qu[E];
        if (kProbs && q)
          load_floats<E>(q + s.index(u * E), s.first + u * kThreads < s.vecs,
                         qu);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t kk =
              race(s.get(u, e), clock[u][e], qu[e], u * E + e);
          if (kk > key) {
            key = kk;
            place = u * E + e;
          }
        }
      }
      if (key) tok = (uint32_t)s.index(place);
      if (s.extra >= 0) {
        const uint32_t kk = race(s.single, clock1,
                                 kProbs && q ? q[s.extra] : 0.0f, S::kSingle);
        if (kk > key || (kk == key && (uint32_t)s.extra < tok)) {
          key = kk;
          tok = (uint32_t)s.extra;
        }
      }
    }
    uint64_t best = wave_max_u64((uint64_t)key << 32 | (uint32_t)~tok);
    if (lane == 0) ldu[wave] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < kWaves; ++w) best = best > ldu[w] ? best : ldu[w];
      const uint32_t k32 = (uint32_t)(best >> 32);
      Best* o = a.best + b * a.chunks + chunk;
      ws_store(&o->key, __uint_as_float(k32 & 0x7fffffffu));
      ws_store(&o->shift, top);
      ws_store(&o->token, k32 ? (int32_t)~(uint32_t)best : -1);
      ws_store(&o->in_r, (int32_t)(k32 >> 31));
      lds_last = arrive(a.arrived + b, (unsigned)a.chunks);
    }
    __syncthreads();
    if (!lds_last) return;
    // The row's last workgroup: the best of all, earlier ones on ties.
    if (wave == 0) {
      float mx = kNegInf;
      for (int i = lane; i < a.chunks; i += kWave)
        mx = fmaxf(mx, ws_load(&a.best[b * a.chunks + i].shift));
      mx = wave_max(mx);
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
  // The words that the next call finds zero (the row's other workgroups have
  // read `stop`), and the result.
  Stat zero;
  zero.top = zero.sum = 0.0f;
  for (int i = threadIdx.x; i < (K + 1) * a.chunks; i += kThreads)
    a.part[b * (K + 1) * a.chunks + i] = zero;
  if (wave == 0) {
    int32_t* out = a.v.sampled + b * (K + 1);
    for (int i = lane; i <= K; i += kWave)
      out[i] = i < at_pos ? a.v.draft[b * K + i] : (i == at_pos ? token : -1);
    if (lane == 0) {
      a.arrived[b] = 0;
      a.stop[b * kStopPitch] = 0;
      a.v.count[b] = at_pos + (token >= 0);
    }
  }
}

int chunks_for(int64_t vocab) {
  return (int)((vocab + kChunk - 1) / kChunk);
}

size_t round_up(size_t x) { return (x + 255) & ~(size_t)255; }

size_t counter_bytes_for(int64_t batch, int64_t k, int64_t vocab) {
  const size_t b = (size_t)batch;
  return b * (size_t)(k + 1) * (size_t)chunks_for(vocab) * sizeof(Stat) +
         b * (1 + kStopPitch) * 4;
}

size_t scratch_bytes_for(int64_t batch, int64_t k, int64_t vocab) {
  const size_t b = (size_t)batch;
  return round_up(b * (size_t)(k + 1) * sizeof(Stat)) +
         b * (size_t)chunks_for(vocab) * sizeof(Best);
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
  const dim3 grid((unsigned)(a.v.batch * (a.v.all_greedy ? 1 : a.chunks)));
  if (a.v.draft_probs && !a.v.all_greedy)
    hipLaunchKernelGGL((k_verify_draw<DT, true>), grid, dim3(kThreads), 0,
                       stream, a);
  else
    hipLaunchKernelGGL((k_verify_draw<DT, false>), grid, dim3(kThreads), 0,
                       stream, a);
  return (int)hipGetLastError();
}

}  // namespace

}  // namespace sfx

using namespace sfx;

extern "C" size_t sfx_verify_workspace_size(int64_t batch, int64_t k,
                                            int64_t vocab) {
  if (!sizes_ok(batch, k, vocab) || batch == 0) return 0;
  return scratch_bytes_for(batch, k, vocab);
}

extern "C" size_t sfx_verify_counter_bytes(int64_t batch, int64_t k,
                                           int64_t vocab) {
  if (!sizes_ok(batch, k, vocab) || batch == 0) return 0;
  return counter_bytes_for(batch, k, vocab);
}

extern "C" int sfx_verify_draft(const sfx_verify* args, void* counters,
                                size_t counter_bytes, void* workspace,
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
  if (!workspace || ((uintptr_t)workspace & 15) ||
      workspace_bytes < scratch_bytes_for(v.batch, v.k, v.vocab))
    return SFX_EINVAL;
  if (!counters || ((uintptr_t)counters & 15) ||
      counter_bytes < counter_bytes_for(v.batch, v.k, v.vocab))
    return SFX_EINVAL;
  a.chunks = chunks_for(v.vocab);
  a.part = (Stat*)counters;
  a.arrived = (unsigned*)(a.part + v.batch * (v.k + 1) * a.chunks);
  a.stop = a.arrived + v.batch;
  a.stat = (Stat*)workspace;
  a.best = (Best*)((char*)workspace +
                   round_up((size_t)v.batch * (size_t)(v.k + 1) * sizeof(Stat)));
  switch (v.dtype) {
    case SFX_BF16: return launch<SFX_BF16>(a, stream);
    case SFX_F16: return launch<SFX_F16>(a, stream);
    default: return launch<SFX_F32>(a, stream);
  }
}
