// What the kernels over a vocabulary's logits share: a workgroup's piece of a row
// in registers, element types, and reductions over a wave.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sfx_common.h"
#include "suffixgpu_amd.h"

namespace sfx {

constexpr int kThreads = 256;
constexpr int kChunk = 8192;  // logits per workgroup
constexpr float kNegInf = -__builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;

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
  // As get, by a shift and a mask that the compiler does not know: it unpacks the
  // element anew, where floats kept from one use to the next would not fit beside
  // each other.
  struct Anew {
    uint32_t shift = 16, mask = 0xffff0000u;
    __device__ Anew() { asm volatile("" : "+s"(shift), "+s"(mask)); }
  };
  __device__ float get(int u, int e, const Anew& by) const {
    if (DT != SFX_BF16) return get(u, e);
    const uint32_t q[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
    return __uint_as_float(e % 2 ? q[e / 2] & by.mask : q[e / 2] << by.shift);
  }
  // The same for the elements of any type, which costs moves.
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
  // The same of step u, by all lanes at once: f(x, index, whether there is such
  // an element).
  template <class F>
  __device__ void again_step(int u, F f) const {
    const int v = first + u * kThreads;
    T x[E];
    const uint4 q = v < vecs ? ((const uint4*)body)[v] : uint4{0, 0, 0, 0};
    __builtin_memcpy(x, &q, 16);
#pragma unroll
    for (int e = 0; e < E; ++e)
      f(Elem<DT>::get(x[e]), head + v * E + e, v < vecs);
  }
};

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

}  // namespace sfx
