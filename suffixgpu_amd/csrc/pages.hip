// Page tables of the paged cache, from the rows' lengths: which pages come from
// the pool's stack of free ones and which go back.
//
// With need_r and back_r the pages that row r lacks or has too many of, row r
// takes those numbered sum_{q < r} need_q and on from the top of the stack, while
// there are any, and its last page goes back as number sum_{q > r} back_q from
// where the stack then ends.  Both are prefix sums over the rows.  Every stack
// entry that changes is then one thread's: it hands its old page to the row that
// takes it and receives the page that comes back to it, so nothing is read after
// another thread has written it.
//
// There are few bytes, so the launches' latency bounds it.  Where the pages that can
// move are few, one workgroup does all (64 rows of 128 pages: 3.5 us); where they are
// many, one plans and others move (256 rows that begin anew with up to 64 pages each:
// 3.2 + 4.8 us).

#include <algorithm>

#include "launch.h"
#include "sfx_common.h"

namespace sfx {

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kMoveThreads = 256;

struct PagesArgs {
  int32_t* stack;
  int32_t* num_free;
  int32_t* held;
  int32_t* table;
  int32_t* plan;
  int64_t num_pages;
  int64_t width;
  int shift;  // log2(page_size)
  int n;
  const void* lengths;
  int len64;
  int32_t* room;
};

// Per row, in LDS: the first page that it takes (numbers from the top of the
// stack), the sum of the pages that it and the rows before it give back, and the
// pages that it held.
struct PlanView {
  int32_t* first;
  int32_t* given;
  int32_t* held;
  __device__ __forceinline__ PlanView(char* lds, int n)
      : first((int32_t*)lds), given(first + n), held(first + 2 * n) {}
};

struct Totals {
  int free, takes, gives;
};

__device__ __forceinline__ uint64_t wave_scan_u64(uint64_t v) {
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const uint64_t w = __shfl_up(v, o);
    if (lane_id() >= o) v += w;
  }
  return v;
}

// The rows' plan by one workgroup; the new number of pages of each row.
__device__ __forceinline__ Totals plan_rows(const PagesArgs& a, PlanView p) {
  __shared__ uint64_t wave_need[kPlanThreads / kWave];
  __shared__ uint32_t wave_give[kPlanThreads / kWave];
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const int64_t free = a.num_free[0];
  uint64_t need0 = 0;
  uint32_t give0 = 0;
  for (int r0 = 0; r0 < a.n; r0 += kPlanThreads) {
    const int r = r0 + (int)threadIdx.x;
    int64_t held = 0, want = 0;
    if (r < a.n) {
      held = a.held[r];
      const int64_t len = load_count(a.lengths, a.len64, r);
      // (a length next to 2^63 shall not wrap)
      want = len < 0 ? held
                     : (len >> a.shift) + ((len & ((1 << a.shift) - 1)) != 0);
      want = want < a.width ? want : a.width;
    }
    const uint64_t need = want > held ? want - held : 0;
    const uint32_t give = held > want ? (uint32_t)(held - want) : 0;
    const uint64_t need_to = wave_scan_u64(need);
    const uint32_t give_to = wave_incl_scan(give);
    if (lane == kWave - 1) {
      wave_need[wave] = need_to;
      wave_give[wave] = give_to;
    }
    __syncthreads();
    uint64_t need1 = need0, need_all = 0;
    uint32_t give1 = give0, give_all = 0;
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
      if (w < wave) {
        need1 += wave_need[w];
        give1 += wave_give[w];
      }
      need_all += wave_need[w];
      give_all += wave_give[w];
    }
    if (r < a.n) {
      const int64_t before = (int64_t)(need1 + need_to - need);
      const int64_t left = before < free ? free - before : 0;
      const int64_t got = (int64_t)need < left ? (int64_t)need : left;
      p.first[r] = (int32_t)(before < free ? before : free);
      p.given[r] = (int32_t)(give1 + give_to);
      p.held[r] = (int32_t)held;
      const int32_t now = (int32_t)(give ? want : held + got);
      a.held[r] = now;
      a.room[r] = now << a.shift;
    }
    need0 += need_all;
    give0 += give_all;
    __syncthreads();
  }
  Totals t;
  t.free = (int)free;
  t.takes = (int)((int64_t)need0 < free ? (int64_t)need0 : free);
  t.gives = (int)give0;
  return t;
}

// Last row whose value is at most x; values ascend, the first is at most x.
__device__ __forceinline__ int last_at_most(const int32_t* v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (v[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// First row whose value is more than x; there is one.
__device__ __forceinline__ int first_above(const int32_t* v, int n, int x) {
  int lo = -1, hi = n - 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (v[mid] > x) hi = mid; else lo = mid;
  }
  return hi;
}

// Stack entries left + i0, left + i0 + step, ...
__device__ __forceinline__ void move_pages(const PagesArgs& a, PlanView p,
                                           Totals t, int64_t i0,
                                           int64_t step) {
  const int64_t left = t.free - t.takes;
  const int64_t moves = t.takes > t.gives ? t.takes : t.gives;
  for (int64_t i = i0; i < moves; i += step) {
    const int64_t s = left + i;
    if (s >= a.num_pages) break;
    int32_t id = -1;
    if (i < t.takes) id = a.stack[s];
    if (i < t.gives) {
      const int r = first_above(p.given, a.n, t.gives - 1 - (int)i);
      const int64_t at =
          p.held[r] - 1 - ((int)i - (t.gives - p.given[r]));
      int32_t* e = a.table + r * a.width + at;
      a.stack[s] = *e;
      *e = -1;
    }
    if (i < t.takes) {
      const int k = t.free - 1 - (int)s;
      const int r = last_at_most(p.first, a.n, k);
      a.table[r * a.width + p.held[r] + (k - p.first[r])] = id;
    }
  }
}

// All by one workgroup: tables of which few entries can move.  64 rows that grow
// by up to 17 tokens: a launch's latency, and three loads that need each other.
__global__ __launch_bounds__(kPlanThreads) void k_pages_resize(PagesArgs a) {
  extern __shared__ __align__(16) char lds[];
  const PlanView p(lds, a.n);
  const Totals t = plan_rows(a, p);
  __syncthreads();
  move_pages(a, p, t, threadIdx.x, kPlanThreads);
  if (threadIdx.x == 0) a.num_free[0] = t.free - t.takes + t.gives;
}

__global__ __launch_bounds__(kPlanThreads) void k_pages_plan(PagesArgs a) {
  extern __shared__ __align__(16) char lds[];
  const PlanView p(lds, a.n);
  const Totals t = plan_rows(a, p);
  __syncthreads();
  for (int i = threadIdx.x; i < 3 * a.n; i += kPlanThreads)
    a.plan[4 + i] = p.first[i];
  if (threadIdx.x == 0) {
    a.plan[0] = t.free;
    a.plan[1] = t.takes;
    a.plan[2] = t.gives;
    a.num_free[0] = t.free - t.takes + t.gives;
  }
}

__global__ __launch_bounds__(kMoveThreads) void k_pages_move(PagesArgs a) {
  extern __shared__ __align__(16) char lds[];
  const PlanView p(lds, a.n);
  const Totals t = {a.plan[0], a.plan[1], a.plan[2]};
  const int64_t i0 = (int64_t)blockIdx.x * kMoveThreads;
  if (i0 >= t.takes && i0 >= t.gives) return;
  for (int i = threadIdx.x; i < 3 * a.n; i += kMoveThreads)
    p.first[i] = a.plan[4 + i];
  __syncthreads();
  move_pages(a, p, t, i0 + threadIdx.x, (int64_t)gridDim.x * kMoveThreads);
}

struct SlotArgs {
  const int32_t* table;
  int64_t num_pages;
  int64_t width;
  int shift;
  const void* start;
  const void* count;
  int start64, count64;
  int64_t tokens;
  int64_t* slots;
};

__global__ __launch_bounds__(256) void k_pages_slots(SlotArgs a) {
  const int64_t r = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.tokens) return;
  const int64_t n = a.count ? load_count(a.count, a.count64, r) : a.tokens;
  const int64_t s0 = load_count(a.start, a.start64, r);
  int64_t slot = -1;
  // in pages: a start next to 2^63 is past the table too
  if (i < n && s0 >= 0 && (s0 >> a.shift) < a.width) {
    const int64_t pos = s0 + i;
    if (pos >> a.shift < a.width) {
      const int64_t id = a.table[r * a.width + (pos >> a.shift)];
      if (id >= 0 && id < a.num_pages)
        slot = (id << a.shift) + (pos & ((1 << a.shift) - 1));
    }
  }
  a.slots[r * a.tokens + i] = slot;
}

bool pool_ok(const sfx_pages* p, int64_t n) {
  return p && p->num_pages >= 0 && p->num_pages <= (int64_t(1) << 30) &&
         p->rows >= 1 && p->rows <= SFX_PAGES_ROWS && n >= 0 && n <= p->rows &&
         p->page_size >= 1 && p->page_size <= 65536 &&
         !(p->page_size & (p->page_size - 1)) && p->table_width >= 1 &&
         p->table_width <= (int64_t(1) << 30) / p->page_size && p->num_free &&
         p->held && p->table && p->plan &&
         (p->num_pages == 0 || p->free_pages);
}

int shift_of(int64_t page_size) {
  int s = 0;
  while ((int64_t(1) << s) < page_size) ++s;
  return s;
}

// Entries of the rows' tables up to which one workgroup moves them all.
constexpr int64_t kAlone = 1 << 16;

}  // namespace

}  // namespace sfx

using namespace sfx;

extern "C" int sfx_pages_resize(const sfx_pages* pool, const void* lengths,
                                int32_t lengths_is64, int64_t n, int32_t* room,
                                hipStream_t stream) {
  if (!pool_ok(pool, n)) return SFX_EINVAL;
  if (n == 0) return 0;
  if (!lengths || !room) return SFX_EINVAL;
  PagesArgs a;
  a.stack = pool->free_pages;
  a.num_free = pool->num_free;
  a.held = pool->held;
  a.table = pool->table;
  a.plan = pool->plan;
  a.num_pages = pool->num_pages;
  a.width = pool->table_width;
  a.shift = shift_of(pool->page_size);
  a.n = (int)n;
  a.lengths = lengths;
  a.len64 = lengths_is64;
  a.room = room;
  const size_t lds = 12 * (size_t)n;
  const int64_t most = std::min<int64_t>(n * a.width, a.num_pages);
  if (most <= kAlone) {
    hipLaunchKernelGGL(k_pages_resize, dim3(1), dim3(kPlanThreads), lds, stream,
                       a);
  } else {
    hipLaunchKernelGGL(k_pages_plan, dim3(1), dim3(kPlanThreads), lds, stream,
                       a);
    const int64_t wgs = (most + kMoveThreads - 1) / kMoveThreads;
    hipLaunchKernelGGL(k_pages_move,
                       dim3((unsigned)std::min<int64_t>(wgs, 1024)),
                       dim3(kMoveThreads), lds, stream, a);
  }
  return (int)hipGetLastError();
}

extern "C" int sfx_pages_slots(const sfx_pages* pool, const void* start,
                               int32_t start_is64, const void* count,
                               int32_t count_is64, int64_t n, int64_t tokens,
                               int64_t* slots, hipStream_t stream) {
  if (!pool_ok(pool, n) || tokens < 0 || tokens > (int64_t(1) << 28))
    return SFX_EINVAL;
  if (n == 0 || tokens == 0) return 0;
  if (!start || !slots) return SFX_EINVAL;
  SlotArgs a;
  a.table = pool->table;
  a.num_pages = pool->num_pages;
  a.width = pool->table_width;
  a.shift = shift_of(pool->page_size);
  a.start = start;
  a.count = count;
  a.start64 = start_is64;
  a.count64 = count_is64;
  a.tokens = tokens;
  a.slots = slots;
  hipLaunchKernelGGL(k_pages_slots,
                     dim3((unsigned)((tokens + 255) / 256), (unsigned)n),
                     dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}
