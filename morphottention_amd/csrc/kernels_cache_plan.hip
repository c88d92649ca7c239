// Page tables and slot maps of the paged cache from the sequences' lengths, on
// the device: what a step of new tokens needs, without the host.
//
// Of sequence b: it holds held[b] pages and wants ceil((lens[b] + new) / P). What
// it holds beyond that goes back to the stack of free pages, all sequences' before
// any is taken; what it lacks comes from the top of the stack, in the order of the
// sequences, and where that does not suffice neither it nor a later one that lacks
// pages gets any (none overtakes another, so none waits for ever). Both are prefix
// sums over the sequences:
//   page j that comes back lies at   free[count + back - 1 - j],
//   page j that is taken comes from  free[count + back - 1 - j],
// so pages that are given back and taken again are the same ones in the same order.
//
// Bound by its launch and its chain: lengths, two scans, pages, table, slots.
#include "common.h"
#include "internal.h"

namespace morpho {

namespace {

struct PlanSeq {
  int64_t want;
  int held, nb;
  bool fits;
  int64_t back, lack;  // pages
};
__device__ __forceinline__ PlanSeq plan_seq(const CachePlanArgs& a, int b) {
  PlanSeq q;
  const int64_t have = max(a.lens[b], 0);
  q.nb = a.new_lens ? min(max(a.new_lens[b], 0), a.n) : a.n;
  q.held = min(max(a.held[b], 0), a.W);
  q.want = (have + q.nb + ((int64_t)1 << a.lp) - 1) >> a.lp;
  q.fits = q.want <= a.W;
  q.back = q.fits ? max(q.held - q.want, (int64_t)0) : 0;
  q.lack = q.fits ? max(q.want - q.held, (int64_t)0) : 0;
  return q;
}

// For the second kernel: a sequence's pages before the call, where its taken ones
// begin, and its tokens (-1: it is left as it was).
struct PlanNote {
  int64_t first;
  int held, granted;
};
constexpr int kPlanHeader = 16;  // bytes before the notes: the pages to take from

// Sums over the lanes before and with this one, of 1024; total: all.
__device__ __forceinline__ int64_t scan1024(int64_t x, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) sums[w] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
  for (int k = 0; k < 16; ++k) {
    if (k < w) before += sums[k];
    total += sums[k];
  }
  return before + x;
}

// Which of 1024 runs, whose ends are `upto`, item j lies in.
__device__ __forceinline__ int run_of(const int64_t* upto, int64_t j) {
  int lo = 0;
#pragma unroll
  for (int step = 512; step; step >>= 1)
    if (upto[lo + step - 1] <= j) lo += step;
  return lo;
}

__device__ __forceinline__ int64_t slot_of(const CachePlanArgs& a, int64_t pos, int page) {
  return page >= 0 ? ((int64_t)page << a.lp) + (pos & ((1 << a.lp) - 1)) : -1;
}

}  // namespace

// One workgroup, 1024 sequences at a time. FUSED: there are no more, and it
// writes table and slots too.
template <bool FUSED>
__global__ __launch_bounds__(1024) void cache_plan_kernel(CachePlanArgs a) {
  __shared__ int64_t sums[16], upto[1024], from[1024];
  __shared__ int first[1024], held[1024], tokens[1024];
  const int t = threadIdx.x;
  const int64_t room = a.room, count = min(max((int64_t)a.free_count[0], (int64_t)0), room);
  int64_t back = 0, total;
  for (int b0 = 0; b0 < a.B; b0 += 1024) {
    scan1024(b0 + t < a.B ? plan_seq(a, b0 + t).back : 0, sums, total);
    back += total;
  }
  const int64_t top = min(count + back, room);
  int64_t back_before = 0, lack_before = 0, taken = 0;
  for (int b0 = 0; b0 < a.B; b0 += 1024) {
    const int b = b0 + t;
    PlanSeq q{};
    if (b < a.B) q = plan_seq(a, b);
    const int64_t backs = scan1024(q.back, sums, total), back_here = total;
    const int64_t lacks = lack_before + scan1024(q.lack, sums, total), lack_here = total;
    const bool ok = b < a.B && q.fits && (q.lack == 0 || lacks <= top);
    upto[t] = backs;
    first[t] = (int)q.want;
    __syncthreads();
    for (int64_t j = t; j < back_here; j += 1024) {
      const int k = run_of(upto, j);
      const int64_t at = count + back - 1 - (back_before + j);
      int* entry = a.table + (int64_t)(b0 + k) * a.W + first[k] + (j - (k ? upto[k - 1] : 0));
      const int page = *entry;
      *entry = -1;
      if (at < room) a.free_pages[at] = page;
    }
    if (b < a.B) {
      a.granted[b] = ok ? q.nb : 0;
      if (ok) a.held[b] = (int)q.want;
      if (!FUSED)
        reinterpret_cast<PlanNote*>(static_cast<char*>(a.workspace) + kPlanHeader)[b] =
            PlanNote{lacks - q.lack, q.held, ok ? q.nb : -1};
    }
    int64_t got;
    const int64_t gets = scan1024(ok ? q.lack : 0, sums, got);  // (its barriers: `upto` is read)
    taken += got;
    if (FUSED) {
      upto[t] = gets;
      held[t] = q.held;
      tokens[t] = ok ? q.nb : 0;
      from[t] = lacks - q.lack;
      __syncthreads();
      for (int64_t j = t; j < got; j += 1024) {
        const int k = run_of(upto, j);
        const int64_t i = j - (k ? upto[k - 1] : 0);
        a.table[(int64_t)k * a.W + held[k] + i] = a.free_pages[top - 1 - (from[k] + i)];
      }
    }
    back_before += back_here;
    lack_before += lack_here;
  }
  if (t == 0) {
    a.free_count[0] = (int)(top - taken);
    if (!FUSED) *static_cast<int64_t*>(a.workspace) = top;
  }
  if (FUSED) {
    __syncthreads();
    for (int e = t; e < a.B * a.n; e += 1024) {
      const int b = e / a.n, i = e - b * a.n;
      const int64_t pos = (int64_t)max(a.lens[b], 0) + i;
      a.slots[e] = i < tokens[b] ? slot_of(a, pos, a.table[(int64_t)b * a.W + (pos >> a.lp)]) : -1;
    }
  }
}

// The taken pages and the slots of 1024 tokens of a sequence a workgroup; the
// first of a sequence writes its table.
__global__ __launch_bounds__(256) void cache_slots_kernel(CachePlanArgs a, int blocks) {
  const int b = blockIdx.x / blocks, part = blockIdx.x % blocks;
  const int64_t top = *static_cast<const int64_t*>(a.workspace);
  const PlanNote note = reinterpret_cast<const PlanNote*>(static_cast<const char*>(a.workspace) + kPlanHeader)[b];
  int* row = a.table + (int64_t)b * a.W;
  const int64_t have = max(a.lens[b], 0);
  auto taken = [&](int64_t k) { return a.free_pages[top - 1 - (note.first + k - note.held)]; };
  if (part == 0) {
    const int64_t want = note.granted >= 0 ? (have + note.granted + ((int64_t)1 << a.lp) - 1) >> a.lp : 0;
    for (int64_t k = note.held + threadIdx.x; k < want; k += 256) row[k] = taken(k);
  }
  for (int i = part * 1024 + threadIdx.x; i < min((part + 1) * 1024, a.n); i += 256) {
    const int64_t pos = have + i, k = pos >> a.lp;
    a.slots[(int64_t)b * a.n + i] = i < note.granted ? slot_of(a, pos, k < note.held ? row[k] : taken(k)) : -1;
  }
}

hipError_t launch_cache_plan(const CachePlanArgs& a, hipStream_t s) {
  if (!a.workspace) {
    MORPHO_KLAUNCH((cache_plan_kernel<true>), dim3(1), dim3(1024), 0, s, a);
    return hipGetLastError();
  }
  MORPHO_KLAUNCH((cache_plan_kernel<false>), dim3(1), dim3(1024), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int blocks = (a.n + 1023) / 1024;
  MORPHO_KLAUNCH(cache_slots_kernel, dim3((unsigned)((int64_t)a.B * blocks)), dim3(256), 0, s, a, blocks);
  return hipGetLastError();
}

}  // namespace morpho
