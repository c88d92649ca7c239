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
// Bound by its launch and its chain: lengths, two scans, pages, table, slots (64
// sequences of 12 new tokens 3.4 us, 512 of 2000 6.0 + 3.8).
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

// Sum over the lanes of a wave up to this one, by register moves. What a wave's 64
// sequences hold or lack stays below 2^31: 2^25 pages each at most.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned add_moved(unsigned x) {
  return x + (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ unsigned wave_upto(unsigned x) {
  x = add_moved<0x111, 0xf>(x);     // row_shr 1, 2, 4, 8
  x = add_moved<0x112, 0xf>(x);
  x = add_moved<0x114, 0xf>(x);
  x = add_moved<0x118, 0xf>(x);
  x = add_moved<0x142, 0xa>(x);     // row_bcast 15: of rows 0 and 2 to 1 and 3
  return add_moved<0x143, 0xc>(x);  // row_bcast 31: of row 1 to 2 and 3
}

// Which of N runs, whose ends are `upto`, item j lies in.
template <int N>
__device__ __forceinline__ int run_of(const int64_t* upto, int64_t j) {
  int lo = 0;
#pragma unroll
  for (int step = N / 2; step; step >>= 1)
    if (upto[lo + step - 1] <= j) lo += step;
  return lo;
}

__device__ __forceinline__ int64_t slot_of(const CachePlanArgs& a, int64_t pos, int page) {
  return page >= 0 ? ((int64_t)page << a.lp) + (pos & ((1 << a.lp) - 1)) : -1;
}

}  // namespace

// One workgroup, N sequences at a time. FUSED: there are no more, and it writes table
// and slots too.
//
// Who gets pages: the sums `lacks` ascend, so those that get none are the ones behind a
// point, and the taken pages are those of the runs before it.
template <int N, bool FUSED>
__global__ __launch_bounds__(N) void cache_plan_kernel(CachePlanArgs a) {
  constexpr int NW = N / 64;
  __shared__ int64_t back_sums[NW], lack_sums[NW], back_upto[N], lack_upto[N];
  __shared__ unsigned long long taken_here;
  __shared__ int first[N], held[N], tokens[N];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int64_t room = a.room, count = min(max((int64_t)a.free_count[0], (int64_t)0), room);
  // sums of a tile's pages over the sequences before and with this one, and all
  auto scan = [&](int64_t& back, int64_t& lack, int64_t& backs, int64_t& lacks) {
    back = wave_upto((unsigned)back);
    lack = wave_upto((unsigned)lack);
    __syncthreads();
    if (lane == 63) {
      back_sums[w] = back;
      lack_sums[w] = lack;
    }
    __syncthreads();
    backs = lacks = 0;
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      if (k == w) {
        back += backs;
        lack += lacks;
      }
      backs += back_sums[k];
      lacks += lack_sums[k];
    }
  };
  PlanSeq q{};
  if (t < a.B) q = plan_seq(a, t);
  int64_t back = q.back, lack = q.lack, back_here, lack_here;
  scan(back, lack, back_here, lack_here);
  int64_t all_back = back_here;
  if (!FUSED)
    for (int b0 = N; b0 < a.B; b0 += N) {
      int64_t x = b0 + t < a.B ? plan_seq(a, b0 + t).back : 0, y = 0, xs, ys;
      scan(x, y, xs, ys);
      all_back += xs;
    }
  const int64_t end = count + all_back, top = min(end, room);
  int64_t back_before = 0, lack_before = 0, taken = 0;
  for (int b0 = 0; b0 < (FUSED ? 1 : a.B); b0 += N) {
    const int b = b0 + t;
    if (b0) {
      q = PlanSeq{};
      if (b < a.B) q = plan_seq(a, b);
      back = q.back;
      lack = q.lack;
      scan(back, lack, back_here, lack_here);
    }
    const int64_t lacks = lack_before + lack;
    const bool ok = b < a.B && q.fits && (q.lack == 0 || lacks <= top);
    back_upto[t] = back;
    first[t] = (int)q.want;
    if (FUSED) {
      lack_upto[t] = lack;
      held[t] = q.held;
      tokens[t] = ok ? q.nb : 0;
    }
    if (t == 0) taken_here = 0;
    __syncthreads();
    if (ok && q.lack > 0) atomicMax(&taken_here, (unsigned long long)lacks);
    for (int64_t j = t; j < back_here; j += N) {
      const int k = run_of<N>(back_upto, j);
      const int64_t at = end - 1 - (back_before + j);
      int* entry = a.table + (int64_t)(b0 + k) * a.W + first[k] + (j - (k ? back_upto[k - 1] : 0));
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
    __syncthreads();
    taken = max(taken, (int64_t)taken_here);
    back_before += back_here;
    lack_before += lack_here;
  }
  if (t == 0) {
    a.free_count[0] = (int)(top - taken);
    if (!FUSED) *static_cast<int64_t*>(a.workspace) = top;
  }
  if (FUSED) {
    for (int64_t j = t; j < taken; j += N) {
      const int k = run_of<N>(lack_upto, j);
      a.table[(int64_t)k * a.W + held[k] + (j - (k ? lack_upto[k - 1] : 0))] = a.free_pages[top - 1 - j];
    }
    // a place on a page that was taken is looked up where that came from
    for (int e = t; e < a.B * a.n; e += N) {
      const int b = e / a.n, i = e - b * a.n;
      int64_t slot = -1;
      if (i < tokens[b]) {
        const int64_t pos = (int64_t)max(a.lens[b], 0) + i, k = pos >> a.lp;
        slot = slot_of(a, pos, k < held[b] ? a.table[(int64_t)b * a.W + k]
                                           : a.free_pages[top - 1 - ((b ? lack_upto[b - 1] : 0) + k - held[b])]);
      }
      a.slots[e] = slot;
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
  // few sequences: fewer waves to wait for at every barrier
  if (!a.workspace) {
    if (a.B <= 256)
      MORPHO_KLAUNCH((cache_plan_kernel<256, true>), dim3(1), dim3(256), 0, s, a);
    else
      MORPHO_KLAUNCH((cache_plan_kernel<1024, true>), dim3(1), dim3(1024), 0, s, a);
    return hipGetLastError();
  }
  MORPHO_KLAUNCH((cache_plan_kernel<1024, false>), dim3(1), dim3(1024), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int blocks = (a.n + 1023) / 1024;
  MORPHO_KLAUNCH(cache_slots_kernel, dim3((unsigned)((int64_t)a.B * blocks)), dim3(256), 0, s, a, blocks);
  return hipGetLastError();
}

}  // namespace morpho
