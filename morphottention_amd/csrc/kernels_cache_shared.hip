// Attention over the paged cache where sequences have their first pages in
// common (forks of one prompt): the rows of all of a group's sequences meet the
// common keys together, so these are read once and not once a sequence; then
// every sequence its own keys (cache_attn.h with CacheShared), and a join.
//
// The softmax over the union of two sets of keys follows from each set's
// reference m, sum of weights l and weighted values o:
//   m = max(m1, m2), l = l1 2^(m1 - m) + l2 2^(m2 - m), o likewise,
// so a piece of the prefix is one more piece of a row to join. A new token sees
// all of its prefix (whole pages of tokens before it), whatever the mask says
// about the new tokens: no masks here.
#include "cache_attn.h"
#include "common.h"
#include "internal.h"

namespace morpho {

namespace {

// 16 R rows of one group: row r of it is new token r % n of its sequence r / n.
struct PrefixBlock {
  int first, rows, row0;  // the group's first place in `members`, its rows, the block's first row
  bool found;
};
// The group and rows of row block rb. A wave looks at 64 groups at a time.
__device__ __forceinline__ PrefixBlock prefix_block(const int* __restrict__ starts, int groups, int members, int n,
                                                    int per, int rb, int lane) {
  PrefixBlock p{0, 0, 0, false};
  for (int g0 = 0; g0 < groups; g0 += 64) {
    const int g = g0 + lane;
    int s0 = 0, s1 = 0;
    if (g < groups) {
      s0 = min(max(starts[g], 0), members);
      s1 = min(max(starts[g + 1], s0), members);
    }
    const int blocks = ((s1 - s0) * n + per - 1) / per;
    int upto = blocks;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o);
      if (lane >= o) upto += x;
    }
    const uint64_t past = __ballot(rb < upto);
    if (past) {
      const int l = __builtin_ctzll(past);
      p.first = __shfl(s0, l);
      p.rows = (__shfl(s1, l) - p.first) * n;
      p.row0 = (rb - (__shfl(upto, l) - __shfl(blocks, l))) * per;
      p.found = true;
      return p;
    }
    rb -= __shfl(upto, 63);
  }
  return p;
}

// A row of the block: its sequence and new token; b < 0: there is none. A
// sequence that skips no keys (cache_attn.h) is not in the group here either.
struct PrefixRow {
  int b, i, keys;
};
__device__ __forceinline__ PrefixRow prefix_row(const CacheAttnArgs& a, const CacheShared& shared, const PrefixBlock& p,
                                                const int* __restrict__ members, const int* __restrict__ lens,
                                                const int* __restrict__ new_lens, int r) {
  PrefixRow x{-1, 0, 0};
  if (p.row0 + r >= p.rows) return x;
  const int b = members[p.first + (p.row0 + r) / a.n];
  if ((unsigned)b >= (unsigned)a.B) return x;
  const SeqLen sq = seq_len(lens, new_lens, b, a.n, a.W << a.lp);
  x.i = (p.row0 + r) % a.n;
  x.keys = shared.skip(b, sq.ctx, a.lp);
  if (x.i < sq.nb && x.keys > 0) x.b = b;
  return x;
}

}  // namespace

struct PrefixArgs {
  int members, rblocks;
};

// What a workgroup works on: heads fastest (as elsewhere), then row blocks, which
// share the keys, then pieces.
struct PrefixPlace {
  int h, rb, sp;
  __device__ __forceinline__ PrefixPlace(int H, int rblocks) {
    int id = blockIdx.x;
    h = id % H;
    id /= H;
    rb = id % rblocks;
    sp = id / rblocks;
  }
};

// 16 QT rows, which the four waves of a workgroup share; each takes every fourth
// tile of the piece's keys straight into registers, one tile ahead.
template <int M, int DV, int QT>
__global__ __launch_bounds__(256) void cache_prefix_kernel(
    CacheAttnArgs a, CacheShared shared, PrefixArgs pa, const int* __restrict__ members,
    const int* __restrict__ starts, const f16* __restrict__ phi, const f16* __restrict__ gate_q,
    const f16* __restrict__ gate_k, const f16* __restrict__ codes, const f16* __restrict__ values,
    const int* __restrict__ table, const int* __restrict__ lens, const int* __restrict__ new_lens,
    float* __restrict__ part_o, float4* __restrict__ part_st) {
  constexpr int NT = DV / 16;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const PrefixPlace at(a.H, pa.rblocks);
  const int h = at.h;
  const PrefixBlock blk = prefix_block(starts, shared.groups, pa.members, a.n, 16 * QT, at.rb, lane);
  if (!blk.found) return;
  PrefixRow row[QT];
  int some = -1, keys = 0;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    row[t] = prefix_row(a, shared, blk, members, lens, new_lens, 16 * t + c16);
    const uint64_t there = __ballot(row[t].b >= 0);
    if (some < 0 && there) {
      some = __shfl(row[t].b, __builtin_ctzll(there));
      keys = __shfl(row[t].keys, __builtin_ctzll(there));
    }
  }
  some = __builtin_amdgcn_readfirstlane(some);
  keys = __builtin_amdgcn_readfirstlane(keys);
  const int kb = at.sp * shared.split;
  if (some < 0 || kb >= keys) return;
  const int ke = at.sp == shared.np - 1 ? keys : min(keys, kb + shared.split);
  const CacheSource<M, DV> src(a, codes, values, table, some, h, lane);

  CacheTile<M, DV> A[1], B[1];
  int tile = kb / 32 + w, pc = 0, pn = 0;
  const int last = ke / 32;  // keys are whole pages, pieces whole tiles
  if (tile < last) {
    pc = src.page_of(tile);
    src.load(A[0], tile, pc);
  }
  if (tile + 4 < last) pn = src.page_of(tile + 4);
  CacheRows<M, DV, QT, true> R;
  float rc[QT];
  R.start_rows(a, gate_q, gate_k, h, lane, rc, [&](int t) {
    const int b = row[t].b >= 0 ? row[t].b : some, i = row[t].b >= 0 ? row[t].i : 0;
    return phi + (((int64_t)b * a.n + i) * a.H + h) * M;
  });
  auto step = [&](CacheTile<M, DV>(&cur)[1], CacheTile<M, DV>(&nxt)[1], int& page, int next) {
    if (tile + 4 < last) src.load(nxt[0], tile + 4, next);
    const bool there = src.exists(page);
    if (tile + 8 < last) page = src.page_of(tile + 8);
    if (there) R.add_clear(cur);
    tile += 4;
  };
  while (tile < last) {
    step(A, B, pc, pn);
    if (tile >= last) break;
    step(B, A, pn, pc);
  }

  __shared__ __align__(16) float so[4][16 * QT][DV + 4];
  __shared__ float sm[4][16 * QT], sl[4][16 * QT], sr[16 * QT];
  __shared__ int64_t place[16 * QT];  // of the row's parts
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float ref, l;
    R.finish(t, ref, l);
#pragma unroll
    for (int c = 0; c < NT; ++c) *reinterpret_cast<f32x4*>(&so[w][16 * t + c16][16 * c + 4 * g]) = R.O[t][c];
    if (g == 0) {
      sm[w][16 * t + c16] = ref;
      sl[w][16 * t + c16] = l;
      if (w == 0) {
        sr[16 * t + c16] = rc[t];
        place[16 * t + c16] =
            row[t].b < 0 ? -1
                         : (((int64_t)row[t].b * a.H + h) * a.n + row[t].i) * (shared.np + a.nsplit) + at.sp;
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 4 * QT * DV; e += 256) {
    const int q = e / (DV / 4), c = 4 * (e % (DV / 4));
    if (place[q] < 0) continue;
    float m = sm[0][q];
#pragma unroll
    for (int k = 1; k < 4; ++k) m = fmaxf(m, sm[k][q]);
    float l = 0.f;
    f32x4 o = {};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = fast_exp2(sm[k][q] - m);
      l += f * sl[k][q];
      o += f * *reinterpret_cast<const f32x4*>(&so[k][q][c]);
    }
    *reinterpret_cast<f32x4*>(part_o + place[q] * DV + c) = o;
    if (c == 0) part_st[place[q]] = float4{m, l, sr[q], 0.f};
  }
}

namespace {
template <int M, int DV>
hipError_t launch_cache_shared_t(const CacheDims& d, const CacheSharedPlan& p, CacheAttnArgs a,
                                 const CacheShared& shared, const CacheSharedCall& call, const f16* phi,
                                 const f16* gate_q, const f16* gate_k, const f16* codes, const f16* values,
                                 const int* table, const int* lens, const int* new_lens, const int64_t* tree,
                                 f16* out, float* lse, const CacheAttnBuffers& part, hipStream_t s) {
  const dim3 block(256);
  const PrefixArgs pa{call.members_count, p.rblocks};
  const dim3 common((unsigned)((int64_t)d.H * p.rblocks * p.np));
#define MORPHO_CACHE_PREFIX(QT)                                                                                    \
  MORPHO_KLAUNCH((cache_prefix_kernel<M, DV, QT>), common, block, 0, s, a, shared, pa, call.members, call.starts, \
                 phi, gate_q, gate_k, codes, values, table, lens, new_lens, part.o, part.st)
  MORPHO_CACHE_PREFIX(1);
#undef MORPHO_CACHE_PREFIX
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)((int64_t)d.B * d.H * p.rest.qblocks * p.rest.nsplit));
#define MORPHO_CACHE_REST(...)                                                                                    \
  MORPHO_KLAUNCH((__VA_ARGS__), grid, block, 0, s, a, shared, phi, gate_q, gate_k, codes, values, table, lens,    \
                 new_lens, tree, out, lse, part.o, part.st)
  if (p.rest.qt == 0)
    MORPHO_CACHE_REST(cache_attn_few_kernel<M, DV, CacheShared>);
  else
    MORPHO_CACHE_REST(cache_attn_rows_kernel<M, DV, 1, true, CacheShared>);
#undef MORPHO_CACHE_REST
  return hipGetLastError();
}
}  // namespace

hipError_t launch_cache_shared(const CacheDims& d, const CacheSharedPlan& plan, const CacheSharedCall& call,
                               const f16* phi, const f16* gate_q, const f16* gate_k, const f16* codes,
                               const f16* values, const int* table, const int* lens, const int* new_lens,
                               const int64_t* tree, f16* out, float* lse, const CacheAttnBuffers& part, float scale,
                               int causal, int mask_diag, hipStream_t s) {
  CacheAttnArgs a = attn_args(d, plan.rest, causal, mask_diag);
  a.sl2e = scale * kLog2e;
  const CacheShared shared{call.group, call.pages, call.groups, plan.np, plan.split_keys};
  MORPHO_MDV_DISPATCH(launch_cache_shared_t, d, plan, a, shared, call, phi, gate_q, gate_k, codes, values, table, lens,
                      new_lens, tree, out, lse, part, s);
}

hipError_t launch_cache_shared_join(const CacheDims& d, const CacheSharedPlan& plan, const CacheSharedCall& call,
                                    const f16* values, const int* table, const int* lens, const int* new_lens,
                                    const int64_t* tree, const CacheAttnBuffers& part, f16* out, float* lse,
                                    int causal, int mask_diag, hipStream_t s) {
  const CacheAttnArgs a = attn_args(d, plan.rest, causal, mask_diag);
  const CacheShared shared{call.group, call.pages, call.groups, plan.np, plan.split_keys};
  const int64_t rows = (int64_t)d.B * d.H * d.n;
#define MORPHO_CACHE_JOIN(DV, NG)                                                                            \
  MORPHO_KLAUNCH((cache_join_kernel<DV, NG, CacheShared>), dim3((unsigned)((rows * (DV / 4) * NG + 255) / 256)), \
                 dim3(256), 0, s, a, shared, rows, values, table, lens, new_lens, tree, part.o, part.st, out, lse)
  const bool many = plan.np + plan.rest.nsplit > 8;
  if (d.DV == 32 && many)
    MORPHO_CACHE_JOIN(32, 32);
  else if (d.DV == 32)
    MORPHO_CACHE_JOIN(32, 1);
  else if (d.DV == 64 && many)
    MORPHO_CACHE_JOIN(64, 16);
  else if (d.DV == 64)
    MORPHO_CACHE_JOIN(64, 1);
  else if (many)
    MORPHO_CACHE_JOIN(128, 8);
  else
    MORPHO_CACHE_JOIN(128, 1);
#undef MORPHO_CACHE_JOIN
  return hipGetLastError();
}

}  // namespace morpho
