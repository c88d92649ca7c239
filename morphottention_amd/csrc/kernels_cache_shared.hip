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
//
// Measured (kernel + join): 32 sequences of 65536 common tokens, H16 m32 dv64, 43 + 5.3 us,
// 5.1 TB/s: reading the keys. 64 of 8192, m16, 15.7 + 4.2; four groups of 12 of 4096 and
// 16 alone, m32, 14.6 + 4.6: the launch, the first keys' latency and the last pieces.
// The 64 with chains of 5 29.4 + 5.1, of 16 68 + 5.6 (matrix work 18).
// 16 trees of 48 drafts behind 4096, H32 m64, 58 + 5.6: VALU and MFMA work (three
// quarters of a SIMD's cycles), which its waves, three at most, overlap only in part.
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
  const int *members, *starts;
  int count, rblocks, blocks;  // members, row blocks, workgroups of the prefixes (before those of the rest)
};

// What a workgroup of the prefixes works on: heads fastest (as elsewhere), then row
// blocks, which share the keys, then pieces.
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
// The part of row x that this piece of head h fills.
__device__ __forceinline__ int64_t part_of(const CacheAttnArgs& a, const CacheShared& shared, const PrefixRow& x, int h,
                                           int sp) {
  return x.b < 0 ? -1 : (((int64_t)x.b * a.H + h) * a.n + x.i) * (shared.np + a.nsplit) + sp;
}

// Few rows: 16 QT of a group, which the four waves of a workgroup share; each takes
// every fourth tile of the piece's keys straight into registers, one tile ahead, so
// that a tile is read once for all of the rows.
template <int M, int DV, int QT>
__device__ __forceinline__ void cache_prefix_few(const CacheAttnArgs& a, const CacheShared& shared, const PrefixArgs& pa,
                                                 const f16* phi, const f16* gate_q, const f16* gate_k,
                                                 const f16* codes, const f16* values, const int* table,
                                                 const int* lens, const int* new_lens, float* part_o, float4* part_st,
                                                 float (&so)[4][16][DV + 4], float (&sm)[4][16], float (&sl)[4][16],
                                                 float (&sr)[16], int64_t (&place)[16]) {
  constexpr int NT = DV / 16;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const PrefixPlace at(a.H, pa.rblocks);
  const int h = at.h, kb = at.sp * shared.split;
  const PrefixBlock blk = prefix_block(pa.starts, shared.groups, pa.count, a.n, 16 * QT, at.rb, lane);
  if (!blk.found) return;
  PrefixRow row[QT];
  int some = -1, keys = 0;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    row[t] = prefix_row(a, shared, blk, pa.members, lens, new_lens, 16 * t + c16);
    const uint64_t there = __ballot(row[t].b >= 0);
    const int first = there ? __builtin_ctzll(there) : 0, b = __shfl(row[t].b, first), k = __shfl(row[t].keys, first);
    keys = some < 0 ? k : keys;
    some = some < 0 ? b : some;
  }
  some = __builtin_amdgcn_readfirstlane(some);
  keys = __builtin_amdgcn_readfirstlane(keys);
  if (some < 0 || kb >= keys) return;
  const int ke = at.sp == shared.np - 1 ? keys : min(keys, kb + shared.split);
  const CacheSource<M, DV> src(a, codes, values, table, some, h, lane);

  CacheTile<M, DV> A[1], B[1];
  int tile = kb / 32 + w, pc = 0, pn = 0;
  const int last = ke / 32;  // prefixes are whole pages, pieces whole tiles
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

  // the waves' sums, 16 rows at a time
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (t) __syncthreads();
    float ref, l;
    R.finish(t, ref, l);
#pragma unroll
    for (int c = 0; c < NT; ++c) *reinterpret_cast<f32x4*>(&so[w][c16][16 * c + 4 * g]) = R.O[t][c];
    if (g == 0) {
      sm[w][c16] = ref;
      sl[w][c16] = l;
      if (w == 0) {
        sr[c16] = rc[t];
        place[c16] = part_of(a, shared, row[t], h, at.sp);
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 4 * DV; e += 256) {
      const int q = e / (DV / 4), c = 4 * (e % (DV / 4));
      if (place[q] < 0) continue;
      float m = sm[0][q];
#pragma unroll
      for (int k = 1; k < 4; ++k) m = fmaxf(m, sm[k][q]);
      l = 0.f;
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
}

// More rows: 64 of a group, 16 for each wave; the keys pass through LDS as in
// cache_attn_rows_kernel, 64 a stage and three stages, every one of them seen by all rows.
template <int M, int DV>
__device__ __forceinline__ void cache_prefix_rows(const CacheAttnArgs& a, const CacheShared& shared,
                                                  const PrefixArgs& pa, const f16* phi, const f16* gate_q,
                                                  const f16* gate_k, const f16* codes, const f16* values,
                                                  const int* table, const int* lens, const int* new_lens,
                                                  float* part_o, float4* part_st,
                                                  char (&lds)[3][2 * CacheTile<M, DV>::kFrags * 1024]) {
  constexpr int KC = CacheTile<M, DV>::KC, NT = DV / 16, NF = CacheTile<M, DV>::kFrags, PER = NF / 2;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const PrefixPlace at(a.H, pa.rblocks);
  const int h = at.h, kb = at.sp * shared.split;
  const PrefixBlock blk = prefix_block(pa.starts, shared.groups, pa.count, a.n, 64, at.rb, lane);
  if (!blk.found) return;
  // lane r looks up row r of the block; all waves find the same
  const PrefixRow all = prefix_row(a, shared, blk, pa.members, lens, new_lens, lane);
  const uint64_t there = __ballot(all.b >= 0);
  if (!there) return;
  const int some = __builtin_amdgcn_readfirstlane(__shfl(all.b, __builtin_ctzll(there)));
  const int keys = __builtin_amdgcn_readfirstlane(__shfl(all.keys, __builtin_ctzll(there)));
  if (kb >= keys) return;
  const int ke = at.sp == shared.np - 1 ? keys : min(keys, kb + shared.split);
  const PrefixRow row{__shfl(all.b, 16 * w + c16), __shfl(all.i, 16 * w + c16), keys};
  const CacheSource<M, DV> src(a, codes, values, table, some, h, lane);
  const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  const int tile0 = kb / 32, tiles = (ke - kb) / 32, stages = (tiles + 1) / 2;
  // a stage lies in one page, or in two of 32 tokens (of which the last stage may have one)
  const bool two = a.lp == 5;
  auto page = [&](int st, int i) {
    return src.row[two ? tile0 + min(2 * st + i, tiles - 1) : (32 * tile0 + 64 * st) >> a.lp];
  };
  // this wave's operands of a stage, as in cache_attn_rows_kernel
  unsigned koff[KC], voff[NT / 2], kto[KC], vto[NT / 2];
#pragma unroll
  for (int i = 0; i < KC; ++i) {
    const int f = w + 4 * i, t = f / (2 * KC), o = f % (2 * KC);
    koff[i] = 2u * (unsigned)(((c16 >> 2) * 8 + (c16 & 3) + 4 * (o / KC) + (two ? 0 : 32 * t)) * M + 32 * (o % KC) +
                              (M == 16 ? 8 * (g & 1) : 8 * g));
    kto[i] = base + 1024u * (unsigned)(NF * t + o);
  }
#pragma unroll
  for (int i = 0; i < NT / 2; ++i) {
    const int f = w + 4 * i, t = f / NT, o = f % NT;
    voff[i] = 2u * (unsigned)((g + (two ? 0 : 4 * t)) * (DV * 8) + c16 * 8 + 128 * o);
    vto[i] = base + 1024u * (unsigned)(NF * t + 2 * KC + o);
  }
  const char* const kh = reinterpret_cast<const char*>(codes + (((int64_t)h * M) << a.lp));
  const char* const vh = reinterpret_cast<const char*>(values + (((int64_t)h * DV) << a.lp));
  const unsigned kpage = (unsigned)(a.H * M * 2) << a.lp, vpage = (unsigned)(a.H * DV * 2) << a.lp;  // bytes, <= 2^25
  constexpr unsigned kStage = 2 * NF * 1024;
  unsigned fill = 0, read = 0;  // where the next stage goes, and the one at hand is
  int slot = (32 * tile0) & ((1 << a.lp) - 1);
  auto issue = [&](const int(&p)[2]) {
    const unsigned pg = src.exists(p[0]) ? (unsigned)p[0] : 0u;
    const char *k[2], *v[2];
    k[0] = k[1] = kh + ((uint64_t)pg * kpage + (unsigned)(slot * M * 2));
    v[0] = v[1] = vh + ((uint64_t)pg * vpage + (unsigned)(slot * DV * 2));
    if (two) {
      const unsigned p1 = src.exists(p[1]) ? (unsigned)p[1] : 0u;
      k[1] = kh + (uint64_t)p1 * kpage;
      v[1] = vh + (uint64_t)p1 * vpage;
    }
#pragma unroll
    for (int i = 0; i < KC; ++i) lds_dma16_so(k[(w + 4 * i) / (2 * KC)], koff[i], kto[i] + fill);
#pragma unroll
    for (int i = 0; i < NT / 2; ++i) lds_dma16_so(v[(w + 4 * i) / NT], voff[i], vto[i] + fill);
    fill = fill == 2 * kStage ? 0 : fill + kStage;
    slot = (slot + 64) & ((1 << a.lp) - 1) & ~63;  // 0 with pages of 32
  };
  int pg[4][2];  // pages of the stage at hand and the next three
  auto pages_of = [&](int st, int(&p)[2]) {
    p[0] = p[1] = page(st, 0);
    if (two) p[1] = page(st, 1);
  };
#pragma unroll
  for (int st = 0; st < 4; ++st) pg[st][0] = pg[st][1] = -1;
#pragma unroll
  for (int st = 0; st < 3; ++st)
    if (st < stages) pages_of(st, pg[st]);
  issue(pg[0]);
  if (stages > 1) issue(pg[1]);

  CacheRows<M, DV, 1, true> R;
  float rc[1];
  R.start_rows(a, gate_q, gate_k, h, lane, rc, [&](int) {
    const int b = row.b >= 0 ? row.b : some, i = row.b >= 0 ? row.i : 0;
    return phi + (((int64_t)b * a.n + i) * a.H + h) * M;
  });
  auto get = [&](CacheTile<M, DV>& T, int i) {
    const char* from = &lds[0][0] + read + 16 * lane + 1024 * NF * i;
#pragma unroll
    for (int f = 0; f < NF - NT; ++f) T.k[f / KC][f % KC] = *reinterpret_cast<const f16x8*>(from + 1024 * f);
#pragma unroll
    for (int c = 0; c < NT; ++c) T.v[c] = *reinterpret_cast<const f16x8*>(from + 1024 * (NF - NT + c));
  };
  for (int st = 0; st < stages; ++st) {
    // this wave's part of the stage has landed (the next stage's may not have)
    if (st + 1 < stages)
      wait_vmcnt_lgkm0<PER>();
    else
      wait_vmcnt_lgkm0<0>();
    asm volatile("s_barrier" ::: "memory");  // ... and every wave's; the stage before is free
    if (st + 2 < stages) issue(pg[2]);
    if (st + 3 < stages) pages_of(st + 3, pg[3]);
    if (2 * st + 1 < tiles && src.exists(pg[0][0]) && src.exists(pg[0][1])) {
      CacheTile<M, DV> T[2];
      get(T[0], 0);
      get(T[1], 1);
      R.add_clear(T);
    } else {
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (2 * st + i >= tiles || !src.exists(pg[0][i])) continue;  // uniform
        CacheTile<M, DV> T[1];
        get(T[0], i);
        R.add_clear(T);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      pg[0][i] = pg[1][i];
      pg[1][i] = pg[2][i];
      pg[2][i] = pg[3][i];
    }
    read = read == 2 * kStage ? 0 : read + kStage;
  }
  float ref, l;
  R.finish(0, ref, l);
  const int64_t place = part_of(a, shared, row, h, at.sp);
  if (place < 0) return;
#pragma unroll
  for (int c = 0; c < NT; ++c) *reinterpret_cast<f32x4*>(part_o + place * DV + 16 * c + 4 * g) = R.O[0][c];
  if (g == 0) part_st[place] = float4{ref, l, rc[0], 0.f};
}

// Both in one launch, the prefixes first, whose workgroups are the longer ones: one
// launch less, and they fill each other's gaps. QT: the prefixes' blocks of 16 rows a
// wave, 0: through LDS.
template <int QT>
struct CacheJoint : CacheShared {
  static constexpr bool kJoint = true;
  PrefixArgs pa;
  __device__ __forceinline__ int first_block() const { return pa.blocks; }
  // Whether this workgroup was one of the prefixes'. ring: the rest's, where it has one.
  template <int M, int DV, class... Ring>
  __device__ __forceinline__ bool prefix(const CacheAttnArgs& a, const f16* phi, const f16* gate_q, const f16* gate_k,
                                         const f16* codes, const f16* values, const int* table, const int* lens,
                                         const int* new_lens, float* part_o, float4* part_st, Ring&... ring) const {
    if ((int)blockIdx.x >= pa.blocks) return false;
    if constexpr (QT > 0) {
      __shared__ __align__(16) float so[4][16][DV + 4];
      __shared__ float sm[4][16], sl[4][16], sr[16];
      __shared__ int64_t place[16];
      cache_prefix_few<M, DV, QT>(a, *this, pa, phi, gate_q, gate_k, codes, values, table, lens, new_lens, part_o,
                                  part_st, so, sm, sl, sr, place);
    } else {
      cache_prefix_rows<M, DV>(a, *this, pa, phi, gate_q, gate_k, codes, values, table, lens, new_lens, part_o, part_st,
                               ring...);
    }
    return true;
  }
};

namespace {
template <int M, int DV>
hipError_t launch_cache_shared_t(const CacheDims& d, const CacheSharedPlan& p, CacheAttnArgs a,
                                 const CacheShared& shared, const CacheSharedCall& call, const f16* phi,
                                 const f16* gate_q, const f16* gate_k, const f16* codes, const f16* values,
                                 const int* table, const int* lens, const int* new_lens, const int64_t* tree,
                                 f16* out, float* lse, const CacheAttnBuffers& part, hipStream_t s) {
  const PrefixArgs pa{call.members, call.starts, call.members_count, p.rblocks, d.H * p.rblocks * p.np};
  const dim3 grid((unsigned)(pa.blocks + (int64_t)d.B * d.H * p.rest.qblocks * p.rest.nsplit)), block(256);
#define MORPHO_CACHE_SHARED(QT, ...)                                                                              \
  MORPHO_KLAUNCH((__VA_ARGS__, CacheJoint<QT>>), grid, block, 0, s, a, (CacheJoint<QT>{shared, pa}), phi, gate_q, gate_k, \
                 codes, values, table, lens, new_lens, tree, out, lse, part.o, part.st)
  if (p.qt == 0)
    MORPHO_CACHE_SHARED(0, cache_attn_rows_kernel<M, DV, 1, true);
  else if (p.qt == 1)
    MORPHO_CACHE_SHARED(1, cache_attn_few_kernel<M, DV);
  else
    MORPHO_CACHE_SHARED(2, cache_attn_few_kernel<M, DV);
#undef MORPHO_CACHE_SHARED
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
