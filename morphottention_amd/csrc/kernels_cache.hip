// Kernels of the paged cache: attention over it (cache_attn.h), appending, page copies and compaction.
#include "cache_attn.h"
#include "common.h"
#include "gemm.h"
#include "internal.h"

namespace morpho {

namespace {
template <int M, int DV>
hipError_t launch_cache_attn_t(const CacheDims& d, const CacheAttnPlan& p, const CacheAttnArgs& a, const f16* phi,
                               const f16* gate_q, const f16* gate_k, const f16* codes, const f16* values,
                               const int* table, const int* lens, const int* new_lens, const int64_t* tree, f16* out,
                               float* lse, const CacheAttnBuffers& part, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)d.B * d.H * p.qblocks * p.nsplit)), block(256);
#define MORPHO_CACHE_ATTN(...)                                                                                     \
  MORPHO_KLAUNCH((__VA_ARGS__), grid, block, 0, s, a, CacheApart{}, phi, gate_q, gate_k, codes, values, table, lens, new_lens, \
                 tree, out, lse, part.o, part.st)
  if (p.qt == 0)
    MORPHO_CACHE_ATTN(cache_attn_few_kernel<M, DV, CacheApart>);
  else if (p.pairs)
    MORPHO_CACHE_ATTN(cache_attn_rows_kernel<M, DV, 1, true, CacheApart>);
  else if (p.qt == 2)
    MORPHO_CACHE_ATTN(cache_attn_rows_kernel<M, DV, 2, false, CacheApart>);
  else if constexpr (M <= 32 && DV <= 64)
    MORPHO_CACHE_ATTN(cache_attn_rows_kernel<M, DV, 1, false, CacheApart>);
#undef MORPHO_CACHE_ATTN
  return hipGetLastError();
}
}  // namespace

hipError_t launch_cache_attn(const CacheDims& d, const CacheAttnPlan& plan, const f16* phi, const f16* gate_q,
                             const f16* gate_k, const f16* codes, const f16* values, const int* table,
                             const int* lens, const int* new_lens, const int64_t* tree, f16* out, float* lse,
                             const CacheAttnBuffers& part, float scale, int causal, int mask_diag, hipStream_t s) {
  CacheAttnArgs a = attn_args(d, plan, causal, mask_diag);
  a.sl2e = scale * kLog2e;
  MORPHO_MDV_DISPATCH(launch_cache_attn_t, d, plan, a, phi, gate_q, gate_k, codes, values, table, lens, new_lens, tree,
                      out, lse, part, s);
}

hipError_t launch_cache_attn_join(const CacheDims& d, const CacheAttnPlan& plan, const f16* values, const int* table,
                                  const int* lens, const int* new_lens, const int64_t* tree,
                                  const CacheAttnBuffers& part, f16* out, float* lse, int causal, int mask_diag,
                                  hipStream_t s) {
  const CacheAttnArgs a = attn_args(d, plan, causal, mask_diag);
  const int64_t rows = (int64_t)d.B * d.H * d.n;
  // few pieces: one group a row, its loads all independent; many: groups that share them
#define MORPHO_CACHE_JOIN(DV, NG)                                                                            \
  MORPHO_KLAUNCH((cache_join_kernel<DV, NG, CacheApart>), dim3((unsigned)((rows * (DV / 4) * NG + 255) / 256)), dim3(256), 0, s, \
                 a, CacheApart{}, rows, values, table, lens, new_lens, tree, part.o, part.st, out, lse)
  const bool many = plan.nsplit > 8;
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

// ---------------------------------------------------------------- append
struct CacheAppendArgs {
  int T, n, D, H, C, HM;  // T = B n tokens, C = H (M + DV) columns, the first HM of them codes
  int lm, ldv;            // log2 of M and DV
  int W, pages, lp, proj;
  int NR, TR, shift;  // rows of a sequence in the tile kernel's row space, rows in all, whether shifted
};

// Where new token i of sequence b goes: the row of its page's head 0 in the
// pool's rows of tokens, [page][head][slot]; -1: nowhere.
__device__ __forceinline__ int64_t token_row(const CacheAppendArgs& a, const int* __restrict__ table,
                                             const int* __restrict__ lens, const int* __restrict__ new_lens, int b,
                                             int i) {
  const int have = max(lens[b], 0), nb = new_lens ? new_lens[b] : a.n;
  const int64_t pos = (int64_t)have + i;
  if (i >= nb || pos >= ((int64_t)a.W << a.lp)) return -1;
  const int page = table[(int64_t)b * a.W + (pos >> a.lp)];
  return (unsigned)page < (unsigned)a.pages ? (((int64_t)page * a.H) << a.lp) + (pos & ((1 << a.lp) - 1)) : -1;
}
// Columns of the projection in the pool: a code, a value (of 8-token groups).
__device__ __forceinline__ f16* code_place(const CacheAppendArgs& a, f16* codes, int64_t row, int c) {
  return codes + ((row + ((int64_t)(c >> a.lm) << a.lp)) << a.lm) + (c & ((1 << a.lm) - 1));
}
__device__ __forceinline__ f16* value_place(const CacheAppendArgs& a, f16* values, int64_t row, int c) {
  const int v = c - a.HM;
  return values + (((row & ~(int64_t)7) + ((int64_t)(v >> a.ldv) << a.lp)) << a.ldv) +
         8 * (v & ((1 << a.ldv) - 1)) + (row & 7);
}

// Few tokens: a workgroup of 8 waves per 16 CT output columns and 16 TT
// tokens. Each wave contracts an eighth of D, 64 wide steps that it brings to
// LDS for itself (no barriers), and the partial tiles are added in LDS, the
// upper four waves' first.
// The operands go through LDS because a lane of the MFMA holds 16 bytes of the
// row lane % 16: loaded so from row-major memory, neighbouring lanes are rows
// apart, and the address unit takes them one at a time. Here eight neighbours
// fetch a 128-byte line of a row (place p of row r holds k chunk p ^ (r / 2 %
// 8), so that the reads of 16 rows of one chunk hit all banks). T 192, D 2048,
// C 4096: 19.4 us loaded directly, 13.1 by half lines (the L1 loses the other
// half before its turn), 10.8 so.
template <int CT, int TT>
__global__ __launch_bounds__(512) void cache_append_rows_kernel(CacheAppendArgs a, const f16* __restrict__ X,
                                                               const f16* __restrict__ Wt, f16* __restrict__ codes,
                                                               f16* __restrict__ values,
                                                               const int* __restrict__ table,
                                                               const int* __restrict__ lens,
                                                               const int* __restrict__ new_lens,
                                                               f16* __restrict__ phi) {
  // operands of a step, 2 KiB each, and steps in LDS: two where three fit (one
  // more was up to 8 % slower; the waves cover each other's waits), one of the
  // smallest, where the first wait counts most
  constexpr int NF = CT + TT, NS = NF == 3 || NF == 4 ? 2 : 1;
  constexpr int kStage = NF * 2048, kSum = 4 * 16 * TT * (16 * CT + 4) * 4;
  __shared__ __align__(1024) char smem[8 * NS * kStage > kSum ? 8 * NS * kStage : kSum];
  auto part = reinterpret_cast<float(*)[16 * TT][16 * CT + 4]>(smem);  // [wave][token][column]
  __shared__ int64_t slot[16 * TT];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int col0 = blockIdx.x * 16 * CT, t0 = blockIdx.y * 16 * TT;
  f32x4 acc[CT][TT];
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[c][t] = f32x4{};
  const int steps = (a.D + 63) / 64, s0 = steps * w / 8, ns = steps * (w + 1) / 8 - s0;  // this wave's steps
  // a lane's byte offsets from the step's first k of row 0 of the tile, 8 rows
  // at a time; rows past the end repeat the last
  unsigned off[NF][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 8 * i + (lane >> 3), chunk = (lane & 7) ^ ((r >> 1) & 7);
#pragma unroll
    for (int c = 0; c < CT; ++c) off[c][i] = (unsigned)(min(16 * c + r, a.C - 1 - col0) * a.D + 8 * chunk) * 2u;
#pragma unroll
    for (int t = 0; t < TT; ++t) off[CT + t][i] = (unsigned)(min(16 * t + r, a.T - 1 - t0) * a.D + 8 * chunk) * 2u;
  }
  // D is a multiple of 32: of a last step of 32 the upper chunks repeat the lower ones, for nothing
  const bool odd = (a.D & 63) != 0;
  const unsigned upper[2] = {((lane & 7) ^ ((lane >> 4) & 7)) >= 4 ? 64u : 0u,
                             ((lane & 7) ^ (((lane >> 4) + 4) & 7)) >= 4 ? 64u : 0u};
  const char* wp = reinterpret_cast<const char*>(Wt + (int64_t)col0 * a.D + 64 * s0);
  const char* xp = reinterpret_cast<const char*>(X + (int64_t)t0 * a.D + 64 * s0);
  const unsigned mine = (unsigned)(w * NS * kStage);
  const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)smem + mine;
  unsigned at = 0;  // place of the step at hand, which the step NS behind it takes
  auto issue = [&](int i, unsigned to) {
    const bool half = odd && s0 + i == steps - 1;
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
      for (int k = 0; k < 2; ++k)
        lds_dma16_so(f < CT ? wp : xp, off[f][k] - (half ? upper[k] : 0u), base + to + 2048u * f + 1024u * k);
    wp += 128;
    xp += 128;
  };
#pragma unroll
  for (int i = 0; i < NS; ++i)
    if (i < ns) issue(i, (unsigned)(i * kStage));
  if (threadIdx.x < 16 * TT) {
    const int t = min(t0 + (int)threadIdx.x, a.T - 1), b = t / a.n;
    slot[threadIdx.x] = token_row(a, table, lens, new_lens, b, t - b * a.n);
  }
  for (int i = 0; i < ns; ++i) {
    // the step has landed, those behind it may not have
    if (NS > 1 && i + NS <= ns)
      wait_vmcnt<(NS - 1) * 2 * NF>();
    else
      wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    f16x8 fr[2][NF];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int f = 0; f < NF; ++f)
        fr[k][f] = *reinterpret_cast<const f16x8*>(smem + mine + at + 2048 * f + 128 * c16 +
                                                   16 * ((4 * k + g) ^ ((c16 >> 1) & 7)));
    // read, so that the next step may take its place
    __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    if (i + NS < ns) issue(i + NS, at);
    at = at == (NS - 1) * kStage ? 0 : at + kStage;
    const bool half = odd && s0 + i == steps - 1;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k == 1 && half) break;  // uniform
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[c][t] = mfma16x16(fr[k][c], fr[k][CT + t], acc[c][t]);
    }
  }
  __syncthreads();  // the sums take the steps' place
  auto place = [&](int c, int t) { return reinterpret_cast<f32x4*>(&part[w & 3][16 * t + c16][16 * c + 4 * g]); };
  if (w >= 4) {
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int t = 0; t < TT; ++t) *place(c, t) = acc[c][t];
  }
  __syncthreads();
  if (w < 4) {  // each place is read and written by one lane
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int t = 0; t < TT; ++t) *place(c, t) += acc[c][t];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 256 * CT * TT; e += 512) {
    const int c = col0 + e % (16 * CT), tok = e / (16 * CT), t = t0 + tok;
    if (t >= a.T || c >= a.C) continue;
    float z = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) z += part[k][tok][e % (16 * CT)];
    const int64_t row = slot[tok];
    if (c < a.HM) {
      const f16 y = (f16)cube_project(z, a.proj);
      phi[(int64_t)t * a.HM + c] = y;
      if (row >= 0) *code_place(a, codes, row, c) = y;
    } else if (row >= 0) {
      *value_place(a, values, row, c) = (f16)z;
    }
  }
}

// Many tokens: 128 x 128 tiles (tokens x columns) of the GEMM main loop. Its
// row space gives each sequence NR rows. With shift, row r of a sequence is
// the position lens % 8 back from the first new one, + r, so that 8 rows of a
// tile are the 8 tokens of a value group and are stored as one; a few rows at
// both ends of a sequence repeat a token and are not stored. What bounds it:
// the main loop's LDS reads and the latency of its two stages (one round of
// tiles 15 us at D 1024, 28 at 2048; three or four stages, one workgroup to a
// CU: 1 us less there and up to 25 % more for more rounds; 256 x 256 tiles: 10 %
// less at T 16384 D 2048 C 4096, up to twice as much for fewer).
struct AppendRows {
  const int* lens;  // null: no shift
  int NR, n;
  __device__ __forceinline__ int shift(int b) const { return lens ? max(lens[b], 0) & 7 : 0; }
  __device__ __forceinline__ int operator()(int r) const {
    const int b = r / NR;
    return b * n + min(max(r - b * NR - shift(b), 0), n - 1);
  }
};

// 4 x 4 halves among the four lanes of a quad: lane q has column q's rows 0 ..
// 3 and gets row q's columns 0 .. 3.
__device__ __forceinline__ f16x4 quad_transpose(f16x4 x, int lane) {
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 d = __builtin_bit_cast(u32x2, x);
  const bool up = lane & 2, odd = lane & 1;
  const unsigned far = (unsigned)__builtin_amdgcn_mov_dpp((int)(up ? d[0] : d[1]), 0x4e /* lane ^ 2 */, 0xf, 0xf, false);
  const unsigned lo = up ? far : d[0], hi = up ? d[1] : far;  // rows 0, 1 (up: 2, 3) of columns q & 1, (q & 1) + 2
  const unsigned l = __builtin_amdgcn_perm(hi, lo, 0x05040100), h = __builtin_amdgcn_perm(hi, lo, 0x07060302);
  const unsigned mine = odd ? h : l;  // row q of the two columns
  const unsigned near = (unsigned)__builtin_amdgcn_mov_dpp((int)(odd ? l : h), 0xb1 /* lane ^ 1 */, 0xf, 0xf, false);
  const unsigned c0 = odd ? near : mine, c1 = odd ? mine : near;
  return __builtin_bit_cast(f16x4, u32x2{__builtin_amdgcn_perm(c1, c0, 0x05040100),
                                         __builtin_amdgcn_perm(c1, c0, 0x07060302)});
}
// v_permlane16_swap: the odd 16-lane rows of a change places with the even
// ones of b (a' = a0 b0 a2 b2, b' = a1 b1 a3 b3).
__device__ __forceinline__ void swap_rows16(f16x4& a, f16x4& b) {
  typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
  u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(x[i], y[i], false, false);
    x[i] = r[0];
    y[i] = r[1];
  }
  a = __builtin_bit_cast(f16x4, x);
  b = __builtin_bit_cast(f16x4, y);
}

__global__ __launch_bounds__(kGemmThreads) void cache_append_tile_kernel(
    CacheAppendArgs a, const f16* __restrict__ X, const f16* __restrict__ Wt, f16* __restrict__ codes,
    f16* __restrict__ values, const int* __restrict__ table, const int* __restrict__ lens,
    const int* __restrict__ new_lens, f16* __restrict__ phi) {
  constexpr int BM = 128, BN = 128;
  using G = Gemm<BM, BN, 2, true, true, 64, 2>;
  static_assert(G::FJ % 2 == 0, "column blocks in pairs");
  __shared__ __align__(16) char lds[G::kLdsBytes];
  const int ntm = (a.TR + BM - 1) / BM, ntn = (a.C + BN - 1) / BN;
  int tr, tc;
  if (!gemm_tile_map(blockIdx.x, ntm, ntn, tr, tc)) return;
  const int m0 = BM * tr, n0 = BN * tc;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const AppendRows rows{a.shift ? lens : nullptr, a.NR, a.n};
  // the tile's rows: token (-1: none) and place in the pool (-1: not stored),
  // looked up before the main loop, which hides the chain of loads
  int my_token = -1;
  int64_t my_place = -1;
  if (threadIdx.x < BM && m0 + (int)threadIdx.x < a.TR) {
    const int r = m0 + threadIdx.x, b = r / a.NR, i = r - b * a.NR - rows.shift(b);
    if (i >= 0 && i < a.n) {
      my_token = b * a.n + i;
      my_place = token_row(a, table, lens, new_lens, b, i);
    }
  }
  f32x4 acc[G::FI][G::FJ];
  G::run(X, a.D, Wt, a.D, a.TR, a.C, m0, n0, 0, a.D, lds, acc, rows);
  auto token = reinterpret_cast<int*>(lds);
  auto place = reinterpret_cast<int64_t*>(lds + BM * 4);
  if (threadIdx.x < BM) {
    token[threadIdx.x] = my_token;
    place[threadIdx.x] = my_place;
  }
  __syncthreads();
  const int wm = w / G::WN, wn = w % G::WN, c16 = lane & 15, g = lane >> 4;
#pragma unroll
  for (int j = 0; j < G::FJ; ++j) {
    const int col = n0 + G::WTN * wn + 16 * j;  // 16 columns of one head's codes or values
    if (col >= a.HM) continue;
#pragma unroll
    for (int i = 0; i < G::FI; ++i) {
      f16x4 y;
#pragma unroll
      for (int r = 0; r < 4; ++r) y[r] = (f16)cube_project(acc[i][j][r], a.proj);
      y = quad_transpose(y, lane);
      const int rt = G::WTM * wm + 16 * i + 4 * g + (c16 & 3), c = col + (c16 & ~3);
      if (token[rt] >= 0) *reinterpret_cast<f16x4*>(phi + (int64_t)token[rt] * a.HM + c) = y;
      if (place[rt] >= 0) *reinterpret_cast<f16x4*>(code_place(a, codes, place[rt], c)) = y;
    }
  }
#pragma unroll
  for (int j = 0; j < G::FJ; j += 2) {
    const int col = n0 + G::WTN * wn + 16 * j;
    if (col + 16 < a.HM || col >= a.C) continue;
    // lane rows 0 and 2: column block j, 1 and 3: block j + 1; 8 rows of each
    const int c = col + 16 * (g & 1) + c16;
    const bool mine = c >= a.HM && c < a.C;
#pragma unroll
    for (int i = 0; i < G::FI; ++i) {
      f16x4 lo, hi;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        lo[r] = (f16)acc[i][j][r];
        hi[r] = (f16)acc[i][j + 1][r];
      }
      swap_rows16(lo, hi);
      const f16x8 y = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      const int rt = G::WTM * wm + 16 * i + 8 * (g >> 1);
      const int64_t first = place[rt], last = place[rt + 7];
      if (!mine) continue;
      // 8 tokens of one group: no two sequences store to one page, and the
      // stored tokens of a sequence follow each other
      if (first >= 0 && (first & 7) == 0 && last == first + 7) {
        *reinterpret_cast<f16x8*>(value_place(a, values, first, c)) = y;
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int64_t p = place[rt + r];
          if (p >= 0) *value_place(a, values, p, c) = y[r];
        }
      }
    }
  }
}

hipError_t launch_cache_append(const CacheDims& d, const f16* X, const f16* W, f16* codes, f16* values,
                               const int* table, const int* lens, const int* new_lens, f16* phi, int proj,
                               hipStream_t s) {
  CacheAppendArgs a{};
  a.T = d.B * d.n;
  a.n = d.n;
  a.D = d.H * d.DV;
  a.H = d.H;
  a.C = d.H * (d.M + d.DV);
  a.HM = d.H * d.M;
  a.lm = log2_of(d.M);
  a.ldv = log2_of(d.DV);
  a.W = d.W;
  a.pages = d.pages;
  a.lp = log2_of(d.P);
  a.proj = proj;
  a.NR = cache_append_rows(d.B, d.n, a.C);
  a.TR = d.B * a.NR;
  a.shift = a.NR != d.n;
  const CacheAppendShape p = cache_append_shape(a.T, a.C);
  if (p.tokens) {
    const dim3 grid((a.C + 16 * p.columns - 1) / (16 * p.columns), (a.T + 16 * p.tokens - 1) / (16 * p.tokens));
#define MORPHO_CACHE_APPEND(CT, TT)                                                                               \
  MORPHO_KLAUNCH((cache_append_rows_kernel<CT, TT>), grid, dim3(512), 0, s, a, X, W, codes, values, table, lens, \
                 new_lens, phi)
    if (p.tokens == 1)
      MORPHO_CACHE_APPEND(1, 1);
    else if (p.tokens == 2 && p.columns == 1)
      MORPHO_CACHE_APPEND(1, 2);
    else if (p.tokens == 2)
      MORPHO_CACHE_APPEND(2, 2);
    else if (p.columns == 2)
      MORPHO_CACHE_APPEND(2, 4);
    else
      MORPHO_CACHE_APPEND(4, 4);
#undef MORPHO_CACHE_APPEND
  } else {
    const dim3 grid(gemm_tile_grid((a.TR + 127) / 128, (a.C + 127) / 128));
    MORPHO_KLAUNCH(cache_append_tile_kernel, grid, dim3(kGemmThreads), 0, s, a, X, W, codes, values, table, lens,
                   new_lens, phi);
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------- page copies
// One launch for all layers: 16 KiB of a page's codes or values a workgroup,
// four loads of a lane in flight. Bound by memory: 550 MB read and written (2
// layers, 700 pages) in 111 us, 5.0 TB/s, a large copy's rate.
constexpr int kCopyBytes = 16384;
__global__ __launch_bounds__(256) void cache_copy_kernel(char* __restrict__ codes, char* __restrict__ values,
                                                        const int* __restrict__ src, const int* __restrict__ dst,
                                                        int pages, int64_t cbytes, int64_t vbytes, int nc, int nv) {
  const int64_t id = blockIdx.x;
  const int piece = (int)(id % (nc + nv));
  const int pair = blockIdx.y, layer = blockIdx.z;
  const int from = src[pair], to = dst[pair];
  if ((unsigned)from >= (unsigned)pages || (unsigned)to >= (unsigned)pages) return;
  const bool val = piece >= nc;
  const int64_t size = val ? vbytes : cbytes, off = (int64_t)(val ? piece - nc : piece) * kCopyBytes;
  char* pool = (val ? values : codes) + (int64_t)layer * pages * size;
  const char* p = pool + from * size + off;
  char* q = pool + to * size + off;
  const int64_t left = size - off;  // a multiple of 16
  i32x4 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int o = 16 * ((int)threadIdx.x + 256 * i);
    if (o < left) x[i] = *reinterpret_cast<const i32x4*>(p + o);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int o = 16 * ((int)threadIdx.x + 256 * i);
    if (o < left) *reinterpret_cast<i32x4*>(q + o) = x[i];
  }
}

hipError_t launch_cache_copy(const CacheDims& d, f16* codes, f16* values, const int* src, const int* dst, int count,
                             hipStream_t s) {
  const int64_t cb = (int64_t)d.H * d.P * d.M * 2, vb = (int64_t)d.H * d.P * d.DV * 2;
  const int nc = (int)((cb + kCopyBytes - 1) / kCopyBytes), nv = (int)((vb + kCopyBytes - 1) / kCopyBytes);
  // grid y and z hold 65535 each
  for (int at = 0; at < count; at += 65535) {
    const dim3 grid(nc + nv, count - at < 65535 ? count - at : 65535, d.layers);
    MORPHO_KLAUNCH(cache_copy_kernel, grid, dim3(256), 0, s, reinterpret_cast<char*>(codes),
                   reinterpret_cast<char*>(values), src + at, dst + at, d.pages, cb, vb, nc, nv);
  }
  return hipGetLastError();
}

// ---------------------------------------------------------------- compaction
// A token's place is at most its source (cache_compact_source leaves out what
// would move forward), so every source lies behind the places of the entries
// before it: a workgroup that moves its share of a sequence's tokens in order,
// each batch read whole before it is written, needs no other memory. A value's line holds 8 tokens of 8 columns, so a lone token
// touches 8 times its bytes; that bounds a tree's accepted path.
struct CompactArgs {
  int B, H, lm, pages, W, lp, K;
};
// A sequence's place in the pool.
struct CompactSeq {
  const int* table;
  int64_t base, cap;
  int H, pages, lp, count;
  __device__ __forceinline__ CompactSeq(const CompactArgs& a, const int* tables, const int* lens,
                                        const int* keep_lens, int b)
      : table(tables + (int64_t)b * a.W), base(max(lens[b], 0)), cap((int64_t)a.W << a.lp), H(a.H), pages(a.pages),
        lp(a.lp), count(keep_lens ? min(max(keep_lens[b], 0), a.K) : a.K) {}
  // row of head 0 of a position, [page][head][slot]; -1: there is none
  __device__ __forceinline__ int64_t place(int64_t pos) const {
    if (pos < 0 || pos >= cap) return -1;
    const int page = table[pos >> lp];
    return (unsigned)page < (unsigned)pages ? (((int64_t)page * H) << lp) + (pos & ((1 << lp) - 1)) : -1;
  }
  // where the k-th kept token, entry k of the row, comes from; -1: it stays or is not there
  __device__ __forceinline__ void move(int k, int entry, int64_t& from, int64_t& to) const {
    const int rel = cache_compact_source(entry, k);
    from = rel < 0 ? -1 : place(base + rel);
    to = place(base + k);
    if (from < 0 || from == to) to = -1;
  }
};

// Few tokens a sequence: one workgroup a (layer, sequence, group of 2^lh
// heads), 16 values a lane and batch. More heads a workgroup take the chain of
// loads up to the first value fewer times (12 layers B32 H16 dv64, up to 9
// tokens: one head 14.6 us, 8 12.6).
constexpr int kCompactValues = 4096;  // of a batch
template <int DV>
__global__ __launch_bounds__(256) void cache_compact_kernel(CompactArgs a, f16* codes, f16* values,
                                                           const int* __restrict__ table,
                                                           const int* __restrict__ lens,
                                                           const int* __restrict__ keep,
                                                           const int* __restrict__ keep_lens, int lh) {
  constexpr int TH = kCompactValues / DV;     // (token, head) pairs of a batch
  constexpr int VPER = kCompactValues / 256;  // values of a lane
  constexpr int CPER = (TH * 8 + 255) / 256;  // 8-code pieces of a lane, at most (cube_m 64)
  __shared__ int64_t from[TH], to[TH];
  const int H = a.H, lm = a.lm, lp = a.lp, groups = (H + (1 << lh) - 1) >> lh;
  int id = blockIdx.x;
  const int h0 = (id % groups) << lh;
  id /= groups;
  const int b = id % a.B, layer = id / a.B;
  const CompactSeq sq(a, table, lens, keep_lens, b);
  const int count = sq.count;
  codes += ((int64_t)layer * a.pages * H) << (lm + lp);
  values += ((int64_t)layer * a.pages * H * DV) << lp;
  const int batch = TH >> lh, heads = min(1 << lh, H - h0), lc = lm - 3;
  for (int k0 = 0; k0 < count; k0 += batch) {
    const int nk = min(batch, count - k0);
    if ((int)threadIdx.x < nk) {
      const int k = k0 + threadIdx.x;
      sq.move(k, keep[(int64_t)b * a.K + k], from[threadIdx.x], to[threadIdx.x]);
    }
    __syncthreads();
    f16x8 cv[CPER];
    f16 vv[VPER];
    // lane's i-th piece of codes: 2^lc of a (token, head) pair, and value
    auto code = [&](int i, const int64_t* at, bool& ok) {
      const int e = threadIdx.x + 256 * i, pair = e >> lc, k = pair >> lh, h = pair & ((1 << lh) - 1);
      ok = k < nk && h < heads && to[k] >= 0;
      return codes + (((ok ? at[k] : 0) + ((int64_t)(h0 + h) << lp)) << lm) + 8 * (e & ((1 << lc) - 1));
    };
    auto value = [&](int i, const int64_t* at, bool& ok) {
      const int e = threadIdx.x + 256 * i, pair = e / DV, k = pair >> lh, h = pair & ((1 << lh) - 1);
      ok = k < nk && h < heads && to[k] >= 0;
      const int64_t row = ok ? at[k] : 0;
      return values + ((row & ~(int64_t)7) + ((int64_t)(h0 + h) << lp)) * DV + 8 * (e % DV) + (row & 7);
    };
    bool ok;
#pragma unroll
    for (int i = 0; i < CPER; ++i) {
      const f16* p = code(i, from, ok);
      if (ok) cv[i] = *reinterpret_cast<const f16x8*>(p);
    }
#pragma unroll
    for (int i = 0; i < VPER; ++i) {
      const f16* p = value(i, from, ok);
      if (ok) vv[i] = *p;
    }
    wait_vmcnt<0>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CPER; ++i) {
      f16* p = code(i, to, ok);
      if (ok) *reinterpret_cast<f16x8*>(p) = cv[i];
    }
#pragma unroll
    for (int i = 0; i < VPER; ++i) {
      f16* p = value(i, to, ok);
      if (ok) *p = vv[i];
    }
    __syncthreads();  // the places are read before the next batch's are written
  }
}

// Many tokens a sequence: one workgroup a (layer, sequence, head, CW value
// columns or 2 CW codes), 4096 / CW tokens a batch, from a whole group of 8
// places on. A lane gathers the 8 values of a group and column and stores them
// as one; the next batch's places are found while this one's values come.
template <int DV, int CW>
__global__ __launch_bounds__(256) void cache_compact_long_kernel(CompactArgs a, f16* codes, f16* values,
                                                                const int* __restrict__ table,
                                                                const int* __restrict__ lens,
                                                                const int* __restrict__ keep,
                                                                const int* __restrict__ keep_lens) {
  constexpr int BT = kCompactValues / CW, CP = CW / 4;  // tokens of a batch; 8-code pieces of a slice
  // three batches' places: one is written while a slower wave still reads the one before last
  __shared__ int64_t from[3][BT], to[3][BT];
  const int H = a.H, lm = a.lm, lp = a.lp, code_slices = max((1 << lm) / (8 * CP), 1);
  int id = blockIdx.x;
  const int slice = id % (code_slices + DV / CW);
  id /= code_slices + DV / CW;
  const int h = id % H;
  id /= H;
  const int b = id % a.B, layer = id / a.B;
  const CompactSeq sq(a, table, lens, keep_lens, b);
  const int begin = -(int)(sq.base & 7);  // kept token of the first place of a group, mostly not one
  auto find = [&](int k0, int buf) {
    for (int at = threadIdx.x; at < BT; at += 256) {
      const int k = k0 + at;
      int64_t f = -1, t = -1;
      if (k >= 0 && k < sq.count) sq.move(k, keep[(int64_t)b * a.K + k], f, t);
      from[buf][at] = f;
      to[buf][at] = t;
    }
  };
  if (sq.count == 0) return;
  find(begin, 0);
  __syncthreads();
  int buf = 0;
  for (int k0 = begin; k0 < sq.count; k0 += BT) {
    const bool more = k0 + BT < sq.count;
    const int next = buf == 2 ? 0 : buf + 1;
    if (slice < code_slices) {
      f16* const pool = codes + (((int64_t)layer * a.pages * H) << (lm + lp)) + ((int64_t)h << (lm + lp)) +
                        8 * CP * slice;
      const int lc = min(lm - 3, __builtin_ctz(CP));  // log2 of the slice's pieces
      f16x8 cv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = threadIdx.x + 256 * i, k = e >> lc;
        if (k < BT && to[buf][k] >= 0)
          cv[i] = *reinterpret_cast<const f16x8*>(pool + (from[buf][k] << lm) + 8 * (e & ((1 << lc) - 1)));
      }
      if (more) find(k0 + BT, next);
      wait_vmcnt<0>();
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = threadIdx.x + 256 * i, k = e >> lc;
        if (k < BT && to[buf][k] >= 0)
          *reinterpret_cast<f16x8*>(pool + (to[buf][k] << lm) + 8 * (e & ((1 << lc) - 1))) = cv[i];
      }
    } else {
      f16* const pool = values + (((int64_t)layer * a.pages * H * DV) << lp) + (((int64_t)h * DV) << lp) +
                        8 * CW * (slice - code_slices);
      // lane: column threadIdx % CW of the slice, two groups
      f16x8 v[2];
      const int c = threadIdx.x % CW, g0 = threadIdx.x / CW;
      auto at = [&](int64_t row) { return pool + (row & ~(int64_t)7) * DV + 8 * c + (row & 7); };
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int k = 8 * (g0 + 256 / CW * i) + j;
          if (to[buf][k] >= 0) v[i][j] = *at(from[buf][k]);
        }
      if (more) find(k0 + BT, next);
      wait_vmcnt<0>();
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = 8 * (g0 + 256 / CW * i);
        bool all = true;  // a group lies in one page
#pragma unroll
        for (int j = 0; j < 8; ++j) all = all && to[buf][k + j] >= 0;
        if (all) {
          *reinterpret_cast<f16x8*>(at(to[buf][k])) = v[i];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (to[buf][k + j] >= 0) *at(to[buf][k + j]) = v[i][j];
        }
      }
    }
    // the barrier above lies between this batch's reads and its writes, and
    // behind the next batch's places; that batch reads nothing written here, for
    // its sources lie behind all of this one's places
    buf = next;
  }
}

template <int DV, int CW>
void launch_cache_compact_long(const CompactArgs& a, int64_t sequences, f16* codes, f16* values, const int* table,
                               const int* lens, const int* keep, const int* keep_lens, hipStream_t s) {
  const int code_slices = (1 << a.lm) / (2 * CW) > 1 ? (1 << a.lm) / (2 * CW) : 1;
  MORPHO_KLAUNCH((cache_compact_long_kernel<DV, CW>), dim3((unsigned)(sequences * a.H * (code_slices + DV / CW))),
                 dim3(256), 0, s, a, codes, values, table, lens, keep, keep_lens);
}

hipError_t launch_cache_compact(const CacheDims& d, f16* codes, f16* values, const int* table, const int* lens,
                                const int* keep, const int* keep_lens, int K, hipStream_t s) {
  const CompactArgs a{d.B, d.H, log2_of(d.M), d.pages, d.W, log2_of(d.P), K};
  const int64_t sequences = (int64_t)d.layers * d.B;
  const int heads = cache_compact_heads(sequences, d.H, d.DV, K);
  const dim3 block(256);
#define MORPHO_CACHE_COMPACT(DV)                                                                                   \
  do {                                                                                                             \
    if (heads)                                                                                                     \
      MORPHO_KLAUNCH((cache_compact_kernel<DV>), dim3((unsigned)(sequences * ((d.H + heads - 1) / heads))), block, \
                     0, s, a, codes, values, table, lens, keep, keep_lens, log2_of(heads));                       \
    else if (K <= 128)                                                                                             \
      launch_cache_compact_long<DV, 32>(a, sequences, codes, values, table, lens, keep, keep_lens, s);            \
    else if (K <= 256)                                                                                             \
      launch_cache_compact_long<DV, 16>(a, sequences, codes, values, table, lens, keep, keep_lens, s);            \
    else                                                                                                           \
      launch_cache_compact_long<DV, 8>(a, sequences, codes, values, table, lens, keep, keep_lens, s);             \
  } while (0)
  if (d.DV == 32)
    MORPHO_CACHE_COMPACT(32);
  else if (d.DV == 64)
    MORPHO_CACHE_COMPACT(64);
  else
    MORPHO_CACHE_COMPACT(128);
#undef MORPHO_CACHE_COMPACT
  return hipGetLastError();
}

}  // namespace morpho
