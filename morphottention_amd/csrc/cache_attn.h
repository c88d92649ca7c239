// Attention over the paged cache: serving a causal attention layer token by token.
//
// The score of a query i and a key j,
//   s_ij = scale sum_c G_c (2 phi_ic phi_jc - phi_ic - phi_jc),  G = gate_q gate_k,
// is s_ij = phi_j . u_i - r_i with u_ic = scale G_c (2 phi_ic - 1) and the row
// constant r_i = scale sum_c G_c phi_ic: what the key adds alone folds into
// the query. So the cache holds the codes phi_j and the values V_j and nothing
// else, both rounded to float16 once, and the attention over it is a plain
// dot product with u_i, exact for these stored numbers to fp32 rounding.
//
// Layout of a layer's pool, P tokens a page:
//   codes  [pages, H, P, M]          a key's codes contiguous
//   values [pages, H, P / 8, DV, 8]  eight tokens of one value column contiguous
// In the value product O^T += V^T P^T the contraction runs over the keys, so a
// lane's MFMA operand is 8 keys of one column: with this layout one 16-byte
// load from memory, without a transpose through LDS.
#pragma once

#include "common.h"
#include "internal.h"

namespace morpho {

namespace {

// What a sequence has: ctx tokens before the new ones, nb new ones, total keys.
struct SeqLen {
  int ctx, nb, total;
};
// Lengths outside their range are cut: a negative one counts as 0, what goes
// past the table's pages is not there.
__device__ __forceinline__ SeqLen seq_len(const int* __restrict__ lens, const int* __restrict__ new_lens, int b, int n,
                                          int cap) {
  SeqLen q;
  const int have = max(lens[b], 0);
  q.nb = new_lens ? min(max(new_lens[b], 0), n) : n;
  q.total = (int)min((int64_t)have + q.nb, (int64_t)cap);
  q.ctx = min(have, q.total);
  return q;
}

// Bits of an fp16 value: an infinity or a NaN.
__device__ __forceinline__ bool not_finite(f16 v) {
  return (__builtin_bit_cast(unsigned short, v) & 0x7c00) == 0x7c00;
}

}  // namespace

// ---------------------------------------------------------------- attention over the cache
struct CacheAttnArgs {
  int B, n, H, W, pages, lp;  // sequences, new tokens, heads, pages a sequence, pages, log2 of the page size
  int qblocks, nsplit, split_keys;
  float sl2e;  // scale log2 e
  int causal, mask_diag;
};

// Which sequences have their first pages in common (kernels_cache_shared.hip): those
// keys are the prefix kernel's, in pieces that come before a row's others.
struct CacheShared {
  static constexpr bool kJoint = false;  // whether a launch does the prefixes too, by its first workgroups
  const int* group;  // [B] a sequence's group; none where it is not one of them
  const int* pages;  // [G] the pages that a group's sequences have in common
  int groups, np, split;  // groups; pieces of a prefix, keys of a piece
  __device__ __forceinline__ int pieces() const { return np; }
  // Keys of sequence b that the prefix kernel takes: all of its group's, or, where
  // the sequence has not as many tokens, none.
  __device__ __forceinline__ int skip(int b, int ctx, int lp) const {
    const int g = group[b];
    if ((unsigned)g >= (unsigned)groups) return 0;
    const int64_t keys = (int64_t)max(pages[g], 0) << lp;
    return keys <= ctx ? (int)keys : 0;
  }
  __device__ __forceinline__ int pieces_of(int keys) const { return min(np, (keys + split - 1) / split); }
  __device__ __forceinline__ constexpr int first_block() const { return 0; }
};
// Nothing in common.
struct CacheApart {
  static constexpr bool kJoint = false;
  __device__ __forceinline__ constexpr int first_block() const { return 0; }
  __device__ __forceinline__ constexpr int pieces() const { return 0; }
  __device__ __forceinline__ constexpr int skip(int, int, int) const { return 0; }
  __device__ __forceinline__ constexpr int pieces_of(int) const { return 0; }
};

// One 32-key tile of one head in registers, as MFMA 16x16x32 A operands.
template <int M, int DV>
struct CacheTile {
  static constexpr int KC = M == 64 ? 2 : 1, NT = DV / 16;
  static constexpr int kFrags = 2 * KC + NT;  // 16 bytes a lane each
  f16x8 k[2][KC];  // block i: rows are keys 8 (r / 4) + 4 i + r % 4, so that the scores of both blocks
                   // come out as the value product's B operand (lane group g: keys 8 g .. 8 g + 7)
  f16x8 v[NT];     // 16 value columns each, keys 8 g .. 8 g + 7
};

// Where a wave reads a tile's operands from.
template <int M, int DV>
struct CacheSource {
  static constexpr int KC = CacheTile<M, DV>::KC, NT = CacheTile<M, DV>::NT;
  const f16 *kbase, *vbase;  // of this head and lane, page 0
  const int* row;            // the sequence's pages
  int64_t kstride, vstride;  // of a page
  int pages, lp;
  __device__ __forceinline__ CacheSource(const CacheAttnArgs& a, const f16* codes, const f16* values,
                                         const int* table, int b, int h, int lane)
      : row(table + (int64_t)b * a.W), pages(a.pages), lp(a.lp) {
    const int c16 = lane & 15, g = lane >> 4, P = 1 << a.lp;
    kbase = codes + (int64_t)h * P * M + ((c16 >> 2) * 8 + (c16 & 3)) * M + (M == 16 ? 8 * (g & 1) : 8 * g);
    vbase = values + (int64_t)h * P * DV + g * (DV * 8) + c16 * 8;
    kstride = (int64_t)a.H * P * M;
    vstride = (int64_t)a.H * P * DV;
  }
  __device__ __forceinline__ int page_of(int tile) const { return row[(tile * 32) >> lp]; }
  // a page that the pool does not have: its keys are left out
  __device__ __forceinline__ bool exists(int page) const { return (unsigned)page < (unsigned)pages; }
  __device__ __forceinline__ int slot(int tile) const { return (tile * 32) & ((1 << lp) - 1); }
  // operand f of the tile: k[f / KC][f % KC], then v[f - 2 KC]
  __device__ __forceinline__ const f16* frag(int f, int tile, int page) const {
    const int64_t pg = exists(page) ? page : 0;
    if (f < 2 * KC) return kbase + pg * kstride + slot(tile) * M + 4 * (f / KC) * M + 32 * (f % KC);
    return vbase + pg * vstride + slot(tile) * DV + 128 * (f - 2 * KC);
  }
  __device__ __forceinline__ void load(CacheTile<M, DV>& T, int tile, int page) const {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < KC; ++c) T.k[i][c] = *reinterpret_cast<const f16x8*>(frag(i * KC + c, tile, page));
#pragma unroll
    for (int c = 0; c < NT; ++c) T.v[c] = *reinterpret_cast<const f16x8*>(frag(2 * KC + c, tile, page));
  }
};

// split_exact of two weights, to places j and j + 1: three instructions (a
// conversion takes two numbers, and the remainder is a mixed multiply-add) where one
// after another they are eight. The remainders are exact, so the halves are the same.
__device__ __forceinline__ void split_two(float x, float y, int j, f16x8& hi, f16x8& lo) {
  asm("" : "+v"(x), "+v"(y));
  int both = __builtin_bit_cast(int, f16x2{(f16)x, (f16)y});
  asm("" : "+v"(both));  // or each is converted once more by itself
  const f16x2 h = __builtin_bit_cast(f16x2, both);
  float minus = -1.f;
  asm("" : "+s"(minus));  // or the multiply-add becomes a conversion and a difference
  hi[j] = h[0];
  hi[j + 1] = h[1];
  lo[j] = (f16)__builtin_fmaf((float)h[0], minus, x);
  lo[j + 1] = (f16)__builtin_fmaf((float)h[1], minus, y);
}

// 16 QT query rows of one (sequence, head) in a wave: the queries, and what
// they have summed. S^T = K u^T and O^T += V^T P^T on v_mfma_f32_16x16x32_f16:
// a lane holds 8 keys of the query lane % 16 in both products, so weights
// never leave their lane. u is an fp16 hi / lo pair, so scores are as exact as
// fp32 sums; their sum starts at `off`, minus the row's softmax reference, and
// comes out as the weight's exponent.
//
// The reference is a score seen before minus 12; it moves only when an exponent
// passes 15, so most tiles rescale nothing. Weights are at most 2^15: fp16
// keeps what is 2^-36 of the largest.
// LO: the weights enter the value product as hi / lo pairs, and the output is
// exact to fp32 rounding too (where reading the keys is the bound, the second
// product is free). Without, they are rounded to fp16 once: each moves its
// value's share by up to 2^-11, the divisor sums them unrounded. (Summing the
// rounded ones, by a product with ones, costs a seventh of the MFMAs; what it
// would take off, their mean error, is 2^-12 over the root of the keys.)
template <int M, int DV, int QT, bool LO>
struct CacheRows {
  static constexpr int KC = CacheTile<M, DV>::KC, NT = CacheTile<M, DV>::NT;
  static constexpr int NU = M == 16 ? 1 : 2 * KC;  // u operands: hi and lo of 32 codes each; at M = 16 one holds both
  f16x8 u[QT][NU];
  f32x4 off[QT];  // minus the reference, in every register
  float thr[QT];  // exponent from which the reference moves: 15, -inf before the first score
  float sum[QT];  // of this lane's weights
  f32x4 O[QT][NT];
  bool ready = false;  // every row has a reference

  // Rows first .. first + 16 QT - 1, those from n on repeating the last; rc: the rows' constants.
  __device__ __forceinline__ void start(const CacheAttnArgs& a, const f16* phi, const f16* gate_q, const f16* gate_k,
                                        int b, int h, int first, int lane, float (&rc)[QT]) {
    start_rows(a, gate_q, gate_k, h, lane, rc, [&](int t) {
      const int row = min(first + 16 * t + (lane & 15), a.n - 1);
      return phi + (((int64_t)b * a.n + row) * a.H + h) * M;
    });
  }
  // codes_of(t): the codes of this lane's row t.
  template <class Codes>
  __device__ __forceinline__ void start_rows(const CacheAttnArgs& a, const f16* gate_q, const f16* gate_k, int h,
                                             int lane, float (&rc)[QT], const Codes& codes_of) {
    const int g = lane >> 4;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float r = 0.f;
      const f16* pr = codes_of(t);
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const int c0 = M == 16 ? 8 * (g & 1) : 32 * c + 8 * g;
        const f16x8 p8 = *reinterpret_cast<const f16x8*>(pr + c0);
        const f16 *gq = gate_q + h * M + c0, *gk = gate_k + h * M + c0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float G = a.sl2e * ((float)gq[j] * (float)gk[j]);
          r += G * (float)p8[j];
          f16 hi, lo;
          split_exact(G * (2.f * (float)p8[j] - 1.f), hi, lo);
          if (M == 16) {
            u[t][0][j] = g < 2 ? hi : lo;
          } else {
            u[t][c][j] = hi;
            u[t][KC + c][j] = lo;
          }
        }
      }
      r += __shfl_xor(r, 16);
      if (M != 16) r += __shfl_xor(r, 32);  // at M = 16 lane groups 2 and 3 hold the codes of 0 and 1 again
      rc[t] = r;
      off[t] = f32x4{};
      thr[t] = kNegInf;
      sum[t] = 0.f;
#pragma unroll
      for (int c = 0; c < NT; ++c) O[t][c] = f32x4{};
    }
  }

  // Exponents of the weights: row t of this lane, its 4 keys of block i.
  __device__ __forceinline__ f32x4 score(const CacheTile<M, DV>& T, int t, int i) const {
    f32x4 s = mfma16x16(T.k[i][0], u[t][0], off[t]);
    if constexpr (M != 16) {
      s = mfma16x16(T.k[i][0], u[t][KC], s);
#pragma unroll
      for (int c = 1; c < KC; ++c) {
        s = mfma16x16(T.k[i][c], u[t][c], s);
        s = mfma16x16(T.k[i][c], u[t][KC + c], s);
      }
    }
    return s;
  }

  // Adds NK tiles. seen(t): bit j: row t of this lane sees key j of its 8; read
  // only if MASKED. again(t, p, seen): called with the weights if MASKED.
  template <bool MASKED, int NK, class Seen, class Again>
  __device__ __forceinline__ void add(const CacheTile<M, DV> (&T)[NK], const Seen& seen, const Again& again) {
    static_assert(!MASKED || NK == 1, "one masked tile at a time");
    f32x4 s[NK][QT][2];
    float top[QT];
    bool move = false;
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[n][t][i] = score(T[n], t, i);
        }
    unsigned vis[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      if constexpr (MASKED) {
        vis[t] = seen(t);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0][t][j >> 2][j & 3] = (vis[t] >> j) & 1 ? s[0][t][j >> 2][j & 3] : kNegInf;
      }
      top[t] = s[0][t][0][0];
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int j = 0; j < 8; ++j) top[t] = fmaxf(top[t], s[n][t][j >> 2][j & 3]);
      move |= top[t] > thr[t];
    }
    if (__any(move)) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        float m = fmaxf(top[t], __shfl_xor(top[t], 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        const bool first = thr[t] == kNegInf, any = m > kNegInf;
        const float up = first ? (any ? m - 12.f : 0.f) : fmaxf(m - 12.f, 0.f);
        const float f = first ? 1.f : fast_exp2(-up);  // before the first score there is nothing to scale
        off[t] -= up;
        thr[t] = first && !any ? kNegInf : 15.f;
#pragma unroll
        for (int n = 0; n < NK; ++n) {
          s[n][t][0] -= up;
          s[n][t][1] -= up;
        }
        sum[t] *= f;
#pragma unroll
        for (int c = 0; c < NT; ++c) O[t][c] *= f;
      }
    }
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        f16x8 hi, lo;
        float p[8];
        // the exponentials go before another wave's products (B4 n1000 over
        // 4096 keys 90.2 -> 87.9 us; the products first 89.2)
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = fast_exp2(s[n][t][j >> 2][j & 3]);
          if constexpr (LO) {
            sum[t] += p[j];  // one after another: few registers (few rows are bound by loads in flight)
            if (j & 1) split_two(p[j - 1], p[j], j - 1, hi, lo);
          } else {
            hi[j] = (f16)p[j];
          }
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (!LO) sum[t] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          O[t][c] = mfma16x16(T[n].v[c], hi, O[t][c]);
          if constexpr (LO) O[t][c] = mfma16x16(T[n].v[c], lo, O[t][c]);
        }
        if constexpr (MASKED) again(t, p, vis[t]);
      }
  }
  // Adds tiles that every row sees all of. Single weights tell by their sum
  // whether the reference has to move: while 8 sum to at most 65504, each is an
  // fp16 number. So no maximum is taken, and the exponentials need not wait for
  // one (B4 n4096 over none 147 -> 140 us, B4 n1000 dv128 82.7 -> 80.8, over
  // 4096 keys dv64 81.2 -> 80.4). Pairs are bound by other things.
  template <int NK>
  __device__ __forceinline__ void add_clear(const CacheTile<M, DV> (&T)[NK]) {
    if constexpr (LO) {
      add<false>(T, [](int) { return 0u; }, [](int, const float(&)[8], unsigned) {});
      return;
    }
    f32x4 s[NK][QT][2];
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) s[n][t][i] = score(T[n], t, i);
    // moves row t's reference by the scores from tile n on: to 10 below the
    // top, or 8 like it would already sum to half of what moves it again
    auto settle = [&](int n, int t) {
      float m = kNegInf;
#pragma unroll
      for (int k = 0; k < NK; ++k)
        if (k >= n)
#pragma unroll
          for (int j = 0; j < 8; ++j) m = fmaxf(m, s[k][t][j >> 2][j & 3]);
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      const bool first = thr[t] == kNegInf;
      const float up = first ? m - 10.f : fmaxf(m - 10.f, 0.f);
      const float f = first ? 1.f : fast_exp2(-up);
      off[t] -= up;
      thr[t] = 15.f;
#pragma unroll
      for (int k = 0; k < NK; ++k)
        if (k >= n) {
          s[k][t][0] -= up;
          s[k][t][1] -= up;
        }
      sum[t] *= f;
#pragma unroll
      for (int c = 0; c < NT; ++c) O[t][c] *= f;
    };
    if (!ready) {
#pragma unroll
      for (int t = 0; t < QT; ++t) settle(0, t);
      ready = true;
    }
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        f16x8 w;
        auto weigh = [&]() {
          float p[8];
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            p[j] = fast_exp2(s[n][t][j >> 2][j & 3]);
            w[j] = (f16)p[j];
          }
          __builtin_amdgcn_s_setprio(0);
          return ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        };
        float part = weigh();
        if (__any(part > 65504.f)) {
          settle(n, t);
          part = weigh();
        }
        sum[t] += part;
#pragma unroll
        for (int c = 0; c < NT; ++c) O[t][c] = mfma16x16(T[n].v[c], w, O[t][c]);
      }
  }

  // After the last tile: the reference and the sum of the weights.
  __device__ __forceinline__ void finish(int t, float& ref, float& l) const {
    ref = thr[t] > 0.f ? -off[t][0] : -1e30f;  // nothing seen: below every other
    l = sum[t] + __shfl_xor(sum[t], 16);       // the lane groups hold their own keys of the same 16 queries
    l += __shfl_xor(l, 32);
  }
};

// What a wave's rows see of a tile near or past the end of what all see. In
// integer arithmetic on 8 bits a lane: 8 compares would take 8 register pairs.
struct CacheMask {
  int ctx, nb, total, causal, mask_diag;
  bool tree;
  __device__ __forceinline__ static unsigned first(int count) { return (1u << min(max(count, 0), 8)) - 1; }
  // row i (of the new tokens; bits: its drafts), keys key0 .. key0 + 7
  __device__ __forceinline__ unsigned operator()(int i, uint64_t bits, int key0) const {
    const int d = key0 - ctx;  // which of the new tokens the first key is
    unsigned seen = first(i < nb ? total - key0 : 0);
    if (tree) {
      const unsigned drafts = d >= 0 ? (unsigned)(d < 64 ? bits >> d : 0)
                                     : (d > -8 ? (unsigned)(bits << -d) | first(-d) : 0xffu);
      return seen & drafts;
    }
    if (causal) seen &= first(i + 1 - d);
    if (mask_diag && (unsigned)(i - d) < 8u) seen &= ~(1u << (i - d));
    return seen;
  }
};

// A tile that some row does not see all of. A place behind the last key may
// hold anything, and 0 times an infinity or a NaN is NaN in every row of the
// value product: such values are taken out of it and added by themselves, to
// the rows that see their key.
template <int M, int DV, int QT, bool LO>
__device__ __forceinline__ void add_masked(CacheRows<M, DV, QT, LO>& R, CacheTile<M, DV> (&Ts)[1],
                                           const CacheSource<M, DV>& src, const CacheMask& mask, int first,
                                           const uint64_t (&bits)[QT], int tile, int page, int lane) {
  constexpr int NT = CacheTile<M, DV>::NT;
  const int c16 = lane & 15, g = lane >> 4, key0 = tile * 32 + 8 * g;
  CacheTile<M, DV>& T = Ts[0];
  unsigned there[4], strange = 0;  // halves of the keys that exist
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = mask.total - key0 - 2 * j;
    there[j] = n >= 2 ? ~0u : n == 1 ? 0xffffu : 0u;
  }
#pragma unroll
  for (int c = 0; c < NT; ++c) {
    i32x4 x = __builtin_bit_cast(i32x4, T.v[c]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // an exponent of all ones carries into bit 15 of its half
      const unsigned bad = ((((unsigned)x[j] & 0x7c007c00u) + 0x04000400u) >> 15 & 0x00010001u) * 0xffffu;
      strange |= bad & there[j];
      x[j] = (int)((unsigned)x[j] & ~bad & there[j]);
    }
    T.v[c] = __builtin_bit_cast(f16x8, x);
  }
  const bool any = __any(strange != 0);
  R.template add<true>(
      Ts, [&](int t) { return mask(first + 16 * t + c16, bits[t], key0); },
      [&](int t, const float(&p)[8], unsigned seen) {
        if (!any) return;
        // column 16 c + 4 g + r of key k
        const f16* v = src.vbase - (g * (DV * 8) + c16 * 8) + page * src.vstride + src.slot(tile) * DV + g * 32;
#pragma unroll 1
        for (int k = 0; k < 32; ++k) {
          const int from = 16 * (k >> 3) + c16;
          float pk = p[0];
#pragma unroll
          for (int j = 1; j < 8; ++j) pk = (k & 7) == j ? p[j] : pk;
          pk = __shfl(pk, from);
          const bool sees = (__shfl((int)seen, from) >> (k & 7)) & 1;
#pragma unroll
          for (int c = 0; c < NT; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const f16 x = v[(k >> 3) * DV * 8 + 128 * c + 8 * r + (k & 7)];
              R.O[t][c][r] += sees && not_finite(x) ? pk * (float)x : 0.f;
            }
        }
      });
}

// Writes 4 columns from c on of a row: the result, or one piece's part of it.
template <int DV>
struct CacheOut {
  f16* out;
  float* lse;
  float* part_o;
  float4* part_st;
  int n, H, b, h, nb, nsplit, sp;
  __device__ __forceinline__ f16* row(int i, int c) const { return out + (((int64_t)b * n + i) * H + h) * DV + c; }
  // m, l: reference and sum of the weights; r: the row constant. Not 0: the
  // result has columns that are not finite (settle_columns).
  __device__ __forceinline__ unsigned operator()(int i, int c, f32x4 o, float m, float l, float r) const {
    if (i >= n) return 0;
    const int64_t at = ((int64_t)b * H + h) * n + i;
    if (nsplit > 1) {
      if (i >= nb) return 0;  // the joining kernel writes padding rows
      *reinterpret_cast<f32x4*>(part_o + (at * nsplit + sp) * DV + c) = o;
      if (c == 0) part_st[at * nsplit + sp] = float4{m, l, r, 0.f};
      return 0;
    }
    const bool some = i < nb && l != 0.f;  // padding rows and rows that see nothing get 0
    const float inv = some ? 1.f / l : 0.f;
    f16x4 y;
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = some ? (f16)(o[k] * inv) : (f16)0.f;
    *reinterpret_cast<f16x4*>(row(i, c)) = y;
    if (c == 0) {
      // a difference of larger numbers: the logarithm of the mantissa alone, in
      // [-1, 0), is good to 2^-24, and the rest is added in 64 bits
      const double lg = (double)fast_log2(__builtin_amdgcn_frexp_mantf(l)) + (double)__builtin_amdgcn_frexp_expf(l);
      lse[at] = some ? (float)((double)m + lg - (double)r) : -kFltMax;
    }
    // an exponent of all ones carries into bit 15 of its half
    const uint64_t bits = __builtin_bit_cast(uint64_t, y);
    return ((((unsigned)bits & 0x7c007c00u) + 0x04000400u) | (((unsigned)(bits >> 32) & 0x7c007c00u) + 0x04000400u)) &
           0x80008000u;
  }
};

// Columns c .. c + 3 of a finished row, those of them that are not finite. The
// weight of every key that a row sees is positive, so a value that is not finite
// decides its column whatever the weight: infinite, or NaN where both infinities
// or a NaN are among them. The value product does not keep to that (0 times an
// infinity where a weight rounds to nothing, infinities of both signs where it is
// a pair of halves), so such a column becomes the sum of the values that are not
// finite. Where all are finite, single weights were rounded up and the largest
// value with them past the range. The keys are read once more, which nothing but
// such a row pays for (15 shapes with and without: -1.7 to 1.9 %, mean -0.1).
// v, stride: the head's values in page 0, and a page's; pages: the sequence's, of
// `count` in the pool; i: the row; bits: its drafts; l: the sum of its weights
// (scores that are not numbers leave nothing to settle); out: column c of it.
template <int DV>
__device__ __forceinline__ void settle_columns(const f16* v, int64_t stride, const int* pages, int count, int lp,
                                               const CacheMask& mask, int i, uint64_t bits, float l, f16* out,
                                               int c) {
  if (!__builtin_isfinite(l)) return;
  f16x4* at = reinterpret_cast<f16x4*>(out);
  f16x4 y = *at;
  if (!(not_finite(y[0]) || not_finite(y[1]) || not_finite(y[2]) || not_finite(y[3]))) return;
  f32x4 sum = {};
#pragma unroll 1
  for (int key = 0; key < mask.total; key += 8) {
    const int page = pages[key >> lp];
    const unsigned seen = mask(i, bits, key);
    if ((unsigned)page >= (unsigned)count || seen == 0) continue;
    const f16* from = v + page * stride + ((key & ((1 << lp) - 1)) * DV + 8 * c);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f16x8 x = *reinterpret_cast<const f16x8*>(from + 8 * k);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[k] += (seen >> j) & 1 && not_finite(x[j]) ? (float)x[j] : 0.f;
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (not_finite(y[k])) y[k] = sum[k] != 0.f ? (f16)sum[k] : (f16)__builtin_copysignf(65504.f, (float)y[k]);
  *at = y;
}

// What a workgroup works on: heads fastest (a page's heads are neighbours in
// memory, and with a multiple of 8 heads all row blocks of a head share an
// XCD's L2), then pieces, then row blocks, then sequences; under a causal
// mask, where the last row blocks are the longest, all sequences' last ones
// before the others (B4 n1000 over 4096 keys 101 -> 95 us, n4096 over none 180
// -> 164; without the mask the first order is 1 to 4 % faster), and every other
// round of 256 workgroups in reverse, 8 (one for each XCD) at a time: a CU that
// takes a long one first takes a short one next (88.6 -> 83.7 us, B8 n500 over
// 1000 to 3000 62.6 -> 57.6; with many rounds it does not matter).
struct CacheBlock {
  int b, h, sp, qb;
  // first: the launch's first workgroup of these
  __device__ __forceinline__ CacheBlock(const CacheAttnArgs& a, int first) {
    int id = blockIdx.x - first;
    if (a.causal && a.qblocks > 1 && (id & 256)) {
      const int round = id & ~255, whole = min(256, (int)gridDim.x - first - round) & ~7;
      if (id - round < whole) id = round + (whole - 8 - ((id - round) & ~7)) + (id & 7);
    }
    h = id % a.H;
    id /= a.H;
    sp = id % a.nsplit;
    id /= a.nsplit;
    if (a.causal) {
      b = id % a.B;
      qb = a.qblocks - 1 - id / a.B;
    } else {
      qb = id % a.qblocks;
      b = id / a.qblocks;
    }
  }
};

// Up to 16 rows: the four waves of a workgroup share them and take every
// fourth tile of the piece's keys, straight into registers, one tile ahead.
// Bound by reading the keys: B64 n1 H16 m16 dv64, 1 to 8191 tokens (158 MB) 34.9
// us, 4.5 TB/s; B1 n1 H16 m32 dv64, 131071 tokens (403 MB) 70 us, 5.7 TB/s. Short
// sequences by the chain lengths, page, key: B1 n1, 99 tokens 4.4 us, of which
// an empty launch is 2.5.
template <int M, int DV, class Shared>
__global__ __launch_bounds__(256) void cache_attn_few_kernel(
    CacheAttnArgs a, Shared shared, const f16* __restrict__ phi, const f16* __restrict__ gate_q, const f16* __restrict__ gate_k,
    const f16* __restrict__ codes, const f16* __restrict__ values, const int* __restrict__ table,
    const int* __restrict__ lens, const int* __restrict__ new_lens, const int64_t* __restrict__ tree,
    f16* __restrict__ out, float* __restrict__ lse, float* __restrict__ part_o, float4* __restrict__ part_st) {
  constexpr int NT = DV / 16;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  if constexpr (Shared::kJoint)
    if (shared.template prefix<M, DV>(a, phi, gate_q, gate_k, codes, values, table, lens, new_lens, part_o, part_st)) return;
  const CacheBlock blk(a, shared.first_block());
  const int b = blk.b, h = blk.h;
  const SeqLen sq = seq_len(lens, new_lens, b, a.n, a.W << a.lp);
  const int kb = shared.skip(b, sq.ctx, a.lp) + blk.sp * a.split_keys, parts = shared.pieces() + a.nsplit;
  if (blk.sp > 0 && kb >= sq.total) return;  // not one of this sequence's pieces
  if (sq.nb == 0 && parts > 1) return;       // padding: the joining kernel writes it

  // keys below `clear` are seen by every row, none from `end` on by any
  const int ke = blk.sp == a.nsplit - 1 ? sq.total : min(sq.total, kb + a.split_keys);
  const bool chunk = tree == nullptr;
  int clear = chunk ? (a.causal ? sq.ctx + (a.mask_diag ? 0 : 1) : a.mask_diag ? sq.ctx : sq.total) : sq.ctx;
  clear = min(clear, sq.total);
  const int end = sq.nb > 0 ? ke : 0;
  const CacheSource<M, DV> src(a, codes, values, table, b, h, lane);

  // the first tile is on its way while the queries are prepared
  CacheTile<M, DV> A[1], B[1];
  int tile = kb / 32 + w, pa = 0, pb = 0;
  auto within = [&](int t) { return t * 32 < end; };
  auto clean = [&](int t, int page) { return t * 32 + 32 <= min(clear, end) && src.exists(page); };
  if (within(tile)) {
    pa = src.page_of(tile);
    src.load(A[0], tile, pa);
  }
  if (within(tile + 4)) pb = src.page_of(tile + 4);

  CacheRows<M, DV, 1, true> R;
  __shared__ float sr[16];  // the row constants, which the main loop need not hold
  float rc[1];
  R.start(a, phi, gate_q, gate_k, b, h, 0, lane, rc);
  if (threadIdx.x < 16) sr[c16] = rc[0];
  const uint64_t bits[1] = {tree ? (uint64_t)tree[(int64_t)b * a.n + min(c16, a.n - 1)] : 0};

  // adds cur, with the next tile's loads in flight
  auto step = [&](CacheTile<M, DV>(&cur)[1], CacheTile<M, DV>(&nxt)[1], int& pc, int pn) {
    if (within(tile + 4)) src.load(nxt[0], tile + 4, pn);
    if (within(tile + 8)) pc = src.page_of(tile + 8);
    R.add_clear(cur);
    tile += 4;
  };
  while (clean(tile, pa)) {
    step(A, B, pa, pb);
    if (!clean(tile, pb)) {
      A[0] = B[0];
      const int p = pa;
      pa = pb;
      pb = p;
      break;
    }
    step(B, A, pb, pa);
  }
  const CacheMask mask{sq.ctx, sq.nb, sq.total, a.causal, a.mask_diag, !chunk};
  while (within(tile)) {
    if (within(tile + 4)) src.load(B[0], tile + 4, pb);
    if (src.exists(pa)) add_masked(R, A, src, mask, 0, bits, tile, pa, lane);
    A[0] = B[0];
    pa = pb;
    tile += 4;
    if (within(tile + 4)) pb = src.page_of(tile + 4);
  }

  __shared__ __align__(16) float so[4][16][DV + 4];
  __shared__ float sm[4][16], sl[4][16];
  float ref, l;
  R.finish(0, ref, l);
#pragma unroll
  for (int c = 0; c < NT; ++c) *reinterpret_cast<f32x4*>(&so[w][c16][16 * c + 4 * g]) = R.O[0][c];
  if (g == 0) {
    sm[w][c16] = ref;
    sl[w][c16] = l;
  }
  __syncthreads();
  const CacheOut<DV> put{out, lse, part_o, part_st, a.n, a.H, b, h, sq.nb, parts, shared.pieces() + blk.sp};
  for (int e = threadIdx.x; e < 4 * DV; e += 256) {
    const int q = e / (DV / 4), c = 4 * (e % (DV / 4));
    if (q >= a.n) break;
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
    if (put(q, c, o, m, l, sr[q]))
      settle_columns<DV>(values + (((int64_t)h * DV) << a.lp), ((int64_t)a.H * DV) << a.lp, table + (int64_t)b * a.W,
                         a.pages, a.lp, mask, q, tree ? (uint64_t)tree[(int64_t)b * a.n + q] : 0, l,
                         put.row(q, c), c);
  }
}

// More rows: each of the four waves of a workgroup has 16 QT of its own, and
// the keys pass through LDS, 64 a stage and three stages, filled by DMA in the
// order in which the lanes read them as operands (a wave fetches every fourth
// operand; 1 KiB each, conflict-free both ways).
// Drafts are bound by reading the keys (B16 n48 H32 m64 dv64, 300 to 4000
// tokens, 198 MB: 43 us, 4.6 TB/s); pieces of prompts by the exponentials,
// conversions and sums beside the matrix products of the few waves of a SIMD, and
// by workgroups of different lengths (B4 n1000 behind 3000 to 4096 tokens H16
// m16 dv64: 80 us, 0.5 PFLOP/s; at n4096 over none 140 us).
template <int M, int DV, int QT, bool LO, class Shared>
__global__ __launch_bounds__(256, M > 32 || DV > 64 ? 2 : LO || QT > 1 ? 3 : 4) void cache_attn_rows_kernel(
    CacheAttnArgs a, Shared shared, const f16* __restrict__ phi, const f16* __restrict__ gate_q, const f16* __restrict__ gate_k,
    const f16* __restrict__ codes, const f16* __restrict__ values, const int* __restrict__ table,
    const int* __restrict__ lens, const int* __restrict__ new_lens, const int64_t* __restrict__ tree,
    f16* __restrict__ out, float* __restrict__ lse, float* __restrict__ part_o, float4* __restrict__ part_st) {
  constexpr int NT = DV / 16, NF = CacheTile<M, DV>::kFrags, PER = NF / 2;  // DMA pieces of a wave and stage
  static_assert(NF % 2 == 0, "a stage's operands divide evenly among four waves");
  __shared__ __align__(1024) char lds[3][2 * NF * 1024];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  if constexpr (Shared::kJoint)
    if (shared.template prefix<M, DV>(a, phi, gate_q, gate_k, codes, values, table, lens, new_lens, part_o, part_st, lds))
      return;
  const CacheBlock blk(a, shared.first_block());
  const int b = blk.b, h = blk.h, q0 = blk.qb * 64 * QT, qw = q0 + 16 * QT * w;
  const SeqLen sq = seq_len(lens, new_lens, b, a.n, a.W << a.lp);
  const int kb = shared.skip(b, sq.ctx, a.lp) + blk.sp * a.split_keys, parts = shared.pieces() + a.nsplit;
  if (blk.sp > 0 && kb >= sq.total) return;
  if (q0 >= sq.nb && parts > 1) return;

  const int ke = blk.sp == a.nsplit - 1 ? sq.total : min(sq.total, kb + a.split_keys);
  // what the wave's rows see: all of them the keys below clear and, where only
  // their own keys are dropped, those from `beyond` on; none a key from end on
  const bool chunk = tree == nullptr;
  const int own = sq.ctx + qw;
  int clear = chunk ? (a.causal ? own + (a.mask_diag ? 0 : 1) : a.mask_diag ? own : sq.total) : sq.ctx;
  clear = min(clear, sq.total);
  const int beyond = chunk && !a.causal && a.mask_diag ? own + 16 * QT : sq.total;
  auto end_of = [&](int first, int count) {
    const int e = chunk && a.causal ? sq.ctx + min(first + count, sq.nb) : sq.total;
    return first < sq.nb ? min(e, ke) : 0;
  };
  const int end = end_of(qw, 16 * QT), endw = end_of(q0, 64 * QT);  // endw: of the workgroup
  const CacheMask mask{sq.ctx, sq.nb, sq.total, a.causal, a.mask_diag, !chunk};
  const CacheSource<M, DV> src(a, codes, values, table, b, h, lane);
  const unsigned base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

  const int tile0 = kb / 32, tiles = endw > kb ? (endw - kb + 31) / 32 : 0, stages = (tiles + 1) / 2;
  // A stage lies in one page, or in two of 32 tokens (then `two`, and the
  // second one of the last stage may not be in the table any more).
  const bool two = a.lp == 5;
  auto page = [&](int st, int i) {
    return src.row[two ? tile0 + min(2 * st + i, tiles - 1) : (32 * tile0 + 64 * st) >> a.lp];
  };
  // This wave's operands of a stage: KC of its 4 KC of codes, NT / 2 of its 2
  // NT of values, every fourth of each. Operand f of a kind with n a tile is
  // f % n of tile f / n. A lane's place in them in bytes from the stage's
  // first token (or its own page's, if there are two), and theirs in LDS.
  constexpr int KC = CacheTile<M, DV>::KC;
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
  unsigned fill = 0;  // where the next stage goes
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
  if (stages > 0) issue(pg[0]);
  if (stages > 1) issue(pg[1]);

  CacheRows<M, DV, QT, LO> R;
  __shared__ float sr[4][16 * QT];  // each wave's row constants
  float rc[QT];
  R.start(a, phi, gate_q, gate_k, b, h, qw, lane, rc);
#pragma unroll
  for (int t = 0; t < QT; ++t)
    if (g == 0) sr[w][16 * t + c16] = rc[t];
  uint64_t bits[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t)
    bits[t] = tree ? tree[(int64_t)b * a.n + min(qw + 16 * t + c16, a.n - 1)] : 0;

  int st = 0;
  // opens stage st: its keys are in LDS, those of stage st + 2 on their way
  auto open = [&]() {
    // this wave's part of the stage has landed (the next stage's may not have)
    if (st + 1 < stages)
      wait_vmcnt_lgkm0<PER>();
    else
      wait_vmcnt_lgkm0<0>();
    asm volatile("s_barrier" ::: "memory");  // ... and every wave's; the stage before is free
    if (st + 2 < stages) issue(pg[2]);
    if (st + 3 < stages) pages_of(st + 3, pg[3]);
  };
  unsigned read = 0;  // where the stage at hand is
  auto close = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      pg[0][i] = pg[1][i];
      pg[1][i] = pg[2][i];
      pg[2][i] = pg[3][i];
    }
    ++st;
    read = read == 2 * kStage ? 0 : read + kStage;
  };
  auto get = [&](CacheTile<M, DV>& T, int i) {
    const char* from = &lds[0][0] + read + 16 * lane + 1024 * NF * i;
#pragma unroll
    for (int f = 0; f < NF - NT; ++f) T.k[f / T.KC][f % T.KC] = *reinterpret_cast<const f16x8*>(from + 1024 * f);
#pragma unroll
    for (int c = 0; c < NT; ++c) T.v[c] = *reinterpret_cast<const f16x8*>(from + 1024 * (NF - NT + c));
  };
  // stages that all of the wave's rows see whole, and the others (every wave
  // opens every stage, so they meet at its barrier from either loop)
  auto clean = [&]() {
    const int from = kb + 64 * st, to = from + 64;
    return to <= end && (to <= clear || from >= beyond) && src.exists(pg[0][0]) && src.exists(pg[0][1]);
  };
  while (st < stages) {
    while (clean()) {
      open();
      CacheTile<M, DV> T[2];
      get(T[0], 0);
      get(T[1], 1);
      R.add_clear(T);
      close();
    }
    if (st == stages) break;
    open();
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      const int tile = tile0 + 2 * st + i, pc = i ? pg[0][1] : pg[0][0];
      if (tile * 32 >= end || !src.exists(pc)) continue;  // uniform in the wave
      CacheTile<M, DV> T[1];
      get(T[0], i);
      add_masked(R, T, src, mask, qw, bits, tile, pc, lane);
    }
    close();
  }
  const CacheOut<DV> put{out, lse, part_o, part_st, a.n, a.H, b, h, sq.nb, parts, shared.pieces() + blk.sp};
  unsigned odd[QT];
  float weights[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    float ref;
    R.finish(t, ref, weights[t]);
    const float r = sr[w][16 * t + c16];
    odd[t] = 0;
#pragma unroll
    for (int c = 0; c < NT; ++c) odd[t] |= put(qw + 16 * t + c16, 16 * c + 4 * g, R.O[t][c], ref, weights[t], r);
  }
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (!odd[t]) continue;
    const int i = qw + 16 * t + c16;
#pragma unroll 1
    for (int c = 4 * g; c < DV; c += 16)
      settle_columns<DV>(reinterpret_cast<const f16*>(vh), vpage / 2, src.row, src.pages, src.lp, mask, i, bits[t],
                         weights[t], put.row(i, c), c);
  }
}

// Joins the pieces of the rows: DV / 4 lanes hold a row's columns, NG such
// groups take its pieces in turn, and the groups are added in order. Bound by
// its launch: B64 n1 H16 of up to 9 pieces 4.4 us where an empty one takes 4.0.
template <int DV, int NG, class Shared>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttnArgs a, Shared shared, int64_t rows, const f16* __restrict__ values,
                                                        const int* __restrict__ table, const int* __restrict__ lens,
                                                        const int* __restrict__ new_lens,
                                                        const int64_t* __restrict__ tree,
                                                        const float* __restrict__ part_o,
                                                        const float4* __restrict__ part_st, f16* __restrict__ out,
                                                        float* __restrict__ lse) {
  constexpr int TC = DV / 4, ROWS = 256 / (TC * NG);
  const int k = threadIdx.x / TC % NG, c = 4 * (threadIdx.x % TC), rl = threadIdx.x / (TC * NG);
  const int64_t at = (int64_t)blockIdx.x * ROWS + rl;  // (b H + h) n + i
  const int i = (int)(at % a.n);
  const int64_t bh = at / a.n;
  const int h = (int)(bh % a.H), b = (int)min(bh / a.H, rows / ((int64_t)a.n * a.H) - 1);
  const SeqLen sq = seq_len(lens, new_lens, b, a.n, a.W << a.lp);
  const bool real = at < rows && i < sq.nb;
  const int skip = real ? shared.skip(b, sq.ctx, a.lp) : 0, before = shared.pieces_of(skip);
  const int pieces = real ? before + min(a.nsplit, (sq.total - skip + a.split_keys - 1) / a.split_keys) : 0;
  const int parts = shared.pieces() + a.nsplit;
  float m = -1e30f, l = 0.f;
  float r = 0.f;
  f32x4 o = {};
  for (int k1 = k; k1 < pieces; k1 += NG) {
    const int64_t s = at * parts + (k1 < before ? k1 : shared.pieces() + k1 - before);
    const float4 st = part_st[s];
    r = st.z;  // the same in every piece
    const f32x4 x = *reinterpret_cast<const f32x4*>(part_o + s * DV + c);
    const float nm = fmaxf(m, st.x), f = fast_exp2(m - nm), fs = fast_exp2(st.x - nm);
    l = l * f + st.y * fs;
    o = o * f + x * fs;
    m = nm;
  }
  if constexpr (NG > 1) {
    __shared__ __align__(16) float so[ROWS][NG][DV];
    __shared__ float2 ss[ROWS][NG];
    *reinterpret_cast<f32x4*>(&so[rl][k][c]) = o;
    if (c == 0) ss[rl][k] = float2{m, l};
    __syncthreads();
    if (k != 0) return;
#pragma unroll
    for (int e = 1; e < NG; ++e) m = fmaxf(m, ss[rl][e].x);
    l = 0.f;
    o = f32x4{};
#pragma unroll
    for (int e = 0; e < NG; ++e) {
      const float2 st = ss[rl][e];
      const float f = fast_exp2(st.x - m);
      l += f * st.y;
      o += f * *reinterpret_cast<const f32x4*>(&so[rl][e][c]);
    }
  }
  if (at >= rows) return;
  const CacheOut<DV> put{out, lse, nullptr, nullptr, a.n, a.H, b, h, sq.nb, 1, 0};
  const CacheMask mask{sq.ctx, sq.nb, sq.total, a.causal, a.mask_diag, tree != nullptr};
  if (put(i, c, o, m, l, r))
    settle_columns<DV>(values + (((int64_t)h * DV) << a.lp), ((int64_t)a.H * DV) << a.lp, table + (int64_t)b * a.W,
                       a.pages, a.lp, mask, i, tree ? (uint64_t)tree[(int64_t)b * a.n + i] : 0, l, put.row(i, c), c);
}

inline int log2_of(int p) { return __builtin_ctz((unsigned)p); }
inline CacheAttnArgs attn_args(const CacheDims& d, const CacheAttnPlan& p, int causal, int mask_diag) {
  CacheAttnArgs a{};
  a.B = d.B;
  a.n = d.n;
  a.H = d.H;
  a.W = d.W;
  a.pages = d.pages;
  a.lp = log2_of(d.P);
  a.qblocks = p.qblocks;
  a.nsplit = p.nsplit;
  a.split_keys = p.split_keys;
  a.causal = causal;
  a.mask_diag = mask_diag;
  return a;
}

}  // namespace morpho
