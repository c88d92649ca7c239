// Verification of drafted tokens: which of them the target keeps, and the next
// token, from given random numbers.
//
// With p the target's distribution behind a token and q the one that its drafts
// were drawn from (or all on the draft, where drafts were not drawn), a draft t
// is kept with probability min(1, r(t) / (q(t) Z)), r = p and Z = 1 at first; one
// that is not leaves r = max(r / Z - q, 0) and Z = sum r to the next draft of the
// same token and, when there is none, to the draw of the next token: what comes
// out then has the target's distribution, whatever q is. Two numbers hold r:
//   r = max(a p - c q, 0), and a rejection makes of them a / Z and c / Z + 1.
// (Where q is all on t, it only takes t out of p.)
//
// The results are whole numbers that depend on which side of a border a sum of
// up to millions of terms falls, so weights and sums are in 64 bits: the order of
// the terms then moves a border by 2^-50 or so, and the same inputs give the same
// tokens as any other 64-bit evaluation. (In 32 bits one of a thousand sampled
// tokens is another one.)
//
// 1. verify_stats_kernel: of every row's chunks the largest logit and the sum of
//    the weights below it (the only pass over all rows; bound by reading them).
// 2. verify_mass_kernel: the decisions up to the first rejection or the end, then
//    what r has in each chunk of that one row.
// 3. verify_kernel: the decisions to the end, and the next token, one workgroup a
//    sequence; a remainder that step 2 did not come to is summed here.
#include <limits.h>

#include "common.h"
#include "internal.h"

namespace morpho {

namespace {

// 2^(i / 32)
__constant__ double kExp2Table[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0, 0x1.172b83c7d517bp+0,
    0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0, 0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0,
    0x1.3dea64c123422p+0, 0x1.44e086061892dp+0, 0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0,
    0x1.6247eb03a5585p+0, 0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0, 0x1.ae89f995ad3adp+0,
    0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0, 0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0,
    0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};

// The weight exp((x - top) / temperature) of a logit, as 2^(v / 32) with v = (x -
// top) c <= 0, c = 32 log2(e) / temperature (the difference first: logits may be as
// large as their type allows): v = 32 e + i + r, |r| <= 1/2, and 2^(r / 32) is a polynomial of degree 5 through its Chebyshev nodes (2^-52.6 off at
// most). The table's 32 numbers are one in each pair of LDS banks, so lanes that
// read any of them never wait for each other. NaN and -inf weigh nothing.
struct Weigh {
  const double* table;  // LDS
  double c, top;        // a finite top
  __device__ __forceinline__ double operator()(float x) const {
    const double v = fmax(((double)x - top) * c, -40000.0);
    const double t = v + 0x1.8p52;
    const int n = (int)__builtin_bit_cast(int64_t, t);
    const double r = v - (t - 0x1.8p52);
    double y = 0x1.5d885e6ef14a6p-35;
    y = fma(y, r, 0x1.3b2b301f1eb9cp-27);
    y = fma(y, r, 0x1.c6b08d70380ddp-20);
    y = fma(y, r, 0x1.ebfbdff7feebap-13);
    y = fma(y, r, 0x1.62e42fefa39efp-6);
    y = fma(y, r, 1.0);
    return __builtin_amdgcn_ldexp(y * table[n & 31], n >> 5);
  }
};
// Any top: of an infinite one its own kind weigh 1, and nothing where all are -inf.
__device__ __forceinline__ double weight_below(const double* table, double c, float x, float top) {
  if (top == __builtin_inff()) return x == top ? 1.0 : 0.0;
  if (top == kNegInf) return 0.0;
  return Weigh{table, c, (double)top}(x);
}

struct Bf16 {
  uint16_t bits;
};
__device__ __forceinline__ float value_of(f16 x) { return (float)x; }
__device__ __forceinline__ float value_of(Bf16 x) { return __builtin_bit_cast(float, (unsigned)x.bits << 16); }
__device__ __forceinline__ float value_of(float x) { return x; }

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
  return x;
}

// The token that token i was drafted behind: the highest bit below its own, or
// (no tree) the one before; -1: none.
__device__ __forceinline__ int parent_of(const VerifyArgs& a, int b, int i) {
  if (!a.tree) return i - 1;
  const uint64_t below = (uint64_t)a.tree[(int64_t)b * a.n + i] & (((uint64_t)1 << i) - 1);
  return below ? 63 - __builtin_clzll(below) : -1;
}
__device__ __forceinline__ int tokens_of(const VerifyArgs& a, int b) {
  return a.new_lens ? min(max(a.new_lens[b], 0), a.n) : a.n;
}
template <class T>
__device__ __forceinline__ const T* row_of(const VerifyRows& r, int b, int i) {
  return static_cast<const T*>(r.data) + b * r.batch_stride + i * r.row_stride;
}

}  // namespace

// One chunk of a row: 256 U pieces of 16 bytes. Rows start anywhere, so the
// pieces are counted from the row's start rounded down to 16 bytes, and the first
// and the last are read by elements.
template <class T, int U, bool BEST>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  constexpr int E = 16 / sizeof(T);
  __shared__ double table[32], sums[4];
  __shared__ float tops[4];
  __shared__ int places[4];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const bool draft = row >= a.B * a.n;
  const int k = draft ? row - a.B * a.n : row, per = draft ? a.n - 1 : a.n, b = k / per, i = k % per;
  const int nb = tokens_of(a, b);
  if (i >= nb) return;
  // what a token without drafts of its own would have drawn from is not asked for
  if (draft && !__any(lane > i && lane < nb && parent_of(a, b, lane) == i)) return;
  if (threadIdx.x < 32) table[threadIdx.x] = kExp2Table[threadIdx.x];
  const T* p = row_of<T>(draft ? a.q : a.p, b, i);
  const int shift = (int)(((uintptr_t)p & 15) / sizeof(T));
  float x[U][E];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int first = ((chunk * U + u) * 256 + (int)threadIdx.x) * E - shift;
    if (first >= 0 && first + E <= a.V) {
      alignas(16) T v[E];
      *reinterpret_cast<i32x4*>(v) = *reinterpret_cast<const i32x4*>(p + first);
#pragma unroll
      for (int e = 0; e < E; ++e) x[u][e] = value_of(v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        x[u][e] = first + e >= 0 && first + e < a.V ? value_of(p[first + e]) : kNegInf;
    }
  }
  float top = kNegInf;
  int place = INT_MAX;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (BEST) {
        if (x[u][e] > top) {  // in ascending order: the lowest of equal ones
          top = x[u][e];
          place = ((chunk * U + u) * 256 + (int)threadIdx.x) * E - shift + e;
        }
      } else {
        top = fmaxf(top, x[u][e]);
      }
    }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float other = __shfl_xor(top, o);
    if constexpr (BEST) {
      const int at = __shfl_xor(place, o);
      if (other > top || (other == top && at < place)) {
        top = other;
        place = at;
      }
    } else {
      top = fmaxf(top, other);
    }
  }
  if (lane == 0) {
    tops[w] = top;
    places[w] = place;
  }
  __syncthreads();
  top = tops[0];
  place = places[0];
#pragma unroll
  for (int e = 1; e < 4; ++e)
    if (tops[e] > top || (BEST && tops[e] == top && places[e] < place)) {
      top = tops[e];
      place = places[e];
    }
  VerifyStat& out = a.stats[(int64_t)row * a.chunks + chunk];
  if constexpr (BEST) {
    if (threadIdx.x == 0) out = VerifyStat{0.0, top, top > kNegInf ? place : -1};
    return;
  }
  double sum = 0.0;
  if (top == __builtin_inff()) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) sum += x[u][e] == top ? 1.0 : 0.0;
  } else if (top > kNegInf) {
    const Weigh weigh{table, a.c, (double)top};
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) sum += weigh(x[u][e]);
  }
  sum = wave_sum(sum);
  if (lane == 0) sums[w] = sum;
  __syncthreads();
  if (threadIdx.x == 0) out = VerifyStat{(sums[0] + sums[1]) + (sums[2] + sums[3]), top, -1};
}

namespace {

// What the decisions of one sequence need; shared by a workgroup of 256.
struct WalkShared {
  double table[32];
  float top[2][64];   // of the target's rows, the drafter's
  double sum[2][64];  // of their weights
  int best[64];       // BEST: the target's best tokens
  int64_t rejected[64];
  double part[4];
};

// The decisions. Lane i of every wave holds draft i; all waves take the same
// steps, so nothing is exchanged between them.
template <class T, bool BEST, bool DRAFT>
struct Walk {
  const VerifyArgs& a;
  WalkShared& s;
  int b, nb, lane;
  int parent = -1;
  int64_t token = -1;
  double p = 0.0, q = 0.0, u = 0.0;  // of the draft: its probabilities, its random number
  // the token at hand, its drafts that are still to be asked, those that were turned down (where q is none)
  int node = 0;
  uint64_t open = 0, gone = 0, taken = 1;
  double pa = 1.0, qc = 0.0, Z = 1.0;  // r = max(pa p - qc q, 0), and its sum
  bool fresh = false;                  // the masses at hand are those of r
  bool none = false;                   // nothing to draw from

  __device__ __forceinline__ Walk(const VerifyArgs& a, WalkShared& s, int b) : a(a), s(s), b(b) {
    lane = threadIdx.x & 63;
    nb = tokens_of(a, b);
    if (lane > 0 && lane < nb) {
      parent = parent_of(a, b, lane);
      token = a.tokens[(int64_t)b * a.n + lane];
      if constexpr (!BEST) u = (double)a.uniform[(int64_t)b * a.n + lane];
    }
    if (threadIdx.x < 32) s.table[threadIdx.x] = kExp2Table[threadIdx.x];
    __syncthreads();
    row_totals();
    __syncthreads();
    if constexpr (!BEST) {
      if (parent >= 0 && token >= 0 && token < a.V) {
        p = chance(0, a.p, parent, token);
        if constexpr (DRAFT) q = chance(1, a.q, parent, token);
      }
    }
    open = __ballot(parent == 0);
  }

  __device__ __forceinline__ double chance(int kind, const VerifyRows& rows, int i, int64_t x) const {
    const double sum = s.sum[kind][i];
    return sum > 0.0 ? weight_below(s.table, a.c, value_of(row_of<T>(rows, b, i)[x]), s.top[kind][i]) / sum : 0.0;
  }

  // Joins the chunks of the rows: 2^k lanes a row, as many rows at a time as the workgroup has.
  __device__ __forceinline__ void row_totals() {
    int per = 1;
    while (per < a.chunks && per < 64) per *= 2;
    const int sub = threadIdx.x & (per - 1);
    uint64_t inner = 0;  // tokens with drafts
    if constexpr (DRAFT)
      for (int i = 0; i < nb; ++i)
        if (__any(parent == i)) inner |= (uint64_t)1 << i;
    for (int r0 = 0; r0 < (DRAFT ? 2 * nb : nb); r0 += 256 / per) {
      const int r = r0 + threadIdx.x / per, kind = r >= nb, i = r - kind * nb;
      const bool real = r < (DRAFT ? 2 * nb : nb) && (!kind || (inner >> i & 1));
      const VerifyStat* st =
          a.stats + (kind ? (int64_t)a.B * a.n + (int64_t)b * (a.n - 1) + i : (int64_t)b * a.n + i) * a.chunks;
      float top = kNegInf;
      int best = INT_MAX;
      for (int c = sub; real && c < a.chunks; c += per) {
        if (BEST) {
          if (st[c].top > top) {
            top = st[c].top;
            best = st[c].best;
          }
        } else {
          top = fmaxf(top, st[c].top);
        }
      }
      for (int o = 1; o < per; o <<= 1) {
        const float x = __shfl_xor(top, o);
        if (BEST) {
          const int at = __shfl_xor(best, o);
          if (x > top || (x == top && at < best)) best = at;
        }
        top = fmaxf(top, x);
      }
      double sum = 0.0;
      if constexpr (!BEST) {
        for (int c = sub; real && c < a.chunks; c += per)
          sum += st[c].sum > 0.0 ? st[c].sum * weight_below(s.table, a.c, st[c].top, top) : 0.0;
        for (int o = 1; o < per; o <<= 1) sum += __shfl_xor(sum, o);
      }
      if (real && sub == 0) {
        if (BEST) s.best[i] = top > kNegInf ? best : -1;
        s.top[kind][i] = top;
        s.sum[kind][i] = sum;
      }
    }
  }

  __device__ __forceinline__ void go_to(int i) {
    node = i;
    taken |= (uint64_t)1 << i;
    pa = Z = 1.0;
    qc = 0.0;
    gone = 0;
    fresh = false;
    open = __ballot(parent == i);
  }

  // On until the end (false), or until the masses of r are asked for (true).
  __device__ __forceinline__ bool asks() {
    while (open) {
      const int i = __builtin_ctzll(open);
      open &= open - 1;
      if constexpr (BEST) {
        if (s.best[node] >= 0 && __shfl(token, i) == (int64_t)s.best[node]) go_to(i);
        continue;
      }
      const double ui = __shfl(u, i), pi = __shfl(p, i);
      if constexpr (DRAFT) {
        const double qi = __shfl(q, i);
        if (ui * qi * Z < pa * pi - qc * qi) {
          go_to(i);
        } else {
          pa /= Z;
          qc = qc / Z + 1.0;
          fresh = false;
          return true;
        }
      } else {
        const bool again = (gone & __ballot(token == __shfl(token, i))) != 0;  // turned down before
        if (ui * Z < (again ? 0.0 : pi)) {
          go_to(i);
        } else {
          gone |= (uint64_t)1 << i;
          if (!again) Z = fmax(Z - pi, 0.0);
          fresh = false;
        }
      }
    }
    return !BEST && !fresh && !none;
  }
  // The sum of the masses that were asked for. Where nothing is left, the row's
  // own distribution takes its place.
  __device__ __forceinline__ void answer(double sum) {
    fresh = true;
    if (sum > 0.0) {
      Z = sum;
    } else {
      none = pa == 1.0 && qc == 0.0 && gone == 0;
      pa = Z = 1.0;
      qc = 0.0;
      gone = 0;
      fresh = false;
    }
  }

  // r over a part of the vocabulary.
  struct Rest {
    const T *p, *q;
    Weigh wp, wq;
    float ptop, qtop;
    double ap, aq;  // 0: not asked for
    const int64_t* rejected;
    int count;
    __device__ __forceinline__ double operator()(int x) const {
      double r = 0.0;
      if (ap > 0.0) {
        const float l = value_of(p[x]);
        r = ap * (ptop < __builtin_inff() ? wp(l) : l == ptop ? 1.0 : 0.0);
      }
      if constexpr (DRAFT) {
        if (aq > 0.0) {
          const float l = value_of(q[x]);
          r -= aq * (qtop < __builtin_inff() ? wq(l) : l == qtop ? 1.0 : 0.0);
        }
      } else {
        for (int k = 0; k < count; ++k)
          if (rejected[k] == x) r = 0.0;
      }
      return fmax(r, 0.0);
    }
  };
  // All of the workgroup calls it; it has barriers.
  __device__ __forceinline__ Rest rest() {
    Rest r;
    r.p = row_of<T>(a.p, b, node);
    r.ptop = s.top[0][node];
    r.wp = Weigh{s.table, a.c, (double)r.ptop};
    r.ap = s.sum[0][node] > 0.0 ? pa / s.sum[0][node] : 0.0;
    r.q = nullptr;
    r.aq = 0.0;
    r.count = 0;
    r.rejected = s.rejected;
    if constexpr (DRAFT) {
      if (qc > 0.0) {
        r.q = row_of<T>(a.q, b, node);
        r.qtop = s.top[1][node];
        r.wq = Weigh{s.table, a.c, (double)r.qtop};
        r.aq = s.sum[1][node] > 0.0 ? qc / s.sum[1][node] : 0.0;
      }
    } else {
      __syncthreads();
      if (threadIdx.x < 64 && (gone >> lane & 1)) s.rejected[__builtin_popcountll(gone & (((uint64_t)1 << lane) - 1))] = token;
      __syncthreads();
      r.count = __builtin_popcountll(gone);
    }
    return r;
  }
  // The mass of a chunk, in every lane.
  __device__ __forceinline__ double mass(const Rest& r, int chunk) {
    double sum = 0.0;
    const int end = min((chunk + 1) * a.chunk, a.V);
    for (int x = chunk * a.chunk + threadIdx.x; x < end; x += 256) sum += r(x);
    sum = wave_sum(sum);
    __syncthreads();
    if (lane == 0) s.part[threadIdx.x >> 6] = sum;
    __syncthreads();
    return (s.part[0] + s.part[1]) + (s.part[2] + s.part[3]);
  }
  // The sum of a row's masses, the same in every wave and kernel.
  __device__ __forceinline__ double total(const double* masses) const {
    double sum = 0.0;
    for (int c = lane; c < a.chunks; c += 64) sum += masses[c];
    return wave_sum(sum);
  }
  __device__ __forceinline__ const double* masses(int round) const {
    return a.masses + ((int64_t)round * a.B + b) * a.chunks;
  }
};

}  // namespace

// Round k: the masses that are asked for after the answers of the rounds before.
template <class T, bool DRAFT>
__global__ __launch_bounds__(256) void verify_mass_kernel(VerifyArgs a, int round) {
  __shared__ WalkShared s;
  const int b = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  if (tokens_of(a, b) == 0) return;
  Walk<T, false, DRAFT> walk(a, s, b);
  for (int k = 0; k < round; ++k) {
    if (!walk.asks()) return;
    walk.answer(walk.total(walk.masses(k)));
  }
  if (!walk.asks()) return;
  const double m = walk.mass(walk.rest(), chunk);
  if (threadIdx.x == 0) a.masses[((int64_t)round * a.B + b) * a.chunks + chunk] = m;
}

template <class T, bool BEST, bool DRAFT>
__global__ __launch_bounds__(256) void verify_kernel(VerifyArgs a) {
  __shared__ WalkShared s;
  __shared__ double mine[kVerifyMaxChunks], scan[4];
  __shared__ int found, last[4];
  const int b = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nb = tokens_of(a, b);
  if (nb == 0) {
    if (threadIdx.x < a.n) a.keep[(int64_t)b * a.n + threadIdx.x] = -1;
    if (threadIdx.x == 0) {
      a.keep_lens[b] = 0;
      a.token[b] = -1;
    }
    return;
  }
  Walk<T, BEST, DRAFT> walk(a, s, b);
  for (int k = 0; walk.asks(); ++k) {
    __syncthreads();  // the masses of the round before are read
    if (k < a.rounds) {
      for (int c = threadIdx.x; c < a.chunks; c += 256) mine[c] = walk.masses(k)[c];
    } else {
      const auto rest = walk.rest();
      for (int c = 0; c < a.chunks; ++c) {
        const double m = walk.mass(rest, c);
        if (threadIdx.x == 0) mine[c] = m;
      }
    }
    __syncthreads();
    walk.answer(walk.total(mine));
  }
  if (w == 0) {
    const int count = __builtin_popcountll(walk.taken), at = __builtin_popcountll(walk.taken & (((uint64_t)1 << lane) - 1));
    int32_t* keep = a.keep + (int64_t)b * a.n;
    if (walk.taken >> lane & 1) keep[at] = lane;
    if (lane >= count && lane < a.n) keep[lane] = -1;
    if (lane == 0) a.keep_lens[b] = count;
  }
  if constexpr (BEST) {
    if (threadIdx.x == 0) a.token[b] = s.best[walk.node];
    return;
  }
  if (walk.none) {
    if (threadIdx.x == 0) a.token[b] = -1;
    return;
  }
  // The first token whose running sum passes u Z: its chunk, then within it. Where
  // rounding leaves none behind a border, the last one that has a mass.
  const double want = (double)a.uniform[(int64_t)b * a.n] * walk.Z;
  auto first_past = [&](double sum, double before, bool some, int index, double& base) {
    // sums of 256 lanes in order; the first lane whose own end passes `want`, or
    // the last with a mass; base: the sum before it
    double upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double x = __shfl_up(upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();
    if (lane == 63) scan[w] = upto;
    if (threadIdx.x == 0) found = INT_MAX;
    __syncthreads();
    for (int k = 0; k < w; ++k) before += scan[k];
    base = before + upto - sum;
    const uint64_t past = __ballot(some && before + upto > want), have = __ballot(some);
    if (lane == 0) {
      last[w] = have ? 64 * w + 63 - __builtin_clzll(have) : -1;
      if (past) atomicMin(&found, 64 * w + __builtin_ctzll(past));
    }
    __syncthreads();
    int at = found;
    if (at == INT_MAX) at = max(max(last[0], last[1]), max(last[2], last[3]));
    return at == index;
  };
  // chunks: a run of them a lane
  const int run = (a.chunks + 255) / 256;
  double sum = 0.0, base;
  for (int c = threadIdx.x * run; c < min((int)(threadIdx.x + 1) * run, a.chunks); ++c) sum += mine[c];
  __shared__ int chunk;
  __shared__ double before_chunk;
  if (first_past(sum, 0.0, sum > 0.0, threadIdx.x, base)) {
    int pick = -1;
    double at = base, pick_at = base;
    for (int c = threadIdx.x * run; c < min((int)(threadIdx.x + 1) * run, a.chunks); ++c) {
      if (mine[c] > 0.0) {
        pick = c;
        pick_at = at;
        if (at + mine[c] > want) break;
      }
      at += mine[c];
    }
    chunk = pick;
    before_chunk = pick_at;
  }
  const auto rest = walk.rest();
  __syncthreads();
  // tokens: a run of them a lane
  const int per = a.chunk / 256, x0 = chunk * a.chunk + threadIdx.x * per, x1 = min(x0 + per, a.V);
  sum = 0.0;
  for (int x = x0; x < x1; ++x) sum += rest(x);
  if (first_past(sum, before_chunk, sum > 0.0, threadIdx.x, base)) {
    int pick = -1;
    for (int x = x0; x < x1; ++x) {
      const double r = rest(x);
      if (r > 0.0) {
        pick = x;
        if (base + r > want) break;
      }
      base += r;
    }
    a.token[b] = pick;
  }
}

namespace {
template <class T>
hipError_t launch_verify_t(const VerifyArgs& a, const VerifyPlan& p, hipStream_t s) {
  const bool draft = a.q.data != nullptr;
  const dim3 block(256), rows((unsigned)((int64_t)a.B * (draft ? 2 * a.n - 1 : a.n) * p.chunks));
#define MORPHO_VERIFY_STATS(U, BEST) MORPHO_KLAUNCH((verify_stats_kernel<T, U, BEST>), rows, block, 0, s, a)
  if (a.best && p.pieces == 1)
    MORPHO_VERIFY_STATS(1, true);
  else if (a.best)
    MORPHO_VERIFY_STATS(4, true);
  else if (p.pieces == 1)
    MORPHO_VERIFY_STATS(1, false);
  else
    MORPHO_VERIFY_STATS(4, false);
#undef MORPHO_VERIFY_STATS
  hipError_t e = hipGetLastError();
  for (int k = 0; k < p.rounds && e == hipSuccess; ++k) {
    const dim3 grid((unsigned)((int64_t)a.B * p.chunks));
    if (draft)
      MORPHO_KLAUNCH((verify_mass_kernel<T, true>), grid, block, 0, s, a, k);
    else
      MORPHO_KLAUNCH((verify_mass_kernel<T, false>), grid, block, 0, s, a, k);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)a.B);
  if (a.best)
    MORPHO_KLAUNCH((verify_kernel<T, true, false>), grid, block, 0, s, a);
  else if (draft)
    MORPHO_KLAUNCH((verify_kernel<T, false, true>), grid, block, 0, s, a);
  else
    MORPHO_KLAUNCH((verify_kernel<T, false, false>), grid, block, 0, s, a);
  return hipGetLastError();
}
}  // namespace

hipError_t launch_verify(const VerifyArgs& a, const VerifyPlan& p, int type, hipStream_t s) {
  if (type == 0) return launch_verify_t<f16>(a, p, s);
  if (type == 1) return launch_verify_t<Bf16>(a, p, s);
  return launch_verify_t<float>(a, p, s);
}

}  // namespace morpho
