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
//    the weights below it (the only pass over all rows).
// 2. verify_mass_kernel, where drafts were drawn: what r has in each chunk after
//    the first, second, ... rejection behind a token, by the whole chip.
// 3. verify_kernel: the decisions and the next token, one workgroup a sequence; a
//    remainder that step 2 did not come to is summed here.
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
// large as their type allows): v = 32 e + i + r, |r| <= 1/2, and 2^(r / 32) is a polynomial
// of degree 5 through its Chebyshev nodes (2^-52.6 off at most). The table's 32
// numbers are one in each pair of LDS banks, so lanes that read any of them never
// wait for each other. NaN and -inf weigh nothing.
__device__ __forceinline__ double exp2_rest(double r) {
  double y = 0x1.5d885e6ef14a6p-35;
  y = fma(y, r, 0x1.3b2b301f1eb9cp-27);
  y = fma(y, r, 0x1.c6b08d70380ddp-20);
  y = fma(y, r, 0x1.ebfbdff7feebap-13);
  y = fma(y, r, 0x1.62e42fefa39efp-6);
  return fma(y, r, 1.0);
}
struct Weigh {
  const double* table;  // LDS
  double c, top;        // a finite top
  __device__ __forceinline__ double operator()(float x) const {
    const double v = fmax(((double)x - top) * c, -40000.0);
    const double t = v + 0x1.8p52;
    const int n = (int)__builtin_bit_cast(int64_t, t);
    return __builtin_amdgcn_ldexp(exp2_rest(v - (t - 0x1.8p52)) * table[n & 31], n >> 5);
  }
};
// For sums: fewer instructions. The product comes before the difference, which
// costs every weight the same factor, 1 + 2^-53 top c / 46: for |top c| below 2^16 or
// so. What weighs less than 2^-1000, NaN and -inf too, weighs that.
struct WeighFast {
  const double* table;
  double c, topc;
  __device__ __forceinline__ double operator()(float x) const {
    const double v = fmax(fma((double)x, c, -topc), -32000.0);
    const double t = v + 0x1.8p52;
    const int n = (int)__builtin_bit_cast(int64_t, t);
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    i32x2 y = __builtin_bit_cast(i32x2, table[n & 31]);
    y[1] += (n & ~31) << 15;
    return exp2_rest(v - (t - 0x1.8p52)) * __builtin_bit_cast(double, y);
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
// Rows start anywhere. A row's chunks are counted from its start rounded down to
// 16 bytes: chunk k begins with element k a.chunk - shift.
template <class T>
__device__ __forceinline__ int shift_of(const T* row) {
  return (int)(((uintptr_t)row & 15) / sizeof(T));
}
// 16 bytes of logits as they are in memory.
template <class T>
struct Piece {
  static constexpr int E = 16 / sizeof(T);
  i32x4 raw;
  __device__ __forceinline__ float operator[](int e) const {
    const unsigned v = (unsigned)raw[e * (int)sizeof(T) / 4];  // (a bit cast of the vector's element itself takes its first)
    if constexpr (sizeof(T) == 4)
      return __builtin_bit_cast(float, v);
    else
      return value_of(__builtin_bit_cast(T, (uint16_t)(v >> 16 * (e & 1))));
  }
  // Elements first .. first + E - 1 of a row of V, -inf where there are none. At the
  // row's ends the load is moved to lie in it, and what is another piece's becomes
  // -inf; rows shorter than a piece are read by elements.
  __device__ __forceinline__ void load(const T* row, int first, int V) {
    constexpr unsigned kNone = sizeof(T) == 4 ? 0xff800000u : __is_same(T, f16) ? 0xfc00u : 0xff80u;
    constexpr int PER = 4 / sizeof(T);  // elements a register
    // register k with element e of the piece replaced, where `so`
    auto with = [](unsigned v, int e, unsigned bits, bool so) {
      const unsigned x = PER == 1 ? bits : e & 1 ? (v & 0xffffu) | bits << 16 : (v & 0xffff0000u) | bits;
      return so ? x : v;
    };
    unsigned v[4];
    if (V < E) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = PER == 1 ? kNone : kNone << 16 | kNone;
#pragma unroll 1
      for (int e = 0; e < V; ++e) {
        const int at = e - first;
        unsigned bits;
        if constexpr (PER == 1)
          bits = __builtin_bit_cast(unsigned, row[e]);
        else
          bits = __builtin_bit_cast(uint16_t, row[e]);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = with(v[k], at, bits, at >= 0 && at / PER == k);
      }
    } else {
      const int from = min(max(first, 0), V - E), d = first - from;  // elements d .. E - 1 + d are the piece's
      __builtin_memcpy(v, row + from, 16);
      if (__any(d != 0)) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e / PER] = with(v[e / PER], e, kNone, e < d || e >= E + d);
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) raw[k] = (int)v[k];
  }
  // the element that position e of the piece holds
  __device__ __forceinline__ static int index(int first, int e, int V) { return V < E ? first + e : min(max(first, 0), V - E) + e; }
};

__device__ __forceinline__ const VerifyStat* stats_of(const VerifyArgs& a, bool draft, int b, int i) {
  return a.stats + (draft ? (int64_t)a.B * a.n + (int64_t)b * (a.n - 1) + i : (int64_t)b * a.n + i) * a.chunks;
}

}  // namespace

// One chunk of a row a workgroup: 256 U pieces of 16 bytes. Bound by the weights'
// instructions (18 of 64 bits and 5 of 32 an element) where the chip is full.
template <class T, int U, bool BEST>
__global__ __launch_bounds__(256, 8) void verify_stats_kernel(VerifyArgs a) {
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
  const int shift = shift_of(p);
  Piece<T> x[U];
#pragma unroll
  for (int u = 0; u < U; ++u) x[u].load(p, ((chunk * U + u) * 256 + (int)threadIdx.x) * E - shift, a.V);
  float top = kNegInf;
  int place = INT_MAX;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (BEST) {
        if (x[u][e] > top) {  // in ascending order: the lowest of equal ones
          top = x[u][e];
          place = Piece<T>::index(((chunk * U + u) * 256 + (int)threadIdx.x) * E - shift, e, a.V);
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
    auto add = [&](const auto& weigh) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // one piece after another: registers for eight waves a SIMD, whose loads
        // and sums overlap
        asm volatile("" : "+v"(x[u].raw));  // converted again, not kept converted
#pragma unroll
        for (int e = 0; e < E; ++e) sum += weigh(x[u][e]);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    const double topc = (double)top * a.c;
    if (fabs(topc) < 65536.0)
      add(WeighFast{table, a.c, topc});
    else
      add(Weigh{table, a.c, (double)top});
  }
  sum = wave_sum(sum);
  if (lane == 0) sums[w] = sum;
  __syncthreads();
  if (threadIdx.x == 0) out = VerifyStat{(sums[0] + sums[1]) + (sums[2] + sums[3]), top, -1};
}

namespace {

// A row's largest logit and the sum of its weights.
struct RowSum {
  float top;
  double sum;
};
// Joins a row's chunks with `per` lanes (a power of two), of which this is number `sub`.
__device__ __forceinline__ RowSum row_sum(const VerifyStat* st, int chunks, bool real, int sub, int per,
                                          const double* table, double c) {
  VerifyStat mine{0.0, kNegInf, -1};
  if (real && sub < chunks) mine = st[sub];
  float top = mine.top;
  for (int k = sub + per; real && k < chunks; k += per) top = fmaxf(top, st[k].top);
  for (int o = 1; o < per; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
  double sum = mine.sum > 0.0 ? mine.sum * weight_below(table, c, mine.top, top) : 0.0;
  for (int k = sub + per; real && k < chunks; k += per)
    sum = fma(st[k].sum, st[k].sum > 0.0 ? weight_below(table, c, st[k].top, top) : 0.0, sum);
  for (int o = 1; o < per; o <<= 1) sum += __shfl_xor(sum, o);
  return {top, sum};
}

// r = max(ap wp - aq wq, 0) of a token's logits, wp and wq their weights below the
// rows' largest; 0 where it is one of `count` that were turned down.
template <bool DRAFT>
struct Rest {
  Weigh p, q;
  double ap, aq;
  bool pinf, qinf;
  const int64_t* gone;
  int count;
  // state (pa, qc) of the decisions: r = max(pa p - qc q, 0)
  __device__ __forceinline__ Rest(const double* table, double c, const RowSum& ps, const RowSum& qs, double pa,
                                  double qc)
      : p{table, c, (double)ps.top}, q{table, c, (double)qs.top}, ap(ps.sum > 0.0 ? pa / ps.sum : 0.0),
        aq(DRAFT && qc > 0.0 && qs.sum > 0.0 ? qc / qs.sum : 0.0), pinf(ps.top == __builtin_inff()),
        qinf(DRAFT && qs.top == __builtin_inff()), gone(nullptr), count(0) {}
  // Of the 16 bytes of elements from `first` on; 0 where there are none.
  template <class T, int E>
  __device__ __forceinline__ void of(const Piece<T>& lp, const Piece<T>& lq, int first, int V, double (&r)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      r[e] = 0.0;
      if (ap > 0.0) r[e] = ap * (pinf ? (lp[e] == __builtin_inff() ? 1.0 : 0.0) : p(lp[e]));
      if constexpr (DRAFT) {
        if (aq > 0.0) r[e] -= aq * (qinf ? (lq[e] == __builtin_inff() ? 1.0 : 0.0) : q(lq[e]));
        r[e] = fmax(r[e], 0.0);
      }
    }
    if constexpr (!DRAFT) {
      for (int k = 0; k < count; ++k) {
        const int64_t t = gone[k];
        if (!__any(t >= first && t < first + E)) continue;
#pragma unroll
        for (int e = 0; e < E; ++e)
          r[e] = t == Piece<T>::index(first, e, V) ? 0.0 : r[e];
      }
    }
  }
};

// The decisions behind one token, drafts that were drawn: drafts of `kids` in
// order. Lane i of the wave holds draft i's p, q and number; all lanes agree, and so
// do the kernels (sums join in one order, no product is fused into a sum but where
// it says so), so that what one asks for another has summed.
struct Asked {
  double pa = 1.0, qc = 0.0, Z = 1.0;  // r = max(pa p - qc q, 0), and its sum
  int kept = -1, rejections = 0;
  bool fresh = false;  // the masses of the last rejection are those of r
  // masses_of(k, pa, qc): the sum of r's masses after rejection k; stop(k): end there
  template <class Sum, class Stop>
  __device__ __forceinline__ bool run(uint64_t kids, double p, double q, double u, const Sum& sum_of, const Stop& stop) {
    for (; kids; kids &= kids - 1) {
      const int i = __builtin_ctzll(kids);
      const double pi = __shfl(p, i), qi = __shfl(q, i), ui = __shfl(u, i);
      if (ui * qi * Z < fma(pa, pi, -(qc * qi))) {
        kept = i;
        return true;
      }
      pa /= Z;
      qc = qc / Z + 1.0;
      if (stop(rejections)) return false;
      Z = sum_of(rejections, pa, qc);
      ++rejections;
      fresh = Z > 0.0;
      if (!fresh) {  // nothing is left: the token's own distribution in its place
        pa = Z = 1.0;
        qc = 0.0;
      }
    }
    return true;
  }
};

// A lane's draft: what it was drafted behind, its token and number.
struct Draft {
  int parent = -1;
  int64_t token = -1;
  double u = 0.0;
  __device__ __forceinline__ Draft(const VerifyArgs& a, int b, int nb, int lane) {
    if (lane > 0 && lane < nb) {
      parent = parent_of(a, b, lane);
      token = a.tokens[(int64_t)b * a.n + lane];
      u = (double)a.uniform[(int64_t)b * a.n + lane];
    }
  }
  __device__ __forceinline__ bool known(const VerifyArgs& a) const { return parent >= 0 && token >= 0 && token < a.V; }
};

// A wave's sum of a row of masses: the same wherever it is taken.
__device__ __forceinline__ double mass_sum(const double* masses, int chunks, int lane) {
  double sum = 0.0;
  for (int c = lane; c < chunks; c += 64) sum += masses[c];
  return wave_sum(sum);
}
__device__ __forceinline__ double* masses_of(const VerifyArgs& a, int round, int b, int node) {
  return a.masses + (((int64_t)round * a.B + b) * (a.n - 1) + node) * a.chunks;
}

}  // namespace

// The sums of all rows of a sequence, by a workgroup of NT: 2^k lanes a row, as many
// rows at a time as it has. `parent`: of the lane's draft.
template <bool DRAFT, int NT>
__device__ __forceinline__ void row_sums(const VerifyArgs& a, int b, int nb, int parent, const double* table,
                                         RowSum (&rows)[2][64]) {
  int per = 1;
  while (per < a.chunks && per < 64) per *= 2;
  const int sub = threadIdx.x & (per - 1);
  uint64_t inner = 0;  // tokens with drafts
  if constexpr (DRAFT)
    for (int i = 0; i < nb; ++i)
      if (__any(parent == i)) inner |= (uint64_t)1 << i;
  for (int r0 = 0; r0 < (DRAFT ? 2 * nb : nb); r0 += NT / per) {
    const int r = r0 + threadIdx.x / per, kind = r >= nb, i = r - kind * nb;
    const bool real = r < (DRAFT ? 2 * nb : nb) && (!kind || (inner >> i & 1));
    const RowSum x = row_sum(stats_of(a, kind, b, real ? i : 0), a.chunks, real, sub, per, table, a.c);
    if (real && sub == 0) rows[kind][i] = x;
  }
  __syncthreads();
}

// What r has in one chunk after rejection number `round` behind a token, if there
// are as many and no draft is kept before. In a chain the token is the one at whose
// draft it ends, known to a workgroup after the sums of all rows; in a tree it is any
// that has drafts (its place on the path is not asked for): there every wave decides
// by itself, and most workgroups end after three round trips to memory.
template <class T, int U, bool CHAIN>
__global__ __launch_bounds__(256) void verify_mass_kernel(VerifyArgs a, int round) {
  constexpr int E = 16 / sizeof(T);
  __shared__ double table[32], sums[4];
  __shared__ RowSum rows[2][64];
  const int chunk = blockIdx.x % a.chunks, k = blockIdx.x / a.chunks, b = CHAIN ? k : k / (a.n - 1);
  int node = CHAIN ? 0 : k % (a.n - 1);
  const int lane = threadIdx.x & 63, nb = tokens_of(a, b);
  if (nb < 2) return;
  const Draft d(a, b, nb, lane);
  if (!CHAIN && __builtin_popcountll(__ballot(d.parent == node)) <= round) return;
  float lp = kNegInf, lq = kNegInf;
  if ((CHAIN || d.parent == node) && d.known(a)) {
    lp = value_of(row_of<T>(a.p, b, d.parent)[d.token]);
    lq = value_of(row_of<T>(a.q, b, d.parent)[d.token]);
  }
  if (threadIdx.x < 32) table[threadIdx.x] = kExp2Table[threadIdx.x];
  __syncthreads();
  RowSum ps, qs;
  if constexpr (CHAIN) {
    row_sums<true, 256>(a, b, nb, d.parent, table, rows);
    ps = rows[0][max(d.parent, 0)];
    qs = rows[1][max(d.parent, 0)];
  } else {
    ps = row_sum(stats_of(a, false, b, node), a.chunks, true, lane, 64, table, a.c);
    qs = row_sum(stats_of(a, true, b, node), a.chunks, true, lane, 64, table, a.c);
  }
  const double p = ps.sum > 0.0 ? weight_below(table, a.c, lp, ps.top) / ps.sum : 0.0;
  const double q = qs.sum > 0.0 ? weight_below(table, a.c, lq, qs.top) / qs.sum : 0.0;
  double pa = 1.0, qc = 1.0;  // after the first rejection
  if constexpr (CHAIN) {
    const uint64_t ends = __ballot(d.parent >= 0 && !(d.u * q < p));
    if (!ends) return;
    node = __builtin_ctzll(ends) - 1;
    ps = rows[0][node];
    qs = rows[1][node];
  } else {
    Asked asked;
    if (asked.run(__ballot(d.parent == node), p, q, d.u,
                  [&](int r, double, double) { return mass_sum(masses_of(a, r, b, node), a.chunks, lane); },
                  [&](int r) { return r == round; }))
      return;
    pa = asked.pa;
    qc = asked.qc;
  }
  const Rest<true> rest(table, a.c, ps, qs, pa, qc);
  const T *prow = row_of<T>(a.p, b, node), *qrow = row_of<T>(a.q, b, node);
  const int first = (chunk * U * 256 + (int)threadIdx.x) * E - shift_of(prow);
  double sum = 0.0;
  Piece<T> x, y;
  x.load(prow, first, a.V);
  y.load(qrow, first, a.V);
#pragma unroll 1
  for (int u = 0; u < U; ++u) {
    const Piece<T> lp0 = x, lq0 = y;
    if (u + 1 < U) {
      x.load(prow, first + (u + 1) * 256 * E, a.V);
      y.load(qrow, first + (u + 1) * 256 * E, a.V);
    }
    double r[E];
    rest.of(lp0, lq0, first + u * 256 * E, a.V, r);
#pragma unroll
    for (int e = 0; e < E; ++e) sum += r[e];
  }
  sum = wave_sum(sum);
  if (lane == 0) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) masses_of(a, round, b, node)[chunk] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The decisions of a sequence from the root on, and its next token.
template <class T, bool BEST, bool DRAFT, int U>
__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(VerifyArgs a) {
  constexpr int E = 16 / sizeof(T), NT = kVerifyThreads, NW = NT / 64;
  __shared__ double table[32], part[NW], masses[kVerifyMaxChunks];
  __shared__ RowSum rows[2][64];
  __shared__ int best[64];
  __shared__ int64_t gone_tokens[64];
  __shared__ int found, last[NW], chosen;
  __shared__ double chosen_before;
  const int b = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nb = tokens_of(a, b);
  int32_t* keep = a.keep + (int64_t)b * a.n;
  if (nb == 0) {
    if (threadIdx.x < a.n) keep[threadIdx.x] = -1;
    if (threadIdx.x == 0) {
      a.keep_lens[b] = 0;
      a.token[b] = -1;
    }
    return;
  }
  // every wave holds the drafts and takes the same steps
  const Draft d(a, b, nb, lane);
  float lp = kNegInf, lq = kNegInf;
  if constexpr (!BEST) {
    if (d.known(a)) {
      lp = value_of(row_of<T>(a.p, b, d.parent)[d.token]);
      if constexpr (DRAFT) lq = value_of(row_of<T>(a.q, b, d.parent)[d.token]);
    }
    if (threadIdx.x < 32) table[threadIdx.x] = kExp2Table[threadIdx.x];
    __syncthreads();
  }
  if constexpr (BEST) {
    int per = 1;
    while (per < a.chunks && per < 64) per *= 2;
    const int sub = threadIdx.x & (per - 1);
    for (int r0 = 0; r0 < nb; r0 += NT / per) {
      const int r = r0 + threadIdx.x / per;
      const VerifyStat* st = stats_of(a, false, b, min(r, nb - 1));
      float top = kNegInf;
      int at = INT_MAX;
      for (int c = sub; c < a.chunks; c += per)
        if (st[c].top > top) {
          top = st[c].top;
          at = st[c].best;
        }
      for (int o = 1; o < per; o <<= 1) {
        const float x = __shfl_xor(top, o);
        const int other = __shfl_xor(at, o);
        if (x > top || (x == top && other < at)) at = other;
        top = fmaxf(top, x);
      }
      if (r < nb && sub == 0) best[r] = top > kNegInf ? at : -1;
    }
    __syncthreads();
  } else {
    row_sums<DRAFT, NT>(a, b, nb, d.parent, table, rows);
  }

  int node = 0;
  uint64_t taken = 1;
  auto write_path = [&]() {
    if (w != 0) return;
    const int count = __builtin_popcountll(taken), at = __builtin_popcountll(taken & (((uint64_t)1 << lane) - 1));
    if (taken >> lane & 1) keep[at] = lane;
    if (lane >= count && lane < a.n) keep[lane] = -1;
    if (lane == 0) a.keep_lens[b] = count;
  };
  if constexpr (BEST) {
    for (;;) {
      const int64_t top = best[node];
      const uint64_t ok = __ballot(d.parent == node && d.token == top && top >= 0);
      if (!ok) break;
      node = __builtin_ctzll(ok);
      taken |= (uint64_t)1 << node;
    }
    write_path();
    if (threadIdx.x == 0) a.token[b] = best[node];
    return;
  }
  double p = 0.0, q = 0.0;
  if (d.known(a)) {
    const RowSum ps = rows[0][d.parent];
    p = ps.sum > 0.0 ? weight_below(table, a.c, lp, ps.top) / ps.sum : 0.0;
    if constexpr (DRAFT) {
      const RowSum qs = rows[1][d.parent];
      q = qs.sum > 0.0 ? weight_below(table, a.c, lq, qs.top) / qs.sum : 0.0;
    }
  }
  // sum of one number a lane over the workgroup
  auto group_sum = [&](double x) {
    x = wave_sum(x);
    __syncthreads();
    if (lane == 0) part[w] = x;
    __syncthreads();
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < NW; ++k) sum += part[k];
    return sum;
  };
  // lane's share of a chunk: a run of pieces of 16 bytes, so that lanes are in the
  // tokens' order
  constexpr int RUN = (256 * U + NT - 1) / NT;
  auto chunk_first = [&](int chunk, int shift) { return (chunk * 256 * U + (int)threadIdx.x * RUN) * E - shift; };
  const bool has_share = (int)threadIdx.x * RUN < 256 * U;
  auto rest_of = [&](const Rest<DRAFT>& rest, const T* prow, const T* qrow, int first, double (&r)[E]) {
    Piece<T> x, y;
    x.load(prow, first, a.V);
    if (DRAFT && rest.aq > 0.0)
      y.load(qrow, first, a.V);
    else
      y = x;
    rest.of(x, y, first, a.V, r);
  };
  auto chunk_mass = [&](const Rest<DRAFT>& rest, const T* prow, const T* qrow, int chunk, int shift) {
    double sum = 0.0;
    if (has_share) {
#pragma unroll
      for (int u = 0; u < RUN; ++u) {
        double r[E];
        rest_of(rest, prow, qrow, chunk_first(chunk, shift) + u * E, r);
#pragma unroll
        for (int e = 0; e < E; ++e) sum += r[e];
      }
    }
    return group_sum(sum);
  };

  double pa = 1.0, qc = 0.0;
  uint64_t gone = 0;   // drafts that were turned down, where they were not drawn
  bool fresh = false;  // `masses` are r's
  for (;;) {
    const uint64_t kids = __ballot(d.parent == node);
    int next = -1;
    if constexpr (DRAFT) {
      Asked asked;
      asked.run(
          kids, p, q, d.u,
          [&](int r, double apa, double aqc) {
            __syncthreads();  // the masses of the rejection before are read
            if (r < a.rounds) {
              const double* from = masses_of(a, r, b, node);
              for (int c = threadIdx.x; c < a.chunks; c += NT) masses[c] = from[c];
            } else {
              const T *prow = row_of<T>(a.p, b, node), *qrow = row_of<T>(a.q, b, node);
              const Rest<DRAFT> rest(table, a.c, rows[0][node], rows[1][node], apa, aqc);
              const int shift = shift_of(prow);
              for (int c = 0; c < a.chunks; ++c) {
                const double m = chunk_mass(rest, prow, qrow, c, shift);
                if (threadIdx.x == 0) masses[c] = m;
              }
            }
            __syncthreads();
            return mass_sum(masses, a.chunks, lane);
          },
          [](int) { return false; });
      next = asked.kept;
      pa = asked.pa;
      qc = asked.qc;
      fresh = asked.fresh;
    } else {
      double Z = 1.0;
      gone = 0;
      for (uint64_t left = kids; left; left &= left - 1) {
        const int i = __builtin_ctzll(left);
        const double pi = __shfl(p, i), ui = __shfl(d.u, i);
        const bool again = (gone & __ballot(d.token == __shfl(d.token, i))) != 0;  // turned down before
        if (ui * Z < (again ? 0.0 : pi)) {
          next = i;
          break;
        }
        gone |= (uint64_t)1 << i;
        if (!again) Z = fmax(Z - pi, 0.0);
      }
    }
    if (next < 0) break;
    node = next;
    taken |= (uint64_t)1 << node;
  }
  write_path();

  // r's masses where the last event was no rejection with any left: the chunks'
  // own, without what was turned down
  const T* prow = row_of<T>(a.p, b, node);
  const T* qrow = DRAFT && qc > 0.0 ? row_of<T>(a.q, b, node) : prow;
  const int shift = shift_of(prow);
  RowSum ps = rows[0][node], qs{0.f, 0.0};
  if (DRAFT && qc > 0.0) qs = rows[1][node];
  Rest<DRAFT> rest(table, a.c, ps, qs, pa, qc);
  double Z = 0.0;
  if (!(DRAFT && fresh)) {
    auto own_masses = [&]() {
      __syncthreads();
      const VerifyStat* st = stats_of(a, false, b, node);
      for (int c = threadIdx.x; c < a.chunks; c += NT)
        masses[c] = st[c].sum > 0.0 ? rest.ap * (st[c].sum * weight_below(table, a.c, st[c].top, ps.top)) : 0.0;
      __syncthreads();
    };
    own_masses();
    if constexpr (!DRAFT) {
      if (gone) {
        if (threadIdx.x < 64 && (gone >> lane & 1))
          gone_tokens[__builtin_popcountll(gone & (((uint64_t)1 << lane) - 1))] = d.token;
        __syncthreads();
        rest.gone = gone_tokens;
        rest.count = __builtin_popcountll(gone);
        for (int k = 0; k < rest.count; ++k) {
          const int64_t t = gone_tokens[k];
          if (t < 0 || t >= a.V) continue;
          const int c = (int)((t + shift) / a.chunk);
          const double m = chunk_mass(rest, prow, prow, c, shift);
          if (threadIdx.x == 0) masses[c] = m;
        }
        __syncthreads();
        if (mass_sum(masses, a.chunks, lane) == 0.0) {  // nothing is left
          rest.count = 0;
          own_masses();
        }
      }
    }
  }
  Z = mass_sum(masses, a.chunks, lane);
  if (!(Z > 0.0)) {
    if (threadIdx.x == 0) a.token[b] = -1;
    return;
  }
  // The first token whose running sum passes u Z: its chunk, then within it. Where
  // rounding leaves none behind a border, the last one that has a mass.
  const double want = (double)a.uniform[(int64_t)b * a.n] * Z;
  // Of the lanes' sums in order: whether this lane's end is the first past `want`,
  // or it is the last with a mass if none is; before: the sum before the first
  // lane's, then before this one's.
  auto is_first_past = [&](double sum, double& before) {
    double upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double x = __shfl_up(upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();
    if (lane == 63) part[w] = upto;
    if (threadIdx.x == 0) found = INT_MAX;
    __syncthreads();
    for (int k = 0; k < w; ++k) before += part[k];
    const uint64_t past = __ballot(sum > 0.0 && before + upto > want), some = __ballot(sum > 0.0);
    before += upto - sum;
    if (lane == 0) {
      last[w] = some ? 64 * w + 63 - __builtin_clzll(some) : -1;
      if (past) atomicMin(&found, 64 * w + __builtin_ctzll(past));
    }
    __syncthreads();
    int at = found;
    if (at == INT_MAX) {
      at = last[0];
#pragma unroll
      for (int k = 1; k < NW; ++k) at = max(at, last[k]);
    }
    return at == (int)threadIdx.x;
  };
  const int run = (a.chunks + NT - 1) / NT, c0 = threadIdx.x * run, c1 = min(c0 + run, a.chunks);
  double sum = 0.0, before = 0.0;
  for (int c = c0; c < c1; ++c) sum += masses[c];
  if (is_first_past(sum, before)) {
    int pick = 0;
    double at = before, pick_at = before;
    for (int c = c0; c < c1; ++c) {
      if (masses[c] > 0.0) {
        pick = c;
        pick_at = at;
        if (at + masses[c] > want) break;
      }
      at += masses[c];
    }
    chosen = pick;
    chosen_before = pick_at;
  }
  __syncthreads();
  double r[RUN][E];
  sum = 0.0;
#pragma unroll
  for (int u = 0; u < RUN; ++u) {
    if (has_share) {
      rest_of(rest, prow, qrow, chunk_first(chosen, shift) + u * E, r[u]);
#pragma unroll
      for (int e = 0; e < E; ++e) sum += r[u][e];
    }
  }
  before = chosen_before;
  if (is_first_past(sum, before)) {
    int pick = -1;
    bool done = false;
#pragma unroll
    for (int u = 0; u < RUN; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!done && r[u][e] > 0.0) {
          pick = Piece<T>::index(chunk_first(chosen, shift) + u * E, e, a.V);
          before += r[u][e];
          done = before > want;
        }
    a.token[b] = pick;
  }
}

namespace {
template <class T, int U>
hipError_t launch_verify_u(const VerifyArgs& a, hipStream_t s) {
  const bool draft = a.q.data != nullptr;
  const dim3 block(256), rows((unsigned)((int64_t)a.B * (draft ? 2 * a.n - 1 : a.n) * a.chunks));
  if (a.best)
    MORPHO_KLAUNCH((verify_stats_kernel<T, U, true>), rows, block, 0, s, a);
  else
    MORPHO_KLAUNCH((verify_stats_kernel<T, U, false>), rows, block, 0, s, a);
  hipError_t e = hipGetLastError();
  for (int k = 0; k < a.rounds && e == hipSuccess; ++k) {
    if (a.tree)
      MORPHO_KLAUNCH((verify_mass_kernel<T, U, false>), dim3((unsigned)((int64_t)a.B * (a.n - 1) * a.chunks)), block, 0, s,
                     a, k);
    else
      MORPHO_KLAUNCH((verify_mass_kernel<T, U, true>), dim3((unsigned)((int64_t)a.B * a.chunks)), block, 0, s, a, k);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)a.B), all(kVerifyThreads);
  if (a.best)
    MORPHO_KLAUNCH((verify_kernel<T, true, false, U>), grid, all, 0, s, a);
  else if (draft)
    MORPHO_KLAUNCH((verify_kernel<T, false, true, U>), grid, all, 0, s, a);
  else
    MORPHO_KLAUNCH((verify_kernel<T, false, false, U>), grid, all, 0, s, a);
  return hipGetLastError();
}
template <class T>
hipError_t launch_verify_t(const VerifyArgs& a, const VerifyPlan& p, hipStream_t s) {
  return p.pieces == 1 ? launch_verify_u<T, 1>(a, s) : launch_verify_u<T, 4>(a, s);
}
}  // namespace

hipError_t launch_verify(const VerifyArgs& a, const VerifyPlan& p, int type, hipStream_t s) {
  if (type == 0) return launch_verify_t<f16>(a, p, s);
  if (type == 1) return launch_verify_t<Bf16>(a, p, s);
  return launch_verify_t<float>(a, p, s);
}

}  // namespace morpho
