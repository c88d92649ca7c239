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
// the terms then moves a border by 2^-45 or so of the row's whole, and the same
// inputs give the same tokens as any other 64-bit evaluation but for numbers that
// close to a border. (In 32 bits one of a thousand sampled tokens is another one.)
// Behind drafts that were turned down r is a difference (of a p and c q, or of p and
// the drafts), so its borders move by that over what is left of the whole; that
// little is left is as rare as it is little.
//
// 1. verify_stats_kernel: of every row's chunks the largest logit and the sum of
//    the weights below it (the only pass over all rows).
// 2. verify_mass_kernel, where drafts were drawn: what r has in each chunk after
//    the first, second, ... rejection behind a token, by the whole chip.
// 3. verify_kernel: the decisions and the next token, one workgroup a sequence; a
//    remainder that step 2 did not come to is summed here.
// A chunk is what one wave takes at a time, 64 U pieces of 16 bytes. Small, since
// the last step draws from one on a single CU.
//
// Measured (kernels, step 1 + 2 + 3): one chain of 5 over 32000 tokens 3.2 + 5.1 + 7.7
// us, 64 of 6 over 128000 (180 MB) 54 + 16 + 12, 16 trees of 48 over 50001, not drawn,
// full (77 MB) 25.5 + 9.4, ragged (17 MB) 11.1 + 8.6, 8 drawn of 24 over 32001 11.7 +
// 6 x 7.9 + 22, 32 of 8 over 65536 at temperature 0 11.0 + 4.0 (34 MB). Step 1 is bound by the
// weights' instructions where its rows fill the chip (3.4 TB/s; the full trees 3.0); of the
// ragged trees' 11.1 us those are 4, the rest is the launch and the waves of the rows that
// are padding, three of four, each with its table and barrier. Steps 2 and 3 are chains
// of loads and decisions on a cold instruction cache: a workgroup of 1024 threads, whose
// waves all decide, is a third slower in step 3 than one of 512.
#include <limits.h>

#include "common.h"
#include "internal.h"

namespace morpho {

namespace {

// Powers of two by a table and a short polynomial, the way of P. T. P. Tang's
// table-driven exponential (ACM Transactions on Mathematical Software 15, 1989). An
// entry is the double next to 2^(i / 256), less i 2^44, so that adding n 2^44 with
// n = 256 e + i gives the bits of 2^(n / 256).
constexpr int kTable = 256;
__constant__ uint64_t kExp2Table[kTable] = {
    0x3ff0000000000000, 0x3feffb1afa5abcbf, 0x3feff63da9fb3335, 0x3feff168143b0281, 0x3fefec9a3e778061, 0x3fefe7d42e11bbcc,
    0x3fefe315e86e7f85, 0x3fefde5f72f654b1, 0x3fefd9b0d3158574, 0x3fefd50a0e3c1f89, 0x3fefd06b29ddf6de, 0x3fefcbd42b72a836,
    0x3fefc74518759bc8, 0x3fefc2bdf66607e0, 0x3fefbe3ecac6f383, 0x3fefb9c79b1f3919, 0x3fefb5586cf9890f, 0x3fefb0f145e46c85,
    0x3fefac922b7247f7, 0x3fefa83b23395dec, 0x3fefa3ec32d3d1a2, 0x3fef9fa55fdfa9c5, 0x3fef9b66affed31b, 0x3fef973028d7233e,
    0x3fef9301d0125b51, 0x3fef8edbab5e2ab6, 0x3fef8abdc06c31cc, 0x3fef86a814f204ab, 0x3fef829aaea92de0, 0x3fef7e95934f312e,
    0x3fef7a98c8a58e51, 0x3fef76a45471c3c2, 0x3fef72b83c7d517b, 0x3fef6ed48695bbc0, 0x3fef6af9388c8dea, 0x3fef672658375d2f,
    0x3fef635beb6fcb75, 0x3fef5f99f8138a1c, 0x3fef5be084045cd4, 0x3fef582f95281c6b, 0x3fef54873168b9aa, 0x3fef50e75eb44027,
    0x3fef4d5022fcd91d, 0x3fef49c18438ce4d, 0x3fef463b88628cd6, 0x3fef42be3578a819, 0x3fef3f49917ddc96, 0x3fef3bdda27912d1,
    0x3fef387a6e756238, 0x3fef351ffb82140a, 0x3fef31ce4fb2a63f, 0x3fef2e85711ece75, 0x3fef2b4565e27cdd, 0x3fef280e341ddf29,
    0x3fef24dfe1f56381, 0x3fef21ba7591bb70, 0x3fef1e9df51fdee1, 0x3fef1b8a66d10f13, 0x3fef187fd0dad990, 0x3fef157e39771b2f,
    0x3fef1285a6e4030b, 0x3fef0f961f641589, 0x3fef0cafa93e2f56, 0x3fef09d24abd886b, 0x3fef06fe0a31b715, 0x3fef0432edeeb2fd,
    0x3fef0170fc4cd831, 0x3feefeb83ba8ea32, 0x3feefc08b26416ff, 0x3feef96266e3fa2d, 0x3feef6c55f929ff1, 0x3feef431a2de883b,
    0x3feef1a7373aa9cb, 0x3feeef26231e754a, 0x3feeecae6d05d866, 0x3feeea401b7140ef, 0x3feee7db34e59ff7, 0x3feee57fbfec6cf4,
    0x3feee32dc313a8e5, 0x3feee0e544ede173, 0x3feedea64c123422, 0x3feedc70df1c5175, 0x3feeda4504ac801c, 0x3feed822c367a024,
    0x3feed60a21f72e2a, 0x3feed3fb2709468a, 0x3feed1f5d950a897, 0x3feecffa3f84b9d4, 0x3feece086061892d, 0x3feecc2042a7d232,
    0x3feeca41ed1d0057, 0x3feec86d668b3237, 0x3feec6a2b5c13cd0, 0x3feec4e1e192aed2, 0x3feec32af0d7d3de, 0x3feec17dea6db7d7,
    0x3feebfdad5362a27, 0x3feebe41b817c114, 0x3feebcb299fddd0d, 0x3feebb2d81d8abff, 0x3feeb9b2769d2ca7, 0x3feeb8417f4531ee,
    0x3feeb6daa2cf6642, 0x3feeb57de83f4eef, 0x3feeb42b569d4f82, 0x3feeb2e2f4f6ad27, 0x3feeb1a4ca5d920f, 0x3feeb070dde910d2,
    0x3feeaf4736b527da, 0x3feeae27dbe2c4cf, 0x3feead12d497c7fd, 0x3feeac0827ff07cc, 0x3feeab07dd485429, 0x3feeaa11fba87a03,
    0x3feea9268a5946b7, 0x3feea84590998b93, 0x3feea76f15ad2148, 0x3feea6a320dceb71, 0x3feea5e1b976dc09, 0x3feea52ae6cdf6f4,
    0x3feea47eb03a5585, 0x3feea3dd1d1929fd, 0x3feea34634ccc320, 0x3feea2b9febc8fb7, 0x3feea23882552225, 0x3feea1c1c70833f6,
    0x3feea155d44ca973, 0x3feea0f4b19e9538, 0x3feea09e667f3bcd, 0x3feea052fa75173e, 0x3feea012750bdabf, 0x3fee9fdcddd47645,
    0x3fee9fb23c651a2f, 0x3fee9f9298593ae5, 0x3fee9f7df9519484, 0x3fee9f7466f42e87, 0x3fee9f75e8ec5f74, 0x3fee9f8286ead08a,
    0x3fee9f9a48a58174, 0x3fee9fbd35d7cbfd, 0x3fee9feb564267c9, 0x3feea024b1ab6e09, 0x3feea0694fde5d3f, 0x3feea0b938ac1cf6,
    0x3feea11473eb0187, 0x3feea17b0976cfdb, 0x3feea1ed0130c132, 0x3feea26a62ff86f0, 0x3feea2f336cf4e62, 0x3feea3878491c491,
    0x3feea427543e1a12, 0x3feea4d2add106d9, 0x3feea589994cce13, 0x3feea64c1eb941f7, 0x3feea71a4623c7ad, 0x3feea7f4179f5b21,
    0x3feea8d99b4492ed, 0x3feea9cad931a436, 0x3feeaac7d98a6699, 0x3feeabd0a478580f, 0x3feeace5422aa0db, 0x3feeae05bad61778,
    0x3feeaf3216b5448c, 0x3feeb06a5e0866d9, 0x3feeb1ae99157736, 0x3feeb2fed0282c8a, 0x3feeb45b0b91ffc6, 0x3feeb5c353aa2fe2,
    0x3feeb737b0cdc5e5, 0x3feeb8b82b5f98e5, 0x3feeba44cbc8520f, 0x3feebbdd9a7670b3, 0x3feebd829fde4e50, 0x3feebf33e47a22a2,
    0x3feec0f170ca07ba, 0x3feec2bb4d53fe0d, 0x3feec49182a3f090, 0x3feec674194bb8d5, 0x3feec86319e32323, 0x3feeca5e8d07f29e,
    0x3feecc667b5de565, 0x3feece7aed8eb8bb, 0x3feed09bec4a2d33, 0x3feed2c980460ad8, 0x3feed503b23e255d, 0x3feed74a8af46052,
    0x3feed99e1330b358, 0x3feedbfe53c12e59, 0x3feede6b5579fdbf, 0x3feee0e521356eba, 0x3feee36bbfd3f37a, 0x3feee5ff3a3c2774,
    0x3feee89f995ad3ad, 0x3feeeb4ce622f2ff, 0x3feeee07298db666, 0x3feef0ce6c9a8952, 0x3feef3a2b84f15fb, 0x3feef68415b749b1,
    0x3feef9728de5593a, 0x3feefc6e29f1c52a, 0x3feeff76f2fb5e47, 0x3fef028cf22749e4, 0x3fef05b030a1064a, 0x3fef08e0b79a6f1f,
    0x3fef0c1e904bc1d2, 0x3fef0f69c3f3a207, 0x3fef12c25bd71e09, 0x3fef16286141b33d, 0x3fef199bdd85529c, 0x3fef1d1cd9fa652c,
    0x3fef20ab5fffd07a, 0x3fef244778fafb22, 0x3fef27f12e57d14b, 0x3fef2ba88988c933, 0x3fef2f6d9406e7b5, 0x3fef33405751c4db,
    0x3fef3720dcef9069, 0x3fef3b0f2e6d1675, 0x3fef3f0b555dc3fa, 0x3fef43155b5bab74, 0x3fef472d4a07897c, 0x3fef4b532b08c968,
    0x3fef4f87080d89f2, 0x3fef53c8eacaa1d6, 0x3fef5818dcfba487, 0x3fef5c76e862e6d3, 0x3fef60e316c98398, 0x3fef655d71ff6075,
    0x3fef69e603db3285, 0x3fef6e7cd63a8315, 0x3fef7321f301b460, 0x3fef77d5641c0658, 0x3fef7c97337b9b5f, 0x3fef81676b197d17,
    0x3fef864614f5a129, 0x3fef8b333b16ee12, 0x3fef902ee78b3ff6, 0x3fef953924676d76, 0x3fef9a51fbc74c83, 0x3fef9f7977cdb740,
    0x3fefa4afa2a490da, 0x3fefa9f4867cca6e, 0x3fefaf482d8e67f1, 0x3fefb4aaa2188510, 0x3fefba1bee615a27, 0x3fefbf9c1cb6412a,
    0x3fefc52b376bba97, 0x3fefcac948dd7274, 0x3fefd0765b6e4540, 0x3fefd632798844f8, 0x3fefdbfdad9cbe14, 0x3fefe1d802243c89,
    0x3fefe7c1819e90d8, 0x3fefedba3692d514, 0x3feff3c22b8f71f1, 0x3feff9d96b2a23d9};

// 2^((n + r) / 256), |r| <= 1/2, n >= -256000: 2^(n / 256) from the table and
// 2^(r / 256) by the cubic that meets it at the four Chebyshev nodes cos((2 k + 1) pi / 8) / 2
// (computed in 60 decimal digits, then rounded; 2^-45 off at most). A table of 64 takes a degree more, and two instructions where the low byte of
// n is the index.
__device__ __forceinline__ double exp2_256(const uint64_t* table, int n, double r) {
  double y = 0x1.c6b0902b5a0abp-29;
  y = fma(y, r, 0x1.ebfbe4e4d7394p-19);
  y = fma(y, r, 0x1.62e42fefa39d9p-9);
  y = fma(y, r, 0x1.fffffffffff62p-1);
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  i32x2 z = __builtin_bit_cast(i32x2, table[n & (kTable - 1)]);  // LDS
  int hi = z[1];
  asm("v_lshl_add_u32 %0, %1, 12, %0" : "+v"(hi) : "v"(n));  // (the compiler adds 64 bits, in five instructions)
  z[1] = hi;
  return y * __builtin_bit_cast(double, z);
}
constexpr double kWhole = 0x1.8p52;  // v + kWhole ends in the whole number next to v
__device__ __forceinline__ double exp2_256(const uint64_t* table, double v) {
  const double t = v + kWhole;
  return exp2_256(table, (int)__builtin_bit_cast(int64_t, t), v - (t - kWhole));
}
// The weight exp((x - top) / temperature) of a logit, 2^(v / 256) with v = (x - top) c
// <= 0, c = 256 log2(e) / temperature. The difference comes first: logits may be as
// large as their type allows. An infinite top is 1e39 here, and so is an infinite x,
// which then weighs 1 where any other weighs nothing. What weighs less than 2^-1000,
// NaN and -inf too, weighs that; below 2^-900 is taken for nothing everywhere.
constexpr double kNothing = 0x1p-900;
struct Weigh {
  const uint64_t* table;
  double c, top;
  __device__ __forceinline__ Weigh(const uint64_t* table, double c, float top)
      : table(table), c(c), top(fmin(fmax((double)top, -1e39), 1e39)) {}
  __device__ __forceinline__ double operator()(float x) const {
    // the lower bound first: it stands for NaN
    return exp2_256(table, fmax((fmin(fmax((double)x, -1e39), 1e39) - top) * c, -256000.0));
  }
  __device__ __forceinline__ double factor() const { return 1.0; }
};
// For long sums with |top c| below 2^40: three instructions less. The weights are over
// 2^(T / 256) with T the whole number next to top c, the sum's factor() puts it over
// top's: t = x c + (kWhole - T) ends in the whole number n next to x c - T, and
// r = x c + (kWhole - T - t) is what is left, the addend being exact in both.
struct WeighFast {
  const uint64_t* table;
  double c, K, rest, low;  // low: 2^-1000 of the top
  __device__ __forceinline__ static bool fits(double c, float top) { return fabs((double)top * c) < 0x1p40; }
  __device__ __forceinline__ WeighFast(const uint64_t* table, double c, float top) : table(table), c(c) {
    const double T = __builtin_rint((double)top * c);
    K = kWhole - T;
    rest = fma(-(double)top, c, T);
    low = (double)top - 256000.0 / c;
  }
  __device__ __forceinline__ double operator()(float x) const {
    const double d = fmax((double)x, low), t = fma(d, c, K);
    return exp2_256(table, (int)__builtin_bit_cast(int64_t, t), fma(d, c, K - t));
  }
  __device__ __forceinline__ double factor() const { return exp2_256(table, 0, rest); }
};
__device__ __forceinline__ double weight_below(const uint64_t* table, double c, float x, float top) {
  const double w = Weigh(table, c, top)(x);
  return w > kNothing && top > kNegInf ? w : 0.0;
}

struct Bf16 {
  uint16_t bits;
};
__device__ __forceinline__ float value_of(f16 x) { return (float)x; }
__device__ __forceinline__ float value_of(Bf16 x) { return __builtin_bit_cast(float, (unsigned)x.bits << 16); }
__device__ __forceinline__ float value_of(float x) { return x; }

// The values that step K of a reduction joins (K of 6: with those of lanes 1, 2, 4, 8,
// 16 and 32 away or their mirror images, which by then hold the same). Lanes' numbers
// go over registers here: through LDS a step of 64 bits takes some 150 cycles, and
// the last kernel is made of such steps.
template <int K>
__device__ __forceinline__ void joined(unsigned x, unsigned& a, unsigned& b) {
  if constexpr (K < 4) {
    constexpr int kDpp[4] = {0xb1, 0x4e, 0x141, 0x140};  // quad_perm 1 0 3 2, 2 3 0 1, row_half_mirror, row_mirror
    a = x;
    b = (unsigned)__builtin_amdgcn_mov_dpp((int)x, kDpp[K], 0xf, 0xf, false);
  } else {
    const auto r = K == 4 ? __builtin_amdgcn_permlane16_swap(x, x, false, false)
                          : __builtin_amdgcn_permlane32_swap(x, x, false, false);
    a = r[0];
    b = r[1];
  }
}
template <int K, class F>
__device__ __forceinline__ double join(double x, const F& f) {
  const uint64_t v = __builtin_bit_cast(uint64_t, x);
  unsigned al, bl, ah, bh;
  joined<K>((unsigned)v, al, bl);
  joined<K>((unsigned)(v >> 32), ah, bh);
  return f(__builtin_bit_cast(double, (uint64_t)ah << 32 | al), __builtin_bit_cast(double, (uint64_t)bh << 32 | bl));
}
template <int K, class F>
__device__ __forceinline__ float join(float x, const F& f) {
  unsigned a, b;
  joined<K>(__builtin_bit_cast(unsigned, x), a, b);
  return f(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
// Over runs of `per` lanes, a power of two.
template <class T, class F>
__device__ __forceinline__ T join_lanes(T x, int per, const F& f) {
  if (per > 1) x = join<0>(x, f);
  if (per > 2) x = join<1>(x, f);
  if (per > 4) x = join<2>(x, f);
  if (per > 8) x = join<3>(x, f);
  if (per > 16) x = join<4>(x, f);
  if (per > 32) x = join<5>(x, f);
  return x;
}
__device__ __forceinline__ double lanes_sum(double x, int per) {
  return join_lanes(x, per, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ float lanes_max(float x, int per) {
  return join_lanes(x, per, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ double wave_sum(double x) { return lanes_sum(x, 64); }
__device__ __forceinline__ float wave_max(float x) { return lanes_max(x, 64); }
__device__ __forceinline__ uint64_t wave_or(uint64_t x) {
  auto either = [](unsigned v) {
    unsigned a, b;
    joined<0>(v, a, b);
    joined<1>(a | b, a, b);
    joined<2>(a | b, a, b);
    joined<3>(a | b, a, b);
    joined<4>(a | b, a, b);
    joined<5>(a | b, a, b);
    return (unsigned)__builtin_amdgcn_readfirstlane((int)(a | b));
  };
  return (uint64_t)either((unsigned)(x >> 32)) << 32 | either((unsigned)x);
}
// The value of lane i, the same i in all of them.
__device__ __forceinline__ int lane_value(int x, int i) { return __builtin_amdgcn_readlane(x, i); }
__device__ __forceinline__ double lane_value(double x, int i) {
  const uint64_t v = __builtin_bit_cast(uint64_t, x);
  const unsigned lo = (unsigned)lane_value((int)(unsigned)v, i), hi = (unsigned)lane_value((int)(unsigned)(v >> 32), i);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over the lanes up to this one.
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_moved(double x) {
  const uint64_t v = __builtin_bit_cast(uint64_t, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, false);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_upto(double x) {
  x = add_moved<0x111, 0xf>(x);     // row_shr 1, 2, 4, 8
  x = add_moved<0x112, 0xf>(x);
  x = add_moved<0x114, 0xf>(x);
  x = add_moved<0x118, 0xf>(x);
  x = add_moved<0x142, 0xa>(x);     // row_bcast 15: of rows 0 and 2 to 1 and 3
  return add_moved<0x143, 0xc>(x);  // row_bcast 31: of row 1 to 2 and 3
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

// A chunk of a row a wave. Bound by the weights' instructions (14.5 an element, nine of
// them of 64 bits, 5.3 cycles each) where the chip is full.
template <class T, int U, bool BEST>
__global__ __launch_bounds__(256, 8) void verify_stats_kernel(VerifyArgs a, int rows) {
  constexpr int E = 16 / sizeof(T);
  static_assert(kTable == 256);
  __shared__ uint64_t table[kTable];
  const int lane = threadIdx.x & 63;
  uint64_t entry = 0;
  if constexpr (!BEST) entry = kExp2Table[threadIdx.x];  // on its way early
  const int id = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int row = min(id / a.chunks, rows - 1), chunk = id - row * a.chunks;
  const bool draft = row >= a.B * a.n;
  const int k = draft ? row - a.B * a.n : row, per = draft ? a.n - 1 : a.n, b = k / per, i = k - b * per;
  const int nb = tokens_of(a, b);
  // what a token without drafts of its own would have drawn from is not asked for
  const bool asked = chunk < a.chunks && i < nb && (!draft || __any(lane > i && lane < nb && parent_of(a, b, lane) == i));
  const T* p = row_of<T>(draft ? a.q : a.p, b, i);
  const int first = (chunk * U * 64 + lane) * E - shift_of(p);
  Piece<T> x[U];
  if (asked) {
#pragma unroll
    for (int u = 0; u < U; ++u) x[u].load(p, first + u * 64 * E, a.V);
  }
  if constexpr (!BEST) {
    table[threadIdx.x] = entry;
    __syncthreads();
  }
  if (!asked) return;
  float top = kNegInf;
  int place = INT_MAX;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = x[u][e];
      if constexpr (BEST) {
        const bool more = v > top;  // in ascending order: the lowest of equal ones
        place = more ? Piece<T>::index(first + u * 64 * E, e, a.V) : place;
        top = more ? v : top;
      } else {
        top = fmaxf(top, v);
      }
    }
  VerifyStat& out = a.stats[(int64_t)row * a.chunks + chunk];
  if constexpr (BEST) {
    const float all = wave_max(top);
    place = top == all ? place : INT_MAX;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) place = min(place, __shfl_xor(place, o));
    if (lane == 0) out = VerifyStat{0.0, all, all > kNegInf ? place : -1};
    return;
  }
  top = wave_max(top);
  double sum = 0.0;
  auto add = [&](const auto& weigh) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // one piece after another: registers for eight waves a SIMD, whose loads and
      // sums overlap
      asm volatile("" : "+v"(x[u].raw));  // converted again, not kept converted
#pragma unroll
      for (int e = 0; e < E; ++e) sum += weigh(x[u][e]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  if (top > kNegInf) {
    if (WeighFast::fits(a.c, top)) {
      const WeighFast weigh(table, a.c, top);
      add(weigh);
      sum *= weigh.factor();
    } else {
      add(Weigh(table, a.c, top));
    }
    sum = wave_sum(sum);
  }
  if (lane == 0) out = VerifyStat{sum, top, -1};
}

namespace {

// A row's largest logit and the sum of its weights.
struct RowSum {
  float top;
  double share;  // 1 / sum, nothing where there is none
};
// Joins a row's chunks with `per` lanes (a power of two), of which this is number `sub`.
__device__ __forceinline__ RowSum row_sum(const VerifyStat* st, int chunks, bool real, int sub, int per,
                                          const uint64_t* table, double c) {
  float top = kNegInf;
#pragma unroll 1
  for (int k = sub; real && k < chunks; k += per) top = fmaxf(top, st[k].top);
  top = lanes_max(top, per);
  double sum = 0.0;
#pragma unroll 1
  for (int k = sub; real && k < chunks; k += per) sum = fma(st[k].sum, weight_below(table, c, st[k].top, top), sum);
  sum = lanes_sum(sum, per);
  return {top, sum > 0.0 ? 1.0 / sum : 0.0};
}
// The sums of the rows that a sequence's drafts ask for, by a workgroup of NT: 2^k
// lanes a row, as many rows at a time as it has. `parent`: of the lane's draft.
template <bool DRAFT, int NT>
__device__ __forceinline__ void row_sums(const VerifyArgs& a, int b, int parent, const uint64_t* table,
                                         RowSum (&rows)[2][64]) {
  int per = 1;
  while (per < a.chunks && per < 64) per *= 2;
  const int lane = threadIdx.x & 63, sub = threadIdx.x & (per - 1);
  const uint64_t inner = wave_or(parent >= 0 ? (uint64_t)1 << parent : 0);  // tokens with drafts
  // lane k holds the k-th of them
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  const int count = __builtin_popcountll(inner);
  const int to = inner >> lane & 1 ? __builtin_popcountll(inner & below) : count + __builtin_popcountll(~inner & below);
  const int with_drafts = __builtin_amdgcn_ds_permute(4 * to, lane);
  for (int r0 = 0; r0 < (DRAFT ? 2 * count : count); r0 += NT / per) {
    const int r = r0 + threadIdx.x / per, kind = r >= count, i = __shfl(with_drafts, r - kind * count);
    const bool real = r < (DRAFT ? 2 * count : count);
    const RowSum x = row_sum(stats_of(a, kind, b, real ? i : 0), a.chunks, real, sub, per, table, a.c);
    if (real && sub == 0) rows[kind][i] = x;
  }
  __syncthreads();
}
// The chance of a logit in its row.
__device__ __forceinline__ double chance(const uint64_t* table, double c, float x, const RowSum& row) {
  return weight_below(table, c, x, row.top) * row.share;
}

// Pieces of the target's and the drafter's row at the same place.
template <class T>
struct PiecePair {
  Piece<T> p, q;
  __device__ __forceinline__ void load(const T* prow, const T* qrow, int first, int V) {
    p.load(prow, first, V);
    q.load(qrow, first, V);
  }
};
// r of logits lp and lq of a token in the target's and the drafter's row.
template <bool DRAFT, class W>
struct Rest {
  W p, q;
  double ap, aq;
  // state (pa, qc) of the decisions: r = max(pa p - qc q, 0)
  __device__ __forceinline__ Rest(const uint64_t* table, double c, const RowSum& ps, const RowSum& qs, double pa,
                                  double qc)
      : p(table, c, ps.top), q(table, c, qs.top), ap(pa * p.factor() * ps.share),
        aq(DRAFT && qc > 0.0 ? qc * q.factor() * qs.share : 0.0) {}
  __device__ __forceinline__ double operator()(float lp, float lq) const {
    double r = fma(ap, p(lp), -kNothing);
    if constexpr (DRAFT) r = fma(-aq, q(lq), r);
    return fmax(r, 0.0);
  }
  // The mass of a chunk, by a wave: a loop with one pair of pieces ahead. Unrolled it
  // takes all 256 registers and spills: 64 chains of 6 over 128000 16.2 -> 44.6 us for
  // the masses and 12 -> 20 in the last kernel (one chain of 5 over 32000 alike).
  template <class T, int U>
  __device__ __forceinline__ double mass(PiecePair<T> x, const T* prow, const T* qrow, int first, int V) const {
    double sum = 0.0;
#pragma unroll 1
    for (int u = 0;;) {
      PiecePair<T> next;
      if (++u < U) next.load(prow, qrow, first + u * 64 * Piece<T>::E, V);
#pragma unroll
      for (int e = 0; e < Piece<T>::E; ++e) sum += (*this)(x.p[e], x.q[e]);
      if (u >= U) break;
      x = next;
    }
    return wave_sum(sum);
  }
};
// The mass of a chunk, of which x is the lane's first pieces.
template <class T, int U>
__device__ __forceinline__ double chunk_mass(const uint64_t* table, double c, const RowSum& ps, const RowSum& qs, double pa,
                                             double qc, const PiecePair<T>& x, const T* prow, const T* qrow, int first,
                                             int V) {
  if (WeighFast::fits(c, ps.top) && WeighFast::fits(c, qs.top))
    return Rest<true, WeighFast>(table, c, ps, qs, pa, qc).template mass<T, U>(x, prow, qrow, first, V);
  return Rest<true, Weigh>(table, c, ps, qs, pa, qc).template mass<T, U>(x, prow, qrow, first, V);
}

// The decisions behind one token, drafts that were drawn: drafts of `kids` in
// order. Lane i of the wave holds draft i's p, q and number; all lanes agree, and so
// do the kernels (sums join in one order, no product is fused into a sum but where
// it says so), so that what one asks for another has summed.
struct Asked {
  double pa = 1.0, qc = 0.0, Z = 1.0;  // r = max(pa p - qc q, 0), and its sum
  int kept = -1, rejections = 0;
  bool fresh = false;  // the masses of the last rejection are those of r
  // sum_of(i, k, pa, qc): the sum of r's masses after rejection k, that of draft i; stop(k): end there (false)
  template <class Sum, class Stop>
  __device__ __forceinline__ bool run(uint64_t kids, double p, double q, double u, const Sum& sum_of, const Stop& stop) {
    for (; kids; kids &= kids - 1) {
      const int i = __builtin_ctzll(kids);
      const double pi = lane_value(p, i), qi = lane_value(q, i), ui = lane_value(u, i);
      if (ui * qi * Z < fma(pa, pi, -(qc * qi))) {
        kept = i;
        return true;
      }
      const double over = 1.0 / Z;
      pa *= over;
      qc = fma(qc, over, 1.0);
      if (stop(rejections)) return false;
      Z = sum_of(i, rejections, pa, qc);
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
    if (lane > 0 && lane < a.n) {  // nb may still be on its way
      parent = parent_of(a, b, lane);
      token = a.tokens[(int64_t)b * a.n + lane];
      u = (double)a.uniform[(int64_t)b * a.n + lane];
    }
    if (lane >= nb) parent = -1, token = -1;
  }
  __device__ __forceinline__ bool known(const VerifyArgs& a) const { return parent >= 0 && token >= 0 && token < a.V; }
};

// A wave's sum of a row of masses: the same wherever it is taken.
__device__ __forceinline__ double mass_sum(const double* masses, int chunks, int lane) {
  double sum = 0.0;
#pragma unroll 1
  for (int c = lane; c < chunks; c += 64) sum += masses[c];
  return wave_sum(sum);
}
__device__ __forceinline__ double* masses_of(const VerifyArgs& a, int round, int b, int node) {
  return a.masses + (((int64_t)round * a.B + b) * (a.n - 1) + node) * a.chunks;
}

}  // namespace

// What r has in a chunk (one a wave) after rejection number `round` behind a token, if
// there are as many and no draft is kept before. In a chain the token is the one at
// whose draft it ends, known to a workgroup after the sums of all rows; in a tree it is
// any that has drafts (its place on the path is not asked for); there a wave takes each
// of the sums that the decisions ask for.
template <class T, int U, bool CHAIN>
__global__ __launch_bounds__(kVerifyMassThreads) void verify_mass_kernel(VerifyArgs a, int round, int groups) {
  constexpr int NT = kVerifyMassThreads, NW = NT / 64;
  static_assert(NW >= 2 + kVerifyMaxRounds - 1 && NT >= kTable);
  __shared__ uint64_t table[kTable];
  __shared__ RowSum rows[2][64];
  __shared__ double sums[kVerifyMaxRounds - 1];  // of the masses of the rounds before
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint64_t entry = kExp2Table[threadIdx.x & (kTable - 1)];  // on its way early
  const int k = blockIdx.x / groups, b = CHAIN ? k : k / (a.n - 1);
  const int chunk = NW * (blockIdx.x - k * groups) + w, nb = tokens_of(a, b);
  int node = CHAIN ? 0 : k - b * (a.n - 1);
  const Draft d(a, b, nb, lane);
  if (nb < 2) return;
  PiecePair<T> x;
  const T *prow, *qrow;
  int first;
  auto load = [&]() {
    prow = row_of<T>(a.p, b, node);
    qrow = row_of<T>(a.q, b, node);
    first = (min(chunk, a.chunks - 1) * U * 64 + lane) * Piece<T>::E - shift_of(prow);
    x.load(prow, qrow, first, a.V);
  };
  const uint64_t kids = __ballot(d.parent == node);
  if (!CHAIN && __builtin_popcountll(kids) <= round) return;
  if (threadIdx.x < kTable) table[threadIdx.x] = entry;
  __syncthreads();
  float lp = kNegInf, lq = kNegInf;
  if ((CHAIN || d.parent == node) && d.known(a)) {
    lp = value_of(row_of<T>(a.p, b, d.parent)[d.token]);
    lq = value_of(row_of<T>(a.q, b, d.parent)[d.token]);
  }
  if constexpr (CHAIN) {
    row_sums<true, NT>(a, b, d.parent, table, rows);
  } else {
    load();  // early: decided while it is on its way
    if (w < 2) {
      const RowSum x = row_sum(stats_of(a, w, b, node), a.chunks, true, lane, 64, table, a.c);
      if (lane == 0) rows[w][0] = x;
    } else if (w < 2 + round) {
      const double sum = mass_sum(masses_of(a, w - 2, b, node), a.chunks, lane);
      if (lane == 0) sums[w - 2] = sum;
    }
    __syncthreads();
  }
  const int mine = CHAIN ? max(d.parent, 0) : 0;
  const double p = chance(table, a.c, lp, rows[0][mine]), q = chance(table, a.c, lq, rows[1][mine]);
  double pa = 1.0, qc = 1.0;  // after the first rejection
  if constexpr (CHAIN) {
    const uint64_t ends = __ballot(d.parent >= 0 && !(d.u * q < p));
    if (!ends) return;
    node = __builtin_ctzll(ends) - 1;
    load();
  } else {
    Asked asked;
    if (asked.run(kids, p, q, d.u, [&](int, int r, double, double) { return sums[r]; }, [&](int r) { return r == round; }))
      return;
    pa = asked.pa;
    qc = asked.qc;
  }
  const RowSum ps = rows[0][CHAIN ? node : 0], qs = rows[1][CHAIN ? node : 0];
  if (chunk >= a.chunks) return;
  const double m = chunk_mass<T, U>(table, a.c, ps, qs, pa, qc, x, prow, qrow, first, a.V);
  if (lane == 0) masses_of(a, round, b, node)[chunk] = m;
}

// The decisions of a sequence from the root on, and its next token.
template <class T, bool BEST, bool DRAFT, int U>
__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(VerifyArgs a) {
  constexpr int E = 16 / sizeof(T), NT = kVerifyThreads, NW = NT / 64;
  __shared__ uint64_t table[kTable];
  __shared__ double part[NW], masses[kVerifyMaxChunks];
  __shared__ RowSum rows[2][64];
  __shared__ double sums[64];
  __shared__ int best[64], found, last[NW];
  const int b = blockIdx.x, lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  uint64_t entry = 0;
  if constexpr (!BEST) entry = kExp2Table[threadIdx.x & (kTable - 1)];  // on its way early
  // every wave holds the drafts and takes the same steps
  const Draft d(a, b, nb, lane);
  float lp = kNegInf, lq = kNegInf;
  if constexpr (!BEST) {
    if (d.known(a)) {
      lp = value_of(row_of<T>(a.p, b, d.parent)[d.token]);
      if constexpr (DRAFT) lq = value_of(row_of<T>(a.q, b, d.parent)[d.token]);
    }
    if (threadIdx.x < kTable) table[threadIdx.x] = entry;
    __syncthreads();
    // the masses that draft i's rejection leaves: of the token behind which it was
    // drafted and the number of its siblings before it (nothing, where it was not asked)
    if constexpr (DRAFT) {
#pragma unroll 1
      for (int i = w; i < nb; i += NW) {
        const int node = lane_value(d.parent, i), r = __builtin_popcountll(__ballot(d.parent == node && lane < i));
        if (node < 0 || r >= a.rounds) continue;
        const double sum = mass_sum(masses_of(a, r, b, node), a.chunks, lane);
        if (lane == 0) sums[i] = sum;
      }
    }
    row_sums<DRAFT, NT>(a, b, d.parent, table, rows);
  } else {
    int per = 1;
    while (per < a.chunks && per < 64) per *= 2;
    const int sub = threadIdx.x & (per - 1);
    for (int r0 = 0; r0 < nb; r0 += NT / per) {
      const int r = r0 + threadIdx.x / per;
      const VerifyStat* st = stats_of(a, false, b, min(r, nb - 1));
      float top = kNegInf;
      int at = INT_MAX;
      for (int c = sub; c < a.chunks; c += per) {
        const VerifyStat x = st[c];
        at = x.top > top ? x.best : at;
        top = fmaxf(top, x.top);
      }
      for (int o = 1; o < per; o <<= 1) {
        const float x = __shfl_xor(top, o);
        const int other = __shfl_xor(at, o);
        at = x > top || (x == top && other < at) ? other : at;
        top = fmaxf(top, x);
      }
      if (r < nb && sub == 0) best[r] = top > kNegInf ? at : -1;
    }
    __syncthreads();
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
  const double u0 = (double)a.uniform[(int64_t)b * a.n];
  const int mine = max(d.parent, 0);
  double p = 0.0, q = 0.0;
#pragma unroll 1
  for (int kind = DRAFT; kind >= 0; --kind) {
    q = p;
    p = chance(table, a.c, kind ? lq : lp, rows[kind][mine]);
  }
  double pa = 1.0, qc = 0.0;
  const int token = d.known(a) ? (int)d.token : -1;
  uint64_t gone = 0;   // drafts that were turned down, where they were not drawn: each token once
  bool fresh = false;  // the masses of the last rejection, at `from` or in `masses`, are r's
  const double* from = nullptr;
  for (;;) {
    const uint64_t kids = __ballot(d.parent == node);
    int next = -1;
    if constexpr (DRAFT) {
      Asked asked;
      asked.run(
          kids, p, q, d.u,
          [&](int i, int r, double apa, double aqc) {
            if (r < a.rounds) {
              from = masses_of(a, r, b, node);
              return sums[i];
            }
            from = nullptr;
            __syncthreads();  // the masses of the rejection before are read
            const T *prow = row_of<T>(a.p, b, node), *qrow = row_of<T>(a.q, b, node);
            for (int c = w; c < a.chunks; c += NW) {
              const int first = (c * U * 64 + lane) * E - shift_of(prow);
              PiecePair<T> x;
              x.load(prow, qrow, first, a.V);
              const double m =
                  chunk_mass<T, U>(table, a.c, rows[0][node], rows[1][node], apa, aqc, x, prow, qrow, first, a.V);
              if (lane == 0) masses[c] = m;
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
        const double pi = lane_value(p, i), ui = lane_value(d.u, i);
        const bool again = (gone & __ballot(token == lane_value(token, i))) != 0;  // turned down before
        if (ui * Z < (again ? 0.0 : pi)) {
          next = i;
          break;
        }
        if (again) continue;
        gone |= (uint64_t)1 << i;
        Z = fmax(Z - pi, 0.0);
      }
    }
    if (next < 0) break;
    node = next;
    taken |= (uint64_t)1 << node;
  }

  // The next token: the first whose running sum of r passes u Z; where rounding leaves
  // none, the last one of the chunk that has a mass.
  const VerifyStat* st = stats_of(a, false, b, node);
  const T* prow = row_of<T>(a.p, b, node);
  const T* qrow = DRAFT && qc > 0.0 ? row_of<T>(a.q, b, node) : prow;
  const int shift = shift_of(prow);
  // (the last of a path has no drafts: its sum is not among the rows')
  const bool inner = __any(d.parent == node);
  const RowSum ps = inner ? rows[0][node] : row_sum(st, a.chunks, true, lane, 64, table, a.c);
  const RowSum qs = DRAFT && qc > 0.0 ? rows[1][node] : ps;
  const Rest<DRAFT, Weigh> rest(table, a.c, ps, qs, pa, qc);
  const int in_chunk = token >= 0 ? (token + shift) / (64 * U * E) : -1;
  // where the last event was no rejection with any left: the chunks' own masses,
  // without what was turned down
  auto own_masses = [&]() {
    __syncthreads();
    for (int c0 = 0; c0 < a.chunks; c0 += NT) {  // every lane: lanes' values are read within
      const int c = c0 + threadIdx.x;
      const VerifyStat x = st[min(c, a.chunks - 1)];
      double m = rest.ap * (x.sum * weight_below(table, a.c, x.top, ps.top));
      for (uint64_t left = gone; left; left &= left - 1) {
        const int i = __builtin_ctzll(left);
        const double there = lane_value(p, i);
        m -= lane_value(in_chunk, i) == c ? there : 0.0;
      }
      if (c < a.chunks) masses[c] = fmax(m, 0.0);
    }
    __syncthreads();
  };
  if (!(DRAFT && fresh)) {
    own_masses();
  } else if (from) {
    __syncthreads();  // a token before may have left its masses here, which a wave behind still sums
#pragma unroll 1
    for (int c = threadIdx.x; c < a.chunks; c += NT) masses[c] = from[c];
    __syncthreads();
  }
  for (;;) {
    // the chunk, by every wave: a run of them a lane
    const int run = (a.chunks + 63) / 64, c0 = lane * run, c1 = min(c0 + run, a.chunks);
    double sum = 0.0;
    for (int c = c0; c < c1; ++c) sum += masses[c];
    const double upto = wave_upto(sum), Z = lane_value(upto, 63), want = u0 * Z;
    const uint64_t some = __ballot(sum > 0.0), past = __ballot(sum > 0.0 && upto > want);
    if (!some) {
      if (gone) {  // nothing is left: the token's own distribution in its place
        gone = 0;
        own_masses();
        continue;
      }
      if (threadIdx.x == 0) a.token[b] = -1;
      break;
    }
    const int at = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
    int chunk = 0;
    double before = upto - sum, chunk_before = 0.0;
    for (int c = c0; c < c1; ++c) {
      const double m = masses[c];
      if (m > 0.0) {
        chunk = c;
        chunk_before = before;
        if (before + m > want) break;
      }
      before += m;
    }
    chunk = lane_value(chunk, at);
    chunk_before = lane_value(chunk_before, at);
    // within it: Q tokens a lane
    constexpr int CHUNK = 64 * U * E, Q = CHUNK > NT ? CHUNK / NT : 1;
    double r[Q];
    sum = 0.0;
    const int x0 = chunk * CHUNK - shift + (int)threadIdx.x * Q;
#pragma unroll
    for (int e = 0; e < Q; ++e) {
      const int x = x0 + e;
      r[e] = 0.0;
      if ((int)threadIdx.x * Q + e < CHUNK && x >= 0 && x < a.V)
        r[e] = rest(value_of(prow[x]), DRAFT ? value_of(qrow[x]) : 0.f);
    }
    if constexpr (!DRAFT) {
      for (uint64_t left = gone; left; left &= left - 1) {
        const int t = lane_value(token, __builtin_ctzll(left));
#pragma unroll
        for (int e = 0; e < Q; ++e) r[e] = t == x0 + e ? 0.0 : r[e];
      }
    }
#pragma unroll
    for (int e = 0; e < Q; ++e) sum += r[e];
    const double here = wave_upto(sum);
    if (lane == 63) part[w] = here;
    if (threadIdx.x == 0) found = INT_MAX;
    __syncthreads();
    before = chunk_before;
#pragma unroll
    for (int k = 0; k < NW; ++k) before += k < w ? part[k] : 0.0;
    const uint64_t in_past = __ballot(sum > 0.0 && before + here > want), in_some = __ballot(sum > 0.0);
    if (lane == 0) {
      last[w] = in_some ? 64 * w + 63 - __builtin_clzll(in_some) : -1;
      if (in_past) atomicMin(&found, 64 * w + __builtin_ctzll(in_past));
    }
    __syncthreads();
    int pick_lane = found;
    if (pick_lane == INT_MAX) {
      pick_lane = -1;
#pragma unroll
      for (int k = 0; k < NW; ++k) pick_lane = max(pick_lane, last[k]);
    }
    if (pick_lane < 0) {
      // rounding had left it a mass, of which there is none
      if (threadIdx.x == 0) masses[chunk] = 0.0;
      __syncthreads();
      continue;
    }
    if (pick_lane == (int)threadIdx.x) {
      before += here - sum;
      int pick = -1;
      bool done = false;
#pragma unroll
      for (int e = 0; e < Q; ++e) {
        const bool take = !done && r[e] > 0.0;
        pick = take ? x0 + e : pick;
        before += r[e];
        done = done || (take && before > want);
      }
      a.token[b] = pick;
    }
    break;
  }
  write_path();
}

namespace {
template <class T, int U>
hipError_t launch_verify_u(const VerifyArgs& a, hipStream_t s) {
  const bool draft = a.q.data != nullptr;
  const int64_t rows = (int64_t)a.B * (draft ? 2 * a.n - 1 : a.n);
  const dim3 block(256), all((unsigned)((rows * a.chunks + 3) / 4));
  if (a.best)
    MORPHO_KLAUNCH((verify_stats_kernel<T, U, true>), all, block, 0, s, a, (int)rows);
  else
    MORPHO_KLAUNCH((verify_stats_kernel<T, U, false>), all, block, 0, s, a, (int)rows);
  hipError_t e = hipGetLastError();
  const int groups = (a.chunks + kVerifyMassThreads / 64 - 1) / (kVerifyMassThreads / 64);
  const dim3 mass_block(kVerifyMassThreads);
  for (int k = 0; k < a.rounds && e == hipSuccess; ++k) {
    if (a.tree)
      MORPHO_KLAUNCH((verify_mass_kernel<T, U, false>), dim3((unsigned)((int64_t)a.B * (a.n - 1) * groups)), mass_block, 0, s,
                     a, k, groups);
    else
      MORPHO_KLAUNCH((verify_mass_kernel<T, U, true>), dim3((unsigned)((int64_t)a.B * groups)), mass_block, 0, s, a, k,
                     groups);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)a.B), threads(kVerifyThreads);
  if (a.best)
    MORPHO_KLAUNCH((verify_kernel<T, true, false, U>), grid, threads, 0, s, a);
  else if (draft)
    MORPHO_KLAUNCH((verify_kernel<T, false, true, U>), grid, threads, 0, s, a);
  else
    MORPHO_KLAUNCH((verify_kernel<T, false, false, U>), grid, threads, 0, s, a);
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
