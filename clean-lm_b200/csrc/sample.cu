// A token per row of logits, drawn by a given random number.
//
//   d_i = (z_i - max z) / T,  w_i = exp(d_i);  the entries in the order of falling logits, lowest index first among equals
//   n   = min(top_k, first m whose w sum to top_p of those of the first top_k, number of w_i >= min_p), at least 1
//   token = the first i, by index, with sum of the kept w_j, j <= i, above u times their sum;  logprob = log(w_token / sum)
//
// The result is a whole number, so sums must not depend on the order in which threads add up, and a draw next to a border must
// fall as it does in exact arithmetic: weights are f64 exponentials, rounded to multiples of 2^-S and added as 64-bit integers
// (S = 62 - log2 of the vocabulary, 50 at most, so that no sum overflows; 2^-47 of the largest weight for 32768 entries, against
// 2^-24 in f32, where one draw in a few hundred of a flat row would fall on another token).
//
// A row is one to four CTAs' work.  They read it two or three times, from L2 but for the first: for the largest logit; where top_k
// is large or top_p is on, for a histogram, which gives a bound that the kept entries reach or a window that the cut lies in; and
// for the candidates, the sums of whole tiles and, around the cut, the entries on a list in shared memory.  The rest is that list
// and one tile.  What bounds it is instructions and barriers, not memory: 148 rows of 32768 bf16 logits (1.5 us at 6.56 TB/s) take
// 4.4 us for the largest, 10.9 for top_k of 50, 13.1 for an unrestricted draw (all weights, in f64) and 28.0 for top_p of 0.9 (a
// histogram and all weights); one row in two CTAs 4.6, 10.8, 10.2 and 23.
//
// What one CTA has to search for alone is far slower (one row of 150001 f32 logits, where an ordinary top_p takes 37 us): top_p of rows
// so flat that the cut's bin, T ln 2 / 64 wide, holds more than 2048 entries (logits that spread less than about 0.17 T, 0.9 ms; of
// 262144 entries 0.4 T, 1.6 ms); a cut among thousands of equal logits (1.2 ms); top_p of a top_k that cuts something, where the bins through
// the k-th hold more than 2048 entries (top_k from about 2040 on; 1.2 ms).
#include "ops.h"
#include "ptx.cuh"

#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>

namespace cdl {
namespace sample {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int CAP = 2048;    // entries of a list
constexpr int BINS = 2048;   // of the logits below the largest, in units of T ln 2 / BIN_PER
constexpr int BIN_PER = 64;
constexpr int TILES = 1024;  // of a row, whose sums are kept
constexpr int SMALL = THREADS;  // entries of a list that are each held against all others (100 to 256, the rest sorted: no faster)
// A CTA's part of top_k up to which a bound from its threads' largest logits finds the candidates.  (Bound / histogram, us, 148
// rows of 32768: top_k of 50 11.9 / 17.0, 100 13.5 / 18.2, 300 29.4 / 30.6; of 150001: 50 29 / 51, 300 51 / 68.)
constexpr int LIST_K = 384;
// And top_k itself: the bounds of three or four CTAs at more of their threads' largest leave more than CAP entries.  (top_k of 1100 of one
// row of 150001 55 us by the bound, 59 by the histogram; of 1300 three passes more, for the list has to be made again.)
constexpr int BOUND_K = CAP / 2;

struct Params {
  const void* z;
  long long ld;
  int vocab;
  const float* u;
  const float *temperature, *top_p, *min_p;  // per row, nullable: the values below
  const int* top_k;
  float all_temperature, all_top_p, all_min_p;
  int all_top_k;
  int* token;
  float* logprob;
  int scale_bits;  // S
  int cluster;     // CTAs of a row
};

// f32 values as unsigned numbers of the same order (-0 as 0).
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
constexpr uint32_t KEY_NONE = 0x007FFFFFu;  // of -inf
// An entry as a number: larger logits first, then lower indices.
__device__ __forceinline__ u64 packed(uint32_t key, int i) {
  return (static_cast<u64>(key) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {  // of two bf16 each
  uint32_t c;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
  return c;
}

// ---- A row of logits, as the 16-byte vectors that it touches.  What a kernel runs once it fetches once: code that is not fetched
// bounds the smallest calls, so there is one copy of each pass and loops are unrolled where loads have to overlap only.
template <typename T>
struct Row {
  static constexpr int N = 16 / sizeof(T);  // logits of a vector
  const T* z;
  int vocab, vectors;
  int lead;  // logits between the 16-byte boundary and the row's first

  // A vector at the row's ends: -inf in front of it and behind it; nothing outside the row is read.
  __device__ __noinline__ static uint4 load_end(const T* z, int vocab, int i) {
    uint4 q;
    T* t = reinterpret_cast<T*>(&q);
    for (int e = 0; e < N; ++e) t[e] = i + e >= 0 && i + e < vocab ? z[i + e] : static_cast<T>(-INFINITY);
    return q;
  }
  __device__ __forceinline__ int first(int v) const { return v * N - lead; }
  // Vectors of a tile: 512 logits, or as many times that as leave at most TILES of them.
  __device__ __forceinline__ int per_tile() const {
    constexpr int BASE = 512 / N;
    return (vectors + BASE * TILES - 1) / (BASE * TILES) * BASE;
  }
  __device__ __forceinline__ uint4 load(int v) const {
    const int i = first(v);
    return i >= 0 && i <= vocab - N ? ld_nc_v4(z + i) : load_end(z, vocab, i);
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (N == 8) return __bfloat162float(z[i]);
    else return z[i];
  }
  // The largest value, NaN where there is one.
  static __device__ __forceinline__ float top(const uint4& q) {
    if constexpr (N == 8) {
      const uint32_t a = max2(max2(q.x, q.y), max2(q.z, q.w));
      return max_nan(bf16_lo(a), bf16_hi(a));
    } else {
      return max_nan(max_nan(__uint_as_float(q.x), __uint_as_float(q.y)), max_nan(__uint_as_float(q.z), __uint_as_float(q.w)));
    }
  }
  // f(vector, index of its first value) for the vectors v0, v0 + step, .. below v1: for little work, D loads and then D times f.
  template <int D, typename F>
  __device__ __forceinline__ void each(int v0, int v1, int step, F f) const {
#pragma unroll 1
    for (int v = v0; v < v1; v += D * step) {
      uint4 q[D];
#pragma unroll
      for (int i = 0; i < D; ++i)
        if (i == 0 || v + i * step < v1) q[i] = load(v + i * step);
#pragma unroll
      for (int i = 0; i < D; ++i)
        if (i == 0 || v + i * step < v1) f(q[i], first(v + i * step));
    }
  }
  // The same for more work, with the next two loads under way.
  template <typename F>
  __device__ __forceinline__ void one_by_one(int v0, int v1, int step, F f) const {
    if (v0 >= v1) return;
    uint4 next = load(v0), after = next;
    if (v0 + step < v1) after = load(v0 + step);
#pragma unroll 1
    for (int v = v0; v < v1; v += step) {
      const uint4 now = next;
      next = after;
      if (v + 2 * step < v1) after = load(v + 2 * step);
      f(now, first(v));
    }
  }
  // f(4 values, index of the first) of a vector.
  template <typename F>
  static __device__ __forceinline__ void fours(const uint4& q, int i, F f) {
    if constexpr (N == 8) {
      uint32_t a = q.x, b = q.y;
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        const float x[4] = {bf16_lo(a), bf16_hi(a), bf16_lo(b), bf16_hi(b)};
        f(x, i + 4 * h);
        a = q.z, b = q.w;
      }
    } else {
      const float x[4] = {__uint_as_float(q.x), __uint_as_float(q.y), __uint_as_float(q.z), __uint_as_float(q.w)};
      f(x, i);
    }
  }
  // The same, all of it at once.
  template <typename F>
  static __device__ __forceinline__ void fours_at_once(const uint4& q, int i, F f) {
    if constexpr (N == 8) {
      uint32_t a = q.x, b = q.y;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x[4] = {bf16_lo(a), bf16_hi(a), bf16_lo(b), bf16_hi(b)};
        f(x, i + 4 * h);
        a = q.z, b = q.w;
      }
    } else {
      const float x[4] = {__uint_as_float(q.x), __uint_as_float(q.y), __uint_as_float(q.z), __uint_as_float(q.w)};
      f(x, i);
    }
  }
};

template <typename T>
__device__ __forceinline__ Row<T> row_of(const Params& p, long long r) {
  Row<T> row;
  row.z = static_cast<const T*>(p.z) + r * p.ld;
  row.vocab = p.vocab;
  row.lead = static_cast<int>((reinterpret_cast<uintptr_t>(row.z) & 15) / sizeof(T));
  row.vectors = (p.vocab + row.lead + Row<T>::N - 1) / Row<T>::N;
  return row;
}

// floor(f n) for f of [0, 1), and whether something is left over: with f = m 2^-s and a product of 128 bits, so that the half of
// an even sum is that.
__device__ __forceinline__ u64 share_of(float f, u64 n, bool& rest) {
  const uint32_t b = __float_as_uint(f);
  const int e = static_cast<int>(b >> 23);
  const u64 m = (b & 0x7FFFFFu) | (e > 0 ? 0x800000u : 0u);
  const int s = 150 - (e > 0 ? e : 1);  // 24 to 149
  const u64 lo = m * n, hi = __umul64hi(m, n);
  u64 q, r;
  if (s < 64) {
    q = (hi << (64 - s)) | (lo >> s);
    r = lo << (64 - s);
  } else if (s < 128) {
    q = s == 64 ? hi : hi >> (s - 64);
    r = lo | (s == 64 ? 0 : hi << (128 - s));
  } else {
    q = 0;
    r = lo | hi;
  }
  rest = r != 0;
  return q;
}
// The least whole sum that top_p of `mass` asks for.
__device__ __forceinline__ u64 least_of(float top_p, u64 mass) {
  bool rest;
  const u64 q = share_of(fmaxf(top_p, 0.f), mass, rest) + rest;
  return q < 1 ? 1 : q;
}

// 2^(j/256), rounded to f64.
__device__ const double POW2[256] = {
    0x1.0000000000000p+0, 0x1.00b1afa5abcbfp+0, 0x1.0163da9fb3335p+0, 0x1.02168143b0281p+0,
    0x1.02c9a3e778061p+0, 0x1.037d42e11bbccp+0, 0x1.04315e86e7f85p+0, 0x1.04e5f72f654b1p+0,
    0x1.059b0d3158574p+0, 0x1.0650a0e3c1f89p+0, 0x1.0706b29ddf6dep+0, 0x1.07bd42b72a836p+0,
    0x1.0874518759bc8p+0, 0x1.092bdf66607e0p+0, 0x1.09e3ecac6f383p+0, 0x1.0a9c79b1f3919p+0,
    0x1.0b5586cf9890fp+0, 0x1.0c0f145e46c85p+0, 0x1.0cc922b7247f7p+0, 0x1.0d83b23395decp+0,
    0x1.0e3ec32d3d1a2p+0, 0x1.0efa55fdfa9c5p+0, 0x1.0fb66affed31bp+0, 0x1.1073028d7233ep+0,
    0x1.11301d0125b51p+0, 0x1.11edbab5e2ab6p+0, 0x1.12abdc06c31ccp+0, 0x1.136a814f204abp+0,
    0x1.1429aaea92de0p+0, 0x1.14e95934f312ep+0, 0x1.15a98c8a58e51p+0, 0x1.166a45471c3c2p+0,
    0x1.172b83c7d517bp+0, 0x1.17ed48695bbc0p+0, 0x1.18af9388c8deap+0, 0x1.1972658375d2fp+0,
    0x1.1a35beb6fcb75p+0, 0x1.1af99f8138a1cp+0, 0x1.1bbe084045cd4p+0, 0x1.1c82f95281c6bp+0,
    0x1.1d4873168b9aap+0, 0x1.1e0e75eb44027p+0, 0x1.1ed5022fcd91dp+0, 0x1.1f9c18438ce4dp+0,
    0x1.2063b88628cd6p+0, 0x1.212be3578a819p+0, 0x1.21f49917ddc96p+0, 0x1.22bdda27912d1p+0,
    0x1.2387a6e756238p+0, 0x1.2451ffb82140ap+0, 0x1.251ce4fb2a63fp+0, 0x1.25e85711ece75p+0,
    0x1.26b4565e27cddp+0, 0x1.2780e341ddf29p+0, 0x1.284dfe1f56381p+0, 0x1.291ba7591bb70p+0,
    0x1.29e9df51fdee1p+0, 0x1.2ab8a66d10f13p+0, 0x1.2b87fd0dad990p+0, 0x1.2c57e39771b2fp+0,
    0x1.2d285a6e4030bp+0, 0x1.2df961f641589p+0, 0x1.2ecafa93e2f56p+0, 0x1.2f9d24abd886bp+0,
    0x1.306fe0a31b715p+0, 0x1.31432edeeb2fdp+0, 0x1.32170fc4cd831p+0, 0x1.32eb83ba8ea32p+0,
    0x1.33c08b26416ffp+0, 0x1.3496266e3fa2dp+0, 0x1.356c55f929ff1p+0, 0x1.36431a2de883bp+0,
    0x1.371a7373aa9cbp+0, 0x1.37f26231e754ap+0, 0x1.38cae6d05d866p+0, 0x1.39a401b7140efp+0,
    0x1.3a7db34e59ff7p+0, 0x1.3b57fbfec6cf4p+0, 0x1.3c32dc313a8e5p+0, 0x1.3d0e544ede173p+0,
    0x1.3dea64c123422p+0, 0x1.3ec70df1c5175p+0, 0x1.3fa4504ac801cp+0, 0x1.40822c367a024p+0,
    0x1.4160a21f72e2ap+0, 0x1.423fb2709468ap+0, 0x1.431f5d950a897p+0, 0x1.43ffa3f84b9d4p+0,
    0x1.44e086061892dp+0, 0x1.45c2042a7d232p+0, 0x1.46a41ed1d0057p+0, 0x1.4786d668b3237p+0,
    0x1.486a2b5c13cd0p+0, 0x1.494e1e192aed2p+0, 0x1.4a32af0d7d3dep+0, 0x1.4b17dea6db7d7p+0,
    0x1.4bfdad5362a27p+0, 0x1.4ce41b817c114p+0, 0x1.4dcb299fddd0dp+0, 0x1.4eb2d81d8abffp+0,
    0x1.4f9b2769d2ca7p+0, 0x1.508417f4531eep+0, 0x1.516daa2cf6642p+0, 0x1.5257de83f4eefp+0,
    0x1.5342b569d4f82p+0, 0x1.542e2f4f6ad27p+0, 0x1.551a4ca5d920fp+0, 0x1.56070dde910d2p+0,
    0x1.56f4736b527dap+0, 0x1.57e27dbe2c4cfp+0, 0x1.58d12d497c7fdp+0, 0x1.59c0827ff07ccp+0,
    0x1.5ab07dd485429p+0, 0x1.5ba11fba87a03p+0, 0x1.5c9268a5946b7p+0, 0x1.5d84590998b93p+0,
    0x1.5e76f15ad2148p+0, 0x1.5f6a320dceb71p+0, 0x1.605e1b976dc09p+0, 0x1.6152ae6cdf6f4p+0,
    0x1.6247eb03a5585p+0, 0x1.633dd1d1929fdp+0, 0x1.6434634ccc320p+0, 0x1.652b9febc8fb7p+0,
    0x1.6623882552225p+0, 0x1.671c1c70833f6p+0, 0x1.68155d44ca973p+0, 0x1.690f4b19e9538p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6b052fa75173ep+0, 0x1.6c012750bdabfp+0, 0x1.6cfdcddd47645p+0,
    0x1.6dfb23c651a2fp+0, 0x1.6ef9298593ae5p+0, 0x1.6ff7df9519484p+0, 0x1.70f7466f42e87p+0,
    0x1.71f75e8ec5f74p+0, 0x1.72f8286ead08ap+0, 0x1.73f9a48a58174p+0, 0x1.74fbd35d7cbfdp+0,
    0x1.75feb564267c9p+0, 0x1.77024b1ab6e09p+0, 0x1.780694fde5d3fp+0, 0x1.790b938ac1cf6p+0,
    0x1.7a11473eb0187p+0, 0x1.7b17b0976cfdbp+0, 0x1.7c1ed0130c132p+0, 0x1.7d26a62ff86f0p+0,
    0x1.7e2f336cf4e62p+0, 0x1.7f3878491c491p+0, 0x1.80427543e1a12p+0, 0x1.814d2add106d9p+0,
    0x1.82589994cce13p+0, 0x1.8364c1eb941f7p+0, 0x1.8471a4623c7adp+0, 0x1.857f4179f5b21p+0,
    0x1.868d99b4492edp+0, 0x1.879cad931a436p+0, 0x1.88ac7d98a6699p+0, 0x1.89bd0a478580fp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8be05bad61778p+0, 0x1.8cf3216b5448cp+0, 0x1.8e06a5e0866d9p+0,
    0x1.8f1ae99157736p+0, 0x1.902fed0282c8ap+0, 0x1.9145b0b91ffc6p+0, 0x1.925c353aa2fe2p+0,
    0x1.93737b0cdc5e5p+0, 0x1.948b82b5f98e5p+0, 0x1.95a44cbc8520fp+0, 0x1.96bdd9a7670b3p+0,
    0x1.97d829fde4e50p+0, 0x1.98f33e47a22a2p+0, 0x1.9a0f170ca07bap+0, 0x1.9b2bb4d53fe0dp+0,
    0x1.9c49182a3f090p+0, 0x1.9d674194bb8d5p+0, 0x1.9e86319e32323p+0, 0x1.9fa5e8d07f29ep+0,
    0x1.a0c667b5de565p+0, 0x1.a1e7aed8eb8bbp+0, 0x1.a309bec4a2d33p+0, 0x1.a42c980460ad8p+0,
    0x1.a5503b23e255dp+0, 0x1.a674a8af46052p+0, 0x1.a799e1330b358p+0, 0x1.a8bfe53c12e59p+0,
    0x1.a9e6b5579fdbfp+0, 0x1.ab0e521356ebap+0, 0x1.ac36bbfd3f37ap+0, 0x1.ad5ff3a3c2774p+0,
    0x1.ae89f995ad3adp+0, 0x1.afb4ce622f2ffp+0, 0x1.b0e07298db666p+0, 0x1.b20ce6c9a8952p+0,
    0x1.b33a2b84f15fbp+0, 0x1.b468415b749b1p+0, 0x1.b59728de5593ap+0, 0x1.b6c6e29f1c52ap+0,
    0x1.b7f76f2fb5e47p+0, 0x1.b928cf22749e4p+0, 0x1.ba5b030a1064ap+0, 0x1.bb8e0b79a6f1fp+0,
    0x1.bcc1e904bc1d2p+0, 0x1.bdf69c3f3a207p+0, 0x1.bf2c25bd71e09p+0, 0x1.c06286141b33dp+0,
    0x1.c199bdd85529cp+0, 0x1.c2d1cd9fa652cp+0, 0x1.c40ab5fffd07ap+0, 0x1.c544778fafb22p+0,
    0x1.c67f12e57d14bp+0, 0x1.c7ba88988c933p+0, 0x1.c8f6d9406e7b5p+0, 0x1.ca3405751c4dbp+0,
    0x1.cb720dcef9069p+0, 0x1.ccb0f2e6d1675p+0, 0x1.cdf0b555dc3fap+0, 0x1.cf3155b5bab74p+0,
    0x1.d072d4a07897cp+0, 0x1.d1b532b08c968p+0, 0x1.d2f87080d89f2p+0, 0x1.d43c8eacaa1d6p+0,
    0x1.d5818dcfba487p+0, 0x1.d6c76e862e6d3p+0, 0x1.d80e316c98398p+0, 0x1.d955d71ff6075p+0,
    0x1.da9e603db3285p+0, 0x1.dbe7cd63a8315p+0, 0x1.dd321f301b460p+0, 0x1.de7d5641c0658p+0,
    0x1.dfc97337b9b5fp+0, 0x1.e11676b197d17p+0, 0x1.e264614f5a129p+0, 0x1.e3b333b16ee12p+0,
    0x1.e502ee78b3ff6p+0, 0x1.e653924676d76p+0, 0x1.e7a51fbc74c83p+0, 0x1.e8f7977cdb740p+0,
    0x1.ea4afa2a490dap+0, 0x1.eb9f4867cca6ep+0, 0x1.ecf482d8e67f1p+0, 0x1.ee4aaa2188510p+0,
    0x1.efa1bee615a27p+0, 0x1.f0f9c1cb6412ap+0, 0x1.f252b376bba97p+0, 0x1.f3ac948dd7274p+0,
    0x1.f50765b6e4540p+0, 0x1.f6632798844f8p+0, 0x1.f7bfdad9cbe14p+0, 0x1.f91d802243c89p+0,
    0x1.fa7c1819e90d8p+0, 0x1.fbdba3692d514p+0, 0x1.fd3c22b8f71f1p+0, 0x1.fe9d96b2a23d9p+0};

// w = exp((z - top) / T) in units of 2^-S: 2^((k + r) / 256) with (z - top) 256 log2(e) / T = k + r, |r| <= 1/2, from a table of
// 2^(S + j/256) and the Taylor series up to r^4, whose rest is 4e-17 (the table-driven method of P. T. P. Tang, 1989).  S <= 50: the
// addition of 1.5 2^52 rounds to whole units.  Constants are members so that they stay in registers: as literals they took two
// moves each, and the pass over a row is bound by the number of its instructions.
struct Weight {
  double top, per_t;          // 256 log2(e) / T
  double c1, c2, c3, c4;      // (ln 2 / 256)^i / i!
  double magic;               // 1.5 2^52
  float least;                // 80 T ln 2 below the top, where w is less than half a unit
  uint32_t pow2;              // the table in shared memory
  // (without meaning for z <= least)
  __device__ __forceinline__ u64 above_least(float z) const {
    const double d = static_cast<double>(z) - top;
    const double k = fma(d, per_t, magic);
    const int n = __double2loint(k);
    const double r = fma(d, per_t, magic - k);
    double y = fma(r, c4, c3);
    y = fma(r, y, c2);
    y = fma(r, y, c1) * r;
    double tab;
    asm("ld.shared.f64 %0, [%1];" : "=d"(tab) : "r"(pow2 + (n & 255) * 8));
    y = fma(tab, y, tab);
    y = __hiloint2double(__double2hiint(y) + ((n << 12) & static_cast<int>(0xFFF00000u)), __double2loint(y)) + magic;
    return static_cast<u64>(__double_as_longlong(y)) & 0x7FFFFFFFFFFFFull;
  }
  __device__ __forceinline__ u64 operator()(float z) const {
    const u64 w = above_least(z);
    return z > least ? w : 0;
  }
};
__device__ __forceinline__ void add_if_from(u64& sum, u64 y, float x, float from) {  // sum += y where x >= from
  asm("{\n\t.reg .pred p;\n\tsetp.ge.f32 p, %2, %3;\n\t@p add.u64 %0, %0, %1;\n\t}" : "+l"(sum) : "l"(y), "f"(x), "f"(from));
}

struct Shared {
  u64 list[CAP], weight_of[CAP];
  union {
    u64 other[CAP];
    uint32_t hist[BINS];
    uint32_t fine[3][THREADS];
  };
  u64 tile[TILES];  // a CTA's tiles at their number in the row
  double pow2[256];
  u64 sums[WARPS];
  float tops[WARPS];
  uint32_t rank_of[256];
  Weight weight;
  // what the cluster's other CTAs read
  float top;
  int at;
  uint32_t count, bound;
  int again;  // (written by the first)
  uint32_t key_min;
  u64 above, all;
  int mode, lo, hi;
  uint32_t before;
  int edge[6];
  uint32_t ahead_of[6], least_of[2];
  // what a CTA's threads tell one another
  u64 word;
  int index;
};

__device__ __forceinline__ u64 warp_sum(u64 x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
struct Sums {
  u64 before, all;
};
// Sum over the threads ahead of this one, and over all of them.  Ends in a barrier.
__device__ __noinline__ Sums block_scan(u64 x, u64* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 y = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) y += o;
  }
  if (lane == 31) sums[warp] = y;
  __syncthreads();
  u64 z = sums[lane & (WARPS - 1)];
#pragma unroll
  for (int d = 1; d < WARPS; d <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, z, d);
    if ((lane & (WARPS - 1)) >= d) z += o;
  }
  const u64 ahead = __shfl_sync(0xffffffffu, z, warp > 0 ? warp - 1 : 0);
  Sums r{y - x + (warp > 0 ? ahead : 0), __shfl_sync(0xffffffffu, z, WARPS - 1)};
  __syncthreads();
  return r;
}

// a[0, n) in falling order, n <= CAP, all different; returns where it is, a or b.  Ends in a barrier.
__device__ __noinline__ u64* sort_down(uint32_t* rank_of, u64* a, u64* b, int n) {
  const int tid = threadIdx.x;
  if (n <= 256) {  // every entry counts those above it
    int p = 32;
    while (p < n) p <<= 1;
    if (tid < 256) rank_of[tid] = 0;
    __syncthreads();
    const int i = tid & (p - 1), part = tid / p, parts = THREADS / p;
    if (i < n) {
      const u64 x = a[i];
      uint32_t r = 0;
#pragma unroll 2
      for (int j = part; j < n; j += parts) r += a[j] > x;
      atomicAdd(&rank_of[i], r);
    }
    __syncthreads();
    if (tid < n) b[rank_of[tid]] = a[tid];
    __syncthreads();
    return b;
  }
  int p = 512;
  while (p < n) p <<= 1;
  for (int i = n + tid; i < p; i += THREADS) a[i] = 0;
#pragma unroll 1
  for (int k = 2; k <= p; k <<= 1)
#pragma unroll 1
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
#pragma unroll 1
      for (int t = tid; t < p / 2; t += THREADS) {
        const int i = 2 * t - (t & (j - 1));  // the pairs i, i + j
        const u64 x = a[i], y = a[i + j];
        if ((x < y) == ((i & k) == 0)) a[i] = y, a[i + j] = x;
      }
    }
  __syncthreads();
  return a;
}

__device__ __forceinline__ uint32_t key_in(u64 entry) { return static_cast<uint32_t>(entry >> 32); }
__device__ __forceinline__ int index_in(u64 entry) { return static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(entry)); }

// The settings of a row.
struct Settings {
  int k;  // 0: all
  float top_p, u;
  uint32_t key_min;  // of min_p; entries below it are not kept
  double t;
};
// How many units of `mass` lie in front of the draw.
__device__ __forceinline__ u64 drawn(float u, u64 mass) {
  bool rest;
  return u > 0.f ? (u < 1.f ? share_of(u, mass, rest) : mass - 1) : 0;
}
__device__ __noinline__ void write_out(const Params& p, const Shared& sh, long long r, double t, int i, float x, u64 mass) {
  p.token[r] = i;
  if (p.logprob)
    p.logprob[r] = static_cast<float>((static_cast<double>(x) - sh.weight.top) / t - log(ldexp(static_cast<double>(mass), -p.scale_bits)));
}

// The draw from a list of more than SMALL entries that holds all that may be kept.
__device__ __noinline__ void draw_sorted(const Params& p, Shared& sh, const Settings& set, long long r, int n) {
  const int tid = threadIdx.x;
  const u64* order = sort_down(sh.rank_of, sh.list, sh.other, n);
  u64* spare = order == sh.list ? sh.other : sh.list;
  const int per = (n + THREADS - 1) / THREADS;  // neighbouring entries of a thread
  const int first = min(n, tid * per), last = min(n, first + per);
  u64 sum = 0;
  for (int i = first; i < last; ++i) sum += sh.weight(of_key(key_in(order[i])));
  u64 upto = block_scan(sum, sh.sums).before;
  for (int i = first; i < last; ++i) {
    upto += sh.weight(of_key(key_in(order[i])));
    spare[i] = upto;
  }
  __syncthreads();
  const int n_k = set.k > 0 && set.k < n ? set.k : n;
  const u64 want_p = set.top_p < 1.f ? least_of(set.top_p, spare[n_k - 1]) : ~0ull;
  u64 keeps = 0;
  for (int i = first; i < min(n_k, last); ++i) keeps += (i == 0 || spare[i - 1] < want_p) && key_in(order[i]) >= set.key_min;
  const int kept = max(1, static_cast<int>(block_scan(keeps, sh.sums).all));
  const u64 mass = spare[kept - 1], want = drawn(set.u, mass);
  __syncthreads();
  // by index
  for (int i = tid; i < kept; i += THREADS) spare[i] = (order[i] << 32) | (order[i] >> 32);
  __syncthreads();
  const u64* line = sort_down(sh.rank_of, spare, const_cast<u64*>(order), kept);
  sum = 0;
  for (int i = first; i < min(kept, last); ++i) sum += sh.weight(of_key(static_cast<uint32_t>(line[i])));
  u64 ahead = block_scan(sum, sh.sums).before;
  for (int i = first; i < min(kept, last); ++i) {
    const float x = of_key(static_cast<uint32_t>(line[i]));
    const u64 w = sh.weight(x);
    if (ahead <= want && want < ahead + w) write_out(p, sh, r, set.t, index_in(line[i] >> 32), x, mass);
    ahead += w;
  }
}

// The draw from up to SMALL entries: each is held against all others, by 32 threads at most, for its place in falling order and
// then, of those that are kept, for what is ahead of it by index.
__device__ __forceinline__ void draw_small(const Params& p, Shared& sh, const Settings& set, long long r, int n) {
  const int tid = threadIdx.x;
  int parts = 32;
  while (parts * n > THREADS) parts >>= 1;
  int i = tid / parts;
  const int part = tid & (parts - 1);
  {
    const u64 me = i < n ? sh.list[i] : 0;
    uint32_t rank = 0;
    if (i < n)
#pragma unroll 4
      for (int j = part; j < n; j += parts) rank += sh.list[j] > me;
    for (int d = 1; d < parts; d <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, d);
    if (i < n && part == 0) sh.other[rank] = me;
  }
  __syncthreads();
  if (set.k > 0 && set.k < n) n = set.k;
  const u64 entry = tid < n ? sh.other[tid] : 0;
  u64 w = tid < n ? sh.weight(of_key(key_in(entry))) : 0;
  const Sums s = block_scan(w, sh.sums);
  const bool kept = tid < n && (tid == 0 || (key_in(entry) >= set.key_min && (!(set.top_p < 1.f) || s.before < least_of(set.top_p, s.all))));
  if (kept) sh.list[tid] = w;
  n = __syncthreads_count(kept);
  if (tid == n - 1) sh.word = s.before + w;
  __syncthreads();
  const u64 mass = sh.word, want = drawn(set.u, mass);
  parts = 32;
  while (parts * n > THREADS) parts >>= 1;
  i = tid / parts;
  u64 ahead = 0;
  const int at = tid & (parts - 1);
  const u64 me = i < n ? sh.other[i] : 0;
  if (i < n)
#pragma unroll 2
    for (int j = at; j < n; j += parts)
      if (static_cast<uint32_t>(sh.other[j]) > static_cast<uint32_t>(me)) ahead += sh.list[j];
  for (int d = 1; d < parts; d <<= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, d);
  if (i < n && at == 0 && ahead <= want && want < ahead + sh.list[i])
    write_out(p, sh, r, set.t, index_in(me), of_key(key_in(me)), mass);
}

// The entry at which the sum over the entries from `cut` on, in falling order, reaches `want`: of their weights, or their number.
// A quarter of the range of logits at a time, then by index.  For windows that hold more than CAP entries: equal logits by the
// thousand, logits far from any scale that the bins have, top_p of a top_k of thousands.
template <typename T>
__device__ __noinline__ u64 select(const Row<T>& row_in, Shared& sh, bool weights, u64 want, u64 cut) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Row<T> row = row_in;
  const Weight weight = sh.weight;
  uint32_t lo = KEY_NONE + 1, hi = key_of(static_cast<float>(weight.top));  // the entry's key is among these
  u64 above = 0;                                                            // sum of the keys above hi
#pragma unroll 1
  while (lo < hi) {
    const uint32_t part = (hi - lo) / 4 + 1;
    const uint32_t p1 = lo + part, p2 = min(hi, p1 + part), p3 = min(hi, p2 + part);
    u64 s1 = 0, s2 = 0, s3 = 0;  // from p1, p2, p3 on
    row.template each<2>(tid, row.vectors, THREADS, [&](const uint4& q, int i0) {
      Row<T>::fours(q, i0, [&](const float (&x)[4], int i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t key = key_of(x[e]);
          if (key < p1 || key > hi || packed(key, i + e) < cut) continue;
          const u64 y = weights ? weight(x[e]) : 1;
          s1 += y;
          if (key >= p2) s2 += y;
          if (key >= p3) s3 += y;
        }
      });
    });
    s1 = above + block_scan(s1, sh.sums).all;
    s2 = above + block_scan(s2, sh.sums).all;
    s3 = above + block_scan(s3, sh.sums).all;
    if (s3 >= want) lo = p3;
    else if (s2 >= want) lo = p2, hi = p3 - 1, above = s3;
    else if (s1 >= want) lo = p1, hi = p2 - 1, above = s2;
    else hi = p1 - 1, above = s1;
  }
  const uint32_t prefix = lo;
  // how many of the entries equal to it, the lowest indices first
  const u64 one = weights ? weight(of_key(prefix)) : 1;
  const u64 ties = one == 0 ? 1 : (want - above + one - 1) / one;
  const int seg = static_cast<int>((static_cast<long long>(row.vocab) + THREADS * WARPS - 1) / (THREADS * WARPS) * THREADS);
  const int i0 = static_cast<int>(min(static_cast<long long>(row.vocab), static_cast<long long>(warp) * seg));
  const int i1 = static_cast<int>(min(static_cast<long long>(row.vocab), static_cast<long long>(i0) + seg));
  auto is = [&](int i) {
    const uint32_t key = key_of(row.at(i));
    return key == prefix && packed(key, i) >= cut;
  };
  u64 n = 0;
  for (int i = i0 + lane; i < i1; i += 32) n += is(i);
  u64 before = __shfl_sync(0xffffffffu, block_scan(n, sh.sums).before, 0);
  n = warp_sum(n);
  if (tid == 0) sh.word = packed(prefix, -1);  // all of them
  __syncthreads();
  if (before < ties && before + n >= ties) {
    for (int i = i0; i < i1; i += 32) {
      const bool hit = i + lane < i1 && is(i + lane);
      const unsigned mask = __ballot_sync(0xffffffffu, hit);
      if (before + __popc(mask) >= ties) {
        if (hit && before + __popc(mask & ((2u << lane) - 1)) == ties) sh.word = packed(prefix, i + lane);
        break;
      }
      before += __popc(mask);
    }
  }
  __syncthreads();
  const u64 at = sh.word;
  __syncthreads();
  return at;
}
// Sums of all tiles, of the entries from `cut` on without those below key_min.
template <typename T>
__device__ __noinline__ void sum_tiles(const Row<T>& row, Shared& sh, int per_tile, int tiles, u64 cut, uint32_t key_min) {
  const int lane = threadIdx.x & 31;
  const Weight weight = sh.weight;
  const uint32_t least = max(key_min, KEY_NONE + 1);
  for (int tile = threadIdx.x >> 5; tile < tiles; tile += WARPS) {
    const int i0 = max(0, row.first(tile * per_tile)), i1 = min(row.vocab, row.first(min(row.vectors, (tile + 1) * per_tile)));
    u64 sum = 0;
    for (int i = i0 + lane; i < i1; i += 32) {
      const float x = row.at(i);
      const uint32_t key = key_of(x);
      if (key >= least && packed(key, i) >= cut) sum += weight(x);
    }
    sum = warp_sum(sum);
    if (lane == 0) sh.tile[tile] = sum;
  }
  __syncthreads();
}
// The cut of a row and its tiles' sums by one CTA alone, whatever the row is like.
template <typename T>
__device__ __noinline__ u64 slow_cut(const Row<T>& row, Shared& sh, const Settings& set, int per_tile, int tiles) {
  u64 cut = 0;
  __syncthreads();
  if (set.k > 0) cut = select(row, sh, false, static_cast<u64>(set.k), 0);
  if (set.top_p < 1.f) {
    sum_tiles(row, sh, per_tile, tiles, cut, 0);
    u64 sum = 0;
    for (int i = threadIdx.x; i < tiles; i += THREADS) sum += sh.tile[i];
    cut = select(row, sh, true, least_of(set.top_p, block_scan(sum, sh.sums).all), cut);
  }
  sum_tiles(row, sh, per_tile, tiles, cut, set.key_min);
  return cut;
}

// The draw where a bound of the threads' largest logits left more than CAP entries: a part of the row lies far below the others
// (masked, or the row is in order), so that its CTA's bound does.  All CTAs of the row find the k-th entry from counts of 11 bits at a
// time, of its key and, where more than CAP are alike, of its index; the list is made again of the entries from there on.  (Half of
// 150001 logits masked, top_k of 50, one row: 43 us, 16 with nothing masked; one CTA searching alone 534.)  It takes all that it needs
// from the parameters, so that the kernel has to keep nothing for it.
template <typename T>
__device__ __noinline__ void draw_again(const Params& p, Shared& sh) {
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, C = p.cluster, rank = static_cast<int>(blockIdx.x % C);
  const long long r = blockIdx.x / C;
  const Row<T> row = row_of<T>(p, r);
  const int per_tile = row.per_tile(), tiles = (row.vectors + per_tile - 1) / per_tile, share = (tiles + C - 1) / C;
  const int v0 = min(row.vectors, min(tiles, rank * share) * per_tile), v1 = min(row.vectors, min(tiles, (rank + 1) * share) * per_tile);
  auto meet = [&]() {
    if (C > 1) cluster.sync();
    else __syncthreads();
  };
  auto of = [&](int other) -> Shared& { return C > 1 ? *cluster.map_shared_rank(&sh, other) : sh; };
  Settings set;
  set.k = p.top_k ? p.top_k[r] : p.all_top_k;
  set.top_p = p.top_p ? p.top_p[r] : p.all_top_p;
  set.u = p.u[r];
  set.key_min = sh.key_min;
  set.t = static_cast<double>(p.temperature ? p.temperature[r] : p.all_temperature);
  const uint32_t k = static_cast<uint32_t>(set.k);
  u64 bound = 0;       // the bits found so far
  uint32_t above = 0;  // the entries above those that have them
  __syncthreads();     // (the list's length was read by all)
#pragma unroll 1
  for (int level = 0; level < 5; ++level) {  // (not an index's last 10 bits: 1024 entries and fewer than BOUND_K above them fit the list)
    static_assert(BOUND_K + 1024 <= CAP, "");
    const int width = level == 2 ? 10 : 11, shift = level == 0 ? 53 : level == 1 ? 42 : level == 2 ? 32 : level == 3 ? 21 : 10;
    const uint32_t mask = (1u << width) - 1;
    for (int i = tid; i < BINS; i += THREADS) sh.hist[i] = 0;
    if (tid == 0) sh.lo = -1, sh.count = 0;
    __syncthreads();
    row.template each<4>(v0 + tid, v1, THREADS, [&](const uint4& q, int i) {
      Row<T>::fours(q, i, [&](const float (&x)[4], int j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t key = key_of(x[e]);
          const u64 entry = packed(key, j + e);
          if (key > KEY_NONE && (level == 0 || (entry ^ bound) >> (shift + width) == 0))
            atomicAdd(&sh.hist[mask - (static_cast<uint32_t>(entry >> shift) & mask)], 1u);
        }
      });
    });
    meet();
    constexpr int PER = BINS / THREADS;
    static_assert(PER == 4, "");
    uint4 bins = make_uint4(0, 0, 0, 0);  // the largest entries first
    for (int c = 0; c < C; ++c) {
      const uint4 o = reinterpret_cast<const uint4*>(of(c).hist)[tid];
      bins.x += o.x, bins.y += o.y, bins.z += o.z, bins.w += o.w;
    }
    const uint32_t count[PER] = {bins.x, bins.y, bins.z, bins.w};
    uint32_t upto = above + static_cast<uint32_t>(block_scan(static_cast<u64>(bins.x) + bins.y + bins.z + bins.w, sh.sums).before);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (upto < k && upto + count[j] >= k) sh.lo = tid * PER + j, sh.ahead_of[0] = upto, sh.ahead_of[1] = upto + count[j];
      upto += count[j];
    }
    meet();
    const int at = sh.lo;
    above = sh.ahead_of[0];
    const uint32_t through = sh.ahead_of[1];
    __syncthreads();  // (read by all before it is written again)
    if (at < 0) break;  // fewer than k entries are not masked: all of them
    bound |= static_cast<u64>(mask - at) << shift;
    if (through <= CAP) break;
  }
  row.template each<4>(v0 + tid, v1, THREADS, [&](const uint4& q, int i) {
    Row<T>::fours(q, i, [&](const float (&x)[4], int j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t key = key_of(x[e]);
        const u64 entry = packed(key, j + e);
        if (key > KEY_NONE && entry >= bound) {
          const uint32_t at = atomicAdd(&sh.count, 1u);
          if (at < CAP) sh.list[at] = entry;
        }
      }
    });
  });
  meet();
  int n = static_cast<int>(sh.count);  // (up to CAP in all)
  if (C > 1) {
    for (int c = 1; rank == 0 && c < C; ++c) {
      const Shared& o = of(c);
      const int m = static_cast<int>(o.count);
      for (int i = tid; i < m && n + i < CAP; i += THREADS) sh.list[n + i] = o.list[i];
      n += m;
    }
    cluster.sync();  // (nobody's shared memory goes while it is read)
    if (rank != 0) return;
  }
  __syncthreads();
  draw_sorted(p, sh, set, r, min(n, CAP));
}

// What the pass over the row's weights has to find.
enum Mode {
  ALL,       // everything (but what min_p leaves out) is kept
  WINDOW_P,  // the cut of top_p lies in a window of bins
  WINDOW_K,  // that of top_k
  LIST,      // what may be kept fits on the list
  SLOW       // one CTA alone searches
};

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int C = p.cluster, rank = static_cast<int>(blockIdx.x % C);
  auto meet = [&]() {
    if (C > 1) cluster.sync();
    else __syncthreads();
  };
  auto of = [&](int other) -> Shared& { return C > 1 ? *cluster.map_shared_rank(&sh, other) : sh; };
  if (tid < 256) sh.pow2[tid] = __hiloint2double(__double2hiint(POW2[tid]) + (p.scale_bits << 20), __double2loint(POW2[tid]));
  if (tid == 0) sh.count = 0, sh.again = 0;
  const long long r = blockIdx.x / C;
  const Row<T> row = row_of<T>(p, r);
  constexpr int N = Row<T>::N;
  const int per_tile = row.per_tile();
  const int tiles = (row.vectors + per_tile - 1) / per_tile;
  const int share = (tiles + C - 1) / C;  // tiles of a CTA
  const int t0 = min(tiles, rank * share), t1 = min(tiles, t0 + share);
  const int v0 = min(row.vectors, t0 * per_tile), v1 = min(row.vectors, t1 * per_tile);
  grid_dep_wait();
  grid_dep_launch();

  // ---- the largest logit; NaN and +inf
  float mine = -INFINITY;
  row.template each<8>(v0 + tid, v1, THREADS, [&](const uint4& q, int) { mine = max_nan(mine, Row<T>::top(q)); });
  const float temperature = p.temperature ? p.temperature[r] : p.all_temperature;
  const float min_p = p.min_p ? p.min_p[r] : p.all_min_p;
  Settings set;
  set.k = p.top_k ? p.top_k[r] : p.all_top_k;
  set.top_p = p.top_p ? p.top_p[r] : p.all_top_p;
  set.u = p.u[r];
  if (set.k < 0 || set.k >= p.vocab) set.k = 0;
  const bool p_on = set.top_p < 1.f;
  float top = mine;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (lane == 0) sh.tops[warp] = top;
  __syncthreads();
  top = sh.tops[lane & (WARPS - 1)];
#pragma unroll
  for (int d = WARPS / 2; d > 0; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (C > 1) {
    if (tid == 0) sh.top = top;
    cluster.sync();
    for (int c = 0; c < C; ++c) top = max_nan(top, of(c).top);
  }
  if (!(top < INFINITY) || top == -INFINITY || !(temperature > 0.f)) {
    const bool bad = !(top < INFINITY) || top == -INFINITY;
    if (tid == 0) sh.at = INT32_MAX;
    __syncthreads();
    if (!bad)  // the first place of the largest
      row.template each<2>(v0 + tid, v1, THREADS, [&](const uint4& q, int i) {
        if (Row<T>::top(q) != top) return;
        Row<T>::fours(q, i, [&](const float (&x)[4], int j) {
          const int e = x[0] == top ? 0 : x[1] == top ? 1 : x[2] == top ? 2 : x[3] == top ? 3 : 4;
          if (e < 4) atomicMin(&sh.at, j + e);
        });
      });
    meet();
    if (rank == 0 && tid == 0) {
      int at = sh.at;
      for (int c = 1; c < C; ++c) at = min(at, of(c).at);
      p.token[r] = bad ? -1 : at;
      if (p.logprob) p.logprob[r] = bad ? __uint_as_float(0x7FC00000u) : 0.f;
    }
    if (C > 1) cluster.sync();
    return;
  }
  set.t = static_cast<double>(temperature);
  constexpr double L = 0.6931471805599453094 / 256;
  const double per_t = 256 * 1.4426950408889634074 / set.t;
  if (tid == 0)
    sh.weight = Weight{static_cast<double>(top), per_t, L, L * L / 2, L * L * L / 6, L * L * L * L / 24, 6755399441055744.0,
                       fminf(__double2float_rd(static_cast<double>(top) - 80 * 0.6931471805599453 * set.t), of_key(key_of(top) - 1)),
                       smem_u32(sh.pow2)};
  // w >= min_p: a bound on the logit, rounded up to the next one in f32
  set.key_min = 0;
  if (min_p > 0.f) {
    const double far = set.t * log(static_cast<double>(fminf(min_p, 1.f)));  // (NaN: of an infinite temperature, where all w are 1)
    set.key_min = isnan(far) ? 0 : min(key_of(top), key_of(__double2float_ru(static_cast<double>(top) + far)));
  }
  if (tid == 0) sh.key_min = set.key_min;

  auto append = [&](uint32_t key, int i) {
    const uint32_t at = atomicAdd(&sh.count, 1u);
    if (at < CAP) sh.list[at] = packed(key, i);
  };
  Mode mode = ALL;
  const float bin_scale = fmaxf(1e-36f, fminf(static_cast<float>(per_t) * (BIN_PER / 256.f), 1e30f));
  // How far a logit lies below the largest; rounded by the addition of 1.5 2^23, infinite distances in the last bin.
  auto bin = [&](float x) { return min(BINS - 1, __float_as_int(fmaf(top - x, bin_scale, 12582912.f)) - 0x4B400000); };
  uint32_t bound = 0;                      // of the list's keys
  float over = 0.f, low = 0.f;             // logits of the window: [low, over)
  const int have = min(THREADS, row.vectors / C);  // threads with a vector, in a CTA
  const int each_k = (set.k + C - 1) / C;
  if ((set.k > 0 || p_on) && p.vocab <= CAP) {
    mode = LIST;
  } else if (set.k > 0 && set.k <= BOUND_K && each_k <= min(LIST_K, have * 3 / 4)) {
    // A CTA's part of top_k: that many of its threads' largest logits reach its bound, so the least of the CTAs' bounds is one that
    // at least top_k logits of the row reach, and not many more where the CTAs' parts of the row are alike.
    mode = LIST;
    const uint32_t key = key_of(mine);
    constexpr int LOW = N == 8 ? 16 : 0;  // bits that tell no two bf16 apart
#pragma unroll 1
    for (int bit = 31; bit >= LOW; --bit) {
      const uint32_t tried = bound | (1u << bit);
      const int n = __syncthreads_count(key >= tried);
      if (n >= each_k) bound = tried;
      if (n == each_k) break;
    }
    if (C > 1) {
      if (tid == 0) sh.bound = bound;
      cluster.sync();
      for (int c = 0; c < C; ++c) bound = min(bound, of(c).bound);
    }
  } else if (set.k > 0 || p_on) {
    // ---- How many logits lie how far below the largest: which bin the cut falls to, almost surely
    for (int i = tid; i < BINS; i += THREADS) sh.hist[i] = 0;
    __syncthreads();
    uint32_t far = 0;
    row.one_by_one(v0 + tid, v1, THREADS, [&](const uint4& q, int i0) {
      Row<T>::fours(q, i0, [&](const float (&x)[4], int) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int b = bin(x[e]);
          if (b < BINS - 1) atomicAdd(&sh.hist[b], 1u);
          else far += x[e] > -INFINITY;
        }
      });
    });
    far = __reduce_add_sync(0xffffffffu, far);
    if (lane == 0 && far) atomicAdd(&sh.hist[BINS - 1], far);
    meet();
    if (rank == 0) {
      constexpr int PER = BINS / THREADS;
      // (the sums fit: at most 2^30 entries, and estimated masses in units of 2^-32)
      u64 sum = 0, mass = 0;
      float squares = 0.f;
      auto estimate = [&](int b, uint32_t n) {
        return static_cast<u64>(n * exp2f((b + 0.5f) * (-1.f / BIN_PER)) * 4294967296.f);
      };
      static_assert(PER == 4, "");
      uint4 bins = reinterpret_cast<const uint4*>(sh.hist)[tid];
#pragma unroll 4
      for (int c = 1; c < C; ++c) {
        const uint4 o = reinterpret_cast<const uint4*>(of(c).hist)[tid];
        bins.x += o.x, bins.y += o.y, bins.z += o.z, bins.w += o.w;
      }
      const uint32_t count[PER] = {bins.x, bins.y, bins.z, bins.w};
      u64 about[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        about[j] = estimate(tid * PER + j, count[j]);
        sum += count[j], mass += about[j];
        squares += static_cast<float>(about[j]) * static_cast<float>(about[j]);
      }
      Sums n = block_scan(sum, sh.sums), m{0, 0};
      if (tid == 0) sh.before = 0, sh.mode = SLOW;
      if (tid < 6) sh.edge[tid] = BINS - 1, sh.ahead_of[tid] = tid & 1 ? static_cast<uint32_t>(n.all) : 0;
      if (set.k > 0 && static_cast<u64>(set.k) < n.all) {  // (a top_k of all finite logits or more cuts nothing: as without it)
        __syncthreads();
        const u64 want = static_cast<u64>(set.k);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (n.before < want && n.before + count[j] >= want) {  // the bin of the k-th
            const u64 through = n.before + count[j];
            sh.before = static_cast<uint32_t>(n.before);
            sh.lo = sh.hi = tid * PER + j;
            if (through <= CAP) sh.mode = LIST;
            else if (!p_on && count[j] <= CAP) sh.mode = WINDOW_K;
          }
          n.before += count[j];
        }
      } else if (!p_on) {
        if (tid == 0) sh.mode = ALL;
      } else {
        m = block_scan(mass, sh.sums);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, d);
        if (lane == 0) sh.tops[warp] = squares;
        __syncthreads();
        squares = 0.f;
        for (int i = 0; i < WARPS; ++i) squares += sh.tops[i];
        // A window around the cut, as wide as the estimates may be wrong.  A logit's place in its bin is worth ln 2 / 128 of its weight
        // at most; the share of what is above an edge is off by half of that, at most 2^-8 of all, and by four standard deviations of
        // errors that are spread evenly and the same for all of a bin (bf16).  Or a quarter of it, or the bin alone, where the list does
        // not hold more.  (Whether the window holds the cut is checked by exact sums.)
        const float all = static_cast<float>(m.all), target = set.top_p * all;
        const float margin = fminf(all * (1.f / 256), 4 * 0.0031f * sqrtf(squares));
        u64 wanted[6];
#pragma unroll
        for (int t = 0; t < 6; ++t) {
          const float reach = t < 2 ? margin : t < 4 ? margin * 0.25f : 0.f;
          wanted[t] = max(u64{1}, static_cast<u64>(fmaxf(0.f, fminf(all, t & 1 ? target + reach : target - reach))));
        }
        const bool has_edge = m.before < wanted[1] && m.before + mass >= wanted[0];  // (all of them lie among these two)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          if (!has_edge) break;
#pragma unroll
          for (int t = 0; t < 6; ++t) {
            const u64 want = wanted[t];
            if (m.before < want && m.before + about[j] >= want) {
              sh.edge[t] = tid * PER + j;
              sh.ahead_of[t] = static_cast<uint32_t>(n.before + (t & 1 ? count[j] : 0));
            }
          }
          m.before += about[j], n.before += count[j];
        }
        __syncthreads();
        if (tid == 0)
          for (int t = 4; t >= 0; t -= 2)
            if (sh.ahead_of[t + 1] - sh.ahead_of[t] <= CAP) sh.mode = WINDOW_P, sh.lo = sh.edge[t], sh.hi = sh.edge[t + 1];
      }
    }
    meet();
    const Shared& o = of(0);
    mode = static_cast<Mode>(o.mode);
    const bool window = mode == WINDOW_P || mode == WINDOW_K || mode == LIST;
    if (window && warp < 2) {  // (a warp each, 32 keys at a time: by halves, in one thread, 3900 cycles)
      // the least logits of the bins up to lo - 1 and up to hi: the logits below have larger bins
      const int last = warp == 0 ? o.lo - 1 : o.hi;
      uint32_t below = KEY_NONE, from = last < 0 ? KEY_NONE + 1 : key_of(top);
#pragma unroll 1
      while (from - below > 1) {
        const uint32_t part = (from - below) / 32 + 1, mid = below + min(part * (lane + 1), from - below);
        const uint32_t low_bins = __ballot_sync(0xffffffffu, bin(of_key(mid)) <= last);  // (from itself among them: its bin is)
        const int first_of = __ffs(low_bins) - 1;  // of the lanes
        from = __shfl_sync(0xffffffffu, mid, first_of);
        if (first_of > 0) below = __shfl_sync(0xffffffffu, mid, first_of - 1);
      }
      if (lane == 0) sh.least_of[warp] = last < 0 ? key_of(INFINITY) : from;
    }
    __syncthreads();
    if (window) over = of_key(sh.least_of[0]), bound = sh.least_of[1], low = of_key(bound);
  }
  __syncthreads();

  u64 cut = 0;
  if (mode == LIST) {
    if (!p_on) bound = max(bound, set.key_min);
    low = of_key(max(bound, KEY_NONE + 1));
    row.template each<4>(v0 + tid, v1, THREADS, [&](const uint4& q, int i) {
      if (!(Row<T>::top(q) >= low)) return;
      Row<T>::fours(q, i, [&](const float (&x)[4], int j) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (x[e] >= low) append(key_of(x[e]), j + e);
      });
    });
  } else if (mode != SLOW) {
    // ---- sums of the tiles above the window and of the whole row; the window's entries on the list.  Where min_p's bound lies
    // above the window, what is above it is summed instead, and nothing of the window is kept.
    const float min_kept = of_key(max(set.key_min, KEY_NONE + 1));
    if (mode == ALL || min_kept >= over) over = min_kept, low = INFINITY;
    const Weight weight = sh.weight;
    const float from = fmaxf(over, of_key(key_of(weight.least) + 1));
    u64 rest = 0, above = 0;
    // f(4 values, index of the first) of each vector that has one from `least` on, tile by tile; the next load is under way
    auto tiles_of = [&](float least, auto f) {
      const int per_lane = per_tile / 32;
      int tile = t0 + warp, in = 0;
      u64 sum = 0;
      auto load = [&](int t, int k) {
        const int v = t * per_tile + k * 32 + lane;
        constexpr uint32_t NONE = N == 8 ? 0xFF80FF80u : 0xFF800000u;  // -inf
        return t < t1 && v < row.vectors ? row.load(v) : make_uint4(NONE, NONE, NONE, NONE);
      };
      uint4 next = load(tile, 0);
#pragma unroll 1
      while (tile < t1) {
        const uint4 now = next;
        const int v = tile * per_tile + in * 32 + lane;
        const bool ends = ++in == per_lane;
        next = ends ? load(tile + WARPS, 0) : load(tile, in);
        if (__any_sync(0xffffffffu, Row<T>::top(now) >= least))  // (by whole warps: lanes that part here would go on apart)
          Row<T>::fours_at_once(now, row.first(v), [&](const float (&x)[4], int i) { f(x, i, sum); });
        if (ends) {
          sum = warp_sum(sum);
          if (lane == 0) sh.tile[tile] = sum;
          above += sum;  // (the same in all lanes)
          sum = 0, in = 0, tile += WARPS;
        }
      }
    };
    if (mode == ALL) {
      tiles_of(from, [&](const float (&x)[4], int, u64& sum) {
#pragma unroll
        for (int e = 0; e < 4; ++e) add_if_from(sum, weight.above_least(x[e]), x[e], from);
      });
    } else {
      const float any = of_key(key_of(weight.least) + 1), least = mode == WINDOW_P ? any : fminf(over, low);
      tiles_of(least, [&](const float (&x)[4], int i, u64& sum) {
        uint32_t inside = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const u64 y = weight.above_least(x[e]);
          add_if_from(rest, y, x[e], any);
          add_if_from(sum, y, x[e], from);
          asm("{\n\t.reg .pred p, q;\n\tsetp.lt.f32 p, %1, %3;\n\tsetp.ge.and.f32 q, %1, %2, p;\n\t@q or.b32 %0, %0, %4;\n\t}"
              : "+r"(inside) : "f"(x[e]), "f"(low), "f"(over), "r"(1 << e));
        }
        if (__any_sync(0xffffffffu, inside != 0)) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (inside >> e & 1) append(key_of(x[e]), i + e);
          __syncwarp();
        }
      });
      rest = block_scan(rest, sh.sums).all;  // (of the whole row, where mode is WINDOW_P)
      above = block_scan(lane == 0 ? above : 0, sh.sums).all;
      if (tid == 0) sh.above = above, sh.all = rest;
    }
  }
  meet();
  int n = static_cast<int>(min(sh.count, static_cast<uint32_t>(CAP + 1)));
  u64 above = sh.above, all = sh.all;
  if (C > 1) {
    if (rank == 0) {
      for (int c = 1; c < C; ++c) {
        const Shared& o = of(c);
        const int m = static_cast<int>(min(o.count, static_cast<uint32_t>(CAP + 1)));
        if (n + m <= CAP)
          for (int i = tid; i < m; i += THREADS) sh.list[n + i] = o.list[i];
        n = min(n + m, CAP + 1);
        above += o.above, all += o.all;
        if (mode == ALL || mode == WINDOW_P || mode == WINDOW_K)
          for (int i = c * share + tid; i < min(tiles, (c + 1) * share); i += THREADS) sh.tile[i] = o.tile[i];
      }
      if (mode == LIST && n > CAP && tid > 0 && tid < C) of(tid).again = 1;
    }
    cluster.sync();
    if (rank != 0 && !sh.again) return;
  }
  if (mode == LIST && (rank != 0 || n > CAP)) {
    draw_again<T>(p, sh);
    return;
  }
  if (mode == LIST) {
    if (n <= SMALL) draw_small(p, sh, set, r, n);
    else draw_sorted(p, sh, set, r, n);
    return;
  }
  if (mode == WINDOW_P || mode == WINDOW_K) {
    // ---- the cut within the window, exactly.  Its entries' weights in 512 parts of the window (as three numbers of 17 bits, whose
    // sums stay below 32 bits), the part in which the sum reaches what is wanted, and that part's entries each against all others.
    constexpr int PER = CAP / THREADS;
    const float edge = fminf(over, top), fine_scale = fminf((THREADS - 1) / (edge - low), 1e30f);
    auto part_of = [&](u64 x) { return min(THREADS - 1, static_cast<int>((edge - of_key(key_in(x))) * fine_scale)); };
    u64 want = static_cast<u64>(set.k) - sh.before;
    if (mode == WINDOW_P) {
      want = least_of(set.top_p, all);
      if (want <= above) mode = SLOW;
      want -= above;
    }
    if (low == INFINITY) {  // min_p's bound is above the window
      if (mode != SLOW) mode = ALL;
    } else {
      for (int i = tid; i < 3 * THREADS; i += THREADS) (&sh.fine[0][0])[i] = 0;
      __syncthreads();
#pragma unroll 1
      for (int j = 0; j < PER; ++j) {
        const int i = tid + j * THREADS;
        if (i >= n) break;
        const u64 x = sh.list[i];
        const int part = part_of(x);
        const u64 w = mode == WINDOW_K ? 1 : sh.weight(of_key(key_in(x)));
        sh.weight_of[i] = w;
        atomicAdd(&sh.fine[0][part], static_cast<uint32_t>(w) & 0x1FFFFu);
        if (w >> 17) atomicAdd(&sh.fine[1][part], static_cast<uint32_t>(w >> 17) & 0x1FFFFu);
        if (w >> 34) atomicAdd(&sh.fine[2][part], static_cast<uint32_t>(w >> 34));
      }
      __syncthreads();
      const u64 mine_in = sh.fine[0][tid] + (static_cast<u64>(sh.fine[1][tid]) << 17) + (static_cast<u64>(sh.fine[2][tid]) << 34);
      if (tid == 0) sh.index = 0;
      const Sums s = block_scan(mine_in, sh.sums);
      if (want > s.all) mode = SLOW;
      if (mode != SLOW) {
        if (s.before < want && want <= s.before + mine_in) sh.lo = tid, sh.word = s.before;
        __syncthreads();
        const int part = sh.lo;
        want -= sh.word;
#pragma unroll 1
        for (int j = 0; j < PER; ++j) {
          const int i = tid + j * THREADS;
          if (i >= n) break;
          const u64 x = sh.list[i];
          if (part_of(x) == part) sh.other[atomicAdd(&sh.index, 1)] = static_cast<u64>(i);
        }
        __syncthreads();
        const int m = sh.index;
#pragma unroll 1
        for (int i = tid; i < m; i += THREADS) {
          const u64 me = sh.list[sh.other[i]];
          u64 ahead = 0;
#pragma unroll 4
          for (int j = 0; j < m; ++j) {
            const u64 at = sh.other[j];
            if (sh.list[at] > me) ahead += sh.weight_of[at];
          }
          if (ahead < want && want <= ahead + sh.weight_of[sh.other[i]]) sh.word = me;
        }
        __syncthreads();
        cut = sh.word;
#pragma unroll 1
        for (int j = 0; j < PER; ++j) {
          const int i = tid + j * THREADS;
          if (i >= n) break;
          const u64 x = sh.list[i];
          if (x >= cut && key_in(x) >= set.key_min)
            atomicAdd(&sh.tile[(index_in(x) + row.lead) / N / per_tile],
                      mode == WINDOW_K ? sh.weight(of_key(key_in(x))) : sh.weight_of[i]);
        }
        __syncthreads();
      }
    }
  }
  if (mode == SLOW) cut = slow_cut(row, sh, set, per_tile, tiles);

  // ---- the draw: which tile, and which entry of it
  const u64 a = 2 * tid < tiles ? sh.tile[2 * tid] : 0, b = 2 * tid + 1 < tiles ? sh.tile[2 * tid + 1] : 0;
  const Sums s = block_scan(a + b, sh.sums);
  const u64 want = drawn(set.u, s.all);
  if (s.before <= want && want < s.before + a + b) {
    const bool second = want >= s.before + a;
    sh.index = 2 * tid + second;
    sh.word = second ? s.before + a : s.before;
  }
  __syncthreads();
  u64 ahead = sh.word;
  const uint32_t least = max(set.key_min, KEY_NONE + 1);
  const int i0 = max(0, row.first(sh.index * per_tile)), i1 = min(row.vocab, row.first(min(row.vectors, (sh.index + 1) * per_tile)));
#pragma unroll 1
  for (int base = i0; base < i1 && ahead <= want; base += THREADS) {
    const int i = base + tid;
    float x = -INFINITY;
    u64 w = 0;
    if (i < i1) {
      x = row.at(i);
      const uint32_t key = key_of(x);
      if (key >= least && packed(key, i) >= cut) w = sh.weight(x);
    }
    const Sums in = block_scan(w, sh.sums);
    const u64 upto = ahead + in.before;
    if (upto <= want && want < upto + w) write_out(p, sh, r, set.t, i, x, s.all);
    ahead += in.all;
  }
}
}  // namespace sample

int32_t sample_execute(const cdl_sample_desc* desc, const cdl_tensor* logits, const cdl_tensor* uniform,
                       const cdl_tensor* temperature, const cdl_tensor* top_k, const cdl_tensor* top_p, const cdl_tensor* min_p,
                       const cdl_tensor* token, const cdl_tensor* logprob, cudaStream_t stream) {
  const char* op = "sample";
  if (!desc || !logits || !uniform || !token) return fail(CDL_ERR_INVALID, "%s: desc, logits, uniform and token are required", op);
  if (logits->rank != 2 || (logits->dtype != CDL_BF16 && logits->dtype != CDL_F32))
    return fail(CDL_ERR_INVALID, "%s: logits must be bf16 or f32 [rows, vocab]", op);
  const long long R = logits->shape[0], V = logits->shape[1];
  if (R < 0 || R > INT32_MAX || V < 0 || V > (1LL << 30))
    return fail(CDL_ERR_UNSUPPORTED, "%s: less than 2^31 rows and a vocabulary of at most 2^30", op);
  if ((V > 1 && logits->stride[1] != 1) || (R > 1 && logits->stride[0] < 0))
    return fail(CDL_ERR_INVALID, "%s: rows of logits must be contiguous", op);
  auto vec = [&](const char* name, const cdl_tensor* t, int32_t dtype) -> int32_t {
    if (t && (t->rank != 1 || t->dtype != dtype || t->shape[0] != R || (R > 1 && t->stride[0] != 1) || (R > 0 && !t->ptr)))
      return fail(CDL_ERR_INVALID, "%s: %s must be a packed %s [rows]", op, name, dtype_name(dtype));
    return CDL_OK;
  };
  CDL_CHECK(vec("uniform", uniform, CDL_F32));
  CDL_CHECK(vec("temperature", temperature, CDL_F32));
  CDL_CHECK(vec("top_k", top_k, CDL_I32));
  CDL_CHECK(vec("top_p", top_p, CDL_F32));
  CDL_CHECK(vec("min_p", min_p, CDL_F32));
  CDL_CHECK(vec("token", token, CDL_I32));
  CDL_CHECK(vec("logprob", logprob, CDL_F32));
  if (R == 0) return CDL_OK;
  if (V == 0 || !logits->ptr) return fail(CDL_ERR_INVALID, "%s: empty vocabulary or null logits", op);
  const cdl_tensor* ins[] = {logits, uniform, temperature, top_k, top_p, min_p};
  for (const cdl_tensor* i : ins)
    if (i && (!views_apart(*token, *i) || (logprob && !views_apart(*logprob, *i))))
      return fail(CDL_ERR_INVALID, "%s: an output overlaps an input", op);
  if (logprob && !views_apart(*token, *logprob)) return fail(CDL_ERR_INVALID, "%s: token and logprob overlap", op);
  sample::Params p{};
  p.z = logits->ptr, p.ld = logits->stride[0], p.vocab = static_cast<int>(V);
  p.u = static_cast<const float*>(uniform->ptr);
  p.temperature = temperature ? static_cast<const float*>(temperature->ptr) : nullptr;
  p.top_k = top_k ? static_cast<const int*>(top_k->ptr) : nullptr;
  p.top_p = top_p ? static_cast<const float*>(top_p->ptr) : nullptr;
  p.min_p = min_p ? static_cast<const float*>(min_p->ptr) : nullptr;
  p.all_temperature = desc->temperature, p.all_top_k = desc->top_k, p.all_top_p = desc->top_p, p.all_min_p = desc->min_p;
  p.token = static_cast<int*>(token->ptr);
  p.logprob = logprob ? static_cast<float*>(logprob->ptr) : nullptr;
  int bits = 0;
  while ((1LL << bits) < V) ++bits;
  p.scale_bits = std::min(50, 62 - bits);
  ProfileScope ps(PROF_ELEMENTWISE, static_cast<double>(R) * V * dtype_size(logits->dtype), stream);
  // CTAs of a row, of 16384 logits each or more: 4 or 3 where such clusters find an SM for each (7/8 of them), pairs where those do;
  // two to an SM where rows are long.  (top_p of 0.9 in 1, 2, 3 and 4 CTAs, us, from HBM: 150001 f32 logits, 16 rows 99, 59, 48,
  // 40, in 6 and 8 slower; 37 rows 101, 62, 49, 56; 48 rows 104, 66, 68, 57; 64 rows 111, 70, 70, 59; 74 rows 115, 71, 70, 87; 148 rows
  // 146, 106, 134, 135.  131072: 48 rows 91, 57, 61, 51; 64 rows 92, 58, 63, 52; of bf16 75, 50, 59, 50 and 76, 50, 60, 51.  65536: 48
  // rows 50, 35, 39, 34; 74 rows 51, 36, 41, 53; 148 rows 55, 52, 75, 83, of which the rule takes the first, 4 us above the second.
  // 32768 bf16: 16 rows 27, 23, 23, 22; 100 rows 28, 32, 45, 46.)
  const long long sms = sm_count(), own_sm = sms * 7 / 8 / R;
  const bool long_rows = V >= 131072;
  const long long fit = own_sm >= 3 ? own_sm : long_rows && 4 * R <= sms * 7 / 4 ? 4 : 2 * R <= (long_rows ? 2 * sms : sms) ? 2 : 1;
  p.cluster = static_cast<int>(std::max<long long>(1, std::min<long long>({4, fit, V / 16384})));
  void (*kernel)(sample::Params) = logits->dtype == CDL_BF16 ? sample::sample_kernel<__nv_bfloat16> : sample::sample_kernel<float>;
  const int smem = static_cast<int>(sizeof(sample::Shared));
  CDL_CUDA(allow_shared_memory(reinterpret_cast<const void*>(kernel), smem));
  const dim3 grid(static_cast<unsigned>(R * p.cluster));
  CDL_CUDA(p.cluster == 1 ? launch_pdl(kernel, grid, dim3(sample::THREADS), smem, stream, p)
                          : launch_pdl_cluster(kernel, grid, dim3(sample::THREADS), smem, p.cluster, stream, p));
  return CDL_OK;
}

}  // namespace cdl

extern "C" {

int32_t cdl_b200_sample(const cdl_sample_desc* desc, const cdl_tensor* logits, const cdl_tensor* uniform,
                        const cdl_tensor* temperature, const cdl_tensor* top_k, const cdl_tensor* top_p, const cdl_tensor* min_p,
                        const cdl_tensor* token, const cdl_tensor* logprob, cdl_stream stream) {
  return cdl::sample_execute(desc, logits, uniform, temperature, top_k, top_p, min_p, token, logprob,
                             static_cast<cudaStream_t>(stream));
}

}  // extern "C"
