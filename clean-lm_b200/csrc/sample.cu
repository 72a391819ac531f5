// A token per row of logits, drawn by a given random number.
//
//   d_i = (z_i - max z) / T,  w_i = exp(d_i);  the entries in the order of falling logits, lowest index first among equals
//   n   = min(top_k, first m whose w sum to top_p of those of the first top_k, number of w_i >= min_p), at least 1
//   token = the first i, by index, with sum of the kept w_j, j <= i, above u times their sum;  logprob = log(w_token / sum)
//
// The result is a whole number, so sums must not depend on the order in which threads add up, and a draw next to a border must
// fall as it does in exact arithmetic: weights are f64 exponentials, rounded to multiples of 2^-S and added as 64-bit integers
// (S = 62 - log2 of the vocabulary, so that no sum overflows; 2^-47 of the largest weight for 32768 entries, against 2^-24 in
// f32, where one draw in a few hundred of a flat row would fall on another token).
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
constexpr int CAP = 2048;    // entries that are sorted at most
constexpr int BINS = 2048;   // of the logits below the largest, in units of T ln 2 / BIN_PER
constexpr int BIN_PER = 64;
constexpr int TILES = 1024;  // of a row, whose sums are kept
constexpr int LIST_K = 384;  // top_k up to which a bound from the threads' largest logits finds the candidates

struct Params {
  const void* z;
  long long ld;
  long long vocab;
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
__device__ __forceinline__ u64 packed(uint32_t key, long long i) {
  return (static_cast<u64>(key) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

template <typename T>
struct Row {
  static constexpr int N = 16 / sizeof(T);  // logits of a 16-byte vector
  const T* z;
  long long vocab, vectors;
  int lead;  // logits between the 16-byte boundary and the row's first
  __device__ __forceinline__ Row(const void* p, long long V) : z(static_cast<const T*>(p)), vocab(V) {
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    vectors = (V + lead + N - 1) / N;
  }
  __device__ __forceinline__ long long first(long long v) const { return v * N - lead; }
  // Vector v of the row, -inf in front of it and behind it; nothing outside the row is read.
  __device__ __forceinline__ uint4 load(long long v) const {
    const long long i = first(v);
    if (i >= 0 && i + N <= vocab) return ld_nc_v4(z + i);
    union {
      T t[N];
      uint4 q;
    } r;
#pragma unroll
    for (int e = 0; e < N; ++e) r.t[e] = i + e >= 0 && i + e < vocab ? z[i + e] : static_cast<T>(-INFINITY);
    return r.q;
  }
  static __device__ __forceinline__ void values(const uint4& q, float (&x)[N]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (N == 8) x[2 * i] = bf16_lo(w[i]), x[2 * i + 1] = bf16_hi(w[i]);
      else x[i] = __uint_as_float(w[i]);
    }
  }
  __device__ __forceinline__ float at(long long i) const {
    if constexpr (N == 8) return __bfloat162float(z[i]);
    else return z[i];
  }
};

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

struct Shared {
  u64 list[CAP];
  union {
    u64 other[CAP];
    uint32_t hist[BINS];
    u64 wide_hist[256];
  };
  u64 tile[TILES];  // a CTA's tiles at their number in the row
  double pow2[256];
  u64 sums[WARPS];
  float fsums[WARPS];
  uint32_t rank_of[256];
  float top_of[WARPS];
  int at_of[WARPS];
  // what the cluster's other CTAs read
  float top;
  int at, bad;
  uint32_t count;
  u64 above, all;
  int mode, lo, hi;
  uint32_t before;
  u64 word;
  long long index;
};

// w = exp((z - top) / T) in units of 2^-S: 2^x with x = (z - top) log2(e) / T, split into n + j / 256 + r with |r| <= 1/512, a table
// of 2^(j/256) and the Taylor series of 2^r up to r^4, whose rest is 4e-17 (the table-driven method of P. T. P. Tang, 1989).
struct Weight {
  double top, per_t;  // log2(e) / T
  const double* pow2;
  int bits;
  __device__ __forceinline__ u64 operator()(float z) const {
    constexpr double L = 0.6931471805599453094, MAGIC = 6755399441055744.0;  // 1.5 2^52
    const double x = (static_cast<double>(z) - top) * per_t;
    if (!(x >= -70.0)) return 0;
    const double k = fma(x, 256.0, MAGIC);
    const int n = __double2loint(k);
    const double r = fma(k - MAGIC, -1.0 / 256.0, x);
    const double tab = pow2[n & 255];
    const double poly = fma(fma(fma(r, L * L * L * L / 24, L * L * L / 6), r, L * L / 2), r, L) * r;
    const long long v = __double_as_longlong(fma(tab, poly, tab));
    const u64 m = (static_cast<u64>(v) & 0xFFFFFFFFFFFFFull) | 0x10000000000000ull;
    const int sh = 52 + 1023 - static_cast<int>(v >> 52) - (n >> 8) - bits;
    if (sh <= 0) return m << -sh;
    return sh < 64 ? (m + (1ull << (sh - 1))) >> sh : 0;
  }
};

__device__ __forceinline__ u64 warp_sum(u64 x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}
// Sum over the threads ahead of this one, and over all of them.  Ends in a barrier.
__device__ __forceinline__ u64 block_scan(u64 x, u64* sums, u64& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 y = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 o = __shfl_up_sync(0xffffffffu, y, d);
    if (lane >= d) y += o;
  }
  if (lane == 31) sums[warp] = y;
  __syncthreads();
  u64 before = y - x;
  all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  __syncthreads();
  return before;
}

// a[0, n) in falling order, n <= CAP, all different; returns where it is, a or b.  Ends in a barrier.
__device__ u64* sort_down(Shared& sh, u64* a, u64* b, int n) {
  const int tid = threadIdx.x;
  if (n <= 256) {  // every entry counts those above it
    int p = 32;
    while (p < n) p <<= 1;
    if (tid < 256) sh.rank_of[tid] = 0;
    __syncthreads();
    const int i = tid & (p - 1), part = tid / p, parts = THREADS / p;
    if (i < n) {
      const u64 x = a[i];
      uint32_t r = 0;
      for (int j = part; j < n; j += parts) r += a[j] > x;
      atomicAdd(&sh.rank_of[i], r);
    }
    __syncthreads();
    if (tid < n) b[sh.rank_of[tid]] = a[tid];
    __syncthreads();
    return b;
  }
  int p = 512;
  while (p < n) p <<= 1;
  for (int i = n + tid; i < p; i += THREADS) a[i] = 0;
  for (int k = 2; k <= p; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int t = tid; t < p / 2; t += THREADS) {
        const int i = 2 * t - (t & (j - 1));  // the pairs i, i + j
        const u64 x = a[i], y = a[i + j];
        if ((x < y) == ((i & k) == 0)) a[i] = y, a[i + j] = x;
      }
    }
  __syncthreads();
  return a;
}

enum Mode { ALL = 0, WINDOW_P = 1, WINDOW_K = 2, LIST = 3, SLOW = 4 };

template <typename T>
struct Work {
  const Params& p;
  Shared& sh;
  Row<T> row;
  long long r;
  Weight weight;
  double t;
  float top, bin_scale;
  uint32_t key_min;           // of min_p; entries below it are not kept
  long long per_tile, tiles;  // vectors of a tile
  static constexpr int N = Row<T>::N;

  __device__ __forceinline__ int bin(float x) const { return min(BINS - 1, static_cast<int>((top - x) * bin_scale)); }

  __device__ __forceinline__ void write(long long i, float x, u64 mass) {
    p.token[r] = static_cast<int>(i);
    if (p.logprob)
      p.logprob[r] = static_cast<float>((static_cast<double>(x) - static_cast<double>(top)) / t -
                                        log(ldexp(static_cast<double>(mass), -p.scale_bits)));
  }
  // How many units of `mass` lie in front of the draw.
  __device__ __forceinline__ u64 drawn(u64 mass) const {
    const float u = p.u[r];
    bool rest;
    return u > 0.f ? (u < 1.f ? share_of(u, mass, rest) : mass - 1) : 0;
  }

  // f(vector's values, index of its first) over [v0, v1), four loads under way.
  template <typename F>
  __device__ __forceinline__ void each(long long v0, long long v1, int from, int step, F f) const {
    for (long long v = v0 + from; v < v1; v += 4 * step) {
      uint4 q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i * step < v1) q[i] = row.load(v + i * step);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i * step < v1) {
          float x[N];
          Row<T>::values(q[i], x);
          f(x, row.first(v + i * step));
        }
    }
  }
  __device__ __forceinline__ void append(uint32_t key, long long i) {
    const uint32_t at = atomicAdd(&sh.count, 1u);
    if (at < CAP) sh.list[at] = packed(key, i);
  }

  // Sums of the tiles [t0, t1): of the entries that are kept, which are those from `cut` on, without those below key_min.
  __device__ void sum_tiles(long long t0, long long t1, u64 cut) {
    const int lane = threadIdx.x & 31;
    const uint32_t least = max(key_min, KEY_NONE + 1);
    for (long long tile = t0 + (threadIdx.x >> 5); tile < t1; tile += WARPS) {
      u64 sum = 0;
      each(tile * per_tile, min(row.vectors, (tile + 1) * per_tile), lane, 32, [&](const float (&x)[N], long long i) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const uint32_t key = key_of(x[e]);
          if (key >= least && packed(key, i + e) >= cut) sum += weight(x[e]);
        }
      });
      sum = warp_sum(sum);
      if (lane == 0) sh.tile[tile] = sum;
    }
  }
  // The draw from the tiles' sums, which all of the block see.
  __device__ void draw_tiles(u64 cut) {
    const int tid = threadIdx.x;
    const u64 a = 2 * tid < tiles ? sh.tile[2 * tid] : 0, b = 2 * tid + 1 < tiles ? sh.tile[2 * tid + 1] : 0;
    u64 mass;
    const u64 before = block_scan(a + b, sh.sums, mass);
    const u64 want = drawn(mass);
    if (before <= want && want < before + a + b) {
      const bool second = want >= before + a;
      sh.index = 2 * tid + second;
      sh.word = second ? before + a : before;
    }
    __syncthreads();
    u64 ahead = sh.word;
    const uint32_t least = max(key_min, KEY_NONE + 1);
    const long long i0 = max(0LL, row.first(sh.index * per_tile));
    const long long i1 = min(row.vocab, row.first((sh.index + 1) * per_tile));
    for (long long base = i0; base < i1 && ahead <= want; base += THREADS) {
      const long long i = base + tid;
      float x = -INFINITY;
      u64 w = 0;
      if (i < i1) {
        x = row.at(i);
        const uint32_t key = key_of(x);
        if (key >= least && packed(key, i) >= cut) w = weight(x);
      }
      u64 all;
      const u64 upto = ahead + block_scan(w, sh.sums, all);
      if (upto <= want && want < upto + w) write(i, x, mass);
      ahead += all;
    }
  }

  // The draw where everything that may be kept is on the list.
  __device__ void draw_list(int n, long long k_in, float top_p) {
    const int tid = threadIdx.x;
    u64* order = sort_down(sh, sh.list, sh.other, n);
    u64* spare = order == sh.list ? sh.other : sh.list;
    const int per = (n + THREADS - 1) / THREADS;  // neighbouring entries of a thread, 4 at most
    u64 w[4], sum = 0, all;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * per + j;
      w[j] = j < per && i < n ? weight(of_key(static_cast<uint32_t>(order[i] >> 32))) : 0;
      sum += w[j];
    }
    u64 upto = block_scan(sum, sh.sums, all);
    const int n_k = k_in > 0 && k_in < n ? static_cast<int>(k_in) : n;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * per + j;
      upto += w[j];
      if (j < per && i < n) {
        spare[i] = upto;
      }
    }
    __syncthreads();
    int kept = n_k;
    const u64 want_p = top_p < 1.f ? least_of(top_p, spare[n_k - 1]) : ~0ull;
    u64 less = 0;  // entries that are kept: below the sum, from the least key on
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * per + j;
      if (j < per && i < n_k) {
        const u64 ahead = i == 0 ? 0 : spare[i - 1];
        less += (i == 0 || ahead < want_p) && static_cast<uint32_t>(order[i] >> 32) >= key_min;
      }
    }
    u64 count;
    block_scan(less, sh.sums, count);
    kept = max(1, static_cast<int>(count));
    const u64 mass = spare[kept - 1];
    const u64 want = drawn(mass);
    __syncthreads();
    // by index
    for (int i = tid; i < kept; i += THREADS) spare[i] = (order[i] << 32) | (order[i] >> 32);
    __syncthreads();
    const u64* line = sort_down(sh, spare, order, kept);
    sum = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * per + j;
      w[j] = j < per && i < kept ? weight(of_key(static_cast<uint32_t>(line[i]))) : 0;
      sum += w[j];
    }
    u64 ahead = block_scan(sum, sh.sums, all);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * per + j;
      if (ahead <= want && want < ahead + w[j])
        write(0xFFFFFFFFu - static_cast<uint32_t>(line[i] >> 32), of_key(static_cast<uint32_t>(line[i])), mass);
      ahead += w[j];
    }
  }

  // The entry at which the sum of f over the entries from `cut` on, in falling order, reaches `want`: 8 bits of the logit at a
  // time, then by index.  For windows that hold more than CAP entries: equal logits by the thousand, logits far from any scale
  // that the bins have.
  template <typename F>
  __device__ u64 select(F f, u64 want, u64 cut) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t prefix = 0;
    u64 above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) sh.wide_hist[tid] = 0;
      __syncthreads();
      each(0, row.vectors, tid, THREADS, [&](const float (&x)[N], long long i) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const uint32_t key = key_of(x[e]);
          if (key > KEY_NONE && packed(key, i + e) >= cut && (shift == 24 || (key >> (shift + 8)) == prefix))
            atomicAdd(&sh.wide_hist[(key >> shift) & 255], f(x[e]));
        }
      });
      __syncthreads();
      if (tid == 0) {
        u64 sum = above;
        int bin = 255;
        while (bin > 0 && sum + sh.wide_hist[bin] < want) sum += sh.wide_hist[bin--];
        sh.index = (prefix << 8) | static_cast<uint32_t>(bin);
        sh.word = sum;
      }
      __syncthreads();
      prefix = static_cast<uint32_t>(sh.index);
      above = sh.word;
      __syncthreads();
    }
    // how many of the entries equal to it, the lowest indices first
    const u64 one = f(of_key(prefix));
    const u64 ties = one == 0 ? 1 : (want - above + one - 1) / one;
    const long long seg = (row.vocab + THREADS * WARPS - 1) / (THREADS * WARPS) * THREADS;
    const long long i0 = min(row.vocab, warp * seg), i1 = min(row.vocab, i0 + seg);
    auto is = [&](long long i) {
      const uint32_t key = key_of(row.at(i));
      return key == prefix && packed(key, i) >= cut;
    };
    u64 n = 0, all;
    for (long long i = i0 + lane; i < i1; i += 32) n += is(i);
    u64 before = block_scan(n, sh.sums, all);
    before = __shfl_sync(0xffffffffu, before, 0);
    n = warp_sum(n);
    if (tid == 0) sh.word = packed(prefix, 0xFFFFFFFFLL);  // all of them
    __syncthreads();
    if (before < ties && before + n >= ties) {
      for (long long i = i0; i < i1; i += 32) {
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
  // One CTA alone, whatever the row is like.
  __device__ void slow(long long k_in, float top_p) {
    u64 cut = 0;
    if (k_in > 0 && k_in < row.vocab) cut = select([](float) { return u64{1}; }, static_cast<u64>(k_in), 0);
    if (top_p < 1.f) {
      const uint32_t least = key_min;
      key_min = 0;
      sum_tiles(0, tiles, cut);
      key_min = least;
      __syncthreads();
      u64 sum = 0, mass;
      for (long long i = threadIdx.x; i < tiles; i += THREADS) sum += sh.tile[i];
      block_scan(sum, sh.sums, mass);
      cut = select(weight, least_of(top_p, mass), cut);
    }
    sum_tiles(0, tiles, cut);
    __syncthreads();
    draw_tiles(cut);
  }
};

template <typename T>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const Params p) {
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
  if (tid < 256) sh.pow2[tid] = exp2(tid / 256.0);
  if (tid == 0) sh.count = 0, sh.above = 0, sh.all = 0;
  grid_dep_wait();
  grid_dep_launch();
  const long long r = blockIdx.x / C;
  Work<T> w{p, sh, Row<T>(static_cast<const T*>(p.z) + r * p.ld, p.vocab), r};
  constexpr int N = Row<T>::N;
  const long long vectors = w.row.vectors;
  constexpr int BASE = 512 / N;  // vectors of a tile: 512 logits, or as many more as leave at most TILES of them
  w.per_tile = (vectors + static_cast<long long>(BASE) * TILES - 1) / (static_cast<long long>(BASE) * TILES) * BASE;
  w.tiles = (vectors + w.per_tile - 1) / w.per_tile;
  const long long share = (w.tiles + C - 1) / C;  // tiles of a CTA
  const long long t0 = min(w.tiles, rank * share), t1 = min(w.tiles, t0 + share);
  const long long v0 = min(vectors, t0 * w.per_tile), v1 = min(vectors, t1 * w.per_tile);
  const float temperature = p.temperature ? p.temperature[r] : p.all_temperature;
  const long long k_in = p.top_k ? p.top_k[r] : p.all_top_k;
  const float top_p = p.top_p ? p.top_p[r] : p.all_top_p;
  const float min_p = p.min_p ? p.min_p[r] : p.all_min_p;

  // ---- the largest logit and its first place; NaN and +inf
  float mine = -INFINITY;
  int at = 0;
  bool bad = false;
  w.each(v0, v1, tid, THREADS, [&](const float (&x)[N], long long i) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      bad |= !(x[e] < INFINITY);
      if (x[e] > mine) mine = x[e], at = static_cast<int>(i) + e;
    }
  });
  float top = mine;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float x = __shfl_xor_sync(0xffffffffu, top, d);
    const int y = __shfl_xor_sync(0xffffffffu, at, d);
    if (x > top || (x == top && y < at)) top = x, at = y;
  }
  if (lane == 0) sh.top_of[warp] = top, sh.at_of[warp] = at;
  bad = __syncthreads_or(bad);
  if (tid == 0) {
    for (int i = 1; i < WARPS; ++i)
      if (sh.top_of[i] > top || (sh.top_of[i] == top && sh.at_of[i] < at)) top = sh.top_of[i], at = sh.at_of[i];
    sh.top = top, sh.at = at, sh.bad = bad;
  }
  meet();
  top = -INFINITY, at = 0, bad = false;
  for (int c = 0; c < C; ++c) {
    const Shared& o = of(c);
    if (o.top > top) top = o.top, at = o.at;
    bad |= o.bad != 0;
  }
  if (bad || top == -INFINITY || !(temperature > 0.f)) {
    if (rank == 0 && tid == 0) {
      const bool none = bad || top == -INFINITY;
      p.token[r] = none ? -1 : at;
      if (p.logprob) p.logprob[r] = none ? __uint_as_float(0x7FC00000u) : 0.f;
    }
    if (C > 1) cluster.sync();
    return;
  }
  w.top = top;
  w.t = static_cast<double>(temperature);
  w.weight = Weight{static_cast<double>(top), 1.4426950408889634074 / w.t, sh.pow2, p.scale_bits};
  w.bin_scale = static_cast<float>(w.weight.per_t) * BIN_PER;
  // w >= min_p: a bound on the logit, rounded up to the next one in f32
  w.key_min = min_p > 0.f ? key_of(__double2float_ru(static_cast<double>(top) + w.t * log(static_cast<double>(fminf(min_p, 1.f))))) : 0;
  w.key_min = min(w.key_min, key_of(top));
  const bool k_on = k_in > 0 && k_in < p.vocab, p_on = top_p < 1.f;

  const long long have = min(static_cast<long long>(THREADS), vectors / C);  // threads with a vector, in a CTA
  if ((k_on && k_in <= min(static_cast<long long>(LIST_K), have * 3 / 4)) || ((k_on || p_on) && p.vocab <= CAP)) {
    // ---- Few entries, all of them on a list.  The k-th of the threads' largest logits is a bound that at least k logits of this
    // CTA reach, and few more than k: its part of the row's k largest are among those.
    uint32_t bound = 0;
    if (k_on && p.vocab > CAP) {
      const uint32_t key = key_of(mine);
      constexpr int LOW = N == 8 ? 16 : 0;  // bits that tell no two bf16 apart
      for (int bit = 31; bit >= LOW; --bit) {
        const uint32_t tried = bound | (1u << bit);
        if (__syncthreads_count(key >= tried) >= k_in) bound = tried;
      }
    }
    if (!p_on) bound = max(bound, w.key_min);
    bound = max(bound, KEY_NONE + 1);
    w.each(v0, v1, tid, THREADS, [&](const float (&x)[N], long long i) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t key = key_of(x[e]);
        if (key >= bound) w.append(key, i + e);
      }
    });
    meet();
    uint32_t n = sh.count;
    if (rank == 0) {
      bool fits = n <= CAP;
      for (int c = 1; c < C; ++c) {
        const Shared& o = of(c);
        const uint32_t m = o.count;
        fits = fits && n + m <= CAP;
        if (fits)
          for (uint32_t i = tid; i < m; i += THREADS) sh.list[n + i] = o.list[i];
        n += m;
      }
      if (!fits) n = CAP + 1;
    }
    meet();
    if (rank != 0) return;
    if (n <= CAP) w.draw_list(static_cast<int>(n), k_in, top_p);
    else w.slow(k_in, top_p);
    return;
  }

  int mode = ALL, lo = 0, hi = 0;
  if (k_on || p_on) {
    // ---- How many logits lie how far below the largest: which bin the cut falls to, almost surely
    for (int i = tid; i < BINS; i += THREADS) sh.hist[i] = 0;
    __syncthreads();
    uint32_t far = 0;
    w.each(v0, v1, tid, THREADS, [&](const float (&x)[N], long long) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (!(x[e] > -INFINITY)) continue;
        const int b = w.bin(x[e]);
        if (b < BINS - 1) atomicAdd(&sh.hist[b], 1u);
        else ++far;
      }
    });
    far = static_cast<uint32_t>(warp_sum(far));
    if (lane == 0 && far) atomicAdd(&sh.hist[BINS - 1], far);
    meet();
    if (rank == 0) {
      constexpr int PER = BINS / THREADS;
      uint32_t n[PER];
      u64 sum = 0;
      float mass = 0.f, m[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int b = tid * PER + j;
        n[j] = sh.hist[b];
        for (int c = 1; c < C; ++c) n[j] += of(c).hist[b];
        m[j] = n[j] * exp2f((b + 0.5f) * (-1.f / BIN_PER));
        sum += n[j], mass += m[j];
      }
      u64 all;
      u64 upto = block_scan(sum, sh.sums, all);
      float fupto = mass;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const float o = __shfl_up_sync(0xffffffffu, fupto, d);
        if (lane >= d) fupto += o;
      }
      if (lane == 31) sh.fsums[warp] = fupto;
      if (tid == 0) sh.lo = sh.hi = BINS - 1, sh.before = 0;
      __syncthreads();
      fupto -= mass;
      float ftotal = 0.f;
      for (int i = 0; i < WARPS; ++i) {
        if (i < warp) fupto += sh.fsums[i];
        ftotal += sh.fsums[i];
      }
      const float target = fmaxf(top_p * ftotal, 1e-30f);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int b = tid * PER + j;
        if (k_on) {
          if (upto < static_cast<u64>(k_in) && upto + n[j] >= static_cast<u64>(k_in)) sh.lo = sh.hi = b, sh.before = static_cast<uint32_t>(upto);
        } else if (fupto < target && fupto + m[j] >= target) {
          sh.lo = sh.hi = b;
        }
        upto += n[j], fupto += m[j];
        sh.hist[b] = n[j];
      }
      __syncthreads();
      if (tid < 32) {
        const int b = sh.lo;
        const u64 through = sh.before + sh.hist[b];  // entries up to the bin of the k-th
        int m_now = SLOW, from = b, to = b;
        if (k_on) {
          if (k_in >= static_cast<long long>(all)) m_now = p_on ? SLOW : ALL;  // (the rest is -inf)
          else if (through <= CAP) m_now = LIST;
          else if (!p_on && sh.hist[b] <= CAP) m_now = WINDOW_K;
        } else {
          // A window around the bin, as wide as its sums may be wrong: by the logits' places within the bins, 2^-8 of all at
          // most.  (Whether it holds the cut is checked by exact sums.)
          const float each_bin = exp2f((b + 0.5f) * (-1.f / BIN_PER));
          const int d = lane + 1;
          uint32_t both = (b - d >= 0 ? sh.hist[b - d] : 0) + (b + d < BINS ? sh.hist[b + d] : 0);
          const float half = min(b - d >= 0 ? sh.hist[b - d] : 0x7FFFFFFFu, b + d < BINS ? sh.hist[b + d] : 0x7FFFFFFFu) * each_bin;
          float reach = half;
#pragma unroll
          for (int s = 1; s < 32; s <<= 1) {
            const uint32_t o = __shfl_up_sync(0xffffffffu, both, s);
            const float f = __shfl_up_sync(0xffffffffu, reach, s);
            if (lane >= s) both += o, reach += f;
          }
          const unsigned fits = __ballot_sync(0xffffffffu, sh.hist[b] + both <= CAP);
          const unsigned wide = __ballot_sync(0xffffffffu, reach >= ftotal * (1.f / 256));
          int width = wide ? __ffs(wide) : 32;         // bins on either side that suffice
          width = min(width, __popc(fits));            // and that the list holds (fits is a run of ones from bit 0)
          if (sh.hist[b] <= CAP) m_now = WINDOW_P, from = max(0, b - width), to = min(BINS - 1, b + width);
        }
        __syncwarp();
        if (lane == 0) sh.mode = m_now, sh.lo = from, sh.hi = to;
      }
    }
    meet();
    const Shared& o = of(0);
    mode = o.mode, lo = o.lo, hi = o.hi;
  }

  if (mode == LIST) {
    w.each(v0, v1, tid, THREADS, [&](const float (&x)[N], long long i) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (x[e] > -INFINITY && w.bin(x[e]) <= hi) w.append(key_of(x[e]), i + e);
    });
  } else if (mode == ALL) {
    w.sum_tiles(t0, t1, 0);
  } else if (mode != SLOW) {
    // ---- sums of the tiles above the window, of all above it and of all; the window's entries on the list
    u64 above = 0, all = 0;
    for (long long tile = t0 + warp; tile < t1; tile += WARPS) {
      u64 sum = 0;
      w.each(tile * w.per_tile, min(vectors, (tile + 1) * w.per_tile), lane, 32, [&](const float (&x)[N], long long i) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int b = w.bin(x[e]);
          if (b > hi && mode == WINDOW_K) continue;
          const uint32_t key = key_of(x[e]);
          if (key <= KEY_NONE) continue;
          const u64 y = w.weight(x[e]);
          all += y;
          if (b < lo) {
            above += y;
            if (key >= w.key_min) sum += y;
          } else if (b <= hi) {
            w.append(key, i + e);
          }
        }
      });
      sum = warp_sum(sum);
      if (lane == 0) sh.tile[tile] = sum;
    }
    u64 total;
    block_scan(above, sh.sums, total);
    if (tid == 0) sh.above = total;
    block_scan(all, sh.sums, total);
    if (tid == 0) sh.all = total;
  }
  meet();
  uint32_t n = sh.count;
  u64 above = sh.above, all = sh.all;
  if (rank == 0 && mode != SLOW) {
    for (int c = 1; c < C; ++c) {
      const Shared& o = of(c);
      const uint32_t m = o.count;
      if (n + m <= CAP)  // (by the bins' counts it is)
        for (uint32_t i = tid; i < m; i += THREADS) sh.list[n + i] = o.list[i];
      n += m;
      above += o.above, all += o.all;
      if (mode != LIST)
        for (long long i = c * share + tid; i < min(w.tiles, (c + 1) * share); i += THREADS) sh.tile[i] = o.tile[i];
    }
  }
  meet();
  if (rank != 0) return;
  if (mode == SLOW || n > CAP) {
    w.slow(k_in, top_p);
  } else if (mode == LIST) {
    w.draw_list(static_cast<int>(n), k_in, top_p);
  } else if (mode == ALL) {
    w.draw_tiles(0);
  } else {
    // ---- the cut within the window, exactly
    const u64* order = sort_down(sh, sh.list, sh.other, static_cast<int>(n));
    int keep;
    const int per = (static_cast<int>(n) + THREADS - 1) / THREADS;
    u64 y[4], sum = 0, inside;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * per + j;
      y[j] = j < per && i < static_cast<int>(n) ? w.weight(of_key(static_cast<uint32_t>(order[i] >> 32))) : 0;
      sum += y[j];
    }
    u64 ahead = above + block_scan(sum, sh.sums, inside);
    if (mode == WINDOW_P) {
      const u64 want = least_of(top_p, all);
      if (!(above < want && want <= above + inside)) {
        w.slow(k_in, top_p);
        return;
      }
      u64 less = 0, count;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = tid * per + j;
        ahead += y[j];
        less += j < per && i < static_cast<int>(n) && ahead < want;
      }
      block_scan(less, sh.sums, count);
      keep = static_cast<int>(count) + 1;
    } else {
      keep = static_cast<int>(k_in - sh.before);
    }
    const u64 cut = order[keep - 1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = tid * per + j;
      if (j < per && i < keep && static_cast<uint32_t>(order[i] >> 32) >= w.key_min) {
        const long long at_i = 0xFFFFFFFFu - static_cast<uint32_t>(order[i]);
        atomicAdd(&sh.tile[(at_i + w.row.lead) / N / w.per_tile], y[j]);
      }
    }
    __syncthreads();
    w.draw_tiles(cut);
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
  p.z = logits->ptr, p.ld = logits->stride[0], p.vocab = V;
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
  p.scale_bits = 62 - bits;
  ProfileScope ps(PROF_ELEMENTWISE, static_cast<double>(R) * V * dtype_size(logits->dtype), stream);
  // CTAs of a row: as many as leave every SM one, with 8192 logits each or more
  p.cluster = static_cast<int>(std::max<long long>(1, std::min<long long>({8, sm_count() / R, V / 8192})));
  void (*kernel)(sample::Params) = logits->dtype == CDL_BF16 ? sample::sample_kernel<__nv_bfloat16> : sample::sample_kernel<float>;
  const int smem = static_cast<int>(sizeof(sample::Shared));
  CDL_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
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
