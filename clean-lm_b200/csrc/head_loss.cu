// Losses of a language-model head: softmax cross entropy and distillation from a teacher's top entries, from the logits or
// from the hidden states and the head's weights without the logits in memory.
//
// Every loss here holds q = softmax(z / tau) of a row of logits against a distribution p that is zero but for a few
// entries (one for a target, K for a teacher), so that the gradient of the logits is
//     G_j = s tau (q_j - p_j),      s = grad_scale * d_loss[row]
// (cross entropy: tau = 1, p = 1 at the target).  With c = log2(e) / tau, M = max z, S = sum 2^(c (z_j - M)):
//     q_j = 2^(c (z_j - M)) / S,   log q_j = ln 2 (c (z_j - M) - log2 S),   lse = M / tau + ln 2 log2 S.
// All statistics are f32.  Differences are taken before they are scaled: a row masked with the type's lowest value, which times c
// overflows, is a uniform one; and what p holds of z - M is summed as it is: loss = tau^2 (sum p log p + ln S) - tau sum p (z - M),
// finite for an entry that is masked that way.
#include "host.h"
#include "ops.h"
#include "ptx.cuh"

#include <cuda_fp16.h>
#include <math.h>

#include <mutex>

namespace cdl {
namespace head {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int MAX_ENTRIES = 1024;  // of a teacher, per row: they are kept in shared memory
constexpr long long MAX_DIM = 1LL << 30;  // of vocabulary and hidden size: indices a few thousand further on are ints, too
constexpr int ROW_THREADS = 512;

static long long up(long long v, long long m) { return (v + m - 1) / m * m; }

// The distributions p of all rows: targets (one entry of probability 1), or a teacher's ids and logits.
struct Entries {
  const int* ids;       // targets, or ids [rows, K]
  const void* teacher;  // logits [rows, K]
  long long ids_ld, teacher_ld;
  int K, kind;  // kind: what the teacher's logits are
};
enum EntryKind { TARGETS, TEACHER_BF16, TEACHER_F32 };

__device__ __forceinline__ float teacher_logit(const Entries& e, long long row, int k) {
  return e.kind == TEACHER_F32 ? static_cast<const float*>(e.teacher)[row * e.teacher_ld + k]
                               : __bfloat162float(static_cast<const __nv_bfloat16*>(e.teacher)[row * e.teacher_ld + k]);
}

// What every row has besides its logits.
struct RowTerms {
  const float* d_loss;  // nullptr: 1
  long long d_loss_stride;
  float* loss;
  float* lse;  // nullptr: not wanted
  float grad_scale, tau;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The three bf16 pieces of an f32 value, v = p0 + p1 + p2 to 24 bits: the first two cut off (no finite value becomes infinite),
// the last rounded.
__device__ __forceinline__ void pieces_of(float v, float (&p)[3]) {
  p[0] = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
  const float r = v - p[0];
  p[1] = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
  p[2] = r - p[1];
}

// Where a row's gradient goes: T [.., ld], or the pieces of f32 values, bf16 [3][.., ld], planes `plane` apart.
struct GradRows {
  void* ptr;  // nullptr: not wanted
  long long ld, plane;
};
template <typename T, bool PIECES>
__device__ __forceinline__ void put(const GradRows& g, long long row, long long j, float v) {
  if constexpr (PIECES) {
    float p[3];
    pieces_of(v, p);
#pragma unroll
    for (int i = 0; i < 3; ++i) static_cast<__nv_bfloat16*>(g.ptr)[i * g.plane + row * g.ld + j] = __float2bfloat16_rn(p[i]);
  } else {
    static_cast<T*>(g.ptr)[row * g.ld + j] = from_f32<T>(v);
  }
}

// A row's entries in shared memory, and what a reduction over the CTA uses.
struct RowEntries {
  int* id;    // -1: does not count
  float* p;   // of the entry
  float* at;  // the row's logit at the id
  __device__ __forceinline__ RowEntries(void* smem, int K) : id(static_cast<int*>(smem)), p(static_cast<float*>(smem) + K), at(p + K) {}
};
constexpr int ENTRY_BYTES = 12;
struct RowShared {
  float part[32];
  float p_log_p;
  int counts;
};

__device__ __forceinline__ float cta_reduce(float v, bool max, float* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  v = max ? warp_max(v) : warp_sum(v);
  __syncthreads();  // (the last reduction's readers are through)
  if (lane == 0) part[warp] = v;
  __syncthreads();
  v = lane < warps ? part[lane] : (max ? -INFINITY : 0.f);
  return max ? warp_max(v) : warp_sum(v);
}

// A row's entries by one warp: ids and p = softmax(teacher / tau) over those that count (id in [0, vocab), logit above
// -inf); sum p log p; whether there are any; and (x != nullptr) the row's logits at the ids.  Four entries of a lane are under way at a
// time: their latency is what this costs.
template <typename T>
__device__ __forceinline__ void load_entries(const RowEntries& e, RowShared& sh, const Entries& src, long long row, int vocab,
                                             float tau, const T* x) {
  const int lane = threadIdx.x & 31;
  const float c = LOG2E / tau;
  if (src.kind == TARGETS) {
    const int id = src.ids[row];
    const bool counts = id >= 0 && id < vocab;
    if (lane == 0) {
      e.id[0] = counts ? id : -1;
      e.p[0] = counts ? 1.f : 0.f;
      if (x != nullptr) e.at[0] = counts ? to_f32(x[id]) : 0.f;
      sh.counts = counts;
      sh.p_log_p = 0.f;
    }
    return;
  }
  const int* ids = src.ids + row * src.ids_ld;
  float m = -INFINITY;
  for (int k0 = lane; k0 < src.K; k0 += 128) {
    int id[4];
    float y[4], at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + 32 * j;
      id[j] = k < src.K ? ids[k] : -1;
      y[j] = k < src.K ? teacher_logit(src, row, k) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (id[j] >= vocab) id[j] = -1;
      if (id[j] < 0) y[j] = -INFINITY;  // (padding may hold anything)
      if (y[j] == -INFINITY) id[j] = -1;
      at[j] = x != nullptr && id[j] >= 0 ? to_f32(x[id[j]]) : 0.f;
      m = fmaxf(m, y[j] != y[j] ? INFINITY : y[j]);  // a NaN makes the row NaN
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = k0 + 32 * j;
      if (k >= src.K) break;
      e.id[k] = id[j];
      e.p[k] = y[j];
      if (x != nullptr) e.at[k] = at[j];
    }
  }
  m = warp_max(m);
  const bool counts = m != -INFINITY;
  float s = 0.f, sy = 0.f;
  for (int k = lane; k < src.K; k += 32) {
    const float y = c * (e.p[k] - m), v = e.id[k] < 0 ? 0.f : ex2(y);
    e.p[k] = v;
    s += v;
    if (v != 0.f) sy += v * y;
  }
  s = warp_sum(s);
  sy = warp_sum(sy);
  const float over = 1.f / s;
  for (int k = lane; k < src.K; k += 32) e.p[k] = counts ? e.p[k] * over : 0.f;
  if (lane == 0) {
    sh.counts = counts;
    sh.p_log_p = counts ? LN2 * (sy * over - log2f(s)) : 0.f;
  }
}

// Which of a row's ids occur more than once: a hash table of more slots than entries, all -1 at first, in which
// an entry meets those of its id; a slot that has met one has the sign bit set.  0 <= id < INT32_MAX.
__device__ __forceinline__ unsigned slot_of(int slots_log2, int id) { return (static_cast<unsigned>(id) * 2654435761u) >> (32 - slots_log2); }
__device__ __forceinline__ void mark_id(int* table, int slots_log2, int id) {
  for (unsigned h = slot_of(slots_log2, id);; h = (h + 1) & ((1u << slots_log2) - 1)) {
    const int was = atomicCAS(&table[h], -1, id);
    if (was == -1 || was == (id | INT32_MIN)) return;
    if (was == id) {
      table[h] = id | INT32_MIN;
      return;
    }
  }
}
__device__ __forceinline__ bool is_marked(const int* table, int slots_log2, int id) {  // of an id that is in the table
  for (unsigned h = slot_of(slots_log2, id);; h = (h + 1) & ((1u << slots_log2) - 1)) {
    if (table[h] == id) return false;
    if (table[h] == (id | INT32_MIN)) return true;
  }
}

// One CTA per row: the row is read twice (the second time from the L2), any alignment and length.
template <typename T, bool PIECES>
__global__ void __launch_bounds__(ROW_THREADS)
    loss_row_kernel(const T* z, long long ld_z, const GradRows g, int vocab, const Entries src, const RowTerms terms) {
  __shared__ int entries[3 * MAX_ENTRIES];
  __shared__ RowShared sh;
  const RowEntries e(entries, src.K);
  grid_dep_wait();
  grid_dep_launch();
  const long long row = blockIdx.x;
  const T* x = z + row * ld_z;
  const float c = LOG2E / terms.tau;
  if (threadIdx.x < 32) load_entries(e, sh, src, row, vocab, terms.tau, x);
  __syncthreads();
  float m = -INFINITY, s = 0.f;
  bool bad = false;
  for (int j = threadIdx.x; j < vocab; j += ROW_THREADS) {
    const float v = to_f32(x[j]);
    bad = bad || v != v;
    if (v > m) {
      s = s * ex2(c * (m - v)) + 1.f;
      m = v;
    } else if (v != -INFINITY) {
      s += ex2(c * (v - m));
    }
  }
  const float top = cta_reduce(m, true, sh.part);
  const float base = top == -INFINITY ? 0.f : top;
  s = cta_reduce((bad ? NAN : s) * (m == -INFINITY ? (bad ? NAN : 0.f) : ex2(c * (m - base))), false, sh.part);
  const float log2_s = log2f(s);
  float cross = 0.f;  // tau sum_k p_k (z_k - M)
  for (int k = threadIdx.x; k < src.K; k += ROW_THREADS)
    if (e.p[k] != 0.f) cross += e.p[k] * terms.tau * (e.at[k] - base);
  cross = cta_reduce(cross, false, sh.part);
  const bool counts = sh.counts;
  if (threadIdx.x == 0) {
    terms.loss[row] = counts ? terms.tau * terms.tau * (sh.p_log_p + LN2 * log2_s) - cross : 0.f;
    if (terms.lse) terms.lse[row] = base / terms.tau + LN2 * log2_s;
  }
  if (g.ptr == nullptr) return;
  const float scale = counts ? terms.grad_scale * terms.tau * (terms.d_loss ? terms.d_loss[row * terms.d_loss_stride] : 1.f) : 0.f;
  const float over_s = scale / s;
  for (int j = threadIdx.x; j < vocab; j += ROW_THREADS)
    put<T, PIECES>(g, row, j, counts ? ex2(c * (to_f32(x[j]) - base)) * over_s : 0.f);
  __syncthreads();
  for (int k = threadIdx.x; k < src.K; k += ROW_THREADS) {
    const int id = e.id[k];
    if (id < 0) continue;
    float p = 0.f;  // each id once: the sum of its entries' probabilities, in their order
    bool again = false;
    for (int i = 0; i < src.K; ++i) {
      if (e.id[i] != id) continue;
      again = again || i < k;
      p += e.p[i];
    }
    if (!again) put<T, PIECES>(g, row, id, scale * (ex2(c * (e.at[k] - base)) / s - p));
  }
}

// The same with a row read from and written to HBM once: a cluster of 1 to 8 CTAs per row, whose warps have a slice of it each, at
// most 32 x VECS vectors of 16 bytes, which stay in registers: the maximum; the exponentials in place of the logits (bf16: as
// f16, 2^15 at the maximum, see store_tile_rows_exp in gemm.cu; their sum is of the f32 values); and, behind the one barrier at
// which the slices' parts of the statistics meet, the gradient.  The row's entries are a thread's each, and their softmax
// meets at the same barrier (8192 x 32768 with 64 entries 215 us, with one 183): where one warp prepared them all, the others waited
// for it, an eighth more time.  One exponential per element: a second one would put 4096 clk of special functions per 64 KB on an SM,
// whose share of the HBM's rate takes 5500.  The slices depend on the vocabulary and on whether rows are on the 16-byte
// grid, not on how many CTAs share a row, so a row's results do not depend on the number of rows.
//
// A vector that starts before the row or ends behind it is read whole where it holds an element of the row (the same 16
// bytes of memory); what is not the row's counts as -inf and is never written.
constexpr int WARPS = 16;              // of a CTA, at most

// Elements of a vector outside [lo, hi) become -inf.
template <typename T>
__device__ __forceinline__ void mask_vector(uint4& q, int lo, int hi) {
  uint32_t* w = &q.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      if (j < lo || j >= hi) w[j] = 0xff800000u;
    } else {
      if (2 * j < lo || 2 * j >= hi) w[j] = (w[j] & 0xffff0000u) | 0xff80u;
      if (2 * j + 1 < lo || 2 * j + 1 >= hi) w[j] = (w[j] & 0xffffu) | 0xff800000u;
    }
  }
}

// Two f32 operations as one.
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

template <typename T, int VECS, bool PIECES>
__global__ void __launch_bounds__(WARPS * 32, VECS <= 8 ? 2 : 1)
    loss_slices_kernel(const T* z, long long ld_z, const GradRows g, long long rows, long long ahead, int vocab, int slice, int ctas,
                       int slots_log2, const Entries src, const RowTerms terms) {
  constexpr bool HALF = sizeof(T) == 2;
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr float OFF = HALF ? 15.f : 0.f;  // the exponentials are 2^(c (z - M) + OFF)
  __shared__ float2 s_part[WARPS];  // (M, S) of the CTA's slices
  // Of 32 entries each: their largest teacher's logit y, w = sum 2^(c (y - largest)), the sum of those times c (y - largest).
  __shared__ float3 s_entries[MAX_ENTRIES / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const long long row = blockIdx.x / ctas;
  const int rank = blockIdx.x - static_cast<int>(row) * ctas;
  const T* x = z + row * ld_z;
  // The row in 16-byte vectors of memory: its first element is element `lead` of vector 0.  Element j of the row is
  // element j + first of the slice, which has n vectors.
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15) / static_cast<int>(sizeof(T));
  const int v0 = (rank * warps + warp) * slice;
  const int n = min(max((lead + vocab + VEC - 1) / VEC - v0, 0), slice), first = lead - v0 * VEC;
  const RowEntries e(smem, src.K);
  grid_dep_wait();
  grid_dep_launch();
  uint4 q[VECS];
  const T* from = x - first + lane * VEC;
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const uint32_t none = HALF ? 0xff80ff80u : 0xff800000u;  // -inf
    q[i] = lane + 32 * i < n ? *reinterpret_cast<const uint4*>(from + i * 32 * VEC) : make_uint4(none, none, none, none);
  }
  const float c = LOG2E / terms.tau;
  const float d_loss = terms.d_loss ? terms.d_loss[row * terms.d_loss_stride] : 1.f;
  // The row of a CTA that will follow this one goes to the L2 meanwhile, so that HBM is read under the arithmetic, too.
  if (lane == 0 && row + ahead < rows && n > 0) {
    const T* later = x + ahead * ld_z;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(later) & 15) / static_cast<int>(sizeof(T));
    const int count = min(max((off + vocab + VEC - 1) / VEC - v0, 0), slice);
    if (count > 0) bulk_prefetch_l2(later - off + static_cast<long long>(v0) * VEC, count * 16);
  }
  int* table = reinterpret_cast<int*>(smem + static_cast<size_t>(ENTRY_BYTES) * src.K);
  for (int i = threadIdx.x; i < 1 << slots_log2; i += blockDim.x) table[i] = -1;
  __syncthreads();
  // A warp has 32 entries at a time.
  float at_first = 0.f;  // the logit at the thread's first one: its load may take until the exponentials are done
  for (int group = warp; group * 32 < src.K; group += warps) {
    const int k = group * 32 + lane;
    int id = -1;
    float y = -INFINITY;
    if (k < src.K) {
      id = src.ids[row * src.ids_ld + k];
      y = src.kind == TARGETS ? 0.f : teacher_logit(src, row, k);
    }
    if (id < 0 || id >= vocab || y == -INFINITY) id = -1, y = -INFINITY;  // (padding may hold anything)
    else mark_id(table, slots_log2, id);
    const float at = id < 0 ? 0.f : to_f32(x[id]);
    const float top = warp_max(y != y ? INFINITY : y);  // (a NaN makes the row NaN)
    const float d = c * (y - top), v = id < 0 ? 0.f : ex2(d);
    if (k < src.K) {
      e.id[k] = id;
      e.p[k] = v;
      if (group != warp) e.at[k] = at;
    }
    if (group == warp) at_first = at;
    const float w = warp_sum(v), wd = warp_sum(v == 0.f ? 0.f : v * d);
    if (lane == 0) s_entries[group] = make_float3(top, w, wd);
  }
  if ((v0 == 0 && lead != 0) || first + vocab < n * VEC) {  // vectors of which the row has a part
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int at = (lane + 32 * i) * VEC;
      if (at < first || at + VEC > first + vocab) mask_vector<T>(q[i], first - at, first + vocab - at);
    }
  }
  float m = -INFINITY;
  if constexpr (HALF) {
    __nv_bfloat162 top = __float2bfloat162_rn(-INFINITY);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q[i]);
      top = __hmax2(__hmax2(top, __hmax2(h[0], h[1])), __hmax2(h[2], h[3]));
    }
    m = fmaxf(__low2float(top), __high2float(top));
  } else {
#pragma unroll
    for (int i = 0; i < VECS; ++i)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(q[i].x), __uint_as_float(q[i].y)), fmaxf(__uint_as_float(q[i].z), __uint_as_float(q[i].w))));
  }
  m = warp_max(m);
  const float own = m == -INFINITY ? 0.f : m;
  const uint64_t c2 = pack_f2(c, c), from2 = pack_f2(-own, -own), off2 = pack_f2(OFF, OFF);
  uint64_t sum2 = pack_f2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    if (32 * i >= n) break;
    uint32_t* w = &q[i].x;
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      float lo, hi;
      if constexpr (HALF) lo = bf16_lo(w[j]), hi = bf16_hi(w[j]);
      else lo = __uint_as_float(w[2 * j]), hi = __uint_as_float(w[2 * j + 1]);
      unpack_f2(fma_f2(add_f2(pack_f2(lo, hi), from2), c2, off2), lo, hi);
      lo = ex2(lo);
      hi = ex2(hi);
      sum2 = add_f2(sum2, pack_f2(lo, hi));
      if constexpr (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[j]) : "f"(hi), "f"(lo));
      else w[2 * j] = __float_as_uint(lo), w[2 * j + 1] = __float_as_uint(hi);
    }
  }
  float s, s_hi;
  unpack_f2(sum2, s, s_hi);
  s = warp_sum(s + s_hi);
  if (lane == 0) s_part[warp] = make_float2(m, s);
  if (threadIdx.x < src.K) e.at[threadIdx.x] = at_first;
  if (ctas > 1) cluster_sync_all();  // (the entries' logits have been read, too: they may be overwritten)
  else __syncthreads();
  auto part = [&](int w) {
    if (ctas == 1) return s_part[w];
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                 : "=f"(v.x), "=f"(v.y)
                 : "r"(mapa_shared(smem_u32(&s_part[w % warps]), w / warps)));
    return v;
  };
  // Up to 32 warps have a part per lane; more go through twice.
  const int all_warps = warps * ctas;
  const float2 mine = lane < all_warps ? part(lane) : make_float2(-INFINITY, 0.f);
  float base = mine.x;
  for (int i = lane + 32; i < all_warps; i += 32) base = fmaxf(base, part(i).x);
  base = warp_max(base);
  if (base == -INFINITY) base = 0.f;
  s = mine.y * ex2(c * (mine.x - base));
  for (int i = lane + 32; i < all_warps; i += 32) {
    const float2 v = part(i);
    s += v.y * ex2(c * (v.x - base));
  }
  s = warp_sum(s);
  if (ctas > 1) cluster_arrive_relaxed();  // this warp has read its peers' parts
  // The teacher's softmax: p of an entry is what it has in its group of 32 times the group's weight.
  const int groups = (src.K + 31) / 32;
  float ent_top = -INFINITY, ent_sum = 0.f;
  for (int i = 0; i < groups; ++i) ent_top = fmaxf(ent_top, s_entries[i].x);
  const bool counts = ent_top != -INFINITY;
  for (int i = 0; i < groups; ++i) ent_sum += s_entries[i].y * ex2(c * (s_entries[i].x - ent_top));  // (where the row counts)
  const float over = 1.f / ent_sum;
  auto weight_of = [&](int k) { return ex2(c * (s_entries[k / 32].x - ent_top)) * over; };
  if (rank == 0 && warp == warps - 1) {
    const float log2_s = log2f(s);
    // (sum p log2 p = sum p c (y - largest) - log2 of the sum)
    const float tau2 = terms.tau * terms.tau * LN2;
    const float rest = tau2 * ((log2_s - OFF) - log2f(ent_sum));
    float sum = 0.f;
    for (int k = lane; k < src.K; k += 32) {
      const float v = e.p[k];
      if (v != 0.f) sum -= v * weight_of(k) * terms.tau * (e.at[k] - base);
    }
    if (lane < groups && s_entries[lane].y != 0.f) {
      const float3 v = s_entries[lane];
      sum += tau2 * weight_of(32 * lane) * (v.z + v.y * (c * (v.x - ent_top)));
    }
    sum = warp_sum(sum) + rest;
    if (lane == 0) {
      terms.loss[row] = counts ? sum : 0.f;
      if (terms.lse) terms.lse[row] = base / terms.tau + LN2 * (log2_s - OFF);
    }
  }
  if (g.ptr != nullptr) {
    T* y = PIECES ? nullptr : static_cast<T*>(g.ptr) + row * g.ld;
    const float scale = counts ? terms.grad_scale * terms.tau * d_loss : 0.f;
    // (a slice of nothing but -inf: 0 wherever the others lie; NaN where the row is)
    const float factor = (m == -INFINITY ? 0.f : ex2(c * (own - base))) * (scale / s);
    const bool in_step = PIECES ? lead == 0 : static_cast<int>(reinterpret_cast<uintptr_t>(y) & 15) == lead * static_cast<int>(sizeof(T));
    const int at0 = lane * VEC - first;  // the row's element at the lane's first vector
    const uint64_t f2 = pack_f2(factor, factor);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      if (32 * i >= n) break;
      uint32_t* w = &q[i].x;
#pragma unroll
      for (int j = 0; j < 4; j += HALF ? 1 : 2) {
        float lo, hi;
        if constexpr (HALF) {
          const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
          unpack_f2(mul_f2(pack_f2(h.x, h.y), f2), lo, hi);
          w[j] = pack_bf16x2(lo, hi);
        } else {
          unpack_f2(mul_f2(pack_f2(__uint_as_float(w[j]), __uint_as_float(w[j + 1])), f2), lo, hi);
          w[j] = __float_as_uint(lo);
          w[j + 1] = __float_as_uint(hi);
        }
      }
      if (!counts) q[i] = make_uint4(0, 0, 0, 0);  // (whatever the logits were)
      if (lane + 32 * i >= n) continue;
      const int at = at0 + i * 32 * VEC;
      if constexpr (PIECES) {
        float v[4][3];
#pragma unroll
        for (int j = 0; j < 4; ++j) pieces_of(__uint_as_float(w[j]), v[j]);
        __nv_bfloat16* to = static_cast<__nv_bfloat16*>(g.ptr) + row * g.ld + at;
#pragma unroll
        for (int k = 0; k < 3; ++k, to += g.plane) {
          const uint2 pair = make_uint2(pack_bf16x2(v[0][k], v[1][k]), pack_bf16x2(v[2][k], v[3][k]));
          if (in_step && at >= 0 && at + VEC <= vocab) {
            *reinterpret_cast<uint2*>(to) = pair;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (at + j >= 0 && at + j < vocab) to[j] = __float2bfloat16_rn(v[j][k]);
          }
        }
      } else if (in_step && at >= 0 && at + VEC <= vocab) {
        *reinterpret_cast<uint4*>(y + at) = q[i];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (at + j >= 0 && at + j < vocab) {
            if constexpr (HALF) reinterpret_cast<uint16_t*>(y)[at + j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
            else reinterpret_cast<uint32_t*>(y)[at + j] = w[j];
          }
      }
    }
    __syncwarp();
    // The entries in this slice, each id once: the sum of its entries' probabilities, in their order.
    for (int k = lane; k < src.K; k += 32) {
      const int id = e.id[k], at = id + first;
      if (id < 0 || at < 0 || at >= n * VEC) continue;
      float p = e.p[k] * weight_of(k);
      if (is_marked(table, slots_log2, id)) {
        p = 0.f;
        bool again = false;
        for (int i = 0; i < src.K; ++i) {
          if (e.id[i] != id) continue;
          again = again || i < k;
          p += e.p[i] * weight_of(i);
        }
        if (again) continue;
      }
      put<T, PIECES>(g, row, id, scale * (ex2(c * (e.at[k] - base) + OFF) / s - p));
    }
  }
  if (ctas > 1) cluster_wait();  // the peers have read this CTA's parts
}

// ------------------------------------------------------------------------------------------ rows behind the fused product
// (matmul_exp_execute in gemm.cu: per row and piece of 128 columns M and S, the exponentials 2^(c (z - M) + 15) in f16, z at the
// entries' ids.)

// What the product and the row kernel read of a row's entries.
struct Prepared {
  const int* ids;               // targets, or a teacher's ids in ascending order, those that do not count behind them
  long long ids_ld;
  const unsigned short* first;  // [rows][pieces + 1]: the first entry at or behind a piece's columns; nullptr: targets
  const float* p;               // [rows][K], in the same order; nullptr: targets
  const float* p_log_p;         // [rows]
  const float* at;              // [rows][K]
};

constexpr int PREPARE_WARPS = 4;  // a row each

// A teacher's entries in the order of their ids (equal ids in their own order), one warp per row.  An entry's place is the
// number of those before it: K^2 comparisons of words in shared memory without a step that waits for another.
__global__ void __launch_bounds__(PREPARE_WARPS * 32)
    prepare_entries_kernel(const Entries src, long long rows, int vocab, float tau, int pieces, int* ids, unsigned short* first, float* p,
                           float* p_log_p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ RowShared shared[PREPARE_WARPS];
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = static_cast<long long>(blockIdx.x) * PREPARE_WARPS + warp;
  if (row >= rows) return;
  const RowEntries e(smem + static_cast<size_t>(warp) * ENTRY_BYTES * src.K, src.K);
  int* sorted = reinterpret_cast<int*>(e.at);
  load_entries<float>(e, shared[warp], src, row, vocab, tau, nullptr);
  __syncwarp();
  for (int k = lane; k < src.K; k += 32) sorted[k] = INT32_MAX;
  __syncwarp();
  if (lane == 0) p_log_p[row] = shared[warp].p_log_p;
  int n = 0;
  for (int k = lane; k < src.K; k += 32) {
    const int id = e.id[k];
    if (id < 0) continue;
    ++n;
    int place = 0;
#pragma unroll 8
    for (int i = 0; i < src.K; ++i)  // (-1 is the largest unsigned)
      place += static_cast<unsigned>(e.id[i]) < static_cast<unsigned>(id) || (e.id[i] == id && i < k);
    sorted[place] = id;
    ids[row * src.K + place] = id;
    p[row * src.K + place] = e.p[k];
  }
  n = __reduce_add_sync(0xffffffffu, n);
  __syncwarp();
  // Where each piece's ids begin: the number of ids before its columns.
  unsigned short* f = first + row * (pieces + 1);
  for (int i = lane; i <= pieces; i += 32) {
    const unsigned col = i == pieces ? 0x7fffffffu : static_cast<unsigned>(i) * 128u;
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (static_cast<unsigned>(sorted[mid]) < col) lo = mid + 1;
      else hi = mid;
    }
    f[i] = static_cast<unsigned short>(lo);
  }
}

constexpr int PIECES_PER_WARP = 64;  // at most: 8192 columns
constexpr int ROWS_PER_CTA = 8;      // a warp's each

// From the pieces' statistics the rows': loss, lse, and (with gradients) the gradient of the logits in bf16 in place of the
// exponentials, which are only multiplied with 2^(c (M - the row's)) s tau / S; the rows of x for the weight gradient's product,
// zeros where a row does not count.  GRAD_TWICE: what bf16 rounds away, in bf16 `rows` rows further on, and the rows of x again
// there: see Linear::twice.  Grid (rows / 8, pieces / per), a row and `per` pieces per warp; the warps have nothing
// to wait for in one another.
enum RowsMode { LOSS_ONLY, GRAD_ONCE, GRAD_TWICE };
template <int MODE>
__global__ void __launch_bounds__(ROWS_PER_CTA * 32)
    softmax_rows_kernel(const float2* stats, float c, __nv_bfloat16* e, long long ld_e, int rows, int vocab, int pieces, int per,
                        int K, const Prepared src, const RowTerms terms, const __nv_bfloat16* x, long long ld_x, __nv_bfloat16* clean,
                        long long ld_clean, int cols) {
  constexpr bool GRAD = MODE != LOSS_ONLY;
  __shared__ float factor[ROWS_PER_CTA][PIECES_PER_WARP];
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * ROWS_PER_CTA + warp;
  if (row >= rows) return;
  stats += static_cast<long long>(row) * pieces;
  const int piece0 = blockIdx.y * per, piece1 = min(pieces, piece0 + per);
  const int target = src.first == nullptr ? src.ids[row] : -1;
  const unsigned short* first = src.first + static_cast<long long>(row) * (pieces + 1);
  const int entries = src.first == nullptr ? (target >= 0 && target < vocab ? 1 : 0) : first[pieces];
  const float d_loss = GRAD && terms.d_loss ? terms.d_loss[row * terms.d_loss_stride] : 1.f;
  float m = -INFINITY, S = 0.f;
  for (int i = lane; i < pieces; i += 256) {  // eight loads under way
    float2 v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = i + 32 * j < pieces ? stats[i + 32 * j] : make_float2(-INFINITY, 0.f);
    float top = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, v[j].x);
    const float from = top == -INFINITY ? 0.f : top;
    S *= ex2(c * (m - from));
#pragma unroll
    for (int j = 0; j < 8; ++j) S += v[j].y * ex2(c * (v[j].x - from));
    m = top;
  }
  const float top = warp_max(m);
  const float base = top == -INFINITY ? 0.f : top;
  S = warp_sum(S * ex2(c * (m - base)));  // (2^15 times the sum)
  const float log2_s = log2f(S) - 15.f;
  const bool counts = entries > 0;
  if (blockIdx.y == 0) {
    const float tau = LN2 * c * (terms.tau * terms.tau);  // (c has what the products put back)
    float cross = 0.f;  // tau sum_k p_k (z_k - M)
    for (int k = lane; k < entries; k += 32) {
      const float p = src.p == nullptr ? 1.f : src.p[static_cast<long long>(row) * K + k];
      if (p != 0.f) cross += p * tau * (src.at[static_cast<long long>(row) * K + k] - base);
    }
    cross = warp_sum(cross);
    if (lane == 0) {
      const float entropy = src.p == nullptr ? 0.f : src.p_log_p[row];
      terms.loss[row] = counts ? terms.tau * terms.tau * (entropy + LN2 * log2_s) - cross : 0.f;
      if (terms.lse) terms.lse[row] = LN2 * (c * base + log2_s);
    }
  }
  if (!GRAD) return;
  const float scale = counts ? terms.grad_scale * terms.tau * d_loss : 0.f, over_s = scale / S;
  for (int i = piece0 + lane; i < piece1; i += 32) factor[warp][i - piece0] = ex2(c * (stats[i].x - base)) * over_s;
  __syncwarp();
  uint4* at = reinterpret_cast<uint4*>(e + row * ld_e + piece0 * 128);
  uint4* rest = reinterpret_cast<uint4*>(e + (static_cast<long long>(rows) + row) * ld_e + piece0 * 128);
  const int vecs = (piece1 - piece0) * 16;  // of 8 columns
  constexpr int DEEP = 2;  // (4 and 8: the same to 2 % more)
  for (int v = lane; v < vecs; v += 32 * DEEP) {
    uint4 q[DEEP];
#pragma unroll
    for (int d = 0; d < DEEP; ++d)
      if (v + 32 * d < vecs) q[d] = at[v + 32 * d];
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      if (v + 32 * d >= vecs) break;
      const float f = factor[warp][(v + 32 * d) >> 4];
      uint4 lo;
      uint32_t *w = &q[d].x, *l = &lo.x;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        w[j] = pack_bf16x2(h.x * f, h.y * f);
        if (MODE == GRAD_TWICE) l[j] = pack_bf16x2(h.x * f - bf16_lo(w[j]), h.y * f - bf16_hi(w[j]));
      }
      at[v + 32 * d] = counts ? q[d] : make_uint4(0, 0, 0, 0);  // (whatever the logits were)
      if (MODE == GRAD_TWICE) rest[v + 32 * d] = counts ? lo : make_uint4(0, 0, 0, 0);
    }
  }
  if (clean != nullptr) {  // the splits share the row of x
    const int per_row = (cols + 7) / 8, share = (per_row + gridDim.y - 1) / gridDim.y;
    const int c1 = min(per_row, static_cast<int>(blockIdx.y + 1) * share);
    for (int i = blockIdx.y * share + lane; i < c1; i += 32) {
      const __nv_bfloat16* from = x + row * ld_x + i * 8;
      __nv_bfloat16* to = clean + row * ld_clean + i * 8;
      if (i * 8 + 8 <= cols) {
        const uint4 v = counts ? *reinterpret_cast<const uint4*>(from) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(to) = v;
        if (MODE == GRAD_TWICE) *reinterpret_cast<uint4*>(to + rows * ld_clean) = v;
      } else {
        for (int j = 0; i * 8 + j < cols; ++j) {
          to[j] = counts ? from[j] : __float2bfloat16_rn(0.f);
          if (MODE == GRAD_TWICE) to[rows * ld_clean + j] = to[j];
        }
      }
    }
  }
  __syncwarp();
  // The entries of these columns, each id once: the sum of its entries' probabilities, in their order.
  if (!counts) return;
  int k0 = 0, k1 = 1;
  if (src.first != nullptr) {
    k0 = first[piece0];
    k1 = first[piece1];
  }
  const int* ids = src.ids + row * src.ids_ld;
  for (int k = k0 + lane; k < k1; k += 32) {
    const int id = ids[k];
    if (src.first == nullptr ? id / 128 < piece0 || id / 128 >= piece1 : k > k0 && ids[k - 1] == id) continue;
    float p = src.p == nullptr ? 1.f : src.p[static_cast<long long>(row) * K + k];
    for (int i = k + 1; i < k1 && ids[i] == id; ++i) p += src.p[static_cast<long long>(row) * K + i];
    const float g = scale * (ex2(c * (src.at[static_cast<long long>(row) * K + k] - base) + 15.f) / S - p);
    const __nv_bfloat16 hi = __float2bfloat16_rn(g);
    e[row * ld_e + id] = hi;
    if (MODE == GRAD_TWICE) e[(static_cast<long long>(rows) + row) * ld_e + id] = __float2bfloat16_rn(g - __bfloat162float(hi));
  }
}

// ------------------------------------------------------------------------------------------ operands and gradients off the grid
// A block has SEGMENT columns of a row, its threads neighbouring ones: any strides and alignment, eight accesses of a thread under
// way.  (381 MB of bf16 rows of odd length 480 -> 173 us against a loop over 256 columns with one.)
constexpr int SEGMENT = 2048;

struct Segment {
  long long row;
  int col;
  __device__ __forceinline__ Segment(int cols) {
    const int per_row = (cols + SEGMENT - 1) / SEGMENT;
    row = blockIdx.x / per_row;
    col = static_cast<int>(blockIdx.x - row * per_row) * SEGMENT + threadIdx.x;
  }
};

// dst[r, c] = src[r, c].
template <typename T>
__global__ void __launch_bounds__(256) copy_kernel(const T* src, long long s_row, long long s_col, T* dst, long long d_row, long long d_col,
                                                          int cols) {
  grid_dep_wait();
  grid_dep_launch();
  const Segment at(cols);
  const T* from = src + at.row * s_row;
  T v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (at.col + 256 * j < cols) v[j] = from[(at.col + 256 * j) * s_col];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (at.col + 256 * j < cols) dst[at.row * d_row + (at.col + 256 * j) * d_col] = v[j];
}

// The same for rows of neighbouring elements, from and to any alignment: a thread has 16 aligned bytes of dst at a time, out
// of the two aligned 16 bytes of src that hold them (both hold an element of the row); what a row has of its first and last 16 bytes
// goes one by one. 190 MB of bf16 rows of 85695: 71 us, 5.4 TB/s; element by element 93.
constexpr int COPY_VECS = 4;  // of a thread, 256 apart
__global__ void __launch_bounds__(256)
    copy_rows_kernel(const __nv_bfloat16* src, long long s_row, __nv_bfloat16* dst, long long d_row, int cols, unsigned per_row, long long all) {
  grid_dep_wait();
  grid_dep_launch();
  const long long first = static_cast<long long>(blockIdx.x) * (256 * COPY_VECS) + threadIdx.x;
  const long long row0 = first / per_row;  // the thread's next vectors lie a few rows further on at most
  const unsigned in_row0 = static_cast<unsigned>(first - row0 * per_row);
  uint4 lo[COPY_VECS], hi[COPY_VECS];
  int at[COPY_VECS];  // the row's element that the vector begins with, INT_MIN: none
  unsigned shift[COPY_VECS];
#pragma unroll
  for (int j = 0; j < COPY_VECS; ++j) {
    at[j] = INT32_MIN;
    if (first + 256 * j >= all) continue;
    const unsigned on = (in_row0 + 256 * j) / per_row;
    const __nv_bfloat16* to = dst + (row0 + on) * d_row;
    at[j] = static_cast<int>(in_row0 + 256 * j - on * per_row) * 8 - static_cast<int>((reinterpret_cast<uintptr_t>(to) & 15) / 2);
    if (at[j] < 0 || at[j] + 8 > cols) continue;
    const uintptr_t from = reinterpret_cast<uintptr_t>(src + (row0 + on) * s_row + at[j]);
    shift[j] = from & 15;
    lo[j] = *reinterpret_cast<const uint4*>(from - shift[j]);
    if (shift[j] != 0) hi[j] = *reinterpret_cast<const uint4*>(from - shift[j] + 16);
  }
#pragma unroll
  for (int j = 0; j < COPY_VECS; ++j) {
    if (at[j] == INT32_MIN || at[j] >= cols) continue;
    const long long row = row0 + (in_row0 + 256 * j) / per_row;
    __nv_bfloat16* to = dst + row * d_row + at[j];
    if (at[j] < 0 || at[j] + 8 > cols) {
      const __nv_bfloat16* from = src + row * s_row + at[j];
      for (int i = 0; i < 8; ++i)
        if (at[j] + i >= 0 && at[j] + i < cols) to[i] = from[i];
      continue;
    }
    uint32_t w[8] = {lo[j].x, lo[j].y, lo[j].z, lo[j].w, hi[j].x, hi[j].y, hi[j].z, hi[j].w};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = shift[j] & 8 ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = shift[j] & 4 ? w[i + 1] : w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = shift[j] & 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The pieces of f32 values.  Zeros where keep (nullptr: all rows count) says that a row does not count.  dst: [3][rows][ld], planes
// `plane` apart.
__global__ void __launch_bounds__(256)
    split_kernel(const float* src, long long s_row, long long s_col, __nv_bfloat16* dst, long long ld, long long plane, int cols,
                 const float* keep) {
  grid_dep_wait();
  grid_dep_launch();
  const Segment at(cols);
  const float* from = src + at.row * s_row;
  const bool zero = keep != nullptr && keep[at.row] == 0.f;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (at.col + 256 * j < cols) v[j] = from[(at.col + 256 * j) * s_col];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (at.col + 256 * j >= cols) break;
    const float x = zero ? 0.f : v[j];
    float p[3];
    pieces_of(x, p);
    __nv_bfloat16* o = dst + at.row * ld + at.col + 256 * j;
    o[0] = __float2bfloat16_rn(p[0]);
    o[plane] = __float2bfloat16_rn(p[1]);
    o[2 * plane] = __float2bfloat16_rn(p[2]);
  }
}

// out[r, c] = the sum of the f32 planes at r, c in their order (+ out[r, c]).  One plane: the end of a gradient that scratch held.
// No plane: zeros.
template <typename T>
__global__ void __launch_bounds__(256)
    sum_planes_kernel(const float* planes, long long ld, long long plane, int slices, T* out, long long o_row, long long o_col, int cols, int add) {
  grid_dep_wait();
  grid_dep_launch();
  const Segment at(cols);
  const float* from = planes + at.row * ld + at.col;
  T* o = out + at.row * o_row + at.col * o_col;
  float v[8] = {};
  for (int s = 0; s < slices; ++s)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at.col + 256 * j < cols) v[j] += from[s * plane + 256 * j];
  if (add) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (at.col + 256 * j < cols) v[j] += to_f32(o[256 * j * o_col]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (at.col + 256 * j < cols) o[256 * j * o_col] = from_f32<T>(v[j]);
}
// The same by vectors of four, where the rows of out and of the planes allow them: a thread has one, SUM_DEPTH loads of it under way
// whatever the number of planes.  (Losses with their gradients, 4 / 8 / 12 / 24 loads: 64 x 512 x 8192, 32 planes, 34.6 / 32.9 / 32.6 / 32.3 us;
// 64 x 2048 x 32768, 36 planes, 104.5 / 103.5 / 102.8 / 102.9; 100 x 2560 x 32768, 14 planes, 119.3 / 118.9 / 118.9 / 119.7.)
constexpr int SUM_DEPTH = MAX_PLANES / 2;
template <typename T>
__global__ void __launch_bounds__(128)
    sum_vectors_kernel(const float* planes, long long ld, long long plane, int slices, T* out, long long o_row, long long all, int cols, int add) {
  grid_dep_wait();
  grid_dep_launch();
  const long long i = static_cast<long long>(blockIdx.x) * 128 + threadIdx.x;
  if (i >= all) return;
  const int per_row = cols / 4;
  const long long r = i / per_row;
  const int c = static_cast<int>(i - r * per_row) * 4;
  const float* from = planes + r * ld + c;
  T* o = out + r * o_row + c;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < slices; s0 += SUM_DEPTH) {
    float4 x[SUM_DEPTH];
#pragma unroll
    for (int i = 0; i < SUM_DEPTH; ++i)
      if (s0 + i < slices) x[i] = *reinterpret_cast<const float4*>(from + (s0 + i) * plane);
#pragma unroll
    for (int i = 0; i < SUM_DEPTH; ++i) {
      if (s0 + i >= slices) break;
      v.x += x[i].x; v.y += x[i].y; v.z += x[i].z; v.w += x[i].w;
    }
  }
  if (add) v.x += to_f32(o[0]), v.y += to_f32(o[1]), v.z += to_f32(o[2]), v.w += to_f32(o[3]);
  if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  else *reinterpret_cast<float4*>(o) = v;
}

// 1 for a row that counts, 0 for one without a target or entries.
__global__ void __launch_bounds__(256) keep_kernel(const Entries src, long long rows, int vocab, float* keep) {
  grid_dep_wait();
  grid_dep_launch();
  const long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  bool any = false;
  for (int k = threadIdx.x & 31; k < src.K; k += 32) {
    const int id = src.ids[row * src.ids_ld + k];
    if (id < 0 || id >= vocab) continue;
    any = any || src.kind == TARGETS || teacher_logit(src, row, k) != -INFINITY;
  }
  any = __any_sync(0xffffffffu, any);
  if ((threadIdx.x & 31) == 0) keep[row] = any ? 1.f : 0.f;
}

// ------------------------------------------------------------------------------------------ few rows of f32 operands
// Up to FEW_ROWS tokens an f32 product reads w once, as it is, and multiplies in f32, two tokens per instruction: 2 T operations per 4
// bytes, at 16 tokens a third of what the SMs do while HBM brings the bytes.  (The pieces of w alone are 2.5 times its
// bytes, written and read by three products: 4 x 2048 x 112256 1546 us, 492 so; 8 tokens 1568 and 562, 16 tokens 1538 and 844.)  TT tokens are a
// thread's accumulators; those behind the last are zeros.  Any alignment: lanes have neighbouring elements.
constexpr int FEW_ROWS = 16, FEW_THREADS = 256, FEW_WARPS = FEW_THREADS / 32;
constexpr int FEW_CHUNK = 512;      // of K in shared memory at a time
constexpr int FEW_OUTER_COLS = 128, FEW_INNER_COLS = 4 * FEW_WARPS;  // of a block

// [k][TT] in shared memory: all tokens of columns k0 .. k0 + n - 1 of a, zeros for tokens that do not exist or (keep: nullptr, or
// a flag per token) do not count.
template <int TT>
__device__ __forceinline__ void few_columns(float* s, const float* a, long long lda, int T, long long k0, int n, const float* keep) {
  for (int k = threadIdx.x; k < n; k += FEW_THREADS) {
#pragma unroll
    for (int q = 0; q < TT / 4; ++q) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = 4 * q + j;
        v[j] = t < T && (keep == nullptr || keep[t] != 0.f) ? a[t * lda + k0 + k] : 0.f;
      }
      *reinterpret_cast<float4*>(s + k * TT + 4 * q) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
}

// out[slice][t, n] = sum over the slice's k of a[t, k] b[k, n]: a block has 128 columns, a lane four of them, the warps every eighth k.
template <int TT>
__global__ void __launch_bounds__(FEW_THREADS, TT == 4 ? 4 : TT == 8 ? 3 : 2)
    few_outer_kernel(const float* a, long long lda, const float* b, long long ldb, int T, int K, int N, int slices, float* out, long long ldo,
                     long long plane) {
  __shared__ __align__(16) float s_a[FEW_CHUNK * TT];
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slice = blockIdx.y, first = blockIdx.x * FEW_OUTER_COLS, n0 = first + lane;
  const bool whole = first + FEW_OUTER_COLS <= N;
  const int k0 = static_cast<int>(static_cast<long long>(K) * slice / slices), k1 = static_cast<int>(static_cast<long long>(K) * (slice + 1) / slices);
  constexpr int U = 4, STEP = FEW_WARPS * U;
  uint64_t acc[4][TT / 2];  // of two tokens each
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int t = 0; t < TT / 2; ++t) acc[c][t] = 0;
  for (int kc = k0; kc < k1; kc += FEW_CHUNK) {
    const int n = min(FEW_CHUNK, k1 - kc);
    __syncthreads();
    few_columns<TT>(s_a, a, lda, T, kc, n, nullptr);
    __syncthreads();
    const float* from = b + static_cast<long long>(kc + warp) * ldb + n0;
    for (int k = warp; k < n; k += STEP, from += STEP * ldb) {
      float v[U][4];
      if (whole && k + FEW_WARPS * (U - 1) < n) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int c = 0; c < 4; ++c) v[u][c] = from[u * FEW_WARPS * ldb + 32 * c];
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int c = 0; c < 4; ++c) v[u][c] = k + FEW_WARPS * u < n && n0 + 32 * c < N ? from[u * FEW_WARPS * ldb + 32 * c] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k + FEW_WARPS * u >= n) break;
        uint64_t w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = pack_f2(v[u][c], v[u][c]);
#pragma unroll
        for (int q = 0; q < TT / 4; ++q) {
          const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(s_a + (k + FEW_WARPS * u) * TT + 4 * q);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            acc[c][2 * q] = fma_f2(x.x, w[c], acc[c][2 * q]);
            acc[c][2 * q + 1] = fma_f2(x.y, w[c], acc[c][2 * q + 1]);
          }
        }
      }
    }
  }
  // The warps' sums in their order, half of the tokens at a time: [warps][TT / 4][128] pairs where the columns of a were.
  constexpr int PAIRS = TT / 4;
  uint64_t* s_sum = reinterpret_cast<uint64_t*>(s_a);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    __syncthreads();
#pragma unroll
    for (int t = 0; t < PAIRS; ++t)
#pragma unroll
      for (int c = 0; c < 4; ++c) s_sum[(warp * PAIRS + t) * FEW_OUTER_COLS + lane + 32 * c] = acc[c][half * PAIRS + t];
    __syncthreads();
    for (int i = threadIdx.x; i < PAIRS * FEW_OUTER_COLS; i += FEW_THREADS) {
      const int t = 2 * (half * PAIRS + i / FEW_OUTER_COLS), col = first + i % FEW_OUTER_COLS;
      uint64_t sum = s_sum[i];
#pragma unroll
      for (int w = 1; w < FEW_WARPS; ++w) sum = add_f2(sum, s_sum[w * PAIRS * FEW_OUTER_COLS + i]);
      float lo, hi;
      unpack_f2(sum, lo, hi);
      if (t < T && col < N) out[slice * plane + t * ldo + col] = lo;
      if (t + 1 < T && col < N) out[slice * plane + (t + 1) * ldo + col] = hi;
    }
  }
}

// out[slice][t, n] = sum over the slice's k of a[t, k] b[n, k]: a warp has four n, its lanes neighbouring k.
template <int TT>
__global__ void __launch_bounds__(FEW_THREADS, TT == 4 ? 4 : TT == 8 ? 3 : 2)
    few_inner_kernel(const float* a, long long lda, const float* b, long long ldb, int T, int K, int N, int slices, float* out, long long ldo,
                     long long plane) {
  __shared__ __align__(16) float2 s_a[TT / 2][FEW_CHUNK];
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slice = blockIdx.y, n0 = blockIdx.x * FEW_INNER_COLS + warp * 4;
  const bool whole = n0 + 4 <= N;
  const int k0 = static_cast<int>(static_cast<long long>(K) * slice / slices), k1 = static_cast<int>(static_cast<long long>(K) * (slice + 1) / slices);
  constexpr int U = 4, STEP = 32 * U;
  uint64_t acc[TT / 2][4];  // of two tokens each
#pragma unroll
  for (int t = 0; t < TT / 2; ++t)
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[t][c] = 0;
  for (int kc = k0; kc < k1; kc += FEW_CHUNK) {
    const int n = min(FEW_CHUNK, k1 - kc);
    __syncthreads();
    for (int k = threadIdx.x; k < FEW_CHUNK; k += FEW_THREADS)
#pragma unroll
      for (int t = 0; t < TT; t += 2)
        s_a[t / 2][k] = make_float2(t < T && k < n ? a[t * lda + kc + k] : 0.f, t + 1 < T && k < n ? a[(t + 1) * lda + kc + k] : 0.f);
    __syncthreads();
    const float* from = b + static_cast<long long>(n0) * ldb + kc + lane;
    for (int k = 0; k < n; k += STEP, from += STEP) {
      float v[U][4];
      if (whole && k + STEP <= n) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int c = 0; c < 4; ++c) v[u][c] = from[c * ldb + 32 * u];
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int c = 0; c < 4; ++c) v[u][c] = k + lane + 32 * u < n && n0 + c < N ? from[c * ldb + 32 * u] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (k + 32 * u >= n) break;
        uint64_t w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = pack_f2(v[u][c], v[u][c]);
#pragma unroll
        for (int t = 0; t < TT / 2; ++t) {
          const uint64_t x = *reinterpret_cast<const uint64_t*>(&s_a[t][k + lane + 32 * u]);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[t][c] = fma_f2(x, w[c], acc[t][c]);
        }
      }
    }
  }
  // Sums over the lanes: in each step a lane keeps one half of its pairs and gives the other away; then it has pair lane of TT * 2, or
  // (fewer tokens) two or four lanes the same one.
  int left = TT * 2;
  uint64_t* flat = &acc[0][0];
  auto other = [](uint64_t v, int o) { return __shfl_xor_sync(0xffffffffu, static_cast<unsigned long long>(v), o); };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (left > 1) {
      left /= 2;
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        if (i >= left) break;
        const uint64_t give = lane & o ? flat[i] : flat[i + left], keep = lane & o ? flat[i + left] : flat[i];
        flat[i] = add_f2(keep, other(give, o));
      }
    } else {
      flat[0] = add_f2(flat[0], other(flat[0], o));
    }
  }
  const int pair = lane * (TT * 2) / 32, t = pair / 4 * 2, col = n0 + pair % 4;
  float lo, hi;
  unpack_f2(flat[0], lo, hi);
  if (t < T && col < N) out[slice * plane + t * ldo + col] = lo;
  if (t + 1 < T && col < N) out[slice * plane + (t + 1) * ldo + col] = hi;
}

// out[m, n] (+)= sum over the tokens of a[t, m] b[t, n]; keep_a, keep_b as above.  A block has 128 columns, whose values of b stay in
// registers, and every `groups`th FEW_OUT_ROWS rows.
constexpr int FEW_OUT_ROWS = 256;
template <int TT>
__global__ void __launch_bounds__(FEW_THREADS, 2)
    few_update_kernel(const float* a, long long lda, const float* keep_a, const float* b, long long ldb, const float* keep_b, int T, int M, int N,
                      float* out, long long ldo, int groups, int add) {
  __shared__ __align__(16) float s_a[FEW_OUT_ROWS * TT];
  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col_blocks = (N + FEW_OUTER_COLS - 1) / FEW_OUTER_COLS;
  const int first = static_cast<int>(blockIdx.x % col_blocks) * FEW_OUTER_COLS, n0 = first + lane;
  const bool whole = first + FEW_OUTER_COLS <= N;
  uint64_t v[4][TT / 2];
#pragma unroll
  for (int t = 0; t < TT; t += 2)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      auto at = [&](int t) { return t < T && n0 + 32 * c < N && (keep_b == nullptr || keep_b[t] != 0.f) ? b[t * ldb + n0 + 32 * c] : 0.f; };
      v[c][t / 2] = pack_f2(at(t), at(t + 1));
    }
  for (int m0 = static_cast<int>(blockIdx.x / col_blocks) * FEW_OUT_ROWS; m0 < M; m0 += groups * FEW_OUT_ROWS) {
    const int rows = min(FEW_OUT_ROWS, M - m0);
    __syncthreads();
    few_columns<TT>(s_a, a, lda, T, m0, rows, keep_a);
    __syncthreads();
    float* to = out + static_cast<long long>(m0 + warp) * ldo + n0;
    for (int m = warp; m < rows; m += FEW_WARPS, to += FEW_WARPS * ldo) {
      uint64_t acc[4] = {0, 0, 0, 0};
#pragma unroll
      for (int q = 0; q < TT / 4; ++q) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(s_a + m * TT + 4 * q);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = fma_f2(x.y, v[c][2 * q + 1], fma_f2(x.x, v[c][2 * q], acc[c]));
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float even, odd;
        unpack_f2(acc[c], even, odd);
        if (whole || n0 + 32 * c < N) to[32 * c] = add ? to[32 * c] + (even + odd) : even + odd;
      }
    }
  }
}

static Entries from_row(Entries e, long long row) {
  e.ids += row * e.ids_ld;
  if (e.kind != TARGETS) e.teacher = static_cast<const char*>(e.teacher) + row * e.teacher_ld * (e.kind == TEACHER_F32 ? 4 : 2);
  return e;
}
static RowTerms from_row(RowTerms t, long long row) {
  if (t.d_loss) t.d_loss += row * t.d_loss_stride;
  t.loss += row;
  if (t.lse) t.lse += row;
  return t;
}

// Warps and slices by the row's size alone: a warp per 4 KB (8 vectors a lane; 6471 x 5047 f32 58 us, with 16 warps 123), per
// 2 KB up to 8 KB (8192 x 2000 bf16 38, 45); rows beyond 64 KB in a cluster of up to 8 CTAs, of 8 warps up to 256 KB
// (1500 x 50000 f32 168; with 16 195), else of 16: 512 KB, and 1 MB with 16 vectors a lane.
// More CTAs share those warps while SMs are without one.  warps = 0: longer rows, which are read twice.
struct Share {
  int warps, slice, ctas, slots_log2;  // warps of a row, vectors of a warp, CTAs of a row, the entries' hash table
  size_t smem;                         // of a CTA
};
static Share choose_share(const void* z, long long ld, long long rows, int vocab, int size, int K) {
  const int vec = 16 / size;
  const bool on_grid = (reinterpret_cast<uintptr_t>(z) & 15) == 0 && (rows == 1 || ld * size % 16 == 0);
  const long long vecs = (static_cast<long long>(vocab) + (on_grid ? 1 : 2) * (vec - 1)) / vec;  // (wherever the row starts in its first)
  Share s = {};
  const int slice = vecs <= 512 ? 128 : 256;
  const int warps = vecs <= 16 * 256 ? static_cast<int>((vecs + slice - 1) / slice) : vecs <= 8 * 8 * 256 ? 8 : 16;  // of a CTA
  const long long ctas = (vecs + warps * 256 - 1) / (warps * 256);
  s.ctas = ctas <= 8 ? static_cast<int>(ctas) : 8;
  s.warps = warps * s.ctas;
  s.slice = static_cast<int>((vecs + s.warps - 1) / s.warps);
  if (s.slice > 512) return {};
  for (int c = s.ctas + 1; c <= 8 && rows * s.ctas < sm_count() && s.slice >= 64; ++c)
    if (s.warps % c == 0) s.ctas = c;
  s.slots_log2 = 5;
  while ((1 << s.slots_log2) < 8 * K) ++s.slots_log2;  // (8192 x 32768 with 64 random ids: 2 K slots 257 us, 4 K 223, 8 K 215)
  s.smem = static_cast<size_t>(ENTRY_BYTES) * K + (4u << s.slots_log2);  // at most 44 KB
  return s;
}

template <typename T, bool PIECES>
static int32_t launch_rows(const void* z, long long ld_z, const GradRows& g, long long rows, int vocab, const Entries& e,
                           const RowTerms& t, cudaStream_t stream) {
  ProfileScope ps(PROF_ELEMENTWISE, static_cast<double>(rows) * vocab * (sizeof(T) + (g.ptr ? (PIECES ? 6 : sizeof(T)) : 0)), stream);
  const Share share = choose_share(z, ld_z, rows, vocab, sizeof(T), e.K);
  if (share.warps == 0 || rows * share.ctas > INT32_MAX) {
    CDL_CUDA(launch_pdl(loss_row_kernel<T, PIECES>, dim3(static_cast<unsigned>(rows)), dim3(ROW_THREADS), 0, stream,
                        static_cast<const T*>(z), ld_z, g, vocab, e, t));
    return CDL_OK;
  }
  auto kernel = share.slice <= 256 ? loss_slices_kernel<T, 8, PIECES> : loss_slices_kernel<T, 16, PIECES>;
  // Rows that run at once: two CTAs of 16 warps, or as many threads in more, per SM.
  const long long ahead = static_cast<long long>(sm_count()) * (share.slice <= 256 ? 1024 : 512) / (share.warps * 32);
  CDL_CUDA(launch_pdl_cluster(kernel, dim3(static_cast<unsigned>(rows * share.ctas)), dim3(share.warps / share.ctas * 32), share.smem,
                              share.ctas, stream, static_cast<const T*>(z), ld_z, g, rows, ahead, vocab, share.slice, share.ctas,
                              share.slots_log2, e, t));
  return CDL_OK;
}

static int32_t prepare_entries(const Entries& e, long long rows, int vocab, float tau, int pieces, int* ids, unsigned short* first, float* p,
                               float* p_log_p, cudaStream_t stream) {
  static std::once_flag once[64];
  int dev = 0;
  CDL_CUDA(cudaGetDevice(&dev));
  cudaError_t err = cudaSuccess;
  constexpr size_t row_bytes = static_cast<size_t>(PREPARE_WARPS) * ENTRY_BYTES;
  std::call_once(once[dev & 63], [&] {
    err = cudaFuncSetAttribute(prepare_entries_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(row_bytes * MAX_ENTRIES));
  });
  if (err != cudaSuccess) return fail(CDL_ERR_CUDA, "cudaFuncSetAttribute failed: %s", cudaGetErrorString(err));
  CDL_CUDA(launch_pdl(prepare_entries_kernel, dim3(static_cast<unsigned>((rows + PREPARE_WARPS - 1) / PREPARE_WARPS)),
                      dim3(PREPARE_WARPS * 32), row_bytes * e.K, stream, e, rows, vocab, tau, pieces, ids, first, p, p_log_p));
  return CDL_OK;
}

static int32_t segments(long long rows, long long cols, dim3* grid) {
  const long long blocks = rows * ((cols + SEGMENT - 1) / SEGMENT);
  if (blocks > INT32_MAX) return fail(CDL_ERR_UNSUPPORTED, "linear loss: operand too large to be copied");
  *grid = dim3(static_cast<unsigned>(blocks));
  return CDL_OK;
}

// dst = src, of which dimension 1 is the nearer one in memory; bf16.
static int32_t copy(const cdl_tensor& src, const cdl_tensor& dst, cudaStream_t stream) {
  using bf = __nv_bfloat16;
  const long long rows = src.shape[0], cols = src.shape[1];
  ProfileScope ps(PROF_ELEMENTWISE, 4.0 * rows * cols, stream);
  if ((src.stride[1] == 1 || cols == 1) && (dst.stride[1] == 1 || cols == 1)) {
    const bool on_grid = (reinterpret_cast<uintptr_t>(dst.ptr) & 15) == 0 && (rows == 1 || dst.stride[0] % 8 == 0);
    const long long per_row = (cols + (on_grid ? 7 : 14)) / 8, all = rows * per_row, blocks = (all + 256 * COPY_VECS - 1) / (256 * COPY_VECS);
    if (blocks > INT32_MAX) return fail(CDL_ERR_UNSUPPORTED, "linear loss: operand too large to be copied");
    CDL_CUDA(launch_pdl(copy_rows_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, static_cast<const bf*>(src.ptr),
                        static_cast<long long>(src.stride[0]), static_cast<bf*>(dst.ptr), static_cast<long long>(dst.stride[0]),
                        static_cast<int>(cols), static_cast<unsigned>(per_row), all));
    return CDL_OK;
  }
  dim3 grid;
  CDL_CHECK(segments(rows, cols, &grid));
  CDL_CUDA(launch_pdl(copy_kernel<bf>, grid, dim3(256), 0, stream, static_cast<const bf*>(src.ptr), static_cast<long long>(src.stride[0]),
                      static_cast<long long>(src.stride[1]), static_cast<bf*>(dst.ptr), static_cast<long long>(dst.stride[0]),
                      static_cast<long long>(dst.stride[1]), static_cast<int>(cols)));
  return CDL_OK;
}

static int32_t split(const cdl_tensor& src, void* dst, long long ld, long long plane, const float* keep, cudaStream_t stream) {
  dim3 grid;
  CDL_CHECK(segments(src.shape[0], src.shape[1], &grid));
  ProfileScope ps(PROF_ELEMENTWISE, 10.0 * src.shape[0] * src.shape[1], stream);
  CDL_CUDA(launch_pdl(split_kernel, grid, dim3(256), 0, stream, static_cast<const float*>(src.ptr), static_cast<long long>(src.stride[0]),
                      static_cast<long long>(src.stride[1]), static_cast<__nv_bfloat16*>(dst), ld, plane, static_cast<int>(src.shape[1]), keep));
  return CDL_OK;
}

// out (dimension 1 the threads' direction) = the sum of f32 planes.
template <typename T>
static int32_t sum_planes_as(const void* planes, long long ld, long long plane, int slices, const cdl_tensor& out, int add, cudaStream_t stream) {
  const long long rows = out.shape[0], cols = out.shape[1], all = rows * (cols / 4);
  const bool vectors = slices > 0 && cols % 4 == 0 && out.stride[1] == 1 && ld % 4 == 0 && plane % 4 == 0 &&
                       reinterpret_cast<uintptr_t>(out.ptr) % (4 * sizeof(T)) == 0 && (rows == 1 || out.stride[0] % 4 == 0);
  if (vectors && (all + 127) / 128 <= INT32_MAX) {
    CDL_CUDA(launch_pdl(sum_vectors_kernel<T>, dim3(static_cast<unsigned>((all + 127) / 128)), dim3(128), 0, stream,
                        static_cast<const float*>(planes), ld, plane, slices, static_cast<T*>(out.ptr),
                        static_cast<long long>(out.stride[0]), all, static_cast<int>(cols), add));
    return CDL_OK;
  }
  dim3 grid;
  CDL_CHECK(segments(rows, cols, &grid));
  CDL_CUDA(launch_pdl(sum_planes_kernel<T>, grid, dim3(256), 0, stream, static_cast<const float*>(planes), ld, plane, slices,
                      static_cast<T*>(out.ptr), static_cast<long long>(out.stride[0]), static_cast<long long>(out.stride[1]),
                      static_cast<int>(cols), add));
  return CDL_OK;
}
static int32_t sum_planes(const void* planes, long long ld, long long plane, int slices, const cdl_tensor& out, int add, cudaStream_t stream) {
  ProfileScope ps(PROF_ELEMENTWISE, static_cast<double>(out.shape[0]) * out.shape[1] * (4 * slices + dtype_size(out.dtype)), stream);
  return out.dtype == CDL_BF16 ? sum_planes_as<__nv_bfloat16>(planes, ld, plane, slices, out, add, stream)
                               : sum_planes_as<float>(planes, ld, plane, slices, out, add, stream);
}

// ------------------------------------------------------------------------------------------ checks
static bool is_float(int32_t t) { return t == CDL_BF16 || t == CDL_F32; }

static int32_t check_desc(const char* op, const cdl_head_loss_desc* d) {
  if (!d) return fail(CDL_ERR_INVALID, "%s: desc is required", op);
  if (!(d->temperature >= 1e-6f && d->temperature <= 1e6f))  // (its square and log2(e) over it are factors)
    return fail(CDL_ERR_INVALID, "%s: temperature must be positive, from 1e-6 to 1e6", op);
  if (d->chunk_rows < 0) return fail(CDL_ERR_INVALID, "%s: chunk_rows must not be negative", op);
  return CDL_OK;
}

static int32_t check_row_values(const char* op, const char* name, const cdl_tensor* t, long long rows, int32_t type, bool packed) {
  if (t->rank != 1 || t->dtype != type || t->shape[0] != rows || (packed && rows > 1 && t->stride[0] != 1))
    return fail(CDL_ERR_INVALID, "%s: %s must be %s%s [tokens]", op, name, packed ? "packed " : "", dtype_name(type));
  return CDL_OK;
}

static int32_t check_terms(const char* op, const cdl_head_loss_desc* desc, long long rows, const cdl_tensor* d_loss,
                           const cdl_tensor* loss, const cdl_tensor* lse, RowTerms* out) {
  if (!loss) return fail(CDL_ERR_INVALID, "%s: loss is required", op);
  CDL_CHECK(check_row_values(op, "loss", loss, rows, CDL_F32, true));
  if (lse) CDL_CHECK(check_row_values(op, "lse", lse, rows, CDL_F32, true));
  if (d_loss) CDL_CHECK(check_row_values(op, "d_loss", d_loss, rows, CDL_F32, false));
  *out = {d_loss ? static_cast<const float*>(d_loss->ptr) : nullptr, d_loss ? (long long)d_loss->stride[0] : 0,
          static_cast<float*>(loss->ptr), lse ? static_cast<float*>(lse->ptr) : nullptr, desc->grad_scale, desc->temperature};
  return CDL_OK;
}

static int32_t check_targets(const char* op, long long rows, const cdl_tensor* targets, Entries* out) {
  if (!targets) return fail(CDL_ERR_INVALID, "%s: targets are required", op);
  CDL_CHECK(check_row_values(op, "targets", targets, rows, CDL_I32, true));
  *out = {static_cast<const int*>(targets->ptr), nullptr, 1, 0, 1, TARGETS};
  return CDL_OK;
}

static int32_t check_teacher(const char* op, long long rows, const cdl_tensor* ids, const cdl_tensor* teacher, Entries* out) {
  if (!ids || !teacher) return fail(CDL_ERR_INVALID, "%s: teacher_ids and teacher_logits are required", op);
  const long long K = ids->rank == 2 ? ids->shape[1] : -1;
  if (ids->rank != 2 || ids->dtype != CDL_I32 || ids->shape[0] != rows || (K > 1 && ids->stride[1] != 1))
    return fail(CDL_ERR_INVALID, "%s: teacher_ids must be i32 [tokens, entries] with contiguous rows", op);
  if (teacher->rank != 2 || !is_float(teacher->dtype) || teacher->shape[0] != rows || teacher->shape[1] != K ||
      (K > 1 && teacher->stride[1] != 1))
    return fail(CDL_ERR_INVALID, "%s: teacher_logits must be bf16 or f32 [tokens, entries] like teacher_ids, with contiguous rows", op);
  if (K > MAX_ENTRIES) return fail(CDL_ERR_UNSUPPORTED, "%s: at most %d entries per token (got %lld)", op, MAX_ENTRIES, K);
  *out = {static_cast<const int*>(ids->ptr), teacher->ptr, ids->stride[0], teacher->stride[0], static_cast<int>(K),
          teacher->dtype == CDL_F32 ? TEACHER_F32 : TEACHER_BF16};
  return CDL_OK;
}

// ------------------------------------------------------------------------------------------ from the logits
static int32_t distillation_execute(const cdl_head_loss_desc* desc, const cdl_tensor* logits, const cdl_tensor* ids,
                                    const cdl_tensor* teacher, const cdl_tensor* d_loss, const cdl_tensor* loss,
                                    const cdl_tensor* lse, const cdl_tensor* d_logits, cudaStream_t stream) {
  const char* op = "distillation";
  CDL_CHECK(check_desc(op, desc));
  if (!logits || logits->rank != 2 || !is_float(logits->dtype))
    return fail(CDL_ERR_INVALID, "%s: logits must be bf16 or f32 [tokens, vocab]", op);
  const long long T = logits->shape[0], V = logits->shape[1];
  if (V > 1 && logits->stride[1] != 1) return fail(CDL_ERR_INVALID, "%s: logits must have contiguous rows", op);
  if (T > INT32_MAX || V > MAX_DIM) return fail(CDL_ERR_UNSUPPORTED, "%s: dimension too large", op);
  RowTerms terms;
  Entries e;
  CDL_CHECK(check_teacher(op, T, ids, teacher, &e));
  CDL_CHECK(check_terms(op, desc, T, d_loss, loss, lse, &terms));
  if (d_logits) {
    if (d_logits->rank != 2 || d_logits->dtype != logits->dtype || d_logits->shape[0] != T || d_logits->shape[1] != V ||
        (V > 1 && d_logits->stride[1] != 1))
      return fail(CDL_ERR_INVALID, "%s: d_logits must have the logits' type and shape and contiguous rows", op);
    if (T > 1 && d_logits->stride[0] < V) return fail(CDL_ERR_INVALID, "%s: rows of d_logits overlap", op);
    if (d_logits->ptr == logits->ptr && T > 1 && d_logits->stride[0] != logits->stride[0])
      return fail(CDL_ERR_INVALID, "%s: d_logits must be the logits themselves or lie elsewhere", op);
  }
  if (T == 0) return CDL_OK;
  if (V == 0) return fail(CDL_ERR_INVALID, "%s: vocab is zero", op);
  auto rows = logits->dtype == CDL_BF16 ? launch_rows<__nv_bfloat16, false> : launch_rows<float, false>;
  const GradRows g = {d_logits ? d_logits->ptr : nullptr, d_logits ? static_cast<long long>(d_logits->stride[0]) : 0, 0};
  return rows(logits->ptr, logits->stride[0], g, T, static_cast<int>(V), e, terms, stream);
}

// ------------------------------------------------------------------------------------------ from the hidden states

// Whether products read and write a bf16 or f32 [rows, cols] view where it is: one dimension contiguous, the other on the
// 16-byte grid.
static bool on_grid(const cdl_tensor& t) {
  const long long r = t.shape[0], c = t.shape[1], sr = t.stride[0], sc = t.stride[1], unit = t.dtype == CDL_BF16 ? 8 : 4;
  if (reinterpret_cast<uintptr_t>(t.ptr) & 15) return false;
  return ((sc == 1 || c == 1) && (r == 1 || (sr % unit == 0 && sr >= c))) || ((sr == 1 || r == 1) && (c == 1 || (sc % unit == 0 && sc >= r)));
}
static bool columns_first(const cdl_tensor& t) { return t.stride[0] < t.stride[1]; }  // dimension 0 is the nearer one in memory

// The stride of a dimension of extent 1, which may be any, becomes the one that columns_first and on_grid read alike: a view on
// the grid then has neighbouring elements along its nearer dimension.
static void settle_strides(cdl_tensor& t) {
  if (t.shape[1] == 1) t.stride[1] = t.shape[0] > 1 && t.stride[0] == 1 ? t.shape[0] : 1;
  if (t.shape[0] == 1) t.stride[0] = t.stride[1] == 1 ? t.shape[1] : 1;
}

struct Linear {
  const char* op;
  cdl_tensor x, w, dx, dw;  // dx, dw: ptr = nullptr where not wanted
  bool has_dx, has_dw, f32;
  long long T, D, V;
  int K;
  // Scratch.  Rows are taken `chunk` at a time.
  long long chunk, ld_x, ld_w, ld_g, ld_sum;
  bool copy_x, copy_w;
  // Few rows of bf16 operands: the bytes of w and dw set the products' time, which take d z as two bf16 pieces then, one below
  // the other: [2 rows, V], the rows of x twice.  With one piece dx and dw are 1.4 times as far off as their own rounding
  // to bf16, give or take what the rounding of a single row's largest value happens to be.
  bool twice;
  bool few;  // few rows of f32 operands
  enum { DIRECT, HELD, SUMMED } dw_way;  // the product stores dw; a bf16 dw off the grid, stored beside it first; an f32 sum over the chunks
  int pieces, slices_z, slices_dx, slices_dw;  // pieces: of the vocabulary, 128 columns each
  size_t at_x, at_w, at_clean, at_keep, at_z, at_g, at_stats, at_ids, at_first, at_p, at_p_log_p, at_at, at_planes, at_sum, bytes;
};

// A view of `rows` rows from `row`.
static cdl_tensor rows_of(const cdl_tensor& t, long long row, long long rows) {
  cdl_tensor o = t;
  o.ptr = static_cast<char*>(t.ptr) + row * t.stride[0] * static_cast<long long>(dtype_size(t.dtype));
  o.shape[0] = rows;
  return o;
}

static cdl_tensor strided2(void* p, int32_t dt, long long r, long long c, long long ld) {
  cdl_tensor t = view2(p, dt, r, c);
  t.stride[0] = ld;
  return t;
}

constexpr long long TARGET_ENTRIES = -1;

// Rows that are taken at a time: up to 1 GB of what grows with them and the vocabulary, but 256 rows at least (w is read once per
// chunk).  16384 x 2048 x 32768 in one go 4.83 ms, in two 5.01: dw is summed in memory then, dx's last wave is emptier.
static long long choose_chunk(long long T, long long bytes_per_row) {
  long long rows = (1LL << 30) / bytes_per_row;
  if (rows < 256) rows = 256;
  if (rows >= T) return T;
  const long long chunks = (T + rows - 1) / rows;
  return up((T + chunks - 1) / chunks, 256);
}

// K slices of a product of few rows, of 512 and more: where there are fewer than four blocks per SM as many as give twelve (two to
// four run at once, and the last ones alone: 5 x 3198 x 102440 with slices for four 912 us, for twelve 792).
static int few_slices(bool inner, long long K, long long N) {
  const int cols = inner ? FEW_INNER_COLS : FEW_OUTER_COLS;
  const long long blocks = (N + cols - 1) / cols, want = blocks < 4 * sm_count() ? 12LL * sm_count() / blocks : 1, most = K / FEW_CHUNK;
  const long long s = want < most ? want : most;
  return s < 1 ? 1 : s > MAX_PLANES ? MAX_PLANES : static_cast<int>(s);
}

static void plan_linear(Linear& p, const cdl_head_loss_desc* desc, long long entries) {
  const bool grad = p.has_dx || p.has_dw, teacher = entries != TARGET_ENTRIES;
  p.f32 = p.x.dtype == CDL_F32;
  p.K = static_cast<int>(entries);
  p.pieces = static_cast<int>(up(p.V, 128) / 128);
  p.copy_x = (reinterpret_cast<uintptr_t>(p.x.ptr) & 15) != 0 || (p.D > 1 && p.x.stride[1] != 1) ||  // (chunks of its rows are on the grid)
             (p.T > 1 && (p.x.stride[0] % 8 != 0 || p.x.stride[0] < p.D));
  p.copy_w = !on_grid(p.w);
  // f32: logits and the pieces of their gradients, or of x; bf16: exponentials, for the loss alone statistics and entries (a target
  // as one entry: the scratch's size is asked for without saying which it is).
  const long long ld = up(p.V, 128), row_bytes = p.f32 ? (grad ? 10 * ld : 4 * ld + 6 * up(p.D, 8))
                                                 : grad ? 2 * ld : 10LL * p.pieces + 12LL * (p.K > 1 ? p.K : 1) + 6;
  p.chunk = desc->chunk_rows > 0 ? desc->chunk_rows : choose_chunk(p.T, row_bytes);
  if (p.chunk > p.T) p.chunk = p.T;
  const bool whole = p.chunk >= p.T, wc = columns_first(p.w), dc = p.has_dw && columns_first(p.dw);
  p.dw_way = Linear::DIRECT;
  p.twice = !p.f32 && grad && whole && p.T <= 64;
  const size_t n = static_cast<size_t>(p.chunk), g_rows = p.twice ? 2 * n : n;
  if (p.has_dw && !(on_grid(p.dw) && (p.dw.dtype == CDL_F32 || whole))) {
    const cdl_tensor near = dc ? transposed(p.dw) : p.dw;
    p.dw_way = p.dw.dtype != CDL_BF16 || !whole || desc->accumulate_dw                                          ? Linear::SUMMED
               : matmul_store_bound(near.shape[0], near.shape[1], static_cast<long long>(g_rows), &near) ? Linear::DIRECT
                                                                                                                : Linear::HELD;
  }
  p.ld_x = up(p.D, 8);
  p.ld_w = up(wc ? p.D : p.V, 8);
  p.ld_g = up(p.V, 128);
  p.ld_sum = p.has_dw ? up(dc ? p.D : p.V, 8) : 0;
  auto near = [](const cdl_tensor& t) {  // a row's elements lie next to one another
    const cdl_tensor n = columns_first(t) ? transposed(t) : t;
    return n.stride[1] == 1 || n.shape[1] == 1;
  };
  p.few = p.f32 && whole && p.T <= FEW_ROWS && (p.x.stride[1] == 1 || p.D == 1) && near(p.w) && (!p.has_dw || near(p.dw));
  if (p.few) {
    p.dw_way = Linear::DIRECT;
    p.slices_z = few_slices(wc, p.D, p.V);
    p.slices_dx = p.has_dx ? few_slices(!wc, p.V, p.D) : 1;
    size_t at = 0;
    auto take = [&](size_t bytes) {
      const size_t here = at;
      at += (bytes + 255) / 256 * 256;
      return here;
    };
    p.at_z = take(n * p.ld_g * 4);
    p.at_keep = take(n * 4);
    const size_t z = p.slices_z > 1 ? p.slices_z * n * up(p.V, 4) : 0, dx = p.slices_dx > 1 ? p.slices_dx * n * up(p.D, 4) : 0;
    p.at_planes = take(4 * (z > dx ? z : dx));
    p.bytes = at;
    return;
  }
  p.slices_z = p.f32 ? matmul_plane_slices(p.chunk, p.V, p.D, true) : 1;
  p.slices_dx = p.has_dx ? matmul_plane_slices(static_cast<long long>(g_rows), p.D, p.V, p.f32) : 1;
  p.slices_dw = p.has_dw && p.f32 ? matmul_plane_slices(dc ? p.V : p.D, dc ? p.D : p.V, p.chunk, true) : 1;
  size_t at = 0;
  auto take = [&](bool want, size_t bytes) {
    const size_t here = at;
    if (want) at += (bytes + 255) / 256 * 256;
    return here;
  };
  const size_t w_rows = wc ? p.V : p.D, dw_rows = dc ? p.V : p.D;
  if (p.f32) {
    p.at_x = take(true, 3 * n * p.ld_x * 2);
    p.at_w = take(true, 3 * w_rows * p.ld_w * 2);
    p.at_clean = take(p.has_dw, 3 * n * p.ld_x * 2);
    p.at_keep = take(p.has_dw, n * 4);
    p.at_z = take(true, n * p.ld_g * 4);
    p.at_g = take(grad, 3 * n * p.ld_g * 2);
  } else {
    p.at_x = take(p.copy_x, static_cast<size_t>(p.T) * p.ld_x * 2);
    p.at_w = take(p.copy_w, w_rows * p.ld_w * 2);
    p.at_clean = take(p.has_dw, g_rows * p.ld_x * 2);
    p.at_g = take(grad, g_rows * p.ld_g * 2);
    p.at_stats = take(true, n * p.pieces * sizeof(float2));
    p.at_at = take(true, n * (teacher ? p.K : 1) * 4);
    p.at_ids = take(teacher, n * p.K * 4);
    p.at_p = take(teacher, n * p.K * 4);
    p.at_p_log_p = take(teacher, n * 4);
    p.at_first = take(teacher, n * (p.pieces + 1) * 2);
  }
  size_t planes = 0;
  auto need = [&](int slices, size_t rows, size_t ld) {
    if (slices > 1 && slices * rows * ld * 4 > planes) planes = slices * rows * ld * 4;
  };
  need(p.slices_z, n, p.ld_g);
  need(p.twice ? 2 * p.slices_dx : p.slices_dx, n, p.ld_x);
  need(p.slices_dw, dw_rows, p.ld_sum);
  p.at_planes = take(planes != 0, planes);
  p.at_sum = take(p.dw_way != Linear::DIRECT, dw_rows * p.ld_sum * (p.dw_way == Linear::SUMMED ? 4 : 2));
  p.bytes = at;
}

static int32_t check_linear(const char* op, const cdl_head_loss_desc* desc, const cdl_tensor* x, const cdl_tensor* w,
                            const cdl_tensor* dx, const cdl_tensor* dw, long long entries, Linear* out) {
  CDL_CHECK(check_desc(op, desc));
  if (!x || !w || x->rank != 2 || w->rank != 2 || !is_float(x->dtype) || x->dtype != w->dtype)
    return fail(CDL_ERR_INVALID, "%s: x must be bf16 or f32 [tokens, hidden], w of the same type [hidden, vocab]", op);
  Linear& p = *out;
  p = Linear{};
  p.op = op;
  p.x = *x;
  p.w = *w;
  settle_strides(p.w);
  p.T = x->shape[0];
  p.D = x->shape[1];
  p.V = w->shape[1];
  p.has_dx = dx != nullptr;
  p.has_dw = dw != nullptr;
  if (w->shape[0] != p.D)
    return fail(CDL_ERR_INVALID, "%s: x is [tokens, %lld], w is [%lld, vocab]: the hidden sizes differ", op, p.D, (long long)w->shape[0]);
  if (p.T > INT32_MAX || p.D > MAX_DIM || p.V > 65535LL * 8 * 128) return fail(CDL_ERR_UNSUPPORTED, "%s: dimension too large", op);
  if (dx) {
    if (dx->rank != 2 || dx->dtype != x->dtype || dx->shape[0] != p.T || dx->shape[1] != p.D || (p.D > 1 && dx->stride[1] != 1) ||
        (p.T > 1 && dx->stride[0] < p.D))
      return fail(CDL_ERR_INVALID, "%s: dx must have x's type and shape and contiguous rows that do not overlap", op);
    // (a chunk's rows of dx are written before the next chunk's rows of x are read)
    if (p.T > 0 && dx->ptr == x->ptr && ((p.T > 1 && dx->stride[0] != x->stride[0]) || (p.D > 1 && dx->stride[1] != x->stride[1])))
      return fail(CDL_ERR_INVALID, "%s: dx must be x itself or lie elsewhere", op);
    p.dx = *dx;
  }
  if (dw) {
    const long long a = dw->rank == 2 ? dw->stride[0] : 0, b = dw->rank == 2 ? dw->stride[1] : 0;
    if (dw->rank != 2 || !(dw->dtype == CDL_F32 || dw->dtype == x->dtype) || dw->shape[0] != p.D || dw->shape[1] != p.V)
      return fail(CDL_ERR_INVALID, "%s: dw must be [hidden, vocab] in f32 or x's type", op);
    const bool apart = p.D == 0 || p.V == 0 ? true : a <= 0 || b <= 0 ? (p.D <= 1 || a > 0) && (p.V <= 1 || b > 0)
                                        : a < b ? (p.V <= 1 || b >= (p.D - 1) * a + 1) : (p.D <= 1 || a >= (p.V - 1) * b + 1);
    if (!apart) return fail(CDL_ERR_INVALID, "%s: elements of dw overlap", op);
    p.dw = *dw;
    settle_strides(p.dw);
  }
  if (p.V == 0 && p.T > 0) return fail(CDL_ERR_INVALID, "%s: vocab is zero", op);
  if (p.D == 0 && p.T > 0) return fail(CDL_ERR_INVALID, "%s: hidden is zero", op);
  if (p.T > 0) plan_linear(p, desc, entries);
  return CDL_OK;
}

// The statistics, losses and logits' gradients of a chunk of rows of bf16 operands on the 16-byte grid.
static int32_t fused_rows(const Linear& p, const cdl_tensor& x, const cdl_tensor& w, const Entries& e, const RowTerms& t,
                          const cdl_tensor& clean, char* base, bool grad, cudaStream_t stream) {
  const int rows = static_cast<int>(x.shape[0]), vocab = static_cast<int>(p.V);
  const bool teacher = e.kind != TARGETS;
  float2* stats = reinterpret_cast<float2*>(base + p.at_stats);
  float* at = reinterpret_cast<float*>(base + p.at_at);
  int* ids = reinterpret_cast<int*>(base + p.at_ids);
  float *probs = reinterpret_cast<float*>(base + p.at_p), *p_log_p = reinterpret_cast<float*>(base + p.at_p_log_p);
  unsigned short* first = reinterpret_cast<unsigned short*>(base + p.at_first);
  const Prepared src = teacher ? Prepared{ids, e.K, first, probs, p_log_p, at} : Prepared{e.ids, e.ids_ld, nullptr, nullptr, nullptr, at};
  if (teacher)
    CDL_CHECK(prepare_entries(e, rows, vocab, t.tau, p.pieces, ids, first, probs, p_log_p, stream));
  void* out = grad ? base + p.at_g : nullptr;
  const float c = matmul_exp_scale(LOG2E / t.tau, p.D);
  CDL_CHECK(matmul_exp_execute(&x, &w, c, out, p.ld_g, {stats, src.ids, src.ids_ld, src.first, at}, stream));
  ProfileScope ps(PROF_ELEMENTWISE, static_cast<double>(rows) * vocab * (grad ? 4 : 0) + 8.0 * rows * p.pieces, stream);
  const dim3 block(ROWS_PER_CTA * 32);
  const unsigned row_ctas = (rows + ROWS_PER_CTA - 1) / ROWS_PER_CTA;
  auto run = [&](auto kernel, unsigned splits, int per) {
    return launch_pdl(kernel, dim3(row_ctas, splits), block, 0, stream, stats, c, static_cast<__nv_bfloat16*>(out), p.ld_g, rows,
                      vocab, p.pieces, per, e.K, src, t, static_cast<const __nv_bfloat16*>(x.ptr), static_cast<long long>(x.stride[0]),
                      p.has_dw ? static_cast<__nv_bfloat16*>(clean.ptr) : nullptr, static_cast<long long>(clean.stride[0]),
                      static_cast<int>(p.D));
  };
  if (!grad) {
    CDL_CUDA(run(softmax_rows_kernel<LOSS_ONLY>, 1, p.pieces));
    return CDL_OK;
  }
  int per = PIECES_PER_WARP;  // fewer where that leaves SMs without a CTA
  while (per > 8 && row_ctas * ((p.pieces + per - 1) / per) < 2u * sm_count()) per /= 2;
  const unsigned splits = (p.pieces + per - 1) / per;
  CDL_CUDA(p.twice ? run(softmax_rows_kernel<GRAD_TWICE>, splits, per) : run(softmax_rows_kernel<GRAD_ONCE>, splits, per));
  return CDL_OK;
}

// [3][rows][cols] pieces (ld), planes `plane` apart; transposed: [3][cols][rows] views of them.
static cdl_tensor pieces3(void* ptr, long long rows, long long cols, long long ld, long long plane, bool transpose = false) {
  cdl_tensor t{};
  t.ptr = ptr;
  t.dtype = CDL_BF16;
  t.rank = 3;
  t.shape[0] = 3;
  t.stride[0] = plane;
  t.shape[transpose ? 2 : 1] = rows;
  t.stride[transpose ? 2 : 1] = ld;
  t.shape[transpose ? 1 : 2] = cols;
  t.stride[transpose ? 1 : 2] = 1;
  return t;
}

// D (+)= A B of pieces, by way of planes if there are slices.
static int32_t pieces_product(const Linear& p, const cdl_tensor& a, const cdl_tensor& b, const cdl_tensor& d, int slices, int add, char* base,
                              cudaStream_t stream) {
  const long long M = d.shape[0], N = d.shape[1], ld = up(N, 8), k_blocks = (a.shape[2] + 63) / 64;
  if (slices > k_blocks) slices = static_cast<int>(k_blocks);  // (the last rows are fewer)
  if (slices == 1)  // (D's rows are neighbouring elements, here and in its planes)
    return matmul_pieces_execute(&a, &b, static_cast<float*>(d.ptr), M > 1 ? d.stride[0] : ld, 1, add, stream);
  float* planes = reinterpret_cast<float*>(base + p.at_planes);
  CDL_CHECK(matmul_pieces_execute(&a, &b, planes, ld, slices, 0, stream));
  return sum_planes(planes, ld, M * ld, slices, d, add, stream);
}

// out [T, N] = a [T, K] times w, of which N (inner: K) is the nearer dimension in memory, by way of planes if there are slices.
static int32_t few_product(const Linear& p, const float* a, long long lda, const cdl_tensor& w_near, bool inner, int slices, const cdl_tensor& out,
                           char* base, cudaStream_t stream) {
  const long long N = inner ? w_near.shape[0] : w_near.shape[1], K = inner ? w_near.shape[1] : w_near.shape[0];
  const long long ldo = slices > 1 ? up(N, 4) : static_cast<long long>(out.stride[0]), plane = p.T * up(N, 4);
  float* to = slices > 1 ? reinterpret_cast<float*>(base + p.at_planes) : static_cast<float*>(out.ptr);
  auto run = [&](auto kernel) -> int32_t {
    const int cols = inner ? FEW_INNER_COLS : FEW_OUTER_COLS;
    const long long blocks = (N + cols - 1) / cols;
    ProfileScope ps(PROF_GEMM, 2.0 * p.T * K * N, stream);
    CDL_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(blocks), slices), dim3(FEW_THREADS), 0, stream, a, lda,
                        static_cast<const float*>(w_near.ptr), static_cast<long long>(w_near.stride[0]), static_cast<int>(p.T),
                        static_cast<int>(K), static_cast<int>(N), slices, to, ldo, plane));
    return CDL_OK;
  };
  if (p.T <= 4) CDL_CHECK(inner ? run(few_inner_kernel<4>) : run(few_outer_kernel<4>));
  else if (p.T <= 8) CDL_CHECK(inner ? run(few_inner_kernel<8>) : run(few_outer_kernel<8>));
  else CDL_CHECK(inner ? run(few_inner_kernel<16>) : run(few_outer_kernel<16>));
  return slices > 1 ? sum_planes(to, ldo, plane, slices, out, 0, stream) : CDL_OK;
}

static int32_t few_execute(Linear& p, const cdl_head_loss_desc* desc, const Entries& e, const RowTerms& terms, char* base, cudaStream_t stream) {
  const bool wc = columns_first(p.w), dc = p.has_dw && columns_first(p.dw);
  const int T = static_cast<int>(p.T), vocab = static_cast<int>(p.V);
  const cdl_tensor w_near = wc ? transposed(p.w) : p.w, z = strided2(base + p.at_z, CDL_F32, p.T, p.V, p.ld_g);
  const float *x = static_cast<const float*>(p.x.ptr), *g = static_cast<const float*>(z.ptr);
  CDL_CHECK(few_product(p, x, p.x.stride[0], w_near, wc, p.slices_z, z, base, stream));
  const GradRows grad = {p.has_dx || p.has_dw ? z.ptr : nullptr, p.ld_g, 0};
  CDL_CHECK((launch_rows<float, false>(z.ptr, p.ld_g, grad, p.T, vocab, e, terms, stream)));
  if (p.has_dw) {  // (ahead of dx, which may be x; rows that do not count add nothing whatever x holds there)
    float* keep = reinterpret_cast<float*>(base + p.at_keep);
    CDL_CUDA(launch_pdl(keep_kernel, dim3((T + 7) / 8), dim3(256), 0, stream, e, p.T, vocab, keep));
    const cdl_tensor d = dc ? transposed(p.dw) : p.dw;
    const int M = static_cast<int>(d.shape[0]), N = static_cast<int>(d.shape[1]);
    auto run = [&](auto kernel) -> int32_t {
      // Six blocks per SM, or as many as there are: a block's columns of b take as long to come as 128 rows to leave.
      const int col_blocks = (N + FEW_OUTER_COLS - 1) / FEW_OUTER_COLS, most = (M + FEW_OUT_ROWS - 1) / FEW_OUT_ROWS;
      const int want = (6 * sm_count() + col_blocks - 1) / col_blocks, groups = want < most ? want : most;
      const long long blocks = static_cast<long long>(col_blocks) * groups;
      ProfileScope ps(PROF_GEMM, 2.0 * p.T * M * N, stream);
      CDL_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(blocks)), dim3(FEW_THREADS), 0, stream, dc ? g : x,
                          dc ? p.ld_g : static_cast<long long>(p.x.stride[0]), dc ? nullptr : keep, dc ? x : g,
                          dc ? static_cast<long long>(p.x.stride[0]) : p.ld_g, dc ? keep : nullptr, T, M, N, static_cast<float*>(d.ptr),
                          static_cast<long long>(d.stride[0]), groups, desc->accumulate_dw));
      return CDL_OK;
    };
    CDL_CHECK(T <= 4 ? run(few_update_kernel<4>) : T <= 8 ? run(few_update_kernel<8>) : run(few_update_kernel<16>));
  }
  if (p.has_dx) CDL_CHECK(few_product(p, g, p.ld_g, w_near, !wc, p.slices_dx, p.dx, base, stream));
  return CDL_OK;
}

static int32_t linear_execute(Linear& p, const cdl_head_loss_desc* desc, const Entries& entries, const RowTerms& terms, void* scratch,
                              size_t scratch_bytes, cudaStream_t stream) {
  const bool grad = p.has_dx || p.has_dw, wc = columns_first(p.w), dc = p.has_dw && columns_first(p.dw);
  const cdl_tensor dw_near = dc ? transposed(p.dw) : p.dw;  // dimension 1 the nearer one in memory
  if (p.T == 0) {  // no rows: no loss, and a gradient of zeros
    if (p.has_dw && !desc->accumulate_dw && p.D > 0 && p.V > 0) CDL_CHECK(sum_planes(nullptr, 0, 0, 0, dw_near, 0, stream));
    return CDL_OK;
  }
  if (p.bytes > 0 && (!scratch || scratch_bytes < p.bytes || (reinterpret_cast<uintptr_t>(scratch) & 255)))
    return fail(CDL_ERR_INVALID, "%s: scratch must hold %zu bytes, 256-byte aligned", p.op, p.bytes);
  const FixedWorkInGraph fixed_work(stream);
  char* base = static_cast<char*>(scratch);
  const int vocab = static_cast<int>(p.V);
  if (p.few) return few_execute(p, desc, entries, terms, base, stream);
  // Where dw's product goes, as [D, V] or (dc) [V, D].
  cdl_tensor dw = dw_near;
  if (p.dw_way != Linear::DIRECT)
    dw = strided2(base + p.at_sum, p.dw_way == Linear::SUMMED ? CDL_F32 : CDL_BF16, dc ? p.V : p.D, dc ? p.D : p.V, p.ld_sum);
  if (p.f32) {
    const cdl_tensor w_near = wc ? transposed(p.w) : p.w;
    const long long w_plane = w_near.shape[0] * p.ld_w, x_plane = p.chunk * p.ld_x, g_plane = p.chunk * p.ld_g;
    CDL_CHECK(split(w_near, base + p.at_w, p.ld_w, w_plane, nullptr, stream));
    const cdl_tensor w3 = pieces3(base + p.at_w, w_near.shape[0], w_near.shape[1], p.ld_w, w_plane, wc);    // [3][D][V]
    const cdl_tensor wt3 = pieces3(base + p.at_w, w_near.shape[0], w_near.shape[1], p.ld_w, w_plane, !wc);  // [3][V][D]
    for (long long row = 0; row < p.T; row += p.chunk) {
      const long long n = p.T - row < p.chunk ? p.T - row : p.chunk;
      const cdl_tensor xc = rows_of(p.x, row, n), z = strided2(base + p.at_z, CDL_F32, n, p.V, p.ld_g);
      const Entries e = from_row(entries, row);
      CDL_CHECK(split(xc, base + p.at_x, p.ld_x, x_plane, nullptr, stream));
      CDL_CHECK(pieces_product(p, pieces3(base + p.at_x, n, p.D, p.ld_x, x_plane), w3, z, p.slices_z, 0, base, stream));
      const GradRows g = {grad ? base + p.at_g : nullptr, p.ld_g, g_plane};
      CDL_CHECK((launch_rows<float, true>(z.ptr, p.ld_g, g, n, vocab, e, from_row(terms, row), stream)));
      if (!grad) continue;
      if (p.has_dw) {  // (the copy with zeros in rows that do not count, see below)
        float* keep = reinterpret_cast<float*>(base + p.at_keep);
        CDL_CUDA(launch_pdl(keep_kernel, dim3(static_cast<unsigned>((n + 7) / 8)), dim3(256), 0, stream, e, n, vocab, keep));
        CDL_CHECK(split(xc, base + p.at_clean, p.ld_x, x_plane, keep, stream));
      }
      if (p.has_dx)
        CDL_CHECK(pieces_product(p, pieces3(base + p.at_g, n, p.V, p.ld_g, g_plane), wt3, rows_of(p.dx, row, n), p.slices_dx, 0, base, stream));
      if (p.has_dw) {
        const bool add = row > 0 || (p.dw_way == Linear::DIRECT && desc->accumulate_dw);
        const cdl_tensor g3 = pieces3(base + p.at_g, n, p.V, p.ld_g, g_plane, dc), x3 = pieces3(base + p.at_clean, n, p.D, p.ld_x, x_plane, !dc);
        CDL_CHECK(pieces_product(p, dc ? g3 : x3, dc ? x3 : g3, dw, p.slices_dw, add, base, stream));
      }
    }
  } else {
    cdl_tensor x = p.x, w = p.w;
    if (p.copy_x) {
      x = strided2(base + p.at_x, CDL_BF16, p.T, p.D, p.ld_x);
      CDL_CHECK(copy(p.x, x, stream));
    }
    if (p.copy_w) {
      const cdl_tensor w_near = wc ? transposed(p.w) : p.w;
      w = strided2(base + p.at_w, CDL_BF16, w_near.shape[0], w_near.shape[1], p.ld_w);
      CDL_CHECK(copy(w_near, w, stream));
      if (wc) w = transposed(w);
    }
    const cdl_tensor wt = transposed(w);
    // Sums over the rows in a fixed order: the same gradient every time.
    cdl_matmul_options fixed = {CDL_GEMM_AUTO, 1};
    for (long long row = 0; row < p.T; row += p.chunk) {
      const long long n = p.T - row < p.chunk ? p.T - row : p.chunk;
      const long long g_rows = p.twice ? 2 * n : n;
      const cdl_tensor g = strided2(base + p.at_g, CDL_BF16, g_rows, p.V, p.ld_g);
      // A row that does not count adds nothing to dw whatever x holds there, infinities and NaN too, which a gradient of zeros
      // alone would not do: the product takes a copy of x with zeros in such rows (made before dx is written, which may
      // be x itself).
      const cdl_tensor clean = strided2(base + p.at_clean, CDL_BF16, g_rows, p.D, p.ld_x);
      CDL_CHECK(fused_rows(p, rows_of(x, row, n), w, from_row(entries, row), from_row(terms, row), clean, base, grad, stream));
      if (p.has_dx) {
        const cdl_tensor d = rows_of(p.dx, row, n);
        const int planes_per_slice = p.twice ? 2 : 1;
        if (p.slices_dx * planes_per_slice > 1) {
          float* planes = reinterpret_cast<float*>(base + p.at_planes);
          CDL_CHECK(matmul_planes_execute(&g, &wt, planes, p.ld_x, p.slices_dx, stream));
          CDL_CHECK(sum_planes(planes, p.ld_x, n * p.ld_x, p.slices_dx * planes_per_slice, d, 0, stream));
        } else {
          CDL_CHECK(matmul_execute(&g, &wt, nullptr, &d, 1.f, 0.f, stream));
        }
      }
      if (p.has_dw) {
        const bool add = row > 0 || (p.dw_way == Linear::DIRECT && desc->accumulate_dw);
        const cdl_tensor a = dc ? transposed(g) : transposed(clean), &b = dc ? clean : g;
        // (beside the kernel ahead, dx's, whose last wave leaves SMs idle: the two share what they read alone)
        const int early = p.has_dx ? 1 : 0;
        if (!add && matmul_store_bound(dw.shape[0], dw.shape[1], a.shape[1], &dw)) CDL_CHECK(matmul_store_execute(&a, &b, &dw, stream, early));
        else CDL_CHECK(matmul_execute(&a, &b, add ? &dw : nullptr, &dw, 1.f, add ? 1.f : 0.f, stream, &fixed, nullptr, 0, early));
      }
    }
  }
  if (p.has_dw && p.dw_way == Linear::HELD) CDL_CHECK(copy(dw, dw_near, stream));
  if (p.has_dw && p.dw_way == Linear::SUMMED) CDL_CHECK(sum_planes(dw.ptr, p.ld_sum, 0, 1, dw_near, desc->accumulate_dw, stream));
  return CDL_OK;
}

}  // namespace head
}  // namespace cdl

extern "C" {

int32_t cdl_b200_distillation(const cdl_head_loss_desc* desc, const cdl_tensor* logits, const cdl_tensor* teacher_ids,
                              const cdl_tensor* teacher_logits, const cdl_tensor* d_loss, const cdl_tensor* loss,
                              const cdl_tensor* lse, const cdl_tensor* d_logits, cdl_stream stream) {
  return cdl::head::distillation_execute(desc, logits, teacher_ids, teacher_logits, d_loss, loss, lse, d_logits,
                                         static_cast<cudaStream_t>(stream));
}

int32_t cdl_b200_linear_loss_scratch_bytes(const cdl_head_loss_desc* desc, const cdl_tensor* x, const cdl_tensor* w,
                                           int64_t entries, const cdl_tensor* dx, const cdl_tensor* dw, size_t* bytes_out) {
  using namespace cdl;
  if (!bytes_out) return fail(CDL_ERR_INVALID, "linear_loss_scratch_bytes: bytes_out is required");
  *bytes_out = 0;
  if (entries < 0 || entries > head::MAX_ENTRIES)
    return fail(CDL_ERR_INVALID, "linear_loss_scratch_bytes: entries must be in 0 .. %d", head::MAX_ENTRIES);
  if (entries == 0) entries = 1;  // (targets have one)
  head::Linear p;
  CDL_CHECK(head::check_linear("linear_loss_scratch_bytes", desc, x, w, dx, dw, entries, &p));
  if (p.T > 0) *bytes_out = p.bytes;
  return CDL_OK;
}

int32_t cdl_b200_linear_cross_entropy(const cdl_head_loss_desc* desc, const cdl_tensor* x, const cdl_tensor* w,
                                      const cdl_tensor* targets, const cdl_tensor* d_loss, const cdl_tensor* loss,
                                      const cdl_tensor* lse, const cdl_tensor* dx, const cdl_tensor* dw, void* scratch,
                                      size_t scratch_bytes, cdl_stream stream) {
  using namespace cdl;
  const char* op = "linear_cross_entropy";
  head::Linear p;
  CDL_CHECK(head::check_linear(op, desc, x, w, dx, dw, head::TARGET_ENTRIES, &p));
  if (desc->temperature != 1.f) return fail(CDL_ERR_UNSUPPORTED, "%s: temperature must be 1", op);
  head::Entries e;
  head::RowTerms terms;
  CDL_CHECK(head::check_targets(op, p.T, targets, &e));
  CDL_CHECK(head::check_terms(op, desc, p.T, d_loss, loss, lse, &terms));
  return head::linear_execute(p, desc, e, terms, scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
}

int32_t cdl_b200_linear_distillation(const cdl_head_loss_desc* desc, const cdl_tensor* x, const cdl_tensor* w,
                                     const cdl_tensor* teacher_ids, const cdl_tensor* teacher_logits, const cdl_tensor* d_loss,
                                     const cdl_tensor* loss, const cdl_tensor* lse, const cdl_tensor* dx, const cdl_tensor* dw,
                                     void* scratch, size_t scratch_bytes, cdl_stream stream) {
  using namespace cdl;
  const char* op = "linear_distillation";
  const long long entries = teacher_ids && teacher_ids->rank == 2 ? teacher_ids->shape[1] : 0;
  if (entries > head::MAX_ENTRIES)
    return fail(CDL_ERR_UNSUPPORTED, "%s: at most %d entries per token (got %lld)", op, head::MAX_ENTRIES, entries);
  head::Linear p;
  CDL_CHECK(head::check_linear(op, desc, x, w, dx, dw, entries, &p));
  head::Entries e;
  head::RowTerms terms;
  CDL_CHECK(head::check_teacher(op, p.T, teacher_ids, teacher_logits, &e));
  CDL_CHECK(head::check_terms(op, desc, p.T, d_loss, loss, lse, &terms));
  return head::linear_execute(p, desc, e, terms, scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
