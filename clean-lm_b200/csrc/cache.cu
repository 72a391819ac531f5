// The paged key-value cache: which pages and slots new tokens get, and the new keys and values' way there.
#include "ops.h"
#include "ptx.cuh"

#include <algorithm>

namespace cdl {
namespace cache {

// ---------------------------------------------------------------- plan
// Per request b, with c = cached, a = added (negative: 0) and P = page_size:
//   E_b = sum of a up to b;  need_b = pages(c + a) - pages(c), 0 where the request does not fit (its table row is too short,
//   E_b > rows or c + a > 2^31 - 1);  C_b = sum of need up to b;  served_b = fits and (need_b == 0 or C_b <= free)
// Served requests with need take stack[free - C_b ..], in the order of the requests: the served ones with need are the first
// ones with it, as C only grows.
// Bound by latency: one kernel, in which every CTA sums the lengths up itself (1024 requests at a time) and then takes its
// share of the rows and pages, each found by a binary search in shared memory.  (5.2 us for 64 requests of a token each, 9.9 for
// 1999 of 1 to 64, two rounds of sums.)
constexpr int THREADS = 256, PER = 4, CHUNK = THREADS * PER;

struct PlanParams {
  const int *cached, *added, *free_pages, *free_count;
  int* table;
  long long table_sb;
  int requests, width, stack, pages, page_size, rows;
  int *seq_lens, *cu, *positions, *slots, *free_left;
};

__global__ void __launch_bounds__(THREADS) plan_kernel(const PlanParams p) {
  __shared__ long long ends[CHUNK + 1], upto[CHUNK + 1];  // of rows and of pages; [i + 1] is request i's
  __shared__ int ctx[CHUNK];                              // cached
  __shared__ unsigned char ok[CHUNK];
  __shared__ long long part[2][THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_wait();
  grid_dep_launch();
  const long long P = p.page_size;
  const long long free = min(max(*p.free_count, 0), p.stack);
  const long long longest = min(p.width * P, static_cast<long long>(INT32_MAX));  // (a table may name a page twice: more keys than slots)
  const int share = blockIdx.x * THREADS + tid, step = gridDim.x * THREADS;
  long long rows_before = 0, pages_before = 0, left = free;
  // sums of x and y over the threads ahead of this one (exclusive), and over all
  auto scan = [&](long long& x, long long& y, long long& all_x, long long& all_y) {
    long long a = x, b = y;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, a, d), v = __shfl_up_sync(0xffffffffu, b, d);
      if (lane >= d) a += u, b += v;
    }
    if (lane == 31) part[0][warp] = a, part[1][warp] = b;
    __syncthreads();
    all_x = all_y = 0;
    x = a - x, y = b - y;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) x += part[0][w], y += part[1][w];
      all_x += part[0][w], all_y += part[1][w];
    }
    __syncthreads();
  };
  for (int r0 = 0; r0 < p.requests; r0 += CHUNK) {
    const int count = min(CHUNK, p.requests - r0);
    long long c[PER], a[PER], sum = 0, none = 0, all, unused;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = tid * PER + i;
      c[i] = r < count ? max(p.cached[r0 + r], 0) : 0;
      a[i] = r < count ? max(p.added[r0 + r], 0) : 0;
      sum += a[i];
    }
    scan(sum, none, all, unused);
    long long e = rows_before + sum, need[PER], pages = 0, end[PER];
    bool fits[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      e += a[i];
      end[i] = e;
      fits[i] = c[i] + a[i] <= longest && e <= p.rows;
      need[i] = fits[i] ? (c[i] + a[i] + P - 1) / P - (c[i] + P - 1) / P : 0;
      pages += need[i];
    }
    long long all_pages;
    none = 0;
    scan(pages, none, all_pages, unused);
    long long at = pages_before + pages;
    const bool mine = (r0 / CHUNK) % gridDim.x == blockIdx.x;
    if (tid == 0) ends[0] = rows_before, upto[0] = pages_before;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = tid * PER + i;
      at += need[i];
      if (r < count) {
        const bool served = fits[i] && (need[i] == 0 || at <= free);
        ends[r + 1] = end[i], upto[r + 1] = at;
        ctx[r] = static_cast<int>(c[i]);
        ok[r] = served;
        if (mine) {
          p.seq_lens[r0 + r] = static_cast<int>(c[i] + (served ? a[i] : 0));
          p.cu[r0 + r + 1] = static_cast<int>(min(end[i], static_cast<long long>(p.rows)));
        }
      }
    }
    __syncthreads();
    // request of the chunk that x falls to: the last one whose sum ahead is not above x
    auto of = [&](const long long* sums, long long x) {
      int lo = 0, hi = count;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= x) lo = mid;
        else hi = mid;
      }
      return lo;
    };
    // ---- the rows of this chunk
    const long long row_end = min(rows_before + all, static_cast<long long>(p.rows));
    for (long long r = rows_before + share; r < row_end; r += step) {
      const int b = of(ends, r);
      const long long pos = ctx[b] + (r - ends[b]);
      long long slot = -1;
      if (ok[b]) {
        const long long page_at = pos / P, old = (ctx[b] + P - 1) / P;
        const int page = page_at < old ? p.table[(r0 + b) * p.table_sb + page_at] : p.free_pages[free - 1 - (upto[b] + page_at - old)];
        if (page >= 0 && page < p.pages) slot = page * P + pos % P;
      }
      p.positions[r] = static_cast<int>(min(pos, static_cast<long long>(INT32_MAX)));
      p.slots[r] = static_cast<int>(slot);
    }
    // ---- and its new pages, those that the stack holds
    for (long long x = pages_before + share; x < min(pages_before + all_pages, free); x += step) {
      const int b = of(upto, x);
      if (!ok[b]) continue;
      const long long old = (ctx[b] + P - 1) / P;
      p.table[(r0 + b) * p.table_sb + old + (x - upto[b])] = p.free_pages[free - 1 - x];
    }
    // the last request that is served takes the stack down to here
    if (blockIdx.x == 0)
      for (int r = tid; r < count; r += THREADS)
        if (ok[r] && upto[r + 1] > upto[r]) left = min(left, free - upto[r + 1]);
    rows_before += all;
    pages_before += all_pages;
    __syncthreads();
  }
  for (long long r = rows_before + share; r < p.rows; r += step) p.positions[r] = -1, p.slots[r] = -1;
  if (blockIdx.x == 0) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) left = min(left, __shfl_xor_sync(0xffffffffu, left, d));
    if (lane == 0) part[0][warp] = left;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) left = min(left, part[0][w]);
      *p.free_left = static_cast<int>(left);
      p.cu[0] = 0;
    }
  }
}

// ---------------------------------------------------------------- write
__device__ __forceinline__ void unpack8(const uint4& q, float (&f)[8]) {
  f[0] = bf16_lo(q.x); f[1] = bf16_hi(q.x); f[2] = bf16_lo(q.y); f[3] = bf16_hi(q.y);
  f[4] = bf16_lo(q.z); f[5] = bf16_hi(q.z); f[6] = bf16_lo(q.w); f[7] = bf16_hi(q.w);
}
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}

struct WriteParams {
  const __nv_bfloat16 *q, *k, *v;
  long long q_st, q_sh, k_st, k_sh, v_st, v_sh;
  __nv_bfloat16 *q_out, *k_out, *k_cache, *v_cache;
  long long qo_st, qo_sh, ko_st, ko_sh, kc_sp, kc_ss, kc_sh, vc_sp, vc_ss, vc_sh;
  const float* cos_sin;
  const int *positions, *slots;
  long long tokens, capacity;  // capacity: slots of the cache
  int heads, kv_heads, half, table_rows, page_size;
};

// Rotate-half RoPE of q and k (x'[i] = x[i] cos - x[i + D/2] sin, x'[i + D/2] = x[i + D/2] cos + x[i] sin) and the way of k and v
// into their slots.  HBM-bound: every element is read and written once.  A CTA has a token, a thread 8 elements of both halves at
// the same place of several heads, whose loads overlap and share the place's cosines and sines.  Loads come ahead of the slot and
// the position, which they do not depend on; three heads at once with 72 registers keep most bytes under way (405 MB, 16384 tokens
// of 48 heads of 128: 64.9 us, 95 % of 6.5 TB/s; two at once 66.1, four 68.3; a thread per place and head, found by 64-bit
// divisions: 90 us).
constexpr int WRITE_THREADS = 128, AT_ONCE = 3;
__device__ __forceinline__ uint4 load_once(const __nv_bfloat16* p) {  // (q and k may be overwritten by this very thread)
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
  return r;
}
__global__ void __launch_bounds__(WRITE_THREADS, 7) write_kernel(const WriteParams p) {
  grid_dep_wait();
  grid_dep_launch();
  const int groups = p.half / 8, step = WRITE_THREADS / groups;  // heads at a time
  const int first = threadIdx.x / groups, g = (threadIdx.x - first * groups) * 8;
  if (first >= step) return;
  const long long token = blockIdx.x;
  const int keys = p.heads, values = p.heads + p.kv_heads, lines = p.heads + 2 * p.kv_heads;
  uint4 a[AT_ONCE], b[AT_ONCE];
  auto load = [&](int line0) {
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int line = line0 + i * step;
      if (line >= lines) break;
      const __nv_bfloat16* from = line < keys     ? p.q + token * p.q_st + line * p.q_sh
                                  : line < values ? p.k + token * p.k_st + (line - keys) * p.k_sh
                                                  : p.v + token * p.v_st + (line - values) * p.v_sh;
      a[i] = load_once(from + g);
      b[i] = load_once(from + g + p.half);
    }
  };
  load(first);  // ahead of the slot and the position, which the loads do not depend on
  const int slot = p.slots[token], pos = p.cos_sin != nullptr ? p.positions[token] : -1;
  const bool cached = slot >= 0 && slot < p.capacity, turn = pos >= 0 && pos < p.table_rows;
  const int page = cached ? slot / p.page_size : 0, in = slot - page * p.page_size;
  float c[8], s[8];
  if (turn) {
    const float* cs = p.cos_sin + static_cast<long long>(pos) * 2 * p.half + g;
    *reinterpret_cast<float4*>(c) = __ldg(reinterpret_cast<const float4*>(cs));
    *reinterpret_cast<float4*>(c + 4) = __ldg(reinterpret_cast<const float4*>(cs + 4));
    *reinterpret_cast<float4*>(s) = __ldg(reinterpret_cast<const float4*>(cs + p.half));
    *reinterpret_cast<float4*>(s + 4) = __ldg(reinterpret_cast<const float4*>(cs + p.half + 4));
  }
  for (int line0 = first; line0 < lines; line0 += AT_ONCE * step) {
    if (line0 != first) load(line0);
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int line = line0 + i * step;
      if (line >= lines) break;
      if (turn && line < values) {
        float lo[8], hi[8], x[8], y[8];
        unpack8(a[i], lo);
        unpack8(b[i], hi);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = lo[j] * c[j] - hi[j] * s[j];
          y[j] = hi[j] * c[j] + lo[j] * s[j];
        }
        a[i] = pack8(x);
        b[i] = pack8(y);
      }
      __nv_bfloat16* to = line < keys                         ? p.q_out + token * p.qo_st + line * p.qo_sh
                          : line < values && p.k_out != nullptr ? p.k_out + token * p.ko_st + (line - keys) * p.ko_sh
                                                                : nullptr;
      if (to != nullptr) {
        *reinterpret_cast<uint4*>(to + g) = a[i];
        *reinterpret_cast<uint4*>(to + g + p.half) = b[i];
      }
      if (line >= keys && cached) {
        to = line < values ? p.k_cache + page * p.kc_sp + in * p.kc_ss + (line - keys) * p.kc_sh
                           : p.v_cache + page * p.vc_sp + in * p.vc_ss + (line - values) * p.vc_sh;
        *reinterpret_cast<uint4*>(to + g) = a[i];
        *reinterpret_cast<uint4*>(to + g + p.half) = b[i];
      }
    }
  }
}
}  // namespace cache

// ---------------------------------------------------------------- host
// Whether no two indices of a view name the same element: sorted by stride, each dimension steps over the ones below it.
bool view_apart_from_itself(const cdl_tensor& t) {
  int order[4], n = 0;
  for (int i = 0; i < t.rank; ++i)
    if (t.shape[i] > 1) order[n++] = i;
  std::sort(order, order + n, [&](int a, int b) { return t.stride[a] < t.stride[b]; });
  long long reach = 1;
  for (int i = 0; i < n; ++i) {
    const int d = order[i];
    if (t.stride[d] < reach) return false;
    reach = t.stride[d] * (t.shape[d] - 1) + reach;
  }
  return true;
}
// Whether two views provably share no element: their extents are apart, or some stride of theirs divides the memory into steps in
// which they lie in different places (q, k and v in the heads of a fused tensor, keys and values in halves of a page, of a head or
// of a row).  Dimensions whose strides are multiples of the step go from one step to another and do not matter.
bool views_apart(const cdl_tensor& a, const cdl_tensor& b) {
  // Bytes from a view's first to behind its last, without the dimensions that are multiples of `step` bytes (0: none is); 0: empty.
  auto reach = [](const cdl_tensor& t, long long step) {
    const long long size = static_cast<long long>(dtype_size(t.dtype));
    long long n = size;
    for (int i = 0; i < t.rank; ++i) {
      if (t.shape[i] == 0) return 0LL;
      if (step == 0 || t.stride[i] * size % step != 0) n += (t.shape[i] - 1) * t.stride[i] * size;
    }
    return n;
  };
  const long long all_a = reach(a, 0), all_b = reach(b, 0);
  if (all_a == 0 || all_b == 0) return true;
  const cdl_tensor* views[] = {&a, &b};
  for (const cdl_tensor* t : views)
    for (int i = 0; i < t->rank; ++i)
      if (t->shape[i] > 1 && t->stride[i] < 0) return false;
  const long long pa = reinterpret_cast<intptr_t>(a.ptr), pb = reinterpret_cast<intptr_t>(b.ptr);
  if (pa + all_a <= pb || pb + all_b <= pa) return true;
  for (const cdl_tensor* t : views)
    for (int i = 0; i < t->rank; ++i) {
      const long long step = t->stride[i] * static_cast<long long>(dtype_size(t->dtype));
      if (step <= 0) continue;
      const long long off = ((pb - pa) % step + step) % step;
      if (reach(a, step) <= off && off + reach(b, step) <= step) return true;
    }
  return false;
}
static bool same_view(const cdl_tensor& a, const cdl_tensor& b) {
  if (a.ptr != b.ptr || a.dtype != b.dtype || a.rank != b.rank) return false;
  for (int i = 0; i < a.rank; ++i)
    if (a.shape[i] != b.shape[i] || (a.shape[i] > 1 && a.stride[i] != b.stride[i])) return false;
  return true;
}

static int32_t check_ints(const char* op, const char* name, const cdl_tensor* t, long long n) {
  if (!t || t->rank != 1 || t->dtype != CDL_I32 || n < 0 || t->shape[0] != n || (n > 1 && t->stride[0] != 1) || (n > 0 && !t->ptr))
    return fail(CDL_ERR_INVALID, "%s: %s must be a packed i32 vector of %lld", op, name, n);
  return CDL_OK;
}

int32_t cache_plan_execute(int32_t page_size, int32_t pages, const cdl_tensor* cached, const cdl_tensor* added,
                           const cdl_tensor* block_table, const cdl_tensor* free_pages, const cdl_tensor* free_count,
                           const cdl_tensor* seq_lens, const cdl_tensor* cu_seqlens, const cdl_tensor* positions,
                           const cdl_tensor* slots, const cdl_tensor* free_left, cudaStream_t stream) {
  const char* op = "cache_plan";
  if (!cached || !block_table || !free_pages || !slots)
    return fail(CDL_ERR_INVALID, "%s: cached, block_table, free_pages and slots are required", op);
  if (page_size <= 0 || pages < 0 || static_cast<long long>(pages) * page_size > INT32_MAX)
    return fail(CDL_ERR_INVALID, "%s: page_size must be positive and the cache hold less than 2^31 slots", op);
  const long long B = cached->shape[0], rows = slots->shape[0];
  if (cached->rank != 1 || B < 0 || B > INT32_MAX / 4 || slots->rank != 1 || rows < 0 || rows > INT32_MAX)
    return fail(CDL_ERR_INVALID, "%s: cached and slots must be vectors of less than 2^29 requests and 2^31 rows", op);
  CDL_CHECK(check_ints(op, "cached", cached, B));
  CDL_CHECK(check_ints(op, "added", added, B));
  CDL_CHECK(check_ints(op, "free_pages", free_pages, free_pages->shape[0]));
  CDL_CHECK(check_ints(op, "free_count", free_count, 1));
  CDL_CHECK(check_ints(op, "seq_lens", seq_lens, B));
  CDL_CHECK(check_ints(op, "cu_seqlens", cu_seqlens, B + 1));
  CDL_CHECK(check_ints(op, "positions", positions, rows));
  CDL_CHECK(check_ints(op, "slots", slots, rows));
  CDL_CHECK(check_ints(op, "free_left", free_left, 1));
  if (block_table->rank != 2 || block_table->dtype != CDL_I32 || block_table->shape[0] != B || block_table->shape[1] < 0 ||
      block_table->shape[1] > INT32_MAX || (block_table->shape[1] > 1 && block_table->stride[1] != 1) ||
      (B > 0 && block_table->shape[1] > 0 && !block_table->ptr) ||
      (B > 1 && block_table->stride[0] < block_table->shape[1]))
    return fail(CDL_ERR_INVALID, "%s: block_table must be i32 [requests, pages of a request] with contiguous rows that do not overlap", op);
  if (free_pages->shape[0] > INT32_MAX) return fail(CDL_ERR_INVALID, "%s: a stack of less than 2^31 pages is needed", op);
  const cdl_tensor* ins[] = {cached, added, free_pages, free_count, block_table};
  const cdl_tensor* outs[] = {seq_lens, cu_seqlens, positions, slots, free_left};
  for (const cdl_tensor* o : outs) {
    for (const cdl_tensor* i : ins)
      if (!views_apart(*o, *i)) return fail(CDL_ERR_INVALID, "%s: an output overlaps an input", op);
    for (const cdl_tensor* q : outs)
      if (q != o && !views_apart(*o, *q)) return fail(CDL_ERR_INVALID, "%s: outputs overlap", op);
  }
  for (int i = 0; i < 4; ++i)
    if (!views_apart(*block_table, *ins[i])) return fail(CDL_ERR_INVALID, "%s: block_table overlaps an input", op);
  cache::PlanParams p{};
  auto ints = [](const cdl_tensor* t) { return static_cast<int*>(t->ptr); };
  p.cached = ints(cached), p.added = ints(added), p.free_pages = ints(free_pages), p.free_count = ints(free_count);
  p.table = ints(block_table), p.table_sb = block_table->stride[0];
  p.requests = static_cast<int>(B), p.width = static_cast<int>(block_table->shape[1]);
  p.stack = static_cast<int>(free_pages->shape[0]), p.pages = pages, p.page_size = page_size, p.rows = static_cast<int>(rows);
  p.seq_lens = ints(seq_lens), p.cu = ints(cu_seqlens), p.positions = ints(positions), p.slots = ints(slots);
  p.free_left = ints(free_left);
  const long long ctas = std::max<long long>(1, std::min<long long>(sm_count(), (rows + cache::THREADS - 1) / cache::THREADS));
  ProfileScope ps(PROF_ELEMENTWISE, 8.0 * rows + 16.0 * B, stream);
  CDL_CUDA(launch_pdl(cache::plan_kernel, dim3(static_cast<unsigned>(ctas)), dim3(cache::THREADS), 0, stream, p));
  return CDL_OK;
}

static int32_t check_heads(const char* op, const char* name, const cdl_tensor* t, long long tokens, long long heads, long long d) {
  if (t->rank != 3 || t->dtype != CDL_BF16 || t->shape[0] != tokens || t->shape[1] != heads || t->shape[2] != d)
    return fail(CDL_ERR_INVALID, "%s: %s must be bf16 [tokens %lld, heads %lld, head_dim %lld]", op, name, tokens, heads, d);
  bool ok = (reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && t->stride[2] == 1;
  for (int i = 0; i < 2; ++i) ok = ok && (t->shape[i] <= 1 || (t->stride[i] % 8 == 0 && t->stride[i] >= 0));
  if (!ok || (tokens * heads > 0 && !t->ptr))
    return fail(CDL_ERR_INVALID, "%s: %s must have a contiguous last dimension and 16-byte aligned strides", op, name);
  return CDL_OK;
}

int32_t cache_write_execute(const cdl_tensor* q, const cdl_tensor* k, const cdl_tensor* v, const cdl_tensor* cos_sin,
                            const cdl_tensor* positions, const cdl_tensor* slots, const cdl_tensor* q_out,
                            const cdl_tensor* k_out, const cdl_tensor* k_cache, const cdl_tensor* v_cache,
                            cudaStream_t stream) {
  const char* op = "cache_write";
  if (!k || !v || !slots || !k_cache || !v_cache)
    return fail(CDL_ERR_INVALID, "%s: k, v, slots, k_cache and v_cache are required", op);
  if ((q == nullptr) != (q_out == nullptr)) return fail(CDL_ERR_INVALID, "%s: q and q_out go together", op);
  if ((cos_sin == nullptr) != (positions == nullptr)) return fail(CDL_ERR_INVALID, "%s: cos_sin and positions go together", op);
  if (!cos_sin && (q || k_out)) return fail(CDL_ERR_INVALID, "%s: q and k_out need the rotation's table", op);
  if (k->rank != 3) return fail(CDL_ERR_INVALID, "%s: k must be bf16 [tokens, kv_heads, head_dim]", op);
  const long long T = k->shape[0], Hkv = k->shape[1], D = k->shape[2], H = q ? (q->rank == 3 ? q->shape[1] : -1) : 0;
  if (T < 0 || T > INT32_MAX || Hkv < 0 || Hkv > 65536 || H < 0 || H > 65536)
    return fail(CDL_ERR_INVALID, "%s: less than 2^31 tokens and at most 65536 heads [tokens, heads, head_dim]", op);
  if (D <= 0 || D % 16 != 0 || D > 16 * cache::WRITE_THREADS)
    return fail(CDL_ERR_INVALID, "%s: head_dim must be a multiple of 16, at most %d", op, 16 * cache::WRITE_THREADS);
  CDL_CHECK(check_heads(op, "k", k, T, Hkv, D));
  CDL_CHECK(check_heads(op, "v", v, T, Hkv, D));
  if (q) {
    CDL_CHECK(check_heads(op, "q", q, T, H, D));
    CDL_CHECK(check_heads(op, "q_out", q_out, T, H, D));
  }
  if (k_out) CDL_CHECK(check_heads(op, "k_out", k_out, T, Hkv, D));
  CDL_CHECK(check_ints(op, "slots", slots, T));
  if (cos_sin) {
    CDL_CHECK(check_ints(op, "positions", positions, T));
    if (cos_sin->rank != 2 || cos_sin->dtype != CDL_F32 || cos_sin->shape[1] != D || cos_sin->shape[0] < 0 ||
        cos_sin->shape[0] > INT32_MAX || cos_sin->stride[1] != 1 || (cos_sin->shape[0] > 1 && cos_sin->stride[0] != D) ||
        (reinterpret_cast<uintptr_t>(cos_sin->ptr) & 15))
      return fail(CDL_ERR_INVALID, "%s: cos_sin must be packed f32 [positions, head_dim], 16-byte aligned", op);
    if (T > 0 && cos_sin->shape[0] > 0 && !cos_sin->ptr) return fail(CDL_ERR_INVALID, "%s: null pointer (cos_sin)", op);
  }
  const cdl_tensor* caches[] = {k_cache, v_cache};
  for (const cdl_tensor* c : caches) {
    bool ok = c->rank == 4 && c->dtype == CDL_BF16 && c->shape[2] == Hkv && c->shape[3] == D && c->stride[3] == 1 &&
              (reinterpret_cast<uintptr_t>(c->ptr) & 15) == 0 && c->shape[0] >= 0 && c->shape[1] > 0;
    for (int i = 0; i < 3 && ok; ++i) ok = c->shape[i] == k_cache->shape[i] && (c->shape[i] <= 1 || (c->stride[i] % 8 == 0 && c->stride[i] >= 0));
    if (!ok)
      return fail(CDL_ERR_INVALID, "%s: the caches must be bf16 [pages, page_size, kv_heads %lld, head_dim %lld] of one shape with a "
                  "contiguous last dimension and 16-byte aligned strides", op, Hkv, D);
    if (T > 0 && c->shape[0] > 0 && Hkv > 0 && !c->ptr) return fail(CDL_ERR_INVALID, "%s: null pointer (a cache)", op);
    if (!view_apart_from_itself(*c)) return fail(CDL_ERR_INVALID, "%s: elements of a cache overlap", op);
  }
  if (k_cache->shape[1] > INT32_MAX || k_cache->shape[0] > INT32_MAX / k_cache->shape[1])
    return fail(CDL_ERR_UNSUPPORTED, "%s: the cache must hold less than 2^31 slots", op);
  const cdl_tensor* outs[] = {q_out, k_out, k_cache, v_cache};
  const cdl_tensor* ins[] = {q, k, v, cos_sin, positions, slots};
  for (int i = 0; i < 4; ++i) {
    if (!outs[i]) continue;
    if (!view_apart_from_itself(*outs[i])) return fail(CDL_ERR_INVALID, "%s: elements of an output overlap", op);
    for (int j = 0; j < 6; ++j) {
      if (!ins[j] || views_apart(*outs[i], *ins[j])) continue;
      if (i == j && i < 2 && same_view(*outs[i], *ins[j])) continue;  // in place
      return fail(CDL_ERR_INVALID, "%s: an output overlaps an input (q_out may be q itself, k_out k)", op);
    }
    for (int j = 0; j < i; ++j)
      if (outs[j] && !views_apart(*outs[i], *outs[j])) return fail(CDL_ERR_INVALID, "%s: outputs overlap", op);
  }
  const long long total = T * (H + 2 * Hkv) * (D / 16);
  if (total == 0) return CDL_OK;
  cache::WriteParams p{};
  auto bf = [](const cdl_tensor* t) { return t ? static_cast<__nv_bfloat16*>(t->ptr) : nullptr; };
  p.q = bf(q), p.k = bf(k), p.v = bf(v), p.q_out = bf(q_out), p.k_out = bf(k_out), p.k_cache = bf(k_cache), p.v_cache = bf(v_cache);
  if (q) p.q_st = q->stride[0], p.q_sh = q->stride[1], p.qo_st = q_out->stride[0], p.qo_sh = q_out->stride[1];
  p.k_st = k->stride[0], p.k_sh = k->stride[1], p.v_st = v->stride[0], p.v_sh = v->stride[1];
  if (k_out) p.ko_st = k_out->stride[0], p.ko_sh = k_out->stride[1];
  p.kc_sp = k_cache->stride[0], p.kc_ss = k_cache->stride[1], p.kc_sh = k_cache->stride[2];
  p.vc_sp = v_cache->stride[0], p.vc_ss = v_cache->stride[1], p.vc_sh = v_cache->stride[2];
  p.cos_sin = cos_sin ? static_cast<const float*>(cos_sin->ptr) : nullptr;
  p.positions = positions ? static_cast<const int*>(positions->ptr) : nullptr;
  p.slots = static_cast<const int*>(slots->ptr);
  p.tokens = T, p.capacity = k_cache->shape[0] * k_cache->shape[1];
  p.heads = static_cast<int>(H), p.kv_heads = static_cast<int>(Hkv), p.half = static_cast<int>(D / 2);
  p.table_rows = cos_sin ? static_cast<int>(cos_sin->shape[0]) : 0, p.page_size = static_cast<int>(k_cache->shape[1]);
  ProfileScope ps(PROF_ELEMENTWISE, static_cast<double>(total) * 64, stream);
  CDL_CUDA(launch_pdl(cache::write_kernel, dim3(static_cast<unsigned>(T)), dim3(cache::WRITE_THREADS), 0, stream, p));
  return CDL_OK;
}

}  // namespace cdl

extern "C" {

int32_t cdl_b200_cache_plan(int32_t page_size, int32_t pages, const cdl_tensor* cached, const cdl_tensor* added,
                            const cdl_tensor* block_table, const cdl_tensor* free_pages, const cdl_tensor* free_count,
                            const cdl_tensor* seq_lens, const cdl_tensor* cu_seqlens, const cdl_tensor* positions,
                            const cdl_tensor* slots, const cdl_tensor* free_left, cdl_stream stream) {
  return cdl::cache_plan_execute(page_size, pages, cached, added, block_table, free_pages, free_count, seq_lens, cu_seqlens,
                                 positions, slots, free_left, static_cast<cudaStream_t>(stream));
}
int32_t cdl_b200_cache_write(const cdl_tensor* q, const cdl_tensor* k, const cdl_tensor* v, const cdl_tensor* cos_sin,
                             const cdl_tensor* positions, const cdl_tensor* slots, const cdl_tensor* q_out,
                             const cdl_tensor* k_out, const cdl_tensor* k_cache, const cdl_tensor* v_cache, cdl_stream stream) {
  return cdl::cache_write_execute(q, k, v, cos_sin, positions, slots, q_out, k_out, k_cache, v_cache,
                                  static_cast<cudaStream_t>(stream));
}

}  // extern "C"
