// Attention of one new token per request over a paged key-value cache.
//
//   s_j = f(scale q . k_j),  f(x) = cap tanh(x / cap) or x;   out = sum_j softmax(s)_j v_j over the keys a request sees,
//   lse = log sum_j exp(s_j)
//
// Bound by reading the keys and values once (2 multiply-adds per 2-byte element and query head of a group; the tensor cores
// see 8 or 16 query columns).  The tiles of 16 or 32 keys of all requests and kv heads form one line, whatever the lengths are,
// that the CTAs share, and the warps of a CTA its part.  SMs do not read at the same rate (equal parts ended after 147 to 204 us,
// the same SMs late each time), so a set of smaller parts follows the first where there is much to read.  Every warp works alone
// on a ring of its own in shared memory, which asynchronous 16-byte copies fill STAGES tiles ahead and across the borders of
// requests, 8 lanes a row, wherever its page lies.  (Loaded straight into the fragments, the next keys on their way behind the
// scores, 12 warps of an SM had too little under way, 270 us for 1.14 GB, which are 174 us at 6.56 TB/s and take 183.7 now; a bulk
// copy per row, which a warp issues one lane after the other, took 262.)  A warp's running maximum, sum and output stay in
// registers.  Where a warp's part cuts the keys of a (request, kv head), the warps of the CTA join what they have of it; what the
// CTA's part cuts goes to the scratch, and a second kernel joins that.
//
// Short work is bound by latency instead, trips to memory one after the other (lengths, page, keys, values, results).  There each
// (request, kv head) has a cluster of CTAs of its own, which join their results by way of shared memory: one request of some
// hundred keys and 16 heads (777 of 128) takes 7.8 us, 10.7 on the common line with its second kernel.  The host knows no lengths, so it
// is the table's width and the window that choose: one of 129 pages of 16 takes the common line whatever its requests hold.
//
// Products are taken transposed, scores^T = K q^T and out^T = V^T p^T, so that the query heads of a group are the 8 columns
// of mma.m16n8k16 (as rows they would leave at least half of it empty) and the pieces of K and V rows that a thread reads are its
// fragments: for the scores the order of d within a product is free, for the output the order of its rows is.  (A tile of the
// 5th-generation tensor cores has 64 or 128 rows of queries, of which one token per request fills 1 to 16.)  Probabilities are
// rounded to bf16 for the second product, as in the prompt's attention; their sum is of the unrounded ones, in f32.
#include "ops.h"
#include "ptx.cuh"

#include <cooperative_groups.h>
#include <float.h>
#include <math.h>

#include <algorithm>

namespace cdl {
namespace decode {

namespace cg = cooperative_groups;

constexpr int WARPS = 4;         // of a CTA
constexpr int STAGES = 2;        // tiles of a warp's ring
// CTAs of an SM: as many as registers (168 of 12 warps, 255 of 8) and rings (70 KB each) allow; nt: tiles of 8 query columns
constexpr int ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }
constexpr int JOIN_WARPS = 8;    // of a CTA of the second kernel
// Where no request sees more keys than this (by the width of its table, by the window), each line has CTAs of its own, as one long line
// among short ones cannot take much longer than the rest.  (Own CTAs / shared ones, us, 16 heads of 128, requests of 1 to L keys:
// L = 512: 1 request 7.2 / 10.8, 37 25 / 30, 256 106 / 126; 2048: 1 10.5 / 14.3, 16 40 / 38, 64 102 / 109; 4096: 1 14.6 / 15.9, 16
// 75 / 61, 37 128 / 120.  24 heads on 2 of 64, L = 2048: 1 9.8 / 10.9, 256 49 / 53; 8192: 1 16.5 / 14.5.  What the rule gives away:
// 4096 lines of 1 to 100 keys, 56 / 51.)
constexpr int OWN_KEYS = 2048;
constexpr int MAX_SPLIT = 8;     // CTAs of a line that has its own
constexpr int MAX_BATCH = 4096;  // the prefix of the lengths is kept in shared memory beside the rings

struct Params {
  const __nv_bfloat16* q;
  long long q_sb, q_sh;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  long long k_sp, k_ss, k_sh, v_sp, v_ss, v_sh;  // page, slot, head
  const int* table;
  long long table_sb;
  const int* lens;
  int batch, heads, kv_heads, group, chunks;  // group: query heads of a kv head; chunks: of COLS of them
  int pages, page_size, width, window;
  float scale, cap;  // of the scores, in natural units; cap 0: none
  __nv_bfloat16* out;
  long long out_sb, out_sh;
  float* lse;
  int set;          // CTAs that run at once
  int split;        // CTAs of a line, where each has its own (a cluster)
  int* prefix;      // [batch + 1] tiles of the requests ahead
  float2* part_ml;  // [2 CTAs][COLS]
  float* part_o;    // [2 CTAs][COLS][D]
  float* warp_o;    // [CTAs][WARPS][COLS][D]
};

// Keys a request sees: [first, end).
__device__ __forceinline__ void visible(const Params& p, int b, int& first, int& end) {
  const long long most = static_cast<long long>(p.width) * p.page_size;
  const int len = p.lens[b];
  end = static_cast<int>(min(static_cast<long long>(max(len, 0)), most));
  first = p.window > 0 ? max(0, end - p.window) : 0;
}

// How the CTAs share `units` tiles: evenly, one or more each (so that all partial results between a line's first and last are
// there); from 192 tiles each on, the CTAs that run at once share 7/8 evenly and a second set of as many the rest, as SMs become
// free.  (Evenly / in two sets, us: 82 tiles each 60.7 / 64.6, 160 106.0 / 105.8, 315 195 / 185, 630 371 / 347.  Four sets of 84,
// 28, 11 and 5 of 128 parts: 70, 109, 186, 343; a CTA's start is not hidden by the others of its SM.)
// Quotients are taken in f64, a tenth of the time of a 64-bit division: exact where units * ctas < 2^53, and in any case the same
// everywhere and never falling.
constexpr int SETS = 2, PARTS = 8, FIRST = 7;
struct Shares {
  long long units;
  int set, ctas;
  __host__ __device__ __forceinline__ Shares(long long units, int set) : units(units), set(set) {
    ctas = units >= 192LL * set ? SETS * set : static_cast<int>(units < set ? units : set);
  }
  __host__ __device__ __forceinline__ long long begin(int c) const {
    const double n = static_cast<double>(units);
    if (ctas <= set) return static_cast<long long>(n * c / ctas);
    return static_cast<long long>(n * (c < set ? FIRST * c : FIRST * set + (PARTS - FIRST) * (c - set)) / (PARTS * set));
  }
  // The CTA that has unit u: the last one that begins at it or ahead of it.
  __host__ __device__ __forceinline__ int of(long long u) const {
    int c;
    if (ctas <= set) {
      c = static_cast<int>(static_cast<double>(u) * ctas / static_cast<double>(units));
    } else {
      const double x = static_cast<double>(u) * PARTS / static_cast<double>(units) * set;
      c = static_cast<int>(x < FIRST * set ? x / FIRST : set + (x - FIRST * set) / (PARTS - FIRST));
    }
    if (c >= ctas) c = ctas - 1;
    while (c > 0 && begin(c) > u) --c;
    while (c + 1 < ctas && begin(c + 1) <= u) ++c;
    return c;
  }
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t word(const uint4& q, int i) { return i == 0 ? q.x : i == 1 ? q.y : i == 2 ? q.z : q.w; }

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Keys of a tile: 16 of D = 128, 32 of D = 64, 8 KB of keys and values either way.
template <int D>
constexpr int tile_keys() { return D == 128 ? 16 : 32; }

// A row in shared memory is 16 bytes longer than in the cache: of the 8 lanes that read 16 bytes each at a time, no two meet in a
// bank then (the pieces 2 t, 2 t + 1, .. of a key row for the scores; piece g of the rows 2 t, 2 t + 1, .. for the output).
template <int D>
constexpr int row_bytes() { return 2 * D + 16; }
template <int D>
constexpr int stage_bytes() { return 2 * tile_keys<D>() * row_bytes<D>(); }

// The partial results of a CTA's warps, two each: of the line (request, kv head) that its part starts within and of the one that
// it ends within.  The output of a warp's last line takes the place of its ring, that of one ahead is in the scratch.
template <int COLS>
struct Cuts {
  long long line[2 * WARPS];  // -1: none
  int starts[2 * WARPS], ends[2 * WARPS], in_ring[2 * WARPS];
  float2 ml[2 * WARPS][COLS];
};

// CTAs of an SM for which it has shared memory: 228 KB, of which the system takes 1 KB per CTA.  (From 576 requests of head_dim 64, 1600
// of 128, the prefix of their lengths leaves room for two.  Parts for CTAs that run at once / for three per SM regardless, the last third
// of them behind the rest, us: 8 heads on 2 of 64, 600 requests of up to 1200 keys 61 / 68, 1024 92 / 108, 2048 of up to 500 97 / 113; of
// 128, 2048 137 / 157.)
inline int ctas_by_memory(int nt, size_t dynamic) {
  const size_t fixed = (nt == 1 ? sizeof(Cuts<8>) : sizeof(Cuts<16>)) + 64;  // and the kernel's few single words
  return static_cast<int>((228 << 10) / ((dynamic + 127) / 128 * 128 + (fixed + 127) / 128 * 128 + 1024));
}

// 16 bytes to shared memory, `bytes` of them from `from` and zeros behind.
__device__ __forceinline__ void copy_16(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Until all but the last N groups of this thread's copies are there.
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// D: head dimension; NT: tiles of 8 query heads of one kv head; OWN: a cluster of p.split CTAs has one line and joins what they have
// of it by way of their shared memory (no second kernel, and nobody looks for its part).
template <int D, int NT, bool OWN>
__global__ void __launch_bounds__(WARPS * 32, ctas_per_sm(NT)) attn_decode_kernel(const Params p) {
  constexpr int COLS = 8 * NT;
  constexpr int KEYS = tile_keys<D>();
  constexpr int SUB = KEYS / 16;   // 16-key products of a tile
  constexpr int KCH = D / 32;      // 16-byte pieces of a key row per thread
  constexpr int VCH = D / 64;      // 16-byte pieces of a value row per thread
  constexpr int MT = D / 16;       // 16-row tiles of the transposed output
  constexpr int RS = row_bytes<D>(), STAGE = stage_bytes<D>();
  static_assert(COLS * D * 4 <= STAGES * STAGE, "an output takes the place of a ring");
  extern __shared__ __align__(128) char smem[];
  int* prefix = reinterpret_cast<int*>(smem + WARPS * STAGES * STAGE);  // [batch + 1]
  __shared__ int warp_sum[WARPS];
  __shared__ Cuts<COLS> cuts;
  __shared__ __align__(16) float own_o[OWN ? COLS * D : 4];  // what this CTA has of its line
  __shared__ float2 own_ml[OWN ? COLS : 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  if (tid < 2 * WARPS) cuts.line[tid] = -1;
  grid_dep_wait();
  grid_dep_launch();

  const int rows = p.kv_heads * p.chunks;  // lines of tiles of a request
  // ---- this CTA's part of the line
  long long c0 = 0, c1 = 0;
  int own_b = 0, own_row = 0, own_n = 0;
  const int own_rank = OWN ? static_cast<int>(blockIdx.x % p.split) : 0;
  bool alone = true;  // one CTA has all of it
  if constexpr (OWN) {
    const int line = static_cast<int>(blockIdx.x / p.split);
    own_b = line / rows, own_row = line - own_b * rows;
    int first, end;
    visible(p, own_b, first, end);
    own_n = static_cast<int>((static_cast<unsigned>(end - first) + (KEYS - 1)) / KEYS);
    c0 = static_cast<long long>(own_n) * own_rank / p.split, c1 = static_cast<long long>(own_n) * (own_rank + 1) / p.split;
    alone = p.split == 1 || own_n <= 1;
    if (own_n == 0) {
      const int kvh = own_row / p.chunks, col0 = (own_row - kvh * p.chunks) * COLS, head0 = kvh * p.group + col0;
      if (own_rank == 0)
        for (int i = tid; i < min(COLS, p.group - col0) * (D / 8); i += WARPS * 32) {
          const int head = head0 + i / (D / 8);
          *reinterpret_cast<uint4*>(p.out + own_b * p.out_sb + head * p.out_sh + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
          if (p.lse != nullptr && i % (D / 8) == 0) p.lse[static_cast<long long>(own_b) * p.heads + head] = -INFINITY;
        }
      return;
    }
    if (tid < COLS) own_ml[tid] = make_float2(-INFINITY, 0.f);
    __syncthreads();
  } else {
    // the tiles ahead of each request
    int run = 0;
    for (int b0 = 0; b0 < p.batch; b0 += WARPS * 32) {
      const int b = b0 + tid;
      int n = 0;
      if (b < p.batch) {
        int first, end;
        visible(p, b, first, end);
        n = static_cast<int>((static_cast<unsigned>(end - first) + (KEYS - 1)) / KEYS);
      }
      int x = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      if (lane == 31) warp_sum[warp] = x;
      __syncthreads();
      int before = run, all = run;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += warp_sum[w];
        all += warp_sum[w];
      }
      if (b < p.batch) prefix[b] = before + x - n;
      run = all;
      __syncthreads();
    }
    if (tid == 0) prefix[p.batch] = run;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int b = tid; b <= p.batch; b += WARPS * 32) p.prefix[b] = prefix[b];

    const long long units = static_cast<long long>(run) * rows;
    if (units == 0) return;
    const Shares shares(units, p.set);
    if (static_cast<int>(blockIdx.x) >= shares.ctas) return;
    c0 = shares.begin(blockIdx.x), c1 = shares.begin(blockIdx.x + 1);
  }
  // Warps with a part, of one tile or more.  (Of 4 tiles or more, so that some had none, a short context took 12.6 us, not 10.9.)
  const long long busy = min(static_cast<long long>(WARPS), c1 - c0);
  long long u = 0, u_end = 0;
  if (warp < busy) u = c0 + (c1 - c0) * warp / busy, u_end = c0 + (c1 - c0) * (warp + 1) / busy;

  // Line and tile of unit x: the largest b with prefix[b] <= x / rows has it.
  struct Place {
    int b, row, tile, n;
  };
  auto place_of = [&](long long x) {
    if constexpr (OWN) return Place{own_b, own_row, static_cast<int>(x), own_n};
    Place at;
    const int ahead = static_cast<int>(static_cast<double>(x) / rows);  // (exact: x < 2^40, rows < 2^17)
    int lo = 0, hi = p.batch;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= ahead) lo = mid;
      else hi = mid;
    }
    at.b = lo;
    at.n = prefix[lo + 1] - prefix[lo];
    const long long rest = x - static_cast<long long>(prefix[lo]) * rows;
    at.row = static_cast<int>(static_cast<double>(rest) / at.n);
    at.tile = static_cast<int>(rest - static_cast<long long>(at.row) * at.n);
    return at;
  };

  // ---- the fetching side: which tile comes next, and where this lane's rows of it lie
  const uint32_t ring = smem_u32(smem + warp * STAGES * STAGE);
  long long next = u;  // unit
  int left = 0;        // tiles of its line from it on
  unsigned key = 0, end = 0;  // (up to 31 behind the last key of a request, which may be 2^31 - 1)
  int page = -1;
  const int* table = nullptr;
  const __nv_bfloat16 *from_k = nullptr, *from_v = nullptr;
  auto look_up = [&]() {  // the page of this lane's key, a tile ahead of the copies
    page = next < u_end && key < end ? table[key / static_cast<unsigned>(p.page_size)] : -1;
  };
  auto enter = [&]() {  // the line of `next`
    const Place at = place_of(next);
    const int kvh = at.row / p.chunks;
    int first, last;
    visible(p, at.b, first, last);
    end = static_cast<unsigned>(last);
    key = static_cast<unsigned>(first) + static_cast<unsigned>(at.tile) * KEYS + (lane & (KEYS - 1));
    left = at.n - at.tile;
    table = p.table + at.b * p.table_sb;
    from_k = p.k + kvh * p.k_sh;
    from_v = p.v + kvh * p.v_sh;
  };
  // Fetches tile `next` into a stage, zeros where a key is not there, and goes on to the one behind it; returns which of its keys
  // there are.
  auto fetch = [&](int stage) -> uint32_t {
    uint32_t mask = 0;
    if (next < u_end) {
      const int slot = static_cast<int>(key % static_cast<unsigned>(p.page_size));
      const bool live = page >= 0 && page < p.pages;
      mask = __ballot_sync(0xffffffffu, live);
      // Where this lane's row lies; D = 128: lanes 16 to 31 have the same keys again and hold the places of their values.
      const bool value = D == 128 && lane >= 16;
      const long long at = value ? page * p.v_sp + slot * p.v_ss : page * p.k_sp + slot * p.k_ss;
      const char* mine = live ? reinterpret_cast<const char*>((value ? from_v : from_k) + at) : nullptr;
      const char* mine_v = live ? reinterpret_cast<const char*>(from_v + page * p.v_sp + slot * p.v_ss) : nullptr;  // (D = 64)
      const uint32_t to = ring + stage * STAGE + (lane >> 3) * RS + (lane & 7) * 16;
#pragma unroll
      for (int j = 0; j < 2 * KEYS / 4; ++j) {
        const char* of = D == 128 || j < KEYS / 4 ? mine : mine_v;
        const char* row =
            reinterpret_cast<const char*>(__shfl_sync(0xffffffffu, reinterpret_cast<long long>(of), (4 * j + (lane >> 3)) & 31));
        const char* from = row != nullptr ? row + (lane & 7) * 16 : reinterpret_cast<const char*>(p.q);
        const int bytes = row != nullptr ? 16 : 0;
#pragma unroll
        for (int h = 0; h < D / 64; ++h) copy_16(to + 4 * j * RS + h * 128, from + (row != nullptr ? h * 128 : 0), bytes);
      }
      ++next, --left, key += KEYS;
      if (left == 0 && next < u_end) enter();
      look_up();
    }
    copies_commit();
    return mask;
  };
  uint32_t live_of[STAGES];
  if (u < u_end) {
    enter();
    look_up();
  }
#pragma unroll
  for (int s = 0; s < STAGES; ++s) live_of[s] = fetch(s);

  const float sm2 = p.scale * LOG2E, cap2 = p.cap * LOG2E;
  const float to_cap = p.cap > 0.f ? p.scale / p.cap : 0.f;
  int stage = 0;
  while (u < u_end) {
    const Place at = place_of(u);
    const int t0 = at.tile, t1 = static_cast<int>(min(static_cast<long long>(at.n), t0 + (u_end - u)));
    const int kvh = at.row / p.chunks, col0 = (at.row - kvh * p.chunks) * COLS;
    const int cols = min(COLS, p.group - col0);
    const int head0 = kvh * p.group + col0;

    // ---- q: thread (g, t) has the pieces 2 t, 2 t + 1 (and those 8 further on) of column g
    uint4 qf[NT][KCH];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < KCH; ++i) {
        qf[j][i] = make_uint4(0, 0, 0, 0);
        if (j * 8 + g < cols)
          qf[j][i] = ld_nc_v4(p.q + at.b * p.q_sb + (head0 + j * 8 + g) * p.q_sh + (2 * t + (i & 1) + 8 * (i >> 1)) * 8);
      }

    float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      m[j][0] = m[j][1] = -INFINITY;
      l[j][0] = l[j][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;
    }
#pragma unroll 1
    for (int tile = t0; tile < t1; ++tile) {
      copies_wait<STAGES - 1>();
      __syncwarp();
      const uint32_t live = live_of[0];
      const char* keys = smem + (warp * STAGES + stage) * STAGE;
      const char* values = keys + KEYS * RS;
      // ---- scores^T: rows are keys, columns query heads
      float s[SUB][NT][4];
#pragma unroll
      for (int x = 0; x < SUB; ++x) {
#pragma unroll
        for (int j = 0; j < NT; ++j) s[x][j][0] = s[x][j][1] = s[x][j][2] = s[x][j][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KCH; ++i) {
          const char* piece = keys + (x * 16 + g) * RS + (2 * t + (i & 1) + 8 * (i >> 1)) * 16;
          const uint4 a = ld_shared_v4(piece), b = ld_shared_v4(piece + 8 * RS);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            mma_bf16(s[x][j], a.x, b.x, a.y, b.y, qf[j][i].x, qf[j][i].y);
            mma_bf16(s[x][j], a.z, b.z, a.w, b.w, qf[j][i].z, qf[j][i].w);
          }
        }
      }
      // ---- this thread's values
      uint4 vf[SUB][4][VCH];
#pragma unroll
      for (int x = 0; x < SUB; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = x * 16 + 2 * t + (r & 1) + (r >> 1) * 8;
#pragma unroll
          for (int i = 0; i < VCH; ++i) vf[x][r][i] = ld_shared_v4(values + row * RS + (g + 8 * i) * 16);
        }
      constexpr uint32_t ALL = KEYS == 32 ? 0xFFFFFFFFu : (1u << (KEYS & 31)) - 1;
      const bool every = (live & ALL) == ALL;
      // ---- the stage is free for the tile STAGES further on
      __syncwarp();
#pragma unroll
      for (int i = 0; i + 1 < STAGES; ++i) live_of[i] = live_of[i + 1];
      live_of[STAGES - 1] = fetch(stage);
      if (++stage == STAGES) stage = 0;

      // ---- running softmax, in powers of 2
      uint32_t pf[SUB][NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < SUB; ++x)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float y = s[x][j][c];
            y = p.cap > 0.f ? cap2 * tanhf(y * to_cap) : y * sm2;
            if (!every) y = (live >> (x * 16 + g + (c >> 1) * 8)) & 1 ? y : -INFINITY;
            s[x][j][c] = y;
            top[c & 1] = fmaxf(top[c & 1], y);
          }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
          top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
        }
        if (__any_sync(0xffffffffu, top[0] > m[j][0] || top[1] > m[j][1])) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float now = fmaxf(m[j][c], top[c]);
            const float f = m[j][c] == -INFINITY ? 0.f : ex2(m[j][c] - now);
            m[j][c] = now;
            l[j][c] *= f;
#pragma unroll
            for (int i = 0; i < MT; ++i) o[j][i][c] *= f, o[j][i][c + 2] *= f;
          }
        }
        const float m0 = m[j][0] == -INFINITY ? 0.f : m[j][0], m1 = m[j][1] == -INFINITY ? 0.f : m[j][1];
#pragma unroll
        for (int x = 0; x < SUB; ++x) {
          const float p0 = ex2(s[x][j][0] - m0), p1 = ex2(s[x][j][1] - m1);
          const float p2 = ex2(s[x][j][2] - m0), p3 = ex2(s[x][j][3] - m1);
          l[j][0] += p0 + p2;
          l[j][1] += p1 + p3;
          pf[x][j][0] = transpose_8x8(pack_bf16x2(p0, p1));
          pf[x][j][1] = transpose_8x8(pack_bf16x2(p2, p3));
        }
      }
      // ---- out^T += V^T p^T: row i of a 16-row tile is an element of piece g (and g + 8) of the value rows
#pragma unroll
      for (int x = 0; x < SUB; ++x)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          constexpr int H = D == 128 ? 0 : 2;  // D = 64: the upper 8 rows are the piece's upper half
          const int w0 = i >> 1, w1 = (i >> 1) + H, c1 = VCH - 1;
          const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
          const uint32_t a0 = __byte_perm(word(vf[x][0][0], w0), word(vf[x][1][0], w0), sel);
          const uint32_t a1 = __byte_perm(word(vf[x][0][c1], w1), word(vf[x][1][c1], w1), sel);
          const uint32_t a2 = __byte_perm(word(vf[x][2][0], w0), word(vf[x][3][0], w0), sel);
          const uint32_t a3 = __byte_perm(word(vf[x][2][c1], w1), word(vf[x][3][c1], w1), sel);
#pragma unroll
          for (int j = 0; j < NT; ++j) mma_bf16(o[j][i], a0, a1, a2, a3, pf[x][j][0], pf[x][j][1]);
        }
    }

    // ---- the sums over the keys; out, or the partial result
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[j][c] += __shfl_xor_sync(0xffffffffu, l[j][c], d);
    const bool whole = t0 == 0 && t1 == at.n, last = u + (t1 - t0) == u_end;
    const int entry = 2 * warp + (t0 == 0);
    if (!whole && last) {  // the ring is empty (copies of nothing but zeros may be under way)
      copies_wait<0>();
      __syncwarp();
    }
    if (!whole && lane == 0) {
      cuts.line[entry] = static_cast<long long>(at.b) * rows + at.row;
      cuts.starts[entry] = t0 == 0, cuts.ends[entry] = t1 == at.n, cuts.in_ring[entry] = last;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = j * 8 + 2 * t + c;
        if (col >= cols) continue;
        // element e of this thread's 8 (D = 128: in each half of the row)
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (D == 128) lo[e] = o[j][e % MT][c], hi[e] = o[j][e % MT][c + 2];
          else lo[e] = e < 4 ? o[j][e & 3][c] : o[j][e & 3][c + 2];
        }
        if (whole) {
          const float inv = l[j][c] == 0.f ? 0.f : 1.f / l[j][c];
          __nv_bfloat16* to = p.out + at.b * p.out_sb + (head0 + col) * p.out_sh + g * 8;
          uint4 w;
          w.x = pack_bf16x2(lo[0] * inv, lo[1] * inv), w.y = pack_bf16x2(lo[2] * inv, lo[3] * inv);
          w.z = pack_bf16x2(lo[4] * inv, lo[5] * inv), w.w = pack_bf16x2(lo[6] * inv, lo[7] * inv);
          *reinterpret_cast<uint4*>(to) = w;
          if (D == 128) {
            w.x = pack_bf16x2(hi[0] * inv, hi[1] * inv), w.y = pack_bf16x2(hi[2] * inv, hi[3] * inv);
            w.z = pack_bf16x2(hi[4] * inv, hi[5] * inv), w.w = pack_bf16x2(hi[6] * inv, hi[7] * inv);
            *reinterpret_cast<uint4*>(to + 64) = w;
          }
          if (p.lse != nullptr && g == 0)
            p.lse[static_cast<long long>(at.b) * p.heads + head0 + col] =
                l[j][c] == 0.f ? -INFINITY : (m[j][c] + log2f(l[j][c])) * LN2;
        } else {
          float* to = (last ? reinterpret_cast<float*>(smem + warp * STAGES * STAGE)
                            : p.warp_o + (static_cast<long long>(blockIdx.x) * WARPS + warp) * COLS * D) + col * D + g * 8;
          *reinterpret_cast<float4*>(to) = make_float4(lo[0], lo[1], lo[2], lo[3]);
          *reinterpret_cast<float4*>(to + 4) = make_float4(lo[4], lo[5], lo[6], lo[7]);
          if (D == 128) {
            *reinterpret_cast<float4*>(to + 64) = make_float4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<float4*>(to + 68) = make_float4(hi[4], hi[5], hi[6], hi[7]);
          }
          if (g == 0) cuts.ml[entry][col] = make_float2(m[j][c], l[j][c]);
        }
      }
    u += t1 - t0;
  }
  __syncthreads();

  // ---- joins what the warps have of the same line, in the order of the keys
  for (int e0 = 0, e1; e0 < 2 * WARPS; e0 = e1) {
    e1 = e0 + 1;
    const long long line = cuts.line[e0];
    if (line < 0) continue;
    int last = e0;
    while (e1 < 2 * WARPS && (cuts.line[e1] < 0 || cuts.line[e1] == line)) {
      if (cuts.line[e1] == line) last = e1;
      ++e1;
    }
    const int b = static_cast<int>(line / rows), row = static_cast<int>(line - static_cast<long long>(b) * rows);
    const int kvh = row / p.chunks, col0 = (row - kvh * p.chunks) * COLS;
    const int cols = min(COLS, p.group - col0), head0 = kvh * p.group + col0;
    const bool whole = cuts.starts[e0] && cuts.ends[last];
    for (int i = tid; i < cols * (D / 4); i += WARPS * 32) {
      const int col = i / (D / 4), d = i % (D / 4) * 4;
      float top = -INFINITY, l = 0.f;
      for (int e = e0; e <= last; ++e)
        if (cuts.line[e] == line) top = fmaxf(top, cuts.ml[e][col].x);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int e = e0; e <= last; ++e) {
        if (cuts.line[e] != line) continue;
        const float2 ml = cuts.ml[e][col];
        const float4 x = cuts.in_ring[e]
                             ? *reinterpret_cast<const float4*>(smem + (e >> 1) * STAGES * STAGE + (col * D + d) * 4)
                             : __ldcg(reinterpret_cast<const float4*>(
                                   p.warp_o + (static_cast<long long>(blockIdx.x) * WARPS + (e >> 1)) * COLS * D + col * D + d));
        const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(ml.x - top);  // (1: NaN, which stays)
        l += f * ml.y;
        sum.x += f * x.x, sum.y += f * x.y, sum.z += f * x.z, sum.w += f * x.w;
      }
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<uint2*>(p.out + b * p.out_sb + (head0 + col) * p.out_sh + d) =
            make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
        if (p.lse != nullptr && d == 0)
          p.lse[static_cast<long long>(b) * p.heads + head0 + col] = l == 0.f ? -INFINITY : (top + log2f(l)) * LN2;
      } else if constexpr (OWN) {
        *reinterpret_cast<float4*>(own_o + col * D + d) = sum;
        if (d == 0) own_ml[col] = make_float2(top, l);
      } else {
        const long long slot = (2LL * blockIdx.x + (cuts.starts[e0] != 0)) * COLS + col;
        *reinterpret_cast<float4*>(p.part_o + slot * D + d) = sum;
        if (d == 0) p.part_ml[slot] = make_float2(top, l);
      }
    }
  }
  if constexpr (OWN) {
    if (alone) return;
    // ---- and what the CTAs have of it
    const cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int kvh = own_row / p.chunks, col0 = (own_row - kvh * p.chunks) * COLS, head0 = kvh * p.group + col0;
    const int cols = min(COLS, p.group - col0);
    for (int i = own_rank * WARPS * 32 + tid; i < cols * (D / 4); i += p.split * WARPS * 32) {
      const int col = i / (D / 4), d = i % (D / 4) * 4;
      float2 ml[MAX_SPLIT];
      float4 x[MAX_SPLIT];
      float top = -INFINITY, l = 0.f;
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c) {
        ml[c] = c < p.split ? *cluster.map_shared_rank(&own_ml[col], c) : make_float2(-INFINITY, 0.f);
        // (a CTA without a tile has no output there)
        x[c] = ml[c].x == -INFINITY && ml[c].y == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                                      : *reinterpret_cast<const float4*>(cluster.map_shared_rank(own_o + col * D + d, c));
        top = fmaxf(top, ml[c].x);
      }
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c) {
        const float f = ml[c].x == -INFINITY ? (ml[c].y == 0.f ? 0.f : 1.f) : ex2(ml[c].x - top);  // (1: NaN, which stays)
        l += f * ml[c].y;
        sum.x += f * x[c].x, sum.y += f * x[c].y, sum.z += f * x[c].z, sum.w += f * x[c].w;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      *reinterpret_cast<uint2*>(p.out + own_b * p.out_sb + (head0 + col) * p.out_sh + d) =
          make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
      if (p.lse != nullptr && d == 0)
        p.lse[static_cast<long long>(own_b) * p.heads + head0 + col] = l == 0.f ? -INFINITY : (top + log2f(l)) * LN2;
    }
    cluster.sync();  // (nobody's shared memory goes while it is read)
  }
}

// Joins the partial results of each (request, head), `items` of them per CTA: a warp takes one that has a few; those that have more
// all warps share, and their sums meet in the order of the warps.  Requests that see no key get zeros and -inf here.
constexpr int FEW = 16;
template <int D, int COLS>
__global__ void __launch_bounds__(JOIN_WARPS * 32) attn_decode_join_kernel(const Params p, int items) {
  __shared__ float4 sums[JOIN_WARPS][D / 4];
  __shared__ float2 mls[JOIN_WARPS];
  __shared__ int firsts[JOIN_WARPS], lasts[JOIN_WARPS];
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int LANES = D / 4;  // of a partial result; D = 64: a warp takes two at a time
  constexpr int PER = 32 / LANES;
  const long long item0 = static_cast<long long>(blockIdx.x) * items, all = static_cast<long long>(p.batch) * p.heads;
  auto column = [&](int head) { return (head % p.group) % COLS; };
  float4 sum;
  float top, l;
  // Partial results c = from, from + step, .. <= last of a line whose first is `first`, into top, l and sum.
  auto take = [&](int first, int last, int from, int step, int col) {
    top = -INFINITY, l = 0.f, sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = from + lane / LANES; c - lane / LANES <= last; c += 4 * step) {
      float2 ml[4];
      float4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int at = c + k * step;
        const long long slot = (2LL * at + (at == first)) * COLS + col;
        ml[k] = at <= last ? p.part_ml[slot] : make_float2(-INFINITY, 0.f);
        x[k] = at <= last ? *reinterpret_cast<const float4*>(p.part_o + slot * D + lane % LANES * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      const float now = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), top);
      const float old = top == -INFINITY ? 1.f : ex2(top - now);  // (1: zeros so far, or NaN, which stays)
      top = now;
      l *= old, sum.x *= old, sum.y *= old, sum.z *= old, sum.w *= old;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = ml[k].x == -INFINITY ? (ml[k].y == 0.f ? 0.f : 1.f) : ex2(ml[k].x - now);
        l += f * ml[k].y;
        sum.x += f * x[k].x, sum.y += f * x[k].y, sum.z += f * x[k].z, sum.w += f * x[k].w;
      }
    }
    if (PER == 2) {  // the halves' sums
      const float other = __shfl_xor_sync(0xffffffffu, top, 16), now = fmaxf(top, other);
      const float f = top == -INFINITY ? 1.f : ex2(top - now), g = other == -INFINITY ? 1.f : ex2(other - now);
      const bool low = lane < 16;  // (in the same order in both)
      auto both = [&](float v) {
        const float o = __shfl_xor_sync(0xffffffffu, v, 16);
        return low ? f * v + g * o : g * o + f * v;
      };
      l = both(l), sum.x = both(sum.x), sum.y = both(sum.y), sum.z = both(sum.z), sum.w = both(sum.w);
      top = now;
    }
  };
  auto write = [&](int b, int head) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (lane < LANES)
      *reinterpret_cast<uint2*>(p.out + b * p.out_sb + head * p.out_sh + lane * 4) =
          make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
    if (p.lse != nullptr && lane == 0)
      p.lse[static_cast<long long>(b) * p.heads + head] = l == 0.f ? -INFINITY : (top + log2f(l)) * LN2;
  };
  if (warp < items) {
    const long long item = item0 + warp;
    int first = 0, last = 0;
    if (item < all) {
      const int b = static_cast<int>(item / p.heads), head = static_cast<int>(item - static_cast<long long>(b) * p.heads);
      const int ahead = p.prefix[b], n = p.prefix[b + 1] - ahead;
      if (n > 0) {
        const int rows = p.kv_heads * p.chunks, row = head / p.group * p.chunks + head % p.group / COLS;
        const Shares shares(static_cast<long long>(p.prefix[p.batch]) * rows, p.set);
        const long long u0 = static_cast<long long>(ahead) * rows + static_cast<long long>(row) * n;
        first = shares.of(u0);
        last = first + 1 >= shares.ctas || shares.begin(first + 1) >= u0 + n ? first : shares.of(u0 + n - 1);
        if (first < last && last - first < FEW) {  // (first == last: one CTA had all of it)
          take(first, last, first, PER, column(head));
          write(b, head);
          last = first;
        }
      } else {
        top = -INFINITY, l = 0.f, sum = make_float4(0.f, 0.f, 0.f, 0.f);
        write(b, head);
      }
    }
    if (lane == 0) firsts[warp] = first, lasts[warp] = last;
  }
  __syncthreads();
  for (int i = 0; i < items; ++i) {
    const int first = firsts[i], last = lasts[i];
    if (first == last) continue;
    const int b = static_cast<int>((item0 + i) / p.heads), head = static_cast<int>(item0 + i - static_cast<long long>(b) * p.heads);
    take(first, last, first + warp * PER, JOIN_WARPS * PER, column(head));
    if (lane < LANES) sums[warp][lane] = sum;
    if (lane == 0) mls[warp] = make_float2(top, l);
    __syncthreads();
    if (warp == 0) {
      top = -INFINITY;
      for (int w = 0; w < JOIN_WARPS; ++w) top = fmaxf(top, mls[w].x);
      l = 0.f, sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < JOIN_WARPS; ++w) {
        const float f = mls[w].x == -INFINITY ? 1.f : ex2(mls[w].x - top);
        const float4 x = sums[w][lane % LANES];
        l += f * mls[w].y;
        sum.x += f * x.x, sum.y += f * x.y, sum.z += f * x.z, sum.w += f * x.w;
      }
      write(b, head);
    }
    __syncthreads();
  }
}
}  // namespace decode

// Bytes of the scratch: tiles ahead of each request, then the partial results, two of a CTA and one of each of its warps.
static size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }
static int tiles_of_columns(long long group) { return group <= 8 ? 1 : 2; }
static int32_t decode_shapes(const char* op, const cdl_tensor* q, const cdl_tensor* k_cache) {
  if (!q || !k_cache) return fail(CDL_ERR_INVALID, "%s: q and k_cache are required", op);
  if (q->rank != 3 || q->dtype != CDL_BF16) return fail(CDL_ERR_INVALID, "%s: q must be bf16 [batch, heads, head_dim]", op);
  if (k_cache->rank != 4 || k_cache->dtype != CDL_BF16)
    return fail(CDL_ERR_INVALID, "%s: the caches must be bf16 [pages, page_size, kv_heads, head_dim]", op);
  const long long d = q->shape[2];
  if (d != 64 && d != 128) return fail(CDL_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128 (got %lld)", op, d);
  if (k_cache->shape[3] != d) return fail(CDL_ERR_INVALID, "%s: head_dim of q and of the cache differ", op);
  if (q->shape[0] < 0 || q->shape[0] > decode::MAX_BATCH)
    return fail(CDL_ERR_UNSUPPORTED, "%s: at most %d requests (got %lld)", op, decode::MAX_BATCH, (long long)q->shape[0]);
  if (q->shape[1] < 0 || k_cache->shape[2] <= 0 || q->shape[1] % k_cache->shape[2] != 0)
    return fail(CDL_ERR_INVALID, "%s: heads (%lld) must be a multiple of kv_heads (%lld)", op, (long long)q->shape[1],
                (long long)k_cache->shape[2]);
  if (q->shape[1] > 65536) return fail(CDL_ERR_UNSUPPORTED, "%s: at most 65536 heads", op);
  return CDL_OK;
}

static size_t decode_scratch_bytes(long long batch, int nt, long long d) {
  const size_t ctas = static_cast<size_t>(decode::SETS) * sm_count() * decode::ctas_per_sm(nt), cols = 8 * nt;
  return align256((batch + 1) * 4) + align256(2 * ctas * cols * 8) + (2 + decode::WARPS) * ctas * cols * d * 4;
}

// Rows of `d` elements from a 16-byte boundary on, whatever the strides of the outer dimensions.
static int32_t check_rows(const char* op, const char* name, const cdl_tensor* t) {
  const int last = t->rank - 1;
  bool ok = (reinterpret_cast<uintptr_t>(t->ptr) & 15) == 0 && (t->shape[last] <= 1 || t->stride[last] == 1);
  for (int i = 0; i < last; ++i) ok = ok && (t->shape[i] <= 1 || (t->stride[i] % 8 == 0 && t->stride[i] >= 0));
  return ok ? CDL_OK
            : fail(CDL_ERR_INVALID, "%s: %s must have a contiguous last dimension, 16-byte aligned, and other strides that are multiples of 8",
                   op, name);
}

int32_t attn_decode_execute(const cdl_attn_decode_desc* desc, const cdl_tensor* q, const cdl_tensor* k_cache,
                            const cdl_tensor* v_cache, const cdl_tensor* block_table, const cdl_tensor* seq_lens,
                            const cdl_tensor* out, const cdl_tensor* lse, void* scratch, size_t scratch_bytes,
                            cudaStream_t stream) {
  const char* op = "attn_decode";
  if (!desc || !v_cache || !block_table || !seq_lens || !out)
    return fail(CDL_ERR_INVALID, "%s: desc, v_cache, block_table, seq_lens and out are required", op);
  CDL_CHECK(decode_shapes(op, q, k_cache));
  const long long B = q->shape[0], H = q->shape[1], D = q->shape[2], Hkv = k_cache->shape[2];
  const long long pages = k_cache->shape[0], page_size = k_cache->shape[1];
  if (v_cache->rank != 4 || v_cache->dtype != CDL_BF16) return fail(CDL_ERR_INVALID, "%s: v_cache must have k_cache's type and shape", op);
  for (int i = 0; i < 4; ++i)
    if (v_cache->shape[i] != k_cache->shape[i]) return fail(CDL_ERR_INVALID, "%s: v_cache must have k_cache's type and shape", op);
  if (page_size <= 0 || pages < 0 || pages > INT32_MAX || page_size > INT32_MAX)
    return fail(CDL_ERR_INVALID, "%s: pages must be 0 to 2^31 - 1 and hold a key at least", op);
  if (block_table->rank != 2 || block_table->dtype != CDL_I32 || block_table->shape[0] != B || block_table->shape[1] < 0 ||
      (block_table->shape[1] > 1 && block_table->stride[1] != 1))
    return fail(CDL_ERR_INVALID, "%s: block_table must be i32 [batch, pages of a request] with contiguous rows", op);
  if (seq_lens->rank != 1 || seq_lens->dtype != CDL_I32 || seq_lens->shape[0] != B || (B > 1 && seq_lens->stride[0] != 1))
    return fail(CDL_ERR_INVALID, "%s: seq_lens must be a packed i32 [batch]", op);
  if (out->rank != 3 || out->dtype != CDL_BF16 || out->shape[0] != B || out->shape[1] != H || out->shape[2] != D)
    return fail(CDL_ERR_INVALID, "%s: out must have q's type and shape", op);
  if (lse && (lse->rank != 2 || lse->dtype != CDL_F32 || lse->shape[0] != B || lse->shape[1] != H ||
              (H > 1 && lse->stride[1] != 1) || (B > 1 && lse->stride[0] != H)))
    return fail(CDL_ERR_INVALID, "%s: lse must be a packed f32 [batch, heads]", op);
  CDL_CHECK(check_rows(op, "q", q));
  CDL_CHECK(check_rows(op, "k_cache", k_cache));
  CDL_CHECK(check_rows(op, "v_cache", v_cache));
  CDL_CHECK(check_rows(op, "out", out));
  if (!(desc->softcap >= 0.f) || isinf(desc->softcap)) return fail(CDL_ERR_INVALID, "%s: softcap must be 0 (none) or positive", op);
  if (isnan(desc->softmax_scale) || isinf(desc->softmax_scale)) return fail(CDL_ERR_INVALID, "%s: softmax_scale must be finite", op);
  const float scale = desc->softmax_scale > 0.f ? desc->softmax_scale : 1.f / sqrtf(static_cast<float>(D));
  // (the kernel's scale / cap, scale log2 e and cap log2 e are finite then, and the first is not denormal)
  if (scale > 0x1p126f || desc->softcap > 0x1p126f ||
      (desc->softcap > 0.f && (scale / desc->softcap < FLT_MIN || scale / desc->softcap > FLT_MAX)))
    return fail(CDL_ERR_INVALID, "%s: softmax_scale and softcap must be at most 2^126 and their quotient a normal f32 number", op);
  if (desc->window < 0) return fail(CDL_ERR_INVALID, "%s: window must be 0 (all keys) or positive", op);
  if (B == 0 || H == 0) return CDL_OK;
  const void* given[] = {q->ptr, seq_lens->ptr, out->ptr};
  for (const void* x : given)
    if (!x) return fail(CDL_ERR_INVALID, "%s: null pointer", op);
  const long long width = pages == 0 ? 0 : block_table->shape[1];
  if ((lse && !lse->ptr) || (width > 0 && (!block_table->ptr || !k_cache->ptr || !v_cache->ptr)))
    return fail(CDL_ERR_INVALID, "%s: null pointer", op);
  if (!view_apart_from_itself(*out)) return fail(CDL_ERR_INVALID, "%s: elements of out overlap", op);
  const cdl_tensor* ins[] = {q, k_cache, v_cache, block_table, seq_lens};
  for (const cdl_tensor* i : ins)
    if (!views_apart(*out, *i) || (lse && !views_apart(*lse, *i))) return fail(CDL_ERR_INVALID, "%s: an output overlaps an input", op);
  if (lse && !views_apart(*out, *lse)) return fail(CDL_ERR_INVALID, "%s: out and lse overlap", op);
  const long long group = H / Hkv;
  const int nt = tiles_of_columns(group), cols = 8 * nt;
  const long long chunks = (group + cols - 1) / cols, rows = Hkv * chunks;
  const long long tile = D == 128 ? decode::tile_keys<128>() : decode::tile_keys<64>();
  long long most = width > INT32_MAX / page_size ? INT32_MAX : width * page_size;  // keys of a request
  if (desc->window > 0) most = std::min<long long>(most, desc->window);
  const long long tiles = B * ((most + tile - 1) / tile);
  if (tiles > INT32_MAX) return fail(CDL_ERR_UNSUPPORTED, "%s: more than 2^31 tiles of keys in the block table", op);
  if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 255) || scratch_bytes < decode_scratch_bytes(B, nt, D))
    return fail(CDL_ERR_INVALID, "%s: scratch must be 256-byte aligned and hold %zu bytes", op, decode_scratch_bytes(B, nt, D));

  if (tiles * rows > (1LL << 40)) return fail(CDL_ERR_UNSUPPORTED, "%s: more than 2^40 tiles of keys", op);
  const size_t rings = decode::WARPS * decode::STAGES * (D == 128 ? decode::stage_bytes<128>() : decode::stage_bytes<64>());
  const size_t smem = rings + (B + 1) * sizeof(int);
  // CTAs that run at once
  const int set = sm_count() * std::min(decode::ctas_per_sm(nt), decode::ctas_by_memory(nt, smem));
  const int grid = std::max(1, decode::Shares(tiles * rows, set).ctas);  // (the lengths may leave some without a part)
  decode::Params p{};
  p.q = static_cast<const __nv_bfloat16*>(q->ptr), p.q_sb = q->stride[0], p.q_sh = q->stride[1];
  p.k = static_cast<const __nv_bfloat16*>(k_cache->ptr), p.v = static_cast<const __nv_bfloat16*>(v_cache->ptr);
  p.k_sp = k_cache->stride[0], p.k_ss = k_cache->stride[1], p.k_sh = k_cache->stride[2];
  p.v_sp = v_cache->stride[0], p.v_ss = v_cache->stride[1], p.v_sh = v_cache->stride[2];
  p.table = static_cast<const int*>(block_table->ptr), p.table_sb = block_table->stride[0];
  p.lens = static_cast<const int*>(seq_lens->ptr);
  p.batch = static_cast<int>(B), p.heads = static_cast<int>(H), p.kv_heads = static_cast<int>(Hkv);
  p.group = static_cast<int>(group), p.chunks = static_cast<int>(chunks);
  p.pages = static_cast<int>(pages), p.page_size = static_cast<int>(page_size);
  p.width = static_cast<int>(std::min<long long>(width, INT32_MAX)), p.window = desc->window;
  p.scale = scale, p.cap = desc->softcap;
  p.out = static_cast<__nv_bfloat16*>(out->ptr), p.out_sb = out->stride[0], p.out_sh = out->stride[1];
  p.lse = lse ? static_cast<float*>(lse->ptr) : nullptr;
  p.set = set;
  char* at = static_cast<char*>(scratch);
  const size_t ctas = static_cast<size_t>(decode::SETS) * set;
  p.prefix = reinterpret_cast<int*>(at), at += align256((B + 1) * 4);
  p.part_ml = reinterpret_cast<float2*>(at), at += align256(2 * ctas * cols * 8);
  p.part_o = reinterpret_cast<float*>(at), at += 2 * ctas * cols * D * 4;
  p.warp_o = reinterpret_cast<float*>(at);

  ProfileScope ps(PROF_ATTN_FWD, 4.0 * B * H * D * most, stream);
  const long long lines = B * rows;
  if (most <= decode::OWN_KEYS) {
    void (*own)(decode::Params) =
        D == 128 ? (nt == 1 ? decode::attn_decode_kernel<128, 1, true> : decode::attn_decode_kernel<128, 2, true>)
                 : (nt == 1 ? decode::attn_decode_kernel<64, 1, true> : decode::attn_decode_kernel<64, 2, true>);
    // CTAs of a line: a tile or more for each warp, and 7/8 of the places, which clusters do not fill (74 lines of 512 keys in 3 CTAs
    // each 10.2 us; in 4, one for each of 296 places, 14.5)
    const long long line_tiles = (most + tile - 1) / tile;
    p.split = static_cast<int>(std::max<long long>(
        1, std::min<long long>({decode::MAX_SPLIT, set * 7LL / 8 / lines, (line_tiles + decode::WARPS - 1) / decode::WARPS})));
    CDL_CUDA(allow_shared_memory(reinterpret_cast<const void*>(own), static_cast<int>(rings)));
    const dim3 of_lines(static_cast<unsigned>(lines * p.split)), block(decode::WARPS * 32);
    CDL_CUDA(p.split == 1 ? launch_pdl(own, of_lines, block, rings, stream, p)
                          : launch_pdl_cluster(own, of_lines, block, rings, p.split, stream, p));
    return CDL_OK;
  }
  void (*kernel)(decode::Params) =
      D == 128 ? (nt == 1 ? decode::attn_decode_kernel<128, 1, false> : decode::attn_decode_kernel<128, 2, false>)
               : (nt == 1 ? decode::attn_decode_kernel<64, 1, false> : decode::attn_decode_kernel<64, 2, false>);
  void (*join)(decode::Params, int) = D == 128 ? (nt == 1 ? decode::attn_decode_join_kernel<128, 8> : decode::attn_decode_join_kernel<128, 16>)
                                          : (nt == 1 ? decode::attn_decode_join_kernel<64, 8> : decode::attn_decode_join_kernel<64, 16>);
  // (the most that any call needs: two threads' calls of different batches never take it from one another)
  CDL_CUDA(allow_shared_memory(reinterpret_cast<const void*>(kernel), static_cast<int>(rings + (decode::MAX_BATCH + 1) * sizeof(int))));
  CDL_CUDA(launch_pdl(kernel, dim3(grid), dim3(decode::WARPS * 32), smem, stream, p));
  // items of a CTA: one while there are few, up to one per warp
  const int items = static_cast<int>(std::max<long long>(1, std::min<long long>(decode::JOIN_WARPS, B * H / (2 * sm_count()))));
  CDL_CUDA(launch_pdl(join, dim3(static_cast<unsigned>((B * H + items - 1) / items)), dim3(decode::JOIN_WARPS * 32), 0, stream, p, items));
  return CDL_OK;
}

}  // namespace cdl

extern "C" {

int32_t cdl_b200_attn_decode(const cdl_attn_decode_desc* desc, const cdl_tensor* q, const cdl_tensor* k_cache,
                             const cdl_tensor* v_cache, const cdl_tensor* block_table, const cdl_tensor* seq_lens,
                             const cdl_tensor* out, const cdl_tensor* lse, void* scratch, size_t scratch_bytes,
                             cdl_stream stream) {
  return cdl::attn_decode_execute(desc, q, k_cache, v_cache, block_table, seq_lens, out, lse, scratch, scratch_bytes,
                                  static_cast<cudaStream_t>(stream));
}
int32_t cdl_b200_attn_decode_scratch_bytes(const cdl_tensor* q, const cdl_tensor* k_cache, size_t* bytes_out) {
  if (!bytes_out) return cdl::fail(CDL_ERR_INVALID, "attn_decode: bytes_out is required");
  CDL_CHECK(cdl::decode_shapes("attn_decode", q, k_cache));
  *bytes_out = cdl::decode_scratch_bytes(q->shape[0], cdl::tiles_of_columns(q->shape[1] / k_cache->shape[2]), q->shape[2]);
  return CDL_OK;
}

}  // extern "C"
