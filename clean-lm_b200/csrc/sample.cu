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

#include <math.h>

namespace cdl {
namespace sample {

constexpr int THREADS = 1024, WARPS = THREADS / 32;
using u64 = unsigned long long;

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
};

// f32 values as unsigned numbers of the same order (-0 as 0).
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t b = __float_as_uint(z + 0.f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

template <typename T>
__device__ __forceinline__ float load(const void* z, long long i);
template <>
__device__ __forceinline__ float load<float>(const void* z, long long i) { return static_cast<const float*>(z)[i]; }
template <>
__device__ __forceinline__ float load<__nv_bfloat16>(const void* z, long long i) {
  return __uint_as_float(static_cast<uint32_t>(static_cast<const unsigned short*>(z)[i]) << 16);
}

__device__ __forceinline__ u64 warp_sum(u64 x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
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

struct Row {
  const void* z;
  long long vocab;
  float top;         // the largest logit
  double inv_t;      // of the temperature: 1 where the row is greedy
  double t;
  double scale;      // 2^S
  __device__ __forceinline__ u64 weight(float x) const {
    return static_cast<u64>(__double2ll_rn(exp((static_cast<double>(x) - static_cast<double>(top)) / t) * scale));
  }
};

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(const Params p) {
  __shared__ u64 sums[WARPS];
  __shared__ u64 hist[256];
  __shared__ float s_top[WARPS];
  __shared__ int s_at[WARPS];
  __shared__ uint32_t s_key;
  __shared__ u64 s_above, s_left;
  __shared__ long long s_index;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_wait();
  grid_dep_launch();
  const long long r = blockIdx.x;
  const long long V = p.vocab;
  const void* z = static_cast<const T*>(p.z) + r * p.ld;
  const float temperature = p.temperature ? p.temperature[r] : p.all_temperature;
  const long long k_in = p.top_k ? p.top_k[r] : p.all_top_k;
  const float top_p = p.top_p ? p.top_p[r] : p.all_top_p;
  const float min_p = p.min_p ? p.min_p[r] : p.all_min_p;

  // ---- the largest logit and its first place; NaN and +inf
  float top = -INFINITY;
  int at = 0;
  bool bad = false;
  for (long long i = tid; i < V; i += THREADS) {
    const float x = load<T>(z, i);
    bad |= !(x < INFINITY);
    if (x > top) top = x, at = static_cast<int>(i);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const float x = __shfl_xor_sync(0xffffffffu, top, d);
    const int y = __shfl_xor_sync(0xffffffffu, at, d);
    if (x > top || (x == top && y < at)) top = x, at = y;
  }
  if (lane == 0) s_top[warp] = top, s_at[warp] = at;
  bad = __syncthreads_or(bad);
  top = s_top[0], at = s_at[0];
  for (int w = 1; w < WARPS; ++w)
    if (s_top[w] > top || (s_top[w] == top && s_at[w] < at)) top = s_top[w], at = s_at[w];
  if (bad || top == -INFINITY) {
    if (tid == 0) {
      p.token[r] = -1;
      if (p.logprob) p.logprob[r] = __uint_as_float(0x7FC00000u);
    }
    return;
  }
  if (!(temperature > 0.f)) {
    if (tid == 0) {
      p.token[r] = at;
      if (p.logprob) p.logprob[r] = 0.f;
    }
    return;
  }
  Row row;
  row.z = z, row.vocab = V, row.top = top;
  row.t = static_cast<double>(temperature);
  row.scale = ldexp(1.0, p.scale_bits);

  // The kept entries: those above `cut` and, of those equal to it, the ones up to index `last`.
  uint32_t cut = 0;
  long long last = V;
  // Finds the entry at which the sum of f(entry) over the entries in falling order reaches `want`, among those kept so far:
  // 8 bits of the value at a time, then by index.  Sets cut and last, returns the sum up to and with that entry.
  auto select = [&](auto f, u64 want) -> u64 {
    const uint32_t old_cut = cut;
    const long long old_last = last;
    auto kept = [&](uint32_t key, long long i) { return key > old_cut || (key == old_cut && i <= old_last); };
    uint32_t prefix = 0;
    u64 above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (long long i = tid; i < V; i += THREADS) {
        const float x = load<T>(z, i);
        const uint32_t key = key_of(x);
        if (kept(key, i) && (shift == 24 || (key >> (shift + 8)) == prefix)) atomicAdd(&hist[(key >> shift) & 255], f(x));
      }
      __syncthreads();
      if (tid == 0) {
        u64 sum = above;
        int bin = 255;
        while (bin > 0 && sum + hist[bin] < want) sum += hist[bin--];
        s_key = (prefix << 8) | bin;
        s_above = sum;
      }
      __syncthreads();
      prefix = s_key;
      above = s_above;
    }
    cut = prefix;
    // how many of the entries equal to it, the lowest indices first
    const u64 each = f(of_key(cut));
    const u64 ties = each == 0 ? 1 : (want - above + each - 1) / each;
    const long long seg = ((V + WARPS - 1) / WARPS + 31) / 32 * 32;
    const long long i0 = warp * seg, i1 = min(V, i0 + seg);
    u64 n = 0;
    for (long long i = i0 + lane; i < i1; i += 32) {
      const uint32_t key = key_of(load<T>(z, i));
      n += key == cut && kept(key, i);
    }
    n = warp_sum(n);
    if (lane == 0) sums[warp] = n;
    if (tid == 0) s_index = old_cut == cut ? old_last : V;
    __syncthreads();
    u64 before = 0, all = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += sums[w];
      all += sums[w];
    }
    if (before < ties && before + n >= ties) {
      for (long long i = i0; i < i1; i += 32) {
        const uint32_t key = i + lane < i1 ? key_of(load<T>(z, i + lane)) : 0;
        const bool is = i + lane < i1 && key == cut && kept(key, i + lane);
        const unsigned mask = __ballot_sync(0xffffffffu, is);
        if (before + __popc(mask) >= ties) {
          if (is && before + __popc(mask & ((2u << lane) - 1)) == ties) s_index = i + lane;
          break;
        }
        before += __popc(mask);
      }
    }
    __syncthreads();
    last = s_index;
    __syncthreads();
    return above + min(ties, all) * each;
  };
  auto weight = [&](float x) { return row.weight(x); };
  u64 mass = 0;
  if (k_in > 0 && k_in < V) select([](float) { return u64{1}; }, static_cast<u64>(k_in));
  // ---- sum of what is kept
  auto kept = [&](float x, long long i) {
    const uint32_t key = key_of(x);
    return key > cut || (key == cut && i <= last);
  };
  const long long seg = ((V + WARPS - 1) / WARPS + 31) / 32 * 32;
  const long long i0 = warp * seg, i1 = min(V, i0 + seg);
  auto total_of = [&](u64& before, u64& mine) -> u64 {
    u64 sum = 0;
    for (long long i = i0 + lane; i < i1; i += 32) {
      const float x = load<T>(z, i);
      if (kept(x, i)) sum += weight(x);
    }
    mine = warp_sum(sum);
    __syncthreads();
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    u64 all = 0;
    before = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += sums[w];
      all += sums[w];
    }
    return all;
  };
  u64 before, mine;
  if (top_p < 1.f) {
    mass = total_of(before, mine);
    // the first entries whose weights sum to top_p of it
    bool rest;
    u64 want = share_of(fmaxf(top_p, 0.f), mass, rest);
    want += rest;
    want = want < 1 ? 1 : want;
    select(weight, want);
  }
  if (min_p > 0.f) {
    // w >= min_p: a bound on the logit, rounded up to the next one in f32
    const double bound = static_cast<double>(top) + row.t * log(static_cast<double>(fminf(min_p, 1.f)));
    const uint32_t key = key_of(__double2float_ru(bound));
    if (key > cut) cut = key, last = V;
  }
  mass = total_of(before, mine);
  // the first entry with a sum above u of all
  const float u = p.u[r];
  bool rest;
  const u64 want = u > 0.f ? (u < 1.f ? share_of(u, mass, rest) : mass - 1) : 0;
  if (before <= want && want < before + mine) {
    for (long long i = i0; i < i1; i += 32) {
      const float x = i + lane < i1 ? load<T>(z, i + lane) : -INFINITY;
      const u64 w = i + lane < i1 && kept(x, i + lane) ? weight(x) : 0;
      u64 upto = w;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > want);
      if (hit != 0) {
        if (lane == __ffs(hit) - 1) {
          p.token[r] = static_cast<int>(i + lane);
          if (p.logprob)
            p.logprob[r] = static_cast<float>((static_cast<double>(x) - static_cast<double>(top)) / row.t -
                                              log(static_cast<double>(mass) / row.scale));
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
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
  CDL_CUDA(launch_pdl(logits->dtype == CDL_BF16 ? sample::sample_kernel<__nv_bfloat16> : sample::sample_kernel<float>,
                      dim3(static_cast<unsigned>(R)), dim3(sample::THREADS), 0, stream, p));
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
