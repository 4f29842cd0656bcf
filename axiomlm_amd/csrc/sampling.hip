// Sampling of one token per row of logits: temperature, top-k, top-p, min-p, from given uniform numbers.
//
// Weights are integers, round(2^shift exp((z - max) / T)) with 2^shift V < 2^63: their sums are exact, so neither
// borders nor the choice depend on the order of threads.
#include "axm.h"
#include "axm_common.h"

namespace {

constexpr int kThreads = 1024;

struct SampleParams {
  const void* logits;
  int64_t ld;
  int V, shift;
  const float* u;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int64_t* tokens;
  float* probs;
};

template <int DT>
__device__ __forceinline__ float logit(const void* row, int i) {
  if (DT == 0) return h2f(((const f16*)row)[i]);
  if (DT == 1) return ((const float*)row)[i];
  return __builtin_bit_cast(float, (uint32_t)((const uint16_t*)row)[i] << 16);
}

// Order of logits: 0 for those never taken (-inf, NaN), else ascending with the value; -0 counts as 0.
__device__ __forceinline__ uint32_t logit_key(float z) {
  if (z != z || z == -INFINITY) return 0u;
  const uint32_t u = __builtin_bit_cast(uint32_t, z + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t s = 0;
  for (int w = 0; w < kThreads / 64; ++w) s += lds[w];
  return s;
}

// Integer weight of a key below or at the row's largest.
struct Weight {
  float top;
  double inv_t;
  int shift;
  __device__ __forceinline__ uint64_t operator()(uint32_t key) const {
    if (key == 0) return 0;
    const float z = key_logit(key);
    if (z == top) return 1ull << shift;
    return (uint64_t)__builtin_rint(ldexp(exp(((double)z - (double)top) * inv_t), shift));
  }
};

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleParams p) {
  __shared__ uint64_t red[kThreads / 64];
  __shared__ uint64_t scan[kThreads];
  const int r = blockIdx.x, V = p.V;
  const uint8_t* row = (const uint8_t*)p.logits + (int64_t)r * p.ld * (DT == 1 ? 4 : 2);
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  auto key_of = [&](int i) { return logit_key(logit<DT>(row, i)); };

  // Largest key, by bisection as the cuts below: f(t) = what lies at or over t.
  auto largest = [&](auto f, uint64_t want) {
    uint32_t cut = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = cut | (1u << bit);
      uint64_t s = 0;
      for (int i = threadIdx.x; i < V; i += kThreads) {
        const uint32_t k = key_of(i);
        if (k >= t) s += f(k);
      }
      if (block_sum(s, red) >= want) cut = t;
    }
    return cut;
  };
  auto count = [](uint32_t) { return (uint64_t)1; };
  const uint32_t top = largest(count, 1);
  if (top == 0) {
    if (threadIdx.x == 0) {
      p.tokens[r] = -1;
      if (p.probs) p.probs[r] = 0.f;
    }
    return;
  }
  const bool greedy = !(temperature > 0.f);
  // Kept: keys over `cut`, and the first `ties` keys equal to it.
  uint32_t cut = 1;
  uint64_t ties = V;
  const int k = greedy ? 1 : top_k;
  Weight weight{key_logit(top), greedy ? 1.0 : 1.0 / (double)temperature, p.shift};
  if (greedy || weight.top == INFINITY) cut = top;  // finite logits weigh nothing beside +inf
  auto over = [&](auto f) {  // what lies over the cut, and at it
    uint64_t a = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const uint32_t x = key_of(i);
      if (x > cut) a += f(x);
    }
    return block_sum(a, red);
  };
  if (k > 0 && k < V) {
    const uint32_t c = largest(count, k);
    if (c >= cut) {
      cut = c;
      ties = k - over(count);
    }
  }
  if (top_p < 1.f && !greedy) {
    uint64_t equal = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) equal += key_of(i) == cut;
    equal = block_sum(equal, red);
    if (equal < ties) ties = equal;
    const uint64_t total = over(weight) + ties * weight(cut);
    // Rank r stays iff the weight before it is under top_p total: the cut is the last key with less over it.
    const double need = (double)top_p * (double)total;
    uint32_t c = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = c | (1u << bit);
      uint64_t s = 0;
      for (int i = threadIdx.x; i < V; i += kThreads) {
        const uint32_t x = key_of(i);
        if (x >= t && x > cut) s += weight(x);
      }
      s = block_sum(s, red);
      if (t <= cut) s += ties * weight(cut);
      if ((double)s >= need) c = t;
    }
    if (c > top) c = top;
    if (c > cut) {
      cut = c;
      ties = V;
    } else if (c < cut) {
      c = cut;
    }
    const uint64_t before = over(weight), each = weight(cut);
    const double room = (need - (double)before) / (double)each;
    uint64_t most = room <= 1.0 ? 1 : (uint64_t)ceil(room);
    if (most < ties) ties = most;
  }
  // min-p by value.
  const double least = (double)min_p * ldexp(1.0, p.shift);
  auto kept_weight = [&](uint32_t x) {
    const uint64_t w = weight(x);
    return (double)w >= least || x == top ? w : 0;
  };
  // Total, then the running sum in index order.
  for (int pass = 0; pass < 2; ++pass) {
    __shared__ uint64_t total_s;
    uint64_t sum = 0, eq_sum = 0;
    const double target = pass ? (double)p.u[r] * (double)total_s : 0.0;
    int found = -1;
    uint64_t w_found = 0;
    for (int base = 0; base < V; base += kThreads) {
      const int i = base + threadIdx.x;
      const uint32_t x = i < V ? key_of(i) : 0u;
      const bool eq = x != 0 && x == cut;
      scan[threadIdx.x] = eq;
      __syncthreads();
      for (int o = 1; o < kThreads; o <<= 1) {
        const uint64_t add = (int)threadIdx.x >= o ? scan[threadIdx.x - o] : 0;
        __syncthreads();
        scan[threadIdx.x] += add;
        __syncthreads();
      }
      const bool keep = x > cut || (eq && eq_sum + scan[threadIdx.x] <= ties);
      eq_sum += scan[kThreads - 1];
      __syncthreads();
      const uint64_t w = keep ? kept_weight(x) : 0;
      scan[threadIdx.x] = w;
      __syncthreads();
      for (int o = 1; o < kThreads; o <<= 1) {
        const uint64_t add = (int)threadIdx.x >= o ? scan[threadIdx.x - o] : 0;
        __syncthreads();
        scan[threadIdx.x] += add;
        __syncthreads();
      }
      const uint64_t here = sum + scan[threadIdx.x];
      sum += scan[kThreads - 1];
      __syncthreads();
      if (pass && found < 0 && w > 0) {
        // The first whose running sum passes the target; the last kept one where rounding leaves none.
        const bool hit = (double)here > target || here == total_s;
        if (hit && !((double)(here - w) > target)) {
          found = i;
          w_found = w;
        }
      }
    }
    if (pass == 0) {
      if (threadIdx.x == 0) total_s = sum;
      __syncthreads();
    } else if (found >= 0) {
      p.tokens[r] = found;
      if (p.probs) p.probs[r] = (float)((double)w_found / (double)total_s);
    }
  }
}

}  // namespace

extern "C" int axm_sample_rows(const void* logits, int dtype, int64_t ld, int rows, int V, const float* u,
                               const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                               float temperature_all, int top_k_all, float top_p_all, float min_p_all, int64_t* tokens,
                               float* probs, void* stream) {
  AXM_CHECK_ARG(logits && u && tokens, -1, "sample_rows: null pointer");
  AXM_CHECK_ARG(dtype >= 0 && dtype <= 2, -1, "sample_rows: bad dtype %d", dtype);
  AXM_CHECK_ARG(rows >= 1 && rows < (1 << 22) && V >= 1 && V <= (1 << 24) && ld >= V, -1, "sample_rows: %d rows of %d logits, %lld apart",
                rows, V, (long long)ld);
  int shift = 46;  // V 2^shift <= 2^63: no sum passes 64 bits
  while ((uint64_t)V << shift > 1ull << 63) --shift;
  SampleParams p{logits, ld, V, shift, u, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all,
                 top_k_all, tokens, probs};
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == 0) hipLaunchKernelGGL((sample_kernel<0>), dim3(rows), dim3(kThreads), 0, s, p);
  else if (dtype == 1) hipLaunchKernelGGL((sample_kernel<1>), dim3(rows), dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((sample_kernel<2>), dim3(rows), dim3(kThreads), 0, s, p);
  AXM_LAUNCH_CHECK("sample_rows");
  return 0;
}
