// Sampling of one token per row of logits: temperature, top-k, top-p, min-p, from given uniform numbers.
//
// One workgroup per row, which it passes over two to four times (later passes come from L2).  The order of tokens is
// (logit descending, index ascending); what top-k and top-p keep is everything up to a cut (z, i) in that order.
// A cut is found from a histogram over (max - z) in steps of 1/64: counts for top-k, weights for top-p; only the bin
// that holds the cut is put in order.  Where top-k leaves no more candidates than the list in LDS holds (the usual
// settings), they are collected in one pass and everything else happens on the list.
//
// Weights are integers, 2^shift exp((z - max) / T) with 2^shift V <= 2^63: their sums are exact, so neither the cuts nor
// the choice depend on the order of threads.
#include "axm.h"
#include "axm_common.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr float kBinsPerUnit = 64.f;
constexpr int kList = 2048;  // candidates in LDS
constexpr int kSums = 3072;  // entries of the running sum

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

// Order of logits as integers (finite values and +inf; -0 counts as 0).
__device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t u = __builtin_bit_cast(uint32_t, z + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o, 64);
  return v;
}

struct Lds {
  double table[256];  // 2^(shift - j / 256)
  union {
    struct {
      uint64_t weight[kBins];
      uint32_t count[kBins];
    } bins;
    uint64_t sums[kSums];
  };
  float z[kList];
  int at[kList];
  float sorted_z[kList];
  int sorted_at[kList];
  uint64_t red[kWaves];
  uint64_t total, before;
  float fred[kWaves], cut_z;
  int ired[kWaves], cut_i, n, bin, where;
};

// Sum over the workgroup, the same in every thread.
__device__ __forceinline__ uint64_t block_sum(uint64_t v, Lds& s) {
  v = wave_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) t += s.red[w];
  return t;
}

// Sum over the threads before this one; *total over all.
__device__ __forceinline__ uint64_t block_before(uint64_t v, Lds& s, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t y = __shfl_up((unsigned long long)x, o, 64);
    x += lane >= o ? y : 0;
  }
  __syncthreads();
  if (lane == 63) s.red[wave] = x;
  __syncthreads();
  uint64_t b = 0, t = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    b += w < wave ? s.red[w] : 0;
    t += s.red[w];
  }
  *total = t;
  return b + x - v;
}

template <int DT>
struct Row {
  static constexpr int E = DT == 1 ? 4 : 8;  // logits of a 16-byte load
  const u32x4* base;                         // the row's first logit is number `lead` from here
  int lead, V, vectors, tile0, tile1;        // tiles (64 loads) of this wave: a contiguous run
  bool inf;                                  // +inf among them: those count 0, all others -inf

  // Loads stay inside the 16-byte blocks that hold the row's first and last logits.
  __device__ __forceinline__ u32x4 load(int tile) const {
    const int v = tile * 64 + (int)(threadIdx.x & 63);
    return base[min(v, vectors - 1)];
  }
  __device__ __forceinline__ int index(int tile, int j) const {
    return (tile * 64 + (int)(threadIdx.x & 63)) * E + j - lead;
  }
  __device__ __forceinline__ void values(int tile, const u32x4& r, float (&z)[E]) const {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (DT == 1) {
        const uint32_t w = r[j];
        z[j] = __builtin_bit_cast(float, w);
      } else {
        const uint32_t w = r[j >> 1];
        z[j] = DT == 0 ? h2f(u16_as_h((uint16_t)(j & 1 ? w >> 16 : w & 0xFFFFu)))
                       : __builtin_bit_cast(float, j & 1 ? w & 0xFFFF0000u : w << 16);
      }
    }
    if (tile == 0 || (tile + 1) * 64 * E - lead > V) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if ((unsigned)index(tile, j) >= (unsigned)V) z[j] = -INFINITY;
    }
    if (inf) {
#pragma unroll
      for (int j = 0; j < E; ++j) z[j] = z[j] == INFINITY ? 0.f : -INFINITY;
    }
  }
  // f(tile, z) for every tile of this wave, four loads on their way.
  template <typename F>
  __device__ __forceinline__ void pass(const F& f) const {
#pragma unroll 1
    for (int t = tile0; t < tile1; t += 4) {
      u32x4 r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) r[k] = load(min(t + k, tile1 - 1));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (t + k < tile1) {
          float z[E];
          values(t + k, r[k], z);
          f(t + k, z);
        }
      }
    }
  }
};

__device__ __forceinline__ int bin_of(float top, float z) {  // -inf and NaN: the last
  return (int)fminf((top - z) * kBinsPerUnit, (float)(kBins - 1));
}

// 2^shift 2^(-(top - z) rate) as an integer: the table's 2^(shift - j / 256), times a polynomial of the rest (under
// 2^-8 octaves: four terms reach 2^-49), rounded by adding 2^52.
struct Weight {
  double top, rate;  // rate: 256 log2(e) / T
  const double* table;
  __device__ __forceinline__ uint64_t operator()(float z) const {
    const double y = fmin((top - (double)z) * rate, 256.0 * 64.0);
    const int i = (int)y;
    const double r = y - (double)i;
    constexpr double a = 0.0027076061740622863;  // ln 2 / 256
    const double q = fma(fma(fma(fma(r, a * a * a * a / 24, -a * a * a / 6), r, a * a / 2), r, -a), r, 1.0);
    const double w = ldexp(table[i & 255] * q, -(i >> 8));
    return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) - 0x4330000000000000ull;
  }
};

// The first logit, in index order, at which the running sum of f passes `target` (by the order of sums as doubles where
// target is no integer), or the last one with a weight.  -> its index in s.where, its f in s.before; s.total the sum.
// f(z, i) >= 0; frac: target is that share of the total.
template <int DT, typename F>
__device__ __forceinline__ void find_in_order(const Row<DT>& row, Lds& s, const F& f, double frac, double target) {
  constexpr int E = Row<DT>::E;
  const int lane = threadIdx.x & 63;
  const int tiles = (row.vectors + 63) / 64, group = (tiles + kSums - 1) / kSums;
  __syncthreads();
  for (int i = threadIdx.x; i < kSums; i += kThreads) s.sums[i] = 0;
  __syncthreads();
  row.pass([&](int tile, const float (&z)[E]) {
    uint64_t w = 0;
#pragma unroll
    for (int j = 0; j < E; ++j) w += f(z[j], row.index(tile, j));
    if (__builtin_amdgcn_ballot_w64(w != 0)) {
      w = wave_sum64(w);
      if (lane == 0) atomicAdd((unsigned long long*)&s.sums[tile / group], (unsigned long long)w);
    }
  });
  __syncthreads();
  constexpr int kEach = kSums / kThreads;
  uint64_t e[kEach], mine = 0, total;
#pragma unroll
  for (int i = 0; i < kEach; ++i) mine += e[i] = s.sums[threadIdx.x * kEach + i];
  uint64_t run = block_before(mine, s, &total);
  if (frac >= 0.0) target = frac * (double)total;
  // Sums as doubles never fall, so one entry passes the target; or none does, and the last with a weight counts.
  auto passes = [&](uint64_t sum) { return (double)sum > target || sum == total; };
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (e[i] != 0 && passes(run + e[i]) && !((double)run > target) && run != total) {
      s.n = threadIdx.x * kEach + i;
      s.before = run;
    }
    run += e[i];
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    run = s.before;
    const int first = s.n * group;
    bool found = false;
    for (int tile = first; tile < min(first + group, tiles) && !found; ++tile) {
      float z[E];
      row.values(tile, row.load(tile), z);
      uint64_t w[E], sum = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) sum += w[j] = f(z[j], row.index(tile, j));
      uint64_t x = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = __shfl_up((unsigned long long)x, o, 64);
        x += lane >= o ? y : 0;
      }
      const uint64_t after = run + __shfl((unsigned long long)x, 63, 64);
      uint64_t here = run + x - sum;
      bool hit = false;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if (w[j] != 0 && passes(here + w[j]) && !((double)here > target) && here != total) {
          hit = true;
          s.where = row.index(tile, j);
          s.total = total;
          s.before = w[j];
        }
        here += w[j];
      }
      found = __builtin_amdgcn_ballot_w64(hit) != 0;
      run = after;
    }
  }
  __syncthreads();
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleParams p) {
  constexpr int E = Row<DT>::E, kSize = DT == 1 ? 4 : 2;
  __shared__ Lds s;
  const int r = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uintptr_t first = (uintptr_t)p.logits + (uintptr_t)((int64_t)r * p.ld * kSize);
  Row<DT> row;
  row.base = (const u32x4*)(first & ~(uintptr_t)15);
  row.lead = (int)(first & 15) / kSize;
  row.V = p.V;
  row.vectors = (row.lead + p.V + E - 1) / E;
  const int tiles = (row.vectors + 63) / 64;
  row.tile0 = (int)((int64_t)tiles * wave / kWaves);
  row.tile1 = (int)((int64_t)tiles * (wave + 1) / kWaves);
  row.inf = false;
  const float temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  const int top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  const double u = fmin(fmax((double)p.u[r], 0.0), 1.0);  // (NaN: 0)

  auto answer = [&](int token, float prob) {
    p.tokens[r] = token;
    if (p.probs) p.probs[r] = prob;
  };

  // ---- the largest logit, lowest index ----
  float top = -INFINITY;
  int top_at = -1;
  row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (z[j] > top) {
        top = z[j];
        top_at = row.index(tile, j);
      }
  });
  auto better = [](float z, int i, float z2, int i2) { return z2 > z || (z2 == z && (unsigned)i2 < (unsigned)i); };
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float z2 = __shfl_xor(top, o, 64);
    const int i2 = __shfl_xor(top_at, o, 64);
    if (better(top, top_at, z2, i2)) {
      top = z2;
      top_at = i2;
    }
  }
  if (lane == 0) {
    s.fred[wave] = top;
    s.ired[wave] = top_at;
  }
  if (threadIdx.x < 256) s.table[threadIdx.x] = exp2((double)p.shift - threadIdx.x * (1.0 / 256));
  __syncthreads();
  for (int w = 0; w < kWaves; ++w)
    if (better(top, top_at, s.fred[w], s.ired[w])) {
      top = s.fred[w];
      top_at = s.ired[w];
    }
  if (top_at < 0 || !(temperature > 0.f)) {  // nothing to take; greedy
    if (threadIdx.x == 0) answer(top_at, top_at < 0 ? 0.f : 1.f);
    return;
  }
  if (top == INFINITY) {
    row.inf = true;
    top = 0.f;
  }
  const Weight weight{(double)top, 256.0 * 1.4426950408889634 / (double)temperature, s.table};
  const uint64_t largest = 1ull << p.shift;
  const double least = (double)min_p * (double)largest;
  auto stays = [&](uint64_t w) { return (double)w >= least || w == largest; };  // min-p
  float cut_z = -INFINITY;  // kept: z > cut_z, or z == cut_z and i <= cut_i
  int cut_i = -1;
  auto kept = [&](float z, int i) { return z > cut_z || (z == cut_z && i <= cut_i); };

  // The cut inside bin `bin`, whose kept logits are too many for the list: by value first, then by index among equal ones.
  // measure(z): what a logit adds; everything before the bin adds `before`; the cut is the logit that reaches `need`.
  auto bisect = [&](int bin, uint64_t before, double need, auto measure) {
    uint32_t lo = ~0u, hi = 0;
    row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (kept(z[j], row.index(tile, j)) && bin_of(top, z[j]) == bin) {
          lo = min(lo, order_key(z[j]));
          hi = max(hi, order_key(z[j]));
        }
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      lo = min(lo, (uint32_t)__shfl_xor((int)lo, o, 64));
      hi = max(hi, (uint32_t)__shfl_xor((int)hi, o, 64));
    }
    __syncthreads();
    if (lane == 0) {
      s.ired[wave] = (int)lo;
      s.fred[wave] = __builtin_bit_cast(float, hi);
    }
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) {
      lo = min(lo, (uint32_t)s.ired[w]);
      hi = max(hi, __builtin_bit_cast(uint32_t, s.fred[w]));
    }
    auto from = [&](uint32_t key) {  // measured in the bin at or over key
      uint64_t a = 0;
      row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (kept(z[j], row.index(tile, j)) && bin_of(top, z[j]) == bin && order_key(z[j]) >= key) a += measure(z[j]);
      });
      return before + block_sum(a, s);
    };
    while (lo < hi) {  // the largest key that reaches `need`
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if ((double)from(mid) >= need) lo = mid;
      else hi = mid - 1;
    }
    const float z_cut = key_value(lo);
    const double over = (double)from(lo + 1), each = (double)measure(z_cut);
    const double rank = fmax(ceil((need - over) / each), 1.0);  // of those equal to it
    find_in_order<DT>(row, s, [&](float z, int i) { return (uint64_t)(z == z_cut && kept(z, i)); }, -1.0, rank - 1.0);
    cut_z = z_cut;
    cut_i = s.where;
  };

  // ---- top-k ----
  const int k = top_k > 0 && top_k < p.V ? top_k : 0;
  if (k > 0) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins.count[i] = 0;
    if (threadIdx.x == 0) s.n = 0, s.bin = -1;
    __syncthreads();
    row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (z[j] > -INFINITY) atomicAdd(&s.bins.count[bin_of(top, z[j])], 1u);
    });
    __syncthreads();
    uint64_t all;
    const uint32_t c0 = s.bins.count[2 * threadIdx.x], c1 = s.bins.count[2 * threadIdx.x + 1];
    const uint64_t before = block_before(c0 + c1, s, &all);
    if (before < (uint64_t)k && before + c0 + c1 >= (uint64_t)k) {
      const bool second = before + c0 < (uint64_t)k;
      s.bin = 2 * threadIdx.x + second;
      s.before = before + (second ? c0 : 0);
    }
    __syncthreads();
    if (s.bin >= 0 || all <= kList) {  // (with no more candidates than k, all of them are kept)
      const int bin = s.bin >= 0 ? s.bin : kBins - 1;
      const uint64_t ahead = s.bin >= 0 ? s.before : all, upto = s.bin >= 0 ? ahead + s.bins.count[bin] : all;
      const bool whole = upto <= (uint64_t)kList;  // the list takes all candidates, not just the bin with the cut
      const int least_bin = whole ? 0 : bin;
      const uint64_t listed = whole ? upto : upto - ahead;
      if (listed <= (uint64_t)kList) {
        row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
          for (int j = 0; j < E; ++j) {
            const int b = bin_of(top, z[j]);
            if (z[j] > -INFINITY && b >= least_bin && b <= bin) {
              const int at = atomicAdd(&s.n, 1);
              s.z[at] = z[j];
              s.at[at] = row.index(tile, j);
            }
          }
        });
        __syncthreads();
        const int n = s.n;
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const float z = s.z[i];
          const int at = s.at[i];
          int rank = 0;
          for (int j = 0; j < n; ++j) rank += s.z[j] > z || (s.z[j] == z && s.at[j] < at);
          s.sorted_z[rank] = z;
          s.sorted_at[rank] = at;
        }
        __syncthreads();
        if (!whole) {
          cut_z = s.sorted_z[k - 1 - (int)ahead];
          cut_i = s.sorted_at[k - 1 - (int)ahead];
        } else {
          // All that is left happens on the list: ranks below `last` stay.
          const int m = min(n, k);
          uint64_t w[2] = {0, 0}, sum;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (2 * (int)threadIdx.x + e < m) w[e] = weight(s.sorted_z[2 * threadIdx.x + e]);
          const uint64_t ahead_w = block_before(w[0] + w[1], s, &sum);
          const double need = top_p < 1.f ? (double)top_p * (double)sum : INFINITY;
          uint64_t mine = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i = 2 * threadIdx.x + e;
            const uint64_t b = ahead_w + (e ? w[0] : 0);
            const bool in = i < m && (i == 0 || (double)b < need) && stays(w[e]);
            mine += in ? 1 : 0;
          }
          const int last = (int)block_sum(mine, s);  // weights fall with the rank, so the kept ranks are the first ones
          uint64_t kept_w = 0;
#pragma unroll
          for (int e = 0; e < 2; ++e) kept_w += 2 * (int)threadIdx.x + e < last ? w[e] : 0;
          const uint64_t total = block_sum(kept_w, s);
          uint64_t* ws = s.sums;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (2 * (int)threadIdx.x + e < last) ws[2 * threadIdx.x + e] = w[e];
          __syncthreads();
          const double target = u * (double)total;
          for (int i = threadIdx.x; i < last; i += kThreads) {
            const uint64_t mine_w = ws[i];
            const int at = s.sorted_at[i];
            uint64_t upto_w = 0;
            for (int j = 0; j < last; ++j) upto_w += s.sorted_at[j] <= at ? ws[j] : 0;
            const bool hit = (double)upto_w > target || upto_w == total;
            if (mine_w != 0 && hit && !((double)(upto_w - mine_w) > target) && upto_w - mine_w != total)
              answer(at, (float)((double)mine_w / (double)total));
          }
          return;
        }
      } else {
        bisect(bin, ahead, (double)k, [](float) { return (uint64_t)1; });
      }
    }
    __syncthreads();
  }

  // ---- top-p ----
  if (top_p < 1.f) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins.weight[i] = 0;
    if (threadIdx.x == 0) s.n = 0, s.bin = 0, s.before = 0;
    __syncthreads();
    row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (kept(z[j], row.index(tile, j)))
          atomicAdd((unsigned long long*)&s.bins.weight[bin_of(top, z[j])], (unsigned long long)weight(z[j]));
    });
    __syncthreads();
    uint64_t all;
    const uint64_t c0 = s.bins.weight[2 * threadIdx.x], c1 = s.bins.weight[2 * threadIdx.x + 1];
    const uint64_t before = block_before(c0 + c1, s, &all);
    const double need = (double)top_p * (double)all;
    // The first bin whose sum reaches `need` (bin 0 where need is 0).
    if ((double)before < need && (double)(before + c0 + c1) >= need) {
      const bool second = (double)(before + c0) < need;
      s.bin = 2 * threadIdx.x + second;
      s.before = before + (second ? c0 : 0);
    }
    __syncthreads();
    const int bin = s.bin;
    const uint64_t ahead = s.before;
    row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (kept(z[j], row.index(tile, j)) && bin_of(top, z[j]) == bin) {
          const int at = atomicAdd(&s.n, 1);
          if (at < kList) {
            s.z[at] = z[j];
            s.at[at] = row.index(tile, j);
          }
        }
    });
    __syncthreads();
    const int n = s.n;
    if (n <= kList) {
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const float z = s.z[i];
        const int at = s.at[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += s.z[j] > z || (s.z[j] == z && s.at[j] < at);
        s.sorted_z[rank] = z;
        s.sorted_at[rank] = at;
      }
      __syncthreads();
      uint64_t w[2] = {0, 0}, sum, mine = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (2 * (int)threadIdx.x + e < n) w[e] = weight(s.sorted_z[2 * threadIdx.x + e]);
      const uint64_t b = ahead + block_before(w[0] + w[1], s, &sum);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * threadIdx.x + e;
        mine += i < n && (i == 0 || (double)(b + (e ? w[0] : 0)) < need) ? 1 : 0;
      }
      const int last = (int)block_sum(mine, s) - 1;  // sums never fall, so the kept ranks are the first ones
      cut_z = s.sorted_z[last];
      cut_i = s.sorted_at[last];
    } else {
      bisect(bin, ahead, need, weight);
    }
  }

  // ---- the token ----
  find_in_order<DT>(row, s, [&](float z, int i) -> uint64_t {
    if (!kept(z, i)) return 0;
    const uint64_t w = weight(z);
    return stays(w) ? w : 0;
  }, u, 0.0);
  if (threadIdx.x == 0) answer(s.where, (float)((double)s.before / (double)s.total));
}

}  // namespace

extern "C" int axm_sample_rows(const void* logits, int dtype, int64_t ld, int rows, int V, const float* u,
                               const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                               float temperature_all, int top_k_all, float top_p_all, float min_p_all, int64_t* tokens,
                               float* probs, void* stream) {
  AXM_CHECK_ARG(logits && u && tokens, -1, "sample_rows: null pointer");
  AXM_CHECK_ARG(dtype >= 0 && dtype <= 2, -1, "sample_rows: bad dtype %d", dtype);
  AXM_CHECK_ARG((uintptr_t)logits % (dtype == 1 ? 4 : 2) == 0, -1, "sample_rows: logits off their type's alignment");
  AXM_CHECK_ARG(rows >= 1 && rows < (1 << 22) && V >= 1 && V <= (1 << 24) && ld >= V, -1,
                "sample_rows: %d rows of %d logits, %lld apart", rows, V, (long long)ld);
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
