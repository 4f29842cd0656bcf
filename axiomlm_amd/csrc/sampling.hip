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
constexpr int kCounted = 256;  // candidates that are put in order by counting
constexpr int kAhead = 2;    // loads of a wave under way
constexpr int kSums = 2048;  // entries of the running sum
constexpr int kTable = 512;  // entries of the table of 2^(j / kTable)

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
  bool order;  // rows with top-p and no top-k first
  // Few rows: `slices` workgroups share a row without top-k (SplitRow); 0: none do.
  int slices;
  struct SliceTop* tops;  // [rows][slices]
  uint64_t* hists;        // [rows][slices][kBins]
  uint64_t* sums;         // [rows][kSums]
  uint64_t* lists;        // [rows][slices][kList]
  struct SplitRow* split; // [rows]
};

struct SliceTop {
  float top;
  int octave;  // the slice's weights are 2^shift 2^(z log2(e) / T - octave)
  int listed;  // candidates of the bin with the cut (second launch)
};
struct SplitRow {  // what the second launch found
  double need;
  uint64_t ahead;
  int bin;
};

// Order of logits as integers (finite values and +inf; -0 counts as 0).
__device__ __forceinline__ uint32_t order_key(float z) {
  const uint32_t u = __builtin_bit_cast(uint32_t, z + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// One candidate as an integer: larger is earlier in the order.
__device__ __forceinline__ uint64_t candidate(float z, int i) { return (uint64_t)order_key(z) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float candidate_z(uint64_t c) { return key_value((uint32_t)(c >> 32)); }
__device__ __forceinline__ int candidate_at(uint64_t c) { return (int)~(uint32_t)c; }

// Inclusive sums over the wave's lanes, on DPP moves: shifts inside rows of 16, then the rows' last lanes onward.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_add64(uint64_t x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, true);
  return x + ((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ uint64_t wave_prefix64(uint64_t x) {
  x = dpp_add64<0x111, 0xF>(x);  // row_shr:1
  x = dpp_add64<0x112, 0xF>(x);
  x = dpp_add64<0x114, 0xF>(x);
  x = dpp_add64<0x118, 0xF>(x);
  x = dpp_add64<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
  return dpp_add64<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
}
__device__ __forceinline__ uint64_t lane63(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, 63);
}

struct Lds {
  double table[kTable];  // of 2^(shift + j / kTable)
  union {
    struct {
      uint64_t weight[kBins];
      uint32_t count[kBins];
    } bins;
    uint64_t sums[kSums];
  };
  uint64_t list[kList];
  uint64_t red[2][kWaves];
  uint64_t total, before;
  int n, bin, where;
  int place[kCounted];
};

// Sum over the workgroup, the same in every thread.  turn: 0 and 1 in turn, so that one barrier is enough.
__device__ __forceinline__ uint64_t block_sum(uint64_t v, Lds& s, int& turn) {
  const uint64_t x = wave_prefix64(v);
  uint64_t* red = s.red[turn ^= 1];
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = x;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) t += red[w];
  return t;
}

// Sum over the threads before this one; *total over all.
__device__ __forceinline__ uint64_t block_before(uint64_t v, Lds& s, int& turn, uint64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t x = wave_prefix64(v);
  uint64_t* red = s.red[turn ^= 1];
  if (lane == 63) red[wave] = x;
  __syncthreads();
  uint64_t b = 0, t = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    b += w < wave ? red[w] : 0;
    t += red[w];
  }
  *total = t;
  return b + x - v;
}

// Largest over the workgroup.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_max64(uint64_t x) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, true);
  const uint64_t y = (uint64_t)hi << 32 | lo;
  return y > x ? y : x;
}
__device__ __forceinline__ uint64_t block_max(uint64_t v, Lds& s, int& turn) {
  v = dpp_max64<0x111, 0xF>(v);
  v = dpp_max64<0x112, 0xF>(v);
  v = dpp_max64<0x114, 0xF>(v);
  v = dpp_max64<0x118, 0xF>(v);
  v = dpp_max64<0x142, 0xA>(v);
  v = dpp_max64<0x143, 0xC>(v);
  uint64_t* red = s.red[turn ^= 1];
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v = red[w] > v ? red[w] : v;
  return v;
}

// s.list[0, n) into descending order (n <= kList); all threads, and a barrier at the end.
__device__ __forceinline__ void sort_list(Lds& s, int n) {
  __syncthreads();
  int size = 64;
  while (size < n) size *= 2;
  if (size <= kCounted) {  // places by counting: each candidate against size^2 / kThreads others in every part of the threads
    const int i = threadIdx.x & (size - 1), each = size * size / kThreads, j0 = threadIdx.x / size * each;
    if ((int)threadIdx.x < size) s.place[i] = 0;
    const uint64_t mine = i < n ? s.list[i] : 0;
    int over = 0;
#pragma unroll 4
    for (int j = j0; j < min(j0 + each, n); ++j) over += s.list[j] > mine;
    __syncthreads();
    if (over) atomicAdd(&s.place[i], over);
    __syncthreads();
    if ((int)threadIdx.x < n) s.list[s.place[i]] = mine;
    __syncthreads();
    return;
  }
  for (int i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = 0;  // less than every candidate
  __syncthreads();
  for (int k = 2; k <= size; k *= 2)  // bitonic
    for (int j = k / 2; j > 0; j /= 2) {
      const int t = threadIdx.x;
      if (t < size / 2) {
        const int a = (t & ~(j - 1)) * 2 + (t & (j - 1)), b = a + j;
        const uint64_t x = s.list[a], y = s.list[b];
        if ((x < y) == ((a & k) == 0)) {
          s.list[a] = y;
          s.list[b] = x;
        }
      }
      __syncthreads();
    }
}

template <int DT>
struct Row {
  static constexpr int E = DT == 1 ? 4 : 8;  // logits of a 16-byte load
  const u32x4* base;                         // the row's first logit is number `lead` from here
  int lead, V, vectors, tile0, tile1;        // tiles (64 loads) of this wave: a contiguous run
  bool inf;                                  // +inf among them: those count 0, all others -inf
  u32x4 first[kAhead];                       // the wave's first tiles stay in registers

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
  // f(tile, z) for every tile of this wave, the next kAhead on their way.
  template <typename F>
  __device__ __forceinline__ void pass(const F& f) const {
    u32x4 r[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) r[k] = first[k];
#pragma unroll 1
    for (int t = tile0; t < tile1; t += kAhead) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (t + k < tile1) {
          float z[E];
          values(t + k, r[k], z);
          if (t + k + kAhead < tile1) r[k] = load(t + k + kAhead);
          f(t + k, z);
        }
      }
    }
  }
};

constexpr double kRate = kTable * 1.4426950408889634;
// Tiles of an entry of the running sum.
__device__ __forceinline__ int tile_group(int vectors) { return ((vectors + 63) / 64 + kSums - 1) / kSums; }
__device__ __forceinline__ int bin_of(float top, float z) {  // -inf and NaN: the last
  return (int)fminf((top - z) * kBinsPerUnit, (float)(kBins - 1));
}

// 2^shift 2^((z - top) rate / kTable) as an integer: the table's 2^(shift + j / kTable), with the whole octaves in its
// exponent, times a polynomial of the rest, at most 2^-10 octaves either way (three terms: 2^-46 of the weight), rounded
// by adding 2^52.  z - top and what follows in 64 bits: differences of fp32 logits do not fit 32.  128 octaves down and
// beyond weigh 0.
struct Weight {
  double top, rate, off;  // rate: kTable log2(e) / T; off: added in kTable-ths of an octave
  const double* table;
  __device__ __forceinline__ uint64_t operator()(float z) const {
    const double y = fmax(fma((double)z - top, rate, off), -128.0 * kTable);
    const double near = y + 6755399441055744.0;  // 1.5 2^52: the nearest integer in the low bits
    const int i = (int)(uint32_t)__builtin_bit_cast(uint64_t, near);
    const double r = y - (near - 6755399441055744.0);
    constexpr double a = 0.6931471805599453 / kTable;
    const double q = fma(fma(fma(r, a * a * a / 6, a * a / 2), r, a), r, 1.0);
    const uint64_t octaves = (uint64_t)((uint32_t)(i & -kTable) * ((1u << 20) / kTable)) << 32;
    const double t = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, table[i & (kTable - 1)]) + octaves);
    return __builtin_bit_cast(uint64_t, fma(q, t, 4503599627370496.0)) - 0x4330000000000000ull;
  }
};
__device__ __forceinline__ void fill_table(Lds& s, int shift) {
  for (int j = threadIdx.x; j < kTable; j += kThreads) s.table[j] = ldexp(exp2((double)j / kTable), shift);
}

// Weights of a lane's logits, all of them before any is used: eight chains of 64-bit operations side by side.  Left to
// itself the compiler moves each into the branch that uses it, one after the other.
template <int E>
__device__ __forceinline__ void weights_of(const Weight& weight, const float (&z)[E], uint64_t (&w)[E]) {
#pragma unroll
  for (int j = 0; j < E; ++j) w[j] = weight(z[j]);
#pragma unroll
  for (int j = 0; j < E; ++j) asm volatile("" : "+v"(w[j]));
}

// Sums of the weights of every `group` tiles, in s.sums; f(tile, z, add) calls add(j, weight) for the tile's logits that
// have one.
template <int DT, typename F>
__device__ __forceinline__ void sum_tiles(const Row<DT>& row, Lds& s, int group, const F& f) {
  constexpr int E = Row<DT>::E;
  __syncthreads();
  for (int i = threadIdx.x; i < kSums; i += kThreads) s.sums[i] = 0;
  __syncthreads();
  row.pass([&](int tile, const float (&z)[E]) {
    uint64_t w = 0;
    f(tile, z, [&](int, uint64_t x) { w += x; });
    if (__builtin_amdgcn_ballot_w64(w != 0)) {
      w = wave_prefix64(w);
      if ((threadIdx.x & 63) == 63) atomicAdd((unsigned long long*)&s.sums[tile / group], (unsigned long long)w);
    }
  });
  __syncthreads();
}

// This lane's share of a tile's weights where few logits are kept: the wave queues those in LDS (where s.list was) and
// weighs them side by side, not every logit that is next to one (us, all weighed / queued: 48.7 / 46.7 for 64 rows of
// 128000 with top-p).  keep(j): whether z[j] is; of(z): its weight.
typedef float __attribute__((may_alias)) lds_float;
template <int E, typename K, typename W>
__device__ __forceinline__ uint64_t kept_sum(const Weight& weight, const float (&z)[E], Lds& s, const K& keep, const W& of) {
  constexpr int kRoom = kList * 2 / kWaves;  // logits of a wave's queue
  lds_float* queue = reinterpret_cast<lds_float*>(s.list) + (threadIdx.x >> 6) * kRoom;
  const int lane = threadIdx.x & 63;
  uint64_t mask[E], sum = 0;
  int n = 0;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    mask[j] = __builtin_amdgcn_ballot_w64(keep(j));
    n += __builtin_popcountll(mask[j]);
  }
  if (n > kRoom) {
    uint64_t w[E];
    weights_of(weight, z, w);
#pragma unroll
    for (int j = 0; j < E; ++j) sum += keep(j) ? of(w[j]) : 0;
    return sum;
  }
  int at = 0;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    if (mask[j] >> lane & 1)
      queue[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask[j], 0u))] =
          z[j];
    at += __builtin_popcountll(mask[j]);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (int i = lane; i < n; i += 64) sum += of(weight(queue[i]));
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  return sum;
}

// The first logit, in index order, at which the running sum of weights (s.sums, and f within a group) passes `target`
// (sums compared as doubles), or the last one with a weight.  -> its index in s.where, its weight in s.before, all
// weights' sum in s.total.  frac >= 0: target is that share of the sum.
template <int DT, typename F>
__device__ __forceinline__ void pick_in_order(const Row<DT>& row, Lds& s, int& turn, int group, const F& f, double frac,
                                              double target) {
  constexpr int E = Row<DT>::E;
  const int tiles = (row.vectors + 63) / 64;
  constexpr int kEach = kSums / kThreads;
  uint64_t e[kEach], mine = 0, total;
#pragma unroll
  for (int i = 0; i < kEach; ++i) mine += e[i] = s.sums[threadIdx.x * kEach + i];
  uint64_t run = block_before(mine, s, turn, &total);
  if (frac >= 0.0) target = frac * (double)total;
  // Sums as doubles never fall, so one entry passes the target; or none does, and the last with a weight counts.
  auto passes = [&](uint64_t before, uint64_t w) {
    return w != 0 && ((double)(before + w) > target || before + w == total) && !((double)before > target);
  };
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (passes(run, e[i])) {
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
      for (int j = 0; j < E; ++j) w[j] = 0;
      f(tile, z, [&](int j, uint64_t x) { sum += w[j] = x; });
      const uint64_t x = wave_prefix64(sum);
      uint64_t here = run + x - sum;
      run += lane63(x);
      bool hit = false;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if (passes(here, w[j])) {
          hit = true;
          s.where = row.index(tile, j);
          s.total = total;
          s.before = w[j];
        }
        here += w[j];
      }
      found = __builtin_amdgcn_ballot_w64(hit) != 0;
    }
  }
  __syncthreads();
}

template <int DT, typename F>
__device__ __forceinline__ void find_in_order(const Row<DT>& row, Lds& s, int& turn, const F& f, double frac,
                                              double target) {
  const int group = tile_group(row.vectors);
  sum_tiles<DT>(row, s, group, f);
  pick_in_order<DT>(row, s, turn, group, f, frac, target);
}

struct Settings {
  float temperature, top_p, min_p;
  int k;  // 0: off
  bool greedy;
};
__device__ __forceinline__ Settings settings_of(const SampleParams& p, int r) {
  Settings t;
  t.temperature = p.temperature ? p.temperature[r] : p.temperature_all;
  const int k = p.top_k ? p.top_k[r] : p.top_k_all;
  t.k = k > 0 && k < p.V ? k : 0;
  t.top_p = p.top_p ? p.top_p[r] : p.top_p_all;
  t.min_p = p.min_p ? p.min_p[r] : p.min_p_all;
  t.greedy = !(t.temperature > 0.f);
  return t;
}

// The row of this workgroup where those with top-p and no top-k, which take longest, start first: where more rows than
// fit the chip at once have settings of their own, some of them would run alone at the end.  us, as they come / slow ones
// first: 500 rows of 50304 in fp32 95.5 / 86.3, 300 in fp16 57.7 / 50.7, 1000 rows of 128000 247 / 205; but 1000 of 32000
// 98 / 102 and 400 of 20000 47 / 50 (finding the row takes 2 us of each), so large vocabularies only.
__device__ __forceinline__ int row_in_order(const SampleParams& p, Lds& s, int& turn) {
  const int rows = gridDim.x, mine = threadIdx.x, wanted = blockIdx.x;
  const Settings t = settings_of(p, min(mine, rows - 1));
  const bool slow = mine < rows && !t.greedy && t.k == 0 && t.top_p < 1.f;
  uint64_t total;
  const int before = (int)block_before(slow, s, turn, &total);
  if (mine < rows && (slow ? before : (int)total + mine - before) == wanted) s.where = mine;
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(s.where);
}

// Row r, with the tiles [tile0, tile1) of a workgroup dealt to its waves in contiguous runs.
template <int DT>
__device__ __forceinline__ Row<DT> row_of(const SampleParams& p, int r) {
  constexpr int E = Row<DT>::E, kSize = DT == 1 ? 4 : 2;
  const uintptr_t first = (uintptr_t)p.logits + (uintptr_t)((int64_t)r * p.ld * kSize);
  Row<DT> row;
  row.base = (const u32x4*)(first & ~(uintptr_t)15);
  row.lead = (int)(first & 15) / kSize;
  row.V = p.V;
  row.vectors = (row.lead + p.V + E - 1) / E;
  row.inf = false;
  return row;
}
template <int DT>
__device__ __forceinline__ void deal_tiles(Row<DT>& row, int tile0, int tile1) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  row.tile0 = tile0 + (int)((int64_t)(tile1 - tile0) * wave / kWaves);
  row.tile1 = tile0 + (int)((int64_t)(tile1 - tile0) * (wave + 1) / kWaves);
  if (row.tile0 < row.tile1) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) row.first[k] = row.load(min(row.tile0 + k, row.tile1 - 1));
  }
}
// Slice `slice` of a row: whole groups of tiles.
template <int DT>
__device__ __forceinline__ void deal_slice(Row<DT>& row, int slice, int slices) {
  const int group = tile_group(row.vectors), tiles = (row.vectors + 63) / 64, groups = (tiles + group - 1) / group;
  deal_tiles<DT>(row, min((int)((int64_t)groups * slice / slices) * group, tiles),
                 min((int)((int64_t)groups * (slice + 1) / slices) * group, tiles));
}

// ---------------------------------------------------------------------------
// Few rows of large vocabularies, without top-k: `slices` workgroups a row.  First launch: every slice's largest logit
// and its histogram of weights, over bins of a grid that all slices share (64 z to the nearest integer) and relative to
// an octave of its own; second: every slice adds the histograms up (shifted by whole bins and octaves), finds the bin
// with the cut, sums its tiles' weights before that bin and lists the bin's candidates; third: one workgroup a row cuts
// the list, adds what stays to the sums and picks the token.  Rows whose largest logit is infinite or passes 2^16 or 2^20
// octaves, and those that list too many, are left to the third launch, which then does everything.  64 rows of 128000
// with top-p: 16, 17 and 11 us; the histogram's pass takes 8, with its additions or without.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t grid_of(float z) {  // 1.5 2^23: the nearest integer in the low bits
  return __builtin_bit_cast(uint32_t, fmaf(z, kBinsPerUnit, 12582912.f));
}
__device__ __forceinline__ int grid_bin(uint32_t top_grid, float z) {  // -inf and NaN: far past the last
  return (int)min(top_grid - grid_of(z), (uint32_t)(kBins - 1));
}
// Weights of a split row: relative to whole octaves.
__device__ __forceinline__ Weight octave_weight(float temperature, int octave, const double* table) {
  return Weight{0.0, kRate / (double)temperature, -(double)kTable * (double)octave, table};
}
// The row's largest logit and octave from its slices'; false: not to be split.
__device__ __forceinline__ bool split_top(const SampleParams& p, int r, float* top, int* octave) {
  const SliceTop x = p.tops[(int64_t)r * p.slices + min((int)threadIdx.x & 15, p.slices - 1)];  // (16 slices or fewer)
  float t = x.top;
  int o = x.octave;
#pragma unroll
  for (int d = 1; d < 16; d *= 2) {
    t = fmaxf(t, __shfl_xor(t, d));
    o = max(o, __shfl_xor(o, d));
  }
  *top = t;
  *octave = o;
  return fabsf(t) < 65536.f && abs(o) < (1 << 20);  // (larger logits have coarser bins)
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_slice_kernel(SampleParams p) {
  constexpr int E = Row<DT>::E;
  __shared__ Lds s;
  const int r = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
  const Settings t = settings_of(p, r);
  if (t.greedy || t.k > 0) return;
  Row<DT> row = row_of<DT>(p, r);
  deal_slice<DT>(row, slice, p.slices);
  int turn = 0;
  fill_table(s, p.shift);
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins.weight[i] = 0;
  float top = -INFINITY;
  row.pass([&](int, const float (&z)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j) top = fmaxf(top, z[j]);
  });
  const uint32_t best = (uint32_t)block_max(top > -INFINITY ? order_key(top) : 0, s, turn);
  top = best ? key_value(best) : -INFINITY;
  const double octave = ceil((double)top * (kRate / kTable) / (double)t.temperature);
  const bool fine = best && fabs(octave) < (double)(1 << 20);
  if (threadIdx.x == 0)
    p.tops[blockIdx.x] = SliceTop{top, fine ? (int)octave : !best || octave < 0.0 ? -(1 << 30) : 1 << 30, 0};
  if (!fine || !(t.top_p < 1.f)) return;
  const Weight weight = octave_weight(t.temperature, (int)octave, s.table);
  const uint32_t top_grid = grid_of(top);
  row.pass([&](int, const float (&z)[E]) {
    uint64_t w[E];
    weights_of(weight, z, w);
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (z[j] > -INFINITY)
        atomicAdd((unsigned long long*)&s.bins.weight[grid_bin(top_grid, z[j])], (unsigned long long)w[j]);
  });
  __syncthreads();
  uint64_t* to = p.hists + (int64_t)blockIdx.x * kBins;
  for (int i = threadIdx.x; i < kBins; i += kThreads) to[i] = s.bins.weight[i];
}

// min-p of a split row: the least weight that stays.
__device__ __forceinline__ uint64_t least_of(float min_p, uint64_t largest) {
  return (uint64_t)fmin(fmax(ceil((double)min_p * (double)largest), 0.0), (double)largest);
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_sums_kernel(SampleParams p) {
  constexpr int E = Row<DT>::E;
  __shared__ Lds s;
  const int r = blockIdx.x / p.slices, slice = blockIdx.x % p.slices;
  const Settings t = settings_of(p, r);
  if (t.greedy || t.k > 0) return;
  float top;
  int octave, turn = 0;
  if (!split_top(p, r, &top, &octave)) return;
  Row<DT> row = row_of<DT>(p, r);
  deal_slice<DT>(row, slice, p.slices);
  fill_table(s, p.shift);
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins.weight[i] = 0;
  if (threadIdx.x == 0) s.n = 0, s.bin = 0, s.before = 0;
  __syncthreads();
  const uint32_t top_grid = grid_of(top);
  int bin = kBins;  // the bin with the cut; past the last: no top-p
  if (t.top_p < 1.f) {
    constexpr int kTogether = 4;  // slices whose histograms are asked for together
    for (int i0 = 0; i0 < p.slices; i0 += kTogether) {
      uint64_t w[kTogether][kBins / kThreads];
      SliceTop x[kTogether];
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const int64_t n = (int64_t)r * p.slices + min(i0 + i, p.slices - 1);
        x[i] = p.tops[n];
#pragma unroll
        for (int e = 0; e < kBins / kThreads; ++e) w[i][e] = p.hists[n * kBins + e * kThreads + threadIdx.x];
      }
#pragma unroll
      for (int i = 0; i < kTogether; ++i) {
        const int down = octave - x[i].octave;
        if (i0 + i >= p.slices || x[i].top == -INFINITY || down > 63) continue;  // (the first: it has no histogram)
        const int by = (int)min(top_grid - grid_of(x[i].top), (uint32_t)kBins);
#pragma unroll
        for (int e = 0; e < kBins / kThreads; ++e)
          if (w[i][e] >> down != 0)
            atomicAdd((unsigned long long*)&s.bins.weight[min(e * kThreads + (int)threadIdx.x + by, kBins - 1)],
                      (unsigned long long)(w[i][e] >> down));
      }
    }
    __syncthreads();
    uint64_t all;
    const uint64_t c0 = s.bins.weight[2 * threadIdx.x], c1 = s.bins.weight[2 * threadIdx.x + 1];
    const uint64_t before = block_before(c0 + c1, s, turn, &all);
    const double need = (double)t.top_p * (double)all;
    if ((double)before < need && (double)(before + c0 + c1) >= need) {
      const bool second = (double)(before + c0) < need;
      s.bin = 2 * threadIdx.x + second;
      s.before = before + (second ? c0 : 0);
    }
    __syncthreads();
    bin = s.bin;
    if (slice == 0 && threadIdx.x == 0) p.split[r] = SplitRow{need, s.before, bin};
  }
  const Weight weight = octave_weight(t.temperature, octave, s.table);
  const uint64_t least = least_of(t.min_p, weight(top));
  uint64_t* list = p.lists + (int64_t)blockIdx.x * kList;
  const int group = tile_group(row.vectors);
  sum_tiles<DT>(row, s, group, [&](int tile, const float (&z)[E], auto add) {
    int b[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      b[j] = z[j] > -INFINITY ? grid_bin(top_grid, z[j]) : kBins + 1;
      if (b[j] == bin) {
        const int at = atomicAdd(&s.n, 1);
        if (at < kList) list[at] = candidate(z[j], row.index(tile, j));
      }
    }
    add(0, kept_sum(weight, z, s, [&](int j) { return b[j] < bin; }, [&](uint64_t w) { return w >= least ? w : 0; }));
  });
  if (threadIdx.x == 0) p.tops[blockIdx.x].listed = s.n;
  const int tiles = (row.vectors + 63) / 64, groups = (tiles + group - 1) / group;
  const int g0 = (int)((int64_t)groups * slice / p.slices), g1 = (int)((int64_t)groups * (slice + 1) / p.slices);
  for (int i = g0 + threadIdx.x; i < g1; i += kThreads) p.sums[(int64_t)r * kSums + i] = s.sums[i];
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleParams p) {
  constexpr int E = Row<DT>::E;
  __shared__ Lds s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int turn = 0;
  const int r = p.order ? row_in_order(p, s, turn) : blockIdx.x;
  Row<DT> row = row_of<DT>(p, r);
  const Settings settings = settings_of(p, r);
  const float temperature = settings.temperature, top_p = settings.top_p, min_p = settings.min_p;
  const bool greedy = settings.greedy;
  const int k = settings.k;
  const double u = fmin(fmax((double)p.u[r], 0.0), 1.0);  // (NaN: 0)

  auto answer = [&](int token, float prob) {
    p.tokens[r] = token;
    if (p.probs) p.probs[r] = prob;
  };
  float split_z;
  int octave;
  if (p.slices > 0 && !greedy && k == 0 && split_top(p, r, &split_z, &octave)) {
    // The slices have summed what lies before the bin with the cut and listed the bin.
    int n = (threadIdx.x & 63) < p.slices ? p.tops[(int64_t)r * p.slices + (threadIdx.x & 63)].listed : 0;
#pragma unroll
    for (int d = 1; d < 16; d *= 2) n += __shfl_xor(n, d);
    n = __builtin_amdgcn_readfirstlane(n);
    if (n <= kList) {
      fill_table(s, p.shift);
      const int group = tile_group(row.vectors), groups = ((row.vectors + 63) / 64 + group - 1) / group;
      for (int i = threadIdx.x; i < kSums; i += kThreads) s.sums[i] = i < groups ? p.sums[(int64_t)r * kSums + i] : 0;
      for (int i = 0, at = 0; i < p.slices; ++i) {
        const int m = p.tops[(int64_t)r * p.slices + i].listed;
        const uint64_t* from = p.lists + ((int64_t)r * p.slices + i) * kList;
        for (int j = threadIdx.x; j < m; j += kThreads) s.list[at + j] = from[j];
        at += m;
      }
      sort_list(s, n);
      const Weight weight = octave_weight(temperature, octave, s.table);
      const uint64_t least = least_of(min_p, weight(split_z));
      float cut_z = -INFINITY;
      int cut_i = -1;
      if (top_p < 1.f) {
        const SplitRow x = p.split[r];
        uint64_t c[2] = {0, 0}, w[2] = {0, 0}, sum, mine = 0;
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (2 * (int)threadIdx.x + e < n) {
            c[e] = s.list[2 * threadIdx.x + e];
            w[e] = weight(candidate_z(c[e]));
          }
        const uint64_t b = x.ahead + block_before(w[0] + w[1], s, turn, &sum);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int i = 2 * threadIdx.x + e;
          const bool in = i < n && (i == 0 || (double)(b + (e ? w[0] : 0)) < x.need);
          mine += in ? 1 : 0;
          if (in && w[e] >= least) {
            const int tile = (candidate_at(c[e]) + row.lead) / (64 * E);
            atomicAdd((unsigned long long*)&s.sums[tile / group], (unsigned long long)w[e]);
          }
        }
        const uint64_t last = s.list[max((int)block_sum(mine, s, turn), 1) - 1];
        cut_z = candidate_z(last);
        cut_i = candidate_at(last);
      }
      __syncthreads();
      pick_in_order<DT>(row, s, turn, group, [&](int tile, const float (&z)[E], auto add) {
        uint64_t w[E];
        weights_of(weight, z, w);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const bool in = (z[j] > cut_z) | ((z[j] == cut_z) & (j <= cut_i - row.index(tile, 0)));
          add(j, in & (w[j] >= least) ? w[j] : 0);
        }
      }, u, 0.0);
      if (threadIdx.x == 0) answer(s.where, (float)((double)s.before / (double)s.total));
      return;
    }
  }
  deal_tiles<DT>(row, 0, (row.vectors + 63) / 64);
  if (!greedy) {
    fill_table(s, p.shift);
    if (k > 0)
      for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins.count[i] = 0;
    if (threadIdx.x == 0) s.n = 0, s.bin = -1;
  }

  // ---- the largest logit, lowest index ----
  float top = -INFINITY;
  int top_at = -1;
  row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const bool more = z[j] > top;
      top = more ? z[j] : top;
      top_at = more ? row.index(tile, j) : top_at;
    }
  });
  const uint64_t best = block_max(top_at < 0 ? 0 : candidate(top, top_at), s, turn);
  const float own = top;
  top = candidate_z(best);
  if (best == 0 || greedy) {  // nothing to take; the largest
    if (threadIdx.x == 0) answer(best == 0 ? -1 : candidate_at(best), best == 0 ? 0.f : 1.f);
    return;
  }
  if (top == INFINITY) {
    row.inf = true;
    top = 0.f;
  }
  const Weight weight{(double)top, kRate / (double)temperature, 0.0, s.table};
  const uint64_t largest = 1ull << p.shift;
  // min-p: weights from `least` on stay (the largest always).
  const uint64_t least = least_of(min_p, largest);
  auto stays = [&](uint64_t w) { return w >= least; };
  // Kept: z > cut_z, or z == cut_z and i <= cut_i; without a cut, what is over -inf.
  float cut_z = -INFINITY;
  int cut_i = -1;
  auto kept = [&](float z, int tile, int j) {
    return (z > cut_z) | ((z == cut_z) & (j <= cut_i - row.index(tile, 0)));
  };

  // The cut inside bin `bin`, whose kept logits are too many for the list: by value first, then by index among equal ones.
  // measure(z): what a logit adds; everything before the bin adds `before`; the cut is the logit that reaches `need`.
  auto bisect = [&](int bin, uint64_t before, double need, auto measure) {
    uint64_t ends = 0;  // largest of the order and of its complement
    uint32_t lo = 0, hi = 0;
    row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (kept(z[j], tile, j) && bin_of(top, z[j]) == bin) {
          lo = max(lo, ~order_key(z[j]));
          hi = max(hi, order_key(z[j]));
        }
    });
    ends = block_max(lo, s, turn);
    lo = ~(uint32_t)ends;
    hi = (uint32_t)block_max(hi, s, turn);
    auto from = [&](uint32_t key) {  // measured in the bin at or over key
      uint64_t a = 0;
      row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (kept(z[j], tile, j) && bin_of(top, z[j]) == bin && order_key(z[j]) >= key) a += measure(z[j]);
      });
      return before + block_sum(a, s, turn);
    };
    while (lo < hi) {  // the largest key that reaches `need`
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      if ((double)from(mid) >= need) lo = mid;
      else hi = mid - 1;
    }
    const float z_cut = key_value(lo);
    const double over = (double)from(lo + 1), each = (double)measure(z_cut);
    const double rank = fmax(ceil((need - over) / each), 1.0);  // of those equal to it
    find_in_order<DT>(row, s, turn, [&](int tile, const float (&z)[E], auto add) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (z[j] == z_cut && kept(z[j], tile, j)) add(j, 1);
    }, -1.0, rank - 1.0);
    cut_z = z_cut;
    cut_i = s.where;
  };

  // ---- top-k ----
  if (k > 0) {
    const float own_top = top_at < 0 ? -INFINITY : row.inf ? (own == INFINITY ? 0.f : -INFINITY) : own;
    // The k-th largest of the threads' own largest logits bounds the cut from below: where few pass it, they are all
    // candidates and no histogram of the row is needed.
    bool listed = false;
    uint64_t all = 0;
    if (k <= kThreads / 4) {
      if (own_top > -INFINITY) atomicAdd(&s.bins.count[bin_of(top, own_top)], 1u);
      __syncthreads();
      const uint32_t c0 = s.bins.count[2 * threadIdx.x], c1 = s.bins.count[2 * threadIdx.x + 1];
      const uint64_t before = block_before(c0 + c1, s, turn, &all);
      if (before < (uint64_t)k && before + c0 + c1 >= (uint64_t)k) s.bin = 2 * threadIdx.x + (before + c0 < (uint64_t)k);
      s.bins.count[2 * threadIdx.x] = s.bins.count[2 * threadIdx.x + 1] = 0;
      __syncthreads();
      const float reach = s.bin >= 0 && s.bin < kBins - 1 ? (float)(s.bin + 1) : 0.f;  // (the last bin has no end)
      if (reach > 0.f) {
        row.pass([&](int tile, const float (&z)[E]) {
          float most = z[0];
#pragma unroll
          for (int j = 1; j < E; ++j) most = fmaxf(most, z[j]);
          if ((top - most) * kBinsPerUnit < reach) {
#pragma unroll
            for (int j = 0; j < E; ++j)
              if ((top - z[j]) * kBinsPerUnit < reach) {
                const int at = atomicAdd(&s.n, 1);
                if (at < kList) s.list[at] = candidate(z[j], row.index(tile, j));
              }
          }
        });
        __syncthreads();
        listed = s.n <= kList;
        __syncthreads();
      }
      if (!listed && threadIdx.x == 0) s.n = 0, s.bin = -1;
      __syncthreads();
    }
    if (!listed) {
      row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (z[j] > -INFINITY) atomicAdd(&s.bins.count[bin_of(top, z[j])], 1u);
      });
      __syncthreads();
      const uint32_t c0 = s.bins.count[2 * threadIdx.x], c1 = s.bins.count[2 * threadIdx.x + 1];
      const uint64_t before = block_before(c0 + c1, s, turn, &all);
      if (before < (uint64_t)k && before + c0 + c1 >= (uint64_t)k) {
        const bool second = before + c0 < (uint64_t)k;
        s.bin = 2 * threadIdx.x + second;
        s.before = before + (second ? c0 : 0);
      }
      __syncthreads();
    }
    if (listed || s.bin >= 0 || all <= kList) {  // (with no more candidates than k, all of them are kept)
      const int bin = s.bin >= 0 ? s.bin : kBins - 1;
      const uint64_t ahead = s.bin >= 0 ? s.before : all, upto = s.bin >= 0 ? ahead + s.bins.count[bin] : all;
      const bool whole = listed || upto <= (uint64_t)kList;  // the list takes all candidates, not just the bin with the cut
      if (whole || upto - ahead <= (uint64_t)kList) {
        if (!listed) {
          const int least_bin = whole ? 0 : bin;
          row.pass([&](int tile, const float (&z)[E]) {
#pragma unroll
            for (int j = 0; j < E; ++j) {
              const int b = bin_of(top, z[j]);
              if (b <= bin && b >= least_bin && z[j] > -INFINITY)
                s.list[atomicAdd(&s.n, 1)] = candidate(z[j], row.index(tile, j));
            }
          });
          __syncthreads();
        }
        const int n = s.n;
        sort_list(s, n);
        if (!whole) {
          const uint64_t c = s.list[k - 1 - (int)ahead];
          cut_z = candidate_z(c);
          cut_i = candidate_at(c);
        } else {
          // All that is left happens on the list, two neighbouring ranks a thread.
          const int m = min(n, k);
          uint64_t c[2] = {0, 0}, w[2] = {0, 0}, sum;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (2 * (int)threadIdx.x + e < m) {
              c[e] = s.list[2 * threadIdx.x + e];
              w[e] = weight(candidate_z(c[e]));
            }
          const uint64_t ahead_w = block_before(w[0] + w[1], s, turn, &sum);
          const double need = top_p < 1.f ? (double)top_p * (double)sum : INFINITY;
          // Sums rise and weights fall with the rank, so the kept ranks are the first ones; the others weigh 0.
          const int i0 = 2 * (int)threadIdx.x;
          const bool in0 = i0 < m && (i0 == 0 || (double)ahead_w < need) && stays(w[0]);
          const bool in1 = i0 + 1 < m && (double)(ahead_w + w[0]) < need && stays(w[1]);
          w[0] = in0 ? w[0] : 0;
          w[1] = in1 ? w[1] : 0;
          const uint64_t total = block_sum(w[0] + w[1], s, turn);
          const double target = u * (double)total;
          if (m <= 64) {  // the same comparisons of places again, of indices: s.sums are the weights before each
            if (threadIdx.x < 64) s.sums[threadIdx.x] = 0;
            if (threadIdx.x < 32) {  // (the pairs of ranks as they lie in registers)
              s.sums[64 + 2 * threadIdx.x] = w[0];
              s.sums[65 + 2 * threadIdx.x] = w[1];
            }
            __syncthreads();
            const int j0 = wave * 4;
            const int at = lane < m ? candidate_at(s.list[lane]) : 0;
            uint64_t part = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              part += j0 + j < m && candidate_at(s.list[j0 + j]) < at ? s.sums[64 + j0 + j] : 0;
            if (lane < m && part != 0) atomicAdd((unsigned long long*)&s.sums[lane], (unsigned long long)part);
            __syncthreads();
            if (wave == 0 && lane < m) {
              const uint64_t b = s.sums[lane], x = s.sums[64 + lane];
              if (x != 0 && ((double)(b + x) > target || b + x == total) && !((double)b > target))
                answer(at, (float)((double)x / (double)total));
            }
            return;
          }
          // Running sums in index order, by 1024 stretches of the vocabulary, then inside the one that passes the target.
          const int each = (p.V + kThreads - 1) / kThreads;
          s.sums[threadIdx.x] = 0;
          if (threadIdx.x == 0) s.n = 0;
          __syncthreads();
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (w[e] != 0) atomicAdd((unsigned long long*)&s.sums[candidate_at(c[e]) / each], (unsigned long long)w[e]);
          __syncthreads();
          uint64_t total2;
          const uint64_t mine = s.sums[threadIdx.x], run = block_before(mine, s, turn, &total2);
          auto passes = [&](uint64_t b, uint64_t x) {
            return x != 0 && ((double)(b + x) > target || b + x == total) && !((double)b > target);
          };
          if (passes(run, mine)) {
            s.where = threadIdx.x;
            s.before = run;
          }
          __syncthreads();
          // (index, weight) of the stretch's candidates; the list itself is in registers.
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (w[e] != 0 && candidate_at(c[e]) / each == s.where) {
              const int at = atomicAdd(&s.n, 1);
              s.list[at] = (uint64_t)candidate_at(c[e]);
              s.sums[at] = w[e];
            }
          __syncthreads();
          const int inside = s.n;
          for (int i = threadIdx.x; i < inside; i += kThreads) {
            uint64_t b = s.before;
            for (int j = 0; j < inside; ++j) b += s.list[j] < s.list[i] ? s.sums[j] : 0;
            if (passes(b, s.sums[i])) answer((int)s.list[i], (float)((double)s.sums[i] / (double)total));
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
      uint64_t w[E];
      weights_of(weight, z, w);
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (kept(z[j], tile, j))
          atomicAdd((unsigned long long*)&s.bins.weight[bin_of(top, z[j])], (unsigned long long)w[j]);
    });
    __syncthreads();
    uint64_t all;
    const uint64_t c0 = s.bins.weight[2 * threadIdx.x], c1 = s.bins.weight[2 * threadIdx.x + 1];
    const uint64_t before = block_before(c0 + c1, s, turn, &all);
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
        if (bin_of(top, z[j]) == bin && kept(z[j], tile, j)) {
          const int at = atomicAdd(&s.n, 1);
          if (at < kList) s.list[at] = candidate(z[j], row.index(tile, j));
        }
    });
    __syncthreads();
    const int n = s.n;
    if (n <= kList) {
      sort_list(s, n);
      uint64_t w[2] = {0, 0}, sum, mine = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (2 * (int)threadIdx.x + e < n) w[e] = weight(candidate_z(s.list[2 * threadIdx.x + e]));
      const uint64_t b = ahead + block_before(w[0] + w[1], s, turn, &sum);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = 2 * threadIdx.x + e;
        mine += i < n && (i == 0 || (double)(b + (e ? w[0] : 0)) < need) ? 1 : 0;
      }
      const uint64_t c = s.list[(int)block_sum(mine, s, turn) - 1];  // sums never fall: the kept ranks are the first ones
      cut_z = candidate_z(c);
      cut_i = candidate_at(c);
    } else {
      bisect(bin, ahead, need, weight);
    }
  }

  // ---- the token ----
  const int group = tile_group(row.vectors);
  auto stayed = [&](uint64_t w) { return stays(w) ? w : 0; };
  auto weights = [&](int tile, const float (&z)[E], auto add) {
    uint64_t w[E];
    weights_of(weight, z, w);
#pragma unroll
    for (int j = 0; j < E; ++j) add(j, kept(z[j], tile, j) ? stayed(w[j]) : 0);
  };
  if (cut_z > -INFINITY)
    sum_tiles<DT>(row, s, group, [&](int tile, const float (&z)[E], auto add) {
      add(0, kept_sum(weight, z, s, [&](int j) { return kept(z[j], tile, j); }, stayed));
    });
  else
    sum_tiles<DT>(row, s, group, weights);
  pick_in_order<DT>(row, s, turn, group, weights, u, 0.0);
  if (threadIdx.x == 0) answer(s.where, (float)((double)s.before / (double)s.total));
}

}  // namespace

namespace {

// Workgroups that share a row, 8192 logits or more each: none where rows or vocabulary are too small for the three
// launches to pay, or where top-k leaves rows a list that one workgroup is as fast with.  us, one workgroup a row / split:
// with top-p 64 rows of 128000 93 / 44 (four slices), 100 of 50000 47 / 42 (two), 20 of 40000 36 / 32 (four), but 8 of
// 30000 30 / 31 (three); without one row of 100000 42 / 21 (twelve), 60 of 50000 23 / 22 and in fp32 28 / 23 (four), but
// 20 of 40000 19 / 21 (four) and 100 of 50000 23 / 26 (two); 60 of 20000 with top-k in most 26 / 45 (two).
int slices_of(int rows, int V, bool top_k, bool top_p) {
  const int by_rows = axm_num_cus() / rows, by_size = V / 8192, n = by_rows < by_size ? by_rows : by_size;
  if (top_k || by_size < (top_p ? 4 : 5) || n < (top_p ? 2 : 4)) return 0;
  return n < 16 ? n : 16;
}
struct SampleWorkspace {
  size_t split, tops, sums, hists, lists, bytes;
};
SampleWorkspace sample_workspace(int rows, int slices) {
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  SampleWorkspace w{};
  if (slices == 0) return w;
  const size_t n = (size_t)rows * slices;
  w.tops = w.split + up(rows * sizeof(SplitRow));
  w.sums = w.tops + up(n * sizeof(SliceTop));
  w.hists = w.sums + up((size_t)rows * kSums * 8);
  w.lists = w.hists + up(n * kBins * 8);
  w.bytes = w.lists + up(n * kList * 8);
  return w;
}

template <int DT>
void launch_sample(const SampleParams& p, int rows, hipStream_t s) {
  if (p.slices > 0) {
    hipLaunchKernelGGL((sample_slice_kernel<DT>), dim3(rows * p.slices), dim3(kThreads), 0, s, p);
    hipLaunchKernelGGL((sample_sums_kernel<DT>), dim3(rows * p.slices), dim3(kThreads), 0, s, p);
  }
  hipLaunchKernelGGL((sample_kernel<DT>), dim3(rows), dim3(kThreads), 0, s, p);
}

}  // namespace

extern "C" size_t axm_sample_rows_workspace_bytes(int rows, int V, int with_top_k, int with_top_p) {
  if (rows < 1 || V < 1) return 0;
  return sample_workspace(rows, slices_of(rows, V, with_top_k != 0, with_top_p != 0)).bytes;
}

extern "C" int axm_sample_rows(const void* logits, int dtype, int64_t ld, int rows, int V, const float* u,
                               const float* temperature, const int* top_k, const float* top_p, const float* min_p,
                               float temperature_all, int top_k_all, float top_p_all, float min_p_all, int64_t* tokens,
                               float* probs, void* workspace, size_t workspace_bytes, void* stream) {
  AXM_CHECK_ARG(logits && u && tokens, -1, "sample_rows: null pointer");
  AXM_CHECK_ARG(dtype >= 0 && dtype <= 2, -1, "sample_rows: bad dtype %d", dtype);
  AXM_CHECK_ARG((uintptr_t)logits % (dtype == 1 ? 4 : 2) == 0, -1, "sample_rows: logits off their type's alignment");
  AXM_CHECK_ARG(rows >= 1 && rows < (1 << 22) && V >= 1 && V <= (1 << 24) && ld >= V, -1,
                "sample_rows: %d rows of %d logits, %lld apart", rows, V, (long long)ld);
  const int slices = slices_of(rows, V, top_k || (top_k_all > 0 && top_k_all < V), top_p || top_p_all < 1.f);
  const SampleWorkspace w = sample_workspace(rows, slices);
  AXM_CHECK_ARG(workspace_bytes >= w.bytes && (w.bytes == 0 || (workspace && (uintptr_t)workspace % 16 == 0)), -1,
                "sample_rows: workspace of %zu bytes needed (16-byte aligned), %zu given", w.bytes, workspace_bytes);
  int shift = 46;  // V 2^shift <= 2^63: no sum passes 64 bits
  while ((uint64_t)V << shift > 1ull << 63) --shift;
  uint8_t* ws = (uint8_t*)workspace;
  SampleParams p{logits, ld, V, shift, u, temperature, top_k, top_p, min_p, temperature_all, top_p_all, min_p_all,
                 top_k_all, tokens, probs,
                 V >= 40960 && rows > axm_num_cus() && rows <= kThreads && (temperature || top_k || top_p),
                 slices, nullptr, nullptr, nullptr, nullptr, nullptr};
  if (slices > 0) {
    p.split = (SplitRow*)(ws + w.split);
    p.tops = (SliceTop*)(ws + w.tops);
    p.sums = (uint64_t*)(ws + w.sums);
    p.hists = (uint64_t*)(ws + w.hists);
    p.lists = (uint64_t*)(ws + w.lists);
  }
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == 0) launch_sample<0>(p, rows, s);
  else if (dtype == 1) launch_sample<1>(p, rows, s);
  else launch_sample<2>(p, rows, s);
  AXM_LAUNCH_CHECK("sample_rows");
  return 0;
}
