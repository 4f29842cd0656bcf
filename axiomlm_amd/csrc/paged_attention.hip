// Decode attention of one new token per sequence over a paged KV cache.
//
//   out[b][hq] = sum_s p_s v_s,  p = softmax(q k_s / sqrt(hd)) over s < seq_lens[b]
//
// Every cached row is read once and serves all query heads of its KV head: their rows (up to 16 a pass) are one tile of
// v_mfma_f32_16x16x32_f16.  The work is the list of 128-key units of all (sequence, KV head) pairs, and every
// workgroup takes an equal run of it, whatever the lengths are: a run holds parts of at most two pairs beside whole ones.
// A pair that one workgroup has whole is stored as fp16; parts leave fp32 (max, sum, sum of p v), joined by a second
// launch, which also turns stored scores into the account of weights.
#include <type_traits>

#include "kv_device.h"
#include "paged_kv.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kBlock = 32;             // keys of a wave's step: the k extent of one P V instruction
constexpr int kUnit = kWaves * kBlock; // keys of a work unit: one step of every wave
constexpr int kRows = 16;              // query rows of a tile
// Weights are held as 2^kShift exp2(s - m): with the running maximum allowed to lag by kSlack, they stay below 2^15 and
// keep fp16's full precision down to 2^-21 of the largest.
constexpr float kSlack = 8.f;
constexpr float kShift = 7.f;

struct DecodeParams {
  PagedKv kv;
  const f16* q;
  int64_t ld_q;
  const int* lens;
  f16* out;
  float* parts;    // [workgroup][2][16 rows][2 + hd]: a run's first and last pair, where it has only part of them
  int* info;       // [pairs][2]: first and last workgroup of a pair
  f32x2* ml;       // [n_seqs][Hq]: (max, sum) of pairs that one workgroup has whole (account only)
  float* scores;   // [n_seqs][Hq][score_len], log2 units (account only)
  int64_t score_len;
  float* mass;
  int64_t mass_len;
  int Hq, n_rep, chunks;  // chunks: tiles of 16 query rows per KV head
  int grid;
  int max_len;
  float scale_log2;
};

typedef float __attribute__((may_alias)) lds_float;  // results in the memory of value tiles
typedef const __attribute__((address_space(4))) int* const_ints;  // read through the scalar cache
__device__ __forceinline__ const_ints as_const(const int* p) { return (const_ints)(uintptr_t)p; }

__device__ __forceinline__ int len_of(const DecodeParams& p, int b) {
  return min(max(as_const(p.lens)[b], 0), p.max_len);
}

// Workgroup w's run of U units: U / grid of them, one more in the first U % grid.
__device__ __forceinline__ uint32_t run_begin(uint32_t U, uint32_t grid, uint32_t w) {
  return U / grid * w + min(w, U % grid);
}
__device__ __forceinline__ uint32_t run_of(uint32_t U, uint32_t grid, uint32_t u) {
  const uint32_t each = U / grid, more = U % grid, head = more * (each + 1);
  return u < head ? u / (each + 1) : more + (u - head) / max(each, 1u);
}

// Bytes of a cached row that one lane loads at a time, and the loads of its share (a quarter: 4 lanes hold a key row).
template <int KVT, int HD>
struct RowShape {
  static constexpr int kBytes = KVT == AXM_KV_FP16 ? 2 * HD : KVT == AXM_KV_FP8 ? HD : HD / 2;
  static constexpr int kLoad = kBytes >= 64 ? 16 : 8;
  static constexpr int kLoads = kBytes / (4 * kLoad);
  static constexpr int kChunks = kLoad * 8 / (KVT == AXM_KV_FP16 ? 16 : KVT == AXM_KV_FP8 ? 8 : 4) / 8;  // of 8 elements
  static constexpr int kScale = HD / 64 * 2;
  // First element of chunk c of load j for lane quarter lq.
  static __device__ __forceinline__ int dim(int j, int c, int lq) { return ((j * 4 + lq) * kChunks + c) * 8; }
};

// One step's rows as loaded: keys 16 h + l16, quarter lq.
template <int KVT, int HD>
struct Step {
  u32x4 k[2][RowShape<KVT, HD>::kLoads], v[2][RowShape<KVT, HD>::kLoads];
  uint32_t ks[2], vs[2];
  int valid[2];  // keys of each half that count
};

template <int KVT, int HD>
__device__ __forceinline__ f16x8 step_chunk(const u32x4& r, uint32_t sc, int j, int c, int lq) {
  KvRaw8 f;
  f.r = r;
  if (KVT == AXM_KV_FP8) f.r = u32x4{r[2 * c], r[2 * c + 1], 0u, 0u};
  if (KVT == AXM_KV_INT4) f.r = u32x4{r[c], 0u, 0u, 0u};
  f.sc = sc;
  if (HD == 128 && KVT == AXM_KV_FP8) f.sc = j == 0 ? sc & 0xFFFFu : sc >> 16;
  if (HD == 128 && KVT == AXM_KV_INT4) f.sc = lq < 2 ? sc & 0xFFFFu : sc >> 16;
  return kv_half8<KVT>(f);
}

template <int KVT, int HD, bool MASS>
__global__ void __launch_bounds__(kThreads, 2) paged_decode_kernel(DecodeParams p) {
  using S = RowShape<KVT, HD>;
  constexpr int KS = HD / 32, DT = HD / 16;
  constexpr int VROW = HD + 16;
  constexpr int kMergeRow = 2 + HD;
  static_assert(kRows * kMergeRow * 4 <= kBlock * VROW * 2, "a wave's result fits its value tile");
  __shared__ __align__(16) f16 vt[kWaves][kBlock * VROW];
  __shared__ __align__(16) f16 pt[kWaves][2][kRows * kBlock];
  const PagedKv& kv = p.kv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int B = kv.n_seqs, pairs = kv.Hkv * p.chunks;

  // ---- this workgroup's run of units ----
  auto units = [&](int b) { return b < B ? (min(max(p.lens[b], 0), p.max_len) + kUnit - 1) / kUnit : 0; };
  auto prefix = [&](int x) {  // inclusive sums over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      x += lane >= o ? y : 0;
    }
    return x;
  };
  int total = 0, mine = units(lane), sums = prefix(mine);
  total = __builtin_amdgcn_readlane(sums, 63);
  for (int b0 = 64; b0 < B; b0 += 64) total += __builtin_amdgcn_readlane(prefix(units(b0 + lane)), 63);
  const uint32_t U = (uint32_t)total * pairs;
  uint32_t u = run_begin(U, p.grid, blockIdx.x);
  const uint32_t u_end = run_begin(U, p.grid, blockIdx.x + 1);
  // Sequences without a key have no unit: zeros.
  for (int b = blockIdx.x; b < B; b += p.grid)
    if (len_of(p, b) == 0)
      for (int i = threadIdx.x; i < p.Hq * HD; i += kThreads) p.out[(int64_t)b * p.Hq * HD + i] = f16(0);
  if (u >= u_end) return;
  const int at = (int)(u / pairs);  // units of a sequence come once per pair
  int b = 0, before = 0;
  {
    int b0 = 0, done = 0;
    while (done + __builtin_amdgcn_readlane(sums, 63) <= at) {
      done += __builtin_amdgcn_readlane(sums, 63);
      b0 += 64;
      mine = units(b0 + lane);
      sums = prefix(mine);
    }
    const int i = __builtin_popcountll(__builtin_amdgcn_ballot_w64(done + sums <= at));
    b = b0 + i;
    before = done + __builtin_amdgcn_readlane(sums, i) - __builtin_amdgcn_readlane(mine, i);
  }
  int n_units = (len_of(p, b) + kUnit - 1) / kUnit;
  uint32_t rest = u - (uint32_t)before * pairs;
  int pair = (int)(rest / n_units), c0 = (int)(rest % n_units);

  while (u < u_end) {
    // ---- one pair: units [c0, c1) of sequence b ----
    const int len = len_of(p, b);
    const int c1 = min(n_units, c0 + (int)(u_end - u));
    const int k_end = min(c1 * kUnit, len);
    const int kvh = pair / p.chunks, chunk = pair % p.chunks;
    const int rows = min(kRows, p.n_rep - chunk * kRows);
    const int hq0 = kvh * p.n_rep + chunk * kRows;
    const const_ints table = as_const(kv.table) + (int64_t)b * kv.max_pages;
    const int mask = (1 << kv.page_shift) - 1;
    const int head_row = kvh << kv.page_shift;

    auto pages_of = [&](int kb, int (&pg)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) pg[h] = table[min(kb + 16 * h, k_end - 1) >> kv.page_shift];
    };
    // Rows past k_end, and those of a page outside the pool, are past their descriptors' ends and read as zeros.
    auto fetch = [&](int kb, const int (&pg)[2], Step<KVT, HD>& st) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = kb + 16 * h;
        const bool ok = (unsigned)pg[h] < (unsigned)kv.n_pages;
        const int n = ok ? min(max(k_end - key, 0), 16) : 0;
        const int64_t page = ok ? pg[h] : 0;
        const int row = head_row + (key & mask);
        const int64_t off = page * kv.page_stride + (int64_t)row * S::kBytes;
        const auto kr = __builtin_amdgcn_make_buffer_rsrc(kv.k + off, (short)0, n * S::kBytes, 0x00020000);
        const auto vr = __builtin_amdgcn_make_buffer_rsrc(kv.v + off, (short)0, n * S::kBytes, 0x00020000);
        const int lo = l16 * S::kBytes + lq * S::kLoad;
#pragma unroll
        for (int j = 0; j < S::kLoads; ++j) {
          if constexpr (S::kLoad == 16) {
            st.k[h][j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, lo + 64 * j, 0, 0));
            st.v[h][j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vr, lo + 64 * j, 0, 0));
          } else {
            const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(kr, lo, 0, 0));
            const u32x2 d = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(vr, lo, 0, 0));
            st.k[h][j] = u32x4{a.x, a.y, 0u, 0u};
            st.v[h][j] = u32x4{d.x, d.y, 0u, 0u};
          }
        }
        st.ks[h] = st.vs[h] = 0u;
        if constexpr (KVT != AXM_KV_FP16) {
          const int64_t so = page * kv.scale_stride + (int64_t)row * S::kScale;
          const auto ksr = __builtin_amdgcn_make_buffer_rsrc(kv.ks + so, (short)0, n * S::kScale, 0x00020000);
          const auto vsr = __builtin_amdgcn_make_buffer_rsrc(kv.vs + so, (short)0, n * S::kScale, 0x00020000);
          if constexpr (HD == 128) {
            st.ks[h] = __builtin_amdgcn_raw_buffer_load_b32(ksr, l16 * 4, 0, 0);
            st.vs[h] = __builtin_amdgcn_raw_buffer_load_b32(vsr, l16 * 4, 0, 0);
          } else {
            st.ks[h] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(ksr, l16 * 2, 0, 0);
            st.vs[h] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vsr, l16 * 2, 0, 0);
          }
        }
        st.valid[h] = n;
      }
    };

    f16x8 qa[KS];
#pragma unroll
    for (int j = 0; j < S::kLoads; ++j)
#pragma unroll
      for (int c = 0; c < S::kChunks; ++c) {
        f16x8 x;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = f16(0);
        if (l16 < rows)
          x = kv_order8<KVT>(
              *reinterpret_cast<const f16x8*>(p.q + b * p.ld_q + (int64_t)(hq0 + l16) * HD + S::dim(j, c, lq)));
        qa[j * S::kChunks + c] = x;
      }
    float m[4], l[4];
    f32x4 o[DT];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      m[v] = kNegBig;
      l[v] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};

    auto step = [&](int kb, const Step<KVT, HD>& st) {
      // Values to LDS as they convert, key-major.
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < S::kLoads; ++j)
#pragma unroll
          for (int c = 0; c < S::kChunks; ++c)
            *reinterpret_cast<f16x8*>(&vt[wave][(16 * h + l16) * VROW + S::dim(j, c, lq)]) =
                step_chunk<KVT, HD>(st.v[h][j], st.vs[h], j, c, lq);
      f32x4 sc[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < S::kLoads; ++j)
#pragma unroll
          for (int c = 0; c < S::kChunks; ++c)
            sc[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qa[j * S::kChunks + c],
                                                          step_chunk<KVT, HD>(st.k[h][j], st.ks[h], j, c, lq), sc[h], 0,
                                                          0, 0);
      }
      // Lane (l16, lq) has rows 4 lq + v of keys 16 h + l16.
      float s2[4][2];
      bool grows = false;
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool seen = l16 < st.valid[h];
          s2[v][h] = seen && 4 * lq + v < rows ? sc[h][v] * p.scale_log2 : kNegBig;
          grows |= s2[v][h] > m[v] + kSlack;
          if constexpr (MASS) {
            const int key = kb + 16 * h + l16;
            if (4 * lq + v < rows && key < k_end)
              p.scores[((int64_t)b * p.Hq + hq0 + 4 * lq + v) * p.score_len + key] = seen ? s2[v][h] : -INFINITY;
          }
        }
      if (__builtin_amdgcn_ballot_w64(grows)) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float m_new = fmaxf(m[v], row16_max(fmaxf(s2[v][0], s2[v][1])));
          const float a = fast_exp2(m[v] - m_new);
          m[v] = m_new;
          l[v] *= a;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d][v] *= a;
        }
      }
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w = s2[v][h] == kNegBig ? 0.f : fast_exp2(s2[v][h] - m[v] + kShift);
          l[v] += w;
          // Two fp16 terms: 22 bits of the weight.
          const f16 hi = f2h(w);
          pt[wave][0][pt_index(4 * lq + v, 16 * h + l16)] = hi;
          pt[wave][1][pt_index(4 * lq + v, 16 * h + l16)] = f2h(w - h2f(hi));
        }
      const f16x8 pa = *reinterpret_cast<const f16x8*>(&pt[wave][0][pt_index(l16, 8 * lq)]);
      const f16x8 pb = *reinterpret_cast<const f16x8*>(&pt[wave][1][pt_index(l16, 8 * lq)]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const f16x8 vb = v_operand(&vt[wave][16 * d], VROW, l16, lq);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pa, vb, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pb, vb, o[d], 0, 0, 0);
      }
    };

    const int kb0 = c0 * kUnit + wave * kBlock;
    if (kb0 < k_end) {
      // Two steps' rows in turn: one is on its way while the other is worked on, and the page numbers a step ahead of it.
      Step<KVT, HD> s0, s1;
      int pg[2];
      pages_of(kb0, pg);
      fetch(kb0, pg, s0);
      pages_of(kb0 + kUnit, pg);
      int kb = kb0;
      for (; kb + kUnit < k_end; kb += 2 * kUnit) {
        fetch(kb + kUnit, pg, s1);
        pages_of(kb + 2 * kUnit, pg);
        step(kb, s0);
        fetch(kb + 2 * kUnit, pg, s0);
        pages_of(kb + 3 * kUnit, pg);
        step(kb + kUnit, s1);
      }
      if (kb < k_end) step(kb, s0);
    }

    // ---- join the four waves ----
    lds_float* mine_r = reinterpret_cast<lds_float*>(vt[wave]);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int row = 4 * lq + v;
      const float sum = row16_sum(l[v]);
      if (l16 == 0) {
        mine_r[row * kMergeRow] = m[v];
        mine_r[row * kMergeRow + 1] = sum;
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) mine_r[row * kMergeRow + 2 + 16 * d + kv_col_dim<KVT>(l16)] = o[d][v];
    }
    __syncthreads();
    const bool whole = c0 == 0 && c1 == n_units;
    const uint32_t run = blockIdx.x;
    for (int t = threadIdx.x; t < rows * HD; t += kThreads) {
      const int row = t / HD, e = t % HD;
      float w[kWaves], mm = kNegBig, ll = 0.f, oo = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        w[i] = reinterpret_cast<const lds_float*>(vt[i])[row * kMergeRow];
        mm = fmaxf(mm, w[i]);
      }
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        const float a = fast_exp2(w[i] - mm);
        ll += a * reinterpret_cast<const lds_float*>(vt[i])[row * kMergeRow + 1];
        oo += a * reinterpret_cast<const lds_float*>(vt[i])[row * kMergeRow + 2 + e];
      }
      const int64_t r = (int64_t)b * p.Hq + hq0 + row;
      if (whole) {
        p.out[r * HD + e] = f2h(ll == 0.f ? 0.f : oo / ll);
        if (MASS && e == 0) p.ml[r] = f32x2{mm, ll};
      } else {
        // A part that begins its pair ends the run (slot 1), any other part begins it (slot 0).
        float* to = p.parts + ((int64_t)(2 * run + (c0 == 0 ? 1 : 0)) * kRows + row) * kMergeRow;
        if (e == 0) {
          to[0] = mm;
          to[1] = ll;
        }
        to[2 + e] = oo;
      }
    }
    if (c0 == 0 && threadIdx.x == 0 && p.info) {
      int* to = p.info + ((int64_t)b * pairs + pair) * 2;
      to[0] = (int)run;
      to[1] = (int)run_of(U, p.grid, u + n_units - 1);
    }
    u += c1 - c0;
    c0 = 0;
    if (u < u_end) {
      if (++pair == pairs) {
        pair = 0;
        do ++b;
        while ((n_units = (len_of(p, b) + kUnit - 1) / kUnit) == 0);
      }
      __syncthreads();  // the value tiles are free again
    }
  }
}

// Second launch.  Workgroups [0, n_seqs Hq) join the parts of one query row each, the waves taking parts in turn.  The
// others (account only) take kMassKeys keys of one (sequence, KV head): the row's maxima and sums first, then
// mass += sum over the group's rows of exp2(score - max) / sum.
constexpr int kMassKeys = 1024;

__device__ __forceinline__ const float* part_of(const DecodeParams& p, int hd, int w, int w0, int row) {
  return p.parts + ((int64_t)(2 * w + (w == w0 ? 1 : 0)) * kRows + row) * (2 + hd);
}

template <int HD>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(DecodeParams p, int join_blocks, int slices) {
  constexpr int E = HD / 64;
  __shared__ float red[kWaves][2 + HD];
  __shared__ f32x2 ml[64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int pairs = p.kv.Hkv * p.chunks;
  if ((int)blockIdx.x < join_blocks) {
    const int b = blockIdx.x / p.Hq, hq = blockIdx.x % p.Hq;
    const int r = hq % p.n_rep, pair = hq / p.n_rep * p.chunks + r / kRows, row = r % kRows;
    if (len_of(p, b) == 0) return;
    const int* info = p.info + ((int64_t)b * pairs + pair) * 2;
    const int w0 = info[0], w1 = info[1];
    if (w0 == w1) return;  // stored already
    float m = kNegBig, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    constexpr int kAhead = 4;  // parts requested together
    for (int w = w0 + wave; w <= w1; w += kWaves * kAhead) {
      float pm[kAhead], pl[kAhead], po[kAhead][E];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const bool in = w + i * kWaves <= w1;
        const float* from = part_of(p, HD, in ? w + i * kWaves : w, w0, row);
        pm[i] = in ? from[0] : kNegBig;
        pl[i] = in ? from[1] : 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) po[i][e] = in ? from[2 + lane + 64 * e] : 0.f;
      }
      float mm = m;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) mm = fmaxf(mm, pm[i]);
      const float a = fast_exp2(m - mm);
      l *= a;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] *= a;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float x = fast_exp2(pm[i] - mm);
        l += x * pl[i];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += x * po[i][e];
      }
      m = mm;
    }
    red[wave][0] = m;
    red[wave][1] = l;
#pragma unroll
    for (int e = 0; e < E; ++e) red[wave][2 + lane + 64 * e] = o[e];
    __syncthreads();
    if (threadIdx.x < HD) {
      float mm = kNegBig, ll = 0.f, oo = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) mm = fmaxf(mm, red[i][0]);
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        const float x = fast_exp2(red[i][0] - mm);
        ll += x * red[i][1];
        oo += x * red[i][2 + threadIdx.x];
      }
      p.out[(int64_t)blockIdx.x * HD + threadIdx.x] = f2h(ll == 0.f ? 0.f : oo / ll);
    }
    return;
  }
  const int item = blockIdx.x - join_blocks;
  const int bh = item / slices, b = bh / p.kv.Hkv, kvh = bh % p.kv.Hkv;
  const int k0 = item % slices * kMassKeys, k1 = min(k0 + kMassKeys, len_of(p, b));
  if (k0 >= k1) return;
  for (int r = wave; r < p.n_rep; r += kWaves) {
    const int64_t hq = (int64_t)b * p.Hq + kvh * p.n_rep + r;
    int w0 = 0, w1 = 0;
    if (p.info) {
      const int* info = p.info + ((int64_t)b * pairs + kvh * p.chunks + r / kRows) * 2;
      w0 = info[0];
      w1 = info[1];
    }
    f32x2 x;
    if (w0 == w1) {
      x = p.ml[hq];
    } else {
      float m = kNegBig, l = 0.f;
      for (int w = w0 + lane; w <= w1; w += 64) {
        const float* from = part_of(p, HD, w, w0, r % kRows);
        const float mm = fmaxf(m, from[0]);
        l = l * fast_exp2(m - mm) + from[1] * fast_exp2(from[0] - mm);
        m = mm;
      }
      const float mm = wave_max(m);
      x = f32x2{mm, wave_sum(l * fast_exp2(m - mm))};
    }
    if (lane == 0) ml[r] = f32x2{x.x - kShift, x.y == 0.f ? 0.f : 1.f / x.y};
  }
  __syncthreads();
  float* mass = p.mass + (int64_t)bh * p.mass_len;
  const float* scores = p.scores + ((int64_t)b * p.Hq + kvh * p.n_rep) * p.score_len;
  for (int key = k0 + threadIdx.x; key < k1; key += kThreads) {
    float sum = 0.f;
    for (int r = 0; r < p.n_rep; ++r) sum += fast_exp2(scores[r * p.score_len + key] - ml[r].x) * ml[r].y;
    mass[key] += sum;
  }
}

template <int KVT, int HD>
void launch_decode(const DecodeParams& p, hipStream_t s) {
  if (p.mass) hipLaunchKernelGGL((paged_decode_kernel<KVT, HD, true>), dim3(p.grid), dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((paged_decode_kernel<KVT, HD, false>), dim3(p.grid), dim3(kThreads), 0, s, p);
}

// Workgroups of the first launch: two per CU, no more than units at the table's capacity.
int decode_grid(int64_t most_units) {
  const int64_t full = 2 * (int64_t)axm_num_cus();
  return (int)(most_units < full ? most_units : full);
}

struct Workspace {
  size_t parts, info, ml, scores, bytes;  // offsets, 256-byte aligned
};
Workspace workspace_of(int n_seqs, int Hq, int Hkv, int hd, int64_t capacity, bool mass) {
  const int64_t per = (capacity + kUnit - 1) / kUnit, pairs = (int64_t)Hkv * ((Hq / Hkv + kRows - 1) / kRows);
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  Workspace w{};
  const bool parts = per > 1;
  w.info = w.parts + up(parts ? (size_t)decode_grid(n_seqs * pairs * per) * 2 * kRows * (2 + hd) * 4 : 0);
  w.ml = w.info + up(parts ? (size_t)n_seqs * pairs * 8 : 0);
  w.scores = w.ml + up(mass ? (size_t)n_seqs * Hq * 8 : 0);
  w.bytes = w.scores + up(mass ? (size_t)n_seqs * Hq * capacity * 4 : 0);
  return w;
}

}  // namespace

extern "C" size_t axm_paged_decode_workspace_bytes(int n_seqs, int n_head, int n_kv_head, int head_dim, int page_size,
                                                   int max_pages, int with_mass) {
  if (n_seqs < 1 || n_kv_head < 1 || n_head < n_kv_head || page_size < 1 || max_pages < 1) return 0;
  return workspace_of(n_seqs, n_head, n_kv_head, head_dim, (int64_t)page_size * max_pages, with_mass != 0).bytes;
}

extern "C" int axm_paged_flash_decode(const void* q, int64_t ld_q, const axm_paged_kv* d, const int* seq_lens, void* out,
                                      int n_head, float* mass, int64_t mass_len, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  DecodeParams p{};
  if (int rc = paged_view(d, "paged_flash_decode", &p.kv)) return rc;
  const PagedKv& kv = p.kv;
  AXM_CHECK_ARG(q && seq_lens && out, -1, "paged_flash_decode: null pointer");
  AXM_CHECK_ARG(n_head >= kv.Hkv && n_head % kv.Hkv == 0 && n_head / kv.Hkv <= 64, -1,
                "paged_flash_decode: n_head=%d not a multiple (up to 64) of n_kv_head=%d", n_head, kv.Hkv);
  AXM_CHECK_ARG(ld_q >= (int64_t)n_head * kv.hd && ld_q % 8 == 0 && (uintptr_t)q % 16 == 0, -1,
                "paged_flash_decode: query rows %lld halves apart must be 16-byte aligned", (long long)ld_q);
  const int64_t capacity = (int64_t)kv.max_pages << kv.page_shift;
  AXM_CHECK_ARG(!mass || mass_len >= capacity, -1, "paged_flash_decode: mass has %lld slots, the table %lld",
                (long long)mass_len, (long long)capacity);
  p.n_rep = n_head / kv.Hkv;
  p.chunks = (p.n_rep + kRows - 1) / kRows;
  const int64_t per = (capacity + kUnit - 1) / kUnit, units = per * kv.n_seqs * kv.Hkv * p.chunks;
  const int slices = (int)((capacity + kMassKeys - 1) / kMassKeys);
  AXM_CHECK_ARG(units < (1ll << 31) && (int64_t)kv.n_seqs * n_head * (1 + slices) < (1 << 24), -1,
                "paged_flash_decode: %d sequences of %d heads and up to %lld slots are too many for one call", kv.n_seqs,
                n_head, (long long)capacity);
  const Workspace w = workspace_of(kv.n_seqs, n_head, kv.Hkv, kv.hd, capacity, mass != nullptr);
  AXM_CHECK_ARG(workspace_bytes >= w.bytes && (w.bytes == 0 || (workspace && (uintptr_t)workspace % 16 == 0)), -1,
                "paged_flash_decode: workspace of %zu bytes needed (16-byte aligned), %zu given", w.bytes,
                workspace_bytes);
  const hipStream_t s = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace;
  const bool parts = per > 1;
  p.q = (const f16*)q;
  p.ld_q = ld_q;
  p.lens = seq_lens;
  p.out = (f16*)out;
  p.parts = parts ? (float*)(ws + w.parts) : nullptr;
  p.info = parts ? (int*)(ws + w.info) : nullptr;
  p.ml = mass ? (f32x2*)(ws + w.ml) : nullptr;
  p.scores = mass ? (float*)(ws + w.scores) : nullptr;
  p.score_len = capacity;
  p.mass = mass;
  p.mass_len = mass_len;
  p.Hq = n_head;
  p.grid = decode_grid(units);
  p.max_len = (int)capacity;
  p.scale_log2 = kLog2e / __builtin_sqrtf((float)kv.hd);
  switch (kv.kv_dtype * 2 + (kv.hd == 128)) {
    case 0: launch_decode<AXM_KV_FP16, 64>(p, s); break;
    case 1: launch_decode<AXM_KV_FP16, 128>(p, s); break;
    case 2: launch_decode<AXM_KV_FP8, 64>(p, s); break;
    case 3: launch_decode<AXM_KV_FP8, 128>(p, s); break;
    case 4: launch_decode<AXM_KV_INT4, 64>(p, s); break;
    default: launch_decode<AXM_KV_INT4, 128>(p, s); break;
  }
  AXM_LAUNCH_CHECK("paged_flash_decode");
  const int join = parts ? kv.n_seqs * n_head : 0, account = mass ? kv.n_seqs * kv.Hkv * slices : 0;
  if (join + account) {
    if (kv.hd == 128)
      hipLaunchKernelGGL((paged_join_kernel<128>), dim3(join + account), dim3(kThreads), 0, s, p, join, slices);
    else
      hipLaunchKernelGGL((paged_join_kernel<64>), dim3(join + account), dim3(kThreads), 0, s, p, join, slices);
    AXM_LAUNCH_CHECK("paged_flash_decode (join)");
  }
  return 0;
}
