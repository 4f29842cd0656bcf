// Decode attention of one new token per sequence over a paged KV cache.
//
//   out[b][hq] = sum_s p_s v_s,  p = softmax(q k_s / sqrt(hd)) over s < seq_lens[b]
//
// Every cached row is read once and serves all query heads of its KV head: their rows (up to 16 a pass) are one tile of
// v_mfma_f32_16x16x32_f16.  The work is the list of 32-key blocks of all (sequence, KV head) pairs, and every wave takes
// an equal run of it, whatever the lengths are, loading a block ahead across the pairs' borders.  A run holds whole pairs
// and a piece of one pair at each end; a workgroup joins its waves' pieces in LDS.  A pair that one workgroup has whole
// is stored as fp16; others leave fp32 (max, sum, sum of p v), joined by a second launch, which also turns stored
// scores into the account of weights.
#include <type_traits>

#include "kv_device.h"
#include "paged_kv.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kBlock = 32;  // keys of a step: the k extent of one P V instruction
constexpr int kRows = 16;   // query rows of a tile
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
  int* info;       // [sequence][pair][2]: first and last workgroup of a pair, -1 where one stored it
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

// Wave w's run of U blocks over `waves`: U / waves of them, one more in the first U % waves.
__device__ __forceinline__ uint32_t run_begin(uint32_t U, uint32_t waves, uint32_t w) {
  return U / waves * w + min(w, U % waves);
}
__device__ __forceinline__ uint32_t run_of(uint32_t U, uint32_t waves, uint32_t u) {
  const uint32_t each = U / waves, more = U % waves, head = more * (each + 1);
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

// One 32-key block of a run.
struct Block {
  int b, kvh, chunk, c, n;  // sequence, KV head, its tile of query rows, block c of the sequence's n
  int len;                  // the sequence's keys; 0: past the run
  int page[2];              // of keys 32 c and 32 c + 16
};

// A value that all lanes of the wave share, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Inclusive sums over the wave's lanes, on DPP moves: shifts inside rows of 16, then the rows' last lanes onward.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, true);
}
__device__ __forceinline__ int wave_prefix(int x) {
  x = dpp_add<0x111, 0xF>(x);  // row_shr:1
  x = dpp_add<0x112, 0xF>(x);
  x = dpp_add<0x114, 0xF>(x);
  x = dpp_add<0x118, 0xF>(x);
  x = dpp_add<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
  return dpp_add<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
}
// Descriptor of n bytes from p + off, built in scalar registers: left to itself the compiler takes some of its words
// for per-lane values (a median of three is a vector instruction) and loops over the lanes around every load.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const uint8_t* p, int64_t off, int n) {
  const uint64_t a = (uint64_t)(uintptr_t)p + (uint64_t)off;
  const uint64_t u = (uint64_t)(uint32_t)uniform((int)(a >> 32)) << 32 | (uint32_t)uniform((int)a);
  return __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)u, (short)0, uniform(n), 0x00020000);
}

// A piece of a pair that a wave could not finish alone, in LDS until the workgroup joins its waves' pieces.
struct Piece {
  int b, pair;    // b < 0: none
  int ended;      // whether the piece reaches the sequence's end
  uint32_t last;  // the pair's last block, in the order of all blocks
};

// NV: query rows of a lane (4 NV or fewer rows in all).  Row r is tile row 4 (r % 4) + r / 4, so that the lanes of a tile
// share the rows evenly: with four heads per KV head every lane has one row to weigh instead of some lanes four (us, NV
// by the rows / always 4: 128 INT4 sequences of 8 rows 25.5 / 28.0, one sequence of one row 5.4 / 6.0, 48 fp16 ones of
// four 50.7 / 51.0).
// Each half of a block has its page looked up: it may be another one with pages of 16, and one lookup for both where it
// is not was no faster (48 fp16 sequences, pages of 64: 50.7 with one, 49.8 with two).
template <int KVT, int HD, int NV>
__global__ void __launch_bounds__(kThreads, 2) paged_decode_kernel(DecodeParams p) {
  using S = RowShape<KVT, HD>;
  constexpr int KS = HD / 32, DT = HD / 16;
  constexpr int VROW = HD + 16;
  constexpr int kMergeRow = 2 + HD;
  static_assert(kRows * kMergeRow * 4 <= kBlock * VROW * 2, "a piece fits a value tile");
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ Piece piece[kWaves][2];
  const PagedKv& kv = p.kv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, lq = lane >> 4;
  const int B = kv.n_seqs, pairs = kv.Hkv * p.chunks, most_rows = min(p.n_rep, kRows);
  f16* vt = reinterpret_cast<f16*>(lds) + wave * (kBlock * VROW);
  f16* pt = reinterpret_cast<f16*>(lds) + kWaves * (kBlock * VROW) + wave * (2 * kRows * kBlock);
  // Pieces: a wave's last one lies where its value tile was, the first one behind the tiles.
  auto piece_at = [&](int w, int slot) {
    return reinterpret_cast<lds_float*>(slot ? lds + w * (kBlock * VROW * 2)
                                             : lds + kWaves * (kBlock * VROW + 2 * kRows * kBlock) * 2 +
                                                   w * (most_rows * kMergeRow * 4));
  };
  if (lane < 2) piece[wave][lane].b = -1;

  // ---- this wave's run of blocks ----
  auto blocks_of = [&](int len) { return (len + kBlock - 1) / kBlock; };
  const uint32_t waves = (uint32_t)p.grid * kWaves;
  uint32_t U = 0, u0 = 0;
  int count;
  Block lead;  // the next block whose pages are asked for
  if (p.info == nullptr) {  // a workgroup per pair
    lead.b = blockIdx.x / pairs;
    lead.kvh = blockIdx.x % pairs / p.chunks;
    lead.chunk = blockIdx.x % pairs % p.chunks;
    lead.len = len_of(p, lead.b);
    lead.n = blocks_of(lead.len);
    lead.c = (int)run_begin(lead.n, kWaves, wave);
    count = (int)run_begin(lead.n, kWaves, wave + 1) - lead.c;
  } else {
    auto len_at = [&](int b) { return b < B ? min(max(p.lens[b], 0), p.max_len) : 0; };
    int len = len_at(lane), sums = wave_prefix(blocks_of(len));
    int total = __builtin_amdgcn_readlane(sums, 63);
    for (int b0 = 64; b0 < B; b0 += 64) total += __builtin_amdgcn_readlane(wave_prefix(blocks_of(len_at(b0 + lane))), 63);
    U = (uint32_t)total * pairs;
    u0 = run_begin(U, waves, blockIdx.x * kWaves + wave);
    count = (int)(run_begin(U, waves, blockIdx.x * kWaves + wave + 1) - u0);
    if (count > 0) {
      const int at = (int)(u0 / pairs);  // a sequence's blocks come once per pair
      int b0 = 0, done = 0;
      while (done + __builtin_amdgcn_readlane(sums, 63) <= at) {
        done += __builtin_amdgcn_readlane(sums, 63);
        b0 += 64;
        len = len_at(b0 + lane);
        sums = wave_prefix(blocks_of(len));
      }
      const int i = __builtin_popcountll(__builtin_amdgcn_ballot_w64(done + sums <= at));
      lead.b = b0 + i;
      lead.len = __builtin_amdgcn_readlane(len, i);
      lead.n = blocks_of(lead.len);
      const uint32_t rest = u0 - (uint32_t)(done + __builtin_amdgcn_readlane(sums, i) - lead.n) * pairs;
      const int pair = (int)(rest / lead.n);
      lead.c = (int)(rest - (uint32_t)pair * lead.n);
      lead.kvh = p.chunks == 1 ? pair : pair / p.chunks;
      lead.chunk = p.chunks == 1 ? 0 : pair % p.chunks;
    }
  }

  if (count > 0) {
    int left = uniform(count);
    lead = Block{uniform(lead.b), uniform(lead.kvh), uniform(lead.chunk), uniform(lead.c), uniform(lead.n),
                 uniform(lead.len), {0, 0}};
    auto next = [&]() {  // the lead block with its pages, and the lead one further
      Block x = lead;
      x.page[0] = x.page[1] = -1;
      if (left == 0) {
        x.len = 0;
        return x;
      }
      const const_ints table = as_const(kv.table) + (int64_t)x.b * kv.max_pages;
      x.page[0] = table[x.c * kBlock >> kv.page_shift];
      x.page[1] = table[min(x.c * kBlock + 16, x.len - 1) >> kv.page_shift];
      if (--left > 0 && ++lead.c == lead.n) {
        lead.c = 0;
        if (++lead.chunk == p.chunks) {
          lead.chunk = 0;
          ++lead.kvh;
        }
        if (lead.kvh == kv.Hkv) {
          lead.kvh = 0;
          do lead.len = len_of(p, ++lead.b);
          while (lead.len == 0);
          lead.n = blocks_of(lead.len);
        }
      }
      return x;
    };
    auto counting = [&](const Block& x, int h) {  // keys of half h that count
      return (unsigned)x.page[h] < (unsigned)kv.n_pages ? min(max(x.len - x.c * kBlock - 16 * h, 0), 16) : 0;
    };
    // Rows past the sequence, and those of a page outside the pool, are past their descriptors' ends and read as zeros.
    auto fetch = [&](const Block& x, Step<KVT, HD>& st) {
      const int mask = (1 << kv.page_shift) - 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool ok = (unsigned)x.page[h] < (unsigned)kv.n_pages;
        const int n = ok ? min(max(x.len - x.c * kBlock - 16 * h, 0), 16) : 0;
        const int64_t page = ok ? x.page[h] : 0;
        const int row = (x.kvh << kv.page_shift) + ((x.c * kBlock + 16 * h) & mask);
        const int64_t off = page * kv.page_stride + row * S::kBytes;
        const auto kr = rows_at(kv.k, off, n * S::kBytes);
        const auto vr = rows_at(kv.v, off, n * S::kBytes);
        const int64_t so = page * kv.scale_stride + row * S::kScale;
        __amdgpu_buffer_rsrc_t ksr = kr, vsr = vr;
        if constexpr (KVT != AXM_KV_FP16) {
          ksr = rows_at(kv.ks, so, n * S::kScale);
          vsr = rows_at(kv.vs, so, n * S::kScale);
        }
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
          if constexpr (HD == 128) {
            st.ks[h] = __builtin_amdgcn_raw_buffer_load_b32(ksr, l16 * S::kScale, 0, 0);
            st.vs[h] = __builtin_amdgcn_raw_buffer_load_b32(vsr, l16 * S::kScale, 0, 0);
          } else {
            st.ks[h] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(ksr, l16 * S::kScale, 0, 0);
            st.vs[h] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(vsr, l16 * S::kScale, 0, 0);
          }
        }
      }
    };

    f16x8 qa[KS];
    float m[NV], l[NV];
    f32x4 o[DT];
    int from = lead.c;  // first block of the piece in hand
    auto begin = [&](const Block& x) {
      const int r = (l16 >> 2) + 4 * (l16 & 3), rows = min(kRows, p.n_rep - x.chunk * kRows);
      const f16* q = p.q + x.b * p.ld_q + (int64_t)(x.kvh * p.n_rep + x.chunk * kRows + r) * HD;
#pragma unroll
      for (int j = 0; j < S::kLoads; ++j)
#pragma unroll
        for (int c = 0; c < S::kChunks; ++c) {
          f16x8 y;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = f16(0);
          if (r < rows) y = kv_order8<KVT>(*reinterpret_cast<const f16x8*>(q + S::dim(j, c, lq)));
          qa[j * S::kChunks + c] = y;
        }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        m[v] = kNegBig;
        l[v] = 0.f;
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
      from = x.c;
    };
    f32x4 sc[2];
    auto take = [&](const Step<KVT, HD>& st) {
      // Values to LDS as they convert, key-major; scores.
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < S::kLoads; ++j)
#pragma unroll
          for (int c = 0; c < S::kChunks; ++c)
            *reinterpret_cast<f16x8*>(&vt[(16 * h + l16) * VROW + S::dim(j, c, lq)]) =
                step_chunk<KVT, HD>(st.v[h][j], st.vs[h], j, c, lq);
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
    };
    auto weigh = [&](const Block& x) {
      const int rows = min(kRows, p.n_rep - x.chunk * kRows);
      // Lane (l16, lq) has rows lq + 4 v of keys 16 h + l16.
      float s2[NV][2];
      bool grows = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool seen = l16 < counting(x, h);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          s2[v][h] = seen && lq + 4 * v < rows ? sc[h][v] * p.scale_log2 : kNegBig;
          grows |= s2[v][h] > m[v] + kSlack;
        }
        if (p.scores != nullptr) {
          const int key = x.c * kBlock + 16 * h + l16;
          const int64_t hq = (int64_t)x.b * p.Hq + x.kvh * p.n_rep + x.chunk * kRows + lq;
#pragma unroll
          for (int v = 0; v < NV; ++v)
            if (lq + 4 * v < rows && key < x.len) p.scores[(hq + 4 * v) * p.score_len + key] = seen ? s2[v][h] : -INFINITY;
        }
      }
      if (__builtin_amdgcn_ballot_w64(grows)) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          const float m_new = fmaxf(m[v], row16_max(fmaxf(s2[v][0], s2[v][1])));
          const float a = fast_exp2(m[v] - m_new);
          m[v] = m_new;
          l[v] *= a;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d][v] *= a;
        }
      }
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float w = s2[v][h] == kNegBig ? 0.f : fast_exp2(s2[v][h] - m[v] + kShift);
          l[v] += w;
          // Two fp16 terms: 22 bits of the weight.  Tile rows of no query row keep what was in LDS: rows do not mix.
          const f16 hi = f2h(w);
          pt[pt_index(4 * lq + v, 16 * h + l16)] = hi;
          pt[kRows * kBlock + pt_index(4 * lq + v, 16 * h + l16)] = f2h(w - h2f(hi));
        }
      const f16x8 pa = *reinterpret_cast<const f16x8*>(&pt[pt_index(l16, 8 * lq)]);
      const f16x8 pb = *reinterpret_cast<const f16x8*>(&pt[kRows * kBlock + pt_index(l16, 8 * lq)]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const f16x8 vb = v_operand(&vt[16 * d], VROW, l16, lq);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pa, vb, o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pb, vb, o[d], 0, 0, 0);
      }
    };
    // The piece in hand ends with block x: out as it is, or kept for the join.
    auto end = [&](const Block& x, int i) {
      const int rows = min(kRows, p.n_rep - x.chunk * kRows);
      const bool ended = x.c + 1 == x.n, whole = from == 0 && ended;
      lds_float* to = piece_at(wave, from == 0);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int row = lq + 4 * v;
        const float sum = row16_sum(l[v]);
        if (row >= rows) continue;
        if (whole) {
          const int64_t r = (int64_t)x.b * p.Hq + x.kvh * p.n_rep + x.chunk * kRows + row;
#pragma unroll
          for (int d = 0; d < DT; ++d)
            p.out[r * HD + 16 * d + kv_col_dim<KVT>(l16)] = f2h(sum == 0.f ? 0.f : o[d][v] / sum);
          if (p.ml != nullptr && l16 == 0) p.ml[r] = f32x2{m[v], sum};
        } else {
          if (l16 == 0) {
            to[row * kMergeRow] = m[v];
            to[row * kMergeRow + 1] = sum;
          }
#pragma unroll
          for (int d = 0; d < DT; ++d) to[row * kMergeRow + 2 + 16 * d + kv_col_dim<KVT>(l16)] = o[d][v];
        }
      }
      if (lane == 0) {
        const int pair = x.kvh * p.chunks + x.chunk;
        if (!whole) piece[wave][from == 0] = Piece{x.b, pair, ended, u0 + i + (x.n - 1 - x.c)};
        else if (p.info) p.info[((int64_t)x.b * pairs + pair) * 2] = -1;
      }
    };

    // A block's rows are asked for as soon as those of the one before have been taken, the page numbers a block earlier.
    Step<KVT, HD> st;
    Block x = next();
    fetch(x, st);
    Block y = next();
    begin(x);
    for (int i = 0; i < count; ++i) {
      take(st);
      fetch(y, st);
      weigh(x);
      const Block z = x;
      x = y;
      y = next();
      if (z.c + 1 == z.n || i + 1 == count) {
        end(z, i);
        begin(x);
      }
    }
  }

  // ---- sequences without a key have no block: zeros ----
#pragma unroll 1
  for (int b = p.info ? blockIdx.x : blockIdx.x % pairs ? B : blockIdx.x / pairs; b < B; b += p.grid) {
    if (len_of(p, b) != 0) continue;
#pragma unroll 1
    for (int i = threadIdx.x; i < p.Hq * HD / 8; i += kThreads)
      reinterpret_cast<u32x4*>(p.out + (int64_t)b * p.Hq * HD)[i] = u32x4{0u, 0u, 0u, 0u};
    if (p.info)
#pragma unroll 1
      for (int i = threadIdx.x; i < pairs; i += kThreads) p.info[((int64_t)b * pairs + i) * 2] = -1;
  }

  // ---- join the waves' pieces ----
  __syncthreads();
#pragma unroll 1
  for (int s = 0; s <= kWaves; ++s) {
    // A chain of pieces of one pair starts with the workgroup's first piece, or with one that begins its pair, and goes on
    // through the following waves' first pieces.
    const int w0 = s == 0 ? 0 : s - 1, slot = s == 0 ? 0 : 1;
    const int b = uniform(piece[w0][slot].b), pair = uniform(piece[w0][slot].pair);
    if (b < 0) continue;
    int w1 = w0, ended = uniform(piece[w0][slot].ended);
    while (!ended && w1 + 1 < kWaves && uniform(piece[w1 + 1][0].b) >= 0) ended = uniform(piece[++w1][0].ended);
    const int kvh = p.chunks == 1 ? pair : pair / p.chunks, chunk = p.chunks == 1 ? 0 : pair % p.chunks;
    const int rows = min(kRows, p.n_rep - chunk * kRows);
    const bool whole = slot == 1 && ended;
    const int64_t r0 = (int64_t)b * p.Hq + kvh * p.n_rep + chunk * kRows;
#pragma unroll 1
    for (int t = threadIdx.x; t < rows * HD; t += kThreads) {
      const int row = t / HD, e = t % HD;
      const lds_float* x = piece_at(w0, slot) + row * kMergeRow;
      float mm = x[0], ll = x[1], oo = x[2 + e];
#pragma unroll 1
      for (int w = w0 + 1; w <= w1; ++w) {
        x = piece_at(w, 0) + row * kMergeRow;
        const float m2 = x[0], top = fmaxf(mm, m2), a = fast_exp2(mm - top), c = fast_exp2(m2 - top);
        mm = top;
        ll = a * ll + c * x[1];
        oo = a * oo + c * x[2 + e];
      }
      if (whole) {
        p.out[(r0 + row) * HD + e] = f2h(ll == 0.f ? 0.f : oo / ll);
        if (p.ml != nullptr && e == 0) p.ml[r0 + row] = f32x2{mm, ll};
      } else {
        // A part that begins its pair ends the run (slot 1), any other part begins it (slot 0).
        float* to = p.parts + ((int64_t)(2 * blockIdx.x + slot) * kRows + row) * kMergeRow;
        if (e == 0) {
          to[0] = mm;
          to[1] = ll;
        }
        to[2 + e] = oo;
      }
    }
    if (slot == 1 && threadIdx.x == 0 && p.info) {
      int* to = p.info + ((int64_t)b * pairs + pair) * 2;
      to[0] = whole ? -1 : (int)blockIdx.x;
      to[1] = (int)(run_of(U, waves, piece[w0][slot].last) / kWaves);
    }
  }
}

// Second launch.  The first join_blocks workgroups join the parts of query rows, WPR waves a row taking parts in turn.  The
// others (account only) take kMassKeys keys of one (sequence, KV head): the row's maxima and sums first, then
// mass += sum over the group's rows of exp2(score - max) / sum.
constexpr int kMassKeys = 1024;

__device__ __forceinline__ const float* part_of(const DecodeParams& p, int hd, int w, int w0, int row) {
  return p.parts + ((int64_t)(2 * w + (w == w0 ? 1 : 0)) * kRows + row) * (2 + hd);
}

template <int HD, int WPR>
__global__ void __launch_bounds__(kThreads) paged_join_kernel(DecodeParams p, int join_blocks, int slices) {
  constexpr int E = HD / 64;
  __shared__ float red[kWaves][2 + HD];
  __shared__ f32x2 ml[64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int pairs = p.kv.Hkv * p.chunks;
  if ((int)blockIdx.x < join_blocks) {
    constexpr int kRowsHere = kWaves / WPR;
    const int64_t r = (int64_t)blockIdx.x * kRowsHere + wave / WPR;  // of n_seqs Hq
    const bool in = r < (int64_t)p.kv.n_seqs * p.Hq;
    const int b = in ? (int)(r / p.Hq) : 0, hq = in ? (int)(r - (int64_t)b * p.Hq) : 0;
    const int kvh = hq / p.n_rep, rr = hq - kvh * p.n_rep, row = rr % kRows;
    const const_ints info = as_const(p.info) + ((int64_t)b * pairs + kvh * p.chunks + rr / kRows) * 2;
    const int w0 = in ? info[0] : -1, w1 = info[1];
    if (WPR == kWaves && w0 < 0) return;  // stored already
    float m = kNegBig, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    if (w0 >= 0) {
      constexpr int kAhead = 4;  // parts requested together
      for (int w = w0 + wave % WPR; w <= w1; w += WPR * kAhead) {
        float pm[kAhead], pl[kAhead], po[kAhead][E];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const bool has = w + i * WPR <= w1;
          const float* from = part_of(p, HD, has ? w + i * WPR : w, w0, row);
          pm[i] = has ? from[0] : kNegBig;
          pl[i] = has ? from[1] : 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) po[i][e] = has ? from[2 + lane + 64 * e] : 0.f;
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
    }
    if constexpr (WPR == 1) {
      if (w0 >= 0)
#pragma unroll
        for (int e = 0; e < E; ++e) p.out[r * HD + lane + 64 * e] = f2h(l == 0.f ? 0.f : o[e] / l);
      return;
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
      p.out[r * HD + threadIdx.x] = f2h(ll == 0.f ? 0.f : oo / ll);
    }
    return;
  }
  const int item = blockIdx.x - join_blocks;
  const int bh = item / slices, b = bh / p.kv.Hkv, kvh = bh % p.kv.Hkv;
  const int k0 = item % slices * kMassKeys, k1 = min(k0 + kMassKeys, len_of(p, b));
  if (k0 >= k1) return;
  for (int r = wave; r < p.n_rep; r += kWaves) {
    const int64_t hq = (int64_t)b * p.Hq + kvh * p.n_rep + r;
    int w0 = -1, w1 = 0;
    if (p.info) {
      const int* info = p.info + ((int64_t)b * pairs + kvh * p.chunks + r / kRows) * 2;
      w0 = info[0];
      w1 = info[1];
    }
    f32x2 x;
    if (w0 < 0) {
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
  const int rows = p.n_rep < kRows ? p.n_rep : kRows;
  const size_t lds = kWaves * ((kBlock * (HD + 16) + 2 * kRows * kBlock) * 2 + rows * (2 + HD) * 4);
  const dim3 grid(p.grid), block(kThreads);
  if (rows <= 4) hipLaunchKernelGGL((paged_decode_kernel<KVT, HD, 1>), grid, block, lds, s, p);
  else if (rows <= 8) hipLaunchKernelGGL((paged_decode_kernel<KVT, HD, 2>), grid, block, lds, s, p);
  else hipLaunchKernelGGL((paged_decode_kernel<KVT, HD, 4>), grid, block, lds, s, p);
}

// Up to this many blocks of capacity a workgroup takes a pair whole and nothing is joined by a second launch (us, one
// launch / two; fp16: one sequence of 100 keys, 4 heads of 64, 5.4 / 7.2; 8 KV heads of 128: one of 256 8.9 / 10.0, 16 of
// 250 8.9 / 10.4; one of 500 12.1 / 10.2, 64 of 500 19.2 / 17.9, one of 1000 19.0 / 10.1).
constexpr int kPairBlocks = 8;

// Workgroups of the first launch otherwise; no more than have a block at the table's capacity.  Per CU two where rows
// are long, three where a wave's registers and its steps' bytes are few (128 sequences, INT4, heads of 64: 28.4 us with
// two, 26.6 with three, 26.8 with four; 48 sequences, fp16, heads of 128: 50.4, 50.8, 52.6).
int decode_grid(int64_t most_blocks, int per_cu) {
  const int64_t full = per_cu * (int64_t)axm_num_cus(), used = (most_blocks + kWaves - 1) / kWaves;
  return (int)(used < full ? used : full);
}
int per_cu(int kv_dtype, int hd) { return paged_row_bytes(kv_dtype, hd) <= 64 ? 3 : 2; }

struct Workspace {
  size_t parts, info, ml, scores, bytes;  // offsets, 256-byte aligned
};
Workspace workspace_of(int n_seqs, int Hq, int Hkv, int hd, int64_t capacity, bool mass) {
  const int64_t per = (capacity + kBlock - 1) / kBlock, pairs = (int64_t)Hkv * ((Hq / Hkv + kRows - 1) / kRows);
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  Workspace w{};
  const bool parts = per > kPairBlocks;
  w.info = w.parts + up(parts ? (size_t)decode_grid(n_seqs * pairs * per, 3) * 2 * kRows * (2 + hd) * 4 : 0);
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
  AXM_CHECK_ARG((uintptr_t)out % 16 == 0, -1, "paged_flash_decode: out must be 16-byte aligned");
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
  const int64_t per = (capacity + kBlock - 1) / kBlock, blocks = per * kv.n_seqs * kv.Hkv * p.chunks;
  const int slices = (int)((capacity + kMassKeys - 1) / kMassKeys);
  AXM_CHECK_ARG(blocks < (1ll << 31) && (int64_t)kv.n_seqs * n_head * (1 + slices) < (1 << 24), -1,
                "paged_flash_decode: %d sequences of %d heads and up to %lld slots are too many for one call", kv.n_seqs,
                n_head, (long long)capacity);
  const Workspace w = workspace_of(kv.n_seqs, n_head, kv.Hkv, kv.hd, capacity, mass != nullptr);
  AXM_CHECK_ARG(workspace_bytes >= w.bytes && (w.bytes == 0 || (workspace && (uintptr_t)workspace % 16 == 0)), -1,
                "paged_flash_decode: workspace of %zu bytes needed (16-byte aligned), %zu given", w.bytes,
                workspace_bytes);
  const hipStream_t s = (hipStream_t)stream;
  uint8_t* ws = (uint8_t*)workspace;
  const bool parts = per > kPairBlocks;
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
  p.grid = parts ? decode_grid(blocks, per_cu(kv.kv_dtype, kv.hd)) : kv.n_seqs * kv.Hkv * p.chunks;
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
  // One wave a row where a pair has few parts (about grid / pairs, one more), four where it has many (us, one / four:
  // 128 INT4 sequences 25.2 / 27.9, 48 fp16 ones 49.8 / 50.3; 8 INT4 ones of 4000 keys 15.4 / 11.7, one FP8 one of 8000
  // 23.2 / 15.3).
  const bool many = parts && (int64_t)p.grid > 4 * (int64_t)kv.n_seqs * kv.Hkv * p.chunks;
  const int rows = kv.n_seqs * n_head, join = !parts ? 0 : many ? rows : (rows + kWaves - 1) / kWaves;
  const int account = mass ? kv.n_seqs * kv.Hkv * slices : 0;
  if (join + account) {
    const dim3 grid(join + account), block(kThreads);
    if (kv.hd == 128 && many) hipLaunchKernelGGL((paged_join_kernel<128, 4>), grid, block, 0, s, p, join, slices);
    else if (kv.hd == 128) hipLaunchKernelGGL((paged_join_kernel<128, 1>), grid, block, 0, s, p, join, slices);
    else if (many) hipLaunchKernelGGL((paged_join_kernel<64, 4>), grid, block, 0, s, p, join, slices);
    else hipLaunchKernelGGL((paged_join_kernel<64, 1>), grid, block, 0, s, p, join, slices);
    AXM_LAUNCH_CHECK("paged_flash_decode (join)");
  }
  return 0;
}
