// Paged KV cache: RoPE and store of new tokens, and eviction by accumulated attention weight.
#include "paged_kv.h"

#include <type_traits>

int paged_view(const axm_paged_kv* d, const char* who, PagedKv* out) {
  AXM_CHECK_ARG(d && d->k && d->v && d->block_table, -1, "%s: null cache or table pointer", who);
  AXM_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, -1, "%s: head_dim=%d must be 64 or 128", who, d->head_dim);
  AXM_CHECK_ARG(d->kv_dtype >= 0 && d->kv_dtype <= 2, -1, "%s: bad kv dtype %d", who, d->kv_dtype);
  const bool quant = d->kv_dtype != AXM_KV_FP16;
  AXM_CHECK_ARG(!quant || (d->k_scales && d->v_scales), -1, "%s: quantized cache needs scales", who);
  AXM_CHECK_ARG(d->page_size >= 16 && d->page_size <= 1024 && (d->page_size & (d->page_size - 1)) == 0, -1,
                "%s: page_size=%d must be a power of two between 16 and 1024", who, d->page_size);
  AXM_CHECK_ARG(d->n_kv_head >= 1 && d->n_kv_head <= 1024 && d->n_pages >= 1 && d->n_seqs >= 1 && d->max_pages >= 1, -1,
                "%s: bad cache shape (%d KV heads, %d pages, %d sequences of %d pages)", who, d->n_kv_head, d->n_pages,
                d->n_seqs, d->max_pages);
  AXM_CHECK_ARG((int64_t)d->max_pages * d->page_size < (1ll << 30), -1, "%s: sequences of %d pages of %d are too long",
                who, d->max_pages, d->page_size);
  const int64_t rows = (int64_t)d->n_kv_head * d->page_size;
  AXM_CHECK_ARG(d->page_stride >= rows * paged_row_bytes(d->kv_dtype, d->head_dim) && d->page_stride % 16 == 0, -1,
                "%s: pages %lld bytes apart (dense pages of this shape take %lld; multiples of 16)", who,
                (long long)d->page_stride, (long long)(rows * paged_row_bytes(d->kv_dtype, d->head_dim)));
  AXM_CHECK_ARG(((uintptr_t)d->k | (uintptr_t)d->v) % 16 == 0, -1, "%s: k and v must be 16-byte aligned", who);
  if (quant) {
    AXM_CHECK_ARG(d->scale_stride >= rows * (d->head_dim / 64) * 2 && d->scale_stride % 4 == 0, -1,
                  "%s: scale pages %lld bytes apart", who, (long long)d->scale_stride);
    AXM_CHECK_ARG(((uintptr_t)d->k_scales | (uintptr_t)d->v_scales) % 4 == 0, -1, "%s: scales must be 4-byte aligned",
                  who);
  }
  int shift = 0;
  while ((1 << shift) < d->page_size) ++shift;
  *out = PagedKv{(uint8_t*)d->k, (uint8_t*)d->v, (uint8_t*)d->k_scales, (uint8_t*)d->v_scales, d->block_table,
                 d->page_stride, d->scale_stride, d->kv_dtype, d->n_kv_head, d->head_dim, shift, d->n_pages, d->n_seqs,
                 d->max_pages};
  return 0;
}

namespace {

// ---------------------------------------------------------------------------
// RoPE + store.  A lane holds 8 elements (four rotation pairs) of a head row of [q | k | v], hd / 8 lanes a row, a wave
// 64 / (hd / 8) rows of one token.  fp32 products and sums, one rounding to fp16 (rope_out), then for quantized pages
// one scale per 64 elements (8 lanes): fp16(amax / 448 | 7) and codes of fp16(x / scale).  Bound by the rows' bytes; with
// 4 bytes a lane and a row a wave it took 57.8 us for 4001 tokens of 48 rows into FP8 pages instead of 22.8 (4.1 TB/s).
// ---------------------------------------------------------------------------
constexpr int kWriteWaves = 4;

template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
  return fmaxf(v, dpp_move<CTRL>(v));
}

// VEC: rows, bias and rotations are 16-byte aligned (else 4-byte loads and stores of the rows).
template <int HD, int KVT, bool VEC>
__global__ void __launch_bounds__(kWriteWaves * 64)
    paged_write_kernel(f16* __restrict__ qkv, int64_t ld, uint32_t items, uint32_t groups, const float* __restrict__ freqs,
                       int rope_len, const int* __restrict__ positions, const int* __restrict__ slots,
                       const int* __restrict__ seq_ids, const f16* __restrict__ bias, PagedKv kv, int Hq) {
  constexpr int LPR = HD / 8, RPW = 64 / LPR;  // lanes of a row, rows of a wave
  const int lane = threadIdx.x & 63;
  const uint32_t item = (uint32_t)__builtin_amdgcn_readfirstlane(blockIdx.x * kWriteWaves + (threadIdx.x >> 6));
  if (item >= items) return;
  const uint32_t t = item / groups;
  const int r = (int)(item - t * groups) * RPW + lane / LPR, e = lane % LPR * 8;
  const int pos = positions[t], slot = slots ? slots[t] : pos, b = seq_ids ? seq_ids[t] : (int)t;
  if (slot < 0 || (unsigned)b >= (unsigned)kv.n_seqs) return;
  const int page = paged_page(kv, b, slot);
  if (page < 0 || r >= Hq + 2 * kv.Hkv) return;
  f16* at = qkv + t * ld + (int64_t)r * HD + e;
  f16x8 x, add;
  auto load8 = [&](const f16* p) {
    if (VEC) return *reinterpret_cast<const f16x8*>(p);
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    return __builtin_bit_cast(f16x8, w);
  };
  x = load8(at);
  if (bias != nullptr) {
    if (VEC) add = load8(bias + r * HD + e);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) add[i] = bias[r * HD + e + i];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = hadd(x[i], add[i]);
  }
  if (r < Hq + kv.Hkv) {
    int p = pos % rope_len;
    if (p < 0) p += rope_len;
    const float* f = freqs + ((int64_t)p * HD + e);
    float cs[8];
    if (VEC) {
      *reinterpret_cast<f32x4*>(cs) = reinterpret_cast<const f32x4*>(f)[0];
      *reinterpret_cast<f32x4*>(cs + 4) = reinterpret_cast<const f32x4*>(f)[1];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) cs[i] = f[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const f16 a = x[i], c = x[i + 1];
      x[i] = rope_out(a, c, cs[i], cs[i + 1], true);
      x[i + 1] = rope_out(a, c, cs[i], cs[i + 1], false);
    }
  }
  if (r < Hq) {
    if (VEC) *reinterpret_cast<f16x8*>(at) = x;
    else
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(at)[i] = __builtin_bit_cast(u32x4, x)[i];
    return;
  }
  const bool is_v = r >= Hq + kv.Hkv;
  const int h = r - Hq - (is_v ? kv.Hkv : 0);
  uint8_t* codes = (is_v ? kv.v : kv.k) + paged_row(kv, page, h, slot, paged_row_bytes(KVT, HD));
  if (KVT == AXM_KV_FP16) {
    *reinterpret_cast<f16x8*>(codes + 2 * e) = x;
    return;
  }
  float amax = fabsf(h2f(x[0]));
#pragma unroll
  for (int i = 1; i < 8; ++i) amax = fmaxf(amax, fabsf(h2f(x[i])));
  amax = dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(amax)));  // over the 8 lanes of the group
  constexpr bool kFp8 = KVT == AXM_KV_FP8;
  const f16 sc = f2h(__fdiv_rn(amax, kFp8 ? 448.f : 7.f));
  if (e % 64 == 0)
    reinterpret_cast<f16*>((is_v ? kv.vs : kv.ks) + paged_scale_row(kv, page, h, slot))[e / 64] = sc;
  float c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = h2f(x[i]);
    c[i] = h2f(sc) == 0.f && v == v ? 0.f : h2f(f2h(__fdiv_rn(v, h2f(sc))));
    if (c[i] == c[i]) c[i] = fminf(fmaxf(c[i], kFp8 ? -448.f : -8.f), kFp8 ? 448.f : 7.f);  // NaN stays
  }
  if (kFp8) {
    u32x2 w = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i / 4] |= (uint32_t)fp8e4m3fn_from_f32(c[i]) << (8 * (i & 3));
    *reinterpret_cast<u32x2*>(codes + e) = w;
  } else {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (c[i] == c[i] ? (uint32_t)(int)__builtin_rintf(c[i]) & 15u : 0u) << (4 * i);
    *reinterpret_cast<uint32_t*>(codes + e / 2) = w;
  }
}

template <int HD, int KVT>
void launch_write(bool vec, unsigned grid, hipStream_t s, f16* qkv, int64_t ld, uint32_t items, uint32_t groups,
                  const float* freqs, int rope_len, const int* positions, const int* slots, const int* seq_ids,
                  const f16* bias, const PagedKv& kv, int Hq) {
  const dim3 block(kWriteWaves * 64);
  if (vec)
    hipLaunchKernelGGL((paged_write_kernel<HD, KVT, true>), dim3(grid), block, 0, s, qkv, ld, items, groups, freqs,
                       rope_len, positions, slots, seq_ids, bias, kv, Hq);
  else
    hipLaunchKernelGGL((paged_write_kernel<HD, KVT, false>), dim3(grid), block, 0, s, qkv, ld, items, groups, freqs,
                       rope_len, positions, slots, seq_ids, bias, kv, Hq);
}

// ---------------------------------------------------------------------------
// Eviction.  Select: one workgroup per (layer, sequence, KV head).  The value that the (budget - recent)-th largest account
// before the recent slots has comes from histograms of its ordered bits (11, 11 and 10; 1024 heads of up to 4096 slots:
// 27 us, mostly the histograms' atomics; 13 bits at first, or counting two bits a step over keys in registers, took
// longer); then every wave counts and writes the kept slots of its own stretch in order.  Move: one workgroup per
// (layer, k | v, sequence, KV head) copies the kept rows down in ascending tiles.  A row never moves up, so what a later
// tile reads lies behind the tile being written: a tile's loads are under way while the one before is stored.  Bound by
// the rows' bytes: 150 us for the same heads cut to 1024 rows of 256 bytes (4.0 TB/s).
// ---------------------------------------------------------------------------
constexpr int kEvictThreads = 256;
constexpr int kEvictWaves = kEvictThreads / 64;
constexpr int kBinBits = 11, kBinsEach = (1 << kBinBits) / kEvictThreads;

// Order of accounts: larger is kept first; -0 counts as 0, NaN as less than every number.
__device__ __forceinline__ uint32_t account_key(float a) {
  if (a != a) return 0u;
  const uint32_t u = __builtin_bit_cast(uint32_t, a + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kEvictThreads)
    evict_select_kernel(const int* __restrict__ lens, int max_len, const float* __restrict__ mass, int64_t mass_len,
                        int n_seqs, int Hkv, int budget, int recent, float* __restrict__ mass_out,
                        int* __restrict__ kept, int* __restrict__ lens_out) {
  constexpr int kHeld = 16;  // keys a lane keeps in registers (4096 slots); the rest is read again
  __shared__ __align__(16) uint32_t bins[kBinsEach * kEvictThreads];
  __shared__ int wave_sum_s[kEvictWaves], found_bin, found_before, found_count;
  __shared__ int wave_over[kEvictWaves], wave_equal[kEvictWaves];
  const int64_t row = blockIdx.x;
  const int b = (int)(row / Hkv % n_seqs);
  const int n = min(max(lens[b], 0), max_len);
  const float* a = mass + row * mass_len;
  float* out = mass_out + row * mass_len;
  int* k = kept + row * budget;
  const int left = min(n, budget), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (row < (int64_t)n_seqs * Hkv && row % Hkv == 0 && threadIdx.x == 0) lens_out[b] = left;
  for (int64_t i = left + threadIdx.x; i < mass_len; i += kEvictThreads) out[i] = 0.f;
  for (int i = left + threadIdx.x; i < budget; i += kEvictThreads) k[i] = -1;
  if (n <= budget) {
    for (int i = threadIdx.x; i < n; i += kEvictThreads) {
      out[i] = a[i];
      k[i] = i;
    }
    return;
  }
  const int old = n - recent;  // slots that compete
  const int want = budget - recent;
  for (int i = threadIdx.x; i < recent; i += kEvictThreads) {
    k[want + i] = old + i;
    out[want + i] = a[old + i];
  }
  if (want == 0) return;
  // A wave's stretch: contiguous, a multiple of 64 slots.
  const int each = ((old + kEvictWaves - 1) / kEvictWaves + 63) / 64 * 64;
  const int begin = min(wave * each, old), end = min(begin + each, old);
  uint32_t held[kHeld];
#pragma unroll
  for (int c = 0; c < kHeld; ++c) {
    const int i = begin + c * 64 + lane;
    held[c] = i < end ? account_key(a[i]) : 0u;
  }
  auto pass = [&](auto f) {  // f(slot, key, whether there is one): all lanes of the wave
#pragma unroll
    for (int c = 0; c < kHeld; ++c)
      if (begin + c * 64 < end) f(begin + c * 64 + lane, held[c], begin + c * 64 + lane < end);
    for (int at = begin + kHeld * 64; at < end; at += 64) {
      const int i = at + lane;
      f(i, i < end ? account_key(a[i]) : 0u, i < end);
    }
  };
  uint32_t cut = 0, mask = 0;  // bits of the cut that are known
  int need = want;             // keys still to take among those that share them
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 32 - kBinBits : level == 1 ? 32 - 2 * kBinBits : 0;
    const uint32_t digit = level == 2 ? (1u << (32 - 2 * kBinBits)) - 1 : (1u << kBinBits) - 1;
    u32x4* all = reinterpret_cast<u32x4*>(bins);
#pragma unroll
    for (int i = 0; i < kBinsEach / 4; ++i) all[i * kEvictThreads + threadIdx.x] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    pass([&](int, uint32_t key, bool in) {
      if (in && (key & mask) == cut) atomicAdd(&bins[(key >> shift) & digit], 1u);
    });
    __syncthreads();
    // From the largest bin down: thread t has kBinsEach of them.
    const int first = kEvictThreads - 1 - threadIdx.x;
    u32x4 c[kBinsEach / 4];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kBinsEach / 4; ++i) {
      c[i] = all[first * (kBinsEach / 4) + i];
      mine += (int)(c[i].x + c[i].y + c[i].z + c[i].w);
    }
    int x = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      x += lane >= o ? y : 0;
    }
    if (lane == 63) wave_sum_s[wave] = x;
    __syncthreads();
    int before = x - mine;
#pragma unroll
    for (int w = 0; w < kEvictWaves; ++w) before += w < wave ? wave_sum_s[w] : 0;
    if (before < need && before + mine >= need) {
      int bin = -1, count = 0;
#pragma unroll
      for (int i = kBinsEach - 1; i >= 0; --i)
        if (bin < 0) {
          count = (int)c[i / 4][i & 3];
          if (before + count >= need) bin = kBinsEach * first + i;
          else before += count;
        }
      found_bin = bin;
      found_before = before;
      found_count = count;
    }
    __syncthreads();
    cut |= (uint32_t)found_bin << shift;
    mask |= digit << shift;
    need -= found_before;
    if (found_count == need && cut != 0) {  // all that share these bits stay: everything over the key below them
      --cut;
      need = 0;
      break;
    }
  }
  // `need` of the keys equal to the cut stay, the lowest slots first.
  int over = 0, equal = 0;
  pass([&](int, uint32_t key, bool in) {
    over += __builtin_popcountll(__builtin_amdgcn_ballot_w64(in && key > cut));
    equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(in && key == cut));
  });
  if (lane == 0) {
    wave_over[wave] = over;
    wave_equal[wave] = equal;
  }
  __syncthreads();
  int to = 0, ties = need;  // rows written before this stretch, ties left for it
  for (int w = 0; w < wave; ++w) {
    const int take = min(wave_equal[w], ties);
    to += wave_over[w] + take;
    ties -= take;
  }
  pass([&](int i, uint32_t key, bool in) {
    const uint64_t o = __builtin_amdgcn_ballot_w64(in && key > cut), q = __builtin_amdgcn_ballot_w64(in && key == cut);
    const uint64_t below = (1ull << lane) - 1;
    const int eq = __builtin_popcountll(q & below);
    if ((o >> lane & 1) || ((q >> lane & 1) && eq < ties)) {
      const int at = to + __builtin_popcountll(o & below) + min(eq, ties);
      k[at] = i;
      out[at] = a[i];
    }
    const int take = min((int)__builtin_popcountll(q), ties);
    to += __builtin_popcountll(o) + take;
    ties -= take;
  });
}

// VPR: 16-byte vectors of a row; a tile is 64 rows, kEach vectors a thread.
template <int VPR, bool QUANT, int SCALE>
__global__ void __launch_bounds__(kEvictThreads)
    evict_move_kernel(PagedKv kv, int64_t layer_stride, int64_t scale_layer_stride, const int* __restrict__ lens,
                      const int* __restrict__ kept, int budget) {
  constexpr int kTile = 64, kEach = kTile * VPR / kEvictThreads > 0 ? kTile * VPR / kEvictThreads : 1;
  constexpr int kAtOnce = 1024;  // rows whose places are looked up together
  constexpr int kBytes = VPR * 16;
  __shared__ int64_t from[kAtOnce], into[kAtOnce];  // page << 32 | row in the page; -1: stays
  int idx = blockIdx.x;
  const int h = idx % kv.Hkv;
  idx /= kv.Hkv;
  const int b = idx % kv.n_seqs;
  idx /= kv.n_seqs;
  const bool is_v = idx & 1;
  const int l = idx >> 1;
  if (lens[b] <= budget) return;
  uint8_t* base = (is_v ? kv.v : kv.k) + l * layer_stride;
  uint8_t* sbase = QUANT ? (is_v ? kv.vs : kv.ks) + l * scale_layer_stride : nullptr;
  const int* k = kept + (((int64_t)l * kv.n_seqs + b) * kv.Hkv + h) * budget;
  const int in_page = (1 << kv.page_shift) - 1;
  auto place = [&](int slot) {
    const int page = paged_page(kv, b, slot);
    return page < 0 ? (int64_t)-1 : (int64_t)page << 32 | (uint32_t)((h << kv.page_shift) + (slot & in_page));
  };
  auto row_at = [&](int64_t at) { return base + (at >> 32) * kv.page_stride + (int64_t)(uint32_t)at * kBytes; };
  auto scale_at = [&](int64_t at) { return sbase + (at >> 32) * kv.scale_stride + (int64_t)(uint32_t)at * SCALE; };
  for (int t0 = 0; t0 < budget; t0 += kAtOnce) {
    const int rows = min(kAtOnce, budget - t0);
    __syncthreads();
    for (int i = threadIdx.x; i < kAtOnce; i += kEvictThreads) {
      int64_t f = -1, t = -1;
      if (i < rows) {
        const int slot = k[t0 + i];
        if (slot != t0 + i) {
          f = place(slot);
          t = place(t0 + i);
        }
      }
      from[i] = t < 0 ? -1 : f;
      into[i] = t;
    }
    __syncthreads();
    u32x4 cur[kEach], next[kEach];
    uint32_t cur_s = 0, next_s = 0;
    auto load = [&](int tile, u32x4 (&x)[kEach], uint32_t& sc) {
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int i = threadIdx.x + j * kEvictThreads, r = tile * kTile + i / VPR;
        if (i < kTile * VPR && r < kAtOnce && from[r] >= 0)
          x[j] = *reinterpret_cast<const u32x4*>(row_at(from[r]) + i % VPR * 16);
      }
      if (QUANT && threadIdx.x < kTile) {
        const int r = tile * kTile + threadIdx.x;
        if (r < kAtOnce && from[r] >= 0)
          sc = SCALE == 4 ? *reinterpret_cast<const uint32_t*>(scale_at(from[r]))
                          : *reinterpret_cast<const uint16_t*>(scale_at(from[r]));
      }
    };
    const int tiles = (rows + kTile - 1) / kTile;
    load(0, cur, cur_s);
#pragma unroll 1
    for (int tile = 0; tile < tiles; ++tile) {
      load(tile + 1, next, next_s);  // (rows past the last are marked as staying)
      // The tile's own loads have arrived in every wave before any of its rows is overwritten.
#pragma unroll
      for (int j = 0; j < kEach; ++j) asm volatile("" : "+v"(cur[j]));
      asm volatile("" : "+v"(cur_s));
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int i = threadIdx.x + j * kEvictThreads, r = tile * kTile + i / VPR;
        if (i < kTile * VPR && from[r] >= 0) *reinterpret_cast<u32x4*>(row_at(into[r]) + i % VPR * 16) = cur[j];
        cur[j] = next[j];
      }
      if (QUANT && threadIdx.x < kTile) {
        const int r = tile * kTile + threadIdx.x;
        if (from[r] >= 0) {
          if (SCALE == 4) *reinterpret_cast<uint32_t*>(scale_at(into[r])) = cur_s;
          else *reinterpret_cast<uint16_t*>(scale_at(into[r])) = (uint16_t)cur_s;
        }
      }
      cur_s = next_s;
    }
  }
}

}  // namespace

extern "C" int axm_rope_paged_kv_write(void* qkv, int64_t ld_qkv, int T, const void* freqs, int rope_len,
                                       const int* positions, const int* slots, const int* seq_ids,
                                       const void* qkv_bias, const axm_paged_kv* d, int q_dim, void* stream) {
  PagedKv kv;
  if (int rc = paged_view(d, "rope_paged_kv_write", &kv)) return rc;
  AXM_CHECK_ARG(qkv && freqs && positions, -1, "rope_paged_kv_write: null pointer");
  AXM_CHECK_ARG(T >= 1 && T <= (1 << 20) && rope_len >= 1, -1, "rope_paged_kv_write: T=%d, rope_len=%d", T, rope_len);
  AXM_CHECK_ARG(q_dim >= kv.hd && q_dim <= (1 << 20) && q_dim % kv.hd == 0, -1,
                "rope_paged_kv_write: q_dim=%d is no multiple of head_dim=%d", q_dim, kv.hd);
  const int rows = q_dim / kv.hd + 2 * kv.Hkv, rows_per_wave = 512 / kv.hd;
  AXM_CHECK_ARG(ld_qkv >= (int64_t)rows * kv.hd && ld_qkv % 2 == 0 && (uintptr_t)qkv % 4 == 0, -1,
                "rope_paged_kv_write: rows of %d halves %lld apart (4-byte aligned)", rows * kv.hd, (long long)ld_qkv);
  const int64_t groups = (rows + rows_per_wave - 1) / rows_per_wave, items = T * groups;
  AXM_CHECK_ARG(items < (1ll << 26), -1, "rope_paged_kv_write: %d tokens of %d heads are too many for one call", T, rows);
  const bool vec = ((uintptr_t)qkv | (uintptr_t)qkv_bias | (uintptr_t)freqs) % 16 == 0 && ld_qkv % 8 == 0;
  const unsigned grid = (unsigned)((items + kWriteWaves - 1) / kWriteWaves);
  auto launch = [&](auto hd, auto kvt) {
    launch_write<decltype(hd)::value, decltype(kvt)::value>(
        vec, grid, (hipStream_t)stream, (f16*)qkv, ld_qkv, (uint32_t)items, (uint32_t)groups, (const float*)freqs, rope_len,
        positions, slots, seq_ids, (const f16*)qkv_bias, kv, q_dim / kv.hd);
  };
  auto launch_hd = [&](auto hd) {
    if (kv.kv_dtype == AXM_KV_FP16) launch(hd, std::integral_constant<int, AXM_KV_FP16>{});
    else if (kv.kv_dtype == AXM_KV_FP8) launch(hd, std::integral_constant<int, AXM_KV_FP8>{});
    else launch(hd, std::integral_constant<int, AXM_KV_INT4>{});
  };
  if (kv.hd == 128) launch_hd(std::integral_constant<int, 128>{});
  else launch_hd(std::integral_constant<int, 64>{});
  AXM_LAUNCH_CHECK("rope_paged_kv_write");
  return 0;
}

extern "C" int axm_evict_paged_kv(const axm_paged_kv* d, int n_layer, int64_t layer_stride, int64_t scale_layer_stride,
                                  const int* seq_lens, const float* mass, int64_t mass_len, int budget, int recent,
                                  float* mass_out, int* kept, int* lens_out, void* stream) {
  PagedKv kv;
  if (int rc = paged_view(d, "evict_paged_kv", &kv)) return rc;
  AXM_CHECK_ARG(seq_lens && mass && mass_out && kept && lens_out && mass != mass_out, -1,
                "evict_paged_kv: null pointer, or mass_out is mass");
  AXM_CHECK_ARG(d->k != d->v, -1, "evict_paged_kv: k and v are the same pages");
  AXM_CHECK_ARG(budget >= 1 && recent >= 0 && recent <= budget, -1, "evict_paged_kv: budget=%d, recent=%d", budget,
                recent);
  const int max_len = kv.max_pages << kv.page_shift;
  AXM_CHECK_ARG(mass_len >= max_len, -1, "evict_paged_kv: mass has %lld slots, the table %d", (long long)mass_len,
                max_len);
  const int64_t heads = (int64_t)n_layer * kv.n_seqs * kv.Hkv;
  AXM_CHECK_ARG(n_layer >= 1 && heads < (1 << 23), -1, "evict_paged_kv: %d layers of %d sequences", n_layer,
                kv.n_seqs);
  AXM_CHECK_ARG(n_layer == 1 || (layer_stride > 0 && layer_stride % 16 == 0 &&
                                 (kv.kv_dtype == AXM_KV_FP16 || (scale_layer_stride > 0 && scale_layer_stride % 4 == 0))),
                -1, "evict_paged_kv: layers %lld bytes apart", (long long)layer_stride);
  hipLaunchKernelGGL(evict_select_kernel, dim3((unsigned)heads), dim3(kEvictThreads), 0, (hipStream_t)stream, seq_lens,
                     max_len, mass, mass_len, kv.n_seqs, kv.Hkv, budget, recent, mass_out, kept, lens_out);
  AXM_LAUNCH_CHECK("evict_paged_kv (select)");
  if (budget < max_len) {
    const dim3 grid((unsigned)(2 * heads)), block(kEvictThreads);
    const hipStream_t st = (hipStream_t)stream;
    switch (kv.kv_dtype * 2 + (kv.hd == 128)) {
#define MOVE(VPR, QUANT, SCALE)                                                                                      \
  hipLaunchKernelGGL((evict_move_kernel<VPR, QUANT, SCALE>), grid, block, 0, st, kv, layer_stride, scale_layer_stride, \
                     seq_lens, kept, budget)
      case 0: MOVE(8, false, 2); break;
      case 1: MOVE(16, false, 4); break;
      case 2: MOVE(4, true, 2); break;
      case 3: MOVE(8, true, 4); break;
      case 4: MOVE(2, true, 2); break;
      default: MOVE(4, true, 4); break;
#undef MOVE
    }
    AXM_LAUNCH_CHECK("evict_paged_kv (move)");
  }
  return 0;
}
