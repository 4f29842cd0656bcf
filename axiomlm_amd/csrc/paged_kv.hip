// Paged KV cache: RoPE and store of new tokens, and eviction by accumulated attention weight.
#include "paged_kv.h"

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
// RoPE + store.  One wave per (token, head row of [q | k | v]); lane l holds the EPL = hd / 64 elements from EPL l on
// (hd 128: one rotation pair; hd 64: half of one, the other half a lane away).  fp32 products and sums, one rounding
// to fp16 (rope_out), then for quantized pages one scale per 64 elements: fp16(amax / 448 | 7) and codes of
// fp16(x / scale).
// ---------------------------------------------------------------------------
constexpr int kWriteWaves = 4;

template <int EPL>
using hvec = _Float16 __attribute__((ext_vector_type(EPL)));

template <int EPL>
__device__ __forceinline__ void store_row(const PagedKv& kv, bool is_v, int page, int h, int slot, int lane,
                                          hvec<EPL> x) {
  constexpr int LPG = 64 / EPL;  // lanes per group of 64
  uint8_t* codes = (is_v ? kv.v : kv.k) + paged_row(kv, page, h, slot, paged_row_bytes(kv.kv_dtype, kv.hd));
  if (kv.kv_dtype == AXM_KV_FP16) {
    *reinterpret_cast<hvec<EPL>*>(codes + 2 * EPL * lane) = x;
    return;
  }
  float amax = fabsf(h2f(x[0]));
#pragma unroll
  for (int e = 1; e < EPL; ++e) amax = fmaxf(amax, fabsf(h2f(x[e])));
#pragma unroll
  for (int off = LPG / 2; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
  const bool fp8 = kv.kv_dtype == AXM_KV_FP8;
  const f16 sc = f2h(__fdiv_rn(amax, fp8 ? 448.f : 7.f));
  if (lane % LPG == 0)
    reinterpret_cast<f16*>((is_v ? kv.vs : kv.ks) + paged_scale_row(kv, page, h, slot))[lane / LPG] = sc;
  const float most = fp8 ? 448.f : 8.f;
  float c[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) {
    const float xf = h2f(x[e]);
    c[e] = h2f(sc) == 0.f && xf == xf ? 0.f : h2f(f2h(__fdiv_rn(xf, h2f(sc))));
    if (c[e] == c[e]) c[e] = fminf(fmaxf(c[e], -most), fp8 ? most : 7.f);  // NaN stays
  }
  if (fp8) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < EPL; ++e) w |= (uint32_t)fp8e4m3fn_from_f32(c[e]) << (8 * e);
    if (EPL == 1) codes[lane] = (uint8_t)w;
    else *reinterpret_cast<uint16_t*>(codes + 2 * lane) = (uint16_t)w;
    return;
  }
  int n[EPL];
#pragma unroll
  for (int e = 0; e < EPL; ++e) n[e] = c[e] == c[e] ? (int)__builtin_rintf(c[e]) & 15 : 0;
  if (EPL == 1) {
    const int next = __shfl_xor(n[0], 1, 64);
    if ((lane & 1) == 0) codes[lane / 2] = (uint8_t)(n[0] | next << 4);
  } else {
    codes[lane] = (uint8_t)(n[0] | n[EPL - 1] << 4);
  }
}

template <int EPL>
__global__ void __launch_bounds__(kWriteWaves * 64)
    paged_write_kernel(f16* __restrict__ qkv, int64_t ld, int T, const float* __restrict__ freqs, int rope_len,
                       const int* __restrict__ positions, const int* __restrict__ slots,
                       const int* __restrict__ seq_ids, const f16* __restrict__ bias, PagedKv kv, int Hq) {
  constexpr int HD = 64 * EPL;
  const int lane = threadIdx.x & 63;
  const int rows = Hq + 2 * kv.Hkv;
  const int64_t item = (int64_t)blockIdx.x * kWriteWaves + (threadIdx.x >> 6);
  if (item >= (int64_t)T * rows) return;
  const int t = (int)(item / rows), r = (int)(item % rows);
  const int pos = positions[t];
  const int slot = slots ? slots[t] : pos;
  const int b = seq_ids ? seq_ids[t] : t;
  if (slot < 0 || (unsigned)b >= (unsigned)kv.n_seqs) return;
  const int page = paged_page(kv, b, slot);
  if (page < 0) return;
  f16* row = qkv + t * ld + (int64_t)r * HD;
  hvec<EPL> x = *reinterpret_cast<const hvec<EPL>*>(row + EPL * lane);
  if (bias != nullptr) {
#pragma unroll
    for (int e = 0; e < EPL; ++e) x[e] = hadd(x[e], bias[r * HD + EPL * lane + e]);
  }
  if (r < Hq + kv.Hkv) {
    int p = pos % rope_len;
    if (p < 0) p += rope_len;
    const float* f = freqs + ((int64_t)p * (HD / 2) + EPL * lane / 2) * 2;
    if (EPL == 2) {
      const f16 a = x[0], c = x[EPL - 1];
      x[0] = rope_out(a, c, f[0], f[1], true);
      x[EPL - 1] = rope_out(a, c, f[0], f[1], false);
    } else {
      const f16 other = u16_as_h((uint16_t)__shfl_xor((int)h_as_u16(x[0]), 1, 64));
      x[0] = (lane & 1) == 0 ? rope_out(x[0], other, f[0], f[1], true) : rope_out(other, x[0], f[0], f[1], false);
    }
  }
  if (r < Hq) {
    *reinterpret_cast<hvec<EPL>*>(row + EPL * lane) = x;
    return;
  }
  const bool is_v = r >= Hq + kv.Hkv;
  store_row<EPL>(kv, is_v, page, r - Hq - (is_v ? kv.Hkv : 0), slot, lane, x);
}

// ---------------------------------------------------------------------------
// Eviction.  Select: one workgroup per (layer, sequence, KV head) finds the value that the (budget - recent)-th
// largest account before the recent slots has, by bisection over the ordered bits, then writes the kept slots in order
// with one prefix count.  Move: one workgroup per (layer, k | v, sequence, KV head) copies the kept rows down in
// ascending tiles: a row never moves up, so every row a later tile reads lies behind the tile being written.
// ---------------------------------------------------------------------------
constexpr int kEvictThreads = 256;

// Order of accounts: larger is kept first; -0 counts as 0, NaN as less than every number.
__device__ __forceinline__ uint32_t account_key(float a) {
  if (a != a) return 0u;
  const uint32_t u = __builtin_bit_cast(uint32_t, a + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int block_sum(int v, int* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  int s = 0;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) s += lds[w];
  return s;
}

__global__ void __launch_bounds__(kEvictThreads)
    evict_select_kernel(const int* __restrict__ lens, int max_len, const float* __restrict__ mass, int64_t mass_len,
                        int n_seqs, int Hkv, int budget, int recent, float* __restrict__ mass_out,
                        int* __restrict__ kept, int* __restrict__ lens_out) {
  __shared__ int red[kEvictThreads / 64];
  __shared__ int scan[kEvictThreads];
  const int64_t row = blockIdx.x;
  const int b = (int)(row / Hkv % n_seqs);
  const int n = min(max(lens[b], 0), max_len);
  const float* a = mass + row * mass_len;
  float* out = mass_out + row * mass_len;
  int* k = kept + row * budget;
  const int left = min(n, budget);
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
  // Largest t with at least `want` keys >= t (want >= 1), found bit by bit.
  uint32_t cut = 0;
  if (want > 0) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = cut | (1u << bit);
      int c = 0;
      for (int i = threadIdx.x; i < old; i += kEvictThreads) c += account_key(a[i]) >= t;
      if (block_sum(c, red) >= want) cut = t;
    }
  }
  int above = 0;
  for (int i = threadIdx.x; i < old; i += kEvictThreads) above += account_key(a[i]) > cut;
  above = block_sum(above, red);
  int ties = want - above;  // of the slots whose account equals the cut, the lowest ones
  int at = 0;
  for (int base = 0; base < old && want > 0; base += kEvictThreads) {
    const int i = base + threadIdx.x;
    const uint32_t key = i < old ? account_key(a[i]) : 0u;
    const bool over = i < old && key > cut, equal = i < old && key == cut;
    // Counts of both in one word: equal in the low half, over in the high half.
    scan[threadIdx.x] = (over ? 1 << 16 : 0) | (equal ? 1 : 0);
    __syncthreads();
    for (int o = 1; o < kEvictThreads; o <<= 1) {
      const int add = (int)threadIdx.x >= o ? scan[threadIdx.x - o] : 0;
      __syncthreads();
      scan[threadIdx.x] += add;
      __syncthreads();
    }
    const int incl = scan[threadIdx.x], all = scan[kEvictThreads - 1];
    const int eq_before = (incl & 0xFFFF) - (equal ? 1 : 0), over_before = (incl >> 16) - (over ? 1 : 0);
    if (over || (equal && eq_before < ties)) {
      const int to = at + over_before + min(eq_before, ties);
      k[to] = i;
      out[to] = a[i];
    }
    at += (all >> 16) + min(all & 0xFFFF, ties);
    ties -= min(all & 0xFFFF, ties);
    __syncthreads();
  }
  for (int i = threadIdx.x; i < recent; i += kEvictThreads) {
    k[want + i] = old + i;
    out[want + i] = a[old + i];
  }
}

__global__ void __launch_bounds__(kEvictThreads)
    evict_move_kernel(PagedKv kv, int64_t layer_stride, int64_t scale_layer_stride, const int* __restrict__ lens,
                      const int* __restrict__ kept, int budget) {
  __shared__ __align__(16) uint8_t tile[64 * 256];
  __shared__ uint32_t tile_sc[64];
  int idx = blockIdx.x;
  const int h = idx % kv.Hkv;
  idx /= kv.Hkv;
  const int b = idx % kv.n_seqs;
  idx /= kv.n_seqs;
  const bool is_v = idx & 1;
  const int l = idx >> 1;
  const int n = lens[b];
  if (n <= budget) return;
  const int rb = paged_row_bytes(kv.kv_dtype, kv.hd), vpr = rb / 16;  // 16-byte vectors per row
  uint8_t* base = (is_v ? kv.v : kv.k) + l * layer_stride;
  uint8_t* sbase = (is_v ? kv.vs : kv.ks) + l * scale_layer_stride;
  const bool quant = kv.kv_dtype != AXM_KV_FP16;
  const int* k = kept + (((int64_t)l * kv.n_seqs + b) * kv.Hkv + h) * budget;
  for (int t0 = 0; t0 < budget; t0 += 64) {
    const int rows = min(64, budget - t0);
    for (int i = threadIdx.x; i < rows * vpr; i += kEvictThreads) {
      const int slot = k[t0 + i / vpr];
      const int page = paged_page(kv, b, slot);
      if (page >= 0)
        reinterpret_cast<u32x4*>(tile)[i] =
            *reinterpret_cast<const u32x4*>(base + paged_row(kv, page, h, slot, rb) + i % vpr * 16);
    }
    if (quant && (int)threadIdx.x < rows) {
      const int slot = k[t0 + threadIdx.x];
      const int page = paged_page(kv, b, slot);
      if (page >= 0) {
        const uint8_t* s = sbase + paged_scale_row(kv, page, h, slot);
        tile_sc[threadIdx.x] = kv.hd == 128 ? *reinterpret_cast<const uint32_t*>(s) : *reinterpret_cast<const uint16_t*>(s);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * vpr; i += kEvictThreads) {
      const int slot = t0 + i / vpr;
      const int page = paged_page(kv, b, slot);
      if (page >= 0 && paged_page(kv, b, k[slot]) >= 0)
        *reinterpret_cast<u32x4*>(base + paged_row(kv, page, h, slot, rb) + i % vpr * 16) =
            reinterpret_cast<const u32x4*>(tile)[i];
    }
    if (quant && (int)threadIdx.x < rows) {
      const int slot = t0 + threadIdx.x;
      const int page = paged_page(kv, b, slot);
      if (page >= 0 && paged_page(kv, b, k[slot]) >= 0) {
        uint8_t* s = sbase + paged_scale_row(kv, page, h, slot);
        if (kv.hd == 128) *reinterpret_cast<uint32_t*>(s) = tile_sc[threadIdx.x];
        else *reinterpret_cast<uint16_t*>(s) = (uint16_t)tile_sc[threadIdx.x];
      }
    }
    __syncthreads();
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
  const int rows = q_dim / kv.hd + 2 * kv.Hkv;
  AXM_CHECK_ARG(ld_qkv >= (int64_t)rows * kv.hd && ld_qkv % 2 == 0 && (uintptr_t)qkv % 4 == 0, -1,
                "rope_paged_kv_write: rows of %d halves %lld apart (4-byte aligned)", rows * kv.hd, (long long)ld_qkv);
  const int64_t items = (int64_t)T * rows;
  AXM_CHECK_ARG(items < (1ll << 26), -1, "rope_paged_kv_write: %d tokens of %d heads are too many for one call", T, rows);
  const dim3 grid((unsigned)((items + kWriteWaves - 1) / kWriteWaves));
  if (kv.hd == 128)
    hipLaunchKernelGGL((paged_write_kernel<2>), grid, dim3(kWriteWaves * 64), 0, (hipStream_t)stream, (f16*)qkv, ld_qkv,
                       T, (const float*)freqs, rope_len, positions, slots, seq_ids, (const f16*)qkv_bias, kv,
                       q_dim / kv.hd);
  else
    hipLaunchKernelGGL((paged_write_kernel<1>), grid, dim3(kWriteWaves * 64), 0, (hipStream_t)stream, (f16*)qkv, ld_qkv,
                       T, (const float*)freqs, rope_len, positions, slots, seq_ids, (const f16*)qkv_bias, kv,
                       q_dim / kv.hd);
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
    hipLaunchKernelGGL(evict_move_kernel, dim3((unsigned)(2 * heads)), dim3(kEvictThreads), 0, (hipStream_t)stream, kv,
                       layer_stride, scale_layer_stride, seq_lens, kept, budget);
    AXM_LAUNCH_CHECK("evict_paged_kv (move)");
  }
  return 0;
}
