// Decode attention of one new token per sequence over a paged KV cache.
#include "paged_kv.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Element e of a cached row as axm_dequantize_kv gives it.
__device__ __forceinline__ float kv_value(const PagedKv& kv, const uint8_t* codes, const uint8_t* scales, int e) {
  if (kv.kv_dtype == AXM_KV_FP16) return h2f(reinterpret_cast<const f16*>(codes)[e]);
  const float sc = h2f(reinterpret_cast<const f16*>(scales)[e / 64]);
  if (kv.kv_dtype == AXM_KV_FP8) return h2f(f2h(fp8e4m3fn_to_f32(codes[e]) * sc));
  return h2f(f2h((float)((int)((codes[e / 2] >> (4 * (e & 1)) & 15) ^ 8) - 8) * sc));
}

// One workgroup per (sequence, query head): a wave takes every fourth key.
__global__ void __launch_bounds__(256) paged_decode_kernel(PagedKv kv, const f16* __restrict__ q, int64_t ld_q,
                                                           const int* __restrict__ lens, f16* __restrict__ out, int Hq,
                                                           f32x2* __restrict__ ml) {
  __shared__ float part[4][2 + 128];
  const int b = blockIdx.x / Hq, hq = blockIdx.x % Hq, h = hq / (Hq / kv.Hkv);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, hd = kv.hd;
  const int n = min(max(lens[b], 0), kv.max_pages << kv.page_shift);
  const float scale = kLog2e / __builtin_sqrtf((float)hd);
  float x[2], o[2] = {0.f, 0.f}, m = -INFINITY, l = 0.f;
  for (int e = 0; e < 2; ++e) x[e] = lane + 64 * e < hd ? h2f(q[b * ld_q + hq * hd + lane + 64 * e]) : 0.f;
  for (int key = wave; key < n; key += 4) {
    const int page = paged_page(kv, b, key);
    if (page < 0) continue;
    const int64_t row = paged_row(kv, page, h, key, paged_row_bytes(kv.kv_dtype, hd));
    const int64_t srow = paged_scale_row(kv, page, h, key);
    float d = 0.f;
    for (int e = 0; e < hd / 64; ++e) d += x[e] * kv_value(kv, kv.k + row, kv.ks + srow, lane + 64 * e);
    const float s = wave_sum(d) * scale;
    const float m_new = fmaxf(m, s);
    const float a = m_new == -INFINITY ? 1.f : exp2f(m - m_new), p = exp2f(s - m_new);
    m = m_new;
    l = l * a + p;
    for (int e = 0; e < hd / 64; ++e) o[e] = o[e] * a + p * kv_value(kv, kv.v + row, kv.vs + srow, lane + 64 * e);
  }
  if (lane == 0) {
    part[wave][0] = m;
    part[wave][1] = l;
  }
  for (int e = 0; e < hd / 64; ++e) part[wave][2 + lane + 64 * e] = o[e];
  __syncthreads();
  float mm = -INFINITY, ll = 0.f;
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, part[w][0]);
  for (int w = 0; w < 4; ++w) ll += part[w][0] == -INFINITY ? part[w][1] : part[w][1] * exp2f(part[w][0] - mm);
  for (int e = threadIdx.x; e < hd; e += 256) {
    float oo = 0.f;
    for (int w = 0; w < 4; ++w) oo += part[w][0] == -INFINITY ? part[w][2 + e] : part[w][2 + e] * exp2f(part[w][0] - mm);
    out[((int64_t)b * Hq + hq) * hd + e] = f2h(ll == 0.f ? 0.f : oo / ll);
  }
  if (ml && threadIdx.x == 0) ml[(int64_t)b * Hq + hq] = f32x2{mm, ll};
}

// mass[b][kvh][key] += the group's softmax weights of the key: one wave per key.
__global__ void __launch_bounds__(256) paged_mass_kernel(PagedKv kv, const f16* __restrict__ q, int64_t ld_q,
                                                         const int* __restrict__ lens, int Hq,
                                                         const f32x2* __restrict__ ml, float* __restrict__ mass,
                                                         int64_t mass_len) {
  const int b = blockIdx.x / kv.Hkv, h = blockIdx.x % kv.Hkv, R = Hq / kv.Hkv;
  const int lane = threadIdx.x & 63, hd = kv.hd;
  const int n = min(max(lens[b], 0), kv.max_pages << kv.page_shift);
  const float scale = kLog2e / __builtin_sqrtf((float)hd);
  for (int key = blockIdx.y * 4 + (threadIdx.x >> 6); key < n; key += 4 * gridDim.y) {
    const int page = paged_page(kv, b, key);
    if (page < 0) continue;
    const int64_t row = paged_row(kv, page, h, key, paged_row_bytes(kv.kv_dtype, hd));
    const int64_t srow = paged_scale_row(kv, page, h, key);
    float sum = 0.f;
    for (int r = 0; r < R; ++r) {
      float d = 0.f;
      for (int e = 0; e < hd / 64; ++e)
        d += h2f(q[b * ld_q + (h * R + r) * hd + lane + 64 * e]) * kv_value(kv, kv.k + row, kv.ks + srow, lane + 64 * e);
      const f32x2 x = ml[(int64_t)b * Hq + h * R + r];
      sum += exp2f(wave_sum(d) * scale - x.x) / x.y;
    }
    if (lane == 0) mass[((int64_t)b * kv.Hkv + h) * mass_len + key] += sum;
  }
}

}  // namespace

extern "C" size_t axm_paged_decode_workspace_bytes(int n_seqs, int n_head, int n_kv_head, int head_dim, int page_size,
                                                   int max_pages, int with_mass) {
  return with_mass ? (size_t)n_seqs * n_head * 8 : 0;
}

extern "C" int axm_paged_flash_decode(const void* q, int64_t ld_q, const axm_paged_kv* d, const int* seq_lens, void* out,
                                      int n_head, float* mass, int64_t mass_len, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  PagedKv kv;
  if (int rc = paged_view(d, "paged_flash_decode", &kv)) return rc;
  AXM_CHECK_ARG(q && seq_lens && out, -1, "paged_flash_decode: null pointer");
  AXM_CHECK_ARG(n_head >= kv.Hkv && n_head % kv.Hkv == 0 && n_head / kv.Hkv <= 64, -1,
                "paged_flash_decode: n_head=%d not a multiple (up to 64) of n_kv_head=%d", n_head, kv.Hkv);
  AXM_CHECK_ARG((int64_t)kv.n_seqs * n_head < (1 << 23), -1, "paged_flash_decode: %d sequences of %d heads", kv.n_seqs,
                n_head);
  AXM_CHECK_ARG(ld_q >= (int64_t)n_head * kv.hd && ld_q % 8 == 0 && (uintptr_t)q % 16 == 0, -1,
                "paged_flash_decode: query rows %lld halves apart must be 16-byte aligned", (long long)ld_q);
  AXM_CHECK_ARG(!mass || mass_len >= ((int64_t)kv.max_pages << kv.page_shift), -1,
                "paged_flash_decode: mass has %lld slots, the table %lld", (long long)mass_len,
                (long long)kv.max_pages << kv.page_shift);
  const size_t need = axm_paged_decode_workspace_bytes(kv.n_seqs, n_head, kv.Hkv, kv.hd, 1 << kv.page_shift,
                                                       kv.max_pages, mass != nullptr);
  AXM_CHECK_ARG(workspace_bytes >= need && (need == 0 || workspace), -1,
                "paged_flash_decode: workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  const hipStream_t s = (hipStream_t)stream;
  hipLaunchKernelGGL(paged_decode_kernel, dim3(kv.n_seqs * n_head), dim3(256), 0, s, kv, (const f16*)q, ld_q, seq_lens,
                     (f16*)out, n_head, (f32x2*)workspace);
  AXM_LAUNCH_CHECK("paged_flash_decode");
  if (mass) {
    hipLaunchKernelGGL(paged_mass_kernel, dim3(kv.n_seqs * kv.Hkv, 16), dim3(256), 0, s, kv, (const f16*)q, ld_q,
                       seq_lens, n_head, (const f32x2*)workspace, mass, mass_len);
    AXM_LAUNCH_CHECK("paged_flash_decode (mass)");
  }
  return 0;
}
