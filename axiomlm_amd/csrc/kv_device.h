// Device helpers that the matrix-core attention kernels share: cached codes to fp16, row reductions, the weight tile
// and the transposed value operand.
#pragma once
#include "axm.h"
#include "axm_common.h"

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegBig = -1e30f;

// A raw 8-element key/value chunk (fp16: 16 B, fp8: 8 B, int4: 4 B) and its fp16
// group scale become eight fp32 values with the rounding of load_kv8.
// HW: fp8 codes through v_cvt_pk_f32_fp8 (OCP E4M3FN on gfx950; every finite
// code converts exactly, so the result equals the table-free decode below for
// all non-NaN codes).  The attention kernels use it; the dequantization entry
// point keeps the bitwise decode so that NaN codes keep their exact pattern.
typedef float f32x2_hw __attribute__((ext_vector_type(2)));
template <int KVT, bool HW = false>
__device__ __forceinline__ void kv8_convert(u32x4 r, float sc, float out[8]) {
  if (KVT == AXM_KV_FP8 && HW) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const uint32_t word = r[w];
      const f32x2_hw lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false);
      const f32x2_hw hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
      out[4 * w + 0] = h2f(f2h(lo.x * sc));
      out[4 * w + 1] = h2f(f2h(lo.y * sc));
      out[4 * w + 2] = h2f(f2h(hi.x * sc));
      out[4 * w + 3] = h2f(f2h(hi.y * sc));
    }
    return;
  }
  if (KVT == AXM_KV_FP16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = r[i];
      const f16x2 h = as_h2(w);
      out[2 * i] = h2f(h.x);
      out[2 * i + 1] = h2f(h.y);
    }
  } else if (KVT == AXM_KV_FP8) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = r[i >> 2];
      out[i] = h2f(f2h(fp8e4m3fn_to_f32((w >> (8 * (i & 3))) & 0xFFu) * sc));
    }
  } else {
    const uint32_t w = r.x;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int q = (int)(((w >> (4 * i)) & 0xFu) ^ 0x8u) - 8;
      out[i] = h2f(f2h((float)q * sc));
    }
  }
}

// Eight raw codes of a cache row and their group's scale.
struct KvRaw8 {
  u32x4 r;
  uint32_t sc;  // fp16 bits in the low half
};

// Position e of an f16x8 from kv_half8 holds element kv_dim_of<KVT>(e) of the chunk:
// the int4 form delivers the even elements 0, 2, 4, 6, then the odd ones.
template <int KVT>
__device__ __forceinline__ constexpr int kv_dim_of(int e) {
  return KVT == AXM_KV_INT4 ? ((e & 3) << 1) | (e >> 2) : e;
}

// Eight consecutive query elements in the order kv_half8 delivers the chunk's
// elements (the MFMA k index then pairs each query element with its key element).
template <int KVT>
__device__ __forceinline__ f16x8 kv_order8(f16x8 v) {
  f16x8 r;
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = v[kv_dim_of<KVT>(e)];
  return r;
}

template <int KVT>
__device__ __forceinline__ f16x8 kv_half8(const KvRaw8& f) {
  if (KVT == AXM_KV_FP16) return __builtin_bit_cast(f16x8, f.r);
  if (KVT == AXM_KV_INT4) {
    // u = nibble ^ 8 = q + 8 in [0, 15].  The even nibbles (one per byte of lo) and
    // the odd ones (hi) become, by one byte permute per pair with the exponent byte
    // 0x64, the exact halves 1024 + u; minus 1032 gives q exactly, and one fp16
    // multiply by the scale rounds q * scale once (the fp32 product of a 4-bit
    // integer and an fp16 scale is exact, so this equals fp16(float(q) * scale)).
    const uint32_t u = f.r.x ^ 0x88888888u;
    const uint32_t lo = u & 0x0F0F0F0Fu, hi = (u >> 4) & 0x0F0F0F0Fu;
    const f16 sc = u16_as_h((uint16_t)f.sc);
    const f16x2 s2 = {sc, sc};
    const f16x2 off = {(f16)1032.f, (f16)1032.f};
    const uint32_t pr[4] = {__builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u),
                            __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u),
                            __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u),
                            __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)};
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = as_u32((as_h2(pr[i]) - off) * s2);
    return __builtin_bit_cast(f16x8, o);
  }
  if (KVT == AXM_KV_FP8) {
    // Two E4M3FN codes -> two fp16 per conversion (scale 1.0: every finite code is
    // an exact fp16), then one fp16 multiply rounds code * scale once, as the fp32
    // product (exact: 4 x 11 significant bits) rounded to fp16 does.
    const f16 sc = u16_as_h((uint16_t)f.sc);
    const f16x2 s2 = {sc, sc};
    u32x4 o;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      o[2 * w] = as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(f.r[w], 1.0f, false) * s2);
      o[2 * w + 1] = as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(f.r[w], 1.0f, true) * s2);
    }
    return __builtin_bit_cast(f16x8, o);
  }
  float x[8];
  kv8_convert<KVT, true>(f.r, h2f(u16_as_h((uint16_t)f.sc)), x);
  f16x8 h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = f2h(x[i]);
  return h;
}

template <int CTRL>
__device__ __forceinline__ float dpp_sum_step(float v) {
  const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false);
  return v + __builtin_bit_cast(float, o);
}

// 2^x with the bare v_exp_f32: softmax weights below 2^-126 of the running
// maximum are flushed to zero instead of kept as denormals, which changes no
// fp16 output.
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

template <int CTRL>
__device__ __forceinline__ float dpp_max_step(float v) {
  const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false);
  return fmaxf(v, __builtin_bit_cast(float, o));
}
__device__ __forceinline__ float row16_max(float v) {
  v = dpp_max_step<0xB1>(v);
  v = dpp_max_step<0x4E>(v);
  v = dpp_max_step<0x141>(v);
  return dpp_max_step<0x140>(v);
}
__device__ __forceinline__ float row16_sum(float v) {
  v = dpp_sum_step<0xB1>(v);
  v = dpp_sum_step<0x4E>(v);
  v = dpp_sum_step<0x141>(v);
  return dpp_sum_step<0x140>(v);
}

constexpr int kTreeKeys = 32;    // keys per block (the k extent of one P V MFMA)

// P tile of the matrix-core attention kernels, [row][key] with 32 keys per row:
// written 4 rows x 16 keys at a time, read 8 keys per row; the 8-key groups of
// row r are XOR-swizzled by bits 2-3 of r (2-way bank conflicts at most).
__device__ __forceinline__ int pt_index(int row, int key) {
  return row * kTreeKeys + (((key >> 3) ^ ((row >> 2) & 3)) << 3) + (key & 7);
}

// B operand of O += P V from V rows stored key-major (row stride vrow halves;
// seg = row 0 of a 16-dim tile): lane (l16, lq) needs dim column l16 of keys
// 8 lq .. 8 lq + 7.  ds_read_b64_tr_b16 over a 16-lane group returns to lane i
// column i of the 4 x 16 block whose row r is the 4 x 8 bytes the group's lanes
// 4 r .. 4 r + 3 address, so lane i addresses key (i / 4) of the group's four,
// dims 4 (i % 4) .. + 3; two reads give keys 8 lq .. + 3 and 8 lq + 4 .. + 7.
typedef short tr_v4s __attribute__((vector_size(8)));
__device__ __forceinline__ f16x8 v_operand(const f16* seg, int vrow, int l16, int lq) {
  typedef __attribute__((address_space(3))) tr_v4s lds_v4s;
  const f16* p0 = seg + (8 * lq + (l16 >> 2)) * vrow + 4 * (l16 & 3);
  const tr_v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)p0);
  const tr_v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(p0 + 4 * vrow));
  f16x8 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    r[e] = __builtin_bit_cast(f16, (short)a[e]);
    r[4 + e] = __builtin_bit_cast(f16, (short)b[e]);
  }
  return r;
}
// Dim of output column c of a 16-dim tile whose V rows were stored in kv_half8's
// order (int4: positions 0..7 of each 8-dim chunk hold dims 0, 2, 4, 6, 1, 3, 5, 7).
template <int KVT>
__device__ __forceinline__ int kv_col_dim(int c) {
  return (c & 8) | kv_dim_of<KVT>(c & 7);
}
