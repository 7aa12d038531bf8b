// Shared by the paged K/V cache kernels (kv_cache.hip, attention_paged.hip): argument checks, the codes of the 8-bit
// pages, and the device-side checks of what the host cannot see.
#pragma once
#include "mapa_common.h"

namespace mapa_paged {

constexpr int HD = 64;  // head dim, as every attention of the library
constexpr unsigned FAULT_KV_RANGE = 4u;  // MAPA_FAULT_KV_RANGE

__device__ __forceinline__ void kv_fault(unsigned* fault) {
  if (fault) __hip_atomic_fetch_or(fault, FAULT_KV_RANGE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Tokens in the cache of sequence b, held within what the host stated (max_kv, the table's width).
__device__ __forceinline__ int checked_len(int len, int cap, unsigned* fault) {
  if (len < 0 || len > cap) {
    kv_fault(fault);
    len = len < 0 ? 0 : cap;
  }
  return len;
}
// Page number held within the cache.
__device__ __forceinline__ int checked_page(int page, int num_pages, unsigned* fault) {
  if ((unsigned)page >= (unsigned)num_pages) {
    kv_fault(fault);
    page = 0;
  }
  return page;
}

// Row exponents of the 8-bit pages.  amax_bits: the row's largest |value| as fp32 bits (an integer maximum, so an
// infinity or a NaN wins it).  With |max| = m 2^k, 1 <= m < 2, the largest code is t 2^c (448 = 1.75 2^8, 127 =
// 1.984375 2^6): the exponent is k - c, one more if m > t.  Rows below 2^-100 share its exponent, so the scaling by
// 2^-exponent stays a normal number; 255 marks a row with a value that is not finite.
template <bool I8>
__device__ __forceinline__ uint32_t row_exponent(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const uint32_t a = max(amax_bits, (uint32_t)(127 - 100) << 23);
  return (a >> 23) - (I8 ? 6u : 8u) + ((a & 0x7fffffu) > (I8 ? 0x7e0000u : 0x600000u) ? 1u : 0u);
}
__device__ __forceinline__ float exponent_value(uint32_t byte) { return __uint_as_float(byte << 23); }  // 255: +inf
__device__ __forceinline__ float exponent_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Four codes of a word as fp32, times the row's scale (exact: a power of two).  A row held as NaN has the scale +inf:
// its codes are e4m3's NaN, or int8's 0 (0 * inf).
template <bool I8>
__device__ __forceinline__ f32x4 decode4(uint32_t w, float s) {
  f32x4 r;
  if constexpr (I8) {
    r[0] = (float)(int8_t)(w & 0xffu) * s;
    r[1] = (float)(int8_t)((w >> 8) & 0xffu) * s;
    r[2] = (float)(int8_t)((w >> 16) & 0xffu) * s;
    r[3] = (float)(int8_t)(w >> 24) * s;
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    r[0] = lo[0] * s;
    r[1] = lo[1] * s;
    r[2] = hi[0] * s;
    r[3] = hi[1] * s;
  }
  return r;
}

inline int check_cache(const mapa_kv_cache& c, const char* who) {
  MAPA_CHECK_ARG(c.dtype == MAPA_BF16 || c.dtype == MAPA_F16 || c.dtype == MAPA_FP8 || c.dtype == MAPA_I8,
                 "%s: pages must be bf16, f16, fp8 or i8", who);
  MAPA_CHECK_ARG(c.heads > 0 && c.heads <= 2048 && c.num_pages > 0, "%s: bad cache (%d heads, %d pages)", who, c.heads,
                 c.num_pages);
  MAPA_CHECK_ARG(c.page_size >= 16 && c.page_size <= 1024 && (c.page_size & (c.page_size - 1)) == 0,
                 "%s: page size %d must be a power of two, 16 to 1024", who, c.page_size);
  MAPA_CHECK_ARG(c.k && c.v && (uintptr_t)c.k % 16 == 0 && (uintptr_t)c.v % 16 == 0,
                 "%s: pages must be 16-byte aligned device memory", who);
  const bool codes = c.dtype == MAPA_FP8 || c.dtype == MAPA_I8;
  MAPA_CHECK_ARG(!codes || (c.k_exp && c.v_exp), "%s: 8-bit pages need exponent bytes", who);
  return 0;
}
inline int check_batch(const mapa_kv_batch& b, const char* who) {
  MAPA_CHECK_ARG(b.seqs >= 0 && b.seqs <= 65535 && b.table_stride >= 0 && b.new_rows >= 0 && b.max_new >= 0 &&
                     b.max_kv >= 0 && b.max_kv <= (1 << 30),
                 "%s: bad batch (%d sequences, %d table columns, %d rows, max_kv %d)", who, b.seqs, b.table_stride,
                 b.new_rows, b.max_kv);
  MAPA_CHECK_ARG(b.seqs == 0 || (b.kv_lens && b.cu_new && (b.table || b.table_stride == 0)),
                 "%s: null batch array", who);
  return 0;
}
inline int log2_of(int v) { return __builtin_ctz((unsigned)v); }
// largest token count of a sequence that the table and the host's bound allow
inline int kv_cap(const mapa_kv_cache& c, const mapa_kv_batch& b) {
  const int64_t t = (int64_t)b.table_stride * c.page_size;
  return (int)(t < b.max_kv ? t : b.max_kv);
}

}  // namespace mapa_paged
