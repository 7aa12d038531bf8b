// Write and read back of a paged K/V cache (mapa_kv_cache_write, mapa_kv_cache_read).
//
// Both are memory-bound row copies with a page lookup and, for 8-bit pages, one power-of-two exponent per row of 64
// values: eight lanes hold a row, eight values each (16 B of a 16-bit row), so its largest value is three exchanges
// away and a wave moves eight whole rows.  A workgroup takes a few tokens; its threads find their sequences by looking
// at all row offsets at once (thread i holds the interval of sequence i: one trip to memory however many sequences
// there are, where a binary search makes log2 of them) and one thread per token looks its page up.  The rows follow as
// (K or V, head, token): a wave's eight rows are neighbours in the page (512 B of 8-bit codes and eight exponent bytes
// in a row), where (token, head) order scatters them over eight heads' parts of it.  Measured: 25 thousand tokens of 16
// heads into int8 pages, 153 MB, 36.7 us (4.2 TB/s), 59 thousand back out of them, 365 MB, 80.8 us (4.5 TB/s; copy: 5.04);
// 32 tokens of 12 heads, 3.4 us, which is a launch and the three trips to memory of offsets, table and rows.
#include <type_traits>

#include "paged.h"

namespace {
using namespace mapa_paged;

constexpr int TPB = 256;
constexpr int MAX_TB = 8;  // tokens per workgroup

struct CopyArgs {
  void* page[2];  // K, V
  uint8_t* exp[2];
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* cu;
  void* row[2];
  int64_t rs[2], hs[2];
  unsigned* fault;
  int seqs, table_stride, rows, cap, heads, psl, num_pages;
  int tb, tbl;  // tokens per workgroup (a power of two), its logarithm
};

constexpr int U = 8;  // rows in flight per group of eight lanes (4: 2 % slower)

// largest of the eight lanes of a row
__device__ __forceinline__ uint32_t max8(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xf, 0xf, true));  // quad_perm 1, 0, 3, 2
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xf, 0xf, true));  // quad_perm 2, 3, 0, 1
  return max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xf, 0xf, true));  // row_half_mirror: 7 - lane
}

// 8 values of a row as they lie in memory
struct Float8 {
  f32x4 a, b;
};
template <int DT>
struct Row8 {
  typedef uint4 T;
};
template <>
struct Row8<MAPA_F32> {
  typedef Float8 T;
};
template <int DT>
__device__ __forceinline__ void unpack8(const typename Row8<DT>::T& u, float* f) {
  if constexpr (DT == MAPA_F32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = u.a[j];
      f[4 + j] = u.b[j];
    }
  } else {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = lp_to_f32(DT == MAPA_F16, (uint16_t)(w[j] & 0xffff));
      f[2 * j + 1] = lp_to_f32(DT == MAPA_F16, (uint16_t)(w[j] >> 16));
    }
  }
}
template <int DT>
__device__ __forceinline__ typename Row8<DT>::T pack8(const float* f) {
  if constexpr (DT == MAPA_F32)
    return Float8{f32x4{f[0], f[1], f[2], f[3]}, f32x4{f[4], f[5], f[6], f[7]}};
  else
    return uint4{pack_lp2(DT == MAPA_F16, f[0], f[1]), pack_lp2(DT == MAPA_F16, f[2], f[3]),
                 pack_lp2(DT == MAPA_F16, f[4], f[5]), pack_lp2(DT == MAPA_F16, f[6], f[7])};
}

// Rows written once and not read here again go past the caches' keeping (views read back: 35.5 us without, 32.2 with)
__device__ __forceinline__ void st_stream(void* p, const uint4& v) {
  __builtin_nontemporal_store(__builtin_bit_cast(f32x4, v), reinterpret_cast<f32x4*>(p));
}
__device__ __forceinline__ void st_stream(void* p, const Float8& v) {
  __builtin_nontemporal_store(v.a, reinterpret_cast<f32x4*>(p));
  __builtin_nontemporal_store(v.b, reinterpret_cast<f32x4*>(p) + 1);
}

// Rows read once (a third of a projection's rows: 120 us without, 106 with, for 25 thousand tokens into int8 pages)
template <int DT>
__device__ __forceinline__ typename Row8<DT>::T ld_stream(const char* p) {
  const f32x4* q = reinterpret_cast<const f32x4*>(p);
  if constexpr (DT == MAPA_F32) return Float8{__builtin_nontemporal_load(q), __builtin_nontemporal_load(q + 1)};
  else return __builtin_bit_cast(uint4, __builtin_nontemporal_load(q));
}

// Sequence of each of the workgroup's rows t0 .. t0 + nt - 1 into `seq` (-1: none), by the packed offsets cu.
__device__ __forceinline__ void find_sequences(const CopyArgs& a, int t0, int nt, int* seq) {
  if (threadIdx.x < MAX_TB) seq[threadIdx.x] = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < a.seqs; i += TPB) {
    const int c0 = a.cu[i], c1 = a.cu[i + 1];
    if (c0 < 0 || c1 < c0 || c1 > a.rows) {
      if (blockIdx.x == 0) kv_fault(a.fault);
      continue;
    }
    for (int t = max(c0, t0); t < min(c1, t0 + nt); ++t) seq[t - t0] = i;
  }
  __syncthreads();
}

// SRC: type of the new rows; PAGE: type of the pages
template <int SRC, int PAGE>
__global__ void __launch_bounds__(TPB) kv_write_kernel(CopyArgs a) {
  constexpr bool CODES = PAGE == MAPA_FP8 || PAGE == MAPA_I8;
  __shared__ int seq[MAX_TB];
  __shared__ int64_t at[MAX_TB];  // row of the page that takes the token, for head 0; -1: nothing to write
  const int t0 = blockIdx.x * a.tb, nt = min(a.rows - t0, a.tb);
  find_sequences(a, t0, nt, seq);
  if (threadIdx.x < a.tb) {
    const int t = t0 + threadIdx.x, b = seq[threadIdx.x];  // -1 past the last row
    int64_t r = -1;
    if (b >= 0) {
      const int c0 = a.cu[b], c1 = a.cu[b + 1];
      const int pos = a.kv_lens[b] - (c1 - c0) + (t - c0);
      if (pos < 0 || pos >= a.cap) {
        kv_fault(a.fault);
      } else {
        const int page = a.table[(int64_t)b * a.table_stride + (pos >> a.psl)];
        if ((unsigned)page >= (unsigned)a.num_pages) kv_fault(a.fault);
        else r = (((int64_t)page * a.heads) << a.psl) + (pos & ((1 << a.psl) - 1));
      }
    }
    at[threadIdx.x] = r;
  }
  __syncthreads();

  // rows (K or V, head, token); the eight lanes of a row stay together, U rows per lane group in flight
  const int rows = 2 * a.heads << a.tbl;
  const int l8 = threadIdx.x & 7;
  for (int r0 = threadIdx.x >> 3; r0 < rows; r0 += U * (TPB / 8)) {
    typename Row8<SRC>::T x[U];
    int64_t dst[U];
    bool isv[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int r = r0 + k * (TPB / 8);
      const int kh = r >> a.tbl, tl = r & (a.tb - 1);
      isv[k] = kh >= a.heads;
      const int h = isv[k] ? kh - a.heads : kh;
      dst[k] = -1;
      if (r < rows && at[tl] >= 0) {
        dst[k] = at[tl] + ((int64_t)h << a.psl);
        const int64_t src = (int64_t)(t0 + tl) * (isv[k] ? a.rs[1] : a.rs[0]) + h * (isv[k] ? a.hs[1] : a.hs[0]) + l8 * 8;
        x[k] = ld_stream<SRC>(reinterpret_cast<const char*>(isv[k] ? a.row[1] : a.row[0]) + src * (SRC == MAPA_F32 ? 4 : 2));
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (dst[k] < 0) continue;  // the same for the eight lanes of the row
      void* page = isv[k] ? a.page[1] : a.page[0];
      if constexpr (SRC == PAGE) {
        reinterpret_cast<uint4*>(page)[dst[k] * 8 + l8] = __builtin_bit_cast(uint4, x[k]);
      } else {
        float f[8];
        unpack8<SRC>(x[k], f);
        if constexpr (!CODES) {
          reinterpret_cast<uint4*>(page)[dst[k] * 8 + l8] = __builtin_bit_cast(uint4, pack8<PAGE>(f));
        } else {
          uint32_t m = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
          m = max8(m);
          const uint32_t e = row_exponent<PAGE == MAPA_I8>(m);
          const float inv = exponent_inverse(e);
          uint2 w;
          if constexpr (PAGE == MAPA_FP8) {
            int lo = 0, hi = 0;
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inv, f[1] * inv, lo, false);
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * inv, f[3] * inv, lo, true);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * inv, f[5] * inv, hi, false);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * inv, f[7] * inv, hi, true);
            w = uint2{(uint32_t)lo, (uint32_t)hi};
            if (e == 255u) w = uint2{0x7f7f7f7fu, 0x7f7f7f7fu};  // e4m3's NaN
          } else {
            // x 2^-e + 1.5 2^23: the sum's last bits are the integer, rounded to nearest even (|code| <= 127)
            uint32_t c[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j] = __float_as_uint(__builtin_fmaf(f[j], inv, 12582912.f));
            const uint32_t c01 = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), c23 = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
            const uint32_t c45 = __builtin_amdgcn_perm(c[5], c[4], 0x0c0c0400u), c67 = __builtin_amdgcn_perm(c[7], c[6], 0x04000c0cu);
            w = uint2{c01 | c23, c45 | c67};
            if (e == 255u) w = uint2{0u, 0u};
          }
          reinterpret_cast<uint2*>(page)[dst[k] * 8 + l8] = w;
          if (l8 == 0) (isv[k] ? a.exp[1] : a.exp[0])[dst[k]] = (uint8_t)e;
        }
      }
    }
  }
}

template <int PAGE, int OUT>
__global__ void __launch_bounds__(TPB) kv_read_kernel(CopyArgs a) {
  constexpr bool CODES = PAGE == MAPA_FP8 || PAGE == MAPA_I8;
  __shared__ int seq[MAX_TB];
  __shared__ int64_t at[MAX_TB];  // row of the page that holds the token, for head 0; -1: zero, -2: not a row of ours
  const int t0 = blockIdx.x * a.tb, nt = min(a.rows - t0, a.tb);
  find_sequences(a, t0, nt, seq);
  if (threadIdx.x < a.tb) {
    const int b = seq[threadIdx.x];  // -1 past the last row
    int64_t r = -2;
    if (b >= 0) {
      const int pos = t0 + threadIdx.x - a.cu[b];
      r = -1;
      if (pos < checked_len(a.kv_lens[b], a.cap, a.fault)) {
        const int page = checked_page(a.table[(int64_t)b * a.table_stride + (pos >> a.psl)], a.num_pages, a.fault);
        r = (((int64_t)page * a.heads) << a.psl) + (pos & ((1 << a.psl) - 1));
      }
    }
    at[threadIdx.x] = r;
  }
  __syncthreads();

  const int rows = 2 * a.heads << a.tbl;
  const int l8 = threadIdx.x & 7;
  for (int r0 = threadIdx.x >> 3; r0 < rows; r0 += U * (TPB / 8)) {
    uint4 x[U];  // 16-bit pages: 8 values; codes: 8 codes and the exponent byte
    char* dst[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int r = r0 + k * (TPB / 8);
      const int kh = r >> a.tbl, tl = r & (a.tb - 1);
      const bool isv = kh >= a.heads;
      const int h = isv ? kh - a.heads : kh;
      dst[k] = nullptr;
      x[k] = uint4{0, 0, 0, 0};
      if (r < rows && at[tl] != -2) {
        const int64_t from = at[tl], src = from + ((int64_t)h << a.psl);
        dst[k] = reinterpret_cast<char*>(isv ? a.row[1] : a.row[0]) +
                 ((int64_t)(t0 + tl) * (isv ? a.rs[1] : a.rs[0]) + h * (isv ? a.hs[1] : a.hs[0]) + l8 * 8) *
                     (OUT == MAPA_F32 ? 4 : 2);
        if (from >= 0) {
          const void* page = isv ? a.page[1] : a.page[0];
          if constexpr (!CODES) {
            x[k] = reinterpret_cast<const uint4*>(page)[src * 8 + l8];
          } else {
            const uint2 w = reinterpret_cast<const uint2*>(page)[src * 8 + l8];
            x[k] = uint4{w.x, w.y, (isv ? a.exp[1] : a.exp[0])[src], 0};
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (!dst[k]) continue;
      if constexpr (PAGE == OUT) {
        st_stream(dst[k], x[k]);
      } else {
        float f[8];
        if constexpr (!CODES) {
          unpack8<PAGE>(x[k], f);
        } else {
          const float s = exponent_value(x[k].z);
          const f32x4 lo = decode4<PAGE == MAPA_I8>(x[k].x, s), hi = decode4<PAGE == MAPA_I8>(x[k].y, s);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f[j] = lo[j];
            f[4 + j] = hi[j];
          }
        }
        st_stream(dst[k], pack8<OUT>(f));
      }
    }
  }
}

template <typename F>
int by_page(int dtype, F f) {
  switch (dtype) {
    case MAPA_BF16: f(std::integral_constant<int, MAPA_BF16>()); break;
    case MAPA_F16: f(std::integral_constant<int, MAPA_F16>()); break;
    case MAPA_FP8: f(std::integral_constant<int, MAPA_FP8>()); break;
    default: f(std::integral_constant<int, MAPA_I8>()); break;
  }
  return 0;
}
template <typename F>
int by_row(int dtype, F f) {
  switch (dtype) {
    case MAPA_F32: f(std::integral_constant<int, MAPA_F32>()); break;
    case MAPA_BF16: f(std::integral_constant<int, MAPA_BF16>()); break;
    default: f(std::integral_constant<int, MAPA_F16>()); break;
  }
  return 0;
}

int fill_args(CopyArgs& a, const mapa_kv_cache* c, const mapa_kv_batch* b, const void* k, const void* v, int dtype,
              int64_t krs, int64_t khs, int64_t vrs, int64_t vhs, const char* who) {
  MAPA_CHECK_ARG(c && b, "%s: null descriptor", who);
  if (int rc = check_cache(*c, who)) return rc;
  if (int rc = check_batch(*b, who)) return rc;
  MAPA_CHECK_ARG(dtype == MAPA_F32 || dtype == MAPA_BF16 || dtype == MAPA_F16, "%s: rows must be f32, bf16 or f16", who);
  MAPA_CHECK_ARG(k && v, "%s: null rows", who);
  const int el = dtype == MAPA_F32 ? 4 : 8;
  MAPA_CHECK_ARG((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && krs % el == 0 && khs % el == 0 && vrs % el == 0 &&
                     vhs % el == 0,
                 "%s: row bases and strides must keep 16-byte alignment", who);
  a.page[0] = c->k; a.page[1] = c->v;
  a.exp[0] = c->k_exp; a.exp[1] = c->v_exp;
  a.table = b->table; a.kv_lens = b->kv_lens;
  a.row[0] = const_cast<void*>(k); a.row[1] = const_cast<void*>(v);
  a.rs[0] = krs; a.rs[1] = vrs; a.hs[0] = khs; a.hs[1] = vhs;
  a.fault = mapa_gemm_impl::fault_word();
  a.seqs = b->seqs; a.table_stride = b->table_stride;
  a.cap = kv_cap(*c, *b);
  a.heads = c->heads; a.psl = log2_of(c->page_size); a.num_pages = c->num_pages;
  return 0;
}
// tokens per workgroup: one while that leaves fewer than four workgroups per CU, so that a step's few tokens spread
int tokens_per_block(int rows) {
  int tb = 1;
  while (tb < MAX_TB && rows / (2 * tb) >= 1024) tb *= 2;
  return tb;
}

}  // namespace

extern "C" int mapa_kv_cache_write(const mapa_kv_cache* c, const mapa_kv_batch* b, const void* k, const void* v,
                                   int dtype, int64_t k_rstride, int64_t k_hstride, int64_t v_rstride,
                                   int64_t v_hstride, hipStream_t stream) {
  CopyArgs a = {};
  if (b && c && (b->seqs == 0 || b->new_rows == 0)) {
    if (int rc = check_cache(*c, "mapa_kv_cache_write")) return rc;
    return check_batch(*b, "mapa_kv_cache_write");
  }
  if (int rc = fill_args(a, c, b, k, v, dtype, k_rstride, k_hstride, v_rstride, v_hstride, "mapa_kv_cache_write"))
    return rc;
  const bool codes = c->dtype == MAPA_FP8 || c->dtype == MAPA_I8;
  MAPA_CHECK_ARG(c->k != c->v && !(codes && c->k_exp == c->v_exp),
                 "mapa_kv_cache_write: keys and values share their pages or exponents");
  a.cu = b->cu_new;
  a.rows = b->new_rows;
  a.tb = tokens_per_block(a.rows);
  a.tbl = log2_of(a.tb);
  const dim3 grid((unsigned)((a.rows + a.tb - 1) / a.tb));
  by_row(dtype, [&](auto src) {
    by_page(c->dtype, [&](auto page) {
      hipLaunchKernelGGL((kv_write_kernel<decltype(src)::value, decltype(page)::value>), grid, dim3(TPB), 0, stream, a);
    });
  });
  MAPA_CHECK_LAUNCH("mapa_kv_cache_write");
  return 0;
}

extern "C" int mapa_kv_cache_read(const mapa_kv_cache* c, const mapa_kv_batch* b, const int32_t* cu_rows, int rows,
                                  void* k_out, void* v_out, int dtype, int64_t k_rstride, int64_t k_hstride,
                                  int64_t v_rstride, int64_t v_hstride, hipStream_t stream) {
  CopyArgs a = {};
  MAPA_CHECK_ARG(rows >= 0, "mapa_kv_cache_read: bad row count %d", rows);
  if (b && c && (b->seqs == 0 || rows == 0)) {
    if (int rc = check_cache(*c, "mapa_kv_cache_read")) return rc;
    return check_batch(*b, "mapa_kv_cache_read");
  }
  if (int rc = fill_args(a, c, b, k_out, v_out, dtype, k_rstride, k_hstride, v_rstride, v_hstride,
                         "mapa_kv_cache_read"))
    return rc;
  MAPA_CHECK_ARG(cu_rows != nullptr, "mapa_kv_cache_read: null cu_rows");
  MAPA_CHECK_ARG(k_out != v_out, "mapa_kv_cache_read: keys and values have one output");
  a.cu = cu_rows;
  a.rows = rows;
  a.tb = tokens_per_block(a.rows);
  a.tbl = log2_of(a.tb);
  const dim3 grid((unsigned)((a.rows + a.tb - 1) / a.tb));
  by_row(dtype, [&](auto out) {
    by_page(c->dtype, [&](auto page) {
      hipLaunchKernelGGL((kv_read_kernel<decltype(page)::value, decltype(out)::value>), grid, dim3(TPB), 0, stream, a);
    });
  });
  MAPA_CHECK_LAUNCH("mapa_kv_cache_read");
  return 0;
}
