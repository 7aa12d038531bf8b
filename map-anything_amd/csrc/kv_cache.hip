// Write and read back of a paged K/V cache (mapa_kv_cache_write, mapa_kv_cache_read).
//
// Both are memory-bound row copies with a page lookup and, for 8-bit pages, one power-of-two exponent per row of 64
// values: eight lanes hold a row, eight values each (16 B of a 16-bit row), so its largest value is three exchanges
// away and a wave moves eight whole rows.  A workgroup takes a few tokens; its threads find their sequences by looking
// at all row offsets at once (thread i holds the interval of sequence i: one trip to memory however many sequences
// there are, where a binary search makes log2 of them), one thread per token looks its page up, and the (token, K or V,
// head) rows follow in an order that keeps neighbouring lanes on neighbouring memory.
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
  int seqs, table_stride, rows, cap, heads, psl, num_pages, tb;
};

struct Place {
  int seq, pos;
};

// 8 values of a row in fp32
template <int DT>
__device__ __forceinline__ void ld8(const void* p, float* f) {
  if constexpr (DT == MAPA_F32) {
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = a[j];
      f[4 + j] = b[j];
    }
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = lp_to_f32(DT == MAPA_F16, (uint16_t)(w[j] & 0xffff));
      f[2 * j + 1] = lp_to_f32(DT == MAPA_F16, (uint16_t)(w[j] >> 16));
    }
  }
}
template <int DT>
__device__ __forceinline__ void st8(void* p, const float* f) {
  if constexpr (DT == MAPA_F32) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{f[0], f[1], f[2], f[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{f[4], f[5], f[6], f[7]};
  } else {
    *reinterpret_cast<uint4*>(p) =
        uint4{pack_lp2(DT == MAPA_F16, f[0], f[1]), pack_lp2(DT == MAPA_F16, f[2], f[3]),
              pack_lp2(DT == MAPA_F16, f[4], f[5]), pack_lp2(DT == MAPA_F16, f[6], f[7])};
  }
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
  if (threadIdx.x < nt) {
    const int t = t0 + threadIdx.x, b = seq[threadIdx.x];
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

  const int rows = nt * 2 * a.heads;
  const int l8 = threadIdx.x & 7;
  for (int r = threadIdx.x >> 3; r < rows; r += TPB / 8) {  // the eight lanes of a row stay together
    const int tk = r / a.heads, h = r - tk * a.heads, tl = tk >> 1, kv = tk & 1;
    const int64_t to = at[tl];
    if (to < 0) continue;
    const int64_t dst = to + ((int64_t)h << a.psl);
    const int64_t src = (int64_t)(t0 + tl) * a.rs[kv] + h * a.hs[kv] + l8 * 8;
    if constexpr (SRC == PAGE) {
      reinterpret_cast<uint4*>(a.page[kv])[dst * 8 + l8] =
          *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.row[kv]) + src);
    } else {
      float f[8];
      ld8<SRC>(reinterpret_cast<const char*>(a.row[kv]) + src * (SRC == MAPA_F32 ? 4 : 2), f);
      if constexpr (!CODES) {
        st8<PAGE>(reinterpret_cast<uint16_t*>(a.page[kv]) + dst * HD + l8 * 8, f);
      } else {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(f[j]) & 0x7fffffffu);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
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
          uint32_t c[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) c[j] = (uint32_t)(int)rintf(e == 255u ? 0.f : f[j] * inv) & 0xffu;
          w = uint2{c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24), c[4] | (c[5] << 8) | (c[6] << 16) | (c[7] << 24)};
        }
        reinterpret_cast<uint2*>(a.page[kv])[dst * 8 + l8] = w;
        if (l8 == 0) a.exp[kv][dst] = (uint8_t)e;
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
  if (threadIdx.x < nt) {
    const int b = seq[threadIdx.x];
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

  const int rows = nt * 2 * a.heads;
  const int l8 = threadIdx.x & 7;
  for (int r = threadIdx.x >> 3; r < rows; r += TPB / 8) {
    const int tk = r / a.heads, h = r - tk * a.heads, tl = tk >> 1, kv = tk & 1;
    const int64_t from = at[tl];
    if (from == -2) continue;
    const int64_t src = from + ((int64_t)h << a.psl);
    char* dst = reinterpret_cast<char*>(a.row[kv]) +
                ((int64_t)(t0 + tl) * a.rs[kv] + h * a.hs[kv] + l8 * 8) * (OUT == MAPA_F32 ? 4 : 2);
    if constexpr (PAGE == OUT) {
      *reinterpret_cast<uint4*>(dst) = from < 0 ? uint4{0, 0, 0, 0} : reinterpret_cast<const uint4*>(a.page[kv])[src * 8 + l8];
    } else {
      float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (from >= 0) {
        if constexpr (!CODES) {
          ld8<PAGE>(reinterpret_cast<const uint16_t*>(a.page[kv]) + src * HD + l8 * 8, f);
        } else {
          const uint2 w = reinterpret_cast<const uint2*>(a.page[kv])[src * 8 + l8];
          const float s = exponent_value(a.exp[kv][src]);
          const f32x4 x = decode4<PAGE == MAPA_I8>(w.x, s), y = decode4<PAGE == MAPA_I8>(w.y, s);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            f[j] = x[j];
            f[4 + j] = y[j];
          }
        }
      }
      st8<OUT>(dst, f);
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
  a.cu = b->cu_new;
  a.rows = b->new_rows;
  a.tb = tokens_per_block(a.rows);
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
  a.cu = cu_rows;
  a.rows = rows;
  a.tb = tokens_per_block(a.rows);
  const dim3 grid((unsigned)((a.rows + a.tb - 1) / a.tb));
  by_row(dtype, [&](auto out) {
    by_page(c->dtype, [&](auto page) {
      hipLaunchKernelGGL((kv_read_kernel<decltype(page)::value, decltype(out)::value>), grid, dim3(TPB), 0, stream, a);
    });
  });
  MAPA_CHECK_LAUNCH("mapa_kv_cache_read");
  return 0;
}
