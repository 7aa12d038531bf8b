// Rotary positions with several axes (mapa_rope_axes): the general form of mapa_rope2d.  Pair i of axis a turns by
// t = p_a f_i: u' = u cos t - v sin t, v' = v cos t + u sin t; the backward pass is the same turn by -t.
//
// Memory-bound: every value is read and written once, 3 flop per value, and a token's S cosines and sines serve all of
// its heads (both tensors).  A workgroup takes TB tokens: one thread per (token, pair) computes its cosine and sine
// into LDS, then the threads walk the tokens' (head, group of W pairs) items in the tensor's own memory order, 16 B per
// access where sections and strides allow.  A thread keeps its group of pairs for all of its items, so an item costs
// one small division and two LDS address lookups beside its loads.  The angle is formed and reduced to a fraction of a turn in 64 bits (a
// far time times a frequency of one keeps no fraction in 32), then sincospif; per token that is S of them against
// 2 * heads * S values moved.  Measured: queries and keys of 137 thousand tokens, 12 heads each, bf16, 845 MB in 164 us
// (5.15 TB/s; copy: 5.04), of 11 thousand, 15 us (4.5), of 16 alone, 4.3 us; eight items in flight per thread, 16 tokens
// per workgroup and non-temporal accesses were no faster.
#include "mapa_common.h"

namespace {

constexpr int TPB = 256;
constexpr int MAX_TB = 8;

struct RopeArgs {
  const void* x[2];
  void* y[2];
  int64_t xb[2], xh[2], xn[2], yb[2], yh[2], yn[2];
  int heads[2];
  const void* pos;
  int64_t pb, pn, pa;
  int pos_f32, batch, tokens, S, rest, tb, head_major;
  int den;       // items of the inner loop: tb tokens or all heads
  uint32_t div;  // small_div's multiplier of den
  int first[MAPA_ROPE_MAX_AXES + 1];  // first pair of each axis (unused axes: S)
  float sign;
  double turns[MAPA_ROPE_MAX_PAIRS];  // turns per unit of position
};

template <int DT>
struct Elem {
  typedef uint16_t T;
};
template <>
struct Elem<MAPA_F32> {
  typedef float T;
};

template <int BYTES>
struct Word;
template <>
struct Word<2> { typedef uint16_t T; };
template <>
struct Word<4> { typedef uint32_t T; };
template <>
struct Word<8> { typedef uint2 T; };
template <>
struct Word<16> { typedef uint4 T; };

template <int DT>
__device__ __forceinline__ float to_f32(typename Elem<DT>::T v) {
  if constexpr (DT == MAPA_F32) return v;
  else if constexpr (DT == MAPA_F16) return f16_to_f32(v);
  else return bf16_to_f32(v);
}
template <int DT>
__device__ __forceinline__ typename Elem<DT>::T from_f32(float v) {
  if constexpr (DT == MAPA_F32) return v;
  else if constexpr (DT == MAPA_F16) return f32_to_f16(v);
  else return f32_to_bf16(v);
}

template <int DT, int N>
struct Vec {
  typename Elem<DT>::T e[N];
};
template <int DT, int N>
__device__ __forceinline__ Vec<DT, N> ld(const typename Elem<DT>::T* p) {
  typedef typename Word<N * sizeof(typename Elem<DT>::T)>::T W;
  return __builtin_bit_cast(Vec<DT, N>, *reinterpret_cast<const W*>(p));
}
template <int DT, int N>
__device__ __forceinline__ void st(typename Elem<DT>::T* p, const Vec<DT, N>& v) {
  typedef typename Word<N * sizeof(typename Elem<DT>::T)>::T W;
  *reinterpret_cast<W*>(p) = __builtin_bit_cast(W, v);
}

// n / d for 0 <= n < 2^16, 0 < d < 2^14 (m = ceil(2^31 / d))
__device__ __forceinline__ int small_div(int n, uint32_t m) { return (int)__umulhi((uint32_t)n << 1, m); }

// W pairs per item; PAIRED: u and v are neighbours (interleaved columns), one access of 2 W values instead of two of W
template <int DT, int W, bool PAIRED, bool AXIAL>
__global__ void __launch_bounds__(TPB) rope_axes_kernel(RopeArgs a) {
  typedef typename Elem<DT>::T T;
  __shared__ __attribute__((aligned(16))) float cs[MAX_TB * MAPA_ROPE_MAX_PAIRS], sn[MAX_TB * MAPA_ROPE_MAX_PAIRS];
  __shared__ int64_t xat[2][MAX_TB], yat[2][MAX_TB];  // element offsets of the workgroup's tokens
  const int total = a.batch * a.tokens;  // fits (checked on the host)
  const int t0 = blockIdx.x * a.tb;
  const int nt = min(total - t0, a.tb);
  for (int e = threadIdx.x; e < nt * a.S; e += TPB) {
    const int tl = e / a.S, i = e - tl * a.S;
    const int t = t0 + tl, b = t / a.tokens, n = t - b * a.tokens;
    const int ax = (i >= a.first[1]) + (i >= a.first[2]) + (i >= a.first[3]);
    const int64_t at = b * a.pb + n * a.pn + ax * a.pa;
    const double p = a.pos_f32 ? (double)reinterpret_cast<const float*>(a.pos)[at]
                               : (double)reinterpret_cast<const int64_t*>(a.pos)[at];
    if (i == 0) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        xat[w][tl] = b * a.xb[w] + n * a.xn[w];
        yat[w][tl] = b * a.yb[w] + n * a.yn[w];
      }
    }
    const double turn = p * a.turns[i];
    float s, c;
    sincospif(2.f * (float)(turn - rint(turn)), &s, &c);
    cs[tl * a.S + i] = c;
    sn[tl * a.S + i] = a.sign * s;
  }
  __syncthreads();

  // items (token, head) of this thread's group of pairs, walked as the tensor lies in memory: heads inside tokens, or
  // tokens inside heads
  const int heads = a.heads[0] + a.heads[1], groups = a.S / W, rows = TPB / groups;
  const int q0 = threadIdx.x / groups, i = (threadIdx.x - q0 * groups) * W;
  int col = PAIRED ? 2 * i : i, step = a.S;
  if constexpr (AXIAL) {  // the axis' block begins at column 2 first: u at i - first in it, v section columns on
    const int f = i >= a.first[3] ? a.first[3] : i >= a.first[2] ? a.first[2] : i >= a.first[1] ? a.first[1] : 0;
    const int e = i >= a.first[3] ? a.first[4] : i >= a.first[2] ? a.first[3] : i >= a.first[1] ? a.first[2] : a.first[1];
    col = f + i;
    step = e - f;
  }
  auto split = [&](int q, int& tl, int& h) __attribute__((always_inline)) {
    const int outer = small_div(q, a.div), inner = q - outer * a.den;
    tl = a.head_major ? inner : outer;
    h = a.head_major ? outer : inner;
  };
  // (a partial last workgroup walks the places of its missing tokens too, and skips them)
  const int items = a.tb * heads;
  constexpr int U = 4;  // items in flight per thread
  for (int base = q0; base < items && q0 < rows; base += rows * U) {
    Vec<DT, PAIRED ? 2 * W : W> lo[U], hi[U];
    T* out[U];
    int tab[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int q = base + k * rows;
      out[k] = nullptr;
      int tl, h;
      split(q, tl, h);
      if (q < items && tl < nt) {
        const bool w = h >= a.heads[0];
        const int hh = w ? h - a.heads[0] : h;
        const T* src = reinterpret_cast<const T*>(w ? a.x[1] : a.x[0]) + xat[w][tl] + hh * (w ? a.xh[1] : a.xh[0]) + col;
        out[k] = reinterpret_cast<T*>(w ? a.y[1] : a.y[0]) + yat[w][tl] + hh * (w ? a.yh[1] : a.yh[0]) + col;
        tab[k] = tl * a.S + i;
        if constexpr (PAIRED && W == 1) {  // no alignment beyond the element's
          lo[k].e[0] = src[0];
          lo[k].e[1] = src[1];
        } else if constexpr (PAIRED) {
          lo[k] = ld<DT, 2 * W>(src);
        } else {
          lo[k] = ld<DT, W>(src);
          hi[k] = ld<DT, W>(src + step);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (out[k]) {
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const float c = cs[tab[k] + j], s = sn[tab[k] + j];
          T& ur = PAIRED ? lo[k].e[PAIRED ? 2 * j : j] : lo[k].e[j];
          T& vr = PAIRED ? lo[k].e[PAIRED ? 2 * j + 1 : j] : hi[k].e[j];
          const float u = to_f32<DT>(ur), v = to_f32<DT>(vr);
          float nu = __builtin_fmaf(u, c, -(v * s)), nv = __builtin_fmaf(v, c, u * s);
          // fp32 first in every variant: some took an fma that rounds to fp16 at once, so that fp16 results differed by
          // alignment
          if constexpr (DT == MAPA_F16) asm("" : "+v"(nu), "+v"(nv));
          ur = from_f32<DT>(nu);
          vr = from_f32<DT>(nv);
        }
        if constexpr (PAIRED && W == 1) {
          out[k][0] = lo[k].e[0];
          out[k][1] = lo[k].e[1];
        } else if constexpr (PAIRED) {
          st<DT, 2 * W>(out[k], lo[k]);
        } else {
          st<DT, W>(out[k], lo[k]);
          st<DT, W>(out[k] + step, hi[k]);
        }
      }
    }
  }
  // the dims behind the rotated ones, copied (rest is 0 when the tensors are rotated in place)
  for (int it = threadIdx.x; it < items * a.rest; it += TPB) {
    const int q = it / a.rest, c = it - q * a.rest;
    int tl, h;
    split(q, tl, h);
    if (tl >= nt) continue;
    const bool w = h >= a.heads[0];
    const int hh = w ? h - a.heads[0] : h;
    reinterpret_cast<T*>(w ? a.y[1] : a.y[0])[yat[w][tl] + hh * (w ? a.yh[1] : a.yh[0]) + 2 * a.S + c] =
        reinterpret_cast<const T*>(w ? a.x[1] : a.x[0])[xat[w][tl] + hh * (w ? a.xh[1] : a.xh[0]) + 2 * a.S + c];
  }
}

template <int DT, int W, bool PAIRED>
void launch_w(const RopeArgs& a, bool axial, unsigned grid, hipStream_t stream) {
  if (axial)
    hipLaunchKernelGGL((rope_axes_kernel<DT, W, PAIRED, true>), dim3(grid), dim3(TPB), 0, stream, a);
  else
    hipLaunchKernelGGL((rope_axes_kernel<DT, W, PAIRED, false>), dim3(grid), dim3(TPB), 0, stream, a);
}

template <int DT>
void launch(const RopeArgs& a, int layout, int W, unsigned grid, hipStream_t stream) {
  constexpr bool F = DT == MAPA_F32;
  if (layout == MAPA_ROPE_INTERLEAVED) {
    auto go = [&](auto w) {
      hipLaunchKernelGGL((rope_axes_kernel<DT, decltype(w)::value, true, false>), dim3(grid), dim3(TPB), 0, stream, a);
    };
    if (!F && W >= 4) go(std::integral_constant<int, F ? 2 : 4>());
    else if (W >= 2) go(std::integral_constant<int, 2>());
    else go(std::integral_constant<int, 1>());
    return;
  }
  const bool axial = layout == MAPA_ROPE_AXIAL;
  if (!F && W >= 8) launch_w<DT, F ? 4 : 8, false>(a, axial, grid, stream);
  else if (W >= 4) launch_w<DT, 4, false>(a, axial, grid, stream);
  else if (W >= 2) launch_w<DT, 2, false>(a, axial, grid, stream);
  else launch_w<DT, 1, false>(a, axial, grid, stream);
}

}  // namespace

extern "C" int mapa_rope_axes(const mapa_rope_axes_desc* d, hipStream_t stream) {
  MAPA_CHECK_ARG(d != nullptr, "mapa_rope_axes: null descriptor");
  MAPA_CHECK_ARG(d->dtype == MAPA_F32 || d->dtype == MAPA_BF16 || d->dtype == MAPA_F16,
                 "mapa_rope_axes: dtype must be f32, bf16 or f16");
  MAPA_CHECK_ARG(d->batch >= 0 && d->tokens >= 0 && d->head_dim > 0, "mapa_rope_axes: bad shape b=%d n=%d d=%d",
                 d->batch, d->tokens, d->head_dim);
  MAPA_CHECK_ARG(d->axes >= 1 && d->axes <= MAPA_ROPE_MAX_AXES, "mapa_rope_axes: %d axes (1 to %d)", d->axes,
                 MAPA_ROPE_MAX_AXES);
  MAPA_CHECK_ARG(d->layout >= MAPA_ROPE_AXIAL && d->layout <= MAPA_ROPE_INTERLEAVED, "mapa_rope_axes: bad layout");
  MAPA_CHECK_ARG(d->pos_dtype == MAPA_POS_I64 || d->pos_dtype == MAPA_POS_F32, "mapa_rope_axes: bad pos_dtype");
  RopeArgs a = {};
  for (int i = 0; i < d->axes; ++i) {
    MAPA_CHECK_ARG(d->section[i] > 0 && d->section[i] <= MAPA_ROPE_MAX_PAIRS, "mapa_rope_axes: section %d is %d", i,
                   d->section[i]);
    a.first[i + 1] = a.first[i] + d->section[i];
  }
  a.S = a.first[d->axes];
  for (int i = d->axes; i < MAPA_ROPE_MAX_AXES; ++i) a.first[i + 1] = a.S;
  MAPA_CHECK_ARG(a.S <= MAPA_ROPE_MAX_PAIRS && 2 * a.S <= d->head_dim,
                 "mapa_rope_axes: %d pairs do not fit head dim %d (at most %d pairs)", a.S, d->head_dim,
                 MAPA_ROPE_MAX_PAIRS);
  const int64_t total = (int64_t)d->batch * d->tokens;
  bool in_place = true;
  int heads = 0;
  for (int i = 0; i < 2; ++i) {
    MAPA_CHECK_ARG(d->heads[i] >= 0 && d->heads[i] <= 2048, "mapa_rope_axes: bad head count %d (at most 2048)",
                   d->heads[i]);
    a.heads[i] = d->x[i] ? d->heads[i] : 0;
    heads += a.heads[i];
    if (!a.heads[i]) continue;
    MAPA_CHECK_ARG(d->y[i] != nullptr, "mapa_rope_axes: null output");
    a.x[i] = d->x[i];
    a.y[i] = d->y[i];
    a.xb[i] = d->x_bstride[i]; a.xh[i] = d->x_hstride[i]; a.xn[i] = d->x_nstride[i];
    a.yb[i] = d->y_bstride[i]; a.yh[i] = d->y_hstride[i]; a.yn[i] = d->y_nstride[i];
    const bool same = d->x[i] == d->y[i];
    MAPA_CHECK_ARG(!same || (a.xb[i] == a.yb[i] && a.xh[i] == a.yh[i] && a.xn[i] == a.yn[i]),
                   "mapa_rope_axes: in place needs equal strides");
    in_place = in_place && same;
  }
  if (total == 0 || heads == 0) return 0;
  MAPA_CHECK_ARG(!a.heads[0] || !a.heads[1] || a.y[0] != a.y[1], "mapa_rope_axes: both tensors have one output");
  MAPA_CHECK_ARG(d->positions != nullptr, "mapa_rope_axes: null positions");
  MAPA_CHECK_ARG(total <= (int64_t)0x7fffffff, "mapa_rope_axes: too many tokens");
  const int size = d->dtype == MAPA_F32 ? 4 : 2;
  for (int i = 0; i < 2; ++i)
    MAPA_CHECK_ARG(!a.heads[i] || ((uintptr_t)a.x[i] % size == 0 && (uintptr_t)a.y[i] % size == 0),
                   "mapa_rope_axes: base pointers must be aligned to their element");
  // pairs per item: the widest of 16 B per access that every section, stride and base allows
  const bool paired = d->layout == MAPA_ROPE_INTERLEAVED;
  int W = 16 / size / (paired ? 2 : 1);
  for (; W > 1; W /= 2) {
    const int64_t el = paired ? 2 * W : W;
    bool ok = a.S % W == 0;
    if (d->layout == MAPA_ROPE_AXIAL)
      for (int i = 0; i < d->axes; ++i) ok = ok && d->section[i] % W == 0;
    for (int i = 0; i < 2; ++i) {
      if (!a.heads[i]) continue;
      ok = ok && (uintptr_t)a.x[i] % (el * size) == 0 && (uintptr_t)a.y[i] % (el * size) == 0 && a.xb[i] % el == 0 &&
           a.xh[i] % el == 0 && a.xn[i] % el == 0 && a.yb[i] % el == 0 && a.yh[i] % el == 0 && a.yn[i] % el == 0;
    }
    if (ok) break;
  }
  a.pos = d->positions;
  a.pos_f32 = d->pos_dtype == MAPA_POS_F32;
  a.pb = d->pos_bstride; a.pn = d->pos_nstride; a.pa = d->pos_astride;
  a.batch = d->batch;
  a.tokens = d->tokens;
  a.rest = in_place ? 0 : d->head_dim - 2 * a.S;
  a.sign = d->inverse ? -1.f : 1.f;
  for (int i = 0; i < a.S; ++i) a.turns[i] = d->freq[i] * 0.15915494309189533577;  // 1 / (2 pi)
  const int w0 = a.heads[0] ? 0 : 1;
  a.head_major = a.xh[w0] > a.xn[w0];
  a.tb = 1;  // tokens per workgroup: one while that leaves fewer than four workgroups per CU
  while (a.tb < MAX_TB && total / (2 * a.tb) >= 1024) a.tb *= 2;
  a.den = a.head_major ? a.tb : heads;
  a.div = ((1u << 31) + a.den - 1) / a.den;
  const unsigned grid = (unsigned)((total + a.tb - 1) / a.tb);
  if (d->dtype == MAPA_F32) launch<MAPA_F32>(a, d->layout, W, grid, stream);
  else if (d->dtype == MAPA_BF16) launch<MAPA_BF16>(a, d->layout, W, grid, stream);
  else launch<MAPA_F16>(a, d->layout, W, grid, stream);
  MAPA_CHECK_LAUNCH("mapa_rope_axes");
  return 0;
}
