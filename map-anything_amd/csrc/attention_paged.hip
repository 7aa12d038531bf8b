// Attention of new tokens over a paged K/V cache (mapa_attention_paged): head dim 64, grouped heads, bf16 / f16 queries
// over 16-bit, e4m3 or int8 pages, full / causal / block-causal.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp2(c s_ij - m_i),  s_ij = q_i . k_j,  c = scale log2(e),  j < limit(i)
//
// Rows are (new token, query head of the group) pairs, token-major, so that all query heads of a K/V head share its
// tiles.  Q enters the MFMA as it is and c is applied to the fp32 scores: folding c into a 16-bit Q would round it once
// more, which costs as much accuracy as the rounding of the output.  P is rounded to 16 bits as an MFMA operand, its
// sum is not.  The sums' reference m_i is the row's first tile's maximum (2^7 below it in fp16), moved only when a
// tile's sum passes 2^8 (2^15).
//
//  * attn_paged_chunk: 4 or 8 waves x 32 rows over 64-key tiles (as mapa_attention): S^T = K Q^T on 32x32x16 MFMAs, so
//    a lane owns a row and P feeds O^T = V^T P^T without leaving registers.  16-bit pages go to LDS by DMA, 8-bit pages
//    through registers (decoded exactly: code times a power of two), into the same swizzled image.  The softmax's 112
//    vector operations per tile of a wave and its 16 MFMAs share the issue port (70 % busy) at a clock that power holds
//    at 1.6 to 1.9 GHz: 576 Gflop of a 1370-token view over a 100-view scene in 654 us, 0.88 Pflop/s (large matrix
//    product: 1.235).  The pipelined step took it from 723 to 651 us on one card.
//  * attn_paged_step: few rows (single tokens): every wave walks its own 32-key tiles with 16x16x32 MFMAs, K from
//    memory straight into operand registers, V through a wave-private LDS tile for its transpose; no barrier until the
//    four waves are joined.  Memory-bound: 64 scenes' tokens over 556 MB of e4m3 pages 113 us, 4.9 TB/s (copy: 5.04);
//    one token over 11 thousand keys, 34 MB, is a chain of trips to memory instead, 10.9 us and 3.9 for its merge.
//  * keys are cut into ranges of `chunk` when rows alone do not fill the chip; the merge kernels join the fp32 partials
//    in a fixed order (3.9 us of the single token, 11 and 18 us of the chunks above).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged.h"
#include "index_math.h"

namespace {
using namespace mapa_paged;

constexpr int NT = 256;
constexpr int MAX_GROUP = 128;  // query heads per K/V head
constexpr int KT = 64;   // keys of a chunk tile
constexpr int ST = 32;   // keys of a step tile
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
// A row's reference moves when a tile's sum of probabilities passes REBASE_SUM.  In fp16 the reference lies LIFT below the
// row's first maximum and probabilities go up to 2^15: fp16's smallest steps then lose 2^-32 of the row's largest at
// most, not 2^-25.  20 thousand keys 18 below a single one, which weigh 3e-4 together, came out as nothing without it.
template <bool F16>
struct Softmax {
  static constexpr float LIFT = F16 ? 7.f : 0.f;  // log2
  static constexpr float REBASE_SUM = F16 ? 32768.f : 256.f;
};

struct PagedArgs {
  const char* page[2];  // K, V
  const uint8_t* exp[2];
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* cu;
  const uint16_t* q;
  uint16_t* o;
  float* lse;
  int64_t qr, qh, orr, oh;
  float* part_o;    // [slot][rows of a workgroup][64], normalised
  float* part_lse;  // [slot][rows of a workgroup], log2 domain
  unsigned* fault;
  float c;  // scale * log2(e)
  int seqs, table_stride, new_rows, max_new, cap, num_pages, psl;
  int heads, kv_heads, group;
  int block;    // mask_block
  int splits, chunk;  // key ranges of a split task, keys of a range
  int whole;     // tasks [0, whole) of the chunk kernel walk all their keys, the others are split
  int tiles;     // row tiles of the grid (upper bound)
  int per_tile;  // tokens of a row tile
  int slot_rows; // rows of a chunk slot
  int tile_passes, range_passes;  // passes over a head's row tiles and key ranges
};

typedef short s4v __attribute__((ext_vector_type(4)));
typedef short s8v __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;

typedef int i4v __attribute__((ext_vector_type(4)));

// 16 B per lane from a buffer into LDS at lds + 16 lane, lanes past the buffer's end as zeros.  In asm so that the
// compiler, which takes any LDS-DMA in flight for a writer of what a transposed LDS read reads, does not wait for it
// there: it has no register output, and its completion is waited for by hand before the barrier that precedes the reads.
// The five wait states before the load cover an operand SGPR that a vector instruction wrote just before (and M0, which
// nothing else in these kernels uses).
__device__ __forceinline__ void lds_dma16(i4v rsrc, int voffset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds"
               :: "v"(voffset), "s"(rsrc), "s"(lds) : "memory");
}

__device__ __forceinline__ s4v tr_read(const char* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v*)(p));
}

// keys that a query at position pos sees
__device__ __forceinline__ int key_limit(int pos, int len, int block) {
  if (block == 0) return len;
  if (pos < 0) return 0;
  const int64_t end = ((int64_t)(pos / block) + 1) * block;
  return end < len ? (int)end : len;
}

// New tokens of sequence b: its row interval, checked
__device__ __forceinline__ int new_tokens(const PagedArgs& p, int c0, int c1) {
  if (c0 < 0 || c1 < c0 || c1 > p.new_rows || c1 - c0 > p.max_new) {
    kv_fault(p.fault);
    return 0;
  }
  return c1 - c0;
}

template <bool F16>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (F16) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});  // v_cvt_pk_f16_f32
  } else {
    return pack_bf16x2(a, b);
  }
}

// 8 codes -> 8 operand words of the query's type, times the row's power of two s (exact unless it leaves the type);
// e4m3 pairs have an instruction that scales as it converts
template <bool F16, bool I8>
__device__ __forceinline__ bf16x8 decode8(uint2 w, float s) {
  if constexpr (I8) {
    const f32x4 a = decode4<true>(w.x, s), b = decode4<true>(w.y, s);
    return __builtin_bit_cast(bf16x8, uint4{pack16<F16>(a[0], a[1]), pack16<F16>(a[2], a[3]), pack16<F16>(b[0], b[1]),
                                            pack16<F16>(b[2], b[3])});
  } else if constexpr (F16) {
    return __builtin_bit_cast(
        bf16x8, uint4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, s, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, s, true))});
  } else {
    return __builtin_bit_cast(
        bf16x8, uint4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, s, true)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, s, false)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, s, true))});
  }
}

// Bits 15 and 31 of the result: whether any of 8 operand words is an infinity or a NaN (an exponent of all ones carries)
template <bool F16>
__device__ __forceinline__ uint32_t special_bits(uint32_t w) {
  constexpr uint32_t E = F16 ? 0x7c007c00u : 0x7f807f80u, ONE = F16 ? 0x04000400u : 0x00800080u;
  return ((w & E) + ONE) & 0x80008000u;
}
template <bool F16>
__device__ __forceinline__ uint32_t special_bits(bf16x8 v) {
  const uint4 u = __builtin_bit_cast(uint4, v);
  return special_bits<F16>(u.x) | special_bits<F16>(u.y) | special_bits<F16>(u.z) | special_bits<F16>(u.w);
}
// 8 operand words with zeros for the infinities and NaNs (SPECIAL: for all others)
template <bool F16, bool SPECIAL>
__device__ __forceinline__ bf16x8 part_of(bf16x8 v) {
  const uint4 u = __builtin_bit_cast(uint4, v);
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = special_bits<F16>(w[i]), m = (b - (b >> 15)) | b;  // 16 ones for each
    w[i] &= SPECIAL ? m : ~m;
  }
  return __builtin_bit_cast(bf16x8, uint4{w[0], w[1], w[2], w[3]});
}
// element j of 8 operand words if `on`, the others zero
__device__ __forceinline__ bf16x8 only(bf16x8 v, int j, bool on) {
  const uint4 u = __builtin_bit_cast(uint4, v);
  const uint32_t m = !on ? 0u : (j & 1) ? 0xffff0000u : 0xffffu;
  const int w = j >> 1;
  const uint4 r = {w == 0 ? u.x & m : 0u, w == 1 ? u.y & m : 0u, w == 2 ? u.z & m : 0u, w == 3 ? u.w & m : 0u};
  return __builtin_bit_cast(bf16x8, r);
}

// A row's sum l over the keys it sees, at the reference m (log2 domain), is positive unless all their scores are -inf.
// The whole row is 0 / 0 = NaN then; a range of it (part) leaves zeros and a logarithm of -inf, which weigh nothing beside
// the other ranges.
__device__ __forceinline__ float range_inverse(float l, bool part) { return part && l == 0.f ? 1.f : 1.f / l; }
__device__ __forceinline__ float range_lse(float m, float l, bool part) {
  return l > 0.f ? m + __log2f(l) : part && l == 0.f ? -INFINITY : __builtin_nanf("");
}

// Row tile of the chunk kernel -> (sequence, its first packed row, its new and its cached tokens, tile in it), by a
// wave-wide prefix sum over the sequences' tile counts, 64 at a time; seq -1: no such tile.
struct RowTile {
  int seq, c0, nq, len, tile;
};
__device__ __forceinline__ RowTile find_tile(const PagedArgs& p, int tile, int lane) {
  int before = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < p.seqs; s0 += 64) {
    const int s = s0 + lane;
    int q0 = 0, n = 0, len = 0;
    if (s < p.seqs) {
      q0 = p.cu[s];
      len = p.kv_lens[s];
      n = new_tokens(p, q0, p.cu[s + 1]);
      len = checked_len(len, p.cap, p.fault);
    }
    int sum = (n + p.per_tile - 1) / p.per_tile;
    const int own = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(sum, o, 64);
      if (lane >= o) sum += up;
    }
    const uint64_t past = __ballot(before + sum > tile);
    if (past) {
      const int l = __builtin_ctzll(past);
      return RowTile{s0 + l, __builtin_amdgcn_readlane(q0, l), __builtin_amdgcn_readlane(n, l),
                     __builtin_amdgcn_readlane(len, l), tile - before - __builtin_amdgcn_readlane(sum - own, l)};
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return RowTile{-1, 0, 0, 0, 0};
}

// ------------------------------------------------------------------------------------------------ chunk
// CK: 0 = 16-bit pages of the query's type, 1 = e4m3, 2 = int8.  NW: waves of a workgroup, 32 rows each (the plan's rule
// and both sides' figures are at chunk_waves).
template <bool F16, int CK, int NW>
__global__ void __launch_bounds__(NW * 64, 2) attn_paged_chunk(PagedArgs p) {
  constexpr int QB = NW * 32;
  constexpr int PIECES = 8 / NW;  // 8-row pieces of a 64-row tile per wave
  constexpr int TILE = KT * 128;  // 64 rows x 128 B
  __shared__ __attribute__((aligned(1024))) char lds[2 * 2 * TILE];  // K by tile parity, then V
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, l32 = lane & 31;

  int task, split, slot, hk, tile;
  mapa_idx::paged_chunk_work(blockIdx.x, p.whole, p.tiles, p.kv_heads, p.splits, p.range_passes, task, split, slot);
  mapa_idx::paged_task(task, p.tiles, p.tile_passes, hk, tile);
  const RowTile rt0 = find_tile(p, tile, lane);
  const int b = rt0.seq, nq = rt0.nq, c0 = rt0.c0, len = rt0.len;
  tile = rt0.tile;
  if (b < 0) return;
  const int t0 = tile * p.per_tile;                       // first token of the tile, in its sequence
  const int rows = min(p.per_tile, nq - t0) * p.group;    // rows of the tile
  const int pos0 = len - nq + t0;                         // position of the first token
  const int lim_lo = key_limit(pos0, len, p.block);
  const int lim_hi = key_limit(pos0 + (rows - 1) / p.group, len, p.block);
  if (lim_hi <= p.chunk && split == 0) slot = -1;  // one range holds all of the tile's keys: no partials
  const int k_begin = split * p.chunk, k_end = slot < 0 ? lim_hi : min(k_begin + p.chunk, lim_hi);

  // this lane's row
  const int r = wave * 32 + l32;
  const int rc = min(r, rows - 1);
  const int rt = rc / p.group, rg = rc - rt * p.group;
  const int tok = c0 + t0 + rt, head = hk * p.group + rg;
  const int limit = key_limit(pos0 + rt, len, p.block);
  if (k_begin >= k_end) {  // no key of this range is seen by any row of the tile (the merge knows which ranges are)
    if (slot < 0 && r < rows) {
      uint16_t* o = p.o + (int64_t)tok * p.orr + head * p.oh + hl * 32;
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<uint4*>(o)[i] = uint4{0, 0, 0, 0};
      if (p.lse && hl == 0) p.lse[(int64_t)head * p.new_rows + tok] = -INFINITY;
    }
    return;
  }
  const int kt0 = k_begin / KT, kt1 = (k_end + KT - 1) / KT;
  const int kt_free = min(lim_lo, k_end) / KT;  // tiles below: every key seen by every row

  bf16x8 qf[4];
  {
    const uint16_t* q = p.q + (int64_t)tok * p.qr + head * p.qh;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qf[kk] = *reinterpret_cast<const bf16x8*>(q + kk * 16 + 8 * hl);
  }

  // Places.  A wave fetches NA pieces of every tile's K and of its V: of 16-bit pages 8 rows each, of 8-bit pages 16.
  // Lane i holds where piece i % NA of tile wt0 + i / NA begins in the cache (in bytes for 16-bit pages, in rows for
  // codes and their exponents), so that a piece's place is two v_readlanes away from being scalar (a view over a
  // 100-view scene: 655 us with this arithmetic in scalar instructions per tile, 647 so).  The next 64 pieces' pages are
  // fetched a window ahead.  Pieces past the sequence's last page get page 0: what they bring is hidden.
  constexpr int NA = CK == 0 ? PIECES : 1;
  const int32_t* trow = p.table + (int64_t)b * p.table_stride;
  const int pages = (len + (1 << p.psl) - 1) >> p.psl;
  int wt0 = kt0, raw;  // raw: the table's entries of the window after
  int64_t win;
  const int lane_key = lane * (KT / NA) + (CK == 0 ? wave * 8 : (wave & 3) * 16);
  auto fetch_raw = [&](int t) __attribute__((always_inline)) {
    const int lp = (t * KT + lane_key) >> p.psl;
    raw = lp < pages ? trow[lp] : 0;
  };
  auto set_window = [&]() __attribute__((always_inline)) {
    const int64_t row = (int64_t)checked_page(raw, p.num_pages, p.fault) * p.kv_heads + hk;
    win = ((row << p.psl) + ((wt0 * KT + lane_key) & ((1 << p.psl) - 1))) * (CK == 0 ? 128 : 1);
    fetch_raw(wt0 + 64 / NA);
  };
  fetch_raw(wt0);
  set_window();

  // Staging.  A tile's K is needed one step before its V, so step t brings K of tile t + 2 and V of tile t; the V rows'
  // place in the cache is K's of two steps ago (`at`, by tile parity).  Tile numbers past the range are clamped: what
  // they bring is not used.
  //  * 16-bit pages: a wave moves 8-row pieces of K and of V (8 rows x 128 B lie in one page: a scalar base and a fixed
  //    offset per lane), the 16-B column XOR-swizzled on the source so that the LDS image stays lane-linear.  V's buffer
  //    ends where the sequence does, so that rows past it arrive as zeros: whatever their memory holds must not meet a
  //    zero probability (hidden scores are replaced, so K needs no such care).
  //  * 8-bit pages: four waves take a tile's 64 rows, four lanes a row of 16 codes each, fetched a step earlier and
  //    decoded on the way into LDS; of eight waves, four take K and four V.
  int64_t at[2][NA];
  const int prow8 = lane >> 3;
  const int koff = prow8 * 128 + (((lane & 7) ^ (((wave & 1) * 4 + (lane >> 4)) & 7)) << 4);
  const int voff = prow8 * 128 + (((lane & 7) ^ (((lane >> 4) & 1) << 2)) << 4);
  auto place = [&](int kt, auto par_tag) __attribute__((always_inline)) {
    constexpr int par = decltype(par_tag)::value;
    if (__builtin_expect(kt - wt0 >= 64 / NA, 0)) {
      wt0 += 64 / NA;
      set_window();
    }
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int l = (kt - wt0) * NA + i;
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)win, l);
      const uint32_t hi = __builtin_amdgcn_readlane((int)(win >> 32), l);
      at[par][i] = (int64_t)(((uint64_t)hi << 32) | lo);
    }
  };
  const uint32_t lds_base = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
  auto dma = [&](auto x_tag, int kt, auto par_tag, auto full_tag) __attribute__((always_inline)) {  // x: 0 K, 1 V
    constexpr int x = decltype(x_tag)::value, par = decltype(par_tag)::value;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int k8 = (i * NW + wave) * 8;
      int bytes = 1024;
      if constexpr (x == 1 && !decltype(full_tag)::value) {
        const int rows_left = len - kt * KT - k8;
        bytes = rows_left >= 8 ? 1024 : rows_left > 0 ? rows_left * 128 : 0;
      }
      const uint64_t base = (uint64_t)(p.page[x] + at[par][i]);
      lds_dma16(i4v{(int)(uint32_t)base, (int)(base >> 32), bytes, 0x00020000}, x == 0 ? koff : voff,
                lds_base + (2 * x + par) * TILE + k8 * 128);
    }
  };
  uint4 creg[2] = {};
  uint32_t ereg[2] = {};
  // x: 0 K, 1 V; r: register set
  auto fetch8 = [&](int x, int r, auto par_tag) __attribute__((always_inline)) {
    constexpr int par = decltype(par_tag)::value;
    const char* page = x == 0 ? p.page[0] : p.page[1];
    const uint8_t* exp = x == 0 ? p.exp[0] : p.exp[1];
    creg[r] = reinterpret_cast<const uint4*>(page + at[par][0] * 64)[lane];
    ereg[r] = (exp + at[par][0])[lane >> 2];
  };
  auto store8 = [&](int x, int r, int kt, auto par_tag) __attribute__((always_inline)) {
    constexpr int par = decltype(par_tag)::value;
    char* dst = lds + (2 * x + par) * TILE;
    const int row = (tid & 255) >> 2, ch = (lane & 3) * 2;
    const float s = exponent_value(ereg[r]);
    bf16x8 lo = decode8<F16, CK == 2>(uint2{creg[r].x, creg[r].y}, s);
    bf16x8 hi = decode8<F16, CK == 2>(uint2{creg[r].z, creg[r].w}, s);
    if (kt * KT + row >= len) lo = hi = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
    const int sw = x == 0 ? (row >> 1) & 7 : ((row >> 1) & 1) << 2;
    *reinterpret_cast<bf16x8*>(dst + row * 128 + ((ch ^ sw) << 4)) = lo;
    *reinterpret_cast<bf16x8*>(dst + row * 128 + (((ch + 1) ^ sw) << 4)) = hi;
  };
  // eight waves: this wave's tensor, and its tile that step t stores (K t + 2, V t) and fetches (one further)
  const int mine = wave >> 2;
  auto tile_of = [&](int t) __attribute__((always_inline)) { return mine == 0 ? t + 2 : t; };
  using T_ = std::integral_constant<bool, true>;
  using F_ = std::integral_constant<bool, false>;
  using P0 = std::integral_constant<int, 0>;
  using P1 = std::integral_constant<int, 1>;
  // the steps' barrier: this wave's DMA has landed and its LDS accesses are done
  auto step_barrier = [&]() __attribute__((always_inline)) {
    if constexpr (CK == 0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  place(kt0, P0());
  if constexpr (CK == 0) {
    dma(P0(), kt0, P0(), F_());
    place(min(kt0 + 1, kt1 - 1), P1());
    dma(P0(), kt0 + 1, P1(), F_());
  } else if constexpr (NW == 4) {
    fetch8(0, 0, P0());
    store8(0, 0, kt0, P0());
    place(min(kt0 + 1, kt1 - 1), P1());
    fetch8(0, 0, P1());
    fetch8(1, 1, P0());
    store8(0, 0, kt0 + 1, P1());
    place(min(kt0 + 2, kt1 - 1), P0());
    fetch8(0, 0, P0());
  } else {
    if (mine == 0) {
      fetch8(0, 0, P0());
      place(min(kt0 + 1, kt1 - 1), P1());
      fetch8(0, 1, P1());
      store8(0, 0, kt0, P0());
      store8(0, 1, kt0 + 1, P1());
    }
    place(min(tile_of(kt0), kt1 - 1), P0());
    fetch8(mine, 0, P0());
  }

  f32x16 o[2], st[2][2];  // output rows; scores by tile parity
  bf16x8 pf[4];           // probabilities of the tile before, waiting for its V
#pragma unroll
  for (int d = 0; d < 2; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  float m_ref = 0.f, l_run = 0.f;
  const float c = p.c;

  // K fragment: keys 32 kb + l32, dims 16 kk + 8 hl ..; V^T fragment: dims 32 dt + l32, keys 16 f + 8 (j / 4) + 4 hl + j % 4
  // (transposed LDS reads), the order in which the scores come out of K Q^T
  auto k_frag = [&](const char* Ks, int kb, int kk) __attribute__((always_inline)) {
    const int row = kb * 32 + l32;
    return *reinterpret_cast<const bf16x8*>(Ks + row * 128 + (((kk * 2 + hl) ^ ((row >> 1) & 7)) << 4));
  };
  auto v_frag = [&](const char* Vs, int dt, int f) __attribute__((always_inline)) {
    const int i4 = lane & 15, q4 = i4 >> 2, p4 = i4 & 3, grp = (lane >> 4) & 1;
    const int cc = dt * 32 + 16 * grp + 4 * p4, ch = cc >> 3, within = (cc & 7) * 2;
    const int R0 = 16 * f + 4 * hl + q4, R1 = R0 + 8;
    const s4v lo = tr_read(Vs + R0 * 128 + ((ch ^ (((R0 >> 1) & 1) << 2)) << 4) + within);
    const s4v hi = tr_read(Vs + R1 * 128 + ((ch ^ (((R1 >> 1) & 1) << 2)) << 4) + within);
    return (bf16x8)s8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  auto row_max = [&](const f32x16* s) __attribute__((always_inline)) {
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
    return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * c;
  };
  auto hide = [&](f32x16* s, int kt) __attribute__((always_inline)) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = kt * KT + kb * 32 + (i & 3) + 8 * (i >> 2) + 4 * hl;
        s[kb][i] = key < limit ? s[kb][i] : -INFINITY;
      }
  };
  // O^T += V^T P^T of tile kt, with a look at V first: an infinity or NaN of a key that some rows do not see, times
  // their zero probability, must not reach them.  The product takes zeros in their place (so that a row's sum is formed
  // the same way whatever its hidden keys hold), and they are added key by key, where they are seen.
  auto pv_checked = [&](const char* Vs, int kt) __attribute__((always_inline)) {
    bf16x8 vf[2][4];
    uint32_t bits = 0;
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
      for (int dt = 0; dt < 2; ++dt) {
        vf[dt][f] = v_frag(Vs, dt, f);
        bits |= special_bits<F16>(vf[dt][f]);
      }
    const bool special = __any(bits != 0);
    if (__builtin_expect(special, 0)) {
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) vf[dt][f] = part_of<F16, false>(vf[dt][f]);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f)
#pragma unroll
      for (int dt = 0; dt < 2; ++dt) o[dt] = mfma32x32x16<F16>(vf[dt][f], pf[f], o[dt]);
    if (__builtin_expect(special, 0)) {
      asm volatile("" ::: "memory");  // the fragments are read again: kept over the product, they would spill
      const bf16x8 p0 = pf[0], p1 = pf[1], p2 = pf[2], p3 = pf[3];
#pragma unroll
      for (int dt = 0; dt < 2; ++dt)
#pragma unroll 1
        for (int fj = 0; fj < 64; ++fj) {
          const int f = fj >> 4, j = fj & 7, h2 = (fj >> 3) & 1;
          const int key = kt * KT + 16 * f + (j & 3) + 8 * (j >> 2) + 4 * h2;
          const bf16x8 pr = f == 0 ? p0 : f == 1 ? p1 : f == 2 ? p2 : p3;
          // (the transposed read takes no notice of EXEC: all lanes read, in no branch)
          const bf16x8 vs = part_of<F16, true>(v_frag(Vs, dt, f));
          const bf16x8 pk = only(pr, j, hl == h2), vk = only(vs, j, hl == h2);
          f32x16 t;
#pragma unroll
          for (int i = 0; i < 16; ++i) t[i] = 0.f;
          t = mfma32x32x16<F16>(vk, pk, t);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[dt][i] = key < limit ? o[dt][i] + t[i] : o[dt][i];
        }
    }
  };

  // Step t (parity PAR): the softmax of tile t's scores, the products K Q^T of tile t + 1 and V^T P^T of tile t - 1.
  // The two MFMA chains and the softmax are independent, so the matrix unit runs under the exponentials: 16 MFMAs of 32
  // cycles between 16 groups of two scores (2 fma, 2 exp, 2 add, 1 conversion: 36 cycles).
  auto step = [&](int t, auto first_tag, auto mask_tag, auto par_tag) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(first_tag)::value;
    constexpr bool MASK = decltype(mask_tag)::value;
    constexpr int par = decltype(par_tag)::value, nxt = par ^ 1;
    using PN = std::integral_constant<int, nxt>;
    f32x16(&s)[2] = st[par];
    f32x16(&sn)[2] = st[nxt];
    const char* Ks = lds + nxt * TILE;        // K of tile t + 1
    const char* Vs = lds + (2 + nxt) * TILE;  // V of tile t - 1
    constexpr bool PV = !MASK && !FIRST;
    bf16x8 kf[2][2], vf[2][2];
    auto frags = [&](int i) __attribute__((always_inline)) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        kf[i & 1][x] = k_frag(Ks, x, i);
        if constexpr (PV) vf[i & 1][x] = v_frag(Vs, x, i);
      }
    };
    frags(0);
    if constexpr (CK == 0) {
      dma(P1(), t, par_tag, std::integral_constant<bool, !MASK>());
      place(min(t + 2, kt1 - 1), par_tag);
      dma(P0(), t + 2, par_tag, F_());
    } else {
      if constexpr (NW == 4) {
        store8(1, 1, t, par_tag);
        store8(0, 0, t + 2, par_tag);
        fetch8(1, 1, PN());
        place(min(t + 3, kt1 - 1), PN());
        fetch8(0, 0, PN());
      } else {
        store8(mine, 0, tile_of(t), par_tag);
        place(min(tile_of(t + 1), kt1 - 1), PN());
        fetch8(mine, 0, PN());
      }
    }
    if constexpr (MASK) hide(s, t);
    // finite also for a row that sees none of the range
    if constexpr (FIRST) m_ref = fmaxf(row_max(s), -1e38f) - Softmax<F16>::LIFT;
    const float nm = -m_ref;
    if constexpr (MASK && !FIRST) pv_checked(Vs, t - 1);
    // Group n: MFMA n; the exponents of scores 2n, 2n + 1; behind them the sums and the conversion of the two before,
    // ahead the fma of the two after (an exponential's result is late).  Scores in register order: key block, then
    // accumulator element, which is the order of P's fragments.
    float a[4] = {0.f, 0.f, 0.f, 0.f}, x[2], e[2], y[2];
    uint32_t pk[4];
    x[0] = __builtin_fmaf(s[0][0], c, nm);
    x[1] = __builtin_fmaf(s[0][1], c, nm);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 17; ++n) {
      const int i = n >> 2, g = n & 3;
      if (n < 16) {
        if (g < 2) {
          if (i == 0) {
#pragma unroll
            for (int z = 0; z < 16; ++z) sn[g][z] = 0.f;
          }
          sn[g] = mfma32x32x16<F16>(kf[i & 1][g], qf[i], sn[g]);
        } else if constexpr (PV) {
          o[g - 2] = mfma32x32x16<F16>(vf[i & 1][g - 2], pf[i], o[g - 2]);
        }
        if (g == 0 && i < 3) frags(i + 1);
        e[0] = __builtin_amdgcn_exp2f(x[0]);
        e[1] = __builtin_amdgcn_exp2f(x[1]);
        if (n < 15) {
          x[0] = __builtin_fmaf(s[(2 * n + 2) >> 4][(2 * n + 2) & 15], c, nm);
          x[1] = __builtin_fmaf(s[(2 * n + 3) >> 4][(2 * n + 3) & 15], c, nm);
        }
      }
      if (n > 0) {
        const int b2 = 2 * ((n - 1) & 1);
        a[b2] = n < 3 ? y[0] : a[b2] + y[0];
        a[b2 + 1] = n < 3 ? y[1] : a[b2 + 1] + y[1];
        pk[(n - 1) & 3] = pack16<F16>(y[0], y[1]);
        asm volatile("" : "+v"(pk[(n - 1) & 3]));  // here, not sunk behind the check below
        if (((n - 1) & 3) == 3) pf[(n - 1) >> 2] = __builtin_bit_cast(bf16x8, uint4{pk[0], pk[1], pk[2], pk[3]});
      }
      y[0] = e[0];
      y[1] = e[1];
      __builtin_amdgcn_sched_barrier(0);
    }
    float ls = (a[0] + a[1]) + (a[2] + a[3]);
    if constexpr (!FIRST) {
      const uint64_t over = __ballot(!(ls <= Softmax<F16>::REBASE_SUM));  // NaN rebases too
      if (__builtin_expect(over != 0, 0)) {
        // a row (its two lanes) moves its reference by its own scores: the wave's other rows compute what they have again.
        // The maximum exchanges values between lanes, so all of them take part in it (kept out of a branch by the asm).
        const bool mine = ((over | over << 32 | over >> 32) >> lane) & 1;
        float m = fmaxf(row_max(s) - Softmax<F16>::LIFT, m_ref);
        asm volatile("" : "+v"(m));
        m = mine ? m : m_ref;
        const float alpha = __builtin_amdgcn_exp2f(m_ref - m);
        m_ref = m;
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < 2; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[dt][i] *= alpha;
        float again = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t pk[4];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int e = 8 * (i & 1) + 2 * g;
            const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 1][e], c, -m));
            const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 1][e + 1], c, -m));
            again += e0 + e1;
            pk[g] = pack16<F16>(e0, e1);
          }
          pf[i] = __builtin_bit_cast(bf16x8, uint4{pk[0], pk[1], pk[2], pk[3]});
        }
        asm volatile("" : "+v"(again));
        ls = mine ? again : ls;
      }
    }
    l_run += ls;
    step_barrier();
  };

  step_barrier();
#pragma unroll
  for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
    for (int i = 0; i < 16; ++i) st[0][kb][i] = 0.f;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) st[0][kb] = mfma32x32x16<F16>(k_frag(lds, kb, kk), qf[kk], st[0][kb]);
  }
  step_barrier();  // K of the first tile is read: its slot is free
  // Nothing is in flight here.  The compiler does not see that in the asm above: without its own wait it may put one for
  // Q's loads into the loop, where it waits for the step's DMA (5 % of a view over a 100-view scene)
  if constexpr (CK == 0) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  int kt = kt0;
  if (kt < kt_free) step(kt, T_(), F_(), P0());
  else step(kt, T_(), T_(), P0());
  ++kt;
#pragma unroll 1
  for (; kt + 1 < kt_free; kt += 2) {
    step(kt, F_(), F_(), P1());
    step(kt + 1, F_(), F_(), P0());
  }
  // the rest: at most one more free tile, then the masked ones (an extra mask on a free tile changes nothing)
#pragma unroll 1
  for (; kt < kt1; kt += 2) {
    step(kt, F_(), T_(), P1());
    if (kt + 1 < kt1) step(kt + 1, F_(), T_(), P0());
  }
  pv_checked(lds + (2 + ((kt1 - 1 - kt0) & 1)) * TILE, kt1 - 1);

  const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
  const bool seen = limit > k_begin;
  const bool part = slot >= 0;
  const float inv = !seen ? 0.f : range_inverse(l_tot, part);
  const float lse2 = !seen ? -INFINITY : range_lse(m_ref, l_tot, part);
  if (!seen) {
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
  }
  if (slot < 0) {
    uint16_t* obase = p.o + (int64_t)tok * p.orr + head * p.oh;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int gp = 0; gp < 2; ++gp) {  // 16-B row segments out of the two half-lanes' 8-B pieces
        uint32_t y[2], x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          y[i] = pack16<F16>(o[dt][8 * gp + 2 * i] * inv, o[dt][8 * gp + 2 * i + 1] * inv);
          x[i] = pack16<F16>(o[dt][8 * gp + 4 + 2 * i] * inv, o[dt][8 * gp + 4 + 2 * i + 1] * inv);
          const auto sw = __builtin_amdgcn_permlane32_swap(y[i], x[i], false, false);
          y[i] = sw[0];
          x[i] = sw[1];
        }
        if (r < rows) *reinterpret_cast<uint4*>(obase + dt * 32 + 16 * gp + 8 * hl) = uint4{y[0], y[1], x[0], x[1]};
      }
    if (p.lse && r < rows && hl == 0) p.lse[(int64_t)head * p.new_rows + tok] = lse2 * LN2;
  } else if (r < rows) {
    const int64_t prow = (int64_t)slot * QB + r;
    float* po = p.part_o + prow * HD;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(po + dt * 32 + 8 * g + 4 * hl) =
            f32x4{o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv, o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv};
    if (hl == 0) p.part_lse[prow] = lse2;
  }
}

// ------------------------------------------------------------------------------------------------ step
// RB blocks of 16 rows (new tokens x query heads of the group) per workgroup; each of the 4 waves walks every fourth
// 32-key tile of the workgroup's key range.
template <bool F16, int CK, int RB>
__global__ void __launch_bounds__(NT, 2) attn_paged_step(PagedArgs p) {
  constexpr int VT = ST * 128;  // V tile of a wave
  constexpr int RS = RB * 16;   // rows
  constexpr int JOIN = 4 * RS * HD * 4;
  __shared__ __attribute__((aligned(1024))) char lds[JOIN > 4 * VT ? JOIN : 4 * VT];
  __shared__ float join_m[4][RS], join_l[4][RS];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, l16 = lane & 15;

  int b, split, hk;
  mapa_idx::paged_step_work(blockIdx.x, p.kv_heads, p.splits, b, split, hk);
  // The page window and, for one sequence alone, the first tiles are fetched before its length is known (the range's
  // place is not a matter of it; what lies past the sequence is hidden later): one trip to memory less in a chain of
  // four.  Of several sequences most ranges may be past the end, and other workgroups cover the wait.  Pages are held
  // within the cache here and reported once the length says which of them are the sequence's.
  const int32_t* trow = p.table + (int64_t)b * p.table_stride;
  const int k_begin = split * p.chunk;
  const int pmask = (1 << p.psl) - 1;
  const int64_t page_rows = (int64_t)p.kv_heads << p.psl, head_rows = (int64_t)hk << p.psl;
  int w0 = k_begin >> p.psl, raw = 0;
  int64_t win;
  auto fetch_window = [&]() __attribute__((always_inline)) {
    raw = w0 + lane < p.table_stride ? trow[w0 + lane] : 0;
    win = (int64_t)((unsigned)raw < (unsigned)p.num_pages ? raw : 0) * page_rows + head_rows;
  };
  fetch_window();
  // row of the cache (head hk) of a 16-row-aligned key of the window
  auto cache_row = [&](int key) __attribute__((always_inline)) {
    const int i = min(key >> p.psl, p.table_stride - 1) - w0;
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)win, i);
    const int hi = __builtin_amdgcn_readlane((int)(win >> 32), i);
    return (int64_t)(((uint64_t)(uint32_t)hi << 32) | lo) + (key & pmask);
  };
  struct Tile {
    uint4 k[CK == 0 ? 4 : 2];  // 16-bit: [key block][32 dims]; codes: [key block]
    uint4 v[CK == 0 ? 4 : 2];  // 16-bit: rows 8 i + lane / 8; codes: rows 16 i + lane / 4
    uint32_t ke[2], ve[2];
  };
  auto load_tile = [&](Tile& t, int key0) __attribute__((always_inline)) {  // a tile of the window
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int64_t at = cache_row(key0 + 16 * kb);
      if constexpr (CK == 0) {
        const char* kp = p.page[0] + (at + l16) * 128 + g * 16;
        t.k[2 * kb] = *reinterpret_cast<const uint4*>(kp);
        t.k[2 * kb + 1] = *reinterpret_cast<const uint4*>(kp + 64);
        const char* vp = p.page[1] + (at + (lane >> 3)) * 128 + (lane & 7) * 16;
        t.v[2 * kb] = *reinterpret_cast<const uint4*>(vp);
        t.v[2 * kb + 1] = *reinterpret_cast<const uint4*>(vp + 8 * 128);
      } else {
        t.k[kb] = *reinterpret_cast<const uint4*>(p.page[0] + (at + l16) * 64 + g * 16);
        t.ke[kb] = p.exp[0][at + l16];
        t.v[kb] = *reinterpret_cast<const uint4*>(p.page[1] + (at + (lane >> 2)) * 64 + (lane & 3) * 16);
        t.ve[kb] = p.exp[1][at + (lane >> 2)];
      }
    }
  };

  constexpr int STEP = 4 * ST;
  Tile ta, tb;
  int key = k_begin + wave * ST;
  // (a window has at least 64 pages of 16 rows: the range's first eight tiles are in it)
  const bool early = p.seqs == 1 && p.table_stride > 0;
  if (early) {
    load_tile(ta, key);
    if (p.chunk > STEP) load_tile(tb, key + STEP);
  }
  const int c0 = p.cu[b];
  const int nq = new_tokens(p, c0, p.cu[b + 1]);
  const int len = checked_len(p.kv_lens[b], p.cap, p.fault);
  const int rows = nq * p.group;
  if (rows == 0) return;
  const int pos0 = len - nq;
  const int lim_lo = key_limit(pos0, len, p.block), lim_hi = key_limit(len - 1, len, p.block);
  const int k_end = min(k_begin + p.chunk, lim_hi);

  int limit[RB], tok[RB], head[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = min(rb * 16 + l16, rows - 1);
    const int rt = r / p.group;
    tok[rb] = c0 + rt;
    head[rb] = hk * p.group + r - rt * p.group;
    limit[rb] = key_limit(pos0 + rt, len, p.block);
  }
  if (k_begin >= k_end) {  // uniform: the whole workgroup leaves (the merge knows which ranges are empty)
    for (int i = tid; split == 0 && i < rows * 8; i += NT) {
      const int r = i >> 3, rt = r / p.group, h = hk * p.group + r - rt * p.group, t = c0 + rt;
      reinterpret_cast<uint4*>(p.o + (int64_t)t * p.orr + h * p.oh)[i & 7] = uint4{0, 0, 0, 0};
      if (p.lse && (i & 7) == 0) p.lse[(int64_t)h * p.new_rows + t] = -INFINITY;
    }
    return;
  }

  const int pages = (len + (1 << p.psl) - 1) >> p.psl;
  auto report_pages = [&]() __attribute__((always_inline)) {
    if (w0 + lane < pages && (unsigned)raw >= (unsigned)p.num_pages) kv_fault(p.fault);
  };
  report_pages();
  if (!early) {
    load_tile(ta, key);
    if (p.chunk > STEP) load_tile(tb, key + STEP);
  }
  auto load = [&](Tile& t, int key0) __attribute__((always_inline)) {
    const int last = min((key0 + ST - 1) >> p.psl, p.table_stride - 1);
    if (__builtin_expect(last - w0 >= 64, 0)) {
      w0 = key0 >> p.psl;
      fetch_window();
      report_pages();
    }
    load_tile(t, key0);
  };

  bf16x8 qf[RB][2];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const uint16_t* q = p.q + (int64_t)tok[rb] * p.qr + head[rb] * p.qh;
    // 8-bit pages hand a lane 16 neighbouring dims of a key (one 16-B load): Q follows that order
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
      qf[rb][kk] = *reinterpret_cast<const bf16x8*>(q + (CK == 0 ? kk * 32 + 8 * g : 16 * g + 8 * kk));
  }

  f32x4 o[RB][4];
  float m_ref[RB], l_run[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    m_ref[rb] = -INFINITY;
    l_run[rb] = 0.f;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[rb][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const float c = p.c;
  char* Vs = lds + wave * VT;
  // V's 16-B column is XOR-swizzled by its row, so that the transposed reads of four rows hit different banks
  auto vslot = [&](int row, int ch) __attribute__((always_inline)) { return Vs + row * 128 + ((ch ^ ((row & 3) << 1)) << 4); };

  auto tile_step = [&](const Tile& t, int key0) __attribute__((always_inline)) {
    const bool mask = key0 + ST > lim_lo;
    // V to LDS (rows past the sequence as zeros: whatever their memory holds must not meet a zero weight)
#pragma unroll
    for (int i = 0; i < (CK == 0 ? 4 : 2); ++i) {
      if constexpr (CK == 0) {
        const int row = 8 * i + (lane >> 3);
        uint4 v = t.v[i];
        if (mask && key0 + row >= len) v = uint4{0, 0, 0, 0};
        *reinterpret_cast<uint4*>(vslot(row, lane & 7)) = v;
      } else {
        const int row = 16 * i + (lane >> 2);
        const float s = exponent_value(t.ve[i]);
        bf16x8 lo = decode8<F16, CK == 2>(uint2{t.v[i].x, t.v[i].y}, s);
        bf16x8 hi = decode8<F16, CK == 2>(uint2{t.v[i].z, t.v[i].w}, s);
        if (mask && key0 + row >= len) lo = hi = bf16x8{0, 0, 0, 0, 0, 0, 0, 0};
        *reinterpret_cast<bf16x8*>(vslot(row, (lane & 3) * 2)) = lo;
        *reinterpret_cast<bf16x8*>(vslot(row, (lane & 3) * 2 + 1)) = hi;
      }
    }
    bf16x8 kf[2][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      if constexpr (CK == 0) {
        kf[kb][0] = __builtin_bit_cast(bf16x8, t.k[2 * kb]);
        kf[kb][1] = __builtin_bit_cast(bf16x8, t.k[2 * kb + 1]);
      } else {
        const float s = exponent_value(t.ke[kb]);
        kf[kb][0] = decode8<F16, CK == 2>(uint2{t.k[kb].x, t.k[kb].y}, s);
        kf[kb][1] = decode8<F16, CK == 2>(uint2{t.k[kb].z, t.k[kb].w}, s);
      }
    }
    // V^T fragments: dims 16 dt + l16, keys 4 g .. + 3 and 16 + 4 g .. + 3 (the order the scores come in)
    auto v_frag = [&](int dt) __attribute__((always_inline)) {
      const int q4 = l16 >> 2, p4 = l16 & 3;
      const int row = 4 * g + q4, ch = dt * 2 + (p4 >> 1), within = (p4 & 1) * 8;
      const s4v lo = tr_read(vslot(row, ch) + within);
      const s4v hi = tr_read(vslot(row + 16, ch) + within);
      return (bf16x8)s8v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    bf16x8 vf[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) vf[dt] = v_frag(dt);
    bool special = false;  // as in the chunk kernel's pv_checked
    if (mask) {
      uint32_t bits = 0;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) bits |= special_bits<F16>(vf[dt]);
      special = __any(bits != 0);
    }
    if (__builtin_expect(special, 0)) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) vf[dt] = part_of<F16, false>(vf[dt]);
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      f32x4 st[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        st[kb] = mfma16x16x32<F16>(kf[kb][0], qf[rb][0], f32x4{0.f, 0.f, 0.f, 0.f});
        st[kb] = mfma16x16x32<F16>(kf[kb][1], qf[rb][1], st[kb]);
      }
      if (mask) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[kb][i] = key0 + 16 * kb + 4 * g + i < limit[rb] ? st[kb][i] : -INFINITY;
      }
      float mx = fmaxf(fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3])),
                       fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c;
      const float m_new = fmaxf(m_ref[rb], mx - Softmax<F16>::LIFT);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;  // nothing seen yet
      const float alpha = __builtin_amdgcn_exp2f(m_ref[rb] - m_use);
      m_ref[rb] = m_new;
      float e[8], ls = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i >> 2][i & 3], c, -m_use));
        ls += e[i];
      }
      l_run[rb] = l_run[rb] * alpha + ls;
      const bf16x8 pf = __builtin_bit_cast(bf16x8, uint4{pack16<F16>(e[0], e[1]), pack16<F16>(e[2], e[3]),
                                                         pack16<F16>(e[4], e[5]), pack16<F16>(e[6], e[7])});
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o[rb][dt] *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o[rb][dt] = mfma16x16x32<F16>(vf[dt], pf, o[rb][dt]);
      if (__builtin_expect(special, 0)) {
#pragma unroll 1
        for (int dt = 0; dt < 4; ++dt) {
          const bf16x8 vs = part_of<F16, true>(v_frag(dt));
          f32x4 sum = o[rb][0];
#pragma unroll
          for (int x = 1; x < 4; ++x) sum = dt == x ? o[rb][x] : sum;
#pragma unroll 1
          for (int jj = 0; jj < 32; ++jj) {
            const int j = jj & 7, g2 = jj >> 3;
            const int key = key0 + 4 * g2 + (j & 3) + 16 * (j >> 2);
            const bf16x8 pk = only(pf, j, g == g2), vk = only(vs, j, g == g2);
            const f32x4 x = mfma16x16x32<F16>(vk, pk, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = key < limit[rb] ? sum[i] + x[i] : sum[i];
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) o[rb][x] = dt == x ? sum : o[rb][x];
        }
      }
    }
  };

  // two tiles in registers: the loads of one fly while the other is used
#pragma unroll 1
  while (key < k_end) {
    tile_step(ta, key);
    if (key + 2 * STEP < k_end) load(ta, key + 2 * STEP);
    key += STEP;
    if (key >= k_end) break;
    tile_step(tb, key);
    if (key + 2 * STEP < k_end) load(tb, key + 2 * STEP);
    key += STEP;
  }

  // join the four waves: fp32 rows, maxima and sums through LDS
  __syncthreads();
  float* jo = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    float l = l_run[rb];
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const int row = rb * 16 + l16;
    if (g == 0) {
      join_m[wave][row] = m_ref[rb];
      join_l[wave][row] = l;
    }
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
      *reinterpret_cast<f32x4*>(jo + (wave * RS + row) * HD + dt * 16 + 4 * g) = o[rb][dt];
  }
  __syncthreads();
  for (int i = tid; i < rows * 16 && i < RS * 16; i += NT) {
    const int row = i >> 4, d = (i & 15) * 4;
    const int rt = row / p.group, h = hk * p.group + row - rt * p.group, t = c0 + rt;
    float m = join_m[0][row];
#pragma unroll
    for (int x = 1; x < 4; ++x) m = fmaxf(m, join_m[x][row]);
    const bool seen = key_limit(pos0 + rt, len, p.block) > k_begin;
    const float m_use = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float wgt = __builtin_amdgcn_exp2f(join_m[x][row] - m_use);
      l += wgt * join_l[x][row];
      acc += wgt * *reinterpret_cast<const f32x4*>(jo + (x * RS + row) * HD + d);
    }
    const bool part = lim_hi > p.chunk;
    const float lse2 = !seen ? -INFINITY : range_lse(m_use, l, part);
    f32x4 v = acc * range_inverse(l, part);
    if (!seen) v = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!part) {  // one range holds all keys: no partials
      *reinterpret_cast<uint2*>(p.o + (int64_t)t * p.orr + h * p.oh + d) =
          uint2{pack16<F16>(v[0], v[1]), pack16<F16>(v[2], v[3])};
      if (p.lse && d == 0) p.lse[(int64_t)h * p.new_rows + t] = lse2 * LN2;
    } else {
      const int64_t pr = mapa_idx::paged_step_slot(b, hk, split, p.kv_heads, p.splits) * RS + row;
      *reinterpret_cast<f32x4*>(p.part_o + pr * HD + d) = v;
      if (d == 0) p.part_lse[pr] = lse2;
    }
  }
}

// ------------------------------------------------------------------------------------------------ merge
// Eight ranges' partials (their log2 sums ls, normalised rows v) into the running maximum, weight and row
__device__ __forceinline__ void merge_ranges(const float* ls, const f32x4* v, float& m, float& l, f32x4& acc) {
  float mx = m;
#pragma unroll
  for (int i = 0; i < 8; ++i) mx = fmaxf(mx, ls[i]);
  const float use = mx == -INFINITY ? 0.f : mx;
  const float keep = __builtin_amdgcn_exp2f(m - use);
  l *= keep;
  acc *= keep;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float w = __builtin_amdgcn_exp2f(ls[i] - use);
    l += w;
    acc += w * v[i];
  }
  m = mx;
}
template <bool F16>
__device__ __forceinline__ void merge_store(const PagedArgs& p, int n, float m, float l, f32x4 acc, int tok, int head,
                                            int d) {
  const float inv = n > 0 ? 1.f / l : 0.f;
  *reinterpret_cast<uint2*>(p.o + (int64_t)tok * p.orr + head * p.oh + d) =
      uint2{pack16<F16>(acc[0] * inv, acc[1] * inv), pack16<F16>(acc[2] * inv, acc[3] * inv)};
  if (p.lse && d == 0)
    p.lse[(int64_t)head * p.new_rows + tok] = n > 0 ? range_lse(m, l, false) * LN2 : -INFINITY;
}

// One wave per row: four groups of 16 lanes x 4 columns, group g over the key ranges g, g + 4, ...; 32 ranges' partials
// are in flight at once, joined in a fixed order.  `first`: the row in its first range's slot, `r`: its first 32 ranges'
// partials, fetched before it is known how many of them the row sees; `n`: that number.
struct Ranges {
  float ls[8];
  f32x4 v[8];
};
template <int ROWS>
__device__ __forceinline__ void load_ranges(const PagedArgs& p, int64_t first, int s0, int lane, Ranges& r) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int s = s0 + 4 * i + (lane >> 4);
    r.ls[i] = -INFINITY;
    r.v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (s < p.splits) {
      const int64_t at = first + (int64_t)s * ROWS;
      r.ls[i] = p.part_lse[at];
      r.v[i] = *reinterpret_cast<const f32x4*>(p.part_o + at * HD + (lane & 15) * 4);
    }
  }
}
template <bool F16, int ROWS>
__device__ __forceinline__ void merge_row(const PagedArgs& p, int64_t first, Ranges& r, int n, int tok, int head,
                                          int lane) {
  const int d = (lane & 15) * 4, g = lane >> 4;
  float m = -INFINITY, l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int s0 = 0; s0 < n; s0 += 32) {
    if (s0 > 0) load_ranges<ROWS>(p, first, s0, lane, r);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (s0 + 4 * i + g >= n) {  // a range that the row does not see: never written
        r.ls[i] = -INFINITY;
        r.v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    merge_ranges(r.ls, r.v, m, l, acc);
  }
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    const float m2 = __shfl_xor(m, o, 64), l2 = __shfl_xor(l, o, 64);
    const float mx = fmaxf(m, m2), use = mx == -INFINITY ? 0.f : mx;
    const float wa = __builtin_amdgcn_exp2f(m - use), wb = __builtin_amdgcn_exp2f(m2 - use);
    l = l * wa + l2 * wb;
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = acc[j] * wa + __shfl_xor(acc[j], o, 64) * wb;
    m = mx;
  }
  if (g == 0) merge_store<F16>(p, n, m, l, acc, tok, head, d);
}

// The split tasks of the chunk kernel: blockIdx.x = task, blockIdx.y = 32 of its rows; 16 lanes x 4 columns per row
// (there are many rows, so nothing is gained by spreading a row's ranges over lanes)
template <bool F16>
__global__ void __launch_bounds__(NT) attn_paged_merge_chunk(PagedArgs p) {
  const int lane = threadIdx.x & 63, d = (threadIdx.x & 15) * 4;
  const int j = blockIdx.x;
  int hk, tile;
  mapa_idx::paged_task(p.whole + j, p.tiles, p.tile_passes, hk, tile);
  const RowTile rt = find_tile(p, tile, lane);
  if (rt.seq < 0) return;
  const int len = rt.len;
  const int t0 = rt.tile * p.per_tile, pos0 = len - rt.nq + t0;
  const int rows = min(p.per_tile, rt.nq - t0) * p.group;
  if (key_limit(pos0 + (rows - 1) / p.group, len, p.block) <= p.chunk) return;  // one range: written where computed
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = blockIdx.y * 32 + i * 16 + (threadIdx.x >> 4);
    if (r >= rows) return;
    const int t = r / p.group, tok = rt.c0 + t0 + t, head = hk * p.group + r - t * p.group;
    const int n = (key_limit(pos0 + t, len, p.block) + p.chunk - 1) / p.chunk;
    const int64_t first = (int64_t)j * p.splits * p.slot_rows + r;
    float m = -INFINITY, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int s0 = 0; s0 < n; s0 += 8) {
      float ls[8];
      f32x4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        ls[k] = -INFINITY;
        v[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (s0 + k < n) {
          const int64_t at = first + (int64_t)(s0 + k) * p.slot_rows;
          ls[k] = p.part_lse[at];
          v[k] = *reinterpret_cast<const f32x4*>(p.part_o + at * HD + d);
        }
      }
      merge_ranges(ls, v, m, l, acc);
    }
    merge_store<F16>(p, n, m, l, acc, tok, head, d);
  }
}

// The step kernel's rows: blockIdx.x = (sequence, K/V head), blockIdx.y = 4 of its rows
template <bool F16, int RB>
__global__ void __launch_bounds__(NT) attn_paged_merge_step(PagedArgs p) {
  constexpr int RS = RB * 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.x / p.kv_heads, hk = blockIdx.x - b * p.kv_heads, r = blockIdx.y * 4 + wave;
  const int64_t first = mapa_idx::paged_step_slot(b, hk, 0, p.kv_heads, p.splits) * RS + r;
  Ranges part;
  load_ranges<RS>(p, first, 0, lane, part);
  const int c0 = p.cu[b];
  const int nq = new_tokens(p, c0, p.cu[b + 1]);
  if (r >= nq * p.group) return;
  const int len = checked_len(p.kv_lens[b], p.cap, p.fault);
  if (key_limit(len - 1, len, p.block) <= p.chunk) return;  // one range: written where computed
  const int t = r / p.group;
  const int limit = key_limit(len - nq + t, len, p.block);
  merge_row<F16, RS>(p, first, part, (limit + p.chunk - 1) / p.chunk, c0 + t, hk * p.group + r - t * p.group, lane);
}

// ------------------------------------------------------------------------------------------------ plan
struct Plan {
  int rb;     // row blocks of the step kernel (0: the chunk kernel)
  int waves;  // of a chunk workgroup
  int slot_rows;
  int tiles, per_tile;
  int whole, splits, chunk;
  int64_t slots;  // workgroups that leave partials
  int64_t ws;     // bytes of the partials
};

int cu_count() {
  static int cache[16] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 16) dev = 0;
  if (cache[dev]) return cache[dev];
  int cus = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
  return cache[dev] = cus;
}

// Key ranges per task when all tasks are alike (one sequence): n of them cost ceil(tasks n / slots) rounds of
// (tiles / n + fixed) tile times each, where a workgroup's fixed part (prologue, partial rows, their merge) is worth
// `fixed` tiles; the n with the least cost.
int even_splits(int64_t tasks, int tiles, int slots, double fixed, int most) {
  int best = 1;
  double cost = 0;
  for (int n = 1; n <= most && n <= tiles; ++n) {
    const int64_t rounds = (tasks * n + slots - 1) / slots;
    const double c = (double)rounds * ((tiles + n - 1) / n + (n > 1 ? fixed : 0.0));
    if (n == 1 || c < cost * 0.98) {
      best = n;
      cost = c;
    }
  }
  return best;
}
// ... when the sequences' lengths may differ (the host knows the longest only): the last workgroup to start ends
// one range after the others, so the time is about tasks (tiles + n fixed) / slots + (tiles / n + fixed), least at
// n = sqrt(tiles slots / (tasks fixed)).
int ragged_splits(int64_t tasks, int tiles, int slots, double fixed, int most) {
  const double n = std::sqrt((double)tiles * slots / ((double)tasks * fixed));
  return std::max(1, std::min({most, tiles, (int)(n + 0.5)}));
}

// Waves of a chunk workgroup (32 rows each).  Eight share a tile's decoding where two workgroups of four do it twice, and
// leave more rows of the last tile empty.  One sequence over 12 heads and 55 thousand keys, eight against four waves, by
// the ratio of their padded rows: int8 pages 0.83 to 0.91 of the time at 1 to 1.11 (1370 rows 308 and 340 us), 0.96 at
// 1.14, 0.99 at 1.2, 1.10 at 1.33; e4m3, cheaper to decode, 0.89 to 0.97 at 1 to 1.11 (291 and 304 us), 1.03 at 1.14, 1.15
// at 1.33; over 6 thousand keys eight are no slower anywhere.  16-bit pages have nothing to decode (an 8-view chunk 642
// and 633 us), and ragged batches want the finer pieces (ragged causal int8 chunks 133 and 122 us).
int chunk_waves(const mapa_attn_paged_desc& d) {
  const int64_t rows = (int64_t)d.batch.max_new * (d.heads / d.cache.heads);
  const int64_t four = (rows + 127) / 128 * 128, eight = (rows + 255) / 256 * 256;
  if (d.batch.seqs != 1) return 4;
  if (d.cache.dtype == MAPA_I8) return eight * 5 <= four * 6 ? 8 : 4;
  return d.cache.dtype == MAPA_FP8 && eight * 8 <= four * 9 ? 8 : 4;
}

// Passes over a head's row tiles or key ranges: as many as cut it where the 8 XCDs' equal runs of the work end, so that an
// XCD whose run ends inside a head gets its share of the long and the short pieces.  8 views, each seeing the earlier
// ones, 12 heads 673 us in one pass and 638 in two, 12 heads over one 732 and 649 in eight; 11 thousand causal tokens 273
// and 240; eight ragged causal chunks of 1370 tokens over 4 heads 193 and 180.  Ragged batches keep their row tiles in
// one pass: neighbours share their sequence's keys (ragged causal int8 chunks 122 us in one pass, 130 in two).
int xcd_passes(int heads, int things) {
  int c = 8;
  for (int h = heads; c > 1 && h % 2 == 0; h /= 2) c /= 2;
  return std::min(c, things);
}

Plan make_plan(const mapa_attn_paged_desc& d) {
  Plan pl = {};
  const int group = d.heads / d.cache.heads;
  const int cap = kv_cap(d.cache, d.batch);
  const int64_t rows = (int64_t)d.batch.max_new * group;
  int slots = 2 * cu_count();  // resident workgroups
  int unit, tiles_k;
  int64_t tasks;
  if (rows <= 32) {
    pl.rb = rows <= 16 ? 1 : 2;
    pl.slot_rows = 16 * pl.rb;
    tasks = (int64_t)d.batch.seqs * d.cache.heads;
    unit = 4 * ST;
    tiles_k = std::max(1, (cap + unit - 1) / unit);
    pl.splits = d.batch.seqs == 1 ? even_splits(tasks, tiles_k, slots, 4.0, 128)
                                  : ragged_splits(tasks, tiles_k, slots, 4.0, 128);
  } else {
    pl.waves = chunk_waves(d);
    if (pl.waves == 8) slots /= 2;
    pl.slot_rows = pl.waves * 32;
    pl.per_tile = std::max(1, pl.slot_rows / group);
    const int64_t a = (int64_t)d.batch.new_rows / pl.per_tile + d.batch.seqs;
    const int64_t b = (int64_t)d.batch.seqs * ((d.batch.max_new + pl.per_tile - 1) / pl.per_tile);
    pl.tiles = (int)std::min(a, b);
    tasks = (int64_t)pl.tiles * d.cache.heads;
    unit = KT;
    tiles_k = std::max(1, (cap + unit - 1) / unit);
    if (d.batch.seqs == 1) {  // full rounds of whole tasks, the rest cut so that it fills the chip too
      pl.whole = (int)(tasks / slots * slots);
      const int64_t rest = tasks - pl.whole;
      pl.splits = rest ? even_splits(rest, tiles_k, slots, 4.0, 64) : 1;
      if (pl.splits == 1) pl.whole = (int)tasks;
    } else {
      pl.splits = ragged_splits(tasks, tiles_k, slots, 12.0, 64);
      if (pl.splits == 1) pl.whole = (int)tasks;
    }
  }
  const int per = (tiles_k + pl.splits - 1) / pl.splits;
  pl.splits = (tiles_k + per - 1) / per;
  pl.chunk = per * unit;
  pl.slots = pl.splits > 1 ? (tasks - pl.whole) * pl.splits : 0;
  pl.ws = pl.slots * pl.slot_rows * (HD + 1) * 4;
  return pl;
}
// the same work without a workspace: every task walks all its keys
void unsplit(Plan& pl, const mapa_attn_paged_desc& d) {
  pl.splits = 1;
  pl.chunk = 1 << 30;
  pl.whole = pl.rb ? 0 : pl.tiles * d.cache.heads;
  pl.slots = pl.ws = 0;
}

int check_desc(const mapa_attn_paged_desc* d) {
  const char* who = "mapa_attention_paged";
  MAPA_CHECK_ARG(d != nullptr, "%s: null descriptor", who);
  if (int rc = check_cache(d->cache, who)) return rc;
  if (int rc = check_batch(d->batch, who)) return rc;
  MAPA_CHECK_ARG(d->dtype == MAPA_BF16 || d->dtype == MAPA_F16, "%s: queries must be bf16 or f16", who);
  MAPA_CHECK_ARG(d->cache.dtype == MAPA_FP8 || d->cache.dtype == MAPA_I8 || d->cache.dtype == d->dtype,
                 "%s: 16-bit pages must have the queries' type", who);
  MAPA_CHECK_ARG(d->heads > 0 && d->heads <= 65535 && d->heads % d->cache.heads == 0 &&
                     d->heads / d->cache.heads <= MAX_GROUP,
                 "%s: %d query heads over %d K/V heads", who, d->heads, d->cache.heads);
  MAPA_CHECK_ARG(d->mask_block >= 0, "%s: bad mask_block %d", who, d->mask_block);
  MAPA_CHECK_ARG(d->scale >= 0.f && d->scale < 1e30f, "%s: bad scale %g", who, (double)d->scale);
  return 0;
}

template <bool F16, int CK>
void launch(const PagedArgs& a, const Plan& pl, unsigned grid, hipStream_t stream) {
  if (CK != 0 && pl.rb == 0 && pl.waves == 8)
    hipLaunchKernelGGL((attn_paged_chunk<F16, CK, CK != 0 ? 8 : 4>), dim3(grid), dim3(512), 0, stream, a);
  else if (pl.rb == 0) hipLaunchKernelGGL((attn_paged_chunk<F16, CK, 4>), dim3(grid), dim3(256), 0, stream, a);
  else if (pl.rb == 1) hipLaunchKernelGGL((attn_paged_step<F16, CK, 1>), dim3(grid), dim3(NT), 0, stream, a);
  else hipLaunchKernelGGL((attn_paged_step<F16, CK, 2>), dim3(grid), dim3(NT), 0, stream, a);
}
template <bool F16>
int launch_all(const PagedArgs& a, const Plan& pl, int page_dtype, int64_t wgs, hipStream_t stream) {
  if (page_dtype == MAPA_FP8) launch<F16, 1>(a, pl, (unsigned)wgs, stream);
  else if (page_dtype == MAPA_I8) launch<F16, 2>(a, pl, (unsigned)wgs, stream);
  else launch<F16, 0>(a, pl, (unsigned)wgs, stream);
  MAPA_CHECK_LAUNCH("mapa_attention_paged");
  if (pl.slots == 0) return 0;
  if (pl.rb == 0) {
    const dim3 grid(a.tiles * a.kv_heads - a.whole, a.slot_rows / 32);
    hipLaunchKernelGGL((attn_paged_merge_chunk<F16>), grid, dim3(NT), 0, stream, a);
  } else {
    const dim3 grid(a.seqs * a.kv_heads, (std::min(a.max_new * a.group, 16 * pl.rb) + 3) / 4);
    if (pl.rb == 1) hipLaunchKernelGGL((attn_paged_merge_step<F16, 1>), grid, dim3(NT), 0, stream, a);
    else hipLaunchKernelGGL((attn_paged_merge_step<F16, 2>), grid, dim3(NT), 0, stream, a);
  }
  MAPA_CHECK_LAUNCH("mapa_attention_paged (merge)");
  return 0;
}

}  // namespace

extern "C" int64_t mapa_attention_paged_workspace_bytes(const mapa_attn_paged_desc* d) {
  if (check_desc(d) || d->batch.seqs == 0 || d->batch.new_rows == 0) return 0;
  return make_plan(*d).ws;
}

extern "C" int mapa_attention_paged(const mapa_attn_paged_desc* d, hipStream_t stream) {
  if (int rc = check_desc(d)) return rc;
  const mapa_kv_batch& b = d->batch;
  if (b.seqs == 0 || b.new_rows == 0 || b.max_new == 0) return 0;
  MAPA_CHECK_ARG(d->q && d->o && (uintptr_t)d->q % 16 == 0 && (uintptr_t)d->o % 16 == 0 && d->q_rstride % 8 == 0 &&
                     d->q_hstride % 8 == 0 && d->o_rstride % 8 == 0 && d->o_hstride % 8 == 0,
                 "mapa_attention_paged: query / output bases and strides must keep 16-byte alignment");
  Plan pl = make_plan(*d);
  if (pl.ws && !(d->workspace && (uintptr_t)d->workspace % 16 == 0 && d->workspace_bytes >= pl.ws)) unsplit(pl, *d);
  PagedArgs a = {};
  a.page[0] = (const char*)d->cache.k; a.page[1] = (const char*)d->cache.v;
  a.exp[0] = d->cache.k_exp; a.exp[1] = d->cache.v_exp;
  a.table = b.table; a.kv_lens = b.kv_lens; a.cu = b.cu_new;
  a.q = (const uint16_t*)d->q; a.o = (uint16_t*)d->o; a.lse = d->lse;
  a.qr = d->q_rstride; a.qh = d->q_hstride; a.orr = d->o_rstride; a.oh = d->o_hstride;
  a.fault = mapa_gemm_impl::fault_word();
  a.c = (d->scale > 0.f ? d->scale : 0.125f) * LOG2E;
  a.seqs = b.seqs; a.table_stride = b.table_stride; a.new_rows = b.new_rows; a.max_new = b.max_new;
  a.cap = kv_cap(d->cache, b);
  a.num_pages = d->cache.num_pages; a.psl = log2_of(d->cache.page_size);
  a.heads = d->heads; a.kv_heads = d->cache.heads; a.group = d->heads / d->cache.heads;
  a.block = d->mask_block;
  a.splits = pl.splits; a.chunk = pl.chunk; a.whole = pl.whole; a.tiles = pl.tiles; a.per_tile = pl.per_tile;
  a.slot_rows = pl.slot_rows;
  a.tile_passes = b.seqs == 1 && pl.rb == 0 ? xcd_passes(a.kv_heads, pl.tiles) : 1;
  a.range_passes = xcd_passes(a.kv_heads, pl.splits);
  const int64_t wgs = pl.rb ? (int64_t)b.seqs * a.kv_heads * a.splits : pl.whole + pl.slots;
  MAPA_CHECK_ARG(wgs <= 0x7fffffff && (int64_t)pl.tiles * a.kv_heads <= 0x7fffffff,
                 "mapa_attention_paged: too many workgroups");
  if (pl.slots) {
    a.part_o = (float*)d->workspace;
    a.part_lse = a.part_o + pl.slots * pl.slot_rows * HD;
  }
  return d->dtype == MAPA_F16 ? launch_all<true>(a, pl, d->cache.dtype, wgs, stream)
                              : launch_all<false>(a, pl, d->cache.dtype, wgs, stream);
}
