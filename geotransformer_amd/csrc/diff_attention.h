// diff_attention.h -- kernels of the differential attention (geotr_diff_attn_*, include/geotr.h), instantiated per type in
// diff_attention_{f32,bf16,f16}.hip.
//
//   out_h = sum_j (P1_ij - lam_h P2_ij) v_j,   Pa_ij = softmax_j(s q_a,i . k_a,j),   heads 2h and 2h + 1 of q and k are the two maps.
//
// One pass over the keys with a running maximum and sum for each map and an accumulator for each map: 4 D + 4 Dv operations per (row, key).
//   Joining the weights first would need the sums before the pass: one V product less, but every score and exponential twice.
// Backward, from lse_a = log2 of the sums and del_a = dO . O_a (attention output of map a):
//   dP = dO V^T;  dS1 = P1 (dP - del1);  dS2 = -lam P2 (dP - del2);  dQa = s dSa Ka;  dKa = s dSa^T Qa;  dV = (P1 - lam P2)^T dO;
//   dlam = - sum_ij P2 dP.  Blocks that own query rows (dQ, dlam) and blocks that own keys (dK, dV): the scores are computed twice, and no sum
//   depends on the order of atomics.
//
// Buckets of widths (32, 64, 128; values one or two times that) and groups of heads rounded up to a power of two pad what lies between: a head
// of 80 or 96 takes the time of 128 (52 and 53 us against 56, causal 2 x 2 048 rows, 4 heads, bf16), a group of 5 or 7 nearly that of 8 (62, 65 and
// 68 us, 2 key heads, 64, 128).
// Layout of the matrix work (32 x 32 MFMA, a wave = 32 rows of one kind): scores are computed TRANSPOSED to how they are consumed, so the
// accumulator a lane holds (16 of 32 contraction indices of ONE row) is the B operand of the next product as it stands: no exchange
// between lanes and no LDS round trip for P and dS.  The other operand of that product is read transposed from LDS (ds_read_b64_tr_b16;
// 32-bit: ds_read_b32 along the row), contraction indices in the same order: 8 (r / 4) + 4 half + r % 4 for accumulator register r.
// A row of a head group: with g query heads to a key head the heads of a query are consecutive rows r = (i << gsh) + h of the tile (g rounded
// up to a power of two), so they share every K and V fragment, and one query row over a long cache still fills g rows of the tile.
// Tiles go global -> LDS by 16-byte buffer loads (no registers), rows that do not exist or are masked and channels beyond D / Dv at an
// offset past the buffer's end: the hardware writes zeros, so what a masked row holds (NaN included) never enters a product.  The chunk
// order inside a row is permuted by the row (swizzle): row reads and transposed reads both spread over all banks.
#pragma once
#include "common.h"

namespace geotr {
namespace dattn {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;
#define GEOTR_LDS __attribute__((address_space(3)))
#define GEOTR_INLINE __attribute__((always_inline))
// LDS reads are not moved ahead over this (registers)
#define GEOTR_FENCE __builtin_amdgcn_sched_barrier(0)

struct Args {
  geotr_heads q, k, v, dout;             // dout: backward only
  void *out, *gq, *gk, *gv;              // contiguous (rows, heads, channels)
  float* maps;                           // (rows, heads, 2, dv): the maps' outputs, for the backward pass
  float *lse, *part, *drow;              // (hk, 4, nq, g): see store_sums; split partials; (hk, nq, g)
  float* rows;                           // backward, (hk, 4, nq, g, 2): lse1, lse2 - log2 |lam|; del1, del2; sign of lam, rest of lse1; of lse2, -
  const float* amax;                     // 16-bit floats of narrow range: largest |dout| and |v| (backward)
  const float* lam;
  const int64_t *q_len, *k_len;
  const uint8_t* masks;                  // (nk) 1 = ignored key
  int64_t nq, nk;                        // all rows
  int batch, stacked, n, m;              // batch mode: n, m rows per sequence
  int hk, g, gsh, d, dv, causal, splits; // query heads to a key head; packed rows r = (i << gsh) + h, h < g <= 1 << gsh
  int tiles, tile0, seq0;                // tiles of a head; a launch's first tile and (batch mode) first sequence: a grid may not hold them all
  float scale, scale_log2;
};

// ---- types: E elements in 16 bytes, a contraction step of 2 E, one 16-byte fragment per lane and step -----------------------------------
template <typename T>
struct Ops;
template <>
struct Ops<__bf16> {
  using Frag = __attribute__((ext_vector_type(8))) __bf16;
  static __device__ __forceinline__ void mma(f32x16& c, Frag a, Frag b) { c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Ops<_Float16> {
  using Frag = __attribute__((ext_vector_type(8))) _Float16;
  static __device__ __forceinline__ void mma(f32x16& c, Frag a, Frag b) { c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Ops<float> {
  using Frag = f32x4;
  static __device__ __forceinline__ void mma(f32x16& c, Frag a, Frag b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  }
};

template <typename T>
constexpr int kE = 16 / sizeof(T);         // elements of a fragment
template <typename T>
constexpr int kStep = 2 * kE<T>;           // channels (row reads) or contraction indices of one step
template <typename T>
constexpr int kPSteps = 32 / kStep<T>;     // steps of a 32-deep product

// the type whose exponents are narrow
template <typename T>
struct Narrow {
  static constexpr bool value = false;
};
template <>
struct Narrow<_Float16> {
  static constexpr bool value = true;
};
// waves that a SIMD unit holds at a time, by the registers of the accumulators (rows: one map to a wave, half of them)
template <typename T, int DB, int DVB>
constexpr int kWaves = sizeof(T) * DB <= 128 ? 2 : 1;
template <typename T, int DB, int DVB>
constexpr int kWavesRows = sizeof(T) == 4 ? (DB <= 32 ? 3 : DB <= 64 ? 2 : 1) : DVB <= 64 ? 4 : DVB <= 128 ? 3 : 2;

// fragment t of the accumulator's 32 contraction indices: registers E t .. E t + E - 1 (rounded to T: the one rounding of P and dS)
template <typename T>
__device__ __forceinline__ typename Ops<T>::Frag pack(const f32x16& p, int t) {
  typename Ops<T>::Frag f;
#pragma unroll
  for (int i = 0; i < kE<T>; ++i) f[i] = (T)p[kE<T> * t + i];
  return f;
}

// what pack(p, t) = w rounded away: p - w in one instruction as a product of a pair with (-1, 0) or (0, -1), where expanding w would take one
// more.  The pairs are kept from the compiler: bfloat16's (-1, 0) as an immediate is read as (0, -1).
template <typename T>
__device__ __forceinline__ typename Ops<T>::Frag pack_rest(const f32x16& p, int t, const typename Ops<T>::Frag& w) {
  using Pair = __attribute__((ext_vector_type(2))) T;
  unsigned one = Narrow<T>::value ? 0xbc00u : 0xbf80u, other = one << 16;
  asm("" : "+s"(one), "+s"(other));
  const Pair minus[2] = {__builtin_bit_cast(Pair, one), __builtin_bit_cast(Pair, other)};
  typename Ops<T>::Frag f;
#pragma unroll
  for (int i = 0; i < kE<T>; ++i) {
    const Pair x = {w[i & ~1], w[i | 1]};
    if constexpr (Narrow<T>::value) f[i] = (T)__builtin_amdgcn_fdot2(x, minus[i & 1], p[kE<T> * t + i], false);
    else f[i] = (T)__builtin_amdgcn_fdot2_f32_bf16(x, minus[i & 1], p[kE<T> * t + i], false);
  }
  return f;
}

// ---- LDS tiles ------------------------------------------------------------------------------------------------------------------------
// A tile of rows of C 16-byte chunks; chunk c of row r lies at position c ^ swz(r).  256 bytes (all banks) hold 16 / C rows.  swz moves row
// bits to chunk bits (linear over xor): eight rows read at one chunk, and the 4 rows x 2 chunks of a transposed read, fall on distinct banks.
template <int C>
__device__ __host__ constexpr int swz(int row) {
  return C >= 16 ? ((row << 1) & 14) | ((row >> 3) & 1) : ((row * C / 16) << 1) & (C - 1);
}
template <class V>
__device__ __forceinline__ V lds_load(unsigned at) {
  return *(const GEOTR_LDS V*)(uintptr_t)at;
}
__device__ __forceinline__ unsigned lds_at(const void* p) { return (unsigned)(uintptr_t)(const GEOTR_LDS char*)p; }

// Row reads: lane % 32 = row, chunks c0 + 2 q + half of the CM from c0 (a multiple of CM) on.  One address for each xor pattern, everything
// else in the instruction's offset.
template <typename T, int C, int CM = C>
struct Rows {
  static constexpr int N = (CM >= 16 ? 16 : CM) / 2;
  unsigned a[N];
  __device__ __forceinline__ Rows(int col, int half, int c0 = 0) {
#pragma unroll
    for (int j = 0; j < N; ++j) a[j] = col * C * 16 + ((c0 + 2 * j + half) ^ swz<C>(col)) * 16;
  }
  __device__ __forceinline__ typename Ops<T>::Frag get(unsigned tile, int row0, int q) const {  // row0 a multiple of 32
    return lds_load<typename Ops<T>::Frag>(tile + a[q % N] + (unsigned)(row0 * C * 16 + (q / N) * 256));
  }
};
// Transposed reads: lane % 32 = channel 32 v + lane % 32; contraction indices = rows, in the order of the accumulator registers, step t
template <typename T, int C, int SIZE = sizeof(T)>
struct Cols;
template <typename T, int C>
struct Cols<T, C, 2> {
  static constexpr int NU = C >= 16 ? 2 : 1, NV = (C >= 16 ? 16 : C) / 4;
  unsigned a[NV * NU];
  __device__ __forceinline__ Cols(int lane) {
    const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), lp = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int u = 0; u < NU; ++u) a[v * NU + u] = row * C * 16 + ((4 * v + lp) ^ swz<C>(row + 8 * u)) * 16 + (lane & 1) * 8;
  }
  __device__ __forceinline__ typename Ops<T>::Frag get(unsigned tile, int row0, int t, int v) const {  // row0 a multiple of 32
    const unsigned o = (row0 + 16 * t) * C * 16 + (v / NV) * 256, i = (v % NV) * NU;
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GEOTR_LDS s16x4*)(uintptr_t)(tile + a[i] + o));
    const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GEOTR_LDS s16x4*)(uintptr_t)(tile + a[i + NU - 1] + o + 8 * C * 16));
    return __builtin_bit_cast(typename Ops<T>::Frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  }
};
template <typename T, int C>
struct Cols<T, C, 4> {
  static constexpr int NT = C >= 16 ? 2 : 1, NV = C >= 16 ? 2 : 1;
  unsigned a[4 * NT * NV];
  __device__ __forceinline__ Cols(int lane) {
    const int row = 4 * (lane >> 5), c = (lane & 31) >> 2;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < NV; ++v) a[(i * NT + t) * NV + v] = (row + i) * C * 16 + ((8 * v + c) ^ swz<C>(row + i + 8 * t)) * 16 + (lane & 3) * 4;
  }
  __device__ __forceinline__ typename Ops<T>::Frag get(unsigned tile, int row0, int t, int v) const {
    typename Ops<T>::Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f[i] = lds_load<float>(tile + a[(i * NT + t % NT) * NV + v % NV] + (unsigned)((row0 + 8 * t) * C * 16 + (v / NV) * 256));
    return f;
  }
};

constexpr int kNumRecords = 0x40000000, kOutside = 0x7fffff00;  // a chunk at kOutside lies past every buffer: zeros
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, kNumRecords, 0x00020000);
}
// 16 bytes per lane from byte offset + scalar into 1 024 bytes of LDS.  Issued by asm (it writes no register): the compiler takes a
// transposed LDS read for one that may depend on every such load in flight and would wait for the next tile before this one's products
// (causal 8 192: 489 us with the builtin).  The loops wait themselves (tile_ready).
using i32x4 = __attribute__((ext_vector_type(4))) int;
__device__ __forceinline__ i32x4 words(const void* p) {
  const uint64_t u = (uint64_t)p;
  int lo = __builtin_amdgcn_readfirstlane((int)u), hi = __builtin_amdgcn_readfirstlane((int)(u >> 32)) & 0xffff;
  // a buffer load may read what v_readfirstlane wrote after five wait states, and the compiler does not look into the asm for that
  asm volatile("s_nop 4" : "+s"(lo), "+s"(hi));
  return i32x4{lo, hi, kNumRecords, 0x00020000};
}
__device__ __forceinline__ void load_lds(i32x4 d, unsigned lds, int offset, int scalar = 0) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(offset), "s"(d), "s"(scalar)
               : "m0", "memory");
}
// the descriptor `bytes` further on
__device__ __forceinline__ i32x4 advance(i32x4 d, unsigned bytes) {
  const uint64_t u = (((uint64_t)(unsigned)d[1] << 32) | (unsigned)d[0]) + bytes;
  return i32x4{(int)u, (int)(u >> 32), d[2], d[3]};
}
// this wave's tile loads have arrived, all but the youngest PENDING
template <int PENDING = 0>
__device__ __forceinline__ void tile_ready() {
  static_assert(PENDING < 64, "six bits");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PENDING) : "memory");
}
// Ends the compiler's own wait for what it loaded into x: a use inside a loop would wait for the tile loads in flight as well.
template <class V>
__device__ __forceinline__ void arrived(V& x) {
  asm volatile("" : "+v"(x));
}
// x lies in accumulation registers here: without it the compiler takes the same ones for the scores, 64 moves a tile (dK/dV 327 -> 276 us at
// 2 x 4 096 causal rows and 8 heads).  Only in kernels that spill nothing: in dQ of 32-bit heads of 128
// (432 registers of fragments and accumulators) the compiler, out of registers, takes apart the four registers of a Q fragment around the pinned
// accumulators and loses the copy of one: the first product read an accumulator in its place, and dQ of the first map was wrong.  The marker is
// what a test finds pinned kernels by; it also looks for accumulators among the factors of every product.
__device__ __forceinline__ void held(f32x16& x) { asm volatile("; held" : "+a"(x)); }
template <typename T>
__device__ __forceinline__ typename Ops<T>::Frag load_frag(__amdgpu_buffer_rsrc_t r, int offset) {
  return __builtin_bit_cast(typename Ops<T>::Frag, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0));
}

// ROWS rows of NM maps of `width` channels (bucket DB) into a tile, dealt over the SHARE waves that use it (wave w of them).  row_at(row)
// is a row's byte offset, and 16 rows further on it is rs16 more.  A step of the waves covers S rows; the swizzle repeats after 16 (and is
// linear over xor), so a lane keeps one offset for each of NB steps and reaches the others by a scalar: no vector arithmetic per load
// where every row exists.
template <typename T, int ROWS, int NM, int DB, int SHARE>
struct Stage {
  static constexpr int CM = DB * (int)sizeof(T) / 16, C = NM * CM, N = ROWS * C / 64, S = SHARE * 64 / C > 0 ? SHARE * 64 / C : 1;
  static constexpr int NS = (N + SHARE - 1) / SHARE, NB = C < 16 || S >= 16 ? 1 : 16 / S < NS ? 16 / S : NS;
  static_assert(ROWS * C % 64 == 0 && C <= 64, "whole wave loads");
  int base[NB], row0;
  template <class At>
  __device__ __forceinline__ Stage(int width, int map_bytes, int w, int lane, At row_at) {
    const int p = w * 64 + lane;
    row0 = p / C;
    const int pos = (p % C) ^ swz<C>(row0);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int c = pos ^ swz<C>(j * S), map = NM == 1 ? 0 : c / CM, cc = NM == 1 ? c : c % CM;
      base[j] = cc * kE<T> >= width ? kOutside : row_at(j * S + row0) + map * map_bytes + cc * 16;
    }
  }
  template <class Row>
  __device__ __forceinline__ void load_some(unsigned tile, i32x4 r, int rs16, int w, Row row) const {
#pragma unroll
    for (int it = 0; it < NS; ++it) {
      if (N % SHARE != 0 && it * SHARE + w >= N) break;
      load_lds(r, tile + (it * SHARE + w) * 1024, row(it * S + row0) ? base[it % NB] : kOutside, (it - it % NB) * S * (rs16 / 16));
    }
  }
  // every row exists
  __device__ __forceinline__ void load_all(unsigned tile, i32x4 r, int rs16, int w) const {
    load_some(tile, r, rs16, w, [](int) { return true; });
  }
  // rows `bits` of the tile
  __device__ __forceinline__ void load(unsigned tile, i32x4 r, int rs16, int w, uint64_t bits) const {
    if (bits == (ROWS == 64 ? ~0ull : 0xffffffffull)) load_all(tile, r, rs16, w);
    else load_some(tile, r, rs16, w, [&](int x) { return (bits >> x) & 1; });
  }
};

// the same for rows at offsets of their own: src(row) gives a byte offset or kOutside
template <typename T, int ROWS, int NM, int DB, int SHARE, class Src>
__device__ __forceinline__ void stage_at(unsigned tile, i32x4 r, int width, int map_bytes, int w, int lane, Src src) {
  using L = Stage<T, ROWS, NM, DB, SHARE>;
  asm volatile("" : "+v"(lane));  // recomputed for every tile: kept in registers the offsets would be spilled
  const int p = w * 64 + lane, row0 = p / L::C, pos = (p % L::C) ^ swz<L::C>(row0);
#pragma unroll
  for (int it = 0; it < L::NS; ++it) {
    if (L::N % SHARE != 0 && it * SHARE + w >= L::N) break;
    const int c = pos ^ swz<L::C>(it * L::S);  // swz is linear and row0 < S
    const int map = NM == 1 ? 0 : c / L::CM, cc = NM == 1 ? c : c % L::CM;
    const int o = src(it * L::S + row0);
    load_lds(r, tile + (it * SHARE + w) * 1024, o == kOutside || cc * kE<T> >= width ? kOutside : o + map * map_bytes + cc * 16);
  }
}

// ---- sequences ------------------------------------------------------------------------------------------------------------------------
struct Seq {
  int b;             // address index of the batch (0 in stack mode)
  int64_t q0, k0;    // first row in all rows
  int n, m, tile;    // tile < 0: behind the last sequence
  int spare, spares; // index and number of the blocks behind the last sequence
  int64_t q_end, k_end;
};
constexpr int kMostRows = 1 << 30;
__device__ __forceinline__ int clamp_len(int64_t v, int64_t most) { return (int)(v < 0 ? 0 : v > most ? most : v); }
__device__ __forceinline__ int add_sat(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)kMostRows); }

// Sequence and tile (TILE packed query rows, or keys when KEYS) of block `t`.  Stack mode: lengths on the device, one scan of 64 clouds at
// a time by every wave; sums are held at 2^30 and rows clamped to what exists, so lengths that do not fit never address past the arrays.
template <int TILE, bool KEYS>
__device__ __forceinline__ Seq find_seq(const Args& a, int b, int t, int tiles) {
  Seq s;
  s.spare = 0, s.spares = 1, s.q_end = a.nq, s.k_end = a.nk;
  if (!a.stacked) {
    s.b = b, s.q0 = (int64_t)b * a.n, s.k0 = (int64_t)b * a.m, s.tile = t;
    s.n = a.q_len ? clamp_len(a.q_len[b], a.n) : a.n;
    s.m = a.k_len ? clamp_len(a.k_len[b], a.m) : a.m;
    return s;
  }
  const int lane = lane_id();
  int qs = 0, ks = 0, ts = 0;
  s.b = 0, s.tile = -1, s.n = s.m = 0, s.q0 = s.k0 = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int i = b0 + lane;
    int ql = i < a.batch ? clamp_len(a.q_len[i], a.nq) : 0, kl = i < a.batch ? clamp_len(a.k_len[i], a.nk) : 0;
    const int ql0 = ql, kl0 = kl;
    int tl = KEYS ? (kl + TILE - 1) / TILE : (int)((((int64_t)ql << a.gsh) + TILE - 1) / TILE);
    const int tl0 = tl;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(ql, o, 64), y = __shfl_up(kl, o, 64), z = __shfl_up(tl, o, 64);
      if (lane >= o) ql = add_sat(ql, x), kl = add_sat(kl, y), tl = add_sat(tl, z);
    }
    ql = add_sat(ql, qs), kl = add_sat(kl, ks), tl = add_sat(tl, ts);
    const uint64_t hit = __ballot(tl > t && tl - tl0 <= t && tl0 > 0);
    if (hit && s.tile < 0) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      const int qe = __shfl(ql, l, 64), ke = __shfl(kl, l, 64), te = __shfl(tl, l, 64);
      const int qn = __shfl(ql0, l, 64), kn = __shfl(kl0, l, 64), tn = __shfl(tl0, l, 64);
      s.q0 = qe - qn, s.k0 = ke - kn, s.tile = t - (te - tn);
      s.n = (int)(s.q0 < a.nq ? (s.q0 + qn > a.nq ? a.nq - s.q0 : qn) : 0);
      s.m = (int)(s.k0 < a.nk ? (s.k0 + kn > a.nk ? a.nk - s.k0 : kn) : 0);
      s.tile = __builtin_amdgcn_readfirstlane(s.tile);
      s.n = __builtin_amdgcn_readfirstlane(s.n), s.m = __builtin_amdgcn_readfirstlane(s.m);
      s.q0 = __builtin_amdgcn_readfirstlane((int)s.q0), s.k0 = __builtin_amdgcn_readfirstlane((int)s.k0);
      return s;
    }
    qs = __shfl(ql, 63, 64), ks = __shfl(kl, 63, 64), ts = __shfl(tl, 63, 64);
  }
  s.spare = t - ts, s.spares = max(1, tiles - ts);
  s.q_end = min((int64_t)qs, a.nq), s.k_end = min((int64_t)ks, a.nk);
  return s;
}

// keys key0 .. key0 + 63 that exist and are not masked
__device__ __forceinline__ uint64_t key_bits(const Args& a, const Seq& s, int key0, int end, int lane) {
  if (a.masks) {
    const int j = key0 + lane;
    return __ballot(j < end && !a.masks[s.k0 + j]);
  }
  const int left = end - key0;
  return left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
}

__device__ __forceinline__ float swap_max(float x) {
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
}
__device__ __forceinline__ float swap_add(float x) {
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// Scores beyond 2^20 (in powers of two): s c - b with a product of its own.  An fma keeps the exact product, whose distance from the
// rounded maximum b grows with it until the exponential overflows; rounded alike, the largest score gives exactly 0.
constexpr float kHuge = 1048576.f;
template <class B>
__device__ __forceinline__ void exponents(f32x16& s, float c, B b, bool huge, float rest = 0.f) {
  if (__builtin_expect(huge, 0)) {  // a branch of the wave, not a choice per element
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = (s[i] * c - b(i)) - rest;
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = fmaf(s[i], c, -b(i));
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i]);
}

// One packed query row of a lane: its query, head within the group, whether it exists and whether it is written (batch mode: rows beyond
// their sequence's length get zeros)
struct Row {
  int i, h;
  bool in, out;
};
__device__ __forceinline__ Row row_of(const Args& a, const Seq& s, int r) {
  Row x;
  x.i = r >> a.gsh, x.h = r & ((1 << a.gsh) - 1);
  x.in = x.i < s.n && x.h < a.g;
  x.out = x.i < (a.stacked ? s.n : a.n) && x.h < a.g;
  return x;
}
__device__ __forceinline__ int64_t stat_at(const Args& a, int kvh, int map, int64_t row, int h) {
  return (((int64_t)kvh * 4 + map) * a.nq + row) * a.g + h;
}

// pairs of the numbers of a row lie side by side: what a wave reads of them stays near one address however many rows there are
__device__ __forceinline__ int64_t row_stat_at(const Args& a, int kvh, int pair, int64_t row, int h) {
  return ((((int64_t)kvh * 4 + pair) * a.nq + row) * a.g + h) * 2;
}

// What the backward pass takes weights from: log2 of the sum, m + log2 l.  Beyond 2^20 that would round log2 l away (weights off by 4 % at
// 2^20, all 1 further on), so there m and log2 l are kept apart.  Rows without a key: infinity, weights of zero.
__device__ __forceinline__ void store_sums(const Args& a, int64_t at, float m, float l, bool some) {
  const float log = log2f(l);
  const bool far = fabsf(m) > kHuge;
  a.lse[at] = some ? (far ? m : m + log) : INFINITY;
  a.lse[at + 2 * a.nq * a.g] = some && far ? log : 0.f;
}

// four consecutive channels of an output row
template <typename T>
__device__ __forceinline__ void store4(T* p, float x, float y, float z, float w) {
  struct alignas(4 * sizeof(T)) V { T v[4]; };
  *(V*)p = V{{(T)x, (T)y, (T)z, (T)w}};
}

// ---- forward ----------------------------------------------------------------------------------------------------------------------------
// Order of the tiles of one sequence: causal rows cost what lies before them.  Where all blocks run at once (two to a compute
// unit) the second half goes up from the shortest (a long block shares its unit with a short one); else the longest go first.
__device__ __forceinline__ int tile_order(const Args& a, int y, int tiles, int others, int at_once = 512) {
  if (!a.causal) return y;
  if ((int64_t)tiles * others > at_once) return tiles - 1 - y;
  return y < (tiles + 1) / 2 ? tiles - 1 - y : y - (tiles + 1) / 2;
}
// keys of this block when they are dealt over blockIdx.z
__device__ __forceinline__ void split_keys(const Args& a, int& begin, int& end) {
  const int tiles = (end + 31) / 32, per = (tiles + a.splits - 1) / a.splits;
  begin = min(end, (int)blockIdx.z * per * 32);
  end = min(end, begin + per * 32);
}
// rows behind the last sequence: zero results
template <typename T>
__device__ __forceinline__ void zero_rows(const Args& a, const Seq& s, int kvh, int threads) {
  const int64_t rows = s.q_end < a.nq ? a.nq - s.q_end : 0, per = (int64_t)a.g * a.dv, first = (int64_t)s.spare * threads + threadIdx.x,
                step = (int64_t)s.spares * threads;
  if (a.splits > 1) {  // no keys: the join writes zeros
    const int w = a.dv + 4;
    for (int64_t e = first; e < rows * a.g; e += step) {
      float* p = a.part + (((int64_t)blockIdx.z * a.nq + s.q_end + e / a.g) * a.hk * a.g + kvh * a.g + e % a.g) * 2 * w;
      p[0] = p[w] = -INFINITY, p[1] = p[w + 1] = 0.f;
    }
    return;
  }
  for (int64_t e = first; e < rows * per; e += step) {
    const int64_t i = e / per, o = ((s.q_end + i) * a.hk + kvh) * per + (e - i * per);
    ((T*)a.out)[o] = (T)0.f;
  }
  for (int64_t e = first; a.maps && e < 2 * rows * per; e += step) {
    const int64_t i = e / (2 * per);
    a.maps[((s.q_end + i) * a.hk + kvh) * 2 * per + (e - i * 2 * per)] = 0.f;
  }
  for (int64_t e = first; a.lse && e < rows * a.g; e += step) {
    const int64_t at = stat_at(a, kvh, 0, s.q_end, 0) + e;
    a.lse[at] = a.lse[at + a.nq * a.g] = INFINITY;
    a.lse[at + 2 * a.nq * a.g] = a.lse[at + 3 * a.nq * a.g] = 0.f;
  }
}

// Many rows: the waves are two maps x G groups of 32 packed rows; a wave owns 32 rows of ONE map, so it needs half the accumulators (three
// waves to a SIMD unit at d = 64, v 128, where both maps in a wave leave one) and the maps meet in LDS at the end.  Tiles of 32 keys in two
// buffers: the next one loads while this one is consumed.  8 192 causal rows, 16 heads on 4, 64, 128, bf16: 416 us, 0.99 PFLOP/s of the four
// products where a large library product of this card reaches 1.2.  Counters of that call: matrix core busy 0.51 of the cycles, vector
// instructions 0.50, LDS 0.42 (and 0.17 in conflicts), 2.5 waves to a SIMD unit that wait for an issue slot 0.36 of their life and for data 0.30:
// the two kinds of work take about their sum; what keeps them from overlapping is not established.  32 bits, 2 048 rows: 112 of 138 TFLOP/s.
// P is rounded to the type before its product (outputs in 16 bits are off by 1.2 to 1.4 times what rounding the exact ones gives): a 32-bit
// product takes 16 times as long.  EXACT (below) keeps the rest as well, so a training call's output differs from the same call without
// gradients in the last bits.
// The accumulators are rescaled only when a row's maximum grew by more than 2^8: weights stay below 2^8, sums are exact either way.
// FEW (a token over a cache, wide heads): the G groups share 32 rows and take 32 keys each of every tile, joined at the end.
// EXACT (16-bit, for training): what rounding P to 16 bits takes away goes through a second product, because the gradients subtract
// dout . O_map from dout . v: an error of O is one of every dS of the row, and was as large as all others of dQ and dK together.
template <typename T, int DB, int DVB, int G, bool FEW, bool EXACT>
__global__ __launch_bounds__(128 * G, (kWavesRows<T, DB, DVB>)) void fwd_kernel(Args a) {
  using Frag = typename Ops<T>::Frag;
  constexpr int CK = 2 * DB * (int)sizeof(T) / 16, CV = DVB * (int)sizeof(T) / 16, NT = DVB / 32, QS = DB / kStep<T>, TILE = FEW ? 32 : 32 * G;
  constexpr int BN = FEW ? 32 * G : 32, kTile = BN * (CK + CV) * 16, kJoin = G * (NT * 16 + 2) * 64 * 4;
  constexpr int kSmem = 2 * kTile > kJoin ? 2 * kTile : kJoin;
  constexpr bool kAgain = NT * 16 + QS * 4 <= 80;  // registers left for computing scores again
  __shared__ __attribute__((aligned(1024))) char smem[kSmem];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
  const int map = wave & 1, group = wave >> 1, rows_at = FEW ? 0 : 32 * group;
  const int kvh = a.stacked ? blockIdx.x : blockIdx.x % a.hk;
  const int t = tile_order(a, a.tile0 + blockIdx.y, a.tiles, gridDim.x);
  const Seq s = find_seq<TILE, false>(a, a.stacked ? 0 : a.seq0 + blockIdx.x / a.hk, t, a.tiles);
  if (s.tile < 0) {
    zero_rows<T>(a, s, kvh, 128 * G);
    return;
  }
  const int row_base = s.tile * TILE;
  if (row_base >> a.gsh >= (a.stacked ? s.n : a.n)) return;

  // Q: B operand, lane = row, straight from global memory
  const Row row = row_of(a, s, row_base + rows_at + col);
  Frag q[QS];
  {
    const int i0 = row_base >> a.gsh;
    const auto rq = buffer((const T*)a.q.data + s.b * a.q.batch_stride + ((a.stacked ? s.q0 : 0) + i0) * a.q.row_stride +
                           ((int64_t)kvh * 2 * a.g + map) * a.q.head_stride);
    const int o = (int)(((row.i - i0) * a.q.row_stride + 2 * row.h * a.q.head_stride) * (int)sizeof(T));
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      const int c = (2 * i + half) * kE<T>;
      q[i] = load_frag<T>(rq, row.in && c < a.d ? o + c * (int)sizeof(T) : kOutside);
    }
  }
#pragma unroll
  for (int i = 0; i < QS; ++i) arrived(q[i]);
  f32x16 acc[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc[i] = zero16();
  float m = -INFINITY, l = 0.f;
  bool huge = false;

  const T* const kp = (const T*)a.k.data + s.b * a.k.batch_stride + (a.stacked ? s.k0 : 0) * a.k.row_stride + (int64_t)kvh * 2 * a.k.head_stride;
  const T* const vp = (const T*)a.v.data + s.b * a.v.batch_stride + (a.stacked ? s.k0 : 0) * a.v.row_stride + (int64_t)kvh * a.v.head_stride;
  const int off = s.m - s.n;  // causal: key j for query i iff j <= i + off
  int begin = 0, end = s.m, seen = 0x7fffffff;  // seen: keys that all rows of this wave see
  if (a.causal) {  // no key beyond the last row's limit
    const int last = min((row_base + TILE - 1) >> a.gsh, s.n - 1);
    end = min(end, max(0, last + off + 1));
    seen = ((row_base + rows_at) >> a.gsh) + off + 1;
  }
  if (a.splits > 1) split_keys(a, begin, end);

  const int krs = (int)(a.k.row_stride * sizeof(T)), vrs = (int)(a.v.row_stride * sizeof(T));
  // four waves load K, four (from the other end) V
  const Stage<T, BN, 2, DB, 4> kst(a.d, (int)(a.k.head_stride * sizeof(T)), wave, lane, [&](int x) { return x * krs; });
  const Stage<T, BN, 1, DVB, 4> vst(a.dv, 0, 2 * G - 1 - wave, lane, [&](int x) { return x * vrs; });
  auto fill = [&](unsigned tile, int key0, uint64_t bits) GEOTR_INLINE {
    if (G == 2 || wave < 4) kst.load(tile, words(kp + (int64_t)key0 * a.k.row_stride), 16 * krs, wave, bits);
    if (G == 2 || wave >= 2 * G - 4) vst.load(tile + BN * CK * 16, words(vp + (int64_t)key0 * a.v.row_stride), 16 * vrs, 2 * G - 1 - wave, bits);
  };

  const Rows<T, CK, CK / 2> krow(col, half, map * (CK / 2));
  const Cols<T, CV> vcol(lane);
  const unsigned base = lds_at(smem);
  auto scores = [&](unsigned tile, int key0, unsigned there) GEOTR_INLINE {
    f32x16 x = zero16();
#pragma unroll
    for (int i = 0; i < QS; ++i) Ops<T>::mma(x, krow.get(tile, 0, i), q[i]);
    if (there != 0xffffffffu || key0 + 32 > seen) {
      const int above = a.causal ? row.i + off - key0 : 31;  // keys of the tile up to this one
      unsigned lo = there;
      if (above < 31) lo = above < 0 ? 0u : lo & ((2u << above) - 1);
      lo >>= 4 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = (lo >> (8 * (i / 4) + i % 4)) & 1 ? x[i] : -INFINITY;
    }
    return x;
  };
  auto sum = [&](const f32x16& x) GEOTR_INLINE {
    float u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = (x[i] + x[4 + i]) + (x[8 + i] + x[12 + i]);
    return (u[0] + u[1]) + (u[2] + u[3]);
  };
  auto raise = [&](const f32x16& x) GEOTR_INLINE {  // the reference b to the maximum of scores x
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) top = fmaxf(top, x[i]);
    top = fmaxf(m, swap_max(top) * a.scale_log2);
    const float c = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - top);
    m = top, l *= c;
    huge = __any(fabsf(m) > kHuge && m > -INFINITY);
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[i][j] *= c;
  };
  auto consume = [&](unsigned tile, unsigned vt, int key0, unsigned there) GEOTR_INLINE {
    f32x16 p = scores(tile, key0, there);
    float u;
    if constexpr (kAgain) {
      exponents(p, a.scale_log2, [&](int) { return m; }, huge);  // no reference yet: infinite
      u = sum(p);
      if (!__all(u < 256.f)) {
        p = scores(tile, key0, there);
        raise(p);
        const float from = m == -INFINITY ? 0.f : m;  // no key yet: the weights are zero
        exponents(p, a.scale_log2, [&](int) { return from; }, huge);
        u = sum(p);
      }
    } else {
      float top = p[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) top = fmaxf(top, p[i]);
      if (__any(swap_max(top) * a.scale_log2 > m + 8.f)) raise(p);
      const float from = m == -INFINITY ? 0.f : m;
      exponents(p, a.scale_log2, [&](int) { return from; }, huge);
      u = sum(p);
    }
    l += u;
#pragma unroll
    for (int x = 0; x < kPSteps<T>; ++x) {
      const Frag w = pack<T>(p, x);
      if constexpr (EXACT) {
        const Frag rest = pack_rest<T>(p, x, w);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const Frag v = vcol.get(vt, 0, x, i);
          Ops<T>::mma(acc[i], v, w);
          Ops<T>::mma(acc[i], v, rest);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NT; ++i) Ops<T>::mma(acc[i], vcol.get(vt, 0, x, i), w);
      }
    }
  };

  // Tiles without a missing or masked row (the first `whole` keys) are loaded from descriptors that run along; the others look at every row
  const int whole = a.masks ? begin : begin + (end - begin) / BN * BN;
  i32x4 rk = words(kp + (int64_t)begin * a.k.row_stride), rv = words(vp + (int64_t)begin * a.v.row_stride);
  constexpr uint64_t kAll = BN == 64 ? ~0ull : 0xffffffffull;
  uint64_t bits = 0;
  auto next = [&](int key0, unsigned tile) GEOTR_INLINE {
    if (key0 < whole) {
      if (G == 2 || wave < 4) kst.load_all(tile, rk, 16 * krs, wave);
      if (G == 2 || wave >= 2 * G - 4) vst.load_all(tile + BN * CK * 16, rv, 16 * vrs, 2 * G - 1 - wave);
      rk = advance(rk, BN * krs), rv = advance(rv, BN * vrs);
      return kAll;
    }
    const uint64_t x = key0 < end ? key_bits(a, s, key0, end, lane) & kAll : 0;
    if (key0 < end) fill(tile, key0, x);
    return x;
  };
  auto step = [&](int key0, unsigned tile, unsigned other) GEOTR_INLINE {
    tile_ready();
    __syncthreads();  // the tile is complete, and nobody reads the other buffer any more
    const uint64_t now = bits;
    bits = next(key0 + BN, other);
    if constexpr (FEW) {
      if ((unsigned)(now >> (32 * group))) consume(tile + group * 32 * CK * 16, tile + BN * CK * 16 + group * 32 * CV * 16, key0 + 32 * group, (unsigned)(now >> (32 * group)));
    } else {
      if (now) consume(tile, tile + BN * CK * 16, key0, (unsigned)now);
    }
  };
  bits = next(begin, base);
  for (int key0 = begin; key0 < end; key0 += 2 * BN) {  // two tiles: the buffers are constants of the addresses
    step(key0, base, base + kTile);
    if (key0 + BN < end) step(key0 + BN, base + kTile, base);
  }

  l = swap_add(l);
  if constexpr (FEW) {  // the other groups' sums and accumulators through LDS
    static_assert(!FEW || G == 2, "one other group");
    float* const box = (float*)smem + map * (NT * 16 + 2) * 64 + lane;
    __syncthreads();
    if (group == 1) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) box[(i * 16 + j) * 64] = acc[i][j];
      box[NT * 16 * 64] = m, box[(NT * 16 + 1) * 64] = l;
    }
    __syncthreads();
    if (group == 0) {
      const float om = box[NT * 16 * 64], n = fmaxf(m, om), u = n == -INFINITY ? 0.f : n;
      const float c = __builtin_amdgcn_exp2f(m - u), o = __builtin_amdgcn_exp2f(om - u);
      l = l * c + box[(NT * 16 + 1) * 64] * o;
      m = n;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = acc[i][j] * c + box[(i * 16 + j) * 64] * o;
    }
  }
  if (!row.in) m = -INFINITY, l = 0.f;
  const bool mine = !FEW || group == 0;
  const int head = kvh * a.g + row.h;
  if (a.splits > 1) {  // unnormalised, with its maximum and sum: (split, row, head, 2, 4 + dv)
    if (!row.out || !mine) return;
    float* p = a.part + ((((int64_t)blockIdx.z * a.nq + s.q0 + row.i) * a.hk * a.g + head) * 2 + map) * (a.dv + 4);
    if (half == 0) p[0] = m, p[1] = l;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 32 * i + 8 * j + 4 * half;
        if (c < a.dv) store4<float>(p + 4 + c, acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]);
      }
    return;
  }
  __syncthreads();
  float* const box = (float*)smem + (FEW ? 0 : group) * NT * 16 * 64 + lane;
  const bool some = l != 0.f;  // false: no key, zero rows; a NaN stays one
  const float inv = 1.f / l;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[i][j] = some ? acc[i][j] * inv : 0.f;
  const int64_t at = s.q0 + row.i;
  if (row.out && mine) {
    if (a.lse && half == 0) store_sums(a, stat_at(a, kvh, map, at, row.h), m, l, some);
    if (a.maps) {
      float* const p = a.maps + ((at * a.hk * a.g + head) * 2 + map) * a.dv;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = 32 * i + 8 * j + 4 * half;
          if (c < a.dv) store4<float>(p + c, acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]);
        }
    }
  }
  if (map == 1 && mine) {
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) box[(i * 16 + j) * 64] = acc[i][j];
  }
  __syncthreads();
  if (map == 1 || !row.out || !mine) return;
  const float lam = a.lam[head];
  T* const p = (T*)a.out + (at * a.hk * a.g + head) * a.dv;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 32 * i + 8 * j + 4 * half;
      if (c < a.dv) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = fmaf(-lam, box[(i * 16 + 4 * j + e) * 64], acc[i][4 * j + e]);
        store4<T>(p + c, y[0], y[1], y[2], y[3]);
      }
    }
}

// Few rows (a token over a cache; in 32 bits five rows and more): the NW waves own the same 32 packed rows, both maps, and every wave streams
// key tiles of its own (no barrier), joined at the end; with a.splits > 1 the keys are dealt over blockIdx.z and the partials joined by the next
// launch.  Bound: HBM.  8 tokens over caches of up to 32 768 keys, 16 heads on 4, 64, 128, bf16: 81 us, 4.9 of the 5.1 TB/s of a large copy, and
// 6 us for the join (with the two maps' waves sharing tiles behind barriers, 103).  4 tokens of 32 heads on 4 over 8 192 keys, 32, 64, 32 bits:
// 26 us, 13 at the copy's rate.  P is rounded to the type before its product.
template <typename T, int DB, int DVB, int NW>
__global__ __launch_bounds__(NW * 64, (kWaves<T, DB, DVB>)) void fwd_keys_kernel(Args a) {
  using Frag = typename Ops<T>::Frag;
  constexpr int CK = 2 * DB * (int)sizeof(T) / 16, CV = DVB * (int)sizeof(T) / 16, NT = DVB / 32, QS = DB / kStep<T>;
  constexpr int BN = 32, TILE = 32, kTile = BN * (CK + CV) * 16, kJoin = (NW / 2) * 64 * (2 * NT * 16 + 4) * 4;
  constexpr int kSmem = kTile * NW > kJoin ? kTile * NW : kJoin;
  __shared__ __attribute__((aligned(1024))) char smem[kSmem];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
  const int kvh = a.stacked ? blockIdx.x : blockIdx.x % a.hk;
  const Seq s = find_seq<TILE, false>(a, a.stacked ? 0 : a.seq0 + blockIdx.x / a.hk, a.tile0 + blockIdx.y, a.tiles);
  T* const out = (T*)a.out;
  if (s.tile < 0) {
    zero_rows<T>(a, s, kvh, NW * 64);
    return;
  }
  const int row_base = s.tile * TILE;
  if (row_base >> a.gsh >= (a.stacked ? s.n : a.n)) return;
  const int r = row_base + col;
  const Row row = row_of(a, s, r);

  // Q: B operand, lane = row, straight from global memory
  Frag q1[QS], q2[QS];
  {
    const auto rq = buffer((const T*)a.q.data + s.b * a.q.batch_stride + (a.stacked ? s.q0 : 0) * a.q.row_stride +
                           (int64_t)kvh * 2 * a.g * a.q.head_stride + (int64_t)(row_base >> a.gsh) * a.q.row_stride);
    const int o = (int)(((row.i - (row_base >> a.gsh)) * a.q.row_stride + 2 * row.h * a.q.head_stride) * (int)sizeof(T));
    const int hs = (int)(a.q.head_stride * sizeof(T));
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      const int c = (2 * i + half) * kE<T>;
      const bool in = row.in && c < a.d;
      q1[i] = load_frag<T>(rq, in ? o + c * (int)sizeof(T) : kOutside);
      q2[i] = load_frag<T>(rq, in ? o + hs + c * (int)sizeof(T) : kOutside);
    }
  }
#pragma unroll
  for (int i = 0; i < QS; ++i) arrived(q1[i]), arrived(q2[i]);
  f32x16 acc1[NT], acc2[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) acc1[i] = zero16(), acc2[i] = zero16();
  float m1 = -INFINITY, m2 = -INFINITY, l1 = 0.f, l2 = 0.f;
  bool huge = false;

  const T* const kp = (const T*)a.k.data + s.b * a.k.batch_stride + (a.stacked ? s.k0 : 0) * a.k.row_stride + (int64_t)kvh * 2 * a.k.head_stride;
  const T* const vp = (const T*)a.v.data + s.b * a.v.batch_stride + (a.stacked ? s.k0 : 0) * a.v.row_stride + (int64_t)kvh * a.v.head_stride;
  const int off = s.m - s.n;                         // causal: key j for query i iff j <= i + off
  const int limit = a.causal ? row.i + off : 0x7fffffff;
  int end = s.m;
  if (a.causal) {  // no key beyond the last row's limit
    const int last = min((row_base + TILE - 1) >> a.gsh, s.n - 1);
    end = min(end, max(0, last + off + 1));
  }
  int begin = 0;
  if (a.splits > 1) split_keys(a, begin, end);

  const int krs = (int)(a.k.row_stride * sizeof(T)), vrs = (int)(a.v.row_stride * sizeof(T)), hs = (int)(a.k.head_stride * sizeof(T));
  auto fill = [&](unsigned tile, int key0, uint64_t bits) GEOTR_INLINE {
    const auto rk = words(kp + (int64_t)key0 * a.k.row_stride), rv = words(vp + (int64_t)key0 * a.v.row_stride);
    if (bits == 0xffffffffull) {
      stage_at<T, 32, 2, DB, 1>(tile, rk, a.d, hs, 0, lane, [&](int x) { return x * krs; });
      stage_at<T, 32, 1, DVB, 1>(tile + BN * CK * 16, rv, a.dv, 0, 0, lane, [&](int x) { return x * vrs; });
    } else {
      stage_at<T, 32, 2, DB, 1>(tile, rk, a.d, hs, 0, lane, [&](int x) { return (bits >> x) & 1 ? x * krs : kOutside; });
      stage_at<T, 32, 1, DVB, 1>(tile + BN * CK * 16, rv, a.dv, 0, 0, lane, [&](int x) { return (bits >> x) & 1 ? x * vrs : kOutside; });
    }
  };

  const Rows<T, CK> krow(col, half);
  const Cols<T, CV> vcol(lane);
  // 32 keys of a staged tile
  auto consume = [&](const char* at, int sub, int key0, uint64_t bits) GEOTR_INLINE {
    const unsigned tile = lds_at(at), vt = tile + BN * CK * 16;
    f32x16 s1 = zero16(), s2 = zero16();
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      Ops<T>::mma(s1, krow.get(tile, 32 * sub, i), q1[i]);
      Ops<T>::mma(s2, krow.get(tile, 32 * sub, CK / 4 + i), q2[i]);
    }
    const int k0 = key0 + 32 * sub;
    unsigned lo = (unsigned)(bits >> (32 * sub));
    const int above = limit - k0;  // keys of the tile up to this one
    if (lo != 0xffffffffu || __any(above < 31)) {
      if (above < 31) lo = above < 0 ? 0u : lo & ((2u << above) - 1);
      lo >>= 4 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool in = (lo >> (8 * (i / 4) + i % 4)) & 1;
        s1[i] = in ? s1[i] : -INFINITY;
        s2[i] = in ? s2[i] : -INFINITY;
      }
    }
    float x1 = s1[0], x2 = s2[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) x1 = fmaxf(x1, s1[i]), x2 = fmaxf(x2, s2[i]);
    x1 = swap_max(x1) * a.scale_log2, x2 = swap_max(x2) * a.scale_log2;
    // the accumulators are rescaled only when a maximum grew by more than 2^8: weights stay below 2^8, sums are exact either way
    if (__any(x1 > m1 + 8.f || x2 > m2 + 8.f)) {
      const float n1 = fmaxf(m1, x1), n2 = fmaxf(m2, x2);
      const float c1 = n1 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m1 - n1), c2 = n2 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m2 - n2);
      m1 = n1, m2 = n2, l1 *= c1, l2 *= c2;
      huge = __any((fabsf(m1) > kHuge && m1 > -INFINITY) || (fabsf(m2) > kHuge && m2 > -INFINITY));
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc1[i][j] *= c1, acc2[i][j] *= c2;
    }
    const float b1 = m1 == -INFINITY ? 0.f : m1, b2 = m2 == -INFINITY ? 0.f : m2;
    exponents(s1, a.scale_log2, [&](int) { return b1; }, huge);
    exponents(s2, a.scale_log2, [&](int) { return b2; }, huge);
#pragma unroll
    for (int i = 0; i < 16; ++i) l1 += s1[i], l2 += s2[i];
#pragma unroll
    for (int p = 0; p < kPSteps<T>; ++p) {
      const Frag p1 = pack<T>(s1, p), p2 = pack<T>(s2, p);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const Frag f = vcol.get(vt, 32 * sub, p, i);
        Ops<T>::mma(acc1[i], f, p1);
        Ops<T>::mma(acc2[i], f, p2);
      }
    }
  };

  char* const mine = smem + wave * kTile;
  for (int key0 = begin + 32 * wave; key0 < end; key0 += 32 * NW) {
    const uint64_t bits = key_bits(a, s, key0, end, lane) & 0xffffffffull;
    if (!bits) continue;
    fill(lds_at(mine), key0, bits);
    tile_ready();  // this wave's own: no barrier
    consume(mine, 0, key0, bits);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }

  l1 = swap_add(l1), l2 = swap_add(l2);
  {  // join the waves' partials, the upper half of them through LDS, twice
#pragma unroll
    for (int step = NW / 2; step >= 1; step /= 2) {
      __syncthreads();
      float* const box = (float*)smem + (wave % step) * 64 * (2 * NT * 16 + 4);
      if (wave >= step && wave < 2 * step) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) box[(i * 16 + j) * 64 + lane] = acc1[i][j], box[((NT + i) * 16 + j) * 64 + lane] = acc2[i][j];
        float* st = box + 2 * NT * 16 * 64;
        st[lane] = m1, st[64 + lane] = m2, st[128 + lane] = l1, st[192 + lane] = l2;
      }
      __syncthreads();
      if (wave < step) {
        const float* st = box + 2 * NT * 16 * 64;
        const float om1 = st[lane], om2 = st[64 + lane], n1 = fmaxf(m1, om1), n2 = fmaxf(m2, om2);
        const float u1 = n1 == -INFINITY ? 0.f : n1, u2 = n2 == -INFINITY ? 0.f : n2;
        const float c1 = __builtin_amdgcn_exp2f(m1 - u1), c2 = __builtin_amdgcn_exp2f(m2 - u2);
        const float d1 = __builtin_amdgcn_exp2f(om1 - u1), d2 = __builtin_amdgcn_exp2f(om2 - u2);
        l1 = l1 * c1 + st[128 + lane] * d1, l2 = l2 * c2 + st[192 + lane] * d2;
        m1 = n1, m2 = n2;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            acc1[i][j] = acc1[i][j] * c1 + box[(i * 16 + j) * 64 + lane] * d1;
            acc2[i][j] = acc2[i][j] * c2 + box[((NT + i) * 16 + j) * 64 + lane] * d2;
          }
      }
    }
    if (wave) return;
  }

  if (!row.out) return;
  if (!row.in) m1 = m2 = -INFINITY, l1 = l2 = 0.f;
  const int64_t at = s.q0 + row.i;
  const int head = kvh * a.g + row.h;
  if (a.splits > 1) {  // unnormalised, with its maximum and sum: (split, row, head, 2, 4 + dv)
    const int w = a.dv + 4;
    float* p1 = a.part + (((int64_t)blockIdx.z * a.nq + at) * a.hk * a.g + head) * 2 * w;
    float* p2 = p1 + w;
    if (half == 0) p1[0] = m1, p1[1] = l1, p2[0] = m2, p2[1] = l2;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = 32 * i + 8 * j + 4 * half;
        if (c < a.dv) {
          store4<float>(p1 + 4 + c, acc1[i][4 * j], acc1[i][4 * j + 1], acc1[i][4 * j + 2], acc1[i][4 * j + 3]);
          store4<float>(p2 + 4 + c, acc2[i][4 * j], acc2[i][4 * j + 1], acc2[i][4 * j + 2], acc2[i][4 * j + 3]);
        }
      }
    return;
  }
  const float lam = a.lam[head];
  const bool some = l1 != 0.f;  // false: no key (the maps share their keys), zero rows; a NaN stays one
  const float i1 = 1.f / l1, i2 = 1.f / l2;
  T* const po = out + (at * a.hk * a.g + head) * a.dv;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 32 * i + 8 * j + 4 * half;
      if (c < a.dv) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = some ? fmaf(-lam, acc2[i][4 * j + e] * i2, acc1[i][4 * j + e] * i1) : 0.f;
        store4<T>(po + c, y[0], y[1], y[2], y[3]);
      }
    }
}

// A row or a few of them in 32 bits: a matrix product of 32 rows takes as long for one (6 144 cycles for 32 keys at 32, 64), so these are
// vector instructions.  A wave load is whole rows of K, 16 bytes a lane, LK lanes to the two maps of a key, KPL keys; sums of q . k over the
// lanes of a map by DPP; the same lanes then take VE channels of the key's row of V.  Every key slot of a wave keeps a softmax of its own (no
// exchange between slots, nothing in LDS), joined at the end.  Bound: latency at one row of 257 keys (6.0 us; the tiles below took 18.3), HBM on
// long caches: 4 tokens over 8 192 keys, 4 heads, 64, 128: 24 us, 5.6 TB/s from the caches (52 by tiles); 128, 256: 49 us (155).
// dpp: lanes of a row of 16; swap: the pair (rows or halves of the first map, of the second), each in both places
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}
// the values of the first and the second map's lanes of a key, LK lanes to a key
template <int LK>
__device__ __forceinline__ void both(float x, bool second, float& one, float& two) {
  if constexpr (LK == 16) {
    const float o = dpp<0x128>(x);  // row_ror:8
    one = second ? o : x, two = second ? x : o;
  } else {
    const auto w = LK == 32 ? __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false)
                            : __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    one = __uint_as_float(w[0]), two = __uint_as_float(w[1]);
  }
}
template <int DB, int DVB, int R>
__global__ __launch_bounds__(512) void fwd_rows_kernel(Args a) {
  constexpr int NW = 8, U = 8, LK = DB / 2, KPL = 64 / LK, VE = DVB / LK, BN = U * KPL, W = 2 * DVB + 4;
  static_assert((VE == 2 || VE == 4) && R <= NW, "values of a lane, a row to a wave at the end");
  __shared__ __attribute__((aligned(16))) float box[NW][R][W];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int slot = lane / LK, in_slot = lane % LK, map = in_slot / (LK / 2), chunk = in_slot % (LK / 2);
  const int kvh = a.stacked ? blockIdx.x : blockIdx.x % a.hk;
  const Seq s = find_seq<R, false>(a, a.stacked ? 0 : a.seq0 + blockIdx.x / a.hk, a.tile0 + blockIdx.y, a.tiles);
  if (s.tile < 0) {
    zero_rows<float>(a, s, kvh, NW * 64);
    return;
  }
  const int row_base = s.tile * R, i0 = row_base >> a.gsh, off = s.m - s.n;
  if (i0 >= (a.stacked ? s.n : a.n)) return;
  const auto rq = buffer((const float*)a.q.data + s.b * a.q.batch_stride + ((a.stacked ? s.q0 : 0) + i0) * a.q.row_stride +
                         (int64_t)kvh * 2 * a.g * a.q.head_stride);
  f32x4 q[R];
  float m[R], l[R], acc1[R][VE], acc2[R][VE];
  int limit[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const Row row = row_of(a, s, row_base + r);
    q[r] = load_frag<float>(rq, row.in && 4 * chunk < a.d ? (int)(((row.i - i0) * a.q.row_stride + (2 * row.h + map) * a.q.head_stride + 4 * chunk) * 4) : kOutside);
    limit[r] = a.causal ? row.i + off : 0x7fffffff;
    m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
    for (int e = 0; e < VE; ++e) acc1[r][e] = acc2[r][e] = 0.f;
  }
  const float* const kp = (const float*)a.k.data + s.b * a.k.batch_stride + (a.stacked ? s.k0 : 0) * a.k.row_stride + (int64_t)kvh * 2 * a.k.head_stride;
  const float* const vp = (const float*)a.v.data + s.b * a.v.batch_stride + (a.stacked ? s.k0 : 0) * a.v.row_stride + (int64_t)kvh * a.v.head_stride;
  int begin = 0, end = s.m;
  if (a.causal) end = min(end, max(0, min((row_base + R - 1) >> a.gsh, s.n - 1) + off + 1));  // no key beyond the last row's limit
  if (a.splits > 1) split_keys(a, begin, end);
  const int krs = (int)(a.k.row_stride * 4), vrs = (int)(a.v.row_stride * 4);
  const int ko = 4 * chunk < a.d ? (int)(map * a.k.head_stride + 4 * chunk) * 4 : kOutside, vo = VE * in_slot < a.dv ? VE * in_slot * 4 : kOutside;
  using Vec = __attribute__((ext_vector_type(VE))) float;
  for (int key0 = begin + wave * BN; key0 < end; key0 += NW * BN) {
    const uint64_t bits = key_bits(a, s, key0, end, lane) >> slot;
    const auto rk = buffer(kp + (int64_t)key0 * a.k.row_stride), rv = buffer(vp + (int64_t)key0 * a.v.row_stride);
    f32x4 k[U];
    Vec v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = load_frag<float>(rk, (bits >> (u * KPL)) & 1 && ko != kOutside ? (u * KPL + slot) * krs + ko : kOutside);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int o = (bits >> (u * KPL)) & 1 && vo != kOutside ? (u * KPL + slot) * vrs + vo : kOutside;
      if constexpr (VE == 4) v[u] = load_frag<float>(rv, o);
      else v[u] = __builtin_bit_cast(Vec, __builtin_amdgcn_raw_buffer_load_b64(rv, o, 0, 0));
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float x[U], top = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float t = q[r][0] * k[u][0];
#pragma unroll
        for (int e = 1; e < 4; ++e) t = fmaf(q[r][e], k[u][e], t);
        t += dpp<0xB1>(t);   // quad_perm [1,0,3,2]
        t += dpp<0x4E>(t);   // quad_perm [2,3,0,1]
        t += dpp<0x141>(t);  // row_half_mirror: the sum of 8 lanes
        if constexpr (LK >= 32) t += dpp<0x140>(t);  // row_mirror: of 16
        if constexpr (LK == 64) {
          const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(t), __float_as_uint(t), false, false);
          t = __uint_as_float(w[0]) + __uint_as_float(w[1]);
        }
        const bool seen = (bits >> (u * KPL)) & 1 && key0 + u * KPL + slot <= limit[r];
        x[u] = seen ? t * a.scale_log2 : -INFINITY, top = fmaxf(top, x[u]);
      }
      const float n = fmaxf(m[r], top), from = n == -INFINITY ? 0.f : n, c = __builtin_amdgcn_exp2f(m[r] - from);
      float c1, c2;
      both<LK>(c, map, c1, c2);
      m[r] = n, l[r] *= c;
#pragma unroll
      for (int e = 0; e < VE; ++e) acc1[r][e] *= c1, acc2[r][e] *= c2;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = __builtin_amdgcn_exp2f(x[u] - from);
        float p1, p2;
        both<LK>(p, map, p1, p2);
        l[r] += p;
#pragma unroll
        for (int e = 0; e < VE; ++e) acc1[r][e] = fmaf(p1, v[u][e], acc1[r][e]), acc2[r][e] = fmaf(p2, v[u][e], acc2[r][e]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int o = LK; o < 64; o *= 2) {  // the wave's key slots
      const float om = __shfl_xor(m[r], o, 64), n = fmaxf(m[r], om), from = n == -INFINITY ? 0.f : n;
      const float c = __builtin_amdgcn_exp2f(m[r] - from), d = __builtin_amdgcn_exp2f(om - from);
      float c1, c2, d1, d2;
      both<LK>(c, map, c1, c2), both<LK>(d, map, d1, d2);
      m[r] = n, l[r] = l[r] * c + __shfl_xor(l[r], o, 64) * d;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        acc1[r][e] = acc1[r][e] * c1 + __shfl_xor(acc1[r][e], o, 64) * d1;
        acc2[r][e] = acc2[r][e] * c2 + __shfl_xor(acc2[r][e], o, 64) * d2;
      }
    }
    if (lane < LK) {
#pragma unroll
      for (int e = 0; e < VE; ++e) box[wave][r][VE * in_slot + e] = acc1[r][e], box[wave][r][DVB + VE * in_slot + e] = acc2[r][e];
      if (chunk == 0) box[wave][r][2 * DVB + map] = m[r], box[wave][r][2 * DVB + 2 + map] = l[r];
    }
  }
  __syncthreads();
  if (wave >= R) return;
  const Row row = row_of(a, s, row_base + wave);
  const int c = 4 * lane;
  if (!row.out) return;
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, y[2][4] = {};
#pragma unroll
  for (int x = 0; x < 2; ++x) {
#pragma unroll
    for (int w = 0; w < NW; ++w) top[x] = fmaxf(top[x], box[w][wave][2 * DVB + x]);
    const float from = top[x] == -INFINITY ? 0.f : top[x];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(box[w][wave][2 * DVB + x] - from);
      sum[x] = fmaf(box[w][wave][2 * DVB + 2 + x], f, sum[x]);
      if (c < DVB) {
        const f32x4 t = *(const f32x4*)&box[w][wave][x * DVB + c];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[x][e] = fmaf(t[e], f, y[x][e]);
      }
    }
    if (!row.in) top[x] = -INFINITY, sum[x] = 0.f;
  }
  const int64_t at = s.q0 + row.i;
  const int head = kvh * a.g + row.h;
  if (a.splits > 1) {  // unnormalised, with its maximum and sum: (split, row, head, 2, 4 + dv)
    float* const p = a.part + (((int64_t)blockIdx.z * a.nq + at) * a.hk * a.g + head) * 2 * (a.dv + 4);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (lane == 0) p[x * (a.dv + 4)] = top[x], p[x * (a.dv + 4) + 1] = sum[x];
      if (c < a.dv) store4<float>(p + x * (a.dv + 4) + 4 + c, y[x][0], y[x][1], y[x][2], y[x][3]);
    }
    return;
  }
  const float lam = a.lam[head], f1 = 1.f / sum[0], f2 = 1.f / sum[1];
  const bool some = sum[0] != 0.f;  // false: no key, zero rows; a NaN stays one
#pragma unroll
  for (int e = 0; e < 4; ++e) y[0][e] = some ? fmaf(-lam, y[1][e] * f2, y[0][e] * f1) : 0.f;
  if (c < a.dv) store4<float>((float*)a.out + (at * a.hk * a.g + head) * a.dv + c, y[0][0], y[0][1], y[0][2], y[0][3]);
}

// ---- backward: query rows (dQ, sum of P2 dP) --------------------------------------------------------------------------------------------
// fp16: the power of two that brings |dP - del| <= 2 Dv max|dout| max|v| below 2^15, so that dS neither overflows nor underflows for the small
// gradients of a mean loss; 1 for the types with the exponent range of 32 bits
template <typename T>
__device__ __forceinline__ float grad_scale(const Args& a) {
  if constexpr (Narrow<T>::value) {
    const float top = 2.f * a.dv * a.amax[0] * a.amax[1];
    if (top > 0.f && top < INFINITY) return ldexpf(1.f, 14 - ilogbf(top));
  }
  return 1.f;
}

// A wave owns 32 packed rows.  Where two tiles of 64 keys fit into LDS the four waves are two groups of rows x two of the keys, joined at the
// end: blocks of 64 rows fill the chip at half the rows, and the longest causal block ends after half the steps (2 x 4 096 causal rows, 8
// heads, 64, 128: 175 -> 157 us, 147 by now; 128, 256 at 2 x 2 048 and 4 heads: 187 -> 116).  Bound: latency of 1.6 waves to a SIMD unit (matrix
// core busy 0.31, vector instructions 0.46, 0.30 of a wave's life in waits for data), 0.70 PFLOP/s.  dS is rounded to the type before its product.
template <typename T, int DB, int DVB>
constexpr int kKeyGroups = 128 * (2 * DB + DVB) * (int)sizeof(T) <= 131072 ? 2 : 1;
template <typename T, int DB, int DVB, int NW>
constexpr int kSmemQ() {
  constexpr int KG = kKeyGroups<T, DB, DVB>, kTile = 32 * KG * (2 * DB + DVB) * (int)sizeof(T), NB = 2 * kTile <= 131072 ? 2 : 1;
  constexpr int kJoin = KG == 1 ? 0 : NW / KG * (2 * DB / 32 * 16 + 1) * 64 * 4;
  return NB * kTile > kJoin ? NB * kTile : kJoin;
}
// block `y` of `blocks` of a head
template <typename T, int DB, int DVB, int NW>
__device__ __forceinline__ void dq_block(const Args& a, char* smem, int y, int blocks) {
  using Frag = typename Ops<T>::Frag;
  constexpr int CK = 2 * DB * (int)sizeof(T) / 16, CV = DVB * (int)sizeof(T) / 16, ND = DB / 32, QS = DB / kStep<T>, VS = DVB / kStep<T>;
  constexpr int KG = kKeyGroups<T, DB, DVB>, RG = NW / KG, BN = 32 * KG, TILE = 32 * RG;
  constexpr int kTile = BN * (CK + CV) * 16, NB = 2 * kTile <= 131072 ? 2 : 1;
  constexpr uint64_t kAll = BN == 64 ? ~0ull : 0xffffffffull;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
  const int kvh = a.stacked ? blockIdx.x : blockIdx.x % a.hk;
  const int rg = wave % RG, kg = wave / RG;
  const int t = tile_order(a, y, blocks, gridDim.x, 256 * kWaves<T, DB, DVB>);
  const Seq s = find_seq<TILE, false>(a, a.stacked ? 0 : a.seq0 + blockIdx.x / a.hk, t, blocks);
  T* const dq = (T*)a.gq;
  if (s.tile < 0) {
    const int64_t rows = s.q_end < a.nq ? a.nq - s.q_end : 0, per = (int64_t)a.g * 2 * a.d;
    for (int64_t e = (int64_t)s.spare * (NW * 64) + threadIdx.x; e < rows * per; e += (int64_t)s.spares * (NW * 64)) {
      const int64_t i = e / per;
      dq[((s.q_end + i) * a.hk + kvh) * per + (e - i * per)] = (T)0.f;
    }
    for (int64_t e = (int64_t)s.spare * (NW * 64) + threadIdx.x; e < rows * a.g; e += (int64_t)s.spares * (NW * 64))
      a.drow[((int64_t)kvh * a.nq + s.q_end) * a.g + e] = 0.f;
    return;
  }
  const int row_base = s.tile * TILE;
  if (row_base >> a.gsh >= (a.stacked ? s.n : a.n)) return;
  const int r = row_base + 32 * rg + col;
  const Row row = row_of(a, s, r);
  const int64_t at = s.q0 + row.i;
  const int head = kvh * a.g + row.h;
  const float gs = grad_scale<T>(a);

  Frag q1[QS], q2[QS], go[VS];
  {
    const int i0 = row_base >> a.gsh;
    const auto rq = buffer((const T*)a.q.data + s.b * a.q.batch_stride + ((a.stacked ? s.q0 : 0) + i0) * a.q.row_stride +
                           (int64_t)kvh * 2 * a.g * a.q.head_stride);
    const auto ro = buffer((const T*)a.dout.data + s.b * a.dout.batch_stride + ((a.stacked ? s.q0 : 0) + i0) * a.dout.row_stride +
                           (int64_t)kvh * a.g * a.dout.head_stride);
    const int oq = (int)(((row.i - i0) * a.q.row_stride + 2 * row.h * a.q.head_stride) * (int)sizeof(T)), hs = (int)(a.q.head_stride * sizeof(T));
    const int oo = (int)(((row.i - i0) * a.dout.row_stride + row.h * a.dout.head_stride) * (int)sizeof(T));
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      const int c = (2 * i + half) * kE<T>;
      const bool in = row.in && c < a.d;
      q1[i] = load_frag<T>(rq, in ? oq + c * (int)sizeof(T) : kOutside);
      q2[i] = load_frag<T>(rq, in ? oq + hs + c * (int)sizeof(T) : kOutside);
    }
#pragma unroll
    for (int i = 0; i < VS; ++i) {
      const int c = (2 * i + half) * kE<T>;
      go[i] = load_frag<T>(ro, row.in && c < a.dv ? oo + c * (int)sizeof(T) : kOutside);
    }
  }
  float lse1 = INFINITY, lse2 = INFINITY, rest1 = 0.f, rest2 = 0.f, del1 = 0.f, del2 = 0.f, lam = 0.f;
  if (row.in) {
    const int64_t st = stat_at(a, kvh, 0, at, row.h);
    lse1 = a.lse[st], lse2 = a.lse[st + a.nq * a.g], rest1 = a.lse[st + 2 * a.nq * a.g], rest2 = a.lse[st + 3 * a.nq * a.g], lam = a.lam[head];
    const int64_t rs = row_stat_at(a, kvh, 1, at, row.h);
    del1 = a.rows[rs], del2 = a.rows[rs + 1];
  }
  arrived(lse1), arrived(lse2), arrived(rest1), arrived(rest2), arrived(del1), arrived(del2), arrived(lam);
#pragma unroll
  for (int i = 0; i < QS; ++i) arrived(q1[i]), arrived(q2[i]);
#pragma unroll
  for (int i = 0; i < VS; ++i) arrived(go[i]);
  const bool huge = __any((fabsf(lse1) > kHuge && lse1 < INFINITY) || (fabsf(lse2) > kHuge && lse2 < INFINITY));
  f32x16 acc1[ND], acc2[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i) acc1[i] = zero16(), acc2[i] = zero16();
  float dsum = 0.f;

  const T* const kp = (const T*)a.k.data + s.b * a.k.batch_stride + (a.stacked ? s.k0 : 0) * a.k.row_stride + (int64_t)kvh * 2 * a.k.head_stride;
  const T* const vp = (const T*)a.v.data + s.b * a.v.batch_stride + (a.stacked ? s.k0 : 0) * a.v.row_stride + (int64_t)kvh * a.v.head_stride;
  const int off = s.m - s.n;
  const int limit = a.causal ? row.i + off : 0x7fffffff;
  int end = s.m;
  if (a.causal) {
    const int last = min((row_base + TILE - 1) >> a.gsh, s.n - 1);
    end = min(end, max(0, last + off + 1));
  }
  const int krs = (int)(a.k.row_stride * sizeof(T)), vrs = (int)(a.v.row_stride * sizeof(T));
  const Stage<T, BN, 2, DB, NW> kst(a.d, (int)(a.k.head_stride * sizeof(T)), wave, lane, [&](int x) { return x * krs; });
  const Stage<T, BN, 1, DVB, NW> vst(a.dv, 0, wave, lane, [&](int x) { return x * vrs; });
  auto fill = [&](unsigned tile, int key0, uint64_t bits) GEOTR_INLINE {
    kst.load(tile, words(kp + (int64_t)key0 * a.k.row_stride), 16 * krs, wave, bits);
    vst.load(tile + BN * CK * 16, words(vp + (int64_t)key0 * a.v.row_stride), 16 * vrs, wave, bits);
  };
  const Rows<T, CK> krow(col, half);
  const Rows<T, CV> vrow(col, half);
  const Cols<T, CK> kcol(lane);
  auto consume = [&](unsigned at, int key0, uint64_t bits) GEOTR_INLINE {
    const unsigned tile = at + kg * 32 * CK * 16, vt = at + BN * CK * 16 + kg * 32 * CV * 16;
    unsigned lo = (unsigned)(bits >> (32 * kg));
    if (!lo) return;
    key0 += 32 * kg;
    f32x16 s1 = zero16(), s2 = zero16(), dp = zero16();
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      Ops<T>::mma(s1, krow.get(tile, 0, i), q1[i]);
      Ops<T>::mma(s2, krow.get(tile, 0, CK / 4 + i), q2[i]);
    }
    if constexpr (kWaves<T, DB, DVB> == 1 && !(sizeof(T) == 4 && DB == 128)) {
#pragma unroll
      for (int i = 0; i < ND; ++i) held(acc1[i]), held(acc2[i]);
    }
#pragma unroll
    for (int i = 0; i < VS; ++i) Ops<T>::mma(dp, vrow.get(vt, 0, i), go[i]);
    const int above = limit - key0;
    if (above < 31) lo = above < 0 ? 0u : lo & ((2u << above) - 1);
    const bool some = __any(lo != 0xffffffffu);
    lo >>= 4 * half;
    exponents(s1, a.scale_log2, [&](int) { return lse1; }, huge, rest1);
    exponents(s2, a.scale_log2, [&](int) { return lse2; }, huge, rest2);
    if (__builtin_expect(some, 0)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool in = (lo >> (8 * (i / 4) + i % 4)) & 1;
        s1[i] = in ? s1[i] : 0.f, s2[i] = in ? s2[i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float p1 = s1[i], p2 = s2[i];
      dsum = fmaf(p2, dp[i], dsum);
      s1[i] = p1 * (dp[i] - del1), s2[i] = p2 * (dp[i] - del2);
      if constexpr (Narrow<T>::value) s1[i] *= gs, s2[i] *= gs;
    }
#pragma unroll
    for (int p = 0; p < kPSteps<T>; ++p) {
      const Frag d1 = pack<T>(s1, p), d2 = pack<T>(s2, p);
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        Ops<T>::mma(acc1[i], kcol.get(tile, 0, p, i), d1);
        Ops<T>::mma(acc2[i], kcol.get(tile, 0, p, ND + i), d2);
      }
    }
  };
  const unsigned base = lds_at(smem);
  if constexpr (NB == 2) {
    int which = 0;
    uint64_t bits = key_bits(a, s, 0, end, lane) & kAll;
    if (0 < end) fill(base, 0, bits);
    for (int key0 = 0; key0 < end; key0 += BN) {
      tile_ready();
      __syncthreads();
      uint64_t next = 0;
      if (key0 + BN < end) {
        next = key_bits(a, s, key0 + BN, end, lane) & kAll;
        fill(base + (kTile - which), key0 + BN, next);
      }
      consume(base + which, key0, bits);
      bits = next;
      which = kTile - which;
    }
  } else {
    for (int key0 = 0; key0 < end; key0 += BN) {
      const uint64_t bits = key_bits(a, s, key0, end, lane) & kAll;
      if (!bits) continue;
      __syncthreads();
      fill(base, key0, bits);
      tile_ready();
      __syncthreads();
      consume(base, key0, bits);
    }
  }
  if constexpr (KG == 2) {
    float* const box = (float*)smem + rg * (2 * ND * 16 + 1) * 64 + lane;
    __syncthreads();
    if (kg == 1) {
#pragma unroll
      for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) box[(i * 16 + j) * 64] = acc1[i][j], box[((ND + i) * 16 + j) * 64] = acc2[i][j];
      box[2 * ND * 16 * 64] = dsum;
    }
    __syncthreads();
    if (kg == 1) return;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc1[i][j] += box[(i * 16 + j) * 64], acc2[i][j] += box[((ND + i) * 16 + j) * 64];
    dsum += box[2 * ND * 16 * 64];
  }
  if (!row.out) return;
  dsum = swap_add(dsum);
  if (!row.in) dsum = 0.f;
  if (half == 0) a.drow[((int64_t)kvh * a.nq + at) * a.g + row.h] = dsum;
  const float f = a.scale / gs, f2 = -lam * f;
  T* const p1 = dq + (at * a.hk * a.g + head) * 2 * a.d;
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 32 * i + 8 * j + 4 * half;
      if (c < a.d) {
        if (row.in) {
          store4<T>(p1 + c, acc1[i][4 * j] * f, acc1[i][4 * j + 1] * f, acc1[i][4 * j + 2] * f, acc1[i][4 * j + 3] * f);
          store4<T>(p1 + a.d + c, acc2[i][4 * j] * f2, acc2[i][4 * j + 1] * f2, acc2[i][4 * j + 2] * f2, acc2[i][4 * j + 3] * f2);
        } else {
          store4<T>(p1 + c, 0.f, 0.f, 0.f, 0.f);
          store4<T>(p1 + a.d + c, 0.f, 0.f, 0.f, 0.f);
        }
      }
    }
}
template <typename T, int DB, int DVB, int NW>
__global__ __launch_bounds__(NW * 64, (kWaves<T, DB, DVB>)) void dq_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) char smem[kSmemQ<T, DB, DVB, NW>()];
  dq_block<T, DB, DVB, NW>(a, smem, a.tile0 + blockIdx.y, a.tiles);
}

// ---- backward: keys (dK, dV) --------------------------------------------------------------------------------------------------------------
// A wave owns 32 keys; K and V are the B operands (lane = key).  16-bit K and V stay in registers, V of wide heads in LDS; in 32 bits they are
// read again from memory for every tile of 32 packed query rows (a product takes 16 times as long as the load; held: 136 against 129 us at
// 32 clouds of 295, spilled).  Bound: latency of one wave to a SIMD unit (matrix core busy 0.24, vector instructions 0.36), 0.55 PFLOP/s at
// 2 x 4 096 causal rows, 8 heads, 64, 128 (251 us); two waves spill (989 us).  Where both gradients' accumulators leave no registers (16-bit heads
// of 128, values of 256) dK and dV are two launches, the scores twice: 20 instead of 16 products of d, 334 instead of 462 us at 2 x 2 048 rows and
// 4 heads (255 by now).  Narrower heads lose by it (64, 128: 370 against 274 us at 2 x 4 096 causal rows and 8 heads; 128, 128 at 2 x 2 048 and 4:
// 162 against 142).  P1 - lam P2 and dS are rounded to the type before their products.
enum Part { kBoth, kKeysOnly, kValuesOnly };
template <typename T, int DVB>
constexpr bool kSplitKV = sizeof(T) == 2 && DVB == 256;
template <typename T, int DB, int DVB, int PART>
constexpr int kWavesKV = DB <= 32 ? 2 : 1;
// V stays in LDS
template <typename T, int DB, int PART>
constexpr bool kLdsV = PART != kValuesOnly && sizeof(T) == 2 && (int)sizeof(T) * DB > 128;
// bytes of 32 query rows, of dout's, and of 8 x 32 numbers of the rows
template <typename T, int DB, int DVB>
constexpr int kRowTile = 32 * (2 * DB + DVB) * (int)sizeof(T) + 1024;
// QG = 2: the waves are two groups of keys x two of the query rows.  Not for 16-bit heads of 128 whose dK and dV are one launch: the tiles' second
// addresses spill 17 registers there, and accumulators are pinned only where nothing spills (held, above; 232 instead of 212 us at 2 x 2 048
// rows and 4 heads; spilled without the pins 312, dK and dV apart 252).
template <typename T, int DB, int DVB, int PART>
constexpr int kRowGroups = sizeof(T) == 2 && DB == 128 && PART == kBoth ? 1 : 4 * kRowTile<T, DB, DVB> + (kLdsV<T, DB, PART> ? 64 * DVB * (int)sizeof(T) : 0) <= 160 * 1024 ? 2 : 1;
template <typename T, int DB, int DVB, int NW, int PART, int QG>
constexpr int kSmemKV() {
  constexpr int kBuf = QG * kRowTile<T, DB, DVB>, NB = 2 * kBuf <= 140000 ? 2 : 1, kV = kLdsV<T, DB, PART> ? 32 * NW / QG * DVB * (int)sizeof(T) : 0;
  constexpr int kJoin = QG == 1 ? 0 : NW / QG * ((PART != kValuesOnly ? 2 * DB / 32 : 0) + (PART != kKeysOnly ? DVB / 32 : 0)) * 16 * 64 * 4;
  return NB * kBuf + kV > kJoin ? NB * kBuf + kV : kJoin;
}
template <typename T, int DB, int DVB, int NW, int PART, int QG>
__device__ __forceinline__ void dkv_block(const Args& a, char* smem, int y, int blocks) {
  using Frag = typename Ops<T>::Frag;
  constexpr int CQ = 2 * DB * (int)sizeof(T) / 16, CO = DVB * (int)sizeof(T) / 16, ND = DB / 32, NV = DVB / 32, QS = DB / kStep<T>, VS = DVB / kStep<T>;
  constexpr bool kHold = sizeof(T) == 2, kInLds = kLdsV<T, DB, PART>, kHoldV = PART != kValuesOnly && kHold && !kInLds;
  constexpr bool DK = PART != kValuesOnly, DV = PART != kKeysOnly;
  constexpr int KG = NW / QG, TILE = 32 * KG, BN = 32 * QG;
  constexpr int kRowBytes = 32 * (CQ + CO) * 16, kTile = kRowTile<T, DB, DVB>, kBuf = QG * kTile;
  constexpr int NB = 2 * kBuf <= 140000 ? 2 : 1;
  constexpr int kJoin = QG == 1 ? 0 : KG * ((DK ? 2 * ND : 0) + (DV ? NV : 0)) * 16 * 64 * 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
  const int kg = wave % KG, qg = wave / KG;
  const int kvh = a.stacked ? blockIdx.x : blockIdx.x % a.hk;
  const Seq s = find_seq<TILE, true>(a, a.stacked ? 0 : a.seq0 + blockIdx.x / a.hk, y, blocks);
  T* const dk = (T*)a.gk;
  T* const dv = (T*)a.gv;
  if (s.tile < 0) {
    const int64_t rows = s.k_end < a.nk ? a.nk - s.k_end : 0;
    for (int64_t e = (int64_t)s.spare * (NW * 64) + threadIdx.x; DK && e < rows * (2 * a.d); e += (int64_t)s.spares * (NW * 64)) {
      const int64_t i = e / (2 * a.d);
      dk[((s.k_end + i) * a.hk + kvh) * 2 * a.d + (e - i * 2 * a.d)] = (T)0.f;
    }
    for (int64_t e = (int64_t)s.spare * (NW * 64) + threadIdx.x; DV && e < rows * a.dv; e += (int64_t)s.spares * (NW * 64)) {
      const int64_t i = e / a.dv;
      dv[((s.k_end + i) * a.hk + kvh) * a.dv + (e - i * a.dv)] = (T)0.f;
    }
    return;
  }
  const int key_base = s.tile * TILE;
  const int keys_here = a.stacked ? s.m : a.m;
  if (key_base >= keys_here) return;
  const int key = key_base + 32 * kg + col;
  const bool in = key < s.m && !(a.masks && a.masks[s.k0 + key]);
  float gs = grad_scale<T>(a), boost = 1.f;
  bool minus = false;
  if constexpr (Narrow<T>::value) {  // fp16: P 2^8 in the product with dout, the weights of a long row stay normal numbers; less where |lam| > 2^6
    float most = 1.f;
    for (int h = 0; h < a.g; ++h) most = fmaxf(most, fabsf(a.lam[kvh * a.g + h]));
    const int power = ilogbf(most) + (most > 1.f);
    gs = ldexpf(gs, -power), boost = ldexpf(1.f, min(8, 14 - power));
  }

  const auto rk = buffer((const T*)a.k.data + s.b * a.k.batch_stride + ((a.stacked ? s.k0 : 0) + key_base) * a.k.row_stride +
                         (int64_t)kvh * 2 * a.k.head_stride);
  const auto rv = buffer((const T*)a.v.data + s.b * a.v.batch_stride + ((a.stacked ? s.k0 : 0) + key_base) * a.v.row_stride +
                         (int64_t)kvh * a.v.head_stride);
  const int ok = (int)((32 * kg + col) * a.k.row_stride * (int)sizeof(T)), hs = (int)(a.k.head_stride * sizeof(T));
  const int ov = (int)((32 * kg + col) * a.v.row_stride * (int)sizeof(T));
  auto k_frag = [&](int map, int i) GEOTR_INLINE {
    const int c = (2 * i + half) * kE<T>;
    return load_frag<T>(rk, in && c < a.d ? ok + map * hs + c * (int)sizeof(T) : kOutside);
  };
  auto v_frag = [&](int i) GEOTR_INLINE {
    const int c = (2 * i + half) * kE<T>;
    return load_frag<T>(rv, in && c < a.dv ? ov + c * (int)sizeof(T) : kOutside);
  };
  Frag k1[kHold ? QS : 1], k2[kHold ? QS : 1], vv[kHoldV ? VS : 1];
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < QS; ++i) k1[i] = k_frag(0, i), k2[i] = k_frag(1, i);
#pragma unroll
    for (int i = 0; i < QS; ++i) arrived(k1[i]), arrived(k2[i]);
  }
  if constexpr (kHoldV) {
#pragma unroll
    for (int i = 0; i < VS; ++i) vv[i] = v_frag(i);
#pragma unroll
    for (int i = 0; i < VS; ++i) arrived(vv[i]);
  }
  const unsigned vt = lds_at(smem) + NB * kBuf + kg * 32 * CO * 16;  // this wave's keys of V
  if constexpr (kInLds) {
    const i32x4 r = words((const T*)a.v.data + s.b * a.v.batch_stride + ((a.stacked ? s.k0 : 0) + key_base + 32 * kg) * a.v.row_stride +
                          (int64_t)kvh * a.v.head_stride);
    const unsigned there = (unsigned)__ballot(in);
    stage_at<T, 32, 1, DVB, 1>(vt, r, a.dv, 0, 0, lane, [&](int x) GEOTR_INLINE {
      return (there >> x) & 1 ? x * (int)(a.v.row_stride * sizeof(T)) : kOutside;
    });
  }
  f32x16 ak1[DK ? ND : 1], ak2[DK ? ND : 1], av[DV ? NV : 1];
  if constexpr (DK) {
#pragma unroll
    for (int i = 0; i < ND; ++i) ak1[i] = zero16(), ak2[i] = zero16();
  }
  if constexpr (DV) {
#pragma unroll
    for (int i = 0; i < NV; ++i) av[i] = zero16();
  }

  const int off = s.m - s.n;
  const int rows = s.n << a.gsh;
  int first = 0;
  if (a.causal) first = (min(s.n, max(0, key_base - off)) << a.gsh) / 32 * 32;  // rows before see none of these keys
  // key j is seen by query i iff j <= i + off, by packed row r iff (j - off) << gsh <= r
  auto sees = [&](int j) GEOTR_INLINE { return a.causal ? max(0, min(j - off, s.n)) << a.gsh : 0; };  // below zero it would pass 32 bits
  const int from = sees(key), last = sees(key_base + TILE - 1);
  for (int h = 0; h < a.g; ++h) minus |= a.lam[kvh * a.g + h] < 0.f;

  const T* const qp = (const T*)a.q.data + s.b * a.q.batch_stride + (a.stacked ? s.q0 : 0) * a.q.row_stride + (int64_t)kvh * 2 * a.g * a.q.head_stride;
  const T* const op = (const T*)a.dout.data + s.b * a.dout.batch_stride + (a.stacked ? s.q0 : 0) * a.dout.row_stride +
                      (int64_t)kvh * a.g * a.dout.head_stride;
  const float* const sp = a.rows + row_stat_at(a, kvh, 0, s.q0, 0);
  const int qrs = (int)(a.q.row_stride * sizeof(T)), qhs = (int)(a.q.head_stride * sizeof(T)), ors = (int)(a.dout.row_stride * sizeof(T)),
            ohs = (int)(a.dout.head_stride * sizeof(T));
  const int group = 1 << a.gsh, q16 = group <= 16 ? (16 >> a.gsh) * qrs : 32 * qhs, o16 = group <= 16 ? (16 >> a.gsh) * ors : 16 * ohs;
  const Stage<T, 32, 2, DB, NW> qst(a.d, qhs, wave, lane, [&](int x) { return (x >> a.gsh) * qrs + (x & (group - 1)) * 2 * qhs; });
  const Stage<T, 32, 1, DVB, NW> ost(a.dv, 0, wave, lane, [&](int x) { return (x >> a.gsh) * ors + (x & (group - 1)) * ohs; });
  // numbers of the rows: a wave load takes a pair of the kinds, lane = kind and row
  const int so = (((col >> a.gsh) * a.g + (col & (group - 1))) * 2 + half) * 4;
  auto fill32 = [&](unsigned tile, int r0) GEOTR_INLINE {
    const int i0 = r0 >> a.gsh, h0 = r0 & (group - 1);
    const i32x4 rq = words(qp + i0 * a.q.row_stride + 2 * h0 * a.q.head_stride), ro = words(op + i0 * a.dout.row_stride + h0 * a.dout.head_stride);
    auto there = [&](int x) GEOTR_INLINE { return r0 + x < rows && ((r0 + x) & (group - 1)) < a.g; };
    if (r0 + 32 <= rows && a.g == group) {
      qst.load_all(tile, rq, q16, wave);
      ost.load_all(tile + 32 * CQ * 16, ro, o16, wave);
    } else {
      qst.load_some(tile, rq, q16, wave, there);
      ost.load_some(tile + 32 * CQ * 16, ro, o16, wave, there);
    }
    // rows that do not exist: zeros, and their products are zero because q and dout are
    for (int x = wave; x < 4; x += NW) {
      const i32x4 rs = words(sp + (((int64_t)x * a.nq + i0) * a.g + h0) * 2);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                   :
                   : "s"(__builtin_amdgcn_readfirstlane(tile + kRowBytes + x * 256)), "v"(there(col) ? so : kOutside), "s"(rs)
                   : "m0", "memory");
    }
  };
  auto fill = [&](unsigned tile, int r0) GEOTR_INLINE {
    fill32(tile, r0);
    if (QG == 2 && r0 + 32 < rows) fill32(tile + kTile, r0 + 32);
  };
  const Rows<T, CQ> qrow(col, half);
  const Rows<T, CO> orow(col, half);
  const Cols<T, CQ> qcol(lane);
  const Cols<T, CO> ocol(lane);
  auto consume = [&](unsigned qt, int r0) GEOTR_INLINE {
    if constexpr (QG == 2) {
      qt += qg * kTile, r0 += 32 * qg;
      if (r0 >= rows) return;
    }
    const unsigned ot = qt + 32 * CQ * 16, st = qt + kRowBytes + 16 * half;
    auto stat = [&](int which, int j) GEOTR_INLINE { return lds_load<f32x4>(st + 128 * which + 32 * j); };
    f32x16 s1 = zero16(), s2 = zero16(), dp = zero16();  // scores, then P1 and |lam| P2
#pragma unroll
    for (int i = 0; i < QS; ++i) {
      Ops<T>::mma(s1, qrow.get(qt, 0, i), kHold ? k1[i % (kHold ? QS : 1)] : k_frag(0, i));
      Ops<T>::mma(s2, qrow.get(qt, 0, CQ / 4 + i), kHold ? k2[i % (kHold ? QS : 1)] : k_frag(1, i));
    }
    if constexpr (kWavesKV<T, DB, DVB, PART> == 1) {
      if constexpr (DK) {
#pragma unroll
        for (int i = 0; i < ND; ++i) held(ak1[i]), held(ak2[i]);
      }
      if constexpr (DV) {
#pragma unroll
        for (int i = 0; i < NV; ++i) held(av[i]);
      }
    }
    if constexpr (PART == kKeysOnly) GEOTR_FENCE;
    auto weights = [&](auto from, auto far) GEOTR_INLINE {  // beside the products of dP
      if constexpr (DK) {
#pragma unroll
        for (int i = 0; i < VS; ++i) {
          if (PART == kKeysOnly && i % 2 == 0) GEOTR_FENCE;
          Ops<T>::mma(dp, orow.get(ot, 0, i), kHoldV ? vv[i % (kHoldV ? VS : 1)] : kInLds ? orow.get(vt, 0, i) : v_frag(i));
        }
        if constexpr (PART == kKeysOnly) GEOTR_FENCE;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 e1 = stat(0, j), e2 = stat(1, j);
        f32x4 r1 = {}, r2 = {};
        if constexpr (decltype(far)::value) r1 = stat(5, j), r2 = stat(6, j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * j + e;
          s1[i] = __builtin_amdgcn_exp2f(from(s1[i], e1[e], r1[e])), s2[i] = __builtin_amdgcn_exp2f(from(s2[i], e2[e], r2[e]));
        }
      }
    };
    const float own = fabsf(lds_load<float>(qt + kRowBytes + 128 * half + 4 * col));  // lane: row and map
    if (__builtin_expect(__any(own > kHuge && own < INFINITY), 0)) weights([&](float x, float e, float r) { return (x * a.scale_log2 - e) - r; }, std::true_type{});
    else weights([&](float x, float e, float) { return fmaf(x, a.scale_log2, -e); }, std::false_type{});
    if (a.causal && r0 < last) {  // rows that do not see some key of the block
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (r0 + 8 * (i / 4) + 4 * half + i % 4 < from) s1[i] = 0.f, s2[i] = 0.f;
    }
    if (minus) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4 sg = stat(4, j);
#pragma unroll
        for (int e = 0; e < 4; ++e) s2[4 * j + e] *= sg[e];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f32x4 d1 = {}, d2 = {};
      if constexpr (DK) d1 = stat(2, j), d2 = stat(3, j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 4 * j + e;
        const float p1 = s1[i], p2 = s2[i], g = dp[i];
        if constexpr (DK) s1[i] = p1 * (g - d1[e]), s2[i] = p2 * (d2[e] - g);
        if constexpr (DV) dp[i] = p1 - p2;
        if constexpr (Narrow<T>::value) s1[i] *= gs, s2[i] *= gs, dp[i] *= boost;
      }
    }
#pragma unroll
    for (int p = 0; p < kPSteps<T>; ++p) {
      if constexpr (DV) {
        const Frag f = pack<T>(dp, p);
#pragma unroll
        for (int i = 0; i < NV; ++i) Ops<T>::mma(av[i], ocol.get(ot, 0, p, i), f);
      }
      if constexpr (DK) {
        const Frag f1 = pack<T>(s1, p), f2 = pack<T>(s2, p);
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          Ops<T>::mma(ak1[i], qcol.get(qt, 0, p, i), f1);
          Ops<T>::mma(ak2[i], qcol.get(qt, 0, p, ND + i), f2);
        }
      }
    }
  };
  const unsigned base = lds_at(smem);
  if constexpr (NB == 2) {
    if (first < rows) fill(base, first);
    int which = 0;
    for (int r0 = first; r0 < rows; r0 += BN) {
      tile_ready();
      __syncthreads();
      if (r0 + BN < rows) fill(base + (kBuf - which), r0 + BN);
      consume(base + which, r0);
      which = kBuf - which;
    }
  } else {
    for (int r0 = first; r0 < rows; r0 += BN) {
      __syncthreads();
      fill(base, r0);
      tile_ready();
      __syncthreads();
      consume(base, r0);
    }
  }
  if constexpr (QG == 2) {  // the other query group's sums
    float* box = (float*)smem + kg * (kJoin / 4 / KG) + lane;
    auto meet = [&](f32x16& x) GEOTR_INLINE {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (qg == 1) box[j * 64] = x[j];
        else x[j] += box[j * 64];
      }
      box += 16 * 64;
    };
    auto all = [&]() GEOTR_INLINE {
      if constexpr (DK) {
#pragma unroll
        for (int i = 0; i < ND; ++i) meet(ak1[i]), meet(ak2[i]);
      }
      if constexpr (DV) {
#pragma unroll
        for (int i = 0; i < NV; ++i) meet(av[i]);
      }
    };
    __syncthreads();
    if (qg == 1) all();
    __syncthreads();
    if (qg == 1) return;
    all();
  }
  if (key >= keys_here) return;
  const float fk = a.scale / gs, fv = 1.f / boost;
  const int64_t at = s.k0 + key;
  T* const pk = dk + (at * a.hk + kvh) * 2 * a.d;
  T* const pv = dv + (at * a.hk + kvh) * a.dv;
  // a key that is masked or does not exist: zero, whatever its lane accumulated
  auto out4 = [&](T* p, const f32x16& x, int j, float f) GEOTR_INLINE {
    if (in) store4<T>(p, x[4 * j] * f, x[4 * j + 1] * f, x[4 * j + 2] * f, x[4 * j + 3] * f);
    else store4<T>(p, 0.f, 0.f, 0.f, 0.f);
  };
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (DK) {
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        const int c = 32 * i + 8 * j + 4 * half;
        if (c < a.d) out4(pk + c, ak1[i], j, fk), out4(pk + a.d + c, ak2[i], j, fk);
      }
    }
    if constexpr (DV) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 32 * i + 8 * j + 4 * half;
        if (c < a.dv) out4(pv + c, av[i], j, fv);
      }
    }
  }
}
template <typename T, int DB, int DVB, int NW, int PART, int QG>
__global__ __launch_bounds__(NW * 64, (kWavesKV<T, DB, DVB, PART>)) void dkv_kernel(Args a) {
  __shared__ __attribute__((aligned(1024))) char smem[kSmemKV<T, DB, DVB, NW, PART, QG>()];
  dkv_block<T, DB, DVB, NW, PART, QG>(a, smem, a.tile0 + blockIdx.y, a.tiles);
}
// Both in one launch where both take two waves to a SIMD unit, the first key_blocks of a head for the keys: the last blocks of one fill what the
// other's leave empty (32 clouds of 295 in 32 bits, 32, 64: 215 -> 169 us, 25 registers spilled in 32 bits; 2 x 2 048 rows, 4 heads, bf16: 81 -> 60).
template <typename T, int DB, int DVB, int NW, int QG>
__global__ __launch_bounds__(NW * 64, 2) void backward_kernel(Args a, int key_blocks) {
  constexpr int kQ = kSmemQ<T, DB, DVB, NW>(), kKV = kSmemKV<T, DB, DVB, NW, kBoth, QG>();
  __shared__ __attribute__((aligned(1024))) char smem[kQ > kKV ? kQ : kKV];
  const int y = a.tile0 + blockIdx.y;
  if (y < key_blocks) dkv_block<T, DB, DVB, NW, kBoth, QG>(a, smem, y, key_blocks);
  else dq_block<T, DB, DVB, NW>(a, smem, y - key_blocks, a.tiles - key_blocks);
}

// ---- launches -------------------------------------------------------------------------------------------------------------------------------
enum Which { kForward, kForwardKeys, kBackward };

// stack mode: every sequence may end inside a tile, and one block more takes the rows behind the last
inline int64_t tiles_of(const Args& a, bool keys, int tile) {
  const int64_t rows = keys ? (a.stacked ? a.nk : a.m) : (a.stacked ? a.nq : a.n) << a.gsh;
  return (rows + tile - 1) / tile + (a.stacked ? a.batch + 1 : 0);
}

template <typename T, int DB, int DVB>
int launch_dims(const Args& a, Which which, hipStream_t s) {
  constexpr int G = 2, NWB = 4, kWide = 64 * (2 * DB + DVB) * (int)sizeof(T);  // bytes of 64 keys
  // few rows: narrow heads stream a tile per wave; wide ones share tiles of 64 keys, where two buffers of them fit
  constexpr bool kNarrow = (int)sizeof(T) * DB < 256, kFew = !kNarrow && 2 * kWide <= 160 * 1024;
  const bool keys = which == kForwardKeys && (kNarrow || kFew);
  // A grid holds 65 535 tiles of a head and 2^32 threads over the heads and sequences: what is more takes further launches
  const int seqs = a.stacked ? 1 : a.batch, most_seqs = std::max(1, (1 << 22) / a.hk), most_tiles = 65535;
  auto go = [&](auto kernel, int64_t blocks, int threads, auto... more) -> int {
    for (int seq0 = 0; seq0 < seqs; seq0 += most_seqs)
      for (int64_t tile0 = 0; tile0 < blocks; tile0 += most_tiles) {
        Args part = a;
        part.tiles = (int)blocks, part.tile0 = (int)tile0, part.seq0 = seq0;
        const dim3 grid((unsigned)(std::min(most_seqs, seqs - seq0) * a.hk), (unsigned)std::min<int64_t>(most_tiles, blocks - tile0),
                        which == kBackward ? 1u : (unsigned)a.splits);
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, s, part, more...);
        GEOTR_CHECK_LAUNCH("differential attention");
      }
    return GEOTR_OK;
  };
  auto run = [&](auto kernel, int tile, int threads) -> int { return go(kernel, tiles_of(a, false, tile), threads); };
  if (which == kBackward) {
    // Two query groups halve a block's keys and its steps, but load every query row twice as often.  They win while all their blocks run at
    // once (2 x 2 048 rows and 4 heads, 128 against 64 blocks: 64/64 139 against 246 us) and lose with more
    // (2 x 4 096 causal rows and 8 heads: 404 against 316).  32-bit products take 16 times as long as the loads: always (32 clouds of 295
    // rows: 119 against 128 us; 4 x 2 048 rows, 4 heads: 368 against 481).
    const int64_t tiles = a.stacked ? (a.nk / (32 * NWB) + a.batch / 2) : (int64_t)a.batch * ((a.m + 32 * NWB - 1) / (32 * NWB));
    const bool small = tiles * a.hk <= 128 * kWavesKV<T, DB, DVB, kBoth>;
    const int64_t rows = tiles_of(a, false, 32 * NWB / kKeyGroups<T, DB, DVB>);
    auto keys_of = [&](auto part, auto use) -> int {  // use(query groups, blocks)
      constexpr int PART = decltype(part)::value, QG = kRowGroups<T, DB, DVB, PART>;
      if constexpr (QG == 2)
        if (sizeof(T) == 4 || small) return use(std::integral_constant<int, 2>{}, tiles_of(a, true, 16 * NWB));
      if constexpr (QG == 1 || sizeof(T) == 2) return use(std::integral_constant<int, 1>{}, tiles_of(a, true, 32 * NWB));
      return GEOTR_OK;
    };
    if constexpr (kWaves<T, DB, DVB> == 2 && kWavesKV<T, DB, DVB, kBoth> == 2) {
      return keys_of(std::integral_constant<int, kBoth>{}, [&](auto qg, int64_t blocks) {
        return go(backward_kernel<T, DB, DVB, NWB, decltype(qg)::value>, blocks + rows, 64 * NWB, (int)blocks);
      });
    } else {
      if (a.nq)
        if (const int r = go(dq_kernel<T, DB, DVB, NWB>, rows, 64 * NWB)) return r;
      if (a.nk == 0) return GEOTR_OK;
      auto keys = [&](auto part) {
        return keys_of(part, [&](auto qg, int64_t blocks) {
          return go(dkv_kernel<T, DB, DVB, NWB, decltype(part)::value, decltype(qg)::value>, blocks, 64 * NWB);
        });
      };
      if constexpr (kSplitKV<T, DVB>) {
        if (const int r = keys(std::integral_constant<int, kKeysOnly>{})) return r;
        return keys(std::integral_constant<int, kValuesOnly>{});
      } else {
        return keys(std::integral_constant<int, kBoth>{});
      }
    }
  }
  if constexpr (sizeof(T) == 4) {
    const int64_t rows = (a.stacked ? (a.nq + a.batch - 1) / std::max(a.batch, 1) : a.n) << a.gsh;
    if (which == kForwardKeys && rows <= 4)
      return rows == 1 ? run(fwd_rows_kernel<DB, DVB, 1>, 1, 512) : run(fwd_rows_kernel<DB, DVB, 4>, 4, 512);
  }
  if (keys) {
    if constexpr (kNarrow) return run(fwd_keys_kernel<T, DB, DVB, 4>, 32, 256);
    if constexpr (kFew) return run(fwd_kernel<T, DB, DVB, G, true, false>, 32, 128 * G);
  }
  if constexpr (sizeof(T) == 2)
    if (a.maps) return run(fwd_kernel<T, DB, DVB, G, false, true>, 32 * G, 128 * G);
  return run(fwd_kernel<T, DB, DVB, G, false, false>, 32 * G, 128 * G);
}

// head dimensions: the next of 32, 64, 128 for q and k; one or two times that for v
template <typename T>
int launch_type(const Args& a, Which which, hipStream_t s) {
  if (a.d <= 32 && a.dv <= 32) return launch_dims<T, 32, 32>(a, which, s);
  if (a.d <= 32 && a.dv <= 64) return launch_dims<T, 32, 64>(a, which, s);
  if (a.d <= 64 && a.dv <= 64) return launch_dims<T, 64, 64>(a, which, s);
  if (a.d <= 64 && a.dv <= 128) return launch_dims<T, 64, 128>(a, which, s);
  if (a.d <= 128 && a.dv <= 128) return launch_dims<T, 128, 128>(a, which, s);
  return launch_dims<T, 128, 256>(a, which, s);
}

int launch_f32(const Args& a, Which which, hipStream_t s);
int launch_bf16(const Args& a, Which which, hipStream_t s);
int launch_f16(const Args& a, Which which, hipStream_t s);

}  // namespace dattn
}  // namespace geotr
