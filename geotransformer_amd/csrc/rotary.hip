// rotary.hip -- rotary positions: pairs of channels of query and key heads turned by an angle proportional to the token's position
// (geotr_rotary, include/geotr.h), for integer positions of sequences and for coordinates of points with one frequency set per axis.
//
//   y_a = g (x_a cos t - x_b sin t),  y_b = g (x_b cos t + x_a sin t),   t = 2 pi p[axis_i] turns_i,
//   (a, b) = (i, i + R/2) (half layout) or (2i, 2i + 1) (interleaved); channels R .. D pass through.
// The gradient is the transposed rotation with the same g: the same kernel with -t (`inverse`).
//
// Bound: HBM, every element read once and written once (the trigonometry is one sine and cosine per (token, pair), shared by all heads
// of the query and of the key, which one launch covers).  A thread owns one 16-byte chunk position of a token (two chunks in the half
// layout), computes the E (half) or E / 2 (interleaved) angles once and walks the heads with four of them in flight.  32 768 tokens of 40
// heads of 128, bf16: 157 us, 4.3 of the 5.1 TB/s of a large copy; 9 583 points of 16 heads of 32, 32 bits: 8.8 us (4.5 TB/s); one token: 6 us,
// the launch.
#include <algorithm>

#include "common.h"

namespace geotr {
namespace {

template <typename T, int E>
struct alignas(sizeof(T) * E) Chunk {
  T v[E];
};

struct RotaryArgs {
  geotr_heads q, qo, k, ko;
  int64_t rows, pos_batch, pos_row, pos_axis;
  const void* positions;
  const double* turns;
  const int32_t* axis;
  float gain, sign;
  int pos_type, dim, rot, tiles, tokens, heads, heads_per_block, copy_rest;
  unsigned block0;  // a launch's first block: a grid holds 2^32 threads along an axis
};

__device__ __forceinline__ double position_at(const void* p, int type, int64_t i) {
  switch (type) {
    case GEOTR_POS_I32: return (double)((const int32_t*)p)[i];
    case GEOTR_POS_I64: return (double)((const int64_t*)p)[i];
    case GEOTR_POS_F32: return (double)((const float*)p)[i];
    default: return ((const double*)p)[i];
  }
}

// cos and sin of 2 pi t.  The angle is kept in turns and 64 bits until it is within 1/8 turn of a quarter (a position of 10^6 in 32-bit
// radians is off by 0.06): the rest, |x| <= pi/4, is two Taylor polynomials whose remainders are below 2^-28 of the result.
__device__ __forceinline__ void sincos_turns(double t, float& c, float& s) {
  const double q = rint(4.0 * t);
  const float x = (float)(6.283185307179586 * fma(-0.25, q, t));
  const int quadrant = (int)(q - 4.0 * floor(0.25 * q));
  const float x2 = x * x;
  float ps = fmaf(x2, 2.7557319e-6f, -1.9841270e-4f);
  ps = fmaf(x2, ps, 8.3333333e-3f);
  ps = fmaf(x2, ps, -1.6666667e-1f);
  ps = fmaf(x * x2, ps, x);
  float pc = fmaf(x2, -2.7557319e-7f, 2.4801587e-5f);
  pc = fmaf(x2, pc, -1.3888889e-3f);
  pc = fmaf(x2, pc, 4.1666667e-2f);
  pc = fmaf(x2, pc, -0.5f);
  pc = fmaf(x2, pc, 1.0f);
  const bool odd = quadrant & 1;
  const float a = odd ? ps : pc, b = odd ? pc : ps;
  c = (quadrant == 1 || quadrant == 2) ? -a : a;
  s = (quadrant & 2) ? -b : b;
}

// E elements per chunk; IL: pairs inside a chunk, else between two chunks R/2 apart.  E = 1: scalar accesses, pairs (2i, 2i+1) or
// (i, i + R/2): odd strides and layouts whose halves are not a multiple of any chunk.
template <typename T, int E, bool IL>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  constexpr bool kTwo = !IL || E == 1;            // two chunks per head
  constexpr int NP = kTwo ? E : E / 2;            // pairs per thread
  const int half = a.rot / 2;
  const int n_rot = half / NP, n_all = n_rot + (a.copy_rest ? (a.dim - a.rot) / E : 0);
  const unsigned block = a.block0 + blockIdx.x, b = block / (unsigned)a.tiles;
  const int64_t row0 = (int64_t)(block - b * (unsigned)a.tiles) * a.tokens;
  const int h0 = blockIdx.y * a.heads_per_block, h1 = min(h0 + a.heads_per_block, a.heads);
  const int hq = (int)a.q.heads;
  for (int u = threadIdx.x; u < a.tokens * n_all; u += 256) {
    const int t = u / n_all, c = u - t * n_all;
    const int64_t row = row0 + t;
    if (row >= a.rows) continue;
    const T* qi = (const T*)a.q.data + b * a.q.batch_stride + row * a.q.row_stride;
    const T* ki = (const T*)a.k.data + b * a.k.batch_stride + row * a.k.row_stride;
    T* qo = (T*)a.qo.data + b * a.qo.batch_stride + row * a.qo.row_stride;
    T* ko = (T*)a.ko.data + b * a.ko.batch_stride + row * a.ko.row_stride;
    const bool turn = c < n_rot;
    int e0, e1 = 0;
    float cs[NP], sn[NP];
    if (turn) {
      e0 = kTwo ? (IL ? 2 * c : c * E) : c * E;
      e1 = kTwo ? (IL ? 2 * c + 1 : e0 + half) : 0;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int i = c * NP + p;
        const double pos = position_at(a.positions, a.pos_type, b * a.pos_batch + row * a.pos_row + a.axis[i] * a.pos_axis);
        sincos_turns(pos * a.turns[i], cs[p], sn[p]);
        cs[p] *= a.gain;
        sn[p] *= a.gain * a.sign;
      }
    } else {
      e0 = a.rot + (c - n_rot) * E;
    }
    constexpr int U = 4;  // heads in flight
    for (int h = h0; h < h1; h += U) {
      Chunk<T, E> x[U], y[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int hh = h + j;
        if (hh < h1) {
          const T* src = hh < hq ? qi + hh * a.q.head_stride : ki + (hh - hq) * a.k.head_stride;
          x[j] = *(const Chunk<T, E>*)(src + e0);
          if (kTwo && turn) y[j] = *(const Chunk<T, E>*)(src + e1);
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int hh = h + j;
        if (hh < h1) {
          T* dst = hh < hq ? qo + hh * a.qo.head_stride : ko + (hh - hq) * a.ko.head_stride;
          if (turn) {
#pragma unroll
            for (int p = 0; p < NP; ++p) {  // products and sums in 32 bits, one rounding to T at the end
              T& xa = kTwo ? x[j].v[p] : x[j].v[2 * p];
              T& xb = kTwo ? y[j].v[p] : x[j].v[2 * p + 1 < E ? 2 * p + 1 : 0];
              const float fa = (float)xa, fb = (float)xb;
              xa = (T)fmaf(fa, cs[p], -(fb * sn[p]));
              xb = (T)fmaf(fb, cs[p], fa * sn[p]);
            }
            if (kTwo) *(Chunk<T, E>*)(dst + e1) = y[j];
          }
          *(Chunk<T, E>*)(dst + e0) = x[j];
        }
      }
    }
  }
}

template <typename T, int E>
void rotary_launch(const RotaryArgs& a, bool interleaved, dim3 grid, hipStream_t s) {
  if (interleaved) hipLaunchKernelGGL((rotary_kernel<T, E, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((rotary_kernel<T, E, false>), grid, dim3(256), 0, s, a);
}

template <typename T>
void rotary_dispatch(const RotaryArgs& a, int e, bool interleaved, dim3 grid, hipStream_t s) {
  switch (e) {
    case 8: if constexpr (sizeof(T) == 2) rotary_launch<T, 8>(a, interleaved, grid, s); break;
    case 4: rotary_launch<T, 4>(a, interleaved, grid, s); break;
    case 2: rotary_launch<T, 2>(a, interleaved, grid, s); break;
    default: rotary_launch<T, 1>(a, interleaved, grid, s);
  }
}

}  // namespace
}  // namespace geotr

using namespace geotr;

extern "C" int geotr_rotary(const geotr_heads* q, const geotr_heads* q_out, const geotr_heads* k, const geotr_heads* k_out, int dtype,
                            int64_t batch, int64_t rows, int64_t dim, int64_t rotary_dim, int interleaved, const void* positions,
                            int position_type, int64_t pos_batch_stride, int64_t pos_row_stride, int64_t pos_axis_stride,
                            const double* turns, const int32_t* axis, float gain, int inverse, void* stream) {
  GEOTR_CHECK_ARG(q && q_out, "geotr_rotary: null descriptor");
  GEOTR_CHECK_ARG(!k == !k_out, "geotr_rotary: k and k_out go together");
  GEOTR_CHECK_ARG(dtype >= GEOTR_F32 && dtype <= GEOTR_F16, "geotr_rotary: unknown dtype %d", dtype);
  GEOTR_CHECK_ARG(position_type >= GEOTR_POS_I32 && position_type <= GEOTR_POS_F64, "geotr_rotary: unknown position type %d", position_type);
  GEOTR_CHECK_ARG(batch >= 0 && rows >= 0 && dim >= 2 && dim <= 1024, "geotr_rotary: batch %lld, rows %lld, head dimension %lld (2 .. 1024)",
                  (long long)batch, (long long)rows, (long long)dim);
  GEOTR_CHECK_ARG(rotary_dim >= 2 && rotary_dim <= dim && rotary_dim % 2 == 0, "geotr_rotary: rotary dimension %lld of a head of %lld",
                  (long long)rotary_dim, (long long)dim);
  const geotr_heads none = {nullptr, 0, 0, 0, 0};
  RotaryArgs a;
  a.q = *q, a.qo = *q_out, a.k = k ? *k : none, a.ko = k_out ? *k_out : none;
  GEOTR_CHECK_ARG(a.q.heads >= 0 && a.q.heads <= 65536 && a.k.heads >= 0 && a.k.heads <= 65536 && a.qo.heads == a.q.heads && a.ko.heads == a.k.heads,
                  "geotr_rotary: %lld query and %lld key heads in, %lld and %lld out", (long long)a.q.heads, (long long)a.k.heads,
                  (long long)a.qo.heads, (long long)a.ko.heads);
  if (batch == 0 || rows == 0 || a.q.heads + a.k.heads == 0) return GEOTR_OK;
  GEOTR_CHECK_ARG((a.q.heads == 0 || (a.q.data && a.qo.data)) && (a.k.heads == 0 || (a.k.data && a.ko.data)) && positions && turns && axis,
                  "geotr_rotary: null pointer");
  // the widest chunk that every address is a multiple of
  const int size = dtype == GEOTR_F32 ? 4 : 2;
  int e = 16 / size;
  auto fits = [&](int w) {
    const int64_t span = interleaved ? rotary_dim : rotary_dim / 2;
    if (span % w || dim % w || rotary_dim % w) return false;
    const geotr_heads* all[4] = {&a.q, &a.qo, &a.k, &a.ko};
    for (const geotr_heads* v : all)
      if (v->heads && (((uintptr_t)v->data) % (w * size) || v->batch_stride % w || v->row_stride % w || v->head_stride % w)) return false;
    return true;
  };
  while (e > 1 && !fits(e)) e /= 2;
  const bool in_place = (a.q.heads == 0 || a.q.data == a.qo.data) && (a.k.heads == 0 || a.k.data == a.ko.data);
  a.rows = rows, a.pos_batch = pos_batch_stride, a.pos_row = pos_row_stride, a.pos_axis = pos_axis_stride;
  a.positions = positions, a.turns = turns, a.axis = axis, a.gain = gain, a.sign = inverse ? -1.f : 1.f;
  a.pos_type = position_type, a.dim = (int)dim, a.rot = (int)rotary_dim, a.copy_rest = in_place ? 0 : 1;
  const int pairs = interleaved && e > 1 ? e / 2 : e;
  const int n_all = (int)(rotary_dim / 2) / pairs + (a.copy_rest ? (int)(dim - rotary_dim) / e : 0);
  a.tokens = std::max(1, 256 / n_all);
  const int64_t tiles = rows / a.tokens + (rows % a.tokens != 0);
  GEOTR_CHECK_ARG(tiles <= 0x7fffffff / batch, "geotr_rotary: %lld x %lld tokens in one call", (long long)batch, (long long)rows);
  const int64_t blocks = tiles * batch;
  a.tiles = (int)tiles, a.heads = (int)(a.q.heads + a.k.heads);
  // all heads in one thread once the tokens alone give 2 048 blocks (the angles are computed once); fewer tokens: heads over more blocks
  const int64_t want = std::min<int64_t>(a.heads, (2048 + blocks - 1) / blocks);
  a.heads_per_block = (int)((a.heads + want - 1) / want);
  hipStream_t s = (hipStream_t)stream;
  constexpr int64_t kMost = 1 << 23;
  for (int64_t first = 0; first < blocks; first += kMost) {
    a.block0 = (unsigned)first;
    const dim3 grid((unsigned)std::min(kMost, blocks - first), (unsigned)((a.heads + a.heads_per_block - 1) / a.heads_per_block));
    if (dtype == GEOTR_F32) rotary_dispatch<float>(a, e, interleaved, grid, s);
    else if (dtype == GEOTR_BF16) rotary_dispatch<__bf16>(a, e, interleaved, grid, s);
    else rotary_dispatch<_Float16>(a, e, interleaved, grid, s);
    GEOTR_CHECK_LAUNCH("geotr_rotary");
  }
  return GEOTR_OK;
}
