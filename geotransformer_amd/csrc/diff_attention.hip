// diff_attention.hip -- entry points of the differential attention (include/geotr.h) and its small kernels: joining the partials of keys
// dealt over several blocks, del = dout . output of each map, and the gradient of lam.  The matrix work is in diff_attention.h.
#include <algorithm>

#include "diff_attention.h"

namespace geotr {
namespace dattn {
namespace {

constexpr int kMostSplits = 64;  // the join holds one split per lane

// Every wave holds the splits' maxima and sums in its lanes and four channels of both maps in a lane.  W waves to a (row, head) take the
// splits in turn and meet in LDS in a fixed order: four for many splits (single tokens, where latency counts: one wave took 82 us for 16
// rows of 64 splits, four 6), one for few (many rows: 12 us against 28 at 16 384 rows of two splits).
template <typename T, int W>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
  __shared__ f32x4 box[W][2][64];
  const int lane = threadIdx.x & 63, wave = W == 1 ? 0 : threadIdx.x >> 6, heads = a.hk * a.g;
  const int64_t e = W == 1 ? blockIdx.x * 4ll + (threadIdx.x >> 6) : blockIdx.x, row = e / heads;
  if (W == 1 && e >= a.nq * heads) return;
  const int head = (int)(e - row * heads), w = a.dv + 4, c = 4 * lane;
  const int64_t step = a.nq * heads * 2 * (int64_t)w;
  const float* p = a.part + e * 2 * w;
  float m[2], l[2], f[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    m[x] = lane < a.splits ? p[lane * step + x * w] : -INFINITY;
    l[x] = lane < a.splits ? p[lane * step + x * w + 1] : 0.f;
    float top = m[x];
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    f[x] = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[x] - top);
    float sum = l[x] * f[x];
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    m[x] = top, l[x] = sum;
  }
  f32x4 y = {}, z = {};
#pragma unroll 4
  for (int s = wave; s < a.splits; s += W) {
    const float f1 = __shfl(f[0], s, 64), f2 = __shfl(f[1], s, 64);
    if (c < a.dv) {
      const f32x4 u = *(const f32x4*)(p + s * step + 4 + c), v = *(const f32x4*)(p + s * step + w + 4 + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // a split without keys may have written nothing
        if (f1 != 0.f) y[i] = fmaf(u[i], f1, y[i]);
        if (f2 != 0.f) z[i] = fmaf(v[i], f2, z[i]);
      }
    }
  }
  if constexpr (W > 1) {
    box[wave][0][lane] = y, box[wave][1][lane] = z;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int x = 1; x < W; ++x) {
      const f32x4 u = box[x][0][lane], v = box[x][1][lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += u[i], z[i] += v[i];
    }
  }
  const bool some = l[0] != 0.f;
  const float lam = a.lam[head];
  if (c < a.dv) {
    float o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[i] = some ? y[i] / l[0] : 0.f, z[i] = some ? z[i] / l[1] : 0.f;
      o[i] = fmaf(-lam, z[i], y[i]);
    }
    store4<T>((T*)a.out + e * a.dv + c, o[0], o[1], o[2], o[3]);
    if (a.maps) {
      store4<float>(a.maps + 2 * e * a.dv + c, y[0], y[1], y[2], y[3]);
      store4<float>(a.maps + (2 * e + 1) * a.dv + c, z[0], z[1], z[2], z[3]);
    }
  }
  if (a.lse && lane < 2) {
    const int kvh = head / a.g;
    store_sums(a, stat_at(a, kvh, lane, row, head - kvh * a.g), lane ? m[1] : m[0], lane ? l[1] : l[0], some);
  }
}

// What the backward pass reads of a row: the sums, del_a = dout . O_a in 32 bits (16 lanes per (row, head)), |lam| folded into the second
// sum.  fp16: the largest |dout| of the rows that exist (an order-free maximum).  Bound: HBM.  The blocks take the rows in turn: a grid holds
// 2^32 threads, 16 of them to a (row, head).
template <typename T>
__global__ __launch_bounds__(256) void del_kernel(Args a, float* amax) {
  using Frag = typename Ops<T>::Frag;
  const int lane = threadIdx.x & 63, heads = a.hk * a.g, c0 = lane & 15;
  const int64_t all = a.nq * heads;
  float most = 0.f;
  int64_t exist = a.nq;  // stack mode: rows behind the last sequence say nothing
  if constexpr (Narrow<T>::value) {
    if (a.stacked) {
      exist = 0;
      for (int b = lane; b < a.batch; b += 64) exist += clamp_len(a.q_len[b], a.nq);
#pragma unroll
      for (int o = 32; o; o >>= 1) exist += __shfl_xor(exist, o, 64);
    }
  }
  for (int64_t e0 = (int64_t)blockIdx.x * 16; e0 < all; e0 += (int64_t)gridDim.x * 16) {
    const int64_t e = e0 + 4 * (threadIdx.x >> 6) + (lane >> 4);
    const bool in = e < all;
    float x = 0.f, z = 0.f, top = 0.f;
    const int64_t row = in ? e / heads : 0;
    const int head = in ? (int)(e - row * heads) : 0;
    const int64_t b = a.stacked ? 0 : row / a.n, i = a.stacked ? row : row - b * a.n;
    if (in) {
      const T* g = (const T*)a.dout.data + b * a.dout.batch_stride + i * a.dout.row_stride + head * a.dout.head_stride;
      const float* y = a.maps + 2 * e * a.dv;
      for (int c = c0 * kE<T>; c < a.dv; c += 16 * kE<T>) {
        const Frag fg = *(const Frag*)(g + c);
#pragma unroll
        for (int j = 0; j < kE<T>; j += 4) {
          const f32x4 y1 = *(const f32x4*)(y + c + j), y2 = *(const f32x4*)(y + a.dv + c + j);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = (float)fg[j + i];
            x = fmaf(v, y1[i], x), z = fmaf(v, y2[i], z);
            if constexpr (Narrow<T>::value) top = fmaxf(top, fabsf(v));
          }
        }
      }
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) x += __shfl_xor(x, o, 64), z += __shfl_xor(z, o, 64);
    if (in && c0 == 0) {
      const int kvh = head / a.g;
      const int64_t at = stat_at(a, kvh, 0, row, head - kvh * a.g);
      const int64_t to = row_stat_at(a, kvh, 0, row, head - kvh * a.g), step = a.nq * a.g;
      const float lam = a.lam[head], e2 = a.lse[at + step], r2 = a.lse[at + 3 * step], log = log2f(fabsf(lam));
      const bool far = fabsf(e2) > kHuge && e2 < INFINITY;
      float2* const p = (float2*)(a.rows + to);
      p[0] = float2{a.lse[at], lam == 0.f ? INFINITY : far ? e2 : e2 - log};
      p[step] = float2{x, z};
      p[2 * step] = float2{lam < 0.f ? -1.f : 1.f, a.lse[at + 2 * step]};
      p[3 * step] = float2{far && lam != 0.f ? r2 - log : 0.f, 0.f};
    }
    if constexpr (Narrow<T>::value) {  // gradients of rows that do not exist say nothing
      if (a.stacked ? row >= exist : in && a.q_len && i >= a.q_len[b]) top = 0.f;
      most = fmaxf(most, top);
    }
  }
  if constexpr (Narrow<T>::value) {
#pragma unroll
    for (int o = 32; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    if (lane == 0 && most > 0.f) atomicMax((int*)amax, __float_as_int(most));
  }
}

// fp16: the largest |v| of the keys that exist and are not masked
__global__ __launch_bounds__(256) void v_max_kernel(Args a, float* amax) {
  const int lane = threadIdx.x & 63, per = a.hk * (a.dv / 8);
  int64_t end = a.nk;
  if (a.stacked) {
    int64_t sum = 0;
    for (int b = lane; b < a.batch; b += 64) sum += clamp_len(a.k_len[b], a.nk);
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
    end = min(end, sum);
  }
  float top = 0.f;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < end * per; e += (int64_t)gridDim.x * 256) {
    const int64_t row = e / per, b = a.stacked ? 0 : row / a.m, i = a.stacked ? row : row - b * a.m;
    if ((a.masks && a.masks[row]) || (!a.stacked && a.k_len && i >= a.k_len[b])) continue;
    const int rest = (int)(e - row * per), head = rest / (a.dv / 8);
    const auto x = *(const typename Ops<_Float16>::Frag*)((const _Float16*)a.v.data + b * a.v.batch_stride + i * a.v.row_stride +
                                                          head * a.v.head_stride + 8 * (rest - head * (a.dv / 8)));
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf((float)x[j]));
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  if (lane == 0 && top > 0.f) atomicMax((int*)amax, __float_as_int(top));
}

// dlam_h = - sum over rows, in a fixed order: 1 024 partial sums in 64 bits, then a tree
__global__ __launch_bounds__(1024) void dlam_kernel(const float* drow, int64_t nq, int g, float* dlam) {
  __shared__ double box[1024];
  const int kvh = blockIdx.x / g, h = blockIdx.x - kvh * g;
  const float* p = drow + (int64_t)kvh * nq * g + h;
  double s = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < nq; i += 1024) s += (double)p[i * g];
  box[threadIdx.x] = s;
  for (int o = 512; o; o >>= 1) {
    __syncthreads();
    if (threadIdx.x < o) box[threadIdx.x] += box[threadIdx.x + o];
  }
  if (threadIdx.x == 0) dlam[blockIdx.x] = (float)-box[0];
}

int launch(int dtype, const Args& a, Which which, hipStream_t s) {
  return dtype == GEOTR_F32 ? launch_f32(a, which, s) : dtype == GEOTR_BF16 ? launch_bf16(a, which, s) : launch_f16(a, which, s);
}

// near: rows and heads that a tile reaches by 32-bit offsets from its first element, below the 1 GiB a buffer descriptor here covers; other
// heads and rows have 64-bit addresses of their own
int check_view(const geotr_heads& v, int64_t heads, int size, int64_t batch, int64_t rows, int64_t near_rows, int64_t near_heads, const char* what) {
  GEOTR_CHECK_ARG(v.heads == heads, "differential attention: %s has %lld heads, expected %lld", what, (long long)v.heads, (long long)heads);
  if (batch * rows == 0) return GEOTR_OK;
  GEOTR_CHECK_ARG(v.data, "differential attention: %s is a null pointer", what);
  const int e = 16 / size;
  GEOTR_CHECK_ARG((uintptr_t)v.data % 16 == 0 && v.batch_stride % e == 0 && v.row_stride % e == 0 && v.head_stride % e == 0,
                  "differential attention: %s is not a 16-byte aligned view", what);
  const int64_t most = 1ll << 40;  // no product below passes 64 bits
  GEOTR_CHECK_ARG(v.row_stride >= 0 && v.head_stride >= 0 && v.row_stride < most && v.head_stride < most &&
                      (near_rows * v.row_stride + near_heads * v.head_stride + 512) * size < kNumRecords,
                  "differential attention: strides of %s (rows %lld, heads %lld elements): %lld rows and %lld heads on have to lie within 1 GiB, "
                  "which a contiguous tensor's do", what, (long long)v.row_stride, (long long)v.head_stride, (long long)near_rows, (long long)near_heads);
  return GEOTR_OK;
}

int make_args(const geotr_diff_attn* op, Args& a) {
  GEOTR_CHECK_ARG(op, "differential attention: null descriptor");
  GEOTR_CHECK_ARG(op->dtype >= GEOTR_F32 && op->dtype <= GEOTR_F16, "differential attention: unknown dtype %d", op->dtype);
  GEOTR_CHECK_ARG(op->batch >= 0 && op->n >= 0 && op->m >= 0 && op->batch <= (1 << 20), "differential attention: batch %lld, rows %lld and %lld",
                  (long long)op->batch, (long long)op->n, (long long)op->m);
  GEOTR_CHECK_ARG(op->dim >= 8 && op->dim <= 128 && op->dim % 8 == 0 && op->v_dim >= 8 && op->v_dim <= 256 && op->v_dim % 8 == 0,
                  "differential attention: head dimensions %lld and %lld (multiples of 8 up to 128 and 256)", (long long)op->dim, (long long)op->v_dim);
  const int64_t hk = op->v.heads, h = op->q.heads / 2;
  GEOTR_CHECK_ARG(hk >= 1 && h >= hk && h % hk == 0 && op->q.heads % 2 == 0 && h / hk <= 64 && hk <= 65535,
                  "differential attention: %lld query, %lld key and %lld value heads", (long long)op->q.heads, (long long)op->k.heads, (long long)hk);
  GEOTR_CHECK_ARG(op->scale > 0.f && op->scale < 1e30f, "differential attention: scale %g", (double)op->scale);
  GEOTR_CHECK_ARG(op->lam, "differential attention: lam is a null pointer");
  GEOTR_CHECK_ARG(!op->stacked || op->batch == 0 || (op->q_lengths && op->k_lengths), "differential attention: stack mode needs both lengths");
  const int size = op->dtype == GEOTR_F32 ? 4 : 2;
  const int64_t g = h / hk;
  a.gsh = 0;
  while ((1 << a.gsh) < g) ++a.gsh;
  const int64_t most = 1ll << 40;  // the products stay below 2^63
  a.nq = std::min(op->n, most) * (op->stacked ? 1 : op->batch), a.nk = std::min(op->m, most) * (op->stacked ? 1 : op->batch);
  GEOTR_CHECK_ARG(op->n <= kMostRows && op->m <= kMostRows && (a.nq << a.gsh) <= kMostRows && a.nk <= kMostRows, "differential attention: %lld query rows (x %lld heads) and %lld keys in one call",
                  (long long)a.nq, (long long)g, (long long)a.nk);
  int rc;
  if ((rc = check_view(op->q, 2 * h, size, op->batch, op->n, 64, 2ll << a.gsh, "q")) || (rc = check_view(op->k, 2 * hk, size, op->batch, op->m, 128, 1, "k")) ||
      (rc = check_view(op->v, hk, size, op->batch, op->m, 128, 0, "v")))
    return rc;
  a.q = op->q, a.k = op->k, a.v = op->v, a.dout = geotr_heads{nullptr, 0, 0, 0, 0};
  a.out = a.gq = a.gk = a.gv = nullptr, a.maps = a.lse = a.part = a.drow = a.rows = nullptr, a.amax = nullptr;
  a.lam = op->lam, a.q_len = op->q_lengths, a.k_len = op->k_lengths, a.masks = op->key_masks;
  a.batch = (int)op->batch, a.stacked = op->stacked != 0, a.n = (int)op->n, a.m = (int)op->m;
  a.hk = (int)hk, a.g = (int)g, a.d = (int)op->dim, a.dv = (int)op->v_dim, a.causal = op->causal != 0, a.splits = 1, a.tiles = a.tile0 = a.seq0 = 0;
  a.scale = op->scale, a.scale_log2 = (float)((double)op->scale * 1.4426950408889634);
  return GEOTR_OK;
}

// Few rows to a sequence (32 packed rows or less) without a gradient: blocks of one 32-row tile whose waves stream keys of their own.  Keys are dealt over
// blocks until there are two for each compute unit, as long as every block keeps 256 keys.
bool keys_form(const Args& a) {
  const int64_t rows = a.stacked ? (a.nq + a.batch - 1) / std::max(a.batch, 1) : a.n;
  return rows << a.gsh <= 32;
}
int choose_splits(const Args& a) {
  const int64_t per = a.stacked ? a.nk / std::max(a.batch, 1) : a.m, seqs = std::max(a.batch, 1);
  const int64_t rows = (a.stacked ? (a.nq + seqs - 1) / seqs : a.n) << a.gsh, tile = keys_form(a) ? 32 : 64;
  const int64_t blocks = seqs * a.hk * std::max<int64_t>(1, (rows + tile - 1) / tile);
  return (int)std::max<int64_t>(1, std::min<int64_t>({kMostSplits, 512 / blocks, per / 256}));
}
size_t part_bytes(const Args& a, int splits) {
  return splits > 1 ? align_up((size_t)splits * a.nq * a.hk * a.g * 2 * (a.dv + 4) * sizeof(float)) : 0;
}

}  // namespace
}  // namespace dattn
}  // namespace geotr

using namespace geotr;
using namespace geotr::dattn;

extern "C" {

size_t geotr_diff_attn_workspace_bytes(const geotr_diff_attn* op) {
  Args a;
  if (make_args(op, a) != GEOTR_OK) return 0;
  return part_bytes(a, choose_splits(a));
}

int geotr_diff_attn_forward(const geotr_diff_attn* op, void* out, float* maps, float* lse, void* ws, size_t ws_bytes, void* stream) {
  Args a;
  const int rc = make_args(op, a);
  if (rc != GEOTR_OK) return rc;
  if (a.nq == 0) return GEOTR_OK;
  GEOTR_CHECK_ARG(out, "geotr_diff_attn_forward: out is a null pointer");
  GEOTR_CHECK_ARG(!maps == !lse, "geotr_diff_attn_forward: maps and lse go together");
  GEOTR_CHECK_ARG((uintptr_t)out % 16 == 0 && (uintptr_t)maps % 16 == 0, "geotr_diff_attn_forward: results are not 16-byte aligned");
  a.out = out, a.maps = maps, a.lse = lse, a.splits = choose_splits(a);
  const size_t need = part_bytes(a, a.splits);
  if (need) {
    if (!ws || ws_bytes < need) return fail(GEOTR_E_WORKSPACE, "geotr_diff_attn_forward: workspace of %zu bytes, %zu needed", ws_bytes, need);
    a.part = (float*)ws;
  }
  hipStream_t s = (hipStream_t)stream;
  if (const int r = launch(op->dtype, a, keys_form(a) && !maps ? kForwardKeys : kForward, s)) return r;
  if (a.splits > 1) {
    const int64_t rows = a.nq * a.hk * a.g;
    const bool many = a.splits > 4;
    const dim3 grid((unsigned)(many ? rows : (rows + 3) / 4));
    auto join = [&](auto one, auto four) { hipLaunchKernelGGL(many ? four : one, grid, dim3(256), 0, s, a); };
    if (op->dtype == GEOTR_F32) join(join_kernel<float, 1>, join_kernel<float, 4>);
    else if (op->dtype == GEOTR_BF16) join(join_kernel<__bf16, 1>, join_kernel<__bf16, 4>);
    else join(join_kernel<_Float16, 1>, join_kernel<_Float16, 4>);
    GEOTR_CHECK_LAUNCH("geotr_diff_attn_forward");
  }
  return GEOTR_OK;
}

size_t geotr_diff_attn_backward_workspace_bytes(const geotr_diff_attn* op) {
  Args a;
  if (make_args(op, a) != GEOTR_OK) return 0;
  const size_t rows = (size_t)a.nq * a.hk * a.g;
  return align_up(8 * rows * sizeof(float)) + align_up(rows * sizeof(float)) + align_up(2 * sizeof(float));
}

int geotr_diff_attn_backward(const geotr_diff_attn* op, const geotr_heads* dout, const float* maps, const float* lse,
                             void* dq, void* dk, void* dv, float* dlam, void* ws, size_t ws_bytes, void* stream) {
  Args a;
  const int rc = make_args(op, a);
  if (rc != GEOTR_OK) return rc;
  GEOTR_CHECK_ARG(dout && dlam, "geotr_diff_attn_backward: null pointer");
  const int size = op->dtype == GEOTR_F32 ? 4 : 2;
  if (const int r = check_view(*dout, (int64_t)a.hk * a.g, size, op->batch, op->n, 64, 1ll << a.gsh, "dout")) return r;
  GEOTR_CHECK_ARG((a.nq == 0 || (maps && lse && dq)) && (a.nk == 0 || (dk && dv)), "geotr_diff_attn_backward: null pointer");
  GEOTR_CHECK_ARG((uintptr_t)maps % 16 == 0 && (uintptr_t)dq % 16 == 0 && (uintptr_t)dk % 16 == 0 && (uintptr_t)dv % 16 == 0,
                  "geotr_diff_attn_backward: results are not 16-byte aligned");
  const size_t rows = (size_t)a.nq * a.hk * a.g, need = geotr_diff_attn_backward_workspace_bytes(op);
  if (!ws || ws_bytes < need) return fail(GEOTR_E_WORKSPACE, "geotr_diff_attn_backward: workspace of %zu bytes, %zu needed", ws_bytes, need);
  Carver c(ws);
  a.rows = c.take<float>(8 * rows), a.drow = c.take<float>(rows);
  float* amax = c.take<float>(2);
  a.dout = *dout, a.maps = const_cast<float*>(maps), a.lse = const_cast<float*>(lse);
  a.gq = dq, a.gk = dk, a.gv = dv, a.amax = amax;
  hipStream_t s = (hipStream_t)stream;
  if (op->dtype == GEOTR_F16) {
    if (const int r = zero_async(amax, 2 * sizeof(float), s)) return r;
    const int64_t chunks = a.nk * a.hk * (a.dv / 8);
    if (chunks) hipLaunchKernelGGL(v_max_kernel, dim3((unsigned)std::min<int64_t>(1024, (chunks + 255) / 256)), dim3(256), 0, s, a, amax + 1);
    GEOTR_CHECK_LAUNCH("geotr_diff_attn_backward");
  }
  if (a.nq) {
    const dim3 grid((unsigned)std::min<size_t>(1 << 20, (rows + 15) / 16));
    if (op->dtype == GEOTR_F32) hipLaunchKernelGGL((del_kernel<float>), grid, dim3(256), 0, s, a, amax);
    else if (op->dtype == GEOTR_BF16) hipLaunchKernelGGL((del_kernel<__bf16>), grid, dim3(256), 0, s, a, amax);
    else hipLaunchKernelGGL((del_kernel<_Float16>), grid, dim3(256), 0, s, a, amax);
    GEOTR_CHECK_LAUNCH("geotr_diff_attn_backward");
  }
  if (const int r = launch(op->dtype, a, kBackward, s)) return r;
  hipLaunchKernelGGL(dlam_kernel, dim3((unsigned)(a.hk * a.g)), dim3(1024), 0, s, a.drow, a.nq, a.g, dlam);
  GEOTR_CHECK_LAUNCH("geotr_diff_attn_backward");
  return GEOTR_OK;
}

}  // extern "C"
