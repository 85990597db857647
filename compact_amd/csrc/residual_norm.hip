// What lies between two blocks of a language model, forward and backward: the
// norm of a block's output, its gate and scale, the residual add, and the norm
// that feeds the next block.
//
//   n1 = y rho1, rho1 = (mean y^2 + eps)^-1/2, u = n1 w_post    (no w_post: u = y)
//   r' = beta r + alpha g u
//   n2 = r' rho2, rho2 = (mean r'^2 + eps)^-1/2, x = n2 w_pre
// The gate g is absent, a value per channel, per (sequence, channel) or per
// token.  Backward, with dx and dr' given and mu(.) a row's mean:
//   t = dr' + rho2 (dn2 - n2 mu(dn2 n2)), dn2 = dx w_pre;   dr = beta t
//   dn1 = alpha g t w_post,  dy = rho1 (dn1 - n1 mu(dn1 n1))   (no w_post: dy = alpha g t)
//   dw_pre = sum dx n2;  G = sum t n1 over tokens:  dw_post = alpha g G,
//   dg = alpha w_post G;  a token's gate: dg = alpha sum_j t u.
// Every sum, statistic and product is fp32; each output is rounded once.  x is
// the norm of the unrounded r', which is still in registers.
//
// HBM-bound: the forward reads two and writes two row tensors, the backward
// reads four and writes two.  A group of `tr` threads holds a row in registers,
// eight columns per thread and vector; a block has `groups` of them side by
// side and goes over its rows with the weights (and the backward's sums over
// tokens, those of more than 8192 columns in LDS) kept in registers.
//
// Measured on one MI355X: forward of 8192 x 2048 bf16 with both norms 27 us (5.0
// TB/s), of 8192 x 4096 49 (5.5); backward of 8192 x 4096 82 us and 5 for the
// partial sums (4.6 TB/s), of 3009 x 1999 fp32, every row unaligned, 31 and 4, of
// 2000 x 16000 bf16 125 in all (3.1 TB/s), of 49923 x 128 fp16 23 in all (3.4
// TB/s).  A large copy reaches 5.0.

#include "compact_amd.h"
#include "row_ops.h"

namespace cpt {
namespace resnorm {

constexpr int kMaxThreads = 1024;
constexpr int kMaxWaves = kMaxThreads / 64;
enum Gate : int { kNone = 0, kChannel = 1, kSequence = 2, kToken = 3 };

struct Shape {
  int64_t rows;        // all tokens
  int64_t seq;         // tokens per sequence (rows without a sequence gate)
  int64_t d;
  int tr, groups;      // threads per row, rows side by side in a block
  int gate, wdt;       // Gate, weights' type
  float alpha, beta, eps;
};

// Sums of N values over the threads of each row group, in every thread: of 16 or 32
// threads by rotations within 16 lanes, of more with one barrier; `red` alternates
// between two buffers from call to call.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float (*red)[kMaxWaves], int tr) {
  if (tr < 64) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] += dpp<0x128, 0xF>(0.f, v[i]);   // row_ror:8
      v[i] += dpp<0x124, 0xF>(0.f, v[i]);
      v[i] += dpp<0x122, 0xF>(0.f, v[i]);
      v[i] += dpp<0x121, 0xF>(0.f, v[i]);
      if (tr == 32) v[i] += __shfl_xor(v[i], 16);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  const int wave = threadIdx.x >> 6, per = tr >> 6;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i][wave] = v[i];
  }
  __syncthreads();
  const int w0 = wave / per * per;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.f;
    for (int w = 0; w < per; ++w) s += red[i][w0 + w];
    v[i] = s;
  }
}

// A thread's eight weights of DT or fp32, ones where there is no tensor.
template <int DT, bool TINY>
__device__ __forceinline__ void ld_weights(const void* w, int wdt, int64_t base, int64_t j,
                                           int64_t d, float v[8]) {
  if (!w) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 1.f;
  } else if (wdt == DT) {
    const Cols<DT, TINY> c(j, d);
    Row8<DT>::unpack(c.ld((const typename Row8<DT>::T*)w + base), v);
  } else {
    const Cols<kF32, TINY> c(j, d);
    Row8<kF32>::unpack(c.ld((const float*)w + base), v);
  }
}

template <int DT, int NV, bool TINY>
__global__ __launch_bounds__(kMaxThreads) void forward_kernel(
    Shape s, const void* __restrict__ residual, int64_t ld_res, const void* __restrict__ y,
    int64_t ld_y, const void* __restrict__ w_post, const void* __restrict__ w_pre,
    const void* __restrict__ gate, void* residual_out, void* x, float* stats) {
  using R = Row8<DT>;
  using T = typename R::T;
  using C = Cols<DT, TINY>;
  __shared__ float red[2][2][kMaxWaves];
  const int group = threadIdx.x / s.tr, tid = threadIdx.x - group * s.tr;
  float a[NV][8], wp[NV][8];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int64_t j = 8 * ((int64_t)c * s.tr + tid);
    float g[8];
    ld_weights<DT, TINY>(w_post, s.wdt, 0, j, s.d, a[c]);
    ld_weights<DT, TINY>(s.gate == kChannel ? gate : nullptr, s.wdt, 0, j, s.d, g);
    ld_weights<DT, TINY>(w_pre, s.wdt, 0, j, s.d, wp[c]);
#pragma unroll
    for (int e = 0; e < 8; ++e) a[c][e] *= s.alpha * g[e];
  }
  const bool ragged = s.d % 8 != 0 || s.tr * NV * 8 != s.d;
  const float inv_d = 1.f / (float)s.d;
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * s.groups;
  struct Loaded {
    typename R::Raw y[NV], r[NV];
  };
  const auto load = [&](int64_t row0, Loaded& q) {
    const int64_t row = min(row0 + group, s.rows - 1);   // groups past it repeat the last row
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const C cols(8 * ((int64_t)c * s.tr + tid), s.d);
      q.y[c] = cols.ld((const T*)(y ? y : residual) + row * (y ? ld_y : ld_res));
      q.r[c] = cols.ld((const T*)residual + row * ld_res);
    }
  };
  Loaded q;
  int64_t row0 = (int64_t)blockIdx.x * s.groups;
  load(row0, q);
  for (; row0 < s.rows; row0 += step, turn ^= 1) {
    const bool in = row0 + group < s.rows;
    const int64_t row = in ? row0 + group : s.rows - 1;
    // the next row's loads go ahead of this one's stores, which would be waited for
    Loaded next;
    load(row0 + step, next);
    if (!TINY && ragged) {
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const C cols(8 * ((int64_t)c * s.tr + tid), s.d);
        R::mask(q.y[c], (1u << cols.skip) - 1, 0);
        R::mask(q.r[c], (1u << cols.skip) - 1, 0);
      }
    }
    const auto& ry = q.y;
    const auto& rr = q.r;
    float r[NV][8];
    float rho1 = 1.f;
    if (y) {
      if (w_post) {
        float sum[1] = {0.f};
#pragma unroll
        for (int c = 0; c < NV; ++c) {
          float v[8];
          R::unpack(ry[c], v);
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[0] += v[e] * v[e];
        }
        group_sum<1>(sum, red[turn], s.tr);
        rho1 = 1.f / sqrtf(sum[0] * inv_d + s.eps);
      }
      float k = rho1;
      if (s.gate == kToken) k *= ld_any(gate, s.wdt, row);
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const C cols(8 * ((int64_t)c * s.tr + tid), s.d);
        float v[8], g[8];
        R::unpack(rr[c], r[c]);
        R::unpack(ry[c], v);
        if (s.gate == kSequence) {
          ld_weights<DT, TINY>(gate, s.wdt, row / s.seq * s.d, 8 * ((int64_t)c * s.tr + tid), s.d,
                               g);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= g[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) r[c][e] = s.beta * r[c][e] + a[c][e] * (v[e] * k);
        if (in) cols.st_own((T*)residual_out + row * s.d, R::pack(r[c]));
      }
    } else {
#pragma unroll
      for (int c = 0; c < NV; ++c) R::unpack(rr[c], r[c]);
    }
    float rho2 = 1.f;
    if (x) {
      float sum[1] = {0.f};
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[0] += r[c][e] * r[c][e];
      group_sum<1>(sum, red[turn] + 1, s.tr);
      rho2 = 1.f / sqrtf(sum[0] * inv_d + s.eps);
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const C cols(8 * ((int64_t)c * s.tr + tid), s.d);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = r[c][e] * rho2 * wp[c][e];
        if (in) cols.st_own((T*)x + row * s.d, R::pack(v));
      }
    }
    if (tid == 0 && in) {
      stats[row] = rho1;
      stats[s.rows + row] = rho2;
    }
    q = next;
  }
}

// grid (chunks of a sequence's rows, sequences).  Block (c, b) takes the row
// groups c, c + chunks, ... of sequence b and leaves its sums over them in
// partial[b * chunks + c]: dw_pre's columns, then G's.
template <int DT, int NV, bool TINY>
__global__ __launch_bounds__(kMaxThreads) void backward_kernel(
    Shape s, const void* __restrict__ d_res_out, int64_t ld_dro, const void* __restrict__ d_x,
    int64_t ld_dx, const void* __restrict__ res_out, int64_t ld_ro, const void* __restrict__ y,
    int64_t ld_y, const float* __restrict__ stats, const void* __restrict__ w_post,
    const void* __restrict__ w_pre, const void* __restrict__ gate, void* d_res, void* d_y,
    void* d_gate, float* partial) {
  using R = Row8<DT>;
  using T = typename R::T;
  using C = Cols<DT, TINY>;
  extern __shared__ __align__(16) float combine[];
  __shared__ float red[2][3][kMaxWaves];
  const int group = threadIdx.x / s.tr, tid = threadIdx.x - group * s.tr;
  const int64_t b = blockIdx.y;
  // Two vectors a thread leave no registers for the weights' sums: LDS has them, a
  // slot of its own for each thread (such a block has one group).  2000 x 16000 bf16
  // with all of it in registers, which spill: 268 us; so 125.
  constexpr bool kInLds = NV > 1;
  float a[NV][8], wp[NV][8], acc_pre[kInLds ? 1 : NV][8], acc_g[kInLds ? 1 : NV][8];
  float4* const slot = reinterpret_cast<float4*>(combine) + tid;
  const auto take = [&](int i, float (&v)[8]) {
    const float4 lo = slot[2 * i * s.tr], hi = slot[(2 * i + 1) * s.tr];
    v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w;
    v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
  };
  const auto put = [&](int i, const float (&v)[8]) {
    slot[2 * i * s.tr] = make_float4(v[0], v[1], v[2], v[3]);
    slot[(2 * i + 1) * s.tr] = make_float4(v[4], v[5], v[6], v[7]);
  };
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    const int64_t j = 8 * ((int64_t)c * s.tr + tid);
    float g[8];
    ld_weights<DT, TINY>(w_post, s.wdt, 0, j, s.d, a[c]);
    ld_weights<DT, TINY>(s.gate == kChannel || s.gate == kSequence ? gate : nullptr, s.wdt,
                         s.gate == kSequence ? b * s.d : 0, j, s.d, g);
    ld_weights<DT, TINY>(w_pre, s.wdt, 0, j, s.d, wp[c]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      a[c][e] *= s.alpha * g[e];
      acc_pre[kInLds ? 0 : c][e] = acc_g[kInLds ? 0 : c][e] = 0.f;
    }
    if (kInLds) put(c, acc_pre[0]), put(NV + c, acc_g[0]);
  }
  const bool ragged = s.d % 8 != 0 || s.tr * NV * 8 != s.d;
  const float inv_d = 1.f / (float)s.d;
  const int64_t step = (int64_t)gridDim.x * s.groups;
  struct Loaded {
    typename R::Raw dr[NV], dx[NV], r[NV], y[NV];
    float rho1, rho2, gate;
  };
  const auto load = [&](int64_t row0, Loaded& q) {
    const int64_t row = b * s.seq + min(row0 + group, s.seq - 1);
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const C cols(8 * ((int64_t)c * s.tr + tid), s.d);
      q.dr[c] = q.dx[c] = q.r[c] = q.y[c] = R::zero();
      if (d_res_out) q.dr[c] = cols.ld((const T*)d_res_out + row * ld_dro);
      if (d_x) {
        q.dx[c] = cols.ld((const T*)d_x + row * ld_dx);
        q.r[c] = cols.ld((const T*)res_out + row * ld_ro);
      }
      if (y) q.y[c] = cols.ld((const T*)y + row * ld_y);
    }
    q.rho1 = stats[row], q.rho2 = stats[s.rows + row];
    q.gate = s.gate == kToken ? ld_any(gate, s.wdt, row) : 1.f;
  };
  int turn = 0;
  Loaded q;
  int64_t row0 = (int64_t)blockIdx.x * s.groups;
  for (; row0 < s.seq; row0 += step, turn ^= 1) {
    const bool in = row0 + group < s.seq;
    const int64_t row = b * s.seq + row0 + group;
    load(row0, q);
    if (!in || (!TINY && ragged)) {   // a group past the last row adds nothing
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const C cols(8 * ((int64_t)c * s.tr + tid), s.d);
        const uint32_t off = !in ? 255 : TINY ? 0 : (1u << cols.skip) - 1;
        R::mask(q.dr[c], off, 0);
        R::mask(q.dx[c], off, 0);
        R::mask(q.r[c], off, 0);
        R::mask(q.y[c], off, 0);
      }
    }
    const float rho1 = q.rho1, rho2 = q.rho2, gt = q.gate;
    // one reduction for both norms: with t = dr' + rho2 (dn2 - n2 m2) left open in m2,
    // sum a n1 t = sum a n1 (dr' + rho2 dn2) - rho2 m2 sum a n1 n2
    float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      float dr[8], dx[8], r[8], v[8];
      R::unpack(q.dr[c], dr);
      R::unpack(q.dx[c], dx);
      R::unpack(q.r[c], r);
      R::unpack(q.y[c], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n2 = r[e] * rho2, dn2 = dx[e] * wp[c][e], an1 = a[c][e] * (v[e] * rho1);
        sum[0] += dn2 * n2;
        sum[1] += an1 * (dr[e] + rho2 * dn2);
        sum[2] += an1 * n2;
      }
    }
    group_sum<3>(sum, red[turn], s.tr);
    if (kInLds) {
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        repack<DT>(q.dr[c]), repack<DT>(q.dx[c]);
        repack<DT>(q.r[c]), repack<DT>(q.y[c]);
      }
    }
    const float m2 = sum[0] * inv_d;
    const float dgt = sum[1] - rho2 * m2 * sum[2];
    const float m1 = w_post ? gt * dgt * inv_d : 0.f;
    if (s.gate == kToken && in && tid == 0) st_any(d_gate, s.wdt, row, dgt);
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const C cols(8 * ((int64_t)c * s.tr + tid), s.d);
      float dr[8], dx[8], r[8], v[8];
      R::unpack(q.dr[c], dr);
      R::unpack(q.dx[c], dx);
      R::unpack(q.r[c], r);
      R::unpack(q.y[c], v);
      float(&sum_pre)[8] = acc_pre[kInLds ? 0 : c];
      float(&sum_g)[8] = acc_g[kInLds ? 0 : c];
      if (kInLds) take(c, sum_pre), take(NV + c, sum_g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float n2 = r[e] * rho2, n1 = v[e] * rho1;
        const float t = dr[e] + rho2 * (dx[e] * wp[c][e] - n2 * m2);
        sum_pre[e] += dx[e] * n2;
        sum_g[e] += gt * t * n1;
        dr[e] = s.beta * t;
        v[e] = rho1 * (gt * a[c][e] * t - n1 * m1);
      }
      if (kInLds) put(c, sum_pre), put(NV + c, sum_g);
      if (in) {
        cols.st_own((T*)d_res + row * s.d, R::pack(dr));
        if (y) cols.st_own((T*)d_y + row * s.d, R::pack(v));
      }
    }
  }
  float* out = partial + (b * gridDim.x + blockIdx.x) * 2 * s.d;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    auto& acc = which ? acc_g : acc_pre;
    if (s.groups == 1) {
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const Cols<kF32, TINY> cols(8 * ((int64_t)c * s.tr + tid), s.d);
        if (kInLds) take(which * NV + c, acc[0]);
        cols.st_own(out + which * s.d, Row8<kF32>::pack(acc[kInLds ? 0 : c]));
      }
    } else if constexpr (!kInLds) {
      // the groups' sums, a column a thread, in group order
      const int64_t pitch = (s.d + 7) / 8 * 8;
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const C cols(8 * ((int64_t)c * s.tr + tid), s.d);
        float* const to = combine + group * pitch + cols.at;
        if (!TINY && cols.skip == 0) {   // aligned: 8 floats a thread
          reinterpret_cast<float4*>(to)[0] =
              make_float4(acc[c][0], acc[c][1], acc[c][2], acc[c][3]);
          reinterpret_cast<float4*>(to)[1] =
              make_float4(acc[c][4], acc[c][5], acc[c][6], acc[c][7]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e >= cols.skip && e < cols.skip + cols.n) to[e] = acc[c][e];
        }
      }
      __syncthreads();
      for (int64_t j = threadIdx.x; j < s.d; j += blockDim.x) {
        float v = combine[j];
#pragma unroll 8
        for (int g = 1; g < s.groups; ++g) v += combine[g * pitch + j];
        out[which * s.d + j] = v;
      }
    }
  }
}

template <int DT>
auto backward_of(int64_t d, int nv) {
  return d < 8     ? backward_kernel<DT, 1, true>
         : nv == 1 ? backward_kernel<DT, 1, false>
                   : backward_kernel<DT, 2, false>;
}

constexpr int kFinCols = 64, kFinSlices = 16;

// grid (columns / 64, results from `base`, 0 or 2): the chunks' sums of 64 columns,
// sixteen slices of them added side by side and then in order.  Result 0: dw_pre; 1:
// dw_post, and dg of a channel gate from the same sum; 2 + b: dg of sequence b, where
// it has a gate of its own.
__global__ __launch_bounds__(kFinCols* kFinSlices) void finish_kernel(
    Shape s, int base, const float* __restrict__ partial, int64_t chunks, int64_t seqs,
    const void* __restrict__ w_post, const void* __restrict__ gate, void* d_w_pre, void* d_w_post,
    void* d_gate) {
  __shared__ float part[kFinSlices][kFinCols];
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const int64_t j = (int64_t)blockIdx.x * kFinCols + lane;
  const int what = base + blockIdx.y;
  const bool in = j < s.d;
  const int64_t first = what >= 2 ? (what - 2) * chunks : 0;
  const int64_t n = what >= 2 ? chunks : chunks * seqs;
  const int64_t per = (n + kFinSlices - 1) / kFinSlices;
  const int64_t c0 = min(n, slice * per), c1 = min(n, c0 + per);
  const float* p = partial + (what ? s.d : 0) + (in ? j : 0);
  float v = 0.f;
  if (what == 1 && s.gate == kSequence) {
    for (int64_t c = c0; c < c1; ++c)
      v += p[(first + c) * 2 * s.d] * (in ? ld_any(gate, s.wdt, c / chunks * s.d + j) : 0.f);
  } else {
#pragma unroll 8
    for (int64_t c = c0; c < c1; ++c) v += p[(first + c) * 2 * s.d];
  }
  part[slice][lane] = v;
  __syncthreads();
  if (slice > 0 || !in) return;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kFinSlices; ++k) sum += part[k][lane];
  if (what == 0) {
    if (d_w_pre) st_any(d_w_pre, s.wdt, j, sum);
    return;
  }
  const float wq = w_post ? ld_any(w_post, s.wdt, j) : 1.f;
  if (what >= 2) {
    st_any(d_gate, s.wdt, (int64_t)(what - 2) * s.d + j, s.alpha * wq * sum);
    return;
  }
  if (s.gate == kChannel) {
    if (d_w_post) st_any(d_w_post, s.wdt, j, s.alpha * ld_any(gate, s.wdt, j) * sum);
    st_any(d_gate, s.wdt, j, s.alpha * wq * sum);
  } else if (d_w_post) {
    st_any(d_w_post, s.wdt, j, s.alpha * sum);
  }
}

inline int launched() { return hipGetLastError() == hipSuccess ? kOk : kErrLaunch; }

constexpr int64_t kMaxD = 8 * kMaxThreads * 2;

// Of a grid's second extent (16 bits wide): more sequences take further launches.
constexpr int64_t kMaxExtent = 65535;
unsigned extent(int64_t n) { return (unsigned)(n < kMaxExtent ? n : kMaxExtent); }
void* from(const void* p, int64_t element, int type) {
  return p ? (char*)p + element * (type == kF32 ? 4 : 2) : nullptr;
}

// Vectors per thread, and the threads and row groups of a block of about `threads`.
// Rows of up to 256 columns share a wavefront, so that its lanes all have columns
// (16 or 32 threads a row against 64: forward of 100000 x 128 bf16 19 and 52 us, of
// 64000 x 256 26 and 36; backward of 49923 x 128 fp16 23 and 50, half of that from
// the groups' sums being added a column a thread).
int plan(Shape& s, int threads) {
  const int64_t vecs = (s.d + 7) / 8;
  const int nv = vecs <= kMaxThreads ? 1 : 2;
  const int64_t t = (vecs + nv - 1) / nv;
  s.tr = t <= 16 ? 16 : t <= 32 ? 32 : (int)((t + 63) / 64 * 64);
  s.groups = threads / s.tr > 1 ? threads / s.tr : 1;
  if (s.groups > s.seq) s.groups = s.seq > 0 ? (int)s.seq : 1;
  return nv;
}

// The backward's blocks: two of 512 threads a CU, which wait for their barriers
// apart (30000 x 512 bf16: 47 us, one of 1024 52); for rows of more than 2048
// columns one of 1024, which leaves half the partial sums (4000 x 8192: 93 us,
// against 102).
int backward_threads(int64_t d) { return d <= 2048 ? 512 : 1024; }

// Chunks of a sequence's rows in the backward: as many blocks as run at a time,
// over all sequences, as far as there are rows.
int64_t backward_chunks(const Shape& s, int64_t seqs) {
  const int64_t blocks = 256 * (1024 / backward_threads(s.d));
  int64_t c = (blocks + seqs - 1) / seqs;
  const int64_t most = (s.seq + s.groups - 1) / s.groups;
  if (c > most) c = most;
  return c < 1 ? 1 : c;
}

bool shape_ok(int64_t rows, int64_t seq, int64_t d, int gate) {
  return rows >= 0 && seq >= 0 && d >= 1 && gate >= kNone && gate <= kToken &&
         (rows == 0 || (seq > 0 && rows % seq == 0)) && (gate == kSequence || seq == rows);
}

}  // namespace resnorm
}  // namespace cpt

using namespace cpt;
using namespace cpt::resnorm;

extern "C" {

int cpt_residual_norm(int dtype, int weight_dtype, const void* residual, int64_t ld_residual,
                      const void* y, int64_t ld_y, const void* w_post, const void* w_pre,
                      const void* gate, int gate_kind, int64_t rows, int64_t seq, int64_t d,
                      float scale, float residual_scale, float eps, void* residual_out, void* x,
                      void* stats, void* stream) {
  if (dtype < kF32 || dtype > kBF16 || (weight_dtype != kF32 && weight_dtype != dtype))
    return kErrDType;
  if (!shape_ok(rows, seq, d, gate_kind)) return kErrShape;
  if (d > kMaxD) return kErrTooLarge;
  if ((gate_kind != kNone) != (gate != nullptr)) return kErrShape;
  if (!y && (w_post || gate || residual_scale != 1.f)) return kErrShape;
  if ((y != nullptr) != (residual_out != nullptr) || (w_pre != nullptr) != (x != nullptr) ||
      (!y && !x))
    return kErrShape;
  if (rows == 0) return kOk;
  if (!residual || !stats || ld_residual < 0 || ld_y < 0) return kErrShape;
  Shape s{rows, seq, d, 0, 0, gate_kind, weight_dtype, scale, residual_scale, eps};
  s.seq = rows;   // blocks take rows of any sequence
  const int nv = plan(s, 256);
  s.seq = seq;
  const int threads = s.tr * s.groups;
  const int64_t blocks = (rows + s.groups - 1) / s.groups;
  const int64_t most = 256 * (2048 / threads);   // as many as can run at a time
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
#define CPT_FWD(DT, NV, TINY)                                                                    \
  forward_kernel<DT, NV, TINY><<<grid, threads, 0, (hipStream_t)stream>>>(                             \
      s, residual, ld_residual, y, ld_y, w_post, w_pre, gate, residual_out, x, (float*)stats)
#define CPT_FWD_NV(DT) \
  (d < 8 ? CPT_FWD(DT, 1, true) : nv == 1 ? CPT_FWD(DT, 1, false) : CPT_FWD(DT, 2, false))
  dtype == kF32 ? CPT_FWD_NV(kF32) : dtype == kF16 ? CPT_FWD_NV(kF16) : CPT_FWD_NV(kBF16);
  return launched();
}

int64_t cpt_residual_norm_backward_workspace_bytes(int64_t rows, int64_t seq, int64_t d,
                                                   int gate_kind) {
  if (!shape_ok(rows, seq, d, gate_kind) || d > kMaxD) return -1;
  if (rows == 0) return 0;
  Shape s{rows, seq, d, 0, 0, gate_kind, kF32, 1.f, 1.f, 0.f};
  plan(s, backward_threads(d));
  const int64_t seqs = rows / seq;
  return seqs * backward_chunks(s, seqs) * 2 * d * 4;
}

int cpt_residual_norm_backward(int dtype, int weight_dtype, const void* d_residual_out,
                               int64_t ld_dro, const void* d_x, int64_t ld_dx,
                               const void* residual_out, int64_t ld_ro, const void* y,
                               int64_t ld_y, const void* stats, const void* w_post,
                               const void* w_pre, const void* gate, int gate_kind, int64_t rows,
                               int64_t seq, int64_t d, float scale, float residual_scale,
                               void* d_residual, void* d_y, void* d_w_pre, void* d_w_post,
                               void* d_gate, void* workspace, void* stream) {
  if (dtype < kF32 || dtype > kBF16 || (weight_dtype != kF32 && weight_dtype != dtype))
    return kErrDType;
  if (!shape_ok(rows, seq, d, gate_kind)) return kErrShape;
  if (d > kMaxD) return kErrTooLarge;
  if ((gate_kind != kNone) != (gate != nullptr) || (gate != nullptr) != (d_gate != nullptr) ||
      (w_post != nullptr) != (d_w_post != nullptr) || (w_pre != nullptr) != (d_w_pre != nullptr) ||
      (w_pre != nullptr) != (d_x != nullptr) || (y != nullptr) != (d_y != nullptr))
    return kErrShape;
  if (!y && (w_post || gate || residual_scale != 1.f)) return kErrShape;
  if (!y && !d_x) return kErrShape;
  const int64_t seqs = rows == 0 ? 0 : rows / seq;
  if (rows > 0 && (!stats || !d_residual || !workspace || (d_x && !residual_out) || ld_dro < 0 ||
                   ld_dx < 0 || ld_ro < 0 || ld_y < 0))
    return kErrShape;
  Shape s{rows, seq, d, 0, 0, gate_kind, weight_dtype, scale, residual_scale, 0.f};
  const int nv = plan(s, backward_threads(d));
  const int64_t chunks = seqs == 0 ? 0 : backward_chunks(s, seqs);
  const hipStream_t st = (hipStream_t)stream;
  if (rows > 0) {
    const int threads = s.tr * s.groups;
    const auto kern = dtype == kF32   ? backward_of<kF32>(d, nv)
                      : dtype == kF16 ? backward_of<kF16>(d, nv)
                                      : backward_of<kBF16>(d, nv);
    // the sums over tokens of rows with two vectors a thread; the groups' of others
    const int64_t floats = nv > 1         ? 2 * nv * s.tr * 8
                           : s.groups > 1 ? s.groups * ((d + 7) / 8 * 8)
                                          : 0;
    const size_t lds = 4 * (size_t)floats;
    if (lds > 62 * 1024 &&
        hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                            (int)lds) != hipSuccess)
      return kErrLaunch;
    for (int64_t seq0 = 0; seq0 < seqs; seq0 += kMaxExtent) {   // tensors from sequence seq0 on
      const int64_t row0 = seq0 * seq;
      const dim3 grid((unsigned)chunks, extent(seqs - seq0));
      kern<<<grid, threads, lds, st>>>(
          s, from(d_residual_out, row0 * ld_dro, dtype), ld_dro, from(d_x, row0 * ld_dx, dtype),
          ld_dx, from(residual_out, row0 * ld_ro, dtype), ld_ro, from(y, row0 * ld_y, dtype), ld_y,
          (const float*)stats + row0, w_post, w_pre, from(gate, seq0 * d, weight_dtype),
          from(d_residual, row0 * d, dtype), from(d_y, row0 * d, dtype), d_gate,
          (float*)workspace + seq0 * chunks * 2 * d);
      const int rc = launched();
      if (rc != kOk) return rc;
    }
  }
  if (d_w_pre || d_w_post || gate_kind == kChannel || gate_kind == kSequence) {
    const auto finish = [&](int base, int64_t seq0, unsigned results) {
      const dim3 grid((unsigned)((d + kFinCols - 1) / kFinCols), results);
      finish_kernel<<<grid, kFinCols * kFinSlices, 0, st>>>(
          s, base, (const float*)workspace + seq0 * chunks * 2 * d, chunks, seqs, w_post, gate,
          d_w_pre, d_w_post, from(d_gate, seq0 * d, weight_dtype));
      return launched();
    };
    const int64_t gated = gate_kind == kSequence ? seqs : 0;
    int rc = finish(0, 0, extent(2 + gated));
    for (int64_t seq0 = kMaxExtent - 2; rc == kOk && seq0 < gated; seq0 += kMaxExtent)
      rc = finish(2, seq0, extent(gated - seq0));
    return rc;
  }
  return kOk;
}

}  // extern "C"
