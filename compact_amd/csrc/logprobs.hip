// Log probabilities of given tokens, with each row's entropy and its likeliest
// alternatives, and their gradient.
//
// Over a row of V logits x, z = x / T:
//   lse = log sum e^z;  log p = z - lse;  H = -sum p log p
//   outputs log p[target], H, lse, and the k largest log p with their columns
//   (ties to the lowest column)
//   d x_j = (a (1[j = target] - p_j) - b p_j (log p_j + H)) / T
// with a, b the gradients of log p[target] and H.
//
// Bound: HBM, one read of the logits (backward: and one write).  The forward is one
// pass: a thread keeps the maximum of its own columns, their sum of e^(z - max) and
// of e^(z - max) (z - max), both rebased once in four vectors; the entropy is then
// log s - w / s, a sum of terms of one sign.  Alternatives cost no more reading of
// note: the k-th largest of the threads' maxima (a bound that at least k columns
// reach) leaves about k threads with candidates, and only those threads' columns are
// looked at again, dealt out over the block.  Where a bound leaves too many (constant
// rows, rows with little but -inf, NaN), a radix selection takes its place.

#include <type_traits>

#include "compact_amd.h"
#include "row_ops.h"

namespace cpt {
namespace {

constexpr int kMaxTop = 128;          // alternatives
constexpr int kMaxCand = 1024;        // candidates that are sorted
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LogArgs {
  const void* x;
  const void* targets;
  float* logp;
  float* entropy;
  float* lse;
  float* stats;
  float* top_logp;
  int64_t* top_idx;
  int64_t rows, seq, ld_b, ld_s, ignore;
  int v, k, wide;
  float inv_t;
};

// A value's place in the order of a selection: NaN first, then by size; -0 is 0.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = x == x ? __float_as_uint(x + 0.f) : 0x7FC00000u;
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float x, int col) {
  return (uint64_t)order_bits(x) << 32 | (uint32_t)~col;
}
__device__ __forceinline__ float order_value(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b >> 31 ? b & 0x7FFFFFFFu : ~b);
}

// max, sum of 2^(t - max) and of 2^(t - max) (t - max) over t = x log2(e) / T, the max
// kept as x.
struct Stats {
  float m, s, w;
};
__device__ __forceinline__ void rebase(Stats& a, float m, float k) {
  if (a.m == -INFINITY) {
    a.m = m;                  // s and w are 0 (or NaN)
    return;
  }
  const float d = (a.m - m) * k, f = exp2f(d);
  // far below: 0, not 0 * inf
  a.w = (a.w + fmaxf(d, -1024.f) * a.s) * f;
  a.s *= f;
  a.m = m;
}

template <int NT>
struct Shared {
  float red[3][NT / 64];
  float bound[NT / 64];
  int count, active, need;
  uint32_t prefix;
  int hist[256];
  int scan[NT / 64];
  uint16_t list[NT];
  uint64_t cand[kMaxCand];
};

template <int DT>
__device__ __forceinline__ typename Row8<DT>::Raw ld_vec(const typename Row8<DT>::T* row, int vec,
                                                         int v) {
  return row_ld<DT>(row, (int64_t)vec * 8, v, Row8<DT>::kNegInf);
}

// Candidates by radix selection: the k largest keys' columns into S.cand.
template <int DT, int NT>
__device__ void radix_candidates(const typename Row8<DT>::T* row, int v, int k, Shared<NT>& S) {
  const int vecs = (v + 7) / 8;
  if (threadIdx.x == 0) S.prefix = 0, S.need = k;
  uint32_t mask = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += NT) S.hist[i] = 0;
    __syncthreads();
    const uint32_t prefix = S.prefix;
    for (int i = threadIdx.x; i < vecs; i += NT) {
      float x[8];
      Row8<DT>::unpack(ld_vec<DT>(row, i, v), x);
      for (int j = 0; j < 8 && i * 8 + j < v; ++j) {
        const uint32_t o = order_bits(x[j]);
        if ((o & mask) == prefix) atomicAdd(&S.hist[o >> shift & 255], 1);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int need = S.need, b = 255;
      while (S.hist[b] < need) need -= S.hist[b--];
      S.need = need;
      S.prefix = prefix | (uint32_t)b << shift;
    }
    mask |= 255u << shift;
    __syncthreads();
  }
  // all above the k-th value, and of its equals the first S.need by column
  const uint32_t kth = S.prefix;
  const int need = S.need;
  if (threadIdx.x == 0) S.count = 0;
  __syncthreads();
  int before = 0;
  for (int i0 = 0; i0 < vecs; i0 += NT) {
    const int i = i0 + threadIdx.x;
    float x[8];
    int equal = 0;
    if (i < vecs) {
      Row8<DT>::unpack(ld_vec<DT>(row, i, v), x);
      for (int j = 0; j < 8 && i * 8 + j < v; ++j) {
        const uint32_t o = order_bits(x[j]);
        if (o > kth) S.cand[atomicAdd(&S.count, 1)] = order_key(x[j], i * 8 + j);
        equal += o == kth;
      }
    }
    // the equals of the threads before this one
    int run = equal;
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(run, o);
      if ((threadIdx.x & 63) >= o) run += u;
    }
    if ((threadIdx.x & 63) == 63) S.scan[threadIdx.x >> 6] = run;
    __syncthreads();
    int rank = before + run - equal;
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) rank += S.scan[w];
    for (int w = 0; w < NT / 64; ++w) before += S.scan[w];
    if (equal)
      for (int j = 0; j < 8 && i * 8 + j < v; ++j)
        if (order_bits(x[j]) == kth && rank++ < need)
          S.cand[atomicAdd(&S.count, 1)] = order_key(x[j], i * 8 + j);
    __syncthreads();
  }
}

template <int DT, int NT>
__global__ __launch_bounds__(NT) void logprobs_kernel(const LogArgs A) {
  __shared__ Shared<NT> S;
  using R = Row8<DT>;
  constexpr int kWaves = NT / 64;
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int v = A.v, k = A.k;
  int64_t y = -1;
  if (A.targets) {
    y = ld_index(A.targets, A.wide, r);
    if (y == A.ignore || y < 0 || y >= v) {    // left out
      if (threadIdx.x == 0) {
        A.logp[r] = A.entropy[r] = A.lse[r] = 0.f;
        if (A.stats) A.stats[r] = A.stats[A.rows + r] = 0.f;
      }
      for (int i = threadIdx.x; i < k; i += NT) {
        A.top_logp[r * k + i] = -INFINITY;
        A.top_idx[r * k + i] = -1;
      }
      return;
    }
  }
  const int64_t b = r / A.seq;
  const auto* row = (const typename R::T*)A.x + b * A.ld_b + (r - b * A.seq) * A.ld_s;
  const float c = A.inv_t * kLog2e;
  const float chosen = threadIdx.x == 0 && A.targets ? Elem<DT>::ld(row + y) : 0.f;
  const int vecs = (v + 7) / 8, whole = v / 8;

  // 1. maximum, sum and weighted sum of this thread's columns
  Stats st{-INFINITY, 0.f, 0.f};
  auto take = [&](const typename R::Raw* raw, auto count) {
    constexpr int N = decltype(count)::value;
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float x[8];
      R::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
    }
    if (top > st.m) rebase(st, top, c);
    const float base = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float x[8];
      R::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = (x[j] - base) * c;     // exact near the maximum, of any size
        const float e = __builtin_amdgcn_exp2f(t);
        st.s += e;
        st.w = fmaf(e, fmaxf(t, -256.f), st.w);
      }
    }
  };
  int i = threadIdx.x;
  for (; i + 3 * NT < whole; i += 4 * NT) {
    typename R::Raw raw[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) raw[u] = R::ld(row + (int64_t)(i + u * NT) * 8);
    take(raw, std::integral_constant<int, 4>{});
  }
  for (; i < vecs; i += NT) {
    const typename R::Raw raw = ld_vec<DT>(row, i, v);
    take(&raw, std::integral_constant<int, 1>{});
  }

  // 2. the row's
  const float mine = st.m;
  const float wm = wave_max(mine);
  if (lane == 0) S.red[0][wave] = wm;
  // wavefronts whose lanes all have columns, and the first
  const int full = max(1, min(kWaves, vecs / 64));
  if (k > 0) {
    // the wave's k / full-th largest maximum of a lane (rounded up)
    float left = mine, bound = wm;
    for (int n = (k + full - 1) / full; n > 1 && bound > -INFINITY; --n) {
      const uint64_t who = __ballot(left == bound);
      if (lane == (int)__builtin_ctzll(who)) left = -INFINITY;
      bound = wave_max(left);
    }
    if (lane == 0) S.bound[wave] = bound;
    if (threadIdx.x == 0) S.count = S.active = 0;
  }
  __syncthreads();
  float m = S.red[0][0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, S.red[0][w]);
  rebase(st, m, c);
  const float ws = wave_sum(st.s), ww = wave_sum(st.w);
  if (lane == 0) S.red[1][wave] = ws, S.red[2][wave] = ww;
  __syncthreads();
  float s = 0.f, w2 = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) s += S.red[1][w], w2 += S.red[2][w];
  const bool empty = m == -INFINITY && s == 0.f;      // -inf alone
  const float log_s = logf(s);
  if (threadIdx.x == 0) {
    A.lse[r] = empty ? -INFINITY : fmaf(m, A.inv_t, log_s);
    A.entropy[r] = empty ? 0.f : log_s - (w2 / s) * kLn2;
    if (A.targets)
      A.logp[r] = empty ? -INFINITY : (chosen - m) * A.inv_t - log_s;
    if (A.stats) {
      A.stats[r] = m;
      A.stats[A.rows + r] = log_s;
    }
  }
  if (k == 0) return;

  // 3. the columns that reach the bound
  float bound = S.bound[0];
  for (int w = 1; w < full; ++w) bound = fminf(bound, S.bound[w]);
  bool far = !(s < INFINITY) || bound == -INFINITY;   // NaN, or too few
  if (!far) {
    if (mine >= bound) S.list[atomicAdd(&S.active, 1)] = (uint16_t)threadIdx.x;
    __syncthreads();
    const int per = (vecs + NT - 1) / NT, total = S.active * per;
    for (int q = threadIdx.x; q < total; q += NT) {
      const int a = q / per, vec = S.list[a] + (q - a * per) * NT;
      if (vec >= vecs) continue;
      float x[8];
      R::unpack(ld_vec<DT>(row, vec, v), x);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (x[j] >= bound && vec * 8 + j < v) {
          const int at = atomicAdd(&S.count, 1);
          if (at < kMaxCand) S.cand[at] = order_key(x[j], vec * 8 + j);
        }
    }
    __syncthreads();
    far = S.count > kMaxCand;
    __syncthreads();
  }
  if (far) radix_candidates<DT, NT>(row, v, k, S);

  // 4. in order
  const int count = S.count;
  for (int a = threadIdx.x; a < count; a += NT) {
    const uint64_t key = S.cand[a];
    int rank = 0;
    for (int o = 0; o < count; ++o) rank += S.cand[o] > key;
    if (rank < k) {
      const float x = order_value(key);
      A.top_logp[r * k + rank] =
          x == -INFINITY && s == s ? -INFINITY : (x - m) * A.inv_t - log_s;
      A.top_idx[r * k + rank] = (uint32_t)~(uint32_t)key;
    }
  }
}

struct LogGradArgs {
  const void* x;
  const void* targets;
  const float* lse;
  const float* stats;
  const float* entropy;
  const float* d_logp;
  const float* d_entropy;
  void* grad;
  int64_t rows, seq, ld_b, ld_s, gld_b, gld_s, ignore;
  int v, wide, chunks;
  float inv_t;
};

constexpr int kGradThreads = 256, kGradVecs = 4;

template <int DT>
__global__ __launch_bounds__(kGradThreads) void logprobs_grad_kernel(const LogGradArgs A) {
  using R = Row8<DT>;
  const int64_t r = blockIdx.x / A.chunks;
  const int chunk = (int)(blockIdx.x - r * A.chunks), v = A.v;
  const int64_t b = r / A.seq, n = r - b * A.seq;
  const auto* row = (const typename R::T*)A.x + b * A.ld_b + n * A.ld_s;
  auto* out = (typename R::T*)A.grad + b * A.gld_b + n * A.gld_s;
  int64_t y = -1;
  bool live = true;
  if (A.targets) {
    y = ld_index(A.targets, A.wide, r);
    live = y != A.ignore && y >= 0 && y < v;
  }
  // lse = m / T + l; one number of 32 bits would not hold l beside a large m
  const float m = A.stats ? A.stats[r] : 0.f, l = A.stats ? A.stats[A.rows + r] : A.lse[r];
  const float ga = live && A.targets && A.d_logp ? A.d_logp[r] * A.inv_t : 0.f;
  const float gb = live && A.d_entropy ? A.d_entropy[r] * A.inv_t : 0.f;
  const float h = live && A.d_entropy ? A.entropy[r] : 0.f;
  // nothing to choose from, or nothing asked: zeros, whatever the logits are
  live = live && m != -INFINITY && l != -INFINITY && (ga != 0.f || gb != 0.f);
  const int at = (chunk * kGradVecs * kGradThreads + (int)threadIdx.x) * 8;
  typename R::Raw raw[kGradVecs];
  if (live) {
#pragma unroll
    for (int u = 0; u < kGradVecs; ++u)
      raw[u] = row_ld<DT>(row, at + u * kGradThreads * 8, v, R::kNegInf);
  }
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int j0 = at + u * kGradThreads * 8;
    float x[8];
    if (live) {
      R::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float lp = fmaf(x[j] - m, A.inv_t, -l);
        const float p = __builtin_amdgcn_exp2f(lp * kLog2e);
        // p = 0 has no entropy, at -inf too
        x[j] = -p * fmaf(gb, fmaxf(lp, -1024.f) + h, ga);
        if (j0 + j == y) x[j] += ga;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 0.f;
    }
    row_st<DT>(out, j0, v, R::pack(x));
  }
}

int check_logits(int dtype, int64_t rows, int64_t vocab, int64_t seq, const void* logits,
                 float temperature) {
  if (dtype < 0 || dtype > 2) return kErrDType;
  if (rows < 0 || vocab <= 0 || seq <= 0 || !(temperature > 0.f) || !(temperature < INFINITY))
    return kErrShape;
  if (vocab > 1 << 24 || rows > 0x7FFFFFFF) return kErrTooLarge;
  return rows && !logits ? kErrShape : kOk;
}

}  // namespace
}  // namespace cpt

using namespace cpt;

extern "C" {

int cpt_token_logprobs(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t seq,
                       int64_t ld_batch, int64_t ld_row, int target_wide, const void* targets,
                       int64_t ignore_index, float temperature, int64_t k, void* logprobs,
                       void* entropy, void* lse, void* stats, void* top_logprobs,
                       void* top_indices, void* stream) {
  if (const int rc = check_logits(dtype, rows, vocab, seq, logits, temperature)) return rc;
  if (k < 0 || k > vocab) return kErrShape;
  if (k > kMaxTop) return kErrTooLarge;
  if (rows == 0) return kOk;
  if (!entropy || !lse || (targets != nullptr) != (logprobs != nullptr) ||
      (k && (!top_logprobs || !top_indices)))
    return kErrShape;
  const LogArgs A{logits, targets, (float*)logprobs, (float*)entropy, (float*)lse,
                  (float*)stats, (float*)top_logprobs, (int64_t*)top_indices, rows, seq, ld_batch, ld_row,
                  ignore_index, (int)vocab, (int)k, target_wide, 1.f / temperature};
  const hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)rows;
  // few rows: a row is a chain of loads, shorter with more threads
  const bool wide = rows <= 512 && vocab > 4096;
#define CPT_LP(DT) \
  (wide ? logprobs_kernel<DT, 1024><<<grid, 1024, 0, st>>>(A) : logprobs_kernel<DT, 256><<<grid, 256, 0, st>>>(A))
  if (dtype == kF32)
    CPT_LP(kF32);
  else if (dtype == kF16)
    CPT_LP(kF16);
  else
    CPT_LP(kBF16);
#undef CPT_LP
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

int cpt_token_logprobs_backward(int dtype, const void* logits, int64_t rows, int64_t vocab,
                                int64_t seq, int64_t ld_batch, int64_t ld_row, int target_wide,
                                const void* targets, int64_t ignore_index, float temperature,
                                const void* lse, const void* stats, const void* entropy,
                                const void* d_logprobs, const void* d_entropy, void* grad, int64_t gld_batch,
                                int64_t gld_row, void* stream) {
  if (const int rc = check_logits(dtype, rows, vocab, seq, logits, temperature)) return rc;
  if (rows == 0) return kOk;
  if ((!lse && !stats) || !grad || (d_logprobs && !targets) || (d_entropy && !entropy)) return kErrShape;
  LogGradArgs A{logits, targets, (const float*)lse, (const float*)stats, (const float*)entropy,
                (const float*)d_logprobs, (const float*)d_entropy, grad, rows, seq, ld_batch,
                ld_row, gld_batch, gld_row, ignore_index, (int)vocab, target_wide, 0,
                1.f / temperature};
  A.chunks = (int)((vocab + kGradThreads * kGradVecs * 8 - 1) / (kGradThreads * kGradVecs * 8));
  const int64_t grid = rows * A.chunks;
  if (grid > 0x7FFFFFFF) return kErrTooLarge;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == kF32)
    logprobs_grad_kernel<kF32><<<(unsigned)grid, kGradThreads, 0, st>>>(A);
  else if (dtype == kF16)
    logprobs_grad_kernel<kF16><<<(unsigned)grid, kGradThreads, 0, st>>>(A);
  else
    logprobs_grad_kernel<kBF16><<<(unsigned)grid, kGradThreads, 0, st>>>(A);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // extern "C"
