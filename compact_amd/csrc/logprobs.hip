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
// looked at again, dealt out over the block.  Where a bound leaves too many (more than
// 1024 candidates or maxima, in a row of one wavefront 256 or 128: constant rows, rows with
// little but -inf) or there is none (NaN; more than 64 alternatives for each wavefront
// whose lanes all have columns, as 65 of a row under 1024 columns), a radix selection
// takes its place: five more readings of the row.
//
// Measured on one MI355X, 15% of the rows left out, us a pass among others: 8192 x 32000
// bf16 83 without alternatives (5.4 TB/s), 93 with 20, 115 with 50 in all; 1531 x 50021
// fp16, 50 of them, 45; 7 x 32000, 5 of them, 13 (the kernel 11); the gradient of 8192 x
// 32000 bf16 181 (5.4 TB/s, in part from the Infinity Cache).

#include <algorithm>

#include "compact_amd.h"
#include "row_ops.h"

namespace cpt {
namespace logprobs {

constexpr int kMaxTop = 128;          // alternatives
constexpr int kSlots = 4;             // of a thread: four maxima each, of some of its vectors
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
  int64_t rows, ld_b, ld_s, ignore;
  FastDivU32 seq;
  int v, k, wide, shift;              // 1 << shift vectors a maximum
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

// A maximum m, and the sums of 2^(t - base) and of 2^(t - base) (t - base) over t = x c,
// c = log2(e) / T.  base is the whole number next to m c: then t - base is one fused
// multiply-add, and bases differ exactly.  Past 2^22 (`wide`; whole numbers end at
// 2^24) it is m c itself, and t - base is (x - m) c.
struct Stats {
  float m, base, s, w;
  bool wide;
};
__device__ __forceinline__ bool is_wide(float m, float c) { return !(fabsf(m * c) < 4194304.f); }
__device__ __forceinline__ void rebase(Stats& a, float m, float c) {
  const bool wide = is_wide(m, c);
  const float base = wide ? 0.f : rintf(m * c);
  float d = a.base - base;
  if (wide || a.wide)
    d = wide && a.wide ? (a.m - m) * c : wide ? fmaf(-c, m, a.base) : fmaf(c, a.m, -base);
  if (a.m > -INFINITY) {        // else s and w are 0, or NaN
    const float f = exp2f(d);
    a.w = (a.w + fmaxf(d, -1024.f) * a.s) * f;    // far below: 0, not 0 * inf
    a.s *= f;
  }
  a.m = m, a.base = base, a.wide = wide;
}

// One wavefront's rows are narrow: its block is kept small, so that many run side by side.
template <int NT>
struct Shared {
  static constexpr int kCand = NT == 64 ? 256 : 1024;   // candidates that are sorted
  static constexpr int kList = NT == 64 ? 128 : 1024;   // maxima that reach the bound
  float red[3][NT / 64];
  float bound[NT / 64];
  int count, active, need;
  uint32_t prefix;
  int scan[NT / 64];
  uint16_t list[kList];
  union {
    uint2 top[kSlots][NT];
    int hist[256];
  };
  uint64_t cand[kCand];
};

template <int DT>
__device__ __forceinline__ typename Row8<DT>::Raw ld_vec(const typename Row8<DT>::T* row, int vec,
                                                         int v) {
  return row_ld<DT>(row, (int64_t)vec * 8, v, Row8<DT>::kNegInf);
}

// Four vectors of a row, `step` apart, from the whole ones below `n` (past them the last
// again).
template <int DT>
struct Four {
  typename Row8<DT>::Raw raw[4];
  __device__ __forceinline__ void ld(const typename Row8<DT>::T* row, int i, int step, int n) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      raw[u] = Row8<DT>::ld(row + (int64_t)min(i + u * step, n - 1) * 8);
  }
};

// N vectors into a thread's statistics, and their maxima into those of the slot.  CUT: the
// first `count` of them, the others being other threads'.
template <int DT, int N, bool CUT>
__device__ __forceinline__ void take(Stats& st, const typename Row8<DT>::Raw* raw, float c,
                                     float slot[N], bool first, int count) {
  float top = -INFINITY, low = INFINITY;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    float x[8];
    Row8<DT>::unpack(raw[u], x);
    float most = x[0];
    low = fminf(low, x[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) most = fmaxf(most, x[j]), low = fminf(low, x[j]);
    if (CUT && u >= count) most = -INFINITY;
    slot[u] = first ? most : fmaxf(slot[u], most);
    top = fmaxf(top, most);
  }
  if (top > st.m) rebase(st, top, c);
  if (low * c > -1e38f && !st.wide) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      float x[8], s = CUT ? 0.f : st.s, w = CUT ? 0.f : st.w;
      Row8<DT>::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = fmaf(x[j], c, -st.base);
        const float e = __builtin_amdgcn_exp2f(t);
        s += e;
        w = fmaf(e, t, w);
      }
      st.s = !CUT ? s : u < count ? st.s + s : st.s;
      st.w = !CUT ? w : u < count ? st.w + w : st.w;
    }
  } else {                      // -inf among them (0 * inf), or far from 0
    const float m = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      if (CUT && u >= count) break;
      float x[8];
      Row8<DT>::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = st.wide ? (x[j] - m) * c : fmaf(x[j], c, -st.base);
        const float e = __builtin_amdgcn_exp2f(t);
        st.s += e;
        st.w = fmaf(e, fmaxf(t, -256.f), st.w);
      }
    }
  }
}

// A maximum in 16 bits: the type's own, of fp32 the next bf16 number from it upwards.
template <int DT>
__device__ __forceinline__ uint32_t top_bits(float x) {
  const uint32_t b = __float_as_uint(x);
  if (DT == kF16) return f32_to_f16_bits(x);
  return (b + (DT == kF32 && !(b >> 31) ? 0xFFFFu : 0u)) >> 16;
}
template <int DT>
__device__ __forceinline__ float top_value(uint32_t b) {
  return DT == kF16 ? f16_bits_to_f32((uint16_t)b) : __uint_as_float(b << 16);
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
  const uint32_t b = A.seq.div((uint32_t)r), n = (uint32_t)r - b * A.seq.d;
  const auto* row = (const typename R::T*)A.x + b * A.ld_b + n * A.ld_s;
  const float c = A.inv_t * kLog2e;
  const float chosen = threadIdx.x == 0 && A.targets ? Elem<DT>::ld(row + y) : 0.f;
  const int vecs = (v + 7) / 8, whole = v / 8;

  // 1. maximum, sum and weighted sum of this thread's columns: four vectors at a time
  Stats st{-INFINITY, 0.f, 0.f, 0.f, false};
  if (whole > 0) {
    Four<DT> cur;
    const int first = threadIdx.x & ~63;      // the wave's: branches on it are uniform
    float slot[4];
    int group = 0;
    for (int i = threadIdx.x, w = first; w < whole; i += 4 * NT, w += 4 * NT) {
      cur.ld(row, i, NT, whole);
      const bool fresh = (group & ((1 << A.shift) - 1)) == 0;
      if (w + 3 * NT + 63 < whole)
        take<DT, 4, false>(st, cur.raw, c, slot, fresh, 4);
      else if (i < whole)
        take<DT, 4, true>(st, cur.raw, c, slot, fresh, (whole - i + NT - 1) / NT);
      if (k > 0) {
        S.top[group >> A.shift][threadIdx.x] =
            make_uint2(top_bits<DT>(slot[0]) | top_bits<DT>(slot[1]) << 16,
                       top_bits<DT>(slot[2]) | top_bits<DT>(slot[3]) << 16);
        ++group;
      }
    }
  }
  if (threadIdx.x == 0 && whole < vecs) {
    const typename R::Raw raw = ld_vec<DT>(row, whole, v);
    float slot[1];
    take<DT, 1, false>(st, &raw, c, slot, true, 1);
  }

  // 2. the row's
  const float mine = st.m;
  const float wm = wave_max(mine);
  if (lane == 0) S.red[0][wave] = wm;
  // wavefronts whose lanes all have columns, and the first
  const int full = max(1, min(kWaves, whole / 64));
  if (k > 0) {
    // a number that k / full of the wave's maxima reach and, in eight halvings, few more
    const int want = (k + full - 1) / full;
    float bound = wm;
    if (want > 1) {
      const uint64_t has = __ballot(mine > -INFINITY);
      bound = __popcll(has) < want ? -INFINITY : -wave_max(mine > -INFINITY ? -mine : -INFINITY);
      float high = wm;
      for (int n = 0; n < 8 && bound < high && bound > -INFINITY; ++n) {
        const float mid = 0.5f * bound + 0.5f * high;
        const int reach = __popcll(__ballot(mine >= mid));
        if (reach < want) {
          high = mid;
        } else {
          bound = mid;
          if (reach == want) break;
        }
      }
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
  // of e^(z - m / T)
  const float log_s = logf(s) - (st.wide ? 0.f : fmaf(m, c, -st.base) * kLn2);
  if (threadIdx.x == 0) {
    A.lse[r] = empty ? -INFINITY : fmaf(m, A.inv_t, log_s);
    const float h = logf(s) - (w2 / s) * kLn2;
    A.entropy[r] = empty || h < 0.f ? 0.f : h;    // no less than 0 by rounding; NaN stays
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
    // the maxima that reach it
    if (mine >= bound)
      for (int g = 0, w = threadIdx.x; w < whole; ++g, w += (4 * NT) << A.shift) {
        const uint2 tops = S.top[g][threadIdx.x];
        const uint32_t bits[4] = {tops.x & 0xFFFFu, tops.x >> 16, tops.y & 0xFFFFu, tops.y >> 16};
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (top_value<DT>(bits[u]) >= bound) {
            const int at = atomicAdd(&S.active, 1);
            if (at < S.kList) S.list[at] = (uint16_t)((g * 4 + u) * NT + threadIdx.x);
          }
      }
    __syncthreads();
    // and their vectors again: every fourth of the thread's from the slot's start on
    const int per = A.shift, active = S.active;
    far = active > S.kList;
    for (int q = threadIdx.x; !far && q < active << per; q += NT) {
      const int entry = S.list[q >> per], slot = entry / NT;
      const int nth = ((slot >> 2 << per) + (q & ((1 << per) - 1))) * 4 + (slot & 3);
      const int vec = (entry & (NT - 1)) + nth * NT;
      if (vec >= whole) continue;
      float x[8];
      R::unpack(R::ld(row + (int64_t)vec * 8), x);
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) hits |= x[j] >= bound ? 1u << j : 0u;
      if (hits == 0) continue;
      int at = atomicAdd(&S.count, __popc(hits));
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (hits >> j & 1) {
          if (at < S.kCand) S.cand[at] = order_key(x[j], vec * 8 + j);
          ++at;
        }
    }
    // columns past the last whole vector
    const int rest = whole * 8 + (int)threadIdx.x;
    if (threadIdx.x < 8 && rest < v) {
      const float x = Elem<DT>::ld(row + rest);
      if (x >= bound) {
        const int at = atomicAdd(&S.count, 1);
        if (at < S.kCand) S.cand[at] = order_key(x, rest);
      }
    }
    __syncthreads();
    far = far || S.count > S.kCand;
    __syncthreads();
  }
  if (far) radix_candidates<DT, NT>(row, v, k, S);

  // 4. in order
  const int count = S.count;
  for (int a = threadIdx.x; a < count; a += NT) {
    const uint64_t key = S.cand[a];
    int rank = 0;
#pragma unroll 8
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
  int64_t rows, ld_b, ld_s, gld_b, gld_s, ignore;
  FastDivU32 seq, chunks;
  int v, wide;
  float inv_t;
};

constexpr int kGradThreads = 256, kGradVecs = 4;

template <int DT>
__global__ __launch_bounds__(kGradThreads) void logprobs_grad_kernel(const LogGradArgs A) {
  using R = Row8<DT>;
  const uint32_t r = A.chunks.div(blockIdx.x), b = A.seq.div(r), n = r - b * A.seq.d;
  const int chunk = (int)(blockIdx.x - r * A.chunks.d), v = A.v;
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
  if (rows < 0 || vocab <= 0 || seq <= 0 || !(temperature > 0.f) || !(temperature < INFINITY) ||
      !(kLog2e / temperature < INFINITY))
    return kErrShape;
  if (vocab > 1 << 24 || rows > 0x7FFFFFFF) return kErrTooLarge;
  return rows && !logits ? kErrShape : kOk;
}

}  // namespace logprobs
}  // namespace cpt

using namespace cpt;
using namespace cpt::logprobs;

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
  // A row is one wavefront's where it is short: nothing to wait for (with 20 alternatives,
  // 16384 x 12000 bf16 83 us, with 256 threads 105; 8192 x 16000 58 and 59, without
  // alternatives 49 and 45; 8192 x 16000 fp32 93 and 85), unless so many are asked that its
  // lanes' maxima are a weak bound.  A row for each CU or fewer: the chain of loads is
  // shorter with more threads.
  const bool narrow = vocab * (dtype == kF32 ? 4 : 2) <= (k > 0 ? 32768 : 24576);
  const int threads = rows <= 256 && vocab > 8192 ? 1024 : narrow && k <= 48 ? 64 : 256;
  int shift = 0;
  while ((vocab / 8 + ((4 * threads) << shift) - 1) / ((4 * threads) << shift) > kSlots) ++shift;
  const LogArgs A{logits, targets, (float*)logprobs, (float*)entropy, (float*)lse,
                  (float*)stats, (float*)top_logprobs, (int64_t*)top_indices, rows, ld_batch,
                  ld_row, ignore_index,
                  FastDivU32::make((uint32_t)std::min<int64_t>(seq, 0x7FFFFFFF)), (int)vocab,
                  (int)k, target_wide, shift, 1.f / temperature};
  const hipStream_t st = (hipStream_t)stream;
  const unsigned grid = (unsigned)rows;
#define CPT_LP(DT)                                                           \
  (threads == 64    ? logprobs_kernel<DT, 64><<<grid, 64, 0, st>>>(A)        \
   : threads == 256 ? logprobs_kernel<DT, 256><<<grid, 256, 0, st>>>(A)      \
                    : logprobs_kernel<DT, 1024><<<grid, 1024, 0, st>>>(A))
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
                                const void* d_logprobs, const void* d_entropy, void* grad,
                                int64_t gld_batch, int64_t gld_row, void* stream) {
  if (const int rc = check_logits(dtype, rows, vocab, seq, logits, temperature)) return rc;
  if (rows == 0) return kOk;
  if ((!lse && !stats) || !grad || (d_logprobs && !targets) || (d_entropy && !entropy))
    return kErrShape;
  LogGradArgs A{logits, targets, (const float*)lse, (const float*)stats, (const float*)entropy,
                (const float*)d_logprobs, (const float*)d_entropy, grad, rows, ld_batch,
                ld_row, gld_batch, gld_row, ignore_index,
                FastDivU32::make((uint32_t)std::min<int64_t>(seq, 0x7FFFFFFF)), {}, (int)vocab,
                target_wide, 1.f / temperature};
  constexpr int kChunk = kGradThreads * kGradVecs * 8;
  const int64_t chunks = (vocab + kChunk - 1) / kChunk;
  A.chunks = FastDivU32::make((uint32_t)chunks);
  const int64_t grid = rows * chunks;
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
