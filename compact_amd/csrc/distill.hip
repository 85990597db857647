// Distillation from a teacher's top logits: the loss of each row of student
// logits z [rows, V] and its gradient, in one pass over them.
//
// With q = softmax(z / tau) and the teacher's K entries (index, logit t):
//   no log-sum-exp:  p_k = softmax(t / tau) over the entries, p_rest = 0
//   with it (lse):   p_k = exp(t_k / tau - lse), p_rest = max(0, 1 - sum p),
//                    q_rest = the sum of q outside the entries
//   soft = tau^2 (sum p_k (log p_k - log q_k) + p_rest (log p_rest - log q_rest))
//   hard = log sum exp z - z_y
//   loss = alpha soft + (1 - alpha) hard
//   dz_j = alpha tau (q_j P - p_j - [j no entry] p_rest q_j / q_rest)
//          + (1 - alpha) (softmax(z)_j - [j = y]),         P = sum p + p_rest
// An entry whose index lies outside [0, V) is absent; a row with no entries has
// no soft term.  A row whose label is `ignore` or outside [0, V) is not read:
// its loss and gradient are zero.
//
// HBM-bound: a row is read once and its gradient written once.  A block holds a
// row in registers between the two (as stored, 16 bytes a vector), so the
// softmax's maximum and sums and the gradient are three passes over registers.
// Rows too wide for the registers are read again for the gradient.  The first
// wavefront reads the teacher's entries meanwhile; the gradient of an entry's or
// the label's column is written over the general one after a barrier.
// Statistics are fp32, kept as (maximum, sum of exponentials): one exchange over
// the block per row.  With a tail the columns outside the entries are summed
// about their own maximum, so q_rest keeps its digits however small it is; where
// nothing is left outside (all of it -inf), the p_rest term falls away.

#include "compact_amd.h"
#include "row_ops.h"

namespace cpt {
namespace distill {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kMaxWaves = 16;
constexpr int kMaxEntries = 2048;
constexpr int64_t kMaxVocab = 1 << 19;
constexpr int kStream = 0;   // NV of the kernel that reads a row twice

struct Args {
  int64_t rows, vocab;
  const void* logits;
  int64_t seq, ld_b, ld_s;        // row = (b, s): b * ld_b + s * ld_s
  void* grad;
  int64_t gld_b, gld_s;
  const void* top;                // [rows, K] teacher logits and indices
  const void* idx;
  int top_dtype, idx_wide;
  int k;
  const float* lse;
  const void* labels;
  int label_wide;
  int64_t ignore;
  float tau, alpha, grad_scale;
  const float* grad_out;          // null, one value or one per row
  int grad_out_rows, mean;
  float* row_loss;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// -inf stands for "no element": its differences with itself would be NaN.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ bool row_live(const Args& a, int64_t row) {
  if (!a.labels) return true;
  const int64_t y = ld_index(a.labels, a.label_wide, row);
  return y != a.ignore && y >= 0 && y < a.vocab;
}

// Rows that count, over the whole batch (each block for itself: the labels are
// read from cache once per block, which saves a launch).
__device__ int64_t count_live(const Args& a, float* tmp) {
  if (!a.labels) return a.rows;
  int n = 0;
  for (int64_t r = threadIdx.x; r < a.rows; r += blockDim.x) n += row_live(a, r);
  int* const t = reinterpret_cast<int*>(tmp);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off);
  if ((threadIdx.x & 63) == 0) t[threadIdx.x >> 6] = n;
  __syncthreads();
  int64_t s = 0;
  for (unsigned w = 0; w < blockDim.x / 64; ++w) s += t[w];
  __syncthreads();
  return s;
}

// What the first wavefront leaves in LDS about a row's teacher.
struct Teacher {
  float mass;      // sum p
  float rest;      // p_rest
  float z_label;
  int repeated;    // an index occurs twice
  float m, st, s1; // with a tail: maximum and sums over the entries' columns
};

// The compiler would keep every unpacked column of one pass over the registers
// for the next: eight registers a vector more than it has.
template <int DT>
__device__ __forceinline__ void repack(typename Row8<DT>::Raw& r) {
  asm volatile("" : "+v"(r.w));
  if constexpr (DT == kF32) asm volatile("" : "+v"(r.x));
}

// Whether entry k is the first of its index.
__device__ __forceinline__ bool first_of(const int* idx, int k) {
  for (int i = 0; i < k; ++i)
    if (idx[i] == idx[k]) return false;
  return true;
}

template <int DT, int NV>
__global__ __launch_bounds__(1024) void distill_kernel(Args a) {
  using R = Row8<DT>;
  using T = typename R::T;
  constexpr int kN = NV == kStream ? 1 : NV;
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ float red_m[2][kMaxWaves], red_t[2][kMaxWaves], red_1[2][kMaxWaves];
  __shared__ Teacher teach;
  __shared__ float tmp[kMaxWaves];
  // entries: index (-1 absent), logit of the student, p, log p; then a bit per column
  int* const s_idx = reinterpret_cast<int*>(smem);
  float* const s_z = reinterpret_cast<float*>(smem + a.k);
  float* const s_p = reinterpret_cast<float*>(smem + 2 * a.k);
  float* const s_lp = reinterpret_cast<float*>(smem + 3 * a.k);
  uint32_t* const bits = smem + 4 * a.k;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const int64_t v = a.vocab, vecs = (v + 7) / 8;
  const bool tail = a.lse != nullptr;
  const bool hard = a.alpha != 1.f;
  const bool two = hard && a.tau != 1.f;   // a second softmax, at temperature 1
  const float kt = kLog2e / a.tau, k1 = kLog2e;
  for (int64_t w = tid; w < (v + 31) / 32; w += blockDim.x) bits[w] = 0;
  float norm = a.grad_scale;
  if (a.mean) {
    const int64_t live = count_live(a, tmp);
    norm /= (float)(live > 0 ? live : 1);
  }
  __syncthreads();

  // with a tail, the entries' columns leave the row: the first wavefront has them,
  // and what the block sums is the rest, about a maximum of its own
  auto mask = [&](float x[8], int64_t j) {
    if (tail && j < v) {
      const uint32_t top = bits[j >> 5] >> (j & 31);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = top >> e & 1 ? -INFINITY : x[e];
    }
  };

  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const z = (const T*)a.logits + row / a.seq * a.ld_b + row % a.seq * a.ld_s;
    T* const g = a.grad ? (T*)a.grad + row / a.seq * a.gld_b + row % a.seq * a.gld_s : nullptr;
    const int64_t label = a.labels ? ld_index(a.labels, a.label_wide, row) : -1;
    if (!row_live(a, row)) {
      if (tid == 0) a.row_loss[row] = 0.f;
      if (g)
        for (int64_t c = tid; c < vecs; c += blockDim.x) row_st<DT>(g, 8 * c, v, R::zero());
      continue;
    }
    typename R::Raw q[kN];
    if constexpr (NV != kStream) {
#pragma unroll
      for (int c = 0; c < kN; ++c)
        q[c] = row_ld<DT>(z, 8 * ((int64_t)c * blockDim.x + tid), v, R::kNegInf);
    }
    if (wave == 0) {
      // the teacher: entries, their probabilities, the student's logits there
      float m = -INFINITY;
      int again = 0;
      for (int k = lane; k < a.k; k += 64) {
        const int64_t id = ld_index(a.idx, a.idx_wide, row * a.k + k);
        const bool ok = id >= 0 && id < v;
        const float t = ok ? ld_any(a.top, a.top_dtype, row * a.k + k) / a.tau : -INFINITY;
        s_idx[k] = ok ? (int)id : -1;
        s_z[k] = ok ? Elem<DT>::ld(z + id) : 0.f;
        s_lp[k] = t;
        m = fmaxf(m, t);
        if (ok) again |= atomicOr(&bits[id >> 5], 1u << (id & 31)) >> (id & 31) & 1;
      }
      again = __ballot(again) != 0;
      float base, sum = 0.f;
      if (tail) {
        base = a.lse[row];
      } else {
        m = base_of(wave_max(m));
        for (int k = lane; k < a.k; k += 64) sum += exp2_fast((s_lp[k] - m) * kLog2e);
        sum = wave_sum(sum);
        base = m + __log2f(sum) * kLn2;
      }
      float mass = 0.f;
      for (int k = lane; k < a.k; k += 64) {
        const float lp = s_lp[k] - base;
        const float p = s_idx[k] < 0 || (!tail && sum == 0.f) ? 0.f : exp2_fast(lp * kLog2e);
        s_lp[k] = lp;
        s_p[k] = p;
        mass += p;
      }
      mass = wave_sum(mass);
      float mz = -INFINITY, st = 0.f, s1 = 0.f;
      if (tail) {
        for (int k = lane; k < a.k; k += 64)
          if (s_idx[k] >= 0) mz = fmaxf(mz, s_z[k]);
        mz = wave_max(mz);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int k = lane; k < a.k; k += 64) {
          if (s_idx[k] < 0 || (again && !first_of(s_idx, k))) continue;
          const float y = s_z[k] - base_of(mz);
          st += exp2_fast(y * kt);
          if (two) s1 += exp2_fast(y * k1);
        }
        st = wave_sum(st);
        s1 = wave_sum(s1);
      }
      if (lane == 0) {
        teach.rest = tail ? fmaxf(0.f, 1.f - mass) : 0.f;
        teach.mass = mass;
        teach.z_label = hard ? Elem<DT>::ld(z + label) : 0.f;
        teach.repeated = again;
        teach.m = mz, teach.st = st, teach.s1 = s1;
      }
    }
    if (tail) __syncthreads();   // the bits are read below

    // maximum and sums over the thread's columns
    float m = -INFINITY, st = 0.f, s1 = 0.f;
    if constexpr (NV != kStream) {
#pragma unroll
      for (int c = 0; c < kN; ++c) {
        float x[8];
        R::unpack(q[c], x);
        if (tail) {
          mask(x, 8 * ((int64_t)c * blockDim.x + tid));
          q[c] = R::pack(x);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);
        repack<DT>(q[c]);
      }
      const float mb = base_of(m);
#pragma unroll
      for (int c = 0; c < kN; ++c) {
        float x[8];
        R::unpack(q[c], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = x[e] - mb;
          st += exp2_fast(y * kt);
          if (two) s1 += exp2_fast(y * k1);
        }
        repack<DT>(q[c]);
      }
    } else {
      for (int64_t c = tid; c < vecs; c += blockDim.x) {
        float x[8], mc = m;
        R::unpack(row_ld<DT>(z, 8 * c, v, R::kNegInf), x);
        mask(x, 8 * c);
#pragma unroll
        for (int e = 0; e < 8; ++e) mc = fmaxf(mc, x[e]);
        const float mb = base_of(mc);
        const float back = m == -INFINITY ? 0.f : m - mb;
        st *= exp2_fast(back * kt);
        if (two) s1 *= exp2_fast(back * k1);
        m = mc;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = x[e] - mb;
          st += exp2_fast(y * kt);
          if (two) s1 += exp2_fast(y * k1);
        }
      }
    }
    // over the wavefront, then the block: sums are brought to the common maximum.  A
    // maximum of -inf comes with sums of 0, or of NaN where every logit is NaN: both
    // stay as they are
    {
      const float mw = wave_max(m), back = base_of(m) - base_of(mw);
      st = wave_sum(m == -INFINITY ? st : st * exp2_fast(back * kt));
      if (two) s1 = wave_sum(m == -INFINITY ? s1 : s1 * exp2_fast(back * k1));
      if (lane == 0) {
        red_m[turn][wave] = mw;
        red_t[turn][wave] = st;
        red_1[turn][wave] = s1;
      }
    }
    __syncthreads();
    m = -INFINITY;
    for (int w = 0; w < waves; ++w) m = fmaxf(m, red_m[turn][w]);
    const float mb = base_of(m);
    st = s1 = 0.f;
    for (int w = 0; w < waves; ++w) {
      const float mw = red_m[turn][w], back = base_of(mw) - mb;
      const float t = red_t[turn][w], u = red_1[turn][w];
      st += mw == -INFINITY ? t : t * exp2_fast(back * kt);
      if (two) s1 += mw == -INFINITY ? u : u * exp2_fast(back * k1);
    }
    turn ^= 1;
    // the block's maximum and sum (the rest's, with a tail) and the whole row's
    const float sr = st;
    float mz = mb, c_t = 1.f, c_1 = 1.f;
    if (tail) {
      const float mt = teach.m;
      mz = base_of(fmaxf(m, mt));
      c_t = exp2_fast((mb - mz) * kt);
      c_1 = exp2_fast((mb - mz) * k1);
      // an empty side's sum is 0 whatever its factor
      if (m == -INFINITY) c_t = c_1 = 1.f;
      const float back = mt == -INFINITY ? 0.f : base_of(mt) - mz;
      st = st * c_t + teach.st * exp2_fast(back * kt);
      if (two) s1 = s1 * c_1 + teach.s1 * exp2_fast(back * k1);
    }
    if (!two) s1 = st, c_1 = c_t;
    const float log_st = __log2f(st) * kLn2, log_s1 = __log2f(s1) * kLn2;
    const float rest = sr == 0.f ? 0.f : teach.rest;
    const float mass = teach.mass + rest;   // P
    if (wave == 0) {
      float soft = 0.f;
      for (int k = lane; k < a.k; k += 64) {
        const float p = s_p[k];
        if (p != 0.f) soft += p * (s_lp[k] - ((s_z[k] - mz) / a.tau - log_st));
      }
      soft = wave_sum(soft);
      if (rest > 0.f)
        soft += rest * (__log2f(rest) * kLn2 - (__log2f(sr) * kLn2 + (mb - mz) / a.tau - log_st));
      if (lane == 0) {
        float loss = a.alpha * a.tau * a.tau * soft;
        if (hard) loss += (1.f - a.alpha) * (log_s1 - (teach.z_label - mz));
        a.row_loss[row] = loss;
      }
    }
    if (g) {
      const float go = norm * (a.grad_out ? a.grad_out[a.grad_out_rows ? row : 0] : 1.f);
      const float cs = go * a.alpha * a.tau, ch = go * (1.f - a.alpha);
      // factors of e_tau and e_1 (about mz at an entry, about mb elsewhere)
      const float f_top = cs * mass / st, f_top1 = ch / s1;
      const float f_t = f_top * c_t - (rest > 0.f ? cs * rest / sr : 0.f), f_1 = f_top1 * c_1;
      auto grad_of = [&](float x) {
        const float y = x - mb, et = exp2_fast(y * kt);
        float d = f_t * et;
        if (two)
          d += f_1 * exp2_fast(y * k1);
        else if (hard)
          d += f_1 * et;
        return d;
      };
      auto grad8 = [&](const typename R::Raw& raw, int64_t j) {
        float x[8];
        R::unpack(raw, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = grad_of(x[e]);
        row_st<DT>(g, j, v, R::pack(x));
      };
      if constexpr (NV != kStream) {
#pragma unroll
        for (int c = 0; c < kN; ++c) grad8(q[c], 8 * ((int64_t)c * blockDim.x + tid));
      } else {
        for (int64_t c = tid; c < vecs; c += blockDim.x)
          grad8(row_ld<DT>(z, 8 * c, v, R::kNegInf), 8 * c);
      }
      __syncthreads();   // the columns below are written again
      if (wave == 0) {
        for (int k = lane; k < a.k; k += 64) {
          const int id = s_idx[k];
          if (id < 0) continue;
          float p = s_p[k];
          if (teach.repeated) {
            p = 0.f;
            for (int i = 0; i < a.k; ++i) p += s_idx[i] == id ? s_p[i] : 0.f;
          }
          const float y = s_z[k] - mz, et = exp2_fast(y * kt);
          float x = f_top * et - cs * p;
          if (hard) x += f_top1 * (two ? exp2_fast(y * k1) : et) - (id == label ? ch : 0.f);
          Elem<DT>::st(g + id, x);
        }
        if (hard && lane == 0 && !(bits[label >> 5] >> (label & 31) & 1))
          Elem<DT>::st(g + label, grad_of(teach.z_label) - ch);
      }
    }
    if (wave == 0) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (int k = lane; k < a.k; k += 64)
        if (s_idx[k] >= 0) bits[s_idx[k] >> 5] = 0;
    }
    // the first wavefront writes `teach` again for the next row: all have read it
    // before the barrier above, where there is one
    if (!g) __syncthreads();
  }
}

constexpr int kSumThreads = 1024;

// The rows' losses to one: their sum, over the rows that count for a mean.
__global__ __launch_bounds__(kSumThreads) void total_kernel(Args a, float* loss) {
  __shared__ float tmp[kMaxWaves];
  const int64_t live = a.mean ? count_live(a, tmp) : 1;
  float s = 0.f;
  for (int64_t r = threadIdx.x; r < a.rows; r += kSumThreads) s += a.row_loss[r];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x > 0) return;
  s = 0.f;
  for (int w = 0; w < kMaxWaves; ++w) s += tmp[w];
  *loss = s / (float)(live > 0 ? live : 1);
}

// x[row] *= f (one factor, or one per row): nothing is read where it is 1.
template <int DT>
__global__ __launch_bounds__(256) void scale_kernel(void* x, int64_t rows, int64_t v,
                                                    const float* __restrict__ f, int per_row) {
  using R = Row8<DT>;
  using T = typename R::T;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float s = f[per_row ? row : 0];
    if (s == 1.f) continue;
    T* const p = (T*)x + row * v;
    for (int64_t j = 8 * (int64_t)threadIdx.x; j < v; j += 8 * 256) {
      float t[8];
      R::unpack(row_ld<DT>(p, j, v, 0), t);
#pragma unroll
      for (int e = 0; e < 8; ++e) t[e] *= s;
      row_st<DT>(p, j, v, R::pack(t));
    }
  }
}

inline int launched() { return hipGetLastError() == hipSuccess ? kOk : kErrLaunch; }

// Columns up to 32768: four vectors a thread of as few threads as hold the row;
// then eight of 1024 threads; wider rows are read twice.
int vectors(int64_t v, int* threads) {
  const int64_t vecs = (v + 7) / 8;
  *threads = 1024;
  if (vecs <= 256) return *threads = 256, 1;
  if (vecs <= 512) return *threads = 256, 2;
  if (vecs <= 1024) return *threads = 256, 4;
  if (vecs <= 2048) return *threads = 512, 4;
  if (vecs <= 4096) return 4;
  if (vecs <= 8192) return 8;
  return kStream;
}

}  // namespace distill
}  // namespace cpt

using namespace cpt;
using namespace cpt::distill;

extern "C" {

int cpt_distill_topk(int dtype, const void* logits, int64_t rows, int64_t vocab, int64_t seq,
                     int64_t ld_batch, int64_t ld_row, int top_dtype, const void* top_logits,
                     int idx_wide, const void* top_indices, int64_t k, const void* top_lse,
                     int label_wide, const void* labels, int64_t ignore_index, float temperature,
                     float alpha, int reduction, float grad_scale, const void* grad_out,
                     void* row_loss, void* loss, void* grad, int64_t gld_batch, int64_t gld_row,
                     void* stream) {
  if (dtype < kF32 || dtype > kBF16 || top_dtype < kF32 || top_dtype > kBF16) return kErrDType;
  if (rows < 0 || vocab < 1 || k < 0 || !(temperature > 0.f) || reduction < 0 || reduction > 2 ||
      ld_batch < 0 || ld_row < 0 || gld_batch < 0 || gld_row < 0)
    return kErrShape;
  // LDS: 16 bytes an entry and a bit a column
  if (k > kMaxEntries || vocab > kMaxVocab) return kErrTooLarge;
  if (reduction != 2 && !loss) return kErrShape;
  if (alpha != 1.f && !labels && rows > 0) return kErrShape;
  if (rows > 0 && (!logits || !row_loss || seq < 1 || (k > 0 && (!top_logits || !top_indices))))
    return kErrShape;
  const hipStream_t st = (hipStream_t)stream;
  Args a{rows, vocab, logits, seq, ld_batch, ld_row, grad, gld_batch, gld_row, top_logits,
         top_indices, top_dtype, idx_wide, (int)k, (const float*)top_lse, labels, label_wide,
         ignore_index, temperature, alpha, grad_scale, (const float*)grad_out, reduction == 2,
         reduction == 0, (float*)row_loss};
  if (rows > 0) {
    int threads;
    const int nv = vectors(vocab, &threads);
    const int64_t most = 256 * (2048 / threads);   // as many blocks as can run at a time
    const unsigned grid = (unsigned)(rows < most ? rows : most);
    const size_t lds = 16 * (size_t)k + (size_t)(vocab + 31) / 32 * 4;
#define CPT_DISTILL(DT, NV)                                                              \
  do {                                                                                  \
    if (lds > 62 * 1024 &&                                                              \
        hipFuncSetAttribute((const void*)distill_kernel<DT, NV>,                        \
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) \
      return kErrLaunch;                                                                \
    distill_kernel<DT, NV><<<grid, threads, lds, st>>>(a);                              \
  } while (0)
#define CPT_DISTILL_NV(DT)                      \
  switch (nv) {                                 \
    case 1: CPT_DISTILL(DT, 1); break;          \
    case 2: CPT_DISTILL(DT, 2); break;          \
    case 4: CPT_DISTILL(DT, 4); break;          \
    case 8: CPT_DISTILL(DT, 8); break;          \
    default: CPT_DISTILL(DT, kStream); break;   \
  }
    if (dtype == kF32) {
      CPT_DISTILL_NV(kF32)
    } else if (dtype == kF16) {
      CPT_DISTILL_NV(kF16)
    } else {
      CPT_DISTILL_NV(kBF16)
    }
    if (launched() != kOk) return kErrLaunch;
  }
  if (reduction != 2) {
    total_kernel<<<1, kSumThreads, 0, st>>>(a, (float*)loss);
    return launched();
  }
  return kOk;
}

int cpt_scale_rows(int dtype, void* x, int64_t rows, int64_t cols, const void* factor,
                   int per_row, void* stream) {
  if (dtype < kF32 || dtype > kBF16) return kErrDType;
  if (rows < 0 || cols < 0) return kErrShape;
  if (rows == 0 || cols == 0) return kOk;
  if (!x || !factor) return kErrShape;
  const unsigned grid = (unsigned)(rows < 2048 ? rows : 2048);
  const auto kern = dtype == kF32   ? scale_kernel<kF32>
                    : dtype == kF16 ? scale_kernel<kF16>
                                    : scale_kernel<kBF16>;
  kern<<<grid, 256, 0, (hipStream_t)stream>>>(x, rows, cols, (const float*)factor, per_row);
  return launched();
}

}  // extern "C"
