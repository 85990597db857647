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
// Bound by HBM: a row is read once and its gradient written once.  A block holds a
// row in registers between the two (as stored, 16 bytes a vector), so the
// softmax's maximum and sums and the gradient are three passes over registers; of
// rows too wide for them the rest is read again.  The first wavefront reads the
// teacher's entries meanwhile; the gradient of an entry's or the label's column is
// written over the general one after a barrier.  Statistics are fp32, kept as
// (maximum, sum of exponentials): one exchange over the block per row.  With a
// tail the columns outside the entries are summed about their own maximum, so
// q_rest keeps its digits however small it is (a finite logit counts however low it
// lies); where nothing is left outside (all of it -inf), the p_rest term falls away.
// Where the entries hold little, p_rest and q_rest are both near 1 and what counts is
// taken from the entries' shares.
//
// Measured on one MI355X: 8192 rows of 32000 bf16 columns (15% left out, both
// terms, tau 2) 229 us, 4.2 TB/s of rows read and gradients written; a large copy
// reaches 5.0.  Of it the stores are 65 us and the exponentials 15; loading the
// next row ahead of the gradient's stores made it slower (247), as loads then
// wait for stores in order.  Evaluation of 1024 x 32000 fp32: 22 us, 5.1 TB/s.

#include "compact_amd.h"
#include "row_ops.h"

namespace cpt {
namespace distill {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
constexpr int kMaxWaves = 16;
constexpr int kMaxEntries = 2048;
constexpr int64_t kMaxVocab = 1 << 19;
constexpr int kBatch = 2;   // vectors in flight of a row that is read again

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
  float* loss;
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The exponentials are taken in powers of two about a whole number near the
// maximum: 2^(k z - C), C = rint(k max).  The product and difference are one
// fused operation, rounded once, and two bases differ by an exact power of two.
// C stops at 2^28, beyond which its own spacing would count: rows that lie
// there are moved to 0 first.
constexpr float kFar = 268435456.f;
__device__ __forceinline__ float base_of(float m, float k) {
  return rintf(fminf(fmaxf(m * k, -kFar), kFar));
}

// 1 / x to fp32's last place (one Newton step from the instruction's estimate)
// in three instructions, where a correctly rounded division takes ten.
__device__ __forceinline__ float inverse(float x) {
  const float r = __builtin_amdgcn_rcpf(x);
  return fmaf(r, fmaf(-x, r, 1.f), r);
}

__device__ __forceinline__ bool live_label(const Args& a, int64_t y) {
  return y != a.ignore && y >= 0 && y < a.vocab;
}

// A value that all lanes share, in a scalar register.
__device__ __forceinline__ float uniform(float x) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}

// Rows that count, over the whole batch, by each block for itself: the labels are read
// from cache once per block.  That costs no more than a launch where rows are wide or
// few (8192 x 32000 bf16: mean 223 us, sum 219), but grows with rows times blocks:
// 8192 x 1024 34 and 20 us, 100000 x 1024 373 and 226.
__device__ __forceinline__ int64_t count_live(const Args& a, float* tmp) {
  if (!a.labels) return a.rows;
  int n = 0;
  constexpr int kAhead = 8;
  for (int64_t r = threadIdx.x; r < a.rows; r += kAhead * (int64_t)blockDim.x) {
    int64_t y[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t at = r + i * (int64_t)blockDim.x;
      y[i] = at < a.rows ? ld_index(a.labels, a.label_wide, at) : -1;
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) n += live_label(a, y[i]);
  }
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

// A teacher's entry as it is stored: the words of its index and of its logit.
struct Entry {
  uint32_t index, index_high;
  uint16_t low, high;
  __device__ __forceinline__ int id(uint32_t vocab, int wide) const {
    return (wide ? index_high == 0 : true) && index < vocab ? (int)index : -1;
  }
  __device__ __forceinline__ float logit(int dt) const {
    if (dt == kF32) return __uint_as_float((uint32_t)high << 16 | low);
    return dt == kF16 ? f16_bits_to_f32(low) : bf16_to_f32(low);
  }
};

// Whether entry k is the first of its index.
__device__ __forceinline__ bool first_of(const int* idx, int k) {
  for (int i = 0; i < k; ++i)
    if (idx[i] == idx[k]) return false;
  return true;
}

// Sum and maximum over 16 lanes (one value a wavefront of the block), in all.
__device__ __forceinline__ float row16_sum(float x) {
  x += dpp<0x111, 0xF>(0.f, x);
  x += dpp<0x112, 0xF>(0.f, x);
  x += dpp<0x114, 0xF>(0.f, x);
  x += dpp<0x118, 0xF>(0.f, x);
  return lane63(x);
}
__device__ __forceinline__ float row16_max(float x) {
  x = fmaxf(x, dpp<0x111, 0xF>(x, x));
  x = fmaxf(x, dpp<0x112, 0xF>(x, x));
  x = fmaxf(x, dpp<0x114, 0xF>(x, x));
  x = fmaxf(x, dpp<0x118, 0xF>(x, x));
  return lane63(x);
}

// POW: the softmax at temperature 1 from the one at tau.  0: not wanted, or the
// same (tau = 1); 1: exponentials of its own; 2: tau = 2, their squares.
template <int DT, int NV, int POW, bool GRAD, int THREADS, int WAVES>
__global__ __launch_bounds__(THREADS, WAVES) void distill_kernel(Args a) {
  using R = Row8<DT>;
  using T = typename R::T;
  using Raw = typename R::Raw;
  constexpr uint32_t kBytes = 8 * sizeof(T);
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
  const uint32_t tid = threadIdx.x;
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // whole vectors; the ragged end, one column a thread
  const uint32_t v = (uint32_t)a.vocab, vecs = v / 8, ragged = v & 7;
  const bool tail = a.lse != nullptr;
  const bool hard = a.alpha != 1.f;
  const float kt = kLog2e / a.tau, k1 = kLog2e;
  // well before a base stops, at the temperature or at temperature 1
  const uint32_t far_from =
      __float_as_uint(uniform(0.5f * kFar / (POW == 1 ? fmaxf(kt, k1) : kt)));
  for (uint32_t w = tid; w < (v + 31) / 32; w += THREADS) bits[w] = 0;
  if (tid < 2 * kMaxWaves && tid % kMaxWaves >= THREADS / 64) {   // wavefronts there are not
    red_m[tid / kMaxWaves][tid % kMaxWaves] = -INFINITY;
    red_t[tid / kMaxWaves][tid % kMaxWaves] = red_1[tid / kMaxWaves][tid % kMaxWaves] = 0.f;
  }
  float norm = a.grad_scale;
  if (a.mean) {
    const int64_t live = count_live(a, tmp);
    norm /= (float)(live > 0 ? live : 1);
    if (blockIdx.x == 0 && tid == 0) *a.loss = (float)(live > 0 ? live : 1);   // for the total
  }
  __syncthreads();

  const auto offset = [&](int64_t r, int64_t ld_b, int64_t ld_s) {
    if (a.seq >= a.rows) return r * ld_s * (int64_t)sizeof(T);   // one batch
    const uint32_t rb = (uint32_t)r / (uint32_t)a.seq, rs = (uint32_t)r - rb * (uint32_t)a.seq;
    return (rb * ld_b + rs * ld_s) * (int64_t)sizeof(T);
  };
  const auto label_of = [&](int64_t r) {
    return a.labels && r < a.rows ? ld_index(a.labels, a.label_wide, r) : -1;
  };

  int turn = 0;
  int64_t next_label = label_of(blockIdx.x);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const char* const z = (const char*)a.logits + offset(row, a.ld_b, a.ld_s);
    char* const g = GRAD ? (char*)a.grad + offset(row, a.gld_b, a.gld_s) : nullptr;
    const auto elem = [&](int64_t j) { return Elem<DT>::ld((const T*)z + j); };
    const auto vec8 = [&](uint32_t vec) { return R::ld((const T*)(z + vec * kBytes)); };
    const int64_t label = next_label;
    if (a.labels && !live_label(a, label)) {
      next_label = label_of(row + gridDim.x);
      if (tid == 0) a.row_loss[row] = 0.f;
      if (GRAD) {
        for (uint32_t c = tid; c < vecs; c += THREADS) R::st((T*)(g + c * kBytes), R::zero());
        if (tid < ragged) Elem<DT>::st((T*)g + vecs * 8 + tid, 0.f);
      }
      continue;
    }
    // Loads come back in order: the first entries', needed first, lead.  They are
    // loaded as words of either width without a branch, which would be waited for.
    const auto load_entry = [&](int k) {
      const int64_t i = row * a.k + k;
      const int64_t w = i << a.idx_wide, h = i << (a.top_dtype == kF32);
      const uint32_t* const idx = (const uint32_t*)a.idx;
      const uint16_t* const top = (const uint16_t*)a.top;
      return Entry{idx[w], idx[w + a.idx_wide], top[h], top[h + (a.top_dtype == kF32)]};
    };
    Entry first{};
    if (wave == 0 && a.k > 0) first = load_entry(min(lane, a.k - 1));
    Raw q[NV > 0 ? NV : 1];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      q[c] = R::fill(R::kNegInf);
      if (c * THREADS + tid < vecs) q[c] = vec8(c * THREADS + tid);
    }
    float xr = tid < ragged ? elem(vecs * 8 + tid) : -INFINITY;
    next_label = label_of(row + gridDim.x);
    if (wave == 0) {
      // the teacher: entries, their probabilities, the student's logits there
      float m = -INFINITY;
      int again = 0;
      for (int k = lane; k < a.k; k += 64) {
        if (k >= 64) first = load_entry(k);
        const int e_id = first.id(v, a.idx_wide);
        const float t = e_id >= 0 ? first.logit(a.top_dtype) : -INFINITY;
        s_idx[k] = e_id;
        s_z[k] = e_id >= 0 ? elem(e_id) : 0.f;
        s_lp[k] = t;
        m = fmaxf(m, t);
        if (e_id >= 0)
          again |= atomicOr(&bits[e_id >> 5], 1u << (e_id & 31)) >> (e_id & 31) & 1;
      }
      again = __ballot(again) != 0;
      // log p = (t - base) / tau - ls: the difference of two logits rounded once, so that
      // log p is good about 0 however large the logits are
      float base, ls = 0.f, sum = 0.f;
      if (tail) {
        base = a.lse[row];   // at the temperature
      } else {
        m = wave_max(m);
        m = m == -INFINITY ? 0.f : m;
        for (int k = lane; k < a.k; k += 64) sum += exp2_fast((s_lp[k] - m) * kt);
        sum = wave_sum(sum);
        base = m, ls = __log2f(sum) * kLn2;
      }
      float mass = 0.f;
      for (int k = lane; k < a.k; k += 64) {
        const float t = s_lp[k];
        const float lp = (tail ? fmaf(-base, a.tau, t) : t - base) / a.tau - ls;
        const float p = s_idx[k] < 0 || (!tail && sum == 0.f) ? 0.f : exp2_fast(lp * kLog2e);
        s_lp[k] = lp;
        s_p[k] = p;
        mass += p;
      }
      mass = wave_sum(mass);
      if (lane == 0) {
        teach.rest = tail ? fmaxf(0.f, 1.f - mass) : 0.f;
        teach.mass = mass;
        teach.z_label = hard ? elem(label) : 0.f;
        teach.repeated = again;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (tail) {
      // the entries' columns leave the row: the first wavefront has them, and what
      // the block sums is the rest, about a maximum of its own
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const uint32_t vec = c * THREADS + tid;
        const uint32_t top = vec < vecs ? bits[vec >> 2] >> (8 * (vec & 3)) & 255 : 0;
        if (top) R::mask(q[c], top, R::kNegInf);
      }
      if (tid < ragged && bits[vecs >> 2] >> (8 * (vecs & 3) + tid) & 1) xr = -INFINITY;
    }
    // Columns past the registers are read again, kBatch vectors at a time: with a
    // tail without the entries', and -inf past the row's end.
    float shift = 0.f, below = 0.f;   // taken off the entries and the label; off the columns
    const auto load_batch = [&](uint32_t first, Raw (&r)[kBatch]) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) r[i] = vec8(min(first + i * THREADS, vecs - 1));
    };
    const auto unpack_again = [&](uint32_t vec, Raw& r, float x[8]) {
      if (tail) {
        const uint32_t at = min(vec, vecs - 1);
        const uint32_t top = bits[at >> 2] >> (8 * (at & 3)) & 255;
        if (top) R::mask(r, top, R::kNegInf);
      }
      if (vec >= vecs) r = R::fill(R::kNegInf);
      R::unpack(r, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] -= below;
    };

    float m, st, s1, c_t, c_1, sr;
    for (bool moved = false;; moved = true) {
      // maximum and sums over the thread's columns
      m = xr;
      st = s1 = 0.f;
      float ct = 0.f, c1 = 0.f;
      const auto add = [&](float x, float& to_t, float& to_1) {
        const float et = exp2_fast(fmaf(x, kt, -ct));
        to_t += et;
        if (POW == 1) to_1 += exp2_fast(fmaf(x, k1, -c1));
        if (POW == 2) to_1 = fmaf(et, et, to_1);
      };
      // a vector's eight first by themselves: the chain of the widest row (65536 vectors)
      // has 137 terms, not 1024
      const auto add_vec = [&](const float x[8]) {
        float vt = 0.f, v1 = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) add(x[e], vt, v1);
        st += vt;
        if (POW) s1 += v1;
      };
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        float x[8];
        R::unpack(q[c], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);
        repack<DT>(q[c]);
      }
      ct = base_of(m, kt), c1 = base_of(m, k1);
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        float x[8];
        R::unpack(q[c], x);
        add_vec(x);
        repack<DT>(q[c]);
      }
      for (uint32_t first = NV * THREADS + tid; first < vecs; first += kBatch * THREADS) {
        Raw r[kBatch];
        load_batch(first, r);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          float x[8], mc = m;
          unpack_again(first + i * THREADS, r[i], x);
#pragma unroll
          for (int e = 0; e < 8; ++e) mc = fmaxf(mc, x[e]);
          if (mc > m) {
            const float nt = base_of(mc, kt), n1 = base_of(mc, k1);
            st *= exp2_fast(ct - nt);
            if (POW == 1) s1 *= exp2_fast(c1 - n1);
            if (POW == 2) s1 *= exp2_fast(2.f * (ct - nt));
            m = mc, ct = nt, c1 = n1;
          }
          add_vec(x);
        }
      }
      add(xr, st, s1);
      // over the wavefront, then the block: sums are brought to the common base
      const float mw = wave_max(m), back = exp2_fast(ct - base_of(mw, kt));
      st = wave_sum(st * back);
      if (POW == 1) s1 = wave_sum(s1 * exp2_fast(c1 - base_of(mw, k1)));
      if (POW == 2) s1 = wave_sum(s1 * back * back);
      if (lane == 0) {
        red_m[turn][wave] = mw;
        red_t[turn][wave] = st;
        if (POW) red_1[turn][wave] = s1;
      }
      if (tail && wave == 0) {
        // the same over the entries' columns, each once
        float me = -INFINITY, te = 0.f, e1 = 0.f;
        for (int k = lane; k < a.k; k += 64)
          if (s_idx[k] >= 0) me = fmaxf(me, s_z[k] - shift);
        me = wave_max(me);
        for (int k = lane; k < a.k; k += 64) {
          if (s_idx[k] < 0 || (teach.repeated && !first_of(s_idx, k))) continue;
          const float et = exp2_fast(fmaf(s_z[k] - shift, kt, -base_of(me, kt)));
          te += et;
          if (POW == 1) e1 += exp2_fast(fmaf(s_z[k] - shift, k1, -base_of(me, k1)));
          if (POW == 2) e1 = fmaf(et, et, e1);
        }
        te = wave_sum(te);
        e1 = wave_sum(e1);
        if (lane == 0) teach.m = me, teach.st = te, teach.s1 = e1;
      }
      __syncthreads();
      {
        const int w = lane & (kMaxWaves - 1);
        const float mw = red_m[turn][w];
        m = row16_max(mw);
        c_t = base_of(m, kt), c_1 = POW == 2 ? 2.f * c_t : POW == 1 ? base_of(m, k1) : 0.f;
        const float back = exp2_fast(base_of(mw, kt) - c_t);
        st = row16_sum(red_t[turn][w] * back);
        if (POW == 1) s1 = row16_sum(red_1[turn][w] * exp2_fast(base_of(mw, k1) - c_1));
        if (POW == 2) s1 = row16_sum(red_1[turn][w] * back * back);
      }
      turn ^= 1;
      // values that are far (masked by the type's lowest) are moved to 0 and summed again:
      // a row of nothing else, and with a tail what lies outside the entries, each by its
      // own maximum
      const auto far = [&](float x) {   // in scalar registers, as all share x
        const uint32_t size = __float_as_uint(uniform(x)) & 0x7FFFFFFFu;
        return size - far_from < 0x7F800000u - far_from;   // and finite
      };
      if (moved || !(far(m) || (tail && far(fmaxf(m, teach.m))))) break;
      const float m_row = tail ? fmaxf(m, teach.m) : m;
      shift = uniform(fabsf(m_row) == INFINITY ? 0.f : m_row);
      below = uniform(m == -INFINITY ? shift : m);
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        float x[8];
        R::unpack(q[c], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] -= below;
        q[c] = R::pack(x);
      }
      xr -= below;
      __syncthreads();   // `teach` is written again
    }
    // c_t, c_1: the base of the block's sums.  sr: its sum (the rest's, with a tail);
    // st, s1: the whole row's, about b_t and b_1, u_t and u_1 apart; `apart` is how far
    // the columns were moved more than the entries
    sr = st;
    float b_t = c_t, b_1 = c_1, u_t = 1.f, u_1 = 1.f;
    const float apart = below - shift;
    float q_top = 0.f;   // the student's share of the entries' columns, with a tail
    if (tail) {
      const float et = base_of(teach.m, kt), e1 = POW == 2 ? 2.f * et : base_of(teach.m, k1);
      const float r_t = fmaf(apart, kt, c_t), r_1 = fmaf(apart, k1, c_1);
      b_t = fmaxf(r_t, et), b_1 = fmaxf(r_1, e1);
      u_t = exp2_fast(r_t - b_t), u_1 = exp2_fast(r_1 - b_1);
      q_top = teach.st * exp2_fast(et - b_t);
      st = st * u_t + q_top;
      q_top *= inverse(st);
      if (POW) s1 = s1 * u_1 + teach.s1 * exp2_fast(e1 - b_1);
    }
    if (!POW) s1 = st, b_1 = b_t, u_1 = u_t;
    if (st == INFINITY) st = s1 = NAN;   // +inf among the logits
    const float rest = sr == 0.f ? 0.f : teach.rest;
    const float mass = teach.mass + rest;   // P
    // Of a large rest, two shares near 1 (many classes, a high temperature), only the
    // difference counts, and it is taken between the entries' shares instead:
    //   log(rest / q_rest) = log(1 + (q_top - p_top) / (1 - q_top))
    //   P q_rest - rest = p_top - P q_top
    const bool large_rest = tail && q_top < 0.5f && teach.mass < 0.5f;
    if (wave == 0) {
      const float l_t = __log2f(st), l_1 = __log2f(s1);   // of the row's sums, less b_t and b_1
      float soft = 0.f;
      for (int k = lane; k < a.k; k += 64) {
        const float p = s_p[k];
        if (p != 0.f) soft += p * (s_lp[k] - kLn2 * (fmaf(s_z[k] - shift, kt, -b_t) - l_t));
      }
      soft = wave_sum(soft);
      if (rest > 0.f)
        soft += rest * (large_rest ? log1pf((q_top - teach.mass) / (1.f - q_top))
                                   : kLn2 * (__log2f(rest) - (__log2f(sr) - l_t + (c_t - b_t))) -
                                         apart * (kt * kLn2));
      if (lane == 0) {
        float loss = a.alpha * a.tau * a.tau * soft;
        if (hard) loss += (1.f - a.alpha) * kLn2 * (l_1 - fmaf(teach.z_label - shift, k1, -b_1));
        a.row_loss[row] = loss;
      }
    }
    if constexpr (GRAD) {
      const float go = norm * (a.grad_out ? a.grad_out[a.grad_out_rows ? row : 0] : 1.f);
      const float cs = go * a.alpha * a.tau, ch = go * (1.f - a.alpha);
      // factors of the exponentials: about the row's base at an entry, the block's elsewhere
      const float f_top = cs * mass * inverse(st), f_top1 = ch * inverse(s1);
      float f_t = f_top * u_t, f_1 = f_top1 * u_1;
      if (rest > 0.f)
        f_t = large_rest ? cs * (teach.mass - mass * q_top) * inverse(sr)
                         : f_t - cs * rest * inverse(sr);
      if (!POW) f_t += f_1;   // one softmax for both terms (f_1 is 0 without labels' term)
      const auto grad_of = [&](float x) {
        const float et = exp2_fast(fmaf(x, kt, -c_t));
        if (POW == 1) return fmaf(f_t, et, f_1 * exp2_fast(fmaf(x, k1, -c_1)));
        if (POW == 2) return et * fmaf(f_1, et, f_t);
        return f_t * et;
      };
#pragma unroll
      for (int c = 0; c < NV; ++c) {
        const uint32_t vec = c * THREADS + tid;
        float x[8];
        R::unpack(q[c], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = grad_of(x[e]);
        if (vec < vecs) R::st((T*)(g + vec * kBytes), R::pack(x));
      }
      for (uint32_t first = NV * THREADS + tid; first < vecs; first += kBatch * THREADS) {
        Raw r[kBatch];
        load_batch(first, r);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const uint32_t vec = first + i * THREADS;
          float x[8];
          unpack_again(vec, r[i], x);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = grad_of(x[e]);
          if (vec < vecs) R::st((T*)(g + vec * kBytes), R::pack(x));
        }
      }
      if (tid < ragged) Elem<DT>::st((T*)g + vecs * 8 + tid, grad_of(xr));
      __syncthreads();   // the columns below are written again
      if (wave == 0) {
        const auto top_of = [&](float x) {
          const float et = exp2_fast(fmaf(x, kt, -b_t));
          if (POW == 1) return fmaf(f_top, et, f_top1 * exp2_fast(fmaf(x, k1, -b_1)));
          if (POW == 2) return et * fmaf(f_top1, et, f_top);
          return (f_top + f_top1) * et;
        };
        for (int k = lane; k < a.k; k += 64) {
          const int id = s_idx[k];
          if (id < 0) continue;
          float p = s_p[k];
          if (teach.repeated) {
            p = 0.f;
            for (int i = 0; i < a.k; ++i) p += s_idx[i] == id ? s_p[i] : 0.f;
          }
          Elem<DT>::st((T*)g + id, top_of(s_z[k] - shift) - cs * p - (id == label ? ch : 0.f));
        }
        if (hard && lane == 0 && !(bits[label >> 5] >> (label & 31) & 1))
          Elem<DT>::st((T*)g + label, grad_of(teach.z_label - below) - ch);
      }
    }
    if (wave == 0) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      for (int k = lane; k < a.k; k += 64)
        if (s_idx[k] >= 0) bits[s_idx[k] >> 5] = 0;
    }
    // the first wavefront writes `teach` again for the next row: all have read it
    // before the barrier above, where there is one
    if (!GRAD) __syncthreads();
  }
}

constexpr int kSumThreads = 1024;

// The rows' losses to one: their sum, or over the count that stands in its place.
__global__ __launch_bounds__(kSumThreads) void total_kernel(Args a) {
  __shared__ float tmp[kMaxWaves];
  const float count = a.mean && a.rows > 0 ? *a.loss : 1.f;
  float s = 0.f;
#pragma unroll 8
  for (int64_t r = threadIdx.x; r < a.rows; r += kSumThreads) s += a.row_loss[r];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x > 0) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < kMaxWaves; ++w) s += tmp[w];
  *a.loss = s / count;
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

// Launches one shape of block.  As many blocks as can run at a time go over the rows.
template <int DT, int NV, bool GRAD, int THREADS, int WAVES>
int launch(const Args& a, hipStream_t st) {
  const bool two = a.alpha != 1.f && a.tau != 1.f;
  const int64_t most = 256 * (WAVES * 256 / THREADS);
  const unsigned grid = (unsigned)(a.rows < most ? a.rows : most);
  const size_t lds = 16 * (size_t)a.k + (size_t)(a.vocab + 31) / 32 * 4;
  const auto kern = !two           ? distill_kernel<DT, NV, 0, GRAD, THREADS, WAVES>
                    : a.tau == 2.f ? distill_kernel<DT, NV, 2, GRAD, THREADS, WAVES>
                                   : distill_kernel<DT, NV, 1, GRAD, THREADS, WAVES>;
  if (lds > 62 * 1024 &&
      hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                          (int)lds) != hipSuccess)
    return kErrLaunch;
  kern<<<grid, THREADS, lds, st>>>(a);
  return launched();
}

// Threads of a row's block and the vectors each keeps of it for the gradient: 32
// registers of the row's own type, and as few threads as hold it that way, so that
// several rows are in flight on a CU and few wavefronts wait for each other (8000
// rows of 8000 bf16 columns: 69 us with 128 threads, 102 with 256 and half the
// vectors).  Rows past 32768 columns do not fit; a few more registers each then pay
// (1500 x 50000 fp32 131 us, 139 with 4 vectors; 1531 x 50021 bf16 84, 86 with 8),
// and the rest is read twice.  Without a gradient nothing is kept: one pass.
template <int DT>
int launch(const Args& a, hipStream_t st) {
  const int64_t vecs = a.vocab / 8;
  if (!a.grad)
    return vecs <= 1024 ? launch<DT, 0, false, 256, 8>(a, st)
                        : launch<DT, 0, false, 512, 8>(a, st);
  if (vecs <= 128) return launch<DT, 1, true, 128, 6>(a, st);
  if (vecs <= 256) return launch<DT, 2, true, 128, 6>(a, st);
  if (vecs <= 512) return launch<DT, 4, true, 128, 4>(a, st);
  constexpr int kFull = DT == kF32 ? 4 : 8, kWide = DT == kF32 ? 2 : 1;
  if (vecs <= 1024) return launch<DT, kFull, true, 128 * kWide, 4>(a, st);
  if (vecs <= 2048) return launch<DT, kFull, true, 256 * kWide, 4>(a, st);
  if (vecs <= 4096) return launch<DT, kFull, true, 512 * kWide, 4>(a, st);
  return launch<DT, kFull + 2, true, 512 * kWide, 4>(a, st);
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
  if (k > kMaxEntries || vocab > kMaxVocab || rows > 0x7FFFFFFF) return kErrTooLarge;
  if (reduction != 2 && !loss) return kErrShape;
  if (alpha != 1.f && !labels && rows > 0) return kErrShape;
  if (rows > 0 && (!logits || !row_loss || seq < 1 || (k > 0 && (!top_logits || !top_indices))))
    return kErrShape;
  const hipStream_t st = (hipStream_t)stream;
  Args a{rows, vocab, logits, seq, ld_batch, ld_row, grad, gld_batch, gld_row, top_logits,
         top_indices, top_dtype, idx_wide != 0, (int)k, (const float*)top_lse, labels, label_wide,
         ignore_index, temperature, alpha, grad_scale, (const float*)grad_out, reduction == 2,
         reduction == 0, (float*)row_loss, (float*)loss};
  if (rows > 0) {
    const int rc = dtype == kF32   ? launch<kF32>(a, st)
                   : dtype == kF16 ? launch<kF16>(a, st)
                                   : launch<kBF16>(a, st);
    if (rc != kOk) return rc;
  }
  if (reduction != 2) {
    total_kernel<<<1, kSumThreads, 0, st>>>(a);
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
