// An AdamW step over many tensors in few launches, with the gradients' global norm
// and clipping, and moments in fp32 or in 8 bits.
//
//   g <- g * grad_scale * min(1, max_norm / (norm + 1e-6)),  norm over all tensors
//   m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2
//   p <- p - lr wd p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
// A norm that is not finite leaves everything as it was.  Each product and sum of
// the moments is rounded by itself (no fused multiply-add), so that they are the
// same bits wherever they are computed.
//
// 8-bit moments: blocks of 128 elements share a power of two 2^s, kept as the byte
// s + 134 (255: the block is NaN).  A second moment is five bits E and three bits M
// and stands for M 2^s (E = 0) or (8 + M) 2^(E - 1 + s): a float's own layout with
// fewer bits, so that encoding is a shift of the scaled float's.  A first moment has
// a sign and a four-bit E.  s puts the block's largest value into the top binade
// (one that would round past it stays at 15/16 of its end).  An average that moves
// by a thousandth a step would never leave a code of three bits by rounding to
// nearest, so values are rounded up or down in proportion, by 16 bits of a hash of
// (seed, step, tensor, element); a nonzero second moment is never rounded to zero,
// where m / (sqrt(v) + eps) would be large.
//
// Bound: HBM, 22 bytes an element with 16-bit parameters and gradients and fp32
// moments, 28 with an fp32 copy of the parameters, 10 with 8-bit moments.  The
// tensors' pointers are kernel arguments, up to 90 a launch: no table to upload or keep.  A
// launch has one step number on the host: tensors whose numbers change from one to the next
// take one each (counts on the device do not divide a call).
//
// Measured on one MI355X, a trace's mean of 12: 1.1 G bf16 parameters with an fp32 copy 5750
// us (5.4 TB/s) and 430 for the norm; 371 M with 8-bit moments 780 (4.8; the least 741),
// their values 394; 31.6 M in 320 tensors 136 in four launches (5.1) and 27 for the norm;
// 0.2 M fp32 4.7.

#include <algorithm>
#include <cmath>

#include "compact_amd.h"
#include "row_ops.h"

namespace cpt {
namespace adamw {

constexpr int kThreads = 256;
constexpr int kArgBytes = 4096;       // of a kernel
constexpr int kPass = kThreads * 8;   // elements a block has in registers at a time
constexpr int kBlockLog = 7;          // 128 elements share a scale
constexpr int kScaleBias = 134;

// Whether a step clips and goes ahead, decided on the device.
struct Control {
  float clip;
  int skip;
};
// A tensor's bias corrections 1 / (1 - b^t) and its dither's key, likewise.
struct DeviceStep {
  float inv1, inv2;
  uint32_t key;
};

// A tensor of a launch; what a kind of step has none of takes no room, so that one
// launch has as many tensors as fit (90 with fp32 moments alone).
template <bool BITS8>
struct ScaleAddress {};
template <>
struct ScaleAddress<true> {
  uint8_t* ms;
  uint8_t* vs;
};
template <bool MASTER>
struct MasterAddress {};
template <>
struct MasterAddress<true> {
  float* master;
};
template <bool BITS8, bool MASTER>
struct Tensor : ScaleAddress<BITS8>, MasterAddress<MASTER> {
  void* p;
  const void* g;
  void* m;
  void* v;
  int64_t n;
};
struct StepCommon {
  const Control* control;         // null: no clipping, or
  const double* partial;          // the squares' sums, from which each block decides itself
  float* norm;
  int partials;
  float max_norm;
  const DeviceStep* device_step;  // null: inv1, inv2, and keys of seed and step
  const float* lr_device;         // null: lr
  int64_t chunk;                  // elements a block, a multiple of 2048
  int count, base;                // tensors, and the first one's place in the call
  uint32_t seed, step;
  float lr, wd, b1, b2, c1, c2, eps, grad_scale, inv1, inv2;   // c = 1 - b
};
template <bool BITS8, bool MASTER>
struct StepArgs : StepCommon {
  static constexpr int kTensors =
      (kArgBytes - (int)sizeof(StepCommon) - 16) / ((int)sizeof(Tensor<BITS8, MASTER>) + 4);
  int first[kTensors];            // first block
  Tensor<BITS8, MASTER> t[kTensors];
};

__host__ __device__ __forceinline__ uint32_t mix(uint32_t h) {
  h ^= h >> 16;
  h *= 0x243F6A89u;
  h ^= h >> 15;
  h *= 0x1E3779B1u;
  return h ^ (h >> 16);
}
__host__ __device__ __forceinline__ uint32_t tensor_key(uint32_t seed, uint32_t step, uint32_t i) {
  return mix(seed * 0x37E15163u + step * 0x6A09E667u + i * 0x3C6EF373u);
}

// The tensor that a block works on: the last whose first block is not past it.  All
// loads before the first wait.
template <int MOST>
__device__ __forceinline__ int find_tensor(const int (&first)[MOST], int count, int block) {
  constexpr int kLoads = (MOST + 63) / 64;
  const int lane = threadIdx.x & 63;
  int v[kLoads], n = 0;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) v[i] = first[min(i * 64 + lane, count - 1)];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) n += __popcll(__ballot(i * 64 + lane < count && v[i] <= block));
  return __builtin_amdgcn_readfirstlane(n - 1);
}

// Rounded by themselves, whatever they are inlined into.
__device__ __forceinline__ float mul(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}
__device__ __forceinline__ float add(float a, float b) {
#pragma clang fp contract(off)
  return a + b;
}

// Eight elements [i, i + 8) of a tensor of n: whole vectors unless they end past it.
template <int DT>
__device__ __forceinline__ typename Row8<DT>::Raw ld8(const void* p, int64_t i, int64_t n) {
  const auto* q = (const typename Row8<DT>::T*)p + i;
  return i + 8 <= n ? Row8<DT>::ld(q) : Row8<DT>::ld_n(q, (int)(n - i), 0);
}
template <int DT>
__device__ __forceinline__ void st8(void* p, int64_t i, int64_t n, const float v[8]) {
  auto* q = (typename Row8<DT>::T*)p + i;
  if (i + 8 <= n)
    Row8<DT>::st(q, Row8<DT>::pack(v));
  else
    Row8<DT>::st_n(q, Row8<DT>::pack(v), (int)(n - i));
}
typedef uint32_t u32x2_a1 __attribute__((ext_vector_type(2), aligned(1)));
__device__ __forceinline__ void ld_codes(const void* p, int64_t i, int64_t n, uint32_t c[2]) {
  const uint8_t* q = (const uint8_t*)p + i;
  if (i + 8 <= n) {
    const u32x2_a1 w = *reinterpret_cast<const u32x2_a1*>(q);
    c[0] = w.x, c[1] = w.y;
  } else {
    c[0] = c[1] = 0;
    for (int j = 0; j < (int)(n - i); ++j) c[j >> 2] |= (uint32_t)q[j] << (8 * (j & 3));
  }
}
__device__ __forceinline__ void st_codes(void* p, int64_t i, int64_t n, const uint32_t c[2]) {
  uint8_t* q = (uint8_t*)p + i;
  if (i + 8 <= n) {
    *reinterpret_cast<u32x2_a1*>(q) = u32x2_a1{c[0], c[1]};
  } else {
    for (int j = 0; j < (int)(n - i); ++j) q[j] = (uint8_t)(c[j >> 2] >> (8 * (j & 3)));
  }
}

// A code's value: its bits in a float's place, times 2^(129 + s).
template <bool SIGNED>
__device__ __forceinline__ float decode(uint32_t code, int scale) {
  const float y = __builtin_ldexpf(__uint_as_float((SIGNED ? code & 127 : code) << 20),
                                   scale - (kScaleBias - 129));
  const float v = SIGNED ? __uint_as_float(__float_as_uint(y) | (code & 128) << 24) : y;
  return scale == 255 ? __uint_as_float(0x7FC00000u) : v;
}
template <bool SIGNED>
__device__ __forceinline__ uint32_t encode(float x, int s, uint32_t dither16) {
  const uint32_t y = __float_as_uint(__builtin_ldexpf(fabsf(x), -s - 129));
  uint32_t code = (y + (dither16 << 4)) >> 20;
  if (SIGNED) return min(code, 127u) | (__float_as_uint(x) >> 24 & 128u);
  code = min(code, 255u);
  return x > 0.f ? max(code, 1u) : code;
}
// The largest of 16 lanes' values, in each of them.
__device__ __forceinline__ uint32_t max16(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xF, 0xF, false));  // row_ror
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xF, 0xF, false));
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xF, 0xF, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xF, 0xF, false));
}
// s of a block whose largest magnitude has these bits; 2^(s + top) is its binade's start.
__device__ __forceinline__ int block_scale(uint32_t bits, int top) {
  return max((int)(bits >> 23) - 127 - top, 1 - kScaleBias);
}

__device__ __forceinline__ Control decide(float norm, float max_norm) {
  return Control{fminf(1.f, max_norm / add(norm, 1e-6f)), !(norm < INFINITY)};
}
// The root of n numbers' sum, in every thread of a block of THREADS.
template <int THREADS>
__device__ __forceinline__ float root_of_sum(const double* p, int n) {
  __shared__ double part[THREADS / 64];
  double s = 0;
  for (int i = threadIdx.x; i < n; i += THREADS) s += p[i];
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  double t = 0;
  for (int i = 0; i < THREADS / 64; ++i) t += part[i];
  return (float)sqrt(t);
}

// m / (sqrt(v) + eps).  Beside moments of three bits the hardware's root and reciprocal,
// good to one unit in the last place (and a root of a denormal to nothing) are exact
// enough; the IEEE ones are 25 instructions of about 80 an element there.
template <bool BITS8>
__device__ __forceinline__ float quotient(float m, float v, float eps) {
  if (!BITS8 || eps < 1e-18f) return m / (sqrtf(v) + eps);
  return m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) + eps);
}

// PD: the parameters' type, GD: the gradients', BITS8: moments in 8 bits, MASTER: an
// fp32 copy of the parameters that is stepped in their place.
template <int PD, int GD, bool BITS8, bool MASTER>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const StepArgs<BITS8, MASTER> A) {
  const int ti = find_tensor(A.first, A.count, blockIdx.x);
  const auto& T = A.t[ti];
  float clip = 1.f;
  if (A.control || A.partial) {
    Control c;
    if (A.partial) {
      const float norm = root_of_sum<kThreads>(A.partial, A.partials);
      if (blockIdx.x == 0 && threadIdx.x == 0) *A.norm = norm;
      c = decide(norm, A.max_norm);
    } else {
      c = *A.control;
    }
    if (c.skip) return;
    clip = c.clip;
  }
  float inv1 = A.inv1, inv2 = A.inv2;
  uint32_t key = tensor_key(A.seed, A.step, A.base + ti);
  if (A.device_step) {
    inv1 = A.device_step[ti].inv1;
    inv2 = A.device_step[ti].inv2;
    key = A.device_step[ti].key;
  }
  const float lr = A.lr_device ? *A.lr_device : A.lr;
  const float step = lr * inv1, decay = -lr * A.wd;
  const int64_t start = (int64_t)(blockIdx.x - A.first[ti]) * A.chunk;
  const int64_t n = T.n;
  int64_t end = min(start + A.chunk, n);
  // the 16 lanes of a block of moments stay together: each takes part in its maximum
  if (BITS8) end = (end + 127) & ~(int64_t)127;
  for (int64_t i = start + threadIdx.x * 8; i < end; i += kPass) {
    const auto rg = ld8<GD>(T.g, i, n);
    typename Row8<MASTER ? kF32 : PD>::Raw rp;
    if constexpr (MASTER)
      rp = ld8<kF32>(T.master, i, n);
    else
      rp = ld8<PD>(T.p, i, n);
    float g[8], p[8], m[8], v[8];
    int sm = 0, sv = 0;
    if constexpr (BITS8) {
      uint32_t cm[2], cv[2];
      ld_codes(T.m, i, n, cm);
      ld_codes(T.v, i, n, cv);
      sm = T.ms[i >> kBlockLog];
      sv = T.vs[i >> kBlockLog];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        m[j] = decode<true>(cm[j >> 2] >> (8 * (j & 3)) & 255, sm);
        v[j] = decode<false>(cv[j >> 2] >> (8 * (j & 3)) & 255, sv);
      }
    } else {
      const auto rm = ld8<kF32>(T.m, i, n), rv = ld8<kF32>(T.v, i, n);
      Row8<kF32>::unpack(rm, m);
      Row8<kF32>::unpack(rv, v);
    }
    Row8<GD>::unpack(rg, g);
    Row8<MASTER ? kF32 : PD>::unpack(rp, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = mul(mul(g[j], A.grad_scale), clip);
      m[j] = add(mul(A.b1, m[j]), mul(A.c1, x));
      v[j] = add(mul(A.b2, v[j]), mul(A.c2, mul(x, x)));
      p[j] = fmaf(decay, p[j], p[j]) - step * quotient<BITS8>(m[j], v[j] * inv2, A.eps);
    }
    if constexpr (BITS8) {
      // what lies past the tensor's end is zero and stays so
      uint32_t am = 0, av = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        am = max(am, __float_as_uint(m[j]) & 0x7FFFFFFFu);
        av = max(av, __float_as_uint(v[j]) & 0x7FFFFFFFu);
      }
      am = max16(am);
      av = max16(av);
      sm = block_scale(am, 17);
      sv = block_scale(av, 33);
      const uint32_t at = key + (uint32_t)i * 0x1E3779B9u;
      uint32_t cm[2] = {0, 0}, cv[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t r = mix(at + j * 0x1E3779B9u);
        cm[j >> 2] |= encode<true>(m[j], sm, r & 0xFFFFu) << (8 * (j & 3));
        cv[j >> 2] |= encode<false>(v[j], sv, r >> 16) << (8 * (j & 3));
      }
      const bool bm = am >= 0x7F800000u, bv = av >= 0x7F800000u;
      if (bm) cm[0] = cm[1] = 0;
      if (bv) cv[0] = cv[1] = 0;
      st_codes(T.m, i, n, cm);
      st_codes(T.v, i, n, cv);
      if ((i & ((1 << kBlockLog) - 1)) == 0) {
        T.ms[i >> kBlockLog] = (uint8_t)(bm ? 255 : sm + kScaleBias);
        T.vs[i >> kBlockLog] = (uint8_t)(bv ? 255 : sv + kScaleBias);
      }
    } else {
      st8<kF32>(T.m, i, n, m);
      st8<kF32>(T.v, i, n, v);
    }
    if constexpr (MASTER) st8<kF32>(T.master, i, n, p);
    st8<PD>(T.p, i, n, p);
  }
}

// ---------------------------------------------------------------------------
// the gradients' norm
// ---------------------------------------------------------------------------

struct NormTensor {
  const void* g;
  int64_t n;
};
struct NormArgs {
  static constexpr int kTensors = (kArgBytes - 48) / 20;
  int64_t chunk;        // elements a block, a multiple of 2048
  double* partial;      // one a block
  int count;
  float grad_scale;
  int first[kTensors];
  NormTensor t[kTensors];
};

// In 64 bits: no gradient's square is out of range, and neither the sum's order nor its
// rounding shows in the norm.  It costs nothing beside the reading.
__device__ __forceinline__ double squares(const float g[8], float scale) {
  double s = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const double x = mul(g[j], scale);
    s = fma(x, x, s);
  }
  return s;
}

template <int GD>
__global__ __launch_bounds__(kThreads) void grad_squares(const NormArgs A) {
  __shared__ double part[kThreads / 64];
  const int ti = find_tensor(A.first, A.count, blockIdx.x);
  const NormTensor& T = A.t[ti];
  const int64_t start = (blockIdx.x - A.first[ti]) * A.chunk, end = min(start + A.chunk, T.n);
  double sum = 0;
  int64_t i = start + threadIdx.x * 8;
  for (; i + 3 * kPass + 8 <= end; i += 4 * kPass) {
    typename Row8<GD>::Raw r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      r[u] = Row8<GD>::ld((const typename Row8<GD>::T*)T.g + i + u * kPass);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      float g[8];
      Row8<GD>::unpack(r[u], g);
      sum += squares(g, A.grad_scale);
    }
  }
  for (; i < end; i += kPass) {
    float g[8];
    Row8<GD>::unpack(ld8<GD>(T.g, i, T.n), g);
    sum += squares(g, A.grad_scale);
  }
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) A.partial[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

__global__ void decide_kernel(const float* norm, float max_norm, Control* control) {
  *control = decide(*norm, max_norm);
}

// The norm, and what the step does with it.  One block.
__global__ __launch_bounds__(1024) void norm_kernel(const double* partial, int n, float max_norm,
                                                    float* norm, Control* control) {
  const float f = root_of_sum<1024>(partial, n);
  if (threadIdx.x == 0) {
    *norm = f;
    if (control) *control = decide(f, max_norm);
  }
}

// ---------------------------------------------------------------------------
// step counts on the device
// ---------------------------------------------------------------------------

constexpr int kCounts = 256;
struct CountArgs {
  int64_t* step[kCounts];
  const Control* control;
  DeviceStep* out;
  int count, base;
  uint32_t seed;
  double b1, b2;
};
__global__ __launch_bounds__(kCounts) void count_kernel(const CountArgs A) {
  const int i = threadIdx.x;
  if (i >= A.count || (A.control && A.control->skip)) return;
  const int64_t t = *A.step[i] + 1;
  *A.step[i] = t;
  A.out[i].inv1 = (float)(1.0 / (1.0 - pow(A.b1, (double)t)));
  A.out[i].inv2 = (float)(1.0 / (1.0 - pow(A.b2, (double)t)));
  A.out[i].key = tensor_key(A.seed, (uint32_t)t, (uint32_t)(A.base + i));
}

// ---------------------------------------------------------------------------
// what 8-bit moments stand for
// ---------------------------------------------------------------------------

struct ValueTensor {
  const void* m;
  const void* v;
  const uint8_t* ms;
  const uint8_t* vs;
  uint16_t* om;
  uint16_t* ov;
  int64_t n;
};
struct ValueArgs {
  static constexpr int kTensors = (kArgBytes - 24) / 60;
  int64_t chunk;
  int count;
  int first[kTensors];
  ValueTensor t[kTensors];
};
// Every value is a bf16 number: four bits times a power of two.
__global__ __launch_bounds__(kThreads) void values_kernel(const ValueArgs A) {
  const int ti = find_tensor(A.first, A.count, blockIdx.x);
  const ValueTensor& T = A.t[ti];
  const int64_t start = (blockIdx.x - A.first[ti]) * A.chunk;
  const int64_t n = T.n, end = min(start + A.chunk, n);
  for (int64_t i = start + threadIdx.x * 8; i < end; i += kPass) {
    uint32_t cm[2], cv[2];
    ld_codes(T.m, i, n, cm);
    ld_codes(T.v, i, n, cv);
    const int sm = T.ms[i >> kBlockLog], sv = T.vs[i >> kBlockLog];
    float m[8], v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = decode<true>(cm[j >> 2] >> (8 * (j & 3)) & 255, sm);
      v[j] = decode<false>(cv[j >> 2] >> (8 * (j & 3)) & 255, sv);
    }
    st8<kBF16>(T.om, i, n, m);
    st8<kBF16>(T.ov, i, n, v);
  }
}

int ok() { return hipGetLastError() == hipSuccess ? kOk : kErrLaunch; }
int64_t chunks(int64_t n, int64_t c) { return (n + c - 1) / c; }

// Elements a block, so that all of a call's are about `blocks` blocks: a multiple of a
// pass, `most` passes at most.
int64_t chunk_for(int64_t total, int64_t blocks, int64_t most) {
  return std::min(std::max<int64_t>(total / blocks / kPass, 1), most) * kPass;
}
// The step's: few passes, so that a CU has many blocks (31 M elements in 320 tensors: 155
// us with one pass a block, 174 with four); two where a pass's start shows (8-bit: 144
// and 154) or blocks are many.
int64_t step_chunk(int64_t total, bool bits8) {
  return (bits8 || total >= 1 << 27 ? 2 : 1) * kPass;
}
// A small step's blocks add the norm's sums themselves, a launch less (0.5 M elements
// clipped: 21 us, 17.6 without it); more blocks than the chip holds would each wait for them.
constexpr int64_t kOwnNorm = 2048 * kPass;
// The norm's: four passes together, few enough blocks for what adds their sums.
int64_t norm_chunk(int64_t total) {
  return 4 * chunk_for(total, total <= kOwnNorm ? 1024 : 8192, 1 << 30);
}

struct Sizes {
  int64_t total = 0;
};
int tensor_sizes(const cpt_adamw_tensor* t, int64_t count, Sizes* s) {
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].n < 0) return kErrShape;
    if (t[i].n > 1ll << 40) return kErrTooLarge;
    s->total += t[i].n;
  }
  return s->total > 1ll << 40 ? kErrTooLarge : kOk;
}

// Workspace: a Control, a DeviceStep a tensor, partial sums.
constexpr int64_t kControlBytes = 16;
int64_t step_bytes(int64_t count) { return (count * (int64_t)sizeof(DeviceStep) + 15) / 16 * 16; }
int64_t workspace_bytes(int64_t count, int64_t total) {
  return kControlBytes + step_bytes(count) + 8 * (count + chunks(total, norm_chunk(total)) + 1);
}

template <int GD>
int launch_squares(const cpt_adamw_tensor* t, int64_t count, int64_t chunk, float grad_scale,
                   double* partial, int64_t* blocks, hipStream_t st) {
  int64_t done = 0;
  for (int64_t i = 0; i < count;) {
    NormArgs A;
    A.count = 0;
    A.chunk = chunk, A.grad_scale = grad_scale, A.partial = partial + done;
    int64_t grid = 0;
    for (; i < count && A.count < NormArgs::kTensors; ++i) {
      if (t[i].n == 0) continue;
      A.first[A.count] = (int)grid;
      A.t[A.count++] = NormTensor{t[i].g, t[i].n};
      grid += chunks(t[i].n, chunk);
    }
    if (A.count == 0) break;
    grad_squares<GD><<<(unsigned)grid, kThreads, 0, st>>>(A);
    if (ok()) return kErrLaunch;
    done += grid;
  }
  *blocks = done;
  return kOk;
}

int grad_norm(int gd, const cpt_adamw_tensor* t, int64_t count, int64_t total, float grad_scale,
              float max_norm, float* norm, Control* control, double* partial, int64_t* partials,
              hipStream_t st) {
  int64_t blocks = 0;
  const int64_t chunk = norm_chunk(total);
  const auto squares = gd == kF32   ? launch_squares<kF32>
                       : gd == kF16 ? launch_squares<kF16>
                                    : launch_squares<kBF16>;
  const int rc = squares(t, count, chunk, grad_scale, partial, &blocks, st);
  if (rc) return rc;
  if (partials) {       // left to the step
    *partials = blocks;
    return kOk;
  }
  norm_kernel<<<1, 1024, 0, st>>>(partial, (int)blocks, max_norm, norm, control);
  return ok();
}

// All launches of a step of one kind, a run of tensors with one step number each.
template <int PD, int GD, bool BITS8, bool MASTER>
int launch_step(StepCommon C, const cpt_adamw_tensor* t, int64_t count, double beta1, double beta2,
                hipStream_t st) {
  using Args = StepArgs<BITS8, MASTER>;
  static_assert(sizeof(Args) <= kArgBytes);
  const DeviceStep* steps = C.device_step;
  for (int64_t i = 0; i < count;) {
    Args A;
    static_cast<StepCommon&>(A) = C;
    A.count = 0;
    A.base = (int)i;
    A.device_step = steps ? steps + i : nullptr;
    if (!steps) {
      A.step = (uint32_t)t[i].step;
      A.inv1 = (float)(1.0 / (1.0 - std::pow(beta1, (double)t[i].step)));
      A.inv2 = (float)(1.0 / (1.0 - std::pow(beta2, (double)t[i].step)));
    }
    int64_t grid = 0;
    // an empty tensor keeps its place (keys and device steps go by it) and has no block
    for (const int64_t step = t[i].step; i < count && A.count < Args::kTensors; ++i) {
      if (!steps && t[i].step != step) break;
      auto& T = A.t[A.count];
      A.first[A.count++] = (int)grid;
      T.p = t[i].p, T.g = t[i].g, T.m = t[i].m, T.v = t[i].v, T.n = t[i].n;
      if constexpr (BITS8) T.ms = (uint8_t*)t[i].m_scale, T.vs = (uint8_t*)t[i].v_scale;
      if constexpr (MASTER) T.master = (float*)t[i].master;
      grid += chunks(t[i].n, C.chunk);
    }
    if (grid == 0) continue;
    adamw_kernel<PD, GD, BITS8, MASTER><<<(unsigned)grid, kThreads, 0, st>>>(A);
    if (ok()) return kErrLaunch;
  }
  return kOk;
}
template <int PD, int GD>
int launch_kind(const StepCommon& C, const cpt_adamw_tensor* t, int64_t count, double beta1,
                double beta2, bool bits8, bool master, hipStream_t st) {
  if (PD != kF32 && master)
    return bits8 ? launch_step<PD, GD, true, PD != kF32>(C, t, count, beta1, beta2, st)
                 : launch_step<PD, GD, false, PD != kF32>(C, t, count, beta1, beta2, st);
  return bits8 ? launch_step<PD, GD, true, false>(C, t, count, beta1, beta2, st)
               : launch_step<PD, GD, false, false>(C, t, count, beta1, beta2, st);
}

}  // namespace adamw
}  // namespace cpt

using namespace cpt;
using namespace cpt::adamw;

extern "C" {

int64_t cpt_adamw_workspace_bytes(int64_t count, int64_t elements) {
  if (count < 0 || elements < 0 || count > 1 << 24 || elements > 1ll << 40) return -1;
  return workspace_bytes(count, elements);
}

int cpt_grad_norm(int grad_dtype, const cpt_adamw_tensor* tensors, int64_t count, float grad_scale,
                  void* norm, void* workspace, void* stream) {
  if (grad_dtype < 0 || grad_dtype > 2) return kErrDType;
  if (count < 0 || (count && !tensors) || !norm || !workspace) return kErrShape;
  Sizes s;
  if (const int rc = tensor_sizes(tensors, count, &s)) return rc;
  for (int64_t i = 0; i < count; ++i)
    if (tensors[i].n && !tensors[i].g) return kErrShape;
  return grad_norm(grad_dtype, tensors, count, s.total, grad_scale, 0.f, (float*)norm, nullptr,
                   (double*)workspace, nullptr, (hipStream_t)stream);
}

int cpt_adamw(int dtype, int grad_dtype, int bits8, int has_master, const cpt_adamw_tensor* tensors,
              int64_t count, double lr, const void* lr_device, double beta1, double beta2,
              double eps, double weight_decay, double grad_scale, double max_norm, int norm_given,
              int64_t seed, void* norm, void* workspace, void* stream) {
  if (dtype < 0 || dtype > 2 || (grad_dtype != dtype && grad_dtype != kF32)) return kErrDType;
  if (has_master && dtype == kF32) return kErrDType;
  if (count < 0 || (count && !tensors) || !(beta1 >= 0 && beta1 < 1) ||
      !(beta2 >= 0 && beta2 < 1) || !(eps >= 0))
    return kErrShape;
  const bool clip = max_norm > 0;
  Sizes s;
  if (const int rc = tensor_sizes(tensors, count, &s)) return rc;
  bool on_device = false;
  for (int64_t i = 0; i < count; ++i) {
    const cpt_adamw_tensor& t = tensors[i];
    if (i == 0) on_device = t.step_device != nullptr;
    if ((t.step_device != nullptr) != on_device || (!on_device && t.step < 1)) return kErrShape;
    if (t.n && (!t.p || !t.g || !t.m || !t.v || (bits8 && (!t.m_scale || !t.v_scale)) ||
                (has_master && !t.master)))
      return kErrShape;
  }
  if ((clip && !norm) || ((clip || on_device) && !workspace)) return kErrShape;
  const hipStream_t st = (hipStream_t)stream;
  StepCommon C{};
  Control* control = nullptr;
  DeviceStep* steps = nullptr;
  if (clip) {
    control = (Control*)workspace;
    bool one = !on_device && !norm_given && s.total > 0 && s.total <= kOwnNorm &&
               count <= StepArgs<true, true>::kTensors;
    for (int64_t i = 1; i < count; ++i) one = one && tensors[i].step == tensors[0].step;
    double* partial = (double*)((char*)workspace + kControlBytes + step_bytes(count));
    int64_t partials = 0;
    if (norm_given) {
      decide_kernel<<<1, 1, 0, st>>>((const float*)norm, (float)max_norm, control);
      if (ok()) return kErrLaunch;
    } else if (const int rc = grad_norm(grad_dtype, tensors, count, s.total, (float)grad_scale,
                                        (float)max_norm, (float*)norm, control, partial,
                                        one ? &partials : nullptr, st)) {
      return rc;
    }
    if (one) {
      C.partial = partial, C.partials = (int)partials;
      C.norm = (float*)norm, C.max_norm = (float)max_norm;
      control = nullptr;
    }
  }
  if (on_device) {
    steps = (DeviceStep*)((char*)workspace + kControlBytes);
    for (int64_t i = 0; i < count; i += kCounts) {
      CountArgs N;
      N.count = (int)std::min<int64_t>(count - i, kCounts);
      for (int k = 0; k < N.count; ++k) N.step[k] = (int64_t*)tensors[i + k].step_device;
      N.control = control, N.out = steps + i, N.base = (int)i, N.seed = (uint32_t)seed;
      N.b1 = beta1, N.b2 = beta2;
      count_kernel<<<1, kCounts, 0, st>>>(N);
      if (ok()) return kErrLaunch;
    }
  }
  C.control = control, C.device_step = steps, C.lr_device = (const float*)lr_device;
  C.chunk = step_chunk(s.total, bits8), C.seed = (uint32_t)seed;
  C.lr = (float)lr, C.wd = (float)weight_decay, C.b1 = (float)beta1, C.b2 = (float)beta2;
  C.c1 = (float)(1 - beta1), C.c2 = (float)(1 - beta2);
  C.eps = (float)eps, C.grad_scale = (float)grad_scale;
#define CPT_STEP(PD, GD) \
  launch_kind<PD, GD>(C, tensors, count, beta1, beta2, bits8, has_master, st)
  if (dtype == kF32) return CPT_STEP(kF32, kF32);
  if (dtype == kF16) return grad_dtype == kF32 ? CPT_STEP(kF16, kF32) : CPT_STEP(kF16, kF16);
  return grad_dtype == kF32 ? CPT_STEP(kBF16, kF32) : CPT_STEP(kBF16, kBF16);
#undef CPT_STEP
}

int cpt_adamw_8bit_values(const cpt_adamw_tensor* tensors, int64_t count, void* stream) {
  if (count < 0 || (count && !tensors)) return kErrShape;
  Sizes s;
  if (const int rc = tensor_sizes(tensors, count, &s)) return rc;
  for (int64_t i = 0; i < count; ++i) {
    const cpt_adamw_tensor& t = tensors[i];
    if (t.n && (!t.p || !t.g || !t.m || !t.v || !t.m_scale || !t.v_scale)) return kErrShape;
  }
  for (int64_t i = 0; i < count;) {
    ValueArgs A;
    A.count = 0;
    A.chunk = step_chunk(s.total, true);
    int64_t grid = 0;
    for (; i < count && A.count < ValueArgs::kTensors; ++i) {
      const cpt_adamw_tensor& t = tensors[i];
      if (t.n == 0) continue;
      A.first[A.count] = (int)grid;
      A.t[A.count++] = ValueTensor{t.m, t.v, (const uint8_t*)t.m_scale, (const uint8_t*)t.v_scale,
                                   (uint16_t*)t.p, (uint16_t*)t.g, t.n};
      grid += chunks(t.n, A.chunk);
    }
    if (A.count == 0) break;
    values_kernel<<<(unsigned)grid, kThreads, 0, (hipStream_t)stream>>>(A);
    if (ok()) return kErrLaunch;
  }
  return kOk;
}

}  // extern "C"
