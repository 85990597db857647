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
// tensors' pointers are kernel arguments, 48 a launch: no table to upload or keep.

#include <algorithm>
#include <cmath>

#include "compact_amd.h"
#include "row_ops.h"

namespace cpt {
namespace {

constexpr int kThreads = 256;
constexpr int kStepTensors = 48;      // 80 bytes each in 4 KB of kernel arguments
constexpr int kChunk = 8192;          // elements a block of the step, a multiple of 128
constexpr int kBlockLog = 7;          // 128 elements share a scale
constexpr int kScaleBias = 134;
constexpr int kNormBlocks = 2048;     // blocks that the squares' sum is cut into, about

struct Tensor {
  void* p;
  const void* g;
  void* m;
  void* v;
  uint8_t* ms;
  uint8_t* vs;
  float* master;
  int64_t n;
  int first;            // first block of this tensor
  uint32_t key;         // the dither's
  float inv1, inv2;     // 1 / (1 - b^t)
};

// What a step on the device decides: one float4 for all tensors {clip, skip}, then
// {inv1, inv2, key} a tensor where the step counts are on the device.
struct Control {
  float clip;
  int skip;
};
struct DeviceStep {
  float inv1, inv2;
  uint32_t key;
};

struct StepArgs {
  Tensor t[kStepTensors];
  const Control* control;         // null: no clipping
  const DeviceStep* device_step;  // null: the tensors' own
  const float* lr_device;         // null: lr
  int count;
  float lr, wd, b1, b2, c1, c2, eps, grad_scale;   // c = 1 - b
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

// The tensor that a block works on: the last whose first block is not past it.
template <class Args>
__device__ __forceinline__ int find_tensor(const Args& A, int block) {
  const int lane = threadIdx.x & 63;
  const int first = lane < A.count ? A.t[lane].first : 0x7FFFFFFF;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(first <= block)) - 1);
}

__device__ __forceinline__ float mul(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ float add(float a, float b) { return __fadd_rn(a, b); }

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
  const float y =
      __builtin_ldexpf(__uint_as_float((SIGNED ? code & 127 : code) << 20), scale - (kScaleBias - 129));
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

// PD: the parameters' type, GD: the gradients', BITS8: moments in 8 bits, MASTER: an
// fp32 copy of the parameters that is stepped in their place.
template <int PD, int GD, bool BITS8, bool MASTER>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const StepArgs A) {
  const int ti = find_tensor(A, blockIdx.x);
  const Tensor& T = A.t[ti];
  float clip = 1.f;
  if (A.control) {
    if (A.control->skip) return;
    clip = A.control->clip;
  }
  float inv1 = T.inv1, inv2 = T.inv2;
  uint32_t key = T.key;
  if (A.device_step) {
    inv1 = A.device_step[ti].inv1;
    inv2 = A.device_step[ti].inv2;
    key = A.device_step[ti].key;
  }
  const float lr = A.lr_device ? *A.lr_device : A.lr;
  const float step = lr * inv1, decay = -lr * A.wd;
  const int64_t start = (int64_t)(blockIdx.x - T.first) * kChunk;
  const int64_t n = T.n;
  int64_t end = min(start + kChunk, n);
  // the 16 lanes of a block of moments stay together: each takes part in its maximum
  if (BITS8) end = (end + 127) & ~(int64_t)127;
  for (int64_t i = start + threadIdx.x * 8; i < end; i += kThreads * 8) {
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
      const float den = sqrtf(v[j] * inv2) + A.eps;
      p[j] = fmaf(decay, p[j], p[j]) - step * m[j] / den;
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
  int first;
};
constexpr int kNormTensors = 64;      // a lane each in find_tensor
struct NormArgs {
  NormTensor t[kNormTensors];
  int count;
  int64_t chunk;
  float grad_scale;
  double* partial;      // one a block
};

// Squares are summed in 64 bits: no gradient's square is out of range, and the order
// of the sum does not show.
template <int GD>
__global__ __launch_bounds__(kThreads) void grad_squares(const NormArgs A) {
  __shared__ double part[kThreads / 64];
  const NormTensor& T = A.t[find_tensor(A, blockIdx.x)];
  const int64_t start = (blockIdx.x - T.first) * A.chunk, end = min(start + A.chunk, T.n);
  double s[2] = {0, 0};
  for (int64_t i = start + threadIdx.x * 8; i < end; i += kThreads * 8) {
    float g[8];
    Row8<GD>::unpack(ld8<GD>(T.g, i, T.n), g);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double x = mul(g[j], A.grad_scale);
      s[j & 1] += x * x;
    }
  }
  double sum = s[0] + s[1];
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) A.partial[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

__device__ __forceinline__ void decide(float norm, float max_norm, Control* control) {
  control->clip = fminf(1.f, max_norm / add(norm, 1e-6f));
  control->skip = !(norm < INFINITY);
}
__global__ void decide_kernel(const float* norm, float max_norm, Control* control) {
  decide(*norm, max_norm, control);
}

// The norm, and what the step does with it.  One block.
__global__ __launch_bounds__(1024) void norm_kernel(const double* partial, int n, float max_norm,
                                                    float* norm, Control* control) {
  __shared__ double part[16];
  double s = 0;
  for (int i = threadIdx.x; i < n; i += 1024) s += partial[i];
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = 0;
    for (int i = 0; i < 16; ++i) t += part[i];
    const float f = (float)sqrt(t);
    *norm = f;
    if (control) decide(f, max_norm, control);
  }
}

// ---------------------------------------------------------------------------
// step counts on the device
// ---------------------------------------------------------------------------

struct CountArgs {
  int64_t* step[kStepTensors];
  const Control* control;
  DeviceStep* out;
  int count, base;
  uint32_t seed;
  double b1, b2;
};
__global__ __launch_bounds__(64) void count_kernel(const CountArgs A) {
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
  int first;
};
constexpr int kValueTensors = 56;
struct ValueArgs {
  ValueTensor t[kValueTensors];
  int count;
};
// Every value is a bf16 number: four bits times a power of two.
__global__ __launch_bounds__(kThreads) void values_kernel(const ValueArgs A) {
  const ValueTensor& T = A.t[find_tensor(A, blockIdx.x)];
  const int64_t start = (int64_t)(blockIdx.x - T.first) * kChunk;
  const int64_t n = T.n, end = min(start + kChunk, n);
  for (int64_t i = start + threadIdx.x * 8; i < end; i += kThreads * 8) {
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

// Elements a block of the norm's first launch: all gradients in about kNormBlocks.
int64_t norm_chunk(int64_t total) {
  return std::max<int64_t>(kThreads * 8, (total / kNormBlocks + 2047) / 2048 * 2048);
}

struct Sizes {
  int64_t total = 0, live = 0;
};
int tensor_sizes(const cpt_adamw_tensor* t, int64_t count, Sizes* s) {
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].n < 0) return kErrShape;
    if (t[i].n > 1ll << 40) return kErrTooLarge;
    s->total += t[i].n;
    s->live += t[i].n > 0;
  }
  return s->total > 1ll << 42 ? kErrTooLarge : kOk;
}

// Workspace: {Control, 16 bytes}, a DeviceStep a tensor of a launch's, partial sums.
int64_t workspace_bytes(int64_t count, int64_t total) {
  const int64_t steps = (count + kStepTensors) * 16;
  return 16 + steps + 8 * (count + chunks(total, norm_chunk(total)) + 1);
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
    for (; i < count && A.count < kNormTensors; ++i) {
      if (t[i].n == 0) continue;
      A.t[A.count++] = NormTensor{t[i].g, t[i].n, (int)grid};
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
              float max_norm, float* norm, Control* control, double* partial, hipStream_t st) {
  int64_t blocks = 0;
  const int64_t chunk = norm_chunk(total);
  const int rc = gd == kF32 ? launch_squares<kF32>(t, count, chunk, grad_scale, partial, &blocks, st)
                 : gd == kF16
                     ? launch_squares<kF16>(t, count, chunk, grad_scale, partial, &blocks, st)
                     : launch_squares<kBF16>(t, count, chunk, grad_scale, partial, &blocks, st);
  if (rc) return rc;
  norm_kernel<<<1, 1024, 0, st>>>(partial, (int)blocks, max_norm, norm, control);
  return ok();
}

template <int PD, int GD>
void launch_step(const StepArgs& A, int64_t grid, bool bits8, bool master, hipStream_t st) {
  const unsigned b = (unsigned)grid;
  if (bits8) {
    if (master && PD != kF32)
      adamw_kernel<PD, GD, true, PD != kF32><<<b, kThreads, 0, st>>>(A);
    else
      adamw_kernel<PD, GD, true, false><<<b, kThreads, 0, st>>>(A);
  } else if (master && PD != kF32) {
    adamw_kernel<PD, GD, false, PD != kF32><<<b, kThreads, 0, st>>>(A);
  } else {
    adamw_kernel<PD, GD, false, false><<<b, kThreads, 0, st>>>(A);
  }
}

}  // namespace
}  // namespace cpt

using namespace cpt;

extern "C" {

int64_t cpt_adamw_workspace_bytes(int64_t count, int64_t elements) {
  if (count < 0 || elements < 0 || count > 1 << 24 || elements > 1ll << 42) return -1;
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
                   (double*)workspace, (hipStream_t)stream);
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
  Control* control = nullptr;
  DeviceStep* steps = nullptr;
  if (clip) {
    control = (Control*)workspace;
    double* partial = (double*)((char*)workspace + 16 + (count + kStepTensors) * 16);
    if (norm_given) {
      decide_kernel<<<1, 1, 0, st>>>((const float*)norm, (float)max_norm, control);
      if (ok()) return kErrLaunch;
    } else if (const int rc = grad_norm(grad_dtype, tensors, count, s.total, (float)grad_scale,
                                        (float)max_norm, (float*)norm, control, partial, st)) {
      return rc;
    }
  }
  if (on_device) steps = (DeviceStep*)((char*)workspace + 16);
  StepArgs A;
  A.control = control;
  A.lr_device = (const float*)lr_device;
  A.lr = (float)lr, A.wd = (float)weight_decay;
  A.b1 = (float)beta1, A.b2 = (float)beta2;
  A.c1 = (float)(1 - beta1), A.c2 = (float)(1 - beta2);
  A.eps = (float)eps, A.grad_scale = (float)grad_scale;
  int64_t last_step = 0;
  float inv1 = 0, inv2 = 0;
  for (int64_t i = 0; i < count;) {
    CountArgs C;
    A.count = 0;
    A.device_step = steps;
    C.base = (int)i;
    int64_t grid = 0;
    for (int k = 0; i < count && k < kStepTensors; ++i, ++k) {
      const cpt_adamw_tensor& t = tensors[i];
      C.step[k] = (int64_t*)t.step_device;
      C.count = k + 1;
      if (!on_device && t.step != last_step) {
        last_step = t.step;
        inv1 = (float)(1.0 / (1.0 - std::pow(beta1, (double)t.step)));
        inv2 = (float)(1.0 / (1.0 - std::pow(beta2, (double)t.step)));
      }
      // an empty tensor keeps its place (the device's step counts go by it) and no block
      A.t[A.count++] = Tensor{t.p, t.g, t.m, t.v, (uint8_t*)t.m_scale, (uint8_t*)t.v_scale,
                              (float*)t.master, t.n, (int)grid,
                              tensor_key((uint32_t)seed, (uint32_t)t.step, (uint32_t)i), inv1,
                              inv2};
      grid += chunks(t.n, kChunk);
    }
    if (on_device) {
      C.control = control, C.out = steps, C.seed = (uint32_t)seed, C.b1 = beta1, C.b2 = beta2;
      count_kernel<<<1, 64, 0, st>>>(C);
      if (ok()) return kErrLaunch;
      steps += C.count;
    }
    if (grid == 0) continue;
#define CPT_STEP(PD, GD) launch_step<PD, GD>(A, grid, bits8, has_master, st)
    if (dtype == kF32)
      CPT_STEP(kF32, kF32);
    else if (dtype == kF16)
      grad_dtype == kF32 ? CPT_STEP(kF16, kF32) : CPT_STEP(kF16, kF16);
    else
      grad_dtype == kF32 ? CPT_STEP(kBF16, kF32) : CPT_STEP(kBF16, kBF16);
#undef CPT_STEP
    if (ok()) return kErrLaunch;
  }
  return kOk;
}

int cpt_adamw_8bit_values(const cpt_adamw_tensor* tensors, int64_t count, void* stream) {
  if (count < 0 || (count && !tensors)) return kErrShape;
  Sizes s;
  if (const int rc = tensor_sizes(tensors, count, &s)) return rc;
  for (int64_t i = 0; i < count; ++i) {
    const cpt_adamw_tensor& t = tensors[i];
    if (t.n && (!t.p || !t.master || !t.m || !t.v || !t.m_scale || !t.v_scale)) return kErrShape;
  }
  for (int64_t i = 0; i < count;) {
    ValueArgs A;
    A.count = 0;
    int64_t grid = 0;
    for (; i < count && A.count < kValueTensors; ++i) {
      const cpt_adamw_tensor& t = tensors[i];
      if (t.n == 0) continue;
      A.t[A.count++] = ValueTensor{t.m, t.v, (const uint8_t*)t.m_scale, (const uint8_t*)t.v_scale,
                                   (uint16_t*)t.p, (uint16_t*)t.master, t.n, (int)grid};
      grid += chunks(t.n, kChunk);
    }
    if (A.count == 0) break;
    values_kernel<<<(unsigned)grid, kThreads, 0, (hipStream_t)stream>>>(A);
    if (ok()) return kErrLaunch;
  }
  return kOk;
}

}  // extern "C"
