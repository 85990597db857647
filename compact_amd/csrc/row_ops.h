// Helpers of the row kernels (embedding.hip, residual_norm.hip, distill.hip):
// eight consecutive elements of a row at any element alignment, and sums and
// maxima over a wavefront.
#pragma once

#include "common.h"

namespace cpt {

// A 16-byte access needs no more than the element's own alignment: gfx950
// takes an unaligned global_load_dwordx4 / store_dwordx4 as it is, so rows of
// odd width (every row at another offset) run on the same code as aligned ones.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

// Eight elements as they are stored: Raw, 4 or 8 registers.
template <int DT> struct Row8;

template <int DT> struct Row8Half {   // 16-bit formats
  using T = uint16_t;
  struct Raw { u32x4 w; };
  static __device__ __forceinline__ Raw ld(const T* p) {
    return Raw{*reinterpret_cast<const u32x4_a2*>(p)};
  }
  // the first n < 8 elements, the rest `fill` (the format's bits)
  static __device__ __forceinline__ Raw ld_n(const T* p, int n, uint32_t fill) {
    Raw r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = 2 * j < n ? p[2 * j] : fill;
      const uint32_t hi = 2 * j + 1 < n ? p[2 * j + 1] : fill;
      r.w[j] = lo | (hi << 16);
    }
    return r;
  }
  static __device__ __forceinline__ void st(T* p, const Raw& r) {
    *reinterpret_cast<u32x4_a2*>(p) = r.w;
  }
  static __device__ __forceinline__ void st_n(T* p, const Raw& r, int n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (2 * j < n) p[2 * j] = (uint16_t)(r.w[j] & 0xFFFFu);
      if (2 * j + 1 < n) p[2 * j + 1] = (uint16_t)(r.w[j] >> 16);
    }
  }
  // elements k .. 7
  static __device__ __forceinline__ void st_from(T* p, const Raw& r, int k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (2 * j >= k) p[2 * j] = (uint16_t)(r.w[j] & 0xFFFFu);
      if (2 * j + 1 >= k) p[2 * j + 1] = (uint16_t)(r.w[j] >> 16);
    }
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float v[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (DT == kBF16) {
        v[2 * j] = __uint_as_float(r.w[j] << 16);
        v[2 * j + 1] = __uint_as_float(r.w[j] & 0xFFFF0000u);
      } else {
        v[2 * j] = f16_bits_to_f32((uint16_t)(r.w[j] & 0xFFFFu));
        v[2 * j + 1] = f16_bits_to_f32((uint16_t)(r.w[j] >> 16));
      }
    }
  }
  static __device__ __forceinline__ Raw pack(const float v[8]) {
    Raw r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (DT == kBF16)
        r.w[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
      else
        r.w[j] = (uint32_t)f32_to_f16_bits(v[2 * j]) |
                 ((uint32_t)f32_to_f16_bits(v[2 * j + 1]) << 16);
    }
    return r;
  }
  static __device__ __forceinline__ Raw fill(uint32_t bits) {
    const uint32_t w = bits | (bits << 16);
    return Raw{u32x4{w, w, w, w}};
  }
  static __device__ __forceinline__ Raw zero() { return fill(0); }
  // `bits` in the elements whose bit of `which` is set
  static __device__ __forceinline__ void mask(Raw& r, uint32_t which, uint32_t bits) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (which >> (2 * j) & 1) r.w[j] = (r.w[j] & 0xFFFF0000u) | bits;
      if (which >> (2 * j + 1) & 1) r.w[j] = (r.w[j] & 0xFFFFu) | (bits << 16);
    }
  }
};
template <> struct Row8<kBF16> : Row8Half<kBF16> {
  static constexpr uint32_t kNegInf = 0xFF80u;
};
template <> struct Row8<kF16> : Row8Half<kF16> {
  static constexpr uint32_t kNegInf = 0xFC00u;
};
template <> struct Row8<kF32> {
  using T = float;
  struct Raw { u32x4 w, x; };
  static constexpr uint32_t kNegInf = 0xFF800000u;
  static __device__ __forceinline__ Raw ld(const T* p) {
    const u32x4_a4* q = reinterpret_cast<const u32x4_a4*>(p);
    return Raw{q[0], q[1]};
  }
  static __device__ __forceinline__ Raw ld_n(const T* p, int n, uint32_t fill) {
    Raw r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.w[j] = j < n ? __float_as_uint(p[j]) : fill;
      r.x[j] = 4 + j < n ? __float_as_uint(p[4 + j]) : fill;
    }
    return r;
  }
  static __device__ __forceinline__ void st(T* p, const Raw& r) {
    u32x4_a4* q = reinterpret_cast<u32x4_a4*>(p);
    q[0] = r.w;
    q[1] = r.x;
  }
  static __device__ __forceinline__ void st_n(T* p, const Raw& r, int n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j < n) p[j] = __uint_as_float(r.w[j]);
      if (4 + j < n) p[4 + j] = __uint_as_float(r.x[j]);
    }
  }
  static __device__ __forceinline__ void st_from(T* p, const Raw& r, int k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= k) p[j] = __uint_as_float(r.w[j]);
      if (4 + j >= k) p[4 + j] = __uint_as_float(r.x[j]);
    }
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float v[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = __uint_as_float(r.w[j]);
      v[4 + j] = __uint_as_float(r.x[j]);
    }
  }
  static __device__ __forceinline__ Raw pack(const float v[8]) {
    Raw r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r.w[j] = __float_as_uint(v[j]);
      r.x[j] = __float_as_uint(v[4 + j]);
    }
    return r;
  }
  static __device__ __forceinline__ Raw fill(uint32_t b) {
    return Raw{u32x4{b, b, b, b}, u32x4{b, b, b, b}};
  }
  static __device__ __forceinline__ Raw zero() { return fill(0); }
  static __device__ __forceinline__ void mask(Raw& r, uint32_t which, uint32_t bits) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (which >> j & 1) r.w[j] = bits;
      if (which >> (4 + j) & 1) r.x[j] = bits;
    }
  }
};

// The compiler would keep the columns that it unpacked for one pass over a row in
// registers for the next pass: eight a vector more.  This makes it unpack again.
template <int DT>
__device__ __forceinline__ void repack(typename Row8<DT>::Raw& r) {
  asm volatile("" : "+v"(r.w));
  if constexpr (DT == kF32) asm volatile("" : "+v"(r.x));
}

// Elements [j, j + 8) of a row of d columns: `fill` past its end.
template <int DT>
__device__ __forceinline__ typename Row8<DT>::Raw row_ld(const typename Row8<DT>::T* row, int64_t j,
                                                         int64_t d, uint32_t fill) {
  if (j + 8 <= d) return Row8<DT>::ld(row + j);
  const int n = j < d ? (int)(d - j) : 0;
  return Row8<DT>::ld_n(row + j, n, fill);
}
template <int DT>
__device__ __forceinline__ void row_st(typename Row8<DT>::T* row, int64_t j, int64_t d,
                                       const typename Row8<DT>::Raw& r) {
  if (j + 8 <= d)
    Row8<DT>::st(row + j, r);
  else if (j < d)
    Row8<DT>::st_n(row + j, r, (int)(d - j));
}

// A thread's eight columns [j, j + 8) of a row of d, without a branch before the
// load (each would be waited for by itself): past the end the row's last eight are
// taken, of which the first `skip` are other threads' too.  Rows of fewer than
// eight columns (TINY) go element by element.
template <int DT, bool TINY>
struct Cols {
  using R = Row8<DT>;
  using T = typename R::T;
  int64_t at;
  int skip, n;
  __device__ __forceinline__ Cols(int64_t j, int64_t d) {
    at = TINY ? j : min(j, d - 8);
    skip = (int)min(j - at, (int64_t)8);
    n = (int)max(min(d - j, (int64_t)8), (int64_t)0);
  }
  __device__ __forceinline__ typename R::Raw ld(const T* row) const {
    return TINY ? R::ld_n(row + at, n, 0) : R::ld(row + at);
  }
  // shared columns are stored by each that has them: with the same values
  __device__ __forceinline__ void st(T* row, const typename R::Raw& r) const {
    if (TINY)
      R::st_n(row + at, r, n);
    else if (skip < 8)
      R::st(row + at, r);
  }
  // only the thread's own: where what is stored depends on what was there
  __device__ __forceinline__ void st_own(T* row, const typename R::Raw& r) const {
    if (TINY)
      R::st_n(row + at, r, n);
    else if (skip == 0)
      R::st(row + at, r);
    else
      R::st_from(row + at, r, skip);
  }
};

// Sum and maximum over a wavefront, in every lane: four shifts within rows of
// 16 lanes and two broadcasts across them (DPP), a fixed order.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float old, float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(old), __float_as_uint(x),
                                                     CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float lane63(float x) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 63));
}
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp<0x111, 0xF>(0.f, x);   // row_shr:1
  x += dpp<0x112, 0xF>(0.f, x);
  x += dpp<0x114, 0xF>(0.f, x);
  x += dpp<0x118, 0xF>(0.f, x);
  x += dpp<0x142, 0xA>(0.f, x);   // row_bcast:15 into rows 1 and 3
  x += dpp<0x143, 0xC>(0.f, x);   // row_bcast:31 into rows 2 and 3
  return lane63(x);
}
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<0x111, 0xF>(x, x));
  x = fmaxf(x, dpp<0x112, 0xF>(x, x));
  x = fmaxf(x, dpp<0x114, 0xF>(x, x));
  x = fmaxf(x, dpp<0x118, 0xF>(x, x));
  x = fmaxf(x, dpp<0x142, 0xA>(x, x));
  x = fmaxf(x, dpp<0x143, 0xC>(x, x));
  return lane63(x);
}

// An element of a tensor whose type is known at run time only.
__device__ __forceinline__ float ld_any(const void* p, int dt, int64_t i) {
  if (dt == kF32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t h = reinterpret_cast<const uint16_t*>(p)[i];
  return dt == kF16 ? f16_bits_to_f32(h) : bf16_to_f32(h);
}
__device__ __forceinline__ void st_any(void* p, int dt, int64_t i, float v) {
  if (dt == kF32)
    reinterpret_cast<float*>(p)[i] = v;
  else
    reinterpret_cast<uint16_t*>(p)[i] =
        dt == kF16 ? f32_to_f16_bits(v) : (uint16_t)f32_to_bf16_bits(v);
}
// An index tensor of 32 or 64 bits.
__device__ __forceinline__ int64_t ld_index(const void* p, int wide, int64_t i) {
  return wide ? reinterpret_cast<const int64_t*>(p)[i] : reinterpret_cast<const int32_t*>(p)[i];
}

}  // namespace cpt
