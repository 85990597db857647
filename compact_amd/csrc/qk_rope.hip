// The queries' and keys' norms and position rotation, and their gradient.
//
// Per head of d columns, at position t:
//   n = x / sqrt(mean x^2 + eps) * w            (no weights: n = x)
//   the first R columns turn by pairs (a, b) -> (a c - b s, b c + a s) with
//   c, s = scaling * cos, sin(t * inv_freq[pair]); a pair is two neighbours
//   (interleaved) or column i of each half of the R.
// Backward, with dn = the gradient turned back and rho = 1 / sqrt(mean x^2 + eps):
//   dw = sum over tokens and heads of dn * x * rho
//   dx = rho * (dn w - x rho^2 mean(dn w x))
// Nothing is kept between the two: a head's row is in registers when rho is needed.
//
// Bound: HBM, two (backward with norms three) passes over q and k.  A lane holds
// eight pairs, so a head is d / 16 lanes and the norm's sums are a few exchanges
// within them.  All d columns are pairs here; those past R are normed and left so.
// Angles are products in 64 bits reduced to a turn (a position of 10^6 times a
// frequency rounded in 32 bits is 0.03 off; these are 1e-7 off at 2 10^9, 1e-4 at
// 10^12), once per token and pair into LDS for all heads.
//
// Measured on one MI355X: 8192 tokens x 36 heads x 64 bf16 13.6 us a pass (5.5 TB/s, in part
// from the Infinity Cache); with norms 8192 x 64 x 128 bf16 46; kernel time of a trace's
// mean: the gradient of that 82 us (4.9 TB/s) and 4.7 for the partial sums, 4 tokens 4.1.

#include <algorithm>

#include "compact_amd.h"
#include "row_ops.h"

namespace cpt {
namespace qkrope {

constexpr int kRopeThreads = 256;
constexpr int kRopeTableBytes = 19456;    // cos and sin of a tile of tokens
constexpr int kRopeMaxTile = 64;          // tokens a tile
constexpr int kRopeBlocks = 2048;         // of the backward, each with a partial sum
constexpr int kSumThreads = 1024;

struct RopeSide {                         // queries or keys
  const void* x;
  const void* dy;
  void* out;
  const void* w;
  float* partial;                         // [blocks, d]
  int64_t xs[3], ys[3], os[3];            // elements between sequences, tokens, heads
  FastDivU32 heads;
  int blocks, tile;
};

struct RopeArgs {
  RopeSide side[2];
  const void* positions;
  const float* inv_freq;
  int64_t pos_stride;
  FastDivU32 seq;
  int tokens, d, rot, lanes, width, pos_wide, wdt;   // width: columns of the table side by side
  float eps, scaling;
};

// A lane's eight pairs of a head, pair(t) for t = 0 .. 7.  VEC: eight neighbours, moved 16
// bytes at a time at any alignment; where they would end past the head's (or, in
// halves, past those that turn) they are the last eight, of which the lane before has
// the first `skip` too.  Otherwise (fewer than eight of a kind) every `lanes`-th, an
// element at a time.
template <int DT, bool VEC, bool INTER>
struct HeadLane {
  using R = Row8<DT>;
  using T = typename R::T;
  int lane, lanes, pairs, rot, d, first, skip;

  __device__ __forceinline__ HeadLane(int lane, int lanes, int rot, int d)
      : lane(lane), lanes(lanes), pairs(d / 2), rot(rot), d(d) {
    // in halves a lane has turning pairs or others: not both
    const int ahead = INTER ? 0 : (rot / 2 + 7) / 8;
    const bool turns = INTER || lane < ahead;
    const int begin = turns ? 0 : rot / 2, end = INTER || !turns ? pairs : rot / 2;
    const int want = begin + 8 * (turns ? lane : lane - ahead);
    first = max(min(want, end - 8), 0);
    skip = min(want - first, 8);
  }
  __device__ __forceinline__ bool on(int t) const {
    return VEC ? t >= skip : lane + t * lanes < pairs;
  }
  // without VEC pairs past the end are taken as the last one
  __device__ __forceinline__ int pair(int t) const {
    return VEC ? first + t : min(lane + t * lanes, pairs - 1);
  }
  __device__ __forceinline__ int col_a(int i) const {
    if (INTER) return 2 * i;
    return i < rot / 2 ? i : i + rot / 2;
  }
  __device__ __forceinline__ int col_b(int i) const {
    if (INTER) return 2 * i + 1;
    return i < rot / 2 ? i + rot / 2 : i + d / 2;
  }
  __device__ __forceinline__ void ld(const T* row, float a[8], float b[8]) const {
    if constexpr (VEC) {
      const int i = pair(0);
      if constexpr (INTER) {
        float v[16];
        R::unpack(R::ld(row + 2 * i), v);
        R::unpack(R::ld(row + 2 * i + 8), v + 8);
#pragma unroll
        for (int t = 0; t < 8; ++t) a[t] = v[2 * t], b[t] = v[2 * t + 1];
      } else {
        const auto ra = R::ld(row + col_a(i)), rb = R::ld(row + col_b(i));
        R::unpack(ra, a);
        R::unpack(rb, b);
      }
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int i = pair(t);
        a[t] = Elem<DT>::ld(row + col_a(i));
        b[t] = Elem<DT>::ld(row + col_b(i));
      }
    }
  }
  __device__ __forceinline__ void st(T* row, const float a[8], const float b[8]) const {
    if constexpr (VEC) {
      if (skip == 8) return;
      const int i = first;      // shared pairs are stored by each: with the same values
      if constexpr (INTER) {
        float v[16];
#pragma unroll
        for (int t = 0; t < 8; ++t) v[2 * t] = a[t], v[2 * t + 1] = b[t];
        R::st(row + 2 * i, R::pack(v));
        R::st(row + 2 * i + 8, R::pack(v + 8));
      } else {
        R::st(row + col_a(i), R::pack(a));
        R::st(row + col_b(i), R::pack(b));
      }
    } else {
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (on(t)) {
          Elem<DT>::st(row + col_a(pair(t)), a[t]);
          Elem<DT>::st(row + col_b(pair(t)), b[t]);
        }
    }
  }
};

// A token's row of the table, a hole after eight pairs: lanes that each read eight in a row
// do not meet in LDS's banks.
__host__ __device__ __forceinline__ int table_at(int pair) { return pair + (pair >> 3); }
__host__ __device__ __forceinline__ int table_row(int d) { return table_at(d / 2) + 1; }

// A head's weights as a lane has its columns: one branch, then loads alone (a load
// under a branch of its own is waited for by itself).
template <int DT, bool VEC, bool INTER>
__device__ __forceinline__ void ld_weights(const HeadLane<DT, VEC, INTER>& io, const void* w,
                                           int wdt, float a[8], float b[8]) {
  if (DT != kF32 && wdt == kF32) {
    const HeadLane<kF32, VEC, INTER> wide(io.lane, io.lanes, io.rot, io.d);
    wide.ld((const float*)w, a, b);
  } else {
    io.ld((const typename Elem<DT>::T*)w, a, b);
  }
}

// Pairs turned by their cos and sin, `back` or forth.  Those that do not turn are left
// alone: with cos 1 and sin 0 an infinity would make its partner NaN.
template <int DT, bool VEC, bool INTER>
__device__ __forceinline__ void turn(const HeadLane<DT, VEC, INTER>& io, const float2* table,
                                     bool back, float a[8], float b[8]) {
  // in halves a lane's eight are of a kind
  if (VEC && !INTER && io.first >= io.rot / 2) return;
  const float sign = back ? -1.f : 1.f;
  const bool all = (VEC && !INTER) || io.rot == io.d;
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int p = io.pair(t);
    const float2 cs = table[table_at(p)];
    const float s = sign * cs.y;
    const float u = a[t] * cs.x - b[t] * s, v = b[t] * cs.x + a[t] * s;
    a[t] = all || p < io.rot / 2 ? u : a[t];
    b[t] = all || p < io.rot / 2 ? v : b[t];
  }
}

// A thread's place: heads lie side by side in a wavefront, the lanes past the last whole
// head idle (lane -1 of a group that no head goes to).
struct Place {
  int lane, group, groups;
  __device__ __forceinline__ explicit Place(int lanes) {
    const int in_wave = threadIdx.x & 63, per_wave = 64 / lanes, g = in_wave / lanes;
    lane = in_wave - g * lanes;
    groups = per_wave * (kRopeThreads / 64);
    group = g < per_wave ? (int)(threadIdx.x >> 6) * per_wave + g : 1 << 30;
  }
};

// The sum over a head's lanes, in each of them: by exchanges where they are a power of
// two, otherwise folded into the first and read from there.
__device__ __forceinline__ float head_sum(float v, int lane, int lanes) {
  if ((lanes & (lanes - 1)) == 0) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
  }
  int left = lanes;
  while (left > 1) {
    const int half = (left + 1) >> 1;
    const float u = __shfl_down(v, half);
    v += lane + half < left ? u : 0.f;
    left = half;
  }
  return __shfl(v, (int)(threadIdx.x & 63) - lane);
}

// cos and sin of `turn` turns: reduced to an eighth of a turn in 64 bits, so that what is
// left fits 32, then both Taylor series (cos 1.2e-10, sin 1.8e-9 off at most there; both
// 2 x 2^-24 in fp32).
__device__ __forceinline__ float2 cos_sin(double turn) {
  turn -= rint(turn);
  const double quarter = rint(4.0 * turn);
  const float x = 6.283185307179586f * (float)fma(-0.25, quarter, turn), y = x * x;
  float c = fmaf(y, -1.f / 3628800, 1.f / 40320), s = fmaf(y, 1.f / 362880, -1.f / 5040);
  c = fmaf(y, fmaf(y, fmaf(y, c, -1.f / 720), 1.f / 24), -0.5f);
  s = fmaf(y, fmaf(y, s, 1.f / 120), -1.f / 6);
  c = fmaf(y, c, 1.f);
  s = fmaf(x * y, s, x);
  const int q = (int)quarter & 3;
  const float u = q & 1 ? s : c, v = q & 1 ? c : s;
  return make_float2(q == 1 || q == 2 ? -u : u, q >= 2 ? -v : v);
}

// cos and sin of a tile's tokens, a column of pairs a thread, and where the tokens start.
template <bool BWD>
__device__ __forceinline__ void rope_table(const RopeArgs& A, const RopeSide& S, int t0, int nt,
                                           float2* table, int64_t (*base)[kRopeMaxTile]) {
  const int pairs = A.d / 2, turning = A.rot / 2, width = A.width, row = table_row(A.d);
  for (int p = threadIdx.x & (width - 1); p < pairs; p += width) {
    const double f = p < turning ? (double)A.inv_freq[p] * 0.15915494309189533577 : 0.0;
    for (int tok = threadIdx.x / width; tok < nt; tok += kRopeThreads / width) {
      float2 cs = make_float2(1.f, 0.f);
      if (p < turning) {
        const uint32_t b = A.seq.div(t0 + tok), n = t0 + tok - b * A.seq.d;
        const int64_t pos = A.positions ? ld_index(A.positions, A.pos_wide, b * A.pos_stride + n)
                                        : (int64_t)n;
        cs = cos_sin((double)pos * f);
        cs.x *= A.scaling;
        cs.y *= A.scaling;
      }
      table[tok * row + table_at(p)] = cs;
    }
  }
  if (threadIdx.x < nt) {
    const uint32_t b = A.seq.div(t0 + threadIdx.x), n = t0 + threadIdx.x - b * A.seq.d;
    base[0][threadIdx.x] = b * S.xs[0] + n * S.xs[1];
    base[1][threadIdx.x] = b * S.os[0] + n * S.os[1];
    if (BWD) base[2][threadIdx.x] = b * S.ys[0] + n * S.ys[1];
  }
}

// INVERSE turns back (the gradient without norms).
template <int DT, bool VEC, bool INTER, bool NORM>
__global__ __launch_bounds__(kRopeThreads) void rope_forward(const RopeArgs A, int inverse) {
  extern __shared__ float2 table[];
  __shared__ int64_t base[2][kRopeMaxTile];
  using T = typename Elem<DT>::T;
  const int k_side = blockIdx.x >= A.side[0].blocks;
  const RopeSide& S = A.side[k_side];
  const int block = blockIdx.x - (k_side ? A.side[0].blocks : 0);
  const Place at(A.lanes);
  const int row = table_row(A.d);
  const HeadLane<DT, VEC, INTER> io(at.lane, A.lanes, A.rot, A.d);
  float wa[8], wb[8];
  if (NORM) ld_weights(io, S.w, A.wdt, wa, wb);
  const int t0 = block * S.tile, nt = min(S.tile, A.tokens - t0);
  rope_table<false>(A, S, t0, nt, table, base);
  __syncthreads();
  const int items = nt * S.heads.d;
  for (int it = at.group; it < items; it += at.groups) {
    const uint32_t tok = S.heads.div(it), h = it - tok * S.heads.d;
    float a[8], b[8];
    io.ld((const T*)S.x + base[0][tok] + h * S.xs[2], a, b);
    if (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int t = 0; t < 8; ++t) ss += io.on(t) ? a[t] * a[t] + b[t] * b[t] : 0.f;
      const float rho = rsqrtf(head_sum(ss, at.lane, A.lanes) / A.d + A.eps);
#pragma unroll
      for (int t = 0; t < 8; ++t) a[t] *= rho * wa[t], b[t] *= rho * wb[t];
    }
    turn(io, table + tok * row, inverse, a, b);
    io.st((T*)S.out + base[1][tok] + h * S.os[2], a, b);
  }
}

// Four wavefronts a SIMD for the 16-bit types: 128 registers (300 columns fp16 61 -> 56 us).
template <int DT, bool VEC, bool INTER>
__global__ __launch_bounds__(kRopeThreads, VEC && DT != kF32 ? 4 : 1)
void rope_norm_backward(const RopeArgs A) {
  extern __shared__ float2 table[];
  __shared__ int64_t base[3][kRopeMaxTile];
  using T = typename Elem<DT>::T;
  // the keys first: with few heads their blocks are few and long (8192 tokens of 8 heads x
  // 256 and one: 38 us, 35 so)
  const int k_side = blockIdx.x < A.side[1].blocks;
  const RopeSide& S = A.side[k_side];
  const int block = blockIdx.x - (k_side ? 0 : A.side[1].blocks);
  const Place at(A.lanes);
  const int row = table_row(A.d);
  const HeadLane<DT, VEC, INTER> io(at.lane, A.lanes, A.rot, A.d);
  float wa[8], wb[8], da[8], db[8];
  ld_weights(io, S.w, A.wdt, wa, wb);
#pragma unroll
  for (int t = 0; t < 8; ++t) da[t] = db[t] = 0.f;
  const float inv_d = 1.f / A.d;
  for (int64_t t0 = (int64_t)block * S.tile; t0 < A.tokens; t0 += (int64_t)S.blocks * S.tile) {
    const int nt = (int)min((int64_t)S.tile, A.tokens - t0);
    rope_table<true>(A, S, (int)t0, nt, table, base);
    __syncthreads();
    const int items = nt * S.heads.d;
    for (int it = at.group; it < items; it += at.groups) {
      const uint32_t tok = S.heads.div(it), h = it - tok * S.heads.d;
      float a[8], b[8], ga[8], gb[8];
      io.ld((const T*)S.x + base[0][tok] + h * S.xs[2], a, b);
      io.ld((const T*)S.dy + base[2][tok] + h * S.ys[2], ga, gb);
      turn(io, table + tok * row, true, ga, gb);
      float ss = 0.f, sd = 0.f;
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const float xa = io.on(t) ? a[t] : 0.f, xb = io.on(t) ? b[t] : 0.f;
        ss += xa * xa + xb * xb;
        sd += ga[t] * wa[t] * xa + gb[t] * wb[t] * xb;
      }
      ss = head_sum(ss, at.lane, A.lanes);
      sd = head_sum(sd, at.lane, A.lanes);
      const float rho = rsqrtf(ss * inv_d + A.eps);
      const float m = rho * rho * (sd * inv_d);
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        da[t] += ga[t] * (a[t] * rho);
        db[t] += gb[t] * (b[t] * rho);
        a[t] = rho * (ga[t] * wa[t] - a[t] * m);
        b[t] = rho * (gb[t] * wb[t] - b[t] * m);
      }
      io.st((T*)S.out + base[1][tok] + h * S.os[2], a, b);
    }
    __syncthreads();
  }
  // the groups' sums, in their order: within a wavefront by exchange where lanes are a power
  // of two, then one row a wavefront, otherwise a group, in LDS
  float* sums = reinterpret_cast<float*>(table);
  const bool even = (A.lanes & (A.lanes - 1)) == 0;
  if (even)
    for (int o = A.lanes; o < 64; o <<= 1)
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        da[t] += __shfl_xor(da[t], o);
        db[t] += __shfl_xor(db[t], o);
      }
  const int rows = even ? kRopeThreads / 64 : at.groups;
  if (even ? (threadIdx.x & 63) < A.lanes : at.group < at.groups) {
    float* mine = sums + (even ? (int)threadIdx.x >> 6 : at.group) * A.d;
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (io.on(t)) {
        mine[io.col_a(io.pair(t))] = da[t];
        mine[io.col_b(io.pair(t))] = db[t];
      }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < A.d; j += kRopeThreads) {
    float s = 0.f;
#pragma unroll 4
    for (int r = 0; r < rows; ++r) s += sums[r * A.d + j];
    S.partial[(int64_t)block * A.d + j] = s;
  }
}

// dw[j] = the blocks' partial sums, 16 columns a block, 64 threads each.
__global__ __launch_bounds__(kSumThreads) void rope_weight_sums(const float* pq, int nq, void* dwq,
                                                                const float* pk, int nk, void* dwk,
                                                                int d, int wdt) {
  __shared__ float part[kSumThreads / 16][17];
  const float* p = blockIdx.y ? pk : pq;
  const int n = blockIdx.y ? nk : nq;
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, j = min((int)blockIdx.x * 16 + c, d - 1);
  float s[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) s[u] = 0.f;
  for (int i = r; i < n; i += 512) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = p[(int64_t)min(i + 64 * u, n - 1) * d + j];
#pragma unroll
    for (int u = 0; u < 8; ++u) s[u] += i + 64 * u < n ? v[u] : 0.f;
  }
  part[r][c] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  // 16 columns' 64 sums: four lanes a column, then those four
  if (threadIdx.x < 64) {
    float t = 0.f;
#pragma unroll
    for (int u = 0; u < 16; ++u) t += part[(threadIdx.x >> 4) * 16 + u][c];
    t += __shfl_xor(t, 16);
    t += __shfl_xor(t, 32);
    if (threadIdx.x < 16 && (int)blockIdx.x * 16 + c < d)
      st_any(blockIdx.y ? dwk : dwq, wdt, j, t);
  }
}

int pow2_at_least(int n) {
  int l = 1;
  while (l < n) l <<= 1;
  return l;
}

// Eights of a head's pairs: in halves those that turn and the others apart.
int rope_eights(int64_t d, int64_t rot, bool inter) {
  return (int)(inter ? (d / 2 + 7) / 8 : (rot / 2 + 7) / 8 + ((d - rot) / 2 + 7) / 8);
}
// Whether a head moves 16 bytes at a time: eight pairs of a kind at least, and a lane each.
bool rope_vec(int64_t d, int64_t rot, bool inter) {
  return (inter ? d >= 16 : rot >= 16 && (d == rot || d - rot >= 16)) &&
         rope_eights(d, rot, inter) <= 64;
}
// Where the eights leave lanes of a power of two idle and more heads fit a wavefront
// without, they are the lanes (8192 x 40 x 80 bf16, gradient: 43 us, 49 with 8 lanes for 5;
// 4000 x 24 x 300 fp16 forward 24.5 and 29).
int rope_lanes(int64_t d, int64_t rot, bool inter) {
  if (!rope_vec(d, rot, inter)) return pow2_at_least((int)((d / 2 + 7) / 8));
  const int eights = rope_eights(d, rot, inter), even = pow2_at_least(eights);
  return 64 / eights > 64 / even ? eights : even;
}

// Tokens a tile: as many as give every group of the block a head, and up to four times that
// as far as the table holds: forward where there are 1024 blocks a side all the same,
// backward, where a block's start and end cost as much as two heads a group and the
// chip holds 1024, where there are more than 1024 of both sides.  (3009 tokens of 12 and
// 3 heads x 80 fp32: gradient 20 us, 22.5 by the forward's rule, 28 where a block had no
// regard to its groups.)
int rope_tile(int64_t tokens, int64_t heads, int64_t all_heads, int64_t d, int lanes,
              bool backward) {
  const int64_t groups = 64 / lanes * (kRopeThreads / 64);
  const int64_t once = std::max<int64_t>(1, groups / heads);
  const int64_t full = backward ? (tokens * all_heads + groups * 1024 - 1) / (groups * 1024)
                                : tokens / (once * 1024);
  const int64_t rounds = std::min<int64_t>(4, std::max<int64_t>(1, full));
  const int64_t most = std::min<int64_t>(kRopeTableBytes / (8 * table_row((int)d)), kRopeMaxTile);
  return (int)std::max<int64_t>(1, std::min(std::min(once * rounds, most), tokens));
}

int64_t rope_blocks(int64_t tokens, int tile) { return (tokens + tile - 1) / tile; }
// The backward's, which loop over tiles: kRopeBlocks by the sides' heads.
int64_t rope_blocks_bounded(int64_t tokens, int tile, int64_t heads, int64_t all_heads) {
  return std::min(rope_blocks(tokens, tile),
                  std::max<int64_t>(1, kRopeBlocks * heads / all_heads));
}

int rope_check(int dtype, int wdt, int64_t batch, int64_t seq, int64_t hq, int64_t hk, int64_t d,
               int64_t rot) {
  if (dtype < 0 || dtype > 2 || (wdt != dtype && wdt != kF32)) return kErrDType;
  if (batch < 0 || seq < 0 || hq < 0 || hk < 0 || d < 2 || d % 2 || rot < 2 || rot % 2 || rot > d)
    return kErrShape;
  if (d > 1024 || hq > 65536 || hk > 65536) return kErrTooLarge;
  if (seq > 0 && batch > ((1ll << 30) - 1) / seq) return kErrTooLarge;
  return kOk;
}

RopeSide rope_side(const void* x, const int64_t* xs, const void* dy, const int64_t* ys, void* out,
                   const int64_t* os, const void* w, int64_t heads) {
  RopeSide s{};
  s.x = x, s.dy = dy, s.out = out, s.w = w;
  for (int i = 0; i < 3; ++i) {
    s.xs[i] = xs[i];
    s.ys[i] = ys ? ys[i] : 0;
    s.os[i] = os[i];
  }
  s.heads = FastDivU32::make((uint32_t)std::max<int64_t>(heads, 1));
  return s;
}

template <int DT>
int launch_forward(const RopeArgs& A, bool vec, bool inter, bool norm, int inverse, size_t lds,
                   hipStream_t st) {
  const int grid = A.side[0].blocks + A.side[1].blocks;
#define CPT_ROPE(V, I, N) \
  rope_forward<DT, V, I, N><<<grid, kRopeThreads, lds, st>>>(A, inverse)
  if (vec) {
    if (inter) { if (norm) CPT_ROPE(true, true, true); else CPT_ROPE(true, true, false); }
    else { if (norm) CPT_ROPE(true, false, true); else CPT_ROPE(true, false, false); }
  } else {
    if (inter) { if (norm) CPT_ROPE(false, true, true); else CPT_ROPE(false, true, false); }
    else { if (norm) CPT_ROPE(false, false, true); else CPT_ROPE(false, false, false); }
  }
#undef CPT_ROPE
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

template <int DT>
int launch_backward(const RopeArgs& A, bool vec, bool inter, size_t lds, hipStream_t st) {
  const int grid = A.side[0].blocks + A.side[1].blocks;
#define CPT_ROPE(V, I) rope_norm_backward<DT, V, I><<<grid, kRopeThreads, lds, st>>>(A)
  if (vec) { if (inter) CPT_ROPE(true, true); else CPT_ROPE(true, false); }
  else { if (inter) CPT_ROPE(false, true); else CPT_ROPE(false, false); }
#undef CPT_ROPE
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // namespace qkrope
}  // namespace cpt

using namespace cpt;
using namespace cpt::qkrope;

extern "C" {

int cpt_qk_rope(int dtype, int weight_dtype, int interleaved, int inverse, const void* q,
                int64_t q_batch, int64_t q_token, int64_t q_head, const void* k, int64_t k_batch,
                int64_t k_token, int64_t k_head, const void* w_q, const void* w_k,
                const void* positions, int pos_wide, int64_t pos_batch, const void* inv_freq,
                int64_t batch, int64_t seq, int64_t heads_q, int64_t heads_k, int64_t d,
                int64_t rotary, float eps, float scaling, void* q_out, int64_t qo_batch,
                int64_t qo_token, int64_t qo_head, void* k_out, int64_t ko_batch, int64_t ko_token,
                int64_t ko_head, void* stream) {
  const int rc = rope_check(dtype, weight_dtype, batch, seq, heads_q, heads_k, d, rotary);
  if (rc) return rc;
  if ((w_q == nullptr) != (w_k == nullptr) || (w_q && inverse) || !inv_freq || !(eps >= 0.f))
    return kErrShape;
  const int64_t tokens = batch * seq;
  if (tokens == 0 || heads_q + heads_k == 0) return kOk;
  if ((heads_q && (!q || !q_out)) || (heads_k && (!k || !k_out))) return kErrShape;
  RopeArgs A{};
  const int64_t xq[3] = {q_batch, q_token, q_head}, xk[3] = {k_batch, k_token, k_head};
  const int64_t oq[3] = {qo_batch, qo_token, qo_head}, ok[3] = {ko_batch, ko_token, ko_head};
  A.side[0] = rope_side(q, xq, nullptr, nullptr, q_out, oq, w_q, heads_q);
  A.side[1] = rope_side(k, xk, nullptr, nullptr, k_out, ok, w_k, heads_k);
  const int64_t heads[2] = {heads_q, heads_k};
  int most = 1;
  for (int i = 0; i < 2; ++i) {
    A.side[i].tile = rope_tile(tokens, std::max<int64_t>(heads[i], 1), heads_q + heads_k, d,
                               rope_lanes(d, rotary, interleaved), false);
    A.side[i].blocks = heads[i] ? (int)rope_blocks(tokens, A.side[i].tile) : 0;
    if (heads[i]) most = std::max(most, A.side[i].tile);
  }
  A.positions = positions, A.pos_wide = pos_wide, A.pos_stride = pos_batch;
  A.inv_freq = (const float*)inv_freq;
  A.seq = FastDivU32::make((uint32_t)seq);
  A.tokens = (int)tokens, A.d = (int)d, A.rot = (int)rotary;
  A.lanes = rope_lanes(d, rotary, interleaved);
  A.width = std::min(kRopeThreads, pow2_at_least((int)d / 2));
  A.wdt = weight_dtype, A.eps = eps, A.scaling = scaling;
  const size_t lds = (size_t)most * table_row((int)d) * 8;
  const bool vec = rope_vec(d, rotary, interleaved), norm = w_q != nullptr;
  const hipStream_t st = (hipStream_t)stream;
  if (dtype == kF32) return launch_forward<kF32>(A, vec, interleaved, norm, inverse, lds, st);
  if (dtype == kF16) return launch_forward<kF16>(A, vec, interleaved, norm, inverse, lds, st);
  return launch_forward<kBF16>(A, vec, interleaved, norm, inverse, lds, st);
}

int64_t cpt_qk_rope_backward_workspace_bytes(int64_t tokens, int64_t heads_q, int64_t heads_k,
                                             int64_t d) {
  if (tokens < 0 || heads_q < 0 || heads_k < 0 || d < 2 || d > 1024 || tokens >= 1ll << 30)
    return -1;
  if (tokens == 0 || heads_q == 0 || heads_k == 0) return 0;
  // a token a tile at the least
  const int64_t all = heads_q + heads_k;
  return (rope_blocks_bounded(tokens, 1, heads_q, all) +
          rope_blocks_bounded(tokens, 1, heads_k, all)) *
         d * 4;
}

int cpt_qk_rope_backward(int dtype, int weight_dtype, int interleaved, const void* d_q,
                         int64_t dq_batch, int64_t dq_token, int64_t dq_head, const void* d_k,
                         int64_t dk_batch, int64_t dk_token, int64_t dk_head, const void* q,
                         int64_t q_batch, int64_t q_token, int64_t q_head, const void* k,
                         int64_t k_batch, int64_t k_token, int64_t k_head, const void* w_q,
                         const void* w_k, const void* positions, int pos_wide, int64_t pos_batch,
                         const void* inv_freq, int64_t batch, int64_t seq, int64_t heads_q,
                         int64_t heads_k, int64_t d, int64_t rotary, float eps, float scaling,
                         void* q_grad, void* k_grad, void* dw_q, void* dw_k, void* workspace,
                         void* stream) {
  const int rc = rope_check(dtype, weight_dtype, batch, seq, heads_q, heads_k, d, rotary);
  if (rc) return rc;
  const int64_t tokens = batch * seq;
  if (!w_q || !w_k || !dw_q || !dw_k || !inv_freq || !(eps >= 0.f)) return kErrShape;
  if (tokens == 0 || heads_q == 0 || heads_k == 0) return kErrShape;
  if (!q || !k || !d_q || !d_k || !q_grad || !k_grad || !workspace) return kErrShape;
  RopeArgs A{};
  const int64_t xq[3] = {q_batch, q_token, q_head}, xk[3] = {k_batch, k_token, k_head};
  const int64_t yq[3] = {dq_batch, dq_token, dq_head}, yk[3] = {dk_batch, dk_token, dk_head};
  const int64_t oq[3] = {seq * heads_q * d, heads_q * d, d};
  const int64_t ok[3] = {seq * heads_k * d, heads_k * d, d};
  A.side[0] = rope_side(q, xq, d_q, yq, q_grad, oq, w_q, heads_q);
  A.side[1] = rope_side(k, xk, d_k, yk, k_grad, ok, w_k, heads_k);
  const int64_t heads[2] = {heads_q, heads_k};
  float* ws = (float*)workspace;
  int most = 1;
  for (int i = 0; i < 2; ++i) {
    RopeSide& s = A.side[i];
    s.tile = rope_tile(tokens, heads[i], heads_q + heads_k, d, rope_lanes(d, rotary, interleaved),
                       true);
    s.blocks = (int)rope_blocks_bounded(tokens, s.tile, heads[i], heads_q + heads_k);
    s.partial = ws;
    ws += (int64_t)s.blocks * d;
    most = std::max(most, s.tile);
  }
  A.positions = positions, A.pos_wide = pos_wide, A.pos_stride = pos_batch;
  A.inv_freq = (const float*)inv_freq;
  A.seq = FastDivU32::make((uint32_t)seq);
  A.tokens = (int)tokens, A.d = (int)d, A.rot = (int)rotary;
  A.lanes = rope_lanes(d, rotary, interleaved);
  A.width = std::min(kRopeThreads, pow2_at_least((int)d / 2));
  A.wdt = weight_dtype, A.eps = eps, A.scaling = scaling;
  // the table, and at the end the sums of the wavefronts, or groups, in its place
  const bool even = (A.lanes & (A.lanes - 1)) == 0;
  const size_t rows = even ? 4 : 64 / A.lanes * 4;
  const size_t lds = std::max<size_t>((size_t)most * table_row((int)d) * 8, rows * d * 4);
  const bool vec = rope_vec(d, rotary, interleaved);
  const hipStream_t st = (hipStream_t)stream;
  const int err = dtype == kF32   ? launch_backward<kF32>(A, vec, interleaved, lds, st)
                  : dtype == kF16 ? launch_backward<kF16>(A, vec, interleaved, lds, st)
                                  : launch_backward<kBF16>(A, vec, interleaved, lds, st);
  if (err) return err;
  rope_weight_sums<<<dim3((unsigned)((d + 15) / 16), 2), kSumThreads, 0, st>>>(
      A.side[0].partial, A.side[0].blocks, dw_q, A.side[1].partial, A.side[1].blocks, dw_k, (int)d,
      weight_dtype);
  return hipGetLastError() == hipSuccess ? kOk : kErrLaunch;
}

}  // extern "C"
