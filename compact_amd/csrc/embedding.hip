// Embedding lookup with a scale, and its gradient by sorted tokens.
//
//   out[n] = scale W[id_n]                     (an id outside the table: zeros)
//   dW[v]  = scale sum_{n: id_n = v} dy[n]     (v != padding_idx)
//
// The lookup is HBM-bound: one thread per eight columns.
//
// The gradient adds no floats atomically.  The tokens' (id, position) pairs are
// sorted by id with their order kept, so one id's tokens lie side by side in the
// order of the batch: up to 32768 tokens in one launch, each of 32 blocks sorting a
// range of ids in LDS; beyond by a radix sort of 8 bits a pass (a block ranks 2048
// pairs by ballots).  The table's zeros are written by further blocks of the same
// launches: sorting is latency and compares, the zeros are HBM.  The sorted list is
// cut into tiles of equal length, whatever ids they hold, so a frequent token's rows
// are spread over as many wavefronts as it needs; sums of an id over several tiles
// are joined in tile order.  The result is the same from run to run.  Bound by HBM:
// dy is read once, the table written once (rows with tokens twice).
//
// Measured on one MI355X: the lookup of 8192 x 2048 bf16 9.8 us (4.6 TB/s), its
// gradient into 32000 rows 43 (3.7 TB/s of what it must read and write; 35 where dy
// lies in the Infinity Cache), of 65536 tokens 118.  The sums take 11 us of the first,
// 71 of the second, at 4.3 TB/s; the second's three launches of the sort 37.

#include "compact_amd.h"
#include "row_ops.h"

namespace cpt {
namespace embed {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
constexpr int kItems = 8;                    // pairs per thread of a sort block
constexpr int kSortTile = kBlock * kItems;
constexpr int kRadix = 256;
constexpr int kCols = 512;                   // columns of a wavefront

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------

template <int DT>
__global__ __launch_bounds__(kBlock) void lookup_kernel(const void* __restrict__ weight,
                                                        int64_t vocab, int64_t d,
                                                        const void* __restrict__ ids, int wide,
                                                        int64_t id0, uint32_t total,
                                                        FastDivU32 per_row, float scale,
                                                        void* __restrict__ out) {
  using R = Row8<DT>;
  using T = typename R::T;
  const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
  if (i >= total) return;
  const uint32_t r = per_row.div(i);
  const int64_t j = 8 * (int64_t)(i - r * per_row.d);
  const int64_t n = id0 + r, id = ld_index(ids, wide, n);
  typename R::Raw q = R::zero();
  if (id >= 0 && id < vocab) {
    q = row_ld<DT>((const T*)weight + id * d, j, d, 0);
    if (scale != 1.f) {
      float v[8];
      R::unpack(q, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= scale;
      q = R::pack(v);
    }
  }
  row_st<DT>((T*)out + n * d, j, d, q);
}

// ---------------------------------------------------------------------------
// sort
// ---------------------------------------------------------------------------

struct Pair {
  uint32_t id, pos;
};

// The key of a token: its id, or `vocab` (sorted last, never summed) for padding
// and ids outside the table.
__device__ __forceinline__ uint32_t token_key(const void* ids, int wide, int64_t n, int64_t vocab,
                                              int64_t padding) {
  const int64_t id = ld_index(ids, wide, n);
  return id >= 0 && id < vocab && id != padding ? (uint32_t)id : (uint32_t)vocab;
}

// The share of the table's zeros that a launch of the sort writes beside it, in
// blocks past its own.
struct Zeros {
  void* out;
  int64_t begin, end;   // elements, of a row type
  unsigned first;       // block
};
template <int OT>
__device__ __forceinline__ bool zeros_here(const Zeros& z) {
  if (blockIdx.x < z.first) return false;
  using R = Row8<OT>;
  const int64_t step = (int64_t)(gridDim.x - z.first) * blockDim.x * 8;
  int64_t i = z.begin + 8 * ((int64_t)(blockIdx.x - z.first) * blockDim.x + threadIdx.x);
  for (; i < z.end; i += step) row_st<OT>((typename R::T*)z.out, i, z.end, R::zero());
  return true;
}

// counts[block][digit] of the pairs' digit (key >> shift) & 255 (of the tokens
// themselves where `in` is null), and zeros for the `later` passes' counts.
template <int OT>
__global__ __launch_bounds__(kBlock) void count_kernel(const Pair* __restrict__ in,
                                                       const void* __restrict__ ids, int wide,
                                                       int64_t n, int64_t vocab, int64_t padding,
                                                       int shift, uint32_t* __restrict__ counts,
                                                       unsigned blocks, int later, Zeros zeros) {
  __shared__ uint32_t hist[kRadix];
  if (zeros_here<OT>(zeros)) return;
  hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kSortTile;
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = i0 + k * kBlock + threadIdx.x;
    if (i >= n) continue;
    const uint32_t key = in ? in[i].id : token_key(ids, wide, i, vocab, padding);
    atomicAdd(&hist[(key >> shift) & (kRadix - 1)], 1u);
  }
  __syncthreads();
  for (int p = 0; p <= later; ++p)
    counts[((int64_t)p * blocks + blockIdx.x) * kRadix + threadIdx.x] =
        p == 0 ? hist[threadIdx.x] : 0;
}

// One pass of the sort: pairs of `in` (the tokens themselves in the first) to
// their places by digit (key >> shift) & 255, equal digits in their order.  `next`
// (or null) takes the next digit's counts of the blocks that the pairs move to:
// gathered in LDS (1 KiB a block), as a frequent token's pairs all add to one.
template <int OT>
__global__ __launch_bounds__(kBlock) void scatter_kernel(const Pair* __restrict__ in,
                                                         const void* __restrict__ ids, int wide,
                                                         int64_t n, int64_t vocab, int64_t padding,
                                                         int shift,
                                                         const uint32_t* __restrict__ counts,
                                                         unsigned blocks, uint32_t* next,
                                                         Pair* __restrict__ out, Zeros zeros) {
  extern __shared__ uint32_t moved[];   // [blocks][digit]
  __shared__ uint32_t wave_count[kWaves][kRadix];
  __shared__ uint32_t base[kRadix];
  __shared__ uint32_t scan[kWaves];
  if (zeros_here<OT>(zeros)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int w = 0; w < kWaves; ++w) wave_count[w][tid] = 0;
  if (next)
    for (unsigned b = 0; b < blocks; ++b) moved[b * kRadix + tid] = 0;
  __syncthreads();
  // a wavefront ranks 512 consecutive pairs, 64 at a time
  const int64_t i0 = (int64_t)blockIdx.x * kSortTile + wave * (kSortTile / kWaves) + lane;
  Pair q[kItems];
  uint32_t rank[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = i0 + k * 64;
    q[k] = Pair{0, 0};
    if (i < n) q[k] = in ? in[i] : Pair{token_key(ids, wide, i, vocab, padding), (uint32_t)i};
  }
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const bool live = i0 + k * 64 < n;
    const uint32_t digit = (q[k].id >> shift) & (kRadix - 1);
    uint64_t same = __ballot(live);
#pragma unroll
    for (int bit = 0; bit < 8; ++bit) {
      const uint64_t set = __ballot((digit >> bit) & 1);
      same &= (digit >> bit) & 1 ? set : ~set;
    }
    const uint64_t below = same & ((1ull << lane) - 1);
    const uint32_t before = live ? wave_count[wave][digit] : 0;
    rank[k] = before + __popcll(below);
    // the wavefront's accesses to its own counters stay in order: read, then written
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (live && below == 0) wave_count[wave][digit] = before + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // thread t: where digit t starts for this block
  uint32_t total = 0, mine = 0;
#pragma unroll 8
  for (unsigned b = 0; b < blocks; ++b) {
    const uint32_t c = counts[(int64_t)b * kRadix + tid];
    mine += b < blockIdx.x ? c : 0;
    total += c;
  }
  uint32_t inc = total;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t u = __shfl_up(inc, off);
    if (lane >= off) inc += u;
  }
  if (lane == 63) scan[wave] = inc;
  __syncthreads();
  uint32_t at = inc - total + mine;
  for (int w = 0; w < wave; ++w) at += scan[w];
  base[tid] = at;
  uint32_t run = 0;
  for (int w = 0; w < kWaves; ++w) {
    const uint32_t c = wave_count[w][tid];
    wave_count[w][tid] = run;
    run += c;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    if (i0 + k * 64 >= n) continue;
    const uint32_t digit = (q[k].id >> shift) & (kRadix - 1);
    const uint32_t to = base[digit] + wave_count[wave][digit] + rank[k];
    out[to] = q[k];
    if (next)
      atomicAdd(&moved[to / kSortTile * kRadix + (q[k].id >> (shift + 8) & (kRadix - 1))], 1u);
  }
  if (!next) return;
  __syncthreads();
  for (unsigned b = 0; b < blocks; ++b) {
    const uint32_t c = moved[b * kRadix + tid];
    if (c) atomicAdd(&next[(int64_t)b * kRadix + tid], c);
  }
}

// The sort of up to 32768 tokens in one launch.  Each of 32 blocks takes a range of
// ids: it reads all tokens into registers, counts those below its range and packs
// those inside, in their order, into LDS as (id - first id) << 15 | position; sorts
// them there by the id's bits in stable passes of up to 8; and writes them behind the
// tokens of the ranges below.  Tokens that are summed nowhere fill the list's end.  Bound by
// latency and, in the reading of all tokens by each block, by the vector pipe: 18 us
// at 8192 tokens beside 131 MB of zeros (which alone take 20), 16 at 20011 (20 where
// the tokens are read a second time to be packed).  The whole gradient, dy in the
// Infinity Cache, against the radix sort's three launches: 8192 tokens into 32000 x
// 2048 bf16 35 and 48 us, 16000 into 5000 x 1000 31 and 37, 20011 x 1001 fp32 43 and
// 52, 32768 into 32000 x 2048 82 and 84.
constexpr int kRanges = 32;
constexpr int kRangeThreads = 1024;
constexpr int kRangeWaves = kRangeThreads / 64;
constexpr int kPosBits = 15;
constexpr int kRangeRounds = (1 << kPosBits) / kRangeThreads;   // of 64 tokens a wavefront

template <int OT>
__global__ __launch_bounds__(kRangeThreads) void range_sort_kernel(
    const void* __restrict__ ids, int wide, int n, uint32_t vocab, int64_t padding, uint32_t span,
    int bits, Pair* __restrict__ out, Zeros zeros) {
  extern __shared__ uint32_t list[];   // [n]
  __shared__ uint16_t count[kRangeWaves][kRadix];
  __shared__ uint32_t base[kRadix], tmp[2][kRangeWaves];
  if (zeros_here<OT>(zeros)) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t lo = min(blockIdx.x * span, vocab), width_in = min(span, vocab - lo);
  const uint64_t lower = (1ull << lane) - 1;
  // a wavefront has consecutive tokens, 64 at a time; one compare each tells what lies
  // inside the range and below it (a negative id of 32 bits is above every other)
  int each = (n + kRangeThreads - 1) / kRangeThreads * 64, i0 = wave * each;
  const int i1 = min(n, i0 + each);
  constexpr int kAhead = 16;
  const uint32_t pad = padding >= 0 ? (uint32_t)padding : ~0u;
  uint32_t key[kRangeRounds];
  uint32_t inside = 0, below = 0;
#pragma unroll
  for (int h = 0; h < kRangeRounds; h += kAhead) {
    if (i0 + 64 * h >= i1) break;
    uint32_t top[kAhead];
    if (wide) {
#pragma unroll
      for (int t = 0; t < kAhead; ++t) {
        const uint2 id =
            reinterpret_cast<const uint2*>(ids)[min(i0 + 64 * (h + t) + lane, n - 1)];
        key[h + t] = id.x, top[t] = id.y;
      }
    } else {
#pragma unroll
      for (int t = 0; t < kAhead; ++t) {
        key[h + t] = reinterpret_cast<const uint32_t*>(ids)[min(i0 + 64 * (h + t) + lane, n - 1)];
        top[t] = 0;
      }
    }
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      uint32_t& k = key[h + t];
      if (top[t] != 0 || i0 + 64 * (h + t) + lane >= i1 || k == pad) k = ~0u;
      inside += __popcll(__ballot(k - lo < width_in));
      below += __popcll(__ballot(k < lo));
    }
  }
  if (lane == 0) tmp[0][wave] = inside, tmp[1][wave] = below;
  __syncthreads();
  int to = 0, m = 0, first = 0;
  for (int w = 0; w < kRangeWaves; ++w) {
    to += w < wave ? tmp[0][w] : 0;
    m += tmp[0][w];
    first += tmp[1][w];
  }
#pragma unroll
  for (int t = 0; t < kRangeRounds; ++t) {
    if (i0 + 64 * t >= i1) break;
    const bool in = key[t] - lo < width_in;
    const uint64_t mask = __ballot(in);
    if (in) list[to + __popcll(mask & lower)] = (key[t] - lo) << kPosBits | (i0 + 64 * t + lane);
    to += __popcll(mask);
  }
  // stable passes over the packed list, its pairs in registers between LDS and LDS
  each = (m + kRangeThreads - 1) / kRangeThreads * 64, i0 = wave * each;
  const int rounds = each / 64;
  const int passes = (bits + 7) / 8, width = passes > 0 ? (bits + passes - 1) / passes : 0;
  for (int p = 0; p < passes; ++p) {
    const int shift = kPosBits + p * width;
    for (int c = tid; c < kRangeWaves * kRadix / 2; c += kRangeThreads)
      reinterpret_cast<uint32_t*>(&count[0][0])[c] = 0;
    __syncthreads();
    uint32_t q[kRangeRounds], rank[kRangeRounds];
#pragma unroll
    for (int r = 0; r < kRangeRounds; ++r) {
      if (r >= rounds) break;
      const int i = i0 + 64 * r + lane;
      const bool live = i < m;
      q[r] = live ? list[i] : 0;
      const uint32_t digit = q[r] >> shift & ((1u << width) - 1);
      uint64_t same = __ballot(live);
      for (int b = 0; b < width; ++b) {
        const uint64_t set = __ballot(digit >> b & 1);
        same &= digit >> b & 1 ? set : ~set;
      }
      const uint32_t before = live ? count[wave][digit] : 0;
      rank[r] = before + __popcll(same & lower);
      // the wavefront's accesses to its own counters stay in order: read, then written
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (live && (same & lower) == 0) count[wave][digit] = (uint16_t)(before + __popcll(same));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    // thread d: digit d's pairs by wavefront, and where they start
    uint32_t total = 0, upto = 0;
    if (tid < kRadix) {
      for (int w = 0; w < kRangeWaves; ++w) {
        const uint32_t c = count[w][tid];
        count[w][tid] = (uint16_t)total;
        total += c;
      }
      upto = total;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const uint32_t u = __shfl_up(upto, off);
        if (lane >= off) upto += u;
      }
      if (lane == 63) tmp[0][wave] = upto;
    }
    __syncthreads();
    if (tid < kRadix) {
      for (int w = 0; w < wave; ++w) upto += tmp[0][w];
      base[tid] = upto - total;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRangeRounds; ++r) {
      if (r >= rounds) break;
      if (i0 + 64 * r + lane >= m) continue;
      const uint32_t digit = q[r] >> shift & ((1u << width) - 1);
      list[base[digit] + count[wave][digit] + rank[r]] = q[r];
    }
    __syncthreads();
  }
  if (passes == 0) __syncthreads();
  for (int i = tid; i < m; i += kRangeThreads)
    out[first + i] = Pair{lo + (list[i] >> kPosBits), list[i] & ((1u << kPosBits) - 1)};
  if (blockIdx.x == kRanges - 1)
    for (int i = first + m + tid; i < n; i += kRangeThreads) out[i] = Pair{vocab, 0};
}

// ---------------------------------------------------------------------------
// sums
// ---------------------------------------------------------------------------

// Zeros over the whole table.
template <int DT>
__global__ __launch_bounds__(kBlock) void zero_kernel(void* out, int64_t total) {
  using R = Row8<DT>;
  const int64_t stride = (int64_t)gridDim.x * kBlock * 8;
  for (int64_t i = 8 * ((int64_t)blockIdx.x * kBlock + threadIdx.x); i < total; i += stride)
    row_st<DT>((typename R::T*)out, i, total, R::zero());
}

template <int OT, bool TINY, bool ADD>
__device__ __forceinline__ void write_row(void* out, int64_t v, const Cols<OT, TINY>& cols,
                                          int64_t d, float scale, const float acc[8]) {
  using R = Row8<OT>;
  typename R::T* row = (typename R::T*)out + v * d;
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = acc[e] * scale;
  if (ADD) {
    float o[8];
    R::unpack(cols.ld(row), o);
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] += o[e];
    cols.st_own(row, R::pack(r));
  } else {
    cols.st(row, R::pack(r));
  }
}

// A wavefront sums 512 columns of the ids that begin in one tile of TILE sorted
// tokens.  The tile's last id is followed to its end if that lies in the next
// tile (which then leaves it out): 2 TILE pairs, one a lane.  An id that goes on
// further is summed tile by tile; `edge` (fp32 [tiles][2][d]) takes the sums of
// the tile that it begins in (1) and of those that it runs on into (0).
constexpr int kAhead = 4;   // rows loaded while as many are added

template <int DT, int OT, bool TINY, bool ADD, int TILE>
__global__ __launch_bounds__(kBlock) void sum_kernel(const void* __restrict__ grad, int64_t ld,
                                                     const Pair* __restrict__ pairs, int64_t n,
                                                     int64_t vocab, int64_t d, unsigned strips,
                                                     float scale, void* out, float* edge) {
  using R = Row8<DT>;
  using T = typename R::T;
  const int lane = threadIdx.x & 63;
  const uint32_t unit = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = unit / strips, i0 = t * TILE;
  const int64_t j = (unit - t * strips) * kCols + 8 * lane;
  if (i0 >= n) return;
  const Cols<DT, TINY> cols(j, d);
  const Cols<OT, TINY> to(j, d);
  const Cols<kF32, TINY> sums(j, d);
  const uint32_t none = (uint32_t)vocab;
  const Pair p = lane < 2 * TILE && i0 + lane < n ? pairs[i0 + lane] : Pair{none, 0};
  const uint32_t first = __builtin_amdgcn_readfirstlane(p.id);
  if (first == none) return;
  // three ids around the tile, each in its lane (none where there is no such pair)
  const int64_t beside = lane == 0 ? i0 - 1 : lane == 1 ? i0 - TILE - 1 : i0 + 2 * TILE;
  const uint32_t around = beside >= 0 && beside < n ? pairs[beside].id : none;
  const bool entered = __builtin_amdgcn_readlane(around, 0) == first;
  const bool older = __builtin_amdgcn_readlane(around, 1) == first;   // than the last tile
  const uint32_t far = __builtin_amdgcn_readlane(around, 2);
  const int live = __popcll(__ballot(p.id != none));
  const int run = __popcll(__ballot(p.id == first));
  int begin = 0, end = live < TILE ? live : TILE;
  bool head = false, tail = false;   // of an id that goes over further tiles
  if (entered) {
    if (!older && run <= TILE) {
      begin = run;                   // the last tile has it whole
    } else {
      head = true;
    }
  }
  if (live > TILE && !(entered && run > TILE)) {
    const uint32_t id = __builtin_amdgcn_readlane(p.id, TILE - 1);
    const int upto = __popcll(__ballot(p.id <= id));
    if (upto > TILE) {
      if (upto == 2 * TILE && far == id)
        tail = true;
      else
        end = upto;
    }
  }
  if (begin >= end) return;
  const uint32_t before = __shfl_up(p.id, 1);
  const uint64_t starts = __ballot(lane > 0 && p.id != before);
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  typename R::Raw q[2][kAhead];
  const auto load = [&](int k0, typename R::Raw (&r)[kAhead]) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      // past the end: the last row again, not added
      const uint32_t pos = __builtin_amdgcn_readlane(p.pos, min(k0 + k, end - 1));
      r[k] = cols.ld((const T*)grad + (int64_t)pos * ld);
    }
  };
  const auto add = [&](int k0, const typename R::Raw (&r)[kAhead]) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int at = k0 + k;
      if (at >= end) break;
      float v[8];
      R::unpack(r[k], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += v[e];
      const bool stop = at + 1 == end;
      if (!stop && !(starts >> (at + 1) & 1)) continue;
      if ((stop && tail) || (head && at < run))
        sums.st(edge + (2 * t + (head && at < run ? 0 : 1)) * d, Row8<kF32>::pack(acc));
      else
        write_row<OT, TINY, ADD>(out, __builtin_amdgcn_readlane(p.id, at), to, d, scale, acc);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    }
  };
  load(begin, q[0]);
  for (int k = begin; k < end; k += 2 * kAhead) {
    load(k + kAhead, q[1]);
    add(k, q[0]);
    load(k + 2 * kAhead, q[0]);
    add(k + kAhead, q[1]);
  }
}

// The ids that go over three tiles or more.  A block looks at four tiles, and for
// each such id that begins in one of them adds the tiles' sums of 512 columns:
// each wavefront a part of the tiles, then the parts in order.
constexpr int kJoinTiles = 4;
constexpr int kJoinThreads = 512;
// Sums loaded together, and added without a branch: one that left the loop would
// draw each load behind it, to be waited for by itself (90000 x 100 bf16 55 us, 50
// so; 4 together 50.5).
constexpr int kJoinAhead = 8;

template <int OT, bool TINY, bool ADD, int TILE>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const Pair* __restrict__ pairs, int64_t n,
                                                      int64_t vocab, int64_t d, float scale,
                                                      void* out, const float* __restrict__ edge) {
  constexpr int kParts = kJoinThreads / 64;
  __shared__ float part[kParts][8][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t j = (int64_t)blockIdx.y * kCols + 8 * lane;
  const Cols<OT, TINY> to(j, d);
  const Cols<kF32, TINY> sums(j, d);
  uint32_t id = 0;
  bool is = false;
  {
    const int64_t i = ((int64_t)blockIdx.x * kJoinTiles + (lane & (kJoinTiles - 1))) * TILE;
    const auto at = [&](int64_t k) { return pairs[min(max(k, (int64_t)0), n - 1)].id; };
    const uint32_t before = at(i - 1), head = at(i), end = at(i + TILE - 1), far = at(i + 2 * TILE);
    id = at(i + TILE);
    is = (lane < kJoinTiles) & (i + 2 * TILE < n) & (id != (uint32_t)vocab) & (end == id) &
         (far == id) & !((head == id) & (i > 0) & (before == id));
  }
  for (uint64_t heads = __ballot(is); heads; heads &= heads - 1) {
    const int h = __builtin_ctzll(heads);
    const int64_t t0 = (int64_t)blockIdx.x * kJoinTiles + h;
    const uint32_t v = __builtin_amdgcn_readlane(id, h);
    // the last tile that begins with the id: 64 tiles looked at together, and of a
    // long run every 64th of 4096, beyond every 4096th
    int64_t last = t0 + 2;
    const auto runs_to = [&](int64_t step) {
      const int64_t i = (last + (lane + 1) * step) * TILE;
      const uint32_t there = pairs[min(n - 1, i)].id;
      return (there == v) & (i < n);
    };
    const auto reach = [&](bool in, int64_t step) {
      const int r = __popcll(__ballot(in));
      last += r * step;
      return r;
    };
    const bool near = runs_to(1), far = runs_to(64);
    if (__popcll(__ballot(near)) < 64) {
      reach(near, 1);
    } else {
      if (reach(far, 64) == 64) {
        while (reach(runs_to(4096), 4096) == 64) {}
        reach(runs_to(64), 64);
      }
      reach(runs_to(1), 1);
    }
    const int64_t count = last - t0 + 1, per = (count + kParts - 1) / kParts;
    const int64_t c0 = wave * per, c1 = min(count, c0 + per);
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int64_t c = c0; c < c1; c += kJoinAhead) {
      Row8<kF32>::Raw q[kJoinAhead];
#pragma unroll
      for (int i = 0; i < kJoinAhead; ++i) {
        const int64_t at = min(c + i, c1 - 1);   // past the end: the last one again, not added
        q[i] = sums.ld(edge + (2 * (t0 + at) + (at == 0 ? 1 : 0)) * d);
      }
#pragma unroll
      for (int i = 0; i < kJoinAhead; ++i) {
        float x[8];
        Row8<kF32>::unpack(q[i], x);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += c + i < c1 ? x[e] : 0.f;
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) part[wave][e][lane] = acc[e];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        for (int w = 1; w < kParts; ++w) acc[e] += part[w][e][lane];
      write_row<OT, TINY, ADD>(out, v, to, d, scale, acc);
    }
  }
}

// The ids of a range, and whether the tokens' places fit beside their bits.
uint32_t range_span(int64_t vocab) { return (uint32_t)((vocab + kRanges - 1) / kRanges); }
int bits_of(uint32_t v) {   // 0 .. v
  int b = 0;
  while (b < 32 && (v >> b) != 0) ++b;
  return b;
}
bool by_ranges(int64_t n, int64_t vocab) {
  return n <= (1 << kPosBits) && bits_of(range_span(vocab) - 1) <= 32 - kPosBits;
}

constexpr unsigned kMovedBlocks = 56;   // 56 KiB of LDS: 114688 tokens
constexpr int kZeroThreads = 1 << 20;   // of a launch's blocks of zeros

inline int launched() { return hipGetLastError() == hipSuccess ? kOk : kErrLaunch; }

int passes_of(int64_t vocab) {   // keys 0 .. vocab
  int bits = 1;
  while (bits < 32 && (vocab >> bits) != 0) ++bits;
  return (bits + 7) / 8;
}

// 16 tokens a tile where 32 would leave the chip short of wavefronts: 8192 tokens
// of 2048 columns 41 against 44 us, 32768 91 against 86.
int tile_of(int64_t n, int64_t d) {
  return n * ((d + kCols - 1) / kCols) <= 40000 ? 16 : 32;
}

struct Plan {
  int passes, tile;
  int64_t sort_blocks, tiles;
  int64_t counts, pairs, edge, bytes;   // offsets into the workspace
};

int64_t up(int64_t v) { return (v + 255) / 256 * 256; }

Plan plan(int64_t n, int64_t vocab, int64_t d) {
  Plan p;
  p.passes = passes_of(vocab);
  p.tile = tile_of(n, d);
  p.sort_blocks = (n + kSortTile - 1) / kSortTile;
  p.tiles = (n + p.tile - 1) / p.tile;
  p.counts = 0;
  p.pairs = up(p.passes * p.sort_blocks * kRadix * 4);
  p.edge = p.pairs + 2 * up(n * (int64_t)sizeof(Pair));
  p.bytes = p.edge + up(p.tiles * 2 * d * 4);
  return p;
}

bool sizes_ok(int64_t n, int64_t vocab, int64_t d) { return n >= 0 && vocab >= 0 && d >= 0; }
// positions and keys are 32 bits wide, a grid's second extent 16, its first 31
bool too_large(int64_t n, int64_t vocab, int64_t d) {
  return n >= (1ll << 31) || vocab >= (1ll << 31) || d > 65535ll * kCols ||
         (n / 16 + 1) * (d / kCols + 1) >= (1ll << 31);
}

}  // namespace embed
}  // namespace cpt

using namespace cpt;
using namespace cpt::embed;

extern "C" {

int cpt_embedding(int dtype, const void* weight, int64_t vocab, int64_t d, const void* ids,
                  int ids_wide, int64_t n, float scale, void* out, void* stream) {
  if (dtype < kF32 || dtype > kBF16) return kErrDType;
  if (!sizes_ok(n, vocab, d)) return kErrShape;
  if (n == 0 || d == 0) return kOk;
  if ((vocab > 0 && !weight) || !ids || !out) return kErrShape;
  const int64_t per_row = (d + 7) / 8;
  if (per_row >= (1ll << 30)) return kErrTooLarge;
  const FastDivU32 div = FastDivU32::make((uint32_t)per_row);
  const int64_t most = (1ll << 30) / per_row;   // rows of a launch
  for (int64_t r0 = 0; r0 < n; r0 += most) {
    const uint32_t total = (uint32_t)((n - r0 < most ? n - r0 : most) * per_row);
    const unsigned grid = (total + kBlock - 1) / kBlock;
    const auto kern = dtype == kF32   ? lookup_kernel<kF32>
                      : dtype == kF16 ? lookup_kernel<kF16>
                                      : lookup_kernel<kBF16>;
    kern<<<grid, kBlock, 0, (hipStream_t)stream>>>(weight, vocab, d, ids, ids_wide, r0, total, div,
                                                   scale, out);
    if (launched() != kOk) return kErrLaunch;
  }
  return kOk;
}

int64_t cpt_embedding_backward_workspace_bytes(int64_t n, int64_t vocab, int64_t d) {
  if (!sizes_ok(n, vocab, d) || too_large(n, vocab, d)) return -1;
  return plan(n, vocab, d).bytes;
}

int cpt_embedding_backward(int dtype, int out_dtype, const void* grad, int64_t ld_grad,
                           const void* ids, int ids_wide, int64_t n, int64_t vocab, int64_t d,
                           int64_t padding_idx, float scale, int accumulate, void* out,
                           void* workspace, void* stream) {
  if (dtype < kF32 || dtype > kBF16 || (out_dtype != dtype && out_dtype != kF32)) return kErrDType;
  if (!sizes_ok(n, vocab, d) || ld_grad < 0) return kErrShape;
  if (too_large(n, vocab, d)) return kErrTooLarge;
  if (vocab == 0 || d == 0) return kOk;
  if (!out || (n > 0 && (!grad || !ids || !workspace))) return kErrShape;
  const hipStream_t st = (hipStream_t)stream;
  const int64_t total = accumulate ? 0 : vocab * d;
  if (n == 0) {
    const int64_t want = (total + 8 * kBlock - 1) / (8 * kBlock);
    const unsigned grid = (unsigned)(want < 2048 ? want : 2048);
    const auto kern = out_dtype == kF32   ? zero_kernel<kF32>
                      : out_dtype == kF16 ? zero_kernel<kF16>
                                          : zero_kernel<kBF16>;
    if (total > 0) kern<<<grid, kBlock, 0, st>>>(out, total);
    return launched();
  }
  const Plan p = plan(n, vocab, d);
  uint8_t* const ws = (uint8_t*)workspace;
  uint32_t* const counts = (uint32_t*)(ws + p.counts);
  Pair* pairs[2] = {(Pair*)(ws + p.pairs), (Pair*)(ws + p.pairs + up(n * sizeof(Pair)))};
  float* const edge = (float*)(ws + p.edge);
  // part `k` of `parts` of the zeros, in blocks of `threads` after the first `own`
  const auto zeros = [&](int k, int parts, unsigned own, int threads, unsigned* grid) {
    const int64_t each = (total / parts + 7) / 8 * 8;
    Zeros z{out, each * k, k + 1 == parts || each * (k + 1) > total ? total : each * (k + 1), own};
    const int64_t want = z.end <= z.begin ? 0 : (z.end - z.begin + 8 * threads - 1) / (8 * threads);
    *grid = own + (unsigned)(want < kZeroThreads / threads ? want : kZeroThreads / threads);
    return z;
  };
  const Pair* in = pairs[0];
  unsigned grid;
  if (by_ranges(n, vocab)) {
    const Zeros z = zeros(0, 1, kRanges, kRangeThreads, &grid);
    const auto kern = out_dtype == kF32   ? range_sort_kernel<kF32>
                      : out_dtype == kF16 ? range_sort_kernel<kF16>
                                          : range_sort_kernel<kBF16>;
    const size_t lds = 4 * (size_t)n;
    if (lds > 32 * 1024 &&
        hipFuncSetAttribute((const void*)kern, hipFuncAttributeMaxDynamicSharedMemorySize,
                            (int)lds) != hipSuccess)
      return kErrLaunch;
    const uint32_t span = range_span(vocab);
    kern<<<grid, kRangeThreads, lds, st>>>(ids, ids_wide, (int)n, (uint32_t)vocab, padding_idx,
                                           span, bits_of(span - 1), pairs[0], z);
  } else {
    const unsigned own = (unsigned)p.sort_blocks;
    const auto count = out_dtype == kF32   ? count_kernel<kF32>
                       : out_dtype == kF16 ? count_kernel<kF16>
                                           : count_kernel<kBF16>;
    const auto scatter = out_dtype == kF32   ? scatter_kernel<kF32>
                         : out_dtype == kF16 ? scatter_kernel<kF16>
                                             : scatter_kernel<kBF16>;
    in = nullptr;
    // a pass counts for the next one where the blocks' counts fit LDS
    const bool ahead = own <= kMovedBlocks;
    const int parts = ahead ? p.passes + 1 : 2 * p.passes;
    int part = 0;
    for (int k = 0; k < p.passes; ++k) {
      uint32_t* const c = counts + (ahead ? (int64_t)k * own * kRadix : 0);
      if (k == 0 || !ahead) {
        const Zeros z = zeros(part++, parts, own, kBlock, &grid);
        count<<<grid, kBlock, 0, st>>>(in, ids, ids_wide, n, vocab, padding_idx, 8 * k, c, own,
                                       ahead ? p.passes - 1 : 0, z);
      }
      const bool counts_next = ahead && k + 1 < p.passes;
      const Zeros z = zeros(part++, parts, own, kBlock, &grid);
      scatter<<<grid, kBlock, counts_next ? own * kRadix * 4 : 0, st>>>(
          in, ids, ids_wide, n, vocab, padding_idx, 8 * k, c, own,
          counts_next ? c + (int64_t)own * kRadix : nullptr, pairs[k & 1], z);
      in = pairs[k & 1];
    }
  }
  if (launched() != kOk) return kErrLaunch;
  const unsigned strips = (unsigned)((d + kCols - 1) / kCols);
  const unsigned sums = (unsigned)((p.tiles * strips + kWaves - 1) / kWaves);
  const dim3 joins((unsigned)((p.tiles + kJoinTiles - 1) / kJoinTiles), strips);
#define CPT_SUM_T(DT, OT, TINY, ADD, TILE)                                                      \
  (sum_kernel<DT, OT, TINY, ADD, TILE><<<sums, kBlock, 0, st>>>(                                \
       grad, ld_grad, in, n, vocab, d, strips, scale, out, edge),                               \
   join_kernel<OT, TINY, ADD, TILE><<<joins, kJoinThreads, 0, st>>>(in, n, vocab, d, scale, out, edge))
#define CPT_SUM_A(DT, OT, TINY, TILE) \
  (accumulate ? CPT_SUM_T(DT, OT, TINY, true, TILE) : CPT_SUM_T(DT, OT, TINY, false, TILE))
#define CPT_SUM(DT, OT)                                                                         \
  (d < 8 ? (p.tile == 16 ? CPT_SUM_A(DT, OT, true, 16) : CPT_SUM_A(DT, OT, true, 32))            \
         : (p.tile == 16 ? CPT_SUM_A(DT, OT, false, 16) : CPT_SUM_A(DT, OT, false, 32)))
  if (dtype == kF32)
    CPT_SUM(kF32, kF32);
  else if (dtype == kF16)
    out_dtype == kF32 ? CPT_SUM(kF16, kF32) : CPT_SUM(kF16, kF16);
  else
    out_dtype == kF32 ? CPT_SUM(kBF16, kF32) : CPT_SUM(kBF16, kBF16);
  return launched();
}

}  // extern "C"
