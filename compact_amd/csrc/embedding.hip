// Embedding lookup with a scale, and its gradient by sorted tokens.
//
//   out[n] = scale W[id_n]                     (an id outside the table: zeros)
//   dW[v]  = scale sum_{n: id_n = v} dy[n]     (v != padding_idx)
//
// The lookup is HBM-bound: one thread per eight columns.
//
// The gradient adds no floats atomically.  The tokens' (id, position) pairs are
// sorted by id with their order kept (a radix sort of 8 bits a pass, each pass
// ranking 2048 pairs a block by ballots), so one id's tokens lie side by side in
// the order of the batch.  The sorted list is cut into tiles of equal length,
// whatever ids they hold, so a frequent token's rows are spread over as many
// wavefronts as it needs: a wavefront sums 512 columns of one tile in fp32,
// writes each id that lies wholly inside it, and leaves the sums of an id that
// goes on over a tile's edge to be joined in tile order.  The result is the same
// from run to run.  Bound by HBM: dy is read once, the table written once.

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

// counts[0][block][digit] of the lowest digit, and zeros for the later passes'.
__global__ __launch_bounds__(kBlock) void count_kernel(const void* __restrict__ ids, int wide,
                                                       int64_t n, int64_t vocab, int64_t padding,
                                                       int passes, uint32_t* counts) {
  __shared__ uint32_t hist[kRadix];
  hist[threadIdx.x] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * kSortTile;
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = i0 + k * kBlock + threadIdx.x;
    if (i < n) atomicAdd(&hist[token_key(ids, wide, i, vocab, padding) & (kRadix - 1)], 1u);
  }
  __syncthreads();
  for (int p = 0; p < passes; ++p)
    counts[((int64_t)p * gridDim.x + blockIdx.x) * kRadix + threadIdx.x] =
        p == 0 ? hist[threadIdx.x] : 0;
}

// One pass of the sort: pairs of `in` (the tokens themselves in the first) to
// their places by digit (key >> shift) & 255, equal digits in their order.
// `next` (null in the last pass) collects the next digit's counts by block.
__global__ __launch_bounds__(kBlock) void scatter_kernel(const Pair* __restrict__ in,
                                                         const void* __restrict__ ids, int wide,
                                                         int64_t n, int64_t vocab, int64_t padding,
                                                         int shift,
                                                         const uint32_t* __restrict__ counts,
                                                         uint32_t* next, Pair* __restrict__ out) {
  __shared__ uint32_t wave_count[kWaves][kRadix];
  __shared__ uint32_t base[kRadix];
  __shared__ uint32_t scan[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int w = 0; w < kWaves; ++w) wave_count[w][tid] = 0;
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
  for (unsigned b = 0; b < gridDim.x; ++b) {
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
      atomicAdd(&next[(int64_t)(to / kSortTile) * kRadix + ((q[k].id >> (shift + 8)) & 255)], 1u);
  }
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

template <int OT>
__device__ __forceinline__ void write_row(void* out, int64_t v, int64_t j, int64_t d, float scale,
                                          int accumulate, const float acc[8]) {
  using R = Row8<OT>;
  typename R::T* row = (typename R::T*)out + v * d;
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = acc[e] * scale;
  if (accumulate) {
    float o[8];
    R::unpack(row_ld<OT>(row, j, d, 0), o);
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] += o[e];
  }
  row_st<OT>(row, j, d, R::pack(r));
}

// grid (tiles, columns / 512 / 4): a wavefront sums 512 columns of one tile.
// edge: fp32 [tiles][2][d]: sums of the id that came in over the tile's first
// edge (0), and of the id that starts inside and goes on past its end (1).
template <int DT, int OT>
__global__ __launch_bounds__(kBlock) void sum_kernel(const void* __restrict__ grad, int64_t ld,
                                                     const Pair* __restrict__ pairs, int64_t n,
                                                     int64_t vocab, int64_t d, int tile,
                                                     float scale, int accumulate, void* out,
                                                     float* edge) {
  using R = Row8<DT>;
  using T = typename R::T;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t j = ((int64_t)blockIdx.y * kWaves + wave) * kCols + 8 * lane;
  if (j - 8 * lane >= d) return;
  const int64_t i0 = (int64_t)blockIdx.x * tile;
  const int64_t i1 = min(n, i0 + tile);
  const uint32_t none = (uint32_t)vocab;
  uint32_t id = pairs[i0].id;
  bool entered = i0 > 0 && pairs[i0 - 1].id == id;
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  constexpr int kAhead = 8;
  for (int64_t i = i0; i < i1 && id != none; i += kAhead) {
    Pair p[kAhead];
    typename R::Raw q[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      p[k] = i + k < i1 ? pairs[i + k] : Pair{none, 0};
      q[k] = p[k].id != none ? row_ld<DT>((const T*)grad + (int64_t)p[k].pos * ld, j, d, 0)
                             : R::zero();
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i + k >= i1) break;
      if (p[k].id != id) {
        if (entered)
          row_st<kF32>(edge + 2 * blockIdx.x * d, j, d, Row8<kF32>::pack(acc));
        else
          write_row<OT>(out, id, j, d, scale, accumulate, acc);
        entered = false;
        id = p[k].id;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
        if (id == none) break;
      }
      float v[8];
      R::unpack(q[k], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += v[e];
    }
  }
  if (id == none) return;
  const bool leaves = i1 < n && pairs[i1].id == id;
  if (entered || leaves)
    row_st<kF32>(edge + (2 * blockIdx.x + (entered ? 0 : 1)) * d, j, d, Row8<kF32>::pack(acc));
  else
    write_row<OT>(out, id, j, d, scale, accumulate, acc);
}

// grid (tiles, columns / 512): the ids that start in a tile and end in a later
// one.  Four wavefronts add a quarter of the tiles each, then in order.
template <int OT>
__global__ __launch_bounds__(kBlock) void join_kernel(const Pair* __restrict__ pairs, int64_t n,
                                                      int64_t vocab, int64_t d, int tile,
                                                      float scale, int accumulate, void* out,
                                                      const float* __restrict__ edge) {
  __shared__ float part[kWaves][8][64];
  const int64_t t0 = blockIdx.x, i1 = (t0 + 1) * tile;
  if (i1 >= n) return;
  const uint32_t id = pairs[i1 - 1].id;
  if (id == (uint32_t)vocab || pairs[i1].id != id) return;
  if (pairs[i1 - tile].id == id && t0 > 0 && pairs[i1 - tile - 1].id == id) return;
  // the last tile that the id reaches: the first later one that does not end with it
  // still holds its last tokens
  int64_t lo = t0 + 1, hi = (n + tile - 1) / tile - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (pairs[min(n, (mid + 1) * tile) - 1].id == id && (mid + 1) * tile < n &&
        pairs[(mid + 1) * tile].id == id)
      lo = mid + 1;
    else
      hi = mid;
  }
  const int64_t count = lo - t0 + 1, per = (count + kWaves - 1) / kWaves;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t j = (int64_t)blockIdx.y * kCols + 8 * lane;
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  const int64_t c0 = wave * per, c1 = min(count, c0 + per);
#pragma unroll 4
  for (int64_t c = c0; c < c1; ++c) {
    float v[8];
    Row8<kF32>::unpack(row_ld<kF32>(edge + (2 * (t0 + c) + (c == 0 ? 1 : 0)) * d, j, d, 0), v);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += v[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) part[wave][e][lane] = acc[e];
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    for (int w = 1; w < kWaves; ++w) acc[e] += part[w][e][lane];
  write_row<OT>(out, id, j, d, scale, accumulate, acc);
}

inline int launched() { return hipGetLastError() == hipSuccess ? kOk : kErrLaunch; }

int passes_of(int64_t vocab) {   // keys 0 .. vocab
  int bits = 1;
  while (bits < 32 && (vocab >> bits) != 0) ++bits;
  return (bits + 7) / 8;
}

// Tokens of a tile: 32, more where the batch still gives 4096 wavefronts (each
// edge costs an fp32 row written and read again).
int tile_of(int64_t n, int64_t d) {
  const int64_t strips = (d + kCols - 1) / kCols;
  int tile = 32;
  while (tile < 256 && n * strips / (2 * tile) >= 4096) tile *= 2;
  return tile;
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
// positions and keys are 32 bits wide, a grid's second extent 16
bool too_large(int64_t n, int64_t vocab, int64_t d) {
  return n >= (1ll << 31) || vocab >= (1ll << 31) || d > 65535ll * kCols;
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
  if (!accumulate) {
    const int64_t total = vocab * d, want = (total + 8 * kBlock - 1) / (8 * kBlock);
    const unsigned grid = (unsigned)(want < 2048 ? want : 2048);
    const auto kern = out_dtype == kF32   ? zero_kernel<kF32>
                      : out_dtype == kF16 ? zero_kernel<kF16>
                                          : zero_kernel<kBF16>;
    kern<<<grid, kBlock, 0, st>>>(out, total);
    if (launched() != kOk) return kErrLaunch;
  }
  if (n == 0) return kOk;
  const Plan p = plan(n, vocab, d);
  uint8_t* const ws = (uint8_t*)workspace;
  uint32_t* const counts = (uint32_t*)(ws + p.counts);
  Pair* pairs[2] = {(Pair*)(ws + p.pairs), (Pair*)(ws + p.pairs + up(n * sizeof(Pair)))};
  float* const edge = (float*)(ws + p.edge);
  const unsigned sb = (unsigned)p.sort_blocks;
  count_kernel<<<sb, kBlock, 0, st>>>(ids, ids_wide, n, vocab, padding_idx, p.passes, counts);
  const Pair* in = nullptr;
  for (int k = 0; k < p.passes; ++k) {
    uint32_t* const c = counts + (int64_t)k * sb * kRadix;
    scatter_kernel<<<sb, kBlock, 0, st>>>(in, ids, ids_wide, n, vocab, padding_idx, 8 * k, c,
                                          k + 1 < p.passes ? c + (int64_t)sb * kRadix : nullptr,
                                          pairs[k & 1]);
    in = pairs[k & 1];
  }
  if (launched() != kOk) return kErrLaunch;
  const int64_t strips = (d + kCols - 1) / kCols;
  const dim3 sums((unsigned)p.tiles, (unsigned)((strips + kWaves - 1) / kWaves));
  const dim3 joins((unsigned)p.tiles, (unsigned)strips);
#define CPT_SUM(DT, OT)                                                                          \
  (sum_kernel<DT, OT><<<sums, kBlock, 0, st>>>(grad, ld_grad, in, n, vocab, d, p.tile, scale,     \
                                               accumulate, out, edge),                           \
   join_kernel<OT><<<joins, kBlock, 0, st>>>(in, n, vocab, d, p.tile, scale, accumulate, out,     \
                                             edge))
  if (dtype == kF32)
    CPT_SUM(kF32, kF32);
  else if (dtype == kF16)
    out_dtype == kF32 ? CPT_SUM(kF16, kF32) : CPT_SUM(kF16, kF16);
  else
    out_dtype == kF32 ? CPT_SUM(kBF16, kF32) : CPT_SUM(kBF16, kBF16);
  return launched();
}

}  // extern "C"
