/*
 * Embedding look-up with scaling and its gradient, for binary32, binary16 and bfloat16 tables.
 *
 *   EmbedTake       out[i] = scale * table[index[i]]                (0 where index[i] is outside the table)
 *   EmbedTakeGrad   grad[r] (=|+=) scale * sum of g[i], index[i] == r  (an index outside names no row)
 *
 * Products with scale and sums are binary32, in ascending order of i up to the grouping below, and
 * rounded once to the element type.  No atomics on values: results do not depend on timing.
 *
 * The look-up moves 16-byte groups, four in flight per thread, and is bound by memory.
 *
 * The gradient sorts (index, position) stably (radix_sort.cuh) and sums segments of the sorted list:
 *   - the list is cut into chunks of kChunk entries; a chunk's CTA owns the runs that begin in it
 *     and follows the last one past the chunk's end;
 *   - only a run of more than kChunk entries (a frequent token) is split: each chunk leaves its
 *     part as a binary32 row in scratch memory, and a second kernel adds the parts, in order;
 *   - when the gradient is assigned rather than added to, further CTAs of the same launch write
 *     zeros to the rows that no index names, so that every row of the table is written exactly
 *     once.
 * A short list (up to kFewTokens) is not sorted: the CTA of an entry that is the first of its index
 * finds the later ones by scanning the list.
 */
#ifndef MSHADOW_GPU_EMBED_TAKE_CUH_
#define MSHADOW_GPU_EMBED_TAKE_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../bfloat.h"
#include "./radix_sort.cuh"

namespace mshadow {
namespace cuda {
namespace embtake {

const int kChunk = 64;        // sorted entries per CTA; also the longest run that is not split
const int kFewTokens = 512;   // lists up to this are not sorted
const int kOneCta = 8192;     // lists up to this are sorted by one CTA
const int kDepth = 8;         // source rows in flight per thread
const uint32_t kManyParts = 32;  // a split run of more chunks than this is shared by a CTA's warps
const int kZeroRows = 32;     // table rows per CTA that writes zeros

// ---- element types: groups of 16 bytes (or single elements) as binary32 ----------------------------

/*!
 * \brief how rows are accessed: kOne element at a time; kAligned, 16-byte groups; kAnywhere, rows that start at any
 *  element: two 32-bit elements or one 16-bit element per thread.  16-bit elements in fours spread each store of
 *  a warp over four times the sectors: 16384 gradient rows of 2047 into 131072, assigned, took 414 us instead
 *  of 198; 32-bit elements in twos: 262144 rows of 511 into 65536 in 212 us, one at a time 264.
 */
enum Form { kOne = 0, kAligned = 1, kAnywhere = 2 };

template <typename T, int kVec>
struct Group {
  static const int kLanes = (kVec == kAligned ? 16 / static_cast<int>(sizeof(T)) : kVec == kAnywhere && sizeof(T) == 4 ? 2 : 1);
};

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(half::half_t v) { return __half2float(__ushort_as_half(v.half_)); }
__device__ __forceinline__ float ToFloat(bfloat::bf16_t v) { return __uint_as_float(static_cast<uint32_t>(v.bits_) << 16); }
__device__ __forceinline__ void FromFloat(float v, float *out) { *out = v; }
__device__ __forceinline__ void FromFloat(float v, half::half_t *out) { out->half_ = __half_as_ushort(__float2half_rn(v)); }
__device__ __forceinline__ void FromFloat(float v, bfloat::bf16_t *out) {
  out->bits_ = __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

/*! \brief raw bits of one group */
template <typename T, int kVec>
struct Bits {
  T raw[Group<T, kVec>::kLanes];
};
template <typename T>
struct Bits<T, kAligned> {
  uint4 raw;
};

/*! \brief `left`: elements of the row from p on; an aligned group is whole */
template <typename T>
__device__ __forceinline__ void LoadStream(const T *p, uint32_t, Bits<T, kAligned> *b) {
  b->raw = __ldcs(reinterpret_cast<const uint4 *>(p));
}
template <typename T>
__device__ __forceinline__ void Load(const T *p, uint32_t, Bits<T, kAligned> *b) {
  b->raw = *reinterpret_cast<const uint4 *>(p);
}
template <typename T>
__device__ __forceinline__ void Store(T *p, uint32_t, const Bits<T, kAligned> &b) {
  *reinterpret_cast<uint4 *>(p) = b.raw;
}
template <typename T, int kVec>
__device__ __forceinline__ void Load(const T *p, uint32_t left, Bits<T, kVec> *b) {
#pragma unroll
  for (int l = 0; l < Group<T, kVec>::kLanes; ++l) {
    if (l < static_cast<int>(left)) b->raw[l] = p[l];
    else memset(&b->raw[l], 0, sizeof(T));
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void LoadStream(const T *p, uint32_t left, Bits<T, kVec> *b) {
  Load(p, left, b);
}
template <typename T, int kVec>
__device__ __forceinline__ void Store(T *p, uint32_t left, const Bits<T, kVec> &b) {
#pragma unroll
  for (int l = 0; l < Group<T, kVec>::kLanes; ++l) {
    if (l < static_cast<int>(left)) p[l] = b.raw[l];
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void Unpack(const Bits<T, kVec> &b, float (&v)[Group<T, kVec>::kLanes]) {
  T e[Group<T, kVec>::kLanes];
  memcpy(e, &b.raw, sizeof(e));
#pragma unroll
  for (int l = 0; l < Group<T, kVec>::kLanes; ++l) v[l] = ToFloat(e[l]);
}
template <typename T, int kVec>
__device__ __forceinline__ void Pack(const float (&v)[Group<T, kVec>::kLanes], Bits<T, kVec> *b) {
  T e[Group<T, kVec>::kLanes];
#pragma unroll
  for (int l = 0; l < Group<T, kVec>::kLanes; ++l) FromFloat(v[l], &e[l]);
  memcpy(&b->raw, e, sizeof(e));
}

// ---- look-up -------------------------------------------------------------------------------------------

/*!
 * \brief rows on 16-byte boundaries: grid-stride over (token, group) pairs, four per thread and sweep: the look-ups of the
 *  four row numbers and then the four groups are in flight together
 */
template <typename T>
__global__ void __launch_bounds__(256)
EmbedTakeKernel(T *out, int64_t ld_out, const int32_t *index, const T *table, int64_t ld_table, uint32_t total,
                gpu_rt::FastDiv groups, int32_t rows, float scale) {
  gpu_rt::GridDependencySync();
  typedef Group<T, kAligned> G;
  const uint32_t step = gridDim.x * 256;
  for (uint32_t e0 = blockIdx.x * 256 + threadIdx.x; e0 < total; e0 += 4 * step) {
    Bits<T, kAligned> b[4];
    uint32_t token[4], col[4];
    int32_t r[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t e = e0 + u * step;
      r[u] = -1;
      if (e < total) {
        col[u] = groups.DivMod(e, &token[u]) * G::kLanes;
        r[u] = index[token[u]];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      memset(&b[u], 0, sizeof(b[u]));
      if (r[u] >= 0 && r[u] < rows) Load(table + r[u] * ld_table + col[u], G::kLanes, &b[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (e0 + u * step >= total) continue;
      float v[G::kLanes];
      Unpack<T, kAligned>(b[u], v);
      const bool named = r[u] >= 0 && r[u] < rows;
#pragma unroll
      for (int l = 0; l < G::kLanes; ++l) v[l] = named ? v[l] * scale : 0.0f;
      Pack<T, kAligned>(v, &b[u]);
      Store(out + token[u] * ld_out + col[u], G::kLanes, b[u]);
    }
  }
}

const int kTakeDeep = 8;            // loads of a lane in flight
const uint32_t kTakeSegment = 512;  // elements of a row taken at a time where rows start anywhere

/*!
 * \brief rows that start at any element: a segment of a row goes to 4 to 32 lanes, so that what depends on the row is found once,
 *  and 16-bit elements go in pairs, as the 4-byte words of the output row (its first and last element may be
 *  left over).  16384 x 2047 bf16: 50 us; with row and column found for each pair of elements 79 us.
 */
template <typename T>
__global__ void __launch_bounds__(256)
EmbedTakeAnywhereKernel(T *out, int64_t ld_out, const int32_t *index, const T *table, int64_t ld_table, uint32_t total,
                        gpu_rt::FastDiv segments, uint32_t width, int32_t rows, float scale, int lanes_log2) {
  gpu_rt::GridDependencySync();
  constexpr int kDeep = kTakeDeep;
  const uint32_t lanes = 1u << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const uint32_t teams = gridDim.x * (256u >> lanes_log2);
  for (uint32_t e = blockIdx.x * (256u >> lanes_log2) + (threadIdx.x >> lanes_log2); e < total; e += teams) {
    uint32_t token;
    const uint32_t begin = segments.DivMod(e, &token) * kTakeSegment, end = min(width, begin + kTakeSegment);
    const int32_t r = index[token];
    const bool named = r >= 0 && r < rows;
    T *dst = out + token * ld_out;
    const T *src = table + (named ? r : 0) * ld_table;
    if (sizeof(T) == 2) {
      const uint32_t head = begin + (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(dst + begin) >> 1) & 1u);
      const uint32_t words = end > head ? (end - head) / 2 : 0;
      const bool even = reinterpret_cast<uintptr_t>(src + head) % 4 == 0;
      for (uint32_t w0 = lane; w0 < words; w0 += lanes * kDeep) {
        T v[kDeep][2];
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
          const T *from = src + head + 2 * (w0 + lanes * u);
          if (w0 + lanes * u >= words || !named) {
            memset(v[u], 0, sizeof(v[u]));
          } else if (even) {
            memcpy(v[u], reinterpret_cast<const uint32_t *>(from), 4);
          } else {
            v[u][0] = from[0], v[u][1] = from[1];
          }
        }
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
          if (w0 + lanes * u >= words) continue;
          T o[2];
          FromFloat(named ? ToFloat(v[u][0]) * scale : 0.0f, &o[0]);
          FromFloat(named ? ToFloat(v[u][1]) * scale : 0.0f, &o[1]);
          uint32_t bits;
          memcpy(&bits, o, 4);
          *reinterpret_cast<uint32_t *>(dst + head + 2 * (w0 + lanes * u)) = bits;
        }
      }
      const uint32_t rest = lane == 0 ? begin : head + 2 * words;  // the elements before the first and behind the last word
      if ((lane == 0 && head > begin && begin < end) || (lane == 1 && rest < end)) {
        FromFloat(named ? ToFloat(src[rest]) * scale : 0.0f, &dst[rest]);
      }
    } else {
      for (uint32_t c0 = begin + lane; c0 < end; c0 += lanes * kDeep) {
        float v[kDeep];
#pragma unroll
        for (int u = 0; u < kDeep; ++u) v[u] = c0 + lanes * u < end && named ? ToFloat(src[c0 + lanes * u]) : 0.0f;
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
          if (c0 + lanes * u < end) FromFloat(named ? v[u] * scale : 0.0f, &dst[c0 + lanes * u]);
        }
      }
    }
  }
}

// ---- gradient -------------------------------------------------------------------------------------------

template <typename T>
struct GradArgs {
  T *grad;
  int64_t ld_grad;
  const T *g;
  int64_t ld_g;
  const int32_t *keys, *rows;  // sorted indices, their positions (-1: names no row)
  const int32_t *index;        // short lists: the indices as given
  uint32_t n, width, table_rows;
  float scale;
  int add;
  uint32_t chunks, slabs;      // CTAs that sum; the ones after them write zeros
  float *parts;                // [2 * chunks][width_pad]: parts of split runs
  int64_t ld_parts;
  int32_t *spans;              // [0], [1] = number of split runs of few / many parts, then (first, last chunk) of
                               // the runs of few parts from the front, of many parts from the back
};

/*!
 * \brief -0, the sum of nothing: a run of entries that name no row (they are sorted among those of the first and the last row).
 *  Adding it, or a sum of -0 alone, changes no value, so a row is not written then: another call may be adding to it at
 *  the same time on another stream, and a NaN would not keep its bits.
 */
template <int kLanes>
__device__ __forceinline__ bool AddsNothing(const float (&sum)[kLanes]) {
  bool nothing = true;
#pragma unroll
  for (int l = 0; l < kLanes; ++l) nothing = nothing && __float_as_uint(sum[l]) == 0x80000000u;
  return nothing;
}
/*! \brief scale * sum; the sum of nothing stays it, whatever the scale */
__device__ __forceinline__ float Scaled(float scale, float sum) {
  return __float_as_uint(sum) == 0x80000000u ? sum : __fmul_rn(scale, sum);
}

template <typename T, int kVec>
__device__ __forceinline__ void WriteRow(const GradArgs<T> &a, int32_t row, uint32_t col,
                                         const float (&acc)[Group<T, kVec>::kLanes]) {
  T *p = a.grad + row * a.ld_grad + col;
  Bits<T, kVec> b;
  float v[Group<T, kVec>::kLanes];
  if (a.add) {
    if (AddsNothing(acc)) return;
    Load(p, a.width - col, &b);
    Unpack<T, kVec>(b, v);
#pragma unroll
    for (int l = 0; l < Group<T, kVec>::kLanes; ++l) v[l] = __fadd_rn(v[l], Scaled(a.scale, acc[l]));
  } else {
#pragma unroll
    for (int l = 0; l < Group<T, kVec>::kLanes; ++l) v[l] = __fadd_rn(Scaled(a.scale, acc[l]), 0.0f);
  }
  Pack<T, kVec>(v, &b);
  Store(p, a.width - col, b);
}

/*! \brief zeros for the rows [first, last) whose flag is not set */
template <typename T, int kVec>
__device__ __forceinline__ void WriteZeros(const GradArgs<T> &a, uint32_t first, uint32_t last, const uint8_t *named) {
  Bits<T, kVec> zero;
  memset(&zero, 0, sizeof(zero));
  const uint32_t warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  for (uint32_t r = first + warp; r < last; r += warps) {
    if (named[r - first]) continue;
    for (uint32_t c = lane * Group<T, kVec>::kLanes; c < a.width; c += 32 * Group<T, kVec>::kLanes) {
      Store(a.grad + r * a.ld_grad + c, a.width - c, zero);
    }
  }
}

/*! \brief first position of keys[0, n) that is not below k; by one warp, 32 places looked at per step */
__device__ __forceinline__ uint32_t WarpLowerBound(const int32_t *keys, uint32_t n, int32_t k) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t lo = 0, hi = n;  // the answer lies in [lo, hi]
  while (lo < hi) {
    const uint32_t span = hi - lo, part = (span + 31) / 32;
    const uint32_t at = lo + lane * part;  // ends of 32 parts: keys[at] < k for the parts before the answer's
    const bool below = at < hi && keys[at] < k;
    const uint32_t count = __popc(__ballot_sync(0xffffffffu, below));
    if (count == 0) return lo;
    lo = lo + (count - 1) * part + 1;
    hi = min(hi, lo + part - 1);
  }
  return lo;
}

/*! \brief adds the source rows of window entries [from, to) to acc, kDepth of them in flight */
template <typename T, int kVec>
__device__ __forceinline__ void AddRows(const GradArgs<T> &a, const int32_t *rows, uint32_t from, uint32_t to, uint32_t col,
                                        float (&acc)[Group<T, kVec>::kLanes]) {
  for (uint32_t i = from; i < to; i += kDepth) {
    Bits<T, kVec> b[kDepth];
    int32_t r[kDepth];
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      r[u] = i + u < to ? rows[i + u] : -1;
      if (r[u] >= 0) LoadStream(a.g + r[u] * a.ld_g + col, a.width - col, &b[u]);
    }
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      if (r[u] >= 0) {
        float v[Group<T, kVec>::kLanes];
        Unpack<T, kVec>(b[u], v);
#pragma unroll
        for (int l = 0; l < Group<T, kVec>::kLanes; ++l) acc[l] = __fadd_rn(acc[l], v[l]);
      }
    }
  }
}

/*!
 * \brief stable sort of the (clipped index, position) pairs of up to kOneCta indices by one CTA of 1024 threads, least
 *  significant digit first, and the start values of the list of split runs: one launch instead of six and a
 *  memory set.  The pairs live in shared memory (4 + 2 bytes each); in a pass every warp takes a
 *  contiguous part of them into registers, counts its digits (ranks within a round of 32 from a
 *  warp-wide match), and after a scan over warps and digits scatters them back.  Bound by latency: two passes
 *  of eight bits take 5 us for 1024 pairs and 22 us for 8192, where the many-CTA sort takes 25 us in six
 *  launches, whose issue alone costs the host 15 us more.
 *  Dynamic shared memory: SortOneBytes(n, digit_bits).
 */
template <int kUnused>
__global__ void __launch_bounds__(1024)
EmbedSortKernel(int32_t *keys, int32_t *rows, const int32_t *index, uint32_t n, uint32_t table_rows, int passes, int digit_bits,
                int32_t *spans) {
  gpu_rt::GridDependencySync();
  constexpr int kItems = kOneCta / 1024;
  extern __shared__ uint32_t s_key[];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rounds = (n + 1023) / 1024;  // a warp's part: `rounds` times 32 consecutive pairs
  const uint32_t digits = 1u << digit_bits, mask = digits - 1u;
  uint16_t *s_val = reinterpret_cast<uint16_t *>(s_key + rounds * 1024);
  uint16_t *count = s_val + rounds * 1024;             // [32 warps][digits]
  uint32_t *base = reinterpret_cast<uint32_t *>(count + 32 * digits);  // [digits]
  __shared__ uint32_t s_sum[32];
  if (threadIdx.x < 2) spans[threadIdx.x] = 0;
  for (uint32_t i = threadIdx.x; i < n; i += 1024) {
    const int32_t k = index[i];
    const bool named = k >= 0 && static_cast<uint32_t>(k) < table_rows;
    s_key[i] = named ? static_cast<uint32_t>(k) : 0u;
    s_val[i] = named ? static_cast<uint16_t>(i) : 0xffffu;  // i < kOneCta
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    for (uint32_t i = threadIdx.x; i < 16 * digits; i += 1024) reinterpret_cast<uint32_t *>(count)[i] = 0;
    __syncthreads();
    uint32_t key[kItems];
    uint32_t val_rank[kItems];  // value in the upper half, rank among the warp's equal digits in the lower
    uint16_t *mine = count + warp * digits;
    const uint32_t first = warp * rounds * 32 + lane;
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      const uint32_t i = first + r * 32;
      if (r >= static_cast<int>(rounds)) break;
      const bool in = i < n;
      key[r] = in ? s_key[i] : 0u;
      const uint32_t digit = in ? (key[r] >> shift) & mask : digits;
      const uint32_t peers = __match_any_sync(0xffffffffu, digit);
      const uint32_t before = __popc(peers & ((1u << lane) - 1u));
      const uint32_t seen = in ? mine[digit] : 0u;
      __syncwarp();
      if (in && before == 0) mine[digit] = static_cast<uint16_t>(seen + __popc(peers));
      __syncwarp();
      val_rank[r] = (in ? static_cast<uint32_t>(s_val[i]) << 16 : 0u) | (seen + before);
    }
    __syncthreads();
    // per digit: the warps' counts become the warps' places within the digit, and their sum the digit's size
    uint32_t size = 0;
    if (threadIdx.x < digits) {
      for (int w = 0; w < 32; ++w) {
        const uint32_t c = count[w * digits + threadIdx.x];
        count[w * digits + threadIdx.x] = static_cast<uint16_t>(size);
        size += c;
      }
    }
    uint32_t incl = size;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= static_cast<uint32_t>(o)) incl += up;
    }
    if (lane == 31) s_sum[warp] = incl;
    __syncthreads();
    uint32_t below = 0;
    for (uint32_t w = 0; w < warp; ++w) below += s_sum[w];
    if (threadIdx.x < digits) base[threadIdx.x] = below + incl - size;
    __syncthreads();
    const bool last = pass == passes - 1;
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      if (r >= static_cast<int>(rounds)) break;
      if (first + r * 32 < n) {
        const uint32_t digit = (key[r] >> shift) & mask;
        const uint32_t at = base[digit] + mine[digit] + (val_rank[r] & 0xffffu), val = val_rank[r] >> 16;
        if (last) {
          keys[at] = static_cast<int32_t>(key[r]);
          rows[at] = val == 0xffffu ? -1 : static_cast<int32_t>(val);
        } else {
          s_key[at] = key[r];
          s_val[at] = static_cast<uint16_t>(val);
        }
      }
    }
    __syncthreads();
  }
}

/*!
 * \brief sums of the runs of a sorted list, and zeros for the rows that are not in it.
 *  grid: chunks * slabs CTAs that sum, then (when assigning) CTAs that write zeros.
 *  A thread walks its chunk's entries eight at a time whatever runs they belong to, with the eight source
 *  rows (and, when adding, the table rows of the runs that end among them) in flight together: with one run
 *  after the other, 600 tokens of mostly different rows took 48 us.
 */
template <typename T, int kVec, bool kAdd>
__global__ void __launch_bounds__(256) EmbedSumKernel(const GradArgs<T> a) {
  gpu_rt::GridDependencySync();
  typedef Group<T, kVec> G;
  if (blockIdx.x >= a.chunks * a.slabs) {
    __shared__ uint8_t named[kZeroRows];
    const uint32_t first = (blockIdx.x - a.chunks * a.slabs) * kZeroRows;
    const uint32_t last = min(a.table_rows, first + kZeroRows);
    for (uint32_t r = threadIdx.x; r < kZeroRows; r += blockDim.x) named[r] = 0;
    const uint32_t from = WarpLowerBound(a.keys, a.n, static_cast<int32_t>(first));
    __syncthreads();
    // the entries of these rows; after a stretch of 128 of them (a frequent token) a search finds the next row
    if (threadIdx.x < 32) {
      for (uint32_t i = from; i < a.n;) {
        const uint32_t e = i + threadIdx.x * 4;
        int32_t k = 0x7fffffff;
        for (uint32_t j = e; j < min(e + 4, a.n); ++j) {
          k = a.keys[j];
          if (k < static_cast<int64_t>(last)) named[k - first] = 1;
        }
        const int32_t top = __shfl_sync(0xffffffffu, k, 31);  // of the last entry looked at, or past the list
        if (top >= static_cast<int64_t>(last)) break;
        i = WarpLowerBound(a.keys, a.n, top + 1);
      }
    }
    __syncthreads();
    WriteZeros<T, kVec>(a, first, last, named);
    return;
  }
  static_assert(kChunk == 64, "the ends of runs are kept in 64-bit words");
  __shared__ int32_t s_keys[3 * kChunk + 1], s_rows[3 * kChunk];
  __shared__ uint32_t s_ends[3 * kChunk / 32];
  const uint32_t chunk = blockIdx.x / a.slabs, slab = blockIdx.x - chunk * a.slabs;
  const int64_t begin = static_cast<int64_t>(chunk) * kChunk;
  // entries [begin - kChunk, begin + 2 kChunk] of the list; keys outside the list differ from all others
  for (uint32_t i = threadIdx.x; i < 3 * kChunk + 1; i += blockDim.x) {
    const int64_t e = begin - kChunk + i;
    const bool in = e >= 0 && e < a.n;
    s_keys[i] = in ? a.keys[e] : -1;
    if (i < 3 * kChunk) s_rows[i] = in ? a.rows[e] : -1;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < 3 * kChunk; i += blockDim.x) {
    const uint32_t ends = __ballot_sync(0xffffffffu, s_keys[i] != s_keys[i + 1]);  // (blocks are whole warps, 192 too)
    if ((i & 31) == 0) s_ends[i / 32] = ends;
  }
  __syncthreads();
  // bit p of `ends` of chunk c of the window: a run ends with entry p
  uint64_t ends[3];
#pragma unroll
  for (int c = 0; c < 3; ++c) ends[c] = s_ends[2 * c] | static_cast<uint64_t>(s_ends[2 * c + 1]) << 32;
  // (all below in positions of the chunk: entry 0 is list entry `begin`)
  const int count = static_cast<int>(min(static_cast<int64_t>(kChunk), a.n - begin));
  auto end_of = [&](int p) -> int {  // one past the end of the run of entry p, 0 <= p; kChunk * 2 if further
    const uint64_t here = p < 64 ? ends[1] >> p : 0;
    if (here != 0) return p + __ffsll(static_cast<long long>(here));
    return ends[2] != 0 ? 64 + __ffsll(static_cast<long long>(ends[2])) : 128;
  };
  int from = 0, head = 0;  // entries before `head` belong to a split run that began in an earlier chunk
  if (!(ends[0] >> 63)) {
    // the first run began in an earlier chunk: that chunk adds it up, unless it is longer than a chunk
    const int start = ends[0] == 0 ? -64 : -static_cast<int>(__clzll(static_cast<long long>(ends[0])));
    const int stop = end_of(0);
    if (ends[0] == 0 || stop - start > kChunk) head = min(stop, count);
    else from = min(stop, count);
  }
  // the last run, if it is not the first one: followed past the chunk's end, unless it is longer than a chunk
  int to = count;
  bool tail = false;
  const int begun = from > head ? from : head;  // runs from here on begin in this chunk
  if (begun < count) {
    const uint64_t before = count >= 2 ? ends[1] & ((uint64_t(1) << (count - 1)) - 1) : 0;  // ends before the last entry
    int last = before == 0 ? 0 : 64 - __clzll(static_cast<long long>(before));
    if (last < begun) last = begun;
    const int stop = end_of(count - 1);
    tail = stop - last > kChunk;
    if (!tail) to = stop;
  }
  const uint32_t col = (slab * blockDim.x + threadIdx.x) * G::kLanes;
  if (tail && slab == 0 && threadIdx.x < 32) {
    const uint32_t last = (WarpLowerBound(a.keys, a.n, s_keys[kChunk + count - 1] + 1) - 1) / kChunk;  // key < rows <= 2^31 - 1
    if (threadIdx.x == 0) {
      const bool many = last - chunk >= kManyParts;
      const uint32_t place = static_cast<uint32_t>(atomicAdd(a.spans + (many ? 1 : 0), 1));
      int2 *list = reinterpret_cast<int2 *>(a.spans + 2);
      list[many ? a.chunks - 1 - place : place] = make_int2(static_cast<int>(chunk), static_cast<int>(last));
    }
  }
  if (col >= a.width) return;
  float acc[G::kLanes];
#pragma unroll
  for (int l = 0; l < G::kLanes; ++l) acc[l] = -0.0f;  // the sum of nothing
  for (int i = from; i < to; i += kDepth) {
    Bits<T, kVec> b[kDepth], d[kAdd ? kDepth : 1];
    int32_t r[kDepth];
    uint32_t stops = 0;  // bit u: a run ends with entry i + u
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const int p = i + u;
      r[u] = p < to ? s_rows[kChunk + p] : -1;
      if (r[u] >= 0) LoadStream(a.g + r[u] * a.ld_g + col, a.width - col, &b[u]);
      const bool stop = p < to && (p == to - 1 || ((p < 64 ? ends[1] >> p : ends[2] >> (p - 64)) & 1u));
      if (stop) stops |= 1u << u;
      if (kAdd && stop && p >= head && !(tail && p == to - 1)) {
        Load(a.grad + s_keys[kChunk + p] * a.ld_grad + col, a.width - col, &d[kAdd ? u : 0]);
      }
    }
#pragma unroll
    for (int u = 0; u < kDepth; ++u) {
      const int p = i + u;
      float v[G::kLanes];
      if (r[u] >= 0) {
        Unpack<T, kVec>(b[u], v);
#pragma unroll
        for (int l = 0; l < G::kLanes; ++l) acc[l] = __fadd_rn(acc[l], v[l]);
      }
      if (!(stops >> u & 1u)) continue;
      if (p < head || (tail && p == to - 1)) {
        float *part = a.parts + (2 * static_cast<int64_t>(chunk) + (p < head ? 0 : 1)) * a.ld_parts + col;
#pragma unroll
        for (int l = 0; l < G::kLanes; ++l) part[l] = acc[l];
      } else if (!kAdd || !AddsNothing(acc)) {
        if (kAdd) Unpack<T, kVec>(d[kAdd ? u : 0], v);
#pragma unroll
        for (int l = 0; l < G::kLanes; ++l) v[l] = __fadd_rn(Scaled(a.scale, acc[l]), kAdd ? v[l] : 0.0f);
        Pack<T, kVec>(v, &b[u]);
        Store(a.grad + s_keys[kChunk + p] * a.ld_grad + col, a.width - col, b[u]);
      }
#pragma unroll
      for (int l = 0; l < G::kLanes; ++l) acc[l] = -0.0f;
    }
  }
}

/*! \brief adds the parts c, c + step, ... up to `last` of a run that begins in `chunk`, 4 columns, eight in flight */
template <typename T>
__device__ __forceinline__ void AddParts(const GradArgs<T> &a, uint32_t c, uint32_t step, uint32_t chunk, uint32_t last,
                                         uint32_t col, float (&acc)[4]) {
  for (; c <= last; c += step * 8) {
    float4 p[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t q = c + step * u;
      p[u] = make_float4(-0.0f, -0.0f, -0.0f, -0.0f);
      if (q <= last) {
        const int64_t row = q == chunk ? 2 * static_cast<int64_t>(q) + 1 : 2 * static_cast<int64_t>(q);
        p[u] = __ldcs(reinterpret_cast<const float4 *>(a.parts + row * a.ld_parts + col));
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      acc[0] = __fadd_rn(acc[0], p[u].x);
      acc[1] = __fadd_rn(acc[1], p[u].y);
      acc[2] = __fadd_rn(acc[2], p[u].z);
      acc[3] = __fadd_rn(acc[3], p[u].w);
    }
  }
}
template <typename T>
__device__ __forceinline__ void WriteFour(const GradArgs<T> &a, int32_t key, uint32_t col, const float (&acc)[4]) {
#pragma unroll
  for (int l = 0; l < 4; ++l) {
    const float one[1] = {acc[l]};
    if (col + l < a.width) WriteRow<T, kOne>(a, key, col + l, one);
  }
}

/*!
 * \brief adds the parts of the split runs.  A run of few parts is one warp's, 128 columns at a time.  A run of many is
 *  shared: a CTA takes 32 of its columns, each quarter of its sixteen warps every 64th part, and they are
 *  joined in order.  Bound by the latency of dependent loads, so what counts is parts in flight.  (One list of runs, a
 *  CTA of eight warps and 128 columns at a time for each: 118 us behind the sums of 2^20 Zipf(1.1) tokens, most
 *  of it for the 2300 parts of the most frequent one; shared by 128 columns and sixteen warps: 59 us.)
 */
template <typename T>
__global__ void __launch_bounds__(512) EmbedSpanKernel(const GradArgs<T> a) {
  gpu_rt::GridDependencySync();
  __shared__ float s_sum[16][32];
  const uint32_t few = static_cast<uint32_t>(a.spans[0]), many = static_cast<uint32_t>(a.spans[1]);
  const int2 *list = reinterpret_cast<const int2 *>(a.spans + 2);
  const uint32_t slabs = (a.width + 127) / 128, strips = (a.width + 31) / 32;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (uint32_t w = blockIdx.x; w < many * strips; w += gridDim.x) {
    const int2 run = list[a.chunks - 1 - w / strips];
    const uint32_t chunk = static_cast<uint32_t>(run.x), last = static_cast<uint32_t>(run.y);
    const int32_t key = a.keys[last * kChunk];
    const uint32_t strip = (w % strips) * 32;
    float acc[4] = {-0.0f, -0.0f, -0.0f, -0.0f};
    AddParts(a, chunk + warp * 4 + lane / 8, 64, chunk, last, strip + (lane & 7) * 4, acc);
#pragma unroll
    for (int l = 0; l < 4; ++l) {
      acc[l] = __fadd_rn(acc[l], __shfl_xor_sync(0xffffffffu, acc[l], 8));
      acc[l] = __fadd_rn(acc[l], __shfl_xor_sync(0xffffffffu, acc[l], 16));
    }
    if (lane < 8) *reinterpret_cast<float4 *>(&s_sum[warp][lane * 4]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    __syncthreads();
    if (threadIdx.x < 32 && strip + threadIdx.x < a.width) {
      float sum[1] = {s_sum[0][threadIdx.x]};
#pragma unroll
      for (int q = 1; q < 16; ++q) sum[0] = __fadd_rn(sum[0], s_sum[q][threadIdx.x]);
      WriteRow<T, kOne>(a, key, strip + threadIdx.x, sum);
    }
    __syncthreads();
  }
  for (uint32_t w = blockIdx.x * 16 + warp; w < few * slabs; w += gridDim.x * 16) {
    const int2 run = list[w / slabs];
    const uint32_t chunk = static_cast<uint32_t>(run.x), last = static_cast<uint32_t>(run.y);
    const int32_t key = a.keys[last * kChunk];
    const uint32_t col = (w % slabs) * 128 + lane * 4;
    float acc[4] = {-0.0f, -0.0f, -0.0f, -0.0f};
    AddParts(a, chunk, 1, chunk, last, col, acc);
    WriteFour(a, key, col, acc);
  }
}

/*!
 * \brief short lists, in one launch and without a sort.  grid: n * slabs CTAs, then (when assigning) CTAs that
 *  write zeros.  The CTA of an entry whose index occurred before does nothing.
 */
template <typename T, int kVec>
__global__ void __launch_bounds__(256) EmbedFewKernel(const GradArgs<T> a) {
  gpu_rt::GridDependencySync();
  typedef Group<T, kVec> G;
  __shared__ int32_t s_rows[kFewTokens];
  __shared__ uint32_t s_votes[kFewTokens / 32];
  __shared__ uint8_t named[kZeroRows];
  __shared__ int s_earlier;
  if (blockIdx.x >= a.n * a.slabs) {
    const uint32_t first = (blockIdx.x - a.n * a.slabs) * kZeroRows;
    const uint32_t last = min(a.table_rows, first + kZeroRows);
    for (uint32_t r = threadIdx.x; r < kZeroRows; r += blockDim.x) named[r] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < a.n; i += blockDim.x) {
      const int32_t k = a.index[i];
      if (k >= static_cast<int64_t>(first) && k < static_cast<int64_t>(last)) named[k - first] = 1;
    }
    __syncthreads();
    WriteZeros<T, kVec>(a, first, last, named);
    return;
  }
  const uint32_t entry = blockIdx.x / a.slabs, slab = blockIdx.x - entry * a.slabs;
  const int32_t key = a.index[entry];
  if (key < 0 || key >= static_cast<int64_t>(a.table_rows)) return;
  if (threadIdx.x == 0) s_earlier = 0;
  __syncthreads();
  for (uint32_t i0 = 0; i0 < a.n; i0 += blockDim.x) {
    const uint32_t i = i0 + threadIdx.x;
    const bool same = i < a.n && a.index[i] == key;
    const uint32_t votes = __ballot_sync(0xffffffffu, same);
    if ((threadIdx.x & 31) == 0 && i < kFewTokens) s_votes[i / 32] = votes;
    if (same && i < entry) s_earlier = 1;
  }
  __syncthreads();
  if (s_earlier) return;
  const uint32_t words = (a.n + 31) / 32;
  uint32_t count = 0;
  for (uint32_t w = 0; w < words; ++w) {
    uint32_t bits = s_votes[w];
    if (threadIdx.x == 0) {
      uint32_t at = count, left = bits;
      while (left != 0) {
        s_rows[at++] = static_cast<int32_t>(w * 32 + __ffs(left) - 1);
        left &= left - 1;
      }
    }
    count += __popc(bits);
  }
  __syncthreads();
  const uint32_t col = (slab * blockDim.x + threadIdx.x) * G::kLanes;
  if (col >= a.width) return;
  float acc[G::kLanes];
#pragma unroll
  for (int l = 0; l < G::kLanes; ++l) acc[l] = -0.0f;
  AddRows<T, kVec>(a, s_rows, 0, count, col, acc);
  WriteRow<T, kVec>(a, key, col, acc);
}

// ---- host side ------------------------------------------------------------------------------------------

template <typename T>
inline bool Aligned(const T *p, int64_t ld, int64_t width) {
  const int64_t lanes = 16 / sizeof(T);
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % lanes == 0 && width % lanes == 0;
}

inline unsigned TakeGrid(uint32_t items, uint32_t per_cta) {
  const int64_t cap = static_cast<int64_t>(gpu_rt::CurrentDevice().sm_count) * 8;
  return static_cast<unsigned>(std::min<int64_t>((static_cast<int64_t>(items) + per_cta - 1) / per_cta, cap));
}

/*! \brief out[i] = scale * table[index[i]]; rows and columns of the tensors as given by n, rows, width */
template <typename T>
inline void TakeLaunch(T *out, int64_t ld_out, const int32_t *index, const T *table, int64_t ld_table, int64_t n,
                       int64_t rows, int64_t width, float scale, cudaStream_t stream) {
  if (n == 0 || width == 0) return;
  const bool aligned = Aligned(out, ld_out, width) && Aligned(table, ld_table, width);
  const uint32_t pieces = static_cast<uint32_t>(aligned ? width / Group<T, kAligned>::kLanes
                                                        : (width + kTakeSegment - 1) / kTakeSegment);
  // the kernels count (token, piece) pairs in 32 bits, with room for a last sweep past the end
  const int64_t block = std::max<int64_t>(1, (int64_t(1) << 30) / pieces);
  for (int64_t i = 0; i < n; i += block) {
    const uint32_t total = static_cast<uint32_t>(std::min(block, n - i)) * pieces;
    if (aligned) {
      gpu_rt::LaunchAfterDrain(EmbedTakeKernel<T>, dim3(TakeGrid(total, 256)), dim3(256), 0, stream, out + i * ld_out, ld_out,
                               index + i, table, ld_table, total, gpu_rt::FastDiv(pieces), static_cast<int32_t>(rows), scale);
    } else {
      // as few lanes as take a segment in one sweep of kTakeDeep loads: short rows share a warp
      const int64_t units = std::min<int64_t>(width, kTakeSegment) * static_cast<int64_t>(sizeof(T)) / 4;
      int lanes_log2 = 2;
      while (lanes_log2 < 5 && (int64_t(kTakeDeep) << lanes_log2) < units) ++lanes_log2;
      gpu_rt::LaunchAfterDrain(EmbedTakeAnywhereKernel<T>, dim3(TakeGrid(total, 256 >> lanes_log2)), dim3(256), 0, stream, out + i * ld_out,
                               ld_out, index + i, table, ld_table, total, gpu_rt::FastDiv(pieces),
                               static_cast<uint32_t>(width), static_cast<int32_t>(rows), scale, lanes_log2);
    }
    MSHADOW_CUDA_POST_KERNEL_CHECK(EmbedTakeKernel);
  }
}

struct GradPlan {
  bool few;
  uint32_t chunks;
  int64_t ld_parts;
  int64_t keys, rows, sort, parts, spans, bytes;  // offsets
};

inline GradPlan MakeGradPlan(int64_t n, int64_t width) {
  GradPlan p = {};
  p.few = n <= kFewTokens;
  if (p.few) return p;
  p.chunks = static_cast<uint32_t>((n + kChunk - 1) / kChunk);
  p.ld_parts = (width + 127) / 128 * 128;
  int64_t at = 0;
  auto take = [&at](int64_t bytes) {
    const int64_t was = at;
    at += (bytes + 255) / 256 * 256;
    return was;
  };
  p.keys = take(n * 4);
  p.rows = take(n * 4);
  p.sort = take(static_cast<int64_t>(sortdetail::ScratchBytes(n)));
  p.parts = take(2ll * p.chunks * p.ld_parts * 4);
  p.spans = take((1ll + p.chunks) * 8);
  p.bytes = at;
  return p;
}

template <typename T, int kVec>
inline void GradGo(GradArgs<T> a, const GradPlan &p, char *ws, cudaStream_t stream) {
  const uint32_t items = (a.width + Group<T, kVec>::kLanes - 1) / Group<T, kVec>::kLanes;
  const uint32_t threads = std::min(256u, (items + 31) / 32 * 32);
  a.slabs = (items + threads - 1) / threads;
  const uint32_t zero = a.add ? 0 : (a.table_rows + kZeroRows - 1) / kZeroRows;
  CHECK_LT(static_cast<uint64_t>(p.few ? a.n : p.chunks) * a.slabs + zero, uint64_t(1) << 31)
      << "EmbedTakeGrad: more indices times columns than one launch covers";
  if (p.few) {
    const uint32_t grid = a.n * a.slabs + zero;
    if (grid == 0) return;
    gpu_rt::LaunchAfterDrain(EmbedFewKernel<T, kVec>, dim3(grid), dim3(threads), 0, stream, a);
    MSHADOW_CUDA_POST_KERNEL_CHECK(EmbedFewKernel);
    return;
  }
  int32_t *keys = reinterpret_cast<int32_t *>(ws + p.keys), *rows = reinterpret_cast<int32_t *>(ws + p.rows);
  int bits = 1;
  while (bits < 31 && (int64_t(1) << bits) < a.table_rows) ++bits;
  a.spans = reinterpret_cast<int32_t *>(ws + p.spans);
  if (a.n <= static_cast<uint32_t>(kOneCta)) {
    const int passes = (bits + 8) / 9, digit_bits = (bits + passes - 1) / passes;
    const size_t pairs = (a.n + 1023) / 1024 * 1024, digits = size_t(1) << digit_bits;
    const size_t smem = pairs * 6 + digits * (32 * 2 + 4), most = size_t(kOneCta) * 6 + 512 * (32 * 2 + 4);
    gpu_rt::AllowSharedMemory(EmbedSortKernel<0>, most);
    gpu_rt::LaunchAfterDrain(EmbedSortKernel<0>, dim3(1), dim3(1024), smem, stream, keys, rows, a.index, a.n, a.table_rows, passes,
                             digit_bits, a.spans);
    MSHADOW_CUDA_POST_KERNEL_CHECK(EmbedSortKernel);
  } else {
    // (Writing the zeros by further CTAs of the sort's launches instead was slower: 186 against 165 us for 16384 indices
    // into 131072 x 2048 bf16 -- writes alone run at 3.9 TB/s however they are issued, and each of the six launches
    // drained its share of them before the next began.)
    MSHADOW_CUDA_CALL(cudaMemsetAsync(a.spans, 0, 8, stream));
    const sortdetail::Source named = {static_cast<int>(a.table_rows), 1};
    sortdetail::SortPairs<int32_t, int32_t>(keys, rows, a.index, a.n, bits, true, named, ws + p.sort, stream);
  }
  a.keys = keys, a.rows = rows;
  a.chunks = p.chunks;
  a.parts = reinterpret_cast<float *>(ws + p.parts), a.ld_parts = p.ld_parts;
  if (a.add) {
    gpu_rt::LaunchAfterDrain(EmbedSumKernel<T, kVec, true>, dim3(a.chunks * a.slabs), dim3(threads), 0, stream, a);
  } else {
    gpu_rt::LaunchAfterDrain(EmbedSumKernel<T, kVec, false>, dim3(a.chunks * a.slabs + zero), dim3(threads), 0, stream, a);
  }
  MSHADOW_CUDA_POST_KERNEL_CHECK(EmbedSumKernel);
  const int64_t most = static_cast<int64_t>(p.chunks) * ((a.width + 127) / 128);
  const int64_t cap = static_cast<int64_t>(gpu_rt::CurrentDevice().sm_count) * 4;
  gpu_rt::LaunchAfterDrain(EmbedSpanKernel<T>, dim3(static_cast<unsigned>(std::min(most, cap))), dim3(512), 0, stream, a);
  MSHADOW_CUDA_POST_KERNEL_CHECK(EmbedSpanKernel);
}

/*! \brief grad[r] (=|+=) scale * sum of the rows of g whose index is r */
template <typename T>
inline void GradLaunch(T *grad, int64_t ld_grad, const T *g, int64_t ld_g, const int32_t *index, int64_t n, int64_t rows,
                       int64_t width, float scale, bool add, const GradPlan &p, char *ws, cudaStream_t stream) {
  if (rows == 0 || width == 0 || (n == 0 && add)) return;
  GradArgs<T> a = {};
  a.grad = grad, a.ld_grad = ld_grad, a.g = g, a.ld_g = ld_g, a.index = index;
  a.n = static_cast<uint32_t>(n), a.width = static_cast<uint32_t>(width), a.table_rows = static_cast<uint32_t>(rows);
  a.scale = scale, a.add = add;
  if (Aligned(grad, ld_grad, width) && (n == 0 || Aligned(g, ld_g, width))) GradGo<T, kAligned>(a, p, ws, stream);
  else GradGo<T, kAnywhere>(a, p, ws, stream);
}

}  // namespace embtake
}  // namespace cuda
}  // namespace mshadow
#endif  // MSHADOW_GPU_EMBED_TAKE_CUH_
