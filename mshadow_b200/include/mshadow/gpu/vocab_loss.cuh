/*
 * Softmax cross entropy over a large vocabulary without keeping the logits, and its gradients.
 *
 *   z = x W^T (n tokens x v classes, contraction over h),  m = max z,  lse = m + log sum exp(z - m)
 *   loss = lse - (1 - a) z_label - a / (v - 1) * (sum z - z_label)
 *   d    = (exp(z - lse) - q) * row_scale,  q = 1 - a at the label, a / (v - 1) elsewhere
 *   grad x = d W,   grad W (=|+=) d^T x
 *
 * A token whose label is `ignore`, or lies outside [0, v), is not live: loss, lse and gradient 0.
 *
 * The products run on the tensor cores: 16-bit operands, binary32 accumulators in tensor memory,
 * one persistent CTA (or pair of CTAs) per SM (or pair of SMs) whose warps have fixed roles -- one
 * thread issues the tiled copies of the operands, one the products, eight warps (two threads per
 * tile row) take the finished accumulators while the next tile's products run into the other
 * half of the tensor memory.  All waits are bounded.
 *
 * Forward: a tile of logits never leaves tensor memory; its row maxima and sums of
 * exponentials (8 bytes per row and tile) do, and a second kernel joins them over the tiles.
 *
 * Backward, piece of the vocabulary after piece: the tile of logits is computed again, turned into
 * d, rounded to the operands' type and stored (n x piece); d W adds to the binary32 gradient of x,
 * and d^T x is the piece's gradient of W.  The rounding of d is the one rounding between inputs and
 * outputs besides the final one: it is what lets the second and third product run on 16-bit
 * operands, and it is relative to each d (half a unit of its last place), so the gradients come
 * out about as exact as their own final rounding leaves them.  What is stored is not d itself but
 *     d' = (p - q) / (1 - a) * gloss * 2^k,     d = d' * scale * (1 - a) * 2^-k
 * with 2^k bringing the largest finite |gloss| / (1 - a) to 2^14 .. 2^15, and the factor on the right applied to the
 * finished sums: a mean over thousands of tokens would put most of d below the smallest binary16 number, and the
 * label's term, which carries most of the gradient while p is small, would be rounded by the same fraction in every
 * row -- as stored it is a power of two.  (With scale and 1 - a inside: gradients of 0.31 % instead of 0.17 %
 * relative error, bf16, smoothing 0.1; 0.21 instead of 0.17 % without smoothing.)
 * binary16 has too few exponents for one k: a token whose |gloss| is less than 2^-6 of the largest gets a k of its own for the
 * gradient of x, whose row it alone determines, and its row of d' is brought back to the common k before the gradient
 * of W, where it stands beside the others.  There an entry of d below 2^-39 of the largest |gloss| / (1 - a) is lost.
 *
 * Live tokens are packed together first (PackRowsKernel): tiles of padding cost nothing, whatever
 * their hidden states hold -- an infinity in a padded row does not meet a zero of d -- and the
 * packed rows are aligned for the tiled copies whatever the caller's layout.
 */
#ifndef MSHADOW_GPU_VOCAB_LOSS_CUH_
#define MSHADOW_GPU_VOCAB_LOSS_CUH_

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "./tcgen05.cuh"

namespace mshadow {
namespace cuda {
namespace vloss {

const int kTileN = 256;       // columns of a tile
const int kStepK = 64;        // contraction elements per stage (one 128-byte swizzle row)
const int kThreads = 384;     // warp 0: copies, warp 1: products, warp 2: tensor memory, warps 4-11: epilogue
const int kHalfN = kTileN / 2;  // columns of a tile that one epilogue group (four warps, a thread per row) takes
const uint32_t kBoxOut = 128 * 128;  // a box of 128 rows by 128 bytes, on its way out through shared memory
const int kWideSteps = 24;    // steps from which d and grad W are computed in tiles of 512 columns (below)
const int kPadRows = 256;     // token rows of the scratch matrices are padded to this
const float kLog2e = 1.4426950408889634f;

/*! \brief what the kernel does with a finished tile, and how its operands lie */
enum Mode {
  kStat,        // A = tokens, B = vocabulary rows, both along the contraction; row maxima and sums
  kDelta,       // same product; d stored
  kDataGrad,    // A = d (along), B = vocabulary rows (across); binary32 partial gradient of x
  kWeightGrad,  // A = d (across), B = tokens (across); gradient of a piece of W
};

template <int kMode>
struct Layout {
  static const bool kAAcross = kMode == kWeightGrad;
  static const bool kBAcross = kMode == kDataGrad || kMode == kWeightGrad;
};

/*!
 * \brief stages per run of accumulation in tensor memory (VocabGemmKernel): 1024 contraction elements for the loss; 8192 for the
 *  logits of the gradient, whose exponentials are rounded to 16 bits, and for sums that stay binary32; 16384 for
 *  sums that are rounded to 16 bits themselves
 */
__host__ __device__ __forceinline__ int RunSteps(int mode, bool wide_out) {
  return mode == kStat ? 16 : mode == kDelta || wide_out ? 128 : 256;
}
/*! \brief first stage of run `run` of a contraction of `steps` */
template <int kMode>
__device__ __forceinline__ int RunBegin(int run, int runs, int steps, int run_steps) {
  return kMode == kStat ? run * steps / runs : run < runs ? run * run_steps : steps;
}

/*! \brief kWide: a pair's tile is 512 columns wide, two sets of 256, and fills the tensor memory */
template <int kMode, int kCtas, bool kWide>
struct StageShape {
  static const int kRowsN = kTileN / kCtas;                          // rows of B that a CTA holds, of a set
  static const int kSets = kWide ? 2 : 1;                            // sets of accumulators per tile
  static const uint32_t kBytesA = 128 * kStepK * 2;
  static const uint32_t kBytesB = kRowsN * kStepK * 2;
  static const uint32_t kStage = kBytesA + kSets * kBytesB;
  // Five stages of 32 KB are enough where there is something to send: the sixth's place is worth more as a second
  // outgoing box for each epilogue group (d of 8192 x 32768 x 512: 3 %).  kStat sends nothing (and is 2 % faster with
  // six than with five; seven are no better).
  static const int kStages = kCtas != 2 || kWide ? 4 : kMode == kStat ? 6 : 5;
  static const int kBoxes = kMode == kStat ? 0 : kCtas == 2 && !kWide ? 2 : 1;  // outgoing boxes of an epilogue group
  static const uint32_t kOut = kStage * kStages;
  static const size_t kSmem = kOut + 2 * kBoxes * kBoxOut + 1024;    // + alignment to the swizzle's 1024 bytes
};

struct GemmArgs {
  // extents
  const int32_t *live;   // device word: token rows that count; null: `tokens` do
  int32_t tokens;
  int32_t m_tiles;       // kWeightGrad: row tiles of the piece (else from the live rows)
  int32_t n_tiles;
  int32_t k_blocks;      // kWeightGrad: from the live rows
  int32_t k_plan;        // kDataGrad: k_blocks of the first piece, by which all pieces are cut into the same parts
  int32_t room;          // kDataGrad: tiles that there is room for beside the gradient itself, for parts of tiles
  float step_cycles, tile_cycles;  // kDataGrad: what CutOf counts
  int32_t group;         // row tiles that are walked before the next column tile
  int32_t b_row0;        // first row of B (the piece's first vocabulary row)
  uint32_t instr;
  // kStat, kDelta
  int32_t cols;          // columns of the piece that exist
  int32_t col0;          // class of the piece's first column
  int32_t tile_n;        // kStat: columns of a tile, a multiple of 16 * CTAs and at most kTileN
  int32_t tile0;         // kStat: tiles of the pieces before this one
  int64_t pad_rows;
  const int32_t *label;
  float2 *part;          // [tile][half][row]: maximum and sum of exp(z - maximum)
  float *part_sum;       // [tile][half][row]: sum of z, or null
  float *label_logit;    // [row]
  const float *lse2;     // [row]: lse in base 2
  const float *row_scale;
  float q_label, q_other;
  int bf16;
  // kDataGrad
  int accumulate;
  // kWeightGrad
  const float *inv_scale;  // device word: what takes sums of d' to the gradient
  void *out;
  int64_t ld_out;
  int32_t out_rows, out_cols;
  int out_type;          // kFloat32, kFloat16, kBfloat16
  int out_add;
  int out_vec;           // rows of `out` start on 16-byte boundaries
  int out_tiled;         // written by tiled copies (map_out)
  int run_steps;         // RunSteps
  float4 *earlier;       // kRuns: sums of earlier runs (EarlierOf)
  int *status;
};

__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t PackPair(float a, float b, int bf16) {
  if (bf16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
  }
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&p);
}
__device__ __forceinline__ float Widen(uint16_t bits, int bf16) {
  return bf16 ? __uint_as_float(static_cast<uint32_t>(bits) << 16) : __half2float(__ushort_as_half(bits));
}

/*! \brief a piece of work: tile (m, n), part `slice` of `parts` of its contraction; `spare`: its place beside the gradient */
struct Unit {
  int m, n, slice, parts, spare;
};

/*!
 * \brief how the walk over `tiles` tiles is cut: the first `full` of them whole, whole rounds over the GPU, and the
 *  `rest`, which would leave part of it idle for a round, in `parts` parts of their contraction each
 */
struct Cut {
  int full, rest, parts;
  __device__ __forceinline__ int Units() const { return full + rest * parts; }
};

/*!
 * \brief the cut for grad x, the same in every thread of a warp that asks.  n x h has few tiles and a contraction as long
 *  as the vocabulary piece.  Of 1 .. 16 parts, at least eight steps long and as many as there is room for,
 *  the cheapest by this count: rounds over the `slots` of the GPU, step_cycles a step, some 4000 to begin and
 *  end a part, and tile_cycles to write a part of a tile and read it again.  Decided on the device, by the
 *  tokens that count.
 */
__device__ __forceinline__ Cut CutOf(int m_tiles, int n_tiles, int k_blocks, int room, int slots, float step_cycles,
                                     float tile_cycles) {
  Cut cut;
  const int tiles = m_tiles * n_tiles;
  cut.full = tiles / slots * slots;
  cut.rest = tiles - cut.full;
  const int parts = (threadIdx.x & 15) + 1;
  const bool fits = parts == 1 || (parts * 8 <= k_blocks && parts * cut.rest <= room);
  const float rounds = static_cast<float>((cut.rest * parts + slots - 1) / slots);
  const float steps = static_cast<float>((k_blocks + parts - 1) / parts);
  // (each operation rounded by itself: the two kernels that ask must not differ by how theirs is compiled)
  float cost = __fadd_rn(__fmul_rn(rounds, __fadd_rn(__fmul_rn(steps, step_cycles), 4000.0f)),
                         __fmul_rn(static_cast<float>(parts * cut.rest), tile_cycles));
  if (!fits) cost = INFINITY;
  cut.parts = parts;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, cost, o);
    const int which = __shfl_xor_sync(0xffffffffu, cut.parts, o);
    if (other < cost || (other == cost && which < cut.parts)) cost = other, cut.parts = which;
  }
  return cut;
}

/*! \brief work w of the walk: `group` row tiles by all column tiles, then the next group; parts outermost */
__device__ __forceinline__ Unit UnitOf(int w, const Cut &cut, int m_tiles, int n_tiles, int group) {
  Unit t = {0, 0, 0, 1, 0};
  int r = w;
  if (w >= cut.full) {
    t.parts = cut.parts;
    t.slice = (w - cut.full) / cut.rest;
    r = w - t.slice * cut.rest;
    t.spare = (r - cut.full) * cut.parts + t.slice;
  }
  const int band = group * n_tiles;
  const int g = r / band;
  const int first = g * group;
  const int height = min(group, m_tiles - first);
  const int q = r - g * band;
  t.n = q / height;
  t.m = first + (q - t.n * height);
  return t;
}
/*! \brief place of tile (m, n) in that walk */
__device__ __forceinline__ int PlaceOf(int m, int n, int m_tiles, int n_tiles, int group) {
  const int first = m / group * group;
  return first * n_tiles + n * min(group, m_tiles - first) + (m - first);
}

// ---- epilogues: one thread per row of the tile and half of its columns ----------------------------

/*! \brief what an epilogue group (four warps) knows about its half of a tile */
struct Half {
  uint32_t acc;      // tensor memory of this thread's row, first column of the half
  int64_t row;       // row of the matrix
  int col;           // first column of the half, within the piece
  uint32_t boxes, box;  // shared memory of the group's first outgoing box; which one is filled next
  int group, thread; // 0 / 1; thread of the group: 0 .. 127
  float4 *earlier;   // kRuns: this thread's sums of the tile's earlier runs, or null: there are none
  __device__ __forceinline__ uint32_t Box() const { return boxes + box * 2 * kBoxOut; }
};

// ---- sums of earlier runs: 128 columns of a row per thread and set of accumulators, read and written by that thread alone -----

const int kEarlierStep = 256;  // groups of four columns of a thread are this far apart: a warp's lie side by side
const int64_t kEarlierBytes = int64_t(2) * (kHalfN / 4) * kEarlierStep * 16;  // of a CTA: two sets
__device__ __forceinline__ float4 *EarlierOf(float4 *all, int set) {
  return all + (static_cast<int64_t>(blockIdx.x) * 2 + set) * (kHalfN / 4) * kEarlierStep + (threadIdx.x - 128);
}
/*! \brief accumulators of the columns from `col` on, plus those of the earlier runs */
template <bool kRuns, int kColumns>
__device__ __forceinline__ void AddEarlier(const Half &t, int col, uint32_t (&r)[kColumns]) {
  if (!kRuns || t.earlier == nullptr) return;
#pragma unroll
  for (int q = 0; q < kColumns / 4; ++q) {
    const float4 e = t.earlier[(col / 4 + q) * kEarlierStep];
    r[4 * q] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * q]), e.x));
    r[4 * q + 1] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * q + 1]), e.y));
    r[4 * q + 2] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * q + 2]), e.z));
    r[4 * q + 3] = __float_as_uint(__fadd_rn(__uint_as_float(r[4 * q + 3]), e.w));
  }
}
/*! \brief a run that is not its tile's last: its sums, and those of the runs before it, are kept */
__device__ __forceinline__ void KeepHalf(const Half &t, float4 *keep) {
#pragma unroll 1
  for (int b = 0; b < kHalfN / 32; ++b) {
    uint32_t r[32];
    tc5::LoadColumns(t.acc + b * 32, r);
    tc5::WaitColumns(r);
    AddEarlier<true>(t, b * 32, r);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      keep[(b * 8 + q) * kEarlierStep] = make_float4(__uint_as_float(r[4 * q]), __uint_as_float(r[4 * q + 1]),
                                                     __uint_as_float(r[4 * q + 2]), __uint_as_float(r[4 * q + 3]));
    }
  }
}

/*!
 * \brief before a box is filled.  With two boxes the next one is known to be free already (BoxSend); a single one is
 *  waited for.
 */
template <int kBoxes>
__device__ __forceinline__ void BoxFree(Half *t) {
  if (kBoxes == 2) {
    t->box ^= 1u;
    return;
  }
  if (t->thread == 0) tc5::WaitStoresRead();
  tc5::NamedBarrier(1 + t->group, 128);
}
/*! \brief 16 bytes of this thread's row of the box, in the place the 128-byte swizzle gives them */
__device__ __forceinline__ void BoxPut(const Half &t, int chunk, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t at = t.Box() + t.thread * 128 + ((chunk ^ (t.thread & 7)) << 4);
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
/*!
 * \brief the box is full: one thread sends it to column x, row y of the output.  With two boxes that thread first sees to
 *  it that the other one has been read (it was sent a box ago), so that one barrier says both.
 */
template <int kBoxes, bool kAdd>
__device__ __forceinline__ void BoxSend(const Half &t, const CUtensorMap *map, int x, int y) {
  tma::FenceAsyncShared();
  if (kBoxes == 2 && t.thread == 0) tc5::WaitStoresRead();
  tc5::NamedBarrier(1 + t.group, 128);
  if (t.thread == 0) tc5::StoreBox<kAdd>(map, x, y, t.Box());
}

/*!
 * \brief maximum and sum of exponentials of the half row, 128 logits in pairs.
 *
 *  The change of base and the difference to the maximum are one multiply-add, z log2 e - r, with r = the rounded
 *  m log2 e; what r was rounded by is taken out of the sum again, so that its largest term is 1 and the loss of a
 *  token whose label has the largest logit is log(sum) with nothing cancelled.  In pairs these and the
 *  additions run at twice the rate of single ones; bound by the exponentials, 16 a cycle and SM.  (Single
 *  operations, difference first: 33 % more time at 128 features.)
 */
__device__ __forceinline__ void StatHalf(uint64_t (&v)[kHalfN / 2], const Half &own, int limit, int label, int64_t at,
                                         const GemmArgs &a) {
  if (limit < kHalfN) {  // columns past the vocabulary weigh nothing
#pragma unroll
    for (int i = 0; i < kHalfN / 2; ++i) {
      float lo, hi;
      tc5::Unpair(v[i], &lo, &hi);
      v[i] = tc5::Pair(2 * i < limit ? lo : -INFINITY, 2 * i + 1 < limit ? hi : -INFINITY);
    }
  }
  if (a.part_sum != nullptr) {
    uint64_t t[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kHalfN / 2; ++i) {
      float lo, hi;
      tc5::Unpair(v[i], &lo, &hi);
      t[i & 3] = tc5::AddPair(t[i & 3], tc5::Pair(2 * i < limit ? lo : 0.0f, 2 * i + 1 < limit ? hi : 0.0f));
    }
    float lo, hi;
    tc5::Unpair(tc5::AddPair(tc5::AddPair(t[0], t[1]), tc5::AddPair(t[2], t[3])), &lo, &hi);
    a.part_sum[at] = lo + hi;
  }
  float m[8];
#pragma unroll
  for (int i = 0; i < kHalfN / 2; ++i) {
    float lo, hi;
    tc5::Unpair(v[i], &lo, &hi);
    m[i & 7] = i < 8 ? fmaxf(lo, hi) : fmaxf(fmaxf(m[i & 7], lo), hi);
  }
#pragma unroll
  for (int i = 4; i > 0; i >>= 1) {
#pragma unroll
    for (int j = 0; j < i; ++j) m[j] = fmaxf(m[j], m[j + i]);
  }
  if (label >= 0 && label < min(limit, kHalfN)) {
    uint64_t z = v[0];
#pragma unroll
    for (int i = 1; i < kHalfN / 2; ++i) z = i == label >> 1 ? v[i] : z;
    float lo, hi;
    tc5::Unpair(z, &lo, &hi);
    a.label_logit[own.row] = label & 1 ? hi : lo;
  }
  const float from = m[0] == -INFINITY ? 0.0f : m[0];  // nothing but -infinity: any finite reference serves
  const float base = -from * kLog2e;
  const uint64_t log2e = tc5::Pair(kLog2e, kLog2e), bases = tc5::Pair(base, base);
  uint64_t s[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < kHalfN / 2; ++i) {
    float lo, hi;
    tc5::Unpair(tc5::FmaPair(v[i], log2e, bases), &lo, &hi);
    s[i & 3] = tc5::AddPair(s[i & 3], tc5::Pair(Exp2(lo), Exp2(hi)));
  }
  float lo, hi;
  tc5::Unpair(tc5::AddPair(tc5::AddPair(s[0], s[1]), tc5::AddPair(s[2], s[3])), &lo, &hi);
  a.part[at] = make_float2(m[0], (lo + hi) * Exp2(-__fmaf_rn(from, kLog2e, base)));
}

/*! \brief d' of 32 columns, in pairs */
__device__ __forceinline__ void DeltaColumns(const uint32_t (&r)[32], int limit, int label, float lse2, float scale,
                                             const GemmArgs &a, uint32_t (&out)[16]) {
  const float other = -a.q_other * scale;
  const uint64_t log2e = tc5::Pair(kLog2e, kLog2e), bases = tc5::Pair(-lse2, -lse2), scales = tc5::Pair(scale, scale),
                 others = tc5::Pair(other, other);
  float d[32];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float lo, hi;
    tc5::Unpair(tc5::FmaPair(tc5::Pair(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), log2e, bases), &lo, &hi);
    tc5::Unpair(tc5::FmaPair(tc5::Pair(Exp2(lo), Exp2(hi)), scales, others), &d[2 * i], &d[2 * i + 1]);
  }
  if (static_cast<unsigned>(label) < 32u) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i == label) d[i] = (Exp2(__fmaf_rn(__uint_as_float(r[i]), kLog2e, -lse2)) - a.q_label) * scale;
    }
  }
  if (limit < 32) {
#pragma unroll
    for (int i = 0; i < 32; ++i) d[i] = i < limit ? d[i] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) out[i] = PackPair(d[2 * i], d[2 * i + 1], a.bf16);
}

template <int kBoxes, bool kRuns>
__device__ __forceinline__ void DeltaHalf(Half &t, int limit, int label, float lse2, float scale, const CUtensorMap *map,
                                          int row0, const GemmArgs &a) {
#pragma unroll 1
  for (int b = 0; b < kHalfN / 64; ++b) {
    uint32_t r0[32], r1[32], p0[16], p1[16];
    tc5::LoadColumns(t.acc + b * 64, r0);
    tc5::LoadColumns(t.acc + b * 64 + 32, r1);
    tc5::WaitColumns(r0);
    tc5::WaitColumns(r1);
    AddEarlier<kRuns>(t, b * 64, r0);
    AddEarlier<kRuns>(t, b * 64 + 32, r1);
    DeltaColumns(r0, limit - b * 64, label - b * 64, lse2, scale, a, p0);
    DeltaColumns(r1, limit - b * 64 - 32, label - b * 64 - 32, lse2, scale, a, p1);
    BoxFree<kBoxes>(&t);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      BoxPut(t, q, p0[4 * q], p0[4 * q + 1], p0[4 * q + 2], p0[4 * q + 3]);
      BoxPut(t, 4 + q, p1[4 * q], p1[4 * q + 1], p1[4 * q + 2], p1[4 * q + 3]);
    }
    BoxSend<kBoxes, false>(t, map, t.col + b * 64, row0);
  }
}

/*! \brief the half tile as binary32, times `factor`, stored or added */
template <int kBoxes, bool kRuns, bool kAdd>
__device__ __forceinline__ void FloatHalf(Half &t, float factor, const CUtensorMap *map, int x, int y) {
#pragma unroll 1
  for (int b = 0; b < kHalfN / 32; ++b) {
    uint32_t r[32];
    tc5::LoadColumns(t.acc + b * 32, r);
    tc5::WaitColumns(r);
    AddEarlier<kRuns>(t, b * 32, r);
#pragma unroll
    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * factor);
    BoxFree<kBoxes>(&t);
#pragma unroll
    for (int q = 0; q < 8; ++q) BoxPut(t, q, r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
    BoxSend<kBoxes, kAdd>(t, map, x + b * 32, y);
  }
}

/*! \brief the half tile in the operands' type, times `factor` */
template <int kBoxes, bool kRuns>
__device__ __forceinline__ void PackedHalf(Half &t, float factor, int bf16, const CUtensorMap *map, int row0) {
#pragma unroll 1
  for (int b = 0; b < kHalfN / 64; ++b) {
    uint32_t r0[32], r1[32];
    tc5::LoadColumns(t.acc + b * 64, r0);
    tc5::LoadColumns(t.acc + b * 64 + 32, r1);
    tc5::WaitColumns(r0);
    tc5::WaitColumns(r1);
    AddEarlier<kRuns>(t, b * 64, r0);
    AddEarlier<kRuns>(t, b * 64 + 32, r1);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      r0[i] = PackPair(__uint_as_float(r0[2 * i]) * factor, __uint_as_float(r0[2 * i + 1]) * factor, bf16);
      r1[i] = PackPair(__uint_as_float(r1[2 * i]) * factor, __uint_as_float(r1[2 * i + 1]) * factor, bf16);
    }
    BoxFree<kBoxes>(&t);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      BoxPut(t, q, r0[4 * q], r0[4 * q + 1], r0[4 * q + 2], r0[4 * q + 3]);
      BoxPut(t, 4 + q, r1[4 * q], r1[4 * q + 1], r1[4 * q + 2], r1[4 * q + 3]);
    }
    BoxSend<kBoxes, false>(t, map, t.col + b * 64, row0);
  }
}

/*! \brief 32 columns of a row of grad W by plain accesses: rows that the tiled copy cannot address, and additions */
__device__ __forceinline__ void WeightColumns(const uint32_t (&r)[32], int64_t row, int col, float inv, const GemmArgs &a) {
  const int left = a.out_cols - col;
  if (left <= 0) return;
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) * inv;
  if (a.out_type == kFloat32) {
    float *out = static_cast<float *>(a.out) + row * a.ld_out + col;
    if (a.out_vec && left >= 32) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float4 *p = reinterpret_cast<float4 *>(out) + q;
        float4 w = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        if (a.out_add) {
          const float4 o = *p;
          w.x += o.x, w.y += o.y, w.z += o.z, w.w += o.w;
        }
        *p = w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (i < left) out[i] = a.out_add ? out[i] + v[i] : v[i];
      }
    }
    return;
  }
  const int bf16 = a.out_type == kBfloat16;
  uint16_t *out = static_cast<uint16_t *>(a.out) + row * a.ld_out + col;
  if (a.out_vec && left >= 32) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint4 *p = reinterpret_cast<uint4 *>(out) + q;
      if (a.out_add) {
        const uint4 o = *p;
        const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[8 * q + 2 * j] += Widen(static_cast<uint16_t>(w[j] & 0xffffu), bf16);
          v[8 * q + 2 * j + 1] += Widen(static_cast<uint16_t>(w[j] >> 16), bf16);
        }
      }
      uint4 w;
      w.x = PackPair(v[8 * q], v[8 * q + 1], bf16);
      w.y = PackPair(v[8 * q + 2], v[8 * q + 3], bf16);
      w.z = PackPair(v[8 * q + 4], v[8 * q + 5], bf16);
      w.w = PackPair(v[8 * q + 6], v[8 * q + 7], bf16);
      *p = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i < left) {
        const float t = a.out_add ? v[i] + Widen(out[i], bf16) : v[i];
        out[i] = static_cast<uint16_t>(PackPair(t, 0.0f, bf16) & 0xffffu);
      }
    }
  }
}

/*!
 * \brief 32 columns of grad W of the warp's 32 rows, for rows that start at any element: the accumulators change places
 *  in shared memory (the warp's own part of the outgoing box), so that a warp writes a row's 32 columns at
 *  once instead of every thread its own row, element by element (60000 x 300 bf16: 202 us, now 72)
 */
__device__ __forceinline__ void WeightRows(const uint32_t (&r)[32], const Half &t, int64_t row0, int col, float inv,
                                           const GemmArgs &a) {
  const int lane = t.thread & 31;
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 8; ++q) BoxPut(t, q, r[4 * q], r[4 * q + 1], r[4 * q + 2], r[4 * q + 3]);
  __syncwarp();
  const bool in = col + lane < a.out_cols;
  const uint32_t box = t.Box() + (t.thread & ~31) * 128;
  const int64_t first = (row0 + (t.thread & ~31)) * a.ld_out + col + lane;
  const int rows = static_cast<int>(min(static_cast<int64_t>(32), a.out_rows - (row0 + (t.thread & ~31))));
#pragma unroll 8
  for (int i = 0; i < rows; ++i) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(box + i * 128 + (((lane >> 2) ^ (i & 7)) << 4) + (lane & 3) * 4) : "memory");
    v *= inv;
    if (!in) continue;
    if (a.out_type == kFloat32) {
      float *out = static_cast<float *>(a.out) + first + i * a.ld_out;
      *out = a.out_add ? *out + v : v;
    } else {
      const int bf16 = a.out_type == kBfloat16;
      uint16_t *out = static_cast<uint16_t *>(a.out) + first + i * a.ld_out;
      if (a.out_add) v += Widen(*out, bf16);
      *out = static_cast<uint16_t>(PackPair(v, 0.0f, bf16) & 0xffffu);
    }
  }
}

/*!
 * \brief persistent product kernel of all four modes.  kCtas CTAs (a cluster) share a tile of
 *  128 * kCtas rows by 256 columns (kStat: a.tile_n; kWide: 512).  Dynamic shared memory StageShape::kSmem.
 *
 *  Tensor memory holds two sets of accumulators; the products of one run into them while the epilogue empties the
 *  other.  The contraction is cut into runs (RunSteps) that are added up in binary32 outside of it, because the
 *  tensor cores cut off, rather than round, each time they add to an accumulator, always towards zero.  kStat adds its runs
 *  of 1024 elements up in registers: over 4096 elements the loss was off by 1.8e-6 of its value in one run, by 4e-7 in
 *  these, which cost 1 % of the time (plain binary32: 6e-7 there, 3e-8 to 4e-8 at 1000 to 2000 features; runs of 512:
 *  2.5e-7 and another 3 %; of 256: 17 %).  The other modes keep the sums of a tile's runs in memory (38 MB for all CTAs,
 *  written and read once per run, some 20 000 cycles).  Without runs the gradient of W of a class that 65536 tokens name was
 *  off by 4.2e-4 of its value, and by 1.7e-3 at 262144, however well the rounding of d' averages out; now by 5e-5, for 1 %
 *  of the time of 2048 x 32000 x 4096 and 1.5 % of 32768 x 32000 x 2048 with the gradient of W as binary32 (with runs of
 *  8192 for all sums: 3.5 % of 8192 x 131072 x 4096).  kRuns: for calls with a contraction longer than a run; kernels apart,
 *  since the registers of those sums keep the next kernel off the SM, 1 to 3 us of a small call.
 *
 *  kWide: both sets belong to one tile.  A step's rows of A then serve 512 columns, a quarter less is read from the L2
 *  and, where A is d', from memory; in return the products wait while a tile is emptied.  For long contractions (not
 *  in kStat, whose runs would be emptied too often).
 */
template <int kMode, int kCtas, bool kWide, bool kRuns>
__global__ void __launch_bounds__(kThreads, 1)
VocabGemmKernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_out, const GemmArgs a) {
  // map_x: the rows of x where the caller has them; kDataGrad: the parts of tiles beside the gradient
  typedef StageShape<kMode, kCtas, kWide> S;
  typedef Layout<kMode> L;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  const uint32_t smem = (tma::SharedAddr(raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kCtas == 2 ? tc5::ClusterRank() : 0u;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      tma::BarrierInit(&full[s], 1);
      tma::BarrierInit(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      tma::BarrierInit(&acc_full[s], 1);
      tma::BarrierInit(&acc_empty[s], 8 * kCtas);
    }
    tc5::PrefetchMap(&map_a);
    tc5::PrefetchMap(&map_b);
    tc5::PrefetchMap(&map_x);
    if (kMode != kStat) tc5::PrefetchMap(&map_out);
  }
  if (warp == 2) tc5::AllocTensorMemory<kCtas>(&tmem_slot);
  tc5::FenceBefore();
  __syncthreads();
  if (kCtas == 2) tc5::ClusterSync();
  tc5::FenceAfter();
  const uint32_t tmem = tmem_slot;
  gpu_rt::GridDependencySync();

  const int live = a.live != nullptr ? a.live[0] : a.tokens;
  // every token counts: the rows of x were not packed, and are read from where the caller has them
  const bool in_place = kMode != kDataGrad && a.live != nullptr && a.live[2] != 0;
  const CUtensorMap *from_a = (kMode == kStat || kMode == kDelta) && in_place ? &map_x : &map_a;
  const CUtensorMap *from_b = kMode == kWeightGrad && in_place ? &map_x : &map_b;
  const int tile_m = 128 * kCtas;
  const int tile_n = kMode == kStat ? a.tile_n : S::kSets * kTileN;
  const int rows_n = kMode == kStat ? tile_n / kCtas : S::kRowsN;  // rows of B that this CTA loads, of a set
  // an empty batch still passes one tile of zeros through the products that end in d and in grad W
  const int m_tiles = kMode == kWeightGrad ? a.m_tiles
                      : kMode == kDelta    ? max(1, (live + tile_m - 1) / tile_m)
                                           : (live + tile_m - 1) / tile_m;
  const int k_blocks = kMode == kWeightGrad ? max(1, (live + kStepK - 1) / kStepK) : a.k_blocks;
  Cut cut = {m_tiles * a.n_tiles, 0, 1};
  if (kMode == kDataGrad) cut = CutOf(m_tiles, a.n_tiles, a.k_plan, a.room, gridDim.x / kCtas, a.step_cycles, a.tile_cycles);
  const int units = cut.Units();
  const int first = blockIdx.x / kCtas, step = gridDim.x / kCtas;

  if (warp < 4) {
    if (warp == 0 && lane == 0) {
      uint32_t fill = 0;  // stages filled so far
      bool ok = true;
      for (int w = first; ok && w < units; w += step) {
        const Unit u = UnitOf(w, cut, m_tiles, a.n_tiles, a.group);
        const int k_begin = u.slice * k_blocks / u.parts, k_end = (u.slice + 1) * k_blocks / u.parts;
        const int m0 = u.m * tile_m + static_cast<int>(rank) * 128;
        const int n0 = u.n * tile_n + static_cast<int>(rank) * rows_n;
        for (int kb = k_begin; kb < k_end; ++kb, ++fill) {
          const int s = fill % S::kStages;
          const uint32_t use = fill / S::kStages;
          if (use > 0 && !tma::WaitBounded(&empty[s], (use - 1) & 1u)) {
            ok = false;
            break;
          }
          const uint32_t bar = kCtas == 2 ? tc5::MapToRank(tma::SharedAddr(&full[s]), 0) : tma::SharedAddr(&full[s]);
          if (rank == 0) tma::BarrierExpect(&full[s], (S::kBytesA + S::kSets * rows_n * kStepK * 2) * kCtas);
          const uint32_t sa = smem + s * S::kStage, sb = sa + S::kBytesA;
          const int k0 = kb * kStepK;
          if (L::kAAcross) {
#pragma unroll
            for (int j = 0; j < 2; ++j) tc5::LoadBox<kCtas>(sa + j * tc5::kBoxBytes, from_a, m0 + 64 * j, k0, bar);
          } else {
            tc5::LoadBox<kCtas>(sa, from_a, k0, m0, bar);
          }
          if (L::kBAcross) {
#pragma unroll
            for (int j = 0; j < S::kSets * S::kRowsN / 64; ++j) {
              const int set = j / (S::kRowsN / 64), x = n0 + set * kTileN + 64 * (j % (S::kRowsN / 64));
              tc5::LoadBox<kCtas>(sb + j * tc5::kBoxBytes, from_b, x, a.b_row0 + k0, bar);
            }
          } else {
#pragma unroll
            for (int set = 0; set < S::kSets; ++set) {
              tc5::LoadBox<kCtas>(sb + set * S::kBytesB, from_b, k0, a.b_row0 + n0 + set * kTileN, bar);
            }
          }
        }
      }
      if (!ok) atomicExch(a.status, tma::kStatusBulkCopyTimeout);
      // every stage handed back: the products have read all copies of this CTA, and no arrival is
      // still on its way to these barriers when the CTA leaves
      for (uint32_t i = fill > S::kStages ? fill - S::kStages : 0; i < fill; ++i) {
        if (!tma::WaitBounded(&empty[i % S::kStages], (i / S::kStages) & 1u)) atomicExch(a.status, tma::kStatusBulkCopyTimeout);
      }
    } else if (warp == 1 && lane == 0 && rank == 0) {
      uint32_t fill = 0, turn = 0;
      bool ok = true;
      for (int w = first; ok && w < units; w += step) {
        const Unit u = UnitOf(w, cut, m_tiles, a.n_tiles, a.group);
        const int k_first = u.slice * k_blocks / u.parts, k_count = (u.slice + 1) * k_blocks / u.parts - k_first;
        if (k_count == 0) continue;  // the last piece of the vocabulary may have fewer steps than there are parts
        const int runs = kRuns || kMode == kStat ? (k_count + a.run_steps - 1) / a.run_steps : 1;
        for (int run = 0; ok && run < runs; ++run, turn += S::kSets) {
          const int k_begin = k_first + RunBegin<kMode>(run, runs, k_count, a.run_steps);
          const int k_end = k_first + RunBegin<kMode>(run + 1, runs, k_count, a.run_steps);
          for (int kb = k_begin; ok && kb < k_end; ++kb, ++fill) {
            const int s = fill % S::kStages;
            const uint32_t sa = smem + s * S::kStage;
#pragma unroll
            for (int set = 0; set < S::kSets; ++set) {
              // the set's accumulators have been emptied (asked once per run), the stage has been filled
              const uint32_t half = (turn + set) & 1u, use = (turn + set) >> 1;
              if (ok && kb == k_begin && use > 0) ok = tma::WaitBounded(&acc_empty[half], (use - 1) & 1u);
              if (ok && set == 0) ok = tma::WaitBounded(&full[s], (fill / S::kStages) & 1u);
              if (!ok) break;
              tc5::FenceAfter();
              const uint32_t acc = tmem + half * kTileN, sb = sa + S::kBytesA + set * S::kBytesB;
              const uint64_t da = L::kAAcross ? tc5::DescAcrossK(sa) : tc5::DescAlongK(sa);
              const uint64_t db = L::kBAcross ? tc5::DescAcrossK(sb) : tc5::DescAlongK(sb);
              const uint32_t step_a = L::kAAcross ? 2048 >> 4 : 32 >> 4, step_b = L::kBAcross ? 2048 >> 4 : 32 >> 4;
#pragma unroll
              for (int j = 0; j < kStepK / 16; ++j) {
                tc5::Multiply<kCtas>(acc, da + j * step_a, db + j * step_b, a.instr, kb > k_begin || j > 0);
              }
              if (set == S::kSets - 1) tc5::CommitTo<kCtas>(&empty[s]);
              if (kb == k_end - 1) tc5::CommitTo<kCtas>(&acc_full[half]);
            }
          }
        }
      }
      if (!ok) atomicExch(a.status, tma::kStatusBulkCopyTimeout);
    }
  } else {
    Half t;
    t.group = (warp - 4) >> 2;
    t.thread = threadIdx.x - 128 - t.group * 128;
    t.box = 0u;
    t.boxes = smem + S::kOut + t.group * kBoxOut;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    uint32_t turn = 0;
    bool late = false;
    // accumulators ready / handed back.  A wait that gave up is not repeated: the warps of a group go on together, so that
    // their barriers stay matched, with results that the status word declares void.
    auto ready = [&]() {
      if (!late && !__all_sync(0xffffffffu, tma::WaitBounded(&acc_full[turn & 1u], (turn >> 1) & 1u))) late = true;
      tc5::FenceAfter();
      t.acc = tmem + (turn & 1u) * kTileN + t.group * kHalfN + lanes;
    };
    auto release = [&]() {
      tc5::FenceBefore();
      __syncwarp();
      if (lane == 0) {
        if (kCtas == 2) tc5::ArriveCluster(tc5::MapToRank(tma::SharedAddr(&acc_empty[turn & 1u]), 0));
        else tma::BarrierArrive(&acc_empty[turn & 1u]);
      }
      ++turn;
    };
    for (int w = first; w < units; w += step) {
      const Unit u = UnitOf(w, cut, m_tiles, a.n_tiles, a.group);
      const int k_count = (u.slice + 1) * k_blocks / u.parts - u.slice * k_blocks / u.parts;
      if (kMode == kDataGrad && k_count == 0) continue;
      const int runs = kRuns || kMode == kStat ? (k_count + a.run_steps - 1) / a.run_steps : 1;
      const int row0 = u.m * tile_m + static_cast<int>(rank) * 128;
      t.row = row0 + t.thread;
      t.col = u.n * tile_n + t.group * kHalfN;
      const int label = (kMode == kStat || kMode == kDelta) && t.row < live ? a.label[t.row] : -1;
      if (kMode == kStat) {
        uint64_t v[kHalfN / 2];
#pragma unroll
        for (int i = 0; i < kHalfN / 2; ++i) v[i] = 0;
        for (int run = 0; run < runs; ++run) {
          ready();
#pragma unroll
          for (int c = 0; c < kHalfN / 16; ++c) {
            uint32_t r[16];
            tc5::LoadColumns(t.acc + c * 16, r);
            tc5::WaitColumns(r);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              v[c * 8 + i] = tc5::AddPair(v[c * 8 + i], tc5::Pair(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])));
            }
          }
          release();
        }
        if (row0 + (warp & 3) * 32 >= live) continue;  // no row of this warp's exists
        const int limit = min(a.cols - t.col, tile_n - t.group * kHalfN);  // columns of this half that exist
        const int64_t at = (static_cast<int64_t>(a.tile0 + u.n) * 2 + t.group) * a.pad_rows + t.row;
        StatHalf(v, t, limit, label < 0 ? -1 : label - a.col0 - t.col, at, a);
        continue;
      }
      for (int i = 0; i < runs * S::kSets; ++i) {
        const int run = i / S::kSets, set = i - run * S::kSets;
        t.col = u.n * tile_n + t.group * kHalfN + set * kTileN;
        if (kRuns) t.earlier = run > 0 ? EarlierOf(a.earlier, set) : nullptr;
        ready();
        if (kRuns && run < runs - 1) {
          KeepHalf(t, EarlierOf(a.earlier, set));
        } else if (kMode == kDelta) {
          // rows past the live ones: no column of theirs exists, so that d' is zero there whatever the logits of a zero data
          // row are (NaN beside a class with an infinite weight); the product for grad W reads them up to a whole step
          DeltaHalf<S::kBoxes, kRuns>(t, t.row < live ? a.cols - t.col : 0, label < 0 ? -1 : label - a.col0 - t.col,
                                      a.lse2[t.row], a.row_scale[t.row], &map_out, row0, a);
        } else if (kMode == kDataGrad) {
          // a whole tile goes to its place in the gradient, a part of one to a tile of its own beside it
          const bool whole = u.parts == 1;
          const CUtensorMap *to = whole ? &map_out : &map_x;
          const int x = whole ? t.col : t.group * kHalfN + set * kTileN;
          const int y = whole ? row0 : u.spare * tile_m + static_cast<int>(rank) * 128;
          if (a.accumulate) FloatHalf<S::kBoxes, kRuns, true>(t, 1.0f, to, x, y);
          else FloatHalf<S::kBoxes, kRuns, false>(t, 1.0f, to, x, y);
        } else {
          const float inv = a.inv_scale[0];
          if (a.out_tiled) {
            if (a.out_type == kFloat32 && a.out_add) FloatHalf<S::kBoxes, kRuns, true>(t, inv, &map_out, t.col, row0);
            else if (a.out_type == kFloat32) FloatHalf<S::kBoxes, kRuns, false>(t, inv, &map_out, t.col, row0);
            else PackedHalf<S::kBoxes, kRuns>(t, inv, a.out_type == kBfloat16, &map_out, row0);
          } else {
#pragma unroll 1
            for (int c = 0; c < kHalfN / 32; ++c) {
              uint32_t r[32];
              tc5::LoadColumns(t.acc + c * 32, r);
              tc5::WaitColumns(r);
              AddEarlier<kRuns>(t, c * 32, r);
              if (!a.out_vec) WeightRows(r, t, row0, t.col + c * 32, inv, a);
              else if (t.row < a.out_rows) WeightColumns(r, t.row, t.col + c * 32, inv, a);
            }
          }
        }
        release();
      }
    }
    if (late && lane == 0) atomicExch(a.status, tma::kStatusBulkCopyTimeout);
    if (kMode != kStat && t.thread == 0) tc5::WaitStores();
  }
  __syncwarp();
  tc5::FenceBefore();
  __syncthreads();
  if (kCtas == 2) tc5::ClusterSync();
  tc5::FenceAfter();
  if (warp == 2) tc5::FreeTensorMemory<kCtas>(tmem);
}

// ---- the kernels around the products ------------------------------------------------------------

struct PackArgs {
  const uint16_t *x;
  int64_t ld_x;
  const int32_t *label;
  int32_t ignore;
  int32_t n, v, h;
  int64_t pad_rows;      // n rounded up to kPadRows
  uint16_t *packed;      // [pad_rows][ld_packed]
  int64_t ld_packed;
  int32_t *words;        // [0] = live rows, [1] = what takes d' to d (a float), [2] = rows of x left where they are
  int32_t *row_of;       // [pad_rows] token of packed row (forward)
  int32_t *pos_of;       // [n] packed row of token, or -1 (backward)
  int32_t *label_of;     // [pad_rows] label of packed row
  float *loss, *lse_out; // forward: rows that do not count become 0
  const float *lse;      // backward
  const float *gloss;    // backward, may be null
  float scale, q_label;
  float *lse2, *row_scale;  // [pad_rows], backward
  float *row_down;       // [pad_rows] 2^-(a row's own k - the common one), or null: all rows have the common one
  int vec;               // 16-byte copies possible
  int tiled;             // the tiled copies can read x itself: nothing is packed if all its rows count
  int rows_per_cta;
  float2 *counts;        // [pad_rows / 256] (count as bits, largest |gloss|), or null: the labels are counted directly
};

__device__ __forceinline__ bool IsLive(int32_t label, int32_t ignore, int32_t v) {
  return label != ignore && label >= 0 && label < v;
}

/*! \brief |gloss| where it is a number that a scale can be chosen by: an infinite one must not leave the other rows without */
__device__ __forceinline__ float FiniteSize(float gloss) {
  const float size = fabsf(gloss);
  return size < INFINITY ? size : 0.0f;
}
/*! \brief the power of two that brings `size` to [2^14, 2^15); 0 for one that has none */
__device__ __forceinline__ int ScaleExponent(float size) {
  return size > 0.0f && size < INFINITY ? 14 - ilogbf(size) : 0;  // -113 .. 163
}

/*! \brief live rows, and the largest finite |gloss| among them, of every 256 tokens: for lists too long to be counted by each CTA below */
template <int kUnused>
__global__ void __launch_bounds__(256) CountRowsKernel(const PackArgs a) {
  gpu_rt::GridDependencySync();
  __shared__ int s_count[8];
  __shared__ float s_top[8];
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const bool on = i < a.n && IsLive(a.label[i], a.ignore, a.v);
  float top = on && a.gloss != nullptr ? FiniteSize(a.gloss[i]) : 0.0f;
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const int count = __popc(__ballot_sync(0xffffffffu, on));
  if ((threadIdx.x & 31) == 0) s_count[threadIdx.x >> 5] = count, s_top[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  int total = 0;
  top = 0.0f;
  for (int w = 0; w < 8; ++w) total += s_count[w], top = fmaxf(top, s_top[w]);
  a.counts[blockIdx.x] = make_float2(__int_as_float(total), top);
}

/*!
 * \brief packs the live rows of x and what belongs to them, in token order.  A CTA takes
 *  rows_per_cta tokens (at most 256); where its first live row goes it finds by counting the labels before it
 *  itself (4 bytes per token from the L2), which spares a scan kernel and its launch.  The rows
 *  from the last live one up to the next multiple of kPadRows become zeros.  Where all rows are live and the
 *  products can read x as it is, nothing is copied.
 */
template <int kUnused>
__global__ void __launch_bounds__(256) PackRowsKernel(const PackArgs a) {
  gpu_rt::GridDependencySync();
  __shared__ int s_before[8], s_total[8];
  __shared__ float s_top[8];
  __shared__ int s_src[256];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int base = blockIdx.x * a.rows_per_cta;
  int before = 0, total = 0;
  float top = 0.0f;
  if (a.counts != nullptr) {  // (then rows_per_cta is 256)
    for (int64_t b = tid; b < a.pad_rows / 256; b += 256) {
      const float2 c = a.counts[b];
      total += __float_as_int(c.x);
      before += b < blockIdx.x ? __float_as_int(c.x) : 0;
      top = fmaxf(top, c.y);
    }
  } else {
    for (int i = tid; i < a.n; i += 256) {
      const int on = IsLive(a.label[i], a.ignore, a.v) ? 1 : 0;
      total += on;
      before += i < base ? on : 0;
      if (a.gloss != nullptr && on) top = fmaxf(top, FiniteSize(a.gloss[i]));
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (lane == 0) s_before[warp] = before, s_total[warp] = total, s_top[warp] = top;
  __syncthreads();
  before = total = 0;
  top = 0.0f;
  for (int w = 0; w < 8; ++w) before += s_before[w], total += s_total[w], top = fmaxf(top, s_top[w]);
  __syncthreads();

  const int common = a.row_scale != nullptr ? ScaleExponent((a.gloss != nullptr ? top : 1.0f) / a.q_label) : 0;
  const int end = (total + kPadRows - 1) / kPadRows * kPadRows;  // rows up to here are read by the products
  const int i = base + tid;
  const bool mine = tid < a.rows_per_cta && i < a.n;
  const int32_t label = mine ? a.label[i] : -1;
  const bool on = mine && IsLive(label, a.ignore, a.v);
  const unsigned votes = __ballot_sync(0xffffffffu, on);
  if (lane == 0) s_before[warp] = __popc(votes);
  __syncthreads();
  int pos = before + __popc(votes & ((1u << lane) - 1u));
  for (int w = 0; w < warp; ++w) pos += s_before[w];
  s_src[tid] = on ? pos : -1;
  if (on) {
    a.label_of[pos] = label;
    if (a.row_of != nullptr) a.row_of[pos] = i;
    if (a.row_scale != nullptr) {
      const float factor = (a.gloss != nullptr ? a.gloss[i] : 1.0f) / a.q_label;
      int own = common;
      if (a.row_down != nullptr) {
        const int best = FiniteSize(factor) > 0.0f ? ScaleExponent(fabsf(factor)) : common;
        if (best - common > 6) own = min(best, common + 100);
        a.row_down[pos] = __int_as_float((127 + common - own) << 23);
      }
      a.row_scale[pos] = ldexpf(factor, own);
      a.lse2[pos] = a.lse[i] * kLog2e;
    }
  }
  if (mine && a.pos_of != nullptr) a.pos_of[i] = on ? pos : -1;
  if (mine && !on && a.loss != nullptr) a.loss[i] = 0.0f, a.lse_out[i] = 0.0f;
  if (tid < a.rows_per_cta && i >= total && i < max(end, kPadRows)) {
    a.label_of[i] = -1;
    if (a.row_scale != nullptr) a.row_scale[i] = 0.0f, a.lse2[i] = 0.0f;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.words[0] = total;
    // (with no token that counts the sums are empty, and zero whatever the scale: 1 / 0 tokens, say)
    reinterpret_cast<float *>(a.words)[1] = total > 0 ? ldexpf(a.scale * a.q_label, -common) : 0.0f;
    a.words[2] = a.tiled && total == a.n;
  }
  if (a.tiled && total == a.n) return;
  __syncthreads();
  for (int t = warp; t < a.rows_per_cta; t += 8) {
    const int from = base + t;
    if (from < a.n && s_src[t] >= 0) {
      const uint16_t *src = a.x + from * a.ld_x;
      uint16_t *dst = a.packed + s_src[t] * a.ld_packed;
      if (a.vec) {
        for (int c = lane; c < a.h / 8; c += 32) reinterpret_cast<uint4 *>(dst)[c] = __ldcs(reinterpret_cast<const uint4 *>(src) + c);
        for (int c = a.h / 8 * 8 + lane; c < a.h; c += 32) dst[c] = src[c];
      } else {
        for (int c = lane; c < a.h; c += 32) dst[c] = src[c];
      }
    }
    if (from >= total && from < max(end, kPadRows)) {
      uint4 *dst = reinterpret_cast<uint4 *>(a.packed + from * a.ld_packed);
      for (int c = lane; c < a.ld_packed / 8; c += 32) dst[c] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

/*!
 * \brief copies rows of 16-bit elements to rows that start on 16-byte boundaries: a thread assembles eight elements (the
 *  groups of all rows dealt out to threads; a CTA per row and an element per thread took three times as long)
 */
template <int kUnused>
__global__ void __launch_bounds__(256)
AlignRowsKernel(uint16_t *dst, int64_t ld_dst, const uint16_t *src, int64_t ld_src, int64_t total, gpu_rt::FastDiv groups,
                int cols) {
  gpu_rt::GridDependencySync();
  for (int64_t e = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; e < total; e += static_cast<int64_t>(gridDim.x) * 256) {
    uint32_t row;
    const int col = static_cast<int>(groups.DivMod(static_cast<uint32_t>(e), &row)) * 8;
    const uint16_t *from = src + row * ld_src + col;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = col + j < cols ? from[j] : 0u;
    *reinterpret_cast<uint4 *>(dst + row * ld_dst + col) =
        make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
  }
}

/*! \brief rows of d' with a k of their own back to the common one, between the gradients of x and W: a warp per row */
template <int kUnused>
__global__ void __launch_bounds__(256)
CommonScaleKernel(uint16_t *delta, int64_t ld, const int32_t *live, const float *row_down, int cols) {
  gpu_rt::GridDependencySync();
  const int lane = threadIdx.x & 31;
  for (int row = blockIdx.x * 8 + (threadIdx.x >> 5); row < live[0]; row += gridDim.x * 8) {
    const float down = row_down[row];
    if (down == 1.0f) continue;
    uint4 *p = reinterpret_cast<uint4 *>(delta + row * ld);
    for (int c = lane; c < (cols + 7) / 8; c += 32) {
      uint4 v = p[c];
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = PackPair(Widen(static_cast<uint16_t>(w[j] & 0xffffu), 0) * down, Widen(static_cast<uint16_t>(w[j] >> 16), 0) * down, 0);
      }
      v.x = w[0], v.y = w[1], v.z = w[2], v.w = w[3];
      p[c] = v;
    }
  }
}

struct JoinArgs {
  const int32_t *live;
  int32_t tokens, parts, v;
  int64_t pad_rows;
  const float2 *part;
  const float *part_sum, *label_logit;
  const int32_t *label, *row_of;  // row_of null: packed row = token
  int32_t ignore;
  float smooth;
  float *loss, *lse;
};

/*!
 * \brief joins the maxima and sums of the tile halves row by row.  512 threads share kRows rows: a thread takes every
 *  (512 / kRows)-th part of its row, eight at a time with their loads in flight together, and the threads of a row are
 *  joined pairwise.  Bound by the latency of a few round trips: few rows per CTA (4) while there are few tokens (834
 *  parts of 48 rows: 15 us with 32 rows per CTA), 32 rows (256-byte loads) when there are many.
 */
template <int kRows>
__global__ void __launch_bounds__(512) JoinTilesKernel(const JoinArgs a) {
  gpu_rt::GridDependencySync();
  constexpr int kShare = 512 / kRows;
  __shared__ float s_ref[kShare / 2][kRows], s_sum[kShare / 2][kRows], s_total[kShare / 2][kRows];
  const int live = a.live != nullptr ? *a.live : a.tokens;
  const int r = threadIdx.x % kRows, q = threadIdx.x / kRows;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + r;
  if (static_cast<int64_t>(blockIdx.x) * kRows >= live) return;
  float ref = -INFINITY, sum = 0.0f, total = 0.0f;
  const int32_t label = q == 0 && row < live ? a.label[row] : -1;
  const double z = q == 0 && row < live ? a.label_logit[row] : 0.0f;  // of no meaning for a row that does not count
  if (row < live) {
    for (int t0 = q; t0 < a.parts; t0 += kShare * 8) {
      float2 p[8];
      float top = ref;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int t = t0 + kShare * u;
        p[u] = t < a.parts ? a.part[t * a.pad_rows + row] : make_float2(-INFINITY, 0.0f);
        if (a.part_sum != nullptr && t < a.parts) total += a.part_sum[t * a.pad_rows + row];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) top = fmaxf(top, p[u].x);
      const float from = top == -INFINITY ? 0.0f : top;
      sum *= Exp2((ref - from) * kLog2e);
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += p[u].y * Exp2((p[u].x - from) * kLog2e);
      ref = top;
    }
  }
#pragma unroll
  for (int half = kShare / 2; half > 0; half >>= 1) {
    if (q >= half && q < 2 * half) s_ref[q - half][r] = ref, s_sum[q - half][r] = sum, s_total[q - half][r] = total;
    __syncthreads();
    if (q < half) {
      const float other = s_ref[q][r], top = fmaxf(ref, other), from = top == -INFINITY ? 0.0f : top;
      sum = sum * Exp2((ref - from) * kLog2e) + s_sum[q][r] * Exp2((other - from) * kLog2e);
      ref = top;
      total += s_total[q][r];
    }
    __syncthreads();
  }
  if (q != 0 || row >= live) return;
  const int64_t to = a.row_of != nullptr ? a.row_of[row] : row;
  if (!IsLive(label, a.ignore, a.v)) {
    a.loss[to] = 0.0f, a.lse[to] = 0.0f;
    return;
  }
  // a handful of operations per row, in 64 bits: the maximum is tens of units large, the loss may be small
  const double log_sum = log(static_cast<double>(sum));
  double loss = (ref - z) + log_sum;
  if (a.part_sum != nullptr) {
    const double smooth = a.smooth;
    loss += smooth * z - smooth / (a.v - 1) * (total - z);
  }
  a.loss[to] = static_cast<float>(loss);
  a.lse[to] = static_cast<float>(ref + log_sum);
}

struct FinishArgs {
  const float *acc, *spare;
  int64_t ld_acc;
  const int32_t *live;
  int n_tiles, tile_n, group, k_plan, room, slots, ctas;  // of the kernel that wrote the parts
  float step_cycles, tile_cycles;
  const int32_t *pos_of;
  const float *inv_scale, *row_down;
  uint16_t *out;
  int64_t ld_out;
  int32_t n, h;
  int bf16, vec;
  gpu_rt::FastDiv groups;  // (h + 7) / 8
};

/*!
 * \brief gradient of x: parts of the contraction added in order, rounded once, rows back in token order.  A thread keeps
 *  its eight columns and takes four rows at a time, so that what it computes about tiles is little and
 *  eight 16-byte loads are in flight (a CTA for each row: 54 us for 8192 x 2560; so: 42 us, 3.8 TB/s).
 *  kOwnScales: rows of d' had scales of their own.
 */
template <bool kOwnScales>
__global__ void __launch_bounds__(256) DataGradFinishKernel(const FinishArgs a) {
  gpu_rt::GridDependencySync();
  constexpr int kRows = 4;
  const float inv = a.inv_scale[0];
  const int groups = (a.h + 7) / 8;
  const int tile_m = 128 * a.ctas, m_tiles = (a.live[0] + tile_m - 1) / tile_m;
  const Cut cut = CutOf(m_tiles, a.n_tiles, a.k_plan, a.room, a.slots, a.step_cycles, a.tile_cycles);
  const int64_t part_stride = static_cast<int64_t>(tile_m) * a.tile_n;
  // (row blocks) x (groups of eight columns), dealt out to threads
  const uint32_t total = static_cast<uint32_t>((a.n + kRows - 1) / kRows) * static_cast<uint32_t>(groups);
  for (uint32_t e = blockIdx.x * 256 + threadIdx.x; e < total; e += gridDim.x * 256) {
    uint32_t block;
    const int g = static_cast<int>(a.groups.DivMod(e, &block));
    const int n = 8 * g / a.tile_n, col = 8 * g - n * a.tile_n;
    const int64_t i0 = static_cast<int64_t>(block) * kRows;
    int pos[kRows], parts[kRows], most = 1;
    const float *from[kRows];
    float v[kRows][8];
#pragma unroll
    for (int r = 0; r < kRows; ++r) pos[r] = i0 + r < a.n ? a.pos_of[i0 + r] : -1;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      parts[r] = pos[r] >= 0 ? 1 : 0;
      from[r] = a.acc + pos[r] * a.ld_acc + 8 * g;
      if (pos[r] >= 0 && cut.parts > 1) {
        const int m = pos[r] / tile_m;
        const int place = PlaceOf(m, n, m_tiles, a.n_tiles, a.group) - cut.full;
        if (place >= 0) {
          parts[r] = most = cut.parts;
          from[r] = a.spare + place * cut.parts * part_stride + static_cast<int64_t>(pos[r] - m * tile_m) * a.tile_n + col;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[r][j] = 0.0f;
    }
#pragma unroll 4  // (two at a time, as the compiler would have it: 16 tokens 19.5 -> 22 us)
    for (int s = 0; s < most; ++s) {
      float4 lo[kRows], hi[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        lo[r] = hi[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (s < parts[r]) {
          const float4 *p = reinterpret_cast<const float4 *>(from[r] + s * part_stride);
          lo[r] = __ldcs(p), hi[r] = __ldcs(p + 1);
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        v[r][0] += lo[r].x, v[r][1] += lo[r].y, v[r][2] += lo[r].z, v[r][3] += lo[r].w;
        v[r][4] += hi[r].x, v[r][5] += hi[r].y, v[r][6] += hi[r].z, v[r][7] += hi[r].w;
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (i0 + r >= a.n) break;
      uint16_t *out = a.out + (i0 + r) * a.ld_out;
      const float factor = parts[r] > 0 ? inv : 0.0f;  // (inv may be infinite, and the zeros of a row that does not count are zeros)
      const float down = kOwnScales && parts[r] > 0 ? a.row_down[pos[r]] : 1.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[r][j] = kOwnScales ? v[r][j] * down * factor : v[r][j] * factor;
      if (a.vec && 8 * g + 8 <= a.h) {
        uint4 w;
        w.x = PackPair(v[r][0], v[r][1], a.bf16);
        w.y = PackPair(v[r][2], v[r][3], a.bf16);
        w.z = PackPair(v[r][4], v[r][5], a.bf16);
        w.w = PackPair(v[r][6], v[r][7], a.bf16);
        reinterpret_cast<uint4 *>(out)[g] = w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (8 * g + j < a.h) out[8 * g + j] = static_cast<uint16_t>(PackPair(v[r][j], 0.0f, a.bf16) & 0xffffu);
        }
      }
    }
  }
}

// ---- host side ------------------------------------------------------------------------------------

const int64_t kDeltaBytes = int64_t(512) << 20;  // piece of d: larger pieces mean fewer passes over the gradient of x
const int64_t kCountDirectly = 16384;            // tokens up to which each CTA of PackRowsKernel counts all labels itself
const int64_t kCopyBytes = int64_t(128) << 20;   // piece of W copied to aligned rows where the caller's are not

inline int64_t RoundUp(int64_t a, int64_t b) { return (a + b - 1) / b * b; }
inline int64_t Ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Problem {
  const uint16_t *x, *w;
  const int32_t *label;
  int64_t n, v, h, ld_x, ld_w;
  bool bf16;
  int32_t ignore;
  float smooth;
  int type() const { return bf16 ? kBfloat16 : kFloat16; }
};

inline bool Aligned16(const void *p, int64_t ld, int64_t elem) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * elem % 16 == 0;
}

/*!
 * \brief one CTA or a pair per tile.  A pair reads each operand half as often and runs a long grid of tiles
 *  about 6 % faster (8192 x 131072 x 4096: 6.06 against 6.50 ms), but its tiles are twice as high: where that
 *  costs more rounds of tiles over the SMs than it saves (257 rows: two pairs high for three CTAs'
 *  worth of rows), single CTAs are used.
 */
inline int CtasFor(int64_t rows, int64_t other_tiles, int sms) {
  const int64_t single = Ceil(Ceil(rows, 128) * other_tiles, sms), pair = Ceil(Ceil(rows, 256) * other_tiles, sms / 2);
  return single * 107 < pair * 100 ? 1 : 2;
}

/*!
 * \brief tiles of 512 columns (kWide) for a product with `tiles` tiles of 256, `across` of them side by side, and a
 *  contraction of `steps`: steps enough that emptying a tile while nothing multiplies costs less than the quarter
 *  of the copies that is saved (grad W: 14 % less time at 128 steps, 13 % at 64, 7 % at 32; d: 7 % at 64, 5 % at 32, 4 %
 *  more at 16), and tiles enough that whole rounds over the SMs lose little
 */
inline bool WideFor(int64_t tiles, int64_t across, int64_t steps, int sms) {
  return across % 2 == 0 && tiles / 2 >= sms && steps >= kWideSteps;
}
/*!
 * \brief cycles that CutOf counts for a step of a tile: as measured with all SMs busy (the operand copies, not the
 *  products, set them).  Tiles of grad x: 0 = one CTA, 128 x 256; 1 = a pair, 256 x 256; 2 = a pair, 256 x 512
 */
inline double StepCycles(int shape) { return shape == 0 ? 850.0 : shape == 1 ? 810.0 : 1250.0; }
/*! \brief cycles to write a part of a tile and read it again, at about 2400 bytes a cycle */
inline double TileCycles(int shape) { return (shape == 0 ? 128.0 : 256.0) * (shape == 2 ? 512.0 : 256.0) * 8.0 / 2400.0; }
/*!
 * \brief the tile shape of grad x for n tokens, h_tiles blocks of 256 features and a contraction of `steps` (the vocabulary
 *  piece): the one whose best cut (CutOf) costs least when all tokens count.  Wide tiles where there are enough
 *  rows (8192 x 4096: 10 % less time than 256 x 256, 2048 x 4096: 14 %, 4096 x 1024: 12 %), single CTAs for 257 rows
 */
inline int DataShape(int64_t n, int64_t h_tiles, int64_t steps, int sms) {
  int best = 0;
  double least = 0.0;
  for (int shape = 0; shape < 3; ++shape) {
    if (shape == 2 && (h_tiles % 2 != 0 || steps < 4 * kWideSteps)) continue;
    const int64_t slots = shape == 0 ? sms : sms / 2;
    const int64_t tiles = Ceil(n, shape == 0 ? 128 : 256) * (shape == 2 ? h_tiles / 2 : h_tiles);
    const int64_t full = tiles / slots, rest = tiles % slots;
    double cut = 0.0;
    for (int64_t parts = 1; parts <= 16 && rest > 0 && (parts == 1 || (parts * 8 <= steps && parts * rest <= 4 * slots)); ++parts) {
      const double cost = Ceil(rest * parts, slots) * (Ceil(steps, parts) * StepCycles(shape) + 4000.0) + parts * rest * TileCycles(shape);
      if (parts == 1 || cost < cut) cut = cost;
    }
    const double cost = full * (steps * StepCycles(shape) + 4000.0) + cut;
    if (shape == 0 || cost < least) least = cost, best = shape;
  }
  return best;
}

/*! \brief how a call is cut, and where its scratch matrices lie (offsets in bytes) */
struct Plan {
  bool pack, copy_w;
  int64_t pad_rows, ld_x, ld_w, piece, ld_acc, tile_n, tiles;
  int room, ctas, ctas_gx, shape_gx;
  bool wide_gx, runs;
  int64_t counts, words, row_of, pos_of, label_of, lse2, row_scale, row_down, x, w, part, part_sum, label_logit, delta, acc, spare, earlier, bytes;
};

/*! \brief layout of a call; sms = multiprocessors of the device */
inline Plan MakePlan(int64_t n, int64_t v, int64_t h, bool gradient, bool want_gx, bool smooth, bool pack, bool copy_w,
                     int sms) {
  Plan p = {};
  p.pack = pack;
  p.copy_w = copy_w;
  p.pad_rows = RoundUp(n, kPadRows);
  p.ld_x = RoundUp(h, 8);
  p.ld_w = RoundUp(h, 8);
  p.ld_acc = RoundUp(h, kTileN);
  p.tile_n = kTileN;
  p.piece = RoundUp(v, kTileN);
  if (gradient) p.piece = std::min(p.piece, std::max<int64_t>(kTileN, kDeltaBytes / (2 * p.pad_rows) / kTileN * kTileN));
  if (copy_w) p.piece = std::min(p.piece, std::max<int64_t>(kTileN, kCopyBytes / (2 * p.ld_w) / kTileN * kTileN));
  p.ctas = CtasFor(n, p.piece / kTileN, sms);
  if (!gradient && n <= 128 && p.piece >= v) {
    // a call bound by reading W once: as many columns per tile as make whole rounds over the SMs (32000 classes: 143
    // tiles of 224 columns instead of 125 of 256)
    p.ctas = 1;
    const int64_t rounds = Ceil(Ceil(v, kTileN), sms);
    p.tile_n = std::min<int64_t>(kTileN, RoundUp(Ceil(v, rounds * sms), 16));
  }
  p.tiles = Ceil(v, p.tile_n);
  const int64_t h_tiles = p.ld_acc / kTileN;
  p.shape_gx = DataShape(n, h_tiles, Ceil(std::min(p.piece, v), kStepK), sms);
  p.ctas_gx = p.shape_gx == 0 ? 1 : 2;
  p.wide_gx = p.shape_gx == 2;
  p.room = 4 * (sms / p.ctas_gx);  // parts of tiles: four rounds over the GPU
  int64_t at = 0;
  auto take = [&at](int64_t bytes) {
    const int64_t was = at;
    at += RoundUp(bytes, 256);
    return was;
  };
  p.words = take(256);
  p.counts = take(pack && p.pad_rows > kCountDirectly ? p.pad_rows / 256 * 8 : 0);
  p.label_of = take(pack ? p.pad_rows * 4 : 0);
  p.row_of = take(pack && !gradient ? p.pad_rows * 4 : 0);
  p.pos_of = take(gradient ? p.pad_rows * 4 : 0);
  p.x = take(pack ? p.pad_rows * p.ld_x * 2 : 0);
  p.w = take(copy_w ? p.piece * p.ld_w * 2 : 0);
  if (gradient) {
    p.lse2 = take(p.pad_rows * 4);
    p.row_scale = take(p.pad_rows * 4);
    p.row_down = take(want_gx ? p.pad_rows * 4 : 0);
    p.delta = take(p.pad_rows * p.piece * 2);
    p.acc = take(want_gx ? p.pad_rows * p.ld_acc * 4 : 0);
    // (whether a contraction is longer than a run)
    p.runs = Ceil(h, kStepK) > RunSteps(kDelta, false) || Ceil(n, kStepK) > RunSteps(kWeightGrad, true) ||
             Ceil(std::min(p.piece, v), kStepK) > RunSteps(kDataGrad, false);
    p.earlier = take(p.runs ? sms * kEarlierBytes : 0);
    p.spare = take(want_gx ? static_cast<int64_t>(p.room) * 128 * p.ctas_gx * kTileN * (p.wide_gx ? 2 : 1) * 4 : 0);
  } else {
    p.part = take(2 * p.tiles * p.pad_rows * 8);
    p.part_sum = take(smooth ? 2 * p.tiles * p.pad_rows * 4 : 0);
    p.label_logit = take(p.pad_rows * 4);
  }
  p.bytes = at;
  return p;
}

/*! \brief the kernels count tiles in 32 bits */
inline void CheckExtents(const Problem &q) {
  CHECK(q.n <= (int64_t(1) << 30) && q.h < (int64_t(1) << 22) && Ceil(q.n, 4) * Ceil(q.h, 8) < (int64_t(1) << 30) &&
        Ceil(q.n, 128) * Ceil(q.v, 16) < (int64_t(1) << 31) && Ceil(q.v, 128) * Ceil(q.h, 256) < (int64_t(1) << 31))
      << "LinearSoftmaxLoss: more tokens, classes or features than one call covers";
}
inline Plan PlanForward(const Problem &q, int sms) {
  CheckExtents(q);
  // packing costs a launch (some 4 us), and saves whole tiles of rows that do not count: 512 rows are two pairs' worth
  const bool pack = q.n > 512 || !Aligned16(q.x, q.ld_x, 2);
  return MakePlan(q.n, q.v, q.h, false, false, q.smooth != 0.0f, pack, !Aligned16(q.w, q.ld_w, 2), sms);
}
inline Plan PlanBackward(const Problem &q, bool want_gx, int sms) {
  CheckExtents(q);
  return MakePlan(q.n, q.v, q.h, true, want_gx, q.smooth != 0.0f, true, !Aligned16(q.w, q.ld_w, 2), sms);
}
/*! \brief scratch that suffices for every call of these sizes, whatever its layouts and options */
inline size_t WorkspaceNeed(int64_t n, int64_t v, int64_t h, bool gradient, int sms) {
  int64_t most = 0;
  for (int copy_w = 0; copy_w < 2; ++copy_w) {
    most = std::max(most, MakePlan(n, v, h, gradient, true, true, true, copy_w != 0, sms).bytes);
  }
  return static_cast<size_t>(most);
}

template <int kMode, int kCtas, bool kWide, bool kRuns>
inline void LaunchRuns(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mx, const CUtensorMap &mo, const GemmArgs &args, int64_t units,
                       int sms, cudaStream_t stream) {
  auto kernel = VocabGemmKernel<kMode, kCtas, kWide, kRuns>;
  const size_t smem = StageShape<kMode, kCtas, kWide>::kSmem;
  gpu_rt::AllowSharedMemory(kernel, smem);
  cudaLaunchConfig_t cfg = {};
  // (the parts of kDataGrad are counted by the kernel: it gets every slot)
  const int64_t slots = kMode == kDataGrad ? sms / kCtas : std::min<int64_t>(std::max<int64_t>(units, 1), sms / kCtas);
  cfg.gridDim = dim3(static_cast<unsigned>(slots) * kCtas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = MSHADOW_B200_EARLY_LAUNCH ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCtas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kCtas > 1 ? 2 : 1;
  MSHADOW_CUDA_CALL(cudaLaunchKernelEx(&cfg, kernel, ma, mb, mx, mo, args));
  MSHADOW_CUDA_POST_KERNEL_CHECK(VocabGemmKernel);
}

/*! \brief `steps`: of the longest contraction, which may be shorter on the device where not all tokens count */
template <int kMode, int kCtas, bool kWide>
inline void LaunchGemm(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mx, const CUtensorMap &mo, const GemmArgs &args,
                       int64_t steps, int64_t units, int sms, cudaStream_t stream) {
  if (kMode != kStat && steps > args.run_steps) {
    LaunchRuns<kMode, kCtas, kWide, kMode != kStat>(ma, mb, mx, mo, args, units, sms, stream);
  } else {
    LaunchRuns<kMode, kCtas, kWide, false>(ma, mb, mx, mo, args, units, sms, stream);
  }
}

template <int kMode>
inline void Gemm(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mx, const CUtensorMap &mo, const GemmArgs &args,
                 int64_t steps, int64_t units, int ctas, int sms, cudaStream_t stream) {
  if (ctas == 2) LaunchGemm<kMode, 2, false>(ma, mb, mx, mo, args, steps, units, sms, stream);
  else LaunchGemm<kMode, 1, false>(ma, mb, mx, mo, args, steps, units, sms, stream);
}

/*!
 * \brief row tiles walked before the next column tile, so that what the tiles in flight read again stays in the L2.
 *  8192 x 131072 x 4096: the two products over h take 6 % less time in bands of 16 row tiles than of 4 or 32, the
 *  two gradients 2 % less in bands of 8 than of 16.
 */
inline int GroupOf(int64_t m_tiles, int64_t most) {
  return static_cast<int>(std::min<int64_t>(std::max<int64_t>(m_tiles, 1), most));
}

// The functions below that launch kernels are templates so that a program that includes the headers and calls no vocabulary
// operator holds none of their kernels, and needs no architecture that has tcgen05.

/*! \brief the weight rows [p0, p0 + rows) as the products read them: map over W itself, or over an aligned copy */
template <int kUnused>
inline CUtensorMap WeightMap(const Problem &q, const Plan &p, char *ws, int64_t p0, int64_t rows, int box_rows,
                             cudaStream_t stream, bool copy_now, int32_t *row0) {
  if (!p.copy_w) {
    *row0 = static_cast<int32_t>(p0);
    return tc5::MatrixMap(q.w, q.type(), q.v, q.h, q.ld_w, box_rows);
  }
  uint16_t *w = reinterpret_cast<uint16_t *>(ws + p.w);
  if (copy_now) {
    const int64_t groups = Ceil(q.h, 8), total = rows * groups;  // below 2^31: a piece holds at most 2^30 elements
    gpu_rt::LaunchAfterDrain(AlignRowsKernel<kUnused>, dim3(static_cast<unsigned>(std::min<int64_t>(Ceil(total, 256), 4096))), dim3(256),
                             0, stream, w, p.ld_w, q.w + p0 * q.ld_w, q.ld_w, total, gpu_rt::FastDiv(static_cast<uint32_t>(groups)),
                             static_cast<int>(q.h));
    MSHADOW_CUDA_POST_KERNEL_CHECK(AlignRowsKernel);
  }
  *row0 = 0;
  return tc5::MatrixMap(w, q.type(), rows, q.h, p.ld_w, box_rows);
}

template <int kUnused>
inline void PackLaunch(const Problem &q, const Plan &p, char *ws, PackArgs a, cudaStream_t stream) {
  a.x = q.x, a.ld_x = q.ld_x, a.label = q.label, a.ignore = q.ignore;
  a.n = static_cast<int32_t>(q.n), a.v = static_cast<int32_t>(q.v), a.h = static_cast<int32_t>(q.h);
  a.pad_rows = p.pad_rows;
  a.packed = reinterpret_cast<uint16_t *>(ws + p.x), a.ld_packed = p.ld_x;
  a.words = reinterpret_cast<int32_t *>(ws + p.words);
  a.label_of = reinterpret_cast<int32_t *>(ws + p.label_of);
  a.vec = a.tiled = Aligned16(q.x, q.ld_x, 2);
  a.rows_per_cta = 16;
  a.counts = nullptr;
  if (p.pad_rows > kCountDirectly) {
    a.rows_per_cta = 256;
    a.counts = reinterpret_cast<float2 *>(ws + p.counts);
    gpu_rt::LaunchAfterDrain(CountRowsKernel<kUnused>, dim3(static_cast<unsigned>(p.pad_rows / 256)), dim3(256), 0, stream, a);
    MSHADOW_CUDA_POST_KERNEL_CHECK(CountRowsKernel);
  }
  gpu_rt::LaunchAfterDrain(PackRowsKernel<kUnused>, dim3(static_cast<unsigned>(p.pad_rows / a.rows_per_cta)), dim3(256), 0, stream, a);
  MSHADOW_CUDA_POST_KERNEL_CHECK(PackRowsKernel);
}

template <int kUnused>
inline void ForwardLaunch(float *loss, float *lse, const Problem &q, const Plan &p, char *ws, int sms, cudaStream_t stream) {
  if (p.pack) {
    PackArgs k = {};
    k.row_of = reinterpret_cast<int32_t *>(ws + p.row_of);
    k.loss = loss, k.lse_out = lse;
    PackLaunch<kUnused>(q, p, ws, k, stream);
  }
  GemmArgs a = {};
  a.live = p.pack ? reinterpret_cast<const int32_t *>(ws + p.words) : nullptr;
  a.tokens = static_cast<int32_t>(q.n);
  a.k_blocks = static_cast<int32_t>(Ceil(q.h, kStepK));
  a.run_steps = RunSteps(kStat, false);
  const int64_t m_tiles = Ceil(q.n, 128 * p.ctas);
  a.group = GroupOf(m_tiles, 16);
  a.instr = tc5::InstrDesc(q.bf16, false, false, 128 * p.ctas, static_cast<int>(p.tile_n));
  a.tile_n = static_cast<int32_t>(p.tile_n);
  a.pad_rows = p.pad_rows;
  a.label = p.pack ? reinterpret_cast<const int32_t *>(ws + p.label_of) : q.label;
  a.part = reinterpret_cast<float2 *>(ws + p.part);
  a.part_sum = q.smooth != 0.0f ? reinterpret_cast<float *>(ws + p.part_sum) : nullptr;
  a.label_logit = reinterpret_cast<float *>(ws + p.label_logit);
  a.bf16 = q.bf16;
  a.status = gpu_rt::StatusWord();
  const CUtensorMap ma = p.pack ? tc5::MatrixMap(ws + p.x, q.type(), p.pad_rows, q.h, p.ld_x, 128)
                                : tc5::MatrixMap(q.x, q.type(), q.n, q.h, q.ld_x, 128);
  const CUtensorMap mx = Aligned16(q.x, q.ld_x, 2) ? tc5::MatrixMap(q.x, q.type(), q.n, q.h, q.ld_x, 128) : ma;
  for (int64_t p0 = 0; p0 < q.v; p0 += p.piece) {
    const int64_t cols = std::min(p.piece, q.v - p0);
    const CUtensorMap mb = WeightMap<kUnused>(q, p, ws, p0, cols, static_cast<int>(p.tile_n) / p.ctas, stream, true, &a.b_row0);
    a.cols = static_cast<int32_t>(cols);
    a.col0 = static_cast<int32_t>(p0);
    a.tile0 = static_cast<int32_t>(p0 / p.tile_n);
    a.n_tiles = static_cast<int32_t>(Ceil(cols, p.tile_n));
    Gemm<kStat>(ma, mb, mx, mb, a, a.k_blocks, m_tiles * a.n_tiles, p.ctas, sms, stream);
  }
  JoinArgs j = {};
  j.live = a.live, j.tokens = a.tokens, j.parts = static_cast<int32_t>(2 * p.tiles), j.v = static_cast<int32_t>(q.v);
  j.pad_rows = p.pad_rows, j.part = a.part, j.part_sum = a.part_sum, j.label_logit = a.label_logit;
  j.label = a.label, j.row_of = p.pack ? reinterpret_cast<const int32_t *>(ws + p.row_of) : nullptr;
  j.ignore = q.ignore, j.smooth = q.smooth, j.loss = loss, j.lse = lse;
  if (q.n <= 1024) {
    gpu_rt::LaunchAfterDrain(JoinTilesKernel<4>, dim3(gpu_rt::CeilDiv(q.n, 4)), dim3(512), 0, stream, j);
  } else {
    gpu_rt::LaunchAfterDrain(JoinTilesKernel<32>, dim3(gpu_rt::CeilDiv(q.n, 32)), dim3(512), 0, stream, j);
  }
  MSHADOW_CUDA_POST_KERNEL_CHECK(JoinTilesKernel);
}

struct GradOut {
  uint16_t *gx;
  int64_t ld_gx;
  void *gw;
  int64_t ld_gw;
  int gw_type;
  bool gw_add;
  const float *lse, *gloss;
  float scale;
};

template <int kUnused>
inline void BackwardLaunch(const GradOut &g, const Problem &q, const Plan &p, char *ws, int sms, cudaStream_t stream) {
  PackArgs k = {};
  k.pos_of = reinterpret_cast<int32_t *>(ws + p.pos_of);
  k.lse = g.lse, k.gloss = g.gloss, k.scale = g.scale, k.q_label = static_cast<float>(1.0 - q.smooth);
  k.lse2 = reinterpret_cast<float *>(ws + p.lse2);
  k.row_scale = reinterpret_cast<float *>(ws + p.row_scale);
  // (bfloat16 has the exponents for a common scale; without the gradient of x there is no use for another)
  if (!q.bf16 && g.gloss != nullptr && g.gx != nullptr) k.row_down = reinterpret_cast<float *>(ws + p.row_down);
  PackLaunch<kUnused>(q, p, ws, k, stream);

  const int32_t h_tiles = static_cast<int32_t>(p.ld_acc / kTileN);
  const int type = q.type();
  float *acc = reinterpret_cast<float *>(ws + p.acc);
  char *delta = ws + p.delta;
  GemmArgs a = {};
  a.live = reinterpret_cast<const int32_t *>(ws + p.words);
  a.inv_scale = reinterpret_cast<const float *>(ws + p.words) + 1;
  a.pad_rows = p.pad_rows;
  a.label = reinterpret_cast<const int32_t *>(ws + p.label_of);
  a.lse2 = k.lse2;
  a.row_scale = k.row_scale;
  a.q_label = static_cast<float>(1.0 - q.smooth);
  a.q_other = q.smooth != 0.0f ? static_cast<float>(static_cast<double>(q.smooth) / (q.v - 1)) : 0.0f;
  a.bf16 = q.bf16;
  a.status = gpu_rt::StatusWord();
  a.earlier = p.runs ? reinterpret_cast<float4 *>(ws + p.earlier) : nullptr;
  const CUtensorMap x_along = tc5::MatrixMap(ws + p.x, type, p.pad_rows, q.h, p.ld_x, 128);
  const CUtensorMap x_across = tc5::MatrixMap(ws + p.x, type, p.pad_rows, q.h, p.ld_x, 64);
  const bool tiled = Aligned16(q.x, q.ld_x, 2);
  const CUtensorMap x_along_in_place = tiled ? tc5::MatrixMap(q.x, type, q.n, q.h, q.ld_x, 128) : x_along;
  const CUtensorMap x_across_in_place = tiled ? tc5::MatrixMap(q.x, type, q.n, q.h, q.ld_x, 64) : x_across;
  const CUtensorMap d_along = tc5::MatrixMap(delta, type, p.pad_rows, p.piece, p.piece, 128);
  const CUtensorMap d_across = tc5::MatrixMap(delta, type, p.pad_rows, p.piece, p.piece, 64);
  for (int64_t p0 = 0; p0 < q.v; p0 += p.piece) {
    const int64_t cols = std::min(p.piece, q.v - p0);
    const int64_t m_tiles = Ceil(q.n, 128 * p.ctas);
    a.cols = static_cast<int32_t>(cols);
    a.col0 = static_cast<int32_t>(p0);
    a.n_tiles = static_cast<int32_t>(Ceil(cols, kTileN));
    a.k_blocks = static_cast<int32_t>(Ceil(q.h, kStepK));
    a.run_steps = RunSteps(kDelta, false);
    a.group = GroupOf(m_tiles, 16);
    a.instr = tc5::InstrDesc(q.bf16, false, false, 128 * p.ctas, kTileN);
    const CUtensorMap w_along = WeightMap<kUnused>(q, p, ws, p0, cols, kTileN / p.ctas, stream, true, &a.b_row0);
    if (p.ctas == 2 && WideFor(m_tiles * a.n_tiles, a.n_tiles, a.k_blocks, sms)) {
      a.n_tiles /= 2;
      LaunchGemm<kDelta, 2, true>(x_along, w_along, x_along_in_place, d_along, a, a.k_blocks, m_tiles * a.n_tiles, sms, stream);
    } else {
      Gemm<kDelta>(x_along, w_along, x_along_in_place, d_along, a, a.k_blocks, m_tiles * a.n_tiles, p.ctas, sms, stream);
    }
    if (g.gx != nullptr) {
      const CUtensorMap w_across = WeightMap<kUnused>(q, p, ws, p0, cols, 64, stream, false, &a.b_row0);
      const CUtensorMap out = tc5::MatrixMap(acc, kFloat32, p.pad_rows, p.ld_acc, p.ld_acc, 128);
      const int64_t tile_n = kTileN * (p.wide_gx ? 2 : 1);
      const CUtensorMap spare =
          tc5::MatrixMap(ws + p.spare, kFloat32, static_cast<int64_t>(p.room) * 128 * p.ctas_gx, tile_n, tile_n, 128);
      const int64_t x_tiles = Ceil(q.n, 128 * p.ctas_gx);
      a.n_tiles = p.wide_gx ? h_tiles / 2 : h_tiles;
      a.step_cycles = static_cast<float>(StepCycles(p.shape_gx));
      a.tile_cycles = static_cast<float>(TileCycles(p.shape_gx));
      a.k_blocks = static_cast<int32_t>(Ceil(cols, kStepK));
      a.k_plan = static_cast<int32_t>(Ceil(std::min(p.piece, q.v), kStepK));
      a.run_steps = RunSteps(kDataGrad, false);
      a.room = p.room;
      a.accumulate = p0 > 0;
      a.group = GroupOf(x_tiles, 8);
      a.instr = tc5::InstrDesc(q.bf16, false, true, 128 * p.ctas_gx, kTileN);
      if (p.wide_gx) LaunchGemm<kDataGrad, 2, true>(d_along, w_across, spare, out, a, a.k_blocks, x_tiles * a.n_tiles, sms, stream);
      else Gemm<kDataGrad>(d_along, w_across, spare, out, a, a.k_blocks, x_tiles * a.n_tiles, p.ctas_gx, sms, stream);
    }
    if (g.gw != nullptr && k.row_down != nullptr) {
      gpu_rt::LaunchAfterDrain(CommonScaleKernel<kUnused>, dim3(static_cast<unsigned>(std::min<int64_t>(Ceil(q.n, 8), 8 * sms))), dim3(256),
                               0, stream, reinterpret_cast<uint16_t *>(delta), p.piece, a.live,
                               static_cast<const float *>(k.row_down), static_cast<int>(cols));
      MSHADOW_CUDA_POST_KERNEL_CHECK(CommonScaleKernel);
    }
    if (g.gw != nullptr) {
      const int64_t elem = g.gw_type == kFloat32 ? 4 : 2;
      const int ctas = CtasFor(cols, h_tiles, sms);
      a.m_tiles = static_cast<int32_t>(Ceil(cols, 128 * ctas));
      a.n_tiles = h_tiles;
      a.run_steps = RunSteps(kWeightGrad, g.gw_type == kFloat32);
      a.b_row0 = 0;
      a.group = GroupOf(a.m_tiles, 8);
      a.instr = tc5::InstrDesc(q.bf16, true, true, 128 * ctas, kTileN);
      a.out = static_cast<char *>(g.gw) + p0 * g.ld_gw * elem;
      a.ld_out = g.ld_gw;
      a.out_rows = static_cast<int32_t>(cols);
      a.out_cols = static_cast<int32_t>(q.h);
      a.out_type = g.gw_type;
      a.out_add = g.gw_add;
      a.out_vec = Aligned16(a.out, g.ld_gw, elem);
      // (a tiled copy leaves out columns past the matrix in units of 16 bytes: rows that do not end on such a
      // boundary would lose up to 14 bytes behind them to zeros.  It also adds, binary32 to binary32 (numbers below
      // 2^-126 count as zero); a 16-bit sum would be rounded twice, so those additions are plain accesses.)
      a.out_tiled = a.out_vec && (!a.out_add || a.out_type == kFloat32) && q.h * elem % 16 == 0;
      const CUtensorMap out = a.out_tiled ? tc5::MatrixMap(a.out, g.gw_type, cols, q.h, g.ld_gw, 128) : x_across;
      const int64_t tiles = static_cast<int64_t>(a.m_tiles) * h_tiles;
      if (ctas == 2 && WideFor(tiles, h_tiles, Ceil(q.n, kStepK), sms)) {
        a.n_tiles = h_tiles / 2;
        LaunchGemm<kWeightGrad, 2, true>(d_across, x_across, x_across_in_place, out, a, Ceil(q.n, kStepK), tiles / 2, sms, stream);
      } else {
        Gemm<kWeightGrad>(d_across, x_across, x_across_in_place, out, a, Ceil(q.n, kStepK), tiles, ctas, sms, stream);
      }
    }
  }
  if (g.gx != nullptr) {
    FinishArgs f = {};
    f.acc = acc, f.spare = reinterpret_cast<const float *>(ws + p.spare), f.ld_acc = p.ld_acc, f.live = a.live;
    f.n_tiles = p.wide_gx ? h_tiles / 2 : h_tiles;
    f.tile_n = p.wide_gx ? 2 * kTileN : kTileN;
    f.group = GroupOf(Ceil(q.n, 128 * p.ctas_gx), 8);
    f.k_plan = a.k_plan, f.room = p.room, f.slots = sms / p.ctas_gx, f.ctas = p.ctas_gx;
    f.step_cycles = a.step_cycles, f.tile_cycles = a.tile_cycles;
    f.pos_of = k.pos_of, f.inv_scale = a.inv_scale, f.row_down = k.row_down;
    f.out = g.gx, f.ld_out = g.ld_gx, f.n = static_cast<int32_t>(q.n), f.h = static_cast<int32_t>(q.h);
    f.bf16 = q.bf16, f.vec = Aligned16(g.gx, g.ld_gx, 2);
    f.groups = gpu_rt::FastDiv(static_cast<uint32_t>(Ceil(q.h, 8)));
    const int64_t blocks = std::min<int64_t>(Ceil(Ceil(q.n, 4) * Ceil(q.h, 8), 256), 4 * sms);
    const dim3 grid(static_cast<unsigned>(blocks));
    if (f.row_down != nullptr) gpu_rt::LaunchAfterDrain(DataGradFinishKernel<true>, grid, dim3(256), 0, stream, f);
    else gpu_rt::LaunchAfterDrain(DataGradFinishKernel<false>, grid, dim3(256), 0, stream, f);
    MSHADOW_CUDA_POST_KERNEL_CHECK(DataGradFinishKernel);
  }
}

}  // namespace vloss
}  // namespace cuda
}  // namespace mshadow
#endif  // MSHADOW_GPU_VOCAB_LOSS_CUH_
