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
 * thread issues the tiled copies of the operands, one the products, four warps (a thread per
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
 * out about as exact as their own final rounding leaves them.  Before it d is multiplied by a power
 * of two that brings the largest row scale to 2^14 .. 2^15 -- a mean over thousands of tokens puts most
 * of d below the smallest binary16 number otherwise -- and the results are divided by it again, exactly.
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
const int kThreads = 256;     // warp 0: copies, warp 1: products, warp 2: tensor memory, warps 4-7: epilogue
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

template <int kCtas>
struct StageShape {
  static const int kRowsN = kTileN / kCtas;                          // rows of B that a CTA holds
  static const uint32_t kBytesA = 128 * kStepK * 2;
  static const uint32_t kBytesB = kRowsN * kStepK * 2;
  static const uint32_t kStage = kBytesA + kBytesB;
  static const int kStages = kCtas == 2 ? 6 : 4;
  static const size_t kSmem = kStage * kStages + 1024;               // + alignment to the swizzle's 1024 bytes
};

struct GemmArgs {
  // extents
  const int32_t *live;   // device word: token rows that count; null: `tokens` do
  int32_t tokens;
  int32_t m_tiles;       // kWeightGrad: row tiles of the piece (else from the live rows)
  int32_t n_tiles;
  int32_t k_blocks;      // kWeightGrad: from the live rows
  int32_t slices;        // kDataGrad: the contraction is cut into this many parts
  int32_t group;         // row tiles that are walked before the next column tile
  int32_t b_row0;        // first row of B (the piece's first vocabulary row)
  uint32_t instr;
  // kStat, kDelta
  int32_t cols;          // columns of the piece that exist
  int32_t col0;          // class of the piece's first column
  int32_t tile0;         // kStat: tiles of the pieces before this one
  int64_t pad_rows;
  const int32_t *label;
  float2 *part;          // [tile][row]: maximum and sum of exp(z - maximum)
  float *part_sum;       // [tile][row]: sum of z, or null
  float *label_logit;    // [row]
  const float *lse2;     // [row]: lse in base 2
  const float *row_scale;
  float q_label, q_other;
  int bf16;
  uint16_t *delta;       // [row][ld_delta]
  int64_t ld_delta;
  // kDataGrad
  float *acc;            // [slice][row][ld_acc]
  int64_t ld_acc, acc_slice;
  int accumulate;
  // kWeightGrad
  const float *inv_scale;  // device word: what undoes the power of two in row_scale
  void *out;
  int64_t ld_out;
  int32_t out_rows, out_cols;
  int out_type;          // kFloat32, kFloat16, kBfloat16
  int out_add;
  int out_vec;           // rows of `out` start on 16-byte boundaries
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

/*! \brief one tile of the walk */
struct Unit {
  int m, n, slice;
};

/*! \brief unit u of the walk: `group` row tiles by all column tiles, then the next group; slices outermost */
__device__ __forceinline__ Unit UnitOf(int u, int m_tiles, int n_tiles, int group) {
  Unit t;
  const int plane = m_tiles * n_tiles;
  t.slice = u / plane;
  const int r = u - t.slice * plane;
  const int band = group * n_tiles;
  const int g = r / band;
  const int first = g * group;
  const int height = min(group, m_tiles - first);
  const int q = r - g * band;
  t.n = q / height;
  t.m = first + (q - t.n * height);
  return t;
}

// ---- epilogues: one thread per row of the tile, 32 columns at a time ----------------------------

/*!
 * \brief running maximum and sum of exponentials of one row.  The difference to the maximum is taken before the
 *  change of base (a product with log2 e folded into one multiply-add would save an addition, but it
 *  rounds at the size of the logit): the largest term is then exactly 1, and the loss of a token whose
 *  label has the largest logit is log(sum) with nothing cancelled, never negative.
 */
struct RowStat {
  float ref, sum, total;
  int label;  // column of the label within the tile, or outside [0, kTileN)
};

template <bool kTotal>
__device__ __forceinline__ void StatColumns(const uint32_t (&r)[32], int c0, int limit, RowStat *st, float *label_logit) {
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
  if (kTotal) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += c0 + i < limit ? v[i] : 0.0f;
    st->total += t;
  }
  if (c0 + 32 > limit) {  // columns past the vocabulary weigh nothing
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (c0 + i >= limit) v[i] = -INFINITY;
    }
  }
  float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int i = 4; i < 32; ++i) m[i & 3] = fmaxf(m[i & 3], v[i]);
  const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  const float ref = fmaxf(st->ref, top);
  const float from = ref == -INFINITY ? 0.0f : ref;  // nothing but -infinity so far: any finite reference serves
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i & 3] += Exp2((v[i] - from) * kLog2e);
  st->sum = st->sum * Exp2((st->ref - from) * kLog2e) + ((s[0] + s[1]) + (s[2] + s[3]));
  st->ref = ref;
  if (static_cast<unsigned>(st->label - c0) < 32u) {
    const int at = st->label - c0;
    float z = v[0];
#pragma unroll
    for (int i = 1; i < 32; ++i) z = i == at ? v[i] : z;
    *label_logit = z;
  }
}

__device__ __forceinline__ void DeltaColumns(const uint32_t (&r)[32], int c0, int limit, int label, float lse2,
                                             float scale, const GemmArgs &a, uint16_t *out) {
  float d[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) d[i] = (Exp2(__fmaf_rn(__uint_as_float(r[i]), kLog2e, -lse2)) - a.q_other) * scale;
  if (static_cast<unsigned>(label - c0) < 32u) {
    const int at = label - c0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i == at) d[i] = (Exp2(__fmaf_rn(__uint_as_float(r[i]), kLog2e, -lse2)) - a.q_label) * scale;
    }
  }
  if (c0 + 32 > limit) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (c0 + i >= limit) d[i] = 0.0f;
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 p;
    p.x = PackPair(d[8 * q], d[8 * q + 1], a.bf16);
    p.y = PackPair(d[8 * q + 2], d[8 * q + 3], a.bf16);
    p.z = PackPair(d[8 * q + 4], d[8 * q + 5], a.bf16);
    p.w = PackPair(d[8 * q + 6], d[8 * q + 7], a.bf16);
    reinterpret_cast<uint4 *>(out)[q] = p;
  }
}

__device__ __forceinline__ void AccColumns(const uint32_t (&r)[32], float *out, int accumulate) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    float4 v = make_float4(__uint_as_float(r[4 * q]), __uint_as_float(r[4 * q + 1]), __uint_as_float(r[4 * q + 2]),
                           __uint_as_float(r[4 * q + 3]));
    float4 *p = reinterpret_cast<float4 *>(out) + q;
    if (accumulate) {
      const float4 o = *p;
      v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
    }
    *p = v;
  }
}

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

template <int kMode>
__device__ __forceinline__ void FinishTile(const Unit &u, uint32_t acc, int64_t row, int live, const GemmArgs &a) {
  uint32_t r[32];
  if (kMode == kStat || kMode == kDelta) {
    const int limit = a.cols - u.n * kTileN;  // columns of this tile that exist
    const int col = a.col0 + u.n * kTileN;    // class of its first column
    const int label = row < live ? a.label[row] : -1;
    if (kMode == kStat) {
      RowStat st = {-INFINITY, 0.0f, 0.0f, label < 0 ? -1 : label - col};
      const int chunks = min(kTileN / 32, (limit + 31) / 32);
      for (int c = 0; c < chunks; ++c) {
        tc5::LoadColumns(acc + c * 32, r);
        tc5::WaitColumns(r);
        if (a.part_sum != nullptr) StatColumns<true>(r, c * 32, limit, &st, a.label_logit + row);
        else StatColumns<false>(r, c * 32, limit, &st, a.label_logit + row);
      }
      const int64_t at = static_cast<int64_t>(a.tile0 + u.n) * a.pad_rows + row;
      a.part[at] = make_float2(st.ref, st.sum);
      if (a.part_sum != nullptr) a.part_sum[at] = st.total;
    } else {
      const int at = label < 0 ? -1 : label - col;
      const float lse2 = a.lse2[row], scale = a.row_scale[row];  // rows past the live ones: 0 and 0
      uint16_t *out = a.delta + row * a.ld_delta + u.n * kTileN;
      for (int c = 0; c < kTileN / 32; ++c) {
        tc5::LoadColumns(acc + c * 32, r);
        tc5::WaitColumns(r);
        DeltaColumns(r, c * 32, limit, at, lse2, scale, a, out + c * 32);
      }
    }
  } else if (kMode == kDataGrad) {
    float *out = a.acc + u.slice * a.acc_slice + row * a.ld_acc + u.n * kTileN;
    for (int c = 0; c < kTileN / 32; ++c) {
      tc5::LoadColumns(acc + c * 32, r);
      tc5::WaitColumns(r);
      AccColumns(r, out + c * 32, a.accumulate);
    }
  } else {
    const float inv = a.inv_scale[0];
    for (int c = 0; c < kTileN / 32; ++c) {
      tc5::LoadColumns(acc + c * 32, r);
      tc5::WaitColumns(r);
      if (row < a.out_rows) WeightColumns(r, row, u.n * kTileN + c * 32, inv, a);
    }
  }
}

/*!
 * \brief persistent product kernel of all four modes.  kCtas CTAs (a cluster) share a tile of
 *  128 * kCtas rows by 256 columns.  Block of 256 threads; dynamic shared memory StageShape<kCtas>::kSmem.
 */
template <int kMode, int kCtas>
__global__ void __launch_bounds__(kThreads, 1)
VocabGemmKernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GemmArgs a) {
  typedef StageShape<kCtas> S;
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
      tma::BarrierInit(&acc_empty[s], 128 * kCtas);
    }
    tc5::PrefetchMap(&map_a);
    tc5::PrefetchMap(&map_b);
  }
  if (warp == 2) tc5::AllocTensorMemory<kCtas>(&tmem_slot);
  tc5::FenceBefore();
  __syncthreads();
  if (kCtas == 2) tc5::ClusterSync();
  tc5::FenceAfter();
  const uint32_t tmem = tmem_slot;
  gpu_rt::GridDependencySync();

  const int live = a.live != nullptr ? *a.live : a.tokens;
  const int tile_m = 128 * kCtas;
  // an empty batch still passes one tile of zeros through the products that end in d and in grad W
  const int m_tiles = kMode == kWeightGrad ? a.m_tiles
                      : kMode == kDelta    ? max(1, (live + tile_m - 1) / tile_m)
                                           : (live + tile_m - 1) / tile_m;
  const int k_blocks = kMode == kWeightGrad ? max(1, (live + kStepK - 1) / kStepK) : a.k_blocks;
  const int units = m_tiles * a.n_tiles * a.slices;
  const int first = blockIdx.x / kCtas, step = gridDim.x / kCtas;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t fill = 0;  // stages filled so far
      bool ok = true;
      for (int w = first; ok && w < units; w += step) {
        const Unit u = UnitOf(w, m_tiles, a.n_tiles, a.group);
        const int k_begin = u.slice * k_blocks / a.slices, k_end = (u.slice + 1) * k_blocks / a.slices;
        const int m0 = u.m * tile_m + static_cast<int>(rank) * 128;
        const int n0 = u.n * kTileN + static_cast<int>(rank) * S::kRowsN;
        for (int kb = k_begin; kb < k_end; ++kb, ++fill) {
          const int s = fill % S::kStages;
          const uint32_t use = fill / S::kStages;
          if (use > 0 && !tma::WaitBounded(&empty[s], (use - 1) & 1u)) {
            ok = false;
            break;
          }
          const uint32_t bar = kCtas == 2 ? tc5::MapToRank(tma::SharedAddr(&full[s]), 0) : tma::SharedAddr(&full[s]);
          if (rank == 0) tma::BarrierExpect(&full[s], S::kStage * kCtas);
          const uint32_t sa = smem + s * S::kStage, sb = sa + S::kBytesA;
          const int k0 = kb * kStepK;
          if (L::kAAcross) {
#pragma unroll
            for (int j = 0; j < 2; ++j) tc5::LoadBox<kCtas>(sa + j * tc5::kBoxBytes, &map_a, m0 + 64 * j, k0, bar);
          } else {
            tc5::LoadBox<kCtas>(sa, &map_a, k0, m0, bar);
          }
          if (L::kBAcross) {
#pragma unroll
            for (int j = 0; j < S::kRowsN / 64; ++j)
              tc5::LoadBox<kCtas>(sb + j * tc5::kBoxBytes, &map_b, n0 + 64 * j, a.b_row0 + k0, bar);
          } else {
            tc5::LoadBox<kCtas>(sb, &map_b, k0, a.b_row0 + n0, bar);
          }
        }
      }
      if (!ok) atomicExch(a.status, tma::kStatusBulkCopyTimeout);
      // every stage handed back: the products have read all copies of this CTA, and no arrival is
      // still on its way to these barriers when the CTA leaves
      for (uint32_t i = fill > S::kStages ? fill - S::kStages : 0; i < fill; ++i) {
        if (!tma::WaitBounded(&empty[i % S::kStages], (i / S::kStages) & 1u)) atomicExch(a.status, tma::kStatusBulkCopyTimeout);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      uint32_t fill = 0, tile = 0;
      bool ok = true;
      for (int w = first; ok && w < units; w += step, ++tile) {
        const Unit u = UnitOf(w, m_tiles, a.n_tiles, a.group);
        const int k_begin = u.slice * k_blocks / a.slices, k_end = (u.slice + 1) * k_blocks / a.slices;
        const uint32_t half = tile & 1u, use = tile >> 1;
        if (use > 0 && !tma::WaitBounded(&acc_empty[half], (use - 1) & 1u)) {
          ok = false;
          break;
        }
        tc5::FenceAfter();
        const uint32_t acc = tmem + half * kTileN;
        for (int kb = k_begin; kb < k_end; ++kb, ++fill) {
          const int s = fill % S::kStages;
          if (!tma::WaitBounded(&full[s], (fill / S::kStages) & 1u)) {
            ok = false;
            break;
          }
          tc5::FenceAfter();
          const uint32_t sa = smem + s * S::kStage, sb = sa + S::kBytesA;
          const uint64_t da = L::kAAcross ? tc5::DescAcrossK(sa) : tc5::DescAlongK(sa);
          const uint64_t db = L::kBAcross ? tc5::DescAcrossK(sb) : tc5::DescAlongK(sb);
          const uint32_t step_a = L::kAAcross ? 2048 >> 4 : 32 >> 4, step_b = L::kBAcross ? 2048 >> 4 : 32 >> 4;
#pragma unroll
          for (int j = 0; j < kStepK / 16; ++j) {
            tc5::Multiply<kCtas>(acc, da + j * step_a, db + j * step_b, a.instr, kb > k_begin || j > 0);
          }
          tc5::CommitTo<kCtas>(&empty[s]);
        }
        if (ok) tc5::CommitTo<kCtas>(&acc_full[half]);
      }
      if (!ok) atomicExch(a.status, tma::kStatusBulkCopyTimeout);
    }
  } else if (warp >= 4) {
    const int quarter = warp - 4;
    uint32_t tile = 0;
    for (int w = first; w < units; w += step, ++tile) {
      const Unit u = UnitOf(w, m_tiles, a.n_tiles, a.group);
      const uint32_t half = tile & 1u;
      const bool ready = tma::WaitBounded(&acc_full[half], (tile >> 1) & 1u);
      if (!__all_sync(0xffffffffu, ready)) {
        if (lane == 0) atomicExch(a.status, tma::kStatusBulkCopyTimeout);
        break;
      }
      tc5::FenceAfter();
      const int64_t row = static_cast<int64_t>(u.m) * tile_m + static_cast<int>(rank) * 128 + quarter * 32 + lane;
      FinishTile<kMode>(u, tmem + half * kTileN + (static_cast<uint32_t>(quarter * 32) << 16), row, live, a);
      tc5::FenceBefore();
      if (kCtas == 2) tc5::ArriveCluster(tc5::MapToRank(tma::SharedAddr(&acc_empty[half]), 0));
      else tma::BarrierArrive(&acc_empty[half]);
    }
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
  int32_t *words;        // [0] = live rows, [1] = inv_scale (a float)
  int32_t *row_of;       // [pad_rows] token of packed row (forward)
  int32_t *pos_of;       // [n] packed row of token, or -1 (backward)
  int32_t *label_of;     // [pad_rows] label of packed row
  float *loss, *lse_out; // forward: rows that do not count become 0
  const float *lse;      // backward
  const float *gloss;    // backward, may be null
  float scale;
  float *lse2, *row_scale;  // [pad_rows], backward
  int vec;               // 16-byte copies possible
  int rows_per_cta;
};

__device__ __forceinline__ bool IsLive(int32_t label, int32_t ignore, int32_t v) {
  return label != ignore && label >= 0 && label < v;
}

/*!
 * \brief packs the live rows of x and what belongs to them, in token order.  A CTA takes
 *  rows_per_cta tokens (at most 256); where its first live row goes it finds by counting the labels before it
 *  itself (4 bytes per token from the L2), which spares a scan kernel and its launch.  The rows
 *  from the last live one up to the next multiple of kPadRows become zeros.
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
  for (int i = tid; i < a.n; i += 256) {
    const int on = IsLive(a.label[i], a.ignore, a.v) ? 1 : 0;
    total += on;
    before += i < base ? on : 0;
    if (a.gloss != nullptr && on) top = fmaxf(top, fabsf(a.gloss[i]));
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

  // the power of two that brings the largest row scale to [2^14, 2^15)
  float up = 1.0f, down = 1.0f;
  if (a.row_scale != nullptr) {
    const float largest = fabsf(a.scale) * (a.gloss != nullptr ? top : 1.0f);
    if (largest > 0.0f && largest < INFINITY) {
      const int e = min(100, max(-100, 14 - ilogbf(largest)));
      up = __int_as_float((127 + e) << 23);
      down = __int_as_float((127 - e) << 23);
    }
  }
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
      a.row_scale[pos] = a.scale * (a.gloss != nullptr ? a.gloss[i] : 1.0f) * up;
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
    reinterpret_cast<float *>(a.words)[1] = down;
  }
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

/*! \brief copies rows of 16-bit elements to rows that start on 16-byte boundaries */
template <int kUnused>
__global__ void __launch_bounds__(256)
AlignRowsKernel(uint16_t *dst, int64_t ld_dst, const uint16_t *src, int64_t ld_src, int rows, int cols) {
  gpu_rt::GridDependencySync();
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    for (int c = threadIdx.x; c < cols; c += 256) dst[r * ld_dst + c] = src[r * ld_src + c];
  }
}

struct JoinArgs {
  const int32_t *live;
  int32_t tokens, tiles, v;
  int64_t pad_rows;
  const float2 *part;
  const float *part_sum, *label_logit;
  const int32_t *label, *row_of;  // row_of null: packed row = token
  int32_t ignore;
  float smooth;
  float *loss, *lse;
};

/*! \brief joins the tiles' maxima and sums row by row: 32 rows per CTA, eight threads of a row share its tiles */
template <int kUnused>
__global__ void __launch_bounds__(256) JoinTilesKernel(const JoinArgs a) {
  gpu_rt::GridDependencySync();
  __shared__ float s_ref[8][33], s_sum[8][33], s_total[8][33];
  const int live = a.live != nullptr ? *a.live : a.tokens;
  const int r = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 32 + r;
  if (blockIdx.x * 32 >= live) return;
  float ref = -INFINITY, sum = 0.0f, total = 0.0f;
  if (row < live) {
    for (int t = q; t < a.tiles; t += 8) {
      const float2 p = a.part[t * a.pad_rows + row];
      const float top = fmaxf(ref, p.x), from = top == -INFINITY ? 0.0f : top;
      sum = sum * Exp2((ref - from) * kLog2e) + p.y * Exp2((p.x - from) * kLog2e);
      ref = top;
      if (a.part_sum != nullptr) total += a.part_sum[t * a.pad_rows + row];
    }
  }
  s_ref[q][r] = ref, s_sum[q][r] = sum, s_total[q][r] = total;
  __syncthreads();
  if (q != 0 || row >= live) return;
  for (int w = 1; w < 8; ++w) {
    const float other = s_ref[w][r], top = fmaxf(ref, other), from = top == -INFINITY ? 0.0f : top;
    sum = sum * Exp2((ref - from) * kLog2e) + s_sum[w][r] * Exp2((other - from) * kLog2e);
    ref = top;
    total += s_total[w][r];
  }
  const int32_t label = a.label[row];
  const int64_t to = a.row_of != nullptr ? a.row_of[row] : row;
  if (!IsLive(label, a.ignore, a.v)) {
    a.loss[to] = 0.0f, a.lse[to] = 0.0f;
    return;
  }
  // a handful of operations per row, in 64 bits: the maximum is tens of units large, the loss may be small
  const double log_sum = log(static_cast<double>(sum)), z = a.label_logit[row];
  double loss = (ref - z) + log_sum;
  if (a.part_sum != nullptr) {
    const double smooth = a.smooth;
    loss += smooth * z - smooth / (a.v - 1) * (total - z);
  }
  a.loss[to] = static_cast<float>(loss);
  a.lse[to] = static_cast<float>(ref + log_sum);
}

struct FinishArgs {
  const float *acc;
  int64_t ld_acc, acc_slice;
  int slices;
  const int32_t *pos_of;
  const float *inv_scale;
  uint16_t *out;
  int64_t ld_out;
  int32_t n, h;
  int bf16, vec;
};

/*! \brief gradient of x: parts of the contraction added in order, rounded once, rows back in token order */
template <int kUnused>
__global__ void __launch_bounds__(256) DataGradFinishKernel(const FinishArgs a) {
  gpu_rt::GridDependencySync();
  const float inv = a.inv_scale[0];
  const int groups = (a.h + 7) / 8;
  for (int64_t i = blockIdx.x; i < a.n; i += gridDim.x) {
    const int pos = a.pos_of[i];
    uint16_t *out = a.out + i * a.ld_out;
    for (int g = threadIdx.x; g < groups; g += 256) {
      float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      if (pos >= 0) {
        for (int s = 0; s < a.slices; ++s) {
          const float4 *p = reinterpret_cast<const float4 *>(a.acc + s * a.acc_slice + pos * a.ld_acc) + 2 * g;
          const float4 lo = __ldcs(p), hi = __ldcs(p + 1);
          v[0] += lo.x, v[1] += lo.y, v[2] += lo.z, v[3] += lo.w;
          v[4] += hi.x, v[5] += hi.y, v[6] += hi.z, v[7] += hi.w;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= inv;
      if (a.vec && 8 * g + 8 <= a.h) {
        uint4 w;
        w.x = PackPair(v[0], v[1], a.bf16);
        w.y = PackPair(v[2], v[3], a.bf16);
        w.z = PackPair(v[4], v[5], a.bf16);
        w.w = PackPair(v[6], v[7], a.bf16);
        reinterpret_cast<uint4 *>(out)[g] = w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (8 * g + j < a.h) out[8 * g + j] = static_cast<uint16_t>(PackPair(v[j], 0.0f, a.bf16) & 0xffffu);
        }
      }
    }
  }
}

// ---- host side ------------------------------------------------------------------------------------

const int64_t kDeltaBytes = int64_t(512) << 20;  // piece of d: larger pieces mean fewer passes over the gradient of x
const int64_t kCopyBytes = int64_t(128) << 20;   // piece of W copied to aligned rows where the caller's are not

inline int64_t RoundUp(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

/*! \brief how a call is cut, and where its scratch matrices lie (offsets in bytes) */
struct Plan {
  bool pack, copy_w;
  int64_t pad_rows, ld_x, ld_w, piece, ld_acc, tiles;
  int slices, ctas;
  int64_t words, row_of, pos_of, label_of, lse2, row_scale, x, w, part, part_sum, label_logit, delta, acc, bytes;
};

struct Problem {
  const uint16_t *x, *w;
  const int32_t *label;
  int64_t n, v, h, ld_x, ld_w;
  bool bf16;
  int32_t ignore;
  float smooth;
};

inline bool Aligned16(const void *p, int64_t ld, int64_t elem) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * elem % 16 == 0;
}

/*! \brief layout of a call; sms = multiprocessors of the device */
inline Plan MakePlan(int64_t n, int64_t v, int64_t h, bool gradient, bool want_gx, bool smooth, bool pack, bool copy_w,
                     int sms, int ctas) {
  Plan p = {};
  p.pack = pack;
  p.copy_w = copy_w;
  p.ctas = ctas;
  p.pad_rows = RoundUp(n, kPadRows);
  p.ld_x = RoundUp(h, 8);
  p.ld_w = RoundUp(h, 8);
  p.ld_acc = RoundUp(h, kTileN);
  p.tiles = (v + kTileN - 1) / kTileN;
  p.piece = p.tiles * kTileN;
  if (gradient) p.piece = std::min(p.piece, std::max<int64_t>(kTileN, kDeltaBytes / (2 * p.pad_rows) / kTileN * kTileN));
  if (copy_w) p.piece = std::min(p.piece, std::max<int64_t>(kTileN, kCopyBytes / (2 * p.ld_w) / kTileN * kTileN));
  p.slices = 1;
  if (gradient && want_gx) {
    // enough parts of the contraction to give every SM a tile, each at least eight steps long
    const int64_t tiles = RoundUp(p.pad_rows, 128 * ctas) / (128 * ctas) * (p.ld_acc / kTileN);
    const int64_t want = (sms / ctas + tiles - 1) / tiles, most = p.piece / kStepK / 8;
    p.slices = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(16, std::min(want, most))));
  }
  int64_t at = 0;
  auto take = [&at](int64_t bytes) {
    const int64_t was = at;
    at += RoundUp(bytes, 256);
    return was;
  };
  p.words = take(256);
  p.label_of = take(pack ? p.pad_rows * 4 : 0);
  p.row_of = take(pack && !gradient ? p.pad_rows * 4 : 0);
  p.pos_of = take(gradient ? p.pad_rows * 4 : 0);
  p.x = take(pack ? p.pad_rows * p.ld_x * 2 : 0);
  p.w = take(copy_w ? p.piece * p.ld_w * 2 : 0);
  if (gradient) {
    p.lse2 = take(p.pad_rows * 4);
    p.row_scale = take(p.pad_rows * 4);
    p.delta = take(p.pad_rows * p.piece * 2);
    p.acc = take(want_gx ? p.slices * p.pad_rows * p.ld_acc * 4 : 0);
  } else {
    p.part = take(p.tiles * p.pad_rows * 8);
    p.part_sum = take(smooth ? p.tiles * p.pad_rows * 4 : 0);
    p.label_logit = take(p.pad_rows * 4);
  }
  p.bytes = at;
  return p;
}

#ifndef MSHADOW_B200_VLOSS_CTAS
#define MSHADOW_B200_VLOSS_CTAS 1
#endif
inline Plan PlanForward(const Problem &q, int sms) {
  const bool pack = q.n > 256 || !Aligned16(q.x, q.ld_x, 2);
  return MakePlan(q.n, q.v, q.h, false, false, q.smooth != 0.0f, pack, !Aligned16(q.w, q.ld_w, 2), sms, MSHADOW_B200_VLOSS_CTAS);
}
inline Plan PlanBackward(const Problem &q, bool want_gx, int sms) {
  return MakePlan(q.n, q.v, q.h, true, want_gx, q.smooth != 0.0f, true, !Aligned16(q.w, q.ld_w, 2), sms, MSHADOW_B200_VLOSS_CTAS);
}
/*! \brief scratch that suffices for every call of these sizes, whatever its layouts and options */
inline size_t WorkspaceNeed(int64_t n, int64_t v, int64_t h, bool gradient, int sms) {
  int64_t most = 0;
  for (int copy_w = 0; copy_w < 2; ++copy_w) {
    most = std::max(most, MakePlan(n, v, h, gradient, true, true, true, copy_w != 0, sms, MSHADOW_B200_VLOSS_CTAS).bytes);
  }
  return static_cast<size_t>(most);
}

template <int kMode, int kCtas>
inline void LaunchGemm(const CUtensorMap &ma, const CUtensorMap &mb, const GemmArgs &args, int64_t units, int sms,
                       cudaStream_t stream) {
  auto kernel = VocabGemmKernel<kMode, kCtas>;
  const size_t smem = StageShape<kCtas>::kSmem;
  MSHADOW_CUDA_CALL(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(units, 1), sms / kCtas)) * kCtas);
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
  MSHADOW_CUDA_CALL(cudaLaunchKernelEx(&cfg, kernel, ma, mb, args));
  MSHADOW_CUDA_POST_KERNEL_CHECK(VocabGemmKernel);
}

template <int kMode>
inline void Gemm(const CUtensorMap &ma, const CUtensorMap &mb, const GemmArgs &args, int64_t units, int ctas, int sms,
                 cudaStream_t stream) {
  if (ctas == 2) LaunchGemm<kMode, 2>(ma, mb, args, units, sms, stream);
  else LaunchGemm<kMode, 1>(ma, mb, args, units, sms, stream);
}

/*! \brief row tiles walked before the next column tile: together their operand rows stay in the L2 */
inline int GroupOf(int64_t m_tiles) { return static_cast<int>(std::min<int64_t>(std::max<int64_t>(m_tiles, 1), 16)); }

/*! \brief the weight rows [p0, p0 + rows) as the products read them: map over W itself, or over an aligned copy */
inline CUtensorMap WeightMap(const Problem &q, const Plan &p, char *ws, int64_t p0, int64_t rows, int box_rows,
                             cudaStream_t stream, bool copy_now, int32_t *row0) {
  if (!p.copy_w) {
    *row0 = static_cast<int32_t>(p0);
    return tc5::MatrixMap(q.w, q.bf16, q.v, q.h, q.ld_w, box_rows);
  }
  uint16_t *w = reinterpret_cast<uint16_t *>(ws + p.w);
  if (copy_now) {
    gpu_rt::LaunchAfterDrain(AlignRowsKernel<0>, dim3(static_cast<unsigned>(std::min<int64_t>(rows, 4096))), dim3(256), 0,
                             stream, w, p.ld_w, q.w + p0 * q.ld_w, q.ld_w, static_cast<int>(rows), static_cast<int>(q.h));
    MSHADOW_CUDA_POST_KERNEL_CHECK(AlignRowsKernel);
  }
  *row0 = 0;
  return tc5::MatrixMap(w, q.bf16, rows, q.h, p.ld_w, box_rows);
}

inline void PackLaunch(const Problem &q, const Plan &p, char *ws, PackArgs a, cudaStream_t stream) {
  a.x = q.x, a.ld_x = q.ld_x, a.label = q.label, a.ignore = q.ignore;
  a.n = static_cast<int32_t>(q.n), a.v = static_cast<int32_t>(q.v), a.h = static_cast<int32_t>(q.h);
  a.pad_rows = p.pad_rows;
  a.packed = reinterpret_cast<uint16_t *>(ws + p.x), a.ld_packed = p.ld_x;
  a.words = reinterpret_cast<int32_t *>(ws + p.words);
  a.label_of = reinterpret_cast<int32_t *>(ws + p.label_of);
  a.vec = Aligned16(q.x, q.ld_x, 2);
  a.rows_per_cta = p.pad_rows >= 65536 ? 64 : 16;
  gpu_rt::LaunchAfterDrain(PackRowsKernel<0>, dim3(static_cast<unsigned>(p.pad_rows / a.rows_per_cta)), dim3(256), 0, stream, a);
  MSHADOW_CUDA_POST_KERNEL_CHECK(PackRowsKernel);
}

inline void ForwardLaunch(float *loss, float *lse, const Problem &q, const Plan &p, char *ws, int sms, cudaStream_t stream) {
  if (p.pack) {
    PackArgs k = {};
    k.row_of = reinterpret_cast<int32_t *>(ws + p.row_of);
    k.loss = loss, k.lse_out = lse;
    PackLaunch(q, p, ws, k, stream);
  }
  GemmArgs a = {};
  a.live = p.pack ? reinterpret_cast<const int32_t *>(ws + p.words) : nullptr;
  a.tokens = static_cast<int32_t>(q.n);
  a.k_blocks = gpu_rt::CeilDiv(q.h, kStepK);
  a.slices = 1;
  const int64_t m_tiles = (q.n + 128 * p.ctas - 1) / (128 * p.ctas);
  a.group = GroupOf(m_tiles);
  a.instr = tc5::InstrDesc(q.bf16, false, false, 128 * p.ctas, kTileN);
  a.pad_rows = p.pad_rows;
  a.label = p.pack ? reinterpret_cast<const int32_t *>(ws + p.label_of) : q.label;
  a.part = reinterpret_cast<float2 *>(ws + p.part);
  a.part_sum = q.smooth != 0.0f ? reinterpret_cast<float *>(ws + p.part_sum) : nullptr;
  a.label_logit = reinterpret_cast<float *>(ws + p.label_logit);
  a.bf16 = q.bf16;
  a.status = gpu_rt::StatusWord();
  const CUtensorMap ma = p.pack ? tc5::MatrixMap(ws + p.x, q.bf16, p.pad_rows, q.h, p.ld_x, 128)
                                : tc5::MatrixMap(q.x, q.bf16, q.n, q.h, q.ld_x, 128);
  for (int64_t p0 = 0; p0 < q.v; p0 += p.piece) {
    const int64_t cols = std::min(p.piece, q.v - p0);
    const CUtensorMap mb = WeightMap(q, p, ws, p0, cols, kTileN / p.ctas, stream, true, &a.b_row0);
    a.cols = static_cast<int32_t>(cols);
    a.col0 = static_cast<int32_t>(p0);
    a.tile0 = static_cast<int32_t>(p0 / kTileN);
    a.n_tiles = gpu_rt::CeilDiv(cols, kTileN);
    Gemm<kStat>(ma, mb, a, m_tiles * a.n_tiles, p.ctas, sms, stream);
  }
  JoinArgs j = {};
  j.live = a.live, j.tokens = a.tokens, j.tiles = static_cast<int32_t>(p.tiles), j.v = static_cast<int32_t>(q.v);
  j.pad_rows = p.pad_rows, j.part = a.part, j.part_sum = a.part_sum, j.label_logit = a.label_logit;
  j.label = a.label, j.row_of = p.pack ? reinterpret_cast<const int32_t *>(ws + p.row_of) : nullptr;
  j.ignore = q.ignore, j.smooth = q.smooth, j.loss = loss, j.lse = lse;
  gpu_rt::LaunchAfterDrain(JoinTilesKernel<0>, dim3(gpu_rt::CeilDiv(q.n, 32)), dim3(256), 0, stream, j);
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

inline void BackwardLaunch(const GradOut &g, const Problem &q, const Plan &p, char *ws, int sms, cudaStream_t stream) {
  PackArgs k = {};
  k.pos_of = reinterpret_cast<int32_t *>(ws + p.pos_of);
  k.lse = g.lse, k.gloss = g.gloss, k.scale = g.scale;
  k.lse2 = reinterpret_cast<float *>(ws + p.lse2);
  k.row_scale = reinterpret_cast<float *>(ws + p.row_scale);
  PackLaunch(q, p, ws, k, stream);

  const int rows = 128 * p.ctas;
  const int64_t m_tiles = (q.n + rows - 1) / rows;
  const int h_tiles = static_cast<int>(p.ld_acc / kTileN);
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
  a.delta = reinterpret_cast<uint16_t *>(ws + p.delta);
  a.ld_delta = p.piece;
  a.acc = reinterpret_cast<float *>(ws + p.acc);
  a.ld_acc = p.ld_acc;
  a.acc_slice = p.pad_rows * p.ld_acc;
  a.status = gpu_rt::StatusWord();
  const CUtensorMap x_along = tc5::MatrixMap(ws + p.x, q.bf16, p.pad_rows, q.h, p.ld_x, 128);
  const CUtensorMap x_across = tc5::MatrixMap(ws + p.x, q.bf16, p.pad_rows, q.h, p.ld_x, 64);
  const CUtensorMap d_along = tc5::MatrixMap(a.delta, q.bf16, p.pad_rows, p.piece, p.piece, 128);
  const CUtensorMap d_across = tc5::MatrixMap(a.delta, q.bf16, p.pad_rows, p.piece, p.piece, 64);
  for (int64_t p0 = 0; p0 < q.v; p0 += p.piece) {
    const int64_t cols = std::min(p.piece, q.v - p0);
    a.cols = static_cast<int32_t>(cols);
    a.col0 = static_cast<int32_t>(p0);
    a.slices = 1;
    a.n_tiles = gpu_rt::CeilDiv(cols, kTileN);
    a.k_blocks = gpu_rt::CeilDiv(q.h, kStepK);
    a.group = GroupOf(m_tiles);
    a.instr = tc5::InstrDesc(q.bf16, false, false, rows, kTileN);
    const CUtensorMap w_along = WeightMap(q, p, ws, p0, cols, kTileN / p.ctas, stream, true, &a.b_row0);
    Gemm<kDelta>(x_along, w_along, a, m_tiles * a.n_tiles, p.ctas, sms, stream);
    if (g.gx != nullptr) {
      const CUtensorMap w_across = WeightMap(q, p, ws, p0, cols, 64, stream, false, &a.b_row0);
      a.n_tiles = h_tiles;
      a.k_blocks = gpu_rt::CeilDiv(cols, kStepK);
      a.slices = std::min(p.slices, a.k_blocks);  // the last piece may be shorter than the parts are many
      a.accumulate = p0 > 0;
      a.instr = tc5::InstrDesc(q.bf16, false, true, rows, kTileN);
      Gemm<kDataGrad>(d_along, w_across, a, m_tiles * a.n_tiles * a.slices, p.ctas, sms, stream);
    }
    if (g.gw != nullptr) {
      const int64_t elem = g.gw_type == kFloat32 ? 4 : 2;
      a.m_tiles = gpu_rt::CeilDiv(cols, rows);
      a.n_tiles = h_tiles;
      a.slices = 1;
      a.b_row0 = 0;
      a.group = GroupOf(a.m_tiles);
      a.instr = tc5::InstrDesc(q.bf16, true, true, rows, kTileN);
      a.out = static_cast<char *>(g.gw) + p0 * g.ld_gw * elem;
      a.ld_out = g.ld_gw;
      a.out_rows = static_cast<int32_t>(cols);
      a.out_cols = static_cast<int32_t>(q.h);
      a.out_type = g.gw_type;
      a.out_add = g.gw_add;
      a.out_vec = Aligned16(a.out, g.ld_gw, elem);
      Gemm<kWeightGrad>(d_across, x_across, a, static_cast<int64_t>(a.m_tiles) * a.n_tiles, p.ctas, sms, stream);
    }
  }
  if (g.gx != nullptr) {
    FinishArgs f = {};
    f.acc = a.acc, f.ld_acc = p.ld_acc, f.acc_slice = a.acc_slice, f.slices = p.slices;
    f.pos_of = k.pos_of, f.inv_scale = a.inv_scale;
    f.out = g.gx, f.ld_out = g.ld_gx, f.n = static_cast<int32_t>(q.n), f.h = static_cast<int32_t>(q.h);
    f.bf16 = q.bf16, f.vec = Aligned16(g.gx, g.ld_gx, 2);
    gpu_rt::LaunchAfterDrain(DataGradFinishKernel<0>, dim3(static_cast<unsigned>(std::min<int64_t>(q.n, 8192))), dim3(256), 0, stream, f);
    MSHADOW_CUDA_POST_KERNEL_CHECK(DataGradFinishKernel);
  }
}

}  // namespace vloss
}  // namespace cuda
}  // namespace mshadow
#endif  // MSHADOW_GPU_VOCAB_LOSS_CUH_
