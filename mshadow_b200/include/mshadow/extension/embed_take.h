/*
 * EmbedTake / EmbedTakeGrad: the embedding look-up of a language model and its gradient.
 *
 *   EmbedTake(dst, table, index, scale):             dst[i] = scale * table[index[i]]
 *   EmbedTakeGrad<Saver>(dst, src, index, scale):    dst[r] (Saver) scale * sum of src[i] over index[i] == r
 *
 * They stand beside take() (mshadow/extension/take.h) and AddTakeGrad (mshadow/tensor_gpu-inl.h:216-235)
 * and differ from them where a language model needs it: binary16 and bfloat16 tables beside
 * binary32 ones, summed in binary32 and rounded once; a scale; and an index outside the table is a
 * token without a row -- padding, or a row another GPU holds -- which looks up zeros and adds nothing
 * (take and AddTakeGrad clip it to the table).  EmbedTakeGrad sorts the indices itself; Saver is sv::saveto
 * (every row of dst is written, zeros where no index names it) or sv::plusto (rows that are not named are not
 * written).  dst shares no element with another operand.  Equal calls give equal bits.
 *
 * `workspace`: at least EmbedTakeGradWorkspace() bytes of device memory, or NULL for the stream's scratch memory.
 * A call that is captured into a graph must bring its own.
 */
#ifndef MSHADOW_EXTENSION_EMBED_TAKE_H_
#define MSHADOW_EXTENSION_EMBED_TAKE_H_

#include "../bfloat.h"
#if MSHADOW_USE_CUDA && defined(__CUDACC__)
#include "../gpu/embed_take.cuh"

namespace mshadow {

template <typename DType>
inline void EmbedTake(Tensor<gpu, 2, DType> dst, const Tensor<gpu, 2, DType> &table, const Tensor<gpu, 1, int32_t> &index,
                      float scale = 1.0f) {
  CHECK_EQ(dst.size(0), index.size(0)) << "EmbedTake: shape mismatch";
  CHECK_EQ(dst.size(1), table.size(1)) << "EmbedTake: shape mismatch";
  cuda::embtake::TakeLaunch(dst.dptr_, dst.stride_, index.dptr_, table.dptr_, table.stride_, dst.size(0), table.size(0),
                            dst.size(1), scale, Stream<gpu>::GetStream(dst.stream_));
}

/*! \brief bytes of workspace for `n` indices and rows of `width` elements */
inline size_t EmbedTakeGradWorkspace(index_t n, index_t width) {
  return gpu_rt::WorkspaceBytes(static_cast<size_t>(cuda::embtake::MakeGradPlan(n, width).bytes));
}

template <typename Saver, typename DType>
inline void EmbedTakeGrad(Tensor<gpu, 2, DType> dst, const Tensor<gpu, 2, DType> &src, const Tensor<gpu, 1, int32_t> &index,
                          float scale = 1.0f, void *workspace = NULL,
                          size_t workspace_bytes = 0) {
  static_assert(std::is_same<Saver, sv::saveto>::value || std::is_same<Saver, sv::plusto>::value,
                "EmbedTakeGrad assigns or adds");
  CHECK_EQ(src.size(0), index.size(0)) << "EmbedTakeGrad: shape mismatch";
  CHECK_EQ(dst.size(1), src.size(1)) << "EmbedTakeGrad: shape mismatch";
  const cudaStream_t stream = Stream<gpu>::GetStream(dst.stream_);
  const cuda::embtake::GradPlan plan = cuda::embtake::MakeGradPlan(src.size(0), src.size(1));
  char *ws = gpu_rt::Workspace(workspace, workspace_bytes, static_cast<size_t>(plan.bytes), stream, "EmbedTakeGrad");
  cuda::embtake::GradLaunch(dst.dptr_, dst.stride_, src.dptr_, src.stride_, index.dptr_, src.size(0), dst.size(0),
                            dst.size(1), scale, std::is_same<Saver, sv::plusto>::value, plan, ws, stream);
}

}  // namespace mshadow
#endif  // MSHADOW_USE_CUDA && __CUDACC__
#endif  // MSHADOW_EXTENSION_EMBED_TAKE_H_
