/*
 * LinearSoftmaxLoss / LinearSoftmaxLossGrad: softmax cross entropy of a linear layer over a large
 * vocabulary, without the matrix of logits.
 *
 *   LinearSoftmaxLoss(loss, lse, data, weight, label):
 *     z = dot(data, weight.T());  lse[i] = log sum_k exp z[i][k]
 *     loss[i] = lse[i] - (1 - smooth) z[i][label[i]] - smooth / (v - 1) * (sum over the other classes of z[i])
 *   LinearSoftmaxLossGrad<Saver>(gdata, gweight, data, weight, label, lse, gloss, scale):
 *     the gradients of sum_i scale * gloss[i] * loss[i]  (gloss: NULL data pointer = all ones);
 *     gdata is assigned, gweight assigned (sv::saveto) or added to (sv::plusto)
 *
 * Composed from the framework's other operators this is a matrix product, Softmax, and SoftmaxGrad or
 * SmoothSoftmaxGrad (mshadow/tensor_gpu-inl.h:157-214; the smoothing is theirs) with two more products,
 * and holds tokens x vocabulary logits and probabilities.  Here the products run in the same kernels.
 * What the gradient holds is a piece of the vocabulary of bounded size; the loss holds 16 bytes for each token
 * and 256 classes (24 with smoothing).
 *
 * data (n x h) and weight (v x h) are binary16 or bfloat16; loss and lse are binary32; gdata has the type of
 * data; gweight that type or float.  Sums are binary32, of products that the tensor cores add: they cut off where
 * a rounding would round, which is bounded by adding long sums in runs (sums of one sign come out up to 6e-5 too
 * small, 1.2e-4 where the result has 16 bits).  In the gradients each entry of softmax - target is rounded to the operands'
 * type between the two products, whatever the type of gweight.  A class whose weight is -infinity has probability 0
 * and a zero row in gweight; gdata is NaN then, as 0 * infinity is.  In binary16 what a token adds to gweight is lost below
 * 2^-39 of the largest finite |gloss| / (1 - smooth).  float gradients that are added to may lose what they hold below
 * 2^-126.  A token whose label equals ignore_label, or lies
 * outside [0, v), contributes nothing: its loss and lse are 0, its gdata row is zero, and whatever
 * its data row holds reaches no result.  gdata or gweight may be empty (dptr_ == NULL): not computed.  Outputs share
 * no element with other operands, but gdata may lie in the memory of data.  Equal calls give equal bits.
 *
 * `workspace`: at least LinearSoftmaxLossWorkspace() bytes of device memory, or NULL for the stream's scratch memory.
 * A call that is captured into a graph must bring its own, and another call on the device precede it.
 */
#ifndef MSHADOW_EXTENSION_LINEAR_SOFTMAX_LOSS_H_
#define MSHADOW_EXTENSION_LINEAR_SOFTMAX_LOSS_H_

#include "../bfloat.h"
#if MSHADOW_USE_CUDA && defined(__CUDACC__)
#include "../gpu/vocab_loss.cuh"

namespace mshadow {

/*! \brief bytes of workspace for n tokens, v classes and h features; gradient: of the gradient, else of the loss */
inline size_t LinearSoftmaxLossWorkspace(index_t n, index_t v, index_t h, bool gradient) {
  if (n == 0) return 0;
  return gpu_rt::WorkspaceBytes(cuda::vloss::WorkspaceNeed(n, v, h, gradient, gpu_rt::CurrentDevice().sm_count));
}

namespace vlossdetail {
template <typename DType>
inline cuda::vloss::Problem MakeProblem(const Tensor<gpu, 2, DType> &data, const Tensor<gpu, 2, DType> &weight,
                                        const Tensor<gpu, 1, int32_t> &label, int ignore_label, float smooth) {
  static_assert(DataType<DType>::kFlag == kFloat16 || DataType<DType>::kFlag == kBfloat16,
                "LinearSoftmaxLoss: data and weight are half_t or bf16_t");
  CHECK_EQ(data.size(1), weight.size(1)) << "LinearSoftmaxLoss: shape mismatch";
  CHECK_EQ(data.size(0), label.size(0)) << "LinearSoftmaxLoss: shape mismatch";
  CHECK(weight.size(0) >= 1 && weight.size(1) >= 1) << "LinearSoftmaxLoss: empty weight";
  CHECK(smooth >= 0.0f && smooth < 1.0f) << "LinearSoftmaxLoss: smoothing outside [0, 1)";
  CHECK(smooth == 0.0f || weight.size(0) > 1) << "LinearSoftmaxLoss: smoothing over a single class";
  cuda::vloss::Problem q;
  q.x = reinterpret_cast<const uint16_t *>(data.dptr_), q.ld_x = data.stride_;
  q.w = reinterpret_cast<const uint16_t *>(weight.dptr_), q.ld_w = weight.stride_;
  q.label = label.dptr_;
  q.n = data.size(0), q.v = weight.size(0), q.h = data.size(1);
  q.bf16 = DataType<DType>::kFlag == kBfloat16;
  q.ignore = ignore_label;
  q.smooth = smooth;
  return q;
}
}  // namespace vlossdetail

template <typename DType>
inline void LinearSoftmaxLoss(Tensor<gpu, 1, float> loss, Tensor<gpu, 1, float> lse, const Tensor<gpu, 2, DType> &data,
                              const Tensor<gpu, 2, DType> &weight, const Tensor<gpu, 1, int32_t> &label,
                              int ignore_label = -1, float smooth = 0.0f, void *workspace = NULL,
                              size_t workspace_bytes = 0) {
  const cuda::vloss::Problem q = vlossdetail::MakeProblem(data, weight, label, ignore_label, smooth);
  CHECK(loss.size(0) == data.size(0) && lse.size(0) == data.size(0)) << "LinearSoftmaxLoss: shape mismatch";
  if (q.n == 0) return;
  const cudaStream_t stream = Stream<gpu>::GetStream(loss.stream_);
  const int sms = gpu_rt::CurrentDevice().sm_count;
  const cuda::vloss::Plan plan = cuda::vloss::PlanForward(q, sms);
  char *ws = gpu_rt::Workspace(workspace, workspace_bytes, static_cast<size_t>(plan.bytes), stream, "LinearSoftmaxLoss");
  cuda::vloss::ForwardLaunch<0>(loss.dptr_, lse.dptr_, q, plan, ws, sms, stream);
}

template <typename Saver, typename DType, typename GType>
inline void LinearSoftmaxLossGrad(Tensor<gpu, 2, DType> gdata, Tensor<gpu, 2, GType> gweight,
                                  const Tensor<gpu, 2, DType> &data, const Tensor<gpu, 2, DType> &weight,
                                  const Tensor<gpu, 1, int32_t> &label, const Tensor<gpu, 1, float> &lse,
                                  const Tensor<gpu, 1, float> &gloss, float scale, int ignore_label = -1,
                                  float smooth = 0.0f, void *workspace = NULL, size_t workspace_bytes = 0) {
  static_assert(std::is_same<Saver, sv::saveto>::value || std::is_same<Saver, sv::plusto>::value,
                "LinearSoftmaxLossGrad assigns or adds the weight's gradient");
  static_assert(std::is_same<GType, DType>::value || std::is_same<GType, float>::value,
                "LinearSoftmaxLossGrad: the weight's gradient has the weight's type or float");
  const cuda::vloss::Problem q = vlossdetail::MakeProblem(data, weight, label, ignore_label, smooth);
  CHECK_EQ(lse.size(0), data.size(0)) << "LinearSoftmaxLossGrad: shape mismatch";
  CHECK(gloss.dptr_ == NULL || gloss.size(0) == data.size(0)) << "LinearSoftmaxLossGrad: shape mismatch";
  CHECK(gdata.dptr_ == NULL || gdata.shape_ == data.shape_) << "LinearSoftmaxLossGrad: shape mismatch";
  CHECK(gweight.dptr_ == NULL || gweight.shape_ == weight.shape_) << "LinearSoftmaxLossGrad: shape mismatch";
  if (gdata.dptr_ == NULL && gweight.dptr_ == NULL) return;
  const cudaStream_t stream = Stream<gpu>::GetStream(gdata.dptr_ != NULL ? gdata.stream_ : gweight.stream_);
  const bool add = std::is_same<Saver, sv::plusto>::value;
  if (q.n == 0) {
    if (gweight.dptr_ != NULL && !add) {
      MSHADOW_CUDA_CALL(cudaMemset2DAsync(gweight.dptr_, gweight.stride_ * sizeof(GType), 0, q.h * sizeof(GType), q.v, stream));
    }
    return;
  }
  const int sms = gpu_rt::CurrentDevice().sm_count;
  const cuda::vloss::Plan plan = cuda::vloss::PlanBackward(q, gdata.dptr_ != NULL, sms);
  char *ws = gpu_rt::Workspace(workspace, workspace_bytes, static_cast<size_t>(plan.bytes), stream, "LinearSoftmaxLossGrad");
  cuda::vloss::GradOut g;
  g.gx = reinterpret_cast<uint16_t *>(gdata.dptr_), g.ld_gx = gdata.stride_;
  g.gw = gweight.dptr_, g.ld_gw = gweight.stride_;
  g.gw_type = DataType<GType>::kFlag;
  g.gw_add = add;
  g.lse = lse.dptr_, g.gloss = gloss.dptr_, g.scale = scale;
  cuda::vloss::BackwardLaunch<0>(g, q, plan, ws, sms, stream);
}

}  // namespace mshadow
#endif  // MSHADOW_USE_CUDA && __CUDACC__
#endif  // MSHADOW_EXTENSION_LINEAR_SOFTMAX_LOSS_H_
