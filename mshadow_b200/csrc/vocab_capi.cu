/*
 * C entries of the two ends of a language model over its vocabulary table: embedding look-up and gradient, and
 * softmax cross entropy over the table without the logits (declared in include/mshadow_b200.h).
 * Arguments are checked here; the work is EmbedTake*, LinearSoftmaxLoss* of the C++ API.
 */
#include "mshadow_b200.h"

#include <cmath>
#include <string>

#include "mshadow/tensor.h"

namespace msb_internal {
void SetLastError(const char *message);  // defined next to msb_last_error()
}

using namespace mshadow;  // NOLINT(*)
typedef mshadow::half::half_t half_t;
typedef mshadow::bfloat::bf16_t bf16_t;

// every entry that launches work runs inside an NVTX range named after it (-DMSHADOW_B200_NVTX=0: none)
#ifndef MSHADOW_B200_NVTX
#define MSHADOW_B200_NVTX 1
#endif
#if MSHADOW_B200_NVTX
#include <nvtx3/nvToolsExt.h>
#endif

namespace {

struct TraceRange {
#if MSHADOW_B200_NVTX
  explicit TraceRange(const char *name) { nvtxRangePushA(name); }
  ~TraceRange() { nvtxRangePop(); }
#else
  explicit TraceRange(const char *) {}
#endif
};

int Refuse(const char *name, int code, const std::string &msg) {
  msb_internal::SetLastError((std::string(name) + ": " + msg).c_str());
  return code;
}

#define VOCAB_REQUIRE(cond, code, msg) \
  if (!(cond)) return Refuse(__func__, code, msg)

/*! \brief runs `body`, turning whatever it throws into a status; nothing leaves through the C boundary */
template <typename Body>
int Guarded(const char *name, Body body) {
  TraceRange range(name);
  try {
    body();
  } catch (const gpu_rt::WorkspaceError &e) {
    return Refuse(name, MSB_ERR_ARGUMENT, e.what());
  } catch (const dmlc::Error &e) {
    const std::string what = e.what();
    const bool cuda = what.find("CUDA") != std::string::npos || what.find("ErrStr") != std::string::npos;
    return Refuse(name, cuda ? MSB_ERR_CUDA : MSB_ERR_SHAPE, what);
  } catch (const std::exception &e) {
    return Refuse(name, MSB_ERR_MEMORY, e.what());
  }
  return MSB_OK;
}

/*! \brief address of an element of `dtype` */
inline bool ElementAligned(const void *p, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % (dtype == kFloat32 ? 4 : 2) == 0;
}
/*! \brief addresses of int32 / float arrays */
template <typename... Pointers>
inline bool WordAligned(Pointers... p) {
  return ((reinterpret_cast<uintptr_t>(p) % 4 == 0) && ...);
}
inline bool FitsIndex(int64_t v) { return v >= 0 && v <= 0x7fffffffLL; }
inline bool LdOk(int64_t ld, int64_t width) { return ld >= width && FitsIndex(ld); }

/*! \brief a call recorded into a graph brings its workspace, and the device was used before the recording */
int CaptureCheck(const char *name, const void *workspace, bool needs_workspace, msb_stream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  const cudaError_t err = cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &status);
  if (err != cudaSuccess) return Refuse(name, MSB_ERR_CUDA, cudaGetErrorString(err));
  if (status == cudaStreamCaptureStatusNone) return MSB_OK;
  if (needs_workspace && workspace == nullptr) {
    return Refuse(name, MSB_ERR_ARGUMENT, "a call captured into a graph needs a workspace of the caller's");
  }
  if (!gpu_rt::StatusWordReady()) {
    return Refuse(name, MSB_ERR_ARGUMENT, "the first call on a device (or msb_stream_wait) must precede a capture");
  }
  return MSB_OK;
}

/*!
 * \brief every pointer that is not null names memory of the current device (or managed memory).  A kernel given host
 *  memory, or memory of a GPU it cannot reach, faults, and takes the process's context with it; asking costs a fraction of a
 *  microsecond.
 */
template <typename... Pointers>
int PlaceCheck(const char *name, Pointers... pointers) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return Refuse(name, MSB_ERR_CUDA, std::string("CUDA: ") + cudaGetErrorString(err));
  const void *all[] = {static_cast<const void *>(pointers)...};
  for (const void *p : all) {
    if (p == nullptr) continue;
    cudaPointerAttributes at;
    err = cudaPointerGetAttributes(&at, p);
    if (err != cudaSuccess) {
      (void)cudaGetLastError();
      return Refuse(name, MSB_ERR_CUDA, std::string("CUDA: ") + cudaGetErrorString(err));
    }
    if (at.type == cudaMemoryTypeManaged) continue;
    if (at.type != cudaMemoryTypeDevice) return Refuse(name, MSB_ERR_ARGUMENT, "an operand is not device memory");
    if (at.device != dev) {
      return Refuse(name, MSB_ERR_ARGUMENT, "an operand is memory of device " + std::to_string(at.device) + " while device " +
                                                std::to_string(dev) + " is current");
    }
  }
  return MSB_OK;
}

template <typename DType>
inline Tensor<gpu, 2, DType> Mat(const void *p, int64_t r, int64_t c, int64_t ld, Stream<gpu> *s) {
  return Tensor<gpu, 2, DType>(static_cast<DType *>(const_cast<void *>(p)), Shape2(r, c), static_cast<index_t>(ld), s);
}
template <typename DType>
inline Tensor<gpu, 1, DType> Vec(const void *p, int64_t n, Stream<gpu> *s) {
  return Tensor<gpu, 1, DType>(static_cast<DType *>(const_cast<void *>(p)), Shape1(n), s);
}

struct Borrowed {
  Stream<gpu> s;
  explicit Borrowed(msb_stream_t raw) { s.stream_ = static_cast<cudaStream_t>(raw); }
};

}  // namespace

extern "C" {

int msb_embed_take(void *dst, const void *table, const int32_t *index, int64_t n, int64_t rows, int64_t width,
                   int64_t ld_dst, int64_t ld_table, int dtype, float scale, msb_stream_t stream) {
  VOCAB_REQUIRE(dtype == kFloat32 || dtype == kFloat16 || dtype == kBfloat16, MSB_ERR_ARGUMENT,
                "dtype must be 0 (float32), 2 (float16) or 12 (bfloat16)");
  VOCAB_REQUIRE(FitsIndex(n) && FitsIndex(rows) && FitsIndex(width), MSB_ERR_SHAPE, "extent out of range");
  VOCAB_REQUIRE(LdOk(ld_dst, width) && LdOk(ld_table, width), MSB_ERR_SHAPE, "stride < width");
  if (n == 0 || width == 0) return MSB_OK;
  VOCAB_REQUIRE(dst && index && (table || rows == 0), MSB_ERR_ARGUMENT, "null pointer");
  VOCAB_REQUIRE(ElementAligned(dst, dtype) && ElementAligned(table, dtype) && WordAligned(index), MSB_ERR_LAYOUT,
                "operands must be aligned to their elements");
  const int rc = PlaceCheck(__func__, dst, table, index);
  if (rc != MSB_OK) return rc;
  return Guarded(__func__, [&] {
    Borrowed st(stream);
    const Tensor<gpu, 1, int32_t> idx = Vec<int32_t>(index, n, &st.s);
    if (dtype == kFloat32) {
      EmbedTake(Mat<float>(dst, n, width, ld_dst, &st.s), Mat<float>(table, rows, width, ld_table, &st.s), idx, scale);
    } else if (dtype == kFloat16) {
      EmbedTake(Mat<half_t>(dst, n, width, ld_dst, &st.s), Mat<half_t>(table, rows, width, ld_table, &st.s),
                idx, scale);
    } else {
      EmbedTake(Mat<bf16_t>(dst, n, width, ld_dst, &st.s),
                Mat<bf16_t>(table, rows, width, ld_table, &st.s), idx, scale);
    }
  });
}

int msb_embed_take_grad_workspace(int64_t n, int64_t width, int64_t *bytes) {
  VOCAB_REQUIRE(bytes != nullptr, MSB_ERR_ARGUMENT, "null output");
  VOCAB_REQUIRE(FitsIndex(n) && FitsIndex(width), MSB_ERR_SHAPE, "extent out of range");
  return Guarded(__func__, [&] {
    *bytes = static_cast<int64_t>(EmbedTakeGradWorkspace(static_cast<index_t>(n), static_cast<index_t>(width)));
  });
}

int msb_embed_take_grad(void *dst, const void *src, const int32_t *index, int64_t n, int64_t rows, int64_t width,
                        int64_t ld_dst, int64_t ld_src, int dtype, float scale, int saver, void *workspace,
                        int64_t workspace_bytes, msb_stream_t stream) {
  VOCAB_REQUIRE(dtype == kFloat32 || dtype == kFloat16 || dtype == kBfloat16, MSB_ERR_ARGUMENT,
                "dtype must be 0 (float32), 2 (float16) or 12 (bfloat16)");
  VOCAB_REQUIRE(saver == 0 || saver == 1, MSB_ERR_ARGUMENT, "saver must be 0 (assign) or 1 (add)");
  VOCAB_REQUIRE(FitsIndex(n) && FitsIndex(rows) && FitsIndex(width), MSB_ERR_SHAPE, "extent out of range");
  VOCAB_REQUIRE(LdOk(ld_dst, width) && LdOk(ld_src, width), MSB_ERR_SHAPE, "stride < width");
  if (rows == 0 || width == 0 || (n == 0 && saver == 1)) return MSB_OK;
  VOCAB_REQUIRE(dst && (n == 0 || (src && index)), MSB_ERR_ARGUMENT, "null pointer");
  VOCAB_REQUIRE(ElementAligned(dst, dtype) && ElementAligned(src, dtype) && WordAligned(index), MSB_ERR_LAYOUT,
                "operands must be aligned to their elements");
  int64_t need = 0;
  int rc = msb_embed_take_grad_workspace(n, width, &need);
  if (rc != MSB_OK) return rc;
  VOCAB_REQUIRE(workspace == nullptr || workspace_bytes >= need, MSB_ERR_ARGUMENT, "workspace too small");
  rc = PlaceCheck(__func__, dst, src, index, workspace);
  if (rc == MSB_OK) rc = CaptureCheck(__func__, workspace, need > 0, stream);
  if (rc != MSB_OK) return rc;
  return Guarded(__func__, [&] {
    Borrowed st(stream);
    const Tensor<gpu, 1, int32_t> idx = Vec<int32_t>(index, n, &st.s);
    const size_t bytes = static_cast<size_t>(workspace_bytes < 0 ? 0 : workspace_bytes);
#define VOCAB_GRAD(T)                                                                                        \
  if (saver == 1) EmbedTakeGrad<sv::plusto>(Mat<T>(dst, rows, width, ld_dst, &st.s),                         \
                                            Mat<T>(src, n, width, ld_src, &st.s), idx, scale, workspace, bytes); \
  else EmbedTakeGrad<sv::saveto>(Mat<T>(dst, rows, width, ld_dst, &st.s), Mat<T>(src, n, width, ld_src, &st.s), \
                                 idx, scale, workspace, bytes)
    if (dtype == kFloat32) {
      VOCAB_GRAD(float);
    } else if (dtype == kFloat16) {
      VOCAB_GRAD(half_t);
    } else {
      VOCAB_GRAD(bf16_t);
    }
#undef VOCAB_GRAD
  });
}

int msb_linear_softmax_loss_workspace(int64_t n, int64_t v, int64_t h, int gradient, int64_t *bytes) {
  VOCAB_REQUIRE(bytes != nullptr, MSB_ERR_ARGUMENT, "null output");
  VOCAB_REQUIRE(FitsIndex(n) && FitsIndex(v) && FitsIndex(h) && v >= 1 && h >= 1, MSB_ERR_SHAPE, "extent out of range");
  return Guarded(__func__, [&] {
    *bytes = static_cast<int64_t>(LinearSoftmaxLossWorkspace(static_cast<index_t>(n), static_cast<index_t>(v),
                                                             static_cast<index_t>(h), gradient != 0));
  });
}

int msb_linear_softmax_loss(float *loss, float *lse, const void *data, const void *weight, const int32_t *label,
                            int64_t n, int64_t v, int64_t h, int64_t ld_data, int64_t ld_weight, int dtype,
                            int32_t ignore_label, float smooth, void *workspace, int64_t workspace_bytes,
                            msb_stream_t stream) {
  VOCAB_REQUIRE(dtype == kFloat16 || dtype == kBfloat16, MSB_ERR_ARGUMENT, "dtype must be 2 (float16) or 12 (bfloat16)");
  VOCAB_REQUIRE(FitsIndex(n) && FitsIndex(v) && FitsIndex(h) && v >= 1 && h >= 1, MSB_ERR_SHAPE, "extent out of range");
  VOCAB_REQUIRE(LdOk(ld_data, h) && LdOk(ld_weight, h), MSB_ERR_SHAPE, "stride < width");
  VOCAB_REQUIRE(smooth >= 0.0f && smooth < 1.0f && (smooth == 0.0f || v > 1), MSB_ERR_ARGUMENT,
                "smoothing must lie in [0, 1) and needs two classes");
  if (n == 0) return MSB_OK;
  VOCAB_REQUIRE(loss && lse && data && weight && label, MSB_ERR_ARGUMENT, "null pointer");
  VOCAB_REQUIRE(ElementAligned(data, dtype) && ElementAligned(weight, dtype) && WordAligned(loss, lse, label), MSB_ERR_LAYOUT,
                "operands must be aligned to their elements");
  int rc = PlaceCheck(__func__, loss, lse, data, weight, label, workspace);
  if (rc == MSB_OK) rc = CaptureCheck(__func__, workspace, true, stream);
  if (rc != MSB_OK) return rc;
  return Guarded(__func__, [&] {
    Borrowed st(stream);
    const size_t bytes = static_cast<size_t>(workspace_bytes < 0 ? 0 : workspace_bytes);
    const Tensor<gpu, 1, int32_t> lab = Vec<int32_t>(label, n, &st.s);
    if (dtype == kFloat16) {
      LinearSoftmaxLoss(Vec<float>(loss, n, &st.s), Vec<float>(lse, n, &st.s), Mat<half_t>(data, n, h, ld_data, &st.s),
                        Mat<half_t>(weight, v, h, ld_weight, &st.s), lab, ignore_label, smooth, workspace, bytes);
    } else {
      LinearSoftmaxLoss(Vec<float>(loss, n, &st.s), Vec<float>(lse, n, &st.s),
                        Mat<bf16_t>(data, n, h, ld_data, &st.s),
                        Mat<bf16_t>(weight, v, h, ld_weight, &st.s), lab, ignore_label, smooth, workspace, bytes);
    }
  });
}

int msb_linear_softmax_loss_grad(void *gdata, void *gweight, const void *data, const void *weight, const int32_t *label,
                                 const float *lse, const float *gloss, float scale, int64_t n, int64_t v, int64_t h,
                                 int64_t ld_gdata, int64_t ld_gweight, int64_t ld_data, int64_t ld_weight, int dtype,
                                 int gweight_dtype, int saver, int32_t ignore_label, float smooth, void *workspace,
                                 int64_t workspace_bytes, msb_stream_t stream) {
  VOCAB_REQUIRE(dtype == kFloat16 || dtype == kBfloat16, MSB_ERR_ARGUMENT, "dtype must be 2 (float16) or 12 (bfloat16)");
  VOCAB_REQUIRE(gweight_dtype == dtype || gweight_dtype == kFloat32, MSB_ERR_ARGUMENT,
                "the weight's gradient has the weight's type or float32");
  VOCAB_REQUIRE(saver == 0 || saver == 1, MSB_ERR_ARGUMENT, "saver must be 0 (assign) or 1 (add)");
  VOCAB_REQUIRE(FitsIndex(n) && FitsIndex(v) && FitsIndex(h) && v >= 1 && h >= 1, MSB_ERR_SHAPE, "extent out of range");
  VOCAB_REQUIRE(LdOk(ld_data, h) && LdOk(ld_weight, h) && (gdata == nullptr || LdOk(ld_gdata, h)) &&
                    (gweight == nullptr || LdOk(ld_gweight, h)),
                MSB_ERR_SHAPE, "stride < width");
  VOCAB_REQUIRE(smooth >= 0.0f && smooth < 1.0f && (smooth == 0.0f || v > 1), MSB_ERR_ARGUMENT,
                "smoothing must lie in [0, 1) and needs two classes");
  if (gdata == nullptr && gweight == nullptr) return MSB_OK;
  VOCAB_REQUIRE(n == 0 || (data && weight && label && lse), MSB_ERR_ARGUMENT, "null pointer");
  VOCAB_REQUIRE(ElementAligned(data, dtype) && ElementAligned(weight, dtype) && ElementAligned(gdata, dtype) &&
                    ElementAligned(gweight, gweight_dtype) && WordAligned(label, lse, gloss),
                MSB_ERR_LAYOUT, "operands must be aligned to their elements");
  int rc = PlaceCheck(__func__, gdata, gweight, data, weight, label, lse, gloss, workspace);
  if (rc == MSB_OK) rc = CaptureCheck(__func__, workspace, n > 0, stream);
  if (rc != MSB_OK) return rc;
  return Guarded(__func__, [&] {
    Borrowed st(stream);
    const size_t bytes = static_cast<size_t>(workspace_bytes < 0 ? 0 : workspace_bytes);
    const Tensor<gpu, 1, int32_t> lab = Vec<int32_t>(label, n, &st.s);
    const Tensor<gpu, 1, float> ls = Vec<float>(lse, n, &st.s), gl = Vec<float>(gloss, n, &st.s);
#define VOCAB_LOSS_GRAD(S, T, G)                                                                                     \
  LinearSoftmaxLossGrad<S>(Mat<T>(gdata, n, h, ld_gdata, &st.s), Mat<G>(gweight, v, h, ld_gweight, &st.s),           \
                           Mat<T>(data, n, h, ld_data, &st.s), Mat<T>(weight, v, h, ld_weight, &st.s), lab, ls, gl, \
                           scale, ignore_label, smooth, workspace, bytes)
#define VOCAB_LOSS_GRAD_T(T)                                                \
  if (gweight_dtype == kFloat32) {                                          \
    if (saver == 1) VOCAB_LOSS_GRAD(sv::plusto, T, float);                  \
    else VOCAB_LOSS_GRAD(sv::saveto, T, float);                             \
  } else {                                                                  \
    if (saver == 1) VOCAB_LOSS_GRAD(sv::plusto, T, T);                      \
    else VOCAB_LOSS_GRAD(sv::saveto, T, T);                                 \
  }
    if (dtype == kFloat16) {
      VOCAB_LOSS_GRAD_T(half_t)
    } else {
      VOCAB_LOSS_GRAD_T(bf16_t)
    }
#undef VOCAB_LOSS_GRAD_T
#undef VOCAB_LOSS_GRAD
  });
}

}  // extern "C"
