/*
 * The vocabulary operators as a C++ user of the headers calls them: Tensor handles, a Stream, element
 * types as template arguments.  Built into its own shared library by mshadow_b200/build.py and driven by
 * tests/test_vocab_table.py with device pointers; returns 0, or the number of the step that failed.
 */
#include <mshadow/tensor.h>

using namespace mshadow;  // NOLINT(*)
typedef mshadow::bfloat::bf16_t bf16;

template <typename DType>
static int Step(DType *table, int32_t *tokens, int32_t *label, DType *gtable, DType *hidden, DType *ghidden, float *loss,
                float *lse, int n, int v, int h, float scale) {
  Stream<gpu> *stream = NewStream<gpu>(false, false);
  Tensor<gpu, 2, DType> t(table, Shape2(v, h), stream), gt(gtable, Shape2(v, h), stream);
  Tensor<gpu, 2, DType> x(hidden, Shape2(n, h), stream), gx(ghidden, Shape2(n, h), stream);
  Tensor<gpu, 1, int32_t> tok(tokens, Shape1(n), stream), lab(label, Shape1(n), stream);
  Tensor<gpu, 1, float> l(loss, Shape1(n), stream), s(lse, Shape1(n), stream), ones;
  EmbedTake(x, t, tok, 2.0f);
  LinearSoftmaxLoss(l, s, x, t, lab);
  LinearSoftmaxLossGrad<sv::saveto>(gx, gt, x, t, lab, s, ones, scale);
  EmbedTakeGrad<sv::plusto>(gt, gx, tok, 2.0f);
  stream->Wait();
  int failed = 0;
  try {  // shapes that do not agree are refused on the host
    Tensor<gpu, 2, DType> narrow(hidden, Shape2(n, h - 1), stream);
    EmbedTake(narrow, t, tok);
    failed = 1;
  } catch (const dmlc::Error &) {
  }
  try {
    LinearSoftmaxLoss(l, s.Slice(0, n - 1), x, t, lab);
    failed = 2;
  } catch (const dmlc::Error &) {
  }
  try {
    LinearSoftmaxLoss(l, s, x, t, lab, -1, 1.0f);
    failed = 3;
  } catch (const dmlc::Error &) {
  }
  try {
    LinearSoftmaxLossGrad<sv::saveto>(gx, gt, x, t, lab, s, ones, scale, -1, 0.0f, lse, 64);  // workspace too small
    failed = 4;
  } catch (const dmlc::Error &) {
  }
  DeleteStream(stream);
  return failed;
}

extern "C" int msb_vocab_step_f16(void *table, int32_t *tokens, int32_t *label, void *gtable, void *hidden, void *ghidden,
                                  float *loss, float *lse, int n, int v, int h, float scale) {
  typedef mshadow::half::half_t T;
  return Step(static_cast<T *>(table), tokens, label, static_cast<T *>(gtable), static_cast<T *>(hidden),
              static_cast<T *>(ghidden), loss, lse, n, v, h, scale);
}
extern "C" int msb_vocab_step_bf16(void *table, int32_t *tokens, int32_t *label, void *gtable, void *hidden, void *ghidden,
                                   float *loss, float *lse, int n, int v, int h, float scale) {
  return Step(static_cast<bf16 *>(table), tokens, label, static_cast<bf16 *>(gtable), static_cast<bf16 *>(hidden),
              static_cast<bf16 *>(ghidden), loss, lse, n, v, h, scale);
}

/*! \brief host conversions of the element type: bits of the rounded value, or the value of bits */
extern "C" int msb_bf16_round(const float *in, uint16_t *bits, float *back, int n) {
  for (int i = 0; i < n; ++i) {
    const bf16 b(in[i]);
    bits[i] = b.bits_;
    back[i] = static_cast<float>(b);
  }
  return DataType<bf16>::kFlag;
}
