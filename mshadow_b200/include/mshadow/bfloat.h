/*
 * bfloat16 element type for tensors: mshadow::bfloat::bf16_t, 16 bits holding the upper half of a
 * binary32.  It is a storage type of the function-form operators that take 16-bit tensors
 * (EmbedTake, LinearSoftmaxLoss and their gradients): conversions only, round to nearest even, no
 * arithmetic of its own.  The type tag is the one dmlc/mshadow reserves for it
 * (mshadow/base.h, kBfloat16 = 12).
 */
#ifndef MSHADOW_BFLOAT_H_
#define MSHADOW_BFLOAT_H_

#include <stdint.h>
#include <string.h>

#include "./base.h"

namespace mshadow {
namespace bfloat {

class MSHADOW_ALIGNED(2) bf16_t {
 public:
  uint16_t bits_;

  MSHADOW_XINLINE bf16_t() {}
  MSHADOW_XINLINE explicit bf16_t(const float &value) : bits_(FromFloat(value)) {}
  MSHADOW_XINLINE operator float() const {  // NOLINT(*)
    const uint32_t f = static_cast<uint32_t>(bits_) << 16;
    float r;
    memcpy(&r, &f, sizeof(r));
    return r;
  }
  /*! \brief the value whose bit pattern is `bits` */
  MSHADOW_XINLINE static bf16_t Binary(uint16_t bits) {
    bf16_t r;
    r.bits_ = bits;
    return r;
  }

 private:
  MSHADOW_XINLINE static uint16_t FromFloat(float value) {
    uint32_t f;
    memcpy(&f, &value, sizeof(f));
    if ((f & 0x7fffffffu) > 0x7f800000u) return static_cast<uint16_t>((f >> 16) | 0x0040u);  // NaN stays one
    return static_cast<uint16_t>((f + 0x7fffu + ((f >> 16) & 1u)) >> 16);
  }
};

}  // namespace bfloat

template <>
struct DataType<bfloat::bf16_t> {
  static const int kFlag = kBfloat16;
  static const int kLanes = 1;
};

}  // namespace mshadow
#endif  // MSHADOW_BFLOAT_H_
