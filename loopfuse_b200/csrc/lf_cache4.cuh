// The records of a 4-bit cache (include/lf_sm100.h has the format), as the kernels that write and read them see it.
#pragma once

#include "lf_common.cuh"

namespace lf {

template <int D>
struct Record4 {
  static constexpr int kGroups = D / 32;       // groups of 32 columns, each with a scale and a midpoint
  static constexpr int kBytes = LF_RECORD4_BYTES(D);
  static constexpr int kScales = D / 2;        // byte of the first scale
  static constexpr int kMids = D / 2 + D / 16; // byte of the first midpoint
  static constexpr int kKeyPiece = D / 8;      // bytes of one of a key's four pieces
  static constexpr int kValuePiece = D / 16;   // bytes of one of a value's eight pieces
  static constexpr int kAlign = D / 8;         // 16 or 8 bytes: what a copy moves at once
};

inline bool record4_aligned(const void* p, const int64_t (&stride)[3], int D) {
  const int64_t a = D / 8;
  return reinterpret_cast<uintptr_t>(p) % a == 0 && stride[0] % a == 0 && stride[1] % a == 0 && stride[2] % a == 0;
}

}  // namespace lf
