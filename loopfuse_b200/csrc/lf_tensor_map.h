// Tensor maps of the TMA copies: the driver's encoder, and a cached encode for bf16 tensors of up to
// five dimensions.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <stdint.h>

namespace lf {

// The driver's cuTensorMapEncodeTiled; null (with the error recorded) where it has none.
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();

// A bf16 tensor of five dimensions, innermost first and of stride 1, and the box that one copy moves: 64
// columns, in the 128-byte swizzle that the MMA descriptors read. Elements outside are read as zero.
struct TileMapSpec {
  const void* base;
  int64_t dim[5];     // dim[0] = columns
  int64_t stride[4];  // elements between steps of dimensions 1 to 4
  int32_t box[4];     // extent of the box in dimensions 1 to 4
};

// Map of `spec`, from a small cache where it is there (a map depends on nothing but the spec).
int make_map_5d(CUtensorMap* map, const TileMapSpec& spec);

}  // namespace lf
