// Cached tensor maps of the packed kernels: their boxes span heads and tokens, or the slots of a page.
#include "lf_tensor_map.h"

#include <string.h>

#include <mutex>

#include "lf_common.cuh"

namespace lf {

static int encode_map_5d(CUtensorMap* map, const TileMapSpec& s) {
  const auto fn = get_encode_fn();
  if (!fn) return LF_ERR_CUDA;
  cuuint64_t dims[5], strides[4];
  cuuint32_t box[5] = {64, 0, 0, 0, 0}, estr[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i < 5; ++i) dims[i] = static_cast<cuuint64_t>(s.dim[i]);
  for (int i = 0; i < 4; ++i) {
    box[i + 1] = static_cast<cuuint32_t>(s.box[i]);
    strides[i] = static_cast<cuuint64_t>(s.stride[i]) * 2;
    // (A dimension of extent 1 may carry any stride; keep it a valid multiple of 16 bytes.)
    if (s.stride[i] <= 0 || (strides[i] & 15)) {
      if (dims[i + 1] != 1) return LF_ERR_ALIGNMENT;
      strides[i] = 16 * ((dims[0] * 2 + 15) / 16);
    }
  }
  const CUresult r =
      fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(s.base), dims, strides, box,
         estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_cuda_error(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
    return LF_ERR_CUDA;
  }
  return LF_OK;
}

// Direct-mapped, one mutex, like the cache of the prefill kernels: a miss encodes again, and an entry
// whose buffer was freed refers to nothing.
struct MapEntry {
  bool valid = false;
  TileMapSpec spec;
  CUtensorMap map;
};
constexpr int kMapSlots = 256;
static std::mutex g_map_mutex;
static MapEntry g_maps[kMapSlots];

int make_map_5d(CUtensorMap* map, const TileMapSpec& spec) {
  TileMapSpec key;  // (with the padding zeroed: entries are compared as bytes)
  memset(&key, 0, sizeof(key));
  key.base = spec.base;
  uint64_t h = reinterpret_cast<uintptr_t>(spec.base) * 0x9E3779B97F4A7C15ull;
  for (int i = 0; i < 5; ++i) {
    key.dim[i] = spec.dim[i];
    h = (h ^ static_cast<uint64_t>(spec.dim[i])) * 0xC2B2AE3D27D4EB4Full;
  }
  for (int i = 0; i < 4; ++i) {
    key.stride[i] = spec.stride[i];
    key.box[i] = spec.box[i];
    h = (h ^ static_cast<uint64_t>(spec.stride[i]) ^ static_cast<uint64_t>(spec.box[i]) << 48) *
        0x165667B19E3779F9ull;
  }
  const int slot = static_cast<int>((h >> 32) % kMapSlots);
  {
    std::lock_guard<std::mutex> lock(g_map_mutex);
    const MapEntry& e = g_maps[slot];
    if (e.valid && memcmp(&e.spec, &key, sizeof(key)) == 0) {
      *map = e.map;
      return LF_OK;
    }
  }
  const int rc = encode_map_5d(map, key);
  if (rc != LF_OK) return rc;
  std::lock_guard<std::mutex> lock(g_map_mutex);
  MapEntry& e = g_maps[slot];
  memcpy(&e.spec, &key, sizeof(key));
  e.map = *map;
  e.valid = true;
  return LF_OK;
}

}  // namespace lf
