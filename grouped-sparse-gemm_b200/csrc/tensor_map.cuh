// Host side of the TMA descriptors: the driver's encoder and a cache of the maps it made.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <mutex>

#include "common.cuh"

namespace pnv {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                   CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(sym);
  });
  return fn;
}

// Tensor maps are pure functions of (base pointer, extents, box, swizzle).  A serving loop calls with
// the same few operand buffers over and over, so the most recent maps are kept and the driver's
// encoder is only called for a new key.  A map holds no reference to the memory it describes: a
// buffer freed and reallocated at the same address with the same shape yields the same map.
struct MapKey {
  const void* base;
  uint64_t row_bytes, rows, experts;
  uint32_t box_rows, box_inner, kind;   // kind: which function made it; swizzle in the high bits
  bool operator==(const MapKey& o) const {
    return base == o.base && row_bytes == o.row_bytes && rows == o.rows && experts == o.experts &&
           box_rows == o.box_rows && box_inner == o.box_inner && kind == o.kind;
  }
};
constexpr int kMapCacheSize = 64;
struct MapCache {
  std::mutex mu;
  MapKey keys[kMapCacheSize];
  CUtensorMap maps[kMapCacheSize];
  int used = 0, next = 0;
};

template <class Encode>
int cached_map(MapCache& cache, CUtensorMap* out, const MapKey& key, Encode encode) {
  std::lock_guard<std::mutex> lock(cache.mu);
  for (int i = 0; i < cache.used; ++i)
    if (cache.keys[i] == key) { *out = cache.maps[i]; return PNV_OK; }
  if (int rc = encode(out)) return rc;
  const int slot = cache.used < kMapCacheSize ? cache.used++ : (cache.next++ % kMapCacheSize);
  cache.keys[slot] = key;
  cache.maps[slot] = *out;
  return PNV_OK;
}

}  // namespace pnv
