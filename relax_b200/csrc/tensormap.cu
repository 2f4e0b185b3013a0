#include "tensormap.h"

#include <cstring>
#include <mutex>

namespace rb200 {
namespace {
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);
EncodeFn g_encode = nullptr;
std::once_flag g_once;
}  // namespace

static int resolve_encode() {
  std::call_once(g_once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<EncodeFn>(fn);
  });
  RB200_CHECK(g_encode != nullptr, "cuTensorMapEncodeTiled is not available from this driver");
  return 0;
}

namespace {
// Encoding a tensor map costs a driver call of a microsecond or two; a serving loop asks for the
// same few maps (same buffers, same shapes) on every step.  Small per-thread cache, keyed by
// everything the encoding depends on.
struct MapKey {
  const void* base;
  int dtype, rank, swizzle, promotion;
  unsigned long long dims[5], strides[4];
  unsigned box[5];
  bool operator==(const MapKey& o) const { return memcmp(this, &o, sizeof(MapKey)) == 0; }
};
struct MapEntry {
  MapKey key;
  CUtensorMap map;
  bool valid;
};
constexpr int kMapCacheSlots = 256;
thread_local MapEntry t_map_cache[kMapCacheSlots];
unsigned hash_key(const MapKey& k) {
  const unsigned char* b = reinterpret_cast<const unsigned char*>(&k);
  unsigned h = 2166136261u;
  for (size_t i = 0; i < sizeof(MapKey); ++i) h = (h ^ b[i]) * 16777619u;
  return h;
}
}  // namespace

int make_tensor_map(CUtensorMap* out, const void* base, CUtensorMapDataType dtype, int rank,
                    const unsigned long long* dims, const unsigned long long* strides_bytes,
                    const unsigned* box, CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion) {
  RB200_CHECK(rank >= 1 && rank <= 5, "tensor map rank %d out of range", rank);
  MapKey key;
  memset(&key, 0, sizeof(key));
  key.base = base;
  key.dtype = (int)dtype;
  key.rank = rank;
  key.swizzle = (int)swizzle;
  key.promotion = (int)promotion;
  for (int i = 0; i < rank; ++i) {
    key.dims[i] = dims[i];
    key.box[i] = box[i];
    if (i + 1 < rank) key.strides[i] = strides_bytes[i];
  }
  MapEntry& slot = t_map_cache[hash_key(key) % kMapCacheSlots];
  if (slot.valid && slot.key == key) {
    *out = slot.map;
    return 0;
  }
  if (resolve_encode() != 0) return -1;
  RB200_CHECK((reinterpret_cast<uintptr_t>(base) & 15u) == 0, "tensor map needs a 16-byte aligned base");
  cuuint64_t d[5];
  cuuint64_t st[4];
  cuuint32_t bx[5];
  cuuint32_t es[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = dims[i];
    bx[i] = box[i];
    es[i] = 1;
    if (i + 1 < rank) {
      RB200_CHECK(strides_bytes[i] % 16 == 0, "tensor map pitch %llu is not a multiple of 16", strides_bytes[i]);
      st[i] = strides_bytes[i];
    }
  }
  CUresult r = g_encode(out, dtype, (cuuint32_t)rank, const_cast<void*>(base), d, st, bx, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, promotion,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RB200_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  slot.key = key;
  slot.map = *out;
  slot.valid = true;
  return 0;
}

int make_tensor_map_2d(CUtensorMap* out, const void* base, CUtensorMapDataType dtype,
                       unsigned long long dim0, unsigned long long dim1,
                       unsigned long long stride1_bytes, unsigned box0, unsigned box1,
                       CUtensorMapSwizzle swizzle, CUtensorMapL2promotion promotion) {
  const unsigned long long dims[2] = {dim0, dim1};
  const unsigned long long strides[1] = {stride1_bytes};
  const unsigned box[2] = {box0, box1};
  return make_tensor_map(out, base, dtype, 2, dims, strides, box, swizzle, promotion);
}
}  // namespace rb200
