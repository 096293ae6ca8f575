#include "tmap.cuh"

#include <mutex>

namespace moddit {

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn g_encode = nullptr;
static std::once_flag g_once;
static cudaError_t g_lookup_error = cudaSuccess;

static void lookup_encode() {
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult qres;
  g_lookup_error = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
  if (g_lookup_error == cudaSuccess && qres == cudaDriverEntryPointSuccess) g_encode = reinterpret_cast<EncodeFn>(fn);
}

// The descriptor is a pure function of these arguments, and a caller runs the same tensors through the same
// kernels step after step: the last few encodings are kept per host thread (the driver call costs microseconds,
// which is visible once a step is a few milliseconds long).
namespace {
struct CachedMap {
  const void* base;
  int dtype, BH, N, rows, D, box_rows;
  CUtensorMap map;
};
constexpr int kCachedMaps = 16;
thread_local CachedMap t_maps[kCachedMaps];
thread_local int t_maps_used = 0, t_maps_next = 0;
}  // namespace

int make_tmap_rows(CUtensorMap* map, const void* base, int dtype, int BH, int N, int D, int box_rows) {
  return make_tmap_first_rows(map, base, dtype, BH, N, N, D, box_rows);
}

int make_tmap_first_rows(CUtensorMap* map, const void* base, int dtype, int BH, int N, int rows, int D, int box_rows) {
  for (int i = 0; i < t_maps_used; ++i) {
    const CachedMap& c = t_maps[i];
    if (c.base == base && c.dtype == dtype && c.BH == BH && c.N == N && c.rows == rows && c.D == D && c.box_rows == box_rows) {
      *map = c.map;
      return MODDIT_OK;
    }
  }
  std::call_once(g_once, lookup_encode);
  if (!g_encode) return fail(MODDIT_E_CUDA, "cuTensorMapEncodeTiled is not available from the driver (%s)",
                             cudaGetErrorString(g_lookup_error));
  // The driver wants a current context.  A thread that has made no runtime call that needs one (a backward pass runs on a
  // thread of the autograd engine) has none yet; cudaSetDevice on the current device gives it one, also during a capture.
  int dev = 0;
  MODDIT_CHECK_CUDA(cudaGetDevice(&dev));
  MODDIT_CHECK_CUDA(cudaSetDevice(dev));
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(BH)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(N) * D * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapDataType dt = (dtype == MODDIT_BF16) ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult res = g_encode(map, dt, 3, const_cast<void*>(base), dims, strides, box, estr,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (res != CUDA_SUCCESS) return fail(MODDIT_E_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", static_cast<int>(res));
  CachedMap& slot = t_maps[t_maps_next];
  slot = CachedMap{base, dtype, BH, N, rows, D, box_rows, *map};
  t_maps_next = (t_maps_next + 1) % kCachedMaps;
  if (t_maps_used < kCachedMaps) ++t_maps_used;
  return MODDIT_OK;
}

}  // namespace moddit
