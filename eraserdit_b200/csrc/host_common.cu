#include "host_common.h"

#include <mutex>

#include "../../include/eraserdit_b200.h"

namespace erd {

namespace {
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
    }
  });
  return fn;
}
}  // namespace

int check_device_sm100() {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  int major = 0, minor = 0;
  e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  e = cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  return (major == 10 && minor == 0) ? kErrOk : kErrUnsupportedDevice;
}

int encode_tensor_map(CUtensorMap* map, CUtensorMapDataType dtype, uint32_t rank, void* base,
                      const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box,
                      CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return kErrTensorMap;
  cuuint32_t elem_strides[5] = {1, 1, 1, 1, 1};
  auto encode = [&] {
    return fn(map, dtype, rank, base, reinterpret_cast<const cuuint64_t*>(dims),
              reinterpret_cast<const cuuint64_t*>(strides_bytes),
              reinterpret_cast<const cuuint32_t*>(box), elem_strides,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {
    // A host thread whose first CUDA call this is: the driver wants the context that
    // the runtime binds to a thread only with its first launch or device choice.
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess)
      return kErrTensorMap;
    r = encode();
  }
  return r == CUDA_SUCCESS ? kErrOk : kErrTensorMap;
}

}  // namespace erd

extern "C" int erd_abi_version(void) { return ERD_ABI_VERSION; }

extern "C" const char* erd_error_string(int code) {
  switch (code) {
    case erd::kErrOk: return "ok";
    case erd::kErrNullPointer: return "null pointer argument";
    case erd::kErrBadShape: return "unsupported or inconsistent shape";
    case erd::kErrMisaligned: return "pointer or stride not 16-byte aligned";
    case erd::kErrUnsupportedDevice: return "current device is not sm_100 (B200)";
    case erd::kErrTensorMap: return "tensor map encoding failed";
    case erd::kErrTooLarge: return "size exceeds the entry point's limit";
    default: break;
  }
  if (code > 0) return cudaGetErrorString(static_cast<cudaError_t>(code));
  return "unknown error";
}
