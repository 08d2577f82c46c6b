// Tensor maps for the tensor-core kernels (host side of umma.cuh).
#include "umma.cuh"

namespace fl {

namespace {
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                              CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once (concurrent first calls store the same value).
EncodeFn encoder() {
    static std::atomic<void*> fn{nullptr};
    void* f = fn.load(std::memory_order_acquire);
    if (f == nullptr) {
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault,
                                             &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            return nullptr;
        fn.store(f, std::memory_order_release);
    }
    return reinterpret_cast<EncodeFn>(f);
}
}  // namespace

int make_tensor_map(CUtensorMap* map, CUtensorMapDataType type, int elem_bytes, const void* base,
                    int64_t inner, int64_t outer, int64_t ld, int box_inner, int box_outer) {
    EncodeFn encode = encoder();
    if (encode == nullptr) {
        set_error("cuTensorMapEncodeTiled is not available in this driver");
        return FL_ERR_CUDA;
    }
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * elem_bytes};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_outer)};
    const cuuint32_t one[2] = {1, 1};
    auto attempt = [&] {
        return encode(map, type, 2, const_cast<void*>(base), dims, strides, box, one,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = attempt();
    if (r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) {
        // a host thread that has made no runtime call yet has a device but no context
        int dev = 0;
        FL_CUDA(cudaGetDevice(&dev));
        FL_CUDA(cudaSetDevice(dev));
        r = attempt();
    }
    if (r != CUDA_SUCCESS) {
        set_error("tensor map of (%lld, %lld), row stride %lld, refused (driver error %d)",
                  (long long)outer, (long long)inner, (long long)ld, (int)r);
        return FL_ERR_CUDA;
    }
    return FL_OK;
}

}  // namespace fl
