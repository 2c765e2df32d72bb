#include "rows_map.cuh"

#include <atomic>

namespace smla {

namespace {
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                             const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
}  // namespace

int encode_map(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base, const uint64_t* dims, const uint64_t* strides, const uint32_t* box,
               CUtensorMapL2promotion promotion) {
    static std::atomic<EncodeFn> encode{nullptr};
    if (encode.load() == nullptr) {
        cudaDriverEntryPointQueryResult qres;
        void* fn = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres) != cudaSuccess || fn == nullptr)
            return set_error(SMLA_E_DEVICE, "the driver has no cuTensorMapEncodeTiled");
        encode = (EncodeFn)fn;
    }
    cuuint64_t d[3] = {}, s[2] = {};
    cuuint32_t b[3] = {};
    const cuuint32_t estr[3] = {1, 1, 1};
    for (int i = 0; i < rank; ++i) { d[i] = dims[i]; b[i] = box[i]; }
    for (int i = 0; i + 1 < rank; ++i) s[i] = strides[i];
    const CUresult r = encode.load()(map, type, rank, const_cast<void*>(base), d, s, b, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                     CU_TENSOR_MAP_SWIZZLE_128B, promotion, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : set_error(SMLA_E_DEVICE, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

int rows_tensor_map(const uint8_t* kv, CUtensorMap* map) {
    const uint64_t dims[2] = {ROW_BYTES / 4, (uint64_t)NO_ROW}, strides[1] = {ROW_BYTES};
    const uint32_t box[2] = {32, 1};
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_INT32, 2, kv, dims, strides, box, CU_TENSOR_MAP_L2_PROMOTION_NONE);
}

}  // namespace smla
