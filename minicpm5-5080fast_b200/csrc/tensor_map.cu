// tensor_map.cu -- encoded TMA tensor maps of row-major matrices, cached by address and shape.
#include "tcgen05.cuh"

#include <mutex>
#include <unordered_map>

namespace mcl {

namespace {

// cuTensorMapEncodeTiled through the runtime's driver entry point (no link against libcuda).
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    if (fn == nullptr) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    }
    return fn;
}

// An encoded tensor map depends only on (address, shape, box): a step launched eagerly would
// otherwise pay two driver encodes per GEMM.  Small process-wide cache, cleared when full.
struct MapKey {
    const void* ptr; uint32_t rows, K, pitch, elem, box_k, box_rows, swz;
    bool operator==(const MapKey& o) const {
        return ptr == o.ptr && rows == o.rows && K == o.K && pitch == o.pitch && elem == o.elem && box_k == o.box_k && box_rows == o.box_rows && swz == o.swz;
    }
};
struct MapKeyHash {
    size_t operator()(const MapKey& k) const {
        uint64_t h = 0xCBF29CE484222325ull;
        const uint64_t v[5] = {(uint64_t)(uintptr_t)k.ptr, ((uint64_t)k.rows << 32) | k.K, ((uint64_t)k.box_k << 32) | k.box_rows,
                               ((uint64_t)k.elem << 32) | k.swz, k.pitch};
        for (uint64_t x : v) { h ^= x; h *= 0x100000001B3ull; }
        return (size_t)h;
    }
};
constexpr size_t kMapCacheMax = 4096;

}  // namespace

// Row-major [rows, K] matrix of 1- or 2-byte elements, box = [box_rows x box_k]; out-of-range
// rows / columns read as zero (ragged N, M < Mpad, K tail).
mc_status_t tma_encode_2d(CUtensorMap* map, const void* ptr, uint32_t rows, uint32_t K, uint32_t pitch, uint32_t elem_bytes,
                          uint32_t box_k, uint32_t box_rows, bool swizzle128) {
    EncodeTiledFn fn = encode_fn();
    if (fn == nullptr) {
        set_error("tensor map: cuTensorMapEncodeTiled is not available from this driver");
        return MC_E_CUDA;
    }
    const cuuint64_t dims[2] = {K, rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch * elem_bytes};   // row pitch in bytes (a multiple of 16)
    const cuuint32_t box[2] = {box_k, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    auto encode = [&]() {
        return fn(map, elem_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
                  const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzle128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {      // a host thread's first CUDA call: the runtime gives it its device's context
        int device = 0;
        if (cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) r = encode();
    }
    if (r != CUDA_SUCCESS) {
        set_error("tensor map: cuTensorMapEncodeTiled failed (%d) for rows=%u K=%u", (int)r, rows, K);
        return MC_E_CUDA;
    }
    return MC_OK;
}

mc_status_t tma_map_2d(CUtensorMap* map, const void* ptr, uint32_t rows, uint32_t K, uint32_t pitch, uint32_t elem_bytes,
                       uint32_t box_k, uint32_t box_rows, bool swizzle128) {
    static std::mutex mu;
    static std::unordered_map<MapKey, CUtensorMap, MapKeyHash> cache;
    const MapKey key{ptr, rows, K, pitch, elem_bytes, box_k, box_rows, swizzle128 ? 1u : 0u};
    {
        std::lock_guard<std::mutex> lock(mu);
        auto it = cache.find(key);
        if (it != cache.end()) { *map = it->second; return MC_OK; }
    }
    const mc_status_t s = tma_encode_2d(map, ptr, rows, K, pitch, elem_bytes, box_k, box_rows, swizzle128);
    if (s != MC_OK) return s;
    std::lock_guard<std::mutex> lock(mu);
    if (cache.size() >= kMapCacheMax) cache.clear();
    cache.emplace(key, *map);
    return MC_OK;
}

}  // namespace mcl
