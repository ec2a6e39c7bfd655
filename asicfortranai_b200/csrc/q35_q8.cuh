// q35_q8.cuh -- what the 8-bit operators share (q35_norm8.cu, q35_fp8.cu, q35_kv8.cu,
// q35_sample_filtered.cu): element types, the two 8-bit codes and their rounding,
// argument checks.
//
// A code stands for code * scale, with the largest magnitude of the block at +-Q (127 for int8, 448 for
// e4m3).  encode8 rounds a binary32 quotient to the nearest code, ties to even, clamped to [-Q, Q]; how
// the scale and the quotient are formed is each operator's own: the append's are IEEE operations that a plain program
// repeats bit for bit (q35_kv8.cu), the norm's have other roundings than a division (q35_norm8.cu), so a
// value next to a rounding boundary may get the code on its other side.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "q35_internal.cuh"

namespace q35 {

constexpr int Q8_BLOCK = 128;   // elements per scale along a row (norm output, e4m3 product)

inline size_t dtype_size(int dtype) { return dtype == Q35_DT_F32 ? 4 : 2; }
inline int check_dtype(int dtype) {
    if (dtype != Q35_DT_F32 && dtype != Q35_DT_BF16 && dtype != Q35_DT_F16)
        return set_error(Q35_ERR_INVALID, "unknown element type");
    return Q35_OK;
}
inline int check_code(int code) {
    if (code != Q35_CODE_INT8 && code != Q35_CODE_E4M3) return set_error(Q35_ERR_INVALID, "unknown 8-bit code");
    return Q35_OK;
}
inline bool aligned_to(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

#ifdef __CUDACC__
// Launches with programmatic dependent launch (and a cluster of `cluster` CTAs along x when
// that is above 1): the grid may begin while the previous kernel of the stream ends, so a
// kernel launched this way calls dependency_wait() before it touches global memory.
template <typename... P, typename... A>
inline cudaError_t launch_dependent(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t s, int cluster,
                                    A... args) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
}
__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dependency_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// two floats to the packed pair of a 16-bit type (low half first)
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

template <int CODE> __device__ __forceinline__ constexpr float code_max() {
    return CODE == Q35_CODE_INT8 ? 127.0f : 448.0f;
}

// the code nearest to v (ties to even, clamped); NaN gives 0 (int8) or NaN (e4m3)
template <int CODE> __device__ __forceinline__ uint8_t encode8(float v) {
    if (CODE == Q35_CODE_INT8) {
        const int q = __float2int_rn(v);               // saturates; NaN gives 0
        return (uint8_t)(int8_t)max(-127, min(127, q));
    }
    return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
// four of them, the first in the lowest byte
template <int CODE> __device__ __forceinline__ uint32_t encode8x4(float a, float b, float c, float d) {
    if (CODE == Q35_CODE_INT8)
        return encode8<CODE>(a) | ((uint32_t)encode8<CODE>(b) << 8) | ((uint32_t)encode8<CODE>(c) << 16) |
               ((uint32_t)encode8<CODE>(d) << 24);
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
template <int CODE> __device__ __forceinline__ float decode8(uint8_t c) {
    if (CODE == Q35_CODE_INT8) return (float)(int8_t)c;
    const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
    return __half2float(__half(h));
}
#endif

}  // namespace q35
