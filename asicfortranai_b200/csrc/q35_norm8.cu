// q35_norm8.cu -- RMSNorm with the residual's addition and an 8-bit output with scales:
//   h = x + r                                  (binary32; stored rounded to x's type)
//   y = h * rsqrt(mean(h^2) + eps) * w         (of the unrounded h)
//   scale_g = max |y| of group g / Q,  code = nearest code to y / scale_g
// with groups of 128 elements (the e4m3 product's scales of x) or one group per row.
//
// One CTA per row; the row stays in registers between the sum of squares and the codes, so
// x and r are read once.  Bound by HBM for many rows (2 or 3 element passes in and out plus
// one byte a code) and by latency for one.  A thread holds chunks of V consecutive
// elements, V * sizeof(T) = 16 bytes (one vector load), so a group of 128 is 128 / V
// neighbouring lanes and its maximum a few shuffles.
#include <algorithm>

#include "q35_q8.cuh"

namespace q35 {
namespace {

constexpr int NORM_MAX_DIM = 32768;

struct Norm8Params {
    const void *x, *res;
    void *res_out;
    const float *w;
    uint8_t *q;
    float *scales;
    int64_t ldx, ldr, ldo, ldq;   // elements between rows
    int32_t dim, groups;
    float eps;
    bool vec;                      // rows start on vector boundaries and dim is a multiple of V
};

// the larger of a and b, NaN if either is: a row with a NaN or infinite element gets NaN scales
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T, int V>
__device__ __forceinline__ void load_chunk(const T *p, int i, int dim, bool vec, float (&v)[V]) {
    if (vec) {
        if (i < dim) {
            const uint4 u = *reinterpret_cast<const uint4 *>(p + i);
            const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = to_f32<T>(t[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = 0.0f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = i + j < dim ? to_f32<T>(p[i + j]) : 0.0f;
    }
}

// NC chunks per thread: thread t's chunk c covers elements (c * blockDim + t) * V ...
template <typename T, int CODE, int NC, bool ROW>
__global__ void __launch_bounds__(1024) norm8_kernel(const Norm8Params p) {
    constexpr int V = 16 / sizeof(T);
    constexpr int LANES = Q8_BLOCK / V;       // lanes of a group of 128: 32 (fp32) or 16
    __shared__ float part[32];
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, nw = blockDim.x >> 5;
    const T *x = static_cast<const T *>(p.x) + row * p.ldx;
    const T *r = static_cast<const T *>(p.res) + (p.res ? row * p.ldr : 0);
    T *ro = static_cast<T *>(p.res_out) + (p.res_out ? row * p.ldo : 0);
    uint8_t *q = p.q + row * p.ldq;

    float h[NC][V];
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int i = (c * blockDim.x + t) * V;
        load_chunk<T, V>(x, i, p.dim, p.vec, h[c]);
        if (p.res) {
            float b[V];
            load_chunk<T, V>(r, i, p.dim, p.vec, b);
#pragma unroll
            for (int j = 0; j < V; ++j) h[c][j] += b[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) ss = fmaf(h[c][j], h[c][j], ss);
        if (p.res_out) {
            if (p.vec) {
                if (i < p.dim) {
                    uint4 u;
                    T *o = reinterpret_cast<T *>(&u);
#pragma unroll
                    for (int j = 0; j < V; ++j) o[j] = from_f32<T>(h[c][j]);
                    *reinterpret_cast<uint4 *>(ro + i) = u;
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (i + j < p.dim) ro[i + j] = from_f32<T>(h[c][j]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) part[warp] = ss;
    __syncthreads();
    float tot = lane < nw ? part[lane] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, o);
    const float inv = 1.0f / sqrtf(tot / (float)p.dim + p.eps);

    float amax[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int i = (c * blockDim.x + t) * V;
        amax[c] = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float w = i + j < p.dim ? p.w[i + j] : 0.0f;
            h[c][j] = i + j < p.dim ? h[c][j] * inv * w : 0.0f;
            amax[c] = max_nan(amax[c], fabsf(h[c][j]));
        }
    }
    if (ROW) {
        float m = amax[0];
#pragma unroll
        for (int c = 1; c < NC; ++c) m = max_nan(m, amax[c]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        __syncthreads();
        if (lane == 0) part[warp] = m;
        __syncthreads();
        m = lane < nw ? part[lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
        for (int c = 0; c < NC; ++c) amax[c] = m;
    } else {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) amax[c] = max_nan(amax[c], __shfl_xor_sync(0xffffffffu, amax[c], o));
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int i = (c * blockDim.x + t) * V;
        if (i >= p.dim) continue;
        const float s = __fdiv_rn(amax[c], code_max<CODE>());
        const int g = ROW ? 0 : i / Q8_BLOCK;
        if (ROW ? i == 0 : (i % Q8_BLOCK) == 0) p.scales[row * p.groups + g] = s;
        uint8_t b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) b[j] = s == 0.0f ? 0 : encode8<CODE>(__fdiv_rn(h[c][j], s));
        if (p.vec) {
            if (V == 8) *reinterpret_cast<uint2 *>(q + i) = *reinterpret_cast<const uint2 *>(b);
            else *reinterpret_cast<uint32_t *>(q + i) = *reinterpret_cast<const uint32_t *>(b);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (i + j < p.dim) q[i + j] = b[j];
        }
    }
}

template <typename T, int CODE, bool ROW>
int launch_norm8(const Norm8Params &p, int32_t rows, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int chunks = (int)ceil_div(p.dim, V);
    // (V = 8: 32768 elements are 4096 chunks; only fp32 rows above 16384 reach 8 a thread)
    const int nc = chunks <= 1024 ? 1 : chunks <= 2048 ? 2 : chunks <= 4096 ? 4 : 8;
    const int threads = (int)round_up(ceil_div(chunks, nc), 32);
    switch (nc) {
    case 1: norm8_kernel<T, CODE, 1, ROW><<<rows, threads, 0, s>>>(p); break;
    case 2: norm8_kernel<T, CODE, 2, ROW><<<rows, threads, 0, s>>>(p); break;
    case 4: norm8_kernel<T, CODE, 4, ROW><<<rows, threads, 0, s>>>(p); break;
    default:
        if constexpr (V == 4) norm8_kernel<T, CODE, 8, ROW><<<rows, threads, 0, s>>>(p);
        break;
    }
    Q35_CUDA_TRY(cudaGetLastError());
    return Q35_OK;
}

template <typename T>
int launch_norm8(const Norm8Params &p, int code, bool row, int32_t rows, cudaStream_t s) {
    if (code == Q35_CODE_INT8)
        return row ? launch_norm8<T, Q35_CODE_INT8, true>(p, rows, s) : launch_norm8<T, Q35_CODE_INT8, false>(p, rows, s);
    return row ? launch_norm8<T, Q35_CODE_E4M3, true>(p, rows, s) : launch_norm8<T, Q35_CODE_E4M3, false>(p, rows, s);
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int q35_rms_norm_quant_dev(q35_ctx ctx, int dtype, const void *x, int64_t ldx, const void *residual,
                                      int64_t ldr, void *residual_out, int64_t ldo, const float *weight, float eps,
                                      int32_t rows, int32_t dim, int code, int32_t group, void *q, int64_t ldq,
                                      float *scales) {
    if (!ctx) return set_error(Q35_ERR_INVALID, "rms_norm_quant: ctx is NULL");
    int st = check_dtype(dtype);
    if (!st) st = check_code(code);
    if (st) return st;
    if (rows < 0) return set_error(Q35_ERR_INVALID, "rms_norm_quant: negative row count");
    if (dim < 1 || dim > NORM_MAX_DIM) return set_error(Q35_ERR_INVALID, "rms_norm_quant: dim must be in [1,32768]");
    if (group != 0 && group != Q8_BLOCK) return set_error(Q35_ERR_INVALID, "rms_norm_quant: group must be 128 or 0 (the row)");
    if (!(eps >= 0.0f)) return set_error(Q35_ERR_INVALID, "rms_norm_quant: eps must not be negative");
    if (rows == 0) return Q35_OK;
    if (!x || !weight || !q || !scales) return set_error(Q35_ERR_INVALID, "rms_norm_quant: NULL argument");
    if (ldx < dim || ldq < dim || (residual && ldr < dim) || (residual_out && ldo < dim))
        return set_error(Q35_ERR_INVALID, "rms_norm_quant: a row stride is below dim");
    const size_t es = dtype_size(dtype);
    if (!aligned_to(x, es) || !aligned_to(residual, es) || !aligned_to(residual_out, es) || !aligned_to(weight, 4) ||
        !aligned_to(scales, 4))
        return set_error(Q35_ERR_INVALID, "rms_norm_quant: a pointer is not aligned to its elements");
    // residual_out may be x or residual themselves (each thread reads its elements before it
    // writes them); a shifted overlap would read sums
    if (residual_out) {
        auto overlaps = [&](const void *p, int64_t ld) {
            const char *a = static_cast<const char *>(p), *o = static_cast<const char *>(residual_out);
            const size_t na = ((size_t)(rows - 1) * ld + dim) * es, no = ((size_t)(rows - 1) * ldo + dim) * es;
            return p && a < o + no && o < a + na && !(a == o && ld == ldo);
        };
        if (overlaps(x, ldx) || overlaps(residual, ldr))
            return set_error(Q35_ERR_INVALID, "rms_norm_quant: residual_out partly overlaps an input");
    }
    DeviceGuard g(ctx->device);
    Norm8Params p;
    p.x = x; p.res = residual; p.res_out = residual_out; p.w = weight;
    p.q = static_cast<uint8_t *>(q);
    p.scales = scales;
    p.ldx = ldx; p.ldr = ldr; p.ldo = ldo; p.ldq = ldq;
    p.dim = dim;
    p.groups = group ? (int32_t)ceil_div(dim, Q8_BLOCK) : 1;
    p.eps = eps;
    const int V = (int)(16 / es);
    auto vec_ok = [&](const void *ptr, int64_t ld) { return !ptr || (aligned_to(ptr, 16) && ld % V == 0); };
    p.vec = dim % V == 0 && vec_ok(x, ldx) && vec_ok(residual, ldr) && vec_ok(residual_out, ldo) &&
            aligned_to(q, V) && ldq % V == 0;
    switch (dtype) {
    case Q35_DT_F32: return launch_norm8<float>(p, code, group == 0, rows, ctx->stream);
    case Q35_DT_BF16: return launch_norm8<__nv_bfloat16>(p, code, group == 0, rows, ctx->stream);
    default: return launch_norm8<__half>(p, code, group == 0, rows, ctx->stream);
    }
}
