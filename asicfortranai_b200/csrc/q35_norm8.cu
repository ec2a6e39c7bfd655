// q35_norm8.cu -- RMSNorm with the residual's addition and an 8-bit output with scales:
//   h = x + r                                  (binary32; stored rounded to x's type)
//   y = h * rsqrt(mean(h^2) + eps) * w         (of the unrounded h)
//   scale_g = max |y| of group g / Q,  code = nearest code to y / scale_g
// with groups of 128 elements (the e4m3 product's scales of x) or one group per row.
//
// A row at a time per CTA; it stays in registers between the sum of squares and the codes, so
// x and r are read once.  Bound by HBM for many rows (2 or 3 element passes in and out plus
// one byte a code) and by latency for one.  A thread holds chunks of V consecutive
// elements, V * sizeof(T) = 16 bytes (one vector load), so a group of 128 is 128 / V
// neighbouring lanes and its maximum a few shuffles.
//
// 1/rms is split into a power of two and a factor f in [1, 2): y' = h 2^e w has one rounding,
// the codes are round(y' (Q / max |y'|)) -- f cancels -- and f enters the scale alone, so a code
// sees fewer roundings than y / scale has, and no division per element.
//
// A row with an element that is no number, or with squares next to the ends of binary32's range, takes a
// path of its own (far_row): NaN scales in every group, or the row's codes with the sum of squares taken
// once more behind a power of two.
//
// Measured: 4099 rows of 5120 in bf16 with the residual and its sum 28 us (147 MB, 5.2 TB/s; a
// copy reaches 6.5); one row of 8192 6.5 us a call back to back, which is the host's time.
#include <algorithm>
#include <cfloat>
#include <cstring>

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
    int32_t rows, dim, groups;
    float eps, inv_dim;
    bool vec;                      // rows start on vector boundaries and dim is a multiple of V
};

// the larger of a and b, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// V consecutive elements as they stand in memory
template <typename T, int V> struct Chunk { T e[V]; };
template <typename T, int V> __device__ __forceinline__ Chunk<T, V> chunk_of(uint4 u) {
    Chunk<T, V> c;
    memcpy(&c, &u, 16);
    return c;
}
template <typename T, int V> __device__ __forceinline__ uint4 words_of(const Chunk<T, V> &c) {
    uint4 u;
    memcpy(&u, &c, 16);
    return u;
}

// VEC: rows start on 16-byte boundaries and dim is a multiple of V.  The words are taken apart
// where they are used: doing it here would wait for the load here.  (volatile: a load issued
// ahead of a barrier is not moved down to its use)
template <typename T, int V, bool VEC>
__device__ __forceinline__ uint4 load_chunk(const T *p, int i, int dim) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (VEC) {
        if (i < dim)
            asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p + i));
    } else {
        Chunk<T, V> c;
#pragma unroll
        for (int j = 0; j < V; ++j) c.e[j] = i + j < dim ? p[i + j] : from_f32<T>(0.0f);
        u = words_of<T, V>(c);
    }
    return u;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// One row, read from memory again in every pass: the largest element, then the sum of squares behind the
// power of two that brings it next to 1 (eps with it), then codes by groups of 128 elements, a warp each.
// All threads of the CTA call it, behind the loop over the rows (within it, in line or as a call, it cost
// that loop registers: 30.5 us at 4099 rows of 5120 in bf16, 28.4 here, 27.5 without it).
template <typename T, int CODE, bool ROW>
__device__ __forceinline__ void far_row(const Norm8Params &p, int64_t row, float (*part)[32]) {
    constexpr float Q = code_max<CODE>();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, nw = blockDim.x >> 5;
    const T *x = static_cast<const T *>(p.x) + row * p.ldx;
    const T *r = static_cast<const T *>(p.res) + (p.res ? row * p.ldr : 0);
    T *ro = static_cast<T *>(p.res_out) + (p.res_out ? row * p.ldo : 0);
    uint8_t *q = p.q + row * p.ldq;
    auto sum = [&](int i) { return p.res ? to_f32<T>(x[i]) + to_f32<T>(r[i]) : to_f32<T>(x[i]); };
    auto over_cta = [&](float v, int slot, auto join) {
        v = join(v);
        __syncthreads();
        if (lane == 0) part[slot][warp] = v;
        __syncthreads();
        return join(lane < nw ? part[slot][lane] : 0.0f);
    };
    float m = 0.0f, ss = 0.0f, top = 0.0f;
#pragma unroll 1
    for (int i = t; i < p.dim; i += blockDim.x) m = max_nan(m, fabsf(sum(i)));
    m = over_cta(m, 0, warp_max_nan);
    const int e = max(-126, min(126, (int)(__float_as_uint(fmaxf(m, sqrtf(p.eps))) >> 23) - 127));
    const float by = m <= FLT_MAX ? __uint_as_float((uint32_t)(127 - e) << 23) : NAN;   // (NaN for the whole row)
#pragma unroll 1
    for (int i = t; i < p.dim; i += blockDim.x) {
        const float y = sum(i) * by;
        ss = fmaf(y, y, ss);
    }
    ss = over_cta(ss, 1, warp_sum);
    const float f = rsqrtf(fmaf(ss, p.inv_dim, p.eps * by * by));       // 1/rms = by f
    if (ROW) {
#pragma unroll 1
        for (int i = t; i < p.dim; i += blockDim.x) top = max_nan(top, fabsf(sum(i) * by * p.w[i]));
        top = over_cta(top, 0, warp_max_nan);
    }
#pragma unroll 1
    for (int g = warp; g * Q8_BLOCK < p.dim; g += nw) {
        float y[Q8_BLOCK / 32], amax = top;
#pragma unroll
        for (int j = 0; j < Q8_BLOCK / 32; ++j) {
            const int i = g * Q8_BLOCK + 32 * j + lane;
            y[j] = 0.0f;
            if (i < p.dim) {
                const float h = sum(i);
                y[j] = h * by * p.w[i];
                if (p.res_out) ro[i] = from_f32<T>(h);
            }
            if (!ROW) amax = max_nan(amax, fabsf(y[j]));
        }
        if (!ROW) amax = warp_max_nan(amax);
        if (lane == 0 && (!ROW || g == 0)) p.scales[row * p.groups + g] = amax * f * (1.0f / Q);
#pragma unroll
        for (int j = 0; j < Q8_BLOCK / 32; ++j) {
            const int i = g * Q8_BLOCK + 32 * j + lane;
            if (i < p.dim) q[i] = encode8<CODE>(amax > 0.0f ? __fdiv_rn(y[j], __fdiv_rn(amax, Q)) : amax);
        }
    }
}

// NC chunks per thread: thread t's chunk c covers elements (c * blockDim + t) * V ...  A CTA takes
// rows blockIdx, blockIdx + gridDim, ...; the next row's loads are issued before this row's
// barrier, so that memory is busy through the reductions.  MT: the largest CTA, MB: CTAs an
// SM should hold.  WS: the weights stand in shared memory (CTAs of several rows), four floats of
// every chunk in a plane.
template <typename T, int CODE, int NC, bool ROW, bool VEC, bool WS, int MT, int MB>
__global__ void __launch_bounds__(MT, MB) norm8_kernel(const __grid_constant__ Norm8Params p) {
    constexpr int V = 16 / sizeof(T);
    constexpr int LANES = Q8_BLOCK / V;       // lanes of a group of 128: 32 (fp32) or 16
    constexpr float Q = code_max<CODE>();
    extern __shared__ float4 weights[];
    __shared__ float part[2][2][32];          // (by the row's parity: a row's values outlive one barrier)
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, nw = blockDim.x >> 5;
    dependency_trigger();
    dependency_wait();

    uint4 nx[NC], nr[NC];
    auto fetch = [&](int64_t row) {
        const T *x = static_cast<const T *>(p.x) + row * p.ldx;
        const T *r = static_cast<const T *>(p.res) + (p.res ? row * p.ldr : 0);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * blockDim.x + t) * V;
            nx[c] = load_chunk<T, V, VEC>(x, i, p.dim);
            if (p.res) nr[c] = load_chunk<T, V, VEC>(r, i, p.dim);
        }
    };
    int64_t row = blockIdx.x;
    if (row < p.rows) fetch(row);
    const int chunks = p.dim / V;
    if (WS) {                                 // (each thread reads back what it wrote)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int ch = c * blockDim.x + t;
#pragma unroll
            for (int j = 0; j < V / 4; ++j)
                if (ch < chunks) weights[j * chunks + ch] = *reinterpret_cast<const float4 *>(p.w + ch * V + 4 * j);
        }
    }
    bool any_far = false;
    for (int par = 0; row < p.rows; par ^= 1) {
        float h[NC][V];
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const Chunk<T, V> x = chunk_of<T, V>(nx[c]);
#pragma unroll
            for (int j = 0; j < V; ++j) h[c][j] = to_f32<T>(x.e[j]);
            if (p.res) {
                const Chunk<T, V> r = chunk_of<T, V>(nr[c]);
#pragma unroll
                for (int j = 0; j < V; ++j) h[c][j] += to_f32<T>(r.e[j]);
            }
#pragma unroll
            for (int j = 0; j < V; ++j) ss = fmaf(h[c][j], h[c][j], ss);
        }
        const int64_t next = row + gridDim.x;
        if (next < p.rows) fetch(next);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane == 0) part[par][0][warp] = ss;
        __syncthreads();
        float tot = lane < nw ? part[par][0][lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) tot += __shfl_xor_sync(0xffffffffu, tot, o);
        const float mean = fmaf(tot, p.inv_dim, p.eps);
        // a row for far_row: marked in its first scale; what else is written of it here is written again
        const bool far = !(tot < INFINITY) || mean < 0x1p-100f;
        any_far |= far;
        if (p.res_out && !far) {              // (not before: far_row reads the inputs, which this may be)
            T *ro = static_cast<T *>(p.res_out) + row * p.ldo;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int i = (c * blockDim.x + t) * V;
                Chunk<T, V> o;
#pragma unroll
                for (int j = 0; j < V; ++j) o.e[j] = from_f32<T>(h[c][j]);
                if (VEC) {
                    if (i < p.dim) *reinterpret_cast<uint4 *>(ro + i) = words_of<T, V>(o);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (i + j < p.dim) ro[i + j] = o.e[j];
                }
            }
        }
        const float inv = rsqrtf(mean);      // within 2 ulp
        const float pow2 = __uint_as_float(__float_as_uint(inv) & 0x7f800000u);
        const float f = __uint_as_float((__float_as_uint(inv) & 0x007fffffu) | 0x3f800000u);

        float amax[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * blockDim.x + t) * V;
            float w[V];
            if (VEC) {
                // (chunks behind the row's end are zeros times zeros)
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (i < p.dim)
                        u = WS ? weights[(j / 4) * chunks + c * blockDim.x + t] : *reinterpret_cast<const float4 *>(p.w + i + j);
                    w[j] = u.x; w[j + 1] = u.y; w[j + 2] = u.z; w[j + 3] = u.w;
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) w[j] = i + j < p.dim ? p.w[i + j] : 0.0f;
            }
            amax[c] = 0.0f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[c][j] = VEC || i + j < p.dim ? h[c][j] * pow2 * w[j] : 0.0f;
                amax[c] = max_nan(amax[c], fabsf(h[c][j]));
            }
        }
        if (ROW) {
            float m = amax[0];
#pragma unroll
            for (int c = 1; c < NC; ++c) m = max_nan(m, amax[c]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (lane == 0) part[par][1][warp] = m;
            __syncthreads();
            m = lane < nw ? part[par][1][lane] : 0.0f;
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
        uint8_t *q = p.q + row * p.ldq;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * blockDim.x + t) * V;
            if (i >= p.dim) continue;
            const int g = ROW ? 0 : i / Q8_BLOCK;
            if (ROW ? i == 0 : (i % Q8_BLOCK) == 0) p.scales[row * p.groups + g] = far ? -1.0f : amax[c] * f * (1.0f / Q);
            uint32_t b[V / 4];
            if (amax[c] < 1e-30f) {                    // Q / amax would overflow (0: codes 0)
                const float s = __fdiv_rn(amax[c], Q);
                auto code = [&](float v) { return s == 0.0f ? 0.0f : __fdiv_rn(v, s); };
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    b[j / 4] = encode8x4<CODE>(code(h[c][j]), code(h[c][j + 1]), code(h[c][j + 2]), code(h[c][j + 3]));
            } else {
                const float r = __fdiv_rn(Q, amax[c]);
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    b[j / 4] = encode8x4<CODE>(h[c][j] * r, h[c][j + 1] * r, h[c][j + 2] * r, h[c][j + 3] * r);
            }
            if (VEC) {
                if (V == 8) *reinterpret_cast<uint2 *>(q + i) = make_uint2(b[0], b[V / 4 - 1]);
                else *reinterpret_cast<uint32_t *>(q + i) = b[0];
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (i + j < p.dim) q[i + j] = (uint8_t)(b[j / 4] >> (8 * (j & 3)));
            }
        }
        row = next;
    }
    if (any_far) {
        __syncthreads();                      // (the marks of thread 0)
        for (row = blockIdx.x; row < p.rows; row += gridDim.x)
            if (p.scales[row * p.groups] == -1.0f) far_row<T, CODE, ROW>(p, row, part[0]);
    }
}

template <typename T, int CODE, bool ROW, bool VEC>
int launch_norm8(const Norm8Params &p, cudaStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int chunks = (int)ceil_div(p.dim, V);
    // one row per CTA and as many threads as there are chunks while an SM has one row at most
    // (latency); else persistent CTAs of up to 512 threads with one chunk or more each
    const bool few = p.rows <= 148;
    const int most = few ? 1024 : 512;
    int nc = chunks <= most ? 1 : chunks <= 2 * most ? 2 : 4;
    if (chunks > 4096) nc = 8;                 // (fp32 rows above 16384)
    const int threads = (int)round_up(ceil_div(chunks, nc), 32);
    auto kern = norm8_kernel<T, CODE, 1, ROW, VEC, false, 1024, 1>;
    if (few || threads > 512) {
        if (nc == 2) kern = norm8_kernel<T, CODE, 2, ROW, VEC, false, 1024, 1>;
        if (nc == 4) kern = norm8_kernel<T, CODE, 4, ROW, VEC, false, 1024, 1>;
        if constexpr (V == 4)
            if (nc == 8) kern = norm8_kernel<T, CODE, 8, ROW, VEC, false, 1024, 1>;
        const int grid = few ? p.rows : std::min(p.rows, 148);
        Q35_CUDA_TRY(launch_dependent(kern, dim3((unsigned)grid), threads, 0, s, 1, p));
        return Q35_OK;
    }
    kern = nc == 1   ? norm8_kernel<T, CODE, 1, ROW, VEC, VEC, 512, 3>
           : nc == 2 ? norm8_kernel<T, CODE, 2, ROW, VEC, VEC, 512, 2>
                     : norm8_kernel<T, CODE, 4, ROW, VEC, VEC, 512, 1>;
    const size_t smem = VEC ? (size_t)p.dim * 4 : 0;
    if (smem > 48 * 1024) {
        // the limit is the function's, for every call of the process: the largest row of this branch, once
        static bool configured[64] = {};
        int dev = 0;
        Q35_CUDA_TRY(cudaGetDevice(&dev));
        if (dev < 0 || dev >= 64 || !configured[dev]) {
            Q35_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * 512 * V * 4));
            if (dev >= 0 && dev < 64) configured[dev] = true;
        }
    }
    int per = 0;                                   // resident CTAs per SM
    Q35_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, threads, smem));
    const int grid = (int)std::min<int64_t>(p.rows, (int64_t)std::max(1, per) * 148);
    Q35_CUDA_TRY(launch_dependent(kern, dim3((unsigned)grid), threads, smem, s, 1, p));
    return Q35_OK;
}

template <typename T, int CODE, bool ROW> int launch_norm8(const Norm8Params &p, cudaStream_t s) {
    return p.vec ? launch_norm8<T, CODE, ROW, true>(p, s) : launch_norm8<T, CODE, ROW, false>(p, s);
}

template <typename T> int launch_norm8(const Norm8Params &p, int code, bool row, cudaStream_t s) {
    if (code == Q35_CODE_INT8)
        return row ? launch_norm8<T, Q35_CODE_INT8, true>(p, s) : launch_norm8<T, Q35_CODE_INT8, false>(p, s);
    return row ? launch_norm8<T, Q35_CODE_E4M3, true>(p, s) : launch_norm8<T, Q35_CODE_E4M3, false>(p, s);
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
    // writes them; one row has no stride); a shifted overlap would read sums
    if (residual_out) {
        auto overlaps = [&](const void *p, int64_t ld) {
            const char *a = static_cast<const char *>(p), *o = static_cast<const char *>(residual_out);
            const size_t na = ((size_t)(rows - 1) * ld + dim) * es, no = ((size_t)(rows - 1) * ldo + dim) * es;
            return p && a < o + no && o < a + na && !(a == o && (ld == ldo || rows == 1));
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
    p.rows = rows;
    p.dim = dim;
    p.groups = group ? (int32_t)ceil_div(dim, Q8_BLOCK) : 1;
    p.eps = eps;
    p.inv_dim = 1.0f / (float)dim;
    const int V = (int)(16 / es);
    auto vec_ok = [&](const void *ptr, int64_t ld) { return !ptr || (aligned_to(ptr, 16) && ld % V == 0); };
    p.vec = dim % V == 0 && aligned_to(weight, 16) && vec_ok(x, ldx) && vec_ok(residual, ldr) && vec_ok(residual_out, ldo) &&
            aligned_to(q, V) && ldq % V == 0;
    switch (dtype) {
    case Q35_DT_F32: return launch_norm8<float>(p, code, group == 0, ctx->stream);
    case Q35_DT_BF16: return launch_norm8<__nv_bfloat16>(p, code, group == 0, ctx->stream);
    default: return launch_norm8<__half>(p, code, group == 0, ctx->stream);
    }
}
