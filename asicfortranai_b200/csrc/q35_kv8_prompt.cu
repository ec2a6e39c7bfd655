// q35_kv8_prompt.cu -- causal attention of many rows over the 8-bit KV cache on the 5th-generation
// tensor cores; q35_kv8.cu has the definition, the cache and the other forms.
//
// One CTA per tile of 128 (row, head) pairs of a sequence and kv head, two CTAs per SM where the
// memory takes them (one's softmax under the other's MMAs).  Per 64 keys:
//   * converters: warps 4, 5 turn K's codes into fp16 (exact) in shared memory, keys as rows; warps
//     6, 7 V's, transposed on the way (a thread's 8 keys x 16 d become 16 rows of 8 keys), so both
//     MMA operands are K-major with the 128-byte swizzle;
//   * MMA issuer (warp 8, one thread): S = Q K^T into one of two tensor-memory buffers, then
//     O += P V with P from tensor memory;
//   * softmax (warps 0..3, a row per thread): S from tensor memory, times the row's and the
//     block's scale, masked; weights relative to a reference that follows the running maximum
//     only when that has grown by 2^4 (fp32 queries: 2), so O is rarely moved; weights times the
//     block's v scale over the largest one so far go back as fp16 into S's buffer, with a factor that
//     spends fp16's range on small ones.
// fp32 queries and their weights take two fp16 terms each (22 bits), with two MMAs for one, the low terms
// first.
//
// Sums and O are fp32.  The tensor cores' additions do not round to nearest: each loses up to a bit of what
// has been summed so far, always towards zero.  With 16-bit queries that is 7e-5 of an output over 20
// thousand keys of like weight, below the outputs' own rounding (half a step of fp16: 4.9e-4).  With fp32
// queries (1.4e-4: two products a key) P V adds up two steps at a time, in one of two buffers, and the
// softmax warps add these to sums in registers, rounded; a head_dim of 256 is two CTAs then, 128 d of the
// values each.
//
// Measured, 2048 rows of 40 heads of 128 over 2001 older tokens, bf16: 250 us (75 are the operations at
// the fp16 rate), f32 555 (445 with all of O in the tensor cores' accumulators).  A CTA's step of 64 keys
// (bf16) takes 3300 clocks, of which a softmax warp works 2000 (1500 of them on the weights: 16 exponentials a clock
// and SM alone are 512 for each of the SM's two CTAs) and the tensor pipe is busy for 640.
//
// Waits are bounded as in q35_fp8.cu.
#include <cfloat>
#include <type_traits>

#include "q35_kv8.cuh"
#include "q35_tc.cuh"

namespace q35 {
namespace {

constexpr int PT_ROWS = 128;               // (row, head) pairs per CTA
constexpr int PT_KEYS = 64;                // keys per step
constexpr int PT_THREADS = 288;

// TERMS: fp16 terms of a query element and of a weight (2 for fp32 queries: 22 bits)
template <int TERMS, int D> struct Prompt {
    // d of the values a CTA takes (fp32 queries of 256: two CTAs, each with all scores), and whether a group of
    // steps' outputs is added up outside the tensor cores
    static constexpr int DV = TERMS == 2 && D > 128 ? 128 : D;
    static constexpr bool apart = TERMS == 2;
    static constexpr int group = 2;                                    // steps that P V adds up in its accumulator
    static constexpr uint32_t Q = PT_ROWS * D * 2, K = PT_KEYS * D * 2, V = DV * PT_KEYS * 2;  // Q: one term
    static constexpr int stages = TERMS * D > 256 ? 1 : 2;             // of K and V: what the memory takes
    static constexpr int ctas = apart || D > 128 ? 1 : 2;              // per SM
    // (sums outside the tensor cores take registers, which the converters give up: 232 + 96 of twice 168.  The
    // issuer's warpgroup is filled up with idle warps, so that each is whole)
    static constexpr int threads = apart ? 384 : PT_THREADS;
    static constexpr int softmax_regs = 232, converter_regs = 96, launch_regs = (softmax_regs + converter_regs) / 2;
    static constexpr uint32_t tmem = 128 + (apart ? 2 : 1) * DV > 256 ? 512 : 256;    // columns: S 2 x 64, O (2 of a step)
    static constexpr uint32_t off_k = TERMS * Q, off_v = off_k + stages * K, off_bar = off_v + stages * V;
    static constexpr size_t smem = 1024 + off_bar + 8 * 18 + 16 + 4 * 32;
    // A row's maximum may pass its reference by 2^slack, and the weights carry a factor `boost` in fp16:
    // 2^15 together.  The factor keeps the bits of weights far below the reference (a key high above the
    // others whose value is small, a block of large values without weight): 11 bits down to 2^-25 of it and
    // 2^-36 at most below, with fp32 queries 22 bits down to 2^-17 and 2^-39.  Measured with factors of
    // 2^7 / 2^11 / 2^13 / 2^14 at 2048 rows of 40 heads of 128 over 2001 older tokens, append included: bf16 276 /
    // 279 / 283 / 285 us (O moves more often), fp32 477 at all four.
    static constexpr float slack = TERMS == 2 ? 1.0f : 4.0f, boost = TERMS == 2 ? 16384.0f : 2048.0f;
};

__device__ __forceinline__ void tc_mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// A from tensor memory
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0],"
                 " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16,"
                 " %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                   "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
                   "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
                   "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
                 : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
                 " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                   "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D fp32, A and B fp16, both K-major
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void st_shared16(uint32_t addr, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// makes this thread's shared-memory writes visible to the tensor cores' reads
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// byte offset of 16-byte chunk `chunk` (0..7) of row `row` in a block of 128-byte rows, 128-byte swizzle
__device__ __forceinline__ uint32_t swz(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

template <typename T, int CODE, int D>
__global__ void __launch_bounds__((Prompt<std::is_same<T, float>::value ? 2 : 1, D>::threads), (Prompt<std::is_same<T, float>::value ? 2 : 1, D>::ctas))
kv8_prompt_kernel(const AttnParams p) {
    constexpr int TERMS = std::is_same<T, float>::value ? 2 : 1;
    using L = Prompt<TERMS, D>;
    constexpr int ST = L::stages, DV = L::DV;
    const int d0 = DV < D ? (int)blockIdx.z * DV : 0;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t *sbase = smem_raw + (base - raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t bars = base + L::off_bar;
    auto k_full = [&](int i) { return bars + 8u * i; };            // 2 converter warps
    auto k_empty = [&](int i) { return bars + 8u * (2 + i); };     // commit of Q K^T
    auto v_full = [&](int i) { return bars + 8u * (4 + i); };      // 2 converter warps
    auto pv_done = [&](int i) { return bars + 8u * (6 + i); };     // commit of P V (frees V's stage and S's buffer)
    auto s_full = [&](int i) { return bars + 8u * (8 + i); };      // commit of Q K^T
    auto p_full = [&](int i) { return bars + 8u * (10 + i); };     // 4 softmax warps
    const uint32_t q_full = bars + 8u * 12, drain = bars + 8u * 13;
    auto sc_full = [&](int i) { return bars + 8u * (14 + i); };    // a step's scales stand in slot i of 4
    uint8_t *misc = sbase + L::off_bar + 8 * 18;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(misc);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(misc + 4);
    float *scales = reinterpret_cast<float *>(misc + 16);          // [4][4 of k, 4 of v]: by 16 keys

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full(i), 2); mbar_init(k_empty(i), 1); mbar_init(v_full(i), 2);
            mbar_init(pv_done(i), 1); mbar_init(s_full(i), 1); mbar_init(p_full(i), 4);
        }
        for (int i = 0; i < 4; ++i) mbar_init(sc_full(i), 1);
        mbar_init(q_full, 4);
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void *)tmem_slot)), "r"(L::tmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;          // S buffers at 0 and 64, O at 128
    dependency_trigger();
    dependency_wait();

    // the tiles with most keys first
    const int mt = gridDim.x - 1 - blockIdx.x;
    const int KVH = p.H / p.G;
    const int seq = blockIdx.y / KVH, kvh = blockIdx.y - seq * KVH;
    const SeqRows sr = seq_rows(p.row_start, p.past, seq, p.rows, p.max_rows, p.max_seq, p.err);
    const int f0 = mt * PT_ROWS;
    const int fn = min(PT_ROWS, sr.n * p.G - f0);
    const int kend = fn > 0 ? sr.past + (f0 + fn - 1) / p.G + 1 : 0;   // keys the tile's last row sees
    const int steps = (kend + PT_KEYS - 1) / PT_KEYS;                  // (0: nothing to do)
    const int64_t hb = seq * p.seq_stride + (int64_t)kvh * p.max_seq * D;
    const int64_t sb = seq * p.scale_seq_stride + (int64_t)kvh * p.nblk;
    // where P V of step j adds up
    auto o_at = [&](int j) { return 128u + (uint32_t)(L::apart ? j / L::group % 2 * DV : 0); };
    bool ok = true;
    auto fail = [&]() {
        ok = false;
        *abort_flag = 1;
        atomicExch(p.err, Q35_ERR_TIMEOUT);
    };

    if (warp < 4) {
        // ---------------- Q, softmax, output: row `tid` of the tile ----------------
        if constexpr (L::apart) regs_up<L::softmax_regs>();
        const int r = tid, f = f0 + r;
        const bool live = r < fn;
        const int lim = live ? sr.past + f / p.G + 1 : 0;
        const int64_t row = sr.r0 + (live ? f / p.G : 0);
        const int head = kvh * p.G + (live ? f % p.G : 0);
        float qs = 0.0f;
        if (steps > 0) {
            const T *src = static_cast<const T *>(p.q) + row * p.ldq + (int64_t)head * D;
            const bool vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
            auto load8 = [&](int d, T (&x)[8]) {
                if (vec) {
#pragma unroll
                    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                        reinterpret_cast<uint4 *>(x)[i] = reinterpret_cast<const uint4 *>(src + d)[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = src[d + i];
                }
            };
            float a = 0.0f;
            if (live) {
#pragma unroll 4
                for (int d = 0; d < D; d += 8) {
                    __align__(16) T x[8];
                    load8(d, x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(to_f32<T>(x[i])));
                }
            }
            // a power of two brings the row's largest element to 2^13..2^14 (the scale's sign with it, so
            // that the largest product is the largest score)
            const int e = min(126, 13 - ((int)(__float_as_uint(a) >> 23) - 127));
            const float up = copysignf(a > 0.0f ? __uint_as_float((uint32_t)(e + 127) << 23) : 1.0f, p.scale);
            qs = fabsf(p.scale) * 1.4426950408889634f * (a > 0.0f ? __uint_as_float((uint32_t)(127 - e) << 23) : 1.0f);
#pragma unroll 2
            for (int d = 0; d < D; d += 8) {
                __align__(16) T x[8];
                uint32_t w[4], lo[4] = {0u, 0u, 0u, 0u};
                if (live) load8(d, x);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y0 = to_f32<T>(x[2 * i]) * up, y1 = to_f32<T>(x[2 * i + 1]) * up;
                    w[i] = live ? pack2<__half>(y0, y1) : 0u;
                    if (TERMS == 2 && live) {
                        const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                        lo[i] = pack2<__half>(y0 - h.x, y1 - h.y);
                    }
                }
                const uint32_t at = base + (uint32_t)(d / 64) * (PT_ROWS * 128) + swz(r, (d % 64) / 8);
                st_shared16(at, make_uint4(w[0], w[1], w[2], w[3]));
                if (TERMS == 2) st_shared16(at + L::Q, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }

        const int all_see = fn > 0 ? sr.past + f0 / p.G + 1 : 0;       // keys below this: every row sees them
        const uint32_t lanes = (uint32_t)(32 * warp) << 16;
        float m = -INFINITY, l = 0.0f;            // reference of the weights, their sum
        // largest v scale that the row has seen and its reciprocal (a later row's would cost an earlier
        // one bits of its weights); 2^-126 times the weights' factor stands for less
        float vref = L::boost * FLT_MIN, vinv = 1.0f / FLT_MIN;        // (the reciprocal times L::boost)
        float acc[L::apart ? DV : 1];             // outputs of the steps before the last one
        if constexpr (L::apart) {
#pragma unroll
            for (int i = 0; i < DV; ++i) acc[i] = 0.0f;
        }
        // adds the outputs of the steps up to j, which are relative to the references that acc has
        auto add_step = [&](int j) {
            if (!__all_sync(0xffffffffu, mbar_wait(pv_done(j & 1), (uint32_t)((j >> 1) & 1), abort_flag))) { fail(); return; }
            tc_fence_after();
            if constexpr (L::apart) {
#pragma unroll
                for (int d = 0; d < DV; d += 32) {
                    float o[32];
                    tc_ld32(tmem + lanes + o_at(j) + (uint32_t)d, o);
                    tc_wait_ld(o);
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[d + i] += o[i];
                }
            }
        };
        for (int j = 0; j < steps && ok; ++j) {
            const int b = j & 1, kk = j * PT_KEYS;
            const uint32_t ph = (uint32_t)((j >> 1) & 1);
            // (a slot is written again for step j + 4, which the K converters reach only after P V of step
            // j, so its phase is still the one to wait for)
            if (!__all_sync(0xffffffffu, mbar_wait(sc_full(j & 3), (uint32_t)((j >> 2) & 1), abort_flag) &&
                                             mbar_wait(s_full(b), ph, abort_flag))) { fail(); break; }
            const float4 k4 = *reinterpret_cast<const float4 *>(scales + 8 * (j & 3));
            const float4 v4 = *reinterpret_cast<const float4 *>(scales + 8 * (j & 3) + 4);
            // (never 0: a masked score times 0 would be NaN)
            const float ks[4] = {fmaxf(k4.x * qs, 1e-37f), fmaxf(k4.y * qs, 1e-37f), fmaxf(k4.z * qs, 1e-37f), fmaxf(k4.w * qs, 1e-37f)};
            const bool edge = kk + PT_KEYS > all_see;                  // some row does not see some key
            float vs[4] = {v4.x, v4.y, v4.z, v4.w};
            if (edge) {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (kk + 16 * u >= lim) vs[u] = 0.0f;
            }
            const float vtop = fmaxf(fmaxf(vref, fmaxf(vs[0], vs[1])), fmaxf(vs[2], vs[3]));
            tc_fence_after();
            // the scores are read twice, 32 at a time: for the maximum, then for the weights (all 64 with
            // their weights would not fit the registers of two CTAs an SM)
            float mx = -INFINITY;
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                float s[32];
                tc_ld32(tmem + lanes + (uint32_t)(64 * b + 32 * hh), s);
                tc_wait_ld(s);
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (kk + 32 * hh + i >= lim) s[i] = -INFINITY;
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    float x = s[16 * u];
#pragma unroll
                    for (int i = 1; i < 16; ++i) x = fmaxf(x, s[16 * u + i]);
                    mx = fmaxf(mx, x * ks[2 * hh + u]);
                }
            }
            // O moves to new references only where a row's maximum has passed its own by 2^slack, or for
            // a larger v scale
            float down = 1.0f;
            if (__any_sync(0xffffffffu, mx > m + L::slack || vtop > vref)) {
                if (vtop > vref) vinv = L::boost / vtop;
                const float vdown = vtop > vref ? vref * vinv * (1.0f / L::boost) : 1.0f;
                vref = vtop;
                const float to = mx > m + L::slack ? mx : m;
                down = to == -INFINITY ? 1.0f : ex2(m - to);
                m = to;
                l *= down;
                down *= vdown;
                if (L::apart ? j % L::group > 0 : j > 0) {
                    if (!__all_sync(0xffffffffu, mbar_wait(pv_done(b ^ 1), (uint32_t)(((j - 1) >> 1) & 1), abort_flag))) { fail(); break; }
                    tc_fence_after();
                    constexpr int W = L::apart ? 16 : 32;              // (registers)
#pragma unroll 1
                    for (int d = 0; d < DV; d += W) {
                        float o[W];
                        uint32_t w[W];
                        const uint32_t at = tmem + lanes + o_at(j) + (uint32_t)d;
                        if constexpr (W == 16) tc_ld16(at, o);
                        else tc_ld32(at, o);
                        tc_wait_ld(o);
#pragma unroll
                        for (int i = 0; i < W; ++i) w[i] = __float_as_uint(o[i] * down);
                        if constexpr (W == 16) tc_st16(at, w);
                        else tc_st32(at, w);
                    }
                    tc_wait_st();
                }
            }
            const float mu = m == -INFINITY ? 0.0f : m;                // a row that has seen no key yet
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                // (the weights of the first half take the place of its own scores, the second's too: 16
                // columns of high terms, then 16 of low ones)
                float s[32];
                uint32_t pk[16], pl[TERMS == 2 ? 16 : 1];
                float sum = 0.0f;                                      // (of 32: l takes two additions a step)
                tc_ld32(tmem + lanes + (uint32_t)(64 * b + 32 * hh), s);
                tc_wait_ld(s);
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (kk + 32 * hh + i >= lim) s[i] = -INFINITY;
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float c = ks[2 * hh + u], v = vs[2 * hh + u];
                    const float w = v == vref ? L::boost : v * vinv;
#pragma unroll
                    for (int i = 16 * u; i < 16 * u + 16; i += 2) {
                        const float e0 = ex2(fmaf(s[i], c, -mu)), e1 = ex2(fmaf(s[i + 1], c, -mu));
                        sum += e0 + e1;
                        pk[i / 2] = pack2<__half>(e0 * w, e1 * w);
                        if constexpr (TERMS == 2) {
                            const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&pk[i / 2]));
                            pl[i / 2] = pack2<__half>(fmaf(e0, w, -h.x), fmaf(e1, w, -h.y));
                        }
                    }
                }
                l += sum;
                tc_st16(tmem + lanes + (uint32_t)(64 * b + 32 * hh), pk);
                if constexpr (TERMS == 2) tc_st16(tmem + lanes + (uint32_t)(64 * b + 32 * hh + 16), pl);
            }
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full(b));
            if constexpr (L::apart) {
                // (P V does not come back to the buffer before the next arrivals on p_full)
                if (j > 0 && j % L::group == 0) add_step(j - 1);
                if (__any_sync(0xffffffffu, down != 1.0f)) {
#pragma unroll
                    for (int i = 0; i < DV; ++i) acc[i] *= down;
                }
            }
        }
        if (steps > 0 && ok) {
            add_step(steps - 1);
            const float inv = 1.0f / (l * L::boost);
            T *dst = static_cast<T *>(p.out) + row * p.ldo + (int64_t)head * D + d0;
            const bool vec = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
#pragma unroll(L::apart ? DV / 32 : 1)
            for (int d = 0; d < DV; d += 32) {
                float o[32];
                if (!ok) break;
                if constexpr (L::apart) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = acc[d + i];
                } else {
                    __syncwarp();
                    tc_ld32(tmem + lanes + 128u + (uint32_t)d, o);
                    tc_wait_ld(o);
                }
                if (!live) continue;
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = o[i] * inv * vref;
                if (p.out_q) {
                    uint32_t c[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        c[i] = (uint32_t)(uint8_t)quant127(o[4 * i]) | (uint32_t)(uint8_t)quant127(o[4 * i + 1]) << 8 |
                               (uint32_t)(uint8_t)quant127(o[4 * i + 2]) << 16 | (uint32_t)(uint8_t)quant127(o[4 * i + 3]) << 24;
                    uint4 *dq = reinterpret_cast<uint4 *>(p.out_q + (row * p.H + head) * D + d0 + d);
                    dq[0] = make_uint4(c[0], c[1], c[2], c[3]);
                    dq[1] = make_uint4(c[4], c[5], c[6], c[7]);
                } else if (vec) {
                    if constexpr (TERMS == 2) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4 *>(dst + d + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
                            *reinterpret_cast<uint4 *>(dst + d + i) =
                                make_uint4(pack2<T>(o[i], o[i + 1]), pack2<T>(o[i + 2], o[i + 3]), pack2<T>(o[i + 4], o[i + 5]),
                                           pack2<T>(o[i + 6], o[i + 7]));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) dst[d + i] = from_f32<T>(o[i]);
                }
            }
        }
    } else if (warp < 8) {
        if constexpr (L::apart) regs_down<L::converter_regs>();
        if (warp < 6) {
            // ---------------- K: fp16 rows ----------------
            // D / 16 neighbouring lanes take a key's row (whole lines); a thread has D / 16 pieces of 16 codes
            constexpr int LK = D / 16, KR = 64 / LK;                     // lanes per key, keys per round of 64 threads
            const int t = tid - 128, ch = t % LK, key0 = t / LK;
            const uint8_t *kb = p.k + hb + 16 * ch;
            uint4 c[LK];
            auto load = [&](int j) {
#pragma unroll
                for (int i = 0; i < LK; ++i) c[i] = ldg16(kb + (int64_t)min(j * PT_KEYS + KR * i + key0, kend - 1) * D);
            };
            // lanes 0..3 of warp 4 the step's k scales, 4..7 its v scales
            const float *sp = (t < 4 ? p.ks : p.vs) + sb;
            float sc = 0.0f;
            auto load_scale = [&](int j) {
                const int key = j * PT_KEYS + 16 * (t & 3);
                sc = 0.0f;
                if (t < 8 && key < kend) sc = ldg(sp + (key >> p.block_shift));
            };
            if (steps > 0) { load(0); load_scale(0); }
            for (int j = 0; j < steps && ok; ++j) {
                const int b = j % ST;
                if (!__all_sync(0xffffffffu, mbar_wait(k_empty(b), (uint32_t)((j / ST) & 1) ^ 1u, abort_flag))) { fail(); break; }
                const uint32_t dst = base + L::off_k + (uint32_t)b * L::K;
                const uint32_t blk = dst + (uint32_t)(ch / 4) * (PT_KEYS * 128);
                const int odd = (ch / 4) & 1;                            // (neighbouring 64-d blocks' lanes write the
#pragma unroll                                                       // halves in opposite order: no bank conflicts)
                for (int i = 0; i < LK; ++i) {
                    uint4 x, y;
                    codes_f16<CODE>(c[i].x, x.x, x.y);
                    codes_f16<CODE>(c[i].y, x.z, x.w);
                    codes_f16<CODE>(c[i].z, y.x, y.y);
                    codes_f16<CODE>(c[i].w, y.z, y.w);
                    const int key = KR * i + key0;
                    st_shared16(blk + swz(key, 2 * (ch % 4) + odd), odd ? y : x);
                    st_shared16(blk + swz(key, 2 * (ch % 4) + 1 - odd), odd ? x : y);
                }
                if (t < 8) scales[8 * (j & 3) + t] = sc;
                if (j + 1 < steps) { load(j + 1); load_scale(j + 1); }
                fence_async();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(k_full(b));
                    if (warp == 4) mbar_arrive(sc_full(j & 3));
                }
            }
        } else {
            // ---------------- V: fp16, transposed ----------------
            constexpr int VG = DV > 128 ? DV / 128 : 1;                    // pieces of 16 d x 8 keys a thread
            const int t = tid - 192, kg = t & 7, dg0 = t >> 3;           // keys 8 kg .., d 16 dg .. (8 groups, DV / 16 in all)
            const uint8_t *vb = p.v + hb + d0 + 16 * dg0;
            uint4 c[VG][8];
            const bool live = dg0 < DV / 16;
            auto load = [&](int j) {
#pragma unroll
                for (int g = 0; g < VG; ++g)
#pragma unroll
                    for (int i = 0; i < 8; ++i) c[g][i] = ldg16(vb + 128 * g + (int64_t)min(j * PT_KEYS + 8 * kg + i, kend - 1) * D);
            };
            if (steps > 0 && live) load(0);
            for (int j = 0; j < steps && ok; ++j) {
                const int b = j % ST;
                // the stage is free: P V of step j - ST
                if (j >= ST && !__all_sync(0xffffffffu, mbar_wait(pv_done((j - ST) & 1), (uint32_t)((j - ST) >> 1) & 1u, abort_flag))) { fail(); break; }
                if (live) {
                    // past the last key: whatever is stored there must not count
                    if ((j + 1) * PT_KEYS > kend) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (j * PT_KEYS + 8 * kg + i >= kend) {
#pragma unroll
                                for (int g = 0; g < VG; ++g) c[g][i] = make_uint4(0u, 0u, 0u, 0u);
                            }
                    }
                    const uint32_t dst = base + L::off_v + (uint32_t)b * L::V;
                    auto word = [&](const uint4 &u, int w) { return w == 0 ? u.x : w == 1 ? u.y : w == 2 ? u.z : u.w; };
#pragma unroll
                    for (int g = 0; g < VG; ++g)
#pragma unroll
                        for (int w = 0; w < 4; ++w)
#pragma unroll
                            for (int hh = 0; hh < 2; ++hh) {
                                uint4 x, y;                               // d = 16 dg + 4 w + 2 hh, and the next
                                const uint32_t sel = hh ? 0x7362 : 0x5140;
                                codes_f16<CODE>(__byte_perm(word(c[g][0], w), word(c[g][1], w), sel), x.x, y.x);
                                codes_f16<CODE>(__byte_perm(word(c[g][2], w), word(c[g][3], w), sel), x.y, y.y);
                                codes_f16<CODE>(__byte_perm(word(c[g][4], w), word(c[g][5], w), sel), x.z, y.z);
                                codes_f16<CODE>(__byte_perm(word(c[g][6], w), word(c[g][7], w), sel), x.w, y.w);
                                const int d = 16 * (dg0 + 8 * g) + 4 * w + 2 * hh;
                                st_shared16(dst + swz(d, kg), x);
                                st_shared16(dst + swz(d + 1, kg), y);
                            }
                    if (j + 1 < steps) load(j + 1);
                }
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full(b));
            }
        }
    } else if (warp == 8 && lane == 0 && steps > 0) {
        // ---------------- MMA issuer ----------------
        const uint32_t is = idesc_f16(PT_ROWS, PT_KEYS), io = idesc_f16(PT_ROWS, DV);
        const uint64_t qd = smem_desc_sw128(base);
        if (!mbar_wait(q_full, 0, abort_flag)) fail();
        auto scores = [&](int j) {
            const int b = j & 1, sb = j % ST;
            // the buffer's weights have been read: P V of step j - 2
            if (!mbar_wait(k_full(sb), (uint32_t)((j / ST) & 1), abort_flag) ||
                (j >= 2 && !mbar_wait(pv_done(b), (uint32_t)((j >> 1) & 1) ^ 1u, abort_flag))) { fail(); return; }
            tc_fence_after();
            const uint64_t kd = smem_desc_sw128(base + L::off_k + (uint32_t)sb * L::K);
#pragma unroll
            for (int term = TERMS - 1; term >= 0; --term)              // (small sums first: they lose less)
#pragma unroll
                for (int i = 0; i < D / 16; ++i)
                    tc_mma_f16(tmem + (uint32_t)(64 * b), qd + (uint64_t)((term * L::Q + (i / 4) * (PT_ROWS * 128)) / 16 + 2 * (i % 4)),
                               kd + (uint64_t)((i / 4) * (PT_KEYS * 128 >> 4) + 2 * (i % 4)), is, term < TERMS - 1 || i > 0 ? 1u : 0u);
            tc_commit(k_empty(sb));
            tc_commit(s_full(b));
        };
        if (ok) scores(0);
        for (int j = 0; j < steps && ok; ++j) {
            const int b = j & 1, sb = j % ST;
            if (j + 1 < steps) scores(j + 1);
            if (!ok) break;
            if (!mbar_wait(p_full(b), (uint32_t)((j >> 1) & 1), abort_flag) ||
                !mbar_wait(v_full(sb), (uint32_t)((j / ST) & 1), abort_flag)) { fail(); break; }
            tc_fence_after();
            const uint64_t vd = smem_desc_sw128(base + L::off_v + (uint32_t)sb * L::V);
#pragma unroll
            for (int term = TERMS - 1; term >= 0; --term)
#pragma unroll
                for (int i = 0; i < PT_KEYS / 16; ++i)
                    tc_mma_f16_ts(tmem + o_at(j), tmem + (uint32_t)(64 * b + 32 * (i / 2) + 16 * term + 8 * (i % 2)),
                                  vd + (uint64_t)(2 * i), io, (L::apart ? j % L::group : j) > 0 || i > 0 || term < TERMS - 1 ? 1u : 0u);
            tc_commit(pv_done(b));
        }
        tc_commit(drain);
        if (!mbar_wait(drain, 0, abort_flag)) fail();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 8) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::tmem) : "memory");
    }
}

template <typename T, int CODE, int D> int launch_prompt(const AttnParams &p, int zs, cudaStream_t s) {
    using L = Prompt<std::is_same<T, float>::value ? 2 : 1, D>;
    auto kern = kv8_prompt_kernel<T, CODE, D>;
    static bool configured[64] = {};
    int dev = 0;
    Q35_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        Q35_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem));
        if (L::apart) {
            // the split of the registers takes what the CTA has at launch: with less it would wait for ever
            cudaFuncAttributes a;
            Q35_CUDA_TRY(cudaFuncGetAttributes(&a, kern));
            if (a.numRegs < L::launch_regs) return set_error(Q35_ERR_INVALID, "kv8_attention: the prompt kernel was built with too few registers");
        }
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    const dim3 grid((unsigned)ceil_div((int64_t)p.max_rows * p.G, PT_ROWS), (unsigned)zs, (unsigned)(D / L::DV));
    Q35_CUDA_TRY(launch_dependent(kern, grid, L::threads, L::smem, s, 1, p));
    return Q35_OK;
}
template <typename T, int CODE> int launch_prompt(const AttnParams &p, int D, int zs, cudaStream_t s) {
    return D == 64 ? launch_prompt<T, CODE, 64>(p, zs, s) : D == 128 ? launch_prompt<T, CODE, 128>(p, zs, s) : launch_prompt<T, CODE, 256>(p, zs, s);
}
template <typename T> int launch_prompt(const AttnParams &p, int code, int D, int zs, cudaStream_t s) {
    return code == Q35_CODE_INT8 ? launch_prompt<T, Q35_CODE_INT8>(p, D, zs, s) : launch_prompt<T, Q35_CODE_E4M3>(p, D, zs, s);
}

}  // namespace

// Half a tile of (row, head) pairs at least, and tiles for a good part of the SMs: the 16-row form
// splits few tiles' keys over all SMs, this one walks them alone.  Append and attention over 4000
// older tokens, 16-row form against this one: bf16 8 tiles 48 / 84 us (head_dim 128), 89 / 119 (256);
// 16 tiles 64 / 93, 118 / 121; 32 tiles 94 / 89, 172 / 128; 160 tiles 330 / 135, 600 / 262.  fp32 with head_dim
// 64, 128, 256: 32 tiles 68 / 86, 119 / 124, 251 / 184; 64 tiles 99 / 90, 192 / 149, 415 / 240; 160 tiles
// 227 / 180, 478 / 257, 944 / 647.
bool kv8_prompt_takes(const q35_kv8_cache &c, int32_t heads, int32_t max_rows) {
    const int64_t pairs = (int64_t)max_rows * (heads / c.kv_heads);
    return pairs >= PT_ROWS / 2 && ceil_div(pairs, PT_ROWS) * c.seqs * c.kv_heads >= 32;
}

int launch_kv8_prompt(const AttnParams &p, int dtype, int code, int D, int zs, cudaStream_t s) {
    if (dtype == Q35_DT_F32) return launch_prompt<float>(p, code, D, zs, s);
    return dtype == Q35_DT_BF16 ? launch_prompt<__nv_bfloat16>(p, code, D, zs, s) : launch_prompt<__half>(p, code, D, zs, s);
}

}  // namespace q35
