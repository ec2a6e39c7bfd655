// q35_kv8.cu -- a KV cache held in 8 bits with a scale for each block of tokens and head:
// the append that fills it and the causal grouped-query attention that reads it.
//
//   codes  k, v [seq][kv_head][max_seq][head_dim], one byte each (int8 or e4m3)
//   scales k_scale, v_scale [seq][kv_head][ceil(max_seq / block)], block of 16..128 tokens
//
// Append.  Tokens that join a block can be larger than the ones it holds, so the block's
// scale is s' = max(s, max |new| (1/Q)) (s = 0 for a block without older tokens, 1/Q and the
// product rounded to binary32); where it grew, the older codes become the codes nearest to (code * s) / s'.  One CTA per (block,
// head, k or v): it alone reads and writes the block, so nothing races.  Non-finite input
// does not enter the maximum; infinities are stored as +-Q, NaN as 0.
//
// Attention.  o = sum_j softmax_j(scale q . k_j) v_j over the row's own position and all
// before it.  The group's query heads read a kv head's codes once: its (row, head) pairs
// are one side of m16n8k16 tensor-core tiles -- the 8 columns (kv8_attn8_kernel, up to 8 pairs
// in all: single tokens) or the 16 rows (kv8_attn_kernel).  Codes become fp16 exactly (both codes
// fit its 11 bits), the scale multiplies the fp32 scores of its block, and v's scale the
// probabilities, relative to the largest v scale that the row has seen (at most 1).  They are the
// other operand in fp16: 11 bits of a weight, with a factor that spends fp16's range on small ones
// (ATT_BOOST).  A query row is scaled by a power of two to use fp16's range; fp32 queries and their
// probabilities take two fp16 terms each (22 bits).  Maximum, sum and outputs are fp32.
//
// Measured, append and attention together: 16 sequences of 301 to 8100 tokens, 8 kv heads and 64
// heads of 128 45 us (130 MB of codes, 2.9 TB/s), three of 40 to 65 thousand with 32 heads 75 us (306
// MB, 4.1 TB/s); one token after 2000 13 us, three launches.  The append of 2048 tokens of
// 40 heads 28 us (64 MB): conversions and roundings, about 20 instructions an element.
//
// Prompts take 128-row tiles on tcgen05 instead (q35_kv8_prompt.cu).
//
// Single tokens are bound by latency on the way to HBM (a warp has one step of 16 keys on its way; DRAM 41 %,
// SM 33 %, tensor pipe 10 % busy for the 16 sequences above); their form takes K and V^T as the 16-row
// operand, so that half the MMAs and half the accumulators do, and turns the weights around with movmatrix.
//
// No shared-memory staging of codes: a lane's 16 consecutive bytes of a key serve four
// k-steps of Q K^T (the order of the d indices is free as long as Q uses the same), and its
// 16 bytes of each of four keys serve 16 column tiles of P V (the order of the output
// columns is free), so every load is a 16-byte register load and there is no transpose.
#include <algorithm>
#include <cfloat>
#include <cstring>
#include <type_traits>

#include "q35_kv8.cuh"

namespace q35 {
namespace {

struct AppendParams {
    const void *x[2];          // k, v rows
    uint8_t *codes[2];
    float *scales[2];
    int64_t ld;                // elements between rows of x
    int64_t seq_stride, scale_seq_stride;
    const int32_t *row_start, *past;
    int32_t rows, max_rows, G, max_seq, nblk;
    bool vec;                  // rows of x start on 16-byte boundaries
    int *err;
};

constexpr int APPEND_THREADS = 256;

// Four codes of x / s.  A code is the fp32 quotient, rounded; x * r with r = 1/s rounded is within
// 2^-22 of it, so where no rounding boundary lies that near the product rounds to the same code and
// the division is left out (it costs ten instructions or so a value, the product with its check
// five).  `fast` is off where r could overflow.
template <int CODE> __device__ __forceinline__ uint32_t encode_quotients(const float (&x)[4], float s, float r, bool fast) {
    float t[4];
    bool near = !fast;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = x[i] * r;
    if (CODE == Q35_CODE_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float k = __fadd_rn(t[i], 12582912.0f);     // 3 2^22: the sum's last bits are the whole number
            near |= !(fabsf(t[i] - __fadd_rn(k, -12582912.0f)) <= 0.4999f);    // (infinities and NaN too)
            word |= (__float_as_uint(k) & 0xffu) << (8 * i);
        }
    } else {
        // boundaries lie half way between numbers of 3 fraction bits (from 2^-6 on)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            near |= !(fabsf(t[i]) >= 0.015626f) || ((__float_as_uint(t[i]) - 0x7fff8u) & 0xfffffu) < 16u;
        word = encode8x4<CODE>(t[0], t[1], t[2], t[3]);
    }
    if (near) {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = s == 0.0f || x[i] != x[i] ? 0.0f : __fdiv_rn(x[i], s);
        word = encode8x4<CODE>(t[0], t[1], t[2], t[3]);
    }
    return word;
}

template <typename T, int CODE, int D, int TB>
__global__ void __launch_bounds__(APPEND_THREADS) kv8_append_kernel(const AppendParams p) {
    __shared__ float part[APPEND_THREADS / 32];
    dependency_trigger();
    dependency_wait();
    const int s = blockIdx.z >> 1, which = blockIdx.z & 1, head = blockIdx.y;
    const SeqRows q = seq_rows(p.row_start, p.past, s, p.rows, p.max_rows, p.max_seq, p.err);
    if (q.n == 0) return;
    const int blk = q.past / TB + blockIdx.x;
    const int t0 = blk * TB;                              // first token of the block
    const int first = max(t0, q.past), last = min(t0 + TB, q.past + q.n);   // new tokens [first, last)
    if (first >= last) return;
    const T *x = static_cast<const T *>(which ? p.x[1] : p.x[0]) + (int64_t)(q.r0 + first - q.past) * p.ld + (int64_t)head * D;
    uint8_t *codes = (which ? p.codes[1] : p.codes[0]) + s * p.seq_stride + ((int64_t)head * p.max_seq + t0) * D;
    float *scale = (which ? p.scales[1] : p.scales[0]) + s * p.scale_seq_stride + (int64_t)head * p.nblk + blk;
    const int held = first - t0, fresh = last - first;

    // four elements a thread and round, all of the block's rounds in flight (a whole block of 128
    // tokens by 256 is 32 rounds: those take several passes over the input)
    constexpr int STEP = 4 * APPEND_THREADS, ROUNDS = TB * D / STEP, R = ROUNDS < 8 ? ROUNDS : 8;
    static_assert(STEP % D == 0 && ROUNDS >= 1, "a round is whole tokens, a block whole rounds");
    const bool vec = p.vec;
    const int64_t next = (int64_t)(STEP / D) * p.ld;         // elements of x between rounds
    const T *mine = x + (int64_t)(4 * threadIdx.x / D) * p.ld + 4 * threadIdx.x % D;
    // (held as they stand in memory: half the registers for 16-bit types)
    using Raw = typename std::conditional<sizeof(T) == 4, uint4, uint2>::type;
    Raw raw[R];
    const int total = fresh * D;
    auto load = [&](int e0) {                                // rounds e0 / STEP .. of this thread's elements
        const T *s = mine + e0 / STEP * next;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            raw[r] = Raw{};                                  // (zeros)
            if (e0 + r * STEP + 4 * (int)threadIdx.x >= total) continue;
            if (vec) raw[r] = *reinterpret_cast<const Raw *>(s + r * next);
            else {
                T w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = s[r * next + i];
                memcpy(&raw[r], w, sizeof(w));
            }
        }
    };
    auto values = [&](int r, float (&v)[4]) {
        T w[4];
        memcpy(w, &raw[r], sizeof(w));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32<T>(w[i]);
    };
    auto over_cta = [&](float amax) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < APPEND_THREADS / 32; ++w) amax = fmaxf(amax, part[w]);
        return amax;
    };
    const float old = held ? *scale : 0.0f;
    float amax = 0.0f;                                       // (fmaxf leaves NaN out)
    for (int e0 = 0; e0 < total; e0 += R * STEP) {
        load(e0);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float v[4];
            values(r, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(v[i]));
        }
    }
    amax = over_cta(amax);
    if (amax > FLT_MAX) {                                    // infinities do not count: once more without
        amax = 0.0f;
#pragma unroll 1
        for (int e = threadIdx.x; e < total; e += APPEND_THREADS) {
            const float a = fabsf(to_f32<T>(x[(int64_t)(e / D) * p.ld + e % D]));
            if (a <= FLT_MAX) amax = fmaxf(amax, a);
        }
        __syncthreads();
        amax = over_cta(amax);
    }
    const float now = fmaxf(old, __fmul_rn(amax, 1.0f / code_max<CODE>()));
    if (threadIdx.x == 0) *scale = now;
    const float recip = __fdiv_rn(1.0f, now);
    const bool fast = now >= 1e-30f;
    if (held && now != old) {
        uint32_t *w = reinterpret_cast<uint32_t *>(codes) + threadIdx.x;
        const int n = held * D / 4 - (int)threadIdx.x;       // words from this thread's first one on
        for (int i0 = 0; i0 < n; i0 += R * APPEND_THREADS) {
            uint32_t c[R];                                   // (a round's loads together: one latency)
#pragma unroll
            for (int r = 0; r < R; ++r) c[r] = i0 + r * APPEND_THREADS < n ? w[i0 + r * APPEND_THREADS] : 0u;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = __fmul_rn(decode8<CODE>((uint8_t)(c[r] >> (8 * i))), old);
                if (i0 + r * APPEND_THREADS < n) w[i0 + r * APPEND_THREADS] = encode_quotients<CODE>(v, now, recip, fast);
            }
        }
    }
    codes += held * D;
    for (int e0 = 0; e0 < total; e0 += R * STEP) {
        if (total > R * STEP) load(e0);                      // (else the values are still here)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int e = e0 + r * STEP + 4 * threadIdx.x;
            float v[4];
            values(r, v);
            if (e < total) *reinterpret_cast<uint32_t *>(codes + e) = encode_quotients<CODE>(v, now, recip, fast);
        }
    }
}

// ---- attention ------------------------------------------------------------------------

constexpr int ATT_WARPS = 8;
constexpr int ATT_THREADS = 32 * ATT_WARPS;
constexpr int ATT_M = 16;                 // (row, head) pairs per CTA
constexpr int ATT_MAX_SPLITS = 64;        // CTAs that share a tile's keys
// Factor of the weights in fp16.  A weight is at most 1 (the row's largest score, the largest v scale) and
// the ones that carry a row can be far below it: a key high above the others whose value is small, a block
// of large values without weight.  With 2^15 a weight keeps its 11 bits down to 2^-29 and is off by 2^-40
// at most below that (without: 2^-14 and 2^-25).  fp32 queries' second term, the rest of the first, carries
// another 2^11: 22 bits, or 2^-51.
constexpr float ATT_BOOST = 32768.0f, ATT_LOW = 2048.0f;

__device__ __forceinline__ uint2 ldg8(const uint8_t *p) {
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint4 &a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
                 " {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}

template <int D> struct AttnShape {
    // keys per warp and step: 32, 16, 16 (twice as many for D = 64 and 128 left room for one CTA an
    // SM, whose two warps a scheduler waited for memory: 104 against 91 us for three long sequences)
    static constexpr int KC = D == 64 ? 32 : 16;
    static constexpr int CTAS = D == 256 ? 1 : 2;   // per SM
    static constexpr int KS = D / 16;          // k-steps of Q K^T
    static constexpr int ROWS_O = D + 4;       // padded row of the merge buffer, floats
};
template <int D> constexpr size_t attn_smem(int terms) {
    // Q fragments, then (after the key loop) the merge buffer, in the same bytes
    const size_t qf = (size_t)terms * AttnShape<D>::KS * 32 * 16;
    const size_t mg = (size_t)ATT_WARPS * ATT_M * AttnShape<D>::ROWS_O * 4;
    return qf > mg ? qf : mg;
}

// quant127's caller-visible form: int8 trunc(127 o), clamped
template <typename T, int D>
__device__ __forceinline__ void store_out(const AttnParams &p, int64_t row, int head, int d, float v) {
    if (p.out_q) p.out_q[(row * p.H + head) * D + d] = quant127(v);
    else static_cast<T *>(p.out)[row * p.ldo + (int64_t)head * D + d] = from_f32<T>(v);
}

// CTAs that share a tile of `steps` steps: at most `splits`, each with a step for every warp
__device__ __forceinline__ int tile_parts(int steps, int splits) { return max(1, min(splits, steps / ATT_WARPS)); }

// grid (split, tile of 16 (row, head) pairs, seq * kv_heads + kv head)
template <typename T, int CODE, int D>
__global__ void __launch_bounds__(ATT_THREADS, AttnShape<D>::CTAS) kv8_attn_kernel(const AttnParams p) {
    constexpr int TERMS = std::is_same<T, float>::value ? 2 : 1;
    constexpr int KC = AttnShape<D>::KC, KS = AttnShape<D>::KS, NT = KC / 8, VT = D / 8;
    constexpr int RO = AttnShape<D>::ROWS_O;
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ float qscale[ATT_M];
    __shared__ float2 ml[ATT_WARPS][ATT_M];
    uint32_t *qf = reinterpret_cast<uint32_t *>(sm);   // [TERMS][KS][32][4]
    float *mg = reinterpret_cast<float *>(sm);         // [ATT_WARPS][16][RO]

    dependency_trigger();
    dependency_wait();
    const int split = blockIdx.x, mt = blockIdx.y;
    const int KVH = p.H / p.G;
    const int seq = blockIdx.z / KVH, kvh = blockIdx.z - seq * KVH;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const SeqRows sr = seq_rows(p.row_start, p.past, seq, p.rows, p.max_rows, p.max_seq, p.err);
    const int f0 = mt * ATT_M;                          // first (row, head) pair of the tile
    const int fn = min(ATT_M, sr.n * p.G - f0);
    if (fn <= 0) return;
    const int64_t tile = (int64_t)blockIdx.z * gridDim.y + mt;

    // keys of this CTA: an equal share of the keys the tile's last row sees
    const int kend_all = sr.past + (f0 + fn - 1) / p.G + 1;
    const int steps = (kend_all + KC - 1) / KC;
    const int parts = tile_parts(steps, p.splits);
    if (split >= parts) return;
    const int k0 = (int)((int64_t)steps * split / parts) * KC;
    const int k1 = min(kend_all, (int)((int64_t)steps * (split + 1) / parts) * KC);

    // Q rows: a power of two brings each row's largest element to 2^13..2^14
    for (int r = warp; r < ATT_M; r += ATT_WARPS) {
        const int f = f0 + r;
        const bool live = r < fn;
        const T *src = static_cast<const T *>(p.q) + (live ? (int64_t)(sr.r0 + f / p.G) * p.ldq +
                                                                 (int64_t)(kvh * p.G + f % p.G) * D : 0);
        float x[D / 32], a = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            x[i] = live ? to_f32<T>(src[lane + 32 * i]) : 0.0f;
            a = fmaxf(a, fabsf(x[i]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        const int e = min(126, 13 - ((int)(__float_as_uint(a) >> 23) - 127));
        const float up = a > 0.0f ? __uint_as_float((uint32_t)(e + 127) << 23) : 1.0f;
        if (lane == 0) qscale[r] = p.scale * 1.4426950408889634f * (a > 0.0f ? __uint_as_float((uint32_t)(127 - e) << 23) : 1.0f);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int d = lane + 32 * i;
            const int ks = (d / 64) * 4 + (d % 16) / 4, ln = (r % 8) * 4 + (d % 64) / 16;
            const int reg = (d & 2) + (r >> 3), half = d & 1;
            const float y = x[i] * up;
            const __half hi = __float2half_rn(y);
            __half *dst = reinterpret_cast<__half *>(qf + ((ks * 32 + ln) * 4 + reg)) + half;
            *dst = hi;
            if (TERMS == 2) dst[KS * 32 * 8] = __float2half_rn(y - __half2float(hi));
        }
    }
    __syncthreads();

    // rows g and g + 8 of the tile: limits, scales, running maximum and sum
    int lim[2];
    float qs[2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = g + 8 * h;
        lim[h] = r < fn ? sr.past + (f0 + r) / p.G + 1 : 0;
        qs[h] = qscale[r];
    }
    const int all_see = min(k1, sr.past + f0 / p.G + 1);     // keys below this: every row sees them
    const int64_t hb = seq * p.seq_stride + (int64_t)kvh * p.max_seq * D;
    const uint8_t *kb = p.k + hb, *vb = p.v + hb;
    const int64_t sb = seq * p.scale_seq_stride + (int64_t)kvh * p.nblk;
    const float *ksb = p.ks + sb, *vsb = p.vs + sb;

    float o[VT][4];
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] = 0.0f;
    // largest v scale that each of the two rows has seen and its reciprocal (a later row's would cost
    // an earlier one bits of its weights); the smallest normal number stands for less
    float vref[2] = {FLT_MIN, FLT_MIN}, vinv[2] = {1.0f / FLT_MIN, 1.0f / FLT_MIN};

    constexpr int KL = D / 64;                  // 16-byte loads per key and lane: 1, 2, 4
    uint4 kr[NT][KL];                           // K codes of a step: key 8t + g, bytes 64 j + 16 c ..
    constexpr int VW = D == 64 ? 2 : 4;         // words per V load
    constexpr int VL = D == 256 ? 2 : 1;
    uint32_t vr[NT / 2][4][VL][VW];             // V codes: keys 16 s + 2c, +1, +8, +9, bytes 16 g (8 g) ..

    auto load_k = [&](int kk) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint8_t *a = kb + (int64_t)(kk + KC > k1 ? min(kk + 8 * t + g, k1 - 1) : kk + 8 * t + g) * D + 16 * c;
#pragma unroll
            for (int j = 0; j < KL; ++j) kr[t][j] = ldg16(a + 64 * j);
        }
    };
    auto load_v = [&](int kk) {
#pragma unroll
        for (int s = 0; s < NT / 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = kk + 16 * s + 2 * c + (i & 1) + 8 * (i >> 1);
                const uint8_t *a = vb + (int64_t)(kk + KC > k1 ? min(key, k1 - 1) : key) * D;
                if constexpr (D == 64) {
                    const uint2 u = ldg8(a + 8 * g);
                    vr[s][i][0][0] = u.x; vr[s][i][0][1] = u.y;
                } else {
#pragma unroll
                    for (int j = 0; j < VL; ++j) {
                        const uint4 u = ldg16(a + 128 * j + 16 * g);
                        vr[s][i][j][0] = u.x; vr[s][i][j][1] = u.y; vr[s][i][j][2] = u.z; vr[s][i][j][3] = u.w;
                    }
                }
            }
    };
    // past the last key: whatever is stored there must not count (where the codes are used: a
    // selection behind the load would wait for it)
    auto clear_v = [&](int kk) {
#pragma unroll
        for (int s = 0; s < NT / 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (kk + 16 * s + 2 * c + (i & 1) + 8 * (i >> 1) >= k1) {
#pragma unroll
                    for (int j = 0; j < VL; ++j)
#pragma unroll
                        for (int w = 0; w < VW; ++w) vr[s][i][j][w] = 0u;
                }
    };

    // scales of the next step's 16-key pieces (blocks hold 16 tokens or more); as the codes, they
    // are on their way a step ahead
    float nks[NT / 2], nvs[NT / 2];
    auto load_scales = [&](int kk) {
#pragma unroll
        for (int u = 0; u < NT / 2; ++u) {
            const int key = kk + 16 * u;
            nks[u] = nvs[u] = 0.0f;
            if (key < k1) {
                nks[u] = ldg(ksb + (key >> p.block_shift));
                nvs[u] = ldg(vsb + (key >> p.block_shift));
            }
        }
    };

    int kk = k0 + warp * KC;
    if (kk < k1) { load_k(kk); load_scales(kk); load_v(kk); }
    for (; kk < k1; kk += ATT_WARPS * KC) {
        const int nk = kk + ATT_WARPS * KC;
        float s[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] = 0.0f;
        // scores: k-step (j, i) takes byte quad i of load j
#pragma unroll
        for (int j = 0; j < KL; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint4 qa = *reinterpret_cast<const uint4 *>(qf + ((j * 4 + i) * 32 + lane) * 4);
                uint4 ql;
                if (TERMS == 2) ql = *reinterpret_cast<const uint4 *>(qf + ((KS + j * 4 + i) * 32 + lane) * 4);
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    uint32_t b0, b1;
                    codes_f16<CODE>(i == 0 ? kr[t][j].x : i == 1 ? kr[t][j].y : i == 2 ? kr[t][j].z : kr[t][j].w, b0, b1);
                    mma16816(s[t], qa, b0, b1);
                    if (TERMS == 2) mma16816(s[t], ql, b0, b1);
                }
            }
        float ksc[NT / 2], vsc[NT / 2][2], vtop[2] = {vref[0], vref[1]};
#pragma unroll
        for (int u = 0; u < NT / 2; ++u) {
            ksc[u] = nks[u];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                vsc[u][h] = kk + 16 * u < min(lim[h], k1) ? nvs[u] : 0.0f;
                vtop[h] = fmaxf(vtop[h], vsc[u][h]);
            }
        }
        if (nk < k1) { load_k(nk); load_scales(nk); }
        float mx[2] = {m[0], m[1]};
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[t][i] *= qs[i >> 1] * ksc[t / 2];
        if (kk + KC > all_see) {                 // some row does not see some key of the step
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = kk + 8 * t + 2 * c + (i & 1);
                    if (key >= lim[i >> 1] || key >= k1) s[t][i] = -INFINITY;
                }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx[i >> 1] = fmaxf(mx[i >> 1], s[t][i]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        }
        // the outputs so far move to the new maximum and the new reference v scale
        float mu[2], down[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float vdown = 1.0f;
            if (vtop[h] > vref[h]) {
                vinv[h] = 1.0f / vtop[h];
                vdown = vref[h] * vinv[h];
                vref[h] = vtop[h];
            }
            mu[h] = mx[h] == -INFINITY ? 0.0f : mx[h];     // a row that has seen no key yet
            down[h] = ex2(m[h] - mu[h]);
            l[h] *= down[h];
            down[h] *= vdown;
            m[h] = mx[h];
        }
        if (__any_sync(0xffffffffu, down[0] != 1.0f || down[1] != 1.0f)) {
#pragma unroll
            for (int t = 0; t < VT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][i] *= down[i >> 1];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = ex2(s[t][i] - mu[i >> 1]);
                l[i >> 1] += e;
                s[t][i] = e;
            }
        // outputs
        if (kk + KC > k1) clear_v(kk);
#pragma unroll
        for (int u = 0; u < NT / 2; ++u) {
            const float w[2] = {vsc[u][0] == vref[0] ? ATT_BOOST : vsc[u][0] * vinv[0] * ATT_BOOST,
                                vsc[u][1] == vref[1] ? ATT_BOOST : vsc[u][1] * vinv[1] * ATT_BOOST};
            uint4 pa, pl;
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[i] = s[2 * u][i] * w[i >> 1]; x[4 + i] = s[2 * u + 1][i] * w[i >> 1]; }
            pa = make_uint4(pack2<__half>(x[0], x[1]), pack2<__half>(x[2], x[3]), pack2<__half>(x[4], x[5]),
                            pack2<__half>(x[6], x[7]));
            if (TERMS == 2) {
                uint32_t *hp = reinterpret_cast<uint32_t *>(&pa), *lp = reinterpret_cast<uint32_t *>(&pl);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 hf = __half22float2(*reinterpret_cast<const __half2 *>(&hp[i]));
                    lp[i] = pack2<__half>((x[2 * i] - hf.x) * ATT_LOW, (x[2 * i + 1] - hf.y) * ATT_LOW);
                }
            }
#pragma unroll
            for (int j = 0; j < VL; ++j)
#pragma unroll
                for (int w4 = 0; w4 < VW; ++w4) {
                    // keys 2c, 2c+1 interleaved byte by byte, and keys 2c+8, 2c+9
                    const uint32_t a0 = vr[u][0][j][w4], a1 = vr[u][1][j][w4], a2 = vr[u][2][j][w4], a3 = vr[u][3][j][w4];
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        uint32_t b0, b1, b2, b3;
                        codes_f16<CODE>(__byte_perm(a0, a1, hh ? 0x7362 : 0x5140), b0, b1);
                        codes_f16<CODE>(__byte_perm(a2, a3, hh ? 0x7362 : 0x5140), b2, b3);
                        const int t = (j * VW + w4) * 4 + 2 * hh;
                        if (TERMS == 2) {
                            // (rounded additions over the steps)
                            float lo0[4] = {0, 0, 0, 0}, lo1[4] = {0, 0, 0, 0};
                            mma16816(lo0, pl, b0, b2);
                            mma16816(lo1, pl, b1, b3);
#pragma unroll
                            for (int i = 0; i < 4; ++i) { lo0[i] *= 1.0f / ATT_LOW; lo1[i] *= 1.0f / ATT_LOW; }
                            mma16816(lo0, pa, b0, b2);
                            mma16816(lo1, pa, b1, b3);
#pragma unroll
                            for (int i = 0; i < 4; ++i) { o[t][i] += lo0[i]; o[t + 1][i] += lo1[i]; }
                        } else {
                            mma16816(o[t], pa, b0, b2);
                            mma16816(o[t + 1], pa, b1, b3);
                        }
                    }
                }
        }
        if (nk < k1) load_v(nk);
    }

    // merge the warps: every warp's rows relative to its own maximum
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (c == 0) ml[warp][g + 8 * h] = make_float2(m[h], l[h]);
    }
    __syncthreads();       // Q fragments are read no more
#pragma unroll
    for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = 2 * c + (i & 1);      // column tile t, column n: see load_v
            const int d = D == 64 ? n * 8 + t : (t / 16) * 128 + n * 16 + t % 16;
            mg[(warp * ATT_M + g + 8 * (i >> 1)) * RO + d] = o[t][i] * (1.0f / ATT_BOOST) * vref[i >> 1];
        }
    __syncthreads();
    for (int r = warp; r < fn; r += ATT_WARPS) {
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < ATT_WARPS; ++w) mm = fmaxf(mm, ml[w][r].x);
        const float mu = mm == -INFINITY ? 0.0f : mm;
        float sum = 0.0f, f[ATT_WARPS];
#pragma unroll
        for (int w = 0; w < ATT_WARPS; ++w) {
            f[w] = ex2(ml[w][r].x - mu);
            sum = fmaf(ml[w][r].y, f[w], sum);
        }
        const int fr = f0 + r;
        const int64_t slot = (tile * p.splits + split) * ATT_M + r;
        if (parts > 1 && lane == 0) p.part_ml[slot] = make_float2(mm, sum);
        const float inv = 1.0f / sum;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int d = lane + 32 * i;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < ATT_WARPS; ++w) v = fmaf(mg[(w * ATT_M + r) * RO + d], f[w], v);
            if (parts > 1) p.part_o[slot * D + d] = v;
            else store_out<T, D>(p, sr.r0 + fr / p.G, kvh * p.G + fr % p.G, d, v * inv);
        }
    }
}

// ---- up to 8 (row, head) pairs --------------------------------------------------------

template <int D> struct Attn8Shape {
    static constexpr int U = D == 64 ? 2 : 1;                // 16-key pieces per warp and step (twice as many spilled)
    static constexpr int KC = 16 * U;
    static constexpr int KS = D / 16;
    static constexpr int ROWS_O = D + 4;
};
template <int D> constexpr size_t attn8_smem(int terms) {
    const size_t qf = (size_t)terms * Attn8Shape<D>::KS * 32 * 8;
    const size_t mg = (size_t)ATT_WARPS * 8 * Attn8Shape<D>::ROWS_O * 4;
    return qf > mg ? qf : mg;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// grid (split, tile of 8 (row, head) pairs, seq * kv_heads + kv head)
template <typename T, int CODE, int D>
__global__ void __launch_bounds__(ATT_THREADS, D == 256 ? 1 : 2) kv8_attn8_kernel(const AttnParams p) {
    constexpr int TERMS = std::is_same<T, float>::value ? 2 : 1;
    constexpr int U = Attn8Shape<D>::U, KC = Attn8Shape<D>::KC, KS = Attn8Shape<D>::KS, OT = D / 16;
    constexpr int RO = Attn8Shape<D>::ROWS_O, TM = 8;
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ float qscale[TM];
    __shared__ float2 ml[ATT_WARPS][TM];
    uint32_t *qf = reinterpret_cast<uint32_t *>(sm);   // [KS][32][TERMS][2]
    float *mg = reinterpret_cast<float *>(sm);         // [ATT_WARPS][8][RO]

    dependency_trigger();
    dependency_wait();
    const int split = blockIdx.x, mt = blockIdx.y;
    const int KVH = p.H / p.G;
    const int seq = blockIdx.z / KVH, kvh = blockIdx.z - seq * KVH;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const SeqRows sr = seq_rows(p.row_start, p.past, seq, p.rows, p.max_rows, p.max_seq, p.err);
    const int f0 = mt * TM;
    const int fn = min(TM, sr.n * p.G - f0);
    if (fn <= 0) return;
    const int64_t tile = (int64_t)blockIdx.z * gridDim.y + mt;
    const int kend_all = sr.past + (f0 + fn - 1) / p.G + 1;
    const int steps = (kend_all + KC - 1) / KC;
    const int parts = tile_parts(steps, p.splits);
    if (split >= parts) return;
    const int k0 = (int)((int64_t)steps * split / parts) * KC;
    const int k1 = min(kend_all, (int)((int64_t)steps * (split + 1) / parts) * KC);
    const int all_see = min(k1, sr.past + f0 / p.G + 1);     // keys below this: every row sees them
    const int64_t hb = seq * p.seq_stride + (int64_t)kvh * p.max_seq * D;
    const uint8_t *kb = p.k + hb + 16 * c, *vb = p.v + hb + (D == 64 ? 8 : 16) * g;
    const int64_t sb = seq * p.scale_seq_stride + (int64_t)kvh * p.nblk;
    const float *ksb = p.ks + sb, *vsb = p.vs + sb;

    constexpr int KL = D / 64;                  // 16-byte loads per key and lane
    constexpr int VW = D == 64 ? 2 : 4;         // words per V load
    constexpr int VL = D == 256 ? 2 : 1;
    uint4 kr[U][2][KL];                         // keys 16 u + g, + 8: bytes 64 j + 16 c ..
    uint32_t vr[U][4][VL][VW];                  // keys 16 u + 2c, +1, +8, +9
    float nks[U], nvs[U];
    auto load_k = [&](int kk) {
        const bool tail = kk + KC > k1;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                int key = kk + 16 * u + 8 * h + g;
                if (tail) key = min(key, k1 - 1);
#pragma unroll
                for (int j = 0; j < KL; ++j) kr[u][h][j] = ldg16(kb + (int64_t)key * D + 64 * j);
            }
            const int key = min(kk + 16 * u, k1 - 1);
            nks[u] = ldg(ksb + (key >> p.block_shift));
            nvs[u] = ldg(vsb + (key >> p.block_shift));
        }
    };
    auto load_v = [&](int kk) {
        const bool tail = kk + KC > k1;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int key = kk + 16 * u + 2 * c + (i & 1) + 8 * (i >> 1);
                if (tail) key = min(key, k1 - 1);
                const uint8_t *a = vb + (int64_t)key * D;
                if constexpr (D == 64) {
                    const uint2 w = ldg8(a);
                    vr[u][i][0][0] = w.x; vr[u][i][0][1] = w.y;
                } else {
#pragma unroll
                    for (int j = 0; j < VL; ++j) {
                        const uint4 w = ldg16(a + 128 * j);
                        vr[u][i][j][0] = w.x; vr[u][i][j][1] = w.y; vr[u][i][j][2] = w.z; vr[u][i][j][3] = w.w;
                    }
                }
            }
    };
    int kk = k0 + warp * KC;
    if (kk < k1) { load_k(kk); load_v(kk); }

    // Q rows, scaled as in kv8_attn_kernel: warp r prepares row r
    {
        const int r = warp, f = f0 + r;
        const bool live = r < fn;
        const T *src = static_cast<const T *>(p.q) + (live ? (int64_t)(sr.r0 + f / p.G) * p.ldq +
                                                                 (int64_t)(kvh * p.G + f % p.G) * D : 0);
        float x[D / 32], a = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            x[i] = live ? to_f32<T>(src[lane + 32 * i]) : 0.0f;
            a = fmaxf(a, fabsf(x[i]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        const int e = min(126, 13 - ((int)(__float_as_uint(a) >> 23) - 127));
        const float up = a > 0.0f ? __uint_as_float((uint32_t)(e + 127) << 23) : 1.0f;
        if (lane == 0) qscale[r] = p.scale * 1.4426950408889634f * (a > 0.0f ? __uint_as_float((uint32_t)(127 - e) << 23) : 1.0f);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int d = lane + 32 * i;
            const int ks = (d / 64) * 4 + (d % 16) / 4, ln = r * 4 + (d % 64) / 16, reg = (d >> 1) & 1, half = d & 1;
            const float y = x[i] * up;
            const __half hi = __float2half_rn(y);
            __half *dst = reinterpret_cast<__half *>(qf + (ks * 32 + ln) * 2 * TERMS + reg) + half;
            *dst = hi;
            if (TERMS == 2) dst[4] = __float2half_rn(y - __half2float(hi));
        }
    }
    __syncthreads();

    // pairs 2c and 2c + 1: limits, scales, running maximum (the same in every lane of a column)
    // and this lane's share of the sum
    int lim[2];
    float qs[2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = 2 * c + h;
        lim[h] = r < fn ? sr.past + (f0 + r) / p.G + 1 : 0;
        qs[h] = qscale[r];
    }
    float o[OT][4];
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] = 0.0f;
    // largest v scale that each of the two rows has seen and its reciprocal (a later row's would cost
    // an earlier one bits of its weights); the smallest normal number stands for less
    float vref[2] = {FLT_MIN, FLT_MIN}, vinv[2] = {1.0f / FLT_MIN, 1.0f / FLT_MIN};

    for (; kk < k1; kk += ATT_WARPS * KC) {
        const int nk = kk + ATT_WARPS * KC;
        // (the tensor cores' sums lose what lies below the accumulator's last bit, each time: the low
        // terms of fp32 queries have a sum of their own)
        float s[U][4], sl[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] = sl[u][i] = 0.0f;
#pragma unroll
        for (int j = 0; j < KL; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t q0, q1, q2, q3;
                if (TERMS == 2) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(qf + ((j * 4 + i) * 32 + lane) * 4);
                    q0 = v.x; q1 = v.y; q2 = v.z; q3 = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2 *>(qf + ((j * 4 + i) * 32 + lane) * 2);
                    q0 = v.x; q1 = v.y; q2 = q3 = 0u;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    uint4 a;
                    const uint4 &x = kr[u][0][j], &y = kr[u][1][j];
                    codes_f16<CODE>(i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w, a.x, a.z);
                    codes_f16<CODE>(i == 0 ? y.x : i == 1 ? y.y : i == 2 ? y.z : y.w, a.y, a.w);
                    mma16816(s[u], a, q0, q1);
                    if (TERMS == 2) mma16816(sl[u], a, q2, q3);
                }
            }
        float ksc[U], vsc[U][2], vtop[2] = {vref[0], vref[1]};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ksc[u] = nks[u];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                vsc[u][h] = kk + 16 * u < min(lim[h], k1) ? nvs[u] : 0.0f;
                vtop[h] = fmaxf(vtop[h], vsc[u][h]);
            }
        }
        if (nk < k1) load_k(nk);
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] = (TERMS == 2 ? s[u][i] + sl[u][i] : s[u][i]) * (qs[i & 1] * ksc[u]);
        if (kk + KC > all_see) {                 // some row does not see some key of the step
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = kk + 16 * u + g + 8 * (i >> 1);
                    if (key >= lim[i & 1] || key >= k1) s[u][i] = -INFINITY;
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx[i & 1] = fmaxf(mx[i & 1], s[u][i]);
        // a larger score or v scale than before: the outputs so far move to the new references
        if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1] || vtop[0] > vref[0] || vtop[1] > vref[1])) {
            float down[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float vdown = 1.0f;
                if (vtop[h] > vref[h]) {
                    vinv[h] = 1.0f / vtop[h];
                    vdown = vref[h] * vinv[h];
                    vref[h] = vtop[h];
                }
                float x = fmaxf(mx[h], m[h]);
#pragma unroll
                for (int b = 4; b < 32; b <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, b));
                down[h] = x == -INFINITY ? 1.0f : ex2(m[h] - x);
                m[h] = x;
                l[h] *= down[h];
                down[h] *= vdown;
            }
#pragma unroll
            for (int t = 0; t < OT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[t][i] *= down[i & 1];
        }
        if (kk + KC > k1) {
            // past the last key: whatever is stored there must not count (cleared where the codes
            // are used: a selection behind the load would wait for it)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (kk + 16 * u + 2 * c + (i & 1) + 8 * (i >> 1) >= k1) {
#pragma unroll
                        for (int j = 0; j < VL; ++j)
#pragma unroll
                            for (int w = 0; w < VW; ++w) vr[u][i][j][w] = 0u;
                    }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float w[2] = {vsc[u][0] == vref[0] ? ATT_BOOST : vsc[u][0] * vinv[0] * ATT_BOOST,
                                vsc[u][1] == vref[1] ? ATT_BOOST : vsc[u][1] * vinv[1] * ATT_BOOST};
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float mu = m[i & 1] == -INFINITY ? 0.0f : m[i & 1];     // a row that has seen no key yet
                const float e = ex2(s[u][i] - mu);
                l[i & 1] += e;
                x[i] = e * w[i & 1];
            }
            const uint32_t h0 = pack2<__half>(x[0], x[1]), h1 = pack2<__half>(x[2], x[3]);
            const uint32_t b0 = transpose8x8(h0), b1 = transpose8x8(h1);
            uint32_t c0 = 0u, c1 = 0u;
            if (TERMS == 2) {
                const float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&h0));
                const float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&h1));
                c0 = transpose8x8(pack2<__half>((x[0] - f0.x) * ATT_LOW, (x[1] - f0.y) * ATT_LOW));
                c1 = transpose8x8(pack2<__half>((x[2] - f1.x) * ATT_LOW, (x[3] - f1.y) * ATT_LOW));
            }
#pragma unroll
            for (int j = 0; j < VL; ++j)
#pragma unroll
                for (int w4 = 0; w4 < VW; ++w4)
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        // keys 2c, 2c+1 interleaved byte by byte, and keys 2c+8, 2c+9: two d of each
                        uint4 a;
                        codes_f16<CODE>(__byte_perm(vr[u][0][j][w4], vr[u][1][j][w4], hh ? 0x7362 : 0x5140), a.x, a.y);
                        codes_f16<CODE>(__byte_perm(vr[u][2][j][w4], vr[u][3][j][w4], hh ? 0x7362 : 0x5140), a.z, a.w);
                        const int t = (j * VW + w4) * 2 + hh;
                        if (TERMS == 2) {
                            float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};        // (rounded additions over the steps)
                            mma16816(x, a, c0, c1);
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[i] *= 1.0f / ATT_LOW;
                            mma16816(x, a, b0, b1);
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[t][i] += x[i];
                        } else mma16816(o[t], a, b0, b1);
                    }
        }
        if (nk < k1) load_v(nk);
    }

    // merge the warps: every warp's rows relative to its own maximum
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], b);
        if (g == 0) ml[warp][2 * c + h] = make_float2(m[h], l[h]);
    }
    __syncthreads();       // Q fragments are read no more
#pragma unroll
    for (int t = 0; t < OT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = (D == 64 ? 8 * g : (t / 8) * 128 + 16 * g) + 2 * (t % 8) + (i >> 1);
            mg[(warp * TM + 2 * c + (i & 1)) * RO + d] = o[t][i] * (1.0f / ATT_BOOST) * vref[i & 1];
        }
    __syncthreads();
    if (warp < fn) {
        const int r = warp;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < ATT_WARPS; ++w) mm = fmaxf(mm, ml[w][r].x);
        const float mu = mm == -INFINITY ? 0.0f : mm;
        float sum = 0.0f, f[ATT_WARPS];
#pragma unroll
        for (int w = 0; w < ATT_WARPS; ++w) {
            f[w] = ex2(ml[w][r].x - mu);
            sum = fmaf(ml[w][r].y, f[w], sum);
        }
        const int fr = f0 + r;
        const int64_t slot = (tile * p.splits + split) * TM + r;
        if (parts > 1 && lane == 0) p.part_ml[slot] = make_float2(mm, sum);
        const float inv = 1.0f / sum;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int d = lane + 32 * i;
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < ATT_WARPS; ++w) v = fmaf(mg[(w * TM + r) * RO + d], f[w], v);
            if (parts > 1) p.part_o[slot * D + d] = v;
            else store_out<T, D>(p, sr.r0 + fr / p.G, kvh * p.G + fr % p.G, d, v * inv);
        }
    }
}

// joins the splits of a tile: grid (rows of a tile, tile, seq * kv_heads + kv head), four
// warps that take the splits in turn
constexpr int COMBINE_THREADS = 128;
template <typename T, int D>
__global__ void __launch_bounds__(COMBINE_THREADS) kv8_combine_kernel(const AttnParams p) {
    constexpr int E = D / 32;                  // outputs per lane
    __shared__ float acc[4][D];
    __shared__ float factor[ATT_MAX_SPLITS], norm;
    dependency_trigger();
    dependency_wait();
    const int r = blockIdx.x, mt = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int KVH = p.H / p.G;
    const int seq = blockIdx.z / KVH, kvh = blockIdx.z - seq * KVH;
    const SeqRows sr = seq_rows(p.row_start, p.past, seq, p.rows, p.max_rows, p.max_seq, p.err);
    const int f0 = mt * p.tile_rows, f = f0 + r, fn = min(p.tile_rows, sr.n * p.G - f0);
    if (r >= fn) return;
    const int parts = tile_parts((sr.past + (f0 + fn - 1) / p.G + p.step_keys) / p.step_keys, p.splits);
    if (parts == 1) return;                    // (written by the attention itself)
    const int64_t tile = (int64_t)blockIdx.z * gridDim.y + mt;
    const int64_t slot0 = tile * p.splits * p.tile_rows + r;
    if (warp == 0) {
        float2 a[ATT_MAX_SPLITS / 32];
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int i = 0; i < ATT_MAX_SPLITS / 32; ++i) {
            const int s = lane + 32 * i;
            a[i] = s < parts ? p.part_ml[slot0 + (int64_t)s * p.tile_rows] : make_float2(-INFINITY, 0.0f);
            m = fmaxf(m, a[i].x);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < ATT_MAX_SPLITS / 32; ++i) {
            const float e = ex2(a[i].x - mu);
            factor[lane + 32 * i] = e;
            l = fmaf(a[i].y, e, l);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane == 0) norm = l;
    }
    __syncthreads();
    float v[E] = {};
#pragma unroll 4
    for (int s = warp; s < parts; s += 4) {
        const float *src = p.part_o + (slot0 + (int64_t)s * p.tile_rows) * D + lane * E;
        const float e = factor[s];
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const float2 u = *reinterpret_cast<const float2 *>(src + i);
            v[i] = fmaf(u.x, e, v[i]);
            v[i + 1] = fmaf(u.y, e, v[i + 1]);
        }
    }
#pragma unroll
    for (int i = 0; i < E; ++i) acc[warp][lane * E + i] = v[i];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += COMBINE_THREADS)
        store_out<T, D>(p, sr.r0 + f / p.G, kvh * p.G + f % p.G, d, ((acc[0][d] + acc[1][d]) + (acc[2][d] + acc[3][d])) / norm);
}

struct AttnPlan { int tile_rows, step_keys, mtiles, splits; int64_t tiles; size_t ml_bytes, o_bytes; };

// tiles of 8 (row, head) pairs where a sequence has no more, else of 16.  splits: six CTAs for
// every SM where the tiles alone are fewer, so that sequences of different lengths even out; at
// least one step of every warp each
AttnPlan attn_plan(const q35_kv8_cache &c, int32_t heads, int32_t max_rows) {
    AttnPlan pl;
    const int G = heads / c.kv_heads, D = c.head_dim;
    pl.tile_rows = (int64_t)max_rows * G <= 8 ? 8 : ATT_M;
    pl.step_keys = D == 64 ? 32 : 16;
    pl.mtiles = (int)ceil_div((int64_t)max_rows * G, pl.tile_rows);
    pl.tiles = (int64_t)pl.mtiles * c.seqs * c.kv_heads;
    const int64_t keys = (int64_t)ATT_WARPS * pl.step_keys;
    pl.splits = (int)std::max<int64_t>(
        1, std::min<int64_t>({ATT_MAX_SPLITS, 6 * 148 / std::max<int64_t>(1, pl.tiles), c.max_seq / keys}));
    const int64_t slots = pl.splits > 1 ? pl.tiles * pl.splits * pl.tile_rows : 0;
    pl.ml_bytes = (size_t)round_up(slots * (int64_t)sizeof(float2), 256);
    pl.o_bytes = (size_t)slots * c.head_dim * sizeof(float);
    return pl;
}

template <typename T, int CODE, int D>
int launch_attn(const AttnParams &p, const AttnPlan &pl, int zs, cudaStream_t s) {
    constexpr int terms = std::is_same<T, float>::value ? 2 : 1;
    static_assert(AttnShape<D>::KC == (D == 64 ? 32 : 16) && Attn8Shape<D>::KC == AttnShape<D>::KC, "attn_plan's steps");
    const bool small = pl.tile_rows == 8;
    auto kern = small ? kv8_attn8_kernel<T, CODE, D> : kv8_attn_kernel<T, CODE, D>;
    const size_t smem = small ? attn8_smem<D>(terms) : attn_smem<D>(terms);
    static bool configured[64][2] = {};
    int dev = 0;
    Q35_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev][small]) {
        Q35_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (dev >= 0 && dev < 64) configured[dev][small] = true;
    }
    Q35_CUDA_TRY(launch_dependent(kern, dim3(pl.splits, pl.mtiles, zs), ATT_THREADS, smem, s, 1, p));
    if (pl.splits > 1)
        Q35_CUDA_TRY(launch_dependent(kv8_combine_kernel<T, D>, dim3(pl.tile_rows, pl.mtiles, zs), COMBINE_THREADS, 0, s, 1, p));
    return Q35_OK;
}

template <typename T, int CODE>
int launch_attn(const AttnParams &p, const AttnPlan &pl, int D, int zs, cudaStream_t s) {
    if (D == 64) return launch_attn<T, CODE, 64>(p, pl, zs, s);
    if (D == 128) return launch_attn<T, CODE, 128>(p, pl, zs, s);
    return launch_attn<T, CODE, 256>(p, pl, zs, s);
}
template <typename T>
int launch_attn(const AttnParams &p, const AttnPlan &pl, int code, int D, int zs, cudaStream_t s) {
    return code == Q35_CODE_INT8 ? launch_attn<T, Q35_CODE_INT8>(p, pl, D, zs, s) : launch_attn<T, Q35_CODE_E4M3>(p, pl, D, zs, s);
}

template <typename T, int CODE, int D>
int launch_append_b(const AppendParams &p, int block, dim3 grid, cudaStream_t s) {
    auto kern = block == 16   ? kv8_append_kernel<T, CODE, D, 16>
                : block == 32 ? kv8_append_kernel<T, CODE, D, 32>
                : block == 64 ? kv8_append_kernel<T, CODE, D, 64>
                              : kv8_append_kernel<T, CODE, D, 128>;
    Q35_CUDA_TRY(launch_dependent(kern, grid, APPEND_THREADS, 0, s, 1, p));
    return Q35_OK;
}
template <typename T, int CODE>
int launch_append_d(const AppendParams &p, int D, int block, dim3 grid, cudaStream_t s) {
    if (D == 64) return launch_append_b<T, CODE, 64>(p, block, grid, s);
    if (D == 128) return launch_append_b<T, CODE, 128>(p, block, grid, s);
    return launch_append_b<T, CODE, 256>(p, block, grid, s);
}
template <typename T>
int launch_append_c(const AppendParams &p, int code, int D, int block, dim3 grid, cudaStream_t s) {
    return code == Q35_CODE_INT8 ? launch_append_d<T, Q35_CODE_INT8>(p, D, block, grid, s)
                                 : launch_append_d<T, Q35_CODE_E4M3>(p, D, block, grid, s);
}

int nblk(const q35_kv8_cache &c) { return (int)ceil_div(c.max_seq, c.block); }
int64_t seq_stride(const q35_kv8_cache &c) {
    return c.seq_stride ? c.seq_stride : (int64_t)c.kv_heads * c.max_seq * c.head_dim;
}
int64_t scale_seq_stride(const q35_kv8_cache &c) {
    return c.scale_seq_stride ? c.scale_seq_stride : (int64_t)c.kv_heads * nblk(c);
}

int check_rows(const q35_kv8_cache &c, const Kv8Rows &r) {
    if (r.rows < 0 || r.max_rows < 0 || r.max_rows > r.rows)
        return set_error(Q35_ERR_INVALID, "kv8: rows and max_rows must satisfy 0 <= max_rows <= rows");
    if (r.rows > 0 && r.max_rows == 0) return set_error(Q35_ERR_INVALID, "kv8: max_rows is 0");
    if (r.max_rows > c.max_seq) return set_error(Q35_ERR_INVALID, "kv8: more rows than the cache has positions");
    if (r.rows > 0 && (!r.row_start || !r.past)) return set_error(Q35_ERR_INVALID, "kv8: NULL row table");
    return Q35_OK;
}

int check_heads(const q35_kv8_cache &c, int32_t heads) {
    if (heads < 1 || heads % c.kv_heads)
        return set_error(Q35_ERR_INVALID, "kv8_attention: heads must be a multiple of kv_heads");
    return Q35_OK;
}
// the kernels count a sequence's (row, head) pairs of a kv head in 32 bits
int check_pairs(const q35_kv8_cache &c, int32_t heads, int32_t max_rows) {
    if ((int64_t)max_rows * (heads / c.kv_heads) > INT32_MAX - 128)
        return set_error(Q35_ERR_INVALID, "kv8_attention: max_rows * heads / kv_heads above 2^31 - 129");
    return Q35_OK;
}

}  // namespace

int kv8_check(const q35_kv8_cache *c) {
    if (!c) return set_error(Q35_ERR_INVALID, "kv8: cache is NULL");
    int st = check_code(c->code);
    if (st) return st;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return set_error(Q35_ERR_INVALID, "kv8: head_dim must be 64, 128 or 256");
    if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
        return set_error(Q35_ERR_INVALID, "kv8: block must be 16, 32, 64 or 128 tokens");
    if (c->seqs < 1 || c->kv_heads < 1 || c->max_seq < 1) return set_error(Q35_ERR_INVALID, "kv8: non-positive size");
    if ((int64_t)c->seqs * c->kv_heads > 32767) return set_error(Q35_ERR_INVALID, "kv8: more than 32767 sequences x kv heads");
    if (c->max_seq > (1 << 30)) return set_error(Q35_ERR_INVALID, "kv8: max_seq above 2^30");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return set_error(Q35_ERR_INVALID, "kv8: NULL cache array");
    if (!aligned_to(c->k, 16) || !aligned_to(c->v, 16) || seq_stride(*c) % 16)
        return set_error(Q35_ERR_INVALID, "kv8: codes must start on 16-byte boundaries");
    if (!aligned_to(c->k_scale, 4) || !aligned_to(c->v_scale, 4))
        return set_error(Q35_ERR_INVALID, "kv8: scales are not aligned");
    if (c->seqs > 1 && (seq_stride(*c) < (int64_t)c->kv_heads * c->max_seq * c->head_dim ||
                        scale_seq_stride(*c) < (int64_t)c->kv_heads * nblk(*c)))
        return set_error(Q35_ERR_INVALID, "kv8: a sequence stride is below a sequence's size");
    return Q35_OK;
}

int launch_kv8_append(const q35_kv8_cache &c, int dtype, const void *k, const void *v, int64_t ld, const Kv8Rows &r,
                      int *err, cudaStream_t s) {
    if (r.rows == 0) return Q35_OK;
    AppendParams p;
    p.x[0] = k; p.x[1] = v;
    p.codes[0] = static_cast<uint8_t *>(c.k); p.codes[1] = static_cast<uint8_t *>(c.v);
    p.scales[0] = c.k_scale; p.scales[1] = c.v_scale;
    p.ld = ld;
    p.seq_stride = seq_stride(c); p.scale_seq_stride = scale_seq_stride(c);
    p.row_start = r.row_start; p.past = r.past;
    p.rows = r.rows; p.max_rows = r.max_rows;
    p.G = c.kv_heads; p.max_seq = c.max_seq; p.nblk = nblk(c);
    p.vec = aligned_to(k, 16) && aligned_to(v, 16) && ld * (int64_t)dtype_size(dtype) % 16 == 0;
    p.err = err;
    // blocks a run of max_rows tokens can touch, wherever it starts
    const int bx = (int)((r.max_rows + (int64_t)c.block - 2) / c.block + 1);
    const dim3 grid((unsigned)bx, (unsigned)c.kv_heads, (unsigned)(2 * c.seqs));
    switch (dtype) {
    case Q35_DT_F32: return launch_append_c<float>(p, c.code, c.head_dim, c.block, grid, s);
    case Q35_DT_BF16: return launch_append_c<__nv_bfloat16>(p, c.code, c.head_dim, c.block, grid, s);
    default: return launch_append_c<__half>(p, c.code, c.head_dim, c.block, grid, s);
    }
}

size_t kv8_attention_workspace(const q35_kv8_cache &c, int32_t heads, int32_t rows, int32_t max_rows) {
    if (rows <= 0 || kv8_prompt_takes(c, heads, max_rows)) return 0;
    const AttnPlan pl = attn_plan(c, heads, max_rows);
    return pl.ml_bytes + pl.o_bytes;
}

size_t kv8_workspace_bound(const q35_kv8_cache &c, int32_t heads) {
    // tiles * splits is at most 6 * 148 wherever a tile is split at all (attn_plan)
    (void)heads;
    return (size_t)6 * 148 * ATT_M * (sizeof(float2) + sizeof(float) * (size_t)c.head_dim) + 256;
}

int launch_kv8_attention(const q35_kv8_cache &c, int dtype, const void *q, int64_t ldq, int32_t heads, void *out,
                         int64_t ldo, int8_t *out_q, const Kv8Rows &r, float scale, void *workspace, int *err,
                         cudaStream_t s) {
    if (r.rows == 0) return Q35_OK;
    const bool prompt = kv8_prompt_takes(c, heads, r.max_rows);
    const AttnPlan pl = attn_plan(c, heads, r.max_rows);
    AttnParams p;
    p.q = q; p.out = out; p.out_q = out_q;
    p.k = static_cast<const uint8_t *>(c.k); p.v = static_cast<const uint8_t *>(c.v);
    p.ks = c.k_scale; p.vs = c.v_scale;
    p.ldq = ldq; p.ldo = ldo;
    p.seq_stride = seq_stride(c); p.scale_seq_stride = scale_seq_stride(c);
    p.row_start = r.row_start; p.past = r.past;
    p.rows = r.rows; p.max_rows = r.max_rows;
    p.H = heads; p.G = heads / c.kv_heads; p.max_seq = c.max_seq; p.nblk = nblk(c);
    p.splits = pl.splits; p.tile_rows = pl.tile_rows; p.step_keys = pl.step_keys;
    p.block_shift = c.block == 16 ? 4 : c.block == 32 ? 5 : c.block == 64 ? 6 : 7;
    p.scale = scale;
    p.part_ml = static_cast<float2 *>(workspace);
    p.part_o = reinterpret_cast<float *>(static_cast<char *>(workspace) + pl.ml_bytes);
    p.err = err;
    const int zs = c.seqs * c.kv_heads;
    if (prompt) return launch_kv8_prompt(p, dtype, c.code, c.head_dim, zs, s);
    // (tiles along grid.y: fewer than 32 of 128 pairs)
    switch (dtype) {
    case Q35_DT_F32: return launch_attn<float>(p, pl, c.code, c.head_dim, zs, s);
    case Q35_DT_BF16: return launch_attn<__nv_bfloat16>(p, pl, c.code, c.head_dim, zs, s);
    default: return launch_attn<__half>(p, pl, c.code, c.head_dim, zs, s);
    }
}

}  // namespace q35

using namespace q35;

extern "C" {

int q35_kv8_append_dev(q35_ctx ctx, const q35_kv8_cache *cache, int dtype, const void *k, const void *v, int64_t ld,
                       const int32_t *row_start, const int32_t *past, int32_t rows, int32_t max_rows) {
    if (!ctx) return set_error(Q35_ERR_INVALID, "kv8_append: ctx is NULL");
    int st = kv8_check(cache);
    if (!st) st = check_dtype(dtype);
    if (st) return st;
    const Kv8Rows r{row_start, past, rows, max_rows};
    st = check_rows(*cache, r);
    if (st) return st;
    if (rows == 0) return Q35_OK;
    if (!k || !v) return set_error(Q35_ERR_INVALID, "kv8_append: NULL argument");
    if (ld < (int64_t)cache->kv_heads * cache->head_dim)
        return set_error(Q35_ERR_INVALID, "kv8_append: the row stride is below kv_heads * head_dim");
    if (!aligned_to(k, dtype_size(dtype)) || !aligned_to(v, dtype_size(dtype)))
        return set_error(Q35_ERR_INVALID, "kv8_append: a pointer is not aligned to its elements");
    DeviceGuard g(ctx->device);
    st = ensure_workspace(ctx, 0, 0);
    if (st) return st;
    return launch_kv8_append(*cache, dtype, k, v, ld, r, ctx->ws.err, ctx->stream);
}

int64_t q35_kv8_attention_workspace(const q35_kv8_cache *cache, int32_t heads, int32_t rows, int32_t max_rows) {
    if (kv8_check(cache)) return -1;
    const int32_t dummy = 0;
    if (check_heads(*cache, heads) || check_rows(*cache, Kv8Rows{&dummy, &dummy, rows, max_rows}) ||
        check_pairs(*cache, heads, max_rows))
        return -1;
    return (int64_t)kv8_attention_workspace(*cache, heads, rows, max_rows);
}

int q35_kv8_attention_dev(q35_ctx ctx, const q35_kv8_cache *cache, int dtype, const void *q, int64_t ldq,
                          int32_t heads, void *out, int64_t ldo, const int32_t *row_start, const int32_t *past,
                          int32_t rows, int32_t max_rows, float scale, void *workspace, size_t workspace_bytes) {
    if (!ctx) return set_error(Q35_ERR_INVALID, "kv8_attention: ctx is NULL");
    int st = kv8_check(cache);
    if (!st) st = check_dtype(dtype);
    if (st) return st;
    st = check_heads(*cache, heads);
    const Kv8Rows r{row_start, past, rows, max_rows};
    if (!st) st = check_rows(*cache, r);
    if (!st) st = check_pairs(*cache, heads, max_rows);
    if (st) return st;
    if (rows == 0) return Q35_OK;
    if (!q || !out) return set_error(Q35_ERR_INVALID, "kv8_attention: NULL argument");
    const int64_t width = (int64_t)heads * cache->head_dim;
    if (ldq < width || ldo < width) return set_error(Q35_ERR_INVALID, "kv8_attention: a row stride is below heads * head_dim");
    if (!aligned_to(q, dtype_size(dtype)) || !aligned_to(out, dtype_size(dtype)))
        return set_error(Q35_ERR_INVALID, "kv8_attention: a pointer is not aligned to its elements");
    if (!(scale == scale) || scale > 3.402823466e38f || scale < -3.402823466e38f)
        return set_error(Q35_ERR_INVALID, "kv8_attention: scale is not finite");
    const size_t need = kv8_attention_workspace(*cache, heads, rows, max_rows);
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned_to(workspace, 16)))
        return set_error(Q35_ERR_INVALID, "kv8_attention: workspace missing, too small or not 16-byte aligned");
    DeviceGuard g(ctx->device);
    st = ensure_workspace(ctx, 0, 0);
    if (st) return st;
    return launch_kv8_attention(*cache, dtype, q, ldq, heads, out, ldo, nullptr, r, scale, workspace, ctx->ws.err,
                                ctx->stream);
}

}  // extern "C"
