// q35_sample_filtered.cu -- sampling with temperature, top-k, top-p and min-p together, each
// row with its own parameters and its own uniform draw, for any vocabulary up to 2^22.
//
//   z_i = (l_i - max l) / T,  w_i = e^{z_i}                    (T <= 0: the first maximum)
//   the k largest logits (equal ones: lowest index first);
//   of those, in descending order, the shortest prefix whose mass reaches p times theirs;
//   of those, the ones with w_i >= min_p;
//   the token is the first kept index whose running mass (in index order) passes u * mass.
//
// w is formed in binary64 (a difference of logits is exact there; within 2^-44) and summed as
// integers of 2^-40, so that sums, histograms and prefix sums are exact, independent of
// their order, and a draw next to a border falls on the same side as in binary64.
// Cut-offs come from a radix descent over the order-preserving 32-bit keys of the logits
// (counts for top-k, masses for top-p), not from a sort.
#include <cfloat>

#include "q35_q8.cuh"

namespace q35 {
namespace {

constexpr int FT = 1024;                  // threads per row
constexpr int FW = FT / 32;
constexpr int FMAXV = 1 << 22;            // 2^22 weights of at most 2^40
constexpr double FSCALE = 1099511627776.0;   // 2^40
constexpr unsigned KEY_NONE = 0x007fffffu;   // key of -infinity: masked entries (NaN counts as one)

using u64 = unsigned long long;

struct FilteredParams {
    const void *logits;
    int64_t ld;
    int32_t V;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *tokens;
    float *probs;
};

struct FShared {
    u64 hist[256];
    u64 wsum[FW];
    unsigned redu[FW];
    int redi[FW];
    unsigned lo, hi;
    u64 carry;
    int hit;
};

__device__ __forceinline__ unsigned key_of(float f) {
    if (f != f) return KEY_NONE;
    f += 0.0f;                            // -0 and +0 are equal logits
    const unsigned b = __float_as_uint(f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

template <typename T> struct Row {
    const T *p;
    int V;
    double mx, invT;                      // of the row; T > 0
    float mxf;
    __device__ __forceinline__ unsigned key(int i) const { return key_of(to_f32<T>(p[i])); }
    __device__ __forceinline__ double weight(unsigned k) const {
        if (k <= KEY_NONE) return 0.0;
        const float l = key_value(k);
        if (l == mxf) return 1.0;          // also for +infinity
        return exp(((double)l - mx) * invT);
    }
    __device__ __forceinline__ u64 mass(unsigned k) const { return (u64)__double2ull_rn(weight(k) * FSCALE); }
};

__device__ unsigned block_max_u(FShared &sh, unsigned v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) sh.redu[threadIdx.x >> 5] = v;
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, sh.redu[threadIdx.x & 31]);
    __syncthreads();
    return v;
}
__device__ int block_min_i(FShared &sh, int v) {
    v = __reduce_min_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) sh.redi[threadIdx.x >> 5] = v;
    __syncthreads();
    v = __reduce_min_sync(0xffffffffu, sh.redi[threadIdx.x & 31]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ u64 block_sum(FShared &sh, u64 v) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) sh.wsum[threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_sum(sh.wsum[threadIdx.x & 31]);
    __syncthreads();
    return v;
}

// the largest key v in [lo, hi] whose weight W(v) = sum of w(key) over the entries with
// key >= v reaches target (W(lo) >= target >= 1, nothing above hi); *above = W of the keys
// greater than v
template <typename T, typename WF>
__device__ unsigned descend(FShared &sh, const Row<T> &row, unsigned lo, unsigned hi, u64 target, WF w, u64 *above) {
    const int t = threadIdx.x;
    u64 carry = 0;
    for (int level = 0; lo < hi && level < 8; ++level) {      // at most 5: each level leaves 1/128 of the range
        const unsigned range = hi - lo;
        int sft = 0;
        while ((range >> sft) >= 256u) ++sft;
        const int nb = (int)(range >> sft) + 1;
        for (int i = t; i < 256; i += FT) sh.hist[i] = 0;
        __syncthreads();
        for (int i = t; i < row.V; i += FT) {
            const unsigned k = row.key(i);
            if (k >= lo && k <= hi) atomicAdd(&sh.hist[(k - lo) >> sft], w(k));
        }
        __syncthreads();
        if (t < 32) {
            u64 m[8], mine = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int d = nb - 1 - 8 * t - i;
                m[i] = d >= 0 ? sh.hist[d] : 0;
                mine += m[i];
            }
            u64 incl = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const u64 n = __shfl_up_sync(0xffffffffu, incl, o);
                if (t >= o) incl += n;
            }
            u64 c = carry + incl - mine;
            if (c < target && carry + incl >= target) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int d = nb - 1 - 8 * t - i;
                    if (d >= 0 && c + m[i] >= target) {
                        const unsigned b0 = lo + ((unsigned)d << sft);
                        sh.lo = b0;
                        sh.hi = min(hi, b0 + ((1u << sft) - 1u));
                        sh.carry = c;
                        break;
                    }
                    c += m[i];
                }
            }
        }
        __syncthreads();
        lo = sh.lo;
        hi = sh.hi;
        carry = sh.carry;
        __syncthreads();
    }
    *above = carry;
    return lo;
}

template <typename T>
__global__ void __launch_bounds__(FT, 1) sample_filtered_kernel(const FilteredParams p) {
    __shared__ FShared sh;
    const int r = blockIdx.x, t = threadIdx.x, warp = t >> 5, lane = t & 31;
    Row<T> row;
    row.p = static_cast<const T *>(p.logits) + (int64_t)r * p.ld;
    row.V = p.V;
    unsigned kmax = 0, kmin = 0;          // kmin as the largest complement, of the entries that count
    for (int i = t; i < p.V; i += FT) {
        const unsigned k = row.key(i);
        kmax = max(kmax, k);
        if (k > KEY_NONE) kmin = max(kmin, ~k);
    }
    kmax = block_max_u(sh, kmax);
    kmin = ~block_max_u(sh, kmin);
    if (kmax <= KEY_NONE) {               // every logit is masked
        if (t == 0) {
            p.tokens[r] = 0;
            if (p.probs) p.probs[r] = 0.0f;
        }
        return;
    }
    const float Tf = p.temperature ? p.temperature[r] : 1.0f;
    const float pf = p.top_p ? p.top_p[r] : 1.0f, mf = p.min_p ? p.min_p[r] : 0.0f;
    const int k = p.top_k ? p.top_k[r] : 0;
    if (!(Tf > 0.0f) || k == 1 || !(mf <= 1.0f) || !(pf > 0.0f)) {
        // only the first maximum is kept
        int first = p.V;
        for (int i = t; i < p.V; i += FT)
            if (row.key(i) == kmax) { first = i; break; }
        first = block_min_i(sh, first);
        if (t == 0) {
            p.tokens[r] = first + 1;
            if (p.probs) p.probs[r] = 1.0f;
        }
        return;
    }
    row.mxf = key_value(kmax);
    row.mx = (double)row.mxf;
    row.invT = 1.0 / (double)Tf;

    // top-k: keys above `cut`, and the first `ties` entries equal to it
    unsigned cut = kmin;
    u64 ties = (u64)p.V;
    if (k > 0 && k < p.V) {
        u64 n = 0;
        for (int i = t; i < p.V; i += FT) n += row.key(i) > KEY_NONE ? 1 : 0;
        n = block_sum(sh, n);
        if ((u64)k < n) {
            u64 above;
            cut = descend(sh, row, kmin, kmax, (u64)k, [](unsigned) { return (u64)1; }, &above);
            ties = (u64)k - above;
        }
    }
    // top-p over what top-k kept
    if (pf < 1.0f) {
        u64 z = 0, eq = 0;
        for (int i = t; i < p.V; i += FT) {
            const unsigned key = row.key(i);
            if (key > cut) z += row.mass(key);
            else if (key == cut) ++eq;
        }
        z = block_sum(sh, z);
        eq = block_sum(sh, eq);
        eq = eq < ties ? eq : ties;
        const u64 wc = row.mass(cut);
        z += eq * wc;
        u64 target = (u64)ceil((double)pf * (double)z);
        target = target < 1 ? 1 : target > z ? z : target;
        u64 above;
        // (entries equal to the cut count with their kept share: they are the lowest)
        const u64 over = z - eq * wc;
        if (target <= over) {
            const unsigned v = descend(sh, row, cut, kmax, target, [&](unsigned q) { return q > cut ? row.mass(q) : (u64)0; }, &above);
            const u64 wv = row.mass(v);
            ties = (target - above + wv - 1) / wv;
            cut = v;
        } else if (wc > 0) {
            ties = min(eq, (target - over + wc - 1) / wc);
        }
    }
    // min-p
    const double floor_w = (double)mf;
    // kept mass of each warp's contiguous segment, the ties taken in index order
    const int seg = (int)round_up(ceil_div(p.V, FW), 32);
    const int s0 = min(p.V, warp * seg), s1 = min(p.V, s0 + seg);
    u64 wm = 0, we = 0;
    for (int i = s0 + lane; i < s1; i += 32) {
        const unsigned key = row.key(i);
        if (key == cut) ++we;
        else if (key > cut && row.weight(key) >= floor_w) wm += row.mass(key);
    }
    wm = warp_sum(wm);
    we = warp_sum(we);
    const u64 wcut = row.weight(cut) >= floor_w ? row.mass(cut) : 0;
    if (lane == 0) { sh.wsum[warp] = we; sh.hist[warp] = wm; }
    __syncthreads();
    u64 run = 0, eqs = 0, mine0 = 0, eq0 = 0;
    for (int w = 0; w < FW; ++w) {
        if (w == warp) { mine0 = run; eq0 = eqs; }
        const u64 e1 = min(ties, eqs + sh.wsum[w]);
        run += sh.hist[w] + (e1 - min(ties, eqs)) * wcut;
        eqs += sh.wsum[w];
    }
    const u64 total = run;
    const float uf = p.u[r];
    if (!(uf > 0.0f)) {
        // the first kept index of any mass, also one that rounds to no unit of 2^-40 (the first
        // entry equal to the cut is always kept)
        int first = p.V;
        for (int i = t; i < p.V; i += FT) {
            const unsigned key = row.key(i);
            if (key < cut) continue;
            const double w = row.weight(key);
            if (w > 0.0 && w >= floor_w) { first = i; break; }
        }
        first = block_min_i(sh, first);
        if (t == 0) {
            p.tokens[r] = first + 1;
            if (p.probs) p.probs[r] = (float)(row.weight(row.key(first)) * FSCALE / (double)total);
        }
        return;
    }
    u64 goal = (u64)((double)uf * (double)total) + 1;    // the running mass that passes u * mass
    if (goal > total) goal = total;
    // the segment that holds the goal walks it in index order
    const u64 e1 = min(ties, eq0 + we);
    const u64 mine1 = mine0 + wm + (e1 - min(ties, eq0)) * wcut;
    if (mine0 < goal && goal <= mine1) {
        u64 c = mine0, ec = eq0;
        for (int i0 = s0; i0 < s1; i0 += 32) {
            const int i = i0 + lane;
            const unsigned key = i < s1 ? row.key(i) : 0u;
            const unsigned eqm = __ballot_sync(0xffffffffu, i < s1 && key == cut);
            const u64 rank = ec + __popc(eqm & ((1u << lane) - 1u));
            u64 w = 0;
            if (i < s1) {
                if (key == cut) w = rank < ties ? wcut : 0;
                else if (key > cut && row.weight(key) >= floor_w) w = row.mass(key);
            }
            u64 incl = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 n = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += n;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, w > 0 && c + incl >= goal);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    p.tokens[r] = i + 1;
                    if (p.probs) p.probs[r] = (float)(row.weight(key) * FSCALE / (double)total);
                }
                break;
            }
            c += __shfl_sync(0xffffffffu, incl, 31);
            ec += __popc(eqm);
        }
    }
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int q35_sample_filtered_dev(q35_ctx ctx, int dtype, const void *logits, int64_t ld, int32_t rows,
                                       int32_t vocab, const float *temperature, const int32_t *top_k,
                                       const float *top_p, const float *min_p, const float *u, int32_t *tokens,
                                       float *probs) {
    if (!ctx) return set_error(Q35_ERR_INVALID, "sample_filtered: ctx is NULL");
    int st = check_dtype(dtype);
    if (st) return st;
    if (rows < 0) return set_error(Q35_ERR_INVALID, "sample_filtered: negative row count");
    if (vocab < 1 || vocab > FMAXV) return set_error(Q35_ERR_INVALID, "sample_filtered: vocabulary must be 1..4194304");
    if (rows == 0) return Q35_OK;
    if (!logits || !u || !tokens) return set_error(Q35_ERR_INVALID, "sample_filtered: NULL argument");
    if (ld < vocab) return set_error(Q35_ERR_INVALID, "sample_filtered: the row stride is below the vocabulary");
    if (!aligned_to(logits, dtype_size(dtype)) || !aligned_to(temperature, 4) || !aligned_to(top_k, 4) ||
        !aligned_to(top_p, 4) || !aligned_to(min_p, 4) || !aligned_to(u, 4) || !aligned_to(tokens, 4) || !aligned_to(probs, 4))
        return set_error(Q35_ERR_INVALID, "sample_filtered: a pointer is not aligned to its elements");
    DeviceGuard g(ctx->device);
    FilteredParams p;
    p.logits = logits; p.ld = ld; p.V = vocab;
    p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
    p.u = u; p.tokens = tokens; p.probs = probs;
    switch (dtype) {
    case Q35_DT_F32: sample_filtered_kernel<float><<<rows, FT, 0, ctx->stream>>>(p); break;
    case Q35_DT_BF16: sample_filtered_kernel<__nv_bfloat16><<<rows, FT, 0, ctx->stream>>>(p); break;
    default: sample_filtered_kernel<__half><<<rows, FT, 0, ctx->stream>>>(p); break;
    }
    Q35_CUDA_TRY(cudaGetLastError());
    return Q35_OK;
}
