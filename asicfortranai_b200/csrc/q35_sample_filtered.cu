// q35_sample_filtered.cu -- sampling with temperature, top-k, top-p and min-p together, each
// row with its own parameters and its own uniform draw, for any vocabulary up to 401,408.
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
//
// One cluster of 1 to 8 CTAs per row, each holding a contiguous slice of the row in shared
// memory, so a row is read once.  No sort: the cut-offs of top-k (counts) and top-p (masses)
// come from a histogram over 1024 equal steps of the logit below the maximum.  Masses enter it
// as three pieces of 14 bits, which native 32-bit shared-memory additions sum exactly.  Then
// every warp drops the entries below the step that holds the cut from its segment (in place, in
// order), and the entries of that step (a few tens as a rule) are ranked directly by every CTA;
// where they are too many (long runs of equal or close logits) further histograms take 10 bits
// of the key at a time.  The masses of what is kept are then summed over what is left.  The draw
// finds its CTA, its warp's segment and its 32 entries by exact prefix sums, and the entry's index by
// its rank among the kept ones of its segment.
//
// CTAs exchange by remote stores ahead of a cluster barrier, after which all that is read is local
// (24 remote loads by every thread had cost 2900 to 5400 clocks at each exchange): totals, the
// sums of 32 groups of 32 bins, the entries of one bin.  Only the bins of the group that holds
// the cut are loaded from the other CTAs, by one warp.
//
// Bound by the exponentials (15 binary64 operations and about as many integer ones an entry)
// where nothing cuts the vocabulary first, and by barrier latency for one row.  Measured: 64 rows
// of 100,277 62 us (26 MB, 4 us of HBM; of a top-p row's 97 k clocks 23 k are exponentials, 22 k
// the histogram of masses, 9 k each loading and dropping), one row of 32,000 14 us.
#include <cfloat>

#include "q35_q8.cuh"

namespace q35 {
namespace {

constexpr int FT = 512;                   // threads per CTA (what every warp repeats costs a quarter of
                                          // the warps' number of clocks per instruction: 1024 were slower)
constexpr int FW = FT / 32;
constexpr int FMAXC = 8;                  // CTAs per row (the portable cluster size)
constexpr int FNB = 1024;                 // histogram bins: 32 groups of 32
constexpr int FLIST = 1024;               // entries of the cut's bin ranked directly (all CTAs)
constexpr int FRES = 50176;               // entries a CTA keeps in shared memory (196 KB); sums of that
                                          // many 14-bit pieces fit 32 bits
constexpr int FMAXV = FMAXC * FRES;
constexpr double FSCALE = 1099511627776.0;   // 2^40

using u64 = unsigned long long;

struct FilteredParams {
    const void *logits;
    int64_t ld;
    int32_t V, C;                         // CTAs per row
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *tokens;
    float *probs;
};

// what the CTAs of a row exchange: slot q of an array is CTA q's, stored there by CTA q in
// every CTA's copy.  Each array is used once between barriers that separate the uses.
struct FPublic {
    unsigned hist[3][FNB];                // this CTA's histogram
    u64 group[FMAXC][32];                 // sums of 32 neighbouring bins
    u64 lmass[FLIST];                     // the cut's bin: CTA q's entries from q * FLIST / C on,
    float lval[FLIST];                    // then all of them in a row (flat)
    unsigned lcount[FMAXC];
    u64 top[FMAXC];                       // (largest key, lowest index)
    unsigned low[FMAXC], n[FMAXC], n_inf[FMAXC];   // complement of the smallest counting key, counting entries
    u64 mass[2][FMAXC], eq[2][FMAXC];
    int first[FMAXC];
};
struct FShared {
    FPublic pub;
    double table[16];                     // 2^(j/16)
    u64 scan[FW];
    u64 wmass[FW], weq[FW];
    u64 found_above;
    unsigned found;
    unsigned appended;
    int loff[FMAXC];
    unsigned fine[3 * FMAXC][32];
    int holder, at;
    u64 hmass, heq;
};

// order-preserving image of a logit (no NaN; -0 and +0 alike) and back
__device__ __forceinline__ unsigned key_of(float f) {
    f += 0.0f;
    const unsigned b = __float_as_uint(f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// NaN counts as masked
template <typename T> __device__ __forceinline__ float logit(const T *p) {
    const float f = to_f32<T>(*p);
    return f != f ? -INFINITY : f;
}
// 2^(j/16)
__constant__ double root16[16] = {
    1.0, 1.0442737824274138, 1.0905077326652577, 1.1387886347566916,
    1.189207115002721, 1.241857812073484, 1.2968395546510096, 1.3542555469368927,
    1.4142135623730951, 1.4768261459394993, 1.5422108254079407, 1.6104903319492543,
    1.681792830507429, 1.7562521603732995, 1.8340080864093424, 1.9152065613971474};
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// the address of this CTA's shared variable in CTA rank's shared memory
__device__ __forceinline__ uint32_t remote(const void *p, int rank) {
    uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ unsigned ld_remote(const unsigned *p, int rank) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void st_remote(const void *p, int rank, unsigned v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void st_remote(const void *p, int rank, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory");
}
// (three 32-bit reductions: shorter than five dependent pairs of shuffles)
__device__ __forceinline__ u64 warp_sum(u64 v) {
    const unsigned a = __reduce_add_sync(0xffffffffu, (unsigned)v & 0xffffffu);
    const unsigned b = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 24) & 0xffffffu);
    const unsigned c = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 48));
    return (u64)a + ((u64)b << 24) + ((u64)c << 48);
}
__device__ __forceinline__ u64 warp_max(u64 v) {
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(v >> 32) == hi ? (unsigned)v : 0u);
    return ((u64)hi << 32) | lo;
}
__device__ __forceinline__ u64 warp_scan(u64 v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
    }
    return v;
}

extern __shared__ float slice_values[];

// a row's weights
struct Weigh {
    double mx, c;                         // maximum (finite), 16 / (ln 2 * T)
    const double *table;

    // 2^40 w rounded to an integer; *scaled gets 2^40 w.  Table-driven exponential (Tang's
    // method): w = 2^(-s) * 2^(j/16) * 2^(f/16), |f| <= 1/2, the last factor by its series to
    // the sixth power (2^-51); 16 doubles fill the 32 banks once, so the look-up has no conflicts
    __device__ __forceinline__ u64 mass(float l, double *scaled) const {
        double t = ((double)l - mx) * c;
        t = t > -686.0 ? t : -686.0;                            // 2^-42.9: mass 0
        const double magic = 6755399441055744.0;                // 1.5 * 2^52: the sum's low bits are rint(t)
        const double tn = t + magic;
        const int n = __double2loint(tn);
        const double f = t - (tn - magic);
        // (ln2/16)^i / i!
        double q = 9.181219573844436e-12;
        q = fma(q, f, 1.271587195055813e-09);
        q = fma(q, f, 1.467610032291943e-07);
        q = fma(q, f, 1.3550807779497455e-05);
        q = fma(q, f, 9.383847928089871e-04);
        q = fma(q, f, 4.332169878499658e-02);
        q = fma(q, f, 1.0);
        const double v = q * table[n & 15];                     // within [0.97, 2.05)
        // times 2^(40 - s), s = -(n >> 4) in 0 .. 43
        const double r = __hiloint2double(__double2hiint(v) + ((n >> 4) + 40) * (1 << 20), __double2loint(v));
        *scaled = r;
        return (u64)__double_as_longlong(r + 4503599627370496.0) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 mass(float l) const {
        double r;
        return mass(l, &r);
    }
    // w in full range
    __device__ __forceinline__ double weight(float l) const {
        return l == -INFINITY ? 0.0 : exp(((double)l - mx) * c * 4.332169878499658e-02);
    }
};

__device__ __forceinline__ void hist_mass(unsigned (*h)[FNB], int bin, u64 w) {
    atomicAdd(&h[0][bin], (unsigned)w & 0x3fffu);
    atomicAdd(&h[1][bin], (unsigned)(w >> 14) & 0x3fffu);
    if (w >> 28) atomicAdd(&h[2][bin], (unsigned)(w >> 28));
}

// this CTA's sums of 32 neighbouring bins to every CTA (all threads; before a cluster barrier)
__device__ __forceinline__ void publish_groups(FShared &sh, int C, int rank) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
#pragma unroll
    for (int g = warp; g < FNB / 32; g += FW) {
        const int i = 32 * g + lane;
        const u64 s = warp_sum(sh.pub.hist[0][i] + ((u64)sh.pub.hist[1][i] << 14) + ((u64)sh.pub.hist[2][i] << 28));
        if (lane < C) st_remote(&sh.pub.group[rank][g], lane, s);
    }
}
// after that barrier: the first bin at which carry + the running sum of all CTAs' histograms
// reaches target; *above = that sum before the bin.  All threads call it.
__device__ int find_bin(FShared &sh, int C, u64 target, u64 carry, u64 *above) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    u64 g = 0;
    for (int q = 0; q < C; ++q) g += sh.pub.group[q][lane];
    u64 incl = carry + warp_scan(g);
    unsigned hit = __ballot_sync(0xffffffffu, incl >= target);
    const int gi = hit ? __ffs(hit) - 1 : 31;                    // (target is always reached)
    const u64 before = __shfl_sync(0xffffffffu, incl - g, gi);
    for (int i = warp; i < 3 * C; i += FW)                       // the warps share the loads
        sh.fine[i][lane] = ld_remote(&sh.pub.hist[i % 3][32 * gi + lane], i / 3);
    __syncthreads();
    if (warp == 0) {
        u64 m = 0;
        for (int q = 0; q < C; ++q)
            m += sh.fine[3 * q][lane] + ((u64)sh.fine[3 * q + 1][lane] << 14) + ((u64)sh.fine[3 * q + 2][lane] << 28);
        incl = before + warp_scan(m);
        hit = __ballot_sync(0xffffffffu, incl >= target);
        if (lane == (hit ? __ffs(hit) - 1 : 31)) { sh.found = (unsigned)(32 * gi + lane); sh.found_above = incl - m; }
    }
    __syncthreads();
    *above = sh.found_above;
    return (int)sh.found;                   // (not written again before the next barrier)
}

template <typename T>
__global__ void __launch_bounds__(FT, 1) sample_filtered_kernel(const FilteredParams p) {
    __shared__ FShared sh;
    const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
    const int C = p.C, rank = (int)cluster_rank();
    const int r = blockIdx.x / C;
    const int per = (p.V + C - 1) / C;
    const int base = min(p.V, rank * per), n = min(p.V, base + per) - base;   // this CTA's slice
    const T *lg = static_cast<const T *>(p.logits) + (int64_t)r * p.ld + base;
    const float Tf = p.temperature ? p.temperature[r] : 1.0f;
    const float pf = p.top_p ? p.top_p[r] : 1.0f, mf = p.min_p ? p.min_p[r] : 0.0f;
    const int k = p.top_k ? p.top_k[r] : 0;
    const float uf = p.u[r];
    // a warp's segment of the slice: its first entry and, after the first loop, how many of
    // its entries are still in the list that starts there
    const int seg = (int)round_up(ceil_div(max(n, 1), FW), 32);
    const int s0 = min(n, warp * seg), s1 = min(n, s0 + seg);
    int len = s1 - s0;
    float *mine = slice_values + s0;

    // values, largest (its lowest index), smallest, how many count
    float vmax = -INFINITY, vmin = INFINITY;
    int imax = 0;
    unsigned cnt = 0;
#pragma unroll 16
    for (int i = lane; i < len; i += 32) {
        const float l = logit(lg + s0 + i);
        mine[i] = l;
        if (l > vmax) { vmax = l; imax = i; }
        if (l > -INFINITY) { vmin = fminf(vmin, l); ++cnt; }
    }
    for (int i = t; i < 3 * FNB; i += FT) (&sh.pub.hist[0][0])[i] = 0;
    if (t < 16) sh.table[t] = root16[t];
    if (t == 0) sh.appended = 0;
    u64 top = warp_max(((u64)key_of(vmax) << 32) | (unsigned)~(base + s0 + imax));
    unsigned low = __reduce_max_sync(0xffffffffu, ~key_of(vmin));
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    if (lane == 0) { sh.scan[warp] = top; sh.wmass[warp] = low; sh.weq[warp] = cnt; }
    if (C > 1) cluster_arrive();           // every CTA of the row has begun: its memory can be written
    __syncthreads();
    if (C > 1) cluster_wait();
    if (warp == 0) {
        top = warp_max(lane < FW ? sh.scan[lane] : 0);
        low = __reduce_max_sync(0xffffffffu, lane < FW ? (unsigned)sh.wmass[lane] : 0u);
        cnt = __reduce_add_sync(0xffffffffu, lane < FW ? (unsigned)sh.weq[lane] : 0u);
        if (lane < C) {
            st_remote(&sh.pub.top[rank], lane, top);
            st_remote(&sh.pub.low[rank], lane, low);
            st_remote(&sh.pub.n[rank], lane, cnt);
        }
    }
    cluster_sync();
    top = warp_max(lane < C ? sh.pub.top[lane] : 0);
    low = __reduce_max_sync(0xffffffffu, lane < C ? sh.pub.low[lane] : 0u);
    cnt = __reduce_add_sync(0xffffffffu, lane < C ? sh.pub.n[lane] : 0u);
    const unsigned kmax = (unsigned)(top >> 32), kmin = ~low;
    const int first_max = (int)~(unsigned)top;
    if (cnt == 0 || !(Tf > 0.0f) || k == 1 || !(mf <= 1.0f) || !(pf > 0.0f)) {
        // every logit is masked, or only the first maximum is kept
        if (rank == 0 && t == 0) {
            p.tokens[r] = cnt == 0 ? 0 : first_max + 1;
            if (p.probs) p.probs[r] = cnt == 0 ? 0.0f : 1.0f;
        }
        return;
    }
    // +infinity: the entries that are it share all the mass (0 stands for them, the rest is masked)
    float top_value = key_value(kmax), least = key_value(kmin);
    const bool infinite = top_value == INFINITY;
    auto value = [&](int i) {               // entry i of the slice as it stands in the lists
        const float l = logit(lg + i);
        return infinite ? (l == INFINITY ? 0.0f : -INFINITY) : l;
    };
    if (infinite) {
        unsigned c = 0;
        for (int i = lane; i < len; i += 32) {
            mine[i] = mine[i] == INFINITY ? 0.0f : -INFINITY;
            c += mine[i] == 0.0f;
        }
        __syncwarp();
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0) sh.weq[warp] = c;
        __syncthreads();
        c = __reduce_add_sync(0xffffffffu, lane < FW ? (unsigned)sh.weq[lane] : 0u);
        if (t < C) st_remote(&sh.pub.n_inf[rank], t, c);
        cluster_sync();
        cnt = __reduce_add_sync(0xffffffffu, lane < C ? sh.pub.n_inf[lane] : 0u);
        top_value = least = 0.0f;
    }
    Weigh s;
    s.table = sh.table;
    s.mx = (double)top_value;
    s.c = 23.083120654223414 / (double)Tf;                     // 16 / ln 2

    // the histogram: equal steps below the maximum, the last bin open.  The range covers
    // every weight that counts (e^-32) or the whole row, whichever is less.
    const float span = fminf(top_value - least, 32.0f * Tf);
    const float iw = span > 1e-30f ? FNB / span : 0.0f;
    auto lin = [&](float l) {
        const float d = (top_value - l) * iw;                  // never rises with the logit
        return d > 0.0f ? (d < FNB - 1 ? (int)d : FNB - 1) : 0;
    };
    // drops the entries for which keep() is false from the warp's list, in place and in order
    auto compact = [&](auto keep) {
        int m = 0;
        for (int i0 = 0; i0 < len; i0 += 128) {                // four words in flight
            float l[4];
            unsigned b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = i0 + 32 * j + lane;
                l[j] = i < len ? mine[i] : -INFINITY;
                b[j] = __ballot_sync(0xffffffffu, i < len && keep(l[j]));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (b[j] >> lane & 1u) mine[m + __popc(b[j] & ((1u << lane) - 1u))] = l[j];
                m += __popc(b[j]);
            }
        }
        __syncwarp();
        len = m;
    };
    // a value below which no entry of the bins up to b lies, and one above which none of bin b and
    // beyond does: the bin's edges with room for the roundings of lin
    auto lower_edge = [&](int b) {
        return b == FNB - 1 || iw == 0.0f ? least : fmaxf(least, __double2float_rd(s.mx - (double)(b + 1) / iw * (1.0 + 1e-6)));
    };
    auto upper_edge = [&](int b) {
        return b == 0 || iw == 0.0f ? top_value : fminf(top_value, __double2float_ru(s.mx - (double)b / iw * (1.0 - 1e-6)));
    };
    // The cut of a selection whose histogram has been found to cross target in bin b, with
    // `above` before it: the largest value v with W(entries >= v) >= target, among the entries
    // above `floor` (masses) or all (counts); *above becomes W(entries > v).
    const int cap = FLIST / C;
    auto cut_in_bin = [&](int b, u64 *above, u64 target, bool count, float floor) {
        // the bin's entries of this CTA, then their masses, to every CTA
        for (int i = lane; i < len; i += 32) {
            const float l = mine[i];
            if (lin(l) != b || !(count ? l > -INFINITY : l > floor)) continue;
            const unsigned at = atomicAdd(&sh.appended, 1u);
            if (at < (unsigned)cap) sh.pub.lval[rank * cap + at] = l;
        }
        __syncthreads();
        const int got = (int)sh.appended;
        for (int i = t; i < min(got, cap); i += FT) {
            const float l = sh.pub.lval[rank * cap + i];
            const u64 w = count ? 1 : s.mass(l);
            for (int q = 0; q < C; ++q) {
                st_remote(&sh.pub.lval[rank * cap + i], q, __float_as_uint(l));
                st_remote(&sh.pub.lmass[rank * cap + i], q, w);
            }
        }
        if (t < C) st_remote(&sh.pub.lcount[rank], t, (unsigned)got);
        cluster_sync();
        if (t == 0) sh.appended = 0;
        const unsigned mine_n = lane < C ? sh.pub.lcount[lane] : 0u;
        if (__all_sync(0xffffffffu, mine_n <= (unsigned)cap)) {
            // the lists in a row, then four threads per entry add up what is above and equal to it
            int off = (int)mine_n;
#pragma unroll
            for (int o = 1; o < FMAXC; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, off, o);
                if (lane >= o) off += v;
            }
            const int all = __shfl_sync(0xffffffffu, off, FMAXC - 1);
            if (warp == 0 && lane < FMAXC) sh.loff[lane] = off - (int)mine_n;
            __syncthreads();
            float *flat_v = reinterpret_cast<float *>(sh.pub.hist[0]);        // (the histogram is done with)
            u64 *flat_w = reinterpret_cast<u64 *>(sh.pub.hist[1]);
            for (int e = t; e < cap * C; e += FT) {
                const int q = e / cap, j = e - q * cap;
                if (j < (int)sh.pub.lcount[q]) {
                    flat_v[sh.loff[q] + j] = sh.pub.lval[e];
                    flat_w[sh.loff[q] + j] = sh.pub.lmass[e];
                }
            }
            __syncthreads();
            for (int e0 = 0; e0 < all; e0 += FT / 4) {
                const int e = e0 + (t >> 2);
                const float v = e < all ? flat_v[e] : INFINITY;
                u64 more = 0, same = 0;
#pragma unroll 4
                for (int j = t & 3; j < all; j += 4) {
                    const float l = flat_v[j];
                    const u64 w = flat_w[j];
                    if (l > v) more += w;
                    else if (l == v) same += w;
                }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    more += __shfl_xor_sync(0xffffffffu, more, o);
                    same += __shfl_xor_sync(0xffffffffu, same, o);
                }
                more += *above;
                if (e < all && more < target && more + same >= target) { sh.found = key_of(v); sh.found_above = more; }
            }
            __syncthreads();
            *above = sh.found_above;
            return key_value(sh.found);
        }
        // too many: histograms of 10 bits of the key, within the keys the bin can hold
        unsigned hi = key_of(upper_edge(b)), lo = key_of(lower_edge(b));
        if (!count) lo = max(lo, key_of(floor));
        for (int level = 0; lo < hi && level < 8; ++level) {     // at most 4
            int sft = 0;
            while (((hi - lo) >> sft) >= (unsigned)FNB) ++sft;
            // (every CTA has read the previous histogram: a barrier has passed since)
            for (int i = t; i < 3 * FNB; i += FT) (&sh.pub.hist[0][0])[i] = 0;
            __syncthreads();
            for (int i = lane; i < len; i += 32) {
                const float l = mine[i];
                const unsigned key = key_of(l);
                if (key >= lo && key <= hi && lin(l) == b && (count || l > floor)) {
                    const int bin = (int)((hi - key) >> sft);
                    if (count) atomicAdd(&sh.pub.hist[0][bin], 1u);
                    else hist_mass(sh.pub.hist, bin, s.mass(l));
                }
            }
            publish_groups(sh, C, rank);
            cluster_sync();
            const int d = find_bin(sh, C, target, *above, above);
            const unsigned top_key = hi - ((unsigned)d << sft);
            const unsigned width = (1u << sft) - 1u;
            lo = top_key - lo > width ? top_key - width : lo;
            hi = top_key;
            cluster_sync();
        }
        return key_value(lo);
    };

    // top-k: entries above `cut`, and the first `ties` equal to it
    float cut = least;
    u64 ties = (u64)p.V;
    if (k > 0 && (unsigned)k < cnt) {
#pragma unroll 4
        for (int i = lane; i < len; i += 32) {
            const float l = mine[i];
            if (l > -INFINITY) atomicAdd(&sh.pub.hist[0][lin(l)], 1u);
        }
        publish_groups(sh, C, rank);
        cluster_sync();
        u64 above;
        const int b = find_bin(sh, C, (u64)k, 0, &above);
        const float edge = lower_edge(b);
        compact([&](float l) { return l >= edge; });
        cut = cut_in_bin(b, &above, (u64)k, true, 0.0f);
        ties = (u64)k - above;
        compact([&](float l) { return l >= cut; });
        // (every CTA has read the histogram: cut_in_bin has passed a barrier since)
        for (int i = t; i < 3 * FNB; i += FT) (&sh.pub.hist[0][0])[i] = 0;
        __syncthreads();
    }

    // masses above the cut by warp segment, entries equal to it; min-p here unless top-p comes first
    const bool by_p = pf < 1.0f;
    double floor_w = by_p ? 0.0 : (double)mf * FSCALE;
    u64 wm = 0, we = 0;                     // of this warp
    u64 before_m, before_e, all_m, all_e;   // of the CTAs before this one, of all CTAs
    auto segment_sums = [&](auto add, int slot) {
        wm = 0;
        unsigned ne = 0;
#pragma unroll 4
        for (int i = lane; i < len; i += 32) {
            const float l = mine[i];
            double scaled;
            const u64 w = s.mass(l, &scaled);
            const bool in = l > cut;
            wm += in && (!(floor_w > 0.0) || scaled >= floor_w) ? w : 0;
            ne += l == cut;
            add(l, in ? w : 0);
        }
        wm = warp_sum(wm);
        we = __reduce_add_sync(0xffffffffu, ne);
        if (lane == 0) { sh.wmass[warp] = wm; sh.weq[warp] = we; }
        __syncthreads();
        if (warp == 0) {
            const u64 a = warp_sum(lane < FW ? sh.wmass[lane] : 0);
            const unsigned e = __reduce_add_sync(0xffffffffu, lane < FW ? (unsigned)sh.weq[lane] : 0u);
            if (lane < C) { st_remote(&sh.pub.mass[slot][rank], lane, a); st_remote(&sh.pub.eq[slot][rank], lane, (u64)e); }
        }
        if (slot == 0 && by_p) publish_groups(sh, C, rank);
        cluster_sync();
        const u64 m = lane < C ? sh.pub.mass[slot][lane] : 0;
        const unsigned e = lane < C ? (unsigned)sh.pub.eq[slot][lane] : 0u;
        all_m = warp_sum(m);
        all_e = __reduce_add_sync(0xffffffffu, e);
        before_m = warp_sum(lane < rank ? m : 0);
        before_e = __reduce_add_sync(0xffffffffu, lane < rank ? e : 0u);
    };
    if (by_p) segment_sums([&](float l, u64 w) { if (w > 0) hist_mass(sh.pub.hist, lin(l), w); }, 0);
    else segment_sums([](float, u64) {}, 0);
    double cut_scaled;
    u64 wcut = s.mass(cut, &cut_scaled);

    if (by_p) {
        // (entries equal to the top-k cut count with their kept share: they are the lowest)
        const u64 eq = all_e < ties ? all_e : ties;
        const u64 z = all_m + eq * wcut;
        u64 target = (u64)ceil((double)pf * (double)z);
        target = target < 1 ? 1 : target > z ? z : target;
        if (target <= all_m) {
            u64 above;
            const int b = find_bin(sh, C, target, 0, &above);
            const float edge = lower_edge(b);
            compact([&](float l) { return l > cut && l >= edge; });
            cut = cut_in_bin(b, &above, target, false, cut);
            wcut = s.mass(cut, &cut_scaled);
            ties = (target - above + wcut - 1) / wcut;
        } else if (wcut > 0) {
            ties = min(eq, (target - all_m + wcut - 1) / wcut);
        }
        compact([&](float l) { return l >= cut; });
        // the masses of what is left, with min-p
        floor_w = (double)mf * FSCALE;
        segment_sums([](float, u64) {}, 1);
    }
    if (cut_scaled < floor_w) wcut = 0;
    auto with_ties = [&](u64 m, u64 e) { return m + (e < ties ? e : ties) * wcut; };   // running mass after m, e
    const u64 total = with_ties(all_m, all_e);
    const double prob1 = FSCALE / (double)total;

    if (!(uf > 0.0f)) {
        // the first kept index of any mass, also one that rounds to no unit of 2^-40 (the first
        // entry equal to the cut is always kept)
        int first = INT32_MAX;
        for (int i = t; i < n; i += FT) {
            const float l = value(i);
            if (!(l >= cut)) continue;
            const double w = s.weight(l);
            if (w > 0.0 && w * FSCALE >= floor_w) { first = base + i; break; }
        }
        first = __reduce_min_sync(0xffffffffu, first);
        __syncthreads();
        if (lane == 0) sh.scan[warp] = (u64)first;
        __syncthreads();
        first = __reduce_min_sync(0xffffffffu, lane < FW ? (int)sh.scan[lane] : INT32_MAX);
        if (t < C) st_remote(&sh.pub.first[rank], t, (unsigned)first);
        cluster_sync();
        int lowest = INT32_MAX;
        for (int q = 0; q < C; ++q) lowest = min(lowest, sh.pub.first[q]);
        if (t == 0 && first == lowest && lowest != INT32_MAX) {
            p.tokens[r] = lowest + 1;
            if (p.probs) p.probs[r] = (float)(s.weight(value(lowest - base)) * prob1);
        }
        return;
    }
    u64 goal = (u64)((double)uf * (double)total) + 1;         // the running mass that passes u * mass
    if (goal > total) goal = total;
    // the warp whose segment holds the goal
    if (lane == 0) sh.scan[warp] = (u64)len;
    if (t == 0) sh.holder = -1;
    __syncthreads();
    if (warp == 0) {
        const u64 m0 = lane < FW ? sh.wmass[lane] : 0, e0 = lane < FW ? sh.weq[lane] : 0;
        const u64 sm = warp_scan(m0), se = warp_scan(e0);
        const u64 m = before_m + sm - m0, e = before_e + se - e0;
        if (with_ties(m, e) < goal && goal <= with_ties(before_m + sm, before_e + se)) {
            sh.holder = lane;
            sh.hmass = m;
            sh.heq = e;
        }
    }
    __syncthreads();
    const int holder = sh.holder;
    if (holder >= 0) {
        // the CTA's warps share that segment's list: the piece, then the entry
        const int hlen = (int)sh.scan[holder], h0 = min(n, holder * seg), h1 = min(n, h0 + seg);
        const float *list = slice_values + h0;
        const int sub = (int)round_up(ceil_div(max(hlen, 1), FW), 32);
        const int a0 = min(hlen, warp * sub), a1 = min(hlen, a0 + sub);
        auto entry = [&](int i, bool &eq) -> u64 {
            const float l = i < a1 ? list[i] : -INFINITY;
            eq = i < a1 && l == cut;
            if (!(l > cut)) return 0;
            double scaled;
            const u64 w = s.mass(l, &scaled);
            return scaled >= floor_w ? w : 0;
        };
        wm = 0; we = 0;
        for (int i0 = a0; i0 < a1; i0 += 32) {
            bool eq;
            wm += entry(i0 + lane, eq);
            we += eq ? 1 : 0;
        }
        wm = warp_sum(wm);
        we = warp_sum(we);
        __syncthreads();
        if (lane == 0) { sh.wmass[warp] = wm; sh.weq[warp] = we; }
        __syncthreads();
        u64 m = sh.hmass + warp_sum(lane < warp ? sh.wmass[lane] : 0), e = sh.heq + warp_sum(lane < warp ? sh.weq[lane] : 0);
        if (with_ties(m, e) < goal && goal <= with_ties(m + wm, e + we)) {
            for (int i0 = a0; i0 < a1; i0 += 32) {
                bool eq;
                const u64 incl = warp_scan(entry(i0 + lane, eq));
                const unsigned eqm = __ballot_sync(0xffffffffu, eq);
                const u64 after = with_ties(m + incl, e + __popc(eqm & (0xffffffffu >> (31 - lane))));
                const unsigned hit = __ballot_sync(0xffffffffu, after >= goal);
                if (hit) {
                    if (lane == 0) sh.at = i0 + __ffs(hit) - 1;      // position in the list
                    break;
                }
                m += __shfl_sync(0xffffffffu, incl, 31);
                e += __popc(eqm);
            }
        }
        __syncthreads();
        // its index: the list holds the segment's entries of at least the cut, in order, or all of
        // them; the warps count pieces of the segment
        int at = sh.at;
        const float drawn = list[at];
        int index = h0 + at;
        bool writer = t == 0;
        if (hlen < h1 - h0) {
            const int part = (int)round_up(ceil_div(h1 - h0, FW), 32);
            const int b0 = min(h1, h0 + warp * part), b1 = min(h1, b0 + part);
            int c = 0;
            for (int i0 = b0; i0 < b1; i0 += 32)
                c += __popc(__ballot_sync(0xffffffffu, i0 + lane < b1 && value(i0 + lane) >= cut));
            if (lane == 0) sh.scan[warp] = (u64)c;
            __syncthreads();
            at -= (int)warp_sum(lane < warp ? sh.scan[lane] : 0);
            writer = lane == 0 && at >= 0 && at < c;
            if (at >= 0 && at < c)
                for (int i0 = b0; i0 < b1; i0 += 32) {
                    const unsigned b = __ballot_sync(0xffffffffu, i0 + lane < b1 && value(i0 + lane) >= cut);
                    const int c1 = __popc(b);
                    if (at < c1) {
                        index = i0 + (int)__fns(b, 0, at + 1);
                        break;
                    }
                    at -= c1;
                }
        }
        if (writer) {
            p.tokens[r] = base + index + 1;
            if (p.probs) p.probs[r] = (float)(s.weight(drawn) * prob1);
        }
    }
    // (the last remote accesses, find_bin's loads and segment_sums's stores, lie before a barrier
    // that every CTA has passed, so a CTA may leave)
}

// CTAs per row: enough to hold the row in shared memory, then as many as leave an SM for
// each, down to 4096 entries a CTA
int filtered_ctas(int32_t rows, int32_t V) {
    int c = 1;
    while (c < FMAXC && ((int64_t)c * FRES < V || ((int64_t)2 * c * rows <= 148 && V / c > 4096))) c *= 2;
    return c;
}

template <typename T> int launch_filtered(const FilteredParams &p, int32_t rows, cudaStream_t s) {
    auto kern = sample_filtered_kernel<T>;
    static bool configured[64] = {};
    int dev = 0;
    Q35_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        Q35_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FRES * 4));
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * p.C));
    cfg.blockDim = dim3(FT);
    cfg.dynamicSmemBytes = (size_t)ceil_div(p.V, p.C) * 4;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    Q35_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return Q35_OK;
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
    if (vocab < 1 || vocab > FMAXV) return set_error(Q35_ERR_INVALID, "sample_filtered: vocabulary must be 1..401408");
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
    p.C = filtered_ctas(rows, vocab);
    if ((int64_t)rows * p.C > INT32_MAX) return set_error(Q35_ERR_INVALID, "sample_filtered: too many rows in one call");
    switch (dtype) {
    case Q35_DT_F32: return launch_filtered<float>(p, rows, ctx->stream);
    case Q35_DT_BF16: return launch_filtered<__nv_bfloat16>(p, rows, ctx->stream);
    default: return launch_filtered<__half>(p, rows, ctx->stream);
    }
}
