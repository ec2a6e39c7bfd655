// q35_kv8.cuh -- launchers of the 8-bit KV cache (q35_kv8.cu), shared with the model runtime
#pragma once
#include "q35_q8.cuh"

namespace q35 {

struct Kv8Rows {
    const int32_t *row_start;   // device [seqs + 1]: rows row_start[s] .. row_start[s+1]-1 belong to sequence s
    const int32_t *past;        // device [seqs]: tokens of the sequence before these rows
    int32_t rows, max_rows;     // rows in all; no sequence has more than max_rows of them
};

int kv8_check(const q35_kv8_cache *c);
int launch_kv8_append(const q35_kv8_cache &c, int dtype, const void *k, const void *v, int64_t ld, const Kv8Rows &r,
                      int *err, cudaStream_t s);
// bytes that cover every call on the cache with at most max_rows rows a sequence
size_t kv8_workspace_bound(const q35_kv8_cache &c, int32_t heads);
size_t kv8_attention_workspace(const q35_kv8_cache &c, int32_t heads, int32_t rows, int32_t max_rows);
// out (q's type, row stride ldo) or, when out_q is set, trunc(127 o) as the next int8 matmul takes it
// (rows heads * head_dim apart)
int launch_kv8_attention(const q35_kv8_cache &c, int dtype, const void *q, int64_t ldq, int32_t heads, void *out,
                         int64_t ldo, int8_t *out_q, const Kv8Rows &r, float scale, void *workspace, int *err,
                         cudaStream_t s);

// ---- shared by the attention kernels (q35_kv8.cu, q35_kv8_prompt.cu) ----

struct AttnParams {
    const void *q;
    void *out;
    int8_t *out_q;
    const uint8_t *k, *v;
    const float *ks, *vs;
    int64_t ldq, ldo, seq_stride, scale_seq_stride;
    const int32_t *row_start, *past;
    int32_t rows, max_rows, H, G, max_seq, nblk;   // G: heads per kv head
    int32_t splits, tile_rows, step_keys;          // rows of a tile, keys of a warp's step
    int32_t block_shift;                           // log2 of the tokens per scale
    float scale;
    float *part_o;                                 // [tile][split][16][D] unnormalised outputs
    float2 *part_ml;                               // [tile][split][16] maximum (log2 units) and sum
    int *err;
};

// whether rows of this number take the prompt kernel
bool kv8_prompt_takes(const q35_kv8_cache &c, int32_t heads, int32_t max_rows);
int launch_kv8_prompt(const AttnParams &p, int dtype, int code, int D, int zs, cudaStream_t s);

#ifdef __CUDACC__
// the rows of sequence s: first row, count (0 with the error word set when the tables are
// inconsistent or the cache would overflow) and the tokens before them
struct SeqRows { int r0, n, past; };
__device__ __forceinline__ SeqRows seq_rows(const int32_t *row_start, const int32_t *past, int s, int rows,
                                            int max_rows, int max_seq, int *err) {
    SeqRows q;
    q.r0 = row_start[s];
    const int r1 = row_start[s + 1];
    q.n = r1 - q.r0;
    q.past = past[s];
    const bool ok = q.r0 >= 0 && r1 >= q.r0 && r1 <= rows && q.n <= max_rows && q.past >= 0 &&
                    (int64_t)q.past + q.n <= max_seq;
    if (!ok) {
        if (threadIdx.x == 0) atomicExch(err, Q35_ERR_INVALID);
        q.n = 0;
    }
    return q;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// (coherent loads: these grids start while the append that writes codes and scales still runs, and the
// read-only path is for memory that nobody writes while the grid lives)
__device__ __forceinline__ uint4 ldg16(const uint8_t *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ float ldg(const float *p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
    return v;
}
// four codes to two fp16 pairs (bytes 0,1 and 2,3)
template <int CODE> __device__ __forceinline__ void codes_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if (CODE == Q35_CODE_INT8) {
        // 0x64xx is the fp16 number 1024 + xx: biased bytes, minus 1024 + 128, exactly
        const uint32_t u = w ^ 0x80808080u;
        const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        asm("sub.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
        asm("sub.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
    } else {
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi) : "r"(w));
    }
}
#endif

}  // namespace q35
