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

}  // namespace q35
