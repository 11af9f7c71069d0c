// Paged serving: the step's tables, queries and keys into the paged cache
// (paged.hip; 8-bit pages paged_q8.hip), attention over the pages
// (paged_attention.hip; 8-bit pages paged_attention_q8.hip).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

namespace rq {

// The device side of rqmv_paged_batch / rqmv_paged_cache (include/rqmv.h).
struct PagedBatch {
    int* q_start;
    int* kv_len;
    int* table;
    int64_t table_stride;
    int max_blocks, seqs, tokens;
    int* positions;
    int* slots;
};

struct PagedCache {
    __half* k;
    __half* v;
    int blocks;       // (blocks * block_size < 2^31)
    int block_shift;  // log2 block_size
    int kv_heads, head_dim;
};

// What 8-bit pages hold in place of PagedCache's k and v (which are null then): codes, and a scale byte for each 16
// rows of a block and head.
struct PagedCodes {
    int8_t* k;
    int8_t* v;
    uint8_t* k_scale;
    uint8_t* v_scale;
};

constexpr int kPagedMaxSeqs = 8192;

hipError_t launch_paged_plan(const PagedBatch& b, int blocks, int block_shift, const int* cached_len,
                             const int* new_len, const int* free_list, int free_count, const int* free_head,
                             int* free_head_out, int* status, hipStream_t stream);

struct QkNormRope {
    const void* qkv;
    int64_t ld;
    int q_heads;
    const float* q_norm;
    const float* k_norm;
    float eps;
    const float2* rope;
    int rot_dim, rope_rows;
    void* q_out;
    int64_t ldq;
};
hipError_t launch_qk_norm_rope(const PagedBatch& b, const PagedCache& c, const QkNormRope& p, bool x_f16, bool q_f16,
                               hipStream_t stream);

hipError_t launch_qk_norm_rope_q8(const PagedBatch& b, const PagedCache& c, const PagedCodes& codes, const QkNormRope& p,
                                  bool x_f16, bool q_f16, hipStream_t stream);
// Every value of the codes into the pages k and v of the same shape.
hipError_t launch_paged_values_q8(const PagedCache& c, const PagedCodes& codes, __half* k, __half* v, hipStream_t stream);

// Whether the launches' grids hold this batch.
bool paged_attention_fits(const PagedBatch& b, const PagedCache& c, int q_heads);
size_t paged_attention_workspace(const PagedBatch& b, const PagedCache& c, int q_heads, int cus);
hipError_t launch_paged_attention(const PagedBatch& b, const PagedCache& c, const void* q, bool f32, int64_t ldq,
                                  int q_heads, float scale, int window, void* workspace, void* out, int64_t ldo, int cus,
                                  hipStream_t stream);
size_t paged_attention_q8_workspace(const PagedBatch& b, const PagedCache& c, int q_heads, int cus);
hipError_t launch_paged_attention_q8(const PagedBatch& b, const PagedCache& c, const PagedCodes& codes, const void* q, bool f32,
                                     int64_t ldq, int q_heads, float scale, int window, void* workspace, void* out,
                                     int64_t ldo, int cus, hipStream_t stream);

}  // namespace rq
