// A serving step's tables, and its queries and keys on their way into a paged
// cache (rqmv_paged_plan, rqmv_qk_norm_rope).
#include "paged.h"

#include <limits.h>

#include "lanes.h"
#include "paged_rows.h"

namespace rq {

// --------------------------------------------------------------- tables ----

// Sequence s holds h_s = ceil(cached_s / B) pages and needs n_s = ceil((cached_s
// + new_s) / B); with S the exclusive prefix sum of n - h, its page p >= h_s is
// free_list[head + S_s + p - h_s]. Row t belongs to the sequence with start_s <=
// t < start_{s+1}, start the prefix sum of new.
//
// One workgroup makes everything that depends on all sequences: a first pass
// over them adds up and checks (nothing is written before it is known that the
// step fits), a second scans and writes the starts, lengths and new table
// entries, the starts and page starts kept in LDS for the searches by row and
// by page. Rows are independent of each other once the starts are known: up
// to kPlanRows of them the same workgroup writes them, more go to a second
// launch over the whole device.
constexpr int kPlanThreads = 1024;
constexpr int kPlanRows = 2048;

// Inclusive prefix sums of two values over the workgroup; `total` gets the sums.
__device__ __forceinline__ void scan2(int& a, int& b, int (&total)[2], int (*part)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    a = (int)wave_scan((unsigned)a);
    b = (int)wave_scan((unsigned)b);
    if (lane == 63) part[wave][0] = a, part[wave][1] = b;
    __syncthreads();
    total[0] = total[1] = 0;
    int ba = 0, bb = 0;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wave) ba += part[w][0], bb += part[w][1];
        total[0] += part[w][0], total[1] += part[w][1];
    }
    a += ba, b += bb;
    __syncthreads();
}

// The last s in 0..n-1 with start[s] <= t (start[0] <= t).
__device__ __forceinline__ int last_at(const int* start, int n, int t) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int slot_of(int block, int row, int blocks, int shift) {
    return (unsigned)block < (unsigned)blocks ? (block << shift) + row : -1;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedBatch b, int blocks, int shift,
                                                                  const int* cached_len, const int* new_len,
                                                                  const int* free_list, int free_count,
                                                                  const int* free_head, int* free_head_out,
                                                                  int* status, bool rows_too) {
    extern __shared__ int lds[];
    int* start = lds;                 // seqs + 1 entries
    int* page = lds + b.seqs + 1;     // seqs + 1 entries
    __shared__ int part[kPlanThreads / 64][2];
    __shared__ unsigned long long sums[2];
    __shared__ int bad;
    const int t = threadIdx.x;
    const int64_t most = (int64_t)b.max_blocks << shift;
    const int head = *free_head;
    if (t < 2) sums[t] = 0;
    if (t == 2) bad = 0;
    __syncthreads();
    // sums in 64 bits: 8192 sequences of 2^31 rows pass 32
    unsigned long long rows = 0, fresh = 0;
    bool wrong = false;
    for (int s = t; s < b.seqs; s += kPlanThreads) {
        const int c = cached_len[s], n = new_len[s];
        if (c < 0 || n < 0 || (int64_t)c + n > most) {
            wrong = true;
            continue;
        }
        rows += n;
        fresh += (((int64_t)c + n + (1 << shift) - 1) >> shift) - (((int64_t)c + (1 << shift) - 1) >> shift);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) rows += __shfl_xor(rows, d), fresh += __shfl_xor(fresh, d);
    if ((t & 63) == 0) {
        atomicAdd(&sums[0], rows);
        atomicAdd(&sums[1], fresh);
    }
    if (wrong) atomicOr(&bad, 1);
    __syncthreads();
    int err = bad;
    if (sums[0] > (unsigned long long)b.tokens) err |= 2;
    if (head < 0 || head > free_count || sums[1] > (unsigned long long)(free_count - head)) err |= 4;
    // the starts, page starts and lengths (on an error: no rows, lengths unchanged)
    int row0 = 0, page0 = 0;
    for (int s0 = 0; s0 < b.seqs; s0 += kPlanThreads) {
        const int s = s0 + t;
        int c = 0, n = 0, need = 0;
        if (s < b.seqs) {
            c = cached_len[s];
            if (!err) {
                n = new_len[s];
                need = (int)((((int64_t)c + n + (1 << shift) - 1) >> shift) - (((int64_t)c + (1 << shift) - 1) >> shift));
            }
        }
        int a = n, p = need, total[2];
        scan2(a, p, total, part);
        if (s < b.seqs) {
            start[s] = row0 + a - n;
            page[s] = page0 + p - need;
            b.q_start[s] = row0 + a - n;
            b.kv_len[s] = c + n;
        }
        row0 += total[0];
        page0 += total[1];
    }
    if (t == 0) {
        start[b.seqs] = row0;
        page[b.seqs] = page0;
        b.q_start[b.seqs] = row0;
        *free_head_out = head + page0;
        *status = err;
    }
    __syncthreads();
    // the pages taken, each by its number in the step: its sequence ends with its last new pages
    for (int p = t; p < page0; p += kPlanThreads) {
        const int s = last_at(page, b.seqs, p);
        const int end = (int)(((int64_t)b.kv_len[s] + (1 << shift) - 1) >> shift);
        b.table[s * b.table_stride + end - (page[s + 1] - p)] = free_list[head + p];
    }
    if (!rows_too) return;
    for (int r = t; r < b.tokens; r += kPlanThreads) {
        int pos = 0, slot = -1;
        if (r < row0) {
            const int s = last_at(start, b.seqs, r);
            const int kv = b.kv_len[s];
            pos = kv - (start[s + 1] - r);
            const int end = (int)(((int64_t)kv + (1 << shift) - 1) >> shift);
            const int at = pos >> shift, p = page[s + 1] - (end - at);  // (a new page's number in the step)
            const int block = p >= page[s] ? free_list[head + p] : b.table[s * b.table_stride + at];
            slot = slot_of(block, pos & ((1 << shift) - 1), blocks, shift);
        }
        b.positions[r] = pos;
        b.slots[r] = slot;
    }
}

// Positions and slots by row, from the starts, lengths and tables of the launch before.
__global__ void __launch_bounds__(256) paged_rows_kernel(PagedBatch b, int blocks, int shift) {
    extern __shared__ int start[];  // seqs + 1 entries
    for (int s = threadIdx.x; s <= b.seqs; s += 256) start[s] = b.q_start[s];
    __syncthreads();
    for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < b.tokens; r += (int64_t)gridDim.x * 256) {
        int pos = 0, slot = -1;
        if (r < start[b.seqs]) {
            const int s = last_at(start, b.seqs, (int)r);
            pos = b.kv_len[s] - (start[s + 1] - (int)r);
            slot = slot_of(b.table[s * b.table_stride + (pos >> shift)], pos & ((1 << shift) - 1), blocks, shift);
        }
        b.positions[r] = pos;
        b.slots[r] = slot;
    }
}

hipError_t launch_paged_plan(const PagedBatch& b, int blocks, int block_shift, const int* cached_len,
                             const int* new_len, const int* free_list, int free_count, const int* free_head,
                             int* free_head_out, int* status, hipStream_t stream) {
    const bool rows_too = b.tokens <= kPlanRows;
    const size_t lds = 2 * (size_t)(b.seqs + 1) * sizeof(int);
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(paged_plan_kernel),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), lds, stream, b, blocks, block_shift, cached_len,
                       new_len, free_list, free_count, free_head, free_head_out, status, rows_too);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || rows_too) return e;
    const int grid = (b.tokens - 1) / 256 + 1;
    hipLaunchKernelGGL(paged_rows_kernel, dim3(grid < 2048 ? grid : 2048), dim3(256),
                       (size_t)(b.seqs + 1) * sizeof(int), stream, b, blocks, block_shift);
    return hipGetLastError();
}

// -------------------------------------- norms, rotation and the append ----

template <int HD, typename X, typename Q>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(PagedBatch b, PagedCache c, QkNormRope p) {
    constexpr int LPH = HD / 8;  // lanes per head
    const int token = blockIdx.x;
    const int head = blockIdx.y * (256 / LPH) + threadIdx.x / LPH;
    const int u = threadIdx.x % LPH;
    if (head >= p.q_heads + 2 * c.kv_heads) return;  // (whole lane groups leave)
    const bool value = head >= p.q_heads + c.kv_heads;
    const HeadPlace at = head_place<HD>(p, value, u);
    const int lo = at.lo, hi = at.hi;
    float x[8];
    const X* src = static_cast<const X*>(p.qkv) + (int64_t)token * p.ld + head * HD;
    load4<X>(src + lo, x);
    load4<X>(src + hi, x + 4);
    if (!value) {
        const float* norm = head < p.q_heads ? p.q_norm : p.k_norm;
        HeadLane h;
        if (norm) load_norm(norm, at, h);
        if (at.turns) load_turn(p, b.positions[token], u, h);
        norm_and_turn<HD>(norm, at.turns, p.eps, h, x);
    }
    if (head < p.q_heads) {
        Q* dst = static_cast<Q*>(p.q_out) + (int64_t)token * p.ldq + head * HD;
        store4(dst + lo, x);
        store4(dst + hi, x + 4);
        return;
    }
    const int slot = b.slots[token];
    if (slot < 0 || (slot >> c.block_shift) >= c.blocks) return;
    const int kh = head - p.q_heads - (value ? c.kv_heads : 0);
    const int64_t row = (((int64_t)(slot >> c.block_shift) * c.kv_heads + kh) << c.block_shift) +
                        (slot & ((1 << c.block_shift) - 1));
    __half* dst = (value ? c.v : c.k) + row * HD;
    store4(dst + lo, x);
    store4(dst + hi, x + 4);
}

template <int HD, typename X>
static void launch_qk_x(const PagedBatch& b, const PagedCache& c, const QkNormRope& p, bool q_f16, hipStream_t stream) {
    constexpr int HPB = 256 / (HD / 8);  // heads per workgroup
    const dim3 grid(b.tokens, (p.q_heads + 2 * c.kv_heads + HPB - 1) / HPB);
    if (q_f16) hipLaunchKernelGGL((qk_norm_rope_kernel<HD, X, __half>), grid, dim3(256), 0, stream, b, c, p);
    else hipLaunchKernelGGL((qk_norm_rope_kernel<HD, X, float>), grid, dim3(256), 0, stream, b, c, p);
}

template <int HD>
static void launch_qk_hd(const PagedBatch& b, const PagedCache& c, const QkNormRope& p, bool x_f16, bool q_f16,
                         hipStream_t stream) {
    if (x_f16) launch_qk_x<HD, __half>(b, c, p, q_f16, stream);
    else launch_qk_x<HD, float>(b, c, p, q_f16, stream);
}

hipError_t launch_qk_norm_rope(const PagedBatch& b, const PagedCache& c, const QkNormRope& p, bool x_f16, bool q_f16,
                               hipStream_t stream) {
    if (c.head_dim == 64) launch_qk_hd<64>(b, c, p, x_f16, q_f16, stream);
    else if (c.head_dim == 128) launch_qk_hd<128>(b, c, p, x_f16, q_f16, stream);
    else launch_qk_hd<256>(b, c, p, x_f16, q_f16, stream);
    return hipGetLastError();
}

}  // namespace rq
