// Attention of several sequences' new tokens over their pages: what the kernels
// over fp16 pages (paged_attention.hip, rqmv_paged_attention) and over 8-bit pages
// (paged_attention_q8.hip, rqmv_paged_attention_q8) share.
//
// For query head h of a token at position p of its sequence:
//     out = sum_k e^(s_k) v_k / sum_k e^(s_k),  s_k = scale q . k_k,
// over the positions k of max(0, p - window + 1)..p whose pages are present, in
// one pass over the keys with a running reference m (e^(s - m) throughout; a sum
// is rescaled when its reference moves).
//
// Rows. A sequence with n new tokens has n * group rows per kv head (row r:
// token r / group, head r % group of its group), cut into tiles of TM rows that
// share the keys and values read. Tile i of sequence s is number floor(q_start[s]
// * group / TM) + s + i: no two tiles share a number, the numbers grow with s, so
// a workgroup finds its sequence by searching q_start, and tokens * group / TM +
// seqs numbers always suffice (some stay empty).
//
// Matrix cores. S^T = K Q^T in 32 x 32 tiles: a lane then holds one query (its
// column) and 16 of the tile's 32 keys, the other 16 in lane ^ 32, so a row's
// maximum is taken over registers and one lane swap, and the weights already
// lie where the second product takes them: O^T = V^T P^T needs, per 16 keys,
// eight of them per lane, which may come in any order as long as V's operand has
// the same; keys 4h..4h+3 and 8+4h..8+4h+3 (h = lane / 32) are the lane's own
// scores. V's operand is read transposed from LDS (ds_read_b64_tr_b16).
// Queries stay in registers. fp16 queries: the weights are rounded to fp16 (2^-12
// of each weight on average, as fp16 outputs are rounded; references move
// only when a maximum passes them by 2^8, and the weights are taken times 2^6,
// so that they lie in fp16's normal range down to 2^-20 of the largest). fp32
// queries: queries and weights are split into a high and a low fp16 part, two
// products each (22 bits; queries scaled by a power of two per row, weights by
// 2^15). Sums are fp32.
//
// Keys and values lie in LDS as fp16, 16 keys of one page at a time, 32 or 64 keys
// per step. A row's 16-byte pieces are stored XORed with the row number, so that
// the operand reads hit every bank once.
//
// Masked places: a masked score is -infinity by selection, and V must not meet
// its zero weight as a NaN: in steps where some row may not see some key, the
// values of keys that no row sees are zeroed in LDS, and so are NaN and infinite
// ones of the others; where there are such, they are read again from the cache
// after the last step and added to the rows that see them.
#pragma once

#include "lanes.h"
#include "paged.h"

#include <float.h>
#include <limits.h>

#include "halfcode.h"

namespace rq {

struct AttnArgs {
    const void* q;
    void* out;
    int64_t ldq, ldo;
    PagedBatch b;
    PagedCache c;
    int group, cap;     // query heads per kv head; positions that the table reaches
    int window;         // 0: none
    float scale;        // times log2 e: scores are taken to the base 2
    int tiles, splits, min_chunk;
    // partial results, where a tile's keys are split (a part is one row's: head_dim sums, and
    // reference and weight sum), and for each token and head of a group where its are
    float* o;           // [parts][head_dim]
    float2* ml;         // [parts]
    int most;           // splits of a tile at most, where parts are [split][token][query head]; 0: by item (paged_few_kernel)
    int2* info;         // [tokens][group]: live splits, and where parts are by item 32 first part + row; null: nothing is split
    const int2* items;  // paged_items_kernel's; null: at most kItemSeqs sequences, or paged_many_kernel
    int64_t parts;
};

struct AttnPlan {
    bool few, join, items;
    int splits, min_chunk, most;
    int64_t tiles, parts;
};

// `few_tiles`: tiles of 32 rows over all heads up to which few rows are assumed.
AttnPlan plan_attention(int tokens, int seqs, int64_t cap, int kv_heads, int group, int hd, bool f32, int cus,
                        int64_t few_tiles);
size_t attention_workspace_bytes(const AttnPlan& p, int tokens, int seqs, int group, int hd);
// A call's arguments; where the plan has items, launches the count of them.
hipError_t attention_args(const AttnPlan& p, const PagedBatch& b, const PagedCache& c, const void* q, int64_t ldq, int q_heads,
                          float scale, int window, void* workspace, void* out, int64_t ldo, hipStream_t stream,
                          AttnArgs* args);
// The splits' join, where the plan has one.
hipError_t launch_attention_join(const AttnPlan& p, const AttnArgs& a, bool f32, hipStream_t stream);

inline dim3 attention_grid(const AttnPlan& p, const AttnArgs& a) {
    return dim3((unsigned)((p.tiles + (p.few ? p.splits : 0)) * a.c.kv_heads), p.few ? 1 : p.splits);
}
// Waves of a large tile, 32 rows each.
constexpr int many_waves(int hd) { return hd == 256 ? 4 : 8; }
constexpr int few_lds(int hd) { return 4 * 2 * 32 * hd * 2; }
constexpr int many_lds(int hd) { return 2 * 2 * 64 * hd * 2; }

namespace {

typedef float f16_t __attribute__((ext_vector_type(16)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef short s4_t __attribute__((ext_vector_type(4)));

constexpr int kMaxSplits = 64;  // of one tile's keys

// One tile of rows and its keys.
struct Tile {
    int seq, token0, n, kv;  // the sequence, its first row of q, its new tokens, its positions
    int row0, rows;          // the tile's first row in the sequence, the sequence's rows
    int first, end;          // keys first..end-1 (first a multiple of 64)
    int chunk, live;         // keys per split, splits that have any
    int all_from, all_to;    // every row sees keys all_from..all_to-1
};

// The last sequence s for which at_most(s) holds (it holds up to some s >= 0), 64 candidates at a time.
template <typename F>
__device__ __forceinline__ int last_seq(int seqs, F at_most) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = seqs;
    while (n > 1) {
        const int step = (n + 63) >> 6, i = lane * step;
        const int c = max((int)__popcll(__ballot(i < n && at_most(lo + min(i, n - 1)))), 1) - 1;
        lo += c * step;
        n = min(step, n - c * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}
__device__ __forceinline__ int start_of(const PagedBatch& b, int s) { return min(max(b.q_start[s], 0), b.tokens); }
// Of tile `number`: floor(q_start[s] * group / TM) + s <= number.
template <int TM>
__device__ __forceinline__ int find_seq(const PagedBatch& b, int group, int number) {
    return last_seq(b.seqs, [&](int s) { return start_of(b, s) * group / TM + s <= number; });
}

// A sequence's first row of q, new tokens and positions, read as they are found and brought into range.
struct Seq {
    int token0, n, kv;
};
__device__ __forceinline__ Seq load_seq(const AttnArgs& a, int s) {
    const int from = start_of(a.b, s);
    return Seq{from, min(max(a.b.q_start[s + 1], from), a.b.tokens) - from, max(a.b.kv_len[s], 0)};
}

template <int TM>
__device__ __forceinline__ Tile make_tile(const AttnArgs& a, int seq, const Seq& of, int row0) {
    Tile t;
    t.seq = seq;
    t.token0 = of.token0;
    t.n = of.n;
    t.kv = of.kv;
    t.row0 = row0;
    t.rows = t.n * a.group;
    const int last = min(row0 + TM, t.rows) - 1;
    const int p0 = t.kv - t.n + row0 / a.group, p1 = t.kv - t.n + max(last, 0) / a.group;
    t.end = max(min(p1 + 1, a.cap), 0);
    t.first = a.window ? max(p0 - a.window + 1, 0) & ~63 : 0;
    if (t.first > t.end) t.first = t.end & ~63;
    const int len = t.end - t.first;
    const int even = (len + a.splits - 1) / a.splits;
    t.chunk = max((even + 63) & ~63, a.min_chunk);
    t.live = (len + t.chunk - 1) / t.chunk;
    t.all_from = a.window ? max(p1 - a.window + 1, 0) : 0;
    t.all_to = min(p0 + 1, a.cap);
    return t;
}

// 16 bytes per lane from `base` + `offset` (bytes) straight into LDS at `lds` +
// 16 lane. Inline assembly, so that the compiler does not make every later LDS
// read wait for it: the kernel waits for these loads itself. (M0 holds the LDS
// address; a write of M0 needs one wait state before a load to LDS.)
__device__ __forceinline__ void load_lds(const void* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(offset), "s"(base), "s"(lds)
                 : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

template <int HD>
struct Lay {
    static constexpr int PCS = HD / 8;    // 16-byte pieces per row
    static constexpr int RPI = 64 / PCS;  // rows per load instruction
    static constexpr int NI = 16 / RPI;   // instructions per 16 keys
    static constexpr int ROW = HD * 2;    // bytes per row
    // the XOR of a row's piece numbers: K is read 16 rows at one piece, V four
    // rows at four pieces in a row (a row of 64 dims is half the banks)
    __device__ static constexpr int kx(int row) { return HD == 64 ? (row >> 1) & 7 : row & 15; }
    __device__ static constexpr int vx(int row) { return HD == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2; }
};

// The ids of a sequence's pages, 64 at a time in a wave's lanes.
struct Pages {
    const int* row;
    int last, blocks, shift, from, held;
    __device__ __forceinline__ void fetch(int page) {
        from = page;
        held = row[min(page + (int)(threadIdx.x & 63), last)];
    }
    __device__ __forceinline__ void need(int page0, int page1) {  // pages page0..page1 (at most 4)
        if (page0 < from || page1 >= from + 64) fetch(page0);
    }
    __device__ __forceinline__ int at(int page) const { return __builtin_amdgcn_readlane(held, page - from); }
    __device__ __forceinline__ bool absent(int id) const { return (unsigned)id >= (unsigned)blocks; }
};


// A wave's rows: queries as operands, output sums, references, weight sums.
template <int HD, int QT, bool F32>
struct Rows {
    static constexpr int NK = HD / 16, ND = HD / 32, QP = F32 ? 2 : 1;
    h8_t q[QT][NK][QP];
    f16_t o[QT][ND];
    float m[QT], l[QT], c[QT];  // reference (times c), weight sum of the lane's own keys, factor of the scores
    int lo[QT], hi[QT];         // the row sees keys lo..hi
};

__device__ __forceinline__ h8_t cvt8(const float (&v)[8]) {
    h8_t r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const h2_t p = __builtin_convertvector((f2_t{v[2 * e], v[2 * e + 1]}), h2_t);
        r[2 * e] = p[0];
        r[2 * e + 1] = p[1];
    }
    return r;
}

// A row's values as they are in memory, while they are on their way. (fp16: the operands)
template <int HD, bool F32>
struct RawRows {
    float4 v[F32 ? HD / 16 : 1][2];
};

// Requests the wave's rows, with the first page ids on their way. `arrived` waits for them: the compiler
// would wait for them at their first use in the loop, in every step, and for the step's own loads, which it does not
// count, with them. fp32 rows are asked for before the first step's loads to LDS and become operands while these
// are on their way (one token over 4,096: 4 % less); fp16 rows, which are operands already, come
// behind those loads (32 sequences: 1 % less).
// HALVES: a lane holds the row's dims h HD / 2 + 8 k .. in operand k instead of 16 k + 8 h (the sum over a row's dims may go in
// any order, if the keys' is the same).
template <int HD, bool F32, bool HALVES = false>
__device__ __forceinline__ void load_rows(const AttnArgs& a, const Tile& t, int kh, int row, Rows<HD, 1, F32>& w,
                                          RawRows<HD, F32>& raw) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int r = min(row + (lane & 31), t.rows - 1);  // (rows past the last repeat it)
    const int tok = r / a.group, pos = t.kv - t.n + tok;
    const int64_t at = (int64_t)(t.token0 + tok) * a.ldq + (kh * a.group + r % a.group) * HD + (HALVES ? HD / 2 : 8) * h;
    w.hi[0] = min(pos, a.cap - 1);
    w.lo[0] = a.window ? pos - a.window + 1 : 0;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
        if constexpr (F32) {
            const float* src = static_cast<const float*>(a.q) + at + (HALVES ? 8 : 16) * k;
            raw.v[k][0] = *reinterpret_cast<const float4*>(src);
            raw.v[k][1] = *reinterpret_cast<const float4*>(src + 4);
        } else {
            w.q[0][k][0] = *reinterpret_cast<const h8_t*>(static_cast<const _Float16*>(a.q) + at + (HALVES ? 8 : 16) * k);
        }
    }
}
template <int HD, bool F32>
__device__ __forceinline__ void arrived(Rows<HD, 1, F32>& w, RawRows<HD, F32>& raw) {
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float4& v = raw.v[k][j];
                asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
            }
        } else {
            asm volatile("" : "+v"(w.q[0][k][0]));
        }
    }
}
// Rows to operands (fp32: two fp16 parts), and nothing added up yet.
template <int HD, bool F32>
__device__ __forceinline__ void start_rows(const AttnArgs& a, Rows<HD, 1, F32>& w, const RawRows<HD, F32>& raw) {
    w.m[0] = -INFINITY;
    w.l[0] = 0.f;
    w.c[0] = a.scale;
    if constexpr (F32) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float4 x = raw.v[k][j];
                top = fmaxf(fmaxf(top, fabsf(x.x)), fmaxf(fabsf(x.y), fmaxf(fabsf(x.z), fabsf(x.w))));
            }
        top = swap32_max(top);
        // 2^up brings the row's largest magnitude into [2^13, 2^14); the low
        // part's smallest step is then 2^-37 of it
        int up = top > 0.f && top < INFINITY ? 14 - __builtin_amdgcn_frexp_expf(top) : 0;
        up = min(max(up, -115), 100);
        // The scores' factor stays a normal number: 0 or infinite it would make NaN of masked scores or of zeros. (A lower
        // `up` is for rows whose scores are below 2^-80, a lowered factor for scores far past fp32's range or 0.)
        up = min(up, __builtin_amdgcn_frexp_expf(a.scale) + 125);
        w.c[0] = fminf(ldexpf(a.scale, -up), FLT_MAX);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
            const float4 x = raw.v[k][0], y = raw.v[k][1];
            float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = ldexpf(v[e], up);
            w.q[0][k][0] = cvt8(v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] -= (float)w.q[0][k][0][e];
            w.q[0][k][1] = cvt8(v);
        }
    }
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) w.o[0][d][e] = 0.f;
}

// S^T of 32 KT keys: s[i][t] holds, per lane, query lane % 32 of row tile i and
// keys 32 t + 8 (e / 4) + 4 h + e % 4.
template <int HD, int QT, int KT, bool F32>
__device__ __forceinline__ void scores(const char* K, const Rows<HD, QT, F32>& w, f16_t (&s)[QT][KT]) {
    typedef Lay<HD> L;
    const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[i][t][e] = 0.f;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k)
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int r = 32 * t + (lane & 31);
            const h8_t key = *reinterpret_cast<const h8_t*>(K + r * L::ROW + ((2 * k + h) ^ L::kx(r)) * 16);
#pragma unroll
            for (int i = 0; i < QT; ++i)
#pragma unroll
                for (int p = 0; p < Rows<HD, QT, F32>::QP; ++p)
                    s[i][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key, w.q[i][k][p], s[i][t], 0, 0, 0);
        }
    if constexpr (HD == 128 && KT == 2) {
        // four key operands ahead of their products (2048 tokens over 14,336, fp16: 533 us, without 549; heads of 64
        // and 256 lose 3 % and 1 % so)
        constexpr int READS = HD / 16 * KT, EACH = QT * Rows<HD, QT, F32>::QP;
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < READS - 4; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, EACH, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4 * EACH, 0);
    }
}

// -infinity for the keys that a row does not see.
template <int HD, int QT, int KT, bool F32>
__device__ __forceinline__ void mask_scores(const Rows<HD, QT, F32>& w, f16_t (&s)[QT][KT], int key0, unsigned bad) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        // keys key0 + 4 h + off with off - from <= width, unsigned (a row without keys: none)
        const bool some = w.hi[i] >= w.lo[i];
        const int from = some ? w.lo[i] - key0 - 4 * h : 1 << 30;
        const unsigned width = some ? (unsigned)(w.hi[i] - w.lo[i]) : 0u;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if ((unsigned)(32 * t + 8 * (e / 4) + e % 4 - from) > width) s[i][t][e] = -INFINITY;
    }
    if (bad) {
#pragma unroll
        for (int g = 0; g < 2 * KT; ++g)
            if ((bad >> g) & 1) {
#pragma unroll
                for (int i = 0; i < QT; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[i][g / 2][8 * (g % 2) + e] = -INFINITY;
            }
    }
}

// The rows' largest scores (NaNs apart).
template <int QT, int KT>
__device__ __forceinline__ void largest(const f16_t (&s)[QT][KT], float (&top)[QT]) {
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        float m = s[i][0][0];
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) m = fmaxf(m, s[i][t][e]);
        top[i] = swap32_max(m);
    }
}

// Moves the references to the rows' maxima where one lies more than the slack above.
template <int HD, int QT, bool F32>
__device__ __forceinline__ void move_references(Rows<HD, QT, F32>& w, const float (&largest)[QT]) {
    constexpr float SLACK = F32 ? 0.f : 8.f;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        const float top = largest[i] * w.c[i];
        if (__any(top - w.m[i] > SLACK)) {  // (no key yet and none now: NaN, which moves nothing)
            const float m = fmaxf(w.m[i], top);
            const float f = m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(w.m[i] - m);
            w.m[i] = m;
            w.l[i] *= f;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) w.o[i][d][e] *= f;
        }
    }
}

// Scores to weights, added up and rounded to the second product's operands.
template <int HD, int QT, int KT, bool F32>
__device__ __forceinline__ void weights(Rows<HD, QT, F32>& w, f16_t (&s)[QT][KT],
                                        h8_t (&p)[QT][2 * KT][F32 ? 2 : 1]) {
    // fp32 rows: 2^15 comes after the exponential. With 15 added to the argument its last bit is 2^-20, and rows of
    // six keys were off by 1.8e-7 instead of 1.2e-7 (as fast). fp16 rows: 2^6 in the argument is one
    // instruction less and below the weights' own rounding.
    // fp16, up to 128 dims: the sum of the rounded weights, two at a time. What a large weight's rounding adds
    // to the row it adds to the divisor too, so a row of one large weight is off by its output's rounding alone
    // (2048 tokens over 14,336: 533 us, with the weights added before they are rounded 538; 4,096 over 6,000, 8/4
    // heads of 256: 492 and 484, so there they are added before).
    constexpr bool PAIRS = !F32 && HD <= 128;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
        float ref = w.m[i] == -INFINITY ? 0.f : w.m[i] - (F32 ? 0.f : 6.f), c = w.c[i];
        // Scores of 2^20 and more: the reference is a rounded product, and the exact ones may lie so far from it
        // that every weight leaves fp16's range. Then products are rounded before the difference. (The branch
        // takes 5 % at 64 and 3 % at 256 dims of fp16, nothing at 128.)
        if (__any(fabsf(w.m[i]) > 0x1p20f && w.m[i] > -INFINITY)) {
#pragma clang fp contract(off)
            ref = w.m[i] == -INFINITY ? 0.f : w.m[i];
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float x = s[i][t][e] * c;
                    s[i][t][e] = x - ref;
                }
            c = 1.f;
            ref = F32 ? 0.f : -6.f;
        }
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = __builtin_amdgcn_exp2f(fmaf(s[i][t][8 * b + e], c, -ref));
                    if constexpr (F32) v[e] *= 0x1p15f;
                    if constexpr (!PAIRS) w.l[i] += v[e];
                }
                h8_t& hi = p[i][2 * t + b][0];
                hi = cvt8(v);
                if constexpr (PAIRS) {
                    const h2_t one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
                    for (int e = 0; e < 8; e += 2)
                        w.l[i] = __builtin_amdgcn_fdot2(h2_t{hi[e], hi[e + 1]}, one, w.l[i], false);
                }
                if constexpr (F32) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] -= (float)hi[e];
                    p[i][2 * t + b][1] = cvt8(v);
                }
            }
    }
}

// O^T += V^T P^T over 32 KT keys.
template <int HD, int QT, int KT, bool F32>
__device__ __forceinline__ void add_values(const char* V, Rows<HD, QT, F32>& w,
                                           const h8_t (&p)[QT][2 * KT][F32 ? 2 : 1]) {
    typedef Lay<HD> L;
    const int lane = threadIdx.x & 63;
    // 16 lanes read 16 dims of four keys; key bits 0-1 are (lane & 15) / 4
    const int r = 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int low = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
#pragma unroll
    for (int b = 0; b < 2 * KT; ++b)
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) {
            const char* at = V + (16 * b + r) * L::ROW + ((4 * d + low) ^ L::vx(r)) * 16 + (lane & 1) * 8;
            const char* at8 = V + (16 * b + 8 + r) * L::ROW + ((4 * d + low) ^ L::vx(8 + r)) * 16 + (lane & 1) * 8;
            typedef __attribute__((address_space(3))) s4_t lds4;
            const s4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)at);
            const s4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)at8);
            const h8_t v = __builtin_bit_cast(h8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int i = 0; i < QT; ++i)
#pragma unroll
                for (int part = 0; part < (F32 ? 2 : 1); ++part)
                    w.o[i][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[i][b][part], w.o[i][d], 0, 0, 0);
        }
}

// fp16 pairs with an exponent of all ones leave 0x8000 bits here.
__device__ __forceinline__ uint32_t odd_bits(uint32_t x) { return ((x & 0x7C007C00u) + 0x04000400u) & 0x80008000u; }
__device__ __forceinline__ uint32_t even_part(uint32_t x) { return x & ~((odd_bits(x) >> 15) * 0xFFFFu); }

// A step in which some row may not see some key: zeroes the values of keys that
// no row sees (key0 + row >= end, absent pages) and the others' that are NaN or infinite.
// Returns whether there are such (they come into the sums at the end, add_odd). `thread`
// of `threads` walks the tile.
template <int HD, int KEYS>
__device__ __forceinline__ bool zero_dead(char* V, int key0, int end, unsigned bad, int thread, int threads) {
    bool any = false;
    for (int u = thread; u < KEYS * (HD / 8); u += threads) {
        const int row = u / (HD / 8);
        uint4* at = reinterpret_cast<uint4*>(V + u * 16);
        if (key0 + row >= end || ((bad >> (row >> 4)) & 1)) {
            *at = make_uint4(0, 0, 0, 0);
        } else {
            const uint4 x = *at;
            if (odd_bits(x.x) | odd_bits(x.y) | odd_bits(x.z) | odd_bits(x.w)) {
                any = true;
                *at = make_uint4(even_part(x.x), even_part(x.y), even_part(x.z), even_part(x.w));
            }
        }
    }
    return any;
}

// The NaN and infinite values of keys from..to-1 in present pages, read from the cache, added to the
// rows that see them: rare, after the last step (the sums are final but for the division).
// (`read`(row, dim): four values of row `row` of a cache of head_dim columns)
template <int HD, int QT, bool F32, typename F>
__device__ __forceinline__ void add_odd(const AttnArgs& a, const Tile& t, int kh, int from, int to,
                                        Rows<HD, QT, F32>& w, F read) {
    const int h = (threadIdx.x & 63) >> 5, shift = a.c.block_shift;
    const int* table = a.b.table + t.seq * a.b.table_stride;
#pragma unroll 1
    for (int key = from; key < to; ++key) {
        const int id = table[key >> shift];
        if ((unsigned)id >= (unsigned)a.c.blocks) continue;
        const int64_t row = (((int64_t)id * a.c.kv_heads + kh) << shift) + (key & ((1 << shift) - 1));
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // dims 32 d + 8 e + 4 h ..
                const h4_t v = read(row, 32 * d + 8 * e + 4 * h);
                asm volatile("" ::: "memory");  // (a read at a time: few registers)
#pragma unroll
                for (int i = 0; i < QT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float x = (float)v[j];
                        w.o[i][d][4 * e + j] += key >= w.lo[i] && key <= w.hi[i] && !(fabsf(x) < INFINITY) ? x : 0.f;
                    }
            }
    }
}

// Four consecutive dims of a row to the output or, with several live splits, to the workspace.
__device__ __forceinline__ void put4(const AttnArgs& a, bool f16_out, bool whole, int64_t part, int token, int head,
                                     int hd, int dim, const float (&v)[4]) {
    if (whole) {
        if (f16_out) {
            uint2 u;
            u.x = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t{v[0], v[1]}), h2_t));
            u.y = __builtin_bit_cast(uint32_t, __builtin_convertvector((f2_t{v[2], v[3]}), h2_t));
            *reinterpret_cast<uint2*>(static_cast<_Float16*>(a.out) + (int64_t)token * a.ldo + head * hd + dim) = u;
        } else {
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + (int64_t)token * a.ldo + head * hd + dim) =
                make_float4(v[0], v[1], v[2], v[3]);
        }
    } else {
        *reinterpret_cast<float4*>(a.o + part * hd + dim) = make_float4(v[0], v[1], v[2], v[3]);
    }
}

// The factor of sums with reference m when they join others with reference `to` >= m (sums
// without a reference are 0, or NaN, which stays).
__device__ __forceinline__ float part_weight(float m, float l, float to) {
    return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(m - to);
}
__device__ __forceinline__ float reciprocal(float l) { return l == 0.f ? 0.f : 1.f / l; }  // (no key: zeros)
// The weight sum of a row that has seen keys, all of whose scores are -infinity: beside another part's sum it adds nothing,
// and alone its reciprocal is infinite, which makes the row's sums of 0 NaN.
constexpr float kNoWeight = 0x1p-140f;
// Whether any of keys from..to of the sequence is in a present page.
__device__ __forceinline__ bool sees_key(const AttnArgs& a, int seq, int from, int to) {
    if (from > to) return false;
    const int* table = a.b.table + seq * a.b.table_stride;
#pragma unroll 1
    for (int page = from >> a.c.block_shift; page <= to >> a.c.block_shift; ++page)
        if ((unsigned)table[page] < (unsigned)a.c.blocks) return true;
    return false;
}


// Items: see paged_attention.hip on few rows.
struct Item {
    int seq, tile, split, first, chunk, live;
    int part;  // its number among the items of split tiles
    Seq of;
};

// A sequence's tiles, and the first and the number of its keys.
template <int TM>
__device__ __forceinline__ void seq_size(const AttnArgs& a, const Seq& of, int* tiles, int* first, int* keys) {
    *tiles = (of.n * a.group + TM - 1) / TM;
    *first = a.window ? max(min(of.kv - of.n, a.cap) - a.window + 1, 0) & ~63 : 0;
    *keys = max(min(of.kv, a.cap) - *first, 0);
}
// 64-key units per item, for a batch of `total` units.
__device__ __forceinline__ int chunk_units(const AttnArgs& a, int64_t total, int units) {
    const int even = (int)min((total + a.splits - 1) / a.splits, (int64_t)(1 << 24));
    return max(max(even, a.min_chunk / 64), (units + kMaxSplits - 1) / kMaxSplits);
}
__device__ __forceinline__ int64_t sum_wave(int64_t v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor((long long)v, d);
    return v;
}

// A sequence's items: chunk (in units), live splits of each tile, items.
template <int TM>
__device__ __forceinline__ int seq_items(const AttnArgs& a, int64_t total, int tiles, int keys, int* chunk, int* live) {
    const int units = (keys + 63) >> 6;
    *chunk = chunk_units(a, total, units);
    *live = max((units + *chunk - 1) / *chunk, 1);
    return tiles * *live;
}
// Items, and those of split tiles in the upper half.
__device__ __forceinline__ unsigned long long both_counts(int items, int live) {
    return (unsigned long long)(live > 1 ? items : 0) << 32 | (unsigned)items;
}

// Item `number` of the batch (of 256 threads); false: there is none. Of the items only those of
// split tiles have partial results, and these are at most 2 `splits`: a tile of u units in chunks of c < u
// has at most 2 u / c. Up to kItemSeqs sequences every workgroup adds them up by itself, a sequence a
// thread; more are added up by a launch before (32/8 heads of 128, 100 to 300 positions each: 8192 sequences
// 1370 us, by every workgroup 4840; 512 sequences 95, 107).
constexpr int kItemSeqs = 256;

// LONG_FIRST (of at most kItemSeqs sequences): the last item of each tile, which is shorter than the others, comes after
// all those; a CU that is done with its long ones then finds short ones to fill the rest.
template <int TM, bool LONG_FIRST = false>
__device__ __forceinline__ bool find_item(const AttnArgs& a, int number, Item* item) {
    int tiles = 0, first = 0, keys = 0, chunk, live;
    if (a.items) {
        const int s = last_seq(a.b.seqs, [&](int i) { return a.items[i].x <= number; });
        const int2 from = a.items[s], sum = a.items[a.b.seqs];
        const Seq of = load_seq(a, s);
        seq_size<TM>(a, of, &tiles, &first, &keys);
        const int items = seq_items<TM>(a, (int64_t)sum.y << 32 | (unsigned)sum.x, tiles, keys, &chunk, &live);
        const int at = number - from.x;
        if (at < 0 || at >= items) return false;
        *item = Item{s, at / live, at % live, first, chunk * 64, live, from.y + at, of};
    } else {
        __shared__ unsigned long long upto_of[4];
        __shared__ int64_t totals[4];
        __shared__ Item found;
        const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
        Seq of{};
        if (t < a.b.seqs) {
            of = load_seq(a, t);
            seq_size<TM>(a, of, &tiles, &first, &keys);
        }
        if (t == 0) found.seq = -1;
        const unsigned long long upto_total = wave_scan((unsigned long long)tiles * (unsigned)((keys + 63) >> 6));
        if (lane == 63) totals[wave] = (int64_t)upto_total;
        __syncthreads();
        const int items = seq_items<TM>(a, totals[0] + totals[1] + totals[2] + totals[3], tiles, keys, &chunk, &live);
        if constexpr (LONG_FIRST) {
            __shared__ unsigned parts_of[4];
            // short items in the upper half, long ones in the lower
            const unsigned long long own = (unsigned long long)(unsigned)tiles << 32 | (unsigned)(tiles * (live - 1));
            const unsigned own_parts = live > 1 ? items : 0;
            const unsigned long long upto = wave_scan(own);
            const unsigned upto_parts = wave_scan(own_parts);
            if (lane == 63) upto_of[wave] = upto, parts_of[wave] = upto_parts;
            __syncthreads();
            unsigned long long from = upto - own;
            unsigned part = upto_parts - own_parts, longs = 0;
            for (int w = 0; w < 4; ++w) {
                from += w < wave ? upto_of[w] : 0;
                part += w < wave ? parts_of[w] : 0;
                longs += (unsigned)upto_of[w];
            }
            const bool is_long = (unsigned)number < longs;
            const int at = is_long ? number - (int)(unsigned)from : number - (int)longs - (int)(from >> 32);
            if (at >= 0 && at < (is_long ? tiles * (live - 1) : tiles)) {
                const int tile = is_long ? at / (live - 1) : at, split = is_long ? at % (live - 1) : live - 1;
                found = Item{t, tile, split, first, chunk * 64, live, (int)part + tile * live + split, of};
            }
        } else {
            const unsigned long long own = both_counts(items, live), upto = wave_scan(own);
            if (lane == 63) upto_of[wave] = upto;
            __syncthreads();
            unsigned long long from = upto - own;
            for (int w = 0; w < 3; ++w) from += w < wave ? upto_of[w] : 0;
            const int at = number - (int)(unsigned)from;
            if (at >= 0 && at < items)
                found = Item{t, at / live, at % live, first, chunk * 64, live, (int)(from >> 32) + at, of};
        }
        __syncthreads();
        if (found.seq < 0) return false;
        *item = found;
    }
    item->seq = __builtin_amdgcn_readfirstlane(item->seq);
    item->tile = __builtin_amdgcn_readfirstlane(item->tile);
    item->split = __builtin_amdgcn_readfirstlane(item->split);
    item->first = __builtin_amdgcn_readfirstlane(item->first);
    item->chunk = __builtin_amdgcn_readfirstlane(item->chunk);
    item->live = __builtin_amdgcn_readfirstlane(item->live);
    item->part = __builtin_amdgcn_readfirstlane(item->part);
    item->of.token0 = __builtin_amdgcn_readfirstlane(item->of.token0);
    item->of.n = __builtin_amdgcn_readfirstlane(item->of.n);
    item->of.kv = __builtin_amdgcn_readfirstlane(item->of.kv);
    return true;
}

// The waves' sums of an item, joined and written: to the output, or as the item's part; PARTS of the row's dims
// after each other, each wave's in its own 128 HD / PARTS bytes of LDS (32 rows, 16-byte pieces XORed with the row).
// `begin`..`end`: the item's keys, of which wave i took every fourth step of KEYS from begin + i KEYS on.
template <int HD, bool F32, int KEYS, int PARTS = 1>
__device__ __forceinline__ void finish_few(const AttnArgs& a, const Tile& t, const Item& item, int kh, int begin, int end,
                                           int64_t part0, const Rows<HD, 1, F32>& w, char* lds) {
    constexpr int TM = 32, ROW = HD / PARTS * 4, PCS = ROW / 16, X = PCS < 16 ? PCS - 1 : 15, BYTES = TM * ROW;
    __shared__ float2 sums[4][32];
    const bool whole = item.live <= 1;
    const int seq = item.seq, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* K = lds + wave * BYTES;
    const int q = lane & 31, h = lane >> 5;
    float l = 0.f;
    const int rows = min(t.rows - t.row0, TM);
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        if (p) __syncthreads();
#pragma unroll
        for (int d = 0; d < HD / 32 / PARTS; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int piece = (32 * d + 8 * e + 4 * h) / 4, at = p * (HD / 32 / PARTS) + d;
                *reinterpret_cast<float4*>(K + q * ROW + (piece ^ (q & X)) * 16) =
                    make_float4(w.o[0][at][4 * e], w.o[0][at][4 * e + 1], w.o[0][at][4 * e + 2], w.o[0][at][4 * e + 3]);
            }
        if (p == 0) {
            l = swap32_sum(w.l[0]);
            // (the wave's keys and what lies between: a row that sees one of those has its weight in another wave)
            if (l == 0.f && sees_key(a, seq, max(w.lo[0], begin + wave * KEYS), min(w.hi[0], end - 1))) l = kNoWeight;
            if (h == 0) sums[wave][q] = make_float2(w.m[0], l);
        }
        __syncthreads();
        if (p == 0 && a.info && kh == 0 && item.split == 0)
            for (int u = threadIdx.x; u < rows; u += 256)
                a.info[(int64_t)t.token0 * a.group + t.row0 + u] = make_int2(item.live, item.part << 5 | u);
        for (int u = threadIdx.x; u < rows * PCS; u += 256) {
            const int row = u / PCS, piece = u % PCS;
            float m = sums[0][row].x, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 1; i < 4; ++i) m = fmaxf(m, sums[i][row].x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 ml = sums[i][row];
                const float f = part_weight(ml.x, ml.y, m);
                const float4 x = *reinterpret_cast<const float4*>(lds + i * BYTES + row * ROW + (piece ^ (row & X)) * 16);
                sum = fmaf(f, ml.y, sum);
                v[0] = fmaf(f, x.x, v[0]), v[1] = fmaf(f, x.y, v[1]), v[2] = fmaf(f, x.z, v[2]), v[3] = fmaf(f, x.w, v[3]);
            }
            const int tok = (t.row0 + row) / a.group, head = kh * a.group + (t.row0 + row) % a.group;
            const int64_t part = a.most ? ((int64_t)item.split * a.b.tokens + t.token0 + tok) * (a.group * a.c.kv_heads) + head
                                        : part0 + row;
            if (whole) {
                const float inv = reciprocal(sum);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] *= inv;
            } else if (p == 0 && piece == 0) {
                a.ml[part] = make_float2(m, sum);
            }
            put4(a, !F32, whole, part, t.token0 + tok, head, HD, p * (HD / PARTS) + 4 * piece, v);
        }
    }
}

// A wave's rows of a large tile, written: to the output, or as the split's part.
template <int HD, bool F32>
__device__ __forceinline__ void finish_many(const AttnArgs& a, const Tile& t, int kh, int split, int begin, int end,
                                            int row, const Rows<HD, 1, F32>& w) {
    const int lane = threadIdx.x & 63;
    const bool whole = t.live <= 1;
    const int h = lane >> 5, r = row + (lane & 31);
    float l = swap32_sum(w.l[0]);
    if (l == 0.f && sees_key(a, t.seq, max(w.lo[0], begin), min(w.hi[0], end - 1))) l = kNoWeight;
    const float f = whole ? reciprocal(l) : 1.f;
    if (r >= t.rows) return;
    const int tok = t.token0 + r / a.group, head = kh * a.group + r % a.group;
    const int64_t part = ((int64_t)split * a.b.tokens + tok) * (a.group * a.c.kv_heads) + head;
    if (!whole && h == 0) a.ml[part] = make_float2(w.m[0], l);
    if (a.info && kh == 0 && split == 0 && h == 0) a.info[(int64_t)t.token0 * a.group + r] = make_int2(t.live, 0);
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float v[4] = {w.o[0][d][4 * e] * f, w.o[0][d][4 * e + 1] * f, w.o[0][d][4 * e + 2] * f,
                                w.o[0][d][4 * e + 3] * f};
            put4(a, !F32, whole, part, tok, head, HD, 32 * d + 8 * e + 4 * h, v);
        }
}

}  // namespace

}  // namespace rq
