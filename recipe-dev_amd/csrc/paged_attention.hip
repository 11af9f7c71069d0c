// Attention of several sequences' new tokens over their pages
// (rqmv_paged_attention).
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
// Keys and values go from the pages straight into LDS (global_load_lds, 16
// bytes a lane), 16 keys of one page at a time, 32 or 64 keys per step. A row's
// 16-byte pieces are stored XORed with the row number, so that the operand reads
// hit every bank once.
//
// Masked places: a masked score is -infinity by selection, and V must not meet
// its zero weight as a NaN: in steps where some row may not see some key, the
// values of keys that no row sees are zeroed in LDS, and so are NaN and infinite
// ones of the others; where there are such, they are read again from the cache
// after the last step and added to the rows that see them.
#include "lanes.h"
#include "paged.h"

#include <float.h>
#include <limits.h>

#include "halfcode.h"

namespace rq {

namespace {

typedef float f16_t __attribute__((ext_vector_type(16)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef short s4_t __attribute__((ext_vector_type(4)));

constexpr int kMaxSplits = 64;  // of one tile's keys
constexpr int64_t kEarlyBytes = int64_t(1) << 20;  // of parts that a join may ask for unseen

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

// The 16 keys from `key` on of one page (id clamped into the cache) of `cache`, to LDS.
template <int HD, bool VALUES>
__device__ __forceinline__ void load_group(const __half* cache, const PagedCache& c, int kh, int id, int key,
                                           uint32_t lds) {
    typedef Lay<HD> L;
    const int lane = threadIdx.x & 63;
    const int64_t row = (((int64_t)id * c.kv_heads + kh) << c.block_shift) + (key & ((1 << c.block_shift) - 1));
    const __half* base = cache + row * HD;
#pragma unroll
    for (int i = 0; i < L::NI; ++i) {
        const int r = i * L::RPI + lane / L::PCS;
        const int piece = (lane % L::PCS) ^ (VALUES ? L::vx(r) : L::kx(r));
        load_lds(base, (uint32_t)(r * L::ROW + piece * 16), lds + i * 1024);
    }
}

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
template <int HD, bool F32>
__device__ __forceinline__ void load_rows(const AttnArgs& a, const Tile& t, int kh, int row, Rows<HD, 1, F32>& w,
                                          RawRows<HD, F32>& raw) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int r = min(row + (lane & 31), t.rows - 1);  // (rows past the last repeat it)
    const int tok = r / a.group, pos = t.kv - t.n + tok;
    const int64_t at = (int64_t)(t.token0 + tok) * a.ldq + (kh * a.group + r % a.group) * HD + 8 * h;
    w.hi[0] = min(pos, a.cap - 1);
    w.lo[0] = a.window ? pos - a.window + 1 : 0;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
        if constexpr (F32) {
            const float* src = static_cast<const float*>(a.q) + at + 16 * k;
            raw.v[k][0] = *reinterpret_cast<const float4*>(src);
            raw.v[k][1] = *reinterpret_cast<const float4*>(src + 4);
        } else {
            w.q[0][k][0] = *reinterpret_cast<const h8_t*>(static_cast<const _Float16*>(a.q) + at + 16 * k);
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
template <int HD, int QT, bool F32>
__device__ __forceinline__ void add_odd(const AttnArgs& a, const Tile& t, int kh, int from, int to,
                                        Rows<HD, QT, F32>& w) {
    typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
    const int h = (threadIdx.x & 63) >> 5, shift = a.c.block_shift;
    const int* table = a.b.table + t.seq * a.b.table_stride;
#pragma unroll 1
    for (int key = from; key < to; ++key) {
        const int id = table[key >> shift];
        if ((unsigned)id >= (unsigned)a.c.blocks) continue;
        const _Float16* row = reinterpret_cast<const _Float16*>(a.c.v) +
                              ((((int64_t)id * a.c.kv_heads + kh) << shift) + (key & ((1 << shift) - 1))) * HD + 4 * h;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // dims 32 d + 8 e + 4 h ..
                const h4_t v = *reinterpret_cast<const h4_t*>(row + 32 * d + 8 * e);
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

// ------------------------------------------- few rows: keys over the waves ----

// At most 32 rows a tile (a decode step, a few speculated tokens): bound by
// reading the keys and values.
//
// Items. The lengths are known on the device alone, and may differ by orders of magnitude: every
// workgroup adds up the batch's keys and cuts each tile's into chunks of one length, about
// total / `splits`, so that tiles + splits items per kv head suffice whatever the
// lengths are, and finds its own among them.
//
// Each of four waves takes every fourth step of 32
// keys of the split into LDS of its own, without barriers; its K buffer is filled
// again while it works on the values and the other way round, and a second workgroup
// on the CU fills the rest. At the end the waves' sums are joined through LDS.
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

// The first item of each sequence and the first of its partial results; behind them the total.
template <int TM>
__global__ void __launch_bounds__(1024) paged_items_kernel(AttnArgs a, int2* out) {
    __shared__ unsigned long long upto_of[16];
    __shared__ int64_t totals[16];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int tiles, first, keys, chunk, live;
    int64_t total = 0;
    for (int s = t; s < a.b.seqs; s += 1024) {
        seq_size<TM>(a, load_seq(a, s), &tiles, &first, &keys);
        total += (int64_t)tiles * ((keys + 63) >> 6);
    }
    total = sum_wave(total);
    if (lane == 0) totals[wave] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < 16; ++w) total += totals[w];
    unsigned long long before = 0;
    for (int s0 = 0; s0 < a.b.seqs; s0 += 1024) {
        const int s = s0 + t;
        unsigned long long own = 0;
        if (s < a.b.seqs) {
            seq_size<TM>(a, load_seq(a, s), &tiles, &first, &keys);
            const int items = seq_items<TM>(a, total, tiles, keys, &chunk, &live);
            own = both_counts(items, live);
        }
        const unsigned long long upto = wave_scan(own);
        __syncthreads();
        if (lane == 63) upto_of[wave] = upto;
        __syncthreads();
        unsigned long long from = before + upto - own;
        for (int w = 0; w < 16; ++w) {
            from += w < wave ? upto_of[w] : 0;
            before += upto_of[w];
        }
        if (s < a.b.seqs) out[s] = make_int2((int)(unsigned)from, (int)(from >> 32));
    }
    if (t == 0) out[a.b.seqs] = make_int2((int)(unsigned)total, (int)(total >> 32));
}

template <int TM>
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
        const int64_t own_total = sum_wave((int64_t)tiles * ((keys + 63) >> 6));
        if (lane == 0) totals[wave] = own_total;
        __syncthreads();
        const int items = seq_items<TM>(a, totals[0] + totals[1] + totals[2] + totals[3], tiles, keys, &chunk, &live);
        const unsigned long long own = both_counts(items, live), upto = wave_scan(own);
        if (lane == 63) upto_of[wave] = upto;
        __syncthreads();
        unsigned long long from = upto - own;
        for (int w = 0; w < 3; ++w) from += w < wave ? upto_of[w] : 0;
        const int at = number - (int)(unsigned)from;
        if (at >= 0 && at < items)
            found = Item{t, at / live, at % live, first, chunk * 64, live, (int)(from >> 32) + at, of};
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

template <int HD, bool F32>
__global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) paged_few_kernel(AttnArgs a) {
    typedef Lay<HD> L;
    constexpr int TM = 32, KEYS = 32, HALF = KEYS * HD * 2;  // HALF: bytes of a wave's K (and V) buffer
    extern __shared__ __align__(16) char lds[];
    __shared__ float2 sums[4][32];
    const int kh = blockIdx.x % a.c.kv_heads;
    Item item;
    if (!find_item<TM>(a, blockIdx.x / a.c.kv_heads, &item)) return;
    // (starts out of order may count past what the workspace holds)
    const bool whole = item.live <= 1;
    const int64_t part0 = ((int64_t)item.part * a.c.kv_heads + kh) * TM;
    if (!whole && (a.most ? item.split >= a.most : part0 < 0 || part0 + TM > a.parts)) return;
    const int seq = item.seq;
    const Tile t = make_tile<TM>(a, seq, item.of, item.tile * TM);
    const int begin = item.first + item.split * item.chunk, end = min(begin + item.chunk, t.end);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* K = lds + wave * 2 * HALF;
    char* V = K + HALF;
    const uint32_t k_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)K, v_lds = k_lds + HALF;
    Pages pages{a.b.table + seq * a.b.table_stride, a.b.max_blocks - 1, a.c.blocks, a.c.block_shift, INT_MIN / 2, 0};
    Rows<HD, 1, F32> w;

    int id[2], next[2];
    auto look = [&](int key0, int (&ids)[2]) {  // the page ids of keys key0.. and key0 + 16..
        const int p0 = key0 >> pages.shift, p1 = (key0 + 16) >> pages.shift;
        pages.need(p0, p1);
        ids[0] = pages.at(p0);
        ids[1] = pages.at(p1);
    };
    auto load = [&](auto values, int key0, const int (&ids)[2]) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
            load_group<HD, decltype(values)::value>(decltype(values)::value ? a.c.v : a.c.k, a.c, kh,
                                                    pages.absent(ids[g]) ? 0 : ids[g], key0 + 16 * g,
                                                    (decltype(values)::value ? v_lds : k_lds) + g * 16 * L::ROW);
    };
    int key0 = begin + wave * KEYS;
    bool odd = false;
    if (key0 < end) pages.fetch(key0 >> pages.shift);
    RawRows<HD, F32> raw;
    if constexpr (F32) {  // (they are converted while the first step is on its way)
        load_rows<HD, F32>(a, t, kh, t.row0, w, raw);
        arrived(w, raw);
    }
    if (key0 < end) {
        look(key0, id);
        load(std::false_type{}, key0, id);
        load(std::true_type{}, key0, id);
    }
    if constexpr (!F32) {
        load_rows<HD, F32>(a, t, kh, t.row0, w, raw);
        arrived(w, raw);
    }
    start_rows(a, w, raw);
    while (key0 < end) {
        const int after = key0 + 4 * KEYS;
        const bool more = after < end;
        wait_loads<2 * L::NI>();  // K (V's loads were issued after it)
        f16_t s[1][1];
        scores<HD, 1, 1, F32>(K, w, s);
        if (more) {
            look(after, next);
            // the operand reads have returned (their products are the scores)
            asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(s[0][0]) : : "memory");
            load(std::false_type{}, after, next);
        }
        const unsigned bad = (pages.absent(id[0]) ? 1 : 0) | (pages.absent(id[1]) ? 2 : 0);
        const bool masked = key0 < t.all_from || key0 + KEYS > t.all_to || bad;
        if (masked) mask_scores<HD, 1, 1, F32>(w, s, key0, bad);
        float top[1];
        largest<1, 1>(s, top);
        move_references<HD, 1, F32>(w, top);
        h8_t p[1][2][F32 ? 2 : 1];
        weights<HD, 1, 1, F32>(w, s, p);
        if (more) wait_loads<2 * L::NI>();
        else wait_loads<0>();
        if (masked && __any(zero_dead<HD, KEYS>(V, key0, t.end, bad, lane, 64))) odd = true;
        add_values<HD, 1, 1, F32>(V, w, p);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(w.o[0][0]) : : "memory");
            load(std::true_type{}, after, next);
            id[0] = next[0], id[1] = next[1];
        }
        key0 = after;
    }
    wait_loads<0>();
    if (odd) {  // (the wave's own steps; what unmasked ones let through is there already, and stays)
        for (int k = begin + wave * KEYS; k < end; k += 4 * KEYS)
            add_odd<HD, 1, F32>(a, t, kh, k, min(k + KEYS, t.end), w);
    }
    // the waves' sums, each in its own LDS (32 rows of HD values, pieces XORed with the row)
    const int q = lane & 31, h = lane >> 5;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int piece = (32 * d + 8 * e + 4 * h) / 4;
            *reinterpret_cast<float4*>(K + q * HD * 4 + (piece ^ (q & 15)) * 16) =
                make_float4(w.o[0][d][4 * e], w.o[0][d][4 * e + 1], w.o[0][d][4 * e + 2], w.o[0][d][4 * e + 3]);
        }
    float l = swap32_sum(w.l[0]);
    // (the wave's keys and what lies between: a row that sees one of those has its weight in another wave)
    if (l == 0.f && sees_key(a, seq, max(w.lo[0], begin + wave * KEYS), min(w.hi[0], end - 1))) l = kNoWeight;
    if (h == 0) sums[wave][q] = make_float2(w.m[0], l);
    __syncthreads();
    const int rows = min(t.rows - t.row0, TM);
    if (a.info && kh == 0 && item.split == 0)
        for (int u = threadIdx.x; u < rows; u += 256)
            a.info[(int64_t)t.token0 * a.group + t.row0 + u] = make_int2(item.live, item.part << 5 | u);
    for (int u = threadIdx.x; u < rows * (HD / 4); u += 256) {
        const int row = u / (HD / 4), piece = u % (HD / 4);
        float m = sums[0][row].x, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 1; i < 4; ++i) m = fmaxf(m, sums[i][row].x);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 ml = sums[i][row];
            const float f = part_weight(ml.x, ml.y, m);
            const float4 x = *reinterpret_cast<const float4*>(lds + i * 2 * HALF + row * HD * 4 + (piece ^ (row & 15)) * 16);
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
        } else if (piece == 0) {
            a.ml[part] = make_float2(m, sum);
        }
        put4(a, !F32, whole, part, t.token0 + tok, head, HD, 4 * piece, v);
    }
}

// --------------------------------------------- many rows: rows over the waves ----

// TM = 32 WAVES rows a tile (prompts, chunks of prompts): bound by the matrix
// cores and the exponentials. Each wave has 32 rows; the waves share steps of 64 keys in
// two LDS buffers, one barrier a step. Eight waves (two per SIMD, 256 registers each), so
// that one multiplies while the other takes exponentials; at 256 dims four, which may have 512 registers
// (fp16 takes 291, fp32 363; fp16 in 256 registers, with steps of 32 keys, spilled inside the loop, and the
// reloads waited for the step's own loads to LDS: 2048 tokens over 6,000, 32/8 heads, 1,015 us against 659).
// 2048 tokens over 14,336, 32/8 heads of 128, fp16: 509 to 533 us by the card, 1,012 to 967 TFLOP/s (a library product
// of 8192^3: 1,162 to 1,145). Four waves of 64 rows took 1,224 us: their sums lay in accumulator registers and were
// moved at every step.
constexpr int many_waves(int hd) { return hd == 256 ? 4 : 8; }

template <int HD, bool F32>
__global__ void __launch_bounds__(64 * many_waves(HD), many_waves(HD) / 4) paged_many_kernel(AttnArgs a) {
    typedef Lay<HD> L;
    constexpr int WAVES = many_waves(HD), TM = 32 * WAVES, KEYS = 64, KT = KEYS / 32;
    constexpr int HALF = KEYS * HD * 2;
    extern __shared__ __align__(16) char lds[];
    // the last tiles first: of one sequence's they have the most keys
    const int kh = blockIdx.x % a.c.kv_heads, number = a.tiles - 1 - blockIdx.x / a.c.kv_heads, split = blockIdx.y;
    const int seq = find_seq<TM>(a.b, a.group, number);
    const int first = start_of(a.b, seq) * a.group / TM + seq;
    const Tile t = make_tile<TM>(a, seq, load_seq(a, seq), (number - first) * TM);
    if (t.row0 < 0 || t.row0 >= t.rows) return;  // (below 0: starts out of order)
    const int begin = t.first + split * t.chunk, end = min(begin + t.chunk, t.end);
    if (split && begin >= end) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = t.row0 + 32 * wave;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
    Pages pages{a.b.table + seq * a.b.table_stride, a.b.max_blocks - 1, a.c.blocks, a.c.block_shift, INT_MIN / 2, 0};
    Rows<HD, 1, F32> w;

    // Step i is in buffer i % 2, keys before values. Of eight waves, four load 16 rows of keys each and
    // four of values; of four, each loads both. Returns which groups are absent.
    auto load = [&](int key0, int buffer) -> unsigned {
        pages.need(key0 >> pages.shift, (key0 + KEYS - 16) >> pages.shift);
        unsigned bad = 0;
#pragma unroll
        for (int g = 0; g < KEYS / 16; ++g) bad |= pages.absent(pages.at((key0 + 16 * g) >> pages.shift)) ? 1u << g : 0u;
        const int g = wave % (KEYS / 16), key = key0 + 16 * g, id = pages.at(key >> pages.shift);
        const int page = pages.absent(id) ? 0 : id;
        const uint32_t at = lds0 + buffer * 2 * HALF + g * 16 * L::ROW;
        if (WAVES == 4 || wave < 4) load_group<HD, false>(a.c.k, a.c, kh, page, key, at);
        if (WAVES == 4 || wave >= 4) load_group<HD, true>(a.c.v, a.c, kh, page, key, at + HALF);
        return bad;
    };
    // the keys that any of the wave's rows sees
    const int p0 = t.kv - t.n + row / a.group, p1 = t.kv - t.n + (min(row + 32, t.rows) - 1) / a.group;
    const int wave_to = row < t.rows ? p1 + 1 : 0, wave_from = a.window ? p0 - a.window + 1 : 0;
    unsigned bad = 0, bad_next = 0;
    int buffer = 0;
    bool odd = false;
    if (begin < end) pages.fetch(begin >> pages.shift);
    RawRows<HD, F32> raw;
    load_rows<HD, F32>(a, t, kh, row, w, raw);
    arrived(w, raw);
    if (begin < end) bad = load(begin, 0);
    start_rows(a, w, raw);
    for (int key0 = begin; key0 < end; key0 += KEYS) {
        wait_loads<0>();
        __syncthreads();  // the step is in LDS, and the other buffer is free
        if (key0 + KEYS < end) bad_next = load(key0 + KEYS, buffer ^ 1);
        char* K = lds + buffer * 2 * HALF;
        char* V = K + HALF;
        const bool masked = key0 < t.all_from || key0 + KEYS > t.all_to || bad;
        if (masked && __syncthreads_or(zero_dead<HD, KEYS>(V, key0, t.end, bad, threadIdx.x, 64 * WAVES))) odd = true;
        if (key0 < wave_to && key0 + KEYS > wave_from) {  // (a wave whose rows see none of the step only loads)
            f16_t s[1][KT];
            scores<HD, 1, KT, F32>(K, w, s);
            if (masked) mask_scores<HD, 1, KT, F32>(w, s, key0, bad);
            float top[1];
            largest<1, KT>(s, top);
            move_references<HD, 1, F32>(w, top);
            h8_t p[1][2 * KT][F32 ? 2 : 1];
            weights<HD, 1, KT, F32>(w, s, p);
            add_values<HD, 1, KT, F32>(V, w, p);
        }
        bad = bad_next;
        buffer ^= 1;
    }
    if (odd) add_odd<HD, 1, F32>(a, t, kh, begin, end, w);
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

// ---------------------------------------------------------- the splits' join ----

// out = sum_c 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c over a row's live splits (EARLY: of all places that
// there are, before it is known which hold one). HD / 4
// threads take a split's 16-byte columns, SIDE of them in a row (token, query head) take every
// SIDE-th split, four at a time.
template <int HD, int SIDE, bool F32, bool EARLY>
__global__ void __launch_bounds__(256) paged_join_kernel(AttnArgs a) {
    constexpr int TPR = HD / 4, ROWS = 256 / (TPR * SIDE);
    __shared__ float4 part[SIDE > 1 ? 256 : 1];
    __shared__ float2 sums[SIDE > 1 ? SIDE : 1];
    const int heads = a.group * a.c.kv_heads;
    const int64_t unit = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * ROWS + threadIdx.x / (TPR * SIDE);
    if (unit >= (int64_t)a.b.tokens * heads) return;  // (SIDE > 1: a row per workgroup, all of it leaves)
    const int token = (int)(unit / heads), head = (int)(unit % heads), kh = head / a.group;
    const int col = threadIdx.x % TPR, side = threadIdx.x / TPR % SIDE;
    const int2 info = a.info[(int64_t)token * a.group + head % a.group];
    const int from = a.b.q_start[0], to = a.b.q_start[a.b.seqs];
    // (rows of no sequence have no info; that of rows of starts out of order may be an older call's)
    int live = info.x, most = a.most;
    int64_t at = unit, next = (int64_t)a.b.tokens * heads;
    if (!EARLY) {
        if (token < from || token >= to || live <= 1 || live > kMaxSplits) return;
        most = live;
        if (!a.most) {
            at = ((int64_t)(info.y >> 5) * a.c.kv_heads + kh) * 32 + (info.y & 31);
            next = (int64_t)a.c.kv_heads * 32;
        }
        if (at < 0 || at + (live - 1) * next >= a.parts) return;
    }
    float m = -INFINITY, sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](float2 ml, float4 x) {
        const float to = fmaxf(m, ml.x);
        const float f = part_weight(m, sum, to), g = part_weight(ml.x, ml.y, to);
        m = to;
        sum = f * sum + g * ml.y;
        v[0] = f * v[0] + g * x.x, v[1] = f * v[1] + g * x.y, v[2] = f * v[2] + g * x.z, v[3] = f * v[3] + g * x.w;
    };
    for (int c = side; c < most; c += 4 * SIDE) {
        float4 x[4];
        float2 ml[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t row = at + min(c + k * SIDE, most - 1) * next;
            x[k] = *reinterpret_cast<const float4*>(a.o + row * HD + 4 * col);
            ml[k] = a.ml[row];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c + k * SIDE < live) add(ml[k], x[k]);
    }
    if (EARLY && (token < from || token >= to || live <= 1 || live > most)) return;
    if constexpr (SIDE > 1) {
        part[threadIdx.x] = make_float4(v[0], v[1], v[2], v[3]);
        if (col == 0) sums[side] = make_float2(m, sum);
        __syncthreads();
        if (side) return;
#pragma unroll
        for (int k = 1; k < SIDE; ++k) add(sums[k], part[k * TPR + col]);
    }
    const float inv = reciprocal(sum);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= inv;
    put4(a, !F32, true, 0, token, head, HD, 4 * col, v);
}

// ------------------------------------------------------------------ launches ----

constexpr int few_lds(int hd) { return 4 * 2 * 32 * hd * 2; }
constexpr int many_lds(int hd) { return 2 * 2 * 64 * hd * 2; }

struct AttnPlan {
    bool few, join, items;
    int splits, min_chunk, most;
    int64_t tiles, parts;
};

AttnPlan plan_attention(int tokens, int seqs, int64_t cap, int kv_heads, int group, int hd, bool f32, int cus) {
    AttnPlan p;
    const int heads = kv_heads * group;
    // The few-rows form up to 128 rows a sequence and kv head on average, or where there are so few that
    // the large tiles leave CUs idle: tiles of 32 rows over all heads up to 4 a CU (64 and 256 dims, fp16),
    // 2 (128 dims; 64, fp32) or a half (256, fp32, whose large tiles have 128 rows). Over 222
    // batches of 1 to 16 sequences, 64 to 1024 new tokens and 0 to 6,000 cached ones the choice takes 0.5 to
    // 4.5 % more than the better form; at 256 dims of fp16 11 % over 131 batches. Few against many, 32/8 heads of 128,
    // fp16, us: 32 sequences of 128 rows over 6,000 positions 238 / 341, of 256 398 / 350; one of 1024 rows over 1,000
    // 23 / 27; four of 2048 over 6,000 350 / 221. One form takes the whole batch: 100 decoding requests over 2,000 beside
    // 2048 tokens over 6,000 take 494 (few), as two batches 157 + 255; 32 beside them 298 (many), 53 + 255.
    p.tiles = (int64_t)tokens * group / 32 + seqs;
    const int64_t few_tiles = hd == 128 ? 2 * cus : hd == 64 ? (f32 ? 2 : 4) * cus : f32 ? cus / 2 : 4 * cus;
    p.few = (int64_t)tokens * group <= (int64_t)128 * seqs || (int64_t)tokens * heads / 32 <= few_tiles;
    p.items = p.few && seqs > kItemSeqs;
    if (p.few) {
        // Two items per CU over the whole batch (32 requests of 60 to 8,192 positions, with the join: 39.1 us; one
        // per CU 41.2, four 41.3), of two steps for each wave at least (one request at 4,097: 12.4 us; of
        // one step 14.8, of four 14.6; the 32 requests with a window of 1,024 24.3, of four 20.3).
        p.min_chunk = 256;
        const int64_t want = 2 * cus / kv_heads, most = p.tiles * ((cap + p.min_chunk - 1) / p.min_chunk);
        p.splits = (int)(most < want ? most : want < 1 ? 1 : want);
        p.join = cap > p.min_chunk;
        p.parts = p.join ? (int64_t)2 * p.splits * kv_heads * 32 : 0;
        // Parts have fixed places where all that there could be take up to 1 MiB: the join then asks for them before
        // it knows which there are (one token over 4,096, 0.3 MB: 12.4 us, otherwise 13.0; 40 over up to 3,000, 8 MB:
        // 26.4 so, 25.8 otherwise).
        const int64_t all = (cap + p.min_chunk - 1) / p.min_chunk;
        p.most = (int)(all < kMaxSplits ? all : kMaxSplits);
        if (!p.join || (int64_t)tokens * heads * p.most * hd * 4 > kEarlyBytes) p.most = 0;
        else p.parts = (int64_t)tokens * heads * p.most;
    } else {
        p.tiles = (int64_t)tokens * group / (32 * many_waves(hd)) + seqs;
        // Keys are split where the tiles take at most half of the CUs (at less, a split's uneven second part
        // costs more than it gives: eight sequences of 300 tokens, 8/4 heads of 256, 41 us split, 25 whole).
        p.min_chunk = 128;
        const int64_t wgs = p.tiles * kv_heads;
        int64_t s = cus / wgs;
        const int64_t most = (cap + p.min_chunk - 1) / p.min_chunk;
        if (s > most) s = most;
        p.splits = (int)(s > kMaxSplits ? kMaxSplits : s < 1 ? 1 : s);
        p.join = p.splits > 1;
        p.parts = p.join ? (int64_t)p.splits * tokens * heads : 0;
        p.most = p.splits;
    }
    return p;
}

size_t workspace_bytes(const AttnPlan& p, int tokens, int seqs, int group, int hd) {
    return (p.join ? p.parts * (hd * sizeof(float) + sizeof(float2)) + (size_t)tokens * group * sizeof(int2) : 0) +
           (p.items ? ((size_t)seqs + 1) * sizeof(int2) : 0);
}

template <int HD, bool F32>
hipError_t launch_attention_hd(const AttnPlan& p, const AttnArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)((p.tiles + (p.few ? p.splits : 0)) * a.c.kv_heads), p.few ? 1 : p.splits);
    const void* f = p.few ? reinterpret_cast<const void*>(paged_few_kernel<HD, F32>)
                          : reinterpret_cast<const void*>(paged_many_kernel<HD, F32>);
    const int lds = p.few ? few_lds(HD) : many_lds(HD);
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    if (p.few) hipLaunchKernelGGL((paged_few_kernel<HD, F32>), grid, dim3(256), lds, stream, a);
    else hipLaunchKernelGGL((paged_many_kernel<HD, F32>), grid, dim3(64 * many_waves(HD)), lds, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.join) return e;
    // A workgroup per row for few of them, for 1024 / HD rows of many (eight sequences of 300 tokens, 16 heads of
    // 64: 24 us less). One row of 33 splits: 3.8 us by a workgroup, 6.3 by HD / 4 threads.
    const int64_t rows = (int64_t)a.b.tokens * a.group * a.c.kv_heads;
    constexpr int SIDE = 1024 / HD;
    // (2^26 rows of 256 dims are 2^24 workgroups, more threads than a grid's one dimension holds)
    const unsigned groups = (unsigned)((rows + SIDE - 1) / SIDE), across = groups < (1u << 20) ? groups : 1u << 20;
    const dim3 wide((unsigned)rows), narrow(across, (groups - 1) / across + 1), threads(256);
    if (p.few && p.most) hipLaunchKernelGGL((paged_join_kernel<HD, SIDE, F32, true>), wide, threads, 0, stream, a);
    else if (rows <= 2048) hipLaunchKernelGGL((paged_join_kernel<HD, SIDE, F32, false>), wide, threads, 0, stream, a);
    else hipLaunchKernelGGL((paged_join_kernel<HD, 1, F32, false>), narrow, threads, 0, stream, a);
    return hipGetLastError();
}

}  // namespace

bool paged_attention_fits(const PagedBatch& b, const PagedCache& c, int q_heads) {
    return ((int64_t)b.tokens * (q_heads / c.kv_heads) / 32 + b.seqs) * c.kv_heads <= (1 << 23) &&
           (int64_t)b.tokens * q_heads <= (1 << 26);
}

size_t paged_attention_workspace(const PagedBatch& b, const PagedCache& c, int q_heads, int cus) {
    const int group = q_heads / c.kv_heads;
    const int64_t cap = (int64_t)b.max_blocks << c.block_shift;
    size_t most = 0;
    for (const bool f32 : {false, true}) {  // (one workspace serves both types)
        const AttnPlan p = plan_attention(b.tokens, b.seqs, cap, c.kv_heads, group, c.head_dim, f32, cus);
        const size_t bytes = workspace_bytes(p, b.tokens, b.seqs, group, c.head_dim);
        most = bytes > most ? bytes : most;
    }
    return most;
}

hipError_t launch_paged_attention(const PagedBatch& b, const PagedCache& c, const void* q, bool f32, int64_t ldq,
                                  int q_heads, float scale, int window, void* workspace, void* out, int64_t ldo, int cus,
                                  hipStream_t stream) {
    const int group = q_heads / c.kv_heads;
    const int64_t cap = (int64_t)b.max_blocks << c.block_shift;
    const AttnPlan p = plan_attention(b.tokens, b.seqs, cap, c.kv_heads, group, c.head_dim, f32, cus);
    AttnArgs a;
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.b = b;
    a.c = c;
    a.group = group;
    a.cap = (int)cap;
    a.window = window > (1 << 30) ? 0 : window;  // (the table reaches 2^30 positions at most)
    a.scale = scale * 1.44269504088896340736f;
    a.tiles = (int)p.tiles;
    a.splits = p.splits;
    a.min_chunk = p.min_chunk;
    a.most = p.most;
    a.o = static_cast<float*>(workspace);
    a.ml = reinterpret_cast<float2*>(a.o + p.parts * c.head_dim);
    int2* behind = reinterpret_cast<int2*>(a.ml + p.parts);
    a.info = p.join ? behind : nullptr;
    int2* items = p.items ? behind + (p.join ? (int64_t)b.tokens * group : 0) : nullptr;
    a.items = items;
    a.parts = p.parts;
    if (items) {
        hipLaunchKernelGGL(paged_items_kernel<32>, dim3(1), dim3(1024), 0, stream, a, items);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (c.head_dim == 64) return f32 ? launch_attention_hd<64, true>(p, a, stream) : launch_attention_hd<64, false>(p, a, stream);
    if (c.head_dim == 128)
        return f32 ? launch_attention_hd<128, true>(p, a, stream) : launch_attention_hd<128, false>(p, a, stream);
    return f32 ? launch_attention_hd<256, true>(p, a, stream) : launch_attention_hd<256, false>(p, a, stream);
}

}  // namespace rq
