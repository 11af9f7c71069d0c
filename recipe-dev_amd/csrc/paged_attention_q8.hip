// Attention over 8-bit pages (rqmv_paged_attention_q8): the mathematics, tiles,
// splits and joins of paged_attention.h, over codes and scales.
//
// Codes become the fp16 numbers that they stand for on their way to the matrix
// cores, which is exact (q8.h); from then on the arithmetic is that of fp16 pages.
#include "paged_attention.h"
#include "q8.h"

namespace rq {

namespace {

// How a wave takes 16 rows of codes: contiguous, 1024 bytes an instruction.
template <int HD>
struct Lay8 {
    static constexpr int PCS = HD / 16;   // 16-byte pieces per row
    static constexpr int RPI = 64 / PCS;  // rows per load instruction
    static constexpr int NI = HD / 64;    // instructions per 16 keys
};

// 16 keys of one page, on their way.
template <int HD>
struct Keys16 {
    uint4 x[Lay8<HD>::NI];
    unsigned scale;
};

template <int HD>
__device__ __forceinline__ void fetch16(const int8_t* codes, const uint8_t* scales, const PagedCache& c, int kh, int id,
                                        int key, Keys16<HD>& to) {
    const int64_t row = (((int64_t)id * c.kv_heads + kh) << c.block_shift) + (key & ((1 << c.block_shift) - 1));
    const uint4* from = reinterpret_cast<const uint4*>(codes + row * HD) + (threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < Lay8<HD>::NI; ++i) to.x[i] = from[i * 64];
    to.scale = scales[row >> 4];
}

// To 16 rows of fp16 in LDS.
template <int HD, bool VALUES>
__device__ __forceinline__ void put16(const Keys16<HD>& from, char* lds) {
    typedef Lay<HD> L;
    typedef Lay8<HD> L8;
    const int lane = threadIdx.x & 63, c = lane % L8::PCS;
    const Scale s = scale_of(__builtin_amdgcn_readfirstlane(from.scale));
#pragma unroll
    for (int i = 0; i < L8::NI; ++i) {
        const int r = i * L8::RPI + lane / L8::PCS, x = VALUES ? L::vx(r) : L::kx(r);
        const uint4 w = from.x[i];
        *reinterpret_cast<uint4*>(lds + r * L::ROW + ((2 * c) ^ x) * 16) = codes_to_h(make_uint2(w.x, w.y), s);
        *reinterpret_cast<uint4*>(lds + r * L::ROW + ((2 * c + 1) ^ x) * 16) = codes_to_h(make_uint2(w.z, w.w), s);
    }
}

// Four values of a row of the cache.
template <int HD>
struct Q8Values {
    const int8_t* v;
    const uint8_t* scale;
    __device__ __forceinline__ h4_t operator()(int64_t row, int dim) const {
        const uint32_t c = *reinterpret_cast<const uint32_t*>(v + row * HD + dim);
        const uint4 o = codes_to_h(make_uint2(c, 0), scale_of(scale[row >> 4]));
        const hv2_t a = __builtin_bit_cast(hv2_t, o.x), b = __builtin_bit_cast(hv2_t, o.y);
        return h4_t{a[0], a[1], b[0], b[1]};
    }
};

// ------------------------------------------- few rows: keys over the waves ----

// Four waves take every fourth step of 32 keys, without barriers. A step's keys go from the pages into registers,
// where they become operands of the first product without a detour: a lane takes half of a row's dims (h HD / 2 ..,
// and the queries' operands hold theirs in that order). The values go straight to LDS as codes, two
// buffers a wave, and are read transposed (ds_read_b64_tr_b8); the next step's keys and values are asked for
// once the scores are done. Codes lie in LDS as rows of HD bytes, 16-byte pieces XORed so that a read of
// two pieces of sixteen rows hits every bank alike. (Keys through LDS, as over fp16 pages, 101.9 us for the first size
// below, so 86.4; then a tile's last item behind all longer ones 77.5.)
// Bound: HBM (32/8 heads of 128, fp16, with the join: 48 requests of 100 to 12,000 positions 77 us, 4.4 TB/s, over fp16
// pages 142; 200 of 1,000 to 3,000 148, 5.1 TB/s); for one sequence the chain lengths -> table -> keys and the
// join (one token over 8,000, fp32: 12.8 us, of which 10.8 and 3.8 in a trace).
template <int HD>
__device__ constexpr int code_xor(int row) {
    return HD == 64 ? ((row >> 2) & 1) << 1 : HD == 128 ? ((row >> 1) & 3) << 1 : (row & 7) << 1;
}

// A lane's half of row lane % 32 of a step of 32 keys, and the row's scale byte.
template <int HD>
struct KeyHalf {
    uint4 x[HD / 32];
    unsigned scale;
};
template <int HD>
__device__ __forceinline__ void fetch_keys(const PagedCodes& codes, const PagedCache& c, int kh, const int (&ids)[2], int key0,
                                           KeyHalf<HD>& to) {
    const int lane = threadIdx.x & 63, r = lane & 31;
    const int id = r < 16 ? ids[0] : ids[1];
    const int64_t row = (((int64_t)id * c.kv_heads + kh) << c.block_shift) + ((key0 + r) & ((1 << c.block_shift) - 1));
    const uint4* from = reinterpret_cast<const uint4*>(codes.k + row * HD + (lane >> 5) * (HD / 2));
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) to.x[i] = from[i];
    to.scale = codes.k_scale[row >> 4];
}

// S^T of 32 keys, as scores() of paged_attention.h leaves it, but for their scales' `more`.
template <int HD, bool F32>
__device__ __forceinline__ void scores_of_codes(const KeyHalf<HD>& keys, const Scale& scale, const Rows<HD, 1, F32>& w,
                                                f16_t& s) {
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
        const uint4 x = keys.x[k / 2];
        const h8_t key = __builtin_bit_cast(h8_t, codes_to_low(k % 2 ? make_uint2(x.z, x.w) : make_uint2(x.x, x.y), scale));
#pragma unroll
        for (int p = 0; p < Rows<HD, 1, F32>::QP; ++p) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(key, w.q[0][k][p], s, 0, 0, 0);
    }
}

// O^T += V^T P^T over a step's 32 keys, whose scale bytes are v_scale. (A scale above 2^5 is 2^5, as often as it takes.)
template <int HD, bool F32>
__device__ __forceinline__ void add_codes(const char* V, const unsigned (&v_scale)[2], Rows<HD, 1, F32>& w,
                                          const h8_t (&p)[2][F32 ? 2 : 1]) {
    typedef int i2_t __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i2_t lds2;
    const int lane = threadIdx.x & 63, h = lane >> 5;
    // 16 lanes read 16 dims of eight keys, two lanes a key: 4 h .. 4 h + 3 and 8 + 4 h ..
    const int i = (lane & 15) >> 1, r = (i < 4 ? 0 : 4) + 4 * h + i;
    const char* at = V + r * HD + (lane & 1) * 8;
    i2_t x[2][HD / 32];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
            x[b][d] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (lds2*)(at + 16 * b * HD + ((2 * d + ((lane >> 4) & 1)) ^ code_xor<HD>(r)) * 16));
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const Scale scale = scale_of(v_scale[b]);
        int again = 1 << scale.more;
        do {
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {
                const h8_t v = __builtin_bit_cast(h8_t, codes_to_low(make_uint2(x[b][d][0], x[b][d][1]), scale));
#pragma unroll
                for (int part = 0; part < (F32 ? 2 : 1); ++part)
                    w.o[0][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[b][part], w.o[0][d], 0, 0, 0);
            }
        } while (--again);
    }
}

constexpr int q8_few_lds(int hd) { return 4 * 2 * 32 * hd; }
constexpr int q8_few_wgs(int hd, bool f32) { return hd == 256 ? 1 : 2; }

template <int HD, bool F32>
__global__ void __launch_bounds__(256, q8_few_wgs(HD, F32)) paged_q8_few(AttnArgs a, PagedCodes codes) {
    constexpr int TM = 32, KEYS = 32, STEP = KEYS * HD;  // STEP: bytes of a step's values
    extern __shared__ __align__(16) char lds[];
    const int kh = blockIdx.x % a.c.kv_heads;
    Item item;
    if (!find_item<TM, true>(a, blockIdx.x / a.c.kv_heads, &item)) return;
    // (starts out of order may count past what the workspace holds)
    const bool whole = item.live <= 1;
    const int64_t part0 = ((int64_t)item.part * a.c.kv_heads + kh) * TM;
    if (!whole && (a.most ? item.split >= a.most : part0 < 0 || part0 + TM > a.parts)) return;
    const int seq = item.seq;
    const Tile t = make_tile<TM>(a, seq, item.of, item.tile * TM);
    const int begin = item.first + item.split * item.chunk, end = min(begin + item.chunk, t.end);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char* V = lds + wave * 2 * STEP;
    const uint32_t v_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)V;
    Pages pages{a.b.table + seq * a.b.table_stride, a.b.max_blocks - 1, a.c.blocks, a.c.block_shift, INT_MIN / 2, 0};
    Rows<HD, 1, F32> w;

    KeyHalf<HD> keys;
    unsigned v_scale[2], v_next[2];
    unsigned bad = 0, bad_next = 0;  // which 16 keys of the step are in no page
    int buffer = 0;
    auto fetch = [&](int key0, int to) {
        const int p0 = key0 >> pages.shift, p1 = (key0 + 16) >> pages.shift;
        pages.need(p0, p1);
        int ids[2] = {pages.at(p0), pages.at(p1)};
        bad_next = (pages.absent(ids[0]) ? 1 : 0) | (pages.absent(ids[1]) ? 2 : 0);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (pages.absent(ids[g])) ids[g] = 0;
            const int key = key0 + 16 * g;
            const int64_t row = (((int64_t)ids[g] * a.c.kv_heads + kh) << a.c.block_shift) + (key & ((1 << a.c.block_shift) - 1));
            v_next[g] = codes.v_scale[row >> 4];
#pragma unroll
            for (int i = 0; i < Lay8<HD>::NI; ++i) {
                const int r = i * Lay8<HD>::RPI + lane / Lay8<HD>::PCS;
                const int piece = (lane % Lay8<HD>::PCS) ^ code_xor<HD>(r);
                load_lds(codes.v + row * HD, (uint32_t)(r * HD + piece * 16), v_lds + to * STEP + g * 16 * HD + i * 1024);
            }
        }
        fetch_keys<HD>(codes, a.c, kh, ids, key0, keys);
    };
    int key0 = begin + wave * KEYS;
    bool odd = false;
    if (key0 < end) pages.fetch(key0 >> pages.shift);
    RawRows<HD, F32> raw;
    load_rows<HD, F32, true>(a, t, kh, t.row0, w, raw);
    arrived(w, raw);
    if (key0 < end) fetch(key0, 0);
    start_rows(a, w, raw);
    while (key0 < end) {
        const int after = key0 + 4 * KEYS;
        bad = bad_next;
        wait_loads<0>();
        const Scale scale = scale_of(keys.scale);
#pragma unroll
        for (int g = 0; g < 2; ++g) v_scale[g] = __builtin_amdgcn_readfirstlane(v_next[g]);
        f16_t s[1][1];
        scores_of_codes<HD, F32>(keys, scale, w, s[0][0]);
        if (__any(scale.more)) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const float by = (float)(1 << __builtin_amdgcn_readlane(scale.more, 16 * g));
#pragma unroll
                for (int e = 0; e < 8; ++e) s[0][0][8 * g + e] *= by;
            }
        }
        if (after < end) {
            // (the reads of the other buffer have returned: their products are behind)
            asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(s[0][0]) : : "memory");
            fetch(after, buffer ^ 1);
        }
        const bool masked = key0 < t.all_from || key0 + KEYS > t.all_to || bad;
        if (masked) mask_scores<HD, 1, 1, F32>(w, s, key0, bad);
        float top[1];
        largest<1, 1>(s, top);
        move_references<HD, 1, F32>(w, top);
        h8_t p[1][2][F32 ? 2 : 1];
        weights<HD, 1, 1, F32>(w, s, p);
        if (masked) {
            // A NaN scale must not meet a weight of 0: groups that no row sees count as 0, and NaN groups too, which come
            // to the rows that see them at the end (add_odd).
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const bool dead = ((bad >> b) & 1) || key0 + 16 * b >= t.end, nan = v_scale[b] == kScaleNan;
                odd |= nan && !dead;
                if (dead || nan) v_scale[b] = 0;
            }
        }
        add_codes<HD, F32>(V + buffer * STEP, v_scale, w, p[0]);
        buffer ^= 1;
        key0 = after;
    }
    if (odd) {  // (the wave's own steps; what unmasked ones let through is there already, and stays)
        for (int k0 = begin + wave * KEYS; k0 < end; k0 += 4 * KEYS)
            add_odd<HD, 1, F32>(a, t, kh, k0, min(k0 + KEYS, t.end), w, Q8Values<HD>{codes.v, codes.v_scale});
    }
    finish_few<HD, F32, KEYS, 2>(a, t, item, kh, begin, end, part0, w, lds);
}

// --------------------------------------------- many rows: rows over the waves ----

// The waves share steps of 64 keys in two LDS buffers, one barrier a step. Codes go from the pages into registers, 16
// keys of one page at a time (one scale), and from there, a step later, to LDS as fp16. Bound: matrix cores and VALU in
// turn (2000 tokens over 12,000, 32/8 heads of 128, fp16: 456 us, 935 TFLOP/s; over fp16 pages 432, as there is no
// conversion).
template <int HD, bool F32>
__global__ void __launch_bounds__(64 * many_waves(HD), many_waves(HD) / 4) paged_q8_many(AttnArgs a, PagedCodes codes) {
    typedef Lay<HD> L;
    constexpr int WAVES = many_waves(HD), TM = 32 * WAVES, KEYS = 64, KT = KEYS / 32;
    constexpr int HALF = KEYS * HD * 2;
    constexpr bool BOTH = WAVES == 4;  // each wave loads keys and values; of eight, four load each
    extern __shared__ __align__(16) char lds[];
    // the last tiles first: of one sequence's they have the most keys
    const int kh = blockIdx.x % a.c.kv_heads, number = a.tiles - 1 - blockIdx.x / a.c.kv_heads, split = blockIdx.y;
    const int seq = find_seq<TM>(a.b, a.group, number);
    const int first = start_of(a.b, seq) * a.group / TM + seq;
    const Tile t = make_tile<TM>(a, seq, load_seq(a, seq), (number - first) * TM);
    if (t.row0 < 0 || t.row0 >= t.rows) return;  // (below 0: starts out of order)
    const int begin = t.first + split * t.chunk, end = min(begin + t.chunk, t.end);
    if (split && begin >= end) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = t.row0 + 32 * wave;
    Pages pages{a.b.table + seq * a.b.table_stride, a.b.max_blocks - 1, a.c.blocks, a.c.block_shift, INT_MIN / 2, 0};
    Rows<HD, 1, F32> w;

    const int g = wave % (KEYS / 16);
    Keys16<HD> one, two;  // BOTH: keys, values; else what the wave loads
    // Asks for the wave's part of a step; returns which groups are absent.
    auto fetch = [&](int key0) -> unsigned {
        pages.need(key0 >> pages.shift, (key0 + KEYS - 16) >> pages.shift);
        unsigned bad = 0;
#pragma unroll
        for (int i = 0; i < KEYS / 16; ++i) bad |= pages.absent(pages.at((key0 + 16 * i) >> pages.shift)) ? 1u << i : 0u;
        const int key = key0 + 16 * g, id = pages.at(key >> pages.shift);
        const int page = pages.absent(id) ? 0 : id;
        const bool keys = BOTH || wave < 4;
        fetch16<HD>(keys ? codes.k : codes.v, keys ? codes.k_scale : codes.v_scale, a.c, kh, page, key, one);
        if (BOTH) fetch16<HD>(codes.v, codes.v_scale, a.c, kh, page, key, two);
        return bad;
    };
    auto put = [&](int buffer) {
        char* at = lds + buffer * 2 * HALF + g * 16 * L::ROW;
        if (BOTH || wave < 4) put16<HD, false>(one, at);
        if (BOTH) put16<HD, true>(two, at + HALF);
        else if (wave >= 4) put16<HD, true>(one, at + HALF);
    };
    // the keys that any of the wave's rows sees
    const int p0 = t.kv - t.n + row / a.group, p1 = t.kv - t.n + (min(row + 32, t.rows) - 1) / a.group;
    const int wave_to = row < t.rows ? p1 + 1 : 0, wave_from = a.window ? p0 - a.window + 1 : 0;
    unsigned bad = 0, bad1 = 0, bad2 = 0;
    int buffer = 0;
    bool odd = false;
    if (begin < end) pages.fetch(begin >> pages.shift);
    RawRows<HD, F32> raw;
    load_rows<HD, F32>(a, t, kh, row, w, raw);
    arrived(w, raw);
    if (begin < end) bad = fetch(begin);
    start_rows(a, w, raw);
    if (begin < end) {
        put(0);
        if (begin + KEYS < end) bad1 = fetch(begin + KEYS);
    }
    // The next step to the other buffer, and those behind it asked for: at a step's beginning at 128 dims (2000 tokens over
    // 12,000, fp16: 461 us, at its end 468), at its end at 64 and 256 (over 4,000: 145 and 566 us, 147 and 599).
    constexpr bool FIRST = HD == 128;
    auto go_on = [&](int key0) {
        if (key0 + KEYS < end) put(buffer ^ 1);
        if (key0 + 2 * KEYS < end) bad2 = fetch(key0 + 2 * KEYS);
    };
    for (int key0 = begin; key0 < end; key0 += KEYS) {
        __syncthreads();  // the step is in LDS, and the other buffer is free
        if (FIRST) go_on(key0);
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
        if (!FIRST) go_on(key0);
        bad = bad1;
        bad1 = bad2;
        buffer ^= 1;
    }
    if (odd) add_odd<HD, 1, F32>(a, t, kh, begin, end, w, Q8Values<HD>{codes.v, codes.v_scale});
    finish_many<HD, F32>(a, t, kh, split, begin, end, row, w);
}

template <int HD, bool F32>
hipError_t launch_hd(const AttnPlan& p, const AttnArgs& a, const PagedCodes& codes, hipStream_t stream) {
    const void* f = p.few ? reinterpret_cast<const void*>(paged_q8_few<HD, F32>)
                          : reinterpret_cast<const void*>(paged_q8_many<HD, F32>);
    const int lds = p.few ? q8_few_lds(HD) : many_lds(HD);
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    if (p.few) hipLaunchKernelGGL((paged_q8_few<HD, F32>), attention_grid(p, a), dim3(256), lds, stream, a, codes);
    else hipLaunchKernelGGL((paged_q8_many<HD, F32>), attention_grid(p, a), dim3(64 * many_waves(HD)), lds, stream, a, codes);
    return hipGetLastError();
}

// Tiles of 32 rows over all heads up to which few rows are assumed: 4 a CU, of fp16 rows of 128 dims 2. Over 380 batches
// of 1 to 32 sequences, 16 to 1024 new tokens and 0 to 6,000 cached ones, of seven combinations of heads and type, the
// choice takes 2 to 5 % more than the better form on average (32/8 heads of 128, fp16, few against many, us: 32
// sequences of 16 tokens over 6,000 115 / 148, of 64 370 / 390; 4 of 512 356 / 224). At 4 a CU the fewest rows that take
// the form for many have tiles for more than half of the CUs, so it splits keys at fp16 rows of 128 dims alone.
AttnPlan plan_q8(const PagedBatch& b, const PagedCache& c, int q_heads, bool f32, int cus) {
    return plan_attention(b.tokens, b.seqs, (int64_t)b.max_blocks << c.block_shift, c.kv_heads, q_heads / c.kv_heads,
                          c.head_dim, f32, cus, (c.head_dim == 128 && !f32 ? 2 : 4) * cus);
}

}  // namespace

size_t paged_attention_q8_workspace(const PagedBatch& b, const PagedCache& c, int q_heads, int cus) {
    size_t most = 0;
    for (const bool f32 : {false, true}) {  // (one workspace serves both types)
        const size_t bytes = attention_workspace_bytes(plan_q8(b, c, q_heads, f32, cus), b.tokens, b.seqs,
                                                       q_heads / c.kv_heads, c.head_dim);
        most = bytes > most ? bytes : most;
    }
    return most;
}

hipError_t launch_paged_attention_q8(const PagedBatch& b, const PagedCache& c, const PagedCodes& codes, const void* q, bool f32,
                                     int64_t ldq, int q_heads, float scale, int window, void* workspace, void* out,
                                     int64_t ldo, int cus, hipStream_t stream) {
    const AttnPlan p = plan_q8(b, c, q_heads, f32, cus);
    AttnArgs a;
    hipError_t e = attention_args(p, b, c, q, ldq, q_heads, scale, window, workspace, out, ldo, stream, &a);
    if (e != hipSuccess) return e;
    if (c.head_dim == 64) e = f32 ? launch_hd<64, true>(p, a, codes, stream) : launch_hd<64, false>(p, a, codes, stream);
    else if (c.head_dim == 128)
        e = f32 ? launch_hd<128, true>(p, a, codes, stream) : launch_hd<128, false>(p, a, codes, stream);
    else e = f32 ? launch_hd<256, true>(p, a, codes, stream) : launch_hd<256, false>(p, a, codes, stream);
    return e == hipSuccess ? launch_attention_join(p, a, f32, stream) : e;
}

}  // namespace rq
