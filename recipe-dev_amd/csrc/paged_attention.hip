// Attention of several sequences' new tokens over fp16 pages
// (rqmv_paged_attention); the mathematics and what 8-bit pages share is in
// paged_attention.h.
//
// Keys and values go from the pages straight into LDS (global_load_lds, 16
// bytes a lane).
#include "paged_attention.h"

namespace rq {

namespace {

constexpr int64_t kEarlyBytes = int64_t(1) << 20;  // of parts that a join may ask for unseen

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

// Four values of a row of the cache.
template <int HD>
struct F16Values {
    const __half* v;
    __device__ __forceinline__ h4_t operator()(int64_t row, int dim) const {
        return *reinterpret_cast<const h4_t*>(reinterpret_cast<const _Float16*>(v) + row * HD + dim);
    }
};

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

template <int HD, bool F32>
__global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) paged_few_kernel(AttnArgs a) {
    typedef Lay<HD> L;
    constexpr int TM = 32, KEYS = 32, HALF = KEYS * HD * 2;  // HALF: bytes of a wave's K (and V) buffer
    extern __shared__ __align__(16) char lds[];
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
            add_odd<HD, 1, F32>(a, t, kh, k, min(k + KEYS, t.end), w, F16Values<HD>{a.c.v});
    }
    finish_few<HD, F32, KEYS>(a, t, item, kh, begin, end, part0, w, lds);
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
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
    if (odd) add_odd<HD, 1, F32>(a, t, kh, begin, end, w, F16Values<HD>{a.c.v});
    finish_many<HD, F32>(a, t, kh, split, begin, end, row, w);
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

template <int HD, bool F32>
hipError_t join_hd(const AttnPlan& p, const AttnArgs& a, hipStream_t stream) {
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

template <int HD, bool F32>
hipError_t launch_attention_hd(const AttnPlan& p, const AttnArgs& a, hipStream_t stream) {
    const void* f = p.few ? reinterpret_cast<const void*>(paged_few_kernel<HD, F32>)
                          : reinterpret_cast<const void*>(paged_many_kernel<HD, F32>);
    const int lds = p.few ? few_lds(HD) : many_lds(HD);
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    if (p.few) hipLaunchKernelGGL((paged_few_kernel<HD, F32>), attention_grid(p, a), dim3(256), lds, stream, a);
    else hipLaunchKernelGGL((paged_many_kernel<HD, F32>), attention_grid(p, a), dim3(64 * many_waves(HD)), lds, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.join) return e;
    return join_hd<HD, F32>(p, a, stream);
}

// Tiles of 32 rows over all heads up to which few rows are assumed: 4 a CU (64 and 256 dims, fp16),
// 2 (128 dims; 64, fp32) or a half (256, fp32, whose large tiles have 128 rows). Over 222
// batches of 1 to 16 sequences, 64 to 1024 new tokens and 0 to 6,000 cached ones the choice takes 0.5 to
// 4.5 % more than the better form; at 256 dims of fp16 11 % over 131 batches. Few against many, 32/8 heads of 128,
// fp16, us: 32 sequences of 128 rows over 6,000 positions 238 / 341, of 256 398 / 350; one of 1024 rows over 1,000
// 23 / 27; four of 2048 over 6,000 350 / 221.
int64_t few_tiles(int hd, bool f32, int cus) {
    return hd == 128 ? 2 * cus : hd == 64 ? (f32 ? 2 : 4) * cus : f32 ? cus / 2 : 4 * cus;
}

}  // namespace

AttnPlan plan_attention(int tokens, int seqs, int64_t cap, int kv_heads, int group, int hd, bool f32, int cus,
                        int64_t few_tiles) {
    AttnPlan p;
    const int heads = kv_heads * group;
    // The few-rows form up to 128 rows a sequence and kv head on average, or where there are so few that
    // the large tiles leave CUs idle. One form takes the whole batch: 100 decoding requests over 2,000 beside
    // 2048 tokens over 6,000 take 494 us (few, fp16 pages, 32/8 heads of 128), as two batches 157 + 255; 32 beside them 298
    // (many), 53 + 255.
    p.tiles = (int64_t)tokens * group / 32 + seqs;
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

size_t attention_workspace_bytes(const AttnPlan& p, int tokens, int seqs, int group, int hd) {
    return (p.join ? p.parts * (hd * sizeof(float) + sizeof(float2)) + (size_t)tokens * group * sizeof(int2) : 0) +
           (p.items ? ((size_t)seqs + 1) * sizeof(int2) : 0);
}

hipError_t launch_attention_join(const AttnPlan& p, const AttnArgs& a, bool f32, hipStream_t stream) {
    if (!p.join) return hipSuccess;
    if (a.c.head_dim == 64) return f32 ? join_hd<64, true>(p, a, stream) : join_hd<64, false>(p, a, stream);
    if (a.c.head_dim == 128) return f32 ? join_hd<128, true>(p, a, stream) : join_hd<128, false>(p, a, stream);
    return f32 ? join_hd<256, true>(p, a, stream) : join_hd<256, false>(p, a, stream);
}

bool paged_attention_fits(const PagedBatch& b, const PagedCache& c, int q_heads) {
    return ((int64_t)b.tokens * (q_heads / c.kv_heads) / 32 + b.seqs) * c.kv_heads <= (1 << 23) &&
           (int64_t)b.tokens * q_heads <= (1 << 26);
}

size_t paged_attention_workspace(const PagedBatch& b, const PagedCache& c, int q_heads, int cus) {
    const int group = q_heads / c.kv_heads;
    const int64_t cap = (int64_t)b.max_blocks << c.block_shift;
    size_t most = 0;
    for (const bool f32 : {false, true}) {  // (one workspace serves both types)
        const AttnPlan p = plan_attention(b.tokens, b.seqs, cap, c.kv_heads, group, c.head_dim, f32, cus,
                                          few_tiles(c.head_dim, f32, cus));
        const size_t bytes = attention_workspace_bytes(p, b.tokens, b.seqs, group, c.head_dim);
        most = bytes > most ? bytes : most;
    }
    return most;
}

hipError_t attention_args(const AttnPlan& p, const PagedBatch& b, const PagedCache& c, const void* q, int64_t ldq, int q_heads,
                          float scale, int window, void* workspace, void* out, int64_t ldo, hipStream_t stream,
                          AttnArgs* args) {
    const int group = q_heads / c.kv_heads;
    AttnArgs& a = *args;
    a.q = q;
    a.out = out;
    a.ldq = ldq;
    a.ldo = ldo;
    a.b = b;
    a.c = c;
    a.group = group;
    a.cap = (int)((int64_t)b.max_blocks << c.block_shift);
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
    return hipSuccess;
}

hipError_t launch_paged_attention(const PagedBatch& b, const PagedCache& c, const void* q, bool f32, int64_t ldq,
                                  int q_heads, float scale, int window, void* workspace, void* out, int64_t ldo, int cus,
                                  hipStream_t stream) {
    const AttnPlan p = plan_attention(b.tokens, b.seqs, (int64_t)b.max_blocks << c.block_shift, c.kv_heads,
                                      q_heads / c.kv_heads, c.head_dim, f32, cus, few_tiles(c.head_dim, f32, cus));
    AttnArgs a;
    const hipError_t e = attention_args(p, b, c, q, ldq, q_heads, scale, window, workspace, out, ldo, stream, &a);
    if (e != hipSuccess) return e;
    if (c.head_dim == 64) return f32 ? launch_attention_hd<64, true>(p, a, stream) : launch_attention_hd<64, false>(p, a, stream);
    if (c.head_dim == 128)
        return f32 ? launch_attention_hd<128, true>(p, a, stream) : launch_attention_hd<128, false>(p, a, stream);
    return f32 ? launch_attention_hd<256, true>(p, a, stream) : launch_attention_hd<256, false>(p, a, stream);
}

}  // namespace rq

