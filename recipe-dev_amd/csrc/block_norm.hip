// The norms between two blocks, with the gate and the residual stream between
// them, of many rows (rqmv_block_norm).
//
//     d = delta / sqrt(mean(delta^2) + eps) * post     (the norm after a block)
//     u = x + scale * gate * d                         (the residual stream)
//     out = u / sqrt(mean(u^2) + eps) * pre            (the norm before the next)
// A row lies in the registers of T threads (V float4 each), so that it is read
// and written once, whatever of the three a call asks for; its two sums of squares are two joins
// over the T threads. Bound: HBM at prefill (4096 rows of 4,096 with one gate, fp16 out: 41.2 us, 5.7 TB/s); at a few rows the
// chain of loads, two joins and stores, for which T is 1024 (5 rows of 5,120: 5.6 us, 4.5 in a trace).
#include "block_norm.h"

#include <hip/hip_fp16.h>

namespace rq {

namespace {

// The sum over a row's T threads.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    if constexpr (T == 64) return v;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += part[w];
    return v;
}

__device__ __forceinline__ float squares(float4 v) { return v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w; }

// Rows pass by the caches: outputs always, x and delta where each is more than the L2s hold (4096 rows of 4,096 with one
// gate, fp16 out: 41.4 us, with outputs alone 42.2, without 52.1; with the reads of what comes next 57, 68 and 76; 1000
// rows with a gate each, outputs alone, 13.0, with all 14.6). Calls of 5 to 2,000 rows of 4,096 and a product over their
// fp16 rows take as long together as after plain stores; of 4096 rows 155.0 us and 153.2, of 4096 and the next norm 79.8
// and 75.4.
constexpr int64_t kCached = int64_t(32) << 20;
typedef float nt4_t __attribute__((ext_vector_type(4)));
typedef uint32_t nt2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float4 stream4(const float* p) {
    const nt4_t v = __builtin_nontemporal_load(reinterpret_cast<const nt4_t*>(p));
    return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void put(float* p, float4 v) {
    __builtin_nontemporal_store(nt4_t{v.x, v.y, v.z, v.w}, reinterpret_cast<nt4_t*>(p));
}
__device__ __forceinline__ void put(__half* p, float4 v) {
    const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    __builtin_nontemporal_store(nt2_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)},
                                reinterpret_cast<nt2_t*>(p));
}

template <int T, int V, typename O>
__global__ void __launch_bounds__(T < 256 ? 256 : T) block_norm_kernel(BlockNorm p) {
    __shared__ float part[2][16];
    const int64_t row = T < 256 ? (int64_t)blockIdx.x * (256 / T) + threadIdx.x / T : blockIdx.x;
    if (row >= p.rows) return;  // (T < 256 has no barriers)
    const int t = threadIdx.x % T, n4 = p.n / 4;
    const float inv_n = 1.f / (float)p.n;
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    auto at = [&](const float* base, int i) { return *reinterpret_cast<const float4*>(base + 4 * (t + i * T)); };
    float4 u[V], d[V];
    const float* x = p.x + row * p.ldx;
    const float* delta = p.delta + row * p.ldd;
    if (p.n * 4 * (int64_t)p.rows > kCached) {
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = t + i * T < n4 ? stream4(x + 4 * (t + i * T)) : zero;
        if (p.delta) {
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = t + i * T < n4 ? stream4(delta + 4 * (t + i * T)) : zero;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = t + i * T < n4 ? at(x, i) : zero;
        if (p.delta) {
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = t + i * T < n4 ? at(delta, i) : zero;
        }
    }
    if (p.delta) {
        float r = p.scale;
        if (p.post) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) ss += squares(d[i]);
            r = 1.f / sqrtf(row_sum<T>(ss, part[0]) * inv_n + p.eps);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (t + i * T >= n4) continue;
            float4 f = make_float4(r, r, r, r);
            if (p.post) {
                const float4 w = at(p.post, i);
                f = make_float4(r * w.x * p.scale, r * w.y * p.scale, r * w.z * p.scale, r * w.w * p.scale);
            }
            if (p.gate) {
                const float4 g = at(p.gate + row * p.ldg, i);
                f = make_float4(f.x * g.x, f.y * g.y, f.z * g.z, f.w * g.w);
            }
            u[i] = make_float4(fmaf(f.x, d[i].x, u[i].x), fmaf(f.y, d[i].y, u[i].y), fmaf(f.z, d[i].z, u[i].z),
                               fmaf(f.w, d[i].w, u[i].w));
        }
    }
    if (p.x_out) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (t + i * T < n4) put(p.x_out + row * p.ldxo + 4 * (t + i * T), u[i]);
    }
    if (!p.pre) return;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) ss += squares(u[i]);
    const float r = 1.f / sqrtf(row_sum<T>(ss, part[1]) * inv_n + p.eps);
    O* out = static_cast<O*>(p.out) + row * p.ldo;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (t + i * T >= n4) continue;
        const float4 w = at(p.pre, i);
        put(out + 4 * (t + i * T), make_float4(u[i].x * r * w.x, u[i].y * r * w.y, u[i].z * r * w.z, u[i].w * r * w.w));
    }
}

template <int T, int V>
void launch(const BlockNorm& p, bool out_f16, hipStream_t stream) {
    constexpr int THREADS = T < 256 ? 256 : T, ROWS = THREADS / T;
    const dim3 grid((p.rows + ROWS - 1) / ROWS), threads(THREADS);
    if (out_f16) hipLaunchKernelGGL((block_norm_kernel<T, V, __half>), grid, threads, 0, stream, p);
    else hipLaunchKernelGGL((block_norm_kernel<T, V, float>), grid, threads, 0, stream, p);
}

}  // namespace

hipError_t launch_block_norm(const BlockNorm& p, bool out_f16, int cus, hipStream_t stream) {
    // 1024 threads a row while all rows are resident at once, two a CU (500 rows of 4,096 6.3 us, of 256 threads 7.7; of
    // 8,192 10.0 and 12.4); past that 256, whose rows end and begin at different times (750 rows of 4,096 8.8 us, of 1024
    // threads 9.6; 4096 rows 40.7 and 45.6), from 4,097 values on, where these have fewer rows a CU, for more than
    // four (1100 of 5,120 13.8 and 16.0; 1000 of 8,192 equal).
    const int n4 = p.n / 4;
    if (n4 <= 64) launch<64, 1>(p, out_f16, stream);
    else if (n4 <= 256) launch<64, 4>(p, out_f16, stream);
    else if (p.rows > 2 * cus && n4 <= 1024) launch<256, 4>(p, out_f16, stream);
    else if (p.rows > 4 * cus && n4 <= 2048) launch<256, 8>(p, out_f16, stream);
    else if (n4 <= 1024) launch<1024, 1>(p, out_f16, stream);
    else if (n4 <= 2048) launch<1024, 2>(p, out_f16, stream);
    else if (n4 <= 4096) launch<1024, 4>(p, out_f16, stream);
    else launch<1024, 8>(p, out_f16, stream);
    return hipGetLastError();
}

}  // namespace rq
