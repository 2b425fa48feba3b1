// Append to a paged KV cache with the keys' rotation on the way
// (SLC_OP_EXT_PAGED_APPEND).
//
// Row t of sequence b (starts[b] <= t < starts[b + 1]) sits at position
// pos = past[b] + t - starts[b], in page table[b][pos / page] at offset
// pos % page of the state [pages, layers, 2, page, kv_heads, head_dim]:
//   key[2p], key[2p+1] (GPT-J) or key[p], key[p + D/2] (NeoX) are turned by
//   pos / theta^(2p / D) and written to parity 0, the value to parity 1.
// The arithmetic is rope_kernel's: f64 angle from the host-computed f64
// denominators, f64 sine and cosine rounded to f32, two IEEE products and one
// sum per output, so an F32 cache receives bit for bit what Rope followed by
// KvAppend stores; an F16 / BF16 cache receives those values rounded to
// nearest.
//
// HBM-bound: 8 * T * Hkv * D bytes in, 2 * T * Hkv * D * size out. A CTA takes
// kTokens tokens at a time: its threads first evaluate the tokens' sines and
// cosines (each once for all heads), then move 4 pairs of keys and 8 values
// per item with 128-bit accesses. Measured: prompts of 11598 tokens, 8 kv heads
// of 128 in f32 (190 MB) 33.5 us, 5.7 TB/s; one token 2.4 us in a graph, 5.3 us
// as a call (the host's part).
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "tma.cuh"

namespace slc {
namespace k {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = kPagedMaxHeadDim / 2;

struct AppendArgs {
    const float *k, *v;
    PagedCache cache;
    PagedBatch batch;
    int kv_heads, head_dim, tokens;
    int rotate, gptj;
    uint32_t *err;
    double denom[kMaxHalf];  // theta^(2 p / D), host libm pow
};

// Four floats at a 4-byte aligned address (`vec`: 16-byte aligned).
__device__ __forceinline__ void load4(const float *p, int vec, float (&x)[4]) {
    if (vec) {
        const float4 a = ld_stream_f4(p);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = p[i];
    }
}

template <typename T>
__device__ __forceinline__ void store4(T *p, const float (&x)[4]);
template <>
__device__ __forceinline__ void store4<float>(float *p, const float (&x)[4]) {
    *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
template <>
__device__ __forceinline__ void store4<__half>(__half *p, const float (&x)[4]) {
    const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a),
                                               *reinterpret_cast<const uint32_t *>(&b));
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16 *p, const float (&x)[4]) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a),
                                               *reinterpret_cast<const uint32_t *>(&b));
}

// kTokens: tokens per CTA pass. head_dim is a multiple of 8, so a head's half
// is a multiple of 4 and every store below is 8- or 16-byte aligned.
template <typename T, int kTokens>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const __grid_constant__ AppendArgs p) {
    pdl_trigger();
    extern __shared__ float trig[];  // [kTokens][half] sines, then cosines
    __shared__ long long dst_s[kTokens];  // byte offset of the token's keys, -1: none
    __shared__ uint32_t pos_s[kTokens];
    const int half = p.head_dim / 2, Hkv = p.kv_heads;
    float *cos_s = trig + kTokens * half;
    const int total = (int)p.batch.starts[p.batch.seqs];
    const int vec = aligned16(p.k) && aligned16(p.v);
    bool waited = false;
    for (int t0 = blockIdx.x * kTokens; t0 < p.tokens && t0 < total; t0 += gridDim.x * kTokens) {
        if (threadIdx.x < kTokens) {
            const int t = t0 + threadIdx.x;
            long long dst = -1;
            uint32_t pos = 0;
            if (t < p.tokens && t < total) {
                const int b = paged_sequence_of(p.batch, (uint32_t)t);
                pos = p.batch.past[b] + (uint32_t)t - p.batch.starts[b];
                dst = paged_row(p.cache, p.batch, b, (int)pos, p.err);
            }
            dst_s[threadIdx.x] = dst;
            pos_s[threadIdx.x] = pos;
        }
        __syncthreads();
        if (p.rotate)
            for (int i = threadIdx.x; i < kTokens * half; i += kThreads) {
                const int j = i / half, pr = i - j * half;
                if (dst_s[j] < 0) continue;
                double sn, cs;
                sincos((double)pos_s[j] / p.denom[pr], &sn, &cs);
                trig[i] = (float)sn;
                cos_s[i] = (float)cs;
            }
        if (!waited) pdl_wait();  // the tables above are written by uploads alone
        waited = true;
        __syncthreads();
        const int quads = half / 4, work = kTokens * Hkv * quads;
        for (int i = threadIdx.x; i < work; i += kThreads) {
            const int c = i % quads, th = i / quads, h = th % Hkv, j = th / Hkv;
            if (dst_s[j] < 0) continue;
            const size_t src = ((size_t)(t0 + j) * Hkv + h) * p.head_dim;
            T *kd = reinterpret_cast<T *>(p.cache.base + dst_s[j]) + (size_t)h * p.head_dim;
            T *vd = reinterpret_cast<T *>(p.cache.base + dst_s[j] + p.cache.parity_stride) +
                    (size_t)h * p.head_dim;
            // NeoX: dims 4c .. 4c+3 and the same past the half; GPT-J: 8c .. 8c+7.
            const int d0 = p.gptj ? 8 * c : 4 * c, d1 = p.gptj ? 8 * c + 4 : 4 * c + half;
            float a[4], b[4], x[4], y[4];
            load4(p.k + src + d0, vec, a);
            load4(p.k + src + d1, vec, b);
            load4(p.v + src + d0, vec, x);
            load4(p.v + src + d1, vec, y);
            if (p.rotate) {
                const float *sn = trig + j * half + 4 * c, *cs = cos_s + j * half + 4 * c;
                float o0[4], o1[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float f = p.gptj ? (e < 2 ? a[2 * e] : b[2 * e - 4]) : a[e];
                    const float g = p.gptj ? (e < 2 ? a[2 * e + 1] : b[2 * e - 3]) : b[e];
                    const float r0 = __fsub_rn(__fmul_rn(f, cs[e]), __fmul_rn(g, sn[e]));
                    const float r1 = __fadd_rn(__fmul_rn(f, sn[e]), __fmul_rn(g, cs[e]));
                    if (p.gptj) {
                        (e < 2 ? o0[2 * e] : o1[2 * e - 4]) = r0;
                        (e < 2 ? o0[2 * e + 1] : o1[2 * e - 3]) = r1;
                    } else {
                        o0[e] = r0;
                        o1[e] = r1;
                    }
                }
                store4<T>(kd + d0, o0);
                store4<T>(kd + d1, o1);
            } else {
                store4<T>(kd + d0, a);
                store4<T>(kd + d1, b);
            }
            store4<T>(vd + d0, x);
            store4<T>(vd + d1, y);
        }
        __syncthreads();
    }
    if (!waited) pdl_wait();
}

template <typename T, int kTokens>
void launch(cudaStream_t s, const AppendArgs &a) {
    const int grid = grid_for((size_t)a.tokens, kTokens);
    launch_k(paged_append_kernel<T, kTokens>, grid, kThreads,
             (size_t)kTokens * a.head_dim * sizeof(float), s, a);
}

template <typename T>
void launch_for(cudaStream_t s, const AppendArgs &a) {
    // One token per CTA while that leaves SMs free, four beyond.
    if (a.tokens <= 4 * kSmCount)
        launch<T, 1>(s, a);
    else
        launch<T, 4>(s, a);
}

}  // namespace

cudaError_t paged_append(cudaStream_t s, const float *k, const float *v, const PagedCache &cache,
                         const PagedBatch &batch, size_t kv_heads, size_t head_dim, size_t tokens,
                         float theta, int gptj, uint32_t *err) {
    if (tokens == 0 || batch.seqs == 0 || kv_heads == 0) return cudaSuccess;
    AppendArgs a{};
    a.k = k;
    a.v = v;
    a.cache = cache;
    a.batch = batch;
    a.kv_heads = (int)kv_heads;
    a.head_dim = (int)head_dim;
    a.tokens = (int)tokens;
    a.rotate = theta != 0.f;
    a.gptj = gptj;
    a.err = err;
    if (a.rotate)
        for (size_t p = 0; p < head_dim / 2; p++)
            a.denom[p] = pow((double)theta, 2.0 * (double)p / (double)head_dim);
    switch (cache.type) {
    case kPagedF16: launch_for<__half>(s, a); break;
    case kPagedBf16: launch_for<__nv_bfloat16>(s, a); break;
    default: launch_for<float>(s, a); break;
    }
    count_launch();
    return cudaGetLastError();
}

}  // namespace k
}  // namespace slc
