// Paged KV cache: addressing shared by the append and attention kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "tensormap.h"
#include "tma.cuh"

namespace slc {
namespace k {

// pos / page by a multiplication (set_page below).
__device__ __forceinline__ int page_of(const PagedCache &c, int pos) {
    return (int)((__umulhi((uint32_t)pos, c.page_mul) + (uint32_t)pos) >> c.page_shift);
}

// Byte offset (from cache.base) of the key row of position `pos` of sequence
// `b`, head 0. The host has checked every page id that a position in use
// names; the guard keeps a wrong one from leaving the cache (page 0 then
// stands in, and the device error word is set).
__device__ __forceinline__ long long paged_row(const PagedCache &c, const PagedBatch &batch, int b,
                                               int pos, uint32_t *err) {
    const int pg = page_of(c, pos), off = pos - pg * c.page;
    uint32_t id = 0;
    if (pg < batch.per_seq) id = batch.table[(long long)b * batch.per_seq + pg];
    if (pg >= batch.per_seq || id >= (uint32_t)c.pages) {
        report_error(err, kErrGatherId);
        id = 0;
    }
    return (long long)id * c.page_stride + (long long)off * c.row_stride;
}

// The sequence that row t belongs to: the largest b with starts[b] <= t
// (starts is nondecreasing, starts[seqs] > t).
__device__ __forceinline__ int paged_sequence_of(const PagedBatch &batch, uint32_t t) {
    int lo = 0, hi = batch.seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (batch.starts[mid] <= t)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

// The cache's layer as a tensor map [pages][2][page][kv_heads][head_dim] with
// boxes of 128 bytes by `unit` keys: the largest power of two, at least 8 (the
// rows of a swizzle) and at most `most`, that divides the page, so that boxes
// stack to any tile. Returns unit, or 1 where there is none.
inline int paged_boxes(const PagedAttention &a, int most, size_t size, bool f16, bool swizzle, CUtensorMap *map) {
    const PagedCache &c = a.cache;
    int unit = most;
    while (unit >= 8 && c.page % unit) unit /= 2;
    if (unit < 8) return 1;
    const uint64_t dims[5] = {(uint64_t)a.head_dim, (uint64_t)a.kv_heads, (uint64_t)c.page, 2, (uint64_t)c.pages};
    const uint64_t strides[4] = {(uint64_t)a.head_dim * size, (uint64_t)c.row_stride, (uint64_t)c.parity_stride,
                                 (uint64_t)c.page_stride};
    const uint32_t box[5] = {128 / (uint32_t)size, 1, (uint32_t)unit, 1, 1};
    const CUtensorMapDataType type = size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : f16     ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return encode_tensor_map_5d(map, type, c.base, dims, strides, box, swizzle) ? unit : 1;
}

__device__ __forceinline__ void tma_load_5d(void *dst, const void *map, int x, int y, int z, int u, int w,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(u), "r"(w), "r"(smem_addr(bar))
        : "memory");
}
// One pass of the attention: the rows of each sequence against its own keys,
// or all rows against the shared prefix.
struct PagedPass {
    PagedAttention a;
    int prefix_pass;  // one segment list over all rows, keys [0, prefix), no mask
    int first;        // keys below it are left out (a prefix pass saw them)
    float *pre_o;     // [tokens * heads][head_dim] unnormalised, and
    float *pre_ml;    // [tokens * heads][2]: written by the prefix pass, merged by the other
    float *part_o;    // pieces of segments: unnormalised outputs, and
    float *part_ml;   // their (m, l)
    float scale_log2;
    // Sequences of more query rows per kv head (tokens * group) than this go
    // to paged_rows_kernel, the others to paged_attention_kernel.
    int small_rows;
};

// Whether some row of the segment may see key index i.
template <typename C>
__device__ __forceinline__ bool live_key(const PagedPass &p, const C &c, int i) {
    const int pos = i < c.sink ? i : i - c.sink + c.low;
    return i < c.keys && (pos >= c.from || ((i < c.sink || c.sink == c.low) && pos < p.a.sinks));
}

constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// Powers of two that bring the largest magnitude of a set (its bits) to
// [2^k, 2^(k + 1)): the scale is pow2(k - scale_exponent(bits)).
__device__ __forceinline__ int scale_exponent(uint32_t bits) {
    return bits ? max((int)(bits >> 23) - 127, -100) : 0;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// 16 bytes of a cache row as floats, and one element of it.
template <typename T>
struct Frag;
template <>
struct Frag<float> {
    __device__ static __forceinline__ void ld(const void *p, float (&x)[4]) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    }
    __device__ static __forceinline__ float get(const void *p) { return *static_cast<const float *>(p); }
};
template <>
struct Frag<__nv_bfloat16> {
    __device__ static __forceinline__ void ld(const void *p, float (&x)[8]) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ static __forceinline__ float get(const void *p) {
        return __bfloat162float(*static_cast<const __nv_bfloat16 *>(p));
    }
};
template <>
struct Frag<__half> {
    __device__ static __forceinline__ void ld(const void *p, float (&x)[8]) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
    __device__ static __forceinline__ float get(const void *p) {
        return __half2float(*static_cast<const __half *>(p));
    }
};

// One query row against the keys i in [k0, k1) for which pos(i) is not
// negative, in plain f32, by one warp: for rows whose tiles hold values that
// are not finite. o[y]: dimension lane + 32 y, unnormalised; m in log2 units.
// A lane takes a key's score, the warp 32 keys' values with two or four of them
// in flight: 90 cycles a key where one key at a time took 800. A score that is NaN
// or +infinity makes the whole row NaN and ends it.
template <typename T, int DP, typename Pos>
__device__ __noinline__ void plain_row(const PagedPass &p, const float *q, int b, int kvh, int k0, int k1, Pos pos,
                                       float &m, float &l, float (&o)[DP / 32]) {
    constexpr int kEpl = 16 / (int)sizeof(T), kFly = DP > 128 ? 2 : 4;
    const int lane = threadIdx.x & 31, D = p.a.head_dim;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int y = 0; y < DP / 32; y++) o[y] = 0.f;
    for (int i0 = k0; i0 < k1; i0 += 32) {
        const int at = i0 + lane < k1 ? pos(i0 + lane) : -1;
        long long off = 0;
        float x = -INFINITY;
        if (at >= 0) {
            off = paged_row(p.a.cache, p.a.batch, b, at, p.a.err) + (long long)kvh * D * (int)sizeof(T);
            const char *src = p.a.cache.base + off;
            float part[kEpl];
#pragma unroll
            for (int e = 0; e < kEpl; e++) part[e] = 0.f;
#pragma unroll 2
            for (int d = 0; d < D; d += kEpl) {
                float kv[kEpl];
                Frag<T>::ld(src + d * (int)sizeof(T), kv);
#pragma unroll
                for (int e = 0; e < kEpl; e++) part[e] = fmaf(q[d + e], kv[e], part[e]);
            }
#pragma unroll
            for (int w = kEpl / 2; w; w /= 2)
#pragma unroll
                for (int e = 0; e < w; e++) part[e] += part[e + w];
            x = part[0] * p.scale_log2;
        }
        if (__any_sync(0xffffffffu, !(x < INFINITY))) {
            l = __int_as_float(0x7fffffff);
#pragma unroll
            for (int y = 0; y < DP / 32; y++) o[y] = l;
            return;
        }
        const float nm = fmaxf(m, warp_max(x)), mu = nm == -INFINITY ? 0.f : nm;
        const float f = ex2(m - mu), e = ex2(x - mu);
        l = fmaf(l, f, warp_sum(e));
        m = nm;
#pragma unroll
        for (int y = 0; y < DP / 32; y++) o[y] *= f;
        const unsigned seen = __ballot_sync(0xffffffffu, at >= 0);
        for (int j0 = 0; j0 < 32; j0 += kFly) {
            float ej[kFly], v[kFly][DP / 32];
#pragma unroll
            for (int j = 0; j < kFly; j++) {
                const bool live = (seen >> (j0 + j)) & 1;
                ej[j] = __shfl_sync(0xffffffffu, e, j0 + j);
                const char *src = p.a.cache.base + p.a.cache.parity_stride + __shfl_sync(0xffffffffu, off, j0 + j);
#pragma unroll
                for (int y = 0; y < DP / 32; y++) {
                    const int d = lane + 32 * y;
                    v[j][y] = live && d < D ? Frag<T>::get(src + d * (int)sizeof(T)) : 0.f;
                }
            }
#pragma unroll
            for (int j = 0; j < kFly; j++)
#pragma unroll
                for (int y = 0; y < DP / 32; y++) o[y] = fmaf(ej[j], v[j][y], o[y]);
        }
    }
}

// paged_rows.cu: the pass on the tensor cores, 128 query rows at a time.
bool paged_rows_supported(const PagedAttention &a);
size_t paged_rows_part_floats(const PagedAttention &a);
cudaError_t paged_rows(cudaStream_t s, const PagedPass &p);

}  // namespace k
}  // namespace slc
