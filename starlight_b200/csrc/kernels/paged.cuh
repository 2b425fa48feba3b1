// Paged KV cache: addressing shared by the append and attention kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "tma.cuh"

namespace slc {
namespace k {

// Byte offset (from cache.base) of the key row of position `pos` of sequence
// `b`, head 0. The host has checked every page id that a position in use
// names; the guard keeps a wrong one from leaving the cache (page 0 then
// stands in, and the device error word is set).
__device__ __forceinline__ long long paged_row(const PagedCache &c, const PagedBatch &batch, int b,
                                               int pos, uint32_t *err) {
    const int pg = pos / c.page, off = pos - pg * c.page;
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

}  // namespace k
}  // namespace slc
