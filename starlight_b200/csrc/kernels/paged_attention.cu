// Attention over a paged KV cache: rows of a ragged batch against their own
// sequence's keys (causal, optionally a sliding window with first tokens that
// stay visible), or rows of the whole batch against a prefix that all
// sequences share (SLC_OP_EXT_PAGED_ATTENTION, SLC_OP_EXT_PREFIX_ATTENTION).
//
//   s_p = scale * q . k_p over the positions p that the row sees,
//   m = max s, l = sum exp(s - m), o = sum exp(s - m) v_p / l,
// computed in one pass over the keys with a running m, l and o.
//
// Work. A segment is (sequence, block of kRows query rows, kv head); its keys
// are cut into tiles of kTileKeys. All tiles of all segments form one line
// that the CTAs (one per SM) share out in equal contiguous ranges, so a batch
// of any lengths keeps every SM busy to the end. The cuts are computed on the
// device from the batch's lengths: a captured graph replays with new ones. A
// segment that crosses a cut is merged by the last of its CTAs to finish
// (ticket, no waiting), its pieces in ascending order: results do not depend
// on the order of execution.
//
// A tile is 16 keys for each of the CTA's warps. A warp fetches its keys and
// values row by row (one bulk copy per row and lane) into a ring of its own,
// kStages tiles ahead and across segment borders, and shares nothing with the
// other warps until the segment's end, where the warps' m, l and o merge in
// shared memory.
//
// Arithmetic. mma.sync m16n8k8 on tf32 pairs: x = hi + lo with hi the top 11
// significant bits and lo the rest, three products (hi hi, hi lo, lo hi) for
// an F32 cache: 2^-21 relative, f32 accumulators. F16 and BF16 values are
// exact as one tf32, two products. The tiles are transposed (S^T = K Q^T,
// O^T = V^T P^T), so that the 16 of the MMA are keys and dimensions and the 8
// are query rows: decode has 1 to 8 rows per kv head (GQA), and rows beyond
// that would be padding. Dimensions and keys inside a tile are permuted so
// that every fragment is one 128-bit shared load without bank conflicts (row
// strides of 16 mod 32 words for keys, 8 mod 32 for values).
//
// Rows that meet a NaN or an infinity are recomputed in plain f32 over the
// keys that they see alone (the MMA multiplies masked values by zero, and the
// split of an infinity is NaN).
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "tma.cuh"

namespace slc {
namespace k {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;
constexpr int kWarpKeys = 16;
constexpr int kTileKeys = kWarps * kWarpKeys;
constexpr int kSmallRows = 32;  // query rows per kv head taken here; more go to paged_rows.cu

template <typename T, int DP>
struct Cfg {
    static constexpr int kEpl = 16 / (int)sizeof(T);  // elements of a 128-bit shared load
    static constexpr int kKBlk = 4 * kEpl;             // dims per K fragment block
    static constexpr int kVBlk = 8 * kEpl;             // dims per V fragment block
    static constexpr int kKStride = DP * (int)sizeof(T) + 64;
    static constexpr int kVStride = DP * (int)sizeof(T) + 32;
    static constexpr int kStageBytes = kWarpKeys * (kKStride + kVStride);
    static constexpr int kMergeStride = DP + 4;  // floats
    static constexpr int kFixed = 2 * kRows * DP * 4 + kWarps * kRows * (kMergeStride + 2) * 4 + 4096;
    static constexpr int kFit = (220 * 1024 - kFixed) / (kWarps * kStageBytes);
    static constexpr int kStages = kFit > 4 ? 4 : (kFit < 1 ? 1 : kFit);
    static constexpr int kSmem = kFixed + kStages * kWarps * kStageBytes;
};

// Segment and tile of a unit of the work line, walked forward.
struct Cursor {
    long long left;  // units of this sequence from the current one on, itself included
    int b;           // sequence
    int tok0, ntok, past;
    int sink, low, keys;  // visible keys: [0, sink) and [low, low + keys - sink)
    int tiles, kvh, rb, tile;
};

__device__ __forceinline__ void seq_load(const PagedPass &p, int b, Cursor &c) {
    c.b = b;
    if (p.prefix_pass) {
        c.b = paged_sequence_of(p.a.batch, 0);  // the first with tokens: its table row
        c.tok0 = 0;
        c.ntok = (int)p.a.batch.starts[p.a.batch.seqs];
        c.past = p.a.prefix;
        c.sink = 0;
        c.low = 0;
        c.keys = p.a.prefix;
    } else {
        c.tok0 = (int)p.a.batch.starts[b];
        c.ntok = (int)p.a.batch.starts[b + 1] - c.tok0;
        if ((long long)c.ntok * (p.a.heads / p.a.kv_heads) > p.small_rows) c.ntok = 0;
        c.past = (int)p.a.batch.past[b];
        c.sink = 0;
        c.low = p.first;
        if (p.a.window) {
            c.low = max(c.past + 1 - p.a.window, 0);
            c.sink = min(p.a.sinks, c.low);
        }
        c.keys = c.sink + c.past + c.ntok - c.low;
    }
    c.tiles = (c.keys + kTileKeys - 1) / kTileKeys;
}
__device__ __forceinline__ long long seq_units(const PagedPass &p, const Cursor &c) {
    const long long rb = (c.ntok * (long long)(p.a.heads / p.a.kv_heads) + kRows - 1) / kRows;
    return c.ntok > 0 ? rb * p.a.kv_heads * c.tiles : 0;
}

// Places the cursor on unit `at` counted from the start of sequence c.b.
__device__ __forceinline__ void cursor_at(const PagedPass &p, Cursor &c, long long at) {
    const int seqs = p.prefix_pass ? 1 : p.a.batch.seqs;
    long long n = seq_units(p, c);
    while (!p.prefix_pass && at >= n && c.b + 1 < seqs) {
        at -= n;
        seq_load(p, c.b + 1, c);
        n = seq_units(p, c);
    }
    c.left = n - at;
    const long long seg = at / max(c.tiles, 1);
    c.tile = (int)(at - seg * c.tiles);
    c.rb = (int)(seg / p.a.kv_heads);
    c.kvh = (int)(seg - (long long)c.rb * p.a.kv_heads);
}

__device__ __forceinline__ void cursor_next(const PagedPass &p, Cursor &c) {
    if (--c.left == 0) {
        cursor_at(p, c, seq_units(p, c));
        return;
    }
    if (++c.tile == c.tiles) {
        c.tile = 0;
        if (++c.kvh == p.a.kv_heads) {
            c.kvh = 0;
            c.rb++;
        }
    }
}

__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32_hi(float x) { return __float_as_uint(x) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf32_lo(float x, uint32_t hi) {
    return __float_as_uint(x - __uint_as_float(hi));
}
// Position of compressed key index i.
__device__ __forceinline__ int key_pos(const Cursor &c, int i) {
    return i < c.sink ? i : i - c.sink + c.low;
}
// Whether row position `at` sees key index i.
__device__ __forceinline__ bool sees(const PagedPass &p, const Cursor &c, int i, int at) {
    if (i >= c.keys) return false;
    if (p.prefix_pass) return true;
    const int pos = key_pos(c, i);
    return pos <= at && (!p.a.window || pos > at - p.a.window || pos < p.a.sinks);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) paged_attention_kernel(const __grid_constant__ PagedPass p) {
    using C = Cfg<T, DP>;
    constexpr int EPL = C::kEpl, KB = DP / C::kKBlk, VB = DP / C::kVBlk, NT = DP / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char *ring = smem;
    float *q_hi = reinterpret_cast<float *>(ring + C::kStages * kWarps * C::kStageBytes);
    float *q_lo = q_hi + kRows * DP;
    float *mo = q_lo + kRows * DP;                          // [kWarps][kRows][kMergeStride]
    float *mml = mo + kWarps * kRows * C::kMergeStride;     // [kWarps][kRows][2]
    float *row_ml = mml + kWarps * kRows * 2;               // [kRows][2]
    long long *sums = reinterpret_cast<long long *>(row_ml + kRows * 2);  // [kThreads + 1]
    uint64_t *full = reinterpret_cast<uint64_t *>(sums + kThreads + 1);   // [kWarps][kStages]
    int *flags = reinterpret_cast<int *>(full + kWarps * C::kStages);
    volatile int *abort = flags;
    int *last_s = flags + 1, *bad_s = flags + 2;  // bad_s: bit per row

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int D = p.a.head_dim, H = p.a.heads, Hkv = p.a.kv_heads, G = H / Hkv;
    const int seqs = p.prefix_pass ? 1 : p.a.batch.seqs;
    uint64_t *my_full = full + warp * C::kStages;

    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int i = 0; i < kWarps * C::kStages; i++) mbar_init(&full[i], 1);
        fence_mbar_init();
        *abort = 0;
        *bad_s = 0;
    }
    // Dims past head_dim stay zero in the ring (never copied).
    if (D < DP)
        for (int i = threadIdx.x; i < C::kStages * kWarps * C::kStageBytes / 16; i += kThreads)
            reinterpret_cast<uint4 *>(ring)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();

    // The work line: every thread adds up a run of sequences, thread 0 the runs.
    const int per = (seqs + kThreads - 1) / kThreads;
    {
        long long n = 0;
        for (int i = 0; i < per; i++) {
            const int b = threadIdx.x * per + i;
            if (b < seqs) {
                Cursor c;
                seq_load(p, b, c);
                n += seq_units(p, c);
            }
        }
        sums[threadIdx.x + 1] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sums[0] = 0;
        for (int i = 1; i <= kThreads; i++) sums[i] += sums[i - 1];
    }
    __syncthreads();
    const long long U = sums[kThreads];
    const long long grid = min((long long)gridDim.x, U);
    if (blockIdx.x >= grid) {
        pdl_wait();
        return;
    }
    const long long u0 = U * blockIdx.x / grid, u1 = U * (blockIdx.x + 1) / grid;
    Cursor cc, pc;  // consumer and producer
    {
        int lo = 0;
        for (int i = kThreads; i > 0; i >>= 1)
            while (lo + i <= kThreads && sums[lo + i] <= u0) lo += i;
        seq_load(p, min(lo * per, seqs - 1), cc);
        cursor_at(p, cc, u0 - sums[lo]);
        pc = cc;
    }
    pdl_wait();  // q and the cache come from earlier kernels; workspace use may overlap none

    const uint64_t policy = policy_evict_first();
    const uint32_t row_bytes = (uint32_t)(D * sizeof(T));
    // Copies the warp's 16 keys (lanes 0..15) and values (lanes 16..31) of
    // the producer's unit into a stage. Rows past the segment's keys: values
    // are zeroed (they meet zero probabilities), scores are masked.
    auto issue = [&](int stage) {
        unsigned char *st = ring + (warp * C::kStages + stage) * C::kStageBytes;
        const int r = lane & 15, parity = lane >> 4;
        const int i = pc.tile * kTileKeys + warp * kWarpKeys + r;
        const bool live = i < pc.keys;
        unsigned char *dst = parity ? st + kWarpKeys * C::kKStride + r * C::kVStride : st + r * C::kKStride;
        const int rows = __popc(__ballot_sync(0xffffffffu, live));
        if (!live && parity)
            for (int j = 0; j < DP * (int)sizeof(T) / 16; j++)
                reinterpret_cast<uint4 *>(dst)[j] = make_uint4(0, 0, 0, 0);
        if (rows < 32) fence_proxy_async_smem();
        if (lane == 0) mbar_arrive_expect_tx(&my_full[stage], rows * row_bytes);
        __syncwarp();
        if (live) {
            const char *src = p.a.cache.base + paged_row(p.a.cache, p.a.batch, pc.b, key_pos(pc, i), p.a.err) +
                              parity * p.a.cache.parity_stride + (long long)pc.kvh * row_bytes;
            bulk_g2s(dst, src, row_bytes, &my_full[stage], policy);
        }
    };
    const int units = (int)(u1 - u0);
    int issued = 0;
    for (; issued < C::kStages && issued < units; issued++) {
        if (issued) cursor_next(p, pc);
        issue(issued);
    }

    float acc[NT][4];  // O^T: dims x rows
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    int at0 = 0, at1 = 0;      // positions of rows 2t, 2t + 1
    long long seg_u0 = u0;     // this CTA's first unit of the current segment
    bool fresh = true;
    int done = 0;
    for (long long u = u0; u < u1; u++) {
        if (fresh) {
            // Queries of the segment as tf32 pairs, in fragment order: block j
            // of kKBlk dims, lane (g, t) holds row g, dims j kKBlk + EPL t + e.
            for (int i = threadIdx.x; i < kRows * DP; i += kThreads) {
                const int e = i % 4, ln = (i / 4) % 32, x = i / 128;  // x = j * (EPL / 4) + e / 4
                const int j = x / (EPL / 4), ee = (x % (EPL / 4)) * 4 + e;
                const int r = ln >> 2, d = j * C::kKBlk + EPL * (ln & 3) + ee;
                const int row = cc.rb * kRows + r, tok = row / G;
                float v = 0.f;
                if (tok < cc.ntok && d < D)
                    v = p.a.q[((size_t)(cc.tok0 + tok) * H + cc.kvh * G + (row - tok * G)) * D + d];
                const uint32_t hi = tf32_hi(v);
                q_hi[i] = __uint_as_float(hi);
                q_lo[i] = __uint_as_float(tf32_lo(v, hi));
            }
            at0 = cc.past + (cc.rb * kRows + 2 * t) / G;
            at1 = cc.past + (cc.rb * kRows + 2 * t + 1) / G;
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = 0.f;
            m0 = m1 = -INFINITY;
            l0 = l1 = 0.f;
            seg_u0 = u;
            fresh = false;
            __syncthreads();
        }
        const int stage = done % C::kStages;
        mbar_wait(&my_full[stage], (done / C::kStages) & 1, p.a.err, abort);
        const unsigned char *ks = ring + (warp * C::kStages + stage) * C::kStageBytes;
        const unsigned char *vs = ks + kWarpKeys * C::kKStride;

        // S^T: keys g, g + 8 x rows 2t, 2t + 1.
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) s[i][j] = 0.f;
#pragma unroll
        for (int j = 0; j < KB; j++) {
            float ka[EPL], kb[EPL];
            Frag<T>::ld(ks + g * C::kKStride + (j * C::kKBlk + EPL * t) * sizeof(T), ka);
            Frag<T>::ld(ks + (g + 8) * C::kKStride + (j * C::kKBlk + EPL * t) * sizeof(T), kb);
#pragma unroll
            for (int x = 0; x < EPL / 4; x++) {
                const float4 qh = reinterpret_cast<const float4 *>(q_hi)[(j * (EPL / 4) + x) * 32 + lane];
                const float4 ql = reinterpret_cast<const float4 *>(q_lo)[(j * (EPL / 4) + x) * 32 + lane];
                const float h4[4] = {qh.x, qh.y, qh.z, qh.w}, w4[4] = {ql.x, ql.y, ql.z, ql.w};
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int e = 4 * x + 2 * y;
                    const float f[4] = {ka[e], kb[e], ka[e + 1], kb[e + 1]};
                    uint32_t hi[4];
#pragma unroll
                    for (int z = 0; z < 4; z++) hi[z] = sizeof(T) == 4 ? tf32_hi(f[z]) : __float_as_uint(f[z]);
                    const uint32_t b0 = __float_as_uint(h4[2 * y]), b1 = __float_as_uint(h4[2 * y + 1]);
                    mma_tf32(s[2 + y], hi, __float_as_uint(w4[2 * y]), __float_as_uint(w4[2 * y + 1]));
                    mma_tf32(s[y], hi, b0, b1);
                    if (sizeof(T) == 4) {
                        uint32_t lo[4];
#pragma unroll
                        for (int z = 0; z < 4; z++) lo[z] = tf32_lo(f[z], hi[z]);
                        mma_tf32(s[2 + y], lo, b0, b1);
                    }
                }
            }
        }
        const int i0 = cc.tile * kTileKeys + warp * kWarpKeys + g, i1 = i0 + 8;
        float sc[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float x = ((s[2][j] + s[3][j]) + (s[0][j] + s[1][j])) * p.scale_log2;
            sc[j] = sees(p, cc, j < 2 ? i0 : i1, (j & 1) ? at1 : at0) ? x : -INFINITY;
        }
        float n0 = fmaxf(sc[0], sc[2]), n1 = fmaxf(sc[1], sc[3]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
            n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
        }
        n0 = fmaxf(n0, m0);
        n1 = fmaxf(n1, m1);
        const float u_0 = n0 == -INFINITY ? 0.f : n0, u_1 = n1 == -INFINITY ? 0.f : n1;
        float pr[4];
        pr[0] = ex2(sc[0] - u_0);
        pr[1] = ex2(sc[1] - u_1);
        pr[2] = ex2(sc[2] - u_0);
        pr[3] = ex2(sc[3] - u_1);
        const float f0 = ex2(m0 - u_0), f1 = ex2(m1 - u_1);
        l0 *= f0;
        l1 *= f1;
        m0 = n0;
        m1 = n1;
        l0 += pr[0] + pr[2];
        l1 += pr[1] + pr[3];
        // P as the B fragments of the two 8-key steps: row g, keys t and t + 4.
        uint32_t bh[2][2], bl[2][2];
#pragma unroll
        for (int ks8 = 0; ks8 < 2; ks8++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int src = (t + 4 * x) * 4 + (g >> 1);
                const float a = __shfl_sync(0xffffffffu, pr[2 * ks8], src);
                const float b = __shfl_sync(0xffffffffu, pr[2 * ks8 + 1], src);
                const float v = (g & 1) ? b : a;
                bh[ks8][x] = tf32_hi(v);
                bl[ks8][x] = tf32_lo(v, bh[ks8][x]);
            }
        // The tile's P V starts from zero and is added to the running output
        // outside the tensor core, whose accumulation truncates: over
        // thousands of keys that bias would grow past f32 rounding.
#pragma unroll
        for (int j = 0; j < VB; j++) {
            float o[EPL / 2][4];
#pragma unroll
            for (int x = 0; x < EPL / 2; x++)
#pragma unroll
                for (int z = 0; z < 4; z++) o[x][z] = 0.f;
#pragma unroll
            for (int ks8 = 0; ks8 < 2; ks8++) {
                float va[EPL], vb[EPL];
                Frag<T>::ld(vs + (8 * ks8 + t) * C::kVStride + (j * C::kVBlk + EPL * g) * sizeof(T), va);
                Frag<T>::ld(vs + (8 * ks8 + t + 4) * C::kVStride + (j * C::kVBlk + EPL * g) * sizeof(T), vb);
#pragma unroll
                for (int x = 0; x < EPL / 2; x++) {
                    const float f[4] = {va[2 * x], va[2 * x + 1], vb[2 * x], vb[2 * x + 1]};
                    uint32_t hi[4];
#pragma unroll
                    for (int z = 0; z < 4; z++) hi[z] = sizeof(T) == 4 ? tf32_hi(f[z]) : __float_as_uint(f[z]);
                    mma_tf32(o[x], hi, bl[ks8][0], bl[ks8][1]);
                    if (sizeof(T) == 4) {
                        uint32_t lo[4];
#pragma unroll
                        for (int z = 0; z < 4; z++) lo[z] = tf32_lo(f[z], hi[z]);
                        mma_tf32(o[x], lo, bh[ks8][0], bh[ks8][1]);
                    }
                    mma_tf32(o[x], hi, bh[ks8][0], bh[ks8][1]);
                }
            }
#pragma unroll
            for (int x = 0; x < EPL / 2; x++) {
                float(&a)[4] = acc[j * (EPL / 2) + x];
                a[0] = fmaf(a[0], f0, o[x][0]);
                a[1] = fmaf(a[1], f1, o[x][1]);
                a[2] = fmaf(a[2], f0, o[x][2]);
                a[3] = fmaf(a[3], f1, o[x][3]);
            }
        }
        __syncwarp();
        done++;
        if (issued < units && !*abort) {
            cursor_next(p, pc);
            issue(stage);
            issued++;
        }

        const bool seg_end = cc.tile == cc.tiles - 1;
        if (!seg_end && u + 1 < u1) {
            cc.tile++;
            cc.left--;
            continue;
        }

        // ---- end of this CTA's piece of the segment: merge the warps.
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            l0 += __shfl_xor_sync(0xffffffffu, l0, o);
            l1 += __shfl_xor_sync(0xffffffffu, l1, o);
        }
        float *w0 = mo + (warp * kRows + 2 * t) * C::kMergeStride, *w1 = w0 + C::kMergeStride;
#pragma unroll
        for (int i = 0; i < NT; i++) {
            const int d = (i / (EPL / 2)) * C::kVBlk + EPL * g + 2 * (i % (EPL / 2));
            *reinterpret_cast<float2 *>(w0 + d) = make_float2(acc[i][0], acc[i][2]);
            *reinterpret_cast<float2 *>(w1 + d) = make_float2(acc[i][1], acc[i][3]);
        }
        if (g == 0) {
            float *ml = mml + (warp * kRows + 2 * t) * 2;
            ml[0] = m0, ml[1] = l0, ml[2] = m1, ml[3] = l1;
        }
        __syncthreads();
        const int rows = min(kRows, cc.ntok * G - cc.rb * kRows);
        // Row r, dims d .. d + 3 of the merge, d = 4 (i % (DP / 4)).
        for (int i = threadIdx.x; i < kRows * DP / 4; i += kThreads) {
            const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
            float mm = -INFINITY;
            for (int w = 0; w < kWarps; w++) mm = fmaxf(mm, mml[(w * kRows + r) * 2]);
            const float mu = mm == -INFINITY ? 0.f : mm;
            float ll = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            bool odd = false;
            for (int w = 0; w < kWarps; w++) {
                const float mw = mml[(w * kRows + r) * 2], lw = mml[(w * kRows + r) * 2 + 1];
                const float f = ex2(mw - mu);
                const float4 x = *reinterpret_cast<const float4 *>(mo + (w * kRows + r) * C::kMergeStride + d);
                ll = fmaf(lw, f, ll);
                o.x = fmaf(x.x, f, o.x);
                o.y = fmaf(x.y, f, o.y);
                o.z = fmaf(x.z, f, o.z);
                o.w = fmaf(x.w, f, o.w);
                odd |= !(mw < INFINITY);
            }
            odd |= !finite(ll) || !finite(o.x) || !finite(o.y) || !finite(o.z) || !finite(o.w);
            if (odd && r < rows && d < D) atomicOr(bad_s, 1 << r);
            *reinterpret_cast<float4 *>(mo + r * C::kMergeStride + d) = o;  // warp 0's rows, read above by this thread alone
            if (d == 0) {
                row_ml[2 * r] = mm;
                row_ml[2 * r + 1] = ll;
            }
        }
        __syncthreads();
        if (*bad_s) {
            // Plain f32 over the visible keys of the piece, a warp per row.
            const int k0 = (cc.tile - (int)(u - seg_u0)) * kTileKeys;
            const int k1 = min(cc.keys, (cc.tile + 1) * kTileKeys);
            for (int r = warp; r < rows; r += kWarps) {
                if (!((*bad_s >> r) & 1)) continue;
                const int row = cc.rb * kRows + r, tok = row / G, at = cc.past + tok;
                const float *q = p.a.q + ((size_t)(cc.tok0 + tok) * H + cc.kvh * G + (row - tok * G)) * D;
                float mm, ll, o[DP / 32];
                plain_row<T, DP>(
                    p, q, cc.b, cc.kvh, k0, k1, [&](int i) { return sees(p, cc, i, at) ? key_pos(cc, i) : -1; }, mm,
                    ll, o);
#pragma unroll
                for (int y = 0; y < DP / 32; y++) mo[r * C::kMergeStride + lane + 32 * y] = o[y];
                if (lane == 0) {
                    row_ml[2 * r] = mm;
                    row_ml[2 * r + 1] = ll;
                }
            }
            __syncthreads();
            if (threadIdx.x == 0) *bad_s = 0;
        }

        // ---- the segment's result, or a piece of it for the merge.
        const long long a0 = u - cc.tile, a1 = a0 + cc.tiles;  // the segment's units
        bool write = true;
        if (a0 < u0 || a1 > u1) {
            const int c_first = (int)(((a0 + 1) * grid - 1) / U), c_last = (int)((a1 * grid - 1) / U);
            const int slot = 2 * blockIdx.x + (a0 >= u0 ? 1 : 0);
            float *po = p.part_o + (size_t)slot * kRows * DP, *pml = p.part_ml + (size_t)slot * kRows * 2;
            for (int i = threadIdx.x; i < rows * DP / 4; i += kThreads) {
                const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
                *reinterpret_cast<float4 *>(po + r * DP + d) =
                    *reinterpret_cast<const float4 *>(mo + r * C::kMergeStride + d);
            }
            if (threadIdx.x < 2 * rows) pml[threadIdx.x] = row_ml[threadIdx.x];
            __syncthreads();
            if (threadIdx.x == 0) {
                __threadfence();
                const unsigned ticket = atomicAdd(&p.a.tickets[c_first], 1u);
                *last_s = ticket == (unsigned)(c_last - c_first);
                if (*last_s) p.a.tickets[c_first] = 0u;
                __threadfence();
            }
            __syncthreads();
            write = *last_s;
            if (write) {
                const int pieces = c_last - c_first + 1;
                for (int i = threadIdx.x; i < rows * DP / 4; i += kThreads) {
                    const int r = i / (DP / 4), d = 4 * (i % (DP / 4));
                    float mm = -INFINITY, ll = 0.f;
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
                    for (int x = 0; x < pieces; x++) {
                        const size_t sl = x == 0 ? 2 * (size_t)c_first + 1 : 2 * (size_t)(c_first + x);
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p.part_ml) + sl * kRows + r);
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(p.part_o + (sl * kRows + r) * DP + d));
                        const float nm = fmaxf(mm, ml.x), mu = nm == -INFINITY ? 0.f : nm;
                        const float f = ex2(mm - mu), e = ex2(ml.x - mu);
                        ll = fmaf(ml.y, e, ll * f);
                        o.x = fmaf(v.x, e, o.x * f);
                        o.y = fmaf(v.y, e, o.y * f);
                        o.z = fmaf(v.z, e, o.z * f);
                        o.w = fmaf(v.w, e, o.w * f);
                        mm = nm;
                    }
                    *reinterpret_cast<float4 *>(mo + r * C::kMergeStride + d) = o;
                    if (d == 0) {
                        row_ml[2 * r] = mm;
                        row_ml[2 * r + 1] = ll;
                    }
                }
                __syncthreads();
            }
        }
        if (write) {
            for (int i = threadIdx.x; i < rows * D / 4; i += kThreads) {
                const int r = i / (D / 4), d = 4 * (i % (D / 4));
                const int row = cc.rb * kRows + r, tok = row / G;
                const size_t at = (size_t)(cc.tok0 + tok) * H + cc.kvh * G + (row - tok * G);
                float4 o = *reinterpret_cast<const float4 *>(mo + r * C::kMergeStride + d);
                float mm = row_ml[2 * r], ll = row_ml[2 * r + 1];
                if (p.prefix_pass) {
                    *reinterpret_cast<float4 *>(p.pre_o + at * D + d) = o;
                    if (d == 0) *reinterpret_cast<float2 *>(p.pre_ml + at * 2) = make_float2(mm, ll);
                    continue;
                }
                if (p.pre_o) {
                    const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p.pre_ml) + at);
                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(p.pre_o + at * D + d));
                    const float nm = fmaxf(mm, ml.x), mu = nm == -INFINITY ? 0.f : nm;
                    const float f = ex2(mm - mu), e = ex2(ml.x - mu);
                    ll = fmaf(ml.y, e, ll * f);
                    o.x = fmaf(v.x, e, o.x * f);
                    o.y = fmaf(v.y, e, o.y * f);
                    o.z = fmaf(v.z, e, o.z * f);
                    o.w = fmaf(v.w, e, o.w * f);
                }
                float *dst = p.a.out + at * D + d;  // 4-byte aligned
                dst[0] = __fdiv_rn(o.x, ll);
                dst[1] = __fdiv_rn(o.y, ll);
                dst[2] = __fdiv_rn(o.z, ll);
                dst[3] = __fdiv_rn(o.w, ll);
            }
        }
        __syncthreads();
        fresh = true;
        if (u + 1 < u1) cursor_next(p, cc);
    }
    // After a wait that gave up, copies may still be in flight: let them land
    // before the CTA's shared memory is released.
    if (*abort) {
        const int from = issued > C::kStages ? issued - C::kStages : 0;
        for (int i = from; i < issued; i++) {
            const uint64_t t0 = global_ns();
            while (!mbar_try_wait(&my_full[i % C::kStages], (i / C::kStages) & 1) &&
                   global_ns() - t0 < 100000000ull) {
            }
        }
    }
}

int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

size_t partial_floats(int dp) { return (size_t)2 * kSmCount * kRows * (dp + 2); }
size_t prefix_floats(const PagedAttention &a) {
    return a.prefix ? (size_t)a.tokens * a.heads * (a.head_dim + 2) : 0;
}

template <typename T, int DP>
cudaError_t launch_pass(cudaStream_t s, const PagedPass &p) {
    using C = Cfg<T, DP>;
    static_assert(C::kSmem <= 227 * 1024, "shared layout");
    static std::atomic<uint64_t> smem_set{0};
    set_smem_limit_once(paged_attention_kernel<T, DP>, C::kSmem, &smem_set);
    launch_k(paged_attention_kernel<T, DP>, kSmCount, kThreads, C::kSmem, s, p);
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_dim(cudaStream_t s, const PagedPass &p) {
    switch (padded_dim(p.a.head_dim)) {
    case 64: return launch_pass<T, 64>(s, p);
    case 128: return launch_pass<T, 128>(s, p);
    default: return launch_pass<T, 256>(s, p);
    }
}

cudaError_t launch_type(cudaStream_t s, const PagedPass &p) {
    switch (p.a.cache.type) {
    case kPagedF16: return launch_dim<__half>(s, p);
    case kPagedBf16: return launch_dim<__nv_bfloat16>(s, p);
    default: return launch_dim<float>(s, p);
    }
}

// Whether rows * group query rows of one kv head are too many for
// paged_attention_kernel, which reads the keys once per kRows of them.
bool many_rows(const PagedAttention &a, size_t rows) {
    return paged_rows_supported(a) && rows * (size_t)(a.heads / a.kv_heads) > (size_t)kSmallRows;
}

size_t part_floats(const PagedAttention &a) {
    const size_t few = partial_floats(padded_dim(a.head_dim));
    const bool rows = many_rows(a, a.max_new) || (a.prefix && many_rows(a, a.tokens));
    return rows ? std::max(few, paged_rows_part_floats(a)) : few;
}

}  // namespace

size_t paged_attention_workspace_bytes(const PagedAttention &a) {
    return (part_floats(a) + prefix_floats(a)) * sizeof(float);
}

cudaError_t paged_attention(cudaStream_t s, const PagedAttention &a) {
    if (a.tokens == 0 || a.batch.seqs == 0) return cudaSuccess;
    if (paged_attention_workspace_bytes(a) > a.workspace_bytes) return cudaErrorMemoryAllocation;
    PagedPass p{};
    p.a = a;
    p.scale_log2 = a.scale * kLog2e;
    p.part_o = static_cast<float *>(a.workspace);
    p.part_ml = p.part_o + (size_t)2 * kSmCount * kRows * padded_dim(a.head_dim);
    p.small_rows = INT32_MAX;
    cudaError_t e = cudaSuccess;
    if (a.prefix) {
        p.pre_o = p.part_o + part_floats(a);
        p.pre_ml = p.pre_o + (size_t)a.tokens * a.heads * a.head_dim;
        p.prefix_pass = 1;
        e = many_rows(a, a.tokens) ? paged_rows(s, p) : launch_type(s, p);
        if (e != cudaSuccess) return e;
        p.prefix_pass = 0;
        p.first = a.prefix;
    }
    // Sequences with many rows first, those with few after them.
    if (many_rows(a, a.max_new)) {
        p.small_rows = kSmallRows;
        e = paged_rows(s, p);
        if (e != cudaSuccess) return e;
    }
    return launch_type(s, p);
}

}  // namespace k
}  // namespace slc
