// Attention over a paged KV cache for many query rows: prompts, and the rows
// of a whole batch against the prefix that its sequences share. The same
// definition and work line as paged_attention.cu; a segment is (sequence, 128
// query rows, kv head), a tile 128 keys, and the products run on tcgen05.
//
// Arithmetic. kind::f16 with f32 accumulators on pairs of f16: x = hi + lo
// keeps 22 bits, and f16's denormals keep 2^-39 of the largest value below
// that, given scales (powers of two, exact) that bring the largest value of a
// query row, of a key tile and of a value tile to [2^14, 2^15). Probabilities
// are taken 2^14 times as large for the same reason. An F32 cache needs three
// products (lo hi, hi lo, hi hi) for S = Q K^T and for P V; F16 and BF16
// values are one f16 each (to the same 2^-39), two products. A value that is
// more than 2^18 times smaller than its tile's largest keeps fewer than 22
// bits. Every tile's P V starts from zero and is added in f32 registers
// (TMEM accumulation over thousands of keys would truncate thousands of
// times).
//
// One CTA per SM, 16 warps:
//   0..3   softmax: one thread per row; Q of a segment to TMEM as f16 pairs;
//          S from TMEM, running maximum, P as f16 pairs back into the TMEM
//          columns that S held
//   4..7   output: one thread per row; O += P V of each tile in registers,
//          the merge of a split segment, the result
//   8..14  producers: K and V tiles from the pages by 16-byte asynchronous
//          copies into a ring of slots, then in place (the tile's largest
//          value, scale, f16 or f16 pair) the 128-byte swizzled operand
//   15     issues the MMAs: Q K^T of the next tile before P V of this one
// The ring holds operands in the order of their MMAs (K0 K1 V0 K2 V1 ...), so
// a slot is free as soon as the MMA kSlots back is done; three slots of pairs
// or six of single f16. Q and P are A operands from TMEM; K is read K-major
// and V MN-major from the same layout ([key][64 dims] rows of 128 bytes).
// TMEM: Q, two S / P buffers and O, 128 columns each.
//
// Tensor-bound: 4 * pairs * D flops take 4 (16-bit cache) or 6 (F32) passes of
// half as many MMA flops each.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace slc {
namespace k {
namespace {

constexpr int kM = 128;     // query rows per segment
constexpr int kKeys = 128;  // keys per tile
constexpr int kProducers = 7;
constexpr int kThreads = 16 * 32;
constexpr int kShift = 14;  // largest scaled value in [2^14, 2^15)
// Registers a thread: 128 at launch; softmax, output, and the two warpgroups of
// producers (the MMA warp is the last of them).
constexpr int kLaunchRegs = 128, kSoftRegs = 104, kOutRegs = 200, kProdRegs = 104;
static_assert(kSoftRegs + kOutRegs + 2 * kProdRegs <= 4 * kLaunchRegs, "register split");
constexpr uint64_t kLimitNs = 4000000000ull;  // rows of values that are not finite take long

template <typename T, int DP>
struct Cfg {
    static constexpr bool kPair = sizeof(T) == 4;            // keys and values are f16 pairs
    static constexpr bool kRaw = std::is_same<T, __half>::value;  // taken as they are
    static constexpr int kBlocks = DP / 64;                  // 128-byte blocks along the dims
    static constexpr int kBlockBytes = kKeys * 128;          // 16 KiB
    static constexpr int kHalfBytes = kBlocks * kBlockBytes;  // one of hi, lo
    static constexpr int kTileBytes = kHalfBytes * (kPair ? 2 : 1);
    static constexpr int kSlots = kPair && DP == 128 ? 3 : 6;
    static constexpr int kAhead = kSlots / 2;                // operands copied ahead of the one converted
    static constexpr int kRing = kSlots * kTileBytes;
    static constexpr int kSmall = 4 * (2 * 4 * kM + 4 * kM + 4 * 8 + 8 + 4 * DP + 16) + 8 * (8 + 2 * kSlots + 8 + 20);
    static constexpr int kSmem = 1024 + kRing + kSmall;
    static constexpr int kEpl = 16 / (int)sizeof(T);    // elements of a 16-byte load
    static constexpr int kLpr = DP / kEpl;               // lanes per cache row
    static constexpr int kRpi = 32 / kLpr;               // rows per warp load
    static constexpr int kLoads = (kKeys / kRpi + kProducers - 1) / kProducers;
    // f32 accumulators, f16 operands, K-major A; B K-major (S) or MN-major (O).
    static constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
    static constexpr uint32_t kIdescO =
        (1u << 4) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
};

// A segment of the work line and a place in it.
struct Cursor {
    int b, rt, kvh, tile;  // sequence, row tile, kv head, key tile
    int tok0, ntok, past;  // of the sequence
    int r0, rows;          // of the row tile
    int sink, low, keys, tiles;
};

__device__ __forceinline__ int group_of(const PagedPass &p) { return p.a.heads / p.a.kv_heads; }
__device__ __forceinline__ int seq_count(const PagedPass &p) { return p.prefix_pass ? 1 : p.a.batch.seqs; }

__device__ __forceinline__ void seq_load(const PagedPass &p, int b, Cursor &c) {
    c.b = b;
    if (p.prefix_pass) {
        c.b = paged_sequence_of(p.a.batch, 0);  // the first with tokens: its table row
        c.tok0 = 0;
        c.ntok = (int)p.a.batch.starts[p.a.batch.seqs];
        c.past = p.a.prefix;
    } else {
        c.tok0 = (int)p.a.batch.starts[b];
        c.ntok = (int)p.a.batch.starts[b + 1] - c.tok0;
        c.past = (int)p.a.batch.past[b];
        if ((long long)c.ntok * group_of(p) <= p.small_rows) c.ntok = 0;
    }
}
__device__ __forceinline__ int row_tiles(const PagedPass &p, const Cursor &c) {
    return (int)(((long long)c.ntok * group_of(p) + kM - 1) / kM);
}
// The keys of row tile c.rt: those that any of its rows sees.
__device__ __forceinline__ void row_tile_load(const PagedPass &p, Cursor &c) {
    const int G = group_of(p);
    c.r0 = c.rt * kM;
    c.rows = min(kM, c.ntok * G - c.r0);
    c.sink = 0;
    c.low = p.first;
    if (p.prefix_pass) {
        c.keys = p.a.prefix;
    } else {
        const int first = c.past + c.r0 / G, last = c.past + (c.r0 + c.rows - 1) / G;
        if (p.a.window) {
            c.low = max(first + 1 - p.a.window, 0);
            c.sink = min(p.a.sinks, c.low);
        }
        c.keys = c.sink + last + 1 - c.low;
    }
    c.tiles = (c.keys + kKeys - 1) / kKeys;
}
__device__ __forceinline__ long long seq_units(const PagedPass &p, Cursor &c) {
    long long n = 0;
    const int rts = row_tiles(p, c);
    for (c.rt = 0; c.rt < rts; c.rt++) {
        row_tile_load(p, c);
        n += c.tiles;
    }
    return n * p.a.kv_heads;
}
// Places the cursor on unit `at` of the line from sequence c.b on (c.rt 0).
__device__ __forceinline__ void cursor_at(const PagedPass &p, Cursor &c, long long at) {
    for (;;) {
        const int rts = row_tiles(p, c);
        for (c.rt = 0; c.rt < rts; c.rt++) {
            row_tile_load(p, c);
            const long long n = (long long)c.tiles * p.a.kv_heads;
            if (at < n) {
                c.kvh = (int)(at / c.tiles);
                c.tile = (int)(at - (long long)c.kvh * c.tiles);
                return;
            }
            at -= n;
        }
        if (p.prefix_pass || c.b + 1 >= p.a.batch.seqs) return;
        seq_load(p, c.b + 1, c);
    }
}
// The next unit; the line's end is the caller's to know.
__device__ __forceinline__ void cursor_next(const PagedPass &p, Cursor &c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.kvh < p.a.kv_heads) return;
    c.kvh = 0;
    if (++c.rt < row_tiles(p, c)) {
        row_tile_load(p, c);
        return;
    }
    if (p.prefix_pass || c.b + 1 >= p.a.batch.seqs) return;
    seq_load(p, c.b + 1, c);
    cursor_at(p, c, 0);
}

__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// (a, b) as an f16 pair, a low; and the value that it holds.
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
// Element (row, dim) of a swizzled operand: block dim / 64 of rows of 128
// bytes, 16-byte chunks xored with the row.
__device__ __forceinline__ uint32_t operand_at(int row, int dim) {
    return (uint32_t)((dim >> 6) * kKeys * 128 + row * 128 + ((((dim & 63) >> 3) ^ (row & 7)) << 4) + (dim & 7) * 2);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) paged_rows_kernel(const __grid_constant__ PagedPass p) {
    using C = Cfg<T, DP>;
    constexpr int S = C::kSlots;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    const uint32_t raw = smem_addr(smem_raw);
    unsigned char *smem = smem_raw + ((1024 - (raw & 1023)) & 1023);
    unsigned char *ring = smem;                         // [S] operands: hi[, lo]
    float *row_ml = reinterpret_cast<float *>(smem + C::kRing);  // [4 tiles][kM][2]
    float *alpha = row_ml + 4 * kM * 2;                 // [4 tiles][kM]
    float *k_scale = alpha + 4 * kM;                    // [8 tiles]
    float *v_scale = k_scale + 8;                       // [8 tiles]
    uint32_t *k_max = reinterpret_cast<uint32_t *>(v_scale + 8);  // [4 tiles]
    uint32_t *v_max = k_max + 4;                        // [4 tiles]
    int *poison = reinterpret_cast<int *>(v_max + 4);   // [8 segments]
    float *scratch = reinterpret_cast<float *>(poison + 8);       // [4 warps][DP]
    int *flags = reinterpret_cast<int *>(scratch + 4 * DP);
    volatile int *abort = flags;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(flags + 1);
    int *last_s = flags + 2;
    long long *sums = reinterpret_cast<long long *>(flags + 4);   // [4] a scan's warps, [2] what it found
    uint64_t *bars = reinterpret_cast<uint64_t *>(sums + 6);
    uint64_t *full = bars, *empty = full + S;           // [S] the ring's
    uint64_t *q_full = empty + S, *s_full = q_full + 1, *p_full = s_full + 2, *o_full = p_full + 2,
             *o_empty = o_full + 1, *done = o_empty + 1;
    // What threads pass each other beside the operands, in rings long enough
    // for the lead that the barriers above allow.
    uint64_t *k_sc = done + 1, *v_sc = k_sc + 8, *a_full = v_sc + 8;  // [8], [8], [4]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int D = p.a.head_dim, H = p.a.heads, G = group_of(p);

    pdl_trigger();
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; i++) {
            mbar_init(&full[i], kProducers);
            mbar_init(&empty[i], 1);
        }
        mbar_init(q_full, 4);
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        mbar_init(o_full, 1);
        mbar_init(o_empty, 4);
        mbar_init(done, 1);
        for (int i = 0; i < 8; i++) {
            mbar_init(&k_sc[i], 1);
            mbar_init(&v_sc[i], 1);
        }
        for (int i = 0; i < 4; i++) mbar_init(&a_full[i], 4);
        fence_mbar_init();
        *abort = 0;
        for (int i = 0; i < 4; i++) k_max[i] = v_max[i] = 0;
        for (int i = 0; i < 8; i++) poison[i] = 0;
    }
    // The work line, as in paged_attention_kernel (the first kM threads).
    const int seqs = seq_count(p);
    const int per = (seqs + kM - 1) / kM;
    long long mine = 0, upto = 0;
    if (warp < 4) {
        for (int i = 0; i < per; i++) {
            const int b = threadIdx.x * per + i;
            if (b < seqs) {
                Cursor c;
                seq_load(p, b, c);
                mine += seq_units(p, c);
            }
        }
        upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) sums[warp] = upto;
    }
    __syncthreads();
    long long U = 0;
    for (int w = 0; w < 4; w++) {
        if (w < warp) upto += sums[w];
        U += sums[w];
    }
    const long long grid = min((long long)gridDim.x, U);
    if (blockIdx.x >= grid) {
        pdl_wait();
        return;
    }
    if (warp == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_addr(tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const long long u0 = U * blockIdx.x / grid, u1 = U * (blockIdx.x + 1) / grid;
    if (warp < 4 && upto - mine <= u0 && u0 < upto) {
        sums[4] = threadIdx.x;
        sums[5] = upto - mine;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t s_tm = tmem, o_tm = tmem + 256, q_tm = tmem + 384;  // S: two buffers
    const int N = (int)(u1 - u0);
    Cursor c;
    seq_load(p, (int)sums[4] * per, c);
    cursor_at(p, c, u0 - sums[5]);
    pdl_wait();

    // No wait below ends a loop: after one that gave up (the abort word is
    // set) every role runs through its remaining steps without waiting, so
    // that the barriers between its own threads stay matched.
    if (warp < 4)
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    else if (warp < 8)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kOutRegs));
    else
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProdRegs));
    if (warp < 4) {
        // ---- softmax ------------------------------------------------------
        const int r = threadIdx.x;
        const uint32_t lane_tm = (uint32_t)(warp * 32) << 16;
        float m = -INFINITY, l = 0.f, qs = 1.f;
        int hi = 0, lo = 0;
        bool first = true;
        for (int n = 0; n < N; n++) {
            if (first) {
                // The row to TMEM: hi in columns 0 .. DP / 2, lo behind them.
                // The segment before is through with Q (its last S is read).
                const int row = c.r0 + r, tok = row / G;
                const bool live = r < c.rows;
                const float *q = p.a.q + (live ? ((size_t)(c.tok0 + tok) * H + c.kvh * G + (row - tok * G)) * D : 0);
                const bool vec = aligned16(p.a.q);
                auto load4 = [&](int d, float(&x)[4]) {
                    if (live && d < D && vec) {
                        const float4 v = *reinterpret_cast<const float4 *>(q + d);
                        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; e++) x[e] = live && d < D ? q[d + e] : 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] *= p.scale_log2;
                };
                uint32_t top = 0;
#pragma unroll 8
                for (int d = 0; d < DP; d += 4) {
                    float x[4];
                    load4(d, x);
#pragma unroll
                    for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
                }
                const int ex = scale_exponent(top);
                const float sc = pow2(kShift - ex);
                qs = pow2(ex - kShift);
#pragma unroll 1
                for (int h = 0; h < DP / 32; h++) {
                    uint32_t qh[16], ql[16];
#pragma unroll
                    for (int d = 0; d < 32; d += 4) {
                        float x[4];
                        load4(32 * h + d, x);
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const float u = x[e] * sc, v = x[e + 1] * sc;
                            qh[(d + e) / 2] = pack_h2(u, v);
                            const float2 b = unpack_h2(qh[(d + e) / 2]);
                            ql[(d + e) / 2] = pack_h2(u - b.x, v - b.y);
                        }
                    }
                    tmem_st16(q_tm + lane_tm + 16 * h, qh);
                    tmem_st16(q_tm + lane_tm + DP / 2 + 16 * h, ql);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
                m = -INFINITY;
                l = 0.f;
                // Row r sees key indexes i < hi with i >= lo or i < sinks.
                hi = c.keys;
                lo = 0;
                if (!p.prefix_pass) {
                    const int at = c.past + tok;
                    hi = min(hi, at + 1 - c.low + c.sink);
                    if (p.a.window) lo = max(at - p.a.window + 1 - c.low, 0) + c.sink;
                }
            }
            mbar_wait(&s_full[n & 1], (n >> 1) & 1, p.a.err, abort, kLimitNs);
            mbar_wait(&k_sc[n & 7], (n >> 3) & 1, p.a.err, abort, kLimitNs);
            tc_fence_after();
            const int i0 = c.tile * kKeys;
            // Rows past the tile's last hold zeros; they need no mask.
            const bool whole = i0 + kKeys <= hi && (i0 >= lo || i0 + kKeys <= p.a.sinks);
            const bool masked = __any_sync(0xffffffffu, !whole);
            const float f = qs * k_scale[n & 7];
            const uint32_t st = s_tm + (n & 1) * 128 + lane_tm;
            // Both passes over the row, with the mask only where a row needs it.
            float nm, a, sum = 0.f;
            auto row = [&](auto mask) {
                constexpr bool kMask = decltype(mask)::value;
                const int h0 = hi - i0, l0 = lo - i0, s0 = p.a.sinks - i0;
                float mx = -INFINITY;
#pragma unroll 1
                for (int h = 0; h < 4; h++) {
                    uint32_t x[32];
                    tmem_ld32_async(st + 32 * h, x);
                    tmem_wait_ld(x);
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const int i = 32 * h + j;
                        if (!kMask || (i < h0 && (i >= l0 || i < s0))) mx = fmaxf(mx, __uint_as_float(x[j]));
                    }
                }
                nm = fmaxf(m, mx == -INFINITY ? mx : mx * f);
                const float mu = nm == -INFINITY ? 0.f : nm - (float)kShift;
                a = m == -INFINITY ? 0.f : ex2(m - nm);
#pragma unroll 1
                for (int h = 0; h < 4; h++) {
                    uint32_t x[32], ph[16], pl[16];
                    tmem_ld32_async(st + 32 * h, x);
                    tmem_wait_ld(x);
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        float e[2];
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            const int i = 32 * h + 2 * j + y;
                            e[y] = ex2(fmaf(__uint_as_float(x[2 * j + y]), f, -mu));
                            if (kMask && !(i < h0 && (i >= l0 || i < s0))) e[y] = 0.f;
                        }
                        sum += e[0] + e[1];
                        ph[j] = pack_h2(e[0], e[1]);
                        const float2 b = unpack_h2(ph[j]);
                        pl[j] = pack_h2(e[0] - b.x, e[1] - b.y);
                    }
                    tmem_st16(st + 32 * h, ph);
                    tmem_st16(st + 32 * h + 16, pl);
                }
            };
            if (masked)
                row(std::true_type());
            else
                row(std::false_type());
            m = nm;
            l = fmaf(l, a, sum);
            alpha[(n & 3) * kM + r] = a;
            first = c.tile == c.tiles - 1;
            if (first || n == N - 1) {
                row_ml[((n & 3) * kM + r) * 2] = m == -INFINITY ? m : m - (float)kShift;
                row_ml[((n & 3) * kM + r) * 2 + 1] = l;
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&a_full[n & 3]);
                mbar_arrive(&p_full[n & 1]);
            }
            if (n + 1 < N) cursor_next(p, c);
        }
    } else if (warp < 8) {
        // ---- output -------------------------------------------------------
        const int r = threadIdx.x - 128, ow = warp - 4;
        const uint32_t lane_tm = (uint32_t)(ow * 32) << 16;
        float acc[DP];
        int seg = 0, seg_n = 0;
#pragma unroll
        for (int d = 0; d < DP; d++) acc[d] = 0.f;
        for (int n = 0; n < N; n++) {
            mbar_wait(&a_full[n & 3], (n >> 2) & 1, p.a.err, abort, kLimitNs);
            mbar_wait(&v_sc[n & 7], (n >> 3) & 1, p.a.err, abort, kLimitNs);
            mbar_wait(o_full, n & 1, p.a.err, abort, kLimitNs);
            tc_fence_after();
            const float a = alpha[(n & 3) * kM + r], vs = v_scale[n & 7];
            float m = row_ml[((n & 3) * kM + r) * 2], l = row_ml[((n & 3) * kM + r) * 2 + 1];
            const uint32_t ot = o_tm + lane_tm;
#pragma unroll
            for (int h = 0; h < DP / 16; h++) {
                float x[16];
                tmem_ld16(ot + 16 * h, x);
#pragma unroll
                for (int j = 0; j < 16; j++) acc[16 * h + j] = fmaf(acc[16 * h + j], a, x[j] * vs);
            }
            tc_fence_before();
            const bool seg_end = c.tile == c.tiles - 1;
            if (!seg_end && n + 1 < N) {
                __syncwarp();
                if (lane == 0) mbar_arrive(o_empty);
                cursor_next(p, c);
                continue;
            }
            // ---- end of this CTA's piece of the segment.
            const bool bad_tiles = poison[seg & 7] != 0;
            bar_sync(2, 128);
            if (r == 0) poison[seg & 7] = 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty);
            const bool live = r < c.rows;
            const int row = c.r0 + r, tok = row / G, at = c.past + tok;
            const size_t qrow = (size_t)(c.tok0 + tok) * H + c.kvh * G + (row - tok * G);
            bool bad = bad_tiles || !finite(l) || !(m < INFINITY);
#pragma unroll
            for (int d = 0; d < DP; d++) bad |= !finite(acc[d]);
            unsigned todo = __ballot_sync(0xffffffffu, bad && live);
            while (todo) {
                const int src = __ffs(todo) - 1;
                todo &= todo - 1;
                const size_t qr = __shfl_sync(0xffffffffu, (unsigned long long)qrow, src);
                const int rat = __shfl_sync(0xffffffffu, at, src);
                const int k0 = (c.tile - (n - seg_n)) * kKeys, k1 = min(c.keys, (c.tile + 1) * kKeys);
                float rm, rl, ro[DP / 32];
                plain_row<T, DP>(
                    p, p.a.q + qr * D, c.b, c.kvh, k0, k1,
                    [&](int i) {
                        const int pos = i < c.sink ? i : i - c.sink + c.low;
                        if (p.prefix_pass) return pos;
                        const bool sees =
                            pos <= rat && (!p.a.window || pos > rat - p.a.window || pos < p.a.sinks);
                        return sees ? pos : -1;
                    },
                    rm, rl, ro);
#pragma unroll
                for (int y = 0; y < DP / 32; y++) scratch[ow * DP + lane + 32 * y] = ro[y];
                __syncwarp();
                if (lane == src) {
                    m = rm;
                    l = rl;
#pragma unroll
                    for (int d = 0; d < DP; d++) acc[d] = scratch[ow * DP + d];
                }
                __syncwarp();
            }
            const long long a0 = u0 + n - c.tile, a1 = a0 + c.tiles;  // the segment's units
            bool write = true;
            if (a0 < u0 || a1 > u1) {
                const int c_first = (int)(((a0 + 1) * grid - 1) / U), c_last = (int)((a1 * grid - 1) / U);
                const size_t slot = 2 * blockIdx.x + (a0 >= u0 ? 1 : 0);
                float4 *po = reinterpret_cast<float4 *>(p.part_o) + slot * (DP / 4) * kM + r;
#pragma unroll
                for (int d = 0; d < DP / 4; d++)
                    po[d * kM] = make_float4(acc[4 * d], acc[4 * d + 1], acc[4 * d + 2], acc[4 * d + 3]);
                reinterpret_cast<float2 *>(p.part_ml)[slot * kM + r] = make_float2(m, l);
                bar_sync(2, 128);
                if (r == 0) {
                    __threadfence();
                    const unsigned ticket = atomicAdd(&p.a.tickets[c_first], 1u);
                    *last_s = ticket == (unsigned)(c_last - c_first);
                    if (*last_s) p.a.tickets[c_first] = 0u;
                    __threadfence();
                }
                bar_sync(2, 128);
                write = *last_s;
                bar_sync(2, 128);
                if (write) {
                    m = -INFINITY;
                    l = 0.f;
                    for (int x = 0; x <= c_last - c_first; x++) {
                        const size_t sl = x == 0 ? 2 * (size_t)c_first + 1 : 2 * (size_t)(c_first + x);
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p.part_ml) + sl * kM + r);
                        const float4 *pp = reinterpret_cast<const float4 *>(p.part_o) + sl * (DP / 4) * kM + r;
                        const float nm = fmaxf(m, ml.x), mu = nm == -INFINITY ? 0.f : nm;
                        const float f = x == 0 ? 0.f : ex2(m - mu), e = ex2(ml.x - mu);
                        l = fmaf(ml.y, e, l * f);
#pragma unroll
                        for (int d = 0; d < DP / 4; d++) {
                            const float4 v = __ldcg(pp + d * kM);
                            acc[4 * d] = fmaf(v.x, e, x == 0 ? 0.f : acc[4 * d] * f);
                            acc[4 * d + 1] = fmaf(v.y, e, x == 0 ? 0.f : acc[4 * d + 1] * f);
                            acc[4 * d + 2] = fmaf(v.z, e, x == 0 ? 0.f : acc[4 * d + 2] * f);
                            acc[4 * d + 3] = fmaf(v.w, e, x == 0 ? 0.f : acc[4 * d + 3] * f);
                        }
                        m = nm;
                    }
                }
            }
            if (write && live) {
                if (p.prefix_pass) {
                    float *dst = p.pre_o + qrow * D;
#pragma unroll
                    for (int d = 0; d < DP; d += 4)
                        if (d < D)
                            *reinterpret_cast<float4 *>(dst + d) =
                                make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]);
                    *reinterpret_cast<float2 *>(p.pre_ml + qrow * 2) = make_float2(m, l);
                } else {
                    float f = 1.f, e = 0.f;
                    const float *pre = p.pre_o ? p.pre_o + qrow * D : nullptr;
                    if (pre) {
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p.pre_ml) + qrow);
                        const float nm = fmaxf(m, ml.x), mu = nm == -INFINITY ? 0.f : nm;
                        f = ex2(m - mu);
                        e = ex2(ml.x - mu);
                        l = fmaf(ml.y, e, l * f);
                    }
                    float *dst = p.a.out + qrow * D;
                    const bool vec = aligned16(p.a.out);
#pragma unroll
                    for (int d = 0; d < DP; d += 4) {
                        if (d >= D) continue;
                        float4 o = make_float4(acc[d], acc[d + 1], acc[d + 2], acc[d + 3]);
                        if (pre) {
                            const float4 v = __ldcg(reinterpret_cast<const float4 *>(pre + d));
                            o.x = fmaf(v.x, e, o.x * f);
                            o.y = fmaf(v.y, e, o.y * f);
                            o.z = fmaf(v.z, e, o.z * f);
                            o.w = fmaf(v.w, e, o.w * f);
                        }
                        o.x = __fdiv_rn(o.x, l);
                        o.y = __fdiv_rn(o.y, l);
                        o.z = __fdiv_rn(o.z, l);
                        o.w = __fdiv_rn(o.w, l);
                        if (vec) {
                            *reinterpret_cast<float4 *>(dst + d) = o;
                        } else {
                            dst[d] = o.x;
                            dst[d + 1] = o.y;
                            dst[d + 2] = o.z;
                            dst[d + 3] = o.w;
                        }
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < DP; d++) acc[d] = 0.f;
            seg++;
            seg_n = n + 1;
            if (n + 1 < N) cursor_next(p, c);
        }
    } else if (warp < 15) {
        // ---- producers ----------------------------------------------------
        const int pw = warp - 8;
        // Load i of a warp covers rows (i kProducers + pw) kRpi + sub.
        const int sub = lane / C::kLpr, col = (lane % C::kLpr) * C::kEpl;  // row of a load, first dim
        // Where a row's 16 bytes land: in the operand's own place, or, for
        // pairs, in the row's bytes of the slot (hi and lo blocks) in order.
        auto raw_at = [&](int r) {
            const int ch = lane % C::kLpr;
            return C::kPair ? (uint32_t)((ch >> 3) * C::kBlockBytes + r * 128 + (ch & 7) * 16) : operand_at(r, col);
        };
        const long long row_bytes = (long long)D * (int)sizeof(T);
        // Operand j is K of tile 0, then K of tile (j + 1) / 2 (odd j) or V of
        // tile j / 2 - 1 (even j), while those tiles last: 2 N of them.
        const int total = 2 * N;
        auto is_v = [&](int j) { return j == total - 1 || (j > 0 && j % 2 == 0); };
        auto tile_of = [&](int j) { return j == total - 1 ? N - 1 : j == 0 ? 0 : j % 2 ? (j + 1) / 2 : j / 2 - 1; };
        // Rows that the lanes copy: of the tile whose keys come next, and of
        // the one before it, whose values follow.
        long long off_k = -1, off_v = -1;
        // Segments of the operands being converted, for the poison flags.
        Cursor cv = c;
        int seg_k = 0, seg_v = 0;
        auto copy = [&](int j) {
            const bool v = is_v(j);
            if (!v) {
                if (j) {
                    cursor_next(p, c);
                    off_v = off_k;
                }
                // Lane i kRpi + sub looks up the row that load i takes there.
                const int r = (lane / C::kRpi * kProducers + pw) * C::kRpi + lane % C::kRpi;
                const int i = c.tile * kKeys + r;
                off_k = -1;
                if (r < kKeys && i < c.keys)
                    off_k = paged_row(p.a.cache, p.a.batch, c.b, i < c.sink ? i : i - c.sink + c.low, p.a.err) +
                            c.kvh * row_bytes;
            }
            const long long mine = v ? (j == total - 1 ? off_k : off_v) : off_k;
            if (j >= S) mbar_wait(&empty[j % S], (j / S - 1) & 1, p.a.err, abort, kLimitNs);
            unsigned char *slot = ring + (j % S) * C::kTileBytes;
            const char *base = p.a.cache.base + (v ? p.a.cache.parity_stride : 0) + col * (int)sizeof(T);
#pragma unroll
            for (int i = 0; i < C::kLoads; i++) {
                const int r = (i * kProducers + pw) * C::kRpi + sub;
                const long long off = __shfl_sync(0xffffffffu, mine, i * C::kRpi + sub);
                const bool live = off >= 0 && col < D;
                if (r < kKeys) cp_async16_zfill(slot + raw_at(r), base + (live ? off : 0), live ? 16 : 0);
            }
        };
        auto convert = [&](int j) {
            const bool v = is_v(j);
            const int n = tile_of(j);
            unsigned char *slot = ring + (j % S) * C::kTileBytes;
            const uint32_t at = smem_addr(slot);
            int ex = kShift;  // the scale is 2^(kShift - ex)
            if (!C::kRaw) {
                // The tile's largest magnitude, over all producer warps.
                uint4 x[C::kLoads];
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < C::kLoads; i++) {
                    const int r = (i * kProducers + pw) * C::kRpi + sub;
                    x[i] = make_uint4(0, 0, 0, 0);
                    if (r < kKeys) x[i] = *reinterpret_cast<const uint4 *>(slot + raw_at(r));
                    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        if (C::kPair) {
                            top = max(top, w[y] & 0x7fffffffu);
                        } else {
                            top = max(top, (w[y] << 16) & 0x7fffffffu);
                            top = max(top, w[y] & 0x7fff0000u);
                        }
                    }
                }
                top = __reduce_max_sync(0xffffffffu, top);
                uint32_t *most = v ? v_max : k_max;
                if (lane == 0) atomicMax(&most[n & 3], top);
                bar_sync(1, kProducers * 32);  // also: every row of the slot has been read
                top = *reinterpret_cast<volatile uint32_t *>(&most[n & 3]);
                // Next used in two tiles; last read two tiles ago.
                if (threadIdx.x == 8 * 32) most[(n + 2) & 3] = 0;
                ex = scale_exponent(top);
                if (threadIdx.x == 8 * 32 && top >= 0x7f800000u) poison[(v ? seg_v : seg_k) & 7] = 1;
                const float sc = pow2(kShift - ex);
#pragma unroll
                for (int i = 0; i < C::kLoads; i++) {
                    const int r = (i * kProducers + pw) * C::kRpi + sub;
                    if (r >= kKeys) continue;
                    const uint32_t to = at + operand_at(r, col);
                    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                    if (C::kPair) {
                        const float a = __uint_as_float(w[0]) * sc, b = __uint_as_float(w[1]) * sc,
                                    d = __uint_as_float(w[2]) * sc, e = __uint_as_float(w[3]) * sc;
                        const uint32_t h0 = pack_h2(a, b), h1 = pack_h2(d, e);
                        const float2 f0 = unpack_h2(h0), f1 = unpack_h2(h1);
                        sts64(to, h0, h1);
                        sts64(to + C::kHalfBytes, pack_h2(a - f0.x, b - f0.y), pack_h2(d - f1.x, e - f1.y));
                    } else {
                        uint32_t h[4];
#pragma unroll
                        for (int y = 0; y < 4; y++)
                            h[y] = pack_h2(__uint_as_float(w[y] << 16) * sc, __uint_as_float(w[y] & 0xffff0000u) * sc);
                        sts128(to, make_uint4(h[0], h[1], h[2], h[3]));
                    }
                }
            }
            if (threadIdx.x == 8 * 32) {
                (v ? v_scale : k_scale)[n & 7] = pow2(ex - kShift);
                mbar_arrive(&(v ? v_sc : k_sc)[n & 7]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[j % S]);
        };
        for (int j = 0; j < total + C::kAhead; j++) {
            if (j < total) copy(j);
            cp_async_commit();
            const int k = j - C::kAhead;
            if (k < 0) continue;
            cp_async_wait<C::kAhead>();
            if (C::kRaw) {
                convert(k);
                continue;
            }
            if (!is_v(k) && k > 0) {
                seg_v = seg_k;  // the values that follow are of the tile before
                seg_k += cv.tile == cv.tiles - 1;
                cursor_next(p, cv);
            }
            if (k == total - 1) seg_v = seg_k;
            convert(k);
        }
    } else {
        // ---- MMA issue ----------------------------------------------------
        if (lane == 0) {
        const uint32_t ra = smem_addr(ring);
        int seg = 0, j = 0;  // j: the next operand
        bool first = true;
        auto slot_wait = [&] {
            mbar_wait(&full[j % S], (j / S) & 1, p.a.err, abort, kLimitNs);
            return ra + (j % S) * C::kTileBytes;
        };
        auto qk = [&](int n) {
            if (first) mbar_wait(q_full, seg++ & 1, p.a.err, abort, kLimitNs);
            const uint32_t kb = slot_wait();
            if (!*abort) {
                tc_fence_after();
                const uint32_t d = s_tm + (n & 1) * 128;
#pragma unroll
                for (int ks = 0; ks < DP / 16; ks++) {
                    const uint32_t off = (ks / 4) * C::kBlockBytes + (ks % 4) * 32;
                    const uint32_t qh = q_tm + ks * 8;
                    const uint64_t kh = sw128_desc(kb + off);
                    mma_ts(d, qh + DP / 2, kh, C::kIdescS, ks > 0);
                    if (C::kPair) mma_ts(d, qh, sw128_desc(kb + C::kHalfBytes + off), C::kIdescS, 1u);
                    mma_ts(d, qh, kh, C::kIdescS, 1u);
                }
                mma_commit(&empty[j % S]);
                mma_commit(&s_full[n & 1]);
            }
            j++;
            first = c.tile == c.tiles - 1;  // of the next tile
            if (n + 1 < N) cursor_next(p, c);
        };
        auto pv = [&](int n) {
            mbar_wait(&p_full[n & 1], (n >> 1) & 1, p.a.err, abort, kLimitNs);
            const uint32_t vb = slot_wait();
            if (n >= 1) mbar_wait(o_empty, (n - 1) & 1, p.a.err, abort, kLimitNs);
            if (!*abort) {
                tc_fence_after();
                const uint32_t pt = s_tm + (n & 1) * 128;
#pragma unroll
                for (int ks = 0; ks < kKeys / 16; ks++) {
                    const uint32_t ph = pt + (ks / 2) * 32 + (ks % 2) * 8;
                    const uint64_t vh = sw128_desc_mn(vb + ks * 2048, C::kBlockBytes);
                    mma_ts(o_tm, ph + 16, vh, C::kIdescO, ks > 0);
                    if (C::kPair)
                        mma_ts(o_tm, ph, sw128_desc_mn(vb + C::kHalfBytes + ks * 2048, C::kBlockBytes), C::kIdescO, 1u);
                    mma_ts(o_tm, ph, vh, C::kIdescO, 1u);
                }
                mma_commit(&empty[j % S]);
                mma_commit(o_full);
            }
            j++;
        };
        qk(0);
        for (int n = 0; n < N; n++) {
            if (n + 1 < N) qk(n + 1);
            pv(n);
        }
        // Every MMA issued must complete before TMEM is freed.
        mma_commit(done);
        drain_wait(done, 0);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 15) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

int padded_dim(int d) { return d <= 64 ? 64 : 128; }

template <typename T, int DP>
cudaError_t launch(cudaStream_t s, const PagedPass &p) {
    using C = Cfg<T, DP>;
    static_assert(C::kSmem <= 227 * 1024, "shared layout");
    static std::atomic<uint64_t> smem_set{0};
    cudaError_t e = set_smem_limit_once(paged_rows_kernel<T, DP>, C::kSmem, &smem_set);
    if (e != cudaSuccess) return e;
    // The register split above needs the launch to hold kLaunchRegs a thread.
    static const int regs = [] {
        cudaFuncAttributes at{};
        return cudaFuncGetAttributes(&at, paged_rows_kernel<T, DP>) == cudaSuccess ? at.numRegs : 0;
    }();
    if (regs < kLaunchRegs) return cudaErrorInvalidConfiguration;
    launch_k(paged_rows_kernel<T, DP>, kSmCount, kThreads, C::kSmem, s, p);
    count_launch();
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_dim(cudaStream_t s, const PagedPass &p) {
    return padded_dim(p.a.head_dim) == 64 ? launch<T, 64>(s, p) : launch<T, 128>(s, p);
}

}  // namespace

// Wider heads leave no room for Q, K and V tiles in shared memory.
bool paged_rows_supported(const PagedAttention &a) { return a.head_dim <= 128; }

size_t paged_rows_part_floats(const PagedAttention &a) {
    return (size_t)2 * kSmCount * kM * (padded_dim(a.head_dim) + 2);
}

// part_o [2 * grid][DP / 4][kM] float4, part_ml [2 * grid][kM] float2.
cudaError_t paged_rows(cudaStream_t s, const PagedPass &pass) {
    PagedPass p = pass;
    p.part_ml = p.part_o + (size_t)2 * kSmCount * kM * padded_dim(p.a.head_dim);
    switch (p.a.cache.type) {
    case kPagedF16: return launch_dim<__half>(s, p);
    case kPagedBf16: return launch_dim<__nv_bfloat16>(s, p);
    default: return launch_dim<float>(s, p);
    }
}

}  // namespace k
}  // namespace slc
