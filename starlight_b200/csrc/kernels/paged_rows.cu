// Attention over a paged KV cache for many query rows: prompts, and the rows
// of a whole batch against the prefix that its sequences share. The same
// definition and work line as paged_attention.cu; a segment is (sequence, 128
// query rows, kv head), a tile 128 keys, and the products run on tcgen05.
//
// Arithmetic. kind::f16 with f32 accumulators on pairs of f16: x = hi + lo
// keeps 22 bits, down to a step of 2^-24 where f16 ends, given scales (powers
// of two, exact): of a query row, whose largest value comes to [2^14, 2^15); of
// a key, whose largest comes to [2^3, 2^15); of a value channel (a dim) in a
// tile, whose largest comes to [2, 2^15). So an element is off by at most 2^-22
// of itself or 2^-39 of the row's, 2^-28 of the key's, 2^-26 of the channel's
// largest. Probabilities are taken 2^14 times as large for the same reason.
// Keys share a scale within a tile and channels keep theirs from tile to tile
// as long as those ranges hold, so most tiles are converted once, with scales
// known beforehand, and the output is held in units of the channels' scales. An
// F32 cache needs three products (lo hi, hi lo, hi hi) for S = Q K^T and for
// P V; F16 values are taken as they are and BF16 values are one f16 each, two
// products. Every tile's P V starts from zero and is added in f32 registers
// (TMEM accumulation over thousands of keys would truncate thousands of times).
//
// Infinities and NaN. A key's reach S by themselves; a score that they make NaN
// is taken once more from the cache, for it may be -infinity, and its row goes
// on without it. A value's are taken out of the operand, where they would reach
// the rows that do not see them, and put into the results at the segment's end.
// What is done twice is the conversion of their tiles, one product for every
// such score, and a look through the values between a segment's first such tile
// and its last.
//
// One CTA per SM, 20 warps:
//   0..3   softmax: one thread per row; Q of a segment to TMEM as f16 pairs;
//          S from TMEM, running maximum, P as f16 pairs back into the TMEM
//          columns that S held (16-bit caches: with warps 8..11, two threads
//          per row, each half of the keys)
//   4..7   output: one thread per row; O += P V of each tile in registers,
//          the result, or this CTA's piece of a split segment
//   8..15  (16-bit caches: 12..15) conversion in place: scale, f16 or f16
//          pair, zeros in rows that no query sees (they may hold anything).
//          Keys or values that the scales at hand do not suit are read from the
//          cache once more (a pass over each tile for its maxima would cost a
//          quarter of the shared memory's bandwidth, which is what bounds an
//          F32 cache).
//   16     issues the MMAs: Q K^T of the next tile before P V of this one
//   17     copies: TMA boxes of 8 to 128 keys of a page and 128 bytes into a
//          ring of slots (pages that are not a multiple of 8 keys: 16-byte
//          asynchronous copies, by warps 17..19)
// The ring holds operands in the order K0 K1 V0 K2 V1 ..., so a slot is free
// as soon as the MMAs kSlots back are done; three slots of pairs or six of
// single f16. Q and P are A operands from TMEM; K is read K-major and V
// MN-major from the same layout ([key][64 dims] rows of 128 bytes, 128-byte
// swizzle). TMEM: Q, two S / P buffers and O, 128 columns each.
//
// Bound: 4 * pairs * D flops take 4 (16-bit cache) or 6 (F32) passes of half as
// many MMA flops each: 2048 cycles a tile, 3/2 of that for F32. Two prompts of
// 2048 tokens, 32 heads of 128, window 4096 (254 GFLOP), three sets of inputs in
// turn: f32 943 us, some 8300 cycles a tile (conversion and the MMAs share the
// shared memory; the tensor pipe is active for 37 %), bf16 817 us (29 %: four
// warps convert), f16 552 us, some 4900 (43 %: the softmax warps' chain of TMEM
// reads, exponentials and splits). The roles' code is more than the instruction
// caches hold: each of the rare ways below costs 1 to 3 % of an f32 prompt's time
// where it is never taken.
#include <float.h>
#include <limits.h>
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
constexpr int kCopy = 3;    // copying warps where TMA boxes do not fit the pages
constexpr int kThreads = 20 * 32;
constexpr int kShift = 14;  // a query row's largest value in [2^14, 2^15), probabilities up to 2^14
constexpr int kTop = 11;    // a scale takes the largest value to 2^11 and serves from 2^1 to 2^15
constexpr int kFirst = 2;   // exponent expected at first
constexpr int kNear = 8;    // keys down to 2^-8 of the expected largest value share its scale
constexpr float kLarge = 4194304.f;  // 2^22
constexpr int kDeep = 60;   // octaves that a channel's scale may fall within a segment
constexpr int kLaunchRegs = 96;  // registers a thread at launch
template <typename T, int DP>
struct Cfg {
    static constexpr bool kPair = sizeof(T) == 4;            // keys and values are f16 pairs
    static constexpr bool kRaw = std::is_same<T, __half>::value;  // taken as they are
    static constexpr int kBlocks = DP / 64;                  // 128-byte blocks along the dims
    static constexpr int kBlockBytes = kKeys * 128;          // 16 KiB
    static constexpr int kHalfBytes = kBlocks * kBlockBytes;  // one of hi, lo
    static constexpr int kTileBytes = kHalfBytes * (kPair ? 2 : 1);
    static constexpr int kSlots = kPair && DP == 128 ? 3 : 6;
    static constexpr int kAhead = kSlots / 2;                // asynchronous copies: operands in flight
    static constexpr int kRing = kSlots * kTileBytes;
    static constexpr int kSmall = 4 * (22 * kM + 8 * kKeys + 18 * DP + 96 + 8 * 12 + 16 + 2 * DP / 32 * kM) +
                                  8 * (3 * kKeys + 8 + 3 * kSlots + 8 + 20);
    static constexpr int kSmem = 1024 + kRing + kSmall;
    static constexpr int kEpl = 16 / (int)sizeof(T);    // elements of a 16-byte load
    static constexpr int kLpr = DP / kEpl;               // lanes per cache row
    static constexpr int kRpi = 32 / kLpr;               // rows per warp load
    // An F32 cache keeps eight warps converting; 16-bit ones leave four of
    // them to a second softmax warpgroup, each with half the keys of a tile.
    static constexpr int kSoft = kPair ? 1 : 2;
    static constexpr int kConv = kPair ? 8 : 4;
    static constexpr int kConvWarp = 16 - kConv;
    static constexpr int kRows = kKeys / kConv / kRpi;   // 16-byte pieces per conversion lane
    // Registers a thread, by warpgroup, out of those of the launch.
    static constexpr int kSoftRegs = kPair ? 96 : 88, kOutRegs = kPair ? 200 : 192, kConvRegs = kPair ? 64 : 56,
                         kRestRegs = 56;
    static_assert(kSoft * kSoftRegs + kOutRegs + kConv / 4 * kConvRegs + kRestRegs <= 5 * kLaunchRegs, "registers");
    // f32 accumulators, f16 operands, K-major A; B K-major (S) or MN-major (O).
    static constexpr uint32_t kIdescS = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
    static constexpr uint32_t kIdescO =
        (1u << 4) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(kM >> 4) << 24);
};

struct RowsArgs {
    PagedPass pass;
    CUtensorMap map;
    int unit;  // keys per box (paged_boxes); 1: no boxes
    int join;  // split segments are merged by rows_join_kernel
    uint64_t limit;  // of a wait, ns: the output warps may look through a segment's values (odd_values)
};
constexpr uint64_t kLimitNs = 1000000000ull, kLimitKeyNs = 500;  // a key took them 150 ns

// Where a segment has values that are not finite: key indexes [from, to) of
// whole tiles.
struct OddKeys {
    int from, to;
};

// A segment of the work line and a place in it. Key indexes run over
// positions [0, sink) and from `low` on, both widened to whole boxes; the
// positions that some row sees are those below `sinks` and from `from` on.
struct Cursor {
    int b, rt, kvh, tile;  // sequence, row tile, kv head, key tile
    int tok0, ntok, past;  // of the sequence
    int r0, rows;          // of the row tile
    int sink, low, from, keys, tiles;
};

__device__ __forceinline__ int group_of(const PagedPass &p) { return p.a.heads / p.a.kv_heads; }
__device__ __forceinline__ int seq_count(const PagedPass &p) { return p.prefix_pass ? 1 : p.a.batch.seqs; }

__device__ __forceinline__ void seq_load(const PagedPass &p, int b, Cursor &c) {
    c.b = b;
    if (p.prefix_pass) {
        // The first with tokens: its table row. Mostly sequence 0: one read
        // instead of a chain of them.
        c.b = p.a.batch.starts[1] ? 0 : paged_sequence_of(p.a.batch, 0);
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
__device__ __forceinline__ void row_tile_load(const PagedPass &p, int unit, Cursor &c) {
    const int G = group_of(p);
    c.r0 = c.rt * kM;
    c.rows = min(kM, c.ntok * G - c.r0);
    c.sink = 0;
    c.from = p.first;
    c.low = p.first - p.first % unit;
    if (p.prefix_pass) {
        c.keys = p.a.prefix;
    } else {
        const int first = c.past + c.r0 / G, last = c.past + (c.r0 + c.rows - 1) / G;
        if (p.a.window) {
            c.from = max(first + 1 - p.a.window, 0);
            c.low = c.from - c.from % unit;
            const int sinks = min(p.a.sinks, c.from);
            c.sink = (sinks + unit - 1) / unit * unit;
            if (c.sink >= c.low) c.sink = c.low = 0;
        }
        c.keys = c.sink + last + 1 - c.low;
    }
    c.tiles = (c.keys + kKeys - 1) / kKeys;
}
// Places the cursor on unit `at` of the line counted from row tile c.rt of
// sequence c.b.
__device__ __forceinline__ void cursor_at(const PagedPass &p, int unit, Cursor &c, long long at) {
    for (;;) {
        const int rts = row_tiles(p, c);
        for (; c.rt < rts; c.rt++) {
            row_tile_load(p, unit, c);
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
        c.rt = 0;
    }
}
// The next unit; the line's end is the caller's to know.
__device__ __forceinline__ void cursor_next(const PagedPass &p, int unit, Cursor &c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.kvh < p.a.kv_heads) return;
    c.kvh = 0;
    if (++c.rt < row_tiles(p, c)) {
        row_tile_load(p, unit, c);
        return;
    }
    if (p.prefix_pass || c.b + 1 >= p.a.batch.seqs) return;
    seq_load(p, c.b + 1, c);
    c.rt = 0;
    cursor_at(p, unit, c, 0);
}

// The work line, added up by the first kM threads, each over a run of it: an
// equal share of a sequence's row tiles, or several sequences. (A thread per
// sequence took 14 us for two of 64 row tiles.)
struct Line {
    long long mine, upto;  // of this thread's run; up to its end
    long long total;
    int parts, per;  // runs per sequence, sequences per run
};
// The first row tile of a run and how many it has of that sequence (-1: the
// run is whole sequences).
__device__ __forceinline__ int run_start(const PagedPass &p, const Line &x, int run, Cursor &c) {
    seq_load(p, run / x.parts * x.per, c);
    c.rt = 0;
    if (x.parts == 1) return -1;
    const int rts = row_tiles(p, c), part = run % x.parts;
    c.rt = (int)((long long)rts * part / x.parts);
    return (int)((long long)rts * (part + 1) / x.parts) - c.rt;
}
// Every thread of the CTA calls it; sums: 6 words shared.
__device__ __forceinline__ Line line_scan(const PagedPass &p, int unit, long long *sums) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, seqs = seq_count(p);
    Line x;
    x.mine = x.upto = x.total = 0;
    x.parts = max(kM / seqs, 1);
    x.per = (seqs + kM - 1) / kM;
    if (warp < 4) {
        const int first = (int)threadIdx.x / x.parts * x.per;
        for (int b = first; b < min(first + x.per, seqs); b++) {
            Cursor c;
            int n = -1;
            if (b == first)
                n = run_start(p, x, threadIdx.x, c);
            else
                seq_load(p, b, c), c.rt = 0;
            const int end = n < 0 ? row_tiles(p, c) : c.rt + n;
            for (; c.rt < end; c.rt++) {
                row_tile_load(p, unit, c);
                x.mine += (long long)c.tiles * p.a.kv_heads;
            }
        }
        x.upto = x.mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x.upto, o);
            if (lane >= o) x.upto += y;
        }
        if (lane == 31) sums[warp] = x.upto;
    }
    __syncthreads();
    for (int w = 0; w < 4; w++) {
        if (w < warp) x.upto += sums[w];
        x.total += sums[w];
    }
    return x;
}
// The thread whose run holds unit u leaves where that begins; after a barrier
// line_place sets the cursor there.
__device__ __forceinline__ void line_find(const Line &x, long long u, long long *sums) {
    if (threadIdx.x < kM && x.upto - x.mine <= u && u < x.upto) {
        sums[4] = threadIdx.x;
        sums[5] = x.upto - x.mine;
    }
}
__device__ __forceinline__ void line_place(const PagedPass &p, int unit, const Line &x, long long u,
                                           const long long *sums, Cursor &c) {
    run_start(p, x, (int)sums[4], c);
    cursor_at(p, unit, c, u - sums[5]);
}

// Position of key index i.
__device__ __forceinline__ int key_pos(const Cursor &c, int i) { return i < c.sink ? i : i - c.sink + c.low; }
// What the copying warp tells the others of a tile.
struct Tile {
    int begins, whole;  // first of a segment; every key index is seen by some row
    int seg;            // its segment, counted from this CTA's first
    int b, kvh, i0;
    int sink, low, from, keys;
};

// Called by a whole warp, issued by one lane (always the same).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "elect.sync _|q, 0xffffffff;\n"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void commit_one(uint64_t *bar) {
    asm volatile(
        "{\n"
        ".reg .pred q;\n"
        "elect.sync _|q, 0xffffffff;\n"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
        "}\n" ::"r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void bar_sync(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// The same, and whether some thread passes true.
__device__ __forceinline__ bool bar_or(int id, int threads, bool x) {
    uint32_t any;
    asm volatile(
        "{\n"
        ".reg .pred p, q;\n"
        "setp.ne.u32 p, %3, 0;\n"
        "barrier.red.or.pred q, %1, %2, p;\n"
        "selp.u32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(any)
        : "r"(id), "r"(threads), "r"((uint32_t)x)
        : "memory");
    return any != 0;
}
// (a, b) as an f16 pair, a low; and the value that it holds.
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 unpack_h2(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
}
// Two f32 operations at a time.
struct F2 {
    uint64_t v;
    __device__ __forceinline__ F2() {}
    __device__ __forceinline__ F2(float a, float b) {
        asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    }
    __device__ __forceinline__ float2 get() const {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
// An f16 pair of x, and of what it leaves.
__device__ __forceinline__ void split2(F2 x, uint32_t &hi, uint32_t &lo) {
    const float2 f = x.get();
    hi = pack_h2(f.x, f.y);
    const float2 b = unpack_h2(hi);
    const float2 r = fma2(F2(b.x, b.y), F2(-1.f, -1.f), x).get();
    lo = pack_h2(r.x, r.y);
}

// Element (row, dim) of a swizzled operand: block dim / 64 of rows of 128
// bytes, 16-byte chunks xored with the row.
__device__ __forceinline__ uint32_t operand_at(int row, int dim) {
    return (uint32_t)((dim >> 6) * kKeys * 128 + row * 128 + ((((dim & 63) >> 3) ^ (row & 7)) << 4) + (dim & 7) * 2);
}

// Of a tile of keys: what takes its scale out of S; a byte for each conversion
// warp, whether keys of its have scales of their own.
struct KeyTile {
    float scale;
    uint32_t none;
    unsigned char own[8];
};
// a / b of powers of two, from 2^-126 to 2^127.
__device__ __forceinline__ float ratio2(float a, float b) {
    return pow2(min(max((int)(__float_as_uint(a) >> 23) - (int)(__float_as_uint(b) >> 23), -126), 127));
}

// Cache values to operands: a conversion lane's 16 raw bytes at a time, of
// row (i kConv + warp) kRpi + sub, from dim `col` on.
template <typename T, int DP>
struct Operand {
    using C = Cfg<T, DP>;
    static constexpr int kStep = C::kConv * C::kRpi * 128;
    // To f16, or f16 pairs, with a scale for each element.
    __device__ static __forceinline__ void convert(uint4 x, const F2 (&sc)[C::kEpl / 2], uint32_t dst) {
        if constexpr (C::kPair) {
            uint32_t h0, h1, l0, l1;
            split2(mul2(F2(__uint_as_float(x.x), __uint_as_float(x.y)), sc[0]), h0, l0);
            split2(mul2(F2(__uint_as_float(x.z), __uint_as_float(x.w)), sc[1]), h1, l1);
            sts64(dst, h0, h1);
            sts64(dst + C::kHalfBytes, l0, l1);
        } else if constexpr (!C::kRaw) {
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            uint32_t h[4];
#pragma unroll
            for (int z = 0; z < 4; z++) {
                const float2 f = mul2(F2(__uint_as_float(w[z] << 16), __uint_as_float(w[z] & 0xffff0000u)), sc[z]).get();
                h[z] = pack_h2(f.x, f.y);
            }
            sts128(dst, make_uint4(h[0], h[1], h[2], h[3]));
        }
    }
    // Magnitudes as bits, by word: one of f32 or two of 16 bits.
    __device__ static __forceinline__ uint32_t size_of(uint32_t w) {
        return w & (C::kPair ? 0x7fffffffu : 0x7fff7fffu);
    }
    __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        return C::kPair ? max(a, b) : __vmaxu2(a, b);
    }
    // Takes what is not finite out of 16 bytes; whether there was any.
    __device__ static __forceinline__ bool clean(uint4 &x) {
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
        bool any = false;
#pragma unroll
        for (int z = 0; z < 4; z++) {
            if constexpr (C::kPair) {
                if (size_of(w[z]) >= 0x7f800000u) any = true, w[z] = 0;
            } else {
                constexpr uint32_t kInf = C::kRaw ? 0x7c00u : 0x7f80u;
                if ((size_of(w[z]) & 0xffffu) >= kInf) any = true, w[z] &= 0xffff0000u;
                if (size_of(w[z]) >> 16 >= kInf) any = true, w[z] &= 0xffffu;
            }
        }
        x = make_uint4(w[0], w[1], w[2], w[3]);
        return any;
    }
    // The largest magnitude of 16 bytes, as the bits of an f32.
    __device__ static __forceinline__ uint32_t largest(uint4 x) {
        const uint32_t t = larger(larger(size_of(x.x), size_of(x.y)), larger(size_of(x.z), size_of(x.w)));
        return C::kPair ? t : max(t << 16, t & 0xffff0000u);
    }
    // The scale of an operand's channel, from what takes it out of the outputs.
    __device__ static __forceinline__ float inverse(float x) { return ratio2(pow2(-kShift), x); }
    // 16 bytes of the tile's keys or values from the cache; zeros where no row sees them.
    __device__ static __forceinline__ uint4 fetch(const PagedPass &p, const Tile &cu, int row, int col, bool v) {
        const int key = cu.i0 + row, pos = key < cu.sink ? key : key - cu.sink + cu.low, D = p.a.head_dim;
        if (!live_key(p, cu, key) || col >= D) return make_uint4(0, 0, 0, 0);
        return __ldcg(reinterpret_cast<const uint4 *>(
            p.a.cache.base + paged_row(p.a.cache, p.a.batch, cu.b, pos, p.a.err) + (v ? p.a.cache.parity_stride : 0) +
            (cu.kvh * D + col) * (long long)sizeof(T)));
    }
};

// The rare ways of the conversion and of the softmax, behind branches marked as
// unlikely: what is not executed costs as well, in instruction fetches. They
// are part of their roles' code, not calls, so that each keeps to the registers
// that its role has given itself.
//
// A conversion warp's keys from the cache again: those outside 2^-kNear to 2^3
// of the expected largest value get a scale of their own, from their own.
template <typename T, int DP>
__device__ __forceinline__ void keys_again(const PagedPass &p, const Tile &cu, uint32_t to, int expect, float *rel) {
    using C = Cfg<T, DP>;
    using O = Operand<T, DP>;
    const int lane = threadIdx.x & 31, pw = (threadIdx.x >> 5) - C::kConvWarp;
    const int sub = lane / C::kLpr, ch = lane % C::kLpr, col = ch * C::kEpl;
#pragma unroll 1
    for (int i = 0; i < C::kRows; i++) {
        const int row = (i * C::kConv + pw) * C::kRpi + sub;
        const uint4 x = O::fetch(p, cu, row, col, false);
        uint32_t t = O::largest(x);
#pragma unroll 1
        for (int o = 1; o < C::kLpr; o <<= 1) t = max(t, __shfl_xor_sync(0xffffffffu, t, o));
        int ex = t ? scale_exponent(t) : expect;
        if (ex >= expect - kNear && ex <= expect + 3) ex = expect;
        const float f = pow2(kTop - ex);
        F2 sc[C::kEpl / 2];
#pragma unroll
        for (int e = 0; e < C::kEpl / 2; e++) sc[e] = F2(f, f);
        O::convert(x, sc, to + i * O::kStep);
        if (ch == 0) rel[row] = pow2(min(max(ex - expect, -126), 127));
    }
}
// S's columns of keys with scales of their own.
template <typename T, int DP>
__device__ __forceinline__ void rescale_scores(uint32_t st, int first, const KeyTile *tile, const float *rel) {
    using C = Cfg<T, DP>;
#pragma unroll 1
    for (int i = first; i < first + kKeys / C::kSoft; i++)
        if (tile->own[i / C::kRpi % C::kConv])
            tmem_st1(st + i, __float_as_uint(__uint_as_float(tmem_ld1(st + i)) * rel[i]));
    tmem_wait_st();
}
// S less a number of the row.
template <typename T, int DP>
__device__ __forceinline__ void shift_scores(uint32_t st, int first, float by) {
    for (int i = first; i < first + kKeys / Cfg<T, DP>::kSoft; i++)
        tmem_st1(st + i, __float_as_uint(__uint_as_float(tmem_ld1(st + i)) - by));
    tmem_wait_st();
}
__device__ __forceinline__ void note_odd(OddKeys *odd, int i0) {
    atomicMin(&odd->from, i0);
    atomicMax(&odd->to, i0 + kKeys);
}
// All conversion warps' values of a tile from the cache again, with new scales
// from the tile's own largest values. `now` takes them out of the outputs, as
// `was` did. A scale falls by at most kDeep octaves within a segment, whose
// outputs so far are held in units of it.
template <typename T, int DP>
__device__ __forceinline__ void values_again(const PagedPass &p, const Tile &cu, uint32_t to, uint32_t *most, int *high,
                                          int *high_seg, const float *was, float *now, OddKeys *odd) {
    using C = Cfg<T, DP>;
    using O = Operand<T, DP>;
    const int lane = threadIdx.x & 31, pw = (threadIdx.x >> 5) - C::kConvWarp, ct = threadIdx.x - C::kConvWarp * 32;
    const int sub = lane / C::kLpr, ch = lane % C::kLpr, col = ch * C::kEpl;
    uint32_t top[C::kEpl];
#pragma unroll
    for (int e = 0; e < C::kEpl; e++) top[e] = 0;
#pragma unroll 1
    for (int i = 0; i < C::kRows; i++) {
        const uint4 x = O::fetch(p, cu, (i * C::kConv + pw) * C::kRpi + sub, col, true);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < C::kEpl; e++) {
            const uint32_t a = O::size_of(w[C::kPair ? e % 4 : e / 2 % 4]);
            const uint32_t t = C::kPair ? a : e % 2 ? a & 0xffff0000u : a << 16;
            if (t < 0x7f800000u) top[e] = max(top[e], t);
        }
    }
#pragma unroll
    for (int e = 0; e < C::kEpl; e++) {
#pragma unroll 1
        for (int o = C::kLpr; o < 32; o <<= 1) top[e] = max(top[e], __shfl_xor_sync(0xffffffffu, top[e], o));
        if (sub == 0) most[pw * DP + col + e] = top[e];
    }
    bar_sync(1, C::kConv * 32);
    if (ct < DP) {
        uint32_t t = 0;
#pragma unroll 1
        for (int w = 0; w < C::kConv; w++) t = max(t, most[w * DP + ct]);
        const int before = (int)(__float_as_uint(was[ct]) >> 23) - 127 + kTop + kShift;
        const int held = cu.begins ? -kDeep - 100 : *high_seg == cu.seg ? max(high[ct], before) : before;
        const int ex = max(t ? scale_exponent(t) : before, held - kDeep);
        now[ct] = pow2(ex - kTop - kShift);
        high[ct] = max(ex, held);
    }
    bar_sync(1, C::kConv * 32);
    if (ct == 0) *high_seg = cu.seg;
    F2 sc[C::kEpl / 2];
#pragma unroll
    for (int e = 0; e < C::kEpl / 2; e++) sc[e] = F2(O::inverse(now[col + 2 * e]), O::inverse(now[col + 2 * e + 1]));
#pragma unroll 1
    for (int i = 0; i < C::kRows; i++) {
        uint4 x = O::fetch(p, cu, (i * C::kConv + pw) * C::kRpi + sub, col, true);
        if (O::clean(x)) note_odd(odd, cu.i0);
        O::convert(x, sc, to + i * O::kStep);
    }
}
// A conversion lane's part of a tile of F16 values, which is otherwise taken
// as it is, cleaned.
template <typename T, int DP>
__device__ __forceinline__ void clean_values(unsigned char *at, int i0, OddKeys *odd) {
    for (int i = 0; i < Cfg<T, DP>::kRows; i++) {
        uint4 x = *reinterpret_cast<const uint4 *>(at + i * Operand<T, DP>::kStep);
        if (!Operand<T, DP>::clean(x)) continue;
        *reinterpret_cast<uint4 *>(at + i * Operand<T, DP>::kStep) = x;
        note_odd(odd, i0);
    }
}
// The values that are not finite, zero in the operand, into the results of a
// piece of a segment: four warps look through the keys [k0, k1) once more and
// note for every dim which rows see a +infinity and which a -infinity (a NaN is
// both); then thread r puts them into row r's result, dim d at
// dst[d / 4 * step + d % 4]. bits: zero, and left so.
template <typename T, int DP>
__device__ __noinline__ void odd_values(const PagedPass &p, Cursor c, int k0, int k1, float *dst, int step, bool live,
                                        uint32_t *bits) {
    using C = Cfg<T, DP>;
    constexpr int kFly = 4, kWords = kM / 32;
    const int r = threadIdx.x & (kM - 1), warp = r >> 5, lane = r & 31, D = p.a.head_dim, G = group_of(p);
    const int col = lane % C::kLpr * C::kEpl;
    const char *base = p.a.cache.base + p.a.cache.parity_stride + (c.kvh * D + col) * (long long)sizeof(T);
    for (int i0 = k0 + warp * C::kRpi + lane / C::kLpr; __any_sync(0xffffffffu, i0 < k1); i0 += 4 * C::kRpi * kFly) {
        uint4 x[kFly];
#pragma unroll
        for (int y = 0; y < kFly; y++) {
            const int i = i0 + y * 4 * C::kRpi, pos = i < c.sink ? i : i - c.sink + c.low;
            x[y] = make_uint4(0, 0, 0, 0);
            if (i < k1 && col < D)
                x[y] = __ldcg(
                    reinterpret_cast<const uint4 *>(base + paged_row(p.a.cache, p.a.batch, c.b, pos, p.a.err)));
        }
#pragma unroll 1
        for (int y = 0; y < kFly; y++) {
            uint4 kept = x[y];
            if (!Operand<T, DP>::clean(kept)) continue;
            const int i = i0 + y * 4 * C::kRpi, pos = i < c.sink ? i : i - c.sink + c.low;
            // Rows [from, to) see the key.
            long long from = 0, to = c.rows;
            if (!p.prefix_pass) {
                if (pos < p.first || (pos < c.from && pos >= p.a.sinks)) continue;
                from = max((long long)(pos - c.past) * G - c.r0, 0ll);
                if (p.a.window && pos >= p.a.sinks)
                    to = min((((long long)pos + p.a.window) - c.past) * G - c.r0, to);
            }
            float v[C::kEpl];
            Frag<T>::ld(&x[y], v);
#pragma unroll 1
            for (int w = 0; w < kWords; w++) {
                const int lo = (int)max(from - 32 * w, 0ll), hi = (int)min(to - 32 * w, 32ll);
                if (lo >= hi) continue;
                const uint32_t rows = (0xffffffffu >> (32 - hi)) & (0xffffffffu << lo);
#pragma unroll
                for (int e = 0; e < C::kEpl; e++) {
                    if (finite(v[e])) continue;
                    uint32_t *word = bits + (col + e) * kWords + w;
                    if (!(v[e] < 0.f) && (*word & rows) != rows) atomicOr(word, rows);
                    if (!(v[e] > 0.f) && (word[DP * kWords] & rows) != rows) atomicOr(word + DP * kWords, rows);
                }
            }
        }
    }
    __syncwarp();
    bar_sync(2, kM);
    for (int d = 0; d < D; d++) {
        const uint32_t plus = bits[d * kWords + warp] >> lane & 1, minus = bits[(DP + d) * kWords + warp] >> lane & 1;
        if (!live || !(plus | minus)) continue;
        float &o = dst[(size_t)(d / 4) * step + d % 4];
        o = (plus ? INFINITY : 0.f) - (minus ? INFINITY : 0.f) + o;
    }
    bar_sync(2, kM);
    for (int i = r; i < 2 * DP * kWords; i += kM) bits[i] = 0;
    bar_sync(2, kM);
}
// S's columns that the row does not see, all but i < hi with i >= lo or
// i < sinks, to -infinity.
template <typename T, int DP>
__device__ __forceinline__ void mask_scores(uint32_t st, int first, int hi, int lo, int sinks) {
#pragma unroll 1
    for (int i = first; i < first + kKeys / Cfg<T, DP>::kSoft; i += 16) {
        float s[16];
        uint32_t x[16];
        tmem_ld16(st + i, s);
#pragma unroll
        for (int j = 0; j < 16; j++)
            x[j] = __float_as_uint(i + j < hi && (i + j >= lo || i + j < sinks) ? s[j] : -INFINITY);
        tmem_st16(st + i, x);
    }
    tmem_wait_st();
}
// The scores of row q against the tile's keys that came out NaN though the row
// holds none and is not NaN yet (alive): a key with an infinity has a score of
// +-infinity, or NaN after all. Takes those from the cache, in f32. Columns
// first .. first + kKeys / kSoft of S. Returns the row's largest.
template <typename T, int DP>
__device__ __forceinline__ float repair_scores(const PagedPass &p, uint32_t st, int first, const float *q, int b, int kvh,
                                               int i0, int sink, int low, bool alive) {
    using C = Cfg<T, DP>;
    const int D = p.a.head_dim;
    const float sign = p.scale_log2 < 0.f ? -1.f : 1.f;
    float mx = -INFINITY;
    for (int i = first; i < first + kKeys / C::kSoft; i++) {
        float x = __uint_as_float(tmem_ld1(st + i));
        const bool wrong = alive && x != x;
        if (__any_sync(0xffffffffu, wrong)) {
            if (wrong) {
                const int key = i0 + i, pos = key < sink ? key : key - sink + low;
                const char *src = p.a.cache.base + paged_row(p.a.cache, p.a.batch, b, pos, p.a.err) +
                                  (long long)kvh * D * (int)sizeof(T);
                x = 0.f;
#pragma unroll 4
                for (int d = 0; d < D; d++) x = fmaf(q[d] * sign, Frag<T>::get(src + d * (int)sizeof(T)), x);
                alive = x == x;
            }
            __syncwarp();
            tmem_st1(st + i, __float_as_uint(x));
        }
        mx = fmaxf(mx, x);
    }
    tmem_wait_st();
    return mx;
}

// Where a row's result goes: (o f + prefix o e) / l to the output, or for a
// prefix pass o, m and l to where the next pass reads them.
struct RowEnd {
    float *dst;
    const float *pre;
    float l, f, e;
    bool vec;  // dst is aligned for 16 bytes
};
__device__ __forceinline__ RowEnd row_end(const PagedPass &p, size_t qrow, float m, float l) {
    const size_t at = qrow * p.a.head_dim;
    if (p.prefix_pass) {
        *reinterpret_cast<float2 *>(p.pre_ml + qrow * 2) = make_float2(m, l);
        return {p.pre_o + at, nullptr, 1.f, 1.f, 0.f, true};
    }
    RowEnd x{p.a.out + at, nullptr, l, 1.f, 0.f, aligned16(p.a.out)};
    if (p.pre_o) {
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p.pre_ml) + qrow);
        const float nm = fmaxf(m, ml.x), mu = nm == -INFINITY ? 0.f : nm;
        x.pre = p.pre_o + at;
        x.f = ex2(m - mu);
        x.e = ex2(ml.x - mu);
        x.l = fmaf(ml.y, x.e, l * x.f);
    }
    return x;
}
__device__ __forceinline__ void row_store(const RowEnd &x, int d, float4 o) {
    if (x.pre) {
        const float4 v = __ldcg(reinterpret_cast<const float4 *>(x.pre + d));
        o.x = fmaf(v.x, x.e, o.x * x.f);
        o.y = fmaf(v.y, x.e, o.y * x.f);
        o.z = fmaf(v.z, x.e, o.z * x.f);
        o.w = fmaf(v.w, x.e, o.w * x.f);
    }
    o.x = __fdiv_rn(o.x, x.l);
    o.y = __fdiv_rn(o.y, x.l);
    o.z = __fdiv_rn(o.z, x.l);
    o.w = __fdiv_rn(o.w, x.l);
    if (x.vec) {
        *reinterpret_cast<float4 *>(x.dst + d) = o;
    } else {
        x.dst[d] = o.x;
        x.dst[d + 1] = o.y;
        x.dst[d + 2] = o.z;
        x.dst[d + 3] = o.w;
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) paged_rows_kernel(const __grid_constant__ RowsArgs args) {
    const PagedPass &p = args.pass;
    const int unit = args.unit;
    using C = Cfg<T, DP>;
    constexpr int S = C::kSlots;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    unsigned char *ring = smem;                         // [S] operands: hi[, lo]
    float *row_ml = reinterpret_cast<float *>(smem + C::kRing);  // [4 tiles][kM][2]
    float *alpha = row_ml + 4 * kM * 2;                 // [4 tiles][kM]
    float *row_l2 = alpha + 4 * kM;                     // [4 tiles][kM] the second group's sums
    float *half_max = row_l2 + 4 * kM;                  // [2 groups][3][kM] tiles in turn, Q
    float *k_rel = half_max + 6 * kM;                   // [8 tiles][kKeys] keys' scales by their tile's
    float *v_scale = k_rel + 8 * kKeys;                 // [8 changes][DP]
    int *v_high = reinterpret_cast<int *>(v_scale + 8 * DP);      // [DP] largest exponents within the segment
    uint32_t *v_most = reinterpret_cast<uint32_t *>(v_high + DP);  // [8 warps][DP] a tile's largest values
    int *v_seg = reinterpret_cast<int *>(v_most + 8 * DP);  // the segment of v_high (4 words)
    uint32_t *k_most = reinterpret_cast<uint32_t *>(v_seg + 4);  // [2][8 warps] keys' largest
    int *v_change = reinterpret_cast<int *>(k_most + 16);  // [8 tiles] the channels' scales change here
    KeyTile *key_tile = reinterpret_cast<KeyTile *>(v_change + 8);  // [8 tiles]
    OddKeys *seg_odd = reinterpret_cast<OddKeys *>(key_tile + 8);  // [8 segments]
    uint32_t *odd_bits = reinterpret_cast<uint32_t *>(seg_odd + 8);  // [+, -][DP][kM / 32] outputs that see such
    Tile *tiles = reinterpret_cast<Tile *>(odd_bits + 2 * DP / 32 * kM);  // [8 tiles]
    long long *row_off = reinterpret_cast<long long *>(tiles + 8);  // [3 tiles][kKeys]
    int *flags = reinterpret_cast<int *>(row_off + 3 * kKeys);
    volatile int *abort = flags;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(flags + 1);
    int *last_s = flags + 2;
    long long *sums = reinterpret_cast<long long *>(flags + 4);   // [4] a scan's warps, [2] what it found
    uint64_t *bars = reinterpret_cast<uint64_t *>(sums + 6);
    uint64_t *raw = bars, *full = raw + S, *empty = full + S;  // [S] the ring's: copied, converted, used
    uint64_t *q_full = empty + S, *s_full = q_full + 1, *p_full = s_full + 2, *o_full = p_full + 2,
             *o_empty = o_full + 1, *done = o_empty + 1;
    // What threads pass each other beside the operands, in rings long enough
    // for the lead that the barriers above allow.
    uint64_t *k_sc = done + 1, *v_sc = k_sc + 8, *a_full = v_sc + 8;  // [8], [8], [4]

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int D = p.a.head_dim, H = p.a.heads, G = group_of(p);

    pdl_trigger();
    if (threadIdx.x == kM) {  // its warp has no part in the scan below
        for (int i = 0; i < S; i++) {
            mbar_init(&raw[i], unit > 1 ? 1 : kCopy);
            mbar_init(&full[i], C::kConv);
            mbar_init(&empty[i], 1);
        }
        mbar_init(q_full, 4 * C::kSoft);
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4 * C::kSoft);
        }
        mbar_init(o_full, 1);
        mbar_init(o_empty, 4);
        mbar_init(done, 1);
        for (int i = 0; i < 8; i++) {
            mbar_init(&k_sc[i], C::kConv);
            mbar_init(&v_sc[i], C::kConv);
        }
        for (int i = 0; i < 4; i++) mbar_init(&a_full[i], 4 * C::kSoft);
        fence_mbar_init();
        *abort = 0;
        for (int i = 0; i < 8; i++) key_tile[i] = KeyTile{};
        for (int i = 0; i < 8; i++) seg_odd[i] = {INT_MAX, 0};
        *v_seg = -1;
    }
    for (int i = threadIdx.x; i < 2 * DP / 32 * kM; i += kThreads) odd_bits[i] = 0;
    if (threadIdx.x >= kThreads - DP) v_scale[threadIdx.x - (kThreads - DP)] = pow2(kFirst - kTop - kShift);
    const Line line = line_scan(p, unit, sums);
    const long long U = line.total;
    const long long grid = min((long long)gridDim.x, U);
    if (blockIdx.x >= grid) {
        pdl_wait();
        return;
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_addr(tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const long long u0 = U * blockIdx.x / grid, u1 = U * (blockIdx.x + 1) / grid;
    line_find(line, u0, sums);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t s_tm = tmem, o_tm = tmem + 256, q_tm = tmem + 384;  // S: two buffers
    const int N = (int)(u1 - u0);
    Cursor c;
    line_place(p, unit, line, u0, sums, c);
    pdl_wait();

    // Operand j of the ring: K of tile 0, then K of tile (j + 1) / 2 (odd j)
    // or V of tile j / 2 - 1 (even j) while those last, 2 N in all.
    const int total = 2 * N;
    auto is_v = [&](int j) { return j == total - 1 || (j > 0 && j % 2 == 0); };
    auto tile_of = [&](int j) { return j == total - 1 ? N - 1 : j == 0 ? 0 : j % 2 ? (j + 1) / 2 : j / 2 - 1; };

    const bool soft = warp < 4 || (C::kSoft == 2 && warp >= 8 && warp < C::kConvWarp);
    // No wait below ends a loop: after one that gave up (the abort word is
    // set) every role runs through its remaining steps without waiting, so
    // that the barriers between its own threads stay matched.
    if (soft) {
        // ---- softmax ------------------------------------------------------
        if (C::kSoftRegs < kLaunchRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kSoftRegs));
        const int r = threadIdx.x & (kM - 1), group = warp >> 3;
        const uint32_t lane_tm = (uint32_t)((warp & 3) * 32) << 16;
        // The larger of both groups' values for the row.
        auto both = [&](float x, int buffer) {
            if (C::kSoft == 1) return x;
            half_max[(3 * group + buffer) * kM + r] = x;
            bar_sync(4, 2 * kM);
            return max_nan(x, half_max[(3 * (1 - group) + buffer) * kM + r]);
        };
        // Queries are taken with the scale's sign; its size comes after the product.
        const float sign = p.scale_log2 < 0.f ? -1.f : 1.f, size = fabsf(p.scale_log2);
        float m = -INFINITY, l = 0.f, qs = 1.f;
        int hi = 0, lo = 0;
        bool first = true, sound = true;  // sound: a row with a finite query
        for (int n = 0; n < N; n++) {
            if (first) {
                // The row to TMEM: first as it is, 128 columns, while its largest
                // value is found, then every 32 columns in place as 16 of hi
                // and 16 of lo. The segment before is through with Q (its
                // last S is read).
                const int row = c.r0 + r, tok = row / G;
                const bool live = r < c.rows;
                const float *q = p.a.q + (live ? ((size_t)(c.tok0 + tok) * H + c.kvh * G + (row - tok * G)) * D : 0);
                const bool vec = aligned16(p.a.q);
                float top = 0.f;
#pragma unroll 1
                for (int h = group * (DP / 2); h < (C::kSoft == 1 ? DP : (group + 1) * (DP / 2)); h += 32) {
                    float4 v[8];
#pragma unroll
                    for (int y = 0; y < 8; y++) {
                        const float *at = q + h + 4 * y;
                        v[y] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (live && h + 4 * y < D)
                            v[y] = vec ? *reinterpret_cast<const float4 *>(at)
                                       : make_float4(at[0], at[1], at[2], at[3]);
                    }
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        uint32_t x[16];
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            const float4 f = v[4 * y + z];
                            x[4 * z] = __float_as_uint(f.x * sign);
                            x[4 * z + 1] = __float_as_uint(f.y * sign);
                            x[4 * z + 2] = __float_as_uint(f.z * sign);
                            x[4 * z + 3] = __float_as_uint(f.w * sign);
                        }
#pragma unroll
                        for (int z = 0; z < 16; z++) top = max_nan(top, fabsf(__uint_as_float(x[z])));
                        tmem_st16(q_tm + lane_tm + h + 16 * y, x);
                    }
                }
                tmem_wait_st();
                top = both(top, 2);
                const int ex = scale_exponent(__float_as_uint(top));
                sound = live && top < INFINITY;
                const float sc = pow2(kShift - ex);
                qs = pow2(ex - kShift);
#pragma unroll 1
                for (int h = group * (DP / 2); h < (C::kSoft == 1 ? DP : (group + 1) * (DP / 2)); h += 32) {
                    uint32_t x[32], qh[16], ql[16];
                    tmem_ld32_async(q_tm + lane_tm + h, x);
                    tmem_wait_ld(x);
#pragma unroll
                    for (int d = 0; d < 16; d++)
                        split2(mul2(F2(__uint_as_float(x[2 * d]), __uint_as_float(x[2 * d + 1])), F2(sc, sc)), qh[d],
                               ql[d]);
                    tmem_st16(q_tm + lane_tm + h, qh);
                    tmem_st16(q_tm + lane_tm + h + 16, ql);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
                m = -INFINITY;
                l = 0.f;
                // Row r sees key indexes i < hi with i >= lo or i < sinks.
                hi = c.keys;
                lo = c.from - c.low + c.sink;
                if (!p.prefix_pass) {
                    const int at = c.past + tok;
                    hi = min(hi, at + 1 - c.low + c.sink);
                    if (p.a.window) lo = max(at - p.a.window + 1 - c.low, 0) + c.sink;
                }
            }
            mbar_wait(&s_full[n & 1], (n >> 1) & 1, p.a.err, abort, args.limit);
            if (!C::kRaw) mbar_wait(&k_sc[n & 7], (n >> 3) & 1, p.a.err, abort, args.limit);
            tc_fence_after();
            const int i0 = c.tile * kKeys;
            // Rows past the tile's last hold zeros; they need no mask.
            const bool whole = i0 + kKeys <= hi && (i0 >= lo || i0 + kKeys <= p.a.sinks);
            const bool masked = __any_sync(0xffffffffu, !whole);
            const uint4 kt = *reinterpret_cast<const uint4 *>(key_tile + (n & 7));
            // Not 0, which would make NaN of -infinity.
            const float f = max_nan(C::kRaw ? qs * size : qs * __uint_as_float(kt.x) * size, FLT_MIN);
            const uint32_t st = s_tm + (n & 1) * 128 + lane_tm;
            const int h_first = group * 2;
            if (!C::kRaw && __builtin_expect((kt.z | kt.w) != 0, 0))
                rescale_scores<T, DP>(st, 32 * h_first, key_tile + (n & 7), k_rel + (n & 7) * kKeys);
            // Where some row's mask hides keys of the tile, S there becomes
            // -infinity first: two forms of the passes below would be twice the
            // code, whose fetches cost the other roles more.
            if (masked) mask_scores<T, DP>(st, 32 * h_first, hi - i0, lo - i0, p.a.sinks - i0);
            float mx = -INFINITY;
#pragma unroll 1
            for (int h = h_first; h < h_first + 4 / C::kSoft; h++) {
                uint32_t x[32];
                tmem_ld32_async(st + 32 * h, x);
                tmem_wait_ld(x);
#pragma unroll
                for (int j = 0; j < 32; j++) mx = max_nan(mx, __uint_as_float(x[j]));
            }
            float other = -INFINITY;
            float *mine = half_max + (3 * group + (n & 1)) * kM + r, *theirs = mine + (1 - 2 * group) * 3 * kM;
            if (C::kSoft == 2) {
                *mine = mx;
                bar_sync(4, 2 * kM);
                other = *theirs;
            }
            // NaN among a finite query's scores: a key holds what is not finite.
            // The two warps of a row see the same and meet once more.
            if (__builtin_expect(__any_sync(0xffffffffu, sound && (mx != mx || other != other)), 0)) {
                const int tok = (c.r0 + r) / G;
                const float *q = p.a.q + ((size_t)(c.tok0 + tok) * H + c.kvh * G + (c.r0 + r - tok * G)) * D;
                mx = repair_scores<T, DP>(p, st, 32 * h_first, q, c.b, c.kvh, i0, c.sink, c.low, sound && l == l);
                if (C::kSoft == 2) {
                    bar_sync(5 + (warp & 3), 64);
                    *mine = mx;
                    bar_sync(5 + (warp & 3), 64);
                    other = *theirs;
                }
            }
            mx = fmaxf(mx, other);
            const float own = mx == -INFINITY ? mx : mx * f, nm = fmaxf(m, own);
            float mu = nm == -INFINITY ? 0.f : nm - (float)kShift;
            // Scores past 2^22, whose rounding is not small against 1: their
            // distance from the largest is taken first, or that one's
            // probability would not be near 1.
            const bool large = fabsf(nm) >= kLarge && fabsf(nm) < INFINITY;
            if (__builtin_expect(__any_sync(0xffffffffu, large), 0)) {
                shift_scores<T, DP>(st, 32 * h_first, large ? own >= m ? mx : m / f : 0.f);
                mu = large ? -(float)kShift : mu;
            }
            const float a = m == -INFINITY ? 0.f : ex2(m - nm);
            F2 sum2(0.f, 0.f);
#pragma unroll 1
            for (int h = h_first; h < h_first + 4 / C::kSoft; h++) {
                uint32_t x[32], ph[16], pl[16];
                tmem_ld32_async(st + 32 * h, x);
                tmem_wait_ld(x);
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float2 z =
                        fma2(F2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), F2(f, f), F2(-mu, -mu)).get();
                    const F2 e(ex2(z.x), ex2(z.y));
                    sum2 = add2(sum2, e);
                    split2(e, ph[j], pl[j]);
                }
                tmem_st16(st + 32 * h, ph);
                tmem_st16(st + 32 * h + 16, pl);
            }
            m = nm;
            l = fmaf(l, a, sum2.get().x + sum2.get().y);
            if (group == 0) alpha[(n & 3) * kM + r] = a;
            first = c.tile == c.tiles - 1;
            if (first || n == N - 1) {
                if (group == 0) {
                    row_ml[((n & 3) * kM + r) * 2] = m;
                    row_ml[((n & 3) * kM + r) * 2 + 1] = l * pow2(-kShift);
                } else {
                    row_l2[(n & 3) * kM + r] = l * pow2(-kShift);
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&a_full[n & 3]);
                mbar_arrive(&p_full[n & 1]);
            }
            if (n + 1 < N) cursor_next(p, unit, c);
        }
    } else if (warp < 8) {
        // ---- output -------------------------------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kOutRegs));
        const int r = threadIdx.x - 128, ow = warp - 4;
        const uint32_t lane_tm = (uint32_t)(ow * 32) << 16;
        F2 acc[DP / 2];  // in units of the channels' scales
        int change = 0, seg = 0;
#pragma unroll
        for (int d = 0; d < DP / 2; d++) acc[d] = F2(0.f, 0.f);
        for (int n = 0; n < N; n++) {
            mbar_wait(&a_full[n & 3], (n >> 2) & 1, p.a.err, abort, args.limit);
            mbar_wait(&v_sc[n & 7], (n >> 3) & 1, p.a.err, abort, args.limit);
            mbar_wait(o_full, n & 1, p.a.err, abort, args.limit);
            tc_fence_after();
            const float a = alpha[(n & 3) * kM + r];
            if (!C::kRaw && __builtin_expect(v_change[n & 7], 0)) {
                const float *was = v_scale + (change++ & 7) * DP, *now = v_scale + (change & 7) * DP;
#pragma unroll
                for (int d = 0; d < DP / 2; d++) {
                    const float2 x = *reinterpret_cast<const float2 *>(was + 2 * d),
                                 y = *reinterpret_cast<const float2 *>(now + 2 * d);
                    acc[d] = mul2(acc[d], F2(ratio2(x.x, y.x), ratio2(x.y, y.y)));
                }
            }
            float m = row_ml[((n & 3) * kM + r) * 2], l = row_ml[((n & 3) * kM + r) * 2 + 1];
            if (C::kSoft == 2) l += row_l2[(n & 3) * kM + r];
            const uint32_t ot = o_tm + lane_tm;
#pragma unroll
            for (int h = 0; h < DP / 16; h++) {
                float x[16];
                tmem_ld16(ot + 16 * h, x);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    F2 &d = acc[8 * h + j];
                    d = fma2(d, F2(a, a), F2(x[2 * j], x[2 * j + 1]));
                }
            }
            tc_fence_before();
            const bool seg_end = c.tile == c.tiles - 1;
            if (!seg_end && n + 1 < N) {
                __syncwarp();
                if (lane == 0) mbar_arrive(o_empty);
                cursor_next(p, unit, c);
                continue;
            }
            // ---- end of this CTA's piece of the segment.
            auto four = [&](int d) {
                const float2 x = acc[2 * d].get(), y = acc[2 * d + 1].get();
                return make_float4(x.x, x.y, y.x, y.y);
            };
            const float *vs = v_scale + (change & 7) * DP;
#pragma unroll
            for (int d = 0; d < DP / 2; d++) {
                const float2 x = C::kRaw ? make_float2(pow2(-kShift), pow2(-kShift))
                                         : *reinterpret_cast<const float2 *>(vs + 2 * d);
                acc[d] = mul2(acc[d], F2(x.x, x.y));
            }
            const OddKeys odd = seg_odd[seg & 7];
            const bool has_odd = bar_or(2, 128, odd.to != 0);  // one answer for all, whatever was waited for
            if (r == 0) seg_odd[seg & 7] = {INT_MAX, 0};
            __syncwarp();
            if (lane == 0) mbar_arrive(o_empty);
            const bool live = r < c.rows;
            auto add_odd = [&](float *dst, int step, bool mine) {
                odd_values<T, DP>(p, c, odd.from, min(c.keys, odd.to), dst, step, mine, odd_bits);
            };
            const int row = c.r0 + r, tok = row / G;
            const size_t qrow = (size_t)(c.tok0 + tok) * H + c.kvh * G + (row - tok * G);
            const long long a0 = u0 + n - c.tile, a1 = a0 + c.tiles;  // the segment's units
            bool write = live;
            if (a0 < u0 || a1 > u1) {
                const int c_first = (int)(((a0 + 1) * grid - 1) / U), c_last = (int)((a1 * grid - 1) / U);
                const size_t slot = 2 * blockIdx.x + (a0 >= u0 ? 1 : 0);
                float4 *po = reinterpret_cast<float4 *>(p.part_o) + slot * (DP / 4) * kM + r;
#pragma unroll
                for (int d = 0; d < DP / 4; d++) po[d * kM] = four(d);
                reinterpret_cast<float2 *>(p.part_ml)[slot * kM + r] = make_float2(m, l);
                if (__builtin_expect(has_odd, 0)) add_odd(reinterpret_cast<float *>(po), 4 * kM, true);
                if (args.join) {
                    write = false;
                } else {
                    bar_sync(2, 128);
                    if (r == 0) {
                        __threadfence();
                        const unsigned ticket = atomicAdd(&p.a.tickets[c_first], 1u);
                        *last_s = ticket == (unsigned)(c_last - c_first);
                        if (*last_s) p.a.tickets[c_first] = 0u;
                        __threadfence();
                    }
                    bar_sync(2, 128);
                    write = live && *last_s;
                    bar_sync(2, 128);
                }
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
                            const F2 z(0.f, 0.f);
                            acc[2 * d] = fma2(F2(v.x, v.y), F2(e, e), x == 0 ? z : mul2(acc[2 * d], F2(f, f)));
                            acc[2 * d + 1] =
                                fma2(F2(v.z, v.w), F2(e, e), x == 0 ? z : mul2(acc[2 * d + 1], F2(f, f)));
                        }
                        m = nm;
                    }
                }
            }
            if (write) {
                const RowEnd end = row_end(p, qrow, m, l);
#pragma unroll
                for (int d = 0; d < DP; d += 4)
                    if (d < D) row_store(end, d, four(d / 4));
            }
            if (__builtin_expect(has_odd && a0 >= u0 && a1 <= u1, 0))
                add_odd((p.prefix_pass ? p.pre_o : p.a.out) + (live ? qrow * D : 0), 4, live);
#pragma unroll
            for (int d = 0; d < DP / 2; d++) acc[d] = F2(0.f, 0.f);
            seg++;
            if (n + 1 < N) cursor_next(p, unit, c);
        }
    } else if (warp < 16) {
        // ---- conversion ---------------------------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kConvRegs));
        using O = Operand<T, DP>;
        const int pw = warp - C::kConvWarp;
        // Piece i of a lane: row (i kConv + pw) kRpi + sub, 16 raw bytes from
        // dim `col` on. A piece on is a multiple of 8 rows on.
        const int sub = lane / C::kLpr, ch = lane % C::kLpr, col = ch * C::kEpl;
        constexpr int kBatch = 2, kStep = C::kConv * C::kRpi * 128;
        static_assert(C::kRows % kBatch == 0 && C::kConv * C::kRpi % 8 == 0, "batches of pieces 8 rows apart");
        auto row_of = [&](int i) { return (i * C::kConv + pw) * C::kRpi + sub; };
        const uint32_t op0 = operand_at(row_of(0), col);
        const uint32_t raw0 = C::kPair ? (ch >> 3) * C::kBlockBytes + row_of(0) * 128 + (ch & 7) * 16 : op0;
        int e_k = kFirst;    // exponent of the largest value expected of a tile's keys
        F2 vs[C::kEpl / 2];  // this lane's channels' scales
        int change = 0;      // of them
#pragma unroll
        for (int e = 0; e < C::kEpl / 2; e++) vs[e] = F2(pow2(kTop - kFirst), pow2(kTop - kFirst));
        for (int j = 0; j < total; j++) {
            const bool v = is_v(j);
            const int n = tile_of(j);
            mbar_wait(&raw[j % S], (j / S) & 1, p.a.err, abort, args.limit);
            unsigned char *slot = ring + (j % S) * C::kTileBytes;
            const Tile &cu = tiles[n & 7];
            const bool whole = cu.whole;
            // Rows that no query sees may hold anything, or be of a tile before.
            if (!whole && (v || !C::kRaw))
#pragma unroll 1
                for (int i = 0; i < C::kRows; i++)
                    if (!live_key(p, cu, cu.i0 + row_of(i)))
                        *reinterpret_cast<uint4 *>(slot + raw0 + i * kStep) = make_uint4(0, 0, 0, 0);
            const uint32_t to = smem_addr(slot) + op0;
            if (!C::kRaw && !v) {
                const float f = pow2(kTop - e_k);
                F2 sc[C::kEpl / 2];
#pragma unroll
                for (int e = 0; e < C::kEpl / 2; e++) sc[e] = F2(f, f);
                uint32_t top = 0, low = 0xffffffffu;  // low: less 1, so that zeros do not count
#pragma unroll 1
                for (int ib = 0; ib < C::kRows; ib += kBatch) {
                    uint4 x[kBatch];
#pragma unroll
                    for (int y = 0; y < kBatch; y++)
                        x[y] = *reinterpret_cast<const uint4 *>(slot + raw0 + (ib + y) * kStep);
                    __syncwarp();  // a row of pairs is read whole before it is written
#pragma unroll
                    for (int y = 0; y < kBatch; y++) {
                        const uint32_t t = O::largest(x[y]);
                        top = max(top, t);
                        low = min(low, t - 1);
                        O::convert(x[y], sc, to + (ib + y) * kStep);
                    }
                }
                top = __reduce_max_sync(0xffffffffu, top);
                // A warp with 16 bytes (a key, perhaps) that the scale does not
                // suit takes its keys from the cache once more.
                const bool off = __any_sync(0xffffffffu, (top && scale_exponent(top) > e_k + 3) ||
                                                             (int)(low >> 23) - 127 < e_k - kNear);
                if (__builtin_expect(off, 0))
                    keys_again<T, DP>(p, cu, to, e_k, k_rel + (n & 7) * kKeys);
                if (lane == 0) {
                    k_most[8 * (n & 1) + pw] = top;
                    key_tile[n & 7].own[pw] = off;
                    if (pw == 0) key_tile[n & 7].scale = pow2(e_k - kTop);
                }
            } else if (!C::kRaw) {
                uint32_t top[4] = {0, 0, 0, 0};
#pragma unroll 1
                for (int ib = 0; ib < C::kRows; ib += kBatch) {
                    uint4 x[kBatch];
#pragma unroll
                    for (int y = 0; y < kBatch; y++)
                        x[y] = *reinterpret_cast<const uint4 *>(slot + raw0 + (ib + y) * kStep);
                    __syncwarp();  // a row of pairs is read whole before it is written
#pragma unroll
                    for (int y = 0; y < kBatch; y++) {
                        top[0] = O::larger(top[0], O::size_of(x[y].x));
                        top[1] = O::larger(top[1], O::size_of(x[y].y));
                        top[2] = O::larger(top[2], O::size_of(x[y].z));
                        top[3] = O::larger(top[3], O::size_of(x[y].w));
                        O::convert(x[y], vs, to + (ib + y) * kStep);
                    }
                }
                // Channels keep their scales while the largest value of this
                // lane's keys, scaled, is from 2^1 to 2^15.
                bool off = false;
#pragma unroll
                for (int e = 0; e < C::kEpl; e++) {
                    const uint32_t t =
                        C::kPair ? top[e % 4] : e % 2 ? top[e / 2 % 4] & 0xffff0000u : top[e / 2 % 4] << 16;
                    const float2 f = vs[e / 2].get();
                    const float at = __uint_as_float(t) * (e % 2 ? f.y : f.x);
                    off |= t && !(at >= 2.f && at < 32768.f);
                }
                off = bar_or(1, C::kConv * 32, off);
                if (__builtin_expect(off, 0)) {
                    const float *was = v_scale + (change++ & 7) * DP;
                    float *now = v_scale + (change & 7) * DP;
                    values_again<T, DP>(p, cu, to, v_most, v_high, v_seg, was, now, &seg_odd[cu.seg & 7]);
#pragma unroll
                    for (int e = 0; e < C::kEpl / 2; e++)
                        vs[e] = F2(O::inverse(now[col + 2 * e]), O::inverse(now[col + 2 * e + 1]));
                }
                // The keys' largest values that the barrier has brought together.
                const uint32_t t = __reduce_max_sync(
                    0xffffffffu, lane < C::kConv ? k_most[8 * (min(n + 1, N - 1) & 1) + lane] : 0u);
                if (t && t < 0x7f800000u) e_k = scale_exponent(t);
                if (lane == 0 && pw == 0) v_change[n & 7] = off;
            }
            if (C::kRaw && v) {
                uint32_t odd = 0;  // bit 15 of each half: its magnitude is 0x7c00 or more
#pragma unroll 4
                for (int i = 0; i < C::kRows; i++) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(slot + raw0 + i * kStep);
                    odd |= (O::size_of(x.x) + 0x04000400u) | (O::size_of(x.y) + 0x04000400u) |
                           (O::size_of(x.z) + 0x04000400u) | (O::size_of(x.w) + 0x04000400u);
                }
                if (__builtin_expect((odd & 0x80008000u) != 0, 0)) clean_values<T, DP>(slot + raw0, cu.i0, &seg_odd[cu.seg & 7]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (!v)
                    mbar_arrive(&k_sc[n & 7]);
                else
                    mbar_arrive(&v_sc[n & 7]);
                mbar_arrive(&full[j % S]);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRestRegs));
        if (warp > 16) {
            // ---- copies -------------------------------------------------------
            int seg = 0;
            // Before the copy of a tile's keys: the ring of eight is far behind.
            auto tell = [&](int n, bool begins) {
                Tile t;
                t.begins = begins;
                t.i0 = c.tile * kKeys;
                t.whole = t.i0 + kKeys <= c.keys &&
                          (key_pos(c, t.i0) >= c.from || key_pos(c, t.i0 + kKeys - 1) < p.a.sinks);
                t.seg = seg;
                t.b = c.b, t.kvh = c.kvh;
                t.sink = c.sink, t.low = c.low, t.from = c.from, t.keys = c.keys;
                tiles[n & 7] = t;
            };
            if (unit > 1) {
                if (warp == 17) {
                    // Lane i copies box row i of the tile: `unit` keys of a page.
                    const int boxes = kKeys / unit;
                    constexpr int kBlk = DP * (int)sizeof(T) / 128;
                    uint32_t id = 0, id_v = 0;
                    int z = -1, z_v = -1, kvh_v = 0;  // key within the page; -1: no keys there
                    auto look_up = [&] {
                        const int i = c.tile * kKeys + lane * unit;
                        z = -1;
                        if (lane < boxes && i < c.keys) {
                            const int pos = key_pos(c, i), pg = page_of(p.a.cache, pos);
                            z = pos - pg * p.a.cache.page;
                            id = pg < p.a.batch.per_seq
                                     ? p.a.batch.table[(long long)c.b * p.a.batch.per_seq + pg]
                                     : ~0u;
                        }
                    };
                    auto copy = [&](int j, uint32_t page_id, int at, int kvh, int parity, int n, bool begins) {
                        if (j >= S) mbar_wait(&empty[j % S], (j / S - 1) & 1, p.a.err, abort, args.limit);
                        if (__any_sync(0xffffffffu, *abort)) return;
                        if (at >= 0 && page_id >= (uint32_t)p.a.cache.pages) {  // checked on the host; see paged_row
                            report_error(p.a.err, kErrGatherId);
                            page_id = 0;
                        }
                        const int count = __popc(__ballot_sync(0xffffffffu, at >= 0));
                        if (lane == 0) {
                            if (!parity) tell(n, begins);
                            mbar_arrive_expect_tx(&raw[j % S], count * unit * 128 * kBlk);
                        }
                        __syncwarp();
                        unsigned char *slot = ring + (j % S) * C::kTileBytes + lane * unit * 128;
                        if (at >= 0)
#pragma unroll
                            for (int y = 0; y < kBlk; y++)
                                tma_load_5d(slot + y * C::kBlockBytes, &args.map, y * (128 / (int)sizeof(T)), kvh, at,
                                            parity, (int)page_id, &raw[j % S]);
                    };
                    if (lane == 0) prefetch_tensormap(&args.map);
                    look_up();
                    bool begins = true;
                    for (int n = 0; n < N; n++) {
                        copy(n ? 2 * n - 1 : 0, id, z, c.kvh, 0, n, begins);
                        if (n) copy(2 * n, id_v, z_v, kvh_v, 1, n, false);
                        id_v = id;
                        z_v = z;
                        kvh_v = c.kvh;
                        begins = c.tile == c.tiles - 1;
                        seg += begins;
                        if (n + 1 < N) {
                            cursor_next(p, unit, c);
                            look_up();
                        }
                    }
                    copy(total - 1, id_v, z_v, kvh_v, 1, N, false);
                    // Copies still in flight must land before the CTA's shared
                    // memory is released (after a wait that gave up; else the
                    // MMAs have used them all).
                    if (*abort)
                        for (int j = max(total - S, 0); j < total; j++) drain_wait(&raw[j % S], (j / S) & 1);
                }
            } else {
                // Rows kRpi at a time, every kCopy-th of them a warp's, by 16-byte
                // pieces; their places in the cache through a ring of three tiles.
                const int w = warp - 17, sub = lane / C::kLpr, ch = lane % C::kLpr, col = ch * C::kEpl;
                auto look_up = [&](int n) {
                    for (int r = threadIdx.x - 17 * 32; r < kKeys; r += kCopy * 32) {
                        const int i = c.tile * kKeys + r;
                        long long off = -1;
                        if (i < c.keys)
                            off = paged_row(p.a.cache, p.a.batch, c.b, key_pos(c, i), p.a.err) +
                                  c.kvh * D * (long long)sizeof(T);
                        row_off[n % 3 * kKeys + r] = off;
                    }
                    bar_sync(3, kCopy * 32);
                };
                auto copy = [&](int j, int n, int parity) {
                    if (j >= S) mbar_wait(&empty[j % S], (j / S - 1) & 1, p.a.err, abort, args.limit);
                    unsigned char *slot = ring + (j % S) * C::kTileBytes;
                    const char *base = p.a.cache.base + (parity ? p.a.cache.parity_stride : 0) + col * (int)sizeof(T);
#pragma unroll 4
                    for (int r = w * C::kRpi + sub; r < kKeys; r += kCopy * C::kRpi) {
                        const long long off = row_off[n % 3 * kKeys + r];
                        const bool live = off >= 0 && col < D;
                        cp_async16_zfill(slot + (C::kPair ? (ch >> 3) * C::kBlockBytes + r * 128 + (ch & 7) * 16
                                                          : operand_at(r, col)),
                                         live ? base + off : p.a.cache.base, live ? 16 : 0);
                    }
                };
                int done_j = 0;
                auto landed = [&](int j) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&raw[j % S]);
                };
                for (int j = 0; j < total; j++) {
                    const bool v = is_v(j);
                    const int n = tile_of(j);
                    if (!v) {
                        bool begins = n == 0;
                        if (n) {
                            begins = c.tile == c.tiles - 1;
                            seg += begins;
                            cursor_next(p, unit, c);
                        }
                        look_up(n);
                        if (w == 0 && lane == 0) tell(n, begins);
                    }
                    copy(j, n, v);
                    cp_async_commit();
                    if (j >= C::kAhead) {
                        cp_async_wait<C::kAhead>();
                        landed(done_j++);
                    }
                }
                cp_async_wait<0>();
                while (done_j < total) landed(done_j++);
            }
        } else {
            // ---- MMA issue ----------------------------------------------------
            // The whole warp walks the loop and one elected lane issues. Inside
            // one lane's branch 16 MMAs took 1600 cycles to issue, 1024 to run;
            // uniform control flow took 10 % off two prompts of 2048 tokens over
            // an f16 cache, 3 % over f32. With all steps unrolled the code of the
            // roles outgrew the instruction caches (1.2 times as long in either);
            // rolled up, f32 and bf16 took 2 to 4 % less than half unrolled, f16
            // 7 % more.
            // The small products of a tile come before all large ones: the
            // tensor core cuts its sums off at the size of what they hold, and
            // the order halves the error (1.0e-6 to 4.6e-7 of the outputs'
            // norm over 1100 f32 keys, 7.2e-7 to 4.5e-7 f16) for 3 to 4 % of time.
            const uint32_t ra = smem_addr(ring);
            int seg = 0;
            auto slot_wait = [&](int j) {
                mbar_wait(&full[j % S], (j / S) & 1, p.a.err, abort, args.limit);
                return ra + (j % S) * C::kTileBytes;
            };
            auto qk = [&](int n, bool begins, uint32_t kb) {
                const int j = n ? 2 * n - 1 : 0;
                if (begins) mbar_wait(q_full, seg++ & 1, p.a.err, abort, args.limit);
                if (!__any_sync(0xffffffffu, *abort)) {
                    tc_fence_after();
                    const uint32_t d = s_tm + (n & 1) * 128;
                    const uint64_t desc = sw128_desc(kb);
#pragma unroll 1
                    for (int b = 0; b < C::kBlocks; b++) {
                        // 64 dims: descriptors hold addresses in 16-byte units.
                        const uint64_t kh = desc + b * (C::kBlockBytes / 16);
                        const uint32_t qh = q_tm + b * 64;
#pragma unroll(C::kRaw ? 4 : 1)
                        for (int ks = 0; ks < 4; ks++) {
                            const uint32_t at = qh + ks / 2 * 32 + ks % 2 * 8;
                            mma_ts(d, at + 16, kh + ks * 2, C::kIdescS, b + ks);
                            if (C::kPair) mma_ts(d, at, kh + ks * 2 + C::kHalfBytes / 16, C::kIdescS, 1u);
                        }
                    }
#pragma unroll 1
                    for (int b = 0; b < C::kBlocks; b++) {
                        const uint64_t kh = desc + b * (C::kBlockBytes / 16);
                        const uint32_t qh = q_tm + b * 64;
#pragma unroll(C::kRaw ? 4 : 1)
                        for (int ks = 0; ks < 4; ks++)
                            mma_ts(d, qh + ks / 2 * 32 + ks % 2 * 8, kh + ks * 2, C::kIdescS, 1u);
                    }
                    commit_one(&empty[j % S]);
                    commit_one(&s_full[n & 1]);
                }
            };
            auto pv = [&](int n) {
                mbar_wait(&p_full[n & 1], (n >> 1) & 1, p.a.err, abort, args.limit);
                const int j = n == N - 1 ? total - 1 : 2 * n + 2;
                const uint32_t vb = slot_wait(j);
                if (n >= 1) mbar_wait(o_empty, (n - 1) & 1, p.a.err, abort, args.limit);
                if (!__any_sync(0xffffffffu, *abort)) {
                    tc_fence_after();
                    const uint32_t pt = s_tm + (n & 1) * 128;
                    const uint64_t desc = sw128_desc_mn(vb, C::kBlockBytes);
#pragma unroll 1
                    for (int b = 0; b < kKeys / 32; b++) {
                        const uint64_t vh = desc + b * (2 * 2048 / 16);
                        const uint32_t ph = pt + b * 32;
#pragma unroll(C::kRaw ? 2 : 1)
                        for (int ks = 0; ks < 2; ks++) {
                            mma_ts(o_tm, ph + ks * 8 + 16, vh + ks * 128, C::kIdescO, b + ks);
                            if (C::kPair)
                                mma_ts(o_tm, ph + ks * 8, vh + ks * 128 + C::kHalfBytes / 16, C::kIdescO, 1u);
                        }
                    }
#pragma unroll 1
                    for (int b = 0; b < kKeys / 32; b++) {
                        const uint64_t vh = desc + b * (2 * 2048 / 16);
                        const uint32_t ph = pt + b * 32;
#pragma unroll(C::kRaw ? 2 : 1)
                        for (int ks = 0; ks < 2; ks++) mma_ts(o_tm, ph + ks * 8, vh + ks * 128, C::kIdescO, 1u);
                    }
                    commit_one(&empty[j % S]);
                    commit_one(o_full);
                }
            };
            // Q K^T one tile ahead, but a segment's first waits for its Q, which
            // the softmax warps write after the tile before: P V goes first there.
            bool begins = true;
            uint32_t kb = 0;
            for (int nq = 0, np = 0, known = 0; np < N;) {
                if (nq < N && nq <= np + 1 && known <= nq) {
                    kb = slot_wait(nq ? 2 * nq - 1 : 0);
                    begins = tiles[nq & 7].begins;
                    known = nq + 1;
                }
                if (nq < N && nq <= np + 1 && !(begins && np < nq)) {
                    qk(nq, begins, kb);
                    nq++;
                } else {
                    pv(np++);
                }
            }
            // Every MMA issued must complete before TMEM is freed.
            commit_one(done);
            drain_wait(done, 0);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 16) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Merges the pieces of the segments that cuts of the work line split, a block
// for every cut: a segment in k + 1 pieces has k of them, each for an equal
// part of its rows. The pieces are added in ascending order, eight reads in
// flight. Launched where segments are fewer than CTAs, and so in many pieces
// each: for a prefix of 8192 keys in ten, the last CTA to finish one took 23 us
// to merge it alone, this launch takes 6. With more segments than CTAs a
// segment is in two pieces mostly, and a launch less was better by 17 us in 930
// (two prompts of 2048 tokens).
constexpr int kJoinThreads = 512;
template <int DP>
__global__ void __launch_bounds__(kJoinThreads) rows_join_kernel(const __grid_constant__ PagedPass p, int unit,
                                                                 int ctas) {
    __shared__ long long sums[6];
    pdl_trigger();
    const Line line = line_scan(p, unit, sums);
    const long long U = line.total;
    const long long grid = min((long long)ctas, U);
    const int cut = 1 + blockIdx.x;  // before CTA `cut`
    if (cut >= grid) {
        pdl_wait();
        return;
    }
    const long long u = U * cut / grid;
    line_find(line, u, sums);
    __syncthreads();
    Cursor c;
    line_place(p, unit, line, u, sums, c);
    pdl_wait();
    if (c.tile == 0) return;  // the cut lies between two segments
    const long long a0 = u - c.tile, a1 = a0 + c.tiles;
    const int first = (int)(((a0 + 1) * grid - 1) / U), last = (int)((a1 * grid - 1) / U);
    const int shares = last - first, share = cut - first - 1;
    const int lo = (int)((long long)c.rows * share / shares), n = (int)((long long)c.rows * (share + 1) / shares) - lo;
    const int G = group_of(p), D = p.a.head_dim;
    for (int i = threadIdx.x; i < n * (D / 4); i += kJoinThreads) {
        const int d = i / n, r = lo + i % n, row = c.r0 + r, tok = row / G;
        const size_t qrow = (size_t)(c.tok0 + tok) * p.a.heads + c.kvh * G + (row - tok * G);
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int x = first; x <= last; x += 8) {
            float2 ml[8];
            float4 v[8];
#pragma unroll
            for (int y = 0; y < 8; y++) {
                ml[y] = make_float2(-INFINITY, 0.f);
                v[y] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (x + y > last) continue;
                const size_t slot = 2 * (size_t)(x + y) + (x + y == first ? 1 : 0);
                ml[y] = __ldcg(reinterpret_cast<const float2 *>(p.part_ml) + slot * kM + r);
                v[y] = __ldcg(reinterpret_cast<const float4 *>(p.part_o) + (slot * (DP / 4) + d) * kM + r);
            }
            float nm = m;
#pragma unroll
            for (int y = 0; y < 8; y++) nm = fmaxf(nm, ml[y].x);
            const float mu = nm == -INFINITY ? 0.f : nm, f = ex2(m - mu);
            l *= f;
            o.x *= f;
            o.y *= f;
            o.z *= f;
            o.w *= f;
#pragma unroll
            for (int y = 0; y < 8; y++) {
                const float e = ex2(ml[y].x - mu);
                l = fmaf(ml[y].y, e, l);
                o.x = fmaf(v[y].x, e, o.x);
                o.y = fmaf(v[y].y, e, o.y);
                o.z = fmaf(v[y].z, e, o.z);
                o.w = fmaf(v[y].w, e, o.w);
            }
            m = nm;
        }
        row_store(row_end(p, qrow, m, l), 4 * d, o);
    }
}

int padded_dim(int d) { return d <= 64 ? 64 : 128; }

template <typename T, int DP>
cudaError_t launch(cudaStream_t s, const PagedPass &p) {
    using C = Cfg<T, DP>;
    static_assert(C::kSmem <= 227 * 1024, "shared layout");
    RowsArgs args{};
    args.pass = p;
    args.limit = kLimitNs + kLimitKeyNs * (uint64_t)p.a.batch.per_seq * (uint64_t)p.a.cache.page;
    args.join = ((size_t)p.a.tokens * (p.a.heads / p.a.kv_heads) + kM - 1) / kM * p.a.kv_heads < (size_t)kSmCount;
    args.unit = paged_boxes(p.a, kKeys, sizeof(T), C::kRaw, !C::kPair, &args.map);
    static std::atomic<uint64_t> smem_set{0};
    cudaError_t e = set_smem_limit_once(paged_rows_kernel<T, DP>, C::kSmem, &smem_set);
    if (e != cudaSuccess) return e;
    // The register split above needs the launch to hold kLaunchRegs a thread.
    static const int regs = [] {
        cudaFuncAttributes at{};
        return cudaFuncGetAttributes(&at, paged_rows_kernel<T, DP>) == cudaSuccess ? at.numRegs : 0;
    }();
    if (regs < kLaunchRegs) return cudaErrorInvalidConfiguration;
    launch_k(paged_rows_kernel<T, DP>, kSmCount, kThreads, C::kSmem, s, args);
    count_launch();
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    if (args.join) {
        launch_k(rows_join_kernel<DP>, kSmCount - 1, kJoinThreads, 0, s, p, args.unit, kSmCount);
        count_launch();
    }
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
