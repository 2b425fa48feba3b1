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
// are cut into tiles of kTileKeys. All tiles of all segments, and one more unit
// for a segment's end, which takes about a tile's time, form one line
// that the CTAs (one or two per SM) share out in equal contiguous ranges, so a batch
// of any lengths keeps every SM busy to the end. The cuts are computed on the
// device from the batch's lengths: a captured graph replays with new ones. A
// segment that crosses a cut is merged by the last of its CTAs to finish
// (ticket, no waiting), its pieces in ascending order: results do not depend
// on the order of execution.
//
// A tile is 16 or 32 keys for each of the CTA's warps. A warp fetches its keys
// and values into a ring of its own, kStages tiles ahead and across segment
// borders, and shares nothing with the other warps until the segment's end,
// where the warps' m, l and o merge in shared memory. (Independent warps, each
// with a range of the line and a warp that copies for all, were slower: 430
// instead of 363 us over 64 long sequences, 19 instead of 8 over a short one,
// whose pieces are then eight times as many to merge.) It fetches them as TMA
// boxes of 8 to 32 keys by 128 bytes, swizzled. (Pages that are not a
// multiple of 8 keys go by 16-byte asynchronous copies: twice the
// instructions in all, which is what bounds two warps per scheduler. Bulk
// copies of single rows, 256 or 512 bytes, were bound by the copy unit, about
// 35 cycles each.)
//
// Arithmetic. The tiles are transposed (S^T = K Q^T, O^T = V^T P^T), so that
// the 16 of the MMA are keys and dimensions and the 8 are query rows: decode
// has 1 to 8 rows per kv head (GQA), and rows beyond that would be padding.
//   F32   m16n8k8 on tf32 pairs: x = hi + lo with hi rounded to 11 bits, three
//         products (lo hi, hi lo, hi hi), 2^-21 relative.
//   F16   m16n8k16; keys and values are exact, queries (each row scaled by a
//         power of two to 2^14) and probabilities (times 2^14) are pairs of
//         f16, 22 bits, two products.
//   BF16  m16n8k16; queries and probabilities are three bf16, 24 bits, three
//         products.
// Keys are fragments by ldmatrix, values by its transposed form (16 bit) or
// by 128-bit loads with keys and dims permuted (F32), without bank conflicts.
// The probabilities of a tile turn from S^T's accumulator layout into B
// fragments by shuffles (F32) or movmatrix (16 bit), without shared memory.
//
// Rows that meet a NaN or an infinity are recomputed in plain f32 over the
// keys that they see alone (the MMA multiplies masked values by zero, and the
// split of an infinity is NaN), until a score of NaN or +infinity ends them. One
// infinite value in each of 64 sequences of 3000 keys makes 0.25 ms 8.9 ms, one
// NaN among the keys 0.29 ms.
//
// Bound by HBM over long sequences: 64 of 300 to 16000 keys in bf16 (1.97 GB)
// 334 us, 5.9 TB/s; 8 of 1000 to 8000 in f32 (282 MB) 55 us, 5.1 TB/s; heads
// of 64 f32, 64 sequences (1.09 GB), 182 us, 6.0 TB/s. Short segments are
// bound by latency: with 8 warps an SM three of four issue slots are empty, a
// segment's start and end (queries, merge, result) cost about 5000 cycles and
// a tile of 256 keys 4500. One sequence of 512 keys takes 8.0 us, a launch
// chain of dependent reads.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.cuh"
#include "tma.cuh"

namespace slc {
namespace k {
namespace {

constexpr int kRows = 8;

template <typename T, int DP>
struct Cfg {
    static constexpr bool kHalf = sizeof(T) == 2;
    // CTAs per SM: the warps wait for latencies, not for a unit (3 in 4 issue
    // slots are empty), so two are better where registers (128 a thread) and
    // shared memory allow it. Heads of 64: 64 sequences of 8 kv heads in f32
    // up to 8000 long 249 -> 182 us, up to 600 41 -> 35 us, f16 136 -> 126 us;
    // one short sequence 7.9 -> 8.4 us. For 128, two of four warps each gain
    // 1 % over long sequences in bf16 and lose 2 to 6 % over short ones, and
    // with half the keys a tile the 16-bit types take 1.4 times as long.
    static constexpr int kCtas = DP == 64 ? 2 : 1;
    static constexpr int kWarps = !kHalf && DP == 256 ? 4 : 8;
    static constexpr int kThreads = kWarps * 32;
    // 16 keys an MMA; two of them a tile give a warp independent work to
    // overlap and halve the rest (16-bit rows fit twice).
    static constexpr int kSub = kHalf && DP <= 128 ? 2 : 1;
    static constexpr int kWarpKeys = 16 * kSub;
    static constexpr int kTileKeys = kWarps * kWarpKeys;
    static constexpr int kTerms = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;  // of a query or probability
    static constexpr int kShift = std::is_same<T, __half>::value ? 14 : 0;        // f16: scaled by 2^14
    static constexpr int kEpl = 16 / (int)sizeof(T);  // elements of 16 bytes
    static constexpr int kLpr = DP / kEpl;             // 16-byte pieces of a cache row
    static constexpr int kBlk = DP * (int)sizeof(T) / 128;      // 128-byte blocks of one
    static constexpr int kHalfStage = kBlk * kWarpKeys * 128;  // keys, or values: [block][key][128 bytes]
    static constexpr int kStageBytes = 2 * kHalfStage;
    static constexpr int kMergeStride = DP + 4;  // floats
    static constexpr int kQBytes = kRows * DP * (kHalf ? 2 * kTerms : 8);
    static constexpr int kFixed = kQBytes + kWarps * kRows * (kMergeStride + 2) * 4 + 1024 + 1024;
    static constexpr int kFit = ((kCtas == 1 ? 224 : 113) * 1024 - kFixed) / (kWarps * kStageBytes);
    static constexpr int kStages = kFit > 4 ? 4 : kFit;
    static constexpr int kSmem = kFixed + kStages * kWarps * kStageBytes;
};

// Segment and tile of a unit of the work line, walked forward (kTile: keys of
// a tile).
template <int kTile>
struct Cursor {
    long long left;  // units of this sequence from the current one on, itself included
    int b;           // sequence
    int tok0, ntok, past;
    // Key indexes run over positions [0, sink) and from `low` on, both widened
    // to whole boxes; visible are those below `sinks` and from `from` on.
    int sink, low, from, keys;
    int tiles, kvh, rb, tile;
};

template <int kTile>
__device__ __forceinline__ void seq_load(const PagedPass &p, int unit, int b, Cursor<kTile> &c) {
    c.b = b;
    if (p.prefix_pass) {
        // The first with tokens: its table row. Mostly sequence 0: one read
        // instead of a chain of them.
        c.b = p.a.batch.starts[1] ? 0 : paged_sequence_of(p.a.batch, 0);
        c.tok0 = 0;
        c.ntok = (int)p.a.batch.starts[p.a.batch.seqs];
        c.past = p.a.prefix;
        c.sink = c.low = c.from = 0;
        c.keys = p.a.prefix;
    } else {
        c.tok0 = (int)p.a.batch.starts[b];
        c.ntok = (int)p.a.batch.starts[b + 1] - c.tok0;
        if ((long long)c.ntok * (p.a.heads / p.a.kv_heads) > p.small_rows) c.ntok = 0;
        c.past = (int)p.a.batch.past[b];
        c.sink = 0;
        c.from = p.first;
        if (p.a.window) c.from = max(c.past + 1 - p.a.window, 0);
        c.low = c.from - c.from % unit;
        if (p.a.window) {
            c.sink = (min(p.a.sinks, c.from) + unit - 1) / unit * unit;
            if (c.sink >= c.low) c.sink = c.low = 0;
        }
        c.keys = c.sink + c.past + c.ntok - c.low;
    }
    c.tiles = c.ntok > 0 ? (c.keys + kTile - 1) / kTile : 0;
}
template <int kTile>
__device__ __forceinline__ long long seq_units(const PagedPass &p, const Cursor<kTile> &c) {
    const long long rb = (c.ntok * (long long)(p.a.heads / p.a.kv_heads) + kRows - 1) / kRows;
    return c.ntok > 0 ? rb * p.a.kv_heads * (c.tiles + 1) : 0;
}

// Places the cursor on the tile at unit `at` counted from the start of sequence
// c.b, or on the next one where that unit is a segment's end. Returns the units
// passed over.
template <int kTile>
__device__ __forceinline__ int cursor_at(const PagedPass &p, int unit, Cursor<kTile> &c, long long at) {
    const int seqs = p.prefix_pass ? 1 : p.a.batch.seqs;
    long long n = seq_units(p, c), seg;
    for (int passed = 0;; passed++, at++) {
        while (!p.prefix_pass && at >= n && c.b + 1 < seqs) {
            at -= n;
            seq_load(p, unit, c.b + 1, c);
            n = seq_units(p, c);
        }
        seg = at / (c.tiles + 1);
        c.tile = (int)(at - seg * (c.tiles + 1));
        if (c.tile < c.tiles || at >= n) {
            c.left = n - at;
            c.rb = (int)(seg / p.a.kv_heads);
            c.kvh = (int)(seg - (long long)c.rb * p.a.kv_heads);
            return passed;
        }
    }
}

// To the next tile: a unit on, at a segment's end two.
template <int kTile>
__device__ __forceinline__ void cursor_next(const PagedPass &p, int unit, Cursor<kTile> &c) {
    const bool ends = ++c.tile == c.tiles;
    c.left -= ends ? 2 : 1;
    if (!ends) return;
    if (c.left == 0) {
        cursor_at(p, unit, c, seq_units(p, c));
        return;
    }
    c.tile = 0;
    if (++c.kvh == p.a.kv_heads) {
        c.kvh = 0;
        c.rb++;
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
__device__ __forceinline__ uint32_t tf32_hi(float x) { return (__float_as_uint(x) + 0x1000u) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf32_lo(float x, uint32_t hi) {
    return __float_as_uint(x - __uint_as_float(hi));
}
template <typename T>
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (std::is_same<T, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool kTrans>
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    if (kTrans)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// (a, b) rounded to a pair of T, a in the low half; a and b become what is left.
template <typename T>
__device__ __forceinline__ uint32_t take_pair(float &a, float &b) {
    if (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        a -= f.x;
        b -= f.y;
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const uint32_t w = *reinterpret_cast<const uint32_t *>(&h);
    a -= __uint_as_float(w << 16);
    b -= __uint_as_float(w & 0xffff0000u);
    return w;
}

// Position of compressed key index i.
template <int kTile>
__device__ __forceinline__ int key_pos(const Cursor<kTile> &c, int i) {
    return i < c.sink ? i : i - c.sink + c.low;
}
// Whether row position `at` sees key index i.
template <int kTile>
__device__ __forceinline__ bool sees(const PagedPass &p, const Cursor<kTile> &c, int i, int at) {
    if (i >= c.keys) return false;
    if (p.prefix_pass) return true;
    const int pos = key_pos(c, i);
    return pos <= at && pos >= p.first && (!p.a.window || pos > at - p.a.window || pos < p.a.sinks);
}
// Whether every row of the segment sees every key of [i0, i1).
template <int kTile>
__device__ __forceinline__ bool all_see(const PagedPass &p, const Cursor<kTile> &c, int i0, int i1) {
    if (p.prefix_pass) return i1 <= c.keys;
    if (i1 > c.keys - (c.ntok - 1)) return false;
    const int from = p.a.window ? max(c.past + c.ntok - p.a.window, c.from) : c.from;
    return i0 >= c.sink + from - c.low || (i1 <= max(c.sink, c.from) && i1 <= p.a.sinks);
}

struct PassArgs {
    PagedPass pass;
    CUtensorMap map;
    int unit;  // keys per box (paged_boxes); 1: no boxes
};

template <typename T, int DP>
__global__ void __launch_bounds__(Cfg<T, DP>::kThreads, Cfg<T, DP>::kCtas)
    paged_attention_kernel(const __grid_constant__ PassArgs args) {
    const PagedPass &p = args.pass;
    const int unit = args.unit;
    using C = Cfg<T, DP>;
    using Cur = Cursor<C::kTileKeys>;
    constexpr int kWarps = C::kWarps, kThreads = C::kThreads, kTileKeys = C::kTileKeys, S = C::kStages;
    constexpr int kWarpKeys = C::kWarpKeys, kSub = C::kSub;
    constexpr int NT = DP / 16;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char *ring = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    unsigned char *q_s = ring + S * kWarps * C::kStageBytes;            // fragments of the queries
    float *mo = reinterpret_cast<float *>(q_s + C::kQBytes);           // [kWarps][kRows][kMergeStride]
    float *mml = mo + kWarps * kRows * C::kMergeStride;                 // [kWarps][kRows][2]
    float *row_ml = mml + kWarps * kRows * 2;                           // [kRows][2]
    float *q_scale = row_ml + kRows * 2;                                // [kRows]
    long long *sums = reinterpret_cast<long long *>(q_scale + kRows);   // [kWarps]
    int *last_s = reinterpret_cast<int *>(sums + kWarps), *bad_s = last_s + 1;  // bad_s: bit per row
    long long *found = sums + kWarps + 1;                               // [2]
    uint64_t *bars = reinterpret_cast<uint64_t *>(found + 2);           // [kWarps][S][2] keys, values landed
    volatile int *abort = reinterpret_cast<int *>(bars + kWarps * S * 2);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int D = p.a.head_dim, H = p.a.heads, Hkv = p.a.kv_heads, G = H / Hkv;
    const int seqs = p.prefix_pass ? 1 : p.a.batch.seqs;

    pdl_trigger();

    // The work line: every thread adds up a run of sequences; a scan over the
    // threads finds the run in which this CTA's share begins.
    const int per = (seqs + kThreads - 1) / kThreads;
    long long mine = 0;
    for (int i = 0; i < per; i++) {
        const int b = threadIdx.x * per + i;
        if (b < seqs) {
            Cur c;
            seq_load(p, unit, b, c);
            mine += seq_units(p, c);
        }
    }
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) sums[warp] = upto;
    __syncthreads();
    long long U = 0;
    for (int w = 0; w < kWarps; w++) {
        if (w < warp) upto += sums[w];
        U += sums[w];
    }
    const long long grid = min((long long)gridDim.x, U);
    if (blockIdx.x >= grid) {
        pdl_wait();
        return;
    }
    const long long u0 = U * blockIdx.x / grid, u1 = U * (blockIdx.x + 1) / grid;
    if (upto - mine <= u0 && u0 < upto) {
        found[0] = threadIdx.x;
        found[1] = upto - mine;
    }
    if (threadIdx.x == 0) {
        *bad_s = 0;
        *abort = 0;
        for (int i = 0; i < kWarps * S * 2; i++) mbar_init(&bars[i], 1);
        fence_mbar_init();
    }
    __syncthreads();
    Cur cc, pc;  // consumer and producer
    seq_load(p, unit, (int)found[0] * per, cc);
    long long u = u0 + cursor_at(p, unit, cc, u0 - found[1]), pu = u;  // their units
    pc = cc;
    if (u >= u1) {  // nothing but a segment's end
        pdl_wait();
        return;
    }
    // The producer's unit: lane b holds the table entry and the place in its
    // page of box b of the warp's keys, or, without boxes, lane r those of key
    // r (modulo the keys); read a tile before their use.
    uint64_t *bar = bars + warp * S * 2;
    uint32_t next_id = 0;
    int next_in = -1;  // -1: past the segment's keys
    auto look_up = [&] {
        const int k = unit > 1 ? lane * unit : lane % kWarpKeys, i = pc.tile * kTileKeys + warp * kWarpKeys + k;
        next_in = -1;
        if (k < kWarpKeys && i < pc.keys) {
            const int pos = key_pos(pc, i), pg = page_of(p.a.cache, pos);
            next_in = pos - pg * p.a.cache.page;
            next_id = pg < p.a.batch.per_seq ? p.a.batch.table[(long long)pc.b * p.a.batch.per_seq + pg] : ~0u;
        }
    };
    const int head_bytes = D * (int)sizeof(T);
    // Copies the warp's keys of the producer's unit into a stage, or its
    // values. (checked on the host: page ids; see paged_row)
    auto issue = [&](int stage, int parity) {
        unsigned char *st = ring + (warp * S + stage) * C::kStageBytes + parity * C::kHalfStage;
        if (next_in >= 0 && next_id >= (uint32_t)p.a.cache.pages) {
            report_error(p.a.err, kErrGatherId);
            next_id = 0;
        }
        if (unit > 1) {
            if (__any_sync(0xffffffffu, *abort)) return;
            uint64_t *full = bar + 2 * stage + parity;
            const int count = __popc(__ballot_sync(0xffffffffu, next_in >= 0));
            if (lane == 0) mbar_arrive_expect_tx(full, count * unit * 128 * C::kBlk);
            __syncwarp();
            if (next_in >= 0)
#pragma unroll
                for (int y = 0; y < C::kBlk; y++)
                    tma_load_5d(st + (y * kWarpKeys + lane * unit) * 128, &args.map, y * (128 / (int)sizeof(T)), pc.kvh,
                                next_in, parity, (int)next_id, full);
            return;
        }
        // Zeros for rows past the segment's keys and for dims past head_dim.
        long long off = -1;
        if (next_in >= 0)
            off = next_id * p.a.cache.page_stride + next_in * p.a.cache.row_stride + (long long)pc.kvh * head_bytes;
        const char *base = p.a.cache.base + (parity ? p.a.cache.parity_stride : 0);
#pragma unroll 2
        for (int x = 0; x < kWarpKeys * C::kLpr / 32; x++) {
            const int r = (x * 32 + lane) / C::kLpr, c = (x * 32 + lane) % C::kLpr;
            const long long o = __shfl_sync(0xffffffffu, off, r);
            const bool live = o >= 0 && c * 16 < head_bytes;
            cp_async16_zfill(st + (c / 8 * kWarpKeys + r) * 128 + ((c % 8) ^ (r & 7)) * 16,
                             base + (live ? o + c * 16 : 0), live ? 16 : 0);
        }
        cp_async_commit();
    };
    auto landed = [&](int stage, int parity, int phase) {
        if (unit > 1)
            mbar_wait(bar + 2 * stage + parity, phase, p.a.err, abort);
        else
            cp_async_wait<2 * S - 1>();
        __syncwarp();
    };
    if (unit > 1 && threadIdx.x == 0) prefetch_tensormap(&args.map);
    look_up();   // lengths and tables come from uploads alone,
    pdl_wait();  // q and the cache from earlier kernels; workspace use may overlap none
    auto advance = [&] {
        pu += pc.tile + 1 == pc.tiles ? 2 : 1;
        if (pu < u1) {
            cursor_next(p, unit, pc);
            look_up();
        }
    };
    for (int i = 0; i < S; i++) {
        if (pu < u1) {
            issue(i, 0);
            issue(i, 1);
            advance();
        } else if (unit == 1) {  // one group a half, empty ones at the end
            cp_async_commit();
            cp_async_commit();
        }
    }

    // Queries of a segment, a warp per row: read a tile before they are used,
    // then put into fragment order.
    constexpr int kOwn = kRows / kWarps, kItems = (kRows * DP / 4 + kThreads - 1) / kThreads;
    float qv[kOwn][DP / 32];
    auto load_q = [&](const Cur &c) {
#pragma unroll
        for (int x = 0; x < kOwn; x++) {
            const int row = c.rb * kRows + warp + x * kWarps, tok = row / G;
            const float *q = p.a.q + ((size_t)(c.tok0 + tok) * H + c.kvh * G + (row - tok * G)) * D;
#pragma unroll
            for (int y = 0; y < DP / 32; y++) {
                const int d = lane + 32 * y;
                qv[x][y] = tok < c.ntok && d < D ? q[d] : 0.f;
            }
        }
    };
    auto stage_q = [&] {
#pragma unroll
        for (int o = 0; o < kOwn; o++) {
            const int r = warp + o * kWarps;
            float(&v)[DP / 32] = qv[o];
            float f = p.scale_log2;
            if (C::kShift) {
                float top = 0.f;
#pragma unroll
                for (int y = 0; y < DP / 32; y++) top = fmaxf(top, fabsf(v[y]));
                const int ex = scale_exponent(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
                f *= pow2(ex - C::kShift);
#pragma unroll
                for (int y = 0; y < DP / 32; y++) v[y] *= pow2(C::kShift - ex);
            }
            if (lane == 0) q_scale[r] = f;
#pragma unroll
            for (int y = 0; y < DP / 32; y++) {
                const int d = lane + 32 * y, j = d / 16, k = d % 16;
                if (C::kHalf) {
                    // k step j, lane (r, t): b0 = dims 2t, 2t + 1, b1 = 8 + 2t, ...
                    T *dst = reinterpret_cast<T *>(q_s) + (j * C::kTerms * 32 + r * 4 + (k % 8) / 2) * 4 + k / 8 * 2 +
                             k % 2;
#pragma unroll
                    for (int x = 0; x < C::kTerms; x++) {
                        float none = 0.f;
                        const uint32_t w = take_pair<T>(v[y], none);
                        *reinterpret_cast<uint16_t *>(dst + x * 128) = (uint16_t)w;
                    }
                } else {
                    // k step d / 8, lane (r, t): dims t and 4 + t, hi and lo.
                    float *dst = reinterpret_cast<float *>(q_s) + (d / 8 * 32 + r * 4 + d % 4) * 4 + d / 4 % 2;
                    const uint32_t hi = tf32_hi(v[y]);
                    dst[0] = __uint_as_float(hi);
                    dst[2] = __uint_as_float(tf32_lo(v[y], hi));
                }
            }
        }
    };
    load_q(cc);
    stage_q();
    __syncthreads();

    float acc[NT][4];  // O^T: dims x rows
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float qf0 = 0.f, qf1 = 0.f;  // S to log2 units, rows 2t and 2t + 1
    int at0 = 0, at1 = 0;        // their positions
    long long seg_u0 = u;        // this CTA's first unit of the current segment
    bool fresh = true;
    int stage = 0, phase = 0;
    Cur nc = cc;                 // first unit of the segment after this one
    // The outputs of a segment that this thread merges and writes: item i is
    // row r, dims d .. d + 3; what a prefix pass left for them.
    float4 pre_v[kItems];
    float2 pre_ml[kItems];
    auto item = [&](int i, int &r, int &d) {
        const int x = threadIdx.x + i * kThreads;
        r = x / (DP / 4);
        d = 4 * (x % (DP / 4));
    };
    auto out_row = [&](int r) {
        const int row = cc.rb * kRows + r, tok = row / G;
        return (size_t)(cc.tok0 + tok) * H + cc.kvh * G + (row - tok * G);
    };
    while (u < u1) {
        const bool seg_end = cc.tile == cc.tiles - 1, ends = seg_end || u + 1 == u1;
        const bool last = u + (seg_end ? 2 : 1) >= u1;  // of this CTA
        if (ends) {
            if (!last) {
                nc = cc;
                cursor_next(p, unit, nc);
                load_q(nc);
            }
            if (p.pre_o && !p.prefix_pass)
#pragma unroll
                for (int i = 0; i < kItems; i++) {
                    int r, d;
                    item(i, r, d);
                    if (r < min(kRows, cc.ntok * G - cc.rb * kRows) && d < D) {
                        pre_ml[i] = __ldcg(reinterpret_cast<const float2 *>(p.pre_ml) + out_row(r));
                        pre_v[i] = __ldcg(reinterpret_cast<const float4 *>(p.pre_o + out_row(r) * D + d));
                    }
                }
        }
        if (fresh) {
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
            qf0 = q_scale[2 * t];
            qf1 = q_scale[2 * t + 1];
        }
        landed(stage, 0, phase);
        const int w0i = cc.tile * kTileKeys + warp * kWarpKeys;
        const bool more = pu < u1, work = w0i < cc.keys;
        unsigned char *ks = ring + (warp * S + stage) * C::kStageBytes, *vs = ks + C::kHalfStage;

        // A warp past the segment's keys has no work in its last tile.
        // S^T: keys g, g + 8 x rows 2t, 2t + 1; small products apart.
        float s[kSub][4][4];
#pragma unroll
        for (int h = 0; h < kSub; h++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[h][i][j] = 0.f;
        if (work) {
            // 32 bytes of 16 keys a step: row lane % 16, 16-byte piece 2 (j % 4)
            // + lane / 16 of its 128-byte block, xored with the row.
            const uint32_t ka = smem_addr(ks) + (lane & 15) * 128, x0 = (((lane >> 4) ^ (lane & 7)) << 4);
#pragma unroll
            for (int j = 0; j < 4 * C::kBlk; j++) {
                uint32_t a[kSub][4];
#pragma unroll
                for (int h = 0; h < kSub; h++)
                    ldmatrix4<false>(ka + (j / 4 * kWarpKeys + h * 16) * 128 + (x0 ^ (j % 4 * 32)), a[h]);
                if constexpr (C::kHalf) {
#pragma unroll
                    for (int x = 0; x < C::kTerms; x++) {
                        const uint2 b = reinterpret_cast<const uint2 *>(q_s)[(j * C::kTerms + x) * 32 + lane];
#pragma unroll
                        for (int h = 0; h < kSub; h++) mma_16<T>(s[h][x], a[h], b.x, b.y);
                    }
                } else {
                    const float4 b = reinterpret_cast<const float4 *>(q_s)[j * 32 + lane];
                    const uint32_t h0 = __float_as_uint(b.x), h1 = __float_as_uint(b.y);
#pragma unroll
                    for (int h = 0; h < kSub; h++) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            const float f = __uint_as_float(a[h][z]);
                            hi[z] = tf32_hi(f);
                            lo[z] = tf32_lo(f, hi[z]);
                        }
                        mma_tf32(s[h][2 + (j & 1)], hi, __float_as_uint(b.z), __float_as_uint(b.w));
                        mma_tf32(s[h][j & 1], hi, h0, h1);
                        mma_tf32(s[h][2 + (j & 1)], lo, h0, h1);
                    }
                }
            }
        }
        // The keys are read: their slot takes those of S tiles on.
        __syncwarp();
        if (more)
            issue(stage, 0);
        else if (unit == 1)
            cp_async_commit();

        float pr[kSub][4], f0, f1;
        bool clear;
        if (work) {
#pragma unroll
            for (int h = 0; h < kSub; h++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    pr[h][j] =
                        ((s[h][3][j] + s[h][2][j]) + (s[h][1][j] + s[h][0][j])) * ((j & 1) ? qf1 : qf0);
            clear = all_see(p, cc, w0i, w0i + kWarpKeys);
            if (!clear)
#pragma unroll
                for (int h = 0; h < kSub; h++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (!sees(p, cc, w0i + h * 16 + g + j / 2 * 8, (j & 1) ? at1 : at0)) pr[h][j] = -INFINITY;
            float n0 = fmaxf(pr[0][0], pr[0][2]), n1 = fmaxf(pr[0][1], pr[0][3]);
            if (kSub == 2) {
                n0 = fmaxf(n0, fmaxf(pr[kSub - 1][0], pr[kSub - 1][2]));
                n1 = fmaxf(n1, fmaxf(pr[kSub - 1][1], pr[kSub - 1][3]));
            }
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, o));
                n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, o));
            }
            n0 = fmaxf(n0, m0);
            n1 = fmaxf(n1, m1);
            const float u_0 = n0 == -INFINITY ? 0.f : n0, u_1 = n1 == -INFINITY ? 0.f : n1;
            f0 = ex2(m0 - u_0);
            f1 = ex2(m1 - u_1);
            l0 *= f0;
            l1 *= f1;
            m0 = n0;
            m1 = n1;
#pragma unroll
            for (int h = 0; h < kSub; h++) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    // The distance first: of scores past 2^24 it is exact, u less kShift is not.
                    const float d = pr[h][j] - ((j & 1) ? u_1 : u_0);
                    pr[h][j] = ex2(C::kShift ? d + C::kShift : d);
                }
                l0 += pr[h][0] + pr[h][2];
                l1 += pr[h][1] + pr[h][3];
            }
        }
        landed(stage, 1, phase);
        if (work) {
            if (!clear && unit > 1) {
                // Values of keys that no row sees may be anything, and meet zero
                // probabilities: they become zero.
                const unsigned dead = __ballot_sync(0xffffffffu, lane < kWarpKeys && !live_key(p, cc, w0i + lane));
                constexpr int kPieces = C::kBlk * 8, kStep = kPieces < 32 ? 32 / kPieces : 1;  // lanes: pieces, rows
                const int c = lane % kPieces;
#pragma unroll
                for (int r0 = 0; r0 < kWarpKeys; r0 += kStep) {
                    const int r = r0 + (kPieces < 32 ? lane / kPieces : 0);
                    if ((dead >> r) & 1)
                        for (int x = c; x < kPieces; x += 32)
                            *reinterpret_cast<uint4 *>(vs + (x / 8 * kWarpKeys + r) * 128 + x % 8 * 16) =
                                make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();
                __syncwarp();
            }

            // A tile's P V starts from zero and is added to the running output
            // outside the tensor core, whose accumulation truncates: over
            // thousands of keys that bias would grow past f32 rounding.
            if constexpr (C::kHalf) {
                // B fragments: row g, keys 2t, 2t + 1 and 8 + 2t, 9 + 2t.
                uint32_t b[kSub][C::kTerms][2];
#pragma unroll
                for (int x = 0; x < C::kTerms; x++)
#pragma unroll
                    for (int h = 0; h < kSub; h++) {
                        b[h][x][0] = movmatrix(take_pair<T>(pr[h][0], pr[h][1]));
                        b[h][x][1] = movmatrix(take_pair<T>(pr[h][2], pr[h][3]));
                    }
                // Key lane % 8 + 8 (lane / 16), 16-byte piece 2 (i % 4) + lane / 8 % 2.
                const uint32_t va = smem_addr(vs) + ((lane & 7) + (lane >> 4) * 8) * 128,
                               x0 = ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < kSub; h++) {
                        uint32_t a[4];
                        ldmatrix4<true>(va + (i / 4 * kWarpKeys + h * 16) * 128 + (x0 ^ (i % 4 * 32)), a);
#pragma unroll
                        for (int x = C::kTerms - 1; x >= 0; x--) mma_16<T>(o, a, b[h][x][0], b[h][x][1]);
                    }
                    acc[i][0] = fmaf(acc[i][0], f0, o[0]);
                    acc[i][1] = fmaf(acc[i][1], f1, o[1]);
                    acc[i][2] = fmaf(acc[i][2], f0, o[2]);
                    acc[i][3] = fmaf(acc[i][3], f1, o[3]);
                }
            } else {
                // B fragments of the two 8-key steps: row g, keys 2t and 2t + 1.
                uint32_t bh[2][2], bl[2][2];
#pragma unroll
                for (int k8 = 0; k8 < 2; k8++)
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const int src = (2 * t + x) * 4 + (g >> 1);
                        const float a = __shfl_sync(0xffffffffu, pr[0][2 * k8], src);
                        const float b = __shfl_sync(0xffffffffu, pr[0][2 * k8 + 1], src);
                        const float v = (g & 1) ? b : a;
                        bh[k8][x] = tf32_hi(v);
                        bl[k8][x] = tf32_lo(v, bh[k8][x]);
                    }
#pragma unroll
                for (int j = 0; j < DP / 32; j++) {
                    float o[2][4] = {};
#pragma unroll
                    for (int k8 = 0; k8 < 2; k8++) {
                        float va[4], vb[4];
                        const unsigned char *v0 = vs + (j * kWarpKeys + 8 * k8 + 2 * t) * 128;
                        Frag<T>::ld(v0 + ((g ^ (2 * t)) << 4), va);
                        Frag<T>::ld(v0 + 128 + ((g ^ (2 * t + 1)) << 4), vb);
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const float f[4] = {va[2 * x], va[2 * x + 1], vb[2 * x], vb[2 * x + 1]};
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int z = 0; z < 4; z++) {
                                hi[z] = tf32_hi(f[z]);
                                lo[z] = tf32_lo(f[z], hi[z]);
                            }
                            mma_tf32(o[x], hi, bl[k8][0], bl[k8][1]);
                            mma_tf32(o[x], lo, bh[k8][0], bh[k8][1]);
                            mma_tf32(o[x], hi, bh[k8][0], bh[k8][1]);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        float(&a)[4] = acc[2 * j + x];
                        a[0] = fmaf(a[0], f0, o[x][0]);
                        a[1] = fmaf(a[1], f1, o[x][1]);
                        a[2] = fmaf(a[2], f0, o[x][2]);
                        a[3] = fmaf(a[3], f1, o[x][3]);
                    }
                }
            }
        }
        __syncwarp();
        if (more) {
            issue(stage, 1);
            advance();
        } else if (unit == 1) {
            cp_async_commit();
        }
        if (++stage == S) {
            stage = 0;
            phase ^= 1;
        }

        if (!ends) {
            cc.tile++;
            cc.left--;
            u++;
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
            if (C::kHalf) {  // tile i: dims 16 i + g and 16 i + 8 + g
                w0[16 * i + g] = acc[i][0];
                w1[16 * i + g] = acc[i][1];
                w0[16 * i + 8 + g] = acc[i][2];
                w1[16 * i + 8 + g] = acc[i][3];
            } else {  // dims 32 (i / 2) + 4 g + 2 (i % 2) and the next
                const int d = i / 2 * 32 + 4 * g + i % 2 * 2;
                *reinterpret_cast<float2 *>(w0 + d) = make_float2(acc[i][0], acc[i][2]);
                *reinterpret_cast<float2 *>(w1 + d) = make_float2(acc[i][1], acc[i][3]);
            }
        }
        m0 -= C::kShift;  // l and o are 2^kShift times as large
        m1 -= C::kShift;
        if (g == 0) {
            float *ml = mml + (warp * kRows + 2 * t) * 2;
            ml[0] = m0, ml[1] = l0, ml[2] = m1, ml[3] = l1;
        }
        __syncthreads();  // q_s is free from here on
        const int rows = min(kRows, cc.ntok * G - cc.rb * kRows);
        float4 o[kItems];
        float mm[kItems], ll[kItems];
#pragma unroll
        for (int i = 0; i < kItems; i++) {
            o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            mm[i] = -INFINITY;
            ll[i] = 0.f;
        }
        auto add = [&](int i, float m, float l, float4 v) {  // to an item's running sums
            const float nm = fmaxf(mm[i], m), mu = nm == -INFINITY ? 0.f : nm;
            const float f = ex2(mm[i] - mu), e = ex2(m - mu);
            ll[i] = fmaf(l, e, ll[i] * f);
            o[i].x = fmaf(v.x, e, o[i].x * f);
            o[i].y = fmaf(v.y, e, o[i].y * f);
            o[i].z = fmaf(v.z, e, o[i].z * f);
            o[i].w = fmaf(v.w, e, o[i].w * f);
            mm[i] = nm;
        };
#pragma unroll
        for (int i = 0; i < kItems; i++) {
            int r, d;
            item(i, r, d);
            if (r >= rows || d >= D) continue;
            for (int w = 0; w < kWarps; w++) mm[i] = fmaxf(mm[i], mml[(w * kRows + r) * 2]);
            const float mu = mm[i] == -INFINITY ? 0.f : mm[i];
            bool odd = false;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float mw = mml[(w * kRows + r) * 2], lw = mml[(w * kRows + r) * 2 + 1], f = ex2(mw - mu);
                const float4 x = *reinterpret_cast<const float4 *>(mo + (w * kRows + r) * C::kMergeStride + d);
                ll[i] = fmaf(lw, f, ll[i]);
                o[i].x = fmaf(x.x, f, o[i].x);
                o[i].y = fmaf(x.y, f, o[i].y);
                o[i].z = fmaf(x.z, f, o[i].z);
                o[i].w = fmaf(x.w, f, o[i].w);
                odd |= !(mw < INFINITY);
            }
            odd |= !finite(ll[i]) || !finite(o[i].x) || !finite(o[i].y) || !finite(o[i].z) || !finite(o[i].w);
            if (odd) atomicOr(bad_s, 1 << r);
        }
        if (!last) stage_q();
        __syncthreads();
        if (const int bad = *bad_s) {
            // Plain f32 over the visible keys of the piece, a warp per row.
            const int k0 = (cc.tile - (int)(u - seg_u0)) * kTileKeys;
            const int k1 = min(cc.keys, (cc.tile + 1) * kTileKeys);
            for (int r = warp; r < rows; r += kWarps) {
                if (!((bad >> r) & 1)) continue;
                const int at = cc.past + (cc.rb * kRows + r) / G;
                float m, l, v[DP / 32];
                plain_row<T, DP>(
                    p, p.a.q + out_row(r) * D, cc.b, cc.kvh, k0, k1,
                    [&](int i) { return sees(p, cc, i, at) ? key_pos(cc, i) : -1; }, m, l, v);
#pragma unroll
                for (int y = 0; y < DP / 32; y++) mo[r * C::kMergeStride + lane + 32 * y] = v[y];
                if (lane == 0) {
                    row_ml[2 * r] = m;
                    row_ml[2 * r + 1] = l;
                }
            }
            __syncthreads();
            if (threadIdx.x == 0) *bad_s = 0;
#pragma unroll
            for (int i = 0; i < kItems; i++) {
                int r, d;
                item(i, r, d);
                if (r >= rows || !((bad >> r) & 1)) continue;
                o[i] = *reinterpret_cast<const float4 *>(mo + r * C::kMergeStride + d);
                mm[i] = row_ml[2 * r];
                ll[i] = row_ml[2 * r + 1];
            }
            __syncthreads();
        }

        // ---- the segment's result, or a piece of it for the merge.
        const long long a0 = u - cc.tile, a1 = a0 + cc.tiles;  // the segment's tiles
        bool write = true;
        if (a0 < u0 || a1 > u1) {
            const int c_first = (int)(((a0 + 1) * grid - 1) / U), c_last = (int)((a1 * grid - 1) / U);
            const int slot = 2 * blockIdx.x + (a0 >= u0 ? 1 : 0);
#pragma unroll
            for (int i = 0; i < kItems; i++) {
                int r, d;
                item(i, r, d);
                if (r >= rows || d >= D) continue;
                *reinterpret_cast<float4 *>(p.part_o + ((size_t)slot * kRows + r) * DP + d) = o[i];
                if (d == 0)
                    reinterpret_cast<float2 *>(p.part_ml)[(size_t)slot * kRows + r] = make_float2(mm[i], ll[i]);
            }
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
#pragma unroll
                for (int i = 0; i < kItems; i++) {
                    int r, d;
                    item(i, r, d);
                    if (r >= rows || d >= D) continue;
                    mm[i] = -INFINITY;
                    ll[i] = 0.f;
                    o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    // Eight pieces in flight, added in ascending order.
                    for (int x = c_first; x <= c_last; x += 8) {
                        float2 ml[8];
                        float4 v[8];
#pragma unroll
                        for (int y = 0; y < 8; y++) {
                            const size_t sl = 2 * (size_t)min(x + y, c_last) + (x + y == c_first ? 1 : 0);
                            ml[y] = __ldcg(reinterpret_cast<const float2 *>(p.part_ml) + sl * kRows + r);
                            v[y] = __ldcg(reinterpret_cast<const float4 *>(p.part_o + (sl * kRows + r) * DP + d));
                        }
#pragma unroll
                        for (int y = 0; y < 8; y++)
                            if (x + y <= c_last) add(i, ml[y].x, ml[y].y, v[y]);
                    }
                }
            }
            __syncthreads();  // last_s is read
        }
        if (write) {
#pragma unroll
            for (int i = 0; i < kItems; i++) {
                int r, d;
                item(i, r, d);
                if (r >= rows || d >= D) continue;
                const size_t at = out_row(r);
                if (p.prefix_pass) {
                    *reinterpret_cast<float4 *>(p.pre_o + at * D + d) = o[i];
                    if (d == 0) *reinterpret_cast<float2 *>(p.pre_ml + at * 2) = make_float2(mm[i], ll[i]);
                    continue;
                }
                if (p.pre_o) add(i, pre_ml[i].x, pre_ml[i].y, pre_v[i]);
                float *dst = p.a.out + at * D + d;  // 4-byte aligned
                dst[0] = __fdiv_rn(o[i].x, ll[i]);
                dst[1] = __fdiv_rn(o[i].y, ll[i]);
                dst[2] = __fdiv_rn(o[i].z, ll[i]);
                dst[3] = __fdiv_rn(o[i].w, ll[i]);
            }
        }
        fresh = true;
        cc = nc;
        u += seg_end ? 2 : 1;
    }
    // After a wait that gave up, copies may still be in flight: let them land
    // before the CTA's shared memory is released.
    if (unit > 1 && *abort && lane == 0)
        for (int i = 0; i < 2 * S; i++) {
            const uint64_t t0 = global_ns();
            while (!mbar_try_wait(bar + i, phase ^ (i / 2 < stage)) && global_ns() - t0 < 100000000ull) {
            }
        }
}

int padded_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

constexpr size_t kPieces = 2 * 2 * kSmCount;  // two a CTA
size_t partial_floats(int dp) { return kPieces * kRows * (dp + 2); }
size_t prefix_floats(const PagedAttention &a) {
    return a.prefix ? (size_t)a.tokens * a.heads * (a.head_dim + 2) : 0;
}

template <typename T, int DP>
cudaError_t launch_pass(cudaStream_t s, const PagedPass &p) {
    using C = Cfg<T, DP>;
    static_assert(C::kStages >= 1 && C::kCtas * (C::kSmem + 1024) <= 228 * 1024, "shared layout");
    static std::atomic<uint64_t> smem_set{0};
    const cudaError_t e = set_smem_limit_once(paged_attention_kernel<T, DP>, C::kSmem, &smem_set);
    if (e != cudaSuccess) return e;
    PassArgs args{};
    args.pass = p;
    args.unit = paged_boxes(p.a, C::kWarpKeys, sizeof(T), std::is_same<T, __half>::value, true, &args.map);
    launch_k(paged_attention_kernel<T, DP>, kSmCount * C::kCtas, C::kThreads, C::kSmem, s, args);
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

// Query rows of one kv head up to which a sequence is paged_attention_kernel's,
// which reads the keys once per kRows of them; more are paged_rows.cu's.
// Measured, 16 sequences of 1000 to 4000 keys, 8 kv heads of 128, with 16, 32
// and 48 rows: f32 109, 169, 245 us here and 121, 139, 141 there; bf16 60, 90,
// 129 and 103, 107, 108. (paged_rows.cu takes heads up to 128: wider ones come
// here with any rows, 2048 tokens of 16 heads of 256 in bf16 580 us.)
int small_rows(const PagedAttention &a) { return a.cache.type == kPagedF32 ? 16 : 32; }
// Where all keys that the call's shapes allow are few, tokens in all times keys
// counted in blocks of kRows rows by a tile, it takes them whatever the rows:
// paged_rows.cu has 20 us to start up and end. 1 sequence of 38 tokens over 160
// keys (76 units) 7.2 us here and 28 there, of 128 new tokens in f32 (512) 18
// and 28, of 20 over 1000 (640) 21.6 and 20.9, of 64 over 1000 (2304) 41 and
// 30. Known from the shapes alone, so that a call gives the same results
// captured and not.
constexpr size_t kFewUnits = 1024;
bool many_rows(const PagedAttention &a, size_t new_tokens, size_t runs, size_t keys) {
    const size_t group = a.heads / a.kv_heads, tile = a.cache.type == kPagedF32 ? 128 : 256;
    if (!paged_rows_supported(a) || new_tokens * group <= (size_t)small_rows(a)) return false;
    const size_t blocks = (size_t)a.tokens * group / kRows + runs;
    return blocks * a.kv_heads * ((keys + tile - 1) / tile) > kFewUnits;
}
bool many_rows(const PagedAttention &a) {
    size_t keys = (size_t)a.batch.per_seq * a.cache.page;
    if (a.window) keys = std::min(keys, (size_t)a.window + a.sinks + a.max_new);
    return many_rows(a, a.max_new, a.batch.seqs, keys);
}
bool many_prefix_rows(const PagedAttention &a) { return a.prefix && many_rows(a, a.tokens, 1, a.prefix); }

size_t part_floats(const PagedAttention &a) {
    const size_t few = partial_floats(padded_dim(a.head_dim));
    return many_rows(a) || many_prefix_rows(a) ? std::max(few, paged_rows_part_floats(a)) : few;
}

// A pass over the shared prefix saves the others' reads of it (from L2, mostly)
// and costs launches and the merge, 4 to 15 us: it is taken where those reads
// are kPrefixPass bytes or more. Measured, with the pass and without: 64
// sequences of 8 kv heads of 128 bf16, prefix 256 (67 MB) 35 and 32 us, 512
// (134 MB) 44 and 43, 1024 49 and 61, 8192 72 and 313; 8 sequences, 1024 (34
// MB) 18 and 16, 2048 (67 MB) 19 and 21, 4096 24 and 29; 64 sequences of 4 kv
// heads of 64 f32, 777 (102 MB) 28 and 33; 6 of them (10 MB) 18 and 11. The
// border is a compromise: few sequences gain from 60 MB on, many from 150 MB,
// and between those the two differ by 2 us. Without it the rows read the pages by
// their own table rows, which are the same.
constexpr size_t kPrefixPass = (size_t)96 << 20;
size_t prefix_bytes(const PagedAttention &a) {
    const size_t row = (size_t)2 * a.kv_heads * a.head_dim * (a.cache.type == kPagedF32 ? 4 : 2);
    return (size_t)a.batch.seqs * a.prefix * row;
}
// The call without its prefix where there is no pass over it: for the reads
// that it saves, or because the workspace does not hold its results, one row
// of head_dim + 2 floats for every query row (prompts, whose passes are bound
// by the products in either case).
PagedAttention as_run(const PagedAttention &call) {
    PagedAttention a = call;
    if (prefix_bytes(a) < kPrefixPass || (part_floats(a) + prefix_floats(a)) * sizeof(float) > a.workspace_bytes)
        a.prefix = 0;
    return a;
}

}  // namespace

size_t paged_attention_workspace_bytes(const PagedAttention &call) {
    const PagedAttention a = as_run(call);
    return (part_floats(a) + prefix_floats(a)) * sizeof(float);
}

cudaError_t paged_attention(cudaStream_t s, const PagedAttention &call) {
    if (call.tokens == 0 || call.batch.seqs == 0) return cudaSuccess;
    const PagedAttention a = as_run(call);
    if (paged_attention_workspace_bytes(a) > a.workspace_bytes) return cudaErrorMemoryAllocation;
    PagedPass p{};
    p.a = a;
    p.scale_log2 = a.scale * kLog2e;
    p.part_o = static_cast<float *>(a.workspace);
    p.part_ml = p.part_o + kPieces * kRows * padded_dim(a.head_dim);
    p.small_rows = INT32_MAX;
    cudaError_t e = cudaSuccess;
    if (a.prefix) {
        p.pre_o = p.part_o + part_floats(a);
        p.pre_ml = p.pre_o + (size_t)a.tokens * a.heads * a.head_dim;
        p.prefix_pass = 1;
        e = many_prefix_rows(a) ? paged_rows(s, p) : launch_type(s, p);
        if (e != cudaSuccess) return e;
        p.prefix_pass = 0;
        p.first = a.prefix;
    }
    // Sequences with many rows first, those with few after them (a sequence
    // alone has its kernel: a launch for nothing takes 4 us).
    if (many_rows(a)) {
        p.small_rows = a.batch.seqs == 1 ? 0 : small_rows(a);
        e = paged_rows(s, p);
        if (e != cudaSuccess || a.batch.seqs == 1) return e;
    }
    return launch_type(s, p);
}

}  // namespace k
}  // namespace slc
