"""GPU tests of the paged KV-cache operators against their definitions in 64
bits (tests/paged_util.py), at the lengths, masks, layouts and contents where
they can go wrong.

Append: an F32 cache holds bit for bit what the Rope operator gives, a 16-bit
cache those values rounded to nearest; every other slot keeps its bits.

Attention: the bound, elementwise. A tf32 pair keeps x to 2^-20 (its low part
has 13 bits, of which the MMA reads 11), the product of two low parts is left
out (2^-20): a product is off by 3 * 2^-20 of its size, and a sum of D of them
in f32 by at most as much again for D <= 256 and the accumulators used: a
score's error is below ds = 8 * 2^-20 * scale * sum |q k|. A probability is
then off by a factor of exp(ds), numerator and denominator both: 2 ds of
sum p |v|. The products p v add 3 * 2^-20, the exponential 2^-22, the sums
over the keys (32 or more apart in separate accumulators, 2^-23 a step) at
most 2^-20 for 64 keys, the merges and the division the rest of 8 * 2^-20.
The split of rows and keys over CTAs changes which sums are made first, not
the bound. Rows on the tcgen05 path use f16 pairs (22 bits, inside the above)
whose smallest step is 2^-34 of a tile's largest key or value and 2^-39 of the
query's largest element: as much again, rounded up to 2^-33, times the largest
value, and times what multiplies it in a score."""
import math
import random
import time

import numpy as np
import pytest

from starlight_b200.device import (BufferRef, CudaDevice, DeviceError, DType, Op, OpCode, RopeVariant, Value,
                                   ValueRole, state_words)
from tests.gpu_util import get, new_f32, put_f32, put_u32
from tests.paged_util import HOLE, Batch, from_bits, put_at, to_bits, upload

pytestmark = pytest.mark.gpu

F32, F16, BF16 = DType.F32, DType.F16, DType.BF16


@pytest.fixture(scope="module")
def dev():
    d = CudaDevice(0)
    yield d
    d.close()


def attend(dev, b, scale=None, window=0, sinks=0, offset=0, refs=None, max_new=None, out=None):
    """PagedAttention (PrefixAttention where the batch has a prefix) over the
    batch; the output buffer holds 7.5 before."""
    scale = 1 / math.sqrt(b.dim) if scale is None else scale
    tables, cache = refs or upload(dev, b)
    x = Value.f32((b.tokens, b.heads * b.dim))
    q = put_at(dev, b.q, offset)
    out = out or put_at(dev, np.full(b.q.size, 7.5, np.float32), offset)
    new = b.max_new() if max_new is None else max_new
    code, scalars = (OpCode.PrefixAttention, [new, b.prefix]) if b.prefix else (OpCode.PagedAttention,
                                                                                [new, window, sinks])
    dev.dispatch(b.op(code, scale=scale), [q, *tables, cache], [x, *b.described(), b.state()], [out], [x], scalars)
    return get(dev, out).reshape(b.tokens, -1)


def check(got, b, scale=None, window=0, sinks=0):
    scale = 1 / math.sqrt(b.dim) if scale is None else scale
    want, tol = b.attention(scale, window, sinks)
    live = int(b.starts[-1])
    err = np.abs(got[:live] - want[:live])
    assert np.all(np.isfinite(got[:live]))
    assert np.all(err <= tol[:live]), (err / np.maximum(tol[:live], 1e-30)).max()
    assert np.all(got[live:] == 7.5)  # rows behind the last sequence


# ---------------------------------------------------------------- append ----

APPENDS = [
    dict(lens=[(0, 1)]),
    dict(lens=[(5, 1)], page=1, dim=8, kv_heads=1),
    dict(lens=[(20, 3), (0, 17), (7, 0), (33, 1)], page=5, dim=72, kv_heads=3, layers=3),
    dict(lens=[(511, 1)] * 9, page=16, dim=128, kv_heads=8, pad=4),
    dict(lens=[(3, 700), (0, 1), (90, 130)], page=64, dim=64, kv_heads=4, layers=1, layer=0),
    dict(lens=[(1, 33)], page=100, dim=256, kv_heads=2),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("variant", [RopeVariant.Neox, RopeVariant.GptJ])
@pytest.mark.parametrize("case", range(len(APPENDS)))
@pytest.mark.parametrize("offset", [0, 1])
def test_append(dev, case, dtype, variant, offset):
    b = Batch(**APPENDS[case], dtype=dtype, seed=case)
    tables, cache = upload(dev, b)
    T, kv = b.tokens, b.kv_heads * b.dim
    k, v = put_at(dev, b.k, offset), put_at(dev, b.v, offset)
    x = Value.f32((T, kv))
    for theta in (500000.0, 0.0):
        turned = b.k
        pos = np.zeros(T, np.uint32)
        for i, (p, n) in enumerate(b.lens):
            pos[b.starts[i]:b.starts[i + 1]] = p + np.arange(n)
        if theta:
            out = new_f32(dev, b.k.size)
            y = Value.f32((T, b.kv_heads, 1, b.dim))
            dev.dispatch(Op(OpCode.Rope, theta=theta, variant=variant), [k, put_u32(dev, pos)],
                         [y, Value.u32((T, 1))], [out], [y])
            turned = get(dev, out)
        dev.upload_f32(cache.buffer, b.words)
        dev.dispatch(b.append_op(theta, variant), [k, v, *tables, cache], [x, x, *b.described(), b.state()], [], [])
        got = from_bits(get(dev, cache), b.shape, dtype)
        want = b.stored.copy()
        turned, value = (to_bits(a, dtype)[0].reshape(T, b.kv_heads, b.dim) for a in (turned, b.v))
        for i, (p, n) in enumerate(b.lens):
            at = p + np.arange(n)
            where = b.table[i][at // b.page].astype(np.int64)
            rows = slice(int(b.starts[i]), int(b.starts[i + 1]))
            want[where, b.layer, 0, at % b.page] = turned[rows]
            want[where, b.layer, 1, at % b.page] = value[rows]
        assert np.array_equal(got, want, equal_nan=True)


def test_append_positions_far_out(dev):
    # Angles of positions near 2^24: the f64 path, as the Rope operator's.
    b = Batch([(0, 2)], page=1 << 23, layers=1, layer=0, kv_heads=1, heads=1, dim=8, extra_pages=0,
              width=4)
    b.past[:] = (1 << 24) - 2
    b.table[0] = [HOLE, 0, HOLE, HOLE]
    tables = [put_u32(dev, a) for a in (b.table, b.past, b.starts)]
    cache = new_f32(dev, state_words(b.shape, F32))
    k, v = put_f32(dev, b.k), put_f32(dev, b.v)
    x = Value.f32((2, 8))
    dev.dispatch(b.append_op(), [k, v, *tables, cache], [x, x, *b.described(), b.state()], [], [])
    out = new_f32(dev, 16)
    y = Value.f32((2, 1, 1, 8))
    pos = put_u32(dev, (1 << 24) - 2 + np.arange(2))
    dev.dispatch(Op(OpCode.Rope, theta=500000.0), [k, pos], [y, Value.u32((2, 1))], [out], [y])
    got = get(dev, cache).reshape(b.shape)
    assert np.array_equal(got[0, 0, 0, -2:, 0].ravel(), get(dev, out))
    assert np.array_equal(got[0, 0, 1, -2:, 0].ravel(), b.v.ravel())


# ------------------------------------------------------------- attention ----

SHAPES = [
    dict(heads=1, kv_heads=1, dim=8, page=1),
    dict(heads=4, kv_heads=4, dim=64, page=16),
    dict(heads=8, kv_heads=2, dim=128, page=16),
    dict(heads=6, kv_heads=2, dim=72, page=5),
    dict(heads=16, kv_heads=2, dim=128, page=64, layers=3),
    dict(heads=16, kv_heads=1, dim=96, page=7),
    dict(heads=71, kv_heads=1, dim=64, page=32),
    dict(heads=2, kv_heads=1, dim=256, page=16),
    dict(heads=3, kv_heads=1, dim=200, page=100, layers=1, layer=0),
]
LENGTHS = [
    [(0, 1)],
    [(1, 1), (63, 1), (64, 1), (65, 1), (500, 1)],
    [(0, 1), (130, 0), (17, 2), (15, 1), (0, 5)],
    [(40, 33), (3, 1), (0, 70)],
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", range(len(LENGTHS)))
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(dev, shape, lens, dtype):
    b = Batch(LENGTHS[lens], **SHAPES[shape], dtype=dtype, seed=10 * shape + lens, pad=lens)
    refs = upload(dev, b)
    check(attend(dev, b, offset=lens % 2, refs=refs), b)
    check(attend(dev, b, window=16, sinks=4, refs=refs), b, window=16, sinks=4)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (64, 4), (65, 63), (100, 1000), (1 << 31, 5),
                                          (400, 0)])
def test_windows_and_sinks(dev, window, sinks, dtype):
    b = Batch([(0, 1), (300, 1), (62, 9), (390, 20), (5, 130)], heads=8, kv_heads=2, dim=64, page=16, dtype=dtype)
    check(attend(dev, b, window=window, sinks=sinks), b, window=window, sinks=sinks)


@pytest.mark.parametrize("new", [1, 40])
def test_pages_behind_the_window_may_be_gone(dev, new):
    b = Batch([(200, new), (90, new)], heads=4, kv_heads=2, dim=64, page=8)
    want, tol = b.attention(0.125, 24, 3)
    for i, (p, _) in enumerate(b.lens):
        b.table[i, 1:(p + 1 - 24) // 8] = HOLE
    got = attend(dev, b, scale=0.125, window=24, sinks=3)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype,lens", [(F32, [(70000, 1)]), (BF16, [(70000, 1), (9, 1), (33333, 3)]),
                                        (F16, [(20000, 1)] * 3 + [(0, 1)] * 40)])
def test_long_sequences(dev, dtype, lens):
    b = Batch(lens, heads=4, kv_heads=1, dim=128, page=16, layers=1, layer=0, dtype=dtype)
    check(attend(dev, b), b)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 128), (8, 4, 64)])
def test_few_rows_over_many_keys(dev, dtype, heads, kv_heads, dim):
    # More rows than the kernel for few takes, in far fewer segments than CTAs.
    b = Batch([(9000, 40), (10, 2)], heads=heads, kv_heads=kv_heads, dim=dim, page=16, layers=1, layer=0, dtype=dtype)
    refs = upload(dev, b)
    check(attend(dev, b, refs=refs), b)
    check(attend(dev, b, window=3000, sinks=5, refs=refs), b, window=3000, sinks=5)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window,sinks,page", [(1, 0, 16), (7, 2, 5), (64, 4, 32), (65, 63, 8), (200, 1000, 64)])
def test_windows_of_many_rows(dev, window, sinks, page, dtype):
    b = Batch([(300, 150), (0, 200), (62, 9), (390, 120), (5, 130)], heads=16, kv_heads=8, dim=64, page=page,
              dtype=dtype, layers=1, layer=0)
    check(attend(dev, b, window=window, sinks=sinks), b, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("page", [5, 16])
def test_many_rows_over_few_keys(dev, page, dtype):
    # A table with no room for more keys: the kernel for few rows takes them.
    b = Batch([(40, 33), (3, 1), (0, 70), (100, 25)], heads=6, kv_heads=2, dim=72, page=page, dtype=dtype, pad=2,
              narrow=True)
    refs = upload(dev, b)
    check(attend(dev, b, refs=refs), b)
    check(attend(dev, b, window=20, sinks=3, refs=refs), b, window=20, sinks=3)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("past,new", [(0, 300), (1000, 1), (333, 40)])
def test_one_sequence(dev, past, new, dtype):
    # Alone in the batch, with max_new above what it has: one kernel does all.
    b = Batch([(past, new)], heads=16, kv_heads=4, dim=128, page=16, dtype=dtype, width=4096)
    check(attend(dev, b, max_new=500), b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [8, 24, 256])
def test_page_sizes(dev, page, dtype):
    b = Batch([(700, 1), (255, 2), (256, 70), (7, 1)], heads=8, kv_heads=2, dim=128, page=page, dtype=dtype)
    refs = upload(dev, b)
    check(attend(dev, b, refs=refs), b)
    check(attend(dev, b, window=100, sinks=9, refs=refs), b, window=100, sinks=9)


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("heads", [2, 40])
def test_more_sequences_than_threads(dev, heads, window):
    b = Batch([(i % 90, i % 3) for i in range(700)], heads=heads, kv_heads=2, dim=64, page=16, layers=1, layer=0)
    check(attend(dev, b, window=window, sinks=2 if window else 0), b, window=window, sinks=2 if window else 0)


def test_offsets_past_32_bits(dev):
    # A cache of more than 2^32 bytes; the sequence lives in its last pages.
    pages, page, hkv, d = 5000, 64, 8, 128
    shape = (pages, 2, 2, page, hkv, d)
    n = int(np.prod(shape))
    assert n * 4 > 1 << 32
    b = Batch([(100, 1)], heads=8, kv_heads=8, dim=128, page=page, layers=2, layer=1, extra_pages=0)
    buf = dev.allocate_f32(n)
    last = b.stored.astype(np.float32)
    per_page = n // pages
    import torch

    class Memory:
        __cuda_array_interface__ = dict(shape=(2 * per_page,), typestr="<f4", version=3,
                                        data=(dev.device_ptr(buf) + 4 * (n - 2 * per_page), False))

    dev.synchronize()
    torch.as_tensor(Memory(), device="cuda").copy_(torch.from_numpy(last.ravel()))
    torch.cuda.synchronize()
    b.table = b.table + np.uint32(pages - 2)
    b.pages, b.shape = pages, shape
    tables = [put_u32(dev, a) for a in (b.table, b.past, b.starts)]
    got = attend(dev, b, refs=(tables, BufferRef(buf, 0, n)))
    b.stored = np.zeros((0,))
    b.keys = lambda i: tuple(last[(b.table[0] - pages + 2).astype(np.int64)][:, 1, x].reshape(-1, hkv, d)[:101]
                             .astype(np.float64) for x in (0, 1))
    check(got, b)
    # Append there as well.
    x = Value.f32((1, hkv * d))
    dev.dispatch(b.append_op(theta=0.0), [put_f32(dev, b.k), put_f32(dev, b.v), *tables, BufferRef(buf, 0, n)],
                 [x, x, *b.described(), b.state()], [], [])
    dev.synchronize()
    tail = torch.as_tensor(Memory(), device="cuda").cpu().numpy().reshape(2, *shape[1:])
    at = tail[int(b.table[0, 1]) - pages + 2, 1, :, 100 - 64]
    assert np.array_equal(at[0].ravel(), b.k.ravel()) and np.array_equal(at[1].ravel(), b.v.ravel())
    dev.release(buf)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new", [1, 40])
def test_positions_near_31_bits(dev, new, dtype):
    b = Batch([(4090, new)], heads=8, kv_heads=2, dim=64, page=4096, layers=1, layer=0, dtype=dtype)
    want, tol = b.attention(0.125, 100)
    pages = (1 << 19) - 4
    table = np.full((1, pages + 2), HOLE, np.uint32)
    table[0, pages:] = b.table[0, :2]
    b.table, b.past = table, b.past + np.uint32(4096 * pages)
    got = attend(dev, b, scale=0.125, window=100)
    assert np.all(np.abs(got - want) <= tol)


# ------------------------------------------------- values out of the ordinary

def put_values(b, places):
    """Sets keys / values of (sequence, position) to given numbers."""
    for seq, pos, parity, value in places:
        b.stored[int(b.table[seq, pos // b.page]), b.layer, parity, pos % b.page] = value
    b.stored, b.words = to_bits(b.stored.astype(np.float32), b.dtype)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("heads,new", [(2, 6), (16, 40)])
def test_keys_and_values_that_a_row_does_not_see(dev, value, dtype, heads, new):
    # Position 100 + 3 is not finite: it belongs to the fourth new token, so
    # three rows of the same block must come out clean; and position 60 is
    # behind the window of the rows from 60 + 50 on.
    b = Batch([(100, new), (10, 1)], heads=heads, kv_heads=2, dim=64, page=16, dtype=dtype)
    put_values(b, [(0, 103, 0, value), (0, 103, 1, value)])
    got = attend(dev, b)
    want, tol = b.attention(0.125)
    clean = [0, 1, 2, new]  # the last: the other sequence
    assert np.all(np.abs(got[clean] - want[clean]) <= tol[clean])
    assert not np.any(np.isfinite(got[3]))
    b = Batch([(100, new)], heads=heads, kv_heads=2, dim=64, page=16, dtype=dtype)
    put_values(b, [(0, 60, 0, value), (0, 60, 1, value)])
    got = attend(dev, b, window=41 + 3)  # rows 0 .. 3 see positions > 56 .. 59, row 4 onward not 60
    want, tol = b.attention(0.125, 44)
    assert np.all(np.abs(got[4:] - want[4:]) <= tol[4:])
    assert not np.any(np.isfinite(got[:4]))


def seconds(dev, b, calls=3):
    """The shortest of a few calls over the batch, with its upload left out."""
    tables, cache = upload(dev, b)
    x = Value.f32((b.tokens, b.heads * b.dim))
    q, out = put_f32(dev, b.q), new_f32(dev, b.q.size)
    cmd = dev.command(b.op(OpCode.PagedAttention, scale=b.dim ** -0.5), [q, *tables, cache],
                      [x, *b.described(), b.state()], [out], [x], [b.max_new(), 0, 0])
    took = []
    for _ in range(calls):
        dev.synchronize()
        start = time.perf_counter()
        cmd()
        dev.synchronize()
        took.append(time.perf_counter() - start)
    got = get(dev, out).reshape(b.tokens, -1)
    for ref in (*tables, cache, q, out):
        dev.release(ref.buffer)
    return min(took), got


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("parity,value,most", [(0, np.nan, 10), (0, np.inf, 10), (1, np.inf, 100)])
def test_what_a_value_that_is_not_finite_costs_few_rows(dev, parity, value, most, dtype):
    # One early position of every sequence. A NaN score ends its row (1.2 times
    # the time of the clean call measured); a value's rows are done again in
    # plain f32 (25 to 50 times).
    b = Batch([(3000, 1)] * 32, heads=32, kv_heads=8, dim=128, page=16, layers=1, layer=0, dtype=dtype)
    clean, _ = seconds(dev, b)
    put_values(b, [(s, 5, parity, value) for s in range(32)])
    hurt, got = seconds(dev, b)
    assert not np.any(np.isfinite(got))
    assert hurt < most * clean, (hurt, clean)


@pytest.mark.parametrize("new", [1, 70])
def test_scores_of_minus_infinity_leave_the_others(dev, new):
    # A visible key of -inf times a positive query: its probability is 0.
    b = Batch([(100, new)], heads=2, kv_heads=2, dim=8, page=16)
    b.q = np.abs(b.q) + 0.1
    put_values(b, [(0, 50, 0, -np.inf)])
    got = attend(dev, b)
    with np.errstate(invalid="ignore"):
        k, v = b.keys(0)
    keep = np.arange(100 + new) != 50
    for t in range(new):
        for h in range(2):
            seen = keep & (np.arange(100 + new) <= 100 + t)
            s = k[seen, h] @ b.q[t, 8 * h:8 * h + 8].astype(np.float64) / math.sqrt(8)
            w = np.exp(s - s.max())
            want = (w / w.sum()) @ v[seen, h]
            # ds for scores of up to 8 terms of size 5; see the module's note.
            assert np.all(np.abs(got[t, 8 * h:8 * h + 8] - want) <= 1e-3)


def outputs(b, window=0, sinks=0):
    """The definition in 64 bits, infinities and NaN with it: a value counts by
    its sign where its key's score is not -infinity."""
    scale, G = b.dim ** -0.5, b.heads // b.kv_heads
    out = np.full((b.tokens, b.heads, b.dim), np.nan)
    with np.errstate(invalid="ignore"):
        for i, (p, n) in enumerate(b.lens):
            k, v = b.keys(i)
            for t in range(n):
                pos = np.arange(p + t + 1)
                if window:
                    pos = pos[(pos > p + t - window) | (pos < sinks)]
                for h in range(b.heads):
                    row = int(b.starts[i]) + t
                    s = k[pos, h // G] @ b.q[row, h * b.dim:(h + 1) * b.dim].astype(np.float64) * scale
                    if np.all(s < np.inf) and np.any(s > -np.inf):
                        w = np.exp(s - s.max())
                        seen = s > -np.inf
                        out[row, h] = ((w / w.sum())[seen, None] * v[pos[seen], h // G]).sum(0)
    return out.reshape(b.tokens, -1)


def check_odd(got, b, window=0, sinks=0, some=True):
    """Infinities and NaN where the definition has them, and the rest (some,
    where the batch is made for it) within the bound that the same batch has
    with small numbers in their places."""
    want = outputs(b, window, sinks)
    places = ~np.isfinite(b.stored)
    keep = b.stored.copy()
    b.stored[places] = 0
    tol = b.attention(b.dim ** -0.5, window, sinks)[1] * 2
    b.stored = keep
    live = int(b.starts[-1])
    got, want, tol = got[:live], want[:live], tol[:live]
    assert np.array_equal(np.isnan(got), np.isnan(want))
    for sign in (np.inf, -np.inf):
        assert np.array_equal(got == sign, want == sign)
    ok = np.isfinite(want)
    assert np.any(ok) or not some
    assert np.all(np.abs(got[ok] - want[ok]) <= tol[ok])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("heads,new,page", [(2, 5, 16), (4, 150, 16), (16, 40, 5)])
def test_channels_that_are_not_finite(dev, dtype, window, heads, new, page):
    # Single values: their channels alone are lost, in the rows that see them.
    b = Batch([(100, new), (0, new), (33, 1)], heads=heads, kv_heads=2, dim=64, page=page, layers=1, layer=0, dtype=dtype)
    for seq, pos, head, d, value in [(0, 3, 0, 1, np.inf), (0, 90, 1, 63, -np.inf), (0, 103, 0, 2, np.nan),
                                     (0, 102, 0, 1, -np.inf), (1, 2, 1, 8, np.inf), (1, new - 1, 0, 31, np.inf)]:
        b.stored[int(b.table[seq, pos // page]), 0, 1, pos % page, head, d] = value
    b.stored, b.words = to_bits(b.stored.astype(np.float32), dtype)
    check_odd(attend(dev, b, window=window, sinks=2 if window else 0), b, window, 2 if window else 0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens", [[(2500, 40), (2000, 3), (30, 50)], [(3000 - 20 * i, 30 + i) for i in range(12)]])
def test_channels_that_are_not_finite_far_apart(dev, lens, dtype):
    # In the first, a middle and the last tile of segments, split ones too.
    b = Batch(lens, heads=8, kv_heads=2, dim=64, page=16, layers=1, layer=0, dtype=dtype)
    for seq in range(0, len(lens), 2):
        end = sum(lens[seq])
        for pos, head, d, value in [(1, 0, 3, np.inf), (end // 2, 1, 40, -np.inf), (end - 4, 0, 9, np.nan)]:
            b.stored[int(b.table[seq, pos // 16]), 0, 1, pos % 16, head, d] = value
    b.stored, b.words = to_bits(b.stored.astype(np.float32), dtype)
    check_odd(attend(dev, b), b)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,new", [(2, 5), (4, 150), (16, 70)])
def test_scores_that_are_infinite(dev, dtype, heads, new):
    # Keys with one infinity: scores of +infinity end a row, -infinity leaves
    # it without that key.
    b = Batch([(100, new), (0, new)], heads=heads, kv_heads=2, dim=64, page=16, layers=1, layer=0, dtype=dtype)
    b.q.reshape(b.tokens, heads, 64)[:, :, 7] = np.where(np.arange(b.tokens) % 3, 0.5, -0.5)[:, None]
    for seq, pos, value in [(0, 20, -np.inf), (0, 21, -np.inf), (0, 104, -np.inf), (1, 1, -np.inf), (1, 3, -np.inf)]:
        b.stored[int(b.table[seq, pos // 16]), 0, 0, pos % 16, :, 7] = value
    b.stored, b.words = to_bits(b.stored.astype(np.float32), dtype)
    check_odd(attend(dev, b), b)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,new", [(2, 3), (8, 60)])
def test_rows_whose_scores_are_all_minus_infinity(dev, dtype, heads, new):
    # The first row sees one key, of score -infinity: it is NaN, the others
    # leave that key out.
    b = Batch([(0, new), (20, 1)], heads=heads, kv_heads=2, dim=64, page=16, layers=1, layer=0, dtype=dtype)
    b.q.reshape(b.tokens, heads, 64)[:, :, 7] = 0.5
    b.stored[int(b.table[0, 0]), 0, 0, 0, :, 7] = -np.inf
    b.stored, b.words = to_bits(b.stored.astype(np.float32), dtype)
    got = attend(dev, b)
    assert np.all(np.isnan(got[0]))
    check_odd(got, b)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,new", [(2, 5), (4, 150)])
@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_queries_that_are_not_finite(dev, value, dtype, heads, new):
    b = Batch([(100, new), (9, 1)], heads=heads, kv_heads=2, dim=64, page=16, layers=1, layer=0, dtype=dtype)
    q = b.q.reshape(b.tokens, heads, 64)
    q[1, 0, 5] = q[new, heads - 1, 63] = value
    got = attend(dev, b).reshape(q.shape)
    assert np.all(np.isnan(got[1, 0])) and np.all(np.isnan(got[new, heads - 1]))
    q[1, 0, 5] = q[new, heads - 1, 63] = 0
    want, tol = (x.reshape(q.shape) for x in b.attention(0.125))
    rest = np.ones((b.tokens, heads), bool)
    rest[1, 0] = rest[new, heads - 1] = False
    assert np.all(np.abs(got - want)[rest] <= tol[rest])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("parity,value", [(0, np.nan), (0, -np.inf), (1, np.inf)])
def test_what_a_value_that_is_not_finite_costs_many_rows(dev, parity, value, dtype):
    # One early position, or one in eight, in a prompt whose rows nearly all see it.
    b = Batch([(0, 2048)], heads=8, kv_heads=2, dim=128, page=16, layers=1, layer=0, dtype=dtype)
    clean, _ = seconds(dev, b)
    put_values(b, [(0, 5, parity, value)])
    hurt, got = seconds(dev, b)
    assert np.all(np.isfinite(got[:5])) and not np.any(np.isfinite(got[5:]))
    assert hurt < 10 * clean, (hurt, clean)
    put_values(b, [(0, pos, parity, value) for pos in range(5, 2048, 8)])
    hurt, got = seconds(dev, b)
    assert np.all(np.isfinite(got[:5])) and not np.any(np.isfinite(got[5:]))
    assert hurt < 100 * clean, (hurt, clean)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -12, 2.0 ** 12, 2.0 ** 60])
def test_sizes_of_keys_values_and_queries(dev, size, dtype, new):
    # The same scores from keys and queries of any size, values of any size.
    if dtype == F16 and not 2.0 ** -13 < size < 2.0 ** 13:
        pytest.skip("beyond F16")
    b = Batch([(150, new)], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
    b.stored, b.words = to_bits((b.stored * size).astype(np.float32), dtype)
    check(attend(dev, b, scale=0.125 / size), b, scale=0.125 / size)
    b.q = (b.q / np.float32(size)).astype(np.float32)
    check(attend(dev, b, scale=0.125), b, scale=0.125)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_values_of_very_different_sizes(dev, dtype, new):
    # One key with a huge value that no row gives weight, among small ones.
    b = Batch([(150, new)], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
    b.q = np.abs(b.q) + 0.5
    put_values(b, [(0, 30, 0, -200.0), (0, 30, 1, 2.0 ** 14)])
    got = attend(dev, b)
    want, tol = b.attention(0.125)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("dim", [64, 128])
def test_value_channels_of_very_different_sizes(dev, dim, page, dtype):
    # Each channel is held as finely as if it were alone: to 2^-22 of a value
    # or 2^-26 of the channel's largest among a tile's keys, 2^-25 with those
    # of the probabilities. Sizes change along the keys too, so that the scales
    # of a tile do not suit the next.
    b = Batch([(150, 40), (300, 90)], heads=8, kv_heads=2, dim=dim, page=page, layers=1, layer=0, dtype=dtype)
    b.stored[..., 1, :, :, :] *= 2.0 ** (-10.0 * (np.arange(dim) % 4))
    put = [(1, pos, 2.0 ** (9 * (pos // 100 % 3))) for pos in range(390)]
    for seq, pos, size in put:
        b.stored[int(b.table[seq, pos // page]), 0, 1, pos % page] *= size
    b.stored, b.words = to_bits(b.stored.astype(np.float32), dtype)
    scale = dim ** -0.5
    got = attend(dev, b).reshape(b.tokens, 8, dim)
    want = b.attention(scale)[0].reshape(b.tokens, 8, dim)
    for i, (p, n) in enumerate(b.lens):
        k, v = b.keys(i)
        for t in range(n):
            for h in range(8):
                kk, vv = k[:p + t + 1, h // 4], v[:p + t + 1, h // 4]
                tile = v[:min(p + n, 128 * ((p + t) // 128 + 1)), h // 4]
                q = b.q[b.starts[i] + t].reshape(8, dim)[h].astype(np.float64)
                s = kk @ q * scale
                w = np.exp(s - s.max())
                ds = 9 * 2.0 ** -20 * scale * (np.abs(kk) @ np.abs(q)).max()
                tol = (w / w.sum()) @ np.abs(vv) * (2 * ds + (8 + len(kk) / 64) * 2.0 ** -20)
                tol += 2.0 ** -25 * np.abs(tile).max(0)
                row = b.starts[i] + t
                assert np.all(np.abs(got[row, h] - want[row, h]) <= tol), (row, h)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("sizes", [[0, 25, -25, 20, -10], [0, 90, -100, 80, 3]])
def test_values_that_rise_and_fall(dev, sizes, window, dtype):
    # Blocks of 400 positions of one size: the channels' scales follow, up and
    # down, and what the rows hold so far with them. A value counts to 2^-26 of
    # the largest of its dim among 128 neighbours, and to 2^-90 of the largest
    # of all.
    b = Batch([(0, 2000), (1900, 100)], heads=4, kv_heads=2, dim=64, page=16, layers=1, layer=0, dtype=dtype)
    for seq in range(2):
        for pos in range(2000):
            b.stored[int(b.table[seq, pos // 16]), 0, 1, pos % 16] *= 2.0 ** sizes[pos // 400]
    b.stored, b.words = to_bits(b.stored.astype(np.float32), dtype)
    got = attend(dev, b, window=window).reshape(b.tokens, 4, 64)
    for i, rows in (0, range(0, 2000, 37)), (1, range(0, 100, 9)):
        k, v = b.keys(i)
        for t in rows:
            at, row = b.lens[i][0] + t, int(b.starts[i]) + t
            low = max(at + 1 - window, 0) if window else 0
            for h in range(4):
                kk, vv, q = k[low:at + 1, h // 2], v[low:at + 1, h // 2], b.q[row, 64 * h:64 * h + 64].astype(np.float64)
                s = kk @ q / 8
                w = np.exp(s - s.max())
                w /= w.sum()
                ds = 9 * 2.0 ** -20 / 8 * (np.abs(kk) @ np.abs(q)).max()
                near = np.abs(v[max(low - 127, 0):at + 128, h // 2]).max(0)
                tol = w @ np.abs(vv) * (2 * ds + (8 + len(kk) / 64) * 2.0 ** -20) + 2.0 ** -25 * near
                tol += 2.0 ** -89 * np.abs(v[:, h // 2]).max(0)
                assert np.all(np.abs(got[row, h] - w @ vv) <= tol), (row, h)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads", [2, 8])
def test_large_keys_that_a_row_does_not_see(dev, heads, dtype):
    # From position 40 on keys are 2^13 or 2^24 times as large: the rows before
    # keep their precision, which the bound takes from what they see.
    b = Batch([(0, 100), (30, 60)], heads=heads, kv_heads=2, dim=64, page=16, layers=1, layer=0, dtype=dtype)
    for seq in range(2):
        for pos in range(40, sum(b.lens[seq])):
            b.stored[int(b.table[seq, pos // 16]), 0, 0, pos % 16] *= 2.0 ** (13 if dtype == F16 else 24)
    b.stored, b.words = to_bits(b.stored.astype(np.float32), dtype)
    check(attend(dev, b), b)


def test_extreme_scores(dev):
    # Scores of +-20000: only differences count.
    b = Batch([(200, 1), (90, 40)], heads=4, kv_heads=2, dim=64, page=16)
    check(attend(dev, b, scale=300.0), b, scale=300.0)
    check(attend(dev, b, scale=0.0), b, scale=0.0)
    check(attend(dev, b, scale=-0.125), b, scale=-0.125)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new", [1, 40])
def test_scores_past_24_bits(dev, new, dtype):
    # Scores of 10^8 and more, whose steps in f32 are larger than 1: nothing
    # overflows, and a row whose largest score leads by more than the steps of
    # all has that key's value (to 2^-16: a probability of at most e^-40 beside
    # one, and what its pair and the value's keep).
    b = Batch([(200, new), (30, new)], heads=4, kv_heads=2, dim=64, page=16, dtype=dtype)
    for scale in (1e7, -1e8):
        got = attend(dev, b, scale=scale)
        want, _ = b.attention(scale)
        assert np.all(np.isfinite(got))
        for i, (p, n) in enumerate(b.lens):
            k, v = b.keys(i)
            for t in range(n):
                for h in range(4):
                    row = int(b.starts[i]) + t
                    q = b.q[row, 64 * h:64 * h + 64].astype(np.float64)
                    s = k[:p + t + 1, h // 2] @ q * scale
                    ds = 16 * 2.0 ** -20 * abs(scale) * (np.abs(k[:p + t + 1, h // 2]) @ np.abs(q)).max()
                    top = np.sort(s)[::-1]
                    if len(top) == 1 or top[0] - top[1] > 2 * ds + 40:
                        x, w = got[row, 64 * h:64 * h + 64], want[row, 64 * h:64 * h + 64]
                        assert np.all(np.abs(x - w) <= 2.0 ** -16 * np.abs(v).max())


def random_batch(r, seed):
    """A batch and (window, sinks) of any sizes that a test can afford."""
    while True:
        kv, G = r.choice([1, 1, 2, 3, 4, 8]), r.choice([1, 1, 2, 4, 7, 8, 16])
        seqs = r.choice([1, 1, 2, 3, 5, 9, 30, 150])
        hi = r.choice([3, 40, 300, 1500]) // (8 if seqs > 20 else 1) + 1
        most = r.choice([1, 1, 2, 5, 40, 200]) // (10 if seqs > 20 else 1) + 1
        lens = [(r.randrange(hi), r.randrange(most + 1)) for _ in range(seqs)]
        if sum(n for _, n in lens) and sum(n for _, n in lens) * kv * G * (hi + most) < 1.5e6:
            break
    prefix = window = sinks = 0
    kind = r.random()
    if kind < 0.25:
        prefix = r.randrange(1, hi + 1)
        lens = [(p + prefix, n) for p, n in lens]
    elif kind < 0.6:
        window, sinks = r.choice([1, 2, 15, 16, 17, 33, 100, 1000]), r.choice([0, 0, 1, 4, 16, 33, 200])
    layers = r.choice([1, 2])
    b = Batch(lens, heads=kv * G, kv_heads=kv, dim=8 * r.choice([1, 4, 8, 8, 9, 12, 16, 16, 16, 25, 32]),
              page=r.choice([3, 5, 8, 16, 16, 24, 32, 64, 100, 128]), layers=layers, layer=r.randrange(layers),
              dtype=r.choice([F32, F16, BF16]), prefix=prefix, pad=r.randrange(3), seed=seed, narrow=r.random() < 0.4)
    return b, window, sinks


@pytest.mark.parametrize("seed", range(40))
def test_random_batches(dev, seed):
    r = random.Random(seed)
    b, window, sinks = random_batch(r, seed)
    got = attend(dev, b, window=window, sinks=sinks, offset=seed % 2, max_new=b.max_new() + r.choice([0, 0, 50]))
    check(got, b, window=window, sinks=sinks)


@pytest.mark.parametrize("seed", range(40))
def test_random_batches_with_values_that_are_not_finite(dev, seed):
    r = random.Random(1000 + seed)
    b, window, sinks = random_batch(r, seed)
    used = set()
    seen = [(i, pos) for i, (p, n) in enumerate(b.lens) if n for pos in range(p + n)]
    for _ in range(r.choice([1, 3, 20])):
        i, pos = r.choice(seen)
        slot = (int(b.table[i, pos // b.page]), pos % b.page)
        if slot in used:  # a key and its value at once: 0 times infinity
            continue
        used.add(slot)
        parity = int(r.random() < 0.7)
        value = r.choice([np.inf, -np.inf, np.nan]) if parity else r.choice([np.inf, -np.inf, -np.inf, np.nan])
        b.stored[slot[0], b.layer, parity, slot[1], r.randrange(b.kv_heads), r.randrange(b.dim)] = value
    b.stored, b.words = to_bits(b.stored.astype(np.float32), b.dtype)
    check_odd(attend(dev, b, window=window, sinks=sinks, offset=seed % 2), b, window, sinks, some=False)


# ---------------------------------------------------------------- prefix ----

@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", [
    dict(lens=[(20, 1)], prefix=1, page=16),
    dict(lens=[(20, 1), (40, 1), (16, 1)], prefix=16, page=16, heads=8, kv_heads=2, dim=128),
    dict(lens=[(300, 1), (301, 3), (257, 0), (700, 1)], prefix=257, page=16, heads=4, kv_heads=4, dim=64),
    dict(lens=[(130, 0), (130, 1), (131, 17)], prefix=130, page=5, heads=6, kv_heads=2, dim=72, pad=3),
    dict(lens=[(2000 + i, 1) for i in range(40)], prefix=2000, page=64, heads=8, kv_heads=1, dim=128, layers=1,
         layer=0),
    dict(lens=[(90, 2), (99, 1)], prefix=64, page=16, heads=2, kv_heads=1, dim=256),
    dict(lens=[(200, 70), (150, 1)], prefix=150, page=32, heads=16, kv_heads=2, dim=64),
])
def test_prefix(dev, case, dtype):
    b = Batch(**case, dtype=dtype)
    check(attend(dev, b, offset=1), b)
    prefix, b.prefix = b.prefix, 0
    plain = attend(dev, b)  # the operator without a prefix gives the same
    check(plain, b)
    b.prefix = prefix


# The prefix is read in a pass of its own from this many bytes of reads by all
# sequences on; below, every sequence reads it by itself.
PASS_BYTES = 96 << 20
PASSES = [
    # rows of one kv head: 16, 64, 328, wide heads, odd pages; the last two over enough keys for the kernel for many
    dict(lens=[(1700 + i, 1) for i in range(16)], prefix=1650, heads=8, kv_heads=8, dim=128, page=16),
    dict(lens=[(800 + 3 * i, 1) for i in range(64)], prefix=799, heads=8, kv_heads=8, dim=128, page=64),
    dict(lens=[(640 + i % 9, i % 3) for i in range(80)], prefix=640, heads=32, kv_heads=8, dim=64, page=16, pad=2),
    dict(lens=[(1000 + i, 1) for i in range(16)], prefix=900, heads=16, kv_heads=8, dim=256, page=24),
    dict(lens=[(1500 + i, i % 2) for i in range(31)], prefix=1500, heads=8, kv_heads=8, dim=72, page=5),
    dict(lens=[(702, 0)] + [(702 + i, 1) for i in range(64)], prefix=701, heads=64, kv_heads=8, dim=72, page=7),
    dict(lens=[(1300 + i, 1) for i in range(48)], prefix=1290, heads=64, kv_heads=8, dim=128, page=16),
]


def pass_batch(case, dtype, **kw):
    b = Batch(**case, layers=1, layer=0, dtype=dtype, **kw)
    assert len(b.lens) * b.prefix * 2 * b.kv_heads * b.dim * (4 if dtype == F32 else 2) >= PASS_BYTES
    return b


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(PASSES)))
def test_prefix_in_a_pass_of_its_own(dev, case, dtype):
    b = pass_batch(PASSES[case], dtype, seed=case)
    refs = upload(dev, b)
    first = attend(dev, b, offset=case % 2, refs=refs)
    check(first, b)
    for _ in range(3):
        assert np.array_equal(first, attend(dev, b, offset=case % 2, refs=refs))


@pytest.mark.parametrize("case", [0, 1, 4, 6])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_prefix_pass_with_values_that_are_not_finite(dev, value, case):
    b = pass_batch(PASSES[case], F32, seed=case)
    hurt = 3 if case != 4 else 5  # a sequence with a token of its own
    put_values(b, [(hurt, b.lens[hurt][0], 1, value)])
    got = attend(dev, b)
    want, tol = b.attention(1 / math.sqrt(b.dim))
    # Where the position lies in the prefix's last page, longer sequences see it too.
    clean = np.all(np.isfinite(want), axis=1)
    assert not clean[int(b.starts[hurt])] and np.any(clean)
    assert np.all(np.abs(got[clean] - want[clean]) <= tol[clean])
    assert not np.any(np.isfinite(got[~clean]))
    put_values(b, [(hurt, 100, 0, np.nan)])  # shared: no row is left
    assert not np.any(np.isfinite(attend(dev, b)))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_prefix_whose_pass_does_not_fit_the_workspace(dev, dtype):
    b = pass_batch(PASSES[6], dtype, seed=6)
    # Room for the pieces of split segments (19.7 MB) and 0.9 MB; the pass would leave 1.6 MB of results.
    small = CudaDevice(0, workspace_bytes=2 * (2 * 148 * 128 * 130 * 4 + (9 << 17)))
    try:
        start = small.launch_count()
        got = attend(small, b)
        without = small.launch_count() - start
        check(got, b)
    finally:
        small.close()
    refs, start = upload(dev, b), dev.launch_count()
    check(attend(dev, b, refs=refs), b)
    assert dev.launch_count() - start > without
    b.prefix = 0
    assert np.array_equal(attend(dev, b, refs=refs), got)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prompts_under_one_prefix(dev, dtype):
    # Their results do not fit the workspace: the rows read the prefix themselves.
    b = Batch([(512, 1)] * 4, prefix=512, heads=32, kv_heads=8, dim=128, page=16, layers=1, layer=0, dtype=dtype)
    new, width = 2048, (512 + 2048) // 16
    own = 32 + np.arange(4 * 128).reshape(4, 128)
    b.table = np.concatenate([np.tile(np.arange(32), (4, 1)), own], 1).astype(np.uint32)
    b.lens, b.tokens, b.pages = [(512, new)] * 4, 4 * new, 32 + 4 * 128
    b.starts, b.shape = np.arange(5, dtype=np.uint32) * new, (b.pages, 1, 2, 16, 8, 128)
    assert b.table.shape == (4, width)
    r = np.random.RandomState(1)
    b.stored, b.words = to_bits(r.standard_normal(b.shape).astype(np.float32), dtype)
    b.q = r.standard_normal((b.tokens, 32 * 128)).astype(np.float32)
    refs = upload(dev, b)
    got = attend(dev, b, refs=refs)
    b.prefix = 0
    assert np.array_equal(got, attend(dev, b, refs=refs))
    # A few rows against the definition.
    k, v = b.keys(2)
    for t in (0, 1000, 2047):
        for h in (0, 31):
            kk, vv = k[:513 + t, h // 4], v[:513 + t, h // 4]
            s = kk @ b.q[2 * new + t, 128 * h:128 * h + 128].astype(np.float64) / math.sqrt(128)
            w = np.exp(s - s.max())
            ds = 9 * 2.0 ** -20 / math.sqrt(128) * (np.abs(kk) @ np.abs(b.q[2 * new + t, 128 * h:128 * h + 128])).max()
            tol = (w / w.sum()) @ np.abs(vv) * (2 * ds + (8 + len(kk) / 64) * 2.0 ** -20)
            assert np.all(np.abs(got[2 * new + t, 128 * h:128 * h + 128] - (w / w.sum()) @ vv) <= tol)


def test_prefix_of_zero(dev):
    b = Batch([(20, 1), (3, 2)], heads=4, kv_heads=2, dim=64)
    refs = upload(dev, b)
    x = Value.f32((b.tokens, 256))
    out = new_f32(dev, b.q.size)
    dev.dispatch(b.op(OpCode.PrefixAttention, scale=0.125), [put_f32(dev, b.q), *refs[0], refs[1]],
                 [x, *b.described(), b.state()], [out], [x], [2, 0])
    check(get(dev, out).reshape(b.tokens, -1), b, scale=0.125)


@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_prefix_with_a_value_that_is_not_finite_in_one_sequence(dev, value):
    b = Batch([(40, 1), (50, 1), (41, 1)], prefix=40, page=8, heads=4, kv_heads=2, dim=64)
    put_values(b, [(1, 45, 1, value)])
    got = attend(dev, b)
    want, tol = b.attention(0.125)
    assert np.all(np.abs(got[[0, 2]] - want[[0, 2]]) <= tol[[0, 2]])
    assert not np.any(np.isfinite(got[1]))


# ------------------------------------------------------- the device's manner

@pytest.mark.parametrize("prefix", [0, 64])
def test_results_do_not_depend_on_the_run(dev, prefix):
    b = Batch([(5000, 1), (64, 1), (900, 3), (300, 60)], prefix=prefix, heads=8, kv_heads=2, dim=128, layers=1, layer=0)
    refs = upload(dev, b)
    first = attend(dev, b, refs=refs)
    for _ in range(5):
        assert np.array_equal(first, attend(dev, b, refs=refs))


def test_empty_calls(dev):
    for lens, pad in ([], 0), ([(5, 0)], 0), ([(5, 0), (3, 0)], 2):
        b = Batch(lens, pad=pad)
        tables, cache = upload(dev, b)
        x, y = Value.f32((b.tokens, b.heads * b.dim)), Value.f32((b.tokens, b.kv_heads * b.dim))
        out = new_f32(dev, b.q.size, 7.5)
        for code, scalars in (OpCode.PagedAttention, [0, 0, 0]), (OpCode.PrefixAttention, [0, 0]):
            dev.dispatch(b.op(code, scale=1.0), [put_f32(dev, b.q), *tables, cache],
                         [x, *b.described(), b.state()], [out], [x], scalars)
        dev.dispatch(b.append_op(), [put_f32(dev, b.k), put_f32(dev, b.v), *tables, cache],
                     [y, y, *b.described(), b.state()], [], [])
        assert np.all(get(dev, out) == 7.5)


def test_refusals_leave_the_device_usable(dev):
    b = Batch([(20, 3), (5, 1)])
    refs = upload(dev, b)
    bad = b.table.copy()
    bad[0, 0] = b.pages
    with pytest.raises(DeviceError, match="page id out of range"):
        attend(dev, b, refs=([put_u32(dev, bad), *refs[0][1:]], refs[1]))
    with pytest.raises(DeviceError, match="max_new"):
        attend(dev, b, refs=refs, max_new=2)
    check(attend(dev, b, refs=refs), b)


def test_small_workspace_is_refused():
    d = CudaDevice(0, workspace_bytes=1 << 20)
    try:
        b = Batch([(20, 3)])
        with pytest.raises(DeviceError, match="workspace is too small"):
            attend(d, b)
    finally:
        d.close()


def test_two_devices_on_one_gpu(dev):
    # Separate streams and workspaces: both run the same batch at once.
    other = CudaDevice(0)
    try:
        b = Batch([(4000, 1), (700, 2)], heads=8, kv_heads=2, dim=128, layers=1, layer=0)
        sides = []
        for d in (dev, other):
            tables, cache = upload(d, b)
            x = Value.f32((b.tokens, b.heads * b.dim))
            out = new_f32(d, b.q.size)
            cmd = d.command(b.op(OpCode.PagedAttention, scale=0.088), [put_f32(d, b.q), *tables, cache],
                            [x, *b.described(), b.state()], [out], [x], [2, 0, 0])
            sides.append((d, cmd, out))
        for _ in range(20):
            for _, cmd, _ in sides:
                cmd()
        for d, _, out in sides:
            check(get(d, out).reshape(b.tokens, -1), b, scale=0.088)
    finally:
        other.close()


class Server:
    """A decoding loop over two layers as a serving program writes it: per
    layer PagedAppend, Rope of the queries, attention; the batch's description
    uploaded once per step."""

    def __init__(self, dev, heads, kv_heads, dim, page, seqs, width, pages, dtype, prefix=0, shape=None):
        self.dev, self.n, self.prefix, self.dtype = dev, seqs, prefix, dtype
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.shape = (pages, 2, 2, page, kv_heads, dim)
        state = Value(dtype, self.shape, ValueRole.State)
        self.cache = new_f32(dev, state_words(self.shape, dtype))
        self.table, self.past, self.starts, self.pos = (
            put_u32(dev, np.zeros(s)) for s in ((seqs, width), seqs, seqs + 1, seqs))
        described = [Value.u32((seqs, width)), Value.u32((seqs,)), Value.u32((seqs + 1,))]
        ports = [self.table, self.past, self.starts]
        x, y = Value.f32((seqs, heads * dim)), Value.f32((seqs, kv_heads * dim))
        r = Value.f32((seqs, heads, 1, dim))
        self.q, self.k, self.v, self.turned, self.out = [], [], [], [], []
        self.commands = []
        code = OpCode.PrefixAttention if prefix else OpCode.PagedAttention
        scalars = [1, prefix] if prefix else [1, 0, 0]
        for layer in range(2):
            q, k, v = new_f32(dev, seqs * heads * dim), new_f32(dev, seqs * kv_heads * dim), new_f32(
                dev, seqs * kv_heads * dim)
            turned, out = new_f32(dev, seqs * heads * dim), new_f32(dev, seqs * heads * dim)
            attrs = dict(layer=layer, heads=heads, kv_heads=kv_heads, head_dim=dim)
            self.commands += [
                dev.command(Op(OpCode.PagedAppend, theta=500000.0, **attrs), [k, v, *ports, self.cache],
                            [y, y, *described, state], [], []),
                dev.command(Op(OpCode.Rope, theta=500000.0), [q, self.pos], [r, Value.u32((seqs, 1))], [turned], [r]),
                dev.command(Op(code, scale=1 / math.sqrt(dim), **attrs), [turned, *ports, self.cache],
                            [x, *described, state], [out], [x], scalars)]
            for name, ref in zip(("q", "k", "v", "turned", "out"), (q, k, v, turned, out)):
                getattr(self, name).append(ref)

    def step(self, table, past, qkv):
        d = self.dev
        d.upload_u32(self.table.buffer, table)
        d.upload_u32(self.past.buffer, past)
        d.upload_u32(self.starts.buffer, np.arange(self.n + 1))
        d.upload_u32(self.pos.buffer, past)
        for layer, (q, k, v) in enumerate(qkv):
            d.upload_f32(self.q[layer].buffer, q)
            d.upload_f32(self.k[layer].buffer, k)
            d.upload_f32(self.v[layer].buffer, v)
        for cmd in self.commands:
            cmd()
        d.synchronize()
        return [get(d, o).reshape(self.n, -1) for o in self.out]


@pytest.mark.parametrize("prefix", [0, 24])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decoding_captured_and_replayed(dtype, prefix):
    # Three sequences of different lengths decode 12 steps; the captured run
    # replays one graph while lengths and tables change, and gives what the
    # eager one gives, bit for bit.
    heads, kv_heads, dim, page, steps = 8, 2, 64, 8, 12
    rng = np.random.RandomState(3)
    table = np.full((3, 8), 63, np.uint32)
    table[:, :3] = [4, 9, 2]
    free = iter(rng.permutation(np.arange(10, 60)))
    for b in range(3):
        table[b, 3:] = [next(free) for _ in range(5)]
    results, replays = [], []
    for capture in (False, True):
        d = CudaDevice(0)
        try:
            d.set_capture(capture)
            s = Server(d, heads, kv_heads, dim, page, 3, 8, 64, dtype, prefix)
            r = np.random.RandomState(5)
            past = np.array([24, 31, 26], np.uint32)
            fill = r.randn(int(np.prod(s.shape))).astype(np.float32)
            d.upload_f32(s.cache.buffer, to_bits(fill, dtype)[1])
            outs = []
            for i in range(steps):
                qkv = [(r.randn(3, heads * dim), r.randn(3, kv_heads * dim), r.randn(3, kv_heads * dim))
                       for _ in range(2)]
                outs.append(s.step(table, past, qkv))
                past = past + 1
            results.append((outs, get(d, s.cache)))
            replays.append(d.capture_stats()["replays"])
        finally:
            d.close()
    assert replays[0] == 0 and replays[1] >= steps - 3
    for a, b in zip(results[0][0], results[1][0]):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))
    assert np.array_equal(results[0][1].view(np.uint32), results[1][1].view(np.uint32))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("window", [0, 33])
def test_prompts_captured_and_replayed(dtype, window):
    # Chunks of prompts of changing lengths through one captured command, then
    # a second graph on the same workspace.
    batches = [Batch([(p, n), (20, 1), (m, 9)], heads=8, kv_heads=2, dim=64, page=16, dtype=dtype, width=400,
                     extra_pages=40, pad=120 - n, seed=i)
               for i, (p, n, m) in enumerate([(300, 90, 0), (0, 120, 7), (500, 1, 90), (17, 64, 400), (100, 33, 5),
                                              (250, 100, 60)])]
    pages = max(b.pages for b in batches)
    shape = (pages, 2, 2, 16, 2, 64)
    d = CudaDevice(0)
    try:
        d.set_capture(True)
        cache = new_f32(d, state_words(shape, dtype))
        table, past, starts = (put_u32(d, np.zeros(n)) for n in ((3, 400), 3, 4))
        q, outs = new_f32(d, 130 * 512), [new_f32(d, 130 * 512) for _ in range(2)]
        x = Value.f32((130, 512))
        first = batches[0]
        cmds = [d.command(first.op(OpCode.PagedAttention, scale=0.125), [q, table, past, starts, cache],
                          [x, *first.described(), Value(dtype, shape, ValueRole.State)], [out], [x], [120, window, 1])
                for out in outs]
        for b in batches * 2:
            assert b.tokens == 130
            words = np.zeros(cache.len, np.float32)
            words[:b.words.size] = b.words
            d.upload_f32(cache.buffer, words)
            d.upload_u32(table.buffer, b.table)
            d.upload_u32(past.buffer, b.past)
            d.upload_u32(starts.buffer, b.starts)
            d.upload_f32(q.buffer, b.q)
            for cmd in cmds:
                cmd()
            d.synchronize()
            a, c = (get(d, out).reshape(130, -1) for out in outs)
            live = int(b.starts[-1])
            want, tol = b.attention(0.125, window, 1 if window else 0)
            assert np.all(np.abs(a[:live] - want[:live]) <= tol[:live])
            assert np.array_equal(a[:live], c[:live])
        assert d.capture_stats()["replays"] >= 6
    finally:
        d.close()


def test_decoding_matches_the_dense_cache(dev):
    # The same tokens through Rope, CausalAttention and a dense cache, one
    # sequence at a time.
    heads, kv_heads, dim, page, steps, width = 4, 2, 64, 4, 9, 4
    s = Server(dev, heads, kv_heads, dim, page, 2, width, 16, F32)
    table = np.array([[3, 8, 1, 15], [7, 2, 9, 4]], np.uint32)
    r = np.random.RandomState(8)
    max_seq = width * page
    dense = [new_f32(dev, 2 * 2 * max_seq * kv_heads * dim) for _ in range(2)]
    state = Value.f32((1, 2, 2, max_seq, kv_heads, dim), ValueRole.State)
    for i in range(steps):
        past = np.array([i, i], np.uint32)
        qkv = [[r.randn(2, n * dim).astype(np.float32) for n in (heads, kv_heads, kv_heads)] for _ in range(2)]
        got = s.step(table, past, qkv)
        for b in range(2):
            pos = put_u32(dev, [i])
            for layer, (q, k, v) in enumerate(qkv):
                x, y = Value.f32((1, heads, 1, dim)), Value.f32((1, kv_heads, 1, dim))
                tq, tk, out = new_f32(dev, heads * dim), new_f32(dev, kv_heads * dim), new_f32(dev, heads * dim)
                for val, src, dst in (x, q, tq), (y, k, tk):
                    dev.dispatch(Op(OpCode.Rope, theta=500000.0), [put_f32(dev, src[b]), pos],
                                 [val, Value.u32((1, 1))], [dst], [val])
                dev.dispatch(Op(OpCode.CausalAttention, layer=layer, heads=heads, kv_heads=kv_heads, head_dim=dim,
                                scale=1 / math.sqrt(dim)), [tq, tk, put_f32(dev, v[b]), dense[b]],
                             [x, y, y, state], [out], [x], [i])
                # Both are within 2^-14 of the definition (values up to 4).
                assert np.all(np.abs(get(dev, out) - got[layer][b]) <= 2.0 ** -13)
    # The caches agree bit for bit.
    paged = get(dev, s.cache).reshape(s.shape)
    for b in range(2):
        rows = paged[table[b].astype(np.int64)].transpose(1, 2, 0, 3, 4, 5).reshape(2, 2, max_seq, kv_heads, dim)
        assert np.array_equal(rows[:, :, :steps], get(dev, dense[b]).reshape(2, 2, max_seq, kv_heads, dim)[:, :, :steps])
