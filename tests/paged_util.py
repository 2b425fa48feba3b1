"""Paged KV cache test helpers (not collected as tests): ragged batches over a
paged cache and the operators' definitions in 64 bits."""
import numpy as np

from starlight_b200.device import BufferRef, DType, Op, OpCode, RopeVariant, Value, ValueRole, state_words

HOLE = 0xFFFFFFFF  # a table entry that must not be followed


def to_bits(x, dtype):
    """f32 array -> (stored values as f64, 32-bit words of the state)."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == DType.F32:
        return x.astype(np.float64), x.ravel()
    import torch
    t = torch.from_numpy(x).to(torch.float16 if dtype == DType.F16 else torch.bfloat16)
    raw = t.contiguous().view(torch.int16).numpy().ravel()
    if raw.size % 2:
        raw = np.concatenate([raw, np.zeros(1, np.int16)])
    return t.double().numpy(), raw.view(np.float32)


def from_bits(words, shape, dtype):
    """32-bit words of a state -> stored values as f64."""
    n = int(np.prod(shape))
    if dtype == DType.F32:
        return np.asarray(words, np.float32)[:n].reshape(shape).astype(np.float64)
    import torch
    raw = torch.from_numpy(np.ascontiguousarray(words, np.float32).view(np.int16)[:n].copy())
    return raw.view(torch.float16 if dtype == DType.F16 else torch.bfloat16).double().numpy().reshape(shape)


def dim_sum(k, q):
    """The sizes that the smallest steps of f16 pairs multiply in q . k."""
    return np.abs(k).max() * np.abs(q).sum() + np.abs(q).max() * np.abs(k).sum(1).max()


class Batch:
    """Sequences of (past, new) over a paged cache of random values; every
    slot that no sequence holds is NaN, every table entry past a sequence's
    pages is HOLE. `prefix` leading positions are shared pages."""

    def __init__(self, lens, heads=4, kv_heads=2, dim=64, page=16, layers=2, layer=1, dtype=DType.F32,
                 prefix=0, pad=0, extra_pages=3, seed=0, width=None, narrow=False):
        self.lens, self.heads, self.kv_heads, self.dim = lens, heads, kv_heads, dim
        self.page, self.layers, self.layer, self.dtype, self.prefix = page, layers, layer, dtype, prefix
        r = self.rng = np.random.RandomState(seed)
        need = [-(-(p + n) // page) for p, n in lens]
        shared = -(-prefix // page)
        self.pages = shared + sum(max(k - shared, 0) for k in need) + extra_pages
        order = r.permutation(self.pages)
        if width is None:
            # Rows in numbers have their own kernel where the table leaves room
            # for many keys; `narrow` tables have no more than they need.
            many = max([n for _, n in lens] + [0]) * heads // kv_heads > 16
            width = max(need + [1] + ([] if narrow or not many else [-(-(1 << 18) // page)]))
        self.table = np.full((len(lens), width), HOLE, np.uint32)
        used = shared
        for b, k in enumerate(need):
            self.table[b, :min(shared, width)] = order[:min(shared, width)]
            own = max(k - shared, 0)
            self.table[b, shared:shared + own] = order[used:used + own]
            used += own
        self.past = np.array([p for p, _ in lens], np.uint32)
        self.starts = np.concatenate([[0], np.cumsum([n for _, n in lens])]).astype(np.uint32)
        self.tokens = int(self.starts[-1]) + pad
        self.shape = (self.pages, layers, 2, page, kv_heads, dim)
        values = np.full(self.shape, np.nan, np.float32)
        for b, (p, n) in enumerate(lens):
            for j in range(need[b]):
                count = min(page, p + n - j * page)
                values[self.table[b, j], :, :, :count] = r.randn(layers, 2, count, kv_heads, dim)
        self.stored, self.words = to_bits(values, dtype)
        self.q = r.randn(self.tokens, heads * dim).astype(np.float32)
        self.k = r.randn(self.tokens, kv_heads * dim).astype(np.float32)
        self.v = r.randn(self.tokens, kv_heads * dim).astype(np.float32)

    def keys(self, b):
        """K, V [positions, kv_heads, dim] of sequence b (f64, as stored)."""
        p, n = self.lens[b]
        pos = np.arange(p + n)
        at = self.table[b][pos // self.page].astype(np.int64)
        return (self.stored[at, self.layer, 0, pos % self.page], self.stored[at, self.layer, 1, pos % self.page])

    def attention(self, scale, window=0, sinks=0):
        """(output, bound) [tokens, heads * dim] in f64; bound: what a correct
        kernel may be off by, elementwise (derived in test_gpu_paged.py)."""
        H, G, D = self.heads, self.heads // self.kv_heads, self.dim
        out = np.full((self.tokens, H, D), np.nan)
        tol = np.zeros((self.tokens, H, D))
        for b, (p, n) in enumerate(self.lens):
            if n == 0:
                continue
            k, v = self.keys(b)
            for t in range(n):
                row = int(self.starts[b]) + t
                at = p + t
                pos = np.arange(at + 1)
                if window:
                    pos = pos[(pos > at - window) | (pos < sinks)]
                for h in range(H):
                    kk, vv = k[pos, h // G], v[pos, h // G]
                    q = self.q[row, h * D:(h + 1) * D].astype(np.float64)
                    s = kk @ q * scale
                    w = np.exp(s - s.max())
                    out[row, h] = (w / w.sum()) @ vv
                    ds = 8 * 2.0 ** -20 * abs(scale) * (np.abs(kk) @ np.abs(q)).max()
                    ds += 2.0 ** -33 * abs(scale) * dim_sum(kk, q)
                    tol[row, h] = (w / w.sum()) @ np.abs(vv) * (2 * ds + (8 + len(pos) / 64) * 2.0 ** -20)
                    tol[row, h] += 2.0 ** -33 * np.abs(vv).max()
        return out.reshape(self.tokens, -1), tol.reshape(self.tokens, -1)

    # ---- ports -----------------------------------------------------------
    def described(self):
        return [Value.u32(self.table.shape), Value.u32(self.past.shape), Value.u32(self.starts.shape)]

    def state(self):
        return Value(self.dtype, self.shape, ValueRole.State)

    def op(self, code, **kw):
        return Op(code, layer=self.layer, heads=self.heads, kv_heads=self.kv_heads, head_dim=self.dim, **kw)

    def append_op(self, theta=500000.0, variant=RopeVariant.Neox):
        return self.op(OpCode.PagedAppend, theta=theta, variant=variant)

    def max_new(self):
        return max([n for _, n in self.lens] + [0])


def upload(dev, batch):
    """The batch's table, past and starts, and its cache, as BufferRefs."""
    from tests.gpu_util import put_f32, put_u32
    refs = [put_u32(dev, a) for a in (batch.table, batch.past, batch.starts)]
    cache = put_f32(dev, batch.words)
    assert cache.len == state_words(batch.shape, batch.dtype)
    return refs, cache


def put_at(dev, arr, offset):
    """An f32 array at an element offset of its buffer."""
    from tests.gpu_util import put_f32
    a = np.ascontiguousarray(arr, np.float32).ravel()
    ref = put_f32(dev, np.concatenate([np.full(offset, 7.5, np.float32), a]))
    return BufferRef(ref.buffer, offset, a.size)
