"""What dispatch refuses of the paged KV-cache operators, on the CPU: the
library's own checks run on a device without a GPU (host_dispatch.cpp), which
records accepted commands and launches nothing."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

from starlight_b200 import build, device as D
from starlight_b200.device import (BufferRef, Command, CudaDevice, DeviceError, DType, Op, OpCode, Status, Value,
                                   ValueRole)
from tests.paged_util import HOLE, Batch

HERE = os.path.dirname(os.path.abspath(__file__))


class HostDevice(CudaDevice):
    def __init__(self, lib):
        self._lib = lib
        self._d = C.c_void_p(lib.host_device_new())

    def close(self):
        if self._d:
            self._lib.host_device_free(self._d)
            self._d = C.c_void_p()

    def f32(self, words):
        return BufferRef(self._lib.host_buffer(self._d, words, None), 0, words)

    def u32(self, data):
        a = np.ascontiguousarray(data, np.uint32).ravel()
        keep = a if a.size else np.zeros(1, np.uint32)
        b = self._lib.host_buffer(self._d, a.size, keep.ctypes.data_as(C.POINTER(C.c_uint32)))
        return BufferRef(b, 0, a.size)


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    build.build()
    tmp = tmp_path_factory.mktemp("host_dispatch")
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    obj, so = str(tmp / "host.o"), str(tmp / "host.so")
    objects = [os.path.join(build.BUILD, f) for f in sorted(os.listdir(build.BUILD))
               if f.endswith(".o") and f not in ("capture.cpp.o", "decode_run.cpp.o", "engine.cpp.o")]
    subprocess.run([nvcc, "-x", "cu", *build.NVCC_FLAGS, "-c", os.path.join(HERE, "host_dispatch.cpp"), "-o", obj],
                   check=True)
    subprocess.run([nvcc, *build.ARCH, "-shared", "-o", so, obj, *objects, "-ldl", "-lpthread"], check=True)
    real, host = D.load_library(), C.CDLL(so)
    for name in ("slc_dispatch", "slc_last_error"):
        getattr(host, name).restype = getattr(real, name).restype
        getattr(host, name).argtypes = getattr(real, name).argtypes
    host.host_device_new.restype = C.c_void_p
    host.host_device_free.argtypes = [C.c_void_p]
    host.host_buffer.argtypes = [C.c_void_p, C.c_uint64, C.POINTER(C.c_uint32)]
    host.host_buffer.restype = C.c_uint32
    host.host_recorded.restype = C.c_uint64
    return host


@pytest.fixture
def dev(lib):
    d = HostDevice(lib)
    yield d
    d.close()


LENS = [(20, 3), (0, 1), (7, 0), (33, 1)]


class Call:
    """One dispatch's arguments, to be changed before it is made."""

    def __init__(self, dev, kind, batch=None, **kw):
        self.dev, self.kind = dev, kind
        b = self.b = batch or Batch(LENS, **kw)
        self.batch = [b.table.copy(), b.past.copy(), b.starts.copy()]
        self.described, self.state = b.described(), b.state()
        self.rows = b.tokens
        self.scalars = {"append": [], "attend": [b.max_new(), 0, 0], "prefix": [b.max_new(), b.prefix]}[kind]
        code = {"append": OpCode.PagedAppend, "attend": OpCode.PagedAttention, "prefix": OpCode.PrefixAttention}
        self.op = dict(code=code[kind], layer=b.layer, heads=b.heads, kv_heads=b.kv_heads, head_dim=b.dim,
                       theta=1e4, scale=0.125)
        self.width = (b.kv_heads if kind == "append" else b.heads) * b.dim
        self.out_shape = None
        self.state_offset = 0

    def __call__(self):
        d = self.dev
        before = d._lib.host_recorded()
        tables = [d.u32(a) for a in self.batch]
        half = self.state.dtype in (DType.F16, DType.BF16)
        words = D.state_words(self.state.shape, self.state.dtype if half else DType.F32)
        state = d.f32(words + self.state_offset)
        state = BufferRef(state.buffer, self.state_offset, words)
        x = Value.f32((self.rows, self.width))
        n = self.rows * self.width
        if self.kind == "append":
            ins, vals, outs, ovals = [d.f32(n), d.f32(n)], [x, x], [], []
        else:
            o = Value.f32(self.out_shape or (self.rows, self.width))
            ins, vals, outs, ovals = [d.f32(n)], [x], [d.f32(o.element_count())], [o]
        d.dispatch(Op(**self.op), ins + tables + [state], vals + self.described + [self.state], outs, ovals,
                   self.scalars)
        assert d._lib.host_recorded() == before + 1

    def refused(self, match, status=Status.Execution):
        before = self.dev._lib.host_recorded()
        with pytest.raises(DeviceError, match=match) as e:
            self()
        assert e.value.status == status
        assert self.dev._lib.host_recorded() == before


KINDS = ["append", "attend", "prefix"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [DType.F32, DType.F16, DType.BF16])
def test_accepts(dev, kind, dtype):
    Call(dev, kind, dtype=dtype)()
    Call(dev, kind, dtype=dtype, pad=5)()
    Call(dev, kind, dtype=dtype, page=5, dim=8, kv_heads=1, heads=1)()
    Call(dev, kind, batch=Batch([], dtype=dtype))()
    Call(dev, kind, batch=Batch([(5, 0)], dtype=dtype, pad=2))()


@pytest.mark.parametrize("kind", KINDS)
def test_refuses_page_ids_out_of_range(dev, kind):
    c = Call(dev, kind)
    c.batch[0][0, 1] = c.b.pages
    c.refused("page id out of range")
    c = Call(dev, kind)
    c.batch[0][3, 2] = HOLE
    c.refused("page id out of range")


@pytest.mark.parametrize("kind", KINDS)
def test_table_entries_beyond_the_sequences_are_not_looked_at(dev, kind):
    c = Call(dev, kind)
    c.batch[0][1, 1:] = HOLE
    c.batch[0][2, :] = HOLE  # a sequence without new tokens
    c()


def test_pages_behind_the_window_are_not_looked_at(dev):
    b = Batch([(100, 2)], page=8)
    c = Call(dev, "attend", batch=b)
    c.scalars = [2, 20, 3]
    low = 100 + 1 - 20
    c.batch[0][0, 1:low // 8] = HOLE
    c()
    c.batch[0][0, low // 8] = HOLE
    c.refused("page id out of range")
    c = Call(dev, "attend", batch=b)
    c.scalars = [2, 20, 9]  # the ninth sink is in page 1
    c.batch[0][0, 1:low // 8] = HOLE
    c.refused("page id out of range")


def test_append_looks_at_written_pages_only(dev):
    c = Call(dev, "append", batch=Batch([(100, 2)], page=8))
    c.batch[0][0, :12] = HOLE
    c()


@pytest.mark.parametrize("kind", KINDS)
def test_refuses_lengths(dev, kind):
    c = Call(dev, kind)
    c.batch[1][0] = 16 * c.batch[0].shape[1] - 2
    c.refused("exceed the table's pages")
    c = Call(dev, kind)
    c.batch[1][0] = 0xFFFFFFFF
    c.refused("exceed the table's pages")
    c = Call(dev, kind)
    c.batch[2][0] = 1
    c.refused("begin at 0")
    c = Call(dev, kind)
    c.batch[2][2] = 2
    c.refused("must not decrease")
    c = Call(dev, kind)
    c.batch[2][-1] += 1
    if kind != "append":
        c.scalars[0] = 9
    c.refused("exceed the token rows")


def test_refuses_a_page_written_twice(dev):
    c = Call(dev, "append")
    c.batch[0][3, 2] = c.batch[0][0, 1]
    c.refused("writes one page twice")
    c = Call(dev, "append", batch=Batch([(0, 40)], page=16))
    c.batch[0][0, 2] = c.batch[0][0, 0]
    c.refused("writes one page twice")
    # Pages that are read alone may be shared, here and by an attention.
    b = Batch([(40, 1), (40, 1)], page=16, prefix=32)
    Call(dev, "append", batch=b)()
    Call(dev, "attend", batch=b)()


@pytest.mark.parametrize("kind", ["attend", "prefix"])
def test_refuses_more_tokens_than_max_new(dev, kind):
    c = Call(dev, kind)
    c.scalars[0] = 2
    c.refused("more tokens than max_new")


def test_refuses_a_prefix_that_is_not_shared(dev):
    b = Batch([(40, 1), (50, 1), (5, 0)], page=16, prefix=30)
    Call(dev, "prefix", batch=b)()
    c = Call(dev, "prefix", batch=b)
    c.batch[0][1, 1] = c.batch[0][1, 2]
    c.refused("pages differ")
    c = Call(dev, "prefix", batch=b)
    c.batch[0][2, :] = HOLE  # no new tokens: not looked at
    c()
    c = Call(dev, "prefix", batch=b)
    c.scalars[1] = 41
    c.refused("exceeds a sequence's past")


@pytest.mark.parametrize("kind", KINDS)
def test_refuses_shapes(dev, kind):
    for change, match in [
        (lambda c: c.op.update(kv_heads=3), "width|state shape|multiple"),
        (lambda c: c.op.update(layer=2), "layer is out of range"),
        (lambda c: c.described.__setitem__(0, Value.u32((c.b.table.size,))), "batch shapes"),
        (lambda c: (c.described.__setitem__(1, Value.u32((3,))), c.batch.__setitem__(1, c.batch[1][:3])),
         "batch shapes"),
        (lambda c: (c.described.__setitem__(2, Value.u32((4,))), c.batch.__setitem__(2, c.batch[2][:4])),
         "batch shapes"),
        (lambda c: setattr(c, "width", c.width + 8), "width must equal"),
        (lambda c: setattr(c, "state", Value(DType.F32, c.b.shape[1:], ValueRole.State)), "state shape"),
        (lambda c: setattr(c, "state", Value(DType.F32, (*c.b.shape[:3], 0, *c.b.shape[4:]), ValueRole.State)),
         "nonzero page"),
    ]:
        c = Call(dev, kind)
        change(c)
        c.refused(match)


def test_refuses_heads_and_dims(dev):
    c = Call(dev, "attend", heads=4, kv_heads=2)
    c.op["heads"], c.width = 3, 3 * 64
    c.refused("multiple of kv_heads")
    c = Call(dev, "attend", heads=4, kv_heads=2)
    c.op["heads"], c.width = 0, 0
    c.refused("heads must be nonzero")
    for dim in (4, 12, 264):
        Call(dev, "append", dim=dim).refused("multiple of 8 up to 256", Status.Unimplemented)
    c = Call(dev, "attend")
    c.out_shape = (c.width, c.rows)
    c.refused("output shape")


@pytest.mark.parametrize("kind", KINDS)
def test_refuses_states(dev, kind):
    c = Call(dev, kind)
    c.state_offset = 2
    c.refused("16-byte boundary", Status.Unimplemented)
    c = Call(dev, kind)
    c.state_offset = 4
    c()
    c = Call(dev, kind)
    c.state = Value(DType.I8, c.b.shape, ValueRole.State)
    c.refused("dtype is not supported", Status.Unimplemented)
    c = Call(dev, kind)
    c.state = Value(DType.F32, c.b.shape, ValueRole.Temp)
    c.refused("exactly one State")


def test_sixteen_bit_states_belong_to_the_paged_operators(dev):
    # The dense operators keep refusing them.
    x, shape = Value.f32((1, 1, 1, 8)), (1, 1, 2, 4, 1, 8)
    with pytest.raises(DeviceError, match="dtype is not supported"):
        dev.dispatch(Op(OpCode.KvAppend), [dev.f32(8), dev.f32(8), dev.f32(64)],
                     [x, x, Value(DType.BF16, shape, ValueRole.State)], [], [], [0])
    with pytest.raises(DeviceError, match="16-bit state size"):
        c = Call(dev, "append", dtype=DType.BF16)
        b = c.b
        tables = [dev.u32(a) for a in c.batch]
        n = c.rows * c.width
        dev.dispatch(Op(**c.op), [dev.f32(n), dev.f32(n), *tables, dev.f32(int(np.prod(b.shape)))],
                     [Value.f32((c.rows, c.width))] * 2 + b.described() + [b.state()], [], [])


@pytest.mark.parametrize("theta", [-1.0, float("inf"), float("nan")])
def test_refuses_theta(dev, theta):
    c = Call(dev, "append")
    c.op["theta"] = theta
    c.refused("theta must be finite")


def test_refuses_port_counts_and_aliases(dev):
    c = Call(dev, "attend")
    c.scalars = [3, 0]
    c.refused("scalar count")
    b = Batch(LENS)
    n = b.tokens * b.heads * b.dim
    q, tables = dev.f32(n), [dev.u32(a) for a in (b.table, b.past, b.starts)]
    state = dev.f32(D.state_words(b.shape, b.dtype))
    x = Value.f32((b.tokens, b.heads * b.dim))
    op = b.op(OpCode.PagedAttention, scale=1.0)
    with pytest.raises(DeviceError, match="aliases an overlapping input"):
        dev.dispatch(op, [q, *tables, state], [x, *b.described(), b.state()], [q], [x], [3, 0, 0])
    with pytest.raises(DeviceError, match="too many command ports"):
        dev.dispatch(op, [q, *tables, state, dev.f32(4), dev.f32(4)],
                     [x, *b.described(), b.state(), Value.f32((4,)), Value.f32((4,))], [dev.f32(n)], [x], [3, 0, 0])
    with pytest.raises(DeviceError, match="state must be the last input"):
        dev.dispatch(op, [q, state, *tables], [x, b.state(), *b.described()], [dev.f32(n)], [x], [3, 0, 0])


def test_command_repeats_a_dispatch_with_other_scalars(dev):
    b = Batch(LENS)
    n = b.tokens * b.heads * b.dim
    x = Value.f32((b.tokens, b.heads * b.dim))
    state = dev.f32(D.state_words(b.shape, b.dtype))
    tables = [dev.u32(a) for a in (b.table, b.past, b.starts)]
    cmd = dev.command(b.op(OpCode.PagedAttention, scale=1.0), [dev.f32(n), *tables, state],
                      [x, *b.described(), b.state()], [dev.f32(n)], [x], [3, 0, 0])
    assert isinstance(cmd, Command)
    cmd()
    cmd([4, 16, 2])
    with pytest.raises(DeviceError, match="max_new"):
        cmd([2, 0, 0])
    cmd()
    with pytest.raises(DeviceError, match="different lengths"):
        dev.command(b.op(OpCode.PagedAttention), [dev.f32(n)], [], [], [])


def test_sizes_past_32_bits_are_refused(dev):
    c = Call(dev, "attend")
    # 70000 entries of pages of 65536 positions: 2^32 positions.
    c.described[0] = Value.u32((1, 70000))
    c.described[1], c.described[2] = Value.u32((1,)), Value.u32((2,))
    c.batch = [np.zeros((1, 70000), np.uint32), np.zeros(1, np.uint32), np.array([0, 1], np.uint32)]
    c.state = Value(DType.F32, (1, 2, 2, 65536, 2, 64), ValueRole.State)
    c.refused("exceeds 2\\^31")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1 << 31, (1 << 31) + 1, (1 << 32) - 1])
def test_page_sizes_past_31_bits_are_refused(dev, kind, page):
    # A table without pages does not bound the page by their product.
    c = Call(dev, kind, batch=Batch([(0, 0), (0, 0)], width=0))
    c.state = Value(DType.F32, (0, 2, 2, page, 2, 64), ValueRole.State)
    c.refused("exceed 2\\^31 - 1 positions")
    c.state = Value(DType.F32, (0, 2, 2, (1 << 31) - 1, 2, 64), ValueRole.State)
    c()


@pytest.mark.parametrize("dtype", [DType.F32, DType.BF16])
@pytest.mark.parametrize("heads", [32, 64])
@pytest.mark.parametrize("seqs,new,prefix", [(4, 2048, 512), (8, 1024, 512), (7, 1000, 512), (8, 1024, 64),
                                             (16, 4096, 20000), (1, 1, 16), (64, 1, 8192)])
def test_prefix_takes_what_attention_takes(dev, seqs, new, prefix, heads, dtype):
    # Prompts under one prefix: their rows' results do not all fit the workspace.
    b = Batch([], heads=heads, kv_heads=8, dim=128, layers=1, layer=0, dtype=dtype)
    b.lens = [(prefix, new)] * seqs
    width = -(-(prefix + new) // b.page)
    b.table = np.tile(np.arange(width, dtype=np.uint32), (seqs, 1))
    b.past, b.starts = np.full(seqs, prefix, np.uint32), np.arange(seqs + 1, dtype=np.uint32) * new
    b.tokens, b.pages, b.shape, b.prefix = seqs * new, width, (width, *b.shape[1:]), prefix
    Call(dev, "attend", batch=b)()
    Call(dev, "prefix", batch=b)()


@pytest.mark.parametrize("kind", KINDS)
def test_counts_near_31_bits_are_refused(dev, kind):
    # The kernels round positions, tokens and rows up to tiles and steps in 32 bits.
    most = (1 << 31) - 8192
    width = (1 << 31) // 4096 - 1
    b = Batch([], heads=1, kv_heads=1, dim=8, page=4096, layers=1, layer=0)
    b.lens, b.tokens, b.pages, b.shape = [(most - 1, 1)], 1, width, (width, 1, 2, 4096, 1, 8)
    b.table = np.arange(width, dtype=np.uint32)[None]
    b.past, b.starts = np.array([most - 1], np.uint32), np.array([0, 1], np.uint32)
    Call(dev, kind, batch=b)()
    b.past[0] += 1
    Call(dev, kind, batch=b).refused("exceeds 2\\^31 - 8192 positions")
    b = Batch([(5, 1)], heads=1, kv_heads=1, dim=8)
    c = Call(dev, kind, batch=b)
    c.rows = most
    c()
    c.rows = most + 1
    c.refused("exceeds 2\\^31 - 8192 tokens")


@pytest.mark.parametrize("kind", ["attend", "prefix"])
def test_query_rows_near_31_bits_are_refused(dev, kind):
    b = Batch([(5, 1)], heads=8, kv_heads=1, dim=8)
    c = Call(dev, kind, batch=b)
    c.rows = ((1 << 31) - 8192) // 8
    c()
    c.rows += 1
    c.refused("exceeds 2\\^31 - 8192 query rows")


@pytest.mark.parametrize("kind", KINDS)
def test_kv_heads_past_16_bits_are_refused(dev, kind):
    b = Batch([], heads=1 << 16, kv_heads=1 << 16, dim=8, page=1, layers=1, layer=0, extra_pages=1)
    Call(dev, kind, batch=b)()
    b = Batch([], heads=(1 << 16) + 1, kv_heads=(1 << 16) + 1, dim=8, page=1, layers=1, layer=0, extra_pages=1)
    Call(dev, kind, batch=b).refused("support 65536 heads", Status.Unimplemented)


def test_dispatch_prepares_no_command(dev, monkeypatch):
    # A dispatch made once does not pay for one that is repeated.
    def refuse(*args):
        raise AssertionError("a Command was made")
    b = Batch(LENS)
    n = b.tokens * b.heads * b.dim
    x, state = Value.f32((b.tokens, b.heads * b.dim)), dev.f32(D.state_words(b.shape, b.dtype))
    ports = [dev.f32(n), *[dev.u32(a) for a in (b.table, b.past, b.starts)], state]
    out = dev.f32(n)
    monkeypatch.setattr(D, "Command", refuse)
    before = dev._lib.host_recorded()
    dev.dispatch(b.op(OpCode.PagedAttention, scale=1.0), ports, [x, *b.described(), b.state()], [out], [x], [3, 0, 0])
    assert dev._lib.host_recorded() == before + 1
    with pytest.raises(DeviceError, match="different lengths"):
        dev.dispatch(b.op(OpCode.PagedAttention), ports, [x], [out], [x], [3, 0, 0])
