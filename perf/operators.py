"""Paged KV-cache operators of the serving path: what is timed, their plain forms and their exact values.

Three operators work on one cache, a State value of shape [pages, layers, 2, page, kv_heads, head_dim] (F32, F16 or
BF16), and one description of a ragged batch: `table` [sequences, pages per sequence] names each sequence's pages in
order, `past` [sequences] counts the positions that it has cached, and the rows starts[b] .. starts[b + 1] of the
token-major inputs are its new tokens, at positions past[b], past[b] + 1, ...

  append   PagedAppend: rotates the new keys by their positions and writes keys and values into the pages
  attend   PagedAttention: causal attention over the pages, with a sliding window and first tokens that stay visible
  prefix   PrefixAttention: the same attention where all sequences begin with the same pages, those read once for all

Both attentions run after the append of the same tokens, so a token sees its own key. Sizes are those of the
Llama-3 8B and 70B shapes (32/8 and 64/8 heads of 128, or a tensor-parallel share of them) and of the small fixture
model (4/4 heads of 64)."""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_THETA = 500000.0


def _case(name, op, **kw):
    c = dict(name=name, op=op, heads=32, kv_heads=8, dim=128, page=16, layers=1, dtype="f32", seqs=1, short=0,
             new=1, past_lo=0, past_hi=0, window=0, sinks=0, prefix=0, gptj=False, lens=1)
    c.update(kw)
    return c


def listed():
    return [
        # One user's decode step: the smallest call, all latency.
        _case("append one token", "append", past_lo=511, past_hi=511, layers=4),
        # A serving batch's decode step into a 16-bit cache.
        _case("append 64 tokens bf16", "append", seqs=64, past_lo=100, past_hi=8000, dtype="bf16", layers=2),
        # Several prompts admitted at once.
        _case("append prompts", "append", seqs=7, new=2048, past_lo=0, past_hi=700, page=64),
        # One user early in a conversation.
        _case("decode one short", "attend", past_lo=511, past_hi=511, layers=4),
        # The benchmark's batch of 8 with conversations of different lengths.
        _case("decode 8 ragged", "attend", seqs=8, past_lo=1030, past_hi=8000),
        # A busy server: many sequences, from just begun to long.
        _case("decode 64 bf16", "attend", seqs=64, past_lo=300, past_hi=16000, dtype="bf16"),
        # Long streams held to a window with four sinks, one tensor-parallel share of the 70B shape.
        _case("decode streams f16", "attend", heads=16, kv_heads=2, seqs=24, past_lo=3000, past_hi=60000,
              window=4096, sinks=4, page=64, dtype="f16"),
        # Long prompts fed in chunks, with a window.
        _case("prefill chunks windowed", "attend", seqs=2, new=2048, short=0, past_lo=5000, past_hi=7001,
              window=4096, sinks=4, page=64),
        # Two prompts among decoding sequences in one call, on the fixture's heads and an odd page.
        _case("mixed batch", "attend", heads=4, kv_heads=4, dim=64, seqs=27, short=24, new=777, past_lo=3,
              past_hi=1500, page=5),
        # A few answers sampled from one question.
        _case("prefix 6 small", "prefix", heads=4, kv_heads=4, dim=64, seqs=6, prefix=777, past_lo=778,
              past_hi=1000),
        # A batch under one system prompt.
        _case("prefix 64 bf16", "prefix", seqs=64, prefix=8192, past_lo=8200, past_hi=9700, dtype="bf16"),
        # Many questions about one long document, the 70B shape.
        _case("prefix 128 long f16", "prefix", heads=64, kv_heads=8, seqs=128, prefix=32768, past_lo=32768,
              past_hi=33300, page=64, dtype="f16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "prefix"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (64, 8, 128), (16, 2, 128), (8, 1, 128), (4, 4, 64)])
    c = dict(op=op, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([5, 16, 16, 32, 64]),
             layers=rng.choice([1, 1, 2]), dtype=rng.choice(["f32", "f16", "bf16"]), seqs=_spread(rng, 1, 64), short=0,
             new=1, window=0, sinks=0, prefix=0, gptj=rng.random() < 0.3, lens=rng.randrange(1 << 20))
    if op == "append":
        c["new"] = _spread(rng, 1, max(1, 8192 // c["seqs"]))
        c["past_lo"] = rng.randrange(0, 300)
        c["past_hi"] = c["past_lo"] + _spread(rng, 1, 4000)
        return c
    if op == "prefix":
        c["prefix"] = _spread(rng, 17, 16000)
        c["past_lo"] = c["prefix"] + rng.randrange(0, 50)
        c["past_hi"] = c["past_lo"] + _spread(rng, 1, 800)
        c["new"] = rng.choice([1, 1, 1, 2, 4])
        return c
    c["past_lo"] = rng.randrange(0, 500)
    if rng.random() < 0.4:  # prompts, some with decoding sequences beside them
        c["seqs"] = _spread(rng, 1, 12)
        c["short"] = rng.randrange(0, c["seqs"])
        c["new"] = _spread(rng, 2, max(2, 1024 // c["seqs"]))
        c["past_hi"] = c["past_lo"] + _spread(rng, 1, 4000)
    else:
        c["past_hi"] = c["past_lo"] + _spread(rng, 1, min(60000, 300000 // c["seqs"]))
    if rng.random() < 0.4:
        c["window"], c["sinks"] = _spread(rng, 16, 4096), rng.choice([0, 1, 4, 16])
    return c


def _lengths(case):
    """(past, new) of every sequence, as the case alone gives them: the first `short` decode, the others bring up to
    `new` tokens (exactly `new` where that is at most 4)."""
    r = np.random.RandomState(case["lens"])
    n = case["seqs"]
    past = r.randint(case["past_lo"], case["past_hi"] + 1, n)
    new = np.full(n, case["new"]) if case["new"] <= 4 else r.randint(case["new"] // 2, case["new"] + 1, n)
    if case["new"] > 4 and not case["short"] and n > 1:
        new[0] = case["new"]
    new[: case["short"]] = 1
    return past.astype(np.int64), new.astype(np.int64)


def prepare(case, seed):
    past, new = _lengths(case)
    n, page, layers = case["seqs"], case["page"], case["layers"]
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    starts = np.concatenate([[0], np.cumsum(new)])
    need = -(-(past + new) // page)
    shared = -(-case["prefix"] // page)
    pages = int(shared + (need - shared).sum()) + 3
    r = np.random.RandomState(seed % (1 << 32))
    order = r.permutation(pages)
    table = np.zeros((n, int(need.max())), np.int64)
    used = shared
    for b in range(n):
        table[b, :shared] = order[:shared]
        table[b, shared : need[b]] = order[used : used + need[b] - shared]
        used += need[b] - shared
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = int(starts[-1])

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    # Keys have a few strong channels, as trained ones do; queries are scaled so that scores spread by one or two.
    strong = torch.ones(D, device="cuda")
    strong[torch.randperm(D, generator=g, device="cuda")[: D // 32]] = 4.0
    cache = normal(pages, layers, 2, page, Hkv, D, dtype=_DTYPES[case["dtype"]])
    cache[:, :, 0] *= strong.to(cache.dtype)
    state = dict(case=case, layer=layers - 1, cache=cache, tokens=T, max_new=int(new.max()),
                 host=(table.astype(np.uint32), past.astype(np.uint32), starts.astype(np.uint32)),
                 table=torch.from_numpy(table).cuda(), past=torch.from_numpy(past).cuda(),
                 starts=torch.from_numpy(starts).cuda())
    if case["op"] == "append":
        state["k"], state["v"] = normal(T, Hkv * D) * strong.repeat(Hkv), normal(T, Hkv * D)
    else:
        state["q"], state["out"] = normal(T, H * D), torch.zeros(T, H * D, device="cuda")
    if own:
        _bind(state)
    return state


# ---- the framework's operators ---------------------------------------------------------------------------------------

_device = []


class _Buffers:
    """The buffers of one state on the framework's device, given back when the state goes."""

    def __init__(self, dev):
        self.dev, self.ids = dev, []

    def __del__(self):
        for b in self.ids:
            self.dev.release(b)

    def u32(self, array):
        from starlight_b200.device import BufferRef
        b = self.dev.allocate_u32(array.size)
        self.ids.append(b)
        self.dev.upload_u32(b, array)
        return BufferRef(b, 0, array.size)

    def f32(self, tensor):
        """A buffer with the tensor's bytes and a tensor over the buffer's memory."""
        from starlight_b200.device import BufferRef
        words = tensor.numel() * tensor.element_size() // 4
        b = self.dev.allocate_f32(words)
        self.ids.append(b)
        self.dev.synchronize()
        view = torch.as_tensor(_Memory(self.dev.device_ptr(b), words, self), device="cuda")
        view = view.view(tensor.dtype).view(tensor.shape)
        view.copy_(tensor)
        return BufferRef(b, 0, words), view


class _Memory:
    def __init__(self, pointer, words, keep):
        self.keep = keep
        self.__cuda_array_interface__ = dict(shape=(words,), typestr="<f4", data=(pointer, False), version=3)


def _bind(s):
    """Puts the state's tensors on the framework's device and makes the command that a step dispatches."""
    from starlight_b200.device import CudaDevice, DType, Op, OpCode, RopeVariant, Value, ValueRole
    if not _device:
        _device.append(CudaDevice(0))
    dev, c = _device[0], s["case"]
    buffers = _Buffers(dev)
    table, past, starts = (buffers.u32(a) for a in s["host"])
    described = [Value.u32(a.shape) for a in s["host"]]
    cache, s["cache"] = buffers.f32(s["cache"])
    state = Value(DType[c["dtype"].upper()], tuple(s["cache"].shape), ValueRole.State)
    T, kv, hd = s["tokens"], c["kv_heads"] * c["dim"], c["heads"] * c["dim"]
    attrs = dict(layer=s["layer"], heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["dim"])
    if c["op"] == "append":
        (k, s["k"]), (v, s["v"]) = buffers.f32(s["k"]), buffers.f32(s["v"])
        op = Op(OpCode.PagedAppend, theta=_THETA, variant=RopeVariant.GptJ if c["gptj"] else RopeVariant.Neox, **attrs)
        s["call"] = dev.command(op, [k, v, table, past, starts, cache],
                                [Value.f32((T, kv)), Value.f32((T, kv)), *described, state], [], [])
    else:
        (q, s["q"]), (out, s["out"]) = buffers.f32(s["q"]), buffers.f32(s["out"])
        prefix = c["op"] == "prefix"
        op = Op(OpCode.PrefixAttention if prefix else OpCode.PagedAttention, scale=1 / math.sqrt(c["dim"]), **attrs)
        scalars = [s["max_new"], c["prefix"]] if prefix else [s["max_new"], c["window"], c["sinks"]]
        s["call"] = dev.command(op, [q, table, past, starts, cache], [Value.f32((T, hd)), *described, state],
                                [out], [Value.f32((T, hd))], scalars)
    torch.cuda.synchronize()


# ---- the plain forms ---------------------------------------------------------------------------------------------------


def _tokens(s):
    """Sequence and position of every new token."""
    t = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["starts"][1:], t, right=True)
    return b, s["past"][b] + t - s["starts"][b]


def _append(s):
    c = s["case"]
    Hkv, D, page = c["kv_heads"], c["dim"], c["page"]
    b, pos = _tokens(s)
    pair = torch.arange(D // 2, device="cuda", dtype=torch.float64)
    angle = pos.double()[:, None] / _THETA ** (2 * pair / D)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    k = s["k"].view(-1, Hkv, D)
    first, second = (k[..., 0::2], k[..., 1::2]) if c["gptj"] else (k[..., : D // 2], k[..., D // 2 :])
    turned = [first * cos - second * sin, first * sin + second * cos]
    k = torch.stack(turned, -1).view(-1, Hkv, D) if c["gptj"] else torch.cat(turned, -1)
    where, off = s["table"][b, pos // page], pos % page
    cache = s["cache"]
    cache[where, s["layer"], 0, off] = k.to(cache.dtype)
    cache[where, s["layer"], 1, off] = s["v"].view(-1, Hkv, D).to(cache.dtype)
    return cache


def _rows(s, b, pos):
    """Keys and values [..., kv_heads, head_dim] in 32 bits at positions `pos` of sequences `b`."""
    page = s["case"]["page"]
    at = (s["table"][b, pos // page], s["layer"])
    return s["cache"][(*at, 0, pos % page)].float(), s["cache"][(*at, 1, pos % page)].float()


def _padded(s):
    """Queries as [sequences, kv_heads, group * max_new, head_dim], and (sequence, place) of every token."""
    c = s["case"]
    n, H, Hkv, D, M = c["seqs"], c["heads"], c["kv_heads"], c["dim"], s["max_new"]
    b, pos = _tokens(s)
    place = pos - s["past"][b]
    q = torch.zeros(n, M, H, D, device="cuda")
    q[b, place] = s["q"].view(-1, H, D)
    return q.view(n, M, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(n, Hkv, -1, D), b, place


def _unpadded(s, o, b, place):
    c = s["case"]
    n, H, Hkv, D, M = c["seqs"], c["heads"], c["kv_heads"], c["dim"], s["max_new"]
    o = o.view(n, Hkv, H // Hkv, M, D).permute(0, 3, 1, 2, 4).reshape(n, M, H * D)
    return o[b, place]


def _own_keys(s, q, first):
    """Masked scores of the padded queries against each sequence's keys from `first` on (and its sinks, where it has a
    window), and those keys' values."""
    c = s["case"]
    M, window, sinks = s["max_new"], c["window"], c["sinks"]
    end = s["past"] + s["starts"][1:] - s["starts"][:-1]
    low = torch.full_like(s["past"], first)
    if window:
        low = torch.clamp(s["past"] + 1 - window, min=sinks)
    count = int((end - low).max()) + sinks  # the program knows its lengths
    j = torch.arange(count, device="cuda")[None]
    pos = torch.where(j < sinks, j, low[:, None] + j - sinks)
    real = pos < end[:, None]
    k, v = _rows(s, torch.arange(c["seqs"], device="cuda")[:, None], pos * real)
    k, v = k.permute(0, 2, 3, 1), v.permute(0, 2, 1, 3)
    score = (q @ k).view(c["seqs"], c["kv_heads"], -1, M, count) / math.sqrt(c["dim"])
    at = (s["past"][:, None] + torch.arange(M, device="cuda"))[:, :, None]
    seen = real[:, None] & (pos[:, None] <= at)
    if window:
        seen = seen & ((pos[:, None] > at - window) | (pos[:, None] < sinks))
    score = torch.where(seen[:, None, None], score, -math.inf).view(c["seqs"], c["kv_heads"], -1, count)
    return score, v


def _attend(s):
    q, b, place = _padded(s)
    score, v = _own_keys(s, q, 0)
    # Places without a token may see nothing: their rows are not returned.
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
    return _unpadded(s, (p @ v) / p.sum(-1, keepdim=True), b, place)


def _prefix(s):
    c = s["case"]
    n, Hkv, D = c["seqs"], c["kv_heads"], c["dim"]
    q, b, place = _padded(s)
    pos = torch.arange(c["prefix"], device="cuda")
    k, v = _rows(s, torch.zeros_like(pos), pos)
    shared = q.transpose(0, 1).reshape(Hkv, -1, D) @ k.permute(1, 2, 0) / math.sqrt(D)
    score, v_own = _own_keys(s, q, c["prefix"])
    top = torch.maximum(shared.amax(-1).view(Hkv, n, -1).transpose(0, 1), score.amax(-1))[..., None]
    p_shared = torch.exp(shared - top.transpose(0, 1).reshape(Hkv, -1, 1))
    p = torch.exp(score - top)
    o = (p_shared @ v.transpose(0, 1)).view(Hkv, n, -1, D).transpose(0, 1) + p @ v_own
    total = p_shared.sum(-1, keepdim=True).view(Hkv, n, -1, 1).transpose(0, 1) + p.sum(-1, keepdim=True)
    return _unpadded(s, o / total, b, place)


def run(state):
    if own:
        state["call"]()
        return state["cache"] if state["case"]["op"] == "append" else state["out"]
    return {"append": _append, "attend": _attend, "prefix": _prefix}[state["case"]["op"]](state)


# ---- what a pass cannot do without, and exact values --------------------------------------------------------------------


def _visible(case):
    """(distinct keys read, query-key pairs) of one layer's pass, for one key/value head and one query head."""
    past, new = _lengths(case)
    window, sinks, prefix = case["window"], case["sinks"], case["prefix"]
    keys, pairs = (prefix, int((new * prefix).sum())) if prefix else (0, 0)
    for p, m in zip(past, new):
        at = np.arange(p, p + m)
        seen = at + 1 - prefix
        if window:
            low = np.maximum(at + 1 - window, 0)
            seen = np.where(low > sinks, at + 1 - low + sinks, at + 1)
            keys += int(min(p + m, p + m - max(p + 1 - window, 0) + min(sinks, max(p + 1 - window, 0))))
        else:
            keys += int(p + m - prefix)
        pairs += int(seen.sum())
    return keys, pairs


def work(case):
    past, new = _lengths(case)
    T, size = int(new.sum()), 4 if case["dtype"] == "f32" else 2
    kv, hd = case["kv_heads"] * case["dim"], case["heads"] * case["dim"]
    described = 4 * (int((-(-(past + new) // case["page"])).sum()) + 2 * case["seqs"] + 1)
    if case["op"] == "append":
        return {"bytes": 2 * T * kv * (4 + size) + 4 * (3 * case["seqs"] + 1), "flops": 3 * T * kv}
    keys, pairs = _visible(case)
    return {"bytes": 2 * keys * kv * size + 8 * T * hd + described, "flops": 4 * pairs * hd}


def exact(case, seed):
    s, c = prepare(case, seed), case
    H, Hkv, D, page, layer = c["heads"], c["kv_heads"], c["dim"], c["page"], s["layer"]
    table, past, starts = (a.astype(np.int64) for a in s["host"])
    if c["op"] == "append":
        cache = s["cache"].double()
        for b in range(c["seqs"]):
            n = int(starts[b + 1] - starts[b])
            pos = int(past[b]) + torch.arange(n, device="cuda")
            k = s["k"][starts[b] : starts[b + 1]].double().view(n, Hkv, D)
            z = torch.view_as_complex(k.view(n, Hkv, D // 2, 2) if c["gptj"] else
                                      torch.stack([k[..., : D // 2], k[..., D // 2 :]], -1))
            w = _THETA ** (-2 * torch.arange(D // 2, device="cuda", dtype=torch.float64) / D)
            z = torch.view_as_real(z * torch.polar(torch.ones_like(w), pos.double()[:, None] * w)[:, None])
            k = z.reshape(n, Hkv, D) if c["gptj"] else torch.cat([z[..., 0], z[..., 1]], -1)
            rows = torch.from_numpy(table[b]).cuda()[pos // page], layer
            cache[(*rows, 0, pos % page)] = k
            cache[(*rows, 1, pos % page)] = s["v"][starts[b] : starts[b + 1]].double().view(n, Hkv, D)
        return cache
    out = torch.zeros(s["tokens"], H, D, device="cuda", dtype=torch.float64)
    for b in range(c["seqs"]):
        t0, t1, end = int(starts[b]), int(starts[b + 1]), int(past[b] + starts[b + 1] - starts[b])
        if t0 == t1:
            continue
        used = torch.from_numpy(table[b]).cuda()[: -(-end // page)]
        kv = s["cache"][used, layer].double()  # [pages, 2, page, kv_heads, head_dim]
        kv = kv.permute(1, 3, 0, 2, 4).reshape(2, Hkv, -1, D)[:, :, :end]
        at, pos = torch.arange(end - (t1 - t0), end, device="cuda")[:, None], torch.arange(end, device="cuda")[None]
        hidden = pos > at
        if c["window"]:
            hidden |= (pos <= at - c["window"]) & (pos >= c["sinks"])
        for h in range(H):
            a = s["q"][t0:t1].view(-1, H, D)[:, h].double() @ kv[0, h * Hkv // H].T / math.sqrt(D)
            out[t0:t1, h] = torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ kv[1, h * Hkv // H]
    return out.view(-1, H * D)
