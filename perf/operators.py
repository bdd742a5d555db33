"""The operators that serve requests behind one shared prefix (an instruction, few-shot examples, a
document), as calls of the public Python binding (qattn.py) that can be timed and compared: rotary
positions, the paged K/V cache's write and read, and attention of a batch over the cached prefix and
its own keys.

A case is a dict of plain values.  `kind` names the call:

  rope    Context.rope: q and k head vectors rotated to given positions
  write   Context.kv_write: K and V rows into cache slots, quantised as they are written
  read    Context.kv_read: cache slots back into rows
  attend  SharedRun.encode: packed queries over `prefix` cached keys and their own keys

`queries` and `own` are packed lengths ("1*16", "37,150*2"): the queries of a sequence are the last
positions of its own keys.  With `own` a false value every own key is a query's (a whole prompt)."""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LOCAL_PREFIX, LOCAL_WINDOW = 176, 432  # the model's sparse mask
THETA, YARN_CONTEXT, YARN_FAST, YARN_SLOW = 1e6, 32768, 32.0, 1.0
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
MOST_FLOPS, MOST_ROWS = 3.4e11, 20000


def listed():
    return [
        # One step of 16 requests behind a 500-token instruction, a few tokens of their own each:
        # the smallest call, where latency counts.
        {"name": "step_16", "kind": "attend", "queries": "1*16", "own": "9,1,30,17,4,22,12,27,6,31,19,3,25,14,8,11",
         "prefix": 500, "heads": 16, "kv_heads": 8, "dim": 128, "dtype": "f16", "cache": "e4m3", "page": 16,
         "own_in": "pages", "mask": "causal"},
        # One step of 64 requests behind a document of 8,192 tokens in an int8 cache.
        {"name": "step_64_long", "kind": "attend", "queries": "1*64",
         "own": "150,37,600,1,222,95*5,412,333,77*4,512*6,18,240,64*8,589,131*9,301,45*7,260,3,199*5,470,88,160*5",
         "prefix": 8192, "heads": 16, "kv_heads": 8, "dim": 128, "dtype": "f16", "cache": "int8", "page": 64,
         "own_in": "pages", "mask": "causal"},
        # A step of 8 conversations, seven query heads to a key head, in a bf16 cache.
        {"name": "step_8_group7", "kind": "attend", "queries": "1*8", "own": "1500,700,33,1201,64,950,410,1",
         "prefix": 4000, "heads": 28, "kv_heads": 4, "dim": 128, "dtype": "bf16", "cache": "16bit", "page": 32,
         "own_in": "pages", "mask": "causal"},
        # A micro-batch of 16 short queries behind an instruction, under the model's sparse mask; their
        # own K and V are the projections' rows and never enter the cache.
        {"name": "queries_16_ragged", "kind": "attend",
         "queries": "36,84,150,10,121,67,139,95,52,143,18,110,78,129,101,86", "own": "",
         "prefix": 500, "heads": 16, "kv_heads": 8, "dim": 128, "dtype": "f16", "cache": "16bit", "page": 64,
         "own_in": "rows", "mask": "prefix_local"},
        # 16 documents of 500 tokens behind 5,000 tokens of examples: the largest.
        {"name": "documents_16x500", "kind": "attend", "queries": "500*16", "own": "", "prefix": 5000, "heads": 16,
         "kv_heads": 8, "dim": 128, "dtype": "f16", "cache": "e4m3", "page": 64, "own_in": "rows", "mask": "causal"},
        # A chunk of one long document read in pieces: its last 1,500 tokens, 2,500 earlier ones in the
        # int8 cache, heads of 64.
        {"name": "chunk_1500_dim64", "kind": "attend", "queries": "1500", "own": "2500", "prefix": 1500, "heads": 16,
         "kv_heads": 8, "dim": 64, "dtype": "bf16", "cache": "int8", "page": 16, "own_in": "pages", "mask": "causal"},
        # The 16 new tokens of a step, half of each head rotated in pairs of neighbours.
        {"name": "rope_16", "kind": "rope", "tokens": 16, "heads": 28, "kv_heads": 4, "dim": 128, "rotary": 64,
         "layout": "interleaved", "dtype": "bf16", "scaling": "linear", "factor": 4.0, "far": 30000, "in_qkv": False},
        # A full batch, Q and K in place of the projection's rows, positions past the trained context.
        {"name": "rope_8000_far", "kind": "rope", "tokens": 8000, "heads": 16, "kv_heads": 8, "dim": 128, "rotary": 128,
         "layout": "half", "dtype": "f16", "scaling": "yarn", "factor": 4.0, "far": 131000, "in_qkv": True},
        # The new keys of a step of 64 requests.
        {"name": "write_64", "kind": "write", "tokens": 64, "kv_heads": 8, "dim": 128, "dtype": "f16", "cache": "int8",
         "page": 64},
        # A full batch's keys.
        {"name": "write_8000", "kind": "write", "tokens": 8000, "kv_heads": 8, "dim": 128, "dtype": "f16",
         "cache": "e4m3", "page": 64},
        # An instruction's keys back into rows.
        {"name": "read_500", "kind": "read", "tokens": 500, "kv_heads": 4, "dim": 128, "dtype": "bf16", "cache": "int8",
         "page": 32},
        # Four documents' keys back into rows.
        {"name": "read_20000", "kind": "read", "tokens": 20000, "kv_heads": 8, "dim": 128, "dtype": "f16",
         "cache": "e4m3", "page": 16},
    ]


def _log_int(rng, low, high):
    return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _lengths_text(lengths):
    return ",".join(str(n) for n in lengths)


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "attend", "rope", "write", "read"))
    case = {"kind": kind, "dtype": rng.choice(("f16", "bf16"))}
    case["heads"], case["kv_heads"] = rng.choice(((16, 8), (16, 8), (28, 4), (8, 8), (12, 1), (32, 8)))
    case["dim"] = rng.choice((64, 128, 128))
    if kind == "rope":
        rotary = rng.choice((case["dim"], case["dim"], case["dim"] // 2, 48))
        scaling = rng.choice(("none", "linear", "yarn"))
        return {**case, "tokens": _log_int(rng, 1, MOST_ROWS), "rotary": rotary,
                "layout": rng.choice(("half", "interleaved")), "scaling": scaling,
                "factor": 1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)),
                "far": _log_int(rng, 10, 1 << 20), "in_qkv": rng.random() < 0.5}
    case["cache"], case["page"] = rng.choice(("16bit", "e4m3", "int8")), rng.choice((16, 32, 64, 128))
    if kind != "attend":
        del case["heads"]
        return {**case, "tokens": _log_int(rng, 1, MOST_ROWS)}
    case["prefix"] = 0 if rng.random() < 0.1 else _log_int(rng, 1, 8192)
    case["own_in"], case["mask"] = rng.choice(("rows", "pages")), rng.choice(("causal", "causal", "prefix_local"))
    if rng.random() < 0.5:  # a step: one token each, seldom a few
        count = _log_int(rng, 1, 64)
        queries = [1 if rng.random() < 0.8 else rng.randint(1, 8) for _ in range(count)]
        top = _log_int(rng, 1, 2000)
        lengths = [max(n, rng.randint(1, top)) for n in queries]
        return {**case, "queries": _lengths_text(queries), "own": _lengths_text(lengths)}
    count = rng.choice((1, 1, 2, 4, 8, 16))
    top = _log_int(rng, 8, 8000 // count)
    queries = [rng.randint(max(1, top // 8), top) for _ in range(count)]
    while sum(queries) * case["heads"] * case["dim"] * 4 * (case["prefix"] + max(queries)) > MOST_FLOPS:
        queries = [n // 2 + 1 for n in queries]
        case["prefix"] = case["prefix"] * 3 // 4
    return {**case, "queries": _lengths_text(queries), "own": ""}


# ---- the library ----------------------------------------------------------------------------


def _binding():
    if "qattn" not in sys.modules:
        path = os.path.join(ROOT, "qwen3-embedding-webgpu-prepacked_amd", "qattn.py")
        spec = importlib.util.spec_from_file_location("qattn", path)
        sys.modules["qattn"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["qattn"])
    return sys.modules["qattn"]


_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        _ctx = _binding().Context(0)
    return _ctx


# ---- inputs ---------------------------------------------------------------------------------


class State:
    """What a program holds between calls; the library's handles are released with it."""

    def __init__(self, **parts):
        self.run = None
        self.__dict__.update(parts)

    def __del__(self):
        if self.run is not None:
            self.run.destroy()


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _lengths(text):
    out = []
    for part in text.split(","):
        length, _, times = part.partition("*")
        out += [int(length)] * int(times or 1)
    return np.array(out, dtype=np.int64)


def _offsets(lengths):
    return np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)


def _own_lengths(case):
    return _lengths(case["own"] or case["queries"])


def _slots(case, g, count):
    """Slots of `count` tokens in order, in pages taken from the pool in no order."""
    used = -(-count // case["page"])
    pages = used + used // 4 + 1
    order = torch.randperm(pages, generator=g, device="cuda")
    token = torch.arange(count, device="cuda")
    return pages, order[token // case["page"]] * case["page"] + token % case["page"]


def _pool(case, g, pages):
    """A pool of pages as writes leave it: (k, v, k_scale, v_scale), values of unit variance."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    if case["cache"] == "16bit":
        return _normal(g, DTYPES[case["dtype"]], *shape), _normal(g, DTYPES[case["dtype"]], *shape), None, None
    pairs = [_quantised(_normal(g, DTYPES[case["dtype"]], *shape), case["cache"]) for _ in range(2)]
    return pairs[0][0], pairs[1][0], pairs[0][1], pairs[1][1]


def _rope_inputs(case, seed):
    g = _generator(seed)
    tokens, dim = case["tokens"], case["dim"]
    q_width, k_width = case["heads"] * dim, case["kv_heads"] * dim
    row = q_width + 2 * k_width if case["in_qkv"] else q_width + k_width
    rows = _normal(g, DTYPES[case["dtype"]], tokens, row)
    far = torch.randint(0, max(1, case["far"] - tokens), (1,), generator=g, device="cuda")
    positions = (far + torch.arange(tokens, device="cuda")).to(torch.int32)
    return rows, positions


def _cache_inputs(case, seed):
    """(pool, slots, rows of K, rows of V) of a write or a read."""
    g = _generator(seed)
    pages, slots = _slots(case, g, case["tokens"])
    width, dtype = case["kv_heads"] * case["dim"], DTYPES[case["dtype"]]
    if case["kind"] == "read":
        return _pool(case, g, pages), slots, None, None
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    stored = {"16bit": dtype, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}[case["cache"]]
    pool = [torch.zeros(shape, device="cuda", dtype=stored) for _ in range(2)]
    pool += [None, None] if case["cache"] == "16bit" else [torch.zeros(shape[:3], device="cuda") for _ in range(2)]
    # Keys and values as projected: heads and channels of unlike sizes.
    k, v = (_normal(g, torch.float32, case["tokens"], width) *
            torch.exp(0.7 * torch.randn(width, generator=g, device="cuda")) for _ in range(2))
    return tuple(pool), slots, k.to(dtype), v.to(dtype)


def _attend_inputs(case, seed):
    g, dtype = _generator(seed), DTYPES[case["dtype"]]
    queries, lengths, page = _lengths(case["queries"]), _own_lengths(case), case["page"]
    q = _normal(g, dtype, int(queries.sum()), case["heads"] * case["dim"])
    paged = case["own_in"] == "pages"
    need = [-(-case["prefix"] // page)] + ([-(-int(n) // page) for n in lengths] if paged else [])
    pages = sum(need) + sum(need) // 4 + 1
    order = np.random.RandomState(seed % (1 << 32)).permutation(pages).astype(np.int32)
    ends = np.cumsum(need)
    tables = [order[a:b] for a, b in zip(ends - need, ends)]
    pool = _pool(case, g, pages)
    k = v = None
    if not paged:
        k, v = (_normal(g, dtype, int(lengths.sum()), case["kv_heads"] * case["dim"]) for _ in range(2))
    return q, pool, tables, k, v


def prepare(case, seed):
    kind = case["kind"]
    if kind == "rope":
        rows, positions = _rope_inputs(case, seed)
        dtype, tokens = DTYPES[case["dtype"]], case["tokens"]
        out = [torch.zeros(tokens, case[h] * case["dim"], device="cuda", dtype=dtype) for h in ("heads", "kv_heads")]
        state = State(case=case, rows=rows, positions=positions, out=out, turns=_frequencies(case).cuda())
        if own:
            b = _binding()
            width = case["heads"] * case["dim"]
            scaling = {"none": b.ROPE_PLAIN, "linear": b.ROPE_LINEAR, "yarn": b.ROPE_YARN}[case["scaling"]]
            layout = {"half": b.ROPE_HALF, "interleaved": b.ROPE_INTERLEAVED}[case["layout"]]
            state.desc = b.make_rope_desc(
                positions.data_ptr(), tokens, q=(rows.data_ptr(), out[0].data_ptr(), case["heads"]),
                k=(rows[:, width:].data_ptr(), out[1].data_ptr(), case["kv_heads"]), head_dim=case["dim"],
                rotary_dim=case["rotary"], layout=layout, dtype=b.BF16 if case["dtype"] == "bf16" else b.F16,
                q_row_stride=rows.shape[1], k_row_stride=rows.shape[1], theta=THETA, scaling=scaling,
                factor=case["factor"], original_context=YARN_CONTEXT, beta_fast=YARN_FAST, beta_slow=YARN_SLOW)
            state.ctx = _context()
        return state
    if kind in ("write", "read"):
        pool, slots, k, v = _cache_inputs(case, seed)
        state = State(case=case, pool=pool, slots=slots, k=k, v=v)
        if kind == "read":
            width, dtype = case["kv_heads"] * case["dim"], DTYPES[case["dtype"]]
            state.out = [torch.zeros(case["tokens"], width, device="cuda", dtype=dtype) for _ in range(2)]
        if own:
            state.cache, state.ctx = _own_cache(case, pool), _context()
        return state
    q, pool, tables, k, v = _attend_inputs(case, seed)
    queries, lengths = _lengths(case["queries"]), _own_lengths(case)
    state = State(case=case, q=q, pool=pool, k=k, v=v, out=torch.zeros_like(q), tables=tables)
    # The packing as index tensors, which the plain form gathers by.
    longest_q, longest_k = int(queries.max()), int(lengths.max())
    step_q, step_k = np.arange(longest_q), np.arange(longest_k)
    starts_q, starts_k = _offsets(queries)[:-1, None], _offsets(lengths)[:-1, None]
    to_gpu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    state.pad_q = to_gpu(starts_q + np.minimum(step_q, queries[:, None] - 1).clip(0))
    state.pad_k = to_gpu(starts_k + np.minimum(step_k, lengths[:, None] - 1).clip(0))
    state.seq = to_gpu(np.repeat(np.arange(len(queries)), queries))
    state.step = to_gpu(np.concatenate([np.arange(n) for n in queries]))
    state.position = to_gpu(case["prefix"] + np.repeat(lengths - queries, queries)) + state.step
    state.lengths = to_gpu(lengths)
    state.prefix_table = to_gpu(tables[0]).long()
    if case["own_in"] == "pages":
        width = max(len(t) for t in tables[1:])
        state.own_table = to_gpu(np.stack([np.pad(t, (0, width - len(t))) for t in tables[1:]])).long()
    if own:
        b = _binding()
        paged = case["own_in"] == "pages"
        desc = b.make_shared_desc(
            q.data_ptr(), state.out.data_ptr(), _own_cache(case, pool), _offsets(queries), lengths,
            q_heads=case["heads"], prefix_pages=tables[0], prefix_len=case["prefix"],
            own_pages=np.concatenate(tables[1:]) if paged else None, k=None if paged else k.data_ptr(),
            v=None if paged else v.data_ptr(),
            mask=b.MASK_CAUSAL if case["mask"] == "causal" else b.MASK_PREFIX_LOCAL, prefix=LOCAL_PREFIX,
            window=LOCAL_WINDOW)
        state.run = _context().shared_run(desc)
    return state


def _own_cache(case, pool):
    b = _binding()
    fmt = {"16bit": b.KV_16BIT, "e4m3": b.KV_E4M3, "int8": b.KV_INT8}[case["cache"]]
    k_scale, v_scale = (None if s is None else s.data_ptr() for s in pool[2:])
    return b.make_kv_cache(pool[0].data_ptr(), pool[1].data_ptr(), len(pool[0]), case["page"], case["kv_heads"],
                           case["dim"], dtype=b.BF16 if case["dtype"] == "bf16" else b.F16, format=fmt,
                           k_scale=k_scale, v_scale=v_scale)


# ---- a pass ---------------------------------------------------------------------------------


def run(state):
    kind = state.case["kind"]
    if not own:
        return {"rope": _plain_rope, "write": _plain_write, "read": _plain_read, "attend": _plain_attend}[kind](state)
    if kind == "rope":
        state.ctx.rope(state.desc)
        return state.out
    if kind == "write":
        state.ctx.kv_write(state.cache, state.k.data_ptr(), state.v.data_ptr(), state.slots.data_ptr(),
                           state.case["tokens"])
        return state.pool
    if kind == "read":
        state.ctx.kv_read(state.cache, state.slots.data_ptr(), state.case["tokens"], state.out[0].data_ptr(),
                          state.out[1].data_ptr())
        return state.out
    state.run.encode()
    return state.out


# ---- the plain forms ------------------------------------------------------------------------


def _frequencies(case):
    """Angle per position of each pair, in 64 bits."""
    pair = torch.arange(case["rotary"] // 2, dtype=torch.float64)
    f = THETA ** (-2 * pair / case["rotary"])
    if case["scaling"] == "linear":
        f = f / case["factor"]
    if case["scaling"] == "yarn":
        def turns(n):  # the pair that turns n times in the original context
            return case["rotary"] * math.log(YARN_CONTEXT / (n * 2 * math.pi)) / (2 * math.log(THETA))
        low = max(math.floor(turns(YARN_FAST)), 0)
        high = min(math.ceil(turns(YARN_SLOW)), case["rotary"] - 1)
        ramp = ((pair - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / case["factor"] * ramp
    return f


def _magnitude(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "yarn" else 1.0


def _plain_rope(state):
    case = state.case
    tokens, dim, rotary, half = case["tokens"], case["dim"], case["rotary"], case["rotary"] // 2
    angle = state.positions.double()[:, None] * state.turns  # far positions: 32 bits would lose the angle
    cos = (torch.cos(angle) * _magnitude(case)).float()[:, None, :]
    sin = (torch.sin(angle) * _magnitude(case)).float()[:, None, :]

    def rotated(x):
        x = x.reshape(tokens, -1, dim).float()
        a, b = (x[..., :half], x[..., half:rotary]) if case["layout"] == "half" else (x[..., 0:rotary:2], x[..., 1:rotary:2])
        a, b = a * cos - b * sin, b * cos + a * sin
        turned = torch.cat([a, b], -1) if case["layout"] == "half" else torch.stack([a, b], -1).flatten(-2)
        return torch.cat([turned, x[..., rotary:]], -1).to(DTYPES[case["dtype"]]).reshape(tokens, -1)

    width = case["heads"] * dim
    return [rotated(state.rows[:, :width]), rotated(state.rows[:, width:width + case["kv_heads"] * dim])]


def _quantised(x, form):
    """(codes, scales) of vectors along the last axis: e4m3 with the least power of two that fits the
    largest value into 448, int8 with the largest value over 127."""
    x = x.float()
    most = x.abs().amax(-1)
    if form == "int8":
        full = torch.full_like(most, 127.0)
        scale = torch.where(most > 0, most / full, torch.ones_like(most))
        codes = torch.round(x * torch.where(most > 0, full / most, torch.ones_like(most))[..., None])
        return codes.to(torch.int8), scale
    mantissa, exponent = torch.frexp(most)  # most = mantissa 2^exponent, mantissa in [0.5, 1)
    exponent = exponent - 9 + (mantissa > 448.0 / 512.0).to(exponent.dtype)
    scale = torch.where(most > 0, torch.ldexp(torch.ones_like(most), exponent), torch.ones_like(most))
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _put(pool, slots, page, values):
    narrow = values.element_size() == 1
    target, values = (pool.view(torch.uint8), values.view(torch.uint8)) if narrow else (pool, values)
    target[slots // page, :, slots % page] = values


def _plain_write(state):
    case, pool = state.case, state.pool
    shape = (case["tokens"], case["kv_heads"], case["dim"])
    if case["cache"] == "16bit":
        _put(pool[0], state.slots, case["page"], state.k.view(shape))
        _put(pool[1], state.slots, case["page"], state.v.view(shape))
        return pool
    k, k_scale = _quantised(state.k.view(shape), case["cache"])
    v, v_scale = _quantised(state.v.view(shape), case["cache"])
    _put(pool[0], state.slots, case["page"], k)
    _put(pool[1], state.slots, case["page"], v)
    _put(pool[2], state.slots, case["page"], k_scale)
    _put(pool[3], state.slots, case["page"], v_scale)
    return pool


def _values(codes, scale):
    return codes.float() if scale is None else codes.float() * scale[..., None]


def _narrow(codes):
    """A view that can be indexed: 8-bit floats by their bytes."""
    return codes.view(torch.uint8) if codes.dtype == torch.float8_e4m3fn else codes


def _taken(codes, *index):
    return _narrow(codes)[index].view(codes.dtype)


def _plain_read(state):
    case, pool = state.case, state.pool
    index = (state.slots // case["page"], slice(None), state.slots % case["page"])
    rows = [_values(_taken(c, *index), None if s is None else s[index]) for c, s in zip(pool[:2], pool[2:])]
    return [r.to(DTYPES[case["dtype"]]).reshape(case["tokens"], -1) for r in rows]


def _plain_attend(state):
    case = state.case
    dim, kv, prefix = case["dim"], case["kv_heads"], case["prefix"]
    group = case["heads"] // kv
    tokens, sequences = len(state.q), len(state.lengths)

    def pages_of(codes, scale, table):  # [..., pages] -> [..., kv, keys, dim]
        x = _values(_taken(codes, table), None if scale is None else scale[table])
        return x.movedim(-3, -4).flatten(-3, -2)

    shared = [pages_of(c, s, state.prefix_table)[:, :prefix] for c, s in zip(state.pool[:2], state.pool[2:])]
    if case["own_in"] == "pages":
        mine = [pages_of(c, s, state.own_table) for c, s in zip(state.pool[:2], state.pool[2:])]
    else:
        mine = [x[state.pad_k].float().view(sequences, -1, kv, dim).transpose(1, 2) for x in (state.k, state.v)]
    keys = mine[0].shape[2]
    q = state.q.float().view(tokens, kv, group, dim) / math.sqrt(dim)

    def seen(position, at):
        keep = at <= position
        if case["mask"] == "prefix_local":
            keep = keep & ((at < LOCAL_PREFIX) | (at + LOCAL_WINDOW > position))
        return keep

    # Scores over the shared keys [kv, tokens, group, prefix] and over each sequence's own, for which
    # the queries are padded to [sequences, kv, longest, group, dim] and the scores packed again.
    at = torch.arange(prefix, device="cuda")
    far = (q.permute(1, 0, 2, 3).reshape(kv, tokens * group, dim) @ shared[0].transpose(1, 2)).view(kv, tokens, group, prefix)
    far = far.masked_fill(~seen(state.position[:, None], at)[None, :, None], -math.inf)
    padded = q[state.pad_q].permute(0, 2, 1, 3, 4)
    longest = padded.shape[2]
    near = padded.reshape(sequences, kv, longest * group, dim) @ mine[0].transpose(2, 3)
    near = near.view(sequences, kv, longest, group, keys)
    place = torch.arange(keys, device="cuda")
    where = state.position[state.pad_q]
    keep = seen(where[..., None], prefix + place) & (place < state.lengths[:, None, None])
    near = near.masked_fill(~keep[:, None, :, None], -math.inf)
    near_rows = near[state.seq, :, state.step].transpose(0, 1)  # [kv, tokens, group, keys]
    most = near_rows.amax(-1) if not prefix else torch.maximum(near_rows.amax(-1), far.amax(-1))
    most = torch.where(most == -math.inf, torch.zeros_like(most), most)
    far = torch.exp(far - most[..., None])
    near = torch.exp(near - most.transpose(0, 1)[state.pad_q].permute(0, 2, 1, 3)[..., None])
    total = far.sum(-1) + near.sum(-1)[state.seq, :, state.step].transpose(0, 1)
    out = (far.view(kv, tokens * group, prefix) @ shared[1]).view(kv, tokens, group, dim)
    close = (near.view(sequences, kv, longest * group, keys) @ mine[1]).view(sequences, kv, longest, group, dim)
    out = out + close[state.seq, :, state.step].transpose(0, 1)
    out = torch.where(total[..., None] > 0, out / total[..., None], torch.zeros_like(out))
    return out.permute(1, 0, 2, 3).reshape(tokens, -1).to(DTYPES[case["dtype"]])


# ---- what a pass cannot do without ----------------------------------------------------------


def _seen_pairs(case):
    """(visible (query, key) pairs, shared keys that some query sees, own keys that some query sees)."""
    queries, lengths, prefix = _lengths(case["queries"]), _own_lengths(case), case["prefix"]
    position = prefix + np.repeat(lengths - queries, queries) + np.concatenate([np.arange(n) for n in queries])
    count, shared, mine = position + 1, prefix, int(lengths.sum())
    if case["mask"] == "prefix_local":
        always = np.minimum(position + 1, LOCAL_PREFIX)
        count = always + (position - np.maximum(position - LOCAL_WINDOW + 1, always) + 1).clip(0)
        start = prefix + lengths - queries - LOCAL_WINDOW + 1  # first key in the window of the first query
        gap = lambda first, last: np.maximum(0, last - np.maximum(first, LOCAL_PREFIX))  # noqa: E731
        shared -= int(min(gap(0, np.minimum(start, prefix))))
        mine -= int(gap(prefix, np.minimum(start, prefix + lengths)).sum())
    return int(count.sum()), shared, mine


def work(case):
    kind, dim = case["kind"], case["dim"]
    if kind == "rope":
        values = case["tokens"] * (case["heads"] + case["kv_heads"]) * dim
        return {"bytes": 4 * values + 4 * case["tokens"], "flops": 3 * values}
    key = 2 * case["kv_heads"] * (2 * dim if case["cache"] == "16bit" else dim + 4)  # K and V of one token
    row = 4 * case["kv_heads"] * dim
    if kind != "attend":
        return {"bytes": case["tokens"] * (key + row + 8), "flops": case["tokens"] * case["kv_heads"] * dim * 4}
    pairs, shared, mine = _seen_pairs(case)
    tokens = int(_lengths(case["queries"]).sum())
    return {"bytes": 4 * tokens * case["heads"] * dim + shared * key + mine * (key if case["own_in"] == "pages" else row),
            "flops": 4 * dim * case["heads"] * pairs}


# ---- the same calls in 64 bits --------------------------------------------------------------


def _exact_rope(case, seed):
    rows, positions = _rope_inputs(case, seed)
    half = case["rotary"] // 2
    angles = torch.zeros(case["tokens"], half, dtype=torch.float64, device="cuda")
    for i in range(half):
        f = math.exp(-2 * i / case["rotary"] * math.log(THETA))
        if case["scaling"] == "linear":
            f /= case["factor"]
        if case["scaling"] == "yarn":
            edge = [case["rotary"] / 2 * math.log(YARN_CONTEXT / (2 * math.pi * n)) / math.log(THETA)
                    for n in (YARN_FAST, YARN_SLOW)]
            low, high = max(math.floor(edge[0]), 0), min(math.ceil(edge[1]), case["rotary"] - 1)
            share = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            f = share * f / case["factor"] + (1 - share) * f
        angles[:, i] = positions.double() * f
    turn = torch.polar(torch.full_like(angles, _magnitude(case)), angles)[:, None]
    out, first = [], 0
    for heads in (case["heads"], case["kv_heads"]):
        x = rows[:, first:first + heads * case["dim"]].double().view(case["tokens"], heads, case["dim"]).clone()
        first += heads * case["dim"]
        at = [slice(0, half), slice(half, case["rotary"])] if case["layout"] == "half" else \
            [slice(0, case["rotary"], 2), slice(1, case["rotary"], 2)]
        z = torch.complex(x[..., at[0]], x[..., at[1]]) * turn
        x[..., at[0]], x[..., at[1]] = z.real, z.imag
        out.append(x.view(case["tokens"], -1))
    return out


def _exact_codes(x, form):
    """(the values that the codes stand for, or None; scales) in 64 bits."""
    most = x.abs().amax(-1)
    if form == "int8":
        return None, most / 127
    scale = torch.exp2(torch.ceil(torch.log2(most / 448)))
    y = x / scale[..., None]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step, scale


def _exact_write(case, seed):
    pool, slots, k, v = _cache_inputs(case, seed)
    shape, page = (case["tokens"], case["kv_heads"], case["dim"]), case["page"]
    out = []
    for x in (k, v):
        values, scale = (x.double().view(shape), None) if case["cache"] == "16bit" else \
            _exact_codes(x.double().view(shape), case["cache"])
        codes = None
        if values is not None:
            codes = torch.zeros(pool[0].shape, dtype=torch.float64, device="cuda")
            codes[slots // page, :, slots % page] = values
        scales = None
        if scale is not None:
            scales = torch.zeros(pool[0].shape[:3], dtype=torch.float64, device="cuda")
            scales[slots // page, :, slots % page] = scale
        out.append((codes, scales))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _cached(pool, which, pages, page, length):
    """Keys (which = 0) or values (1) 0 .. length - 1 of a page table, [length, kv, dim] in 64 bits."""
    slot = torch.arange(length, device="cuda")
    table = torch.from_numpy(np.asarray(pages, dtype=np.int64)).cuda()
    at = (table[slot // page], slice(None), slot % page)
    x = _taken(pool[which], *at).to(torch.float32).double()
    return x if pool[2] is None else x * pool[2 + which][at].double()[..., None]


def _exact_attend(case, seed):
    q, pool, tables, k, v = _attend_inputs(case, seed)
    dim, page, group = case["dim"], case["page"], case["heads"] // case["kv_heads"]
    out = torch.zeros(len(q), case["heads"], dim, dtype=torch.float64, device="cuda")
    shared = [_cached(pool, w, tables[0], page, case["prefix"]) for w in range(2)]
    at_q = at_k = 0
    for i, (m, n) in enumerate(zip(_lengths(case["queries"]).tolist(), _own_lengths(case).tolist())):
        if case["own_in"] == "pages":
            mine = [_cached(pool, w, tables[1 + i], page, n) for w in range(2)]
        else:
            mine = [x[at_k:at_k + n].double().view(n, case["kv_heads"], dim) for x in (k, v)]
        keys, values = (torch.cat(pair) for pair in zip(shared, mine))
        rows = q[at_q:at_q + m].double().view(m, case["heads"], dim)
        key = torch.arange(len(keys), device="cuda")[None, :]
        query = torch.arange(len(keys) - m, len(keys), device="cuda")[:, None]
        hidden = key > query
        if case["mask"] == "prefix_local":
            hidden |= (key >= LOCAL_PREFIX) & (query - key >= LOCAL_WINDOW)
        for h in range(case["heads"]):
            scores = rows[:, h] @ keys[:, h // group].T / math.sqrt(dim)
            out[at_q:at_q + m, h] = torch.softmax(scores.masked_fill(hidden, -math.inf), -1) @ values[:, h // group]
        at_q, at_k = at_q + m, at_k + n
    return out.view(len(q), -1)


def exact(case, seed):
    kind = case["kind"]
    if kind == "rope":
        return _exact_rope(case, seed)
    if kind == "write":
        return _exact_write(case, seed)
    if kind == "read":
        pool, slots, _, _ = _cache_inputs(case, seed)
        at = (slots // case["page"], slice(None), slots % case["page"])
        rows = [_taken(pool[w], *at).to(torch.float32).double() for w in range(2)]
        if pool[2] is not None:
            rows = [r * pool[2 + w][at].double()[..., None] for w, r in enumerate(rows)]
        return [r.reshape(case["tokens"], -1) for r in rows]
    return _exact_attend(case, seed)
