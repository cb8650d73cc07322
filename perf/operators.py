"""Workloads of the paged KIVI cache: ragged sequences whose quantized tokens lie in pages that a
scheduler hands out, as a continuously batched server keeps them.

Three operators, each in the types, head widths, groups and code widths it is used with:

  write   new tokens of a ragged batch go into the cache (``PagedCache.append_device``: what leaves
          the full-precision windows is quantized into the pages), and what the call touched is read
          back as rows (``PagedCache.read_device``)
  read    whole sequences are read back as rows
  attend  a chunk of new tokens of each sequence attends to its cache
          (``PagedCache.attention_device``): one token (decode), a few (drafted tokens to verify) or
          thousands (a piece of a prompt), with or without the chunk's own keys and values as rows,
          with or without a sliding window and a few first tokens that stay visible

A sequence of n tokens holds, per KV head, its first n // R * R keys quantized per channel over
groups of G tokens, its first max(0, n - R) values quantized per token over groups of G channels,
and its last rows in windows of 2 R rows (token t in row t % (2 R)); R is the residual length.

``own = False`` computes the same from plain tensors (one code per byte) with elementary torch
operations in float32; ``exact`` restates it from the tokens themselves in float64 (codes, scales
and zeros by the format's own float32 rule: they are defined bit for bit). Keys are N(0, 1) with 1%
of each KV head's channels ten times larger, values N(0, 1)."""
import importlib.util
import math
import os

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_package = []


def _kivi():
    """kivi-cache-rs_amd/kivi.py (the folder's name is no module name)."""
    if not _package:
        spec = importlib.util.spec_from_file_location("kivi", os.path.join(_ROOT, "kivi-cache-rs_amd", "kivi.py"))
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        _package.append(module)
    return _package[0]


# ---------------------------------------------------------------- the cases


def _case(op, name, dtype, bits, group, residual, page, kv, q, dim, sequences, shortest, longest, rows, **more):
    """`sequences` sequences of `shortest` to `longest` cached tokens; the first `long_chunks` of
    them bring `rows` new tokens, the others `rows_least`. `padded` rows follow the last sequence."""
    c = {"op": op, "dtype": dtype, "bits": bits, "group": group, "residual": residual, "page": page,
         "kv_heads": kv, "q_heads": q, "head_dim": dim, "sequences": sequences, "shortest": shortest,
         "longest": longest, "rows": rows, "rows_least": more.pop("rows_least", rows),
         "long_chunks": more.pop("long_chunks", sequences), "fresh": more.pop("fresh", True),
         "window": more.pop("window", 0), "sinks": more.pop("sinks", 0), "padded": more.pop("padded", 0)}
    if name is not None:
        c["name"] = name
    assert not more, more
    return c


def listed():
    return [
        # one user's chat: the next token goes in (latency alone)
        _case("write", "write one token", "bf16", 2, 32, 128, 64, 8, 8, 128, 1, 1000, 1000, 1),
        # a full decode batch, ragged lengths, drafted tokens among the new ones
        _case("write", "write 64 sequences' next tokens", "f16", 4, 32, 128, 128, 8, 8, 128, 64, 5, 32768, 7,
              rows_least=1, long_chunks=9, padded=3),
        # prompts of a batch encoded whole, and handed on as rows
        _case("write", "write prompts", "f32", 2, 32, 128, 64, 8, 8, 128, 9, 0, 0, 8191, rows_least=1500, long_chunks=4),
        # long sequences handed to another worker as rows, heads of 96 channels, byte codes
        _case("read", "read long sequences", "bf16", 8, 32, 96, 96, 16, 16, 96, 5, 2000, 45001, 0),
        # one user's chat: one token of a layer with grouped heads
        _case("attend", "decode one sequence", "bf16", 2, 32, 128, 64, 8, 32, 128, 1, 1000, 1000, 1),
        # a full decode batch of ragged lengths
        _case("attend", "decode 64 sequences", "bf16", 2, 32, 128, 64, 8, 32, 128, 64, 500, 32768, 1),
        # one very long document, eight query heads per KV head, the token written first
        _case("attend", "decode one 131072-token sequence", "f16", 4, 32, 128, 256, 8, 64, 128, 1, 131071, 131071, 1,
              fresh=False),
        # drafted tokens of a small batch verified, already written, float32
        _case("attend", "verify 5 tokens of 16 sequences", "f32", 2, 32, 128, 64, 8, 32, 128, 16, 100, 9001, 5,
              fresh=False),
        # a piece of a long prompt over what is cached of it
        _case("attend", "chunk of 2048 tokens", "bf16", 2, 32, 128, 64, 8, 32, 128, 1, 16384, 16384, 2048),
        # a serving step: one ragged piece of a prompt among decoding sequences, seven query heads per KV head
        _case("attend", "mixed step", "f16", 4, 64, 128, 128, 4, 28, 128, 24, 300, 12000, 517, rows_least=1,
              long_chunks=2, padded=5),
        # decoding far past a sliding window with four first tokens kept
        _case("attend", "windowed decode", "bf16", 4, 32, 128, 64, 8, 32, 128, 32, 3000, 65536, 1, window=4096, sinks=4),
        # a piece of a prompt under a sliding window, small heads
        _case("attend", "windowed chunk", "f16", 2, 32, 64, 64, 8, 32, 64, 2, 5000, 20000, 1500, window=1024, sinks=4),
    ]


def _odd_log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "write", "read", "attend", "attend", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    bits = rng.choice([2, 2, 4, 8])
    dim = rng.choice([128] * 5 + [64, 64, 80, 96, 256])
    group = rng.choice([g for g in (32, 32, 32, 64, 16, 128) if dim % g == 0 and g * bits % 32 == 0] or [16])
    residual = max(32, group) * rng.choice([1, 2, 4]) if group < 128 else group
    page = max(32, group) * rng.choice([1, 2, 2, 4])
    kv = rng.choice([1, 2, 4, 8, 8, 8, 16])
    gq = rng.choice([1, 2, 4, 4, 7, 8, 16] if kv <= 8 else [1, 2])
    sequences = _odd_log(rng, 1, 64)
    longest = _odd_log(rng, 1, 131072)
    shortest = min(longest, _odd_log(rng, 1, 131072))
    more = {"padded": rng.choice([0, 0, 1, 6])}
    rows = 1
    if op == "write":
        gq = 1
        if rng.random() < 0.5:  # whole prompts
            longest = shortest = 0
            rows = _odd_log(rng, 2, 8191)
            more.update(rows_least=rng.randint(1, rows), long_chunks=rng.randint(1, sequences))
        else:  # the next tokens: no more than a window takes back
            rows = rng.choice([1, 1, 2, 5, 8, residual])
            more.update(rows_least=1, long_chunks=rng.randint(1, sequences))
    elif op == "read":
        gq, rows, more["padded"] = 1, 0, 0
    else:
        form = rng.choice(["decode", "decode", "verify", "chunk", "mixed"])
        if form == "verify":
            rows = rng.randint(2, 16)
        elif form != "decode":
            rows = _odd_log(rng, 20, 2048)
            sequences = min(sequences, _odd_log(rng, 1, 24))
        if form == "mixed":
            more.update(rows_least=1, long_chunks=1)
        # rows that are written first lie in the cache: the shortest sequence has to hold them all
        more["fresh"] = rng.random() < 0.6 or shortest < rows
        if rng.random() < 0.35:
            more.update(window=_odd_log(rng, 16, 8192), sinks=rng.choice([0, 1, 4, 37]))
    case = _case(op, None, dtype, bits, group, residual, page, kv, kv * gq, dim, sequences, shortest, longest, rows, **more)
    # no more than the largest listed cases move and compute
    most = [work(c) for c in listed()]
    bound = {what: max(m[what] for m in most) for what in ("bytes", "flops")}
    if dtype == "f32":
        bound["flops"] /= 8
    while any(work(case)[what] > bound[what] for what in bound) or _held_elements(case) > 2 ** 30:
        if case["sequences"] > 1 and rng.random() < 0.7:
            case["sequences"] = (case["sequences"] + 1) // 2
            case["long_chunks"] = min(case["long_chunks"], case["sequences"])
        elif case["longest"] > 1:
            case["longest"] = max(case["rows"] if not case["fresh"] else 1, case["longest"] * 2 // 3)
            case["shortest"] = min(case["shortest"], case["longest"])
        else:
            case["rows"] = max(1, case["rows"] * 2 // 3)
            case["rows_least"] = min(case["rows_least"], case["rows"])
    return case


# ---------------------------------------------------------------- a case's layout


def _lengths(c):
    """Cached tokens of each sequence: spread evenly over the logarithm, in mixed order."""
    n, lo, hi = c["sequences"], c["shortest"], c["longest"]
    if n == 1 or hi == lo:
        return [hi] * n
    spread = [int(round(math.exp(math.log(max(lo, 1)) + (math.log(hi) - math.log(max(lo, 1))) * i / (n - 1))))
              for i in range(n)]
    step = next(s for s in (7, 5, 3, 11, 13, 1) if math.gcd(s, n) == 1)
    return [spread[i * step % n] for i in range(n)]


def _chunks(c):
    """New tokens of each sequence; reading takes whole sequences."""
    if c["op"] == "read":
        return _lengths(c)
    return [c["rows"] if i < c["long_chunks"] else c["rows_least"] for i in range(c["sequences"])]


def _held_elements(c):
    return (sum(_lengths(c)) + sum(_chunks(c))) * c["kv_heads"] * c["head_dim"]


def _packed(c, n):
    """(quantized key tokens, quantized value tokens) of a sequence of n tokens."""
    r = c["residual"]
    return n // r * r, max(0, n - r)


def _touched(c, n):
    """First token that a write behind n cached tokens can change: the oldest value still in the window."""
    return _packed(c, n)[1]


def _visible(c, n, m):
    """(sink tokens, first token of the rest) that some row of m at the end of n tokens sees."""
    if not c["window"]:
        return 0, 0
    lo = max(0, n - m + 1 - c["window"])
    return min(c["sinks"], lo), lo


def _starts(c):
    at = [0]
    for m in _chunks(c):
        at.append(at[-1] + m)
    return at


def _pages_of(c, n):
    return -(-n // c["page"])


def _scale(c):
    return 1.0 / math.sqrt(c["head_dim"])


# ---------------------------------------------------------------- inputs


def _rng(seed, salt):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + salt)


def _tokens(c, seed):
    """Per sequence (keys, values) of all its tokens, cached ones and the new rows behind them:
    [tokens, kv_heads, head_dim] in the case's type."""
    dtype, kv, dim = _TYPES[c["dtype"]], c["kv_heads"], c["head_dim"]
    new = [0] * c["sequences"] if c["op"] == "read" or not c["fresh"] else _chunks(c)
    lengths = [n + m for n, m in zip(_lengths(c), new)]
    many = max(1, round(dim / 100))
    hot = torch.rand(kv, dim, generator=_rng(seed, 1), device="cuda").topk(many, 1).indices
    factor = torch.ones(kv, dim, device="cuda").scatter_(1, hot, 10.0).to(dtype)
    keys = torch.randn(sum(lengths), kv, dim, generator=_rng(seed, 2), device="cuda", dtype=dtype).mul_(factor)
    values = torch.randn(sum(lengths), kv, dim, generator=_rng(seed, 3), device="cuda", dtype=dtype)
    return list(zip(keys.split(lengths), values.split(lengths)))


def _queries(c, seed):
    rows = _starts(c)[-1] + c["padded"]
    return torch.randn(rows, c["q_heads"], c["head_dim"], generator=_rng(seed, 4), device="cuda",
                       dtype=_TYPES[c["dtype"]])


def _ragged(c, rows):
    """Rows of the sequences one after the other, and the padding behind the last."""
    pad = torch.zeros(c["padded"], *rows[0].shape[1:], dtype=rows[0].dtype, device="cuda")
    return torch.cat(list(rows) + [pad])


class _State:
    """What the program has in hand: tensors and handles by name."""

    def __init__(self, case, **held):
        self.case = case
        self.__dict__.update(held)


def _table(c, seed):
    """(page table, pages of the pool, window slot of each sequence): pages in any order, entries of
    no page -1. Under a sliding window the pages that nothing reads any more are handed back."""
    chunks, lengths = _chunks(c), _lengths(c)
    new = chunks if c["op"] == "write" else [0] * len(lengths)
    need = [_pages_of(c, n + m) for n, m in zip(lengths, new)]
    g = torch.Generator().manual_seed(int(seed) * 1000003 + 5)
    order = torch.randperm(sum(need) + 3, generator=g, dtype=torch.int32)
    table = torch.full((c["sequences"], max(need) + 2), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    slots = torch.randperm(c["sequences"] + 1, generator=g, dtype=torch.int32)[:c["sequences"]]
    return table.cuda(), order.numel(), slots.cuda()


def _forget(c, table):
    if c["op"] == "attend" and c["window"]:
        for i, (n, m) in enumerate(zip(_lengths(c), _chunks(c))):
            sinks, lo = _visible(c, n + m if c["fresh"] else n, m)
            table[i, _pages_of(c, sinks):lo // c["page"]] = -1


def prepare(case, seed):
    c = case
    dtype, kv, dim = _TYPES[c["dtype"]], c["kv_heads"], c["head_dim"]
    lengths, chunks, starts = _lengths(c), _chunks(c), _starts(c)
    tokens = _tokens(c, seed)
    table, pages, slots = _table(c, seed)
    cache = (_OwnCache if own else _PlainCache)(c, pages, c["sequences"] + 1)
    s = _State(c, cache=cache, table=table, slots=slots, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
               starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    if sum(lengths):  # what is cached by now
        held = [(k[:n], v[:n]) for (k, v), n in zip(tokens, lengths)]
        cache.fill(s, torch.cat([k for k, _ in held]), torch.cat([v for _, v in held]), lengths)
    _forget(c, table)
    rows = starts[-1] + c["padded"]
    if c["op"] == "read":
        s.k_out = torch.zeros(rows, kv, dim, dtype=dtype, device="cuda")
        s.v_out = torch.zeros_like(s.k_out)
    elif c["op"] == "write":
        s.k = _ragged(c, [k[n:] for (k, _), n in zip(tokens, lengths)])
        s.v = _ragged(c, [v[n:] for (_, v), n in zip(tokens, lengths)])
        # read back: from the oldest token that the call can change to the newest
        first = [_touched(c, n) for n in lengths]
        after = [n + m for n, m in zip(lengths, chunks)]
        at = [0]
        for n, f in zip(after, first):
            at.append(at[-1] + n - f)
        s.first = torch.tensor(first, dtype=torch.int32, device="cuda")
        s.after = torch.tensor(after, dtype=torch.int32, device="cuda")
        s.back = torch.tensor(at, dtype=torch.int32, device="cuda")
        s.k_out = torch.zeros(at[-1], kv, dim, dtype=dtype, device="cuda")
        s.v_out = torch.zeros_like(s.k_out)
    else:
        s.q = _queries(c, seed)
        s.out = torch.zeros_like(s.q)
        if c["fresh"]:
            s.k = _ragged(c, [k[n:] for (k, _), n in zip(tokens, lengths)])
            s.v = _ragged(c, [v[n:] for (_, v), n in zip(tokens, lengths)])
    cache.ready(s)
    return s


def run(state):
    c, cache = state.case, state.cache
    if c["op"] == "write":
        cache.write(state)
        cache.read_back(state)
        return [state.k_out, state.v_out]
    if c["op"] == "read":
        cache.read(state)
        return [state.k_out, state.v_out]
    cache.attend(state)
    return state.out


# ---------------------------------------------------------------- the framework's calls


def _stream():
    return torch.cuda.current_stream().cuda_stream


class _OwnCache:
    def __init__(self, c, pages, slots):
        kivi = _kivi()
        self.amd = kivi.Backend.amd()
        config = kivi.KiviConfig(c["bits"], c["group"], c["residual"])
        self.cache = kivi.PagedCache(self.amd, config, c["kv_heads"], c["head_dim"], c["dtype"], c["page"], pages, slots)

    def _batch(self, s, lengths, starts, rows, max_rows, max_length):
        return _kivi().PagedBatch(s.case["sequences"], s.slots.data_ptr(), lengths.data_ptr(), starts.data_ptr(),
                                  s.table.data_ptr(), s.table.shape[1], rows, max_rows, max_length)

    def fill(self, s, k, v, lengths):
        at = torch.zeros(len(lengths) + 1, dtype=torch.int32)
        at[1:] = torch.tensor(lengths).cumsum(0)
        at = at.cuda()
        nothing = torch.zeros_like(s.lengths)
        batch = self._batch(s, nothing, at, k.shape[0], max(lengths), max(lengths))
        self.cache.append_device(batch, k.data_ptr(), k.numel(), v.data_ptr(), v.numel(), stream=_stream())
        torch.cuda.current_stream().synchronize()  # k and v are let go

    def ready(self, s):
        """The batch descriptors and the workspace that a serving loop keeps."""
        c = s.case
        longest, rows = c["longest"], c["longest"] if c["op"] == "read" else c["rows"]
        tensor = {"read": "k_out", "write": "k", "attend": "q"}[c["op"]]
        s.batch = self._batch(s, s.lengths, s.starts, getattr(s, tensor).shape[0], rows, longest + rows)
        if c["op"] == "write":
            s.batch_back = self._batch(s, s.after, s.back, s.k_out.shape[0], rows + c["residual"], longest + rows)
        if c["op"] == "attend":
            size = self.cache.attention_workspace_bytes(s.batch, c["q_heads"])
            s.workspace = torch.empty(size, dtype=torch.uint8, device="cuda")

    def write(self, s):
        self.cache.append_device(s.batch, s.k.data_ptr(), s.k.numel(), s.v.data_ptr(), s.v.numel(), stream=_stream())

    def read_back(self, s):
        self.cache.read_device(s.batch_back, s.k_out.data_ptr(), s.k_out.numel(), s.v_out.data_ptr(), s.v_out.numel(),
                               first_ptr=s.first.data_ptr(), stream=_stream())

    def read(self, s):
        self.cache.read_device(s.batch, s.k_out.data_ptr(), s.k_out.numel(), s.v_out.data_ptr(), s.v_out.numel(),
                               stream=_stream())

    def attend(self, s):
        c = s.case
        rows = {}
        if c["fresh"]:
            rows = {"k_ptr": s.k.data_ptr(), "k_len": s.k.numel(), "v_ptr": s.v.data_ptr(), "v_len": s.v.numel()}
        self.cache.attention_device(s.batch, s.q.data_ptr(), s.q.numel(), c["q_heads"], _scale(c), s.out.data_ptr(),
                                    s.out.numel(), s.workspace.data_ptr(), s.workspace.numel(), window=c["window"],
                                    sinks=c["sinks"], stream=_stream(), **rows)


# ---------------------------------------------------------------- the same in plain torch


def _code(x, levels):
    """(codes, scale, zero) of groups along the last axis by the format's float32 rule:
    scale = span / levels, code = round-half-even((x - zero) / scale)."""
    zero, top = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = (top - zero) / torch.full_like(top, levels)  # by a tensor: torch takes a number's reciprocal
    safe = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = torch.where(scale == 0, torch.zeros_like(x), ((x - zero) / safe).round_().clamp_(0, levels))
    return codes.to(torch.uint8), scale.squeeze(-1), zero.squeeze(-1)


class _PlainCache:
    """Pools of codes (one per byte) and (scale, zero) pairs by page, windows by slot."""

    def __init__(self, c, pages, slots):
        kv, dim, p, g, r = c["kv_heads"], c["head_dim"], c["page"], c["group"], c["residual"]
        dtype = _TYPES[c["dtype"]]
        self.k_codes = torch.zeros(pages, p, kv, dim, dtype=torch.uint8, device="cuda")
        self.v_codes = torch.zeros_like(self.k_codes)
        self.k_pairs = torch.zeros(pages, p // g, kv, dim, 2, device="cuda")
        self.v_pairs = torch.zeros(pages, p, kv, dim // g, 2, device="cuda")
        self.k_window = torch.zeros(slots, 2 * r, kv, dim, dtype=dtype, device="cuda")
        self.v_window = torch.zeros_like(self.k_window)

    def _append(self, c, table, slot, n, k, v):
        m, r, g, p = k.shape[0], c["residual"], c["group"], c["page"]
        levels = 2 ** c["bits"] - 1
        kq, vq = _packed(c, n)
        kq2, vq2 = _packed(c, n + m)
        ring = torch.arange(max(0, n - r), n, device="cuda")
        old = max(0, n - r)
        if kq2 > kq:
            rows = torch.cat([self.k_window[slot, ring[kq - old:] % (2 * r)], k[:kq2 - n]]).float()
            groups = rows.view(-1, g, *rows.shape[1:]).permute(0, 2, 3, 1)  # [group, kv, dim, token]
            codes, scale, zero = _code(groups, levels)
            t = torch.arange(kq, kq2, device="cuda")
            self.k_codes[table[t // p], t % p] = codes.permute(0, 3, 1, 2).reshape(rows.shape)
            t = t[::g]
            self.k_pairs[table[t // p], t % p // g] = torch.stack([scale, zero], -1)
        if vq2 > vq:
            rows = torch.cat([self.v_window[slot, ring % (2 * r)], v])[:vq2 - vq].float()
            codes, scale, zero = _code(rows.view(*rows.shape[:2], -1, g), levels)
            t = torch.arange(vq, vq2, device="cuda")
            self.v_codes[table[t // p], t % p] = codes.view(rows.shape)
            self.v_pairs[table[t // p], t % p] = torch.stack([scale, zero], -1)
        t = torch.arange(max(n, n + m - r), n + m, device="cuda")
        self.k_window[slot, t % (2 * r)] = k[t - n]
        self.v_window[slot, t % (2 * r)] = v[t - n]

    def _rows(self, c, table, slot, n, t, k=None, v=None):
        """Keys and values of tokens t (ascending) of a sequence of n cached tokens as float32 rows;
        tokens from n on are rows of k and v."""
        p, g, r = c["page"], c["group"], c["residual"]
        kq, vq = _packed(c, n)
        cached = t[t < n]
        a, b = cached[cached < kq], cached[cached >= kq]
        pair = self.k_pairs[table[a // p], a % p // g]
        keys = [self.k_codes[table[a // p], a % p].float() * pair[..., 0] + pair[..., 1],
                self.k_window[slot, b % (2 * r)].float()]
        a, b = cached[cached < vq], cached[cached >= vq]
        pair = self.v_pairs[table[a // p], a % p]
        codes = self.v_codes[table[a // p], a % p].float().view(*pair.shape[:3], g)
        values = [(codes * pair[..., :1] + pair[..., 1:]).flatten(2), self.v_window[slot, b % (2 * r)].float()]
        if k is not None:
            new = t[t >= n] - n
            keys.append(k[new].float())
            values.append(v[new].float())
        return torch.cat(keys), torch.cat(values)

    def _each(self, s):
        """(page table, slot, cached tokens, new tokens, first row) of each sequence; its program
        knows the lengths on the host too."""
        c = s.case
        table, slots = s.table.long(), s.slots.tolist()
        return [(table[i], slots[i], n, m, at)
                for i, (n, m, at) in enumerate(zip(_lengths(c), _chunks(c), _starts(c)))]

    def fill(self, s, k, v, lengths):
        table, slots = s.table.long(), s.slots.tolist()
        for i, (ki, vi) in enumerate(zip(k.split(lengths), v.split(lengths))):
            self._append(s.case, table[i], slots[i], 0, ki, vi)

    def ready(self, s):
        s.each = self._each(s)

    def write(self, s):
        for table, slot, n, m, at in s.each:
            self._append(s.case, table, slot, n, s.k[at:at + m], s.v[at:at + m])

    def read_back(self, s):
        at = 0
        for table, slot, n, m, _ in s.each:
            t = torch.arange(_touched(s.case, n), n + m, device="cuda")
            keys, values = self._rows(s.case, table, slot, n + m, t)
            s.k_out[at:at + len(t)] = keys.to(s.k_out.dtype)
            s.v_out[at:at + len(t)] = values.to(s.v_out.dtype)
            at += len(t)

    def read(self, s):
        for table, slot, n, _, at in s.each:
            keys, values = self._rows(s.case, table, slot, n, torch.arange(n, device="cuda"))
            s.k_out[at:at + n] = keys.to(s.k_out.dtype)
            s.v_out[at:at + n] = values.to(s.v_out.dtype)

    def attend(self, s):
        c = s.case
        kv, dim, gq = c["kv_heads"], c["head_dim"], c["q_heads"] // c["kv_heads"]
        for table, slot, n, m, at in s.each:
            k, v = (s.k[at:at + m], s.v[at:at + m]) if c["fresh"] else (None, None)
            total = n + m if c["fresh"] else n
            sinks, lo = _visible(c, total, m)
            t = torch.cat([torch.arange(sinks, device="cuda"), torch.arange(lo, total, device="cuda")])
            keys, values = self._rows(c, table, slot, n, t, k, v)
            position = torch.arange(total - m, total, device="cuda")[:, None]
            seen = t <= position
            if c["window"]:
                seen &= (t > position - c["window"]) | (t < c["sinks"])
            q = s.q[at:at + m].float().view(m, kv, gq, dim).permute(1, 2, 0, 3)  # [kv, gq, m, dim]
            logits = q.reshape(kv, gq * m, dim) @ keys.permute(1, 2, 0) * _scale(c)
            logits = logits.view(kv, gq, m, -1).masked_fill(~seen, -math.inf)
            weights = torch.exp(logits - logits.amax(-1, keepdim=True))
            weights = weights / weights.sum(-1, keepdim=True)
            out = weights.view(kv, gq * m, -1) @ values.permute(1, 0, 2)
            s.out[at:at + m] = out.view(kv, gq, m, dim).permute(2, 0, 1, 3).reshape(m, kv * gq, dim).to(s.out.dtype)


# ---------------------------------------------------------------- what a pass cannot do without


def _size(c):
    return {"f32": 4, "f16": 2, "bf16": 2}[c["dtype"]]


def _held_bytes(c, lo, hi, n):
    """Bytes that tokens [lo, hi) of a sequence of n cached tokens hold: codes, pairs, window rows."""
    kq, vq = _packed(c, n)
    d, g, b = c["head_dim"], c["group"], c["bits"]
    kp, vp = max(0, min(hi, kq) - lo), max(0, min(hi, vq) - lo)
    packed = kp * (d * b / 8 + d / g * 8) + vp * (d * b / 8 + d / g * 8)
    return c["kv_heads"] * (packed + (2 * (hi - lo) - kp - vp) * d * _size(c))


def work(case):
    c = case
    row = c["kv_heads"] * c["head_dim"] * _size(c)  # one token's keys, or values
    spent = flops = 0.0
    for n, m in zip(_lengths(c), _chunks(c)):
        if c["op"] == "read":
            spent += _held_bytes(c, 0, n, n) + 2 * n * row
            flops += 4.0 * n * c["kv_heads"] * c["head_dim"]
        elif c["op"] == "write":
            (kq, vq), (kq2, vq2) = _packed(c, n), _packed(c, n + m)
            first = _touched(c, n)
            spent += 2 * m * row  # the new rows
            spent += (max(0, min(n, kq2) - kq) + max(0, min(n, vq2) - vq)) * row  # rows that leave the windows
            written = _held_bytes(c, first, n + m, n + m) - (max(0, n - max(kq2, first)) + max(0, n - max(vq2, first))) * row
            if kq2 == kq:
                written -= (kq - first) * c["kv_heads"] * (c["head_dim"] * c["bits"] / 8 + c["head_dim"] / c["group"] * 8)
            spent += max(0.0, written)
            spent += _held_bytes(c, first, n + m, n + m) + 2 * (n + m - first) * row  # read back
            flops += 12.0 * (n + m - first) * c["kv_heads"] * c["head_dim"]
        else:
            total = n + m if c["fresh"] else n
            sinks, lo = _visible(c, total, m)
            spent += _held_bytes(c, 0, sinks, n) + _held_bytes(c, min(lo, n), n, n)
            spent += 2 * m * row if c["fresh"] else 0
            spent += 2 * m * c["q_heads"] * c["head_dim"] * _size(c)
            # pairs of a row and a token that it sees
            pairs = 0
            if c["window"]:
                for p in range(total - m, total):
                    inside = min(p + 1, c["window"])
                    pairs += inside + min(c["sinks"], max(0, p + 1 - inside))
            else:
                pairs = m * total - m * (m - 1) // 2
            flops += 4.0 * pairs * c["q_heads"] * c["head_dim"]
    return {"bytes": spent, "flops": flops}


# ---------------------------------------------------------------- from the definition, in float64


def _quantized(x, levels):
    """What the codes of groups along the last axis stand for, in float64."""
    low, high = torch.min(x, -1, keepdim=True)[0], torch.max(x, -1, keepdim=True)[0]
    step = torch.div(high - low, torch.full_like(low, levels))
    place = torch.div(x - low, step)
    place = torch.where(step == 0, torch.zeros_like(place), torch.round(place)).clamp(0, levels)
    return low.double() + place.double() * step.double()


def _definition(c, k, v, n):
    """Rows [n, kv, dim] of one sequence as its cache holds them, in float64."""
    levels, g = 2 ** c["bits"] - 1, c["group"]
    kd, vd = k.double(), v.double()
    kq, vq = _packed(c, n)
    if kq:
        by_group = k[:kq].float().view(kq // g, g, *k.shape[1:]).movedim(1, -1).contiguous()
        kd[:kq] = _quantized(by_group, levels).movedim(-1, 1).reshape(kq, *k.shape[1:])
    if vq:
        by_group = v[:vq].float().view(vq, v.shape[1], -1, g)
        vd[:vq] = _quantized(by_group, levels).view(vq, *v.shape[1:])
    return kd, vd


def exact(case, seed):
    c = case
    tokens, lengths, chunks, starts = _tokens(c, seed), _lengths(c), _chunks(c), _starts(c)
    if c["op"] == "read":
        both = [_definition(c, k, v, n) for (k, v), n in zip(tokens, lengths)]
        return [torch.cat([k for k, _ in both]), torch.cat([v for _, v in both])]
    if c["op"] == "write":
        both = []
        for (k, v), n in zip(tokens, lengths):
            kd, vd = _definition(c, k, v, k.shape[0])
            both.append((kd[_touched(c, n):], vd[_touched(c, n):]))
        return [torch.cat([k for k, _ in both]), torch.cat([v for _, v in both])]
    q = _queries(c, seed).double()
    out = torch.zeros_like(q)
    gq = c["q_heads"] // c["kv_heads"]
    for i, ((k, v), n, m) in enumerate(zip(tokens, lengths, chunks)):
        total = n + m if c["fresh"] else n
        kd, vd = _definition(c, k[:n], v[:n], n)
        kd, vd = torch.cat([kd, k[n:].double()]), torch.cat([vd, v[n:].double()])
        sinks, lo = _visible(c, total, m)
        if lo > sinks:
            kd, vd = torch.cat([kd[:sinks], kd[lo:]]), torch.cat([vd[:sinks], vd[lo:]])
        place = torch.arange(total, device="cuda")
        place = torch.cat([place[:sinks], place[lo:]]) if lo > sinks else place
        row = torch.arange(m, device="cuda")[:, None] + (total - m)
        hidden = place[None, :] > row
        if c["window"]:
            hidden |= (place[None, :] <= row - c["window"]) & (place[None, :] >= c["sinks"])
        for h in range(c["q_heads"]):
            logits = (q[starts[i]:starts[i] + m, h] @ kd[:, h // gq].T) * _scale(c)
            logits[hidden] = -math.inf
            out[starts[i]:starts[i] + m, h] = torch.softmax(logits, dim=-1) @ vd[:, h // gq]
    return out
