"""A paged cache under test beside a plain model of it.

``Rig`` owns a ``kivi.PagedCache``, the page tables and slots a scheduler would keep, and the tokens
of every sequence as numpy rows; ``held`` restates from those rows what the cache holds (the format's
float32 rule), ``attend`` the attention in float64 with a bound on the error the kernels' roundings
can add."""

import ctypes as C

import numpy as np

import kivi
from helpers import DeviceArrays

#: Half a step relative to the value: what one rounding to the type can be off.
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def to_bits(x, dtype):
    """float32 values rounded to nearest even into the type's bits."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    out = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), out)


def to_floats(bits, dtype):
    if dtype == "bf16":
        return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)
    return np.asarray(bits).astype(np.float32)


def rounded(x, dtype):
    return to_floats(to_bits(x, dtype), dtype)


def coded(x, bits):
    """(codes, scale, zero) of groups along the last axis, float32 as src/quant.rs:453-485 has it."""
    x = np.asarray(x, np.float32)
    levels = np.float32(2 ** bits - 1)
    zero, top = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    scale = (top - zero) / levels
    safe = np.where(scale == 0, np.float32(1), scale)
    codes = np.where(scale == 0, np.float32(0), np.clip(np.rint((x - zero) / safe), np.float32(0), levels))
    return codes, scale, zero


def _fma(a, b, c):
    return (a.astype(np.longdouble) * b + c).astype(np.float32)


def held(cfg, k, v, n):
    """Rows [n, heads, dim] as a cache of n tokens holds them, in float32: code * scale + zero rounded
    once (an fma, as src/quant.rs:379-451 has it; the sum is exact in 64 bits of mantissa)."""
    g, r = cfg.group_size, cfg.residual_length
    k, v = k[:n].copy(), v[:n].copy()
    kq, vq = n // r * r, max(0, n - r)
    if kq:
        x = k[:kq].reshape(kq // g, g, *k.shape[1:]).transpose(0, 2, 3, 1)
        codes, scale, zero = coded(x, cfg.bits)
        k[:kq] = _fma(codes, scale, zero).transpose(0, 3, 1, 2).reshape(k[:kq].shape)
    if vq:
        codes, scale, zero = coded(v[:vq].reshape(vq, v.shape[1], -1, g), cfg.bits)
        v[:vq] = _fma(codes, scale, zero).reshape(v[:vq].shape)
    return k, v


class Device(DeviceArrays):
    """Device buffers of any element type."""

    def put(self, host):
        host = np.ascontiguousarray(host)
        p = self.alloc(max(1, -(-host.nbytes // 4)))
        if host.nbytes:
            self._ok(self._hip.hipMemcpy(C.c_void_p(p), host.ctypes.data_as(C.c_void_p), C.c_size_t(host.nbytes), 1),
                     "hipMemcpy H2D")
        return p

    def write(self, p, host):
        host = np.ascontiguousarray(host)
        self._ok(self._hip.hipMemcpy(C.c_void_p(p), host.ctypes.data_as(C.c_void_p), C.c_size_t(host.nbytes), 1),
                 "hipMemcpy H2D")

    def get(self, p, shape, np_type):
        out = np.empty(shape, np_type)
        self.wait()
        self._ok(self._hip.hipMemcpy(out.ctypes.data_as(C.c_void_p), C.c_void_p(p), C.c_size_t(out.nbytes), 2),
                 "hipMemcpy D2H")
        return out

    def wait(self):
        self._ok(self._hip.hipDeviceSynchronize(), "hipDeviceSynchronize")


RAW = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


class Rig:
    """Sequences of one paged cache. Lengths grow by ``append``; ``chunks`` are the new tokens of
    each call (0 allowed)."""

    def __init__(self, amd, bits=2, group=32, residual=128, heads=2, dim=64, dtype="f32", page=64, pages=40, slots=6,
                 sequences=3, per_sequence=12, gq=2, seed=0):
        self.cfg = kivi.KiviConfig(bits, group, residual)
        self.heads, self.dim, self.dtype, self.page, self.gq = heads, dim, dtype, page, gq
        self.qh = heads * gq
        self.cache = kivi.PagedCache(amd, self.cfg, heads, dim, dtype, page, pages, slots)
        self.rng = np.random.default_rng(4200 + seed)
        self.mem = Device()
        self.table = np.full((sequences, per_sequence), -1, np.int32)
        order = self.rng.permutation(pages)[:sequences * per_sequence].astype(np.int32)
        self.table.reshape(-1)[:order.size] = order
        self.slots = self.rng.permutation(slots)[:sequences].astype(np.int32)
        self.lengths = np.zeros(sequences, np.int64)
        self.k = [np.zeros((0, heads, dim), np.float32) for _ in range(sequences)]
        self.v = [np.zeros((0, heads, dim), np.float32) for _ in range(sequences)]

    @property
    def sequences(self):
        return len(self.lengths)

    def tokens(self, n, spread=None):
        """n rows of keys and values, representable in the type; 1% (one at least) of the key channels x10."""
        k = self.rng.standard_normal((n, self.heads, self.dim)).astype(np.float32)
        k[..., :max(1, self.dim // 100)] *= 10
        v = self.rng.standard_normal((n, self.heads, self.dim)).astype(np.float32)
        if spread is not None:
            k, v = k * np.float32(spread), v * np.float32(spread)
        return rounded(k, self.dtype), rounded(v, self.dtype)

    def queries(self, rows):
        return rounded(self.rng.standard_normal((rows, self.qh, self.dim)).astype(np.float32), self.dtype)

    def batch(self, lengths, chunks, rows=None, max_rows=None, max_length=0, table=None, slots=None, starts=None):
        if starts is None:
            starts = np.concatenate([[0], np.cumsum(chunks)])
        starts = np.asarray(starts, np.int32)
        rows = int(starts[-1]) if rows is None else rows
        table = self.table if table is None else table
        put = self.mem.put
        return kivi.PagedBatch(len(lengths), put(np.asarray(self.slots if slots is None else slots, np.int32)),
                               put(np.asarray(lengths, np.int32)), put(starts), put(np.asarray(table, np.int32)),
                               table.shape[1], rows, max(chunks, default=0) if max_rows is None else max_rows, max_length)

    def upload(self, x, stride=None, offset=0):
        """Rows on the device: (address, elements, stride); `stride` and `offset` in elements."""
        rows = x.shape[0]
        flat = to_bits(x.reshape(rows, int(np.prod(x.shape[1:]))), self.dtype)
        width = flat.shape[1]
        stride = width if stride is None else stride
        buffer = np.full(offset + rows * stride, to_bits(np.float32(np.nan), self.dtype)[()], RAW[self.dtype])
        buffer[offset:].reshape(rows, stride)[:, :width] = flat
        return self.mem.put(buffer) + offset * SIZE[self.dtype], rows * stride, stride

    def append(self, chunks, tokens=None, padded=0, stride=None, offset=0, keep=True, lengths=None):
        """Appends `chunks` new tokens to each sequence, on the device and in the model."""
        lengths = self.lengths.copy() if lengths is None else np.asarray(lengths)
        new = [self.tokens(m) for m in chunks] if tokens is None else tokens
        pad = self.tokens(padded)
        k = np.concatenate([k for k, _ in new] + [pad[0]])
        v = np.concatenate([v for _, v in new] + [pad[1]])
        kp, kn, ks = self.upload(k, stride, offset)
        vp, vn, vs = self.upload(v, stride, offset)
        self.cache.append_device(self.batch(lengths, chunks, rows=len(k)), kp, kn, vp, vn, k_stride=ks, v_stride=vs)
        self.mem.wait()
        if keep:
            for i, (kk, vv) in enumerate(new):
                self.k[i] = np.concatenate([self.k[i][:lengths[i]], kk])
                self.v[i] = np.concatenate([self.v[i][:lengths[i]], vv])
            self.lengths = lengths + np.asarray(chunks)
        return new

    def read(self, first, counts, lengths=None, fill=0.0, rows=None, **more):
        """(keys, values) rows of tokens first[i] .. first[i] + counts[i]."""
        lengths = self.lengths if lengths is None else lengths
        total = int(sum(counts)) if rows is None else rows
        shape = (total, self.heads, self.dim)
        kp, n, _ = self.upload(np.full(shape, fill, np.float32))
        vp, n, _ = self.upload(np.full(shape, fill, np.float32))
        self.cache.read_device(self.batch(lengths, counts, rows=total, **more), kp, n, vp, n,
                               first_ptr=self.mem.put(np.asarray(first, np.int32)))
        return [to_floats(self.mem.get(p, shape, RAW[self.dtype]), self.dtype) for p in (kp, vp)]

    def attention(self, q, chunks, scale, new=None, window=0, sinks=0, lengths=None, rows=None, stride=None, offset=0,
                  stream=0, fill=7.0, **more):
        """The cache's attention; `new`: per sequence (k, v) rows given with the call."""
        lengths = self.lengths if lengths is None else lengths
        qp, qn, qs = self.upload(q, stride, offset)
        op, on, os_ = self.upload(np.full(q.shape, fill, np.float32), stride, offset)
        batch = self.batch(lengths, chunks, rows=len(q), **more)
        given = {}
        if new is not None:
            pad = np.full((len(q) - int(sum(chunks)), self.heads, self.dim), np.nan, np.float32)
            kp, kn, ks = self.upload(np.concatenate([k for k, _ in new] + [pad]), stride, offset)
            vp, vn, vs = self.upload(np.concatenate([v for _, v in new] + [pad]), stride, offset)
            given = {"k_ptr": kp, "k_len": kn, "v_ptr": vp, "v_len": vn, "k_stride": ks, "v_stride": vs}
        size = self.cache.attention_workspace_bytes(batch, self.qh)
        # what is in the workspace before a call is nothing a call may use
        work = self.mem.put(np.full(size // 4 + 1, np.nan, np.float32))
        self.cache.attention_device(batch, qp, qn, self.qh, scale, op, on, work, size, window=window, sinks=sinks,
                                    q_stride=qs, out_stride=os_, stream=stream, **given)
        start = op - offset * SIZE[self.dtype]
        raw = self.mem.get(start, (offset + len(q) * os_,), RAW[self.dtype])[offset:].reshape(len(q), os_)
        return to_floats(raw[:, :self.qh * self.dim].reshape(q.shape), self.dtype)

    def expected(self, q, chunks, scale, new=None, window=0, sinks=0, lengths=None, hidden=None):
        """(out, bound) in float64; `hidden[i]`: tokens of sequence i that no query sees."""
        lengths = self.lengths if lengths is None else lengths
        out, bound = np.zeros(q.shape), np.zeros(q.shape)
        at = 0
        for i, m in enumerate(chunks):
            k, v = held(self.cfg, self.k[i], self.v[i], int(lengths[i]))
            if new is not None:
                k, v = np.concatenate([k, new[i][0]]), np.concatenate([v, new[i][1]])
            gone = None if hidden is None else hidden[i]
            out[at:at + m], bound[at:at + m] = attend(q[at:at + m], k, v, scale, self.dtype, window, sinks, gone)
            at += m
        return out, bound

    def check(self, q, chunks, scale, new=None, window=0, sinks=0, lengths=None, hidden=None, **more):
        got = self.attention(q, chunks, scale, new, window, sinks, lengths, **more)
        want, bound = self.expected(q, chunks, scale, new, window, sinks, lengths, hidden)
        n = int(sum(chunks))
        err = np.abs(got[:n].astype(np.float64) - want[:n])
        assert np.isfinite(got[:n]).all()
        worst = np.unravel_index(np.argmax(err - bound[:n]), err.shape) if err.size else None
        assert (err <= bound[:n]).all(), f"at {worst}: off {err[worst]:.3g}, bound {bound[worst]:.3g}, want {want[worst]:.4g}"
        assert (got[n:] == 7.0).all(), "rows behind the last sequence were written"
        return got

    def close(self):
        self.mem.free()


def attend(q, k, v, scale, dtype, window=0, sinks=0, hidden=None):
    """Causal attention of q [m, qh, dim], the last m of L positions, over k, v [L, heads, dim] in
    float64, and a bound on what the kernels' arithmetic can add.

    The kernels round keys, values and weights to the type at most once each (half a step u), add
    products in float32 in any order (D terms of a logit, L of an output; half a step e = 2^-24 each,
    twice that for the running rescales), multiply a logit by the scale (2 roundings) and take exp2
    (2 ulp). A logit is then off by at most a = |scale| sum |q k| (u + (D + 4) e) + 4 e |logit|; the
    same of the row's maximum cancels, since it divides out; weights by a factor within exp(2 a), so
    by 2.5 a for a <= 0.2 (numerator and normalizer together, u and 4 e more for their own rounding); the output
    by that times sum p |v|, and its own rounding."""
    u, e = HALF[dtype], 2.0 ** -24
    m, qh, dim = q.shape
    total, heads = k.shape[0], k.shape[1]
    gq = qh // heads
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    t = np.arange(total)
    kd, vd, qd = k.astype(np.float64), v.astype(np.float64), q.astype(np.float64)
    for j in range(m):
        p = total - m + j
        seen = t <= p
        if window:
            seen &= (t > p - window) | (t < sinks)
        if hidden is not None:
            seen &= ~hidden
        if not seen.any():
            continue
        ks, vs = kd[seen], vd[seen]
        for h in range(qh):
            kh, vh = ks[:, h // gq], vs[:, h // gq]
            logits = kh @ qd[j, h] * scale
            size = np.abs(kh) @ np.abs(qd[j, h]) * abs(scale)
            a = float((size * (u + (dim + 4) * e) + 4 * e * np.abs(logits)).max())
            w = np.exp(logits - logits.max())
            w /= w.sum()
            out[j, h] = w @ vh
            rel = 2.5 * a + 2 * u + (2 * len(ks) + 16) * e if a <= 0.2 else np.expm1(2 * a) + 2 * u + (2 * len(ks) + 16) * e
            bound[j, h] = rel * (w @ np.abs(vh)) + 2 * u * np.abs(out[j, h]) + 1e-30
    return out, bound
