"""The paged cache (``kivi_paged_*``): refusals on the CPU, and under ``-m gpu`` writes, reads and
attention of ragged batches against a plain model, the oracle's KiviCache and float64 attention
(tolerances derived in paged_helpers.attend)."""

import ctypes as C

import numpy as np
import pytest

import kivi
from conftest import amd_backend
from kivi import KiviCache, KiviConfig, KiviError, PagedBatch, PagedCache
from paged_helpers import RAW, Rig, held, rounded, to_bits, to_floats

# ---------------------------------------------------------------- refusals (no device needed)


def _refused(fn):
    with pytest.raises(KiviError) as e:
        fn()
    return e.value


@pytest.mark.parametrize("args,variant,payload", [
    ((KiviConfig(3, 32, 128), 8, 128, "bf16", 64, 4, 4), "InvalidBits", {"bits": 3}),
    ((KiviConfig(2, 12, 128), 8, 128, "bf16", 64, 4, 4), "MisalignedGroup", {"group_size": 12, "bits": 2}),
    ((KiviConfig(2, 32, 48), 8, 128, "bf16", 64, 4, 4), "ResidualLength", {"residual_length": 48, "group_size": 32}),
    ((KiviConfig(2, 32, 128), 0, 128, "bf16", 64, 4, 4), "ZeroDimension", {"name": "num_kv_heads"}),
    ((KiviConfig(2, 32, 128), 8, 100, "bf16", 64, 4, 4), "HeadDim", {"head_dim": 100, "group_size": 32}),
    ((KiviConfig(2, 32, 128), 8, 0, "bf16", 64, 4, 4), "HeadDim", {"head_dim": 0, "group_size": 32}),
    ((KiviConfig(2, 32, 128), 8, 128, "f64", 64, 4, 4), "Unsupported", {}),
    ((KiviConfig(2, 32, 128), 8, 512, "bf16", 64, 4, 4), "Unsupported", {}),
    ((KiviConfig(8, 100, 100), 1, 200, "bf16", 800, 4, 4), "Unsupported", {}),
    ((KiviConfig(2, 32, 128), 8, 128, "bf16", 0, 4, 4), "TokenGroup", {"tokens": 0, "group_size": 32}),
    ((KiviConfig(2, 48, 48), 8, 96, "bf16", 64, 4, 4), "TokenGroup", {"tokens": 64, "group_size": 96}),
    ((KiviConfig(2, 32, 128), 8, 128, "bf16", 64, 0, 4), "ZeroDimension", {"name": "num_pages"}),
    ((KiviConfig(2, 32, 128), 8, 128, "bf16", 64, 4, 0), "ZeroDimension", {"name": "num_slots"}),
    ((KiviConfig(2, 32, 128), 8, 128, "bf16", 64, 2 ** 31, 4), "Unsupported", {}),
    ((KiviConfig(2, 32, 128), 8, 128, "bf16", 64, 4, 2 ** 31), "Unsupported", {}),
    ((KiviConfig(2, 32, 128), 2 ** 16, 128, "bf16", 64, 4, 4), "Unsupported", {}),
])
def test_new_refuses(args, variant, payload):
    e = _refused(lambda: PagedCache(amd_backend(), *args))
    assert (e.variant, e.payload) == (variant, payload)


def test_null_cache_and_out_are_refused():
    b = amd_backend()
    batch = PagedBatch(0, 0, 0, 0, 0, 0, 0)
    err = kivi._Error()
    assert b["paged_append_device"](None, C.byref(batch._c), None, 0, 0, None, 0, 0, None, C.byref(err)) == 100
    assert err.name == b"cache"
    assert b["paged_new"](C.byref(KiviConfig()._c()), 1, 128, 0, 64, 1, 1, None, C.byref(err)) == 100
    assert err.name == b"out"
    b["paged_free"](None)
    assert b["paged_device_bytes"](None) == 0


def test_a_cache_without_a_device_fails_loudly():
    b = amd_backend()
    if b["device_count"]() > 0:
        pytest.skip("a HIP device is present")
    assert _refused(lambda: PagedCache(b, KiviConfig(), 8, 128, "bf16", 64, 4, 4)).variant == "Device"


@pytest.fixture
def rig(amd):
    made = []

    def make(**more):
        made.append(Rig(amd, **more))
        return made[-1]

    yield make
    for r in made:
        r.close()


def _call(r, op, batch, n=1 << 20, p=None, **more):
    p = r.mem.alloc(16) if p is None else p
    if op == "append":
        r.cache.append_device(batch, p, n, p, n, **more)
    elif op == "read":
        r.cache.read_device(batch, p, n, p, n, **more)
    else:
        r.cache.attention_device(batch, p, n, more.pop("qh", r.qh), 1.0, p, n, p, more.pop("work", 1 << 40), **more)


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["append", "read", "attention"])
def test_calls_refuse(rig, op):
    """Refused on the host: none of these enqueues anything."""
    r = rig()
    width = r.heads * r.dim

    def batch(**more):
        c = dict(sequences=1, slots_ptr=16, lengths_ptr=16, starts_ptr=16, pages_ptr=16, pages_per_sequence=1, rows=3)
        c.update(more)
        return PagedBatch(**c)

    for bad, name in (("slots_ptr", "slots"), ("lengths_ptr", "lengths"), ("starts_ptr", "starts"), ("pages_ptr", "pages")):
        e = _refused(lambda: _call(r, op, batch(**{bad: 0})))
        assert (e.variant, e.name) == ("NullArgument", name)
    for bad in ({"sequences": 65536}, {"rows": 2 ** 31}, {"rows": 2 ** 24 + 1}, {"pages_per_sequence": 2 ** 31}):
        assert _refused(lambda: _call(r, op, batch(**bad))).variant == "Unsupported"
    stride = "q_stride" if op == "attention" else "k_stride"
    row = r.qh * r.dim if op == "attention" else width
    e = _refused(lambda: _call(r, op, batch(), **{stride: row - 1}))
    assert (e.variant, e.payload) == ("Shape", {"expected": row, "actual": row - 1})
    e = _refused(lambda: _call(r, op, batch(), n=3 * row - 1))
    assert (e.variant, e.payload) == ("Shape", {"expected": 3 * row, "actual": 3 * row - 1})
    assert _refused(lambda: _call(r, op, batch(), p=0)).variant == "NullArgument"
    assert _refused(lambda: _call(r, op, batch(), p=2)).variant == "Unsupported"  # not on an element
    err = kivi._Error()
    assert amd_backend()["paged_read_device"](r.cache._h, None, None, None, 0, 0, None, 0, 0, None, C.byref(err)) == 100
    if op == "attention":
        for qh in (0, 3):
            assert _refused(lambda: _call(r, op, batch(), qh=qh)).variant == "QueryHeads"
        # one of keys and values alone
        assert _refused(lambda: _call(r, op, batch(), k_ptr=16, k_len=1 << 20)).variant == "NullArgument"
        big = batch(rows=1, max_length=8192, pages_per_sequence=128)
        need = r.cache.attention_workspace_bytes(big, r.qh)
        assert need > 0
        e = _refused(lambda: _call(r, op, big, work=need - 1))
        assert (e.variant, e.a, e.b) == ("Capacity", need, need - 1)


@pytest.mark.gpu
def test_nothing_to_do_is_no_error(rig):
    r = rig()
    none = PagedBatch(0, 0, 0, 0, 0, 0, 0)
    for op in ("append", "read", "attention"):
        _call(r, op, none, n=0, p=0)
    assert r.cache.attention_workspace_bytes(none, r.qh) == 0
    r.append([0, 0, 0])
    r.append([5, 0, 3])
    assert r.read([0, 0, 0], [0, 0, 0])[0].shape[0] == 0


@pytest.mark.gpu
def test_getters(rig):
    r = rig(bits=4, group=32, residual=64, heads=3, dim=96, dtype="bf16", page=96, pages=36, slots=7)
    c = r.cache
    assert c.config() == KiviConfig(4, 32, 64)
    assert (c.num_kv_heads(), c.head_dim(), c.dtype(), c.page_tokens(), c.num_pages(), c.num_slots()) == (3, 96, "bf16", 96, 36, 7)
    per_token = 2 * (96 * 4 // 8 + 96 // 32 * 8)  # codes and (scale, zero) pairs, keys and values
    assert c.device_bytes() == 36 * 96 * 3 * per_token + 2 * 7 * 3 * 2 * 64 * 96 * 2


# ---------------------------------------------------------------- writes and reads

SHAPES = [
    # bits, group, residual, heads, dim, page
    (2, 32, 128, 2, 128, 64),
    (2, 16, 16, 1, 80, 32),    # a residual that ends inside a block, padded channels
    (2, 32, 32, 2, 32, 32),
    (4, 64, 128, 2, 64, 128),
    (4, 8, 24, 3, 24, 32),     # small groups, a residual of odd blocks
    (4, 32, 96, 1, 96, 96),
    (8, 4, 12, 2, 20, 32),     # channels that fill no 8
    (8, 128, 128, 1, 128, 256),
    (2, 48, 48, 1, 96, 96),    # spans of lcm(32, 48)
    (8, 20, 40, 1, 40, 160),
    (2, 16, 32, 1, 256, 32),
]


def _same(a, b):
    return np.array_equal(np.asarray(a, np.float32).view(np.uint32), np.asarray(b, np.float32).view(np.uint32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_write_and_read_back_bit_for_bit(rig, shape, dtype):
    """Ragged pieces of many sizes, read back after each: what the model holds, to the bit."""
    bits, group, residual, heads, dim, page = shape
    span = max(7 * residual, 300) + 200
    r = rig(bits=bits, group=group, residual=residual, heads=heads, dim=dim, dtype=dtype, page=page,
            per_sequence=-(-span // page) + 1, pages=3 * (-(-span // page) + 1) + 2, seed=bits * dim + page)
    for chunks in ([1, 0, residual - 1], [residual, 3, 1], [2 * residual + 5, 1, 1], [1, 77, 0], [1, residual + 1, 3 * residual],
                   [1, 1, 1], [residual, residual, residual]):
        r.append(chunks)
        n = [int(x) for x in r.lengths]
        first = [max(0, x - 2 * residual - 9) for x in n]
        for f in ([0] * 3, first):
            k, v = r.read(f, [x - y for x, y in zip(n, f)])
            want = [held(r.cfg, r.k[i], r.v[i], n[i]) for i in range(3)]
            assert _same(k, rounded(np.concatenate([w[0][y:] for w, y in zip(want, f)]), dtype))
            assert _same(v, rounded(np.concatenate([w[1][y:] for w, y in zip(want, f)]), dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("bits,group,residual,dim", [(2, 32, 128, 128), (4, 16, 48, 80), (8, 32, 64, 96)])
def test_a_sequence_is_a_kivi_cache(rig, oracle, bits, group, residual, dim):
    """The same tokens in the oracle's KiviCache: the same reconstruction, to the bit."""
    r = rig(bits=bits, group=group, residual=residual, dim=dim, page=96)
    for chunks in ([300, 5, 129], [1, 1, 1], [50, 200, 3]):
        r.append(chunks)
    n = [int(x) for x in r.lengths]
    k, v = r.read([0] * 3, n)
    at = 0
    for i in range(3):
        c = KiviCache(oracle, r.cfg, 1, r.heads, dim)
        c.append(r.k[i].transpose(1, 0, 2), r.v[i].transpose(1, 0, 2), n[i])
        wk, wv = (x.reshape(r.heads, n[i], dim).transpose(1, 0, 2) for x in c.dequantize())
        assert _same(k[at:at + n[i]], wk) and _same(v[at:at + n[i]], wv)
        at += n[i]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("stride,offset", [(2 * 64 + 8, 0), (2 * 64 + 3, 0), (2 * 64 + 8, 1), (5 * 64, 8)])
def test_strided_and_unaligned_rows(rig, dtype, stride, offset):
    r = rig(dtype=dtype)
    r.append([100, 31, 200], stride=stride, offset=offset, padded=3)
    r.append([1, 131, 7], stride=stride, offset=offset)
    n = [int(x) for x in r.lengths]
    k, v = r.read([0] * 3, n)
    want = [held(r.cfg, r.k[i], r.v[i], n[i]) for i in range(3)]
    assert _same(k, rounded(np.concatenate([w[0] for w in want]), dtype))
    assert _same(v, rounded(np.concatenate([w[1] for w in want]), dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 9, 128])
def test_appends_of_up_to_a_residual_length_are_taken_back(rig, m):
    """Drafted tokens refused: other tokens in their place, from any length in between, give what the
    sequence would hold without the draft; a repeated append changes nothing."""
    r = rig(sequences=2, per_sequence=12)
    r.append([250, 511])
    base = r.lengths.copy()
    draft = [r.tokens(m) for _ in range(2)]
    r.append([m, m], tokens=draft)
    r.append([m, m], tokens=draft, lengths=base)
    kept = m // 2
    r.append([m, m], lengths=base + kept)
    r.append([1, 1], lengths=base + m)
    n = [int(x) for x in r.lengths]
    k, v = r.read([0, 0], n)
    want = [held(r.cfg, r.k[i], r.v[i], n[i]) for i in range(2)]
    assert _same(k, np.concatenate([w[0] for w in want])) and _same(v, np.concatenate([w[1] for w in want]))


@pytest.mark.gpu
def test_values_outside_their_ranges_do_no_harm(rig):
    """Bad slots, pages, lengths and starts: others' tokens stay as they were, unheld tokens read as zeros."""
    r = rig(sequences=3, per_sequence=10)
    r.append([400, 300, 260])
    before = r.read([0] * 3, [400, 300, 260])
    k, v = r.tokens(60)
    kp, n, _ = r.upload(k)
    vp, n, _ = r.upload(v)

    def append(**more):
        args = dict(lengths=[400, 300, 260], chunks=[20, 20, 20], rows=60)
        args.update(more)
        r.cache.append_device(r.batch(args.pop("lengths"), args.pop("chunks"), **args), kp, n, vp, n)

    append(slots=[-1, 6, 2 ** 31 - 1])
    nowhere = np.full_like(r.table, -1)
    nowhere[:, ::2] = 10 ** 6
    # windows of slots that no sequence has: nothing of it is seen again
    free = [s for s in range(6) if s not in r.slots]
    append(table=nowhere, slots=free)
    append(starts=[-5, -1, -1, -1])
    append(starts=[2 ** 31 - 1, 60, 70, 60], slots=free)
    append(lengths=[2 ** 31 - 1] * 3, slots=free, table=nowhere)
    append(starts=[50, 10, 5, 2], slots=free)
    assert all(_same(a, b) for a, b in zip(before, r.read([0] * 3, [400, 300, 260])))

    gk, gv = r.read([0] * 3, [30] * 3, slots=[-1, 6, -2 ** 31])
    assert not gk.any() and not gv.any()
    gk, gv = r.read([0] * 3, [30] * 3, lengths=[-1, -2 ** 31, 0])
    assert not gk.any() and not gv.any()
    holes = r.table.copy()
    holes[0, 1] = -1
    holes[1, 0] = 40
    gk, gv = r.read([0] * 3, [400, 300, 260], table=holes)
    want = [x.copy() for x in before]
    for w in want:
        w[64:128] = 0
        w[400:464] = 0
    assert _same(gk, want[0]) and _same(gv, want[1])
    # behind the table, and behind the sequence
    gk, gv = r.read([390, 2 ** 31 - 40, -7], [30, 30, 5])
    wk, wv = before
    assert _same(gk[:10], wk[390:400]) and not gk[10:60].any() and _same(gk[60:], wk[700:705])
    assert _same(gv[:10], wv[390:400]) and not gv[10:60].any() and _same(gv[60:], wv[700:705])


@pytest.mark.gpu
def test_rows_behind_the_last_sequence_are_left(rig):
    r = rig()
    r.append([40, 300, 7])
    k, v = r.read([0, 0, 0], [40, 300, 7], fill=3.5, rows=360)
    assert (k[347:] == 3.5).all() and (v[347:] == 3.5).all()
    # a chunk longer than max_rows is cut to it
    k, v = r.read([0, 0, 0], [40, 300, 7], fill=3.5, rows=347, max_rows=50)
    assert (k[90:340] == 3.5).all() and not (k[:90] == 3.5).any() and not (k[340:] == 3.5).any()


@pytest.mark.gpu
def test_special_values(rig, oracle):
    """Constant groups, zeros of both signs, infinities and NaN go through as the reference's rule has it."""
    r = rig(sequences=1, dim=64, per_sequence=8)
    k, v = r.tokens(260)
    k[:32, 0, 3] = 5.0
    k[32:64, 0, 4] = np.where(np.arange(32) % 2, 0.0, -0.0)
    k[64:70, 1, 5] = np.nan
    k[96:128, 1, 6] = np.nan
    k[100, 0, 7] = np.inf
    v[3, 0, :32] = -2.0
    v[4, 1, 32:] = np.nan
    v[5, 1, 33] = np.nan
    v[6, 0, 1] = -np.inf
    v[7, 0, 2] = 1e-42
    r.append([260], tokens=[(k, v)])
    got = r.read([0], [260])
    c = KiviCache(oracle, r.cfg, 1, r.heads, 64)
    c.append(k.transpose(1, 0, 2), v.transpose(1, 0, 2), 260)
    want = [x.reshape(r.heads, 260, 64).transpose(1, 0, 2) for x in c.dequantize()]
    for a, b in zip(got, want):
        assert np.array_equal(np.isnan(a), np.isnan(b))
        assert np.array_equal(a[~np.isnan(b)], b[~np.isnan(b)])


# ---------------------------------------------------------------- attention

ATTEND = [
    # bits, group, residual, heads, gq, dim, page
    (2, 32, 128, 2, 4, 128, 64),
    (4, 32, 128, 2, 1, 64, 128),
    (8, 16, 32, 1, 7, 80, 32),
    (2, 16, 16, 1, 3, 96, 32),
    (4, 8, 24, 2, 2, 24, 32),
    (8, 20, 40, 1, 5, 40, 160),
    (2, 48, 48, 1, 2, 96, 96),
    (4, 64, 64, 1, 8, 256, 64),
    (2, 128, 128, 1, 16, 128, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", ATTEND, ids=lambda s: "-".join(map(str, s)))
def test_attention(rig, shape, dtype):
    """Decode, drafted tokens and chunks, with the new rows given or written first, ragged lengths from nothing."""
    bits, group, residual, heads, gq, dim, page = shape
    per = -(-900 // page)
    r = rig(bits=bits, group=group, residual=residual, heads=heads, gq=gq, dim=dim, dtype=dtype, page=page,
            sequences=4, per_sequence=per, pages=4 * per, slots=4, seed=dim + gq)
    scale = dim ** -0.5
    r.append([650, 1, residual, 0])
    for chunks in ([1, 1, 1, 1], [5, 1, 3, 2], [70, 0, 33, 1], [1, 130, 1, 61]):
        q = r.queries(sum(chunks) + 2)
        new = [r.tokens(m) for m in chunks]
        r.check(q, chunks, scale, new=new)
        r.append(chunks, tokens=new)
        r.check(q, chunks, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (40, 0), (64, 4), (200, 37), (500, 130), (10 ** 12, 10 ** 13)])
def test_window_and_sinks(rig, window, sinks, dtype):
    r = rig(dtype=dtype, sequences=4, gq=4, slots=4, pages=48, page=32, residual=64, per_sequence=12, dim=64)
    r.append([300, 20, 0, 111])
    for chunks in ([1, 1, 1, 1], [7, 2, 1, 3], [45, 50, 30, 1]):
        q, new = r.queries(sum(chunks)), [r.tokens(m) for m in chunks]
        r.check(q, chunks, 0.125, new=new, window=window, sinks=sinks)
    r.check(r.queries(9), [3, 3, 0, 3], 0.125, window=window, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks,chunk", [(100, 5, 1), (64, 0, 3), (65, 33, 40)])
def test_pages_behind_a_window_are_not_read(rig, window, sinks, chunk):
    r = rig(sequences=2, slots=2, per_sequence=20, dim=64, page=32, residual=32)
    r.append([600, 333])
    chunks = [chunk, chunk]
    q, new = r.queries(2 * chunk), [r.tokens(chunk) for _ in range(2)]
    whole = r.check(q, chunks, 0.2, new=new, window=window, sinks=sinks)
    table = r.table.copy()
    for i, n in enumerate((600, 333)):
        table[i, -(-sinks // 32):(n + 1 - window) // 32] = -1
    assert (table != r.table).any()
    assert _same(whole, r.check(q, chunks, 0.2, new=new, window=window, sinks=sinks, table=table))


@pytest.mark.gpu
def test_tokens_of_no_page_are_seen_by_no_query(rig):
    r = rig(sequences=2, slots=2, per_sequence=10)
    r.append([500, 260])
    holes = r.table.copy()
    holes[0, [0, 3]] = -1
    holes[1, :] = 10 ** 7
    gone = [np.zeros(500, bool), np.zeros(260, bool)]
    gone[0][:64] = gone[0][192:256] = True
    gone[1][:256] = True  # keys behind 256 lie in the window
    for chunks in ([1, 1], [20, 3]):
        r.check(r.queries(sum(chunks)), chunks, 0.1, table=holes, hidden=gone)


@pytest.mark.gpu
def test_rows_that_see_nothing_are_zero(rig):
    """More queries than tokens, sequences of no tokens, no slot: zeros, and neighbours untouched."""
    r = rig(sequences=3, slots=4)
    r.append([3, 200, 0])
    q = r.queries(12)
    got = r.check(q, [5, 2, 5], 0.3)
    assert not got[:2].any() and not got[7:].any() and got[2:7].any()
    got = r.attention(q, [5, 2, 5], 0.3, slots=[9, int(r.slots[1]), -1])
    assert not got[:5].any() and not got[7:].any() and got[5:7].any()
    # no slot but rows of its own: attention over those
    new = [r.tokens(m) for m in (5, 2, 5)]
    got = r.attention(q, [5, 2, 5], 0.3, new=new, slots=[-1, -1, -1])
    want, bound = r.expected(q, [5, 2, 5], 0.3, new=new, lengths=[0, 0, 0])
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stride,offset", [(4 * 64 + 8, 0), (4 * 64 + 5, 0), (4 * 64 + 16, 3)])
def test_attention_of_strided_and_unaligned_rows(rig, dtype, stride, offset):
    r = rig(dtype=dtype)
    r.append([300, 40, 129])
    for chunks in ([1, 1, 1], [40, 3, 17]):
        q, new = r.queries(sum(chunks) + 1), [r.tokens(m) for m in chunks]
        r.check(q, chunks, 0.125, new=new, stride=stride, offset=offset)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
@pytest.mark.parametrize("m", [1, 40])
def test_other_scales(rig, scale, m):
    r = rig(sequences=2, slots=2)
    r.append([400, 17])
    r.check(r.queries(2 * m), [m, m], scale, new=[r.tokens(m) for _ in range(2)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,spread", [("f32", 1e12), ("f32", 1e-12), ("bf16", 1e10), ("bf16", 1e-10), ("f16", 3e2), ("f16", 1e-3)])
@pytest.mark.parametrize("m", [1, 33])
def test_magnitudes(rig, dtype, spread, m):
    """Keys and values of any magnitude that the type holds, queries scaled against them."""
    r = rig(dtype=dtype, sequences=1, slots=1, per_sequence=8)
    tokens = r.tokens(400, spread)
    r.append([400], tokens=[tokens])
    q = r.queries(m)
    r.check(q, [m], 0.125 / spread, new=[r.tokens(m, spread)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_what_a_row_does_not_see_does_not_reach_it(rig, dtype):
    """NaN and infinities in tokens behind a row's position, in front of its window, in unused window
    rows and pages, and in padding: rows that do not see them are as without them."""
    r = rig(dtype=dtype, sequences=2, slots=3, per_sequence=10, residual=32, page=32, dim=64)
    bad = [r.tokens(300), r.tokens(130)]
    for k, v in bad:
        k[:, 0, 5], v[:, 1, 7] = np.inf, np.nan
    r.append([300, 130], tokens=bad)      # old content of pages and windows
    r.lengths[:] = 0
    r.k, r.v = [x[:0] for x in r.k], [x[:0] for x in r.v]
    r.append([150, 70])
    chunks = [40, 7]
    new = [r.tokens(m) for m in chunks]
    clean = r.check(r_q := r.queries(47), chunks, 0.125, new=new)
    poisoned = [(k.copy(), v.copy()) for k, v in new]
    poisoned[0][0][20, 0, 1], poisoned[0][1][20, 0, 2], poisoned[0][1][33, 1, 9] = np.nan, np.inf, np.nan
    poisoned[1][1][6] = np.nan
    got = r.attention(r_q, chunks, 0.125, new=poisoned)
    assert _same(got[:20], clean[:20]) and _same(got[40:46], clean[40:46])
    assert not np.isfinite(got[20:40]).all() and np.isnan(got[46]).any()
    # the window's front edge
    got = r.attention(r_q, chunks, 0.125, new=poisoned, window=5)
    want = r.attention(r_q, chunks, 0.125, new=new, window=5)
    for rows in (slice(0, 20), slice(25, 33), slice(38, 40), slice(40, 46)):
        assert _same(got[rows], want[rows])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("f32", 96), ("bf16", 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (300, 70)])
def test_chunks_over_many_tiles(rig, dtype, dim, window, sinks):
    """Packed tiles, tiles of rows and those that are neither in the walk of one workgroup (enough rows to fill the
    device) and cut into splits (few), with a page missing among the packed ones, the new rows given or written."""
    r = rig(dtype=dtype, dim=dim, heads=4, gq=8, sequences=6, slots=6, residual=64, page=64, per_sequence=20, pages=120)
    r.append([700, 640, 10, 0, 1000, 333])
    holes = r.table.copy()
    holes[0, 9] = holes[4, 12] = -1
    gone = [np.zeros(n, bool) for n in (700, 640, 10, 0, 1000, 333)]
    gone[0][576:640] = gone[4][768:832] = True
    chunks = [200] * 6
    for few in (False, True):
        counts = [200, 0, 0, 0, 0, 0] if few else chunks
        new = [r.tokens(m) for m in counts]
        r.check(r.queries(sum(counts)), counts, dim ** -0.5, new=new, window=window, sinks=sinks, table=holes,
                hidden=[np.concatenate([g, np.zeros(m, bool)]) for g, m in zip(gone, counts)])
    r.append(chunks)
    r.check(r.queries(400), [200, 0, 0, 0, 200, 0], dim ** -0.5, window=window, sinks=sinks)


@pytest.mark.gpu
def test_bounds_only_plan(rig):
    """`max_length` and the table's size change the plan, never the meaning."""
    r = rig(sequences=2, slots=2, per_sequence=20, pages=40, dim=64)
    r.append([1100, 90])
    q, chunks = r.queries(2), [1, 1]
    want, bound = r.expected(q, chunks, 0.125)
    for more in ({"max_length": 1}, {"max_length": 500}, {"max_length": 1100}, {"max_length": 10 ** 9}):
        assert (np.abs(r.attention(q, chunks, 0.125, **more) - want) <= bound).all()


@pytest.mark.gpu
def test_shared_pages(rig):
    """Two sequences read the same pages (a prefix both have), in one call."""
    r = rig(sequences=2, slots=4, per_sequence=10, residual=64)
    r.append([512, 0])
    # a second window with the first one's rows: the last 128 tokens appended again to another slot
    k, v = r.k[0], r.v[0]
    scratch = np.full_like(r.table, -1)
    kp, n, _ = r.upload(np.concatenate([k[384:], k[:0]]))
    vp, n, _ = r.upload(v[384:])
    r.cache.append_device(r.batch([384, 0], [128, 0], table=scratch, slots=[int(r.slots[1]), int(r.slots[1])]), kp, n, vp, n)
    r.mem.wait()
    r.k[1], r.v[1], r.lengths[1] = k, v, 512
    r.table[1] = r.table[0]
    r.check(r.queries(6), [3, 3], 0.125, new=[r.tokens(3) for _ in range(2)])


@pytest.mark.gpu
def test_records_behind_four_gigabytes(rig):
    """Pages and windows whose offsets pass 32 bits in bytes and in words."""
    heads, dim, page, residual = 4, 128, 1024, 128
    record = page * 2 * (dim // 4 + dim // 32 * 8) * heads
    pages = (17 << 30) // record
    slots = (5 << 30) // (heads * 2 * residual * dim * 2)
    r = rig(heads=heads, dim=dim, page=page, residual=residual, dtype="bf16", pages=pages, slots=slots, sequences=2, per_sequence=2)
    r.table[:] = [[pages - 1, 0], [pages // 2, pages - 2]]
    r.slots[:] = [slots - 1, slots // 2]
    r.append([1200, 900])
    r.append([1, 200])
    k, v = r.read([1000, 800], [201, 300])
    want = [held(r.cfg, r.k[i], r.v[i], int(r.lengths[i])) for i in range(2)]
    assert _same(k, rounded(np.concatenate([want[0][0][1000:], want[1][0][800:]]), "bf16"))
    assert _same(v, rounded(np.concatenate([want[0][1][1000:], want[1][1][800:]]), "bf16"))
    r.check(r.queries(4), [1, 3], 0.088, new=[r.tokens(1), r.tokens(3)])


# ---------------------------------------------------------------- streams and graphs


@pytest.mark.gpu
def test_a_captured_step_replays_for_growing_sequences(rig):
    """One graph of a serving step (attention over the cache and the new rows, then their append),
    replayed with other rows and lengths in the same arrays."""
    r = rig(sequences=3, slots=3, dtype="bf16", per_sequence=10, residual=32, page=32, gq=4)
    hip = C.CDLL("libamdhip64.so.7")
    r.append([190, 31, 0])
    chunks = [1, 2, 1]
    q, new = r.queries(4), [r.tokens(m) for m in chunks]
    qp, qn, _ = r.upload(q)
    op, on, _ = r.upload(np.zeros_like(q))
    kp, kn, _ = r.upload(np.concatenate([k for k, _ in new]))
    vp, vn, _ = r.upload(np.concatenate([v for _, v in new]))
    batch = r.batch(r.lengths, chunks)
    size = r.cache.attention_workspace_bytes(batch, r.qh)
    work = r.mem.put(np.zeros(size // 4 + 1, np.float32))
    stream = C.c_void_p()
    assert hip.hipStreamCreate(C.byref(stream)) == 0

    def step():
        r.cache.attention_device(batch, qp, qn, r.qh, 0.125, op, on, work, size, k_ptr=kp, k_len=kn, v_ptr=vp, v_len=vn,
                                 stream=stream.value)
        r.cache.append_device(batch, kp, kn, vp, vn, stream=stream.value)

    graph, exe = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 0) == 0
    step()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    for turn in range(40):
        q, new = r.queries(4), [r.tokens(m) for m in chunks]
        r.mem.write(qp, to_bits(q, "bf16"))
        r.mem.write(kp, to_bits(np.concatenate([k for k, _ in new]), "bf16"))
        r.mem.write(vp, to_bits(np.concatenate([v for _, v in new]), "bf16"))
        r.mem.write(batch._c.lengths, r.lengths.astype(np.int32))
        assert hip.hipGraphLaunch(exe, stream) == 0
        assert hip.hipStreamSynchronize(stream) == 0
        got = to_floats(r.mem.get(op, q.shape, RAW["bf16"]), "bf16")
        want, bound = r.expected(q, chunks, 0.125, new=new)
        assert (np.abs(got - want) <= bound).all(), turn
        for i, (k, v) in enumerate(new):
            r.k[i], r.v[i] = np.concatenate([r.k[i], k]), np.concatenate([r.v[i], v])
        r.lengths += chunks
        if turn % 13 == 0:  # the program's own eager work in between
            k, v = r.read([0] * 3, [int(x) for x in r.lengths])
            w = [held(r.cfg, r.k[i], r.v[i], int(r.lengths[i])) for i in range(3)]
            assert _same(k, rounded(np.concatenate([x[0] for x in w]), "bf16"))
    assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0 and hip.hipStreamDestroy(stream) == 0


@pytest.mark.gpu
def test_calls_on_two_streams(rig):
    """Two halves of the sequences served on two streams at once, each with its workspace."""
    r = rig(sequences=4, slots=4, per_sequence=10, gq=4)
    hip = C.CDLL("libamdhip64.so.7")
    r.append([600, 200, 555, 31])
    q = r.queries(4)
    new = [r.tokens(1) for _ in range(4)]
    want, bound = r.expected(q, [1] * 4, 0.125, new=new)
    streams = [C.c_void_p(), C.c_void_p()]
    jobs = []
    for i, s in enumerate(streams):
        assert hip.hipStreamCreate(C.byref(s)) == 0
        mine = slice(2 * i, 2 * i + 2)
        batch = r.batch(r.lengths[mine], [1, 1], table=r.table[mine], slots=r.slots[mine])
        size = r.cache.attention_workspace_bytes(batch, r.qh)
        jobs.append((batch, r.upload(q[mine]), r.upload(np.zeros_like(q[mine])),
                     r.upload(np.concatenate([k for k, _ in new[mine]])), r.upload(np.concatenate([v for _, v in new[mine]])),
                     r.mem.put(np.zeros(size // 4 + 1, np.float32)), size, s))
    for _ in range(5):
        for batch, qu, out, k, v, work, size, s in jobs:
            r.cache.attention_device(batch, qu[0], qu[1], r.qh, 0.125, out[0], out[1], work, size, k_ptr=k[0], k_len=k[1],
                                     v_ptr=v[0], v_len=v[1], stream=s.value)
            r.cache.append_device(batch, k[0], k[1], v[0], v[1], stream=s.value)
    got = np.concatenate([to_floats(r.mem.get(job[2][0], (2, r.qh, r.dim), RAW["f32"]), "f32") for job in jobs])
    assert (np.abs(got - want) <= bound).all()
    for s in streams:
        assert hip.hipStreamDestroy(s) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_prompt_in_pieces_then_tokens(rig, oracle, dtype):
    """A run of the operators as a server has them: prompts in pieces over what is cached so far, then
    tokens one by one; each step's outputs and at the end the whole cache."""
    r = rig(dtype=dtype, sequences=2, slots=3, per_sequence=12, gq=4, residual=64)
    for chunks in ([200, 90], [130, 64], [1, 150], [1, 1], [1, 1], [64, 1], [1, 1]):
        q, new = r.queries(sum(chunks)), [r.tokens(m) for m in chunks]
        r.check(q, chunks, 0.125, new=new)
        r.append(chunks, tokens=new)
    n = [int(x) for x in r.lengths]
    k, v = r.read([0, 0], n)
    want = [held(r.cfg, r.k[i], r.v[i], n[i]) for i in range(2)]
    assert _same(k, rounded(np.concatenate([w[0] for w in want]), dtype))
    assert _same(v, rounded(np.concatenate([w[1] for w in want]), dtype))
    # a decoded token over the finished caches, beside the oracle's cache of the same tokens
    q = r.queries(2)
    got = r.check(q, [1, 1], 0.125)
    if dtype == "f32":
        for i in range(2):
            c = KiviCache(oracle, r.cfg, 1, r.heads, r.dim)
            c.append(r.k[i].transpose(1, 0, 2), r.v[i].transpose(1, 0, 2), n[i])
            np.testing.assert_allclose(got[i].reshape(-1), c.attention(q[i], r.qh, 0.125), rtol=1e-4, atol=1e-5)
