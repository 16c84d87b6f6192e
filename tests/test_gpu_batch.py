"""Several requests at once over a cache in 4 bits, each operator against its definition in 64 bits (batch_plain.py) at the sizes and
masks where it can go wrong, then a run of all of them together, captured and on streams of their own."""
import ctypes
import zlib

import numpy as np
import pytest

import batch_plain as plain
from batch_plain import DTYPES, EPS, PAGE, pages

pytestmark = pytest.mark.gpu


@pytest.fixture
def dev(torch_gpu, awq, lib):
    return Device(torch_gpu, awq, lib)


class Device:
    def __init__(self, torch, awq, lib):
        self.torch, self.awq, self.lib = torch, awq, lib
        self.types = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

    def stream(self):
        return ctypes.c_void_p(self.torch.cuda.current_stream().cuda_stream)

    def act(self, x, dtype):
        """(tensor, the values it holds)"""
        t = self.torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda().to(self.types[dtype])
        return t, self.host(t)

    def ints(self, x):
        return self.torch.tensor(np.asarray(x, np.int64), dtype=self.torch.int32, device="cuda")

    def floats(self, x):
        return self.torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()

    def full(self, shape, fill, dtype):
        return self.torch.full(shape, fill, dtype=self.types.get(dtype, dtype), device="cuda")

    def host(self, t):
        self.torch.cuda.synchronize()
        return t.double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()

    def bits(self, t):
        return self.host(t.view(self.torch.int16 if t.element_size() == 2 else self.torch.int32))


def rng_of(*seed):
    return np.random.default_rng([zlib.crc32(s.encode()) if isinstance(s, str) else int(s) for s in seed])


def tables(rng, n_requests, held, width, spare=5):
    """(table, n_pages) of random pages"""
    total = sum(held)
    order = rng.permutation(total + spare)
    table, at = np.full((n_requests, width), -1, np.int64), 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    return table, total + spare


# --- pages and slots ----------------------------------------------------------------------------------------------------
def run_plan(dev, cached, fresh, table, stack, n_pages, max_tokens, in_place=True, keys=True):
    n, width = table.shape
    d_table, free = dev.ints(table), dev.ints(list(stack) + [-7] * (n_pages - len(stack)))
    count, out = dev.ints([len(stack)]), dev.ints([-7])
    i = lambda m: dev.full((m,), -7, dev.torch.int32)  # noqa: E731
    lengths, starts, key_starts, positions, slots, left = i(max(n, 1)), i(n + 1), i(n + 1), i(max_tokens + 3), i(max_tokens + 3), i(1)
    c, f = dev.ints(cached if n else [0]), dev.ints(fresh if n else [0])
    a = dev.awq.AwqPagePlanArgs(c.data_ptr(), f.data_ptr(), d_table.data_ptr() if n else None, free.data_ptr(), count.data_ptr(),
                                count.data_ptr() if in_place else out.data_ptr(), lengths.data_ptr(), starts.data_ptr(),
                                key_starts.data_ptr() if keys else None, positions.data_ptr(), slots.data_ptr(), left.data_ptr() if keys else None,
                                max_tokens, n, width, n_pages, 0)
    dev.awq.check(dev.lib.awq_page_plan(ctypes.byref(a), dev.stream()))
    h = dev.host
    if not in_place:
        assert h(count)[0] == len(stack)
        count = out
    assert (h(positions)[max_tokens:] == -7).all() and (h(slots)[max_tokens:] == -7).all()
    if not keys:
        assert (h(key_starts) == -7).all() and h(left)[0] == -7
    return (h(d_table), h(free), int(h(count)[0]), h(lengths)[:n], h(starts), h(key_starts), h(positions)[:max_tokens], h(slots)[:max_tokens], int(h(left)[0]))


def check_plan(got, want, n_free, keys=True):
    table, given, count, lengths, starts, key_starts, positions, slots, left = want
    assert np.array_equal(got[0], table) and got[2] == count
    assert got[1][:len(given)].tolist() == given and (got[1][len(given):] == -7).all()
    assert got[3].tolist() == lengths and got[4].tolist() == starts
    if keys:
        assert got[5].tolist() == key_starts and got[8] == left
    assert got[6].tolist() == positions and got[7].tolist() == slots


@pytest.mark.parametrize("n", [0, 1, 2, 5, 200, 1023, 1024, 1025, 3000])
@pytest.mark.parametrize("plenty", [True, False], ids=["plenty", "short"])
def test_plan(dev, n, plenty):
    rng = rng_of(n, plenty)
    width = 20
    cached = rng.choice([0, 1, 63, 64, 65, 128, 700, 64 * width - 1, 64 * width], n)
    fresh = rng.choice([-1, 0, 1, 1, 1, 1, 64, 65, 300], n)
    held = [pages(c) for c in cached]
    table, n_pages = tables(rng, n, held, width, 20 * n + 40)
    used = set(table[table >= 0].tolist())
    spare = [p for p in range(n_pages) if p not in used]
    stack = spare if plenty else spare[:max(1, n // 3)]
    total = int(np.maximum(fresh, 0).sum())
    print("plan", n, plenty, total, flush=True)
    for max_tokens, in_place, keys in ((total, True, True), (total + 70, False, False), (max(0, total - 3), True, True)):
        want = plain.plan(cached, fresh, table, stack, n_pages, max_tokens)
        got = run_plan(dev, cached, fresh, table, stack, n_pages, max_tokens, in_place, keys)
        check_plan(got, want, len(stack), keys)


def test_plan_of_numbers_out_of_range(dev):
    """counts and entries that no program should pass: nothing is read or written out of range"""
    cached, fresh = [-5, 10 ** 9, 100, 64], [3, 1, 10 ** 9, 2]
    table = np.array([[1, 2], [3, 4], [99, -8], [7, 7]])
    got = run_plan(dev, cached, fresh, table, [5, 6, 77], 9, 40)
    # cached as 0 and 128 of 128; the second and the third do not fit; the first takes the list's last entry, which is no page
    assert got[3].tolist() == [3, 128, 100, 66] and got[8] == 2 and got[2] == 1
    assert got[0].tolist() == [[77, 2], [3, 4], [99, -8], [7, 6]]
    assert got[7][:4].tolist() == [-1, -1, -1, -1] and got[6][:4].tolist() == [0, 1, 2, 128]


# --- rotary positions, append, rows ---------------------------------------------------------------------------------------
def append(dev, dtype, q, k, v, cos, sin, positions, slots, cache, heads, kv, dim, rot, interleaved, q_out, k_out):
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    a = dev.awq.AwqPagedAppendArgs(at(q), at(q_out), at(k), at(k_out), at(v), at(cos), at(sin), at(positions), at(slots), at(cache), ld(q), ld(q_out),
                                   ld(k), ld(k_out), ld(v), len(positions), 0 if cos is None else cos.shape[0], heads, kv, dim, rot, int(interleaved),
                                   0 if cache is None else cache.shape[0])
    if rot == 0:
        a.max_pos = 1 << 20
    dev.awq.check(dev.lib.awq_paged_append(ctypes.byref(a), DTYPES[dtype], dev.stream()))


SHAPES = [(1, 1, 64), (6, 2, 64), (8, 8, 128), (12, 3, 128), (4, 1, 256), (20, 2, 256)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("turn", [(0, False), (16, True), (16, False), (48, False), ("all", True), ("all", False)], ids=str)
def test_append(dev, dtype, shape, turn):
    heads, kv, dim = shape
    rot, interleaved = dim if turn[0] == "all" else turn[0], turn[1]
    rng = rng_of(dtype, heads, dim, rot, interleaved)
    T, n_pages, max_pos = 37, 4, 500
    print("append", dtype, shape, turn, flush=True)
    x = rng.standard_normal((T, (heads + 2 * kv) * dim + 24)) * np.exp(rng.standard_normal((T, 1)))
    x[5] = 0.0            # one value throughout
    x[6] = 3.0
    x[7] *= 1e-6          # below binary16's normal numbers
    d_x, vx = dev.act(x, dtype)
    cut = np.cumsum([0, heads, kv, kv]) * dim
    q, k, v = (d_x[:, a:b] for a, b in zip(cut, cut[1:]))
    vq, vk, vv = (vx[:, a:b].reshape(T, -1, dim) for a, b in zip(cut, cut[1:]))
    positions = rng.integers(0, max_pos, T)
    positions[3], positions[4] = -1, max_pos
    slots = rng.permutation(n_pages * PAGE)[:T]
    slots[10], slots[11] = -1, n_pages * PAGE
    angle = rng.random((max_pos, max(rot // 2, 1))) * 7
    cos, sin = dev.floats(np.cos(angle)), dev.floats(np.sin(angle))
    if rot == 0:
        positions[4] = 1 << 20
    there = (positions >= 0) & (positions < (max_pos if rot else 1 << 20))
    at = np.where(there, positions, 0) % max_pos
    c, s = (np.asarray(dev.host(t)[at], np.float64)[:, :rot // 2] for t in (cos, sin))
    want_q, want_k = (plain.nearest(plain.turned(w, c, s, rot, interleaved), dtype) for w in (vq, vk))
    empty = rng.integers(0, 256, (n_pages, kv, 72 * dim), dtype=np.uint8)
    expect = empty.copy()
    kn, ks, kz = plain.quantised(want_k)
    vn, vs, vz = plain.quantised(vv)
    kept = there & (slots >= 0) & (slots < n_pages * PAGE)
    for t in np.flatnonzero(kept):
        page, p = divmod(int(slots[t]), PAGE)
        one = plain.packed_pages(*(tuple(np.repeat(y[t][None, :, None], PAGE, 2) for y in z) for z in ((kn, ks, kz), (vn, vs, vz))))[0]
        half = 64 * dim
        for lo, hi, step in ((0, half, dim // 2), (half, 72 * dim, 2)):
            rows = expect[page, :, lo:hi].reshape(kv, -1, PAGE, step)
            rows[:, :, p] = one[:, lo:hi].reshape(kv, -1, PAGE, step)[:, :, p]
    for in_place in (False, True):
        cache = dev.torch.from_numpy(empty.copy()).cuda()
        mine = d_x.clone()
        q, k, v = (mine[:, a:b] for a, b in zip(cut, cut[1:]))
        q_out, k_out = (q, k) if in_place else (dev.full((T, heads * dim + 8), 9.0, dtype), dev.full((T, kv * dim), 9.0, dtype))
        append(dev, dtype, q, k, v, cos if rot else None, sin if rot else None, dev.ints(positions), dev.ints(slots), cache, heads, kv, dim, rot,
               interleaved, q_out, k_out)
        for got, w, was in ((q_out, want_q, vq), (k_out, want_k, vk)):
            got = dev.host(got)[:, :w[0].size].reshape(w.shape)
            assert np.array_equal(got[there], w[there])
            assert np.array_equal(got[~there], was[~there]) if in_place else (got[~there] == 9.0).all()
        if not in_place:
            assert (dev.host(q_out)[:, heads * dim:] == 9.0).all()
        assert np.array_equal(dev.host(cache), expect)
    # the rotary positions alone, of queries alone, and the append without k_out and queries
    q_out = dev.full((T, heads * dim), 9.0, dtype)
    q, k, v = (d_x[:, a:b] for a, b in zip(cut, cut[1:]))
    d_pos, d_slots = dev.ints(positions), dev.ints(slots)
    append(dev, dtype, q, None, None, cos if rot else None, sin if rot else None, d_pos, None, None, heads, kv, dim, rot, interleaved, q_out, None)
    assert np.array_equal(dev.host(q_out).reshape(want_q.shape)[there], want_q[there])
    cache = dev.torch.from_numpy(empty.copy()).cuda()
    append(dev, dtype, None, k, v, cos if rot else None, sin if rot else None, d_pos, d_slots, cache, heads, kv, dim, rot, interleaved, None, None)
    assert np.array_equal(dev.host(cache), expect)


def rows_of(dev, dtype, cache, table, first, lengths, starts, n_rows, kv, dim, want=(True, True), fill=9.0, pad=8):
    k, v = (dev.full((n_rows, kv * dim + pad), fill, dtype) if w else None for w in want)
    n, width = table.shape
    tensors = [dev.ints(table), None if first is None else dev.ints(first), dev.ints(lengths), dev.ints(starts)]
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    a = dev.awq.AwqPagedRowsArgs(cache.data_ptr(), *(at(t) for t in tensors), at(k), at(v), kv * dim + pad, kv * dim + pad, n_rows, n, width, cache.shape[0],
                                 kv, dim, 0)
    dev.awq.check(dev.lib.awq_paged_rows(ctypes.byref(a), DTYPES[dtype], dev.stream()))
    return [None if t is None else dev.host(t) for t in (k, v)]


def cache_of(dev, rng, n_pages, kv, dim, scale=1.0):
    """a random cache: (tensor, keys, values) [pages][heads][64][dim], and the nibble parts of the values without their offsets"""
    out, values, parts = [], [], []
    for _ in range(2):
        n = rng.integers(0, 16, (n_pages, kv, PAGE, dim)).astype(np.float64)
        s = plain.nearest(scale * np.exp(0.5 * rng.standard_normal((n_pages, kv, PAGE, dim // 64))) * 0.2, "f16")
        z = plain.nearest(s * (-7.5 + 2 * rng.standard_normal(s.shape)), "f16")
        out.append((n, s, z))
        values.append(plain.value_of(n, s, z))
        parts.append(plain.value_of(n, s, np.abs(z)))
    return dev.torch.from_numpy(plain.packed_pages(*out)).cuda(), values[0], values[1], parts[1]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kv,dim", [(1, 64), (3, 128), (2, 256)])
def test_rows(dev, dtype, kv, dim):
    rng = rng_of(dtype, kv, dim)
    lengths, first = [0, 1, 64, 200, 65, 3, 130], [0, 0, 10, 150, 65, 9, 0]
    width = 4
    table, n_pages = tables(rng, len(lengths), [pages(x) for x in lengths], width)
    table[3, 3], table[6, 0] = -1, n_pages
    cache, k, v, _ = cache_of(dev, rng, n_pages, kv, dim)
    counts = [max(0, a - b) for a, b in zip(lengths, first)]
    counts[2] += 4  # rows that no position has
    starts = np.cumsum([2] + counts)
    n_rows = int(starts[-1]) + 5
    wants = []
    for x in (k, v):
        w = np.full((n_rows, kv, dim), 9.0)
        for i, (lo, hi) in enumerate(zip(first, lengths)):
            for p in range(lo, hi):
                page = table[i, p // PAGE]
                w[starts[i] + p - lo] = plain.nearest(x[page, :, p % PAGE], dtype) if 0 <= page < n_pages else 0.0
        wants.append(w.reshape(n_rows, -1))
    for want in ((True, True), (True, False), (False, True)):
        got = rows_of(dev, dtype, cache, table, first, lengths, starts, n_rows, kv, dim, want)
        for g, w in zip(got, wants):
            if g is not None:
                assert np.array_equal(g[:, :kv * dim], w) and (g[:, kv * dim:] == 9.0).all()
    # from the first position on; the rows given out are fewer than there are positions
    got = rows_of(dev, dtype, cache, table, None, lengths, np.cumsum([0] + lengths), 100, kv, dim)
    assert np.array_equal(got[0][1:65, :kv * dim], plain.nearest(k[table[2, 0]].transpose(1, 0, 2).reshape(64, -1), dtype))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_append_of_what_is_not_finite_or_large(dev, dtype):
    """64 values with a NaN or an infinity read as NaN, their neighbours as they are; large bfloat16 values as binary16's largest"""
    kv, dim, T = 2, 128, 6
    x = rng_of(dtype).standard_normal((T, kv * dim))
    x[0, 5], x[1, 70], x[2, 130], x[3, 255] = np.nan, np.inf, -np.inf, np.nan
    if dtype == "bf16":
        x[4, 3], x[4, 100], x[5, 130], x[5, 140] = 1e30, -1e30, 3e38, -3e38
    d_x, vx = dev.act(x, dtype)
    cache = dev.torch.zeros((1, kv, 72 * dim), dtype=dev.torch.uint8, device="cuda")
    append(dev, dtype, None, d_x, d_x, None, None, dev.ints(range(T)), dev.ints(range(T)), cache, 1, kv, dim, 0, False, None, None)
    with np.errstate(invalid="ignore"):
        want = plain.nearest(plain.value_of(*plain.quantised(vx.reshape(T, kv, dim))), dtype).reshape(T, -1)
    got = rows_of(dev, dtype, cache, np.array([[0]]), None, [T], [0, T], T, kv, dim, pad=0)
    assert np.isnan(want).sum() == 4 * 64
    for g in got:
        assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(g[~np.isnan(g)], want[~np.isnan(want)])


def test_two_tokens_of_one_slot_leave_its_neighbours_alone(dev):
    kv, dim, T = 2, 64, 8
    d_x, _ = dev.act(rng_of(9).standard_normal((T, kv * dim)), "f16")
    cache = dev.torch.full((2, kv, 72 * dim), 77, dtype=dev.torch.uint8, device="cuda")
    append(dev, "f16", None, d_x, d_x, None, None, dev.ints(range(T)), dev.ints([5, 5, 5, 70, 5, 70, 5, 5]), cache, 1, kv, dim, 0, False, None, None)
    got = dev.host(cache)
    for page, p in ((0, 5), (1, 6)):
        data, par = got[page, :, :64 * dim].reshape(kv, 2, PAGE, -1), got[page, :, 64 * dim:].reshape(kv, -1, PAGE, 2)
        others = np.arange(PAGE) != p
        assert (data[:, :, others] == 77).all() and (par[:, :, others] == 77).all()


# --- attention over pages ---------------------------------------------------------------------------------------------------
def paged(dev, dtype, q, cache, table, lengths, heads, kv, dim, scale, ctx, width=None):
    n, w = table.shape
    size = dev.lib.awq_paged_workspace_bytes(n, heads, kv, dim, w)
    ws = dev.full((size // 4,), float("nan"), "f32")
    d_table, d_lengths = dev.ints(table), dev.ints(lengths)
    a = dev.awq.AwqPagedAttentionArgs(q.data_ptr(), cache.data_ptr(), d_table.data_ptr(), d_lengths.data_ptr(), ctx.data_ptr(), ws.data_ptr(), q.stride(0),
                                      ctx.stride(0), size, n, w, cache.shape[0], heads, kv, dim, scale, 0)
    dev.awq.check(dev.lib.awq_paged_attention(ctypes.byref(a), DTYPES[dtype], dev.stream()))
    return dev.host(ctx)


def check_paged(got, dtype, vq, table, lengths, keys, values, spread, n_pages, scale):
    """A weight times its scale is rounded to binary16 (2^-11 of it), scores are sums in binary32 that lose some 2^-20 of their terms' size: weights
    are off by so much more.  The result is rounded once: by half a step of the type, relative or, in binary16 below 2^-14 where numbers are 2^-24
    apart, of 2^-25."""
    n, heads, dim = vq.shape
    for i in range(n):
        L = min(max(int(lengths[i]), 0), table.shape[1] * PAGE)
        at = table[i, np.arange(L) // PAGE]
        seen = (at >= 0) & (at < n_pages)
        at, p = np.where(seen, at, 0), np.arange(L) % PAGE
        k, v, s = (x[at, :, p] for x in (keys, values, spread))
        want, size = plain.attention(vq[i:i + 1], k, v, scale, seen[None], s)
        terms = (np.abs(vq[i]).sum(-1).max() * (np.abs(k[seen]).max() if seen.any() else 0.0)) * abs(scale)
        limit = EPS[dtype] / 2 * np.abs(want) + (2.0 ** -11 + terms * 2.0 ** -20 + 2.0 ** -18) * size + (2.0 ** -25 if dtype == "f16" else 1e-30)
        assert (np.abs(got[i] - want[0]) <= limit[0]).all(), (i, L, np.abs(got[i] - want[0]).max(), limit.max())


LENGTHS = [0, 1, 63, 64, 65, 130, 1000, 3000]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (16, 16, 64), (12, 4, 64), (8, 8, 128), (32, 8, 128), (20, 1, 128), (32, 2, 128), (8, 2, 256), (3, 1, 256),
                                          (40, 2, 256)])
def test_paged_attention(dev, dtype, heads, kv, dim):
    rng = rng_of(dtype, heads, kv, dim)
    lengths = LENGTHS
    width = 50
    table, n_pages = tables(rng, len(lengths), [pages(x) for x in lengths], width)
    print("paged", dtype, heads, kv, dim, flush=True)
    cache, k, v, spread = cache_of(dev, rng, n_pages, kv, dim)
    # what lies behind a request's last position and in pages that nobody has is not a number
    raw = cache.view(dev.torch.float16).reshape(n_pages, kv, 36 * dim)[:, :, 32 * dim:].reshape(n_pages, kv, 2, dim // 64, 2, PAGE)
    used = np.zeros((n_pages, PAGE), bool)
    for i, L in enumerate(lengths):
        used[table[i, np.arange(L) // PAGE], np.arange(L) % PAGE] = True
    raw.masked_fill_(~dev.torch.from_numpy(used).cuda()[:, None, None, None, None, :], float("nan"))
    x = rng.standard_normal((len(lengths), heads * dim + 16)) * 1.5
    x[5] *= 1e-3
    d_x, vx = dev.act(x, dtype)
    vq = vx[:, :heads * dim].reshape(-1, heads, dim)
    ctx = dev.full((len(lengths) + 1, heads * dim + 8), 9.0, dtype)
    got = paged(dev, dtype, d_x, cache, table, lengths, heads, kv, dim, dim ** -0.5, ctx)
    assert (got[-1] == 9.0).all() and (got[:, heads * dim:] == 9.0).all() and (got[0, :heads * dim] == 0.0).all()
    got = got[:-1, :heads * dim].reshape(-1, heads, dim)
    check_paged(got, dtype, vq, table, lengths, k, v, spread, n_pages, dim ** -0.5)
    # pages that are none, lengths that the table does not hold
    table = table.copy()
    table[4, 0], table[6, 3], table[7, 46], table[2, 0] = -1, n_pages, -5, 1 << 30
    lengths = [-3, 1, 63, 64, 65, 130, 1000, 3000]
    got = paged(dev, dtype, d_x, cache, table, lengths, heads, kv, dim, dim ** -0.5, dev.full((len(lengths), heads * dim), 9.0, dtype))
    assert (got[0] == 0.0).all() and (got[2] == 0.0).all()
    check_paged(got.reshape(-1, heads, dim), dtype, vq, table, lengths, k, v, spread, n_pages, dim ** -0.5)
    got = paged(dev, dtype, d_x, cache, table[:, :3].copy(), lengths, heads, kv, dim, dim ** -0.5, dev.full((len(lengths), heads * dim), 9.0, dtype))
    check_paged(got.reshape(-1, heads, dim), dtype, vq, table[:, :3], lengths, k, v, spread, n_pages, dim ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("size", [1e-5, 1e-2, 300.0])
@pytest.mark.parametrize("gain", [1e-3, 1.0, 30.0])
def test_paged_attention_of_small_and_large_values(dev, dtype, size, gain):
    """values near binary16's least and largest, flat weights and weights on one position"""
    heads, kv, dim, lengths = 4, 2, 128, [700, 2000, 64]
    rng = rng_of(dtype, size * 1e6, gain * 1e3)
    table, n_pages = tables(rng, 3, [pages(x) for x in lengths], 32)
    cache, k, v, spread = cache_of(dev, rng, n_pages, kv, dim, size)
    d_q, vq = dev.act(rng.standard_normal((3, heads * dim)) * min(gain / size, 8000.0), dtype)  # (binary16 ends at 65504)
    got = paged(dev, dtype, d_q, cache, table, lengths, heads, kv, dim, dim ** -0.5, dev.full((3, heads * dim), 9.0, dtype))
    check_paged(got.reshape(3, heads, dim), dtype, vq.reshape(3, heads, dim), table, lengths, k, v, spread, n_pages, dim ** -0.5)


@pytest.mark.parametrize("n", [65, 300, 2000])
def test_paged_attention_of_many_requests(dev, n):
    heads, kv, dim = 4, 2, 64
    rng = rng_of(n)
    lengths = rng.choice([0, 1, 5, 64, 100, 257], n)
    table, n_pages = tables(rng, n, [pages(x) for x in lengths], 5)
    cache, k, v, spread = cache_of(dev, rng, n_pages, kv, dim)
    d_q, vq = dev.act(rng.standard_normal((n, heads * dim)), "f16")
    got = paged(dev, "f16", d_q, cache, table, lengths, heads, kv, dim, 0.125, dev.full((n, heads * dim), 9.0, "f16"))
    check_paged(got.reshape(n, heads, dim), "f16", vq.reshape(n, heads, dim), table, lengths, k, v, spread, n_pages, 0.125)


def test_paged_attention_far_into_a_large_cache(dev):
    """pages behind the first 4 GiB"""
    heads, kv, dim, n_pages = 8, 8, 128, 66000
    rng = rng_of(1)
    lengths = [150, 70]
    small, k, v, spread = cache_of(dev, rng, 5, kv, dim)
    cache = dev.torch.empty((n_pages, kv, 72 * dim), dtype=dev.torch.uint8, device="cuda")
    table = np.array([[65999, 3, 65000], [58254, 65500, -1]])
    small_table = np.array([[0, 1, 2], [3, 4, -1]])
    for t, s in zip(table.ravel(), small_table.ravel()):
        if t >= 0:
            cache[int(t)] = small[int(s)]
    d_q, vq = dev.act(rng.standard_normal((2, heads * dim)), "f16")
    got = paged(dev, "f16", d_q, cache, table, lengths, heads, kv, dim, 0.1, dev.full((2, heads * dim), 9.0, "f16"))
    check_paged(got.reshape(2, heads, dim), "f16", vq.reshape(2, heads, dim), small_table, lengths, k, v, spread, 5, 0.1)
    # and rows of them, and an append there
    k_rows, _ = rows_of(dev, "f16", cache, table, None, lengths, [0, 150, 220], 220, kv, dim, pad=0)
    assert np.array_equal(k_rows[149], plain.nearest(k[2, :, 149 - 128], "f16").ravel())
    d_x, vx = dev.act(rng.standard_normal((1, kv * dim)), "f16")
    append(dev, "f16", None, d_x, d_x, None, None, dev.ints([150]), dev.ints([65000 * 64 + 22]), cache, heads, kv, dim, 0, False, None, None)
    k_rows, _ = rows_of(dev, "f16", cache, table, None, [151, 70], [0, 151, 221], 221, kv, dim, pad=0)
    assert np.array_equal(k_rows[150], plain.nearest(plain.value_of(*plain.quantised(vx.reshape(kv, dim))), "f16").ravel())


# --- attention of packed prompts ----------------------------------------------------------------------------------------------
def packed(dev, dtype, q, k, v, q_starts, k_starts, heads, kv, dim, causal, scale, ctx, n_tokens=None, n_keys=None):
    starts = [dev.ints(q_starts), None if k_starts is None else dev.ints(k_starts)]
    a = dev.awq.AwqPackedAttentionArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), ctx.data_ptr(), starts[0].data_ptr(),
                                       None if k_starts is None else starts[1].data_ptr(), q.stride(0), k.stride(0), v.stride(0), ctx.stride(0),
                                       q.shape[0] if n_tokens is None else n_tokens, k.shape[0] if n_keys is None else n_keys, len(q_starts) - 1, heads, kv, dim,
                                       int(causal), scale)
    dev.awq.check(dev.lib.awq_packed_attention(ctypes.byref(a), DTYPES[dtype], dev.stream()))
    return dev.host(ctx)


def check_packed(got, dtype, vq, vk, vv, q_starts, k_starts, causal, scale, fill=9.0):
    """A weight is rounded to the activations' type, and so is the sum that divides them: half a step of each, and of the result.  Scores are sums in
    binary32 that lose some 2^-20 of their terms' size."""
    known = np.zeros(len(got), bool)
    for a, b, c, d in zip(q_starts, q_starts[1:], k_starts, k_starts[1:]):
        nq, nk = b - a, d - c
        known[a:b] = True
        if nq == 0:
            continue
        i, j = np.arange(nq)[:, None], np.arange(nk)[None, :]
        seen = j <= i + nk - nq if causal else np.ones((nq, nk), bool)
        if nk == 0:
            assert (got[a:b] == 0.0).all()
            continue
        want, size = plain.attention(vq[a:b], vk[c:d], vv[c:d], scale, seen)
        assert (got[a:b][~seen.any(1)] == 0.0).all()
        terms = np.abs(vq[a:b]).sum(-1).max() * np.abs(vk[c:d]).max() * abs(scale)
        limit = EPS[dtype] / 2 * (2 * np.abs(want) + size) * 1.01 + (terms * 2.0 ** -20 + 2.0 ** -18) * size + 1e-30
        assert (np.abs(got[a:b] - want) <= limit).all(), (a, b, nk, np.abs(got[a:b] - want).max())
    assert (got[~known] == fill).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (6, 2, 64), (8, 8, 128), (8, 2, 128), (5, 1, 128), (4, 2, 256), (3, 1, 256)])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
def test_packed_attention(dev, dtype, heads, kv, dim, causal):
    rng = rng_of(dtype, heads, kv, dim, causal)
    new = [0, 1, 2, 31, 32, 33, 0, 63, 64, 65, 127, 128, 129, 300, 1]
    keys = [5, 1, 70, 31, 100, 33, 0, 20, 64, 400, 0, 128, 257, 300, 600]
    print("packed", dtype, heads, kv, dim, causal, flush=True)
    q_starts, k_starts = np.cumsum([3] + new), np.cumsum([2] + keys)
    n_q, n_k = int(q_starts[-1]) + 6, int(k_starts[-1]) + 4
    x, y = rng.standard_normal((n_q, heads * dim + 8)) * 1.3, rng.standard_normal((n_k, 2 * kv * dim + 16))
    y[:2], y[-4:] = np.nan, np.nan  # rows of nobody
    d_x, vx = dev.act(x, dtype)
    d_y, vy = dev.act(y, dtype)
    ctx = dev.full((n_q, heads * dim + 8), 9.0, dtype)
    got = packed(dev, dtype, d_x, d_y, d_y[:, kv * dim:], q_starts, k_starts, heads, kv, dim, causal, dim ** -0.5, ctx)
    assert (got[:, heads * dim:] == 9.0).all()
    vq = vx[:, :heads * dim].reshape(n_q, heads, dim)
    vk, vv = (vy[:, a:a + kv * dim].reshape(n_k, kv, dim) for a in (0, kv * dim))
    check_packed(got[:, :heads * dim].reshape(vq.shape), dtype, vq, vk, vv, q_starts, k_starts, causal, dim ** -0.5)
    # the queries' starts for the keys too
    got = packed(dev, dtype, d_x, d_y, d_y[:, kv * dim:], q_starts, None, heads, kv, dim, causal, 0.05, dev.full((n_q, heads * dim), 9.0, dtype))
    check_packed(got.reshape(vq.shape), dtype, vq, vk, vv, q_starts, q_starts, causal, 0.05)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_packed_attention_beside_what_is_not_finite(dev, dtype, dim):
    """keys and values of later positions that are not finite do not reach the queries ahead of them, and do reach those behind"""
    heads, kv, new = 2, 1, [150, 90, 40]
    rng = rng_of(dtype, dim)
    starts = np.cumsum([0] + new)
    n = int(starts[-1])
    d_q, vq = dev.act(rng.standard_normal((n, heads * dim)), dtype)
    k, v = rng.standard_normal((2, n, kv * dim))
    k[100, 3], k[200, 5] = np.nan, np.nan
    v[100, 7], v[60 + 150, 9], v[n - 1, 0] = np.inf, np.nan, -np.inf
    d_k, vk = dev.act(k, dtype)
    d_v, vv = dev.act(v, dtype)
    got = packed(dev, dtype, d_q, d_k, d_v, starts, None, heads, kv, dim, True, dim ** -0.5, dev.full((n, heads * dim), 9.0, dtype)).reshape(n, heads, dim)
    ahead = np.zeros(n, bool)
    ahead[:100] = ahead[150:200] = ahead[240:n - 1] = True
    assert np.isfinite(got[ahead]).all()
    assert np.isnan(got[100:150]).all() and np.isnan(got[200:240]).all() and (got[n - 1, :, 0] == -np.inf).all() and np.isfinite(got[n - 1, :, 1:]).all()
    for a, b in ((0, 100), (150, 200), (240, n - 1)):
        q_starts, k_starts = [0, b - a], [0, b - a]
        check_packed(got[a:b], dtype, vq[a:b].reshape(-1, heads, dim), vk[a:b].reshape(-1, kv, dim), vv[a:b].reshape(-1, kv, dim), q_starts, k_starts, True,
                     dim ** -0.5)


def test_packed_attention_of_scores_far_from_zero(dev):
    """scores of one sign, far beyond the range of an exponential, in bfloat16"""
    heads, kv, dim, n = 2, 1, 64, 200
    rng = rng_of(4)
    q = np.abs(rng.standard_normal((n, heads * dim))) * 1e18
    k = -np.abs(rng.standard_normal((n, kv * dim))) * 1e16
    v = rng.standard_normal((n, kv * dim))
    k[n // 2:] = k[n // 2 - 1]  # (equal scores: the weights are equal too)
    (d_q, vq), (d_k, vk), (d_v, vv) = (dev.act(x, "bf16") for x in (q, k, v))
    got = packed(dev, "bf16", d_q, d_k, d_v, [0, n], None, heads, kv, dim, True, 0.125, dev.full((n, heads * dim), 9.0, "bf16")).reshape(n, heads, dim)
    assert np.isfinite(got).all()
    assert np.abs(got[0] - vv[0].reshape(kv, dim)).max() <= 2.0 ** -8 * np.abs(vv[0]).max()


@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales_that_do_not_favour_the_largest_product(dev, scale):
    """0: all keys seen weigh the same; below 0: the least products the most"""
    heads, kv, dim, new = 4, 2, 128, [70, 140]
    rng = rng_of(6)
    starts = np.cumsum([0] + new)
    (d_q, vq), (d_k, vk), (d_v, vv) = (dev.act(rng.standard_normal((210, h * dim)), "f16") for h in (heads, kv, kv))
    got = packed(dev, "f16", d_q, d_k, d_v, starts, None, heads, kv, dim, True, scale, dev.full((210, heads * dim), 9.0, "f16"))
    shape = lambda x: x.reshape(210, -1, dim)  # noqa: E731
    check_packed(shape(got), "f16", shape(vq), shape(vk), shape(vv), starts, starts, True, scale)
    table, n_pages = tables(rng, 2, [2, 3], 4)
    cache, k, v, spread = cache_of(dev, rng, n_pages, kv, dim)
    got = paged(dev, "f16", d_q[:2], cache, table, [70, 140], heads, kv, dim, scale, dev.full((2, heads * dim), 9.0, "f16"))
    check_paged(got.reshape(2, heads, dim), "f16", shape(vq)[:2], table, [70, 140], k, v, spread, n_pages, scale)


@pytest.mark.parametrize("n", [70, 500])
def test_packed_attention_of_many_requests(dev, n):
    heads, kv, dim = 2, 1, 64
    rng = rng_of(n)
    new = rng.choice([0, 1, 2, 7, 130], n)
    starts = np.cumsum([0] + list(new))
    T = int(starts[-1])
    (d_q, vq), (d_k, vk), (d_v, vv) = (dev.act(rng.standard_normal((T, h * dim)), "bf16") for h in (heads, kv, kv))
    got = packed(dev, "bf16", d_q, d_k, d_v, starts, None, heads, kv, dim, True, 0.125, dev.full((T, heads * dim), 9.0, "bf16"))
    check_packed(got.reshape(T, heads, dim), "bf16", vq.reshape(T, heads, dim), vk.reshape(T, kv, dim), vv.reshape(T, kv, dim), starts, starts, True, 0.125)


# --- sampling -------------------------------------------------------------------------------------------------------------------
def sample(dev, dtype, x, u, temperature=None, top_k=None, top_p=None, min_p=None, vocab=None, ws=None):
    n, V = x.shape[0], x.shape[1] if vocab is None else vocab
    ids = dev.full((n + 1,), -7, dev.torch.int32)
    size = dev.lib.awq_sample_workspace_bytes(n, V)
    ws = dev.full((size // 4 + 1,), float("nan"), "f32") if ws is None else ws
    keep = [dev.floats(t) if t is not None else None for t in (temperature, top_p, min_p, u)] + [None if top_k is None else dev.ints(top_k)]
    at = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    a = dev.awq.AwqSampleArgs(x.data_ptr(), at(keep[0]), at(keep[4]), at(keep[1]), at(keep[2]), at(keep[3]), ids.data_ptr(), ws.data_ptr(), x.stride(0), V, n, size)
    dev.awq.check(dev.lib.awq_sample(ctypes.byref(a), DTYPES[dtype], dev.stream()))
    got = dev.host(ids)
    assert got[n] == -7
    return got[:n].tolist()


def check_sample(dev, dtype, vx, got, u, temperature, top_k, top_p, min_p):
    f = lambda v, i, other: other if v is None else float(np.float32(v[i]))  # noqa: E731
    want = [plain.sample(vx[i], f(temperature, i, 1.0), 0 if top_k is None else int(top_k[i]), f(top_p, i, 1.0), f(min_p, i, 0.0), f(u, i, 0.0))
            for i in range(len(got))]
    assert got == want


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 500, 8191, 8192, 8193, 32771, 151936])
@pytest.mark.parametrize("spread", [0.3, 2.0, 8.0])
def test_sample(dev, dtype, vocab, spread):
    n = 24
    rng = rng_of(dtype, vocab, spread * 10)
    print("sample", dtype, vocab, spread, flush=True)
    x = spread * rng.standard_normal((n, vocab + 3))
    x[3, : vocab // 2] = -np.inf
    x[4, vocab // 3] = np.nan
    d_x, vx = dev.act(x, dtype)
    vx = vx[:, :vocab]
    u = rng.random(n).astype(np.float32)
    u[:3] = 0.0, 1.0 - 2.0 ** -24, 0.5
    of = lambda *v: [v[i % len(v)] for i in range(n)]  # noqa: E731
    temperature, top_k, top_p, min_p = of(0.0, 0.7, 1.0, 1.5, 0.01), of(0, 1, 5, 50, 1000, 100000, -2), of(1.0, 0.9, 0.3, 0.999), of(0.0, 0.0, 0.05, 0.5, 1.0)
    for t, k, p, m in ((None, None, None, None), (temperature, None, None, None), (temperature, top_k, None, None), (temperature, None, top_p, None),
                       (temperature, None, None, min_p), (temperature, top_k, top_p, min_p), (of(1.3), None, of(0.95), of(0.001)), (of(0.8), of(40), of(0.9), None)):
        check_sample(dev, dtype, vx, sample(dev, dtype, d_x, u, t, k, p, m, vocab), u, t, k, p, m)


def test_sample_among_equals(dev):
    """rows of equal logits and of few different ones: ties go to the lowest ids, whatever their number"""
    rng = rng_of(5)
    V, n = 20011, 12
    x = rng.integers(0, 3, (n, V)).astype(np.float64)
    x[:3] = 1.5
    x[3, 100:] = -3.0
    x[4] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    d_x, vx = dev.act(x, "f32")
    u = rng.random(n).astype(np.float32)
    of = lambda *v: [v[i % len(v)] for i in range(n)]  # noqa: E731
    for k, p, m in ((of(10, 9000, 15000, 50), None, None), (None, of(0.5, 0.01, 0.9), None), (of(12000, 700), of(0.7, 0.2, 0.95), None), (None, None, of(1.0, 0.3)),
                    (None, None, None)):
        check_sample(dev, "f32", vx, sample(dev, "f32", d_x, u, None, k, p, m), u, None, k, p, m)


def test_sample_rows_without_a_choice(dev):
    inf, V = np.inf, 9001
    x = np.full((10, V), -1.0)
    x[0], x[1] = -inf, np.nan
    x[2, [70, 8500]] = inf
    x[3, 8999] = inf
    x[4] = -3.4e38                 # a mask's lowest value throughout, and everywhere but at one place
    x[5], x[5, 4000] = -3.4e38, 2.0
    x[6], x[6, [5, 6000]] = -inf, -5.0
    x[7, 17] = 3e38
    x[8] = -1e30
    x[9, :] = 60000.0
    d_x, vx = dev.act(x, "f32")
    u = np.full(10, 0.75, np.float32)
    for t, k, p, m in ((None, None, None, None), ([0.0] * 10, None, None, None), ([1.0] * 10, [5] * 10, [0.9] * 10, [0.1] * 10), ([float("nan")] * 10, None, None, None),
                       ([2.0 ** -20] * 10, None, [0.5] * 10, None), ([1.0] * 10, None, [0.0] * 10, None), ([1.0] * 10, [0] * 10, [float("nan")] * 10, [float("nan")] * 10),
                       ([1e-3] * 10, [7] * 10, None, [2.0] * 10)):
        got = sample(dev, "f32", d_x, u, t, k, p, m)
        m = None if m is None or m[0] != m[0] else m
        p = None if p is None or p[0] != p[0] else p
        check_sample(dev, "f32", vx, got, u, t, k, p, m)


def test_sample_follows_the_weights(dev):
    """every token of a short row comes as often as uniform numbers at even distances say"""
    x, n = np.array([0.1, -2.0, 1.3, -np.inf, 0.7]), 4096
    d_x, vx = dev.act(np.repeat(x[None], n, 0), "f32")
    u = (np.arange(n) + 0.5) / n
    got = np.bincount(sample(dev, "f32", d_x, u, [0.7] * n), minlength=5)
    w = np.exp(vx[0] / np.float64(np.float32(0.7)))
    assert np.abs(got / n - w / w.sum()).max() <= 1.0 / n


# --- together --------------------------------------------------------------------------------------------------------------------
class Server:
    """A batch of requests of one layer: queries, keys and values of a token are rows of tables, its logits the attention's result."""

    def __init__(self, dev, dtype, heads=4, kv=2, dim=64, vocab=97, n_pages=60, width=8, seed=3):
        rng = np.random.default_rng(seed)
        self.dev, self.dtype, self.heads, self.kv, self.dim, self.vocab, self.n_pages, self.width = dev, dtype, heads, kv, dim, vocab, n_pages, width
        self.rows, self.v_rows = dev.act(rng.standard_normal((vocab, (heads + 2 * kv) * dim)), dtype)
        self.head, self.v_head = dev.act(rng.standard_normal((vocab, heads * dim)) * 0.3, dtype)
        angle = np.arange(width * PAGE)[:, None] * 100.0 ** (-np.arange(dim // 4) * 4.0 / dim)
        self.cos, self.sin = dev.floats(np.cos(angle)), dev.floats(np.sin(angle))
        self.cache = dev.torch.zeros((n_pages, kv, 72 * dim), dtype=dev.torch.uint8, device="cuda")
        self.free, self.count = dev.ints(rng.permutation(n_pages)), dev.ints([n_pages])

    def start(self, n):
        dev = self.dev
        self.n, self.table = n, dev.full((n, self.width), -1, dev.torch.int32)
        self.lengths = dev.ints([0] * n)
        self.cached = dev.ints([0] * n)
        self.ids = dev.ints([0] * n)
        self.ws = dev.full((max(dev.lib.awq_paged_workspace_bytes(n, self.heads, self.kv, self.dim, self.width),
                                dev.lib.awq_sample_workspace_bytes(n, self.vocab)) // 4,), float("nan"), "f32")
        self.starts, self.keys = dev.ints([0] * (n + 1)), dev.ints([0] * (n + 1))

    def step(self, tokens, fresh, prompt, u, max_tokens):
        """one pass; `tokens`, `fresh` and u on the device.  Logits, and the sampled ids in self.ids"""
        dev, T, D = self.dev, max_tokens, self.dim
        self.cached.copy_(self.lengths)
        positions, slots = dev.full((T,), 0, dev.torch.int32), dev.full((T,), 0, dev.torch.int32)
        a = dev.awq.AwqPagePlanArgs(self.cached.data_ptr(), fresh.data_ptr(), self.table.data_ptr(), self.free.data_ptr(), self.count.data_ptr(),
                                    self.count.data_ptr(), self.lengths.data_ptr(), self.starts.data_ptr(), self.keys.data_ptr(), positions.data_ptr(),
                                    slots.data_ptr(), None, T, self.n, self.width, self.n_pages, 0)
        dev.awq.check(dev.lib.awq_page_plan(ctypes.byref(a), dev.stream()))
        x = self.rows[tokens.long()]
        q, k, v = x[:, :self.heads * D], x[:, self.heads * D:(self.heads + self.kv) * D], x[:, (self.heads + self.kv) * D:]
        append(dev, self.dtype, q, k, v, self.cos, self.sin, positions, slots, self.cache, self.heads, self.kv, D, D // 2, False, q, k)
        ctx = dev.full((T, self.heads * D), 0.0, self.dtype)
        if prompt:
            n_rows = self.n * self.width * PAGE
            kv_rows = dev.full((n_rows, 2 * self.kv * D), 0.0, self.dtype)
            b = dev.awq.AwqPagedRowsArgs(self.cache.data_ptr(), self.table.data_ptr(), None, self.lengths.data_ptr(), self.keys.data_ptr(), kv_rows.data_ptr(),
                                         kv_rows.data_ptr() + 2 * self.kv * D, kv_rows.stride(0), kv_rows.stride(0), n_rows, self.n, self.width, self.n_pages,
                                         self.kv, D, 0)
            dev.awq.check(dev.lib.awq_paged_rows(ctypes.byref(b), DTYPES[self.dtype], dev.stream()))
            c = dev.awq.AwqPackedAttentionArgs(q.data_ptr(), kv_rows.data_ptr(), kv_rows.data_ptr() + 2 * self.kv * D, ctx.data_ptr(), self.starts.data_ptr(),
                                               self.keys.data_ptr(), q.stride(0), kv_rows.stride(0), kv_rows.stride(0), ctx.stride(0), T, n_rows, self.n, self.heads,
                                               self.kv, D, 1, D ** -0.5)
            dev.awq.check(dev.lib.awq_packed_attention(ctypes.byref(c), DTYPES[self.dtype], dev.stream()))
            last = ctx[(self.starts[1:].long() - 1).clamp(min=0)]
        else:
            d = dev.awq.AwqPagedAttentionArgs(q.data_ptr(), self.cache.data_ptr(), self.table.data_ptr(), self.lengths.data_ptr(), ctx.data_ptr(),
                                              self.ws.data_ptr(), q.stride(0), ctx.stride(0), self.ws.numel() * 4, self.n, self.width, self.n_pages, self.heads,
                                              self.kv, D, D ** -0.5, 0)
            dev.awq.check(dev.lib.awq_paged_attention(ctypes.byref(d), DTYPES[self.dtype], dev.stream()))
            last = ctx
        logits = (last.float()[:, None, :] * self.head.float()[None]).sum(-1)
        e = dev.awq.AwqSampleArgs(logits.data_ptr(), None, None, None, None, u.data_ptr(), self.ids.data_ptr(), self.ws.data_ptr(), self.vocab, self.vocab, self.n,
                                  self.ws.numel() * 4)
        dev.awq.check(dev.lib.awq_sample(ctypes.byref(e), DTYPES["f32"], dev.stream()))
        return logits

    def plain_logits(self, ids):
        """logits behind a request's tokens, in 64 bits: keys and values as the cache holds them"""
        D, n = self.dim, len(ids)
        x = self.v_rows[ids].reshape(n, -1, D)
        cos, sin = (self.dev.host(t).astype(np.float64)[:n] for t in (self.cos, self.sin))
        q = plain.nearest(plain.turned(x[:, :self.heads], cos, sin, D // 2, False), self.dtype)
        k = plain.nearest(plain.turned(x[:, self.heads:self.heads + self.kv], cos, sin, D // 2, False), self.dtype)
        k, v = (plain.value_of(*plain.quantised(y)) for y in (k, x[:, self.heads + self.kv:]))
        ctx, _ = plain.attention(q[-1:], k, v, D ** -0.5, np.ones((1, n), bool))
        return ctx.reshape(-1) @ self.v_head.T


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_batch_from_prompts_to_answers(dev, dtype):
    """prompts in two parts, then single tokens, the requests of different lengths; pages run from the list and back to it"""
    rng = rng_of(dtype, "batch")
    s, torch = Server(dev, dtype), dev.torch
    s.start(4)
    texts = [rng.integers(0, s.vocab, n).tolist() for n in (5, 150, 64, 90)]
    cuts = [3, 100, 64, 1]
    ids = [[], [], [], []]
    for part in range(2):
        pieces = [t[:c] if part == 0 else t[c:] for t, c in zip(texts, cuts)]
        tokens = sum(pieces, [])
        logits = s.step(dev.ints(tokens + [0] * 7), dev.ints([len(p) for p in pieces]), True, dev.floats(rng.random(4)), len(tokens) + 7)
        ids = [i + p for i, p in zip(ids, pieces)]
    got, drawn = dev.host(logits), dev.host(s.ids)
    # (a request without new positions has no logits in a pass)
    fresh = [len(t) > c for t, c in zip(texts, cuts)]
    # rounded: keys and values out of the cache (once), weights and the result; 0.3 of 256 products of numbers of size 1
    limit = {"f16": 0.02, "bf16": 0.15}[dtype]
    for i in range(4):
        if fresh[i]:
            assert np.abs(got[i] - s.plain_logits(ids[i])).max() < limit
    for _ in range(70):
        drawn = dev.host(s.ids).tolist()
        ids = [i + [t] for i, t in zip(ids, drawn)]
        logits = s.step(dev.ints(drawn), dev.ints([1] * 4), False, dev.floats(rng.random(4)), 4)
    got = dev.host(logits)
    for i in range(4):
        assert np.abs(got[i] - s.plain_logits(ids[i])).max() < limit
    assert dev.host(s.lengths).tolist() == [len(i) for i in ids]
    held = sum(pages(len(i)) for i in ids)
    assert int(dev.host(s.count)[0]) == s.n_pages - held
    # all end: every page is back, once
    s.cached.copy_(s.lengths)
    s.step(dev.ints([0] * 4), dev.ints([-1] * 4), False, dev.floats([0.5] * 4), 4)
    torch.cuda.synchronize()
    assert int(dev.host(s.count)[0]) == s.n_pages and sorted(dev.host(s.free).tolist()) == list(range(s.n_pages))


def test_a_captured_step(dev):
    """a decode step as a graph, replayed with the host's own work and waits in between: the ids of the same steps run one by one"""
    torch = dev.torch
    runs = []
    for captured in (False, True):
        rng = rng_of(11)
        s = Server(dev, "f16")
        s.start(3)
        texts = [rng.integers(0, s.vocab, n).tolist() for n in (60, 7, 126)]
        s.step(dev.ints(sum(texts, [])), dev.ints([len(t) for t in texts]), True, dev.floats(rng.random(3)), sum(map(len, texts)))
        u, fresh, tokens, got = dev.floats([0.0] * 3), dev.ints([1] * 3), s.ids.clone(), []
        graph = None
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            saved = [t.clone() for t in (s.lengths, s.count, s.table, s.ids, s.cache)]
            with torch.cuda.stream(side):  # (once ahead of the capture, as torch's own calls need it)
                s.step(tokens, fresh, False, u, 3)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            for t, was in zip((s.lengths, s.count, s.table, s.ids, s.cache), saved):
                t.copy_(was)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                s.step(tokens, fresh, False, u, 3)
        for _ in range(12):
            u.copy_(dev.floats(rng.random(3)))
            tokens.copy_(s.ids)
            if graph is not None:
                graph.replay()
            else:
                s.step(tokens, fresh, False, u, 3)
            got.append(dev.host(s.ids).tolist())
            (torch.ones(1000, device="cuda") * 2).sum().item()
        runs.append((got, dev.host(s.lengths).tolist(), dev.host(s.cache).tobytes()))
    assert runs[0] == runs[1]


def test_calls_on_streams_of_their_own(dev):
    """two attentions and two samplings side by side, each with a workspace of its own, give what they give one after the other"""
    torch, heads, kv, dim = dev.torch, 8, 2, 128
    rng = rng_of(12)
    lengths = [3000, 10, 700]
    table, n_pages = tables(rng, 3, [pages(x) for x in lengths], 50)
    cache, *_ = cache_of(dev, rng, n_pages, kv, dim)
    q = [dev.act(rng.standard_normal((3, heads * dim)), "bf16")[0] for _ in range(2)]
    x = [dev.act(3 * rng.standard_normal((8, 50021)), "f16")[0] for _ in range(2)]
    u = rng.random(8)
    alone = [(paged(dev, "bf16", a, cache, table, lengths, heads, kv, dim, 0.1, dev.full((3, heads * dim), 9.0, "bf16")), sample(dev, "f16", b, u, top_p=[0.9] * 8))
             for a, b in zip(q, x)]
    n, w = table.shape
    size, more = dev.lib.awq_paged_workspace_bytes(n, heads, kv, dim, w), dev.lib.awq_sample_workspace_bytes(8, 50021)
    d_table, d_lengths, d_u, d_p = dev.ints(table), dev.ints(lengths), dev.floats(u), dev.floats([0.9] * 8)
    outs = [(dev.full((3, heads * dim), 9.0, "bf16"), dev.full((8,), -7, torch.int32), dev.full((size // 4,), 0.0, "f32"), dev.full((more // 4 + 1,), 0.0, "f32"))
            for _ in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for st, a, b, (ctx, ids, ws, ws2) in zip(streams, q, x, outs):
            args = dev.awq.AwqPagedAttentionArgs(a.data_ptr(), cache.data_ptr(), d_table.data_ptr(), d_lengths.data_ptr(), ctx.data_ptr(), ws.data_ptr(),
                                                 a.stride(0), ctx.stride(0), size, n, w, n_pages, heads, kv, dim, 0.1, 0)
            dev.awq.check(dev.lib.awq_paged_attention(ctypes.byref(args), 1, ctypes.c_void_p(st.cuda_stream)))
            args = dev.awq.AwqSampleArgs(b.data_ptr(), None, None, d_p.data_ptr(), None, d_u.data_ptr(), ids.data_ptr(), ws2.data_ptr(), 50021, 50021, 8, more)
            dev.awq.check(dev.lib.awq_sample(ctypes.byref(args), 3, ctypes.c_void_p(st.cuda_stream)))
    for (ctx, ids, _, _), (want, want_ids) in zip(outs, alone):
        assert np.array_equal(dev.host(ctx), want) and dev.host(ids).tolist() == want_ids


def test_captured_parts_of_prompts(dev):
    """passes of three requests with 5, 1 and 30 new positions each, behind what they have, as a graph that is replayed: the ids of the same passes
    run one by one"""
    torch, new = dev.torch, [5, 1, 30]
    runs = []
    for captured in (False, True):
        rng = rng_of(13)
        s = Server(dev, "bf16")
        s.start(3)
        u, fresh, tokens, got = dev.floats([0.0] * 3), dev.ints(new), dev.ints([0] * 40), []
        state = (s.lengths, s.count, s.table, s.ids, s.cache)
        graph = None
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            saved = [t.clone() for t in state]
            with torch.cuda.stream(side):
                s.step(tokens, fresh, True, u, 40)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            for t, was in zip(state, saved):
                t.copy_(was)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                s.step(tokens, fresh, True, u, 40)
        for _ in range(6):
            u.copy_(dev.floats(rng.random(3)))
            tokens.copy_(dev.ints(rng.integers(0, s.vocab, 40)))
            if graph is not None:
                graph.replay()
            else:
                s.step(tokens, fresh, True, u, 40)
            got.append(dev.host(s.ids).tolist())
            (torch.ones(1000, device="cuda") * 2).sum().item()
        runs.append((got, dev.host(s.lengths).tolist(), dev.host(s.cache).tobytes()))
    assert runs[0][1] == [30, 6, 180] and runs[0] == runs[1]


def test_packed_attention_of_rows_far_apart(dev):
    """strides with which rows lie further than 2^32 bytes from the first"""
    heads, kv, dim, new = 2, 1, 128, [100, 64]
    rng, n, ld = rng_of(14), 164, (1 << 24) + 8
    print("rows far apart", flush=True)
    x = dev.torch.empty((n, ld), dtype=dev.torch.float16, device="cuda")
    d_y, vy = dev.act(rng.standard_normal((n, (heads + 2 * kv) * dim)), "f16")
    x[:, :d_y.shape[1]] = d_y
    ctx = x[:, 1024:1024 + heads * dim]
    ctx.fill_(9.0)
    starts = np.cumsum([0] + new)
    got = packed(dev, "f16", x, x[:, heads * dim:], x[:, (heads + kv) * dim:], starts, None, heads, kv, dim, True, dim ** -0.5, ctx)
    parts = [vy[:, a * dim:b * dim].reshape(n, b - a, dim) for a, b in ((0, heads), (heads, heads + kv), (heads + kv, heads + 2 * kv))]
    check_packed(got.reshape(n, heads, dim), "f16", *parts, starts, starts, True, dim ** -0.5)


def test_sample_of_the_largest_vocabulary_and_of_rows_far_apart(dev):
    V, n = 524288, 3
    rng, ld = rng_of(15), (1 << 30) + 8
    print("largest vocabulary", flush=True)
    d_x, vx = dev.act(2.0 * rng.standard_normal((n, V)), "f16")
    x = dev.torch.empty((n, ld), dtype=dev.torch.float16, device="cuda")
    x[:, :V] = d_x
    u = rng.random(n).astype(np.float32)
    for t, k, p, m in ((None, None, None, None), ([0.0] * n, None, None, None), ([0.7, 1.0, 1.4], [50, 4000, 300000], None, None), ([1.0, 0.5, 1.3], None, [0.9, 0.99, 0.95], None),
                       (None, [400] * n, [0.9] * n, [0.02] * n)):
        check_sample(dev, "f16", vx, sample(dev, "f16", x, u, t, k, p, m, V), u, t, k, p, m)
