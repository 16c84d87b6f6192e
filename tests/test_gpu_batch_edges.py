"""Several requests at once: what lies at the edges of the operators' definitions, against batch_plain.py's 64 bits."""
import ctypes

import numpy as np
import pytest

import batch_plain as plain
from test_gpu_batch import append, cache_of, check_paged, check_plan, check_sample, dev, packed, paged, rng_of, rows_of, run_plan, sample, tables  # noqa: F401

pytestmark = pytest.mark.gpu


# --- pages and slots ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,width", [(1, 3), (6, 9), (40, 70), (300, 20), (1500, 5)])
@pytest.mark.parametrize("plenty", [True, False], ids=["plenty", "short"])
def test_plan_of_ended_requests_with_entries_that_are_no_pages(dev, n, width, plenty):
    """what is no page does not go on the list, and nobody is given it"""
    rng = rng_of("holes", n, plenty)
    cached = rng.integers(0, 64 * width + 1, n)
    fresh = rng.choice([-1, -1, 0, 1, 70], n)
    fresh[0] = -1
    table, n_pages = tables(rng, n, [plain.pages(c) for c in cached], width, 3 if n == 1 else 5 * n)
    spare = np.setdiff1d(np.arange(n_pages), table)[: None if plenty else 1].tolist()
    holes = rng.random(table.shape) < 0.2
    table[holes] = rng.choice([-1, n_pages, -2 ** 31, 2 ** 31 - 1], holes.sum())
    if n == 1:
        table[0, 0] = -1
    print("plan, holes", n, width, plenty, flush=True)
    ended = fresh < 0
    back = [p for i in np.flatnonzero(ended) for p in table[i, :plain.pages(cached[i])] if 0 <= p < n_pages]
    total = int(np.maximum(fresh, 0).sum())
    for max_tokens in (total, total + 5000):  # one launch and two
        want = plain.plan(np.where(ended, 0, cached), np.where(ended, 0, fresh), table, spare + back, n_pages, max_tokens)
        check_plan(run_plan(dev, cached, fresh, table, spare, n_pages, max_tokens), want, len(spare))

@pytest.mark.parametrize("n", [5, 300, 1500])
@pytest.mark.parametrize("more", [0, 5000])
def test_plan_with_the_lengths_in_the_place_of_those_before(dev, n, more):
    """one buffer of lengths, step after step: in one launch and in two"""
    rng = rng_of("in place", n, more)
    width = 12
    print("plan, in place", n, more, flush=True)
    lengths = rng.integers(0, 64 * width - 100, n)
    table, n_pages = tables(rng, n, [plain.pages(c) for c in lengths], width, 4 * n)
    spare = np.setdiff1d(np.arange(n_pages), table).tolist()
    d = {name: dev.ints(x) for name, x in (("table", table), ("free", spare + [-7] * (n_pages - len(spare))), ("count", [len(spare)]), ("lengths", lengths))}
    for _ in range(3):
        fresh = rng.choice([-1, 0, 1, 1, 65, 200], n)
        total = int(np.maximum(fresh, 0).sum())
        T = total + more
        stack = dev.host(d["free"])[:int(dev.host(d["count"])[0])].tolist()
        want = plain.plan(dev.host(d["lengths"]), fresh, dev.host(d["table"]), stack, n_pages, T)
        d_fresh, starts, keys, positions, slots, left = dev.ints(fresh), *(dev.full((m,), -7, dev.torch.int32) for m in (n + 1, n + 1, T + 1, T + 1, 1))
        a = dev.awq.AwqPagePlanArgs(d["lengths"].data_ptr(), d_fresh.data_ptr(), d["table"].data_ptr(), d["free"].data_ptr(), d["count"].data_ptr(),
                                    d["count"].data_ptr(), d["lengths"].data_ptr(), starts.data_ptr(), keys.data_ptr(), positions.data_ptr(), slots.data_ptr(),
                                    left.data_ptr(), T, n, width, n_pages, 0)
        dev.awq.check(dev.lib.awq_page_plan(ctypes.byref(a), dev.stream()))
        h = dev.host
        assert h(d["lengths"]).tolist() == want[3] and h(starts).tolist() == want[4] and h(keys).tolist() == want[5] and int(h(left)[0]) == want[8]
        assert np.array_equal(h(d["table"]), want[0]) and int(h(d["count"])[0]) == want[2]
        assert h(positions)[:T].tolist() == want[6] and h(slots)[:T].tolist() == want[7] and h(positions)[T] == h(slots)[T] == -7


# --- append and rows ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("written", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_at_the_end_of_binary16_stay_finite(dev, written, dim):
    """groups that span all of binary16, whose fifteenth step lies beyond it: its largest number, for the rows and for the attention"""
    kv, T = 2, 20
    rng = rng_of("end", written, dim)
    x = rng.choice([-65504.0, 65504.0, 0.0, 3.0], (T, kv * dim))
    x[:4, 0], x[:4, 1] = -65504.0, 65504.0
    x[4] = 65504.0
    x[5], x[5, ::64] = -65504.0, 65504.0
    x[6, ::64] = np.nan
    if written == "bf16":
        x[7] = rng.choice([-1e30, 1e30], kv * dim)
    d_x, vx = dev.act(x, written)
    cache = dev.torch.zeros((1, kv, 72 * dim), dtype=dev.torch.uint8, device="cuda")
    append(dev, written, None, d_x, d_x, None, None, dev.ints(range(T)), dev.ints(range(T)), cache, 1, kv, dim, 0, False, None, None)
    with np.errstate(invalid="ignore"):
        values = plain.value_of(*plain.quantised(vx.reshape(T, kv, dim)))
    assert np.abs(values[[0, 1, 2, 3, 5]]).max() > 65520.0
    for dtype in ("f16", "bf16"):
        want = plain.nearest(np.clip(values, -65504.0, 65504.0) if dtype == "f16" else values, dtype).reshape(T, -1)
        for g in rows_of(dev, dtype, cache, np.array([[0]]), None, [T], [0, T], T, kv, dim, pad=0):
            assert np.array_equal(np.isnan(g), np.isnan(want)) and np.array_equal(g[~np.isnan(g)], want[~np.isnan(want)])
    # one position a request is the attention's result as it is; 3 requests, and one after the other
    order = [0, 3, 5]
    pages = dev.torch.cat([cache[:, :, :]] * T)
    for i in range(T):  # position i first in page i
        data, par = (t[i].view(kv, -1, 64, w) for t, w in ((pages[:, :, :64 * dim], dim // 2), (pages[:, :, 64 * dim:], 2)))
        first = data[:, :, i].clone(), par[:, :, i].clone()
        pages[i, :, :64 * dim].view(kv, 2, 64, dim // 2)[:, :, 0] = first[0]
        pages[i, :, 64 * dim:].view(kv, -1, 64, 2)[:, :, 0] = first[1]
    d_q, _ = dev.act(np.zeros((3, kv * dim)), "f16")
    got = paged(dev, "f16", d_q, pages, np.array(order)[:, None], [1, 1, 1], kv, kv, dim, 0.1, dev.full((3, kv * dim), 9.0, "f16"))
    want = np.clip(values[order], -65504.0, 65504.0).reshape(3, -1)
    size = np.abs(values[order]).reshape(3, -1)
    assert np.isfinite(got).all()
    # a value's product and offset are rounded to 2^-11 of them, the result once more
    assert (np.abs(got - want) <= 2.0 ** -11 * (np.abs(want) + 131008.0 + size)).all()


# --- attention over pages ---------------------------------------------------------------------------------------------------
def cache_of_scales(dev, rng, n_pages, kv, dim, v_scales, k_signs=False):
    """a random cache with values of these scales [pages][heads][64][dim / 64]: (tensor, keys, values, the size of the values' parts)"""
    shape = (n_pages, kv, 64, dim)
    n = [rng.integers(0, 16, shape).astype(np.float64) for _ in range(2)]
    s = [plain.nearest(x, "f16") for x in (0.2 * (rng.choice([-1.0, 1.0], v_scales.shape) if k_signs else np.ones(v_scales.shape)), v_scales)]
    z = [plain.nearest(x * (-7.5 + rng.standard_normal(x.shape)), "f16") for x in s]
    cache = dev.torch.from_numpy(plain.packed_pages(*zip(n, s, z))).cuda()
    return cache, plain.value_of(n[0], s[0], z[0]), plain.value_of(n[1], s[1], z[1]), plain.value_of(n[1], np.abs(s[1]), np.abs(z[1]))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (12, 2, 128), (16, 1, 128), (8, 2, 256), (16, 1, 256)])
@pytest.mark.parametrize("gain", [0.3, 6.0])
@pytest.mark.parametrize("kind", ["keys", "groups", "both", "pages", "none"])
def test_paged_attention_of_scales_far_apart(dev, dtype, heads, kv, dim, gain, kind):
    """scales of values that differ by up to 2^20 between keys, between groups, between both or from page to page, and groups without any: the tolerance is
    that of even ones, which counts what each key weighs"""
    lengths = [700, 1300, 64, 3]
    rng = rng_of("far", dtype, heads, dim, gain * 10, kind)
    print("paged, scales", dtype, heads, kv, dim, gain, kind, flush=True)
    table, n_pages = tables(rng, 4, [plain.pages(x) for x in lengths], 21)
    shape = (n_pages, kv, 64, dim // 64)
    cut = {"keys": (n_pages, kv, 64, 1), "groups": (1, kv, 1, dim // 64), "both": shape, "pages": (n_pages, 1, 1, 1), "none": (n_pages, kv, 64, 1)}[kind]
    scales = np.broadcast_to(2.0 ** rng.uniform(-12, 8, cut), shape).copy()
    if kind == "none":
        scales[..., 0] = 0.0
        scales[:, :, 5:9] = 0.0
    cache, k, v, spread = cache_of_scales(dev, rng, n_pages, kv, dim, scales)
    d_q, vq = dev.act(rng.standard_normal((4, heads * dim)) * gain, dtype)
    got = paged(dev, dtype, d_q, cache, table, lengths, heads, kv, dim, dim ** -0.5, dev.full((4, heads * dim), 9.0, dtype))
    check_paged(got.reshape(4, heads, dim), dtype, vq.reshape(4, heads, dim), table, lengths, k, v, spread, n_pages, dim ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (12, 2, 128), (16, 1, 256)])
@pytest.mark.parametrize("size", [1e-4, 1.0, 500.0])
@pytest.mark.parametrize("mixed", [True, False], ids=["mixed", "negative"])
def test_paged_attention_of_scales_below_zero(dev, dtype, heads, kv, dim, size, mixed):
    lengths = [700, 64, 129]
    rng = rng_of("below", dtype, heads, dim, size * 1e4, mixed)
    print("paged, below zero", dtype, heads, kv, dim, size, mixed, flush=True)
    table, n_pages = tables(rng, 3, [plain.pages(x) for x in lengths], 11)
    shape = (n_pages, kv, 64, dim // 64)
    scales = size * np.exp(0.5 * rng.standard_normal(shape)) * (rng.choice([-1.0, 1.0], shape) if mixed else -1.0)
    cache, k, v, spread = cache_of_scales(dev, rng, n_pages, kv, dim, scales, k_signs=True)
    d_q, vq = dev.act(rng.standard_normal((3, heads * dim)), dtype)
    got = paged(dev, dtype, d_q, cache, table, lengths, heads, kv, dim, dim ** -0.5, dev.full((3, heads * dim), 9.0, dtype))
    check_paged(got.reshape(3, heads, dim), dtype, vq.reshape(3, heads, dim), table, lengths, k, v, spread, n_pages, dim ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (12, 2, 128), (16, 1, 128), (8, 2, 256), (16, 1, 256)])
@pytest.mark.parametrize("position", [0, 70])
def test_paged_attention_of_one_key_is_its_value(dev, dtype, heads, kv, dim, position):
    """where one key has all the weight its product with the scale is exact: the value is rounded once, behind sums in binary32"""
    rng = rng_of("one key", dtype, heads, dim, position)
    n, L = 40, position + 1
    table, n_pages = tables(rng, n, [plain.pages(L)] * n, 2)
    cache, k, v, spread = cache_of(dev, rng, n_pages, kv, dim)
    q = np.ones((n, heads * dim))
    if position:  # all other keys have none: theirs are far below
        raw = cache.view(dev.torch.float16).reshape(n_pages, kv, 36 * dim)[:, :, 32 * dim:34 * dim].reshape(n_pages, kv, dim // 64, 2, 64)
        raw[:, :, :, 0], raw[:, :, :, 1] = 0.0, -60000.0
        raw[:, :, :, 1, position % 64].fill_(100.0)
        raw[dev.torch.from_numpy(table[:, 0]).cuda(), :, :, 1] = -60000.0
    d_q, _ = dev.act(q, dtype)
    got = paged(dev, dtype, d_q, cache, table, [L] * n, heads, kv, dim, dim ** -0.5, dev.full((n, heads * dim), 9.0, dtype)).reshape(n, heads, dim)
    of = table[:, position // 64], slice(None), position % 64
    want, size = (np.repeat(t[of], heads // kv, 1) for t in (v, spread))
    assert (np.abs(got - want) <= plain.EPS[dtype] / 2 * np.abs(want) + 2.0 ** -21 * size + (2.0 ** -25 if dtype == "f16" else 0.0)).all()


@pytest.mark.parametrize("dim,long", [(64, 2500), (256, 1250)])
def test_paged_attention_of_many_pages_a_wavefront(dev, dim, long):
    """128 key/value heads leave a wavefront more than 64 pages of one request: its page numbers are read anew while pages are on their way"""
    kv, few = 128, [0, 77]
    lengths = [200, 64 * long - 7, 1, 64 * 90]
    rng = rng_of("many pages", dim)
    print("paged, many pages", dim, flush=True)
    n_pages, width = 9, long
    cache, k, v, spread = cache_of(dev, rng, n_pages, kv, dim)
    table = rng.integers(0, n_pages, (4, width))
    table[rng.random(table.shape) < 0.1] = -1
    table[1, 60:130] = np.where(np.arange(70) % 7 == 0, 3, -1)
    x = rng.standard_normal((4, kv * dim))
    d_q, vq = dev.act(x, "f16")
    got = paged(dev, "f16", d_q, cache, table, lengths, kv, kv, dim, dim ** -0.5, dev.full((4, kv * dim), 9.0, "f16")).reshape(4, kv, dim)
    k, v, spread = (t[:, few] for t in (k, v, spread))
    check_paged(got[:, few], "f16", vq.reshape(4, kv, dim)[:, few], table, lengths, k, v, spread, n_pages, dim ** -0.5)


# --- attention of packed prompts ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("behind", [32, 96, 160])
def test_packed_attention_beside_what_is_not_finite_in_a_step_that_some_wavefronts_skip(dev, dtype, dim, behind):
    """Requests with positions ahead of their queries: the first wavefronts of a tile are done some steps ahead of the last ones, and all of them look
    for values that are not finite.  Those of keys that a query does not see do not reach it, those of keys it sees do."""
    heads, kv, new = 2, 1, [150, 128, 200, 129]
    rng = rng_of(dtype, dim, behind)
    print("packed, not finite", dtype, dim, behind, flush=True)
    q_starts, k_starts = np.cumsum([0] + new), np.cumsum([0] + [n + behind for n in new])
    n_q, n_k = int(q_starts[-1]), int(k_starts[-1])
    d_q, vq = dev.act(rng.standard_normal((n_q, heads * dim)), dtype)
    d_k, vk = dev.act(rng.standard_normal((n_k, kv * dim)), dtype)
    v = rng.standard_normal((n_k, kv * dim))
    for c in k_starts[:-1]:
        v[c + behind + 97, 0], v[c + behind + 99, 7], v[c + behind + 127, dim - 1] = -np.inf, np.inf, np.nan
    d_v, vv = dev.act(v, dtype)
    got = packed(dev, dtype, d_q, d_k, d_v, q_starts, k_starts, heads, kv, dim, True, dim ** -0.5, dev.full((n_q, heads * dim), 9.0, dtype))
    got = got.reshape(n_q, heads, dim)
    finite = np.where(np.isfinite(vv), vv, 0.0)
    for a, c, n in zip(q_starts, k_starts, new):
        at = np.arange(n)
        for first, column, want in ((97, 0, -np.inf), (99, 7, np.inf), (127, dim - 1, np.nan)):
            x = got[a:a + n, :, column]
            assert np.isfinite(x[at < first]).all()
            assert np.isnan(x[at >= first]).all() if np.isnan(want) else (x[at >= first] == want).all()
            got[a:a + n, :, column][at >= first] = 0.0
    # the columns without them are those of finite values, and so are the queries ahead of them
    limit_of = [0, 7, dim - 1]
    others = np.setdiff1d(np.arange(dim), limit_of)
    shape = lambda x: x.reshape(len(x), -1, dim)  # noqa: E731
    for columns, many in ((others, None), (limit_of, 97)):
        for a, c, n in zip(q_starts, k_starts, new):
            m = n if many is None else many
            i, j = np.arange(m)[:, None], np.arange(m + behind)[None, :]
            want, size = plain.attention(shape(vq)[a:a + m], shape(vk)[c:c + m + behind], shape(finite)[c:c + m + behind], dim ** -0.5, j <= i + behind)
            terms = np.abs(shape(vq)[a:a + m]).sum(-1).max() * np.abs(vk[c:c + m + behind]).max() * dim ** -0.5
            limit = plain.EPS[dtype] / 2 * (2 * np.abs(want) + size) * 1.01 + (terms * 2.0 ** -20 + 2.0 ** -18) * size + 1e-30
            assert (np.abs(got[a:a + m] - want) <= limit)[:, :, columns].all(), (a, n, dim, columns[:3])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("score", [0.716796875, 1.3984375, 3.494140625])
def test_packed_attention_of_values_at_the_end_of_binary16(dev, dim, score):
    """weights e^score that binary16 rounds up by some 4.5e-4, of values that are its largest number: their mean is that number"""
    n, q = 2048, np.zeros((5, dim))
    q[:, 0] = 1.0
    k, v = np.zeros((n, dim)), np.full((n, dim), 65504.0)
    k[64:, 0] = score
    v[:, 1::2] *= -1.0
    (d_q, _), (d_k, _), (d_v, vv) = (dev.act(x, "f16") for x in (q, k, v))
    got = packed(dev, "f16", d_q, d_k, d_v, [0, 5], [0, n], 1, 1, dim, False, 1.0, dev.full((5, dim), 9.0, "f16"))
    assert np.isfinite(got).all() and (np.abs(got - vv[:5]) <= 2.0 ** -10 * 65504.0).all()


# --- sampling -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [5, 31, 5000, 8193, 40000])
def test_sample_of_uniform_numbers_next_to_zero(dev, dtype, vocab):
    """the first token kept, however little it weighs: also where fewer tokens than top-k keeps, or than weigh min-p, are within e^-64 of the largest"""
    rng = rng_of("zero", dtype, vocab)
    print("sample, zero", dtype, vocab, flush=True)
    n = 12
    x = rng.standard_normal((n, vocab))
    x[0, vocab // 2:vocab // 2 + 10] += 90
    x[1] = np.round(2 * x[1]) * 40              # many equals
    x[2] = np.where(np.arange(vocab) % 3 == 1, 9.0, -1e4)
    x[3] = -np.inf
    x[3, [vocab // 3, vocab - 1]] = -100.0, 0.0
    x[4, vocab // 2] = np.inf
    x[5, : vocab // 2] = np.nan
    x[6] *= 40
    x[7, vocab // 4:] = -np.inf
    d_x, vx = dev.act(x, dtype)
    of = lambda *v: [v[i % len(v)] for i in range(n)]  # noqa: E731
    k = of(50, 3, 2, 5, 1000, 4, 20, 4999, 1, 8190)
    for u in (0.0, 1e-30, 2.0 ** -61, 2.0 ** -149):
        for t, kk, p, m in ((of(1.0), k, None, None), (of(0.02, 0.05), k, None, None), (of(0.01), None, None, of(1e-30, 1e-35, 1e-28, 1e-27)), (of(0.02), k, None, of(1e-30, 0.0, 1e-37)),
                            (of(0.02), k, of(1.0, 0.9, 0.999999), of(0.0, 1e-20)), (of(1e-3, 3e38, 1e-30), k, None, None), (of(0.02), None, None, None)):
            us = np.full(n, u, np.float32)
            check_sample(dev, dtype, vx, sample(dev, dtype, d_x, us, t, kk, p, m), us, t, kk, p, m)
