"""Several requests at once over a key/value cache that is held in 4 bits: the operators of such a step, for timing and for
comparing results.

  plan       pages and slots of a step's new positions, from the requests' lengths
  append     rotary positions on queries and keys, keys and values into the pages; read back as the values they stand for
  attention  one query of each request over its pages
  packed     prompts of different lengths, one behind the other, each seeing its own keys up to its own position
  sample     a token of each row of logits: temperature, top-k, top-p, min-p, from given uniform numbers

A page holds 64 positions of every key/value head, 72 dim bytes a head: keys and values in nibbles (low one first), then the
keys' and the values' parameters, [dim / 64][scale, offset][64 positions] in binary16.  64 values of a position share a scale s and
an offset z, and nibble n stands for s n + z.  Nibble k dim / 4 + 16 g + e of a key's row is its value 64 g + 16 k + e, nibble
c dim / 16 + 4 g + e of a value's row its value 64 g + 4 c + e.

Lengths belong to the case, values to the seed."""
import ctypes
import importlib
import math
import random

import numpy as np
import torch

PACKAGE = "cuda-kernel-qwen3-8b-awq_amd"
PAGE = 64
VOCAB = 151936

own = False


def listed():
    return [
        # a decode step of a busy server: one new position a request
        {"name": "plan 200 answers", "op": "plan", "requests": 200, "prompts": 0, "longest": 8000, "fresh": 1, "ended": 5},
        # the same with prompts that came in, and requests that ended
        {"name": "plan 40 prompts among 240", "op": "plan", "requests": 240, "prompts": 40, "longest": 8000, "fresh": 2000, "ended": 17},
        # a decode step's new rows, the int4 model's number format and pairs
        {"name": "append 64 answers f16", "op": "append", "dtype": "float16", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "interleaved": True},
        # a prompt pass, half of each head rotated, positions scaled for a long context
        {"name": "append 8000 positions bf16", "op": "append", "dtype": "bfloat16", "tokens": 8000, "heads": 32, "kv_heads": 8, "dim": 128,
         "rot": 64, "interleaved": False},
        # the smallest call: a few chats just begun, small heads without groups
        {"name": "attention 12 short f16", "op": "attention", "dtype": "float16", "requests": 12, "shortest": 5, "longest": 300, "heads": 16,
         "kv_heads": 16, "dim": 64},
        # one document at the positions the int4 model holds
        {"name": "attention 1 of 40960 f16", "op": "attention", "dtype": "float16", "requests": 1, "shortest": 40960, "longest": 40960,
         "heads": 32, "kv_heads": 8, "dim": 128},
        # a busy server's decode step
        {"name": "attention 64 ragged bf16", "op": "attention", "dtype": "bfloat16", "requests": 64, "shortest": 100, "longest": 8000,
         "heads": 32, "kv_heads": 8, "dim": 128},
        # prompts that came in together
        {"name": "packed 13 prompts f16", "op": "packed", "dtype": "float16", "requests": 13, "shortest": 60, "longest": 1000, "behind": 0,
         "heads": 32, "kv_heads": 8, "dim": 128},
        # parts of long prompts behind what has been read of them
        {"name": "packed 3 chunks bf16", "op": "packed", "dtype": "bfloat16", "requests": 3, "shortest": 500, "longest": 1100, "behind": 3500,
         "heads": 32, "kv_heads": 8, "dim": 128},
        # one row of the int4 model
        {"name": "sample 1 row f16", "op": "sample", "dtype": "float16", "rows": 1, "vocab": VOCAB, "filters": True},
        # a large batch of binary32 logits, every row with settings of its own
        {"name": "sample 256 rows f32", "op": "sample", "dtype": "float32", "rows": 256, "vocab": VOCAB, "filters": True},
        # a middling batch that is only tempered, odd vocabulary
        {"name": "sample 33 rows bf16", "op": "sample", "dtype": "bfloat16", "rows": 33, "vocab": 32771, "filters": False},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "packed", "packed", "sample", "sample"])
    if op == "plan":
        n = _spread(rng, 1, 240)
        return {"op": op, "requests": n, "prompts": rng.randrange(n // 4 + 1), "longest": _spread(rng, 64, 8000),
                "fresh": _spread(rng, 1, 2000), "ended": rng.randrange(n // 8 + 1)}
    dtype = rng.choice(["float16", "bfloat16"])
    if op == "sample":
        return {"op": op, "dtype": rng.choice(["float16", "bfloat16", "float32"]), "rows": _spread(rng, 1, 256), "vocab": _spread(rng, 500, VOCAB),
                "filters": rng.random() < 0.7}
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = {"heads": kv * rng.choice([1, 2, 4] if dim == 128 else [1, 2, 3]), "kv_heads": kv, "dim": dim}
    if op == "append":
        return {"op": op, "dtype": dtype, "tokens": _spread(rng, 1, 8000), "rot": rng.choice([dim // 4, dim // 2, dim]),
                "interleaved": rng.random() < 0.5, **heads}
    if op == "attention":
        lo = _spread(rng, 1, 2000)
        return {"op": op, "dtype": dtype, "requests": _spread(rng, 1, 64), "shortest": lo, "longest": _spread(rng, lo, 8000), **heads}
    lo = _spread(rng, 1, 700)
    return {"op": op, "dtype": dtype, "requests": _spread(rng, 1, 10), "shortest": lo, "longest": _spread(rng, lo, 1100),
            "behind": rng.choice([0, _spread(rng, 1, 2000)]), **heads}


# --- inputs --------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _type(case):
    return getattr(torch, case["dtype"])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prefix(values):
    return [sum(values[:i]) for i in range(len(values) + 1)]


def _ragged(case, n):
    """n lengths between the shortest and the longest, both among them"""
    rng = random.Random("%d %d %d" % (n, case["shortest"], case["longest"]))
    got = [_spread(rng, case["shortest"], case["longest"]) for _ in range(n)]
    got[0] = case["longest"]
    return got


def _plan_lengths(case):
    """(held, new) positions of every request; -1 new ones: the request has ended"""
    n = case["requests"]
    rng = random.Random("%d %d %d" % (n, case["prompts"], case["longest"]))
    cached, fresh = [], []
    for i in range(n):
        prompt = i % max(1, n // max(1, case["prompts"])) == 0 and sum(f > 1 for f in fresh) < case["prompts"]
        cached.append(rng.choice([0, 0, 64, _spread(rng, 1, case["longest"])]) if prompt else _spread(rng, 1, case["longest"]))
        fresh.append(_spread(rng, 1, case["fresh"]) if prompt else 1)
    for i in rng.sample(range(n), case["ended"]):
        fresh[i] = -1
    return cached, fresh


def _pages(n):
    return -(-n // PAGE)


def prepare(case, seed):
    return {"op": case["op"], **_prepare[case["op"]](case, _gen(seed), seed)}


def _prepare_plan(case, g, seed):
    cached, fresh = _plan_lengths(case)
    held = [_pages(c) for c in cached]
    width = _pages(case["longest"] + case["fresh"]) + 1
    need = sum(_pages(c + f) - _pages(c) for c, f in zip(cached, fresh) if f > 0)
    n_pages = sum(held) + need + 100
    order = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.full((len(cached), width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None, :] < torch.tensor(held, device="cuda")[:, None]
    table[at] = order[:sum(held)]
    free = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    free[:n_pages - sum(held)] = order[sum(held):]
    return {"cached": _ints(cached), "fresh": _ints(fresh), "table": table, "free": free, "count": _ints([n_pages - sum(held)]),
            "tokens": sum(max(f, 0) for f in fresh)}


def _rotary(rot, positions, factor):
    """cosines and sines, the positions divided by `factor`"""
    freq = 10000.0 ** (-2.0 * torch.arange(rot // 2, device="cuda", dtype=torch.float64) / rot)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] / factor * freq[None, :]
    return angle.cos().float(), angle.sin().float()


def _prepare_append(case, g, seed):
    T, H, KV, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    # a few requests' positions, some behind others, into pages in no order
    n = min(T, 64)
    fresh = [T // n + (i < T % n) for i in range(n)]
    first = [(997 * i) % 3001 for i in range(n)]
    width = max(_pages(a + f) for a, f in zip(first, fresh))
    table = torch.randperm(n * width, generator=g, device="cuda").int().reshape(n, width)
    request = torch.repeat_interleave(torch.arange(n, device="cuda"), torch.tensor(fresh, device="cuda"))
    starts = torch.tensor(_prefix(fresh), device="cuda")
    positions = torch.arange(T, device="cuda") - starts[request] + torch.tensor(first, device="cuda")[request]
    slots = table[request, positions // PAGE].long() * PAGE + positions % PAGE
    qkv = torch.randn(T, (H + 2 * KV) * d, generator=g, device="cuda") * (0.5 + torch.rand((H + 2 * KV) * d, generator=g, device="cuda"))
    cos, sin = _rotary(case["rot"], 12000, 4.0)
    return {"case": case, "qkv": qkv.to(_type(case)), "cos": cos, "sin": sin, "positions": positions.int(), "slots": slots.int(), "table": table,
            "first": _ints(first), "lengths": _ints([a + f for a, f in zip(first, fresh)]), "starts": starts.int(),
            "cache": torch.zeros(n * width, KV, 72 * d, dtype=torch.uint8, device="cuda")}


def _prepare_attention(case, g, seed):
    n, H, KV, d = case["requests"], case["heads"], case["kv_heads"], case["dim"]
    lengths = _ragged(case, n)
    held = [_pages(x) for x in lengths]
    width, n_pages = max(held), sum(held) + 3
    cache = torch.randint(0, 256, (n_pages, KV, 72 * d), generator=g, device="cuda", dtype=torch.uint8)
    scale = 0.1 + 0.3 * torch.rand(n_pages, KV, 2, d // 64, 1, PAGE, generator=g, device="cuda")
    offset = scale * (-7.5 + torch.randn(scale.shape, generator=g, device="cuda"))
    cache[:, :, 64 * d:] = torch.cat([scale, offset], 4).half().reshape(n_pages, KV, -1).view(torch.uint8)
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda")[None, :] < torch.tensor(held, device="cuda")[:, None]
    table[at] = torch.randperm(n_pages, generator=g, device="cuda").int()[:sum(held)]
    q = (torch.randn(n, H * d, generator=g, device="cuda") * 1.5).to(_type(case))
    return {"case": case, "q": q, "cache": cache, "table": table, "lengths": _ints(lengths)}


def _packed_lengths(case):
    new = _ragged(case, case["requests"])
    return new, [n + (case["behind"] * (i + 1) // case["requests"]) for i, n in enumerate(new)]


def _prepare_packed(case, g, seed):
    H, KV, d = case["heads"], case["kv_heads"], case["dim"]
    new, keys = _packed_lengths(case)
    q, k = (torch.randn(sum(n), h * d, generator=g, device="cuda") * 1.2 for n, h in ((new, H), (keys, KV)))
    v = torch.randn(sum(keys), KV * d, generator=g, device="cuda")
    return {"case": case, "q": q.to(_type(case)), "kv": torch.cat([k, v], 1).to(_type(case)), "q_starts": _ints(_prefix(new)),
            "k_starts": _ints(_prefix(keys))}


def _prepare_sample(case, g, seed):
    n, V = case["rows"], case["vocab"]
    logits = 2.0 * torch.randn(n, V, generator=g, device="cuda")
    # tokens that fit, and tokens that are not allowed
    fits = torch.randint(0, V, (n, 60), generator=g, device="cuda")
    logits.scatter_add_(1, fits, 2.0 + 3.0 * torch.rand(n, 60, generator=g, device="cuda"))
    logits[:, torch.randint(0, V, (V // 50,), generator=g, device="cuda")] = -math.inf
    pick = lambda *of: torch.tensor(of, device="cuda")[torch.randint(0, len(of), (n,), generator=g, device="cuda")]  # noqa: E731
    state = {"case": case, "logits": logits.to(_type(case)), "temperature": pick(0.6, 0.8, 1.0, 1.0, 1.3), "u": torch.rand(n, generator=g, device="cuda"),
             "top_k": None, "top_p": None, "min_p": None}
    if case["filters"]:
        state |= {"temperature": pick(0.0, 0.6, 0.8, 1.0, 1.3), "top_k": pick(0, 0, 20, 50, 400).int(), "top_p": pick(1.0, 0.5, 0.9, 0.95),
                  "min_p": pick(0.0, 0.0, 0.02, 0.1)}
    return state


_prepare = {"plan": _prepare_plan, "append": _prepare_append, "attention": _prepare_attention, "packed": _prepare_packed, "sample": _prepare_sample}


# --- the framework's operators ---------------------------------------------------------------------------------------
_kept = {}  # the package and the scratch memory that a program keeps


def _awq():
    if "awq" not in _kept:
        _kept["awq"] = importlib.import_module(PACKAGE)
    return _kept["awq"], _kept["awq"].load_library(), torch.cuda.current_stream().cuda_stream


def _scratch(n):
    if "scratch" not in _kept or _kept["scratch"].numel() < n:
        _kept["scratch"] = torch.empty(max(n, 1 << 20), dtype=torch.uint8, device="cuda")
    return _kept["scratch"]


_code = {torch.bfloat16: 1, torch.float32: 2, torch.float16: 3}


def _own_plan(s):
    awq, lib, stream = _awq()
    n, width = s["table"].shape
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    lengths, starts, keys, positions, slots, count, left = new(n), new(n + 1), new(n + 1), new(s["tokens"]), new(s["tokens"]), new(1), new(1)
    a = awq.AwqPagePlanArgs(s["cached"].data_ptr(), s["fresh"].data_ptr(), s["table"].data_ptr(), s["free"].data_ptr(), s["count"].data_ptr(),
                            count.data_ptr(), lengths.data_ptr(), starts.data_ptr(), keys.data_ptr(), positions.data_ptr(), slots.data_ptr(),
                            left.data_ptr(), s["tokens"], n, width, s["free"].numel(), 0)
    awq.check(lib.awq_page_plan(ctypes.byref(a), stream))
    return {"table": s["table"], "free": s["free"], "count": count, "lengths": lengths, "starts": starts, "keys": keys, "positions": positions,
            "slots": slots, "left": left}


def _own_append(s):
    awq, lib, stream = _awq()
    c, x = s["case"], s["qkv"]
    T, H, KV, d, ld, size = c["tokens"], c["heads"], c["kv_heads"], c["dim"], x.shape[1], 2
    q, k, kc, vc = (torch.empty(T, h * d, dtype=x.dtype, device="cuda") for h in (H, KV, KV, KV))
    at = x.data_ptr()
    n, width = s["table"].shape
    a = awq.AwqPagedAppendArgs(at, q.data_ptr(), at + size * H * d, k.data_ptr(), at + size * (H + KV) * d, s["cos"].data_ptr(), s["sin"].data_ptr(),
                               s["positions"].data_ptr(), s["slots"].data_ptr(), s["cache"].data_ptr(), ld, H * d, ld, KV * d, ld, T,
                               s["cos"].shape[0], H, KV, d, c["rot"], int(c["interleaved"]), n * width)
    awq.check(lib.awq_paged_append(ctypes.byref(a), _code[x.dtype], stream))
    b = awq.AwqPagedRowsArgs(s["cache"].data_ptr(), s["table"].data_ptr(), s["first"].data_ptr(), s["lengths"].data_ptr(), s["starts"].data_ptr(),
                             kc.data_ptr(), vc.data_ptr(), KV * d, KV * d, T, n, width, n * width, KV, d, 0)
    awq.check(lib.awq_paged_rows(ctypes.byref(b), _code[x.dtype], stream))
    return {"q": q, "k": k, "keys": kc, "values": vc}


def _own_attention(s):
    awq, lib, stream = _awq()
    c, q = s["case"], s["q"]
    H, KV, d = c["heads"], c["kv_heads"], c["dim"]
    n, width = s["table"].shape
    ctx = torch.empty_like(q)
    size = lib.awq_paged_workspace_bytes(n, H, KV, d, width)
    a = awq.AwqPagedAttentionArgs(q.data_ptr(), s["cache"].data_ptr(), s["table"].data_ptr(), s["lengths"].data_ptr(), ctx.data_ptr(),
                                  _scratch(size).data_ptr(), H * d, H * d, size, n, width, s["cache"].shape[0], H, KV, d, d ** -0.5, 0)
    awq.check(lib.awq_paged_attention(ctypes.byref(a), _code[q.dtype], stream))
    return ctx


def _own_packed(s):
    awq, lib, stream = _awq()
    c, q, kv = s["case"], s["q"], s["kv"]
    H, KV, d = c["heads"], c["kv_heads"], c["dim"]
    ctx = torch.empty_like(q)
    a = awq.AwqPackedAttentionArgs(q.data_ptr(), kv.data_ptr(), kv.data_ptr() + 2 * KV * d, ctx.data_ptr(), s["q_starts"].data_ptr(),
                                   s["k_starts"].data_ptr(), H * d, 2 * KV * d, 2 * KV * d, H * d, q.shape[0], kv.shape[0], c["requests"], H, KV, d, 1,
                                   d ** -0.5)
    awq.check(lib.awq_packed_attention(ctypes.byref(a), _code[q.dtype], stream))
    return ctx


def _own_sample(s):
    awq, lib, stream = _awq()
    x = s["logits"]
    n, V = x.shape
    ids = torch.empty(n, dtype=torch.int32, device="cuda")
    size = lib.awq_sample_workspace_bytes(n, V)
    of = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    a = awq.AwqSampleArgs(x.data_ptr(), s["temperature"].data_ptr(), of(s["top_k"]), of(s["top_p"]), of(s["min_p"]), s["u"].data_ptr(), ids.data_ptr(),
                          _scratch(size).data_ptr(), V, V, n, size)
    awq.check(lib.awq_sample(ctypes.byref(a), _code[x.dtype], stream))
    return ids


# --- the plain forms -------------------------------------------------------------------------------------------------
def _to(x, dtype):
    """64 bits to 16 in one rounding (by way of 32 bits a value next to a border is rounded twice)"""
    digits, least = (11, -13) if dtype == torch.float16 else (8, -125)
    step = torch.ldexp(torch.ones_like(x), torch.frexp(x)[1].clamp(min=least) - digits)
    return (torch.round(x / step) * step).to(dtype)


def _plain_plan(s):
    cached, fresh, table = s["cached"].long(), s["fresh"].long(), s["table"].clone()
    n, width = table.shape
    held = (cached + PAGE - 1) // PAGE
    at = torch.arange(width, device="cuda")[None, :]
    given = table[(fresh < 0)[:, None] & (at < held[:, None])]
    free = s["free"].clone()
    place = s["count"].long() + torch.arange(given.numel(), device="cuda")
    free[place] = given
    available = s["count"].long() + given.numel()
    fits = cached + fresh <= width * PAGE
    need = torch.where((fresh > 0) & fits, (cached + fresh + PAGE - 1) // PAGE - held, 0)
    total = need.cumsum(0)
    served = fits & ((need == 0) | (total <= available))
    new = served[:, None] & (at >= held[:, None]) & (at < (held + need)[:, None])
    which = available - 1 - (total - need)[:, None] - (at - held[:, None])
    table = torch.where(new, free[which.clamp(0, free.numel() - 1)], table)
    taken = torch.where(served, total * (need > 0), 0).max()
    lengths = torch.where(fresh < 0, 0, cached + torch.where(served, fresh, 0))
    put = fresh.clamp(min=0)
    zero = torch.zeros(1, dtype=torch.long, device="cuda")
    starts, keys = torch.cat([zero, put.cumsum(0)]), torch.cat([zero, lengths.cumsum(0)])
    token = torch.arange(s["tokens"], device="cuda")
    request = torch.searchsorted(starts, token, right=True) - 1
    positions = cached[request] + token - starts[request]
    slots = table[request, (positions // PAGE).clamp(max=width - 1)] * PAGE + positions % PAGE
    slots = torch.where(served[request], slots, -1)
    return {"table": table, "free": free, "count": (available - taken).int(), "lengths": lengths.int(), "starts": starts.int(), "keys": keys.int(),
            "positions": positions.int(), "slots": slots.int(), "left": (~served).sum().int().reshape(1)}


def _plain_append(s):
    c = s["case"]
    T, H, KV, d, rot = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rot"]
    x = s["qkv"].double().reshape(T, H + 2 * KV, d)
    at = s["positions"].long()
    cos, sin = s["cos"][at].double()[:, None, :], s["sin"][at].double()[:, None, :]
    turn, rest = x[:, :H + KV, :rot], x[:, :H + KV, rot:]
    if c["interleaved"]:
        a, b = turn[..., 0::2], turn[..., 1::2]
        turn = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).reshape(T, H + KV, rot)
    else:
        a, b = turn[..., :rot // 2], turn[..., rot // 2:]
        turn = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    qk = _to(torch.cat([turn, rest], -1), s["qkv"].dtype)
    rows = torch.cat([qk[:, H:].double(), x[:, H + KV:]], 1).reshape(T, 2 * KV, d // 64, 64)
    z = _to(rows.amin(-1, keepdim=True), torch.float16).double()
    scale = _to((rows.amax(-1, keepdim=True) - rows.amin(-1, keepdim=True)) / 15.0, torch.float16).double()
    n = torch.round((rows - z) / torch.where(scale > 0, scale, 1.0)).clamp(0.0, 15.0) * (scale > 0)
    rows = _to(n * scale + z, s["qkv"].dtype).reshape(T, 2, KV * d)
    return {"q": qk[:, :H].reshape(T, H * d), "k": qk[:, H:].reshape(T, KV * d), "keys": rows[:, 0].contiguous(), "values": rows[:, 1].contiguous()}


def _unpacked(cache, d):
    """keys and values [page][head][64][dim] in 32 bits"""
    pages, KV = cache.shape[:2]
    G = d // 64
    byte = cache[:, :, :64 * d].reshape(pages, KV, 2, PAGE, d // 2)
    n = torch.stack([byte & 15, byte >> 4], -1).reshape(pages, KV, 2, PAGE, d).float()
    par = cache[:, :, 64 * d:].contiguous().view(torch.float16).float().reshape(pages, KV, 2, G, 2, PAGE)
    s, z = par[..., 0, :].transpose(3, 4), par[..., 1, :].transpose(3, 4)  # [page][head][k, v][64][G]
    k = n[:, :, 0].reshape(pages, KV, PAGE, 4, G, 16).transpose(3, 4) * s[:, :, 0, :, :, None, None] + z[:, :, 0, :, :, None, None]
    v = n[:, :, 1].reshape(pages, KV, PAGE, 16, G, 4).transpose(3, 4) * s[:, :, 1, :, :, None, None] + z[:, :, 1, :, :, None, None]
    return k.reshape(pages, KV, PAGE, d), v.reshape(pages, KV, PAGE, d)


def _plain_attention(s):
    c, lengths = s["case"], s["lengths"]
    n, H, KV, d = c["requests"], c["heads"], c["kv_heads"], c["dim"]
    width = s["table"].shape[1]
    at = s["table"].clamp(min=0).long()
    k, v = (x[at].transpose(1, 2).reshape(n, KV, width * PAGE, d) for x in _unpacked(s["cache"], d))
    q = s["q"].float().reshape(n, KV, H // KV, d) * d ** -0.5
    p = torch.matmul(q, k.transpose(2, 3).contiguous())
    p = p.masked_fill(torch.arange(width * PAGE, device="cuda") >= lengths[:, None, None, None], -math.inf)
    p = (p - p.amax(-1, keepdim=True)).exp()
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(n, H * d).to(s["q"].dtype)


def _plain_packed(s):
    c = s["case"]
    n, H, KV, d = c["requests"], c["heads"], c["kv_heads"], c["dim"]
    of_q, of_k = s["q_starts"].long(), s["k_starts"].long()
    nq, nk = of_q.diff(), of_k.diff()
    row, col = torch.arange(c["longest"], device="cuda"), torch.arange(c["longest"] + c["behind"], device="cuda")
    q = s["q"][(of_q[:-1, None] + row).clamp(max=s["q"].shape[0] - 1)].float().reshape(n, -1, KV, H // KV, d).permute(0, 2, 3, 1, 4) * d ** -0.5
    kv = s["kv"][(of_k[:-1, None] + col).clamp(max=s["kv"].shape[0] - 1)].float().reshape(n, -1, 2, KV, 1, d).permute(2, 0, 3, 4, 1, 5)
    seen = col[None, None, :] <= (row[None, :] + (nk - nq)[:, None])[:, :, None]
    p = torch.matmul(q, kv[0].transpose(3, 4).contiguous()).masked_fill(~seen[:, None, None], -math.inf)
    p = (p - p.amax(-1, keepdim=True)).exp()
    o = torch.matmul(p, kv[1].contiguous()) / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(n, -1, H * d)[row[None, :] < nq[:, None]].to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"]
    n, V = x.shape
    greedy = s["temperature"] <= 0
    T = torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    ordered, index = x.sort(dim=-1, descending=True, stable=True)
    w = ((ordered.double() - ordered[:, :1].double()) / T).exp()
    keep = torch.ones(n, V, dtype=torch.bool, device="cuda")
    if s["top_k"] is not None:
        place = torch.arange(V, device="cuda")[None, :]
        k = torch.where(s["top_k"] > 0, s["top_k"], V)[:, None]
        sums = torch.where(place < k, w, 0.0).cumsum(-1)
        ahead = torch.cat([torch.zeros_like(sums[:, :1]), sums[:, :-1]], 1)
        p = s["top_p"].double()[:, None]
        keep = (place < k) & ((p >= 1) | (place == 0) | (ahead < p * sums[:, -1:])) & (w >= s["min_p"].double()[:, None])
    w = torch.zeros_like(w).scatter_(1, index, torch.where(keep, w, 0.0))
    sums = w.cumsum(-1)
    chosen = ((sums > s["u"].double()[:, None] * sums[:, -1:]) & (w > 0)).int().argmax(-1)
    return torch.where(greedy, index[:, 0], chosen).int()


def run(state):
    if own:
        return _own[state["op"]](state)
    return _plain[state["op"]](state)


_own = {"plan": _own_plan, "append": _own_append, "attention": _own_attention, "packed": _own_packed, "sample": _own_sample}
_plain = {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "packed": _plain_packed, "sample": _plain_sample}


# --- what the operators' definitions give, in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _exact[case["op"]](s)


def _exact_plan(s):
    cached, fresh, table, free = (s[x].cpu().numpy().copy() for x in ("cached", "fresh", "table", "free"))
    n, width = table.shape
    stack = free[:int(s["count"])].tolist()
    for i in range(n):
        if fresh[i] < 0:
            stack += table[i, :_pages(int(cached[i]))].tolist()
    free[:len(stack)] = stack
    available, taken, left = len(stack), 0, 0
    lengths, starts, keys, positions, slots = [], [0], [0], [], []
    for i in range(n):
        a, f = int(cached[i]), int(fresh[i])
        need = _pages(a + f) - _pages(a) if f > 0 else 0
        served = a + f <= width * PAGE and (need == 0 or taken + need <= available)
        if a + f <= width * PAGE:
            if need and served:
                table[i, _pages(a):_pages(a + f)] = [stack[available - 1 - taken - j] for j in range(need)]
            taken += need if served else 1 << 40  # whoever comes behind one that has to wait waits too
        left += not served
        lengths.append(0 if f < 0 else a + f if served else a)
        starts.append(starts[-1] + max(f, 0))
        keys.append(keys[-1] + lengths[-1])
        for p in range(a, a + max(f, 0)):
            positions.append(p)
            slots.append(int(table[i, p // PAGE]) * PAGE + p % PAGE if served else -1)
    if taken >= 1 << 40:
        return None  # (no case of these runs out of pages)
    as_ints = lambda v: np.array(v, dtype=np.int32)  # noqa: E731
    return {"table": table, "free": free, "count": as_ints([available - taken]), "lengths": as_ints(lengths), "starts": as_ints(starts),
            "keys": as_ints(keys), "positions": as_ints(positions), "slots": as_ints(slots), "left": as_ints([left])}


def _nearest(x, dtype):
    """the numbers of a 16-bit type nearest to x, even ones of two, as 64-bit numbers"""
    if dtype == torch.float16:
        return x.astype(np.float16).astype(np.float64)
    m, e = np.frexp(x)
    return np.ldexp(np.rint(np.ldexp(m, 8)), e - 8)


def _exact_append(s):
    c = s["case"]
    T, H, KV, d, rot, dtype = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rot"], s["qkv"].dtype
    x = s["qkv"].double().cpu().numpy().reshape(T, H + 2 * KV, d)
    at = s["positions"].cpu().numpy()
    cos, sin = s["cos"].double().cpu().numpy()[at][:, None], s["sin"].double().cpu().numpy()[at][:, None]
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if c["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    y = x[:, :H + KV].copy()
    y[..., one] = x[:, :H + KV, one] * cos - x[:, :H + KV, two] * sin
    y[..., two] = x[:, :H + KV, two] * cos + x[:, :H + KV, one] * sin
    rows = []
    for r in (_nearest(y[:, H:], dtype), x[:, H + KV:]):
        r = r.reshape(T, KV, d // 64, 64)
        lo, hi = r.min(-1, keepdims=True), r.max(-1, keepdims=True)
        z, scale = _nearest(lo, torch.float16), _nearest((hi - lo) / 15.0, torch.float16)
        with np.errstate(divide="ignore", invalid="ignore"):
            n = np.where(scale > 0, np.clip(np.rint((r - z) / scale), 0, 15), 0)
        rows.append((n * scale + z).reshape(T, KV * d))
    return {"q": y[:, :H].reshape(T, H * d), "k": y[:, H:].reshape(T, KV * d), "keys": rows[0], "values": rows[1]}


def _exact_attention(s):
    c = s["case"]
    H, KV, d = c["heads"], c["kv_heads"], c["dim"]
    G = d // 64
    i = torch.arange(d, device="cuda")
    of_key = (i % 64 // 16) * (d // 4) + 16 * (i // 64) + i % 16
    of_value = (i % 64 // 4) * (d // 16) + 4 * (i // 64) + i % 4
    out = []
    for r, n in enumerate(s["lengths"].tolist()):
        pages = s["cache"][s["table"][r, :_pages(n)].long()]  # [pages][KV][72 d]
        par = pages[:, :, 64 * d:].contiguous().view(torch.float16).double().reshape(-1, KV, 2, G, 2, PAGE)
        kv = []
        for which, order in ((0, of_key), (1, of_value)):
            byte = pages[:, :, 32 * d * which:32 * d * (which + 1)].reshape(-1, KV, PAGE, d // 2)
            nib = torch.where(order % 2 == 0, byte[..., order // 2] & 15, byte[..., order // 2] >> 4).double()
            values = nib * par[:, :, which, i // 64, 0].transpose(2, 3) + par[:, :, which, i // 64, 1].transpose(2, 3)
            kv.append(values.transpose(0, 1).reshape(KV, -1, d)[:, :n])
        q = s["q"][r].double().reshape(KV, H // KV, d)
        p = torch.softmax(torch.matmul(q, kv[0].transpose(1, 2).contiguous()) / math.sqrt(d), -1)
        out.append(torch.matmul(p, kv[1]).reshape(H * d))
    return torch.stack(out)


def _exact_packed(s):
    c = s["case"]
    H, KV, d = c["heads"], c["kv_heads"], c["dim"]
    out, (new, keys) = [], _packed_lengths(c)
    for nq, nk, a, b in zip(new, keys, _prefix(new), _prefix(keys)):
        q = s["q"][a:a + nq].double().reshape(nq, H, d).transpose(0, 1)
        k, v = (x.double().reshape(nk, KV, d).transpose(0, 1) for x in s["kv"][b:b + nk].chunk(2, 1))
        hidden = torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1)
        o = []
        for h in range(H):
            x = (q[h] @ k[h * KV // H].T.contiguous() / math.sqrt(d)).masked_fill(hidden, -math.inf)
            o.append(torch.softmax(x, -1) @ v[h * KV // H])
        out.append(torch.stack(o, 1).reshape(nq, H * d))
    return torch.cat(out)


def _exact_sample(s):
    V = s["logits"].shape[1]
    host = {x: None if s[x] is None else s[x].double().cpu().numpy() for x in ("logits", "temperature", "top_k", "top_p", "min_p", "u")}
    ids = []
    for r, x in enumerate(host["logits"]):
        order = np.argsort(-x, kind="stable")
        T = host["temperature"][r]
        if T <= 0:
            ids.append(order[0])
            continue
        w = np.exp((x[order] - x[order[0]]) / T)
        n = V
        if host["top_k"] is not None:
            n = int(host["top_k"][r]) or V
            if host["top_p"][r] < 1:
                sums = np.cumsum(w[:n])
                n = min(n, int(np.searchsorted(sums, host["top_p"][r] * sums[-1])) + 1)
            n = min(n, max(1, int(np.count_nonzero(w >= host["min_p"][r]))))
        kept = np.sort(order[:n])
        sums = np.cumsum(np.exp((x[kept] - x[order[0]]) / T))
        ids.append(kept[min(len(kept) - 1, int(np.searchsorted(sums, host["u"][r] * sums[-1], side="right")))])
    return np.array(ids, dtype=np.int32)


_exact = {"plan": _exact_plan, "append": _exact_append, "attention": _exact_attention, "packed": _exact_packed, "sample": _exact_sample}


# --- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "plan":
        cached, fresh = _plan_lengths(case)
        tokens, ended = sum(max(f, 0) for f in fresh), sum(_pages(c) for c, f in zip(cached, fresh) if f < 0)
        new = sum(_pages(c + f) - _pages(c) for c, f in zip(cached, fresh) if f > 0)
        return {"bytes": 20 * len(cached) + 8 * tokens + 8 * ended + 8 * new, "flops": 0}
    if op == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * (4 if case["dtype"] == "float32" else 2) + 24), "flops": 2 * case["rows"] * case["vocab"]}
    H, KV, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "append":
        T = case["tokens"]
        held = 2 * 72 * d * KV / 64  # bytes of a position's keys and values, written once and read back once
        return {"bytes": T * (2 * (2 * H + 3 * KV) * d + 4 * case["rot"] + 8 + held + 4 * KV * d), "flops": T * (3 * (H + KV) * case["rot"] + 8 * KV * d)}
    if op == "attention":
        lengths = _ragged(case, case["requests"])
        return {"bytes": sum(lengths) * KV * 72 * d / 64 + case["requests"] * 4 * H * d, "flops": 4 * H * d * sum(lengths)}
    new, keys = _packed_lengths(case)
    pairs = sum(n * (k - n) + n * (n + 1) // 2 for n, k in zip(new, keys))
    return {"bytes": 4 * (sum(new) * H + sum(keys) * KV) * d, "flops": 4 * H * d * pairs}
