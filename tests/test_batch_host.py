"""Several requests at once: what is refused before anything is launched, the cache's layout and the rotary tables (no GPU)."""
import ctypes

import numpy as np
import pytest

import batch_plain as plain
from helpers import host_program, ptr

P = 0x100000  # an address that nothing reads


def refused(lib, rc, words):
    return rc == 1 and words.encode() in lib.awq_last_error()


def changed(struct, good, **kw):
    a = struct(**good)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


PLAN = dict(cached=P, fresh=P, table=P, free_pages=P, free_in=P, free_out=P, lengths=P, starts=P, positions=P, slots=P, max_tokens=8,
            n_requests=4, max_pages=10, n_pages=50)


@pytest.mark.parametrize("kw,words", [
    (dict(n_requests=-1), "out of range"), (dict(max_pages=-1), "out of range"), (dict(n_pages=1 << 25), "out of range"),
    (dict(n_requests=70000, max_pages=1000), "too many"), (dict(max_tokens=-1), "max_tokens"), (dict(free_in=None), "NULL"),
    (dict(cached=None), "NULL"), (dict(table=None), "NULL"), (dict(slots=None), "NULL"), (dict(free_pages=None), "NULL")], ids=str)
def test_plan_refuses(awq, lib, kw, words):
    assert refused(lib, lib.awq_page_plan(changed(awq.AwqPagePlanArgs, PLAN, **kw), None), words)


APPEND = dict(q=P, q_out=P, k=P, k_out=P, v=P, cosines=P, sines=P, positions=P, slots=P, cache=P, ldq=1024, ldq_out=1024, ldk=256, ldk_out=256,
              ldv=256, n_tokens=3, max_pos=100, heads=8, kv_heads=2, dim=128, rot=64, interleaved=0, n_pages=5)


@pytest.mark.parametrize("kw,words", [
    (dict(dim=96), "64, 128 or 256"), (dict(kv_heads=0), "heads"), (dict(heads=7), "multiple of kv_heads"), (dict(rot=24), "rot"),
    (dict(rot=144), "rot"), (dict(rot=-16), "rot"), (dict(ldq=1000), "overlap"), (dict(ldq=1028), "16-byte"), (dict(q=P + 8), "16-byte"),
    (dict(ldq=1032), "one stride"), (dict(q_out=None), "q:"), (dict(ldk=128), "k:"), (dict(v=None), "append needs"), (dict(slots=None), "append needs"),
    (dict(k=None), "append needs"), (dict(cache=P + 4), "cache is"), (dict(cosines=None), "NULL"), (dict(sines=P + 4), "tables"),
    (dict(positions=None), "NULL"), (dict(n_pages=1 << 25), "out of range"), (dict(n_tokens=-1), "out of range"), (dict(ldv=250), "v:")], ids=str)
def test_append_refuses(awq, lib, kw, words):
    assert refused(lib, lib.awq_paged_append(changed(awq.AwqPagedAppendArgs, APPEND, **kw), 3, None), words)


ROWS = dict(cache=P, table=P, first=P, lengths=P, starts=P, k=P, v=P, ldk=256, ldv=256, n_rows=4, n_requests=2, max_pages=3, n_pages=5, kv_heads=2, dim=128)


@pytest.mark.parametrize("kw,words", [
    (dict(dim=32), "64, 128 or 256"), (dict(cache=None), "NULL"), (dict(starts=None), "NULL"), (dict(ldk=248), "overlap"), (dict(ldv=260), "16-byte"),
    (dict(k=P + 2), "16-byte"), (dict(n_rows=-1), "out of range"), (dict(max_pages=-1), "out of range")], ids=str)
def test_rows_refuse(awq, lib, kw, words):
    assert refused(lib, lib.awq_paged_rows(changed(awq.AwqPagedRowsArgs, ROWS, **kw), 1, None), words)


PAGED = dict(q=P, cache=P, table=P, lengths=P, ctx=P, workspace=P, ldq=1024, ldc=1024, workspace_bytes=1 << 30, n_requests=2, max_pages=3, n_pages=5, heads=8,
             kv_heads=2, dim=128, scale=0.1)


@pytest.mark.parametrize("kw,words", [
    (dict(dim=80), "64, 128 or 256"), (dict(heads=9), "multiple"), (dict(kv_heads=0), "multiple"), (dict(n_requests=-1), "range"), (dict(q=None), "NULL"),
    (dict(table=None), "NULL"), (dict(workspace=None), "NULL"), (dict(workspace=P + 8), "16-byte"), (dict(ldc=1020), "16-byte"), (dict(ldq=512), "overlap"),
    (dict(workspace_bytes=100), "too small"), (dict(scale=float("nan")), "scale"), (dict(n_requests=1 << 20, max_pages=1 << 20), "range")], ids=str)
def test_paged_attention_refuses(awq, lib, kw, words):
    assert refused(lib, lib.awq_paged_attention(changed(awq.AwqPagedAttentionArgs, PAGED, **kw), 3, None), words)


PACKED = dict(q=P, k=P, v=P, ctx=P, q_starts=P, k_starts=P, ldq=1024, ldk=256, ldv=256, ldc=1024, n_tokens=9, n_keys=20, n_requests=2, heads=8, kv_heads=2,
              dim=128, causal=1, scale=0.1)


@pytest.mark.parametrize("kw,words", [
    (dict(dim=512), "64, 128 or 256"), (dict(heads=3), "multiple"), (dict(n_tokens=-1), "out of range"), (dict(k_starts=None, n_keys=5), "starts of their own"),
    (dict(k=None), "NULL"), (dict(q_starts=None), "NULL"), (dict(ldv=252), "16-byte"), (dict(ctx=P + 8), "16-byte"), (dict(ldk=128), "overlap"), (dict(scale=float("inf")), "scale"),
    (dict(ldv=(1 << 25) + 8), "apart")], ids=str)
def test_packed_attention_refuses(awq, lib, kw, words):
    assert refused(lib, lib.awq_packed_attention(changed(awq.AwqPackedAttentionArgs, PACKED, **kw), 1, None), words)


SAMPLE = dict(logits=P, uniform=P, ids=P, workspace=P, ld=1000, vocab=1000, n_rows=3, workspace_bytes=1 << 30)


@pytest.mark.parametrize("kw,words", [
    (dict(vocab=0), "out of range"), (dict(vocab=524289, ld=600000), "out of range"), (dict(n_rows=-1), "out of range"), (dict(uniform=None), "NULL"),
    (dict(ids=None), "NULL"), (dict(ld=999), "overlap"), (dict(workspace=P + 8), "misaligned"), (dict(logits=P + 2), "misaligned"),
    (dict(workspace_bytes=10), "too small")], ids=str)
def test_sample_refuses(awq, lib, kw, words):
    assert refused(lib, lib.awq_sample(changed(awq.AwqSampleArgs, SAMPLE, **kw), 2, None), words)


def test_number_formats(awq, lib):
    """the cache's operators take 16-bit activations, sampling binary32 too; awq_open does not know binary16"""
    for dtype in (0, 2, 4):
        assert refused(lib, lib.awq_paged_append(changed(awq.AwqPagedAppendArgs, APPEND), dtype, None), "binary16")
        assert refused(lib, lib.awq_paged_rows(changed(awq.AwqPagedRowsArgs, ROWS), dtype, None), "binary16")
        assert refused(lib, lib.awq_paged_attention(changed(awq.AwqPagedAttentionArgs, PAGED), dtype, None), "binary16")
        assert refused(lib, lib.awq_packed_attention(changed(awq.AwqPackedAttentionArgs, PACKED), dtype, None), "binary16")
    assert refused(lib, lib.awq_sample(changed(awq.AwqSampleArgs, SAMPLE), 4, None), "dtype")
    options, handle = awq.AwqOpenOptions(awq.DTYPE_FLOAT16, 0, 0), ctypes.c_void_p()
    assert refused(lib, lib.awq_open(b"/nowhere", ctypes.byref(options), ctypes.byref(handle)), "unknown dtype")


def test_nothing_to_do_needs_no_device(awq, lib):
    assert lib.awq_paged_append(changed(awq.AwqPagedAppendArgs, APPEND, n_tokens=0), 1, None) == 0
    assert lib.awq_paged_rows(changed(awq.AwqPagedRowsArgs, ROWS, n_rows=0), 1, None) == 0
    assert lib.awq_paged_attention(changed(awq.AwqPagedAttentionArgs, PAGED, n_requests=0), 1, None) == 0
    assert lib.awq_packed_attention(changed(awq.AwqPackedAttentionArgs, PACKED, n_tokens=0), 1, None) == 0
    assert lib.awq_sample(changed(awq.AwqSampleArgs, SAMPLE, n_rows=0), 2, None) == 0
    for call in (lib.awq_page_plan, ):
        assert refused(lib, call(None, None), "args is NULL")
    for call in (lib.awq_paged_append, lib.awq_paged_rows, lib.awq_paged_attention, lib.awq_packed_attention, lib.awq_sample):
        assert refused(lib, call(None, 1, None), "args is NULL")


def test_sizes(lib):
    assert lib.awq_page_bytes(8, 128) == 8 * 72 * 128 and lib.awq_page_bytes(0, 128) == 0 and lib.awq_page_bytes(2, 96) == 0
    for n, heads, kv, dim, width in [(1, 8, 8, 64, 1), (64, 32, 8, 128, 640), (3, 40, 2, 256, 9), (1000, 1, 1, 64, 3)]:
        size = lib.awq_paged_workspace_bytes(n, heads, kv, dim, width)
        assert size > 0 and size % 16 == 0
    assert lib.awq_paged_workspace_bytes(2, 9, 2, 128, 4) == 0 and lib.awq_sample_workspace_bytes(1, 0) == 0
    assert lib.awq_sample_workspace_bytes(3, 524288) > lib.awq_sample_workspace_bytes(3, 1) > 0


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_layout_and_bad_pages(lib, tmp_path, dim):
    """every nibble and parameter of a head's part of a page has a place of its own; entries and slots outside the cache hold nothing"""
    program = """
#include <stdio.h>
#include "batch.hpp"
int main() {
  for (int i = 0; i < %d; ++i) printf("%%d %%d\\n", key_nibble(%d, i), value_nibble(%d, i));
  for (int v = 0; v < 2; ++v) for (int g = 0; g < %d / 64; ++g) for (int w = 0; w < 2; ++w) for (int p = 0; p < 64; ++p)
    printf("%%d\\n", page_parameter(%d, v, g, w, p));
  int n = 7;
  for (int e : {-2147483647 - 1, -1, 0, 6, 7, 2147483647}) printf("%%d\\n", held_page(e, n));
  for (int s : {-2147483647 - 1, -1, 0, 63, 64, 447, 448, 2147483647}) printf("%%d\\n", slot_page(s, n));
  printf("%%lld\\n", (long long)page_head_bytes(%d));
}""" % ((dim,) * 6)
    got = host_program(tmp_path, program)
    keys, values, got = got[0:2 * dim:2], got[1:2 * dim:2], got[2 * dim:]
    assert keys == plain.key_order(dim).tolist() and values == plain.value_order(dim).tolist()
    assert sorted(keys) == sorted(values) == list(range(dim))
    n = 2 * dim // 64 * 2 * 64
    assert sorted(got[:n]) == list(range(64 * dim, 72 * dim, 2))
    assert got[n:] == [-1, -1, 0, 6, -1, -1] + [-1, -1, 0, 0, 1, 6, -1, -1] + [72 * dim]


@pytest.mark.parametrize("spec", [(0, 128, 1e4, 1.0, 0, 0, 0), (0, 2, 1e4, 1.0, 0, 0, 0), (1, 64, 5e5, 8.0, 0, 0, 0), (2, 96, 1e4, 4.0, 0, 0, 0),
                                  (3, 128, 1e4, 16.0, 4096, 1, 32), (3, 64, 1e6, 1.0, 32768, 1, 32)], ids=str)
def test_rotary_tables(awq, lib, spec):
    kind, rot, base, factor, original, slow, fast = spec
    n = 3000
    s = awq.AwqRotarySpec(kind, rot, base, factor, original, slow, fast)
    cos, sin = np.zeros((n, rot // 2), np.float32), np.zeros((n, rot // 2), np.float32)
    awq.check(lib.awq_rotary_tables(ctypes.byref(s), n, ptr(cos), ptr(sin)))
    want = plain.rotary(kind, rot, n, base, factor, original, slow, fast)
    # half a step of binary32 below an amplitude of 2, and angles up to 3,000 that differ in the last bits of 64
    for got, w in zip((cos, sin), want):
        assert np.abs(got - w).max() <= 2.0 ** -24 + 1e-11


@pytest.mark.parametrize("spec,words", [((4, 64, 1e4, 1, 0, 0, 0), "kind"), ((0, 63, 1e4, 1, 0, 0, 0), "rot"), ((0, 64, 1.0, 1, 0, 0, 0), "base"),
                                        ((1, 64, 1e4, 0.5, 0, 0, 0), "factor"), ((1, 64, 1e4, float("nan"), 0, 0, 0), "factor"),
                                        ((2, 2, 1e4, 2, 0, 0, 0), "pair"), ((3, 64, 1e4, 2, 4096, 32, 1), "bands"), ((3, 64, 1e4, 2, 0, 1, 32), "bands")], ids=str)
def test_rotary_tables_refuse(awq, lib, spec, words):
    s = awq.AwqRotarySpec(*spec)
    assert refused(lib, lib.awq_rotary_tables(ctypes.byref(s), 4, P, P), words)
    s = awq.AwqRotarySpec(0, 64, 1e4, 1, 0, 0, 0)
    assert refused(lib, lib.awq_rotary_tables(ctypes.byref(s), 4, None, P), "NULL")
