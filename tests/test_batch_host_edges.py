"""Several requests at once: refusals at the edges of what can be launched, the rotary tables' ramps (no GPU)."""
import ctypes
import math

import numpy as np
import pytest

from helpers import ptr
from test_batch_host import APPEND, PACKED, PAGED, ROWS, SAMPLE, changed, refused


@pytest.mark.parametrize("call", [
    # work-items of a launch that 32 bits do not hold, each within the ranges of the single numbers
    lambda awq, lib: lib.awq_paged_append(changed(awq.AwqPagedAppendArgs, APPEND, n_tokens=1 << 24), 1, None),
    lambda awq, lib: lib.awq_paged_rows(changed(awq.AwqPagedRowsArgs, ROWS, n_rows=1 << 26), 1, None),
    lambda awq, lib: lib.awq_packed_attention(changed(awq.AwqPackedAttentionArgs, PACKED, n_tokens=1 << 28, n_keys=1 << 28), 1, None),
    lambda awq, lib: lib.awq_paged_attention(changed(awq.AwqPagedAttentionArgs, PAGED, n_requests=1 << 23, workspace_bytes=1 << 40), 1, None),
    lambda awq, lib: lib.awq_sample(changed(awq.AwqSampleArgs, SAMPLE, n_rows=1 << 24, workspace_bytes=1 << 40), 2, None),
    lambda awq, lib: lib.awq_sample(changed(awq.AwqSampleArgs, SAMPLE, n_rows=1 << 23, workspace_bytes=1 << 40), 2, None),
    lambda awq, lib: lib.awq_sample(changed(awq.AwqSampleArgs, SAMPLE, n_rows=1 << 20, vocab=500000, ld=500000, workspace_bytes=1 << 50), 2, None),
], ids=["append", "rows", "packed", "paged", "sample", "choose", "scan"])
def test_more_work_than_a_launch_takes_is_refused(awq, lib, call):
    assert refused(lib, call(awq, lib), "too many")


def tables_of(awq, lib, spec, n):
    s = awq.AwqRotarySpec(*spec)
    cos, sin = np.zeros((n, spec[1] // 2), np.float32), np.zeros((n, spec[1] // 2), np.float32)
    awq.check(lib.awq_rotary_tables(ctypes.byref(s), n, ptr(cos), ptr(sin)))
    return cos, sin


def check_tables(got, f, amplitude):
    # half a step of binary32 below an amplitude of 2, and angles up to 3,000 that differ in the last bits of 64
    angle = np.arange(len(got[0]))[:, None] * f
    assert np.abs(got[0] - amplitude * np.cos(angle)).max() <= 2.0 ** -24 + 1e-11
    assert np.abs(got[1] - amplitude * np.sin(angle)).max() <= 2.0 ** -24 + 1e-11


RAMPS = [(128, 1e4, 16.0, 4096.0, 1.0, 32.0), (128, 1e6, 4.0, 32768.0, 1.0, 32.0), (64, 5e5, 8.0, 8192.0, 0.5, 3.0), (2, 1e4, 2.0, 100.0, 1.0, 32.0)]


@pytest.mark.parametrize("rot,base,factor,original,slow,fast", RAMPS, ids=str)
def test_rotary_ramp_over_the_number_of_turns(awq, lib, rot, base, factor, original, slow, fast):
    """as the YaRN paper has it: with r = original / wavelength, gamma = 0 below slow, 1 above fast, (r - slow) / (fast - slow) between them, a frequency f
    becomes (1 - gamma) f / factor + gamma f"""
    wavelength = 2 * math.pi * base ** (2.0 * np.arange(rot // 2) / rot)
    gamma = np.clip((original / wavelength - slow) / (fast - slow), 0.0, 1.0)
    f = (1 - gamma) * (2 * math.pi / wavelength) / factor + gamma * (2 * math.pi / wavelength)
    assert rot == 2 or ((gamma > 0) & (gamma < 1)).any()
    check_tables(tables_of(awq, lib, (awq.ROTARY_TURNS, rot, base, factor, original, slow, fast), 3000), f, 0.1 * math.log(factor) + 1)


@pytest.mark.parametrize("rot,base,factor,original,slow,fast", RAMPS[:3], ids=str)
def test_rotary_ramp_between_whole_indices(awq, lib, rot, base, factor, original, slow, fast):
    """the ramp over the index with its bounds rounded outwards, by the turns that a frequency of those indices makes"""
    low, high = (rot * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (fast, slow))
    low, high = math.floor(low), math.ceil(high)
    share = np.clip((np.arange(rot // 2) - low) / (high - low), 0.0, 1.0)
    f = base ** (-2.0 * np.arange(rot // 2) / rot)
    turns = [original * base ** (-2.0 * b / rot) / (2 * math.pi) for b in (high, low)]
    check_tables(tables_of(awq, lib, (awq.ROTARY_BANDS, rot, base, factor, original, *turns), 3000), f * (1 - share) + f / factor * share, 0.1 * math.log(factor) + 1)


@pytest.mark.parametrize("spec,words", [((5, 64, 1e4, 2, 4096, 32, 1), "bands"), ((5, 64, 1e4, 2, 0, 1, 32), "bands"), ((5, 64, 1e4, 0.5, 4096, 1, 32), "factor"),
                                        ((4, 64, 1e4, 2, 4096, 1, 32), "kind"), ((6, 64, 1e4, 2, 4096, 1, 32), "kind"), ((-1, 64, 1e4, 2, 4096, 1, 32), "kind")], ids=str)
def test_rotary_ramps_refuse(awq, lib, spec, words):
    s, out = awq.AwqRotarySpec(*spec), np.zeros((4, 32), np.float32)
    assert refused(lib, lib.awq_rotary_tables(ctypes.byref(s), 4, ptr(out), ptr(out)), words)
