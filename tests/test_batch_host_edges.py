"""Several requests at once: refusals at the edges of what can be launched (no GPU)."""
import pytest

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
