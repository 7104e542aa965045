"""Order of instructions in the kernels over a paged cache and of the log probabilities, read from their sources: what it guards against cannot be shown by running it."""
import re

import pytest

from test_kernel_order import CSRC, kernels


def _kernel(source, name):
    (body,) = [b for n, b in kernels(CSRC / source) if n == name]
    return body


def test_reads_ahead_of_the_wait_are_acquired():
    """A launch that reads starts, lengths, queries or pages without having waited for the one in front of it could find older copies in the SM's own cache: the
    acquiring load (and the proxy fence, for what copies read) comes before all of them."""
    merge = _kernel("paged_attention.cu", "merge_kernel")
    assert 0 < merge.index("acquire_ahead(c)") < min(merge.index(x) for x in ("sequence_by_warp(", "sequence(c,", "seen_of(", "cost_of(", "grid_dependency_wait()"))
    many = _kernel("paged_attention_tc.cu", "attention_tc_kernel")
    begin = re.search(r"if \(w\.beside\) \{\s*acquire_ahead\(c\);\s*asm volatile\(\"fence\.proxy\.async\.global;\" ::: \"memory\"\);\s*\} else grid_dependency_wait\(\);", many)
    assert begin and begin.end() < min(many.index(x) for x in ("sequence(c,", "c.q_start", "a.q)", "table[", "tma_load_2d("))
    # whoever comes next waits for this launch alone: it ends behind the one that it ran beside
    assert re.search(r"if \(w\.beside\) grid_dependency_wait\(\);\s*\}$", many)
    for source, name in (("paged_attention.cu", "paged_split_kernel"), ("paged_append.cu", "paged_append_kernel"), ("logprobs.cu", "token_logprobs_kernel")):
        body = _kernel(source, name)
        assert body.index("grid_dependency_wait()") < min([body.index(x) for x in ("sequence(c,", "a.tokens[", "entry_of(", "load8(p", "bulk_load_1d(") if x in body])


@pytest.mark.parametrize("source,name", [("paged_attention.cu", "paged_split_kernel"), ("paged_attention_tc.cu", "attention_tc_kernel"), ("logprobs.cu", "token_logprobs_kernel")])
def test_copies_in_flight_are_waited_for(source, name):
    """A block that gives up a bounded wait does not leave with its bulk copies in flight."""
    body = _kernel(source, name)
    loads = [m.start() for m in re.finditer(r"\b(tma_load_\dd|bulk_load_1d)\(", body)]
    assert loads and body.find("mbar_drain(", loads[-1]) > 0


def test_one_thread_writes_the_status():
    """A contradiction on the device is met by any number of threads, and the status word is host memory: it is behind a device word that one of them takes."""
    text = (CSRC / "paged.cuh").read_text()
    assert len(re.findall(r"atomicCAS\(c\.status, 0, 5\)", text)) == 1
    assert "== 0 && atomicExch(c.told, 1u) == 0) atomicCAS(c.status, 0, 5)" in text
    assert not any("status, 0, 5" in (CSRC / s).read_text() for s in ("paged_append.cu", "paged_attention.cu", "paged_attention.cuh", "paged_attention_tc.cu"))
    # and the flush that reports it clears that word
    assert "c.told = ctx->d_abort + 8;" in text and "cudaMemsetAsync(ctx->d_abort, 0, 64, ctx->stream)" in (CSRC / "ctx.cu").read_text()
