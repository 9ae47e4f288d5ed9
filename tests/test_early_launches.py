"""Kernels that are launched while the kernel in front of them still runs wait for it, and load nothing by instructions that the wait does not order.

The non-coherent load is for data that nobody writes during the kernel's life, which begins before the wait."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "native_sparse_attention_triton_b200", "csrc")
UNORDERED = re.compile(r"__ld(g|cs|cg|ca|lu)\(|ld\.global\.nc")


def _files():
    return {f: open(os.path.join(CSRC, f)).read() for f in sorted(os.listdir(CSRC)) if f.endswith((".cu", ".cuh", ".h"))}


def _body(text, at):
    """From `at` to the brace that closes the first one opened behind it."""
    start = text.index("{", at)
    depth = 0
    for i in range(start, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[at:i + 1]
    raise AssertionError("unbalanced")


def _function(name):
    for f, text in _files().items():
        m = re.search(r"(__device__|__global__)[^;{}]*\b" + name + r"\(", text)
        if m:
            return _body(text, m.end())
    raise AssertionError(name)


def test_kernels_that_wait():
    kernels = {}
    for f, text in _files().items():
        for m in re.finditer(r"__global__[^;{}]*?\b(\w+_kernel)\(", text):
            body = _body(text, m.end())
            if "wait_for_launch_before();" in body:
                kernels[m.group(1)] = body
    assert set(kernels) == {"paged_append_kernel", "evict_select_kernel", "evict_move_kernel", "paged_decode_kernel", "paged_weights_kernel",
                            "sink_fwd_tc_kernel", "sink_dq_tc_kernel", "sink_dkdv_tc_kernel", "sink_finish_kernel"}
    for name, body in kernels.items():
        assert not UNORDERED.search(body), name
        assert "__restrict__" not in body, name


@pytest.mark.parametrize("name", ["visible_rows", "count_tiles", "find_tile", "exact_decode_row", "find_sequence", "find_row_tile", "find_tile_of_rows",
                                  "end_of_rows", "lane_elements", "exact_query_row", "exact_key_row", "fill_row_table", "load_key_tile"])
def test_what_they_call(name):
    body = _function(name)
    assert not UNORDERED.search(body) and "__restrict__" not in body


def test_every_early_launch_is_of_such_a_kernel():
    """launch_early stands in the files of these kernels alone."""
    files = {f for f, text in _files().items() if re.search(r"\blaunch_early\(", text) and f != "host_util.h"}
    assert files == {"attn_bwd.cu", "paged_cache.cu", "paged_decode.cu", "sink_dkdv_tc.cu", "sink_dq_tc.cu", "sink_fwd_tc.cu"}
