"""The workspace of a draft-tree step's end serves every step of up to its requests and rows: its size never falls as
either grows."""
import pytest

import arcllm_amd as arc


def size(requests, tokens):
    return arc.tree_commit_workspace_bytes(arc.PagedBatch(requests, tokens))


@pytest.mark.parametrize("requests", [1, 3, 64, 65, 1000])
def test_more_rows_need_no_less(requests):
    sizes = [size(requests, n) for n in range(0, 9000)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))


def test_more_requests_need_no_less():
    sizes = [size(n, 200) for n in range(0, 3000)]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))


def test_room_for_the_most_parts():
    # rows of logits are read in up to 64 parts of 8 bytes each, of fewer than 4096 in all where rows are fewer than that
    assert size(1, 63) >= 63 * 64 * 8 and size(1, 64) >= 63 * 64 * 8 and size(1, 2048) >= 2047 * 2 * 8
