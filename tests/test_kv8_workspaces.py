"""Workspaces of PagedKv8::attention: needed where one token looks at a long context, and then checked; none for no tokens.
Needs no GPU."""
import pytest

import gie

A, B, C, W, S, T, KS, VS = (0x10000 * i for i in range(1, 9))  # addresses that are never read


def problem(**k):
    return gie.PagedKv(**{**dict(batch=1, total_tokens=1, q_heads=8, kv_heads=2, head_dim=64, page_size=16, num_pages=8,
                                 max_pages=4096, max_new=1, max_len=65536, cache="int8"), **k})


@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("cache", ["int8", "fp8"])
def test_parts_need_a_workspace_and_it_is_checked(dim, cache):
    p = problem(head_dim=dim, cache=cache)
    need = gie.kv8_attention_workspace_size(p)
    assert need > 0 and need % 16 == 0
    for workspace, given, expect in ((W, need - 1, "WorkspaceTooSmall"), (None, 0, "WorkspaceTooSmall"),
                                     (None, need, "WorkspaceTooSmall"), (W + 4, need, "InvalidArgument")):
        with pytest.raises(gie.GieError) as e:
            gie.kv8_attention(p, A, C, W, KS, VS, S, S, T, B, workspace=workspace, ws_bytes=given)
        assert e.value.status == expect


def test_no_tokens_no_workspace():
    for batch in (0, 2):
        assert gie.kv8_attention_workspace_size(problem(batch=batch, total_tokens=0)) == 0
        assert gie.paged_attention_workspace_size(problem(batch=batch, total_tokens=0, cache="")) == 0
