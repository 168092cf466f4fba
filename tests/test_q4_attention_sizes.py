"""Sizes of calls over a 4-bit cache at the end of what a launch takes, on the host."""
import pytest

from shiftaddllm_amd import native

E_INVAL = -1


def describe(*sizes):
    p = native.Q4AttentionPlan()
    return native.cabi().lutgemm_describe_q4_attention_plan(*sizes, p), p


@pytest.mark.parametrize("sizes", [(65535, 1, 257, 257, 32, 32), (65535, 1, 4096, 4096, 32, 32), (8192, 1, 2048, 2048, 32, 32), (65535, 33, 256, 256, 32, 64),
                                   (65535, 200, 64, 64, 128, 256)])
def test_launches_of_2_to_the_32_work_items_are_refused(sizes):
    """batch * kv_heads workgroups of 256 threads each; prompts: of 512 for every block that tokens may fall into."""
    assert describe(*sizes)[0] == E_INVAL
    batch, tokens, heads, kv_heads, head_dim, positions = sizes
    assert native.cabi().lutgemm_q4_attention_workspace(*sizes) == 0


@pytest.mark.parametrize("sizes", [(65535, 1, 256, 256, 32, 32), (65535, 33, 64, 64, 32, 64), (65535, 200, 16, 16, 128, 256)])
def test_sizes_just_below_are_taken(sizes):
    rc, p = describe(*sizes)
    assert rc == 0 and p.workgroups * p.threads < 1 << 32
