"""What the host decides for calls at the edges of attention over pages (no GPU): the workspace, calls that are refused."""
import pytest

from llmx_b200 import ops, runtime


def call(requests=1, rows=1, max_rows=1, max_context=64, heads=32, kv_heads=8, dim=128, page=16, window=0, q=ops.BF16, cache=ops.E4M3, tree_words=0, pages=4096,
         total_context=0):
    """A call of the sizes named, its pointers aligned and of nothing."""
    pointers = [256] * 8 + [256 if tree_words else 0]
    return ops._CALL.pack(*pointers, q, cache, -(-max_context // page), tree_words, requests, rows, max_rows, max_context, total_context, pages, heads, kv_heads,
                          dim, page, window, 0, 1.0, 0, 0, 0, 0)


def room(**sizes):
    packed = call(**sizes)
    return runtime.sized(lambda: runtime.lib().llmx_pages_workspace(packed))


EXPANDED = 2 * 8 * 16 * 128 * 2          # bytes of an expanded page of 8 heads


# ---- prompts' pages -----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("context", [32768, 131072])
def test_room_for_prompts_goes_by_the_rows_that_there_are(context):
    """One prompt among 63 requests of a row each: requests of more than 16 rows are expanded (64 pairs of 4 heads), and 363 rows are
    at most 21 of those."""
    most = room(requests=64, rows=363, max_rows=300, max_context=context)
    assert 21 * (context // 16) * EXPANDED <= most <= 22 * (context // 16 + 32) * EXPANDED


def test_room_for_prompts_alone_is_theirs():
    assert room(requests=4, rows=4 * 512, max_rows=512, max_context=8192) >= 4 * 512 * EXPANDED
    one = room(requests=1, rows=512, max_rows=512, max_context=8192)
    assert 512 * EXPANDED <= one <= 600 * EXPANDED + 32 * 512 * 132 * 4 * 8
    assert room(requests=1, rows=512, max_rows=512, max_context=131072, window=1024) <= 200 * EXPANDED + 32 * 512 * 132 * 4 * 8


# ---- calls without a form -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", [ops.BF16, ops.F32])
@pytest.mark.parametrize("window", [0, 70])
def test_pages_of_other_types_are_attended_under_a_tree_alone(cache, window):
    packed = call(requests=2, rows=20, max_rows=10, cache=cache, window=window)
    assert runtime.lib().llmx_pages_attention(packed) != 0 and "under a tree alone" in runtime.last_error()
    assert runtime.lib().llmx_pages_workspace(packed) == 0
    assert cache == ops.F32 or room(requests=2, rows=20, max_rows=10, cache=cache, tree_words=1) > 0


# ---- engines ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("width, refused", [(256, False), (264, True)])
def test_an_engine_of_wide_heads_is_refused_before_its_first_step(width, refused):
    from configs import TINY_E
    from llmx_b200.engine.engine import StepError, _need_eight_bits
    from llmx_b200.registry import architecture_of
    entry = architecture_of(dict(TINY_E, head_dim=width))
    model = entry.build(entry.config_cls.from_dict(dict(TINY_E, head_dim=width)))
    if refused:
        with pytest.raises(StepError, match="256 values at most"):
            _need_eight_bits(model, model.cache_entry_specs())
    else:
        _need_eight_bits(model, model.cache_entry_specs())
