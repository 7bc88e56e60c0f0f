"""The cache in eight bits and attention for trees of drafted tokens: refusals, and what the host prepares (no GPU)."""
import numpy as np
import pytest
import torch

from llmx_b200 import ops
from llmx_b200.runtime import KernelError


def pages(n=4, g=2, page=16, dim=64):
    return ops.QuantizedPages.zeros(n, g, page, dim, "cpu")


def attention_args(rows=3, heads=4, g=2, dim=64, requests=2, dtype=torch.bfloat16, **changes):
    a = dict(q=torch.zeros(rows, heads * dim, dtype=dtype), cache=pages(g=g, dim=dim), out=torch.zeros(rows, heads * dim, dtype=dtype),
             row_start=torch.tensor([0, 1], dtype=torch.int32), row_count=torch.tensor([1, 2], dtype=torch.int32),
             history=torch.zeros(requests, dtype=torch.int32), block_tables=torch.zeros(requests, 3, dtype=torch.int32), heads=heads, kv_heads=g,
             head_dim=dim, window=None, scale=1.0, max_rows=2, max_context=4)
    a.update(changes)
    return a


def test_a_new_cache_is_rows_of_zeros():
    c = pages()
    assert c.codes.dtype is torch.float8_e4m3fn and int(c.codes.view(torch.uint8).max()) == 0 and set(c.exponents.flatten().tolist()) == {127}
    assert (c.pages, c.kv_heads, c.page_size, c.head_dim) == (4, 2, 16, 64)


@pytest.mark.parametrize("codes, exponents", [
    (torch.zeros(4, 2, 2, 16, 64, dtype=torch.uint8), torch.zeros(4, 2, 2, 16, dtype=torch.uint8)),
    (torch.zeros(4, 1, 2, 16, 64).to(torch.float8_e4m3fn), torch.zeros(4, 1, 2, 16, dtype=torch.uint8)),
    (torch.zeros(4, 2, 2, 16, 64).to(torch.float8_e4m3fn), torch.zeros(4, 2, 2, 15, dtype=torch.uint8)),
    (torch.zeros(4, 2, 2, 16, 64).to(torch.float8_e4m3fn), torch.zeros(4, 2, 2, 16)),
    (torch.zeros(4, 2, 2, 64, 16).to(torch.float8_e4m3fn).transpose(3, 4), torch.zeros(4, 2, 2, 16, dtype=torch.uint8)),
])
def test_quantized_pages_refuse(codes, exponents):
    with pytest.raises(KernelError, match="quantized pages"):
        ops.QuantizedPages(codes, exponents)


@pytest.mark.parametrize("what, changes", [
    ("heads", dict(k=torch.zeros(3, 1, 64), v=torch.zeros(3, 1, 64))),
    ("heads", dict(k=torch.zeros(3, 2, 32), v=torch.zeros(3, 2, 32))),
    ("one type", dict(v=torch.zeros(3, 2, 64, dtype=torch.bfloat16))),
    ("one after another", dict(k=torch.zeros(3, 64, 2).transpose(1, 2))),
    ("one after another", dict(v=torch.zeros(3, 4, 64)[:, ::2])),
    ("int32 slot", dict(slots=torch.zeros(3, dtype=torch.int64))),
    ("int32 slot", dict(slots=torch.zeros(2, dtype=torch.int32))),
    ("not one the kernels take", dict(k=torch.zeros(3, 2, 64, dtype=torch.float16), v=torch.zeros(3, 2, 64, dtype=torch.float16))),
    ("CUDA tensors", dict()),
])
def test_quantize_kv_refuses(what, changes):
    a = dict(k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), slots=torch.zeros(3, dtype=torch.int32), cache=pages())
    a.update(changes)
    with pytest.raises(KernelError, match=what):
        ops.quantize_kv(**a)


def test_quantize_kv_refuses_wide_heads():
    with pytest.raises(KernelError, match="256"):
        ops.quantize_kv(torch.zeros(1, 1, 257), torch.zeros(1, 1, 257), torch.zeros(1, dtype=torch.int32), pages(g=1, dim=257))


@pytest.mark.parametrize("what, changes", [
    ("page ids", dict(pages=torch.zeros(2, dtype=torch.int64))),
    ("page ids", dict(out=torch.zeros(3, 2, 2, 16, 64))),
    ("page ids", dict(out=torch.zeros(2, 2, 2, 64, 16).transpose(3, 4))),
    ("count per page", dict(used=torch.zeros(1, dtype=torch.int32))),
    ("count per page", dict(used=torch.zeros(2))),
    ("not one the kernels take", dict(out=torch.zeros(2, 2, 2, 16, 64, dtype=torch.float16))),
    ("CUDA tensors", dict()),
])
def test_dequantize_pages_refuses(what, changes):
    a = dict(cache=pages(), pages=torch.zeros(2, dtype=torch.int32), out=torch.zeros(2, 2, 2, 16, 64))
    a.update(changes)
    with pytest.raises(KernelError, match=what):
        ops.dequantize_pages(**a)


REFUSED = [
    ("one type", dict(out=torch.zeros(3, 256))),
    ("one type", dict(heads=3)),
    ("one type", dict(kv_heads=3)),
    ("one type", dict(q=torch.zeros(256, 3, dtype=torch.bfloat16).T)),
    ("a cache", dict(cache=pages(g=1))),
    ("a cache", dict(cache=pages(dim=32))),
    ("one per request", dict(row_count=torch.zeros(3, dtype=torch.int32))),
    ("one per request", dict(history=torch.zeros(2))),
    ("block tables", dict(block_tables=torch.zeros(1, 3, dtype=torch.int32))),
    ("block tables", dict(block_tables=torch.zeros(2, 3))),
    ("block tables", dict(block_tables=torch.zeros(3, 2, dtype=torch.int32).T)),
    ("bounds", dict(max_rows=-1)),
    ("bounds", dict(max_context=-1)),
    ("scale above 0", dict(scale=0.0)),
    ("scale above 0", dict(scale=-1.0)),
    ("scale above 0", dict(scale=float("nan"))),
    ("scale above 0", dict(scale=float("inf"))),
    ("scale above 0", dict(scale=1e39)),
    ("CUDA tensors", dict()),
]


@pytest.mark.parametrize("what, changes", REFUSED + [
    ("window", dict(window=0)),
    ("eight bits", dict(cache=torch.zeros(4, 2, 2, 16, 64, dtype=torch.bfloat16))),
    ("not one the kernels take", dict(q=torch.zeros(3, 256, dtype=torch.float16), out=torch.zeros(3, 256, dtype=torch.float16))),
])
def test_attention_quantized_refuses(what, changes):
    with pytest.raises(KernelError, match=what):
        ops.attention_quantized(**attention_args(**changes))


@pytest.mark.parametrize("what, changes", REFUSED + [
    ("words", dict(tree=torch.zeros(2, 1, dtype=torch.int32))),
    ("words", dict(tree=torch.zeros(3, 1, dtype=torch.int64))),
    ("words", dict(tree=torch.zeros(3, dtype=torch.int32))),
    ("words", dict(tree=torch.zeros(3, 0, dtype=torch.int32))),
    ("not one the kernels take", dict(cache=torch.zeros(4, 2, 2, 16, 64, dtype=torch.float16))),
])
def test_attention_tree_refuses(what, changes):
    a = attention_args(tree=torch.zeros(3, 1, dtype=torch.int32))
    a.update(changes)
    del a["window"]
    with pytest.raises(KernelError, match=what):
        ops.attention_tree(**a)


def test_tree_bits_name_a_token_and_what_it_continues():
    parents = [[-1, 0, 0, 2, -1], list(range(-1, 39))]
    bits = ops.tree_bits(parents).view(np.uint32)
    assert bits.shape == (45, 2)
    assert bits[:5, 0].tolist() == [0b1, 0b11, 0b101, 0b1101, 0b10000] and not bits[:5, 1].any()
    for i in range(40):                                   # a chain: every token before it
        assert int(bits[5 + i, 0]) | int(bits[5 + i, 1]) << 32 == (1 << (i + 1)) - 1
    assert ops.tree_bits([]).shape == (0, 1)


@pytest.mark.parametrize("parents", [[[0]], [[-1, 1]], [[-2]], [[-1], [-1, 3]]])
def test_tree_bits_refuse_what_no_tree_is(parents):
    with pytest.raises(KernelError, match="no earlier token"):
        ops.tree_bits(parents)


def test_a_cache_of_one_plane_is_refused_eight_bits():
    from llmx_b200.cache.manager import CacheManager, KVSpec
    with pytest.raises(ValueError, match="planes of their own"):
        CacheManager([KVSpec(2, 64, planes=1)], 16, 64, 2, kv_dtype=torch.float8_e4m3fn, device="cpu")


def test_the_managers_eight_bits():
    from llmx_b200.cache.manager import CacheManager, KVSpec
    m = CacheManager([KVSpec(2, 64), KVSpec(2, 64), KVSpec(2, 64, window=32)], 16, 64, 2, kv_dtype=torch.float8_e4m3fn, device="cpu")
    gi, entry = m.entry_storage(1)
    assert isinstance(entry, ops.QuantizedPages) and gi == 0 and (entry.pages, entry.kv_heads, entry.page_size, entry.head_dim) == (4, 2, 16, 64)
    assert m.storage_bytes() == 3 * 4 * 2 * 2 * 16 * 65


def test_models_with_other_mixers_are_refused_eight_bits():
    from configs import TINY_E
    from llmx_b200.engine.engine import StepError, _need_eight_bits
    from llmx_b200.registry import architecture_of
    from test_zamizen_config import CFG
    for config, refused in ((TINY_E, None), (CFG, "LatentAttention, MaskedAttention")):
        entry = architecture_of(config)
        model = entry.build(entry.config_cls.from_dict(config))
        if refused is None:
            _need_eight_bits(model, model.cache_entry_specs())
        else:
            with pytest.raises(StepError, match=refused):
                _need_eight_bits(model, model.cache_entry_specs())
