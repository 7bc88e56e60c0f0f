"""Calls at the edges of what the operators of the cache in eight bits allow: bounds that lie above the counts.  Tolerances count the
roundings that test_quantized_cache_gpu.py names."""
import math

import pytest
import torch

from llmx_b200 import ops
from test_quantized_cache_gpu import BF16, DEV, Case, gpu


def close(c, got, r, weight_step, least, window=None):
    """Request r's rows of `got` (float64) against 64 bits: a weight's rounding is `weight_step` of it, and `least` of the largest product
    of a row and head for each key that it sees."""
    n, h = c.requests[r]
    half_step = 2.0 ** -8 if c.dtype is BF16 else 2.0 ** -24
    kv, ok = c.keys(r), c.seen(r, window)
    for head in range(c.heads):
        k, v = (kv[:, plane, head // (c.heads // c.g)] for plane in (0, 1))
        x = c.q[c.starts[r]:c.starts[r] + n, head * c.dim:(head + 1) * c.dim].double()
        s = (x @ k.T * c.scale).masked_fill(~ok, -math.inf)
        w = torch.softmax(s, dim=-1)
        o, size = w @ v, w @ v.abs()
        score_error = (c.dim + 8) * 2.0 ** -24 * c.scale * torch.where(ok, x.abs() @ k.abs().T, 0.0).amax(-1, keepdim=True)
        largest = (w[:, :, None] * v.abs().amax(-1)[None, :, None]).amax(1) * ok.sum(-1, keepdim=True)
        limit = half_step * o.abs() + size * (2 * score_error + weight_step + (n + h + 16) * 2.0 ** -23) + least * largest
        mine = got[c.starts[r]:c.starts[r] + n, head * c.dim:(head + 1) * c.dim]
        bad = ~((mine - o).abs() <= limit)
        assert not bool(bad.any()), (r, head, bad.nonzero()[:4].tolist(), mine[bad][:4], o[bad][:4], limit[bad][:4])


# ---- a request of fewer rows than the call's bound ------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("n", [1, 10, 64, 65, 100])
@pytest.mark.parametrize("h", [0, 1500])
@pytest.mark.parametrize("window", [None, 70])
def test_one_request_of_fewer_rows_than_the_bound(n, h, window):
    """100 rows at most, of which the device's count names n.  Weights are bfloat16 where the bound is a prompt's."""
    c = Case([(n, h)], 8, 2, 128, 16, BF16, seed=21, spare_rows=100 - n)
    q, out = c.q.to(DEV), torch.full_like(c.q.to(DEV), 7.0)
    ops.attention_quantized(q, c.cache, out, *c.device(), c.heads, c.g, c.dim, window, c.scale, 100, 100 + h)
    assert bool((out[n:] == 7.0).all())
    close(c, out.double().cpu(), 0, 2.0 ** -8, 0.0, window)


@gpu
@pytest.mark.parametrize("window", [None, 70])
def test_one_request_recorded_at_the_bound_and_replayed_with_fewer_rows(window):
    c = Case([(100, 800)], 8, 2, 128, 16, BF16, seed=22, spare_rows=0)
    q, out = c.q.to(DEV), torch.zeros_like(c.q.to(DEV))
    start, count, history, tables = c.device()

    def call():
        ops.attention_quantized(q, c.cache, out, start, count, history, tables, c.heads, c.g, c.dim, window, c.scale, 100, 900)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for n, h in ((100, 800), (1, 800), (64, 33), (10, 0), (65, 700), (0, 50), (100, 800)):
        count.fill_(n)
        history.fill_(h)
        out.fill_(7.0)
        graph.replay()
        assert bool((out[n:] == 7.0).all())
        c.requests = [(n, h)]
        close(c, out.double().cpu(), 0, 2.0 ** -8, 0.0, window)
