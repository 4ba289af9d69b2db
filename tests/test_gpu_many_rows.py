"""Calls of more (batch, kv head) rows than the workspace's fixed counter area has words, behind smaller calls that left
their keys and records where a larger call's counters would lie: what a call gives does not depend on what ran before."""

import numpy as np
import pytest
import torch

from common import PAGE
from test_gpu_select import attended, bridge_call, chosen64, close, queries, scores64
from test_gpu_tree import filled
from turbopolar_amd import _lib
from turbopolar_amd.kernels import PageSet, decode_attention, fp16_scale

pytestmark = pytest.mark.gpu
AREA = 65536 // 4  # words of the counter area


def repeated(small, rows):
    """``small``'s rows over and over, as a cache of ``rows`` rows."""
    index = [i % small.runtime._batch_size for i in range(rows)]
    return small.fork(rows=index), index


def split_step(device):
    """A decode step over more pages than one workgroup takes, whose records go behind the counter area."""
    cache = filled(device, "default", 1, 4, 4, PAGE * 400, seed=9)
    q = queries(device, 1, 4, 3)[:, :, None]
    k, v = (torch.ones((1, 4, 1, 128), dtype=torch.float16, device=device) for _ in range(2))
    return lambda: cache.decode_attention(q, k, v, 0.1)


def test_selection_behind_smaller_calls(device):
    small = filled(device, "default", 3, 8, 4, PAGE * 6 + 5, seed=1)
    q = queries(device, 3, 8, 2)
    want = chosen64(scores64(q, small.runtime.page_bounds())[0], 3, 1, 0)
    result = attended(q, small, want, fp16_scale(small.config.attention_scale))
    step = split_step(device)
    middle, at_middle = repeated(small, 700)
    big, at = repeated(small, 4200)
    assert len(at) * 4 > AREA > len(at_middle) * 4
    call = lambda cache, index: bridge_call(cache, q[index].contiguous(), cache.runtime.page_bounds(), 3, 1, 0)  # noqa: E731
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        outs = [call(big, at)]
        for between in (step, lambda: call(middle, at_middle), step):
            between()
            outs.append(call(big, at))
    torch.cuda.synchronize()
    for i, (out, selected) in enumerate(outs):
        assert np.array_equal(selected.cpu().numpy(), want[at]), i
        assert torch.equal(out, outs[0][0])
        close(out, result[at], f"call {i}")


def test_selection_in_a_graph(device):
    """More rows than one launch takes, captured and replayed with eager calls between."""
    small = filled(device, "fast", 2, 8, 4, PAGE * 6, seed=1)
    big, at = repeated(small, 4200)
    q = queries(device, 2, 8, 5)[at].contiguous()[:, :, None]
    call = lambda: big.selected_attention(q, 0.1, 3, 1, 0)  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    step = split_step(device)
    for seed in range(3):
        q.copy_(queries(device, 2, 8, 20 + seed)[at][:, :, None])
        out.zero_()
        graph.replay()
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


def test_any_number_of_rows(device):
    """The entry point alone: rows around a launch's, up to the most that a call takes, in one workspace, a call of few
    rows and many pages between, whose keys lie over what a larger area of counters would take."""
    L = _lib.lib()
    g = torch.Generator(device=device).manual_seed(1)

    def made(rows, pages):
        bounds = torch.randn((rows, 1, pages, 2, 128), generator=g, device=device).sort(dim=3).values.half().contiguous()
        return torch.randn((rows, 1, 128), generator=g, device=device).half(), bounds

    few = made(2, 20000)
    ws = torch.zeros(int(L.tp_select_workspace_bytes(65535, 1, 1, 3)), dtype=torch.uint8, device=device)
    assert ws.numel() >= int(L.tp_select_workspace_bytes(2, 1, 1, 20000))

    def call(q, bounds, n):
        rows, pages = bounds.shape[0], bounds.shape[2]
        out = torch.full((rows, 1, n), -1, dtype=torch.int32, device=device)
        st = L.tp_select_pages(q.data_ptr(), rows, 1, 1, bounds.data_ptr(), pages, pages, 0, 0, n, 0.1, out.data_ptr(),
                               ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        assert st == 0, L.tp_last_error()
        return out

    for rows in (AREA, AREA + 1, 2 * AREA, 2 * AREA + 1, 65535):
        q, bounds = made(rows, 3)
        got = [call(q, bounds, 1)]
        call(*few, 7)
        got.append(call(q, bounds, 1))
        want = scores64(q, bounds)[0].argmax(-1)[..., None]
        for out in got:
            assert np.array_equal(out.cpu().numpy(), want), rows


def test_decode_of_many_rows_in_splits(device):
    """Splits asked for where one workgroup a row is the default."""
    small = filled(device, "default", 3, 8, 4, PAGE * 6, seed=4)
    q = queries(device, 3, 8, 2)
    scale = fp16_scale(small.config.attention_scale)
    result = attended(q, small, np.broadcast_to(np.arange(6), (3, 4, 6)), scale)
    step = split_step(device)
    big, at = repeated(small, 4200)
    block, values, *_ = big.runtime.get_fused_attention_inputs()
    pages, many = PageSet(block, values), q[at].contiguous()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        outs = []
        for splits in (1, 2, 1):
            outs.append(decode_attention(many, pages, None, None, PAGE * 6, scale, pages_per_split=splits))
            step()
    torch.cuda.synchronize()
    for out in outs:
        close(out, result[at], "decode")
