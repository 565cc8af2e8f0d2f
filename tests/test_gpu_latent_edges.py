"""The MLA latent-cache operators where calls, streams and values meet: cases beside those of test_gpu_latent.py."""

import math

import pytest
import torch

from test_gpu_latent import (E4M3, SCALE, assert_attention, check, filled_cache, run_attention, slots_of, tables)

pytestmark = pytest.mark.gpu


def test_an_error_that_another_stream_records_while_parts_are_merged(cuda_device):
    """Attention whose parts are merged, beside a stream that records a bad slot at some moment of it: the call is done or
    skipped as a whole, the error is reported, and the next call is right."""
    from pithtrain_b200 import kernels
    from pithtrain_b200.operators.mla import LatentCache, latent_attention, latent_cache_write
    g = torch.Generator(device="cuda").manual_seed(60)
    lens = [3000, 1, 2500, 700]
    cache, table = filled_cache(g, lens, 64, torch.bfloat16)
    q = torch.randn(4, 1, 16, 576, generator=g, device="cuda").bfloat16()
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    other = LatentCache.allocate(1, 16)
    x = torch.ones(1, 1, 576, device="cuda", dtype=torch.bfloat16)
    cos, sin = tables(1)
    bad = torch.full((1, 1), 16, device="cuda")
    w = torch.ones(512, device="cuda")
    attend = lambda: latent_attention(q, cache, table, n, SCALE)  # noqa: E731
    record = lambda: latent_cache_write(other, bad, x[..., :512], x[..., 512:], w, cos, sin, 1e-6)  # noqa: E731
    attend()
    torch.cuda.synchronize()
    graphs = []
    for call, times in ((attend, 20), (record, 1)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(times):
                call()
        graphs.append(graph)
    side = torch.cuda.Stream()
    for i in range(40):
        with torch.cuda.stream(side):
            torch.cuda._sleep(5000 * i)
            graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="a slot given"):
            kernels.check_device_status()
    assert_attention(q, cache, table, lens, SCALE)
