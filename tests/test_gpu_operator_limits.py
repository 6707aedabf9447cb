"""The feature cache and the distillation loss at the ends of what they take: reads under way when their loader closes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_read_under_way_when_the_passes_close(ctx):
    """The consumer's stream is busy when the loader goes: its last read still finds the pages, which the allocator then gives away."""
    from aeon_b200 import _lib as L
    from aeon_b200.dataloader import _CachedPasses
    shape, size = (640, 64), 256
    g = torch.Generator("cuda")
    g.manual_seed(5)
    x = torch.randn((size,) + shape, generator=g, device="cuda")
    torch.cuda.synchronize()
    passes = _CachedPasses(0, "int8", [("audio", shape, L.F32)], size, 1)
    passes.add((("audio", x),))
    assert passes.restart()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(40):
            big = big @ big * 1e-3
        (_, got), = passes.next()
    codes = passes.caches["audio"].codes.numel()
    passes.close()
    del passes
    taken = [torch.full((codes,), 77, dtype=torch.uint8, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(got, x)  # add() has put the kept values into x
    del taken
