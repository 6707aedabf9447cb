"""Ends of the ranges that the feature cache and the distillation loss take, and what the loader's passes from the cache stand on, on a
machine without a GPU."""
import ctypes as C

import pytest
import torch

from aeon_b200 import _lib as L
from tests.test_operator_refusals import cache_desc, fake_context, loader_config

LARGEST_DIM = 2 ** 31 - 1024


@pytest.mark.parametrize("name", ["aeonb_cache_write", "aeonb_cache_read"])
@pytest.mark.parametrize("dim", [LARGEST_DIM + 1, 2 ** 31 - 512, 2 ** 31 - 128, 2 ** 31 - 1])
def test_groups_longer_than_lanes_can_step_through(name, dim):
    """A lane's next place, up to 512 values on, has to fit 32 bits with a sign, or it would pass for one inside the group again."""
    lib = L.load()
    call = getattr(lib, name)
    one = dict(dim=dim, heads=1, pages=1, page_tokens=1, seqs=1, tokens=1)
    assert call(fake_context(), C.byref(cache_desc(**one))) == L.ERR_INVALID
    assert "dim" in lib.aeonb_last_error().decode()
    assert call(fake_context(), C.byref(cache_desc(**dict(one, dim=LARGEST_DIM, seqs=0)))) == L.OK


def test_steps_of_the_largest_group():
    """The place behind a group's last chunk, for every width of chunk a lane takes (values at a time, lanes of a group)."""
    for values, lanes in ((16, 32), (8, 32), (4, 32)):
        step = values * lanes
        for dim in (LARGEST_DIM, LARGEST_DIM - values + 1):
            last = (dim - 1) // values * values  # of some lane
            assert last + step + values < 2 ** 31 and dim + values - 1 < 2 ** 31
    assert LARGEST_DIM + 4 * 32 + 3 * 32 < 2 ** 31  # values apart: four of a lane, 32 apart


def test_cached_pages_are_kept_until_their_reads_are_done(monkeypatch):
    """close() waits for the device before it lets go of anything that a read on the caller's stream may still use."""
    from aeon_b200.dataloader import _CachedPasses
    done = []

    class Held(dict):
        def clear(self):
            done.append("dropped")
            super().clear()

    class Context:
        device = 3

        def close(self):
            done.append("closed")

    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: done.append("waited for %d" % device))
    passes = _CachedPasses.__new__(_CachedPasses)
    passes.ctx, passes.caches, passes.tables, passes.kept = Context(), Held(audio=1), Held(audio=2), Held(label=[3])
    passes.close()
    assert done[0] == "waited for 3" and done.count("dropped") == 3 and done[-1] == "closed"
    assert not passes.caches and not passes.tables and not passes.kept


@pytest.mark.parametrize("changes", [dict(), dict(node_count=2, node_id=1), dict(block_size=4)])
def test_passes_that_differ_are_not_cached(changes):
    """shuffle_manifest deals a new order of the blocks at each reset, and each node other records: not what a first pass has kept."""
    from aeon_b200 import DataLoader
    from aeon_b200.dataloader import check_feature_cache
    with pytest.raises(ValueError, match="shuffle_manifest"):
        DataLoader(loader_config(shuffle_manifest=True, **changes))
    assert check_feature_cache(loader_config(shuffle_manifest=False, **changes)) == "int8"
    assert check_feature_cache(loader_config(feature_cache=None, shuffle_manifest=True, **changes)) is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab,row,at", [(29, 5000, 0), (29, 5001, 3), (500, 40000, 512), (1000, 4100, 1), (29, 36, 3), (1, 64, 0)])
def test_memory_of_a_gradient(dtype, vocab, row, at):
    """The gradient of some columns of longer rows takes the memory of the columns, not of the rows, and lies in its 16 bytes as they do."""
    from aeon_b200.kernels import _distill_grad_like
    size = torch.finfo(dtype).bits // 8
    for shape in ((64,), (4, 16), (1,)):
        logits = torch.empty(shape + (row,), dtype=dtype)[..., at:at + vocab]
        grad = _distill_grad_like(logits)
        assert grad.shape == logits.shape and grad.dtype == dtype
        assert grad.untyped_storage().nbytes() <= 5 * logits.numel() * size + 64 * 9 * size
        assert (grad.data_ptr() - logits.data_ptr()) % 16 == 0
        assert vocab == 1 or grad.stride(-1) == 1
        if shape != (1,):  # (one row is at no distance from another)
            assert (grad.stride(-2) - logits.stride(-2)) * size % 16 == 0 and grad.view(-1, vocab).stride(0) >= vocab
            assert grad.stride() == logits.stride() or row > 4 * vocab
        grad.fill_(1)
