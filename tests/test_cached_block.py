"""A block over a cache: what it refuses, and that a refused call leaves the cache
as it was."""
import pytest
import torch

from headshot_amd.aggregator import BlockWeights, block_forward_cached
from headshot_amd.paged import PagedKV

DEV = "cuda:0"


def i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def cache(lens, device, dtype=torch.float16):
    table = torch.arange(4 * len(lens), dtype=torch.int32, device=device).reshape(len(lens), 4)
    kv = torch.zeros(2, 4 * len(lens), 2, 16, 64, dtype=dtype, device=device)
    return PagedKV(kv[0], kv[1], table, i32(lens, device))


@pytest.mark.parametrize("lens", [[8, 3], [5, 4], [5, 2], [0, 0], [-5, 3]])
def test_prompt_into_held_sequences(lens):
    """Sequences that hold keys before their prompt, or not all of its. (Nothing
    runs: no context is needed.)"""
    with pytest.raises(AssertionError, match="empty sequences"):
        block_forward_cached(None, None, torch.zeros(8, 128), cache(lens, "cpu"), 2, offsets=i32([0, 5, 8], "cpu"))


def test_prompt_offsets():
    for offsets in (i32([0, 8], "cpu"), i32([0, 5, 8], "cpu").long(), i32([[0, 5, 8]], "cpu"), i32([0, 5, 8], "meta")):
        with pytest.raises(AssertionError, match="offsets wants"):
            block_forward_cached(None, None, torch.zeros(8, 128), cache([5, 3], "cpu"), 2, offsets=offsets)


def block(dim=128):
    gen = torch.Generator(device=DEV).manual_seed(5)
    w = BlockWeights.random(dim, 2 * dim, 64, torch.float16, DEV, gen, ls_init=0.1)
    return w, torch.randn((8, dim), generator=gen, device=DEV).half()


@pytest.mark.gpu
def test_second_prompt_is_refused(ctx):
    w, x = block()
    c, offsets = cache([5, 3], DEV), i32([0, 5, 8], DEV)
    first = block_forward_cached(ctx, w, x, c, 2, offsets=offsets)
    kept = c.k.clone(), c.v.clone()
    c.lens += i32([5, 3], DEV)
    with pytest.raises(AssertionError, match="empty sequences"):
        block_forward_cached(ctx, w, x, c, 2, offsets=offsets)
    assert torch.equal(c.k, kept[0]) and torch.equal(c.v, kept[1])
    c.lens.copy_(i32([5, 3], DEV))
    assert torch.equal(block_forward_cached(ctx, w, x, c, 2, offsets=offsets, check=False), first)


@pytest.mark.gpu
def test_captured_prompt(ctx):
    """A prompt can be captured (unchecked) and follows its offsets and lens."""
    w, x = block()
    c, offsets = cache([5, 3], DEV), i32([0, 5, 8], DEV)
    block_forward_cached(ctx, w, x, c, 2, offsets=offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = block_forward_cached(ctx, w, x, c, 2, offsets=offsets)
    for cut in (5, 0, 8, 2):
        offsets.copy_(i32([0, cut, 8], DEV))
        c.lens.copy_(i32([cut, 8 - cut], DEV))
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        assert torch.equal(got, block_forward_cached(ctx, w, x, c, 2, offsets=offsets)), f"cut {cut}"
