"""DecodeStack.share and back again: slots, graphs and tables afterwards, against stacks that never shared, bit for bit."""

import pytest
import torch

from tests.test_gpu_stack_cache8 import CACHES, _ints, _stack, _x, parts  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu
PREFIX = [59, 3, 41]


def _apart(gpu, parts, cache):
    """A stack whose slots' tables do not name the prefix's pages."""
    s = _stack(gpu, parts, 4, cache)
    rest = [p for p in range(60) if p not in PREFIX]
    s.pages.copy_(_ints(rest[:32]).view(4, 8))
    return s


@pytest.mark.parametrize("cache", CACHES)
def test_prompts_after_share_none_are_those_of_a_stack_that_never_shared(gpu, parts, cache):
    gen = torch.Generator(device="cuda").manual_seed(1)
    s, never = (_apart(gpu, parts, cache) for _ in range(2))
    x = _x(gen, 90)
    s.share(_ints(PREFIX))
    s.prompt(x[:48], _ints([0, 48]), _ints([3]))
    s.positions.fill_(-1)
    s.share(None)
    assert torch.equal(s.pages, never.pages)
    for t in (s, never):
        t.prompt(x, _ints([0, 50, 90]), _ints([2, 0]))
    for _ in range(3):
        x0 = _x(gen, 4)
        assert torch.equal(s.forward(x0), never.forward(x0))
    assert torch.equal(s.positions, never.positions)


@pytest.mark.parametrize("cache", CACHES)
def test_slots_under_way_go_on_after_share_none(gpu, parts, cache):
    gen = torch.Generator(device="cuda").manual_seed(2)
    s, never = (_apart(gpu, parts, cache) for _ in range(2))
    x = _x(gen, 48 + 25)
    s.share(_ints(PREFIX))
    s.prompt(x[:48], _ints([0, 48]), _ints([2]))
    s.start_behind(_ints([0, 1]))
    for b in range(3):
        never.prompt(x[:48], _ints([0, 48]), _ints([b]))
    assert torch.equal(s.positions, never.positions)
    for t in (s, never):
        t.prompt(x[48:], _ints([0, 5, 25]), _ints([1, 0]))
    s.share(None)
    assert torch.equal(s.pages, never.pages)
    for _ in range(3):
        x0 = _x(gen, 4)
        assert torch.equal(s.forward(x0), never.forward(x0))
    # One of them ends and another sequence takes its slot: the others' positions are theirs.
    for t in (s, never):
        t.positions[0] = -1
        t.prompt(x[:60], _ints([0, 60]), _ints([0]))
    for _ in range(3):
        x0 = _x(gen, 4)
        assert torch.equal(s.forward(x0), never.forward(x0))


@pytest.mark.parametrize("cache", ["16", "int8"])
def test_a_graphs_handle_outlives_share(gpu, parts, cache):
    gen = torch.Generator(device="cuda").manual_seed(3)
    s, still = (_apart(gpu, parts, cache) for _ in range(2))
    x = _x(gen, 48)
    for t in (s, still):
        t.share(_ints(PREFIX))
        t.prompt(x, _ints([0, 48]), _ints([2]))
        t.start_behind(_ints([0, 1]))
    graph = s.capture()
    s.share(None)
    junk = [torch.full((1 << n,), 0xFF, dtype=torch.uint8, device="cuda") for n in range(8, 24)]  # what was freed is somebody else's
    for _ in range(4):
        x0 = _x(gen, 4)
        s.load(x0)
        graph.replay()
        assert torch.equal(s.output, still.forward(x0))
        torch.cuda.synchronize()
        assert all(bool((j == 0xFF).all()) for j in junk)


def test_share_is_not_captured_and_waits_for_another_streams_steps(gpu, parts):
    gen = torch.Generator(device="cuda").manual_seed(4)
    s, other = (_apart(gpu, parts, "int8") for _ in range(2))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = torch.ones(4, device="cuda") + 1
        with pytest.raises(RuntimeError, match="captured"):
            s.share(None)
    g.replay()
    assert bool((y == 2).all())
    x = [_x(gen, 4) for _ in range(20)]
    for t in (s, other):
        t.share(_ints(PREFIX))
        t.start_behind(_ints(range(4)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x0 in x:
            s.forward(x0)
    s.share(None)  # with the side stream's steps under way
    junk = torch.full((1 << 24,), 0xFF, dtype=torch.uint8, device="cuda")
    want = [other.forward(x0) for x0 in x][-1]
    assert torch.equal(s.output, want) and bool((junk == 0xFF).all()) and s.positions.tolist() == [68] * 4
