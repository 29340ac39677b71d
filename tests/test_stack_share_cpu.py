"""DecodeStack.share's page tables and what lives on behind it, on the CPU: tables, caches and positions are tensors, and no kernel runs."""

import gc
import types
import weakref

import pytest
import torch

from latent_amd import DecodeStack

PAGES, PAGE = 40, 4


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.fixture(autouse=True)
def no_capture(monkeypatch):
    """torch asks a device whether its stream is being captured."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def block(seed, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    cache = lambda: torch.randint(0, 100, (PAGES, PAGE, 2, 8), generator=g).to(dtype)  # noqa: E731
    codes = dtype != torch.float16
    scale = lambda: torch.rand((PAGES, 2, PAGE), generator=g) if codes else None  # noqa: E731
    return types.SimpleNamespace(k_cache=cache(), v_cache=cache(), k_scale=scale(), v_scale=scale(),
                                 workspace_size=lambda n, pages, prefix: 1000 + 8 * prefix)


def stack(pages, positions, blocks):
    s = DecodeStack.__new__(DecodeStack)
    s.T, s.attention, s.graph, s.prefix, s.norms = len(pages), blocks, None, None, None
    s.pages, s.positions = ints(pages), ints(positions)
    s.attention_workspace = torch.empty(1000, dtype=torch.uint8)
    return s


def held(s, b, n):
    """What slot b's first n positions hold in every cache."""
    rows = s.pages[b].long()[torch.arange(n) // PAGE]
    at = torch.arange(n) % PAGE
    got = []
    for a in s.attention:
        for c, z in ((a.k_cache, a.k_scale), (a.v_cache, a.v_scale)):
            got.append(c.float()[rows, at])
            if z is not None:
                got.append(z[rows, :, at])
    return got


TABLE = [[1, 2, 3, 4], [5, 6, 7, 8], [9, 10, 11, 12]]


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8, torch.float8_e4m3fn])
def test_slots_have_pages_of_their_own_again(dtype):
    s = stack(TABLE, [-1, -1, -1], [block(1, dtype), block(2, dtype)])
    s.share(ints([20, 21]))
    assert s.pages.tolist() == [[20, 21, 3, 4], [20, 21, 7, 8], [20, 21, 11, 12]]
    s.positions[1] = 11  # slot 1 is behind the prefix, the others idle
    before = held(s, 1, 11)
    prefix = [c[20:22].float().clone() for a in s.attention for c in (a.k_cache, a.v_cache)]
    s.share(None)
    assert s.prefix is None and s.pages.tolist() == TABLE
    assert all(torch.equal(a, b) for a, b in zip(before, held(s, 1, 11)))
    assert all(torch.equal(a, c[20:22].float()) for a, c in zip(prefix, (c for a in s.attention for c in (a.k_cache, a.v_cache))))


def test_another_prefix_and_none():
    s = stack(TABLE, [-1, -1, -1], [block(1)])
    s.share(ints([20, 21, 22]))
    s.share(ints([30]))
    assert s.pages.tolist() == [[30, 2, 3, 4], [30, 6, 7, 8], [30, 10, 11, 12]]
    s.share(ints([]))
    assert s.pages.tolist() == TABLE and s.prefix is None
    s.share(s.pages[0, :2])  # one slot's own pages
    assert s.pages.tolist() == [[1, 2, 3, 4], [1, 2, 7, 8], [1, 2, 11, 12]]
    s.share(s.pages[0, :3])  # more of them, from the table that this call puts back
    assert s.prefix.tolist() == [1, 2, 3] and s.pages[:, :3].tolist() == [[1, 2, 3]] * 3
    s.share(None)
    assert s.pages.tolist() == TABLE


def test_pages_that_were_given_away_or_never_there():
    """While slots share, a page that their tables named before may have become another slot's."""
    s = stack([[1, 2, 3, 4], [-1, 6, 7, 8], [9, 99, 11, 12]], [-1, -1, -1], [block(1)])
    s.share(ints([20, 21]))
    s.pages[0, 2:] = ints([9, 6])  # slots 2's and 1's first pages, which nobody used
    s.positions.copy_(ints([15, 9, -1]))
    before = [held(s, 0, 15), held(s, 1, 9)]
    s.share(None)
    # Who is under way and has no page of its own keeps the prefix's, an idle slot names none.
    assert s.pages.tolist() == [[1, 2, 9, 6], [20, 21, 7, 8], [-1, 99, 11, 12]]
    for b, n in ((0, 15), (1, 9)):
        assert all(torch.equal(x, y) for x, y in zip(before[b], held(s, b, n)))


def test_a_prefix_of_slots_pages_in_another_order():
    s = stack(TABLE, [-1, -1, -1], [block(1)])
    s.share(ints([6, 1]))
    s.positions.copy_(ints([9, 9, 9]))
    before = [held(s, b, 9) for b in range(3)]
    s.share(None)
    for b in range(3):
        assert all(torch.equal(x, y) for x, y in zip(before[b], held(s, b, 9))), b
    assert s.pages[2].tolist() == TABLE[2]


def test_slots_start_behind_the_prefix():
    s = stack(TABLE, [3, -1, -1], [block(1)])
    with pytest.raises(RuntimeError):
        s.start_behind(ints([1]))
    s.share(ints([20, 21]))
    s.start_behind(ints([2, 1]))
    assert s.positions.tolist() == [3, 8, 8]
    s.start_behind(ints([-1, 3]))
    s.start_behind(ints([]))
    assert s.positions.tolist() == [3, 8, 8]
    for bad in (torch.tensor([1]), ints([[1]]), torch.zeros(1)):
        with pytest.raises(ValueError):
            s.start_behind(bad)


def test_a_graph_keeps_what_it_reads():
    """share replaces scratch and prefix; a graph that was captured with the old ones may still be replayed by whoever has it."""
    s = stack(TABLE, [-1, -1, -1], [block(1)])
    s.share(ints([20, 21]))
    refs = [weakref.ref(s.prefix), weakref.ref(s.attention_workspace)]
    graph = types.SimpleNamespace(held=s._captured_operands())
    s.share(None)
    gc.collect()
    assert all(r() is not None for r in refs)
    del graph
    gc.collect()
    assert all(r() is None for r in refs)


def test_not_while_a_graph_is_captured(monkeypatch):
    s = stack(TABLE, [-1, -1, -1], [block(1)])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError):
        s.share(ints([20]))
    assert s.pages.tolist() == TABLE and s.prefix is None


def test_a_page_that_somebody_goes_on_reading_is_nobody_elses():
    """The prefix is slot 0's own pages; slot 1, which has none, keeps them when slot 0 has ended."""
    s = stack([[1, 2, 3, 4], [-1, -1, 7, 8], [9, 10, 11, 12]], [-1, -1, -1], [block(1)])
    s.share(s.pages[0, :2])
    s.positions.copy_(ints([-1, 9, 9]))
    before = [held(s, b, 9) for b in (1, 2)]
    s.share(None)
    assert s.pages.tolist() == [[-1, -1, 3, 4], [1, 2, 7, 8], [9, 10, 11, 12]]
    for b in (1, 2):
        assert all(torch.equal(x, y) for x, y in zip(before[b - 1], held(s, b, 9)))
