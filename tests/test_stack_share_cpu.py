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


TABLE = [[1, 2, 3, 4], [5, 6, 7, 8], [9, 10, 11, 12]]


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
