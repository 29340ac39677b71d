"""Consecutive LATENT MoE layers decoded as one HIP graph.

Each layer l routes its tokens with its own router and adds the expert FFN to
the residual stream:

    ids_l, w_l = top-k(softmax(x_l . W_r[l]))
    y_l        = sum_k w_l * LATENT_FFN_l(x_l)          (latent_moe_ffn_forward)
    x_{l+1}    = x_l + y_l

With attention blocks each layer first lets its tokens read the sequences'
caches (the new token's own key and value among them):

    h_l        = x_l + Attention_l(x_l)                 (latent_kv_append, latent_attn_decode)

and h_l takes x_l's place above.  Row b of a step is the next token of the
sequence in slot b, at positions[b]; a slot whose position is negative is idle.
A slot whose pages (or whose rotation table) end before its position keeps what
is cached and stores nothing more; behind its pages it attends to what is there,
behind the table its attention is zeros.
`prompt` runs whole prompts, or chunks of them, through the same layers and
leaves the slots ready to decode.  After `share` the slots' first pages are the
same ones, which a step reads once for all slots (latent_attn_decode_shared);
`start_behind` puts slots behind them.

With norms each block, attention and experts alike, reads pre(x) and adds
scale gate post(y) to the stream, in one launch with the next block's pre
(latent_residual_norm):

    x' = x + s g post(Block(pre(x)))

The residual stream stays fp32 on the device; the stack's own buffers are
allocated once (an attention block's projections come from torch's allocator,
from a graph's pool when captured), so the whole stack (2 router kernels + the expert FFN + one add per layer, and
the attention's) can be captured in a torch.cuda.CUDAGraph (a HIP graph) and
replayed.  This is the stacked decode of a llama.cpp graph built by
build_moe_ffn_latent (README.md:111-113): the MoE blocks alone, or with the
attention that graph has between them.
"""

from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from .attention import _CODES, Attention
from .moe import StackedLayer, moe_forward, workspace_size
from .norm import BlockNorm, residual_norm
from .router import Router, route


class DecodeStack:
    def __init__(self, layers: Sequence[StackedLayer], routers: Sequence[Router], n_tokens: int,
                 attention: Optional[Sequence[Attention]] = None, max_pages: int = 0,
                 norms: Optional[Sequence[BlockNorm]] = None):
        """norms: one for each block in their order, a layer's attention (if there is any) and its experts."""
        if len(layers) != len(routers) or not layers:
            raise ValueError("need one router per layer")
        d, k = layers[0].d, routers[0].k
        for L, r in zip(layers, routers):
            if L.d != d or r.n_embd != d or r.n_expert != L.n_expert or r.k != k:
                raise ValueError("layers and routers must share d, k and match expert counts")
        self.layers, self.routers = list(layers), list(routers)
        self.T, self.d, self.k = int(n_tokens), d, k
        dev = layers[0].gate_a.codes.device
        n = len(layers)
        self.x = [torch.zeros((self.T, d), dtype=torch.float32, device=dev) for _ in range(n + 1)]
        self.y = [torch.empty((self.T, d), dtype=torch.float32, device=dev) for _ in range(n)]
        self.ids = [torch.empty((self.T, k), dtype=torch.int32, device=dev) for _ in range(n)]
        self.w = [torch.empty((self.T, k), dtype=torch.float32, device=dev) for _ in range(n)]
        self.logits = [torch.empty((self.T, r.n_expert), dtype=torch.float32, device=dev) for r in routers]
        # One zero-filled workspace shared by every layer (calls are stream ordered
        # and each call leaves the control block zero).
        need = max(workspace_size(L, self.T, k) for L in layers)
        self.workspace = torch.zeros((max(need, 256),), dtype=torch.uint8, device=dev)
        for r in self.routers:
            r.workspace(self.T)
        self.graph: Optional[torch.cuda.CUDAGraph] = None
        self.attention: Optional[List[Attention]] = None
        if attention is not None:
            self._add_attention(list(attention), int(max_pages), dev)
        elif max_pages:
            raise ValueError("max_pages without attention")
        self.norms: Optional[List[BlockNorm]] = None
        if norms is not None:
            self.norms = list(norms)
            per = 1 if self.attention is None else 2
            if len(self.norms) != per * n:
                raise ValueError(f"need {per * n} norms, one for each block")
            if not all(isinstance(b, BlockNorm) for b in self.norms):
                raise TypeError("norms must be BlockNorm")

    def _add_attention(self, blocks: List[Attention], max_pages: int, dev: torch.device) -> None:
        if len(blocks) != len(self.layers):
            raise ValueError("need one attention block per layer")
        for a in blocks:
            if a.n_embd != self.d or a.k_cache.shape[:2] != blocks[0].k_cache.shape[:2] or a.w_qkv.device != dev:
                raise ValueError("attention blocks must share d, the pages' number and size, and the layers' device")
        caches = [t.data_ptr() for a in blocks for t in (a.k_cache, a.v_cache) if t.numel()]
        if len(set(caches)) != len(caches):
            raise ValueError("each layer's attention block needs a cache of its own: layers that share one overwrite each other's keys")
        if max_pages <= 0:
            raise ValueError("max_pages must be positive")
        self.attention = blocks
        # Slot b's pages (of every layer's cache alike) and its next token's position; negative: idle.
        self.pages = torch.full((self.T, max_pages), -1, dtype=torch.int32, device=dev)
        self.positions = torch.full((self.T,), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros((self.T,), dtype=torch.int32, device=dev)
        self.h = [torch.empty((self.T, self.d), dtype=torch.float32, device=dev) for _ in blocks]
        self.prefix: Optional[torch.Tensor] = None
        self.attention_workspace = self._attention_scratch(None)

    def _attention_scratch(self, prefix: Optional[torch.Tensor]) -> torch.Tensor:
        pages = 0 if prefix is None else prefix.numel()
        need = max(a.workspace_size(self.T, self.pages.shape[1], pages) for a in self.attention)
        return torch.empty((max(need, 16),), dtype=torch.uint8, device=self.pages.device)

    def share(self, prefix: Optional[torch.Tensor]) -> None:
        """From now on the first P pages of every slot are those that prefix (int32 [P], P <= max_pages) names, of every
        layer's cache alike: pages[:, :P] is set to them, and steps read them once for all slots.  Whoever fills them does so
        through a slot, by `prompt`: an idle slot's prompt starts at position 0, in the shared pages.  A slot that is to go on behind
        them, with a prompt or a step, is put there by `start_behind`.
        None, or another prefix: first the slots' columns name again what they did before, and a slot
        under way takes a copy of the prefix there; where its page is another slot's by now, or there was none, it keeps the prefix's,
        and an idle slot names none.  The call waits for the device, whose steps under way, on whatever stream, read
        what it replaces, so it cannot be part of a capture.  A captured graph is dropped; who has it by its handle may still replay
        it, over the prefix that it was captured with."""
        if self.attention is None:
            raise RuntimeError("this stack has no attention")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("share cannot be captured")
        if prefix is not None:
            if prefix.dtype != torch.int32 or prefix.dim() != 1 or prefix.device != self.pages.device or prefix.numel() > self.pages.shape[1]:
                raise ValueError(f"prefix must be int32 [pages] on {self.pages.device}, at most {self.pages.shape[1]} of them")
            prefix = prefix.clone() if prefix.numel() else None
        workspace = self._attention_scratch(prefix)
        if self.pages.is_cuda:
            torch.cuda.synchronize(self.pages.device)
        if self.prefix is not None:
            self._unshare()
        self.graph = None
        self.prefix, self.attention_workspace = prefix, workspace
        if prefix is not None:
            self._own = self.pages[:, :prefix.numel()].clone()
            self.pages[:, :prefix.numel()] = prefix

    def start_behind(self, slots: torch.Tensor) -> None:
        """Puts these slots (int32 [B]; others than 0 .. n_tokens - 1 are left out), idle or not, at the first position behind the shared prefix."""
        if self.attention is None or self.prefix is None:
            raise RuntimeError("this stack shares no prefix")
        if slots.dtype != torch.int32 or slots.dim() != 1 or slots.device != self.positions.device:
            raise ValueError(f"slots must be int32 [slots] on {self.positions.device}")
        rows = torch.arange(self.T, dtype=torch.int32, device=slots.device)
        self.positions.masked_fill_((rows[:, None] == slots).any(1), self.prefix.numel() * self.attention[0].k_cache.shape[1])

    def _unshare(self) -> None:
        own, P = self._own, self.prefix.numel()
        shared = self.prefix.expand(self.T, P)
        n_pages = self.attention[0].k_cache.shape[0]
        busy = (self.positions >= 0)[:, None]
        given = torch.isin(own, self.pages[:, P:].contiguous())
        # A page that the prefix has at another place is still to be read from.
        free = (own >= 0) & (own < n_pages) & ~given & (~torch.isin(own, self.prefix) | (own == shared))
        move = free & busy & (shared >= 0) & (shared < n_pages)
        for b in move.any(1).nonzero().flatten().tolist():  # a slot at a time: the copies may be as large as the cache
            to, of = own[b][move[b]].long(), self.prefix[move[b]].long()
            for a in self.attention:
                for t in (a.k_cache, a.v_cache, a.k_scale, a.v_scale):
                    if t is not None:
                        rows = t.view(torch.uint8) if t.dtype in _CODES else t
                        rows[to] = rows[of]
        kept = torch.where(busy & ~free, shared, -1)
        given = given | torch.isin(own, kept)
        self.pages[:, :P] = torch.where(busy & ~free, shared, torch.where(given & ~busy, -1, own))

    @property
    def output(self) -> torch.Tensor:
        return self.x[-1]

    def _body(self) -> None:
        if self.attention is not None:
            torch.add(self.positions, 1, out=self.lengths)
        if self.norms is not None:
            self._normed_layers()
        else:
            for l, (L, r) in enumerate(zip(self.layers, self.routers)):
                x = self.x[l]
                if self.attention is not None:
                    x = torch.add(x, self._attend(l, x), out=self.h[l])
                torch.add(x, self._experts(l, x), out=self.x[l + 1])
        if self.attention is not None:
            self.positions.add_(self.positions >= 0)

    def _attend(self, l: int, x: torch.Tensor) -> torch.Tensor:
        return self.attention[l].decode(x, self.pages, self.positions, self.lengths, workspace=self.attention_workspace, prefix=self.prefix)

    def _experts(self, l: int, x: torch.Tensor) -> torch.Tensor:
        self.routers[l](x, ids=self.ids[l], weights=self.w[l], logits_out=self.logits[l])
        return moe_forward(x, self.ids[l], self.w[l], self.layers[l], out=self.y[l], workspace=self.workspace)

    def _reads(self, i: int) -> torch.dtype:
        """What block i reads: an attention block its weights' type, experts the stream's."""
        return torch.float32 if self.attention is None or i % 2 else self.attention[i // 2].w_qkv.dtype

    def _first(self, x: torch.Tensor) -> torch.Tensor:
        pre = self.norms[0].pre
        return x if pre is None else residual_norm(x, pre=pre, dtype=self._reads(0))[1]

    def _add(self, i: int, x: torch.Tensor, y: torch.Tensor, out: Optional[torch.Tensor] = None):
        last = i + 1 == len(self.norms)
        return self.norms[i].add(x, y, None if last else self.norms[i + 1], torch.float32 if last else self._reads(i + 1), x_out=out)

    def _normed_layers(self) -> None:
        x = self.x[0]
        n, i = self._first(x), 0
        for l in range(len(self.layers)):
            if self.attention is not None:
                x, n = self._add(i, x, self._attend(l, n), out=self.h[l])
                i += 1
            x, n = self._add(i, x, self._experts(l, n), out=self.x[l + 1])
            i += 1

    def load(self, x0: torch.Tensor) -> None:
        self.x[0].copy_(x0)

    def forward(self, x0: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Eager run on the current stream."""
        if x0 is not None:
            self.load(x0)
        self._body()
        return self.output

    def prompt(self, x: torch.Tensor, starts: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
        """New tokens of several sequences through every layer: x [N, d], packed; sequence b is rows starts[b] ..
        starts[b + 1] - 1 (int32 [B + 1], ascending, up to N) and goes on in slot slots[b] (int32 [B], different
        ones of 0 .. n_tokens - 1) at that slot's position, or from 0 where the slot is idle (also
        with no tokens: a slot that is to stay idle is left out; behind a shared prefix: start_behind).  The slots' pages have to have
        room.  Returns the output rows f32 [N, d]; the slots then decode what follows.  Rows of no sequence
        (padding) reach no cache, their attention is zeros, and they pass the experts."""
        if self.attention is None:
            raise RuntimeError("this stack has no attention")
        if x.dim() != 2 or x.shape[1] != self.d:
            raise ValueError(f"expected x [N, {self.d}]")
        if starts.dtype != torch.int32 or slots.dtype != torch.int32 or starts.shape != (slots.numel() + 1,) or slots.dim() != 1:
            raise ValueError("starts must be int32 [B + 1] and slots int32 [B]")
        dev = self.positions.device
        if x.device != dev or starts.device != dev or slots.device != dev:
            raise ValueError(f"x, starts and slots must be on {dev}")
        x = x.to(torch.float32)
        N, B = x.shape[0], slots.numel()
        at = slots.long()
        first, pages = self.positions[at].clamp_min(0), self.pages[at]
        lengths = first + starts[1:] - starts[:-1]
        if N and B:
            row = torch.arange(N, dtype=torch.int32, device=x.device)
            seqs = torch.searchsorted(starts[1:].contiguous(), row, right=True, out_int32=True).clamp_max(B - 1)
            positions = row - starts[seqs.long()] + first[seqs.long()]
            positions = torch.where((row >= starts[0]) & (row < starts[-1]), positions, -1)
        if N:
            ws = torch.zeros((max(max(workspace_size(L, N, self.k) for L in self.layers), 256),), dtype=torch.uint8, device=x.device)
            n = x if self.norms is None else self._first(x)
            for l, (L, r, a) in enumerate(zip(self.layers, self.routers, self.attention)):
                if B or self.norms is not None:
                    y = a.prompt(n, pages, positions, seqs, starts, lengths) if B else x.new_zeros(x.shape)
                    x, n = (x + y,) * 2 if self.norms is None else self._add(2 * l, x, y)
                ids, w = route(r.k, x=n, router=r.weight, drop=r.drop, drop_param=r.drop_param)
                y = moe_forward(n, ids, w, L, workspace=ws)
                x, n = (x + y,) * 2 if self.norms is None else self._add(2 * l + 1, x, y)
        else:
            x = x.clone()
        self.positions.index_copy_(0, at, lengths)
        return x

    def capture(self, warmup: int = 2) -> torch.cuda.CUDAGraph:
        """Capture the stack in a graph; replays read x[0] (and the slots' pages and positions) and write every buffer."""
        at = self.positions.clone() if self.attention is not None else None
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(warmup):
                self._body()
                if at is not None:  # the slots stay where they are: their next token overwrites what this one stored
                    self.positions.copy_(at)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            self._body()
        g.held = self._captured_operands()
        self.graph = g
        return g

    def _captured_operands(self) -> List[Optional[torch.Tensor]]:
        """What a graph reads and writes that the stack may replace while somebody still has the graph: it lives as long as its handle."""
        kept = [] if self.attention is None else [self.prefix, self.attention_workspace]
        for b in self.norms or ():
            kept += [b.gate, *(t for n in (b.pre, b.post) if n is not None for t in (n.weight, n.bias))]
        return kept

    def replay(self) -> torch.Tensor:
        if self.graph is None:
            raise RuntimeError("capture() first")
        self.graph.replay()
        return self.output

    def resident_bytes(self) -> int:
        return sum(L.nbytes() for L in self.layers)

    def router_bytes(self) -> int:
        return sum(r.weight.numel() * r.weight.element_size() for r in self.routers)

    def layer_ids(self) -> List[torch.Tensor]:
        return self.ids
