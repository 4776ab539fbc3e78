"""The attention of a decoder block next to its quantised linear layers: pages, steps and the four calls together.

The reference's FasterTransformer fork runs attention between the QKV projection and the attention output projection
(layers/attention_layers/GptContextAttentionLayer.cc, DecoderSelfAttentionLayer.cc) over a dense fp16 cache.  Here the cache
is paged and holds 8- or 4-bit codes, sequences of any lengths share a step, and a step may bring one token a sequence, a
tree of drafted tokens, whole prompts, or a chunk of a prompt behind what the cache holds.

* :class:`PagedSequences` -- which pages belong to which sequence (host side, no device needed)
* :class:`AttentionStep`  -- one step's tables on the device, made once and used by every layer
* :class:`BlockAttention` -- one layer's cache; called with the fused QKV output, it writes the step's keys and values and attends

``TensorParallelBlockLinears(..., attention=BlockAttention(...))`` calls it where the block otherwise has a stand-in.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Sequence

from . import binding as B


class OutOfPages(RuntimeError):
    pass


class PagedSequences:
    """Pages of a cache (the same for every layer) dealt to sequences of any lengths."""

    def __init__(self, num_pages: int, page_size: int):
        if num_pages <= 0 or page_size <= 0 or page_size % 16 or page_size > 1024:
            raise ValueError(f"{num_pages} pages of {page_size} tokens: pages are multiples of 16 tokens, at most 1024")
        self.num_pages, self.page_size = num_pages, page_size
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._pages: Dict[int, List[int]] = {}
        self._length: Dict[int, int] = {}
        self._next = 0

    def add(self, tokens: int = 0) -> int:
        """A new sequence with room for ``tokens``; its number."""
        seq = self._next
        self._pages[seq], self._length[seq] = [], 0
        try:
            self.extend(seq, tokens)
        except (OutOfPages, ValueError):
            del self._pages[seq], self._length[seq]
            raise
        self._next += 1
        return seq

    def extend(self, seq: int, tokens: int) -> None:
        """``tokens`` more places at the end.  Where pages run out nothing has changed."""
        if tokens < 0:
            raise ValueError("trim() takes tokens away")
        need = -(-(self._length[seq] + tokens) // self.page_size) - len(self._pages[seq])
        if need > len(self._free):
            raise OutOfPages(f"{need} pages wanted, {len(self._free)} of {self.num_pages} free")
        self._pages[seq] += [self._free.pop() for _ in range(need)]
        self._length[seq] += tokens

    def trim(self, seq: int, length: int) -> None:
        """Back to ``length`` tokens (drafts that were not accepted); pages behind it are free again."""
        if not 0 <= length <= self._length[seq]:
            raise ValueError(f"sequence {seq} has {self._length[seq]} tokens")
        keep = -(-length // self.page_size)
        self._free += reversed(self._pages[seq][keep:])
        del self._pages[seq][keep:]
        self._length[seq] = length

    def free(self, seq: int) -> None:
        self.trim(seq, 0)
        del self._pages[seq], self._length[seq]

    def length(self, seq: int) -> int:
        return self._length[seq]

    def pages(self, seq: int) -> List[int]:
        return list(self._pages[seq])

    def slots(self, seq: int, tokens: int) -> List[int]:
        """Places of the last ``tokens`` tokens, as abq_kv_cache_write takes them."""
        n, P = self._length[seq], self.page_size
        if not 0 <= tokens <= n:
            raise ValueError(f"sequence {seq} has {n} tokens")
        return [self._pages[seq][t // P] * P + t % P for t in range(n - tokens, n)]


@dataclass
class AttentionStep:
    """Tables of one step: the last ``new[i]`` tokens of every sequence are its rows, packed in this order."""
    kind: str                # "tokens": the same number of rows of every sequence, over the cache; "prompt": packed prompts or chunks
    rows: int                # rows of a sequence ("tokens")
    total: int               # rows of the step
    longest: int             # rows of the sequence with most
    held: int                # tokens of all sequences, those of the step included
    prefix: bool             # some sequence had tokens before the step (or read_back): a prompt step's keys and values come out of the cache, for all its sequences
    slots: object
    block_table: object
    seq_lens: object
    cu_q: object
    cu_k: object
    tree: object = None
    workspace: object = None
    outgrown: list = field(default_factory=list)  # workspaces that were too small for a later layer: a captured launch may still point to them

    @classmethod
    def make(cls, torch, sequences: PagedSequences, ids: Sequence[int], new: Sequence[int], *, prompt: bool, tree=None, read_back: bool = False,
             device="cuda") -> "AttentionStep":
        """``new`` tokens of every sequence of ``ids`` have places already (:meth:`PagedSequences.extend`).  ``tree``: int64 [batch][rows] as
        abq_cache_attention takes it.

        A prompt step in which no sequence had tokens before attends to the keys and values as they come; as soon as one had, all of its sequences attend to what
        the cache gives back, quantised.  ``read_back``: the latter always, so that a prompt's result depends neither on what it is batched with nor on the chunks
        that it comes in (it costs reading the step's tokens back)."""
        if len(ids) != len(new) or not ids or any(m < 0 or m > sequences.length(s) for s, m in zip(ids, new)):
            raise ValueError("a step needs a number of new tokens for each of its sequences, at most its length")
        if len(set(ids)) != len(ids):
            raise ValueError("a sequence can be in a step once")
        if not prompt and (len(set(new)) != 1 or not 1 <= new[0] <= 64):
            raise ValueError("a token step has the same number of rows, 1 to 64, of every sequence")
        if tree is not None and prompt:
            raise ValueError("prompts are causal: a tree goes with a token step")
        lens = [sequences.length(s) for s in ids]
        pages = [sequences.pages(s) for s in ids]
        width = max(1, max(len(p) for p in pages))
        ints = lambda v, t: torch.tensor(v, dtype=t).to(device)  # noqa: E731
        ends = lambda v: ints([sum(v[:i]) for i in range(len(v) + 1)], torch.int32)  # noqa: E731
        return cls(kind="prompt" if prompt else "tokens", rows=0 if prompt else new[0], total=sum(new), longest=max(new), held=sum(lens),
                   prefix=any(m < n for m, n in zip(new, lens)) or (prompt and read_back),
                   slots=ints([x for s, m in zip(ids, new) for x in sequences.slots(s, m)], torch.int64),
                   block_table=ints([p + [0] * (width - len(p)) for p in pages], torch.int32), seq_lens=ints(lens, torch.int32),
                   cu_q=ends(new), cu_k=ends(lens), tree=tree)

    def scratch(self, torch, nbytes: int, device):
        """The step's workspace, with room for ``nbytes``.  It lives as long as the step, and so do the smaller ones before it."""
        if self.workspace is None or self.workspace.numel() < nbytes:
            if self.workspace is not None:
                self.outgrown.append(self.workspace)
            self.workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        return self.workspace


class BlockAttention:
    """One layer's quantised cache and its attention.  ``step`` is set by the caller before a forward pass; calls write the step's keys
    and values into the cache, then attend.  All on the current stream; the layers of a model share a step (and its workspace, so calls that
    may overlap need a step each).  A captured launch reads the step's tables and uses its workspace: the caller keeps the step as long as the graph."""

    def __init__(self, abq, torch, *, heads: int, kv_heads: int | None = None, head_dim: int = 128, num_pages: int, page_size: int = 16, bits: int = 8, dtype=None,
                 scale: float | None = None, device="cuda", status_word=None):
        self.abq, self.torch = abq, torch
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads or heads, head_dim
        self.dtype = dtype or torch.float16
        self.scale = scale if scale is not None else head_dim ** -0.5
        nbytes = B.kv_cache_bytes(num_pages, page_size, self.kv_heads, head_dim, bits)
        if not nbytes:
            raise ValueError(f"no cache of {bits} bits, {self.kv_heads} heads of {head_dim}, pages of {page_size} tokens")
        self.data = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        self.cache = B.make_kv_cache(self.data, page_size=page_size, kv_heads=self.kv_heads, head_dim=head_dim, bits=bits, dtype=self.dtype)
        self.status_word = status_word
        self.step: AttentionStep | None = None

    def split(self, qkv):
        """Queries, keys and values of a fused projection's output [rows][(heads + 2 kv_heads) * head_dim], as views."""
        H, K = self.heads, self.kv_heads
        x = qkv.view(qkv.shape[0], H + 2 * K, self.head_dim)
        return x[:, :H], x[:, H:H + K], x[:, H + K:]

    def __call__(self, qkv, out=None):
        """qkv [rows][(heads + 2 kv_heads) * head_dim] -> [rows][heads * head_dim] (in ``out`` if given)."""
        step, torch = self.step, self.torch
        if step is None:
            raise RuntimeError("set .step before the forward pass")
        if qkv.shape[0] != step.total:
            raise ValueError(f"{qkv.shape[0]} rows, the step has {step.total}")
        if out is None:
            out = torch.empty((step.total, self.heads * self.head_dim), dtype=self.dtype, device=qkv.device)
        q, k, v = self.split(qkv)
        res = out.view(step.total, self.heads, self.head_dim)
        B.kv_cache_write(B.make_kv_write_params(self.cache, k, v, step.slots))
        if step.kind == "tokens":
            need = B.cache_attention_workspace_bytes(self.cache, step.seq_lens.numel(), step.rows, self.heads)
            B.cache_attention(B.make_cache_attention_params(self.cache, q, res, step.block_table, step.seq_lens, scale=self.scale,
                                                            workspace=step.scratch(torch, need, qkv.device), tree=step.tree, status_word=self.status_word))
            return out
        if step.prefix:  # a chunk behind what the cache holds: whole sequences come out of it, the chunk as it has just been written among them
            k, v = (torch.empty((step.held, self.kv_heads, self.head_dim), dtype=self.dtype, device=qkv.device) for _ in range(2))
            B.kv_cache_read(B.make_kv_read_params(self.cache, k, v, step.block_table, step.cu_k))
        B.prompt_attention(B.make_prompt_attention_params(q, k, v, res, step.cu_q, step.cu_k if step.prefix else step.cu_q, scale=self.scale, max_q=step.longest,
                                                          status_word=self.status_word))
        return out
