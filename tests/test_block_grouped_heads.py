"""A decoder block with grouped heads: the QKV projection's width, what every rank holds of it, and the attention it is given; with numpy in place of the GEMMs here, and
the library's block on the GPU."""
import importlib
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import attention_ref as R


@pytest.fixture
def tp(abq):
    return importlib.import_module("abq_llm_b200.tp_linear")


class Backend:
    class Linear:
        def __init__(self, codes):
            self.w, (self.out_features, self.in_features) = codes.astype(np.float64), codes.shape

        def __call__(self, x):
            return x @ self.w.T

    def make_linear(self, codes, scale, zero, w_bits, group, reduce_output=False):
        return self.Linear(codes)

    def glue_attention(self, qkv, hl, out=None):
        return qkv[:, :hl]

    def glue_residual(self, a, b, out=None):
        return a + b

    def glue_swiglu(self, gu, fl, out=None):
        return gu[:, :fl] * gu[:, fl:]

    def all_reduce(self, t):
        return t


def _weights(tp, hidden, ffn, heads_per_kv, seed=0):
    rng = np.random.default_rng(seed)
    return [(rng.integers(0, 4, size=(s.out_features, s.in_features)), np.ones(s.out_features), None) for s in tp.llama_block_specs(hidden, ffn, heads_per_kv)]


@pytest.mark.parametrize("hidden,heads_per_kv,world", [(4096, 4, 8), (4096, 1, 8), (1536, 3, 2), (2560, 5, 3), (512, 4, 1)])
def test_every_rank_holds_the_query_heads_of_its_key_heads(tp, hidden, heads_per_kv, world):
    qkv, o, *_ = tp.llama_block_specs(hidden, 1024, heads_per_kv)
    kv = hidden // heads_per_kv
    assert qkv.out_features == hidden + 2 * kv and (o.out_features, o.in_features) == (hidden, hidden)
    seen = []
    for rank in range(world):
        rows, _ = tp.shard_of(qkv, rank, world)
        cols = tp.shard_of(o, rank, world)[1]
        own = (cols.stop - cols.start) // heads_per_kv
        queries, keys, values = rows[:own * heads_per_kv], rows[own * heads_per_kv:own * (heads_per_kv + 1)], rows[own * (heads_per_kv + 1):]
        assert queries == list(range(cols.start, cols.stop)), "the output projection reads this rank's query heads"
        assert [x - hidden for x in keys] == [x - hidden - kv for x in values] == list(range(cols.start // heads_per_kv, cols.stop // heads_per_kv))
        seen += rows
    assert sorted(seen) == list(range(qkv.out_features))


@pytest.mark.parametrize("heads,kv_heads,dim,world", [(8, 2, 128, 2), (12, 4, 64, 2), (4, 4, 128, 2)])
def test_ranks_together_are_the_whole_block(tp, heads, kv_heads, dim, world):
    hidden, ffn, g = heads * dim, 256, heads // kv_heads
    weights, x = _weights(tp, hidden, ffn, g), np.random.default_rng(1).normal(size=(3, hidden))

    class Attention:
        """Something of every head that shows which key and value it was given."""
        head_dim = dim

        def __init__(self, heads, kv_heads):
            self.heads, self.kv_heads = heads, kv_heads

        def __call__(self, qkv, out):
            y = qkv.reshape(len(qkv), self.heads + 2 * self.kv_heads, dim)
            q, k, v = y[:, :self.heads], y[:, self.heads:self.heads + self.kv_heads], y[:, self.heads + self.kv_heads:]
            share = (q * np.repeat(k, g, axis=1)).sum(-1, keepdims=True) / hidden ** 3
            return (share * np.repeat(v, g, axis=1)).reshape(len(qkv), -1)

    whole = tp.TensorParallelBlockLinears(Backend(), hidden, ffn, 0, 1, weights, 2, attention=Attention(heads, kv_heads))
    parts = [tp.TensorParallelBlockLinears(Backend(), hidden, ffn, r, world, weights, 2, attention=Attention(heads // world, kv_heads // world)) for r in range(world)]
    assert np.allclose(sum(p.attention_part(x) for p in parts), whole.attention_part(x), rtol=1e-12)
    # a plain callable: the block is told what shares a key head; without an attention the queries stand in
    wrapped = tp.TensorParallelBlockLinears(Backend(), hidden, ffn, 0, 1, weights, 2, attention=lambda qkv, out: whole.attention(qkv, out), heads_per_kv=g)
    assert np.array_equal(wrapped.forward(x), whole.forward(x))
    plain = tp.TensorParallelBlockLinears(Backend(), hidden, ffn, 0, 1, weights, 2, heads_per_kv=g)
    assert np.allclose(plain.attention_part(x), (x @ weights[0][0][:hidden].T) @ weights[1][0].T)


def test_refusals(tp):
    weights = _weights(tp, 512, 256, 2)
    make = lambda att, w=weights, **kw: tp.TensorParallelBlockLinears(Backend(), 512, 256, 0, 1, w, 2, attention=att, **kw)  # noqa: E731
    att = lambda **kw: SimpleNamespace(**{**dict(heads=4, kv_heads=2, head_dim=128, dtype=torch.float16), **kw})  # noqa: E731
    make(att())
    with pytest.raises(ValueError, match="reads"):
        make(att(heads=8, kv_heads=4))
    with pytest.raises(ValueError, match="reads"):
        make(att(head_dim=64))
    with pytest.raises(ValueError, match="reads"):
        make(att(), heads_per_kv=1)
    with pytest.raises(ValueError, match="fp16"):
        make(att(dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="codes"):
        make(att(kv_heads=4))  # the weights are those of two heads a key head
    with pytest.raises(ValueError):
        tp.llama_block_specs(512, 256, 3)


def test_other_callables_are_taken_as_they_are(tp):
    """Names that mean something else there, and a type of its own, are not looked at."""
    class Own:
        heads, kv_heads, head_dim, dtype = [1, 2], {}, "64", torch.bfloat16

        def __call__(self, qkv, out):
            return qkv[:, :512]
    block = tp.TensorParallelBlockLinears(Backend(), 512, 256, 0, 1, _weights(tp, 512, 256, 1), 2, attention=Own())
    x = np.random.default_rng(1).normal(size=(3, 512))
    plain = tp.TensorParallelBlockLinears(Backend(), 512, 256, 0, 1, _weights(tp, 512, 256, 1), 2)
    assert np.array_equal(block.forward(x), plain.forward(x))


@pytest.mark.gpu
def test_a_grouped_block_on_the_gpu(abq, cuda, tp):
    """A prompt and a token step through a block of 8 heads on 2: the attention gets its heads of the projection's rows; with queries and keys turned by a callable
    around it, too."""
    att = importlib.import_module("abq_llm_b200.attention")
    heads, kv_heads, dim, ffn = 8, 2, 64, 1024
    hidden, width = heads * dim, (heads + 2 * kv_heads) * dim
    gen = torch.Generator(device="cuda").manual_seed(0)
    be = tp.AbqBackend(abq, torch, None, x_bits=8, x_scale=16.0, max_tokens=64)
    weights = []
    for spec in tp.llama_block_specs(hidden, ffn, heads // kv_heads):
        codes = torch.randint(0, 16, (spec.out_features, spec.in_features), dtype=torch.int32, device="cuda", generator=gen)
        scale = ((torch.rand(spec.out_features, device="cuda", generator=gen) + 0.5) * (3.4 / (16 * spec.in_features ** 0.5))).half()
        weights.append((codes, scale, torch.full((spec.out_features,), 8, dtype=torch.uint8, device="cuda")))
    pages = att.PagedSequences(8, 16)
    ids = [pages.add(20), pages.add(9)]
    for turn in (lambda qkv: qkv, lambda qkv: torch.cat([-qkv[:, :width - kv_heads * dim], qkv[:, width - kv_heads * dim:]], dim=1)):
        inner = att.BlockAttention(abq, torch, heads=heads, kv_heads=kv_heads, head_dim=dim, num_pages=8)
        block = tp.TensorParallelBlockLinears(be, hidden, ffn, 0, 1, weights, 4, attention=lambda qkv, out: inner(turn(qkv), out), heads_per_kv=heads // kv_heads)
        inner.step = att.AttentionStep.make(torch, pages, ids, [20, 9], prompt=True)
        block.forward(torch.randn((29, hidden), device="cuda", generator=gen).half())
        for s in ids:
            pages.extend(s, 1)
        inner.step = step = att.AttentionStep.make(torch, pages, ids, [1, 1], prompt=False)
        x = torch.randn((2, hidden), device="cuda", generator=gen).half()
        got = block.forward(x).clone()
        qkv = turn(block.layers["qkv"](x).clone())
        q, _, _ = inner.split(qkv)
        want, bound = R.cache_attention(inner.data.cpu().view(8, kv_heads, 1, -1), 16, 8, torch.float16, step.block_table.cpu(), step.seq_lens.tolist(), q.cpu(), 1, dim ** -0.5)
        attn = inner(qkv.contiguous())
        assert bool(((attn.cpu().double().view(2, heads, dim) - want).abs() <= bound).all())
        h, d = block.ffn_part(x, block.layers["o"](attn).clone())
        assert torch.equal(be.glue_residual(h, d), got)
        for s in ids:
            pages.trim(s, pages.length(s) - 1)
    block = tp.TensorParallelBlockLinears(be, hidden, ffn, 0, 1, weights, 4, attention=att.BlockAttention(abq, torch, heads=heads, kv_heads=kv_heads, head_dim=dim, num_pages=8))
    assert block.heads_per_kv == 4
