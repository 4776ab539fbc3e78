"""Pages and steps of the quantised cache on the host (no device), and the block's attention hook with a numpy stand-in."""
import random

import pytest
import torch


@pytest.fixture(scope="module")
def att(abq):
    import importlib
    return importlib.import_module("abq_llm_b200.attention")


def test_pages_belong_to_one_sequence_each(att):
    """A random life of sequences: every page is free or held once, lengths fit, places are distinct."""
    r = random.Random(5)
    p = att.PagedSequences(40, 32)
    live = {}
    for _ in range(600):
        act = r.random()
        if act < 0.3:
            n = r.choice([0, 1, 31, 32, 33, 200])
            try:
                live[p.add(n)] = n
            except att.OutOfPages:
                assert sum(-(-x // 32) for x in live.values()) + -(-n // 32) > 40
        elif live and act < 0.7:
            s = r.choice(list(live))
            n = r.choice([0, 1, 7, 64])
            try:
                p.extend(s, n)
                live[s] += n
            except att.OutOfPages:
                assert p.length(s) == live[s]
        elif live and act < 0.9:
            s = r.choice(list(live))
            live[s] = r.randint(0, live[s])
            p.trim(s, live[s])
        elif live:
            s = r.choice(list(live))
            p.free(s)
            del live[s]
        held = [x for s in live for x in p.pages(s)]
        assert len(set(held)) == len(held) == sum(-(-n // 32) for n in live.values()) and all(0 <= x < 40 for x in held)
        assert all(p.length(s) == n for s, n in live.items())
        slots = [x for s, n in live.items() for x in p.slots(s, n)]
        assert len(set(slots)) == len(slots)


def test_refusals(att):
    for pages, size in ((0, 16), (4, 8), (4, 24), (4, 2048)):
        with pytest.raises(ValueError):
            att.PagedSequences(pages, size)
    p = att.PagedSequences(4, 16)
    a, b = p.add(20), p.add(5)
    with pytest.raises(att.OutOfPages):
        p.add(17)
    assert p.add(16) == 2  # nothing was lost on the way
    with pytest.raises(ValueError):
        p.trim(a, 21)
    with pytest.raises(ValueError):
        p.extend(a, -1)
    with pytest.raises(ValueError):
        p.slots(b, 6)
    make = lambda *x, **k: att.AttentionStep.make(torch, p, *x, device="cpu", **k)  # noqa: E731
    for ids, new, kw in (([a], [1, 1], {}), ([], [], {}), ([a, b], [1, 2], {}), ([a], [21], {}), ([a], [0], {}), ([a, a], [1, 1], {}), ([a], [-1], dict(prompt=True)),
                         ([a], [3], dict(prompt=True, tree=torch.zeros((1, 3), dtype=torch.int64)))):
        with pytest.raises(ValueError):
            make(ids, new, **{"prompt": False, **kw})


def test_step_tables(att):
    p = att.PagedSequences(8, 16)
    a = p.add(20)
    b = p.add(3)
    p.extend(a, 2)
    s = att.AttentionStep.make(torch, p, [a, b], [2, 2], prompt=False, device="cpu")
    assert (s.kind, s.rows, s.total, s.held, s.prefix) == ("tokens", 2, 4, 25, True)
    assert s.seq_lens.tolist() == [22, 3] and s.block_table.tolist() == [p.pages(a), p.pages(b) + [0]]
    assert s.slots.tolist() == [p.pages(a)[1] * 16 + 4, p.pages(a)[1] * 16 + 5, p.pages(b)[0] * 16 + 1, p.pages(b)[0] * 16 + 2]
    q = att.AttentionStep.make(torch, p, [b, a], [3, 22], prompt=True, device="cpu")
    assert not q.prefix and q.cu_q.tolist() == [0, 3, 25] == q.cu_k.tolist() and q.longest == 22


def test_the_block_calls_its_attention(abq):
    """TensorParallelBlockLinears hands the QKV output to the attention it was given, and to the backend's stand-in otherwise."""
    import importlib
    import numpy as np
    TP = importlib.import_module("abq_llm_b200.tp_linear")

    class Linear:
        def __init__(self, codes):
            self.w, self.out_features = codes.astype(np.float64), codes.shape[0]

        def __call__(self, x):
            return x @ self.w.T

    class Backend:
        def make_linear(self, codes, scale, zero, w_bits, group, reduce_output=False):
            return Linear(codes)

        def glue_attention(self, qkv, hl, out=None):
            return qkv[:, :hl]

        def all_reduce(self, t):
            return t

        def glue_residual(self, a, b, out=None):
            return a + b

        def glue_swiglu(self, gu, fl, out=None):
            return gu[:, :fl] * gu[:, fl:]

    rng = np.random.default_rng(0)
    shapes = [(s.out_features, s.in_features) for s in TP.llama_block_specs(128, 256)]
    weights = [(rng.integers(0, 4, size=s), np.ones(s[0]), None) for s in shapes]
    x = rng.normal(size=(3, 128))
    plain = TP.TensorParallelBlockLinears(Backend(), 128, 256, 0, 1, weights, 2)
    seen = []

    def attention(qkv, out):
        seen.append((qkv.shape, out))
        return qkv[:, 256:]
    block = TP.TensorParallelBlockLinears(Backend(), 128, 256, 0, 1, weights, 2, attention=attention)
    a, b = plain.forward(x), block.forward(x)
    assert seen == [((3, 384), None)] and not np.allclose(a, b)
    assert np.allclose(block.attention_part(x), (x @ weights[0][0].T)[:, 256:] @ weights[1][0].T)
