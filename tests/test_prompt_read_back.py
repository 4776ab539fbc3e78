"""Prompt steps that always read back: a prompt's result does not depend on what it is batched with, nor on its chunks beyond rounding."""
import importlib

import pytest
import torch

import attention_ref as R


@pytest.fixture(scope="module")
def att(abq):
    return importlib.import_module("abq_llm_b200.attention")


def test_step(att):
    p = att.PagedSequences(8, 16)
    a, b = p.add(20), p.add(3)
    plain = att.AttentionStep.make(torch, p, [a, b], [20, 3], prompt=True, device="cpu")
    back = att.AttentionStep.make(torch, p, [a, b], [20, 3], prompt=True, read_back=True, device="cpu")
    assert not plain.prefix and back.prefix
    assert back.held == 23 and back.cu_q.tolist() == back.cu_k.tolist() == [0, 20, 23]


@pytest.mark.gpu
@pytest.mark.parametrize("bits,half,heads,kv_heads,dim", [(4, torch.float16, 8, 2, 128), (8, torch.bfloat16, 4, 4, 64)])
def test_alone_and_beside_a_chunk(abq, cuda, att, bits, half, heads, kv_heads, dim):
    gen = torch.Generator().manual_seed(bits)
    pages = att.PagedSequences(80, 16)
    layer = att.BlockAttention(abq, torch, heads=heads, kv_heads=kv_heads, head_dim=dim, num_pages=80, bits=bits, dtype=half)
    rows = lambda n: torch.randn((n, (heads + 2 * kv_heads) * dim), generator=gen).to(half)  # noqa: E731

    def run(x, ids, new):
        layer.step = att.AttentionStep.make(torch, pages, ids, new, prompt=True, read_back=True)
        return layer(x.cuda()).clone()

    x, other, chunk = rows(300), rows(45), rows(70)
    alone = run(x, [pages.add(300)], [300])
    old = pages.add(45)
    run(other, [old], [45])
    pages.extend(old, 70)
    mixed = run(torch.cat([chunk, x]), [old, pages.add(300)], [70, 300])
    assert torch.equal(mixed[70:].view(torch.int16), alone.view(torch.int16)), "the same prompt beside another sequence's chunk"
    parts, seq = [], pages.add(0)
    for n in (100, 1, 199):
        pages.extend(seq, n)
        at = sum(len(p) for p in parts)
        parts.append(run(x[at:at + n], [seq], [n]))
    q, k, v = layer.split(x)
    back = []
    for part in (k, v):  # what the cache holds of it
        codes, scale, low = R.quantise(part.contiguous(), bits)
        back.append(((codes.float() * scale.float()) + low.float()).to(half))
    want, bound = R.prompt_attention(q, *back, [300], [300], dim ** -0.5)
    for got in (alone, torch.cat(parts)):
        assert bool(((got.cpu().double().view(300, heads, dim) - want).abs() <= bound).all())
