"""Inf and NaN among the values of packed prompts over many rounds of blocks, most of which leave one of a block's two row tiles without a key: whether a block's V tiles
held such values is told to each row tile through a few slots that go round."""
import random

import pytest
import torch

from test_gpu_prompt_attention import HALF, _run

pytestmark = pytest.mark.gpu


def _prompts(seed, batch):
    """Long ones (both row tiles have rows), many shorter than half a block, some whose first rows see nothing (only the second row tile has keys), some behind a prefix."""
    r = random.Random(seed)
    nq, nk = [], []
    for _ in range(batch):
        kind = r.random()
        n = r.randint(130, 250) if kind < 0.25 else r.randint(1, 60)
        m = n
        if 0.25 <= kind < 0.4:
            n = r.randint(140, 250)
            m = n - 128 if r.random() < 0.7 else r.randint(1, 20)
        elif kind > 0.85:
            m = n + r.randint(1, 200)
        nq.append(n), nk.append(m)
    return nq, nk


@pytest.mark.parametrize("half", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv_heads,batch", [(64, 48, 48, 45), (64, 64, 16, 30), (128, 48, 48, 45)])
def test_values_of_other_blocks_do_not_count(abq, cuda, half, dim, heads, kv_heads, batch):
    nq, nk = _prompts(dim + batch, batch)
    at = [sum(nk[:b]) for b in range(batch)]

    def edit(q, k, v):
        r = random.Random(batch)
        for b in range(batch):
            if r.random() < 0.3:
                v[at[b] + r.randrange(nk[b]), r.randrange(kv_heads), r.randrange(dim)] = r.choice([float("inf"), float("-inf"), float("nan")])

    first = _run(abq, HALF[half], dim, heads, kv_heads, nq, nk, seed=batch, edit=edit).clone()
    for _ in range(5):
        again = _run_only(abq, HALF[half], dim, heads, kv_heads, nq, nk, batch, edit)
        assert torch.equal(first[:sum(nq)].view(torch.int16), again[:sum(nq)].view(torch.int16))


def _run_only(abq, half, dim, heads, kv_heads, nq, nk, seed, edit):
    from test_gpu_prompt_attention import _ends, _inputs
    q, k, v = _inputs(seed, half, dim, heads, kv_heads, nq, nk)
    edit(q, k, v)
    out = torch.empty((q.shape[0], heads, dim), dtype=half, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    abq.prompt_attention(abq.make_prompt_attention_params(q, k, v, out, _ends(nq), _ends(nk), scale=dim ** -0.5, status_word=status))
    assert int(status.item()) == 0
    return out
