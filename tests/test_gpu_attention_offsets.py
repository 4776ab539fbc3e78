"""Rows so far apart that their offsets pass 32 bits, in elements and in bytes, for each operator that takes strides; and a step whose lengths change under a captured layer."""
import importlib

import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def wide(cuda):
    """300 rows of 2^24 elements (10 GB), of which a few thousand are used."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 10 GB")
    buf = torch.empty((300, 1 << 24), dtype=torch.float16, device="cuda")
    yield buf
    del buf
    torch.cuda.empty_cache()


def _view(wide, heads, dim, at):
    x = wide[:, at:at + heads * dim].view(300, heads, dim)
    x.copy_(torch.randn((300, heads, dim), generator=torch.Generator().manual_seed(at)).half())
    return x


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_far_apart(abq, cuda, wide, dim):
    q, k, v, out = (_view(wide, h, dim, 4096 * i) for i, h in enumerate((4, 2, 2, 4)))
    assert q.stride(0) * 299 > 1 << 32
    scale = dim ** -0.5
    ends = torch.tensor([0, 290, 300], dtype=torch.int32).cuda()
    abq.prompt_attention(abq.make_prompt_attention_params(q, k, v, out, ends, ends, scale=scale))
    want, bound = R.prompt_attention(q.cpu(), k.cpu(), v.cpu(), [290, 10], [290, 10], scale)
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    # an Inf in the last rows: they are fetched once more where they are seen
    v[289, 1, 3] = float("inf")
    abq.prompt_attention(abq.make_prompt_attention_params(q, k, v, out, ends, ends, scale=scale))
    got = out.cpu().double()
    assert bool(got[289, 2:, 3].isinf().all()) and int((~got.isfinite()).sum()) == 2
    v[289, 1, 3] = 1.0
    # the cache: written from rows far apart, read back into such, and attention between such
    table = torch.arange(20, dtype=torch.int32).view(1, 20).cuda()
    held = torch.zeros(abq.kv_cache_bytes(20, 16, 2, dim, 8), dtype=torch.uint8, device="cuda")
    cache = abq.make_kv_cache(held, page_size=16, kv_heads=2, head_dim=dim, bits=8, dtype=torch.float16)
    abq.kv_cache_write(abq.make_kv_write_params(cache, k, v, torch.arange(300).cuda()))
    codes, s, low = R.quantise(k.cpu().contiguous(), 8)
    wanted = (codes.float() * s.float() + low.float()).half()
    far = _view(wide, 2, dim, 4096 * 5), _view(wide, 2, dim, 4096 * 6)
    abq.kv_cache_read(abq.make_kv_read_params(cache, *far, table, torch.tensor([0, 300], dtype=torch.int32).cuda()))
    assert torch.equal(far[0].cpu(), wanted)
    rows = (q[236:300], out[236:300])  # 64 rows of one sequence
    work = torch.empty(abq.cache_attention_workspace_bytes(cache, 1, 64, 4), dtype=torch.uint8, device="cuda")
    abq.cache_attention(abq.make_cache_attention_params(cache, *rows, table, torch.tensor([300], dtype=torch.int32).cuda(), scale=scale, workspace=work))
    want, bound = R.cache_attention(held.cpu().view(20, 2, 1, -1), 16, 8, torch.float16, table.cpu(), [300], rows[0].cpu(), 64, scale)
    assert bool(((rows[1].cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("heads,kv_heads,rows", [(8, 8, 1), (16, 2, 12)])
def test_a_captured_layer_follows_the_steps_tables(abq, cuda, heads, kv_heads, rows):
    """One step's tables, refilled in place for the steps after it: places, lengths, pages and tree."""
    att = importlib.import_module("abq_llm_b200.attention")
    dim, bits = 128, 8
    gen = torch.Generator().manual_seed(heads)
    pages = att.PagedSequences(64, 16)
    layer = att.BlockAttention(abq, torch, heads=heads, kv_heads=kv_heads, head_dim=dim, num_pages=64)
    width = (heads + 2 * kv_heads) * dim
    ids = [pages.add(40), pages.add(3)]
    layer.step = att.AttentionStep.make(torch, pages, ids, [40, 3], prompt=True)
    layer(torch.randn((43, width), generator=gen).half().cuda())
    room = 40
    table = torch.zeros((2, room), dtype=torch.int32, device="cuda")
    tree = torch.zeros((2, rows), dtype=torch.int64, device="cuda")

    def tables():
        for s in ids:
            pages.extend(s, rows)
        step = att.AttentionStep.make(torch, pages, ids, [rows] * 2, prompt=False, tree=R.random_tree(gen, 2, rows).cuda())
        table[:, :step.block_table.shape[1]].copy_(step.block_table)
        tree.copy_(step.tree)
        return step

    held = tables()
    layer.step = held
    held.block_table, held.tree = table, tree
    x = torch.zeros((2 * rows, width), dtype=torch.float16, device="cuda")
    for s in ids:
        pages.trim(s, pages.length(s) - rows)
    layer(x)  # (the workspace is made outside the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
    for _ in range(5):
        step = tables()
        held.slots.copy_(step.slots)
        held.seq_lens.copy_(step.seq_lens)
        x.copy_(torch.randn(x.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        q, _, _ = layer.split(x.cpu())
        want, bound = R.cache_attention(layer.data.cpu().view(64, kv_heads, 1, -1), 16, bits, torch.float16, table.cpu(), step.seq_lens.tolist(), q, rows, dim ** -0.5, tree.cpu())
        assert bool(((out.cpu().double().view(want.shape) - want).abs() <= bound).all())
