"""The attention operators as they are used together: prompts, token steps, a tree of drafts that is verified and trimmed, a chunk behind a prefix, through
BlockAttention in a decoder block, against 64 bits over the same cache; and the torch operators."""
import importlib

import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def att(abq):
    return importlib.import_module("abq_llm_b200.attention")


def _table(step):
    return step.block_table.cpu()


@pytest.mark.parametrize("bits,half,heads,kv_heads,dim", [(8, torch.float16, 4, 4, 128), (4, torch.bfloat16, 8, 2, 64)])
def test_a_conversation(abq, cuda, att, bits, half, heads, kv_heads, dim):
    gen = torch.Generator().manual_seed(bits)
    pages = att.PagedSequences(64, 32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    layer = att.BlockAttention(abq, torch, heads=heads, kv_heads=kv_heads, head_dim=dim, num_pages=64, page_size=32, bits=bits, dtype=half, status_word=status)
    granule = R.granule_bytes(dim, bits)
    mirror = torch.zeros((64, kv_heads, 2, granule), dtype=torch.uint8)
    scale = dim ** -0.5

    def qkv(rows):
        return torch.randn((rows, (heads + 2 * kv_heads) * dim), generator=gen).to(half)

    def run(ids, new, prompt, tree=None):
        step = att.AttentionStep.make(torch, pages, ids, new, prompt=prompt, tree=None if tree is None else tree.cuda())
        layer.step = step
        x = qkv(step.total)
        out = layer(x.cuda())
        torch.cuda.synchronize()
        assert int(status.item()) == 0
        q, k, v = layer.split(x)
        R.encode(mirror, 32, bits, step.slots.cpu(), k.contiguous(), v.contiguous())
        assert torch.equal(layer.data.cpu().view(mirror.shape), mirror)
        return step, x, out.cpu().double().view(step.total, heads, dim), q, k, v

    def near(got, want, bound):
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())

    ids = [pages.add(45), pages.add(1), pages.add(150)]
    step, x, out, q, k, v = run(ids, [45, 1, 150], True)
    near(out, *R.prompt_attention(q, k, v, [45, 1, 150], [45, 1, 150], scale))
    for _ in range(3):  # tokens, one a sequence
        for s in ids:
            pages.extend(s, 1)
        step, x, out, q, *_ = run(ids, [1, 1, 1], False)
        near(out, *R.cache_attention(mirror, 32, bits, half, _table(step), step.seq_lens.tolist(), q, 1, scale))
    n = 9  # a tree of drafts, verified at once; some are taken
    for s in ids:
        pages.extend(s, n)
    tree = R.random_tree(gen, 3, n)
    step, x, out, q, *_ = run(ids, [n] * 3, False, tree)
    near(out, *R.cache_attention(mirror, 32, bits, half, _table(step), step.seq_lens.tolist(), q, n, scale, tree))
    for s in ids:
        pages.trim(s, pages.length(s) - n + 2)
    pages.free(ids[1])
    late = pages.add(40)  # a new prompt, and a chunk behind what the cache holds, in one step
    pages.extend(ids[0], 37)
    step, x, out, q, k, v = run([late, ids[0]], [40, 37], True)
    lens = [40, pages.length(ids[0])]
    back = []
    for b, m in enumerate(lens):
        back.append([((c * s).float() + low.float()).to(half).permute(1, 0, 2) for c, s, low in R.decode(mirror, 32, bits, dim, half, _table(step)[b], m)])
    kk, vv = (torch.cat([x[i] for x in back]) for i in (0, 1))
    near(out, *R.prompt_attention(q, kk, vv, [40, 37], lens, scale))


def test_in_a_block_of_quantised_linears(abq, cuda, att):
    """Two LLaMA-shaped blocks with attention between their GEMMs, prompt and token steps: the attention gets the QKV projection's rows and its result is
    what the output projection reads; a captured token step replays to the same."""
    TP = importlib.import_module("abq_llm_b200.tp_linear")
    hidden, ffn, M = 512, 1024, 3
    gen = torch.Generator(device="cuda").manual_seed(0)
    be = TP.AbqBackend(abq, torch, None, x_bits=8, x_scale=16.0, max_tokens=64)
    pages = att.PagedSequences(16, 16)
    blocks = []
    for _ in range(2):
        weights = []
        for spec in TP.llama_block_specs(hidden, ffn):
            codes = torch.randint(0, 16, (spec.out_features, spec.in_features), dtype=torch.int32, device="cuda", generator=gen)
            scale = ((torch.rand(spec.out_features, device="cuda", generator=gen) + 0.5) * (3.4 / (16 * spec.in_features ** 0.5))).to(torch.float16)
            weights.append((codes, scale, torch.full((spec.out_features,), 8, dtype=torch.uint8, device="cuda")))
        blocks.append(TP.TensorParallelBlockLinears(be, hidden, ffn, 0, 1, weights, 4, 0,
                                                    attention=att.BlockAttention(abq, torch, heads=4, head_dim=128, num_pages=16, page_size=16)))
    ids = [pages.add(7), pages.add(11), pages.add(2)]

    def forward(x, step):
        seen = []
        for b in blocks:
            b.attention.step = step
            x = b.forward(x).clone()
            seen.append(x)
        return seen

    step = att.AttentionStep.make(torch, pages, ids, [7, 11, 2], prompt=True)
    forward(torch.randn((20, hidden), device="cuda", generator=gen).half(), step)
    for s in ids:
        pages.extend(s, 1)
    step = att.AttentionStep.make(torch, pages, ids, [1] * M, prompt=False)
    x = torch.randn((M, hidden), device="cuda", generator=gen).half()
    got = forward(x, step)
    # the first block again, with its attention taken apart
    b = blocks[0]
    qkv = b.layers["qkv"](x).clone()
    q, _, _ = b.attention.split(qkv)
    want, bound = R.cache_attention(b.attention.data.cpu().view(16, 4, 1, -1), 16, 8, torch.float16, _table(step), step.seq_lens.tolist(), q.cpu(), 1, 128 ** -0.5)
    attn = b.attention(qkv.contiguous())
    assert bool(((attn.cpu().double().view(M, 4, 128) - want).abs() <= bound).all())
    o = b.layers["o"](attn).clone()
    h, d = b.ffn_part(x, o)
    again = be.glue_residual(h, d)
    assert torch.equal(again, got[0])
    # captured
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        held = forward(x, step)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held[1], got[1])


def test_torch_operators(abq, cuda):
    importlib.import_module("abq_llm_b200.torch_ops")
    ops = torch.ops.abq_b200
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn((50, 12, 64), generator=gen).half().cuda()
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    cu = torch.tensor([0, 20, 50], dtype=torch.int32).cuda()
    out = ops.prompt_attention(q, k, v, cu, cu, 0.125)
    want, bound = R.prompt_attention(q.cpu(), k.cpu(), v.cpu(), [20, 30], [20, 30], 0.125)
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    cache = torch.zeros((4, 2, 1, R.granule_bytes(64, 8)), dtype=torch.uint8, device="cuda")
    slots = torch.cat([torch.arange(20), 32 + torch.arange(30)]).cuda()
    ops.kv_cache_write(cache, k, v, slots, 8)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32).cuda()
    ko, vo = torch.empty((50, 2, 64), dtype=torch.float16, device="cuda"), torch.empty((50, 2, 64), dtype=torch.float16, device="cuda")
    ops.kv_cache_read(cache, ko, vo, table, cu, 8)
    codes, scale, low = R.quantise(k.cpu().contiguous(), 8)
    assert torch.equal(ko.cpu(), (codes.float() * scale.float() + low.float()).half())
    lens = torch.tensor([20, 30], dtype=torch.int32).cuda()
    got = ops.cache_attention(q[[19, 49]], cache, table, lens, None, 0.125, 8)
    want, bound = R.cache_attention(cache.cpu(), 16, 8, torch.float16, table.cpu(), [20, 30], q[[19, 49]].cpu(), 1, 0.125)
    assert bool(((got.cpu().double() - want).abs() <= bound).all())
    meta = ops.cache_attention(q.to("meta"), cache.to("meta"), table.to("meta"), lens.to("meta"), None, 0.125, 8)
    assert tuple(meta.shape) == (50, 8, 64)
    with pytest.raises(RuntimeError, match="cache of"):
        ops.kv_cache_write(cache, k, v, slots, 4)


def test_many_rounds_of_blocks_no_wait_runs_out(abq, cuda):
    """Over a thousand blocks of prompts, again and again: the same bits, and no barrier's phase is missed (a missed one shows in the status word)."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    for dim in (128, 64):
        lens = [4096, 517, 1]
        cu = torch.tensor([0, 4096, 4613, 4614], dtype=torch.int32).cuda()
        qkv = torch.randn((4614, 40, dim), device="cuda", generator=gen).to(torch.bfloat16)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        outs = [torch.empty((4614, 32, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        params = [abq.make_prompt_attention_params(qkv[:, :32], qkv[:, 32:36], qkv[:, 36:], o, cu, cu, scale=dim ** -0.5, max_q=4096, status_word=status) for o in outs]
        for _ in range(10):
            for p in params:
                abq.prompt_attention(p)
        torch.cuda.synchronize()
        assert int(status.item()) == 0 and torch.equal(outs[0], outs[1])
        # a spot check of the long one against fp32 on the GPU: half a step each for p and the result, and fp32 sums
        q, k, v = (x[:4096, h].float() for x, h in ((qkv[:, :32], 9), (qkv[:, 32:36], 1), (qkv[:, 36:], 1)))
        s = (q @ k.T * dim ** -0.5).masked_fill(~torch.ones((4096, 4096), dtype=torch.bool, device="cuda").tril(), float("-inf"))
        p = torch.softmax(s, dim=-1)
        err = (outs[0][:4096, 9].float() - p @ v).abs()
        assert bool((err <= 2.0 ** -8 * (p @ v).abs() + (2.0 ** -8 + 2.0 ** -12) * (p @ v.abs()) + 1e-6).all())
