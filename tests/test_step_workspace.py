"""The workspace of a step: one for all layers, and none that an earlier call was given goes away while the step lives (a captured launch still points to it)."""
import importlib
import weakref

import pytest
import torch


@pytest.fixture
def att(abq, monkeypatch):
    """attention.py with the library's calls replaced: what they were given as workspace is noted."""
    m = importlib.import_module("abq_llm_b200.attention")

    class Calls:
        need, given = 0, []

        def kv_cache_bytes(self, pages, page_size, heads, dim, bits):
            return 64

        def cache_attention_workspace_bytes(self, *a):
            return self.need

        def make_cache_attention_params(self, *a, workspace, **kw):
            self.given.append((workspace.data_ptr(), workspace.numel(), weakref.ref(workspace)))

        def __getattr__(self, name):
            return lambda *a, **kw: None

    m.calls = Calls()
    m.calls.given = []
    monkeypatch.setattr(m, "B", m.calls)
    return m


def test_a_larger_need_leaves_the_smaller_workspace_alive(att):
    pages = att.PagedSequences(4, 16)
    ids = [pages.add(3), pages.add(5)]
    step = att.AttentionStep.make(torch, pages, ids, [1, 1], prompt=False, device="cpu")
    layers = [att.BlockAttention(None, torch, heads=h, kv_heads=1, head_dim=64, num_pages=4, device="cpu") for h in (2, 4, 3)]
    for layer, need in zip(layers, (256, 1024, 512)):
        layer.step, att.calls.need = step, need
        layer(torch.zeros((2, (layer.heads + 2) * 64), dtype=torch.float16))
    (a, na, ra), (b, nb, rb), (c, nc, rc) = att.calls.given
    assert (na, nb, nc) == (256, 1024, 1024) and b == c, "later layers share the larger one"
    assert ra() is not None, "the first layer's workspace is gone: a launch captured with it writes into freed memory"
    assert a + na <= b or b + nb <= a


@pytest.mark.gpu
def test_a_captured_layer_after_a_wider_one(abq, cuda):
    att = importlib.import_module("abq_llm_b200.attention")
    gen = torch.Generator(device="cuda").manual_seed(0)
    pages = att.PagedSequences(512, 16)
    ids = [pages.add(3000), pages.add(2500)]
    narrow, wide = (att.BlockAttention(abq, torch, heads=h, kv_heads=4, head_dim=128, num_pages=512) for h in (4, 160))
    fill = att.AttentionStep.make(torch, pages, ids, [3000, 2500], prompt=True)
    for layer in (narrow, wide):
        layer.step = fill
        layer(torch.randn((5500, (layer.heads + 8) * 128), device="cuda", generator=gen).half())
    for s in ids:
        pages.extend(s, 2)
    step = att.AttentionStep.make(torch, pages, ids, [2, 2], prompt=False)
    narrow.step = wide.step = step
    x = torch.randn((4, 12 * 128), device="cuda", generator=gen).half()
    want = narrow(x).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = narrow(x)
    before = step.workspace.numel()
    wide(torch.randn((4, 168 * 128), device="cuda", generator=gen).half())
    assert step.workspace.numel() > before and step.outgrown
    junk = [torch.full((before,), 255, dtype=torch.uint8, device="cuda") for _ in range(20)]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(bool((j == 255).all()) for j in junk)
