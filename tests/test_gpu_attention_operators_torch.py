"""The torch operators of the cache and of attention: both types and head sizes, their registration (schema, shape functions, traced graphs) and refusals."""
import importlib

import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(abq, cuda):
    importlib.import_module("abq_llm_b200.torch_ops")
    return torch.ops.abq_b200


def _case(half, dim, bits, seed=0):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn((50, 12, dim), generator=gen).to(half).cuda()
    cache = torch.zeros((4, 2, 1, R.granule_bytes(dim, bits)), dtype=torch.uint8, device="cuda")
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    slots = torch.cat([torch.arange(20), 32 + torch.arange(30)]).cuda()
    return qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], cache, slots, ints([[0, 1], [2, 3]]), ints([0, 20, 50]), ints([20, 30])


@pytest.mark.parametrize("half", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,bits", [(64, 4), (128, 8), (128, 4)])
def test_results(abq, ops, half, dim, bits):
    q, k, v, cache, slots, table, cu, lens = _case(half, dim, bits)
    scale = dim ** -0.5
    want, bound = R.prompt_attention(q.cpu(), k.cpu(), v.cpu(), [20, 30], [20, 30], scale)
    assert bool(((ops.prompt_attention(q, k, v, cu, cu, scale).cpu().double() - want).abs() <= bound).all())
    ops.kv_cache_write(cache, k, v, slots, bits)
    ko, vo = (torch.empty((50, 2, dim), dtype=half, device="cuda") for _ in range(2))
    ops.kv_cache_read(cache, ko, vo, table, cu, bits)
    for x, y in ((k, ko), (v, vo)):
        codes, s, low = R.quantise(x.cpu().contiguous(), bits)
        assert torch.equal(y.cpu(), (codes.float() * s.float() + low.float()).to(half))
    rows, tree = q[[18, 19, 48, 49]], torch.tensor([[1, 3], [1, 2]], device="cuda")
    got = ops.cache_attention(rows, cache, table, lens, tree, scale, bits)
    want, bound = R.cache_attention(cache.cpu(), 16, bits, half, table.cpu(), [20, 30], rows.cpu(), 2, scale, tree.cpu())
    assert bool(((got.cpu().double() - want).abs() <= bound).all())


@pytest.mark.parametrize("half,dim,bits", [(torch.float16, 128, 8), (torch.bfloat16, 64, 4)])
def test_registration(ops, half, dim, bits):
    q, k, v, cache, slots, table, cu, lens = _case(half, dim, bits)
    out = [torch.zeros((50, 2, dim), dtype=half, device="cuda") for _ in range(2)]
    checks = ("test_schema", "test_faketensor")
    torch.library.opcheck(ops.kv_cache_write.default, (cache, k, v, slots, bits), test_utils=checks)
    torch.library.opcheck(ops.kv_cache_read.default, (cache, *out, table, cu, bits), test_utils=checks)
    torch.library.opcheck(ops.cache_attention.default, (q[[19, 49]], cache, table, lens, None, 0.125, bits), test_utils=checks)
    torch.library.opcheck(ops.prompt_attention.default, (q, k, v, cu, cu, 0.125), test_utils=checks)


def test_a_traced_step(ops):
    """Written and attended to in one traced graph: the write is kept and stays in front of the read."""
    from torch.fx.experimental.proxy_tensor import make_fx
    q, k, v, cache, slots, table, cu, lens = _case(torch.float16, 128, 8)

    def step(cache, q, k, v, slots, table, lens):
        ops.kv_cache_write(cache, k, v, slots, 8)
        return ops.cache_attention(q, cache, table, lens, None, 0.1, 8)

    rows = q[[19, 49]]
    want = step(cache.clone(), rows, k, v, slots, table, lens)
    graph = make_fx(step, tracing_mode="fake")(cache, rows, k, v, slots, table, lens)
    assert torch.equal(graph(cache.clone(), rows, k, v, slots, table, lens), want)


def test_refusals(ops):
    q, k, v, cache, slots, table, cu, lens = _case(torch.float16, 128, 8)
    with pytest.raises(RuntimeError, match="cache of"):
        ops.cache_attention(q, cache, table, lens, None, 0.1, 4)
    with pytest.raises(ValueError, match="16-bit type"):
        ops.kv_cache_write(cache, k, v.to(torch.bfloat16), slots, 8)
    with pytest.raises(ValueError, match="slots"):
        ops.kv_cache_write(cache, k, v, slots.int(), 8)
    with pytest.raises(ValueError, match="fp16 or bf16"):
        ops.prompt_attention(q.float(), k.float(), v.float(), cu, cu, 0.1)
    with pytest.raises(Exception):
        ops.prompt_attention(q.cpu(), k.cpu(), v.cpu(), cu.cpu(), cu.cpu(), 0.1)
