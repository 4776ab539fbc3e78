"""abq_kv_cache_read with ends that do not start at 0: rows of no sequence are left as they were, and no position lies in front of its page."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [1, 2, 31, 40])
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4)])
@pytest.mark.parametrize("first", [5, 16, 37, -3, -(2 ** 31)])
def test_rows_before_the_first_sequence(abq, cuda, batch, dim, bits, first):
    """The first start above 0: the rows before it keep what they held.  Below 0 it counts as 0, as abq_prompt_attention takes it."""
    gen = torch.Generator().manual_seed(batch + dim)
    k, v = (torch.randn((64, 3, dim), generator=gen).half().cuda() for _ in range(2))
    held = torch.zeros(abq.kv_cache_bytes(4, 16, 3, dim, bits), dtype=torch.uint8, device="cuda")
    cache = abq.make_kv_cache(held, page_size=16, kv_heads=3, head_dim=dim, bits=bits, dtype=torch.float16)
    abq.kv_cache_write(abq.make_kv_write_params(cache, k, v, torch.arange(64).cuda()))
    table = torch.arange(4, dtype=torch.int32).repeat(batch, 1).cuda()  # page 0 among them: what lies in front of it is not the cache's
    begin = max(first, 0)
    ends = [begin + 20 + i for i in range(batch)]
    cu = torch.tensor([first] + ends, dtype=torch.int32).cuda()
    rows = ends[-1] + 3
    out = torch.full((2, rows, 3, dim), -9.0, dtype=torch.float16, device="cuda")
    abq.kv_cache_read(abq.make_kv_read_params(cache, out[0], out[1], table, cu))
    whole = torch.empty((2, 64, 3, dim), dtype=torch.float16, device="cuda")
    abq.kv_cache_read(abq.make_kv_read_params(cache, whole[0], whole[1], table[:1].contiguous(), torch.tensor([0, 64], dtype=torch.int32).cuda()))
    assert bool((out[:, :begin] == -9).all()) and bool((out[:, ends[-1]:] == -9).all())
    for a, b in zip([begin] + ends, ends):
        assert torch.equal(out[:, a:b], whole[:, :b - a])
