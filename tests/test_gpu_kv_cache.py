"""abq_kv_cache_write / abq_kv_cache_read on the GPU: the cache's bytes against the rule in the header bit for bit, and what is read back."""
import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu
HALF = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _rows(gen, tokens, heads, dim, half, gain=1.0):
    """Slices of one fused buffer, with a large channel, a constant row and a row of zeros."""
    buf = torch.randn((tokens, 3 * heads + 1, dim), generator=gen) * gain
    buf[:, heads:2 * heads, dim // 3] *= 7
    if tokens > 2:
        buf[1, heads] = 1.25
        buf[2, 2 * heads] = 0.0
    buf = buf.to(half).cuda()
    return buf[:, heads:2 * heads], buf[:, 2 * heads:3 * heads]


def _same(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16)) or bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("half", ["fp16", "bf16"])
@pytest.mark.parametrize("tokens,heads,page,gain", [(1, 1, 16, 1.0), (37, 3, 16, 0.02), (130, 8, 48, 30.0), (16, 5, 128, 1e-7), (260, 40, 1024, 1.0)])
def test_write_then_read(abq, cuda, dim, bits, half, tokens, heads, page, gain):
    dtype, gen = HALF[half], torch.Generator().manual_seed(tokens * 7 + dim + bits)
    pages = -(-tokens // page) + 2
    k, v = _rows(gen, tokens, heads, dim, dtype, gain)
    slots = torch.randperm(pages * page, generator=gen)[:tokens].to(torch.int64)
    if tokens > 5:
        slots[3], slots[4] = -1, pages * page  # left out: padding, and a slot behind the cache
    data = torch.randint(0, 256, (pages, heads, page // 16, R.granule_bytes(dim, bits)), dtype=torch.uint8, generator=gen)
    assert data.numel() == abq.kv_cache_bytes(pages, page, heads, dim, bits)
    held = data.cuda()
    cache = abq.make_kv_cache(held, page_size=page, kv_heads=heads, head_dim=dim, bits=bits, dtype=dtype)
    abq.kv_cache_write(abq.make_kv_write_params(cache, k, v, slots.cuda()))
    torch.cuda.synchronize()
    R.encode(data, page, bits, slots, k.cpu().contiguous(), v.cpu().contiguous())
    assert torch.equal(held.cpu(), data), "codes, scales and mins of the written places, and every other byte left as it was"

    # two sequences over the pages in another order, a row of nobody behind them; strided results
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    lens = [page * (pages - 1) - 3, 0, page - 5 if page > 5 else 1]
    table = torch.full((3, pages), 1 << 30, dtype=torch.int32)
    table[0] = order
    table[2, 0] = order[-1]
    cu = torch.tensor([0, lens[0], lens[0], lens[0] + lens[2]], dtype=torch.int32)
    out = torch.full((int(cu[-1]) + 2, 2 * heads + 1, dim), -7.0, dtype=dtype, device="cuda")
    ko, vo = out[:, :heads], out[:, heads + 1:]
    # leftover bytes may decode to anything: make their parameters finite
    rb = dim * bits // 8
    pairs = held[..., 32 * rb:].view(dtype)
    pairs.copy_(torch.where(pairs.isfinite() & (pairs.abs() < 1e3), pairs, torch.ones_like(pairs)))
    data = held.cpu()
    cache = abq.make_kv_cache(held, page_size=page, kv_heads=heads, head_dim=dim, bits=bits, dtype=dtype)
    abq.kv_cache_read(abq.make_kv_read_params(cache, ko, vo, table.cuda(), cu.cuda()))
    torch.cuda.synchronize()
    for b, n in ((0, lens[0]), (2, lens[2])):
        at = int(cu[b])
        for got, (codes, scale, low) in zip((ko, vo), R.decode(data, page, bits, dim, dtype, table[b], n)):
            # code * scale is exact in fp32; the sum is rounded to fp32 and then to 16 bits
            want = ((codes * scale).float() + low.float()).to(dtype).permute(1, 0, 2)
            assert torch.equal(got[at:at + n].cpu().view(torch.int16), want.contiguous().view(torch.int16)) or _same(got[at:at + n].cpu(), want)
    assert bool((out[int(cu[-1]):] == -7).all()) and bool((out[:, heads] == -7).all()), "rows behind the last sequence and the values between the heads"


@pytest.mark.parametrize("half", ["fp16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_error_of_a_row_is_half_a_step(abq, cuda, half, bits):
    """|x - read back| <= scale / 2 and the rounding of the read value; min is kept exactly."""
    dtype, gen = HALF[half], torch.Generator().manual_seed(bits)
    k, v = _rows(gen, 64, 4, 128, dtype)
    held = torch.zeros(abq.kv_cache_bytes(4, 16, 4, 128, bits), dtype=torch.uint8, device="cuda")
    cache = abq.make_kv_cache(held, page_size=16, kv_heads=4, head_dim=128, bits=bits, dtype=dtype)
    abq.kv_cache_write(abq.make_kv_write_params(cache, k, v, torch.arange(64).cuda()))
    ko, vo = torch.empty((64, 4, 128), dtype=dtype, device="cuda"), torch.empty((64, 4, 128), dtype=dtype, device="cuda")
    abq.kv_cache_read(abq.make_kv_read_params(cache, ko, vo, torch.arange(4, dtype=torch.int32).view(1, 4).cuda(), torch.tensor([0, 64], dtype=torch.int32).cuda()))
    step, tiny = R.halves(dtype)
    for x, y in ((k, ko), (v, vo)):
        x, y = x.double(), y.double()
        low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
        scale = (high - low) / ((1 << bits) - 1) * (1 + 2 * step) + tiny  # rounded up by less than a step of the type
        # half a code, the quotient's fp32 rounding (2^-15 of a code), the sum's and the result's own rounding
        assert bool(((x - y).abs() <= scale * (0.5 + 2.0 ** -14) + y.abs() * step * (1 + 2.0 ** -12) + tiny).all())
        assert bool((y.amin(-1, keepdim=True) == low).all())


def test_rows_with_inf_or_nan_read_as_nan(abq, cuda):
    x = torch.randn((6, 2, 64), dtype=torch.float16, device="cuda")
    k, v = x.clone(), x.clone()
    k[1, 0, 5], k[2, 1, 0], v[3, 0, 63] = float("inf"), float("nan"), float("-inf")
    held = torch.zeros(abq.kv_cache_bytes(1, 16, 2, 64, 8), dtype=torch.uint8, device="cuda")
    cache = abq.make_kv_cache(held, page_size=16, kv_heads=2, head_dim=64, bits=8, dtype=torch.float16)
    abq.kv_cache_write(abq.make_kv_write_params(cache, k, v, torch.arange(6).cuda()))
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    abq.kv_cache_read(abq.make_kv_read_params(cache, ko, vo, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.tensor([0, 6], dtype=torch.int32).cuda()))
    bad_k, bad_v = torch.zeros((6, 2), dtype=torch.bool), torch.zeros((6, 2), dtype=torch.bool)
    bad_k[1, 0] = bad_k[2, 1] = bad_v[3, 0] = True
    assert torch.equal(ko.isnan().all(-1).cpu(), bad_k) and torch.equal(ko.isnan().any(-1).cpu(), bad_k)
    assert torch.equal(vo.isnan().all(-1).cpu(), bad_v) and torch.equal(vo.isnan().any(-1).cpu(), bad_v)


def test_pages_outside_the_cache_read_as_zero(abq, cuda):
    held = torch.full((abq.kv_cache_bytes(2, 16, 1, 64, 8),), 60, dtype=torch.uint8, device="cuda")
    cache = abq.make_kv_cache(held, page_size=16, kv_heads=1, head_dim=64, bits=8, dtype=torch.float16)
    k, v = torch.ones((80, 1, 64), dtype=torch.float16, device="cuda"), torch.ones((80, 1, 64), dtype=torch.float16, device="cuda")
    table = torch.tensor([[1, 2, -1, 0]], dtype=torch.int32).cuda()  # (and tokens 64 .. 79 lie behind the table's row)
    abq.kv_cache_read(abq.make_kv_read_params(cache, k, v, table, torch.tensor([0, 80], dtype=torch.int32).cuda()))
    zero = (k == 0).all(-1).view(5, 16).all(1).cpu()
    assert zero.tolist() == [False, True, True, False, True]


@pytest.mark.parametrize("batch", [31, 32, 70])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_sequences_read_together_as_one_by_one(abq, cuda, batch, dim):
    """Empty ones among them, at the start, in a row, and at the end."""
    gen = torch.Generator().manual_seed(batch)
    lens = torch.randint(1, 40, (batch,), generator=gen)
    lens[[0, 1, 5, 6, 7, batch - 1]] = 0
    table = torch.randperm(3 * batch, generator=gen).to(torch.int32).view(batch, 3).cuda()
    held = torch.zeros(abq.kv_cache_bytes(3 * batch, 16, 2, dim, 8), dtype=torch.uint8, device="cuda")
    cache = abq.make_kv_cache(held, page_size=16, kv_heads=2, head_dim=dim, bits=8, dtype=torch.float16)
    k, v = _rows(gen, 48 * batch, 2, dim, torch.float16)
    abq.kv_cache_write(abq.make_kv_write_params(cache, k, v, torch.arange(48 * batch).cuda()))
    cu = [0] + lens.cumsum(0).tolist()
    rows = torch.full((2, cu[-1] + 9, 2, dim), -9.0, dtype=torch.float16, device="cuda")
    abq.kv_cache_read(abq.make_kv_read_params(cache, rows[0], rows[1], table, torch.tensor(cu, dtype=torch.int32).cuda()))
    for b in range(batch):
        n = cu[b + 1] - cu[b]
        if n:
            one = torch.empty((2, n, 2, dim), dtype=torch.float16, device="cuda")
            abq.kv_cache_read(abq.make_kv_read_params(cache, one[0], one[1], table[b:b + 1], torch.tensor([0, n], dtype=torch.int32).cuda()))
            assert torch.equal(one, rows[:, cu[b]:cu[b + 1]]), b
    assert bool((rows[:, cu[-1]:] == -9).all())
