"""Every token of a sequence counts once in abq_cache_attention: weights that are known exactly, so that one token left out, taken twice or read from another place shows,
wherever runs, pieces, tiles and pages begin and end.  That the bounds are tight enough to see it is asserted of each case."""
import pytest
import torch

import attention_ref as R
from test_gpu_cache_attention import HALF, Setup

pytestmark = pytest.mark.gpu

# heads, key heads and rows of the kernels of 8, 16 and 128 rows
KERNELS = [(8, 8, 1), (4, 4, 12), (8, 1, 16)]


def _fill(s):
    """Through abq_kv_cache_write, whose bytes are tested elsewhere."""
    held = s.data.cuda()
    cache = s.abq.make_kv_cache(held, page_size=s.page, kv_heads=s.kv_heads, head_dim=s.dim, bits=s.bits, dtype=s.half)
    s.abq.kv_cache_write(s.abq.make_kv_write_params(cache, s.k.cuda(), s.v.cuda(), s.slots.cuda()))
    s.data = held.cpu()
    return s


def _seen(s, b, length):
    seen = torch.ones((s.n, length), dtype=torch.bool)
    for i in range(s.n):
        bits = (1 << (i + 1)) - 1 if s.tree is None else int(s.tree[b, i]) & ((1 << 64) - 1)
        for j in range(s.n):
            if length - s.n + j >= 0:
                seen[i, length - s.n + j] = bool(bits >> j & 1)
    return seen


def _close(s, out, b, want, bound):
    """want, bound [key heads][n][dim], the same for the query heads of a key head."""
    got = out.cpu().double()[b * s.n:(b + 1) * s.n].view(s.n, s.kv_heads, s.heads // s.kv_heads, s.dim).permute(1, 2, 0, 3)
    err = (got - want.unsqueeze(1)).abs()
    assert bool((err <= bound.unsqueeze(1)).all()), f"sequence {b}: {float((err / bound.unsqueeze(1)).max()):.2f} of the bound"


LENS = [[5000], [4999, 300, 0, 16], [2047, 2048, 2049, 127, 128, 129, 15, 17, 33, 1], [64] * 40 + [2500]]


@pytest.mark.parametrize("heads,kv_heads,n", KERNELS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bits,half", [(8, "fp16"), (4, "fp16"), (8, "bf16")])
@pytest.mark.parametrize("lens,page", list(zip(LENS, (16, 48, 32, 128))))
def test_equal_weights(abq, cuda, heads, kv_heads, n, dim, bits, half, lens, page):
    """Queries of 0: every score is 0 and every weight exactly 1 (2^0 is exact).  Values are +1 or -1 per token and feature: a token changes every feature by about 1 / tokens.

    The bound: the weight times a value's scale is that scale times a power of two, which fp16 holds, so only sums are rounded.  Sums of codes: G granules of 16
    tokens, each adding with at most 2^-21 of the sum so far (at most twice the largest prefix sum, a piece may begin anywhere) and of the 16 products; sums of
    offsets: 2^-23 of at most tokens times the largest, in at most tokens / 4 + 64 additions of a lane and over lanes and pieces; the quotient 2^-21; the
    result's rounding half a step."""
    s = Setup(abq, dim=dim, bits=bits, half=HALF[half], heads=heads, kv_heads=kv_heads, n=n, lens=lens, page=page, tree=n > 1, seed=dim + bits)
    s.q[:] = 0
    s.v = (torch.randint(0, 2, s.v.shape, generator=torch.Generator().manual_seed(n + len(lens))) * 2.0 - 1.0).to(s.half)
    _fill(s)
    out = s.call()
    centre, (step, tiny) = float(1 << (bits - 1)), R.halves(s.half)
    for b, length in enumerate(lens):
        if length == 0:
            assert bool((out[b * n:(b + 1) * n] == 0).all())
            continue
        _, (vc, vs, vm) = R.decode(s.data, page, bits, dim, s.half, s.table[b], length)
        seen = _seen(s, b, length).double()
        count = seen.sum(-1).clamp(min=1).view(1, n, 1)
        want = torch.matmul(seen, vc * vs + vm) / count
        codes, offsets = vs * (vc - centre), (vm + centre * vs).abs().amax()
        prefix = codes.cumsum(1).abs().amax(1, keepdim=True) + 64  # (a row's mask changes it by at most 64 drafts of about 1)
        granules = length // 16 + 8
        bound = 2.0 ** -21 * granules * (2 * prefix + 16 * codes.abs().amax()) / count + 2.0 ** -23 * (length / 4 + 64) * offsets + (step + 2.0 ** -21) * want.abs() + tiny
        _close(s, out, b, want, bound)
        if length >= 100:  # one token more or less shows in several features of every row
            assert bool((((0.99 - want.abs()) / (count + 1) > 2 * bound).sum(-1) >= 8).all()), "the case says nothing"


@pytest.mark.parametrize("heads,kv_heads,n", KERNELS)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("half,lens", [("fp16", [1500, 16, 0, 700]), ("fp16", [1]), ("bf16", [200, 129, 31])])
def test_weights_of_their_own(abq, cuda, heads, kv_heads, n, bits, half, lens):
    """Keys and values that are constant along a row (scale 0): token t has weight exp(scale k_t sum(q)) and value v_t in every feature.

    The bound: a score is one product in fp32 (2^-22 of it, with that of the scale), so a weight is off by 2^-22 (|score| + 1) of itself, and so is their sum; sums as
    above, 2^-24 of the magnitudes in at most tokens / 4 + 64 additions each; the quotient and the result's rounding."""
    dim = 128
    s = Setup(abq, dim=dim, bits=bits, half=HALF[half], heads=heads, kv_heads=kv_heads, n=n, lens=lens, page=16, tree=n > 1, seed=bits + len(lens))
    gen = torch.Generator().manual_seed(n)
    s.q[:] = 0.5
    s.k[:] = ((torch.randint(-16, 17, s.k.shape[:2] + (1,), generator=gen)) / 128.0).to(s.half)  # scores up to 0.125 * 64 / sqrt(128) = 0.71 either way
    s.v[:] = (torch.randint(0, 2, s.v.shape[:2] + (1,), generator=gen) * 2.0 - 1.0).to(s.half)
    _fill(s)
    out = s.call()
    step, tiny = R.halves(s.half)
    for b, length in enumerate(lens):
        if length == 0:
            continue
        (_, _, km), (_, _, vm) = R.decode(s.data, 16, bits, dim, s.half, s.table[b], length)
        score = (km * 0.5 * dim * s.scale).transpose(1, 2)  # [key heads][1][tokens]
        w = torch.exp(score) * _seen(s, b, length).double()
        total = w.sum(-1, keepdim=True)
        share = w / torch.where(total == 0, torch.ones_like(total), total)
        want = torch.matmul(share, vm)
        bound = 2 * 2.0 ** -22 * (1.45 * 0.71 + 1) + 2 * (length / 4 + 64) * 2.0 ** -24 + (step + 2.0 ** -21) * want.abs() + tiny
        _close(s, out, b, want.expand(-1, -1, dim), bound.expand(-1, -1, dim))
        if length >= 100:
            change = share * (vm.transpose(1, 2) - want).abs() / (1 + share)
            assert bool((torch.where(w > 0, change, torch.ones_like(change)) > 2 * bound).all()), "the case says nothing"
