"""abq_cache_attention on the GPU against attention in 64 bits over the same bytes of the cache."""
import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu
HALF = {"fp16": torch.float16, "bf16": torch.bfloat16}


class Setup:
    """A filled cache (every place that no sequence owns holds codes of 255 and NaN parameters), tables and queries as strided slices."""

    def __init__(self, abq, *, dim, bits, half, heads, kv_heads, n, lens, page, tree=False, seed=0, spare=1):
        gen = torch.Generator().manual_seed(seed)
        self.abq, self.dim, self.bits, self.half, self.n, self.lens, self.page = abq, dim, bits, half, n, lens, page
        need = [-(-max(x, 0) // page) for x in lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=gen).to(torch.int32)
        self.table = torch.full((len(lens), max(1, max(need))), -5, dtype=torch.int32)
        self.data = torch.full((pages, kv_heads, page // 16, R.granule_bytes(dim, bits)), 255, dtype=torch.uint8)
        at = 0
        for b, x in enumerate(need):
            self.table[b, :x] = order[at:at + x]
            at += x
        slots = [int(self.table[b, t // page]) * page + t % page for b, x in enumerate(lens) for t in range(max(x, 0))]
        self.slots = torch.tensor(slots, dtype=torch.int64)
        self.k = torch.randn((len(slots), kv_heads, dim), generator=gen).to(half)
        self.k[..., 3] *= 5
        self.v = (torch.randn((len(slots), kv_heads, dim), generator=gen) + 0.25).to(half)
        buf = torch.randn((len(lens) * n, heads + 2, dim), generator=gen).to(half)
        self.q = buf[:, 1:heads + 1]
        self.tree = R.random_tree(gen, len(lens), n) if tree else None
        self.heads, self.kv_heads, self.scale = heads, kv_heads, dim ** -0.5

    def fill(self):
        R.encode(self.data, self.page, self.bits, self.slots, self.k, self.v)
        return self

    def call(self, *, out=None, stream=None, status=None, run=True):
        abq = self.abq
        self.held, self.dtable, self.dlens = self.data.cuda(), self.table.cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda()
        base = torch.empty((self.q.shape[0], self.heads + 2, self.dim), dtype=self.half, device="cuda")
        self.dq = base[:, 1:self.heads + 1]
        self.dq.copy_(self.q)
        self.guard = torch.full((self.q.shape[0], self.heads + 1, self.dim), -9.0, dtype=self.half, device="cuda")
        self.out = self.dq if out == "q" else self.guard[:, :self.heads]
        cache = abq.make_kv_cache(self.held, page_size=self.page, kv_heads=self.kv_heads, head_dim=self.dim, bits=self.bits, dtype=self.half)
        work = torch.full((abq.cache_attention_workspace_bytes(cache, len(self.lens), self.n, self.heads),), 255, dtype=torch.uint8, device="cuda")
        self.params = abq.make_cache_attention_params(cache, self.dq, self.out, self.dtable, self.dlens, scale=self.scale, workspace=work,
                                                      tree=None if self.tree is None else self.tree.cuda(), status_word=status)
        if run:
            abq.cache_attention(self.params, stream)
        return self.out

    def check(self, out, rows=None):
        want, bound = R.cache_attention(self.data, self.page, self.bits, self.half, self.table, self.lens, self.q, self.n, self.scale, self.tree)
        got = out.cpu().double()
        sel = slice(None) if rows is None else rows
        bad = (got[sel] - want[sel]).abs() > bound[sel]
        assert not bool(bad.any()) and not bool(got[sel].isnan().any()), \
            f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / bound.clamp(min=1e-30))[sel].nan_to_num(1e9).max()):.2f} of the bound"
        assert bool((self.guard[:, self.heads] == -9).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("half", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,n,lens,page,tree", [
    (1, 1, 1, [1], 16, False),
    (4, 2, 1, [0, 16, 17, 1, 300, -3], 16, False),
    (3, 3, 1, [5, 129], 48, False),
    (8, 1, 1, [1000, 33], 128, False),
    (14, 2, 2, [40, 2, 1, 0], 32, False),
    (5, 5, 7, [7, 6, 100, 19, 0], 16, True),
    (6, 2, 13, [13, 50, 333], 64, True),
    (2, 1, 64, [64, 200, 63, 1], 16, True),
    (16, 2, 9, [500, 12], 16, True),
    (12, 12, 1, [257] * 9 + [0, 3], 16, False),
    # blocks of 128 rows on the tensor cores: 96, 128, 192 (two blocks) and 256 rows
    (8, 2, 24, [24, 23, 150, 0, 300], 32, True),
    (8, 1, 16, [1, 17, 128, 129, 1500], 16, False),
    (12, 1, 16, [333, 16], 48, True),
    (8, 2, 64, [64, 700, 1, 128], 128, True),
    (16, 2, 16, [200] * 35 + [0, 5], 16, False),
])
def test_against_64_bits(abq, cuda, dim, bits, half, heads, kv_heads, n, lens, page, tree):
    s = Setup(abq, dim=dim, bits=bits, half=HALF[half], heads=heads, kv_heads=kv_heads, n=n, lens=lens, page=page, tree=tree, seed=len(lens) + dim + n).fill()
    s.check(s.call())


@pytest.mark.parametrize("bits,heads,kv_heads,n,lens", [(8, 8, 8, 1, [5000]), (4, 32, 4, 1, [3001, 7, 2048, 4000]), (8, 4, 1, 20, [6100, 900]), (8, 8, 1, 16, [9000, 300])])
def test_sequences_that_many_blocks_share(abq, cuda, bits, heads, kv_heads, n, lens):
    s = Setup(abq, dim=128, bits=bits, half=torch.float16, heads=heads, kv_heads=kv_heads, n=n, lens=lens, page=16, tree=n > 1, seed=bits).fill()
    first = s.call().clone()
    s.check(s.out)
    s.abq.cache_attention(s.params)
    assert torch.equal(first, s.out), "the same bits again: pieces are added in order"


@pytest.mark.parametrize("heads", [2, 48])
def test_rows_that_see_nothing_and_masked_nan(abq, cuda, heads):
    """Tree rows without a bit and nothing before the drafts give 0; drafts whose keys and values are NaN touch only the rows that see them."""
    s = Setup(abq, dim=64, bits=8, half=torch.float16, heads=heads, kv_heads=2, n=4, lens=[4, 30], page=16, tree=True, seed=3)
    s.tree[0] = torch.tensor([0, 2, 0, 8])
    s.tree[1] = torch.tensor([1, 2, 5, 9])
    s.k[4 + 27], s.v[4 + 27] = float("nan"), float("inf")  # sequence 1, draft 1: seen by row 1 alone
    s.v[0] = float("nan")                                  # sequence 0, draft 0: seen by nobody
    s.fill()
    out = s.call()
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all())
    assert bool(out[4 + 1].isnan().all())
    s.check(out, rows=[0, 1, 2, 3, 4, 6, 7])


@pytest.mark.parametrize("n", [1, 64])
def test_many_small_weights_beside_one_large(abq, cuda, n):
    """One key draws almost all weight; 20000 others together hold a part that must not be lost when their weights are held in 16 bits."""
    for half in (torch.float16, torch.bfloat16):
        torch.manual_seed(4)
        s = Setup(abq, dim=64, bits=8, half=half, heads=2 if n > 1 else 1, kv_heads=1, n=n, lens=[20001], page=16)
        s.q[:] = 1.0
        s.k = torch.zeros_like(s.k)
        s.k[:, 0, 0] = torch.rand(20001) * 0.01  # (codes of their own)
        s.k[7, 0] = 1.9
        s.v = (torch.rand(s.v.shape) * 0.01 + 1.0).to(half)
        s.v[7] = -1.0
        s.fill()
        out = s.call()
        s.check(out)
        want, _ = R.cache_attention(s.data, 16, 8, half, s.table, s.lens, s.q, n, s.scale)
        # the others' share is 20000 exp(-1.9 * 64 / 8) = 0.0050, their values lie 2 away: 0.00998, many steps of the result's type
        assert float((want - (-1.0)).abs().min()) > 0.009, "the case says nothing if the small ones do not count"


@pytest.mark.parametrize("heads,n", [(4, 1), (4, 32)])
def test_value_scales_of_all_sizes(abq, cuda, heads, n):
    """Value rows from 2^-14 to 2^14 of the first: the power of two that holds p times the scale in 16 bits follows the largest."""
    s = Setup(abq, dim=128, bits=8, half=torch.bfloat16, heads=heads, kv_heads=1, n=n, lens=[700], page=16, seed=5)
    s.v = (s.v.float() * 2.0 ** torch.randint(-14, 15, (700, 1, 1), generator=torch.Generator().manual_seed(1)).float()).to(torch.bfloat16)
    s.v[:40] = 0.5  # constant rows first: scale 0
    s.fill()
    s.check(s.call())


@pytest.mark.parametrize("n", [1, 16])
def test_queries_of_all_sizes(abq, cuda, n):
    s = Setup(abq, dim=128, bits=8, half=torch.bfloat16, heads=6, kv_heads=1, n=n, lens=[100], page=16, seed=6)
    s.q[0] *= torch.tensor([1e-30, 1e-3, 1.0, 50.0, 0.0, 3e-39]).view(6, 1).to(torch.bfloat16)
    s.fill()
    s.check(s.call())


@pytest.mark.parametrize("heads", [8, 64])
def test_in_place(abq, cuda, heads):
    s = Setup(abq, dim=128, bits=4, half=torch.float16, heads=heads, kv_heads=2, n=3, lens=[900, 31], page=16, tree=True, seed=8).fill()
    s.check(s.call(out="q"))


@pytest.mark.parametrize("heads", [2, 256])
def test_pages_outside_the_cache_are_unseen(abq, cuda, heads):
    s = Setup(abq, dim=64, bits=8, half=torch.float16, heads=heads, kv_heads=2, n=1, lens=[64], page=16, seed=9).fill()
    whole = s.table.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    s.call(status=status)
    assert int(status.item()) == 0
    for bad in (-1, s.data.shape[0], 1 << 30):
        s.table = whole.clone()
        s.table[0, 1] = bad
        status.zero_()
        got = s.call(status=status).clone()
        assert int(status.item()) == abq.STATUS_BAD_PAGE
        # the same result as without those 16 tokens (one row, no mask: the order of the others does not matter)
        s.table, s.lens = torch.cat([whole[:, :1], whole[:, 2:], whole[:, 1:2]], dim=1), [48]
        want, bound = R.cache_attention(s.data, 16, 8, torch.float16, s.table, s.lens, s.q, 1, s.scale)
        assert bool(((got.cpu().double() - want).abs() <= bound).all())
        s.lens = [64]
    # lengths that the table has no room for are cut
    s.table, s.lens = whole, [1000]
    long = s.call().clone()
    s.lens = [64]
    assert torch.equal(long, s.call())


@pytest.mark.parametrize("heads", [8, 192])
def test_a_captured_launch_follows_the_lengths(abq, cuda, heads):
    s = Setup(abq, dim=128, bits=8, half=torch.float16, heads=heads, kv_heads=2, n=1, lens=[400, 90], page=16, seed=10).fill()
    s.call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            abq.cache_attention(s.params)
    for lens in ([400, 90], [1, 0], [17, 90], [399, 16]):
        s.dlens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        s.lens = lens
        s.check(s.out)


@pytest.mark.parametrize("heads,kv_heads,n", [(8, 8, 1), (16, 2, 16)])
def test_two_streams_with_workspaces_of_their_own(abq, cuda, heads, kv_heads, n):
    a = Setup(abq, dim=128, bits=8, half=torch.float16, heads=heads, kv_heads=kv_heads, n=n, lens=[3000], page=16, seed=11).fill()
    b = Setup(abq, dim=128, bits=8, half=torch.float16, heads=heads, kv_heads=kv_heads, n=n, lens=[2900], page=16, seed=12).fill()
    a.call(run=False), b.call(run=False)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for x, st in zip((a, b), streams):
            abq.cache_attention(x.params, st)
    torch.cuda.synchronize()
    a.check(a.out), b.check(b.out)


def test_offsets_beyond_32_bits(abq, cuda):
    """A cache of more than 4 GiB, the sequence in its last pages."""
    page, kv_heads, dim, bits = 1024, 8, 128, 8
    one = abq.kv_cache_bytes(1, page, kv_heads, dim, bits)
    pages = (9 << 29) // one + 2
    held = torch.zeros((pages, one), dtype=torch.uint8, device="cuda")
    assert held.numel() > 1 << 32
    cache = abq.make_kv_cache(held, page_size=page, kv_heads=kv_heads, head_dim=dim, bits=bits, dtype=torch.float16)
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn((1500, kv_heads, dim), generator=gen).half() for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    pos = torch.arange(1500)
    slots = table[0][pos // page].long() * page + pos % page
    abq.kv_cache_write(abq.make_kv_write_params(cache, k.cuda(), v.cuda(), slots.cuda()))
    q = torch.randn((1, 8, dim), generator=gen).half()
    out = torch.empty((1, 8, dim), dtype=torch.float16, device="cuda")
    work = torch.empty(abq.cache_attention_workspace_bytes(cache, 1, 1, 8), dtype=torch.uint8, device="cuda")
    abq.cache_attention(abq.make_cache_attention_params(cache, q.cuda(), out, table.cuda(), torch.tensor([1500], dtype=torch.int32).cuda(), scale=0.1, workspace=work))
    ko, vo = (torch.empty((1500, kv_heads, dim), dtype=torch.float16, device="cuda") for _ in range(2))
    abq.kv_cache_read(abq.make_kv_read_params(cache, ko, vo, table.cuda(), torch.tensor([0, 1500], dtype=torch.int32).cuda()))
    last = held[pages - 2:].cpu().view(2, kv_heads, page // 16, -1)
    want, bound = R.cache_attention(last, page, bits, torch.float16, torch.tensor([[1, 0]]), [1500], q, 1, 0.1)
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    codes, scale, low = R.quantise(k, bits)
    assert torch.equal(ko.cpu(), (codes.float() * scale.float() + low.float()).half())


@pytest.mark.parametrize("group,n", [(79, 1), (5, 16), (53, 3), (40, 4)])
def test_rows_around_the_choice_of_kernel(abq, cuda, group, n):
    s = Setup(abq, dim=64, bits=8, half=torch.float16, heads=2 * group, kv_heads=2, n=n, lens=[500, 61, n, 0], page=32, tree=True, seed=group).fill()
    s.check(s.call())


@pytest.mark.parametrize("dim", [64, 128])
def test_maximum_that_rises_in_either_half_of_a_tile(abq, cuda, dim):
    """Tokens far above all before them, in the second half of a tile of 128, the first half of the next, the second again, and in both of one."""
    s = Setup(abq, dim=dim, bits=8, half=torch.bfloat16, heads=4, kv_heads=1, n=32, lens=[1000], page=16, seed=dim)
    s.q[:] = 1.0
    for token, size in ((200, 3.0), (300, 6.0), (450, 9.0), (530, 12.0), (620, 12.5)):
        s.k[token] = size
    s.fill()
    s.check(s.call())


@pytest.mark.parametrize("heads,kv_heads,n,lens", [(8, 2, 1, [0] * 45 + [70, 1, 0, 300] + [0] * 20), (4, 2, 3, [0, 0]), (8, 1, 12, [0] * 3), (16, 1, 8, [0] * 33 + [20])])
def test_mostly_empty_batches(abq, cuda, heads, kv_heads, n, lens):
    s = Setup(abq, dim=128, bits=4, half=torch.float16, heads=heads, kv_heads=kv_heads, n=n, lens=lens, page=16, tree=n > 1, seed=len(lens)).fill()
    s.check(s.call())


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("heads,kv_heads,n", [(8, 8, 1), (16, 2, 2), (16, 2, 10)])
def test_lengths_that_change_between_calls_without_a_pause(abq, cuda, heads, kv_heads, n, captured):
    """Each call and its second kernel see the lengths as they are at the call's place on the stream, however early the kernels are let in."""
    s = Setup(abq, dim=128, bits=8, half=torch.float16, heads=heads, kv_heads=kv_heads, n=n, lens=[700, 45, 400], page=16, seed=13).fill()
    s.call(run=False)
    steps = torch.tensor([[-37, 0, -399], [30, -20, 350], [5, 19, -1], [2, 1, 50]] * 6, dtype=torch.int32, device="cuda")
    outs = [torch.zeros((s.q.shape[0], heads, 128), dtype=torch.float16, device="cuda") for _ in steps]
    cache = abq.make_kv_cache(s.held, page_size=16, kv_heads=kv_heads, head_dim=128, bits=8, dtype=torch.float16)
    work = torch.empty(abq.cache_attention_workspace_bytes(cache, 3, n, heads), dtype=torch.uint8, device="cuda")
    calls = [abq.make_cache_attention_params(cache, s.dq, o, s.dtable, s.dlens, scale=s.scale, workspace=work) for o in outs]
    start = s.dlens.clone()

    def run(pause):
        s.dlens.copy_(start)
        for step, call in zip(steps, calls):
            s.dlens.add_(step).clamp_(0, 700)
            abq.cache_attention(call)
            abq.cache_attention(call)
            if pause:
                torch.cuda.synchronize()

    run(True)
    want = [o.clone() for o in outs]
    for o in outs:
        o.zero_()
    torch.cuda.synchronize()
    if captured:
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run(False)
        graph.replay()
        graph.replay()
    else:
        run(False)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, outs))
    assert not bool(want[0].isnan().any()) and bool(want[0].any())
