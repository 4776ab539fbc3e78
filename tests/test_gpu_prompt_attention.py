"""abq_prompt_attention on the GPU against attention in 64 bits."""
import pytest
import torch

import attention_ref as R

pytestmark = pytest.mark.gpu
HALF = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _ends(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32).cuda()


def _inputs(seed, half, dim, heads, kv_heads, nq, nk, spare=3):
    """Rows of fused buffers (strided views); `spare` rows of NaN behind the last sequence."""
    gen = torch.Generator().manual_seed(seed)
    qb = torch.randn((sum(nq) + spare, heads + 1, dim), generator=gen)
    kb = torch.randn((sum(nk) + spare, 2 * kv_heads + 1, dim), generator=gen)
    kb[:, :kv_heads, 5] *= 4
    kb[:, kv_heads:] += 0.2
    qb[sum(nq):], kb[sum(nk):] = float("nan"), float("nan")
    qb, kb = qb.to(half).cuda(), kb.to(half).cuda()
    return qb[:, :heads], kb[:, :kv_heads], kb[:, kv_heads:2 * kv_heads]


def _check(out, q, k, v, nq, nk, scale):
    want, bound = R.prompt_attention(q.cpu(), k.cpu(), v.cpu(), nq, nk, scale)
    got, rows = out.cpu().double()[:sum(nq)], sum(nq)
    want, bound = want[:rows], bound[:rows]
    assert bool((got.isfinite() == want.isfinite()).all()), "Inf and NaN reach the rows that see them and no others"
    fine = want.isfinite()
    bad = ((got - want).abs() > bound)[fine]
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / bound.clamp(min=1e-30))[fine].max()):.2f} of the bound"


def _run(abq, half, dim, heads, kv_heads, nq, nk, seed=0, max_q=0, edit=None, total=None):
    q, k, v = _inputs(seed, half, dim, heads, kv_heads, nq, nk)
    if edit:
        edit(q, k, v)
    guard = torch.full((q.shape[0], heads + 1, dim), -9.0, dtype=half, device="cuda")
    out, scale = guard[:, :heads], dim ** -0.5
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    abq.prompt_attention(abq.make_prompt_attention_params(q, k, v, out, _ends(nq), _ends(nk), scale=scale, max_q=max_q, status_word=status))
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    _check(out, q, k, v, nq, nk, scale)
    assert bool((guard[sum(nq):] == -9).all()) and bool((guard[:, heads] == -9).all())
    return out


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("half", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,nq,nk", [
    (1, 1, [1], None),
    (1, 1, [128], None),
    (2, 1, [127], None),
    (4, 4, [129, 1, 0, 256], None),
    (4, 1, [33, 64, 65, 300], None),
    (16, 1, [5, 16, 17, 100], None),
    (32, 1, [40], None),
    (6, 2, [513, 2], None),
    (10, 2, [1000], None),
    (7, 1, [31, 260], None),
    (4, 2, [10, 300, 1, 128], [500, 300, 129, 1000]),   # behind a prefix
    (2, 2, [200, 10, 64], [50, 0, 63]),                  # rows that see nothing
    (8, 2, [1] * 40 + [0] * 5 + [3] * 7, None),          # more sequences than a warp has lanes
    (2, 1, [1], [2500]),
])
def test_against_64_bits(abq, cuda, dim, half, heads, kv_heads, nq, nk):
    _run(abq, HALF[half], dim, heads, kv_heads, nq, nk or nq, seed=sum(nq) + heads)


def test_more_blocks_than_multiprocessors(abq, cuda):
    """Several blocks a CTA, of different lengths: barriers and buffers over many rounds."""
    _run(abq, torch.float16, 128, 32, 8, [900, 3, 700, 129, 0, 1, 512], [1000, 3, 700, 400, 7, 1, 512], seed=1)
    _run(abq, torch.bfloat16, 64, 48, 48, [300, 257, 1, 90, 511] * 2, [300, 257, 1, 90, 511] * 2, seed=2, max_q=511)


def test_the_same_bits_again_and_any_launch_size(abq, cuda):
    a = _run(abq, torch.float16, 128, 8, 2, [700, 50], [700, 50], seed=3).clone()
    b = _run(abq, torch.float16, 128, 8, 2, [700, 50], [700, 50], seed=3, max_q=700)
    c = _run(abq, torch.float16, 128, 8, 2, [700, 50], [700, 50], seed=3, max_q=1)
    assert torch.equal(a[:750], b[:750]) and torch.equal(a[:750], c[:750])


@pytest.mark.parametrize("half", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,heads,kv_heads", [(128, 2, 2), (64, 4, 1)])
def test_inf_and_nan_reach_only_the_rows_that_see_them(abq, cuda, half, dim, heads, kv_heads):
    def edit(q, k, v):
        v[3, 0, 1], v[130, 0, dim - 1], v[299, 0, 7] = float("nan"), float("inf"), float("-inf")  # sequence 0
        v[300 + 64] = float("inf")                                                                # sequence 1
        k[300 + 200:300 + 210] = 0.0
    _run(abq, HALF[half], dim, heads, kv_heads, [300, 260, 1], [300, 260, 1], seed=4, edit=edit)


def test_masked_keys_may_be_nan(abq, cuda):
    """A key of NaN spoils the rows that see it; the rows before it do not notice."""
    q, k, v = _inputs(5, torch.float16, 128, 2, 1, [290], [290])
    k[140] = float("nan")
    out = torch.empty((290, 2, 128), dtype=torch.float16, device="cuda")
    abq.prompt_attention(abq.make_prompt_attention_params(q[:290], k[:290], v[:290], out, _ends([290]), _ends([290]), scale=0.1))
    _check(out[:140], q[:140], k[:140], v[:140], [140], [140], 0.1)
    assert bool(out[140:].isnan().all())


def test_sharp_and_flat_softmax(abq, cuda):
    for gain in (0.0, 30.0):
        def edit(q, k, v):
            q[:400] *= gain
            k[7] *= 3.0
        _run(abq, torch.float16, 128, 4, 2, [400], [400], seed=6, edit=edit)
        _run(abq, torch.bfloat16, 64, 4, 2, [400], [400], seed=6, edit=edit)


def test_rising_maximum(abq, cuda):
    """Scores that grow from key to key: the running maximum is raised, and O scaled, in every tile."""
    def edit(q, k, v):
        q[:1000, :, 0], q[:1000, :, 1:] = 4.0, 0.0
        k[:1000, :, 0] = (torch.arange(1000, device=k.device).view(-1, 1) * 0.125).to(k.dtype)
    _run(abq, torch.float16, 64, 2, 1, [1000], [1000], seed=7, edit=edit)
    _run(abq, torch.bfloat16, 128, 2, 1, [1000], [1000], seed=7, edit=edit)


def test_in_place(abq, cuda):
    q, k, v = _inputs(8, torch.float16, 128, 8, 2, [400, 33], [400, 33])
    first = q.clone()
    abq.prompt_attention(abq.make_prompt_attention_params(q, k, v, q, _ends([400, 33]), _ends([400, 33]), scale=0.1))
    _check(q, first, k, v, [400, 33], [400, 33], 0.1)
    assert bool(q[433:].isnan().all())


def test_ends_beyond_the_rows_are_cut(abq, cuda):
    q, k, v = _inputs(9, torch.float16, 64, 2, 2, [100], [100], spare=0)
    out = torch.full((100, 2, 64), -9.0, dtype=torch.float16, device="cuda")
    abq.prompt_attention(abq.make_prompt_attention_params(q, k, v, out, _ends([60, 1000]), _ends([60, 1000]), scale=0.1))
    _check(out, q, k, v, [60, 40], [60, 40], 0.1)


def test_captured_and_on_two_streams(abq, cuda):
    sets = []
    for seed, lens in ((10, [500, 70]), (11, [333])):
        q, k, v = _inputs(seed, torch.bfloat16, 128, 8, 4, lens, lens)
        out = torch.zeros((q.shape[0], 8, 128), dtype=torch.bfloat16, device="cuda")
        ends = _ends(lens)
        sets.append((abq.make_prompt_attention_params(q, k, v, out, ends, ends, scale=0.1), q, k, v, out, lens))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for s, st in zip(sets, streams):
            abq.prompt_attention(s[0], st)
    torch.cuda.synchronize()
    for _, q, k, v, out, lens in sets:
        _check(out, q, k, v, lens, lens, 0.1)
        out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        abq.prompt_attention(sets[0][0], streams[0])
    graph.replay()
    torch.cuda.synchronize()
    _, q, k, v, out, lens = sets[0]
    _check(out, q, k, v, lens, lens, 0.1)
