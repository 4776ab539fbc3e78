"""abq_cache_attention with ordinary scores against bounds that take each key's own error: a granule left out, or one with another's scores, would show (asserted)."""
import pytest
import torch

import attention_ref as R
from test_gpu_cache_attention import Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,n", [(4, 4, 1), (4, 4, 12), (8, 1, 16)])  # the kernels of 8, 16 and 128 rows
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lens,page", [([1500, 31], 16), ([700, 129, 1], 48)])
def test_each_key_with_its_own_error(abq, cuda, heads, kv_heads, n, dim, bits, lens, page):
    """The bound, for fp16: p_j is off by e_j of itself, so the result by at most sum_j p_j e_j |v_j - result|.  e_j = ln 2 d_j + 2^-21 with the score's error d_j (in
    powers of two): D / 16 steps of the running sum in fp32, 2^-23 each of at most sum|q| times the largest factor, which is 1024 + c or 64 + c in the kernels of few
    rows and |c'| in that of 128; two more roundings for scale and offset.  p times the value's scale is rounded to fp16 once with more than 8 rows (half a step
    of each product with c'), twice (to 2^-22) with up to 8.  Sums in fp32 2^-18 of the magnitudes together, and the result's own rounding."""
    s = Setup(abq, dim=dim, bits=bits, half=torch.float16, heads=heads, kv_heads=kv_heads, n=n, lens=lens, page=page, tree=n > 1, seed=dim + bits + n).fill()
    s.scale = 0.3 * dim ** -0.5  # (flat enough that every granule has a share)
    out = s.call()
    group, centre, most = heads // kv_heads, float(1 << (bits - 1)), float(1 << bits)
    wide = n * group > 79
    for b, length in enumerate(lens):
        (kc, ks, km), (vc, vs, vm) = R.decode(s.data, page, bits, dim, s.half, s.table[b], length)
        k, v = kc * ks + km, vc * vs + vm
        q = s.q[b * n:(b + 1) * n].double().reshape(n, kv_heads, group, dim).permute(1, 2, 0, 3)
        seen = torch.ones((n, length), dtype=torch.bool)
        for i in range(n):
            mask = 1 if s.tree is None else int(s.tree[b, i])
            for j in range(n):
                if length - n + j >= 0:
                    seen[i, length - n + j] = bool(mask >> j & 1)
        p = R.softmax64(torch.matmul(q, k.unsqueeze(1).transpose(2, 3)) * s.scale, seen)
        want = torch.matmul(p, v.unsqueeze(1))
        qsum = q.abs().sum(-1, keepdim=True)
        off = -centre if wide else (1024.0 if bits == 8 else 64.0)
        factor = centre if wide else off + most
        joined = (ks * factor + (km - off * ks).abs()).transpose(1, 2).unsqueeze(1)  # [key heads][1][1][tokens]
        d = 1.4427 * s.scale * qsum * joined * 2.0 ** -23 * (dim // 16 + 2)
        e = 0.6932 * d + 2.0 ** -21
        pe = p * e
        bound = torch.zeros_like(want)
        for h in range(kv_heads):
            for g in range(group):
                for i in range(n):
                    bound[h, g, i] = (pe[h, g, i].unsqueeze(-1) * (v[h] - want[h, g, i]).abs()).sum(0)
        codes, offsets = vs * (vc - centre).abs(), (vm + centre * vs).abs()
        bound = 1.01 * bound + (2.0 ** -22 if n * group <= 8 else 2.0 ** -11) * torch.matmul(p, codes.unsqueeze(1)) + 2.0 ** -18 * torch.matmul(p, (codes + offsets).unsqueeze(1))
        bound = bound + 2.0 ** -11 * want.abs() + 2.0 ** -24 + length * 2.0 ** -39 * (vs * centre + offsets).amax()
        got = out.cpu().double()[b * n:(b + 1) * n].view(n, kv_heads, group, dim).permute(1, 2, 0, 3)
        err = (got - want).abs()
        assert bool((err <= bound).all()), f"sequence {b}: {float((err / bound).max()):.2f} of the bound"
        if length < 600:
            continue
        for at in range(0, length - n - 16, 16):  # without these 16 keys
            part = p[..., at:at + 16]
            change = (torch.matmul(part, v[:, at:at + 16].unsqueeze(1)) - part.sum(-1, keepdim=True) * want) / (1 - part.sum(-1, keepdim=True))
            assert bool((change.abs() > 2 * bound).any(-1).all()), "the case says nothing"
