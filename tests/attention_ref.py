"""Plain restatements of the quantised cache and of attention, for the tests: the layout from its description in include/abq_b200.h,
the quantiser in float32 on the CPU (its operations are correctly rounded there too), attention in float64."""
from __future__ import annotations

import numpy as np
import torch


def halves(dtype):
    """(largest relative rounding error, smallest subnormal step) of a 16-bit type."""
    return (2.0 ** -8, 2.0 ** -133) if dtype == torch.bfloat16 else (2.0 ** -11, 2.0 ** -24)


def place(row_bytes: int, t: int, byte: int) -> int:
    at = t * row_bytes + byte
    line, piece, rest = at // 128, at // 16 % 8, at % 16
    turn = {128: 2 * (line % 4) ^ 4 * (line // 4 % 2), 64: 2 * (line % 4), 32: 4 * (line % 2)}[row_bytes]
    return line * 128 + (piece ^ turn) * 16 + rest


def places(row_bytes: int) -> torch.Tensor:
    return torch.tensor([[place(row_bytes, t, e) for e in range(row_bytes)] for t in range(16)])


def granule_bytes(dim: int, bits: int) -> int:
    return 32 * (dim * bits // 8) + 128


def quantise(x: torch.Tensor, bits: int):
    """16-bit rows [..., dim] (CPU) -> (codes uint8, scale, min) of the rule in the header."""
    half = x.dtype
    f = x.float()
    low, high = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    fine = (high - low) / torch.tensor(float((1 << bits) - 1))
    scale = fine.to(half)
    up = (scale.view(torch.int16) + 1).view(half)
    scale = torch.where(scale.float() < fine, up, scale)
    s = scale.float()
    codes = torch.where(s > 0, torch.round((f - low) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(f))
    bad = ~torch.isfinite(f).all(-1, keepdim=True) | ~torch.isfinite(high - low)
    codes = torch.where(bad, torch.zeros_like(codes), codes)
    nan = torch.full_like(scale, float("nan"))
    return codes.to(torch.uint8), torch.where(bad, nan, scale), torch.where(bad, nan, low.to(half))


def encode(data, page_size: int, bits: int, slots, k, v):
    """Write 16-bit rows k, v [tokens][heads][dim] into ``data`` uint8 [pages][heads][page / 16][granule] (all on the CPU)."""
    dim = k.shape[2]
    rb = dim * bits // 8
    where = places(rb)
    for part, x in ((0, k), (1, v)):
        codes, scale, low = quantise(x, bits)
        rows = codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)
        pair = torch.cat([scale, low], dim=-1).contiguous().view(torch.uint8)
        for i, slot in enumerate(slots.tolist()):
            if slot < 0 or slot >= data.shape[0] * page_size:
                continue
            page, at = divmod(slot, page_size)
            g, t = divmod(at, 16)
            data[page, :, g, 16 * rb * part + where[t]] = rows[i]
            data[page, :, g, 32 * rb + 64 * part + 4 * t:32 * rb + 64 * part + 4 * t + 4] = pair[i]


def decode(data, page_size: int, bits: int, dim: int, half, table_row, length: int):
    """float64 (codes, scale, min) of keys and of values of one sequence: [heads][length][...]."""
    rb = dim * bits // 8
    n = -(-length // page_size)
    g = data[table_row[:n].long()].permute(1, 0, 2, 3)  # [heads][pages][granules][bytes]
    g = g.reshape(g.shape[0], -1, g.shape[-1])
    where = places(rb).reshape(-1)
    out = []
    for part in range(2):
        rows = g[..., 16 * rb * part + where].reshape(g.shape[0], -1, rb)
        codes = rows if bits == 8 else torch.stack([rows & 15, rows >> 4], dim=-1).reshape(g.shape[0], -1, 2 * rb)
        pair = g[..., 32 * rb + 64 * part:32 * rb + 64 * part + 64].contiguous().view(half).reshape(g.shape[0], -1, 2).double()
        out.append((codes[:, :length].double(), pair[:, :length, :1], pair[:, :length, 1:]))
    return out


def softmax64(scores, seen):
    scores = torch.where(seen, scores, torch.full_like(scores, -np.inf))
    top = scores.amax(-1, keepdim=True) if scores.shape[-1] else torch.zeros(scores.shape[:-1] + (1,), dtype=torch.float64)
    e = torch.exp(scores - torch.where(top == -np.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def cache_attention(data, page_size, bits, half, table, lens, q, n, scale, tree=None):
    """(result, error bound) in float64 for 16-bit q [batch * n][q_heads][dim]; everything on the CPU.

    The bound: the result's own rounding (half a step); p vs rounded to fp16 (2^-11 of p vs |c'|, and what underflows below 2^-39 of the
    largest); the score's error d: the codes c are multiplied as o + c (o = 1024 for 8 bits, 64 for 4) in 8 products of 16 and joined with sum(q) (km - o ks), in fp32,
    2^-23 each, so at most 2^-20 of scale log2(e) sum|q| ((o + 2^bits) ks + |km - o ks|),
    plus, for bf16 queries, what the scaled fp16 row loses below its 2^-14 (2^-25 of twice the row's largest per feature), which moves p and the sum of p by
    at most 2 ln 2 d each; sums of p and of p v in fp32 with the exponential's 2^-22, 2^-18 of the sum of magnitudes together."""
    dim, heads = q.shape[2], q.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    centre = float(1 << (bits - 1))
    step, tiny = halves(half)
    for b, length in enumerate(lens):
        if length <= 0:
            continue
        (kc, ks, km), (vc, vs, vm) = decode(data, page_size, bits, dim, half, table[b], length)
        H = kc.shape[0]
        k, v = kc * ks + km, vc * vs + vm
        qq = q[b * n:(b + 1) * n].double().reshape(n, H, heads // H, dim).permute(1, 2, 0, 3)  # [H][group][n][dim]
        s = torch.matmul(qq, k.unsqueeze(1).transpose(2, 3)) * scale
        draft = torch.arange(length) - (length - n)
        seen = torch.zeros((n, length), dtype=torch.bool)
        for i in range(n):
            bits_ = (1 << (i + 1)) - 1 if tree is None else int(tree[b, i]) & ((1 << 64) - 1)
            seen[i] = torch.tensor([d < 0 or bool(bits_ >> d & 1) for d in draft.tolist()])
        clean = torch.where(seen.any(0).view(1, -1, 1), v, torch.zeros_like(v))
        p = softmax64(s, seen)
        got = torch.matmul(p, clean.unsqueeze(1))
        out[b * n:(b + 1) * n] = got.permute(2, 0, 1, 3).reshape(n, heads, dim)
        mags = torch.where(seen.any(0).view(1, -1, 1), vs * centre + (vm + centre * vs).abs(), torch.zeros_like(vs)).nan_to_num(0.0)
        codes = torch.where(seen.any(0).view(1, -1, 1), vs * (vc - centre).abs(), torch.zeros_like(vc)).nan_to_num(0.0)
        o = 1024.0 if bits == 8 else 64.0
        kmag = (ks * (o + 2.0 ** bits) + (km - o * ks).abs()).nan_to_num(0.0).amax((1, 2)).view(H, 1, 1, 1)
        qsum = qq.abs().sum(-1, keepdim=True) * 2.0 ** -20
        if half == torch.bfloat16:
            qsum = qsum + qq.abs().amax(-1, keepdim=True) * dim * 2.0 ** -24
        d = qsum * kmag * scale * 1.4427
        err = 2.0 ** -11 * torch.matmul(p, codes.unsqueeze(1)) + (2.78 * d + 2.0 ** -18) * torch.matmul(p, mags.unsqueeze(1))
        err = err + step * got.abs() + tiny + length * 2.0 ** -39 * mags.amax((1, 2)).view(H, 1, 1, 1)
        bound[b * n:(b + 1) * n] = err.permute(2, 0, 1, 3).reshape(n, heads, dim)
    return out, bound


def random_tree(gen, batch, n):
    """Ancestor masks int64 [batch][n] of random trees: every draft continues an earlier one or the sequence itself."""
    tree = torch.zeros((batch, n), dtype=torch.int64)
    for b in range(batch):
        for j in range(n):
            parent = int(torch.randint(-1, j, (1,), generator=gen)) if j else -1
            mask = (int(tree[b, parent]) & ((1 << 64) - 1) if parent >= 0 else 0) | 1 << j
            tree[b, j] = mask - (1 << 64) if mask >> 63 else mask
    return tree


def prompt_attention(q, k, v, nq, nk, scale):
    """(result, error bound) in float64 of causal attention over packed 16-bit rows (CPU); a value that a row does not see counts as 0.

    The bound: the result's rounding and that of p (half a step each; fp16 weights below 2^-20 of the largest lose at most 2^-31 of it per key); the score's
    error d, at most 2^-20 of scale log2(e) sum|q k| (8 products of 16 in fp32, 2^-23 each), which moves p and the sum of p by at most 2 ln 2 d each; the
    exponential is off by at most 2^-13.7 (bf16) or 2^-18.5 (fp16), in p and in their sum; sums in fp32 and O's scaling: 2^-18 of the sum of magnitudes."""
    half, heads, H = q.dtype, q.shape[1], k.shape[1]
    step, tiny = halves(half)
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    a = b = 0
    for n, m in zip(nq, nk):
        seen = torch.ones((n, m), dtype=torch.bool).tril(m - n)
        for h in range(heads if n and m else 0):
            qq, kk, vv = q[a:a + n, h].double(), k[b:b + m, h * H // heads].double(), v[b:b + m, h * H // heads].double()
            p = softmax64((qq @ kk.T).nan_to_num(0.0, 0.0, 0.0) * scale, seen)
            fine = torch.where(vv.isfinite(), vv, torch.zeros_like(vv))
            got = p @ fine
            d = 2.0 ** -20 * 1.4427 * scale * (qq.abs() @ kk.nan_to_num(0.0, 0.0, 0.0).abs().T).amax(-1, keepdim=True)
            ex = 2.0 * (2.0 ** -13.7 if half == torch.bfloat16 else 2.0 ** -18.5)
            err = (step + 2.78 * d + ex + 2.0 ** -18) * (p @ fine.abs()) + step * got.abs() + tiny + m * 2.0 ** -31 * fine.abs().amax()
            hit = seen.double() @ (~vv.isfinite()).double() > 0  # rows that see an Inf or NaN in this feature
            out[a:a + n, h] = torch.where(hit, torch.full_like(got, float("nan")), got)
            bound[a:a + n, h] = err
        a, b = a + n, b + m
    return out, bound
