"""The attention operators of a decoder block as cases that can be timed and compared: their plain forms and the library's calls.

A case is a dict of plain values; its "kind" says which operator a pass goes through:

  cache    kv_cache_write of the tokens a step brings, then kv_cache_read of the whole sequences: fp16 / bf16 keys and values quantised to
           8 or 4 bits into a paged cache and read back packed (a chunk of a long prompt, a prefix used again)
  cached   cache_attention: the query rows of a token step (one token, or a tree of drafted tokens) over the quantised cache
  prompt   prompt_attention: causal attention over packed prompts of different lengths, grouped heads

Queries, keys and values are slices of one fused QKV buffer, as the QKV projection of a block leaves them.  Head counts are those of
LLaMA-7B (32) and LLaMA-2-13B (40) and grouped ones; keys have the few large channels that such models show.

The cache (one for a layer): uint8 [pages][kv_heads][page_size / 16][granule].  A granule is 16 tokens of one head: 16 rows of key codes,
16 rows of value codes, 16 pairs (scale, min) of the keys, 16 of the values, in the cache's 16-bit type.  A row is head_dim codes in order
(4 bits: the even one in the low nibble); its 16-byte pieces are exchanged inside lines of 128 bytes as _places() says.
"""
from __future__ import annotations

import importlib
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False


def listed():
    return [
        # one token each for three short sequences: the smallest step there is, where the launches are what counts
        dict(name="cache_step_b3_int4", kind="cache", batch=3, shortest=20, longest=75, new=1, kv_heads=8, dim=64, bits=4, bf16=True, page=16, spread=3),
        # a 256-token chunk of four prompts, read back with their prefixes for the attention of the chunk
        dict(name="cache_chunk_b4_int8", kind="cache", batch=4, shortest=300, longest=1111, new=256, kv_heads=8, dim=128, bits=8, bf16=False, page=16, spread=4),
        # a long prompt of a 7B model into a 4-bit cache and out of it
        dict(name="cache_prompt_7b_int4", kind="cache", batch=1, shortest=16001, longest=16001, new=16001, kv_heads=32, dim=128, bits=4, bf16=False, page=64, spread=5),
        # one sequence of a 7B model, token by token: latency
        dict(name="decode_7b_b1", kind="cached", batch=1, idle=0, rows=1, shortest=1024, longest=1024, heads=32, kv_heads=32, dim=128, bits=8, bf16=False, page=16,
             tree=False, spread=6),
        # a served batch of sequences of all lengths in a graph of fixed size (three places idle), grouped heads, 4 bits
        dict(name="decode_b32_gqa_int4", kind="cached", batch=32, idle=3, rows=1, shortest=90, longest=4096, heads=32, kv_heads=8, dim=128, bits=4, bf16=True, page=16,
             tree=False, spread=7),
        # two very long documents, eight key heads
        dict(name="decode_128k_b2", kind="cached", batch=2, idle=0, rows=1, shortest=100003, longest=131072, heads=32, kv_heads=8, dim=128, bits=8, bf16=False, page=64,
             tree=False, spread=8),
        # a tree of 26 drafted tokens for four sequences of a 13B model
        dict(name="tree_13b_b4_n26", kind="cached", batch=4, idle=0, rows=26, shortest=700, longest=2049, heads=40, kv_heads=40, dim=128, bits=8, bf16=False, page=32,
             tree=True, spread=9),
        # the largest trees, heads of 64, 4 bits
        dict(name="tree_b16_n64_d64", kind="cached", batch=16, idle=0, rows=64, shortest=128, longest=1531, heads=16, kv_heads=4, dim=64, bits=4, bf16=True, page=128,
             tree=True, spread=10),
        # a handful of short prompts packed behind one another, one of them of a single token
        dict(name="prompt_short_packed", kind="prompt", batch=7, shortest=1, longest=200, prefix=0, heads=32, kv_heads=8, dim=128, bf16=False, spread=11),
        # one 2048-token prompt of a 7B model
        dict(name="prompt_7b_2048", kind="prompt", batch=1, shortest=2048, longest=2048, prefix=0, heads=32, kv_heads=32, dim=128, bf16=True, spread=12),
        # sixteen prompts of up to 1024 tokens, heads of 64, behind a prefix that the cache held
        dict(name="prompt_prefix_b16_d64", kind="prompt", batch=16, shortest=200, longest=1023, prefix=517, heads=32, kv_heads=4, dim=64, bf16=False, spread=13),
        # one long prompt with grouped heads
        dict(name="prompt_gqa_8k", kind="prompt", batch=1, shortest=8192, longest=8192, prefix=0, heads=32, kv_heads=8, dim=128, bf16=True, spread=14),
    ]


def _spread(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["cache", "cached", "cached", "prompt", "prompt"])
    dim, bf16 = rng.choice([64, 128, 128]), rng.random() < 0.5
    kv_heads, group = rng.choice([(32, 1), (40, 1), (8, 4), (8, 5), (4, 8), (16, 2), (2, 7), (1, 3), (10, 6)])
    c = dict(kind=kind, kv_heads=kv_heads, dim=dim, bf16=bf16, spread=rng.randrange(1 << 20))
    if kind == "cache":
        batch = _spread(rng, 1, 32)
        longest = _spread(rng, 1, min(16000, 16001 * 32 // (kv_heads * batch)))
        return dict(c, batch=batch, shortest=_spread(rng, 1, longest), longest=longest, new=_spread(rng, 1, longest), bits=rng.choice([4, 8]),
                    page=rng.choice([16, 32, 64, 128]))
    if kind == "cached":
        batch, tree = _spread(rng, 1, 64), rng.random() < 0.5
        rows = _spread(rng, 2, 64) if tree else rng.choice([1, 1, 1, 2, 5])
        # neither more bytes than the longest documents nor more products than the largest trees times four
        most = min(131072, 2 * 131072 * 8 // (kv_heads * batch), (1 << 27) // (kv_heads * group * batch * rows))
        longest = _spread(rng, 1, max(1, most))
        return dict(c, batch=batch, idle=rng.choice([0, 0, 1, 4]), rows=rows, shortest=_spread(rng, 1, longest), longest=longest, heads=kv_heads * group,
                    bits=rng.choice([4, 8]), page=rng.choice([16, 32, 64, 128]), tree=tree)
    batch = _spread(rng, 1, 32)
    # scores of all heads and padded sequences: at most those of the longest prompt
    longest = _spread(rng, 1, int(8192 * math.sqrt(32 / (kv_heads * group * batch)) / 1.5))
    return dict(c, batch=batch, shortest=_spread(rng, 1, longest), longest=longest, prefix=rng.choice([0, 0, longest // 3]), heads=kv_heads * group)


# ------------------------------------------------------------------------------------------------------------ inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(c):
    """The longest first, the others between the shortest and it, even over the logarithm."""
    r = random.Random(c["spread"])
    lens = [c["longest"]] + [_spread(r, c["shortest"], c["longest"]) for _ in range(c["batch"] - 1)]
    return lens + [0] * c.get("idle", 0)


def _half(c):
    return torch.bfloat16 if c["bf16"] else torch.float16


def _tensor(values, dtype):
    return torch.tensor(values, dtype=dtype).cuda()


def _ends(lens):
    return _tensor([sum(lens[:i]) for i in range(len(lens) + 1)], torch.int32)


def _keys(gen, shape):
    """Normal values with a few channels six times as large, a little off centre."""
    x = torch.randn(shape, device="cuda", generator=gen)
    gain = 1.0 + 5.0 * (torch.rand(shape[-2:], device="cuda", generator=gen) < 0.04)
    return x * gain + 0.3 * torch.randn(shape[-2:], device="cuda", generator=gen)


def _qkv(c, gen, tokens, heads):
    """Queries (where `heads` is not 0), keys and values as slices of one fused buffer."""
    H, d = c["kv_heads"], c["dim"]
    buf = torch.empty((tokens, heads + 2 * H, d), dtype=_half(c), device="cuda")
    buf[:, :heads] = torch.randn((tokens, heads, d), device="cuda", generator=gen).to(buf.dtype)
    buf[:, heads:heads + H] = _keys(gen, (tokens, H, d)).to(buf.dtype)
    buf[:, heads + H:] = torch.randn((tokens, H, d), device="cuda", generator=gen).to(buf.dtype)
    return buf[:, :heads], buf[:, heads:heads + H], buf[:, heads + H:]


def _row_bytes(c):
    return c["dim"] * c["bits"] // 8


def _places(row_bytes):
    """Where byte e of token t's row lies inside the 16 rows of a granule: int64 [16][row_bytes]."""
    t, e = torch.arange(16).view(16, 1), torch.arange(row_bytes).view(1, row_bytes)
    at = t * row_bytes + e
    line, piece = at // 128, at // 16 % 8
    turn = {128: (line % 4) * 2 ^ (line // 4 % 2) * 4, 64: (line % 4) * 2, 32: (line % 2) * 4}[row_bytes]
    return (line * 128 + (piece ^ turn) * 16 + at % 16).cuda()


def _granule_bytes(c):
    return 32 * _row_bytes(c) + 128


def _codes_of(x, bits, half):
    """float32 rows -> (codes, scale, min): min/max calibration, the scale rounded up to the 16-bit type."""
    top = torch.full((), float((1 << bits) - 1), device="cuda")
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    fine = (high - low) / top
    scale = fine.to(half)
    scale = torch.where(scale.float() < fine, (scale.view(torch.int16) + 1).view(half), scale)
    s = scale.float()
    codes = torch.where(s > 0, torch.round((x - low) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(x))
    return codes.clamp_(0, (1 << bits) - 1).to(torch.uint8), scale, low.to(half)


def _rows_of(codes, bits):
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def _filled_cache(c, gen, pages):
    """A cache whose every place holds a token of earlier steps (those behind a sequence's end are left over from others)."""
    H, d, P, half, rb = c["kv_heads"], c["dim"], c["page"], _half(c), _row_bytes(c)
    data = torch.empty((pages, H, P // 16, _granule_bytes(c)), dtype=torch.uint8, device="cuda")
    where = _places(rb).reshape(-1)
    for part in range(2):
        x = _keys(gen, (pages * P, H, d)) if part == 0 else torch.randn((pages * P, H, d), device="cuda", generator=gen)
        codes, scale, low = _codes_of(x.to(half).float(), c["bits"], half)
        rows = _rows_of(codes, c["bits"]).view(pages, P // 16, 16, H, rb).permute(0, 3, 1, 2, 4)
        data[..., part * 16 * rb + where] = rows.reshape(pages, H, P // 16, 16 * rb)
        pair = torch.cat([scale, low], dim=-1).view(pages, P // 16, 16, H, 2).permute(0, 3, 1, 2, 4).contiguous()
        data[..., 32 * rb + 64 * part:32 * rb + 64 * part + 64] = pair.view(torch.uint8).view(pages, H, P // 16, 64)
    return data


def _pages(c, gen, lens):
    """Pages of every sequence in no order: int32 [batch][most pages]; entries that no token needs are 0."""
    P = c["page"]
    need = [-(-n // P) for n in lens]
    total, most = sum(need) + 2, max(1, max(need))
    order = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros((len(lens), most), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    c, gen = dict(case), _gen(seed)
    if c["kind"] == "prompt":
        lens = _lengths(c)
        klens = [n + c["prefix"] for n in lens]
        if c["prefix"]:
            q, _, _ = _qkv(c, gen, sum(lens), c["heads"])
            _, k, v = _qkv(c, gen, sum(klens), 0)
        else:
            q, k, v = _qkv(c, gen, sum(lens), c["heads"])
        out = torch.empty((sum(lens), c["heads"], c["dim"]), dtype=_half(c), device="cuda")
        return dict(c=c, q=q, k=k, v=v, out=out, cu_q=_ends(lens), cu_k=_ends(klens), longest=max(lens), longest_k=max(klens), scale=c["dim"] ** -0.5)
    lens = _lengths(c)
    table, pages = _pages(c, gen, lens)
    state = dict(c=c, table=table, data=_filled_cache(c, gen, pages), lens=_tensor(lens, torch.int32), longest=max(lens))
    if c["kind"] == "cache":
        new = [min(c["new"], n) for n in lens]
        _, k, v = _qkv(c, gen, sum(new) + 3, c["kv_heads"])  # three places of the step are padding
        seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(new)).cuda()
        pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)]).cuda()
        slots = table[seq, pos // c["page"]].long() * c["page"] + pos % c["page"]
        slots = torch.cat([slots, torch.full((3,), -1, dtype=torch.int64, device="cuda")])
        ks, vs = (torch.empty((sum(lens), c["kv_heads"], c["dim"]), dtype=_half(c), device="cuda") for _ in range(2))
        return dict(state, k=k, v=v, slots=slots, cu=_ends(lens), k_out=ks, v_out=vs)
    rows, B = c["rows"], len(lens)
    q, _, _ = _qkv(c, gen, B * rows, c["heads"])
    tree = None
    if c["tree"]:
        parent = torch.rand((B, rows), device="cuda", generator=gen)
        tree = torch.zeros((B, rows), dtype=torch.int64, device="cuda")
        for j in range(rows):  # every drafted token continues an earlier one, or the sequence itself
            at = (parent[:, j] * (j + 1)).long() - 1
            tree[:, j] = torch.where(at >= 0, tree.gather(1, at.clamp(min=0).view(B, 1)).view(B), 0) | torch.ones((), dtype=torch.int64, device="cuda") << j
    out = torch.empty((B * rows, c["heads"], c["dim"]), dtype=_half(c), device="cuda")
    return dict(state, q=q, tree=tree, out=out, scale=c["dim"] ** -0.5)


# ------------------------------------------------------------------------------------------------------------ plain forms

def _plain_sequences(s):
    """Keys and values of the cached sequences in float32: 2 x [batch][kv_heads][tokens][dim], padded to a page."""
    c = s["c"]
    rb, half, where = _row_bytes(c), _half(c), _places(_row_bytes(c)).reshape(-1)
    data = s["data"][s["table"].long()].permute(0, 2, 1, 3, 4)  # [batch][heads][pages][granules][bytes]
    B, H, n, g, _ = data.shape

    def part(k):
        rows = data[..., 16 * rb * k + where].reshape(B, H, n * g * 16, rb)
        if c["bits"] == 4:
            rows = torch.stack([rows & 15, rows >> 4], dim=-1).reshape(B, H, n * g * 16, 2 * rb)
        pair = data[..., 32 * rb + 64 * k:32 * rb + 64 * k + 64].contiguous().view(half).view(B, H, n * g * 16, 2).float()
        return rows.float() * pair[..., :1] + pair[..., 1:]
    return part(0), part(1)


def _plain_cache(s):
    c = s["c"]
    rb, half, P = _row_bytes(c), _half(c), c["page"]
    kept = (s["slots"] >= 0).nonzero().view(-1)
    slot = s["slots"][kept]
    base = ((slot // P * c["kv_heads"]).view(-1, 1) + torch.arange(c["kv_heads"], device="cuda")) * (P // 16) + (slot % P // 16).view(-1, 1)
    base, t = base * _granule_bytes(c), slot % 16
    flat = s["data"].view(-1)

    def put(x, part):
        codes, scale, low = _codes_of(x[kept].float(), c["bits"], half)
        flat[base.unsqueeze(-1) + 16 * rb * part + _places(rb)[t].unsqueeze(1)] = _rows_of(codes, c["bits"])
        pair = torch.cat([scale, low], dim=-1).view(torch.uint8)
        flat[base.unsqueeze(-1) + (32 * rb + 64 * part + 4 * t).view(-1, 1, 1) + torch.arange(4, device="cuda")] = pair
    put(s["k"], 0)
    put(s["v"], 1)
    k, v = _plain_sequences(s)
    held = torch.arange(k.shape[2], device="cuda") < s["lens"].view(-1, 1)
    return k.transpose(1, 2)[held].to(half), v.transpose(1, 2)[held].to(half)


def _plain_softmax(scores, seen):
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_cached(s):
    c = s["c"]
    B, n, H, d = s["table"].shape[0], c["rows"], c["kv_heads"], c["dim"]
    k, v = _plain_sequences(s)
    q = s["q"].float().view(B, n, H, c["heads"] // H, d).permute(0, 2, 3, 1, 4).reshape(B, H, -1, d)
    scores = (torch.matmul(q, k.transpose(2, 3)) * s["scale"]).view(B, H, -1, n, k.shape[2])
    draft = torch.arange(k.shape[2], device="cuda") - (s["lens"].view(B, 1) - n)  # [batch][tokens]: which of the drafted tokens a place holds
    if s["tree"] is None:
        branch = draft.unsqueeze(1) <= torch.arange(n, device="cuda").view(n, 1)
    else:
        branch = (s["tree"].unsqueeze(2) >> draft.clamp(0, 63).unsqueeze(1)) & 1 == 1
    seen = ((draft < 0).unsqueeze(1) | branch) & (draft < n).unsqueeze(1)
    p = _plain_softmax(scores, seen.view(B, 1, 1, n, -1)).view(B, H, -1, k.shape[2])
    return torch.matmul(p, v).view(B, H, -1, n, d).permute(0, 3, 1, 2, 4).reshape(B * n, c["heads"], d).to(s["out"].dtype)


def _plain_prompt(s):
    c = s["c"]
    B, H, d, L, M = c["batch"], c["kv_heads"], c["dim"], s["longest"], s["longest_k"]

    def padded(x, ends, most):  # packed rows -> [batch][kv_heads][group][most][dim]
        at = (ends[:-1].view(-1, 1) + torch.arange(most, device="cuda")).clamp(max=x.shape[0] - 1).long()
        return x[at].float().view(B, most, H, -1, d).permute(0, 2, 3, 1, 4)
    nq, nk = (e[1:] - e[:-1] for e in (s["cu_q"], s["cu_k"]))
    q, k, v = padded(s["q"], s["cu_q"], L), padded(s["k"], s["cu_k"], M), padded(s["v"], s["cu_k"], M)
    row, key = torch.arange(L, device="cuda").view(1, L, 1), torch.arange(M, device="cuda").view(1, 1, M)
    seen = (key <= row + (nk - nq).view(B, 1, 1)) & (key < nk.view(B, 1, 1))
    p = _plain_softmax(torch.matmul(q, k.transpose(3, 4)) * s["scale"], seen.view(B, 1, 1, L, M))
    out = torch.matmul(p, v).permute(0, 3, 1, 2, 4).reshape(B, L, c["heads"], d)
    return out[torch.arange(L, device="cuda") < nq.view(B, 1)].to(s["out"].dtype)


# ------------------------------------------------------------------------------------------------------------ the library's calls

def _package():
    """The package directory's name has a hyphen: it is registered under an importable one."""
    if "abq_llm_b200" not in sys.modules:
        pkg = Path.cwd() / "abq-llm_b200"
        if not pkg.is_dir():
            pkg = Path(__file__).resolve().parent.parent / "abq-llm_b200"
        spec = importlib.util.spec_from_file_location("abq_llm_b200", pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["abq_llm_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["abq_llm_b200"]


def _own(s):
    """The parameter blocks (and the workspace) are made at a state's first pass and kept, as a program keeps them for its steps."""
    abq, c = _package(), s["c"]
    if "params" not in s:
        if c["kind"] == "prompt":
            s["params"] = abq.make_prompt_attention_params(s["q"], s["k"], s["v"], s["out"], s["cu_q"], s["cu_k"], scale=s["scale"], max_q=s["longest"])
        else:
            cache = abq.make_kv_cache(s["data"], page_size=c["page"], kv_heads=c["kv_heads"], head_dim=c["dim"], bits=c["bits"], dtype=_half(c))
            if c["kind"] == "cache":
                s["params"] = (abq.make_kv_write_params(cache, s["k"], s["v"], s["slots"]),
                               abq.make_kv_read_params(cache, s["k_out"], s["v_out"], s["table"], s["cu"]))
            else:
                work = torch.empty(abq.cache_attention_workspace_bytes(cache, s["table"].shape[0], c["rows"], c["heads"]), dtype=torch.uint8, device="cuda")
                s["params"] = abq.make_cache_attention_params(cache, s["q"], s["out"], s["table"], s["lens"], tree=s["tree"], scale=s["scale"], workspace=work)
    if c["kind"] == "prompt":
        abq.prompt_attention(s["params"])
        return s["out"]
    if c["kind"] == "cached":
        abq.cache_attention(s["params"])
        return s["out"]
    write, read = s["params"]
    abq.kv_cache_write(write)
    abq.kv_cache_read(read)
    return s["k_out"], s["v_out"]


def run(state):
    if own:
        return _own(state)
    return {"cache": _plain_cache, "cached": _plain_cached, "prompt": _plain_prompt}[state["c"]["kind"]](state)


# ------------------------------------------------------------------------------------------------------------ what a pass cannot do without

def _pairs(nq, nk):
    """Keys seen by all the rows of one sequence."""
    return sum(max(0, min(nk, i + 1 + nk - nq)) for i in range(nq))


def work(case):
    c, d, H = case, case["dim"], case["kv_heads"]
    lens = _lengths(c)
    if c["kind"] == "prompt":
        klens = [n + c["prefix"] for n in lens]
        return {"bytes": 2 * d * (2 * sum(lens) * c["heads"] + 2 * sum(klens) * H), "flops": 4 * d * c["heads"] * sum(_pairs(n, m) for n, m in zip(lens, klens))}
    held = 2 * (d * c["bits"] / 8 + 4) * H  # bytes of a token in the cache
    if c["kind"] == "cache":
        new = sum(min(c["new"], n) for n in lens)
        return {"bytes": new * (4 * d * H + held) + sum(lens) * (held + 4 * d * H), "flops": 4 * d * H * (new + sum(lens))}
    rows = c["rows"] * c["heads"]
    return {"bytes": sum(lens) * held + 4 * d * rows * sum(n > 0 for n in lens) + 2 * d * rows * c["idle"], "flops": 4 * d * rows * sum(lens)}


# ------------------------------------------------------------------------------------------------------------ 64 bits

def _exact_tokens(s, granules, part):
    """The values of whole granules [n][bytes] of one head, from the bytes' own addresses: float64 [n * 16][dim]."""
    c = s["c"]
    rb, half = _row_bytes(c), _half(c)
    place = torch.arange(16 * rb, device="cuda")
    line, piece = place // 128, place // 16 % 8
    turn = line % 4 * 2 ^ (line // 4 % 2 * 4) if rb == 128 else line % 4 * 2 if rb == 64 else line % 2 * 4
    order = torch.argsort(line * 128 + (piece ^ turn) * 16 + place % 16)  # the row-major place of every stored byte
    rows = torch.empty((granules.shape[0], 16 * rb), dtype=torch.uint8, device="cuda")
    rows[:, order] = granules[:, 16 * rb * part:16 * rb * (part + 1)]
    rows = rows.view(-1, rb)
    codes = torch.empty((rows.shape[0], c["dim"]), dtype=torch.float64, device="cuda")
    if c["bits"] == 8:
        codes[:] = rows
    else:
        codes[:, 0::2] = rows % 16
        codes[:, 1::2] = rows // 16
    pair = granules[:, 32 * rb + 64 * part:32 * rb + 64 * part + 64].contiguous().view(half).view(-1, 2).double()
    return codes * pair[:, :1] + pair[:, 1:]


def _exact_head(s, b, h, n):
    """Keys and values of the first n tokens of sequence b, head h."""
    pages = s["table"][b, :-(-n // s["c"]["page"])].long()
    granules = s["data"][pages, h].reshape(-1, _granule_bytes(s["c"]))
    return _exact_tokens(s, granules, 0)[:n], _exact_tokens(s, granules, 1)[:n]


def _exact_read(x, bits, half):
    """float64 rows as the cache holds them: the scale is the smallest of its 16-bit type that reaches from the least to the largest value."""
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    fine = (high - low) / ((1 << bits) - 1)
    near = fine.to(half)
    scale = torch.where(near.double() < fine, (near.view(torch.int16) + 1).view(half), near).double()
    codes = torch.where(scale > 0, torch.round((x - low) / scale.clamp(min=1e-300)), 0.0).clamp(0, (1 << bits) - 1)
    return low + codes * scale


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    lens, d, H = _lengths(c), c["dim"], c["kv_heads"]
    if c["kind"] == "cache":
        at = first = 0
        ks, vs = (torch.empty((sum(lens), H, d), dtype=torch.float64, device="cuda") for _ in range(2))
        for b, n in enumerate(lens):
            m = min(c["new"], n)
            for h in range(H):
                for part, to, new in ((0, ks, s["k"]), (1, vs, s["v"])):
                    to[at:at + n, h] = _exact_head(s, b, h, n)[part]
                    to[at + n - m:at + n, h] = _exact_read(new[first:first + m, h].double(), c["bits"], _half(c))
            at, first = at + n, first + m
        return ks, vs
    group = c["heads"] // H
    out = torch.zeros(tuple(s["out"].shape), dtype=torch.float64, device="cuda")
    first = start = 0
    for b, n in enumerate(lens):
        if c["kind"] == "prompt":
            nq, nk, at = n, n + c["prefix"], first
            seen = torch.ones((nq, nk), dtype=torch.bool, device="cuda").tril(nk - nq)
        else:
            nq, nk, at = c["rows"], n, b * c["rows"]
            seen = torch.ones((nq, nk), dtype=torch.bool, device="cuda")
            for i in range(nq):
                bits = (1 << (i + 1)) - 1 if s["tree"] is None else int(s["tree"][b, i]) & ((1 << 64) - 1)
                told = [bool(bits >> j & 1) for j in range(nq)][max(0, nq - nk):]
                if nk:
                    seen[i, nk - len(told):] = torch.tensor(told, dtype=torch.bool, device="cuda")
        for h in range(H):
            if nk == 0:
                continue
            k, v = (s["k"][start:start + nk, h].double(), s["v"][start:start + nk, h].double()) if c["kind"] == "prompt" else _exact_head(s, b, h, nk)
            q = s["q"][at:at + nq, h * group:(h + 1) * group].double()
            w = (q.transpose(0, 1) @ k.T * s["scale"]).masked_fill_(~seen, -math.inf)
            w = torch.softmax(w, dim=-1).nan_to_num_(0.0)
            out[at:at + nq, h * group:(h + 1) * group] = (w @ v).transpose(0, 1)
        if c["kind"] == "prompt":
            first, start = first + nq, start + nk
    return out
