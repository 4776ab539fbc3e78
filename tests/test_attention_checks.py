"""The attention entry points without a GPU: sizes agree with the header, and wrong calls are refused before anything is launched."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
INVALID, WORKSPACE = 1, 3


def test_struct_sizes_match_the_header(abq, tmp_path):
    names = {"abq_kv_cache": abq.KVCache, "abq_kv_write_params": abq.KVWriteParams, "abq_kv_read_params": abq.KVReadParams,
             "abq_cache_attention_params": abq.CacheAttentionParams, "abq_prompt_attention_params": abq.PromptAttentionParams}
    src = tmp_path / "sz.c"
    src.write_text('#include "abq_b200.h"\n#include <stdio.h>\nint main(void){' + "".join(f'printf("%zu\\n", sizeof({n}));' for n in names) + "return 0;}\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "sz")], check=True)
    sizes = [int(x) for x in subprocess.run([str(tmp_path / "sz")], check=True, capture_output=True, text=True).stdout.split()]
    assert sizes == [ctypes.sizeof(t) for t in names.values()]


def test_cache_bytes(abq):
    assert abq.kv_cache_bytes(3, 32, 5, 128, 8) == 3 * 5 * 2 * (16 * 2 * 128 + 128)
    assert abq.kv_cache_bytes(1, 16, 1, 64, 4) == 16 * 2 * 32 + 128
    for bad in ((0, 16, 1, 64, 8), (1, 24, 1, 64, 8), (1, 0, 1, 64, 8), (1, 2048, 1, 64, 8), (1, 16, 0, 64, 8), (1, 16, 1, 96, 8), (1, 16, 1, 64, 2), (1, 16, 1, 64, 16)):
        assert abq.kv_cache_bytes(*bad) == 0, bad


def _cache(abq, **kw):
    c = abq.KVCache(4096, 4, 16, 2, 128, 8, 0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _refused(fn, make, good, changes, status=INVALID):
    for change in changes:
        p = make()
        for k, v in {**good, **change}.items():
            setattr(p, k, v)
        assert fn(ctypes.byref(p), None) == status, change
    assert fn(None, None) == INVALID


CACHE_FAULTS = [dict(data=None), dict(data=4104), dict(num_pages=0), dict(page_size=8), dict(kv_heads=0), dict(head_dim=80), dict(bits=5), dict(half_type=2)]
ROW_FAULTS = [dict(k=None), dict(v=4098), dict(k_stride=260), dict(v_head_stride=4)]


def test_write_refuses(abq):
    good = dict(cache=_cache(abq), k=4096, v=4096, k_stride=256, k_head_stride=128, v_stride=256, v_head_stride=128, slots=4096, tokens=3)
    _refused(abq.lib().abq_kv_cache_write, abq.KVWriteParams, good,
             ROW_FAULTS + [dict(slots=None), dict(slots=4100), dict(tokens=-1), dict(tokens=2**31 - 1)] + [dict(cache=_cache(abq, **c)) for c in CACHE_FAULTS])
    p = abq.KVWriteParams()
    for k, v in {**good, "tokens": 0, "k": None, "v": None, "slots": None}.items():
        setattr(p, k, v)
    assert abq.lib().abq_kv_cache_write(ctypes.byref(p), None) == 0  # nothing to write


def test_read_refuses(abq):
    good = dict(cache=_cache(abq), k=4096, v=4096, k_stride=256, k_head_stride=128, v_stride=256, v_head_stride=128, rows=3, batch=1, block_table=4096, table_stride=4,
                cu_seqlens=4096)
    _refused(abq.lib().abq_kv_cache_read, abq.KVReadParams, good,
             ROW_FAULTS + [dict(block_table=None), dict(block_table=4098), dict(cu_seqlens=None), dict(table_stride=0), dict(rows=-1), dict(rows=2**31 - 1), dict(batch=-1)] +
             [dict(cache=_cache(abq, **c)) for c in CACHE_FAULTS])


def test_cache_attention_refuses(abq):
    c = _cache(abq)
    need = abq.cache_attention_workspace_bytes(c, 2, 1, 4)
    assert need > 0
    good = dict(cache=c, q=4096, out=8192, q_stride=512, q_head_stride=128, out_stride=512, out_head_stride=128, batch=2, rows_per_seq=1, q_heads=4, block_table=4096,
                table_stride=4, seq_lens=4096, scale=0.1, workspace=4096, workspace_bytes=need)
    fn = abq.lib().abq_cache_attention
    _refused(fn, abq.CacheAttentionParams, good,
             [dict(q=None), dict(q=4104), dict(out=None), dict(out=8194), dict(q_stride=4), dict(out_head_stride=130), dict(batch=-1), dict(rows_per_seq=0), dict(rows_per_seq=65),
              dict(q_heads=3), dict(q_heads=0), dict(block_table=None), dict(block_table=4097), dict(table_stride=0), dict(seq_lens=None), dict(seq_lens=4098), dict(tree=4100),
              dict(scale=float("nan")), dict(scale=float("inf")), dict(status_word=4097), dict(out=4096, out_stride=256),
              dict(cache=_cache(abq, num_pages=1 << 30))] + [dict(cache=_cache(abq, **f)) for f in CACHE_FAULTS])
    _refused(fn, abq.CacheAttentionParams, good, [dict(workspace=None), dict(workspace=4104), dict(workspace_bytes=need - 1)], WORKSPACE)
    for rows, heads in ((0, 4), (65, 4), (1, 3), (1, 0)):
        assert abq.cache_attention_workspace_bytes(c, 2, rows, heads) == 0
    assert abq.cache_attention_workspace_bytes(c, 2, 8, 4) > need and abq.cache_attention_workspace_bytes(c, 2, 64, 4) > need


def test_prompt_attention_refuses(abq):
    good = dict(q=4096, k=4096, v=4096, out=8192, q_stride=512, q_head_stride=128, k_stride=256, k_head_stride=128, v_stride=256, v_head_stride=128, out_stride=512,
                out_head_stride=128, total_q=10, total_k=10, q_heads=4, kv_heads=2, head_dim=128, half_type=0, batch=2, cu_q=4096, cu_k=4096, scale=0.1)
    fn = abq.lib().abq_prompt_attention
    _refused(fn, abq.PromptAttentionParams, good,
             [dict(q=None), dict(q=4104), dict(k=None), dict(v=4098), dict(out=None), dict(out=8200), dict(q_stride=4), dict(k_head_stride=129), dict(v_stride=-256), dict(out_stride=0),
              dict(k_stride=0), dict(q_heads=3), dict(q_heads=0), dict(kv_heads=0), dict(head_dim=96), dict(half_type=2), dict(batch=-1), dict(total_q=-1), dict(total_k=-1),
              dict(cu_q=None), dict(cu_k=4098), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(max_q=-1), dict(status_word=4097),
              dict(out=4096, out_stride=1024)])
    for empty in (dict(total_q=0), dict(batch=0)):
        p = abq.PromptAttentionParams()
        for k, v in {**good, **empty}.items():
            setattr(p, k, v)
        assert fn(ctypes.byref(p), None) == 0  # nothing to do


def test_python_layer_refuses(abq):
    """Shapes, types and devices are checked where the parameter block is made: a CPU tensor never becomes a device pointer."""
    c = _cache(abq)
    x = torch.zeros((3, 2, 128), dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        abq.make_kv_write_params(c, x, x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="expected"):
        abq.make_kv_write_params(c, x[:, :1], x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="expected"):
        abq.make_kv_read_params(c, x[..., :64], x, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="same rows"):
        abq.make_cache_attention_params(c, x, x, torch.zeros((2, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int32), scale=1.0, workspace=x)


def test_tensors_of_one_call_are_on_one_device(abq):
    from types import SimpleNamespace as NS
    on = lambda i: NS(device=NS(index=i))  # noqa: E731
    assert abq.binding._one_device(q=on(1), k=on(1), tree=None, status_word=4096) == 1
    with pytest.raises(ValueError, match="different devices.*q on cuda:0.*table on cuda:1"):
        abq.binding._one_device(q=on(0), table=on(1))


def test_calls_go_to_the_device_of_their_tensors(abq, monkeypatch):
    """The call is made with the tensors' device current, on that device's stream, and the old one is current behind it."""
    import torch
    from types import SimpleNamespace as NS
    now, seen = [0], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.old, now[0] = now[0], self.index

        def __exit__(self, *e):
            now[0] = self.old

    monkeypatch.setattr(abq.binding, "_current_device", lambda: now[0])
    monkeypatch.setattr(abq.binding, "_current_raw", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(abq.binding, "_lib", NS(abq_kv_cache_write=lambda p, stream: seen.append((now[0], stream)) or 0))
    for device in (0, 1):
        p = abq.binding.KVWriteParams()
        p._device = device
        abq.kv_cache_write(p)
    assert seen == [(0, 100), (1, 101)] and now == [0]
