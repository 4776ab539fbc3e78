"""abq_cache_attention over values of all sizes that bf16 has, on each of its kernels: one row, 16 rows and 128 rows a key head."""
import pytest
import torch

from test_gpu_cache_attention import Setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,n", [(4, 1), (4, 4), (4, 32)])
@pytest.mark.parametrize("power", [-120, -100, -75, -40, 40, 75, 100])
@pytest.mark.parametrize("bits", [4, 8])
def test_all_values_of_one_size(abq, cuda, bits, power, heads, n):
    s = Setup(abq, dim=64, bits=bits, half=torch.bfloat16, heads=heads, kv_heads=1, n=n, lens=[300], page=16, seed=power + 200)
    s.v = (s.v.float() * 2.0 ** power).to(torch.bfloat16)
    s.fill()
    s.check(s.call())


@pytest.mark.parametrize("heads,n", [(4, 1), (4, 4), (4, 32)])
@pytest.mark.parametrize("power", [-100, 60, 100])
def test_constant_rows(abq, cuda, power, heads, n):
    """Value rows whose scale is 0: their minimum alone counts."""
    s = Setup(abq, dim=128, bits=8, half=torch.bfloat16, heads=heads, kv_heads=1, n=n, lens=[300], page=16, seed=power + 300)
    s.v[:] = (s.v[..., :1].float() * 2.0 ** power).to(torch.bfloat16)
    s.fill()
    s.check(s.call())
