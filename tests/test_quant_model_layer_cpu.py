"""A layer of make_quant_cache, without a GPU: a fake QuantKV stands in for the kernels."""
import pytest
import torch

from test_gpu_quant_model import tiny
from utmist_bigger_bird_b200 import install, make_quant_cache


class FakeKV:
    """Keeps rows as tensors; reads give them back in the dtype that is asked for."""
    capacity, kv_heads, head_dim = 64, 2, 64

    def __init__(self):
        self.rows = torch.zeros(2, 64, 64), torch.zeros(2, 64, 64)

    def write(self, k, v, at, *, values=False):
        for x, rows in zip((k, v), self.rows):
            rows[:, at:at + k.shape[1]] = x.float()
        return (k, v) if values else None

    def read(self, positions=None, *, start=0, stop=None, dtype=torch.bfloat16):
        return tuple(x[:, start:stop].to(dtype) for x in self.rows)


def layer(dtype):
    model = tiny("cpu", dtype)
    install(model, "vs")
    cache = make_quant_cache(model, 64)
    for x in cache.layers:
        x.kv = FakeKV()
    return cache.layers[0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_keys_and_values_have_the_model_s_type(dtype):
    x = layer(dtype)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(1, 2, 5, 64, generator=g).to(dtype) for _ in "kv")
    x.update(k, v)
    assert x.keys.dtype == dtype and x.values.dtype == dtype
    assert torch.equal(x.keys, k) and torch.equal(x.values, v)      # no bits lost on the way
    x.keys, x.values = k[:, :, :3], v[:, :, :3]                     # eviction
    assert x.length == 3 and torch.equal(x.keys, k[:, :, :3]) and x.values.dtype == dtype


def test_what_a_step_cannot_attend_to_is_refused_before_it_is_written():
    """fp32 queries are not attended to over codes: the layer says so while its rows and length are as they were."""
    x = layer(torch.float32)
    k = torch.ones(1, 2, 5, 64)
    x.update(k, k)                                                  # a prompt's attention is the model's own
    rows = [r.clone() for r in x.kv.rows]
    with pytest.raises(ValueError, match="FP16/BF16"):
        x.update(2 * k[:, :, :1], 2 * k[:, :, :1])
    assert x.length == 5 and all(torch.equal(a, b) for a, b in zip(rows, x.kv.rows))
    x.update(k[:, :, :1].half(), k[:, :, :1].half())
    assert x.length == 6
