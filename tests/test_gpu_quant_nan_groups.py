"""A value group that is stored as NaN (it held a NaN or an infinity) makes the dimensions of that group NaN in the tokens
that attend to it, and no others."""
import numpy as np
import pytest
import torch

from oracle import quant_cache_oracle as qo
from test_gpu_quant_cache import check_rounded, f64, filled, rand
from utmist_bigger_bird_b200 import quant_decode

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,group", [(128, 32), (128, 64), (96, 32), (64, 32)])
@pytest.mark.parametrize("g", [4, 5, 12])
@pytest.mark.parametrize("key", [100, 285])                  # among whole steps, and in the last, partial one
def test_nan_stays_in_its_group(bits, d, group, g, key):
    hk, n = 2, 290
    kv, kval, vval, wval = filled(hk, 300, d, bits, group)
    q = rand((hk * g, 1, d), 60)[:, 0]
    want, spread, reach = qo.decode(f64(q[:, None]), kval, vval, None, front=0, window=300, scale=d ** -0.5, n=n, weight=wval)
    meta = kv.v_meta.clone()
    for bad in range(d // group):
        kv.v_meta.copy_(meta)
        kv.v_meta[1, key, bad] = float("nan")
        got = quant_decode(q, kv, front=0, window=300, scale=d ** -0.5, n=n)
        dims = np.arange(d) // group == bad
        assert torch.isnan(got[g:, torch.from_numpy(dims)]).all()
        check_rounded(got[:g, None], want[:g], spread[:g], reach[:g])
        check_rounded(got[g:, None][..., torch.from_numpy(~dims)], want[g:, :, ~dims], spread[g:, :, ~dims], reach[g:])
