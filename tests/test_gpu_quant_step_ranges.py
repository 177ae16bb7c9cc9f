"""Value groups of one token whose steps are far apart, attended to by many small probabilities.

P step is rounded to 11 bits wherever it stays in fp16's normal range, which must not depend on what other groups hold: the
tolerance is that of test_gpu_quant_cache.py. All keys but one are equal and so are their values, so that the roundings of
their P add up instead of cancelling."""
import numpy as np
import pytest
import torch

from oracle import quant_cache_oracle as qo
from test_gpu_quant_cache import check_decode, f64, rand
from utmist_bigger_bird_b200 import QuantKV

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,group,g", [(128, 32, 4), (128, 64, 4), (64, 32, 2), (128, 32, 8), (96, 32, 5), (128, 64, 12)])
@pytest.mark.parametrize("power", [10, 20])
@pytest.mark.parametrize("peak", [3, 2900])
def test_groups_far_apart_keep_their_bits(bits, d, group, g, power, peak):
    hk, n = 2, 3000
    k = torch.zeros(hk, n, d, device=DEV, dtype=torch.bfloat16)
    q = rand((hk * g, 1, d), 61)[:, 0].abs()
    k[:, peak] = 8.0 / float(q.float().sum(-1).mean() * d ** -0.5)       # p of the others: about 2^-12 of its p
    v = rand((hk, 2, d), 62).float()
    for big in range(d // group):                                        # one group large, the others small
        size = torch.ones(d, device=DEV)
        size[big * group:(big + 1) * group] = 2.0 ** power
        rows = v[:, :1].expand(-1, n, -1).clone()
        rows[:, peak] = v[:, 1]
        rows = (rows * size).to(torch.bfloat16)
        kv = QuantKV(hk, n, d, bits=bits, group=group)
        kv.write(k, rows, 0)
        kq, vq = qo.quantise(f64(k), bits, group), qo.quantise(f64(rows), bits, group)
        check_decode(kv, qo.values(*kq), qo.values(*vq), qo.values(vq[0], vq[1], np.abs(vq[2])), q, None, n, 0, n, torch.bfloat16)
