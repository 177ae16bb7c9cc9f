"""More query rows in a call than 65535: follow-up prompts of hundreds of tokens for many heads."""
import numpy as np
import pytest
import torch

from oracle import quant_cache_oracle as qo
from test_gpu_quant_cache import check_rounded, f64, filled, rand
from test_gpu_quant_model import close, tiny
from utmist_bigger_bird_b200 import install, make_quant_cache, quant_decode

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits,d,front,window", [(4, 64, 0, 1000), (8, 32, 7, 150)])
def test_decode_of_many_rows(bits, d, front, window):
    hk, g, t, n = 2, 64, 600, 900                            # 76800 query rows
    kv, kval, vval, wval = filled(hk, 1000, d, bits, 32)
    q = rand((hk * g, t, d), 50)
    got = quant_decode(q, kv, front=front, window=window, scale=d ** -0.5, n=n)
    assert got.shape == q.shape
    for i in (0, 1, 299, 511, 512, 599):                       # a token alone, as of its own position
        want, spread, reach = qo.decode(f64(q[:, i:i + 1]), kval, vval, None, front=front, window=window, scale=d ** -0.5,
                                        n=n - t + i + 1, weight=wval)
        check_rounded(got[:, i:i + 1], want, spread, reach)


def test_a_model_s_long_follow_up():
    """A follow-up prompt of 1100 tokens for 64 heads in one call, and the same in two pieces."""
    model = tiny(DEV, heads=64)
    install(model, "vs", sink=8, window=96, vertical=10 ** 6, n_route=16, exact_tail=32)
    ids = torch.randint(0, 256, (1, 1400), device=DEV)
    one, two = make_quant_cache(model, 1400), make_quant_cache(model, 1400)

    def run(cache, a, b):
        return model(ids[:, a:b], past_key_values=cache, position_ids=torch.arange(a, b, device=DEV)[None]).logits

    with torch.inference_mode():
        run(one, 0, 300), run(two, 0, 300)
        got = run(one, 300, 1400)
        want = torch.cat([run(two, 300, 800), run(two, 800, 1400)], 1)
    close(got, want)
    assert [layer.length for layer in one.layers] == [1400, 1400]


def test_explicit_splits_with_more_tiles_than_counters():
    """More tiles of query rows than a stream keeps counters for: the splits are merged in a second launch."""
    from utmist_bigger_bird_b200 import _lib
    hk, g, t, n, d = 2, 64, 200, 900, 64                     # 2 x 1600 tiles
    kv, kval, vval, wval = filled(hk, 1000, d, 4, 32)
    q = rand((hk * g, t, d), 51)
    before = _lib.lib().bb_kernel_launches()
    got = quant_decode(q, kv, front=0, window=n, scale=d ** -0.5, n=n, splits=2)
    assert _lib.lib().bb_kernel_launches() - before == 2
    for i in (0, 77, 199):
        want, spread, reach = qo.decode(f64(q[:, i:i + 1]), kval, vval, None, front=0, window=n, scale=d ** -0.5,
                                        n=n - t + i + 1, weight=wval)
        check_rounded(got[:, i:i + 1], want, spread, reach)
