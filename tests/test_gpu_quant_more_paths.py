"""Paths of the quantised cache that its other tests pass by: lists for each query head in every kernel, routing over rows longer
than one cluster selects from and under a graph capture, calls of several threads on one stream, an fp16 model. Tolerances are
those of test_gpu_quant_cache.py and test_gpu_quant_model.py."""
import threading

import pytest
import torch

from test_gpu_quant_cache import check_decode, filled, rand
from test_gpu_quant_model import close, plain_cache, tiny
from utmist_bigger_bird_b200 import install, make_quant_cache, quant_decode, quant_pooled_probs, quant_route

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bits,d,group,dtype", [(4, 128, 32, torch.bfloat16), (8, 128, 64, torch.float16), (4, 96, 96, torch.float16),
                                                (8, 96, 32, torch.bfloat16), (4, 32, 32, torch.bfloat16), (8, 64, 64, torch.bfloat16)])
@pytest.mark.parametrize("g,t", [(2, 1), (5, 1), (12, 1), (4, 3), (3, 40)])
def test_lists_for_each_query_head(bits, d, group, dtype, g, t):
    hk, n, front, window, R = 2, 290, 6, 33, 45
    c = filled(hk, 300, d, bits, group, dtype=dtype)
    gen = torch.Generator(device=DEV).manual_seed(70)
    idx = torch.stack([torch.randperm(310, device=DEV, generator=gen)[:R] - 10 for _ in range(hk * g)])
    q = rand((hk * g, t, d), 71, dtype)
    check_decode(*c, q if t > 1 else q[:, 0], idx, n, front, window, dtype)


def test_several_tokens_over_pooled_lists_in_tiles_of_eight():
    c = filled(2, 300, 96, 8, 96)
    gen = torch.Generator(device=DEV).manual_seed(72)
    idx = torch.stack([torch.randperm(259, device=DEV, generator=gen)[:64] for _ in range(2)])
    check_decode(*c, rand((10, 70, 96), 73), idx, 259, 5, 40, torch.bfloat16)


def is_top(idx, probs):
    assert (idx[:, 1:] > idx[:, :-1]).all()
    for h in range(len(idx)):
        rest = probs[h].clone()
        rest[idx[h]] = -2
        assert probs[h, idx[h]].min() >= rest.max()


@pytest.mark.parametrize("cap,n,k_route", [(900_000, 899_990, 512), (900_000, 800_000, 33), (5000, 4001, 4000)])
def test_route_over_long_rows_and_of_many_keys(cap, n, k_route):
    kv, *_ = filled(1, cap, 64, 4, 64)
    q = rand((4, 1, 64), 74)[:, 0]
    for n_arg in (n, torch.tensor([n], device=DEV)):
        kw = dict(front=16, window=100, scale=0.125, n=n_arg)
        idx = quant_route(q, kv, k_route, **kw)
        assert idx.shape == (1, k_route) and idx.min() >= 0 and idx.max() < cap
        is_top(idx, quant_pooled_probs(q, kv, **kw))


@pytest.mark.parametrize("g", [4, 12])
def test_a_captured_routed_step_follows_the_length(g):
    kv, *_ = filled(cap=3000)
    q = rand((2 * g, 1, 128), 75)[:, 0]
    n = torch.tensor([2000], device=DEV)
    kw = dict(front=8, window=300, scale=128 ** -0.5)

    def step(n):
        idx = quant_route(q, kv, 48, n=n, **kw)
        return idx, quant_decode(q, kv, idx, n=n, **kw)

    step(n)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        idx, out = step(n)
        n += 317
    for m in (2000, 2317, 2634):
        graph.replay()
        step(999)                                              # eager calls in between use other buffers
        want = step(m)
        assert torch.equal(idx, want[0]) and torch.equal(out, want[1])


def test_threads_route_on_one_stream():
    made = []
    for i in range(3):
        kv, *_ = filled(cap=4000 + 1000 * i, seed=80 + 2 * i)
        q = rand(((4, 24, 8)[i], 1, 128), 90 + i)[:, 0]             # 24: two launches for the probabilities
        kw = dict(front=8, window=100 + i, scale=128 ** -0.5, n=3900 + 900 * i)
        made.append((kv, q, kw, quant_route(q, kv, 64, **kw), quant_pooled_probs(q, kv, **kw)))
    torch.cuda.synchronize()
    wrong = []

    def work(kv, q, kw, idx, probs):
        for _ in range(60):
            if not torch.equal(quant_route(q, kv, 64, **kw), idx) or not torch.equal(quant_pooled_probs(q, kv, **kw), probs):
                wrong.append(len(q))

    threads = [threading.Thread(target=work, args=m) for m in made]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_fp16_model():
    model = tiny(DEV, torch.float16)
    install(model, "vs", sink=8, window=96, vertical=10 ** 6, n_route=16, exact_tail=32)
    ids = torch.randint(0, 256, (1, 400), device=DEV)
    cache = make_quant_cache(model, 512, bits=8, group=32)
    plain = plain_cache(cache)
    with torch.inference_mode():
        for a, b in ((0, 300), (300, 301), (301, 302)):
            pos = torch.arange(a, b, device=DEV)[None]
            close(model(ids[:, a:b], past_key_values=cache, position_ids=pos).logits,
                  model(ids[:, a:b], past_key_values=plain, position_ids=pos).logits)
    layer = cache.layers[1]
    assert layer.keys.dtype == layer.values.dtype == torch.float16
    assert torch.equal(layer.keys[0], layer.kv.read(stop=302, dtype=torch.float32)[0].half())
