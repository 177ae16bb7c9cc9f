"""A model on the quantised cache (make_quant_cache): prompt, follow-up tokens, single tokens (dense and routed), against
the same model whose cache gives the same stored values back as plain tensors.

Tolerance. Both runs compute in bf16 (8 significant bits) and differ in the roundings of the two layers' attention outputs and
of the stored values (at most four of 2^-8 a layer on the way to the logits, which they reach through sums of many
terms): the logits' difference stays below 8 x 2^-8 of their own root mean square on average, and below 8 times that at
the most."""
import pytest
import torch

from utmist_bigger_bird_b200 import install, make_quant_cache

DEV = "cuda"


def tiny(device, dtype=torch.bfloat16, heads=8, kv_heads=2, head_dim=64):
    from transformers import LlamaConfig, LlamaForCausalLM
    cfg = LlamaConfig(vocab_size=256, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=heads,
                      num_key_value_heads=kv_heads, head_dim=head_dim, max_position_embeddings=4096, attn_implementation="sdpa")
    torch.manual_seed(0)
    return LlamaForCausalLM(cfg).to(device, dtype).eval()


def plain_cache(like):
    """A cache that stores what ``like`` would and returns all of it as tensors."""
    from transformers.cache_utils import Cache
    base = type(like.layers[0])

    class Plain(base):
        def update(self, k, v, *args, **kwargs):
            self.kv.write(k[0], v[0], self.length)
            self.length += k.shape[-2]
            return tuple(x[None] for x in self.kv.read(stop=self.length, dtype=k.dtype))

    layers = []
    for layer in like.layers:
        kv = layer.kv
        layers.append(Plain(type(kv)(kv.kv_heads, kv.capacity, kv.head_dim, bits=kv.bits, group=kv.group), None))
    return Cache(layers=layers)


def close(got, want):
    got, want = got.float(), want.float()
    rms = want.square().mean().sqrt()
    diff = (got - want).abs()
    assert diff.mean() <= 8 * 2.0 ** -8 * rms and diff.max() <= 64 * 2.0 ** -8 * rms, (diff.mean() / rms, diff.max() / rms)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,group", [(8, 64), (4, 32)])
def test_model_on_the_quantised_cache(bits, group):
    model = tiny(DEV)
    install(model, "vs", sink=8, window=96, vertical=10 ** 6, n_route=16, exact_tail=32)
    ids = torch.randint(0, 256, (1, 400), device=DEV)
    cache = make_quant_cache(model, 512, bits=bits, group=group)
    plain = plain_cache(cache)
    with torch.inference_mode():
        for a, b in ((0, 300), (300, 301), (301, 317), (317, 318), (318, 319)):  # prompt, tokens, a follow-up, tokens
            pos = torch.arange(a, b, device=DEV)[None]
            got = model(ids[:, a:b], past_key_values=cache, position_ids=pos).logits
            if b - a > 1 and a:  # the plain run gives each of several new tokens its own past
                want = torch.cat([model(ids[:, i:i + 1], past_key_values=plain, position_ids=pos[:, i - a:i - a + 1]).logits
                                  for i in range(a, b)], 1)
            else:
                want = model(ids[:, a:b], past_key_values=plain, position_ids=pos).logits
            close(got, want)
    assert cache.get_seq_length() == 319 and cache.layers[1].kv.capacity == 512


@pytest.mark.gpu
def test_routed_steps_with_nearly_every_key_routed():
    """Routes that leave out only the one or two least probable keys hardly change a step."""
    model = tiny(DEV)
    install(model, "vs", sink=8, window=96, vertical=10 ** 6, n_route=16, exact_tail=32)
    ids = torch.randint(0, 256, (1, 330), device=DEV)
    dense = make_quant_cache(model, 400)
    routed = make_quant_cache(model, 400, sparse=dict(front=8, window=64, k_route=228))
    with torch.inference_mode():
        for a, b in ((0, 300), (300, 301), (301, 302)):
            pos = torch.arange(a, b, device=DEV)[None]
            got = model(ids[:, a:b], past_key_values=routed, position_ids=pos).logits
            close(got, model(ids[:, a:b], past_key_values=dense, position_ids=pos).logits)


@pytest.mark.gpu
def test_generate_and_eviction():
    model = tiny(DEV)
    install(model, "vs", sink=8, window=96, vertical=32, n_route=16, exact_tail=32, kv_evict=True)
    ids = torch.randint(0, 256, (1, 300), device=DEV)
    cache = make_quant_cache(model, 512, bits=8, group=64)
    with torch.inference_mode():
        model(ids, past_key_values=cache)
        layer = cache.layers[0]
        kept = model.model.layers[0].self_attn.kept
        assert layer.length == kept.shape[-1] < 300
        assert layer.keys.shape == (1, 2, layer.length, 64)
        out = model(ids[:, :1], past_key_values=cache, position_ids=torch.tensor([[300]], device=DEV)).logits
    assert torch.isfinite(out).all() and layer.length == kept.shape[-1] + 1
    install(model, "vs", sink=8, window=96, vertical=32, n_route=16, exact_tail=32)
    cache = make_quant_cache(model, 512, bits=8, group=64, sparse=dict(front=8, window=96, k_route=32))
    out = model.generate(ids, past_key_values=cache, max_new_tokens=6, do_sample=False)
    assert out.shape[1] <= 306 and cache.get_seq_length() >= 300
    cache.reset()
    assert cache.get_seq_length() == 0


def test_refusals():
    model = tiny("cpu")
    with pytest.raises(ValueError, match="RDAttention"):
        make_quant_cache(model, 64)
    install(model, "vs")
    for sparse in (dict(front=1), dict(front=1, window=2, k_route=-1)):
        with pytest.raises(ValueError, match="sparse"):
            make_quant_cache(model, 64, sparse=sparse)
    with pytest.raises(ValueError):
        make_quant_cache(model, 64, bits=5)
    cache = make_quant_cache(model, 64)
    assert cache.get_seq_length() == 0 and len(cache.layers) == 2
    x = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="batch"):
        cache.update(x, x, 0)
