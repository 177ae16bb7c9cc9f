"""A Hugging Face cache whose layers are ``QuantKV``: prefill, decode routing and decode of a model on the quantised
cache, for models whose attention is ``RDAttention`` (``install``).

    install(model, "vs", sink=64, window=4096, vertical=512)
    cache = make_quant_cache(model, capacity=131072, bits=4)
    logits = model(prompt_ids, past_key_values=cache).logits      # or model.generate(..., past_key_values=cache)

``update`` quantises the new rows. The first call of a layer (the prompt) returns the values that the rows now
stand for, so the prefill attends to what later steps read; later calls return a handle whose ``attend``
``RDAttention.exact_attention`` calls: dense attention over the cache, or, for single tokens with ``sparse`` and a
cache longer than front + window + k_route, ``quant_route`` and ``quant_decode`` over front | window | routes (the
routed result at a dense step's price or more: routing reads every key).
Steps after the prompt require FP16 or BF16. ``RDAttention(kv_evict=True)`` works: the kept rows are quantised again in
the place of the prompt.
"""
from __future__ import annotations

import torch

from .quant_cache import QuantKV, quant_decode, quant_route

__all__ = ["make_quant_cache"]


class _Handle:
    """What ``update`` returns in the place of K and V once a cache holds rows."""

    turbo = True  # the attribute by which RDAttention.exact_attention finds ``attend``

    def __init__(self, layer):
        kv = layer.kv
        self.layer, self.shape = layer, (1, kv.kv_heads, layer.length, kv.head_dim)

    def attend(self, q, scaling):
        """q [1, H, t, d] -> [1, H, t, d]: each of the newest t tokens over its own past."""
        layer, t = self.layer, q.shape[2]
        kv, n, s = layer.kv, layer.length, layer.sparse
        if t > 1:
            return quant_decode(q[0], kv, front=0, window=n, scale=scaling, n=n)[None]
        q1 = q[0, :, 0]
        if s and n > s["front"] + s["window"] + s["k_route"]:
            kw = dict(front=s["front"], window=s["window"], scale=scaling, n=n)
            out = quant_decode(q1, kv, quant_route(q1, kv, s["k_route"], **kw), **kw)
        else:
            out = quant_decode(q1, kv, front=0, window=n, scale=scaling, n=n)
        return out[None, :, None]


def _layer_class():
    from transformers.cache_utils import CacheLayerMixin

    class QuantLayer(CacheLayerMixin):
        is_sliding = False

        def __init__(self, kv, sparse):
            self.kv, self.sparse, self.length, self._kept = kv, sparse, 0, None
            self.dtype = torch.bfloat16  # of keys and values as tensors: the model's, once rows have come
            self.is_initialized = True

        def lazy_initialization(self, key_states, value_states):
            pass

        def update(self, key_states, value_states, *args, **kwargs):
            if key_states.shape[0] != 1:
                raise ValueError("batch size 1 only")
            first, t = self.length == 0, key_states.shape[-2]
            if not first and key_states.dtype not in (torch.float16, torch.bfloat16):  # before any row is written
                raise ValueError("attention over a quantised cache requires FP16/BF16")
            self.dtype = key_states.dtype
            values = self.kv.write(key_states[0], value_states[0], self.length, values=first)
            self.length += t
            if first:
                return values[0][None], values[1][None]
            handle = _Handle(self)
            return handle, handle

        # RDAttention.evict sets keys, then values, to the rows that stay
        @property
        def keys(self):
            return self.kv.read(stop=self.length, dtype=self.dtype)[0][None]

        @keys.setter
        def keys(self, rows):
            self._kept = rows

        @property
        def values(self):
            return self.kv.read(stop=self.length, dtype=self.dtype)[1][None]

        @values.setter
        def values(self, rows):
            kept, self._kept = self._kept, None
            if kept is not None and rows is not None:
                self.kv.write(kept[0], rows[0], 0)
                self.length = kept.shape[-2]

        def get_seq_length(self):
            return self.length

        def get_max_cache_shape(self):
            return self.kv.capacity

        def get_mask_sizes(self, query_length):
            return self.length + query_length, 0

        def reset(self):
            self.length = 0

        def offload(self):
            raise NotImplementedError("a quantised cache stays on its device")

        prefetch = offload

        def reorder_cache(self, beam_idx):
            raise NotImplementedError("batch size 1 only")

    return QuantLayer


def make_quant_cache(model, capacity, *, bits=4, group=32, sparse=None):
    """A ``transformers`` Cache of one ``QuantKV`` of ``capacity`` rows a layer of ``model``. ``sparse``: None, or
    ``dict(front=, window=, k_route=)`` for routed single-token steps."""
    from transformers.cache_utils import Cache

    if sparse is not None and (set(sparse) != {"front", "window", "k_route"} or min(sparse.values()) < 0):
        raise ValueError("make_quant_cache: sparse is dict(front=, window=, k_route=), none of them negative")
    layer = _layer_class()
    layers = []
    for block in model.model.layers:
        attn = block.self_attn
        if not hasattr(attn, "exact_attention"):
            raise ValueError("make_quant_cache: install RDAttention in the model first")
        kv = QuantKV(attn.num_kv_heads, capacity, attn.head_dim, bits=bits, group=group, device=attn.k_proj.weight.device)
        layers.append(layer(kv, sparse))
    return Cache(layers=layers)
