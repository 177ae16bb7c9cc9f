"""Quantised KV cache, without a GPU: the 64-bit restatement against its own definition, struct layouts against
the header, and the refusals of the C entries and of the Python wrappers."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import quant_cache_oracle as qo
from utmist_bigger_bird_b200 import QuantKV, _lib, quant_decode, quant_pooled_probs, quant_route

HEADER = Path(__file__).resolve().parent.parent / "include" / "bb_b200.h"


@pytest.mark.parametrize("bits,group,d", [(4, 32, 128), (4, 96, 96), (8, 64, 64), (8, 32, 32)])
def test_oracle_keeps_its_definition(bits, group, d):
    rng = np.random.default_rng(1)
    x = rng.normal(size=(3, 50, d)) * np.exp(rng.normal(size=(3, 50, 1)))
    x[0, 0, :] = 1.5       # a constant group
    x[1, 1, :] = 0.0
    c, step, low = qo.quantise(x, bits, group)
    v = qo.values(c, step, low)
    s = np.repeat(step, group, -1)
    assert c.min() >= 0 and c.max() == 2 ** bits - 1
    assert (np.abs(v - x) <= s / 2 * (1 + 1e-12) + 1e-300).all()      # every value within half a step
    assert (v[0, 0] == 1.5).all() and (v[1, 1] == 0.0).all()
    for t in (step, low):                                                # representable in bf16
        assert (torch.from_numpy(t).to(torch.bfloat16).double().numpy() == t).all()
    for run in (qo.K_RUN, qo.V_RUN):
        assert sorted(qo.place(d, run)) == list(range(d))
        assert (qo.unpack(qo.pack(c, bits, run), bits, run) == c).all()


def test_struct_layouts_match_header(tmp_path):
    structs = {"bb_qkv_cache": _lib.QkvCache, "bb_qkv_write_args": _lib.QkvWriteArgs,
               "bb_qkv_read_args": _lib.QkvReadArgs, "bb_qkv_attn_args": _lib.QkvAttnArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for name, py in structs.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, v = line.split()
        want = C.sizeof(structs[name]) if field == "size" else getattr(structs[name], field).offset
        assert int(v) == want, line


BUF = 1 << 20  # an address that passes the alignment checks; nothing is launched on it here


def cache(**kw):
    base = dict(k_codes=BUF, k_meta=BUF, v_codes=BUF, v_meta=BUF, k_codes_h=64 * 100, k_meta_h=400, v_codes_h=64 * 100,
                v_meta_h=400, kv_heads=8, cap=100, d=128, bits=4, group=32)
    base.update(kw)
    return _lib.QkvCache(**base)


def attn(cache_kw=None, **kw):
    base = dict(heads=32, t=1, n=100, front=4, window=16, scale=0.1, dtype=1)
    base.update(kw)
    return _lib.QkvAttnArgs(cache=cache(**(cache_kw or {})), **base)


@pytest.mark.parametrize("cache_kw,kw,status,msg", [
    (dict(bits=3), {}, 7, "bits"),
    (dict(d=40), {}, 7, "head_dim"),
    (dict(d=160), {}, 7, "head_dim"),
    (dict(group=96), {}, 2, "group"),
    (dict(group=16), {}, 2, "group"),
    (dict(kv_heads=0), {}, 2, "kv_heads"),
    (dict(cap=0), {}, 2, "capacity"),
    (dict(cap=2 ** 31 - 64), {}, 2, "capacity"),
    (dict(k_meta=None), {}, 1, "null"),
    (dict(v_codes=BUF + 8), {}, 4, "16-byte"),
    (dict(k_codes_h=64 * 99), {}, 4, "overlap"),
    (dict(v_meta_h=402), {}, 4, "whole rows"),
    (None, dict(dtype=2), 3, "fp16 or bf16"),
    (None, dict(heads=30), 2, "multiple"),
    (None, dict(t=0), 2, "tokens"),
    (None, dict(n=101), 1, "capacity"),
    (None, dict(front=-1), 1, "front"),
    (None, dict(window=-1), 1, "window"),
    (None, dict(route_k=-1), 1, "route"),
    (None, dict(splits=-1), 1, "splits"),
    (None, dict(route_k=5, route_rows=7), 2, "indices"),
])
def test_decode_refusals(cache_kw, kw, status, msg):
    L, size = _lib.lib(), C.c_size_t(0)
    a = attn(cache_kw, **kw)
    assert L.bb_qkv_decode_workspace_size(C.byref(a), C.byref(size)) == status
    assert msg in L.bb_last_error().decode()
    assert L.bb_qkv_decode(C.byref(a), None, 0, None) == status


def test_call_refusals():
    L, size = _lib.lib(), C.c_size_t(0)
    a = attn()
    assert L.bb_qkv_decode_workspace_size(C.byref(a), C.byref(size)) == 0 and size.value > 0
    assert L.bb_qkv_decode_workspace_size(C.byref(a), None) == 1
    assert L.bb_qkv_decode_workspace_size(None, C.byref(size)) == 1
    assert L.bb_qkv_decode(C.byref(a), None, 0, None) == 5                 # no workspace
    assert L.bb_qkv_decode(C.byref(a), BUF, size.value, None) == 1         # no q / out
    assert L.bb_qkv_route_workspace_size(C.byref(a), C.byref(size)) == 0 and size.value > 0
    assert L.bb_qkv_route(C.byref(a), BUF, size.value, None) == 1          # no q, no output
    b = attn(t=2)
    assert L.bb_qkv_route_workspace_size(C.byref(b), C.byref(size)) == 2
    b = attn(route_k=101)
    assert L.bb_qkv_route_workspace_size(C.byref(b), C.byref(size)) == 1
    w = _lib.QkvWriteArgs(cache=cache(), t=2, at=99, dtype=1)
    assert L.bb_qkv_write(C.byref(w), None) == 1 and "rows" in L.bb_last_error().decode()
    w.at = 98
    assert L.bb_qkv_write(C.byref(w), None) == 1                           # null k
    w.k = w.v = BUF
    w.sk_t = w.sv_t = 4
    assert L.bb_qkv_write(C.byref(w), None) == 4                           # 8-byte rows
    w.t = 0
    assert L.bb_qkv_write(C.byref(w), None) == 0                           # nothing to do
    w.dtype = 7
    assert L.bb_qkv_write(C.byref(w), None) == 3
    assert L.bb_qkv_write(None, None) == 1
    r = _lib.QkvReadArgs(cache=cache(), rows=3, start=98, dtype=1)
    assert L.bb_qkv_read(C.byref(r), None) == 1
    r.start = 97
    assert L.bb_qkv_read(C.byref(r), None) == 1                            # null output
    r.rows = 0
    assert L.bb_qkv_read(C.byref(r), None) == 0
    assert L.bb_qkv_read(None, None) == 1


@pytest.mark.parametrize("kw", [dict(bits=2), dict(head_dim=72), dict(head_dim=256), dict(group=48), dict(group=0),
                                dict(capacity=0), dict(kv_heads=0), dict(group=96)])
def test_holder_refusals(kw):
    base = dict(kv_heads=2, capacity=10, head_dim=128, device="cpu")
    base.update(kw)
    with pytest.raises(ValueError):
        QuantKV(base.pop("kv_heads"), base.pop("capacity"), base.pop("head_dim"), **base)


def test_wrapper_refusals():
    kv = QuantKV(2, 10, 64, bits=8, group=64, device="cpu")
    assert kv.nbytes == 2 * (2 * 10 * 64 + 2 * 10 * 2 * 2)
    x = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        kv.write(x, x, 0)
    q = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: quant_decode(q, kv), lambda: quant_pooled_probs(q, kv), lambda: quant_route(q, kv, 2)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for bad in (lambda: quant_decode(q[0], kv), lambda: quant_pooled_probs(q[None], kv), lambda: quant_route(q, kv, 11)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="dtype"):
        kv.read(dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA"):
        kv.read()
    buf = (kv.k_codes, kv.k_meta, kv.v_codes, kv.v_meta)
    same = QuantKV.from_buffers(*buf, bits=8)
    assert (same.head_dim, same.group, same.capacity, same.kv_heads) == (64, 64, 10, 2)
    for bad in ((buf[0].float(), *buf[1:]), (buf[0][:, ::2], *buf[1:]), (buf[0], buf[1][:, :5], *buf[2:]),
                (buf[0], buf[1].half(), *buf[2:]), (buf[0][:, :, :32].contiguous(), *buf[1:])):
        with pytest.raises(ValueError):
            QuantKV.from_buffers(*bad, bits=8)
