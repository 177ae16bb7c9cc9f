"""Quantised KV cache kernels on the GPU against the 64-bit restatement of their definition.

Tolerances. Writing and reading: codes, steps and low values have to be equal for 16-bit inputs, and values equal
once rounded. Attention: an output is sum_j p_j v_j; the kernels may round each p_j (times a step) to 11 bits,
2^-12 of |step c| + |low| a key, doubled for the normalisation. Scores are fp32 sums of products of up to `reach`:
an error of 2^-20 reach in a score changes its p by that much of itself, and the sum over p again. So before its
rounding an output is within spread (2^-11 + 2^-18 reach) + 2^-24 of the exact one, spread = sum_j p_j (|low| + step c),
and since rounding is monotone the output lies between the two ends of that range, each rounded to its type."""
import numpy as np
import pytest
import torch

from oracle import quant_cache_oracle as qo

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rand(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(*shape, device=DEV, generator=g) * torch.exp(0.7 * torch.randn(shape[0], 1, shape[2], device=DEV, generator=g))
    return (x + 0.5).to(dtype)


def f64(t):
    return t.double().cpu().numpy()


def filled(hk=2, cap=300, d=128, bits=4, group=32, seed=0, dtype=torch.bfloat16):
    """A cache with every row written, the 64-bit values that it stands for, and |low| + step c of its values."""
    from utmist_bigger_bird_b200 import QuantKV
    kv = QuantKV(hk, cap, d, bits=bits, group=group)
    k, v = rand((hk, cap, d), seed, dtype), rand((hk, cap, d), seed + 1, dtype)
    kv.write(k, v, 0)
    kq, vq = qo.quantise(f64(k), bits, group), qo.quantise(f64(v), bits, group)
    return kv, qo.values(*kq), qo.values(*vq), qo.values(vq[0], vq[1], np.abs(vq[2]))


def check_rounded(got, want, spread, reach):
    tol = spread * (2.0 ** -11 + 2.0 ** -18 * reach[..., None]) + 2.0 ** -24
    low, high = (f64(torch.from_numpy(x).float().to(got.dtype)) for x in (want - tol, want + tol))
    x = f64(got).reshape(want.shape)
    off = np.abs(x - want)
    assert ((low <= x) & (x <= high)).all(), f"error {off.max():.3g}, {(off / tol).max():.3g} of the bound before rounding"


def check_decode(kv, kval, vval, wval, q, idx, n, front, window, dtype, n_arg=None, splits=None):
    from utmist_bigger_bird_b200 import quant_decode
    scale = q.shape[-1] ** -0.5
    got = quant_decode(q, kv, idx, front=front, window=window, scale=scale, n=n if n_arg is None else n_arg, splits=splits)
    assert got.shape == q.shape and got.dtype == q.dtype
    q3 = f64(q if q.ndim == 3 else q[:, None])
    want, spread, reach = qo.decode(q3, kval, vval, None if idx is None else idx.cpu().numpy(), front=front,
                                    window=window, scale=scale, n=n, weight=wval)
    check_rounded(got, want, spread, reach)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,group", [(128, 32), (128, 64), (128, 128), (96, 32), (96, 96), (64, 32), (64, 64), (32, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_write_and_read_are_the_definition(bits, d, group, dtype):
    from utmist_bigger_bird_b200 import QuantKV
    hk, t, at, cap = 3, 37, 5, 50
    kv = QuantKV(hk, cap, d, bits=bits, group=group)
    # rows as a projection gives them: [t, hk * d] storage
    k = rand((1, t, hk * d), 1, dtype)[0].view(t, hk, d).transpose(0, 1)
    v = rand((1, t, hk * d), 2, dtype)[0].view(t, hk, d).transpose(0, 1)
    k[0, 3] = 0.25
    got = kv.write(k, v, at, values=True)
    read = kv.read(start=at, stop=at + t, dtype=torch.float32)
    for x, codes, meta, run, val, back in ((k, kv.k_codes, kv.k_meta, qo.K_RUN, got[0], read[0]),
                                           (v, kv.v_codes, kv.v_meta, qo.V_RUN, got[1], read[1])):
        c, step, low = qo.quantise(f64(x), bits, group)
        assert (codes[:, at:at + t].cpu().numpy() == qo.pack(c, bits, run)).all()
        assert (f64(meta[:, at:at + t, :, 0]) == step).all() and (f64(meta[:, at:at + t, :, 1]) == low).all()
        want = torch.from_numpy(qo.values(c, step, low))
        assert val.dtype == dtype and torch.equal(val.cpu(), want.float().to(dtype))
        assert torch.equal(back.cpu(), want.float())
        rest = [*range(at), *range(at + t, cap)]
        assert not codes[:, rest].any() and not meta[:, rest].any(), "other rows are left alone"


@pytest.mark.parametrize("bits", [4, 8])
def test_write_fp32_inputs(bits):
    """fp32 rows: the low value is rounded down and the step up, so every value lies within half a step."""
    from utmist_bigger_bird_b200 import QuantKV
    kv = QuantKV(1, 64, 128, bits=bits, group=64)
    k = rand((1, 64, 128), 3, torch.float32)
    v = rand((1, 64, 128), 4, torch.float32) * 1e-3
    vals = kv.write(k, v, 0, values=True)
    for x, val, meta in ((k, vals[0], kv.k_meta), (v, vals[1], kv.v_meta)):
        step = f64(meta[..., 0]).repeat(64, -1)
        assert (np.abs(f64(val) - f64(x)) <= step * (0.5 + 2.0 ** -18)).all()


def test_write_special_rows():
    """Groups with a NaN or an infinity read back as NaN and leave their neighbours alone; zero, constant, tiny and
    huge groups read back within half a step."""
    from utmist_bigger_bird_b200 import QuantKV
    kv = QuantKV(1, 8, 128, bits=4, group=32)
    x = torch.randn(1, 8, 128, device=DEV)
    x[0, 0, 5], x[0, 1, 40], x[0, 2, 100] = float("nan"), float("inf"), -float("inf")
    x[0, 3] = 0.0
    x[0, 4] = -7.25
    x[0, 5] *= 1e-36
    x[0, 6] *= 1e37
    x[0, 7, :32] = torch.linspace(-3e38, 3e38, 32)     # a range beyond fp32
    k, _ = kv.write(x, x, 0, values=True)
    nan = torch.isnan(k[0].view(8, 4, 32))
    want = torch.zeros(8, 4, dtype=torch.bool, device=DEV)
    want[0, 0] = want[1, 1] = want[2, 3] = want[7, 0] = True
    assert torch.equal(nan.all(-1), want) and torch.equal(nan.any(-1), want)
    assert not k[0, 3].any() and (k[0, 4] == -7.25).all()
    ok = ~want.repeat_interleave(32, -1)
    step = kv.k_meta[0, :, :, 0].float().repeat_interleave(32, -1)
    err = (k[0] - x[0]).abs()
    small = 2.0 ** -99                                   # steps below 2^-100 are stored as zero
    assert (err <= step * 0.501 + 16 * small)[ok].all()


def test_write_at_device_position_and_edges():
    """A device position is read by the kernel; rows that fall outside the cache are skipped."""
    from utmist_bigger_bird_b200 import QuantKV
    x = rand((2, 4, 64), 5)
    for at, inside in ((3, range(4)), (8, range(2)), (-2, range(2, 4)), (10, ()), (-2 ** 40, ())):
        kv = QuantKV(2, 10, 64, bits=4, group=32)
        kv.write(x, x, torch.tensor([at], device=DEV))
        ref = QuantKV(2, 10, 64, bits=4, group=32)
        for r in inside:
            ref.write(x[:, r:r + 1], x[:, r:r + 1], at + r)
        assert torch.equal(kv.k_codes, ref.k_codes) and torch.equal(kv.v_meta, ref.v_meta), at
    kv = QuantKV(2, 10, 64)
    kv.write(x[:, :0], x[:, :0], 10)                      # no rows
    for bad in (-1, 7):
        with pytest.raises(ValueError):
            kv.write(x, x, bad)
    for k, v in ((x[:1], x[:1]), (x, x[:, :3]), (x, x.half()), (x.double(), x.double()), (x[..., :32], x[..., :32])):
        with pytest.raises(ValueError):
            kv.write(k, v, 0)


@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
def test_read_positions(dt):
    small, *_ = filled()
    for kw in (dict(start=-1), dict(start=4, stop=3), dict(stop=301), dict(dtype=torch.float64),
               dict(positions=torch.zeros(3, 4, dtype=dt, device=DEV)), dict(positions=torch.zeros(2, 4, device=DEV)),
               dict(positions=torch.zeros(2, dtype=dt, device=DEV)), dict(positions=torch.zeros(2, 4, dtype=dt))):
        with pytest.raises(ValueError):
            small.read(**kw)
    kv, kval, vval, _ = filled(hk=3, cap=200, d=96, bits=8, group=96)
    pos = torch.randint(0, 200, (3, 77), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(dt)
    pos[0, 0], pos[1, 5] = -1, 200                        # outside: zeros
    wide = torch.stack([pos, pos], -1).flatten(1)[:, ::2]  # a strided list
    for p in (pos, wide):
        k, v = kv.read(p, dtype=torch.float32)
        for got, val in ((k, kval), (v, vval)):
            at = pos.clamp(0, 199).long().cpu().numpy()
            want = np.take_along_axis(val, at[..., None], 1)
            want[0, 0] = want[1, 5] = 0.0
            assert torch.equal(got.cpu(), torch.from_numpy(want).float())
    k, v = kv.read(pos[:, :0])
    assert k.shape == (3, 0, 96) and v.dtype == torch.bfloat16


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d,group", [(128, 32), (128, 64), (128, 128), (96, 32), (96, 96), (64, 32), (64, 64), (32, 32)])
@pytest.mark.parametrize("g,dtype", [(4, torch.bfloat16), (1, torch.float16), (5, torch.bfloat16), (12, torch.float16)])
def test_dense_decode(bits, d, group, g, dtype):
    hk, cap, n = 2, 300, 277
    c = filled(hk, cap, d, bits, group, dtype=dtype)
    q = rand((hk * g, 1, d), 9, dtype)[:, 0]
    check_decode(*c, q, None, n, 0, cap, dtype)


@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 33, 64, 65, 130, 299, 300])
@pytest.mark.parametrize("front,window", [(0, 300), (0, 0), (4, 0), (4, 20), (64, 64), (20, 1), (400, 5)])
def test_decode_lengths_and_ranges(n, front, window):
    """Every key counts once however front and window meet; a row that sees nothing gives zeros."""
    c = filled()
    q = rand((8, 1, 128), 10)[:, 0]
    check_decode(*c, q, None, n, front, window, torch.bfloat16)
    check_decode(*c, q, None, n, front, window, torch.bfloat16, n_arg=torch.tensor([n], device=DEV))


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
@pytest.mark.parametrize("R,window,front", [(1, 20, 4), (37, 100, 16), (128, 0, 0), (17, 290, 16)])
def test_sparse_decode(per_head, dt, R, window, front):
    """Lists of positions, some of them outside [front, n - window): skipped."""
    hk, g, n = 2, 4, 290
    c = filled()
    gen = torch.Generator(device=DEV).manual_seed(4)
    lists = hk * g if per_head else hk
    idx = torch.stack([torch.randperm(310, device=DEV, generator=gen)[:R] - 10 for _ in range(lists)]).to(dt)
    q = rand((hk * g, 1, 128), 11)[:, 0]
    check_decode(*c, q, idx, n, front, window, torch.bfloat16)
    wide = torch.stack([idx, idx], -1).flatten(1)[:, ::2]
    check_decode(*c, q, wide, n, front, window, torch.bfloat16)


@pytest.mark.parametrize("t", [2, 3, 16, 33])
@pytest.mark.parametrize("front,window,R", [(0, 300, 0), (5, 40, 0), (5, 40, 30), (0, 1, 0)])
@pytest.mark.parametrize("bits,d,g", [(4, 128, 4), (8, 64, 3)])
def test_several_tokens(t, front, window, R, bits, d, g):
    """Each token sees its own keys only: causal, with its own window and its own view of the lists."""
    hk, n = 2, 259
    c = filled(hk, 300, d, bits, 32)
    q = rand((hk * g, t, d), 12)
    idx = None
    if R:
        gen = torch.Generator(device=DEV).manual_seed(6)
        idx = torch.stack([torch.randperm(n, device=DEV, generator=gen)[:R] for _ in range(hk)])
    check_decode(*c, q, idx, n, front, window, torch.bfloat16)
    # tokens as a projection gives them: [t, H * d] storage
    check_decode(*c, q.transpose(0, 1).contiguous().transpose(0, 1), idx, n, front, window, torch.bfloat16)


def test_tokens_before_the_first_key_give_zeros():
    """With a device length below the token count, the first tokens see nothing."""
    from utmist_bigger_bird_b200 import quant_decode
    c = filled()
    q = rand((8, 5, 128), 13)
    check_decode(*c, q, None, 3, 0, 300, torch.bfloat16, n_arg=torch.tensor([3], device=DEV))
    out = quant_decode(q, c[0], front=0, window=300, scale=0.1, n=torch.tensor([-7], device=DEV))
    assert not out.any()
    with pytest.raises(ValueError):
        quant_decode(q, c[0], n=3)


@pytest.mark.parametrize("splits", [1, 2, 7, 1000])
def test_explicit_splits(splits):
    c = filled(cap=3000)
    q = rand((8, 1, 128), 14)[:, 0]
    check_decode(*c, q, None, 2999, 0, 3000, torch.bfloat16, splits=splits)


def test_peaked_and_flat_scores():
    """Queries far larger and far smaller than usual: one key takes all, or every key the same."""
    c = filled(bits=8, group=64)
    for scale in (1e-4, 0.0, 30.0, 2000.0):
        q = (rand((8, 1, 128), 15)[:, 0].float() * scale).to(torch.bfloat16)
        check_decode(*c, q, None, 300, 0, 300, torch.bfloat16)


def test_value_steps_of_many_sizes():
    """Steps that differ by 2^20 between tokens, larger and larger or smaller and smaller along the cache."""
    from utmist_bigger_bird_b200 import QuantKV
    hk, cap, d = 2, 300, 128
    ramp = torch.exp2(torch.linspace(-10, 10, cap, device=DEV))[None, :, None]
    for r in (ramp, ramp.flip(1), torch.zeros_like(ramp)):
        kv = QuantKV(hk, cap, d)
        k, v = rand((hk, cap, d), 16), (rand((hk, cap, d), 17).float() * r).to(torch.bfloat16)
        kv.write(k, v, 0)
        kq, vq = qo.quantise(f64(k), 4, 32), qo.quantise(f64(v), 4, 32)
        q = rand((8, 1, d), 18)[:, 0]
        check_decode(kv, qo.values(*kq), qo.values(*vq), qo.values(vq[0], vq[1], np.abs(vq[2])), q, None, 300, 0, 300,
                     torch.bfloat16)


def test_unread_rows_may_hold_anything():
    """NaN in rows beyond n, between front and window, and beyond a token's own position must not matter."""
    from utmist_bigger_bird_b200 import quant_decode, quant_pooled_probs
    q = rand((8, 1, 128), 19)[:, 0]
    for seed in range(2):
        kv, *vals = filled(seed=seed)
        for meta in (kv.k_meta, kv.v_meta):
            meta[:, 250:] = float("nan")
        kw = dict(scale=0.09, n=250)
        probs = quant_pooled_probs(q, kv, front=4, window=8, **kw)
        assert torch.isfinite(probs).all()
        for meta in (kv.k_meta, kv.v_meta):
            meta[:, 10:200] = float("nan")
        idx = torch.arange(15, 40, device=DEV).expand(2, -1).contiguous()
        out = quant_decode(q, kv, None, front=10, window=50, **kw)
        assert torch.isfinite(out).all()
        check_decode(kv, *vals, q, None, 250, 10, 50, torch.bfloat16)
        assert torch.isnan(quant_decode(q, kv, idx, front=10, window=50, **kw)).any(), "read rows do matter"
    kv, *vals = filled()
    q3 = rand((8, 3, 128), 20)
    kv.v_meta[:, 249] = float("nan")                        # the newest token's own row
    out = quant_decode(q3, kv, front=0, window=300, scale=0.09, n=250)
    assert torch.isfinite(out[:, :2]).all() and torch.isnan(out[:, 2]).any()


@pytest.mark.parametrize("bits,d,group,g,dtype", [(4, 128, 32, 4, torch.bfloat16), (8, 64, 64, 2, torch.float16),
                                                  (4, 96, 96, 5, torch.bfloat16), (8, 128, 128, 12, torch.bfloat16)])
@pytest.mark.parametrize("n,front,window", [(300, 4, 20), (277, 0, 0), (17, 4, 20), (1, 0, 0), (0, 0, 0), (130, 64, 64)])
def test_pooled_probs(bits, d, group, g, dtype, n, front, window):
    """|got - want| <= want (2^-18 reach + 2^-17): fp32 scores, exponentials and sums."""
    from utmist_bigger_bird_b200 import quant_pooled_probs
    hk, cap = 2, 300
    kv, kval, _, _ = filled(hk, cap, d, bits, group, dtype=dtype)
    q = rand((hk * g, 1, d), 21, dtype)[:, 0]
    want = qo.pooled_probs(f64(q), kval, front=front, window=window, scale=d ** -0.5, n=n, cap=cap)
    reach = np.abs(f64(q)).sum(-1).max() * np.abs(kval).max() * d ** -0.5
    for n_arg in (n, torch.tensor([n], device=DEV)):
        got = f64(quant_pooled_probs(q, kv, front=front, window=window, scale=d ** -0.5, n=n_arg))
        assert ((got == -1) == (want == -1)).all()
        live = want != -1
        assert (np.abs(got - want)[live] <= want[live] * (2.0 ** -18 * reach + 2.0 ** -17) + 1e-37).all()


@pytest.mark.parametrize("g", [4, 8, 12])
@pytest.mark.parametrize("splits", [1, 3, 1000])
def test_pooled_probs_explicit_splits(splits, g):
    """Few splits: more scores a warp than its CTA keeps. The same bits in one launch, under a graph capture, and in two
    launches (a call without tickets); more query heads than one column tile."""
    import ctypes as C

    from utmist_bigger_bird_b200 import _lib, quant_pooled_probs
    from utmist_bigger_bird_b200.quant_cache import _args
    hk, cap, d, n = 2, 20000, 128, 19990
    kv, kval, _, _ = filled(hk, cap, d)
    q = rand((hk * g, 1, d), 29)[:, 0]
    kw = dict(front=5, window=77, scale=d ** -0.5, n=n, splits=splits)
    got = quant_pooled_probs(q, kv, **kw)
    want = qo.pooled_probs(f64(q), kval, front=5, window=77, scale=d ** -0.5, n=n, cap=cap)
    reach = np.abs(f64(q)).sum(-1).max() * np.abs(kval).max() * d ** -0.5
    live = want != -1
    assert ((f64(got) == -1) == ~live).all()
    assert (np.abs(f64(got) - want)[live] <= want[live] * (2.0 ** -18 * reach + 2.0 ** -17) + 1e-37).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = quant_pooled_probs(q, kv, **kw)
    graph.replay()
    assert torch.equal(again, got)
    a, _ = _args(q, kv, kw["front"], kw["window"], kw["scale"], n, splits, "probs")
    two, size = torch.zeros_like(got), C.c_size_t(0)
    a.out_probs = two.data_ptr()
    _lib.check(_lib.lib().bb_qkv_route_workspace_size(C.byref(a), C.byref(size)), "probs")
    ws = torch.empty(size.value, dtype=torch.uint8, device=DEV)
    _lib.check(_lib.lib().bb_qkv_route(C.byref(a), ws.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream), "probs")
    assert torch.equal(two, got)


def test_decode_without_tickets_takes_two_launches():
    """The C entry without tickets merges in a second launch, with the same result."""
    import ctypes as C

    from utmist_bigger_bird_b200 import _lib, quant_decode
    from utmist_bigger_bird_b200.quant_cache import _args
    L = _lib.lib()
    for g, bits, d, group in ((4, 4, 128, 32), (7, 8, 96, 96)):
        kv, *_ = filled(2, 3000, d, bits, group)
        q = rand((2 * g, 1, d), 33)[:, 0]
        kw = dict(front=3, window=2000, scale=0.1, n=2990)
        before = L.bb_kernel_launches()
        want = quant_decode(q, kv, **kw)
        one = L.bb_kernel_launches() - before
        a, _ = _args(q, kv, kw["front"], kw["window"], kw["scale"], kw["n"], None, "decode")
        out, size = torch.zeros_like(want), C.c_size_t(0)
        a.out, a.so_h = out.data_ptr(), d
        _lib.check(L.bb_qkv_decode_workspace_size(C.byref(a), C.byref(size)), "decode")
        ws = torch.empty(size.value, dtype=torch.uint8, device=DEV)
        before = L.bb_kernel_launches()
        _lib.check(L.bb_qkv_decode(C.byref(a), ws.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream), "decode")
        assert (one, L.bb_kernel_launches() - before) == (1, 2)
        assert torch.equal(out, want)


def test_route_picks_its_own_top_probabilities():
    from utmist_bigger_bird_b200 import quant_pooled_probs, quant_route
    kv, *_ = filled(cap=5000)
    q = rand((8, 1, 128), 22)[:, 0]
    kw = dict(front=16, window=100, scale=128 ** -0.5, n=4001)
    probs = quant_pooled_probs(q, kv, **kw)
    idx = quant_route(q, kv, 64, **kw)
    assert idx.dtype == torch.int64 and idx.shape == (2, 64) and (idx[:, 1:] > idx[:, :-1]).all()
    for h in range(2):
        rest = probs[h].clone()
        rest[idx[h]] = -2
        assert probs[h, idx[h]].min() >= rest.max()
    assert quant_route(q, kv, 0, **kw).shape == (2, 0)


def test_results_do_not_depend_on_stream_or_repetition():
    """The same call on another stream, and again, gives the same bits; a CUDA graph follows the device length."""
    from utmist_bigger_bird_b200 import quant_decode, quant_pooled_probs
    kv, kval, vval, wval = filled(cap=3000)
    q = rand((8, 1, 128), 23)[:, 0]
    n = torch.tensor([2500], device=DEV)
    kw = dict(front=8, window=1000, scale=128 ** -0.5, n=n)
    idx = torch.arange(100, 400, 3, device=DEV).expand(2, -1).contiguous()
    a, p = quant_decode(q, kv, idx, **kw), quant_pooled_probs(q, kv, **kw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            assert torch.equal(quant_decode(q, kv, idx, **kw), a) and torch.equal(quant_pooled_probs(q, kv, **kw), p)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    x = rand((2, 1, 128), 24)
    with torch.cuda.graph(graph):
        kv.write(x, x, n)
        n += 1
        out, probs = quant_decode(q, kv, idx, **kw), quant_pooled_probs(q, kv, **kw)
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        m = 2501 + step
        assert int(n) == m
        kw["n"] = torch.tensor([m], device=DEV)
        assert torch.equal(out, quant_decode(q, kv, idx, **kw)) and torch.equal(probs, quant_pooled_probs(q, kv, **kw))
    assert torch.equal(kv.read(start=2500, stop=2501)[0], kv.read(start=2502, stop=2503)[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_unaligned_rows(dtype):
    """Queries and new rows that start at odd addresses or have odd strides."""
    from utmist_bigger_bird_b200 import QuantKV
    c = filled(dtype=dtype)
    flat = rand((1, 1, 8 * 131 + 1), 30, dtype).flatten()
    q = flat[1:].as_strided((8, 128), (131, 1), 1)
    check_decode(*c, q, None, 290, 4, 40, dtype)
    q = rand((8, 128, 3), 31, dtype).transpose(1, 2)      # dimensions three elements apart
    check_decode(*c, q, None, 290, 4, 40, dtype)
    x = rand((2, 5, 131), 32, dtype)[..., 1:129]
    a, b = QuantKV(2, 5, 128), QuantKV(2, 5, 128)
    a.write(x, x, 0)
    b.write(x.contiguous(), x.contiguous(), 0)
    assert torch.equal(a.k_codes, b.k_codes) and torch.equal(a.v_meta, b.v_meta)
    # rows on 16-byte but not on 32-byte boundaries
    y = torch.empty(2 * 5 * 136 + 8, dtype=dtype, device=DEV)[8:].view(2, 5, 136)[..., :128].copy_(x)
    vals = b.write(y, y, 0, values=True)
    assert torch.equal(a.k_codes, b.k_codes) and torch.equal(vals[0], a.read(dtype=dtype)[0])


def test_buffers_with_gaps_between_heads():
    """Heads that lie further apart than their rows (a view of a longer cache)."""
    from utmist_bigger_bird_b200 import QuantKV
    whole, kval, vval, wval = filled(cap=300)
    part = QuantKV.from_buffers(whole.k_codes[:, :200], whole.k_meta[:, :200], whole.v_codes[:, :200],
                                whole.v_meta[:, :200], bits=4)
    q = rand((8, 1, 128), 25)[:, 0]
    check_decode(part, kval, vval, wval, q, None, 200, 0, 200, torch.bfloat16)
    assert torch.equal(part.read(start=7, stop=150)[1], whole.read(start=7, stop=150)[1])


def test_offsets_beyond_32_bits():
    """A cache whose later heads start beyond 2^32 bytes (8-bit rows of 128 bytes, 18M rows a head)."""
    from utmist_bigger_bird_b200 import QuantKV
    hk, cap, d = 3, 18_000_000, 128
    kv = QuantKV(hk, cap, d, bits=8, group=128)
    rows = [0, 1, cap // 2, cap - 2, cap - 1]
    x = rand((hk, len(rows), d), 26)
    for i, r in enumerate(rows):
        kv.write(x[:, i:i + 1], x[:, i:i + 1].flip(0), r)
    pos = torch.tensor(rows, device=DEV).expand(hk, -1).contiguous()
    k, v = kv.read(pos, dtype=torch.float32)
    for i, r in enumerate(rows):
        a, b = kv.read(start=r, stop=r + 1, dtype=torch.float32)
        assert torch.equal(a[:, 0], k[:, i]) and torch.equal(b[:, 0], v[:, i])
    kq, vq = qo.quantise(f64(x), 8, 128), qo.quantise(f64(x.flip(0)), 8, 128)
    assert torch.equal(k.cpu(), torch.from_numpy(qo.values(*kq)).float())
    # the rows at the end through the attention, as front | window | list of a 5-key problem
    from utmist_bigger_bird_b200 import quant_decode
    q = rand((hk * 2, 1, d), 27)[:, 0]
    idx = torch.tensor([[cap // 2]] * hk, device=DEV)
    got = quant_decode(q, kv, idx, front=2, window=2, scale=0.09)
    want, spread, reach = qo.decode(f64(q[:, None]), qo.values(*kq), qo.values(*vq), np.full((hk, 1), 2), front=2,
                                    window=2, scale=0.09, n=5, weight=qo.values(vq[0], vq[1], np.abs(vq[2])))
    check_rounded(got, want, spread, reach)


def test_refusals_on_the_gpu():
    from utmist_bigger_bird_b200 import quant_decode, quant_pooled_probs
    kv, *_ = filled()
    q = rand((8, 1, 128), 28)[:, 0]
    idx = torch.zeros(2, 4, dtype=torch.int64, device=DEV)
    for bad in (dict(q=q.float()), dict(q=q[:7]), dict(q=q[:, :64]), dict(q=q.cpu()), dict(n=301), dict(n=-1), dict(front=-1),
                dict(window=-1), dict(indices=idx[:1]), dict(indices=idx.float()), dict(indices=idx.cpu()),
                dict(q=q[:, None][:, :0]), dict(splits=-3)):
        kw = dict(q=q, indices=None)
        kw.update(bad)
        with pytest.raises(ValueError):
            quant_decode(kw.pop("q"), kv, kw.pop("indices"), **kw)
    for bad in (dict(q=q.float()), dict(n=301), dict(window=-1)):
        kw = dict(q=q)
        kw.update(bad)
        with pytest.raises(ValueError):
            quant_pooled_probs(kw.pop("q"), kv, **kw)
