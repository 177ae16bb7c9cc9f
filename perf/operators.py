"""The quantised KV cache's operators, as they are measured: inputs, plain forms, exact values and work.

A cache row (one token of one KV head) holds `bits`-bit codes of its `d` values and, for every `group` of them, a
step and a low value in bf16; a code c stands for low + step * c. Four operators work on it:

  write   quantises new rows into the cache and returns the values that the cache now holds
  read    gives rows back as values (a range, or positions chosen for each KV head)
  decode  attention of the newest token or tokens over the cached keys: the first `front`, the last `window` and
          routed ones
  probs   the attention probabilities of every cached key, averaged over the query heads of its KV head

Order of the codes in a row: with G = d / 32, the code of dimension 32 g + run a + i stands at place
(a G + g) run + i, run = 8 for keys and 4 for values. A 4-bit row keeps place 2 b in the low half of byte b and
place 2 b + 1 in its high half; an 8-bit row keeps place b in byte b.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
K_RUN, V_RUN = 8, 4


# ------------------------------------------------------------------------------------------------- cases
def listed():
    base = dict(d=128, hk=8, g=4, bits=4, group=32, dtype="bf16")
    return [
        # one decoding step's new row of every KV head: latency
        dict(base, name="write one token", op="write", t=1, at=131071, cap=131072),
        # a whole 128K-token prompt written after its prefill
        dict(base, name="write 128k prompt", op="write", t=131072, at=0, cap=131072),
        # a short odd-length piece of a prompt, 8-bit, smaller heads, appended at an odd position
        dict(base, name="write odd piece 8-bit", op="write", t=4099, at=1021, cap=8192, d=64, hk=4, bits=8, group=64,
             dtype="fp16"),
        # the rows that a step's routes point at
        dict(base, name="read 512 routed rows", op="read", n=131072, cap=131072, rows=512),
        # the whole 128K-token cache as 16-bit values
        dict(base, name="read 128k", op="read", n=131072, cap=131072, rows=0),
        # a short conversation on a small model: latency
        dict(base, name="decode short 8-bit", op="decode", n=257, cap=1024, t=1, front=0, window=1024, routes=0,
             per_head=False, d=64, hk=4, g=2, bits=8, group=64, dtype="fp16"),
        # the sparse decode step of a 128K-token prompt: sink, window and pooled routes
        dict(base, name="decode sparse 128k", op="decode", n=131072, cap=131072, t=1, front=64, window=16384,
             routes=512, per_head=False),
        # the same step over every key
        dict(base, name="decode dense 128k", op="decode", n=131072, cap=131072, t=1, front=0, window=131072, routes=0,
             per_head=False),
        # a million-token prompt, one step over every key, coarser groups
        dict(base, name="decode dense 1m", op="decode", n=1048573, cap=1048576, t=1, front=0, window=1048576, routes=0,
             per_head=False, group=128),
        # a short follow-up of sixteen tokens on a 32K-token cache of odd length
        dict(base, name="decode 16 tokens 32k", op="decode", n=32771, cap=32800, t=16, front=0, window=32800, routes=0,
             per_head=False),
        # a decode step's routing over a 128K-token cache
        dict(base, name="probs 128k", op="probs", n=131072, cap=131072, front=64, window=16384),
        # routing over an odd 20K-token cache in 8 bits with room to grow
        dict(base, name="probs odd 20k 8-bit", op="probs", n=20011, cap=24576, front=64, window=4096, d=64, hk=4, g=2,
             bits=8, group=64, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "decode", "decode", "probs"])
    d = rng.choice([64, 96, 128, 128])
    c = dict(op=op, d=d, hk=rng.choice([1, 2, 4, 8]), g=rng.choice([1, 2, 4, 5, 8]), bits=rng.choice([4, 4, 8]),
             group=rng.choice([s for s in (32, 64, 96, 128) if d % s == 0]), dtype=rng.choice(["bf16", "fp16"]))
    room = rng.randrange(0, 400)
    if op == "write":
        t = _log(rng, 1, 131072)
        at = rng.randrange(0, 5000)
        return dict(c, t=t, at=at, cap=at + t + room)
    n = _log(rng, 8 if op == "probs" else 1, 400000 if op == "decode" else 131072)
    c.update(n=n, cap=n + room)
    if op == "read":
        return dict(c, rows=0 if rng.random() < 0.5 else _log(rng, 1, 4096))
    front = rng.choice([0, 16, 64])
    window = rng.choice([n + 1, _log(rng, 1, 16384), _log(rng, 1, 16384)])
    if op == "probs":
        return dict(c, front=min(front, n // 4), window=min(window, n // 2))
    t = rng.choice([1, 1, 1, rng.randrange(2, 17)]) if n <= 65536 else 1
    t = min(t, n)
    middle = n - t + 1 - window - front  # keys that routes may point at
    routes = min(_log(rng, 1, 2048), middle) if middle > 0 and t == 1 else 0
    return dict(c, t=t, front=front, window=window, routes=routes, per_head=routes > 0 and rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------- inputs
def _keys_values(case, tokens, gen):
    """Rows as a projection gives them, seen as [hk, tokens, d]: keys with an offset and a scale of their own in every
    channel (some channels far larger), values with a scale of their own in every token."""
    hk, d, dt = case["hk"], case["d"], DTYPES[case["dtype"]]
    new = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    chan = torch.exp(0.4 * new(hk * d)) * torch.where(torch.rand(hk * d, device="cuda", generator=gen) < 0.03, 4.0, 0.7)
    k = (new(tokens, hk * d) * chan + 0.5 * new(hk * d)).to(dt)
    v = (new(tokens, hk * d) * torch.exp(0.3 * new(tokens, 1))).to(dt)
    return k.view(tokens, hk, d).transpose(0, 1), v.view(tokens, hk, d).transpose(0, 1)


def _empty_cache(case):
    hk, cap, d, ng = case["hk"], case["cap"], case["d"], case["d"] // case["group"]
    codes = [torch.zeros(hk, cap, d * case["bits"] // 8, dtype=torch.uint8, device="cuda") for _ in "kv"]
    meta = [torch.zeros(hk, cap, ng, 2, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
    return codes + meta


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kc, vc, km, vm = _empty_cache(case)
    s = dict(case, kc=kc, vc=vc, km=km, vm=vm)
    d, hk, h, dt = case["d"], case["hk"], case["hk"] * case["g"], DTYPES[case["dtype"]]
    if case["op"] == "write":
        s["k"], s["v"] = _keys_values(case, case["t"], gen)
    else:
        n, step = case["n"], 131072
        q = torch.randn(h, case.get("t", 1), d, device="cuda", generator=gen)
        for a in range(0, n, step):  # in pieces, to keep the inputs' own memory small
            b = min(n, a + step)
            k, v = _keys_values(case, b - a, gen)
            if a == 0:  # each query looks for a few of the keys: rows that attention concentrates on
                near = torch.randint(0, b - a, (h, case.get("t", 1)), device="cuda", generator=gen)
                mine = torch.arange(h, device="cuda")[:, None] // case["g"]
                q = q * 0.6 + 0.25 * k[mine, near].float()
            for x, codes, meta, run in ((k, kc, km, K_RUN), (v, vc, vm, V_RUN)):
                c, low, gap = _quantise(x.float(), case["bits"], case["group"])
                codes[:, a:b] = _pack(c, case["bits"], run)
                meta[:, a:b, :, 0], meta[:, a:b, :, 1] = gap, low
        s["q"] = q.to(dt) if case["op"] == "decode" and case["t"] > 1 else q[:, 0].to(dt)
    if case["op"] == "read" and case["rows"]:
        s["positions"] = torch.randint(0, case["n"], (hk, case["rows"]), device="cuda", generator=gen).sort(-1).values
    if case["op"] == "decode" and case["routes"]:
        lo, hi = case["front"], case["n"] - case["window"]
        lists = h if case["per_head"] else hk
        pick = torch.rand(lists, hi - lo, device="cuda", generator=gen).argsort(-1)[:, : case["routes"]]
        s["idx"] = (pick + lo).sort(-1).values.contiguous()
    if own:  # the handle that a program keeps over the same four buffers
        from utmist_bigger_bird_b200 import QuantKV

        s["kv"] = QuantKV.from_buffers(kc, km, vc, vm, bits=case["bits"])
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _bf16_down(x):
    """The largest bf16 number not above x (fp32), as fp32."""
    u = x.contiguous().view(torch.int32)
    cut = u & -65536
    return torch.where((u < 0) & (cut != u), cut + 65536, cut).view(torch.float32)


def _bf16_up(x):
    """The smallest bf16 number not below x >= 0 (fp32), as fp32."""
    return ((x.contiguous().view(torch.int32) + 65535) & -65536).view(torch.float32)


def _quantise(x, bits, group):
    """fp32 [..., d] -> codes [..., d], low and step [..., d / group]. The low value is rounded down and the step up,
    so that every value lies between code 0 and the last code."""
    top = float(2 ** bits - 1)
    g = x.reshape(*x.shape[:-1], -1, group)
    low = _bf16_down(g.amin(-1))
    step = _bf16_up((g.amax(-1) - low) / torch.full_like(low, top))  # a tensor: by a scalar it would be a product
    step = torch.where(step < 2.0 ** -100, 0.0, step)
    c = torch.round((g - low[..., None]) / torch.where(step > 0, step, math.inf)[..., None]).clamp(0.0, top)
    return c.reshape(x.shape), low, step


def _pack(c, bits, run):
    d = c.shape[-1]
    c = c.to(torch.uint8).reshape(*c.shape[:-1], d // 32, 32 // run, run).transpose(-3, -2).reshape(*c.shape[:-1], d)
    return c if bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)


def _unpack(codes, bits, run):
    c = codes if bits == 8 else torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    d = c.shape[-1]
    return c.reshape(*c.shape[:-1], 32 // run, d // 32, run).transpose(-3, -2).reshape(*c.shape[:-1], d)


def _values(codes, meta, bits, run):
    c = _unpack(codes, bits, run).float()
    m = meta.float()
    g = c.reshape(*c.shape[:-1], m.shape[-2], -1)
    return (m[..., 1:2] + m[..., 0:1] * g).reshape(c.shape)


def _plain_write(s):
    out = {}
    rows = slice(s["at"], s["at"] + s["t"])
    for x, name, run in ((s["k"], "k", K_RUN), (s["v"], "v", V_RUN)):
        codes, meta = s[name + "c"], s[name + "m"]
        c, low, step = _quantise(x.float(), s["bits"], s["group"])
        codes[:, rows] = _pack(c, s["bits"], run)
        meta[:, rows, :, 0], meta[:, rows, :, 1] = step, low
        g = c.reshape(*low.shape, -1)
        out[name] = (low[..., None] + step[..., None] * g).reshape(c.shape).to(x.dtype)
        out[name + "_meta"] = meta[:, rows]
    return out


def _plain_read(s):
    out = {}
    for name, run in (("k", K_RUN), ("v", V_RUN)):
        codes, meta = s[name + "c"], s[name + "m"]
        if s["rows"]:
            at = s["positions"]
            heads = torch.arange(s["hk"], device=at.device)[:, None]
            codes, meta = codes[heads, at], meta[heads, at]
        else:
            codes, meta = codes[:, : s["n"]], meta[:, : s["n"]]
        out[name] = _values(codes, meta, s["bits"], run).to(DTYPES[s["dtype"]])
    return out


def _scale(s):
    return s["d"] ** -0.5


def _plain_decode(s):
    n, t, front, window, hk, g, d = s["n"], s["t"], s["front"], s["window"], s["hk"], s["g"], s["d"]
    first = max(min(front, n), n - t + 1 - window)
    dev = s["q"].device
    pos = torch.cat((torch.arange(min(front, n), device=dev), torch.arange(first, n, device=dev)))
    pos = pos.expand(hk, g, -1)
    if s["routes"]:
        idx = s["idx"].reshape(hk, -1, s["routes"]).expand(hk, g, -1)
        pos = torch.cat((pos, idx), -1)
    if not s["per_head"]:  # the query heads of a KV head share its list
        pos = pos[:, :1]
    heads = torch.arange(hk, device=dev)[:, None, None]
    kv = [x[heads, pos] for x in (s["kc"], s["km"], s["vc"], s["vm"])]
    k = _values(kv[0], kv[1], s["bits"], K_RUN)
    v = _values(kv[2], kv[3], s["bits"], V_RUN)
    q = s["q"].float().reshape(hk, pos.shape[1], -1, d)
    last = (n - t + torch.arange(t, device=dev)).repeat(q.shape[2] // t)[:, None]  # position of each row's token
    p = pos[:, :, None, :]
    seen = (p <= last) & ((p < front) | (p > last - window) | (s["routes"] > 0))
    x = torch.matmul(q, k.transpose(-1, -2)) * _scale(s)
    x = torch.where(seen, x, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    out = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    return out.reshape(s["q"].shape).to(s["q"].dtype)


def _plain_probs(s):
    n, hk, g, d = s["n"], s["hk"], s["g"], s["d"]
    k = _values(s["kc"][:, :n], s["km"][:, :n], s["bits"], K_RUN)
    x = torch.matmul(s["q"].float().reshape(hk, g, d), k.transpose(-1, -2)) * _scale(s)
    e = torch.exp(x - x.amax(-1, keepdim=True))
    p = (e / e.sum(-1, keepdim=True)).mean(1)
    out = torch.full((hk, s["cap"]), -1.0, device=k.device)
    out[:, s["front"]: max(s["front"], n - s["window"])] = p[:, s["front"]: max(s["front"], n - s["window"])]
    return out


def run(s):
    op = s["op"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "decode": _plain_decode, "probs": _plain_probs}[op](s)
    from utmist_bigger_bird_b200 import quant_decode, quant_pooled_probs

    kv = s["kv"]
    if op == "write":
        k, v = kv.write(s["k"], s["v"], s["at"], values=True)
        rows = slice(s["at"], s["at"] + s["t"])
        return {"k": k, "v": v, "k_meta": kv.k_meta[:, rows], "v_meta": kv.v_meta[:, rows]}
    if op == "read":
        dt = DTYPES[s["dtype"]]
        k, v = kv.read(s["positions"], dtype=dt) if s["rows"] else kv.read(stop=s["n"], dtype=dt)
        return {"k": k, "v": v}
    if op == "decode":
        return quant_decode(s["q"], kv, s.get("idx"), front=s["front"], window=s["window"], scale=_scale(s), n=s["n"])
    return quant_pooled_probs(s["q"], kv, front=s["front"], window=s["window"], scale=_scale(s), n=s["n"])


# ------------------------------------------------------------------------------------------------- work
def _row_bytes(case):
    return case["d"] * case["bits"] // 8 + case["d"] // case["group"] * 4


def work(case):
    d, hk, h, row = case["d"], case["hk"], case["hk"] * case["g"], _row_bytes(case)
    if case["op"] == "write":  # rows in, their codes and the values that they stand for out
        rows = 2 * hk * case["t"]
        return {"bytes": rows * (2 * d + row + 2 * d), "flops": rows * d * 6}
    if case["op"] == "read":
        rows = 2 * hk * (case["rows"] or case["n"])
        return {"bytes": rows * (row + 2 * d) + (8 * hk * case["rows"]), "flops": rows * d * 2}
    n = case["n"]
    if case["op"] == "probs":
        return {"bytes": hk * (n * row + 4 * case["cap"]) + 2 * h * d, "flops": h * n * (2 * d + 5)}
    t, front, window = case["t"], case["front"], case["window"]
    shared = min(front, n) + n - max(min(front, n), n - t + 1 - window)
    lists = case["routes"] * (h if case["per_head"] else hk)
    pairs = sum(min(front, m) + m - max(min(front, m), m - window) + case["routes"] for m in range(n - t + 1, n + 1))
    return {"bytes": 2 * (hk * shared + lists) * row + 8 * lists + 4 * h * t * d, "flops": h * pairs * 4 * d}


# ------------------------------------------------------------------------------------------------- in 64 bits
def _exact_rows(codes, meta, d, bits, run):
    """Values of rows in float64, dimension by dimension from the definition of the format."""
    dims = torch.arange(d)
    g, r = dims // 32, dims % 32
    place = ((r // run) * (d // 32) + g) * run + r % run
    place = place.to(codes.device)
    if bits == 8:
        c = codes[..., place].double()
    else:
        byte = codes[..., place // 2].to(torch.int32)
        c = ((byte >> ((place % 2) * 4).to(torch.int32)) & 15).double()
    group = (dims // (d // meta.shape[-2])).to(codes.device)
    return meta[..., group, 1].double() + meta[..., group, 0].double() * c


def _bf16_towards(x, up):
    """float64 -> the neighbouring bf16 number (as float64) not below (up) or not above x."""
    y = x.to(torch.bfloat16).double()
    wrong = (y < x) if up else (y > x)
    m, e = torch.frexp(y)
    ulp = torch.ldexp(torch.ones_like(y), (e - 8).to(torch.int32))
    # below a power of two the spacing halves on the side towards zero
    edge = (m.abs() == 0.5) & ((y < 0) if up else (y > 0))
    ulp = torch.where(edge, ulp / 2, ulp)
    return torch.where(wrong, y + ulp if up else y - ulp, y)


def exact(case, seed):
    s = prepare(case, seed)
    d, hk, bits = case["d"], case["hk"], case["bits"]
    if case["op"] == "write":
        out, top = {}, 2 ** bits - 1
        for name in "kv":
            x = s[name].double().reshape(hk, case["t"], -1, case["group"])
            low = _bf16_towards(x.min(-1).values, False)
            step = _bf16_towards((x.max(-1).values - low) / top, True)
            code = torch.where(step[..., None] > 0, torch.round((x - low[..., None]) / step[..., None]), 0.0)
            code = code.clamp(0, top)
            out[name] = (low[..., None] + step[..., None] * code).reshape(hk, case["t"], d)
            out[name + "_meta"] = torch.stack((step, low), -1)
            del x, code
        return out
    if case["op"] == "read":
        out = {}
        for name, run in (("k", K_RUN), ("v", V_RUN)):
            heads = []
            for j in range(hk):
                rows = s["positions"][j] if case["rows"] else torch.arange(case["n"], device="cuda")
                heads.append(_exact_rows(s[name + "c"][j, rows], s[name + "m"][j, rows], d, bits, run))
            out[name] = torch.stack(heads)
        return out
    n, g, scale = case["n"], case["g"], 1.0 / math.sqrt(d)
    if case["op"] == "probs":
        out = torch.full((hk, case["cap"]), -1.0, device="cuda", dtype=torch.float64)
        for j in range(hk):
            k = _exact_rows(s["kc"][j, :n], s["km"][j, :n], d, bits, K_RUN)
            total = torch.zeros(n, device="cuda", dtype=torch.float64)
            for q in s["q"][j * g: (j + 1) * g].double():
                total += torch.softmax((k @ q) * scale, 0)
            a, b = case["front"], n - case["window"]
            if b > a:
                out[j, a:b] = total[a:b] / g
        return out
    t, front, window = case["t"], case["front"], case["window"]
    q = s["q"].double().reshape(hk * g, t, d)
    out = torch.empty_like(q)
    where = torch.arange(n, device="cuda")
    for j in range(hk):
        # the keys of this head that any of its tokens can see, once each, in float64
        any_of = (where < front) | (where > n - t - window)
        if case["routes"]:
            lists = s["idx"][j * g: (j + 1) * g] if case["per_head"] else s["idx"][j: j + 1]
            any_of[lists.flatten()] = True
        rows = where[any_of]
        k = _exact_rows(s["kc"][j, rows], s["km"][j, rows], d, bits, K_RUN)
        v = _exact_rows(s["vc"][j, rows], s["vm"][j, rows], d, bits, V_RUN)
        for a in range(g):
            head = j * g + a
            routed = torch.zeros(n, dtype=torch.bool, device="cuda")
            if case["routes"]:
                routed[s["idx"][head if case["per_head"] else j]] = True
            for i in range(t):
                here = n - t + i
                ok = (rows <= here) & ((rows < front) | (rows > here - window) | routed[rows])
                w = torch.softmax((k[ok] @ q[head, i]) * scale, 0)
                out[head, i] = w @ v[ok]
    return out.reshape(s["q"].shape)
