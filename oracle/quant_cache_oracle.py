"""Plain numpy restatement, in 64 bits, of the quantised KV cache (include/bb_b200.h, bb_qkv_*)."""
import numpy as np

K_RUN, V_RUN = 8, 4


def bf16_neighbour(x, up):
    """The bf16 number next to x (float64 array): the smallest not below it, or the largest not above it."""
    y = np.asarray(x, dtype=np.float64)
    m, e = np.frexp(y)
    scaled = m * 256.0  # 8 significant bits: |scaled| in [128, 256)
    return np.ldexp(np.ceil(scaled) if up else np.floor(scaled), e - 8)


def quantise(x, bits, group):
    """x [..., d] -> codes [..., d] (int), step and low [..., d / group] (float64 holding bf16 numbers)."""
    top = 2 ** bits - 1
    g = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, group)
    low = bf16_neighbour(g.min(-1), False)
    step = bf16_neighbour((g.max(-1) - low) / top, True)
    step = np.where(step < 2.0 ** -100, 0.0, step)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(step[..., None] > 0, np.rint((g - low[..., None]) / step[..., None]), 0.0)
    return np.clip(c, 0, top).astype(np.int64).reshape(x.shape), step, low


def values(codes, step, low):
    g = codes.reshape(*codes.shape[:-1], step.shape[-1], -1)
    return (low[..., None] + step[..., None] * g).reshape(codes.shape)


def place(d, run):
    """Place of every dimension's code in a row."""
    dim = np.arange(d)
    g, r = dim // 32, dim % 32
    return ((r // run) * (d // 32) + g) * run + r % run


def pack(codes, bits, run):
    rows = np.zeros(codes.shape, dtype=np.uint8)
    rows[..., place(codes.shape[-1], run)] = codes
    return rows if bits == 8 else rows[..., 0::2] | (rows[..., 1::2] << 4)


def unpack(rows, bits, run):
    if bits == 4:
        rows = np.stack([rows & 15, rows >> 4], -1).reshape(*rows.shape[:-1], -1)
    return rows[..., place(rows.shape[-1], run)].astype(np.int64)


def seen(n, t, i, front, window, listed):
    """Positions that token i of t attends to (listed ones last, duplicates kept)."""
    p = n - t + i
    if p < 0:
        return np.zeros(0, dtype=np.int64)
    f = min(front, p + 1)
    w0 = max(f, p + 1 - window)
    listed = np.asarray(listed, dtype=np.int64)
    return np.concatenate([np.arange(f), np.arange(w0, p + 1), listed[(listed >= front) & (listed < w0)]])


def decode(q, k, v, idx, *, front, window, scale, n, weight=None):
    """q [H, t, d], k / v [Hkv, cap, d] float64 values, idx [Hkv or H, R] or None -> (out [H, t, d], spread [H, t, d],
    reach [H, t]): the outputs; sum_j p_j weight_j with ``weight`` [Hkv, cap, d] (default |v|); the largest
    scale * sum_d |q_d| max(|k_d|) over the attended keys, both for error bounds."""
    H, t, d = q.shape
    hk = k.shape[0]
    g = H // hk
    out, spread, reach = np.zeros((H, t, d)), np.zeros((H, t, d)), np.zeros((H, t))
    w = np.abs(v) if weight is None else weight
    for h in range(H):
        kv = h // g
        row = [] if idx is None else (idx[h] if len(idx) == H and H != hk else idx[kv])
        for i in range(t):
            pos = seen(n, t, i, front, window, row)
            if not pos.size:
                continue
            s = k[kv, pos] @ q[h, i] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h, i] = p @ v[kv, pos]
            spread[h, i] = p @ w[kv, pos]
            reach[h, i] = (np.abs(k[kv, pos]) @ np.abs(q[h, i])).max() * scale
    return out, spread, reach


def pooled_probs(q, k, *, front, window, scale, n, cap):
    H, d = q.shape
    hk = k.shape[0]
    g = H // hk
    out = np.full((hk, cap), -1.0)
    a, b = front, n - window
    for kv in range(hk):
        if b <= a:
            continue
        s = q[kv * g:(kv + 1) * g] @ k[kv, :n].T * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        out[kv, a:b] = (p / p.sum(-1, keepdims=True)).mean(0)[a:b]
    return out
