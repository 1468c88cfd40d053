"""The paged-cache operators from their definitions, in 64 bits: one sequence, head and row at a time."""
import math

import torch


def rows_of(pages, block_table, b, kv, head):
    """Rows 0 .. kv - 1 of a sequence and key head, [kv, D] in fp64."""
    page = pages.shape[1]
    table = block_table[b].tolist()
    if kv == 0:
        return torch.zeros(0, pages.shape[3], dtype=torch.float64, device=pages.device)
    return torch.cat([pages[table[i], :, head] for i in range(-(-kv // page))])[:kv].double()


def attention(q, k_pages, v_pages, block_table, q_starts, kv_lens, causal, scale):
    """(out, lse, sums [B, Hkv, cap], wv, qk): wv = weights @ |v| and qk = the largest sum of
    |q_d k_d| * scale, what the tests' error bounds are made of."""
    T, Hq, D = q.shape
    Hkv = k_pages.shape[2]
    B, cap = block_table.shape[0], block_table.shape[1] * k_pages.shape[1]
    dev = q.device
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device=dev)
    wv = torch.zeros_like(out)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device=dev)
    sums = torch.zeros(B, Hkv, cap, dtype=torch.float64, device=dev)
    qk = 0.0
    starts, lens = q_starts.tolist(), kv_lens.tolist()
    for b in range(B):
        lq, kv = starts[b + 1] - starts[b], lens[b]
        if lq == 0 or kv == 0:
            continue
        at = slice(starts[b], starts[b + 1])
        i = torch.arange(lq, device=dev).unsqueeze(1)
        seen = torch.arange(kv, device=dev).unsqueeze(0) <= (kv - lq + i if causal else kv + 0 * i)
        for h in range(Hq):
            g = h // (Hq // Hkv)
            k, v = rows_of(k_pages, block_table, b, kv, g), rows_of(v_pages, block_table, b, kv, g)
            x = (q[at, h].double() @ k.t()) * scale
            qk = max(qk, float((q[at, h].double().abs() @ k.abs().t()).max()) * scale)
            x = torch.where(seen, x, torch.full_like(x, -math.inf))
            s = torch.logsumexp(x, -1)
            w = torch.where(seen, torch.exp(x - torch.where(s == -math.inf, torch.zeros_like(s), s)[:, None]),
                            torch.zeros_like(x))
            out[at, h], wv[at, h], lse[at, h] = w @ v, w @ v.abs(), s
            sums[b, g, :kv] += w.sum(0)
    return out, lse, sums, wv, qk


def rotary(x, freq, positions, rot, interleaved, gain=1.0):
    """Pairs of the first `rot` channels of x [T, H, D] turned by positions * freq, times gain; fp64."""
    y = x.double().clone()
    angle = torch.outer(positions.double(), freq.double())
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        c, s = gain * torch.cos(angle[:, i, None]), gain * torch.sin(angle[:, i, None])
        y[..., a] = x[..., a].double() * c - x[..., b].double() * s
        y[..., b] = x[..., a].double() * s + x[..., b].double() * c
    return y


def evict(sums, kv, keep, n_sink, n_recent):
    """Kept rows of one sequence and head, ascending."""
    if kv <= keep:
        return list(range(kv))
    rows = list(range(n_sink)) + list(range(kv - n_recent, kv))
    val = [(-math.inf if math.isnan(s) else s) for s in sums[:kv].tolist()]
    nan = [math.isnan(s) for s in sums[:kv].tolist()]
    rest = sorted(range(n_sink, kv - n_recent), key=lambda i: (nan[i], -val[i], i))
    return sorted(rows + rest[:keep - n_sink - n_recent])
