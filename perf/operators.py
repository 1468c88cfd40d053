"""What the paged-cache operators are measured on.

A serving program holds many sessions' keys and values in pages of one pool.  For
every step it writes the new tokens' rotated keys and their values into the
sessions' pages (paged_rotary_store), attends from the new tokens, one or a chunk
of them for each session, to everything the session's pages hold
(paged_attention), adds up the weight that each cached row received
(paged_attention with weight_sums), and, when a session has grown past its
budget, keeps the rows that received the most (paged_evict).

Every case is one of those calls:
  store    paged_rotary_store: q_out, and the pools with the new rows
  attend   paged_attention: the outputs and the log-sum-exp of every row
  weigh    paged_attention that also adds to weight_sums
  evict    paged_evict: kept rows, new lengths, compacted sums, the pools
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


def listed():
    return [
        # one decoding step of eight sessions: latency of the smallest call
        dict(name="store, 8 single tokens", op="store", batch=8, lq=1, kv=1500, spread=0.9, hq=32, hkv=8, dim=128,
             page=16, dtype="bf16", rot=128, interleaved=False, factor=1.0),
        # four streaming sessions write a chunk of three 880-token frames each, pairs interleaved, half of the head
        # rotated, positions stretched for a long context
        dict(name="store, chunks of 2640", op="store", batch=4, lq=2640, kv=36960, spread=0.0, hq=24, hkv=24, dim=128,
             page=64, dtype="bf16", rot=64, interleaved=True, factor=4.0),
        # one session, a short context: nothing but latency
        dict(name="attend, 1 token, short", op="attend", batch=1, lq=1, kv=511, spread=0.0, hq=8, hkv=2, dim=64,
             page=16, dtype="fp16"),
        # a decoding step of a full batch with ragged lengths
        dict(name="attend, 32 tokens, ragged", op="attend", batch=32, lq=1, kv=8191, spread=0.9, hq=32, hkv=8,
             dim=128, page=16, dtype="bf16"),
        # a decoding step of two sessions with very long contexts
        dict(name="attend, 2 tokens, long", op="attend", batch=2, lq=1, kv=131072, spread=0.3, hq=16, hkv=2, dim=128,
             page=64, dtype="bf16"),
        # prompts read in chunks over what is already cached, sessions at different places
        dict(name="attend, ragged chunks", op="attend", batch=4, lq=701, kv=4500, spread=0.7, hq=32, hkv=8, dim=128,
             page=16, dtype="bf16"),
        # whole prompts from an empty cache, small heads in groups of three
        dict(name="attend, prompts, dim 64", op="attend", batch=3, lq=1501, kv=1501, spread=0.5, hq=12, hkv=4, dim=64,
             page=32, dtype="fp16"),
        # the streaming model's chunk (three frames of 880 tokens, 24 heads) over its 13-chunk cache
        dict(name="attend, chunk of 2640", op="attend", batch=1, lq=2640, kv=34320, spread=0.0, hq=24, hkv=24,
             dim=128, page=16, dtype="bf16"),
        # a decoding step that also keeps the rows' weights for a later eviction
        dict(name="weigh, 16 tokens, ragged", op="weigh", batch=16, lq=1, kv=4096, spread=0.6, hq=32, hkv=8, dim=128,
             page=16, dtype="bf16"),
        # one frame's chunk over five chunks of cache, weights kept
        dict(name="weigh, chunk of 880", op="weigh", batch=1, lq=880, kv=13200, spread=0.0, hq=24, hkv=24, dim=128,
             page=64, dtype="bf16"),
        # one session goes back to half of a short budget
        dict(name="evict, 1000 to 512", op="evict", batch=1, kv=1000, spread=0.0, hkv=8, dim=128, page=16,
             dtype="bf16", keep=512, sink=4, recent=128),
        # eight sessions with long contexts go back to their budget
        dict(name="evict, 32768 to 16384", op="evict", batch=8, kv=32768, spread=0.3, hkv=8, dim=128, page=64,
             dtype="bf16", keep=16384, sink=16, recent=2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "weigh", "evict"])
    case = dict(op=op, dim=rng.choice([64, 128, 128]), page=rng.choice([16, 32, 64]),
                dtype=rng.choice(["bf16", "bf16", "fp16"]), spread=round(rng.uniform(0.0, 0.9), 2))
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    if op == "evict":
        kv = _log(rng, 300, 32768)
        keep = max(64, int(kv * rng.uniform(0.2, 0.8)))
        case.update(batch=_log(rng, 1, 8), kv=kv, hkv=hkv, keep=keep, sink=rng.randint(0, 16),
                    recent=rng.randint(0, keep // 2 - 16))
        return case
    case.update(hq=hkv * group, hkv=hkv)
    if op == "store":
        case.update(batch=_log(rng, 1, 32), lq=_log(rng, 1, 1300), rot=rng.choice([32, 64, case["dim"]]),
                    interleaved=rng.choice([True, False]), factor=rng.choice([1.0, 2.0, 8.0]))
        case["kv"] = case["lq"] + _log(rng, 1, 16000)
    elif rng.random() < 0.5:
        case.update(batch=_log(rng, 1, 32), lq=1, kv=_log(rng, 100, 16000))
    else:
        case.update(batch=_log(rng, 1, 4), lq=_log(rng, 2, 1500))
        case["kv"] = case["lq"] + _log(rng, 1, 6000)
    return case


def _lens(case):
    """(new tokens, cached rows) of every session: between (1 - spread) and 1 times the case's."""
    out = []
    for b in range(case["batch"]):
        f = (0.6180339887498949 * b) % 1.0
        g = (0.7548776662466927 * b) % 1.0
        lq = max(1, int(case.get("lq", 1) * (1 - case["spread"] * g)))
        out.append((lq, max(lq, int(case["kv"] * (1 - case["spread"] * f)))))
    return out


def _inv_freq(case, dtype=torch.float64):
    """Turns of a pair for one step of the position, stretched by `factor`."""
    i = torch.arange(0, case["rot"], 2, device=DEV, dtype=dtype)
    return 10000.0 ** (-i / case["rot"]) / case["factor"]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    lens = _lens(case)
    B, hkv, dim, page = case["batch"], case["hkv"], case["dim"], case["page"]
    width = -(-max(kv for _, kv in lens) // page)               # pages of the longest session
    dst_width = -(-case["keep"] // page) if case["op"] == "evict" else 0
    pages = B * (width + dst_width) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)

    def randn(*shape, gain=1.0):
        return (gain * torch.randn(*shape, generator=g, device=DEV)).to(dt)

    s = dict(case=case, k_pages=randn(pages, page, hkv, dim), v_pages=randn(pages, page, hkv, dim),
             block_table=order[:B * width].view(B, width).contiguous(),
             kv_lens=torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV))
    if case["op"] == "evict":
        s["dst_table"] = order[B * width:B * (width + dst_width)].view(B, dst_width).contiguous()
        # a few rows hold most of the weight
        s["weight_sums"] = torch.exp(2.5 * torch.randn(B, hkv, width * page, generator=g, device=DEV))
        return s
    starts = [0]
    for lq, _ in lens:
        starts.append(starts[-1] + lq)
    T, hq = starts[-1], case["hq"]
    s["q_starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    s["max_q_len"] = max(lq for lq, _ in lens)
    s["q"] = randn(T, hq, dim, gain=1.5)
    # host lists of where each new token stands, as the scheduler of a serving program has them
    s["seq_of"] = torch.tensor([b for b, (lq, _) in enumerate(lens) for _ in range(lq)], device=DEV)
    s["row_of"] = torch.tensor([kv - lq + i for lq, kv in lens for i in range(lq)], device=DEV)
    s["chunk_row"] = torch.tensor([i for lq, _ in lens for i in range(lq)], device=DEV)
    if case["op"] == "store":
        s["k"], s["v"] = randn(T, hkv, dim), randn(T, hkv, dim)
        pos = torch.arange(width * page, device=DEV, dtype=torch.float64)
        angle = torch.outer(pos, _inv_freq(case))
        s["table"] = torch.stack([torch.cos(angle), torch.sin(angle)], dim=-1).float().contiguous()
        s["positions"] = s["row_of"].to(torch.int32)
    if case["op"] == "weigh":
        s["weight_sums"] = torch.zeros(B, hkv, width * page, device=DEV)
    return s


# ------------------------------------------------------------------ plain forms

def _pairs(x, rot, interleaved):
    """First and second member of every rotated pair."""
    return (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])


def _turn(x, c, s, rot, interleaved):
    a, b = _pairs(x, rot, interleaved)
    p, q = a * c - b * s, a * s + b * c
    turned = torch.stack([p, q], dim=-1).flatten(-2) if interleaved else torch.cat([p, q], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _plain_store(s):
    case, dt = s["case"], s["q"].dtype
    rot, inter, page = case["rot"], case["interleaved"], case["page"]
    cs = s["table"][s["positions"].long()].unsqueeze(1)
    c, sn = cs[..., 0], cs[..., 1]
    at = s["block_table"].long()[s["seq_of"], s["row_of"] // page]
    slot = s["row_of"] % page
    s["k_pages"][at, slot] = _turn(s["k"].float(), c, sn, rot, inter).to(dt)
    s["v_pages"][at, slot] = s["v"]
    return _turn(s["q"].float(), c, sn, rot, inter).to(dt), s["k_pages"], s["v_pages"]


def _plain_attend(s):
    case, dt = s["case"], s["q"].dtype
    B, hq, hkv, dim = case["batch"], case["hq"], case["hkv"], case["dim"]
    lq, cap = s["max_q_len"], s["block_table"].shape[1] * case["page"]
    rows = s["block_table"].long()
    k = s["k_pages"][rows].view(B, cap, hkv, dim).permute(0, 2, 3, 1).float()     # [B, hkv, dim, cap]
    v = s["v_pages"][rows].view(B, cap, hkv, dim).permute(0, 2, 1, 3).float()     # [B, hkv, cap, dim]
    q = torch.zeros(B, lq, hq, dim, device=DEV)
    q[s["seq_of"], s["chunk_row"]] = s["q"].float()
    q = q.view(B, lq, hkv, hq // hkv, dim).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, dim)
    last = torch.full((B, lq), -1, dtype=torch.int64, device=DEV)                 # last row that a token sees
    last[s["seq_of"], s["chunk_row"]] = s["row_of"]
    seen = torch.arange(cap, device=DEV) <= last.unsqueeze(-1)                    # [B, lq, cap]
    x = torch.matmul(q, k).mul_(1.0 / math.sqrt(dim)).view(B, hkv, hq // hkv, lq, cap)
    x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    x.div_(torch.where(total > 0, total, torch.ones_like(total)))
    o = torch.matmul(x.view(B, hkv, -1, cap), v)
    o = o.view(B, hkv, hq // hkv, lq, dim).permute(0, 3, 1, 2, 4).reshape(B, lq, hq, dim)
    lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(B, lq, hq)
    at = (s["seq_of"], s["chunk_row"])
    out = [o[at].to(dt), lse[at]]
    if case["op"] == "weigh":
        s["weight_sums"] += x.sum((2, 3))
        out.append(s["weight_sums"])
    return out


def _plain_evict(s):
    case = s["case"]
    B, hkv, page, keep = case["batch"], case["hkv"], case["page"], case["keep"]
    sums, cap = s["weight_sums"], s["weight_sums"].shape[2]
    at = torch.arange(cap, device=DEV)
    lens = s["kv_lens"].long().view(B, 1, 1)
    inf = float("inf")
    rank = torch.where((at < case["sink"]) | (at >= lens - case["recent"]), torch.full_like(sums, inf), sums)
    rank = torch.where(at < lens, rank, torch.full_like(sums, -inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    order = torch.where(torch.arange(keep, device=DEV) < lens, order, cap)        # fewer rows than the budget
    kept = torch.sort(order, dim=-1).values                                       # rows in their own order
    there = kept < cap
    kept = torch.where(there, kept, -1)
    safe = kept.clamp_min(0)
    new = torch.zeros_like(sums)
    new[..., :keep] = torch.where(there, sums.gather(-1, safe), torch.zeros((), device=DEV))
    b = torch.arange(B, device=DEV).view(B, 1, 1)
    h = torch.arange(hkv, device=DEV).view(1, hkv, 1).expand(B, hkv, keep)
    src = s["block_table"].long()[b, safe // page]
    j = torch.arange(keep, device=DEV).expand(B, hkv, keep)
    dst = s["dst_table"].long()[b, j // page]
    to, of = (dst[there], (j % page)[there], h[there]), (src[there], (safe % page)[there], h[there])
    s["k_pages"][to] = s["k_pages"][of]
    s["v_pages"][to] = s["v_pages"][of]
    return kept.to(torch.int32), s["kv_lens"].clamp_max(keep), new, s["k_pages"], s["v_pages"]


def run(s):
    op = s["case"]["op"]
    if not own:
        return (_plain_store if op == "store" else _plain_evict if op == "evict" else _plain_attend)(s)
    from reworld_b200 import paged_attention, paged_evict, paged_rotary_store
    if op == "store":
        q_out = paged_rotary_store(s["k"], s["v"], s["k_pages"], s["v_pages"], s["block_table"], s["q_starts"],
                                   s["kv_lens"], table=s["table"], positions=s["positions"], q=s["q"],
                                   interleaved=s["case"]["interleaved"])
        return q_out, s["k_pages"], s["v_pages"]
    if op == "evict":
        kept, lens, sums = paged_evict(s["k_pages"], s["v_pages"], s["block_table"], s["kv_lens"], s["weight_sums"],
                                       s["case"]["keep"], s["dst_table"], n_sink=s["case"]["sink"],
                                       n_recent=s["case"]["recent"])
        return kept, lens, sums, s["k_pages"], s["v_pages"]
    sums = s.get("weight_sums")
    out, lse = paged_attention(s["q"], s["k_pages"], s["v_pages"], s["block_table"], s["q_starts"], s["kv_lens"],
                               max_q_len=s["max_q_len"], weight_sums=sums, return_lse=True)
    return [out, lse] if sums is None else [out, lse, sums]


def work(case):
    lens = _lens(case)
    T, kv, dim, hkv = sum(q for q, _ in lens), sum(k for _, k in lens), case["dim"], case["hkv"]
    if case["op"] == "store":
        # q, k, v read and written once, the table's rows of the tokens' positions
        return {"bytes": 2 * 2 * T * (case["hq"] + 2 * hkv) * dim + 4 * T * case["rot"],
                "flops": 3 * T * (case["hq"] + hkv) * case["rot"]}
    if case["op"] == "evict":
        kept = sum(min(k, case["keep"]) for _, k in lens)
        # kept rows of k and v read and written, the sums read once and written once, the kept indices
        return {"bytes": hkv * (2 * 2 * 2 * kept * dim + 4 * kv + 8 * kept), "flops": hkv * kv}
    seen = sum(q * k - q * (q - 1) // 2 for q, k in lens)        # (token, row) pairs under the mask
    size = 2 * 2 * T * case["hq"] * dim + 2 * 2 * kv * hkv * dim + 4 * T * case["hq"]
    flops = 4 * seen * case["hq"] * dim
    if case["op"] == "weigh":
        # the sums need every row's total: the scores are needed a second time where a chunk's are too many to hold
        size += 2 * 4 * kv * hkv
        flops += 2 * seen * case["hq"] * dim if case["lq"] > 1 else seen * case["hq"]
    return {"bytes": size, "flops": flops}


# ------------------------------------------------------------------ the definitions, in 64 bits

def exact(case, seed):
    if case["op"] == "evict":
        return None                                              # moves values and computes none
    s = prepare(case, seed)
    page, hkv, group = case["page"], case["hkv"], case["hq"] // case["hkv"]
    lens = _lens(case)
    if case["op"] == "store":
        k, v = s["k_pages"].double(), s["v_pages"].double()
        rot, freq = case["rot"], _inv_freq(case)

        def rotate(x, angle):
            z = x.double().clone()
            first = list(range(0, rot, 2)) if case["interleaved"] else list(range(rot // 2))
            second = [i + (1 if case["interleaved"] else rot // 2) for i in first]
            turn = torch.complex(torch.cos(angle), torch.sin(angle)).unsqueeze(1)
            w = torch.complex(z[..., first], z[..., second]) * turn
            z[..., first], z[..., second] = w.real, w.imag
            return z

        q = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
        t = 0
        for b, (lq, kv) in enumerate(lens):
            rows = torch.arange(kv - lq, kv, device=DEV)
            angle = torch.outer(rows.double(), freq)
            q[t:t + lq] = rotate(s["q"][t:t + lq], angle)
            at = s["block_table"][b].long()[rows // page]
            k[at, rows % page] = rotate(s["k"][t:t + lq], angle)
            v[at, rows % page] = s["v"][t:t + lq].double()
            t += lq
        return q, k, v
    T = s["q"].shape[0]
    out = torch.zeros(T, case["hq"], case["dim"], dtype=torch.float64, device=DEV)
    lse = torch.full((T, case["hq"]), float("-inf"), dtype=torch.float64, device=DEV)
    sums = s["weight_sums"].double() if case["op"] == "weigh" else None
    t = 0
    for b, (lq, kv) in enumerate(lens):
        pages = s["block_table"][b, :-(-kv // page)].long()
        hidden = torch.ones(lq, kv, dtype=torch.bool, device=DEV).triu(kv - lq + 1)
        for h in range(case["hq"]):
            k = s["k_pages"][pages, :, h // group].reshape(-1, case["dim"])[:kv].double()
            v = s["v_pages"][pages, :, h // group].reshape(-1, case["dim"])[:kv].double()
            x = s["q"][t:t + lq, h].double() @ k.t() / math.sqrt(case["dim"])
            x[hidden] = float("-inf")
            lse[t:t + lq, h] = torch.logsumexp(x, -1)
            w = torch.exp(x - lse[t:t + lq, h, None])
            out[t:t + lq, h] = w @ v
            if sums is not None:
                sums[b, h // group, :kv] += w.sum(0)
        t += lq
    return [out, lse] if sums is None else [out, lse, sums]
