"""The paged-cache operators on the GPU against their definitions in 64 bits.

Error bounds (all relative to sums of magnitudes that the oracle gives):
  a score is a sum of D products, exact in fp32, added in fp32: off by at most ds = (D + 2) 2^-24 * sum |q_d k_d| scale;
  a weight exp(s - m) is off by ds and by the exponential's 2^-22, relative; so is the total l, whose n terms add n 2^-24;
  the weights enter the second product rounded to the 16-bit type (half a step, eps / 2 of each), the output is rounded once more.
"""
import math

import pytest
import torch

from oracle import paged as op

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _status_clean():
    from reworld_b200 import _native
    _native.check_status()


def _cache(cuda, lens, page, hkv, D, dtype, seed=0, layout="rows", spare=3, width=None, fill=None):
    """Pools in which every row that no sequence has holds NaN, and a shuffled block table."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) if width is None else width
    total = sum(need) + spare
    shape = (total, page, hkv, D) if layout == "rows" else (total, hkv, page, D)

    def pool():
        t = torch.full(shape, float("nan"), dtype=dtype, device=cuda)
        return t if layout == "rows" else t.transpose(1, 2)

    k, v = pool(), pool()
    order = torch.randperm(total, generator=g, device=cuda).tolist()
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    for b, n in enumerate(lens):
        for i in range(need[b]):
            pg = order.pop()
            table[b, i] = pg
            rows = min(page, n - i * page)
            k[pg, :rows] = torch.randn(rows, hkv, D, generator=g, device=cuda).to(dtype)
            v[pg, :rows] = torch.randn(rows, hkv, D, generator=g, device=cuda).to(dtype)
    return k, v, table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), g


def _starts(cuda, lqs):
    s = [0]
    for n in lqs:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device=cuda)


def _check(out, lse, sums, want, dtype, D, n, before=0.0):
    o, ls, sm, wv, qk = want
    half = torch.finfo(dtype).eps / 2
    ds = (D + 2) * 2.0 ** -24 * qk
    rel = 2 * (ds + 2.0 ** -22 + n * 2.0 ** -24)
    # one more half step of the smallest subnormal where fp16 weights or outputs fall below the normal range
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    tol = (half + rel) * wv + half * (o.abs() + (half + rel) * wv) + tiny * (1 + n)
    bad = (out.double() - o).abs() > tol
    assert not bad.any(), ((out.double() - o).abs() - tol).max().item()
    assert torch.isfinite(out.float()).all()
    if lse is not None:
        fin = torch.isfinite(ls)
        assert torch.equal(fin, torch.isfinite(lse)) and (lse[~fin] == -math.inf).all()
        err = (lse.double() - ls)[fin].abs()
        assert (err <= rel + 2.0 ** -22 * (1 + ls[fin].abs())).all(), err.max().item()
    if sums is not None:
        # a row's weights are taken against its rounded maximum or total: 2^-22 of their size
        top = ls[torch.isfinite(ls)].abs().max().item() if torch.isfinite(ls).any() else 0.0
        r = rel + 2.0 ** -22 * (2 + 2 * top) + n * 2.0 ** -24
        err = (sums.double() - before - sm).abs()
        assert (err <= r * sm + 2.0 ** -23 * (abs(before) + sm) + 1e-37).all(), err.max().item()


def _run(cuda, lqs, lens, hq, hkv, D, dtype, page=16, causal=True, layout="rows", max_q=None, seed=0, sums=True,
         width=None, tail=2):
    from reworld_b200 import paged_attention
    k, v, table, kv, g = _cache(cuda, lens, page, hkv, D, dtype, seed, layout, width=width)
    starts = _starts(cuda, lqs)
    T = sum(lqs) + tail
    q = (1.5 * torch.randn(T, hq, D, generator=g, device=cuda)).to(dtype)
    scale = 1 / math.sqrt(D)
    out = torch.full_like(q, 7.0)
    w = torch.full((len(lens), hkv, table.shape[1] * page + 5), 0.5, device=cuda) if sums else None
    got, lse = paged_attention(q, k, v, table, starts, kv, max_q_len=max(lqs) if max_q is None else max_q,
                               causal=causal, weight_sums=w, return_lse=True, out=out)
    torch.cuda.synchronize()
    _status_clean()
    assert got is out
    n = T - tail
    assert (out[n:] == 7.0).all()                       # behind the last sequence
    want = op.attention(q[:n], k, v, table, starts, kv, causal, scale)
    _check(out[:n], lse[:n], w[..., :-5] if sums else None, want, dtype, D, max(lens + [1]), 0.5)
    if sums:
        assert (w[..., -5:] == 0.5).all()
    if sums:
        # and without the sums
        plain = torch.full_like(q, 7.0)
        _, lse3 = paged_attention(q, k, v, table, starts, kv, max_q_len=max(lqs) if max_q is None else max_q,
                                  causal=causal, return_lse=True, out=plain)
        torch.cuda.synchronize()
        _status_clean()
        assert (plain[n:] == 7.0).all()
        _check(plain[:n], lse3[:n], None, want, dtype, D, max(lens + [1]))
    # the same call again gives the same bits
    if sums:
        w2 = torch.full_like(w, 0.5)
        again, lse2 = paged_attention(q, k, v, table, starts, kv, max_q_len=max(lqs) if max_q is None else max_q,
                                      causal=causal, weight_sums=w2, return_lse=True)
        assert torch.equal(again[:n], out[:n]) and torch.equal(lse2[:n], lse[:n]) and torch.equal(w, w2)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("hq,hkv,D", [(8, 2, 128), (4, 4, 64), (7, 1, 128), (15, 5, 64), (16, 1, 128)])
def test_single_tokens(cuda, dtype, hq, hkv, D):
    _run(cuda, [1] * 6, [1, 17, 64, 65, 777, 3000], hq, hkv, D, dtype)


@pytest.mark.parametrize("page,layout", [(8, "rows"), (32, "heads"), (64, "rows"), (128, "heads"), (256, "rows")])
def test_single_tokens_pages_and_layouts(cuda, page, layout):
    _run(cuda, [1, 1, 1], [5, 600, 257], 8, 2, 128, BF, page=page, layout=layout)


def test_single_tokens_with_empty_sequences(cuda):
    """No new token, no cached row, both; the block table wider than any sequence."""
    _run(cuda, [1, 0, 1, 0, 1], [40, 30, 0, 0, 129], 8, 2, 128, BF, width=40)


@pytest.mark.parametrize("batch", [1, 2, 150, 700])
def test_single_tokens_batches(cuda, batch):
    _run(cuda, [1] * batch, [(37 * i) % 211 + 1 for i in range(batch)], 4, 2, 64, FP, sums=batch < 200)


@pytest.mark.parametrize("lqs,hq", [([1] * 5, 128), ([2, 1, 2, 0, 2], 64)])
def test_weights_of_single_tokens_over_a_very_wide_table(cuda, lqs, hq):
    """512 MiB of scores a sequence: the batch goes in slices of two."""
    from reworld_b200 import _native
    assert _native.lib().rw_paged_attn_workspace_bytes(sum(lqs) + 2, hq, 8, 64, 5, max(lqs), 1 << 20, 1) < 1.1 * 2 ** 30
    _run(cuda, lqs, [700, 3000, 64, 90, 1], hq, 8, 64, BF, page=64, width=16384)


def _widen(table, wide):
    """Few rows over a long table are shared out among all CTAs, over a short one they are a cluster's."""
    return torch.nn.functional.pad(table, (0, 1250 - table.shape[1])) if wide else table


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lqs,lens,hq,hkv,D", [
    ([1], [575], 8, 2, 64),                              # nine tiles
    ([1], [64], 8, 8, 128),
    ([1, 1, 1, 1], [1000, 0, 37, 640], 12, 4, 128),
    ([3, 0, 2, 3, 3, 1], [511, 200, 300, 2, 65, 1], 8, 2, 128),
    ([16], [1024], 3, 3, 64),
    ([4, 2], [1100, 700], 4, 1, 128),
    ([1], [8100], 4, 4, 128),
    ([2], [16000], 2, 1, 64),
    ([1] * 40, [(97 * i) % 500 for i in range(40)], 16, 8, 128),
    ([2] * 90, [(97 * i) % 900 for i in range(90)], 8, 8, 64),
])
def test_few_rows_by_clusters_and_by_shares(cuda, wide, dtype, lqs, lens, hq, hkv, D):
    _run(cuda, lqs, lens, hq, hkv, D, dtype, width=1250 if wide else None, causal=lqs[0] != 3)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lqs,lens,hq,hkv,D", [
    ([2, 5, 16], [2, 70, 400], 8, 2, 128),               # few tokens
    ([130, 1, 257], [130, 300, 1000], 4, 2, 128),        # chunks over what is cached, one token among them
    ([65, 40, 129], [65, 40, 129], 3, 1, 64),            # prompts, groups of three
    ([64, 128, 100], [64, 256, 228], 6, 6, 128),         # whole tiles, a head of its own each
    ([50], [700], 24, 1, 64),                            # a group of 24
    ([33, 20], [33, 300], 40, 1, 128),                   # a group of 40
    ([9, 3], [300, 20], 128, 1, 64),                     # the largest group
])
def test_chunks(cuda, dtype, causal, lqs, lens, hq, hkv, D):
    _run(cuda, lqs, lens, hq, hkv, D, dtype, causal=causal)


@pytest.mark.parametrize("page,layout", [(8, "heads"), (16, "heads"), (32, "rows"), (64, "heads"), (128, "rows"),
                                         (256, "heads")])
def test_chunks_pages_and_layouts(cuda, page, layout):
    _run(cuda, [150, 31], [333, 500], 4, 2, 128, BF, page=page, layout=layout)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("lqs,lens,hq,hkv,D", [
    ([17], [1000], 1, 1, 64),
    ([64], [2000], 8, 8, 128),                           # four blocks of rows, several CTAs each
    ([40, 0, 7, 100], [600, 30, 3, 350], 6, 2, 128),
    ([33, 5], [6000, 100], 4, 2, 64),
    ([9], [130], 40, 2, 128),                            # blocks that end inside a token's heads
])
def test_chunks_by_blocks_and_by_tiles(cuda, causal, wide, lqs, lens, hq, hkv, D):
    _run(cuda, lqs, lens, hq, hkv, D, BF, causal=causal, width=1250 if wide else None)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lqs,lens,hq,hkv,D,dtype", [
    ([1501, 900, 0, 300], [1501, 900, 70, 300], 12, 4, 64, FP),    # more units than CTAs, of many lengths
    ([1300, 700, 90], [1500, 600, 2000], 16, 16, 128, BF),         # (rows that see nothing among them)
    ([300, 20, 150], [2000, 1500, 900], 32, 8, 128, BF),
    ([600], [1000], 32, 8, 128, BF),                               # of about one length
    ([150 + 20 * (i % 5) for i in range(35)], [400 + 90 * (i % 7) for i in range(35)], 6, 2, 128, FP),
])
def test_chunks_by_whole_units(cuda, causal, lqs, lens, hq, hkv, D, dtype):
    _run(cuda, lqs, lens, hq, hkv, D, dtype, causal=causal)


def test_chunks_of_many_sequences(cuda):
    _run(cuda, [(i % 3) + 3 for i in range(1100)], [(13 * i) % 90 + 5 for i in range(1100)], 4, 1, 64, BF, max_q=5)


def test_chunk_rows_that_see_nothing(cuda):
    """More new tokens than rows: the first ones see none; sequences without rows or tokens."""
    _run(cuda, [40, 10, 0, 200], [25, 0, 100, 60], 4, 2, 128, BF)
    _run(cuda, [3, 2], [1, 0], 4, 2, 64, FP)


def test_max_q_len_is_a_bound_and_may_be_left_out(cuda):
    _run(cuda, [3, 90], [60, 200], 4, 2, 128, BF, max_q=5000)
    from reworld_b200 import paged_attention
    k, v, table, kv, g = _cache(cuda, [60, 200], 16, 2, 128, BF)
    q = torch.randn(93, 4, 128, generator=g, device=cuda).to(BF)
    s = _starts(cuda, [3, 90])
    a = paged_attention(q, k, v, table, s, kv)
    b = paged_attention(q, k, v, table, s, kv, max_q_len=93)
    assert torch.equal(a, b)


@pytest.mark.parametrize("lq,wide", [(1, False), (1, True), (40, False), (40, True)])
def test_large_and_infinite_scores(cuda, lq, wide):
    """Scores far apart (one weight is 1), masked rows of the largest finite values."""
    from reworld_b200 import paged_attention
    k, v, table, kv, g = _cache(cuda, [300], 16, 2, 128, BF, 3)
    pages = table[0].tolist()
    table = _widen(table, wide)
    big = torch.finfo(BF).max
    k[pages[-1], 300 % 16:], v[pages[-1], 300 % 16:] = big, -big     # behind the last row
    q = (100 * torch.randn(lq, 4, 128, generator=g, device=cuda)).to(BF)
    s = _starts(cuda, [lq])
    out, lse = paged_attention(q, k, v, table, s, kv, max_q_len=lq, return_lse=True)
    want = op.attention(q, k, v, table, s, kv, True, 1 / math.sqrt(128))
    _check(out, lse, None, want, BF, 128, 300)
    assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("dtype,D,hq,hkv", [(BF, 128, 4, 4), (FP, 64, 6, 2), (BF, 128, 8, 1)])
@pytest.mark.parametrize("lqs,lens,wide", [([5, 3], [40, 200], False), ([5, 3], [40, 200], True), ([2, 2], [700, 1900], False),
                                           ([2, 2], [700, 1900], True), ([300, 17], [300, 900], False),
                                           ([300, 17], [300, 900], True), ([2, 260], [1500, 2000], False),
                                           ([2, 260], [1500, 2000], True)])
def test_values_of_later_tokens_that_are_not_finite(cuda, dtype, D, hq, hkv, lqs, lens, wide):
    """Infinities and NaN in a token's key and value reach that token and those behind it, no other."""
    from reworld_b200 import paged_attention
    k, v, table, kv, g = _cache(cuda, lens, 16, hkv, D, dtype, 12)
    table = _widen(table, wide)
    s = _starts(cuda, lqs)
    q = torch.randn(sum(lqs), hq, D, generator=g, device=cuda).to(dtype)
    ref, lref = paged_attention(q, k, v, table, s, kv, max_q_len=max(lqs), return_lse=True)
    inf, nan = float("inf"), float("nan")
    for b, (lq, n) in enumerate(zip(lqs, lens)):
        # the last token's value, one in the middle, and the last token's key
        for tok, ch, x in ((lq - 1, 3, nan), (lq // 2, 5, inf), (lq // 2, D - 1, -inf), (lq // 2 + 1, 5, -inf)):
            row = n - lq + min(tok, lq - 1)
            v[int(table[b, row // 16]), row % 16, :, ch] = x
        row = n - 1
        k[int(table[b, row // 16]), row % 16, 0, 1] = nan
    out, lse = paged_attention(q, k, v, table, s, kv, max_q_len=max(lqs), return_lse=True)
    torch.cuda.synchronize()
    _status_clean()
    G, t = hq // hkv, 0
    for lq in lqs:
        mid, last = lq // 2, lq - 1
        for i in range(lq):
            got, want = out[t + i].float(), ref[t + i].float().clone()
            if i >= mid:
                want[:, 5], want[:, D - 1] = inf, -inf
            if i >= min(mid + 1, last):
                want[:, 5] = nan if min(mid + 1, last) != mid else -inf
            if i >= last:
                want[:, 3] = nan
                want[:G] = nan                           # its key was NaN too
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (i, lq)
            ok = torch.isfinite(want)
            assert torch.equal(got[~ok & ~torch.isnan(want)], want[~ok & ~torch.isnan(want)])
            # the rest differs by nothing: the same sums, with zeros in the places of what was taken out...
            if i < mid:
                assert torch.equal(got, want), i
        t += lq
    # ...and the weights did not see the values at all
    rows = torch.isfinite(lse)
    assert torch.equal(lse[rows], lref[rows])


@pytest.mark.parametrize("lq", [1, 300])
@pytest.mark.parametrize("dtype,D", [(FP, 64), (FP, 128), (BF, 64)])
def test_scores_of_ten_million(cuda, dtype, D, lq):
    """Scores of 3.6e9 * scale = 2.6e7, where fp32 has steps of 2: the later keys are 7.98 (in powers of two) above the
    first tile's, just what leaves its maximum the base of their weights; 2^7.98 * 2^7 still is an fp16 weight."""
    from reworld_b200 import paged_attention
    g = torch.Generator(device=cuda).manual_seed(61)
    n, page, scale = 500, 16, 0.007203400135040283
    k = torch.zeros(32, page, 1, D, dtype=dtype, device=cuda)
    v = torch.randn(32, page, 1, D, generator=g, device=cuda).to(dtype)
    table = _widen(torch.arange(32, dtype=torch.int32, device=cuda).view(1, 32), lq > 1)   # (by tiles)
    # products and sums below are exact in fp32 (and 61440 and 60000 in their types)
    big = 60000.0 if dtype == FP else 61440.0
    k[..., 0] = big
    k.view(-1, D)[128:, 1] = 48.0
    q = torch.zeros(lq, 1, D, dtype=dtype, device=cuda)
    q[..., 0], q[..., 1] = big, 16.0
    kv = torch.tensor([n], dtype=torch.int32, device=cuda)
    out = paged_attention(q, k, v, table, _starts(cuda, [lq]), kv, max_q_len=lq, causal=False, softmax_scale=scale)
    torch.cuda.synchronize()
    _status_clean()
    if lq == 1:                                          # few rows round the scores themselves, to steps of 2
        assert torch.isfinite(out.float()).all()
        return
    x = torch.where(torch.arange(n, device=cuda) < 128, 0.0, 768.0).double() * scale
    w = torch.softmax(x, 0)
    vals = v.view(-1, D)[:n].double()
    want, wv = w @ vals, w @ vals.abs()
    # the scores' difference is exact; times the scale's fp32 power-of-two form it is off by 2^-23 of 8
    half = torch.finfo(dtype).eps / 2
    tol = half * wv * 1.01 + half * want.abs() + 2.0 ** -17 * wv
    assert ((out[:, 0].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype,D,hq,hkv,lqs,lens", [
    (BF, 128, 4, 4, [1501], [1501]),                     # a prompt: from its first tile on not every row sees all
    (FP, 64, 6, 2, [1501], [1501]),
    (BF, 128, 8, 1, [1501, 400], [1501, 900]),
    (FP, 128, 2, 2, [1501], [4000]),                     # units in parts
    (BF, 64, 1, 1, [2600], [2600]),
])
@pytest.mark.parametrize("early", [(3,), (130, 700), (3, 131, 702, 1100)])
def test_values_early_in_a_prompt_that_are_not_finite(cuda, dtype, D, hq, hkv, lqs, lens, early):
    """Infinities in the values of early tokens, with hundreds of the chunk's rows behind them: the tokens before are
    what they were bit for bit, those behind have them in the channels they are in and what they had elsewhere."""
    from reworld_b200 import paged_attention
    k, v, table, kv, g = _cache(cuda, lens, 16, hkv, D, dtype, 21)
    s = _starts(cuda, lqs)
    q = torch.randn(sum(lqs), hq, D, generator=g, device=cuda).to(dtype)
    w0, w1 = (torch.zeros(len(lens), hkv, table.shape[1] * 16, device=cuda) for _ in range(2))
    ref, lref = paged_attention(q, k, v, table, s, kv, max_q_len=max(lqs), weight_sums=w0, return_lse=True)
    want = ref.float()
    base = lens[0] - lqs[0]
    for i, tok in enumerate(early):                      # channel 5 + i, one sign each
        x = -math.inf if i & 1 else math.inf
        v[int(table[0, (base + tok) // 16]), (base + tok) % 16, :, 5 + i] = x
        want[tok:lqs[0], :, 5 + i] = x
    out, lse = paged_attention(q, k, v, table, s, kv, max_q_len=max(lqs), weight_sums=w1, return_lse=True)
    torch.cuda.synchronize()
    _status_clean()
    assert torch.equal(out.float(), want)
    assert torch.equal(lse, lref) and torch.equal(w0, w1)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("first", [0.0, 1.0])
@pytest.mark.parametrize("D,batch,lq,n", [(64, 160, 130, 60000), (128, 80, 260, 60000), (64, 600, 1, 400000),
                                          (128, 300, 1, 400000)])
def test_many_small_weights_beside_a_large_one(cuda, dtype, first, D, batch, lq, n):
    """Row 0 takes nearly everything and every other row 4.49 * 2^-24 of that, together 1.6 or 10 % of it; their values
    are 1, row 0's is 0 (what such a row usually has: the others are all that is seen) or 1.  As many sequences (of the
    same pages) as a CTA each has whole units.

    Off by at most: the output's rounding; the weights', the same relative to what the small ones give; what is cut off
    where a product is aligned with an fp32 accumulator, less than the accumulator's last place for every key (which is
    large only beside first = 1; of 64 keys a warp of the kernel for few rows sees 16, so that its accumulator has a
    quarter); and the total's additions, n / 32 of them at most, half a step of a number below 2 each."""
    from reworld_b200 import paged_attention
    page = 64
    pages = -(-n // page)
    k = torch.zeros(pages, page, 1, D, dtype=dtype, device=cuda)
    k[0, 0, 0, 0] = 1.0
    v = torch.ones_like(k)
    v[0, 0] = first
    table = torch.arange(pages, dtype=torch.int32, device=cuda).expand(batch, pages).contiguous()
    q = torch.zeros(batch * lq, 1, D, dtype=dtype, device=cuda)
    q[..., 0] = 1.0
    w = 4.49 * 2.0 ** -24
    kv = torch.full((batch,), n, dtype=torch.int32, device=cuda)
    out, lse = paged_attention(q, k, v, table, _starts(cuda, [lq] * batch), kv, max_q_len=lq, causal=False,
                               softmax_scale=-math.log(w), return_lse=True)
    torch.cuda.synchronize()
    _status_clean()
    small = (n - 1) * w
    want = (first + small) / (1 + small)
    half = torch.finfo(dtype).eps / 2
    last = 2.0 ** (math.floor(math.log2(first + small / (1 if lq > 1 else 4))) - 23)
    total = n / 32 * 2.0 ** -24
    tol = half * want + half * small + n * last + total
    assert (out.double() - want).abs().max().item() <= tol
    assert (lse.double() - math.log1p(small) + math.log(w)).abs().max().item() <= total + 2.0 ** -18


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lqs,lens,hq,hkv,D,wide", [
    ([5, 3], [40, 200], 8, 2, 128, False), ([5, 3], [40, 200], 8, 2, 128, True),       # a cluster; shares
    ([64], [500], 4, 4, 64, False), ([64], [500], 4, 4, 64, True),                     # blocks of rows; tiles
    ([300, 150], [300, 900], 6, 2, 128, False), ([400, 200], [500, 200], 4, 1, 64, False)])
def test_weights_of_rows_whose_total_is_nan(cuda, causal, lqs, lens, hq, hkv, D, wide):
    """A row with NaN in its query gives NaN to the rows that it sees and nothing to the others."""
    from reworld_b200 import paged_attention
    k, v, table, kv, g = _cache(cuda, lens, 16, hkv, D, BF, 33)
    table = _widen(table, wide)
    s = _starts(cuda, lqs)
    q = torch.randn(sum(lqs), hq, D, generator=g, device=cuda).to(BF)
    w = [torch.zeros(len(lens), hkv, table.shape[1] * 16, device=cuda) for _ in range(2)]
    paged_attention(q, k, v, table, s, kv, max_q_len=max(lqs), causal=causal, weight_sums=w[0])
    want = w[0].clone()
    G, t = hq // hkv, 0
    for b, (lq, n) in enumerate(zip(lqs, lens)):
        tok = lq // 3
        q[t + tok, G - 1, 7] = math.nan                  # of the first key head's group
        sees = n - lq + tok + 1 if causal else n
        want[b, 0, :sees] = math.nan
        t += lq
    out, lse = paged_attention(q, k, v, table, s, kv, max_q_len=max(lqs), causal=causal, weight_sums=w[1], return_lse=True)
    torch.cuda.synchronize()
    _status_clean()
    assert int(torch.isnan(lse).sum()) == len(lqs)
    assert torch.equal(torch.isnan(w[1]), torch.isnan(want))
    # the NaN row gave the others at most 1, and nothing where it sees nothing
    assert torch.equal(w[1][:, 1:], want[:, 1:])
    t = 0
    for b, (lq, n) in enumerate(zip(lqs, lens)):
        if causal:
            x, y = w[1][b, 0, n - lq + lq // 3 + 1:], w[0][b, 0, n - lq + lq // 3 + 1:]
            assert torch.equal(x, y)


def test_strided_inputs_and_output(cuda):
    from reworld_b200 import paged_attention
    k, v, table, kv, g = _cache(cuda, [100, 50], 16, 2, 128, BF, 4)
    wide = torch.randn(20, 12, 128, generator=g, device=cuda).to(BF)
    q = wide[:, 2:6]                                     # heads of a packed row
    s = _starts(cuda, [12, 8])
    odd = torch.randn(20 * 4 * 128 + 1, generator=g, device=cuda).to(BF)[1:].view(20, 4, 128)   # off by 2 bytes
    out = torch.zeros(20, 9, 128, dtype=BF, device=cuda)[:, 3:7]
    got = paged_attention(q, k, v, table[:, :], s, kv, out=out)
    assert torch.equal(got, paged_attention(q.contiguous(), k, v, table, s, kv))
    assert torch.equal(paged_attention(odd, k, v, table, s, kv), paged_attention(odd.clone(), k, v, table, s, kv))


@pytest.mark.parametrize("lq", [1, 60])
def test_pools_and_tables_as_views(cuda, lq):
    """Keys and values of a page beside one another in one tensor, a block table inside a wider one, one
    page, one head: the strides that a view has, not those that its shape suggests."""
    from reworld_b200 import paged_attention, paged_evict, paged_rotary_store
    k, v, table, kv, g = _cache(cuda, [200, 130], 16, 2, 128, BF, 13)
    both = torch.full((k.shape[0], 2, 16, 3, 160), float("nan"), dtype=BF, device=cuda)
    ks, vs = both[:, 0, :, :2, :128], both[:, 1, :, 1:, 16:144]
    ks.copy_(k)
    vs.copy_(v)
    wide = torch.full((2, table.shape[1] + 5), -7, dtype=torch.int32, device=cuda)
    wide[:, 2:2 + table.shape[1]] = table
    ts = wide[:, 2:2 + table.shape[1]]
    s = _starts(cuda, [lq, lq])
    q = torch.randn(2 * lq, 8, 128, generator=g, device=cuda).to(BF)
    w, ws = (torch.zeros(2, 2, 16 * table.shape[1], device=cuda) for _ in range(2))
    a = paged_attention(q, k, v, table, s, kv, max_q_len=lq, weight_sums=w)
    b = paged_attention(q, ks, vs, ts, s, kv, max_q_len=lq, weight_sums=ws)
    assert torch.equal(a, b) and torch.equal(w, ws)
    kn, vn = (torch.randn(2 * lq, 2, 128, generator=g, device=cuda).to(BF) for _ in range(2))
    for kk, vv, tt in ((k, v, table), (ks, vs, ts)):
        paged_rotary_store(kn, vn, kk, vv, tt, s, kv)
    free = [i for i in range(k.shape[0]) if i not in set(table.flatten().tolist())][:2]
    dst = torch.tensor(free, dtype=torch.int32, device=cuda).view(2, 1)
    for kk, vv, tt in ((k, v, table), (ks, vs, ts)):
        paged_evict(kk, vv, tt, kv, w, 10, dst)
    assert torch.equal(torch.nan_to_num(k, 5.0), torch.nan_to_num(ks, 5.0))
    assert torch.equal(torch.nan_to_num(v, 5.0), torch.nan_to_num(vs, 5.0))
    one = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
    n = torch.tensor([min(16, lq + 3)], dtype=torch.int32, device=cuda)
    lq = min(lq, 16)
    page = both[:1, 0, :, :1, :128].copy_(torch.randn(1, 16, 1, 128, generator=g, device=cuda))
    got = paged_attention(q[:lq], page, page, one, _starts(cuda, [lq]), n, max_q_len=lq)
    want = op.attention(q[:lq], page, page, one, torch.tensor([0, lq]), n, True, 1 / math.sqrt(128))
    _check(got, None, None, want, BF, 128, 16)
    _status_clean()


def test_two_threads_on_one_stream(cuda):
    """Calls of several launches from two host threads that share a stream, and its workspace."""
    import threading
    from reworld_b200 import paged_attention
    k, v, table, kv, g = _cache(cuda, [3000, 2500], 16, 2, 64, BF, 14)
    table = _widen(table, True)
    qs = [torch.randn(n, 8, 64, generator=g, device=cuda).to(BF) for n in (2, 140)]
    ss = [_starts(cuda, [1, 1]), _starts(cuda, [70, 70])]
    want = [paged_attention(q, k, v, table, s, kv, max_q_len=q.shape[0] // 2) for q, s in zip(qs, ss)]
    bad = []

    def work(i):
        for _ in range(60):
            o = paged_attention(qs[i], k, v, table, ss[i], kv, max_q_len=qs[i].shape[0] // 2)
            bad.append(not torch.equal(o, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert len(bad) == 120 and not any(bad)
    _status_clean()


def test_nothing_to_do(cuda):
    from reworld_b200 import paged_attention, paged_evict, paged_rotary_store, rotary, rotary_table
    k, v, table, kv, g = _cache(cuda, [30], 16, 2, 64, BF, 15)
    q = torch.randn(3, 4, 64, generator=g, device=cuda).to(BF)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    out = torch.full_like(q, 3.0)
    paged_attention(q, k, v, table, _starts(cuda, [3]), kv, max_q_len=0, out=out)
    paged_attention(q, k, v, table[:0], _starts(cuda, []), none, out=out)
    assert (out == 3.0).all()
    o, lse = paged_attention(q[:0], k, v, table, _starts(cuda, [0]), kv, return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    assert paged_rotary_store(q[:0, :2], q[:0, :2], k, v, table, _starts(cuda, [0]), kv, q=q[:0]).shape == (0, 4, 64)
    assert rotary(q[:0], rotary_table(8, 32, device=cuda), none).shape == (0, 4, 64)
    kept, lens, sums = paged_evict(k, v, table[:0], none, torch.zeros(0, 2, 32, device=cuda), 8,
                                   torch.zeros(0, 1, dtype=torch.int32, device=cuda))
    assert kept.shape == (0, 2, 8) and lens.shape == (0,) and sums.shape == (0, 2, 32)
    # a table without pages: every row sees nothing
    empty = torch.zeros(1, 0, dtype=torch.int32, device=cuda)
    w = torch.ones(1, 2, 4, device=cuda)
    for mq in (1, 3):
        out, lse = paged_attention(q, k, v, empty, _starts(cuda, [mq]), torch.zeros_like(kv), max_q_len=mq, weight_sums=w,
                                   return_lse=True)
        assert not out[:mq].any() and (lse[:mq] == -math.inf).all() and (w == 1).all()
    _status_clean()


def test_outputs_in_the_pools_are_refused(cuda):
    from reworld_b200 import paged_attention, paged_rotary_store
    k, v, table, kv, g = _cache(cuda, [30, 40], 16, 2, 64, BF, 16)
    s = _starts(cuda, [3, 3])
    q = torch.zeros(6, 2, 64, dtype=BF, device=cuda)
    for pool in (k, v):
        with pytest.raises(ValueError, match="pools"):
            paged_attention(q, k, v, table, s, kv, out=pool[-1, :6])
        with pytest.raises(ValueError, match="pools"):
            paged_rotary_store(q, q, k, v, table, s, kv, q=q, q_out=pool[0, :6])
        with pytest.raises(ValueError, match="pools"):
            paged_rotary_store(q, q, k, v, table, s, kv, q=pool[0, :6], q_out=pool[0, :6])
    # beside the pools in one tensor is well
    page = k[0].numel()
    arena = torch.zeros(2 * k.numel() + 2 * page, dtype=BF, device=cuda)
    ka, va = arena[page:page + k.numel()].view_as(k), arena[page + k.numel():-page].view_as(k)
    ka.copy_(k)
    va.copy_(v)
    for out in (arena[:6 * 128].view(6, 2, 64), arena[-6 * 128:].view(6, 2, 64)):
        paged_attention(q, ka, va, table, s, kv, out=out)
        assert torch.equal(out, paged_attention(q, k, v, table, s, kv))
    _status_clean()


def test_refusals_on_device_tensors(cuda):
    from reworld_b200 import paged_attention, paged_evict, paged_rotary_store, rotary, rotary_table
    k, v, table, kv, g = _cache(cuda, [30, 40], 16, 2, 64, BF, 16)
    q = torch.randn(6, 4, 64, generator=g, device=cuda).to(BF)
    s = _starts(cuda, [3, 3])
    w = torch.zeros(2, 2, table.shape[1] * 16, device=cuda)

    def attend(q=q, k=k, v=v, t=table, s=s, kv=kv, **kw):
        return paged_attention(q, k, v, t, s, kv, **kw)

    for bad in (dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[0]), dict(v=v[:, :8]), dict(v=v.half()),
                dict(t=table.long()), dict(t=table[:1]), dict(s=s.long()), dict(s=s[:2]), dict(kv=kv.long()),
                dict(kv=kv.cpu()), dict(s=s.cpu()), dict(softmax_scale=0.0), dict(softmax_scale=float("nan")),
                dict(max_q_len=-1), dict(out=q), dict(out=q[:3]), dict(out=q.half()), dict(weight_sums=w[:, :1]),
                dict(weight_sums=w.half()), dict(weight_sums=w[..., :-1]), dict(weight_sums=w[:1].expand(2, 2, w.shape[2])),
                dict(out=torch.zeros(1, 4, 64, dtype=BF, device=cuda).expand(6, 4, 64)), dict(k=k[..., ::2], v=v[..., ::2]),
                dict(k=k.transpose(2, 3), v=v.transpose(2, 3))):
        with pytest.raises((ValueError, NotImplementedError)):
            attend(**bad)
    for bad in (dict(k=k[:, :12], v=v[:, :12]), dict(k=k[..., :32].contiguous(), v=v[..., :32].contiguous())):
        with pytest.raises(NotImplementedError):
            attend(**bad)
    with pytest.raises(NotImplementedError):
        attend(q=torch.zeros(6, 258, 64, dtype=BF, device=cuda))
    buf = torch.zeros(12, 4, 64, dtype=BF, device=cuda)
    tab = rotary_table(64, 32, device=cuda)
    pos = torch.zeros(6, dtype=torch.int32, device=cuda)
    for bad in (dict(out=buf[3:9]), dict(table=tab.half()), dict(table=tab[:, :5]), dict(positions=pos.long()),
                dict(positions=pos[:5]), dict(table=rotary_table(64, 128, device=cuda))):
        with pytest.raises(ValueError):
            rotary(**{**dict(x=buf[:6], table=tab, positions=pos), **bad})
    kn = torch.zeros(6, 2, 64, dtype=BF, device=cuda)
    for bad in (dict(k=kn[:5]), dict(v=kn.half()), dict(q=q[:5]), dict(q_out=q), dict(q=kn, q_out=kn[:, :1]),
                dict(positions=pos[:2]), dict(q=q, q_out=torch.zeros(6, 5, 64, dtype=BF, device=cuda)),
                dict(q=torch.zeros_like(kn), q_out=kn)):
        with pytest.raises(ValueError):
            paged_rotary_store(**{**dict(k=kn, v=kn, k_pages=k, v_pages=v, block_table=table, q_starts=s, kv_lens=kv),
                                  **bad})
    dst = torch.zeros(2, 1, dtype=torch.int32, device=cuda)
    for bad in (dict(keep=0), dict(keep=17), dict(n_sink=-1), dict(n_sink=5, n_recent=6), dict(dst_table=dst[:1]),
                dict(dst_table=dst.long()), dict(weight_sums=w[:1])):
        with pytest.raises(ValueError):
            paged_evict(**{**dict(k_pages=k, v_pages=v, block_table=table, kv_lens=kv, weight_sums=w, keep=10,
                                  dst_table=dst), **bad})
    _status_clean()


@pytest.mark.parametrize("lq,hkv,layout", [(1, 2, "rows"), (40, 2, "rows"), (40, 2, "heads")])
def test_pages_behind_eight_gigabytes(cuda, lq, hkv, layout):
    """The same pages at the end of a pool whose offsets pass 32 bits, in bytes and in elements."""
    from reworld_b200 import paged_attention, paged_evict, paged_rotary_store
    page, D, n = 256, 128, 700
    k, v, table, kv, g = _cache(cuda, [n], page, hkv, D, BF, 3, layout, spare=4)
    few = k.shape[0]
    total = 2 ** 33 // (page * hkv * D * 2) + few + 5
    shape = (total, page, hkv, D) if layout == "rows" else (total, hkv, page, D)
    big = [torch.empty(shape, dtype=BF, device=cuda) for _ in range(2)]
    if layout == "heads":
        big = [t.transpose(1, 2) for t in big]
    assert (total - few) * big[0].stride(0) >= 2 ** 32
    for t, s in zip(big, (k, v)):
        t[total - few:] = s
    far = table + (total - few)
    starts = _starts(cuda, [lq])
    q, nk, nv = ((torch.randn(lq, h, D, generator=g, device=cuda)).to(BF) for h in (4 * hkv, hkv, hkv))
    got = []
    free = torch.tensor([i for i in range(few) if i not in table.flatten().tolist()][:2], dtype=torch.int32, device=cuda)
    for kp, vp, tb, at in ((k, v, table, 0), (*big, far, total - few)):
        w = torch.zeros(1, hkv, table.shape[1] * page, device=cuda)
        paged_rotary_store(nk, nv, kp, vp, tb, starts, kv)
        o = paged_attention(q, kp, vp, tb, starts, kv, max_q_len=lq, weight_sums=w)
        kept, lens, sums = paged_evict(kp, vp, tb, kv, w, 300, (free + at)[None], 4, 50)
        pages = (kp[at:at + few].clone(), vp[at:at + few].clone())
        got.append((o, w, kept, lens, sums, *pages))
    torch.cuda.synchronize()
    _status_clean()
    for a, b in zip(*got):
        assert torch.equal(torch.nan_to_num(a.float(), 77.0), torch.nan_to_num(b.float(), 77.0))


@pytest.mark.parametrize("wide", [False, True])
def test_another_stream_and_two_graphs(cuda, wide):
    """Calls on two streams at once, and two captured graphs replayed at once with new lengths."""
    from reworld_b200 import paged_attention
    lens = [3000, 4000]
    k, v, table, kv, g = _cache(cuda, lens, 16, 2, 128, BF, 5)
    table = _widen(table, wide)
    s = _starts(cuda, [1, 1])
    qs = [torch.randn(2, 8, 128, generator=g, device=cuda).to(BF) for _ in range(2)]
    ws = [torch.zeros(2, 2, table.shape[1] * 16, device=cuda) for _ in range(2)]
    ref = [paged_attention(q, k, v, table, s, kv, max_q_len=1) for q in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.zeros_like(qs[0]) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                paged_attention(qs[i], k, v, table, s, kv, max_q_len=1, out=outs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(outs, ref))
    graphs, cap = [], []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o = paged_attention(qs[i], k, v, table, s, kv, max_q_len=1, weight_sums=ws[i])
        graphs.append(gr)
        cap.append(o)
    torch.cuda.synchronize()
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(cap, ref))
    kv.copy_(torch.tensor([70, 1], dtype=torch.int32))   # other lengths, same graph
    new = [paged_attention(q, k, v, table, s, kv, max_q_len=1) for q in qs]
    for i in range(2):
        graphs[i].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(cap, new))
    _status_clean()


@pytest.mark.parametrize("wide", [False, True])
def test_bad_pages_and_lengths_are_reported_and_stay_in_bounds(cuda, wide):
    from reworld_b200 import _native, paged_attention, paged_rotary_store
    k, v, table, kv, g = _cache(cuda, [60], 16, 2, 128, BF, 6)
    table = _widen(table, wide)
    q = torch.randn(1, 4, 128, generator=g, device=cuda).to(BF)
    s = _starts(cuda, [1])
    for bad_table, bad_kv, bad_s in ((table + 100000, kv, s), (table - 100000, kv, s), (table, kv + 100000, s),
                                     (table, kv - 100000, s), (table, kv, s + 50), (table, kv, -s)):
        paged_attention(q, k, v, bad_table, bad_s, bad_kv, max_q_len=1)
        with pytest.raises(RuntimeError):
            _native.check_status(cuda)
        paged_rotary_store(q[:, :2], q[:, 2:], k.clone(), v.clone(), bad_table, bad_s, bad_kv)
        torch.cuda.synchronize()
        try:
            _native.check_status(cuda)                   # a start behind the tokens just leaves no token
        except RuntimeError:
            pass
    _status_clean()


@pytest.mark.parametrize("lq,width", [(1, 64), (1, 1250), (24, 64), (90, 64), (90, 1250)])
def test_a_captured_step_replayed_with_other_lengths(cuda, lq, width):
    """Store, attention with weights and eviction in one graph: replayed with other starts, lengths, pages and tokens it
    gives what the calls give outside a graph, while eager calls of the same stream go on in between."""
    from reworld_b200 import paged_attention, paged_evict, paged_rotary_store, rotary_table
    g = torch.Generator(device=cuda).manual_seed(41)
    B, hq, hkv, D, page, keep = 3, 8, 2, 64, 16, 100
    dw = -(-keep // page)
    pool = torch.randn(B * width + B * dw, page, hkv, D, generator=g, device=cuda).to(BF)
    tab = rotary_table(width * page, D, device=cuda)
    q, k, v = (torch.randn(B * lq, h, D, generator=g, device=cuda).to(BF) for h in (hq, hkv, hkv))
    order = torch.randperm(pool.shape[0], generator=g, device=cuda).to(torch.int32)
    table, dst = order[:B * width].view(B, width).clone(), order[B * width:].view(B, dw).clone()
    s = _starts(cuda, [lq] * B)
    kv = torch.tensor([500, 900, 101], dtype=torch.int32, device=cuda)
    kp, vp = pool.clone(), pool.flip(0).contiguous()
    w = torch.zeros(B, hkv, width * page, device=cuda)

    def step(kp, vp, w):
        qr = paged_rotary_store(k, v, kp, vp, table, s, kv, table=tab, q=q)
        out, lse = paged_attention(qr, kp, vp, table, s, kv, max_q_len=lq, weight_sums=w, return_lse=True)
        return qr, out, lse, *paged_evict(kp, vp, table, kv, w, keep, dst, n_sink=2, n_recent=9)

    step(kp.clone(), vp.clone(), w.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(kp, vp, w)
    for lens, lqs in (([500, 900, 101], [lq] * B), ([120, 1000, 777], [lq, 0, lq]), ([1024, 91, 0], [1, lq, 0]),
                      ([lq, 300, 1000], [lq] * B)):
        order = torch.randperm(pool.shape[0], generator=g, device=cuda).to(torch.int32)
        for to, of in ((table, order[:B * width].view(B, width)), (dst, order[B * width:].view(B, dw)),
                       (s, _starts(cuda, lqs)), (kv, torch.tensor(lens, dtype=torch.int32, device=cuda)),
                       (kp, pool), (vp, pool.flip(0)), (w, torch.full_like(w, 0.25)),
                       (q, torch.randn(q.shape, generator=g, device=cuda).to(BF))):
            to.copy_(of)
        k2, v2, w2 = kp.clone(), vp.clone(), w.clone()
        want = step(k2, v2, w2)
        graph.replay()
        step(pool.clone(), pool.clone(), w.clone())
        torch.cuda.synchronize()
        n = sum(lqs)
        for i, (a, b) in enumerate(zip((*got, kp, vp, w), (*want, k2, v2, w2))):
            if i < 3:                                    # (rows of no sequence are undefined)
                a, b = a[:n], b[:n]
            assert torch.equal(*_bits(a, b)), i
    _status_clean()


BAD = ["page high", "page low", "length beyond", "length negative", "start falls", "start passes", "start negative"]


def _three(cuda, lq, width, hkv=2, D=64, page=16):
    """Three sequences of lq new tokens with `width` pages each, all of them there."""
    g = torch.Generator(device=cuda).manual_seed(31)
    total = 3 * width + 6
    k, v = (torch.randn(total, page, hkv, D, generator=g, device=cuda).to(BF) for _ in range(2))
    table = torch.randperm(total, generator=g, device=cuda)[:3 * width].to(torch.int32).view(3, width).contiguous()
    kv = torch.tensor([500, 390, 450], dtype=torch.int32, device=cuda)
    return k, v, table, _starts(cuda, [lq] * 3), kv, g


def _spoil(kind, lq, table, s, kv, page=16):
    """(table, starts, lengths) with one value out of range, and what they are brought to."""
    bad, good = [table.clone(), s.clone(), kv.clone()], [table.clone(), s.clone(), kv.clone()]
    if kind.startswith("page"):
        bad[0][1] = 2 ** 31 - 1 if kind == "page high" else -1
        good[0][1] = 0
    elif kind.startswith("length"):
        bad[2][1] = 2 ** 31 - 1 if kind == "length beyond" else -5
        good[2][1] = table.shape[1] * page if kind == "length beyond" else 0
    elif kind == "start falls":
        bad[1][0], good[1][0] = 2 * lq, lq               # the first sequence ends before it starts: it has no token
    elif kind == "start passes":
        bad[1][3] = 9 * lq + 1
    else:
        bad[1][0] = -3
    return bad, good


def _bits(*tensors):
    return [t.view(torch.int16 if t.element_size() == 2 else torch.int32) for t in tensors]


@pytest.mark.parametrize("sums", [False, True])
@pytest.mark.parametrize("width", [32, 1250])
@pytest.mark.parametrize("lq", [1, 60, 300])
@pytest.mark.parametrize("kind", BAD)
def test_attention_brings_values_into_range_and_reports_them(cuda, kind, lq, width, sums):
    """Bit for bit what the call gives with the values that they are brought to, for all sequences, and a report."""
    from reworld_b200 import _native, paged_attention
    k, v, table, s, kv, g = _three(cuda, lq, width)
    q = torch.randn(3 * lq, 8, 64, generator=g, device=cuda).to(BF)
    got = []
    for t, st, n in _spoil(kind, lq, table, s, kv):
        out, w = torch.full_like(q, 7.0), torch.full((3, 2, 16 * width), 0.5, device=cuda) if sums else None
        _, lse = paged_attention(q, k, v, t, st, n, max_q_len=lq, weight_sums=w, return_lse=True, out=out)
        torch.cuda.synchronize()
        first = lq if kind == "start falls" else 0       # tokens before the first sequence have no lse
        got.append(_bits(out, lse[first:], *([w] if sums else [])))
        if len(got) == 1:
            with pytest.raises(RuntimeError):
                _native.check_status(cuda)
    _status_clean()
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("lq", [1, 60, 300])
@pytest.mark.parametrize("kind", BAD + ["idle length", "idle start"])
def test_store_brings_values_into_range_and_reports_them(cuda, kind, lq):
    from reworld_b200 import _native, paged_rotary_store
    k, v, table, s, kv, g = _three(cuda, lq, 32)
    kn, vn = (torch.randn(3 * lq, 2, 64, generator=g, device=cuda).to(BF) for _ in range(2))
    q = torch.randn(3 * lq, 4, 64, generator=g, device=cuda).to(BF)
    if kind == "idle length":                            # of a sequence without a token
        s = torch.cat([s[:1], s[:3]])
        bad, good = [table, s, kv.clone()], [table, s, kv]
        bad[2][0] = -1
    elif kind == "idle start":                           # no token's place says that the last sequence's is wrong
        s = torch.cat([s[:3], s[2:3]])
        bad, good = [table, s.clone(), kv], [table, s, kv]
        bad[1][3] = 2 * lq - 1
    else:
        bad, good = _spoil(kind, lq, table, s, kv)
        if kind.startswith("page"):                      # (rows without a page are not written)
            good = [table, s, kv]
    got = []
    for t, st, n in (bad, good):
        kp, vp, qo = k.clone(), v.clone(), torch.full_like(q, 7.0)
        paged_rotary_store(kn, vn, kp, vp, t, st, n, q=q, q_out=qo)
        torch.cuda.synchronize()
        if len(got) == 0:
            with pytest.raises(RuntimeError):
                _native.check_status(cuda)
        got.append((kp, vp, qo))
    if kind == "length negative":                        # (more new tokens than rows, here too)
        with pytest.raises(RuntimeError):
            _native.check_status(cuda)
    if kind.startswith("page"):
        for pool, old in zip(got[1][:2], (k, v)):
            pool[table[1].long()] = old[table[1].long()]
    if kind == "idle start":                             # the token at the place that the start fell to is nobody's
        row = int(kv[1]) - 1
        for pool, old in zip(got[1][:2], (k, v)):
            pool[int(table[1, row // 16]), row % 16] = old[int(table[1, row // 16]), row % 16]
        got[1][2][2 * lq - 1] = 7.0
    if kind == "start falls":                            # tokens before the first sequence
        assert (got[0][2][:lq] == 7.0).all() and (got[1][2][:lq] == 7.0).all()
    for a, b in zip(_bits(*got[0]), _bits(*got[1])):
        assert torch.equal(a, b)
    _status_clean()


@pytest.mark.parametrize("width", [32, 1250])
@pytest.mark.parametrize("kind", ["page high", "page low", "length beyond", "length negative", "new page high",
                                  "new page low"])
def test_evict_brings_values_into_range_and_reports_them(cuda, kind, width):
    from reworld_b200 import _native, paged_evict
    k, v, table, s, kv, g = _three(cuda, 1, width)
    keep = 40
    spare = [i for i in range(k.shape[0]) if i not in set(table.flatten().tolist())]
    dst = torch.tensor(spare[:6] + table[2, -3:].tolist(), dtype=torch.int32, device=cuda).view(3, 3)
    table[2, -3:] = table[2, 0]                          # (behind the last row)
    w = torch.rand(3, 2, 16 * width, generator=g, device=cuda)
    if kind.startswith("new"):
        bad, good = [table, dst.clone(), kv], [table, dst, kv]
        bad[1][1] = 2 ** 31 - 1 if kind == "new page high" else -1
    else:
        (t0, _, n0), (t1, _, n1) = _spoil(kind, 1, table, s, kv)
        bad, good = [t0, dst, n0], [t1, dst, n1]
    got = []
    for t, d, n in (bad, good):
        kp, vp = k.clone(), v.clone()
        kept, lens, sums = paged_evict(kp, vp, t, n, w, keep, d, n_sink=2, n_recent=5)
        torch.cuda.synchronize()
        got.append((kp, vp, kept, lens, sums))
        if len(got) == 1:
            with pytest.raises(RuntimeError):
                _native.check_status(cuda)
    if kind.startswith("new"):                           # rows without a page are not written
        for pool, old in zip(got[1][:2], (k, v)):
            pool[dst[1].long()] = old[dst[1].long()]
    for a, b in zip(_bits(*got[0]), _bits(*got[1])):
        assert torch.equal(a, b)
    _status_clean()


# ------------------------------------------------------------------ rotary positions and the page write

def _freq(rot, theta=10000.0):
    return theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)


def _rot_tol(y, dtype):
    """One rounding to the type; two products and a sum in fp32 of values the size of the pair, with a table off by 2^-25."""
    return torch.finfo(dtype).eps / 2 * y.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D,rot", [(128, 128), (128, 64), (128, 48), (64, 64), (64, 16)])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary(cuda, dtype, D, rot, interleaved):
    from reworld_b200 import rotary, rotary_table
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(37, 5, D, generator=g, device=cuda).to(dtype)
    pos = torch.randint(0, 100000, (37,), generator=g, device=cuda, dtype=torch.int32)
    tab = rotary_table(100000, rot, device=cuda)
    y = rotary(x, tab, pos, interleaved)
    want = op.rotary(x, _freq(rot).to(cuda), pos, rot, interleaved)
    pair = 4 * x.double().abs().max() * 2.0 ** -24
    assert ((y.double() - want).abs() <= _rot_tol(want, dtype) * 1.0001 + pair).all()
    assert torch.equal(y[..., rot:], x[..., rot:])
    z = x.clone()
    assert rotary(z, tab, pos, interleaved, out=z) is z and torch.equal(z, y)      # in place
    packed = torch.zeros(37, 11, D, dtype=dtype, device=cuda)
    packed[:, 3:8] = x
    rotary(packed[:, 3:8], tab, pos, interleaved, out=packed[:, 3:8])
    assert torch.equal(packed[:, 3:8], y) and not packed[:, :3].any() and not packed[:, 8:].any()
    _status_clean()


def test_rotary_of_a_grid(cuda):
    """A table whose row is a token of the model's 3-D grid: what causal_rope_apply makes of a chunk."""
    from oracle import rope as orope
    from reworld_b200 import rotary
    frames, h, w, start = 2, 4, 6, 5
    freqs = orope.build_freqs(128, 12 / 22, 20 / 40)
    st, sh, _ = orope.rope_split(128)
    f, y, x = (i.flatten() for i in torch.meshgrid(torch.arange(start + frames), torch.arange(h), torch.arange(w),
                                                   indexing="ij"))
    z = torch.cat([freqs[f, :st], freqs[y, st:st + sh], freqs[x, st + sh:]], dim=1)      # [tokens, 64] complex
    table = torch.view_as_real(z).float().contiguous().to(cuda)
    g = torch.Generator(device=cuda).manual_seed(51)
    q = torch.randn(frames * h * w, 3, 128, generator=g, device=cuda).to(BF)
    at = torch.arange(start * h * w, (start + frames) * h * w, dtype=torch.int32, device=cuda)
    got = rotary(q, table, at, interleaved=True).float().cpu()
    want = torch.from_numpy(orope.causal_rope_apply(q.float().cpu().numpy()[None], [(frames, h, w)], freqs, start)[0])
    # both are rounded once, from values an fp32 product apart: at most a step
    pair = 4 * q.float().abs().max().item() * 2.0 ** -24
    assert ((got - want).abs() <= torch.finfo(BF).eps * want.abs() + pair).all()
    _status_clean()


def test_rotary_position_outside_the_table(cuda):
    from reworld_b200 import _native, rotary, rotary_table
    tab = rotary_table(10, 64, device=cuda)
    x = torch.randn(2, 1, 64, device=cuda).to(BF)
    rotary(x, tab, torch.tensor([3, 10], dtype=torch.int32, device=cuda))
    with pytest.raises(RuntimeError):
        _native.check_status(cuda)
    rotary(x, tab, torch.tensor([-1, 9], dtype=torch.int32, device=cuda))
    with pytest.raises(RuntimeError):
        _native.check_status(cuda)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("lqs,lens,hq,hkv,D,page,layout", [
    ([1] * 5, [1, 16, 17, 100, 33], 8, 2, 128, 16, "rows"),
    ([1, 0, 40, 7], [9, 30, 40, 300], 6, 3, 64, 32, "heads"),
    ([700, 1500], [900, 1500], 24, 24, 128, 64, "rows"),
    ([2, 3], [20, 30], 0, 1, 128, 8, "rows"),
])
@pytest.mark.parametrize("with_positions", [True, False])
def test_store(cuda, dtype, lqs, lens, hq, hkv, D, page, layout, with_positions):
    from reworld_b200 import paged_rotary_store, rotary_table
    kp, vp, table, kv, g = _cache(cuda, lens, page, hkv, D, dtype, 7, layout)
    k0, v0 = kp.clone(), vp.clone()
    T = sum(lqs) + 3                                     # three tokens behind the last sequence
    k, v = (torch.randn(T, hkv, D, generator=g, device=cuda).to(dtype) for _ in range(2))
    q = torch.randn(T, hq, D, generator=g, device=cuda).to(dtype) if hq else None
    q_out = torch.full_like(q, 9.0) if hq else None
    rows = torch.tensor([n - lq + i for lq, n in zip(lqs, lens) for i in range(lq)] + [0] * 3, device=cuda)
    pos = (rows + 1000).to(torch.int32) if with_positions else None
    tab = rotary_table(4000, D, device=cuda)
    got = paged_rotary_store(k, v, kp, vp, table, _starts(cuda, lqs), kv, table=tab, positions=pos, q=q, q_out=q_out)
    torch.cuda.synchronize()
    _status_clean()
    n = T - 3
    at = rows + 1000 if with_positions else rows
    wk = op.rotary(k, _freq(D).to(cuda), at, D, False)[:n]
    seq = torch.tensor([b for b, lq in enumerate(lqs) for _ in range(lq)], device=cuda)
    r = rows[:n]
    pg, slot = table.long()[seq, r // page], r % page
    pair = 4 * 6.0 * 2.0 ** -24
    assert ((kp[pg, slot].double() - wk).abs() <= _rot_tol(wk, dtype) * 1.0001 + pair).all()
    assert torch.equal(vp[pg, slot], v[:n])
    k0[pg, slot], v0[pg, slot] = kp[pg, slot], vp[pg, slot]         # every other row as it was
    assert torch.equal(torch.nan_to_num(kp, 77.0), torch.nan_to_num(k0, 77.0))
    assert torch.equal(torch.nan_to_num(vp, 77.0), torch.nan_to_num(v0, 77.0))
    if hq:
        wq = op.rotary(q, _freq(D).to(cuda), at, D, False)[:n]
        assert got is q_out and (q_out[n:] == 9.0).all()
        assert ((q_out[:n].double() - wq).abs() <= _rot_tol(wq, dtype) * 1.0001 + pair).all()


def test_store_without_rotation_and_packed_projections(cuda):
    """Slices of one packed q|k|v projection, rotated in place where they are."""
    from reworld_b200 import paged_rotary_store, rotary, rotary_table
    kp, vp, table, kv, g = _cache(cuda, [50, 20], 16, 2, 64, BF, 8)
    qkv = torch.randn(15, 8, 64, generator=g, device=cuda).to(BF)
    ref = qkv.clone()
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    s = _starts(cuda, [10, 5])
    assert paged_rotary_store(k, v, kp, vp, table, s, kv) is None
    rows = torch.cat([torch.arange(40, 50), torch.arange(15, 20)]).to(cuda)
    seq = torch.tensor([0] * 10 + [1] * 5, device=cuda)
    at = (table.long()[seq, rows // 16], rows % 16)
    assert torch.equal(kp[at], k) and torch.equal(vp[at], v)
    tab = rotary_table(64, 32, device=cuda)
    paged_rotary_store(k, v, kp, vp, table, s, kv, table=tab, q=q, q_out=q, interleaved=True)
    pos = rows.to(torch.int32)
    assert torch.equal(q, rotary(ref[:, :4].contiguous(), tab, pos, True))
    assert torch.equal(kp[at], rotary(ref[:, 4:6].contiguous(), tab, pos, True)) and torch.equal(qkv[:, 4:], ref[:, 4:])
    _status_clean()


# ------------------------------------------------------------------ eviction

def _evict_case(cuda, lens, page, hkv, D, keep, sink, recent, dtype=BF, sums=None, layout="rows", seed=0):
    from reworld_b200 import paged_evict
    k, v, table, kv, g = _cache(cuda, lens, page, hkv, D, dtype, seed, layout, spare=len(lens) * -(-keep // page) + 2)
    cap = max(table.shape[1] * page, keep) + 3
    w = torch.exp(torch.randn(len(lens), hkv, cap, generator=g, device=cuda)) if sums is None else sums(cap, g)
    used = set(table.flatten().tolist()) if max(lens) else set()
    free = [i for i in range(k.shape[0]) if i not in used]
    dw = -(-keep // page)
    dst = torch.tensor(free[:len(lens) * dw], dtype=torch.int32, device=cuda).view(len(lens), dw)
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    kept, new_lens, new = paged_evict(k, v, table, kv, w, keep, dst, n_sink=sink, n_recent=recent)
    torch.cuda.synchronize()
    _status_clean()
    assert torch.equal(torch.nan_to_num(w, -1.0), torch.nan_to_num(w0, -1.0))
    for b, n in enumerate(lens):
        assert int(new_lens[b]) == min(n, keep)
        for h in range(hkv):
            want = op.evict(w0[b, h].cpu(), n, keep, sink, recent)
            m = len(want)
            assert kept[b, h].tolist() == want + [-1] * (keep - m)
            at = torch.tensor(want, dtype=torch.int64, device=cuda)
            assert torch.equal(torch.nan_to_num(new[b, h, :m], -1.0), torch.nan_to_num(w0[b, h, at], -1.0))
            assert not new[b, h, m:].any()
            j = torch.arange(m, device=cuda)
            for pool, old in ((k, k0), (v, v0)):
                src = old[table.long()[b, at // page], at % page, h]
                assert torch.equal(pool[dst.long()[b, j // page], j % page, h], src)
                pool[dst.long()[b, j // page], j % page, h] = old[dst.long()[b, j // page], j % page, h]
    assert torch.equal(torch.nan_to_num(k, 77.0), torch.nan_to_num(k0, 77.0))       # nothing else was written
    assert torch.equal(torch.nan_to_num(v, 77.0), torch.nan_to_num(v0, 77.0))


@pytest.mark.parametrize("lens,page,hkv,D,keep,sink,recent", [
    ([1000, 300, 512], 16, 2, 128, 512, 4, 100),
    ([40, 41, 39, 0, 1], 8, 3, 64, 40, 0, 0),
    ([5000, 9000], 64, 1, 128, 2049, 1, 2048),           # nothing left to choose
    ([100], 16, 2, 64, 1, 0, 0),
    ([100], 16, 2, 64, 1, 1, 0),
    ([100, 77], 32, 2, 64, 50, 0, 50),
    ([8192, 8193, 4096], 256, 2, 64, 4095, 3, 5),
    ([40000, 20000, 33, 0], 64, 1, 64, 9000, 16, 100),   # several CTAs a unit
    ([70000], 256, 2, 64, 65000, 0, 0),
    ([17000], 128, 1, 64, 500, 0, 500),
])
@pytest.mark.parametrize("layout", ["rows", "heads"])
def test_evict(cuda, lens, page, hkv, D, keep, sink, recent, layout):
    _evict_case(cuda, lens, page, hkv, D, keep, sink, recent, layout=layout)


def test_evict_keeps_over_a_million_rows(cuda):
    _evict_case(cuda, [1100000, 5], 1024, 1, 128, 1060000, 4, 1000)


@pytest.mark.parametrize("kind", ["equal", "zeros", "few values", "signs and specials", "close"])
def test_evict_ties_and_special_sums(cuda, kind):
    def sums(cap, g):
        x = torch.randn(2, 2, cap, generator=g, device=cuda)
        if kind == "equal":
            return torch.ones_like(x)
        if kind == "zeros":
            return torch.where(x > 0, 0.0, -0.0)         # one value, whatever its sign
        if kind == "few values":
            return torch.round(x)+0.0
        if kind == "close":
            return 1 + (x * 4).round() * 2.0 ** -23      # differ in the last bits only
        x[..., ::7] = float("inf")
        x[..., 1::7] = -float("inf")
        x[..., 2::7] = float("nan")
        return x
    _evict_case(cuda, [5000, 700], 16, 2, 64, 600, 2, 10, sums=sums)
    _evict_case(cuda, [30000], 64, 2, 64, 8000, 2, 10, sums=lambda cap, g: sums(cap, g)[:1])


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("D,dtype", [(128, BF), (64, FP)])
def test_sessions_prompt_decode_evict_decode(cuda, D, dtype):
    """Prompts, decoding with weights kept, eviction to fresh pages, decoding from there: the caches
    hold what a dense restatement holds, and each attention matches the oracle over those rows."""
    from reworld_b200 import paged_attention, paged_evict, paged_rotary_store, rotary_table
    g = torch.Generator(device=cuda).manual_seed(11)
    B, hq, hkv, page, width = 2, 4, 2, 16, 12
    kp, vp = (torch.full((60, page, hkv, D), float("nan"), dtype=dtype, device=cuda) for _ in range(2))
    table = torch.arange(B * width, dtype=torch.int32, device=cuda).view(B, width)
    sums = torch.zeros(B, hkv, width * page, device=cuda)
    tab = rotary_table(512, D, scaling=("linear", 2.0), device=cuda)
    pos = [0, 0]                                         # tokens that a session has had
    lens = [0, 0]
    total = torch.zeros(B, hkv, width * page, dtype=torch.float64, device=cuda)

    def step(lqs):
        T = sum(lqs)
        q, k, v = ((torch.randn(T, h, D, generator=g, device=cuda)).to(dtype) for h in (hq, hkv, hkv))
        for b in range(B):
            lens[b] += lqs[b]
        kv = torch.tensor(lens, dtype=torch.int32, device=cuda)
        s = _starts(cuda, lqs)
        at = torch.tensor([pos[b] + i for b in range(B) for i in range(lqs[b])], dtype=torch.int32, device=cuda)
        qr = paged_rotary_store(k, v, kp, vp, table, s, kv, table=tab, positions=at, q=q)
        out, lse = paged_attention(qr, kp, vp, table, s, kv, max_q_len=max(lqs), weight_sums=sums, return_lse=True)
        for b in range(B):
            pos[b] += lqs[b]
        want = op.attention(qr, kp, vp, table, s, kv, True, 1 / math.sqrt(D))
        _check(out, lse, None, want, dtype, D, max(lens))
        total.add_(want[2])
        assert (sums.double() - total).abs().max() <= 1e-4 * max(1.0, float(total.max()))

    step([70, 41])
    for _ in range(3):
        step([1, 1])
    kv = torch.tensor(lens, dtype=torch.int32, device=cuda)
    dst = torch.arange(30, 30 + B * 3, dtype=torch.int32, device=cuda).view(B, 3)
    kept, new_lens, new_sums = paged_evict(kp, vp, table, kv, sums, 48, dst, n_sink=2, n_recent=8)
    assert new_lens.tolist() == [48, 44]
    for b in range(B):
        for h in range(hkv):
            assert kept[b, h].tolist() == (lambda w: w + [-1] * (48 - len(w)))(op.evict(sums[b, h].cpu(), lens[b], 48, 2, 8))
    ks = kept.clamp_min(0).long()
    total = torch.where(torch.arange(width * page, device=cuda) < new_lens.view(B, 1, 1),
                        torch.nn.functional.pad(total.gather(2, ks), (0, width * page - 48)), 0.0)
    sums.copy_(new_sums)
    table = torch.cat([dst, torch.arange(40, 40 + 4, dtype=torch.int32, device=cuda).view(B, 2)], dim=1)
    table = torch.nn.functional.pad(table, (0, width - 5))
    lens[:] = new_lens.tolist()
    for lqs in ([1, 1], [20, 1], [1, 5]):
        step(lqs)
    _status_clean()
