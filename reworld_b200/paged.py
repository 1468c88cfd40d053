"""A paged KV cache: many sessions' keys and values in pages of one pool.

The contiguous cache of one session (kv_cache.py, attention.py) has a paged form
here, for a ragged batch of sequences with shared key heads, causal order inside
the chunk of new tokens, bf16 or fp16 and head dims 64 and 128:

  rotary_table / rotary   rotary positions (1-D, any part of the head, both pair layouts)
  paged_rotary_store      new keys, rotated, and values into the sequences' pages (and rotated q)
  paged_attention         the new tokens' attention over everything the pages hold; with
                          weight_sums it adds up what weight every cached row received
  paged_evict             keeps the rows with the largest sums and moves them to fresh pages

Pools are [num_pages, page_size, Hkv, D] tensors with any strides of page, row and
head that are multiples of 8 elements (a [num_pages, Hkv, page_size, D] pool is
passed as its transposed view); page_size is a power of two >= 8.  Row r of
sequence b lies in page block_table[b, r // page_size] at row r % page_size.
q_starts [B + 1] gives the sequences' places among the packed tokens and kv_lens
[B] their cached rows, the new tokens' included; both, and the table, are int32
device tensors that are read when the kernels run, so a call needs no
synchronisation and can be captured into a CUDA graph and replayed with new values.
Values out of range are reported through _native.check_status.

The paged form of wan_5b/modules/action_model.py:265-302 (cache write and
attention), of causal_rope_apply (wan_5b/modules/causal_model.py:156-184), and of
the landmark bank's eviction (longctx/inference/landmark_cache_v2.py:465-479) by
attention weight instead of pose.
"""
import ctypes
import functools
import math

import torch

from . import _native
from ._native import RwPaged

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def _stream(device):
    """Handle of the device's current stream (what torch.cuda.current_stream(device).cuda_stream is)."""
    return torch._C._cuda_getCurrentRawStream(device)


# ------------------------------------------------------------------ arguments
# (A decoding step is a few microseconds of GPU time: the checks look at each property once.)

def _heads(t, name, dtype, dev):
    """(strides, data pointer) of a packed [T, heads, D] tensor, which the kernels read or write as it is."""
    if t.dtype != dtype or t.device != dev or t.dim() != 3:
        raise ValueError(f"{name} must be a {dtype} [T, heads, D] tensor on {dev}")
    st, ptr = t.stride(), t.data_ptr()
    if st[2] != 1 or st[0] % 8 or st[1] % 8 or ptr % 16 or st[0] <= 0 or st[1] <= 0:
        T, H, _ = t.shape
        if st[2] != 1 or (T > 1 and (st[0] % 8 or st[0] <= 0)) or (H > 1 and (st[1] % 8 or st[1] <= 0)) or ptr % 16:
            raise ValueError(f"{name}: channels must be contiguous, 16-byte aligned, other strides multiples of 8")
        # strides of a dimension of one are never used, but have to be valid
        st = (st[0] if T > 1 else 8, st[1] if H > 1 else 8, 1)
    return st, ptr


def _in(t, name, dtype, dev):
    """(tensor, strides, data pointer) of an input: one that the kernels cannot read as it is gets copied."""
    try:
        return (t, *_heads(t, name, dtype, dev))
    except ValueError:
        if t.dtype != dtype or t.device != dev or t.dim() != 3:
            raise
        t = t.clone(memory_format=torch.contiguous_format)
        return (t, *_heads(t, name, dtype, dev))


def _ints(t, name, n, dev):
    """Data pointer of a contiguous int32 vector."""
    if t.dtype != torch.int32 or t.device != dev or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous int32 [{n}] tensor on {dev}")
    return t.data_ptr()


def _table(t, name, dev):
    """(sequences, pages of each, stride, data pointer) of a block table."""
    if t.dtype != torch.int32 or t.device != dev or t.dim() != 2:
        raise ValueError(f"{name} must be an int32 [B, pages] tensor on {dev}")
    B, width = t.shape
    s0, s1 = t.stride()
    if (width > 1 and s1 != 1) or (B > 1 and s0 < width):
        raise ValueError(f"{name}: a sequence's pages must be contiguous, and rows apart")
    return B, width, s0 if B > 1 and s0 > width else width, t.data_ptr()


def _cache(k_pages, v_pages, block_table, kv_lens, q_starts=None):
    dev, dt = k_pages.device, k_pages.dtype
    if dev.type != "cuda":
        raise ValueError("a paged cache lives on a CUDA device")
    code = _DTYPES.get(dt)
    if code is None:
        raise ValueError("a paged cache is bf16 or fp16")
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype != dt or v_pages.device != dev:
        raise ValueError("k_pages and v_pages must be alike, [num_pages, page_size, Hkv, D]")
    n, page, hkv, D = shape
    if D != 128 and D != 64:
        raise NotImplementedError(f"head_dim {D}: the paged kernels have 64 and 128")
    if page < 8 or page & (page - 1):
        raise NotImplementedError(f"page_size {page}: must be a power of two >= 8")
    if n < 1 or hkv < 1:
        raise ValueError("the pools have no pages or heads")
    a, b, c, d = k_pages.stride()
    e, f, g, h = v_pages.stride()
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    if d != 1 or h != 1 or (a | b | c | e | f | g) % 8 or (kp | vp) % 16 or min(a, b, c, e, f, g) <= 0:
        raise ValueError("k_pages, v_pages: channels must be contiguous, 16-byte aligned, other strides multiples of 8")
    B, width, ts, tp = _table(block_table, "block_table", dev)
    lp = _ints(kv_lens, "kv_lens", B, dev)
    sp = _ints(q_starts, "q_starts", B + 1, dev) if q_starts is not None else None
    return RwPaged(kp, vp, a, b, c, e, f, g, n, page, hkv, D, code, B, width, 0, tp or kp, ts, sp, lp or kp)


_scratch = {}


def _workspace(dev, stream, nbytes, ncounters):
    """(workspace, counters) of a call: kept for each stream, since calls on different streams may
    overlap (every call leaves the counters zero); a captured call has its own, of its graph's memory."""
    if torch.cuda.is_current_stream_capturing():
        return (torch.empty(nbytes, dtype=torch.uint8, device=dev),
                torch.zeros(ncounters, dtype=torch.int32, device=dev))
    key = (dev.index, stream)
    kept = _scratch.get(key)
    if kept is None or kept[0].numel() < nbytes or kept[1].numel() < ncounters:
        old = (0, 0) if kept is None else (kept[0].numel(), kept[1].numel())
        kept = _scratch[key] = (torch.empty(max(nbytes, old[0]), dtype=torch.uint8, device=dev),
                                torch.zeros(max(ncounters, old[1], 1 << 14), dtype=torch.int32, device=dev))
    return kept


class _on:
    """The device of the call, where it is not the current one."""

    def __init__(self, device):
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)


# ------------------------------------------------------------------ rotary positions

def rotary_table(max_pos, rotary_dim, theta=10000.0, scaling=None, device="cuda"):
    """fp32 [max_pos, rotary_dim / 2, 2] (cos, sin) table; angles in fp64.

    scaling stretches the table for contexts longer than the model was trained on:
      None                       angle = pos * theta^(-2i / rotary_dim)
      ("linear", f)              positions divided by f (the position interpolation that
                                 build_freqs applies to its spatial sections)
      ("ntk", f)                 theta times f^(rotary_dim / (rotary_dim - 2)): the slowest pair turns f times
                                 slower, the fastest as before
      ("bands", f, trained[, slow, fast])
                                 per pair: those that turn more than `fast` (32) times in the `trained`
                                 positions stay, those that turn less than `slow` (1) times are divided by f,
                                 linear in between; cos and sin carry 0.1 ln f + 1, which sharpens
                                 the attention over the longer context
    """
    if rotary_dim < 16 or rotary_dim % 16:
        raise ValueError("rotary_dim must be a positive multiple of 16")
    if max_pos < 1:
        raise ValueError("max_pos must be positive")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    gain = 1.0
    freq = float(theta) ** (-i / rotary_dim)
    if scaling is not None:
        kind, f = scaling[0], float(scaling[1])
        if not f >= 1.0:
            raise ValueError("the scaling factor must be >= 1")
        if kind == "linear":
            freq = freq / f
        elif kind == "ntk":
            freq = (float(theta) * f ** (rotary_dim / (rotary_dim - 2))) ** (-i / rotary_dim)
        elif kind == "bands":
            trained = float(scaling[2])
            slow, fast = (float(scaling[3]), float(scaling[4])) if len(scaling) > 3 else (1.0, 32.0)
            turns = trained * freq / (2 * math.pi)
            keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
            freq = freq * keep + freq / f * (1 - keep)
            gain = 0.1 * math.log(f) + 1.0
        else:
            raise ValueError(f"unknown scaling {kind!r}")
    angle = torch.outer(torch.arange(max_pos, dtype=torch.float64), freq)
    return (torch.stack([angle.cos(), angle.sin()], dim=-1) * gain).float().to(device).contiguous()


def _table_args(table, D, device):
    if table.dtype != torch.float32 or table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous() or \
            table.device != device or table.data_ptr() % 16:
        raise ValueError(f"table must be a contiguous fp32 [max_pos, rotary_dim / 2, 2] tensor on {device}")
    rot = 2 * table.shape[1]
    if rot < 16 or rot % 16 or rot > D or table.shape[0] < 1:
        raise ValueError(f"rotary_dim {rot}: a multiple of 16 up to the head dim ({D}) is needed")
    return table.data_ptr(), table.shape[0], rot


def rotary(x, table, positions, interleaved=False, out=None):
    """Rotary positions of packed tokens x [T, heads, D] (bf16 / fp16, D 64 or 128).

    table: rotary_table(...); its rotary_dim first channels turn, the others pass.
    positions: int32 [T].  interleaved: pairs (2i, 2i + 1), else (i, i + rotary_dim / 2).
    out may be x.  One launch of rw_rotary."""
    dev, dt = x.device, x.dtype
    if dev.type != "cuda" or dt not in _DTYPES or x.dim() != 3:
        raise ValueError("rotary runs on bf16 or fp16 CUDA tensors [T, heads, D]")
    T, H, D = x.shape
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D}: the rotary kernel has 64 and 128")
    tab = _table_args(table, D, dev)
    pp = _ints(positions, "positions", T, dev)
    src, xs, xp = _in(x, "x", dt, dev)
    if out is None:
        out = torch.empty((T, H, D), dtype=dt, device=dev)
    os, op = _out(out, "out", x, (T, H, D), dt, dev)
    if T == 0 or H == 0:
        return out
    with _on(dev):
        code = _native.lib().rw_rotary(xp, op, T, H, D, _DTYPES[dt], xs[0], xs[1], os[0], os[1], *tab,
                                       int(interleaved), pp, _native.status_tensor(dev).data_ptr(), _stream(dev.index))
    _native.check(code, "rw_rotary")
    return out


def _span(t):
    """First byte of a tensor's elements, and the one behind them."""
    lo = t.data_ptr()
    return lo, lo + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _meet(a, b):
    """Whether two tensors may share bytes (two slices of the rows of one packed tensor do not)."""
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.stride() == b.stride() and a.shape[0] == b.shape[0] and a.shape[0] > 1:
        # heads [i, j) and [k, l) of the same rows
        row = a.stride(0) * a.element_size()
        wa, wb = (t.element_size() * (1 + (t.shape[1] - 1) * t.stride(1) + t.shape[2] - 1) for t in (a, b))
        lo, hi, wlo = (a0, b0, wa) if a0 < b0 else (b0, a0, wb)
        whi = wb if a0 < b0 else wa
        d = hi - lo
        return not (wlo <= d and d + whi <= row)
    return True


def _out(out, name, given, shape, dt, dev):
    """(strides, data pointer) of an output, which must be the input itself or apart from it."""
    if tuple(out.shape) != shape:
        raise ValueError(f"{name} must have the shape {list(shape)}")
    st, ptr = _heads(out, name, dt, dev)
    if given is not None and out is not given and out.numel() and \
            not (ptr == given.data_ptr() and out.stride() == given.stride() and given.shape == out.shape) and \
            _meet(out, given):
        raise ValueError(f"{name} overlaps its input without being it")
    return st, ptr


def paged_rotary_store(k, v, k_pages, v_pages, block_table, q_starts, kv_lens, table=None, positions=None, q=None,
                       q_out=None, interleaved=False):
    """Writes the new tokens' keys, rotated, and values into their sequences' pages, in one launch.

    k, v: [T, Hkv, D] of the packed new tokens; token i of sequence b (of lq) becomes row
    kv_lens[b] - lq + i.  With q [T, Hq, D], the rotated q is returned (q_out, which may be q).
    table, interleaved: as rotary(); without a table nothing is rotated.  positions: int32 [T], by
    default a token's row (an evicted cache needs them: its rows are fewer than its positions).
    Tokens behind the last sequence are not written; their rows of q_out stay as they were.
    Replaces the cache write of wan_5b/modules/action_model.py:265-292."""
    pg = _cache(k_pages, v_pages, block_table, kv_lens, q_starts)
    dev, dt = k_pages.device, k_pages.dtype
    k, ks, kp = _in(k, "k", dt, dev)
    v, vs, vp = _in(v, "v", dt, dev)
    T = k.shape[0]
    if k.shape != (T, pg.Hkv, pg.D) or v.shape != k.shape:
        raise ValueError(f"k and v must be [T, {pg.Hkv}, {pg.D}], as the pools")
    Hq, qs, qp, os, op = 0, (0, 0), None, (0, 0), None
    if q is not None:
        given = q
        q, qs, qp = _in(q, "q", dt, dev)
        Hq = q.shape[1]
        if q.shape != (T, Hq, pg.D):
            raise ValueError(f"q must be [{T}, heads, {pg.D}]")
        if q_out is None:
            q_out = torch.empty((T, Hq, pg.D), dtype=dt, device=dev)
            os, op = _heads(q_out, "q_out", dt, dev)
        else:
            os, op = _out(q_out, "q_out", given, (T, Hq, pg.D), dt, dev)
            if q_out.numel() and (_meet(q_out, k) or _meet(q_out, v)):
                raise ValueError("q_out overlaps k or v")
        if Hq == 0:
            qp = op = None
    elif q_out is not None:
        raise ValueError("q_out needs q")
    tab = _table_args(table, pg.D, dev) if table is not None else (None, 0, 0)
    pp = _ints(positions, "positions", T, dev) if positions is not None else None
    if T == 0 or pg.B == 0:
        return q_out
    with _on(dev):
        code = _native.lib().rw_paged_rotary_store(
            pg, kp, vp, qp, op, T, Hq, ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], os[0], os[1], *tab, int(interleaved),
            pp, _native.status_tensor(dev).data_ptr(), _stream(dev.index))
    _native.check(code, "rw_paged_rotary_store")
    return q_out


# ------------------------------------------------------------------ attention

def paged_attention(q, k_pages, v_pages, block_table, q_starts, kv_lens, max_q_len=None, causal=True,
                    softmax_scale=None, weight_sums=None, return_lse=False, out=None):
    """softmax(q k^T * scale) v of the packed new tokens q [T, Hq, D] over their sequences' pages.

    Query heads h of key head h // (Hq // Hkv) share its rows (Hq // Hkv <= 128).  causal: token i
    of a sequence with lq new tokens sees rows 0 .. kv_lens[b] - lq + i, else all kv_lens[b].  A row
    that sees nothing gets zeros (lse -inf).  max_q_len: the most new tokens of a sequence, by
    default T; passing it (1 for a decoding step) is what lets the call choose its kernel.
    weight_sums: fp32 [B, Hkv, cap], cap >= block_table's rows, contiguous last dim; the weight that
    every cached row received from the new tokens (all query heads of the group) is added to it.
    Returns out [T, Hq, D] in q's dtype, or (out, lse [T, Hq] fp32); rows behind the last sequence
    stay as they were in a given `out` and are undefined in a new one.
    The paged form of wan_5b/modules/attention.py:133-179."""
    pg = _cache(k_pages, v_pages, block_table, kv_lens, q_starts)
    dev, dt = k_pages.device, k_pages.dtype
    q, qs, qp = _in(q, "q", dt, dev)
    T, Hq, D = q.shape
    hkv, B, rows = pg.Hkv, pg.B, pg.table_width * pg.page_size
    if D != pg.D or Hq < 1 or Hq % hkv:
        raise ValueError(f"q must be [T, heads, {pg.D}] with a multiple of {hkv} heads")
    if Hq // hkv > 128:
        raise NotImplementedError("more than 128 query heads share a key head")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=dt, device=dev)
        os, op = (Hq * D, D), out.data_ptr()
    else:
        if tuple(out.shape) != (T, Hq, D):
            raise ValueError(f"out must be [{T}, {Hq}, {D}]")
        os, op = _heads(out, "out", dt, dev)
        if out.numel() and _meet(out, q):
            raise ValueError("out overlaps q")
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < 1e30:
        raise ValueError("softmax_scale must be positive and finite")
    longest = T if max_q_len is None else min(int(max_q_len), T)
    if longest < 0:
        raise ValueError("max_q_len must not be negative")
    wp, w0, w1 = _sums_args(weight_sums, B, hkv, rows, dev) if weight_sums is not None else (None, 0, 0)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if T > 0 and B > 0 and longest > 0:
        with _on(dev):
            need, counters = _attn_needs(dev.index, T, Hq, hkv, D, B, longest, rows, wp is not None)
            stream = _stream(dev.index)
            ws, cn = _workspace(dev, stream, need, counters)
            code = _native.lib().rw_paged_attn(
                pg, qp, op, lse.data_ptr() if return_lse else None, T, Hq, longest, qs[0], qs[1], os[0], os[1],
                int(bool(causal)), scale, wp, w0, w1, cn.data_ptr(), counters, ws.data_ptr(), need,
                _native.status_tensor(dev).data_ptr(), stream)
        _native.check(code, "rw_paged_attn")
    return (out, lse) if return_lse else out


def _sums_args(w, B, hkv, rows, dev):
    """(data pointer, strides of sequence and head) of an accumulator of weights."""
    if w.dtype != torch.float32 or w.device != dev or w.dim() != 3:
        raise ValueError(f"weight_sums must be fp32 [{B}, {hkv}, >= {rows}] on {dev}")
    n, h, cap = w.shape
    s0, s1, s2 = w.stride()
    if n != B or h != hkv or cap < rows or (cap > 1 and s2 != 1):
        raise ValueError(f"weight_sums must be fp32 [{B}, {hkv}, >= {rows}] on {dev}")
    if (h > 1 and s1 < cap) or (n > 1 and s0 < cap) or (n > 1 and h > 1 and s0 < (h - 1) * s1 + cap and
                                                      s1 < (n - 1) * s0 + cap):
        raise ValueError("weight_sums: rows overlap")
    return w.data_ptr() or None, s0, s1


@functools.lru_cache(maxsize=4096)
def _attn_needs(device, T, Hq, Hkv, D, B, longest, rows, sums):
    """Workspace bytes and counters of a call of these sizes on the current device."""
    n = ctypes.c_longlong()
    return _native.lib().rw_paged_attn_workspace_bytes(T, Hq, Hkv, D, B, longest, rows, int(sums), n), n.value


# ------------------------------------------------------------------ eviction

def paged_evict(k_pages, v_pages, block_table, kv_lens, weight_sums, keep, dst_table, n_sink=0, n_recent=0):
    """Keeps `keep` rows of every sequence and key head and moves them to dst_table's pages.

    The first n_sink and the last n_recent rows stay; of the others those with the largest
    weight_sums [B, Hkv, >= block_table's rows] (equal sums: the lower row; NaN: below everything).
    A sequence with no more than `keep` rows keeps them all.  Kept rows stay in their order and
    become rows 0, 1, ... of the pages dst_table [B, >= keep / page_size] of the same pools, which
    must not be pages of block_table; those stay as they were (they may be shared).
    Returns (kept, new_lens, new_sums): int32 [B, Hkv, keep], the kept rows, -1 behind the last;
    int32 [B]; and the kept rows' sums, zeros behind them, shaped as weight_sums (contiguous).
    New rows of an evicted sequence need explicit positions in paged_rotary_store."""
    pg = _cache(k_pages, v_pages, block_table, kv_lens)
    dev = k_pages.device
    keep, n_sink, n_recent = int(keep), int(n_sink), int(n_recent)
    if keep < 1 or n_sink < 0 or n_recent < 0 or n_sink + n_recent > keep:
        raise ValueError("keep must be positive and hold n_sink + n_recent rows")
    rows = max(pg.table_width * pg.page_size, keep)
    wp, w0, w1 = _sums_args(weight_sums, pg.B, pg.Hkv, rows, dev)
    cap = weight_sums.shape[2]
    B, width, ds, dp = _table(dst_table, "dst_table", dev)
    if B != pg.B:
        raise ValueError(f"dst_table must be an int32 [{pg.B}, pages] tensor on {dev}")
    if width * pg.page_size < keep:
        raise ValueError(f"dst_table holds {width * pg.page_size} rows, {keep} are kept")
    kept = torch.empty((B, pg.Hkv, keep), dtype=torch.int32, device=dev)
    lens = torch.empty((B,), dtype=torch.int32, device=dev)
    new = torch.empty((B, pg.Hkv, cap), dtype=torch.float32, device=dev)
    if B > 0:
        with _on(dev):
            code = _native.lib().rw_paged_evict(
                pg, wp, w0, w1, new.data_ptr(), cap, kept.data_ptr(), lens.data_ptr(), keep, n_sink, n_recent, dp, ds,
                width, _native.status_tensor(dev).data_ptr(), _stream(dev.index))
        _native.check(code, "rw_paged_evict")
    return kept, lens, new
