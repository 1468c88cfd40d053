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
import math

import torch

from . import _native
from ._native import RwPaged

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


# ------------------------------------------------------------------ arguments

def _check_heads(t, name, dtype, device):
    """A packed [T, heads, D] tensor that the kernels can read as it is."""
    if t.dim() != 3 or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a {dtype} [T, heads, D] tensor on {device}")
    if not _heads_ok(t):
        raise ValueError(f"{name}: channels must be contiguous, 16-byte aligned, other strides multiples of 8")
    return t


def _heads_ok(t):
    st = t.stride()
    return st[2] == 1 and st[0] % 8 == 0 and st[1] % 8 == 0 and t.data_ptr() % 16 == 0 and \
        (st[0] > 0 or t.shape[0] == 1) and (st[1] > 0 or t.shape[1] == 1)


def _in(t, name, dtype, device):
    """Same for an input: one that the kernels cannot read as it is gets copied."""
    if t.dim() != 3 or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be a {dtype} [T, heads, D] tensor on {device}")
    return t if _heads_ok(t) else t.contiguous().clone() if t.is_contiguous() else t.contiguous()


def _ints(t, name, shape, device):
    if t.dtype != torch.int32 or t.device != device or tuple(t.shape) != shape:
        raise ValueError(f"{name} must be an int32 {list(shape)} tensor on {device}")
    if t.dim() == 1 and t.shape[0] > 1 and t.stride(0) != 1:
        raise ValueError(f"{name} must be contiguous")
    return t


def _cache(k_pages, v_pages, block_table, kv_lens, q_starts=None):
    dev, dt = k_pages.device, k_pages.dtype
    if dev.type != "cuda":
        raise ValueError("a paged cache lives on a CUDA device")
    if dt not in _DTYPES:
        raise ValueError("a paged cache is bf16 or fp16")
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != dt or v_pages.device != dev:
        raise ValueError("k_pages and v_pages must be alike, [num_pages, page_size, Hkv, D]")
    n, page, hkv, D = k_pages.shape
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D}: the paged kernels have 64 and 128")
    if page < 8 or page & (page - 1):
        raise NotImplementedError(f"page_size {page}: must be a power of two >= 8")
    if n < 1 or hkv < 1:
        raise ValueError("the pools have no pages or heads")
    ks, vs = k_pages.stride(), v_pages.stride()
    for t, st, name in ((k_pages, ks, "k_pages"), (v_pages, vs, "v_pages")):
        if st[3] != 1 or t.data_ptr() % 16 or any(s <= 0 or s % 8 for s in st[:3]):
            raise ValueError(f"{name}: channels must be contiguous, 16-byte aligned, other strides multiples of 8")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.device != dev:
        raise ValueError(f"block_table must be an int32 [B, pages] tensor on {dev}")
    B, width = block_table.shape
    ts = _table_stride(block_table, "block_table")
    _ints(kv_lens, "kv_lens", (B,), dev)
    if q_starts is not None:
        _ints(q_starts, "q_starts", (B + 1,), dev)
    return RwPaged(k_pages.data_ptr(), v_pages.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], n, page, hkv, D,
                   _DTYPES[dt], B, width, 0, block_table.data_ptr() or k_pages.data_ptr(), ts,
                   q_starts.data_ptr() if q_starts is not None else None,
                   kv_lens.data_ptr() or k_pages.data_ptr())


def _table_stride(t, name):
    B, width = t.shape
    if width > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: a sequence's pages must be contiguous")
    if B > 1 and t.stride(0) < width:
        raise ValueError(f"{name}: rows overlap")
    return max(t.stride(0), width) if B > 1 else width


_counters = {}


def _zeroed(device, n, stream):
    """Counters that every call leaves zero: one buffer for each stream, since calls on
    different streams may overlap; a captured call gets one of its own graph's memory."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(n, dtype=torch.int32, device=device)
    key = (device.index, stream)
    t = _counters.get(key)
    if t is None or t.numel() < n:
        t = _counters[key] = torch.zeros(max(n, 1 << 14), dtype=torch.int32, device=device)
    return t


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
    if not x.is_cuda or x.dtype not in _DTYPES or x.dim() != 3:
        raise ValueError("rotary runs on bf16 or fp16 CUDA tensors [T, heads, D]")
    T, H, D = x.shape
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim {D}: the rotary kernel has 64 and 128")
    dev = x.device
    tab = _table_args(table, D, dev)
    _ints(positions, "positions", (T,), dev)
    src = _in(x, "x", x.dtype, dev)
    if out is None:
        out = torch.empty((T, H, D), dtype=x.dtype, device=dev)
    else:
        _check_out(out, "out", src, (T, H, D), x)
    if T == 0 or H == 0:
        return out
    with _on(dev):
        code = _native.lib().rw_rotary(src.data_ptr(), out.data_ptr(), T, H, D, _DTYPES[x.dtype], *_sl_sh(src),
                                       *_sl_sh(out), *tab, int(interleaved), positions.data_ptr(),
                                       _native.status_tensor(dev).data_ptr(), _native.stream_ptr(dev))
    _native.check(code, "rw_rotary")
    return out


def _sl_sh(t):
    """Strides of token and head; those of a dimension of one are never used, but must be valid."""
    T, H, D = t.shape
    return (t.stride(0) if T > 1 else H * D), (t.stride(1) if H > 1 else D)


def _span(t):
    """First and last byte of a tensor's elements."""
    lo = t.data_ptr()
    return lo, lo + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _check_out(out, name, src, shape, given):
    """An output tensor of the caller's: its form, and that it is the input itself or apart from it."""
    if tuple(out.shape) != shape:
        raise ValueError(f"{name} must have the shape {list(shape)}")
    _check_heads(out, name, src.dtype, src.device)
    for n, s in zip(out.shape, out.stride()):
        if n > 1 and s == 0:
            raise ValueError(f"{name} must not be an expanded tensor")
    if out.numel() and src is given and not (out.data_ptr() == src.data_ptr() and out.stride() == src.stride()):
        a, b = _span(out), _span(src)
        if a[0] < b[1] and b[0] < a[1] and out.untyped_storage().data_ptr() == src.untyped_storage().data_ptr() and \
                not _interleave(out, src):
            raise ValueError(f"{name} overlaps its input without being it")


def _interleave(a, b):
    """Whether two views with the same strides (slices of one packed q|k|v row, say) cannot meet."""
    if a.stride() != b.stride() or a.stride(0) <= 0 or a.shape[0] < 2:
        return False
    row = a.stride(0) * a.element_size()
    width = [t.element_size() * (1 + (t.shape[1] - 1) * t.stride(1) + t.shape[2] - 1) for t in (a, b)]
    if max(width) > row:
        return False
    d = (a.data_ptr() - b.data_ptr()) % row
    return d >= width[1] and d + width[0] <= row


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
    k, v = _in(k, "k", dt, dev), _in(v, "v", dt, dev)
    T = k.shape[0]
    if k.shape != (T, pg.Hkv, pg.D) or v.shape != k.shape:
        raise ValueError(f"k and v must be [T, {pg.Hkv}, {pg.D}], as the pools")
    Hq, qa = 0, (0, 0, 0, 0)
    if q is not None:
        given = q
        q = _in(q, "q", dt, dev)
        Hq = q.shape[1]
        if q.shape != (T, Hq, pg.D):
            raise ValueError(f"q must be [{T}, heads, {pg.D}]")
        if q_out is None:
            q_out = torch.empty((T, Hq, pg.D), dtype=dt, device=dev)
        else:
            _check_out(q_out, "q_out", q, (T, Hq, pg.D), given)
        qa = (*_sl_sh(q), *_sl_sh(q_out))
    elif q_out is not None:
        raise ValueError("q_out needs q")
    tab = _table_args(table, pg.D, dev) if table is not None else (None, 0, 0)
    if positions is not None:
        _ints(positions, "positions", (T,), dev)
    if T == 0 or pg.B == 0:
        return q_out
    with _on(dev):
        code = _native.lib().rw_paged_rotary_store(
            pg, k.data_ptr(), v.data_ptr(), q.data_ptr() if Hq else None, q_out.data_ptr() if Hq else None, T, Hq,
            *_sl_sh(k), *_sl_sh(v), *qa, *tab, int(interleaved), positions.data_ptr() if positions is not None else None,
            _native.status_tensor(dev).data_ptr(), _native.stream_ptr(dev))
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
    q = _in(q, "q", dt, dev)
    T, Hq, D = q.shape
    if D != pg.D or Hq < 1 or Hq % pg.Hkv:
        raise ValueError(f"q must be [T, heads, {pg.D}] with a multiple of {pg.Hkv} heads")
    if Hq // pg.Hkv > 128:
        raise NotImplementedError("more than 128 query heads share a key head")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=dt, device=dev)
    else:
        if tuple(out.shape) != (T, Hq, D):
            raise ValueError(f"out must be [{T}, {Hq}, {D}]")
        _check_heads(out, "out", dt, dev)
        if out.numel() and out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr():
            a, b = _span(out), _span(q)
            if a[0] < b[1] and b[0] < a[1]:
                raise ValueError("out overlaps q")
    scale = 1.0 / math.sqrt(D) if softmax_scale is None else float(softmax_scale)
    if not 0.0 < scale < 1e30:
        raise ValueError("softmax_scale must be positive and finite")
    longest = T if max_q_len is None else int(max_q_len)
    if longest < 0:
        raise ValueError("max_q_len must not be negative")
    rows = pg.table_width * pg.page_size
    sums = (None, 0, 0)
    if weight_sums is not None:
        w = weight_sums
        if w.dtype != torch.float32 or w.device != dev or w.dim() != 3 or w.shape[0] != pg.B or \
                w.shape[1] != pg.Hkv or w.shape[2] < rows or (w.shape[2] > 1 and w.stride(2) != 1):
            raise ValueError(f"weight_sums must be fp32 [{pg.B}, {pg.Hkv}, >= {rows}] on {dev}")
        if (pg.Hkv > 1 and w.stride(1) < rows) or (pg.B > 1 and w.stride(0) < rows):
            raise ValueError("weight_sums: rows overlap")
        sums = (w.data_ptr() or None, w.stride(0), w.stride(1))
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    if T > 0 and pg.B > 0 and longest > 0:
        with _on(dev):
            lib = _native.lib()
            n = ctypes.c_longlong()
            need = lib.rw_paged_attn_workspace_bytes(T, Hq, pg.Hkv, D, pg.B, longest, rows, int(sums[0] is not None),
                                                     n)
            stream = torch.cuda.current_stream(dev).cuda_stream
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            counters = _zeroed(dev, n.value, stream) if n.value else None
            code = lib.rw_paged_attn(
                pg, q.data_ptr(), out.data_ptr(), lse.data_ptr() if lse is not None else None, T, Hq, longest,
                *_sl_sh(q), *_sl_sh(out), int(bool(causal)), scale, *sums, counters.data_ptr() if n.value else None,
                n.value, ws.data_ptr(), need, _native.status_tensor(dev).data_ptr(), stream)
        _native.check(code, "rw_paged_attn")
    return (out, lse) if return_lse else out


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
    w, rows = weight_sums, pg.table_width * pg.page_size
    if w.dtype != torch.float32 or w.device != dev or w.dim() != 3 or w.shape[0] != pg.B or w.shape[1] != pg.Hkv or \
            w.shape[2] < max(rows, keep) or (w.shape[2] > 1 and w.stride(2) != 1):
        raise ValueError(f"weight_sums must be fp32 [{pg.B}, {pg.Hkv}, >= {max(rows, keep)}] on {dev}")
    if dst_table.dim() != 2 or dst_table.dtype != torch.int32 or dst_table.device != dev or \
            dst_table.shape[0] != pg.B:
        raise ValueError(f"dst_table must be an int32 [{pg.B}, pages] tensor on {dev}")
    if dst_table.shape[1] * pg.page_size < keep:
        raise ValueError(f"dst_table holds {dst_table.shape[1] * pg.page_size} rows, {keep} are kept")
    ds = _table_stride(dst_table, "dst_table")
    kept = torch.empty((pg.B, pg.Hkv, keep), dtype=torch.int32, device=dev)
    lens = torch.empty((pg.B,), dtype=torch.int32, device=dev)
    new = torch.empty((pg.B, pg.Hkv, w.shape[2]), dtype=torch.float32, device=dev)
    if pg.B > 0:
        with _on(dev):
            code = _native.lib().rw_paged_evict(
                pg, w.data_ptr(), w.stride(0), w.stride(1), new.data_ptr(), w.shape[2], kept.data_ptr(),
                lens.data_ptr(), keep, n_sink, n_recent, dst_table.data_ptr(), ds, dst_table.shape[1],
                _native.status_tensor(dev).data_ptr(), _native.stream_ptr(dev))
        _native.check(code, "rw_paged_evict")
    return kept, lens, new
