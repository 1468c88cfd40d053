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
import importlib.util
import math
import os
import threading

import torch

from . import _native, build


def _load_bind():
    """The module with the calls' checks (csrc/paged_bind.cpp); there is no other path."""
    path = build.bind_path()
    if not os.path.exists(path):
        raise ImportError(f"reworld_b200 is not built ({path} missing); run `python reworld_b200/build.py`")
    if build.bind_made_for() != build.bind_stamp():
        raise ImportError(f"{path} is built for {build.bind_made_for()}, this is {build.bind_stamp()}; run `python "
                          "reworld_b200/build.py`")
    spec = importlib.util.spec_from_file_location("paged_bind", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    if mod.abi_version() != _native.ABI_VERSION:
        raise ImportError(f"{path}: ABI version {mod.abi_version()} != {_native.ABI_VERSION}")
    return mod


class _Unloaded:
    """Stands for the module until the first paged call: the rest of the package needs the CUDA library alone, and is
    imported where the module is not built too."""
    _lock = threading.Lock()

    def __getattr__(self, name):
        global _bind
        with self._lock:
            if _bind is self:
                _bind = _load_bind()
        return getattr(_bind, name)


_bind = _Unloaded()


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
    if not 0.0 < float(theta) < math.inf:
        raise ValueError("theta must be positive and finite")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    gain = 1.0
    freq = float(theta) ** (-i / rotary_dim)
    if scaling is not None:
        kind = scaling[0]
        if kind not in ("linear", "ntk", "bands"):
            raise ValueError(f"unknown scaling {kind!r}")
        if len(scaling) < (3 if kind == "bands" else 2) or (kind == "bands" and len(scaling) == 4):
            raise ValueError(f"scaling {tuple(scaling)!r}: " + ("(kind, factor, trained) or (kind, factor, trained, slow, "
                             "fast)" if kind == "bands" else "(kind, factor)") + " is needed")
        f = float(scaling[1])
        if not 1.0 <= f < math.inf:
            raise ValueError("the scaling factor must be >= 1 and finite")
        if kind == "linear":
            freq = freq / f
        elif kind == "ntk":
            freq = (float(theta) * f ** (rotary_dim / (rotary_dim - 2))) ** (-i / rotary_dim)
        else:
            trained = float(scaling[2])
            slow, fast = (float(scaling[3]), float(scaling[4])) if len(scaling) > 3 else (1.0, 32.0)
            if not (0.0 < trained < math.inf and -math.inf < slow < fast < math.inf):
                raise ValueError("bands: trained must be positive and slow below fast")
            turns = trained * freq / (2 * math.pi)
            keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
            freq = freq * keep + freq / f * (1 - keep)
            gain = 0.1 * math.log(f) + 1.0
    angle = torch.outer(torch.arange(max_pos, dtype=torch.float64), freq)
    return (torch.stack([angle.cos(), angle.sin()], dim=-1) * gain).float().to(device).contiguous()


def rotary(x, table, positions, interleaved=False, out=None):
    """Rotary positions of packed tokens x [T, heads, D] (bf16 / fp16, D 64 or 128).

    table: rotary_table(...); its rotary_dim first channels turn, the others pass.
    positions: int32 [T].  interleaved: pairs (2i, 2i + 1), else (i, i + rotary_dim / 2).
    out may be x.  One launch of rw_rotary."""
    return _bind.rotary(x, table, positions, interleaved, out)


def paged_rotary_store(k, v, k_pages, v_pages, block_table, q_starts, kv_lens, table=None, positions=None, q=None,
                       q_out=None, interleaved=False):
    """Writes the new tokens' keys, rotated, and values into their sequences' pages, in one launch.

    k, v: [T, Hkv, D] of the packed new tokens; token i of sequence b (of lq) becomes row
    kv_lens[b] - lq + i.  With q [T, Hq, D], the rotated q is returned (q_out, which may be q,
    not in the pools).
    table, interleaved: as rotary(); without a table nothing is rotated.  positions: int32 [T], by
    default a token's row (an evicted cache needs them: its rows are fewer than its positions).
    Tokens of no sequence (behind the last one, before the first) are not written; their rows of q_out stay
    as they were.
    Replaces the cache write of wan_5b/modules/action_model.py:265-292."""
    return _bind.store(k, v, k_pages, v_pages, block_table, q_starts, kv_lens, table, positions, q, q_out, interleaved)


# ------------------------------------------------------------------ attention

def paged_attention(q, k_pages, v_pages, block_table, q_starts, kv_lens, max_q_len=None, causal=True,
                    softmax_scale=None, weight_sums=None, return_lse=False, out=None):
    """softmax(q k^T * scale) v of the packed new tokens q [T, Hq, D] over their sequences' pages.

    Query heads h of key head h // (Hq // Hkv) share its rows (Hq // Hkv <= 128).  causal: token i
    of a sequence with lq new tokens sees rows 0 .. kv_lens[b] - lq + i, else all kv_lens[b].  A row
    that sees nothing gets zeros (lse -inf); what a row does not see has no effect on it, infinities
    and NaN included.  max_q_len: the most new tokens of a sequence, by default T; passing it (1 for a
    decoding step) is what lets the call choose its kernel.  Statistics and accumulation are fp32; the
    weights are rounded to q's type for the product with v, the output once more.
    weight_sums: fp32 [B, Hkv, cap], cap >= block_table's rows, contiguous last dim; the weight that
    every cached row received from the new tokens (all query heads of the group) is added to it; a row
    whose total is NaN gives NaN to the rows that it sees.
    (Few tokens' weights take scratch memory for their scores by the table's width: 4 bytes for every head, token and
    row of block_table, up to 1 GiB, or one sequence's if that is more.)
    out must not lie in the pools.
    Returns out [T, Hq, D] in q's dtype, or (out, lse [T, Hq] fp32).  Rows behind the last sequence
    stay as they were in a given `out` and are undefined in a new one, as are those of a sequence
    with more than max_q_len tokens.
    The paged form of wan_5b/modules/attention.py:133-179."""
    return _bind.attention(q, k_pages, v_pages, block_table, q_starts, kv_lens, max_q_len, causal, softmax_scale,
                           weight_sums, return_lse, out)


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
    return _bind.evict(k_pages, v_pages, block_table, kv_lens, weight_sums, keep, dst_table, n_sink, n_recent)
