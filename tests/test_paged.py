"""The paged-cache entry points' refusals and host logic: nothing here reaches a GPU."""
import ctypes
import math
import os
import shutil
import subprocess
import sys

import pytest
import torch

from reworld_b200 import _native, paged

p = ctypes.c_void_p(256)


def _pg(**kw):
    a = dict(k=256, v=256, k_sp=16 * 2 * 128, k_sl=2 * 128, k_sh=128, v_sp=16 * 2 * 128, v_sl=2 * 128, v_sh=128,
             num_pages=4, page_size=16, Hkv=2, D=128, dtype=0, B=1, table_width=2, pad=0, block_table=256,
             table_stride=2, q_starts=256, kv_lens=256)
    a.update(kw)
    return _native.RwPaged(**a)


BAD_POOLS = [
    (dict(D=96), -2), (dict(D=256), -2), (dict(dtype=2), -2), (dict(page_size=12), -2), (dict(page_size=4), -2),
    (dict(k=None), -1), (dict(v=264), -1), (dict(block_table=None), -1), (dict(kv_lens=None), -1),
    (dict(num_pages=0), -1), (dict(Hkv=0), -1), (dict(B=-1), -1), (dict(table_width=-1), -1),
    (dict(table_stride=1), -1), (dict(k_sl=132), -1), (dict(v_sh=0), -1), (dict(k_sp=-64), -1),
    (dict(page_size=1 << 20, table_width=1 << 12, table_stride=1 << 12), -5),
]


@pytest.mark.parametrize("bad,code", BAD_POOLS)
def test_every_entry_point_refuses_a_bad_cache(bad, code):
    lib, pg = _native.lib(), _pg(**bad)
    assert lib.rw_paged_rotary_store(pg, p, p, None, None, 4, 0, *([128] * 8), None, 0, 0, 0, None, None, None) == code
    assert lib.rw_paged_attn(pg, p, p, None, 4, 4, 1, *([128] * 4), 1, 0.1, None, 0, 0, p, 1 << 40, None, None) == code
    assert lib.rw_paged_evict(pg, p, 64, 32, p, 64, p, p, 16, 0, 0, p, 1, 1, None, None) == code


def test_store_refusals():
    fn, pg = _native.lib().rw_paged_rotary_store, _pg()
    s8 = [256, 128] * 4
    ok = [pg, p, p, p, p, 4, 2, *s8, p, 64, 64, 0, p, None, None]

    def but(**at):
        a = list(ok)
        for i, v in at.items():
            a[int(i[1:])] = v
        return fn(*a)

    assert fn(_pg(), p, p, None, None, 0, 0, *s8, None, 0, 0, 0, None, None, None) == 0     # no tokens
    assert fn(_pg(B=0), p, p, None, None, 4, 0, *s8, None, 0, 0, 0, None, None, None) == 0  # no sequences
    assert but(_1=None) == -1 and but(_2=ctypes.c_void_p(264)) == -1
    assert but(_3=None) == -1 and but(_4=None) == -1                  # q without q_out, q_out without q
    assert but(_5=-1) == -1 and but(_6=0) == -1
    assert but(_7=100) == -1 and but(_14=0) == -1
    assert but(_17=24) == -1 and but(_17=144) == -1 and but(_17=0) == -1   # rotary dim
    assert but(_16=0) == -1 and but(_15=ctypes.c_void_p(264)) == -1       # table size, alignment
    assert fn(_pg(q_starts=None), *ok[1:]) == -1


def test_rotary_refusals():
    fn = _native.lib().rw_rotary
    s4 = [256, 128] * 2
    assert fn(p, p, 0, 2, 128, 0, *s4, p, 64, 64, 0, p, None, None) == 0
    assert fn(p, p, 4, 2, 96, 0, *s4, p, 64, 64, 0, p, None, None) == -2
    assert fn(p, p, 4, 2, 128, 3, *s4, p, 64, 64, 0, p, None, None) == -2
    assert fn(p, p, 4, 2, 128, 0, *s4, None, 64, 64, 0, p, None, None) == -1
    assert fn(p, p, 4, 2, 128, 0, *s4, p, 64, 64, 0, None, None, None) == -1
    assert fn(None, p, 4, 2, 128, 0, *s4, p, 64, 64, 0, p, None, None) == -1
    assert fn(p, p, 4, 2, 128, 0, 0, 128, 256, 128, p, 64, 64, 0, p, None, None) == -1


def test_attention_refusals():
    fn = _native.lib().rw_paged_attn
    s4 = [512, 128] * 2
    big = 1 << 40

    def call(pg=None, q=p, out=p, T=4, Hq=4, mq=1, st=s4, scale=0.1, ws=p, wb=big, sums=None, ss=(0, 0)):
        return fn(pg or _pg(), q, out, None, T, Hq, mq, *st, 1, scale, sums, *ss, ws, wb, None, None)

    assert call(T=0) == 0 and call(mq=0) == 0 and call(pg=_pg(B=0)) == 0
    assert call(q=None) == -1 and call(out=ctypes.c_void_p(8)) == -1
    assert call(T=-1) == -1 and call(Hq=3) == -1 and call(Hq=0) == -1 and call(mq=-1) == -1
    assert call(Hq=258) == -2                                    # 129 query heads on a key head
    assert call(st=[512, 100, 512, 128]) == -1
    assert call(scale=0.0) == -1 and call(scale=-1.0) == -1 and call(scale=math.nan) == -1 and call(scale=math.inf) == -1
    assert call(pg=_pg(q_starts=None)) == -1
    assert call(sums=p, ss=(-1, 0)) == -1


def test_evict_refusals():
    fn, pg = _native.lib().rw_paged_evict, _pg()
    ok = dict(sums=p, ssb=64, ssh=32, new=p, cap=32, kept=p, lens=p, keep=16, sink=2, recent=4, dst=p, dstr=1, dw=1)

    def call(**kw):
        a = dict(ok)
        a.update(kw)
        return fn(pg, a["sums"], a["ssb"], a["ssh"], a["new"], a["cap"], a["kept"], a["lens"], a["keep"], a["sink"],
                  a["recent"], a["dst"], a["dstr"], a["dw"], None, None)

    assert call(keep=0) == -1 and call(sink=-1) == -1 and call(sink=13) == -1 and call(recent=15) == -1
    assert call(sums=None) == -1 and call(new=None) == -1 and call(kept=None) == -1 and call(lens=None) == -1
    assert call(dst=None) == -1 and call(dstr=0) == -1
    assert call(keep=17) == -5 and call(cap=15) == -5            # more than dst_table's rows / new_sums' entries


def test_workspace_of_odd_questions():
    fn = _native.lib().rw_paged_attn_workspace_bytes
    for args in ((0, 8, 2, 128, 1, 1, 64, 0), (1, 8, 3, 128, 1, 1, 64, 0), (1, 8, 2, 96, 1, 1, 64, 0),
                 (1, 8, 2, 128, 0, 1, 64, 0), (1, 8, 2, 128, 1, 0, 64, 0), (1, 8, 2, 128, 1, 1, -1, 0)):
        assert fn(*args) == 0
    assert fn(1, 8, 2, 128, 1, 1, 64, 0) >= 0


def test_workspace_of_weight_sums_is_bounded():
    """Few rows' scores go by the table's width; a batch of any size takes 1 GiB, or one sequence's."""
    fn = _native.lib().rw_paged_attn_workspace_bytes
    small = fn(16, 512, 8, 128, 1, 1, 4096, 1)
    for B in (64, 256, 4000):
        for cap in (131072, 1 << 20, 1 << 22):
            one = 4 * 8 * 16 * cap
            lines = max(1, (1 << 30) // one) * 8 * 16
            got = fn(B, 128, 8, 128, B, 1, cap, 1)
            assert min(B * one, max(1 << 30, one)) - one <= got <= max(1 << 30, one) + 16 * lines + 8 * 8 * B + 1024 + small


def test_python_calls_reject_cpu_tensors():
    z = torch.zeros(1, 8, 2, 128, dtype=torch.bfloat16)
    t = torch.zeros(1, 1, dtype=torch.int32)
    n = torch.zeros(1, dtype=torch.int32)
    s = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        paged.paged_attention(q, z, z, t, s, n)
    with pytest.raises(ValueError):
        paged.paged_rotary_store(q[:, :2], q[:, :2], z, z, t, s, n)
    with pytest.raises(ValueError):
        paged.paged_evict(z, z, t, n, torch.zeros(1, 2, 8), 4, t)
    with pytest.raises(ValueError):
        paged.rotary(q, torch.zeros(4, 64, 2), n)


def test_rotary_table():
    t = paged.rotary_table(50, 32, theta=500.0, device="cpu")
    assert t.shape == (50, 16, 2) and t.dtype == torch.float32
    for pos in (0, 1, 49):
        for i in (0, 7, 15):
            a = pos * 500.0 ** (-2 * i / 32)
            # one rounding of a value of at most 1
            assert abs(float(t[pos, i, 0]) - math.cos(a)) <= 2 ** -24 and abs(float(t[pos, i, 1]) - math.sin(a)) <= 2 ** -24
    lin = paged.rotary_table(50, 32, theta=500.0, scaling=("linear", 4.0), device="cpu")
    assert torch.equal(lin[40], t[10])
    # the fastest pair turns as before, the slowest f times slower
    f = 8.0
    ntk = paged.rotary_table(50, 32, theta=500.0, scaling=("ntk", f), device="cpu")
    assert torch.equal(ntk[:, 0], t[:, 0])
    a = 40 * 500.0 ** (-30 / 32) / f
    assert abs(float(ntk[40, 15, 1]) - math.sin(a)) <= 2 ** -23
    # bands: with 64 trained positions and theta 500 pair 0 turns 10.2 times; pairs under one turn are stretched whole
    g = 0.1 * math.log(f) + 1
    b = paged.rotary_table(50, 32, theta=500.0, scaling=("bands", f, 64, 1.0, 8.0), device="cpu")
    assert abs(float(b[3, 0, 0]) - g * math.cos(3.0)) <= 2 ** -22
    assert abs(float(b[40, 15, 1]) - g * math.sin(a)) <= 2 ** -22
    for bad in (dict(rotary_dim=24), dict(rotary_dim=0), dict(max_pos=0), dict(scaling=("linear", 0.5)),
                dict(scaling=("other", 2.0))):
        with pytest.raises(ValueError):
            paged.rotary_table(**{"max_pos": 8, "rotary_dim": 32, "device": "cpu", **bad})


@pytest.mark.parametrize("kw", [
    dict(scaling=("bands", 8.0, 64, 1.0)), dict(scaling=("bands", 8.0)), dict(scaling=("linear",)),
    dict(scaling=("bands", 8.0, 64, 4.0, 4.0)), dict(scaling=("bands", 8.0, 64, 8.0, 1.0)), dict(scaling=("bands", 8.0, 0)),
    dict(scaling=("bands", 8.0, -64)), dict(scaling=("linear", math.inf)), dict(scaling=("linear", math.nan)),
    dict(theta=0.0), dict(theta=-10000.0), dict(theta=math.nan), dict(theta=math.inf)])
def test_rotary_table_refuses_what_it_has_no_angles_for(kw):
    with pytest.raises(ValueError):
        paged.rotary_table(8, 32, device="cpu", **kw)


def test_rotary_table_between_the_bands():
    """Pairs that turn between `slow` and `fast` times are stretched in part, linear in their turns."""
    f, theta, trained, slow, fast = 4.0, 1000.0, 300, 2.0, 20.0
    t = paged.rotary_table(200, 64, theta=theta, scaling=("bands", f, trained, slow, fast), device="cpu")
    g, between = 0.1 * math.log(f) + 1, 0
    for i in range(32):
        w = theta ** (-2 * i / 64)
        keep = min(1.0, max(0.0, (trained * w / (2 * math.pi) - slow) / (fast - slow)))
        between += 0.0 < keep < 1.0
        for pos in (1, 57, 199):
            a = pos * (keep * w + (1 - keep) * w / f)
            # one rounding of a value of at most g < 2
            assert abs(float(t[pos, i, 0]) - g * math.cos(a)) <= 2 ** -23
            assert abs(float(t[pos, i, 1]) - g * math.sin(a)) <= 2 ** -23
    assert between >= 8


def test_refusals_say_what_was_given():
    """Messages are formatted in C++, which takes one C++ runtime in the process."""
    z = torch.zeros(1, 8, 2, 128, dtype=torch.bfloat16)
    n = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="not on cpu"):
        paged.paged_attention(z[0], z, z, n[None], n, n)
    with pytest.raises(ValueError, match=r"BFloat16 \[8, 2, 128\] on cpu"):
        paged.rotary(z[0], torch.zeros(4, 64, 2), n)


def _in_a_copy(tmp_path, code, **env):
    """Runs `code` where a copy of the package without its built binding is imported."""
    pkg = tmp_path / "reworld_b200"
    shutil.copytree(os.path.dirname(_native.__file__), pkg, ignore=shutil.ignore_patterns("__pycache__", "paged_bind*"))
    shutil.copytree(os.path.join(os.path.dirname(os.path.dirname(_native.__file__)), "include"), tmp_path / "include")
    return subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True,
                          env={**os.environ, "PYTHONPATH": str(tmp_path), **env})


def test_without_the_binding_everything_else_is_imported_and_paged_calls_fail(tmp_path):
    r = _in_a_copy(tmp_path, """
import torch, reworld_b200
from reworld_b200 import attention, paged, self_attn, landmark, ulysses
assert reworld_b200.__file__.startswith({!r})
assert paged.rotary_table(4, 16, device="cpu").shape == (4, 8, 2)
try:
    reworld_b200.rotary(None, None, None)
except ImportError as e:
    print("refused:", e)
""".format(str(tmp_path)))
    assert r.returncode == 0, r.stderr
    assert "refused:" in r.stdout and "build.py" in r.stdout


def test_the_library_is_built_where_the_binding_cannot_be(tmp_path):
    """With a C++ compiler that fails, build() says so, and the library is there."""
    r = _in_a_copy(tmp_path, """
import importlib.util, os
spec = importlib.util.spec_from_file_location("b", "reworld_b200/build.py")
b = importlib.util.module_from_spec(spec)
spec.loader.exec_module(b)
os.remove(b.lib_path())
b._sources = lambda: [os.path.join(b.CSRC, "api.cu")]
try:
    b.build()
except RuntimeError as e:
    print("refused:", e)
assert os.path.exists(b.lib_path()) and not os.path.exists(b.bind_path())
""", CXX="false")
    assert r.returncode == 0, r.stderr
    assert "refused:" in r.stdout


def test_a_binding_for_another_torch_is_refused_and_built_again(tmp_path):
    r = _in_a_copy(tmp_path, """
import importlib.util, os
spec = importlib.util.spec_from_file_location("b", "reworld_b200/build.py")
b = importlib.util.module_from_spec(spec)
spec.loader.exec_module(b)
open(b.bind_path(), "w").close()
open(b.bind_stamp_path(), "w").write("torch 1.0 another")
b._sources = lambda: [os.path.join(b.CSRC, "api.cu")]
b._compile_bind = lambda obj: open(obj, "w").close() or ["touch", b.bind_path() + ".tmp"]
from reworld_b200 import paged
try:
    paged.rotary(None, None, None)
except ImportError as e:
    print("refused:", e)
b.build()
assert b.bind_made_for() == b.bind_stamp() and b.bind_stamp().startswith("torch 2")
b._compile_bind = None
b.build()                                                # up to date now
""")
    assert r.returncode == 0, r.stderr
    assert "refused:" in r.stdout and "torch 1.0 another" in r.stdout
