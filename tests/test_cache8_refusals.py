"""What the entry points of the 8-bit cache, of reading a cache back and of windows refuse, with the reason, before they touch a
GPU (as test_mix_refusals.py: each in a forked process, on addresses that nothing reads), the structure as C lays it out, and
a cache's size."""
import ctypes
import os
import subprocess
import sys
import textwrap

import numpy as np

from cache8_ref import quantise, seen, value

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = textwrap.dedent(
    """
    import ctypes as c, os, sys
    sys.path.insert(0, "tests")
    from conftest import load_package
    m = load_package()
    lib = m.load()
    block = c.create_string_buffer(1 << 16)
    r = m.Rt()
    r.chain = c.addressof(block)
    A = 1 << 30  # addresses that nothing reads: the call is refused first
    at = lambda i: A * (i + 1)

    def seqs(**k):
        return m.Seqs(**{**dict(n=2, t=10, longest=5, start=at(90), past=at(91)), **k})

    def kv(**k):
        return m.Kv(**{**dict(k=at(60), v=at(70), type=8, dim=64, heads=2, page=16, pages=9, table=at(80), table_ld=4), **k})

    ROWS = 9 * 2 * 16  # of that cache, 64 + 4 bytes each

    def rope(s=None, cache=None, **k):
        a = dict(q=at(1), q_ld=256, q_hd=64, q_heads=4, k=at(2), v=at(3), k_ld=128, k_hd=64, v_ld=128, v_hd=64, q_norm=at(4), k_norm=at(5), eps=1e-6, rot=64,
                 pairs=0, freq=at(6), out=at(7), out_ld=256, out_hd=64)
        lib.rt_rope_kv_dev(c.byref(r), c.byref(s or seqs()), c.byref(cache or kv()), c.byref(m.Rope(**{**a, **k})))

    def window(s=None, cache=None, window=5, sinks=1, **k):
        a = dict(q=at(1), q_ld=256, q_hd=64, q_heads=4, scale=0.1, gate=None, gate_ld=0, gate_hd=0, o=at(2), o_ld=256)
        lib.rt_attn_window_dev(c.byref(r), c.byref(s or seqs()), c.byref(cache or kv()), c.byref(m.Attn(**{**a, **k})), window, sinks)

    def read(s=None, cache=None, **k):
        a = dict(type=0, k=at(1), k_ld=128, k_hd=64, v=at(2), v_ld=128, v_hd=64)
        lib.rt_kv_read_dev(c.byref(r), c.byref(s or seqs()), c.byref(cache or kv()), c.byref(m.KvRows(**{**a, **k})))

    def no_init(fn, *args):
        getattr(lib, fn)(c.byref(m.Rt()), *args)

    CASES = [
        ("rt_init has not run", lambda: no_init("rt_attn_window_dev", None, None, None, 1, 0)),
        ("rt_init has not run", lambda: no_init("rt_kv_read_dev", None, None, None)),
        ("struct rt_seqs", lambda: lib.rt_kv_read_dev(c.byref(r), None, None, None)),
        ("struct rt_kv", lambda: lib.rt_kv_read_dev(c.byref(r), c.byref(seqs()), None, None)),
        ("struct rt_kv_rows", lambda: lib.rt_kv_read_dev(c.byref(r), c.byref(seqs()), c.byref(kv()), None)),
        ("struct rt_attn", lambda: lib.rt_attn_window_dev(c.byref(r), c.byref(seqs()), c.byref(kv()), None, 1, 0)),
        ("struct rt_kv", lambda: lib.rt_kv_bytes(None)),
        *[("the cache's type", lambda f=f, k=k: f(cache=kv(type=k))) for f in (rope, window, read) for k in (-1, 3, 7, 9)],
        ("the cache's type", lambda: lib.rt_kv_bytes(c.byref(kv(type=3)))),
        *[("head's size", lambda f=f, k=k: f(cache=kv(dim=k))) for f in (window, read) for k in (16, 48, 288)],
        *[("longest from 1 to t", lambda f=f, k=k: f(seqs(**k))) for f in (window, read) for k in (dict(n=0), dict(t=1 << 23), dict(longest=11))],
        *[("past must be", lambda f=f: f(seqs(past=None))) for f in (window, read)],
        *[("a window of 1 or more", lambda k=k: window(**k)) for k in (dict(window=0), dict(window=-3), dict(sinks=-1))],
        ("query heads, a multiple", lambda: window(q_heads=3)),
        ("o overlaps", lambda: window(o=at(60) + 68 * ROWS - 16)),
        ("out overlaps", lambda: rope(out=at(60) + 68 * ROWS - 16)),
        ("the cache's k overlaps", lambda: rope(cache=kv(v=at(60) + 68 * ROWS - 16))),
        *[("the rows' type", lambda k=k: read(type=k)) for k in (-1, 3, 8)],
        ("needs k or v", lambda: read(k=None, v=None)),
        ("k must be", lambda: read(k=at(1) + 8)),
        ("v must be", lambda: read(v=at(2) + 4)),
        ("strides are multiples of 4", lambda: read(k_ld=130)),
        *[("strides are multiples of 8", lambda k=k: read(**k)) for k in (dict(type=1, k_ld=132), dict(type=2, v_hd=68, v_ld=136))],
        ("its heads must not overlap", lambda: read(v_hd=32)),
        ("its heads must not overlap", lambda: read(k_ld=124)),
        ("k overlaps", lambda: read(k=at(2) + 64)),
        ("k overlaps", lambda: read(k=at(60) + 68 * ROWS - 16)),
        ("v overlaps", lambda: read(v=at(80))),
        ("v overlaps", lambda: read(k=None, v=at(70) - 4 * 128)),
    ]
    bad = 0
    for i, (why, call) in enumerate(CASES):
        rd, wr = os.pipe()
        pid = os.fork()
        if pid == 0:
            os.dup2(wr, 2)
            call()
            os._exit(0)
        os.close(wr)
        text = b""
        while chunk := os.read(rd, 4096):
            text += chunk
        os.close(rd)
        status = os.waitpid(pid, 0)[1]
        if not (os.WIFSIGNALED(status) and os.WTERMSIG(status) == 6) or why not in text.decode():
            bad += 1
            print("case", i, repr(why), "ended with", status, text.decode()[-300:])
    print(len(CASES), "refusals,", bad, "wrong")
    os._exit(1 if bad else 0)
    """
)


def test_every_refusal_says_why():
    env = {k: v for k, v in os.environ.items() if k != "Q8_ABORT_EXIT"}
    p = subprocess.run([sys.executable, "-c", DRIVER], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stdout + p.stderr


def test_structure_is_c_s(q8rt, tmp_path):
    k = q8rt.KvRows
    lines = ['printf("size %zu\\n", sizeof(struct rt_kv_rows));'] + [f'printf("{f} %zu\\n", offsetof(struct rt_kv_rows, {f}));' for f, _ in k._fields_]
    lines.append('printf("q8 %d\\n", RT_Q8);')
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "q8_mix.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got.pop("size")) == ctypes.sizeof(k) and int(got.pop("q8")) == q8rt.TYPES["q8"]
    assert {f: int(v) for f, v in got.items()} == {f: getattr(k, f).offset for f, _ in k._fields_}


def test_bytes(q8rt):
    lib = q8rt.load()
    for kind, row in (("f32", 4 * 96), ("f16", 2 * 96), ("bf16", 2 * 96), ("q8", 96 + 4)):
        kv = q8rt.Kv(type=q8rt.TYPES[kind], dim=96, heads=3, page=7, pages=11, table_ld=1)
        assert lib.rt_kv_bytes(ctypes.byref(kv)) == 3 * 7 * 11 * row


def test_definitions():
    """The references' own facts: a row's largest is 127 steps, every value within half a step, and a window's positions."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((200, 64)) * np.exp(rng.uniform(-40, 40, (200, 1)))).astype(np.float32)
    q, d = quantise(x)
    assert (np.abs(q).max(1) == 127).all() and (np.abs(value(q, d) - x) <= 0.50001 * d[:, None]).all()
    assert seen(5, 3, 0).tolist() == [3, 4, 5] and seen(5, 2, 1).tolist() == [0, 4, 5] and seen(2, 9, 1).tolist() == [0, 1, 2] and seen(1, 1, 4).tolist() == [0, 1]
