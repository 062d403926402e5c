"""What the entry points of include/q8_mix.h refuse, with the reason, before they touch a GPU: the
structures' sizes and fields as C lays them out, and each refusal in a forked process of its own (the
checks read nothing behind the runtime's pointer, so one that has no GPU behind it will do)."""
import os
import subprocess
import sys
import textwrap

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
        return m.Kv(**{**dict(k=at(60), v=at(70), type=1, dim=64, heads=2, page=16, pages=9, table=at(80), table_ld=4), **k})

    def conv(s=None, **k):
        a = {**dict(x=at(1), x_ld=64, ch=64, w=at(2), taps=4, s_in=at(3), s_out=at(4), y=at(5), y_ld=64), **k}
        lib.rt_conv_silu_dev(c.byref(r), c.byref(s or seqs()), *a.values())

    def delta(s=None, **k):
        a = dict(k_heads=2, v_heads=4, k_dim=64, v_dim=32, tiled=0, q=at(1), k=at(2), v=at(3), q_ld=128, k_ld=128, v_ld=128, a=at(4), b=at(5), a_ld=4, b_ld=4,
                 decay=at(6), dt=at(7), eps=1e-6, scale=1.0, s_in=at(8), s_out=at(9), z=None, z_ld=0, nw=None, nw_eps=1e-6, o=at(10), o_ld=128)
        lib.rt_delta_rule_dev(c.byref(r), c.byref(s or seqs()), c.byref(m.Delta(**{**a, **k})))

    def rope(s=None, cache=None, **k):
        a = dict(q=at(1), q_ld=256, q_hd=64, q_heads=4, k=at(2), v=at(3), k_ld=128, k_hd=64, v_ld=128, v_hd=64, q_norm=at(4), k_norm=at(5), eps=1e-6, rot=64,
                 pairs=0, freq=at(6), out=at(7), out_ld=256, out_hd=64)
        lib.rt_rope_kv_dev(c.byref(r), c.byref(s or seqs()), c.byref(cache or kv()), c.byref(m.Rope(**{**a, **k})))

    def attn(s=None, cache=None, **k):
        a = dict(q=at(1), q_ld=256, q_hd=64, q_heads=4, scale=0.1, gate=None, gate_ld=0, gate_hd=0, o=at(2), o_ld=256)
        lib.rt_attn_kv_dev(c.byref(r), c.byref(s or seqs()), c.byref(cache or kv()), c.byref(m.Attn(**{**a, **k})))

    def no_init(fn, *args):
        getattr(lib, fn)(c.byref(m.Rt()), *args)

    CASES = [
        ("rt_init has not run", lambda: no_init("rt_conv_silu_dev", None, None, 0, 0, None, 0, None, None, None, 0)),
        ("rt_init has not run", lambda: no_init("rt_delta_rule_dev", None, None)),
        ("rt_init has not run", lambda: no_init("rt_rope_kv_dev", None, None, None)),
        ("rt_init has not run", lambda: no_init("rt_attn_kv_dev", None, None, None)),
        ("struct rt_seqs", lambda: lib.rt_delta_rule_dev(c.byref(r), None, None)),
        ("struct rt_delta", lambda: lib.rt_delta_rule_dev(c.byref(r), c.byref(seqs()), None)),
        ("struct rt_kv", lambda: lib.rt_attn_kv_dev(c.byref(r), c.byref(seqs()), None, None)),
        ("struct rt_rope", lambda: lib.rt_rope_kv_dev(c.byref(r), c.byref(seqs()), c.byref(kv()), None)),
        ("struct rt_attn", lambda: lib.rt_attn_kv_dev(c.byref(r), c.byref(seqs()), c.byref(kv()), None)),
        *[("longest from 1 to t", lambda f=f, k=k: f(seqs(**k))) for f in (conv, delta, rope, attn)
          for k in (dict(n=0), dict(n=65536), dict(t=0), dict(t=1 << 23), dict(longest=0), dict(longest=11))],
        *[("start must be", lambda f=f: f(seqs(start=None))) for f in (conv, delta, rope, attn)],
        *[("past must be", lambda f=f: f(seqs(past=at(3) + 2))) for f in (rope, attn)],
        *[("multiple of 4 channels", lambda k=k: conv(**k)) for k in (dict(ch=62), dict(ch=0), dict(taps=1), dict(taps=9))],
        *[("16-byte aligned", lambda k=k: conv(**k)) for k in (dict(x=at(1) + 4), dict(w=None), dict(y=0), dict(s_in=None), dict(s_out=at(4) + 8))],
        ("x_ld must be", lambda: conv(x_ld=60)),
        ("y_ld must be", lambda: conv(y_ld=66)),
        ("y overlaps", lambda: conv(y=at(1) + 64)),
        ("y overlaps", lambda: conv(y=at(3))),
        ("y overlaps", lambda: conv(y=at(4) + 16)),
        ("s_out must be s_in or apart", lambda: conv(s_out=at(3) + 16)),
        ("s_out overlaps", lambda: conv(s_out=at(1))),
        ("s_out overlaps", lambda: conv(s_out=at(2) - 16)),
        *[("value heads, a multiple", lambda k=k: delta(**k)) for k in (dict(k_heads=0), dict(v_heads=3), dict(v_heads=4098), dict(v_heads=0))],
        *[("k_dim must be", lambda k=k: delta(k_dim=k)) for k in (0, 48, 160, 512)],
        *[("v_dim must be", lambda k=k: delta(v_dim=k)) for k in (0, 24, 528)],
        *[("must be a multiple of 4 of at least", lambda k=k: delta(**{k: 124})) for k in ("q_ld", "k_ld", "v_ld", "o_ld")],
        ("a_ld and b_ld", lambda: delta(a_ld=3)),
        ("decay must be", lambda: delta(decay=None)),
        ("nw must be", lambda: delta(z=at(20), z_ld=128)),
        ("z_ld must be", lambda: delta(z=at(20), z_ld=100, nw=at(21))),
        *[("o overlaps", lambda k=k: delta(o=at(k))) for k in (1, 2, 3, 4, 5, 6, 7, 8, 9, 90)],
        ("o overlaps", lambda: delta(z=at(10), z_ld=128, nw=at(21))),
        ("s_out overlaps", lambda: delta(s_out=at(3))),
        ("s_out must be s_in or apart", lambda: delta(s_out=at(8) + 64)),
        *[("the cache's type", lambda f=f: f(cache=kv(type=3))) for f in (rope, attn)],
        *[("head's size", lambda f=f, k=k: f(cache=kv(dim=k))) for f in (rope, attn) for k in (16, 48, 288)],
        *[("key-value heads", lambda f=f: f(cache=kv(heads=0))) for f in (rope, attn)],
        *[("needs pages", lambda f=f, k=k: f(cache=kv(**k))) for f in (rope, attn) for k in (dict(page=0), dict(pages=0), dict(table_ld=0), dict(pages=1 << 31))],
        *[("fewer than 2^31 rows", lambda f=f: f(cache=kv(pages=(1 << 31) - 1, page=1 << 30))) for f in (rope, attn)],
        *[("the page table", lambda f=f: f(cache=kv(table=None))) for f in (rope, attn)],
        *[("cache's v must", lambda f=f: f(cache=kv(v=at(70) + 2))) for f in (rope, attn)],
        ("query heads", lambda: rope(q_heads=0)),
        *[("rot must be", lambda k=k: rope(rot=k)) for k in (-2, 7, 66)],
        ("strides are multiples of 4", lambda: rope(q_hd=62)),
        ("strides are multiples of 4", lambda: rope(k_ld=-4)),
        ("its heads must not overlap", lambda: rope(out_hd=60)),
        ("its heads must not overlap", lambda: rope(out_ld=252)),
        ("freq must be", lambda: rope(freq=at(6) + 4)),
        ("out overlaps", lambda: rope(out=at(1), out_ld=512)),
        ("out overlaps", lambda: rope(out=at(2))),
        ("out overlaps", lambda: rope(out=at(60))),
        ("the cache's k overlaps", lambda: rope(cache=kv(v=at(60) + 16))),
        ("the cache's k overlaps", lambda: rope(cache=kv(k=at(3)))),
        ("the cache's v overlaps", lambda: rope(cache=kv(v=at(80)))),
        *[("query heads, a multiple", lambda k=k: attn(q_heads=k)) for k in (0, 3, 4098)],
        ("o_ld must be", lambda: attn(o_ld=252)),
        ("o overlaps", lambda: attn(o=at(1) + 128)),
        ("o overlaps", lambda: attn(o=at(70))),
        ("o overlaps", lambda: attn(o=at(30), gate=at(30) + 1024, gate_ld=256, gate_hd=64)),
        ("gate must be", lambda: attn(gate=at(30) + 4, gate_ld=256, gate_hd=64)),
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


FIELDS = {"rt_seqs": "Seqs", "rt_delta": "Delta", "rt_kv": "Kv", "rt_rope": "Rope", "rt_attn": "Attn"}


def test_structures_are_c_s(q8rt, tmp_path):
    """Every field of the binding's structures at the offset where C has it, and nothing else in them."""
    lines = []
    for name, cls in FIELDS.items():
        k = getattr(q8rt, cls)
        lines.append(f'printf("{name} %zu\\n", sizeof(struct {name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof(struct {name}, {f}));' for f, _ in k._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "q8_mix.h"\nint main(void) {' + "\n".join(lines) + "return 0; }")
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    import ctypes

    for name, cls in FIELDS.items():
        k = getattr(q8rt, cls)
        assert int(got[name]) == ctypes.sizeof(k)
        for f, _ in k._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(k, f).offset, (name, f)
