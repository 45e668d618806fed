"""What the 8-bit page calls and apply_rotary refuse, their plan and their mirrors (no GPU)."""

from __future__ import annotations

import math
import os
import subprocess

import pytest
import torch

from tritonkv_amd import _lib
from tritonkv_amd import paged8 as p8
from tritonkv_amd import pages
from tritonkv_amd import rotary as ro

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I32 = torch.int32


def pool(P=4, HKV=2, page=64, D=64, dtype=torch.int8, block=32):
    return p8.empty_paged8_pool(P, HKV, page, D, dtype, block, device="cpu")


def append_args(**kw):
    a = dict(k_pool=pool(), v_pool=pool(), k_new=torch.zeros(1, 2, 3, 64), v_new=torch.zeros(1, 2, 3, 64),
             block_table=torch.zeros(1, 2, dtype=I32), positions=torch.zeros(1, dtype=I32))
    a.update(kw)
    return a


def decode_args(**kw):
    a = dict(q=torch.zeros(1, 4, 64).half(), k_pool=pool(), v_pool=pool(), block_table=torch.zeros(1, 2, dtype=I32),
             seq_lens=torch.zeros(1, dtype=I32))
    a.update(kw)
    return a


def test_pools():
    for kw, err in ((dict(block=16), ValueError), (dict(block=48), ValueError), (dict(page=48), ValueError),
                    (dict(page=0), ValueError), (dict(P=0), ValueError), (dict(HKV=0), ValueError), (dict(D=80), ValueError),
                    (dict(dtype=torch.uint8), TypeError), (dict(dtype=torch.float8_e5m2), TypeError),
                    (dict(page=2 ** 25), ValueError)):
        with pytest.raises(err):
            pool(**kw)
    p = pool(3, 2, 96, 64, torch.float8_e4m3fn, 32)
    assert p.codes.shape == (3, 2, 96, 64) and p.scale.shape == (3, 2, 3) and p.block == 32 and p.page_size == 96
    assert not p.scale.any()
    codes, scale = p.page_tensors()
    assert codes is p.codes and scale.shape == (3, 1, 1, 8) and scale.data_ptr() == p.scale.data_ptr()
    assert scale.stride(0) * 4 % 16 == 0


def test_pages_of_scales_need_room():
    for scale in (torch.zeros(3, 1, 1), torch.zeros(3, 2, 3), torch.zeros(2, 3, 2).transpose(1, 2)):
        with pytest.raises(ValueError, match="16 bytes"):
            p8.Paged8Pool(torch.zeros(scale.shape[0], scale.shape[1], 32 * scale.shape[2], 64, dtype=torch.int8),
                          scale).page_tensors()
    with pytest.raises(TypeError, match="list"):
        pages.copy_pages(pool(), torch.zeros(1, dtype=I32), torch.zeros(1, dtype=I32))
    with pytest.raises(RuntimeError, match="GPU"):  # taken, but for the device
        pages.copy_pages([pool(), pool()], torch.zeros(1, dtype=I32), torch.zeros(1, dtype=I32))


@pytest.mark.parametrize("name,change", [
    ("codes", lambda p: p8.Paged8Pool(p.codes[0], p.scale)),
    ("dtype", lambda p: p8.Paged8Pool(p.codes.view(torch.uint8), p.scale)),
    ("dense", lambda p: p8.Paged8Pool(torch.zeros(4, 2, 64, 72, dtype=torch.int8)[..., 8:], p.scale)),
    ("expanded", lambda p: p8.Paged8Pool(p.codes[:1].expand(4, 2, 64, 64), p.scale)),
    ("scale shape", lambda p: p8.Paged8Pool(p.codes, p.scale[:, :1])),
    ("scale dtype", lambda p: p8.Paged8Pool(p.codes, p.scale.half())),
    ("scale shared", lambda p: p8.Paged8Pool(p.codes, p.scale[:1].expand(4, 2, 2))),
    ("block", lambda p: p8.Paged8Pool(p.codes, torch.zeros(4, 2, 4))),
    ("not a pool", lambda p: p.codes),
])
def test_malformed_pools(name, change):
    bad = change(pool())
    for call, args in ((p8.paged8_append, append_args(k_pool=bad)), (p8.paged8_decode_attention, decode_args(v_pool=bad))):
        with pytest.raises((ValueError, TypeError)):
            call(**args)
    with pytest.raises((ValueError, TypeError)):
        p8.paged8_read(bad, pool(), torch.zeros(1, 2, dtype=I32), tokens=3)


@pytest.mark.parametrize("kw,err", [
    (dict(k_new=torch.zeros(1, 3, 3, 64)), ValueError),
    (dict(k_new=torch.zeros(1, 2, 3, 64).double()), TypeError),
    (dict(v_new=torch.zeros(1, 2, 4, 64)), ValueError),
    (dict(v_new=torch.zeros(1, 2, 3, 64).half()), ValueError),
    (dict(v_pool=pool(block=64)), ValueError),
    (dict(v_pool=pool(dtype=torch.float8_e4m3fn)), ValueError),
    (dict(block_table=torch.zeros(2, 2, dtype=I32)), ValueError),
    (dict(block_table=torch.zeros(1, 2, dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(2, dtype=I32)), ValueError),
    (dict(counts=torch.zeros(1)), ValueError),
    (dict(q=torch.zeros(1, 4, 3, 64)), ValueError),
    (dict(q_out=torch.zeros(1, 4, 3, 64)), ValueError),
    (dict(rotary=3), TypeError),
    (dict(rotary=ro.Rotary(24, device="cpu")), ValueError),
    (dict(rotary=ro.Rotary(128, device="cpu")), ValueError),
    (dict(rotary=ro.Rotary(64, device="cpu"), q=torch.zeros(1, 4, 2, 64)), ValueError),
    (dict(rotary=ro.Rotary(64, device="cpu"), q=torch.zeros(1, 4, 3, 64).half()), ValueError),
    (dict(rotary=ro.Rotary(64, device="cpu"), q_out=torch.zeros(1, 4, 3, 64)), ValueError),
    (dict(rotary=ro.Rotary(64, device="cpu"), q=torch.zeros(1, 4, 3, 64), q_out=torch.zeros(1, 4, 3, 65)[..., 1:]),
     ValueError),
    (dict(k_new=torch.zeros(1, 2, 3, 64, requires_grad=True)), ValueError),
])
def test_append_refuses(kw, err):
    with pytest.raises(err):
        p8.paged8_append(**append_args(**kw))


def test_append_refuses_outputs_over_inputs():
    rot, q = ro.Rotary(64, device="cpu"), torch.zeros(1, 5, 3, 64)
    with pytest.raises(ValueError, match="share"):
        p8.paged8_append(**append_args(rotary=rot, q=q[:, :4], q_out=q[:, 1:]))
    k = torch.zeros(1, 4, 3, 64)
    with pytest.raises(ValueError, match="share"):
        p8.paged8_append(**append_args(rotary=rot, k_new=k[:, :2], q=q[:, :4].clone(), q_out=k))
    with pytest.raises(RuntimeError, match="GPU"):
        p8.paged8_append(**append_args(rotary=rot, q=q, q_out=q))


@pytest.mark.parametrize("kw,err", [
    (dict(q=torch.zeros(1, 4, 32).half()), ValueError),
    (dict(q=torch.zeros(1, 4, 64)), TypeError),
    (dict(q=torch.zeros(1, 3, 64).half()), ValueError),
    (dict(q=torch.zeros(0, 4, 64).half()), ValueError),
    (dict(q=torch.zeros(1, 4, 33, 64).half()), ValueError),
    (dict(q=torch.zeros(1, 4, 0, 64).half()), ValueError),
    (dict(seq_lens=torch.zeros(2, dtype=I32)), ValueError),
    (dict(counts=torch.zeros(1, dtype=torch.int64)), ValueError),
    (dict(out=torch.zeros(1, 4, 1, 64)), ValueError),
    (dict(out=torch.zeros(1, 4, 64).half()), ValueError),
    (dict(lse=torch.zeros(1, 4, 64)), ValueError),
    (dict(block_table=torch.zeros(1, 0, dtype=I32)), ValueError),
    (dict(piece_tokens=0), ValueError),
])
def test_decode_refuses(kw, err):
    with pytest.raises(err):
        p8.paged8_decode_attention(**decode_args(**kw))


def test_read_refuses():
    t = torch.zeros(1, 2, dtype=I32)
    x = torch.zeros(1, 2, 3, 64)
    for kw, err in ((dict(), ValueError), (dict(tokens=-1), ValueError), (dict(tokens=3, dtype=torch.int8), TypeError),
                    (dict(out=(x, x.half())), ValueError), (dict(out=x), ValueError), (dict(out=(x, x)), ValueError),
                    (dict(out=(x, torch.zeros(1, 2, 4, 64))), ValueError), (dict(out=(x, x.clone()), tokens=4), ValueError),
                    (dict(out=(x.double(), x.double())), TypeError),
                    (dict(out=(x, torch.zeros(1, 2, 3, 65)[..., 1:])), ValueError),
                    (dict(tokens=3, positions=torch.zeros(2, dtype=I32)), ValueError),
                    (dict(tokens=3, counts=torch.zeros(1)), ValueError)):
        with pytest.raises(err):
            p8.paged8_read(pool(), pool(), t, **kw)
    with pytest.raises(RuntimeError, match="GPU"):
        p8.paged8_read(pool(), pool(), t, tokens=3)


def test_rotary_refuses():
    rot = ro.Rotary(64, device="cpu")
    q, k, pos = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 3, 64), torch.zeros(2, dtype=I32)
    for args, kw, err in (
            ((q[0, 0], None, pos, rot), {}, ValueError), ((q.double(), None, pos, rot), {}, TypeError),
            ((q, k[:, :, :2], pos, rot), {}, ValueError), ((q, k.half(), pos, rot), {}, ValueError),
            ((q, k, pos.long(), rot), {}, ValueError), ((q, k, torch.zeros(3, dtype=I32), rot), {}, ValueError),
            ((q, k, pos, ro.Rotary(128, device="cpu")), {}, ValueError), ((q, k, pos, rot.inv_freq), {}, TypeError),
            ((torch.zeros(2, 4, 3, 72), None, pos, rot), {}, ValueError),
            ((torch.zeros(2, 4, 3, 512), None, pos, rot), {}, ValueError),
            ((q, k, pos, rot), dict(out=q), ValueError), ((q, k, pos, rot), dict(out=(q, None)), ValueError),
            ((q, None, pos, rot), dict(out=(q, k)), ValueError), ((q, k, pos, rot), dict(out=(q, q[:, :2])), ValueError),
            ((q, k, pos, rot), dict(out=(q[:, :, :, :].half(), k)), ValueError),
            ((q.clone().requires_grad_(), k, pos, rot), {}, ValueError)):
        with pytest.raises(err):
            ro.apply_rotary(*args, **kw)
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        ro.apply_rotary(q, k, pos, rot)
    for kw, err in ((dict(), ValueError), (dict(dims=3), ValueError), (dict(dims=0), ValueError),
                    (dict(dims=64, base=1.0), ValueError), (dict(dims=64, scaling=dict(type="other", factor=2)), ValueError),
                    (dict(dims=64, scaling=dict(type="linear")), ValueError), (dict(dims=64, factor=math.inf), ValueError),
                    (dict(dims=64, scaling=dict(type="linear", factor=-1)), ValueError),
                    (dict(inv_freq=torch.zeros(4, dtype=I32)), ValueError), (dict(inv_freq=torch.zeros(0)), ValueError),
                    (dict(dims=8, inv_freq=torch.zeros(4)), ValueError)):
        with pytest.raises(err):
            ro.Rotary(device="cpu", **kw)


def test_frequencies():
    """The scalings against their formulas at the ends of the spectrum."""
    plain, one = ro.rotary_frequencies(64, 10000.0)
    assert one == 1.0 and plain[0] == 1.0 and math.isclose(plain[16], 10000.0 ** -0.5)
    assert ro.rotary_frequencies(64, 1e4, dict(type="linear", factor=4))[0] == [w / 4 for w in plain]
    ntk = ro.rotary_frequencies(64, 1e4, dict(type="ntk", factor=4))[0]
    assert ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-12)
    l3 = ro.rotary_frequencies(128, 5e5, dict(type="llama3", factor=8, low_freq_factor=1, high_freq_factor=4,
                                              original_max_position_embeddings=8192))[0]
    p3 = ro.rotary_frequencies(128, 5e5)[0]
    for w, x in zip(p3, l3):
        turns = 8192 * w / (2 * math.pi)
        assert math.isclose(x, w if turns >= 4 else w / 8 if turns <= 1 else
                            w * ((turns - 1) / 3 + (1 - (turns - 1) / 3) / 8), rel_tol=1e-12)
    y, f = ro.rotary_frequencies(64, 1e4, dict(type="yarn", factor=16, original_max_position_embeddings=4096))
    assert math.isclose(f, 0.1 * math.log(16) + 1)
    for w, x in zip(plain, y):
        turns = 4096 * w / (2 * math.pi)
        assert w / 16 <= x * (1 + 1e-12) and x <= w
        if turns > 40:
            assert x == w
        if turns < 0.7:
            assert math.isclose(x, w / 16)


def test_turns():
    """Frequencies as turns in 2**-64, against exact fractions."""
    from fractions import Fraction

    def arctan(n, one):  # of 1 / n
        x = total = one // n
        for k in range(3, 400, 2):
            x //= -n * n
            total += x // k
        return total

    one = 1 << 300
    inv_2pi = Fraction(one, 8 * (4 * arctan(5, one) - arctan(239, one)))
    g = torch.Generator().manual_seed(1)
    w = torch.cat([torch.tensor([1.0, 0.0, -0.25, 7.5, 1e-6, 1e-30, 3e5], dtype=torch.float64),
                   torch.rand(200, generator=g, dtype=torch.float64) * 3 - 1])
    for x, t in zip(w.tolist(), ro._turns(w).tolist()):
        off = (t - int(Fraction(x) * inv_2pi * 2 ** 64)) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= (16 if abs(x) < 10 else 2 ** 20)  # 8 products, each cut


def test_apart():
    x = torch.zeros(2, 7, 10, 8)  # (B, N, heads, D)
    q, k, v = (x[:, :, a:b].transpose(1, 2) for a, b in ((0, 6), (6, 8), (8, 10)))
    assert ro._apart(q, k) and ro._apart(k, v) and ro._apart(q, v) and ro._apart(k, q)
    assert not ro._apart(q, x[:, :, 5:7].transpose(1, 2)) and not ro._apart(q, q) and not ro._apart(x[0, 0], x[0, 0, 3:])
    assert ro._apart(x[0], x[1]) and ro._apart(x[:, :, 0], x[:, :, 1]) and not ro._apart(x[:, 1:], x[:, :6])
    assert ro._apart(x[:0], x)


def test_plan():
    for B, HKV, cols, S, D in ((1, 2, 6, 512, 128), (8, 16, 1, 4096, 64), (16, 8, 32, 8192, 128), (32, 8, 4, 32768, 128),
                               (65535, 1, 1, 64, 64), (3, 1, 33, 70000, 256), (1, 1000, 1, 4096, 128)):
        least, groups, few, long = p8.plan_shares8(B, HKV, cols, S, D)
        assert least >= 1 and 0 <= groups <= 65535 and (few, long) == (0, 0)
        if groups:
            assert groups <= -(-B * -(-S // 32) // least)
    assert p8.plan_shares8(1, 2, 6, 512, 128)[1] == 0 and p8.plan_shares8(1, 2, 6, 1024, 128)[1] > 0
    assert p8.plan_shares8(64, 8, 4, 1024, 128)[1] == 0
    with pytest.raises(ValueError):
        p8.plan_shares8(65536, 1, 1, 64, 64)


def test_mirrors_of_the_structures(tmp_path):
    names = {"tkv_paged8_args": _lib.Paged8Args, "tkv_paged8_append_args": _lib.Paged8AppendArgs,
             "tkv_paged8_read_args": _lib.Paged8ReadArgs, "tkv_rotary_args": _lib.RotaryArgs}
    lines = []
    for n, m in names.items():
        lines.append(f'printf("{n} %zu\\n", sizeof({n}));')
        lines += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for f, _ in m._fields_]
    c = tmp_path / "x.c"
    c.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "tkv.h"\nint main(void) {\n' + "\n".join(lines)
                 + "\nreturn 0; }\n")
    exe = tmp_path / "x"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    import ctypes
    for n, m in names.items():
        assert int(got[n]) == ctypes.sizeof(m)
        for f, _ in m._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(m, f).offset


def test_entries_refuse_malformed_blocks():
    """Argument blocks that the kernels could not take are turned away before anything is launched."""
    lib = _lib.load()
    for entry, block in ((lib.tkv_paged8_decode_attention, _lib.Paged8Args), (lib.tkv_paged8_append, _lib.Paged8AppendArgs),
                         (lib.tkv_paged8_read, _lib.Paged8ReadArgs), (lib.tkv_rotary, _lib.RotaryArgs)):
        assert entry(None, None) == _lib.TKV_EINVAL
        assert entry(block(), None) == _lib.TKV_EINVAL
    good = dict(q=4096, q_strides=(512, 64, 64), k=4096, v=4096, k_strides=(8192, 4096, 64), v_strides=(8192, 4096, 64),
                k_scale=4096, v_scale=4096, k_scale_strides=(4, 2, 1), v_scale_strides=(4, 2, 1), block_table=4096,
                out=4096, B=1, HQ=4, HKV=2, M=1, D=64, block=32, block_table_stride=1, max_pages=1, page_size=64,
                num_pages=4, sm_scale=1.0, least_chunks=1)
    for change in (dict(M=33), dict(M=0), dict(block=16), dict(block=128), dict(k=4100), dict(k_strides=(8192, 4096, 72)),
                   dict(k_strides=(8192, 4096, 0)), dict(k_scale_strides=(-1, 2, 1)), dict(q_strides=(512, 60, 64)),
                   dict(workgroups=4), dict(workgroups=70000), dict(HQ=3), dict(num_pages=0), dict(block_table_stride=0),
                   dict(least_chunks=0), dict(B=70000), dict(out=4100), dict(k_scale=4097)):
        assert lib.tkv_paged8_decode_attention(_lib.Paged8Args(**{**good, **change}), None) == _lib.TKV_EINVAL, change
    assert lib.tkv_paged8_decode_attention(_lib.Paged8Args(**{**good, "D": 96}), None) == _lib.TKV_EUNSUPPORTED
