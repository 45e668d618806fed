"""Rotary positions against the formula in 64 bits, and the gradient's way against differences."""

from __future__ import annotations

import pytest
import torch

import paged8_ref as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def bound(y, a, factor):
    """Rounding to the type, half a step; and 8 * 2^-24 of the pair's magnitudes: cos and sin are off by at
    most 4 * 2^-24 (angle, series), their product with the factor, the two products and the sum by
    one each."""
    eps = torch.finfo(y.dtype).eps / 2
    return eps * y.double().abs() + 8 * 2.0 ** -24 * abs(factor) * a + torch.finfo(y.dtype).tiny


def pair_sum(x, n, interleaved):
    """|a| + |b| of every value's pair."""
    y = x.abs().clone()
    first = torch.arange(n) * 2 if interleaved else torch.arange(n)
    second = first + 1 if interleaved else first + n
    s = y[..., first] + y[..., second]
    y[..., first] = s
    y[..., second] = s
    return y


def check(B, HQ, HKV, N, D, dims, dtype, interleaved=False, factor=1.0, adjoint=False, far=100000, token_major=False,
          explicit=False, seed=0, inside=False, short=False):
    from tritonkv_amd.rotary import Rotary, apply_rotary

    g = torch.Generator().manual_seed(seed)
    w = torch.tensor([10000.0 ** (-2.0 * i / dims) for i in range(dims // 2)], dtype=torch.float64)
    rot = Rotary(inv_freq=w.cuda(), interleaved=interleaved, factor=factor)
    pos = torch.randint(-far, far, (B, N) if explicit else (B,), generator=g, dtype=torch.int32)
    xs = []
    for H in (HQ, HKV):
        x = torch.randn(*((B, N, H, D) if token_major else (B, H, N, D)), generator=g).to(dtype)
        xs.append(x.transpose(1, 2) if token_major else x)
    t = pos.long() if explicit else pos.long()[:, None] + torch.arange(N)
    cuda = [x.cuda() for x in xs]
    if short:
        cuda = [x[:, :, 0] for x in cuda]
    out = tuple(cuda) if inside else None
    got = apply_rotary(*cuda, pos.cuda(), rot, adjoint=adjoint, out=out)
    for x, y in zip(xs, got):
        want = ref.turn(x.double(), t[:, None], w, interleaved, factor, adjoint)
        y = y.cpu().view(x.shape) if short else y.cpu()
        tol = bound(y, pair_sum(x.double(), dims // 2, interleaved), factor)
        ref.assert_within(y, want, tol)
        assert torch.equal(y[..., dims:], x[..., dims:])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,dims", [(64, 64), (128, 128), (256, 256), (128, 64), (128, 32), (128, 20), (64, 2), (80, 24),
                                    (16, 16), (256, 250)])
def test_forms(dtype, interleaved, D, dims):
    check(2, 3, 2, 5, D, dims, dtype, interleaved, seed=D + dims)
    check(2, 3, 2, 5, D, dims, dtype, interleaved, factor=1.3, adjoint=True, token_major=True, seed=dims)


@pytest.mark.parametrize("N", [1, 2, 63, 64, 65])
@pytest.mark.parametrize("explicit", [False, True])
def test_lengths_and_positions(N, explicit):
    check(3, 4, 1, N, 128, 128, BF16, explicit=explicit)
    check(3, 4, 1, N, 128, 128, F32, explicit=explicit, far=2 ** 31 - 100)


@pytest.mark.parametrize("B,N", [(1, 8200), (3, 2731), (4100, 2)])
def test_many_tokens(B, N):
    check(B, 2, 1, N, 64, 64, F16, token_major=B == 3)


def test_one_token_without_its_axis():
    check(5, 4, 2, 1, 128, 128, BF16, short=True)
    check(5, 4, 2, 1, 128, 128, BF16, short=True, inside=True)


@pytest.mark.parametrize("dims,interleaved", [(128, False), (20, False), (20, True)])
def test_in_place(dims, interleaved):
    check(2, 4, 2, 9, 128, dims, BF16, interleaved, inside=True)


def test_queries_and_keys_of_one_projection_in_place():
    from tritonkv_amd.rotary import Rotary, apply_rotary

    B, N, HQ, HKV, D = 2, 7, 4, 2, 64
    qkv = torch.randn(B, N, (HQ + 2 * HKV) * D, device="cuda").bfloat16()
    q = qkv[..., :HQ * D].view(B, N, HQ, D).transpose(1, 2)
    k = qkv[..., HQ * D:(HQ + HKV) * D].view(B, N, HKV, D).transpose(1, 2)
    v = qkv[..., (HQ + HKV) * D:].clone()
    rot, pos = Rotary(D), torch.tensor([3, 1000], dtype=torch.int32, device="cuda")
    want = apply_rotary(q, k, pos, rot)
    ws: dict = {}
    got = apply_rotary(q, k, pos, rot, out=(q, k), _workspace=ws)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0] is q
    assert torch.equal(qkv[..., (HQ + HKV) * D:], v)


def test_queries_alone_and_odd_strides():
    from tritonkv_amd.rotary import Rotary, apply_rotary

    rot, pos = Rotary(64), torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 3, 11, 64, device="cuda").half()
    want, none = apply_rotary(q, None, pos, rot)
    assert none is None
    odd = torch.randn(2, 3, 11, 65, device="cuda").half()[..., 1:]  # rows off 16 bytes: read through a copy
    odd.copy_(q)
    assert torch.equal(apply_rotary(odd, None, pos, rot)[0], want)
    wide = torch.zeros(2, 3, 11, 128, device="cuda").half()
    out = wide[..., 64:]
    assert apply_rotary(q, None, pos, rot, out=(out, None))[0] is out
    assert torch.equal(out, want) and not wide[..., :64].any()
    empty = apply_rotary(q[:, :, :0], None, pos, rot)[0]
    assert empty.shape == (2, 3, 0, 64)
    # positions of every second entry, as they lie
    two = torch.stack([pos, pos + 100], 1)
    assert torch.equal(apply_rotary(q, None, two[:, 0], rot)[0], want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_adjoint_is_the_gradient(interleaved):
    """<g, dy/dx e> by differences of the 64-bit formula equals the call's gradient; and <g, R x> = <R' g, x>."""
    from tritonkv_amd.rotary import Rotary, apply_rotary

    D, dims, factor = 32, 24, 1.25
    gen = torch.Generator().manual_seed(1)
    w = torch.rand(dims // 2, generator=gen, dtype=torch.float64)
    rot = Rotary(inv_freq=w.cuda(), interleaved=interleaved, factor=factor)
    x, g = (torch.randn(1, 2, 3, D, generator=gen) for _ in range(2))
    pos = torch.tensor([12345], dtype=torch.int32)
    t = pos.long()[:, None] + torch.arange(3)
    got = apply_rotary(g.cuda(), None, pos.cuda(), rot, adjoint=True)[0].cpu().double()
    f = lambda z: (ref.turn(z, t[:, None], w, interleaved, factor) * g.double()).sum()  # noqa: E731
    h = 1e-4
    for i in torch.randperm(x.numel(), generator=gen)[:40].tolist():
        e = torch.zeros(x.numel(), dtype=torch.float64)
        e[i] = h
        e = e.view(x.shape)
        diff = (f(x.double() + e) - f(x.double() - e)) / (2 * h)
        assert abs(float(diff) - float(got.flatten()[i])) <= 1e-6 * 10
    leaf = x.double().requires_grad_()
    f(leaf).backward()
    tol = bound(got.float(), pair_sum(g.double(), dims // 2, interleaved), factor)
    ref.assert_within(got, leaf.grad, tol)


def test_kept_calls_streams_and_graphs():
    from tritonkv_amd.rotary import Rotary, apply_rotary

    rot, pos = Rotary(128), torch.tensor([5, 90000], dtype=torch.int32, device="cuda")
    sets = [(torch.randn(2, 4, 1, 128, device="cuda").half(), torch.randn(2, 2, 1, 128, device="cuda").half())
            for _ in range(3)]
    want = [apply_rotary(q, k, pos, rot) for q, k in sets]
    ws: dict = {}
    outs = [tuple(torch.empty_like(x) for x in s) for s in sets]
    for _ in range(2):
        for s, o, w in zip(sets, outs, want):
            assert apply_rotary(*s, pos, rot, out=o, _workspace=ws)[0] is o[0]
            assert all(torch.equal(a, b) for a, b in zip(o, w))
    assert "call" in ws
    # another factor is another call, whatever the workspace holds
    double = Rotary(128, factor=2.0)
    got = apply_rotary(*sets[0], pos, double, out=outs[0], _workspace=ws)
    assert torch.equal(got[0], apply_rotary(*sets[0], pos, double)[0]) and not torch.equal(got[0], want[0][0])
    # outputs that a kept call may not have: over an input
    q, k = sets[1]
    with pytest.raises(ValueError, match="share"):
        apply_rotary(q, k, pos, double, out=(outs[1][0], q[:, :2]), _workspace=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = apply_rotary(*sets[1], pos, rot, out=outs[1], _workspace=ws)
    side.synchronize()
    assert torch.equal(a[0], want[1][0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        apply_rotary(*sets[2], pos, rot, out=outs[2], _workspace=ws)
    for p in (1, 77, 123456):
        pos.fill_(p)
        graph.replay()
        want2 = apply_rotary(*sets[2], pos, rot)
        assert all(torch.equal(a, b) for a, b in zip(outs[2], want2))
