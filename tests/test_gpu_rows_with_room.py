"""Forks of rows that hold room made ahead, on the GPU: tables, counts and bytes against
the definition in Python integers, and the tokens that rows write afterwards.  All of it
is integers and copied bytes, so every comparison is for equality."""

from __future__ import annotations

import random

import pytest
import torch

from tests.rows_with_room import Rows, step

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16 = torch.float16
HKV, D = 2, 64


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _tokens(values):
    """K or V rows (B, HKV, 1, D) that hold the values' numbers."""
    return torch.tensor(values, dtype=F16, device=DEV).view(-1, 1, 1, 1).expand(-1, HKV, 1, D).contiguous()


def _check(m, state, pools):
    table, lens, refs = state
    assert table.tolist() == m.table and lens.tolist() == m.lens and refs.tolist() == m.refs
    for pool, sign in zip(pools, (1, -1)):
        first = pool.cpu()
        assert (first == first[:, :1, :, :1]).all()
        for b in range(m.B):
            row = [sign * float(first[m.table[b][n // m.page], 0, n % m.page, 0]) for n in range(len(m.tokens[b]))]
            assert row == m.tokens[b], b


@pytest.mark.parametrize("seed", range(10))
@pytest.mark.parametrize("workspace", [False, True])
def test_random_lives_with_room(seed, workspace):
    from tritonkv_amd.pages import fork_rows, resize_rows
    from tritonkv_amd.paged16 import paged16_append

    rng = random.Random(seed)
    B, P, page = rng.choice([1, 2, 5, 9, 40]), rng.choice([1, 3, 8]), rng.choice([16, 32, 48])
    m = Rows(B, P, rng.choice([B * P // 2 + 1, B * P + 3, 3000]), page)
    pools = [torch.zeros(m.N, HKV, page, D, dtype=F16, device=DEV) for _ in range(2)]
    state = _i32(m.table), _i32(m.lens), _i32(m.refs)
    ws = {} if workspace else None
    seen = 0
    for _ in range(25):
        parents, new = step(rng, m)
        written = _i32(m.written)
        want, copies = m.fork(parents, new)
        seen += len(copies)
        if parents is None:
            status = resize_rows(pools, *state, _i32(new), _workspace=ws, written=written)
        else:
            status = fork_rows(pools, *state, _i32(parents), None if new is None else _i32(new), _workspace=ws,
                               written=written)
        assert status.tolist() == [want]
        for _ in range(rng.choice([0, 1, page + 1])):
            at = _i32(m.written)
            values = [m.append(b) if m.next < 2048 and rng.random() < 0.7 else 0 for b in range(B)]  # exact in fp16
            x = _tokens(values)
            paged16_append(*pools, x, -x, state[0], torch.where(_i32(values) > 0, at, -1))
        _check(m, state, pools)


@pytest.mark.parametrize("length", [0, 1, 16, 20, 32])
@pytest.mark.parametrize("room", [0, 1, 20, 100])
def test_children_write_their_own_tokens(length, room):
    """Reserve, write some of it, fork, write different tokens in the children, read them by the decode."""
    from tritonkv_amd.paged16 import paged16_append, paged16_decode_attention
    from tritonkv_amd.pages import fork_rows, resize_rows

    m = Rows(4, 10, 40, 16)
    pools = [torch.zeros(40, HKV, 16, D, dtype=F16, device=DEV) for _ in range(2)]
    state = _i32(m.table), _i32(m.lens), _i32(m.refs)
    m.fork(None, [length + room, 0, 0, 5])
    resize_rows(pools, *state, _i32([length + room, 0, 0, 5]))
    values = [m.append(0) for _ in range(length)]
    if length:
        x = _tokens(values).view(1, length, HKV, D).transpose(1, 2)
        paged16_append(*pools, x, -x, state[0][:1], _i32([0]))
    parents = [0, 0, 0, -1]
    written, new = _i32(m.written), [length + room + 1] * 3 + [0]
    m.fork(parents, new)
    assert fork_rows(pools, *state, _i32(parents), _i32(new), written=written).tolist() == [0]
    for _ in range(room + 1):
        at, values = _i32(m.written), [m.append(b) for b in range(3)]
        x = _tokens(values + [0])
        paged16_append(*pools, x, -x, state[0], torch.where(_i32(values + [0]) > 0, at, -1))
    _check(m, state, pools)
    q = torch.zeros(4, HKV, D, dtype=F16, device=DEV)  # equal scores: the mean of the values
    out = paged16_decode_attention(q, *pools, state[0], _i32(m.written))
    for b in range(4):
        mean = -sum(m.tokens[b]) / max(1, len(m.tokens[b]))
        assert torch.allclose(out[b], torch.full_like(out[b], mean), rtol=1e-5, atol=0)


def test_room_is_kept_by_the_heir_and_captured_steps_follow():
    """Beams over rows with room: nothing is handed out while it lasts, in a replayed graph too."""
    from tritonkv_amd.pages import fork_rows

    m = Rows(6, 8, 64, 16)
    pools = [torch.zeros(64, HKV, 16, D, dtype=F16, device=DEV)]
    m.fork(None, [100, 100, 0, 0, 0, 0])
    for _ in range(40):
        m.append(0), m.append(1)
    pages = [list(r) for r in m.table[:2]]
    state = _i32(m.table), _i32(m.lens), _i32(m.refs)
    parents, written, status, ws = _i32([0, 1, 2, 3, 4, 5]), _i32(m.written), _i32([7]), {}
    fork_rows(pools, *state, parents, status=status, _workspace=ws, written=written)
    m.fork([0, 1, 2, 3, 4, 5])
    assert m.table[:2] == pages and state[0].tolist() == m.table and state[2].tolist() == m.refs
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fork_rows(pools, *state, parents, status=status, _workspace=ws, written=written)
    for p in ([0, 1, 0, 1, -1, -1], [2, 1, 0, 0, 4, 5], [1, 1, 1, 1, 1, 1], [5, 3, -1, 2, 0, 1]):
        parents.copy_(_i32(p))
        written.copy_(_i32(m.written))
        want, _ = m.fork(p)
        graph.replay()
        torch.cuda.synchronize()
        assert status.tolist() == [want] == [0]
        assert state[0].tolist() == m.table and state[1].tolist() == m.lens and state[2].tolist() == m.refs
        for b in range(6):
            m.append(b)


@pytest.mark.parametrize("B,P,N", [(300, 6, 2500), (2000, 4, 9000)])
def test_many_rows_with_room(B, P, N):
    """Plans of four and of sixteen waves, rows past a round of them."""
    from tritonkv_amd.pages import fork_rows

    rng = random.Random(B)
    m = Rows(B, P, N, 16)
    m.fork(None, [rng.randint(0, P * 16) if b % 3 == 0 else 0 for b in range(B)])
    for b in range(0, B, 3):
        for _ in range(rng.randint(0, m.lens[b])):
            m.append(b)
    pools = [torch.zeros(N, 1, 16, 8, dtype=F16, device=DEV)]
    state = _i32(m.table), _i32(m.lens), _i32(m.refs)
    parents = [b - b % 3 if rng.random() < 0.8 else b for b in range(B)]
    written = _i32(m.written)
    want, _ = m.fork(parents)
    assert fork_rows(pools, *state, _i32(parents), written=written).tolist() == [want]
    assert state[0].tolist() == m.table and state[1].tolist() == m.lens and state[2].tolist() == m.refs


def test_counts_outside_the_rows():
    """More tokens than a row holds count as all of them, fewer than none as none."""
    from tritonkv_amd.pages import fork_rows

    for given, clamped in (([99, -5, 2 ** 31 - 1], [20, 0, 5]), ([-2 ** 31, 16, 4], [0, 16, 4])):
        results = []
        for written in (given, clamped):
            m = Rows(3, 4, 20, 16)
            m.fork(None, [20, 40, 5])
            state = _i32(m.table), _i32(m.lens), _i32(m.refs)
            pools = [torch.zeros(20, HKV, 16, D, dtype=F16, device=DEV)]
            assert fork_rows(pools, *state, _i32([1, 1, 0]), written=_i32(written)).tolist() == [0]
            results.append([t.tolist() for t in state])
        assert results[0] == results[1]


def test_quantized_pools_and_more_tensors_than_a_launch_takes():
    from tritonkv_amd.paged import empty_paged_pool, paged_append
    from tritonkv_amd.pages import fork_rows

    m = Rows(3, 4, 14, 32)
    m.fork(None, [100, 0, 0])
    for _ in range(40):
        m.append(0)
    pools = [empty_paged_pool(14, HKV, 32, D, 4, 32, DEV) for _ in range(12)]
    state = _i32(m.table), _i32(m.lens), _i32(m.refs)
    x = torch.randn(1, HKV, 40, D, device=DEV).to(F16)
    for p in pools:
        for t in (p.packed, p.scale, p.zero):
            t.zero_()
        paged_append(p, x, state[0][:1], _i32([0]))
    first = [pools[0].packed[p].clone() for p in m.table[0][:2]]
    written = _i32(m.written)
    want, copies = m.fork([0, 0, 0])
    assert fork_rows(pools, *state, _i32([0, 0, 0]), written=written).tolist() == [want] == [0] and len(copies) == 2
    assert state[0].tolist() == m.table and state[2].tolist() == m.refs
    for p in pools:
        for b in range(3):
            assert torch.equal(p.packed[m.table[b][0]], first[0]) and torch.equal(p.packed[m.table[b][1]], first[1])
        paged_append(p, torch.randn(3, HKV, 1, D, device=DEV).to(F16), state[0], _i32(m.written))
        rows = [p.packed[m.table[b][1]] for b in range(3)]
        assert all(torch.equal(r[:, :8], first[1][:, :8]) for r in rows)
        assert not torch.equal(rows[0][:, 8], rows[1][:, 8]) and not torch.equal(rows[1][:, 8], rows[2][:, 8])


@pytest.mark.parametrize("B", [1, 3, 5, 70, 300])
def test_long_rooms_with_pages_that_others_hold(B):
    """The heir keeps its parent's room up to the first page that is not the parent's alone."""
    from tritonkv_amd.pages import fork_rows

    rng = random.Random(B)
    P = 700 if B < 10 else 90
    m = Rows(B, P, B * P + 50, 16)
    m.fork(None, [rng.randint(0, P * 16) if b % 2 == 0 else 0 for b in range(B)])
    for b in range(0, B, 2):
        for _ in range(min(m.lens[b], rng.choice([0, 16, 20, 100]))):
            m.append(b)
    for b in range(0, B, 4):  # a count of the caller's own on some page of the room
        used = -(-m.lens[b] // 16)
        held = len(m.tokens[b]) // 16
        if used > held:
            m.refs[m.table[b][rng.randint(held, used - 1)]] += 1
    pools = [torch.zeros(m.N, 1, 16, 8, dtype=F16, device=DEV)]
    state = _i32(m.table), _i32(m.lens), _i32(m.refs)
    parents = [b - b % 2 if rng.random() < 0.5 else b for b in range(B)]
    rng.shuffle(parents)
    written = _i32(m.written)
    want, _ = m.fork(parents)
    assert fork_rows(pools, *state, _i32(parents), written=written).tolist() == [want]
    assert state[0].tolist() == m.table and state[1].tolist() == m.lens and state[2].tolist() == m.refs


def test_the_most_rows():
    from tritonkv_amd.pages import fork_rows

    m = Rows(8192, 3, 8192 * 4, 16)
    m.fork(None, [48 if b % 2 == 0 else 0 for b in range(8192)])
    for b in range(0, 8192, 2):
        m.tokens[b] = [1] * (b % 33)
    pools = [torch.zeros(m.N, 1, 16, 8, dtype=F16, device=DEV)]
    state = _i32(m.table), _i32(m.lens), _i32(m.refs)
    parents = [b - b % 2 for b in range(8192)]
    written = _i32(m.written)
    want, _ = m.fork(parents)
    assert want == 0 and fork_rows(pools, *state, _i32(parents), written=written).tolist() == [0]
    assert state[0].tolist() == m.table and state[1].tolist() == m.lens and state[2].tolist() == m.refs
