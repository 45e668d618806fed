"""Page bookkeeping on the GPU against a plain model in Python integers: copies,
forks, truncation, growth, freeing and compaction, over 16-bit and 2/4-bit
pools; then all of it together with the append and the decode.

Everything here is integers and copied bytes, so every comparison is for
equality."""

from __future__ import annotations

import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16 = torch.float16


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _pool(num_pages, HKV=2, page=16, D=64, seed=0, dtype=F16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(num_pages, HKV, page, D, device=DEV, generator=g).to(dtype)


def _quant_pool(num_pages, HKV=2, page=32, D=64, nbits=4, seed=0):
    from tritonkv_amd.paged import empty_paged_pool

    g = torch.Generator(device=DEV).manual_seed(seed)
    p = empty_paged_pool(num_pages, HKV, page, D, nbits, 32, DEV)
    p.packed.copy_(torch.randint(0, 256, p.packed.shape, device=DEV, generator=g))
    p.scale.copy_(torch.rand(p.scale.shape, device=DEV, generator=g))
    p.zero.copy_(torch.rand(p.zero.shape, device=DEV, generator=g))
    return p


def _bits(t):
    return t.contiguous().view(torch.uint8)


# ---------------------------------------------------------------------------
# copy_pages
# ---------------------------------------------------------------------------


def _copied(src, dst, src_pages, dst_pages, same):
    """The pairs that are carried out."""
    real = [(i, s, d) for i, (s, d) in enumerate(zip(src, dst))
            if 0 <= s < src_pages and 0 <= d < dst_pages and not (same and s == d)]
    read, taken, done = {s for _, s, _ in real} if same else set(), set(), []
    for _, s, d in real:
        if d not in taken and d not in read:
            done.append((s, d))
        taken.add(d)
    return done


@pytest.mark.parametrize("n", [1, 3, 1024, 1025, 2000, 4096, 4097, 10000])
@pytest.mark.parametrize("kind", ["clean", "wild"])
@pytest.mark.parametrize("other", [False, True])
def test_copy_pairs(n, kind, other):
    from tritonkv_amd.pages import copy_pages

    rng = random.Random(n)
    num = max(4100, 2 * n + 4)
    to_num = num // 2 if other else num
    if kind == "clean":
        order = rng.sample(range(num), num)
        src, dst = order[:n], order[n:2 * n] if not other else rng.sample(range(to_num), n)
    else:  # numbers outside, the same page twice, pages both read and written, pairs of one page
        src = [rng.choice([rng.randrange(-3, num + 3), rng.randrange(max(1, n))]) for _ in range(n)]
        dst = [rng.choice([rng.randrange(-3, to_num + 3), rng.randrange(max(1, n)), src[i]]) for i in range(n)]
    pools = [_pool(num, HKV=1, page=16, D=32, seed=1), _pool(num, HKV=1, page=16, D=8, seed=2)]
    to = [torch.zeros_like(p[:to_num]) for p in pools] if other else None
    want = [p.clone() for p in (to or pools)]
    done = _copied(src, dst, num, to_num, not other)
    assert kind == "wild" or len(done) == n
    if done:
        s, d = (torch.tensor(x, device=DEV) for x in zip(*done))
        for w, p in zip(want, pools):
            w[d] = p[s]
    ws = {}
    for _ in range(2):  # again: nothing that was read was written
        copy_pages(pools, _i32(src), _i32(dst), to, _workspace=ws)
        for w, p in zip(want, to or pools):
            assert torch.equal(_bits(p), _bits(w))


@pytest.mark.parametrize("same", [False, True])
def test_long_copies_check_their_pairs_beforehand(same):
    """Over 32 MiB, with every kind of pair that is skipped, and pages of no whole slices."""
    from tritonkv_amd.pages import copy_pages

    rng = random.Random(5)
    num, n = 300, 200
    src = [rng.randrange(-2, num + 2) for _ in range(n)]
    dst = [rng.choice([rng.randrange(-2, num + 2), src[i]]) for i in range(n)]
    pools = [_pool(num, HKV=4, page=48, D=256, seed=1), _pool(num, HKV=3, page=16, D=64, seed=2),
             _pool(num, HKV=8, page=64, D=128, seed=3)]
    assert n * sum(p[0].numel() * 2 for p in pools) > 32 << 20
    to = pools if same else [torch.zeros_like(p) for p in pools]
    want = [p.clone() for p in to]
    done = _copied(src, dst, num, num, same)
    s, d = (torch.tensor(x, device=DEV) for x in zip(*done))
    for w, p in zip(want, pools):
        w[d] = p[s]
    copy_pages(pools, _i32(src), _i32(dst), None if same else to)
    for w, p in zip(want, to):
        assert torch.equal(_bits(p), _bits(w))


def test_copy_quantized_strided_and_many_tensors():
    from tritonkv_amd.pages import copy_pages

    both = torch.randn(20, 2, 2, 16, 64, device=DEV).to(F16)  # K and V of a page side by side
    token_major = torch.randn(20, 16, 2, 64, device=DEV).to(F16).transpose(1, 2)
    big = torch.randn(20, 8, 64, 128, device=DEV)  # 256 KiB pages: 16 slices
    pools = [_quant_pool(20, nbits=2, seed=3), _quant_pool(20, nbits=4, seed=4), both[:, 0], both[:, 1],
             token_major, big] + [_pool(20, seed=5 + i) for i in range(60)]
    flat = [t for p in pools for t in ([p] if isinstance(p, torch.Tensor) else [p.packed, p.scale, p.zero])]
    want = [t.clone() for t in flat]
    src, dst = [3, 19, 7], [0, 11, 18]
    for w in want:
        w[dst] = w[src]
    copy_pages(pools, _i32(src), _i32(dst))
    for t, w in zip(flat, want):
        assert torch.equal(_bits(t), _bits(w))
    copy_pages(pools, _i32([]), _i32([]))


def test_copy_past_32_bit_offsets():
    from tritonkv_amd.pages import copy_pages

    p = torch.zeros(5 << 20, 1, 16, 64, dtype=F16, device=DEV)  # 10 GiB of 2 KiB pages
    last = p.shape[0] - 1
    p[last].fill_(3)
    p[1].fill_(5)
    copy_pages([p], _i32([last, 1]), _i32([2, last - 1]))
    assert (p[2] == 3).all() and (p[last - 1] == 5).all() and not p[3].any()


# ---------------------------------------------------------------------------
# fork_rows, resize_rows
# ---------------------------------------------------------------------------


class Model:
    """The definition, one row at a time."""

    def __init__(self, B, P, N, page):
        self.B, self.P, self.N, self.page = B, P, N, page
        self.table = [[-1] * P for _ in range(B)]
        self.lens = [0] * B
        self.refs = [0] * N

    def used(self, table, lens):
        return [[p for p in row[:-(-n // self.page)] if 0 <= p < self.N] for row, n in zip(table, lens)]

    def fork(self, parents=None, new_lens=None):
        """Status and copies (source, destination)."""
        B, page = self.B, self.page
        cap = self.P * page
        a = [b if parents is None else p if 0 <= p < B else None for b, p in enumerate(parents or range(B))]
        have = [0 if x is None else max(0, min(self.lens[x], cap)) for x in a]
        want = [0 if x is None else h if new_lens is None else max(0, new_lens[b]) for b, (x, h) in enumerate(zip(a, have))]
        if any(n > cap for n in want):
            return 2, []
        keep = [min(h, n) for h, n in zip(have, want)]
        heirs, most = {}, {}
        for b in range(B):
            most[a[b]] = max(most.get(a[b], 0), keep[b] // page)
        for b in range(B):
            f = keep[b] // page
            if keep[b] % page and self.refs[self.table[a[b]][f]] == 1 and f == most[a[b]]:
                if a[b] not in heirs or b == a[b]:
                    heirs[a[b]] = b
        free = [p for p, n in enumerate(self.refs) if n == 0]
        table, copies = [], []
        for b in range(B):
            f, total = keep[b] // page, -(-want[b] // page)
            row = [] if a[b] is None else self.table[a[b]][:f]
            if keep[b] % page:
                last = self.table[a[b]][f]
                if heirs.get(a[b]) == b:
                    row.append(last)
                else:
                    copies.append((last, free[0] if free else None))
            if total - len(row) > len(free):
                return 1, []
            row += free[:total - len(row)]
            free = free[total - (f + (heirs.get(a[b]) == b if keep[b] % page else 0)):]
            table.append(row + [-1] * (self.P - total))
        for row in self.used(self.table, [max(0, min(n, cap)) for n in self.lens]):
            for p in row:
                self.refs[p] -= 1
        self.table, self.lens = table, want
        for row in self.used(table, want):
            for p in row:
                self.refs[p] += 1
        return 0, copies

    def same_as(self, table, lens, refs):
        return table.tolist() == self.table and lens.tolist() == self.lens and refs.tolist() == self.refs


def _state(m):
    return _i32(m.table), _i32(m.lens), _i32(m.refs)


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("workspace", [False, True])
def test_random_lives_of_a_cache(seed, workspace):
    """Rows forked, reordered, cut, grown and freed at random, shortages among it; tables,
    counts and every page's bytes after each step."""
    from tritonkv_amd.pages import fork_rows, resize_rows

    rng = random.Random(seed)
    B = rng.choice([1, 2, 5, 9, 40])
    page = rng.choice([16, 32, 48])
    P = rng.choice([1, 3, 8])
    N = rng.choice([2, B * P // 2 + 1, B * P + 3, 3000])
    m = Model(B, P, N, page)
    pools = [_pool(N, page=page, seed=seed), _pool(N, HKV=1, page=page, D=8, seed=seed + 1)]
    want = [p.clone() for p in pools]
    table, lens, refs = _state(m)
    ws = {} if workspace else None
    seen = set()
    for step in range(25):
        kind = rng.choice(["resize", "fork", "both", "free"])
        parents = [rng.choice([b, b, rng.randrange(-1, B + 1)]) for b in range(B)]
        cap = P * page + (2 if rng.random() < 0.1 else 0)
        sizes = [rng.choice([m.lens[b], rng.randint(-1, cap), rng.randint(0, min(cap, 2 * page)),
                             page * rng.randint(0, P)]) for b in range(B)]
        if kind == "resize":
            want_status, copies = m.fork(None, sizes)
            status = resize_rows(pools, table, lens, refs, _i32(sizes), _workspace=ws)
        else:
            sizes = None if kind != "both" else sizes
            if kind == "free":
                parents = [b if rng.random() < 0.6 else -1 for b in range(B)]
            want_status, copies = m.fork(parents, sizes)
            status = fork_rows(pools, table, lens, refs, _i32(parents), None if sizes is None else _i32(sizes),
                               _workspace=ws)
        seen.add(want_status)
        assert status.tolist() == [want_status], (step, kind)
        assert m.same_as(table, lens, refs), (step, kind, parents, sizes)
        if copies:
            s, d = (torch.tensor(x, device=DEV) for x in zip(*copies))
            for w in want:
                w[d] = w[s]
        for p, w in zip(pools, want):
            assert torch.equal(_bits(p), _bits(w)), (step, kind)


@pytest.mark.parametrize("B,P,N", [(1500, 4, 4000), (8192, 2, 20000), (3, 5000, 70001), (2, 3, 140000)])
def test_large_tables_and_pools(B, P, N):
    """More rows than a round of the plan, and more pages than a round of its masks."""
    from tritonkv_amd.pages import fork_rows, resize_rows

    page = 16
    rng = random.Random(B)
    m = Model(B, P, N, page)
    for p in rng.sample(range(N), N // 3):  # pages kept by somebody else
        m.refs[p] = 1
    if N > 100000:
        m.refs[:N - 5] = [1] * (N - 5)  # the free ones are the last
    pool = _pool(N, HKV=1, page=page, D=8)
    table, lens, refs = _state(m)
    most = min(P * page, 2 * 16 if B > 3 else P * page)
    sizes = [rng.randint(0, most) for _ in range(B)]
    for parents, new in ((None, sizes), ([rng.randrange(B) for _ in range(B)], None)):
        want, copies = m.fork(parents, new)
        before = pool.clone()
        if parents is None:
            status = resize_rows([pool], table, lens, refs, _i32(new))
        else:
            status = fork_rows([pool], table, lens, refs, _i32(parents))
        assert status.tolist() == [want] and m.same_as(table, lens, refs)
        for s, d in copies[:200]:
            assert torch.equal(pool[d], before[s])


def test_strided_table_shared_counts_and_quantized_pools():
    from tritonkv_amd.pages import fork_rows, resize_rows

    m = Model(4, 3, 20, 32)
    m.refs[1] = 5  # kept by the caller
    pools = [_quant_pool(20, seed=1), _quant_pool(20, nbits=2, seed=2)]
    wide = torch.full((4, 10), -9, dtype=torch.int32, device=DEV)
    table = wide[:, 2:5]
    table.fill_(-1)
    _, lens, refs = _state(m)
    m.fork(None, [40, 0, 96, 1])
    assert resize_rows(pools, table, lens, refs, _i32([40, 0, 96, 1])).tolist() == [0]
    assert m.same_as(table, lens, refs) and (wide[:, :2] == -9).all() and (wide[:, 5:] == -9).all()
    flat = [t for p in pools for t in (p.packed, p.scale, p.zero)]
    want = [t.clone() for t in flat]
    _, copies = m.fork([0, 0, 2, 0], [40, 35, 70, 33])
    assert len(copies) == 2
    for w in want:
        for s, d in copies:
            w[d] = w[s]
    status = fork_rows(pools, table, lens, refs, _i32([0, 0, 2, 0]), _i32([40, 35, 70, 33]))
    assert status.tolist() == [0] and m.same_as(table, lens, refs) and refs[1] == 5
    for t, w in zip(flat, want):
        assert torch.equal(_bits(t), _bits(w))


def test_state_in_one_buffer_off_16_bytes():
    """Counts that start anywhere are read one by one."""
    from tritonkv_amd.pages import compact_pages, fork_rows, resize_rows

    m = Model(3, 4, 37, 16)
    pool = _pool(37)
    state = torch.full((1 + 12 + 3 + 37 + 1,), -1, dtype=torch.int32, device=DEV)
    table, lens, refs = state[1:13].view(3, 4), state[13:16], state[17:54]
    lens.zero_()
    refs.zero_()
    assert refs.data_ptr() % 16
    for new in ([20, 64, 5], [33, 0, 17]):
        m.fork(None, new)
        assert resize_rows([pool], table, lens, refs, _i32(new)).tolist() == [0]
        assert m.same_as(table, lens, refs)
    m.fork([0, 0, 2])
    fork_rows([pool], table, lens, refs, _i32([0, 0, 2]))
    _compacted(m)
    compact_pages([pool], table, refs)
    assert m.same_as(table, lens, refs) and state[0] == -1 and state[16] == -1


def test_more_tensors_than_a_launch_takes():
    from tritonkv_amd.pages import compact_pages, fork_rows

    m = Model(3, 4, 30, 16)
    m.fork(None, [20, 40, 0])
    pools = [_pool(30, seed=i) for i in range(70)]
    want = [p.clone() for p in pools]
    table, lens, refs = _state(m)
    _, copies = m.fork([0, 1, 1])
    fork_rows(pools, table, lens, refs, _i32([0, 1, 1]))
    assert m.same_as(table, lens, refs) and copies
    m.fork([-1, 1, 2])
    fork_rows(pools, table, lens, refs, _i32([-1, 1, 2]))
    moves = _compacted(m)
    compact_pages(pools, table, refs)
    assert m.same_as(table, lens, refs) and moves
    for w, p in zip(want, pools):
        for s, d in copies + moves:
            w[d] = w[s]
        assert torch.equal(p, w)


@pytest.mark.parametrize("each", [1, 2, 3, 39])
@pytest.mark.parametrize("extra", [0, 1, 33])
def test_long_forks_and_compactions(each, extra):
    """Over 32 MiB of copies, of 1 to 39 copies of a page, in pages of no whole slices, in as
    many tensors as the smaller argument block takes, one more, and more than a launch takes."""
    from tritonkv_amd.pages import compact_pages, fork_rows

    groups, page = 40 // each, 48
    B = groups * (each + 1)
    N = 2 * B + 7
    m = Model(B, 2, N, page)
    pools = [_pool(N, HKV=1, page=page, D=8, seed=x) for x in range(extra + 1)] + \
        [_pool(N, HKV=12, page=page, D=264, seed=50 + x) for x in range(3)]
    assert groups * each * sum(p[0].numel() * 2 for p in pools) > 32 << 20
    want = [p.clone() for p in pools]
    # the parents among the others; their pages at the upper end
    parents = [b - b % (each + 1) + each // 2 for b in range(B)]
    for g, b in enumerate(sorted(set(parents))):
        m.lens[b], m.table[b][0], m.refs[N - 1 - g] = 20, N - 1 - g, 1
    table, lens, refs = _state(m)
    status, copies = m.fork(parents)
    assert status == 0 and len(copies) == groups * each
    assert fork_rows(pools, table, lens, refs, _i32(parents)).tolist() == [0]
    assert m.same_as(table, lens, refs)
    kept = [b if b % 2 else -1 for b in range(B)]
    assert m.fork(kept) == (0, [])
    assert fork_rows(pools, table, lens, refs, _i32(kept)).tolist() == [0]
    moves = _compacted(m)
    compact_pages(pools, table, refs)
    assert m.same_as(table, lens, refs)
    for w, p in zip(want, pools):
        for pairs in filter(None, (copies, moves)):
            s, d = (torch.tensor(x, device=DEV) for x in zip(*pairs))
            w[d] = w[s]
        assert torch.equal(_bits(p), _bits(w))


def test_a_long_compaction():
    from tritonkv_amd.pages import compact_pages

    N = 150
    pools = [_pool(N, HKV=3, page=48, D=264, seed=x) for x in range(10)]
    want = [p.clone() for p in pools]
    live = list(range(40)) + list(range(90, 150))
    m = Model(4, 25, N, 48)
    for i, p in enumerate(live):
        m.table[i // 25][i % 25], m.refs[p] = p, 1
    m.lens = [25 * 48] * 4
    table, lens, refs = _state(m)
    moves = _compacted(m)
    assert len(moves) == 50 and len(moves) * sum(p[0].numel() * 2 for p in pools) > 32 << 20
    compact_pages(pools, table, refs)
    assert m.same_as(table, lens, refs)
    s, d = (torch.tensor(x, device=DEV) for x in zip(*moves))
    for w, p in zip(want, pools):
        w[d] = w[s]
        assert torch.equal(_bits(p), _bits(w))


def test_broken_tables_stay_inside():
    """Entries and lengths that no call leaves are not followed out of the pools."""
    from tritonkv_amd.pages import compact_pages, fork_rows

    pool = _pool(8)
    before = pool.clone()
    table = _i32([[5, 99, -4], [2 ** 31 - 1, -2 ** 31, 7]])
    lens, refs = _i32([1000, 20]), _i32([0, 0, 1, 0, 0, 1, 0, 1])
    status = fork_rows([pool], table, lens, refs, _i32([1, 0]), _i32([20, 40]))
    assert status.tolist() == [0] and lens.tolist() == [20, 40]
    assert table.tolist() == [[2 ** 31 - 1, 0, -1], [5, 99, 1]]
    # the partial pages -2**31 and -4 are none: nothing is copied into pages 0 and 1
    assert torch.equal(pool, before)
    compact_pages([pool], _i32([[99, -7, 2 ** 31 - 1]]), refs)


# ---------------------------------------------------------------------------
# compact_pages
# ---------------------------------------------------------------------------


def _compacted(m):
    """Compact the model; the moves."""
    live = sum(n > 0 for n in m.refs)
    moves = list(zip([p for p in range(live, m.N) if m.refs[p] > 0], [p for p in range(live) if m.refs[p] <= 0]))
    to = dict(moves)
    m.table = [[to.get(p, p) for p in row] for row in m.table]
    for s, d in moves:
        m.refs[d], m.refs[s] = m.refs[s], 0
    return moves


@pytest.mark.parametrize("N,share", [(1, 0.0), (1, 1.0), (7, 0.5), (64, 0.5), (1000, 0.1), (1000, 0.9),
                                     (4097, 0.5), (70000, 0.4), (131077, 0.02)])
@pytest.mark.parametrize("into", ["place", "out"])
def test_compaction(N, share, into):
    from tritonkv_amd.pages import compact_pages

    rng = random.Random(N)
    live = rng.sample(range(N), int(N * share))
    P = max(1, len(live) // 3 + 1)
    m = Model(5, P, N, 16)
    for b in range(3):
        m.table[b][:len(live[b::3])] = live[b::3]
    m.table[3][:min(P, len(live))] = live[:P]  # shared pages
    m.table[4][0] = rng.randrange(N)           # a stale entry of a free row
    for p in live:
        m.refs[p] = rng.randint(1, 4)
    pools = [_pool(N, HKV=1, page=16, D=8, seed=N), _pool(N, HKV=1, page=16, D=16, seed=N + 1)]
    want = [p.clone() for p in pools]
    table, lens, refs = _state(m)
    old = table.clone(), refs.clone()
    out = None if into == "place" else (torch.empty_like(table), torch.empty_like(refs))
    ws = {}
    moves = _compacted(m)
    if moves:
        s, d = (torch.tensor(x, device=DEV) for x in zip(*moves))
        for w in want:
            w[d] = w[s]
    for _ in range(2):
        t, r, n = compact_pages(pools, table, refs, out=out, _workspace=ws)
        assert n.tolist() == [len(live)] and t.tolist() == m.table and r.tolist() == m.refs
        for p, w in zip(pools, want):
            assert torch.equal(_bits(p), _bits(w))
        if into == "out":
            assert torch.equal(table, old[0]) and torch.equal(refs, old[1])
        else:
            assert t is table and r is refs  # the second time there is nothing to do
    assert not r[len(live):].any() and (r[:len(live)] > 0).all()


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------


def test_captured_step_of_a_beam_search():
    """A graph of fork, growth, append and decode, replayed with new choices and tokens."""
    from tritonkv_amd.pages import fork_rows, resize_rows
    from tritonkv_amd.paged16 import paged16_decode_attention

    B, P, page, N, D = 6, 8, 16, 60, 64
    m = Model(B, P, N, page)
    m.fork(None, [50, 50, 50, 33, 33, 33])
    pools = [_pool(N, page=page, D=D, seed=s) for s in (1, 2)]
    table, lens, refs = _state(m)
    parents, new_lens = _i32(range(B)), lens.clone()
    q, kn, vn = (torch.zeros(B, h, D, dtype=F16, device=DEV) for h in (4, 2, 2))
    out, status = torch.empty(B, 4, D, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ws = {}

    def step():
        fork_rows(pools, table, lens, refs, parents, new_lens, status=status, _workspace=ws.setdefault(0, {}))
        paged16_decode_attention(q, *pools, table, lens, out=out, _workspace=ws.setdefault(1, {}), k_new=kn, v_new=vn)

    rows = [[pools[i].clone()[torch.tensor(m.table[b], device=DEV)].transpose(0, 1).reshape(2, -1, D)[:, :m.lens[b]]
             for b in range(B)] for i in range(2)]
    saved = [t.clone() for t in (table, lens, refs, *pools)]
    step()  # allocates the workspaces
    for t, s in zip((table, lens, refs, *pools), saved):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator(device=DEV).manual_seed(7)
    rng = random.Random(7)
    for n in range(6):
        choice = [rng.randrange(3) for _ in range(3)] + [3 + rng.randrange(3) for _ in range(3)]
        parents.copy_(_i32(choice))
        new_lens.copy_(lens[parents.long()] + 1)
        for t in (q, kn, vn):
            t.copy_(torch.randn(t.shape, device=DEV, generator=g))
        assert m.fork(choice, [m.lens[a] + 1 for a in choice])[0] == 0
        graph.replay()
        torch.cuda.synchronize()
        assert status.tolist() == [0] and m.same_as(table, lens, refs), n
        rows = [[torch.cat([r[a], new[b][:, None]], 1) for b, a in enumerate(choice)] for r, new in zip(rows, (kn, vn))]
        for b in range(B):
            s = torch.matmul(q[b].double().view(2, 2, D), rows[0][b].double().transpose(1, 2).contiguous()) / D ** 0.5
            want = torch.matmul(torch.softmax(s, -1), rows[1][b].double()).view(4, D)
            assert torch.allclose(out[b].double(), want, atol=1e-5, rtol=0), (n, b)
    assert resize_rows(pools, table, lens, refs, _i32([0] * B)).tolist() == [0]
    assert not refs.any() and (table == -1).all()


def test_quantized_cache_forked_compacted_and_decoded():
    """2/4-bit pools: rows that share a prefix decode as their own contiguous caches do."""
    from tritonkv_amd.kernels import fused_decode_attention
    from tritonkv_amd.paged import empty_paged_pool, paged_append, paged_decode_attention
    from tritonkv_amd.pages import compact_pages, fork_rows, resize_rows
    from tritonkv_amd.quantize import quantize_kv

    B, HKV, page, D, N, P = 4, 2, 32, 128, 40, 6
    pools = [empty_paged_pool(N, HKV, page, D, 4, 32, DEV) for _ in range(2)]
    for p in pools:
        for t in (p.packed, p.scale, p.zero):
            t.zero_()
    table = torch.full((B, P), -1, dtype=torch.int32, device=DEV)
    lens, refs = torch.zeros(B, dtype=torch.int32, device=DEV), torch.zeros(N, dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(3)
    prompt = torch.randn(2, 1, HKV, 75, D, device=DEV, generator=g).to(F16)
    assert resize_rows(pools, table, lens, refs, _i32([75, 160, 0, 0])).tolist() == [0]
    for p, x in zip(pools, prompt):
        paged_append(p, x, table[:1], _i32([0]))
    assert fork_rows(pools, table, lens, refs, _i32([0, -1, 0, 0]), _i32([85, 0, 85, 85])).tolist() == [0]
    tails = torch.randn(2, B, HKV, 10, D, device=DEV, generator=g).to(F16)
    for p, x in zip(pools, tails):
        for b in (0, 2, 3):
            paged_append(p, x[b:b + 1], table[b:b + 1], _i32([75]))
    _, _, live = compact_pages(pools, table, refs)
    assert live.tolist() == [2 + 3] and int(table.max()) == 4
    q = torch.randn(B, 8, D, device=DEV, generator=g).to(F16)
    got = paged_decode_attention(q[:1].expand(3, 8, D).contiguous(), *pools, table[[0, 2, 3]].contiguous(), _i32([85] * 3))
    for i, b in enumerate((0, 2, 3)):
        kv = [torch.cat([x[0], t[b]], 1)[None] for x, t in zip(prompt, tails)]
        kq, vq = quantize_kv(kv[0].contiguous(), kv[1].contiguous(), 4, 32)
        want = fused_decode_attention(q[:1], kq, vq)
        assert torch.allclose(got[i], want[0], atol=2e-3, rtol=0)


def test_another_stream_and_repeated_calls():
    from tritonkv_amd.pages import fork_rows

    m = Model(3, 4, 30, 16)
    m.fork(None, [20, 40, 0])
    pools = [_pool(30, seed=1)]
    table, lens, refs = _state(m)
    ws, status = {}, torch.zeros(1, dtype=torch.int32, device=DEV)
    parents = _i32([0, 1, 1])
    fork_rows(pools, table, lens, refs, parents, status=status, _workspace=ws)
    m.fork([0, 1, 1])
    prep = ws["call"]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.empty(1 << 26, device=DEV).zero_()  # the call has to wait for its own stream
        lens.add_(big[0].to(torch.int32))
        got = fork_rows(pools, table, lens, refs, _i32([1, 2, -1]), _workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    m.fork([1, 2, -1])
    assert ws["call"] is prep and got is not status and got.tolist() == [0]
    assert m.same_as(table, lens, refs)
    with pytest.raises(ValueError):
        fork_rows(pools, table, lens.long(), refs, parents, _workspace=ws)


def test_a_kept_call_checks_that_its_tensors_lie_apart():
    from tritonkv_amd.pages import compact_pages, fork_rows

    m = Model(2, 4, 30, 16)
    pools = [_pool(30, seed=2)]
    table, lens, refs = _state(m)
    ws = {}
    for new in ([20, 40], [40, 20]):
        assert fork_rows(pools, table, lens, refs, _i32([0, 1]), _i32(new), _workspace=ws).tolist() == [0]
        m.fork([0, 1], new)
    prep = ws["call"]
    with pytest.raises(ValueError, match="share memory"):
        fork_rows(pools, table, lens, refs, _i32([0, 1]), lens, _workspace=ws)
    with pytest.raises(ValueError, match="share memory"):
        fork_rows(pools, table, lens, refs, _i32([0, 1]), _i32([9, 9]), status=refs[5:6], _workspace=ws)
    both = _i32([0, 1, 9, 9])
    with pytest.raises(ValueError, match="share memory"):
        fork_rows(pools, table, lens, refs, both[:2], both[2:], status=both[1:2], _workspace=ws)
    same = _i32([1, 0])  # read twice: no fault
    assert fork_rows(pools, table, lens, refs, same, same, _workspace=ws).tolist() == [0]
    m.fork([1, 0], [1, 0])
    assert ws["call"] is prep and m.same_as(table, lens, refs)
    ws = {}
    for _ in range(2):  # in place: the tables are read and written
        compact_pages(pools, table, refs, _workspace=ws)
    with pytest.raises(ValueError, match="share memory"):
        compact_pages(pools, table, refs, live=refs[3:4], _workspace=ws)
