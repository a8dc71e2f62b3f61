"""A step's tables on the GPU against loops in Python."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(lib):
    from longhornai_amd import ops as _ops
    return _ops


def plan(lengths, new, free, left, table, n, tree=None):
    """The rule in loops: (offsets, positions, slots, left, table, free)."""
    B, W = table.shape
    P, table, free = len(free), table.copy(), free.copy()
    held = [min(max(int(x), 0), 64 * W) for x in lengths]
    stack = list(free[:min(max(left, 0), P)])
    for s in range(B):
        if new[s] < 0:
            for p in table[s, :-(-held[s] // 64)]:
                if 0 <= p < P and len(stack) < P:
                    stack.append(p)
    free[:len(stack)] = stack
    offsets, missing, row = [0], 0, 0
    positions, slots = np.full(n, -1, np.int32), np.full(n, -1, np.int64)
    for s in range(B):
        lo = offsets[-1]
        hi = min(n, lo + max(int(new[s]), 0))
        offsets.append(hi)
        for p in range(-(-held[s] // 64), min(W, -(-(held[s] + hi - lo) // 64)) if hi > lo else 0):
            missing += not stack
            table[s, p] = stack.pop() if stack else -1
        T = min(hi - lo, 64)
        for i in range(hi - lo):
            at = held[s] + i
            depth = i if tree is None else max(bin(int(tree[lo + i]) & ((1 << T) - 1)).count("1") - 1, 0)
            positions[lo + i] = held[s] + depth
            if at // 64 < W and 0 <= table[s, at // 64] < P:
                slots[lo + i] = int(table[s, at // 64]) * 64 + at % 64
    return np.array(offsets, np.int32), positions, slots, np.array([len(stack), missing], np.int32), table, free


class Case:
    def __init__(self, lengths, new, width, spare, seed, n=None, over_full=0):
        g = np.random.default_rng(seed)
        self.lengths, self.new = np.array(lengths, np.int32), np.array(new, np.int32)
        need = [min(width, -(-max(int(t), 0) // 64)) for t in lengths]
        P = sum(need) + spare - over_full
        ids = g.permutation(max(P, 1)).astype(np.int32)
        ids = np.concatenate([ids, ids[:over_full]])
        self.table, at = np.full((len(lengths), width), -1, np.int32), 0
        for s, k in enumerate(need):
            self.table[s, :k] = ids[at:at + k]
            at += k
        self.left = max(P - at, 0)
        self.free = np.full(P, -7, np.int32)
        self.free[:self.left] = ids[at:at + self.left]
        self.n = int(np.maximum(self.new, 0).sum()) if n is None else n
        self.tree = None

    def check(self, ops, in_place=False):
        import torch
        table, free = ops.dev(self.table), ops.dev(self.free)
        left = ops.dev(np.array([self.left, 99], np.int32))
        out = None
        if in_place:
            i32 = dict(dtype=torch.int32, device="cuda")
            out = ops.KvPlan(torch.empty(len(self.new) + 1, **i32), torch.empty(self.n, **i32),
                             torch.empty(self.n, dtype=torch.int64, device="cuda"), left)
        p = ops.kv_plan(ops.dev(self.lengths), ops.dev(self.new), free, left, table, self.n,
                        tree=None if self.tree is None else ops.dev(self.tree), out=out)
        got = [ops.host(x) for x in (p.offsets, p.positions, p.slots, p.left, table, free)]
        want = plan(self.lengths, self.new, self.free, self.left, self.table, self.n, self.tree)
        for name, a, b in zip(("offsets", "positions", "slots", "left", "table", "free"), got, want):
            assert np.array_equal(a, b), (name, np.nonzero(a != b)[0][:5], a.ravel()[:8], b.ravel()[:8])


@pytest.mark.parametrize("lengths,new,width,spare", [
    ([0], [1], 4, 3), ([0], [0], 1, 0), ([63, 64, 65, 0], [1, 1, 1, 1], 4, 3), ([5], [-1], 2, 2),
    ([10, 200, 64, 0, 1], [3, -1, 0, 64, 65], 6, 9), ([128, 128], [-1, -3], 2, 0), ([0, 0, 0], [200, 130, 1], 4, 4),
    ([100, 50], [500, 500], 8, 5), ([500], [700], 8, 40), ([512], [64], 8, 10), ([0, 64], [64, 0], 0 + 1, 5)])
@pytest.mark.parametrize("in_place", [False, True])
def test_small_steps(ops, lengths, new, width, spare, in_place):
    Case(lengths, new, width, spare, seed=1).check(ops, in_place)


@pytest.mark.parametrize("B,top,new,n", [(1, 9000, 1, None), (64, 900, 1, None), (65, 300, 5, None), (300, 700, 1, 400),
                                         (1023, 200, 3, None), (1024, 100, 4, 4096), (1024, 100, 4, 4097),
                                         (1025, 200, 1, None), (3000, 300, 2, None), (7, 3000, 3000, None),
                                         (20, 100, 500, 12000)])
def test_many_requests(ops, B, top, new, n):
    g = np.random.default_rng(B)
    lengths = g.integers(0, top + 1, B)
    count = g.integers(0, new + 1, B)
    count[g.random(B) < 0.15] = -1
    c = Case(lengths, count, 64 if top < 4000 else 160, int(count.clip(0).sum()) // 80 + 5, seed=2, n=n)
    c.check(ops)
    c.check(ops, in_place=True)


def test_rows_past_the_room_are_dropped(ops):
    Case([10, 70, 5], [100, 100, 100], 8, 20, seed=3, n=150).check(ops)
    Case([10, 70, 5], [100, 100, 100], 8, 20, seed=3, n=0).check(ops)
    Case([10, 70], [2 ** 31 - 1, 2 ** 31 - 1], 8, 20, seed=3, n=300).check(ops)


def test_lengths_outside_the_table(ops):
    Case([-5, 10 ** 6, -2 ** 31, 2 ** 31 - 1], [3, 4, -1, -1], 4, 9, seed=4).check(ops)


def test_entries_that_are_no_pages_do_not_go_back(ops):
    c = Case([300, 100], [-1, 200], 8, 3, seed=5)
    c.table[0, 1], c.table[0, 3] = -1, 10 ** 6
    c.check(ops)


def test_pages_handed_back_twice_do_not_overflow_the_stack(ops):
    Case([300, 300, 64], [-1, -1, 130], 5, 4, seed=6, over_full=7).check(ops)


@pytest.mark.parametrize("left", [-3, 10 ** 6])
def test_a_count_outside_the_stack_is_clamped(ops, left):
    c = Case([10, 20], [100, 100], 4, 6, seed=7)
    c.free[:] = np.arange(len(c.free))
    c.left = left
    c.check(ops)


def test_positions_of_drafted_trees(ops):
    c = Case([100, 0, 60], [5, 64, 3], 4, 9, seed=8)
    g = np.random.default_rng(8)
    words = []
    for T in c.new:
        masks = []
        for i in range(T):
            parent = int(g.integers(-1, i)) if i else -1
            masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
        words += masks
    words[2] |= 1 << 63  # past the sequence's last token
    words[4] = 0
    c.tree = np.array([w - (1 << 64) if w >> 63 else w for w in words], np.int64)
    c.check(ops)


def test_no_sequences_and_no_pages(ops):
    import torch
    i32 = dict(dtype=torch.int32, device="cuda")
    p = ops.kv_plan(torch.zeros(0, **i32), torch.zeros(0, **i32), torch.zeros(3, **i32), torch.tensor([2, 0], **i32),
                    torch.zeros((0, 4), **i32), 5)
    assert ops.host(p.offsets).tolist() == [0] and ops.host(p.left).tolist() == [2, 0]
    assert (ops.host(p.positions) == -1).all() and (ops.host(p.slots) == -1).all()
    p = ops.kv_plan(torch.tensor([5], **i32), torch.tensor([3], **i32), torch.zeros(0, **i32), torch.tensor([0, 0], **i32),
                    torch.zeros((1, 0), **i32), 4)
    assert ops.host(p.offsets).tolist() == [0, 3] and ops.host(p.positions).tolist() == [0, 1, 2, -1]
    assert (ops.host(p.slots) == -1).all() and ops.host(p.left).tolist() == [0, 0]


def test_a_captured_loop_keeps_its_tables(ops):
    """Decode steps of one graph: the tables live from replay to replay."""
    import torch
    g0 = np.random.default_rng(9)
    B, W, P = 40, 6, 200
    lengths, new = np.zeros(B, np.int32), np.ones(B, np.int32)
    new[3], new[7] = 0, 70
    free = g0.permutation(P).astype(np.int32)
    table = np.full((B, W), -1, np.int32)
    d = [ops.dev(x) for x in (lengths, new, free, table)]
    left = ops.dev(np.array([P, 0], np.int32))
    n = int(new.sum())
    out = ops.KvPlan(torch.empty(B + 1, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda"),
                     torch.empty(n, dtype=torch.int64, device="cuda"), left)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv_plan(d[0], d[1], d[2], left, d[3], n, out=out)
        d[0].add_(d[1])
    have = P
    for step in range(5):
        g.replay()
        torch.cuda.synchronize()
        o, pos, slots, l, table, free = plan(lengths, new, free, have, table, n)
        lengths, have = lengths + new, int(l[0])
        for a, b in zip((out.offsets, out.positions, out.slots, left, d[3], d[2]), (o, pos, slots, l, table, free)):
            assert np.array_equal(ops.host(a), b)
        torch.zeros(1000, device="cuda").add_(1)


class Steps:
    """Steps on tables that live on, what a sequence has counted in `owned`: each checked against
    the rule in lists, and that every page is on the stack or in one row, once."""

    def __init__(self, ops, B, width, pages, seed):
        g = np.random.default_rng(seed)
        self.ops, self.B, self.W, self.P = ops, B, width, pages
        self.stack = [int(p) for p in g.permutation(pages)]
        self.rows = [[] for _ in range(B)]  # the pages that a sequence has
        self.length = np.zeros(B, np.int64)
        self.table = ops.dev(np.full((B, width), -1, np.int32))
        self.free = ops.dev(np.array(self.stack, np.int32))
        self.left = ops.dev(np.array([pages, 0], np.int32))
        self.owned = ops.dev(np.zeros(B, np.int32))

    def step(self, new, n=None, tree=None):
        """Returns the slots."""
        ops, new = self.ops, np.asarray(new)
        n = int(new.clip(0).sum()) if n is None else n
        p = ops.kv_plan(ops.dev(self.length.astype(np.int32)), ops.dev(new.astype(np.int32)), self.free, self.left,
                        self.table, n, tree=tree, owned=self.owned)
        self.left = p.left
        for s in np.nonzero(new < 0)[0]:
            self.stack += self.rows[s]
            self.rows[s] = []
        missing, slots, lo = 0, np.full(n, -1, np.int64), 0
        for s in range(self.B):
            hi = min(n, lo + max(int(new[s]), 0))
            L, row = int(self.length[s]), self.rows[s]
            for _ in range(len(row), min(self.W, -(-(L + hi - lo) // 64)) if hi > lo else 0):
                missing += not self.stack
                if self.stack:
                    row.append(self.stack.pop())
            for i in range(lo, hi):
                at = L + i - lo
                if at // 64 < len(row):
                    slots[i] = 64 * row[at // 64] + at % 64
            lo = hi
        got, owned, table = ops.host(p.slots), ops.host(self.owned), ops.host(self.table)
        assert np.array_equal(got, slots)
        assert ops.host(p.left).tolist() == [len(self.stack), missing]
        assert owned.tolist() == [len(r) for r in self.rows]
        assert all(table[s, :len(r)].tolist() == r for s, r in enumerate(self.rows))
        assert ops.host(self.free)[:len(self.stack)].tolist() == self.stack
        assert sorted(self.stack + [p for r in self.rows for p in r]) == list(range(self.P))
        return got


def test_rejected_drafts_lose_no_pages(ops):
    """A prompt of 60, then drafts of 8 across the end of its page of which one is kept."""
    t = Steps(ops, 1, 8, 10, seed=10)
    assert (t.step([60]) >= 0).all()
    t.length[0] = 60
    for _ in range(4):
        assert (t.step([8]) >= 0).all()
        t.length[0] += 1
    t.step([-1])
    assert ops.host(t.left).tolist() == [10, 0]


def test_a_shortage_can_be_tried_again(ops):
    t = Steps(ops, 2, 8, 4, seed=11)
    t.step([100, 0])
    t.length[0] = 100
    assert (t.step([1, 300])[1:] >= 0).sum() == 128  # two pages of the five
    t.step([0, 300])                                 # none yet: it keeps the two
    t.step([-1, 300])                                # two more
    t.length[0] = 0
    assert (t.step([0, 256]) >= 0).all()
    t.step([0, -1])
    assert ops.host(t.left).tolist() == [4, 0]


def test_a_request_that_ends_before_its_tokens_were_taken(ops):
    t = Steps(ops, 3, 4, 8, seed=12)
    t.step([130, 64, 1])
    t.step([-1, -1, -1])
    assert ops.host(t.left).tolist() == [8, 0]


def test_a_request_that_stays_over_gives_its_pages_back_once(ops):
    t = Steps(ops, 2, 4, 8, seed=13)
    t.step([130, 64])
    t.length[:] = 130, 64
    for _ in range(3):
        t.step([-1, 0])
    t.step([-1, 200])
    t.length[0] = 0
    t.step([256, 0])
    assert ops.host(t.left).tolist() == [0, 0]


@pytest.mark.parametrize("B,width,pages,steps", [(1, 3, 3, 40), (5, 6, 20, 60), (40, 8, 150, 40), (70, 5, 400, 30),
                                                 (1024, 4, 2000, 8), (1100, 6, 4000, 8), (2500, 4, 3000, 6)])
def test_many_steps_of_drafts_shortages_and_ends(ops, B, width, pages, steps):
    g = np.random.default_rng(B)
    t = Steps(ops, B, width, pages, seed=B)
    for _ in range(steps):
        new = np.where(g.random(B) < 0.3, g.integers(0, 150, B), g.integers(0, 9, B))
        new[g.random(B) < 0.15] = -1
        total = int(new.clip(0).sum())
        slots = t.step(new, n=total if g.random() < 0.7 else int(total * g.random()))
        at = 0
        for s in range(B):
            k = max(int(new[s]), 0)
            stored = slots[at:at + k]
            there = int((stored >= 0).sum())  # the first ones
            assert (stored[:there] >= 0).all()
            at += k
            if new[s] < 0:
                t.length[s] = t.length[s] if g.random() < 0.5 else 0  # (the next step may still say that it is over)
                if t.length[s]:
                    new_over = np.zeros(B, np.int64)
                    new_over[s] = -1
                    if g.random() < 0.2:
                        t.step(new_over)
                    t.length[s] = 0
            else:
                t.length[s] += g.integers(0, there + 1)
    t.step(np.full(B, -1))
    assert ops.host(t.left).tolist() == [pages, 0]


def test_counts_outside_the_row_are_clamped(ops):
    t = Steps(ops, 2, 3, 9, seed=14)
    t.owned.copy_(ops.dev(np.array([-5, -2 ** 31], np.int32)))
    t.step([70, 1])
    t.step([-1, -1])
    import torch
    table = ops.dev(np.array([[4, -1, 7]], np.int32))
    free, left, owned = ops.dev(np.zeros(9, np.int32)), ops.dev(np.array([0, 0], np.int32)), ops.dev(np.array([2 ** 31 - 1], np.int32))
    p = ops.kv_plan(ops.dev(np.zeros(1, np.int32)), ops.dev(np.array([-1], np.int32)), free, left, table, 0, owned=owned)
    assert ops.host(p.left).tolist() == [2, 0] and ops.host(free)[:2].tolist() == [4, 7] and ops.host(owned).tolist() == [0]
    assert torch.equal(table.cpu(), torch.tensor([[4, -1, 7]], dtype=torch.int32))


def test_drafted_trees_with_owned_pages(ops):
    """The tree changes positions, not pages."""
    t = Steps(ops, 1, 4, 6, seed=15)
    t.step([62], tree=ops.dev((1 << np.arange(1, 63, dtype=np.int64)) - 1))
    t.length[0] = 62
    for _ in range(3):
        slots = t.step([4], tree=ops.dev(np.array([1, 3, 5, 9], np.int64)))
        assert (slots >= 0).all()
        t.length[0] += 1
    t.step([-1])
    assert ops.host(t.left).tolist() == [6, 0]


def test_a_captured_loop_with_a_request_that_is_over(ops):
    """The host has not looked yet: replays with the same counts give nothing back twice."""
    import torch
    lengths, new = ops.dev(np.array([100, 60], np.int32)), ops.dev(np.array([-1, 1], np.int32))
    table = ops.dev(np.array([[3, 1, -1, -1], [0, -1, -1, -1]], np.int32))
    free, left = ops.dev(np.array([2, 4, 5, -1, -1, -1], np.int32)), ops.dev(np.array([3, 0], np.int32))
    owned = ops.dev(np.array([2, 1], np.int32))
    i32 = dict(dtype=torch.int32, device="cuda")
    out = ops.KvPlan(torch.empty(3, **i32), torch.empty(1, **i32), torch.empty(1, dtype=torch.int64, device="cuda"), left)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv_plan(lengths, new, free, left, table, 1, out=out, owned=owned)
        lengths[1:].add_(1)
    for step in range(7):
        g.replay()
        torch.cuda.synchronize()
        L = 60 + step
        row = [0] if L < 64 else [0, 1]
        assert ops.host(left).tolist() == [5 if L < 64 else 4, 0]
        assert ops.host(free)[:5 if L < 64 else 4].tolist() == [2, 4, 5, 3, 1][:5 if L < 64 else 4]
        assert ops.host(owned).tolist() == [0, len(row)] and ops.host(table)[1, :len(row)].tolist() == row
        assert ops.host(out.slots).tolist() == [64 * row[L // 64] + L % 64]
        torch.zeros(1000, device="cuda").add_(1)
