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
