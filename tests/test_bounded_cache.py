"""The operators of a bounded cache against plain implementations in 64 bits: attention that adds up every cached row's weight,
the choice of the rows that stay, and their move; alone, refused, and one after another as a program uses them."""
import math
import random
import types

import pytest
import torch

from conftest import require_gpu

DEV = "cuda:0"
PAGE = 64
NAN = float("nan")


@pytest.fixture(scope="module")
def ops():
    require_gpu()
    from hilbert_pruned_8b_b200.kernels.ops import Ops
    return Ops(torch.device(DEV))


# ------------------------------------------------------------------------------------------------------- inputs
def _pages(n):
    return (n + PAGE - 1) // PAGE


def _tables(lengths, seed, extra=2, width=None):
    rng = random.Random(seed)
    total = sum(_pages(n) for n in lengths) + extra
    order = list(range(total))
    rng.shuffle(order)
    width = width or max(1, max(_pages(n) for n in lengths))
    rows = []
    for n in lengths:
        mine = [order.pop() for _ in range(_pages(n))]
        rows.append(mine + [-1] * (width - len(mine)))
    return torch.tensor(rows, dtype=torch.int32, device=DEV), total, order


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _step(past, new, table):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    lens = [p + n for p, n in zip(past, new)]
    return types.SimpleNamespace(
        num_tokens=sum(new), num_seqs=len(new), page_tables=[table], positions=_ints([p + i for p, n in zip(past, new) for i in range(n)]),
        tok_seq=_ints([b for b, n in enumerate(new) for _ in range(n)]), seq_start=_ints(starts), seq_pos0=_ints(past), seq_len=_ints(lens),
        max_new=max(new), max_len=max(lens), is_decode=all(n == 1 for n in new), host_new=list(new), host_len=lens, shared={}, tag="")


class Case:
    """Queries as the first columns of wider rows, a paged cache whose rows behind the sequences' ends hold NaN."""

    def __init__(self, dtype, heads, kv, hd, past, new, window, seed=0, strong=1.0, garbage=NAN):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.dtype, self.heads, self.kv, self.hd, self.window = dtype, heads, kv, hd, window
        self.past, self.new = list(past), list(new)
        self.lens = [p + n for p, n in zip(past, new)]
        self.table, self.pages, _ = _tables(self.lens, seed)
        T = sum(new)
        # one more head than is used: rows are further apart than the queries are wide
        self.qkv = (torch.randn(T, (heads + 1) * hd, generator=g, device=DEV) * strong).to(dtype)
        self.k = torch.full((self.pages, kv, PAGE, hd), garbage, dtype=dtype, device=DEV)
        self.v = torch.full((self.pages, kv, PAGE, hd), garbage, dtype=dtype, device=DEV)
        for b, n in enumerate(self.lens):
            j = torch.arange(n, device=DEV)
            page = self.table[b].long()[j // PAGE]
            self.k[page, :, j % PAGE] = torch.randn(n, kv, hd, generator=g, device=DEV).to(dtype)
            self.v[page, :, j % PAGE] = torch.randn(n, kv, hd, generator=g, device=DEV).to(dtype)
        self.before = torch.rand(self.pages, kv, PAGE, generator=g, device=DEV) * 3
        self.step = _step(self.past, self.new, self.table)
        self.cache = types.SimpleNamespace(k=self.k, v=self.v, group=0, window=window)
        self.scale = 1.0 / math.sqrt(hd)

    def run(self, ops, mass, before=None, out=None, **kw):
        if out is None:
            out = torch.full((sum(self.new), self.heads * self.hd), 7.0, dtype=self.dtype, device=DEV)
        ops.attention_mass(self.qkv, self.heads, self.kv, self.hd, self.cache, self.step, out, self.scale, self.window, mass, before=before, **kw)
        return out

    def check(self, out, mass, before, start):
        """``start``: what ``mass`` held before the call."""
        G, t0, u = self.heads // self.kv, 0, 2.0 ** -24
        untouched = torch.ones_like(mass, dtype=torch.bool)
        for b, (p0, n) in enumerate(zip(self.past, self.new)):
            ln = p0 + n
            j = torch.arange(ln, device=DEV)
            page = self.table[b].long()[j // PAGE]
            i = torch.arange(p0, ln, device=DEV)
            hidden = j[None] > i[:, None]
            if self.window:
                hidden |= j[None] <= i[:, None] - self.window
            untouched[page, :, j % PAGE] = False
            for g in range(self.kv):
                k, v = self.k[page, g, j % PAGE].double(), self.v[page, g, j % PAGE].double()
                total, slack = torch.zeros(ln, dtype=torch.float64, device=DEV), torch.zeros(ln, dtype=torch.float64, device=DEV)
                for h in range(g * G, (g + 1) * G):
                    q = self.qkv[t0: t0 + n, h * self.hd: (h + 1) * self.hd].double()
                    w = torch.softmax((q @ k.T * self.scale).masked_fill(hidden, -math.inf), dim=-1)
                    # A score is a sum of hd products in 32 bits: off by at most hd steps of the sum of their sizes, B at
                    # most (the tensor cores' accumulation counts as two of them).  In units of log 2 it is rounded again, and so is
                    # the log-sum, at most B log2(e) + log2(rows) large: a weight's relative error is at most
                    rel = 0.0
                    if n:
                        B = float((q.abs() @ k.abs().T).max()) * self.scale
                        rel = 2 * (2 * self.hd + 8) * u * B + 4 * u * (1.45 * B + math.log2(ln + 1)) + 16 * u
                    total += w.sum(0)
                    slack += w.sum(0) * rel
                    got = out[t0: t0 + n, h * self.hd: (h + 1) * self.hd].double()
                    want, size = w @ v, w @ v.abs()
                    # a weight's error, its rounding for the product, the order of a sum of ln terms, the result's rounding
                    half = torch.finfo(self.dtype).eps / 2
                    tol = size * (2 * rel + (half if self.dtype == torch.bfloat16 else 0.0) + (ln + 16) * u) + want.abs() * half + 1e-30
                    assert torch.isfinite(got).all()
                    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())
                if before is not None:
                    old = torch.where(j < p0, before[page, g, j % PAGE], torch.zeros_like(before[page, g, j % PAGE])).double()
                    total += old
                got = mass[page, g, j % PAGE].double()
                tol = slack + total.abs() * (n * G + 20) * u + 1e-30
                assert torch.isfinite(got).all()
                assert bool(((got - total).abs() <= tol).all()), float(((got - total).abs() / tol).max())
            t0 += n
        assert torch.equal(mass[untouched], start[untouched])         # rows of nobody stay as they were


MANY = [
    # heads, kv heads, head size, rows before, new tokens, window
    (4, 2, 64, [0], [9], None),
    (4, 2, 64, [0, 63, 64, 65], [64, 65, 1, 63], None),
    (8, 2, 128, [0, 1000], [200, 300], None),
    (3, 1, 128, [129, 0, 700], [127, 128, 1], None),
    (6, 3, 128, [500, 0], [300, 257], 100),
    (2, 2, 64, [1000, 3], [40, 700], 1),
    (16, 1, 64, [10], [150], None),
    (17, 1, 64, [100], [30], 64),
    (6, 2, 80, [0, 333], [190, 75], 200),
    (5, 1, 33, [70, 0], [12, 130], None),
    (2, 1, 256, [100], [70], None),
    (4, 4, 200, [0, 64], [64, 100], 65),
    (1, 1, 8, [0], [10], None),
    (4, 2, 128, [9000], [20], None),             # few rows, many keys: the keys are shared out
    (3, 1, 64, [5000, 100], [30, 10], 2000),
    (8, 8, 64, [0, 300], [513, 129], None),
    (6, 2, 128, [0, 131], [400, 255], 130),
    (24, 8, 72, [0, 130], [290, 11], None),      # head sizes between the tensor cores' tiles
    (4, 2, 120, [300, 0], [30, 140], 90),
    (6, 1, 56, [1000], [129], None),
    (2, 1, 16, [0, 5000], [300, 20], None),
]
FEW = [
    (4, 2, 64, [0], [1], None),
    (4, 2, 64, [62, 63, 64, 65, 127, 128], [1, 1, 1, 1, 1, 1], None),
    (32, 8, 128, [3000, 1, 511], [1, 1, 1], None),
    (32, 8, 64, [2999], [1], None),
    (3, 1, 128, [900, 0, 64], [3, 8, 1], None),
    (16, 1, 64, [700, 30], [2, 5], 100),
    (17, 1, 64, [700], [1], None),
    (40, 1, 128, [300], [8], 33),
    (6, 2, 80, [1500, 7], [1, 1], 1),
    (5, 5, 33, [200, 0], [4, 2], None),
    (2, 1, 256, [513], [1], 4096),
    (2, 2, 200, [100, 5000], [1, 2], 70),
    (32, 1, 128, [500, 64], [1, 1], None),
    (33, 1, 64, [500], [1], None),
    (6, 2, 128, [2000, 0, 61, 63], [8, 7, 6, 1], 50),
    (12, 1, 64, [130, 1000], [3, 8], None),
    (16, 2, 152, [1434, 31, 32], [1, 1, 1], None),
    (3, 1, 20, [40, 95], [7, 8], 30),
    (7, 1, 1, [70], [3], None),
    (24, 8, 112, [1500, 63], [1, 1], None),
    (8, 2, 72, [700, 5], [5, 8], 300),
    (3, 1, 8, [200, 64], [1, 2], None),
    (20, 1, 40, [130], [1], None),
]
TYPES = [torch.bfloat16, torch.float32]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,hd,past,new,window", MANY + FEW)
def test_attention_mass(ops, dtype, heads, kv, hd, past, new, window):
    c = Case(dtype, heads, kv, hd, past, new, window, seed=hd + len(past))
    start = torch.full((c.pages, kv, PAGE), 5.0, device=DEV)
    mass = start.clone()
    out = c.run(ops, mass, before=c.before)
    c.check(out, mass, c.before, start)
    # this step's weights alone; then a running sum, in place
    alone = start.clone()
    out2 = c.run(ops, alone)
    c.check(out2, alone, None, start)
    assert torch.equal(out, out2)
    running = c.before.clone()
    c.run(ops, running, before=running)
    seen = mass != start
    assert torch.equal(running[seen], mass[seen])
    again = start.clone()
    assert torch.equal(c.run(ops, again, before=c.before), out) and torch.equal(again, mass)      # the same bits
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv,hd,past,new,window,splits", [
    (8, 2, 128, [0, 1000], [200, 300], None, 1), (8, 2, 128, [0, 1000], [200, 300], None, 5), (6, 3, 64, [500, 0], [300, 257], 100, 7),
    (6, 2, 80, [0, 333], [190, 75], 200, 3), (8, 2, 128, [3000, 10], [1, 1], None, 1), (8, 2, 128, [3000, 10], [2, 8], None, 16),
    (6, 2, 80, [1500, 7], [1, 1], 100, 24)])
def test_shares_of_the_work(ops, dtype, heads, kv, hd, past, new, window, splits):
    """More shares than pages or tiles of queries, and one: the same sums."""
    c = Case(dtype, heads, kv, hd, past, new, window, seed=5)
    start = torch.zeros(c.pages, kv, PAGE, device=DEV)
    mass = start.clone()
    c.check(c.run(ops, mass, before=c.before, splits=splits), mass, c.before, start)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("most", [1, 3, 20])
def test_many_sequences(ops, dtype, most):
    """More sequences than a warp has lanes, some of them without new tokens, one much longer than the others."""
    rng = random.Random(most)
    past = [rng.choice([0, 1, 63, 64, 100]) for _ in range(70)]
    new = [rng.randint(0, most) if p else rng.randint(1, most) for p in past]
    new[-1] = most
    past[40] = 3000
    c = Case(dtype, 4, 2, 64, past, new, None, seed=most)
    start = torch.zeros(c.pages, 2, PAGE, device=DEV)
    mass = start.clone()
    c.check(c.run(ops, mass, before=c.before), mass, c.before, start)
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [[70, 5], [1, 1]])
def test_peaked_and_flat_rows(ops, dtype, new):
    """Scores far apart (one row has nearly all the weight) and all alike."""
    for strong in (30.0, 0.0):
        c = Case(dtype, 8, 2, 128, [300, 64], new, None, seed=9, strong=strong)
        mass = torch.zeros(c.pages, 2, PAGE, device=DEV)
        c.check(c.run(ops, mass), mass, None, torch.zeros_like(mass))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[90, 3], [1, 1]])
def test_output_rows_apart_and_unaligned_queries(ops, new):
    c = Case(torch.bfloat16, 4, 2, 64, [100, 70], new, None, seed=3)
    T = sum(new)
    wide = torch.zeros(T, 4 * 64 + 24, dtype=torch.bfloat16, device=DEV)
    mass = torch.zeros(c.pages, 2, PAGE, device=DEV)
    out = c.run(ops, mass, out=wide[:, 8: 8 + 256])
    c.check(out, mass, None, torch.zeros_like(mass))
    assert not wide[:, :8].any() and not wide[:, 264:].any()
    odd = torch.zeros(T, 4 * 64 + 3, dtype=torch.bfloat16, device=DEV)            # rows at odd places of memory
    odd[:, 1:257] = c.qkv[:, :256]
    was, c.qkv = c.qkv, odd[:, 1:]
    m2 = torch.zeros_like(mass)
    got = c.run(ops, m2)
    c.qkv = was
    c.check(got, m2, None, torch.zeros_like(mass))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 1, 50])
@pytest.mark.parametrize("dtype,heads,kv,hd,past,new", [
    (torch.bfloat16, 8, 2, 64, [0, 383, 64, 5], [1, 1, 1, 1]), (torch.bfloat16, 32, 1, 64, [380], [1]), (torch.bfloat16, 6, 2, 80, [252, 0], [4, 1]),
    (torch.bfloat16, 8, 8, 128, [63, 128, 9], [8, 2, 8]), (torch.float32, 8, 1, 64, [63, 0], [1, 1]), (torch.float32, 3, 3, 7, [61, 40], [3, 2]),
    (torch.bfloat16, 4, 2, 256, [60] * 40, [4] * 40)])
def test_short_sequences_in_one_kernel(ops, dtype, heads, kv, hd, past, new, window):
    """A block with a whole sequence gives what two kernels give, bit for bit: one share, the same order of sums."""
    c = Case(dtype, heads, kv, hd, past, new, window, seed=6)
    start = torch.randn(c.pages, kv, PAGE, device=DEV)
    two, one, was = start.clone(), start.clone(), ops.launches
    want = c.run(ops, two, before=c.before, splits=1)
    assert ops.launches == was + 2
    got = c.run(ops, one, before=c.before)
    assert ops.launches == was + 3
    c.check(got, one, c.before, start)
    assert torch.equal(got, want) and torch.equal(one, two)
    own = c.before.clone()                                   # a running sum in place
    c.run(ops, own, before=own)
    held = two != start
    assert torch.equal(own[held], two[held])
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,heads,kv,hd,window", [(torch.bfloat16, 8, 2, 64, None), (torch.bfloat16, 6, 2, 80, 100), (torch.float32, 4, 2, 33, None)])
@pytest.mark.parametrize("past,new", [
    ([700, 3, 64, 0, 5000, 200, 1], [1, 1, 1, 1, 1, 1, 1]), ([700, 3, 64, 300, 5000, 200, 1], [2, 1, 8, 0, 3, 1, 5]),
    ([40, 3, 64, 0, 20], [1, 1, 1, 1, 1]), ([700, 900, 64, 300, 2000], [0, 3, 1, 1, 0]), ([100, 3000], [1, 0])])
def test_sequences_in_groups(ops, dtype, heads, kv, hd, window, past, new):
    """Scores of a few rows at a time: sequences run one group after another through the same scratch."""
    from hilbert_pruned_8b_b200.kernels.plan import few_groups
    c = Case(dtype, heads, kv, hd, past, new, window, seed=12)
    start = torch.randn(c.pages, kv, PAGE, device=DEV)
    for limit in (1, heads * 2 * 800, heads * 4 * 5100):
        # (a limit below one sequence's scores would send several tokens to the kernels for many)
        ops.MASS_SCORES = max(limit, heads * c.step.max_new * c.step.max_len) if c.step.max_new > 1 else limit
        groups, mass, again, own = few_groups(c.new, c.lens, heads, ops.MASS_SCORES), start.clone(), start.clone(), c.before.clone()
        ops.call_log, log = [], ops.call_log
        try:
            c.check(c.run(ops, mass, before=c.before), mass, c.before, start)
            assert limit > 1 or c.step.max_new > 1 or len(groups) == sum(n > 0 for n in new)
            assert sum(new) == len(new) or ops.call_log == ["hb_attention_mass_few"] * len(groups)
            c.run(ops, again, before=c.before)
            c.run(ops, own, before=own)
        finally:
            ops.call_log = log
            del ops.MASS_SCORES
        assert torch.equal(again, mass) and torch.equal(own[mass != start], mass[mass != start])
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.float32, 33)])
def test_groups_name_the_sequence_of_a_missing_page(ops, dtype, hd):
    """The number in the message is the sequence's in the step, not in its group."""
    from hilbert_pruned_8b_b200.kernels.ops import KernelError
    c = Case(dtype, 4, 2, hd, [100, 200, 150, 300, 90], [1, 2, 1, 1, 1], None, seed=1, garbage=0.0)
    c.table[3, 2] = -1
    ops.MASS_SCORES = 4 * 2 * 320
    try:
        ops.reset_status()
        c.run(ops, torch.zeros(c.pages, 2, PAGE, device=DEV))
        with pytest.raises(KernelError, match="sequence 3 of a step"):
            ops.check_errors()
    finally:
        del ops.MASS_SCORES
        ops.reset_status()


@pytest.mark.gpu
def test_scores_of_one_long_sequence_among_short_ones(ops):
    """64 single tokens, one of them behind 131072 rows: scratch within its limit, captured and eager."""
    past = [50 + b for b in range(64)]
    past[20] = 131072
    c = Case(torch.bfloat16, 32, 1, 64, past, [1] * 64, None, seed=3, garbage=0.0)
    mass, out = torch.zeros(c.pages, 1, PAGE, device=DEV), torch.empty(64, 32 * 64, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    c.run(ops, mass, out=out)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() - held < 300 << 20
    want, sums = out.clone(), mass.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(ops, mass, out=out)
    out.zero_(), mass.zero_()
    graph.replay()
    assert torch.equal(out, want) and torch.equal(mass, sums)
    c.check(out, mass, None, torch.zeros_like(mass))
    ops.check_errors()


@pytest.mark.gpu
def test_many_drafted_tokens_of_a_sequence_too_long_for_its_scores(ops):
    """Several tokens of one sequence whose scores alone are above the limit: the kernels that keep none."""
    c = Case(torch.bfloat16, 8, 2, 64, [900, 100], [5, 2], None, seed=3)
    mass = torch.zeros(c.pages, 2, PAGE, device=DEV)
    ops.MASS_SCORES = 8 * 5 * 800
    try:
        ops.call_log, log = [], ops.call_log
        c.check(c.run(ops, mass, before=c.before), mass, c.before, torch.zeros_like(mass))
        assert ops.call_log == ["hb_attention_mass_tc"]
    finally:
        ops.call_log = log
        del ops.MASS_SCORES
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[90, 3], [1, 2]])
def test_a_sequence_without_new_tokens(ops, new):
    """Rows of a sequence that brings nothing keep their earlier sum."""
    c = Case(torch.bfloat16, 4, 2, 64, [100, 30, 70], [new[0], 0, new[1]], None, seed=4)
    start = torch.zeros(c.pages, 2, PAGE, device=DEV)
    mass = start.clone()
    c.check(c.run(ops, mass, before=c.before), mass, c.before, start)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[90], [1]])
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.bfloat16, 80), (torch.float32, 64)])
def test_attention_mass_notes_a_missing_page(ops, dtype, hd, new):
    from hilbert_pruned_8b_b200.kernels.ops import KernelError
    for bad in (-1, 10 ** 6):
        c = Case(dtype, 4, 2, hd, [200], new, None, seed=1, garbage=0.0)
        c.table[0, 1] = bad
        ops.reset_status()
        c.run(ops, torch.zeros(c.pages, 2, PAGE, device=DEV))
        with pytest.raises(KernelError, match="page"):
            ops.check_errors()
    ops.reset_status()
    # a page in front of every token's window was given back: nobody's fault, and its rows have no place
    c = Case(dtype, 4, 2, hd, [200], new, 20, seed=1, garbage=0.0)
    mass = torch.zeros(c.pages, 2, PAGE, device=DEV)
    want = c.run(ops, mass.clone())
    c.table[0, 0] = -1
    assert torch.equal(c.run(ops, mass), want)
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[300], [90], [5], [1]])
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.bfloat16, 80), (torch.float32, 64)])
def test_pages_given_back_in_front_of_the_window(ops, dtype, hd, new):
    """Pages that no token sees any more may be gone from the table, whatever the cache holds elsewhere (NaN here, in page 0 too)."""
    seed = next(s for s in range(100) if 0 not in _tables([700 + new[0]], s)[0].tolist()[0])
    c = Case(dtype, 6, 2, hd, [700], new, 100, seed=seed)
    start = torch.zeros(c.pages, 2, PAGE, device=DEV)
    full = start.clone()
    want = c.run(ops, full, before=c.before)
    gone = (700 - 100 + 1) // PAGE                       # whole pages in front of the oldest row that the first token sees
    freed = c.table[0, :gone].clone()
    c.table[0, :gone] = -1
    mass = start.clone()
    got = c.run(ops, mass, before=c.before)
    assert torch.isfinite(got).all() and torch.equal(got, want)
    full[freed.long()] = 0.0
    assert torch.equal(mass, full)
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("past,window", [(700, 100), (700, 1), (150, 20), (5000, 1500)])
@pytest.mark.parametrize("new", [[300], [90], [5], [1]])
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.bfloat16, 80), (torch.bfloat16, 200), (torch.float32, 64)])
def test_rows_in_front_of_the_window_do_not_count(ops, dtype, hd, new, past, window):
    """Rows that no token sees any more may hold anything, those of the first visible page too: NaN and infinities there change no bit."""
    c = Case(dtype, 6, 2, hd, [past], new, window, seed=4)
    start = torch.randn(c.pages, 2, PAGE, device=DEV)
    full = start.clone()
    want = c.run(ops, full, before=c.before)
    c.check(want, full, c.before, start)
    j = torch.arange(past - window + 1, device=DEV)       # all rows in front of the oldest that the first token sees
    page = c.table[0].long()[j // PAGE]
    for junk in (NAN, math.inf, -math.inf):
        c.k[page, :, j % PAGE] = junk
        c.v[page, :, j % PAGE] = junk
        mass = start.clone()
        assert torch.equal(c.run(ops, mass, before=c.before), want) and torch.equal(mass, full)
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.float32, 33)])
@pytest.mark.parametrize("new", [[90, 40], [1, 3]])
def test_windows_longer_than_any_sequence(ops, dtype, hd, new):
    """A window that no 32-bit number holds is no window."""
    c = Case(dtype, 4, 2, hd, [300, 64], new, None, seed=7)
    start = torch.zeros(c.pages, 2, PAGE, device=DEV)
    full = start.clone()
    want = c.run(ops, full, before=c.before)
    c.check(want, full, c.before, start)
    for c.window in (2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 40):
        mass = start.clone()
        c.check(c.run(ops, mass, before=c.before), mass, c.before, start)
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("new", [[90, 40], [1, 3]])
def test_captured_and_replayed(ops, new):
    """A captured call follows its inputs; two graphs that are replayed on two streams share nothing."""
    cs = [Case(torch.bfloat16, 8, 2, 128, [300, 64], new, None, seed=s) for s in (1, 2)]
    runs = []
    for c in cs:
        mass = torch.zeros(c.pages, 2, PAGE, device=DEV)
        out = c.run(ops, mass, before=c.before)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            c.run(ops, mass, before=c.before, out=out)
        runs.append((c, graph, out, mass))
    for c, _, out, mass in runs:
        c.qkv.copy_(c.qkv.flip(0))
        out.zero_()
        mass.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (c, graph, out, mass), st in zip(runs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for c, _, out, mass in runs:
        c.check(out, mass, c.before, torch.zeros_like(mass))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd,past,new", [(torch.bfloat16, 128, [300, 64], [90, 40]), (torch.bfloat16, 64, [3000, 10], [300, 20]),
                                               (torch.float32, 64, [300, 64], [90, 40]), (torch.bfloat16, 64, [300, 64], [1, 3]),
                                               (torch.float32, 80, [300, 64], [1, 1]), (torch.bfloat16, 64, [1500, 900], [1, 1])])
def test_metadata_from_the_kernel_in_front(ops, dtype, hd, past, new):
    """A step whose table, starts and places the kernel right in front of the call writes (they held other values before)."""
    c = Case(dtype, 8, 2, hd, past, new, None, seed=13)
    mass = torch.zeros(c.pages, 2, PAGE, device=DEV)
    want, sums = c.run(ops, mass), mass.clone()
    right = [x.clone() for x in (c.step.page_tables[0], c.step.seq_start, c.step.seq_pos0)]
    held = [c.step.page_tables[0], c.step.seq_start, c.step.seq_pos0]
    work = torch.randn(2048, 2048, device=DEV)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        for x, y in zip(held, right):
            torch.add(y, 0, out=x)
        c.run(ops, mass, out=out)
        held[0].fill_(-1)
        held[1].fill_(0)
        held[2].fill_(0)
    for _ in range(10):
        out.zero_(), mass.zero_()
        torch.mm(work, work)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(mass, sums)
    ops.check_errors()


# ------------------------------------------------------------------------------------------------------- the choice
def _chosen(values, n, first, recent, budget):
    """values: the rows' masses (a list)."""
    if n <= budget:
        return list(range(n)) + [-1] * (budget - n)
    order = sorted(range(first, n - recent), key=lambda r: (0 if not math.isnan(values[r]) else 1, -values[r] if not math.isnan(values[r]) else 0.0, r))
    rows = list(range(first)) + order[: budget - first - recent] + list(range(n - recent, n))
    return sorted(rows)


def _select_case(E, kv, lengths, seed, kind):
    g = torch.Generator(device=DEV).manual_seed(seed)
    table, pages, _ = _tables(lengths, seed)
    m = torch.rand(E, pages, kv, PAGE, generator=g, device=DEV)
    if kind == "ties":
        m = (m * 5).round()
    elif kind == "equal":
        m.fill_(0.25)
    elif kind == "wild":
        m = torch.exp((m - 0.5) * 170)                      # zero to infinity
        m[m > 1e36] = math.inf
        m[m < 1e-36] = 0.0
        m[torch.rand(m.shape, generator=g, device=DEV) < 0.05] = NAN
        m[torch.rand(m.shape, generator=g, device=DEV) < 0.05] = -1.5
        m[torch.rand(m.shape, generator=g, device=DEV) < 0.05] = -0.0
        m[torch.rand(m.shape, generator=g, device=DEV) < 0.02] = -math.inf
    return m, table


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["plain", "ties", "equal", "wild"])
@pytest.mark.parametrize("E,kv,lengths,budget,first,recent", [
    (1, 1, [1], 1, 0, 0), (1, 1, [2], 1, 0, 0), (1, 2, [2, 1], 1, 1, 0), (1, 2, [65, 64, 63], 64, 0, 1), (2, 3, [700, 100, 257], 128, 4, 32),
    (2, 3, [700, 100, 257], 128, 100, 28), (1, 1, [0, 5, 300], 17, 3, 2), (3, 2, [5000, 1025], 1000, 0, 0), (1, 2, [40000], 4096, 4, 256),
    (1, 1, [70001], 999, 1, 50), (12, 8, [16000, 300], 512, 4, 60), (1, 1, [300000], 70000, 4, 60)])
def test_evict_select(ops, E, kv, lengths, budget, first, recent, kind):
    m, table = _select_case(E, kv, lengths, 11, kind)
    kept = torch.full((E, len(lengths), kv, budget), 99, dtype=torch.int32, device=DEV)
    ops.evict_select(m, table, _ints(lengths), first, recent, kept)
    host, t = m.cpu(), table.cpu()
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        page = t[b].long()[j // PAGE]
        for e in range(0, E, 5):
            for h in range(0, kv, 3):
                assert kept[e, b, h].tolist() == _chosen(host[e, page, h, j % PAGE].tolist(), n, first, recent, budget)
    # one entry alone, without the axis
    alone = torch.full_like(kept[0], 99)
    ops.evict_select(m[E - 1], table, _ints(lengths), first, recent, alone)
    assert torch.equal(alone, kept[E - 1])
    ops.check_errors()


@pytest.mark.gpu
def test_evict_select_takes_a_missing_page_for_no_mass(ops):
    from hilbert_pruned_8b_b200.kernels.ops import KernelError
    m, table = _select_case(1, 1, [300], 3, "plain")
    table[0, 2] = -1
    kept = torch.empty(1, 1, 1, 100, dtype=torch.int32, device=DEV)
    ops.evict_select(m, table, _ints([300]), 0, 0, kept)
    assert not ((kept >= 128) & (kept < 192)).any()
    with pytest.raises(KernelError, match="page"):
        ops.check_errors()
    ops.reset_status()
    ops.evict_select(m, table, _ints([10 ** 9]), 0, 0, kept)            # a length that the page table cannot hold
    assert int(kept.max()) < 64 * table.shape[1] and int(kept.min()) >= 0
    with pytest.raises(KernelError, match="page"):
        ops.check_errors()
    ops.reset_status()


# --------------------------------------------------------------------------------------------------------- the move
@pytest.mark.gpu
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,kv,hd,v_hd,lengths,budget,first,recent", [
    (1, 1, 64, 64, [1], 1, 0, 0), (2, 3, 128, 128, [700, 100, 257], 128, 4, 32), (1, 2, 80, 80, [3000, 65], 2990, 0, 5),
    (1, 2, 33, 33, [300, 200], 100, 1, 1), (3, 2, 256, 128, [1000], 64, 4, 60), (1, 1, 7, 7, [5000], 1500, 4, 10), (8, 8, 128, 128, [2000, 900], 500, 4, 50)])
def test_evict_rows(ops, dtype, E, kv, hd, v_hd, lengths, budget, first, recent, apart):
    g = torch.Generator(device=DEV).manual_seed(2)
    B, spare = len(lengths), _pages(budget)
    table, pages, rest = _tables(lengths, 6, extra=B * spare + 2)
    k = torch.randn(E, pages, kv, PAGE, hd, generator=g, device=DEV).to(dtype)
    v = torch.randn(E, pages, kv, PAGE, v_hd, generator=g, device=DEV).to(dtype)
    mass = torch.rand(E, pages, kv, PAGE, generator=g, device=DEV)
    kept = torch.empty(E, B, kv, budget, dtype=torch.int32, device=DEV)
    ops.evict_select(mass, table, _ints(lengths), first, recent, kept)
    to = torch.tensor([rest[b * spare: (b + 1) * spare] for b in range(B)], dtype=torch.int32, device=DEV) if apart else None
    want = [x.clone() for x in (k, v, mass)]
    e, b, h, j = torch.nonzero(kept >= 0, as_tuple=True)
    src = kept[e, b, h, j].long()
    dest = (to if apart else table)[b, j // PAGE].long()
    for x, y in zip((k, v, mass), want):
        y[e, dest, h, j % PAGE] = x[e, table[b, src // PAGE].long(), h, src % PAGE]
    ops.evict_rows(kept, k, v, mass, table, to_table=to)
    for x, y in zip((k, v, mass), want):
        assert torch.equal(x, y)
    if not apart:
        k1, v1 = k[0].clone(), v[0].clone()                   # one entry alone, without mass; rows that are in place stay
        again = torch.where(kept[0] >= 0, torch.arange(budget, dtype=torch.int32, device=DEV), kept[0])
        ops.evict_rows(again, k1, v1, None, table)
        assert torch.equal(k1, k[0]) and torch.equal(v1, v[0])
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("dtype,hd,v_hd,offset", [(torch.bfloat16, 72, 72, 0), (torch.bfloat16, 120, 120, 0), (torch.bfloat16, 24, 56, 0), (torch.float32, 36, 4, 0),
                                                  (torch.bfloat16, 128, 128, 8), (torch.float32, 64, 64, 4), (torch.bfloat16, 80, 80, 2),
                                                  (torch.bfloat16, 64, 64, 1)])
def test_evict_rows_in_units_of_fewer_bytes(ops, dtype, hd, v_hd, offset, apart):
    """Rows whose bytes are a multiple of 16 and not of 32, and storage that begins 16, 4 and 2 bytes behind a multiple of 32."""
    E, kv, lengths, budget = 2, 3, [3000, 700, 65], 600
    g = torch.Generator(device=DEV).manual_seed(2)
    B, spare = len(lengths), _pages(budget)
    table, pages, rest = _tables(lengths, 6, extra=B * spare + 2)

    def storage(size):
        n = E * pages * kv * PAGE * size
        return torch.randn(n + offset, generator=g, device=DEV).to(dtype)[offset:].view(E, pages, kv, PAGE, size)
    k, v = storage(hd), storage(v_hd)
    mass = torch.rand(E, pages, kv, PAGE, generator=g, device=DEV)
    kept = torch.empty(E, B, kv, budget, dtype=torch.int32, device=DEV)
    ops.evict_select(mass, table, _ints(lengths), 4, 32, kept)
    to = torch.tensor([rest[b * spare: (b + 1) * spare] for b in range(B)], dtype=torch.int32, device=DEV) if apart else None
    want = [x.clone() for x in (k, v, mass)]
    e, b, h, j = torch.nonzero(kept >= 0, as_tuple=True)
    src = kept[e, b, h, j].long()
    dest = (to if apart else table)[b, j // PAGE].long()
    for x, y in zip((k, v, mass), want):
        y[e, dest, h, j % PAGE] = x[e, table[b, src // PAGE].long(), h, src % PAGE]
    ops.evict_rows(kept, k, v, mass, table, to_table=to)
    for x, y in zip((k, v, mass), want):
        assert torch.equal(x, y)
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("apart", [False, True])
def test_evict_rows_of_very_many_lists(ops, apart):
    """More lists of rows (entries x sequences x kv heads) than a grid's second axis holds."""
    E, B, kv, hd = 32, 1100, 2, 4                         # 70400 lists
    pages = 2 * B
    table = torch.arange(B, dtype=torch.int32, device=DEV).view(B, 1)
    to = (table + B).contiguous() if apart else None
    k, v = (torch.randn(E, pages, kv, PAGE, hd, device=DEV) for _ in range(2))
    mass = torch.rand(E, pages, kv, PAGE, device=DEV)
    kept = torch.empty(E, B, kv, 2, dtype=torch.int32, device=DEV)
    ops.evict_select(mass, table, _ints([3] * B), 0, 1, kept)
    want = [x.clone() for x in (k, v, mass)]
    e, b, h, j = torch.nonzero(kept >= 0, as_tuple=True)
    for x, y in zip((k, v, mass), want):
        y[e, b + (B if apart else 0), h, j] = x[e, b, h, kept[e, b, h, j].long()]
    ops.evict_rows(kept, k, v, mass, table, to_table=to)
    for x, y in zip((k, v, mass), want):
        assert torch.equal(x, y)
    ops.check_errors()


@pytest.mark.gpu
def test_evict_rows_skips_what_has_no_page(ops):
    from hilbert_pruned_8b_b200.kernels.ops import KernelError
    table, pages, _ = _tables([200], 1)
    k = torch.randn(1, pages, 1, PAGE, 64, device=DEV)
    v = torch.randn(1, pages, 1, PAGE, 64, device=DEV)
    for where in (-1, 10 ** 6):
        t, k2, v2 = table.clone(), k.clone(), v.clone()
        t[0, 2] = where
        kept = _ints([[[[0, 130, 3 + 10 ** 6]]]]).view(1, 1, 1, 3)
        ops.evict_rows(kept, k2, v2, None, t)
        assert torch.equal(k2, k) and torch.equal(v2, v)
        with pytest.raises(KernelError, match="page"):
            ops.check_errors()
        ops.reset_status()


# ------------------------------------------------------------------------------------------- one after another
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 80)])
def test_a_conversation_with_a_bounded_cache(ops, dtype, hd):
    """A prompt, single tokens, an eviction in place, more tokens: the attention behind the eviction is that over the rows that
    stayed, and the sums go on from where they were."""
    heads, kv, n, budget = 8, 2, 500, 150
    c = Case(dtype, heads, kv, hd, [0, 0], [n, 90], None, seed=8, garbage=0.0)
    mass = torch.zeros(c.pages, kv, PAGE, device=DEV)
    c.run(ops, mass, before=mass)
    kept = torch.empty(2, kv, budget, dtype=torch.int32, device=DEV)
    ops.evict_select(mass, c.table, _ints(c.lens), 4, 20, kept)
    rows = []
    for b, ln in enumerate(c.lens):
        for g in range(kv):
            r = kept[b, g][kept[b, g] >= 0].long()
            page = c.table[b].long()[r // PAGE]
            rows.append((c.k[page, g, r % PAGE].clone(), c.v[page, g, r % PAGE].clone(), mass[page, g, r % PAGE].clone()))
    ops.evict_rows(kept, c.k, c.v, mass, c.table)
    lens = [min(ln, budget) for ln in c.lens]
    d = Case(dtype, heads, kv, hd, lens, [1, 7], None, seed=21)       # the next tokens: their keys and values behind the kept rows
    gen = torch.Generator(device=DEV).manual_seed(5)
    for b, (p, m) in enumerate(zip(lens, d.new)):
        j = torch.arange(p, p + m, device=DEV)
        page = c.table[b].long()[j // PAGE]
        c.k[page, :, j % PAGE] = torch.randn(m, kv, hd, generator=gen, device=DEV).to(dtype)
        c.v[page, :, j % PAGE] = torch.randn(m, kv, hd, generator=gen, device=DEV).to(dtype)
        for g in range(kv):
            k0, v0, m0 = rows[b * kv + g]
            i = torch.arange(p, device=DEV)
            page = c.table[b].long()[i // PAGE]
            assert torch.equal(c.k[page, g, i % PAGE], k0) and torch.equal(c.v[page, g, i % PAGE], v0) and torch.equal(mass[page, g, i % PAGE], m0)
    d.table, d.pages, d.k, d.v = c.table, c.pages, c.k, c.v
    d.step, d.cache = _step(d.past, d.new, c.table), c.cache
    start = mass.clone()
    out = d.run(ops, mass, before=mass)
    inside = torch.zeros_like(mass, dtype=torch.bool)
    for b, ln in enumerate(d.lens):
        j = torch.arange(ln, device=DEV)
        inside[c.table[b].long()[j // PAGE], :, j % PAGE] = True
    assert torch.equal(mass[~inside], start[~inside])
    d.check(out, mass, start, start)
    ops.check_errors()


def _hidden_attention(hidden):
    """Grouped attention of one whole sequence in 64 bits over what is not hidden: ``hidden`` [kv heads, tokens, tokens]."""
    def attention(q, k, v, window=None):
        T, nh, hd = q.shape
        G = nh // k.shape[1]
        out = torch.empty_like(q)
        for h in range(nh):
            s = (q[:, h] @ k[:, h // G].T / math.sqrt(hd)).masked_fill(hidden[h // G], -math.inf)
            out[:, h] = torch.softmax(s, dim=-1) @ v[:, h // G]
        return out
    return attention


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("model", ["strong_a", "strong_b", "strong_c", "strong_d"])
def test_the_engine_goes_on_behind_an_eviction(model_folders, monkeypatch, model, dtype):
    """Prompts, two evictions in place with tokens between and behind them, in steps of several tokens and in captured ones: the logits
    are those of a plain model whose later tokens see the rows that stayed, rotated by their true positions."""
    require_gpu()
    import plain_llama as pl
    import trace_tools as tt
    from hilbert_pruned_8b_b200.engine.batch import StepEntry
    from hilbert_pruned_8b_b200.engine.step import Engine
    eng = Engine.from_folder(model_folders[model], dtype, max_tokens=1024)
    ops, cfg = eng.ctx.ops, pl.read_config(model_folders[model])
    L, kv = cfg["num_hidden_layers"], cfg["num_key_value_heads"]
    (group,) = eng.cache.groups
    tokens = {b: tt.random_tokens(n, cfg["vocab_size"], 40 + b) for b, n in enumerate((260, 90))}
    seqs = [eng.open_sequence() for _ in tokens]
    done, got = [0, 0], {}
    stood = {(b, e, g): [] for b in tokens for e in range(L) for g in range(kv)}          # positions of a list's rows
    hidden = {b: torch.ones(len(t), len(t), dtype=torch.bool).triu(1).repeat(L, kv, 1, 1) for b, t in tokens.items()}

    def feed(counts):
        entries = [StepEntry(s, tokens[b][done[b]: done[b] + n], list(range(n))) for b, (s, n) in enumerate(zip(seqs, counts))]
        logits = eng.step(entries).double().cpu()
        rows = [(b, done[b] + i) for b, n in enumerate(counts) for i in range(n)]
        got.update({key: row for key, row in zip(rows, logits)})
        for b, n in enumerate(counts):
            for e in range(L):
                for g in range(kv):
                    stood[b, e, g] += range(done[b], done[b] + n)
            done[b] += n

    def cut(budget, first, recent, seed):
        width = max(len(s.pages[0]) for s in seqs)
        table = torch.tensor([s.pages[0] + [-1] * (width - len(s.pages[0])) for s in seqs], dtype=torch.int32, device=DEV)
        mass = torch.rand(group.k.shape[:-1], generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)
        kept = torch.empty(L, len(seqs), kv, budget, dtype=torch.int32, device=DEV)
        ops.evict_select(mass, table, _ints([s.length for s in seqs]), first, recent, kept)
        ops.evict_rows(kept, group.k, group.v, mass, table)
        for b, s in enumerate(seqs):
            before = len(s.pages[0])
            eng.cache.evict(s, min(s.length, budget))
            assert len(s.pages[0]) == min(before, _pages(budget)) and s.length + s.evicted == done[b]
            for e in range(L):
                for g in range(kv):
                    was = stood[b, e, g]
                    stood[b, e, g] = [was[j] for j in kept[e, b, g].tolist() if j >= 0]
                    gone = sorted(set(range(done[b])) - set(stood[b, e, g]))
                    hidden[b][e, g, done[b]:, gone] = True

    feed([200, 40])
    cut(70, 2, 8, 1)                        # the second sequence is shorter than its budget
    for _ in range(5):
        feed([1, 1])
    feed([9, 30])
    cut(40, 0, 5, 2)
    feed([3, 2])
    for _ in range(6):
        feed([1, 1])
    assert eng.graph_replays > 0 and seqs[0].evicted == 130 + 44 and seqs[1].evicted == 35
    ops.check_errors()
    plain = pl.PlainLlama(model_folders[model], round_to=torch.bfloat16 if dtype == "bfloat16" else None)
    for b, s in enumerate(seqs):
        layer = [0]

        def attention(q, k, v, window=None):
            layer[0] += 1
            return _hidden_attention(hidden[b][layer[0] - 1][:, :done[b], :done[b]])(q, k, v)
        monkeypatch.setattr(pl, "attention", attention)
        want = plain.logits(tokens[b][:done[b]])
        tt.compare({k: v for k, v in got.items() if k[0] == b}, {(b, i): row for i, row in enumerate(want)}, dtype, "behind an eviction")


# ------------------------------------------------------------------------------------------- the cache's bookkeeping
def _manager(max_tokens=1024, window=None, stride=1, state=False):
    from hilbert_pruned_8b_b200.cache import CacheManager
    from hilbert_pruned_8b_b200.parts.base import CacheNeed, StateNeed
    needs = {0: CacheNeed(2, 16), 1: CacheNeed(1, 32, window, stride=stride)}
    return CacheManager(needs, {0: StateNeed((3,))} if state else {}, max_tokens, torch.device("cpu"), torch.float32)


def test_an_evicted_sequence_keeps_its_positions():
    from hilbert_pruned_8b_b200.engine.batch import DecodeMeta, StepEntry, build_step
    from hilbert_pruned_8b_b200.engine.workspace import Workspace
    cpu = torch.device("cpu")
    m, ws = _manager(), Workspace(cpu)
    a, b = m.open(), m.open()
    for s, n in ((a, 300), (b, 70)):
        m.reserve([(s, n)])
        m.commit(s, n)
    free = m.pages_free()
    m.evict(a, 130)
    assert (a.length, a.evicted, a.kept) == (130, 170, 130) and (b.length, b.evicted) == (70, 0)
    assert m.pages_free() == [f + 2 for f in free] and [len(p) for p in a.pages] == [3, 3]
    meta = DecodeMeta(2, 8, m, ws, cpu, "meta")
    for n in (3, 1, 1):
        entries = [StepEntry(a, [5] * n, [0]), StepEntry(b, [7], [0])]
        m.reserve([(e.seq, e.seq.length + len(e.tokens)) for e in entries])
        steps = [build_step(entries, m, ws, cpu)] + ([meta.fill(entries)] if n == 1 else [])
        for st in steps:
            assert st.positions.tolist() == [a.length + i for i in range(n)] + [b.length]
            assert st.rope_positions.tolist() == [a.length + 170 + i for i in range(n)] + [b.length]
            assert st.seq_pos0.tolist() == [a.length, b.length]
        for e in entries:
            m.commit(e.seq, e.seq.length + len(e.tokens))
    m.evict(a, 64)
    assert (a.length, a.evicted, a.kept) == (64, 241, 64)
    m.evict(a, 64)                                           # nothing goes
    assert (a.length, a.evicted, a.kept) == (64, 241, 64)
    m.close(a), m.close(b)
    assert m.pages_free() == [16, 16]


def test_rewinds_of_an_evicted_sequence():
    m = _manager()
    s = m.open()
    for n in (100, 200):
        m.reserve([(s, n)])
        m.commit(s, n)
        snap = m.snapshot(s) if n == 100 else snap
    m.evict(s, 120)
    with pytest.raises(ValueError, match="evicted since"):
        m.restore(s, snap)
    m.reserve([(s, 150)])
    m.commit(s, 150)
    later = m.snapshot(s)
    m.reserve([(s, 160)])
    m.commit(s, 160)
    m.restore(s, later)                                      # tokens behind the kept rows may be taken back
    assert (s.length, s.evicted) == (150, 80)
    m.truncate(s, 120)
    for n in (119, 1):
        with pytest.raises(ValueError, match="rewound"):
            m.truncate(s, n)
    assert (s.length, s.evicted, s.kept) == (120, 80, 120)
    m.truncate(s, 0)                                         # a new beginning
    assert (s.length, s.evicted, s.kept) == (0, 0, 0)


def test_evictions_that_are_refused():
    m = _manager()
    s = m.open()
    m.reserve([(s, 100)])
    m.commit(s, 100)
    for rows in (0, -1, 101):
        with pytest.raises(ValueError, match="cannot stay"):
            m.evict(s, rows)
    m.close(s)
    with pytest.raises(ValueError, match="closed"):
        m.evict(s, 50)
    for kw in (dict(window=70), dict(stride=4)):
        n = _manager(**kw)
        s = n.open()
        n.reserve([(s, 100)])
        n.commit(s, 100)
        with pytest.raises(ValueError, match="window or a stride"):
            n.evict(s, 50)
        assert s.length == 100
    n = _manager(state=True)                                 # state of fixed size goes on
    s = n.open()
    n.reserve([(s, 100)])
    n.commit(s, 100)
    n.state_view(0)[s.state_slot] += 2.0
    n.evict(s, 50)
    assert (s.length, s.evicted) == (50, 50) and n.state_view(0)[s.state_slot].tolist() == [2.0] * 3


# ------------------------------------------------------------------------------------------------------- refusals
class _Fake:
    """An ``Ops`` without a device: the checks of arguments run, a call of the library would fail the test."""

    def __new__(cls):
        from hilbert_pruned_8b_b200.kernels.ops import Ops
        o = object.__new__(Ops)
        o.device, o._index, o.sm_count, o.launches = torch.device("cpu"), -1, 148, 0
        o.lib = None

        def call(name, *a):
            raise AssertionError("reached " + name)
        o._call = call
        return o


def _attention_args(**kw):
    n = types.SimpleNamespace
    a = dict(qkv=torch.zeros(3, 64 * 6), heads=4, kv_heads=2, head_dim=64, k=torch.zeros(5, 2, 64, 64), v=torch.zeros(5, 2, 64, 64),
             out=torch.zeros(3, 256), mass=torch.zeros(5, 2, 64), before=None, tokens=3)
    a.update(kw)
    step = n(num_tokens=a.pop("tokens"), num_seqs=1, page_tables=[a.pop("table", torch.zeros(1, 2, dtype=torch.int32))], max_new=3, max_len=3, host_new=[3], host_len=[3])
    cache = n(k=a.pop("k"), v=a.pop("v"), group=0, window=None)
    return dict(dict(scale=0.125, window=None, cache=cache, step=step), **a)


@pytest.mark.parametrize("change,text", [
    (dict(heads=5), "heads"), (dict(kv_heads=0), "heads"), (dict(head_dim=257), "heads"), (dict(head_dim=32), "shape"), (dict(tokens=4), "shape"),
    (dict(out=torch.zeros(2, 256)), "shape"), (dict(out=torch.zeros(3, 255)), "shape"), (dict(qkv=torch.zeros(3, 255)), "shape"),
    (dict(k=torch.zeros(5, 2, 32, 64)), "cache"), (dict(v=torch.zeros(5, 64, 2, 64).transpose(1, 2)), "cache"),
    (dict(out=torch.zeros(3, 256, dtype=torch.bfloat16)), "dtype"), (dict(k=torch.zeros(5, 2, 64, 64).half()), "dtype"),
    (dict(mass=torch.zeros(4, 2, 64)), "mass"), (dict(mass=torch.zeros(5, 2, 64).double()), "mass"), (dict(mass=torch.zeros(5, 64, 2).mT), "mass"),
    (dict(before=torch.zeros(5, 2, 63)), "before"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=NAN), "scale"),
    (dict(window=-5), "window"), (dict(table=torch.zeros(1, 2, dtype=torch.int64)), "page table"), (dict(table=torch.zeros(1, 4, dtype=torch.int32)[:, ::2]), "page table")])
def test_attention_mass_refuses(change, text):
    from hilbert_pruned_8b_b200.kernels.ops import KernelError
    with pytest.raises(KernelError, match=text):
        _Fake().attention_mass(**_attention_args(**change))


@pytest.mark.parametrize("short", ["table", "seq_start", "seq_pos0"])
def test_attention_mass_refuses_a_step_of_fewer_rows_than_sequences(short):
    """What the kernels would read behind the end of."""
    from hilbert_pruned_8b_b200.kernels.ops import KernelError
    a = _attention_args(table=_i32(2, 2))
    st = a["step"]
    st.num_seqs, st.host_new, st.host_len, st.seq_start, st.seq_pos0 = 2, [2, 1], [2, 1], _i32(3), _i32(2)
    if short == "table":
        st.page_tables = [_i32(1, 2)]
    else:
        setattr(st, short, getattr(st, short)[:-1])
    with pytest.raises(KernelError, match="2 sequences"):
        _Fake().attention_mass(**a)


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["page_tables", "seq_start", "seq_pos0"])
def test_attention_mass_refuses_metadata_of_another_device(ops, what):
    from hilbert_pruned_8b_b200.kernels.ops import KernelError
    c = Case(torch.bfloat16, 4, 2, 64, [100], [3], None)
    setattr(c.step, what, [c.table.cpu()] if what == "page_tables" else getattr(c.step, what).cpu())
    with pytest.raises(KernelError, match="tensor on cpu"):
        c.run(ops, torch.zeros(c.pages, 2, PAGE, device=DEV))


@pytest.mark.parametrize("pages,q,called", [(5, None, "hb_attention_mass_tc"), (1 << 22, None, "hb_attention_mass"), ((1 << 22) - 1, None, "hb_attention_mass_tc"),
                                            (5, torch.zeros(1, 256, dtype=torch.bfloat16).expand(20, 256), "hb_attention_mass")])
def test_what_a_tensor_map_does_not_take(pages, q, called):
    """Caches of 2^31 rows and more and one query row for all tokens go to the kernel for every size."""
    o, calls, n = _Fake(), [], types.SimpleNamespace
    o._call, o._elsewhere, o._stream, o.status = lambda name, *a: calls.append(name), lambda: False, lambda: 0, torch.zeros(4, dtype=torch.int32)
    o.use_fast_attention = o.use_tcgen05_attention = True
    o.MASS_FEW_PAIRS, o._mass_plans = 512, {}
    o.lib = n(hb_attention_mass_tc_supported=lambda *a: 1, hb_attention_mass_tc_keys=lambda: 256)

    class Held:
        """Keys and values without memory."""
        shape, dtype = (pages, 8, 64, 8), torch.bfloat16

        def get_device(self):
            return -1

        def is_contiguous(self):
            return True

        def data_ptr(self):
            return 1 << 20
    q = q if q is not None else torch.zeros(20, 64 + 8, dtype=torch.bfloat16)
    heads = 8 if q.shape[1] == 72 else 32

    class Mass(Held):
        shape, dtype = (pages, 8, 64), torch.float32
    step = n(num_tokens=20, num_seqs=1, page_tables=[_i32(1, 2)], seq_start=_i32(2), seq_pos0=_i32(1), max_new=20, max_len=70, host_new=[20], host_len=[70])
    o.attention_mass(q, heads, 8, 8, n(k=Held(), v=Held(), group=0), step, torch.zeros(20, heads * 8, dtype=torch.bfloat16), 0.3, None, Mass())
    assert calls == [called]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
@pytest.mark.parametrize("new", [[90, 40], [1, 3]])
def test_one_query_row_for_all_tokens(ops, dtype, hd, new):
    c = Case(dtype, 4, 2, hd, [300, 64], new, None, seed=17)
    c.qkv = c.qkv[:1].expand(sum(new), -1)
    start = torch.zeros(c.pages, 2, PAGE, device=DEV)
    mass = start.clone()
    c.check(c.run(ops, mass, before=c.before), mass, c.before, start)
    ops.check_errors()


def test_attention_mass_of_no_tokens():
    _Fake().attention_mass(**_attention_args(qkv=torch.zeros(0, 384), out=torch.zeros(0, 256), tokens=0))


def _i32(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("change,text", [
    (dict(mass=torch.zeros(2, 5, 3, 63)), "mass"), (dict(mass=torch.zeros(2, 5, 3, 64).double()), "mass"), (dict(mass=torch.zeros(5, 64)), "mass"),
    (dict(page_table=_i32(4)), "page table"), (dict(page_table=torch.zeros(4, 2)), "page table"), (dict(page_table=_i32(4, 4)[:, ::2]), "page table"),
    (dict(lengths=_i32(3)), "length"), (dict(lengths=torch.zeros(4, dtype=torch.int64)), "length"), (dict(kept=_i32(2, 4, 3, 0)), "kept"),
    (dict(kept=_i32(2, 3, 4, 9)), "kept"), (dict(kept=torch.zeros(2, 4, 3, 9)), "kept"), (dict(kept=_i32(4, 3, 9)), "kept"),
    (dict(first=5, recent=5), "budget"), (dict(first=-1), "budget"), (dict(recent=-1), "budget")])
def test_evict_select_refuses(change, text):
    from hilbert_pruned_8b_b200.kernels.ops import KernelError
    a = dict(mass=torch.zeros(2, 5, 3, 64), page_table=_i32(4, 2), lengths=_i32(4), first=2, recent=3, kept=_i32(2, 4, 3, 9))
    with pytest.raises(KernelError, match=text):
        _Fake().evict_select(**dict(a, **change))


@pytest.mark.parametrize("change,text", [
    (dict(k=torch.zeros(2, 5, 3, 32, 16)), "keys"), (dict(v=torch.zeros(2, 5, 3, 64, 16).double()), "keys"), (dict(v=torch.zeros(2, 6, 3, 64, 16)), "keys"),
    (dict(k=torch.zeros(2, 5, 3, 64, 32)[..., ::2]), "keys"), (dict(k=torch.zeros(2, 5, 3, 64, 16).half(), v=torch.zeros(2, 5, 3, 64, 16).half()), "dtype"),
    (dict(mass=torch.zeros(2, 5, 3, 16)), "mass"), (dict(page_table=_i32(4)), "page table"), (dict(to_table=_i32(3, 2)), "page tables"),
    (dict(to_table=_i32(4, 2).long()), "page table"), (dict(kept=_i32(2, 4, 3, 129), to_table=_i32(4, 2)), "budget"), (dict(kept=_i32(4, 3, 9)), "kept")])
def test_evict_rows_refuses(change, text):
    from hilbert_pruned_8b_b200.kernels.ops import KernelError
    a = dict(kept=_i32(2, 4, 3, 9), k=torch.zeros(2, 5, 3, 64, 16), v=torch.zeros(2, 5, 3, 64, 16), mass=torch.zeros(2, 5, 3, 64),
             page_table=_i32(4, 2), to_table=None)
    with pytest.raises(KernelError, match=text):
        _Fake().evict_rows(**dict(a, **change))


def test_codes_of_waits_that_ran_out_name_their_kernel():
    """The status word holds a code and nothing else: no other kernel notes the codes of these two."""
    import glob
    import os
    import re
    import hilbert_pruned_8b_b200.kernels.build as build
    codes = {}
    for path in glob.glob(os.path.join(os.path.dirname(os.path.dirname(build.__file__)), "csrc", "*.cu*")):
        with open(path) as f:
            codes[os.path.basename(path)] = set(re.findall(r"atomicExch\(\w+, (\d+)\)", f.read()))
    for mine in ("attention_chunk_tc.cu", "attention_mass_tc.cu"):
        assert codes[mine] and codes["moe_tc.cu"]
        for other, theirs in codes.items():
            assert other == mine or not theirs & codes[mine], (mine, other)


@pytest.mark.parametrize("degree,bound", [(4, 2.7e-6), (5, 2.2e-7)])
def test_the_polynomials_of_powers_of_two(degree, bound):
    """2^x in 32-bit steps with the coefficients that stand in the kernels, against 64 bits: the relative errors that are stated there."""
    import os
    import re
    import numpy as np
    import hilbert_pruned_8b_b200.kernels.build as build
    with open(os.path.join(os.path.dirname(os.path.dirname(build.__file__)), "csrc", "exp2_pair.cuh")) as f:
        source = f.read()
    body = source[source.index("if (DEG == 5)"): source.index("float r0, r1;")]
    five, four = body.split("} else {")
    coefficients = [float(a) for a, b in re.findall(r"pair_of\(([-\d.e]+)f, ([-\d.e]+)f\)", five if degree == 5 else four) if a == b]
    assert len(coefficients) == degree + 1
    f32 = np.float32
    x = np.concatenate([np.linspace(-125, 127, 400001), np.linspace(-1, 1, 400001)]).astype(f32)
    r = (x + f32(12582912.0)).astype(f32)
    n = (r - f32(12582912.0)).astype(f32)
    f = (x - n).astype(f32)                                  # exact: x and n lie within a half
    assert np.abs(f).max() <= 0.5
    p = np.full_like(f, f32(coefficients[0]))
    for c in coefficients[1:]:
        p = (f.astype(np.float64) * p.astype(np.float64) + np.float64(f32(c))).astype(f32)       # a fused product and sum, rounded once
    got = p.astype(np.float64) * np.exp2(n.astype(np.float64))
    assert np.abs(got / np.exp2(x.astype(np.float64)) - 1).max() <= bound


def test_groups_of_sequences():
    """Every sequence once and in order, with its tokens, within the limit unless a group has one sequence with new tokens."""
    from hilbert_pruned_8b_b200.kernels.plan import few_groups
    assert few_groups([1] * 8, [300] * 8, 32, 64 << 20) == [(0, 8, 0, 8, 300)]
    assert few_groups([1, 1, 1], [131072, 5, 131072], 32, 32 * 131072) == [(0, 1, 0, 1, 131072), (1, 1, 1, 1, 5), (2, 1, 2, 1, 131072)]
    assert few_groups([0, 1, 0, 2, 0], [7, 1, 900, 2, 65], 4, 1) == [(0, 2, 0, 1, 7), (2, 3, 1, 2, 900)]
    assert few_groups([0, 0], [7, 1], 4, 1) == [] and few_groups([], [], 4, 1) == []
    rng = random.Random(1)
    for _ in range(300):
        n = rng.randint(1, 40)
        new, heads = [rng.choice([0, 1, 1, rng.randint(1, 8)]) for _ in range(n)], rng.choice([1, 8, 32])
        lens = [m + (rng.randint(0, 131072) if rng.random() < 0.2 else rng.randint(0, 900)) for m in new]
        limit = rng.choice([1, 10 ** 6, 64 << 20])
        groups = few_groups(new, lens, heads, limit)
        if sum(new) == 0:
            assert groups == []
            continue
        seq = token = 0
        for first, count, t0, tokens, rows in groups:
            assert (first, t0) == (seq, token) and count > 0 and tokens > 0
            inside = list(range(first, first + count))
            assert tokens == sum(new[b] for b in inside) and rows == max(max(1, lens[b]) for b in inside)
            assert heads * tokens * -(-rows // 64) * 64 <= limit or sum(new[b] > 0 for b in inside) == 1
            seq, token = seq + count, token + tokens
        assert seq == n and token == sum(new)
    # 64 single tokens, one long sequence: 1 GB in one group
    groups = few_groups([1] * 64, [131072] * 64, 32, 64 << 20)
    assert len(groups) == 4 and max(32 * g[3] * g[4] for g in groups) <= 64 << 20


def test_shapes_of_the_launches():
    from hilbert_pruned_8b_b200.kernels.plan import chunk_shares, few_splits, mass_splits, select_shape
    assert few_splits([5], 8, 296) == (5, 1) and few_splits([129] * 8, 8, 296) == (4, 1) and few_splits([100] * 1000, 8, 296) == (1, 1)
    assert few_splits([], 8, 296) == (1, 1) and few_splits([1], 1, 296) == (1, 1)
    for pages in ([33, 126, 9, 65], [1, 1, 2000], [7] * 50 + [900]):
        splits, least = few_splits(pages, 8, 296)
        assert 1 <= splits <= 32 and splits * least >= max(pages)
    assert mass_splits([4096], [4096], 0, 256, 128, 8, 4, 148) == 2 and mass_splits([2048], [32049], 0, 256, 128, 8, 4, 148) == 1
    assert mass_splits([1], [1], 0, 64, 64, 1, 1, 296) == 1 and mass_splits([9000], [9000], 0, 64, 64, 1, 1, 296) == 4
    assert mass_splits([], [], 0, 64, 64, 1, 1, 296) == 1 and 1 <= mass_splits([0, 500], [7, 900], 30, 64, 64, 2, 3, 296) <= 6
    assert chunk_shares([4096], [4096], 0, 128, 128, 16, 4160, 148, 4.5, 8.0) == (1, 32, 0)                 # enough blocks for everybody
    shares, tiles, cut = chunk_shares([128], [100000], 0, 128, 128, 16, 4160, 148, 4.5, 8.0)                  # 16 blocks of 782 tiles
    assert 8 <= shares <= 32 and (shares - 1) * tiles < 782 <= shares * tiles and cut == 128
    assert chunk_shares([10, 0], [100, 7], 0, 128, 128, 16, 4160, 148, 4.5, 8.0) == (1, 1, 0) and chunk_shares([], [], 0, 128, 128, 16, 4160, 148, 4.5, 8.0) == (1, 1, 0)
    for window in (0, 1000):
        for new, lens in (([700, 33, 1], [700, 550, 5000]), ([2000] * 5, [9000] * 5), ([9], [10 ** 6])):
            shares, tiles, cut = chunk_shares(new, lens, window, 256, 64, 5, 100, 148, 1.0, 2.0)
            seen = max(min(ln, window + 256) if window else ln for ln in lens)
            assert 0 <= cut <= sum(new) and (shares == 1 or cut > 0)
            assert 1 <= shares <= 32 and shares * tiles * 64 >= seen               # the device cuts a block into at most that many
    for rows in (1, 64, 1000, 16384, 16385, 70000, 131072, 300000, 10 ** 7):
        for lists in (1, 2, 16, 74, 75, 148, 256, 4096):
            threads, cluster = select_shape(lists, rows, 148)
            assert threads in (512, 1024) and cluster in (1, 2, 4, 8)
            assert cluster == 8 or rows <= threads * cluster * 32
