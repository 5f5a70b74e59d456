"""The serving operators beside one another: on two streams, from two threads, captured once and replayed step after step; and which of its kernels the attention over a shared prefix runs, with items that
lie in one line, whose ranges go on from item to item."""
import threading

import pytest
import torch

from leopard_b200 import _lib, ops
from oracle import serve as O
from test_serve_ops import MANY, attend, close, gen, i32, near, prefix_case

gpu = pytest.mark.gpu
BF16, I32 = torch.bfloat16, torch.int32


class Step:
    """Rows of a step of 40 requests, its tables and its keys' way into a cache; some wait, pages run from a list."""
    B, H, G, D, SIZE, ROWS = 40, 4, 2, 64, 16, 128

    def __init__(self, seed):
        g = gen(seed, "cpu")
        n, t = torch.randint(0, 100, (self.B,), generator=g), torch.randint(0, 4, (self.B,), generator=g)
        width, pages = 12, 800
        order, table, at = torch.randperm(pages, generator=g).int(), torch.full((self.B, width), -1, dtype=I32), 0
        for b in range(self.B):
            held = -(-int(n[b]) // self.SIZE)
            table[b, :held] = order[at:at + held]
            at += held
        self.lengths, self.new, self.table, self.free, self.used = n.int().cuda(), t.int().cuda(), table.cuda(), order[at:].cuda(), i32([2])
        rnd = lambda *s: torch.randn(*s, generator=g).to(BF16).cuda()  # noqa: E731
        self.q, self.k, self.v = rnd(self.ROWS, self.H, self.D), rnd(self.ROWS, self.G, self.D), rnd(self.ROWS, self.G, self.D)
        self.freq = (10000.0 ** (-torch.arange(self.D // 2, dtype=torch.float64) / (self.D // 2))).float().cuda()
        self.pools = [torch.zeros(pages, self.SIZE, self.G, self.D, dtype=BF16, device="cuda") for _ in range(2)]

    def run(self):
        seq, pos, slots, row0 = ops.step_tables(self.lengths, self.new, self.table, self.free, self.used, self.SIZE, self.ROWS)
        q = ops.rotary_append(self.q, self.k, self.v, pos, self.freq, *self.pools, slots)
        self.lengths += self.new
        return seq, pos, slots, row0, q

    def state(self):
        return [x.clone() for x in (self.lengths, self.table, self.used, *self.pools)]

    def check(self, outputs, before):
        """outputs of one `run` from the state `before`, by the definitions"""
        lengths, table, used, k_pool, v_pool = before
        seq, pos, slots, row0, q = outputs
        want = O.step_tables(lengths, self.new, table, self.free, used, self.SIZE, self.ROWS)
        assert [x.tolist() for x in (seq, pos, slots, row0, self.table)] == list(want[:5]) and int(self.used) == want[5]
        assert torch.equal(self.lengths, lengths + self.new)
        near(q, *O.rotary(self.q, pos, self.freq))
        k, size = O.rotary(self.k, pos, self.freq)
        at = slots[slots >= 0]
        assert len(at) == len(set(at.tolist())) == int(self.new.sum())
        near(self.pools[0].view(-1, self.G, self.D)[at], k[slots >= 0], size[slots >= 0])
        assert torch.equal(self.pools[1].view(-1, self.G, self.D)[at], self.v[slots >= 0])
        for pool, old in zip(self.pools, (k_pool, v_pool)):      # all other rows stay
            kept = torch.ones(pool.shape[0] * self.SIZE, dtype=torch.bool, device="cuda")
            kept[at] = False
            assert torch.equal(pool.view(-1, self.G, self.D)[kept], old.view(-1, self.G, self.D)[kept])


@gpu
def test_steps_on_two_streams():
    alone = []
    for seed in (1, 2):
        s = Step(seed)
        outs = []
        for _ in range(6):
            before = s.state()
            outs.append([x.clone() for x in s.run()])
            s.check(outs[-1], before)
        alone.append((outs, s.state()))
    steps, streams = [Step(1), Step(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for s, stream, o in zip(steps, streams, got):
            with torch.cuda.stream(stream):
                o.append(s.run())
    torch.cuda.synchronize()
    for s, o, (outs, state) in zip(steps, got, alone):
        assert all(torch.equal(x, y) for a, b in zip(o, outs) for x, y in zip(a, b)) and all(torch.equal(x, y) for x, y in zip(s.state(), state))


@gpu
def test_a_captured_step_goes_on_from_replay_to_replay():
    s = Step(3)
    start = s.state()
    s.run()                                               # (what is set up at a kernel's first launch)
    for x, y in zip((s.lengths, s.table, s.used, *s.pools), start):
        x.copy_(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.run()
    for i in range(8):
        s.new.copy_(torch.randint(0, 4, (s.B,), generator=gen(i, "cpu")).int())
        s.k.copy_(torch.randn(s.k.shape, generator=gen(i + 50, "cpu")))
        before = s.state()
        graph.replay()
        torch.cuda.synchronize()
        s.check(out, before)


@gpu
def test_two_threads_call_at_once():
    """each thread on a stream of its own, all operators in turn; the same results as one after the other"""
    cases = [prefix_case(6, 1, 32, 8, 128, 900, [5 * b for b in range(6)], page=64, seed=1), prefix_case(20, 1, 32, 8, 128, 4100, [30] * 20, page=64, seed=2)]
    logits = [torch.randn(5, 20000 + 13 * i, generator=gen(i), device="cuda") for i in (0, 1)]
    u = torch.rand(5, generator=gen(9), device="cuda")
    x = [torch.randn(300, 8, 128, generator=gen(i), device="cuda") for i in (0, 1)]
    pos, freq = torch.arange(300, device="cuda"), (10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)).float().cuda()

    def once(i, step):
        return [*step.run(), attend(cases[i]), ops.sample_tokens(logits[i], u, top_k=40, top_p=0.9), ops.rotary(x[i], pos, freq)]
    want = []
    for i in (0, 1):
        s = Step(i + 4)
        want.append([once(i, s) for _ in range(12)])
    steps, got, errors = [Step(4), Step(5)], [[], []], []
    torch.cuda.synchronize()
    meet = threading.Barrier(2, timeout=60)

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                meet.wait()
                for _ in range(12):
                    got[i].append(once(i, steps[i]))
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 (for the thread that waits)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert len(a) == 12 and all(torch.equal(x, y) for p, q in zip(a, b) for x, y in zip(p, q))


# ------------------------------------------------------------------------------------------------------------ which kernels run
def launches(f):
    n = _lib.lib().lp_launch_count()
    f()
    return _lib.lib().lp_launch_count() - n


@gpu
@pytest.mark.parametrize("B, T, H, G, D, prefix, own, new, page", MANY)
def test_many_rows_run_the_tcgen05_kernel(B, T, H, G, D, prefix, own, new, page):
    c = prefix_case(B, T, H, G, D, prefix, own, new, page)
    assert launches(lambda: attend(c)) == 3               # own rows, prefix, join


@gpu
def test_few_rows_and_odd_pages_run_the_other_one():
    for args in ((4, 1, 32, 8, 128, 4796, [40] * 4, None, 64), (2, 1, 4, 4, 128, 100003, [0] * 2, None, 64), (70, 1, 32, 8, 128, 1153, [3] * 70, None, 5)):
        c = prefix_case(*args)
        assert launches(lambda: attend(c)) == 2           # prefix and own rows, join


def around(mean, n):
    """n whole numbers about the mean, whose sum is n times it (n a multiple of 5)"""
    return [mean + i % 5 - 2 for i in range(n)]


# Items that cost too unequal a share each, so that all of them lie in one line and a CTA's range goes on in another item (on 148 SMs): heads of every size, last blocks of at most 128 rows (whose tiles cost less)
# and of more; requests that bring fewer tokens than there is room for, so that there are fewer items than the call's plan has; long items.
LINES = [
    (50, 24, 32, 8, 128, 1028, [i % 21 for i in range(50)], around(12, 50), 16), (30, 60, 16, 4, 128, 1043, [20] * 30, around(40, 30), 48), (100, 24, 8, 2, 96, 1080, [i % 7 for i in range(100)], None, 64),
    (50, 24, 16, 4, 96, 1071, [3] * 50, None, 16), (30, 60, 12, 4, 64, 1272, [20] * 30, None, 64), (100, 24, 12, 4, 64, 1033, [i % 3 for i in range(100)], around(16, 100), 0),
    (35, 8, 32, 8, 128, 6000, [i % 40 for i in range(35)], [8] * 34 + [3], 64),
]


@gpu
@pytest.mark.parametrize("B, T, H, G, D, prefix, own, new, page", LINES)
def test_items_of_one_line(B, T, H, G, D, prefix, own, new, page):
    c = prefix_case(B, T, H, G, D, prefix, own, new, page, seed=B + T)
    out = torch.full((B, T, H, D), 7.0, dtype=BF16, device="cuda")
    assert launches(lambda: attend(c, out=out)) == 3
    close(out, c)
    for b, n in enumerate(new or []):
        assert bool((out[b, n:] == 7.0).all())
    assert torch.equal(attend(c, out=torch.full_like(out, 7.0)), out)
