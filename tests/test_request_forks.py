"""Requests that are forked and truncated: branches that share pages until one of them writes, copied states, pages that go back when the last of their holders has given
them back, tokens that are dropped.  Against the plain implementation of whole sequences, on the kernel sources under the CPU emulator and, marked gpu, on the native library."""
import pytest
import torch

from leopard_b200.seqcache import SequenceCache
from leopard_b200.seqlm import StepEntry
from oracle import ronelorn as OR
from oracle import seqlm as O
import ronelorn_common as R
from seqlm_common import TOL, backend, emu_lib, latent_layer, make_engine, mixed_model, model, rel_err  # noqa: F401  (fixtures)


def tokens(n, vocab, seed):
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def windowed(kinds):
    return model([latent_layer(window=w) for w in kinds])


CASES = {"mixed": (mixed_model, O, make_engine), "pooled": (R.mixed_model, OR, R.make_engine), "attention": (lambda: windowed((9, None)), O, make_engine)}


@pytest.mark.parametrize("which", list(CASES))
@pytest.mark.parametrize("prompt", [3, 4, 11])
def test_branches_go_their_own_ways(backend, which, prompt):
    """one prompt, forked at a page's border and inside of one, forked again later; the branches run in the same steps and alone"""
    make, oracle, engine = CASES[which]
    cfg = make()
    w = oracle.random_weights(cfg, seed=7)
    eng = engine(cfg, w, backend)
    seqs = {"a": tokens(prompt, cfg["vocab"], 1)}
    got = {"a": [eng.step([StepEntry("a", seqs["a"], list(range(prompt)))])]}

    def fork(old, new):
        eng.fork(old, new)
        seqs[new], got[new] = list(seqs[old]), list(got[old])

    def go(keys, n, seed):
        new = {k: tokens(n, cfg["vocab"], seed + i) for i, k in enumerate(keys)}
        out = eng.step([StepEntry(k, new[k], list(range(n))) for k in keys])
        for i, k in enumerate(keys):
            seqs[k] += new[k]
            got[k].append(out[i * n:(i + 1) * n])
    fork("a", "b")
    go(["a", "b"], 1, 10)
    go(["b", "a"], 1, 20)
    fork("b", "c")
    go(["c"], 5, 30)
    go(["a", "b", "c"], 1, 40)
    eng.finish("b")
    fork("c", "d")
    eng.finish("c")
    go(["a", "d"], 6, 50)
    for k in ("a", "b", "d"):
        assert rel_err(torch.cat(got[k], 0), oracle.forward(cfg, w, seqs[k])) < TOL["float32"], k
    eng.finish("a")
    eng.finish("d")
    c = eng.cache
    assert c.pages_in_use() == 0 and not c.held and sorted(c.free_pages) == list(range(c.n_pages))
    assert all(not h for h in c.summary_held) and all(sorted(f) == list(range(n)) for f, n in zip(c.summary_free, c.summary_n_pages))
    assert sorted(c.free_slots) == list(range(c.n_slots))


@pytest.mark.parametrize("keep", [0, 1, 4, 7, 12])
def test_dropped_tokens(backend, keep):
    cfg = windowed((None, None))
    w = O.random_weights(cfg, seed=8)
    eng = make_engine(cfg, w, backend)
    first, then = tokens(13, cfg["vocab"], 1), tokens(6, cfg["vocab"], 2)
    eng.step([StepEntry("a", first, [])])
    eng.fork("a", "b")
    eng.truncate("a", keep)
    got = eng.step([StepEntry("a", then, list(range(6)))])
    assert rel_err(got, O.forward(cfg, w, first[:keep] + then)[keep:]) < TOL["float32"]
    got = eng.step([StepEntry("b", then, list(range(6)))])      # the other holder still has all of it
    assert rel_err(got, O.forward(cfg, w, first + then)[13:]) < TOL["float32"]
    eng.finish("a")
    eng.finish("b")
    assert eng.cache.pages_in_use() == 0 and not eng.cache.held


def test_what_cannot_be_dropped_is_refused(backend):
    cfg = mixed_model()
    eng = make_engine(cfg, O.random_weights(cfg, seed=9), backend)
    eng.step([StepEntry("a", tokens(9, cfg["vocab"], 1), [])])
    with pytest.raises(ValueError, match="recurrent"):
        eng.truncate("a", 5)
    with pytest.raises(ValueError, match="cannot keep 10"):
        eng.truncate("a", 10)
    eng.truncate("a", 9)
    eng.truncate("a", 0)
    with pytest.raises(KeyError):
        eng.fork("nobody", "b")
    with pytest.raises(KeyError):
        eng.fork("a", "a")


# ---- the cache alone ----------------------------------------------------------------------------------------------------
def filled(cache, seq, n):
    """n more rows, each the token's number in the sequence; what was read of the others is checked by the caller"""
    cache.reserve(seq, n)
    for i in range(seq.length, seq.length + n):
        for w, pool in enumerate(cache.pools):
            pool[seq.pages[i // cache.page_size], i % cache.page_size] = i + 1000 * w
    cache.advance(seq, n)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_pages_are_counted(device):
    c = SequenceCache([8, 8, 3], [], None, device, max_tokens=12, page_size=4, max_seqs=2)
    a = c.open("a")
    filled(c, a, 10)
    b = c.fork("a", "b")
    d = c.fork("b", "d")
    assert a.pages == b.pages == d.pages and c.pages_in_use() == 3 and c.held == {p: 3 for p in a.pages}
    filled(c, b, 1)                                       # the page that is being filled is copied, the full ones stay shared
    assert b.pages[:2] == a.pages[:2] and b.pages[2] != a.pages[2] and c.held[a.pages[2]] == 2
    for pool, w in zip(c.pools, range(3)):
        assert torch.equal(pool[b.pages[2], :3, 0].cpu(), torch.tensor([8., 9., 10.]) + 1000 * w)
    filled(c, d, 7)
    filled(c, a, 3)                                       # the last holder writes in place
    assert a.pages[2] not in c.held and len(set(a.pages[2:] + b.pages[2:] + d.pages[2:])) == len(a.pages[2:] + b.pages[2:] + d.pages[2:])
    before = c.pages_in_use()
    c.truncate("d", 6)                                    # inside a page that all three hold
    assert len(d.pages) == 2 and c.pages_in_use() == before - 3
    filled(c, d, 1)
    assert d.pages[0] == a.pages[0] and d.pages[1] != a.pages[1] and c.held[a.pages[1]] == 2
    for key in "bad":
        c.close(key)
    assert c.pages_in_use() == 0 and not c.held


def test_a_window_gives_shared_pages_back_once():
    c = SequenceCache([2], [], 5, "cpu", max_tokens=8, page_size=4, max_seqs=2)
    a = c.open("a")
    filled(c, a, 7)
    b = c.fork("a", "b")
    filled(c, a, 8)
    assert a.pages[0] == -1 and b.pages[0] >= 0 and b.pages[0] not in c.free_pages
    filled(c, b, 8)
    assert b.pages[0] == -1 and sorted(c.free_pages + [p for p in a.pages + b.pages if p >= 0]) == list(range(c.n_pages))
    with pytest.raises(ValueError, match="left the window"):
        c.truncate("a", 8)
    c.truncate("a", 13)
    assert a.length == 13


def test_forked_states_are_copies():
    c = SequenceCache([], [(2, 3), (4,), (6,)], None, "cpu", max_seqs=1)
    a = c.open("a")
    c.advance(a, 5)
    for s in c.states:
        s[a.slot] = 7.0
    b = c.fork("a", "b")
    assert b.slot != a.slot and b.length == 5 and all(bool((s[b.slot] == 7.0).all()) for s in c.states)
    c.states[0][b.slot] = 1.0
    assert bool((c.states[0][a.slot] == 7.0).all())
