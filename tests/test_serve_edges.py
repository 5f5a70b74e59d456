"""Calls of the serving operators and of the sampler at the edges of what they say of themselves: pools without a page, prompts that end inside a page, settings out of range, words equal to the last that top_k keeps, draws without a GPU, numbers of more than 32 bits."""
import json
import textwrap
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from leopard_b200 import _lib, cli, ops
from leopard_b200.sampling import Sampler, SamplingParams
from oracle import serve as O
from test_serve_ops import close
from test_serve_run import DEFINITIONS

gpu = pytest.mark.gpu
BF16, F32, I32, I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------ rotary positions and cache rows
@gpu
@pytest.mark.parametrize("pages, size, G", [(0, 16, 2), (3, 0, 2), (3, 16, 0)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_queries_are_turned_though_the_pool_has_no_rows(pages, size, G, dtype, layout):
    """no slot is a row of the pool, so that no key goes anywhere; the queries are those of `rotary`, to the last bit, as a new tensor, into one given and in place"""
    rows, H, D = 7, 3, 32
    q = torch.randn(rows, H, D, generator=gen(1), device="cuda").to(dtype)
    k, v = (torch.randn(rows, G, D, generator=gen(s), device="cuda").to(dtype) for s in (2, 3))
    pos = torch.arange(5, 5 + rows, device="cuda", dtype=I32)
    freq = (1000.0 ** (-torch.arange(8, dtype=torch.float64) / 8)).float().cuda()
    slots = torch.arange(rows, device="cuda")
    pools = [torch.zeros(pages, size, G, D, dtype=dtype, device="cuda") for _ in range(2)]
    want = ops.rotary(q, pos, freq, layout=layout, scale=1.5)
    assert not torch.equal(want, q)
    rest = (pos, freq, *pools, slots)
    given, mine = torch.full_like(q, 7.0), q.clone()
    got = ops.rotary_append(q, k, v, *rest, layout=layout, scale=1.5)
    assert torch.equal(got, want)
    assert ops.rotary_append(q, k, v, *rest, layout=layout, scale=1.5, q_out=given) is given and torch.equal(given, want)
    assert ops.rotary_append(mine, k, v, *rest, layout=layout, scale=1.5, q_out=mine) is mine and torch.equal(mine, want)
    with pytest.raises(ValueError, match="layout"):
        ops.rotary_append(q, k, v, *rest, layout="pairs")
    assert ops.rotary_append(q[:0], k[:0], v[:0], pos[:0], freq, *pools, slots[:0]).shape == (0, H, D)


# ------------------------------------------------------------------------------------------------------------ a shared prompt, as the user documentation has it
def readme_steps():
    """the documented lines for a shared prompt -> (those of the prompt, those of a step)"""
    text = (Path(__file__).resolve().parents[1] / "README.md").read_text()
    text = text[text.index("## Serving many continuations of one prompt"):]
    code = textwrap.dedent("\n".join(line for line in text.splitlines() if line.startswith("    ")))
    cut = code.index("# once a step")
    return code[:cut], code[cut:]


def by_readme(device, ops, prefix, page_size):
    """Requests that share a prompt's pages by their tables bring a few tokens each, some wait: after each step every request's sequence is in its pages, the prompt's rows and then its own, which nobody else has
    written over, and what it attends to is that sequence."""
    setup, step = readme_steps()
    B, H, G, D, max_pages, n_pages = 5, 8, 2, 64, -(-(prefix + 9) // page_size), 90      # (9 tokens at most behind the prompt)
    g = gen(prefix, "cpu")
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF16).to(device)  # noqa: E731
    i32 = lambda x: torch.tensor(x, dtype=I32, device=device)  # noqa: E731
    k_pages, v_pages = (torch.full((n_pages, page_size, G, D), float("nan"), dtype=BF16, device=device) for _ in range(2))
    order = torch.randperm(n_pages, generator=g).to(I32).to(device)
    n = -(-prefix // page_size)
    freq = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().to(device)
    ns = {"torch": torch, "ops": ops, "B": B, "max_pages": max_pages, "prefix": prefix, "page_size": page_size, "prompt_pages": order[:n].clone(), "k_pages": k_pages, "v_pages": v_pages,
          "free_pages": order[n:].clone(), "used": i32([3]), "inv_freq": freq, "lengths": i32([prefix] * B)}
    prompt = [rnd(prefix, G, D) for _ in range(2)]
    for i in range(prefix):
        for pool, x in zip((k_pages, v_pages), prompt):
            pool[int(order[i // page_size]), i % page_size] = x[i]
    seqs = [[(prompt[0][i].double(), 2.0 ** -20, prompt[1][i]) for i in range(prefix)] for _ in range(B)]      # key, what it may be off by, value
    exec(setup, ns)
    for new in ([3, 0, 1, 4, 2], [1, 1, 0, 1, 1], [4, 4, 4, 4, 4]):
        rows, T = -(-sum(new) // 8) * 8, max(new)
        before = ns["lengths"].clone()
        k, v = rnd(rows, G, D), rnd(rows, G, D)
        logits, u = torch.randn(B, 40, generator=g).to(device), torch.rand(B, generator=g).to(device)
        ns.update(new=i32(new), rows=rows, T=T, q=rnd(rows, H, D), k=k, v=v, logits=logits, uniform=u)
        exec(step, ns)
        r = 0
        for b, t in enumerate(new):
            for i in range(t):
                turned, _ = O.rotary(k[r:r + 1], torch.tensor([len(seqs[b])], device=device), freq)
                seqs[b].append((turned[0], 2.0 ** -8 * turned[0].abs() + 2.0 ** -18 * k[r].double().abs().amax(), v[r]))      # half a step; angles of fp32
                r += 1
        slots = ns["slots"][:r].tolist()
        assert min(slots) >= 0 and len(set(slots)) == r and ns["slots"][r:].tolist() == [-1] * (rows - r)
        assert ns["lengths"].tolist() == [len(s) for s in seqs]
        for b, s in enumerate(seqs):
            at = torch.arange(len(s), device=device)
            where = (ns["page_table"][b, at // page_size].long(), at % page_size)
            for i, (key, off, value) in enumerate(s):
                assert bool(((k_pages[where][i].double() - key).abs() <= off).all()) and torch.equal(v_pages[where][i], value), (b, i)
        close(ns["out"], {"q": ns["q"][ns["at"]], "k": k_pages.nan_to_num(0.0), "v": v_pages.nan_to_num(0.0), "lengths": before, "prefix": prefix, "new": ns["new"], "page_table": ns["page_table"],
                          "prefix_k": None, "prefix_v": None})
        assert ns["token"].tolist() == O.sample_tokens(logits, u, temperature=0.8, top_k=50, top_p=0.95)


@pytest.mark.parametrize("prefix, page_size", [(37, 16), (32, 16), (5, 8), (3, 1)])
def test_the_readme_serves_a_shared_prompt_by_the_definitions(prefix, page_size):
    tables, append, attend, draw, copy_pages = DEFINITIONS
    by_readme("cpu", SimpleNamespace(step_tables=tables, rotary_append=append, sample_tokens=draw, cache_copy_pages=copy_pages,
                                     prefix_attention=lambda q, k, v, lengths, P, new, page_table: attend(q, k, v, lengths, P, new, page_table)), prefix, page_size)


@gpu
@pytest.mark.parametrize("prefix, page_size", [(37, 16), (32, 16), (5, 8), (3, 1), (515, 64)])
def test_the_readme_serves_a_shared_prompt(prefix, page_size):
    by_readme("cuda", ops, prefix, page_size)


# ------------------------------------------------------------------------------------------------------------ the sampler
@pytest.mark.parametrize("option, value", [("top_p", 1.5), ("top_p", 0.0), ("top_p", -0.5), ("top_p", float("nan")), ("min_p", 2.0), ("min_p", -0.1), ("min_p", float("nan"))])
def test_settings_out_of_range_are_refused_before_a_prompt_runs(monkeypatch, option, value):
    with pytest.raises(ValueError, match=option):
        SamplingParams(temperature=0.8, **{option: value})
    with pytest.raises(ValueError, match=option):
        SamplingParams(temperature=0.8, **{"min_p": 0.1, "top_p": 0.9, option: value})
    monkeypatch.setattr(cli, "_load", lambda args: pytest.fail("the model was loaded"))
    with pytest.raises(ValueError, match=option):
        cli.main(["generate", "--model", "m", "--prompt", "1,2", "--temperature", "0.8", f"--{option.replace('_', '-')}={value}"])


def test_settings_at_the_ends_of_their_ranges_are_taken():
    for kw in (dict(), dict(top_p=1.0, min_p=0.0), dict(top_p=1, min_p=1), dict(top_p=1e-9, min_p=1.0)):
        assert SamplingParams(temperature=0.8, **kw).min_p == kw.get("min_p", 0.0)


def keeps_the_same_words(device):
    """logits of few steps, so that many words are equal to the k-th: the draws come from the words that top_k alone keeps, and all of these come up"""
    z = torch.tensor([0.5, 2.0, 1.0, 1.0, 2.0, 0.5, 1.0, -3.0, 1.0], device=device).expand(4000, 9).contiguous()
    for top_k, words in ((1, {1, 4}), (2, {1, 4}), (3, {1, 2, 3, 4, 6, 8}), (6, {1, 2, 3, 4, 6, 8}), (7, {0, 1, 2, 3, 4, 5, 6, 8}), (8, {0, 1, 2, 3, 4, 5, 6, 8}), (9, set(range(9))), (0, set(range(9)))):
        for kw in (dict(), dict(top_p=0.999999), dict(min_p=1e-6), dict(top_p=0.999999, min_p=1e-6)):      # (the least likely word has 1.5 % of the mass)
            drawn = Sampler(SamplingParams(temperature=2.0, top_k=top_k, seed=3, **kw))(z)
            assert set(drawn.tolist()) == words, (top_k, kw)


@gpu
def test_top_k_keeps_the_same_words_with_other_settings_and_without():
    keeps_the_same_words("cuda")


# ------------------------------------------------------------------------------------------------------------ the sampler without a GPU
def test_top_k_keeps_the_same_words_without_a_gpu():
    keeps_the_same_words("cpu")


@pytest.mark.parametrize("kw", [dict(top_p=0.8), dict(min_p=0.1), dict(top_p=0.95, min_p=0.02), dict(top_p=1e-6), dict(min_p=1.0), dict(top_p=0.999, temperature=3.0), dict(top_k=20, top_p=0.9)])
@pytest.mark.parametrize("V", [1, 7, 700])
def test_the_sampler_draws_by_the_definition_without_a_gpu(kw, V):
    z = torch.randn(40, V, generator=gen(V, "cpu")) * 2
    z[3] = -torch.inf
    z[4, V // 2:] = float("nan")
    z[5, ::3] = torch.inf
    z[6, :] = 0.25
    kw = {"temperature": 0.9, **kw}
    rows = [r for r in range(40) if "top_k" not in kw or r not in (4, 5, 6)]      # (numbers that are none, and more than 20 equal ones: the sampler's top_k is another than the draw's)
    got = Sampler(SamplingParams(seed=11, **kw))(z)
    want = O.sample_tokens(z, torch.rand(40, generator=gen(11, "cpu")), **kw)
    assert got.dtype == I64 and [got.tolist()[r] for r in rows] == [want[r] for r in rows]


class FewWords:
    """an engine whose logits are numbers of its own"""
    def __init__(self):
        self.g = gen(9, "cpu")

    def step(self, entries):
        return torch.randn(len(entries), 50, generator=self.g)

    def finish(self, key):
        pass


def test_the_command_line_draws_with_its_settings(monkeypatch, capsys):
    """generate's options reach the draw: the same engine's logits, drawn by the definition"""
    monkeypatch.setattr(cli, "_load", lambda args: FewWords())
    assert cli.main(["generate", "--model", "m", "--prompt", "1,2", "--prompt", "3", "--max-new-tokens", "4", "--temperature", "0.8", "--top-p", "0.7", "--min-p", "0.05", "--seed", "5"]) == 0
    printed = [json.loads(line) for line in capsys.readouterr().out.splitlines()]
    eng, numbers, want = FewWords(), gen(5, "cpu"), [[], []]
    for _ in range(4):
        drawn = O.sample_tokens(eng.step([0, 1]), torch.rand(2, generator=numbers), temperature=0.8, top_p=0.7, min_p=0.05)
        for o, t in zip(want, drawn):
            o.append(t)
    assert printed == [{"prompt": [1, 2], "output": want[0]}, {"prompt": [3], "output": want[1]}]


def least_top_p(device):
    """a top_p that is 0 in 32 bits keeps the likeliest word, as all below its share of the mass do"""
    z = torch.randn(30, 300, generator=gen(2, "cpu")).to(device)
    for top_p in (1e-50, 1e-45, 1e-30, 1e-9):
        assert torch.equal(Sampler(SamplingParams(temperature=1.0, top_p=top_p, seed=1))(z), z.argmax(-1))


def test_the_least_top_p_without_a_gpu():
    least_top_p("cpu")


# ------------------------------------------------------------------------------------------------------------ numbers of more than 32 bits
@gpu
def test_the_least_top_p():
    least_top_p("cuda")


@gpu
def test_a_top_k_of_more_than_32_bits_keeps_all():
    z, u = torch.randn(6, 500, generator=gen(4), device="cuda"), torch.rand(6, generator=gen(5), device="cuda")
    want = O.sample_tokens(z, u)
    for top_k in (2 ** 31 - 1, 2 ** 31, 2 ** 32 - 1, 2 ** 32 + 1, 2 ** 40, 2 ** 63 - 1):
        assert ops.sample_tokens(z, u, top_k=top_k).tolist() == want, top_k
    for top_k in (-2 ** 32, -2 ** 32 + 1, -2 ** 31):
        with pytest.raises(_lib.NativeError, match="top_k"):
            ops.sample_tokens(z, u, top_k=top_k)


@gpu
def test_sizes_of_more_than_32_bits_are_refused():
    i32 = lambda x: torch.tensor(x, dtype=I32, device="cuda")  # noqa: E731
    for size, rows in ((2 ** 32 + 16, 8), (2 ** 31, 8), (16, 2 ** 32 + 8), (16, 2 ** 31)):
        with pytest.raises(ValueError, match="32 bits"):
            ops.step_tables(i32([5, 30]), i32([4, 4]), i32([[-1, -1, -1]] * 2), i32([3, 4, 5, 6]), i32([0]), size, rows)
    q, k = torch.zeros(2, 1, 4, 64, dtype=BF16, device="cuda"), torch.zeros(9, 16, 2, 64, dtype=BF16, device="cuda")
    for prefix in (2 ** 32 + 20, 2 ** 31, -2 ** 32):
        with pytest.raises(ValueError, match="32 bits"):
            ops.prefix_attention(q, k, k, i32([25, 25]), prefix, page_table=i32([[0, 1], [0, 2]]))
