"""The example that answers from retrieved passages, against each request run through on its own."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("answer_from_passages",
                                                  os.path.join(ROOT, "examples", "answer_from_passages.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def alone(model, tokens):
    """Logits of one whole sequence in 32 bits: no cache, no shared prefix, no operator of the library."""
    n, group = tokens.shape[0], model.heads // model.kv
    turns = model.turns[:n]
    half = model.dim // 2

    def attend(i, q, k, v, w, positions):
        def turned(x):
            x = x.float()
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
            a, b = x[..., :half], x[..., half:]
            c, s = turns[:, None, :half], turns[:, None, half:]
            return torch.cat([a * c - b * s, b * c + a * s], -1)
        q, k, v = turned(q), turned(k).repeat_interleave(group, 1), v.float().repeat_interleave(group, 1)
        score = torch.einsum("qhd,khd->hqk", q, k) * model.dim ** -0.5
        score = score.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -float("inf"))
        return torch.einsum("hqk,khd->qhd", score.softmax(-1), v).to(model.embed.dtype)
    return model.forward(tokens, torch.arange(n, device="cuda"), attend)


def test_example_matches_whole_sequences(example):
    torch.manual_seed(1)
    model = example.Decoder(seed=3)
    prompt = torch.randint(0, 2000, (531,), device="cuda")
    cache = example.Cache(model, pages=120)
    shared, first = example.read_prompt(model, cache, prompt)
    questions = torch.randint(0, 2000, (5, 6), device="cuda")
    tokens, logits = example.answer(model, cache, shared, prompt.shape[0], questions, steps=14)
    assert tokens.shape == (5, 14)

    def near(got, want):
        # bf16 activations through two layers: the two orders of rounding differ by a few units of 2^-8 of the scale
        assert (got.float() - want.float()).norm() <= 2.0 ** -5 * want.float().norm()
    near(first, alone(model, prompt))
    for b in range(5):
        fed = torch.cat([questions[b], tokens[b, :-1]])
        want = alone(model, torch.cat([prompt, fed]))[prompt.shape[0]:]
        near(logits[b], want)


def test_example_retrieves_and_answers(example, capsys):
    example.main()
    text = capsys.readouterr().out
    assert "1000 tokens of 25 passages read once; 12 answers of 20 tokens" in text


def test_retrieve_finds_the_nearest(example):
    torch.manual_seed(2)
    passages = torch.randn(3000, 64, device="cuda")
    got = example.retrieve(passages[77:78].contiguous(), passages, 9)
    want = (passages - passages[77]).square().sum(1).argsort()[:9]
    assert got[0] == 77 and set(got.tolist()) == set(want.tolist())
