"""CPU tests of nnzap_b200.score's host side: a model whose step makes logits
up, and a plain form of token_logprobs in place of the kernel."""
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")
VOCAB, PAGE = 50, 4


@pytest.fixture
def score(built_lib, monkeypatch):
    from nnzap_b200 import paged, score

    def token_logprobs(logits, tokens, top_k=0):
        lp = torch.log_softmax(logits.double(), -1)
        val, idx = torch.sort(lp, dim=-1, descending=True, stable=True)
        t = tokens.long()
        none = torch.isneginf(logits).all(-1) | torch.isnan(logits).all(-1)
        ids = torch.where(none[:, None], -1, idx[:, :top_k])
        return types.SimpleNamespace(logprob=torch.where(t < 0, 0.0, lp.gather(1, t.clamp(0)[:, None])[:, 0]), entropy=-(lp.exp() * lp).sum(-1),
                                     top_ids=ids.int(), top_logprobs=val[:, :top_k])
    monkeypatch.setattr(paged, "token_logprobs", token_logprobs)
    monkeypatch.setattr(paged, "stream_check", lambda *a: None)
    return score


class Model:
    """Steps are noted; token t's logits prefer t + 1."""
    def __init__(self, pages=100, max_context=64, logits=None):
        self.device, self.page_size, self.free, self.steps, self.used = torch.device("cpu"), PAGE, list(range(pages)), [], 0
        self.config = types.SimpleNamespace(vocab_size=VOCAB, max_context_length=max_context)
        self.pages, self.logits = pages, logits

    def step(self, tokens, positions, slots, page_table, q_start, kv_len, max_new):
        self.steps.append(tokens.tolist())
        self.used = max(self.used, self.pages - len(self.free))
        if self.logits is not None:
            return self.logits(tokens)
        out = torch.zeros(len(tokens), VOCAB)
        out[torch.arange(len(tokens)), (tokens.long() + 1) % VOCAB] = 5.0
        return out


def test_scores_and_continues(score):
    m = Model()
    out = score.score(m, [[3, 4, 9], [7]], new_tokens=2, budget=3)
    assert [s.tokens for s in out] == [[3, 4, 9, 10, 11], [7, 8, 9]] and sorted(m.free) == list(range(100))
    assert [len(s.logprobs) for s in out] == [4, 2]


@pytest.mark.parametrize("prompts,kw", [([[1, VOCAB]], {}), ([[1], [2, -1]], {}), ([[1], []], {}), ([[1] * 66], {}), ([[1] * 60], dict(new_tokens=6)),
                                        ([[1]], dict(new_tokens=-1)), ([[1]], dict(budget=0)), ([[1]], dict(top_k=0)), ([[1]], dict(top_k=33))])
def test_refusals_come_before_any_step(score, prompts, kw):
    m = Model()
    with pytest.raises(ValueError):
        score.score(m, prompts, **kw)
    assert not m.steps and sorted(m.free) == list(range(100))


@pytest.mark.parametrize("quant", ["q1_0", "q4_mlx"])
def test_embedding_rows_of_ids_that_are_none(score, quant):
    rng = np.random.default_rng(0)
    cfg = types.SimpleNamespace(quant_format=quant, group_size=64, scale_dtype="f16", q1_scales_are_mlx=False)
    M, K = 6, 128
    part = {"weight": rng.integers(0, 256, M * K // (8 if quant == "q1_0" else 2), dtype=np.uint8),
            "scales": rng.standard_normal(M * K // 64).astype(np.float16), "biases": rng.standard_normal(M * K // 64).astype(np.float16)}
    w = score._Weights(cfg, [part], K, "cpu")
    rows = w.rows(torch.tensor([2, -1, M, 2 ** 31 - 1, 5]))
    assert torch.isnan(rows[1:4]).all() and torch.isfinite(rows[[0, 4]]).all()
    assert torch.equal(rows[[0, 4]], w.rows(torch.tensor([2, 5])))


@pytest.mark.parametrize("bad", [float("nan"), -float("inf")])
def test_no_token_to_continue_with(score, bad):
    m = Model(logits=lambda tokens: torch.where((tokens == 8)[:, None], bad, torch.zeros(len(tokens), VOCAB)))
    out = score.score(m, [[8, 1]], new_tokens=1)                     # a row that nobody continues from is no error
    assert out[0].tokens == [8, 1, 0]
    with pytest.raises(RuntimeError, match="prompt 1"):
        score.score(m, [[1, 2], [1, 8]], new_tokens=1)
    assert sorted(m.free) == list(range(100))


def test_pages_of_finished_sequences_serve_the_others(score):
    """Five sequences of 5 to 9 tokens in a pool that holds the longest alone: what a large pool gives."""
    prompts = [list(range(n)) for n in (7, 5, 6, 5, 7)]
    want = score.score(Model(), prompts, new_tokens=2, budget=6)
    m = Model(pages=3)
    got = score.score(m, prompts, new_tokens=2, budget=6)
    assert got == want and sorted(m.free) == [0, 1, 2]
    m = Model()
    score.score(m, prompts, new_tokens=2, budget=100)
    assert m.used == 10                                       # all five in the first step, 2 pages each
    m = Model(pages=2)
    with pytest.raises(MemoryError):
        score.score(m, prompts, new_tokens=3, budget=6)
    assert sorted(m.free) == [0, 1]
