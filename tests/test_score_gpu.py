"""The ragged-serving operators together: a small quantized model that scores
and continues several prompts over one paged cache, against the oracle."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant,gs,style,page,budget", [("q1", 128, "pairwise", 16, 64), ("q4", 64, "half_split", 8, 23), ("q1", 128, "pairwise", 5, 512)])
def test_score_matches_the_oracle(cuda, built_lib, quant, gs, style, page, budget):
    from nnzap_b200 import config_from_dims, synth
    from nnzap_b200.score import PagedModel, score
    from oracle import qwen3_ref as R
    d = synth.ModelDims(vocab=1000, hidden=256, inter=768, layers=2, n_q=4, n_kv=2, head_dim=128, gs=gs, quant=quant, rope_style=style)
    W = synth.make_model(d, seed=3)
    cfg = R.Cfg(vocab=d.vocab, hidden=d.hidden, inter=d.inter, layers=d.layers, n_q=d.n_q, n_kv=d.n_kv, head_dim=d.head_dim, gs=d.gs,
                quant=d.quant, rope_style=style)
    m = PagedModel(config_from_dims(d, max_context_length=256), synth.iter_named_tensors(W), num_pages=300 // page + 8, page_size=page)
    free = len(m.free)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, d.vocab, n).tolist() for n in (70, 1, 33, 2)]
    out = score(m, prompts, new_tokens=3, budget=budget, top_k=4)
    assert len(m.free) == free
    for p, s in zip(prompts, out):
        n = len(p)
        assert s.tokens[:n] == p and len(s.tokens) == n + 3 and len(s.logprobs) == n + 2
        lg = R.forward_tokens(cfg, W, s.tokens).astype(np.float64)
        lp = lg - np.log(np.exp(lg - lg.max(-1, keepdims=True)).sum(-1, keepdims=True)) - lg.max(-1, keepdims=True)
        # logits of the engine's precision are within 2e-2 of the oracle's: log
        # probabilities within twice that
        got = np.array(s.logprobs)
        want = lp[np.arange(n + 2), s.tokens[1:]]
        assert np.abs(got - want).max() <= 4e-2
        ent = -(np.exp(lp) * lp).sum(-1)[:n + 2]
        assert np.abs(np.array(s.entropies) - ent).max() <= 4e-2
        for i in range(n - 1, n + 2):          # greedy: the oracle's largest logit, or within the bar of it
            assert lg[i].max() - lg[i, s.tokens[i + 1]] <= 4e-2
        assert all(a >= b for t in s.top_logprobs for a, b in zip(t, t[1:]))


def test_score_matches_the_engine(cuda, built_lib):
    """The paged path and the engine's contiguous one: the same logits after a prompt."""
    from nnzap_b200 import Model, config_from_dims, synth
    from nnzap_b200.score import PagedModel, score
    d = synth.ModelDims(vocab=1000, hidden=256, inter=768, layers=2, n_q=4, n_kv=2, head_dim=128, gs=128, quant="q1")
    W = synth.make_model(d, seed=0)
    cfg = config_from_dims(d, max_context_length=256)
    m = Model(cfg)
    m.load_weights(synth.iter_named_tensors(W))
    prompt = np.random.default_rng(2).integers(0, d.vocab, 150)
    _, lg = m.prefill(prompt, want_logits=True)
    m.free()
    s = score(PagedModel(cfg, synth.iter_named_tensors(W), num_pages=16), [prompt], new_tokens=1, budget=100, top_k=8)[0]
    lp = lg.astype(np.float64) - lg.max()
    lp -= np.log(np.exp(lp).sum())
    assert np.abs(np.array(s.top_logprobs[-1]) - lp[s.top_ids[-1]]).max() <= 4e-2
    assert np.sort(lp)[-8] - lp[s.top_ids[-1]].min() <= 4e-2


def test_the_layers_share_one_workspace(cuda, built_lib):
    from nnzap_b200 import config_from_dims, synth
    from nnzap_b200.score import PagedModel
    d = synth.ModelDims(vocab=1000, hidden=256, inter=768, layers=3, n_q=4, n_kv=2, head_dim=128, gs=128, quant="q1")
    m = PagedModel(config_from_dims(d, max_context_length=64), synth.iter_named_tensors(synth.make_model(d, seed=0)), num_pages=4)
    assert len({id(L["attend"].workspace) for L in m.layers}) == 1
