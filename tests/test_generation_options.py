"""Command-line options of the generation harness that do not go together: refused before a model is built, not ignored."""
import sys

import pytest

import gpt2_generation as gen


@pytest.mark.parametrize("extra", [["--fused-step-ops"], ["--fused-add-ln", "--fused-step-ops"]], ids=" ".join)
def test_step_ops_are_not_reported_where_they_are_not_used(monkeypatch, capsys, extra):
    """gpt2_greedy_step takes one position for all rows; the paged loop has one for each."""
    monkeypatch.setattr(gen, "build_model", lambda *a, **k: pytest.fail("a model was built"))
    monkeypatch.setattr(sys, "argv", ["gpt2_generation.py", "--device", "cpu", "--kv-cache", "--cache-bits", "4", *extra])
    with pytest.raises(SystemExit) as e:
        gen.main()
    assert e.value.code == 2 and "--fused-step-ops" in capsys.readouterr().err.splitlines()[-1]


@pytest.mark.parametrize("backend", ["NAIVE_PYTORCH", "PYTORCH_SDPA_MATH"])
def test_no_other_attention_is_reported_than_the_one_that_runs(monkeypatch, capsys, backend):
    """The paged loop has its own attention, whatever --backend says."""
    monkeypatch.setattr(gen, "build_model", lambda *a, **k: pytest.fail("a model was built"))
    monkeypatch.setattr(sys, "argv", ["gpt2_generation.py", "--device", "cpu", "--kv-cache", "--cache-bits", "4", "--backend", backend])
    with pytest.raises(SystemExit) as e:
        gen.main()
    assert e.value.code == 2 and "--backend" in capsys.readouterr().err.splitlines()[-1]


def test_a_pool_of_no_pages_is_refused():
    """num_pages=0 is a number of pages, and too few; None is the default."""
    from causal_self_attention import ScaledDotProductAttentionBackend as Backend

    m = gen.build_model("gpt2", Backend.NAIVE_PYTORCH, "cpu", overrides=dict(emb_dim=64, n_heads=1, n_layers=1, vocab_size=11, context_length=32))
    with pytest.raises(ValueError, match="num_pages"):
        gen.PagedGreedyGenerator(m, 1, 32, use_graphs=False, page_size=16, num_pages=0, ops=object())
    assert gen.PagedGreedyGenerator(m, 3, 20, use_graphs=False, page_size=16, ops=object()).cache.num_pages == 6
