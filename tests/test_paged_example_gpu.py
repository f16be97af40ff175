"""The operators together, as examples/parallel_answers.py uses them: reload,
append and attend per layer, fork, single tokens, free, compact."""
from __future__ import annotations

import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import parallel_answers
    return parallel_answers


@pytest.mark.parametrize("answers,chunk,steps", [(4, 75, 6), (2, 128, 3), (1, 1, 2), (5, 53, 4)])
def test_answers_match_attention_over_gathered_keys(example, answers, chunk, steps):
    r = example.run(layers=2, answers=answers, chunk_tokens=chunk, steps=steps, check=True, say=lambda *_: None)
    length = 6 * 128 + chunk + steps
    for s in r["alive"]:
        assert int(r["tables"].lens[s]) == length
    used = int((r["tables"].refs > 0).sum())
    # The shared full pages once, and each answer's own.
    shared = (6 * 128 + chunk) // 128
    assert used == shared + len(r["alive"]) * (-(-length // 128) - shared)
    assert torch.isfinite(r["output"].float()).all()
    # Two bf16 roundings (weights and result) of values up to 4.5: 2 * 2^-8 * 4.5.
    assert r["off"] <= 0.036
