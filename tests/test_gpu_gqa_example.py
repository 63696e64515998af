"""The serving example runs its operators together: logits of every step against a plain recomputation."""
import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_gqa_serve_example(cuda, capsys):
    path = Path(__file__).resolve().parent.parent / "examples" / "gqa_serve.py"
    spec = importlib.util.spec_from_file_location("gqa_serve", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # attention outputs differ by bf16 roundings (2^-8 of a value, twice: the weights and the result); two layers and the
    # projections behind them average over 256 or more of these, so the logits stay well within 2^-6 of the largest
    assert example.main() < 2.0 ** -6
    out = capsys.readouterr().out
    assert "150 from the prefix store" in out and out.count("from the prefix store") == 4
