"""examples/answer_from_search.py, smaller: search, attention over what was found, and training steps."""
import importlib.util
import os

import pytest

torch = pytest.importorskip("torch")

from tests.attend_plain import check, plain

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_search_attention_and_training_run_together():
    spec = importlib.util.spec_from_file_location("answer_from_search", os.path.join(ROOT, "examples", "answer_from_search.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    result = example.main(passages=2000, length=40, queries=5, found=4)
    rows = result["rows"]
    assert rows.shape == (5, 4) and (rows >= 0).all() and result["found_on_topic"] > 0.9
    got = plain(result["new"], result["states"], result["states"], rows=rows, lengths=result["lengths"])
    check("out", result["answers"], got)
    assert result["losses"][-1] < 0.8 * result["losses"][0]
