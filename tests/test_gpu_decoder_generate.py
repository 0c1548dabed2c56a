"""The example decoder's run from its prompts to the beams that are left, with one beam (the prompt's own sequence) and more."""
from __future__ import annotations

import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))


@pytest.mark.parametrize("beams", [1, 2, 4])
def test_generate(beams, capsys):
    from decoder import Decoder, generate

    m = Decoder(layers=2, d=512, heads=4, kv_heads=2, head_dim=128, ffn=512)
    try:
        with torch.cuda.stream(m.stream):
            generate(m, SimpleNamespace(prompt=40, tokens=3, beams=beams))
        said = capsys.readouterr().out
        assert f"{beams + 1} sequences, 3 tokens each" in said
        assert len(eval(said.split("beams left:")[1])) == beams - 1
        assert m.cache.lengths([0, 1]).tolist() == [0, 0]
    finally:
        m.close()
