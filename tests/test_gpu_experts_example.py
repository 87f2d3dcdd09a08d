"""The example of a packed mixture-of-experts block, at a small size: what it says of itself has to hold."""

from __future__ import annotations

import runpy
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).parents[1] / "examples" / "experts_and_adapters.py"


def test_served_trained_and_merged():
    said = runpy.run_path(str(EXAMPLE))["main"](["--hidden", "256", "--inner", "128", "--experts", "8", "--best", "2",
                                                 "--tokens", "200", "--rank", "8", "--steps", "30"])
    # inputs in 4 bits: steps of 2^-1 to 2^-2 of the value, rms about a tenth a product, three products in a row
    assert 0 < said["prompt, 4-bit inputs: distance to 16-bit ones"] < 0.5
    assert said["last token alone: distance to the prompt's"] < 2.0**-6  # the same products, summed in another order
    assert said["LoRA loss, step 30"] < 0.5 * said["LoRA loss, step 1"]
    assert said["adapter merged: distance"] < said["without the adapter: distance"]
    assert said["rows of expert 1 that changed"] == 25
    assert said["rows of other experts that changed"] == 0
