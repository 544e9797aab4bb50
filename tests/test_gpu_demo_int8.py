"""The demo's two new ways: orthogonalised updates, serving in 8 bits."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("orthogonal", [False, True])
def test_demo(dtype, orthogonal):
    from xspmm_amd import feed_forward_demo

    out = feed_forward_demo.run(features=128, hidden=320, tokens=256, density=0.4, steps=5, dtype=dtype,
                                orthogonal=orthogonal)
    assert all(math.isfinite(v) for v in out.values() if isinstance(v, float))
    assert out["served_vs_batch"] < 0.01
    # what is compared is x + the layer's output, of which the roundings are some 2 %
    assert out["served_int8_vs_batch"] < 0.05
