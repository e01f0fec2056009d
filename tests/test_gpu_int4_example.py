"""The example of the 4-bit cache: what it decodes is the attention over what it stored."""

import importlib.util
from pathlib import Path

import pytest
import torch

import int4_reference as ref

pytestmark = pytest.mark.gpu


def _example():
    path = Path(__file__).resolve().parents[1] / "examples" / "int4_long_context.py"
    spec = importlib.util.spec_from_file_location("int4_long_context", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("budget", [4, 64])
def test_the_example_decodes_what_it_stored(budget):
    r = _example().run(requests=3, context=700, budget=budget, layers=2, steps=3, seed=5)
    for layer in range(2):
        view = r["pool"].layer_view(layer)
        o, l, tol_o, tol_l = ref.attend(r["q"][layer][:, None], (view.codes, view.params, view.rope), r["table"],
                                        r["seq_lens"].tolist(), r["sm_scale"])
        out, lse = r["out"]["all"][layer][:, None].double().to(o.device), r["lse"]["all"][layer][:, None].double().to(o.device)
        assert ((out - o).abs() <= tol_o).all()
        assert ((lse - l).abs() <= tol_l).all()
    assert (r["lse"]["chosen"] <= r["lse"]["all"] + 1e-3).all()
    if budget >= 11:  # every page is chosen
        assert torch.equal(r["out"]["all"], r["out"]["chosen"])
