"""What the parts of a model do with weights in 8 bits, as far as it shows without a GPU: the operators are stand-ins that note what they are given."""

import pytest
import torch

from llmserve.ops import library as ops
from llmserve.parts import model as _  # noqa: F401 (registers the parts)
from llmserve.parts.registry import FEED_FORWARDS, BuildContext
from llmserve.parts.spec import PartSpec

CPU = torch.device("cpu")
BF16 = torch.bfloat16


@pytest.fixture
def products(monkeypatch):
    """(x, out) of every product that is asked for."""
    calls = []

    def weight(w):
        *lead, n, k = w.shape
        return ops.Float8(torch.zeros(*lead, n, ops.float8_width(k), dtype=torch.float8_e4m3fn),
                          torch.zeros(*lead, -(-n // 128), ops.float8_scale_columns(k), dtype=torch.uint8).view(torch.float8_e8m0fnu), k)

    def note(out, x, *rest, **options):
        calls.append((x, out))
        return out

    monkeypatch.setattr(ops, "weight_float8", weight)
    monkeypatch.setattr(ops, "gemm_float8", note)
    monkeypatch.setattr(ops, "grouped_float8", note)
    return calls


def loaded(kind, **spec):
    part = FEED_FORWARDS.build(PartSpec(kind, spec), BuildContext(BF16, CPU, "float8"))
    part.load({name: torch.zeros(info.shape, dtype=BF16) for name, info in part.param_infos().items()})
    return part


@pytest.mark.parametrize("m", [1, 16, 17, 32, 33, 64, 65, 300])
@pytest.mark.parametrize("intermediate", [100, 4096, 4100])
def test_units_are_rounded_once_whatever_the_rows(products, m, intermediate):
    """A unit goes from the first product to the second in 8 bits, not in bfloat16 and then in 8 bits, so a step that is filled up rounds as any other."""
    part = loaded("swiglu", hidden=64, intermediate=intermediate)
    part.forward(torch.zeros(m, 64, dtype=BF16))
    (_, act), (x, _) = products
    assert isinstance(act, ops.Float8) and x is act and act.columns == intermediate


@pytest.mark.parametrize("pairs", [1, 16, 64, 65, 200])
def test_units_of_experts_are_rounded_once_whatever_the_rows(products, pairs):
    part = loaded("experts", hidden=64, intermediate=100, experts=4, top=2, unit="silu")
    part._products_float8(torch.zeros(pairs, 64, dtype=BF16), None)
    (_, act), (x, _) = products
    assert isinstance(act, ops.Float8) and x is act and act.columns == 100
