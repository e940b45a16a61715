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


# What each family's mixers and feed-forwards do, and the 8-bit matrices that its parts hold once loaded.
FAMILIES = {
    "tiny-a": (["attention", "swiglu"], []),
    "dibepel-tiny": (["swiglu"], ["composed_attention"]),
    "milozen-tiny": (["swiglu", "experts"], ["latent_attention"]),
    "felavik-tiny": (["experts"], ["composed_attention", "decay_attention"]),
    "nolavik-tiny": (["experts"], ["composed_attention", "gated_delta", "latent_attention", "selective_scan"]),
    "zotunex-tiny": (["experts"], ["composed_attention", "latent_attention", "ungated"]),
    "ramolix-tiny": (["swiglu"], ["composed_attention", "latent_attention", "state_space"]),
}
HELD = {"attention": {"qkv_weight", "o_weight"}, "swiglu": {"gate_up", "down"}, "experts": {"w_gate_up", "w_down"}}


@pytest.mark.parametrize("name", FAMILIES)
def test_which_matrices_a_family_holds_in_8_bits(name, products):
    """And a warning names the parts that keep theirs."""
    import warnings

    from llmserve.config.registry import architecture_of, preset
    from llmserve.parts.model import Model

    config = preset(name)
    arch = architecture_of(config)
    held, kept = FAMILIES[name]
    with warnings.catch_warnings(record=True) as seen:
        warnings.simplefilter("always")
        model = Model(arch.build_spec(arch.config_class.from_dict(config)), BuildContext(BF16, CPU, "float8"))
    got = model.float8_parts()
    assert set(got[0]) == set(held) and set(got[1]) == set(kept)
    assert len(seen) == (1 if kept else 0)
    for kind in kept:
        assert kind in str(seen[0].message)
    model.load({name: torch.zeros(info.shape, dtype=BF16) for name, info in model.param_infos().items()})
    holders = set()
    for _, part in model._parts():
        for one in (part, *getattr(part, "members", ()), getattr(part, "shared_unit", None)):
            if one is None:
                continue
            in_8_bits = {n for n, v in vars(one).items() if isinstance(v, ops.Float8)}
            if in_8_bits:
                assert in_8_bits == HELD[one.spec.kind]
                holders.add(one.spec.kind)
            else:
                assert one.spec.kind not in HELD
    assert set(held) <= holders <= set(held) | {"swiglu"}  # (the unit beside the experts is one)


def test_a_model_in_its_own_type_is_not_warned_of(recwarn):
    from llmserve.config.registry import architecture_of, preset
    from llmserve.parts.model import Model

    config = preset("ramolix-tiny")
    arch = architecture_of(config)
    Model(arch.build_spec(arch.config_class.from_dict(config)), BuildContext(BF16, CPU))
    assert not len(recwarn)


@pytest.mark.parametrize("flags,weights", [([], "model"), (["--weights", "model"], "model"), (["--weights", "float8"], "float8")])
def test_the_command_line_hands_the_option_on(flags, weights, monkeypatch):
    from llmserve import cli
    from llmserve.engine import llm

    class Seen(Exception):
        pass

    def made(model, *, engine, **options):
        engine.validate()
        raise Seen(engine.weights)

    monkeypatch.setattr(llm, "LLM", made)
    with pytest.raises(Seen, match=f"^{weights}$"):
        cli.main(["--model", "tiny", *flags])


def test_the_command_line_refuses_other_weights(capsys):
    from llmserve import cli

    with pytest.raises(SystemExit):
        cli.main(["--model", "tiny", "--weights", "int4"])
    assert "float8" in capsys.readouterr().err


@pytest.mark.parametrize("n,k", [((1 << 32) - (1 << 23), 128), (262144 - 512, 16384), (2, 1 << 23)])
def test_weights_beyond_32_bit_offsets_are_refused(n, k):
    n = n // 128 if k == 128 else n
    w = ops.Float8(torch.empty((n, k), dtype=torch.float8_e4m3fn, device="meta"),
                   torch.empty((-(-n // 128), ops.float8_scale_columns(k)), dtype=torch.float8_e8m0fnu, device="meta"), k)
    with pytest.raises(ValueError, match="too large"):
        ops.gemm_float8(torch.empty((1, n), dtype=torch.float32, device="meta"), torch.empty((1, k), dtype=BF16, device="meta"), w)


def test_a_result_on_its_own_rows_is_refused():
    """Workgroups store theirs while others read X."""
    x8 = ops.empty_float8(4, 256, "cpu")
    x8.values.view(torch.uint8).zero_()
    w = ops.Float8(torch.zeros(512, 256).to(torch.float8_e4m3fn), torch.ones(4, 4).to(torch.float8_e8m0fnu), 256)
    with pytest.raises(ValueError, match="lie on x"):
        ops.gemm_float8(x8, x8, w, swiglu=True)
    x = torch.zeros(4, 256, dtype=BF16)
    with pytest.raises(ValueError, match="lie on x"):
        ops.gemm_float8(x, x, w, swiglu=True)
    with pytest.raises(ValueError, match="GPU tensors only"):  # (beside it in one matrix: not refused for that)
        both = torch.zeros(4, 512, dtype=BF16)
        ops.gemm_float8(both[:, 256:], both[:, :256], w, swiglu=True)
