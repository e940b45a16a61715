"""The layers of engines with weights in 8 bits, product by product on the engine's own rows, against the definition in 64 bits: what is held, what is
multiplied by what, the biases, and one rounding to 8 bits in front of each product."""

import copy

import pytest
import torch

import plain_float8 as plain
from test_float8_engine_gpu import logits, runner
from test_float8_gpu import bound_of
from test_float8_sums_gpu import check_bfloat16, check_steps

pytestmark = pytest.mark.gpu


def exact_rows(out8, x):
    """Rows in 8 bits are the one rounding of the numbers x."""
    values, scale = plain.rows(x.cpu().double())
    assert torch.equal(out8.values.float().cpu().double(), values) and torch.equal(out8.scale.float().cpu().double(), scale)


def numbers(t, block_rows=1):
    return plain.numbers(t.values.float(), t.scale.float(), block_rows)


def held(w8, w):
    """A weight in 8 bits is the definition's of the checkpoint's numbers; returned as what it stands for."""
    values, scale = plain.weight(w.cpu().double())
    assert torch.equal(w8.values.float().cpu().double(), values) and torch.equal(w8.scale.float().cpu().double(), scale)
    return plain.numbers(values, scale, 128)


class Calls:
    """What the operators are given and what they return, copied as the steps go by."""

    def __init__(self, monkeypatch):
        from llmserve.ops import library as ops

        self.ops, self.seen = ops, []
        for name in ("gemm_float8", "grouped_float8", "rmsnorm_float8"):
            monkeypatch.setattr(ops, name, self.wrapped(name, getattr(ops, name)))

    def copied(self, t):
        if isinstance(t, self.ops.Float8):
            return self.ops.Float8(t.values.clone(), t.scale.clone(), t.columns)
        return t.clone() if isinstance(t, torch.Tensor) else t

    def wrapped(self, name, function):
        def call(out, *args, **options):
            before = [self.copied(a) for a in args[:1]] + list(args[1:])
            options_before = {k: self.copied(v) for k, v in options.items()}
            result = function(out, *args, **options)
            left = options.get("resid_out")
            self.seen.append((name, self.copied(result), before, options_before, None if left is None else left.clone()))
            return result
        return call


def check_norm(call, norm):
    """The stream's sum, its norm, and one rounding of that to 8 bits.  (128 units of 2^-24: a sum of squares in 32 bits by threads and then across them, root,
    reciprocal and two products.)"""
    name, out8, (x, weight, eps), options, left = call
    assert name == "rmsnorm_float8" and weight is norm.weight and eps == norm.eps
    r = x.double()
    if options["delta"] is not None:
        summed = r + options["delta"].double()
        assert ((left.double() - summed).abs() <= summed.abs() * (2.0 ** -8 + 2.0 ** -23)).all()
        r = left.double()
    v = (r / torch.sqrt(r.square().mean(dim=1, keepdim=True) + eps) * weight.double()).cpu()
    check_steps(out8, v, v.abs() * 128 * 2.0 ** -24)


def product_of(x, wd, bias=None):
    """(numbers of the rows, the product with a bias in 64 bits)"""
    xd = numbers(x) if not isinstance(x, torch.Tensor) else plain.numbers(*plain.rows(x.cpu().double()))
    xd = xd[:, : wd.shape[1]]
    y = xd @ wd.t()
    return xd, y if bias is None else y + bias.cpu().double()


def check_product(out, x, wd, bias=None, sixteens=None):
    m = out.shape[0]
    xd, y = product_of(x, wd, bias)
    off = bound_of(xd, wd, y, torch.float32, m > 16 if sixteens is None else sixteens)
    if bias is not None:
        off += (y.abs() + bias.cpu().double().abs()) * 2.0 ** -23
    if out.dtype == torch.bfloat16:
        check_bfloat16(out, y, off)
    else:
        assert ((out.cpu().double() - y).abs() <= off).all()
    return y, off


def check_units(act, x, wd, sixteens, limit=None):
    """Gated units are rounded once, to 8 bits."""
    xd, y = product_of(x, wd)
    off = bound_of(xd, wd, y, torch.float32, sixteens)
    inter = wd.shape[0] // 2
    (gate, up), (dg, du) = y.split(inter, dim=1), off.split(inter, dim=1)
    want = plain.unit(gate, up, limit)
    check_steps(act, want, 1.2 * (up.abs() + du + 1) * dg + (gate.abs() + dg) * du + want.abs() * 256 * 2.0 ** -24)


ROWS = (1, 16, 17, 32, 33, 64, 65, 130)


@pytest.mark.parametrize("n", ROWS)
def test_every_product_of_a_model_with_biases(n, monkeypatch):
    """Attention with a bias on q, k and v that is as large as they are and other for each column, and feed-forwards; steps of rows on either side of
    every border between kernels."""
    from llmserve.config.registry import preset

    config = dict(preset("tiny-b"), attention_bias=True)
    options = dict(block_size=4, num_blocks=256, use_graphs=False)
    small, given = runner(config, "float8", **options), runner(config, "model", **options)
    parts = []
    for a, b in zip(small.model.blocks, given.model.blocks):
        for role in a.ROLES:
            if getattr(a.parts[role], "float8", False):
                parts.append((role, a.parts[role], b.parts[role]))
    g = torch.Generator().manual_seed(n)
    for role, part, _ in parts:
        if hasattr(part, "qkv_weight"):
            part.qkv_bias = torch.randn(part.qkv_bias.shape, generator=g).to(torch.bfloat16).to(part.qkv_bias.device)
    calls = Calls(monkeypatch)
    ids = torch.randint(0, config["vocab_size"], (n,), generator=g).tolist()
    logits(small, ids, [n])
    assert len(parts) == 2 * len(small.model.blocks) and len(calls.seen) == 3 * len(parts)
    norms = [blk.parts[role] for blk in small.model.blocks for role in blk.ROLES if hasattr(blk.parts[role], "rms_params")]
    assert len(norms) == len(parts)
    for i, (role, part, plain_part) in enumerate(parts):
        norm, first, second = calls.seen[3 * i: 3 * i + 3]
        check_norm(norm, norms[i])
        (_, out, (x, w, *bias), options, _), (_, out2, (x2, w2, *bias2), options2, _) = first, second
        assert torch.equal(x.values.view(torch.uint8), norm[1].values.view(torch.uint8)) and torch.equal(x.scale.view(torch.uint8), norm[1].scale.view(torch.uint8))
        if hasattr(part, "qkv_weight"):
            assert w is part.qkv_weight and w2 is part.o_weight and not any(b is not None for b in bias2)
            wd = held(w, plain_part.qkv_weight)
            _, off = check_product(out, x, wd, part.qkv_bias)
            assert (part.qkv_bias.cpu().double().abs() > off).double().mean() > 0.9  # (what a lost bias would be)
            check_product(out2, x2, held(w2, plain_part.o_weight))
        else:
            assert w is part.gate_up and w2 is part.down and options["swiglu"]
            # (of up to 64 rows the sums are of exact products)
            check_units(out, x, held(w, plain_part.gate_up), n > 64)
            assert torch.equal(x2.values.view(torch.uint8), out.values.view(torch.uint8))
            check_product(out2, x2, held(w2, plain_part.down))


@pytest.mark.parametrize("name", ["milozen-tiny", "nolavik-tiny", "felavik-tiny", "zotunex-tiny"])
@pytest.mark.parametrize("n", [1, 30, 90])
def test_every_product_of_experts(name, n, monkeypatch):
    """Rows of the step's tokens, sorted by expert; up to 8 pairs an expert in the mean the sums are of exact products.  Few pairs and many."""
    from llmserve.config.registry import preset

    config = copy.deepcopy(preset(name))
    small, given = runner(config, "float8", use_graphs=False), runner(config, "model", use_graphs=False)
    calls = Calls(monkeypatch)
    vocab = config.get("vocab_size") or config["vocab"]
    logits(small, torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(n)).tolist(), [n])
    plain_of = {id(a): b for (_, a), (_, b) in zip(small.model._parts(), given.model._parts()) if hasattr(a, "w_gate_up")}
    part_of = {id(a.w_gate_up): a for _, a in small.model._parts() if hasattr(a, "w_gate_up")}
    groups = [c for c in calls.seen if c[0] == "grouped_float8"]
    assert part_of and len(groups) >= 2 * len({id(a) for a in part_of.values()})
    for (_, act, (x, w, (seg, tiles)), options, _), (_, out, (x2, w2, *_), _, _) in zip(groups[::2], groups[1::2]):
        part = part_of[id(w)]
        assert w2 is part.w_down and torch.equal(x2.values.view(torch.uint8), act.values.view(torch.uint8)) and options["swiglu"]
        assert options["limit"] == (part.limit if part.unit == "clamped" else None)
        kept, ops = plain_of[id(part)], calls.ops
        pairs, experts = x.shape[0], part.experts
        down = kept.w_down
        for e in range(experts):
            a, b = seg[e].item(), seg[e + 1].item()
            if a == b:
                continue
            gate_up = unpaired(kept.w_gate_up[e], part.intermediate)
            wd, dd = (held(ops.Float8(t.values[e], t.scale[e], t.columns), v) for t, v in ((w, gate_up), (w2, down[e])))
            few = pairs <= 8 * experts
            mine = ops.Float8(act.values[a:b], act.scale[a:b], act.columns)
            check_units(mine, x[a:b], wd, not few, options["limit"])
            check_product(out[a:b], ops.Float8(x2.values[a:b], x2.scale[a:b], x2.columns), dd, sixteens=False)
        assert seg[-1].item() == pairs


def unpaired(w, units):
    """[gate; up] of a stacked matrix whose blocks of 32 gate rows and 32 up rows take turns."""
    blocks = w.view(-1, 2, 32, w.shape[-1])
    return torch.cat([blocks[:, 0].reshape(-1, w.shape[-1])[:units], blocks[:, 1].reshape(-1, w.shape[-1])[:units]])
