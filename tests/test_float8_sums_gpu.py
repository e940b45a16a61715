"""Sums of 8-bit products: where nothing of them is dropped, against their definition in 64 bits."""

import pytest
import torch

import plain_float8 as plain
from test_float8_gpu import segments_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ops():
    from llmserve.ops import library

    return library


def operands(m, n, k, seed, groups=0):
    """Rows and weights in 8 bits, and the numbers that they stand for; a column in 16 far above the others, so that what is dropped below it shows."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    x[:, ::16] *= 64
    w = torch.randn(max(groups, 1), n, k, generator=g) * k ** -0.5 / 8
    w8 = ops().weight_float8((w if groups else w[0]).to(torch.bfloat16).to(DEV))
    x8 = ops().rows_float8(ops().empty_float8(m, k, DEV), x.to(torch.bfloat16).to(DEV))
    xd = plain.numbers(x8.values.float(), x8.scale.float())
    wd = [plain.numbers(v.float(), s.float(), 128) for v, s in zip(*((w8.values, w8.scale) if groups else (w8.values[None], w8.scale[None])))]
    return x8, w8, xd, wd


def sums_of(xd, wd):
    """The sums, and how far 32-bit ones of exact products may be off: each of K additions by at most a unit of 2^-23 of the sum of the sizes."""
    return xd @ wd.t(), (xd.abs() @ wd.abs().t()) * xd.shape[1] * 2.0 ** -23


def units_of(y, off, inter):
    """Units and how far off they are: a slope of at most 1.2 |up| in the gate and |gate| in up, and 256 units of 2^-24 for the unit itself (the exponent
    of a gate of up to 88 is rounded at its size)."""
    gate, up = y.split(inter, dim=1)
    dg, du = off.split(inter, dim=1)
    want = plain.unit(gate, up)
    return want, 1.2 * (up.abs() + du) * dg + (gate.abs() + dg) * du + want.abs() * 256 * 2.0 ** -24


def check_steps(out, want, off):
    """Rows in 8 bits of numbers that are `off` from `want` at most: their block's scale is that of a largest number so far off, and each value the rounding of
    a number so far off (rounding does not turn an order, so it lies between the roundings of both ends)."""
    m, k = want.shape
    kp = out.values.shape[1]
    blocks = kp // 128
    want, off = (torch.nn.functional.pad(t, (0, kp - k)).view(m, blocks, 128) for t in (want, off))
    s = out.scale.float().cpu().double()
    assert (s[:, blocks:] == 1).all()
    s = s[:, :blocks]
    least, most = ((want.abs() - off).clamp(min=0).amax(dim=2), (want.abs() + off).amax(dim=2))
    assert (torch.exp2(plain.scale_exponent(least)) <= s).all() and (s <= torch.exp2(plain.scale_exponent(most))).all()
    got, s = out.values.float().cpu().double().view(m, blocks, 128), s.unsqueeze(2)
    low, high = (plain.to_e4m3(((want + d) / s).clamp(-448, 448)) for d in (-off, off))
    wrong = ((got < low) | (got > high)).sum().item()
    assert wrong == 0, f"{wrong} of {m * k} values are not the rounding of any number that 32-bit sums allow"


@pytest.mark.parametrize("m", [1, 9, 16, 17, 40, 64])
@pytest.mark.parametrize("inter,k", [(130, 85), (200, 640), (70, 1023), (129, 1300)])
def test_units_of_few_rows_in_8_bits_are_of_exact_sums(m, inter, k):
    """Whatever K: a unit is one rounding of the unit of exact products' sums."""
    x8, w8, xd, (wd,) = operands(m, 2 * inter, k, m + inter + k)
    want, off = units_of(*sums_of(xd, wd), inter)
    check_steps(ops().gemm_float8(ops().empty_float8(m, inter, DEV), x8, w8, swiglu=True), want, off)


@pytest.mark.parametrize("counts", [[1], [0, 16, 3], [2] * 9])
@pytest.mark.parametrize("inter,k", [(130, 85), (72, 700)])
def test_units_of_few_rows_per_group_in_8_bits_are_of_exact_sums(counts, inter, k):
    pairs, groups = sum(counts), len(counts)
    x8, w8, xd, wd = operands(pairs, 2 * inter, k, pairs + k, groups)
    out = ops().grouped_float8(ops().empty_float8(pairs, inter, DEV), x8, w8, segments_of(counts), swiglu=True)
    group = torch.repeat_interleave(torch.arange(groups), torch.tensor(counts))
    pairs_of = [sums_of(xd[i: i + 1], wd[g]) for i, g in enumerate(group.tolist())]
    want, off = units_of(*(torch.cat(t) for t in zip(*pairs_of)), inter)
    check_steps(out, want, off)
