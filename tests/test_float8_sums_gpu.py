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


def check_bfloat16(out, want, off):
    """Results between the roundings of want - off and want + off."""
    low, high = ((want + d).to(torch.bfloat16).double() for d in (-off, off))  # (rounding keeps the order)
    got = out.cpu().double()
    wrong = ((got < low) | (got > high)).sum().item()
    assert wrong == 0, f"{wrong} of {got.numel()} values are not the rounding of any number that 32-bit sums allow"


@pytest.mark.parametrize("m,inter,k", [(1, 64, 300), (20, 130, 85), (64, 70, 600), (65, 129, 512), (130, 200, 96), (300, 257, 700), (200, 90, 4500)])
def test_exact_sums(m, inter, k):
    """Asked for, at any number of rows: plain with a bias, gated, gated to 8 bits."""
    n = 2 * inter
    x8, w8, xd, (wd,) = operands(m, n, k, m + inter + k)
    y, off = sums_of(xd, wd)
    want, carried = units_of(y, off, inter)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    yb = y + bias.double()
    out = torch.full((m + 1, n + 3), float("nan"), dtype=torch.bfloat16, device=DEV)
    ops().gemm_float8(out[:m, :n], x8, w8, bias.to(DEV), exact=True)
    check_bfloat16(out[:m, :n], yb, off + (yb.abs() + off) * 2.0 ** -23)
    assert torch.isnan(out[m:]).all() and torch.isnan(out[:, n:]).all()
    out = torch.full((m + 1, inter + 3), float("nan"), dtype=torch.bfloat16, device=DEV)
    ops().gemm_float8(out[:m, :inter], x8, w8, swiglu=True, exact=True)
    check_bfloat16(out[:m, :inter], want, carried)
    assert torch.isnan(out[m:]).all() and torch.isnan(out[:, inter:]).all()
    check_steps(ops().gemm_float8(ops().empty_float8(m, inter, DEV), x8, w8, swiglu=True, exact=True), want, carried)
    # a float32 result is exact anyhow
    a, b = (ops().gemm_float8(torch.empty(m, n, device=DEV), x8, w8, exact=e) for e in (False, True))
    assert torch.equal(a, b)


@pytest.mark.parametrize("tile,each", [(0, None), (0, 4), (1, None), (1, 4)])
@pytest.mark.parametrize("m,inter,k", [(70, 45, 1300), (129, 258, 1030)])
def test_exact_sums_of_every_tile_and_part(tile, each, m, inter, k, monkeypatch):
    from llmserve.ops import library

    monkeypatch.setattr(library, "gemm_float8_tiles", lambda *a: (tile, each or -(-k // 128)))
    x8, w8, xd, (wd,) = operands(m, 2 * inter, k, m + inter + k)
    y, off = sums_of(xd, wd)
    want, carried = units_of(y, off, inter)
    room = lambda cols: torch.empty(m, cols, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    check_bfloat16(ops().gemm_float8(room(2 * inter), x8, w8, exact=True), y, off)
    check_bfloat16(ops().gemm_float8(room(inter), x8, w8, swiglu=True, exact=True), want, carried)
    check_steps(ops().gemm_float8(ops().empty_float8(m, inter, DEV), x8, w8, swiglu=True, exact=True), want, carried)


@pytest.mark.parametrize("counts", [[3, 0, 9], [40, 0, 129, 300, 1], [0, 0, 128, 0, 256]])
@pytest.mark.parametrize("inter,k", [(65, 200), (136, 640)])
def test_exact_sums_of_groups(counts, inter, k):
    """Rows behind the last segment are left as they are."""
    pairs, groups, n = sum(counts), len(counts), 2 * inter
    x8, w8, xd, wd = operands(pairs + 2, n, k, pairs + k, groups)
    group = torch.repeat_interleave(torch.arange(groups), torch.tensor(counts))
    segments = segments_of(counts)
    y, off = torch.zeros(pairs, n, dtype=torch.float64), torch.zeros(pairs, n, dtype=torch.float64)
    for g in set(group.tolist()):
        y[group == g], off[group == g] = sums_of(xd[:pairs][group == g], wd[g])
    want, carried = units_of(y, off, inter)
    for cols, swiglu, expected, slack in ((n, False, y, off), (inter, True, want, carried)):
        out = torch.full((pairs + 2, cols + 1), float("nan"), dtype=torch.bfloat16, device=DEV)
        ops().grouped_float8(out[:, :cols], x8, w8, segments, swiglu=swiglu, exact=True)
        check_bfloat16(out[:pairs, :cols], expected, slack)
        assert torch.isnan(out[pairs:]).all() and torch.isnan(out[:, cols:]).all()
    out8 = ops().empty_float8(pairs + 2, inter, DEV)
    out8.values.view(torch.uint8).fill_(7)
    out8.scale.view(torch.uint8).fill_(9)
    ops().grouped_float8(out8, x8, w8, segments, swiglu=True, exact=True)
    check_steps(ops().Float8(out8.values[:pairs], out8.scale[:pairs], inter), want, carried)
    assert (out8.values.view(torch.uint8)[pairs:] == 7).all() and (out8.scale.view(torch.uint8)[pairs:] == 9).all()
    a, b = (ops().grouped_float8(torch.zeros(pairs + 2, n, device=DEV), x8, w8, segments, exact=e) for e in (False, True))
    assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["plain", "gated", "rows"])
def test_exact_sums_in_two_graphs(kind):
    """Two graphs of one call in turn, with other rows each time: the sums' place is a call's own."""
    m, n, k = 90, 406, 700
    w8 = ops().weight_float8((torch.randn(n, k, generator=torch.Generator().manual_seed(n)) * k ** -0.5).to(torch.bfloat16).to(DEV))

    def room():
        return ops().empty_float8(m, n // 2, DEV) if kind == "rows" else torch.empty(m, n if kind == "plain" else n // 2, dtype=torch.bfloat16, device=DEV)

    def call(out, x):
        return ops().gemm_float8(out, x, w8, swiglu=kind != "plain", exact=True)

    def bytes_of(out):
        return [t.clone().view(torch.uint8) for t in (out[:2] if kind == "rows" else (out,))]

    xs, outs, graphs = [torch.empty(m, k, dtype=torch.bfloat16, device=DEV) for _ in range(2)], [room(), room()], []
    for x, out in zip(xs, outs):
        x.normal_()
        call(out, x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(out, x)
        graphs.append(graph)
    for turn in range(4):
        for x in xs:
            x.normal_()
        wanted = [bytes_of(call(room(), x)) for x in xs]
        for graph in graphs if turn % 2 else graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for out, want in zip(outs, wanted):
            assert all(torch.equal(a, b) for a, b in zip(bytes_of(out), want))


@pytest.mark.parametrize("inter,k", [(176, 640), (129, 3000)])
def test_units_in_8_bits_of_a_row_are_the_same_beside_any_others(inter, k):
    """Of up to 64 rows (K in one part, up to 4,096 columns): the same sums in the same order, whichever rows come with it, so a step may be filled up."""
    x8, w8, _, _ = operands(64, 2 * inter, k, inter)
    outs = {}
    for m in (1, 2, 15, 16, 17, 31, 32, 33, 63, 64):
        rows = ops().Float8(x8.values[:m], x8.scale[:m], k)
        outs[m] = ops().gemm_float8(ops().empty_float8(m, inter, DEV), rows, w8, swiglu=True)
    for m, out in outs.items():
        assert torch.equal(out.values.view(torch.uint8), outs[64].values[:m].view(torch.uint8)), m
        assert torch.equal(out.scale.view(torch.uint8), outs[64].scale[:m].view(torch.uint8)), m


@pytest.mark.parametrize("pairs,k,given,kernels", [
    (16, 640, "bfloat16", ["few"]), (17, 640, "bfloat16", ["rows", "few"]), (16, 4104, "bfloat16", ["rows", "few"]), (16, 640, "float8", ["few"]),
    (64, 640, "float8", ["few"]), (65, 640, "float8", ["tiles"]), (65, 640, "bfloat16", ["rows", "tiles"])])
def test_which_kernels_groups_take(pairs, k, given, kernels, monkeypatch):
    """Eight groups: rows become 8 bits inside the product up to 16 of up to 4,096 columns, as one weight's do; tiles beyond eight rows a group in the mean."""
    names = {"llms_rows_float8": "rows", "llms_gemm_float8_few": "few", "llms_gemm_float8": "tiles"}
    taken, real = [], ops()._entry
    w8 = ops().weight_float8(torch.randn(8, 64, k, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV))
    x = torch.randn(pairs, k, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(DEV)
    x8 = ops().rows_float8(ops().empty_float8(pairs, k, DEV), x)
    counts = [pairs - 3, 0, 1, 0, 0, 2, 0, 0]
    monkeypatch.setattr(ops(), "_entry", lambda library, name, arguments: taken.append(names[name]) or real(library, name, arguments))
    out = ops().grouped_float8(torch.empty(pairs, 64, device=DEV), x if given == "bfloat16" else x8, w8, segments_of(counts))
    assert taken == kernels
    assert torch.equal(out, ops().grouped_float8(torch.empty(pairs, 64, device=DEV), x8, w8, segments_of(counts)))


@pytest.mark.parametrize("counts", [[0] * 20 + [400] + [0] * 40 + [3, 90, 7], [1] * 30 + [130] + [1] * 33, [0, 0, 511, 1] + [0] * 60])
@pytest.mark.parametrize("kind", ["rows", "float32"])
def test_uneven_groups_of_few_rows_in_the_mean(counts, kind):
    """One group far above the mean beside empty ones and ones of a row: as many sixteens as it has, one behind another."""
    groups, inter, k = len(counts), 40, 300
    pairs = sum(counts)
    assert pairs <= 8 * groups
    x8, w8, xd, wd = operands(pairs, 2 * inter, k, pairs, groups)
    group = torch.repeat_interleave(torch.arange(groups), torch.tensor(counts))
    y, off = torch.zeros(pairs, 2 * inter, dtype=torch.float64), torch.zeros(pairs, 2 * inter, dtype=torch.float64)
    for g in set(group.tolist()):
        y[group == g], off[group == g] = sums_of(xd[group == g], wd[g])
    if kind == "float32":
        out = ops().grouped_float8(torch.full((pairs, 2 * inter), float("nan"), device=DEV), x8, w8, segments_of(counts))
        assert ((out.cpu().double() - y).abs() <= off).all()
    else:
        check_steps(ops().grouped_float8(ops().empty_float8(pairs, inter, DEV), x8, w8, segments_of(counts), swiglu=True), *units_of(y, off, inter))
