"""Weights in 8 bits of nearly 4 GB, the largest that are taken: offsets beyond 2^31 in every kernel that reads or makes them."""

import pytest
import torch

import plain_float8 as plain
from test_float8_gpu import bound_of, segments_of
from test_float8_sums_gpu import check_bfloat16, units_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
GROUPS, ROWS, K = 2, 128 * 1021, 16384  # 4,282,384,384 bytes; two groups of 2,141,192,192
N = GROUPS * ROWS


def ops():
    from llmserve.ops import library

    return library


@pytest.fixture(scope="module")
def weight():
    """(the weight in 8 bits, [2, ROWS, K]; rows of it by number, in 64 bits)"""
    g = torch.Generator(device=DEV).manual_seed(3)
    w = torch.empty(GROUPS, ROWS, K, dtype=torch.bfloat16, device=DEV)
    for piece in w.view(-1, K).split(1 << 14):
        piece.copy_(torch.randn(piece.shape, generator=g, device=DEV) * K ** -0.5)
    w8 = ops().weight_float8(w)
    # the blocks of rows on both sides of 2^31 bytes of the result, of 2^31 numbers, and the last
    for e, block in ((0, 0), (0, 511), (0, 512), (0, 1020), (1, 0), (1, 3), (1, 1020)):
        at = slice(128 * block, 128 * block + 128)
        values, scale = plain.weight(w[e, at].cpu().double())
        assert torch.equal(w8.values[e, at].float().cpu().double(), values) and torch.equal(w8.scale[e, block: block + 1].float().cpu().double(), scale), (e, block)
    del w
    yield w8
    torch.cuda.empty_cache()


def picked(w8, rows):
    """What rows of the weight [N, K] stand for."""
    values = w8.values.view(N, -1).view(torch.uint8)[rows].view(torch.float8_e4m3fn).float().cpu().double()
    scale = w8.scale.view(N // 128, -1).view(torch.uint8)[[r // 128 for r in rows]].view(torch.float8_e8m0fnu).float().cpu().double()
    return values * scale[:, : K // 128].repeat_interleave(128, dim=1)


def whole(w8):
    return ops().Float8(w8.values.view(N, -1), w8.scale.view(N // 128, -1), K)


def rows_of(m):
    x = torch.randn(m, K, generator=torch.Generator().manual_seed(m)).to(torch.bfloat16).to(DEV)
    x8 = ops().rows_float8(ops().empty_float8(m, K, DEV), x)
    return x, plain.numbers(x8.values.float(), x8.scale.float())


EDGES = [0, 1, 65535, 65536, 131071, 131072, 131073, 196608, N - 130, N - 129, N - 17, *range(N - 9, N)]


@pytest.mark.parametrize("m,few_bytes", [(1, None), (16, None), (40, 1e12), (40, None), (130, None)])
def test_product(weight, m, few_bytes, monkeypatch):
    """Few rows (the weight streamed past them, also past 17 to 64), and tiles."""
    if few_bytes is not None:
        monkeypatch.setattr(ops(), "GEMM_FLOAT8_FEW_BYTES", few_bytes)
    x, xd = rows_of(m)
    wd = picked(weight, EDGES)
    y = xd @ wd.t()
    for dtype in (torch.bfloat16, torch.float32):
        out = ops().gemm_float8(torch.full((m, N), float("nan"), dtype=dtype, device=DEV), x, whole(weight))
        assert not torch.isnan(out).any()
        off = bound_of(xd, wd, y, torch.float32, m > 16 and dtype == torch.bfloat16)
        got = out[:, EDGES]
        if dtype == torch.bfloat16:
            check_bfloat16(got, y, off)
        else:
            assert ((got.cpu().double() - y).abs() <= off).all()


@pytest.mark.parametrize("m", [2, 90])
def test_gated(weight, m):
    x, xd = rows_of(m)
    inter = N // 2
    units = [0, 1, 511, 512, 65535, 65536, inter - 129, *range(inter - 9, inter)]
    wd = picked(weight, units + [inter + u for u in units])
    want, off = units_of(xd @ wd.t(), bound_of(xd, wd, xd @ wd.t(), torch.float32, m > 16), len(units))
    out = ops().gemm_float8(torch.full((m, inter), float("nan"), dtype=torch.bfloat16, device=DEV), x, whole(weight), swiglu=True)
    assert not torch.isnan(out).any()
    check_bfloat16(out[:, units], want, off)


@pytest.mark.parametrize("counts", [[3, 5], [70, 60]])
def test_groups(weight, counts):
    x, xd = rows_of(sum(counts))
    out = ops().grouped_float8(torch.full((sum(counts), ROWS), float("nan"), device=DEV), x, weight, segments_of(counts))
    assert not torch.isnan(out).any()
    columns = [0, 1, ROWS - 129, *range(ROWS - 9, ROWS)]
    at = 0
    for e, n in enumerate(counts):
        wd = picked(weight, [e * ROWS + c for c in columns])
        mine = xd[at: at + n]
        assert ((out[at: at + n][:, columns].cpu().double() - mine @ wd.t()).abs() <= bound_of(mine, wd, mine @ wd.t(), torch.float32)).all()
        at += n


def test_short_rows(weight):
    """The same bytes as rows of 2,048: one token whose X becomes 8 bits inside the product."""
    n, k = N * 8, 2048
    w8 = ops().Float8(weight.values.view(n, k), torch.full((n // 128, 16), 120, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu), k)
    x = torch.randn(1, k, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    xd = plain.numbers(*plain.rows(x.double()))
    edges = [0, (1 << 20) - 1, 1 << 20, n - 129, *range(n - 9, n)]
    wd = w8.values.view(torch.uint8)[edges].view(torch.float8_e4m3fn).float().cpu().double() * 2.0 ** -7
    out = ops().gemm_float8(torch.full((1, n), float("nan"), device=DEV), x.to(DEV), w8)
    assert not torch.isnan(out).any()
    y = xd @ wd.t()
    assert ((out[:, edges].cpu().double() - y).abs() <= bound_of(xd, wd, y, torch.float32)).all()
