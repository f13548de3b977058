"""The predictive operators on the GPU against plain 64-bit statements of their definitions (include/mhlik.h).

Quantized bytes and drawn columns are whole numbers and have to be equal.  Products of float C: the values that 8-bit rows
stand for have 4 significant bits, so products are exact and only the cols - 1 additions round, each by at most a step
2^-23 of the sum of magnitudes.  16-bit C: half a step of the type, and what the 8-bit matrix instruction drops: less than
2^-10 of the sum of magnitudes (it keeps about 16 bits below the largest product of a group); where all products have the
same exponent nothing is dropped and the result is the exact one, rounded once."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def P():
    from mcmc_amd import predictive

    return predictive


# ------------------------------------------------------------------ quantize

E4M3 = np.array([m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127])


def plain_quantize(x):
    """(codes without NaN's payload, powers) of a float64 array."""
    rows, cols = x.shape
    blocks = -(-cols // 128)
    codes = np.zeros((rows, blocks * 128), np.int64)
    ks = np.zeros((rows, blocks), np.int64)
    middle = (E4M3[1:] + E4M3[:-1]) / 2
    for i in range(rows):
        for b in range(blocks):
            v = x[i, b * 128 : (b + 1) * 128]
            top = max([abs(t) for t in v if math.isfinite(t)], default=0.0)
            k = -96
            while k < 119 and top > 448.0 * 2.0 ** k:
                k += 1
            if top == 0.0:
                k = 0
            ks[i, b] = k
            y = v * 2.0 ** -k
            with np.errstate(invalid="ignore"):
                c = np.searchsorted(middle, np.abs(y), side="left")
                tie = (c < 126) & (np.abs(y) == middle[np.minimum(c, 125)]) & (c % 2 == 1)
                c = np.where(np.abs(y) <= 448.0, c + tie, 127)
            codes[i, b * 128 : b * 128 + len(v)] = np.where(c == 127, 127, c + 128 * np.signbit(y))
    return codes, ks


def check_quantized(P, x):
    q = P.quantize(x)
    codes, ks = plain_quantize(x.double().cpu().numpy())
    got = q.data.view(torch.uint8).cpu().numpy().astype(np.int64)
    got = np.where(got % 128 == 127, 127, got)
    assert np.array_equal(got, codes)
    scale = q.scale.cpu().numpy().astype(np.int64)
    assert np.array_equal(scale[:, : ks.shape[1]], ks + 127)
    assert np.all(scale[:, ks.shape[1] :] == 127)
    return q


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (17, 640), (5, 513), (257, 3), (70, 200)])
def test_quantize(P, kind, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(rows * 1000 + cols)
    x = torch.randn(rows, cols, generator=g, device="cuda", dtype=torch.float64) * torch.exp(3 * torch.randn(rows, 1, generator=g, device="cuda", dtype=torch.float64))
    x = x.to(TYPES[kind])
    check_quantized(P, x)
    check_quantized(P, x.t().contiguous().t())  # column by column


@pytest.mark.parametrize("kind", list(TYPES))
def test_quantize_strides(P, kind):
    g = torch.Generator(device="cuda").manual_seed(7)
    big = torch.randn(90, 401, generator=g, device="cuda", dtype=torch.float64).to(TYPES[kind])
    for x in (big[:, 3:], big[::2], big[1:, 1:260], big[:40, ::3], big.t()[5:, 2:], big[0:1].expand(33, 401), big[:, 5:6].expand(90, 150), big[:, 7:8], big.t()[::2, ::5]):
        check_quantized(P, x)


@pytest.mark.parametrize("kind", list(TYPES))
def test_quantize_special_values(P, kind):
    dtype = TYPES[kind]
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    rows = [[0.0] * 130, [-0.0] * 130, [math.inf, 1.0, -math.inf, math.nan] + [0.25] * 126, [math.nan] * 130, [big, -big, 1.0] + [0.0] * 127,
            [tiny, -tiny / 2, tiny * 1.5] + [0.0] * 127, [448.0, 449.0, -447.9] + [1.0] * 127, [448.0, 0.001, 2.0 ** -10] + [3.0] * 127,
            [17.0, 19.0, 21.0, 23.0, 25.0, 27.0, 29.0, 31.0, 448.0] + [0.5] * 121]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype).cuda()
    check_quantized(P, x)
    check_quantized(P, x.repeat(8, 1).t().contiguous().t())


def test_quantize_rounds_a_double_once(P):
    """Values that a detour through float would bring onto a tie of e4m3, and doubles beyond float's range."""
    half = 1.0 + 1.0 / 16  # between 1 and 1.125
    x = torch.tensor([[448.0, half, half + 2.0 ** -40, half - 2.0 ** -40, 1e-300, 5e-324, -half - 2.0 ** -45], [1e300, 1.0, 2.0, 1e-300, 0.0, -1e200, 3.0],
                      [448.0 * 2.0 ** 119, 449.0 * 2.0 ** 119, -1e39, 3e38, 1.0, 0.0, 1.7e38], [448.0 + 2.0 ** -40, 1.0, 0, 0, 0, 0, 0]], dtype=torch.float64, device="cuda")
    check_quantized(P, x)
    check_quantized(P, x.repeat(6, 1).t().contiguous().t())


def test_dequantize(P):
    x = torch.randn(9, 300, device="cuda")
    q = P.quantize(x)
    codes, ks = plain_quantize(x.double().cpu().numpy())
    value = np.where(codes >= 128, -1.0, 1.0) * E4M3[codes % 128] * np.repeat(2.0 ** ks, 128, axis=1)
    assert np.array_equal(q.dequantize().double().cpu().numpy(), value[:, :300])


# ------------------------------------------------------------------- product

SIZES = [(1, 1, 1), (1, 17, 129), (2, 3, 64), (1, 5000, 128), (1, 40, 5000), (3, 300, 20000), (15, 16, 127), (16, 33, 257), (17, 130, 700), (33, 64, 300),
         (64, 65, 256), (64, 19, 2000), (65, 1, 100), (65, 70, 128), (100, 300, 256), (1000, 36, 3), (129, 128, 385), (200, 257, 1300), (300, 129, 513),
         (130, 1000, 640), (4100, 3900, 300)]


def values(q):
    return q.dequantize().double()


def check_product(out, x, w, dtype):
    """x, w: the float64 values that the 8-bit rows stand for."""
    exact = torch.mm(x, w.t().contiguous())
    size = torch.mm(x.abs(), w.abs().t().contiguous())
    off = (out.double() - exact).abs()
    if dtype == torch.float32:
        bound = (x.shape[1] + 8) * 2.0 ** -23 * size
    else:
        bound = torch.finfo(dtype).eps / 2 * exact.abs() + 2.0 ** -10 * size + (6e-8 if dtype == torch.float16 else 0.0)
    assert torch.isfinite(out).all()
    assert (off <= bound).all(), (off - bound).max().item()


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,draws,cols", SIZES)
def test_product(P, rows, draws, cols, out):
    g = torch.Generator(device="cuda").manual_seed(rows + 7 * draws + 13 * cols)
    x = torch.randn(rows, cols, generator=g, device="cuda")
    w = P.quantize(torch.randn(draws, cols, generator=g, device="cuda") / math.sqrt(cols))
    xq = P.quantize(x)
    ready = P.product(xq, w, TYPES[out])
    assert ready.shape == (rows, draws) and ready.dtype == TYPES[out]
    check_product(ready, values(xq), values(w), TYPES[out])
    assert torch.equal(P.product(x, w, TYPES[out]), ready)  # quantized on the way: the same bytes, the same sums


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,cols", [(1, 300), (5, 64), (40, 130), (70, 200), (300, 513)])
def test_product_of_values_of_any_type_and_stride(P, kind, rows, cols):
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    w = P.quantize(torch.randn(150, cols, generator=g, device="cuda"))
    big = torch.randn(2 * rows, cols + 5, generator=g, device="cuda", dtype=torch.float64).to(TYPES[kind])
    for x in (big[:rows, 5:], big[::2, 1 : cols + 1], big[:rows, :cols].t().contiguous().t(), big[-1:, :cols].expand(rows, cols)):
        assert torch.equal(P.product(x, w), P.product(P.quantize(x), w))


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,draws,cols", SIZES)
def test_product_of_equal_exponents_is_exact(P, rows, draws, cols, out):
    """Values +-1 .. +-1.875 and scales that are powers of two a block: sums of multiples of 2^-6 below 2^18, which float holds."""
    g = torch.Generator(device="cuda").manual_seed(rows + draws + cols)

    def some(n):
        v = (1 + torch.randint(0, 8, (n, cols), generator=g, device="cuda") / 8) * (torch.randint(0, 2, (n, cols), generator=g, device="cuda") * 2 - 1)
        return v.double()

    x, w = some(rows), some(draws)
    got = P.product(P.quantize(x), P.quantize(w), TYPES[out])
    exact = torch.mm(x, w.t().contiguous())
    if out == "f16":
        exact = exact.clamp(-65504, 65504)
        got = got.clamp(-65504, 65504)
    assert torch.equal(got, exact.to(TYPES[out]))


@pytest.mark.parametrize("rows", [3, 40, 200])
def test_product_scales_of_each_block(P, rows):
    """Blocks that differ by powers of two, on both sides, each with its own."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    cols, draws = 1500, 190
    e = torch.randint(-30, 30, (rows + draws, 12), generator=g, device="cuda").double()
    v = torch.randn(rows + draws, cols, generator=g, device="cuda", dtype=torch.float64) * torch.exp2(e).repeat_interleave(128, dim=1)[:, :cols]
    x, w = P.quantize(v[:rows]), P.quantize(v[rows:])
    for dtype in (torch.float32, torch.bfloat16):
        check_product(P.product(x, w, dtype), values(x), values(w), dtype)


@pytest.mark.parametrize("rows", [2, 50, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product_keeps_a_nan_to_its_row(P, rows, dtype):
    x = torch.randn(rows, 400, device="cuda")
    x[1, 333] = math.inf
    out = P.product(x, P.quantize(torch.randn(140, 400, device="cuda")), dtype)
    assert torch.isnan(out[1]).all()
    assert torch.isfinite(out[[i for i in range(rows) if i != 1]]).all()


@pytest.mark.parametrize("rows", [1, 20, 64, 100, 300])
@pytest.mark.parametrize("cols", [100, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_product_leaves_the_rest_of_out_alone(P, rows, cols, dtype):
    """A C call with a row stride above the draws, and memory behind the last row."""
    from mcmc_amd import _lib

    draws, stride = 133, 150
    x, w = P.quantize(torch.randn(rows, cols, device="cuda")), P.quantize(torch.randn(draws, cols, device="cuda"))
    want = P.product(x, w, dtype)
    out = torch.full((rows + 2, stride), 77.0, dtype=dtype, device="cuda")
    p = _lib.Q8Operands()
    p.x, p.x_scale, p.w_data, p.w_scale = x.data.data_ptr(), x.scale.data_ptr(), w.data.data_ptr(), w.scale.data_ptr()
    p.out, p.out_stride, p.rows, p.draws, p.cols = out.data_ptr(), stride, rows, draws, cols
    p.out_type = {torch.float32: 2, torch.float16: 4}[dtype]
    assert _lib.load_mhlik().mhlik_q8_product(C.byref(p), -1, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(out[:rows, :draws], want)
    assert (out[:rows, draws:] == 77).all() and (out[rows:] == 77).all()


def test_product_refusals(P):
    w = P.quantize(torch.randn(5, 100, device="cuda"))
    with pytest.raises(ValueError, match="x has 99 columns, w has 100"):
        P.product(torch.randn(3, 99, device="cuda"), w)
    with pytest.raises(ValueError, match="dtype is"):
        P.product(torch.randn(3, 100, device="cuda"), w, torch.float64)
    with pytest.raises(ValueError, match="x has type"):
        P.product(torch.zeros(3, 100, device="cuda", dtype=torch.int32), w)
    with pytest.raises(ValueError, match="2 dimension"):
        P.quantize(torch.randn(3, device="cuda"))
    with pytest.raises(ValueError, match="requires a gradient"):
        P.product(torch.randn(3, 100, device="cuda", requires_grad=True), w)
    with pytest.raises(ValueError, match="scale has shape"):
        P.Block8(w.data, w.scale[:, :2], 100)
    with pytest.raises(ValueError, match="data has 128 columns"):
        P.Block8(w.data, w.scale, 129)
    with pytest.raises(ValueError, match="at least one column"):
        P.quantize(torch.randn(3, 0, device="cuda"))
    assert P.product(torch.randn(0, 100, device="cuda"), w).shape == (0, 5)


# ---------------------------------------------------------------------- draw

def plain_draw(z, u, temperature, top_k, top_p, min_p):
    """One row, float64: (column, log probability)."""
    n = len(z)
    if np.isnan(z).any() or np.isneginf(z).all() or not temperature >= 0 or any(math.isnan(t) for t in (u, top_p, min_p)):
        return -1, math.nan
    z = np.minimum(z, np.finfo(np.float32).max)
    order = np.lexsort((np.arange(n), -z))
    if temperature == 0:
        return order[0], 0.0
    w = np.zeros(n)
    some = ~np.isneginf(z)
    w[some] = np.exp((z[some] - z[order[0]]) / temperature)
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        mass = np.cumsum(w[order])
        before = np.concatenate([[0.0], mass[:-1]])
        order = order[: max(1, int(np.sum(before < top_p * mass[-1])))]
    order = order[w[order] >= min(min_p, 1.0)] if min_p > 0 else order
    kept = np.sort(order)
    kept = kept[w[kept] > 0]
    mass = np.cumsum(w[kept])
    at = min(int(np.searchsorted(mass, max(u, 0.0) * mass[-1], side="right")), len(kept) - 1)
    return kept[at], math.log(w[kept[at]] / mass[-1])


def check_draw(P, z, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    column, logp = P.draw(z, u, temperature, top_k, top_p, min_p)
    rows = z.shape[0]
    assert column.shape == (rows,) and column.dtype == torch.int64 and logp.dtype == torch.float32

    def each(v, off):
        return [off] * rows if v is None else [v] * rows if not isinstance(v, torch.Tensor) else v.double().cpu().tolist()

    zs, us = z.double().cpu().numpy(), u.double().cpu().numpy()
    want = [plain_draw(zs[i], us[i], t, int(k), p, m) for i, (t, k, p, m) in enumerate(zip(each(temperature, 1.0), each(top_k, 0), each(top_p, 1.0), each(min_p, 0.0)))]
    assert column.cpu().tolist() == [int(c) for c, _ in want]
    wl = np.array([l for _, l in want])
    got = logp.double().cpu().numpy()
    assert np.array_equal(np.isnan(wl), np.isnan(got))
    ok = ~np.isnan(wl)
    assert np.all(np.abs(got[ok] - wl[ok]) <= 2.0 ** -24 * np.abs(wl[ok]) + 1e-12)  # half a step of float; weights to 1e-13


def random_row(g, rows, n, dtype, spread=2.0):
    return (spread * torch.randn(rows, n, generator=g, device="cuda")).to(dtype)


CHOICES = [dict(), dict(temperature=0.0), dict(temperature=0.6), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(top_p=0.0), dict(top_p=0.9999),
           dict(min_p=0.05), dict(min_p=1.0), dict(temperature=0.8, top_k=40, top_p=0.9), dict(temperature=1.5, top_k=300, top_p=0.5, min_p=0.01)]
LENGTHS = [1, 2, 63, 64, 65, 128, 129, 512, 513, 2048, 2049, 8192, 8193, 20001]


@pytest.mark.parametrize("choice", CHOICES, ids=lambda c: "-".join("%s%s" % kv for kv in c.items()) or "plain")
@pytest.mark.parametrize("n", LENGTHS)
def test_draw_lengths(P, n, choice):
    g = torch.Generator(device="cuda").manual_seed(n)
    for rows, dtype in ((3, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
        check_draw(P, random_row(g, rows, n, dtype), torch.rand(rows, generator=g, device="cuda", dtype=torch.float64), **choice)


@pytest.mark.parametrize("n", [7, 128, 300, 1500, 3000])
def test_draw_many_rows(P, n):
    """From 512 rows on a row has fewer waves."""
    g = torch.Generator(device="cuda").manual_seed(n)
    rows = 600
    z = random_row(g, rows, n, torch.float32)
    z = torch.where(torch.rand(rows, n, generator=g, device="cuda") < 0.3, -math.inf, z)
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    check_draw(P, z, u)
    check_draw(P, z, u, 0.7, 30, 0.9, 0.02)
    check_draw(P, z.half(), u, 1.3, None, 0.6)


@pytest.mark.parametrize("n,rows", [(70001, 40), (131072, 20), (524289, 2), (600000, 1), (2200000, 1)])
@pytest.mark.parametrize("choice", [dict(), dict(temperature=0.0), dict(top_k=50, top_p=0.95), dict(top_k=5000), dict(top_p=0.9), dict(min_p=0.1)],
                         ids=["plain", "greedy", "k-p", "large-k", "p", "m"])
def test_draw_long_rows(P, n, rows, choice):
    g = torch.Generator(device="cuda").manual_seed(n)
    for dtype in (torch.float32, torch.bfloat16):
        check_draw(P, random_row(g, rows, n, dtype), torch.rand(rows, generator=g, device="cuda", dtype=torch.float64), **choice)


@pytest.mark.parametrize("n", [50, 700, 5000, 30000])
def test_draw_ties(P, n):
    """Few distinct values, so that borders fall among equal ones; all equal; one above many equal ones."""
    g = torch.Generator(device="cuda").manual_seed(n)
    rows = 6
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    few = torch.randint(-3, 3, (rows, n), generator=g, device="cuda").float()
    flat = torch.full((rows, n), -1.25, device="cuda")
    spike = torch.where(torch.arange(n, device="cuda")[None] == n // 3, 60.0, flat)
    for z in (few, flat, spike, few.bfloat16(), torch.sort(few, -1, descending=True)[0], torch.sort(random_row(g, rows, n, torch.float32), -1, descending=True)[0]):
        for choice in (dict(), dict(temperature=0.0), dict(top_k=1), dict(top_k=n // 3), dict(top_k=n - 1), dict(top_p=0.5), dict(top_p=0.97), dict(top_k=n // 2, top_p=0.3), dict(min_p=1.0),
                       dict(min_p=0.4)):
            check_draw(P, z, u, **choice)


@pytest.mark.parametrize("n", [100, 400, 1500, 3000])
def test_draw_many_rows_of_ties(P, n):
    """Fewer waves take a row when there are many; the border falls among hundreds of equal weights."""
    g = torch.Generator(device="cuda").manual_seed(17 * n)
    rows = 515
    z = torch.randint(-2, 2, (rows, n), generator=g, device="cuda").float()
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    check_draw(P, z, u, top_k=n // 3)
    check_draw(P, z.bfloat16(), u, top_p=0.7)
    check_draw(P, z, u, temperature=2.0, top_k=2 * n // 3, top_p=0.5, min_p=0.1)


@pytest.mark.parametrize("rows,n", [(3, 100), (3, 3000), (3, 20000), (515, 100), (515, 400), (515, 1500), (515, 3000)])
def test_draw_border_among_crowded_weights(P, rows, n):
    """One weight far above the rest, which lie so close together that no histogram tells them apart."""
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    z = -30.0 + 1e-3 * torch.rand(rows, n, generator=g, device="cuda")
    z[torch.arange(rows, device="cuda"), torch.randint(0, n, (rows,), generator=g, device="cuda")] = 0.0
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    check_draw(P, z, u, temperature=40.0, top_k=n // 2)
    check_draw(P, z, u, temperature=40.0, top_p=0.6)
    check_draw(P, z, u, temperature=40.0, top_k=n - 5, top_p=0.3, min_p=0.2)


@pytest.mark.parametrize("n", [3, 300, 3000, 20000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_draw_masks(P, n, dtype):
    """-inf and the type's lowest value as masks, rows with one column left or none, +inf, NaN."""
    g = torch.Generator(device="cuda").manual_seed(n)
    low = torch.finfo(dtype).min
    z = random_row(g, 10, n, dtype)
    z[0] = -math.inf
    z[1] = -math.inf
    z[1, n // 2] = -5.0
    z[2, ::2] = -math.inf
    z[3, 1:] = low
    z[4] = low
    z[5, n - 1] = math.nan
    z[6, [0, n - 1]] = math.inf
    z[7] = torch.where(torch.rand(n, generator=g, device="cuda") < 0.99, -math.inf, z[7])
    z[7, 0] = 0.0
    z[8] = -z[8].abs() - torch.finfo(dtype).max / 2
    u = torch.rand(10, generator=g, device="cuda", dtype=torch.float64)
    for choice in (dict(), dict(temperature=0.0), dict(top_k=5), dict(top_p=0.8), dict(min_p=0.01), dict(temperature=0.5, top_k=50, top_p=0.9, min_p=0.001)):
        check_draw(P, z, u, **choice)


@pytest.mark.parametrize("n", [9, 1000, 9000])
def test_draw_ends_of_u(P, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -53, 1.0, 2.0, -1.0, 0.5, math.nan, 2.0 ** -60], dtype=torch.float64, device="cuda")
    z = random_row(g, 8, n, torch.float32)
    z[:, -2:] = -math.inf
    for choice in (dict(), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.2)):
        check_draw(P, z, u, **choice)
        check_draw(P, z, u.float(), **choice)


@pytest.mark.parametrize("n", [20, 1800, 12000])
def test_draw_each_row_its_own(P, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    rows = 12
    z = random_row(g, rows, n, torch.float32)
    u = torch.rand(rows, generator=g, device="cuda")
    t = torch.tensor([1.0, 0.0, 0.5, 2.0, 1e-30, 1e30, math.inf, -1.0, math.nan, 1.0, 0.1, 1.0], device="cuda")
    k = torch.tensor([0, 5, 3, -2, 7, n + 9, 4, 4, 4, n, 1, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    p = torch.tensor([0.5, 1.0, 2.0, -1.0, 0.9, 0.9, 0.3, 0.5, 0.5, math.nan, 0.0, 0.99], device="cuda")
    m = torch.tensor([0.0, 0.1, -3.0, 0.5, 7.0, 0.01, 0.0, 0.0, 0.0, 0.0, math.nan, 0.3], device="cuda")
    check_draw(P, z, u, t, k, p, m)
    check_draw(P, z, u, t)
    check_draw(P, z, u, 1.0, k)
    check_draw(P, z, u, 1.0, 50, p)
    check_draw(P, z, u, 0.5, None, None, m)


@pytest.mark.parametrize("n", [100, 1001, 10001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_draw_strides(P, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(n)
    big = random_row(g, 9, n + 13, dtype)
    u = torch.rand(18, generator=g, device="cuda", dtype=torch.float64)
    for z in (big[:, 1 : n + 1], big[::2, 7 : n + 7], big[:, :n].t().contiguous().t(), big[2:3, :n].expand(9, n), big[:, : 2 * (n // 2) : 2]):
        check_draw(P, z, u[::2][: z.shape[0]], 0.9, 30, 0.9)
        check_draw(P, z, u[: z.shape[0]])


def test_draw_is_the_distribution(P):
    """Equally spaced random numbers give each column its share of the draws, to one draw."""
    n, rows = 50, 4096
    z = torch.randn(n, device="cuda")
    u = (torch.arange(rows, device="cuda", dtype=torch.float64) + 0.5) / rows
    column, _ = P.draw(z.expand(rows, n), u, 0.7)
    share = torch.softmax(z.double() / 0.7, 0) * rows
    assert (torch.bincount(column, minlength=n).double() - share).abs().max() <= 1.0


def test_draw_refusals(P):
    z, u = torch.randn(3, 40, device="cuda"), torch.rand(3, device="cuda")
    for call, text in ((lambda: P.draw(z.double(), u), "z has type"), (lambda: P.draw(z, u[:2]), "2 values for 3 rows"), (lambda: P.draw(z[0], u), "2 dimension"),
                       (lambda: P.draw(z, u.half()), "u has type"), (lambda: P.draw(z[:, :0], u), "at least one column"),
                       (lambda: P.draw(z, u, torch.ones(2, device="cuda")), "temperature has 2 values"), (lambda: P.draw(z, u, 1.0, torch.ones(3, device="cuda")), "top_k has type"),
                       (lambda: P.draw(z.requires_grad_(), u), "requires a gradient")):
        with pytest.raises(ValueError, match=text):
            call()
    z = z.detach()
    from mcmc_amd import MhlikError

    with pytest.raises(MhlikError, match="temperature"):
        P.draw(z, u, -1.0)
    with pytest.raises(MhlikError, match="top_p"):
        P.draw(z, u, top_p=math.nan)
    column, logp = P.draw(z[:0], u[:0])
    assert column.shape == (0,) and logp.shape == (0,)


# ------------------------------------------------------------ streams, graphs

def test_on_another_stream(P):
    """The work goes to the current stream, behind what that stream has to do."""
    x, th = torch.randn(500, 300, device="cuda"), torch.randn(400, 300, device="cuda")
    z, u = torch.randn(30, 20000, device="cuda"), torch.rand(30, device="cuda")
    want = P.product(x, P.quantize(th)), P.draw(z, u, 0.8, 50, 0.9)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(10):
            big = big @ big * 1e-3  # keeps the stream busy
        x2, th2, z2, u2 = x * 1.0, th * 1.0, z * 1.0, u * 1.0  # behind it
        got = P.product(x2, P.quantize(th2)), P.draw(z2, u2, 0.8, 50, 0.9)
    s.synchronize()
    assert torch.equal(got[0], want[0])
    assert all(torch.equal(a, b) for a, b in zip(got[1], want[1]))


def test_two_graphs_replayed(P):
    """Captured calls keep their workspaces to themselves: two graphs, replayed in turn with new inputs and eager work between."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w = P.quantize(torch.randn(9000, 300, generator=g, device="cuda"))
    graphs = []
    for rows, choice in ((70, dict(temperature=0.9, top_k=40, top_p=0.9)), (90, dict(top_p=0.8, min_p=0.001))):
        x = torch.randn(rows, 300, generator=g, device="cuda")
        u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            P.draw(P.product(x, w), u, **choice)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            z = P.product(x, w)
            out = P.draw(z, u, **choice)
        graphs.append((graph, x, u, choice, z, out))
    for _ in range(4):
        for graph, x, u, choice, z, out in graphs:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            u.copy_(torch.rand(u.shape, generator=g, device="cuda", dtype=torch.float64))
            graph.replay()
        for graph, x, u, choice, z, out in graphs:
            want = P.product(x, w)
            assert torch.equal(z, want)
            assert all(torch.equal(a, b) for a, b in zip(out, P.draw(want, u, **choice)))


def test_results_do_not_change_from_call_to_call(P):
    g = torch.Generator(device="cuda").manual_seed(5)
    x, w = torch.randn(300, 900, generator=g, device="cuda"), P.quantize(torch.randn(700, 900, generator=g, device="cuda"))
    z, u = torch.randn(50, 60001, generator=g, device="cuda"), torch.rand(50, generator=g, device="cuda", dtype=torch.float64)
    first = P.product(x, w), *P.draw(z, u, 1.0, None, 0.9)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip((P.product(x, w), *P.draw(z, u, 1.0, None, 0.9)), first))


# -------------------------------------------------------------- all together

def test_posterior_predictive_of_a_chain(P):
    """The kept draws of a sampler's run, new rows, predictions, and draws without a case."""
    from mcmc_amd import samplers
    from mcmc_amd.likelihood import synthetic_host

    N, d = 3000, 5
    X = synthetic_host(11, N, d)
    run = samplers.gpu_sampler(X, 1, 400, 200, 0.05)
    theta = np.asarray(run["samples"])[-300:]
    pp = P.PosteriorPredictive(theta)
    assert pp.theta.rows == 300 and pp.theta.cols == d
    x = torch.from_numpy(np.ascontiguousarray(X[:200])).cuda()
    q = P.quantize(x)
    exact = values(q) @ values(pp.theta).t()
    check_product(pp.predictor(x), values(q), values(pp.theta), torch.float32)
    pp.CHUNK = 300 * 64  # several chunks
    got = pp.probability(x)
    assert (got.double() - torch.sigmoid(exact).mean(1)).abs().max() <= 1e-5  # float sums of 300 values below 1
    # what 8 bits cost: each product within 2 * 2^-4 + 2^-8 relative, a sigmoid a quarter of that
    full = torch.sigmoid(x.double() @ torch.from_numpy(theta).cuda().t()).mean(1)
    size = (x.double().abs() @ torch.from_numpy(np.abs(theta)).cuda().t()).mean(1)
    assert ((got.double() - full).abs() <= 0.25 * (2 * 2.0 ** -4 + 2.0 ** -8) * size + 1e-5).all()
    u = torch.rand(200, device="cuda", dtype=torch.float64)
    index, logp = pp.case_deletion(x, u, 0.9, 100, 0.95)
    z = torch.logaddexp(pp.predictor(x), torch.zeros((), device="cuda"))
    check = P.draw(z, u, 0.9, 100, 0.95)
    assert torch.equal(index, check[0]) and torch.equal(logp, check[1])
    check_draw(P, z, u, 0.9, 100, 0.95)
    each = torch.linspace(0.5, 1.5, 200, device="cuda")
    index, logp = pp.case_deletion(x, u, each)
    check = P.draw(z, u, each)
    assert torch.equal(index, check[0]) and torch.equal(logp, check[1])
    for rows in (199, 201):  # one choice a row, neither fewer nor more
        with pytest.raises(ValueError, match="temperature has %d values for 200 rows" % rows):
            pp.case_deletion(x, u, torch.ones(rows, device="cuda"))
    with pytest.raises(ValueError, match="u has 201 values for 200 rows"):
        pp.case_deletion(x, torch.rand(201, device="cuda"))


def test_no_rows(P):
    x = torch.zeros(0, 300, device="cuda")
    q = P.quantize(x)
    assert q.dequantize().shape == (0, 300)
    w = P.quantize(torch.ones(4, 300, device="cuda"))
    assert P.product(q, w).shape == (0, 4) and P.product(w, q).shape == (4, 0)
    index, logp = P.draw(torch.zeros(0, 9000, device="cuda"), torch.zeros(0, device="cuda"))
    assert index.shape == (0,) and logp.shape == (0,)
    pp = P.PosteriorPredictive(torch.ones(4, 300, device="cuda"))
    assert pp.probability(x).shape == (0,) and pp.case_deletion(x, torch.zeros(0, device="cuda"))[0].shape == (0,)


def test_product_in_parts(P):
    """More rows than a launch has threads for: the last part, and both sides of the borders."""
    rows = (1 << 28) + 70
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.rand(rows, 1, generator=g, device="cuda", dtype=torch.bfloat16)
    w = P.quantize(torch.randn(2, 1, generator=g, device="cuda"))
    out = P.product(x, w, torch.bfloat16)
    for i in (0, 1 << 27, 1 << 28, rows):
        part = slice(max(0, i - 100), min(rows, i + 100))
        want = values(P.quantize(x[part])) @ values(w).T
        assert torch.equal(out[part].double(), want.to(torch.bfloat16).double())  # one product a value, rounded once
    last = x.t()[:, -300:].t()
    assert torch.equal(P.product(last, w, torch.bfloat16), out[-300:])


@pytest.mark.parametrize("rows,n", [((1 << 20) + 70, 3), (16500, 8200)])
def test_draw_in_parts(P, rows, n):
    g = torch.Generator(device="cuda").manual_seed(n)
    z = torch.randn(rows, n, generator=g, device="cuda", dtype=torch.bfloat16)
    u = torch.rand(rows, generator=g, device="cuda")
    each = dict(temperature=0.5 + torch.rand(rows, generator=g, device="cuda"), top_k=torch.randint(1, n, (rows,), generator=g, device="cuda", dtype=torch.int32),
                top_p=torch.rand(rows, generator=g, device="cuda"), min_p=0.01 * torch.rand(rows, generator=g, device="cuda"))
    column, logp = P.draw(z, u, **each)
    border = (1 << 20) if n == 3 else (1 << 27) // n
    for part in (slice(0, 40), slice(border - 40, border + 40), slice(rows - 40, rows)):
        few = {k: v[part] for k, v in each.items()}
        check_draw(P, z[part], u[part], **few)
        want = P.draw(z[part], u[part], **few)
        assert torch.equal(column[part], want[0]) and torch.allclose(logp[part], want[1], rtol=2.0 ** -22, atol=1e-12)  # sums of another shape


def test_threads_at_once(P):
    """Four threads, each on a stream of its own."""
    import threading

    g = torch.Generator(device="cuda").manual_seed(8)
    sets = []
    for i in range(4):
        x = torch.randn(90 + 200 * i, 300, generator=g, device="cuda")
        w = P.quantize(torch.randn(700 + i, 300, generator=g, device="cuda"))
        z = torch.randn(5, 9000 + i, generator=g, device="cuda")
        u = torch.rand(5, generator=g, device="cuda")
        sets.append((x, w, z, u, P.product(x, w), P.draw(z, u, top_p=0.8)))
    torch.cuda.synchronize()
    wrong = []

    def work(x, w, z, u, product, drawn):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                a, b = P.product(x, w), P.draw(z, u, top_p=0.8)
                stream.synchronize()
                if not (torch.equal(a, product) and torch.equal(b[0], drawn[0]) and torch.equal(b[1], drawn[1])):
                    wrong.append(x.shape)

    threads = [threading.Thread(target=work, args=s) for s in sets]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("rows,n", [(515, 100), (515, 400), (3, 400), (515, 1500), (515, 3000), (3, 5000), (3, 30000), (1, (1 << 21) + 5)])
def test_draw_both_borders_among_the_same_ties(P, rows, n):
    """top-k cuts a run of equal weights, and top-p needs all of what is left of it: the run's other columns stay out."""
    g = torch.Generator(device="cuda").manual_seed(rows + n)
    u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
    flat = torch.full((rows, n), -1.25, device="cuda")
    two = torch.where(torch.rand(rows, n, generator=g, device="cuda") < 0.2, 0.0, flat)  # the border lies in the lower, larger run
    for z in (flat, two, two.bfloat16()):
        for choice in (dict(top_k=10, top_p=0.95), dict(top_k=n // 2, top_p=0.99999), dict(top_k=n - 1, top_p=0.9999, min_p=0.1)):
            check_draw(P, z, u, **choice)
    k = torch.randint(1, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
    p = 1.0 - 1e-5 * torch.rand(rows, generator=g, device="cuda")
    check_draw(P, two, u, 0.7, k, p)


@pytest.mark.parametrize("n,spread", [(150_000, 3.9), (1 << 21, 0.0), (1 << 24, 0.0)], ids=["listed", "long", "huge"])
def test_draw_nucleus_of_faint_weights(P, n, spread):
    """One weight of 1, and behind it so many faint ones that they have a mass, of which top-p keeps half.  The border is
    found with weights to 2^-51, 2^-52 off each at most, and sums in double: a draw is off by n 2^-51 of the mass at most."""
    g = torch.Generator(device="cuda").manual_seed(n)
    z = -36.0 + spread * (2 * torch.rand(1, n, generator=g, device="cuda") - 1)
    z[0, n - 1] = 0.0
    w = np.exp(z[0].double().cpu().numpy()).astype(np.longdouble)
    tail = w[:-1].sum()
    top_p = float(1 - tail / 2 / (1 + tail))
    order = np.lexsort((np.arange(n), -w))
    mass = np.cumsum(w[order])
    kept = order[: int(np.searchsorted(mass, top_p * mass[-1])) + 1]
    weight = np.zeros(n, np.longdouble)
    weight[kept] = w[kept]
    upto = np.cumsum(weight)
    for share in (0.1, 0.25, 0.4):
        u = float(share * tail)
        column, logp = P.draw(z, torch.tensor([u], dtype=torch.float64, device="cuda"), top_p=top_p)
        column = int(column)
        assert column < n - 1 and weight[column] > 0
        aim, off = u * upto[-1], n * 2.0 ** -51
        assert upto[column] - weight[column] - off <= aim <= upto[column] + off
        assert abs(float(logp) - math.log(weight[column])) <= 2.0 ** -24 * 40 + n * 2.0 ** -51


def test_draw_masks_in_rows_too_long_for_units(P):
    """A NaN, nothing but -inf, +inf, the type's lowest value: the way of one workgroup a row."""
    n = (1 << 21) + 7
    g = torch.Generator(device="cuda").manual_seed(n)
    z = random_row(g, 5, n, torch.bfloat16)
    z[0, n - 2] = math.nan
    z[1] = -math.inf
    z[2, n // 3] = math.inf
    z[3] = torch.where(torch.rand(n, generator=g, device="cuda") < 0.999, torch.finfo(torch.bfloat16).min, z[3])
    u = torch.rand(5, generator=g, device="cuda", dtype=torch.float64)
    for choice in (dict(), dict(temperature=0.0), dict(top_p=0.8), dict(temperature=0.5, top_k=50, top_p=0.9, min_p=0.001)):
        check_draw(P, z, u, **choice)


def test_tensors_with_the_negative_bit(P):
    """torch keeps the sign of c.conj().imag as a mark on the tensor; the memory holds the other sign."""
    g = torch.Generator(device="cuda").manual_seed(4)

    def negative(v):
        t = torch.complex(torch.zeros_like(v), -v).conj().imag
        assert t.is_neg() and torch.equal(t, v)
        return t

    x, z = torch.randn(3, 200, generator=g, device="cuda"), torch.randn(3, 70, generator=g, device="cuda")
    w = P.quantize(torch.randn(40, 200, generator=g, device="cuda"))
    check_quantized(P, negative(x))
    check_quantized(P, negative(x.double()))
    assert torch.equal(P.product(negative(x), w), P.product(x, w))
    many = torch.randn(100, 200, generator=g, device="cuda")
    assert torch.equal(P.product(negative(many), w), P.product(many, w))
    u = torch.rand(3, generator=g, device="cuda")
    each = [torch.tensor(v, device="cuda") for v in ([0.5, 1.0, 2.0], [0.9, 0.8, 0.5], [0.01, 0.1, 0.2])]
    for rows in (3, 1):  # one value a row: contiguous at any stride
        t, p, m = (negative(v[:rows]) for v in each)
        want = P.draw(z[:rows], u[:rows], each[0][:rows], 30, each[1][:rows], each[2][:rows])
        got = P.draw(negative(z[:rows]), negative(u[:rows]), t, 30, p, m)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    empty = negative(torch.full((2, 1), -math.inf, device="cuda"))
    assert P.draw(empty, u[:2])[0].tolist() == [-1, -1]
    pp = P.PosteriorPredictive(negative(x))
    assert torch.equal(pp.probability(negative(many)), P.PosteriorPredictive(x).probability(many))


def test_forward_mode_is_refused(P):
    """A dual tensor's tangent would be lost."""
    import torch.autograd.forward_ad as forward

    x, w = torch.randn(3, 200, device="cuda"), P.quantize(torch.randn(5, 200, device="cuda"))
    z, u = torch.randn(3, 70, device="cuda"), torch.rand(3, device="cuda")
    pp = P.PosteriorPredictive(torch.randn(6, 200, device="cuda"))
    with forward.dual_level():
        def dual(t):
            return forward.make_dual(t, torch.ones_like(t))

        for call in (lambda: P.quantize(dual(x)), lambda: P.product(dual(x), w), lambda: P.draw(dual(z), u), lambda: P.draw(z, dual(u)), lambda: P.draw(z, u, dual(u)),
                     lambda: pp.probability(dual(x)), lambda: pp.case_deletion(dual(x), u)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        plain = P.product(x, w), P.draw(z, u)  # tensors without a tangent
        assert torch.equal(P.product(dual(x).detach(), w), plain[0])
        assert torch.equal(P.PosteriorPredictive(dual(x)).theta.scale, P.quantize(x).scale)  # keeps its draws detached
    assert torch.equal(P.product(x, w), plain[0]) and torch.equal(P.draw(z, u)[0], plain[1][0])


def test_errors_of_other_calls_are_not_reported_again(P):
    """A call on a device that is not there is refused, and the calls after it know nothing of it; nor of an error that
    other code has left behind, which stays there for it."""
    from mcmc_amd import Likelihood, _lib
    from mcmc_amd.likelihood import synthetic_host

    lib = _lib.load_mhlik()
    x = torch.randn(100, 200, device="cuda")
    z, u = torch.randn(3, 9000, device="cuda"), torch.rand(3, device="cuda")

    def calls():
        q = P.quantize(x)
        return q.data.view(torch.uint8), P.product(x, q), P.product(q, q, torch.bfloat16), *P.draw(z, u, top_p=0.9), *P.draw(z[:, :50], u)

    want = calls()
    q = P.quantize(x)
    nowhere = torch.cuda.device_count()
    assert lib.mhlik_q8_quantize(x.data_ptr(), 2, 100, 200, 200, 1, q.data.data_ptr(), q.scale.data_ptr(), nowhere, None) == 3  # MHLIK_EHIP
    assert "invalid device" in lib.mhlik_last_error(None).decode()
    assert all(torch.equal(a, b) for a, b in zip(calls(), want))
    assert lib.mhlik_q8_quantize(x.data_ptr(), 2, 100, 200, 200, 1, q.data.data_ptr(), q.scale.data_ptr(), nowhere, None) == 3
    with Likelihood(3000, 5, device=0) as lk:  # the samplers' calls ask for the last error too
        lk.upload(synthetic_host(3, 3000, 5))
        assert math.isfinite(lk.loglik(np.zeros(5)))
    assert lib.hipSetDevice(nowhere) != 0  # the runtime's own call
    got = calls()
    assert lib.hipGetLastError() != 0 and lib.hipGetLastError() == 0  # taken back before torch's kernels look for it
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("out", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols", [64, 200])
@pytest.mark.parametrize("draws,stride", [(1000, 1000), (1001, 1001), (1024, 1024), (1024, 1031), (1023, 1040)])
def test_product_narrow_with_several_chunks_a_workgroup(P, draws, stride, cols, out):
    """Rows enough that a workgroup goes along four and more times 128 draws: two buffers in turn, lines carried from one
    chunk to the next, rows of C that do and do not begin at 16 bytes.  Values as in the exact test, so that a stale one shows."""
    from mcmc_amd import _lib

    rows, dtype = 77_003, TYPES[out]
    g = torch.Generator(device="cuda").manual_seed(draws + stride + cols)

    def some(n):
        v = (1 + torch.randint(0, 8, (n, cols), generator=g, device="cuda") / 8) * (torch.randint(0, 2, (n, cols), generator=g, device="cuda") * 2 - 1)
        return v.double()

    x, w = some(rows), some(draws)
    xq, wq = P.quantize(x), P.quantize(w)
    got = torch.full((rows + 1, stride), 77.0, dtype=dtype, device="cuda")
    p = _lib.Q8Operands()
    p.x, p.x_scale, p.w_data, p.w_scale = xq.data.data_ptr(), xq.scale.data_ptr(), wq.data.data_ptr(), wq.scale.data_ptr()
    p.out, p.out_stride, p.rows, p.draws, p.cols = got.data_ptr(), stride, rows, draws, cols
    p.out_type = {"f32": 2, "bf16": 3, "f16": 4}[out]
    assert _lib.load_mhlik().mhlik_q8_product(C.byref(p), -1, torch.cuda.current_stream().cuda_stream) == 0
    exact = torch.mm(x, w.t().contiguous()).to(dtype)  # at most 200 * 3.6: no infinities
    assert torch.equal(got[:rows, :draws], exact)
    assert (got[:rows, draws:] == 77).all() and (got[rows:] == 77).all()


@pytest.mark.parametrize("out", ["bf16", "f16"])
@pytest.mark.parametrize("rows,draws,cols", [(2000, 1000, 64), (2000, 1000, 128), (2000, 1000, 256), (1000, 1000, 400), (1000, 1000, 4096), (4096, 4096, 1000)])
def test_product_accuracy_of_16_bit_results(P, rows, draws, cols, out):
    """What the 8-bit matrix instruction drops is 1.6e-5 of the result's norm, beside the rounding to 16 bits.  The two
    errors are independent, so squares add up; twice the stated 1.6e-5, and 1 % of the rounding's share, which the same
    values rounded after another error have within 1 / sqrt(2 rows draws) (1e-3 here)."""
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = P.quantize(torch.randn(rows, cols, generator=g, device="cuda"))
    w = P.quantize(torch.randn(draws, cols, generator=g, device="cuda") / math.sqrt(cols))
    exact = torch.mm(values(x), values(w).t().contiguous())
    got = P.product(x, w, TYPES[out])
    size = exact.norm()
    off, rounding = ((got.double() - exact).norm() / size).item(), ((exact.to(TYPES[out]).double() - exact).norm() / size).item()
    assert off ** 2 <= (1.01 * rounding) ** 2 + (2 * 1.6e-5) ** 2, (off, rounding)


def test_posterior_predictive_in_a_graph(P):
    """Captured as one, replayed with new rows, eager work between: one mean over a million draws, draws without a case."""
    g = torch.Generator(device="cuda").manual_seed(12)
    pp = P.PosteriorPredictive(torch.randn(1 << 20, 4, generator=g, device="cuda"))
    x, u = torch.randn(2, 4, generator=g, device="cuda"), torch.rand(2, generator=g, device="cuda")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        pp.probability(x), pp.case_deletion(x, u)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pp.probability(x), *pp.case_deletion(x, u, 0.9, top_p=0.95)
    for _ in range(4):
        x.copy_(torch.randn(2, 4, generator=g, device="cuda"))
        u.copy_(torch.rand(2, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = pp.probability(x), *pp.case_deletion(x, u, 0.9, top_p=0.95)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
