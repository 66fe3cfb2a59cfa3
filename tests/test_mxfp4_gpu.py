"""Microscaled 4-bit matrices: quantisation against its definition in 64 bits, and the products with them.

Where a product's terms are small whole numbers every order of sums gives the same bits, so that the results are compared
exactly; others with a bound on the sums: a sum of n terms in 32 bits, each addition cut or rounded, is off by at most
(n + 8) 2^-23 of the terms' magnitudes (the 8 for the join of the waves' sums), the bias and the stream included among the terms."""
import math

import pytest
import torch

import qwen_engine_amd  # noqa: F401

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


@pytest.fixture(scope="module")
def ops():
    from qwen_engine_amd.kernels import ops
    ops.load_library()
    return ops


def gen(seed):
    return torch.Generator().manual_seed(seed)


def codes_of(x):
    """Codes [T, blocks, 32] and scale bytes [T, blocks] of x by the definition: the nearest of the eight magnitudes, the even code
    where two are as near."""
    T, K = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -K % 32)).view(T, -1, 32)
    top = b.abs().amax(-1)
    # a float64's own exponent: exact, also next to powers of two
    e = torch.frexp(top)[1] - 1 - 2
    e = torch.where(top > 0, e.clamp(min=-127), torch.full_like(e, -127))
    bad = ~torch.isfinite(top)
    e = torch.where(bad, torch.zeros_like(e), e)
    a = torch.where(bad.unsqueeze(-1), torch.zeros_like(b), b).abs() / torch.exp2(e.double()).unsqueeze(-1)
    far = (a.clamp(max=6.0).unsqueeze(-1) - GRID).abs()
    best = far.amin(-1, keepdim=True)
    near = far == best
    even = near & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1), even.int().argmax(-1), near.int().argmax(-1))
    code = code + 8 * torch.signbit(b)
    return torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code), torch.where(bad, torch.full_like(e, 255), e + 127)


def values_of(code, scale, K):
    v = torch.cat([GRID, -GRID])[code.long()] * torch.exp2(scale.double() - 127).unsqueeze(-1)
    v = torch.where((scale == 255).unsqueeze(-1), torch.full_like(v, math.nan), v)
    return v.reshape(code.shape[0], -1)[:, :K]


def unpack(codes):
    return torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1, 32)


def packed(code):
    p = code.reshape(code.shape[0], -1, 2)
    return (p[..., 0] + 16 * p[..., 1]).to(torch.uint8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 32), (3, 31), (5, 33), (7, 64), (2, 100), (65, 96), (1, 4096), (130, 257), (1031, 1000)])
def test_quantize(ops, dtype, T, K):
    x = (torch.randn(T, K, generator=gen(1)) * torch.exp2(torch.randint(-20, 20, (T, 1), generator=gen(2)).float())).to(dtype)
    m = ops.mxfp4_quantize(x.to(DEV))
    code, scale = codes_of(x)
    assert m.columns == K and m.codes.shape == (T, (K + 31) // 32 * 16) and m.scales.shape == (T, (K + 31) // 32)
    assert torch.equal(m.scales.cpu().int(), scale.int())
    assert torch.equal(unpack(m.codes.cpu()).int(), code.int())
    for out in (torch.float32, torch.bfloat16):
        assert torch.equal(ops.mxfp4_values(m, out).double().cpu(), values_of(code, scale, K))


def test_quantize_borders(ops):
    """Ties, the largest code's border, signs of zero, the smallest and largest numbers there are, blocks of zeros, NaN, infinities."""
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.999, 0.2500001, 0.7499999, 4.9999995, 5.0000005, 0.0, -0.0])
    rows = []
    for e in (-126, -100, -3, 0, 1, 90, 124):
        for top in (4.0, 6.0, 7.999):
            r = torch.cat([ties, -ties]).double() * 2.0 ** e
            r[0] = top * 2.0 ** e
            rows.append(r.float())
    tiny = torch.zeros(32)
    tiny[:6] = torch.tensor([2.0 ** -149, 2.0 ** -148, -(2.0 ** -128), 2.0 ** -129, 2.0 ** -127, 1.5 * 2.0 ** -127])
    rows.append(tiny)
    for top in (2.0 ** -125, 2.0 ** -126, 2.0 ** -127, 1.99 * 2.0 ** -126, 3.4e38):
        r = torch.linspace(-1, 1, 32) * top
        rows.append(r)
    rows.append(torch.zeros(32))
    rows.append(-torch.zeros(32))
    for bad in (math.nan, math.inf, -math.inf):
        r = torch.ones(32)
        r[17] = bad
        rows.append(r)
    x = torch.stack(rows)
    m = ops.mxfp4_quantize(x.to(DEV))
    code, scale = codes_of(x)
    assert torch.equal(m.scales.cpu().int(), scale.int())
    assert torch.equal(unpack(m.codes.cpu()).int(), code.int())
    for dtype in (torch.float32, torch.bfloat16):
        got, want = ops.mxfp4_values(m, dtype).double().cpu(), values_of(code, scale, 32)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_every_code_and_scale(ops):
    """All 16 codes under all 256 scales stand for what they should, in both types."""
    code = torch.arange(32).repeat(256, 1, 1) % 16
    scale = torch.arange(256).view(256, 1)
    m = ops.MxFp4(packed(code).to(DEV), scale.to(torch.uint8).to(DEV), 32)
    want = values_of(code, scale, 32)
    for dtype in (torch.float32, torch.bfloat16):
        got = ops.mxfp4_values(m, dtype).double().cpu()
        w = torch.where(want.abs() > torch.finfo(dtype).max, want.sign() * math.inf, want)     # (6 * 2^127 and 4 * 2^127: beyond both types)
        assert torch.equal(got.isnan(), w.isnan()) and torch.equal(got.nan_to_num(), w.nan_to_num())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_at_odd_elements(ops, dtype):
    """x and the values' place at no whole 16-byte piece; nothing beside the result is written."""
    buf = torch.randn(1 + 6 * 64, generator=gen(5)).to(dtype).to(DEV)
    x = buf[1:].view(6, 64)
    m = ops.mxfp4_quantize(x)
    code, scale = codes_of(x.cpu())
    assert torch.equal(unpack(m.codes.cpu()).int(), code.int()) and torch.equal(m.scales.cpu().int(), scale.int())


def whole_matrix(N, K, seed):
    """A 4-bit matrix of whole numbers and halves, junk behind its columns."""
    blocks = (K + 31) // 32
    code = torch.randint(0, 16, (N, blocks, 32), generator=gen(seed))
    scale = torch.randint(127, 129, (N, blocks), generator=gen(seed + 1))
    return packed(code), scale.to(torch.uint8), values_of(code, scale, K)


ROWS = [1, 2, 16, 17, 33, 64, 65, 130, 300]
SHAPES = [(16, 32), (48, 128), (77, 100), (1, 1), (30, 257), (512, 1024), (300, 992), (20, 4160)]


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("M", ROWS)
def test_product_of_whole_numbers(ops, kind, M):
    """Every order of sums is exact: the results are equal, whatever the split; in bfloat16 rounded once."""
    for N, K in SHAPES:
        codes, scales, v = whole_matrix(N, K, N + K)
        w = ops.MxFp4(codes.to(DEV), scales.to(DEV), K)
        if kind == "fp4":
            xc, xs, xv = whole_matrix(M, K, 7)
            x = ops.MxFp4(xc.to(DEV), xs.to(DEV), K)
        else:
            xv = torch.randint(-4, 5, (M, K), generator=gen(9)).double()
            x = xv.to(torch.float32 if kind == "float32" else torch.bfloat16).to(DEV)
        want = xv @ v.T                                        # halves (fp4: quarters) below 2^22: exact in 32 bits
        got = ops.gemm_mxfp4(x, w, out_dtype=torch.float32).cpu()
        assert torch.equal(got.double(), want), (N, K)
        got = ops.gemm_mxfp4(x, w, out_dtype=torch.bfloat16).cpu()
        assert torch.equal(got, want.float().to(torch.bfloat16)), (N, K)
        bias = torch.randint(-50, 50, (N,), generator=gen(3)).float()
        stream = torch.randint(-50, 50, (M, N), generator=gen(4)).float()
        out = stream.to(DEV)
        assert ops.gemm_mxfp4(x, w, bias.to(DEV), out=out, epilogue=ops.EPI_RESIDUAL) is out
        assert torch.equal(out.cpu().double(), want + bias + stream), (N, K)


def sums_bound(n, magnitudes):
    return (n + 8) * 2.0 ** -23 * magnitudes


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("M,N,K", [(1, 96, 512), (5, 64, 330), (33, 100, 256), (130, 160, 320), (257, 384, 96)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_silu_and_bias(ops, kind, M, N, K, out_dtype):
    w_raw = torch.randn(N, K, generator=gen(11)) * 0.2
    x_raw = torch.randn(M, K, generator=gen(12))
    w = ops.mxfp4_quantize(w_raw.to(DEV))
    v = values_of(*codes_of(w_raw), K)
    if kind == "fp4":
        x, xv = ops.mxfp4_quantize(x_raw.to(DEV)), values_of(*codes_of(x_raw), K)
    else:
        x = x_raw.to(torch.float32 if kind == "float32" else torch.bfloat16)
        x, xv = x.to(DEV), x.double()
    bias = torch.randn(N, generator=gen(13))
    y = xv @ v.T + bias.double()
    off = sums_bound(3 * K + 1, xv.abs() @ v.abs().T + bias.double().abs())    # (32-bit x: three terms a number)
    got = ops.gemm_mxfp4(x, w, bias.to(DEV), out_dtype=out_dtype).cpu()
    half = torch.finfo(out_dtype).eps / 2
    assert got.dtype == out_dtype
    assert ((got.double() - y).abs() <= off + half * (y.abs() + off)).all()
    got = ops.gemm_mxfp4(x, w, bias.to(DEV), out_dtype=out_dtype, epilogue=ops.EPI_SILU_MUL).cpu().double()
    g, u, og, ou = y[:, :N // 2], y[:, N // 2:], off[:, :N // 2], off[:, N // 2:]
    want = g * torch.sigmoid(g) * u
    # silu's slope is at most 1.1; its own arithmetic (an exponential good to 2 units in the last place of its argument's
    # rounding, a sum, a quotient, a product): at most (4 + |g|) units
    off = 1.1 * og * (u.abs() + ou) + (g * torch.sigmoid(g)).abs() * ou + (4 + g.abs()) * 2.0 ** -23 * want.abs()
    assert ((got - want).abs() <= off + half * (want.abs() + off)).all()


@pytest.mark.parametrize("M", [1, 16, 70, 300])
def test_gate_and_up_rows_in_turn(ops, M):
    """A matrix whose gate and up rows alternate in blocks of 32, as a loaded model's: the plain store and silu_mul over such columns give what
    the epilogue gives of gate rows followed by up rows.  (Both are within the sums' and the activation's arithmetic, as in test_silu_and_bias.)"""
    I, K = 352, 512
    gate, up = (torch.randn(I, K, generator=gen(i)) * 0.2 for i in (61, 62))
    x = torch.randn(M, K, generator=gen(63)).to(DEV)
    w, turn = (ops.mxfp4_quantize(t.to(DEV)) for t in (torch.cat([gate, up]), ops.interleave_gate_up(gate, up)))
    v = ops.mxfp4_values(w, torch.float32).double()
    y, off = x.double() @ v.T, sums_bound(3 * K, x.double().abs() @ v.abs().T)
    g, u, og, ou = y[:, :I], y[:, I:], off[:, :I], off[:, I:]
    want = g * torch.sigmoid(g) * u
    off = 1.1 * og * (u.abs() + ou) + (g * torch.sigmoid(g)).abs() * ou + (5 + g.abs()) * 2.0 ** -23 * want.abs()
    for got in (ops.silu_mul(ops.gemm_mxfp4(x, turn), interleaved=True), ops.gemm_mxfp4(x, w, epilogue=ops.EPI_SILU_MUL)):
        assert ((got.double() - want).abs() <= off).all()


def test_float32_rows_lose_nothing(ops):
    """Three numbers a row, of all magnitudes: a product that leaves out any of the 24 bits is off by more than the bound."""
    M, N, K = 20, 48, 640
    x = torch.zeros(M, K)
    for m in range(M):
        at = torch.randperm(K, generator=gen(m))[:3]
        x[m, at] = torch.randn(3, generator=gen(100 + m)) * 2.0 ** (m * 6 - 60)
    w_raw = torch.randn(N, K, generator=gen(21))
    w = ops.mxfp4_quantize(w_raw.to(DEV))
    v = values_of(*codes_of(w_raw), K)
    got = ops.gemm_mxfp4(x.to(DEV), w).cpu().double()
    assert ((got - x.double() @ v.T).abs() <= sums_bound(9, x.double().abs() @ v.abs().T)).all()


@pytest.mark.parametrize("M,N,K", [(17, 130, 2600), (20, 302, 4160), (40, 20100, 200), (90, 302, 6000), (70, 20100, 200), (200, 8230, 712),
                                   (330, 1000, 12000), (500, 4200, 1312), (300, 8230, 712), (512, 8192, 4096), (3100, 302, 1312), (470, 8230, 712),
                                   (600, 1000, 12000), (1000, 4200, 330), (3100, 302, 12000), (3100, 4200, 768), (600, 1000, 4160)])
def test_float32_rows_lose_nothing_in_tiles(ops, M, N, K):
    """The same where the planes are walked one after the other by tiles of 64, 96, 128, 160 and 256 rows, in one piece and in cuts that begin and end
    inside a plane (and by the tiles of 32 rows of all three): three numbers a row, all over K, the last ones of K among them.  (Nine terms that are
    not zero; the others are added without a rounding.)"""
    m = torch.arange(M)
    x = torch.zeros(M, K)
    for i, at in enumerate((m * 131 % K, K - 1 - m % 40, torch.randint(0, K, (M,), generator=gen(6)))):
        x[m, at] = torch.randn(M, generator=gen(100 + i)) * torch.exp2((m % 20 * 6 - 60).float())
    w_raw = torch.randn(N, K, generator=gen(21))
    w = ops.mxfp4_quantize(w_raw.to(DEV))
    x, v = x.to(DEV), ops.mxfp4_values(w, torch.float32).double()
    off = sums_bound(9, x.double().abs() @ v.abs().T)
    assert ((ops.gemm_mxfp4(x, w).double() - x.double() @ v.T).abs() <= off).all()
    # (the test would see it: without the last eight bits, and without the eight before, many sums are off by more)
    for bits in (0xff, 0xff00):
        less = (x.view(torch.int32) & ~bits).view(torch.float32)
        assert (((less.double() - x.double()) @ v.T).abs() > off).any()


@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("N,K", [(130, 1), (130, 3), (130, 255), (130, 257), (16390, 257), (130, 1023), (16390, 2570), (130, 4096)])
def test_few_float32_rows(ops, M, N, K):
    """Rows of any length from any number of an allocation on, NaN on both sides of them and infinities inside: nothing of a neighbour's joins,
    the lowest bits count, and a row's infinity stays its own."""
    w_raw = torch.randn(N, K, generator=gen(K)).abs() + 0.5                # (no zeros: infinity stays infinity)
    w = ops.mxfp4_quantize(w_raw.to(DEV))
    v = values_of(*codes_of(w_raw), K)
    x = torch.randn(M, K, generator=gen(M)) * torch.exp2(torch.randint(-30, 31, (M, K), generator=gen(M + 1)).float())
    for before in (0, 1, 2, 3):
        room = torch.full((M * K + 16,), math.nan, device=DEV)
        room[before:before + M * K] = x.to(DEV).view(-1)
        got = ops.gemm_mxfp4(room[before:before + M * K].view(M, K), w).cpu().double()
        assert ((got - x.double() @ v.T).abs() <= sums_bound(3 * K, x.double().abs() @ v.abs().T)).all()
    x[M // 2, K // 2] = math.inf
    got = ops.gemm_mxfp4(x.to(DEV), w).cpu()
    assert (got[M // 2] == math.inf).all()
    others = [m for m in range(M) if m != M // 2]
    want = x[others].double() @ v.T
    assert ((got[others].double() - want).abs() <= sums_bound(3 * K, x[others].double().abs() @ v.abs().T)).all()


@pytest.mark.parametrize("M", [1, 2, 7, 16, 17, 32])
@pytest.mark.parametrize("N,K", [(130, 2), (130, 6), (130, 31), (130, 254), (130, 258), (16390, 260), (130, 1022), (16390, 2566), (130, 4100)])
def test_few_bfloat16_rows(ops, M, N, K):
    """Rows whose last 16 bytes go on in the next row, from any number of an allocation on, NaN on both sides of them; a row of NaN stays alone."""
    w_raw = torch.randn(N, K, generator=gen(K))
    w = ops.mxfp4_quantize(w_raw.to(DEV))
    w.codes[:, (K + 1) // 2:] = 0x77                               # (behind the columns: sixes)
    v = values_of(*codes_of(w_raw), K).to(DEV)
    x = torch.randn(M, K, generator=gen(M)).to(torch.bfloat16)
    if M > 2:
        x[1::3] = math.nan
    want = x.to(DEV).double() @ v.T
    bound = sums_bound(K, x.to(DEV).double().abs() @ v.abs().T)
    for before in (0, 1, 2, 4, 7):
        room = torch.full((M * K + 16,), math.nan, dtype=torch.bfloat16, device=DEV)
        room[before:before + M * K] = x.to(DEV).view(-1)
        got = ops.gemm_mxfp4(room[before:before + M * K].view(M, K), w, out_dtype=torch.float32).double()
        assert torch.equal(got.isnan(), want.isnan())
        assert ((got - want).nan_to_num().abs() <= bound.nan_to_num()).all()


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
def test_nan_and_infinities(ops, kind):
    """A NaN block of the matrix spoils its own output column and no other; a row with a NaN or an infinity its own row."""
    M, N, K = 70, 80, 160
    w_raw = torch.randn(N, K, generator=gen(31)).abs() + 1.0             # (no zeros: infinity stays infinity)
    w_raw[33, 100] = math.nan
    x_raw = torch.randn(M, K, generator=gen(32)).abs() + 1.0
    x_raw[3, 64] = math.nan
    x_raw[66, 5] = math.inf
    w = ops.mxfp4_quantize(w_raw.to(DEV))
    x = ops.mxfp4_quantize(x_raw.to(DEV)) if kind == "fp4" else x_raw.to(getattr(torch, kind)).to(DEV)
    got = ops.gemm_mxfp4(x, w, out_dtype=torch.float32).cpu()
    assert got[3].isnan().all() and got[:, 33].isnan().all()
    if kind == "fp4":
        assert got[66].isnan().all()
    else:
        assert (got[66, torch.arange(N) != 33] == math.inf).all()
    keep_m, keep_n = [m for m in range(M) if m not in (3, 66)], [n for n in range(N) if n != 33]
    assert got[keep_m][:, keep_n].isfinite().all()


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("M,N,K", [(1, 130, 256), (7, 130, 250), (16, 16390, 330), (20, 48, 640), (40, 300, 256), (200, 8230, 712), (300, 8230, 712),
                                   (470, 8230, 712), (130, 302, 4160), (3100, 4200, 256), (3, 20, 400001)])
def test_scales_at_the_ends(ops, kind, M, N, K):
    """The smallest scales (also where sums lie below the least normal number: there a sum of n terms is off by at most n + 8 times 2^-149 more),
    the largest that quantisation gives, 252, and the two beyond it, under which the larger codes are beyond float32: beside rows in 16 or 32
    bits a column that has such a one is infinite or NaN and no other is touched, beside rows in 4 bits every sum is right."""
    blocks = (K + 31) // 32

    def matrix(rows, scales, seed, some=None):
        code = torch.randint(0, 16, (rows, blocks, 32), generator=gen(seed))
        if some is not None:                                   # (every other row has no code of 2 or more)
            code = torch.where((torch.arange(rows) % 2 == some).view(-1, 1, 1), code & 11, code)
        scale = torch.tensor(scales)[torch.arange(rows) // 2 % len(scales)].view(-1, 1).expand(rows, blocks).contiguous()
        v = values_of(code, scale, K).to(DEV)
        return ops.MxFp4(packed(code).to(DEV), scale.to(torch.uint8).to(DEV), K), v

    def rows(power):
        x = (torch.randn(M, K, generator=gen(8)) * 2.0 ** power).to(torch.float32 if kind == "float32" else torch.bfloat16).to(DEV)
        return x, x.double()

    def check(x, xv, w, v, infinite=None):
        want, off = xv @ v.T, sums_bound(3 * K, xv.abs() @ v.abs().T) + (3 * K + 8) * 2.0 ** -149
        assert float((want.abs() + off).max()) < torch.finfo(torch.float32).max or infinite is not None
        got = ops.gemm_mxfp4(x, w, out_dtype=torch.float32).double()
        if infinite is not None:
            assert not got[:, infinite].isfinite().any()
            got, want, off = got[:, ~infinite], want[:, ~infinite], off[:, ~infinite]
        assert ((got - want).abs() <= off).all()

    if kind == "fp4":
        for x_scales, w_scales in (([252, 253, 254], [100, 101]), ([0, 1], [252, 253, 254]), ([0, 1, 2], [127]), ([0, 1], [0, 1]), ([127], [0, 1, 2])):
            check(*matrix(M, x_scales, 7), *matrix(N, w_scales, 5))
        return
    for power, scales in ((20, [0, 1]), (0, [0, 1]), (-10, [0, 1]), (-30, [251, 252])):
        check(*rows(power), *matrix(N, scales, 5))
    w, v = matrix(N, [127, 253, 252, 254], 5, some=0)
    beyond = (v.abs() > torch.finfo(torch.float32).max).any(1)
    assert beyond.any() and not beyond.all()
    check(*rows(-30), w, v, beyond)


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("K", [40, 64, 96, 160, 200, 700, 1312])
def test_large_tiles_and_what_lies_behind_a_row(ops, kind, K):
    """Enough rows and columns for the largest tiles; K ends inside a stage, and the row behind is NaN: every other column is exact."""
    M, N = 3100, 4200
    codes, scales, v = whole_matrix(N, K, K)
    scales[1::7] = 255
    v = torch.where((scales == 255).any(1, keepdim=True), torch.full_like(v, math.nan), v).to(DEV)
    w = ops.MxFp4(codes.to(DEV), scales.to(DEV), K)
    if kind == "fp4":
        xc, xs, xv = whole_matrix(M, K, 7)
        xs[1::5] = 255
        xv = torch.where((xs == 255).any(1, keepdim=True), torch.full_like(xv, math.nan), xv)
        x = ops.MxFp4(xc.to(DEV), xs.to(DEV), K)
    else:
        xv = torch.randint(-4, 5, (M, K), generator=gen(9)).double()
        xv[1::5] = math.nan
        x = xv.to(torch.float32 if kind == "float32" else torch.bfloat16).to(DEV)
    want = xv.to(DEV) @ v.T
    for m in (M, 200):
        part = ops.MxFp4(x.codes[:m], x.scales[:m], K) if kind == "fp4" else x[:m]
        got = ops.gemm_mxfp4(part, w, out_dtype=torch.float32).double()
        assert torch.equal(got.isnan(), want[:m].isnan()) and torch.equal(got.nan_to_num(), want[:m].nan_to_num())
        # (gates and ups that are 0 or NaN: the places of the activation's operands)
        up = want[:m, N // 2:]
        gate = want[:m, :N // 2]
        got = ops.gemm_mxfp4(part, w, out_dtype=torch.float32, epilogue=ops.EPI_SILU_MUL).double()
        act = gate * torch.sigmoid(gate) * up
        assert torch.equal(got.isnan(), act.isnan())
        # (below a gate of -88.73 the exponential, beyond 2^128, is infinite in 32 bits and silu 0 instead of 88.73 * 2^-128 < 2^-121 at the most)
        bound = (8 + gate.abs()).nan_to_num() * 2.0 ** -23 * act.nan_to_num().abs() + 2.0 ** -121 * up.nan_to_num().abs()
        assert ((got - act).nan_to_num().abs() <= bound).all()


@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
@pytest.mark.parametrize("M,N,K", [(200, 8230, 712), (300, 8230, 712), (470, 8230, 712), (500, 4200, 1312), (1000, 4200, 330), (70, 20100, 200),
                                   (330, 1000, 12000), (600, 1000, 12000), (600, 1000, 4160), (3100, 302, 12000), (270, 1002, 4168),
                                   (20, 302, 4160), (40, 20100, 200), (3100, 302, 1312), (20, 4200, 4160)])
def test_tiles_of_every_height(ops, kind, M, N, K):
    """Rows and columns that tiles of 32, 64, 96, 128, 160 and 256 rows are taken for, with K in one piece and in cuts; every seventh column
    and every fifth row is NaN, every other sum exact (halves of at most 48 K < 2^21), the activation within its own arithmetic."""
    codes, scales, v = whole_matrix(N, K, K)
    scales[1::7] = 255
    v = torch.where((scales == 255).any(1, keepdim=True), torch.full_like(v, math.nan), v).to(DEV)
    w = ops.MxFp4(codes.to(DEV), scales.to(DEV), K)
    xv = torch.randint(-4, 5, (M, K), generator=gen(9)).double()
    xv[1::5] = math.nan
    x = xv.to(getattr(torch, kind)).to(DEV)
    want = xv.to(DEV) @ v.T
    same = lambda got, to: torch.equal(got.isnan(), to.isnan()) and torch.equal(got.nan_to_num(), to.nan_to_num())
    assert same(ops.gemm_mxfp4(x, w, out_dtype=torch.float32).double(), want)
    bias = torch.randint(-50, 50, (N,), generator=gen(3)).float().to(DEV)
    stream = torch.randint(-50, 50, (M, N), generator=gen(4)).float().to(DEV)
    to = want + bias + stream
    assert same(ops.gemm_mxfp4(x, w, bias, out=stream, epilogue=ops.EPI_RESIDUAL).double(), to)
    up, gate = want[:, N // 2:], want[:, :N // 2]
    got = ops.gemm_mxfp4(x, w, out_dtype=torch.float32, epilogue=ops.EPI_SILU_MUL).double()
    act = gate * torch.sigmoid(gate) * up
    assert torch.equal(got.isnan(), act.isnan())
    # (the bound of the large tiles' test)
    bound = (8 + gate.abs()).nan_to_num() * 2.0 ** -23 * act.nan_to_num().abs() + 2.0 ** -121 * up.nan_to_num().abs()
    assert ((got - act).nan_to_num().abs() <= bound).all()


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("M,N,K", [(70, 301, 128), (70, 301, 640), (300, 517, 384), (300, 1030, 1152), (3100, 4200, 768), (3100, 4200, 128)])
@pytest.mark.parametrize("at", [0, 1, 4])
def test_scales_of_rows_that_end_inside_a_span(ops, kind, M, N, K, at):
    """Scales travel 16 at a time, from any whole word on: rows of 4, 12, 20 or more scales, from the given byte of an allocation on, between
    others that are NaN; every sum exact (halves of at most 48 K)."""
    codes, scales, v = whole_matrix(N, K, K)
    scales[1::7] = 255
    v = torch.where((scales == 255).any(1, keepdim=True), torch.full_like(v, math.nan), v).to(DEV)

    def placed(s):
        room = torch.full((s.numel() + 64,), 255, dtype=torch.uint8, device=DEV)
        room[at:at + s.numel()] = s.to(DEV).view(-1)
        return room[at:at + s.numel()].view(s.shape)
    w = ops.MxFp4(codes.to(DEV), placed(scales), K)
    if kind == "fp4":
        xc, xs, xv = whole_matrix(M, K, 7)
        x = ops.MxFp4(xc.to(DEV), placed(xs), K)
    else:
        xv = torch.randint(-4, 5, (M, K), generator=gen(9)).double()
        x = xv.to(getattr(torch, kind)).to(DEV)
    want = xv.to(DEV) @ v.T
    got = ops.gemm_mxfp4(x, w, out_dtype=torch.float32).double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_rows_at_odd_elements(ops):
    """x, bias and out at no whole 16-byte piece; the numbers before and behind out stay."""
    M, N, K = 19, 40, 96
    codes, scales, v = whole_matrix(N, K, 3)
    w = ops.MxFp4(codes.to(DEV), scales.to(DEV), K)
    for dtype in (torch.bfloat16, torch.float32):
        xv = torch.randint(-4, 5, (M, K), generator=gen(9)).double()
        x = torch.zeros(M * K + 1, dtype=dtype, device=DEV)[1:].view(M, K)
        x.copy_(xv)
        bias = torch.arange(N + 1, device=DEV, dtype=torch.float32)[1:]
        hold = torch.full((M * N + 6,), 7.0, dtype=dtype, device=DEV)
        out = hold[3:3 + M * N].view(M, N)
        ops.gemm_mxfp4(x, w, bias, out=out)
        assert torch.equal(out.cpu(), (xv @ v.T + torch.arange(1, N + 1)).float().to(dtype))
        assert (hold[:3] == 7).all() and (hold[3 + M * N:] == 7).all()


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("K", [330016, 400001])
def test_very_wide_rows(ops, kind, K):
    """Rows whose scales leave no room in shared memory.  One number in a thousand is not zero: the sums stay below 2^22."""
    M, N = 3, 20
    codes, scales, v = whole_matrix(N, K, 5)
    w = ops.MxFp4(codes.to(DEV), scales.to(DEV), K)
    some = torch.rand(M, K, generator=gen(6)) < 1e-3
    some[:, -3:] = True
    if kind == "fp4":
        code = torch.zeros(M, (K + 31) // 32 * 32, dtype=torch.int64)
        code[:, :K] = torch.where(some, 5, 0)                     # (threes)
        code[:, K:] = 7
        scale = torch.full((M, (K + 31) // 32), 127)
        code = code.view(M, -1, 32)
        x, xv = ops.MxFp4(packed(code).to(DEV), scale.to(torch.uint8).to(DEV), K), values_of(code, scale, K)
    else:
        xv = torch.where(some, torch.randint(-4, 5, (M, K), generator=gen(9)), 0).double()
        x = xv.to(torch.float32 if kind == "float32" else torch.bfloat16).to(DEV)
    want = xv @ v.T
    assert torch.equal(ops.gemm_mxfp4(x, w, out_dtype=torch.float32).cpu().double(), want)
    half = N // 2
    act = want[:, :half] * torch.sigmoid(want[:, :half]) * want[:, half:]
    got = ops.gemm_mxfp4(x, w, out_dtype=torch.float32, epilogue=ops.EPI_SILU_MUL).cpu().double()
    # (the activation's own arithmetic, and gates below -88.73, as above)
    assert ((got - act).abs() <= (8 + want[:, :half].abs()) * 2.0 ** -23 * act.abs() + 2.0 ** -121 * want[:, half:].abs()).all()


# The widest rows whose scales still leave a wave of the few rows' kernel its place in shared memory: with one tile of columns, and with two.
@pytest.mark.parametrize("kind,M,one,two", [("bfloat16", 2, 321472, 158688), ("bfloat16", 8, 315328, 155616), ("bfloat16", 16, 307136, 151520),
                                            ("bfloat16", 32, 290752, 143328), ("float32", 2, 313280, 154592), ("float32", 4, 303040, 149472),
                                            ("float32", 8, 298944, 147424), ("float32", 16, 274368, 135136), ("fp4", 2, 285728, 149344),
                                            ("fp4", 8, 214304, 126944), ("fp4", 16, 159712, 105088), ("fp4", 32, 105088, 77792),
                                            ("fp4", 64, 61408, 50496)])
def test_rows_at_the_limit_of_shared_memory(ops, kind, M, one, two):
    """Rows just within these widths, where one to three waves are left, and just beyond, where other kernels take over; junk behind the columns.
    One number in twenty is not zero, so that all sums stay below 2^21 (32 bits of them are exact from there on down to eighths)."""
    N = 20
    widest = one + 1
    codes, scales, v = whole_matrix(N, widest, 5)
    some = torch.rand(M, widest, generator=gen(6)) < 0.05
    if kind == "fp4":
        code, scale = torch.where(some, 5, 0).long(), torch.full((M, (widest + 31) // 32), 127)      # (threes)
    else:
        xv_all = torch.where(some, torch.randint(-4, 5, (M, widest), generator=gen(9)), 0).double()
    for K in (two - 30000, two - 9001, two - 2047, two, two + 1, one - 30000, one - 9001, one - 2047, one, one + 1):
        blocks = (K + 31) // 32
        w = ops.MxFp4(codes[:, :blocks * 16].contiguous().to(DEV), scales[:, :blocks].contiguous().to(DEV), K)
        if kind == "fp4":
            c = torch.full((M, blocks * 32), 7, dtype=torch.int64)
            c[:, :K] = code[:, :K]
            c = c.view(M, -1, 32)
            x, xv = ops.MxFp4(packed(c).to(DEV), scale[:, :blocks].to(torch.uint8).to(DEV), K), values_of(c, scale[:, :blocks], K)
        else:
            xv = xv_all[:, :K]
            x = xv.to(getattr(torch, kind)).to(DEV)
        want = xv @ v[:, :K].T
        assert float((xv.abs() @ v[:, :K].abs().T).max()) < 2.0 ** 21
        assert torch.equal(ops.gemm_mxfp4(x, w, out_dtype=torch.float32).cpu().double(), want), K
        gate, up = want[:, :N // 2], want[:, N // 2:]
        act = gate * torch.sigmoid(gate) * up
        got = ops.gemm_mxfp4(x, w, out_dtype=torch.float32, epilogue=ops.EPI_SILU_MUL).cpu().double()
        # (the activation's own arithmetic, and gates below -88.73, as in the very wide rows' test)
        assert ((got - act).abs() <= (8 + gate.abs()) * 2.0 ** -23 * act.abs() + 2.0 ** -121 * up.abs()).all(), K


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("M", [1, 9, 30, 50, 90])
def test_rows_of_a_larger_matrix(ops, kind, M):
    """Matrices that begin inside others, their scales at no whole word: x and w from their second row on."""
    for N, K in ((40, 96), (333, 544), (256, 1024)):
        codes, scales, v = whole_matrix(N + 1, K, 13)
        codes, scales = codes.to(DEV), scales.to(DEV)
        w = ops.MxFp4(codes[1:], scales[1:], K)
        if kind == "fp4":
            xc, xs, xv = whole_matrix(M + 1, K, 7)
            x = ops.MxFp4(xc.to(DEV)[1:], xs.to(DEV)[1:], K)
        else:
            xv = torch.randint(-4, 5, (M + 1, K), generator=gen(9)).double()
            x = xv.to(torch.float32 if kind == "float32" else torch.bfloat16).to(DEV)[1:]
        want = xv[1:] @ v[1:].T
        assert torch.equal(ops.gemm_mxfp4(x, w, out_dtype=torch.float32).cpu().double(), want), (N, K)
        assert torch.equal(ops.mxfp4_values(w, torch.float32).cpu().double(), v[1:])


def test_matrices_beyond_32_bits(ops):
    """A matrix of more than 2^31 bytes of codes: its last columns, by every number of rows."""
    N, K = 540001, 8192
    some = torch.tensor([0, 1, 262143, 262144, 524287, 524289, N - 2, N - 1])
    g = torch.Generator(device=DEV).manual_seed(1)
    codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=DEV, generator=g)
    scales = torch.randint(127, 129, (N, K // 32), device=DEV, generator=g).to(torch.uint8)
    w = ops.MxFp4(codes, scales, K)
    v = values_of(unpack(codes[some.to(DEV)].cpu()), scales[some.to(DEV)].cpu().int(), K)
    for M in (1, 20, 40):
        xv = torch.randint(-4, 5, (M, K), generator=gen(M)).double()
        for x in (xv.to(torch.bfloat16).to(DEV), xv.float().to(DEV), ops.mxfp4_quantize(xv.float().to(DEV))):
            want = (ops.mxfp4_values(x, torch.float32).cpu().double() if isinstance(x, ops.MxFp4) else xv) @ v.T
            got = ops.gemm_mxfp4(x, w, out_dtype=torch.float32)[:, some.to(DEV)].cpu().double()
            assert torch.equal(got, want), M
    last = ops.mxfp4_values(ops.MxFp4(codes[-3:], scales[-3:], K), torch.bfloat16)
    assert torch.equal(ops.mxfp4_values(w, torch.bfloat16)[-3:], last)


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("K", [64, 1100, 4128])
def test_more_than_a_million_rows(ops, kind, K):
    """More rows than a grid's second axis holds tiles of 16, by tiles and, where the rows are more than 2^31 bytes, 16 at a time; every sum
    exact (halves of at most 48 K < 2^18), the row behind the last one as it was."""
    M, N = 65535 * 16 + 21, 6
    codes, scales, v = whole_matrix(N, K, 3)
    w, v = ops.MxFp4(codes.to(DEV), scales.to(DEV), K), v.to(DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    if kind == "fp4":
        blocks = (K + 31) // 32
        x = ops.MxFp4(torch.randint(0, 256, (M, blocks * 16), dtype=torch.uint8, device=DEV, generator=g),
                      torch.randint(127, 129, (M, blocks), device=DEV, generator=g).to(torch.uint8), K)
        part = lambda a, b: ops.mxfp4_values(ops.MxFp4(x.codes[a:b], x.scales[a:b], K), torch.float32)
    else:
        x = torch.randint(-4, 5, (M, K), dtype=torch.int8, device=DEV, generator=g).to(getattr(torch, kind))
        part = lambda a, b: x[a:b]
    hold = torch.full((M + 1, N), 7.0, device=DEV)
    bias = torch.arange(N, device=DEV, dtype=torch.float32)
    ops.gemm_mxfp4(x, w, bias, out_dtype=torch.float32, out=hold[:M])
    half = ops.gemm_mxfp4(x, w, out_dtype=torch.bfloat16, epilogue=ops.EPI_SILU_MUL)
    assert (hold[M] == 7).all()
    for a in range(0, M, 1 << 17):
        b = min(M, a + (1 << 17))
        want = part(a, b).double() @ v.T
        assert torch.equal(hold[a:b].double(), want + bias.double()), a
        gate, up = want[:, :N // 2], want[:, N // 2:]
        act = gate * torch.sigmoid(gate) * up
        # (the activation's own arithmetic and gates below -88.73, as in the large tiles' test, and a rounding to bfloat16)
        bound = (8 + gate.abs()) * 2.0 ** -23 * act.abs() + 2.0 ** -121 * up.abs()
        assert ((half[a:b].double() - act).abs() <= bound + 2.0 ** -8 * (act.abs() + bound)).all(), a


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
def test_results_beyond_32_bits(ops, kind):
    """More than 2^31 numbers of a result, by tiles, stored and added into a stream: exact sums (halves of at most 48 K), in bfloat16 rounded once."""
    M, N, K = 66003, 33002, 64
    codes, scales, v = whole_matrix(N, K, 3)
    w, v = ops.MxFp4(codes.to(DEV), scales.to(DEV), K), v.to(DEV)
    if kind == "fp4":
        xc, xs, xv = whole_matrix(M, K, 7)
        x = ops.MxFp4(xc.to(DEV), xs.to(DEV), K)
    else:
        xv = torch.randint(-4, 5, (M, K), generator=gen(9)).double()
        x = xv.to(getattr(torch, kind)).to(DEV)
    xv = xv.to(DEV)
    got = ops.gemm_mxfp4(x, w, out_dtype=torch.bfloat16)
    stream = torch.ones(M, N, device=DEV)
    ops.gemm_mxfp4(x, w, out=stream, epilogue=ops.EPI_RESIDUAL)
    for a in (0, 32000, 64000, 65071, M - 100):
        want = xv[a:a + 100] @ v.T
        assert torch.equal(got[a:a + 100], want.float().to(torch.bfloat16)), a
        assert torch.equal(stream[a:a + 100].double(), want + 1), a


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("M", [1, 5, 12, 40, 200])
@pytest.mark.parametrize("K", [1, 33, 500])
def test_narrowest_gate_and_up(ops, kind, M, K):
    """One to three gate columns with their ups, beside numbers that stay: the activation within its own arithmetic (exact sums)."""
    for I in (1, 2, 3):
        codes, scales, v = whole_matrix(2 * I, K, I)
        w = ops.MxFp4(codes.to(DEV), scales.to(DEV), K)
        if kind == "fp4":
            xc, xs, xv = whole_matrix(M, K, 7)
            x = ops.MxFp4(xc.to(DEV), xs.to(DEV), K)
        else:
            xv = torch.randint(-4, 5, (M, K), generator=gen(9)).double()
            x = xv.to(getattr(torch, kind)).to(DEV)
        want = xv @ v.T
        gate, up = want[:, :I], want[:, I:]
        act = gate * torch.sigmoid(gate) * up
        hold = torch.full((M * I + 2,), 7.0, device=DEV)
        ops.gemm_mxfp4(x, w, out_dtype=torch.float32, out=hold[1:-1].view(M, I), epilogue=ops.EPI_SILU_MUL)
        got = hold[1:-1].view(M, I).cpu().double()
        assert ((got - act).abs() <= (8 + gate.abs()) * 2.0 ** -23 * act.abs() + 2.0 ** -121 * up.abs()).all()
        assert hold[0] == 7 and hold[-1] == 7


def test_quantize_beyond_32_bits(ops):
    T, K = 66000, 32768                                        # more than 2^31 numbers
    rows = torch.randn(7, K, generator=gen(3)).to(torch.bfloat16).to(DEV)
    x = rows.repeat(T // 7 + 1, 1)[:T]
    m, few = ops.mxfp4_quantize(x), ops.mxfp4_quantize(rows)
    at = torch.tensor([0, 1, 32767, 65535, 65536, T - 1], device=DEV)
    assert torch.equal(m.codes[at], few.codes[at % 7]) and torch.equal(m.scales[at], few.scales[at % 7])


def test_no_rows(ops):
    w = ops.mxfp4_quantize(torch.randn(8, 64, device=DEV))
    assert ops.gemm_mxfp4(torch.empty(0, 64, device=DEV), w).shape == (0, 8)
    assert ops.gemm_mxfp4(ops.mxfp4_quantize(torch.empty(0, 64, device=DEV)), w).shape == (0, 8)


@pytest.mark.parametrize("kind", ["bfloat16", "float32", "fp4"])
@pytest.mark.parametrize("M", [1, 20, 100, 260])
def test_recorded_and_on_another_stream(ops, kind, M):
    """A recorded quantisation and product replayed on new numbers, twice over, with eager work between; a stream of its own."""
    N, K = 256, 1024
    w_raw = torch.randn(N, K, generator=gen(41)).to(DEV)
    first = torch.randn(M, K, generator=gen(42)).to(DEV)
    dtype = torch.float32 if kind == "float32" else torch.bfloat16

    def go(x):
        w = ops.mxfp4_quantize(w_raw)
        x = x.to(dtype)
        return ops.gemm_mxfp4(ops.mxfp4_quantize(x) if kind == "fp4" else x, w, out_dtype=torch.float32)

    inputs = [torch.randn(M, K, generator=gen(50 + i)).to(DEV) for i in range(4)]
    want = [go(x) for x in inputs]
    static = first.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alone = go(static)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(alone, go(first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go(static)
    for _ in range(2):
        for x, w in zip(inputs, want):
            static.copy_(x)
            graph.replay()
            go(first)
            torch.cuda.synchronize()
            assert torch.equal(out, w)
