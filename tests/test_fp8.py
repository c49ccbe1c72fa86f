"""8-bit dense layers: quant_fp8 and gemm_fp8 against their definition in
64 bits, and the calls that they refuse (those run without a GPU).

Tolerances. e4m3 values and scales are compared exactly: each of their two
roundings (the quotient to f32, then to e4m3) belongs to the definition. A
product is rounded once at the store, by half a step of bf16. Its sums carry
the matrix unit's own arithmetic, which single products of known size show: a
product 2^3 next to one of 2^16 among the same 8 neighbours along K is kept, a
product of 2^2 is lost; in another group of 8 it is kept down to 2^-7. So of
each 8 products 7 lose less than 2^-13 of the largest one, and each addition
of a group to the running sum drops less than 2^-23 of it: 16 groups a block
and one addition for each of the K/128 blocks.
"""
import math

import pytest
import torch

E4M3 = torch.float8_e4m3fn
TINY = 2.0 ** -126


@pytest.fixture(scope="module")
def E():
    from tensorflow_web_deploy_amd.ops.native import ext
    return ext()


def up128(n):
    return -(-n // 128) * 128


def quant_ref(x, block_rows):
    """(e4m3 values as f64 [M, Kp], scales f32) of x in 64 bits, on the CPU."""
    x = x.detach().cpu().double()
    m, k = x.shape
    full = torch.zeros(up128(m) if block_rows == 128 else m, up128(k),
                       dtype=torch.float64)
    full[:m, :k] = x
    b = full.reshape(full.shape[0] // block_rows, block_rows, -1, 128)
    top = b.abs().amax((1, 3))
    s = (top / 448.0).float().clamp_min(TINY).double()
    q = (b / s[:, None, :, None]).float().double()
    step = torch.exp2(torch.floor(torch.log2(
        q.abs().clamp(2.0 ** -6, 448.0))) - 3)
    q = torch.round(q / step) * step  # ties to even
    return q.reshape(full.shape)[:m], s.float()


def run_quant(E, x, block_rows=1):
    m, k = x.shape
    kb = up128(k) // 128
    q = torch.full((m, kb * 128), 7.0, device=x.device).to(E4M3)
    s = torch.full((kb, m) if block_rows == 1 else (up128(m) // 128, kb), -1.0,
                   device=x.device)
    E.quant_fp8(x, q, s, block_rows)
    return q, s


def check_quant(x, q, s, block_rows):
    rq, rs = quant_ref(x, block_rows)
    got = s.cpu().t() if block_rows == 1 else s.cpu()
    assert torch.equal(got, rs)
    assert torch.equal(q.cpu().double(), rq)


# ------------------------------------------------------------- refusals


def _gemm_args(m=4, n=5, k=128, **kw):
    a = {"A": torch.zeros(m, k).to(E4M3), "SA": torch.zeros(k // 128, m),
         "B": torch.zeros(n, k).to(E4M3),
         "SB": torch.zeros(up128(n) // 128, k // 128),
         "C": torch.zeros(m, n, dtype=torch.bfloat16)}
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,word", [
    ({"A": torch.zeros(4, 100).to(E4M3)}, "whole blocks"),
    ({"A": torch.zeros(4, 128)}, "A must be Float8_e4m3fn"),
    ({"A": torch.zeros(3, 128).to(E4M3)}, "A must be"),
    ({"A": torch.zeros(0, 0).to(E4M3)}, "whole blocks"),
    ({"SA": torch.zeros(4, 1)}, "SA must be"),
    ({"SA": torch.zeros(1, 4, dtype=torch.float64)}, "SA must be Float"),
    ({"B": torch.zeros(5, 256).to(E4M3)}, "B must be"),
    ({"B": torch.zeros(128, 5).to(E4M3).t()}, "B must be contiguous"),
    ({"SB": torch.zeros(2, 1)}, "SB must be"),
    ({"C": torch.zeros(4, 5)}, "C must be BFloat16"),
    ({"C": torch.zeros(5, 4, dtype=torch.bfloat16).t()}, "contiguous rows"),
    ({"C": torch.zeros(1, 5, dtype=torch.bfloat16).expand(4, 5)}, "overlap"),
    ({"C": torch.zeros(20, dtype=torch.bfloat16)}, "2D"),
    ({"bias": torch.zeros(4)}, "bias must be"),
    ({"bias": torch.zeros(5, dtype=torch.bfloat16)}, "bias must be Float"),
    ({"residual": torch.zeros(4, 5)}, "residual must be BFloat16"),
    ({"residual": torch.zeros(4, 6, dtype=torch.bfloat16)},
     "residual must be"),
    ({"act": 3}, "act must be"),
    ({"act": -1}, "act must be"),
    ({"C": torch.empty(4, 1 << 27, dtype=torch.bfloat16, device="meta")},
     "C is too large"),
    ({"A": torch.zeros(4 * 128 + 4).to(E4M3)[4:].view(4, 128)},
     "A must start at a multiple of 16"),
    ({"B": torch.zeros(5 * 128 + 8).to(E4M3)[8:].view(5, 128)},
     "B must start at a multiple of 16"),
    ({}, "A must be on GPU"),
])
def test_gemm_refuses(E, kw, word):
    with pytest.raises(RuntimeError, match=word):
        E.gemm_fp8(**_gemm_args(**kw))


@pytest.mark.parametrize("x,q,s,rows,word", [
    (torch.zeros(4, 130, dtype=torch.float64), (4, 256), (2, 4), 1,
     "bf16 or f32"),
    (torch.zeros(4, 130), (4, 130), (2, 4), 1, "Q must be"),
    (torch.zeros(4, 130), (4, 256), (4, 2), 1, "S must be"),
    (torch.zeros(4, 130), (4, 256), (2, 4), 128, "S must be"),
    (torch.zeros(4, 130), (4, 256), (2, 4), 64, "block_rows"),
    (torch.zeros(4, 0), (4, 0), (0, 4), 1, "K must be"),
    (torch.zeros(130, 4).t(), (4, 256), (2, 4), 1, "contiguous rows"),
    (torch.zeros(130), (4, 256), (2, 4), 1, "2D"),
    (torch.empty(1 << 27, 1, device="meta"), (4, 128), (1, 4), 1,
     "X is too large"),
    (torch.zeros(4, 130), (4, 256), (2, 4), 1, "on GPU"),
])
def test_quant_refuses(E, x, q, s, rows, word):
    with pytest.raises(RuntimeError, match=word):
        E.quant_fp8(x, torch.zeros(q).to(E4M3), torch.zeros(s), rows)


def test_reference_rounds_to_even_and_keeps_zeros():
    x = torch.tensor([[448.0, 17.0, 19.0, -17.0, 0.0, 2.0 ** -10, 460.0]])
    x = torch.cat([x[:, :6], torch.zeros(1, 122)], 1)
    q, s = quant_ref(x, 1)
    assert s.item() == 1.0
    assert q[0, :6].tolist() == [448.0, 16.0, 20.0, -16.0, 0.0, 0.0]


# ------------------------------------------------------------ quant_fp8

SIZES = [(1, 1), (1, 128), (3, 127), (17, 129), (2, 768), (33, 1000),
         (257, 640), (5, 4099)]


@pytest.mark.gpu
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", SIZES)
def test_quant(E, m, k, dtype, block_rows):
    g = torch.Generator().manual_seed(m * 1000 + k)
    x = torch.randn(m, k, generator=g) * torch.exp2(
        torch.randint(-30, 30, (m, 1), generator=g).float())
    x = x.to(dtype).cuda()
    check_quant(x, *run_quant(E, x, block_rows), block_rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quant_ends_of_the_range(E, dtype):
    """Blocks of zeros, of the smallest and of the largest numbers."""
    g = torch.Generator().manual_seed(5)
    rows = [torch.zeros(128), torch.randn(128, generator=g) * 2.0 ** -140,
            torch.randn(128, generator=g) * 2.0 ** -118,
            torch.randn(128, generator=g).clamp(-1, 1) * 3e38,
            torch.full((128,), 1e-45), torch.full((128,), -0.0)]
    x = torch.stack(rows).to(dtype).cuda()
    check_quant(x, *run_quant(E, x), 1)


@pytest.mark.gpu
def test_quant_infinity_and_nan_stay_in_their_block(E):
    g = torch.Generator().manual_seed(6)
    x = torch.randn(4, 384, generator=g)
    x[1, 130] = math.inf
    x[2, 5] = math.nan
    q, s = run_quant(E, x.cuda())
    q, s = q.float().cpu(), s.cpu()
    assert s[1, 1] == math.inf and s[0, 2].isnan()
    assert q[1, 130].isnan() and q[2, :128].isnan().all()
    # finite values over an infinite scale
    assert q[1, 128:130].abs().sum() == 0 and q[1, 131:256].abs().sum() == 0
    x[1, 128:256] = 0
    x[2, :128] = 0
    keep = torch.ones(4, 384, dtype=torch.bool)
    keep[1, 128:256] = keep[2, :128] = False
    rq, rs = quant_ref(x, 1)
    assert torch.equal(q[keep].double(), rq[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset,width", [(0, 300), (1, 300), (7, 301)])
def test_quant_rows_that_lie_apart(E, dtype, offset, width):
    g = torch.Generator().manual_seed(7)
    x = torch.randn(9, 400, generator=g).to(dtype).cuda()
    v = x[:, offset:offset + width]
    for rows in (1, 128):
        check_quant(v, *run_quant(E, v, rows), rows)


@pytest.mark.gpu
def test_quant_no_rows(E):
    q, s = run_quant(E, torch.zeros(0, 200, device="cuda"))
    assert q.shape == (0, 256) and s.shape == (2, 0)


# ------------------------------------------------------------- gemm_fp8


def act_ref(y, act):
    return {0: lambda v: v, 1: torch.relu, 2: lambda v: v.clamp(0, 6),
            5: lambda v: 0.5 * v * torch.erfc(-v / math.sqrt(2))}[act](y)


def operands(E, m, n, k, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp2(
        (torch.rand(m, 1, generator=g) - 0.5) * 2 * spread)
    w = torch.randn(n, k, generator=g) * k ** -0.5
    w *= torch.exp2((torch.rand(n, 1, generator=g) - 0.5) * 2 * spread)
    return (*run_quant(E, x.cuda()), *run_quant(E, w.cuda(), 128))


def values64(q, s, block_rows):
    q, s = q.cpu().double(), s.cpu().double()
    s = s.t() if block_rows == 1 else s.repeat_interleave(128, 0)[:len(q)]
    return q * s.repeat_interleave(128, 1)


def check_gemm(got, qa, sa, qb, sb, bias=None, res=None, act=0):
    a, b = values64(qa, sa, 1), values64(qb, sb, 128)
    y, size = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        y, size = y + bias.cpu().double(), size + bias.cpu().double().abs()
    if res is not None:
        y, size = y + res.cpu().double(), size + res.cpu().double().abs()
    # relu, relu6 and erf-GELU have slopes below 1.13; erff is within
    # 2^-21 of erf, times half the value
    ref = act_ref(y, act)
    k = qa.shape[1]
    lost = torch.zeros_like(y)
    for i in range(0, k, 8):  # 7/2^13 of the largest product of each 8
        top = [a[:, None, j].abs() * b[None, :, j].abs()
               for j in range(i, i + 8)]
        lost += 7 * 2.0 ** -13 * torch.stack(top).amax(0)
    tol = 1.13 * (lost + (k / 128 + 16) * 2.0 ** -23 * size)
    tol = tol + 2.0 ** -22 * y.abs()
    tol = tol + 2.0 ** -8 * ref.abs() + 1e-38
    off = (got.cpu().double() - ref).abs()
    assert (off <= tol).all(), (off / tol).max()


GEMMS = [(1, 1, 1), (1, 16, 128), (2, 17, 300), (16, 1000, 768),
         (17, 129, 129), (63, 64, 1000), (65, 200, 4096), (128, 128, 128),
         (130, 257, 640), (300, 96, 2048), (5, 4096, 1280), (257, 513, 384),
         (31, 77, 1100), (32, 160, 128), (20, 4100, 256), (29, 40, 4200)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", GEMMS)
def test_gemm(E, m, n, k):
    ops = operands(E, m, n, k, seed=m + n + k)
    c = torch.full((m, n), math.nan, dtype=torch.bfloat16, device="cuda")
    E.gemm_fp8(*ops, c)
    check_gemm(c, *ops)


@pytest.mark.gpu
@pytest.mark.parametrize("act,residual", [(0, True), (5, False), (2, True)])
@pytest.mark.parametrize("m,n,k", [(12500, 761, 128), (4000, 4055, 4096),
                                   (6200, 768, 256), (500, 2000, 1024)])
def test_gemm_many_tiles(E, m, n, k, act, residual):
    """Some of the rows, among them each tile's first and last ones."""
    qa, sa, qb, sb = operands(E, m, n, k, seed=m)
    bias = torch.randn(n, device="cuda")
    res = (torch.randn(m, n, device="cuda").to(torch.bfloat16) if residual
           else None)
    c = torch.full((m, n), math.nan, dtype=torch.bfloat16, device="cuda")
    E.gemm_fp8(qa, sa, qb, sb, c, bias, res, act)
    assert not c.isnan().any()
    rows = sorted({0, 1, 63, 64, 127, 128, 159, 160, 255, 256, m - 130, m - 2,
                   m - 1, *range(5, m, m // 10)})
    check_gemm(c[rows], qa.view(torch.uint8)[rows].view(E4M3),
               sa[:, rows], qb, sb, bias, None if res is None else res[rows],
               act)


@pytest.mark.gpu
@pytest.mark.parametrize("act", [0, 1, 2, 5])
@pytest.mark.parametrize("m,n,k", [(3, 40, 256), (64, 96, 4096),
                                   (200, 250, 384)])
def test_gemm_epilogue(E, m, n, k, act):
    ops = operands(E, m, n, k, seed=act)
    g = torch.Generator().manual_seed(1)
    bias = torch.randn(n, generator=g).cuda()
    res = torch.randn(m, n, generator=g).to(torch.bfloat16).cuda()
    for b, r in ((bias, None), (None, res), (bias, res)):
        c = torch.full((m, n), math.nan, dtype=torch.bfloat16, device="cuda")
        E.gemm_fp8(*ops, c, b, r, act)
        check_gemm(c, *ops, b, r, act)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("m,n,k", [(40, 72, 256), (40, 71, 8192)])
def test_gemm_into_a_slice(E, m, n, k, offset):
    """Columns of a wider tensor: only they are written."""
    ops = operands(E, m, n, k)
    wide = torch.full((m + 2, n + 20), 3.0, dtype=torch.bfloat16, device="cuda")
    res = torch.randn(m, n + 9, device="cuda").to(torch.bfloat16)[:, 3:n + 3]
    c = wide[1:m + 1, offset:offset + n]
    E.gemm_fp8(*ops, c, None, res, 0)
    check_gemm(c, *ops, None, res, 0)
    wide[1:m + 1, offset:offset + n] = 3.0
    assert (wide == 3.0).all()


@pytest.mark.gpu
def test_gemm_residual_in_place(E):
    ops = operands(E, 70, 130, 512)
    c = torch.randn(70, 130, device="cuda").to(torch.bfloat16)
    res = c.clone()
    E.gemm_fp8(*ops, c, None, c, 0)
    check_gemm(c, *ops, None, res, 0)


@pytest.mark.gpu
def test_gemm_nan_stays_in_its_row(E):
    qa, sa, qb, sb = operands(E, 20, 33, 256)
    want = torch.empty(20, 33, dtype=torch.bfloat16, device="cuda")
    E.gemm_fp8(qa, sa, qb, sb, want)
    sa[1, 7] = math.nan
    c = torch.empty_like(want)
    E.gemm_fp8(qa, sa, qb, sb, c)
    assert c[7].isnan().all()
    c[7], want[7] = 0, 0
    assert torch.equal(c, want)


@pytest.mark.gpu
def test_gemm_no_rows_and_same_bits_again(E):
    ops = operands(E, 77, 200, 4096)
    c = [torch.empty(77, 200, dtype=torch.bfloat16, device="cuda")
         for _ in range(2)]
    for y in c:
        E.gemm_fp8(*ops, y)
    assert torch.equal(*c)
    qa, sa, qb, sb = ops
    E.gemm_fp8(qa[:0], sa[:, :0].contiguous(), qb, sb, c[0][:0])


@pytest.mark.gpu
def test_layer_on_a_stream_and_in_a_graph(E):
    """Rounding and product as a layer runs them: captured, replayed with new
    inputs, with other work between the replays."""
    g = torch.Generator().manual_seed(3)
    x = torch.zeros(50, 700, dtype=torch.bfloat16, device="cuda")
    qb, sb = run_quant(E, torch.randn(90, 700, generator=g).cuda(), 128)
    q = torch.empty(50, 768, dtype=E4M3, device="cuda")
    s = torch.empty(6, 50, device="cuda")
    c = torch.empty(50, 90, dtype=torch.bfloat16, device="cuda")

    def layer(y):
        E.quant_fp8(x, q, s)
        E.gemm_fp8(q, s, qb, sb, y, None, None, 5)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        layer(c)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(c)
    for i in range(3):
        x.copy_(torch.randn(50, 700, generator=g))
        graph.replay()
        got = c.clone()
        eager = torch.empty_like(c)
        layer(eager)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        check_gemm(got, q, s, qb, sb, None, None, 5)


# ------------------------------------------------- offsets past 32 bits


def far_rows(m, n, apart, dtype=torch.bfloat16):
    """Rows of n values that lie `apart` from each other."""
    return torch.empty((m - 1) * apart + n, dtype=dtype,
                       device="cuda").as_strided((m, n), (apart, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quant_far_rows(E, block_rows):
    x = far_rows(20, 200, 2 ** 28 + 3)
    x.copy_(torch.randn(20, 200, device="cuda"))
    check_quant(x.clone(), *run_quant(E, x, block_rows), block_rows)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k", [(12, 256), (40, 256), (40, 8192)])
def test_gemm_far_rows(E, m, k):
    ops = operands(E, m, 70, k)
    c, res = (far_rows(m, 70, 2 ** 28 + 5) for _ in range(2))
    res.copy_(torch.randn(m, 70, device="cuda"))
    E.gemm_fp8(*ops, c, None, res, 0)
    check_gemm(c.clone(), *ops, None, res.clone(), 0)


@pytest.mark.gpu
def test_gemm_operands_past_4_gb(E):
    n = 2 ** 25 + 5
    g = torch.Generator("cuda").manual_seed(1)
    long = torch.randint(0, 256, (n, 128), generator=g, device="cuda",
                         dtype=torch.uint8)
    long[long & 127 == 127] = 0  # no NaN
    long = long.view(E4M3)
    some = [0, 1, 2 ** 24 - 1, 2 ** 25 - 1, 2 ** 25, n - 2, n - 1]
    part = long.view(torch.uint8)[some].view(E4M3)
    for m in (2, 40):  # as weights
        qa, sa, _, _ = operands(E, m, 8, 128, seed=m)
        sb = torch.rand(up128(n) // 128, 1, generator=g, device="cuda")
        c = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
        E.gemm_fp8(qa, sa, long, sb, c)
        # one at a time: each has a block's scale of its own
        for i, at in enumerate(some):
            check_gemm(c[:, at:at + 1], qa, sa,
                       part.view(torch.uint8)[i:i + 1].view(E4M3),
                       sb[at // 128][None])
    del c
    _, _, qb, sb = operands(E, 8, 16, 128)  # as rows
    sa = torch.rand(1, n, generator=g, device="cuda")
    c = torch.empty(n, 16, dtype=torch.bfloat16, device="cuda")
    E.gemm_fp8(long, sa, qb, sb, c)
    check_gemm(c[some], part, sa[:, some], qb, sb)


# ------------------------------------------------------------ f32 results


def check_gemm_f32(got, qa, sa, qb, sb, bias=None, res=None, act=0):
    """Products of e4m3 values are exact in f32. A block's 128 of them, the
    blocks (two roundings each: of the scales' product and of the addition),
    slices of K (32 at most), bias and residual are added in f32, no addition
    off by more than 2^-23 of the terms' size. The activation's slope is 1.13
    at most; GELU's tail is off by 1e-7 times the value, under 2^-21 of it,
    and its operations by less than 2^-20 of the largest that it reaches on
    the negative side, 0.17."""
    a, b = values64(qa, sa, 1), values64(qb, sb, 128)
    y, size = a @ b.t(), a.abs() @ b.abs().t()
    for add in (bias, res):
        if add is not None:
            add = add.cpu().double()
            y, size = y + add, size + add.abs()
    ref = act_ref(y, act)
    n = 128 + 2 * qa.shape[1] / 128 + 32 + 4
    tol = 1.13 * n * 2.0 ** -23 * size + 2.0 ** -21 * y.abs() + 1e-38
    if act == 5:
        tol = tol + 2.0 ** -20 * 0.17
    off = (got.cpu().double() - ref).abs()
    assert (off <= tol).all(), (off / tol).max()


def test_gemm_refuses_f32_elsewhere(E):
    for c in (torch.zeros(4, 5), torch.zeros(4, 5, device="meta")):
        with pytest.raises(RuntimeError, match="C must be"):
            E.gemm_fp8(**_gemm_args(C=c))
    with pytest.raises(RuntimeError, match="C must be"):
        E.gemm_fp8(**_gemm_args(C=torch.zeros(4, 5, dtype=torch.float16)))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", GEMMS)
def test_gemm_f32(E, m, n, k):
    ops = operands(E, m, n, k, seed=m + n + k)
    c = torch.full((m, n), math.nan, device="cuda")
    E.gemm_fp8(*ops, c)
    check_gemm_f32(c, *ops)


@pytest.mark.gpu
@pytest.mark.parametrize("act", [0, 1, 2, 5])
@pytest.mark.parametrize("m,n,k", [(3, 40, 256), (64, 96, 4096),
                                   (200, 250, 384), (700, 520, 256)])
def test_gemm_f32_epilogue(E, m, n, k, act):
    ops = operands(E, m, n, k, seed=act)
    g = torch.Generator().manual_seed(1)
    bias = torch.randn(n, generator=g).cuda()
    res = torch.randn(m, n, generator=g).to(torch.bfloat16).cuda()
    for b, r in ((bias, None), (None, res), (bias, res)):
        c = torch.full((m, n), math.nan, device="cuda")
        E.gemm_fp8(*ops, c, b, r, act)
        check_gemm_f32(c, *ops, b, r, act)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(6200, 768, 256), (500, 2000, 1024),
                                   (3000, 2055, 1100)])
def test_gemm_f32_many_tiles(E, m, n, k):
    qa, sa, qb, sb = operands(E, m, n, k, seed=m)
    bias = torch.randn(n, device="cuda")
    res = torch.randn(m, n, device="cuda").to(torch.bfloat16)
    c = torch.full((m, n), math.nan, device="cuda")
    E.gemm_fp8(qa, sa, qb, sb, c, bias, res, 5)
    assert not c.isnan().any()
    rows = sorted({0, 1, 63, 64, 127, 128, 255, 256, m - 130, m - 2, m - 1,
                   *range(5, m, m // 10)})
    check_gemm_f32(c[rows], qa.view(torch.uint8)[rows].view(E4M3),
                   sa[:, rows], qb, sb, bias, res[rows], 5)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("m,n,k", [(12, 72, 256), (40, 72, 256),
                                   (40, 71, 8192)])
def test_gemm_f32_into_a_slice(E, m, n, k, offset):
    ops = operands(E, m, n, k)
    wide = torch.full((m + 2, n + 20), 3.0, device="cuda")
    c = wide[1:m + 1, offset:offset + n]
    E.gemm_fp8(*ops, c)
    check_gemm_f32(c, *ops)
    c.fill_(3.0)
    assert (wide == 3.0).all()


@pytest.mark.gpu
def test_gemm_f32_in_a_graph(E):
    ops = operands(E, 40, 200, 8192)
    c = torch.empty(40, 200, device="cuda")
    want = torch.empty_like(c)
    E.gemm_fp8(*ops, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.gemm_fp8(*ops, c)
    for _ in range(3):
        c.fill_(math.nan)
        graph.replay()
        assert torch.equal(c, want)
        E.gemm_fp8(*ops, want)
        torch.cuda.synchronize()


@pytest.mark.parametrize("m,n", [(4, (1 << 27) - 1), (16, (1 << 27) - 15),
                                 (20, (1 << 27) - 1)])
def test_gemm_refuses_a_launch_too_large(E, m, n):
    """16 columns to 512 threads: a launch of 2^32 threads isn't one."""
    c = torch.empty(m, n, dtype=torch.bfloat16, device="meta")
    with pytest.raises(RuntimeError, match="C is too large"):
        E.gemm_fp8(**_gemm_args(m=m, C=c))


# ------------------------- scales whose product leaves the range of f32

WAYS = [(2, 8, 256), (20, 100, 512), (40, 72, 384), (40, 70, 8192),
        (300, 96, 2048), (500, 520, 1024), (6200, 768, 256), (12500, 761, 128),
        (4000, 4055, 512), (2300, 2000, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", WAYS)
def test_gemm_zero_block_with_any_scales(E, m, n, k, dtype):
    """A block of weights that are all zero adds nothing, however large its
    scale and those of the rows are."""
    qa, sa, qb, sb = operands(E, m, n, k + 128, seed=m)
    qb.view(torch.uint8)[:, 128:256] = 0
    want = torch.full((m, n), math.nan, dtype=dtype, device="cuda")
    E.gemm_fp8(qa, sa, qb, sb, want)
    sa[1], sb[:, 1] = 0.0, 1.0
    assert want.isfinite().all()
    sa[1, ::3], sa[1, 1::3], sb[:, 1] = 1e30, 3e38, 1e20
    got = torch.full_like(want, math.nan)
    E.gemm_fp8(qa, sa, qb, sb, got)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", WAYS)
def test_gemm_scales_far_from_one(E, m, n, k, dtype):
    """Both scales near 2^-73, and near 2^66 with weights of 2^-9 in one
    place: the result is that of scales near 1 times a power of two. Off by
    the rounding to C's type, and by two f32 roundings more a block."""
    eps = torch.finfo(dtype).eps / 2 + (k / 128 + 1) * 3 * 2.0 ** -24
    sa = torch.full((k // 128, m), 1.3, device="cuda")
    sb = torch.full((up128(n) // 128, k // 128), 1.2, device="cuda")
    for value, e in ((448.0, -73), (2.0 ** -9, 66)):
        qa = torch.full((m, k), value, device="cuda").to(E4M3)
        qb = torch.full((n, k), value, device="cuda").to(E4M3)
        if e > 0:  # one product a row, 2^-18
            qa.view(torch.uint8)[:, 1:] = 0
        c = torch.full((m, n), math.nan, dtype=dtype, device="cuda")
        E.gemm_fp8(qa, sa * 2.0 ** e, qb, sb * 2.0 ** e, c)
        want = (value ** 2 * (k if e < 0 else 1) * sa[0, 0].double().item()
                * sb[0, 0].double().item())
        off = (c.double() * 2.0 ** (-2 * e) / want - 1).abs().max().item()
        assert off <= eps, (e, off, eps)


# ------------------------------------------------ outputs over inputs


def rows_of(buffer, offset, m, n, apart=None, dtype=torch.bfloat16):
    """m rows of n values within a buffer of bytes"""
    size = torch.empty(0, dtype=dtype).element_size()
    b = buffer[offset:]
    return b[:len(b) // size * size].view(dtype).as_strided(
        (m, n), (apart or n, 1))


def test_gemm_refuses_overlaps(E):
    b = torch.zeros(1 << 16, dtype=torch.uint8)
    c = rows_of(b, 1024, 4, 5, 64)
    same = rows_of(b, 1024, 4, 5, 64)
    beside = rows_of(b, 1024 + 10, 4, 5, 64)  # the columns behind C's
    for res in (rows_of(b, 1024 + 8, 4, 5, 64), rows_of(b, 1024 - 8, 4, 5, 64),
                rows_of(b, 1024 + 128, 4, 5, 64), rows_of(b, 1024, 4, 5, 63),
                rows_of(b, 1030, 4, 5)):
        with pytest.raises(RuntimeError, match="C must not overlap residual"):
            E.gemm_fp8(**_gemm_args(C=c, residual=res))
    for res in (same, beside, rows_of(b, 1024 + 3 * 128 + 10, 4, 5, 64)):
        with pytest.raises(RuntimeError, match="A must be on GPU"):
            E.gemm_fp8(**_gemm_args(C=c, residual=res))
    for name, t in (("A", rows_of(b, 1024, 4, 128, dtype=E4M3)),
                    ("SA", rows_of(b, 1024, 1, 4, dtype=torch.float32)),
                    ("B", rows_of(b, 1408, 5, 128, dtype=E4M3)),
                    ("SB", rows_of(b, 1024, 1, 1, dtype=torch.float32)),
                    ("bias", rows_of(b, 1024, 1, 5, dtype=torch.float32)[0])):
        with pytest.raises(RuntimeError, match=f"C must not overlap {name}$"):
            E.gemm_fp8(**_gemm_args(C=c, **{name: t}))


def test_quant_refuses_overlaps(E):
    b = torch.zeros(1 << 16, dtype=torch.uint8)
    x = rows_of(b, 1024, 4, 130)
    for q, s, word in ((1024, 30000, "Q must not overlap X"),
                       (1600, 30000, "Q must not overlap X"),
                       (30000 // 16 * 16, 1024, "S must not overlap X"),
                       (8192, 8192 + 512, "S must not overlap Q")):
        with pytest.raises(RuntimeError, match=word):
            E.quant_fp8(x, rows_of(b, q, 4, 256, dtype=E4M3),
                        rows_of(b, s, 2, 4, dtype=torch.float32))
