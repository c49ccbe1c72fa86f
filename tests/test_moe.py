"""Mixture-of-experts layers: moe_route, moe_mlp_bf16 and moe_mlp_fp8 against
their definition in 64 bits, and the calls that they refuse (those run without
a GPU).

Tolerances. Experts are compared exactly: the choice is that of the scores in
64 bits, with ties to the lower index. Weights are f32 numbers of at most 128
roundings. An expert layer's error is bounded from its parts, row by row and
column by column: see bound().
"""
import math

import pytest
import torch

from test_fp8 import (act_ref, far_rows, quant_ref, rows_of, up128,
                      values64)

E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def E():
    from tensorflow_web_deploy_amd.ops.native import ext
    return ext()


# ------------------------------------------------------------ references


def route_ref(x, bias, k, score, groups, kept, best, renorm, scale):
    """Row by row in Python floats (64 bits); x, bias on the CPU."""
    ids, weights = [], []
    for row in x.double().tolist():
        shut = [math.isnan(v) or v == -math.inf for v in row]
        if score == 1:
            p = [0.0 if s else 1.0 if v > 700 else
                 1 / (1 + math.exp(-v)) if v > -700 else math.exp(v)
                 for v, s in zip(row, shut)]
        else:
            live = [v for v, s in zip(row, shut) if not s]
            top = max(live, default=0.0)
            p = [0.0 if s else 1.0 if v == top else math.exp(v - top)
                 for v, s in zip(row, shut)]
            total = math.fsum(p)
            p = [v / total if total else 0.0 for v in p]
        key = [-math.inf if s else v + (bias[i].item() if bias is not None
                                        else 0.0)
               for i, (v, s) in enumerate(zip(p, shut))]
        key = [-math.inf if math.isnan(v) else v for v in key]
        if groups > 1:
            size = len(key) // groups
            tops = []
            for g in range(groups):
                part = sorted((v for v in key[g * size:(g + 1) * size]
                               if v > -math.inf), reverse=True)[:best]
                tops.append(sum(part) if part else -math.inf)
            keep = sorted(range(groups), key=lambda g: (-tops[g], g))[:kept]
            key = [v if i // size in keep else -math.inf
                   for i, v in enumerate(key)]
        at = sorted((i for i in range(len(key)) if key[i] > -math.inf),
                    key=lambda i: (-key[i], i))[:k]
        w = [p[i] for i in at]
        if renorm:
            total = math.fsum(w)
            w = [v / total if total else 0.0 for v in w]
        ids.append(at + [-1] * (k - len(at)))
        weights.append([v * scale for v in w] + [0.0] * (k - len(at)))
    return (torch.tensor(ids, dtype=torch.int32).reshape(-1, k),
            torch.tensor(weights, dtype=torch.float64).reshape(-1, k))


def route(E, x, bias, k, score=0, groups=1, kept=1, best=1, renorm=True,
          scale=1.0):
    ids = torch.full((x.shape[0], k), -7, dtype=torch.int32, device=x.device)
    w = torch.full((x.shape[0], k), math.nan, device=x.device)
    E.moe_route(x, bias, ids, w, score, groups, kept, best, renorm, scale)
    return ids, w


def check_route(E, x, bias, k, *a, **kw):
    got = route(E, x, bias, k, *a, **kw)
    full = dict(zip(("score", "groups", "kept", "best", "renorm", "scale"),
                    (0, 1, 1, 1, True, 1.0)))
    full.update(zip(full, a))
    full.update(kw)
    ids, w = route_ref(x.cpu(), None if bias is None else bias.cpu(), k,
                       **full)
    assert torch.equal(got[0].cpu(), ids)
    off = (got[1].cpu().double() - w).abs()
    assert (off <= 2.0 ** -17 * w.abs() + 1e-37).all(), off.max()


def test_reference_by_hand():
    x = torch.tensor([[0.0, math.log(3.0), -math.inf, 0.0]])
    ids, w = route_ref(x, None, 3, 0, 1, 1, 1, False, 2.0)
    assert ids.tolist() == [[1, 0, 3]]
    assert torch.allclose(w, torch.tensor([[1.2, 0.4, 0.4]]).double())
    b = torch.tensor([0.0, -5.0, 9.0, 0.0])
    ids, w = route_ref(x, b, 4, 1, 2, 1, 2, True, 1.0)
    assert ids.tolist() == [[3, -1, -1, -1]] and w[0].tolist() == [1, 0, 0, 0]


# ------------------------------------------------------------- refusals


@pytest.mark.parametrize("kw,word", [
    ({"logits": torch.zeros(3, 8, dtype=torch.float64)}, "bf16 or f32"),
    ({"logits": torch.zeros(8, 3).t()}, "contiguous rows"),
    ({"logits": torch.zeros(24)}, "2D"),
    ({"logits": torch.zeros(3, 520)}, "512 experts"),
    ({"logits": torch.zeros(3, 0)}, "512 experts"),
    ({"bias": torch.zeros(7)}, "bias must be"),
    ({"bias": torch.zeros(8, dtype=torch.bfloat16)}, "bias must be Float"),
    ({"ids": torch.zeros(3, 2, dtype=torch.int64)}, "ids must be Int"),
    ({"ids": torch.zeros(2, 2, dtype=torch.int32)}, "ids must be"),
    ({"ids": torch.zeros(3, 0, dtype=torch.int32)}, "k must be"),
    ({"ids": torch.zeros(3, 9, dtype=torch.int32)}, "k must be"),
    ({"weights": torch.zeros(3, 3)}, "weights must be"),
    ({"score": 2}, "score must be"),
    ({"groups": 3}, "groups must"),
    ({"groups": 0}, "groups must"),
    ({"groups": 4, "kept": 5}, "kept must"),
    ({"kept": 0}, "kept must"),
    ({"groups": 8, "kept": 1}, "k must be"),
    ({"best": 3}, "best must"),
    ({"logits": torch.empty(1 << 27, 8, device="meta")}, "too many rows"),
    ({}, "logits must be on GPU"),
])
def test_route_refuses(E, kw, word):
    a = {"logits": torch.zeros(3, 8), "bias": None,
         "ids": torch.zeros(3, 2, dtype=torch.int32),
         "weights": torch.zeros(3, 2)}
    a.update(kw)
    with pytest.raises(RuntimeError, match=word):
        E.moe_route(**a)


def _mlp_args(fp8, t=3, k=2, e=4, d=100, h=70):
    unit, dt = (128, E4M3) if fp8 else (64, torch.bfloat16)
    dp, hp = -(-d // unit) * unit, -(-h // unit) * unit
    a = {"X": torch.zeros(t, d, dtype=torch.bfloat16),
         "ids": torch.zeros(t, k, dtype=torch.int32),
         "weights": torch.zeros(t, k), "W1": torch.zeros(e, h, dp).to(dt),
         "b1": torch.zeros(e, h), "W2": torch.zeros(e, d, hp).to(dt),
         "b2": torch.zeros(e, d),
         "Y": torch.zeros(t, d, dtype=torch.bfloat16)}
    if fp8:
        a["S1"] = torch.zeros(e, up128(h) // 128, dp // 128)
        a["S2"] = torch.zeros(e, up128(d) // 128, hp // 128)
    return a


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("kw,word", [
    ({"X": torch.zeros(3, 100)}, "X must be BFloat16"),
    ({"X": torch.zeros(100, 3, dtype=torch.bfloat16).t()}, "contiguous rows"),
    ({"ids": torch.zeros(3, 2, dtype=torch.int64)}, "ids must be Int"),
    ({"ids": torch.zeros(3, dtype=torch.int32)}, "ids must be 2D"),
    ({"ids": torch.zeros(3, 0, dtype=torch.int32)}, "experts a row"),
    ({"ids": torch.zeros(4, 2, dtype=torch.int32)}, "ids must be"),
    ({"weights": torch.zeros(3, 1)}, "weights must be"),
    ({"W1": torch.zeros(4, 70, 100)}, "W1 must be"),
    ({"W1": torch.zeros(4, 70)}, "3D"),
    ({"W2": torch.zeros(4, 100, 70)}, "W2 must be"),
    ({"b1": torch.zeros(4, 71)}, "b1 must be"),
    ({"b2": torch.zeros(100)}, "b2 must be"),
    ({"Y": torch.zeros(3, 101, dtype=torch.bfloat16)}, "Y must be"),
    ({"Y": torch.zeros(3, 100)}, "Y must be BFloat16"),
    ({"residual": torch.zeros(3, 100)}, "residual must be BFloat16"),
    ({"residual": torch.zeros(2, 100, dtype=torch.bfloat16)},
     "residual must be"),
    ({"act": 4}, "act must be"),
    ({}, "X must be on GPU"),
])
def test_mlp_refuses(E, fp8, kw, word):
    a = _mlp_args(fp8)
    a.update(kw)
    with pytest.raises(RuntimeError, match=word):
        (E.moe_mlp_fp8 if fp8 else E.moe_mlp_bf16)(**a)


@pytest.mark.parametrize("kw", [{"S1": torch.zeros(4, 1, 2)},
                                {"S2": torch.zeros(4, 1, 1).double()}])
def test_mlp_fp8_refuses_scales(E, kw):
    a = _mlp_args(True)
    a.update(kw)
    with pytest.raises(RuntimeError, match="S[12] must be"):
        E.moe_mlp_fp8(**a)


# ------------------------------------------------------------- moe_route


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("t,e,k,groups,kept,best", [
    (1, 1, 1, 1, 1, 1), (5, 3, 2, 1, 1, 1), (9, 8, 8, 1, 1, 1),
    (70, 64, 2, 1, 1, 1), (33, 65, 6, 1, 1, 2), (17, 100, 8, 4, 2, 1),
    (40, 128, 4, 8, 3, 2), (23, 256, 8, 8, 4, 2), (11, 257, 9, 1, 1, 1),
    (13, 512, 33, 64, 20, 2), (7, 511, 64, 7, 7, 2), (6, 96, 5, 32, 5, 2),
    (4, 6, 3, 6, 3, 2), (30, 256, 2, 1, 1, 1), (31, 250, 3, 10, 4, 2),
    (50, 256, 13, 1, 1, 1), (50, 256, 14, 8, 4, 1), (19, 64, 16, 1, 1, 1),
    (12, 300, 31, 1, 1, 1), (12, 300, 32, 3, 2, 2), (18, 14, 13, 1, 1, 1)])
@pytest.mark.parametrize("bias", [False, True])
def test_route(E, t, e, k, groups, kept, best, score, dtype, bias):
    g = torch.Generator().manual_seed(t * e + k)
    x = (torch.randn(t, e, generator=g) * 2).to(dtype).cuda()
    b = torch.randn(e, generator=g).cuda() * 0.3 if bias else None
    check_route(E, x, b, k, score, groups, kept, best, renorm=k % 2 == 0,
                scale=2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
@pytest.mark.parametrize("best", [1, 2])
def test_route_shut_experts(E, score, groups, kept, best):
    """Rows with few experts left, with none, with NaN, with infinities and
    with values whose scores all round to one number in 32 bits."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(12, 16, generator=g)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 1:] = -math.inf
    x[3, :12] = -math.inf
    x[4, ::2] = math.nan
    x[5, [3, 9]] = math.inf
    x[6] = -3.4e38
    x[7] = 20 + torch.arange(16) / 64.0
    x[8] = 0.5
    x[9] = -120 - torch.arange(16) * 1.0
    x[10, 5] = 80.0
    x[11] = torch.arange(16) * 2.0 ** -20
    for b in (None, torch.randn(16, generator=g).cuda() * 0.1,
              torch.full((16,), -2.0).cuda()):
        check_route(E, x.cuda(), b, 4, score, groups, kept, best)


@pytest.mark.gpu
def test_route_bias_that_shuts_and_forces(E):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(50, 24, generator=g).cuda()
    b = torch.zeros(24)
    b[3], b[7], b[11], b[20] = -math.inf, math.nan, math.inf, 1e30
    for score in (0, 1):
        check_route(E, x, b.cuda(), 6, score)
        check_route(E, x, b.cuda(), 6, score, 4, 2, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("groups,kept,best", [(1, 1, 1), (8, 3, 1), (8, 3, 2)])
def test_route_close_scores(E, score, groups, kept, best):
    """Scores apart by less than 32 bits can tell, everywhere in the row."""
    g = torch.Generator().manual_seed(8)
    # with groups over a wider range, so that two groups' sums are as a rule
    # not the sums of the same steps, which differ by 2^-52 only
    steps = torch.randint(0, 40 if groups == 1 else 4000, (64, 64),
                          generator=g)
    x = 1 + steps * 2.0 ** -23
    b = torch.randint(0, 5, (64,), generator=g) * 2.0 ** -26 + 0.25
    check_route(E, x.cuda(), None, 8, score, groups, kept, best)
    check_route(E, x.cuda(), b.cuda(), 8, score, groups, kept, best)


@pytest.mark.gpu
def test_route_rows_that_lie_apart_and_none(E):
    g = torch.Generator().manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(20, 90, generator=g).to(dtype).cuda()
        check_route(E, wide[:, 7:77], None, 5, 1)
        ids, w = route(E, wide[:0], None, 5)
        assert ids.shape == (0, 5)


# --------------------------------------------------------------- moe_mlp


class Layer:
    """Random experts, their weights in the layout that a call takes."""

    def __init__(self, E, fp8, e, d, h, bias=True, seed=0):
        g = torch.Generator().manual_seed(seed + e * d + h)
        self.E, self.fp8, self.d, self.h, self.e = E, fp8, d, h, e
        self.b1 = torch.randn(e, h, generator=g).cuda() * 0.2 if bias else None
        self.b2 = torch.randn(e, d, generator=g).cuda() * 0.2 if bias else None
        self.w, self.s = [], []
        for n, k in ((h, d), (d, h)):
            w = torch.randn(e, n, k, generator=g) * k ** -0.5
            if fp8:
                q = torch.zeros(e, n, up128(k)).to(E4M3).cuda()
                s = torch.zeros(e, up128(n) // 128, up128(k) // 128).cuda()
                for i in range(e):
                    E.quant_fp8(w[i].cuda(), q[i], s[i], 128)
                self.w.append(q), self.s.append(s)
            else:
                p = torch.zeros(e, n, -(-k // 64) * 64)
                p[..., :k] = w
                self.w.append(p.to(torch.bfloat16).cuda())

    def __call__(self, x, ids, w, residual=None, act=0, y=None):
        if y is None:
            y = torch.full(x.shape, math.nan, dtype=x.dtype, device="cuda")
        if self.fp8:
            self.E.moe_mlp_fp8(x, ids, w, self.w[0], self.s[0], self.b1,
                               self.w[1], self.s[1], self.b2, y, residual, act)
        else:
            self.E.moe_mlp_bf16(x, ids, w, self.w[0], self.b1, self.w[1],
                                self.b2, y, residual, act)
        return y

    def values(self, i, j):
        """Layer j of expert i in 64 bits."""
        k = (self.d, self.h)[j]
        if self.fp8:
            return values64(self.w[j][i], self.s[j][i], 128)[:, :k]
        return self.w[j][i].cpu().double()[:, :k]

    def check(self, got, x, ids, w, residual=None, act=0):
        """A row's error, from its parts: the hidden row h is off by
          its sums' error times the activation's slope (1.13 at most), then
          half a step of its type: bf16 2^-8 |h|; for e4m3, where its value
          moved over a border, a whole step, 2^-3 |h| at most, and a scale's
          own rounding, 2^-23 |h|; that part counts only for the values that
          lie within their error of a border, so all get the sums' error and
          each border case a step. The second product passes those on by |W2|,
          adds its own sums' error; the k rows are summed in f32, and the
          result is rounded to bf16."""
        x64, ids, w = x.cpu().double(), ids.cpu(), w.cpu().double()
        t, k = ids.shape
        y = torch.zeros(t, self.d, dtype=torch.float64)
        tol = torch.zeros_like(y)
        if self.fp8:
            q, s = quant_ref(x.cpu(), 1)
            x64 = (q * s.double().repeat_interleave(128, 1))[:, :self.d]
        zero1 = torch.zeros(self.h, dtype=torch.float64)
        zero2 = torch.zeros(self.d, dtype=torch.float64)
        for i in range(self.e):
            r, j = torch.nonzero(ids == i, as_tuple=True)
            if not len(r):
                continue
            w1, w2 = self.values(i, 0), self.values(i, 1)
            b1 = zero1 if self.b1 is None else self.b1[i].cpu().double()
            b2 = zero2 if self.b2 is None else self.b2[i].cpu().double()
            pre = x64[r] @ w1.t() + b1
            h = act_ref(pre, act)
            eh = 1.13 * self.sums(x64[r], w1, b1) + 2.0 ** -22 * pre.abs()
            if self.fp8:
                hq, sq = quant_ref(h, 1)
                f = sq.double().repeat_interleave(128, 1)[:, :self.h]
                raw, h = h, (hq[:, :self.h] * f)
                # the border next to a value is half a step from its rounding
                step = torch.exp2(torch.floor(torch.log2(
                    (raw / f).abs().clamp(2.0 ** -6, 448.0))) - 3) * f
                err = eh + 2.0 ** -22 * raw.abs()
                # a scale moves with the largest value of its block
                b = torch.nn.functional.pad(raw, (0, up128(self.h) - self.h))
                e = torch.nn.functional.pad(eh, (0, up128(self.h) - self.h))
                b = b.reshape(len(r), -1, 128).abs()
                e = e.reshape(len(r), -1, 128)
                move = (e.amax(-1) / b.amax(-1).clamp_min(1e-300) + 2.0 ** -22)
                move = move.repeat_interleave(128, 1)[:, :self.h]
                err = err + move * raw.abs()
                near = (step / 2 - (raw - h).abs()).abs() <= err
                eh = move * h.abs() + near * step * 1.01
            else:
                eh = eh + 2.0 ** -8 * h.abs()
            z = h @ w2.t() + b2
            ez = eh @ w2.abs().t() + self.sums(h.abs() + eh, w2, b2)
            ww = w[r, j][:, None]
            y.index_add_(0, r, z * ww)
            tol.index_add_(0, r, (ez + 2.0 ** -23 * z.abs()) * ww.abs()
                           + k * 2.0 ** -23 * (z * ww).abs())
        if residual is not None:
            y += residual.cpu().double()
        tol += 2.0 ** -8 * (y.abs() + tol) + 1e-38
        off = (got.cpu().double() - y).abs()
        assert (off <= tol).all(), (off / tol).max()

    def sums(self, a, w, b):
        """How far a product's sums may be off: additions in f32 with their
        low bits dropped for bf16; for e4m3 what test_fp8 says, with 7/2^13 of
        the largest product of 8 no more than that of all of them."""
        size = a.abs() @ w.abs().t() + b.abs()
        if not self.fp8:
            return (a.shape[1] + 2) * 2.0 ** -23 * size
        lost = torch.zeros_like(size)
        aa, ww = a.abs(), w.abs()
        for i in range(0, a.shape[1], 8):
            # the largest product of 8 is at most the product of the largest
            lost += (aa[:, i:i + 8].amax(1, keepdim=True)
                     * ww[:, i:i + 8].amax(1)[None])
        return (7 * 2.0 ** -13 * lost
                + (a.shape[1] / 128 + 17) * 2.0 ** -23 * size)


def some_rows(t, e, k, d, seed=0):
    g = torch.Generator().manual_seed(seed + t)
    x = torch.randn(t, d, generator=g).to(torch.bfloat16).cuda()
    ids = torch.stack([torch.randperm(e, generator=g)[:k] for _ in range(t)])
    w = torch.rand(t, k, generator=g)
    return x, ids.to(torch.int32).cuda(), w.cuda()


MLPS = [(1, 2, 1, 64, 64), (1, 16, 2, 192, 320), (2, 4, 4, 128, 128),
        (7, 3, 2, 72, 40), (33, 8, 3, 100, 130), (16, 64, 4, 136, 72),
        (130, 4, 2, 256, 192), (300, 5, 2, 65, 257), (700, 2, 1, 128, 64),
        (40, 32, 8, 131, 129)]


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t,e,k,d,h", MLPS)
def test_mlp(E, t, e, k, d, h, fp8):
    layer = Layer(E, fp8, e, d, h)
    x, ids, w = some_rows(t, e, k, d)
    layer.check(layer(x, ids, w, None, 5), x, ids, w, None, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t,e,k,d,h", [
    (16, 20, 1, 200, 136), (8, 70, 4, 72, 200), (3, 40, 5, 100, 100),
    (2000, 5, 1, 490, 700), (1000, 5, 2, 1000, 990)])
def test_mlp_every_way(E, t, e, k, d, h, fp8):
    """Without a plan for up to 32 assignments, tiles of 64 and 128 rows."""
    layer = Layer(E, fp8, e, d, h)
    x, ids, w = some_rows(t, e, k, d)
    res = torch.randn(t, d, device="cuda").to(torch.bfloat16)
    for act in (0, 1, 5):
        layer.check(layer(x, ids, w, res, act), x, ids, w, res, act)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("act", [0, 1, 2, 5])
@pytest.mark.parametrize("t", [3, 150])
def test_mlp_epilogue(E, fp8, act, t):
    for bias in (True, False):
        layer = Layer(E, fp8, 3, 96, 200, bias)
        x, ids, w = some_rows(t, 3, 2, 96)
        res = torch.randn(t, 96, device="cuda").to(torch.bfloat16)
        layer.check(layer(x, ids, w, res, act), x, ids, w, res, act)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t", [1, 5, 64, 3000])
def test_mlp_ids_that_name_no_expert(E, fp8, t):
    """-1, numbers past the last expert, rows without any, the same expert
    twice, all rows with one expert."""
    layer = Layer(E, fp8, 6, 64, 72)
    x, ids, w = some_rows(t, 6, 3, 64)
    res = torch.randn(t, 64, device="cuda").to(torch.bfloat16)
    for bad in (-1, 6, 2 ** 31 - 1, -2 ** 31):
        i = ids.clone()
        i[:, 1] = bad
        i[::3] = bad
        y = layer(x, i, w, res, 1)
        layer.check(y, x, i, w, res, 1)
        assert torch.equal(y[::3], res[::3])
    twice = ids.clone()
    twice[:, 2] = twice[:, 0]
    layer.check(layer(x, twice, w), x, twice, w)
    one = torch.full_like(ids, 4)
    layer.check(layer(x, one, w), x, one, w)
    assert (layer(x, torch.full_like(ids, -1), w) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d,offset", [(64, 0), (64, 8), (64, 3), (70, 1)])
def test_mlp_rows_that_lie_apart(E, fp8, d, offset):
    layer = Layer(E, fp8, 4, d, 80)
    x, ids, w = some_rows(50, 4, 2, 200)
    v = x[:, offset:offset + d]
    out = torch.full((52, 130), 3.0, dtype=torch.bfloat16, device="cuda")
    y = out[1:51, offset:offset + d]
    res = torch.randn(50, 111, device="cuda").to(torch.bfloat16)[:, 2:2 + d]
    layer(v, ids, w, res, 5, y)
    layer.check(y, v, ids, w, res, 5)
    y.fill_(3.0)
    assert (out == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_mlp_in_place_and_no_rows(E, fp8):
    layer = Layer(E, fp8, 4, 96, 64)
    x, ids, w = some_rows(20, 4, 2, 96)
    res = torch.randn(20, 96, device="cuda").to(torch.bfloat16)
    y = res.clone()
    layer(x, ids, w, y, 1, y)
    layer.check(y, x, ids, w, res, 1)
    assert layer(x[:0], ids[:0], w[:0]).shape == (0, 96)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_mlp_nan_stays_in_its_row(E, fp8):
    layer = Layer(E, fp8, 3, 100, 90)
    x, ids, w = some_rows(40, 3, 2, 100)
    want = layer(x, ids, w, None, 5)
    x[11, 3] = math.nan
    x[12, 4] = math.inf
    y = layer(x, ids, w, None, 5)
    assert y[11].isnan().all()
    keep = torch.ones(40, dtype=torch.bool)
    keep[11] = keep[12] = False
    assert torch.equal(y[keep], want[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t", [2, 40, 300])
def test_mlp_infinity_stays_in_its_column(E, fp8, t):
    """A term that is infinite takes nothing from the columns beside it."""
    layer = Layer(E, fp8, 4, 200, 130)
    x, ids, w = some_rows(t, 4, 2, 200)
    ids[:, 0] = 1
    ids[:, 1] = 2
    spots = {5: math.inf, 70: -math.inf, 133: math.nan}
    for c, v in spots.items():
        layer.b2[1, c] = v
    got = layer(x, ids, w)
    for c, v in spots.items():
        layer.b2[1, c] = 0
    zero = layer(x, ids, w)
    for c, v in spots.items():
        if v == v:
            assert (got[:, c] == v * w[:, 0].sign()).all()
        else:
            assert got[:, c].isnan().all()
        got[:, c] = zero[:, c]
    layer.check(got, x, ids, w)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_mlp_rows_stand_alone(E, fp8):
    """A row's bits hang neither on its place nor on the rows beside it, where
    both calls take the same path."""
    layer = Layer(E, fp8, 8, 128, 128)
    x, ids, w = some_rows(9000, 8, 2, 128)
    y = layer(x, ids, w, None, 5)
    assert torch.equal(y, layer(x, ids, w, None, 5))
    p = torch.randperm(9000, generator=torch.Generator().manual_seed(1)).cuda()
    assert torch.equal(y[p], layer(x[p], ids[p], w[p], None, 5))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_mlp_more_rows_than_a_pass_takes(E, fp8):
    layer = Layer(E, fp8, 4, 64, 64)
    t = 2 ** 16 + 77
    g = torch.Generator().manual_seed(2)
    x = torch.randn(t, 64, generator=g).to(torch.bfloat16).cuda()
    ids = torch.randint(-1, 4, (t, 2), generator=g, dtype=torch.int32).cuda()
    w = torch.rand(t, 2, generator=g).cuda()
    layer.check(layer(x, ids, w, None, 1), x, ids, w, None, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t", [1, 4, 90, 2100])
def test_layer_in_a_graph(E, fp8, t):
    """Router and experts as a layer runs them, captured, replayed with new
    inputs and with eager calls between the replays; two graphs of the same
    layer take turns."""
    layer = Layer(E, fp8, 8, 96, 64)
    g = torch.Generator().manual_seed(9)
    logits = torch.zeros(t, 8, device="cuda")
    x = torch.zeros(t, 96, dtype=torch.bfloat16, device="cuda")
    ids = torch.zeros(t, 2, dtype=torch.int32, device="cuda")
    w = torch.zeros(t, 2, device="cuda")

    def run(y):
        E.moe_route(logits, None, ids, w, 0, 1, 1, 1, True, 1.0)
        layer(x, ids, w, x, 5, y)

    ys = [torch.empty_like(x) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(ys[0])
    side.synchronize()
    graphs = []
    for y in ys:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            run(y)
    for i in range(4):
        x.copy_(torch.randn(t, 96, generator=g))
        logits.copy_(torch.randn(t, 8, generator=g))
        ys[i % 2].fill_(math.nan)
        graphs[i % 2].replay()
        got = ys[i % 2].clone()
        eager = torch.empty_like(x)
        run(eager)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        layer.check(got, x, ids, w, x, 5)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_two_streams_at_once(E, fp8):
    layer = Layer(E, fp8, 4, 128, 256)
    rows = [some_rows(500, 4, 2, 128, seed=s) for s in range(2)]
    want = [layer(*r, None, 5) for r in rows]
    streams = [torch.cuda.Stream() for _ in rows]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for s, r, o in zip(streams, rows, got):
            with torch.cuda.stream(s):
                o.append(layer(*r, None, 5))
    torch.cuda.synchronize()
    for o, y in zip(got, want):
        assert all(torch.equal(z, y) for z in o)


# ------------------------------------------------- offsets past 32 bits


@pytest.mark.gpu
def test_route_far_rows(E):
    x = far_rows(20, 70, 2 ** 28 + 3)
    x.copy_(torch.randn(20, 70, device="cuda"))
    ids, w = route(E, x, None, 5, 1)
    again = route(E, x.clone(), None, 5, 1)
    assert torch.equal(ids, again[0]) and torch.equal(w, again[1])


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t", [4, 40])
def test_mlp_far_rows(E, fp8, t):
    layer = Layer(E, fp8, 12, 64, 72)
    x, ids, w = some_rows(t, 12, 2, 64)
    apart = (2 ** 33 if t < 10 else 2 ** 29) + 8
    v, res, y = (far_rows(t, 64, apart // 4) for _ in range(3))
    v.copy_(x)
    res.copy_(torch.randn(t, 64, device="cuda"))
    layer(v, ids, w, res, 1, y)
    layer.check(y.clone(), x, ids, w, res.clone(), 1)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t", [3, 40])
def test_mlp_experts_past_4_gb(E, fp8, t):
    """The last 8 of many large experts, and the same 8 alone."""
    e, d, h = (70, 8192, 8192) if fp8 else (70, 4096, 8192)
    g = torch.Generator("cuda").manual_seed(t)
    w, s = [], []
    for n, k in ((h, d), (d, h)):
        if fp8:
            q = torch.zeros(e, n, k, dtype=torch.uint8, device="cuda")
            q[-8:] = torch.randint(0, 120, (8, n, k), generator=g,
                                   device="cuda", dtype=torch.uint8)
            w.append(q.view(E4M3))
            s.append(torch.rand(e, n // 128, k // 128, generator=g,
                                device="cuda") * 1e-4)
        else:
            q = torch.zeros(e, n, k, dtype=torch.bfloat16, device="cuda")
            q[-8:] = torch.randn(8, n, k, generator=g, device="cuda") * k ** -.5
            w.append(q)
    b1, b2 = (torch.randn(e, n, generator=g, device="cuda") for n in (h, d))
    x = torch.randn(t, d, generator=g, device="cuda").to(torch.bfloat16)
    ids = torch.randint(0, 8, (t, 1), generator=g, device="cuda",
                        dtype=torch.int32)
    pw = torch.rand(t, 1, generator=g, device="cuda")

    def run(first):
        y = torch.full_like(x, math.nan)
        a = [x, ids + (62 - first), pw]
        for j, b in ((0, b1), (1, b2)):
            a.append(w[j].view(torch.uint8)[first:].view(E4M3) if fp8
                     else w[j][first:])
            a += [s[j][first:]] if fp8 else []
            a.append(b[first:])
        (E.moe_mlp_fp8 if fp8 else E.moe_mlp_bf16)(*a, y, None, 1)
        return y

    y = run(0)
    assert not y.isnan().any() and (y != 0).any(1).all()
    assert torch.equal(y, run(62))


# ------------------------------------------------- the last choice of a row


@pytest.mark.gpu
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("bias", [None, 0.0, 0.25])
def test_route_rival_behind_a_tie_at_the_cut(E, score, bias):
    """The last place and the first one without are equal in 64 bits; a third
    expert is larger than both by less than 32 bits can tell."""
    for row, k in (([0, 0, 1e-9, -5], 1), ([3, 0, 0, 1e-8], 2),
                   ([0, 0, 0, 0, 0, 1e-9], 1), ([5, 4, 3, 0, 0, 0, 1e-9], 4)):
        x = torch.tensor([row])
        b = None if bias is None else torch.full((len(row),), bias).cuda()
        check_route(E, x.cuda(), b, k, score)


@pytest.mark.gpu
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("e,k,groups,kept", [
    (8, 1, 1, 1), (8, 3, 1, 1), (64, 2, 1, 1), (64, 8, 1, 1), (64, 13, 1, 1),
    (64, 14, 1, 1), (256, 8, 1, 1), (256, 8, 8, 4), (512, 20, 1, 1),
    (100, 33, 1, 1)])
def test_route_many_ties_at_the_cut(E, score, e, k, groups, kept):
    """Rows of few values: some large, most equal, here and there one that is
    larger or smaller by less than 32 bits can tell."""
    g = torch.Generator().manual_seed(e + k)
    x = torch.zeros(60, e)
    at = torch.rand(60, e, generator=g)
    x[at < 1.5 / e] = 1e-9
    x[at > 1 - 1.5 / e] = -1e-9
    x[(at > 0.5) & (at < 0.5 + 0.8 * k / e)] = 1.0
    x[(at > 0.2) & (at < 0.2 + 0.2 * k / e)] = 1.0 + 2.0 ** -23
    check_route(E, x.cuda(), None, k, score, groups, kept, 2)
    # one bias for all where groups' sums are compared: sums of the same terms
    # in other pairs differ by their roundings in 64 bits
    b = torch.where(torch.rand(e, generator=g) < 0.3, 0.125, 0.25)
    b = (b if groups == 1 else torch.full((e,), 0.25)).cuda()
    check_route(E, x.cuda(), b, k, score, groups, kept, 2)
    x = x.to(torch.bfloat16)  # equal logits alone
    check_route(E, x.cuda(), None, k, score, groups, kept, 2)


# ------------------------------------------------------------ moe_logits


def in_parts(w):
    """f32 [E, D] as the sum of three bf16 numbers each, D filled up to 64s"""
    w = torch.nn.functional.pad(w, (0, -w.shape[1] % 64))
    parts = []
    for _ in range(3):
        parts.append(w.to(torch.bfloat16))
        w = w - parts[-1].float()
    return torch.stack(parts)


@pytest.mark.parametrize("kw,word", [
    ({"X": torch.zeros(3, 100)}, "X must be BFloat16"),
    ({"X": torch.zeros(100, 3, dtype=torch.bfloat16).t()}, "contiguous rows"),
    ({"X": torch.zeros(300, dtype=torch.bfloat16)}, "2D"),
    ({"X": torch.zeros(3, 0, dtype=torch.bfloat16)}, "width must be"),
    ({"X": torch.empty(1 << 27, 100, dtype=torch.bfloat16, device="meta")},
     "too many rows"),
    ({"W": torch.zeros(3, 8, 128)}, "W must be BFloat16"),
    ({"W": torch.zeros(3, 8, 100, dtype=torch.bfloat16)}, "W must be"),
    ({"W": torch.zeros(2, 8, 128, dtype=torch.bfloat16)}, "W must be"),
    ({"W": torch.zeros(3, 513, 128, dtype=torch.bfloat16)}, "512 experts"),
    ({"W": torch.zeros(3 * 8 * 128 + 4, dtype=torch.bfloat16)[4:].view(
        3, 8, 128)}, "W must start at a multiple of 16"),
    ({"logits": torch.zeros(3, 8, dtype=torch.bfloat16)}, "logits must be"),
    ({"logits": torch.zeros(3, 7)}, "logits must be"),
    ({}, "X must be on GPU"),
])
def test_logits_refuses(E, kw, word):
    a = {"X": torch.zeros(3, 100, dtype=torch.bfloat16),
         "W": torch.zeros(3, 8, 128, dtype=torch.bfloat16),
         "logits": torch.zeros(3, 8)}
    a.update(kw)
    with pytest.raises(RuntimeError, match=word):
        E.moe_logits(**a)


def logits_error(x, w):
    """3 D products, which are exact, added in f32, no addition off by more
    than 2^-23 of the terms' size; what three bf16 numbers lose of an f32 one
    is under 2^-24 of it."""
    n = 3 * w.shape[1] + 32
    return n * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t())


def check_logits(E, x, w):
    got = torch.full((x.shape[0], w.shape[0]), math.nan, device="cuda")
    E.moe_logits(x, in_parts(w).cuda(), got)
    x = x.cpu()
    off = (got.cpu().double() - x.double() @ w.double().t()).abs()
    assert (off <= logits_error(x, w) + 1e-38).all()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("t,d,e", [
    (1, 1, 1), (1, 768, 64), (3, 64, 16), (16, 100, 17), (17, 7, 33),
    (64, 72, 12), (65, 130, 500), (196, 768, 64), (1000, 2048, 8),
    (1030, 513, 130), (5000, 200, 64), (9001, 100, 35)])
def test_logits(E, t, d, e):
    g = torch.Generator().manual_seed(t + d + e)
    x = torch.randn(t, d, generator=g).to(torch.bfloat16)
    w = torch.randn(e, d, generator=g) * d ** -0.5
    check_logits(E, x.cuda(), w)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [5, 3000])
def test_logits_of_rows_that_lie_apart(E, t):
    g = torch.Generator().manual_seed(t)
    wide = torch.randn(t, 151, generator=g).to(torch.bfloat16).cuda()
    w = torch.randn(20, 97, generator=g)
    for at in (0, 1, 8):
        check_logits(E, wide[:, at:at + 97], w)
    assert check_logits(E, wide[:0, :97], w).shape == (0, 20)
    x = far_rows(5, 97, 2 ** 30 + 3)
    x.copy_(wide[:5, :97])
    check_logits(E, x, w)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [6, 3000])
def test_logits_of_infinite_rows(E, t):
    """As the products by definition: infinite by the weight's sign, NaN where
    two of them differ; the other rows aren't touched."""
    g = torch.Generator().manual_seed(t)
    x = torch.randn(t, 80, generator=g).to(torch.bfloat16)
    w = torch.randn(10, 80, generator=g).bfloat16().float()  # parts are 0
    want = check_logits(E, x.cuda(), w)
    x[1, 3], x[2, 4], x[2, 5], x[4, 79] = (math.inf, math.inf, math.inf,
                                           -math.inf)
    x[5, 0] = math.nan
    got = torch.empty_like(want)
    E.moe_logits(x.cuda(), in_parts(w).cuda(), got)
    ref = x.double() @ w.double().t()
    for r in (1, 2, 4, 5):
        assert torch.equal(got[r].cpu().isnan(), ref[r].isnan())
        assert torch.equal(got[r].cpu().nan_to_num(nan=0, posinf=1, neginf=-1),
                           ref[r].float().nan_to_num(nan=0, posinf=1,
                                                     neginf=-1))
        got[r] = want[r]
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_logits_in_a_graph(E):
    g = torch.Generator().manual_seed(1)
    x = torch.zeros(300, 96, dtype=torch.bfloat16, device="cuda")
    w = in_parts(torch.randn(24, 96, generator=g)).cuda()
    y, eager = (torch.empty(300, 24, device="cuda") for _ in range(2))
    E.moe_logits(x, w, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        E.moe_logits(x, w, y)
    for _ in range(3):
        x.copy_(torch.randn(300, 96, generator=g))
        graph.replay()
        E.moe_logits(x, w, eager)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


def test_logits_refuses_a_launch_too_large(E):
    """128 rows and 32 experts to 512 threads, fewer than 2^32 of them"""
    t = 1 << 26
    with pytest.raises(RuntimeError, match="too many rows"):
        E.moe_logits(
            torch.empty(t, 64, dtype=torch.bfloat16, device="meta"),
            torch.zeros(3, 512, 64, dtype=torch.bfloat16),
            torch.empty(t, 512, device="meta"))


# ------------------------- scales whose product leaves the range of f32


@pytest.mark.gpu
@pytest.mark.parametrize("t,e,k", [(1, 4, 2), (8, 4, 2), (40, 8, 2),
                                   (1500, 4, 2), (9000, 4, 2)])
def test_mlp_zero_blocks_with_any_scales(E, t, e, k):
    """Blocks of weights that are all zero add nothing, however large their
    scales and those of the rows are: in the first product by rows that are
    large there, in the second by the hidden values' bias."""
    layer = Layer(E, True, e, 256, 300)
    x, ids, w = some_rows(t, e, k, 256)
    x[:, 128:] = 0
    layer.w[0].view(torch.uint8)[:, :, 128:] = 0
    layer.w[1].view(torch.uint8)[:, :, 128:256] = 0
    layer.s[0][:, :, 1] = 1.0
    layer.s[1][:, :, 1] = 1.0
    want = layer(x, ids, w, None, 5)
    layer.check(want, x, ids, w, None, 5)
    x[:, 128:] = 1e35
    layer.b1[:, 128:256] = 1e35
    layer.s[0][:, :, 1] = 1e20
    layer.s[1][:, :, 1] = 1e20
    assert torch.equal(layer(x, ids, w, None, 5), want)


@pytest.mark.gpu
def test_route_large_scale(E):
    """The scale over a small sum of scores leaves f32's range, the weights
    don't."""
    x = torch.tensor([[-60.0, -61, -62], [-55, -58, -50], [0, 1, 2]]).cuda()
    for scale in (1e35, 1e38, -1e36):
        check_route(E, x, None, 2, 1, renorm=True, scale=scale)


# ------------------------------------------------ outputs over inputs


def test_logits_and_route_refuse_overlaps(E):
    b = torch.zeros(1 << 16, dtype=torch.uint8)
    f32, i32 = torch.float32, torch.int32
    x, w = rows_of(b, 0, 3, 100), rows_of(b, 4096, 24, 128).view(3, 8, 128)
    for at, name in ((8, "X"), (4096 + 6000, "W")):
        with pytest.raises(RuntimeError,
                           match=f"logits must not overlap {name}"):
            E.moe_logits(x, w, rows_of(b, at, 3, 8, dtype=f32))
    x, bias = rows_of(b, 0, 3, 8, dtype=f32), rows_of(b, 512, 1, 8,
                                                      dtype=f32)[0]
    for ids, w, word in ((4, 2048, "ids must not overlap logits"),
                         (520, 2048, "ids must not overlap bias"),
                         (2048, 4, "weights must not overlap logits"),
                         (2048, 520, "weights must not overlap bias"),
                         (2048, 2056, "weights must not overlap ids")):
        with pytest.raises(RuntimeError, match=word):
            E.moe_route(x, bias, rows_of(b, ids, 3, 2, dtype=i32),
                        rows_of(b, w, 3, 2, dtype=f32))


@pytest.mark.parametrize("fp8", [False, True])
def test_mlp_refuses_overlaps(E, fp8):
    call = E.moe_mlp_fp8 if fp8 else E.moe_mlp_bf16
    b = torch.zeros(1 << 16, dtype=torch.uint8)
    y = rows_of(b, 1024, 3, 100)
    other = rows_of(b, 1026, 3, 100)
    for name in ("X", "residual"):
        a = _mlp_args(fp8)
        a.update({"Y": y, name: other})
        with pytest.raises(RuntimeError, match=f"Y must not overlap {name}"):
            call(**a)
        a[name] = rows_of(b, 1024, 3, 100)  # Y itself
        with pytest.raises(RuntimeError, match="must be on GPU"):
            call(**a)
    for name in ("ids", "weights", "W1", "W2", "b1", "b2") + (
            ("S1", "S2") if fp8 else ()):
        a = _mlp_args(fp8)
        t = a[name]
        big = torch.zeros(t.numel() * t.element_size() + 600,
                          dtype=torch.uint8)
        a[name] = big[:-600].view(t.dtype).view(t.shape)
        a["Y"] = rows_of(big[t.numel() * t.element_size() - 4:], 0, 3, 100)
        with pytest.raises(RuntimeError, match=f"Y must not overlap {name}$"):
            call(**a)


@pytest.mark.parametrize("scale", [math.inf, -math.inf, math.nan, 1e39])
def test_route_refuses_an_infinite_scale(E, scale):
    """It would make NaN of the 0 that a place without an expert has."""
    with pytest.raises(RuntimeError, match="scale must be finite"):
        E.moe_route(torch.zeros(3, 8), None,
                    torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2),
                    scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t", [3, 60, 1500, 2 ** 16 + 70])
def test_mlp_into_its_input(E, fp8, t):
    """X as the output, and as the residual too, in every way and pass."""
    layer = Layer(E, fp8, 6, 64, 72)
    g = torch.Generator().manual_seed(t)
    x = torch.randn(t, 64, generator=g).to(torch.bfloat16).cuda()
    ids = torch.randint(-1, 6, (t, 2), generator=g, dtype=torch.int32).cuda()
    w = torch.rand(t, 2, generator=g).cuda()
    for residual in (False, True):
        want = layer(x, ids, w, x if residual else None, 5)
        y = x.clone()
        layer(y, ids, w, y if residual else None, 5, y)
        assert torch.equal(y, want)
