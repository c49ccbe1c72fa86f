"""Mixtures of experts as a graph op, and dense layers in 8 bits, through the
executors.

The CPU executor is compared with a plain loop in 64 bits. The GPU executor is
compared bit for bit with its layers' calls made by hand on what the plan's
own buffers hold: that each call is right is what test_fp8.py and test_moe.py
show.
"""
import math

import numpy as np
import pytest
import torch

from test_moe import route_ref
from tensorflow_web_deploy_amd.conf.config import Config
from tensorflow_web_deploy_amd.ckpt import graphdef as gd
from tensorflow_web_deploy_amd.engine import ir
from tensorflow_web_deploy_amd.engine.executor import Executor, route_experts
from tensorflow_web_deploy_amd.models.builder import GraphBuilder

E4M3 = torch.float8_e4m3fn
H, W, C, DIM, HID, CLASSES = 4, 6, 8, 72, 100, 10
MIXES = [dict(experts=6, k=2),
         dict(experts=12, k=3, score="sigmoid", groups=4, kept=2, best=2,
              renorm=False, scale=2.5, act="relu", router_bias=True)]


def model(mix, seed=3):
    """Patches -> tokens -> two dense branches -> experts -> a classifier."""
    b = GraphBuilder(seed=seed)
    x = b.placeholder("input", [-1, H, W, C])
    x = b.reshape(x, "tokens", [-1, H * W, C])

    def dense(x, name, i, o):
        y = b.node("BatchMatMulV2", name, [x, b.weight(f"{name}/w", (i, o))])
        bias = b.rng.standard_normal(o).astype(np.float32) * 0.1
        return b.node("AddV2", f"{name}/bias",
                      [y, b.const(f"{name}/b", bias)])

    x = b.relu(dense(x, "embed", C, DIM), "embed_relu")
    y = b.node("AddV2", "branches", [dense(x, "left", DIM, DIM),
                                     dense(x, "right", DIM, DIM)])
    if mix:
        y = b.node("AddV2", "sum", [b.moe(y, "experts", DIM, HID, **mix), y])
    ax = b.const("gap/axis", np.array([1], np.int32))
    y = b.node("Mean", "gap", [y, ax], keep_dims=False)
    b.softmax(b.dense(y, "head", DIM, CLASSES))
    return b


def graph(mix, seed=3):
    return ir.optimize(ir.from_graphdef(model(mix, seed).graphdef(),
                                        outputs=["softmax"]))


def config(**kw):
    return Config(input_height=H, input_width=W, input_channels=C,
                  num_classes=CLASSES, **kw)


def images(n, seed=0):
    return np.random.default_rng(seed).standard_normal(
        (n, H, W, C)).astype(np.float32)


# ------------------------------------------------------------------- CPU


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("groups,kept,best", [(1, 1, 1), (4, 2, 1), (4, 2, 2),
                                              (4, 1, 2)])
def test_route_experts(score, groups, kept, best):
    g = torch.Generator().manual_seed(groups + best)
    x = torch.randn(40, 16, generator=g, dtype=torch.float64)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 1:] = -math.inf
    x[3, 3:] = -math.inf
    x[4, ::2] = math.nan
    x[5, [3, 9]] = math.inf
    x[6] = 0.5
    x[7, 4:] = x[7, :1]
    for bias in (None, torch.randn(16, generator=g, dtype=torch.float64)):
        for renorm in (False, True):
            k = min(4, kept * 16 // groups)
            ids, w = route_experts(x, bias, k, ("softmax", "sigmoid")[score],
                                   groups, kept, best, renorm, 1.5)
            want = route_ref(x, bias, k, score, groups, kept, best, renorm,
                             1.5)
            assert torch.equal(ids.int(), want[0])
            assert ((w - want[1]).abs() <= 1e-13).all()


@pytest.mark.parametrize("mix", MIXES)
def test_moe_on_the_cpu(mix, tmp_path):
    """f32 sums of at most 100 terms, in three layers: 1e-4 of the values'
    size, and the graph survives a file."""
    path = str(tmp_path / "moe.pb")
    model(mix).save(path)
    g = ir.load_model(path, ["sum"])
    node = g.node_map()["experts"]
    assert node.op == "MoeMLP" and node.attrs["k"] == mix["k"]
    x, y = Executor(g).run({"input": torch.from_numpy(images(3))},
                           ["branches", "experts"])
    c = {n: torch.from_numpy(v).double() for n, v in g.consts.items()
         if v.dtype == np.float32}
    rows = x.double().flatten(0, 1)
    a = node.attrs
    ids, w = route_ref((x.flatten(0, 1) @ c["experts/router/w"].float()),
                       c.get("experts/router/bias"), a["k"],
                       a["score"] == "sigmoid", a["groups"], a["kept"],
                       a["best"], a["renorm"], a["scale"])
    want = torch.zeros_like(rows)
    for t in range(len(rows)):
        for j, e in enumerate(ids[t].tolist()):
            h = rows[t] @ c["experts/fc1/w"][e] + c["experts/fc1/b"][e]
            h = (torch.relu(h) if a["act"] == "relu"
                 else torch.nn.functional.gelu(h))
            want[t] += w[t, j] * (h @ c["experts/fc2/w"][e]
                                  + c["experts/fc2/b"][e])
    off = (y.double().flatten(0, 1) - want).abs()
    assert off.max() <= 1e-4 * want.abs().max()


def test_vit_with_experts():
    from tensorflow_web_deploy_amd.models import vit
    g = ir.optimize(ir.from_graphdef(
        vit.build_vit_b16(experts=2, experts_per_token=1),
        outputs=["softmax"]))
    moe = [n for n in g.nodes if n.op == "MoeMLP"]
    assert [n.name for n in moe] == [f"layer{i}/moe" for i in (1, 3, 5, 7, 9,
                                                               11)]
    assert all(n.attrs["k"] == 1 for n in moe)
    # per layer 4 projections, in every second one 2 of the MLP
    assert sum(n.op == "DenseND" for n in g.nodes) == 12 * 4 + 6 * 2


# ------------------------------------------------------------------- GPU


def engine(g, **kw):
    from tensorflow_web_deploy_amd.engine.service import LocalEngine
    return LocalEngine(config(device="cuda", **kw), graph=g)


def quant(E, x, rows):
    kb = -(-x.shape[1] // 128)
    q = torch.empty(x.shape[0], kb * 128, dtype=E4M3, device="cuda")
    s = torch.empty((kb, x.shape[0]) if rows == 1 else
                    (-(-x.shape[0] // 128), kb), device="cuda")
    E.quant_fp8(x, q, s, rows)
    return q, s


def on_gpu(a, *shape):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda().reshape(*shape)


def dense_by_hand(E, g, name, x, act):
    """The layer's call on x; its weights from the graph."""
    n = g.node_map()[name]
    w = on_gpu(g.consts[n.inputs[1]].T, -1, x.shape[-1]).contiguous()
    y = torch.empty(x[..., 0].numel(), len(w), dtype=torch.bfloat16,
                    device="cuda")
    E.gemm_fp8(*quant(E, x.reshape(-1, x.shape[-1]), 1), *quant(E, w, 128), y,
               on_gpu(g.consts[n.attrs["bias"]], -1), None, act)
    return y.view(*x.shape[:-1], -1)


def moe_by_hand(E, g, x, fp8):
    n = g.node_map()["experts"]
    a, c = n.attrs, {i: g.consts[i] for i in n.inputs[1:]}
    wr, w1, b1, w2, b2, *rb = (c[i] for i in n.inputs[1:])
    x = x.view(-1, DIM)
    k64 = -(-DIM // 64) * 64
    lin = torch.zeros(-(-wr.shape[1] // 8) * 8, k64, device="cuda")
    lin[:wr.shape[1], :DIM] = on_gpu(wr.T, -1, DIM)
    logits = torch.empty(len(x), len(lin), dtype=torch.bfloat16, device="cuda")
    E.gemm_bf16(x, lin.bfloat16(), logits, None, None, DIM, 0)
    ids = torch.empty(len(x), a["k"], dtype=torch.int32, device="cuda")
    pw = torch.empty(len(x), a["k"], device="cuda")
    E.moe_route(logits[:, :wr.shape[1]].contiguous(),
                on_gpu(rb[0], -1) if rb else None, ids, pw,
                int(a["score"] == "sigmoid"), a["groups"], a["kept"],
                a["best"], a["renorm"], a["scale"])
    y = torch.empty_like(x)
    act = {"relu": 1, "gelu": 5}[a["act"]]
    b1, b2 = on_gpu(b1, len(b1), -1), on_gpu(b2, len(b2), -1)
    if fp8:
        (w1, s1), (w2, s2) = (
            [torch.stack(t) for t in zip(*(
                quant(E, on_gpu(e.T, *e.T.shape), 128) for e in w))]
            for w in (w1, w2))
        E.moe_mlp_fp8(x, ids, pw, w1, s1, b1, w2, s2, b2, y, None, act)
    else:
        def fill(w):
            t = torch.zeros(len(w), w.shape[2], -(-w.shape[1] // 64) * 64,
                            dtype=torch.bfloat16, device="cuda")
            t[..., :w.shape[1]] = on_gpu(w, *w.shape).transpose(1, 2)
            return t
        E.moe_mlp_bf16(x, ids, pw, fill(w1), b1, fill(w2), b2, y, None, act)
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("n", [1, 8, 40])
def test_layers_are_their_calls(mix, dtype, n):
    from tensorflow_web_deploy_amd.ops.native import ext
    E, g = ext(), graph(mix)
    eng = engine(g, dtype=dtype)
    eng.ex.run({"input": torch.from_numpy(images(n))})
    torch.cuda.synchronize()
    bufs = eng.ex._plans[n].bufs
    names = {v.op + ":" + v.name for v in g.nodes}
    assert "MoeMLP:experts" in names and "DenseND:embed_relu" in names
    assert torch.equal(bufs["experts"].view(-1, DIM),
                       moe_by_hand(E, g, bufs["branches"], dtype == "fp8"))
    if dtype == "fp8":
        for name, src, act in (("embed_relu", "tokens", 1),
                               ("left/bias", "embed_relu", 0),
                               ("right/bias", "embed_relu", 0),
                               ("head/bias_add", "gap", 0)):
            assert torch.equal(bufs[name],
                               dense_by_hand(E, g, name, bufs[src], act))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
def test_graphs_streams_and_padding_change_nothing(dtype, monkeypatch):
    g = graph(MIXES[0])
    x = images(8)
    eng = engine(g, dtype=dtype)
    first = eng.infer(x)
    assert eng.ex._plans[8].sched is not None  # two branches, two streams
    eng.infer(images(8, 1))
    for _ in range(3):
        assert np.array_equal(eng.infer(x), first)
    assert np.array_equal(eng.infer(x[:5]), first[:5])  # 5 rows run as 8
    eager = engine(g, dtype=dtype, use_hip_graphs=False)
    assert np.array_equal(eager.infer(x), first)
    monkeypatch.setenv("TWD_EXEC_STREAMS", "1")
    alone = engine(g, dtype=dtype)
    assert np.array_equal(alone.infer(x), first)


@pytest.mark.gpu
def test_fp8_model_against_f32():
    """Without experts, so that no choice can flip. An e4m3 value is off by
    2^-4 of itself at most, and so are both factors of each product, and bf16
    adds 2^-8 a layer: an interval through the layers bounds the logits."""
    g = graph(None)
    x = images(6)
    eng = engine(g, dtype="fp8")
    eng.ex.run({"input": torch.from_numpy(x)})
    got = eng.ex._plans[6].bufs["head/bias_add"].double().cpu()
    c, nodes = g.consts, g.node_map()

    def weights(name):
        n = nodes[name]
        return (torch.from_numpy(c[n.inputs[1]]).double(),
                torch.from_numpy(c[n.attrs["bias"]]).double().reshape(-1))

    def dense(v, off, name):
        w, b = weights(name)
        y = v @ w + b
        r = 2.0 ** -4 + 2.0 ** -9  # a scale's smallest values lose 2^-10 more
        top = v.abs().amax(-1, keepdim=True) + off.amax(-1, keepdim=True)
        wtop = w.abs().max()
        dv = off + r * (v.abs() + off) + top * 2.0 ** -18
        dw = r * w.abs() + wtop * 2.0 ** -18
        t = dv @ (w.abs() + dw) + v.abs() @ dw
        return y, t + 2.0 ** -7 * (y.abs() + t)

    v = torch.from_numpy(x).double().reshape(6, H * W, C)
    off = 2.0 ** -8 * v.abs()
    v, off = dense(v, off, "embed_relu")
    v = torch.relu(v)
    (a, oa), (b, ob) = dense(v, off, "left/bias"), dense(v, off, "right/bias")
    v, off = a + b, oa + ob
    off = off + 2.0 ** -7 * (v.abs() + off)
    v, off = v.mean(1), off.mean(1)
    off = off + 2.0 ** -7 * (v.abs() + off)
    v, off = dense(v, off, "head/bias_add")
    assert ((got - v).abs() <= off).all()


@pytest.mark.gpu
def test_fp8_lenet():
    """A built-in model in 8 bits, its input one that a dense layer's rows
    come to over a reshape of pooled maps."""
    from tensorflow_web_deploy_amd.engine.service import LocalEngine
    cfg = Config(model_name="lenet", dtype="fp8", device="cuda")
    p = LocalEngine(cfg).infer(np.random.default_rng(0).random(
        (8, 28, 28, 1), dtype=np.float32))
    assert p.shape == (8, 10) and (p >= 0).all()
    np.testing.assert_allclose(p.sum(1), 1.0, atol=1e-3)


# ----------------------------------------------------- the router's logits


def test_vit_routes_on_f32():
    from tensorflow_web_deploy_amd.models import vit
    g = ir.optimize(ir.from_graphdef(vit.build_vit_b16(experts=2),
                                     outputs=["softmax"]))
    moe = [n for n in g.nodes if n.op == "MoeMLP"]
    assert moe and all(n.attrs["logits"] == "f32" for n in moe)


def test_builder_refuses_other_logits():
    with pytest.raises(ValueError, match="logits"):
        model(dict(experts=4, k=1, logits="f16"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_router_decides_on_f32_logits(dtype, score, monkeypatch):
    """The engine's choices against those on logits in 64 bits, of the same
    bf16 rows and the graph's own weights: another expert only where the
    scores lie within what the f32 sums may be off. Logits rounded to bf16
    choose others in some rows."""
    from test_moe import logits_error
    from tensorflow_web_deploy_amd.ops.native import ext
    E, k = ext(), 4
    g = graph(dict(experts=64, k=k, score=score, logits="f32"))
    seen = []
    route = E.moe_route

    def spy(logits, bias, ids, *a):
        route(logits, bias, ids, *a)
        seen.append((logits, ids))

    monkeypatch.setattr(E, "moe_route", spy)
    eng = engine(g, dtype=dtype, use_hip_graphs=False)
    eng.ex.run({"input": torch.from_numpy(images(40))})
    torch.cuda.synchronize()
    (logits, ids), = seen
    assert logits.dtype == torch.float32
    x = eng.ex._plans[40].bufs["branches"].view(-1, DIM).cpu().double()
    w = torch.from_numpy(g.consts["experts/router/w"]).t().contiguous()
    exact, err = x @ w.double().t(), logits_error(x, w)
    p = (torch.softmax(exact, -1) if score == "softmax"
         else torch.sigmoid(exact))
    # a score moves by no more than itself times two logits' errors
    err = 2 * err.amax(1, keepdim=True) * p * 1.01 + 2.0 ** -50
    best = p.sort(-1, descending=True).values[:, :k]
    mine = p.gather(1, ids.cpu().long())
    assert (mine >= best - 2 * err.amax(1, keepdim=True)).all()
    a = ("softmax", "sigmoid").index(score), 1, 1, 1, True, 1.0
    want = route_ref(exact, None, k, *a)[0]
    rounded = route_ref(exact.to(torch.bfloat16), None, k, *a)[0]
    assert (rounded != want).any()
    assert (ids.cpu() != want).sum() * 10 < (rounded != want).sum()


# ------------------------------------------- weights of another width


def mismatched(op):
    """Rows of 16 values: before a dense weight for 24 of them, before experts
    for 8."""
    b = GraphBuilder(seed=1)
    x = b.placeholder("input", [-1, H, W, C])
    x = b.reshape(x, "tokens", [-1, H * W * C // 16, 16])
    if op == "experts":
        x = b.moe(x, "layer", 8, 40, experts=4, k=2)
    elif op == "DenseND":
        x = b.node("BatchMatMulV2", "layer", [x, b.weight("w", (24, 16))])
        x = b.node("AddV2", "layer/bias", [
            x, b.const("layer/b", np.zeros(16, np.float32))])
    else:
        x = b.reshape(x, "rows", [-1, 16])
        x = b.dense(x, "layer", 24, 16)
    b.node("Relu", "out", [x])
    return ir.optimize(ir.from_graphdef(b.graphdef(), outputs=["out"]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("op", ["Dense", "DenseND", "experts"])
def test_a_weight_of_another_width_is_refused(op, dtype):
    g = mismatched(op)
    eng = engine(g, dtype=dtype, use_hip_graphs=False)
    with pytest.raises((AssertionError, RuntimeError),
                       match="mismatch|invalid for input of size"):
        eng.ex.run({"input": torch.from_numpy(images(4))})


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
@pytest.mark.parametrize("part,shape", [("fc1", (6, 70, HID)),
                                        ("fc2", (6, HID - 4, DIM))])
def test_experts_of_another_width_are_refused(part, shape, dtype):
    g = graph(MIXES[0])
    g.consts[f"experts/{part}/w"] = np.ones(shape, np.float32)
    eng = engine(g, dtype=dtype, use_hip_graphs=False)
    with pytest.raises(AssertionError, match="mismatch"):
        eng.ex.run({"input": torch.from_numpy(images(4))})


# --------------------------------- choices by the CPU, on logits in f32


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_experts_decides_in_64_bits(score, dtype):
    """Scores that f32 can't tell apart; the weights are of the rows' type."""
    g = torch.Generator().manual_seed(score)
    x = (torch.randint(0, 40, (60, 16), generator=g) * 1e-9).to(dtype)
    x[:20] += 1 + torch.randint(0, 4, (20, 16), generator=g) * 2.0 ** -23
    x[0] = torch.tensor([0, 0, 1e-9, -5] * 4).to(dtype)
    bias = torch.randint(0, 3, (16,), generator=g) * 2.0 ** -26 + 0.25
    for b in (None, bias):
        ids, w = route_experts(x, b, 4, ("softmax", "sigmoid")[score],
                               scale=2.5)
        want = route_ref(x, b, 4, score, 1, 1, 1, True, 2.5)
        assert w.dtype == dtype and torch.equal(ids.int(), want[0])
        off = (w.double() - want[1]).abs()
        assert (off <= torch.finfo(dtype).eps * want[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp8"])
def test_f32_logits_in_graphs_and_padded_batches(dtype):
    g = graph(dict(experts=20, k=3, logits="f32"))
    x = images(8)
    eng = engine(g, dtype=dtype)
    first = eng.infer(x)
    eng.infer(images(8, 1))
    for _ in range(3):
        assert np.array_equal(eng.infer(x), first)
    assert np.array_equal(eng.infer(x[:5]), first[:5])  # 5 rows run as 8
    eager = engine(g, dtype=dtype, use_hip_graphs=False)
    assert np.array_equal(eager.infer(x), first)
