"""The norms before and after a block, forward and backward, against their formulas in 64 bits."""
import pytest
import torch

from block_reference import DEPTH, close, post, round8, rstd_of, through

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5


def _rand(*shape, dtype, seed, scale=1.0, offset=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + offset).to(dtype)


def _case(rows, n, dtype, gate, wdtype=None, scale="tensor", seed=0):
    w = wdtype or dtype
    c = {"y": _rand(rows, n, dtype=dtype, seed=seed), "x": _rand(rows, n, dtype=dtype, seed=seed + 1, scale=3.0),
         "w1": _rand(n, dtype=w, seed=seed + 2, scale=0.2, offset=1.0), "w2": _rand(n, dtype=w, seed=seed + 3, scale=0.2, offset=-1.0),
         "gate": None, "scale": None}
    if gate:
        shape = {"column": (n,), "row": (rows, 1), "element": (rows, n)}[gate]
        c["gate"] = _rand(*shape, dtype=w, seed=seed + 4)
    if scale == "tensor":
        c["scale"] = torch.full((1,), 0.7, dtype=w, device="cuda")
    elif scale is not None:
        c["scale"] = scale
    c["dout"], c["dh"] = _rand(rows, n, dtype=dtype, seed=seed + 5), _rand(rows, n, dtype=dtype, seed=seed + 6)
    return c


def _d(t):
    return t.detach().double() if isinstance(t, torch.Tensor) else t


def _check_forward(mode, c, got):
    z, size = _d(c["x"]), None
    if mode != "pre":
        s = 1.0 if c["scale"] is None else _d(c["scale"])
        ref, size = post(_d(c["y"]), z, _d(c["w1"]), _d(c["gate"]), s, EPS)
        out = got[0] if mode == "post_pre" else got
        close(out, ref, size)
        z = _d(out)                                          # the second norm is one of the stored sum
    if mode != "post":
        h = got[1] if mode == "post_pre" else got
        ref = z * rstd_of(z, EPS) * (1 if c["w2"] is None else _d(c["w2"]))
        close(h, ref, ref.abs())


def _check_backward(mode, c, out, grads, kept8, rows):
    """grads: name → gradient.  The column sums are of `rows` terms, added up in at most rows / groups + groups / 32 + 32 steps."""
    depth = DEPTH + 64 + rows // 4
    dz, size = (_d(c["dout"]), _d(c["dout"]).abs()) if mode != "pre" and c["dout"] is not None else (0.0, 0.0)
    if mode != "post" and c["dh"] is not None:
        z = _d(out) if mode == "post_pre" else _d(c["x"])
        r, k = rstd_of(z, EPS), (round8(z) if kept8 else z)
        dh, w2 = _d(c["dh"]), 1 if c["w2"] is None else _d(c["w2"])
        if "w2" in grads:
            close(grads["w2"], (dh * k * r).sum(0), (dh * k * r).abs().sum(0), depth)
        d, more = through(k, r, dh * w2, (dh * w2).abs())
        dz, size = dz + d, size + more
    if "x" in grads:
        close(grads["x"], dz, size)
    if mode == "pre":
        return
    y, s = _d(c["y"]), 1.0 if c["scale"] is None else _d(c["scale"])
    r, k = rstd_of(y, EPS), (round8(y) if kept8 else y)
    n, w1, gate = k * r, 1 if c["w1"] is None else _d(c["w1"]), 1 if c["gate"] is None else _d(c["gate"])
    s1 = abs(s) if isinstance(s, float) else s.abs()
    a1, ag = (w1.abs() if torch.is_tensor(w1) else 1), (gate.abs() if torch.is_tensor(gate) else 1)
    if "y" in grads:
        ref, terms = through(k, r, s * gate * w1 * dz, s1 * ag * a1 * size)
        close(grads["y"], ref, terms, 2 * DEPTH)
    if "w1" in grads:
        close(grads["w1"], (s * gate * dz * n).sum(0), (s1 * ag * size * n.abs()).sum(0), depth)
    if "scale" in grads:
        close(grads["scale"], (gate * w1 * dz * n).sum().view(1), (ag * a1 * size * n.abs()).sum().view(1), depth)
    if "gate" in grads:
        full, terms = s * w1 * dz * n, s1 * a1 * size * n.abs()
        shape = c["gate"].shape
        if shape == full.shape:
            close(grads["gate"], full, terms, depth)
        elif len(shape) == 1:
            close(grads["gate"], full.sum(0), terms.sum(0), depth)
        else:
            close(grads["gate"], full.sum(1, keepdim=True), terms.sum(1, keepdim=True), depth)


def _call(mode, c, checkpoint=False):
    from roc_shmem_b200.ops.norms import post_norm, post_pre_norm, rms_norm
    if mode == "pre":
        return rms_norm(c["x"], c["w2"], EPS, checkpoint=checkpoint)
    kw = dict(gate=c["gate"], scale=c["scale"], eps=EPS, checkpoint=checkpoint)
    if mode == "post":
        return post_norm(c["y"], c["x"], c["w1"], **kw)
    return post_pre_norm(c["y"], c["x"], c["w1"], c["w2"], **kw)


def _train(mode, c, checkpoint=False):
    names = {"pre": ("x", "w2"), "post": ("y", "x", "w1", "gate", "scale"), "post_pre": ("y", "x", "w1", "w2", "gate", "scale")}[mode]
    names = [n for n in names if isinstance(c[n], torch.Tensor)]
    for n in names:
        c[n] = c[n].detach().requires_grad_(True)
    got = _call(mode, c, checkpoint)
    outs = got if mode == "post_pre" else (got,)
    dys = {"pre": (c["dh"],), "post": (c["dout"],), "post_pre": (c["dout"], c["dh"])}[mode]
    pairs = [(o, d) for o, d in zip(outs, dys) if d is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], [c[n] for n in names], [d for _, d in pairs])
    for n, g in zip(names, grads):
        assert g.dtype == c[n].dtype and g.shape == c[n].shape, n
    return got, dict(zip(names, grads))


SHAPES = [(1, 1), (1, 8), (3, 7), (5, 64), (2, 257), (33, 1000), (300, 2048), (7, 8192), (5, 8200), (3, 16384), (2, 12001), (5000, 40)]


@pytest.mark.parametrize("mode", ["pre", "post", "post_pre"])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_forward(mode, rows, n):
    for i, (dtype, w, gate, scale) in enumerate([(BF, BF, None, "tensor"), (HF, F32, "column", 0.5), (F32, F32, "row", None), (BF, F32, "element", "tensor")]):
        c = _case(rows, n, dtype, gate, w, scale, seed=10 * i + n)
        _check_forward(mode, c, _call(mode, c))


@pytest.mark.parametrize("mode", ["pre", "post", "post_pre"])
@pytest.mark.parametrize("rows,n", SHAPES)
@pytest.mark.parametrize("kept8", [False, True])
def test_gradients(mode, rows, n, kept8):
    for i, (dtype, w, gate, scale) in enumerate([(BF, BF, "column", "tensor"), (HF, F32, "row", "tensor"), (F32, F32, "element", 0.5), (BF, BF, None, None)]):
        c = _case(rows, n, dtype, gate, w, scale, seed=7 * i + n + rows)
        got, grads = _train(mode, c, kept8)
        _check_forward(mode, c, got)
        _check_backward(mode, c, got[0] if mode == "post_pre" else got, grads, kept8, rows)


@pytest.mark.parametrize("absent", ["dout", "dh"])
def test_one_result_unused(absent):
    c = _case(19, 520, BF, "column")
    c[absent] = None
    got, grads = _train("post_pre", c)
    if absent == "dh":
        assert not grads.pop("w2").any()
        _check_backward("post", {**c}, got[0], grads, False, 19)
    else:
        _check_backward("post_pre", c, got[0], grads, False, 19)


def test_weights_left_out_and_partial_gradients():
    c = _case(21, 300, BF, None, scale=None)
    c["w1"] = c["w2"] = None
    got, grads = _train("post_pre", c)
    assert set(grads) == {"y", "x"}
    _check_forward("post_pre", c, got)
    _check_backward("post_pre", c, got[0], grads, False, 21)
    # a single leaf of several: the others cost nothing and get nothing
    c = _case(21, 300, BF, "row")
    for only in ("y", "x", "w1", "w2", "gate", "scale"):
        d = {**c, only: c[only].clone().requires_grad_(True)}
        outs = _call("post_pre", d)
        g, = torch.autograd.grad(outs, d[only], (c["dout"], c["dh"]))
        _check_backward("post_pre", c, outs[0], {only: g}, False, 21)


def test_layouts():
    """Rows apart, rows off their 16-byte boundary, a repeated row, more dimensions, a turned matrix; all give what plain copies give."""
    base = _case(12, 264, BF, "element", seed=3)
    expect, eg = _train("post_pre", {**base})
    wide = torch.zeros(12, 400, dtype=BF, device="cuda")

    def apart(t, at):
        w = wide.clone()
        w[:, at:at + 264] = t
        return w[:, at:at + 264]
    for at in (8, 3):
        c = {k: apart(v, at) if isinstance(v, torch.Tensor) and v.shape == (12, 264) else v for k, v in base.items()}
        got, g = _train("post_pre", c)
        _check_forward("post_pre", c, got)
        _check_backward("post_pre", c, got[0], g, False, 12)
        if at == 8:
            assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1]) and all(torch.equal(g[k], eg[k]) for k in g)
    c = {k: v.t().contiguous().t() if isinstance(v, torch.Tensor) and v.shape == (12, 264) else v for k, v in base.items()}
    got, g = _train("post_pre", c)
    assert torch.equal(got[0], expect[0]) and all(torch.equal(g[k], eg[k]) for k in g)
    c = {k: v.view(3, 4, 264) if isinstance(v, torch.Tensor) and v.shape == (12, 264) else v for k, v in base.items()}
    got, g = _train("post_pre", c)
    assert got[0].shape == (3, 4, 264) and torch.equal(got[1].view(12, 264), expect[1]) and torch.equal(g["gate"].view(12, 264), eg["gate"])
    one = _rand(1, 264, dtype=BF, seed=9)
    many = {**base, "y": one.expand(12, 264)}
    got = _call("post_pre", many)
    again = _call("post_pre", {**base, "y": one.expand(12, 264).contiguous()})
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])
    v = _rand(264, dtype=BF, seed=9)                          # one row without a dimension of rows
    from roc_shmem_b200.ops.norms import rms_norm
    assert torch.equal(rms_norm(v, base["w2"], EPS), rms_norm(v[None], base["w2"], EPS)[0])
    w = _rand(528, dtype=BF, seed=8)[::2]                     # a weight with a stride
    assert torch.equal(rms_norm(base["x"], w, EPS), rms_norm(base["x"], w.contiguous(), EPS))


def test_zero_rows_and_zero_sizes():
    from roc_shmem_b200.ops.norms import post_pre_norm, rms_norm
    c = _case(6, 128, BF, "column")
    c["y"][2] = 0
    c["x"][2] = 0
    c["x"][4] = 0
    got, grads = _train("post_pre", c)
    _check_forward("post_pre", c, got)
    _check_backward("post_pre", c, got[0], grads, False, 6)
    assert not got[1][2].any()
    c = _case(6, 128, BF, "row", scale=0.0)                  # nothing of the block comes through
    c["scale"] = torch.zeros(1, dtype=BF, device="cuda")
    got, grads = _train("post_pre", c)
    assert torch.equal(got[0], c["x"]) and not grads["y"].any() and not grads["w1"].any() and not grads["gate"].any()
    _check_backward("post_pre", c, got[0], grads, False, 6)
    x = torch.empty(0, 128, dtype=BF, device="cuda", requires_grad=True)
    w = torch.ones(128, dtype=BF, device="cuda", requires_grad=True)
    h = rms_norm(x, w)
    gx, gw = torch.autograd.grad(h, (x, w), torch.empty_like(h))
    assert h.shape == (0, 128) and gx.shape == x.shape and not gw.any()
    assert [t.shape for t in post_pre_norm(x, x, w, w)] == [(0, 128)] * 2
    # a NaN or an infinity stays in its row
    c = _case(5, 96, F32, None)
    c["y"][1, 3], c["x"][3, 4] = float("nan"), float("inf")
    out, h = _call("post_pre", c)
    assert torch.isfinite(out[[0, 2, 4]]).all() and torch.isfinite(h[[0, 2, 4]]).all() and torch.isnan(out[1]).all()


def test_against_differences():
    """Directional differences of a weighted sum of the results, fp32, step 2^-6.  The third derivative along the direction is below
    10 per unit of length cubed for unit-size rows, so the difference is within 10 * 2^-12 / 6 of the slope, relative to the terms' size;
    fp32 adds 64 * 2^-24 * 2^6.  Both together are below 2^-7."""
    c = _case(9, 260, F32, "column", seed=77)
    c["x"] = c["x"] / 3
    got, grads = _train("post_pre", c)

    def loss(d):
        out, h = _call("post_pre", d)
        return (out.double() * c["dout"].double()).sum() + (h.double() * c["dh"].double()).sum()
    with torch.no_grad():
        for i, name in enumerate(grads):
            v = _rand(*c[name].shape, dtype=F32, seed=200 + i)
            step = 2.0 ** -6
            up, down = ({**c, name: (c[name] + s * step * v).detach()} for s in (1, -1))
            slope = (loss(up) - loss(down)) / (2 * step)
            expect = (grads[name].double() * v.double()).sum()
            size = (grads[name].double() * v.double()).norm() * 4
            assert (slope - expect).abs() <= 2.0 ** -7 * torch.maximum(size, (grads[name].double() * v.double()).abs().sum()), name


def test_same_bits_again_and_other_streams():
    c = _case(1500, 1024, BF, "row")
    _, first = _train("post_pre", {**c})
    _, second = _train("post_pre", {**c})
    assert all(torch.equal(first[k], second[k]) for k in first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _, third = _train("post_pre", {**c})
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first[k], third[k]) for k in first)


def test_graph_capture_forward_and_backward():
    c = _case(40, 512, BF, "column")
    names = ("y", "x", "w1", "w2", "gate", "scale")
    for n in names:
        c[n] = c[n].clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = _call("post_pre", c, True)
        torch.autograd.grad(outs, [c[n] for n in names], (c["dout"], c["dh"]))
    torch.cuda.current_stream().wait_stream(side)
    del outs
    graphs = []
    for _ in range(2):                                        # two graphs replayed in turn share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = _call("post_pre", c, True)
            grads = torch.autograd.grad(outs, [c[n] for n in names], (c["dout"], c["dh"]))
        graphs.append((g, [o.detach() for o in outs], grads))
    with torch.no_grad():
        c["y"].copy_(_rand(40, 512, dtype=BF, seed=99))
    for g, _, _ in graphs:
        g.replay()
    outs = _call("post_pre", c, True)
    grads = torch.autograd.grad(outs, [c[n] for n in names], (c["dout"], c["dh"]))
    for _, o, d in graphs:
        assert all(torch.equal(a, b) for a, b in zip(o, outs)) and all(torch.equal(a, b) for a, b in zip(d, grads))


def test_refusals():
    from roc_shmem_b200.ops.norms import post_norm, post_pre_norm, rms_norm
    c = _case(4, 64, BF, "column")
    x, y, w = c["x"], c["y"], c["w1"]
    for bad in (lambda: rms_norm(x.double()), lambda: rms_norm(x, w[:63]), lambda: rms_norm(x, w.half()), lambda: rms_norm(x, w.cpu()),
                lambda: rms_norm(x, eps=0.0), lambda: rms_norm(x, eps=float("nan")), lambda: rms_norm(x[:, :0]),
                lambda: rms_norm(torch.zeros(2, 16385, dtype=BF, device="cuda")), lambda: rms_norm(torch.tensor(1.0, device="cuda")),
                lambda: post_norm(y, x[:3]), lambda: post_norm(y.float(), x), lambda: post_norm(y, x, gate=w[:1]), lambda: post_norm(y, x, gate=x[:, :2]),
                lambda: post_norm(y, x, gate=x.half()), lambda: post_norm(y, x, scale=w[:2]), lambda: post_norm(y, x, scale=torch.ones(1)),
                lambda: post_pre_norm(y, x, w, w.double())):
        with pytest.raises(ValueError):
            bad()
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(rms_norm(leaf, w).float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), leaf)


# Rows enough for blocks that walk over them, with every kind of call that has a kernel of its own.
@pytest.mark.parametrize("rows,n", [(5000, 520), (700, 8192), (400, 8208), (5001, 232)])
@pytest.mark.parametrize("mode,dtype,w,gate,scale,kept8,absent", [
    ("post_pre", BF, BF, "element", "tensor", True, None), ("post_pre", BF, BF, "element", 0.5, False, None),
    ("post_pre", BF, F32, "element", 0.5, False, None), ("post_pre", HF, F32, "element", "tensor", True, None),
    ("post_pre", HF, HF, None, "tensor", False, "dout"), ("post_pre", BF, BF, "row", None, True, "dh"),
    ("post_pre", F32, F32, "column", "tensor", False, None), ("post_pre", BF, BF, None, None, True, None),
    ("post", F32, F32, "element", "tensor", True, None), ("post", BF, BF, "column", 0.5, False, None), ("post", HF, HF, "row", "tensor", True, None),
    ("pre", HF, F32, None, None, True, None), ("pre", BF, BF, None, None, False, None), ("pre", F32, F32, None, None, True, None)])
def test_many_rows_of_every_kind(rows, n, mode, dtype, w, gate, scale, kept8, absent):
    c = _case(rows, n, dtype, gate, w, scale, seed=n + rows)
    if absent:
        c[absent] = None
    got, grads = _train(mode, c, kept8)
    _check_forward(mode, c, got)
    if absent == "dh":
        assert not grads.pop("w2").any()
        mode, got = "post", got[0]
    _check_backward(mode, c, got[0] if mode == "post_pre" else got, grads, kept8, rows)


@pytest.mark.parametrize("kept8", [False, True])
def test_many_rows_whose_first_norm_has_no_gradient(kept8):
    c = _case(2000, 1024, BF, "element", BF, "tensor", seed=3)
    names = ("x", "w1", "w2", "gate", "scale")
    for name in names:
        c[name] = c[name].requires_grad_(True)
    out, h = _call("post_pre", c, kept8)
    grads = torch.autograd.grad([out, h], [c[name] for name in names], [c["dout"], c["dh"]])
    _check_backward("post_pre", c, out, dict(zip(names, grads)), kept8, 2000)


@pytest.mark.parametrize("n", [8200, 12288, 16384])
@pytest.mark.parametrize("mode,dtype,w,gate", [("post_pre", BF, BF, "column"), ("post_pre", F32, F32, None), ("post", HF, F32, "element"), ("pre", BF, F32, None)])
def test_many_long_rows(mode, dtype, w, gate, n):
    c = _case(450, n, dtype, gate, w, 0.5, seed=n)
    _check_forward(mode, c, _call(mode, c))
