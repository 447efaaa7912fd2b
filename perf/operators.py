"""Operators around a decoder block's gated MLP, measured on one GPU: the norms before and after the block, activations kept
in 8 bits between the forward and the backward pass, and products with 4-bit weights.

``listed()`` names twelve cases, ``draw(rng)`` gives further ones of the same ranges, ``prepare`` builds what a program holds
before the call, ``run`` is one pass through an operator, ``work`` what the pass cannot do without and ``exact`` its outputs in
64 bits.  With ``own`` false ``run`` computes the formulas with elementary torch operations in 32 bits; with ``own`` true it
makes the calls of ``roc_shmem_b200.ops``.

Kinds of case and what each stands for:

  norm      RMS norms of a residual stream of ``rows`` tokens.  ``form`` "pre" is h = norm(x) w, "post" is
            out = residual + scale * gate * norm(y) w, "post_pre" is that and the next block's h = norm(out) w' in one call.
            ``train`` adds the backward pass (gradients of everything), ``checkpoint`` keeps what it needs in 8 bits
  store     activations to 8 bits (e4m3 with one power of two per row and 128 columns) and back
  swiglu    act = silu(gate) * up that keeps its input in 8 bits, and the backward pass from those
  linear4   x @ w.T with weights of 4 bits, one bf16 scale (and a zero point) per row and ``group`` columns
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
# (in features, out features): shards of the 70B Llama MLP at eight ranks, Mixtral's expert matrices, square problems
LINEAR_SHAPES = [(3584, 8192), (8192, 7168), (4096, 4096), (8192, 8192), (4096, 14336), (14336, 4096), (2048, 2048)]


def _norm(form, rows, hidden, dtype, gate, train=False, checkpoint=False, weight32=False):
    return {"kind": "norm", "form": form, "rows": rows, "hidden": hidden, "dtype": dtype, "gating": gate, "train": train,
            "checkpoint": checkpoint, "weight32": weight32}


def listed() -> list[dict]:
    return [
        # decode of one sequence through a 70B-sized block: nothing but latency
        {"name": "norms decode 1", **_norm("post_pre", 1, 8192, "bf16", "none")},
        # decode batch of a small fp16 model whose hidden size is no multiple of a vector, gate per token
        {"name": "norms decode 48 odd", **_norm("post_pre", 48, 2050, "fp16", "token", weight32=True)},
        # prefill of the 70B-sized block with a learned gate per channel
        {"name": "norms prefill 8192", **_norm("post_pre", 8192, 8192, "bf16", "channel")},
        # training step of the same norms
        {"name": "norms train 8192", **_norm("post_pre", 8192, 8192, "bf16", "channel", train=True)},
        # fp32 fine-tuning of a block that has a norm before it only, packed batch of no round size
        {"name": "norm train fp32 1000", **_norm("pre", 1000, 4100, "fp32", "none", train=True)},
        # training of a Mixtral-sized block with a gate per element, inputs of the norms kept in 8 bits
        {"name": "norms train 8 bits 16384", **_norm("post_pre", 16384, 4096, "bf16", "element", train=True, checkpoint=True)},
        # the input of a linear layer, kept in 8 bits and brought back for its weight gradient
        {"name": "store 16384", "kind": "store", "rows": 16384, "cols": 4096, "dtype": "bf16"},
        # the same of an fp32 activation whose last block of columns is not full
        {"name": "store ragged 777", "kind": "store", "rows": 777, "cols": 1000, "dtype": "fp32"},
        # activation of one rank's MLP shard, forward and backward
        {"name": "swiglu train 8192", "kind": "swiglu", "rows": 8192, "ffn": 3584},
        # decode of one sequence through the gate + up shard
        {"name": "linear4 decode 1", "kind": "linear4", "tokens": 1, "k": 8192, "n": 7168, "group": 128, "zeros": False},
        # decode batch through the down shard, finer groups with zero points
        {"name": "linear4 decode 16", "kind": "linear4", "tokens": 16, "k": 3584, "n": 8192, "group": 64, "zeros": True},
        # prefill of an expert-sized matrix
        {"name": "linear4 prefill 2000", "kind": "linear4", "tokens": 2000, "k": 4096, "n": 14336, "group": 32, "zeros": False},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "norm", "norm", "store", "swiglu", "linear4", "linear4", "linear4"])
    if kind == "norm":
        hidden = _log_int(rng, 64, 16384)
        if rng.random() < 0.7:
            hidden = max(64, hidden // 64 * 64)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        form = rng.choice(["pre", "post", "post_pre", "post_pre"])
        rows = _log_int(rng, 1, max(2, min(16384, 8192 * 8192 // (hidden * (2 if dtype == "fp32" else 1)))))
        train = rng.random() < 0.5
        gate = "none" if form == "pre" else rng.choice(["none", "channel", "token", "element"])
        checkpoint, weight32 = train and rng.random() < 0.5, rng.random() < 0.3
        if train and form == "post_pre":
            # the second norm's input is a rounded result here: one that falls the other way at a border is a step of its type
            # (of 8 bits, if kept so) off, which shows in gradients of 32 bits and says nothing
            weight32, checkpoint = False, checkpoint and dtype != "fp32"
        return _norm(form, rows, hidden, dtype, gate, train, checkpoint, weight32)
    if kind == "store":
        cols = _log_int(rng, 32, 16384)
        if rng.random() < 0.7:
            cols = max(32, cols // 32 * 32)
        return {"kind": kind, "rows": _log_int(rng, 1, min(16384, (1 << 26) // cols)), "cols": cols, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    if kind == "swiglu":
        ffn = 32 * _log_int(rng, 1, 448)
        return {"kind": kind, "rows": _log_int(rng, 1, min(16384, 8192 * 3584 // ffn)), "ffn": ffn}
    group = rng.choice([32, 64, 128, 128])
    if rng.random() < 0.6:
        k, n = rng.choice(LINEAR_SHAPES)
    else:
        k, n = group * rng.randint(1, 8192 // group), 8 * rng.randint(8, 1024)
    tokens = _log_int(rng, 1, 64) if rng.random() < 0.75 else _log_int(rng, 64, 2000)
    return {"kind": kind, "tokens": tokens, "k": k, "n": n, "group": group, "zeros": rng.random() < 0.4}


# ---- inputs --------------------------------------------------------------------------------------------------------------

def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0, offset=0.0, dtype=torch.float32):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + offset).to(dtype)
    kind = case["kind"]
    state = dict(case)
    if kind == "norm":
        R, H, dt = case["rows"], case["hidden"], DTYPES[case["dtype"]]
        wt = torch.float32 if case["weight32"] else dt
        post, pre = case["form"] != "pre", case["form"] != "post"
        leaves = []

        def leaf(name, t):
            state[name] = t.requires_grad_(case["train"])
            leaves.append(name)
        # a residual stream has a few channels far above the others and tokens of different size
        channels = torch.where(torch.rand(H, device="cuda", generator=g) < 0.01, 20.0, 1.0)
        tokens = torch.exp(torch.randn(R, 1, device="cuda", generator=g) * 0.5)
        leaf("x", (randn(R, H) * channels * tokens).to(dt))
        if post:
            leaf("y", randn(R, H, scale=0.7, dtype=dt))
            leaf("w", randn(H, scale=0.1, offset=1.0, dtype=wt))
            leaf("scale", randn(1, scale=0.05, offset=0.6))
            shape = {"none": None, "channel": (H,), "token": (R, 1), "element": (R, H)}[case["gating"]]
            if shape:
                leaf("gate", randn(*shape, scale=0.3, offset=0.5, dtype=wt if case["gating"] == "channel" else dt))
        if pre:
            leaf("w_next", randn(H, scale=0.1, offset=1.0, dtype=wt))
        if case["train"]:
            state["grads"] = [randn(R, H, scale=0.3, dtype=dt) for _ in range(post + pre)]
            if post:                                         # the loss pulls the block's output along, so the scale has a gradient
                state["grads"][0] = (state["grads"][0].float() + 0.1 * state["y"].detach().float()).to(dt)
        state["leaves"] = leaves
    elif kind == "store":
        x = randn(case["rows"], case["cols"]) * torch.exp(torch.randn(1, case["cols"], device="cuda", generator=g))
        state["x"] = x.to(DTYPES[case["dtype"]])
    elif kind == "swiglu":
        state["gu"] = randn(case["rows"], 2 * case["ffn"], scale=1.5, dtype=torch.bfloat16)
        state["dact"] = randn(case["rows"], case["ffn"], scale=0.2, dtype=torch.bfloat16)
    else:
        T, K, N, group = case["tokens"], case["k"], case["n"], case["group"]
        state["x"] = randn(T, K, dtype=torch.bfloat16)
        state["q"] = torch.randint(0, 256, (N, K // 2), device="cuda", generator=g, dtype=torch.uint8)
        state["scales"] = (torch.rand(N, K // group, device="cuda", generator=g) * 0.01 + 0.002).to(torch.bfloat16)
        state["zero_points"] = (torch.randint(5, 11, (N, K // group), device="cuda", generator=g, dtype=torch.uint8)
                                if case["zeros"] else None)
    return state


# ---- the formulas in elementary operations, 32 bits -------------------------------------------------------------------------

def _round8(x: torch.Tensor) -> torch.Tensor:
    """The values that the 8 bits of x stand for: e4m3 times the smallest power of two that holds the block's largest value."""
    rows, cols = x.shape
    pad = -cols % 128
    b = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, 128)
    mantissa, exponent = torch.frexp(b.abs().amax(dim=2, keepdim=True))              # mantissa in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.clamp(exponent - 9 + (mantissa > 0.875).int(), -126, 126)
    up, down = ((e + 127) << 23).view(torch.float32), ((127 - e) << 23).view(torch.float32)      # 2^e, 2^-e
    return ((b * down).to(torch.float8_e4m3fn).float() * up).view(rows, -1)[:, :cols]


def _rstd(v: torch.Tensor) -> torch.Tensor:
    return torch.rsqrt((v * v).sum(dim=1, keepdim=True) / v.shape[1] + EPS)


def _through_norm(v, rstd, u):
    """Gradient of v * rstd(v) for the gradient u of the result."""
    n = v * rstd
    return rstd * (u - n * ((u * n).sum(dim=1, keepdim=True) / v.shape[1]))


def _plain_norm(s: dict) -> list:
    dt = s["x"].dtype
    post, pre = s["form"] != "pre", s["form"] != "post"
    z = s["x"].float()
    outputs = []
    if post:
        y, w, scale = s["y"].float(), s["w"].float(), s["scale"].float()
        gate = s["gate"].float() if "gate" in s else torch.ones(1, device="cuda")
        r1 = _rstd(y)
        out = (z + scale * gate * (y * r1) * w).to(dt)
        outputs.append(out)
        z = out.float()                                      # the next norm reads what was stored
    if pre:
        w_next, r2 = s["w_next"].float(), _rstd(z)
        outputs.append((z * r2 * w_next).to(dt))
    if not s["train"]:
        return outputs
    grads = [g.float() for g in s["grads"]]
    found = {}
    dz = torch.zeros_like(z) if not post else grads[0]
    if pre:
        dh, kept = grads[-1], (_round8(z) if s["checkpoint"] else z)
        found["w_next"] = (dh * kept * r2).sum(dim=0)
        dz = dz + _through_norm(kept, r2, dh * w_next)
    found["x"] = dz
    if post:
        kept = _round8(y) if s["checkpoint"] else y
        n = kept * r1
        found["y"] = _through_norm(kept, r1, scale * gate * w * dz)
        found["w"] = (scale * gate * dz * n).sum(dim=0)
        found["scale"] = (gate * w * dz * n).sum().view(1)
        if "gate" in s:
            dgate = scale * w * dz * n
            found["gate"] = {"channel": lambda: dgate.sum(dim=0), "token": lambda: dgate.sum(dim=1, keepdim=True),
                             "element": lambda: dgate}[s["gating"]]()
    return outputs + [found[name].to(s[name].dtype) for name in s["leaves"]]


def _silu_parts(gu: torch.Tensor):
    """gate and up of the interleaved layout: 32 columns of one, 32 of the other."""
    rows, cols = gu.shape
    b = gu.view(rows, cols // 64, 2, 32)
    return b[:, :, 0], b[:, :, 1]


def _plain_swiglu(s: dict) -> list:
    rows, F = s["rows"], s["ffn"]
    g, u = _silu_parts(s["gu"].float())
    act = (g * torch.sigmoid(g) * u).reshape(rows, F)
    g, u = _silu_parts(_round8(s["gu"]).contiguous())
    d = s["dact"].float().view(rows, F // 32, 32)
    sig = torch.sigmoid(g)
    dgu = torch.stack((d * u * sig * (1 + g * (1 - sig)), d * g * sig), dim=2).view(rows, 2 * F)
    again = (g * sig * u).reshape(rows, F)
    return [v.to(torch.bfloat16) for v in (act, dgu, again)]


def _plain_linear4(s: dict) -> torch.Tensor:
    q = torch.stack((s["q"] & 15, s["q"] >> 4), dim=2).view(s["n"], -1, s["group"]).float()       # the low half comes first
    zero = 8.0 if s["zero_points"] is None else s["zero_points"].float().unsqueeze(2)
    w = ((q - zero) * s["scales"].float().unsqueeze(2)).view(s["n"], s["k"])
    return (s["x"].float() @ w.t()).to(torch.bfloat16)


# ---- one pass ---------------------------------------------------------------------------------------------------------------

def _own_norm(s: dict):
    from roc_shmem_b200.ops.norms import post_norm, post_pre_norm, rms_norm
    form, ckpt = s["form"], s["checkpoint"]
    if form == "pre":
        outputs = (rms_norm(s["x"], s["w_next"], eps=EPS, checkpoint=ckpt),)
    elif form == "post":
        outputs = (post_norm(s["y"], s["x"], s["w"], gate=s.get("gate"), scale=s["scale"], eps=EPS, checkpoint=ckpt),)
    else:
        outputs = post_pre_norm(s["y"], s["x"], s["w"], s["w_next"], gate=s.get("gate"), scale=s["scale"], eps=EPS, checkpoint=ckpt)
    if not s["train"]:
        return list(outputs)
    return [o.detach() for o in outputs] + list(torch.autograd.grad(outputs, [s[name] for name in s["leaves"]], s["grads"]))


def run(state: dict):
    kind = state["kind"]
    if not own:
        if kind == "norm":
            with torch.no_grad():
                return _plain_norm(state)
        if kind == "store":
            return _round8(state["x"]).to(state["x"].dtype)
        return _plain_swiglu(state) if kind == "swiglu" else _plain_linear4(state)
    if kind == "norm":
        return _own_norm(state)
    if kind == "store":
        from roc_shmem_b200.ops.checkpoint8 import restore, store
        return restore(store(state["x"]), state["x"].dtype)
    if kind == "swiglu":
        from roc_shmem_b200.ops.checkpoint8 import swiglu_backward, swiglu_store
        act, kept = swiglu_store(state["gu"])
        dgu, again = swiglu_backward(kept, state["dact"], act=True)
        return [act, dgu, again]
    from roc_shmem_b200.ops.gemm_w4 import W4Tensor, linear_w4
    return linear_w4(state["x"], W4Tensor(state["q"], state["scales"], state["zero_points"]))


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "norm":
        n, b = case["rows"] * case["hidden"], 4 if case["dtype"] == "fp32" else 2
        post, pre = case["form"] != "pre", case["form"] != "post"
        vector = case["hidden"] * (4 if case["weight32"] else b)
        gate = {"none": 0, "channel": vector, "token": case["rows"] * b, "element": n * b}[case["gating"]]
        forward = n * b * (1 + post + post + pre) + vector * (post + pre) + gate              # x and y in, out and h out
        backward = n * b * (post + pre + 1 + post) + vector * (post + pre) + gate             # their gradients in, dx and dy out
        return {"bytes": forward + case["train"] * backward,
                "flops": n * (6 * post + 4 * pre) + case["train"] * n * (12 * post + 10 * pre)}
    if kind == "store":
        n, b = case["rows"] * case["cols"], 4 if case["dtype"] == "fp32" else 2
        kept = n + case["rows"] * -(-case["cols"] // 128)
        return {"bytes": 2 * (n * b + kept), "flops": 4 * n}
    if kind == "swiglu":
        n = case["rows"] * case["ffn"]
        kept = 2 * n + case["rows"] * -(-2 * case["ffn"] // 128)
        return {"bytes": 4 * n + 2 * n + kept + kept + 2 * n + 4 * n + 2 * n, "flops": 30 * n}
    T, K, N = case["tokens"], case["k"], case["n"]
    return {"bytes": N * K // 2 + N * (K // case["group"]) * (3 if case["zeros"] else 2) + 2 * T * (K + N), "flops": 2 * T * K * N}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------------

def _exact8(x: torch.Tensor) -> torch.Tensor:
    """The 8-bit values of x: for each row and 128 columns the smallest e with max |x| <= 448 * 2^e (not under -126), and x / 2^e
    at the nearest of the numbers with 3 bits behind the first one, ties to even, whose smallest step is 2^-9."""
    x = x.double()
    parts = []
    for b in x.split(128, dim=1):
        top = b.abs().amax(dim=1, keepdim=True)
        e = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 448)).clamp(-126, 126)
        e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
        e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e).clamp(min=-126)
        v = b / torch.exp2(e)
        size = torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -6)))
        size = torch.where(torch.exp2(size) > torch.clamp(v.abs(), min=2.0 ** -6), size - 1, size)
        size = torch.where(torch.exp2(size + 1) <= v.abs(), size + 1, size)
        step = torch.exp2(size - 3)
        parts.append(torch.round(v / step) * step * torch.exp2(e))
    return torch.cat(parts, dim=1)


def _exact_norm(s: dict) -> list:
    # the gradients are autograd's through the definition; where a norm's input is kept in 8 bits, they are those of a norm whose
    # own input is the kept one while its size (the mean square) is still the true one's
    post, pre, H = s["form"] != "pre", s["form"] != "post", s["hidden"]
    v = {name: s[name].detach().double() for name in s["leaves"]}
    gate = v.get("gate", 1.0)

    def gradient(values, kept, power, dn):
        """d of n = values / sqrt(mean square + eps) by the rule dn/sqrt - n <dn, n> / (H sqrt), n taken of `kept`."""
        n = kept / power
        return dn / power - n * (dn * n).sum(1, keepdim=True) / (H * power)
    outputs, z = [], v["x"]
    if post:
        p1 = (v["y"].pow(2).mean(1, keepdim=True) + EPS).sqrt()
        z = v["x"] + v["scale"] * gate * v["w"] * (v["y"] / p1)
        outputs.append(z)
        z = z.to(s["x"].dtype).double()                      # the next norm is one of the stored sum
    if pre:
        p2 = (z.pow(2).mean(1, keepdim=True) + EPS).sqrt()
        outputs.append(z / p2 * v["w_next"])
    if not s["train"]:
        return outputs
    found, dz = {}, (s["grads"][0].double() if post else 0.0)
    if pre:
        dh = s["grads"][-1].double()
        kept = _exact8(z) if s["checkpoint"] else z
        found["w_next"] = torch.einsum("ij,ij->j", dh, kept / p2)
        dz = dz + gradient(z, kept, p2, dh * v["w_next"])
    found["x"] = dz
    if post:
        kept = _exact8(v["y"]) if s["checkpoint"] else v["y"]
        n = kept / p1
        found["y"] = gradient(v["y"], kept, p1, dz * v["scale"] * gate * v["w"])
        found["w"] = (dz * n * gate).sum(0) * v["scale"]
        found["scale"] = (dz * n * gate * v["w"]).sum().reshape(1)
        if "gate" in v:
            dg = dz * n * v["w"] * v["scale"]
            found["gate"] = dg.sum(0) if s["gating"] == "channel" else dg.sum(1, keepdim=True) if s["gating"] == "token" else dg
    return outputs + [found[name] for name in s["leaves"]]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(s)
    if case["kind"] == "store":
        return _exact8(s["x"])
    if case["kind"] == "swiglu":
        def parts(gu):
            columns = gu.double().unflatten(1, (-1, 64))
            return columns[..., :32].flatten(1), columns[..., 32:].flatten(1)
        gate, up = parts(s["gu"])
        act = gate / (1 + torch.exp(-gate)) * up
        gate, up = (t.detach().requires_grad_(True) for t in parts(_exact8(s["gu"])))
        again = gate / (1 + torch.exp(-gate)) * up
        dgate, dup = torch.autograd.grad(again, (gate, up), s["dact"].double())
        dgu = torch.cat((dgate.unflatten(1, (-1, 32)), dup.unflatten(1, (-1, 32))), dim=2).flatten(1)
        return [act, dgu, again.detach()]
    low, high = s["q"].double() % 16, torch.div(s["q"].double(), 16, rounding_mode="floor")
    w = torch.stack((low, high), dim=-1).flatten(1)
    w = w - (8 if s["zero_points"] is None else s["zero_points"].double().repeat_interleave(case["group"], dim=1))
    return s["x"].double() @ (w * s["scales"].double().repeat_interleave(case["group"], dim=1)).t()
