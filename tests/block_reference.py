"""The block operators' formulas in 64 bits, with bounds on what fp32 arithmetic and one rounding at the end may differ by."""
import torch

F32 = 2.0 ** -24                     # half a step of fp32, relative
# Operations in a row between an input and a result: up to 32 products per thread, 5 shuffles and 16 words of a row's sum, halved by
# the root, and a dozen products around them.
DEPTH = 64


def half_step(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def close(got: torch.Tensor, ref: torch.Tensor, size: torch.Tensor, depth: int = DEPTH) -> None:
    """|got - ref| is at most half a step of got's type at ref plus `depth` fp32 roundings of terms of `size`."""
    assert got.shape == ref.shape
    g = got.double()
    if not torch.equal(torch.isnan(g), torch.isnan(ref)):
        raise AssertionError("NaN in different places")
    fp32 = depth * F32 * size
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps       # steps below the smallest normal number are all alike
    tol = half_step(got.dtype) * (ref.abs() + fp32) + fp32 + tiny
    bad = ~((g - ref).abs() <= tol) & ~torch.isnan(ref)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((g - ref).abs() / tol)[bad].max()):.3g} of the bound"


def rstd_of(v, eps):
    return 1 / (v.pow(2).mean(-1, keepdim=True) + eps).sqrt()


def post(y, x, w, gate, s, eps):
    """out and the size of its terms; None stands for ones."""
    f = y * rstd_of(y, eps) * (1 if w is None else w) * (1 if gate is None else gate) * s
    return x + f, x.abs() + f.abs()


def through(kept, rstd, u, size):
    """Gradient of v * rstd(v) for the gradient u (with terms of `size`) of the result, at the kept v."""
    n = kept * rstd
    return (rstd * (u - n * (u * n).mean(-1, keepdim=True)), rstd * (size + n.abs() * (size * n.abs()).mean(-1, keepdim=True)))


def round8(x: torch.Tensor) -> torch.Tensor:
    """What 8 bits keep of x [rows, columns], in 64 bits: e4m3 times the smallest power of two that holds the block's largest finite
    value; what is not finite is NaN, and nothing rounds up to a power of two that x's type does not have."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -cols % 128)).view(rows, -1, 128)
    fine = torch.isfinite(b)
    top = torch.where(fine, b, 0.0).abs().amax(2, keepdim=True)
    m, e = torch.frexp(top)
    e = torch.clamp(e - 9 + (m > 0.875).int(), min=-126).double()
    v = b / torch.exp2(e)
    q = v.float()
    top_block = e == (8 if x.dtype is torch.float16 else 120)
    q = torch.where(top_block, q.clamp(-240, 240), q.clamp(-448, 448)).to(torch.float8_e4m3fn).double() * torch.exp2(e)
    return torch.where(fine, q, torch.nan).view(rows, -1)[:, :cols]
