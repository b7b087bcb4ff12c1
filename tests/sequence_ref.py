"""The operators over packed rows in 64 bits on the CPU, row by row from their definitions, as differentiable
torch code (gradients come from autograd over these loops), and the magnitudes that error bounds need."""
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}   # half a step at zero
U32 = 2.0 ** -24


def silu(v):
    return v / (1 + torch.exp(-v))


def bounds(offsets, rows):
    off = [0, rows] if offsets is None else [int(v) for v in offsets]
    return list(zip(off[:-1], off[1:]))


def causal_conv(x, weight, bias=None, offsets=None, act=False, initial=None):
    """(y, state); rows in no sequence are zero."""
    k, ch = weight.shape[1], x.shape[1]
    y = [None] * x.shape[0]
    states = []
    for s, (lo, hi) in enumerate(bounds(offsets, x.shape[0])):
        head = initial[s] if initial is not None else x.new_zeros(k - 1, ch)
        line = torch.cat([head, x[lo:hi]])
        for t in range(hi - lo):
            p = (line[t:t + k] * weight.t()).sum(0)
            if bias is not None:
                p = p + bias
            y[lo + t] = silu(p) if act else p
        states.append(line[len(line) - (k - 1):])
    zero = x.new_zeros(ch)
    y = torch.stack([zero if v is None else v for v in y]) if y else x.new_zeros(0, ch)
    return y, torch.stack(states) if states else x.new_zeros(0, k - 1, ch)


def softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def selective_scan(u, delta, A, B, C, D=None, delta_bias=None, offsets=None, plus=False, initial=None):
    """(y, final states); B and C are (rows, groups, N)."""
    rows, ch = u.shape
    g, n = B.shape[1], A.shape[1]
    d = delta if delta_bias is None else delta + delta_bias
    if plus:
        d = softplus(d)
    y, finals = [None] * rows, []
    for s, (lo, hi) in enumerate(bounds(offsets, rows)):
        h = initial[s] if initial is not None else u.new_zeros(ch, n)
        for t in range(lo, hi):
            b = B[t].repeat_interleave(ch // g, 0)
            c = C[t].repeat_interleave(ch // g, 0)
            h = torch.exp(d[t, :, None] * A) * h + (d[t] * u[t])[:, None] * b
            y[t] = (h * c).sum(1) + (D * u[t] if D is not None else 0)
        finals.append(h)
    zero = u.new_zeros(ch)
    y = torch.stack([zero if v is None else v for v in y]) if y else u.new_zeros(0, ch)
    return y, torch.stack(finals) if finals else u.new_zeros(0, ch, n)


def norm(v, kind, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def add_norm(x, residual=None, weight=None, bias=None, scale=None, kind="rms", eps=1e-5):
    r = x if scale is None else x * scale
    if residual is not None:
        r = r + residual
    return affine(norm(r, kind, eps), weight, bias), r


def affine(v, weight, bias):
    if weight is not None:
        v = v * weight
    return v if bias is None else v + bias


def gate_norm(x, z, weight=None, bias=None, kind="rms", groups=1, gate_first=True, eps=1e-5):
    rows, ch = x.shape
    v = x * silu(z) if gate_first else x
    v = affine(norm(v.reshape(rows, groups, ch // groups), kind, eps).reshape(rows, ch), weight, bias)
    return v if gate_first else v * silu(z)


def leaves(*tensors, grad=True):
    """64-bit CPU copies."""
    return [None if t is None else t.detach().double().cpu().requires_grad_(grad) for t in tensors]


def assert_close(got, want, dtype, magnitude, steps, what=""):
    """|got - want| <= half a step of the type at `want` + steps * 2^-24 * magnitude, where `magnitude` is the sum of
    the absolute values of everything added up to make the number and `steps` the roundings on the longest way
    through them."""
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    magnitude = magnitude.detach() if isinstance(magnitude, torch.Tensor) else magnitude
    limit = HALF_STEP[dtype] * want.abs() + TINY[dtype] + steps * U32 * (1 + HALF_STEP[dtype]) * magnitude
    excess = ((got - want).abs() - limit)
    if excess.numel() and excess.max() > 0:
        i = int(excess.argmax())
        raise AssertionError(f"{what}: element {i} of {tuple(want.shape)}: {got.flatten()[i]} against {want.flatten()[i]}, "
                             f"{int((excess > 0).sum())} elements beyond the bound")


def lengths_to_offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def scan_steps(lengths):
    """Roundings on the longest way through a scan: each row multiplies by a decay exp(d A) whose relative error is
    at most (4 + 12 |d A|) 2^-24 (d itself is off by up to 8 units: its exp and log; the product with A and with
    log2 e one each; v_exp_f32 one) with |d A| < 1 in the tests, and adds one product of four factors."""
    return 16 * (max(lengths, default=1) + 4)

