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



def scan_gradient_case(device, case, dtype, seed, scan_case):
    """A case of a scan's gradients: (u, delta, A, B, C, D, bias), initial states, dy, the final states' gradient, offsets."""
    lengths, tail, ch, n, groups, plus, has_D, has_bias = case
    g, u, delta, A, B, C, D, bias = scan_case(device, *case, dtype, seed)
    more = lambda *s: torch.randn(*s, generator=g, device=device)
    init, dstate, dy = more(len(lengths), ch, n), more(len(lengths), ch, n), more(*u.shape).to(dtype)
    clean = sum(lengths)
    for t in (u, delta, B, C, dy):
        t[clean:] = float("nan")
    off = torch.tensor(lengths_to_offsets(lengths), dtype=torch.int64, device=device)
    return (u, delta, A, B, C, D, bias), init, dy, dstate, off, plus, clean


def scan_gradients(dy, u, delta, A, B, C, D, bias, off, plus, init, dstate, clean):
    """({name: gradient}, {name: the same sums of absolute values}, {name: roundings on the longest way}) of a scan, by
    the backward recurrence g = C dy + a g written out; the gradients themselves by autograd of the definition."""
    u, delta, B, C, dy = (t[:clean] for t in (u, delta, B, C, dy))
    ru, rd, rA, rB, rC, rD, rb, ri = leaves(u, delta, A, B, C, D, bias, init)
    v = (rd if rb is None else rd + rb).detach()
    d, slope = (softplus(v), torch.sigmoid(v)) if plus else (v, torch.ones_like(v))
    d.requires_grad_()            # autograd of softplus's own form above is not its derivative where v is exactly zero
    y, final = selective_scan(ru, d, rA, rB, rC, rD, None, off, False, ri)
    dy, dstate = dy.double().cpu(), dstate.double().cpu()
    named = dict(u=ru, delta=d, A=rA, B=rB, C=rC, D=rD, initial_state=ri)
    named = {k: v for k, v in named.items() if v is not None}
    refs = torch.autograd.grad((y * dy).sum() + (final * dstate).sum(), list(named.values()), allow_unused=True)
    refs = {k: torch.zeros_like(v) if r is None else r for (k, v), r in zip(named.items(), refs)}
    refs["delta"] = refs["delta"] * slope
    if rb is not None:
        refs["delta_bias"] = refs["delta"].sum(0)
    with torch.no_grad():
        ch, n, per = u.shape[1], A.shape[1], u.shape[1] // B.shape[1]
        wide = lambda m, t: m[t].abs().repeat_interleave(per, 0)
        narrow = lambda m: m.reshape(-1, per, n).sum(1)
        ua, ya, decay = ru.abs(), dy.abs(), lambda t: torch.exp(d[t, :, None] * rA)
        s = {k: torch.zeros_like(t) for k, t in named.items()}
        dd = torch.zeros_like(ru)
        for q, (lo, hi) in enumerate(zip(off[:-1], off[1:])):
            hs = [ri[q].abs()]
            for t in range(lo, hi):
                hs.append(decay(t) * hs[-1] + (d[t].abs() * ua[t])[:, None] * wide(rB, t))
            carry = dstate[q].abs()
            for t in range(hi - 1, lo - 1, -1):
                g = carry + ya[t, :, None] * wide(rC, t)
                s["C"][t], s["B"][t] = narrow(ya[t, :, None] * hs[t - lo + 1]), narrow(g * (d[t].abs() * ua[t])[:, None])
                carry = g * decay(t)
                gB, w = (g * wide(rB, t)).sum(1), carry * hs[t - lo]
                s["u"][t] = d[t].abs() * gB + (0 if rD is None else rD.abs() * ya[t])
                dd[t] = ua[t] * gB + (w * rA.abs()).sum(1)
                s["A"] += w * d[t, :, None].abs()
            s["initial_state"][q] = carry
        s["delta"] = dd * slope
        if rD is not None:
            s["D"] = (ua * ya).sum(0)
        if rb is not None:
            s["delta_bias"] = s["delta"].sum(0)
    # a state, and the gradient of one, each come through at most the longest sequence's decays; then the sum over the
    # states or the channels, the slope's functions (8), products; and the sum over rows
    longest = max((hi - lo for lo, hi in zip(off[:-1], off[1:])), default=0)
    way = 2 * scan_steps([longest])
    extra = dict(u=n + 8, delta=n + 16, A=clean + 8, B=ch + 8, C=ch + 8, D=clean + 4, delta_bias=clean + n + 16, initial_state=8)
    return refs, s, {k: way + extra[k] for k in refs}
