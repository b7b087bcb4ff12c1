"""Operators over packed rows (speech_to_text_amd/sequence.py) against 64-bit definitions: values and gradients of
every type, ragged and empty sequences, odd widths and strides, carried states, single tokens, captured graphs."""
import numpy as np
import pytest
import torch

from tests import sequence_ref as R

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def gen(gpu, seed):
    g = torch.Generator(device=gpu)
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=g.device) * scale).to(dtype)


def rand(g, *shape, lo=0.0, hi=1.0):
    return torch.rand(*shape, generator=g, device=g.device) * (hi - lo) + lo


def device_offsets(lengths, gpu):
    return torch.tensor(R.lengths_to_offsets(lengths), dtype=torch.int64, device=gpu)


# ---- causal convolution --------------------------------------------------------------------------------------
CONV = [  # lengths, rows behind them, channels, width
    ([1], 0, 1, 1), ([1], 0, 8, 4), ([3, 0, 1, 2, 70], 5, 65, 4), ([0, 0, 40], 0, 130, 3), ([2, 2, 2, 2], 3, 7, 5),
    ([150], 0, 520, 2), ([33, 64, 31], 1, 24, 8), ([130, 1, 7], 64, 9, 6), ([17, 5], 0, 16, 7),
]


def conv_case(gpu, lengths, tail, ch, width, dtype, initial, seed):
    g = gen(gpu, seed)
    rows = sum(lengths) + tail
    x = randn(g, rows, ch, dtype=dtype)
    w, b = randn(g, ch, width, scale=0.5), randn(g, ch, scale=0.3)
    init = randn(g, len(lengths), width - 1, ch, dtype=dtype) if initial else None
    return g, x, w, b, init


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(CONV)))
def test_causal_conv(gpu, case, dtype):
    import speech_to_text_amd as S

    lengths, tail, ch, width = CONV[case]
    act, initial = case % 2 == 0, case % 3 != 0
    g, x, w, b, init = conv_case(gpu, lengths, tail, ch, width, dtype, initial, case)
    if case == 1:
        b = None
    off = device_offsets(lengths, gpu)
    dy = randn(g, *x.shape, dtype=dtype)
    dstate = randn(g, len(lengths), width - 1, ch, dtype=dtype) if case % 2 else None
    clean = sum(lengths)
    if tail:                                    # what lies behind the sequences is never looked at
        x[clean:], dy[clean:] = float("nan"), float("inf")
    y, state = S.causal_conv(x, w, b, off, activation="silu" if act else None, initial_state=init, return_state=True)
    grads = S.causal_conv_backward(dy, x, w, b, off, activation="silu" if act else None, initial_state=init, dstate=dstate)

    rx, rw, rb, ri = R.leaves(x[:clean], w, b, init)
    want, want_state = R.causal_conv(rx, rw, rb, off.tolist(), act, ri)
    mx, mw, mb, mi = R.leaves(x[:clean].abs(), w.abs(), None if b is None else b.abs(), None if init is None else init.abs(), grad=False)
    size, _ = R.causal_conv(mx, mw, mb, off.tolist(), False, mi)          # sum |w| |x| + |b|
    # K products and sums, then x sigmoid(x), whose slope is below 1.1, with six roundings
    R.assert_close(y[:clean], want, dtype, size, 1.1 * (width + 1) + 6, "y")
    assert (y[clean:] == 0).all()
    assert torch.equal(state.double().cpu(), want_state.detach())         # copies of rows

    loss = (want * dy[:clean].double().cpu()).sum()
    if dstate is not None:
        loss = loss + (want_state * dstate.double().cpu()).sum()
    wrt = [t for t in (rx, rw, rb, ri) if t is not None]
    got = [t for t in (grads.x[:clean], grads.weight, grads.bias, grads.initial_state) if t is not None]
    kinds = [dtype, F32, F32, dtype]
    refs = torch.autograd.grad(loss, wrt, allow_unused=True)
    # |dp| <= 1.1 |dy|, formed with its slope in 10 + K roundings (the slope's own error from p's: another 0.5 |p|);
    # dx adds K of them, dweight and dbias all rows
    dp = 1.1 * dy[:clean].double().cpu().abs() * (1 + size)
    for name, gv, ref, kind in zip([n for n, t in zip(["x", "weight", "bias", "initial"], (rx, rw, rb, ri)) if t is not None],
                                   got, refs, kinds if b is not None else [dtype, F32, dtype]):
        ref = torch.zeros_like(gv.double().cpu()) if ref is None else ref
        biggest = float(dp.max()) if dp.numel() else 0.0
        extra = 0.0 if dstate is None else float(dstate.double().abs().max()) if dstate.numel() else 0.0
        if name in ("x", "initial"):
            mag = width * biggest * float(w.abs().max()) + extra
            R.assert_close(gv, ref, kind, mag, 2 * width + 14, name)
        else:
            both = torch.cat([rx.detach().abs().flatten(), torch.zeros(1) if ri is None else ri.detach().abs().flatten(), torch.ones(1)])
            mag = dp.sum(0).max() * float(both.max()) if dp.numel() else 0.0
            R.assert_close(gv, ref, kind, mag, clean + width + 14, name)
    assert (grads.x[clean:] == 0).all()


def test_causal_conv_of_column_ranges_and_out(gpu):
    """Inputs and outputs that are odd column ranges of wider matrices; rows outside are left alone in `out`."""
    import speech_to_text_amd as S

    g = gen(gpu, 3)
    wide = randn(g, 41, 203, dtype=BF16)
    x = wide[:, 5:102]
    w = randn(g, 97, 4)
    off = torch.tensor([2, 20, 37], dtype=torch.int64, device=gpu)
    base = torch.full((41, 300), 7.0, dtype=BF16, device=gpu)
    out = base[:, 101:198]
    res = S.causal_conv(x, w, None, off, out=out)
    assert res is out
    want = S.causal_conv(x.contiguous(), w, None, off)
    assert torch.equal(out[2:37], want[2:37])
    assert (out[:2] == 7).all() and (out[37:] == 7).all() and (want[:2] == 0).all() and (want[37:] == 0).all()
    assert (base[:, :101] == 7).all() and (base[:, 198:] == 7).all()
    # a column range of the same matrix beside the input may take the result, the input's own may not
    both = wide.clone()
    S.causal_conv(both[:, 5:102], w, None, off, out=both[:, 102:199])
    assert torch.equal(both[2:37, 102:199], want[2:37]) and torch.equal(both[:, :102], wide[:, :102])
    with pytest.raises(S.ParameterError):
        S.causal_conv(both[:, 5:102], w, None, off, out=both[:, 100:197])
    # rows of stride zero (one row, expanded) and host offsets
    e = x[3:4].expand(41, 97)
    assert torch.equal(S.causal_conv(e, w, None, [2, 20, 37]), S.causal_conv(e.contiguous(), w, None, off))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", [1, 2, 4, 8])
def test_causal_conv_carried_on(gpu, width, dtype):
    """A sequence in pieces, the last ones token by token, is the sequence in one."""
    import speech_to_text_amd as S

    g = gen(gpu, width)
    x, w, b = randn(g, 40, 21, dtype=dtype), randn(g, 21, width), randn(g, 21)
    whole, last = S.causal_conv(x, w, b, activation="silu", return_state=True)
    state, parts = None, []
    for lo, hi in [(0, 1), (1, 3), (3, 20), (20, 21), (21, 30)]:
        y, state = S.causal_conv(x[lo:hi], w, b, [0, hi - lo], activation="silu", initial_state=state, return_state=True)
        parts.append(y)
    for t in range(30, 40):
        parts.append(S.causal_conv_step(x[t:t + 1], state, w, b, activation="silu"))
    assert torch.equal(torch.cat(parts), whole) and torch.equal(state, last)


@pytest.mark.parametrize("dtype", TYPES)
def test_steps_with_slots(gpu, dtype):
    """Slots in any order, a slot named several times, slots outside the pool, a second pool for the results."""
    import speech_to_text_amd as S

    g = gen(gpu, 11)
    ch, n, width, pool = 37, 11, 4, 9
    slots = torch.tensor([4, 0, 4, -1, 8, 9, 4, 2, 0], dtype=torch.int32, device=gpu)
    m = len(slots)
    x, w, b = randn(g, m, ch, dtype=dtype), randn(g, ch, width), randn(g, ch)
    conv0 = randn(g, pool, width - 1, ch, dtype=dtype)
    u, delta = randn(g, m, ch, dtype=dtype), rand(g, m, ch, hi=0.5).to(dtype)
    A, B, C, D = -rand(g, ch, n, lo=0.1, hi=1.0), randn(g, m, n, dtype=dtype), randn(g, m, n, dtype=dtype), randn(g, ch)
    scan0 = randn(g, pool, ch, n)
    for fresh in (False, True):
        conv, scan = conv0.clone(), scan0.clone()
        nc, ns = (torch.full_like(conv, 5), torch.full_like(scan, 5)) if fresh else (None, None)
        y = S.causal_conv_step(x, conv, w, b, slots=slots, new_state=nc)
        v = S.selective_scan_step(u, delta, A, B, C, scan, D, slots=slots, new_state=ns)
        if fresh:
            assert torch.equal(conv, conv0) and torch.equal(scan, scan0)
            conv, scan = nc, ns
        for slot in range(pool):
            rows = [i for i in range(m) if int(slots[i]) == slot]
            if not rows:
                keep = (torch.full_like(conv0, 5), torch.full_like(scan0, 5)) if fresh else (conv0, scan0)
                assert torch.equal(conv[slot], keep[0][slot]) and torch.equal(scan[slot], keep[1][slot])
                continue
            c1, s1 = conv0[slot:slot + 1].clone(), scan0[slot:slot + 1].clone()
            for i in rows:                                 # the same tokens one call each
                assert torch.equal(S.causal_conv_step(x[i:i + 1], c1, w, b)[0], y[i])
                assert torch.equal(S.selective_scan_step(u[i:i + 1], delta[i:i + 1], A, B[i:i + 1], C[i:i + 1], s1, D)[0], v[i])
            assert torch.equal(c1[0], conv[slot]) and torch.equal(s1[0], scan[slot])
        for i in (3, 5):
            assert (y[i] == 0).all() and (v[i] == 0).all()


def test_step_with_many_entries(gpu):
    """More entries than a wavefront looks through at once, one repeated slot far apart."""
    import speech_to_text_amd as S

    g = gen(gpu, 12)
    m, ch = 700, 10
    slots = torch.randperm(m, generator=g, device=gpu).to(torch.int32)
    slots[690] = slots[3]
    x, w, state = randn(g, m, ch), randn(g, ch, 3), randn(g, m, 2, ch)
    s0 = state.clone()
    y = S.causal_conv_step(x, state, w, slots=slots)
    a, b = int(slots[3]), int(slots[100])
    line = torch.cat([s0[a], x[3:4], x[690:691]])
    assert torch.equal(state[a], line[2:])
    for row, lo in ((3, 0), (690, 1)):
        want = (line[lo:lo + 3].double() * w.t().double()).sum(0).cpu()
        R.assert_close(y[row], want, F32, (line[lo:lo + 3].double().abs() * w.t().double().abs()).sum(0).cpu(), 4, "y")
    assert torch.equal(state[b], torch.cat([s0[b][1:], x[100:101]]))


# ---- selective scan ---------------------------------------------------------------------------------------------
SCAN = [  # lengths, rows behind them, channels, states, groups, softplus, D, bias
    ([1], 0, 1, 1, 1, True, True, True), ([2, 0, 1, 90], 3, 70, 16, 1, True, True, True),
    ([64], 0, 64, 4, 1, False, False, False), ([65], 0, 66, 13, 2, True, False, True),
    ([0, 31, 33, 0, 64, 1], 40, 48, 8, 3, False, True, True), ([300], 0, 130, 16, 1, True, True, False),
    ([5, 200], 0, 12, 64, 1, True, True, True), ([97, 98], 9, 260, 32, 2, True, True, True),
    ([40] * 5, 0, 300, 2, 1, False, True, False), ([33], 0, 9, 16, 9, True, False, False),
]


def scan_case(gpu, lengths, tail, ch, n, groups, plus, has_D, has_bias, dtype, seed):
    g = gen(gpu, 100 + seed)
    rows = sum(lengths) + tail
    u = randn(g, rows, ch, dtype=dtype)
    if plus:
        delta, bias = randn(g, rows, ch, dtype=dtype), randn(g, ch, scale=0.5) - 2 if has_bias else None
        if not has_bias:
            delta = (delta.float() - 2).to(dtype)
    else:
        delta, bias = rand(g, rows, ch, hi=0.2).to(dtype), rand(g, ch, hi=0.1) if has_bias else None
    A = -rand(g, ch, n, lo=0.05, hi=0.5 if plus else 2.0)
    B, C = randn(g, rows, groups, n, dtype=dtype), randn(g, rows, groups, n, dtype=dtype)
    D = randn(g, ch) if has_D else None
    return g, u, delta, A, B, C, D, bias


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(SCAN)))
def test_selective_scan(gpu, case, dtype):
    import speech_to_text_amd as S

    lengths, tail, ch, n, groups, plus, has_D, has_bias = SCAN[case]
    g, u, delta, A, B, C, D, bias = scan_case(gpu, *SCAN[case], dtype, case)
    init = randn(g, len(lengths), ch, n) if case % 2 else None
    dstate = randn(g, len(lengths), ch, n) if case % 3 == 1 else None
    dy = randn(g, *u.shape, dtype=dtype)
    off, clean = device_offsets(lengths, gpu), sum(lengths)
    if tail:
        for t in (u, delta, B, C, dy):
            t[clean:] = float("nan")
    y, final = S.selective_scan(u, delta, A, B, C, D, bias, off, softplus=plus, initial_state=init, return_state=True)
    grads = S.selective_scan_backward(dy, u, delta, A, B, C, D, bias, off, softplus=plus, initial_state=init, dstate=dstate)

    cut = [t[:clean] for t in (u, delta, B, C)]
    ru, rd, rA, rB, rC, rD, rb, ri = R.leaves(cut[0], cut[1], A, cut[2], cut[3], D, bias, init)
    want, want_final = R.selective_scan(ru, rd, rA, rB, rC, rD, rb, off.tolist(), plus, ri)
    # the same with every term positive: what the sums add up in magnitude (the decays are positive anyway)
    step = rd.detach() if rb is None else rd.detach() + rb.detach()
    step = R.softplus(step) if plus else step.abs()
    pos = [ru.abs(), step, rA, rB.abs(), rC.abs(), rD.abs() if rD is not None else None, ri.abs() if ri is not None else None]
    pos = R.leaves(*pos)
    size, size_final = R.selective_scan(pos[0], pos[1], pos[2], pos[3], pos[4], pos[5], None, off.tolist(), False, pos[6])
    steps = R.scan_steps(lengths)
    R.assert_close(y[:clean], want, dtype, size, steps + n, "y")
    assert (y[clean:] == 0).all()
    R.assert_close(final, want_final, F32, size_final, steps, "state")

    loss = (want * dy[:clean].double().cpu()).sum()
    mass = (size * dy[:clean].double().cpu().abs()).sum()
    if dstate is not None:
        loss = loss + (want_final * dstate.double().cpu()).sum()
        mass = mass + (size_final * dstate.double().cpu().abs()).sum()
    names = ["u", "delta", "A", "B", "C", "D", "delta_bias", "initial_state"]
    leaf = dict(zip(names, [ru, rd, rA, rB, rC, rD, rb, ri]))
    pleaf = dict(u=pos[0], delta=pos[1], A=pos[2], B=pos[3], C=pos[4], D=pos[5], initial_state=pos[6])
    wrt = [k for k in names if leaf[k] is not None]
    refs = dict(zip(wrt, torch.autograd.grad(loss, [leaf[k] for k in wrt], allow_unused=True)))
    pw = [k for k in wrt if k != "delta_bias"]
    mags = dict(zip(pw, torch.autograd.grad(mass, [pleaf[k] for k in pw], allow_unused=True)))
    # d(loss)/d(step) is a difference: its positive part comes through B u, its negative one through A; the sum of both
    # magnitudes is at most the gradient of the positive scan plus twice its A part, |A| h-terms: bound by |A dA| per step
    flow = (mags["A"].abs() * rA.detach().abs()).sum() / max(float(step.min()), 1e-3) if mags["A"] is not None else 0
    if clean:
        mags["delta"] = mags["delta"].abs() + flow
        mags["delta_bias"] = mags["delta"].sum(0)
    for k in wrt:
        gv = getattr(grads, k)
        ref = refs[k] if refs[k] is not None else torch.zeros_like(leaf[k])
        mag = mags.get(k)
        mag = torch.zeros_like(ref) if mag is None else mag.abs()
        if k in ("u", "delta", "B", "C"):
            assert (gv[clean:] == 0).all(), k
            gv = gv[:clean]
        R.assert_close(gv, ref, F32 if k in ("A", "D", "delta_bias", "initial_state") else dtype, mag,
                       2 * steps + n + ch + (clean if k in ("A", "D", "delta_bias") else 0), k)


@pytest.mark.parametrize("dtype", TYPES)
def test_scan_carried_on(gpu, dtype):
    """Prompt in pieces, then tokens: the states handed on give the whole sequence's rows."""
    import speech_to_text_amd as S

    g, u, delta, A, B, C, D, bias = scan_case(gpu, [220], 0, 50, 16, 2, True, True, True, dtype, 50)
    whole, last = S.selective_scan(u, delta, A, B, C, D, bias, softplus=True, return_state=True)
    state, parts = None, []
    for lo, hi in [(0, 1), (1, 70), (70, 210)]:
        y, state = S.selective_scan(u[lo:hi], delta[lo:hi], A, B[lo:hi], C[lo:hi], D, bias, [0, hi - lo], softplus=True,
                                    initial_state=state, return_state=True)
        parts.append(y)
    for t in range(210, 220):
        parts.append(S.selective_scan_step(u[t:t + 1], delta[t:t + 1], A, B[t:t + 1], C[t:t + 1], state, D, bias, softplus=True))
    got = torch.cat(parts)
    ru, rd, rA, rB, rC, rD, rb = R.leaves(u, delta, A, B, C, D, bias, grad=False)
    want, final = R.selective_scan(ru, rd, rA, rB, rC, rD, rb, None, True)
    size, size_final = R.selective_scan(ru.abs(), R.softplus(rd + rb), rA, rB.abs(), rC.abs(), rD.abs())
    for v, s, name in ((whole, last, "whole"), (got, state, "pieces")):
        R.assert_close(v, want, dtype, size, R.scan_steps([220]) + 16, name)
        R.assert_close(s, final, F32, size_final, R.scan_steps([220]), name)


def test_scan_reads_column_ranges(gpu):
    """u, delta, B and C as column ranges of one projection's output, as a block has them."""
    import speech_to_text_amd as S

    g = gen(gpu, 60)
    ch, n = 33, 5
    p = randn(g, 90, 2 * ch + 2 * n + 1, dtype=BF16)
    u, delta, B, C = p[:, 1:1 + ch], p[:, 1 + ch:1 + 2 * ch], p[:, 1 + 2 * ch:1 + 2 * ch + n], p[:, 1 + 2 * ch + n:]
    A = -rand(g, ch, n, lo=0.1, hi=1.0)
    args = (u, delta, A, B, C)
    plain = [t.contiguous() for t in args]
    off = [0, 40, 41, 88]
    assert torch.equal(S.selective_scan(*args, None, None, off, softplus=True),
                       S.selective_scan(*plain, None, None, off, softplus=True))
    dy = randn(g, 90, ch + 4, dtype=BF16)[:, 3:3 + ch]
    for a, b in zip(S.selective_scan_backward(dy, *args, None, None, off, softplus=True),
                    S.selective_scan_backward(dy.contiguous(), *plain, None, None, off, softplus=True)):
        assert (a is None and b is None) or torch.equal(a, b)
    out = torch.full((90, ch), 3.0, dtype=BF16, device=gpu)
    S.selective_scan(*args, None, None, off, softplus=True, out=out)
    assert (out[88:] == 3).all() and (out[:88] != 3).any()


def test_scan_extreme_steps(gpu):
    """Steps of zero leave the state alone, huge ones forget it; softplus far out on both sides."""
    import speech_to_text_amd as S

    ch, n, rows = 4, 3, 100
    u = torch.ones(rows, ch, device=gpu)
    A = -torch.ones(ch, n, device=gpu)
    B = C = torch.ones(rows, n, device=gpu)
    init = torch.full((1, ch, n), 2.0, device=gpu)
    zero = torch.zeros(rows, ch, device=gpu)
    y, s = S.selective_scan(u, zero, A, B, C, initial_state=init, return_state=True)
    assert (y == 6).all() and (s == 2).all()
    y = S.selective_scan(u, torch.full_like(zero, 1e4), A, B, C, initial_state=init)
    assert torch.equal(y, torch.full_like(y, 3e4))                        # exp(-1e4) = 0; d u B = 1e4 each
    # softplus: x for large x, exp(x) for very negative ones; nothing overflows in between
    for x in (-100.0, -80.0, -20.0, -5.0, 0.0, 5.0, 30.0, 90.0, 1000.0):
        d = S.selective_scan(u[:1], torch.full((1, ch), x, device=gpu), torch.zeros_like(A), B[:1], C[:1], softplus=True) / n
        want = float(R.softplus(torch.tensor(x, dtype=torch.float64)))
        # exp and log of up to one unit each, the sums two, the division by n and the three additions of y two
        assert abs(float(d[0, 0]) - want) <= 6 * 2.0 ** -24 * want + 2.0 ** -126, x


def test_infinite_rows_stay_in_their_sequence(gpu):
    """An infinite B, a NaN in u: the rows before them, and the other sequences with their gradients, do not see it."""
    import speech_to_text_amd as S

    g = gen(gpu, 63)
    rows, ch, n = 90, 20, 16
    off = [0, 38, 39, 83]
    u, delta, A = rand(g, rows, ch, lo=0.5, hi=1.0), rand(g, rows, ch, lo=0.1, hi=0.2), -rand(g, ch, n, lo=0.1)
    B, C, dy = randn(g, rows, n), randn(g, rows, n), randn(g, rows, ch)
    want, state = S.selective_scan(u, delta, A, B, C, None, None, off, return_state=True)
    grads = S.selective_scan_backward(dy, u, delta, A, B, C, None, None, off)
    B2 = B.clone()
    B2[37] = float("inf")                                   # the last row of the first sequence
    y, s2 = S.selective_scan(u, delta, A, B2, C, None, None, off, return_state=True)
    assert torch.equal(y[:37], want[:37]) and torch.equal(y[38:], want[38:])
    assert torch.equal(s2[1:], state[1:]) and (s2[0] == float("inf")).all()
    u2 = u.clone()
    u2[38] = float("nan")                                   # a sequence of one row
    y, s2 = S.selective_scan(u2, delta, A, B2, C, None, None, off, return_state=True)
    assert torch.equal(y[:37], want[:37]) and torch.equal(y[39:], want[39:]) and torch.equal(s2[2], state[2])
    g2 = S.selective_scan_backward(dy, u2, delta, A, B2, C, None, None, off)
    for a, b in ((g2.u, grads.u), (g2.delta, grads.delta), (g2.B, grads.B), (g2.C, grads.C)):
        assert torch.equal(a[39:], b[39:])


@pytest.mark.parametrize("batch,pool", [(65, 40), (300, 500), (700, 90), (2050, 2000)])
def test_long_lists_of_slots(gpu, batch, pool):
    """Entries that name one slot, anywhere in a list of any length, give what one call per occurrence gives."""
    import speech_to_text_amd as S

    g = gen(gpu, batch)
    ch, n, width = 70, 9, 3
    slots = torch.randint(-3, pool + 3, (batch,), generator=torch.Generator().manual_seed(batch))
    seen, turn = {}, []
    for s in slots.tolist():
        seen[s] = seen.get(s, -1) + 1
        turn.append(seen[s])
    turn = torch.tensor(turn)
    u, delta = randn(g, batch, ch, dtype=BF16), randn(g, batch, ch, dtype=BF16)
    b, c = randn(g, batch, n, dtype=BF16), randn(g, batch, n, dtype=BF16)
    A, w = -rand(g, ch, n, lo=0.1, hi=2.0), randn(g, ch, width)
    h0, x0 = randn(g, pool, ch, n), randn(g, pool, width - 1, ch, dtype=BF16)
    h, line = h0.clone(), x0.clone()
    dev = slots.to(gpu, torch.int32)
    y = S.selective_scan_step(u, delta, A, b, c, h, softplus=True, slots=dev)
    z = S.causal_conv_step(u, line, w, slots=dev)
    h1, line1, y1, z1 = h0.clone(), x0.clone(), torch.empty_like(y), torch.empty_like(z)
    for k in range(int(turn.max()) + 1):
        i = (turn == k).nonzero().flatten().to(gpu)
        part = [t[i] for t in (u, delta, b, c)]
        y1[i] = S.selective_scan_step(part[0], part[1], A, part[2], part[3], h1, softplus=True, slots=dev[i])
        z1[i] = S.causal_conv_step(part[0], line1, w, slots=dev[i])
    assert torch.equal(y, y1) and torch.equal(h, h1) and torch.equal(z, z1) and torch.equal(line, line1)
    outside = (slots < 0) | (slots >= pool)
    assert outside.any() and (y[outside.to(gpu)] == 0).all() and (z[outside.to(gpu)] == 0).all()


# ---- norms ---------------------------------------------------------------------------------------------------------
NORMS = [(1, 1), (3, 7), (9, 64), (5, 513), (2, 1000), (70, 96), (4, 2049), (3, 4100), (2, 9001), (1, 20000), (300, 40),
         (6, 1500), (77, 200), (3, 7000),
         # rows enough that a workgroup of the gradient kernels walks over several, for each number of threads per row
         (20000, 24), (9000, 130), (4500, 300), (2500, 1100), (2300, 600),
         # rows too wide for the registers: two groups, one, the widest
         (450, 16390), (260, 8193), (2, 32768)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(NORMS)))
def test_add_norm(gpu, case, dtype):
    import speech_to_text_amd as S

    rows, ch = NORMS[case]
    g = gen(gpu, 200 + case)
    kind = "layer" if case % 2 else "rms"
    rt = F32 if case % 3 == 0 else dtype
    x, res = randn(g, rows, ch, dtype=dtype), randn(g, rows, ch, dtype=rt, scale=2.0) if case % 4 != 3 else None
    w, b = 1 + randn(g, ch, scale=0.2), randn(g, ch) if case % 2 else None
    scale = rand(g, ch, lo=0.2, hi=1.5) if case % 3 == 1 else 0.75 if case % 3 == 2 else None
    kw = dict(scale=scale, norm=kind, eps=1e-5)
    y, r = S.add_norm(x, res, w, b, residual_dtype=rt, **kw)
    assert r.dtype == rt and y.dtype == dtype
    rx, rr, rw, rb = R.leaves(x, res, w, b)
    rs = scale.double().cpu().requires_grad_() if isinstance(scale, torch.Tensor) else scale
    want, want_r = R.add_norm(rx, rr, rw, rb, rs, kind, 1e-5)
    sum_size = rx.abs() * (1 if rs is None else abs(rs) if not isinstance(rs, torch.Tensor) else rs.abs()) + (rr.abs() if rr is not None else 0)
    R.assert_close(r, want_r, rt, sum_size, 2, "r")
    # a sum over the row is off by at most (its serial part, ch / 64 + 8 halvings) units of its magnitude; the norm divides
    # by the deviation, so the elements' own errors appear relative to it
    chain = ch / 64 + 24
    dev = (want_r if kind == "rms" else want_r - want_r.mean(-1, keepdim=True)).pow(2).mean(-1, keepdim=True).add(1e-5).sqrt()
    size = (sum_size + want_r.abs().mean(-1, keepdim=True)) / dev * rw.abs() * 2 + (rb.abs() if rb is not None else 0)
    R.assert_close(y, want, dtype, size, chain, "y")

    dy, dr = randn(g, rows, ch, dtype=dtype), randn(g, rows, ch, dtype=rt)
    for use in ((dy, dr), (dy, None), (None, dr)):
        got = S.add_norm_backward(use[0], use[1], r, w, b, x=x, dtype=dtype, **kw)
        stored = r.double().cpu().requires_grad_()                        # the backward pass sees the stored sum
        yy = R.affine(R.norm(stored, kind, 1e-5), rw, rb)
        zero = torch.zeros(rows, ch, dtype=torch.float64)
        dyd, drd = (zero if t is None else t.double().cpu() for t in use)
        wrt = [stored, rw] + ([rb] if rb is not None else [])
        gr = torch.autograd.grad((yy * dyd).sum(), wrt)
        total = gr[0] + drd
        n = R.norm(stored.detach(), kind, 1e-5).abs() + 2
        wd = rw.abs() * dyd.abs()
        # dn - mean(dn) - n mean(dn n), over the deviation
        size = (wd + wd.mean(-1, keepdim=True) + n * (wd * n).mean(-1, keepdim=True)) / dev.detach() * (1 + stored.abs() / dev) + drd.abs()
        R.assert_close(got.residual, total, rt, size, 2 * chain, "residual")
        sc = 1 if rs is None else rs
        R.assert_close(got.x, total * sc, dtype, size * (sc.abs() if isinstance(sc, torch.Tensor) else sc), 2 * chain + 1, "x")
        bigrow = (1 + stored.abs() / dev).detach()
        R.assert_close(got.weight, gr[1], F32, (dyd.abs() * n * bigrow).sum(0), rows + 2 * chain, "weight")
        if rb is not None:
            R.assert_close(got.bias, gr[2], F32, dyd.abs().sum(0), rows + 4, "bias")
        if isinstance(rs, torch.Tensor):
            R.assert_close(got.scale, (total * rx).sum(0), F32, (size * rx.abs()).sum(0), rows + 2 * chain, "scale")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(NORMS)))
def test_gate_norm(gpu, case, dtype):
    import speech_to_text_amd as S

    rows, ch = NORMS[case]
    groups = 2 if ch % 2 == 0 and case % 4 else 1
    g = gen(gpu, 300 + case)
    kind, first = "layer" if case % 2 else "rms", case % 3 != 1
    x, z, dy = (randn(g, rows, ch, dtype=dtype) for _ in range(3))
    w, b = 1 + randn(g, ch, scale=0.2), randn(g, ch) if case % 2 else None
    kw = dict(norm=kind, groups=groups, gate_first=first, eps=1e-5)
    y = S.gate_norm(x, z, w, b, **kw)
    rx, rz, rw, rb = R.leaves(x, z, w, b)
    want = R.gate_norm(rx, rz, rw, rb, kind, groups, first, 1e-5)
    gate = R.silu(rz).detach()
    v = (rx * gate if first else rx).detach()
    cut = lambda t: t.reshape(rows, groups, ch // groups)
    mean = cut(v).mean(-1, keepdim=True) if kind == "layer" else 0
    dev = (cut(v) - mean).pow(2).mean(-1, keepdim=True).add(1e-5).sqrt()
    wide = lambda t: t.expand(rows, groups, ch // groups).reshape(rows, ch)
    dev, avg = wide(dev), wide(cut(v).abs().mean(-1, keepdim=True))
    chain = ch / groups / 64 + 34
    after = torch.ones_like(gate) if first else gate.abs() + 1e-30
    size = ((v.abs() + avg) / dev * rw.abs() * 2 + (rb.abs() if rb is not None else 0)) * after
    R.assert_close(y, want, dtype, size, chain, "y")

    got = S.gate_norm_backward(dy, x, z, w, b, **kw)
    dyd = dy.double().cpu()
    wrt = [t for t in (rx, rz, rw, rb) if t is not None]
    refs = torch.autograd.grad((want * dyd).sum(), wrt)
    n = (v.abs() + avg) / dev
    body = dyd.abs() * after
    wd = body * rw.detach().abs()
    back = (wd + wide(cut(wd).mean(-1, keepdim=True)) + n * wide(cut(wd * n).mean(-1, keepdim=True))) / dev * (1 + n)
    via_gate = gate.abs() + 1.1 if first else 1.0
    R.assert_close(got.x, refs[0], dtype, back * via_gate, 2 * chain, "x")
    inner = back * rx.detach().abs() if first else dyd.abs() * (n * rw.detach().abs() + (rb.detach().abs() if rb is not None else 0))
    R.assert_close(got.z, refs[1], dtype, inner * 1.1 * (1 + rz.detach().abs()), 2 * chain, "z")
    R.assert_close(got.weight, refs[2], F32, (body * n * (1 + n)).sum(0), rows + 2 * chain, "weight")
    if rb is not None:
        R.assert_close(got.bias, refs[3], F32, body.sum(0), rows + 12, "bias")


def test_gradients_of_more_wide_rows_than_workgroups(gpu):
    """Every row's gradient is the one it has in a batch of a few rows; the sum over rows holds against 64 bits."""
    import speech_to_text_amd as S

    rows, ch = 65536 + 70, 8193
    g = torch.Generator(device=gpu).manual_seed(77)
    x, z, dy = (torch.empty(rows, ch, dtype=BF16, device=gpu).normal_(generator=g) for _ in range(3))
    w = torch.ones(ch, device=gpu)
    got = S.gate_norm_backward(dy, x, z, w)
    for part in (slice(0, 3), slice(40000, 40005), slice(65530, rows)):
        few = S.gate_norm_backward(dy[part], x[part], z[part], w)
        assert torch.equal(got.x[part], few.x) and torch.equal(got.z[part], few.z)
    want, size = (torch.zeros(ch, dtype=torch.float64, device=gpu) for _ in range(2))
    for i in range(0, rows, 4096):
        p = slice(i, i + 4096)
        n = dy[p].double() * R.norm(x[p].double() * R.silu(z[p].double()), "rms", 1e-5)
        want += n.sum(0)
        size += n.abs().sum(0)
    # each value's own error (the gate's and the norm's, as in the smaller cases), and the sum: a chain of rows / workgroups
    # (409, of five tiles in 2048) in each partial sum and of at least 16 slices over them
    R.assert_close(got.weight, want.cpu(), F32, size.cpu(), rows / 409 + 409 / 16 + 20 + 2 * (ch / 64 + 34), "weight")


def test_norms_of_special_rows(gpu):
    """A row of zeros gives the bias; equal elements under the layer norm too; strided rows and none at all."""
    import speech_to_text_amd as S

    x = torch.zeros(3, 77, device=gpu)
    b = torch.arange(77, device=gpu, dtype=F32)
    for kind in ("rms", "layer"):
        y, r = S.add_norm(x, None, None, b, norm=kind)
        assert torch.equal(y, b.expand(3, 77)) and (r == 0).all()
        assert torch.equal(S.gate_norm(x + 1, x, None, b, norm=kind), b.expand(3, 77))
        g = S.gate_norm_backward(x + 1, x, x, None, b, norm=kind)
        assert torch.isfinite(g.x).all() and torch.isfinite(g.z).all() and g.weight is None and (g.bias == 3).all()
    y, _ = S.add_norm(x + 3, None, None, b, norm="layer")
    assert torch.equal(y, b.expand(3, 77))
    g = gen(gpu, 8)
    wide = randn(g, 12, 300, dtype=F16)
    a, z = wide[:, 1:100], wide[:, 101:200]
    assert torch.equal(S.gate_norm(a, z), S.gate_norm(a.contiguous(), z.contiguous()))
    y, r = S.add_norm(a, z)
    y2, r2 = S.add_norm(a.contiguous(), z.contiguous())
    assert torch.equal(y, y2) and torch.equal(r, r2)
    out = wide.clone()
    S.gate_norm(out[:, 1:100], out[:, 101:200], out=out[:, 201:300])
    assert torch.equal(out[:, :201], wide[:, :201]) and torch.equal(out[:, 201:], S.gate_norm(a, z))
    none = torch.empty(0, 99, device=gpu)
    w = torch.ones(99, device=gpu)
    assert S.gate_norm(none, none).shape == (0, 99) and S.add_norm(none, none)[0].shape == (0, 99)
    assert (S.gate_norm_backward(none, none, none, w).weight == 0).all()
    assert (S.add_norm_backward(none, None, none, w).weight == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,ch,how", [(70, 45, "nan"), (70, 1001, "nan"), (33, 2, "nan"), (9, 2050, "nan"), (1, 45, "nan"),
                                         (70, 45, "expanded"), (5, 3, "expanded"), (41, 1, "expanded")])
def test_what_lies_behind_a_row(gpu, rows, ch, how, dtype):
    """Column ranges of a wider matrix with NaN around them, and one row expanded to many, as their contiguous copies."""
    import speech_to_text_amd as S

    g = gen(gpu, rows + ch)

    def tensor():
        if how == "expanded":
            return randn(g, 1, ch, dtype=dtype).expand(rows, ch)
        around = torch.full((rows, ch + 9), float("nan"), dtype=dtype, device=gpu)
        around[:, 3:3 + ch] = randn(g, rows, ch, dtype=dtype)
        return around[:, 3:3 + ch]

    def same(got, want):
        got, want = (t if isinstance(t, tuple) else (t,) for t in (got, want))
        for a, b in zip(got, want):
            assert (a is None and b is None) or (torch.isfinite(a).all() and torch.equal(a, b))

    x, z, dy, dr = (tensor() for _ in range(4))
    plain = [t.contiguous() for t in (x, z, dy, dr)]
    w, b, taps, scale = randn(g, ch), randn(g, ch), randn(g, ch, 4), rand(g, ch, lo=0.2, hi=1.5)
    call = lambda f: same(f(x, z, dy, dr), f(*plain))
    call(lambda x, z, dy, dr: S.causal_conv(x, taps, b, activation="silu", return_state=True))
    call(lambda x, z, dy, dr: S.causal_conv_backward(dy, x, taps, b, activation="silu"))
    for kind in ("rms", "layer"):
        call(lambda x, z, dy, dr: S.add_norm(x, z, w, b, scale=scale, norm=kind))
        call(lambda x, z, dy, dr: S.add_norm_backward(dy, dr, z, w, b, x=x, scale=scale, norm=kind))
        for first in (True, False):
            for groups in (1, ch):
                if groups == 1 or ch < 50:
                    call(lambda x, z, dy, dr: S.gate_norm(x, z, w, b, norm=kind, gate_first=first, groups=groups))
                    call(lambda x, z, dy, dr: S.gate_norm_backward(dy, x, z, w, b, norm=kind, gate_first=first, groups=groups))


# ---- every choice of tile and chunk ------------------------------------------------------------------------------------
def scan64(u, d, A, B, C, dy, off, rate):
    """Values and gradients row by row in 64 bits on the GPU; `rate` is A, or |A| for magnitudes (d u, B, C, dy then
    positive as well)."""
    rows, ch = u.shape
    n = A.shape[1]
    y, du, dd, dB, dC = (torch.zeros_like(t) for t in (u, u, d, B, C))
    dA = torch.zeros_like(A)
    for lo, hi in zip(off[:-1], off[1:]):
        hs = torch.zeros(hi - lo + 1, ch, n, dtype=torch.float64, device=u.device)
        for t in range(lo, hi):
            hs[t - lo + 1] = torch.exp(d[t, :, None] * A) * hs[t - lo] + (d[t] * u[t])[:, None] * B[t]
            y[t] = (hs[t - lo + 1] * C[t]).sum(1)
        carry = torch.zeros(ch, n, dtype=torch.float64, device=u.device)
        for t in range(hi - 1, lo - 1, -1):
            dC[t] = (hs[t - lo + 1] * dy[t, :, None]).sum(0)
            g = carry + dy[t, :, None] * C[t]
            dB[t] = (g * (d[t] * u[t])[:, None]).sum(0)
            carry = g * torch.exp(d[t, :, None] * A)
            gB, w = (g * B[t]).sum(1), carry * hs[t - lo]
            dA += w * d[t, :, None]
            dd[t], du[t] = u[t] * gB + (w * rate).sum(1), d[t] * gB
    return dict(y=y, u=du, delta=dd, A=dA, B=dB, C=dC)


@pytest.mark.parametrize("rows,ch,n", [
    (16500, 4096, 1), (8300, 4096, 2), (4200, 4096, 3), (1500, 704, 4), (900, 700, 5),     # forward 256, 128, 64 and 16 rows
    (1100, 4096, 16), (2100, 1024, 16), (1600, 1024, 16), (1200, 640, 16),                 # gradient 64, 32 and 16; forward 32
    (600, 512, 16)])                                                                       # both 8
def test_scan_of_every_chunk_length(gpu, rows, ch, n):
    import speech_to_text_amd as S

    g = gen(gpu, rows)
    cuts = [0, 37, rows // 3, rows // 3 + 1, rows - 300, rows]
    u, dy = randn(g, rows, ch, dtype=BF16), randn(g, rows, ch, dtype=BF16)
    delta = rand(g, rows, ch, lo=0.01, hi=0.1).to(BF16)
    B, C = randn(g, rows, n, dtype=BF16), randn(g, rows, n, dtype=BF16)
    A = -rand(g, ch, n, lo=0.5, hi=2.0)
    off = torch.tensor(cuts, dtype=torch.int64, device=gpu)
    y = S.selective_scan(u, delta, A, B, C, None, None, off)
    gr = S.selective_scan_backward(dy, u, delta, A, B, C, None, None, off)
    up = lambda *ts: [t.double() for t in ts]
    ud, dd, Ad, Bd, Cd, dyd = up(u, delta, A, B, C, dy)
    want = scan64(ud, dd, Ad, Bd, Cd, dyd, cuts, Ad)
    size = scan64(ud.abs(), dd, Ad, Bd.abs(), Cd.abs(), dyd.abs(), cuts, Ad.abs())
    # |d A| < 0.2 and A d > 0.005 on average 0.07: a state forgets within some hundred rows; (4 + 12 |d A|) roundings for
    # each of those, and the chunk's own sum of d
    steps = 7 * 400
    for name, got in dict(y=y, u=gr.u, delta=gr.delta, A=gr.A, B=gr.B, C=gr.C).items():
        kind = F32 if name == "A" else BF16
        extra = dict(A=rows, B=ch, C=ch).get(name, 0)
        R.assert_close(got, want[name].cpu(), kind, size[name].cpu(), steps + extra, name)


@pytest.mark.parametrize("rows", [9000, 17000, 34000, 66000, 2010, 3000])
def test_causal_conv_of_every_tile(gpu, rows):
    """Sizes at which a thread of the forward pass takes 16, 32, 64, 128 and 8 rows, of the gradient 32, 64, 128, 8 and 16."""
    import speech_to_text_amd as S

    g = gen(gpu, rows)
    ch, k = 4096, 4
    x = torch.empty(rows, ch, dtype=BF16, device=gpu).normal_(generator=g)
    dy = torch.empty(rows, ch, dtype=BF16, device=gpu).normal_(generator=g)
    w, b = randn(g, ch, k, scale=0.5), randn(g, ch, scale=0.3)
    cuts = [0, 3, 131, rows // 2, rows // 2 + 2, rows - 1000, rows]
    off = torch.tensor(cuts, dtype=torch.int64, device=gpu)
    y = S.causal_conv(x, w, b, off, activation="silu")
    gr = S.causal_conv_backward(dy, x, w, b, off, activation="silu")
    dw, db = torch.zeros(ch, k, dtype=torch.float64, device=gpu), torch.zeros(ch, dtype=torch.float64, device=gpu)
    biggest = 0.0
    for lo, hi in zip(cuts[:-1], cuts[1:]):
        line = torch.cat([torch.zeros(k - 1, ch, dtype=torch.float64, device=gpu), x[lo:hi].double()])
        p = sum(line[j:j + hi - lo] * w[:, j].double() for j in range(k)) + b.double()
        size = sum(line[j:j + hi - lo].abs() * w[:, j].double().abs() for j in range(k)) + b.double().abs()
        sg = torch.sigmoid(p)
        dp = dy[lo:hi].double() * sg * (1 + p * (1 - sg))
        dw += torch.stack([(dp * line[j:j + hi - lo]).sum(0) for j in range(k)], 1)
        db += dp.sum(0)
        biggest = max(biggest, float((dp.abs() * (1 + size)).max()))
        late = torch.cat([dp, torch.zeros(k - 1, ch, dtype=torch.float64, device=gpu)])
        dx = sum(late[k - 1 - j:k - 1 - j + hi - lo] * w[:, j].double() for j in range(k))
        reach = sum(late[k - 1 - j:k - 1 - j + hi - lo].abs() * w[:, j].double().abs() for j in range(k))
        for name, got, want, mag in (("y", y, p * sg, size), ("x", gr.x, dx, reach + dy[lo:hi].double().abs().max() * size)):
            # sigmoid without its second exponent word: |p| more roundings, |p| < 16
            limit = 2.0 ** -8 * want.abs() + 2.0 ** -126 + 40 * 2.0 ** -24 * mag
            assert ((got[lo:hi].double() - want).abs() <= limit).all(), (name, lo)
    for got, want in ((gr.weight, dw), (gr.bias, db)):
        assert (got.double() - want).abs().max() <= (rows + 40) * 2.0 ** -24 * biggest * 6


def test_scan_step_of_many_entries(gpu):
    """Enough entries that a thread takes four; some slots named again, near and far; padded rows at the end."""
    import speech_to_text_amd as S

    g = gen(gpu, 31)
    m, ch, n, pool = 1103, 1024, 16, 1200
    slots = torch.randperm(pool, generator=g, device=gpu)[:m].to(torch.int32)
    slots[1] = slots[0]
    slots[7], slots[9], slots[1000] = slots[4], slots[4], slots[4]
    slots[1098:] = -1
    u, delta = randn(g, m, ch), rand(g, m, ch, hi=0.3)
    A, B, C, D = -rand(g, ch, n, lo=0.1, hi=1.0), randn(g, m, n), randn(g, m, n), randn(g, ch)
    state = randn(g, pool, ch, n)
    want, size = state.double(), state.double().abs()
    got_state = state.clone()
    y = S.selective_scan_step(u, delta, A, B, C, got_state, D, slots=slots)
    for i, slot in enumerate(slots.tolist()):
        if slot < 0:
            assert (y[i] == 0).all()
            continue
        decay = torch.exp(delta[i].double()[:, None] * A.double())
        step = (delta[i].double() * u[i].double())[:, None]
        want[slot] = decay * want[slot] + step * B[i].double()
        size[slot] = decay * size[slot] + step.abs() * B[i].double().abs()
        wy = (want[slot] * C[i].double()).sum(1) + D.double() * u[i].double()
        ws = (size[slot] * C[i].double().abs()).sum(1) + D.double().abs() * u[i].double().abs()
        assert ((y[i].double() - wy).abs() <= (16 * 4 + n) * 2.0 ** -24 * ws).all(), i     # at most four tokens of a slot
    assert ((got_state.double() - want).abs() <= 16 * 4 * 2.0 ** -24 * size).all()


# ---- empty batches, offsets, streams, graphs --------------------------------------------------------------------------
def test_no_rows(gpu):
    import speech_to_text_amd as S

    none, w = torch.empty(0, 6, device=gpu), torch.ones(6, 3, device=gpu)
    init = torch.ones(2, 2, 6, device=gpu)
    y, s = S.causal_conv(none, w, None, [0, 0, 0], initial_state=init, return_state=True)
    assert y.shape == (0, 6) and torch.equal(s, init)
    g = S.causal_conv_backward(none, none, w, w[:, 0].contiguous(), [0, 0, 0], initial_state=init, dstate=2 * init)
    assert (g.weight == 0).all() and (g.bias == 0).all() and torch.equal(g.initial_state, 2 * init)
    A, B = -torch.ones(6, 4, device=gpu), torch.empty(0, 4, device=gpu)
    h = torch.ones(2, 6, 4, device=gpu)
    y, s = S.selective_scan(none, none, A, B, B, None, None, [0, 0, 0], initial_state=h, return_state=True)
    assert y.shape == (0, 6) and torch.equal(s, h)
    g = S.selective_scan_backward(none, none, none, A, B, B, w[:, 0].contiguous(), None, [0, 0, 0], initial_state=h, dstate=3 * h)
    assert (g.A == 0).all() and (g.D == 0).all() and torch.equal(g.initial_state, 3 * h)
    y, s = S.selective_scan(none, none, A, B, B, return_state=True)
    assert (s == 0).all() and s.shape == (1, 6, 4)
    assert S.selective_scan_step(none, none, A, B, B, h).shape == (0, 6)
    assert S.causal_conv_step(none, init, w).shape == (0, 6)
    assert S.causal_conv(none, w, None, torch.zeros(1, dtype=torch.int64, device=gpu)).shape == (0, 6)


def test_offsets_that_do_not_fit(gpu):
    """Device offsets are not seen by the host: values out of order or range address nothing outside the rows."""
    import speech_to_text_amd as S

    g = gen(gpu, 70)
    rows, ch = 100, 16
    buf = torch.full((3 * rows, ch), 9.0, device=gpu)
    x = randn(g, rows, ch)
    w, A, B = randn(g, ch, 4), -rand(g, ch, 4), randn(g, rows, 4)
    delta = rand(g, rows, ch)
    for bad in ([0, 50, 20, 100], [-5, 30, 200], [500, 900], [0, -7, 60], [2 ** 40, -2 ** 40, 3], [0, 10, 10 ** 12]):
        off = torch.tensor(bad, dtype=torch.int64, device=gpu)
        n = len(bad) - 1
        out = buf[rows:2 * rows]
        init, h0 = randn(g, n, 3, ch), randn(g, n, ch, 4)
        S.causal_conv(x, w, None, off, initial_state=init, return_state=True, out=out)
        S.causal_conv_backward(x, x, w, None, off, initial_state=init, dstate=init)
        S.selective_scan(x, delta, A, B, B, None, None, off, initial_state=h0, return_state=True, out=out)
        S.selective_scan_backward(x, x, delta, A, B, B, None, None, off, initial_state=h0, dstate=h0)
        torch.cuda.synchronize()
        assert (buf[:rows] == 9).all() and (buf[2 * rows:] == 9).all()
    # in range at the front, beyond the rows at the end: the last sequence ends with the rows
    off = torch.tensor([0, 40, 1000], dtype=torch.int64, device=gpu)
    assert torch.equal(S.causal_conv(x, w, None, off), S.causal_conv(x, w, None, [0, 40, 100]))


def block_inputs(g, rows, ch, n, dtype):
    return (randn(g, rows, ch, dtype=dtype), rand(g, rows, ch, hi=0.3).to(dtype), randn(g, rows, n, dtype=dtype),
            randn(g, rows, n, dtype=dtype), randn(g, rows, ch, dtype=dtype), randn(g, rows, ch, dtype=dtype))


def run_all(S, x, delta, B, C, z, dy, w, A, D, wn, off):
    """Every operator once, forward and backward."""
    y = S.causal_conv(x, w, D, off, activation="silu")
    v = S.selective_scan(y, delta, A, B, C, D, None, off)
    o = S.gate_norm(v, z, wn)
    n, r = S.add_norm(o, x, wn)
    ga = S.add_norm_backward(dy, None, r, wn)
    gg = S.gate_norm_backward(ga.x, v, z, wn)
    gs = S.selective_scan_backward(gg.x, y, delta, A, B, C, D, None, off)
    gc = S.causal_conv_backward(gs.u, x, w, D, off, activation="silu")
    return [n, r, *ga[1:3], *gg[1:3], *gs[1:6], *gc[:3]]


def test_captured_and_replayed(gpu):
    """Two graphs of the whole chain with different sizes, replayed in turn with new data and new offsets between eager
    calls of the same operators: every replay has the eager bits."""
    import speech_to_text_amd as S

    g = gen(gpu, 80)
    ch, n = 72, 16
    w, A, D, wn = randn(g, ch, 4), -rand(g, ch, n, lo=0.1), randn(g, ch), 1 + randn(g, ch, scale=0.1)
    graphs = []
    with torch.no_grad():
        for rows in (150, 333):
            bufs = block_inputs(g, rows, ch, n, BF16)
            off = torch.tensor([0, rows // 2, rows - 5], dtype=torch.int64, device=gpu)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                run_all(S, *bufs, w, A, D, wn, off)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs = run_all(S, *bufs, w, A, D, wn, off)
            graphs.append((rows, bufs, off, graph, outs))
        for turn in range(4):
            want = []
            for rows, bufs, off, graph, outs in graphs:
                for b, fresh in zip(bufs, block_inputs(g, rows, ch, n, BF16)):
                    b.copy_(fresh)
                off.copy_(torch.tensor([0, 3 + 20 * turn, rows - turn], dtype=torch.int64))
                want.append([t.clone() for t in run_all(S, *bufs, w, A, D, wn, off)])
            for rows, bufs, off, graph, outs in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for (rows, bufs, off, graph, outs), ws in zip(graphs, want):
                for i, (a, b) in enumerate(zip(outs, ws)):
                    assert torch.equal(a, b), (turn, rows, i)


def test_other_streams_and_repeated_calls(gpu):
    """On a side stream, and again: the same bits."""
    import speech_to_text_amd as S

    g = gen(gpu, 81)
    ch, n, rows = 200, 16, 700
    w, A, D, wn = randn(g, ch, 4), -rand(g, ch, n, lo=0.1), randn(g, ch), 1 + randn(g, ch, scale=0.1)
    bufs = block_inputs(g, rows, ch, n, F32)
    off = [0, 130, 131, 690]
    first = run_all(S, *bufs, w, A, D, wn, off)
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                results.append(run_all(S, *bufs, w, A, D, wn, off))
    torch.cuda.synchronize()
    for r in results:
        for a, b in zip(first, r):
            assert torch.equal(a, b)


# ---- autograd -----------------------------------------------------------------------------------------------------------
def test_autograd_is_the_explicit_gradient(gpu):
    import speech_to_text_amd as S

    g = gen(gpu, 90)
    rows, ch, n = 60, 20, 6
    off = [0, 25, 25, 55]
    x = randn(g, rows, ch, dtype=BF16).requires_grad_()
    w, b = randn(g, ch, 4).requires_grad_(), randn(g, ch).requires_grad_()
    init = randn(g, 3, 3, ch, dtype=BF16).requires_grad_()
    dy, ds = randn(g, rows, ch, dtype=BF16), randn(g, 3, 3, ch, dtype=BF16)
    y, s = S.causal_conv(x, w, b, off, activation="silu", initial_state=init, return_state=True)
    got = torch.autograd.grad([y, s], [x, w, b, init], [dy, ds])
    with torch.no_grad():
        want = S.causal_conv_backward(dy, x, w, b, off, activation="silu", initial_state=init, dstate=ds)
    assert all(torch.equal(a, c) for a, c in zip(got, want))

    u, delta = (randn(g, rows, ch).requires_grad_() for _ in range(2))
    A = (-rand(g, ch, n)).requires_grad_()
    B, C = (randn(g, rows, 2, n).requires_grad_() for _ in range(2))
    D, bias = randn(g, ch).requires_grad_(), randn(g, ch).requires_grad_()
    h0 = randn(g, 3, ch, n).requires_grad_()
    y, h = S.selective_scan(u, delta, A, B, C, D, bias, off, softplus=True, initial_state=h0, return_state=True)
    leaves = [u, delta, A, B, C, D, bias, h0]
    dyf, dh = randn(g, rows, ch), randn(g, 3, ch, n)
    got = torch.autograd.grad([y, h], leaves, [dyf, dh], retain_graph=True)
    with torch.no_grad():
        want = S.selective_scan_backward(dyf, *leaves[:7], off, softplus=True, initial_state=h0, dstate=dh)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    only = torch.autograd.grad(h, leaves, dh, retain_graph=True)          # the state alone
    with torch.no_grad():
        want = S.selective_scan_backward(torch.zeros_like(dyf), *leaves[:7], off, softplus=True, initial_state=h0, dstate=dh)
    assert all(torch.equal(a, c) for a, c in zip(only, want))
    ones = torch.autograd.grad(y.sum(), leaves)                           # an expanded gradient
    with torch.no_grad():
        want = S.selective_scan_backward(torch.ones_like(dyf), *leaves[:7], off, softplus=True, initial_state=h0)
    assert all(torch.equal(a, c) for a, c in zip(ones, want))

    res = randn(g, rows, ch, dtype=F32).requires_grad_()
    sc = rand(g, ch, lo=0.5).requires_grad_()
    wn, bn = randn(g, ch).requires_grad_(), randn(g, ch).requires_grad_()
    dr = randn(g, rows, ch)
    y, r = S.add_norm(x, res, wn, bn, scale=sc, norm="layer")
    got = torch.autograd.grad([y, r], [x, res, wn, bn, sc], [dy, dr])
    with torch.no_grad():
        want = S.add_norm_backward(dy, dr, r, wn, bn, x=x, scale=sc, norm="layer")
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    y, r = S.add_norm(x, None, wn)
    assert torch.equal(torch.autograd.grad(r, x, dy)[0], dy)              # the sum alone: x itself

    z = randn(g, rows, ch, dtype=BF16).requires_grad_()
    y = S.gate_norm(x, z, wn, groups=4)
    got = torch.autograd.grad(y, [x, z, wn], dy)
    with torch.no_grad():
        want = S.gate_norm_backward(dy, x, z, wn, groups=4)
    assert all(torch.equal(a, c) for a, c in zip(got, want[:3]))


def test_autograd_of_shared_and_broadcast_inputs(gpu):
    """One B for all groups by expansion, one row of x for all rows, one tensor as two inputs: gradients add up."""
    import speech_to_text_amd as S

    g = gen(gpu, 91)
    rows, ch, n = 30, 12, 4
    u = randn(g, 1, ch).requires_grad_()
    B1 = randn(g, rows, 1, n).requires_grad_()
    A = (-rand(g, ch, n)).requires_grad_()
    wide = u.expand(rows, ch)
    many = B1.expand(rows, 3, n).contiguous()
    y = S.selective_scan(wide, wide, A, many, many, softplus=True)
    dy = randn(g, rows, ch)
    gu, gB, gA = torch.autograd.grad(y, [u, B1, A], dy)
    ru, rB, rA = R.leaves(u, B1, A)
    want, _ = R.selective_scan(ru.expand(rows, ch), ru.expand(rows, ch), rA, rB.expand(rows, 3, n), rB.expand(rows, 3, n), plus=True)
    for got, ref in zip((gu, gB, gA), torch.autograd.grad((want * dy.double().cpu()).sum(), [ru, rB, rA])):
        torch.testing.assert_close(got.double().cpu(), ref, rtol=1e-4, atol=1e-4 * float(ref.abs().max()))


@pytest.mark.parametrize("op", ["conv", "scan", "add", "gate"])
def test_gradient_against_differences(gpu, op):
    """Directional differences of the operator itself.  With step e the quotient is off by the third derivative's
    e^2 / 6 and by the rounding 2^-24 |y| sqrt(n) / e of two values; e = 2^-7 balances them below 1e-3 of the norms."""
    import speech_to_text_amd as S

    g = gen(gpu, 92)
    rows, ch, n = 64, 24, 8
    off = [0, 20, 50]
    ins = {
        "conv": [randn(g, rows, ch), randn(g, ch, 4), randn(g, ch)],
        "scan": [randn(g, rows, ch), randn(g, rows, ch) - 1, -rand(g, ch, n, lo=0.2), randn(g, rows, n), randn(g, rows, n), randn(g, ch)],
        "add": [randn(g, rows, ch), randn(g, rows, ch), 1 + randn(g, ch, scale=0.1), randn(g, ch), rand(g, ch, lo=0.5)],
        "gate": [randn(g, rows, ch), randn(g, rows, ch), 1 + randn(g, ch, scale=0.1), randn(g, ch)],
    }[op]
    f = {
        "conv": lambda x, w, b: S.causal_conv(x, w, b, off, activation="silu"),
        "scan": lambda u, d, A, B, C, D: S.selective_scan(u, d, A, B, C, D, None, off, softplus=True),
        "add": lambda x, r, w, b, s: S.add_norm(x, r, w, b, scale=s, norm="layer")[0],
        "gate": lambda x, z, w, b: S.gate_norm(x, z, w, b, groups=3),
    }[op]
    dy = randn(g, rows, ch)
    e = 2.0 ** -7
    for i in range(len(ins)):
        v = randn(g, *ins[i].shape)
        leaf = [t.clone().requires_grad_(j == i) for j, t in enumerate(ins)]
        grad, = torch.autograd.grad(f(*leaf), leaf[i], dy)
        hi, lo = (f(*[t + s * e * v if j == i else t for j, t in enumerate(ins)]).double() for s in (1, -1))
        quotient = float(((hi - lo) * dy.double()).sum() / (2 * e))
        exact = float((grad.double() * v.double()).sum())
        size = float(grad.double().norm() * v.double().norm())
        assert abs(quotient - exact) <= 1e-3 * size + 1e-3, (op, i, quotient, exact, size)


# ---- together: features -> block -> tokens ---------------------------------------------------------------------------------
def test_block_over_features_and_tokens(gpu):
    """MFCC features of a ragged batch through a whole block with the offsets the feature engine returned: training
    gradients against 64 bits, and serving (prompt, then tokens) against the whole sequence."""
    import speech_to_text_amd as S
    from tests.signals import speech_like

    ys = [speech_like(m, seed=i) for i, m in enumerate([9000, 700, 16000])]
    feats = S.mfcc_batch(ys, n_fft=512, hop_length=160, n_mfcc=13, n_mels=40, return_tensor=True)
    off = np.concatenate([[0], np.cumsum([len(f) for f in feats])])
    rows = torch.cat(feats)
    rows = (rows - rows.mean(0)) / rows.std(0)
    g = gen(gpu, 95)
    d, ch, n = 24, 32, 8
    par = dict(emb=randn(g, 13, d, scale=0.3), w0=1 + randn(g, d, scale=0.1), inp=randn(g, d, 2 * ch, scale=0.2),
               conv=randn(g, ch, 4, scale=0.5), cb=randn(g, ch, scale=0.1), dt=randn(g, ch, ch, scale=0.1),
               bc=randn(g, ch, 2 * n, scale=0.2), A=-rand(g, ch, n, lo=0.2, hi=2.0), D=randn(g, ch), db=randn(g, ch) - 2,
               wn=1 + randn(g, ch, scale=0.1), out=randn(g, ch, d, scale=0.2), w1=1 + randn(g, d, scale=0.1), sc=rand(g, d, lo=0.3))

    def block(p, x, conv, scan, gate, add):
        h = x @ p["emb"]
        v, r = add(h, None, p["w0"], None)
        xz = v @ p["inp"]
        c = conv(xz[:, :ch], p["conv"], p["cb"])
        bc = c @ p["bc"]
        s = scan(c, c @ p["dt"], p["A"], bc[:, :n], bc[:, n:], p["D"], p["db"])
        o = gate(s, xz[:, ch:], p["wn"]) @ p["out"]
        return add(o, r, p["w1"], p["sc"])[0]

    ours = dict(conv=lambda x, w, b: S.causal_conv(x, w, b, off, activation="silu"),
                scan=lambda *a: S.selective_scan(*a, off, softplus=True),
                gate=lambda x, z, w: S.gate_norm(x, z, w, groups=2),
                add=lambda x, r, w, sc: S.add_norm(x, r, w, scale=sc))
    theirs = dict(conv=lambda x, w, b: R.causal_conv(x, w, b, off.tolist(), True)[0],
                  scan=lambda u, dl, A, B, C, D, db: R.selective_scan(u, dl, A, B[:, None], C[:, None], D, db, off.tolist(), True)[0],
                  gate=lambda x, z, w: R.gate_norm(x, z, w, groups=2),
                  add=lambda x, r, w, sc: R.add_norm(x, r, w, scale=sc))
    leaf = {k: v.clone().requires_grad_() for k, v in par.items()}
    ref = dict(zip(par, R.leaves(*par.values())))
    got = block(leaf, rows, **ours)
    want = block(ref, rows.double().cpu(), **theirs)
    # float32 products of at most 2 ch = 64 terms in a chain of six operators: 1e-4 of the largest value is far above
    # their roundings and far below any wrong term
    torch.testing.assert_close(got.double().cpu(), want, rtol=0, atol=1e-4 * float(want.detach().abs().max()))
    dy = randn(g, *got.shape)
    gg = torch.autograd.grad(got, list(leaf.values()), dy)
    rg = torch.autograd.grad(want, list(ref.values()), dy.double().cpu())
    for name, a, b in zip(par, gg, rg):
        torch.testing.assert_close(a.double().cpu(), b, rtol=0, atol=2e-4 * float(b.detach().abs().max()), msg=lambda m: f"{name}: {m}")

    # serving the first utterance: half of it as a prompt, the rest token by token
    f = rows[:int(off[1])]
    half = len(f) // 2
    with torch.no_grad():
        keep = {}

        def conv(x, w, b):
            if "conv" not in keep:
                y, keep["conv"] = S.causal_conv(x, w, b, activation="silu", return_state=True)
                return y
            return S.causal_conv_step(x, keep["conv"], w, b, activation="silu")

        def scan(u, dl, A, B, C, D, db):
            if "scan" not in keep:
                y, keep["scan"] = S.selective_scan(u, dl, A, B, C, D, db, softplus=True, return_state=True)
                return y
            return S.selective_scan_step(u, dl, A, B, C, keep["scan"], D, db, softplus=True)

        serve = dict(ours, conv=conv, scan=scan)
        parts = [block(par, f[:half], **serve)] + [block(par, f[t:t + 1], **serve) for t in range(half, len(f))]
    torch.testing.assert_close(torch.cat(parts).double().cpu(), want[:len(f)].detach(), rtol=0, atol=1e-4 * float(want.detach().abs().max()))


# ---- large offsets -------------------------------------------------------------------------------------------------------------
def test_beyond_2_31_elements(gpu):
    """Row offsets past 32 bits: the last sequence of a large batch against the same rows alone."""
    import speech_to_text_amd as S

    g = gen(gpu, 97)
    ch, last = 4096, 45
    rows = 2 ** 31 // ch + 200
    x = torch.empty(rows, ch, dtype=BF16, device=gpu)
    x.normal_(generator=g)
    off = torch.tensor([0, rows - last, rows], dtype=torch.int64, device=gpu)
    tail = x[-last:].contiguous()
    w = randn(g, ch, 4)
    assert torch.equal(S.causal_conv(x, w, None, off)[-last:], S.causal_conv(tail, w))
    y, r = S.add_norm(x, x)
    y2, r2 = S.add_norm(tail, tail)
    assert torch.equal(y[-last:], y2) and torch.equal(r[-last:], r2)
    del y, r
    assert torch.equal(S.gate_norm(x, x)[-last:], S.gate_norm(tail, tail))
    g1, g2 = S.gate_norm_backward(x, x, x), S.gate_norm_backward(tail, tail, tail)
    assert torch.equal(g1.x[-last:], g2.x) and torch.equal(g1.z[-last:], g2.z)
    del g1
    assert torch.equal(S.causal_conv_backward(x, x, w, None, off).x[-last:], S.causal_conv_backward(tail, tail, w).x)
    A = -rand(g, ch, 2, lo=0.1)
    B = torch.empty(rows, 2, dtype=BF16, device=gpu).normal_(generator=g)
    y = S.selective_scan(x, x, A, B, B, None, None, off, softplus=True)[-last:]
    ru, rA, rB = R.leaves(tail, A, B[-last:, None], grad=False)
    want, _ = R.selective_scan(ru, ru, rA, rB, rB, plus=True)
    size, _ = R.selective_scan(ru.abs(), R.softplus(ru), rA, rB.abs(), rB.abs())
    R.assert_close(y, want, BF16, size, 4 * R.scan_steps([last]), "y")    # |d A| up to 4 here
    gr = S.selective_scan_backward(x, x, x, A, B, B, None, None, off, softplus=True)
    alone = S.selective_scan_backward(tail, tail, tail, A, B[-last:].contiguous(), B[-last:].contiguous(), softplus=True)
    for a, b in ((gr.u, alone.u), (gr.delta, alone.delta), (gr.B, alone.B)):
        # the two calls cut the rows into different chunks: half a step of the type each, and the scan's own roundings
        torch.testing.assert_close(a[-last:].float(), b.float(), rtol=2.0 ** -7, atol=1e-3 * float(b.float().abs().max()))


# ---- refusals --------------------------------------------------------------------------------------------------------------------
def test_refusals(gpu):
    import speech_to_text_amd as S

    x, w = torch.zeros(10, 6, device=gpu), torch.zeros(6, 4, device=gpu)
    A, B = torch.zeros(6, 3, device=gpu), torch.zeros(10, 3, device=gpu)
    bad = [
        lambda: S.causal_conv(x.cpu(), w), lambda: S.causal_conv(x, w.cpu()), lambda: S.causal_conv(x.double(), w.double()),
        lambda: S.causal_conv(x, w.bfloat16()), lambda: S.causal_conv(x, w[:5]), lambda: S.causal_conv(x.t(), w),
        lambda: S.causal_conv(x[None], w), lambda: S.causal_conv(x, torch.zeros(6, 9, device=gpu)),
        lambda: S.causal_conv(x, torch.zeros(6, 0, device=gpu)), lambda: S.causal_conv(x, w, activation="relu"),
        lambda: S.causal_conv(x, w, None, [0, 5, 3]), lambda: S.causal_conv(x, w, None, [0, 11]),
        lambda: S.causal_conv(x, w, None, [-1, 10]), lambda: S.causal_conv(x, w, None, []), lambda: S.causal_conv(x, w, None, [0]),
        lambda: S.causal_conv(x, w, None, torch.zeros(3, dtype=torch.int32, device=gpu)),
        lambda: S.causal_conv(x, w, None, [0, 10], initial_state=torch.zeros(2, 3, 6, device=gpu)),
        lambda: S.causal_conv(x, w, out=x), lambda: S.causal_conv(x, w, out=torch.zeros(1, 6, device=gpu).expand(10, 6)),
        lambda: S.causal_conv(x, w, out=torch.zeros(9, 6, device=gpu)), lambda: S.causal_conv(x, w, torch.zeros(5, device=gpu)),
        lambda: S.causal_conv_backward(x[:9], x, w), lambda: S.causal_conv_backward(x.half(), x, w),
        lambda: S.causal_conv_step(x, torch.zeros(9, 3, 6, device=gpu), w),
        lambda: S.causal_conv_step(x, torch.zeros(10, 2, 6, device=gpu), w), lambda: S.causal_conv_step(x, None, w),
        lambda: S.causal_conv_step(x, torch.zeros(10, 6, 3, device=gpu).transpose(1, 2), w),
        lambda: S.causal_conv_step(x, torch.zeros(10, 3, 6, device=gpu), w, slots=torch.zeros(10, dtype=torch.int64, device=gpu)),
        lambda: S.causal_conv_step(x, torch.zeros(12, 3, 6, device=gpu)[:10], w, new_state=None, slots=torch.zeros(4, dtype=torch.int32, device=gpu)),
        lambda: S.selective_scan(x, x[:9], A, B, B), lambda: S.selective_scan(x, x.half(), A, B, B),
        lambda: S.selective_scan(x, x, torch.zeros(6, 65, device=gpu), torch.zeros(10, 65, device=gpu), torch.zeros(10, 65, device=gpu)),
        lambda: S.selective_scan(x, x, A, B[:, :2], B), lambda: S.selective_scan(x, x, A, B, B.half()),
        lambda: S.selective_scan(x, x, A, torch.zeros(10, 4, 3, device=gpu), torch.zeros(10, 4, 3, device=gpu)),
        lambda: S.selective_scan(x, x, A, torch.zeros(10, 2, 3, device=gpu), B), lambda: S.selective_scan(x, x, A, B, B, out=x),
        lambda: S.selective_scan(x, x, A, B, B, A[:, 0].bfloat16()), lambda: S.selective_scan(x, x, A, B.expand(10, 3).t(), B),
        lambda: S.selective_scan(x, x, A, B, B, initial_state=torch.zeros(1, 6, 3, device=gpu).half()),
        lambda: S.selective_scan_step(x, x, A, B, B, torch.zeros(9, 6, 3, device=gpu)), lambda: S.selective_scan_step(x, x, A, B, B, None),
        lambda: S.add_norm(x, x.half()), lambda: S.add_norm(x.half(), x.bfloat16()), lambda: S.add_norm(x, norm="batch"),
        lambda: S.add_norm(x, eps=0.0), lambda: S.add_norm(x, weight=torch.ones(5, device=gpu)), lambda: S.add_norm(x, x[:, :5]),
        lambda: S.add_norm(torch.zeros(1, 32769, device=gpu)), lambda: S.add_norm(x, scale=torch.ones(6, device=gpu).double()),
        lambda: S.add_norm_backward(x, None, x, scale=torch.ones(6, device=gpu)), lambda: S.add_norm_backward(x.half(), None, x.bfloat16()),
        lambda: S.gate_norm(x, x, groups=4), lambda: S.gate_norm(x, x, groups=0), lambda: S.gate_norm(x, x.half()),
        lambda: S.gate_norm(x, x, out=x), lambda: S.gate_norm_backward(x[:3], x, x),
    ]
    for i, call in enumerate(bad):
        try:
            call()
        except S.ParameterError:
            continue
        pytest.fail(f"call {i} was not refused")
    leaf = w.clone().requires_grad_()
    with pytest.raises(S.ParameterError):                    # single tokens have no gradient
        S.causal_conv_step(x, torch.zeros(10, 3, 6, device=gpu), leaf)
    with pytest.raises(S.ParameterError):
        S.causal_conv(x, leaf, out=torch.empty_like(x))
    state = torch.zeros(11, 3, 6, device=gpu)
    with pytest.raises(S.ParameterError):
        S.causal_conv_step(x, state[:10], w, new_state=state[1:])
    with pytest.raises(S.ParameterError):                    # the result in the middle of the states
        S.causal_conv_step(x, state[:10], w, out=state.view(33, 6)[:10])
    with pytest.raises(S.ParameterError):
        S.causal_conv(x, w, None, [0, 10], initial_state=state[:1], out=state.view(33, 6)[:10])


def test_differentiable_calls_are_not_captured(gpu):
    """Refused before anything is launched, so the capture itself stays valid."""
    import speech_to_text_amd as S

    x = torch.ones(4, 6, device=gpu)
    w = torch.ones(6, 2, device=gpu, requires_grad=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(S.ParameterError):
            S.causal_conv(x, w)
        with pytest.raises(S.ParameterError):
            S.causal_conv(x, w.detach(), None, [0, 4])       # nor host offsets
        with torch.no_grad():
            y = S.causal_conv(x, w)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert y[:, 0].tolist() == [1, 2, 2, 2]
