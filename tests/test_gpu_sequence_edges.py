"""Operators over packed rows (speech_to_text_amd/sequence.py) at their edges: the order of sums, values that are not finite,
what autograd and the tensors' version counters see, float32 results of 16-bit rows, and the scan's gradients against
bounds that a missing term breaks."""
import numpy as np
import pytest
import torch

from tests import sequence_ref as R
from tests.test_gpu_sequence import BF16, F32, SCAN, TYPES, device_offsets, gen, rand, randn, scan_case

pytestmark = pytest.mark.gpu


# ---- the order of sums ----------------------------------------------------------------------------------------
def folded(v):
    """Sum over the last axis, its upper half added to its lower one until one value is left, in float32."""
    while v.shape[-1] > 1:
        v = v[..., :v.shape[-1] // 2] + v[..., v.shape[-1] // 2:]
    return v[..., 0]


@pytest.mark.parametrize("n", [4, 8, 16, 32, 64])
def test_sums_over_channels_have_one_order(gpu, n):
    """dB and dC, bit for bit: over the channels of a wavefront by halves, then over the four wavefronts.  (With no decay,
    steps of one and ones for u, B and C both are the sum of dy.)"""
    import speech_to_text_amd as S

    g = gen(gpu, n)
    ch, rows = 4 * 64 * 4 // n, 21
    one, ones = torch.ones(rows, ch, device=gpu), torch.ones(rows, n, device=gpu)
    dy = randn(g, rows, ch) * torch.exp(randn(g, rows, ch))
    off = torch.arange(rows + 1, device=gpu)                 # rows by themselves: no state is carried
    got = S.selective_scan_backward(dy, one, one, torch.zeros(ch, n, device=gpu), ones, ones, None, None, off)
    waves = folded(dy.cpu().numpy().reshape(rows, 4, ch // 4))
    want = (waves[:, 0] + waves[:, 1]) + (waves[:, 2] + waves[:, 3])
    for t in (got.B, got.C):
        assert np.array_equal(t.cpu().numpy(), np.broadcast_to(want[:, None], (rows, n)))


# ---- values that are not finite ---------------------------------------------------------------------------------
def test_nan_stays_to_the_end_of_its_sequence(gpu):
    """A NaN is in every later row of its sequence and channel, also behind decays whose product is zero; the same
    backwards for the gradients."""
    import speech_to_text_amd as S

    g = gen(gpu, 1)
    rows, ch, n, end, at = 3000, 64, 4, 2900, 3
    u, dy = randn(g, rows, ch), randn(g, rows, ch)
    delta = torch.full((rows, ch), 0.5, device=gpu)
    A = torch.full((ch, n), -16.0, device=gpu)              # exp(-8) a row
    B, C = randn(g, rows, n), randn(g, rows, n)
    off = torch.tensor([0, end, rows], dtype=torch.int64, device=gpu)
    rest = torch.arange(ch, device=gpu) != at
    clean, _ = S.selective_scan(u, delta, A, B, C, None, None, off, return_state=True)
    grads = S.selective_scan_backward(dy, u, delta, A, B, C, None, None, off)
    u2 = u.clone()
    u2[10, at] = float("nan")
    y, state = S.selective_scan(u2, delta, A, B, C, None, None, off, return_state=True)
    assert torch.isnan(y[10:end, at]).all() and torch.isnan(state[0, at]).all()
    assert torch.equal(y[:, rest], clean[:, rest]) and torch.equal(y[:10], clean[:10]) and torch.equal(y[end:], clean[end:])
    dy2 = dy.clone()
    dy2[end - 10, at] = float("nan")
    g2 = S.selective_scan_backward(dy2, u, delta, A, B, C, None, None, off)
    for got, want in ((g2.u, grads.u), (g2.delta, grads.delta)):
        assert torch.isnan(got[:end - 9, at]).all()
        assert torch.equal(got[:, rest], want[:, rest]) and torch.equal(got[end - 9:], want[end - 9:])


@pytest.mark.parametrize("rate", [-3e38, float("-inf")])
def test_states_that_forget_at_once(gpu, rate):
    """A rate whose product with log2 e is infinite: the state is the row's own d u B, in sequences that start and end
    anywhere; a step of zero leaves it alone where the rate is finite."""
    import speech_to_text_amd as S

    g = gen(gpu, 2)
    lengths, ch, n = [5, 60, 1, 45], 9, 4
    off, rows = device_offsets(lengths, gpu), sum(lengths)
    u, dy = randn(g, rows, ch), randn(g, rows, ch)
    delta, B, C = rand(g, rows, ch, lo=0.01, hi=0.1), randn(g, rows, n), randn(g, rows, n)
    A = -rand(g, ch, n, lo=0.1, hi=1.0)
    A[:, 1] = rate
    y, state = S.selective_scan(u, delta, A, B, C, None, None, off, return_state=True)
    ru, rd, rA, rB, rC = R.leaves(u, delta, A, B[:, None], C[:, None], grad=False)
    want, final = R.selective_scan(ru, rd, rA, rB, rC, offsets=off.tolist())
    size, size_final = R.selective_scan(ru.abs(), rd, rA, rB.abs(), rC.abs(), offsets=off.tolist())
    R.assert_close(y, want, F32, size, R.scan_steps(lengths) + n, "y")
    R.assert_close(state, final, F32, size_final, R.scan_steps(lengths), "state")
    got = S.selective_scan_backward(dy, u, delta, A, B, C, None, None, off)
    assert all(torch.isfinite(t).all() for t in got if t is not None)
    assert (got.A[:, 1] == 0).all()
    pool = torch.ones(rows, ch, n, device=gpu)
    S.selective_scan_step(u, delta, A, B, C, pool)
    own = (rd * ru)[..., None] * rB
    R.assert_close(pool[..., 1], own[..., 1], F32, own[..., 1].abs(), 2, "token")
    if rate > float("-inf"):
        zero = torch.zeros_like(delta)
        init = torch.ones(len(lengths), ch, n, device=gpu)
        _, state = S.selective_scan(u, zero, A, B, C, None, None, off, initial_state=init, return_state=True)
        assert torch.equal(state, init)
        S.selective_scan_step(u, zero, A, B, C, pool, new_state=torch.empty_like(pool))


# ---- what autograd sees -------------------------------------------------------------------------------------------
def test_writes_raise_the_version_counter(gpu):
    """Pools and `out` are written as by torch's own in-place operations: a tensor that a backward pass still needs is
    missed there, and a leaf that requires a gradient is not written."""
    import speech_to_text_amd as S

    g = gen(gpu, 3)
    ch, n, m = 6, 3, 4
    x, w, A = randn(g, m, ch), randn(g, ch, 3), -rand(g, ch, n)
    B = randn(g, m, n)
    conv, scan = randn(g, m, 2, ch), randn(g, m, ch, n)
    out, into = torch.empty_like(x), torch.empty_like(conv)
    writes = [
        (lambda: S.causal_conv_step(x, conv, w), [conv], [x, w, out]),
        (lambda: S.causal_conv_step(x, conv, w, new_state=into, out=out), [into, out], [conv, x, w]),
        (lambda: S.selective_scan_step(x, x, A, B, B, scan), [scan], [x, A, B]),
        (lambda: S.selective_scan_step(x, x, A, B, B, scan, out=out), [scan, out], [x, A, B]),
        (lambda: S.causal_conv(x, w, out=out), [out], [x, w]), (lambda: S.selective_scan(x, x, A, B, B, out=out), [out], [x, A, B]),
        (lambda: S.gate_norm(x, x, out=out), [out], [x]),
    ]
    for i, (call, written, read) in enumerate(writes):
        before = [t._version for t in written], [t._version for t in read]
        call()
        assert all(t._version > v for t, v in zip(written, before[0])), i
        assert all(t._version == v for t, v in zip(read, before[1])), i
    leaf = x.clone().requires_grad_()
    for pool, f, step in ((conv, lambda p: S.causal_conv(leaf, w, None, [0, 1, 2, 3, 4], initial_state=p), lambda p: S.causal_conv_step(x, p, w)),
                          (scan, lambda p: S.selective_scan(leaf, x, A, B, B, None, None, [0, 1, 2, 3, 4], initial_state=p),
                           lambda p: S.selective_scan_step(x, x, A, B, B, p))):
        y = f(pool)
        step(pool)                                          # before the backward pass has read it
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    for call in (lambda t: S.causal_conv(x, w, out=t), lambda t: S.gate_norm(x, x, out=t), lambda t: S.selective_scan(x, x, A, B, B, out=t),
                 lambda t: S.causal_conv_step(x, conv, w, out=t), lambda t: S.selective_scan_step(x, x, A, B, B, scan, out=t)):
        with pytest.raises(S.ParameterError):
            call(torch.empty_like(x).requires_grad_())
        with torch.no_grad():
            call(torch.empty_like(x).requires_grad_())
    with pytest.raises(S.ParameterError):
        S.causal_conv_step(x, conv, w, new_state=torch.empty_like(conv).requires_grad_())
    with pytest.raises(S.ParameterError):
        S.selective_scan_step(x, x, A, B, B, scan, new_state=torch.empty_like(scan).requires_grad_())
    with torch.inference_mode():
        pool = conv.clone()
        S.causal_conv_step(x, pool, w)
    S.causal_conv_step(x, pool, w)                          # tensors without a counter are written all the same


def test_frozen_tables_and_rows(gpu):
    """Whatever does not require a gradient gets none, and the others' are those of a call where all do."""
    import speech_to_text_amd as S

    g = gen(gpu, 6)
    m, ch, n = 40, 12, 4
    rows = lambda: randn(g, m, ch)
    per = lambda *s: randn(g, ch, *s)
    init, h0 = randn(g, 1, 2, ch), randn(g, 1, ch, n)
    calls = [
        (lambda x, w, b, i: S.causal_conv(x, w, b, activation="silu", initial_state=i), [rows(), per(3), per(), init]),
        (lambda u, d, A, B, C, D, b, i: S.selective_scan(u, d, A, B, C, D, b, softplus=True, initial_state=i),
         [rows(), rows(), -rand(g, ch, n), randn(g, m, n), randn(g, m, n), per(), per(), h0]),
        (lambda x, r, w, b, s: S.add_norm(x, r, w, b, scale=s)[0], [rows(), rows(), per(), per(), per()]),
        (lambda x, z, w, b: S.gate_norm(x, z, w, b), [rows(), rows(), per(), per()]),
    ]
    for f, ins in calls:
        dy = rows()
        leaves = [t.clone().requires_grad_() for t in ins]
        want = torch.autograd.grad(f(*leaves), leaves, dy)
        for free in range(len(ins)):
            leaves = [t.clone().requires_grad_(i == free) for i, t in enumerate(ins)]
            f(*leaves).backward(dy)
            for i, t in enumerate(leaves):
                assert (t.grad is None) == (i != free)
            assert torch.equal(leaves[free].grad, want[free])


# ---- float32 results of 16-bit rows ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_float32_results_carry_float32_functions(gpu, dtype):
    """Far out, where an exponent rounded once more (|p| 2^-24 and more) would show: the state's softplus, the gradient
    of its bias, and the gradients of taps, biases and norm weights through SiLU."""
    import speech_to_text_amd as S

    at = torch.tensor([-80.0, -61.25, -43.5, -20.75, -9.5, -3.25, 1.5, 7.75, 30.5])     # exact in every type
    ch, p = len(at), at.double()
    x, one = at[None].to(gpu, dtype), torch.ones(1, ch, dtype=dtype, device=gpu)
    ones = torch.ones(1, 1, dtype=dtype, device=gpu)

    def close(got, want, steps, size=None):
        R.assert_close(got.flatten(), want, F32, want.abs() if size is None else size, steps)

    # softplus: its exp 3 units, log 2 (near zero the exp's own), two sums; times u and B
    zero_A = torch.zeros(ch, 1, device=gpu)
    _, h = S.selective_scan(one, x, zero_A, ones, ones, softplus=True, return_state=True)
    close(h, R.softplus(p), 8)
    pool = torch.zeros(1, ch, 1, device=gpu)
    S.selective_scan_step(one, x, zero_A, ones, ones, pool, softplus=True)
    close(pool, R.softplus(p), 8)
    # ddelta_bias = sigmoid(delta) here: exp 3, sum 1, reciprocal 1, product
    zero = torch.zeros(ch, device=gpu)
    grads = S.selective_scan_backward(one, one, x, zero_A, ones, ones, None, zero, softplus=True)
    sig = 1 / (1 + torch.exp(-p))
    close(grads.delta_bias, sig, 8)
    # SiLU'(p) = sig (1 + p (1 - sig)): the sigmoid's units in both factors, and the sum's cancellation
    slope, size = sig * (1 + p * (1 - sig)), sig * (1 + p.abs() * (1 - sig))
    g = S.causal_conv_backward(one, x, torch.ones(ch, 1, device=gpu), zero, activation="silu")
    close(g.bias, slope, 16, size)
    close(g.weight, slope * p, 17, size * p.abs())
    # (norm(x) w + b) silu(z): dbias = dy silu(z), in rows held in registers and in wide ones
    for width in (ch, 8200):
        z = torch.zeros(1, width, dtype=dtype, device=gpu)
        z[:, :ch] = x
        w = torch.ones(width, device=gpu)
        g = S.gate_norm_backward(torch.ones_like(z), torch.ones_like(z), z, w, w, gate_first=False)
        close(g.bias[:ch], p * sig, 8)


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_give_the_bits_of_the_prompt(gpu, dtype):
    """Many values: the convolution token by token rounds as the convolution of the whole sequence does."""
    import speech_to_text_amd as S

    g = gen(gpu, 5)
    rows, ch = 48, 8192
    x, w, b = randn(g, rows, ch, dtype=dtype), randn(g, ch, 4), randn(g, ch)
    whole, last = S.causal_conv(x, w, b, activation="silu", return_state=True)
    state = torch.zeros(1, 3, ch, dtype=dtype, device=gpu)
    tokens = S.causal_conv_step(x, state, w, b, activation="silu", slots=torch.zeros(rows, dtype=torch.int32, device=gpu))
    assert torch.equal(tokens, whole) and torch.equal(state, last)


# ---- the scan's gradients, element by element -------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(SCAN)))
def test_selective_scan_gradients(gpu, case, dtype):
    """Every gradient with initial states and a gradient of the final ones, against bounds from each element's own
    terms (tests/test_sequence_cpu.py shows that a gradient of zero, or one without its A or its B term, breaks them)."""
    import speech_to_text_amd as S

    args, init, dy, dstate, off, plus, clean = R.scan_gradient_case(gpu, SCAN[case], dtype, 300 + case, scan_case)
    grads = S.selective_scan_backward(dy, *args, off, softplus=plus, initial_state=init, dstate=dstate)
    refs, sizes, steps = R.scan_gradients(dy, *args, off.tolist(), plus, init, dstate, clean)
    for k, ref in refs.items():
        got = getattr(grads, k)
        if k in ("u", "delta", "B", "C"):
            assert (got[clean:] == 0).all(), k
            got = got[:clean]
        R.assert_close(got, ref, F32 if k in ("A", "D", "delta_bias", "initial_state") else dtype, sizes[k], steps[k], k)


def test_scan_into_a_column_range(gpu):
    """`out` with rows further apart than its channels: the rows of sequences are those of a plain call, the rest of
    the matrix stays as it was."""
    import speech_to_text_amd as S

    g = gen(gpu, 61)
    for dtype in TYPES:
        for rows, ch, n in ((90, 33, 5), (20, 7, 3), (700, 130, 16)):
            u, delta = randn(g, rows, ch, dtype=dtype), randn(g, rows, ch, dtype=dtype)
            B, C, A = randn(g, rows, n, dtype=dtype), randn(g, rows, n, dtype=dtype), -rand(g, ch, n, lo=0.1)
            off = [3, 9, 9, rows - 2]
            want = S.selective_scan(u, delta, A, B, C, None, None, off, softplus=True)
            base = torch.full((rows, ch + 11), 3.0, dtype=dtype, device=gpu)
            out = base[:, 4:4 + ch]
            assert S.selective_scan(u, delta, A, B, C, None, None, off, softplus=True, out=out) is out
            assert torch.equal(out[3:rows - 2], want[3:rows - 2])
            assert (out[:3] == 3).all() and (out[rows - 2:] == 3).all()
            assert (base[:, :4] == 3).all() and (base[:, 4 + ch:] == 3).all()


# ---- single tokens: one and four entries per thread ------------------------------------------------------------------
@pytest.mark.parametrize("batch,ch,n,listed", [(603, 400, 16, True), (603, 400, 16, False), (511, 400, 16, True), (527, 30, 8, True),
                                               (131, 3001, 64, True), (131, 3001, 64, False)])
def test_scan_step_by_wavefronts(gpu, batch, ch, n, listed):
    """Around the sizes where a thread takes four entries: each as a call of its own, slots out of order and one twice."""
    import speech_to_text_amd as S

    g = gen(gpu, batch + ch)
    u, delta = randn(g, batch, ch, dtype=BF16), randn(g, batch, ch, dtype=BF16)
    B, C, A, D = randn(g, batch, n, dtype=BF16), randn(g, batch, n, dtype=BF16), -rand(g, ch, n, lo=0.1, hi=2.0), randn(g, ch)
    pool = randn(g, batch, ch, n)
    slots = None
    if listed:
        slots = torch.randperm(batch, generator=g, device=gpu).to(torch.int32)
        slots[7], slots[batch - 1] = -1, slots[5]
    got = pool.clone()
    y = S.selective_scan_step(u, delta, A, B, C, got, D, softplus=True, slots=slots)
    few = list(range(0, batch, max(1, batch // 20))) + [5, 7, batch - 2, batch - 1]
    for i in sorted(set(few)):
        at = i if slots is None else int(slots[i])
        if at < 0:
            assert (y[i] == 0).all()
            continue
        one = pool[at:at + 1].clone()
        if listed and i == batch - 1:                       # the second token of its sequence
            S.selective_scan_step(u[5:6], delta[5:6], A, B[5:6], C[5:6], one, D, softplus=True)
        want = S.selective_scan_step(u[i:i + 1], delta[i:i + 1], A, B[i:i + 1], C[i:i + 1], one, D, softplus=True)
        assert torch.equal(y[i], want[0])
        if not (listed and i == 5):
            assert torch.equal(got[at], one[0])


# ---- refusals -----------------------------------------------------------------------------------------------------------
def test_out_over_a_table_is_refused(gpu):
    """Tables, offsets and slots are inputs too."""
    import speech_to_text_amd as S

    ch, n, m = 6, 4, 10
    memory = torch.zeros(200, device=gpu)
    out = memory[40:40 + m * ch].view(m, ch)
    x, free = torch.zeros(m, ch, device=gpu), torch.zeros(m, ch, device=gpu)
    table = lambda *s, at=90: memory[at:at + int(np.prod(s))].view(s)
    w, v, A, B = torch.zeros(ch, 3, device=gpu), torch.zeros(ch, device=gpu), torch.zeros(ch, n, device=gpu), torch.zeros(m, n, device=gpu)
    off = memory[96:102].view(torch.int64)[:2]
    slots = memory[90:100].view(torch.int32)
    pool, states = torch.zeros(m, 2, ch, device=gpu), torch.zeros(m, ch, n, device=gpu)
    calls = [
        lambda o: S.causal_conv(x, table(ch, 3), out=o), lambda o: S.causal_conv(x, w, table(ch), out=o),
        lambda o: S.causal_conv(x, w, None, off, out=o), lambda o: S.selective_scan(x, x, table(ch, n), B, B, out=o),
        lambda o: S.selective_scan(x, x, A, B, B, table(ch), out=o), lambda o: S.selective_scan(x, x, A, B, B, None, table(ch), out=o),
        lambda o: S.selective_scan(x, x, A, B, B, None, None, off, out=o), lambda o: S.gate_norm(x, x, table(ch), out=o),
        lambda o: S.gate_norm(x, x, None, table(ch), out=o), lambda o: S.causal_conv_step(x, pool, table(ch, 3), out=o),
        lambda o: S.causal_conv_step(x, pool, w, table(ch), out=o), lambda o: S.causal_conv_step(x, pool, w, slots=slots, out=o),
        lambda o: S.selective_scan_step(x, x, table(ch, n), B, B, states, out=o),
        lambda o: S.selective_scan_step(x, x, A, B, B, states, table(ch), out=o),
        lambda o: S.selective_scan_step(x, x, A, B, B, states, None, table(ch), out=o),
        lambda o: S.selective_scan_step(x, x, A, B, B, states, slots=slots, out=o),
    ]
    for i, call in enumerate(calls):
        try:
            call(out)
        except S.ParameterError:
            call(free)
            continue
        pytest.fail(f"call {i} was not refused")
