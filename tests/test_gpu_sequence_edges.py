"""Operators over packed rows (speech_to_text_amd/sequence.py) at their edges: the order of sums, values that are not finite,
what autograd and the tensors' version counters see, float32 results of 16-bit rows, and the scan's gradients against
bounds that a missing term breaks."""
import numpy as np
import pytest
import torch

from tests.test_gpu_sequence import gen, randn

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
