"""Host side of the decoder-block operators: rotary frequencies, the generator's oracle, argument checks."""
import math

import pytest
import torch

import decoder_oracle as oracle
from nexar_b200 import ops


def test_frequencies_without_scaling():
    f, m = ops.rotary_frequencies(64, 10000.0)
    assert m == 1.0 and len(f) == 32 and f[0] == 1.0
    assert f[31] == pytest.approx(10000.0 ** (-62 / 64), rel=1e-14)


@pytest.mark.parametrize("dim", [2, 8, 64, 96, 128])
def test_scaled_frequencies_lie_between_plain_and_stretched(dim):
    plain, _ = ops.rotary_frequencies(dim)
    for kind, factor, length in oracle.SCALINGS:
        f, m = ops.rotary_frequencies(dim, scaling=ops.RotaryScaling(kind, factor, length))
        assert len(f) == len(plain)
        for a, b in zip(f, plain):
            assert b / factor * (1 - 1e-12) <= a <= b * (1 + 1e-12)
        assert m == pytest.approx(0.1 * math.log(factor) + 1 if kind == "yarn" else 1.0)


def test_linear_and_ntk_end_points():
    plain, _ = ops.rotary_frequencies(128)
    lin, _ = ops.rotary_frequencies(128, scaling=ops.RotaryScaling("linear", 4.0))
    assert all(a == pytest.approx(b / 4, rel=1e-14) for a, b in zip(lin, plain))
    ntk, _ = ops.rotary_frequencies(128, scaling=ops.RotaryScaling("ntk", 4.0))
    assert ntk[0] == plain[0] and ntk[-1] == pytest.approx(plain[-1] / 4, rel=1e-12)


def test_bands_and_yarn_keep_the_fast_pairs_and_stretch_the_slow_ones():
    plain, _ = ops.rotary_frequencies(128)
    for kind, length in (("bands", 8192), ("yarn", 4096)):
        f, _ = ops.rotary_frequencies(128, scaling=ops.RotaryScaling(kind, 8.0, length))
        assert f[0] == plain[0] and f[-1] == pytest.approx(plain[-1] / 8, rel=1e-12)
    f, m = ops.rotary_frequencies(128, scaling=ops.RotaryScaling("yarn", 8.0, 4096, magnitude=1.0))
    assert m == 1.0


def _yarn_by_definition(dim, base, factor, length, fast=32.0, slow=1.0):
    """The ramp runs over the pairs from the one that turns ``fast`` times in the original length to the one that
    turns ``slow`` times (a pair's number is real: turns(x) = length base^(-2 x / dim) / 2 pi), widened to whole
    numbers and held inside 0 .. dim - 1."""
    def pair_with(turns):
        lo, hi = -2.0 * dim, 2.0 * dim
        for _ in range(200):  # the number of turns falls with the pair
            mid = (lo + hi) / 2
            lo, hi = (mid, hi) if length * base ** (-2 * mid / dim) / (2 * math.pi) > turns else (lo, mid)
        return (lo + hi) / 2
    first, last = max(math.floor(pair_with(fast)), 0), min(math.ceil(pair_with(slow)), dim - 1)
    out = []
    for i in range(dim // 2):
        plain = base ** (-2 * i / dim)
        share = 0.0 if i <= first else min((i - first) / (last - first), 1.0)  # before the ramp: as trained
        out.append(plain * (1 - share) + plain / factor * share)
    return out


@pytest.mark.parametrize("dim,base,factor,length", [
    (128, 10000.0, 8.0, 4096), (64, 10000.0, 16.0, 8192),         # the slowest pairs turn less than once
    (128, 10000.0, 4.0, 65536), (64, 10000.0, 4.0, 131072), (128, 10000.0, 4.0, 262144),  # all turn more than once
    (96, 500.0, 2.0, 100000), (128, 10000.0, 4.0, 10 ** 12)])     # the ramp's end at the last number it may take
def test_yarn_frequencies_by_definition(dim, base, factor, length):
    f, _ = ops.rotary_frequencies(dim, base, ops.RotaryScaling("yarn", factor, length))
    for got, want in zip(f, _yarn_by_definition(dim, base, factor, length)):
        assert got == pytest.approx(want, rel=1e-12)


def test_philox_known_answers():
    """The published test vectors of Philox4x32-10 (Random123)."""
    assert oracle.philox_words((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert oracle.philox_words((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert oracle.philox_words((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0)) == [
        0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_oracle_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, 9, 3, 8, generator=g, dtype=torch.float64) for _ in range(3))
    s = torch.randn(2, 3, 8, 8, generator=g, dtype=torch.float64)
    lam = torch.tensor([-0.1, 0.0, -1.0])
    do, df = torch.randn_like(q), torch.randn_like(s)
    n = torch.tensor([9, 4])

    def loss(q, k, v, s):
        o, f = oracle.decay_attention(q, k, v, lam, s, n)
        return (o * do).sum() + (f * df).sum()
    x = [t.clone().requires_grad_(True) for t in (q, k, v, s)]
    grads = torch.autograd.grad(loss(*x), x)
    for i in range(4):
        d = [torch.randn_like(t) if j == i else torch.zeros_like(t) for j, t in enumerate(x)]
        want = oracle.directional(loss, [t.detach() for t in x], d)
        assert sum((a * b).sum() for a, b in zip(grads, d)) == pytest.approx(want.item(), rel=1e-6, abs=1e-6)


@pytest.mark.parametrize("bad", [dict(kind="cubic", factor=2.0), dict(kind="linear", factor=0.5),
                                 dict(kind="yarn", factor=float("inf")), dict(kind="bands", factor=2.0, low=4.0, high=1.0),
                                 dict(kind="yarn", factor=2.0, fast=1.0, slow=32.0),
                                 dict(kind="linear", factor=2.0, original_length=0)])
def test_scaling_refusals(bad):
    with pytest.raises(ValueError):
        ops.RotaryScaling(**bad)


@pytest.mark.parametrize("args", [(0,), (7,), (64, 1.0), (64, float("nan"))])
def test_frequency_refusals(args):
    with pytest.raises(ValueError):
        ops.rotary_frequencies(*args)


def test_rotary_refusals_on_the_host():
    x, t = torch.zeros(4, 2, 8), torch.zeros(4, 8)
    with pytest.raises(ValueError, match="layout"):
        ops.rotary(x, t, layout="thirds")
    with pytest.raises(ValueError, match="heads"):
        ops.rotary(x, t, heads=-1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rotary(x, t)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rotary_qk(x, x, t)
    with pytest.raises(ValueError, match="position"):
        ops.rotary_table(0, 8)
    with pytest.raises(ValueError, match="GPU"):
        ops.rotary_table(4, 8, device="cpu")


def test_dropout_refusals_on_the_host():
    state = ops.DropoutState(1, device="cpu")
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            ops.dropout(x, p, state)
    with pytest.raises(TypeError, match="DropoutState"):
        ops.dropout(x, 0.1, 7)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.dropout(x, 0.1, state)
    w = torch.ones(8, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="DropoutState"):
        ops.residual_layer_norm(x, x, w, w, p=0.1)
    with pytest.raises(ValueError, match="probability"):
        ops.residual_layer_norm(x, x, w, w, p=2.0, dropout=state)
    with pytest.raises(ValueError, match="elements"):
        ops.residual_layer_norm(x, x[:2], w, w, p=0.1, dropout=state)


def test_dropout_state_on_the_host():
    s = ops.DropoutState((1 << 64) - 1, device="cpu", step=5)  # seeds wrap to 64 bits
    assert s.tensor.tolist() == [-1, 5]
    s.advance()
    assert s.tensor.tolist() == [-1, 6]
    s.set(3)
    assert s.tensor.tolist() == [3, 0]


def test_decay_refusals_on_the_host():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    lam = torch.zeros(2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.decay_attention(q, q, q, lam)
    with pytest.raises(ValueError, match="log_decay"):
        ops.decay_attention(q, q, q, lam.requires_grad_(True))
    with pytest.raises(ValueError, match="qkv"):
        ops.decay_attention_qkv(q, lam)
    one = q[:, 0]
    with pytest.raises(ValueError, match="no gradient"):
        ops.decay_attention_step(one.clone().requires_grad_(True), one, one, lam.detach(), torch.zeros(1, 2, 64, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.decay_attention_step(one, one, one, lam.detach(), torch.zeros(1, 2, 64, 64))


def test_tangents_are_refused():
    """Forward-mode derivatives: an error, not a result without a tangent (on the host the check comes before that of
    the device)."""
    from torch.autograd import forward_ad
    state = ops.DropoutState(1, device="cpu")
    x, t = torch.zeros(4, 2, 8), torch.zeros(4, 8)
    w = torch.ones(8, dtype=torch.bfloat16)
    rows = torch.zeros(4, 8, dtype=torch.bfloat16)
    q, lam, s0 = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(2), torch.zeros(1, 2, 64, 64)
    qkv, one = torch.zeros(1, 4, 3, 2, 64, dtype=torch.bfloat16), q[:, 0].clone()
    with forward_ad.dual_level():
        def dual(v):
            return forward_ad.make_dual(v, torch.ones_like(v))
        calls = [
            lambda: ops.rotary(dual(x), t), lambda: ops.rotary(x, dual(t)), lambda: ops.rotary_qk(x, dual(x), t),
            lambda: ops.dropout(dual(x), 0.1, state), lambda: ops.dropout(dual(x), 0.0, state),
            lambda: ops.residual_layer_norm(dual(rows), rows, w, w, p=0.1, dropout=state),
            lambda: ops.residual_layer_norm(rows, rows, w, dual(w), p=0.1, dropout=state),
            lambda: ops.decay_attention(dual(q), q, q, lam), lambda: ops.decay_attention(q, q, dual(q), lam),
            lambda: ops.decay_attention(q, q, q, dual(lam)), lambda: ops.decay_attention(q, q, q, lam, state=dual(s0)),
            lambda: ops.decay_attention_qkv(dual(qkv), lam), lambda: ops.decay_attention_step(one, dual(one), one, lam, s0),
            lambda: ops.decay_attention_step(one, one, one, lam, dual(s0))]
        for i, call in enumerate(calls):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
