"""Attention with a decay per head against the written-out sums in 64 bits."""
import pytest
import torch

import decoder_oracle as oracle

pytestmark = pytest.mark.gpu

DECAYS = {"mixed": [0.0, -0.002, -0.03, -0.7], "steep": [-5.0, -30.0, -90.0, -1e4], "none": [0.0] * 4}


def _inputs(dev, B, T, H, D, seed, decays="mixed"):
    g = torch.Generator(device=dev).manual_seed(seed)
    q, k, v, do = (torch.randn(B, T, H, D, device=dev, generator=g).to(torch.bfloat16) for _ in range(4))
    s0, ds = (torch.randn(B, H, D, D, device=dev, generator=g) for _ in range(2))
    lam = torch.tensor((DECAYS[decays] * H)[:H], device=dev)
    return q, k, v, do, s0, ds, lam


def _check(got, want, size, T, D, what, state=False):
    """size: the result's sum with every factor in absolute value. A bf16 output is rounded once (half a step). The
    scores and the states that enter it are split into two bf16 parts: each factor keeps 16 bits (2^-16; twice,
    and once more for products of two errors). All sums are fp32 over at most T + D + 64 terms (2^-24 each), and the
    powers of the decay are fp32 values (2^-23 for their products). The state's keys are split into three parts (2^-23).
    """
    f32 = 2.0 ** -24
    extra = ((T + D + 64) * f32 + 2.0 ** -21 + (0 if state else 3 * 2.0 ** -16)) * size
    half = oracle.half_step(got.dtype)
    oracle.assert_within(got, want, half * (want.abs() + extra) + extra + 1e-30, what)


def _sizes(q, k, v, lam, s0, n, scale):
    return oracle.decay_attention(q.abs(), k.abs(), v.abs(), lam, None if s0 is None else s0.abs(), n, scale)


def _compare(dev, B, T, H, D, lengths=None, state=True, decays="mixed", views=None, train=True, scale=None, seed=0):
    from nexar_b200 import ops
    q, k, v, do, s0, ds, lam = _inputs(dev, B, T, H, D, seed + T + D, decays)
    if views:
        q, k, v = views(q, k, v)
    if not state:
        s0 = None
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=dev)
    leaves = [t.requires_grad_(train) for t in (q, k, v) + ((s0,) if state else ())]
    o, final = ops.decay_attention(q, k, v, lam, state=s0, lengths=n, scale=scale, return_state=True)
    x = [t.detach().double().requires_grad_(True) for t in leaves]
    s64 = x[3] if state else None
    ow, fw = oracle.decay_attention(*x[:3], lam, s64, n, scale)
    with torch.no_grad():
        osz, fsz = _sizes(*x[:3], lam, s64, n, scale)
    _check(o.detach(), ow.detach(), osz, T, D, "o")
    _check(final.detach(), fw.detach(), fsz, T, D, "final state", True)
    if not train:
        return
    got = torch.autograd.grad((o, final), leaves, (do, ds))
    want = torch.autograd.grad((ow, fw), x, (do.double(), ds.double()))
    a = [t.detach().abs().requires_grad_(True) for t in x]
    osz, fsz = oracle.decay_attention(*a[:3], lam, a[3] if state else None, n, scale)
    size = torch.autograd.grad((osz, fsz), a, (do.double().abs(), ds.double().abs()))
    for i, name in enumerate(["dq", "dk", "dv"] + (["dstate"] if state else [])):
        _check(got[i], want[i], size[i], T, D, name, name == "dstate")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 127, 130])
def test_short_sequences(cuda0, T, D):
    _compare(cuda0, 2, T, 3, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,H", [(1, 1000, 1), (1, 257, 4), (3, 700, 2), (1, 2049, 2)])
@pytest.mark.parametrize("state", [True, False])
def test_split_over_the_tokens(cuda0, B, T, H, D, state):
    """Few sequences and heads: several segments, the last one ragged."""
    _compare(cuda0, B, T, H, D, state=state)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,H,lengths", [(2, 3000, 4, [3000, 1234]), (1, 5000, 12, None), (3, 4097, 6, [0, 4097, 4000])])
def test_long_sequences_split_in_both_passes(cuda0, B, T, H, lengths, D):
    """The backward pass splits into fewer segments than the forward pass, whose states it reads."""
    _compare(cuda0, B, T, H, D, lengths=lengths)


@pytest.mark.parametrize("D", [64, 128])
def test_many_heads_without_a_split(cuda0, D):
    _compare(cuda0, 16, 190, 12, D)


@pytest.mark.parametrize("decays", ["steep", "none"])
@pytest.mark.parametrize("T", [70, 600])
def test_steep_and_absent_decays(cuda0, decays, T):
    _compare(cuda0, 1, T, 4, 64, decays=decays)


@pytest.mark.parametrize("T", [70, 600])
def test_a_decay_to_nothing(cuda0, T):
    """exp(-inf) and exp(-1e4) are both 0: a token sees itself alone."""
    from nexar_b200 import ops
    q, k, v, do, s0, ds, _ = _inputs(cuda0, 2, T, 3, 128, 5)
    got = []
    for g in (float("-inf"), -1e4):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v, s0)]
        o, s = ops.decay_attention(*leaves[:3], torch.full((3,), g, device=cuda0), state=leaves[3], return_state=True)
        got.append((o.detach(), s.detach()) + torch.autograd.grad((o, s), leaves, (do, ds)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_tensors_at_any_address(cuda0):
    """Inputs and gradients that are handed over as contiguous views at odd addresses."""
    from nexar_b200 import ops
    q, k, v, do, s0, ds, lam = _inputs(cuda0, 1, 70, 2, 64, 6)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda0)
        flat[1:] = t.reshape(-1)
        return flat[1:].view_as(t)

    def run(qkv, a, b):
        o, s = ops.decay_attention(*qkv, lam, return_state=True)
        return (o.detach(), s.detach()) + torch.autograd.grad((o, s), qkv, (a, b))
    odd = [moved(t.detach()).requires_grad_(True) for t in leaves]
    assert all(t.data_ptr() % 16 == 2 for t in odd)
    assert all(torch.equal(x, y) for x, y in zip(run(leaves, do, ds), run(odd, moved(do), moved(ds))))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,lengths", [(100, [0, 1, 64, 99, 100, 37]), (900, [900, 0, 1, 128, 513, 899]), (5, [0, 0])])
def test_lengths(cuda0, T, lengths, D):
    _compare(cuda0, len(lengths), T, 2, D, lengths=lengths)


def test_lengths_outside_the_range_are_clipped(cuda0):
    from nexar_b200 import ops
    q, k, v, _, s0, _, lam = _inputs(cuda0, 2, 80, 2, 64, 3)
    far = ops.decay_attention(q, k, v, lam, s0, torch.tensor([99, -7], dtype=torch.int32, device=cuda0), return_state=True)
    near = ops.decay_attention(q, k, v, lam, s0, torch.tensor([80, 0], dtype=torch.int32, device=cuda0), return_state=True)
    assert all(torch.equal(a, b) for a, b in zip(far, near)) and torch.equal(near[1][1], s0[1])


@pytest.mark.parametrize("T", [100, 1500])
def test_rows_behind_a_sequence_are_not_read(cuda0, T):
    """Infinities and NaN there change nothing and get zero gradients."""
    from nexar_b200 import ops
    q, k, v, do, s0, ds, lam = _inputs(cuda0, 2, T, 2, 64, 4)
    n = torch.tensor([T - 41, 3], dtype=torch.int32, device=cuda0)
    outs = []
    for junk in (0.0, float("nan"), float("inf")):
        x = [t.clone() for t in (q, k, v, do)]
        for t in x:
            t[0, T - 41:] = junk
            t[1, 3:] = junk
        leaves = [t.requires_grad_(True) for t in x[:3] + [s0.clone()]]
        o, f = ops.decay_attention(*leaves[:3], lam, leaves[3], n, return_state=True)
        outs.append([o, f, *torch.autograd.grad((o, f), leaves, (x[3], ds))])
    for a, b, c in zip(*outs):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.isfinite(a).all()
    assert not outs[0][0][1, 3:].any() and not outs[0][2][0, T - 41:].any()


def test_strides_and_shared_heads(cuda0):
    """Views of a packed projection, transposed, unaligned, and keys shared by all heads."""
    def packed(q, k, v):
        return torch.stack([q, k, v], 2).unbind(2)

    def transposed(q, k, v):
        return tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))

    def odd(q, k, v):
        wide = torch.nn.functional.pad(torch.cat([q, k, v], -1), (1, 2))
        return tuple(t.detach() for t in wide[..., 1:-2].split(q.shape[-1], -1))
    for f in (packed, transposed, odd):
        _compare(cuda0, 2, 77, 3, 64, views=f)
    from nexar_b200 import ops
    q, k, v, do, _, _, lam = _inputs(cuda0, 2, 50, 4, 64, 7)
    shared = k[:, :, :1].clone().requires_grad_(True)
    (got,) = torch.autograd.grad(ops.decay_attention(q, shared.expand(-1, -1, 4, -1), v, lam), shared, do)
    full = shared.detach().expand(-1, -1, 4, -1).contiguous().requires_grad_(True)
    (each,) = torch.autograd.grad(ops.decay_attention(q, full, v, lam), full, do)
    assert torch.equal(got, each.sum(2, keepdim=True))


def test_packed_form_is_the_same(cuda0):
    from nexar_b200 import ops
    q, k, v, do, s0, ds, lam = _inputs(cuda0, 2, 200, 3, 64, 8)
    qkv = torch.stack([q, k, v], 2).requires_grad_(True)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o, f = ops.decay_attention_qkv(qkv, lam, state=s0, return_state=True)
    o2, f2 = ops.decay_attention(*x, lam, state=s0, return_state=True)
    assert torch.equal(o, o2) and torch.equal(f, f2)
    (g,) = torch.autograd.grad((o, f), qkv, (do, ds))
    assert torch.equal(g, torch.stack(torch.autograd.grad((o2, f2), x, (do, ds)), 2))
    with torch.no_grad():
        assert torch.equal(ops.decay_attention_qkv(qkv, lam, state=s0), o)


def test_gradient_against_differences(cuda0):
    from nexar_b200 import ops
    q, k, v, do, s0, ds, lam = _inputs(cuda0, 1, 140, 2, 64, 9)
    leaves = [t.requires_grad_(True) for t in (q, k, v, s0)]
    grads = torch.autograd.grad(ops.decay_attention(q, k, v, lam, s0, return_state=True), leaves, (do, ds))

    def loss(q, k, v, s):
        o, f = oracle.decay_attention(q, k, v, lam, s)
        return (o * do.double()).sum() + (f * ds.double()).sum()
    at = [t.detach().double() for t in leaves]
    for i, got in enumerate(grads):
        way = [torch.randn_like(t) if j == i else torch.zeros_like(t) for j, t in enumerate(at)]
        want = oracle.directional(loss, at, way)  # linear in each input: no truncation error
        size = (got.double().abs() * way[i].abs()).sum()
        assert abs((got.double() * way[i]).sum() - want) <= 2 * 2.0 ** -8 * size, i


@pytest.mark.parametrize("which", [(0,), (1,)])
def test_partial_outputs(cuda0, which):
    """Only the output or only the state has a gradient: the formula's with zeros for the other."""
    from nexar_b200 import ops
    q, k, v, do, s0, ds, lam = _inputs(cuda0, 2, 100, 2, 64, 10)
    leaves = [t.requires_grad_(True) for t in (q, k, v, s0)]
    out = ops.decay_attention(q, k, v, lam, s0, return_state=True)
    got = torch.autograd.grad([out[i] for i in which], leaves, [(do, ds)[i] for i in which])
    do, ds = (t if i in which else torch.zeros_like(t) for i, t in enumerate((do, ds)))
    x = [t.detach().double().requires_grad_(True) for t in leaves]
    want = torch.autograd.grad(oracle.decay_attention(*x[:3], lam, x[3]), x, (do.double(), ds.double()))
    a = [t.detach().abs().requires_grad_(True) for t in x]
    size = torch.autograd.grad(oracle.decay_attention(*a[:3], lam, a[3]), a, (do.double().abs(), ds.double().abs()))
    for i, name in enumerate(("dq", "dk", "dv", "dstate")):
        _check(got[i], want[i], size[i], 100, 64, name, name == "dstate")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,H", [(1, 1), (3, 5), (40, 12)])
def test_single_tokens(cuda0, B, H, D):
    from nexar_b200 import ops
    q, k, v, _, s0, _, lam = _inputs(cuda0, B, 1, H, D, 11)
    q, k, v = (t[:, 0] for t in (q, k, v))
    state = s0.clone()
    o = ops.decay_attention_step(q, k, v, lam, state)
    f32 = 2.0 ** -24
    decay = lam.double().exp().view(1, H, 1, 1)
    kv = k.double()[..., None] * v.double()[..., None, :]
    want = decay * s0.double() + kv
    size = decay * s0.double().abs() + kv.abs()
    oracle.assert_within(state, want, 4 * f32 * size, "state")  # the decay, two products and their sum in fp32
    ow = (q.double()[..., None, :] @ want)[..., 0, :] * D ** -0.5
    extra = (D + 8) * f32 * (q.double().abs()[..., None, :] @ size)[..., 0, :] * D ** -0.5
    half = oracle.half_step(torch.bfloat16)
    oracle.assert_within(o, ow, half * (ow.abs() + extra) + extra, "o")


def test_prompt_then_single_tokens(cuda0):
    """A prompt in one call, then token by token, is the whole sequence in one call."""
    from nexar_b200 import ops
    B, T, H, D = 2, 300, 4, 64
    q, k, v, _, _, _, lam = _inputs(cuda0, B, T, H, D, 12)
    whole, last = ops.decay_attention(q, k, v, lam, return_state=True)
    qkv = torch.stack([q, k, v], 2)
    o, state = ops.decay_attention_qkv(qkv[:, :290], lam, return_state=True)
    parts = [o]
    for t in range(290, T):
        parts.append(ops.decay_attention_step(*qkv[:, t].unbind(1), lam, state)[:, None])
    want, fin = oracle.decay_attention(q.double(), k.double(), v.double(), lam)
    osz, fsz = _sizes(q.double(), k.double(), v.double(), lam, None, None, None)
    for got, st in ((whole, last), (torch.cat(parts, 1), state)):
        _check(got, want, osz, T, D, "o")
        _check(st, fin, fsz, T, D, "state", True)


def test_repeats_and_graphs(cuda0):
    """The same bits again, also from captured graphs that live side by side and on another stream."""
    from nexar_b200 import ops
    q, k, v, do, s0, ds, lam = _inputs(cuda0, 1, 1200, 2, 64, 13)
    leaves = [t.requires_grad_(True) for t in (q, k, v, s0)]

    def run():
        o, f = ops.decay_attention(q, k, v, lam, s0, return_state=True)
        return [t.detach() for t in (o, f, *torch.autograd.grad((o, f), leaves, (do, ds)))]
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, run()))
    for g, _ in graphs:
        g.replay()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_step_marks_the_state_as_changed(cuda0):
    from nexar_b200 import ops
    q, k, v, do, s0, _, lam = _inputs(cuda0, 1, 10, 2, 64, 14)
    q.requires_grad_(True)
    o = ops.decay_attention(q, k, v, lam, state=s0)
    with torch.no_grad():
        ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], lam, s0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(o, q, do)


def test_second_derivatives_raise(cuda0):
    from nexar_b200 import ops
    q, k, v, do, s0, _, lam = _inputs(cuda0, 1, 10, 2, 64, 16)
    q.requires_grad_(True)
    first = torch.autograd.grad(ops.decay_attention(q, k, v, lam), q, do)[0]
    (g,) = torch.autograd.grad(ops.decay_attention(q, k, v, lam), q, do, create_graph=True)
    assert torch.equal(g.detach(), first)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.float().sum().backward()


def test_empty_and_refusals(cuda0):
    from nexar_b200 import ops
    q, k, v, _, s0, _, lam = _inputs(cuda0, 2, 8, 2, 64, 15)
    o, f = ops.decay_attention(q[:, :0], k[:, :0], v[:, :0], lam, state=s0, return_state=True)
    assert o.shape == (2, 0, 2, 64) and torch.equal(f, s0)
    assert not ops.decay_attention(q[:, :0], k[:, :0], v[:, :0], lam, return_state=True)[1].any()
    assert ops.decay_attention(q[:0], k[:0], v[:0], lam).shape == (0, 8, 2, 64)
    n = torch.tensor([1, 2], device=cuda0, dtype=torch.int32)
    bad = [lambda: ops.decay_attention(q.half(), k.half(), v.half(), lam), lambda: ops.decay_attention(q, k[:, :4], v, lam),
           lambda: ops.decay_attention(q[..., :32], k[..., :32], v[..., :32], lam),
           lambda: ops.decay_attention(q, k, v, lam.double()), lambda: ops.decay_attention(q, k, v, lam[:1]),
           lambda: ops.decay_attention(q, k, v, lam.cpu()), lambda: ops.decay_attention(q, k, v.cpu(), lam),
           lambda: ops.decay_attention(q, k, v, lam, state=s0.half()), lambda: ops.decay_attention(q, k, v, lam, state=s0[:1]),
           lambda: ops.decay_attention(q, k, v, lam, state=s0.transpose(2, 3)),
           lambda: ops.decay_attention(q, k, v, lam, lengths=n.long()), lambda: ops.decay_attention(q, k, v, lam, lengths=n[:1]),
           lambda: ops.decay_attention_step(q, k, v, lam, s0), lambda: ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], lam, s0[:1]),
           lambda: ops.decay_attention_step(q[:, 0], k[:, 0, :1], v[:, 0], lam, s0)]
    for f in bad:
        with pytest.raises(RuntimeError, match="nexar_b200"):
            f()


def test_inference_mode(cuda0):
    """Under inference_mode, on inference tensors, every operator gives what it gives outside."""
    from nexar_b200 import ops
    q, k, v, do, s0, ds, lam = _inputs(cuda0, 2, 70, 2, 64, 7)
    drop = ops.DropoutState(3, cuda0)
    w = torch.ones(64, dtype=torch.bfloat16, device=cuda0)

    def run():
        table = ops.rotary_table(70, 64, device=cuda0)
        a, b = ops.rotary_qk(q * 1, k * 1, table)
        o, s = ops.decay_attention(a, b, v, lam, return_state=True)
        t = ops.decay_attention_step(a[:, 0], b[:, 0], v[:, 0], lam, s)
        return (o, s, t, ops.dropout(o, 0.2, drop)) + ops.residual_layer_norm(o, v, w, w, p=0.1, dropout=drop)
    want = run()
    with torch.inference_mode():
        got = run()
    assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("D", [64, 128])
def test_long_chains_repeat_to_the_bit(cuda0, D):
    """Many chunks in a row with every place on the SMs taken: the order of the products inside a chunk may not depend
    on how long they take beside another block's."""
    from nexar_b200 import ops
    q, k, v, do, s0, ds, lam = _inputs(cuda0, 4, 1024, 80, D, 21)
    leaves = [t.requires_grad_(True) for t in (q, k, v, s0)]

    def call():
        o, f = ops.decay_attention(*leaves[:3], lam, state=leaves[3], return_state=True)
        return [o.detach(), f.detach(), *torch.autograd.grad((o, f), leaves, (do, ds))]
    first = call()
    for _ in range(6):
        for a, b in zip(first, call()):
            assert torch.equal(a, b)


def _parts(x, n):
    """x as n bf16 parts, each the rounding of what the ones before leave."""
    out = torch.zeros_like(x)
    for _ in range(n):
        out = out + (x - out).to(torch.bfloat16).double()
    return out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [2, 33, 64, 130])
def test_a_state_holds_fp32_values(cuda0, T, D):
    """One token per sequence has a key (a query, for the gradient of the first state), and its value (output
    gradient) is a power of two: a state is then one product, lam^x k 2^e, that only the roundings of its way can
    touch. Relative, in units of 2^-24: the power of the decay 1, its product with the key 1, what three bf16 parts
    leave 1/8, what the accumulator cuts off 2, and for each chunk behind the token 3 (the factor and two sums). Two
    parts leave up to 64, which the bound has to catch."""
    from nexar_b200 import ops
    B, H = 24, 4
    g = torch.Generator(device=cuda0).manual_seed(T + D)
    lam = torch.tensor([-0.0021, -0.0307, -0.011, -0.0043], device=cuda0)
    at = torch.randint(0, T, (B,), device=cuda0, generator=g)
    at[0], at[1] = 0, T - 1
    only = torch.zeros(B, T, 1, 1, device=cuda0)
    only[torch.arange(B, device=cuda0), at] = 1.0
    x = (only * torch.randn(B, T, H, D, device=cuda0, generator=g)).to(torch.bfloat16)
    two = torch.exp2(torch.randint(-3, 4, (B, T, H, D), device=cuda0, generator=g).float())
    two = (two * (1 - 2 * torch.randint(0, 2, two.shape, device=cuda0, generator=g))).to(torch.bfloat16)
    zero = torch.zeros_like(x)
    _, state = ops.decay_attention(zero, x, two, lam, return_state=True)
    s0 = torch.zeros(B, H, D, D, device=cuda0, requires_grad=True)
    o = ops.decay_attention(x, zero, zero, lam, state=s0, scale=0.25)
    (dstate,) = torch.autograd.grad(o, s0, two)
    row, val = (t.double()[torch.arange(B, device=cuda0), at] for t in (x, two))  # [B, H, D]
    chunks = -(-T // 64)
    bound = (4.125 + 3 * (chunks - 1)) * 2.0 ** -24
    for got, steps, scale, what in ((state, T - 1 - at, 1.0, "state"), (dstate, at + 1, 0.25, "dstate")):
        weight = scale * torch.exp(lam.double()[None] * steps.double()[:, None])[..., None]
        want = (row * weight)[..., :, None] * val[..., None, :]
        oracle.assert_within(got, want, bound * want.abs() + 1e-30, what)
        rough = _parts(row * weight, 2)[..., :, None] * val[..., None, :]
        assert ((rough - want).abs() > bound * want.abs()).any() or T == 2


def test_a_long_sum_has_no_bias(cuda0):
    """All keys and values positive, so that errors of one sign add up. Relative root mean square error of a head's
    state, in units of 2^-24: 2 x 13 for the cuts of a chunk's twelve accumulations and of its largest product, 3 for
    each of the 1 / (1 - lam^64) chunks that are left in the sum. One bf16 part for the decayed keys would leave
    about 2^-10.3 / sqrt(tokens left), 2^-15 and more."""
    from nexar_b200 import ops
    T, H, D = 3000, 4, 64
    q, k, v, _, _, _, _ = _inputs(cuda0, 2, T, H, D, 31)
    k, v = k.abs(), v.abs()
    lam = torch.tensor([-0.002, -0.03, -0.008, -0.1], device=cuda0)
    _, got = ops.decay_attention(q, k, v, lam, return_state=True)
    _, want = oracle.decay_attention(*(t.double() for t in (q, k, v)), lam)
    t = torch.arange(T, device=cuda0, dtype=torch.float64)
    end = (64 * (t // 64 + 1)).clamp(max=T) - 1  # of the token's chunk
    g = lam.double()[None, :, None]
    keys = _parts(k.double() * torch.exp(g * (end - t)[:, None, None]), 1) * torch.exp(g * (T - 1 - end)[:, None, None])
    rough = torch.einsum("bthi,bthj->bhij", keys, v.double())

    def error(x):
        return ((x.double() - want).square().sum((0, 2, 3)) / want.square().sum((0, 2, 3))).sqrt()
    bound = (26 + 3 / (1 - torch.exp(64 * lam.double()))) * 2.0 ** -24
    assert (error(got) <= bound).all(), error(got)
    assert (error(rough) > bound).all(), error(rough)


def _beside_ties(shape, dev, g):
    """fp32 values 2^-12 of half a bf16 step beside the middle between two bf16 neighbours, on either side, as the
    three bf16 numbers that add up to them. With the last 2^-12 lost a value is a tie, which rounds to the even
    neighbour, half of the time the wrong one."""
    base = 1 + torch.randint(0, 128, shape, device=dev, generator=g) / 128.0
    sign = 1.0 - 2.0 * torch.randint(0, 2, shape, device=dev, generator=g)
    tail = (1.0 - 2.0 * torch.randint(0, 2, shape, device=dev, generator=g)) * 2.0 ** -20
    power = torch.exp2(torch.randint(-6, 7, shape, device=dev, generator=g).float())
    return [sign * power * t for t in (base, torch.full_like(base, 2.0 ** -8), tail)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("path", ["scores", "state"])
@pytest.mark.parametrize("result", ["o", "dq", "dk", "dv"])
@pytest.mark.parametrize("T", [64, 150, 1000])
def test_outputs_are_rounded_once(cuda0, T, result, path, D):
    """Scores and states enter the bf16 results with all of their fp32 bits. Without decay and with one-hot rows each
    result is one score or one element of the state, exactly, so it has to be the nearest bf16 number."""
    from nexar_b200 import ops
    B, H = 2, 2
    g = torch.Generator(device=cuda0).manual_seed(T + D)
    zero = torch.zeros(B, T, H, D, device=cuda0)
    t = torch.arange(T, device=cuda0)
    hot = zero.clone()
    hot[:, t, :, t % D] = 1.0
    x = {n: zero for n in ("q", "k", "v", "do")}
    state = torch.zeros(B, H, D, D, device=cuda0)
    dstate = torch.zeros_like(state)
    if path == "state":
        s = sum(_beside_ties((B, H, D, D), cuda0, g))
        rows = {"o": "q", "dq": "do", "dk": "v", "dv": "k"}[result]  # one-hot: picks a row or a column of the state
        x[rows] = hot
        if result in ("o", "dq"):
            state = s
        else:
            dstate = s
        pick = s if result in ("o", "dv") else s.transpose(-1, -2)
        want = pick[:, :, t % D].transpose(1, 2)
    else:
        # the score of tokens i and j is the other token's value; tokens behind the 64th have none (one-hot rows end)
        n = 64
        value = _beside_ties((B, n, H), cuda0, g)
        ones, parts = zero.clone(), zero.clone()
        ones[..., :3] = 1.0
        for i, p in enumerate(value):
            parts[:, :n, :, i] = p
        hot[:, n:] = 0.0
        one, other, row = {"o": ("q", "k", "v"), "dq": ("do", "v", "k"), "dk": ("v", "do", "q"), "dv": ("k", "q", "do")}[result]
        x[one], x[other], x[row] = ones, parts, hot
        s = sum(value)  # [B, n, H]: at column j of every token that sees token j
        sees = (t[:, None] >= t[None, :n]) if result in ("o", "dq") else (t[:, None] <= t[None, :n])
        want = zero.clone()
        want[..., :n] = torch.where(sees[None, :, None], s.transpose(1, 2)[:, None], 0.0)
    leaves = [x[n].to(torch.bfloat16).requires_grad_(True) for n in ("q", "k", "v")]
    state.requires_grad_(True)
    o, f = ops.decay_attention(*leaves, torch.zeros(H, device=cuda0), state=state, scale=1.0, return_state=True)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad((o, f), leaves, (x["do"].to(torch.bfloat16), dstate))), o=o)[result]
    assert torch.equal(got.detach(), want.to(torch.bfloat16))
