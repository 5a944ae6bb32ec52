"""Counter-based dropout, alone and inside the residual add + LayerNorm, against 64-bit plain forms."""
import pytest
import torch

import decoder_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 4099])
@pytest.mark.parametrize("p,seed,step,site", [(0.1, 5, 0, 0), (0.5, -3, 17, 9), (0.999, 1 << 40, (1 << 32) + 1, (1 << 32) - 1)])
def test_dropout_draws_the_published_generator(cuda0, n, dtype, p, seed, step, site):
    from nexar_b200 import ops
    x = torch.randn(n, device=cuda0, generator=torch.Generator(device=cuda0).manual_seed(n)).to(dtype).requires_grad_(True)
    state = ops.DropoutState(seed, cuda0, step)
    keep, scale = oracle.dropout_keep(n, seed & ((1 << 64) - 1), step, site, p)
    keep = keep.to(cuda0)
    # one fp32 product, one rounding: exactly these values
    want = torch.where(keep, x.detach().float() * scale, 0.0).to(dtype)
    y = ops.dropout(x, p, state, site)
    assert torch.equal(y, want)
    d = torch.randn(n, device=cuda0).to(dtype)
    state.advance()  # the backward uses the numbers of the forward, not the current ones
    (gx,) = torch.autograd.grad(y, x, d)
    assert torch.equal(gx, torch.where(keep, d.float() * scale, 0.0).to(dtype))


def test_dropout_layouts_and_far_blocks(cuda0):
    """Draws go by the element's place in the tensor, whatever its strides and alignment."""
    from nexar_b200 import ops
    state = ops.DropoutState(11, cuda0)
    x = torch.randn(65, 37, device=cuda0).to(torch.bfloat16)
    y = ops.dropout(x, 0.3, state)
    assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.3, state), y)
    shifted = torch.empty(65 * 37 + 1, device=cuda0, dtype=torch.bfloat16)[1:].view(65, 37).copy_(x)
    assert torch.equal(ops.dropout(shifted, 0.3, state), y)
    assert torch.equal(ops.dropout(x[:1].expand(4, 37), 0.3, state), ops.dropout(x[:1].expand(4, 37).contiguous(), 0.3, state))
    assert ops.dropout(x[:0], 0.3, state).shape == (0, 37)
    big = torch.ones(3, 1 << 20, device=cuda0, dtype=torch.bfloat16)  # more blocks than one sweep of the grid
    got = ops.dropout(big, 0.3, state).flatten()
    at = 3 * (1 << 20) - 64
    t = round(0.3 * 65536)
    for b in range(at // 8, at // 8 + 8):
        words = oracle.philox_words((b, 0, 0, 0), (11, 0))
        draws = [h for w in words for h in (w & 0xFFFF, w >> 16)]
        assert [v != 0 for v in got[8 * b:8 * b + 8].tolist()] == [d >= t for d in draws]


def test_dropout_ends_of_the_range_and_infinities(cuda0):
    from nexar_b200 import ops
    state = ops.DropoutState(3, cuda0)
    x = torch.randn(1000, device=cuda0)
    assert torch.equal(ops.dropout(x, 0.0, state), x)
    assert torch.equal(ops.dropout(x, 1.0, state), torch.zeros_like(x))
    bad = torch.full((1000,), float("inf"), device=cuda0)
    bad[1::2] = float("nan")
    y = ops.dropout(bad, 0.5, state)
    keep = oracle.dropout_keep(1000, 3, 0, 0, 0.5)[0].to(cuda0)
    assert (y[~keep] == 0).all() and not torch.isfinite(y[keep]).any()


def test_dropout_rate_and_mean(cuda0):
    from nexar_b200 import ops
    n = 1 << 22
    y = ops.dropout(torch.ones(n, device=cuda0), 0.1, ops.DropoutState(2024, cuda0))
    kept = (y != 0).double().mean().item()
    # a binomial share of n draws: six standard deviations
    assert abs(kept - (1 - round(0.1 * 65536) / 65536)) < 6 * (0.09 / n) ** 0.5
    assert len({tuple((ops.dropout(torch.ones(64, device=cuda0), 0.5, ops.DropoutState(s, cuda0, t), i) != 0).tolist())
                for s in (0, 1) for t in (0, 1) for i in (0, 1)}) == 8


def test_dropout_in_a_graph_draws_anew(cuda0):
    from nexar_b200 import ops
    state = ops.DropoutState(8, cuda0)
    x = torch.randn(512, device=cuda0).requires_grad_(True)
    d = torch.ones(512, device=cuda0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.dropout(x, 0.5, state), x, d)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.dropout(x, 0.5, state)
        (gx,) = torch.autograd.grad(y, x, d)
        state.advance()
    for step in range(3):
        graph.replay()
        keep = oracle.dropout_keep(512, 8, step, 0, 0.5)[0].to(cuda0)
        assert torch.equal(y != 0, keep & (x != 0)) and torch.equal(gx != 0, keep)
    assert state.tensor.tolist() == [8, 3]


# ---------------------------------------------------------------- residual add + dropout + LayerNorm
def _inputs(dev, R, C, bias, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    bf = torch.bfloat16
    x, r, ds, dy = (torch.randn(R, C, device=dev, generator=g).to(bf) for _ in range(4))
    w = (1 + 0.1 * torch.randn(C, device=dev, generator=g)).to(bf)
    b, rb = ((0.1 * torch.randn(C, device=dev, generator=g)).to(bf) for _ in range(2))
    return x, r, ds, dy, w, b, (rb if bias else None)


@pytest.mark.parametrize("R,C", [(1, 8), (3, 64), (37, 768), (16, 1024), (5, 1336), (9, 2048), (1500, 256), (2500, 40)])
@pytest.mark.parametrize("bias", [True, False])
def test_residual_dropout_layer_norm(cuda0, R, C, bias):
    from nexar_b200 import ops
    p, seed, step, site = 0.2, 77, 4, 2
    x, r, ds, dy, w, b, rb = _inputs(cuda0, R, C, bias)
    state = ops.DropoutState(seed, cuda0, step)
    leaves = [t.requires_grad_(True) for t in (x, r, w, b) + ((rb,) if bias else ())]
    s, y = ops.residual_layer_norm(x, r, w, b, 1e-5, rbias=rb, p=p, dropout=state, site=site)
    state.advance()
    grads = torch.autograd.grad((s, y), leaves, (ds, dy))
    # the same elements as the plain dropout's draws
    ones = torch.ones(R, C, device=cuda0)
    kept = ops.dropout(ones, p, ops.DropoutState(seed, cuda0, step), site).double()
    if R * C <= 50000:
        keep, scale = oracle.dropout_keep(R * C, seed, step, site, p)
        assert torch.equal(kept, keep.to(cuda0).view(R, C).double() * scale)
    half, f32 = oracle.half_step(torch.bfloat16), 2.0 ** -24
    xd, rd, wd, bd = (t.detach().double() for t in (x, r, w, b))
    branch = rd + (rb.detach().double() if bias else 0.0)
    total = xd + kept * branch
    size = xd.abs() + kept * (rd.abs() + (rb.detach().double().abs() if bias else 0.0))
    # s: up to three fp32 roundings, then one to bf16
    oracle.assert_within(s, total, half * (total.abs() + 4 * f32 * size) + 4 * f32 * size, "s")
    # the norm is that of the stored s. mean and variance: sums of C fp32 terms over 256 lanes' partial sums
    # (C / 32 + 5 additions), approximate reciprocal square root and division (2^-22): fp32 relative error `e` of
    # every factor; five factors and terms
    e = (C / 32 + 16) * f32 + 4 * 2.0 ** -22
    sd = s.detach().double()
    want = oracle.residual_layer_norm_grads(sd, wd, ds.double(), dy.double(), kept)
    var_size = sd.abs().amax(-1, keepdim=True) / sd.var(-1, unbiased=False, keepdim=True).add(1e-5).sqrt()
    slack = 8 * e * (1 + var_size)  # an error of the mean is relative to the largest value, in units of the deviation
    yw = want["xh"] * wd + bd
    ysz = (want["xh"].abs() + 1) * wd.abs() + bd.abs()
    oracle.assert_within(y, yw, half * (yw.abs() + slack * ysz) + slack * ysz, "y")
    for name, got in (("dx", grads[0]), ("dr", grads[1])):
        extra = 2 * slack * (want[name + "_size"] + (kept if name == "dr" else 1.0))
        oracle.assert_within(got, want[name], half * (want[name].abs() + extra) + extra, name)
    # column sums: R fp32 terms
    names = ["dw", "db"] + (["drb"] if bias else [])
    for name, got in zip(names, grads[2:]):
        sz = want[name + "_size"]
        extra = R * f32 * sz
        if name == "dw":
            extra = extra + (slack * (dy.double().abs() * (want["xh"].abs() + 1))).sum(0)
        if name == "drb":
            extra = extra + (2 * slack * (want["dr_size"] + kept)).sum(0)
        oracle.assert_within(got, want[name], half * (want[name].abs() + extra) + extra, name)


def test_residual_gradient_against_differences(cuda0):
    from nexar_b200 import ops
    R, C, p = 6, 48, 0.25
    x, r, ds, dy, w, b, rb = _inputs(cuda0, R, C, True, 5)
    state = ops.DropoutState(1, cuda0)
    kept = ops.dropout(torch.ones(R, C, device=cuda0), p, state).double()

    def loss(x, r, w, b, rb):
        s = x + kept * (r + rb)
        y = (s - s.mean(-1, keepdim=True)) / (s.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * w + b
        return (s * ds.double()).sum() + (y * dy.double()).sum()
    leaves = [t.requires_grad_(True) for t in (x, r, w, b, rb)]
    grads = torch.autograd.grad(ops.residual_layer_norm(x, r, w, b, 1e-5, rbias=rb, p=p, dropout=state), leaves, (ds, dy))
    at = [t.detach().double() for t in leaves]
    for i, got in enumerate(grads):
        way = [torch.randn_like(t) if j == i else torch.zeros_like(t) for j, t in enumerate(at)]
        want = oracle.directional(loss, at, way)
        # gradients are rounded to bf16 (2^-8 each, also the s they are taken at): the inner product's error is at
        # most that share of the sum of absolute terms, with a factor for the derivative at the rounded s
        size = (got.double().abs() * way[i].abs()).sum()
        assert abs((got.double() * way[i]).sum() - want) <= 8 * 2.0 ** -8 * size, i


def test_residual_partial_gradients_and_rerun(cuda0):
    from nexar_b200 import ops
    x, r, ds, dy, w, b, rb = _inputs(cuda0, 200, 768, True, 6)
    leaves = [t.requires_grad_(True) for t in (x, r, w, b, rb)]
    state = ops.DropoutState(4, cuda0)

    def run(outs):
        s, y = ops.residual_layer_norm(x, r, w, b, 1e-5, rbias=rb, p=0.1, dropout=state)
        return torch.autograd.grad([(s, y)[i] for i in outs], leaves, [(ds, dy)[i] for i in outs], allow_unused=True)
    both, again = run((0, 1)), run((0, 1))
    assert all(torch.equal(a, c) for a, c in zip(both, again))  # no atomics: the same bits
    only_y = run((1,))
    zeros = torch.zeros_like(ds)
    s, y = ops.residual_layer_norm(x, r, w, b, 1e-5, rbias=rb, p=0.1, dropout=state)
    for a, c in zip(only_y, torch.autograd.grad((s, y), leaves, (zeros, dy))):
        assert torch.equal(a, c)
    only_s = run((0,))
    assert torch.equal(only_s[0], ds) and not only_s[2].any()


def test_residual_gradients_at_any_address(cuda0):
    from nexar_b200 import ops
    x, r, ds, dy, w, b, rb = _inputs(cuda0, 20, 64, True, 8)
    leaves = [t.requires_grad_(True) for t in (x, r, w, b, rb)]
    state = ops.DropoutState(4, cuda0)

    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda0)
        flat[1:] = t.reshape(-1)
        return flat[1:].view_as(t)

    def run(a, c):
        return torch.autograd.grad(ops.residual_layer_norm(x, r, w, b, 1e-5, rbias=rb, p=0.1, dropout=state), leaves, (a, c))
    assert all(torch.equal(a, c) for a, c in zip(run(ds, dy), run(moved(ds), moved(dy))))


@pytest.mark.parametrize("C", [64, 256, 1024, 2048])
def test_residual_constant_rows(cuda0, C):
    """Rows of one value each, far from zero: nothing is left of them after the mean, so dw is exactly 0 and dx is
    that of a norm at its mean. (The sums of C equal bf16 values and the division by a power of two are exact.)"""
    from nexar_b200 import ops
    R = 40
    g = torch.Generator(device=cuda0).manual_seed(C)
    x = (torch.randn(R, 1, device=cuda0, generator=g) * 1000).to(torch.bfloat16).expand(R, C).contiguous()
    _, _, ds, dy, w, b, _ = _inputs(cuda0, R, C, False, 3)
    leaves = [x.requires_grad_(True), torch.zeros_like(x).requires_grad_(True), w.requires_grad_(True), b]
    s, y = ops.residual_layer_norm(*leaves, 1e-5, p=0.2, dropout=ops.DropoutState(3, cuda0))
    dx, dw = torch.autograd.grad((s, y), (leaves[0], w), (ds, dy))
    assert torch.equal(s, x) and torch.equal(y, b.expand(R, C))
    assert torch.count_nonzero(dw) == 0
    # dx = ds + rstd (gw - mean gw): C products and sums in fp32, rstd by an approximate root, rounded once
    gw = dy.double() * w.detach().double()
    rstd, f32, half = 1e-5 ** -0.5, 2.0 ** -24, oracle.half_step(torch.bfloat16)
    want = ds.double() + rstd * (gw - gw.mean(-1, keepdim=True))
    extra = ((C / 32 + 16) * f32 + 4 * 2.0 ** -22) * (ds.double().abs() + rstd * (gw.abs() + gw.abs().mean(-1, keepdim=True)))
    oracle.assert_within(dx, want, half * (want.abs() + extra) + extra, "dx")


@pytest.mark.parametrize("sinks", [False, True])
def test_residual_tensors_at_any_address(cuda0, sinks):
    from nexar_b200 import ops

    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda0)
        flat[1:] = t.reshape(-1)
        return flat[1:].view_as(t)

    def strided(t):
        return torch.stack([t, t + 1], -1)[..., 0]

    def run(how):
        x, r, ds, dy, w, b, rb = (how(t).detach() for t in _inputs(cuda0, 20, 64, True, 8))
        leaves = [t.requires_grad_(True) for t in (x, r, w, b, rb)]
        if sinks:
            for t in (w, b, rb):
                t.main_grad = torch.empty(64, dtype=t.dtype, device=cuda0)
        out = ops.residual_layer_norm(x, r, w, b, 1e-5, rbias=rb, p=0.1, dropout=ops.DropoutState(4, cuda0))
        got = torch.autograd.grad(out, leaves, (ds, dy), allow_unused=True)
        return [*out, *got[:2], *([t.main_grad for t in (w, b, rb)] if sinks else got[2:])]
    want = run(lambda t: t)
    for how in (moved, strided):
        for a, c in zip(want, run(how)):
            assert torch.equal(a, c)


def test_residual_without_dropout_is_unchanged(cuda0):
    from nexar_b200 import ops
    x, r, ds, dy, w, b, rb = _inputs(cuda0, 64, 768, True)
    plain = ops.residual_layer_norm(x, r, w, b, 1e-5, rbias=rb)
    off = ops.residual_layer_norm(x, r, w, b, 1e-5, rbias=rb, p=0.0, dropout=ops.DropoutState(1, cuda0))
    assert all(torch.equal(a, c) for a, c in zip(plain, off))


def test_residual_writes_gradient_sinks(cuda0):
    from nexar_b200 import ops
    x, r, ds, dy, w, b, rb = _inputs(cuda0, 100, 256, True)
    want = None
    for sink in (False, True):
        ps = [torch.nn.Parameter(t.detach().clone()) for t in (w, b, rb)]
        told = []
        if sink:
            for i, q in enumerate(ps):
                q.main_grad = torch.full_like(q, 7.0)
                q._nexar_on_ready = lambda i=i: told.append(i)
        s, y = ops.residual_layer_norm(x, r, ps[0], ps[1], 1e-5, rbias=ps[2], p=0.1, dropout=ops.DropoutState(9, cuda0))
        torch.autograd.backward((s, y), (ds, dy))
        got = [q.main_grad if sink else q.grad for q in ps]
        if sink:
            assert sorted(told) == [0, 1, 2] and all(q.grad is None for q in ps)
            assert all(torch.equal(a, c) for a, c in zip(got, want))
        want = got


def test_dropout_refusals(cuda0):
    from nexar_b200 import ops
    state = ops.DropoutState(1, cuda0)
    x = torch.zeros(4, 16, device=cuda0, dtype=torch.bfloat16)
    w = torch.ones(16, device=cuda0, dtype=torch.bfloat16)
    wide = torch.zeros(2, 2056, device=cuda0, dtype=torch.bfloat16)
    bad = [lambda: ops.dropout(x.double(), 0.1, state), lambda: ops.dropout(x, 0.1, state, site=-1),
           lambda: ops.dropout(x, 0.1, state, site=1 << 32), lambda: ops.dropout(x, 0.1, ops.DropoutState(1, "cpu")),
           lambda: ops.residual_layer_norm(x.float(), x.float(), w, w, p=0.1, dropout=state),
           lambda: ops.residual_layer_norm(x[:, :12], x[:, :12], w[:12], w[:12], p=0.1, dropout=state),
           lambda: ops.residual_layer_norm(wide, wide, wide[0], wide[0], p=0.1, dropout=state),
           lambda: ops.residual_layer_norm(x, x, w[:8], w, p=0.1, dropout=state),
           lambda: ops.residual_layer_norm(x, x, w, w.cpu(), p=0.1, dropout=state)]
    for f in bad:
        with pytest.raises(RuntimeError, match="nexar_b200"):
            f()
