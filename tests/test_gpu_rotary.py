"""Rotary positions on the GPU against the 64-bit rotation."""
import pytest
import torch

import decoder_oracle as oracle

pytestmark = pytest.mark.gpu


def _bound(x, y, m):
    # one rounding of the result (half a step; fp16 results below the normal range: half a subnormal step),
    # after fp32 products of x with cos and sin that are each one fp32 rounding (2^-24) off: at most
    # 4 such roundings of |x| m per term, two terms
    half = oracle.half_step(x.dtype)
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    wide = x.double().abs().amax(dim=-1, keepdim=True) * abs(m)
    slack = 8 * 2.0 ** -24 * wide
    return half * (y.abs() + slack) + slack + tiny


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,H,D,R", [(1, 1, 1, 2, 2), (2, 3, 5, 64, 64), (3, 17, 4, 80, 60), (1, 130, 12, 128, 96),
                                       (2, 5, 3, 33, 10), (1, 7, 2, 24, 20), (5, 64, 9, 32, 24)])
def test_rotary_matches_the_rotation(cuda0, B, T, H, D, R, dtype, layout):
    from nexar_b200 import ops
    g = torch.Generator(device=cuda0).manual_seed(D * T + H)
    x = torch.randn(B, T, H, D, device=cuda0, generator=g).to(dtype)
    freq, m = ops.rotary_frequencies(R)
    table = ops.rotary_table(T + 11, R, device=cuda0)
    for start in (0, 11):
        y = ops.rotary(x, table, start=start, layout=layout)
        want = oracle.rotate(x.double(), start + torch.arange(T, device=cuda0), freq, m, layout)
        assert y.dtype == dtype and y.is_contiguous()
        oracle.assert_within(y, want, _bound(x, want, m))


@pytest.mark.parametrize("kind,factor,length", oracle.SCALINGS)
def test_scaled_tables_at_far_positions(cuda0, kind, factor, length):
    """The angle of position 10^6 is right to fp32 of the cosine, not of the angle."""
    from nexar_b200 import ops
    sc = ops.RotaryScaling(kind, factor, length)
    freq, m = ops.rotary_frequencies(64, 500000.0, sc)
    table = ops.rotary_table(1_000_001, 64, 500000.0, sc, device=cuda0)
    pos = torch.tensor([0, 1, 4095, 131071, 999_999, 1_000_000], device=cuda0)
    cos, sin = oracle.angles(pos, freq, m)
    want = torch.stack([cos, sin], -1).flatten(-2)
    # fp32 rounding of a value up to m, and the 64-bit angle's own rounding (10^6 * 2^-52)
    oracle.assert_within(table[pos], want, torch.full_like(want, m * (2.0 ** -24 + 1e-9)))


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_positions_per_token(cuda0, index):
    from nexar_b200 import ops
    B, T, H, D = 3, 9, 4, 64
    g = torch.Generator(device=cuda0).manual_seed(1)
    x = torch.randn(B, T, H, D, device=cuda0, generator=g).to(torch.bfloat16)
    table = ops.rotary_table(50, D, device=cuda0)
    freq, m = ops.rotary_frequencies(D)
    pos = torch.randint(0, 50, (B, T), device=cuda0, generator=g).to(index)
    for p in (pos, pos[:1], pos[0], pos.t().contiguous().t(), pos[:1].expand(B, T)):
        y = ops.rotary(x, table, positions=p)
        want = oracle.rotate(x.double(), p.long(), freq, m, "half")
        oracle.assert_within(y, want, _bound(x, want, m))


def test_positions_outside_the_table_show_as_nan(cuda0):
    from nexar_b200 import ops
    x = torch.ones(4, 2, 8, device=cuda0)
    table = ops.rotary_table(3, 6, device=cuda0)
    y = ops.rotary(x, table, positions=torch.tensor([0, 3, -1, 1 << 40], device=cuda0))
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1:, :, :6]).all() and torch.equal(y[1:, :, 6:], x[1:, :, 6:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strided_heads_of_a_packed_projection(cuda0, layout):
    """Views of a packed projection, a padded one, an unaligned one and a transposed one."""
    from nexar_b200 import ops
    B, T, H, D = 2, 21, 6, 64
    g = torch.Generator(device=cuda0).manual_seed(2)
    base = torch.randn(B, T, 3 * H + 1, D + 3, device=cuda0, generator=g).to(torch.bfloat16)
    table = ops.rotary_table(T, 32, device=cuda0)
    freq, m = ops.rotary_frequencies(32)
    pos = torch.arange(T, device=cuda0)
    views = [base[:, :, :H, :D], base[:, :, H:2 * H, 3:], base[:, :, ::2, 1:D + 1],
             base.transpose(1, 2)[:, :T, :, :D].transpose(1, 2), base[..., :D].transpose(2, 3).contiguous().transpose(2, 3),
             base[:, :, :1, :D].expand(B, T, H, D)]
    for x in views:
        y = ops.rotary(x, table, layout=layout)
        want = oracle.rotate(x.double(), pos[:x.shape[1]], freq, m, layout)
        oracle.assert_within(y, want, _bound(x, want, m))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cut", [1, 2, 4])
def test_heads_at_any_address(cuda0, dtype, cut):
    """Rows that start `cut` elements behind an aligned address, with strides to match."""
    from nexar_b200 import ops
    g = torch.Generator(device=cuda0).manual_seed(cut)
    wide = torch.randn(2, 9, 4, 64 + cut, device=cuda0, generator=g).to(dtype)
    x = wide[..., cut:]
    flat = torch.empty(x.numel() + cut, dtype=dtype, device=cuda0)[cut:].view(2, 9, 4, 64).copy_(x)
    table = ops.rotary_table(16, 32, device=cuda0)
    want = ops.rotary(x.contiguous(), table, start=3)
    assert torch.equal(ops.rotary(x, table, start=3), want)
    assert torch.equal(ops.rotary(flat, table, start=3), want)


def test_pair_and_packed_forms_agree_with_the_single_one(cuda0):
    from nexar_b200 import ops
    B, T, H, Hk, D = 2, 33, 8, 2, 128
    g = torch.Generator(device=cuda0).manual_seed(3)
    qkv = torch.randn(B, T, H + 2 * Hk, D, device=cuda0, generator=g).to(torch.bfloat16)
    table = ops.rotary_table(T, 96, device=cuda0)
    q, k, v = qkv.split([H, Hk, Hk], 2)
    q1, k1 = ops.rotary_qk(q, k, table)
    assert torch.equal(q1, ops.rotary(q, table)) and torch.equal(k1, ops.rotary(k, table))
    packed = ops.rotary(qkv, table, heads=H + Hk)
    assert torch.equal(packed, torch.cat([q1, k1, v], 2))
    assert torch.equal(ops.rotary(qkv, table, heads=0), qkv)
    assert torch.equal(ops.rotary(qkv[0], table), ops.rotary(qkv, table)[0])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient(cuda0, layout):
    """The gradient is the formula's (the inverse turn), and agrees with differences of the 64-bit rotation."""
    from nexar_b200 import ops
    B, T, H, D = 2, 9, 3, 32
    g = torch.Generator(device=cuda0).manual_seed(4)
    sc = ops.RotaryScaling("yarn", 8.0, 64)
    freq, m = ops.rotary_frequencies(24, scaling=sc)
    table = ops.rotary_table(T, 24, scaling=sc, device=cuda0)
    q, k, dq, dk = (torch.randn(B, T, H, D, device=cuda0, generator=g) for _ in range(4))
    q.requires_grad_(True), k.requires_grad_(True)
    out = ops.rotary_qk(q, k, table, layout=layout)
    gq, gk = torch.autograd.grad(out, (q, k), (dq, dk), retain_graph=True)
    pos = torch.arange(T, device=cuda0)
    for x, got, d in ((q, gq, dq), (k, gk, dk)):
        want = oracle.rotate(d.double(), -pos, freq, m, layout)
        oracle.assert_within(got, want, _bound(d, want, m))
        way = torch.randn_like(x).double()
        diff = oracle.directional(lambda t: (oracle.rotate(t, pos, freq, m, layout) * d.double()).sum(),
                                  [x.detach().double()], [way])
        # linear in x: the difference has rounding error only
        assert (got.double() * way).sum().item() == pytest.approx(diff.item(), rel=1e-4, abs=1e-3)
    # one output unused, and a second derivative through the gradient
    assert torch.equal(torch.autograd.grad(out[1], k, dk, retain_graph=True)[0], gk)
    x, y = q.detach().requires_grad_(True), dq.clone().requires_grad_(True)
    (first,) = torch.autograd.grad(ops.rotary(x, table, layout=layout), x, y, create_graph=True)
    (second,) = torch.autograd.grad(first, y, dk)
    assert torch.equal(second, ops.rotary(dk, table, layout=layout))


def test_packed_gradient_copies_the_values(cuda0):
    from nexar_b200 import ops
    x = torch.randn(2, 5, 9, 64, device=cuda0).to(torch.bfloat16).requires_grad_(True)
    d = torch.randn(2, 5, 9, 64, device=cuda0).to(torch.bfloat16)
    table = ops.rotary_table(5, 64, device=cuda0)
    (gx,) = torch.autograd.grad(ops.rotary(x, table, heads=6), x, d)
    assert torch.equal(gx[:, :, 6:], d[:, :, 6:]) and not torch.equal(gx[:, :, :6], d[:, :, :6])


def test_rotary_empty_and_refusals(cuda0):
    from nexar_b200 import ops
    table = ops.rotary_table(8, 16, device=cuda0)
    assert ops.rotary(torch.zeros(2, 0, 3, 16, device=cuda0), table).shape == (2, 0, 3, 16)
    assert ops.rotary(torch.zeros(0, 4, 3, 16, device=cuda0), table).shape == (0, 4, 3, 16)
    x = torch.zeros(2, 8, 3, 16, device=cuda0)
    bad = [lambda: ops.rotary(x.double(), table), lambda: ops.rotary(x[0, 0], table),
           lambda: ops.rotary(x, table, start=1), lambda: ops.rotary(x, table, start=-1),
           lambda: ops.rotary(x[..., :8], table), lambda: ops.rotary(x, table.half()),
           lambda: ops.rotary(x, table[:, :15]), lambda: ops.rotary(x, table.t().contiguous().t()),
           lambda: ops.rotary(x, table, heads=4), lambda: ops.rotary(x, table.cpu()),
           lambda: ops.rotary(x, table, positions=torch.zeros(2, 7, dtype=torch.int64, device=cuda0)),
           lambda: ops.rotary(x, table, positions=torch.zeros(8, device=cuda0)),
           lambda: ops.rotary(x, table, positions=torch.zeros(8, dtype=torch.int64)),
           lambda: ops.rotary_qk(x, x[:, :4], table), lambda: ops.rotary_qk(x, x.half(), table)]
    for f in bad:
        with pytest.raises(RuntimeError, match="nexar_b200"):
            f()
    with pytest.raises(ValueError, match="gradient"):
        ops.rotary(x.clone().requires_grad_(True), table.clone().requires_grad_(True))


def test_rotary_on_a_stream_and_in_a_graph(cuda0):
    from nexar_b200 import ops
    x = torch.randn(2, 16, 4, 64, device=cuda0)
    table = ops.rotary_table(64, 64, device=cuda0)
    pos = torch.arange(16, device=cuda0)
    want = [ops.rotary(x, table, start=s) for s in (0, 40)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.rotary(x, table, positions=pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.rotary(x, table, positions=pos)
    graph.replay()
    assert torch.equal(y, want[0])
    pos.add_(40)
    graph.replay()
    assert torch.equal(y, want[1])
