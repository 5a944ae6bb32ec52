"""Decoder-block operators on tensors of more than 2^31 elements, and on streams and graphs side by side."""
import pytest
import torch

import decoder_oracle as oracle

pytestmark = pytest.mark.gpu


def _needs(gigabytes):
    free, _ = torch.cuda.mem_get_info()
    if free < gigabytes * 2 ** 30:
        pytest.skip(f"needs {gigabytes} GB of GPU memory")


def test_rotary_past_32_bit_offsets(cuda0):
    from nexar_b200 import ops
    _needs(12)
    T, H, D = 65552, 256, 128  # 2^31 + 524288 elements
    x = torch.empty(1, T, H, D, dtype=torch.bfloat16, device=cuda0)
    x[:, -3:].normal_()
    x[:, :3].normal_()
    table = ops.rotary_table(T, D, device=cuda0)
    y = ops.rotary(x, table, heads=200)
    for part in (slice(0, 3), slice(T - 3, T)):
        pos = torch.arange(T, device=cuda0)[part]
        assert torch.equal(y[:, part], ops.rotary(x[:, part], table, positions=pos, heads=200))
    # element by element where the alignment allows nothing wider
    odd = x.view(-1)[1:1 + (T - 1) * H * D].view(1, T - 1, H, D)
    z = ops.rotary(odd, table, layout="interleaved")
    assert torch.equal(z[:, -2:], ops.rotary(odd[:, -2:], table, positions=torch.arange(T - 3, T - 1, device=cuda0),
                                             layout="interleaved"))


def test_dropout_past_32_bit_offsets(cuda0):
    from nexar_b200 import ops
    _needs(12)
    n = (1 << 31) + 13
    x = torch.ones(n, dtype=torch.bfloat16, device=cuda0)
    y = ops.dropout(x, 0.25, ops.DropoutState(6, cuda0))
    first = (n - 13) // 8
    t = round(0.25 * 65536)
    for b in (first, first + 1):
        draws = [h for w in oracle.philox_words((b, 0, 0, 0), (6, 0)) for h in (w & 0xFFFF, w >> 16)]
        got = y[8 * b:8 * b + 8].tolist()
        assert [v != 0 for v in got] == [d >= t for d in draws][:len(got)]
    assert abs((y[: 1 << 28] != 0).float().mean().item() - 0.75) < 1e-3


def test_decay_attention_past_32_bit_offsets(cuda0):
    """The last tokens of a tensor of 2^31 elements, from the state of the tokens before them."""
    from nexar_b200 import ops
    _needs(24)
    T, H, D = 131136, 128, 128
    g = torch.Generator(device=cuda0).manual_seed(1)
    q, k, v = (torch.empty(1, T, H, D, dtype=torch.bfloat16, device=cuda0).normal_(generator=g) for _ in range(3))
    lam = -torch.rand(H, device=cuda0, generator=g) * 0.05
    cut = T - 100
    o, fin = ops.decay_attention(q, k, v, lam, return_state=True)
    _, mid = ops.decay_attention(q[:, :cut], k[:, :cut], v[:, :cut], lam, return_state=True)
    tail = [t[:, cut:] for t in (q, k, v)]
    want, wf = oracle.decay_attention(*(t.double() for t in tail), lam, mid.double())
    size, fs = oracle.decay_attention(*(t.double().abs() for t in tail), lam, mid.double().abs())
    # one rounding to bf16, and the bounds of the split operands and fp32 sums over 100 tokens
    extra = size * 2.0 ** -13
    oracle.assert_within(o[:, cut:], want, 2.0 ** -8 * (want.abs() + extra) + extra, "o")
    oracle.assert_within(fin, wf, fs * 2.0 ** -15, "state")


def test_operators_on_streams_side_by_side(cuda0):
    """The same calls on four streams at once give what they give one after the other."""
    from nexar_b200 import ops
    g = torch.Generator(device=cuda0).manual_seed(2)
    jobs = []
    for i in range(4):
        x = torch.randn(1, 700, 9, 64, device=cuda0, generator=g).to(torch.bfloat16).requires_grad_(True)
        lam = torch.full((3,), -0.01 * (i + 1), device=cuda0)
        jobs.append((x, lam, ops.rotary_table(700, 64, device=cuda0), ops.DropoutState(i, cuda0),
                     torch.randn(1, 700, 3, 64, device=cuda0, generator=g).to(torch.bfloat16)))

    def run(x, lam, table, state, do):
        qkv = ops.rotary(x, table, heads=6).view(1, 700, 3, 3, 64)
        o = ops.dropout(ops.decay_attention_qkv(qkv, lam), 0.2, state)
        return o.detach(), torch.autograd.grad(o, x, do)[0]
    want = [run(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for s, j in zip(streams, jobs):
        with torch.cuda.stream(s):
            got.append(run(*j))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    from nexar_b200 import _native
    assert _native.cuda().decay_error_flag() == 0
