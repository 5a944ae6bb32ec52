"""64-bit plain forms of the decoder-block operators, for the tests (CPU or GPU tensors)."""
import math

import torch


def angles(pos, freq, magnitude):
    a = pos.double()[..., None] * torch.tensor(freq, dtype=torch.float64, device=pos.device)
    return magnitude * a.cos(), magnitude * a.sin()


def rotate(x, pos, freq, magnitude, layout, heads=None):
    """x [..., T, H, D] fp64, pos [..., T]."""
    R, H = 2 * len(freq), x.shape[-2]
    heads = H if heads is None else heads
    cos, sin = (t[..., None, :] for t in angles(pos, freq, magnitude))
    head = x[..., :heads, :R]
    a, b = (head[..., :R // 2], head[..., R // 2:]) if layout == "half" else (head[..., 0::2], head[..., 1::2])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([torch.cat([turned, x[..., :heads, R:]], -1), x[..., heads:, :]], -2)


def philox_words(counter, key):
    """Philox4x32-10 of one counter (four words) and key (two words)."""
    c, k, low = list(counter), list(key), 0xFFFFFFFF
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & low, (p0 >> 32) ^ c[3] ^ k[1], p0 & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def dropout_keep(n, seed, step, site, p):
    """Bool [n]: the elements that the counter-based dropout keeps, and the factor on them."""
    low = 0xFFFFFFFF
    t = round(p * 65536)
    out = []
    for b in range(-(-n // 8)):
        for w in philox_words((b & low, b >> 32, site, step & low), (seed & low, seed >> 32 & low)):
            out += [(w & 0xFFFF) >= t, (w >> 16) >= t]
    scale = torch.tensor(65536.0 / (65536 - t) if t < 65536 else 0.0, dtype=torch.float64)
    return torch.tensor(out[:n]), scale.float().double().item()


def decay_attention(q, k, v, log_decay, state=None, lengths=None, scale=None):
    """(o, final state) from the written-out sums, fp64 [B, T, H, D] inputs."""
    B, T, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    t = torch.arange(T, device=q.device, dtype=torch.float64)
    n = torch.full((B,), T, device=q.device) if lengths is None else lengths.clamp(0, T)
    live = (t[None] < n[:, None])[:, :, None, None]
    q, k, v = (torch.where(live, x, torch.zeros_like(x)).transpose(1, 2) for x in (q, k, v))
    g = log_decay.double().view(1, H, 1, 1)
    gap = t[:, None] - t[None]
    w = torch.exp(g * gap.clamp(min=0)) * (gap >= 0)
    o = scale * ((q @ k.transpose(-1, -2)) * w) @ v
    left = torch.exp(g * (n.view(B, 1, 1, 1) - 1 - t.view(1, 1, T, 1)).clamp(min=0))
    final = (k * left).transpose(-1, -2) @ v
    if state is not None:
        o = o + scale * torch.exp(g * (t + 1).view(1, 1, T, 1)) * (q @ state)
        final = final + torch.exp(g * n.view(B, 1, 1, 1)) * state
    return o.transpose(1, 2), final


def residual_layer_norm_grads(s, w, ds, dy, keep_scale, eps=1e-5):
    """Gradients of s = x + keep_scale * r, y = LayerNorm(s) w + b at the stored s: a dict of values and of the
    sums of absolute terms that bound their fp32 errors."""
    mean = s.mean(-1, keepdim=True)
    rstd = ((s - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (s - mean) * rstd
    gw = dy * w
    dx = ds + rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    size = ds.abs() + rstd * (gw.abs() + gw.abs().mean(-1, keepdim=True) +
                              xh.abs() * (gw * xh).abs().mean(-1, keepdim=True))
    dr = dx * keep_scale
    return dict(xh=xh, dx=dx, dx_size=size, dr=dr, dr_size=size * keep_scale, dw=(dy * xh).sum(0),
                dw_size=(dy * xh).abs().sum(0), db=dy.sum(0), db_size=dy.abs().sum(0), drb=dr.sum(0),
                drb_size=dr.abs().sum(0))


def half_step(dtype):
    """Largest relative error of one rounding to nearest in ``dtype``."""
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound element by element (fp64), with the worst offender in the message."""
    over = (got.double() - want).abs() - bound
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert not torch.isnan(over).any(), f"{what}: NaN"
    i = int(over.flatten().argmax()) if over.numel() else 0
    assert over.numel() == 0 or over.flatten()[i] <= 0, (
        f"{what}: {got.flatten()[i].item()} against {want.flatten()[i].item()}, bound {bound.flatten()[i].item():.3g}")


def directional(loss, inputs, directions, h=1e-4):
    """Central difference of loss(*inputs) along ``directions``."""
    up = loss(*(x + h * d for x, d in zip(inputs, directions)))
    down = loss(*(x - h * d for x, d in zip(inputs, directions)))
    return (up - down) / (2 * h)


SCALINGS = [("linear", 4.0, 2048), ("ntk", 4.0, 2048), ("bands", 8.0, 8192), ("yarn", 16.0, 4096)]
PI = math.pi
