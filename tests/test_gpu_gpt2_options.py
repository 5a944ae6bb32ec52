"""GPT-2 with rotary positions, dropout and the decay mixer together: against a plain fp32 model with the same masks,
in a captured step, and across a checkpoint."""
import dataclasses

import pytest
import torch
import torch.nn.functional as F

import decoder_oracle as oracle
from nexar_b200 import ops
from nexar_b200.models.gpt2 import GPT2, GPT2Config
from nexar_b200.parallel.dp import DataParallelTrainer

gpu = pytest.mark.gpu


def _config(**kw):
    return GPT2Config(**{**dict(n_layer=2, n_head=2, n_embd=128, vocab_size=1000, padded_vocab=1024, block_size=96), **kw})


OPTIONS = [dict(positions="rotary"), dict(dropout=0.2), dict(mixer="decay"),
           dict(positions="rotary", dropout=0.1, mixer="decay")]


def _keep(cfg, shape, seed, step, site, device):
    """Factors of the model's dropout calls: draws of the published generator."""
    n = shape[0] * shape[1]
    keep, scale = oracle.dropout_keep(n, seed, step, site, cfg.dropout)
    return (keep.double() * scale).view(shape).to(device).float()


def _reference(cfg, p, idx, tgt, seed, step, drop=True):
    """The model written out in fp32 (rotations and decays in 64 bits)."""
    B, T = idx.shape
    C, H = cfg.n_embd, cfg.n_head
    hd = C // H
    dev = idx.device

    def dropped(x, site):
        return x * _keep(cfg, (B * T, C), seed, step, site, dev) if cfg.dropout and drop else x
    x = p["wte"][idx].view(B * T, C)
    if cfg.positions == "learned":
        x = x + p["wpe"][:T].repeat(B, 1)
    x = dropped(x, 0)
    for l in range(cfg.n_layer):
        q = f"h{l}."
        h = F.layer_norm(x, (C,), p[q + "ln1.w"], p[q + "ln1.b"])
        qkv = (h @ p[q + "attn.w"].t() + p[q + "attn.b"]).view(B, T, 3, H, hd)
        if cfg.positions == "rotary":
            freq, m = ops.rotary_frequencies(hd)
            turned = oracle.rotate(qkv[:, :, :2].reshape(B, T, 2 * H, hd).double(), torch.arange(T, device=dev), freq, m, "half")
            qkv = torch.cat([turned.float().view(B, T, 2, H, hd), qkv[:, :, 2:]], 2)
        qq, kk, vv = qkv.unbind(2)
        if cfg.mixer == "decay":
            lam = torch.log1p(-torch.exp2(-(5.0 + torch.arange(H, device=dev, dtype=torch.float64))))
            y = oracle.decay_attention(qq.double(), kk.double(), vv.double(), lam)[0].float()
            y = F.layer_norm(y, (hd,), p[q + "head_norm.w"], p[q + "head_norm.b"])
        else:
            y = F.scaled_dot_product_attention(qq.transpose(1, 2), kk.transpose(1, 2), vv.transpose(1, 2),
                                               is_causal=True).transpose(1, 2)
        x = x + dropped(y.reshape(B * T, C) @ p[q + "proj.w"].t() + p[q + "proj.b"], 1 + 2 * l)
        h = F.layer_norm(x, (C,), p[q + "ln2.w"], p[q + "ln2.b"])
        f = F.gelu(h @ p[q + "fc.w"].t() + p[q + "fc.b"], approximate="tanh")
        x = x + dropped(f @ p[q + "fcproj.w"].t() + p[q + "fcproj.b"], 2 + 2 * l)
    h = F.layer_norm(x, (C,), p["lnf.w"], p["lnf.b"])
    return F.cross_entropy((h @ p["wte"].t())[:, :cfg.vocab_size], tgt.reshape(-1))


@gpu
@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(o))
def test_loss_and_gradients_match_the_plain_model(cuda0, options):
    cfg = _config(**options)
    m = GPT2(cfg, cuda0, seed=6)
    g = torch.Generator(device=cuda0).manual_seed(3)
    with torch.no_grad():  # biases and norms away from their initial values
        for name, p in m.p.items():
            if name.endswith(".b"):
                p.copy_(0.05 * torch.randn(p.shape, device=cuda0, generator=g))
            elif "norm" in name or ".ln" in name or name.startswith("lnf"):
                p.copy_(1 + 0.1 * torch.randn(p.shape, device=cuda0, generator=g))
        m.flat.grad.fill_(7.0)  # stale values must be overwritten
    if cfg.dropout:
        m.dropout_state.set(6, 11)
    idx = torch.randint(0, cfg.vocab_size, (2, 96), device=cuda0, generator=g)
    tgt = torch.randint(0, cfg.vocab_size, (2, 96), device=cuda0, generator=g)
    loss = m(idx, tgt, unit_grad=True)
    loss.backward()
    p = {k: v.detach().float().requires_grad_(True) for k, v in m.p.items()}
    ref = _reference(cfg, p, idx, tgt, 6, 11)
    ref.backward()
    # bf16 activations through two layers: the same bounds as the model without options
    assert abs(loss.item() - ref.item()) < 0.05
    bad = []
    for name in m.p:
        ours, want = m.flat.view(m.flat.grad, name).float(), p[name].grad
        err = ((ours - want).norm() / (want.norm() + 1e-6)).item()
        if not err < 0.05:
            bad.append((name, round(err, 4)))
    assert not bad, bad
    m.eval()  # no dropout outside training
    with torch.no_grad():
        ref = _reference(cfg, p, idx, tgt, 6, 11, drop=False)
        assert abs(m(idx, tgt).item() - ref.item()) < 0.05


@gpu
def test_captured_steps_draw_what_eager_steps_draw(cuda0):
    cfg = _config(positions="rotary", dropout=0.3, mixer="decay")
    g = torch.Generator().manual_seed(1)
    idx = torch.randint(0, cfg.vocab_size, (2, 96), generator=g)
    tgt = torch.randint(0, cfg.vocab_size, (2, 96), generator=g)
    losses = []
    for graph in (False, True):
        # lr 0: the weights stay, so the losses differ by their masks alone
        tr = DataParallelTrainer(cfg, 2, 96, use_cuda_graph=graph, seed=5, lr=0.0)
        tr.set_batch(idx, tgt)
        tr.capture(warmup=3)
        tr.model.dropout_state.set(5, 3)
        losses.append([tr.step(idx, tgt) for _ in range(3)])
        assert tr.model.dropout_state.tensor.tolist() == [5, 6]
    assert losses[0] == pytest.approx(losses[1], rel=1e-5) and len(set(losses[0])) == 3


@gpu
def test_checkpoint_carries_the_generator(cuda0, tmp_path):
    cfg = _config(dropout=0.2)
    g = torch.Generator().manual_seed(2)
    batch = lambda: [torch.randint(0, cfg.vocab_size, (2, 96), generator=g) for _ in range(2)]  # noqa: E731
    a = DataParallelTrainer(cfg, 2, 96, use_cuda_graph=False, seed=9)
    a.step(*batch())
    path = str(tmp_path / "d.pt")
    a.save(path)
    b = DataParallelTrainer(cfg, 2, 96, use_cuda_graph=False, seed=1)
    b.load(path)
    assert torch.equal(a.model.dropout_state.tensor, b.model.dropout_state.tensor)
    x = batch()
    assert a.step(*x) == pytest.approx(b.step(*x), rel=1e-5)
    # a checkpoint from before the options existed loads into a model without them
    plain = DataParallelTrainer(_config(), 2, 96, use_cuda_graph=False)
    sd = plain.state_dict()
    for k in ("dropout", "positions", "mixer"):
        del sd["config"][k]
    del sd["dropout"]
    plain.load_state_dict(sd)
    with pytest.raises(ValueError, match="model"):
        a.load_state_dict(sd)


@pytest.mark.parametrize("bad", [dict(positions="none"), dict(mixer="mlp"), dict(dropout=1.0), dict(dropout=-0.1),
                                 dict(mixer="decay", n_head=4)])
def test_configuration_refusals(bad):
    with pytest.raises(ValueError):
        GPT2(_config(**bad), "cpu")


def test_workspaces_belong_to_their_call():
    from nexar_b200.ops import functional
    a, b = functional._workspace("cpu", 16), functional._workspace("cpu", 16)
    assert a.numel() == 16 and a.data_ptr() != b.data_ptr()


@gpu
def test_a_captured_step_keeps_its_workspaces(cuda0):
    """Calls that need larger workspaces, and memory that is handed out afterwards, neither change a captured step nor
    are written by it."""
    cfg = _config(mixer="decay", positions="rotary")
    g = torch.Generator().manual_seed(4)
    idx = torch.randint(0, cfg.vocab_size, (2, 96), generator=g)
    tgt = torch.randint(0, cfg.vocab_size, (2, 96), generator=g)
    tr = DataParallelTrainer(cfg, 2, 96, seed=5, lr=0.0, weight_decay=0.0)
    tr.set_batch(idx, tgt)
    tr.capture(warmup=1)
    flat = tr.model.flat

    def grads():
        tr.run_step()
        torch.cuda.synchronize()
        return {n: flat.view(flat.grad, n).clone() for n in tr.model.p if n != "wte"}  # wte: atomic sums
    first = grads()
    wide = torch.randn(20000, 2048, device=cuda0).to(torch.bfloat16).requires_grad_(True)
    w, b = (torch.ones(2048, device=cuda0, dtype=torch.bfloat16).requires_grad_(True) for _ in range(2))
    torch.autograd.grad(ops.layer_norm(wide, w, b), (wide, w, b), torch.ones_like(wide))
    held = [torch.full((n,), 3.25, device=cuda0) for n in (1 << 16, 1 << 18, 1 << 20) for _ in range(24)]
    again = grads()
    for n in first:
        assert torch.equal(first[n], again[n]), n
    assert all(bool((t == 3.25).all()) for t in held)


@gpu
def test_layer_norm_backward_on_streams_side_by_side(cuda0):
    g = torch.Generator(device=cuda0).manual_seed(8)
    streams = [torch.cuda.Stream(cuda0) for _ in range(4)]
    cases = []
    for _ in streams:
        x, dy = (torch.randn(6000, 768, device=cuda0, generator=g).to(torch.bfloat16) for _ in range(2))
        w, b = (torch.randn(768, device=cuda0, generator=g).to(torch.bfloat16).requires_grad_(True) for _ in range(2))
        x.requires_grad_(True)
        cases.append((x, w, b, dy))
    want = [torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), dy) for x, w, b, dy in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, (x, w, b, dy) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), dy))
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert all(torch.equal(i, j) for i, j in zip(a, c))


@gpu
def test_attention_backward_on_streams_side_by_side(cuda0):
    """Bit for bit but for dq, whose sums over key blocks are atomic: there two runs of the same call may differ by
    the order of T / 128 = 8 fp32 terms, a unit in the last place of the bf16 result."""
    g = torch.Generator(device=cuda0).manual_seed(9)
    B, T, H = 1, 1024, 2
    streams = [torch.cuda.Stream(cuda0) for _ in range(4)]
    cases = [[torch.randn(B * T, n * H * 64, device=cuda0, generator=g).to(torch.bfloat16) for n in (3, 1)] for _ in streams]
    for qkv, _ in cases:
        qkv.requires_grad_(True)
    want = [torch.autograd.grad(ops.attention(qkv, B, T, H), qkv, dy)[0].float() for qkv, dy in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, (qkv, dy) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(torch.autograd.grad(ops.attention(qkv, B, T, H), qkv, dy)[0])
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            a = a.float()
            assert torch.equal(a[:, 64 * H:], c[:, 64 * H:])
            scale = c[:, :64 * H].abs().amax()
            assert ((a - c)[:, :64 * H].abs() <= 2.0 ** -7 * c[:, :64 * H].abs() + 2.0 ** -20 * scale).all()


def test_flops_per_token():
    """6 per weight; softmax attention grows with the length, the decay mixer with the head's size alone."""
    small = GPT2Config.small()
    dense = 6.0 * (12 * 12 * 768 * 768 + 50304 * 768)

    def flops(cfg, T):
        class Model:
            pass
        m = Model()
        m.cfg = cfg
        return GPT2.flops_per_token(m, T)
    assert flops(small, 1024) == dense + 6.0 * 12 * 1024 * 768
    decay = GPT2Config(mixer="decay")
    # per head and token: S += k v^T and S^T q, 2 * 64^2 each; backward twice that
    assert flops(decay, 1024) == flops(decay, 64) == dense + 12 * 12 * 3 * (2 + 2) * 64 * 64


@pytest.mark.parametrize("missing", ["n_head", "ln_eps", "vocab_size", "block_size"])
def test_checkpoint_without_a_model_field_is_refused(missing):
    """Only the options that are younger than the format may be absent."""
    class Trainer:
        CHECKPOINT_FORMAT = DataParallelTrainer.CHECKPOINT_FORMAT
        CONFIG_ADDED = getattr(DataParallelTrainer, "CONFIG_ADDED", None)
    tr = Trainer()
    # the saved model stands at the defaults, so nothing but the missing field tells the two apart
    tr.cfg = GPT2Config()
    sd = {"format": tr.CHECKPOINT_FORMAT, "config": dataclasses.asdict(tr.cfg)}
    del sd["config"][missing]
    with pytest.raises(ValueError, match="checkpoint is for model"):
        DataParallelTrainer.load_state_dict(tr, sd)


def test_ranks_draw_masks_of_their_own():
    """The trainer's seeds: one per rank, the same for the rank whenever it is seeded again."""
    from types import SimpleNamespace
    states = []
    for rank in (None, 0, 1, 2, 7):
        tr = SimpleNamespace(model=SimpleNamespace(dropout_state=ops.DropoutState(0, "cpu")),
                             comm=None if rank is None else SimpleNamespace(rank=rank))
        DataParallelTrainer._seed_dropout(tr, 5, 3)
        states.append(tuple(tr.model.dropout_state.tensor.tolist()))
    assert states[0] == states[1] == (5, 3)
    assert len(set(states[1:])) == 4 and all(s[1] == 3 for s in states)
    # the masks behind two ranks' seeds differ in about 2 p (1 - p) of their elements
    a, b = (oracle.dropout_keep(4096, s[0], s[1], 1, 0.5)[0] for s in (states[1], states[2]))
    assert 0.4 < (a != b).double().mean() < 0.6


def _moved(t):
    """The same values in a contiguous view at an address that is not a multiple of 16."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    flat[1:] = t.reshape(-1)
    return flat[1:].view_as(t)


@gpu
@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm_tensors_at_any_address(cuda0, residual):
    """The norms that the model uses without dropout, as those with it."""
    g = torch.Generator(device=cuda0).manual_seed(12)
    x, r, ds, dy = (torch.randn(30, 64, device=cuda0, generator=g).to(torch.bfloat16) for _ in range(4))
    w, b, rb = (torch.randn(64, device=cuda0, generator=g).to(torch.bfloat16) for _ in range(3))

    def run(how):
        xx, rr, ww, bb, rbb = (how(t).requires_grad_(True) for t in (x, r, w, b, rb))
        if residual:
            out = ops.residual_layer_norm(xx, rr, ww, bb, rbias=rbb)
            return [*out, *torch.autograd.grad(out, (xx, rr, ww, bb, rbb), (how(ds), how(dy)))]
        out = ops.layer_norm(xx, ww, bb)
        return [out, *torch.autograd.grad(out, (xx, ww, bb), how(dy))]
    assert all(torch.equal(a, c) for a, c in zip(run(lambda t: t.clone()), run(_moved)))


@gpu
def test_embedding_refusals_and_addresses(cuda0):
    tok = torch.randint(0, 50, (2, 12), device=cuda0)
    wte, wpe = (torch.randn(n, 64, device=cuda0).to(torch.bfloat16).requires_grad_(True) for n in (50, 12))
    dout = torch.randn(2, 12, 64, device=cuda0).to(torch.bfloat16)
    for pos in (None, wpe):
        leaves = [wte] + ([wpe] if pos is not None else [])
        out = ops.embedding(tok, wte, pos)
        want = torch.autograd.grad(out, leaves, dout, retain_graph=True)
        got = torch.autograd.grad(out, leaves, _moved(dout))
        # wte: at most 24 atomic bf16 sums per element, in any order
        assert ((want[0] - got[0]).float().abs() <= 24 * 2.0 ** -8 * dout.float().abs().sum((0, 1))).all()
        assert all(torch.equal(a, c) for a, c in zip(want[1:], got[1:]))
    with pytest.raises(RuntimeError, match="position row"):
        ops.embedding(tok, wte, wpe[:11].detach())
    with pytest.raises(RuntimeError, match="aligned"):
        ops.embedding(tok, _moved(wte.detach()))


@gpu
def test_layer_norm_refusals(cuda0):
    x = torch.zeros(4, 64, device=cuda0, dtype=torch.bfloat16)
    w = torch.ones(64, device=cuda0, dtype=torch.bfloat16)
    for f in (lambda: ops.residual_layer_norm(x, x[:2], w, w), lambda: ops.layer_norm(x, w[:32], w),
              lambda: ops.residual_layer_norm(x, x, w, w, rbias=w.float()),
              lambda: ops.residual_layer_norm(x, x.float(), w, w)):
        with pytest.raises(RuntimeError):
            f()

