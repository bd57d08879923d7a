"""SiT with rotary positions, attention over selected key blocks and 8-bit activation checkpoints, one by one and together, against the same
model written down in 64 bits; and a run of the operators in a captured graph."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


@pytest.fixture(scope="module")
def mods():
    import sitk  # noqa: F401
    from sitk import functional, ops
    from sitk.models import mpp, sit
    return sit, ops, functional, mpp


def pack8(x):
    """What the 8-bit form of x stands for: groups of 32 features, the smallest step 2^k whose codes stay within 127."""
    shape = x.shape
    x2 = x.reshape(-1, shape[-1])
    g = torch.nn.functional.pad(x2, (0, -shape[-1] % 32)).view(x2.shape[0], -1, 32)
    amax = g.abs().amax(-1, keepdim=True)
    k = torch.floor(torch.log2(torch.where(amax > 0, amax, torch.ones_like(amax)))) - 6
    step = 2.0 ** torch.where((amax / 2.0 ** k).round() > 127, k + 1, k)
    return ((g / step).round() * step).view(x2.shape[0], -1)[:, :shape[-1]].reshape(shape)


class RefLinear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        ctx.save_for_backward(x, w)
        ctx.has_b = b is not None
        return torch.nn.functional.linear(x, w, b)

    @staticmethod
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        d2, x2 = dy.reshape(-1, dy.shape[-1]), pack8(x).reshape(-1, x.shape[-1])
        return dy @ w, d2.t() @ x2, d2.sum(0) if ctx.has_b else None


class RefGelu8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u):
        ctx.save_for_backward(u)
        return torch.nn.functional.gelu(u)

    @staticmethod
    def backward(ctx, dg):
        u = pack8(ctx.saved_tensors[0])
        return dg * (0.5 * (1 + torch.erf(u / math.sqrt(2))) + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi))


def ref_rope(x, pos, sections, base):                         # x (B, H, N, dh)
    freqs = torch.cat([float(base) ** (-torch.arange(n, dtype=torch.float64, device=x.device) / n) for n in sections])
    axis = torch.repeat_interleave(torch.arange(len(sections)), torch.tensor(sections)).to(x.device)
    ang = pos.double()[:, axis] * freqs
    c, s, P = ang.cos(), ang.sin(), sum(sections)
    a, b = x[..., :P], x[..., P:2 * P]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * P:]), -1)


def reference(model, img, indices):
    """The model's output in 64 bits from (copies of) its parameters; `indices`: the blocks selected, layer by layer."""
    tr = model.transformer
    P = {k: p.detach().double().requires_grad_() for k, p in model.named_parameters()}
    lin = RefLinear8.apply if tr.act8 else torch.nn.functional.linear
    gelu = RefGelu8.apply if tr.act8 else torch.nn.functional.gelu
    B, Cc, Np, V = img.shape
    x = img.double().permute(0, 2, 3, 1).reshape(B, Np, V * Cc)
    x = torch.nn.functional.linear(x, P["to_patch_embedding.1.weight"], P["to_patch_embedding.1.bias"])
    x = torch.cat((P["cls_token"].expand(B, 1, -1), x), 1) + P["pos_embedding"]
    N, D = x.shape[1:]
    for i, (attn, ff) in enumerate(tr.layers):
        a, n = attn.fn, f"transformer.layers.{i}."
        h = torch.nn.functional.layer_norm(x, (D,), P[n + "0.norm.weight"], P[n + "0.norm.bias"])
        q, k, v = lin(h, P[n + "0.fn.to_qkv.weight"], None).view(B, N, 3, a.heads, a.dim_head).permute(2, 0, 3, 1, 4)
        if tr.rotary is not None:
            q, k = (ref_rope(t, tr._positions.to(DEV), tr.rotary, tr.rotary_base) for t in (q, k))
        s = (q @ k.transpose(-1, -2).contiguous()) * a.scale
        if tr.key_blocks is not None:
            block = tr.key_blocks[0]
            nb = -(-N // block)
            idx = indices[i].long()
            chosen = torch.zeros(B, a.heads, N, nb + 1, dtype=torch.bool, device=DEV).scatter_(-1, idx.where(idx >= 0, nb), True)[..., :nb]
            s = s.masked_fill(~chosen.repeat_interleave(block, -1)[..., :N], -math.inf)
        o = (s.softmax(-1) @ v).transpose(1, 2).reshape(B, N, -1)
        x = x + lin(o, P[n + "0.fn.to_out.0.weight"], P[n + "0.fn.to_out.0.bias"])
        h = torch.nn.functional.layer_norm(x, (D,), P[n + "1.norm.weight"], P[n + "1.norm.bias"])
        g = gelu(lin(h, P[n + "1.fn.net.0.weight"], P[n + "1.fn.net.0.bias"]))
        x = x + lin(g, P[n + "1.fn.net.3.weight"], P[n + "1.fn.net.3.bias"])
    x = x.mean(1) if model.pool == "mean" else x[:, 0]
    x = torch.nn.functional.layer_norm(x, (D,), P["mlp_head.0.weight"], P["mlp_head.0.bias"])
    return torch.nn.functional.linear(x, P["mlp_head.1.weight"], P["mlp_head.1.bias"]), P


def build(sit, dtype, seed=0, **opt):
    torch.manual_seed(seed)
    kw = dict(dict(dim=128, depth=2, heads=2, mlp_dim=192, num_patches=200, num_vertices=6, num_channels=2, num_classes=3, pool="mean"), **opt)
    m = sit.SiT(**kw, compute_dtype=dtype).to(DEV)
    if m.transformer.rotary is not None:
        p = torch.randn(kw["num_patches"], len(kw["rotary"]))
        m.set_patch_positions(p / p.norm(dim=-1, keepdim=True) * 20)
    img = torch.randn(3, kw["num_channels"], kw["num_patches"], kw["num_vertices"], device=DEV)
    return m, img, torch.randn(3, 3, device=DEV)


class Recorder:
    """Notes the blocks that block_select picks, and can hand out noted ones instead."""

    def __init__(self, ops, monkeypatch, given=None):
        self.seen, given = [], None if given is None else list(given)
        real = ops.block_select

        def select(q, pool, top_k):
            sel = real(q, pool, top_k) if given is None else ops.block_selection(given[len(self.seen)], pool)
            self.seen.append(sel.index)
            return sel

        monkeypatch.setattr(ops, "block_select", select)


def norm_error(mine, ref):
    """Of all parameters' gradients as one vector."""
    num = sum(float((mine[k].grad.double() - r.grad).square().sum()) for k, r in ref.items())
    return math.sqrt(num / sum(float(r.grad.square().sum()) for r in ref.values()))


OPTIONS = [dict(rotary=(10, 10, 12)), dict(key_blocks=(64, 2)), dict(act8=True), dict(rotary=(10, 10, 12), key_blocks=(64, 1), act8=True),
           dict(rotary=(8,), key_blocks=(128, 1), act8=True, dim_head=32, heads=3, pool="cls"), dict(rotary=(5, 5), dim_head=20),
           dict(heads=1, dim_head=64, dim=64, key_blocks=(64, 4), act8=True)]


@pytest.mark.parametrize("opt", OPTIONS, ids=lambda o: "+".join(k for k in o))
def test_f32_model_matches_the_definition(mods, monkeypatch, opt):
    """Output and gradients in f32 mode.  Values are off by about 1e-6 of themselves (32-bit sums of some hundred terms, two layers).  With
    act8 a value flips to the next code where it lies within 1e-6 |x| of a border between two: at most 2 x 127 x 1e-6 of them, by
    one step of at most 1/63 of the group's largest: sqrt(2.5e-4) / 63 = 2.5e-4 of the norm.  Held to 1e-3, outputs to 1e-4."""
    sit, ops, _, _ = mods
    m, img, w = build(sit, "f32", **opt)
    rec = Recorder(ops, monkeypatch)
    out = m(img)
    (out * w).sum().backward()
    ref, P = reference(m, img, rec.seen) if m.transformer.layers[0][0].fn.project_out else _reference_projection_free(m, img, rec.seen)
    (ref * w.double()).sum().backward()
    assert float((out.detach().double() - ref).norm() / ref.detach().norm()) < 1e-4
    assert norm_error(dict(m.named_parameters()), P) < 1e-3
    for k, p in m.named_parameters():
        assert p.grad.shape == p.shape and bool(torch.isfinite(p.grad).all()), k


def _reference_projection_free(m, img, seen):
    """heads = 1 as wide as the model: an identity in the place of the output projection."""
    kept = [layer[0].fn.to_out for layer in m.transformer.layers]
    for layer in m.transformer.layers:
        eye = torch.nn.Linear(m.dim, m.dim, device=DEV)
        with torch.no_grad():
            eye.weight.copy_(torch.eye(m.dim)), eye.bias.zero_()
        layer[0].fn.to_out = torch.nn.Sequential(eye)
    try:
        ref, P = reference(m, img, seen)
    finally:
        for layer, old in zip(m.transformer.layers, kept):
            layer[0].fn.to_out = old
    names = {k for k, _ in m.named_parameters()}
    return ref, {k: p for k, p in P.items() if k in names}


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_16_bit_models_follow_the_definition(mods, monkeypatch, dtype):
    """All three options, blocks as selected.  A product of two rounded operands is off by at most 2 u of its norm; 5 in a row in each of two
    layers: 20 u, and twice that behind the way back."""
    sit, ops, _, _ = mods
    m, img, w = build(sit, dtype, rotary=(10, 10, 12), key_blocks=(64, 2), act8=True)
    rec = Recorder(ops, monkeypatch)
    out = m(img)
    (out * w).sum().backward()
    ref, P = reference(m, img, rec.seen)
    (ref * w.double()).sum().backward()
    assert float((out.detach().double() - ref).norm() / ref.detach().norm()) < 20 * U[dtype]
    assert norm_error(dict(m.named_parameters()), P) < 40 * U[dtype]


def test_gradients_match_differences(mods, monkeypatch):
    """Rotary positions and block attention in f32 mode with the blocks held: central differences along directions with a part of the
    gradient, h = 1e-3: the third derivative leaves some h^2 = 1e-6 of the slope; the outputs' rounding, 1e-6 of 280 (the norm of the
    weights times that of about 1), 3e-4 / 2 h = 0.14, against a slope of |g| sqrt(77000) = several hundred.  Held to 1e-2."""
    sit, ops, _, _ = mods
    m, img, w = build(sit, "f32", rotary=(10, 10, 12), key_blocks=(64, 2))
    rec = Recorder(ops, monkeypatch)
    x = torch.randn(3, 201, 128, device=DEV).requires_grad_()
    wx = torch.randn(3, 201, 128, device=DEV)
    m.transformer(x)
    monkeypatch.undo()
    held = rec.seen

    def loss(x):
        with monkeypatch.context() as mp:
            Recorder(ops, mp, given=held)
            return (m.transformer(x).double() * wx).sum()

    g, = torch.autograd.grad(loss(x), x)
    for seed in range(3):
        torch.manual_seed(seed)
        d = torch.randn_like(x) + g / g.std()
        h = 1e-3
        with torch.no_grad():
            slope = (loss(x + h * d) - loss(x - h * d)) / (2 * h)
        assert float((slope - (g * d).double().sum()).abs()) < 1e-2 * float((g * d).double().sum().abs())


def test_act8_gradients_match_differences(mods):
    """Gelu8Fn: |gelu''| <= 2 / sqrt(2 pi) = 0.798, so that half a step of u moves the slope by at most 0.4 steps; Linear8Fn: by half a step
    of x times |dy|."""
    _, _, Fn, _ = mods
    torch.manual_seed(1)
    u, dg = torch.randn(70, 100, device=DEV, requires_grad=True), torch.randn(70, 100, device=DEV)
    g, = torch.autograd.grad(Fn.Gelu8Fn.apply(u), u, dg)
    ud, h = u.detach().double(), 1e-4
    slope = (torch.nn.functional.gelu(ud + h) - torch.nn.functional.gelu(ud - h)) / (2 * h)
    amax = torch.nn.functional.pad(ud, (0, 28)).view(70, 4, 32).abs().amax(-1, keepdim=True).expand(70, 4, 32).reshape(70, 128)[:, :100]
    assert bool(((g.double() - dg * slope).abs() <= dg.abs() * (0.4 * amax / 63 + 1e-5)).all())
    x = torch.randn(40, 52, device=DEV)
    wt, b = torch.randn(24, 52, device=DEV, requires_grad=True), torch.randn(24, device=DEV, requires_grad=True)
    dy = torch.randn(40, 24, device=DEV)
    y = Fn.Linear8Fn.apply(x, wt, b, "f32")
    assert torch.equal(y, Fn.LinearFn.apply(x, wt, b, "f32"))
    dw, db = torch.autograd.grad(y, (wt, b), dy)
    xd = x.double()
    ax = torch.nn.functional.pad(xd, (0, 12)).view(40, 2, 32).abs().amax(-1, keepdim=True).expand(40, 2, 32).reshape(40, 64)[:, :52]
    exact = dy.double().t() @ xd                                # the loss is linear in W: the difference quotient for any h
    assert bool(((dw.double() - exact).abs() <= dy.double().abs().t() @ (ax / 126 + 1e-5)).all())
    assert bool(((db.double() - dy.double().sum(0)).abs() <= 1e-5 * dy.double().abs().sum(0)).all())


def test_act8_changes_no_value_and_keeps_less(mods):
    sit, _, _, _ = mods
    opt = dict(rotary=(10, 10, 12), key_blocks=(64, 2), num_patches=1000, mlp_dim=512)
    kept = {}
    for act8 in (False, True):
        m, img, _ = build(sit, "bf16", act8=act8, **opt)
        x = torch.randn(3, 1001, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).requires_grad_()
        m.transformer(x).sum().backward()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = m.transformer(x)
        kept[act8] = (torch.cuda.memory_allocated() - before, y.detach().clone())
        with torch.no_grad():
            assert torch.equal(m.transformer(x), y)
        del y, x, m
    assert torch.equal(kept[False][1], kept[True][1])
    assert kept[True][0] < 0.75 * kept[False][0], {k: v[0] for k, v in kept.items()}


def test_frozen_parts_repeated_backward_and_other_stream(mods):
    sit, _, _, _ = mods
    m, img, w = build(sit, "bf16", rotary=(10, 10, 12), key_blocks=(64, 2), act8=True)
    loss = (m(img) * w).sum()
    loss.backward(retain_graph=True)
    first = {k: p.grad.clone() for k, p in m.named_parameters()}
    m.zero_grad()
    loss.backward()
    del loss
    for k, p in m.named_parameters():                           # (the LayerNorm sums of the module path add atomically)
        assert float((p.grad - first[k]).norm()) <= 1e-5 * float(first[k].norm()) + 1e-12, k
    m.zero_grad()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = m(img)
        (out * w).sum().backward()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(float((p.grad - first[k]).norm()) <= 1e-5 * float(first[k].norm()) + 1e-12 for k, p in m.named_parameters())
    m.zero_grad()
    for p in m.transformer.parameters():
        p.requires_grad_(False)
    m.transformer.layers[1][1].fn.net[3].bias.requires_grad_(True)         # a bias alone
    (m(img) * w).sum().backward()
    assert sum(p.grad is not None for p in m.transformer.parameters()) == 1 and float(m.cls_token.grad.abs().sum()) > 0
    k = "transformer.layers.1.1.fn.net.3.bias"
    assert float((dict(m.named_parameters())[k].grad - first[k]).norm()) <= 1e-2 * float(first[k].norm())


def test_dropout_and_masked_pretraining_take_the_options(mods):
    sit, _, _, mpp = mods
    m, img, _ = build(sit, "bf16", rotary=(10, 10, 12), key_blocks=(64, 2), act8=True, dropout=0.1, emb_dropout=0.1)
    m(img).sum().backward()
    assert all(bool(torch.isfinite(p.grad).all()) for p in m.parameters())
    m, img, _ = build(sit, "bf16", rotary=(10, 10, 12), key_blocks=(64, 2), act8=True)
    ssl = mpp.masked_patch_pretraining(transformer=m, dim_in=128, dim_out=12, device=DEV, channels=2, num_vertices=6).to(DEV)
    loss = ssl(img)
    loss = loss[0] if isinstance(loss, tuple) else loss
    loss.backward()
    assert all(p.grad is None or bool(torch.isfinite(p.grad).all()) for p in ssl.parameters())
    assert float(m.transformer.layers[0][0].fn.to_qkv.weight.grad.abs().sum()) > 0


def test_a_model_needs_its_positions_and_the_engine_refuses(mods):
    sit, _, _, _ = mods
    from sitk.engine import TrainEngine
    from sitk.runtime import SitkError
    kw = dict(dim=64, depth=1, heads=1, dim_head=32, mlp_dim=64, num_patches=20, num_vertices=4, num_channels=2)
    m = sit.SiT(**kw, rotary=(4,)).to(DEV)
    with pytest.raises(SitkError, match="not set"):
        m(torch.zeros(1, 2, 20, 4, device=DEV))
    for opt in (dict(rotary=(4,)), dict(key_blocks=(64, 1)), dict(act8=True)):
        with pytest.raises(SitkError, match="stage by stage"):
            TrainEngine(sit.SiT(**dict(kw, dim_head=64, heads=3), **opt), batch_size=2, input_layout="patched")


def test_operators_in_one_graph_follow_new_inputs(mods):
    """A block's operators in one captured graph, in the order in which they are used, replayed four times with new inputs and eager work in
    between: the same bits as the eager calls."""
    _, ops, _, _ = mods
    B, N, H, D = 2, 333, 2, 128
    sec, td = (10, 10, 12), torch.bfloat16
    freqs = ops.rope_freqs(sec, device=DEV)
    torch.manual_seed(3)
    fresh = lambda: dict(qkv=torch.randn(B, N, 3, H, 64, device=DEV).to(td), do=torch.randn(B, N, H, 64, device=DEV).to(td),   # noqa: E731
                         pos=torch.randn(N, 3, device=DEV) * 20, x=torch.randn(B * N, D, device=DEV).to(td),
                         mask=torch.rand(B, N, device=DEV) > 0.3)
    inp = fresh()

    def run(i):
        q, k, v = i["qkv"].unbind(2)
        q, k = ops.rope_axes(q, k, i["pos"], freqs, sec)
        sel = ops.block_select(q, ops.block_pool(k, 64, i["mask"]), 2)
        o, lse = ops.block_attention_fwd(q, k, v, sel, 0.125)
        dq, dk, dv = ops.block_attention_bwd(q, k, v, o, i["do"], lse, sel, 0.125)
        dq, dk = ops.rope_axes(dq, dk, i["pos"], freqs, sec, inverse=True)
        g, u8 = ops.act8_gelu_fwd(i["x"])
        dw, db = ops.act8_wgrad(o.view(B * N, D), ops.act8_pack(g))
        return [sel.index, o, lse, dq, dk, dv, g, dw, db, ops.act8_gelu_bwd(g, u8), ops.act8_unpack(u8)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run(inp)
    torch.cuda.current_stream().wait_stream(s)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(inp)
    with torch.cuda.graph(second):                              # a second graph of the same inputs has workspaces of its own
        out2 = run(inp)
    for _ in range(4):
        new = fresh()
        for k in inp:
            inp[k].copy_(new[k])
        want = run(new)
        torch.cuda.synchronize()
        graph.replay()
        second.replay()
        torch.cuda.synchronize()
        for a, a2, b in zip(out, out2, want):
            assert torch.equal(a, b) and torch.equal(a2, b)


def test_captured_training_step(mods):
    """Forward and backward pass of a model with all three options in a captured graph, replayed with new inputs and eager steps of another copy
    in between: the eager gradients (atomics in the LayerNorm sums: 1e-5 of their norm)."""
    sit, _, _, _ = mods
    opt = dict(rotary=(10, 10, 12), key_blocks=(64, 2), act8=True)
    m, img, w = build(sit, "bf16", **opt)
    other, _, _ = build(sit, "bf16", **opt)
    other.load_state_dict(m.state_dict())
    other.transformer.set_positions(m.transformer._positions)
    x = img.clone()

    def step(model, inp):
        for p in model.parameters():
            p.grad = None
        out = model(inp)
        (out * w).sum().backward()
        return out.detach()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            step(m, x)
    torch.cuda.current_stream().wait_stream(s)
    for p in m.parameters():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(m, x)
    for i in range(4):
        new = torch.randn(img.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i))
        x.copy_(new)
        want = step(other, new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for (k, p), q in zip(m.named_parameters(), other.parameters()):
            assert float((p.grad - q.grad).norm()) <= 1e-5 * float(q.grad.norm()) + 1e-12, (i, k)


def test_new_positions_leave_a_captured_graph_alone(mods):
    """A graph of the forward pass, replayed behind set_positions and other allocations: the outputs of the positions it was captured with;
    an eager pass takes the new ones, and a pass under capture that would have to bring them to the device is refused."""
    sit, _, _, _ = mods
    m, img, _ = build(sit, "bf16", rotary=(10, 10, 12), key_blocks=(64, 2))
    x = img.clone()
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            want = m(x)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)
        new = m.transformer._positions.flip(0) * 1.5
        m.transformer.set_positions(new)
        junk = [torch.full((n,), 7.0, device=DEV) for n in range(1, 4000, 7)]
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            other = m(x)
            assert not torch.equal(other, want) and len(junk)


def test_training_behind_a_first_pass_in_inference_mode(mods):
    sit, _, _, _ = mods
    opt = dict(rotary=(10, 10, 12), key_blocks=(64, 2), act8=True)
    m, img, w = build(sit, "bf16", **opt)
    other, _, _ = build(sit, "bf16", **opt)
    other.load_state_dict(m.state_dict())
    other.transformer.set_positions(m.transformer._positions)
    with torch.inference_mode():
        seen = m(img).clone()
    for x in (m, other):
        (x(img) * w).sum().backward()
    assert torch.equal(seen, other(img).detach())
    for (k, p), q in zip(m.named_parameters(), other.parameters()):
        assert float((p.grad - q.grad).norm()) <= 1e-5 * float(q.grad.norm()) + 1e-12, k
