"""The ragged grouped products, 4-bit weights and dropout where the package itself uses them: blocks of any
width, the FFN sublayer, the decode stack, and a run of them together. CPU parts: the torch fallbacks and what
is refused."""
import pytest
import torch

from conftest import rel_l2
from nanospeaker_b200 import MoEBlock, MoEFFNSublayer, quantize_int4
from nanospeaker_b200.decode import StackedMoEDecoder

gpu = pytest.mark.gpu


def block(d, e, d_ff, k, s=0, dtype=torch.float32, **kw):
    m = MoEBlock(d, e, d_ff=d_ff, top_k=k, n_shared=s, capacity_factor=kw.pop("capacity_factor", None), **kw)
    with torch.no_grad():
        m.W_in.copy_(torch.randn_like(m.W_in) * d ** -0.5)
        m.W_out.copy_(torch.randn_like(m.W_out) * m.d_hidden ** -0.5)
        if s:
            m.W_sh_in.copy_(torch.randn_like(m.W_sh_in) * d ** -0.5)
            m.W_sh_out.copy_(torch.randn_like(m.W_sh_out) * m.d_hidden ** -0.5)
        for b in (m.b_in, m.b_out):
            if b is not None:
                b.copy_(torch.randn_like(b) * 0.1)
    return m.to(dtype)


# ------------------------------------------------------------------------------------------- CPU
def test_grouped_setting_changes_nothing_off_the_gpu():
    m = block(64, 6, 96, 2, capacity_factor="auto")
    x = torch.randn(30, 64)
    want, cap = m(x), m.capacity_factor
    m.grouped = True
    assert m.capacity_factor == cap and torch.equal(m(x), want)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradient_of_gathered_rows_is_rounded_once(device, dtype):
    """A token's rows of the gradient, of which there are k: their fp32 sum (off by k 2^-24 of the magnitude) and one
    rounding. Summed in the type, one rounding a row, they are not within that."""
    from nanospeaker_b200.moe import _PairRows
    gen = torch.Generator().manual_seed(0)
    n, k, d = 50, 8, 40
    order = torch.randperm(n * k, generator=gen)
    place = torch.empty_like(order).index_copy_(0, order, torch.arange(n * k))
    x, g = torch.randn(n, d, generator=gen), torch.randn(n * k, d, generator=gen)
    x, g = (t.to(device, dtype) for t in (x, g))
    order, place = order.to(device), place.to(device)
    x.requires_grad_()
    out = _PairRows.apply(x, order // k, place)
    assert torch.equal(out, x[order // k])
    got, = torch.autograd.grad(out, x, g)
    rows = g[place].view(n, k, d).double()
    a = k * 2.0 ** -24 * rows.abs().sum(1)
    bound = torch.finfo(dtype).eps / 2 * (rows.sum(1).abs() + a) + a
    assert got.dtype == dtype and bool(((got.double() - rows.sum(1)).abs() <= bound).all())
    in_type = torch.zeros_like(x)
    for j in range(k):
        in_type = in_type + g[place].view(n, k, d)[:, j]
    assert not bool(((in_type.detach().double() - rows.sum(1)).abs() <= bound).all())


def test_sublayer_dropout_on_the_cpu():
    sub = MoEFFNSublayer(block(64, 6, 96, 2), dropout=0.25)
    x = torch.randn(200, 64)
    sub.eval()
    whole, _ = sub(x)
    assert torch.equal(whole, sub(x)[0])
    sub.train()
    torch.manual_seed(3)
    out, _ = sub(x)
    branch, part = whole - x, out - x
    dropped = (part.abs() < 1e-7) & (branch.abs() > 1e-4)
    assert 0.15 < float(dropped.float().mean()) < 0.35
    kept = ~dropped & (branch.abs() > 1e-4)
    assert torch.allclose(part[kept], branch[kept] / 0.75, rtol=1e-3, atol=1e-5)
    torch.manual_seed(3)
    assert torch.equal(sub(x)[0], out)
    for p in (-0.1, 1.0):
        with pytest.raises(ValueError, match="dropout"):
            MoEFFNSublayer(sub.ffn, dropout=p)
    state = torch.get_rng_state()
    MoEFFNSublayer(sub.ffn), MoEFFNSublayer(sub.ffn, dropout=0.5)
    assert torch.equal(torch.get_rng_state(), state)


def test_decoder_of_4_bit_weights_refuses_what_it_does_not_cover():
    for bad in (block(64, 4, 96, 2, bias=True), block(64, 4, 96, 2, capacity_factor=1.5),
                block(64, 4, 60, 2), block(64, 4, 96, 2, activation=torch.sin)):
        with pytest.raises(ValueError, match="4-bit experts"):
            StackedMoEDecoder([bad], weights="int4")
    with pytest.raises(ValueError, match="held in"):
        StackedMoEDecoder([block(64, 4, 96, 2)], weights="fp4")


# ------------------------------------------------------------------------------------------- GPU
def both(m, x, dout):
    """(out, aux, dx, weight gradients) of one step."""
    m.zero_grad()
    x = x.clone().requires_grad_()
    out = m(x)
    (out.float() * dout.float()).sum().backward()
    return [out.detach(), x.grad] + [p.grad.clone() for p in m.parameters()]


# The block's two forms round differently between the same steps (bf16: each rounding at most 2^-9 of a value
# in the mean square, some ten of them in a row in either form); 2e-2 of the norm is their sum, and what the
# kernels' own parity tests allow twice.
TOL = {torch.bfloat16: 2e-2, torch.float16: 4e-3}


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kw", [dict(d=64, e=8, d_ff=96, k=2), dict(d=576, e=76, d_ff=768, k=6, s=2),
                                dict(d=72, e=5, d_ff=60, k=3, bias=True), dict(d=64, e=8, d_ff=96, k=2,
                                                                               capacity_factor=0.5),
                                dict(d=128, e=16, d_ff=192, k=4, activation="gelu", kernel=False)])
def test_block_of_any_width_matches_the_torch_loop(kw, dtype):
    kw = dict(kw)
    m = block(kw.pop("d"), kw.pop("e"), kw.pop("d_ff"), kw.pop("k"), kw.pop("s", 0), dtype, **kw).cuda().train()
    x = torch.randn(777, m.d_model, device="cuda").to(dtype)
    dout = torch.randn_like(x)
    want = both(m, x, dout)
    counts, dropped = m.expert_counts.clone(), m.dropped
    m.grouped = True
    assert m._grouped_ok(x) and m.capacity_factor == kw.get("capacity_factor")
    got = both(m, x, dout)
    assert torch.equal(m.expert_counts, counts) and int(m.dropped) == int(dropped)
    for a, b in zip(got, want):
        assert rel_l2(a, b) < TOL[dtype]
    assert all(torch.equal(a, b) for a, b in zip(both(m, x, dout)[:1], got[:1]))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_grouped_blocks_input_gradient_is_rounded_once(dtype):
    """Every token through all eight experts, whole numbers throughout (weights are signed permutations, so that a
    pair's gradient stays below 256, exact in either type): the token's gradient is the exact sum, rounded once."""
    gen = torch.Generator().manual_seed(1)
    d, e, n = 16, 8, 60
    m = block(d, e, 24, e, dtype=torch.float64, activation="relu")
    assert m.d_hidden == d
    sign = lambda *s: torch.randint(0, 2, s, generator=gen).double() * 2 - 1  # noqa: E731
    perm = lambda: torch.eye(d, dtype=torch.float64)[torch.randperm(d, generator=gen)] * sign(d, 1)  # noqa: E731
    with torch.no_grad():
        for i in range(e):
            m.W_in[i] = torch.cat([perm(), perm()], 1)
            m.W_out[i] = perm()
    x = torch.randint(-2, 3, (n, d), generator=gen).double().requires_grad_()
    dout = torch.randint(-63, 64, (n, d), generator=gen).double()
    idx, tw = torch.arange(e).expand(n, e).contiguous(), torch.ones(n, e, dtype=torch.float64)
    want, = torch.autograd.grad(m._torch_experts(x, tw, idx, 0)[0], x, dout)
    assert float(want.abs().max()) > 256
    m = m.to(dtype).cuda()
    xc = x.detach().to("cuda", dtype).requires_grad_()
    out, _ = m._grouped_experts(xc, tw.to("cuda", dtype), idx.cuda(), 0)
    got, = torch.autograd.grad(out, xc, dout.to("cuda", dtype))
    assert torch.equal(got.cpu(), want.to(dtype))


@gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_dropped_pairs_hold_reaches_nothing(dtype, bias):
    """Tokens whose pairs are all over the capacity hold infinities and NaN: results, gradients of the weights, of the
    router's weights and of the other tokens as the torch loop gives them, which never looks at those pairs."""
    m = block(64, 4, 96, 2, dtype=dtype, bias=bias).cuda()
    gen = torch.Generator().manual_seed(2)
    n, cap = 40, 12
    idx = torch.stack([torch.zeros(n, dtype=torch.long), torch.arange(n) % 3 + 1], 1)   # expert 0: every token
    idx[20:] = torch.tensor([0, 1])
    counts = [0] * 4                       # pairs in expert order, ties in pair order: the first 12 of each are kept
    kept = torch.zeros(n, 2, dtype=torch.bool)
    for t in range(n):
        for j in range(2):
            kept[t, j] = counts[idx[t, j]] < cap
            counts[idx[t, j]] += 1
    lost = ~kept.any(1)
    assert 5 < int(lost.sum()) < n
    x, dout = torch.randn(n, 64, generator=gen), torch.randn(n, 64, generator=gen)
    x[lost] = torch.tensor([float("inf"), float("nan"), float("-inf"), 3e38]).repeat(16)
    tw = torch.rand(n, 2, generator=gen)
    results = []
    for path in (m._torch_experts, m._grouped_experts):
        xc, tc = x.to("cuda", dtype).requires_grad_(), tw.to("cuda", dtype).requires_grad_()
        out, c = path(xc, tc, idx.cuda(), cap)
        params = [p for p in (m.W_in, m.W_out, m.b_in, m.b_out) if p is not None]
        grads = torch.autograd.grad(out, (xc, tc, *params), dout.to("cuda", dtype))
        assert c.tolist() == counts and int(m.dropped) == int((~kept).sum())
        results.append([out.detach(), *grads])
    for a, b in zip(*results):
        assert bool(torch.isfinite(a).all()) and bool(torch.isfinite(b).all())
        assert rel_l2(b, a) < TOL[dtype]
    gone = lost.cuda()
    assert not results[1][0][gone].any() and not results[1][1][gone].any()
    assert not results[1][2][~kept.cuda()].any()


@gpu
def test_wide_block_with_fp32_weights_takes_16_bit_rows():
    """Weights in fp32, cast where they are used: the result of the 16-bit block with the same values, and fp32
    gradients."""
    m = block(64, 8, 96, 2, 2, torch.bfloat16, bias=True).cuda().train()
    full = block(64, 8, 96, 2, 2, bias=True).cuda().train()
    full.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    m.grouped = full.grouped = True
    x = torch.randn(60, 64, device="cuda").bfloat16()
    got, want = both(full, x, x), both(m, x, x)
    assert torch.equal(got[0], want[0]) and got[0].dtype == torch.bfloat16
    for a, b in zip(got[2:], want[2:]):
        assert a.dtype == torch.float32 and rel_l2(a, b) < TOL[torch.bfloat16]


@gpu
def test_block_of_any_width_without_a_sync_and_in_a_graph():
    m = block(64, 8, 96, 2, dtype=torch.bfloat16).cuda().eval()
    m.grouped = True
    x = torch.randn(100, 64, device="cuda").bfloat16()
    with torch.no_grad():
        m(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(x)
        x.copy_(torch.randn(100, 64))
        graph.replay()
        assert torch.equal(out, m(x))


@gpu
def test_sublayer_dropout_masks_and_gradients():
    """Forward and gradient through the same mask; the seed governs it; evaluation has none."""
    sub = MoEFFNSublayer(block(576, 8, 192, 2, 1, torch.bfloat16), dropout=0.5).to(torch.bfloat16).cuda()
    sub.ffn.combine_mode = "store"      # (the combine that repeats bit for bit)
    x = torch.randn(300, 576, device="cuda").bfloat16()
    plain = MoEFFNSublayer(sub.ffn).to(torch.bfloat16).cuda().eval()
    sub.eval()
    assert torch.equal(sub(x)[0], plain(x)[0])
    sub.train()
    torch.manual_seed(1)
    a, _ = sub(x)
    b, _ = sub(x)
    torch.manual_seed(1)
    assert torch.equal(sub(x)[0], a) and not torch.equal(a, b)
    dropped = a == x
    assert 0.45 < float(dropped.float().mean()) < 0.56
    # the branch's gradient is zero where it was dropped: one column's gradient through the output weights
    torch.manual_seed(1)
    out, _ = sub(x)
    dout = torch.zeros_like(x)
    dout[:, 7] = 1
    kept_rows = ~dropped[:, 7]
    grad = torch.autograd.grad(out, sub.ffn.W_out, dout)[0]
    torch.manual_seed(1)
    out, _ = sub(x)
    same = torch.autograd.grad(out, sub.ffn.W_out, dout * kept_rows[:, None])[0]
    assert rel_l2(grad, same) < 1e-2 and float(grad.abs().sum()) > 0


@gpu
@pytest.mark.parametrize("kernel,dtype", [(True, torch.bfloat16), (False, torch.bfloat16), (False, torch.float16)])
def test_sublayer_dropout_under_autocast(kernel, dtype):
    """The result has the type that the sublayer without dropout gives, and gradients flow. (In fp16 the shared
    experts' bf16 products make the block's result fp32.)"""
    ffn = block(64, 8, 96, 2, 1, dtype, kernel=kernel).cuda().train()
    ffn.grouped = not kernel
    x = torch.randn(40, 64, device="cuda").to(dtype).requires_grad_()
    with torch.autocast("cuda", torch.bfloat16):
        want, _ = MoEFFNSublayer(ffn).cuda()(x)
        out, _ = MoEFFNSublayer(ffn, dropout=0.5).cuda()(x)
    assert out.dtype == want.dtype and out.shape == want.shape
    out.float().sum().backward()
    assert bool(torch.isfinite(x.grad).all())


@gpu
@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64), (1, 64), (3, 5, 64)])
def test_wide_sublayer_and_block_of_few_rows_and_none(shape):
    m = block(64, 8, 96, 2, dtype=torch.bfloat16).cuda().train()
    m.grouped = True
    sub = MoEFFNSublayer(m, dropout=0.5).to(torch.bfloat16).cuda()
    x = torch.randn(shape, device="cuda").bfloat16().requires_grad_()
    assert m(x).shape == sub(x)[0].shape == x.shape
    if x.numel():
        sub(x)[0].float().sum().backward()
        assert bool(torch.isfinite(x.grad).all())
    assert StackedMoEDecoder([m], weights="int4").eager(x.detach()).shape == x.shape


@gpu
def test_sublayer_dropout_under_activation_checkpointing():
    """The recomputed forward meets the same mask: gradients as without checkpointing."""
    from torch.utils.checkpoint import checkpoint
    sub = MoEFFNSublayer(block(64, 8, 96, 2, dtype=torch.float32), dropout=0.3).cuda().train()
    sub.ffn.aux_loss = None
    x = torch.randn(100, 64, device="cuda")
    grads = []
    for through in (lambda f, v: f(v), lambda f, v: checkpoint(f, v, use_reentrant=True),
                    lambda f, v: checkpoint(f, v, use_reentrant=False)):
        v = x.clone().requires_grad_()
        torch.manual_seed(5)
        out = through(lambda t: sub(t)[0], v)
        out.square().sum().backward()
        grads.append(v.grad)
    for g in grads[1:]:
        assert rel_l2(g, grads[0]) < 1e-5


def layer_in_4_bits(m, x, group):
    """x + block(x) in 64 bits with the 4-bit values of the experts' weights, routed as the block's router
    routes x."""
    with torch.no_grad():
        topk_w, topk_idx, _ = m.router(x)
        value = lambda w: None if w is None else quantize_int4(w, group, x.dtype).dequantize().double()  # noqa: E731
        w_in, w_out, sh_in, sh_out = (value(w) for w in (m.W_in, m.W_out, m.W_sh_in, m.W_sh_out))
        xd, out = x.double(), x.double().clone()

        def mlp(rows, a, b):
            gate, up = (rows @ a).chunk(2, dim=-1)
            return m.glu(gate, up) @ b

        for e in topk_idx.unique().tolist():
            tok, slot = (topk_idx == e).nonzero(as_tuple=True)
            out.index_add_(0, tok, mlp(xd[tok], w_in[e], w_out[e]) * topk_w.double()[tok, slot, None])
        for e in range(m.n_shared):
            out += mlp(xd, sh_in[e], sh_out[e])
        return out


@gpu
@pytest.mark.parametrize("kw,dtype", [(dict(d=576, e=76, d_ff=192, k=6, s=2), torch.bfloat16),
                                      (dict(d=128, e=8, d_ff=240, k=2), torch.float16)])
@pytest.mark.parametrize("t", [1, 64])
def test_decoder_with_4_bit_weights(kw, dtype, t):
    """Layer by layer against the 4-bit values in 64 bits. Three roundings to the type (the hidden values, the
    experts' sum, the sum with x), each at most half a step of its value: twice that of the rows' norm."""
    blocks = [block(kw["d"], kw["e"], kw["d_ff"], kw["k"], kw.get("s", 0), dtype).cuda().eval() for _ in range(3)]
    dec = StackedMoEDecoder(blocks, weights="int4", group=64)
    x = torch.randn(t, kw["d"], device="cuda").to(dtype)
    first = dec.step(x).clone()
    assert torch.equal(dec.step(x), first) and torch.equal(dec.eager(x), first)
    at = x
    for b in blocks:
        got = StackedMoEDecoder([b], weights="int4", group=64).eager(at)
        want = layer_in_4_bits(b, at, 64)
        off = (got.double() - want).norm(dim=1) / want.norm(dim=1)
        assert float(off.max()) < 3 * torch.finfo(dtype).eps
        at = got
    assert torch.equal(at, first)
    with torch.no_grad():
        blocks[0].W_out.zero_()
    assert torch.equal(dec.step(x), first)      # held as they were ...
    dec.requantize()
    assert not torch.equal(dec.step(x), first)  # ... until they are rounded again


@gpu
@pytest.mark.parametrize("weights", ["16bit", "int4"])
def test_decoder_first_stepped_in_inference_mode(weights):
    blocks = [block(576, 76, 192, 6, 2, torch.bfloat16).cuda() for _ in range(2)]
    dec = StackedMoEDecoder(blocks, weights=weights)
    x = torch.randn(5, 576, device="cuda").bfloat16()
    with torch.inference_mode():
        want = dec.step(x).clone()
        held = x.clone()
    assert torch.equal(dec.step(x), want) and torch.equal(dec.step(held), want)
    with torch.inference_mode():
        assert torch.equal(dec.step(x), want)


@gpu
def test_decoder_packs_its_weights_on_the_callers_stream(monkeypatch):
    """What a replay reads belongs to the stream that it runs on: weights packed during the warm-up were the warm-up
    stream's, and could be handed out again on it while a replay still read them."""
    from nanospeaker_b200 import int4
    seen = []
    pack = int4.quantize_int4
    monkeypatch.setattr(int4, "quantize_int4", lambda *a: (seen.append(torch.cuda.current_stream()), pack(*a))[1])
    dec = StackedMoEDecoder([block(64, 8, 96, 2, 1, torch.bfloat16).cuda() for _ in range(2)], weights="int4")
    x = torch.randn(5, 64, device="cuda").bfloat16()
    mine = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), mine):
        seen.clear()
        dec.requantize()
        with torch.cuda.stream(stream):
            dec.step(x)
        assert len(seen) == 8 and all(s == stream for s in seen)
    torch.cuda.synchronize()


@gpu
def test_trained_with_dropout_on_grouped_products_then_served_in_4_bits():
    """The set as it is used: a wide block trained for a few steps inside the sublayer with dropout, its
    experts rounded to 4 bits, and the decode stack run on them."""
    torch.manual_seed(0)
    m = block(128, 16, 384, 2, 1, torch.bfloat16, capacity_factor="auto").cuda()
    m.grouped = True
    sub = MoEFFNSublayer(m, dropout=0.1).to(torch.bfloat16).cuda().train()
    x = torch.randn(500, 128, device="cuda").bfloat16()
    assert m.capacity_factor is None and m._grouped_ok(x) and not m._kernels_take(x)
    opt = torch.optim.SGD(sub.parameters(), lr=1e-2)
    for _ in range(3):
        opt.zero_grad()
        out, aux = sub(x)
        (out.float().square().mean() + aux.float()).backward()
        assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in sub.parameters())
        opt.step()
    dec = StackedMoEDecoder([m], weights="int4", group=128)
    got, want = dec.step(x[:5]), layer_in_4_bits(m, x[:5], 128)
    off = (got.double() - want).norm(dim=1) / want.norm(dim=1)
    assert float(off.max()) < 3 * torch.finfo(torch.bfloat16).eps
    from nanospeaker_b200 import kernels
    kernels.check_status("cuda")
