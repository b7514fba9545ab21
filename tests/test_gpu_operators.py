"""The ragged grouped products, 4-bit weights and dropout on the GPU, against their definitions in 64 bits.

Bounds, derived and not fitted. A sum of n products in fp32 whose partial sums are rounded (or cut) once per
addition is off by at most n * 2^-23 * S, S the sum of the products' magnitudes; the result is then rounded to
its type, by at most half a step (eps / 2 of the value). Both together, with the value's own magnitude
enlarged by the first: |got - exact| <= (eps / 2) * (|exact| + a) + a, a = n * 2^-23 * S. Results below the
type's normal range add half of its smallest step."""
import pytest
import torch

from nanospeaker_b200 import (Int4Weight, dropout_add, grouped_mm, int4_experts, int4_mm, kernels,
                              quantize_int4)

pytestmark = pytest.mark.gpu

HALF = (torch.bfloat16, torch.float16)


def within(got, exact, n, magnitude, extra=0.0):
    """got against exact (64 bits) under the bound above; extra: an error of the sum's inputs."""
    t = got.dtype
    a = n * 2.0 ** -23 * magnitude + extra
    bound = torch.finfo(t).eps / 2 * (exact.abs() + a) + a + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    off = (got.double() - exact).abs()
    assert got.shape == exact.shape
    assert bool((off <= bound).all()), f"off by up to {float((off / bound).max()):.2f} bounds"



def randn(*shape, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


# ------------------------------------------------------------------------------------- grouped_mm
def runs(counts, before=0, behind=0):
    cut = [before]
    for c in counts:
        cut.append(cut[-1] + c)
    return torch.tensor(cut, dtype=torch.int32, device="cuda"), cut[-1] + behind


def exact_grouped(x, w, off, dy=None):
    """(y, S of y), and with dy the gradients with theirs, by a loop over the runs in 64 bits."""
    cut = off.tolist()
    r, (g, k, n) = x.shape[0], w.shape
    d = dict(dtype=torch.float64, device="cuda")
    y, ys = torch.zeros(r, n, **d), torch.zeros(r, n, **d)
    dx, dxs = torch.zeros(r, k, **d), torch.zeros(r, k, **d)
    dw, dws = torch.zeros(g, k, n, **d), torch.zeros(g, k, n, **d)
    for i, (a, b) in enumerate(zip(cut, cut[1:])):
        xi, wi = x[a:b].double(), w[i].double()
        y[a:b], ys[a:b] = xi @ wi, xi.abs() @ wi.abs()
        if dy is not None:
            di = dy[a:b].double()
            dx[a:b], dxs[a:b] = di @ wi.T, di.abs() @ wi.abs().T
            dw[i], dws[i] = xi.T @ di, xi.abs().T @ di.abs()
    return (y, ys) if dy is None else (y, ys, dx, dxs, dw, dws)


def check_grouped(x, w, off, dy):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = grouped_mm(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ey, ys, edx, dxs, edw, dws = exact_grouped(x.detach(), w.detach(), off, dy)
    within(y.detach(), ey, w.shape[1], ys)
    within(dx, edx, w.shape[2], dxs)
    within(dw, edw, x.shape[0], dws)
    kernels.check_status("cuda")
    return y.detach(), dx, dw


@pytest.mark.parametrize("counts", [[1], [0, 0, 5], [128, 256, 64], [1, 127, 129, 0, 63, 65, 255, 257, 33, 32, 31],
                                    [0], [300, 0, 0, 300], [512] * 3])
@pytest.mark.parametrize("k,n", [(64, 64), (8, 8), (72, 264), (200, 136), (576, 256)])
@pytest.mark.parametrize("dtype", HALF)
def test_grouped_both_directions(counts, k, n, dtype):
    off, r = runs(counts)
    check_grouped(randn(r, k, dtype=dtype), randn(len(counts), k, n, dtype=dtype, seed=1) * k ** -0.5, off,
                  randn(r, n, dtype=dtype, seed=2))


@pytest.mark.parametrize("r", [1, 2, 37, 300, 2000])
def test_grouped_many_groups_mostly_empty(r):
    """More groups than rows, and the most groups there may be."""
    for g in (76, 1024):
        of = torch.randint(0, g, (r,), device="cuda")
        off = torch.cat([of.new_zeros(1), torch.bincount(of, minlength=g).cumsum(0)]).int()
        check_grouped(randn(r, 64), randn(g, 64, 72, seed=1), off, randn(r, 72, seed=2))


def test_grouped_long_runs_are_split_and_joined():
    """Runs of many chunks in the weight gradient, one of them collapsed onto a single group."""
    for counts in ([9000, 1, 0, 3333], [0, 12345, 0]):
        off, r = runs(counts)
        _, _, dw = check_grouped(randn(r, 64), randn(len(counts), 64, 40, seed=1), off, randn(r, 40, seed=2))
        x, w = randn(r, 64), randn(len(counts), 64, 40, seed=1).requires_grad_()
        again, = torch.autograd.grad(grouped_mm(x, w, off), w, randn(r, 40, seed=2))
        assert torch.equal(dw, again)     # a fixed order of the sum


def test_grouped_wide_band_walk():
    """More row tiles than a band holds, several column tiles, both tile widths."""
    for k, n in ((64, 1032), (64, 520)):
        off, r = runs([5000, 700])
        check_grouped(randn(r, k), randn(2, k, n, seed=1) * k ** -0.5, off, randn(r, n, seed=2))


@pytest.mark.parametrize("dtype", HALF)
def test_grouped_transposed_weights_in_place(dtype):
    off, r = runs([70, 0, 200])
    stored = randn(3, 136, 72, dtype=dtype, seed=1)              # [G, N, K]
    w = stored.transpose(1, 2)
    _, _, dw = check_grouped(randn(r, 72, dtype=dtype), w, off, randn(r, 136, dtype=dtype, seed=2))
    assert dw.stride() == (136 * 72, 1, 72)                      # the gradient lies as the weight does


def test_grouped_strides_and_offsets_of_views():
    """Rows of a wider matrix, matrices of a wider stack, a view that does not start on 16 bytes, an
    expanded weight and an expanded gradient."""
    off, r = runs([50, 90])
    wide = randn(r, 200)
    stack = randn(2, 64, 160, seed=1)
    base = randn(r * 64 + 1, seed=3)
    for x in (wide[:, 8:72], wide[:, 3:67], base[1:].view(r, 64), randn(64, r).T):
        for w in (stack[:, :, 16:88], stack[:, :, 3:75], stack[:1, :, :72].expand(2, -1, -1)):
            dy = randn(r, 72, seed=2)
            check_grouped(x, w, off, dy)
    x, w = randn(r, 64).requires_grad_(), stack[:, :, :72].detach().requires_grad_()
    grouped_mm(x, w, off).sum().backward()                       # a gradient with strides of zero
    ones = torch.ones(r, 72, device="cuda", dtype=torch.bfloat16)
    _, _, edx, dxs, edw, dws = exact_grouped(x.detach(), w.detach(), off, ones)
    within(x.grad, edx, 72, dxs)
    within(w.grad, edw, r, dws)


def test_grouped_one_group_is_a_plain_product():
    off, r = runs([333])
    check_grouped(randn(r, 128), randn(1, 128, 96, seed=1), off, randn(r, 96, seed=2))


def test_grouped_rows_of_no_run_are_zero():
    off, r = runs([40, 0, 90], before=17, behind=300)
    x, w = randn(r, 64), randn(3, 64, 72, seed=1)
    x[:17], x[147:] = float("nan"), float("inf")                 # never looked at
    x.requires_grad_(), w.requires_grad_()
    y = grouped_mm(x, w, off)
    dy = randn(r, 72, seed=2)
    dy[:17], dy[147:] = float("inf"), float("nan")
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for t in (y, dx):
        assert (t[:17] == 0).all() and (t[147:] == 0).all()
    _, _, _, _, edw, dws = exact_grouped(x.detach(), w.detach(), off, dy)
    within(dw, edw, 130, dws)


def test_grouped_what_is_not_finite_stays_in_its_run():
    """Infinities and NaN of one run reach neither its neighbours' rows nor their weight gradients."""
    off, r = runs([33, 10, 70])
    x, w = randn(r, 64), randn(3, 64, 72, seed=1)
    dy = randn(r, 72, seed=2)
    x[33], x[35], dy[34], dy[40] = float("inf"), float("nan"), float("-inf"), float("nan")
    x.requires_grad_(), w.requires_grad_()
    y = grouped_mm(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    other = torch.cat([torch.arange(33), torch.arange(43, r)]).cuda()
    clean_x, clean_dy = x.detach().clone(), dy.clone()
    clean_x[33:43], clean_dy[33:43] = 0, 0
    ey, ys, edx, dxs, edw, dws = exact_grouped(clean_x, w.detach(), off, clean_dy)
    within(y.detach()[other], ey[other], 64, ys[other])
    within(dx[other], edx[other], 72, dxs[other])
    within(dw[[0, 2]], edw[[0, 2]], r, dws[[0, 2]])
    assert not torch.isfinite(dw[1]).any() and not torch.isfinite(y[33]).any()


def test_grouped_offsets_out_of_range_are_taken_into_range_and_reported():
    x, w = randn(100, 64), randn(3, 64, 72, seed=1)
    for bad, good in (([0, 50, 30, 100], [0, 50, 50, 100]), ([-5, 20, 60, 1000], [0, 20, 60, 100]),
                      ([0, 2 ** 31 - 1, -2 ** 31, 5], [0, 100, 100, 100])):
        bad, good = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (bad, good))
        y = grouped_mm(x, w, bad)
        with pytest.raises(RuntimeError, match="runs decrease or leave"):
            kernels.check_status("cuda")
        assert torch.equal(y, grouped_mm(x, w, good))
        kernels.check_status("cuda")
        dw = kernels.grouped_wgrad(x, y, bad)
        with pytest.raises(RuntimeError, match="runs decrease or leave"):
            kernels.check_status("cuda")
        assert torch.equal(dw, kernels.grouped_wgrad(x, y, good))


def test_grouped_without_rows():
    w = randn(2, 64, 72).requires_grad_()
    x = randn(0, 64).requires_grad_()
    y = grouped_mm(x, w, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert y.shape == (0, 72)
    y.sum().backward()
    assert x.grad.shape == (0, 64) and (w.grad == 0).all()


def test_grouped_gradient_against_differences():
    """A central difference of sum(y * dy) in one direction of each input, in 64 bits on the outputs: the
    product is linear in x and in w, so the difference is exact but for the outputs' rounding."""
    off, r = runs([20, 45])
    x, w, dy = randn(r, 64), randn(2, 64, 72, seed=1), randn(r, 72, seed=2)
    vx, vw = randn(r, 64, seed=3), randn(2, 64, 72, seed=4)
    _, dx, dw = check_grouped(x, w, off, dy)
    for v, grad, call in ((vx, dx, lambda s: grouped_mm(s, w, off)), (vw, dw, lambda s: grouped_mm(x, s, off))):
        at = call(v).double()                      # linear: the directional derivative itself
        slope = float((at * dy.double()).sum())
        # both sums of products of 16-bit values rounded by at most 2^-9 (half a step of bf16's 2^-8 relative)
        room = 2.0 ** -8 * float((at.abs() * dy.double().abs()).sum() + (grad.double().abs() * v.double().abs()).sum())
        assert abs(slope - float((grad.double() * v.double()).sum())) <= room


def test_grouped_graph_replays_and_other_streams():
    """Captured once, replayed on new inputs; two streams at a time."""
    off, r = runs([100, 0, 333, 67])
    x, w, dy = randn(r, 64), randn(4, 64, 72, seed=1), randn(r, 72, seed=2)
    run = lambda: (grouped_mm(x, w, off), kernels.grouped_wgrad(x, dy, off))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in (5, 6):
        x.copy_(randn(r, 64, seed=seed))
        cut = torch.tensor([0, 10 * seed, 200, 200, 490], dtype=torch.int32, device="cuda")
        off.copy_(cut)
        graph.replay()
        want = run()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([run() for _ in range(5)])
    torch.cuda.synchronize()
    for each in got:
        for pair in each:
            assert all(torch.equal(a, b) for a, b in zip(pair, want))


# ------------------------------------------------------------------------------------ 4-bit weights
def levels(shape, group, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    k, n = shape[-2:]
    q = torch.randint(0, 16, shape, generator=g, device="cuda", dtype=torch.uint8)
    s = torch.rand((*shape[:-2], -(-k // group), n), generator=g, device="cuda") + 0.5
    return q, (s * k ** -0.5 / 4).to(dtype)


def exact_weight(q, s, group):
    row = torch.arange(q.shape[-2], device=q.device) // group
    return (q.double() - 8) * s.double().index_select(-2, row)


@pytest.mark.parametrize("rows", [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 200])
@pytest.mark.parametrize("k,n,group", [(64, 16, 64), (8, 1, 32), (1000, 1537, 32), (576, 100, 64),
                                       (4096, 48, 128), (136, 33, 128), (192, 40, 128)])
@pytest.mark.parametrize("dtype", HALF)
def test_int4_mm(rows, k, n, group, dtype):
    q, s = levels((k, n), group, dtype)
    x = randn(rows, k, dtype=dtype)
    y = int4_mm(x, Int4Weight.from_levels(q, s, group))
    w = exact_weight(q, s, group)
    # (each scale group's sum is multiplied once more: 2 roundings a group, within n = 2 k)
    within(y, x.double() @ w, 2 * k, x.double().abs() @ w.abs())


def test_int4_mm_shapes_and_strides():
    q, s = levels((72, 40), 32, torch.bfloat16)
    w = Int4Weight.from_levels(q, s, 32)
    x = randn(2, 3, 72)
    assert torch.equal(int4_mm(x, w).view(6, 40), int4_mm(x.view(6, 72), w))
    assert torch.equal(int4_mm(x[0, 0], w), int4_mm(x[0], w)[0])
    assert int4_mm(x[:0], w).shape == (0, 3, 40)
    wide = randn(5, 200)
    for view in (wide[:, 8:80], wide[:, 3:75]):
        assert torch.equal(int4_mm(view, w), int4_mm(view.contiguous(), w))
    assert torch.equal(int4_mm(randn(72, 5).T, w), int4_mm(randn(72, 5).T.contiguous(), w))


def test_int4_mm_rows_do_not_mix():
    """What is not finite in one row stays there."""
    q, s = levels((128, 64), 64, torch.bfloat16)
    w = Int4Weight.from_levels(q, s, 64)
    x = randn(9, 128)
    want = int4_mm(x, w)
    x[4] = float("inf")
    got = int4_mm(x, w)
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.equal(got[keep], want[keep]) and not torch.isfinite(got[4]).all()


def test_int4_has_no_gradients():
    q, s = levels((64, 32), 64, torch.bfloat16)
    w = Int4Weight.from_levels(q, s, 64)
    x = randn(2, 64).requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        int4_mm(x, w)
    with torch.no_grad():
        int4_mm(x, w)


def act64(name, g):
    return {"silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * torch.special.ndtr(v),
            "relu": torch.relu, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[name](g)


def act_slope(name):
    """The largest magnitude of the activation's derivative."""
    return {"silu": 1.1, "gelu": 1.13, "relu": 1.0, "sigmoid": 0.25, "tanh": 1.0}[name]


def exact_experts(x, tw, idx, w_in, w_out, sh, act, dtype):
    """(out, its error bound apart from the final rounding): sums of the first product off by
    2 D 2^-23 S each; the activation, whose own evaluation is within 2^-19 of its value plus 2^-20 (fast exp
    and division: a few units of 2^-22, and 2^-22 of |g| <= 16 in the exponent); the hidden value rounded to
    the type; the second product's sum; the sum over the pairs."""
    e, d, h2 = w_in.shape
    u = torch.finfo(dtype).eps / 2
    out, err = torch.zeros_like(x), torch.zeros_like(x)

    def mlp(rows, wi, wo):
        a, s = rows @ wi, rows.abs() @ wi.abs()
        da = 2 * d * 2.0 ** -23 * s
        g, up = a.chunk(2, dim=-1)
        dg, du = da.chunk(2, dim=-1)
        act_v = act64(act, g)
        d_act = act_slope(act) * dg + 2.0 ** -19 * act_v.abs() + 2.0 ** -20 * (1 + g.abs())
        hid = act_v * up
        d_hid = d_act * (up.abs() + du) + act_v.abs() * du
        d_hid = d_hid + u * (hid.abs() + d_hid) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        y, ys = hid @ wo, (hid.abs() + d_hid) @ wo.abs()
        return y, d_hid @ wo.abs() + 2 * (h2 // 2) * 2.0 ** -23 * ys

    for i in range(e):
        tok, slot = (idx == i).nonzero(as_tuple=True)
        if tok.numel():
            y, dy = mlp(x[tok], w_in[i], w_out[i])
            w = tw.double()[tok, slot, None]
            out.index_add_(0, tok, y * w)        # (a token may have an expert twice)
            err.index_add_(0, tok, (dy + 16 * 2.0 ** -23 * (y.abs() + dy)) * w.abs())
    for wi, wo in sh:
        y, dy = mlp(x, wi, wo)
        out += y
        err += dy + 16 * 2.0 ** -23 * (y.abs() + dy)
    return out, err


def experts_case(t, d, h, e, k, s, group, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = randn(t, d, dtype=dtype, seed=seed)
    idx = torch.rand((t, e), generator=g, device="cuda").argsort(1)[:, :k].contiguous()
    tw = torch.rand((t, k), generator=g, device="cuda").to(dtype)
    raw = {}
    for i, (name, shape) in enumerate((("w_in", (e, d, 2 * h)), ("w_out", (e, h, d)), ("shared_in", (s, d, 2 * h)),
                                       ("shared_out", (s, h, d)))):
        raw[name] = levels(shape, group, dtype, seed + 10 + i) if shape[0] else None
    packed = {n: None if v is None else Int4Weight.from_levels(*v, group) for n, v in raw.items()}
    plain = {n: None if v is None else exact_weight(*v, group) for n, v in raw.items()}
    return x, tw, idx, packed, plain


def check_experts(x, tw, idx, packed, plain, act="silu"):
    out = int4_experts(x, tw, idx, packed["w_in"], packed["w_out"], act, packed["shared_in"],
                       packed["shared_out"])
    sh = [] if plain["shared_in"] is None else list(zip(plain["shared_in"], plain["shared_out"]))
    want, err = exact_experts(x.double(), tw, idx, plain["w_in"], plain["w_out"], sh, act, x.dtype)
    within(out, want, 0, torch.zeros((), device="cuda"), extra=err)
    return out


@pytest.mark.parametrize("t", [1, 2, 5, 64, 65, 129, 300])
@pytest.mark.parametrize("d,h,e,k,s,group", [(576, 128, 76, 6, 2, 64), (64, 16, 4, 2, 0, 32), (200, 48, 3, 1, 1, 128),
                                             (1024, 64, 8, 8, 1, 64)])
def test_int4_experts(t, d, h, e, k, s, group):
    for dtype in HALF:
        check_experts(*experts_case(t, d, h, e, k, s, group, dtype))
    kernels.check_status("cuda")


@pytest.mark.parametrize("act", ["silu", "swish", "gelu", "relu", "sigmoid", "tanh"])
def test_int4_experts_activations(act):
    case = experts_case(20, 128, 32, 6, 2, 1, 64, torch.bfloat16)
    check_experts(*case, act={"swish": "silu"}.get(act, act))
    if act == "swish":
        x, tw, idx, p, _ = case
        assert torch.equal(int4_experts(x, tw, idx, p["w_in"], p["w_out"], "swish"),
                           int4_experts(x, tw, idx, p["w_in"], p["w_out"], "silu"))


@pytest.mark.parametrize("t,e", [(30, 1), (30, 2), (8, 1), (64, 2), (200, 8), (1300, 3)])
def test_int4_experts_place_of_a_row_changes_nothing(t, e):
    """Tokens in another order, and again: bit for bit the same rows, in whatever place of a tile or pass they come."""
    d, h = 1024, 64
    w_in, w_out = quantize_int4(randn(e, d, 2 * h)), quantize_int4(randn(e, h, d, seed=1))
    gen = torch.Generator(device="cuda").manual_seed(5)
    x, idx = randn(t, d, seed=2), torch.randint(0, e, (t, 1), device="cuda", generator=gen)
    tw = torch.rand(t, 1, device="cuda", generator=gen).to(torch.bfloat16)
    want = int4_experts(x, tw, idx, w_in, w_out)
    for seed in range(3):
        order = torch.randperm(t, device="cuda", generator=gen)
        assert torch.equal(int4_experts(x[order], tw[order], idx[order], w_in, w_out), want[order])
        assert torch.equal(int4_experts(x, tw, idx, w_in, w_out), want)


def test_int4_experts_windows_of_pairs():
    """More pairs than one look at the expert ids takes, all on one expert or spread."""
    x, tw, idx, packed, plain = experts_case(1500, 64, 16, 5, 3, 1, 64, torch.bfloat16)
    check_experts(x, tw, idx, packed, plain)
    one = torch.zeros_like(idx[:, :1]) + 3
    check_experts(x, tw[:, :1].contiguous(), one, packed, plain)


def test_int4_experts_same_expert_twice_and_ids_out_of_range():
    x, tw, idx, packed, plain = experts_case(10, 64, 16, 4, 3, 0, 32, torch.float16)
    idx[3] = torch.tensor([2, 2, 2])
    check_experts(x, tw, idx, packed, plain)
    kernels.check_status("cuda")
    for bad in (-1, 4, 2 ** 40):
        idx[5, 1] = bad
        check_experts(x, tw, idx, packed, plain)
        with pytest.raises(RuntimeError, match="expert id"):
            kernels.check_status("cuda")


def test_int4_experts_views_and_empty():
    x, tw, idx, p, _ = experts_case(12, 64, 16, 4, 2, 1, 64, torch.bfloat16)
    call = lambda *a: int4_experts(*a, p["w_in"], p["w_out"], "silu", p["shared_in"], p["shared_out"])  # noqa: E731
    want = call(x, tw, idx)
    assert torch.equal(call(torch.cat([x, x], 1)[:, 64:], tw.T.contiguous().T, idx.T.contiguous().T), want)
    assert torch.equal(call(x[:4], tw[:4], idx[:4]), want[:4])
    assert call(x[:0], tw[:0], idx[:0]).shape == (0, 64)


def test_int4_graph_replays_on_new_inputs():
    x, tw, idx, p, _ = experts_case(16, 64, 32, 8, 2, 1, 64, torch.bfloat16)
    w = quantize_int4(randn(64, 200))
    run = lambda: (int4_experts(x, tw, idx, p["w_in"], p["w_out"], "silu", p["shared_in"], p["shared_out"]),  # noqa: E731
                   int4_mm(x, w))
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in (1, 2):
        x.copy_(randn(16, 64, seed=seed))
        idx.copy_((idx + seed) % 8)
        graph.replay()
        for a, b in zip(out, run()):
            assert torch.equal(a, b)


# ----------------------------------------------------------------------------------------- dropout
def words(n, seed, call):
    """The generator in Python integers, for every element of a small tensor."""
    out = []
    for quad in range((n + 3) // 4):
        c = [quad & 0xFFFFFFFF, quad >> 32, call & 0xFFFFFFFF, (call >> 32) & 0xFFFFFFFF]
        k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
        for _ in range(10):
            a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        out += c
    return torch.tensor(out[:n], device="cuda")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1,), (3, 5), (8,), (7, 33), (2, 3, 128), (1025,)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999])
def test_dropout_is_the_generators_mask(dtype, shape, p):
    seed, call = 0x1234567890ABCDEF, -7
    rng = torch.tensor([seed, call], device="cuda")
    x, res, dout = (randn(*shape, dtype=dtype, seed=i) for i in range(3))
    keep = (words(x.numel(), seed, call) >= min(round(p * 2 ** 32), 2 ** 32 - 1)).view(shape)
    for residual in (res, None):
        a = x.clone().requires_grad_()
        b = None if residual is None else residual.clone().requires_grad_()
        out = dropout_add(a, b, p, rng)
        base = 0.0 if residual is None else residual.double()
        part = torch.where(keep, x.double() / (1 - p), 0.0)
        # the scale is rounded to fp32, the product and the sum once more: 4 units of 2^-24
        within(out.detach(), base + part, 2, part.abs() + (0 if residual is None else residual.double().abs()))
        out.backward(dout)
        part = torch.where(keep, dout.double() / (1 - p), 0.0)
        within(a.grad, part, 2, part.abs())
        assert (a.grad[~keep] == 0).all()
        if b is not None:
            assert torch.equal(b.grad, dout)


def test_dropout_share_and_independence():
    """Over 2^20 elements the share dropped is within 6 standard deviations of p, and masks of other calls
    or seeds agree in p^2 + (1 - p)^2 of the places."""
    n, p = 1 << 20, 0.3
    x = torch.ones(n, device="cuda")
    masks = []
    for state in ((1, 0), (1, 1), (2, 0), (1, 1 << 32)):
        out = dropout_add(x, None, p, torch.tensor(state, device="cuda"))
        masks.append(out == 0)
        assert abs(float(masks[-1].double().mean()) - p) < 6 * (p * (1 - p) / n) ** 0.5
    agree = p * p + (1 - p) ** 2
    for m in masks[1:]:
        assert abs(float((m == masks[0]).double().mean()) - agree) < 6 * (agree * (1 - agree) / n) ** 0.5


def test_dropout_backward_uses_the_forwards_state():
    """The state moves on between forward and backward; the mask does not."""
    rng = torch.tensor([5, 0], device="cuda")
    x = randn(1000, dtype=torch.float32).requires_grad_()
    out = dropout_add(x, None, 0.5, rng)
    rng[1] += 1
    out.sum().backward()
    assert torch.equal(x.grad != 0, out != 0)
    assert not torch.equal(dropout_add(x, None, 0.5, rng) != 0, out != 0)


def test_dropout_dropped_elements_add_nothing():
    rng = torch.tensor([3, 4], device="cuda")
    keep = dropout_add(torch.ones(4096, device="cuda"), None, 0.5, rng) != 0
    x = torch.where(keep, 1.0, float("nan")).bfloat16()
    res = torch.full((4096,), 0.25, device="cuda", dtype=torch.bfloat16)
    assert torch.isfinite(dropout_add(x, res, 0.5, rng)).all()
    x[~keep] = float("inf")
    out = dropout_add(x, res, 0.5, rng)
    assert (out[~keep] == 0.25).all() and (out[keep] == 2.25).all()


def test_dropout_views_and_empty():
    """Elements are numbered in row-major order of the shape, whatever the strides and the alignment."""
    rng = torch.tensor([1, 2], device="cuda")
    x = randn(40, 24)
    want = dropout_add(x, x, 0.4, rng)
    assert torch.equal(dropout_add(x.T.contiguous().T, x, 0.4, rng), want)
    shifted = torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(40, 24)
    assert torch.equal(dropout_add(shifted, shifted, 0.4, rng), want)
    e = torch.empty(0, 4, device="cuda").requires_grad_()
    dropout_add(e, None, 0.1, rng).sum().backward()
    assert e.grad.shape == (0, 4)


def test_dropout_gradient_of_the_gradient():
    """Linear: the second derivative goes through the same mask."""
    rng = torch.tensor([1, 2], device="cuda")
    x = randn(256, dtype=torch.float32).requires_grad_()
    v = randn(256, dtype=torch.float32, seed=1).requires_grad_()
    g, = torch.autograd.grad(dropout_add(x, None, 0.5, rng), x, v, create_graph=True)
    h, = torch.autograd.grad(g.sum(), v)
    assert torch.equal(h != 0, g != 0) and torch.allclose(h[h != 0], torch.tensor(2.0, device="cuda"))


def test_dropout_graph_replays_move_on():
    """The state is read, and counted up, on the device: every replay has another mask."""
    rng = torch.tensor([9, 0], device="cuda")
    x = torch.ones(4096, device="cuda")
    dropout_add(x, None, 0.5, rng)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = dropout_add(x, None, 0.5, rng)
        rng[1].add_(1)
    seen = []
    for call in range(3):
        graph.replay()
        assert torch.equal(out, dropout_add(x, None, 0.5, torch.tensor([9, call], device="cuda")))
        seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


# ------------------------------------------------------------------------------ traced and captured
def test_registered_ops_check_out():
    """Schemas, fake kernels and autograd of the ops that traced calls see."""
    off, r = runs([20, 0, 13])
    ops = torch.ops.moe_b200
    check = lambda op, args: torch.library.opcheck(  # noqa: E731
        op, args, test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
    x, w = randn(r, 64).requires_grad_(), randn(3, 64, 72, seed=1).requires_grad_()
    check(ops.grouped_mm, (x, w, off))
    check(ops.grouped_wgrad, (x.detach(), randn(r, 72), off))
    rng = torch.tensor([1, 2], device="cuda")
    check(ops.dropout_add, (x, randn(r, 64, seed=2).requires_grad_(), 0.3, rng))
    check(ops.dropout_bwd, (x, 0.3, rng))
    q = quantize_int4(randn(64, 40))
    check(ops.int4_mm, (x.detach(), q.data, q.group, 40))
    xx, tw, idx, p, _ = experts_case(6, 64, 16, 4, 2, 1, 64, torch.bfloat16)
    check(ops.int4_experts, (xx, tw, idx, p["w_in"].data, p["w_out"].data, p["shared_in"].data,
                             p["shared_out"].data, 16, 64, 0))


def test_registered_ops_give_what_the_eager_calls_give():
    """The two ways into the same kernels, gradients included."""
    off, r = runs([20, 0, 13])
    rng = torch.tensor([1, 2], device="cuda")
    res = randn(r, 72, seed=4)
    for layout in (lambda w: w, lambda w: w.transpose(1, 2).contiguous().transpose(1, 2)):
        both = []
        for mm, drop in ((grouped_mm, dropout_add),
                         (torch.ops.moe_b200.grouped_mm, lambda *a: torch.ops.moe_b200.dropout_add(*a)[0])):
            x, w = randn(r, 64).requires_grad_(), layout(randn(3, 64, 72, seed=1)).requires_grad_()
            b = res.clone().requires_grad_()
            out = drop(mm(x, w, off), b, 0.25, rng)
            both.append((out.detach(), *torch.autograd.grad(out, (x, w, b), randn(r, 72, seed=2))))
        assert all(torch.equal(a, b) for a, b in zip(*both))
    q = quantize_int4(randn(64, 40))
    assert torch.equal(int4_mm(x.detach(), q), torch.ops.moe_b200.int4_mm(x.detach(), q.data, q.group, 40))


def test_second_gradients_of_grouped_products_are_refused():
    off, r = runs([20, 13])
    x, w = randn(r, 64).requires_grad_(), randn(2, 64, 72, seed=1).requires_grad_()
    dx, = torch.autograd.grad(grouped_mm(x, w, off), x, randn(r, 72, seed=2), create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        dx.sum().backward()


def test_training_step_in_a_graph():
    """Forward and gradients captured and replayed on new inputs. (No eager graph of the same leaves may be
    alive meanwhile: torch's engine then joins the leaves' stream to the capture, with any op, and the capture
    fails with an error.)"""
    off, r = runs([100, 0, 57])
    x, w = randn(r, 64).requires_grad_(), randn(3, 64, 72, seed=1).requires_grad_()
    dy, rng = randn(r, 72, seed=2), torch.tensor([3, 0], device="cuda")
    step = lambda: torch.autograd.grad(dropout_add(grouped_mm(x, w, off), None, 0.5, rng), (x, w), dy)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.no_grad():
        x.copy_(randn(r, 64, seed=7))
        rng[1] = 5
    graph.replay()
    for a, b in zip(got, step()):
        assert torch.equal(a, b)


def test_graphs_of_two_calls_share_nothing():
    """Two captured graphs of split weight gradients and of experts, replayed in turn and at once on two
    streams."""
    off, r = runs([3000, 10])
    x, y = randn(r, 64), randn(r, 40, seed=2)
    e = experts_case(16, 64, 32, 8, 2, 1, 64, torch.bfloat16)
    run = lambda: (kernels.grouped_wgrad(x, y, off),  # noqa: E731
                   int4_experts(e[0], e[1], e[2], e[3]["w_in"], e[3]["w_out"], "silu", e[3]["shared_in"],
                                e[3]["shared_out"]))
    want = run()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


# --------------------------------------------------------------------------- places past 31 and 32 bits
def test_grouped_results_past_two_to_the_31():
    """More than 2^31 values in y and in dw: what lies at the ends is what a small call gives."""
    r, n = 540_000, 4096
    x, w = randn(r, 8), randn(2, 8, n, seed=1)
    off = torch.tensor([0, r - 300, r], dtype=torch.int32, device="cuda")
    y = grouped_mm(x, w, off)
    assert y.numel() > 2 ** 31
    tail = torch.tensor([0, 100, 400], dtype=torch.int32, device="cuda")
    assert torch.equal(y[-400:], grouped_mm(x[-400:].contiguous(), w, tail))
    del y
    g, m, n = 260, 2048, 4096
    a, b = randn(40, m), randn(40, n, seed=1)
    off = torch.full((g + 1,), 40, dtype=torch.int32, device="cuda")
    off[:g - 1] = 0
    off[g - 1] = 25
    dw = kernels.grouped_wgrad(a, b, off)
    assert dw.numel() > 2 ** 31
    small = kernels.grouped_wgrad(a, b, torch.tensor([0, 25, 40], dtype=torch.int32, device="cuda"))
    assert torch.equal(dw[-2:], small) and not dw[0].any() and not dw[g // 2].any()


def test_experts_past_two_to_the_32_levels():
    """The last of 2300 experts, whose levels lie beyond 2^32, is what the same weights are in the first place."""
    d, h, e = 1024, 1024, 2300
    one_in, one_out = quantize_int4(randn(1, d, 2 * h)), quantize_int4(randn(1, h, d, seed=1))
    many = [Int4Weight(torch.zeros(e, w.data.shape[1], dtype=torch.uint8, device="cuda"), (e, *w.shape[1:]), 64,
                       torch.bfloat16) for w in (one_in, one_out)]
    for big, w in zip(many, (one_in, one_out)):
        big.data[0] = big.data[-1] = w.data[0]
    assert e * d * 2 * h > 2 ** 32
    x, tw = randn(3, d), torch.ones(3, 1, device="cuda", dtype=torch.bfloat16)
    idx = torch.full((3, 1), e - 1, device="cuda")
    want = int4_experts(x, tw, torch.zeros_like(idx), *many)
    assert torch.equal(int4_experts(x, tw, idx, *many), want) and bool(want.any())


def test_dropout_past_two_to_the_31_elements():
    n = 2 ** 31 + 12_345
    rng = torch.tensor([7, 9], device="cuda")
    out = dropout_add(torch.ones(n, dtype=torch.float16, device="cuda"), None, 0.5, rng)
    for at in (2 ** 31 - 8, n - 9):
        for i in range(at, at + 8):
            c, k = [(i // 4) & 0xFFFFFFFF, (i // 4) >> 32, 9, 0], [7, 0]
            for _ in range(10):
                a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
                c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
                k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
            assert float(out[i]) == (2.0 if c[i % 4] >= 2 ** 31 else 0.0)


def test_int4_mm_many_rows():
    """More rows than one grid line of passes, of which each is 32 rows."""
    q, s = levels((64, 48), 64, torch.bfloat16)
    w = Int4Weight.from_levels(q, s, 64)
    x = randn(40_000, 64)
    y = int4_mm(x, w)
    ew = exact_weight(q, s, 64)
    within(y, x.double() @ ew, 128, x.double().abs() @ ew.abs())


# --------------------------------------------------------------------------- two calls at once
def test_calls_on_two_streams_at_once():
    """The operators on two streams that do not wait for one another, fifty times: what each gives alone."""
    x, w = randn(900, 256), randn(6, 256, 192, seed=1)
    off = torch.tensor([0, 300, 300, 305, 705, 800, 900], dtype=torch.int32, device="cuda")
    dy = randn(900, 192, seed=2)
    d, h, e = 576, 128, 16
    w_in, w_out = quantize_int4(randn(e, d, 2 * h)), quantize_int4(randn(e, h, d, seed=1))
    t, tw = randn(40, d, seed=3), torch.full((40, 4), 0.25, device="cuda", dtype=torch.bfloat16)
    idx = torch.rand(40, e, device="cuda").topk(4).indices
    rng = torch.tensor([3, 4], device="cuda")
    calls = [lambda: grouped_mm(x, w, off), lambda: kernels.grouped_wgrad(x, dy, off),
             lambda: int4_experts(t, tw, idx, w_in, w_out), lambda: dropout_add(x, None, 0.5, rng)]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(50):
        with torch.cuda.stream(streams[i % 2]):
            got.append([c() for c in (calls if i % 4 < 2 else calls[::-1])])
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for a, b in zip(outs if i % 4 < 2 else outs[::-1], want):
            assert torch.equal(a, b)
    kernels.check_status("cuda")
