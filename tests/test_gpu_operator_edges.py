"""The operators beside the block where the larger tests' bounds are too wide to see: inputs chosen so that all
sums but the one under test are exact, calls behind a reported one, and what is refused on the GPU."""
import pytest
import torch

from nanospeaker_b200 import Int4Weight, grouped_mm, int4_experts, int4_mm, kernels
from test_operators import host  # noqa: F401  (the schedule's arithmetic, compiled for the host)

pytestmark = pytest.mark.gpu

HALF = (torch.bfloat16, torch.float16)


def whole(lo, hi, *shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda")


# --------------------------------------------------------------------------- 4-bit products, bit for bit
@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 17, 32, 33, 64, 100])
@pytest.mark.parametrize("k,n,group", [(8, 1, 32), (72, 40, 32), (576, 100, 64), (1000, 1537, 32), (4096, 48, 128),
                                       (4104, 272, 64), (8192, 17, 128)])
@pytest.mark.parametrize("dtype", HALF)
def test_int4_mm_whole_numbers_are_exact(rows, k, n, group, dtype):
    """Rows of -2 .. 2 and scales of 1, 1/2, 1/4 and 1/8: every fp32 sum is exact (below 2^17, in steps of 2^-3), so
    the result is that of 64 bits, rounded once, bit for bit."""
    x, q = whole(-2, 2, rows, k), whole(0, 15, k, n, seed=1)
    s = 0.5 ** whole(0, 3, -(-k // group), n, seed=2).double()
    w = (q - 8).double() * s.repeat_interleave(group, 0)[:k]
    got = int4_mm(x.to(dtype), Int4Weight.from_levels(q.to(torch.uint8), s.to(dtype), group))
    assert torch.equal(got, (x.double() @ w).to(dtype))


# --------------------------------------------------------------------------- 4-bit experts: the hidden values
def whole_experts(t, d, h, e, group, dtype, reach=2):
    """Whole numbers throughout, rows of -reach .. reach: gates and hidden values (relu) are exact in fp32. Returns
    the call's arguments, the hidden values of every token and w_out's rows that they meet, in 64 bits."""
    x = whole(-reach, reach, t, d)
    q_in, q_out = whole(0, 15, e, d, 2 * h, seed=1), whole(0, 15, e, h, d, seed=2)
    s_in = torch.ones(e, -(-d // group), 2 * h, dtype=dtype, device="cuda")
    s_out = torch.full((e, -(-h // group), d), 2.0 ** -14, dtype=dtype, device="cuda")
    idx = whole(0, e - 1, t, 1, seed=3)
    pack = lambda q, s: Int4Weight.from_levels(q.to(torch.uint8), s, group)  # noqa: E731
    args = (x.to(dtype), torch.ones(t, 1, dtype=dtype, device="cuda"), idx, pack(q_in, s_in), pack(q_out, s_out))
    hid = torch.empty(t, h, dtype=torch.float64, device="cuda")
    down = torch.empty(t, h, d, dtype=torch.float64, device="cuda")
    for i in range(e):
        tok = (idx[:, 0] == i).nonzero()[:, 0]
        gate, up = (x[tok].double() @ (q_in[i] - 8).double()).chunk(2, 1)
        hid[tok] = gate.clamp(min=0) * up
        down[tok] = (q_out[i] - 8).double() * 2.0 ** -14
    return args, hid, down


def hidden_bound(args, hid, down):
    """(distance of the call's result from 64 bits, its bound, the result in 64 bits). The hidden value loses at most
    2^-15 of itself (its upper half is cut at 2^-7 of it, the rest rounded at 2^-8 of that); the second product's
    sum, two parts of h values and a scale per group, is off by 4 h 2^-23 of its magnitude; then one rounding."""
    assert bool((hid.abs() <= 2 ** 24).all())
    h, f = hid.shape[1], torch.finfo(args[0].dtype)
    exact = torch.einsum("th,thd->td", hid, down)
    magnitude = torch.einsum("th,thd->td", hid.abs(), down.abs())
    a = (4 * h * 2.0 ** -23 + 2.0 ** -15) * magnitude
    out = int4_experts(*args, "relu").double()
    kernels.check_status("cuda")
    return (out - exact).abs(), f.eps / 2 * (exact.abs() + a) + a + f.smallest_normal * f.eps, exact


@pytest.mark.parametrize("t,e", [(1, 1), (5, 2), (24, 2), (100, 3), (300, 4)])
@pytest.mark.parametrize("d,h,group", [(64, 16, 32), (64, 128, 64), (72, 272, 128), (64, 528, 64), (64, 720, 32)])
@pytest.mark.parametrize("dtype", HALF)
def test_int4_experts_hidden_values_are_not_held_in_the_type(t, e, d, h, group, dtype):
    """Bits below the type's: a bf16 hidden value does not hold the bound (in fp16 its 2^-11, summed up with
    either sign, may)."""
    args, hid, down = whole_experts(t, d, h, e, group, dtype)
    off, bound, exact = hidden_bound(args, hid, down)
    assert bool((off <= bound).all())
    if dtype == torch.bfloat16 and t * h >= 1000:
        held = torch.einsum("th,thd->td", hid.to(dtype).double(), down).to(dtype).double()
        assert not bool(((held - exact).abs() <= bound).all())


@pytest.mark.parametrize("t,d,h,e,group", [(1, 8, 16, 1, 32), (7, 8, 48, 3, 128), (33, 24, 16, 2, 64),
                                           (5000, 40, 80, 3, 64), (70, 584, 48, 300, 32), (20, 64, 1040, 2, 128),
                                           (9, 1096, 64, 3, 64), (2500, 64, 336, 40, 32)])
def test_int4_experts_smallest_widths_and_prompts(t, d, h, e, group):
    args, hid, down = whole_experts(t, d, h, e, group, torch.bfloat16)
    off, bound, _ = hidden_bound(args, hid, down)
    assert bool((off <= bound).all())


@pytest.mark.parametrize("t,h", [(5, 128), (60, 528), (300, 64)])
@pytest.mark.parametrize("dtype", HALF)
def test_int4_experts_hidden_values_past_the_types_range(t, h, dtype):
    """Hidden values that fp16 does not reach, results that it does."""
    args, hid, down = whole_experts(t, 64, h, 2, 64, dtype, reach=8)
    assert float(hid.abs().max()) > 65504
    off, bound, exact = hidden_bound(args, hid, down)
    assert float(exact.abs().max()) < 65504 and bool((off <= bound).all())


@pytest.mark.parametrize("t", [1, 12, 40])
def test_int4_experts_small_gates_of_tanh(t):
    """Gates of some 1e-5: tanh is right relative to its value (2 units of 2^-23 and fp32's rounding of the product:
    2^-21), not to one. tanh by an exponential in fp32 does not hold the bound."""
    d, h, e, dtype = 64, 16, 2, torch.bfloat16
    x, q_in, q_out = whole(-2, 2, t, d), whole(0, 15, e, d, 2 * h, seed=1), whole(0, 15, e, h, d, seed=2)
    s_in = torch.ones(e, 1, 2 * h, device="cuda", dtype=torch.float64)
    s_in[..., :h] = 45 * 2.0 ** -28
    idx = whole(0, e - 1, t, 1, seed=3)
    pack = lambda q, s: Int4Weight.from_levels(q.to(torch.uint8), s.to(dtype), 64)  # noqa: E731
    out = int4_experts(x.to(dtype), torch.ones(t, 1, dtype=dtype, device="cuda"), idx, pack(q_in, s_in),
                       pack(q_out, torch.ones(e, 1, d, device="cuda")), "tanh").double()
    a = torch.einsum("td,tdh->th", x.double(), (q_in - 8).double()[idx[:, 0]]) * s_in[0]
    gate, up = a.chunk(2, 1)
    down = (q_out - 8).double()[idx[:, 0]]
    exact = torch.einsum("th,thd->td", torch.tanh(gate) * up, down)
    magnitude = torch.einsum("th,thd->td", (torch.tanh(gate) * up).abs(), down.abs())
    err = (4 * h * 2.0 ** -23 + 2.0 ** -15 + 2.0 ** -21) * magnitude
    f = torch.finfo(dtype)
    bound = f.eps / 2 * (exact.abs() + err) + err + f.smallest_normal * f.eps
    assert bool(((out - exact).abs() <= bound).all())
    one = 2 / (1 + torch.exp(-2 * gate.float())) - 1
    loose = torch.einsum("th,thd->td", one.double() * up, down)
    assert t < 40 or not bool(((loose.to(dtype).double() - exact).abs() <= bound).all())


def test_int4_experts_what_is_not_finite_stays_with_its_token():
    args, _, _ = whole_experts(40, 64, 128, 3, 64, torch.float16)
    want = int4_experts(*args, "relu")
    x = args[0].clone()
    x[7, 3], x[20, 60] = float("inf"), float("nan")
    out = int4_experts(x, *args[1:], "relu")
    keep = [i for i in range(40) if i not in (7, 20)]
    assert torch.equal(out[keep], want[keep])
    assert not torch.isfinite(out[7]).all() and torch.isnan(out[20]).any()


# --------------------------------------------------------------------------- grouped products, bit for bit
@pytest.mark.parametrize("k,n,rows,groups", [(64, 40, 40000, 14), (72, 264, 40000, 14), (264, 72, 40000, 14),
                                             (304, 520, 100000, 8), (64, 64, 3000, 3)])
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_grouped_whole_numbers_are_exact(k, n, rows, groups, dtype, layout, host):
    """Rows of -1, 0 and 1: every fp32 sum is exact in any order, so results are those of 64 bits, rounded once, bit
    for bit. Runs around one, two and three chunks of the weight gradient, around its 64-row stages and its 16-row
    steps; NaN behind the last run."""
    a, b = (k, n) if layout == "kn" else (n, k)       # (dw of a transposed weight is the product's transpose)
    tiles = -(-a // 256) * -(-b // (256 if b > 128 else 128))
    ks = host.chunk_rows(rows, groups, tiles, 74)
    counts = [ks - 1, ks, ks + 1, 2 * ks - 17, 2 * ks + 63, 3 * ks + 16, 2 * ks, 65, 64, 63, 0, 15, 17, 1]
    counts = counts[:groups] if groups > 3 else [ks + 1, 63, ks - 65]
    cut = [0]
    for c in counts:
        cut.append(cut[-1] + c)
    assert cut[-1] <= rows and max(counts) > ks
    x, w = whole(-1, 1, rows, k).to(dtype), whole(-1, 1, groups, k, n, seed=1).to(dtype)
    dy = whole(-1, 1, rows, n, seed=2).to(dtype)
    if layout == "nk":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    x[cut[-1]:], dy[cut[-1]:] = float("nan"), float("nan")
    x.requires_grad_(), w.requires_grad_()
    y = grouped_mm(x, w, torch.tensor(cut, dtype=torch.int32, device="cuda"))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    kernels.check_status("cuda")
    for g, (lo, hi) in enumerate(zip(cut, cut[1:])):
        xg, wg, dg = x.detach()[lo:hi].double(), w.detach()[g].double(), dy[lo:hi].double()
        assert torch.equal(y.detach()[lo:hi], (xg @ wg).to(dtype))
        assert torch.equal(dx[lo:hi], (dg @ wg.T).to(dtype))
        assert torch.equal(dw[g], (xg.T @ dg).to(dtype))
        if hi - lo > 1:      # a run that is a row short is seen
            assert not torch.equal(dw[g], (xg[:-1].T @ dg[:-1]).to(dtype))
    assert not y.detach()[cut[-1]:].any() and not dx[cut[-1]:].any()


# --------------------------------------------------------------------------- behind a reported input
def test_reported_inputs_stop_no_call():
    """A weight gradient of several ms in which one warp waits for the single ragged run end nearly throughout
    (longer than a wait looks away from the status word): the same bits behind a reported expert id or run start, and
    the report stays what it was."""
    runs, each, m, n = 16, 32768, 2048, 4096
    rows = runs * each - 31
    a = torch.randn(rows, m, device="cuda", dtype=torch.bfloat16)
    b = torch.randn(rows, n, device="cuda", dtype=torch.bfloat16)
    off = (torch.arange(runs + 1, device="cuda") * each).clamp(max=rows).int()
    kernels.check_status("cuda")
    want = kernels.grouped_wgrad(a, b, off)
    kernels.check_status("cuda")
    word = kernels.status_word("cuda")
    for code in (2, 3):
        word.fill_(code)
        assert torch.equal(kernels.grouped_wgrad(a, b, off), want)
        assert int(word) == code
        word.zero_()
    # starts that decrease, reported by the call itself: taken into range, and the rest is right
    bad = off.clone()
    bad[3] = bad[4] + 5
    good = bad.cummax(0).values
    got = kernels.grouped_wgrad(a, b, bad)
    with pytest.raises(RuntimeError, match="runs decrease or leave"):
        kernels.check_status("cuda")
    assert torch.equal(got, kernels.grouped_wgrad(a, b, good))
    kernels.check_status("cuda")


def test_a_report_is_not_replaced_by_a_later_one():
    args, _, _ = whole_experts(3, 64, 16, 2, 32, torch.bfloat16)
    x, w = torch.randn(8, 16, device="cuda").half(), torch.randn(2, 16, 16, device="cuda").half()
    args[2][1, 0] = 7
    int4_experts(*args, "relu")
    grouped_mm(x, w, torch.tensor([0, 9, 8], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="expert id"):
        kernels.check_status("cuda")
    kernels.check_status("cuda")


# --------------------------------------------------------------------------- refusals
def test_low_level_entries_refuse_operands_that_do_not_fit():
    from test_operators import low_level_calls
    for call, args in low_level_calls("cuda"):
        with pytest.raises((ValueError, RuntimeError), match="do not fit together"):
            call(*args)
    kernels.check_status("cuda")


@pytest.mark.parametrize("how", ["dual", "jvp"])
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(how, grad):
    """Whether or not an operand requires a gradient, through the eager calls and through the registered ops."""
    import torch.autograd.forward_ad as fwad
    from nanospeaker_b200 import MoEBlock, MoEFFNSublayer, dropout_add, int4_mm, quantize_int4
    half = lambda *s: torch.randn(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    w, off = half(2, 64, 24).requires_grad_(grad), torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    rng = torch.zeros(2, dtype=torch.int64, device="cuda")
    x, tw, idx = half(6, 64), half(6, 1), torch.zeros(6, 1, dtype=torch.int64, device="cuda")
    res = half(6, 64).requires_grad_(grad)
    one = quantize_int4(half(64, 8))
    w_in, w_out = quantize_int4(half(2, 64, 32)), quantize_int4(half(2, 16, 64))
    block = MoEBlock(576, 76, d_ff=192, top_k=6, n_shared=2, capacity_factor=None).to(torch.bfloat16).cuda()
    block.requires_grad_(grad)
    sub = MoEFFNSublayer(block).to(torch.bfloat16).cuda().requires_grad_(grad)
    calls = [(lambda v: grouped_mm(v, w, off), x), (lambda v: dropout_add(v, res, 0.1, rng), x),
             (lambda v: dropout_add(x, v, 0.1, rng), x)]
    if how == "dual":   # (the sublayer's traced form is an autograd.Function, which refuses in its own words)
        calls += [(block, half(5, 576)), (lambda v: sub(v)[0], half(5, 576))]
    if not grad:
        calls += [(lambda v: int4_mm(v, one), x), (lambda v: int4_experts(v, tw, idx, w_in, w_out), x),
                  (lambda v: int4_experts(x, v, idx, w_in, w_out), tw)]
    for call, at in calls:
        with pytest.raises(NotImplementedError, match="forward mode"):
            if how == "jvp":
                torch.func.jvp(call, (at,), (torch.ones_like(at),))
            else:
                with fwad.dual_level():
                    call(fwad.make_dual(at, torch.ones_like(at)))
