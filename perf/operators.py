"""The operators beside the block's fused kernels, as timed cases: one pass each through the public
entry points, over the range of sizes, types and directions that a user calls them with.

Kinds of a case:
  grouped       grouped_mm(x, w, offsets): every run of rows times its expert's matrix, ragged runs
                back to back; "train" also takes both gradients
  int4_mm       int4_mm(x, weight): few rows against one matrix held in 4 bits with group scales
  int4_experts  int4_experts(x, topk_w, topk_idx, w_in, w_out, ...): the block's routed and shared GLU
                experts with weights in 4 bits, for a batch of tokens that generates
  dropout       dropout_add(x, residual, p, rng): residual + dropout(x) and the gradient of x, the
                mask from a counter-based generator and never stored

Sizes: the model's block (d_model 576, 76 routed + 2 shared experts of hidden width 128, top-6) with
the token counts of the benchmark configurations (64, 2048, 16384, 65536), the wide block of the
package's other timed cases, generic powers of two, and ragged ones in between.

A plain form computes in fp32 and rounds once. Random bits are whole-number arithmetic (Philox4x32-10,
Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011), the state (seed, call) an input.
"""
import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _grouped(rows, k, n, groups, skew=0.0, train=False, dtype="bf16", layout="kn"):
    """skew: spread of the per-group logits that the rows are drawn by (0: even, 0.27: loads with
    CV ~ 1 under top-6 routing, 1.5: many groups nearly or quite empty). layout: w's innermost axis,
    n (the block's weights) or k (a transposed view, as a checkpoint of nn.Linear weights is)."""
    return dict(kind="grouped", rows=rows, k=k, n=n, groups=groups, skew=skew, train=train,
                dtype=dtype, layout=layout)


def _int4_mm(rows, k, n, group, dtype="bf16"):
    return dict(kind="int4_mm", rows=rows, k=k, n=n, group=group, dtype=dtype)


def _int4_experts(tokens, d=576, h=128, experts=76, top_k=6, shared=2, group=64, dtype="bf16",
                  activation="silu"):
    return dict(kind="int4_experts", tokens=tokens, d=d, h=h, experts=experts, top_k=top_k,
                shared=shared, group=group, dtype=dtype, activation=activation)


def _dropout(rows, d, p, dtype="bf16", residual=True):
    return dict(kind="dropout", rows=rows, d=d, p=p, dtype=dtype, residual=residual)


def listed():
    return [
        # the up projection of 64 generating sequences: five rows an expert, weights are what is read
        dict(name="grouped 384 rows", **_grouped(384, 576, 256, 76)),
        # the up projection of the benchmark's training step: 16384 tokens, six experts each
        dict(name="grouped train 98304 rows", **_grouped(98304, 576, 256, 76, 0.27, True)),
        # the wide block with hidden width 512: a ragged batch of 3001 tokens, top-4, half of the
        # experts idle, fp16, weights that lie transposed
        dict(name="grouped train 12004 rows, fp16", **_grouped(12004, 768, 1024, 64, 1.5, True,
                                                               "fp16", "nk")),
        # few large experts on a large batch: products that fill the tensor cores
        dict(name="grouped train 32768 rows, large", **_grouped(32768, 2048, 4096, 16, 0.27, True)),
        # one token through one large matrix: nothing but the weights' bytes
        dict(name="int4_mm 1 row", **_int4_mm(1, 4096, 16384, 128)),
        # a small odd matrix, a few sequences, fine scales
        dict(name="int4_mm 7 rows, odd", **_int4_mm(7, 1000, 1537, 32, "fp16")),
        # a serving batch of 64 sequences
        dict(name="int4_mm 64 rows", **_int4_mm(64, 4096, 4096, 64)),
        # one sequence being generated through the model's experts: latency
        dict(name="int4_experts 1 token", **_int4_experts(1)),
        # a serving batch of 64 sequences: every expert has a few rows
        dict(name="int4_experts 64 tokens", **_int4_experts(64)),
        # a wider block, a larger batch, gelu gates, fp16
        dict(name="int4_experts 200 tokens, wide", **_int4_experts(200, 1024, 768, 32, 4, 1, 128,
                                                                   "fp16", "gelu")),
        # one sequence per micro-batch
        dict(name="dropout 2048 rows", **_dropout(2048, 576, 0.1)),
        # 65536 tokens on a GPU: the largest training batch
        dict(name="dropout 65536 rows", **_dropout(65536, 576, 0.1)),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over the logarithm."""
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["grouped", "grouped", "grouped", "int4_mm", "int4_mm", "int4_experts",
                       "int4_experts", "dropout"])
    half = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "grouped":
        return _grouped(_log(rng, 1, 32768), 8 * _log(rng, 4, 256), 8 * _log(rng, 4, 512),
                        _log(rng, 1, 128) if rng.random() < 0.5 else rng.choice([8, 16, 64, 76]),
                        rng.choice([0.0, 0.27, 1.5]), rng.random() < 0.6, half,
                        rng.choice(["kn", "kn", "nk"]))
    if kind == "int4_mm":
        return _int4_mm(_log(rng, 1, 64), 8 * _log(rng, 8, 1024), _log(rng, 64, 16384),
                        rng.choice([32, 64, 128]), half)
    if kind == "int4_experts":
        experts = rng.choice([8, 16, 32, 64, 76, 128])
        return _int4_experts(_log(rng, 1, 256), 64 * _log(rng, 4, 24), 16 * _log(rng, 4, 64), experts,
                             rng.choice([1, 2, 4, 6, 8]), rng.choice([0, 1, 2]),
                             rng.choice([32, 64, 128]), half, rng.choice(["silu", "silu", "gelu"]))
    return _dropout(_log(rng, 16, 32768), rng.choice([_log(rng, 64, 1024), 8 * _log(rng, 8, 128)]),
                    rng.choice([0.05, 0.1, 0.25, 0.5]), rng.choice(["bf16", "fp16", "fp32"]),
                    rng.random() < 0.7)


# ------------------------------------------------------------------------------------- prepare
def _levels(gen, shape, group, dtype):
    """A matrix of standard deviation k^-1/2 as 4-bit levels (0..15, value level - 8) and the scales
    of its groups of `group` inputs: what rounding a normal matrix to 4 bits leaves."""
    k, n = shape[-2:]
    q = (torch.randn(shape, generator=gen, device=DEV) * 2.8).round_().clamp_(-8, 7).add_(8)
    s = torch.rand((*shape[:-2], -(-k // group), n), generator=gen, device=DEV)
    return q.to(torch.uint8), ((0.9 + 0.2 * s) * (k ** -0.5 / 2.8)).to(dtype)


def _held(q, s, group):
    """The weight a user's program keeps: laid out once where the framework's kernels read it."""
    if own:
        from nanospeaker_b200 import Int4Weight
        return Int4Weight.from_levels(q, s, group)
    return q, s


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEV)  # noqa: E731
    state = dict(case)
    if case["kind"] == "grouped":
        r, k, n, g = case["rows"], case["k"], case["n"], case["groups"]
        load = torch.softmax(normal(g) * case["skew"], 0)
        of = torch.multinomial(load, r, replacement=True, generator=gen)
        counts = torch.bincount(of, minlength=g)
        state["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
        state["longest"] = int(counts.max())
        state["x"] = normal(r, k).to(dtype).requires_grad_(case["train"])
        w = (normal(g, k, n) * k ** -0.5).to(dtype)
        if case["layout"] == "nk":
            w = w.transpose(1, 2).contiguous().transpose(1, 2)
        state["w"] = w.requires_grad_(case["train"])
        state["dy"] = normal(r, n).to(dtype)
    elif case["kind"] == "int4_mm":
        state["x"] = normal(case["rows"], case["k"]).to(dtype)
        state["weight"] = _held(*_levels(gen, (case["k"], case["n"]), case["group"], dtype),
                                case["group"])
    elif case["kind"] == "int4_experts":
        t, d, h, e = case["tokens"], case["d"], case["h"], case["experts"]
        state["x"] = normal(t, d).to(dtype)
        logits, idx = normal(t, e).topk(case["top_k"], dim=1)
        state["topk_w"], state["topk_idx"] = torch.softmax(logits, 1).to(dtype), idx
        state["longest"] = int(torch.bincount(idx.reshape(-1)).max())
        for name, shape in (("w_in", (e, d, 2 * h)), ("w_out", (e, h, d)),
                            ("shared_in", (case["shared"], d, 2 * h)),
                            ("shared_out", (case["shared"], h, d))):
            state[name] = (_held(*_levels(gen, shape, case["group"], dtype), case["group"])
                           if shape[0] else None)
    else:
        shape = (case["rows"], case["d"])
        state["x"] = normal(*shape).to(dtype).requires_grad_()
        state["residual"] = normal(*shape).to(dtype) if case["residual"] else None
        state["dout"] = normal(*shape).to(dtype)
        state["rng"] = torch.randint(0, 1 << 40, (2,), generator=gen, device=DEV)
    return state


# ------------------------------------------------------------------------------ the plain forms
def _in_runs(offsets, rows):
    """(group, place within its run) of every row."""
    at = torch.arange(rows, device=offsets.device)
    group = torch.searchsorted(offsets[1:].contiguous(), at.to(offsets.dtype), right=True)
    return group, at - offsets.long()[group]


def _plain_grouped(s):
    group, place = _in_runs(s["offsets"], s["rows"])
    spread = lambda t: t.new_zeros(s["groups"], s["longest"], t.shape[1],  # noqa: E731
                                   dtype=torch.float32).index_put_((group, place), t.float())
    with torch.no_grad():
        x, w = spread(s["x"]), s["w"].float()
        y = torch.bmm(x, w)[group, place].to(s["x"].dtype)
        if not s["train"]:
            return {"y": y}
        dy = spread(s["dy"])
        dx = torch.bmm(dy, w.transpose(1, 2))[group, place].to(y.dtype)
        return {"y": y, "dx": dx, "dw": torch.bmm(x.transpose(1, 2), dy).to(y.dtype)}


def _plain_weight(weight, group):
    q, s = weight
    return (q.float() - 8) * s.float().repeat_interleave(group, -2)[..., :q.shape[-2], :]


def _plain_act(name, g):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.erf(g * 0.5 ** 0.5))


def _plain_mlp(s, x, w_in, w_out):
    gate, up = torch.matmul(x, _plain_weight(w_in, s["group"])).chunk(2, dim=-1)
    return torch.matmul(_plain_act(s["activation"], gate) * up, _plain_weight(w_out, s["group"]))


def _plain_experts(s):
    x, k, e = s["x"].float(), s["top_k"], s["experts"]
    flat = s["topk_idx"].reshape(-1)
    order = torch.argsort(flat, stable=True)
    counts = torch.zeros(e + 1, dtype=torch.int32, device=DEV).index_add_(
        0, flat + 1, torch.ones_like(flat, dtype=torch.int32))
    group, place = _in_runs(counts.cumsum(0).to(torch.int32), flat.numel())
    runs = x.new_zeros(e, s["longest"], s["d"]).index_put_((group, place), x[order // k])
    y = _plain_mlp(s, runs, s["w_in"], s["w_out"])[group, place]
    pairs = torch.empty_like(y).index_copy_(0, order, y).view(-1, k, s["d"])
    out = (pairs * s["topk_w"].float()[:, :, None]).sum(1)
    if s["shared"]:
        out = out + _plain_mlp(s, x.expand(s["shared"], -1, -1), s["shared_in"],
                               s["shared_out"]).sum(0)
    return out.to(s["x"].dtype)


def _plain_bits(n, rng):
    """n random words of 32 bits: word i is word i % 4 of Philox4x32-10 at counter (i / 4, call) under
    the key seed, in int64 (products by halves, as 64 bits would not hold them)."""
    low = 0xFFFFFFFF
    quad = torch.arange((n + 3) // 4, device=rng.device)
    zero = torch.zeros_like(quad)
    c = [quad & low, quad >> 32, zero + (rng[1] & low), zero + ((rng[1] >> 32) & low)]
    key = [rng[0] & low, (rng[0] >> 32) & low]

    def product(a, m):
        high = (m * (a >> 16) + ((m * (a & 0xFFFF)) >> 16)) >> 16
        return high, (m * a) & low

    for _ in range(10):
        h0, l0 = product(c[0], 0xD2511F53)
        h1, l1 = product(c[2], 0xCD9E8D57)
        c = [h1 ^ c[1] ^ key[0], l1, h0 ^ c[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) & low, (key[1] + 0xBB67AE85) & low]
    return torch.stack(c, 1).reshape(-1)[:n]


def _threshold(p):
    """An element whose random word is below this is dropped."""
    return min(round(p * 2.0 ** 32), 2 ** 32 - 1)


def _plain_dropout(s):
    with torch.no_grad():
        x = s["x"]
        keep = (_plain_bits(x.numel(), s["rng"]) >= _threshold(s["p"])).view(x.shape)
        scale = 1 / (1 - s["p"])
        out = torch.where(keep, x.float() * scale, 0.0)
        if s["residual"] is not None:
            out = out + s["residual"].float()
        dx = torch.where(keep, s["dout"].float() * scale, 0.0)
        return {"out": out.to(x.dtype), "dx": dx.to(x.dtype)}


def _run_plain(s):
    if s["kind"] == "grouped":
        return _plain_grouped(s)
    if s["kind"] == "int4_mm":
        return torch.matmul(s["x"].float(), _plain_weight(s["weight"], s["group"])).to(s["x"].dtype)
    return _plain_experts(s) if s["kind"] == "int4_experts" else _plain_dropout(s)


# -------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    import nanospeaker_b200 as nb
    if s["kind"] == "grouped":
        y = nb.grouped_mm(s["x"], s["w"], s["offsets"])
        if not s["train"]:
            return {"y": y}
        dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if s["kind"] == "int4_mm":
        return nb.int4_mm(s["x"], s["weight"])
    if s["kind"] == "int4_experts":
        return nb.int4_experts(s["x"], s["topk_w"], s["topk_idx"], s["w_in"], s["w_out"],
                               activation=s["activation"], shared_in=s["shared_in"],
                               shared_out=s["shared_out"])
    out = nb.dropout_add(s["x"], s["residual"], s["p"], s["rng"])
    dx, = torch.autograd.grad(out, s["x"], s["dout"])
    return {"out": out.detach(), "dx": dx}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------- work
def _touched(case):
    """How many routed experts a batch is expected to reach."""
    e = case["experts"]
    return e * (1 - (1 - min(case["top_k"], e) / e) ** case["tokens"])


def work(case):
    b = TYPES[case["dtype"]].itemsize
    if case["kind"] == "grouped":
        r, k, n, g = case["rows"], case["k"], case["n"], case["groups"]
        part = (r * k + r * n) * b
        weights = min(g, r) * k * n * b
        if not case["train"]:
            return {"bytes": part + weights, "flops": 2 * r * k * n}
        return {"bytes": 2 * part + weights + g * k * n * b, "flops": 6 * r * k * n}
    if case["kind"] == "int4_mm":
        r, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": n * k / 2 + n * -(-k // case["group"]) * b + r * (k + n) * b,
                "flops": 2 * r * k * n}
    if case["kind"] == "int4_experts":
        t, d, h, k = case["tokens"], case["d"], case["h"], case["top_k"]
        each = 3 * d * h / 2 + (2 * h * -(-d // case["group"]) + d * -(-h // case["group"])) * b
        return {"bytes": (_touched(case) + case["shared"]) * each + 2 * t * d * b + t * k * (8 + b),
                "flops": 6 * t * (k + case["shared"]) * d * h}
    size = case["rows"] * case["d"]
    return {"bytes": size * b * (4 + case["residual"]), "flops": 0}


# --------------------------------------------------------------------------------------- exact
def _exact_weight(weight, group):
    """Input row i of the matrix under the scale of its group i // group."""
    q, s = weight
    return (q.double() - 8) * s.double()[torch.arange(q.shape[0], device=q.device) // group]


def _exact_mlp(case, x, w_in, w_out):
    a = x @ _exact_weight(w_in, case["group"])
    gate, up = a[:, :case["h"]], a[:, case["h"]:]
    gate = (gate * torch.sigmoid(gate) if case["activation"] == "silu"
            else gate * torch.special.ndtr(gate))
    return (gate * up) @ _exact_weight(w_out, case["group"])


def _exact_kept(n, rng, p):
    """The mask of dropout, by unsigned 64-bit arithmetic on the host."""
    seed, call = (int(v) for v in rng.cpu())
    m0, m1, low, half = np.uint64(0xD2511F53), np.uint64(0xCD9E8D57), np.uint64(0xFFFFFFFF), np.uint64(32)
    quad = np.arange((n + 3) // 4, dtype=np.uint64)
    x0, x1 = quad & low, quad >> half
    x2 = np.full_like(quad, call & 0xFFFFFFFF)
    x3 = np.full_like(quad, (call >> 32) & 0xFFFFFFFF)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        p0, p1 = x0 * m0, x2 * m1
        x0, x1, x2, x3 = (p1 >> half) ^ x1 ^ np.uint64(k0), p1 & low, (p0 >> half) ^ x3 ^ np.uint64(k1), p0 & low
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    words = np.stack([x0, x1, x2, x3], axis=1).reshape(-1)[:n]
    return torch.from_numpy(words >= np.uint64(_threshold(p)))


def exact(case, seed):
    global own
    before, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = before
    with torch.no_grad():
        if case["kind"] == "grouped":
            r, k, n = case["rows"], case["k"], case["n"]
            cut = s["offsets"].tolist()
            y = torch.empty(r, n, dtype=torch.float64, device=DEV)
            dx = torch.empty(r, k, dtype=torch.float64, device=DEV)
            dw = torch.empty(case["groups"], k, n, dtype=torch.float64, device=DEV)
            for g, (a, b) in enumerate(zip(cut, cut[1:])):
                x, dy, w = s["x"][a:b].double(), s["dy"][a:b].double(), s["w"][g].double()
                y[a:b] = x @ w
                if case["train"]:
                    dx[a:b] = dy @ w.T
                    dw[g] = x.T @ dy
            return {"y": y, "dx": dx, "dw": dw} if case["train"] else {"y": y}
        if case["kind"] == "int4_mm":
            return s["x"].double() @ _exact_weight(s["weight"], case["group"])
        if case["kind"] == "int4_experts":
            x = s["x"].double()
            out = torch.zeros_like(x)
            for e in range(case["experts"]):
                token, slot = (s["topk_idx"] == e).nonzero(as_tuple=True)
                if token.numel():
                    y = _exact_mlp(case, x[token], [v[e] for v in s["w_in"]],
                                   [v[e] for v in s["w_out"]])
                    out[token] += y * s["topk_w"].double()[token, slot, None]
            for e in range(case["shared"]):
                out += _exact_mlp(case, x, [v[e] for v in s["shared_in"]],
                                  [v[e] for v in s["shared_out"]])
            return out
        x = s["x"].double()
        kept = _exact_kept(x.numel(), s["rng"], case["p"]).to(DEV).view(x.shape)
        out = torch.where(kept, x / (1 - case["p"]), 0.0)
        if s["residual"] is not None:
            out = out + s["residual"].double()
        return {"out": out, "dx": torch.where(kept, s["dout"].double() / (1 - case["p"]), 0.0)}
