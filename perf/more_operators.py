"""A gated feed-forward block and the log probabilities of a vocabulary, timed: the product of both projections with its gradients, from
pre-activations that are kept whole or in 8 bits, and what a loss, a sampler or a scorer asks of a row of logits, with its gradient.

`own` False runs their plain forms, elementary torch operations in 32 bits; True makes the calls of `ml.matmul` and `ml.primitives`.
`listed()` holds the fixed cases, `draw(rng)` makes further ones of the same ranges.
"""
import math
import os
import sys

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
BLOCK = 128
TINY = 2.0 ** -126


def _ml():
    pkg = os.path.join(os.getcwd(), "spiral-s-ml-library_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from ml import matmul, primitives
    return matmul, primitives


def listed():
    return [
        # one token through the block: the read of both weights is all there is
        dict(name="gated_one_token", kind="gated", dtype="bf16", activation="silu", rows=1, inner=4096, cols=8192),
        # an odd number of sequences being decoded, widths that are no multiple of anything but 8
        dict(name="gated_few_rows", kind="gated", dtype="f16", activation="gelu", rows=49, inner=1000, cols=2667),
        # a prompt: the matrix pipes
        dict(name="gated_prompt", kind="gated", dtype="bf16", activation="silu", rows=8192, inner=4096, cols=8192),
        # a training step, forward and backward, pre-activations kept as they are
        dict(name="gated_training", kind="gated_training", dtype="bf16", activation="silu", keep="full", rows=8192, inner=2048, cols=8192),
        # the same with the pre-activations kept in 8 bits, of odd sizes (two thirds of four times the inner width)
        dict(name="gated_training_8bit", kind="gated_training", dtype="bf16", activation="silu", keep="8bit", rows=5008, inner=2048, cols=5461),
        # a small model in f32
        dict(name="gated_training_f32", kind="gated_training", dtype="f32", activation="gelu", keep="full", rows=1003, inner=512, cols=1365),
        # a short batch of a small model
        dict(name="gated_training_short", kind="gated_training", dtype="f16", activation="relu", keep="8bit", rows=256, inner=512, cols=1024),
        # one row of logits whose token has been chosen, with the alternatives to it
        dict(name="tokens_one_row", kind="tokens", dtype="f32", rows=1, cols=32003, top=20, entropy=True, masked=True),
        # a serving batch over a large vocabulary
        dict(name="tokens_batch", kind="tokens", dtype="bf16", rows=256, cols=131072, top=5, entropy=True, masked=False),
        # a text being scored: nothing but the log probabilities
        dict(name="tokens_scoring", kind="tokens", dtype="f16", rows=5001, cols=1003, top=0, entropy=False, masked=False),
        # the loss of a training step and its gradient
        dict(name="tokens_training", kind="tokens_training", dtype="bf16", rows=4096, cols=32003, entropy=False),
        # a policy's gradient with an entropy bonus: many short rows
        dict(name="tokens_policy", kind="tokens_training", dtype="f32", rows=65536, cols=256, entropy=True),
    ]


# ---- drawn cases ---------------------------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    n = _log(rng, lo, hi)
    return max(128, n // 128 * 128) if rng.random() < 0.4 else n


def _draw_gated(rng):
    while True:
        rows = rng.choice([_log(rng, 1, 64), _log(rng, 1, 8192)])
        inner, cols = max(8, _width(rng, 64, 8192) // 8 * 8), _width(rng, 64, 16384)
        if inner * cols <= 1 << 26 and 4.0 * rows * inner * cols <= 1.0e12:
            break
    return dict(kind="gated", dtype=rng.choice(["bf16", "bf16", "f16", "f32"]) if rows <= 1024 else rng.choice(["bf16", "f16"]),
                activation=rng.choice(["silu", "silu", "gelu", "relu"]), rows=rows, inner=inner, cols=cols)


def _draw_gated_training(rng):
    while True:
        rows, inner, cols = _log(rng, 64, 16384), max(64, _width(rng, 128, 4096) // 8 * 8), _width(rng, 128, 16384)
        if 12.0 * rows * inner * cols <= 1.6e12:
            break
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"]) if 12.0 * rows * inner * cols <= 1e11 else rng.choice(["bf16", "f16"])
    # (in f32 a relu's slope at sums next to zero is the order of the sums, not the numbers)
    return dict(kind="gated_training", dtype=dtype, activation=rng.choice(["silu", "silu", "gelu"] if dtype == "f32" else ["silu", "silu", "gelu", "relu"]),
                keep="full" if dtype == "f32" else rng.choice(["full", "8bit"]), rows=rows, inner=inner, cols=cols)


def _draw_tokens(rng):
    while True:
        rows, cols = rng.choice([_log(rng, 1, 16), _log(rng, 1, 16384)]), _log(rng, 64, 262144)
        if rows * cols <= 1 << 25:
            break
    return dict(kind="tokens", dtype=rng.choice(["f32", "bf16", "f16"]), rows=rows, cols=cols, top=rng.choice([0, 0, 1, 5, 20, 32]),
                entropy=rng.random() < 0.5, masked=rng.random() < 0.4)


def _draw_tokens_training(rng):
    while True:
        rows, cols = _log(rng, 16, 131072), _log(rng, 8, 262144)
        if rows * cols <= 1 << 27:
            break
    return dict(kind="tokens_training", dtype=rng.choice(["f32", "bf16", "f16"]), rows=rows, cols=cols, entropy=rng.random() < 0.5)


def draw(rng):
    return rng.choice([_draw_gated, _draw_gated, _draw_gated_training, _draw_gated_training, _draw_tokens, _draw_tokens_training])(rng)


# ---- inputs --------------------------------------------------------------------------------------------------------

def _prepare_gated(case, gen):
    rows, inner, cols, t = case["rows"], case["inner"], case["cols"], DTYPE[case["dtype"]]
    # what a norm hands on, some of its columns larger than the others, and weights that leave the variance alone
    x = torch.randn((rows, inner), generator=gen, device="cuda").mul_(torch.exp(torch.randn((inner,), generator=gen, device="cuda") * 0.3))
    weight = lambda: torch.randn((cols, inner), generator=gen, device="cuda").div_(math.sqrt(inner)).to(t)
    s = {"x": x.to(t), "gate": weight(), "up": weight()}
    if case["kind"] == "gated_training":
        s["dy"] = torch.randn((rows, cols), generator=gen, device="cuda").to(t)
    return s


def _prepare_tokens(case, gen):
    rows, cols = case["rows"], case["cols"]
    u = lambda *shape: torch.rand(shape, generator=gen, device="cuda")
    # a few likely tokens above a broad rest; the text's token is mostly one of the likely ones
    x = torch.randn((rows, cols), generator=gen, device="cuda").mul_(2)
    likely = (u(rows, 8) * cols).long().clamp_(max=cols - 1)
    x.scatter_add_(1, likely, u(rows, 8) * 8)
    tokens = torch.where(u(rows) < 0.8, likely[:, 0], (u(rows) * cols).long().clamp_(max=cols - 1)).int()
    if rows > 2:
        tokens[2::17] = -1                                              # places that do not count
    if case.get("masked"):
        x.masked_fill_(u(rows, cols) < 0.7, -math.inf)
        if rows > 2:
            x[1] = -math.inf                                            # a grammar that has come to its end
    s = {"x": x.to(DTYPE[case["dtype"]]), "tokens": tokens}
    if case["kind"] == "tokens_training":
        s["d_logp"] = torch.randn((rows,), generator=gen, device="cuda")
        s["d_entropy"] = torch.randn((rows,), generator=gen, device="cuda") * 0.1 if case["entropy"] else None
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = (_prepare_gated if case["kind"].startswith("gated") else _prepare_tokens)(case, gen)
    s["case"] = case
    s["most"] = torch.tensor(F8_MAX, device="cuda")
    return s


# ---- one pass, plain -----------------------------------------------------------------------------------------------

def _plain_activation(g, name):
    """act(g) and its derivative."""
    if name == "relu":
        return g.clamp(min=0), (g > 0).to(g.dtype)
    if name == "gelu":
        below = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * below, below + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-g))
    return g * s, s * (1 + g * (1 - s))


def _plain_blocks(x, most):
    """(codes, scales) of x's rows in blocks of 128, the codes zero up to a multiple of 16 columns."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    full = torch.zeros((rows, blocks * BLOCK), device=x.device)
    full[:, :cols] = x
    tiles = full.view(rows, blocks, BLOCK)
    scale = (tiles.abs().amax(2) / most).clamp(min=TINY)
    q = (tiles / scale[:, :, None]).to(F8).view(rows, blocks * BLOCK)
    return q[:, :-(-cols // 16) * 16].contiguous(), scale


def _values(q, scale, cols):
    return q[:, :cols].float() * scale.repeat_interleave(BLOCK, 1)[:, :cols]


def _plain_gated(s):
    case = s["case"]
    t = DTYPE[case["dtype"]]
    x, wg, wu = s["x"].float(), s["gate"].float(), s["up"].float()
    g, u = torch.mm(x, wg.t()), torch.mm(x, wu.t())
    y = (_plain_activation(g, case["activation"])[0] * u).to(t)
    if case["kind"] == "gated":
        return y
    if case["keep"] == "full":
        kept = (g.to(t), u.to(t))
        g, u = kept[0].float(), kept[1].float()
    else:
        kept = _plain_blocks(g, s["most"]) + _plain_blocks(u, s["most"])
        g, u = _values(kept[0], kept[1], case["cols"]), _values(kept[2], kept[3], case["cols"])
    dy = s["dy"].float()
    act, slope = _plain_activation(g, case["activation"])
    dg, du = dy * u * slope, dy * act
    return y, kept, (torch.mm(dg, wg) + torch.mm(du, wu)).to(t), torch.mm(dg.t(), x).to(t), torch.mm(du.t(), x).to(t)


def _plain_tokens(s):
    case, x, tokens = s["case"], s["x"].float(), s["tokens"].long()
    rows, cols = x.shape
    most = x.amax(1, keepdim=True)
    none = most == -math.inf
    centred = x - torch.where(none, 0.0, most)
    e = torch.exp(centred)
    total = e.sum(1, keepdim=True)
    lse = most + torch.log(total)                                       # (-inf where there is nothing)
    counts = (tokens >= 0) & (tokens < cols)
    at = x.gather(1, tokens.clamp(0, cols - 1)[:, None])
    logp = torch.where(none, -math.inf, at - lse)[:, 0]
    out = [torch.where(counts, logp, 0.0)]
    training = case["kind"] == "tokens_training"
    if case["entropy"]:
        p = e / torch.where(none, 1.0, total)
        out.append((torch.log(torch.where(none, 1.0, total)) - (p * torch.where(p > 0, centred, 0.0)).sum(1, keepdim=True))[:, 0])
    if training:
        out.append(lse[:, 0])
        p = torch.exp(x - lse)
        dx = -p * s["d_logp"][:, None] * counts[:, None]
        if case["entropy"]:
            dx = dx - s["d_entropy"][:, None] * p * (torch.where(p > 0, x - lse, 0.0) + out[1][:, None])
        dx = dx.scatter_add(1, tokens.clamp(0, cols - 1)[:, None], (s["d_logp"] * counts)[:, None])
        out.append(torch.where(none, 0.0, dx).to(s["x"].dtype))
    elif case["top"]:
        k = min(case["top"], cols)
        v, j = torch.sort(x, dim=1, descending=True, stable=True)
        v, j = v[:, :k], j[:, :k]
        out += [torch.where(v > -math.inf, v - lse, -math.inf), torch.where(v > -math.inf, j, -1).int()]
    return tuple(out)


# ---- one pass, the framework's -------------------------------------------------------------------------------------

def _own_gated(s):
    case, (matmul, _) = s["case"], _ml()
    if case["kind"] == "gated":
        return matmul.matmul_abt_gated(s["x"], s["gate"], s["up"], activation=case["activation"])
    y, kept = matmul.matmul_abt_gated(s["x"], s["gate"], s["up"], activation=case["activation"], keep=s["x"].dtype if case["keep"] == "full" else F8)
    return (y, kept) + tuple(matmul.matmul_abt_gated_backward(s["dy"], s["x"], s["gate"], s["up"], kept, activation=case["activation"]))


def _own_tokens(s):
    case, (_, primitives) = s["case"], _ml()
    if case["kind"] == "tokens":
        out = primitives.token_log_probs(s["x"], s["tokens"], top=min(case["top"], case["cols"]), want_entropy=case["entropy"])
        return out if isinstance(out, tuple) else (out,)
    out = primitives.token_log_probs(s["x"], s["tokens"], want_entropy=case["entropy"], want_lse=True)
    return tuple(out) + (primitives.token_log_probs_backward(s["d_logp"], s["x"], s["tokens"], out[-1], d_entropy=s["d_entropy"],
                                                             entropy=out[1] if case["entropy"] else None),)


def run(state):
    gated = state["case"]["kind"].startswith("gated")
    if own:
        return _own_gated(state) if gated else _own_tokens(state)
    return _plain_gated(state) if gated else _plain_tokens(state)


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------

def _nearest_e4m3(v):
    """v (f64) to the nearest e4m3 number, ties to the even one; |v| within the type's range."""
    step = torch.exp2(torch.frexp(v).exponent.sub(1).clamp(min=-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-F8_MAX, F8_MAX)


def _exact_blocks(x):
    """A block's scale is a f32, and so is the quotient that is rounded to 8 bits."""
    cols = x.shape[1]
    amax = torch.nn.functional.pad(x.abs(), (0, -cols % BLOCK)).unflatten(1, (-1, BLOCK)).amax(2)
    scale = (amax / F8_MAX).float().clamp(min=TINY)
    each = scale.double().repeat_interleave(BLOCK, 1)[:, :cols]
    q = _nearest_e4m3((x / each).float().double())
    return torch.nn.functional.pad(q, (0, -cols % 16)), scale.double(), q * each


def _exact_activation(g, name):
    if name == "relu":
        return torch.relu(g), torch.heaviside(g, torch.zeros((), dtype=g.dtype, device=g.device))
    if name == "gelu":
        below = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
        return g * below, below + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return g * s, s + g * s * torch.sigmoid(-g)


def _exact_gated(case, s):
    t = DTYPE[case["dtype"]]
    x, wg, wu = s["x"].double(), s["gate"].double(), s["up"].double()
    g, u = x @ wg.t(), x @ wu.t()
    y = _exact_activation(g, case["activation"])[0] * u
    if case["kind"] == "gated":
        return y
    if case["keep"] == "full":                           # the gradients are those at the numbers that were kept
        kept, g, u = (g, u), g.to(t).double(), u.to(t).double()
    else:
        (qg, sg, g), (qu, su, u) = _exact_blocks(g), _exact_blocks(u)
        kept = (qg, sg, qu, su)
    act, slope = _exact_activation(g, case["activation"])
    dy = s["dy"].double()
    dg, du = dy * u * slope, dy * act
    return y, kept, torch.cat((dg, du), 1) @ torch.cat((wg, wu), 0), dg.t() @ x, du.t() @ x


def _exact_tokens(case, s):
    rows, cols = s["x"].shape
    logp = torch.empty((rows,), device="cuda", dtype=torch.float64)
    lse, entropy = torch.empty_like(logp), torch.empty_like(logp)
    training, k = case["kind"] == "tokens_training", min(case.get("top", 0), cols)
    top = torch.empty((rows, k), device="cuda", dtype=torch.float64)
    dx = torch.empty((rows, cols), device="cuda", dtype=torch.float64) if training else None
    step = max(1, (1 << 24) // cols)
    for r in range(0, rows, step):                        # some rows at a time
        x, tokens = s["x"][r:r + step].double(), s["tokens"][r:r + step].long()
        l = torch.logsumexp(x, 1)
        something = l > -math.inf
        logs = torch.where(something[:, None], x - l[:, None], -math.inf)
        p = torch.exp(logs)
        h = -torch.xlogy(p, p).sum(1)
        counted = (tokens >= 0) & (tokens < cols)
        mine = torch.arange(cols, device="cuda")[None] == tokens[:, None]
        logp[r:r + step] = torch.where(counted, torch.where(mine, logs, -math.inf).amax(1), 0.0)
        lse[r:r + step], entropy[r:r + step] = l, h
        if k:
            top[r:r + step] = torch.topk(logs, k, 1).values
        if training:
            d = s["d_logp"][r:r + step, None].double() * (mine.double() - p * counted[:, None])
            if case["entropy"]:
                d -= s["d_entropy"][r:r + step, None].double() * (torch.xlogy(p, p) + p * h[:, None])
            dx[r:r + step] = torch.where(something[:, None], d, 0.0)
    out = [logp] + ([entropy] if case["entropy"] else [])
    return tuple(out + ([lse, dx] if training else [top, None] if k else []))


def exact(case, seed):
    return (_exact_gated if case["kind"].startswith("gated") else _exact_tokens)(case, prepare(case, seed))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------

def work(case):
    e, rows, cols = SIZE[case["dtype"]], case["rows"], case["cols"]
    if case["kind"].startswith("gated"):
        inner = case["inner"]
        weights, x, y = 2 * e * inner * cols, e * rows * inner, e * rows * cols
        if case["kind"] == "gated":
            return {"bytes": weights + x + y, "flops": 4.0 * rows * inner * cols}
        kept = 2 * y if case["keep"] == "full" else 2 * rows * (-(-cols // 16) * 16 + 4 * -(-cols // BLOCK))
        # forward: x and the weights, y and what is kept; backward: dy and what was kept, x and the weights, three gradients
        return {"bytes": 3 * weights + 3 * x + 2 * y + 2 * kept, "flops": 12.0 * rows * inner * cols}
    if case["kind"] == "tokens":
        return {"bytes": e * rows * cols + 4 * rows * (2 + case["entropy"] + 2 * min(case["top"], cols)), "flops": (4.0 + 2 * case["entropy"]) * rows * cols}
    # the forward pass reads the logits, the backward pass reads them again and writes as many
    return {"bytes": 3 * e * rows * cols + 4 * rows * (7 + 3 * case["entropy"]), "flops": (8.0 + 6 * case["entropy"]) * rows * cols}
