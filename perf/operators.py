"""The operators of language-model training that sit beside this framework's optimizers, layers and losses, as a user
calls them, with a plain form of each for comparison.

* orthogonalisation of a matrix by Newton-Schulz products, alone and inside the Muon optimizer;
* the gated feed-forward block, forward and backward;
* log probabilities of given tokens with entropy and the top alternatives, forward and backward.

``own`` selects what :func:`run` does: ``False`` the plain form (elementary torch operations, 32 bits and more, rounded
once at the end), ``True`` this framework's kernels.
"""
import math

import torch

own = False

COEF = (3.4445, -4.7750, 2.0315)       # quintic a s + b s^3 + c s^5 applied to the singular values, five times
STEPS = 5
EPS = 1e-7


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a 7x7 stem filter flattened to [64, 3*7*7]: the smallest matrix of an image classifier, an odd inner size;
        # fifteen tiny products one after the other, so latency counts
        {"name": "orth_stem", "op": "orth", "batch": 1, "rows": 64, "cols": 147, "dtype": "bf16"},
        # the 3x3 filters of a residual network's last stage, stacked: ordinary training work, many wide matrices
        {"name": "orth_batch", "op": "orth", "batch": 8, "rows": 512, "cols": 4608, "dtype": "bf16"},
        # one large projection, taller than wide, with its gradient in 32 bits
        {"name": "orth_tall_fp32", "op": "orth", "batch": 1, "rows": 8192, "cols": 2048, "dtype": "fp32"},
        # LeNet-5: a whole optimizer step over tiny matrices and vectors
        {"name": "muon_lenet5", "op": "muon", "net": "lenet5"},
        # ResNet-50: 54 matrices from 64 x 64 to 2048 x 1024 and 512 x 4608, 107 vectors
        {"name": "muon_resnet50", "op": "muon", "net": "resnet50"},
        # one token through the block: serving, bound by reading the three weights
        {"name": "gated_token", "op": "gated", "tokens": 1, "width": 4096, "hidden": 12288, "act": "silu", "train": False},
        # a prompt of ragged length through a smaller block
        {"name": "gated_prompt", "op": "gated", "tokens": 517, "width": 2048, "hidden": 5632, "act": "gelu", "train": False},
        # a small block trained on a ragged batch, sizes that are no multiple of a tile
        {"name": "gated_train_small", "op": "gated", "tokens": 100, "width": 200, "hidden": 520, "act": "silu", "train": True},
        # a training step of a full-sized block, forward and backward
        {"name": "gated_train", "op": "gated", "tokens": 8192, "width": 4096, "hidden": 12288, "act": "silu", "train": True},
        # one token's distribution while sampling: 32-bit logits, an odd vocabulary, the twenty most likely tokens
        {"name": "logp_token", "op": "logp", "rows": 1, "vocab": 50257, "top": 20, "dtype": "fp32", "train": False},
        # scoring a text against a large vocabulary, five alternatives a token, a tenth of the vocabulary masked out
        {"name": "logp_score", "op": "logp", "rows": 2048, "vocab": 131072, "top": 5, "dtype": "bf16", "train": False},
        # policy training: log probability and entropy of every token, with the gradient; some rows are padding
        {"name": "logp_train", "op": "logp", "rows": 8192, "vocab": 32000, "top": 0, "dtype": "bf16", "train": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    limit = {}
    for c in listed():
        w, old = work(c), limit.get(c["op"], {"bytes": 0, "flops": 0})
        limit[c["op"]] = {k: max(w[k], old[k]) for k in w}
    while True:
        op = rng.choice(["orth", "orth", "muon", "gated", "gated", "gated", "logp", "logp", "logp"])
        if op == "orth":
            case = {"op": op, "batch": _log_int(rng, 1, 12), "rows": _log_int(rng, 16, 8192), "cols": _log_int(rng, 16, 8192),
                    "dtype": rng.choice(["bf16", "fp32"])}
        elif op == "muon":
            case = {"op": op, "net": "mlp", "inputs": _log_int(rng, 16, 2000), "hidden": _log_int(rng, 16, 2500),
                    "layers": rng.randint(1, 6), "classes": _log_int(rng, 5, 1000)}
        elif op == "gated":
            case = {"op": op, "tokens": _log_int(rng, 1, 8192), "width": _log_int(rng, 64, 4096),
                    "hidden": _log_int(rng, 128, 12288), "act": rng.choice(["silu", "gelu"]), "train": rng.random() < 0.5}
            if rng.random() < 0.7:          # model builders take multiples of eight; other sizes are padded
                case["width"], case["hidden"] = case["width"] // 8 * 8, case["hidden"] // 8 * 8
        else:
            case = {"op": op, "rows": _log_int(rng, 1, 8192), "vocab": _log_int(rng, 1000, 150000),
                    "top": rng.choice([0, 1, 5, 20]), "dtype": rng.choice(["bf16", "fp32"]), "train": rng.random() < 0.5}
        w = work(case)
        if all(w[k] <= limit[op][k] for k in w):
            return case


# ------------------------------------------------------------------------------------------------------------ work
def _net_shapes(case):
    """Parameter shapes in registration order."""
    if case["net"] == "lenet5":
        return [(6, 1, 5, 5), (6,), (16, 6, 5, 5), (16,), (120, 400), (120,), (84, 120), (84,), (10, 84), (10,)]
    if case["net"] == "resnet50":
        shapes, cin = [(64, 3, 7, 7), (64,), (64,)], 64
        for width, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
            for b in range(blocks):
                for s in ((width, cin, 1, 1), (width, width, 3, 3), (4 * width, width, 1, 1)):
                    shapes += [s, (s[0],), (s[0],)]
                if b == 0:
                    shapes += [(4 * width, cin, 1, 1), (4 * width,), (4 * width,)]
                cin = 4 * width
        return shapes + [(1000, 2048), (1000,)]
    dims = [case["inputs"]] + [case["hidden"]] * case["layers"] + [case["classes"]]
    out = []
    for i, o in zip(dims[:-1], dims[1:]):
        out += [(o, i), (o,)]
    return out


def _orth_flops(rows, cols):
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (3 * m * m * n + m * m * m)          # X X^T and its square are symmetric: half of each


def work(case):
    op = case["op"]
    if op == "orth":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * n * (2 if case["dtype"] == "bf16" else 4),
                "flops": case["batch"] * _orth_flops(case["rows"], case["cols"])}
    if op == "muon":
        total = flops = 0
        for s in _net_shapes(case):
            n = math.prod(s)
            if len(s) > 1:
                total += 5 * 4 * n                      # weight and momentum read and written, gradient read
                flops += _orth_flops(s[0], n // s[0])
            else:
                total += 7 * 4 * n                      # weight and both moments read and written, gradient read
                flops += 12 * n
        return {"bytes": total, "flops": flops}
    if op == "gated":
        t, d, f = case["tokens"], case["width"], case["hidden"]
        if case["train"]:
            return {"bytes": 2 * (4 * t * d + 6 * d * f), "flops": 18 * t * d * f}
        return {"bytes": 2 * (2 * t * d + 3 * d * f), "flops": 6 * t * d * f}
    size = 2 if case["dtype"] == "bf16" else 4
    n, v = case["rows"], case["vocab"]
    outs = n * (8 + 4 + 4 + case["top"] * 12)
    if case["train"]:
        return {"bytes": 2 * n * v * size + outs + n * (8 + 4 * case["top"]), "flops": 12 * n * v}
    return {"bytes": n * v * size + outs, "flops": 5 * n * v}


# ------------------------------------------------------------------------------------------------------------ inputs
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _inputs(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(1000003 * seed + 17)

    def randn(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    op = case["op"]
    if op == "orth":
        # gradients have a decaying spectrum: a strong part of low rank over a noise floor
        b, m, n = case["batch"], case["rows"], case["cols"]
        r = max(1, min(m, n) // 8)
        low = torch.matmul(randn(b, m, r), randn(b, r, n)) * (1.0 / math.sqrt(r))
        mat = (low + 0.3 * randn(b, m, n)) * 1e-3
        return {"g": (mat if b > 1 else mat[0]).to(DTYPES[case["dtype"]])}
    if op == "muon":
        # one flat buffer for each kind of value, every tensor on a 1024-element boundary, as ParamArena lays them out
        shapes = _net_shapes(case)
        total = sum((math.prod(s) + 1023) // 1024 * 1024 for s in shapes)
        out = {k: torch.zeros(total, device=dev) for k in ("flat_params", "flat_grads", "flat_moments", "flat_squares")}
        out["views"], off = [], 0
        for s in shapes:
            stride = torch.empty(s, memory_format=torch.channels_last if len(s) == 4 else torch.contiguous_format,
                                 device="meta").stride()              # Conv2d keeps its filters channels-last
            views = [torch.as_strided(out[k], s, stride, off)
                     for k in ("flat_params", "flat_grads", "flat_moments", "flat_squares")]
            fan = math.prod(s[1:]) if len(s) > 1 else 1
            for view, scale in zip(views, (fan ** -0.5, 1e-2, 3e-2)):
                view.copy_(randn(*s, scale=scale))
            if len(s) == 1:
                views[2].zero_()                        # vectors go through Adam, from its first step
            out["views"].append(views)
            off += (math.prod(s) + 1023) // 1024 * 1024
        return out
    if op == "gated":
        t, d, f = case["tokens"], case["width"], case["hidden"]
        bf = torch.bfloat16
        out = {"x": randn(t, d, dtype=bf), "w_gate": randn(f, d, scale=d ** -0.5, dtype=bf),
               "w_up": randn(f, d, scale=d ** -0.5, dtype=bf), "w_down": randn(d, f, scale=f ** -0.5, dtype=bf)}
        if case["train"]:
            out["dy"] = randn(t, d, scale=1e-2, dtype=bf)
        return out
    n, v = case["rows"], case["vocab"]
    z = randn(n, v, scale=2.5)
    if not case["train"] and n > 1:
        masked = torch.rand(v, generator=g, device=dev) < 0.1
        z[:, masked] = float("-inf")                    # a constraint that forbids part of the vocabulary
    tok = torch.randint(0, v, (n,), generator=g, device=dev)
    out = {"logits": z.to(DTYPES[case["dtype"]]), "tokens": tok}
    if case["train"]:
        tok[torch.rand(n, generator=g, device=dev) < 0.1] = -100        # padding
        out["g_logp"], out["g_ent"] = randn(n, scale=1.0 / n), randn(n, scale=0.01 / n)
        if case["top"]:
            out["g_top"] = randn(n, case["top"], scale=1.0 / n)
    return out


MUON = {"lr": 0.02, "momentum": 0.95, "weight_decay": 0.01, "adam_lr": 3e-4, "adam_betas": (0.9, 0.95), "adam_eps": 1e-8}


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["op"] == "muon":
        state["step"] = 0
        if own:
            from distributed_deep_learning_amd.optim import Muon
            from distributed_deep_learning_amd.parallel import ParamArena
            leaves = [torch.nn.Parameter(v[0].clone()) for v in state["views"]]
            arena = ParamArena([(f"p{i}", p) for i, p in enumerate(leaves)])
            opt = Muon(arena, **MUON)
            for p, v in zip(leaves, state["views"]):
                p.grad.copy_(v[1])
                opt.state_of(p, "momentum").copy_(v[2])
            state["opt"] = opt
    elif case.get("train"):
        names = ("x", "w_gate", "w_up", "w_down") if case["op"] == "gated" else ("logits",)
        for k in names:
            state[k].requires_grad_(own)
    return state


# ------------------------------------------------------------------------------------------------------------ runs
def run(state):
    op = state["case"]["op"]
    return (_run_own if own else _run_plain)[op](state)


def _own_orth(s):
    from distributed_deep_learning_amd.ops import kernels as K
    return K.orthogonalize(s["g"])


def _own_muon(s):
    s["opt"].step(zero_grad=False)
    return [s["opt"].arena.master, s["opt"].flat_state["momentum"], s["opt"].flat_state["exp_avg_sq"]]


def _own_gated(s):
    from distributed_deep_learning_amd.nn import functional as F
    c = s["case"]
    if not c["train"]:
        with torch.no_grad():
            return F.gated_mlp(s["x"], s["w_gate"], s["w_up"], s["w_down"], activation=c["act"])
    leaves = (s["x"], s["w_gate"], s["w_up"], s["w_down"])
    y = F.gated_mlp(*leaves, activation=c["act"])
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


def _own_logp(s):
    from distributed_deep_learning_amd.nn import functional as F
    c = s["case"]
    if not c["train"]:
        with torch.no_grad():
            return list(F.token_logprobs(s["logits"], s["tokens"], top=c["top"]))
    out = F.token_logprobs(s["logits"], s["tokens"], top=c["top"])
    heads, gs = [out[0], out[1]], [s["g_logp"], s["g_ent"]]
    if c["top"]:
        heads.append(out[2]), gs.append(s["g_top"])
    (dz,) = torch.autograd.grad(heads, s["logits"], gs)
    return [t.detach() for t in out] + [dz]


def _newton_schulz(g):
    """fp32 [.., m, n] -> fp32; the squares of the norm are summed in 64 bits."""
    a, b, c = COEF
    tall = g.shape[-2] > g.shape[-1]
    x = g.transpose(-1, -2) if tall else g
    norm = x.double().pow(2).sum((-2, -1), keepdim=True).sqrt()
    x = (x / (norm + EPS).float()).contiguous()
    for _ in range(STEPS):
        s = torch.matmul(x, x.transpose(-1, -2).contiguous())
        x = a * x + torch.matmul(b * s + c * torch.matmul(s, s), x)
    return x.transpose(-1, -2) if tall else x


def _plain_orth(s):
    return _newton_schulz(s["g"].float()).to(s["g"].dtype).contiguous()


def _plain_muon(s):
    h = MUON
    s["step"] += 1
    b1, b2 = h["adam_betas"]
    c1, c2 = 1.0 - b1 ** s["step"], 1.0 - b2 ** s["step"]
    for p, g, m, v in s["views"]:
        if p.dim() > 1:
            m.mul_(h["momentum"]).add_(g)
            u = (g + h["momentum"] * m).reshape(p.shape[0], -1)
            o = _newton_schulz(u).reshape(p.shape)
            scale = max(1.0, u.shape[0] / u.shape[1]) ** 0.5
            p.mul_(1.0 - h["lr"] * h["weight_decay"]).add_(o, alpha=-h["lr"] * scale)
        else:
            m.mul_(b1).add_(g, alpha=1.0 - b1)
            v.mul_(b2).add_(g * g, alpha=1.0 - b2)
            p.sub_(h["adam_lr"] * (m / c1) / ((v / c2).sqrt() + h["adam_eps"]))
    return [s["flat_params"], s["flat_moments"], s["flat_squares"]]


def _activation(g, act):
    """Value and derivative."""
    if act == "silu":
        sg = torch.sigmoid(g)
        return g * sg, sg * (1.0 + g * (1.0 - sg))
    cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_gated(s):
    c = s["case"]
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    g, u = x @ wg.t(), x @ wu.t()
    act, dact = _activation(g, c["act"])
    h = act * u
    y = h @ wd.t()
    bf = torch.bfloat16
    if not c["train"]:
        return y.to(bf)
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * dact, dh * act
    return [t.to(bf) for t in (y, dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ h)]


def _top(z, k):
    """The k largest of every row, equal values by the lowest index."""
    taken = torch.zeros_like(z, dtype=torch.bool)
    iota = torch.arange(z.shape[1], device=z.device)
    vals, idx = [], []
    for _ in range(k):
        v = z.masked_fill(taken, float("-inf")).amax(1, keepdim=True)
        i = torch.where((z == v) & ~taken, iota, z.shape[1]).amin(1, keepdim=True)
        taken.scatter_(1, i, True)
        vals.append(v), idx.append(i)
    return torch.cat(vals, 1), torch.cat(idx, 1)


def _plain_logp(s):
    c = s["case"]
    z, tok = s["logits"].float(), s["tokens"]
    valid = (tok >= 0) & (tok < z.shape[1])
    t = torch.where(valid, tok, 0)[:, None]
    mx = z.amax(1, keepdim=True)
    e = torch.exp(z - mx)
    total = e.sum(1, keepdim=True)
    lse = mx + torch.log(total)
    p = e / total
    ent = (lse - (p * torch.where(p > 0, z, 0.0)).sum(1, keepdim=True))
    logp = torch.where(valid, (z.gather(1, t) - lse)[:, 0], 0.0)
    if c["top"]:
        tv, ti = _top(z, c["top"])
        tv = tv - lse
    else:
        tv, ti = z.new_empty(z.shape[0], 0), tok.new_empty(z.shape[0], 0)
    out = [logp, ent[:, 0], tv, ti]
    if c["train"]:
        gl = torch.where(valid, s["g_logp"], 0.0)[:, None]
        ge = s["g_ent"][:, None]
        gt = s["g_top"] if c["top"] else None
        total_g = gl + (gt.sum(1, keepdim=True) if c["top"] else 0.0)
        dz = -p * (total_g + ge * torch.where(p > 0, z - lse + ent, 0.0))
        dz.scatter_add_(1, t, gl)
        if c["top"]:
            dz.scatter_add_(1, ti, gt)
        out.append(dz.to(s["logits"].dtype))
    return out


_run_own = {"orth": _own_orth, "muon": _own_muon, "gated": _own_gated, "logp": _own_logp}
_run_plain = {"orth": _plain_orth, "muon": _plain_muon, "gated": _plain_gated, "logp": _plain_logp}


# ------------------------------------------------------------------------------------------------------------ exact
def _poly64(mat):
    """Newton-Schulz steps from the definition, X <- X (a + b X^T X + c (X^T X)^2) on the thin side, 64 bits."""
    a, b, c = COEF
    x = mat.double()
    flip = x.shape[-1] > x.shape[-2]
    if flip:
        x = x.transpose(-1, -2)
    x = (x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + EPS)).contiguous()
    eye = torch.eye(x.shape[-1], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        gram = torch.matmul(x.transpose(-1, -2).contiguous(), x)
        x = torch.matmul(x, a * eye + torch.matmul(gram, b * eye + c * gram))
    return x.transpose(-1, -2) if flip else x


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "orth":
        return _poly64(s["g"]).contiguous()
    if op == "muon":
        h, outs, off = MUON, [torch.zeros_like(s["flat_params"], dtype=torch.float64) for _ in range(3)], 0
        for p, g, m, _ in s["views"]:
            stride, p, g, m, v = p.stride(), p.double(), g.double(), m.double(), None
            if p.dim() > 1:
                m = h["momentum"] * m + g
                rows, cols = p.shape[0], p[0].numel()
                o = _poly64((g + h["momentum"] * m).reshape(rows, cols)).reshape(p.shape)
                p = p - h["lr"] * (math.sqrt(max(1.0, rows / cols)) * o + h["weight_decay"] * p)
            else:                                       # Adam's first step: the corrected moments are g and g^2
                m, v = (1.0 - h["adam_betas"][0]) * g, (1.0 - h["adam_betas"][1]) * g * g
                p = p - h["adam_lr"] * g / (g.abs() + h["adam_eps"])
            for flat, t in zip(outs, (p, m, v)):
                if t is not None:
                    torch.as_strided(flat, t.shape, stride, off).copy_(t)
            off += (p.numel() + 1023) // 1024 * 1024
        return outs
    if op == "gated":
        x, wg, wu, wd = (s[k].double() for k in ("x", "w_gate", "w_up", "w_down"))
        g, u = torch.matmul(x, wg.t().contiguous()), torch.matmul(x, wu.t().contiguous())
        if case["act"] == "silu":
            sg = 1.0 / (1.0 + torch.exp(-g))
            act, slope = g * sg, sg + g * sg * (1.0 - sg)
        else:
            cdf = 0.5 * torch.erfc(-g / math.sqrt(2.0))
            act, slope = g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
        h = act * u
        y = torch.matmul(h, wd.t().contiguous())
        if not case["train"]:
            return y
        dy = s["dy"].double()
        dh = torch.matmul(dy, wd)
        dg, du = dh * u * slope, dh * act
        return [y, torch.matmul(dg, wg) + torch.matmul(du, wu), torch.matmul(dg.t().contiguous(), x),
                torch.matmul(du.t().contiguous(), x), torch.matmul(dy.t().contiguous(), h)]
    z, tok = s["logits"].double(), s["tokens"]
    n, v = z.shape
    inside = (tok >= 0) & (tok < v)
    row = torch.arange(n, device=z.device)
    logq = z - torch.logsumexp(z, 1, keepdim=True)
    q = torch.exp(logq)
    plogp = torch.where(q > 0, q * logq, 0.0)
    ent = -plogp.sum(1)
    logp = torch.where(inside, logq[row, tok.clamp(0, v - 1)], 0.0)
    order = torch.sort(z, dim=1, descending=True, stable=True)[1][:, :case["top"]] if case["top"] else tok.new_empty(n, 0)
    out = [logp, ent, logq.gather(1, order), order.contiguous()]
    if case["train"]:
        gl = torch.where(inside, s["g_logp"].double(), 0.0)
        dz = -s["g_ent"].double()[:, None] * (plogp + q * ent[:, None])
        direct = torch.zeros_like(z)
        direct[row[inside], tok[inside]] += gl[inside]
        if case["top"]:
            direct.scatter_add_(1, order, s["g_top"].double())
        dz += direct - q * direct.sum(1, keepdim=True)
        out.append(dz)
    return out
