"""Workloads of the transformer operators: the gated feed-forward block, the norms around a block with its gate and
residual scale, and the global gradient norm with clipping - as plain torch formulas, as this package's calls, and from
their definitions in 64 bits.

``own`` chooses between the plain form (False) and the package's kernels (True)."""
import array
import math
import random

import torch

own = False

ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token through the feed-forward block of a small model: latency
        {"name": "ff_token", "op": "ff", "train": False, "N": 1, "D": 1024, "F": 2732, "act": "silu"},
        # one decoding step of a batch of sequences, a large layer: every weight is read for eight rows
        {"name": "ff_tokens", "op": "ff", "train": False, "N": 8, "D": 4096, "F": 10924, "act": "silu"},
        # a prompt, ragged in every dimension
        {"name": "ff_prompt", "op": "ff", "train": False, "N": 1021, "D": 2048, "F": 5464, "act": "gelu_tanh"},
        # a training step's forward and backward through one layer, ordinary and large
        {"name": "ff_train", "op": "ff", "train": True, "N": 2048, "D": 2048, "F": 5464, "act": "silu"},
        {"name": "ff_train_large", "op": "ff", "train": True, "N": 8192, "D": 4096, "F": 10924, "act": "silu"},
        # the norms around a block: one decoded token, a long prompt, training at an odd width with one gate row per
        # sequence (512 tokens), training of a wide model with one gate per channel
        {"name": "norm_token", "op": "norm", "train": False, "N": 1, "M": 4096, "gate_rows": 1, "post": True},
        {"name": "norm_prompt", "op": "norm", "train": False, "N": 16384, "M": 4096, "gate_rows": 16384, "post": True},
        {"name": "norm_train", "op": "norm", "train": True, "N": 4096, "M": 2051, "gate_rows": 512, "post": True},
        {"name": "norm_train_wide", "op": "norm", "train": True, "N": 8192, "M": 8192, "gate_rows": 8192, "post": True},
        # gradients of a small network, clipped; of a network of 300 tensors, clipped; of 400 tensors that are views of
        # one flat buffer, below the limit and left where they are
        {"name": "clip_small", "op": "clip", "count": 64, "total": 1000003, "flat": False, "norm": 4.0, "max_norm": 1.0},
        {"name": "clip_large", "op": "clip", "count": 300, "total": 400000000, "flat": False, "norm": 2.5, "max_norm": 1.0},
        {"name": "clip_below", "op": "clip", "count": 400, "total": 100000001, "flat": True, "norm": 0.3, "max_norm": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ff", "norm", "clip"))
    if op == "ff":
        D = _log(rng, 64, 1024) * 4
        return {"op": "ff", "train": rng.random() < 0.5, "N": _log(rng, 1, 8192), "D": D,
                "F": min(10924, int(D * rng.uniform(1.0, 4.0)) // 4 * 4), "act": rng.choice(ACTS)}
    if op == "norm":
        N, M = _log(rng, 1, 8192), _log(rng, 60, 8192)
        # the rows that share one gate row: every row its own, a sequence, or all (0: no gate)
        gate_rows = rng.choice((0, 1, N, max(1, N // rng.randint(1, 16))))
        return {"op": "norm", "train": rng.random() < 0.5, "N": N, "M": M, "gate_rows": gate_rows, "post": rng.random() < 0.8}
    return {"op": "clip", "count": _log(rng, 1, 2000), "total": _log(rng, 2500, 400000000), "flat": rng.random() < 0.5,
            "norm": rng.uniform(0.1, 10.0), "max_norm": 1.0}


def _in_place(case):
    """Whether the gradients are clipped where they are: passes repeat only if they then stay as they were."""
    return case["flat"] and case["norm"] < case["max_norm"] / 3


def _pad4(x):
    return (x + 3) // 4 * 4


def _groups(case):
    """Gate rows: each serves gate_rows consecutive rows, the last what is left."""
    return -(-case["N"] // case["gate_rows"]) if case["gate_rows"] else 0


def _sizes(case):
    """Sizes of the gradients: as in a network, half of them vectors, the rest matrices that hold nearly everything.
    Tensors of their own have padded rows, so a multiple of four elements; views of a flat buffer have any number."""
    r = random.Random(case["count"] * 7919 + case["total"])
    share = [r.uniform(0.5, 1.5) * (1.0 if i % 2 == 0 else 1e-3) for i in range(case["count"])]
    scale = (case["total"] - case["count"]) / sum(share)
    sizes = [1 + int(s * scale) for s in share]
    sizes[0] += case["total"] - sum(sizes)
    return sizes if case["flat"] else [_pad4(n) for n in sizes]


# ---------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, device="cuda", generator=g)  # noqa: E731
    buf = lambda *shape: torch.zeros(shape, device="cuda")  # noqa: E731
    s = dict(case)
    if case["op"] == "ff":
        N, D, F = case["N"], case["D"], case["F"]
        s["X"] = rnd(N, D)
        s["Wg"], s["Wu"] = rnd(D, F) / math.sqrt(D), rnd(D, F) / math.sqrt(D)
        s["Wd"] = rnd(F, D) / math.sqrt(F)
        s["H"], s["Y"] = buf(N, F), buf(N, D)
        s["work"] = buf(32 << 20)        # partial sums of split products, kept by the program
        if case["train"]:
            s["dY"] = rnd(N, D) * 1e-2
            s["G"], s["U"], s["dG"], s["dU"] = buf(N, F), buf(N, F), buf(N, F), buf(N, F)
            s["dX"], s["dWg"], s["dWu"], s["dWd"] = buf(N, D), buf(D, F), buf(D, F), buf(F, D)
        return s
    if case["op"] == "norm":
        N, M, P = case["N"], case["M"], _pad4(case["M"])

        def rows(n, values):
            t = buf(n, P)
            t[:, :M] = values
            return t
        # a few channels carry most of the energy, as residual streams do
        big = 1.0 + 20.0 * (torch.rand((1, M), device="cuda", generator=g) < 0.01)
        s["B"], s["R"] = rows(N, 0.3 * rnd(N, M) * big), rows(N, 2.0 * rnd(N, M) * big)
        s["wpre"] = rows(1, 1.0 + 0.2 * rnd(1, M))[0]
        s["wpost"] = rows(1, 1.0 + 0.2 * rnd(1, M))[0] if case["post"] else None
        s["gate"] = rows(_groups(case), 0.5 * rnd(_groups(case), M)) if case["gate_rows"] else None
        s["rscale"], s["scale"] = 0.9, 0.7
        s["Rout"], s["Y"], s["rstd_post"], s["rstd_pre"] = buf(N, P), buf(N, P), buf(N), buf(N)
        if case["train"]:
            s["dRout"], s["dY"] = rows(N, 1e-2 * rnd(N, M)), rows(N, 1e-2 * rnd(N, M))
            s["dR"], s["dB"], s["dwpre"] = buf(N, P), buf(N, P), buf(P)
            s["dwpost"] = buf(P) if case["post"] else None
            s["dgate"] = buf(_groups(case), P) if case["gate_rows"] else None
            s["work"] = buf(64 << 20)    # partial column sums, kept by the program
        return s
    sizes = _sizes(case)
    stds = [math.exp(x) for x in torch.randn(len(sizes), generator=torch.Generator().manual_seed(seed)).tolist()]
    unit = case["norm"] / math.sqrt(sum(n * d * d for n, d in zip(sizes, stds)))
    if case["flat"]:    # as a bucket for a collective holds them: one behind the other, at any alignment
        s["all"] = rnd(sum(sizes))
        s["grads"] = list(torch.split(s["all"], sizes))
        torch._foreach_mul_(s["grads"], [d * unit for d in stds])
    else:
        s["grads"] = [rnd(n) * (d * unit) for n, d in zip(sizes, stds)]
    if _in_place(case):
        s["clipped"], s["out"] = s["all"], s["grads"]
    else:               # the clipped gradients are kept beside the gradients
        s["clipped"] = buf(sum(sizes))
        s["out"] = list(torch.split(s["clipped"], sizes))
    # what a program keeps beside its gradients: where they are, and how long
    s["sizes"] = array.array("q", sizes)
    s["src"] = array.array("q", [t.data_ptr() for t in s["grads"]])
    s["dst"] = array.array("q", [t.data_ptr() for t in s["out"]])
    s["result"] = buf(2)
    s["work"] = torch.zeros(1 << 16, device="cuda", dtype=torch.float64)
    return s


# ---------------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _own(s)
    return {"ff": _plain_ff, "norm": _plain_norm, "clip": _plain_clip}[s["op"]](s)


def _act(name, x):
    """act(x) and its derivative, elementwise."""
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-x))
        return x * p, p * (1.0 + x * (1.0 - p))
    if name == "gelu":
        c = 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5)))
        return x * c, c + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (x + 0.044715 * x * x * x))
        return 0.5 * x * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * x * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * x * x)
    if name == "relu":
        return torch.where(x > 0, x, torch.zeros_like(x)), (x > 0).to(x.dtype)
    p = 1.0 / (1.0 + torch.exp(-x))
    return p, p * (1.0 - p)


def _plain_ff(s):
    G, U = s["X"] @ s["Wg"], s["X"] @ s["Wu"]
    a, da = _act(s["act"], G)
    H = a * U
    Y = H @ s["Wd"]
    if not s["train"]:
        return [Y]
    dH = s["dY"] @ s["Wd"].T
    dG, dU = dH * U * da, dH * a
    return [Y, dG @ s["Wg"].T + dU @ s["Wu"].T, s["X"].T @ dG, s["X"].T @ dU, H.T @ s["dY"]]


def _spread(s, M):
    """The gate of every row."""
    if s["gate"] is None:
        return 1.0
    return s["gate"][:, :M].repeat_interleave(s["gate_rows"], 0)[:s["N"]]


def _sum_groups(s, x):
    """Sums of x over the rows of each gate row."""
    n = s["gate"].shape[0]
    if s["gate_rows"] * n > x.shape[0]:
        x = torch.cat([x, torch.zeros((s["gate_rows"] * n - x.shape[0], x.shape[1]), device=x.device, dtype=x.dtype)])
    return x.reshape(n, s["gate_rows"], -1).sum(1)


def _padded(s, M, *outs):
    return [torch.nn.functional.pad(t, (0, _pad4(M) - M)) for t in outs]


def _plain_norm(s):
    M = s["M"]
    B, R, wpre, gate = s["B"][:, :M], s["R"][:, :M], s["wpre"][:M], _spread(s, M)
    if s["post"]:
        rb = torch.rsqrt((B * B).mean(1, keepdim=True) + EPS)
        Bn = B * rb
        P = Bn * s["wpost"][:M]
    else:
        P = B
    Rout = s["rscale"] * R + s["scale"] * gate * P
    rr = torch.rsqrt((Rout * Rout).mean(1, keepdim=True) + EPS)
    Rn = Rout * rr
    outs = [Rout, Rn * wpre]
    if s["train"]:
        dY = s["dY"][:, :M]
        q = dY * wpre
        dT = s["dRout"][:, :M] + rr * (q - Rn * (q * Rn).mean(1, keepdim=True))
        dP = s["scale"] * gate * dT
        outs += [s["rscale"] * dT]
        if s["post"]:
            q = dP * s["wpost"][:M]
            outs += [rb * (q - Bn * (q * Bn).mean(1, keepdim=True))]
        else:
            outs += [dP]
        outs += [(dY * Rn).sum(0)]
        if s["post"]:
            outs += [(dP * Bn).sum(0)]
        if s["gate"] is not None:
            outs += [_sum_groups(s, s["scale"] * P * dT)]
    return _padded(s, M, *outs)


def _plain_clip(s):
    flat = torch.cat(s["grads"]).double()
    norm = torch.sqrt((flat * flat).sum())
    keep = torch.clamp(s["max_norm"] / norm, max=1.0)
    return [norm.float(), (flat * keep).float()]


def _own(s):
    import __graft_entry__
    cu32 = __graft_entry__.load_package().cu32
    p = lambda name: s[name].data_ptr() if s.get(name) is not None else 0  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "ff":
        ff, act = cu32.Cuda_gatedFF, ACTS.index(s["act"])
        ff.gatedFF([stream], 1, p("X"), p("Wg"), p("Wu"), p("Wd"), p("G"), p("U"), p("H"), p("Y"),
                   p("work"), s["work"].numel(), s["N"], s["D"], s["F"], act)
        if not s["train"]:
            return [s["Y"]]
        ff.gatedFF_delta([stream], 1, p("dY"), p("X"), p("Wg"), p("Wu"), p("Wd"), p("G"), p("U"), p("H"),
                         p("dG"), p("dU"), p("dX"), p("dWg"), p("dWu"), p("dWd"), p("work"), s["work"].numel(),
                         s["N"], s["D"], s["F"], act)
        return [s["Y"], s["dX"], s["dWg"], s["dWu"], s["dWd"]]
    if s["op"] == "norm":
        nr, M, P = cu32.Cuda_normResidual, s["M"], _pad4(s["M"])
        nr.normResidual(stream, p("B"), p("R"), p("gate"), s["gate_rows"], p("wpost"), p("wpre"), p("Rout"), p("Y"),
                        p("rstd_post"), p("rstd_pre"), s["N"], P, M, s["rscale"], s["scale"], EPS)
        outs = [s["Rout"], s["Y"]]
        if s["train"]:
            nr.normResidual_delta(stream, p("dRout"), p("dY"), p("B"), p("Rout"), p("gate"), s["gate_rows"], p("wpost"),
                                  p("wpre"), p("rstd_post"), p("rstd_pre"), p("dR"), p("dB"), p("dgate"), p("dwpost"),
                                  p("dwpre"), p("work"), s["work"].numel(), s["N"], P, M, s["rscale"], s["scale"])
            outs += [s["dR"], s["dB"], s["dwpre"]]
            outs += [s["dwpost"]] if s["post"] else []
            outs += [s["dgate"]] if s["gate"] is not None else []
        return outs
    cu32.Cuda_gradClip.gradClip(stream, s["src"], s["dst"], s["sizes"], len(s["sizes"]), s["max_norm"], p("result"),
                                p("work"), s["work"].numel())
    return [s["result"][0], s["clipped"]]


# ---------------------------------------------------------------------------------------------------------- floors
def work(case):
    """What a pass cannot do without: each input read once, each output written once."""
    if case["op"] == "ff":
        N, D, F = case["N"], case["D"], case["F"]
        return {"bytes": 4 * ((4 if case["train"] else 2) * N * D + (6 if case["train"] else 3) * D * F),
                "flops": (18 if case["train"] else 6) * N * D * F}
    if case["op"] == "norm":
        n = case["N"] * _pad4(case["M"])
        return {"bytes": 4 * n * (8 if case["train"] else 4), "flops": n * (40 if case["train"] else 12)}
    return {"bytes": 4 * case["total"] * (1 if _in_place(case) else 2), "flops": 3 * case["total"]}


# ---------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()
         if k not in ("work", "out", "G", "U", "H", "dG", "dU", "dX", "dWg", "dWu", "dWd")}
    if case["op"] == "ff":
        X, Wg, Wu, Wd = s["X"], s["Wg"], s["Wu"], s["Wd"]
        G = torch.einsum("nd,df->nf", X, Wg).requires_grad_(case["train"])
        a = {"silu": lambda x: x * torch.sigmoid(x), "gelu": lambda x: x * 0.5 * torch.erfc(-x / 2 ** 0.5),
             "gelu_tanh": lambda x: x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)),
             "relu": lambda x: x.clamp(min=0), "sigmoid": torch.sigmoid}[case["act"]](G)
        U = torch.einsum("nd,df->nf", X, Wu)
        H = a.detach() * U
        Y = torch.einsum("nf,fd->nd", H, Wd)
        if not case["train"]:
            return [Y]
        dH = torch.einsum("nd,fd->nf", s["dY"], Wd)
        (dG,) = torch.autograd.grad(a, G, dH * U)
        dU = dH * a.detach()
        dX = torch.einsum("nf,df->nd", dG, Wg) + torch.einsum("nf,df->nd", dU, Wu)
        return [Y, dX, torch.einsum("nd,nf->df", X, dG), torch.einsum("nd,nf->df", X, dU),
                torch.einsum("nf,nd->fd", H, s["dY"])]
    if case["op"] == "norm":
        M, N = case["M"], case["N"]
        leaf = {k: s[k][..., :M].clone().requires_grad_(True) for k in ("B", "R", "wpre", "wpost", "gate") if s[k] is not None}
        row = torch.arange(N, device="cuda")
        unit = lambda x: x / torch.sqrt(x.square().sum(1, keepdim=True) / M + EPS)  # noqa: E731
        with torch.set_grad_enabled(bool(case["train"])):
            branch = unit(leaf["B"]) * leaf["wpost"] if case["post"] else leaf["B"]
            if case["gate_rows"]:
                branch = leaf["gate"][row // case["gate_rows"]] * branch
            Rout = s["rscale"] * leaf["R"] + s["scale"] * branch
            Y = unit(Rout) * leaf["wpre"]
        outs = [Rout.detach(), Y.detach()]
        if case["train"]:
            by = [k for k in ("R", "B", "wpre", "wpost", "gate") if k in leaf]
            outs += torch.autograd.grad((Rout, Y), [leaf[k] for k in by], (s["dRout"][:, :M], s["dY"][:, :M]))
        wide = []
        for t in outs:
            z = torch.zeros((*t.shape[:-1], _pad4(M)), device="cuda", dtype=torch.float64)
            z[..., :M] = t
            wide.append(z)
        return wide
    total = torch.stack([torch.linalg.vector_norm(t.double()) for t in s["grads"]])
    norm = torch.linalg.vector_norm(total)
    ratio = float(min(1.0, case["max_norm"] / float(norm)))
    return [norm, torch.cat([t.double() * ratio for t in s["grads"]])]
