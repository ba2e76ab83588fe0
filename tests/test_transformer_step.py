"""The transformer operators as they are used together: the feed-forward half of a layer between its two norms, forward and
backward through the engine object, and the gradients it leaves clipped by their global norm - against the same half
layer differentiated in 64 bits.

Tolerance: a result lies behind at most six products (G, U and Y forward; deltaH, deltaX and a weight gradient backward),
each within 1e-6 of its norm, and at most eight elementwise or norm stages of some 3e-7; data are random, so a stage passes
the relative error of its input on about as it is (silu and the norms' factor at most 1.2 times): 1e-5 of the norm.
"""
import pytest


class Pool:
    """The engine's device-memory pool, NaN-filled: nothing may depend on what a scratch buffer held."""

    def __init__(self, torch):
        self.torch = torch

    def __call__(self, nfloats):
        t = self.torch.full((nfloats,), float("nan"), device="cuda")
        return t.data_ptr(), t


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,group,width,hidden", [(1, 1, 64, 128), (6, 2, 130, 260), (48, 24, 258, 1028), (500, 125, 131, 516)])
def test_feed_forward_half_layer_trains(pkg, cuda, tokens, group, width, hidden):
    torch = cuda
    eng = pkg.engine.Cu32Engine(torch.cuda.get_device_properties(0).multi_processor_count, Pool(torch),
                                [torch.cuda.current_stream().cuda_stream])
    M, F = pkg.engine.pad4(width), pkg.engine.pad4(hidden)
    groups = -(-tokens // group)
    g = torch.Generator(device="cuda").manual_seed(tokens + width)

    def make(rows, cols, pitch, scale=1.0, shift=0.0):      # padding zero, as the engine keeps it
        t = torch.zeros((rows, pitch), device="cuda")
        t[:, :cols] = scale * torch.randn((rows, cols), device="cuda", generator=g) + shift
        return t
    leaf = {"B0": make(tokens, width, M), "R0": make(tokens, width, M, 2.0), "gate1": make(groups, width, M),
            "post1": make(1, width, M, 0.2, 1.0), "pre1": make(1, width, M, 0.2, 1.0), "gate2": make(groups, width, M),
            "post2": make(1, width, M, 0.2, 1.0), "pre2": make(1, width, M, 0.2, 1.0),
            "Wg": make(M, hidden, F, width ** -0.5), "Wu": make(M, hidden, F, width ** -0.5), "Wd": make(F, width, M, hidden ** -0.5)}
    for n in ("Wg", "Wu"):
        leaf[n][width:] = 0
    leaf["Wd"][hidden:] = 0
    dR2, dY2 = make(tokens, width, M), make(tokens, width, M)
    new = lambda *s: torch.full(s, float("nan"), device="cuda")  # noqa: E731
    R1, Y1, B1, R2, Y2 = (new(tokens, M) for _ in range(5))
    G, U, H = (new(tokens, F) for _ in range(3))
    rstd = [new(tokens) for _ in range(4)]
    p = lambda t: t.data_ptr()  # noqa: E731
    rs, sc = 0.9, 0.8

    # forward
    eng.normResidual(p(R1), p(Y1), p(leaf["B0"]), p(leaf["R0"]), p(leaf["pre1"]), tokens, M, width, Wpost=p(leaf["post1"]),
                     gate=p(leaf["gate1"]), gate_rows=group, res_scale=rs, scale=sc, rstd_post=p(rstd[0]), rstd_pre=p(rstd[1]))
    eng.gatedFF(p(B1), p(Y1), p(leaf["Wg"]), p(leaf["Wu"]), p(leaf["Wd"]), tokens, M, F, pkg.cu32.Cuda_gatedFF.SILU, H=p(H),
                G=p(G), U=p(U))
    eng.normResidual(p(R2), p(Y2), p(B1), p(R1), p(leaf["pre2"]), tokens, M, width, Wpost=p(leaf["post2"]),
                     gate=p(leaf["gate2"]), gate_rows=group, res_scale=rs, scale=sc, rstd_post=p(rstd[2]), rstd_pre=p(rstd[3]))
    # serving gives the same block output without keeping anything
    served = new(tokens, M)
    eng.gatedFF(p(served), p(Y1), p(leaf["Wg"]), p(leaf["Wu"]), p(leaf["Wd"]), tokens, M, F, pkg.cu32.Cuda_gatedFF.SILU)
    assert torch.equal(served, B1)
    # backward: the second norm, the block, the first norm
    grad = {n: torch.full_like(t, float("nan")) for n, t in leaf.items()}
    dR1, dB1, dY1 = (new(tokens, M) for _ in range(3))
    eng.normResidual_delta(p(dR1), p(dB1), p(grad["pre2"]), p(dR2), p(dY2), p(B1), p(R2), p(leaf["pre2"]), p(rstd[3]), tokens, M,
                           width, Wpost=p(leaf["post2"]), rstd_post=p(rstd[2]), deltaWpost=p(grad["post2"]),
                           gate=p(leaf["gate2"]), gate_rows=group, deltaGate=p(grad["gate2"]), res_scale=rs, scale=sc)
    eng.gatedFF_delta(p(dY1), p(grad["Wg"]), p(grad["Wu"]), p(grad["Wd"]), p(dB1), p(Y1), p(leaf["Wg"]), p(leaf["Wu"]),
                      p(leaf["Wd"]), p(G), p(U), p(H), tokens, M, F, pkg.cu32.Cuda_gatedFF.SILU)
    eng.normResidual_delta(p(grad["R0"]), p(grad["B0"]), p(grad["pre1"]), p(dR1), p(dY1), p(leaf["B0"]), p(R1), p(leaf["pre1"]),
                           p(rstd[1]), tokens, M, width, Wpost=p(leaf["post1"]), rstd_post=p(rstd[0]),
                           deltaWpost=p(grad["post1"]), gate=p(leaf["gate1"]), gate_rows=group, deltaGate=p(grad["gate1"]),
                           res_scale=rs, scale=sc)

    # the same in 64 bits
    ref = {n: t.double().requires_grad_(True) for n, t in leaf.items()}
    unit = lambda x: x / torch.sqrt((x * x).sum(1, keepdim=True) / width + 1e-6)  # noqa: E731
    spread = lambda t: t.repeat_interleave(group, 0)[:tokens]  # noqa: E731
    r1 = rs * ref["R0"] + sc * spread(ref["gate1"]) * unit(ref["B0"]) * ref["post1"]
    y1 = unit(r1) * ref["pre1"]
    b1 = (torch.nn.functional.silu(y1 @ ref["Wg"]) * (y1 @ ref["Wu"])) @ ref["Wd"]
    r2 = rs * r1 + sc * spread(ref["gate2"]) * unit(b1) * ref["post2"]
    y2 = unit(r2) * ref["pre2"]
    want = torch.autograd.grad((r2, y2), [ref[n] for n in leaf], (dR2.double(), dY2.double()))
    off = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
    for got, exact in ((R1, r1), (Y1, y1), (B1, b1), (R2, r2), (Y2, y2)):
        assert off(got, exact.detach()) <= 1e-5
    for n, exact in zip(leaf, want):
        assert off(grad[n], exact) <= 1e-5, n

    # all parameters' gradients, clipped to half their norm, in place
    names = [n for n in leaf if n not in ("B0", "R0")]
    addr, sizes = [p(grad[n]) for n in names], [grad[n].numel() for n in names]
    result = new(2)
    before = {n: grad[n].clone() for n in names}
    norm = torch.sqrt(sum((before[n].double() ** 2).sum() for n in names)).item()
    eng.gradNorm(addr, sizes, p(result))
    assert abs(result[0].item() - norm) <= 1.1 * 2.0 ** -24 * norm
    eng.gradClip(addr, addr, sizes, 0.5 * norm, p(result))
    for n in names:
        exact = 0.5 * before[n].double()
        assert ((grad[n].double() - exact).abs() <= 3 * 2.0 ** -24 * exact.abs() + 1e-45).all(), n
    eng.release()
    assert pkg.cu32.read_status() == 0
