"""Gated feed-forward block (cu32_gatedFF, cu32_gatedFF_delta): H = act(X Wg) * (X Wu), Y = H Wd and the gradients.

Each stage is compared with the formula in 64 bits applied to what the device used as that stage's inputs, so that every
product is held to the library's budget for contractions (relative Frobenius error 1e-6, 1e-4 elementwise over the rms)
and the elementwise stages to a bound in units of the rounding 2^-24:
  - H = act(G) U: the exponential, the reciprocal, the sum and the products are at most 16 roundings; where the
    activation's argument is rounded first, that rounding grows with the argument: 2z of GELU_TANH (s changes by 2z times
    the relative change of 2z: 4 |2z| roundings for the cube, its factor and the sum), x / sqrt 2 of GELU (erfc changes by
    at most x^2 times it: 4 x^2).  Results below 1e-37 lose bits to the denormal range (absolute term).
  - deltaG, deltaU multiply deltaH, which stays inside the kernel, by known factors: deltaH's budget of 1e-6 of its rms
    spread over the factors, plus 1e-6 for the factors themselves.
"""
import ctypes

import pytest

EPS = 2.0 ** -24
ACTS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def act64(torch, act, x):
    """act(x) and act'(x) in 64 bits."""
    import math
    p = torch.sigmoid(x)
    if act == 0:
        return x * p, p + x * p * (1 - p)
    if act == 1:
        phi = 0.5 * torch.erfc(-x / math.sqrt(2))
        return x * phi, phi + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    if act == 2:
        k = 2 * math.sqrt(2 / math.pi)
        s = torch.sigmoid(k * (x + 0.044715 * x ** 3))
        return x * s, s + x * s * (1 - s) * k * (1 + 3 * 0.044715 * x * x)
    if act == 3:
        return x.clamp(min=0), (x > 0).double()
    return p, p * (1 - p)


def act_roundings(act, x):
    """Bound of the relative error of act(x) in units of 2^-24 (see above)."""
    if act == 1:
        return 16 + 4 * x * x
    if act == 2:
        return 16 + 4 * 1.6 * (x.abs() + 0.044715 * x.abs() ** 3)
    return 16 + 0 * x


def near(got, want, frob=1e-6, elem=1e-4):
    d = got.double() - want
    norm = want.norm()
    rms = norm / want.numel() ** 0.5
    assert (d.norm() / norm).item() <= frob, (d.norm() / norm).item()
    assert (d.abs() / want.abs().clamp(min=rms)).max().item() <= elem


class Block:
    """Operands on the device, outputs between canaries."""

    def __init__(self, torch, N, D, F, seed, scale=1.0):
        import gpu_util as G
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
        self.N, self.D, self.F = N, D, F
        self.X, self.Wg, self.Wu = r(N, D), scale * r(D, F) / D ** 0.5, r(D, F) / D ** 0.5
        self.Wd, self.dY = r(F, D) / F ** 0.5, r(N, D)
        out = lambda a, b: G.Out(a * b)  # noqa: E731
        self.G, self.U, self.H, self.Y = out(N, F), out(N, F), out(N, F), out(N, D)
        self.dG, self.dU, self.dX = out(N, F), out(N, F), out(N, D)
        self.dWg, self.dWu, self.dWd = out(D, F), out(D, F), out(F, D)

    def forward(self, pkg, act, save=True, work=None):
        import gpu_util as G
        pkg.cu32.Cuda_gatedFF.gatedFF([G.stream()], 1, self.X.data_ptr(), self.Wg.data_ptr(), self.Wu.data_ptr(),
                                      self.Wd.data_ptr(), self.G.ptr if save else 0, self.U.ptr if save else 0, self.H.ptr,
                                      self.Y.ptr, work.data_ptr() if work is not None else 0,
                                      work.numel() if work is not None else 0, self.N, self.D, self.F, act)

    def backward(self, pkg, act, work=None, over=None):
        """over: "U" or "G" - deltaG lies over H, deltaU over U or G."""
        import gpu_util as G
        pkg.cu32.Cuda_gatedFF.gatedFF_delta(
            [G.stream()], 1, self.dY.data_ptr(), self.X.data_ptr(), self.Wg.data_ptr(), self.Wu.data_ptr(),
            self.Wd.data_ptr(), self.G.ptr, self.U.ptr, self.H.ptr, self.H.ptr if over else self.dG.ptr,
            getattr(self, over).ptr if over else self.dU.ptr, self.dX.ptr, self.dWg.ptr, self.dWu.ptr, self.dWd.ptr,
            work.data_ptr() if work is not None else 0, work.numel() if work is not None else 0, self.N, self.D, self.F, act)

    def get(self, torch, name):
        """An output as a device tensor; checks the canaries."""
        shape = {"Y": (self.N, self.D), "dX": (self.N, self.D), "dWg": (self.D, self.F), "dWu": (self.D, self.F),
                 "dWd": (self.F, self.D)}.get(name, (self.N, self.F))
        return torch.as_tensor(getattr(self, name).host(shape)).cuda()


def check_forward(torch, b, act):
    G, U, H, Y = (b.get(torch, n) for n in "GUHY")
    near(G, b.X.double() @ b.Wg.double())
    near(U, b.X.double() @ b.Wu.double())
    want = act64(torch, act, G.double())[0] * U.double()
    bound = act_roundings(act, G.double()) * EPS * want.abs() + 1e-37
    assert ((H.double() - want).abs() <= bound).all()
    near(Y, H.double() @ b.Wd.double())


def check_backward(torch, b, act, G, U):
    dG, dU = b.get(torch, "dG"), b.get(torch, "dU")
    dH = b.dY.double() @ b.Wd.double().T
    a, da = act64(torch, act, G.double())
    for got, factor in ((dG, U.double() * da), (dU, a)):
        want = dH * factor
        budget = 1e-6 * (dH.norm() / dH.numel() ** 0.5) * factor.norm() + 1e-6 * want.norm()
        assert ((got.double() - want).norm() <= budget).item(), ((got.double() - want).norm() / want.norm()).item()
    near(b.get(torch, "dX"), dG.double() @ b.Wg.double().T + dU.double() @ b.Wu.double().T)
    near(b.get(torch, "dWg"), b.X.double().T @ dG.double())
    near(b.get(torch, "dWu"), b.X.double().T @ dU.double())
    near(b.get(torch, "dWd"), b.get(torch, "H").double().T @ b.dY.double())


# ---------------------------------------------------------------------------------------------------- without a GPU
def test_gated_ff_refusals(pkg):
    lib = pkg.cu32.load()
    s = (ctypes.c_int64 * 10)()
    P = 0x10000

    def fwd(X=P, Wg=P, Wu=P, Wd=P, G=0, U=0, H=P, Y=P, work=0, room=0, N=4, D=8, F=12, act=0, length=1):
        return lib.cu32_gatedFF(s, length, X, Wg, Wu, Wd, G, U, H, Y, work, room, N, D, F, act)

    def bwd(dY=P, X=P, Wg=P, Wu=P, Wd=P, G=P, U=P, H=P, dG=2 * P, dU=P, dX=P, dWg=P, dWu=P, dWd=P, work=0, room=0, N=4, D=8,
            F=12, act=0, length=1):
        return lib.cu32_gatedFF_delta(s, length, dY, X, Wg, Wu, Wd, G, U, H, dG, dU, dX, dWg, dWu, dWd, work, room, N, D, F, act)
    for call in (fwd, bwd):
        assert call(length=0) == -3 and call(length=11) == -3
        for dim in ("N", "D", "F"):
            assert call(**{dim: 0}) == -2 and call(**{dim: -4}) == -2
        assert call(N=1 << 29, D=8) == -2                       # more than 2^31 elements
        assert call(D=6) == -4 and call(F=10) == -4
        assert call(act=-1) == -8 and call(act=5) == -8
        assert call(work=P + 4) == -4
    for name in ("X", "Wg", "Wu", "Wd", "H", "Y"):
        assert fwd(**{name: 0}) == -1 and fwd(**{name: P + 8}) == -4
    assert fwd(G=P) == -1 and fwd(U=P) == -1                    # both or none
    assert fwd(G=P + 4, U=P) == -4
    for name in ("dY", "Wd", "G", "U", "dG", "dU"):
        assert bwd(**{name: 0}) == -1
    assert bwd(Wg=0) == -1 and bwd(X=0) == -1 and bwd(H=0) == -1
    assert bwd(X=0, dWg=0) == -1                                # deltaWu still needs X
    Q = 2 * P
    assert bwd(G=Q) == -8 and bwd(U=Q) == -8 and bwd(dU=Q) == -8 and bwd(dG=P) == -8    # deltaG over G, U or deltaU
    for name in ("dY", "X", "Wg", "Wu", "Wd", "G", "U", "H", "dG", "dU", "dX", "dWg", "dWu", "dWd"):
        assert bwd(**{name: P + 4}) == -4
    with pytest.raises(pkg.cu32.CudaException, match="CU32_E_NULL"):
        pkg.cu32.Cuda_gatedFF.gatedFF([0], 1, 0, P, P, P, 0, 0, P, P, 0, 0, 4, 8, 12, 0)


def test_gated_ff_refuses_overlaps(pkg):
    """An output over an operand or another output, whole or in part: CU32_E_ARG, apart from the replacements the calls
    allow.  (With up to 24 rows deltaU over H would leave deltaWd without its H, and deltaX over deltaY without its deltaY.)"""
    lib = pkg.cu32.load()
    s = (ctypes.c_int64 * 10)()
    for N, D, F in ((4, 8, 12), (40, 8, 12), (300, 8, 12)):
        size = {"X": N * D, "Y": N * D, "dY": N * D, "dX": N * D, "Wg": D * F, "Wu": D * F, "Wd": D * F, "dWg": D * F,
                "dWu": D * F, "dWd": D * F, "G": N * F, "U": N * F, "H": N * F, "dG": N * F, "dU": N * F}
        place, at = {}, 0x10000
        for name, n in size.items():            # one behind the other, without a gap
            place[name] = at
            at += 4 * n

        def fwd(**at):
            a = dict(place, **at)
            return lib.cu32_gatedFF(s, 1, a["X"], a["Wg"], a["Wu"], a["Wd"], a["G"], a["U"], a["H"], a["Y"], 0, 0, N, D, F, 0)

        def bwd(**at):
            a = dict(place, **at)
            return lib.cu32_gatedFF_delta(s, 1, *(a[n] for n in ("dY", "X", "Wg", "Wu", "Wd", "G", "U", "H", "dG", "dU", "dX", "dWg",
                                                                 "dWu", "dWd")), 0, 0, N, D, F, 0)
        for call, outs, ins, allowed in ((fwd, ("G", "U", "H", "Y"), ("X", "Wg", "Wu", "Wd"), ()),
                                         (bwd, ("dG", "dU", "dX", "dWg", "dWu", "dWd"), ("dY", "X", "Wg", "Wu", "Wd", "G", "U", "H"),
                                          (("dG", "H"), ("dU", "G"), ("dU", "U")))):
            for out in outs:
                for other in outs + ins:
                    if other == out:
                        continue
                    for there in (place[other], place[other] + 4 * size[other] - 16, place[other] - 4 * size[out] + 16):
                        if there == place[other] and (out, other) in allowed:
                            continue
                        assert call(**{out: there}) == -8, (N, out, other)


# ---------------------------------------------------------------------------------------------------- on the GPU
SHAPES = [
    # N, D, F: up to 8 rows, up to 128 rows (both: one kernel per power of two), tiles; with every kind of tail
    (1, 4, 4), (1, 64, 132), (2, 36, 260), (3, 516, 64), (4, 128, 128), (5, 132, 1028), (8, 1028, 516), (9, 68, 36),
    (16, 260, 2052), (17, 4, 4), (17, 36, 68), (33, 128, 260), (128, 64, 64), (10, 4, 4), (24, 36, 4100),
    (64, 1028, 516), (65, 260, 260), (100, 2052, 132), (130, 260, 516), (257, 516, 132),
    (520, 132, 1028),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gated_ff_forward_and_gradients(pkg, cuda, shape):
    import gpu_util as G
    torch = cuda
    for act in range(5):
        b = Block(torch, *shape, seed=sum(shape) + act)
        work = torch.full((max(4, pkg.cu32.Cuda_gatedFF.work(*shape)),), float("nan"), device="cuda")
        b.forward(pkg, act, work=work)
        check_forward(torch, b, act)
        b.backward(pkg, act, work=work)
        check_backward(torch, b, act, b.get(torch, "G"), b.get(torch, "U"))
        G.check_status(pkg)


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [1, 3, 4])
def test_gated_ff_on_every_tile(pkg, cuda, tile):
    """The three tile shapes of the gated forms, several tiles in both directions, ragged edges."""
    import gpu_util as G
    torch = cuda
    pkg.cu32.tune("tile", tile)
    for shape in ((600, 260, 580), (300, 100, 1156)):
        b = Block(torch, *shape, seed=tile)
        b.forward(pkg, 0)
        check_forward(torch, b, 0)
        b.backward(pkg, 0)
        check_backward(torch, b, 0, b.get(torch, "G"), b.get(torch, "U"))
        G.check_status(pkg)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 2052, 132), (7, 68, 516), (12, 516, 132), (50, 132, 1028), (200, 516, 260)], ids=str)
def test_serving_gives_the_bits_of_training_and_repeats(pkg, cuda, shape):
    torch = cuda
    b = Block(torch, *shape, seed=3)
    work = torch.full((pkg.cu32.Cuda_gatedFF.work(*shape) + 4,), float("nan"), device="cuda")
    b.forward(pkg, 2, save=True, work=work)
    H, Y = b.get(torch, "H"), b.get(torch, "Y")
    for save in (False, True, False):
        b.H.view.fill_(float("nan"))
        b.Y.view.fill_(float("nan"))
        b.forward(pkg, 2, save=save, work=work)
        assert torch.equal(b.get(torch, "H"), H) and torch.equal(b.get(torch, "Y"), Y)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 8228, 68), (33, 8228, 68), (40, 64, 20004), (130, 8228, 68), (150, 64, 20004)], ids=str)
def test_long_reductions(pkg, cuda, shape):
    """A width beyond the interval after which plain products flush their sums, and a long hidden axis cut into slices."""
    torch = cuda
    b = Block(torch, *shape, seed=4)
    work = torch.full((pkg.cu32.Cuda_gatedFF.work(*shape) + 4,), float("nan"), device="cuda")
    b.forward(pkg, 0, work=work)
    check_forward(torch, b, 0)
    b.backward(pkg, 0, work=work)
    check_backward(torch, b, 0, b.get(torch, "G"), b.get(torch, "U"))


@pytest.mark.gpu
def test_gradients_in_place_and_single_ones(pkg, cuda):
    """deltaG over H and deltaU over U or G give the bits of separate buffers; gradients that are not asked for are
    skipped, with the operands only they need absent."""
    import gpu_util as G
    torch = cuda
    b = Block(torch, 70, 132, 196, seed=5)
    b.forward(pkg, 1)
    kept = {n: getattr(b, n).view.clone() for n in "GUH"}
    b.backward(pkg, 1)
    first = {n: b.get(torch, n) for n in ("dG", "dU", "dX", "dWg", "dWu", "dWd")}
    for over in "UG":
        for n in ("dX", "dWg", "dWu", "dWd"):
            getattr(b, n).view.fill_(float("nan"))
        b.backward(pkg, 1, over=over)
        assert torch.equal(b.get(torch, "H"), first["dG"]) and torch.equal(b.get(torch, over), first["dU"])
        for n in ("dX", "dWg", "dWu", "dWd"):
            assert torch.equal(b.get(torch, n), first[n])
        for n in "GUH":
            getattr(b, n).view.copy_(kept[n])
    call = pkg.cu32.Cuda_gatedFF.gatedFF_delta
    p = lambda t: t.data_ptr()  # noqa: E731
    for n in ("dX", "dWg", "dWu", "dWd"):
        getattr(b, n).view.fill_(float("nan"))
    call([G.stream()], 1, p(b.dY), 0, p(b.Wg), p(b.Wu), p(b.Wd), b.G.ptr, b.U.ptr, 0, b.dG.ptr, b.dU.ptr, b.dX.ptr, 0, 0, 0,
         0, 0, b.N, b.D, b.F, 1)
    assert torch.equal(b.get(torch, "dX"), first["dX"]) and torch.isnan(b.get(torch, "dWg")).all()
    call([G.stream()], 1, p(b.dY), p(b.X), 0, 0, p(b.Wd), b.G.ptr, b.U.ptr, b.H.ptr, b.dG.ptr, b.dU.ptr, 0, 0, b.dWu.ptr,
         b.dWd.ptr, 0, 0, b.N, b.D, b.F, 1)
    assert torch.equal(b.get(torch, "dWu"), first["dWu"]) and torch.equal(b.get(torch, "dWd"), first["dWd"])
    assert torch.isnan(b.get(torch, "dWg")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("act", range(5), ids=ACTS)
@pytest.mark.parametrize("rows", [3, 40])
def test_far_pre_activations(pkg, cuda, act, rows):
    """Pre-activations from 1e-6 to 1e4 in size: exponentials that overflow or vanish leave finite, right values.  The
    products are exact here (one non-zero term each), so H, deltaG and deltaU show the activation alone."""
    torch = cuda
    b = Block(torch, rows, 8, 256, seed=6)
    b.X.zero_()
    b.X[:, 0] = 1.0
    x = torch.logspace(-6, 4, 128, device="cuda")
    b.Wg.zero_()
    b.Wg[0, :128], b.Wg[0, 128:] = x, -x
    b.Wu.zero_()
    b.Wu[0] = 1.0
    b.Wd.zero_()
    b.Wd[:, 0] = 1.0
    b.dY.zero_()
    b.dY[:, 0] = 1.0
    b.forward(pkg, act)
    check = b.get(torch, "G").double()
    a, da = act64(torch, act, check)
    H = b.get(torch, "H").double()
    assert torch.isfinite(H).all()
    assert ((H - a).abs() <= act_roundings(act, check) * EPS * a.abs() + 1e-37).all()
    b.backward(pkg, act)
    dG, dU = b.get(torch, "dG").double(), b.get(torch, "dU").double()
    # act' is a sum of terms of up to about 1.1 in size (x s (1 - s) dz stays below that): 32 roundings of their size
    assert ((dG - da).abs() <= 32 * EPS * (1.1 + 0 * da)).all()
    assert ((dU - a).abs() <= act_roundings(act, check) * EPS * a.abs() + 1e-37).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [20, 128])
def test_without_scratch(pkg, cuda, rows):
    """No scratch, or too little: the same call by another path, nothing written beyond what was given."""
    torch = cuda
    b = Block(torch, rows, 516, 772, seed=10)
    need = pkg.cu32.Cuda_gatedFF.work(rows, 516, 772)
    for room in (0, need // 2 // 4 * 4, need):
        work = torch.full((need + 64,), 7.0, device="cuda")
        b.forward(pkg, 0, work=work[:room] if room else None)
        check_forward(torch, b, 0)
        b.backward(pkg, 0, work=work[:room] if room else None)
        check_backward(torch, b, 0, b.get(torch, "G"), b.get(torch, "U"))
        assert (work[room:] == 7.0).all()


@pytest.mark.gpu
def test_gradients_against_differences(pkg, cuda):
    """deltaX and the weight gradients against central differences of sum(Y deltaY) taken in 64 bits: the formula itself."""
    torch = cuda
    for act in (0, 1, 2, 4):       # the smooth ones
        b = Block(torch, 20, 12, 16, seed=40 + act)
        b.forward(pkg, act)
        b.backward(pkg, act)
        ops = {n: getattr(b, n).double() for n in ("X", "Wg", "Wu", "Wd")}

        def value(o):
            return ((act64(torch, act, o["X"] @ o["Wg"])[0] * (o["X"] @ o["Wu"])) @ o["Wd"] * b.dY.double()).sum()
        step = 1e-5      # third-order remainder 1e-10, rounding 1e-16 / 1e-5
        for n in ("X", "Wg", "Wu", "Wd"):
            got = b.get(torch, "d" + n).double()
            for at in ((0, 0), (3, 7), (got.shape[0] - 1, got.shape[1] - 1)):
                hi, lo = dict(ops), dict(ops)
                hi[n], lo[n] = ops[n].clone(), ops[n].clone()
                hi[n][at] += step
                lo[n][at] -= step
                diff = (value(hi) - value(lo)) / (2 * step)
                # two products' budgets of 1e-6 of the gradient's rms each, elementwise 1e-4 as everywhere
                assert abs(got[at] - diff) <= 1e-4 * max(diff.abs().item(), got.norm().item() / got.numel() ** 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 64, 200])
def test_on_a_stream_of_its_own_and_in_a_graph(pkg, cuda, rows):
    """The calls run on streams[0] alone; captured once, replayed with new inputs, forward and gradients."""
    torch = cuda
    b = Block(torch, rows, 132, 260, seed=8)
    work = torch.empty(pkg.cu32.Cuda_gatedFF.work(rows, 132, 260) + 4, device="cuda")
    b.forward(pkg, 0, work=work)          # first use outside the capture
    b.backward(pkg, 0, work=work)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        b.forward(pkg, 0, work=work)
        b.backward(pkg, 0, work=work)
    b.X.mul_(0.5).add_(0.25)
    b.dY.mul_(-1.5)
    graph.replay()
    torch.cuda.synchronize()
    check_forward(torch, b, 0)
    check_backward(torch, b, 0, b.get(torch, "G"), b.get(torch, "U"))
    del graph


@pytest.mark.gpu
def test_two_streams_at_once(pkg, cuda):
    """Blocks on streams of their own, each with scratch of its own."""
    torch = cuda
    blocks = [Block(torch, n, 260, 1028, seed=50 + n) for n in (5, 30, 300)]
    works = [torch.empty(pkg.cu32.Cuda_gatedFF.work(b.N, b.D, b.F) + 4, device="cuda") for b in blocks]
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    for _ in range(10):
        for b, w, s in zip(blocks, works, streams):
            with torch.cuda.stream(s):
                b.forward(pkg, 0, work=w)
                b.backward(pkg, 0, work=w)
    torch.cuda.synchronize()
    for b in blocks:
        check_forward(torch, b, 0)
        check_backward(torch, b, 0, b.get(torch, "G"), b.get(torch, "U"))


@pytest.mark.gpu
def test_rows_do_not_depend_on_their_company(pkg, cuda):
    """A NaN in one row stays in that row, forward and in deltaX."""
    torch = cuda
    for rows in (4, 40, 140):
        b = Block(torch, rows, 68, 132, seed=9)
        work = torch.empty(pkg.cu32.Cuda_gatedFF.work(rows, 68, 132) + 4, device="cuda")
        b.forward(pkg, 0, work=work)
        clean = b.get(torch, "Y")
        b.X[2, 5] = float("nan")
        b.forward(pkg, 0, work=work)
        Y = b.get(torch, "Y")
        assert torch.isnan(Y[2]).all()
        others = [i for i in range(rows) if i != 2]
        assert torch.equal(Y[others], clean[others])
        b.backward(pkg, 0)
        dX = b.get(torch, "dX")
        assert torch.isnan(dX[2]).all() and torch.isfinite(dX[others]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 40, 128, 140])
def test_bad_weights_stay_in_their_column(pkg, cuda, rows):
    """A NaN weight reaches its hidden unit, whose H makes the rows of Y and, through deltaG, of deltaX NaN; no other column
    of G, U, H, deltaG or of the weights' gradients."""
    torch = cuda
    b = Block(torch, rows, 68, 132, seed=19)
    work = torch.empty(pkg.cu32.Cuda_gatedFF.work(rows, 68, 132) + 4, device="cuda")
    b.Wg[7, 33] = float("nan")
    b.forward(pkg, 0, work=work)
    b.backward(pkg, 0, work=work)
    others = [f for f in range(132) if f != 33]
    for name in ("G", "H", "dG", "dU", "dWg", "dWu"):
        t = b.get(torch, name)
        assert torch.isnan(t[:, 33]).all() and torch.isfinite(t[:, others]).all(), name
    assert torch.isfinite(b.get(torch, "U")).all()
    dWd = b.get(torch, "dWd")
    assert torch.isnan(dWd[33]).all() and torch.isfinite(dWd[others]).all()
    for name in ("Y", "dX"):
        assert torch.isnan(b.get(torch, name)).all(), name


@pytest.mark.gpu
def test_gradients_of_rows_do_not_depend_on_their_company_with_scratch(pkg, cuda):
    """An infinity in one row of deltaY stays in that row of deltaG, deltaU and deltaX."""
    torch = cuda
    for rows in (1, 5, 40, 128, 140):
        b = Block(torch, rows, 68, 132, seed=29)
        work = torch.empty(pkg.cu32.Cuda_gatedFF.work(rows, 68, 132) + 4, device="cuda")
        b.forward(pkg, 0, work=work)
        b.backward(pkg, 0, work=work)
        clean = {n: b.get(torch, n) for n in ("dG", "dU", "dX")}
        b.dY[rows // 2, 5] = float("inf")
        b.backward(pkg, 0, work=work)
        others = [i for i in range(rows) if i != rows // 2]
        for n, was in clean.items():
            now = b.get(torch, n)
            assert not torch.isfinite(now[rows // 2]).any() and torch.equal(now[others], was[others]), n


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 7, 24, 25])
@pytest.mark.parametrize("dims", [(4, 4), (60, 260), (68, 1028), (260, 64), (1500, 1284)], ids=str)
def test_weight_gradients_of_few_rows(pkg, cuda, rows, dims):
    """Edges of the few-row weight gradients' tiles (64 x 256 and multiples), with and without scratch, deltaG over H."""
    torch = cuda
    D, F = dims
    b = Block(torch, rows, D, F, seed=rows)
    work = torch.empty(pkg.cu32.Cuda_gatedFF.work(rows, D, F) + 4, device="cuda")
    b.forward(pkg, 0, work=work)
    G, U, H = (b.get(torch, n) for n in "GUH")
    for w in (work, None):
        b.backward(pkg, 0, work=w)
        check_backward(torch, b, 0, G, U)
    kept = {n: b.get(torch, n) for n in ("dG", "dU", "dWg", "dWu", "dWd")}
    b.backward(pkg, 0, work=None, over="U")            # deltaG over H, deltaU over U: deltaWd has to read H before
    assert torch.equal(b.get(torch, "H"), kept["dG"]) and torch.equal(b.get(torch, "U"), kept["dU"])
    for n in ("dWg", "dWu", "dWd"):
        assert torch.equal(b.get(torch, n), kept[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("wanted", [("dWg",), ("dWu",), ("dWd",), ("dWd", "dWu"), ("dX", "dWd"), ()], ids=str)
def test_few_rows_single_gradients(pkg, cuda, wanted):
    import gpu_util as Gu
    torch = cuda
    N, D, F = 6, 68, 132
    b = Block(torch, N, D, F, seed=77)
    work = torch.empty(pkg.cu32.Cuda_gatedFF.work(N, D, F) + 4, device="cuda")
    b.forward(pkg, 0, work=work)
    b.backward(pkg, 0, work=work)
    all_of = {n: b.get(torch, n) for n in ("dX", "dWg", "dWu", "dWd", "dG", "dU")}
    for n in ("dX", "dWg", "dWu", "dWd", "dG", "dU"):
        getattr(b, n).view.fill_(-7.0)
    o = lambda n: getattr(b, n).ptr if n in wanted else 0  # noqa: E731
    pkg.cu32.Cuda_gatedFF.gatedFF_delta(
        [Gu.stream()], 1, b.dY.data_ptr(), b.X.data_ptr(), b.Wg.data_ptr(), b.Wu.data_ptr(), b.Wd.data_ptr(), b.G.ptr, b.U.ptr,
        b.H.ptr, b.dG.ptr, b.dU.ptr, o("dX"), o("dWg"), o("dWu"), o("dWd"), work.data_ptr(), work.numel(), N, D, F, 0)
    for n, was in all_of.items():
        now = b.get(torch, n)
        assert torch.equal(now, was) if n in wanted or n in ("dG", "dU") else bool((now == -7.0).all()), n


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 40, 200])
def test_delta_over_what_the_call_does_not_read(pkg, cuda, rows):
    """Without deltaWd nothing reads H, without the weights' gradients nothing reads X: they may be replaced."""
    import gpu_util as Gu
    torch = cuda
    D, F = 68, 132
    b = Block(torch, rows, D, F, seed=78)
    work = torch.empty(pkg.cu32.Cuda_gatedFF.work(rows, D, F) + 4, device="cuda")
    b.forward(pkg, 0, work=work)
    b.backward(pkg, 0, work=work)
    want = {n: b.get(torch, n) for n in ("dX", "dG", "dU")}
    b.dG.view.fill_(float("nan"))
    pkg.cu32.Cuda_gatedFF.gatedFF_delta(
        [Gu.stream()], 1, b.dY.data_ptr(), b.X.data_ptr(), b.Wg.data_ptr(), b.Wu.data_ptr(), b.Wd.data_ptr(), b.G.ptr, b.U.ptr,
        b.H.ptr, b.dG.ptr, b.H.ptr, b.X.data_ptr(), 0, 0, 0, work.data_ptr(), work.numel(), rows, D, F, 0)
    assert torch.equal(b.get(torch, "dG"), want["dG"]) and torch.equal(b.get(torch, "H"), want["dU"])
    assert torch.equal(b.X, want["dX"])


@pytest.mark.gpu
@pytest.mark.parametrize("shape,keys", [((3, 64, 20000), (1, 6, 9, 15)), ((8, 64, 132), (3, 12)), ((1, 260, 64), (8, 9))], ids=str)
def test_a_lost_wait_ends_the_call_with_a_status(pkg, cuda, shape, keys):
    """One warp of a block counts a wait as run out while the others of its block, and of its cluster (one, two and four
    blocks), got theirs: the kernels end, the status word names a role of theirs, nothing is written beyond the outputs,
    and the next call is right."""
    torch = cuda
    b = Block(torch, *shape, seed=79)
    try:
        for key in keys:
            pkg.cu32.tune("rows_give_up", key)
            b.forward(pkg, 0)
            word = pkg.cu32.read_status()
            assert word >> 24 in (10, 11, 12), hex(word)
            for name in "GUHY":
                b.get(torch, name)
            pkg.cu32.tune("rows_give_up", 0)
            b.forward(pkg, 0)
            check_forward(torch, b, 0)
            assert pkg.cu32.read_status() == 0
    finally:
        pkg.cu32.tune("rows_give_up", 0)


def test_rows_give_up_key(pkg):
    lib = pkg.cu32.load()
    v = ctypes.c_int(-5)
    assert lib.cu32_get_tune(b"rows_give_up", ctypes.byref(v)) == 0 and v.value == 0
    assert lib.cu32_tune(b"rows_give_up", 17) == -8 and lib.cu32_tune(b"rows_give_up", -1) == -8


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(130, 8228, 68), (200, 20004, 36)], ids=str)
def test_scratch_of_a_long_model_axis(pkg, cuda, shape):
    """deltaH is a product over D: where D is long and F small it alone is cut through the scratch, whose size has to count
    it."""
    import gpu_util as G
    torch = cuda
    b = Block(torch, *shape, seed=80)
    need = pkg.cu32.Cuda_gatedFF.work(*shape)
    assert need >= shape[0] * shape[2]
    work = torch.full((need + 64,), float("nan"), device="cuda")
    b.forward(pkg, 0, work=work[:need])
    check_forward(torch, b, 0)
    work.fill_(float("nan"))
    b.backward(pkg, 0, work=work[:need])
    check_backward(torch, b, 0, b.get(torch, "G"), b.get(torch, "U"))
    assert torch.isfinite(work[:shape[0] * shape[2]]).all() and torch.isnan(work[need:]).all()
    G.check_status(pkg)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,scratch,cut", [
    # the gated launch; it and deltaH; deltaWd, deltaWg and deltaWu, deltaH beside a deltaWd in two pieces; Y
    ((400, 260, 5124), True, (1, 0)), ((1000, 260, 5124), True, (1, 1)), ((260, 1028, 4100), True, (0, 3)),
    ((260, 1028, 4100), False, (0, 3)), ((1021, 2048, 5464), True, (1, 2)), ((1021, 2048, 5464), False, (1, 3)),
    ((2048, 2048, 5464), True, (0, 3)), ((1000, 5124, 1028), False, (1, 3)), ((1300, 3588, 516), True, (1, 0)),
], ids=str)
def test_products_in_two_pieces_of_columns(pkg, cuda, shape, scratch, cut):
    """Columns that fill whole rounds of tiles, and the rest in smaller tiles beside the last round: the offsets of the second
    piece, and what stands beside or behind it.  The counter says that the cuts were made."""
    import gpu_util as G
    torch = cuda

    def cuts():
        v = ctypes.c_int()
        assert pkg.cu32.load().cu32_get_tune(b"column_cuts", ctypes.byref(v)) == 0
        return v.value
    b = Block(torch, *shape, seed=81)
    n = pkg.cu32.Cuda_gatedFF.work(*shape) if scratch else 0
    work = torch.full((n,), float("nan"), device="cuda") if n else None
    counts = [cuts()]
    b.forward(pkg, 0, work=work)
    counts.append(cuts())
    b.backward(pkg, 0, work=work)
    counts.append(cuts())
    assert (counts[1] - counts[0], counts[2] - counts[1]) == cut
    check_forward(torch, b, 0)
    check_backward(torch, b, 0, b.get(torch, "G"), b.get(torch, "U"))
    names = ("dX", "dWg", "dWu", "dWd")
    want = {n: b.get(torch, n) for n in ("dG", "dU", "Y") + names}
    kept = {n: getattr(b, n).view.clone() for n in "GUH"}
    for over in (None, "U", "G"):                 # the same bits again, and with deltaG over H, deltaU over U or G
        for n in names:
            getattr(b, n).view.fill_(float("nan"))
        b.backward(pkg, 0, work=work, over=over)
        assert torch.equal(b.get(torch, "H" if over else "dG"), want["dG"]) and torch.equal(b.get(torch, over or "dU"), want["dU"])
        for n in names:
            assert torch.equal(b.get(torch, n), want[n]), (over, n)
        for n in "GUH":
            getattr(b, n).view.copy_(kept[n])
    b.forward(pkg, 0, save=False, work=work)
    assert torch.equal(b.get(torch, "Y"), want["Y"])
    G.check_status(pkg)
