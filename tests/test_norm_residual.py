"""Norms before and after a block with its gate and residual scale (cu32_normResidual, cu32_normResidual_delta).

P = w_post B / rms(B), R' = rs R + s gate P, Y = w_pre R' / rms(R').  Tolerances, elementwise, in roundings of 2^-24 of the
terms a result is made of (T = the sum of their sizes):
  - a row sum of n squares: 16 additions in a thread, 5 in a warp, 5 over the warps: 26 roundings, 13 after the root; the
    root, the mean's factor, the reciprocal and the products add less than 11: 24 for P and for Y (of the stored R');
    R' itself: 24 for its P term, 3 for the others - 26 of T.
  - gradients: the three row sums carry 26 + 8 roundings of the sum of their terms' sizes, what is built from them less
    than 30 more: 64 of T, where T has every term by its size (sums by the sums of sizes).
  - column sums: a chain of additions of at most N + 100 terms, each term good to 64: (N + 164) of the sum of sizes.
"""
import pytest

EPS = 2.0 ** -24


def pad4(x):
    return (x + 3) // 4 * 4


class Case:
    def __init__(self, torch, N, width, gate_rows, post, seed, pad=0, drout=True):
        import gpu_util as G
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.N, self.width, self.M, self.gate_rows, self.post = N, width, pad4(width) + pad, gate_rows, post
        M = self.M

        def rows(n, scale=1.0, shift=0.0):       # the padding columns hold what nobody may read
            t = torch.full((n, M), float("nan"), device="cuda")
            t[:, :width] = scale * torch.randn((n, width), device="cuda", generator=g) + shift
            return t
        self.groups = -(-N // gate_rows) if gate_rows else 0
        self.B, self.R = rows(N, 0.5), rows(N, 2.0)
        self.B[:, 0] *= 30.0
        self.wpre, self.wpost = rows(1, 0.3, 1.0), rows(1, 0.3, 1.0) if post else None
        self.gate = rows(self.groups, 0.7) if gate_rows else None
        self.dRout, self.dY = rows(N) if drout else None, rows(N)
        self.rs, self.s, self.eps = 0.875, 0.6, 1e-6
        out = lambda n: G.Out(n * M)  # noqa: E731
        self.Rout, self.Y, self.dR, self.dB = out(N), out(N), out(N), out(N)
        self.rstd_post, self.rstd_pre = G.Out(N), G.Out(N)
        self.dgate = out(self.groups) if gate_rows else None
        self.dwpost, self.dwpre = out(1) if post else None, out(1)

    def forward(self, pkg, stream=None):
        import gpu_util as G
        p = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
        pkg.cu32.Cuda_normResidual.normResidual(
            stream or G.stream(), p(self.B), p(self.R), p(self.gate), self.gate_rows, p(self.wpost), p(self.wpre),
            self.Rout.ptr, self.Y.ptr, self.rstd_post.ptr, self.rstd_pre.ptr, self.N, self.M, self.width, self.rs, self.s,
            self.eps)

    def backward(self, pkg, work, stream=None):
        import gpu_util as G
        p = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
        o = lambda t: t.ptr if t is not None else 0  # noqa: E731
        pkg.cu32.Cuda_normResidual.normResidual_delta(
            stream or G.stream(), p(self.dRout), p(self.dY), p(self.B), self.Rout.ptr, p(self.gate), self.gate_rows,
            p(self.wpost), p(self.wpre), self.rstd_post.ptr, self.rstd_pre.ptr, self.dR.ptr, self.dB.ptr, o(self.dgate),
            o(self.dwpost), o(self.dwpre), work.data_ptr(), work.numel(), self.N, self.M, self.width, self.rs, self.s)

    def scratch(self, torch, pkg):
        n = pkg.cu32.Cuda_normResidual.work(self.N, self.M, self.gate_rows)
        return torch.full((n,), float("nan"), device="cuda")

    def out(self, torch, name):
        o = getattr(self, name)
        if name.startswith("rstd"):
            return torch.as_tensor(o.host((self.N,))).cuda()
        full = torch.as_tensor(o.host((-1, self.M))).cuda()
        assert (full[:, self.width:] == 0).all(), name
        return full[:, :self.width].double()

    def gate64(self, torch):
        if self.gate is None:
            return torch.ones((self.N, self.width), device="cuda", dtype=torch.float64)
        return self.gate[:, :self.width].double().repeat_interleave(self.gate_rows, 0)[:self.N]


def check_forward(torch, c):
    w = c.width
    B, R, g = c.B[:, :w].double(), c.R[:, :w].double(), c.gate64(torch)
    P = B
    if c.post:
        rb = 1 / torch.sqrt((B * B).mean(1, keepdim=True) + c.eps)
        P = B * rb * c.wpost[:, :w].double()
        assert ((c.out(torch, "rstd_post").double() - rb[:, 0]).abs() <= 20 * EPS * rb[:, 0]).all()
    Rout = c.out(torch, "Rout")
    a, b = c.rs * R, c.s * g * P
    assert ((Rout - (a + b)).abs() <= 26 * EPS * (a.abs() + b.abs())).all()
    rr = 1 / torch.sqrt((Rout * Rout).mean(1, keepdim=True) + c.eps)
    assert ((c.out(torch, "rstd_pre").double() - rr[:, 0]).abs() <= 20 * EPS * rr[:, 0]).all()
    Y = Rout * rr * c.wpre[:, :w].double()
    assert ((c.out(torch, "Y") - Y).abs() <= 24 * EPS * Y.abs() + 1e-44).all()


def check_backward(torch, c):
    w = c.width
    mean = lambda x: x.mean(1, keepdim=True)  # noqa: E731
    B, Rout, g = c.B[:, :w].double(), c.out(torch, "Rout"), c.gate64(torch)
    dY = c.dY[:, :w].double()
    dRo = c.dRout[:, :w].double() if c.dRout is not None else torch.zeros_like(dY)
    wpre = c.wpre[:, :w].double()
    wpost = c.wpost[:, :w].double() if c.post else torch.ones_like(wpre)
    rr = 1 / torch.sqrt(mean(Rout * Rout) + c.eps)
    rh, q = Rout * rr, dY * wpre
    dT = dRo + rr * (q - rh * mean(q * rh))
    T = dRo.abs() + rr * (q.abs() + rh.abs() * mean((q * rh).abs()))
    rb = 1 / torch.sqrt(mean(B * B) + c.eps) if c.post else torch.ones_like(rr)
    bh = B * rb
    dP, TP = c.s * g * dT, c.s * g.abs() * T
    if c.post:
        dB = rb * (dP * wpost - bh * mean(dP * wpost * bh))
        # c2 is the difference of two sums; their terms by size, c1's size among them
        e = (c.s * g * wpost * bh).abs()
        c2 = mean(e * (dRo.abs() + rr * q.abs())) + mean((q * rh).abs()) * mean(e * rr * rh.abs())
        TB = rb * (TP * wpost.abs() + bh.abs() * c2)
    else:
        dB, TB = dP, TP
    assert ((c.out(torch, "dR") - c.rs * dT).abs() <= 64 * EPS * c.rs * T + 1e-44).all()
    assert ((c.out(torch, "dB") - dB).abs() <= 64 * EPS * TB + 1e-44).all()
    n = (c.N + 164) * EPS
    near = lambda got, want, size: ((got - want).abs() <= n * size + 1e-44).all()  # noqa: E731
    assert near(c.out(torch, "dwpre")[0], (dY * rh).sum(0), (dY * rh).abs().sum(0))
    if c.post:
        assert near(c.out(torch, "dwpost")[0], (dP * bh).sum(0), (TP * bh.abs()).sum(0))
    if c.gate is not None:
        t, size = c.s * bh * wpost * dT, c.s * (bh * wpost).abs() * T
        for k in range(c.groups):
            rows = slice(k * c.gate_rows, (k + 1) * c.gate_rows)
            assert near(c.out(torch, "dgate")[k], t[rows].sum(0), size[rows].sum(0)), k


# ---------------------------------------------------------------------------------------------------- without a GPU
def test_norm_residual_refusals(pkg):
    lib = pkg.cu32.load()
    P = 0x10000

    def fwd(B=P, R=P, gate=0, gate_rows=0, wpost=P, wpre=P, Rout=P, Y=P, rpost=P, rpre=P, N=4, M=8, width=7, eps=1e-6):
        return lib.cu32_normResidual(0, B, R, gate, gate_rows, wpost, wpre, Rout, Y, rpost, rpre, N, M, width, 1.0, 1.0, eps)

    def bwd(dRout=P, dY=P, B=P, Rout=P, gate=P, gate_rows=2, wpost=P, wpre=P, rpost=P, rpre=P, dR=P, dB=P, dgate=P, dwpost=P,
            dwpre=P, work=P, room=1 << 20, N=4, M=8, width=7):
        return lib.cu32_normResidual_delta(0, dRout, dY, B, Rout, gate, gate_rows, wpost, wpre, rpost, rpre, dR, dB, dgate,
                                           dwpost, dwpre, work, room, N, M, width, 1.0, 1.0)
    for call in (fwd, bwd):
        for kw in ({"N": 0}, {"N": -1}, {"M": 0}, {"width": 0}, {"width": 9}, {"M": 16388, "width": 5}, {"gate_rows": -1},
                   {"gate": P, "gate_rows": 0}, {"N": 1 << 30}):
            assert call(**kw) == -2, kw
        assert call(M=6, width=5) == -4
    assert fwd(eps=-1e-6) == -8 and fwd(eps=float("nan")) == -8
    for name in ("B", "R", "wpre", "Rout", "Y"):
        assert fwd(**{name: 0}) == -1 and fwd(**{name: P + 4}) == -4
    assert fwd(gate=P + 4, gate_rows=1) == -4 and fwd(wpost=P + 8) == -4
    for name in ("dY", "B", "Rout", "wpre", "rpre", "dR", "dB", "dwpre", "work"):
        assert bwd(**{name: 0}) == -1
    assert bwd(rpost=0) == -1 and bwd(dwpost=0) == -1 and bwd(dgate=0) == -1
    for name in ("dRout", "dY", "B", "Rout", "gate", "wpost", "wpre", "dR", "dB", "dgate", "dwpost", "dwpre", "work"):
        assert bwd(**{name: P + 4}) == -4
    assert bwd(room=23) == -9
    with pytest.raises(pkg.cu32.CudaException, match="CU32_E_DIM"):
        pkg.cu32.Cuda_normResidual.normResidual(0, P, P, 0, 0, P, P, P, P, 0, 0, 0, 8, 8, 1.0, 1.0, 1e-6)


def test_norm_blocks_are_resident(pkg):
    """The gradients' scratch has a row per block; there are no more of them than an SM holds at a time: 96 registers a thread,
    so 5 warps in each of its four parts, and 228 KB of shared memory for rings of three rows, 1664 bytes and 1 KB a block."""
    import torch
    sms = torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 1
    for M in range(4, 4097, 4):
        units = pkg.cu32.Cuda_normResidual.work(1 << 28, M, 0) // (3 * M)
        warps = ((M // 4 + 1) // 2 + 31) // 32
        ring = 3 * ((M * 16 + 127) // 128 * 128)
        fits = min(20 // warps, 228 * 1024 // (ring + 1664 + 1024))
        assert 1 <= units / sms <= fits, M


# ---------------------------------------------------------------------------------------------------- on the GPU
WIDTHS = [1, 3, 4, 31, 127, 128, 129, 513, 1000, 1024, 2051, 4096, 4099, 8192, 8195, 16381, 16384]


@pytest.mark.gpu
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_widths(pkg, cuda, width):
    torch = cuda
    for k, (N, gate_rows, post) in enumerate([(1, 1, True), (2, 0, True), (7, 3, False), (33, 33, True), (400, 150, True)]):
        c = Case(torch, N, width, gate_rows, post, seed=width + k, pad=4 * (k % 2) if width < 16000 else 0)
        work = c.scratch(torch, pkg)
        c.forward(pkg)
        check_forward(torch, c)
        c.backward(pkg, work)
        check_backward(torch, c)


@pytest.mark.gpu
@pytest.mark.parametrize("gate_rows", [0, 1, 2, 5, 16, 299, 300, 599, 600, 10000])
def test_norm_gate_groups(pkg, cuda, gate_rows):
    """Every way the rows of a gate row are shared among blocks: whole groups in a block, groups cut into chunks, one group."""
    torch = cuda
    for post in (False, True):
        for drout in (False, True):
            c = Case(torch, 600, 68, gate_rows, post, seed=gate_rows, drout=drout)
            c.forward(pkg)
            check_forward(torch, c)
            c.backward(pkg, c.scratch(torch, pkg))
            check_backward(torch, c)


@pytest.mark.gpu
def test_norm_with_little_scratch_and_repeats(pkg, cuda):
    """Fewer units with less scratch, down to one; the same scratch gives the same bits."""
    torch = cuda
    c = Case(torch, 500, 260, 90, True, seed=2)
    c.forward(pkg)
    names = ("dR", "dB", "dgate", "dwpost", "dwpre")
    for units in (1, 2, 5, 6, 7, 40):
        work = torch.full((units * 3 * c.M,), float("nan"), device="cuda")
        kept = None
        for _ in range(2):
            for n in names:
                getattr(c, n).view.fill_(float("nan"))
            c.backward(pkg, work)
            check_backward(torch, c)
            now = [c.out(torch, n) for n in names]
            assert kept is None or all(torch.equal(a, b) for a, b in zip(now, kept))
            kept = now


@pytest.mark.gpu
def test_norm_in_place(pkg, cuda):
    """R' over R, Y over B; deltaR over deltaR', deltaB over deltaY."""
    import gpu_util as G
    torch = cuda
    c = Case(torch, 37, 516, 10, True, seed=4)
    work = c.scratch(torch, pkg)
    c.forward(pkg)
    c.backward(pkg, work)
    want = {n: c.out(torch, n) for n in ("Rout", "Y", "dR", "dB", "dgate", "dwpre")}
    B, R = c.B.clone(), c.R.clone()
    p = lambda t: t.data_ptr()  # noqa: E731
    pkg.cu32.Cuda_normResidual.normResidual(G.stream(), p(B), p(R), p(c.gate), 10, p(c.wpost), p(c.wpre), p(R), p(B), 0, 0,
                                            c.N, c.M, c.width, c.rs, c.s, c.eps)
    assert torch.equal(R[:, :c.width].double(), want["Rout"]) and torch.equal(B[:, :c.width].double(), want["Y"])
    dRout, dY = c.dRout.clone(), c.dY.clone()
    pkg.cu32.Cuda_normResidual.normResidual_delta(
        G.stream(), p(dRout), p(dY), p(c.B), c.Rout.ptr, p(c.gate), 10, p(c.wpost), p(c.wpre), c.rstd_post.ptr, c.rstd_pre.ptr,
        p(dRout), p(dY), c.dgate.ptr, c.dwpost.ptr, c.dwpre.ptr, p(work), work.numel(), c.N, c.M, c.width, c.rs, c.s)
    assert torch.equal(dRout[:, :c.width].double(), want["dR"]) and torch.equal(dY[:, :c.width].double(), want["dB"])
    assert torch.equal(c.out(torch, "dgate"), want["dgate"]) and torch.equal(c.out(torch, "dwpre"), want["dwpre"])


@pytest.mark.gpu
def test_norm_zero_rows_and_bad_rows(pkg, cuda):
    """A row of zeros divides by sqrt(eps); a NaN or an infinity stays in its row (and in the column sums)."""
    torch = cuda
    c = Case(torch, 20, 132, 20, True, seed=6)
    c.B[3] = 0
    c.R[3] = 0
    c.forward(pkg)
    check_forward(torch, c)
    assert (c.out(torch, "Y")[3] == 0).all()
    c.backward(pkg, c.scratch(torch, pkg))
    check_backward(torch, c)
    clean = c.out(torch, "Y"), c.out(torch, "dR")
    c.B[5, 7] = float("nan")
    c.R[9, 1] = float("inf")
    c.forward(pkg)
    c.backward(pkg, c.scratch(torch, pkg))
    Y, dR = c.out(torch, "Y"), c.out(torch, "dR")
    others = [i for i in range(20) if i not in (5, 9)]
    assert torch.equal(Y[others], clean[0][others]) and torch.equal(dR[others], clean[1][others])
    assert torch.isnan(Y[5]).all() and torch.isnan(Y[9, 1])


@pytest.mark.gpu
def test_norm_gradients_against_differences(pkg, cuda):
    """The formulas against central differences of sum(R' deltaR') + sum(Y deltaY) in 64 bits."""
    torch = cuda
    c = Case(torch, 6, 22, 3, True, seed=7)
    c.forward(pkg)
    c.backward(pkg, c.scratch(torch, pkg))
    w = c.width
    ops = {"B": c.B[:, :w].double(), "R": c.R[:, :w].double(), "wpre": c.wpre[:, :w].double(),
           "wpost": c.wpost[:, :w].double(), "gate": c.gate[:, :w].double()}

    def value(o):
        unit = lambda x: x / torch.sqrt((x * x).mean(1, keepdim=True) + c.eps)  # noqa: E731
        Rout = c.rs * o["R"] + c.s * o["gate"].repeat_interleave(3, 0) * unit(o["B"]) * o["wpost"]
        return (Rout * c.dRout[:, :w].double()).sum() + (unit(Rout) * o["wpre"] * c.dY[:, :w].double()).sum()
    for n in ops:
        got = c.out(torch, "d" + n)
        for at in ((0, 0), (got.shape[0] - 1, w - 1), (got.shape[0] // 2, 11)):
            hi, lo = dict(ops), dict(ops)
            hi[n], lo[n] = ops[n].clone(), ops[n].clone()
            hi[n][at] += 1e-5
            lo[n][at] -= 1e-5
            diff = ((value(hi) - value(lo)) / 2e-5).item()
            # FP32 results of sums of some ten terms of size one: 1e-5; the difference itself: 1e-8
            assert abs(got[at].item() - diff) <= 1e-5 * (1 + abs(diff)), (n, at)


@pytest.mark.gpu
def test_norm_in_a_graph_and_on_two_streams(pkg, cuda):
    torch = cuda
    cases = [Case(torch, n, 260, 0, True, seed=n) for n in (3, 700)]
    works = [c.scratch(torch, pkg) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, w, s in zip(cases, works, streams):
            c.forward(pkg, s.cuda_stream)
            c.backward(pkg, w, s.cuda_stream)
    torch.cuda.synchronize()
    for c in cases:
        check_forward(torch, c)
        check_backward(torch, c)
    c, w = cases[1], works[1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.forward(pkg)
        c.backward(pkg, w)
    c.B[:, :c.width].mul_(0.5)
    c.dY[:, :c.width].add_(1.0)
    graph.replay()
    torch.cuda.synchronize()
    check_forward(torch, c)
    check_backward(torch, c)
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("N", [20, 700])
@pytest.mark.parametrize("width", [130, 4097])
@pytest.mark.parametrize("gate_rows", [1, 9, 700])
def test_norm_padding_is_zero_beside_bad_rows(pkg, cuda, N, width, gate_rows):
    """Columns >= width of every output are zeros also where the row's sums are NaN or infinite (out() looks at them)."""
    torch = cuda
    c = Case(torch, N, width, gate_rows, True, seed=61, pad=4)
    work = c.scratch(torch, pkg)
    c.forward(pkg)
    c.backward(pkg, work)
    clean = {n: c.out(torch, n) for n in ("Rout", "Y", "dR", "dB")}
    c.B[5, 7] = float("nan")
    c.R[9, 1] = float("inf")
    c.dY[12, 3] = float("-inf")
    c.forward(pkg)
    c.backward(pkg, work)
    others = [i for i in range(N) if i not in (5, 9, 12)]
    for n, was in clean.items():
        now = c.out(torch, n)
        assert torch.equal(now[others], was[others]), n
    for n in ("dgate", "dwpost", "dwpre"):
        c.out(torch, n)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3000, 5000, 0), (3000, 2052, 300), (1200, 10000, 75), (20000, 260, 1700), (9000, 1536, 2500),
                                   (700, 16384, 70)], ids=str)
def test_norm_many_rows_per_block(pkg, cuda, shape):
    """Rings that go round many times: single blocks, clusters of two and four, two clusters to an SM."""
    torch = cuda
    N, width, gate_rows = shape
    c = Case(torch, N, width, gate_rows, True, seed=62)
    c.forward(pkg)
    check_forward(torch, c)
    c.backward(pkg, c.scratch(torch, pkg))
    check_backward(torch, c)
