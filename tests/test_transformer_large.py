"""The transformer operators on arrays whose offsets pass 32 bits: bytes in the gated block (its extents end at 2^31
elements), elements in the norms and in clipping.  Rows at both ends and around the 2^31st and 2^32nd byte and element are
compared with the formula in 64 bits; the tolerances are those of the operators' own tests."""
import pytest

EPS = 2.0 ** -24


def rows_around(n, pitch):
    """The first and last rows and those where a 32-bit offset (bytes or elements) would wrap."""
    at = {0, 1, n - 2, n - 1}
    for wrap in (1 << 29, 1 << 30, 1 << 31, 1 << 32):
        at |= {wrap // pitch - 1, wrap // pitch, wrap // pitch + 1}
    return sorted(r for r in at if 0 <= r < n)


def randn_(t, g):
    for part in t.view(-1).split(1 << 28):
        part.normal_(generator=g)
    return t


@pytest.mark.gpu
def test_gated_block_beyond_4_gigabytes(pkg, cuda):
    import gpu_util as Gu
    torch = cuda
    N, D, F = 300011, 64, 3604                       # 1.08e9 hidden values, 4.3 GB
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    X, dY = randn_(new(N, D), g), randn_(new(N, D), g)
    Wg, Wu, Wd = randn_(new(D, F), g) / 8, randn_(new(D, F), g) / 8, randn_(new(F, D), g) / 60
    G, U, H, dG, Y, dX = new(N, F), new(N, F), new(N, F), new(N, F), new(N, D), new(N, D)
    ff = pkg.cu32.Cuda_gatedFF
    p = lambda t: t.data_ptr()  # noqa: E731
    ff.gatedFF([Gu.stream()], 1, p(X), p(Wg), p(Wu), p(Wd), p(G), p(U), p(H), p(Y), 0, 0, N, D, F, ff.SILU)
    at = torch.tensor(rows_around(N, F), device="cuda")
    g64, u64 = X[at].double() @ Wg.double(), X[at].double() @ Wu.double()

    def near(got, want):
        assert ((got.double() - want).norm() / want.norm()).item() <= 1e-6
    near(G[at], g64)
    near(U[at], u64)
    near(Y[at], H[at].double() @ Wd.double())
    gk, uk = G[at].double(), U[at].double()
    s = torch.sigmoid(gk)
    want = gk * s * uk
    assert ((H[at].double() - want).abs() <= 16 * EPS * want.abs() + 1e-37).all()
    ff.gatedFF_delta([Gu.stream()], 1, p(dY), p(X), p(Wg), p(Wu), p(Wd), p(G), p(U), 0, p(dG), p(U), p(dX), 0, 0, 0, 0, 0, N, D,
                     F, ff.SILU)
    dh = dY[at].double() @ Wd.double().T
    for got, factor in ((dG[at], uk * (s + gk * s * (1 - s))), (U[at], gk * s)):
        budget = 1e-6 * (dh.norm() / dh.numel() ** 0.5) * factor.norm() + 1e-6 * (dh * factor).norm()
        assert (got.double() - dh * factor).norm() <= budget
    near(dX[at], dG[at].double() @ Wg.double().T + U[at].double() @ Wu.double().T)
    Gu.check_status(pkg)


@pytest.mark.gpu
def test_norms_beyond_2_to_31_elements(pkg, cuda):
    import gpu_util as Gu
    torch = cuda
    N, M = 131099, 16384                             # 2.15e9 elements: just past 2^31
    g = torch.Generator(device="cuda").manual_seed(2)
    new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    B, R = randn_(new(N, M), g), randn_(new(N, M), g)
    w1, w2, gate = randn_(new(M), g), randn_(new(M), g), randn_(new(M), g)
    r1, r2 = new(N), new(N)
    at = torch.tensor(rows_around(N, M), device="cuda")
    b64, r64 = B[at].double(), R[at].double()
    nr = pkg.cu32.Cuda_normResidual
    p = lambda t: t.data_ptr()  # noqa: E731
    Y = new(N, M)
    nr.normResidual(Gu.stream(), p(B), p(R), p(gate), N, p(w1), p(w2), p(R), p(Y), p(r1), p(r2), N, M, M, 0.875, 0.5, 1e-6)

    def rstd(x):
        return torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6)
    term = 0.5 * gate.double() * w1.double() * b64 * rstd(b64)
    want = 0.875 * r64 + term
    assert ((R[at].double() - want).abs() <= 26 * EPS * ((0.875 * r64).abs() + term.abs())).all()
    rk = R[at].double()
    y = w2.double() * rk * rstd(rk)
    assert ((Y[at].double() - y).abs() <= 24 * EPS * y.abs()).all()

    # gradients: deltaY is what Y held; deltaR replaces it, deltaB replaces deltaRout
    dR = randn_(new(N, M), g)
    dy, dr = Y[at].double(), dR[at].double()
    work = new(nr.work(N, M, N))
    dg, d1, d2 = new(M), new(M), new(M)
    nr.normResidual_delta(Gu.stream(), p(dR), p(Y), p(B), p(R), p(gate), N, p(w1), p(w2), p(r1), p(r2), p(Y), p(dR), p(dg), p(d1),
                          p(d2), p(work), work.numel(), N, M, M, 0.875, 0.5)
    s2 = rstd(rk)
    a = dy * w2.double()
    c2 = (a * rk).mean(1, keepdim=True) * s2 ** 3
    t = dr + a * s2 - rk * c2
    t_size = dr.abs() + (a * s2).abs() + (rk * (a * rk).abs().mean(1, keepdim=True) * s2 ** 3).abs()
    assert ((Y[at].double() - 0.875 * t).abs() <= 64 * EPS * 0.875 * t_size).all()
    s1 = rstd(b64)
    q = t * 0.5 * gate.double() * w1.double()
    q_size = t_size * (0.5 * gate.double() * w1.double()).abs()
    want = q * s1 - b64 * (q * b64).mean(1, keepdim=True) * s1 ** 3
    size = q_size * s1 + b64.abs() * (q_size * b64.abs()).mean(1, keepdim=True) * s1 ** 3
    assert ((dR[at].double() - want).abs() <= 2 * 64 * EPS * size).all()
    assert torch.isfinite(dg).all() and torch.isfinite(d1).all() and torch.isfinite(d2).all()
    Gu.check_status(pkg)


@pytest.mark.gpu
def test_clipping_beyond_2_to_32_elements(pkg, cuda):
    import gpu_util as Gu
    from array import array
    torch = cuda
    n = (1 << 32) + 5                                # 17.2 GB
    t = torch.full((n + 4,), 0.5, device="cuda")
    t[0], t[n - 1], t[(1 << 32) + 1], t[1 << 31] = 3.0, -5.0, 7.0, 9.0
    clip = pkg.cu32.Cuda_gradClip
    work = torch.empty(clip.work(1), device="cuda", dtype=torch.float64)
    result = torch.empty(2, device="cuda")
    a, z = array("q", [t.data_ptr()]), array("q", [n])
    clip.gradClip(Gu.stream(), a, a, z, 1, 1.0, result.data_ptr(), work.data_ptr(), work.numel())
    norm = ((n - 4) * 0.25 + 9 + 25 + 49 + 81) ** 0.5    # squares and sums of halves: exact in 64 bits
    got = result.double().cpu().tolist()
    assert abs(got[0] - norm) <= 2 * EPS * norm and abs(got[1] - 1 / norm) <= 2 * EPS / norm
    f = got[1]
    want = [3 * f, 0.5 * f, 9 * f, 7 * f, -5 * f]
    at = [0, 1, 1 << 31, (1 << 32) + 1, n - 1]
    for i, w in zip(at, want):
        assert abs(t[i].item() - w) <= EPS * abs(w), i
    assert (t[n:] == 0.5).all()
    lo, hi = t[1:1 << 31].aminmax()
    assert lo == hi == t[1]
