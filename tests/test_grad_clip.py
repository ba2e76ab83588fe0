"""Global gradient norm and clipping (cu32_gradNorm, cu32_gradClip).

Squares are exact in 64 bits and their sum is off by far less than 2^-24, so the norm and the factor are one rounding to
FP32 off (2^-24 relative, a little more for the sum's own error), a clipped gradient two (the factor's and the product's).
"""
import math
from array import array

import pytest

EPS = 2.0 ** -24


def run(pkg, torch, grads, outs, max_norm, stream=None):
    import gpu_util as G
    gc = pkg.cu32.Cuda_gradClip
    n = len(grads)
    work = torch.full((gc.work(n),), float("nan"), device="cuda", dtype=torch.float64)
    result = torch.full((2,), -1.0, device="cuda")
    gc.gradClip(stream if stream is not None else G.stream(), [t.data_ptr() for t in grads], [t.data_ptr() for t in outs],
                [t.numel() for t in grads], n, max_norm, result.data_ptr(), work.data_ptr(), work.numel())
    torch.cuda.synchronize()
    return result.tolist()


def norm64(grads):
    return math.sqrt(math.fsum(float((t.double() ** 2).sum().item()) for t in grads))


def check(torch, result, before, outs, max_norm):
    norm = norm64(before)
    assert abs(result[0] - norm) <= 1.01 * EPS * norm
    factor = min(1.0, max_norm / norm) if norm > 0 else 1.0
    assert abs(result[1] - factor) <= 1.01 * EPS * factor
    for g, o in zip(before, outs):
        want = g.double() * factor
        if factor == 1.0:
            assert torch.equal(o, g)
        else:
            assert ((o.double() - want).abs() <= 2.1 * EPS * want.abs() + 1e-45).all()


# ---------------------------------------------------------------------------------------------------- without a GPU
def test_grad_clip_refusals(pkg):
    lib = pkg.cu32.load()
    P = 0x10000
    addr = lambda a: a.buffer_info()[0]  # noqa: E731
    src, dst, sizes = array("q", [P, P + 4096]), array("q", [P, P + 4096]), array("q", [8, 0])

    def clip(src=addr(src), dst=addr(dst), sizes=addr(sizes), count=2, max_norm=1.0, result=P, work=P, room=1 << 20):
        return lib.cu32_gradClip(0, src, dst, sizes, count, max_norm, result, work, room)
    for name in ("src", "dst", "sizes", "result", "work"):
        assert clip(**{name: 0}) == -1
    assert clip(count=0) == -2 and clip(count=-1) == -2
    assert clip(max_norm=-1.0) == -8 and clip(max_norm=float("nan")) == -8
    assert clip(work=P + 4) == -4 and clip(result=P + 2) == -4
    assert clip(room=0) == -9
    bad = array("q", [-1, 4])
    assert clip(sizes=addr(bad)) == -2
    null = array("q", [0, P])
    assert clip(src=addr(null)) == -1 and clip(dst=addr(null)) == -1
    odd = array("q", [P + 2, P])
    assert clip(src=addr(odd)) == -4 and clip(dst=addr(odd)) == -4
    assert lib.cu32_gradNorm(0, 0, addr(sizes), 2, P, P, 1 << 20) == -1
    with pytest.raises(ValueError):
        pkg.cu32.Cuda_gradClip.gradClip(0, [P], [P], [4], 2, 1.0, P, P, 1 << 20)
    with pytest.raises(pkg.cu32.CudaException, match="CU32_E_SCRATCH"):
        pkg.cu32.Cuda_gradClip.gradClip(0, [P], [P], [4], 1, 1.0, P, P, 1)


# ---------------------------------------------------------------------------------------------------- on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1], [3], [4], [5, 0, 1], [8191], [8192], [8193, 7], [100003, 1, 2, 3, 65536],
                                   list(range(1, 65)), list(range(0, 130)), [17] * 2100], ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("limit", [0.5, 2.0], ids=["clipped", "below"])
def test_clip_out_of_place_and_in_place(pkg, cuda, sizes, limit):
    import gpu_util as G
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(sum(sizes))
    grads = [torch.randn(n, device="cuda", generator=g) * 10.0 ** (i % 5 - 2) for i, n in enumerate(sizes)]
    max_norm = limit * norm64(grads)
    outs = [G.Out(n) for n in sizes] if len(sizes) < 200 else None
    got = [o.view for o in outs] if outs else [torch.empty_like(t) for t in grads]
    result = run(pkg, torch, grads, got, max_norm)
    check(torch, result, grads, got, max_norm)
    if outs:
        for o in outs:
            o.host((o.n,))      # canaries
    again = run(pkg, torch, grads, got, max_norm)
    assert again == result
    copies = [t.clone() for t in grads]
    assert run(pkg, torch, copies, copies, max_norm) == result
    for a, b in zip(copies, got):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("src_off", range(4))
@pytest.mark.parametrize("dst_off", range(4))
def test_clip_at_every_alignment(pkg, cuda, src_off, dst_off):
    torch = cuda
    for n in (1, 2, 6, 8190, 20001):
        src = torch.randn(n + 8, device="cuda")
        dst = torch.full((n + 8,), 7.0, device="cuda")
        a, b = src[src_off:src_off + n], dst[dst_off:dst_off + n]
        max_norm = 0.25 * norm64([a])
        check(torch, run(pkg, torch, [a], [b], max_norm), [a], [b], max_norm)
        assert (dst[:dst_off] == 7.0).all() and (dst[dst_off + n:] == 7.0).all()


@pytest.mark.gpu
def test_norm_alone_and_extreme_values(pkg, cuda):
    import gpu_util as G
    torch = cuda
    gc = pkg.cu32.Cuda_gradClip
    for scale in (1e-30, 1.0, 1e30):       # squares far outside FP32
        grads = [torch.randn(n, device="cuda") * scale for n in (4099, 12, 70000)]
        keep = [t.clone() for t in grads]
        work = torch.empty(gc.work(3), device="cuda", dtype=torch.float64)
        result = torch.zeros(2, device="cuda")
        gc.gradNorm(G.stream(), [t.data_ptr() for t in grads], [t.numel() for t in grads], 3, result.data_ptr(),
                    work.data_ptr(), work.numel())
        norm = norm64(grads)
        assert abs(result[0].item() - norm) <= 1.01 * EPS * norm and result[1].item() == 1.0
        assert all(torch.equal(a, b) for a, b in zip(grads, keep))
        check(torch, run(pkg, torch, grads, grads, 0.5 * norm), keep, grads, 0.5 * norm)


@pytest.mark.gpu
def test_not_finite_zero_and_empty(pkg, cuda):
    torch = cuda
    for bad in (float("inf"), float("-inf"), float("nan")):
        grads = [torch.randn(1000, device="cuda"), torch.randn(9000, device="cuda")]
        grads[1][8999] = bad
        outs = [torch.zeros_like(t) for t in grads]
        result = run(pkg, torch, grads, outs, 0.1)
        assert not math.isfinite(result[0]) and result[1] == 1.0
        assert all(torch.equal(a.view(torch.int32), b.view(torch.int32)) for a, b in zip(grads, outs))
    zero = [torch.zeros(100, device="cuda")]
    assert run(pkg, torch, zero, zero, 1.0) == [0.0, 1.0]
    assert run(pkg, torch, zero, zero, 0.0) == [0.0, 1.0]
    empty = [torch.zeros(0, device="cuda")] * 3
    assert run(pkg, torch, empty, empty, 1.0) == [0.0, 1.0]
    some = [torch.randn(50, device="cuda")]
    assert run(pkg, torch, some, some, float("inf"))[1] == 1.0
    out = [torch.full((50,), 3.0, device="cuda")]
    assert run(pkg, torch, some, out, 0.0)[1] == 0.0 and (out[0] == 0).all()


@pytest.mark.gpu
def test_clip_in_a_graph_and_beside_another(pkg, cuda):
    """Captured with its addresses, replayed on new gradients; two clips on two streams with scratch of their own."""
    torch = cuda
    gc = pkg.cu32.Cuda_gradClip
    sets = [[torch.randn(n, device="cuda") for n in (30011, 5, 4096)] for _ in range(2)]
    keep = [[t.clone() for t in s] for s in sets]
    works = [torch.empty(gc.work(3), device="cuda", dtype=torch.float64) for _ in sets]
    results = [torch.zeros(2, device="cuda") for _ in sets]

    def call(i, stream):
        p = [t.data_ptr() for t in sets[i]]
        gc.gradClip(stream, p, p, [t.numel() for t in sets[i]], 3, 1.0, results[i].data_ptr(), works[i].data_ptr(), works[i].numel())
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        call(i, s.cuda_stream)
    torch.cuda.synchronize()
    for i in range(2):
        check(torch, results[i].tolist(), keep[i], sets[i], 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0, torch.cuda.current_stream().cuda_stream)
    for factor in (3.0, 0.001):
        for t, k in zip(sets[0], keep[0]):
            t.copy_(k * factor)
        before = [t.clone() for t in sets[0]]
        graph.replay()
        torch.cuda.synchronize()
        check(torch, results[0].tolist(), before, sets[0], 1.0)
    del graph


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2e36, 3e38], ids=str)
@pytest.mark.parametrize("max_norm", [1.0, 1e-12, 1e30])
@pytest.mark.parametrize("sizes", [[4099, 12, 7], [8000003], [3] * 1500], ids=lambda s: f"{len(s)}x{sum(s)}")
def test_norms_and_factors_beyond_the_range_of_fp32(pkg, cuda, size, max_norm, sizes):
    """Finite gradients whose norm, or whose factor, FP32 cannot hold: scaled as the formula says, one rounding off (two
    where the factor is an FP32 number); the norm comes out as FP32 rounds it, infinite beyond its range."""
    torch = cuda
    g = torch.Generator(device="cuda").manual_seed(len(sizes))
    grads = [size * (2 * torch.rand(n, device="cuda", generator=g) - 1) for n in sizes]
    norm = norm64(grads)
    factor = torch.tensor(max_norm, dtype=torch.float32).double().item() / norm      # the limit is an FP32 argument
    for outs in ([torch.full_like(t, 7.0) for t in grads], [t.clone() for t in grads]):
        in_place = torch.equal(outs[0], grads[0])
        src = outs if in_place else grads
        got_norm, got_factor = run(pkg, torch, src, outs, max_norm)
        assert got_norm == math.inf if norm > 3.4028236e38 else abs(got_norm - norm) <= 1.01 * EPS * norm
        assert abs(got_factor - factor) <= 1.01 * EPS * factor + 1e-45 and got_factor < 1.0
        for a, o in zip(grads, outs):
            want = a.double() * factor
            assert ((o.double() - want).abs() <= 2.1 * EPS * want.abs() + 1e-45).all()
