"""The Java_* exports of the transformer operators, through a fake JNIEnv with arrays of its own (slots of the JNI
specification's function table: GetArrayLength 171, GetLongArrayRegion 204)."""
import ctypes
from ctypes import CFUNCTYPE, POINTER, c_float, c_int32, c_int64, c_void_p

import pytest

import test_jni


class ArrayJNI(test_jni.FakeJNI):
    def __init__(self, arrays):
        super().__init__([0])
        self.arrays = arrays

        def length(env, arr):
            return len(self.arrays[arr])

        def region(env, arr, start, count, buf):
            for i in range(count):
                buf[i] = self.arrays[arr][start + i]

        for slot, proto, fn in ((171, CFUNCTYPE(c_int32, c_void_p, c_void_p), length),
                                (204, CFUNCTYPE(None, c_void_p, c_void_p, c_int32, c_int32, POINTER(c_int64)), region)):
            cb = proto(fn)
            self._keep.append(cb)
            self.table[slot] = ctypes.cast(cb, c_void_p).value

    def thrown_code(self):
        return next((e[3] for e in self.log if e[0] == "NewObjectA"), 0)


J, I, P = c_int64, c_int32, c_void_p
CLIP = [J, P, P, P, I, c_float, J, J, J]
FF = [P, I] + [J] * 10 + [I] * 4
FF_DELTA = [P, I] + [J] * 16 + [I] * 4
NORM = [J, J, J, J, I] + [J] * 6 + [I] * 3 + [c_float] * 3
NORM_DELTA = [J] + [J] * 5 + [I] + [J] * 10 + [J, I, I, I] + [c_float] * 2


def test_errors_become_exceptions(pkg):
    lib = pkg.cu32.load()
    clip = test_jni._fn(lib, "gradClip_gradClip", CLIP)
    A = 0x10000
    for arrays, args, code in (
            ({1: [A], 2: [A], 3: [4]}, (1, 2, 3, 2), -2),          # arrays shorter than the count
            ({1: [A], 2: [A], 3: [4]}, (1, 2, 3, 0), -2),
            ({1: [A], 2: [A], 3: [4]}, (0, 2, 3, 1), -1),          # a null array
            ({1: [A], 2: [A], 3: [-4]}, (1, 2, 3, 1), -2),
            ({1: [A + 2], 2: [A], 3: [4]}, (1, 2, 3, 1), -4)):
        jni = ArrayJNI(arrays)
        src, dst, sizes, count = args
        clip(jni.env, None, 0, src or None, dst, sizes, count, 1.0, A, A, 1 << 20)
        assert jni.thrown_code() == code and jni.thrown == 0x3333, args
    jni = ArrayJNI({9: [0]})
    ff = test_jni._fn(lib, "gatedFF_gatedFF", FF)
    ff(jni.env, None, 9, 1, A, A, A, A, 0, 0, A, A, 0, 0, 4, 8, 8, 9)
    assert jni.thrown_code() == -8
    jni = ArrayJNI({})
    norm = test_jni._fn(lib, "normResidual_normResidual", NORM)
    norm(jni.env, None, 0, A, 0, 0, 0, 0, A, A, A, 0, 0, 4, 8, 8, 1.0, 1.0, 1e-6)
    assert jni.thrown_code() == -1
    for name, args in (("gatedFF_work", (64, 64, 64)), ("normResidual_work", (64, 64, 0)), ("gradClip_work", (5,))):
        f = test_jni._fn(lib, name, [I] * len(args))
        f.restype = J
        assert f(None, None, *args) == getattr(lib, "cu32_" + name)(*args) > 0


@pytest.mark.gpu
def test_jni_calls_give_the_bits_of_the_c_calls(pkg, cuda):
    torch = cuda
    lib, cu = pkg.cu32.load(), pkg.cu32
    stream = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    rnd = lambda *s: torch.randn(s, device="cuda")  # noqa: E731
    N, D, F = 20, 68, 132
    jni = ArrayJNI({9: [stream]})
    X, Wg, Wu, Wd, dY = rnd(N, D), rnd(D, F), rnd(D, F), rnd(F, D), rnd(N, D)
    work = rnd(cu.Cuda_gatedFF.work(N, D, F) + 4)
    outs = []
    for java in (True, False):
        o = {n: torch.zeros(s, device="cuda") for n, s in (("G", (N, F)), ("U", (N, F)), ("H", (N, F)), ("Y", (N, D)),
             ("dG", (N, F)), ("dU", (N, F)), ("dX", (N, D)), ("dWg", (D, F)), ("dWu", (D, F)), ("dWd", (F, D)))}
        fwd = (p(X), p(Wg), p(Wu), p(Wd), p(o["G"]), p(o["U"]), p(o["H"]), p(o["Y"]), p(work), work.numel(), N, D, F, 0)
        bwd = (p(dY), p(X), p(Wg), p(Wu), p(Wd), p(o["G"]), p(o["U"]), p(o["H"]), p(o["dG"]), p(o["dU"]), p(o["dX"]), p(o["dWg"]),
               p(o["dWu"]), p(o["dWd"]), p(work), work.numel(), N, D, F, 0)
        if java:
            test_jni._fn(lib, "gatedFF_gatedFF", FF)(jni.env, None, 9, 1, *fwd)
            test_jni._fn(lib, "gatedFF_gatedFF_1delta", FF_DELTA)(jni.env, None, 9, 1, *bwd)
        else:
            cu.Cuda_gatedFF.gatedFF([stream], 1, *fwd)
            cu.Cuda_gatedFF.gatedFF_delta([stream], 1, *bwd)
        outs.append(o)
    torch.cuda.synchronize()
    assert jni.thrown is None and all(torch.equal(outs[0][n], outs[1][n]) and outs[0][n].abs().sum() > 0 for n in outs[0])
    outs = []
    B, R, gate, wpost, wpre, dR, dYn = rnd(N, D), rnd(N, D), rnd(2, D), rnd(D), rnd(D), rnd(N, D), rnd(N, D)
    nwork = rnd(cu.Cuda_normResidual.work(N, D, 10))
    for java in (True, False):
        o = {n: torch.zeros(s, device="cuda") for n, s in (("Ro", (N, D)), ("Y", (N, D)), ("a", (N,)), ("b", (N,)), ("dR", (N, D)),
             ("dB", (N, D)), ("dg", (2, D)), ("dpost", (D,)), ("dpre", (D,)))}
        fwd = (stream, p(B), p(R), p(gate), 10, p(wpost), p(wpre), p(o["Ro"]), p(o["Y"]), p(o["a"]), p(o["b"]), N, D, D - 1, 0.5,
               0.75, 1e-6)
        bwd = (stream, p(dR), p(dYn), p(B), p(o["Ro"]), p(gate), 10, p(wpost), p(wpre), p(o["a"]), p(o["b"]), p(o["dR"]), p(o["dB"]),
               p(o["dg"]), p(o["dpost"]), p(o["dpre"]), p(nwork), nwork.numel(), N, D, D - 1, 0.5, 0.75)
        if java:
            test_jni._fn(lib, "normResidual_normResidual", NORM)(jni.env, None, *fwd)
            test_jni._fn(lib, "normResidual_normResidual_1delta", NORM_DELTA)(jni.env, None, *bwd)
        else:
            cu.Cuda_normResidual.normResidual(*fwd)
            cu.Cuda_normResidual.normResidual_delta(*bwd)
        outs.append(o)
    torch.cuda.synchronize()
    assert jni.thrown is None and all(torch.equal(outs[0][n], outs[1][n]) and outs[0][n].abs().sum() > 0 for n in outs[0])
    grads = [rnd(1000), rnd(33)]
    dst = [[torch.zeros_like(t) for t in grads] for _ in range(2)]
    results = [torch.zeros(2, device="cuda") for _ in range(3)]
    cwork = torch.zeros(cu.Cuda_gradClip.work(2), device="cuda", dtype=torch.float64)
    src, sizes = [p(t) for t in grads], [t.numel() for t in grads]
    jni = ArrayJNI({1: src, 2: [p(t) for t in dst[0]], 3: sizes})
    test_jni._fn(lib, "gradClip_gradClip", CLIP)(jni.env, None, stream, 1, 2, 3, 2, 1.0, p(results[0]), p(cwork), cwork.numel())
    cu.Cuda_gradClip.gradClip(stream, src, [p(t) for t in dst[1]], sizes, 2, 1.0, p(results[1]), p(cwork), cwork.numel())
    test_jni._fn(lib, "gradClip_gradNorm", [J, P, P, I, J, J, J])(jni.env, None, stream, 1, 3, 2, p(results[2]), p(cwork), cwork.numel())
    torch.cuda.synchronize()
    assert jni.thrown is None and torch.equal(results[0], results[1]) and results[2][0] == results[0][0]
    assert all(torch.equal(a, b) and a.abs().sum() > 0 for a, b in zip(*dst))
