"""GPU tests of the 8-bit activation path at its edges: ties of the quantisation, long rows, scales and gates at the ends
of their range, clusters of every size, slow predecessors.

Tolerances count roundings.  U = 2^-24 is half a step of fp32 relative to the value.
"""
import pytest
import torch

from mixed_gemv_b200 import _lib, api
from tests.test_gpu_int8_path import ACTS, U, Product, _check_quantised, _gen, _norm_reference

pytestmark = pytest.mark.gpu


# ---- ties of the quantisation -------------------------------------------------------------------

def _quotient(y):
    """y * 127 / max|y| of rows of up to 24-bit values.  The product has 31 bits, so it is exact; a tie, which has eight, is
    a number that the division returns exactly, and any other quotient of such numbers is further from a tie than it errs."""
    return y * 127 / y.abs().amax(dim=1, keepdim=True)


def _ties(quotient):
    twice = quotient * 2
    return (twice == twice.round()) & (twice.round() % 2 != 0)


# rows to a warp, one and two and four pieces a thread, value by value in registers, in two passes
TIE_SHAPES = [(1500, 256), (3, 4096), (400, 4096), (3, 11008), (400, 11008), (300, 1031), (5, 5001), (400, 5001), (2, 70000), (2, 65536)]


def _tie_rows(M, K, dtype, kind, seed):
    g = _gen(seed)
    if kind == "normal":
        return torch.randn(M, K, generator=g, device="cuda").to(dtype)
    # a grid of up to 122 steps to a row's largest value, an even number of steps: half of it is a tie
    top = torch.randint(23, 62, (M, 1), generator=g, device="cuda") * 2
    x = (torch.rand(M, K, generator=g, device="cuda") * 2 - 1).mul(top).round()
    x[:, K // 2 : K // 2 + 1] = top
    x[:, K - 1:] = -top / 2
    return (x * (2.0 ** -120 if kind == "tiny grid" else 1)).to(dtype)  # tiny: statistics below fp32's, rows done in double precision


@pytest.mark.parametrize("dtype, kind", [(torch.float16, "normal"), (torch.bfloat16, "normal"), (torch.float16, "grid"),
                                         (torch.bfloat16, "grid"), (torch.bfloat16, "tiny grid")])
@pytest.mark.parametrize("M, K", TIE_SHAPES)
def test_ties_go_to_the_even_integer(cuda_lib, M, K, dtype, kind):
    x = _tie_rows(M, K, dtype, kind, seed=K)
    q, s = torch.full((M, K), 99, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    api.RowQuantizer()(api.RowQuantizeArguments(x=x, q=q, scale=s))
    quotient = _quotient(x.double())
    assert kind == "normal" or bool(_ties(quotient).any(dim=1).all())
    # With a value of up to 11 bits a quotient that is no tie is at least 1 / (254 * 2^11) > 2^-19 of itself away from one:
    # fp32 arithmetic to 2^-24 has no other answer than the nearest integer.
    assert torch.equal(q.double(), quotient.round())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K, pad", [(2048, 0), (2048, 1), (2056, 0), (70000, 0)])
def test_every_mantissa_under_every_largest_value(cuda_lib, K, pad, dtype):
    """Row b: all multiples of a step up to b steps, b from half to all of what the type's mantissa holds; then, under the
    same largest value, a half, a quarter ... of them."""
    top = 2048 if dtype == torch.float16 else 256
    b = torch.arange(top // 2, top, device="cuda")
    step = torch.arange(K, device="cuda") % top
    x = torch.empty(len(b), K + pad, dtype=dtype, device="cuda")[:, :K]
    x.copy_(torch.where(step[None, :] <= b[:, None], step, b[:, None] - step))
    q, s = torch.empty(len(b), K, dtype=torch.int8, device="cuda"), torch.empty(len(b), device="cuda")
    for fraction in range(8):
        if fraction:
            x.mul_(0.5)
            x[:, -1] = b.to(dtype)
        api.RowQuantizer()(api.RowQuantizeArguments(x=x, q=q, scale=s))
        assert torch.equal(q.double(), _quotient(x.double()).round())


@pytest.mark.parametrize("dtype, kind", [(torch.float16, "normal"), (torch.bfloat16, "normal"), (torch.float16, "grid"),
                                         (torch.bfloat16, "grid"), (torch.bfloat16, "tiny grid")])
@pytest.mark.parametrize("M, K", TIE_SHAPES)
def test_ties_behind_the_norm(cuda_lib, M, K, dtype, kind):
    """y = h w / rms: its ties are those of h w, in which the root does not occur."""
    x = _tie_rows(M, K, dtype, kind, seed=K + 1)
    w = (torch.randint(4, 13, (K,), generator=_gen(K), device="cuda") / 8).to(dtype)
    q, s = torch.full((M, K), 99, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, eps=0.0))
    quotient = _quotient(x.double() * w.double())
    ties, want = _ties(quotient), quotient.round()
    assert kind == "normal" or bool(ties.any())
    assert torch.equal(q.double()[ties], want[ties])
    # Products of the weights here (4 bits) and x have up to 15 bits: no quotient but a tie is within 1 / (254 * 2^15) > 2^-23
    # of itself of one.
    assert torch.equal(q.double(), want)


# ---- rows of many values ------------------------------------------------------------------------

@pytest.mark.parametrize("K", [1 << 24, (1 << 26) + 3])
def test_norm_of_a_long_row_of_one_value(cuda_lib, K):
    """Equal squares: a sum that loses part of each of them is off by as much in all."""
    x = torch.full((1, K), 0.7, dtype=torch.float16, device="cuda")
    x[0, K // 3] = -1.5
    w = torch.ones(K, dtype=torch.float16, device="cuda")
    q, s = torch.empty(1, K, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, eps=0.0))
    # the scale as in test_rmsnorm of the shorter rows
    _check_quantised(q, s, _norm_reference(x, None, w, 0.0)[1], 4 * U, 154 * U)


# ---- the product's epilogue at the ends of its range --------------------------------------------

PAIR, BLOCK = _lib.GEMM_HINT_PAIR, _lib.GEMM_HINT_BLOCK


@pytest.mark.parametrize("hints", [BLOCK, PAIR])
@pytest.mark.parametrize("act", list(ACTS))
def test_scales_whose_product_is_beyond_fp32(cuda_lib, act, hints):
    """Sums times their scales are numbers, the two scales' product is not: infinite, subnormal or zero."""
    M, N, K = 40, 64, 96
    for xs, ws, bias in ((2.0 ** 120, 2.0 ** 10, True), (2.0 ** -130, 2.0 ** -14, False), (2.0 ** -140, 2.0 ** -14, False),
                         (2.0 ** -110, 2.0 ** -30, False), (2.0 ** -12, 2.0 ** -130, False)):
        p = Product(M, N, K, torch.bfloat16, act=act, bias=bias, seed=3)
        p.xs.copy_(xs * (1 + torch.arange(M, device="cuda") / 64))
        p.ws.copy_(ws * (1 + torch.arange(N, device="cuda") / 128))
        if xs > 1:
            p.w.zero_()  # sums of zero: the bias alone is left
        p.run(hints=hints).check()


@pytest.mark.parametrize("hints", [BLOCK, PAIR])
@pytest.mark.parametrize("act", ["silu", "gated"])
def test_gates_far_below_zero(cuda_lib, act, hints):
    """v / (1 + exp(-v)) for v from -80 to -110: bf16 holds it down to -92 as a normal number, and beyond as a subnormal one."""
    M, N, K = 40, 480, 32
    p = Product(M, N, K, torch.bfloat16, act=act, bias=True, seed=4)
    p.x.zero_()
    gates = -80 - torch.arange(N, device="cuda") / 16
    p.bias.copy_(gates)
    if act == "gated":
        p.bias[1::2] = 3
    p.run(hints=hints)
    v = p.bias.double()
    want = v / (1 + torch.exp(-v))
    if act == "gated":
        want = want[0::2] * 3
    # exp(v): the argument times log2(e) errs by 2^-23 of |v| * 1.44 in its exponent, 2^-16 of the value at 110; ten more roundings
    # of fp32 and one to bf16 (2^-8), whose subnormal step is 2^-133, and fp32's below 2^-126, times up to 3, 2^-149
    off = (p.out.double() - want).abs() - ((2.0 ** -8 + 2.0 ** -15) * want.abs() + 2.0 ** -134 + 2.0 ** -147)
    assert float(off.max()) <= 0, p.out[0, off.argmax().item() % p.out.shape[1]]


# ---- clusters of every size ---------------------------------------------------------------------

@pytest.mark.parametrize("hints", [BLOCK | _lib.gemm_hint_split(s) | _lib.gemm_hint_rows(r) for s in range(1, 9) for r in (16, 32, 96, 256)] +
                         [PAIR | _lib.gemm_hint_split(s) | _lib.gemm_hint_rows(r) for s in (1, 2, 4) for r in (32, 256)])
@pytest.mark.parametrize("M, N, K, act", [(1, 100, 1090, "none"), (77, 300, 1300, "silu"), (263, 642, 2049, "gated")])
def test_every_cluster_size_writes_every_element(cuda_lib, M, N, K, act, hints):
    p = Product(M, N, K, act=act, bias=True, seed=6, ldd=(N // 2 if act == "gated" else N) + 3)
    p.run().check()
    want = p.out.clone()
    p.out.fill_(1234.0)
    p.run(hints=hints)
    assert torch.equal(p.out, want)
    assert api.device_error_state() == 0
    p.check_surroundings()


@pytest.mark.parametrize("M", [4, 300])
def test_rows_beside_one_without_a_scale_are_written(cuda_lib, M):
    p = Product(M, 260, 320, bias=True, seed=2).run()
    want = p.out.clone()
    p.xs[1] = float("nan")
    p.out.fill_(1234.0)
    p.run()
    keep = [i for i in range(M) if i != 1]
    assert bool(p.out[1].isnan().all()) and torch.equal(p.out[keep], want[keep])


# ---- a predecessor that takes long --------------------------------------------------------------

@pytest.fixture(scope="module")
def slow_predecessor(tmp_path_factory):
    """Enqueues a kernel of that many seconds which lets its dependents start at once."""
    import ctypes as C
    import os
    import subprocess
    from mixed_gemv_b200 import build
    out = str(tmp_path_factory.mktemp("slow") / "slow_predecessor.so")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "slow_predecessor.cu")
    subprocess.run([build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-shared", "-Xcompiler", "-fPIC", src,
                    "-o", out], check=True, capture_output=True, timeout=300)
    fn = C.CDLL(out).slow_predecessor
    fn.argtypes = [C.c_ulonglong, C.c_void_p]
    return lambda seconds: fn(int(seconds * 1e9), torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("hints", [BLOCK, PAIR, BLOCK | _lib.gemm_hint_split(4) | _lib.gemm_hint_rows(32),
                                   PAIR | _lib.gemm_hint_split(2) | _lib.gemm_hint_rows(64)])
def test_the_limit_of_the_waits_does_not_count_the_predecessor(cuda_lib, slow_predecessor, hints):
    """The kernels' waits give up after a second; a dependent launch that starts early waits for its predecessor first."""
    p = Product(70, 600, 1100, bias=True, seed=9)
    op = api.GemmI8Adaptor()
    op.initialize(p.arguments(_lib.FLAG_PDL, hints))
    op.run()
    torch.cuda.synchronize()
    p.out.fill_(1234.0)
    torch.cuda.synchronize()
    assert slow_predecessor(1.5) == 0
    op.run()
    torch.cuda.synchronize()
    assert api.device_error_state() == 0
    p.check()


THREADS = """
import threading
import torch
from mixed_gemv_b200 import api
x = [torch.randn(700, 512 + 8 * i, dtype=torch.float32, device="cuda").half() for i in range(8)]
q = [torch.empty(t.shape, dtype=torch.int8, device="cuda") for t in x]
s = [torch.empty(700, device="cuda") for t in x]
torch.cuda.synchronize()
start = threading.Barrier(8)
def one(i):
    start.wait()
    api.RowQuantizer()(api.RowQuantizeArguments(x=x[i], q=q[i], scale=s[i]), torch.cuda.Stream())
threads = [threading.Thread(target=one, args=(i,)) for i in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
for a, b, c in zip(x, q, s):
    y = a.double()
    assert torch.equal(b.double(), (y * 127 / y.abs().amax(dim=1, keepdim=True)).round())
print("threads agree")
"""


def test_first_calls_from_several_threads(cuda_lib):
    import subprocess
    import sys
    from tests.conftest import ROOT
    r = subprocess.run([sys.executable, "-c", THREADS], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "threads agree" in r.stdout, r.stderr[-2000:]
