"""GPU tests of the 8-bit activation path against plain implementations in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of fp32 relative to the value.
"""
import pytest
import torch

from mixed_gemv_b200 import _lib, api
from mixed_gemv_b200.enums import Status

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _strided(rows, cols, dtype, ld, offset=0, fill=None):
    """A [rows, cols] view with `ld` elements between rows, `offset` elements behind its allocation."""
    flat = torch.empty(offset + max(rows, 1) * ld + 64, dtype=dtype, device="cuda")
    if fill is not None:
        flat.fill_(fill)
    return flat[offset:offset + rows * ld].view(rows, ld)[:, :cols], flat


# ---- rows into int8 and back --------------------------------------------------------------------

def _check_quantised(q, scale, y, top_slack, scale_tol):
    """q and scale against the 64-bit rows y: the scale to a relative error, each q to the nearest
    integer of y * 127 / top, where top_slack is the relative error that fp32 may put on that product."""
    top = y.abs().amax(dim=1)
    assert torch.all((scale.double() - top / 127).abs() <= scale_tol * top / 127 + 2.0 ** -149)
    want = torch.where(top[:, None] > 0, y * 127 / top[:, None].clamp_min(1e-300), torch.zeros_like(y))
    assert float((q.double() - want).abs().max()) <= 0.5 + 127 * top_slack
    assert int(q.min()) >= -127


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 64), (5, 100), (64, 1024), (7, 1031), (4, 4096), (3, 5001), (2, 8192), (9, 11008),
          (3, 16392), (2, 28672), (1, 65536), (2, 65543), (2, 70000), (1500, 256), (1000, 24),
          # more rows than blocks at a time
          (12000, 136), (3000, 1031), (1400, 4096), (700, 8200), (500, 9001), (400, 28680)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M, K", SHAPES)
def test_quantize_and_back(cuda_lib, M, K, dtype):
    x = torch.randn(M, K, generator=_gen(K + M), device="cuda").to(dtype)
    q = torch.full((M, K), 99, dtype=torch.int8, device="cuda")
    s, back = torch.empty(M, device="cuda"), torch.empty_like(x)
    api.RowQuantizer()(api.RowQuantizeArguments(x=x, q=q, scale=s))
    api.RowDequantizer()(api.RowDequantizeArguments(q=q, scale=s, out=back))
    # scale: one division.  q: the reciprocal 127/top (u) and one product (u) before the rounding
    _check_quantised(q, s, x.double(), 3 * U, 2 * U)
    # back: one product in fp32 (u) and one rounding to dtype
    want = q.double() * s.double()[:, None]
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    assert torch.all((back.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 2 * U) * want.abs() + tiny)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K, ldx, ldq, ox, oq", [(64, 72, 80, 0, 0), (100, 104, 112, 8, 8), (100, 101, 103, 1, 3), (4096, 4104, 4112, 8, 0),
                                                 (4099, 4100, 4099, 0, 1), (8192, 8194, 8192, 2, 4), (66000, 66008, 66001, 0, 0)])
def test_strides_and_alignments(cuda_lib, K, ldx, ldq, ox, oq, dtype):
    M = 5
    x, _ = _strided(M, K, dtype, ldx, ox)
    x.copy_(torch.randn(M, K, generator=_gen(K), device="cuda"))
    q, qflat = _strided(M, K, torch.int8, ldq, oq, fill=77)
    sflat = torch.full((M + 8,), 5.0, device="cuda")
    back, bflat = _strided(M, K, dtype, ldx, ox, fill=3.0)
    api.RowQuantizer()(api.RowQuantizeArguments(x=x, q=q, scale=sflat[:M]))
    api.RowDequantizer()(api.RowDequantizeArguments(q=q, scale=sflat[:M], out=back))
    _check_quantised(q, sflat[:M], x.double(), 3 * U, 2 * U)
    want = q.double() * sflat[:M].double()[:, None]
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    assert torch.all((back.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 2 * U) * want.abs() + tiny)
    # what lies between and behind the rows is left as it was
    q.fill_(77)
    back.fill_(3.0)
    assert bool((qflat == 77).all()) and bool((bflat == 3.0).all()) and bool((sflat[M:] == 5.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [48, 4096, 5001, 70000])
def test_rows_without_and_beyond_numbers(cuda_lib, K, dtype):
    """Zeros, one value alone, infinities, NaN, the smallest and the largest values, next to an ordinary row."""
    x = torch.randn(9, K, generator=_gen(K), device="cuda").to(dtype)
    x[0] = 0
    x[1] = 0
    x[1, K - 1] = -3
    x[2, K // 2] = float("inf")
    x[3, 0] = float("nan")
    x[4, K - 1] = -float("inf")
    x[5] = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps       # the smallest subnormal
    x[6] = torch.finfo(dtype).max
    x[7, :] = torch.finfo(dtype).smallest_normal * x[8].sign()
    w = torch.ones(K, dtype=dtype, device="cuda")
    for norm in (False, True):
        q, s = torch.full((9, K), 99, dtype=torch.int8, device="cuda"), torch.empty(9, device="cuda")
        if norm:
            api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, eps=0.0))
        else:
            api.RowQuantizer()(api.RowQuantizeArguments(x=x, q=q, scale=s))
        bad = torch.tensor([2, 3, 4], device="cuda")
        assert bool(s[bad].isnan().all()) and not bool(q[bad].any())
        assert float(s[0]) == 0 and not bool(q[0].any())
        assert q[1, K - 1] == -127 and not bool(q[1, :K - 1].any())
        assert bool((q[5] == 127).all()) and bool((q[6] == 127).all())
        good = torch.tensor([0, 1, 5, 6, 7, 8], device="cuda")
        y = x[good].double()
        if norm:
            y = y / y.square().mean(dim=1, keepdim=True).sqrt().clamp_min(1e-300)
        # a subnormal fp32 scale is a whole number of 2^-149, half a step off at most (in _check_quantised);
        # the norm's fp32 statistics as in test_rmsnorm
        _check_quantised(q[good], s[good], y, 4 * U, (2 if not norm else 150) * U)


@pytest.mark.parametrize("K", [136, 1031, 4096, 8200])
def test_wild_rows_among_many(cuda_lib, K):
    """Rows that need double precision, or hold no numbers, between ordinary ones of the same block."""
    M, dtype = 3000, torch.bfloat16
    g = _gen(K)
    x, r = torch.randn(M, K, generator=g, device="cuda").to(dtype), torch.randn(M, K, generator=g, device="cuda").to(dtype)
    for start, factor in ((0, 1e-25), (1, 1e25), (2, 0.0)):
        x[start::7] *= factor
        r[start::7] *= factor
    x[3::700, K // 3] = float("inf")
    x[4::700, K - 1] = float("nan")
    w = (1 + 0.2 * torch.randn(K, generator=g, device="cuda")).to(dtype)
    q, s, ro = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda"), torch.empty_like(x)
    api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, residual=r, residual_out=ro, eps=0.0))
    h, y = _norm_reference(x, r, w, 0.0)
    assert torch.equal(torch.nan_to_num(ro), torch.nan_to_num(h))
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[3::700] = bad[4::700] = True
    assert bool(s[bad].isnan().all()) and not bool(q[bad].any()) and not bool(s[~bad].isnan().any())
    zero = h.float().abs().amax(dim=1) == 0
    assert not bool(q[zero].any()) and not bool(s[zero].any())
    y[zero] = 0
    _check_quantised(q[~bad], s[~bad], y[~bad], 4 * U, 154 * U)


def test_offsets_beyond_32_bits(cuda_lib):
    """Three rows, gigabytes apart."""
    M, K, N, far = 3, 520, 264, 1_500_000_016
    x, _ = _strided(M, K, torch.float16, far)
    x.copy_(torch.randn(M, K, generator=_gen(1), device="cuda"))
    q, _ = _strided(M, K, torch.int8, 2 * far)
    s, w = torch.empty(M, device="cuda"), torch.ones(K, dtype=torch.float16, device="cuda")
    api.RowQuantizer()(api.RowQuantizeArguments(x=x, q=q, scale=s))
    _check_quantised(q, s, x.double(), 3 * U, 2 * U)
    want = x.clone() + x.clone()
    api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, residual=x, residual_out=x))
    assert torch.equal(x, want)
    _check_quantised(q, s, _norm_reference(want, None, w, float(torch.tensor(1e-5)))[1], 4 * U, 154 * U)
    api.RowDequantizer()(api.RowDequantizeArguments(q=q, scale=s, out=x))
    back = q.double() * s.double()[:, None]
    assert torch.all((x.double() - back).abs() <= (2.0 ** -11 + 2 * U) * back.abs() + 2.0 ** -25)
    p = Product(M, N, K, bias=True)
    p.out, _ = _strided(M, N, torch.float16, far)
    p.x, p.xs = q, s
    p.run().check()


# ---- norm ---------------------------------------------------------------------------------------

def _norm_reference(x, residual, weight, eps):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    d = h.double()
    return h, d / (d.square().mean(dim=1, keepdim=True) + eps).sqrt() * weight.double()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("M, K", SHAPES)
def test_rmsnorm(cuda_lib, M, K, with_residual, dtype):
    g = _gen(M * 31 + K)
    x = (torch.randn(M, K, generator=g, device="cuda") * 3).to(dtype)
    r = (torch.randn(M, K, generator=g, device="cuda") * 2).to(dtype) if with_residual else None
    ro = torch.full_like(x, 7.0) if with_residual else None
    w = (1 + 0.3 * torch.randn(K, generator=g, device="cuda")).to(dtype)
    q, s = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, residual=r, residual_out=ro, eps=1e-6))
    h, y = _norm_reference(x, r, w, float(torch.tensor(1e-6)))
    if with_residual:
        assert torch.equal(ro, h)
    # q: product with the weight (u), reciprocal (u), product (u).  Scale: the sum of squares of a thread's up to 260
    # values and of up to 32 partial sums, all positive, errs by at most 290 u, its root by half of that; eight more roundings
    _check_quantised(q, s, y, 4 * U, 154 * U)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [3, 40, 263, 1031, 4100, 9001, 16377])
@pytest.mark.parametrize("offsets", [(0, 1, 2, 3, 1), (1, 1, 1, 0, 0), (5, 3, 5, 2, 7), (7, 0, 3, 5, 2)])
def test_norm_of_operands_apart(cuda_lib, K, offsets, dtype):
    """x, residual, residual_out, weight and q each at an address and a distance of rows of its own; what lies around
    the outputs is left as it was."""
    M, g = 7, _gen(K)
    ox, orr, oro, ow, oq = offsets
    x, _ = _strided(M, K, dtype, K + 1, ox)
    r, _ = _strided(M, K, dtype, K + 3, orr)
    ro, roflat = _strided(M, K, dtype, K + 2, oro, fill=5.0)
    q, qflat = _strided(M, K, torch.int8, K + 5, oq, fill=77)
    w = torch.empty(K + 8, dtype=dtype, device="cuda")[ow:ow + K] if ow else torch.empty(K, dtype=dtype, device="cuda")
    for a in (x, r, w):
        a.copy_(torch.randn(a.shape, generator=g, device="cuda"))
    s = torch.empty(M, device="cuda")
    api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, residual=r, residual_out=ro))
    h, y = _norm_reference(x, r, w, float(torch.tensor(1e-5)))
    assert torch.equal(ro, h)
    _check_quantised(q, s, y, 4 * U, 154 * U)
    ro.fill_(5.0)
    q.fill_(77)
    assert bool((roflat == 5.0).all()) and bool((qflat == 77).all())


def test_rmsnorm_eps_matters_and_large_values_do_not_overflow(cuda_lib):
    K = 4096
    x = torch.randn(4, K, generator=_gen(1), device="cuda")
    x[0] *= 1e-4
    x[1] *= 1e30      # squares beyond fp32
    x[2] *= 1e-30     # squares below fp32
    x = x.to(torch.bfloat16)
    w = torch.full((K,), 1e25, dtype=torch.bfloat16, device="cuda")  # times row 1: beyond fp32 before the division
    q, s = torch.empty(4, K, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    for eps in (1e-5, 0.0, 1e-38):
        api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, eps=eps))
        _, y = _norm_reference(x, None, w, float(torch.tensor(eps)))
        _check_quantised(q, s, y, 4 * U, 154 * U)


@pytest.mark.parametrize("K", [4096, 5001])
def test_rmsnorm_of_one_value_and_the_largest_weights(cuda_lib, K):
    """y is beyond fp32, its scale is not."""
    x = torch.zeros(2, K, dtype=torch.bfloat16, device="cuda")
    x[:, K // 2] = 1
    w = torch.full((K,), 3e38, dtype=torch.bfloat16, device="cuda")
    q, s = torch.empty(2, K, dtype=torch.int8, device="cuda"), torch.empty(2, device="cuda")
    api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, eps=0.0))
    assert bool(s.isfinite().all())
    _check_quantised(q, s, _norm_reference(x, None, w, 0.0)[1], 4 * U, 154 * U)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K, ld", [(512, 520), (5001, 5003), (4096, 4096), (70000, 70000)])
@pytest.mark.parametrize("onto", ["residual", "x"])
def test_residual_in_place(cuda_lib, K, ld, onto, dtype):
    M, g = 6, _gen(K)
    x, _ = _strided(M, K, dtype, ld)
    r, _ = _strided(M, K, dtype, ld)
    x.copy_(torch.randn(M, K, generator=g, device="cuda"))
    r.copy_(torch.randn(M, K, generator=g, device="cuda"))
    w = torch.randn(K, generator=g, device="cuda").to(dtype)
    q, s = torch.empty(M, K, dtype=torch.int8, device="cuda"), torch.empty(M, device="cuda")
    h, y = _norm_reference(x.clone(), r.clone(), w, float(torch.tensor(1e-5)))
    target = r if onto == "residual" else x
    api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=w, q=q, scale=s, residual=r, residual_out=target))
    assert torch.equal(target, h)
    _check_quantised(q, s, y, 4 * U, 154 * U)


# ---- int8 matrix product ------------------------------------------------------------------------

ACTS = {"none": 0, "relu": _lib.FLAG_ACT_RELU, "silu": _lib.FLAG_ACT_SILU, "gated": _lib.FLAG_GATED_SILU}


class Product:
    def __init__(self, M, N, K, dtype=torch.float16, scales=torch.float32, bias=False, act="none", seed=0, pad=0, ldd=None, out_offset=0):
        g = _gen(seed)
        ld = -(-K // 16) * 16 + pad
        self.x, self.xflat = _strided(M, K, torch.int8, ld, fill=113)
        self.w, self.wflat = _strided(N, K, torch.int8, ld, fill=-77)
        self.x.copy_(torch.randint(-128, 128, (M, K), generator=g, device="cuda"))
        self.w.copy_(torch.randint(-128, 128, (N, K), generator=g, device="cuda"))
        self.xs = (torch.rand(M, generator=g, device="cuda") + 0.5) / 64
        self.ws = ((torch.rand(N, generator=g, device="cuda") + 0.5) / (64 * K ** 0.5)).to(scales)
        self.bias = torch.randn(N, generator=g, device="cuda").to(dtype) if bias else None
        self.act, self.dtype, self.cols = act, dtype, N // 2 if act == "gated" else N
        self.out, self.flat = _strided(M, self.cols, dtype, ldd or self.cols, out_offset, fill=1234.0)

    def arguments(self, flags=0, hints=0):
        return api.GemmI8Arguments(x=self.x, x_scale=self.xs, weights=self.w, weight_scale=self.ws, bias=self.bias, out=self.out,
                                   flags=flags | ACTS[self.act], hints=hints)

    def run(self, flags=0, hints=0):
        api.GemmI8Adaptor()(self.arguments(flags, hints))
        return self

    def check(self):
        """Against 64 bits.  v = float(sum) * (sx * sw) + b: three roundings of the product, one of the sum.  silu: e = exp(-v)
        errs by (2 + |v|) steps of fp32 from its argument and its approximation, the quotient by two more; v^2 exp(-|v|) < 1
        bounds what that makes of the value.  Then one rounding to dtype."""
        prod = (self.x.double() @ self.w.double().t()) * self.xs.double()[:, None] * self.ws.double()
        v = prod if self.bias is None else prod + self.bias.double()
        err = 4 * U * prod.abs() + 2 * U * v.abs()
        if self.act == "relu":
            v = v.clamp_min(0)
        elif self.act == "silu":
            err, v = 1.1 * err + 16 * U * (1 + v.abs()), v * torch.sigmoid(v)
        elif self.act == "gated":
            gate, up = v[:, 0::2], v[:, 1::2]
            ge, ue = err[:, 0::2], err[:, 1::2]
            a = gate * torch.sigmoid(gate)
            ae = 1.1 * ge + 16 * U * (1 + gate.abs())
            err, v = ae * up.abs() + a.abs() * ue + 2 * U * (a * up).abs(), a * up
        half = torch.finfo(self.dtype).eps / 2
        tiny = torch.finfo(self.dtype).smallest_normal * half
        off = (self.out.double() - v).abs() - (1.01 * err + half * (v.abs() + err) + tiny)
        assert float(off.max()) <= 0, (float(off.max()), off.argmax().item(), tuple(v.shape))
        return self

    def check_surroundings(self):
        self.out.fill_(1234.0)
        assert bool((self.flat == 1234.0).all())


GEMM_SHAPES = [(1, 1, 1), (1, 2, 16), (2, 3, 5), (1, 128, 128), (16, 130, 100), (17, 34, 129), (3, 1000, 4096), (33, 256, 640),
               (64, 512, 2048), (128, 128, 128), (129, 258, 255), (200, 4096, 1024), (255, 256, 257), (257, 514, 384), (300, 500, 1000),
               (1000, 1026, 520), (5, 4098, 11008), (700, 2050, 300)]


@pytest.mark.parametrize("M, N, K, act", [(*mnk, act) for mnk in GEMM_SHAPES for act in ("none", "gated") if act == "none" or mnk[1] % 2 == 0])
def test_gemm(cuda_lib, M, N, K, act):
    Product(M, N, K, torch.bfloat16 if M % 2 else torch.float16, bias=N % 4 == 0, act=act, seed=M).run().check()


PATHS = [_lib.GEMM_HINT_BLOCK | _lib.gemm_hint_split(s) | _lib.gemm_hint_rows(r) for s in (1, 2, 4, 8) for r in (16, 96, 256)] + \
        [_lib.GEMM_HINT_PAIR | _lib.gemm_hint_split(s) | _lib.gemm_hint_rows(r) for s in (1, 2, 4) for r in (32, 96, 160, 256)]


@pytest.mark.parametrize("hints", PATHS)
@pytest.mark.parametrize("M, N, K, act", [(1, 100, 64, "none"), (77, 300, 1300, "silu"), (500, 642, 2049, "gated"), (513, 1025, 2000, "relu")])
def test_every_kernel_and_tiling_gives_the_same_bits(cuda_lib, M, N, K, act, hints):
    p = Product(M, N, K, act=act, bias=True, seed=6).run(hints=hints).check()
    forced = p.out.clone()
    assert torch.equal(p.run().out, forced)
    assert api.device_error_state() == 0


def test_more_tiles_than_blocks(cuda_lib):
    """Every pair of blocks takes several tiles, whose accumulators and ring slots alternate; the last ones come in
    halves (of 2000 x 5000 and 1800 x 5000 at 256 rows), some of them with no rows left (of 1800)."""
    for M, N, K in ((2000, 5000, 200), (1800, 5000, 200), (4096, 8192, 1100)):
        for rows in (64, 256):
            Product(M, N, K, act="gated", seed=7).run(hints=_lib.GEMM_HINT_PAIR | _lib.gemm_hint_rows(rows)).check()
    assert api.device_error_state() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scales", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M", [3, 300])
def test_gemm_types_and_activations(cuda_lib, M, act, scales, dtype):
    Product(M, 390, 272, dtype, scales, bias=True, act=act, seed=5).run().check()


@pytest.mark.parametrize("act", ["none", "gated"])
@pytest.mark.parametrize("M, N, ldd, offset", [(5, 256, 300, 0), (40, 256, 257, 1), (300, 512, 520, 8), (300, 512, 515, 3), (600, 130, 131, 2)])
def test_gemm_strides(cuda_lib, M, N, ldd, offset, act):
    p = Product(M, N, 200, act=act, pad=48, ldd=ldd, out_offset=offset, seed=9).run().check()
    p.check_surroundings()


@pytest.mark.parametrize("M", [3, 40, 300])
def test_gemm_odd_features_in_even_rows(cuda_lib, M):
    """The last feature stands alone in rows whose others are stored two at a time."""
    p = Product(M, 517, 300, bias=True, ldd=520, seed=12).run().check()
    p.check_surroundings()


@pytest.mark.parametrize("M", [1, 200])
def test_gemm_largest_sums(cuda_lib, M):
    """131071 products of -128 and -128: the largest sum there is, 2147467264."""
    p = Product(M, 8, 131071, seed=3)
    p.x.fill_(-128)
    p.w.fill_(-128)
    p.run().check()
    p.w.fill_(127)
    p.run().check()


@pytest.mark.parametrize("M", [4, 300])
def test_a_row_without_a_scale_spoils_itself_only(cuda_lib, M):
    for act in ACTS:
        p = Product(M, 260, 320, act=act, bias=True, seed=2)
        p.run()
        want = p.out.clone()
        p.xs[1] = float("nan")
        p.run()
        assert bool(p.out[1].isnan().all())
        keep = [i for i in range(M) if i != 1]
        assert torch.equal(p.out[keep], want[keep])


def test_gemm_results_repeat(cuda_lib):
    for M, N, K in ((8, 4096, 4096), (130, 1000, 5000), (1000, 2000, 1000)):
        p = Product(M, N, K, seed=1).run()
        first = p.out.clone()
        for _ in range(3):
            p.out.fill_(0)
            assert torch.equal(p.run().out, first)


def test_no_rows(cuda_lib):
    x, q, s = torch.empty(0, 64, dtype=torch.float16, device="cuda"), torch.empty(0, 64, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda")
    w = torch.zeros(32, 64, dtype=torch.int8, device="cuda")
    api.RowQuantizer()(api.RowQuantizeArguments(x=x, q=q, scale=s))
    api.RowDequantizer()(api.RowDequantizeArguments(q=q, scale=s, out=x))
    api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=x, weight=torch.ones(64, dtype=torch.float16, device="cuda"), q=q, scale=s))
    api.GemmI8Adaptor()(api.GemmI8Arguments(x=q, x_scale=s, weights=w, weight_scale=torch.ones(32, device="cuda"), out=x[:, :32]))
    torch.cuda.synchronize()


def test_python_face_refusals(cuda_lib):
    p = Product(4, 32, 64)
    good = dict(x=p.x, x_scale=p.xs, weights=p.w, weight_scale=p.ws, out=p.out)
    half = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    for change, status in ((dict(x=p.x.float()), Status.UNSUPPORTED), (dict(x_scale=p.xs[:3]), Status.INVALID_ARGUMENT),
                           (dict(x_scale=p.xs.half()), Status.UNSUPPORTED), (dict(weights=p.w[:, :32]), Status.INVALID_ARGUMENT),
                           (dict(out=p.out.float()), Status.UNSUPPORTED), (dict(out=p.out[:, :16]), Status.INVALID_ARGUMENT),
                           (dict(bias=torch.zeros(32, device="cuda")), Status.UNSUPPORTED), (dict(x=p.x[0]), Status.INVALID_ARGUMENT),
                           (dict(x=p.x[:1].expand(4, 64)), Status.INVALID_ARGUMENT),
                           (dict(x=torch.zeros(4, 72, dtype=torch.int8, device="cuda")[:, :64]), Status.MISALIGNED),
                           (dict(weights=torch.zeros(64, 32, dtype=torch.int8, device="cuda").t()), Status.INVALID_ARGUMENT),
                           (dict(x_scale=p.xs.cpu()), Status.INVALID_ARGUMENT)):
        with pytest.raises(api.MgvError) as e:
            api.GemmI8Adaptor()(api.GemmI8Arguments(**{**good, **change}))
        assert e.value.status == status, change
    with pytest.raises(api.MgvError, match="together"):
        api.RmsNormQuantizer()(api.RmsNormQuantizeArguments(x=half, weight=half[0], q=p.x, scale=p.xs, residual=half))
    torch.cuda.synchronize()


# ---- streams, graphs, and the operators in a row ------------------------------------------------

class LayerHalf:
    """Norm, gate/up product, quantisation and down projection of a layer."""

    def __init__(self, M, K, H, dtype, seed):
        g = _gen(seed)
        new = lambda *shape, dtype=dtype: torch.empty(*shape, dtype=dtype, device="cuda")  # noqa: E731
        self.x, self.r = torch.randn(M, K, generator=g, device="cuda").to(dtype), torch.randn(M, K, generator=g, device="cuda").to(dtype)
        self.weight = (1 + 0.1 * torch.randn(K, generator=g, device="cuda")).to(dtype)
        self.up, self.down = Product(M, 2 * H, K, dtype, act="gated", seed=seed + 1), Product(M, K, H, dtype, seed=seed + 2)
        self.ro, self.q, self.s = new(M, K), self.up.x, self.up.xs
        self.q2, self.s2 = self.down.x, self.down.xs
        pdl = _lib.FLAG_PDL
        self.ops = []
        for op, args in ((api.RmsNormQuantizer(), api.RmsNormQuantizeArguments(x=self.x, weight=self.weight, q=self.q, scale=self.s,
                                                                               residual=self.r, residual_out=self.ro, flags=pdl)),
                         (api.GemmI8Adaptor(), self.up.arguments(pdl)),
                         (api.RowQuantizer(), api.RowQuantizeArguments(x=self.up.out, q=self.q2, scale=self.s2, flags=pdl)),
                         (api.GemmI8Adaptor(), self.down.arguments(pdl))):
            op.initialize(args)
            self.ops.append(op)

    def run(self, stream=None):
        for op in self.ops:
            op.run(stream)

    def check(self):
        """Every operator against 64 bits on the inputs that its predecessor gave it."""
        h, y = _norm_reference(self.x, self.r, self.weight, float(torch.tensor(1e-5)))
        assert torch.equal(self.ro, h)
        _check_quantised(self.q, self.s, y, 4 * U, 154 * U)
        self.up.check()
        _check_quantised(self.q2, self.s2, self.up.out.double(), 3 * U, 2 * U)
        self.down.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 16, 100, 600])
def test_operators_in_a_row(cuda_lib, M, dtype):
    layer = LayerHalf(M, 512, 1408, dtype, seed=M)
    for _ in range(3):
        layer.run()
    torch.cuda.synchronize()
    layer.check()


def test_two_streams_at_once(cuda_lib):
    layers = [LayerHalf(m, 768, 1024, torch.float16, seed=m) for m in (24, 500)]
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    for _ in range(20):
        for layer, st in zip(layers, streams):
            layer.run(st)
    torch.cuda.synchronize()
    for layer in layers:
        layer.check()
    assert api.device_error_state() == 0


def test_captured_and_replayed_on_new_inputs(cuda_lib):
    layer = LayerHalf(40, 640, 1000, torch.bfloat16, seed=4)
    layer.run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same calls, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer.run()
        graphs.append(graph)
    for seed in range(4):
        layer.x.copy_(torch.randn(layer.x.shape, generator=_gen(100 + seed), device="cuda"))
        for t in (layer.q, layer.q2, layer.up.out, layer.down.out):
            t.fill_(1)
        graphs[seed % 2].replay()
        torch.cuda.synchronize()
        layer.check()


FIRST_CALL = """
import torch
from tests.test_gpu_int8_path import LayerHalf
layer = LayerHalf(24, 512, 704, torch.float16, seed=3)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    layer.run()
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
layer.check()
print("first call captured")
"""


def test_the_first_run_of_a_process_may_be_captured(cuda_lib):
    """Plans are made before the capture, nothing has been launched."""
    import subprocess
    import sys
    from tests.conftest import ROOT
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "first call captured" in r.stdout, r.stderr[-2000:]


def test_the_call_without_a_plan(cuda_lib):
    import ctypes as C
    for M, act in ((0, "none"), (5, "gated"), (300, "silu")):
        p = Product(M, 130, 200, act=act, bias=True, seed=11)
        c = api.GemmI8Adaptor._to_c(cuda_lib, p.arguments())
        assert cuda_lib.mgv_gemm_i8(C.byref(c), None) == Status.OK
        torch.cuda.synchronize()
        if M:
            p.check()


def test_run_takes_the_stream_it_is_given(cuda_lib):
    p = Product(9, 96, 256, seed=8)
    op = api.GemmI8Adaptor()
    op.initialize(p.arguments())
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        op.run()
        after = p.out.clone()
    st.synchronize()
    assert torch.equal(after, p.out)
    p.check()
