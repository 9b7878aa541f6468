"""The MLP-block operators on a B200 against plain formulas in 64 bits.

Tolerances, with u the unit roundoff of the output's type (half the spacing at
1: 2^-8 for bf16, 2^-11 for fp16, 2^-24 for fp32) and e = 2^-23 the
step of the fp32 sums (a chain of n additions, each off by at most e of the
sum of magnitudes, whether rounded or truncated):
  rows      scale within SCALE_TOL; codes within half a step plus the scale's
            own error in steps;
  products  u |y| + k e sum|x||w| (the latter 0 for int8, whose sums are exact),
            and 4 e for the scales and the bias;
  ffn       the same for g and u, carried through the formulas; gradients add
            one rounding of dg and du (u sum|dg||w|).
"""
import ctypes

import pytest
import torch

import sp24

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
E = 2.0 ** -23
QMAX = {sp24.I8: 127.0, sp24.E4M3: 448.0}


@pytest.fixture(autouse=True)
def _clean_status():
    yield
    torch.cuda.synchronize()
    assert sp24.last_kernel_status() == 0, "a kernel raised its bounded-wait timeout flag"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(*shape, seed=0, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, device=DEV, generator=gen(seed)) * std).to(dtype)


# ------------------------------------------------------------------ rows to 8 bits
# Sum of squares: cols / 128 additions in a thread at the fewest threads, then a
# tree; the rest is a handful of roundings, and the exponential's 2^-21 for the
# arguments drawn here (its argument is scaled by log2(e) in fp32: |g| e).
def scale_tol(cols):
    return (cols / 128 + 64) * E


def check_rows(q, scale, y, qdtype, tol):
    """q, scale against the rows y (64 bits)."""
    amax = y.abs().amax(dim=1)
    want = amax / QMAX[qdtype]
    assert torch.all((scale.double() - want).abs() <= tol * want + 2.0 ** -149)
    v = torch.where(want[:, None] > 0, y / want[:, None].clamp_min(1e-300), 0.0)
    got = q.double()
    slack = QMAX[qdtype] * 2 * tol
    if qdtype == sp24.I8:
        half = 0.5
    else:   # half a step of e4m3: 2^-4 of the power of two at or below |v|, 2^-10 below 2^-6
        half = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 4)
    assert torch.all((got - v).abs() <= half + slack), (got - v).abs().max().item()


def rmsnorm64(x, w, r, eps):
    s = x.double() + (0 if r is None else r.double())
    return s, s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("qdtype", [sp24.I8, sp24.E4M3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (5, 64), (2, 129), (17, 1000),
                                       (33, 2048), (4, 5000), (2, 8192), (3, 14336), (1, 16392),
                                       (2, 40001), (9, 4092), (300, 300), (7, 8190), (3, 10006),
                                       (2, 16380), (2, 16386), (2, 8194)])
def test_rows_sizes(rows, cols, dtype, qdtype):
    x, r = randn(rows, cols, seed=1, dtype=dtype), randn(rows, cols, seed=2, std=3.0, dtype=dtype)
    w = (1 + randn(cols, seed=3, std=0.1)).to(dtype)
    tol = scale_tol(cols)
    q, s, total = sp24.rmsnorm_quant(x, w, residual=r, eps=1e-5, qdtype=qdtype)
    s64, y = rmsnorm64(x, w, r, 1e-5)
    check_rows(q, s, y, qdtype, tol)
    assert torch.equal(total, (x.float() + r.float()).to(dtype))
    q, s = sp24.rmsnorm_quant(x, w, eps=1e-5, qdtype=qdtype)
    check_rows(q, s, rmsnorm64(x, w, None, 1e-5)[1], qdtype, tol)
    q, s = sp24.swiglu_quant(x, r, qdtype=qdtype)
    g = x.double()
    check_rows(q, s, g * torch.sigmoid(g) * r.double(), qdtype, tol)
    q, s = sp24.quantize_rows(x, qdtype=qdtype)
    check_rows(q, s, x.double(), qdtype, tol)


@pytest.mark.parametrize("cols,ld,off", [(64, 72, 0), (64, 65, 0), (64, 64, 1), (1000, 1016, 8),
                                         (4096, 8192, 4096), (4097, 4100, 3),
                                         (100, 102, 2), (100, 104, 4), (96, 100, 4), (98, 98, 2), (64, 66, 0)])
def test_rows_strides(cols, ld, off):
    """Any row stride and any start, including 2-byte aligned ones."""
    buf = [randn(9 * ld + off, seed=i, dtype=torch.bfloat16) for i in range(2)]
    x, r = (b[off:off + 9 * ld].view(9, ld)[:, :cols] for b in buf)
    w = (1 + randn(cols + off, seed=3, std=0.1)).to(torch.bfloat16)[off:]
    q, s, total = sp24.rmsnorm_quant(x, w, residual=r, qdtype=sp24.I8)
    check_rows(q, s, rmsnorm64(x, w, r, 1e-6)[1], sp24.I8, scale_tol(cols))
    assert torch.equal(total, (x.float() + r.float()).to(torch.bfloat16))
    q, s = sp24.swiglu_quant(x, r, qdtype=sp24.E4M3)
    g = x.double()
    check_rows(q, s, g * torch.sigmoid(g) * r.double(), sp24.E4M3, scale_tol(cols))


@pytest.mark.parametrize("cols", [96, 4096, 5001])
def test_rows_in_place_residual_and_padding(cols):
    """residual_out may be the residual; nothing outside the rows is written."""
    ld = cols + 24
    x = randn(5, cols, seed=1, dtype=torch.float16)
    res = torch.full((5, ld), 7.0, device=DEV, dtype=torch.float16)
    res[:, :cols] = randn(5, cols, seed=2, dtype=torch.float16)
    before = res.clone()
    w = torch.ones(cols, device=DEV, dtype=torch.float16)
    q = torch.full((5, ld), 99, device=DEV, dtype=torch.int8)
    scale = torch.full((6,), -1.0, device=DEV)
    d = sp24.RowQuantDesc()
    d.dtype, d.qdtype, d.rows, d.cols = sp24.F16, sp24.I8, 5, cols
    d.x, d.residual, d.residual_out, d.weight = (t.data_ptr() for t in (x, res, res, w))
    d.ld_residual = d.ld_residual_out = d.ldq = ld
    d.q, d.scale, d.eps = q.data_ptr(), scale.data_ptr(), 1e-6
    assert sp24.load().sp24_rmsnorm_quant(ctypes.byref(d), torch.cuda.current_stream().cuda_stream) == 0
    check_rows(q[:, :cols], scale[:5], rmsnorm64(x, w, before[:, :cols], 1e-6)[1], sp24.I8, scale_tol(cols))
    assert torch.equal(res[:, :cols], (x.float() + before[:, :cols].float()).half())
    assert torch.all(res[:, cols:] == 7) and torch.all(q[:, cols:] == 99) and scale[5] == -1


@pytest.mark.parametrize("qdtype", [sp24.I8, sp24.E4M3])
@pytest.mark.parametrize("cols", [64, 77, 4096])
def test_rows_zero_tiny_and_not_finite(cols, qdtype):
    x = randn(8, cols, seed=5, dtype=torch.bfloat16)
    x[1] = 0
    x[2] = 0
    x[2, cols // 2] = float("nan")
    x[3, 3] = float("inf")
    x[4, cols - 1] = -float("inf")
    x[5] = x[5] * 2.0 ** -120          # Q / amax would overflow
    x[6] = 0
    x[6, 5] = 2.0 ** -133              # the smallest bf16
    x[7] = x[7] * 2.0 ** 100
    q, s = sp24.quantize_rows(x, qdtype=qdtype)
    for bad in (2, 3, 4):
        assert torch.isnan(s[bad]) and torch.all(q[bad].float() == 0)
    assert s[1] == 0 and torch.all(q[1].float() == 0)
    keep = [0, 1, 5, 7]
    check_rows(q[keep], s[keep], x[keep].double(), qdtype, scale_tol(cols))
    assert q[6].float().abs().max() == QMAX[qdtype] and (q[6].float() != 0).sum() == 1
    # a zero row through the norm and a zero gate through the product
    w = torch.ones(cols, device=DEV, dtype=torch.bfloat16)
    q, s = sp24.rmsnorm_quant(x, w, qdtype=qdtype)
    assert s[1] == 0 and torch.all(q[1].float() == 0)
    assert all(torch.isnan(s[bad]) for bad in (2, 3, 4)) and torch.isfinite(s[[0, 1, 5]]).all()
    q, s = sp24.swiglu_quant(x, x, qdtype=qdtype)
    assert s[1] == 0 and all(torch.isnan(s[bad]) for bad in (2, 3, 4))


def test_norm_whose_squares_leave_fp32():
    """Sums of squares past fp32's range are flagged, not turned into zeroes."""
    x = randn(4, 512, seed=1, dtype=torch.bfloat16)
    x[1] = x[1] * 2.0 ** 90
    x[2] = x[2] * 2.0 ** -90
    w = torch.ones(512, device=DEV, dtype=torch.bfloat16)
    q, s = sp24.rmsnorm_quant(x, w, eps=0.0)
    assert torch.isnan(s[1]) and torch.isnan(s[2]) and torch.all(q[1:3] == 0)
    keep = [0, 3]
    check_rows(q[keep], s[keep], rmsnorm64(x[keep], w, None, 0.0)[1], sp24.I8, scale_tol(512))
    q, s = sp24.rmsnorm_quant(x, w, eps=1e-6)      # tiny rows are eps's business
    check_rows(q[[2]], s[[2]], rmsnorm64(x[[2]], w, None, 1e-6)[1], sp24.I8, scale_tol(512))


def test_rows_no_rows_and_streams():
    q, s, r = sp24.rmsnorm_quant(torch.empty(0, 64, device=DEV, dtype=torch.bfloat16),
                                 torch.ones(64, device=DEV, dtype=torch.bfloat16),
                                 residual=torch.empty(0, 64, device=DEV, dtype=torch.bfloat16))
    assert q.shape == r.shape == (0, 64) and s.shape == (0,)
    x = randn(64, 4096, seed=1, dtype=torch.bfloat16)
    want = sp24.quantize_rows(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = sp24.quantize_rows(x, stream=side)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rows_past_32_bit_offsets():
    rows, cols = 150000, 14400        # 2.16e9 elements
    x = torch.empty(rows, cols, device=DEV, dtype=torch.bfloat16)
    x[:-3] = 1
    x[-3:] = randn(3, cols, seed=4, dtype=torch.bfloat16)
    q, s = sp24.quantize_rows(x)
    check_rows(q[-3:], s[-3:], x[-3:].double(), sp24.I8, scale_tol(cols))
    assert torch.all(q[:8] == 127) and torch.all(q[rows // 2] == 127)


# ------------------------------------------------------------------ scaled product
def weights_2of4(m, k, qdtype, seed):
    """(a_c, tcgen05 image, dense 64-bit weights) with random patterns; a kept
    value may be zero."""
    g = gen(seed)
    order = torch.rand(m, k // 4, 4, device=DEV, generator=g).argsort(dim=2)[:, :, :2]
    at = order.sort(dim=2).values
    if qdtype == sp24.I8:
        vals = torch.randint(-128, 128, (m, k // 4, 2), device=DEV, generator=g).to(torch.int8)
    else:
        vals = (torch.randn(m, k // 4, 2, device=DEV, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    dense = torch.zeros(m, k // 4, 4, device=DEV, dtype=torch.float64).scatter_(2, at, vals.double())
    code = (at[:, :, 0] | at[:, :, 1] << 2).to(torch.uint8)
    meta = (code[:, 0::2] | code[:, 1::2] << 4).contiguous()
    return vals.reshape(m, k // 2), sp24.repack_meta(meta, m, k, qdtype), dense.reshape(m, k)


def tokens_8bit(n, k, qdtype, seed):
    if qdtype == sp24.I8:
        return torch.randint(-128, 128, (n, k), device=DEV, generator=gen(seed)).to(torch.int8)
    return (torch.randn(n, k, device=DEV, generator=gen(seed)) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)


def check_scaled(c, x, w, sw, sx, bias, qdtype, k):
    both = sw.double()[None, :] * sx.double()[:, None]
    xd = x.double()
    y = (xd @ w.t()) * both
    mag = (xd.abs() @ w.abs().t()) * both.abs()
    b = 0.0 if bias is None else bias.double()
    y = y + b
    acc = 0.0 if qdtype == sp24.I8 else k * E
    tol = U[c.dtype] * y.abs() + (acc + 4 * E) * mag + 4 * E * abs(b) + TINY[c.dtype]
    err = (c.double() - y).abs()
    assert torch.all(err <= tol), (err / tol).max().item()
    # and as a whole: independent roundings of the output, the sums' part far below
    assert torch.linalg.norm(c.double() - y) <= (U[c.dtype] + 2e-6) * torch.linalg.norm(y) + 1e-30


@pytest.mark.parametrize("qdtype", [sp24.I8, sp24.E4M3])
@pytest.mark.parametrize("n,m,k", [
    (1, 1, 64), (1, 64, 64), (1, 128, 128), (1, 256, 4096), (1, 300, 192), (2, 1000, 320),
    (7, 129, 64), (8, 128, 256), (9, 257, 1024), (15, 512, 4160), (16, 100, 128), (17, 256, 448),
    (31, 640, 512), (32, 384, 2048), (33, 255, 256), (64, 1024, 1024), (65, 130, 704),
    (100, 2000, 128), (127, 256, 256), (128, 128, 1024), (129, 512, 192), (200, 300, 4096),
    (255, 257, 512), (256, 256, 256), (257, 511, 320), (300, 2304, 1088), (513, 769, 640),
    (1000, 1000, 1024), (64, 4096, 14336), (3, 14336, 4096),
    (33, 14336, 320), (128, 14080, 192), (1000, 14336, 192), (1111, 14081, 320), (2049, 9000, 64)])
def test_scaled_sizes(n, m, k, qdtype):
    a_c, image, w = weights_2of4(m, k, qdtype, seed=m + k)
    x = tokens_8bit(n, k, qdtype, seed=n)
    sw = 10.0 ** (randn(m, seed=3) * 0.3) * 1e-3
    sx = 10.0 ** (randn(n, seed=4) * 0.3) * 1e-2
    bias = randn(m, seed=5)
    for out in (torch.bfloat16, torch.float16, torch.float32):
        small = 1e-2 if out == torch.float16 else 1.0        # fp16's range
        b = bias if (n + m) % 2 else None
        c = sp24.gemm_scaled(a_c, image, x, sw * small, sx, bias=b, out_dtype=out)
        assert c.shape == (n, m) and c.dtype == out
        check_scaled(c, x, w, sw * small, sx, b, qdtype, k)


def test_scaled_int8_is_exact():
    """fp32 outputs of unit scales are the integers themselves."""
    a_c, image, w = weights_2of4(384, 1024, sp24.I8, seed=1)
    for n in (1, 16, 40, 300):
        x = tokens_8bit(n, 1024, sp24.I8, seed=n)
        c = sp24.gemm_scaled(a_c, image, x, out_dtype=torch.float32)
        assert torch.equal(c.double(), x.double() @ w.t())
    # the largest sums: every product 2^14, past 2^24 and past 2^30
    k = 131072
    a_c = torch.full((128, k // 2), -128, device=DEV, dtype=torch.int8)
    image = sp24.repack_meta(torch.full((128, k // 8), 0x44, device=DEV, dtype=torch.uint8), 128, k, sp24.I8)
    for n in (1, 130):
        x = torch.full((n, k), -128, device=DEV, dtype=torch.int8)
        x[:, 0] = 1
        c = sp24.gemm_scaled(a_c, image, x, out_dtype=torch.float32)
        assert torch.all(c == torch.tensor((k // 2 - 1) * 2.0 ** 14 - 128, dtype=torch.float32))


@pytest.mark.parametrize("n", [3, 50, 300])
def test_scaled_strides_and_padding(n):
    m, k = 200, 256
    a_c, image, w = weights_2of4(m, k, sp24.I8, seed=2)
    wide = torch.zeros(m, k // 2 + 48, device=DEV, dtype=torch.int8)
    wide[:, :k // 2] = a_c
    xw = torch.full((n, k + 32), 55, device=DEV, dtype=torch.int8)
    xw[:, :k] = tokens_8bit(n, k, sp24.I8, seed=1)
    sw, sx = torch.rand(m, device=DEV), torch.rand(n, device=DEV)
    c = sp24.gemm_scaled(wide[:, :k // 2], image, xw[:, :k], sw, sx, out_dtype=torch.float32)
    check_scaled(c, xw[:, :k], w, sw, sx, None, sp24.I8, k)
    # rows off the 16-byte grid are staged by the shim
    odd = torch.zeros(n, k + 5, device=DEV, dtype=torch.int8)[:, 3:3 + k]
    odd.copy_(xw[:, :k])
    assert torch.equal(sp24.gemm_scaled(a_c, image, odd, sw, sx, out_dtype=torch.float32), c)
    # an output with odd strides: only its m columns are written
    for dtype, code in ((torch.float16, sp24.F16), (torch.float32, sp24.F32)):
        out = torch.full((n + 1, m + 3), 9.0, device=DEV, dtype=dtype)
        d = sp24.ScaledDesc()
        d.dtype, d.cdtype, d.m, d.n, d.k = sp24.I8, code, m, n, k
        d.a_c, d.meta, d.x, d.ldx = a_c.data_ptr(), image.data_ptr(), xw.data_ptr(), k + 32
        sws = sw * 1e-3
        d.scale_m, d.scale_n = sws.data_ptr(), sx.data_ptr()
        d.c, d.ldc = out.data_ptr() + out.element_size(), m + 3
        assert sp24.load().sp24_gemm_scaled(ctypes.byref(d), torch.cuda.current_stream().cuda_stream) == 0
        flat = out.reshape(-1)[1:]
        check_scaled(flat[:n * (m + 3)].view(n, m + 3)[:, :m], xw[:, :k], w, sws, sx, None, sp24.I8, k)
        edge = flat[:n * (m + 3)].view(n, m + 3)[:, m:]
        assert torch.all(edge == 9) and torch.all(flat[n * (m + 3):] == 9) and out[0, 0] == 9


@pytest.mark.parametrize("qdtype", [sp24.I8, sp24.E4M3])
def test_scaled_is_reproducible_and_stream_ordered(qdtype):
    for n, m, k in ((1, 4096, 4096), (24, 512, 8192), (200, 700, 2048)):
        a_c, image, _ = weights_2of4(m, k, qdtype, seed=1)
        x = tokens_8bit(n, k, qdtype, seed=2)
        want = sp24.gemm_scaled(a_c, image, x, out_dtype=torch.float32)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for _ in range(3):
            got = sp24.gemm_scaled(a_c, image, x, out_dtype=torch.float32, stream=side)
            side.synchronize()
            assert torch.equal(got, want)
    assert sp24.gemm_scaled(a_c, image, x[:0]).shape == (0, m)


def test_scaled_nan_token_stays_in_its_row():
    """A row whose quantisation met a NaN has scale NaN: its products are NaN,
    its neighbours' are not."""
    xb = randn(20, 256, seed=1, dtype=torch.bfloat16)
    xb[7, 3] = float("nan")
    q, s = sp24.quantize_rows(xb)
    a_c, image, _ = weights_2of4(256, 256, sp24.I8, seed=1)
    c = sp24.gemm_scaled(a_c, image, q, None, s)
    assert torch.isnan(c[7]).all() and torch.isfinite(torch.cat((c[:7], c[8:]))).all()


# ------------------------------------------------------------------ gated feed-forward
def ffn64(x, wg, wu, act):
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    s = torch.sigmoid(g)
    if act == sp24.ACT_SILU:
        a, da = g * s, s * (1 + g * (1 - s))
    elif act == sp24.ACT_GELU_TANH:
        c = (2 / torch.pi) ** 0.5
        t = torch.tanh(c * (g + 0.044715 * g ** 3))
        a = 0.5 * g * (1 + t)
        da = 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)
    else:
        a, da = g, torch.ones_like(g)
    return g, u, a, da


def ffn_inputs(t, h, f, dtype, seed=0):
    return (randn(t, h, seed=seed, dtype=dtype), randn(f, h, seed=seed + 1, std=0.7 / h ** 0.5, dtype=dtype),
            randn(f, h, seed=seed + 2, std=0.7 / h ** 0.5, dtype=dtype), randn(t, f, seed=seed + 3, dtype=dtype))


def check_ffn(x, wg, wu, dh, act, out, grads=None):
    u, tiny = U[x.dtype], TINY[x.dtype]
    t, h = x.shape
    f = wg.shape[0]
    g64, u64, a, da = ffn64(x, wg, wu, act)
    X, WG, WU = x.double().abs(), wg.double().abs(), wu.double().abs()
    eg, eu = (h + 8) * E * (X @ WG.t()), (h + 8) * E * (X @ WU.t())   # of the sums g and u
    # |act'| <= 1.1 and |act''| <= 0.5 for silu, 1.13 and 0.8 for gelu; the
    # activation's own fp32 error is 16 e
    d1, d2 = (1.13, 0.8) if act == sp24.ACT_GELU_TANH else (1.1, 0.5)
    eh = d1 * eg * (u64.abs() + eu) + (a.abs() + d1 * eg) * eu + 16 * E * (a * u64).abs()
    y = a * u64
    err = (out.double() - y).abs()
    assert torch.all(err <= u * y.abs() * (1 + 1e-3) + 1.01 * eh + tiny)
    assert torch.linalg.norm(out.double() - y) <= (u + 1e-5) * torch.linalg.norm(y) + tiny * (t * f) ** 0.5
    if grads is None:
        return
    D = dh.double()
    dg, du = D * u64 * da, D * a
    edg = D.abs() * (d2 * eg * (u64.abs() + eu) + d1 * eu + 16 * E * u64.abs()) + u * dg.abs() * 1.01 + tiny
    edu = D.abs() * (d1 * eg + 16 * E * a.abs()) + u * du.abs() * 1.01 + tiny
    dx, dwg, dwu = grads
    S = (dg.abs() + edg) @ WG + (du.abs() + edu) @ WU
    for got, want, tol in (
            (dx, dg @ wg.double() + du @ wu.double(), edg @ WG + edu @ WU + (2 * f + 8) * E * S),
            (dwg, dg.t() @ x.double(), edg.t() @ X + (t + 8) * E * ((dg.abs() + edg).t() @ X)),
            (dwu, du.t() @ x.double(), edu.t() @ X + (t + 8) * E * ((du.abs() + edu).t() @ X))):
        if got is None:
            continue
        err = (got.double() - want).abs()
        bound = u * want.abs() * 1.01 + tol + tiny
        assert torch.all(err <= bound), (err / bound).max().item()
        # dg's and du's rounding and the output's, independent of each other
        assert torch.linalg.norm(got.double() - want) <= (2 * u + 1e-4) * torch.linalg.norm(want) + \
            tiny * got.numel() ** 0.5


@pytest.mark.parametrize("act", [sp24.ACT_SILU, sp24.ACT_NONE])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,h,f", [(1, 8, 8), (1, 64, 128), (1, 1000, 264), (2, 72, 1000), (5, 136, 96), (8, 256, 512),
                                   (16, 4096, 640), (17, 200, 200), (31, 512, 72), (33, 64, 2744), (64, 1024, 256),
                                   (65, 128, 128), (100, 264, 1032), (128, 256, 256), (129, 512, 136), (257, 320, 512),
                                   (300, 1000, 776), (513, 256, 1024),
                                   (1300, 1280, 264), (1030, 1000, 136), (2600, 264, 512),
                                   (33, 72, 14336), (100, 264, 15000), (129, 200, 18888), (256, 64, 16384),
                                   (300, 2056, 400), (700, 1032, 264), (1200, 1544, 744)])
def test_ffn_sizes(t, h, f, dtype, act):
    x, wg, wu, dh = ffn_inputs(t, h, f, dtype, seed=t + h)
    out, saved = sp24.ffn_gated(x, wg, wu, act=act, save=True)
    grads = sp24.ffn_gated_backward(dh, x, wg, wu, saved, act=act)
    check_ffn(x, wg, wu, dh, act, out, grads)
    assert torch.equal(sp24.ffn_gated(x, wg, wu, act=act), out) or t <= 128
    check_ffn(x, wg, wu, dh, act, sp24.ffn_gated(x, wg, wu, act=act))


@pytest.mark.parametrize("t,h,f", [(3, 37, 51), (40, 129, 100), (200, 77, 333)])
def test_ffn_odd_widths(t, h, f):
    """Widths whose rows are not 16-byte multiples: staged by the shim."""
    x, wg, wu, dh = ffn_inputs(t, h, f, torch.bfloat16)
    out, saved = sp24.ffn_gated(x, wg, wu, save=True)
    check_ffn(x, wg, wu, dh, sp24.ACT_SILU, out, sp24.ffn_gated_backward(dh, x, wg, wu, saved))


@pytest.mark.parametrize("t", [6, 140])
def test_ffn_strides_padding_and_partial_gradients(t):
    h, f, dtype = 120, 72, torch.float16
    x, wg, wu, dh = ffn_inputs(t, h, f, dtype, seed=3)
    xs, wgs, wus, dhs = (torch.full((v.shape[0], v.shape[1] + 16), 77.0, device=DEV, dtype=dtype) for v in (x, wg, wu, dh))
    for s, v in ((xs, x), (wgs, wg), (wus, wu), (dhs, dh)):
        s[:, :v.shape[1]] = v
    out, saved = sp24.ffn_gated(xs[:, :h], wgs[:, :h], wus[:, :h], save=True)
    full = sp24.ffn_gated_backward(dhs[:, :f], xs[:, :h], wgs[:, :h], wus[:, :h], saved)
    check_ffn(x, wg, wu, dh, sp24.ACT_SILU, out, full)
    dx, none_g, none_u = sp24.ffn_gated_backward(dh, x, wg, wu, saved, need_dw=False)
    assert none_g is None and none_u is None and torch.equal(dx, full[0])
    none_x, dwg, dwu = sp24.ffn_gated_backward(dh, x, wg, wu, saved, need_dx=False)
    assert none_x is None and torch.equal(dwg, full[1]) and torch.equal(dwu, full[2])
    # outputs with odd strides and starts: only their own elements are written
    lib, stream = sp24.load(), torch.cuda.current_stream().cuda_stream
    d = sp24.FfnDesc()
    d.dtype, d.t, d.h, d.f, d.act = sp24.F16, t, h, f, sp24.ACT_SILU
    d.x, d.w_gate, d.w_up = x.data_ptr(), wg.data_ptr(), wu.data_ptr()
    o = torch.full((t, f + 3), 9.0, device=DEV, dtype=dtype)
    assert lib.sp24_ffn_forward(ctypes.byref(d), o.data_ptr() + 2, f + 3, stream) == 0
    d.saved, d.saved_bytes = saved.data_ptr(), saved.numel()
    g = sp24.FfnGrads()
    ws = torch.empty(lib.sp24_ffn_workspace_bytes(t, h, f), dtype=torch.uint8, device=DEV)
    bufs = [torch.full((r, h + 5), 9.0, device=DEV, dtype=dtype) for r in (t, f, f)]
    g.d_out, g.dx, g.dw_gate, g.dw_up = (v.data_ptr() for v in [dh] + bufs)
    g.ld_dx = g.ld_dgate = g.ld_dup = h + 5
    g.workspace, g.workspace_bytes = ws.data_ptr(), ws.numel()
    assert lib.sp24_ffn_backward(ctypes.byref(d), ctypes.byref(g), stream) == 0
    torch.cuda.synchronize()
    flat = o.reshape(-1)
    check_ffn(x, wg, wu, dh, sp24.ACT_SILU, torch.stack([flat[1 + i * (f + 3):1 + i * (f + 3) + f] for i in range(t)]))
    assert flat[0] == 9 and (flat == 9).sum() >= 3 * t
    for b, want in zip(bufs, full):
        assert torch.equal(b[:, :h], want) and torch.all(b[:, h:] == 9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,h,f", [(1, 64, 136), (40, 264, 14336), (90, 512, 256), (200, 1024, 264), (300, 320, 512),
                                   (1100, 128, 2000)])
def test_ffn_gelu(t, h, f, dtype):
    """The tanh form of gelu through every forward kernel, and its gradients."""
    x, wg, wu, dh = ffn_inputs(t, h, f, dtype, seed=t)
    x[0] *= 40                       # gates far into both tails
    out, saved = sp24.ffn_gated(x, wg, wu, act=sp24.ACT_GELU_TANH, save=True)
    grads = sp24.ffn_gated_backward(dh, x, wg, wu, saved, act=sp24.ACT_GELU_TANH)
    check_ffn(x, wg, wu, dh, sp24.ACT_GELU_TANH, out, grads)
    check_ffn(x, wg, wu, dh, sp24.ACT_GELU_TANH, sp24.ffn_gated(x, wg, wu, act=sp24.ACT_GELU_TANH))


def test_ffn_no_tokens():
    _, wg, wu, _ = ffn_inputs(1, 64, 96, torch.bfloat16)
    x, dh = (torch.empty(0, n, device=DEV, dtype=torch.bfloat16) for n in (64, 96))
    out, saved = sp24.ffn_gated(x, wg, wu, save=True)
    dx, dwg, dwu = sp24.ffn_gated_backward(dh, x, wg, wu, saved)
    assert out.shape == (0, 96) and dx.shape == (0, 64)
    assert torch.all(dwg == 0) and torch.all(dwu == 0) and dwg.shape == (96, 64)


def test_ffn_extreme_gates():
    """silu and its derivative at both ends, zeroes, and NaN kept to its own
    token (and to every weight gradient, which sums over tokens)."""
    h, f = 64, 64
    x = torch.zeros(6, h, device=DEV, dtype=torch.bfloat16)
    x[0, 0], x[1, 0], x[2, 0], x[4, 0] = 300.0, -300.0, -3e4, float("nan")
    wg = torch.ones(f, h, device=DEV, dtype=torch.bfloat16)
    wu = torch.ones(f, h, device=DEV, dtype=torch.bfloat16)
    out, saved = sp24.ffn_gated(x, wg, wu, save=True)
    dh = torch.ones(6, f, device=DEV, dtype=torch.bfloat16)
    dx, dwg, dwu = sp24.ffn_gated_backward(dh, x, wg, wu, saved)
    ok = [0, 1, 2, 3, 5]
    xs = x[ok]
    check_ffn(xs, wg, wu, dh[ok], sp24.ACT_SILU, out[ok], (dx[ok], None, None))
    assert torch.isnan(out[4]).all() and torch.isnan(dx[4]).all()
    assert torch.isfinite(out[ok].float()).all() and torch.isfinite(dx[ok].float()).all()
    assert torch.isnan(dwg[:, 0]).all() and torch.isnan(dwu[:, 0]).all()


@pytest.mark.parametrize("act", [sp24.ACT_SILU, sp24.ACT_GELU_TANH, sp24.ACT_NONE])
def test_ffn_gradients_against_differences(act):
    """Directional derivatives of the 64-bit formula by central differences
    (error eps^2 / 6 of the third derivative, about 1e-9 here), against the
    kernel's gradients: each inner product sums n values that carry two
    roundings of relative size u, of either sign."""
    t, h, f = 70, 96, 160
    x, wg, wu, dh = ffn_inputs(t, h, f, torch.bfloat16, seed=9)
    _, saved = sp24.ffn_gated(x, wg, wu, act=act, save=True)
    grads = sp24.ffn_gated_backward(dh, x, wg, wu, saved, act=act)

    def loss(x, wg, wu):
        g, u, a, _ = ffn64(x, wg, wu, act)
        return (a * u * dh.double()).sum()

    at = [x.double(), wg.double(), wu.double()]
    for i, got in enumerate(grads):
        v = torch.randn(at[i].shape, device=DEV, dtype=torch.float64, generator=gen(20 + i))
        eps = 1e-4 / v.abs().max()
        lo, hi = list(at), list(at)
        lo[i], hi[i] = at[i] - eps * v, at[i] + eps * v
        want = (loss(*hi) - loss(*lo)) / (2 * eps)
        noise = U[torch.bfloat16] * torch.linalg.norm(got.double() * v)
        assert (got.double() * v).sum().sub(want).abs() <= 2 * 6 * noise + 1e-6 * want.abs()


def test_ffn_streams_and_repeats():
    x, wg, wu, dh = ffn_inputs(300, 512, 768, torch.bfloat16)
    out, saved = sp24.ffn_gated(x, wg, wu, save=True)
    want = sp24.ffn_gated_backward(dh, x, wg, wu, saved)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        o, s = sp24.ffn_gated(x, wg, wu, save=True, stream=side)
        got = sp24.ffn_gated_backward(dh, x, wg, wu, s, stream=side)
        side.synchronize()
        assert torch.equal(o, out) and all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("qdtype,bound", [(sp24.I8, 0.05), (sp24.E4M3, 0.12)])
def test_example_trains_and_serves(qdtype, bound):
    """examples/mlp_block.py.  Served error: four roundings to 8 bits (two of
    activations, two of weights) in quadrature.  int8 rows of normal values
    (largest near 4 sigma) are off by 4 / 127 / sqrt(12) = 0.9% each; e4m3 by up to
    2^-4 / sqrt(3) = 3.6% each, less on average; doubled for the norm's and the
    gate's amplification."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "mlp_block.py")
    spec = importlib.util.spec_from_file_location("mlp_block", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, errors = example.run(tokens=200, hidden=512, inter=1408, qdtype=qdtype)
    assert all(b < a for a, b in zip(losses, losses[1:])), losses
    assert all(e <= bound for e in errors.values()), errors


def test_shim_refuses_wrong_types_and_shapes():
    bf = lambda *s: torch.zeros(*s, device=DEV, dtype=torch.bfloat16)  # noqa: E731
    i8 = lambda *s: torch.zeros(*s, device=DEV, dtype=torch.int8)  # noqa: E731
    image = torch.zeros(sp24.meta_tc_bytes(128, 128), device=DEV, dtype=torch.uint8)
    for call in (lambda: sp24.quantize_rows(bf(4, 64), qdtype=sp24.E5M2),
                 lambda: sp24.quantize_rows(bf(4, 64).float()),
                 lambda: sp24.quantize_rows(bf(64)),
                 lambda: sp24.swiglu_quant(bf(4, 64), bf(4, 64).half()),
                 lambda: sp24.swiglu_quant(bf(4, 64), bf(4, 72)),
                 lambda: sp24.rmsnorm_quant(bf(4, 64), bf(72)),
                 lambda: sp24.rmsnorm_quant(bf(4, 64), bf(64), bf(5, 64)),
                 lambda: sp24.gemm_scaled(i8(128, 64), image, bf(4, 128)),
                 lambda: sp24.gemm_scaled(i8(128, 64), image, i8(4, 64)),
                 lambda: sp24.gemm_scaled(i8(128, 64), image[:-16], i8(4, 128)),
                 lambda: sp24.gemm_scaled(i8(128, 64), image, i8(4, 128), torch.ones(127, device=DEV)),
                 lambda: sp24.gemm_scaled(i8(128, 64), image, i8(4, 128), bf(128)),
                 lambda: sp24.gemm_scaled(i8(128, 64), image, i8(4, 128), out_dtype=torch.int8),
                 lambda: sp24.gemm_scaled(i8(128, 64), image, torch.zeros(4, 128, dtype=torch.int8)),
                 lambda: sp24.ffn_gated(bf(4, 64), bf(96, 64), bf(96, 64).half()),
                 lambda: sp24.ffn_gated(bf(4, 64), bf(96, 64), bf(88, 64)),
                 lambda: sp24.ffn_gated(bf(4, 64), bf(96, 72), bf(96, 72)),
                 lambda: sp24.ffn_gated_backward(bf(4, 88), bf(4, 64), bf(96, 64), bf(96, 64), image)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(sp24.Sp24Error):      # k % 64
        sp24.gemm_scaled(i8(128, 16), image[:2 * 2048], i8(4, 32))
    with pytest.raises(sp24.Sp24Error):      # a saved buffer of another call
        sp24.ffn_gated_backward(bf(4, 96), bf(4, 64), bf(96, 64), bf(96, 64), image[:64])


def test_static_weight_hint_and_graphs_keep_results():
    """SP24_HINT_STATIC_WEIGHTS only moves weight loads ahead of the wait for the
    previous kernel; a captured call replays on new inputs.  The tokens are
    written by the kernel just before each product."""
    a_c, image, w = weights_2of4(512, 1024, sp24.I8, seed=1)
    wg, wu = (randn(512, 1024, seed=s, std=0.02, dtype=torch.bfloat16) for s in (2, 3))
    for n in (1, 40, 300):
        xs = [randn(n, 1024, seed=10 + i, dtype=torch.bfloat16) for i in range(3)]

        def chain(x):
            q, s = sp24.quantize_rows(x)
            return sp24.gemm_scaled(a_c, image, q, None, s, out_dtype=torch.float32), sp24.ffn_gated(x, wg, wu)

        want = [chain(x) for x in xs]
        sp24.set_launch_hints(sp24.HINT_STATIC_WEIGHTS)
        try:
            got = [chain(x) for x in xs]
        finally:
            sp24.set_launch_hints(sp24.HINT_NONE)
        assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q))
        x = xs[0].clone()
        side = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            out = chain(x)
        for i in (1, 2):
            x.copy_(xs[i])
            graph.replay()
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])


def test_calls_from_several_threads():
    """First calls on a device may come from several host threads at once, each
    on its own stream: results as from one."""
    import threading
    a_c, image, _ = weights_2of4(640, 512, sp24.E4M3, seed=1)
    wg, wu = (randn(384, 512, seed=s, std=0.02, dtype=torch.float16) for s in (2, 3))
    xs = [randn(n, 512, seed=n, dtype=torch.float16) for n in (1, 70, 200, 400)]

    def work(x, stream=None):
        q, s = sp24.quantize_rows(x, qdtype=sp24.E4M3, stream=stream)
        return sp24.gemm_scaled(a_c, image, q, None, s, stream=stream), sp24.ffn_gated(x, wg, wu, stream=stream)

    want = [work(x) for x in xs]
    torch.cuda.synchronize()
    got = [None] * len(xs)

    def run(i):
        stream = torch.cuda.Stream()
        for _ in range(20):
            got[i] = work(xs[i], stream)
        stream.synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for p, q in zip(got, want) for a, b in zip(p, q))


def test_products_past_32_bit_offsets():
    """Outputs of more than 2^31 elements: the last rows, and the rows around the
    element 2^31."""
    n, wide, k = 150001, 14400, 64
    at = torch.tensor([0, 2 ** 31 // wide - 1, 2 ** 31 // wide, 2 ** 31 // wide + 1, n - 2, n - 1], device=DEV)
    a_c, image, w = weights_2of4(wide, k, sp24.I8, seed=1)
    x = tokens_8bit(n, k, sp24.I8, seed=2)
    sw, sx = torch.rand(wide, device=DEV) * 1e-3, torch.rand(n, device=DEV)
    c = sp24.gemm_scaled(a_c, image, x, sw, sx)
    check_scaled(c[at], x[at], w, sw, sx[at], None, sp24.I8, k)
    del c
    xb = randn(n, k, seed=3, dtype=torch.bfloat16)
    wg, wu = (randn(wide, k, seed=s, std=0.09, dtype=torch.bfloat16) for s in (4, 5))
    h, saved = sp24.ffn_gated(xb, wg, wu, save=True)
    dh = torch.zeros_like(h)
    dh[at] = randn(len(at), wide, seed=6, dtype=torch.bfloat16)
    dx, dwg, dwu = sp24.ffn_gated_backward(dh, xb, wg, wu, saved)
    # only the chosen tokens carry a gradient, so these are the whole sums
    check_ffn(xb[at], wg, wu, dh[at], sp24.ACT_SILU, h[at], (dx[at], None, None))
    few = sp24.ffn_gated(xb[at], wg, wu, save=True)[1]
    _, eg, eu = sp24.ffn_gated_backward(dh[at].contiguous(), xb[at], wg, wu, few, need_dx=False)
    assert torch.allclose(dwg.float(), eg.float(), rtol=2 ** -7, atol=1e-6)
    assert torch.allclose(dwu.float(), eu.float(), rtol=2 ** -7, atol=1e-6)


def test_inputs_freed_right_after_a_call_on_another_stream():
    """A named stream's inputs may be freed at once: their memory is not handed
    out again before the kernel has read it."""
    side = torch.cuda.Stream()
    want = sp24.quantize_rows(randn(4096, 4096, seed=1, dtype=torch.bfloat16))
    torch.cuda.synchronize()
    for _ in range(10):
        x = randn(4096, 4096, seed=1, dtype=torch.bfloat16)
        side.wait_stream(torch.cuda.current_stream())
        big = [sp24.quantize_rows(x, stream=side) for _ in range(4)]
        del x
        junk = torch.full((4096, 4096), 3.0, device=DEV, dtype=torch.bfloat16)
        side.synchronize()
        assert all(torch.equal(q, want[0]) and torch.equal(s, want[1]) for q, s in big)
        del junk


@pytest.mark.parametrize("t,f", [(1, 8), (3, 72), (5, 264), (70, 776), (4, 51), (2, 128)])
def test_ffn_backward_touches_no_column_past_f(t, f):
    """dg and du are formed from the columns of d_out that exist: what the
    workspace holds past them stays as it was (units of eight columns, rows of
    64), and NaN beside d_out's rows reaches no gradient."""
    h, ld = 64, (f + 63) // 64 * 64
    x, wg, wu, dh = ffn_inputs(t, h, f, torch.float16, seed=f)
    out, saved = sp24.ffn_gated(x, wg, wu, save=True)
    wide = torch.full((t, f + 64), float("nan"), device=DEV, dtype=torch.float16)
    wide[:, :f] = dh
    lib, stream = sp24.load(), torch.cuda.current_stream().cuda_stream
    d = sp24.FfnDesc()
    d.dtype, d.t, d.h, d.f, d.act = sp24.F16, t, h, f, sp24.ACT_SILU
    d.x, d.w_gate, d.w_up = x.data_ptr(), wg.data_ptr(), wu.data_ptr()
    d.saved, d.saved_bytes = saved.data_ptr(), saved.numel()
    size = lib.sp24_ffn_workspace_bytes(t, h, f)
    for d_out, ldd in ((dh, f), (wide, f + 64)):
        ws = torch.full((size // 2,), 0x5A5A, device=DEV, dtype=torch.int16)
        dx, dwg, dwu = (torch.empty(r, h, device=DEV, dtype=torch.float16) for r in (t, f, f))
        g = sp24.FfnGrads()
        g.d_out, g.ld_d_out = d_out.data_ptr(), ldd
        g.dx, g.dw_gate, g.dw_up = (v.data_ptr() for v in (dx, dwg, dwu))
        g.workspace, g.workspace_bytes = ws.data_ptr(), size
        assert lib.sp24_ffn_backward(ctypes.byref(d), ctypes.byref(g), stream) == 0
        check_ffn(x, wg, wu, dh, sp24.ACT_SILU, out, (dx, dwg, dwu))
        planes = ws[:2 * t * ld].view(2, t, ld)
        assert torch.all(planes[:, :, (f + 7) // 8 * 8:] == 0x5A5A)


@pytest.mark.parametrize("n", [1, 60, 300])
def test_static_weight_hint_with_weights_that_are_copied(n):
    """Under the hint, weights whose rows are off the 16-byte grid: the shim's
    copies are made just before each product, over memory that held others."""
    h, f, m, k = 1004, 520, 300, 256
    x = randn(n, h, seed=1, dtype=torch.bfloat16)
    pairs = [[randn(f, h, seed=10 * i + j, std=0.02, dtype=torch.bfloat16) for j in (2, 3)] for i in range(3)]
    packed = [weights_2of4(m, k, sp24.I8, seed=i)[:2] for i in range(3)]
    odd = [torch.zeros(m, k // 2 + 4, device=DEV, dtype=torch.int8)[:, :k // 2].copy_(a) for a, _ in packed]
    q = tokens_8bit(n, k, sp24.I8, seed=4)

    def products():
        return [(sp24.ffn_gated(x, *w), sp24.gemm_scaled(a, image, q, out_dtype=torch.float32))
                for w, a, (_, image) in zip(pairs, odd, packed)]

    want = products()
    torch.cuda.synchronize()
    sp24.set_launch_hints(sp24.HINT_STATIC_WEIGHTS)
    try:
        for _ in range(5):
            assert all(torch.equal(a, b) for p, r in zip(products(), want) for a, b in zip(p, r))
        assert sp24.get_launch_hints() == sp24.HINT_STATIC_WEIGHTS
    finally:
        sp24.set_launch_hints(sp24.HINT_NONE)


@pytest.mark.parametrize("cols", [100, 512, 1001, 4096, 40001])
def test_norm_whose_squares_are_subnormal(cols):
    """Sums of squares that lose digits below 2^-126 are flagged too, in every
    form of the kernel; rows just above, and rows whose eps carries the sum, are
    right to the usual tolerance."""
    powers = (-60, -62, -65, -69, -72, -73, -75)
    x = randn(1, cols, seed=1, dtype=torch.bfloat16).repeat(len(powers) + 1, 1)
    for i, e in enumerate(powers):
        x[i] = x[i] * 2.0 ** e
    x[-1] = 0
    w = (1 + randn(cols, seed=2, std=0.1)).to(torch.bfloat16)
    mean = x.double().square().mean(dim=1)
    bad = (mean > 0) & (mean < 2.0 ** -126)
    assert bad.tolist() == [False, False] + [True] * 5 + [False]
    q, s = sp24.rmsnorm_quant(x, w, eps=0.0)
    assert torch.equal(torch.isnan(s), bad) and torch.all(q[bad] == 0) and s[-1] == 0
    check_rows(q[:2], s[:2], rmsnorm64(x[:2], w, None, 0.0)[1], sp24.I8, scale_tol(cols))
    eps = 2.0 ** -125
    q, s = sp24.rmsnorm_quant(x, w, eps=eps)
    check_rows(q, s, rmsnorm64(x, w, None, eps)[1], sp24.I8, scale_tol(cols))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,h,f", [(1, 8, 8), (1, 4096, 640), (5, 136, 96), (16, 1000, 264), (33, 64, 2744), (64, 1024, 256),
                                   (100, 264, 1032), (128, 256, 256), (40, 264, 14336), (128, 72, 15000)])
def test_ffn_few_tokens_repeat_exactly(t, h, f, dtype):
    """Up to 128 tokens too, a call gives the same bits every time, with g and u
    saved or not: neither the kernel nor its split of K depends on that."""
    x, wg, wu, _ = ffn_inputs(t, h, f, dtype, seed=t)
    want, saved = sp24.ffn_gated(x, wg, wu, save=True)
    for _ in range(3):
        out, again = sp24.ffn_gated(x, wg, wu, save=True)
        assert torch.equal(out, want) and torch.equal(sp24.ffn_gated(x, wg, wu), want)
        # rows of f sums, padded to 64: the padding is not written
        planes, first = (s.view(torch.float32).view(2, t, -1)[:, :, :f] for s in (again, saved))
        assert torch.equal(planes, first)
