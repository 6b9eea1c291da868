"""The block-scaled (MX) operators against plain 64-bit statements of the same operators (mx_oracle): quantisation exactly,
everything else to bounds that are derived where they stand."""
import ctypes

import pytest
import torch

import mx_oracle as O

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# the norm: the sum is taken in fp64, the value is multiplied twice and s is a sum in fp32: 3 2^-24 and the two-part
# reciprocal root 2^-40, far below the bound that an fp32 sum would need, (72 / 2 + 5) 2^-24 < 2^-18
NORM_REL = 2.0 ** -18
# the gate, |x| <= 12: the exponential's argument x^2 / 2 <= 72 is rounded once, and once more when it is taken to base 2:
# 144 2^-24 relative in the result; the fitted polynomial adds 11 2^-24, the reciprocal and the products 10: < 2^-16
GATE_REL = 2.0 ** -16


def ops():
    from stablediffusion_amd import ops
    return ops


def data(rows, k, seed, dtype="bf16", loud=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, k, generator=g)
    if loud and rows:
        x *= torch.exp(2 * torch.randn(rows, 1, generator=g))
        x[:, torch.randint(0, k, (1 + k // 50,), generator=g)] *= 30.0
        x[rows // 2, : k // 2 + 1] = 0.0                       # blocks of zeros
    return x.clamp(-6e4, 6e4).to(TYPES[dtype])


def strided(x, dev, pad):
    """x on the device as a column slice of a wider buffer (pad 0: as it is); the rest of the buffer is NaN."""
    if not pad:
        return x.to(dev)
    wide = torch.full((x.shape[0], x.shape[1] + pad), float("nan"), dtype=x.dtype)
    off = pad // 2
    wide[:, off:off + x.shape[1]] = x
    return wide.to(dev)[:, off:off + x.shape[1]]


def within(got, want, rel, dtype):
    """got (of `dtype`) is a rounding of values within `rel` of want: half a step of the type on top, and half a step of its
    subnormals."""
    fi = torch.finfo(dtype)
    tol = want.abs() * (rel + fi.eps / 2 * (1 + rel)) + fi.smallest_normal * fi.eps / 2
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"largest excess {float((off - tol).max()):.3e} at tolerance {float(tol.max()):.3e}"


# ----------------------------------------------------------------------------- quantisation


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("rows,k,dtype,pad", [(1, 1, "bf16", 0), (1, 32, "f16", 0), (3, 31, "f32", 0), (17, 33, "bf16", 0), (16, 128, "bf16", 8),
                                              (5, 129, "f16", 0), (33, 512, "f32", 4), (9, 515, "bf16", 3), (2, 1283, "f16", 5), (40, 1280, "bf16", 16)])
def test_quantise_is_the_definition(dev, fmt, rows, k, dtype, pad):
    x = data(rows, k, rows * 1000 + k, dtype)
    q = ops().mx_quantize(strided(x, dev, pad), fmt)
    want = O.values(x.double(), fmt)
    assert torch.equal(ops().mx_dequantize(q).double().cpu(), want)
    assert torch.equal(ops().mx_dequantize(q, torch.bfloat16).double().cpu(), want)
    # the layout: codes in planes of 64 bytes a row, scale bytes [ceil(K / 128), rows, 4], codes past K zero
    e = torch.zeros(rows, q.scales.shape[0] * 4, dtype=torch.int64)
    have = O.scale_exponents(x.double(), fmt) + 127
    e[:, : have.shape[1]] = have
    assert torch.equal(q.scales.cpu().permute(1, 0, 2).reshape(rows, -1).long(), e)
    assert q.codes.shape == (q.scales.shape[0] * (2 if fmt == "mxfp8" else 1), rows, 64)
    per = 1 if fmt == "mxfp8" else 2
    assert int(q.codes.permute(1, 0, 2).reshape(rows, -1)[:, -(-k // per):].cpu().count_nonzero()) == 0


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_quantise_ties_ends_and_poison(dev, fmt):
    """Every midpoint between neighbours, subnormal and largest inputs, zeros of both signs, and NaN or infinity in a block."""
    emax, emin, digits, most = O.FORMATS[fmt]
    x = torch.zeros(8, 64)
    ties = torch.arange(0, 31) * 2.0 ** (emin - digits - 1)
    x[0, :31], x[0, 31] = ties, most
    x[1, :32] = torch.linspace(-most * 1.14, most * 1.14, 32)             # values that saturate
    x[2, :32] = torch.arange(32) * 2.0 ** -149                            # fp32 subnormals
    x[3, :32] = torch.linspace(1e38, 3.4e38, 32)
    x[4, :32] = -0.0
    x[5, 3], x[5, 40] = float("nan"), 2.0
    x[6, 5], x[6, 41] = float("-inf"), 3.0
    x[7, :32] = 2.0 ** -126 * torch.arange(32)
    q = ops().mx_quantize(x.to(dev), fmt)
    got, want = ops().mx_dequantize(q).double().cpu(), O.values(x.double(), fmt)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and int(torch.isnan(want).sum()) == 64
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_quantise_shapes_and_empty(dev):
    o = ops()
    x = data(12, 96, 5).to(dev)
    q = o.mx_quantize(x.view(3, 4, 96), "mxfp8")
    assert tuple(q.shape) == (3, 4, 96) and o.mx_dequantize(q).shape == (3, 4, 96)
    assert torch.equal(o.mx_dequantize(q).view(12, 96), o.mx_dequantize(o.mx_quantize(x, "mxfp8")))
    assert torch.equal(o.mx_dequantize(o.mx_quantize(x[::3], "mxfp4")), o.mx_dequantize(o.mx_quantize(x[::3].contiguous(), "mxfp4")))
    assert o.mx_dequantize(o.mx_quantize(x[:0], "mxfp4")).shape == (0, 96)
    one = o.mx_quantize(x[0], "mxfp8")
    assert o.mx_dequantize(one).shape == (96,)


# ----------------------------------------------------------------------------- RMS norm


@pytest.mark.parametrize("fmt", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("rows,c,dtype,pad,res", [(1, 1, "bf16", 0, True), (1, 1280, "bf16", 0, True), (5, 33, "f16", 3, False), (7, 512, "f32", 0, True),
                                                  (6, 520, "bf16", 8, True), (9, 1027, "f16", 5, True), (3, 2056, "bf16", 0, False),
                                                  (4, 5120, "bf16", 0, True), (2, 8192, "f32", 4, True), (2, 16384, "f16", 0, True)])
def test_rmsnorm(dev, fmt, rows, c, dtype, pad, res):
    x = data(rows, c, c, dtype)
    r = data(rows, c, c + 1, dtype) if res else None
    gamma = 1 + 0.2 * torch.randn(c, generator=torch.Generator().manual_seed(c))
    y = ops().rmsnorm(strided(x, dev, pad), gamma.to(dev), 1e-5, res=strided(r, dev, pad) if res else None, fmt=fmt)
    s = x.float()
    if res:
        y, stream = y
        s = x.float() + r.float()
        assert stream.dtype == x.dtype and torch.equal(stream.cpu(), s.to(x.dtype))
    want = O.rmsnorm(s.double(), gamma.double(), 1e-5)
    if fmt is None:
        assert y.dtype == x.dtype
        within(y, want, NORM_REL, x.dtype)
    else:
        assert O.held_within(ops().mx_dequantize(y).double().cpu(), want, NORM_REL, fmt)


@pytest.mark.parametrize("fmt", [None, "mxfp8"])
def test_rmsnorm_rows_of_zeros_poison_and_types(dev, fmt):
    o = ops()
    x = data(6, 320, 1, "f32", loud=False)
    x[1] = 0.0
    x[3, 7] = float("nan")
    gamma = torch.ones(320, device=dev)
    y = o.rmsnorm(x.to(dev), gamma, 1e-6, fmt=fmt)
    y = (y if fmt is None else o.mx_dequantize(y)).cpu()
    assert torch.equal(y[1], torch.zeros(320)) and bool(torch.isnan(y[3]).all()) and bool(torch.isfinite(y[[0, 1, 2, 4, 5]]).all())
    if fmt is None:
        within(o.rmsnorm(x[:1].to(dev), gamma, 1e-6, out_dtype=torch.float16), O.rmsnorm(x[:1].double(), torch.ones(320).double(), 1e-6),
               NORM_REL, torch.float16)
        assert bool(torch.isnan(o.rmsnorm(x[1:2].to(dev), gamma, 0.0)).all())      # 0 / 0, as the formula has it
    assert o.rmsnorm(x[:0].to(dev), gamma).shape == (0, 320)


@pytest.mark.parametrize("scale", [1e-36, 1e-25, 1.0, 1e25, 1e36])
def test_rmsnorm_of_far_magnitudes(dev, scale):
    """Rows whose squares leave fp32 on either side: the norm of a scaled row is that of the row (eps 0)."""
    x = (data(5, 700, 3, "f32", loud=False).double() * scale).float()
    want = O.rmsnorm(x.double(), torch.ones(700).double(), 0.0)
    within(ops().rmsnorm(x.to(dev), torch.ones(700, device=dev), 0.0), want, NORM_REL, torch.float32)
    bad = x.clone()
    bad[2, 5] = float("inf")
    y = ops().rmsnorm(bad.to(dev), torch.ones(700, device=dev), 0.0).cpu()
    assert bool(torch.isnan(y[2, 5])) and int(y[2].nan_to_num().count_nonzero()) == 0 and bool(torch.isfinite(y[[0, 1, 3, 4]]).all())


# ----------------------------------------------------------------------------- gated activation


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("fmt", [None, "mxfp8", "mxfp4"])
@pytest.mark.parametrize("rows,c,dtype,pad", [(1, 1, "f32", 0), (3, 40, "bf16", 0), (2, 129, "f16", 0), (17, 640, "bf16", 8), (5, 517, "f32", 3)])
def test_gated(dev, act, fmt, rows, c, dtype, pad):
    x = torch.cat([data(rows, c, c, dtype), (3 * data(rows, c, c + 7, dtype, loud=False).float()).clamp(-12, 12).to(TYPES[dtype])], dim=1)
    y = ops().gated(strided(x, dev, pad), act=act, fmt=fmt)
    want = x[:, :c].double() * O.gate(x[:, c:].double(), act)
    if fmt is None:
        assert y.dtype == x.dtype
        within(y, want, GATE_REL, x.dtype)
    else:
        assert O.held_within(ops().mx_dequantize(y).double().cpu(), want, GATE_REL, fmt)


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gate_far_values(dev, act):
    """Gates far out: the identity on the right to infinity, nothing (below the smallest normal fp32) on the left, NaN through."""
    b = torch.tensor([40.0, 1e4, 1e30, float("inf"), -100.0, -1e4, -1e30, 0.0, float("nan")])
    y = ops().gated(torch.cat([torch.ones(9), b]).view(1, 18).to(dev), act=act).cpu().view(-1)
    assert torch.equal(y[:4], b[:4]) and bool((y[4:8].abs() < 2.0 ** -126).all()) and bool(torch.isnan(y[8]))


# ----------------------------------------------------------------------------- the product


def group_tops(v):
    """The largest magnitude of every 8 consecutive values of a row."""
    return torch.nn.functional.pad(v.abs(), (0, -v.shape[1] % 8)).reshape(v.shape[0], -1, 8).amax(dim=2)


def product(a, b, fmt, bias, res):
    """(value, bound) of a @ b^T + bias + res in fp32, a and b the operands' values in 64 bits.
    Every partial sum is at most S = sum |a b|, each of the K additions is off by at most one step 2^-23 of it, bias and
    residual by half a step each.  With 8-bit operands the matrix instruction adds the products of 8 consecutive k on a grid
    2^-13 below the power of two of their largest and cuts off what lies below (a product 2^14 below another one among its
    8 neighbours vanishes, one among the next 8 does not): each of the other seven products loses less than 2^-13 of the
    largest product, which is at most the product of the largest operands.  4-bit products span 2^6 and lose nothing."""
    y, s = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        y, s = y + bias.double(), s + bias.double().abs()
    if res is not None:
        y, s = y + res.double(), s + res.double().abs()
    tol = s * ((a.shape[1] + 2) * 2.0 ** -23)
    if fmt == "mxfp8":
        tol = tol + 7 * 2.0 ** -13 * (group_tops(a) @ group_tops(b).t())
    return y, tol


SIZES = [(1, 64, 128), (1, 1, 1), (2, 10, 32), (16, 64, 256), (17, 65, 33), (31, 200, 1000), (48, 320, 1280), (64, 128, 640),
         (65, 130, 129), (130, 257, 300), (231, 1280, 1024), (300, 640, 515), (1, 5120, 1280), (5, 1000, 4096)]


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_mx(dev, fmt, m, n, k):
    o = ops()
    i = SIZES.index((m, n, k))
    dtype = ["bf16", "f16", "f32"][i % 3]
    x = data(m, k, i, dtype, loud=i % 2 == 0)
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(100 + i)) * k ** -0.5
    g = torch.Generator().manual_seed(200 + i)
    bias = torch.randn(n, generator=g) if i % 2 else None
    res = torch.randn(m, n, generator=g).to(x.dtype) if i % 3 != 1 else None
    pw = o.pack_linear_mx(w.to(dev), None if bias is None else bias.to(dev))
    y = o.linear_mx(strided(x, dev, 3 * (i % 4)), pw, fmt=fmt, res=None if res is None else strided(res, dev, 4 * (i % 3)))
    assert y.shape == (m, n) and y.dtype == x.dtype
    xv, wv = O.values(x.double(), fmt), O.values(w.double(), "mxfp4")
    want, tol = product(xv, wv, fmt, bias, res)
    fi = torch.finfo(x.dtype)
    tol = tol + want.abs() * fi.eps / 2 + fi.smallest_normal * fi.eps
    off = (y.double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"largest excess {float((off - tol).max()):.3e}"
    # the same from activations that are quantised already, bit for bit, and to fp32
    q = o.mx_quantize(x.to(dev), fmt)
    assert torch.equal(o.linear_mx(q, pw, res=None if res is None else res.to(dev), out_dtype=x.dtype), y)
    y32 = o.linear_mx(q, pw, out_dtype=torch.float32)
    want, tol = product(xv, wv, fmt, bias, None)
    assert bool(((y32.double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("algo", range(1, 9))
def test_every_kernel(dev, monkeypatch, fmt, algo):
    """Each kernel pinned, at 1 ... 9 k-steps (fewer than its ring holds, and more), tokens and columns that fill no tile and
    one column past one, with a bias and a residual; and the same call again, bit for bit."""
    o = ops()
    monkeypatch.setattr(o, "FORCE_MX_ALGO", algo)
    for i, (m, n, k) in enumerate([(1, 1, 1), (2, 70, 128), (300, 257, 200), (257, 300, 384), (64, 520, 512), (33, 128, 640), (129, 65, 700),
                                   (513, 260, 896), (70, 600, 1024), (260, 130, 1100)]):
        x, w = data(m, k, i, "f32", loud=i % 2 == 0), torch.randn(n, k, generator=torch.Generator().manual_seed(i)) * k ** -0.5
        g = torch.Generator().manual_seed(50 + i)
        bias, res = (torch.randn(n, generator=g), torch.randn(m, n, generator=g)) if i % 3 else (None, None)
        pw, q = o.pack_linear_mx(w.to(dev), None if bias is None else bias.to(dev)), o.mx_quantize(x.to(dev), fmt)
        y = o.linear_mx(q, pw, res=None if res is None else res.to(dev), out_dtype=torch.float32)
        want, tol = product(O.values(x.double(), fmt), O.values(w.double(), "mxfp4"), fmt, bias, res)
        off = (y.double().cpu() - want).abs()
        assert bool((off <= tol).all()), f"{(m, n, k)}: largest excess {float((off - tol).max()):.3e}"
        for _ in range(3):
            assert torch.equal(o.linear_mx(q, pw, res=None if res is None else res.to(dev), out_dtype=torch.float32), y), (m, n, k)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_kernels_agree_on_large_products(dev, monkeypatch, fmt):
    """Many tiles and k-steps at once, where a fill that is not waited for would show: the tiled kernels against each other (the
    same order of sums) and against the direct one (another order), several times."""
    o = ops()
    m, n, k = 2100, 2600, 2700
    q = o.mx_quantize(data(m, k, 1, "bf16", loud=False).to(dev), fmt)
    pw = o.pack_linear_mx(torch.randn(n, k, generator=torch.Generator().manual_seed(1)).to(dev) * k ** -0.5)

    def run(algo):
        monkeypatch.setattr(o, "FORCE_MX_ALGO", algo)
        return o.linear_mx(q, pw, out_dtype=torch.float32)

    first = run(8)
    direct = run(4)
    for algo in (5, 6, 7, 8):
        for _ in range(5):
            assert torch.equal(run(algo), first), algo
    a, b = O.values(data(m, k, 1, "bf16", loud=False).double(), fmt), o.mx_dequantize(q).double().cpu()
    assert torch.equal(a, b)
    s = a[:64].abs() @ O.values(torch.randn(n, k, generator=torch.Generator().manual_seed(1)).mul(k ** -0.5).double(), "mxfp4").abs().t()
    assert bool(((direct - first).double().abs().cpu()[:64] <= 2 * s * ((k + 2) * 2.0 ** -23 + 7 * 2.0 ** -13)).all())


@pytest.mark.parametrize("k", [100, 128, 200, 384, 1000, 1300])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_kernels_agree_over_many_tiles(dev, monkeypatch, fmt, k):
    """More than 512 tiles of 128 x 128 (there 8-bit operands take a shorter ring), one k-step to eleven: every tiled kernel adds
    in the same order, so they agree to the bit, several times over."""
    o = ops()
    m, n = 2990, 3010
    q = o.mx_quantize(data(m, k, 2, "bf16", loud=False).to(dev), fmt)
    pw = o.pack_linear_mx(torch.randn(n, k, generator=torch.Generator().manual_seed(3)).to(dev) * k ** -0.5)

    def run(algo):
        monkeypatch.setattr(o, "FORCE_MX_ALGO", algo)
        return o.linear_mx(q, pw, out_dtype=torch.float32)

    first = run(8)
    for algo in (5, 6, 7):
        for _ in range(4):
            assert torch.equal(run(algo), first), algo


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("algo", range(1, 9))
def test_every_kernel_adds_and_rounds_once(dev, monkeypatch, algo, dtype):
    """Bias and residual of every type, added in fp32 and rounded once: bit for bit what the kernel's own fp32 products give.
    Rows and columns that end inside a tile, a column group and a quad, residuals of any stride, outputs in place of the residual."""
    from stablediffusion_amd import hip
    o = ops()
    monkeypatch.setattr(o, "FORCE_MX_ALGO", algo)
    t = TYPES[dtype]
    for i, (m, n) in enumerate([(1, 64), (15, 66), (130, 128), (260, 323), (400, 576), (257, 1)]):
        k = 150 + 128 * i
        g = torch.Generator().manual_seed(300 + i)
        w, bias, res = torch.randn(n, k, generator=g) * k ** -0.5, torch.randn(n, generator=g).to(dev), torch.randn(m, n, generator=g).to(t)
        q = o.mx_quantize(data(m, k, i, "bf16", loud=False).to(dev), ["mxfp8", "mxfp4"][i % 2])
        bare, with_bias = o.pack_linear_mx(w.to(dev)), o.pack_linear_mx(w.to(dev), bias)
        sums = o.linear_mx(q, bare, out_dtype=torch.float32)
        for pad in (0, 1, 8):
            r = strided(res, dev, pad)
            assert torch.equal(o.linear_mx(q, bare, res=r), (sums + r.float()).to(t)), (m, n, pad)
            assert torch.equal(o.linear_mx(q, with_bias, res=r), (sums + bias + r.float()).to(t)), (m, n, pad)
            assert torch.equal(o.linear_mx(q, with_bias, out_dtype=t), (sums + bias).to(t)), (m, n, pad)
            # in place of the residual, a column slice of a buffer whose other columns stay as they were
            wide = torch.full((m, n + 2 * pad), 7.0, dtype=t, device=dev)
            own = wide[:, pad:pad + n]
            own.copy_(r)
            a = hip.MxGemmArgs()
            a.x_codes, a.x_scales, a.fmt = q.codes_ptr, q.scales_ptr, [hip.MX_FP8, hip.MX_FP4][i % 2]
            a.w_codes, a.w_scales, a.bias = with_bias.codes_ptr, with_bias.scales_ptr, with_bias.bias_ptr
            a.M, a.N, a.K, a.out, a.res, a.ld_out, a.ld_res = m, n, k, own.data_ptr(), own.data_ptr(), own.stride(0), own.stride(0)
            a.out_dtype, a.algo = o._mx_dt(t, "test"), algo
            hip.check(hip.lib().sdmi_mx_gemm(ctypes.byref(a), torch.cuda.current_stream().cuda_stream), "sdmi_mx_gemm")
            assert torch.equal(own, (sums + bias + r.float()).to(t)), (m, n, pad)
            assert bool((wide[:, :pad] == 7.0).all()) and bool((wide[:, pad + n:] == 7.0).all()), (m, n, pad)


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_quantisation_inside_the_product(dev, fmt, dtype):
    """Plain activations that the product quantises itself: the direct kernels' products of what mx_quantize gives, bit for bit
    (their order of sums is one and the same).  Row counts around the powers of two and the tiles, K that ends in a k-step, in a
    block and past the waves' first, second and third k-steps, and rows of any stride whose neighbours are NaN."""
    o = ops()
    for i, (m, n, k) in enumerate([(1, 40, 8), (1, 17000, 136), (3, 130, 1000), (5, 64, 5000), (8, 10300, 1056), (16, 100, 3064), (17, 300, 1032), (33, 1000, 1024),
                                   (100, 4000, 40), (230, 1290, 1016), (257, 1100, 512), (31, 9000, 904), (40, 10000, 968), (300, 70, 2048), (900, 64, 256)]):
        x = data(m, k, i, dtype, loud=i % 2 == 0)
        pw = o.pack_linear_mx(torch.randn(n, k, generator=torch.Generator().manual_seed(i)).to(dev) * k ** -0.5)
        q = o.mx_quantize(x.to(dev), fmt)
        o.FORCE_MX_ALGO = 1
        try:
            want = o.linear_mx(q, pw, out_dtype=torch.float32)
        finally:
            o.FORCE_MX_ALGO = 0
        for pad in (0, 3, 8):
            assert torch.equal(o.linear_mx(strided(x, dev, pad), pw, fmt=fmt, out_dtype=torch.float32), want), (m, n, k, pad)


@pytest.mark.parametrize("m", [1, 20, 150])
@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_linear_mx_picks_single_elements(dev, fmt, m):
    """One-hot rows against weights of all different small integers: a swapped row, column, block or scale shows."""
    o = ops()
    n, k = 130, 300
    g = torch.Generator().manual_seed(m)
    w = torch.randint(-6, 7, (n, k), generator=g).float().clamp(-6, 6)
    w[w.abs() == 5] = 4.0
    w[:, ::32] = 6.0                                                    # the scale of every block is 1
    w *= 2.0 ** torch.randint(-3, 4, (n, 10), generator=g).float().repeat_interleave(32, dim=1)[:, :k]
    x = torch.zeros(m, k)
    at = torch.randint(0, k, (m,), generator=g)
    x[torch.arange(m), at] = 2.0 ** torch.randint(-5, 6, (m,), generator=g).float()
    y = o.linear_mx(x.to(dev), o.pack_linear_mx(w.to(dev)), fmt=fmt)
    assert torch.equal(y.cpu(), x @ w.t())


def test_linear_mx_poison_stays_in_its_rows(dev):
    """A NaN in a row of activations reaches that row alone, an infinity too; one in the weights its column alone."""
    o = ops()
    x, w = data(70, 256, 1, "f32", loud=False), torch.randn(96, 256, generator=torch.Generator().manual_seed(2))
    x[3, 200], x[66, 0] = float("nan"), float("inf")
    y = o.linear_mx(x.to(dev), o.pack_linear_mx(w.to(dev))).cpu()
    bad = torch.isnan(y).all(dim=1)
    assert bad.nonzero().view(-1).tolist() == [3, 66] and bool(torch.isfinite(y[~bad]).all())
    w[50, 9] = float("nan")
    y = o.linear_mx(data(70, 256, 1, "f32", loud=False).to(dev), o.pack_linear_mx(w.to(dev))).cpu()
    bad = torch.isnan(y).all(dim=0)
    assert bad.nonzero().view(-1).tolist() == [50] and bool(torch.isfinite(y[:, ~bad]).all())


def test_linear_mx_repeats(dev):
    """The same call again gives the same bits."""
    o = ops()
    x, w = data(200, 1000, 4).to(dev), torch.randn(300, 1000, generator=torch.Generator().manual_seed(5)).to(dev)
    pw = o.pack_linear_mx(w)
    for m in (1, 16, 33, 200):
        a = o.linear_mx(x[:m], pw)
        for _ in range(3):
            assert torch.equal(o.linear_mx(x[:m], pw), a)


def test_linear_mx_empty_and_shapes(dev):
    o = ops()
    pw = o.pack_linear_mx(torch.randn(40, 64, device=dev), torch.zeros(40, device=dev))
    x = data(12, 64, 1).to(dev)
    assert o.linear_mx(x[:0], pw).shape == (0, 40)
    assert torch.equal(o.linear_mx(x.view(3, 4, 64), pw).view(12, 40), o.linear_mx(x, pw))
    assert o.linear_mx(x[0], pw).shape == (40,)


# ----------------------------------------------------------------------------- refusals that need a device


def test_refusals(dev):
    from stablediffusion_amd import hip
    o = ops()
    x = data(8, 64, 1).to(dev)
    pw = o.pack_linear_mx(torch.randn(40, 64, device=dev))
    gamma = torch.ones(64, device=dev)
    q = o.mx_quantize(x, "mxfp8")
    for call in (lambda: o.mx_quantize(x.t()), lambda: o.mx_quantize(x[:, :0]), lambda: o.mx_quantize(x.to(torch.float64)),
                 lambda: o.mx_quantize(x[0].expand(4, 64)), lambda: o.mx_quantize(x, "mxfp6"), lambda: o.mx_dequantize(q, torch.int8),
                 lambda: o.mx_quantize(x.view(2, 4, 64)[:, :3]),
                 lambda: o.rmsnorm(x, gamma[:63]), lambda: o.rmsnorm(x, gamma.to(torch.bfloat16)), lambda: o.rmsnorm(x, gamma, -1.0),
                 lambda: o.rmsnorm(x, gamma, res=x.float()), lambda: o.rmsnorm(x, gamma, res=x[:4]), lambda: o.rmsnorm(x, gamma.cpu()),
                 lambda: o.rmsnorm(x, gamma, fmt="mxfp8", out_dtype=torch.float32),
                 lambda: o.rmsnorm(torch.zeros(1, 16385, device=dev), torch.ones(16385, device=dev)),
                 lambda: o.gated(x[:, :63]), lambda: o.gated(x, act="tanh"), lambda: o.gated(x, out_dtype=torch.int32),
                 lambda: o.pack_linear_mx(x[0]), lambda: o.pack_linear_mx(x, torch.zeros(9, device=dev)), lambda: o.pack_linear_mx(x, torch.zeros(8)),
                 lambda: o.linear_mx(x[:, :63], pw), lambda: o.linear_mx(q, pw, fmt="mxfp4"), lambda: o.linear_mx(x, pw, res=x),
                 lambda: o.linear_mx(x, pw, out_dtype=torch.int8), lambda: o.linear_mx(x, pw, res=torch.zeros(8, 40, device=dev)),
                 lambda: o.linear_mx(x.cpu(), pw)):
        with pytest.raises(hip.SdmiError):
            call()


# ----------------------------------------------------------------------------- together


@pytest.mark.parametrize("tokens,fmt,act", [(1, "mxfp8", "silu"), (77, "mxfp8", "gelu"), (300, "mxfp4", "silu")])
def test_feed_forward_links(dev, tokens, fmt, act):
    """norm -> product -> gate -> product + residual, as a feed-forward runs; every link is checked on what the link before it
    gave, so that no bound has to cover a rounding that another operator made."""
    o = ops()
    c, inner = 320, 640
    g = torch.Generator().manual_seed(tokens)
    x, r = data(tokens, c, 1), data(tokens, c, 2)
    gamma = 1 + 0.1 * torch.randn(c, generator=g)
    w1, w2 = torch.randn(2 * inner, c, generator=g) * c ** -0.5, torch.randn(c, inner, generator=g) * inner ** -0.5
    p1, p2 = o.pack_linear_mx(w1.to(dev)), o.pack_linear_mx(w2.to(dev))
    y, s = o.rmsnorm(x.to(dev), gamma.to(dev), res=r.to(dev), fmt=fmt)
    h = o.linear_mx(y, p1)
    a = o.gated(h, act=act, fmt=fmt)
    out = o.linear_mx(a, p2, res=s)
    assert out.dtype == torch.bfloat16 and out.shape == (tokens, c)
    yv, av = o.mx_dequantize(y).cpu(), o.mx_dequantize(a).cpu()
    assert O.held_within(yv.double(), O.rmsnorm((x.float() + r.float()).double(), gamma.double(), 1e-6), NORM_REL, fmt)
    for got, xin, w, res in ((h, yv, w1, None), (out, av, w2, s.cpu())):
        want, tol = product(xin.double(), O.values(w.double(), "mxfp4"), fmt, None, res)
        tol = tol + want.abs() * 2.0 ** -8
        assert bool(((got.double().cpu() - want).abs() <= tol).all())
    hc = h.double().cpu()
    assert O.held_within(av.double(), hc[:, :inner] * O.gate(hc[:, inner:], act), GATE_REL, fmt)


def test_calls_of_two_threads_on_one_stream(dev):
    """A product of plain activations is a quantisation and a product; two threads' calls on one stream keep theirs apart."""
    import threading
    o = ops()
    pw = o.pack_linear_mx(torch.randn(96, 512, generator=torch.Generator().manual_seed(1)).to(dev))
    xs = [data(200, 512, i).to(dev) for i in range(2)]
    want = [o.linear_mx(x, pw) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        got = [o.linear_mx(xs[i], pw) for _ in range(200)]
        torch.cuda.synchronize()
        wrong.extend(1 for y in got if not torch.equal(y, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("m", [1, 40, 300])
def test_streams_and_graphs(dev, m):
    """The chain on a stream of its own and captured into two graphs that are replayed in turn, with eager work of the same
    operators between the replays."""
    o = ops()
    g = torch.Generator().manual_seed(m)
    w = torch.randn(256, 320, generator=g).to(dev) * 320 ** -0.5
    pw, gamma = o.pack_linear_mx(w), torch.ones(320, device=dev)
    xs = [data(m, 320, 10 + i).to(dev) for i in range(4)]

    def chain(x):
        y, s = o.rmsnorm(x, gamma, res=x, fmt="mxfp8")
        return o.linear_mx(y, pw, out_dtype=torch.bfloat16), o.linear_mx(s, pw, fmt="mxfp4"), s

    want = [chain(x) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [chain(x) for x in xs]
    side.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    graphs = []
    for _ in range(2):
        x = xs[0].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = chain(x)
        graphs.append((gr, x, out))
    for i in (1, 2, 3, 0, 2):
        for j, (gr, x, out) in enumerate(graphs):
            x.copy_(xs[(i + j) % 4])
            gr.replay()
        chain(xs[(i + 2) % 4])
        torch.cuda.synchronize()
        for j, (gr, x, out) in enumerate(graphs):
            assert all(torch.equal(u, v) for u, v in zip(out, want[(i + j) % 4])), (i, j)


# ----------------------------------------------------------------------------- far offsets


@pytest.mark.parametrize("fmt", ["mxfp8", "mxfp4"])
def test_offsets_past_32_bits(dev, fmt):
    """Rows whose elements, bytes and output positions lie past 2^31 and 2^32: the last rows against the same rows alone."""
    o = ops()
    rows, k, n = (1 << 20) + 37, 4224, 64
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=dev)
    tail = data(200, k, 3).to(dev)
    x[-200:] = tail
    q, alone = o.mx_quantize(x, fmt), o.mx_quantize(tail, fmt)
    assert torch.equal(q.codes[:, -200:], alone.codes) and torch.equal(q.scales[:, -200:], alone.scales)
    assert torch.equal(o.mx_dequantize(q, torch.bfloat16)[-200:], o.mx_dequantize(alone, torch.bfloat16))
    gamma = torch.ones(k, device=dev)
    assert torch.equal(o.rmsnorm(x, gamma)[-200:], o.rmsnorm(tail, gamma))
    assert torch.equal(o.gated(x)[-200:], o.gated(tail))
    pw = o.pack_linear_mx(torch.randn(n, k, generator=torch.Generator().manual_seed(1)).to(dev) * k ** -0.5)
    y = o.linear_mx(q, pw, out_dtype=torch.float32)
    assert y.shape == (rows, n)
    want, at = o.linear_mx(alone, pw, out_dtype=torch.float32), y[-200:]
    tol = o.mx_dequantize(alone).double().abs().sum(dim=1, keepdim=True) * float(k) * 2.0 ** -22
    assert bool(((at.double() - want.double()).abs() <= tol).all())
    assert int(y[: rows - 200].count_nonzero()) == 0


# ----------------------------------------------------------------------------- far values of the SiLU gate


@pytest.mark.parametrize("fmt", [None, "mxfp8"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_silu_where_its_exponential_leaves_fp32(dev, dtype, fmt):
    """x / (1 + exp(-x)) is a normal fp32 number down to x = -91.6, exp(x) only down to -87.3 and 1 / exp(-x) down to -88.7.
    The exponent |x| / (2 ln 2) rounded, times a rounded constant, in a root that counts twice would be 2 |x| 2^-24 relative, 183
    2^-24 at 91.5 and 220 at 110: under GATE_REL = 256 2^-24 with a dozen roundings beside it.  Below the normal numbers the
    relative error stays (1.2e-38 2^-16 = 130 steps of 2^-149), and two products are rounded to half a step each."""
    b = torch.linspace(-91.5, -60.0, 2048).to(TYPES[dtype])
    b = b[b >= -91.5]
    b = b[len(b) % 32:]                                        # (blocks of 32, in order: their values are alike)
    a = torch.ones_like(b)
    a[1::2] = 1024.0
    want = a.double() * O.gate(b.double(), "silu")
    if fmt is None:
        within(ops().gated(torch.stack([a, b], 1).to(dev), act="silu").view(-1), want, GATE_REL, TYPES[dtype])
        b = torch.linspace(-110.0, -91.5, 500)
        y = ops().gated(torch.stack([torch.ones(500), b], 1).to(dev), act="silu").view(-1).double().cpu()
        want = O.gate(b.double(), "silu")
        assert bool(((y - want).abs() <= want.abs() * GATE_REL + 2.0 ** -149).all())
    else:
        y = ops().gated(torch.cat([a, b]).view(1, -1).to(dev), act="silu", fmt=fmt)
        assert O.held_within(ops().mx_dequantize(y).double().cpu(), want.view(1, -1), GATE_REL, fmt)


# ----------------------------------------------------------------------------- what fp32 results hold


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gate_in_fp32(dev, act, dtype):
    """fp32 results, whose errors do not grow with |x|.  In units of 2^-24 of the gate's value, at worst.  SiLU: exp2's one step
    2, its exponent's remainder 1 and the product with it 1, all twice for the square, 1 + h^2 1, its reciprocal 2, three
    products 3, the gate's product 1: 15 < 16.  GELU: the fit 0.7; t = 1 / (1 + 0.35 |x|) 3 (constant, sum, the reciprocal after its
    Newton step), and exp(z^2) erfc(z) moves by 2.3 times that at z = 0, less further out, 7; the polynomial's eight sums, whose
    terms are up to 2.2 times the value, 9; exp2 2, the square's and the exponent's remainders 2, five products 5, the gate's 1: 27 < 32."""
    rel = (32 if act == "gelu" else 16) * 2.0 ** -24
    lo = -13.0 if act == "gelu" else -91.5                     # (Phi leaves the normal numbers at -13.1)
    for b in (torch.linspace(lo, 13.0, 6000), torch.linspace(-2.0, 2.0, 6000), torch.randn(6000, generator=torch.Generator().manual_seed(1))):
        b = b.to(TYPES[dtype])
        b = b[b >= lo]
        for a in (1.0, -3.0):
            y = ops().gated(torch.stack([torch.full_like(b, a), b], 1).to(dev), act=act, out_dtype=torch.float32).view(-1)
            within(y, a * O.gate(b.double(), act), rel, torch.float32)


# ----------------------------------------------------------------------------- the norm at fp32's ends, and what its results hold


@pytest.mark.parametrize("fmt", [None, "mxfp8"])
@pytest.mark.parametrize("dtype,scale", [("f32", 1e-44), ("f32", 1e-42), ("f32", 1e-40), ("f32", 1e-38), ("f32", 1e-30), ("f32", 1e-28), ("f32", 1e28), ("f32", 1e30),
                                         ("f32", 3.3e38), ("bf16", 1e-40), ("bf16", 1e-38), ("bf16", 3.3e38)])
def test_rmsnorm_at_the_ends_of_fp32(dev, dtype, scale, fmt):
    """Rows of subnormals, whose reciprocal root no fp32 number holds, and rows next to the largest number, whose one is
    subnormal (eps 0): the formula's result, to the ordinary bound, and s as it is."""
    x = (torch.randn(6, 700, generator=torch.Generator().manual_seed(4)).double().clamp(-1, 1) * scale).to(TYPES[dtype])
    x[1, 50:] = 0.0
    gamma = 1 + 0.2 * torch.randn(700, generator=torch.Generator().manual_seed(5))
    y, s = ops().rmsnorm(x.to(dev), gamma.to(dev), 0.0, res=torch.zeros_like(x).to(dev), fmt=fmt)
    assert torch.equal(s.cpu(), x)
    want = O.rmsnorm(x.double(), gamma.double(), 0.0)
    if fmt is None:
        within(y, want, 4 * 2.0 ** -24, TYPES[dtype])
    else:
        assert O.held_within(ops().mx_dequantize(y).double().cpu(), want, 4 * 2.0 ** -24, fmt)


@pytest.mark.parametrize("rows,c,dtype", [(64, 33, "f32"), (64, 1027, "f32"), (16, 5120, "f32"), (16, 5120, "bf16"), (4, 16384, "f16")])
def test_rmsnorm_in_fp32(dev, rows, c, dtype):
    """fp32 results.  s is the fp32 sum that the formula states; squares, their sum and the reciprocal root in fp64 and the latter
    as two fp32 numbers leave 2^-40; the value times the root is rounded once and its product with gamma once: 2 x 2^-24.  (A
    root in fp32 would be off by up to half a step more, for all values of its row.)"""
    x, r = data(rows, c, c, dtype), data(rows, c, c + 1, dtype)
    gamma = 1 + 0.2 * torch.randn(c, generator=torch.Generator().manual_seed(c))
    y, _ = ops().rmsnorm(x.to(dev), gamma.to(dev), 1e-5, res=r.to(dev), out_dtype=torch.float32)
    want = O.rmsnorm((x.float() + r.float()).double(), gamma.double(), float(torch.tensor(1e-5)))
    off = (y.double().cpu() - want).abs()
    assert bool((off <= want.abs() * 2.1 * 2.0 ** -24).all()), float((off / want.abs()).max()) * 2 ** 24


# ----------------------------------------------------------------------------- more rows than a launch holds


@pytest.mark.parametrize("op", ["quantise", "gate", "norm"])
def test_more_rows_than_a_launch_holds(dev, op):
    """A launch has fewer than 2^32 threads, 2^24 - 1 workgroups of 256: 16 rows each of the element-wise operators, 4 of the norm's
    narrow rows.  Rows on both sides of that border and the last ones against the same rows alone, nothing elsewhere."""
    o = ops()
    border = ((1 << 24) - 1) * (4 if op == "norm" else 16)
    rows, width = border + 1003, 1 if op == "quantise" else 2
    windows = [(0, 50), (border - 70, border + 70), (rows - 300, rows)]
    parts = [data(b - a, width, i + 1, loud=False).to(dev) for i, (a, b) in enumerate(windows)]
    x = torch.zeros(rows, width, dtype=torch.bfloat16, device=dev)
    for (a, b), part in zip(windows, parts):
        x[a:b] = part
    gamma = torch.ones(width, device=dev)
    run = {"quantise": lambda t: o.mx_dequantize(o.mx_quantize(t, "mxfp4"), torch.bfloat16), "gate": lambda t: o.gated(t),
           "norm": lambda t: o.rmsnorm(t, gamma, 1.0, res=t)}[op]
    got, want = run(x), [run(part) for part in parts]
    for i in range(2 if op == "norm" else 1):
        y, alone = (got[i], [w[i] for w in want]) if op == "norm" else (got, want)
        for (a, b), w in zip(windows, alone):
            assert torch.equal(y[a:b], w), (i, a)
        assert int(torch.count_nonzero(y)) == sum(int(torch.count_nonzero(w)) for w in alone), i


# ----------------------------------------------------------------------------- in a traced step


def test_the_operators_are_seen_by_the_trace(dev, monkeypatch):
    """A traced step lists these calls with the others, each with its work, its sizes and the events around it; a refused call
    leaves no entry, and the results are those of an untraced step."""
    from stablediffusion_amd import hip
    o = ops()
    gamma, beta = torch.ones(256, device=dev), torch.zeros(256, device=dev)
    x = data(40, 256, 1).to(dev)
    pw = o.pack_linear_mx(torch.randn(512, 256, generator=torch.Generator().manual_seed(1)).to(dev))

    def step():
        y, s = o.rmsnorm(x, gamma, res=x, fmt="mxfp8")
        h = o.linear_mx(y, pw)
        a = o.gated(h, act="silu")
        q = o.mx_quantize(a, "mxfp4")
        return s, o.mx_dequantize(q), o.rmsnorm(x, gamma, out_dtype=torch.float32), o.linear_mx(x, pw), o.layernorm(x, gamma, beta)

    want = step()
    monkeypatch.setattr(o, "TRACE", [])
    got = step()
    with pytest.raises(hip.SdmiError):
        o.linear_mx(x, pw, out_dtype=torch.int8)
    o.pack_linear_mx(x)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    plain, codes8, codes4 = 40 * 256 * 2, 40 * (256 + 8), 40 * (128 + 8)
    assert [(k, w, shape) for k, w, _, _, _, shape in o.TRACE] == [
        ("rmsnorm", 3 * plain + 1024 + codes8, (40, 256)), ("linear_mx", 2 * 40 * 512 * 256, (40, 512, 256)), ("gated", 3 * plain, (40, 256)),
        ("mx_quantize", plain + codes4, (40, 256)), ("mx_dequantize", codes4 + 2 * plain, (40, 256)),
        ("rmsnorm", plain + 1024 + 2 * plain, (40, 256)), ("linear_mx", 2 * 40 * 512 * 256, (40, 512, 256)), ("layernorm", 2 * plain, (40, 256))]
    assert all(e0.elapsed_time(e1) > 0 for _, _, e0, e1, _, _ in o.TRACE)


# ----------------------------------------------------------------------------- far offsets of the product


@pytest.mark.parametrize("fmt,k", [("mxfp8", 4224), ("mxfp4", 8448)])
def test_product_of_codes_past_32_bits(dev, monkeypatch, fmt, k):
    """Codes past 2^32 bytes from the last k-steps on, in each kernel and from plain activations: the last rows bit for bit what
    the same kernel makes of them alone (the tiled kernels add in one order, the direct ones in another), and those within the
    product's bound of the 64-bit oracle.  The other rows are ones, all with the same result, so that an offset that wraps
    reads other codes; a last k-step left out is over that bound in every row, in 80 % (mxfp8) and 63 % (mxfp4) of the elements."""
    o = ops()
    rows, n, tail_rows = 65535 * 16, 72, 200                   # (the most rows of the direct kernels of 16)
    tail = data(tail_rows, k, 3, loud=False).to(dev)
    w = torch.randn(n, k, generator=torch.Generator().manual_seed(1)) * k ** -0.5
    pw = o.pack_linear_mx(w.to(dev))
    x = torch.ones(rows, k, dtype=torch.bfloat16, device=dev)
    x[-tail_rows:] = tail
    q, alone, one = o.mx_quantize(x, fmt), o.mx_quantize(tail, fmt), o.mx_quantize(x[:1], fmt)
    assert (k // 128 - 2) * rows * (128 if fmt == "mxfp8" else 64) < 2 ** 32 < q.codes.numel()
    want, tol = product(O.values(tail.double().cpu(), fmt), O.values(w.double(), "mxfp4"), fmt, None, None)
    for algo in range(1, 9):
        monkeypatch.setattr(o, "FORCE_MX_ALGO", algo)
        y, a = o.linear_mx(q, pw, out_dtype=torch.float32), o.linear_mx(alone, pw, out_dtype=torch.float32)
        assert bool(((a.double().cpu() - want).abs() <= tol).all()), algo
        assert torch.equal(y[-tail_rows:], a), algo
        assert bool((y[:-tail_rows] == o.linear_mx(one, pw, out_dtype=torch.float32)).all()), algo
        if algo in (1, 8):
            assert torch.equal(o.linear_mx(x, pw, fmt=fmt, out_dtype=torch.float32), y), algo


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("algo", range(1, 9))
def test_product_into_places_past_32_bits(dev, monkeypatch, algo, dtype):
    """Outputs and residuals past 2^31 elements (2^32 bytes of bf16, 2^33 of fp32), one k-step, columns that end inside a quad: rows
    at the start, across 2^31 elements and at the end are what the kernel makes of them alone, the others 0."""
    o = ops()
    monkeypatch.setattr(o, "FORCE_MX_ALGO", algo)
    rows, n, k, t = (1 << 18) + 77, 8251, 100, TYPES[dtype]
    border = (1 << 31) // n
    windows = [(0, 60), (border - 70, border + 70), (rows - 300, rows)]
    assert border + 70 < rows - 300 and rows * n > 1 << 31
    g = torch.Generator().manual_seed(algo)
    pw = o.pack_linear_mx((torch.randn(n, k, generator=g) * k ** -0.5).to(dev))
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=dev)
    wide = torch.zeros(rows, n + 5, dtype=t, device=dev)
    res = wide[:, 3:3 + n]
    parts = [(data(b - a, k, i + 1, loud=False).to(dev), torch.randn(b - a, n, generator=g).to(t).to(dev)) for i, (a, b) in enumerate(windows)]
    for (a, b), (px, pr) in zip(windows, parts):
        x[a:b], res[a:b] = px, pr
    fmt = ["mxfp8", "mxfp4"][algo % 2]
    y = o.linear_mx(o.mx_quantize(x, fmt), pw, res=res, out_dtype=t)
    left = int(torch.count_nonzero(y))
    for (a, b), (px, pr) in zip(windows, parts):
        alone = o.linear_mx(o.mx_quantize(px, fmt), pw, res=pr, out_dtype=t)
        assert torch.equal(y[a:b], alone), a
        left -= int(torch.count_nonzero(alone))
    assert left == 0


def test_gelu_codes_beside_those_of_an_fp32_erfc(dev):
    """How many e4m3 elements of 16.8 million gate products lie on another side of a rounding border than the exact ones: no
    more than half as many again as a plain fp32 erfc makes on the same values (about a dozen), and four for the chance in it."""
    n = 4096
    g = torch.Generator().manual_seed(11)
    x = torch.randn(n, 2 * n, generator=g).half()
    a, b = x[:, :n], x[:, n:]
    exact = O.values(a.double() * O.gate(b.double(), "gelu"), "mxfp8")
    bd = b.to(dev).float()
    plain = a.to(dev).float() * (0.5 * bd * torch.special.erfc(bd * -0.5 ** 0.5))
    own = ops().mx_dequantize(ops().gated(x.to(dev), act="gelu", fmt="mxfp8")).double().cpu()
    off = int((own != exact).sum()), int((O.values(plain.double().cpu(), "mxfp8") != exact).sum())
    assert off[0] <= 1.5 * off[1] + 4, off
