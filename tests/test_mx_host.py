"""The block-scaled operators' refusals through the C ABI (every one returns before a kernel is launched) and the oracle they
are checked against, on the CPU."""
import ctypes as C

import pytest
import torch

import mx_oracle as O

OK, BAD, ALIGN, WORKSPACE = 0, -1, -2, -3
P = 4096            # stands for a device pointer: never read, the calls below are refused or empty
DT = {"bf16": 0, "f16": 1, "f32": 4}


@pytest.fixture(scope="module")
def lib():
    from stablediffusion_amd import hip
    return hip.lib()


def test_quantise_refusals(lib):
    q = lib.sdmi_mx_quantize
    assert q(P, 64, 0, 64, 0, P, P, 1, None) == OK                     # no rows: an empty call
    for bad in ((None, 64, 4, 64, 0, P, P, 1), (P, 64, 4, 64, 0, None, P, 1), (P, 64, 4, 64, 0, P, None, 1),
                (P, 64, -1, 64, 0, P, P, 1), (P, 64, 4, 0, 0, P, P, 1), (P, 63, 4, 64, 0, P, P, 1), (P, 64, 4, 64, 2, P, P, 1),
                (P, 64, 4, 64, 3, P, P, 1), (P, 64, 4, 64, 0, P, P, 0), (P, 64, 4, 64, 0, P, P, 3), (P, 1 << 25, 4, (1 << 24) + 1, 0, P, P, 1),
                (P, 64, 1 << 31, 64, 0, P, P, 1)):
        assert q(*bad, None) == BAD, bad
    assert q(P, 64, 4, 64, 0, P + 8, P, 1, None) == ALIGN
    assert q(P, 64, 4, 64, 0, P, P + 4, 2, None) == ALIGN


def test_dequantise_refusals(lib):
    d = lib.sdmi_mx_dequantize
    assert d(P, P, 0, 64, 1, P, 64, 0, None) == OK
    for bad in ((None, P, 4, 64, 1, P, 64, 0), (P, None, 4, 64, 1, P, 64, 0), (P, P, 4, 64, 1, None, 64, 0), (P, P, 4, 64, 0, P, 64, 0),
                (P, P, 4, 64, 1, P, 63, 0), (P, P, 4, 0, 1, P, 64, 0), (P, P, -4, 64, 1, P, 64, 0), (P, P, 4, 64, 1, P, 64, 2)):
        assert d(*bad, None) == BAD, bad
    assert d(P + 2, P, 4, 64, 1, P, 64, 0, None) == ALIGN


def test_rmsnorm_refusals(lib):
    n = lib.sdmi_rmsnorm
    good = [P, 64, P, 64, P, 1e-6, 0, 64, 0, P, P, 0, P, 1]
    assert n(*good, None) == OK
    for i, v in ((0, None), (1, 63), (3, 63), (4, None), (5, -1.0), (5, float("nan")), (6, -1), (7, 0), (7, 16385), (8, 2), (9, None),
                 (10, None), (12, None), (13, 3)):
        a = list(good)
        a[i] = v
        a[6] = 4 if i != 6 else a[6]
        if i == 7 and v > 64:
            a[1] = a[3] = v
        assert n(*a, None) == BAD, (i, v)
    a = list(good)
    a[6], a[13], a[11] = 4, 0, 2                                        # plain result of an unknown type
    assert n(*a, None) == BAD
    for i in (4, 10, 12):
        a = list(good)
        a[6], a[i] = 4, P + 4
        assert n(*a, None) == ALIGN, i


def test_gated_refusals(lib):
    g = lib.sdmi_gated
    good = [P, 128, 0, 64, 0, 0, P, 0, P, 1]
    assert g(*good, None) == OK
    for i, v in ((0, None), (1, 127), (2, -1), (3, 0), (4, 3), (5, 2), (5, -1), (6, None), (8, None), (9, 7)):
        a = list(good)
        a[i] = v
        a[2] = 4 if i != 2 else a[2]
        assert g(*a, None) == BAD, (i, v)
    a = list(good)
    a[2], a[6] = 4, P + 2
    assert g(*a, None) == ALIGN


def test_pack_refusals(lib):
    p = lib.sdmi_mx_pack_linear
    for bad in ((None, 64, 8, 64, 4, P, P), (P, 64, 8, 64, 4, None, P), (P, 64, 8, 64, 4, P, None), (P, 63, 8, 64, 4, P, P),
                (P, 64, 0, 64, 4, P, P), (P, 64, 8, 0, 4, P, P), (P, 64, 8, 64, 2, P, P), (P, 64, (1 << 24) + 1, 64, 4, P, P)):
        assert p(*bad, None) == BAD, bad
    assert p(P, 64, 8, 64, 4, P + 1, P, None) == ALIGN


def _gemm(**kw):
    from stablediffusion_amd import hip
    a = hip.MxGemmArgs()
    base = dict(x=P, ldx=64, x_dtype=0, w_codes=P, w_scales=P, out=P, M=0, N=64, K=64, ld_out=64, out_dtype=0, fmt=1)
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


def test_product_refusals(lib):
    g = lambda **kw: lib.sdmi_mx_gemm(C.byref(_gemm(**kw)), None)
    assert g() == OK
    assert g(x=None, x_codes=P, x_scales=P) == OK
    for bad in (dict(w_codes=None), dict(w_scales=None), dict(out=None), dict(x=None), dict(x=None, x_codes=P), dict(ldx=63), dict(x_dtype=3),
                dict(N=0), dict(K=0), dict(M=-1), dict(fmt=0), dict(algo=-1), dict(algo=9), dict(out_dtype=2), dict(ld_out=63), dict(res=P, ld_res=63), dict(K=(1 << 24) + 1, ldx=1 << 25)):
        assert g(**{"M": 4, **bad}) == BAD, bad
    assert lib.sdmi_mx_gemm(None, None) == BAD
    for bad in (dict(w_codes=P + 8), dict(w_scales=P + 2), dict(x=None, x_codes=P + 8, x_scales=P)):
        assert g(M=4, **bad) == ALIGN, bad
    # (a product that quantises by itself - K in whole eights, few tokens - has no use for a workspace)
    assert lib.sdmi_mx_gemm_workspace_bytes(C.byref(_gemm(M=300, K=1000, ldx=1000))) == 0
    need = lib.sdmi_mx_gemm_workspace_bytes(C.byref(_gemm(M=300, K=1001, ldx=1001)))
    assert need > 0
    assert g(M=300, K=1001, ldx=1001) == WORKSPACE
    assert g(M=300, K=1001, ldx=1001, workspace=P, workspace_bytes=need - 1) == WORKSPACE
    assert g(M=300, K=1001, ldx=1001, workspace=P + 4, workspace_bytes=need) == WORKSPACE
    assert lib.sdmi_mx_gemm_workspace_bytes(C.byref(_gemm(M=4, K=0))) == -1


def test_sizes(lib):
    assert lib.sdmi_mx_codes_bytes(3, 129, 1) == 3 * 256 and lib.sdmi_mx_codes_bytes(3, 129, 2) == 3 * 128
    assert lib.sdmi_mx_scales_bytes(3, 129) == 2 * 3 * 4
    assert lib.sdmi_mx_codes_bytes(3, 0, 1) == lib.sdmi_mx_scales_bytes(-1, 4) == lib.sdmi_mx_codes_bytes(3, 4, 0) == -1
    assert lib.sdmi_mx_weight_codes_bytes(65, 129) == 2 * 2 * 4096 and lib.sdmi_mx_weight_scales_bytes(65, 129) == 2 * 2 * 256


def test_python_refusals_need_no_gpu():
    from stablediffusion_amd import hip, ops
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for call in (lambda: ops.mx_quantize(x), lambda: ops.rmsnorm(x, torch.ones(64)), lambda: ops.gated(x), lambda: ops.pack_linear_mx(x),
                 lambda: ops.mx_quantize(x, "fp8"), lambda: ops.gated(x, act="relu"), lambda: ops.mx_quantize(x.to(torch.int8))):
        with pytest.raises(hip.SdmiError):
            call()


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_oracle_against_the_formats_own_tables(fmt):
    """Every value that the oracle gives is scale times a representable element, and no representable element is nearer."""
    emax, emin, digits, most = O.FORMATS[fmt]
    table = {0.0}
    for e in range(emin, emax + 1):
        for m in range(2 ** digits):
            table.add((1 + m / 2 ** digits) * 2.0 ** e)
            table.add(m / 2 ** digits * 2.0 ** emin)
    table = torch.tensor(sorted(t for t in table if t <= most), dtype=torch.float64)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(16, 96, generator=g, dtype=torch.float64) * torch.exp(4 * torch.randn(16, 1, generator=g, dtype=torch.float64))
    scale = O.power(O.scale_exponents(x, fmt)).repeat_interleave(32, dim=1)
    got, want = O.values(x, fmt) / scale, (x / scale).clamp(-most, most)
    far = (got.abs()[..., None] - table).abs().amin(-1)
    assert float(far.max()) == 0.0
    assert bool(((got - want).abs() <= (want.abs()[..., None] - table).abs().amin(-1)).all())


def test_sizes_beyond_the_limits(lib):
    """The size queries give -1 for what the operators refuse, and nothing overflows on the way."""
    assert lib.sdmi_mx_codes_bytes((1 << 31) - 1, 1 << 24, 1) == ((1 << 31) - 1) << 24 and lib.sdmi_mx_scales_bytes((1 << 31) - 1, 1) == ((1 << 31) - 1) * 4
    for rows, k in ((1 << 31, 64), (1 << 62, 1), (4, (1 << 24) + 1), (4, (1 << 62) + 1)):
        assert lib.sdmi_mx_codes_bytes(rows, k, 1) == lib.sdmi_mx_codes_bytes(rows, k, 2) == lib.sdmi_mx_scales_bytes(rows, k) == -1, (rows, k)
        assert lib.sdmi_mx_quantize(P, k, rows, k, 0, P, P, 1, None) == lib.sdmi_mx_dequantize(P, P, rows, k, 1, P, k, 0, None) == BAD, (rows, k)
    assert lib.sdmi_mx_weight_codes_bytes(1 << 24, 8064) == (1 << 18) * 63 * 4096
    # N, K, and the threads of the packing launch (one for 32 values): 2^24 x 8192 would be 2^32
    for n, k in (((1 << 24) + 1, 64), (64, (1 << 24) + 1), (1 << 62, 1), (1 << 24, 8192), (1 << 24, 1 << 24)):
        assert lib.sdmi_mx_weight_codes_bytes(n, k) == lib.sdmi_mx_weight_scales_bytes(n, k) == -1, (n, k)
        assert lib.sdmi_mx_pack_linear(P, k, n, k, 4, P, P, None) == BAD, (n, k)
        assert lib.sdmi_mx_gemm_workspace_bytes(C.byref(_gemm(M=4, N=n, K=k, ldx=k, ld_out=n))) == -1, (n, k)


def test_a_product_is_refused_before_anything_is_launched(lib):
    """Pinned kernels whose grid does not hold the rows: the workspace query says so already, and the product refuses before it
    quantises (a workspace of 0 bytes would be the first complaint otherwise)."""
    size = lambda **kw: lib.sdmi_mx_gemm_workspace_bytes(C.byref(_gemm(N=64, K=64, **kw)))
    call = lambda **kw: lib.sdmi_mx_gemm(C.byref(_gemm(N=64, K=64, **kw)), None)
    for algo, rows in ((1, 16), (2, 16), (3, 32), (4, 48)):              # row tiles along y: at most 65535
        assert size(M=65535 * rows, algo=algo) > 0 and size(M=65535 * rows + 1, algo=algo) == -1, algo
        assert call(M=65535 * rows + 1, algo=algo) == BAD and call(M=65535 * rows, algo=algo) == WORKSPACE, algo
    for algo, rows, threads in ((5, 64, 256), (6, 128, 256), (7, 128, 512), (8, 256, 512)):      # all tiles along x: fewer than 2^32 threads
        most = min((2 ** 32 - 1) // threads * rows, 2 ** 31 - 1)
        assert size(M=most, algo=algo) > 0 and call(M=most, algo=algo) == WORKSPACE, algo
        if most < 2 ** 31 - 1:
            assert size(M=most + 1, algo=algo) == -1 and call(M=most + 1, algo=algo) == BAD, algo
    # left to itself the library takes a kernel that holds them, and none past the largest tiles' last full launch
    assert size(M=65535 * 48 + 1) > 0 and size(M=2 ** 31 - 256) > 0 and size(M=2 ** 31) == -1
    assert size(M=2 ** 31 - 1) == -1 and call(M=2 ** 31 - 1) == BAD
