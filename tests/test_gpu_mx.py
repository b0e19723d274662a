"""Microscaled (MX) operators on the GPU against the 64-bit definitions of mx_ref. Tolerances, u = 2^-24 (half a step of fp32, relative):
  quantise and dequantise   exact (dequantise: one rounding to the output's type)
  product                   fp32 sums of at most n terms and the factor of the FP16 format: (n + 4) u sum |a b|
  norm                      y = s * inv * w from a 64-bit sum rounds four times: 4 u |y| before the element's own half step
  backward                  half a step of dx's type and at most 8 roundings of its terms; dweight (rows + 4) u sum |dy s inv|"""
import numpy as np
import pytest
import torch

import vcsr_mc_b200 as vm
from tests import mx_ref as ref
from tests.helpers import random_csr

pytestmark = pytest.mark.gpu
KINDS = {"mxf8": vm.MXF8, "mxf4": vm.MXF4}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = ref.U


def np64(t):
    return t.detach().double().cpu().numpy()


def codes_of(Q):
    """(element codes, scale codes) of an MXDense."""
    data, scale = Q.data.view(torch.uint8).cpu().numpy(), Q.scale.view(torch.uint8).cpu().numpy()
    return (data[:, :Q.cols] if Q.kind == vm.MXF8 else ref.unpack(data, Q.cols)), scale[:, :-(-Q.cols // 32)]


def to_mx(codes, scales, kind, pitch=None):
    """An MXDense of given codes; pitch: bytes from one element row to the next."""
    data = codes if kind == "mxf8" else ref.pack(codes)
    wide = np.zeros((data.shape[0], pitch or data.shape[1]), np.uint8)
    wide[:, :data.shape[1]] = data
    d = torch.from_numpy(wide).cuda()[:, :data.shape[1]]
    return vm.MXDense(d.view(torch.float8_e4m3fn) if kind == "mxf8" else d, torch.from_numpy(scales).cuda(), cols=codes.shape[1])


def features(rows, O, seed, kind="mxf8"):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, O)) * np.exp2(rng.integers(-6, 7, (rows, 1)))
    x[rng.random(rows) < 0.05] = 0
    return ref.quantize(x.astype(np.float32), kind)


# ---- quantise, dequantise --------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,O", [(1, 1), (3, 31), (5, 32), (7, 33), (4, 100), (129, 128), (2, 1009)])
def test_quantize_exact(cuda, kind, dtype, rows, O):
    rng = np.random.default_rng(rows * O)
    spread = 120 if dtype != "f16" else 12
    x = torch.from_numpy(rng.standard_normal((rows, O)) * np.exp2(rng.integers(-spread, spread, (rows, 1)))).to(TYPES[dtype]).cuda()
    x[0, 0] = 0
    codes, scales = ref.quantize(np64(x), kind)
    Q = vm.mx_quantize(x, KINDS[kind])
    got, got_s = codes_of(Q)
    assert np.array_equal(got_s, scales) and np.array_equal(got, codes)
    for t in TYPES.values():
        want = torch.from_numpy(ref.values(codes, scales, kind).astype(np.float32)).to(t)
        assert torch.equal(vm.mx_dequantize(Q, dtype=t).cpu(), want)


@pytest.mark.parametrize("kind", KINDS)
def test_quantize_borders(cuda, kind):
    """Ties, the largest value of the type, one step beyond it, the ends of fp32, zeros, infinities and NaN."""
    grid = ref._grid(kind)
    mid = (grid[1:] + grid[:-1]) / 2
    top = ref.LARGEST[kind]
    rows = [np.append(mid[-31:], top), np.append(-mid[:31], top), np.append(np.nextafter(np.float32(mid[-31:]), np.float32(9e9)), top)]
    rows += [np.full(32, v) for v in (0.0, -0.0, top, np.nextafter(np.float32(top), np.float32(1e9)), 1e-45, 2.0 ** -126, 2.0 ** -127, 3e38,
                                      3.4028234663852886e38)]
    rows += [np.append(np.ones(31), v) for v in (np.inf, -np.inf, np.nan)]
    width = max(len(r) for r in rows)
    x = np.stack([np.pad(r, (0, width - len(r))) for r in rows]).astype(np.float32)
    codes, scales = ref.quantize(x, kind)
    got, got_s = codes_of(vm.mx_quantize(torch.from_numpy(x).cuda(), KINDS[kind]))
    assert np.array_equal(got_s, scales) and np.array_equal(got, codes)
    assert (scales == 255).sum() == 3
    back = vm.mx_dequantize(vm.mx_quantize(torch.from_numpy(x).cuda(), KINDS[kind])).cpu().numpy()
    assert np.isnan(back[-3:]).all() and not np.isnan(back[:-3]).any()


def test_dequantize_every_code(cuda):
    all8, all4 = np.arange(256, dtype=np.uint8).reshape(8, 32), np.arange(16, dtype=np.uint8).reshape(1, 16)
    for scale in (0, 1, 64, 127, 200, 254, 255):
        for kind, codes in (("mxf8", all8), ("mxf4", all4)):
            s = np.full((codes.shape[0], 1), scale, np.uint8)
            got = vm.mx_dequantize(to_mx(codes, s, kind)).cpu().numpy()
            with np.errstate(over="ignore"):
                assert np.array_equal(got, ref.values(codes, s, kind).astype(np.float32), equal_nan=True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shift,pitch", [(0, 144), (8, 144), (1, 133), (3, 131)])
def test_quantize_strides(cuda, kind, shift, pitch):
    """Rows and columns inside larger buffers, whatever their alignment; what lies around them stays."""
    O = 97
    x = torch.randn(6, pitch, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    view = x[1:5, shift:shift + O]
    nb = O if kind == "mxf8" else (O + 1) // 2
    data = torch.full((6, pitch), 77, dtype=torch.uint8, device="cuda")
    scale = torch.full((6, 9), 66, dtype=torch.uint8, device="cuda")
    d = data[1:5, shift:shift + nb]
    out = vm.MXDense(d.view(torch.float8_e4m3fn) if kind == "mxf8" else d, scale[1:5, 2:6], cols=O)
    vm.mx_quantize(view, KINDS[kind], out=out)
    codes, scales = ref.quantize(np64(view), kind)
    got, got_s = codes_of(out)
    assert np.array_equal(got, codes) and np.array_equal(got_s, scales)
    data[1:5, shift:shift + nb] = 77
    scale[1:5, 2:6] = 66
    assert bool((data == 77).all()) and bool((scale == 66).all())
    y = torch.full((6, pitch), 5.0, device="cuda", dtype=torch.bfloat16)
    vm.mx_quantize(view, KINDS[kind], out=out)
    vm.mx_dequantize(out, out=y[1:5, shift:shift + O])
    want = torch.from_numpy(ref.values(codes, scales, kind)).float().bfloat16()
    assert torch.equal(y[1:5, shift:shift + O].cpu(), want)
    y[1:5, shift:shift + O] = 5
    assert bool((y == 5).all())


def test_no_rows(cuda):
    for kind in KINDS.values():
        Q = vm.mx_quantize(torch.zeros(0, 40, device="cuda"), kind)
        assert Q.shape == (0, 40) and vm.mx_dequantize(Q).shape == (0, 40)
        Q, h, inv = vm.add_rms_norm(torch.zeros(0, 40, device="cuda"), torch.ones(40, device="cuda"), kind=kind)
        assert Q.shape == (0, 40) and inv.shape == (0,)
    dx, dw = vm.add_rms_norm_backward(torch.zeros(0, 40, device="cuda"), torch.ones(40, device="cuda"), torch.zeros(0, 40, device="cuda"),
                                      torch.zeros(0, device="cuda"))
    assert dx.shape == (0, 40) and bool((dw == 0).all())


# ---- product ---------------------------------------------------------------------------------------
def sparse(M, N, density, seed, long_row=None, scale=1.0):
    """CSR with fp16 values; every third row empty; `long_row`: that row holds every column."""
    rp, col, val = random_csr(M, N, density, seed, empty_rows=True, scale=scale)
    if long_row is not None:
        rng = np.random.default_rng(seed + 1)
        col = np.concatenate([col[:rp[long_row]], np.arange(N, dtype=np.int32), col[rp[long_row + 1]:]])
        val = np.concatenate([val[:rp[long_row]], (rng.uniform(-1, 1, N) * scale).astype(np.float32), val[rp[long_row + 1]:]])
        rp = rp.copy()
        rp[long_row + 1:] += N - (rp[long_row + 1] - rp[long_row])
    return rp, col.astype(np.int32), val.astype(np.float16).astype(np.float32)


def handle(M, N, rp, col, val, fp32, built="upload", **kw):
    if built == "upload":
        V = vm.csr_to_vcsr_mc(vm.CSR.from_arrays(M, N, rp, col, val), fp32=fp32, segw=32)
        return vm.upload_vcsr_mc_device(V, plans=[vm.PLAN_ROWS], **kw)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return vm.build_vcsr_mc_device(t(rp.astype(np.int32)), t(col), t(val), M, N, fp32=fp32, segw=32, plans=[vm.PLAN_ROWS], **kw)


def check_product(dV, csr, codes, scales, kind, Q=None, start=None):
    rp, col, val = csr
    O = codes.shape[1]
    B = ref.values(codes, scales, kind)
    want, size, n = ref.product(rp, col, val, B)
    C = torch.full((len(rp) - 1, O), 9.0, device="cuda") if start is None else start.clone()
    vm.spmm(dV, to_mx(codes, scales, kind) if Q is None else Q, C, accumulate=start is not None)
    if start is not None:
        want, size = want + np64(start), size + np.abs(np64(start))
    bound = (n + 4) * U * size
    assert np.all(np.abs(np64(C) - want) <= bound), float(np.max(np.abs(np64(C) - want) - bound))
    return C


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("O", [1, 2, 15, 16, 31, 32, 33, 64, 100, 127, 128, 129, 200, 256])
def test_product_widths(cuda, kind, fp32, O):
    M, N = 90, 70
    csr = sparse(M, N, 0.2, O, long_row=4)
    dV = handle(M, N, *csr, fp32, rows_unit_nnz=16)
    codes, scales = features(N, O, O, kind)
    C = check_product(dV, csr, codes, scales, kind)
    start = torch.randn(M, O, device="cuda", generator=torch.Generator("cuda").manual_seed(O))
    check_product(dV, csr, codes, scales, kind, start=start)
    again = torch.empty_like(C)
    vm.spmm(dV, to_mx(codes, scales, kind), again)
    assert torch.equal(again, C), "the same call gives other bits"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("M,N,density,unit,built", [(1, 1, 1.0, 0, "upload"), (1, 5000, 1.0, 0, "build"), (1, 5000, 1.0, 1024, "upload"),
                                                    (2000, 1, 0.5, 0, "build"), (700, 900, 0.02, 0, "upload"), (700, 900, 0.02, 64, "build"),
                                                    (50, 40, 0.0, 0, "upload"), (33, 3000, 0.3, 32, "build")])
def test_product_shapes(cuda, kind, M, N, density, unit, built):
    csr = sparse(M, N, density, M + N)
    dV = handle(M, N, *csr, False, built, rows_unit_nnz=unit)
    codes, scales = features(N, 72, M, kind)
    check_product(dV, csr, codes, scales, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("O,pitch,shift", [(128, 256, 0), (128, 160, 16), (128, 136, 8), (128, 132, 4), (128, 131, 0), (96, 129, 1), (64, 99, 2), (100, 112, 0), (100, 104, 8), (99, 120, 24), (136, 168, 8),
                                           (45, 61, 3)])
def test_product_strides(cuda, kind, O, pitch, shift):
    """B in a larger buffer at any alignment, its scales too; C in a larger buffer whose other columns and rows stay."""
    M, N = 60, 50
    csr = sparse(M, N, 0.3, O, long_row=0)
    dV = handle(M, N, *csr, False, rows_unit_nnz=16)
    codes, scales = features(N, O, pitch, kind)
    data = codes if kind == "mxf8" else ref.pack(codes)
    buf = torch.full((N + 2, pitch + 32), 0xFF, dtype=torch.uint8, device="cuda")
    sbuf = torch.full((N + 2, 13), 0xFF, dtype=torch.uint8, device="cuda")
    # a row stride of `pitch` bytes, starting `shift` bytes into the buffer
    d = torch.as_strided(buf.view(-1), data.shape, (pitch, 1), pitch + shift)
    s = sbuf[1:N + 1, 3:3 + scales.shape[1]]
    d.copy_(torch.from_numpy(data))
    s.copy_(torch.from_numpy(scales))
    Q = vm.MXDense(d.view(torch.float8_e4m3fn) if kind == "mxf8" else d, s, cols=O)
    want, size, n = ref.product(*csr, ref.values(codes, scales, kind))
    for off, ldc in ((0, O), (1, O + 3), (4, O + 8), (8, O + 24)):
        big = torch.full((M + 2, ldc + off), 3.5, device="cuda")
        C = big[1:M + 1, off:off + O]
        vm.spmm(dV, Q, C)
        assert np.all(np.abs(np64(C) - want) <= (n + 4) * U * size)
        C.fill_(3.5)
        assert bool((big == 3.5).all())
    # the first columns of a wider operand
    C = torch.empty(M, O // 2, device="cuda")
    vm.spmm(dV, Q, C, O=O // 2)
    assert np.all(np.abs(np64(C) - want[:, :O // 2]) <= (n + 4) * U * size[:, :O // 2])


@pytest.mark.parametrize("kind", KINDS)
def test_product_special_values(cuda, kind):
    """NaN scales reach exactly the rows and blocks that use them; unused and padded places reach nothing."""
    M, N, O = 40, 64, 96
    rp, col, val = sparse(M, N, 0.2, 3, long_row=5)  # 64 entries of row 5 in chunks of 16
    keep = np.ones(len(col), bool)
    keep[(col == 0) | (col == 7)] = False  # rows 0 and 7 of B are used by nobody
    keep[rp[5] + 10:rp[5] + 13] = False    # row 5's last chunk is not whole
    lens = np.array([keep[rp[r]:rp[r + 1]].sum() for r in range(M)])
    col, val = col[keep], val[keep]
    rp = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    dV = handle(M, N, rp, col, val, False, rows_unit_nnz=16)
    codes, scales = features(N, O, 4, kind)
    scales[0], scales[7] = 255, 255
    if kind == "mxf8":
        codes[0] = 0x7F
    C = check_product(dV, (rp, col, val), codes, scales, kind)
    assert bool(torch.isfinite(C).all())
    scales[9, 1] = 255
    C2 = torch.empty_like(C)
    vm.spmm(dV, to_mx(codes, scales, kind), C2)
    uses = np.array([9 in col[rp[r]:rp[r + 1]] for r in range(M)])
    nan = torch.isnan(C2).cpu().numpy()
    assert nan[uses][:, 32:64].all() and not nan[~uses].any() and not nan[:, :32].any() and not nan[:, 64:].any()


def test_product_scaled_format_hot_columns_and_extremes(cuda):
    M, N, O = 80, 60, 64
    for scale in (1e6, 1e-7):
        csr = sparse(M, N, 0.3, 5)
        csr = (csr[0], csr[1], (csr[2] * np.float32(scale)).astype(np.float32))
        V = vm.csr_to_vcsr_mc(vm.CSR.from_arrays(M, N, *csr), fp32=False, segw=32)
        assert V.scale != 1.0
        dV = vm.upload_vcsr_mc_device(V, plans=[vm.PLAN_ROWS])
        held = ((csr[2] / np.float32(V.scale)).astype(np.float16).astype(np.float64) * np.float64(np.float32(V.scale)))
        check_product(dV, (csr[0], csr[1], held), *features(N, O, 6, "mxf4"), "mxf4")
    csr = sparse(M, N, 0.3, 5, long_row=2)
    dV = handle(M, N, *csr, True, hot_rows=20)
    assert dV.info()["n_hot"] > 0
    check_product(dV, csr, *features(N, O, 6, "mxf4"), "mxf4")
    # scales at both ends of their range, in different rows and blocks
    codes, scales = features(N, O, 7, "mxf8")
    scales[::2, 0], scales[1::2, 0], scales[:, 1] = 100, 4, 230
    check_product(dV, csr, codes, scales, "mxf8")


def test_product_ends_of_the_scale_range(cuda):
    """Code 0 and subnormal products count as zero, code 254 as what it says; in the FP16 and the FP32 format."""
    M, N, O = 33, 40, 96
    csr = sparse(M, N, 0.4, 9)
    codes, scales = features(N, O, 10, "mxf8")
    scales[:, 0], scales[::2, 1], scales[1::2, 1], scales[:, 2] = 0, 0, 127, 254
    codes[:, 64:] &= 0x87  # subnormal elements, so that the sums stay finite
    known = scales.copy()
    known[known == 0] = 127
    zeroed = codes.copy()
    zeroed[np.repeat(scales == 0, 32, 1)] = 0
    want, size, n = ref.product(*csr, ref.values(zeroed, known, "mxf8"))
    for fp32 in (False, True):
        dV = handle(M, N, *csr, fp32)
        C = torch.empty(M, O, device="cuda")
        vm.spmm(dV, to_mx(codes, scales, "mxf8"), C)
        assert np.all(np.abs(np64(C) - want) <= (n + 4) * U * size)


@pytest.mark.parametrize("M,N", [(0, 7), (7, 0), (1, 1)])
def test_product_empty_matrices(cuda, M, N):
    rp, none = np.zeros(M + 1, np.int32), np.zeros(0)
    dV = handle(M, N, rp, none.astype(np.int32), none.astype(np.float32), False)
    Q = vm.mx_quantize(torch.ones(N, 33, device="cuda"), vm.MXF4)
    C = torch.full((M, 33), 5.0, device="cuda")
    vm.spmm(dV, Q, C, accumulate=True)
    assert bool((C == 5).all())
    vm.spmm(dV, Q, C)
    assert bool((C == 0).all())


def test_product_far_offsets(cuda):
    """An operand and a result past 4 GiB, and scales past 2^31 bytes into their array's rows."""
    N, M, O = 34_000_000, 9_000_000, 130  # elements of 144-byte rows: 4.9 GB; C 4.7 GB
    data = torch.zeros(N, 144, dtype=torch.uint8, device="cuda")
    scale = torch.full((N, 64), 127, dtype=torch.uint8, device="cuda")
    cols = torch.tensor([0, 7, N // 2 + 1, N - 2, N - 1], device="cuda")
    codes, scales = features(5, O, 3, "mxf8")
    data[cols, :O] = torch.from_numpy(codes).cuda()
    scale[cols, 57:62] = torch.from_numpy(scales).cuda()
    Q = vm.MXDense(data[:, :O].view(torch.float8_e4m3fn), scale[:, 57:62], cols=O)
    rp = torch.zeros(M + 1, dtype=torch.int32, device="cuda")
    rp[1:] = 2
    rp[M:] = 5
    dV = vm.build_vcsr_mc_device(rp, cols[torch.tensor([0, 3, 1, 2, 4], device="cuda")].int(), torch.tensor([1.0, 2, 0.5, -1, 4], device="cuda"), M, N,
                                 segw=32, plans=[vm.PLAN_ROWS])
    C = torch.full((M, O), 9.0, device="cuda")
    vm.spmm(dV, Q, C)
    B = ref.values(codes, scales, "mxf8")
    for row, want in ((0, B[0] + 2 * B[3]), (M - 1, 0.5 * B[1] - B[2] + 4 * B[4])):
        assert np.all(np.abs(np64(C[row]) - want) <= 7 * U * np.abs(4 * B).sum(0))
    assert not bool(C[1:M - 1].any())


def test_product_refusals(cuda):
    M, N = 20, 130
    csr = sparse(M, N, 0.3, 5, long_row=1)
    dV = handle(M, N, *csr, False, rows_unit_nnz=16)
    codes, scales = features(N, 64, 1, "mxf8")
    Q, C = to_mx(codes, scales, "mxf8"), torch.empty(M, 64, device="cuda")
    short = to_mx(codes[:-1], scales[:-1], "mxf8")
    for call in (lambda: vm.spmm(dV, short, C), lambda: vm.spmm(dV, Q, C[:-1]), lambda: vm.spmm(dV, Q, C, O=65),
                 lambda: vm.spmm(dV, Q, C.half()), lambda: vm.spmm(dV, Q, C, plan=vm.PLAN_BAND), lambda: vm.spmm(dV, Q, C, tileK=77),
                 lambda: vm.spmm(dV, Q, C.cpu()), lambda: vm.spmm(dV, Q, C, O=0)):
        with pytest.raises(vm.VcsrmcError):
            call()
    from vcsr_mc_b200 import _lib
    with pytest.raises(vm.VcsrmcError):  # no workspace for the split row
        _lib.call("vcsrmc_spmm_mx", dV.handle, Q.data.data_ptr(), Q.kind, 64, Q.scale.data_ptr(), 2, 64, C.data_ptr(), 64, 0, None, 0, None)
    only_segment = vm.upload_vcsr_mc_device(vm.csr_to_vcsr_mc(vm.CSR.from_arrays(M, N, *csr), segw=32), plans=[vm.PLAN_SEGMENT])
    with pytest.raises(vm.VcsrmcError):
        vm.spmm(only_segment, Q, C)
    check_product(dV, csr, codes, scales, "mxf8")


# ---- norm ------------------------------------------------------------------------------------------
def check_norm(Q, inv, s, w, eps, kind):
    y, want_inv = ref.norm(np64(s), np64(w), eps)
    assert np.all(np.abs(np64(inv) - want_inv) <= 2 * U * want_inv)
    codes, scales = codes_of(Q)
    lo, hi = ref.scale_codes(y * (1 - 4 * U), kind), ref.scale_codes(y * (1 + 4 * U), kind)
    assert np.all((scales >= lo) & (scales <= hi))
    two = np.exp2(np.repeat(scales, 32, 1)[:, :y.shape[1]].astype(float) - 127)
    got = ref.element_values(codes, kind)
    grid = ref._grid(kind)
    at = np.searchsorted(grid, np.abs(got))
    up = np.append(grid, 2 * grid[-1] - grid[-2])[at + 1] - np.abs(got)
    down = np.abs(got) - np.where(at > 0, grid[at - 1], -grid[1])
    off = np.abs(y) / two - np.abs(got)
    slack = 4 * U * np.abs(y) / two
    assert np.all(off <= up / 2 + slack) and np.all(-off <= down / 2 + slack)
    assert np.all((np.sign(got) == np.sign(y)) | (got == 0))


COMBOS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
WIDTHS = [1, 7, 32, 33, 64, 100, 128, 250, 256, 500, 1000, 1024, 1025, 2048, 4096, 5000, 16384, 32768, 32769, 40000]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("x,r", COMBOS)
@pytest.mark.parametrize("O", WIDTHS)
def test_norm(cuda, kind, x, r, O):
    rows = 9 if O < 2000 else 3
    g = torch.Generator("cuda").manual_seed(O)
    X = torch.randn(rows, O, device="cuda", generator=g).to(TYPES[x])
    R = (torch.randn(rows, O, device="cuda", generator=g) * 3).to(TYPES[r])
    w = (1 + 0.2 * torch.randn(O, device="cuda", generator=g)).to(TYPES[r])
    X[0], R[0] = 0, 0  # a row of zeros
    Q, h, inv = vm.add_rms_norm(X, w, residual=R, eps=1e-5, kind=KINDS[kind])
    s = (X.float() + R.float()).to(TYPES[r])
    assert torch.equal(h, s)
    check_norm(Q, inv, s, w, 1e-5, kind)
    # in place on the residual, and a weight of another type
    keep = R.clone()
    Q2, h2, inv2 = vm.add_rms_norm(X, w.float(), residual=keep, eps=1e-5, kind=KINDS[kind], residual_out=keep)
    assert h2.data_ptr() == keep.data_ptr() and torch.equal(keep, s) and torch.equal(inv2, inv)
    assert torch.equal(Q2.data.view(torch.uint8), Q.data.view(torch.uint8)) and torch.equal(Q2.scale.view(torch.uint8), Q.scale.view(torch.uint8))
    # without a residual
    Q3, h3, inv3 = vm.add_rms_norm(X, w, eps=1e-5, kind=KINDS[kind])
    assert h3 is X
    check_norm(Q3, inv3, X, w, 1e-5, kind)


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 1000])
def test_norm_rows_and_strides(cuda, rows):
    O, ld = 72, 91
    g = torch.Generator("cuda").manual_seed(rows)
    X, R = torch.randn(rows, ld, device="cuda", generator=g)[:, 3:3 + O], torch.randn(rows, ld, device="cuda", generator=g).half()[:, 5:5 + O]
    w = torch.randn(O, device="cuda", generator=g).half()
    big = torch.full((rows + 2, ld), 2.0, device="cuda", dtype=torch.float16)
    Q, h, inv = vm.add_rms_norm(X, w, residual=R, residual_out=big[1:rows + 1, 7:7 + O])
    s = (X + R.float()).half()
    assert torch.equal(h, s)
    check_norm(Q, inv, s, w, 1e-6, "mxf8")
    h.fill_(2.0)
    assert bool((big == 2).all())


def test_norm_extremes(cuda):
    """Sums of squares that leave fp32's range, infinities and NaN stay in their rows."""
    X = torch.ones(6, 64, device="cuda")
    X[1] *= 1e25
    X[2] *= 1e-25
    X[3, 5] = float("inf")
    X[4, 40] = float("nan")
    w = torch.ones(64, device="cuda")
    Q, _, inv = vm.add_rms_norm(X, w, eps=0.0)
    keep = [0, 1, 2, 5]
    check_norm(vm.MXDense(Q.data[keep].view(torch.uint8).view(torch.float8_e4m3fn), Q.scale.view(torch.uint8)[keep].contiguous()), inv[keep],
               X[keep], w, 0.0, "mxf8")
    y = vm.mx_dequantize(Q)
    assert bool(torch.isnan(y[3, :32]).all()) and bool((y[3, 32:] == 0).all()) and bool(torch.isnan(y[4]).all())


@pytest.mark.parametrize("x,r", COMBOS)
@pytest.mark.parametrize("rows,O", [(1, 1), (5, 32), (70, 33), (300, 128), (2500, 100), (40, 1000), (17, 1025), (700, 2048), (6, 8192), (5, 16385), (3, 40000)])
def test_norm_backward(cuda, x, r, rows, O):
    g = torch.Generator("cuda").manual_seed(rows + O)
    dY = torch.randn(rows, O, device="cuda", generator=g).to(TYPES[x])
    dR, h = (torch.randn(rows, O, device="cuda", generator=g).to(TYPES[r]) for _ in range(2))
    w = (1 + 0.2 * torch.randn(O, device="cuda", generator=g)).to(TYPES[r])
    h[0] = 0
    inv = (1 / torch.sqrt(h.double().square().mean(1) + 1e-5)).float()
    for d_residual in (dR, None):
        dx, dw, size, dw_size = ref.norm_backward(np64(dY), np64(w), np64(h), np64(inv), None if d_residual is None else np64(d_residual))
        got, got_w = vm.add_rms_norm_backward(dY, w, h, inv, d_residual=d_residual)
        half = torch.finfo(TYPES[r]).eps / 2
        tiny = float(torch.finfo(TYPES[r]).smallest_normal) * float(torch.finfo(TYPES[r]).eps)  # a step of the type's subnormals
        assert got.dtype == TYPES[r] and got_w.dtype == torch.float32
        assert np.all(np.abs(np64(got) - dx) <= half * np.abs(dx) + 8 * U * size * (1 + half) + tiny)
        assert np.all(np.abs(np64(got_w) - dw) <= (rows + 4) * U * dw_size)
        again, again_w = vm.add_rms_norm_backward(dY, w, h, inv, d_residual=d_residual)
        assert torch.equal(again, got) and torch.equal(again_w, got_w)
    place = dR.clone()
    out, _ = vm.add_rms_norm_backward(dY, w, h, inv, d_residual=place, out=place)
    assert out.data_ptr() == place.data_ptr()
    want, _ = vm.add_rms_norm_backward(dY, w, h, inv, d_residual=dR)
    assert torch.equal(place, want)


def test_norm_backward_against_differences(cuda):
    """The chain x -> norm -> values, through the library's own forward statistics, against differences of the 64-bit forward."""
    g = torch.Generator("cuda").manual_seed(3)
    X, R = (torch.randn(2, 40, device="cuda", generator=g) for _ in range(2))
    w, G, D = torch.randn(40, device="cuda", generator=g), torch.randn(2, 40, device="cuda", generator=g), torch.randn(2, 40, device="cuda", generator=g)
    _, h, inv = vm.add_rms_norm(X, w, residual=R, eps=1e-3)
    dx, dw = vm.add_rms_norm_backward(G, w, h, inv, d_residual=D)
    x, r, wd, gd, dd = (np64(t) for t in (X, R, w, G, D))

    def loss(x, w):
        s = x + r
        return (ref.norm(s, w, 1e-3)[0] * gd).sum() + (s * dd).sum()

    step = 1e-4  # differences: O(step^2) ~ 1e-7 of terms of order 10; fp32 results: 8 u of terms of order 10
    for i in range(2):
        for j in range(0, 40, 7):
            d = np.zeros((2, 40))
            d[i, j] = step
            assert abs((loss(x + d, wd) - loss(x - d, wd)) / (2 * step) - float(dx[i, j])) < 1e-4
    for j in range(40):
        d = np.zeros(40)
        d[j] = step
        assert abs((loss(x, wd + d) - loss(x, wd - d)) / (2 * step) - float(dw[j])) < 1e-4


def test_products_in_flight_together(cuda):
    """One handle on two streams at once, rows split into chunks: each product has its own workspace."""
    M, N, O = 40, 4000, 128
    csr = sparse(M, N, 0.5, 11)
    dV = handle(M, N, *csr, False, rows_unit_nnz=16)
    Qs = [to_mx(*features(N, O, 20 + i, "mxf4"), "mxf4") for i in range(2)]
    alone = [vm.spmm(dV, Q, torch.empty(M, O, device="cuda")) for Q in Qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = [[torch.empty(M, O, device="cuda") for _ in range(20)] for _ in range(2)]
    torch.cuda.synchronize()
    for k in range(20):
        for i in range(2):
            vm.spmm(dV, Qs[i], results[i][k], stream=streams[i])
    torch.cuda.synchronize()
    assert all(torch.equal(C, alone[i]) for i in range(2) for C in results[i])


# ---- together ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", KINDS)
def test_layers_run_captured_and_on_streams(cuda, kind):
    """Products and norms in turn over one matrix, as feature propagation uses them: eagerly, captured in two graphs that replay in turn
    and on two streams at once, always to the same bits; and the way back through the transposed matrix."""
    M, O = 400, 96
    rp, col, val = sparse(M, M, 0.03, 8, long_row=3)
    dV = handle(M, M, rp, col, val, False, rows_unit_nnz=32)
    g = torch.Generator("cuda").manual_seed(4)
    X0, w = torch.randn(M, O, device="cuda", generator=g).half(), torch.ones(O, device="cuda", dtype=torch.float16)

    def layers(X):
        C = torch.empty(M, O, device="cuda")
        h, Q = X, vm.mx_quantize(X, KINDS[kind])
        for _ in range(3):
            vm.spmm(dV, Q, C)
            Q, h, inv = vm.add_rms_norm(C, w, residual=h, kind=KINDS[kind])
        return C, h, inv

    eager = layers(X0)
    eager += vm.add_rms_norm_backward(eager[0], w, eager[1], eager[2], d_residual=eager[1])
    # layer by layer against the definitions, from the library's own inputs of each step
    Q = vm.mx_quantize(X0, KINDS[kind])
    C = check_product(dV, (rp, col, val), *codes_of(Q), kind)
    Q, h, inv = vm.add_rms_norm(C, w, residual=X0, kind=KINDS[kind])
    check_norm(Q, inv, (C + X0.float()).half(), w, 1e-6, kind)
    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):
        X = X0.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm = layers(X)
            vm.add_rms_norm_backward(warm[0], w, warm[1], warm[2], d_residual=warm[1])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layers(X)
            out += vm.add_rms_norm_backward(out[0], w, out[1], out[2], d_residual=out[1])
        graphs.append((graph, X, out))
    graphs[1][1].copy_(X0 * 2)
    two = layers(X0 * 2)
    two += vm.add_rms_norm_backward(two[0], w, two[1], two[2], d_residual=two[1])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s1):
            graphs[0][0].replay()
        with torch.cuda.stream(s2):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][2], eager)) and all(torch.equal(a, b) for a, b in zip(graphs[1][2], two))
    # an explicit stream that is not the current one
    s1.wait_stream(torch.cuda.current_stream())
    Q = vm.mx_quantize(X0, KINDS[kind], stream=s1)
    C = torch.empty(M, O, device="cuda")
    s1.wait_stream(torch.cuda.current_stream())
    vm.spmm(dV, Q, C, stream=s1.cuda_stream)
    s1.synchronize()
    first = torch.empty_like(C)
    vm.spmm(dV, vm.mx_quantize(X0, KINDS[kind]), first)
    assert torch.equal(C, first)
    # back: dB = A^T dC, with dC microscaled
    order = np.argsort(col, kind="stable")
    rows = np.repeat(np.arange(M), np.diff(rp))[order]
    rpt = np.concatenate([[0], np.cumsum(np.bincount(col, minlength=M))]).astype(np.int32)
    dT = handle(M, M, rpt, rows.astype(np.int32), val[order], False)
    dC = vm.mx_quantize(torch.randn(M, O, device="cuda", generator=g), KINDS[kind])
    dB = check_product(dT, (rpt, rows, val[order]), *codes_of(dC), kind)
    dx, dw = vm.add_rms_norm_backward(dB, w, eager[1], eager[2])
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(dw).all())


@pytest.mark.parametrize("O", [24, 33, 128])
def test_driver_microscaled(cuda, O):
    """spmm_vcsr's microscaled algorithms pass its own check against the fp64 product with the values that B then stands for."""
    import csv
    import io
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([os.path.join(root, "vcsr_mc_b200", "spmm_vcsr"), "--gen", "c1", "--O", str(O), "--algo", "vcsr_mc,vcsr_mc_mxf8,vcsr_mc_mxf4",
                          "--bdist", "normal", "--repeat", "2", "--warmup", "1", "--csv"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    rows = {r["algo"]: r for r in csv.DictReader(io.StringIO(out.stdout))}
    assert set(rows) == {"vcsr_mc", "vcsr_mc_mxf8", "vcsr_mc_mxf4"}
    assert all(r["validation"] == "pass" and float(r["gbps_alg"]) > 0 for r in rows.values())
    # fp16 values of A are all that is rounded: half a step of 2^-11 at most, and the check's bound of 3e-3 is far
    assert all(float(rows[k]["rel_l2"]) <= 2.0 ** -11 for k in ("vcsr_mc_mxf8", "vcsr_mc_mxf4"))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("O", [64, 100, 512, 1056])
def test_norm_scales_at_their_borders(cuda, kind, O):
    """Blocks whose largest value lies within a few units of fp32's last place of the border between two scales: the scale is the
    64-bit definition's, for every block (64-bit sums and three 64-bit roundings reach 2^-50, and no value is built nearer than 2^-40)."""
    rng = np.random.default_rng(O)
    rows, top = 600, ref.LARGEST[kind]
    x = rng.standard_normal((rows, O)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(O)).astype(np.float32)
    # column 3 holds the first block's largest value, at the border's value T but for a few 2^-24: x with x w / sqrt((S + x^2) / O + eps) = T
    x[:, :32] *= 0.2
    border = top * 2.0 ** np.ceil(np.log2(1.4 / top))
    T = border * (1 + rng.integers(-4, 5, rows) * 2.0 ** -24) / w[3].astype(np.float64)
    S = (np.delete(x, 3, 1).astype(np.float64) ** 2).sum(1)
    x[:, 3] = T * np.sqrt((S + O * 1e-6) / (O - T * T))
    y, _ = ref.norm(x, w, 1e-6)
    amax = np.abs(y[:, :32]).max(1)
    off = np.abs(amax / border - 1)
    keep = off > 2.0 ** -40
    Q, _, _ = vm.add_rms_norm(torch.from_numpy(x).cuda(), torch.from_numpy(w).cuda(), eps=1e-6, kind=KINDS[kind])
    codes, scales = codes_of(Q)
    assert np.array_equal(scales[keep, 0], ref.scale_codes(y, kind)[keep, 0])
    check_norm(Q, torch.from_numpy(1 / np.sqrt((x.astype(np.float64) ** 2).mean(1) + 1e-6)).cuda().float(), torch.from_numpy(x), torch.from_numpy(w), 1e-6, kind)
    assert (off < 2.0 ** -21).sum() > 50, "too few rows at the border"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("x,r", [("f32", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("O", [8, 40, 96, 264, 1032, 4104])
def test_norm_in_odd_places(cuda, kind, x, r, O):
    """Every operand at an odd offset of a larger buffer (the weight and the MX matrix too), forward and backward; what lies around them stays."""
    rows, g = 37, torch.Generator("cuda").manual_seed(O)

    def place(t, fill):
        big = torch.full((t.shape[0] + 2, t.shape[1] + 5), fill, dtype=t.dtype, device="cuda")
        view = big[1:-1, 3:3 + t.shape[1]]
        view.copy_(t)
        return big, view

    X = place(torch.randn(rows, O, device="cuda", generator=g).to(TYPES[x]), 7)[1]
    R = place(torch.randn(rows, O, device="cuda", generator=g).to(TYPES[r]), 7)[1]
    w = (1 + 0.2 * torch.randn(O + 1, device="cuda", generator=g)).to(TYPES[r])[1:]
    big_h, H = place(torch.zeros(rows, O, device="cuda", dtype=TYPES[r]), 7)
    nb = O if kind == "mxf8" else O // 2
    big_q, D = place(torch.zeros(rows, nb, dtype=torch.uint8, device="cuda"), 77)
    big_s, S = place(torch.zeros(rows, -(-O // 32), dtype=torch.uint8, device="cuda"), 66)
    out = vm.MXDense(D.view(torch.float8_e4m3fn) if kind == "mxf8" else D, S, cols=O)
    Q, h, inv = vm.add_rms_norm(X, w, residual=R, kind=KINDS[kind], out=out, residual_out=H)
    assert Q is out and h is H
    s = (X.float() + R.float()).to(TYPES[r])
    assert torch.equal(H, s)
    check_norm(out, inv, s, w, 1e-6, kind)
    dY = place(torch.randn(rows, O, device="cuda", generator=g).to(TYPES[x]), 7)[1]
    big_d, dR = place(torch.randn(rows, O, device="cuda", generator=g).to(TYPES[r]), 7)
    dx, dw, size, dw_size = ref.norm_backward(np64(dY), np64(w), np64(H), np64(inv), np64(dR))
    got, got_w = vm.add_rms_norm_backward(dY, w, H, inv, d_residual=dR, out=dR)  # in place
    half = torch.finfo(TYPES[r]).eps / 2
    assert got is dR and np.all(np.abs(np64(got) - dx) <= half * np.abs(dx) + 8 * U * size * (1 + half) + 2.0 ** -24)
    assert np.all(np.abs(np64(got_w) - dw) <= (rows + 4) * U * dw_size)
    for big, view, fill in ((big_h, H, 7), (big_q, D, 77), (big_s, S, 66), (big_d, dR, 7)):
        view.fill_(fill)
        assert bool((big == fill).all())


def test_norm_refusals_with_tensors(cuda):
    X, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    half = X.half()
    Q, h, inv = vm.add_rms_norm(X, w, residual=X)
    for call in (lambda: vm.add_rms_norm(X, w[:63]), lambda: vm.add_rms_norm(X, w.cpu()), lambda: vm.add_rms_norm(X, w.double()),
                 lambda: vm.add_rms_norm(half, w, residual=X), lambda: vm.add_rms_norm(X, w, residual=X[:3]),
                 lambda: vm.add_rms_norm(X, w, residual=half, residual_out=X), lambda: vm.add_rms_norm(X, w, eps=-1.0),
                 lambda: vm.add_rms_norm(X, w, kind=vm.F16), lambda: vm.add_rms_norm(X, w, kind=vm.MXF4, out=Q),
                 lambda: vm.add_rms_norm(X.t(), w), lambda: vm.add_rms_norm(X[0], w), lambda: vm.add_rms_norm(X.expand(2, 4, 64)[0].double(), w),
                 lambda: vm.add_rms_norm(X[:1].expand(4, 64), w), lambda: vm.add_rms_norm(X, None),
                 lambda: vm.add_rms_norm_backward(X, w, h, inv.half()), lambda: vm.add_rms_norm_backward(half, w, h, inv),
                 lambda: vm.add_rms_norm_backward(X, w, h, inv[:3]), lambda: vm.add_rms_norm_backward(X, w, h, inv, out=half),
                 lambda: vm.mx_quantize(X, 9), lambda: vm.mx_quantize(X.long()), lambda: vm.mx_dequantize(Q, dtype=torch.float16, out=X),
                 lambda: vm.mx_dequantize(Q, out=X[:, :32])):
        with pytest.raises((vm.VcsrmcError, RuntimeError)):
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("O", [100, 128, 1000, 16392])
def test_norm_in_place_on_its_first_operand(cuda, O):
    """residual_out is X, and dX is dY: the same bits as in tensors of their own."""
    g = torch.Generator("cuda").manual_seed(O)
    X, R, dY = (torch.randn(70, O, device="cuda", generator=g).half() for _ in range(3))
    w = torch.randn(O, device="cuda", generator=g)
    for residual in (R, None):
        Q, h, inv = vm.add_rms_norm(X, w, residual=residual)
        h = h.clone()
        place = X.clone()
        Q2, h2, inv2 = vm.add_rms_norm(place, w, residual=residual, residual_out=place)
        assert h2 is place and torch.equal(place, h) and torch.equal(inv2, inv)
        assert all(np.array_equal(a, b) for a, b in zip(codes_of(Q), codes_of(Q2)))
        dx, dw = vm.add_rms_norm_backward(dY, w, h, inv, d_residual=residual)
        place = dY.clone()
        dx2, dw2 = vm.add_rms_norm_backward(place, w, h, inv, d_residual=residual, out=place)
        assert dx2 is place and torch.equal(dx2, dx) and torch.equal(dw2, dw)


@pytest.mark.parametrize("rows,O", [(540_000_000, 1), (17_000_000, 136)])
def test_many_rows(cuda, rows, O):
    """More than 2^31 values, and more groups of them than a launch numbers: the first rows, the last, and those around each border."""
    kind, nb = ("mxf4", (O + 1) // 2) if O == 1 else ("mxf8", O)
    X = torch.zeros(rows, O, dtype=torch.float16, device="cuda")
    picks = sorted({r for b in (0, (1 << 31) // O, (1 << 31) // (2 * O), 0x7f000000 // 4, 0x7f000000 // (16 if O == 1 else 32), rows) for r in range(b - 3, b + 3)
                    if 0 <= r < rows})
    at = torch.tensor(picks, device="cuda")
    X[at] = torch.randn(len(picks), O, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    x = np64(X[at])
    data = torch.full((rows, nb), 77, dtype=torch.uint8, device="cuda")
    scale = torch.full((rows, -(-O // 32)), 66, dtype=torch.uint8, device="cuda")
    out = vm.MXDense(data.view(torch.float8_e4m3fn) if kind == "mxf8" else data, scale, cols=O)
    want_codes, want_scales = ref.quantize(x.astype(np.float32), kind)

    def check_rest():
        used = torch.zeros(rows, dtype=torch.bool, device="cuda")
        used[at] = True
        assert int((data != 0).any(1).logical_and(~used).sum()) == 0 and int((scale != 0).any(1).logical_and(~used).sum()) == 0

    vm.mx_quantize(X, KINDS[kind], out=out)
    got = data[at].cpu().numpy() if kind == "mxf8" else ref.unpack(data[at].cpu().numpy(), O)
    assert np.array_equal(got, want_codes) and np.array_equal(scale[at].cpu().numpy(), want_scales)
    check_rest()
    Y = torch.full((rows, O), 9.0, dtype=torch.float16, device="cuda")
    vm.mx_dequantize(out, out=Y)
    assert np.array_equal(np64(Y[at]), ref.values(want_codes, want_scales, kind).astype(np.float16).astype(np.float64))
    assert int((Y != 0).any(1).sum()) <= len(picks)
    # the norm of the same rows; rows of zeros have zeros and 1 / sqrt(eps)
    w = torch.full((O,), 1.5, device="cuda")
    _, h, inv = vm.add_rms_norm(X, w, kind=KINDS[kind], out=out, eps=1e-4)
    check_norm(vm.MXDense(out.data.view(torch.uint8)[at].view(out.data.dtype), scale[at], cols=O), inv[at], X[at], w, 1e-4, kind)
    check_rest()
    dx, dw, size, dw_size = ref.norm_backward(x, np64(w), x, np64(inv[at]), None)
    got, got_w = vm.add_rms_norm_backward(X, w, X, inv, out=Y)
    assert np.all(np.abs(np64(got[at]) - dx) <= 2.0 ** -11 * np.abs(dx) + 8 * U * size * (1 + 2.0 ** -11) + 2.0 ** -24)
    assert np.all(np.abs(np64(got_w) - dw) <= (len(picks) + 4) * U * dw_size)  # terms of zero round nothing
    assert int((got != 0).any(1).sum()) <= len(picks)


def test_default_stream_by_its_handle(cuda):
    """stream=0, the default stream's handle as torch gives it: every call runs behind what that stream already holds, while another stream
    is the current one."""
    from vcsr_mc_b200.api import _stream_guard
    device = torch.device("cuda", torch.cuda.current_device())
    default = torch.cuda.default_stream(device)
    for given in (0, 1, default.cuda_stream, default):
        with _stream_guard(given, device):
            assert torch.cuda.current_stream() == default
    M, O = 64, 40
    csr = sparse(M, M, 0.3, 2)
    dV = handle(M, M, *csr, False)
    g = torch.Generator("cuda").manual_seed(5)
    new, w = torch.randn(M, O, device="cuda", generator=g), torch.ones(O, device="cuda")

    def calls(X, Y, C, h, inv, stream):
        Q = vm.mx_quantize(X, vm.MXF8, stream=stream)
        vm.mx_dequantize(Q, out=Y, stream=stream)
        vm.spmm(dV, Q, C, stream=stream)
        N, H, I = vm.add_rms_norm(C, w, residual=X, stream=stream)
        return (Q.data, Q.scale, Y, C, N.data, N.scale, H, I) + tuple(vm.add_rms_norm_backward(X, w, h, inv, stream=stream))

    inv = 1 / torch.sqrt(new.square().mean(1) + 1e-6)
    want = calls(new, torch.empty_like(new), torch.empty(M, O, device="cuda"), new, inv, None)
    X, h = torch.zeros_like(new), torch.zeros_like(new)
    Y, C, side = torch.empty_like(new), torch.empty(M, O, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda._sleep(40_000_000)  # about 20 ms, before X is there
    X.copy_(new)
    h.copy_(new)
    with torch.cuda.stream(side):
        got = calls(X, Y, C, h, inv, default.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))


def scale_rows(scales, pitch, fill):
    """Scales on rows `pitch` bytes apart, in an array that ends with the last row's last scale; the bytes between rows hold `fill`."""
    N, blocks = scales.shape
    flat = torch.from_numpy(np.resize(np.asarray(fill, np.uint8), (N - 1) * pitch + blocks)).cuda()
    view = torch.as_strided(flat, (N, blocks), (pitch, 1))
    view.copy_(torch.from_numpy(scales))
    return view


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("O,first", [(65, None), (72, None), (96, None), (200, None), (224, None), (256, 70)])
def test_product_padded_scales(cuda, kind, O, first):
    """Scale rows of whole words whose slab has three blocks: whatever stands in the fourth byte (or the blocks of columns that are not asked
    for), the results are the same bits. The last row is an entry, and the array ends with its last scale."""
    M, N = 70, 50
    csr = sparse(M, N, 0.3, O, long_row=4)
    codes, scales = features(N, O, O, kind)
    blocks = scales.shape[1]
    want, size, n = ref.product(*csr, ref.values(codes, scales, kind)[:, :first])
    data = to_mx(codes, scales, kind, pitch=(codes.shape[1] + 15) // 16 * 16 if kind == "mxf8" else None).data
    rng = np.random.default_rng(O)
    for fp32 in (False, True):
        dV, seen = handle(M, N, *csr, fp32, rows_unit_nnz=16), []
        for fill in (0, 255, 1, rng.integers(0, 256, N * 8)):
            held = scales.copy()
            if first:
                held[:, 3:] = np.resize(fill, (N, blocks - 3))
            C = torch.empty(M, first or O, device="cuda")
            vm.spmm(dV, vm.MXDense(data, scale_rows(held, (blocks + 3) // 4 * 4, fill), cols=O), C, O=first)
            assert np.all(np.abs(np64(C) - want) <= (n + 4) * U * size)
            seen.append(C)
        assert all(torch.equal(C, seen[0]) for C in seen)


def test_product_time_does_not_follow_padding(cuda):
    """The bytes behind a row's last scale do not choose the form of the product: the least of ten times is the same within a few percent
    (the fp32 form, which a 255 there once chose, takes 15 % longer here)."""
    M, O = 1 << 18, 96
    g = torch.Generator("cuda").manual_seed(1)
    key = torch.unique(torch.randint(0, M * M, (16 * M,), device="cuda", generator=g))
    rp = torch.zeros(M + 1, dtype=torch.int32, device="cuda")
    rp[1:] = torch.cumsum(torch.bincount(key // M, minlength=M), 0)
    val = (torch.rand(key.numel(), device="cuda", generator=g) * 2 - 1).half().float()
    dV = vm.build_vcsr_mc_device(rp, (key % M).int(), val, M, M, segw=32, plans=[vm.PLAN_ROWS])
    Q = vm.mx_quantize(torch.randn(M, O, device="cuda", generator=g), vm.MXF8)
    rows = torch.as_strided(Q.scale.view(torch.uint8), (M, 4), (4, 1))
    assert Q.scale.stride(0) == 4
    C, best = torch.empty(M, O, device="cuda"), {0: 1e9, 255: 1e9}
    for _ in range(10):
        for fill in best:
            rows[:, 3] = fill
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            torch.cuda._sleep(400_000)
            a.record()
            for _ in range(6):
                vm.spmm(dV, Q, C)
            b.record()
            torch.cuda.synchronize()
            best[fill] = min(best[fill], a.elapsed_time(b))
    assert best[255] < 1.07 * best[0], best


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("O,pitch", [(24, 32), (64, 64), (128, 128), (120, 120), (100, 100), (101, 101)])
def test_product_changes_form_within_a_unit(cuda, kind, O, pitch):
    """FP16 format: batches of eight entries whose scales fit the fp16 form of a unit, then do not, then do again, in rows that end with a batch,
    inside one or after several. Rows of small values stand between rows of large ones, so a factor left behind by a change shows in them."""
    lens = [8, 8, 8, 8, 8, 5, 3, 0, 8, 13, 11, 0, 40, 24, 1, 1, 6, 60, 4, 8, 8]
    codes_by_place = [[127, 190, 127, 40, 127], [127, 127, 180, 127, 90], [60, 127, 127, 200, 127], [127, 100, 150, 127, 127]]
    M, N = 6 * len(lens), 6 * sum(lens)  # every entry its own row of B
    rp = np.concatenate([[0], np.cumsum(np.tile(lens, 6))]).astype(np.int32)
    rng = np.random.default_rng(O)
    col, val = np.arange(N, dtype=np.int32), (rng.uniform(0.5, 1, N) * rng.choice([-1, 1], N)).astype(np.float16).astype(np.float32)
    codes, scales = features(N, O, 3, kind)
    # the scale of entry e in block b: by its place in runs of eight, another sequence for every block and sixth of the matrix
    e = np.arange(N)
    sixth = e // sum(lens)
    for b in range(scales.shape[1]):
        seq = np.array(codes_by_place)[(b + sixth) % 4, (e % sum(lens)) // 8 % 5]
        scales[:, b] = np.where(sixth == 5, 127 + e % 3, seq)  # the last sixth never leaves the fp16 form
    Q = to_mx(codes, scales, kind, pitch=pitch if kind == "mxf8" else (pitch + 1) // 2)
    for unit in (16, 64, 256):
        dV = handle(M, N, rp, col, val, False, rows_unit_nnz=unit)
        C = check_product(dV, (rp, col, val), codes, scales, kind, Q=Q)
        start = C * 0.5
        check_product(dV, (rp, col, val), codes, scales, kind, Q=Q, start=start)


@pytest.fixture(scope="module")
def many_split_rows():
    """20000 rows, most of 65 to 200 entries: more than 8192 rows that are split into chunks of 16, and as many units."""
    M, N = 20000, 3000
    rng = np.random.default_rng(7)
    lens = rng.integers(65, 201, M)
    lens[::50], lens[1::50], lens[2::50] = 0, 3, 16
    rp = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    first, step = rng.integers(0, N, M), rng.integers(1, 14, M)  # N / 14 > 200: a row's columns are distinct
    at = np.arange(rp[-1]) - np.repeat(rp[:-1], lens)
    row = np.repeat(np.arange(M), lens)
    col = (np.repeat(first, lens) + at * np.repeat(step, lens)) % N
    order = np.lexsort((col, row))
    col = col[order].astype(np.int32)
    val = rng.uniform(-1, 1, len(col)).astype(np.float16).astype(np.float32)
    return M, N, rp, col, val


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("O", [129, 132, 160, 192, 300])
def test_product_slabs_and_chunks(cuda, many_split_rows, kind, fp32, O):
    """Columns behind the last whole slab in a launch of their own, and the chunks of many split rows added up behind both: stored and
    accumulated, in contiguous and odd places."""
    M, N, rp, col, val = many_split_rows
    dV = handle(M, N, rp, col, val, fp32, rows_unit_nnz=16)
    codes, scales = features(N, O, O, kind)
    A = torch.zeros(M, N, dtype=torch.float64, device="cuda")
    A[torch.from_numpy(np.repeat(np.arange(M), np.diff(rp))).cuda(), torch.from_numpy(col).long().cuda()] = torch.from_numpy(val).double().cuda()
    B = torch.from_numpy(ref.values(codes, scales, kind)).cuda()
    want, size, n = A @ B, A.abs() @ B.abs(), int(np.diff(rp).max())
    slack = 1 + 2.0 ** -40  # of the 64-bit products
    nb = O if kind == "mxf8" else (O + 1) // 2
    for pitch in (nb, (nb + 15) // 16 * 16, nb + 3):
        Q = to_mx(codes, scales, kind, pitch=pitch)
        first = None
        for off, ldc in ((0, O), (1, O + 3)):
            big = torch.full((M + 2, ldc), 3.5, device="cuda")
            C = big[1:M + 1, off:off + O]
            vm.spmm(dV, Q, C)
            assert bool(((C.double() - want).abs() <= (n + 4) * U * size * slack).all())
            assert first is None or torch.equal(C, first)
            first = C.clone()
            start = torch.randn(M, O, device="cuda", generator=torch.Generator("cuda").manual_seed(O))
            C.copy_(start)
            vm.spmm(dV, Q, C, accumulate=True)
            bound = (n + 4) * U * (size + start.double().abs()) * slack
            assert bool(((C.double() - want - start.double()).abs() <= bound).all())
            C.fill_(3.5)
            assert bool((big == 3.5).all())


@pytest.mark.parametrize("x,r", COMBOS)
@pytest.mark.parametrize("rows,O", [(700, 264), (700, 4097), (700, 5000), (700, 8192), (700, 8193), (650, 16392)])
@pytest.mark.parametrize("aligned", [True, False])
def test_norm_backward_more_rows_than_blocks(cuda, x, r, rows, O, aligned):
    """Wide rows, several to a block (two blocks per SM at most): the next row's loads, the weight's gradient over a block's rows. A row's sum
    has at most O / 256 terms in turn in a thread and ten steps over threads, and the other terms 8 roundings."""
    g = torch.Generator("cuda").manual_seed(rows + O)

    def make(t):
        if aligned:
            return torch.randn(rows, O, device="cuda", generator=g).to(TYPES[t])
        return torch.randn(rows, O + 5, device="cuda", generator=g).to(TYPES[t])[:, 3:3 + O]

    dY, dR, h = make(x), make(r), make(r)
    w = (1 + 0.2 * torch.randn(O, device="cuda", generator=g)).to(TYPES[r])
    inv = (1 / torch.sqrt(h.double().square().mean(1) + 1e-5)).float()
    n, gw = h.double() * inv.double()[:, None], dY.double() * w.double()
    through = inv.double()[:, None] * n
    dw, dw_size = (dY.double() * n).sum(0), (dY.double() * n).abs().sum(0)
    half, roundings = torch.finfo(TYPES[r]).eps / 2, 8 + O / 256 + 10
    results = []
    for d_residual in (dR, None):
        base = 0.0 if d_residual is None else d_residual.double()
        dx = base + inv.double()[:, None] * gw - through * (gw * n).mean(1, keepdim=True)
        size = (base if d_residual is None else base.abs()) + (inv.double()[:, None] * gw).abs() + through.abs() * (gw * n).abs().mean(1, keepdim=True)
        got, got_w = vm.add_rms_norm_backward(dY, w, h, inv, d_residual=d_residual)
        tiny = float(torch.finfo(TYPES[r]).smallest_normal) * float(torch.finfo(TYPES[r]).eps)
        assert bool(((got.double() - dx).abs() <= half * dx.abs() + roundings * U * size * (1 + half) + tiny).all())
        assert bool(((got_w.double() - dw).abs() <= (rows + 4) * U * dw_size).all())
        results.append((got, got_w))
    place = dR.clone() if aligned else torch.cat([dR, dR[:, :5]], 1)[:, :O].copy_(dR)
    out, out_w = vm.add_rms_norm_backward(dY, w, h, inv, d_residual=place, out=place)
    assert out is place and torch.equal(place, results[0][0]) and torch.equal(out_w, results[0][1])
    if x == r:  # in place on dY
        out, out_w = vm.add_rms_norm_backward(dY, w, h, inv, out=dY)
        assert out is dY and torch.equal(dY, results[1][0]) and torch.equal(out_w, results[1][1])


def test_refusals_are_argument_errors(cuda):
    """What is refused is refused as an invalid argument, before anything runs: no other error counts, and the next call is right."""
    X, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    half = X.half()
    Q, h, inv = vm.add_rms_norm(X, w, residual=X)
    other = vm.MXDense.empty(4, 32)
    for call in (lambda: vm.add_rms_norm(X, w[:63]), lambda: vm.add_rms_norm(X, w.cpu()), lambda: vm.add_rms_norm(X, w.double()),
                 lambda: vm.add_rms_norm(half, w, residual=X), lambda: vm.add_rms_norm(X, w, residual=X[:3]),
                 lambda: vm.add_rms_norm(X, w, residual=half, residual_out=X), lambda: vm.add_rms_norm(X, w, eps=-1.0),
                 lambda: vm.add_rms_norm(X, w, kind=vm.F16), lambda: vm.add_rms_norm(X, w, kind=vm.MXF4, out=Q),
                 lambda: vm.add_rms_norm(X.t(), w), lambda: vm.add_rms_norm(X[0], w), lambda: vm.add_rms_norm(X[:1].expand(4, 64), w),
                 lambda: vm.add_rms_norm(X, None), lambda: vm.add_rms_norm(X, w, out=other), lambda: vm.add_rms_norm(X, w, eps=float("inf")),
                 lambda: vm.add_rms_norm(X, torch.ones(128, device="cuda")[::2]), lambda: vm.add_rms_norm(X[:, :0], w[:0]),
                 lambda: vm.add_rms_norm_backward(X, w, h, inv.half()), lambda: vm.add_rms_norm_backward(half, w, h, inv),
                 lambda: vm.add_rms_norm_backward(X, w, h, inv[:3]), lambda: vm.add_rms_norm_backward(X, w, h, inv, out=half),
                 lambda: vm.add_rms_norm_backward(X, w, h, None), lambda: vm.add_rms_norm_backward(X, w, h, inv, d_residual=half),
                 lambda: vm.mx_quantize(X, 9), lambda: vm.mx_quantize(X.long()), lambda: vm.mx_quantize(X[:, :0]), lambda: vm.mx_quantize(X, out=other),
                 lambda: vm.mx_dequantize(Q, dtype=torch.float16, out=X), lambda: vm.mx_dequantize(Q, out=X[:, :32]),
                 lambda: vm.mx_dequantize(Q, out=X.double()), lambda: vm.mx_dequantize(Q, out=X.cpu())):
        with pytest.raises(vm.VcsrmcError) as e:
            call()
        assert e.value.status == 1, str(e.value)  # VCSRMC_INVALID_ARG
    torch.cuda.synchronize()
    again = vm.add_rms_norm(X, w, residual=X)
    assert torch.equal(again[0].data.view(torch.uint8), Q.data.view(torch.uint8)) and torch.equal(again[1], h) and torch.equal(again[2], inv)


def test_mx_tensors_changed_in_place(cuda):
    """A tensor of an MX matrix that was resized, replaced or turned after the matrix was made is refused by every call, for reading and for
    writing; values may change."""
    M, O = 40, 64
    csr = sparse(M, M, 0.2, 1)
    dV, w = handle(M, M, *csr, False), torch.ones(O, device="cuda")
    X, C = torch.randn(M, O, device="cuda"), torch.empty(M, O, device="cuda")
    changes = (lambda t: t.resize_(4, t.shape[1]), lambda t: t.resize_(M, 1), lambda t: t.resize_(0), lambda t: t.t_(), lambda t: t.unsqueeze_(0),
               lambda t: t.as_strided_((M, t.shape[1]), (0, 1)), lambda t: t.set_(torch.empty(M // 2, t.shape[1], dtype=t.dtype, device="cuda")))
    for kind in KINDS.values():
        for which in ("data", "scale"):
            for change in changes:
                Q = vm.mx_quantize(X, kind)
                change(getattr(Q, which))
                for call in (lambda: vm.spmm(dV, Q, C), lambda: vm.mx_dequantize(Q), lambda: vm.mx_quantize(X, kind, out=Q),
                             lambda: vm.add_rms_norm(X, w, kind=kind, out=Q)):
                    with pytest.raises(vm.VcsrmcError) as e:
                        call()
                    assert e.value.status == 1, str(e.value)
        Q = vm.mx_quantize(X, kind)
        Q.scale.view(torch.uint8).fill_(127)
        check_product(dV, csr, *codes_of(Q), "mxf8" if kind == vm.MXF8 else "mxf4", Q=Q)
    torch.cuda.synchronize()
