"""The operators around the microscaled (MX) dense operand, as cases to measure: the product of a sparse matrix with an MX operand,
MX quantisation, and the residual addition with root-mean-square norm that writes an MX operand (with its backward pass).

An MX operand holds a row-major matrix as 8-bit (E4M3) or 4-bit (E2M1) elements and one power-of-two scale (E8M0, one byte) for every
32 consecutive columns of a row; the last block of a row may be shorter.

own = False computes them in elementary torch operations, own = True through vcsr_mc_b200.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 32
LARGEST = {"mxf4": 6.0, "mxf8": 448.0}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "mxf8": 1, "mxf4": 0.5}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6


def listed():
    return [
        # one small product of a feature propagation (4096 rows of about 16 entries, narrow features): launch latency counts
        {"name": "product_4k_rows_mxf4", "op": "product", "pattern": "uniform", "M": 4096, "N": 4096, "degree": 16, "O": 32, "q": "mxf4", "a": "f16"},
        # a handful of requested rows of a large graph, thousands of neighbours each: long rows, little parallelism across rows
        {"name": "product_few_rows_mxf8", "op": "product", "pattern": "few_rows", "M": 8, "N": 262144, "degree": 4000, "O": 128, "q": "mxf8", "a": "f16"},
        # the power-law matrix (empty rows and hub rows) at matched precision of A, with an odd feature width
        {"name": "product_powerlaw_odd_mxf8", "op": "product", "pattern": "powerlaw", "M": 262144, "N": 262144, "degree": 10, "O": 100, "q": "mxf8", "a": "f32"},
        # a scale-free graph whose 4-bit features are about as large as the L2 cache
        {"name": "product_rmat_mxf4", "op": "product", "pattern": "rmat", "M": 1 << 20, "N": 1 << 20, "degree": 16, "O": 128, "q": "mxf4", "a": "f16"},
        # the 27-point stencil on a 100^3 grid: the most entries
        {"name": "product_stencil_mxf4", "op": "product", "pattern": "stencil", "M": 100 ** 3, "N": 100 ** 3, "degree": 27, "O": 128, "q": "mxf4", "a": "f16"},
        # quantising the features of a small batch
        {"name": "quantize_4k_mxf8", "op": "quantize", "rows": 4096, "O": 32, "x": "f32", "q": "mxf8"},
        # a whole feature matrix to 4 bits and back to values
        {"name": "quantize_1m_mxf4", "op": "quantize", "rows": 1 << 20, "O": 128, "x": "f16", "q": "mxf4"},
        # the norm of one wide row: a single token
        {"name": "norm_one_row_mxf8", "op": "norm", "rows": 1, "O": 4096, "x": "bf16", "r": "bf16", "q": "mxf8"},
        # the norm between two products over a million rows: fp32 sums of the product in, an fp16 residual stream
        {"name": "norm_1m_mxf8", "op": "norm", "rows": 1 << 20, "O": 128, "x": "f32", "r": "f16", "q": "mxf8"},
        # wide rows whose last block is short
        {"name": "norm_odd_mxf8", "op": "norm", "rows": 20011, "O": 1009, "x": "f32", "r": "bf16", "q": "mxf8"},
        # the backward pass of a mid-sized batch, fp32 gradient from the transposed product
        {"name": "norm_backward_4k", "op": "norm_backward", "rows": 4096, "O": 128, "x": "f32", "r": "f16"},
        # the backward pass of wide rows
        {"name": "norm_backward_wide", "op": "norm_backward", "rows": 32768, "O": 4096, "x": "bf16", "r": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["product", "product", "quantize", "norm", "norm_backward"])
    if op == "product":
        pattern = rng.choice(["uniform", "few_rows", "powerlaw", "rmat", "stencil"])
        q, a, O = rng.choice(["mxf4", "mxf8"]), rng.choice(["f16", "f32"]), _log(rng, 8, 320)
        if pattern == "stencil":
            n = _log(rng, 8, 100)
            M = N = n ** 3
            degree = 27
        elif pattern == "few_rows":
            M, N, degree = _log(rng, 1, 64), _log(rng, 20000, 400000), _log(rng, 100, 8000)
        elif pattern == "rmat":
            M = N = 1 << rng.randint(10, 20)
            degree = _log(rng, 4, 24)
        else:
            M = _log(rng, 300, 600000)
            N = M if pattern == "powerlaw" else _log(rng, 1000, 600000)
            degree = _log(rng, 2, 24)
        O = max(8, min(O, int(100 ** 3 * 26 * 128 / (M * degree))))
        return {"op": op, "pattern": pattern, "M": M, "N": N, "degree": degree, "O": O, "q": q, "a": a}
    O = _log(rng, 16, 8192)
    rows = max(1, min(_log(rng, 1, 1 << 20), (1 << 27) // O))
    x = rng.choice(["f32", "f16", "bf16"])
    if op == "quantize":
        return {"op": op, "rows": rows, "O": O, "x": x, "q": rng.choice(["mxf4", "mxf8"])}
    r = rng.choice(["f32", "f16", "bf16"]) if x == "f32" else x
    if op == "norm":
        return {"op": op, "rows": rows, "O": O, "x": x, "r": r, "q": "mxf8"}
    return {"op": op, "rows": rows, "O": O, "x": x, "r": r}


# ---- inputs --------------------------------------------------------------------------------------


def _rand(g, *shape):
    return torch.rand(*shape, device="cuda", generator=g)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _sparse(case, g):
    """(row_ptr int32, col int32) of the case's pattern, columns ascending and distinct in a row."""
    M, N, degree = case["M"], case["N"], case["degree"]
    if case["pattern"] == "stencil":
        n = round(M ** (1 / 3))
        at = torch.arange(n, device="cuda")
        cells = torch.stack(torch.meshgrid(at, at, at, indexing="ij"), -1).reshape(-1, 1, 3)
        d = torch.arange(-1, 2, device="cuda")
        steps = torch.stack(torch.meshgrid(d, d, d, indexing="ij"), -1).reshape(1, 27, 3)
        to = cells + steps
        inside = ((to >= 0) & (to < n)).all(-1)
        col = ((to[..., 0] * n + to[..., 1]) * n + to[..., 2])[inside]
        counts = inside.sum(1)
    else:
        if case["pattern"] == "rmat":
            e = M * degree
            row = torch.zeros(e, dtype=torch.int64, device="cuda")
            col = torch.zeros(e, dtype=torch.int64, device="cuda")
            for _ in range(M.bit_length() - 1):
                u = _rand(g, e)
                row = row * 2 + (u >= 0.76)
                col = col * 2 + (((u >= 0.57) & (u < 0.76)) | (u >= 0.95))
        else:
            if case["pattern"] == "powerlaw":
                counts = (0.04 * degree * _rand(g, M).clamp_min(1e-9) ** -1.25).clamp_max(min(8192, N)).long()
            else:
                counts = torch.poisson(torch.full((M,), float(degree), device="cuda"), generator=g).long()
            row = torch.repeat_interleave(torch.arange(M, device="cuda"), counts)
            col = torch.randint(0, N, (row.numel(),), device="cuda", generator=g)
        key = torch.unique(row * N + col)
        row, col = key // N, key % N
        counts = torch.bincount(row, minlength=M)
    row_ptr = torch.zeros(M + 1, dtype=torch.int64, device="cuda")
    torch.cumsum(counts, 0, out=row_ptr[1:])
    return row_ptr.int(), col.int().contiguous()


def _features(g, rows, O):
    """Features of uneven magnitude: each row its own size, one row in 64 all zero."""
    x = _randn(g, rows, O) * torch.exp(_randn(g, rows, 1))
    return x * (_rand(g, rows, 1) > 1 / 64)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "product":
        row_ptr, col = _sparse(case, g)
        val = _rand(g, col.numel()) * 2 - 1
        if case["a"] == "f16":
            val = val.half().float()  # the FP16 format holds fp16 values
        codes, scale = _quantize(_features(g, case["N"], case["O"]), case["q"])
        s.update(row_ptr=row_ptr, col=col, val=val, data=_pack(codes, case["q"]), scale=scale)
        if own:
            import vcsr_mc_b200 as vm

            s["A"] = vm.build_vcsr_mc_device(row_ptr, col, val, case["M"], case["N"], fp32=case["a"] == "f32", segw=32, plans=[vm.PLAN_ROWS])
            s["B"] = vm.MXDense(s["data"], s["scale"], cols=case["O"])
        return s
    rows, O = case["rows"], case["O"]
    if case["op"] == "quantize":
        s["x"] = _features(g, rows, O).to(TYPES[case["x"]])
        return s
    rt = TYPES[case["r"]]
    s["weight"] = (1 + 0.1 * _randn(g, O)).to(rt)
    if case["op"] == "norm":
        s["x"] = _features(g, rows, O).to(TYPES[case["x"]])
        s["residual"] = _randn(g, rows, O).to(rt)
        return s
    s["dy"] = (_randn(g, rows, O) * 0.1).to(TYPES[case["x"]])
    s["d_residual"] = (_randn(g, rows, O) * 0.1).to(rt)
    s["hidden"] = (_randn(g, rows, O) * 2).to(rt)
    s["inv_rms"] = torch.rsqrt(s["hidden"].double().square().mean(1) + EPS).float()
    return s


# ---- plain forms -----------------------------------------------------------------------------------


def _quantize(x, q):
    """(codes uint8 [rows, O], scale float8_e8m0fnu [rows, blocks]): the smallest power of two that lets the block's largest magnitude fit the
    element type, elements rounded to nearest, ties to even."""
    rows, O = x.shape
    blocks = -(-O // BLOCK)
    t = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - O)).view(rows, blocks, BLOCK)
    amax = t.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1
    top = math.frexp(LARGEST[q])
    e = (e - top[1] + (m > top[0])).clamp_min(-127)
    e = torch.where(amax > 0, e, -127)
    fine = torch.isfinite(amax)
    t = torch.where(fine, torch.ldexp(t, -e), 0.0)
    scale = torch.where(fine, e + 127, 255).to(torch.uint8).view(rows, blocks)
    if q == "mxf8":
        codes = t.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = t.abs()
        codes = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)) | (torch.signbit(t).to(torch.uint8) << 3)
    return codes.view(rows, blocks * BLOCK)[:, :O], scale.view(torch.float8_e8m0fnu)


def _pack(codes, q):
    """The elements as they are stored: E4M3 bytes, or two E2M1 codes to a byte, the even column in the low half."""
    if q == "mxf8":
        return codes.contiguous().view(torch.float8_e4m3fn)
    codes = torch.nn.functional.pad(codes, (0, codes.shape[1] % 2))
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def _values(data, scale, q, O):
    """What an MX operand stands for, in fp32."""
    if q == "mxf8":
        t = data.float()
    else:
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=data.device)
        t = torch.stack([table[(data & 15).int()], table[(data >> 4).int()]], -1).flatten(1)[:, :O]
    return t * scale.float().repeat_interleave(BLOCK, 1)[:, :O]


def _run_product(s, case):
    B = _values(s["data"], s["scale"], case["q"], case["O"])
    row = torch.repeat_interleave(torch.arange(case["M"], device="cuda"), s["row_ptr"].diff())
    t = B[s["col"]]
    t *= s["val"][:, None]
    return torch.zeros(case["M"], case["O"], device="cuda").index_add_(0, row, t)


def _mx_outputs(codes, scale, q):
    """8-bit elements as they are (a type of torch), 4-bit ones as the values that they stand for."""
    if q == "mxf8":
        return {"data": codes.contiguous().view(torch.float8_e4m3fn), "scale": scale}
    return {"values": _values(_pack(codes, q), scale, q, codes.shape[1]).bfloat16(), "scale": scale}


def _run_norm(s, case):
    h = (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)
    inv = torch.rsqrt(h.float().square().mean(1) + EPS)
    y = h.float() * inv[:, None] * s["weight"].float()
    return {**_mx_outputs(*_quantize(y, case["q"]), case["q"]), "residual": h, "inv_rms": inv}


def _run_backward(s):
    h, dy, inv = s["hidden"].float(), s["dy"].float(), s["inv_rms"][:, None]
    gw = dy * s["weight"].float()
    dx = s["d_residual"].float() + inv * gw - h * inv ** 3 * (gw * h).mean(1, keepdim=True)
    return {"dx": dx.to(s["hidden"].dtype), "dweight": (dy * h * inv).sum(0)}


def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "product":
            return _run_product(state, case)
        if case["op"] == "quantize":
            return _mx_outputs(*_quantize(state["x"], case["q"]), case["q"])
        return _run_norm(state, case) if case["op"] == "norm" else _run_backward(state)
    import vcsr_mc_b200 as vm

    if case["op"] == "product":
        C = torch.empty(case["M"], case["O"], device="cuda")
        return vm.spmm(state["A"], state["B"], C)
    kind = vm.MXF4 if case.get("q") == "mxf4" else vm.MXF8
    if case["op"] == "norm_backward":
        dx, dweight = vm.add_rms_norm_backward(state["dy"], state["weight"], state["hidden"], state["inv_rms"], d_residual=state["d_residual"])
        return {"dx": dx, "dweight": dweight}
    more = {}
    if case["op"] == "quantize":
        Q = vm.mx_quantize(state["x"], kind)
    else:
        Q, h, inv = vm.add_rms_norm(state["x"], state["weight"], residual=state["residual"], eps=EPS, kind=kind)
        more = {"residual": h, "inv_rms": inv}
    if kind == vm.MXF8:
        return {"data": Q.data, "scale": Q.scale, **more}
    return {"values": vm.mx_dequantize(Q, dtype=torch.bfloat16), "scale": Q.scale}


# ---- the definition in 64 bits ----------------------------------------------------------------------


def _exact_scale(y, q):
    """2^e for every element's block, from the definition: e the least integer from -127 with max|y| <= largest * 2^e."""
    rows, O = y.shape
    blocks = -(-O // BLOCK)
    amax = torch.cat([y[:, b * BLOCK:(b + 1) * BLOCK].abs().amax(1, keepdim=True) for b in range(blocks)], 1)
    e = torch.ceil(torch.log2(amax / LARGEST[q]))
    e = torch.where(amax <= LARGEST[q] * torch.exp2(e - 1), e - 1, e)
    e = torch.where(amax > LARGEST[q] * torch.exp2(e), e + 1, e)
    return torch.exp2(torch.where(amax > 0, e, torch.full_like(e, -127.0)).clamp_min(-127))


def _exact_rounded(t, q):
    """t rounded to the element type, to nearest, ties to even; E4M3 has 3 mantissa bits from 2^-6, E2M1 one from 2^0."""
    least, bits = (0, 1) if q == "mxf4" else (-6, 3)
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp_min(2.0 ** least))) - bits)
    return torch.round(t / step) * step


def _exact_product(s, case):
    M, O, q = case["M"], case["O"], case["q"]
    two = torch.exp2(s["scale"].view(torch.uint8).double() - 127)
    row_ptr = s["row_ptr"].cpu().numpy().astype(np.int64)
    out = torch.zeros(M, O, dtype=torch.float64, device="cuda")
    r0 = 0
    while r0 < M:
        r1 = max(r0 + 1, int(np.searchsorted(row_ptr, row_ptr[r0] + (1 << 22), side="right")) - 1)
        p0, p1 = int(row_ptr[r0]), int(row_ptr[r1])
        col = s["col"][p0:p1].long()
        byte = s["data"].view(torch.uint8)[col]
        if q == "mxf4":
            code = torch.stack([byte % 16, byte // 16], 2).flatten(1)[:, :O].int()
            sign, ex, man, width, bias = code // 8, code // 2 % 4, code % 2, 1, 1
        else:
            code = byte.int()
            sign, ex, man, width, bias = code // 128, code // 8 % 16, code % 8, 3, 7
        v = (1 - 2 * sign) * ((ex > 0) + man.double() / 2 ** width) * torch.exp2((ex.clamp_min(1) - bias).double())
        v = v * two[col][:, torch.arange(O, device="cuda") // BLOCK] * s["val"][p0:p1].double()[:, None]
        row = torch.searchsorted(s["row_ptr"][r0 + 1:r1 + 1].contiguous(), torch.arange(p0, p1, device="cuda", dtype=torch.int32), right=True)
        out[r0:r1].index_add_(0, row, v)
        r0 = r1
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "product":
        return _exact_product(s, case)
    if case["op"] == "norm_backward":
        h, dy, w, inv = s["hidden"].double(), s["dy"].double(), s["weight"].double(), s["inv_rms"].double()
        normed = h * inv[:, None]
        through = dy * w
        dx = through - normed * (through * normed).sum(1, keepdim=True) / case["O"]
        return {"dx": s["d_residual"].double() + dx * inv[:, None], "dweight": torch.einsum("ro,ro->o", dy, normed)}
    if case["op"] == "quantize":
        y = s["x"].double()
        scale = _exact_scale(y, case["q"])
        full = scale.repeat_interleave(BLOCK, 1)[:, :case["O"]]
        t = _exact_rounded(y / full, case["q"])
        return {"values": t * full, "scale": scale} if case["q"] == "mxf4" else {"data": t, "scale": scale}
    # the stored sum is rounded to the residual's type, and it is what the norm sees
    h = (s["x"].double() + s["residual"].double()).float().to(s["residual"].dtype).double()
    inv = (torch.linalg.vector_norm(h, dim=1) ** 2 / case["O"] + EPS) ** -0.5
    y = h * inv[:, None] * s["weight"].double()
    # elements before their rounding to 8 bits: a sum of 32 bits may fall on either side of a border
    scale = _exact_scale(y, case["q"])
    return {"data": y / scale.repeat_interleave(BLOCK, 1)[:, :case["O"]], "scale": scale, "residual": h, "inv_rms": inv}


# ---- what a pass cannot do without ---------------------------------------------------------------------


def work(case):
    q = BYTES.get(case.get("q"), 0)
    if case["op"] == "product":
        M, N, O = case["M"], case["N"], case["O"]
        nnz = M * case["degree"]
        if case["pattern"] == "stencil":
            nnz = (3 * round(M ** (1 / 3)) - 2) ** 3
        used = N * -math.expm1(-nnz / N)  # columns that an entry names, were they uniform
        return {"bytes": nnz * (4 + BYTES[case["a"]]) + 4 * (M + 1) + used * (O * q + -(-O // BLOCK)) + 4 * M * O, "flops": 2 * nnz * O}
    rows, O = case["rows"], case["O"]
    n = rows * O
    if case["op"] == "norm_backward":
        return {"bytes": n * (BYTES[case["x"]] + 3 * BYTES[case["r"]]) + 4 * rows + O * (BYTES[case["r"]] + 4), "flops": 10 * n}
    out = n * (2 if case["q"] == "mxf4" else 1) + rows * -(-O // BLOCK)
    if case["op"] == "quantize":
        return {"bytes": n * BYTES[case["x"]] + out, "flops": 3 * n}
    return {"bytes": n * (BYTES[case["x"]] + 2 * BYTES[case["r"]]) + O * BYTES[case["r"]] + 4 * rows + out, "flops": 8 * n}
