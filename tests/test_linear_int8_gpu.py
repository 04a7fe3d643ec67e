"""ops.quantize_int8 and ops.linear_int8 against integer arithmetic and float64.

The rounding to 8 bits is defined in single-precision steps, so its results are compared for equality.  The product is exact in
integers; behind it come at most five fp32 roundings (the sum as fp32, two scales, bias) and one to the output's type, and with the GELU
its relative error of 4e-6 of |v| Phi(-|v|) beside three more roundings: 2^-21 of the magnitudes that take part covers the former,
8e-6 of |v| the latter."""
import numpy as np
import pytest
import torch

from flashdeberta_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _quantized(x):
    """The definition on the host, step by step in single precision."""
    v = x.detach().float().cpu().numpy().reshape(-1, x.shape[-1])
    top = np.abs(v).max(axis=1)
    scale, q = np.zeros_like(top), np.zeros(v.shape, np.int8)
    for r, t in enumerate(top):
        if not np.isfinite(t):
            scale[r] = t
        elif t >= 2.0 ** -100:
            scale[r] = t / np.float32(127)
            q[r] = np.rint(v[r] * (np.float32(127) / t)).astype(np.int8)
    return torch.from_numpy(q).view(x.shape), torch.from_numpy(scale).view(x.shape[:-1])


def _check(out, xq, xs, wq, ws, bias, gelu, acc=None):
    acc = xq.double().cpu() @ wq.double().cpu().t() if acc is None else acc
    scaled = acc * ws.double().cpu() * xs.double().cpu()[..., None]
    b = 0.0 if bias is None else bias.double().cpu()
    v = scaled + b
    bound = 2.0 ** -21 * (scaled.abs() + (0.0 if bias is None else b.abs()))
    if gelu:
        bound = 1.13 * bound + 8e-6 * v.abs()  # (the GELU's slope is at most 1.13)
        v = 0.5 * v * torch.special.erfc(-v / 2 ** 0.5)
    info = torch.finfo(out.dtype)
    allowed = info.eps / 2 * v.abs() + bound + (2.0 ** -25 if out.dtype == torch.float16 else info.tiny)
    worst = ((out.double().cpu() - v).abs() / allowed).max().item()
    assert worst <= 1.0, f"{worst:.3g} times what is allowed"


def _problem(rows, k, n, dtype, bias, seed, given=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, k, generator=g) * torch.exp(torch.randn(rows, 1, generator=g))).to(dtype).to(DEV)
    w = (torch.randn(n, k, generator=g) * 0.05).to(DEV)
    b = None if bias is None else torch.randn(n, generator=g).to(bias).to(DEV)
    wq, ws = ops.quantize_int8(w)
    return x, wq, ws, b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (4, 255), (9, 256), (37, 264), (5, 1001), (2, 4096), (3, 8192), (2, 8200), (2, 20001), (700, 96)])
def test_rounding_to_8_bits(dtype, rows, cols):
    g = torch.Generator().manual_seed(rows * cols)
    x = (torch.randn(rows, cols, generator=g) * 10 ** torch.linspace(-3, 3, rows)[:, None]).to(dtype).to(DEV)
    q, s = ops.quantize_int8(x)
    wq, ws = _quantized(x)
    assert q.shape == x.shape and q.dtype == torch.int8 and q.stride(0) % 16 == 0
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


def test_rounding_of_ties_zeros_and_what_is_not_finite():
    x = torch.zeros(8, 40, device=DEV)
    x[1] = torch.arange(40, device=DEV) - 20.0
    x[2] = 127.0
    x[2, :20] = torch.arange(20, device=DEV) + 0.5          # ties go to the even number
    x[3, 5] = float("inf")
    x[4, 6] = float("nan")
    x[4, 7] = float("inf")
    x[5] = 1e-31                                             # below 2^-100
    x[6] = 2.0 ** -99
    x[7] = torch.finfo(torch.float32).max
    q, s = ops.quantize_int8(x)
    wq, ws = _quantized(x)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu().view(torch.int32)[:4], ws.view(torch.int32)[:4])
    assert torch.isinf(s[3]) and torch.isnan(s[4]) and s[5] == 0 and s[0] == 0 and (q[6] == 127).all()
    assert q[2, :6].tolist() == [0, 2, 2, 4, 4, 6]
    y, t = ops.quantize_int8(x[None, :, ::2])                # leading dimensions, strides
    assert torch.equal(y[0].cpu(), _quantized(x[:, ::2])[0]) and t.shape == (1, 8)


@pytest.mark.parametrize("rows,k,n", [
    (1, 1, 1), (1, 16, 8), (1, 1024, 4096), (2, 100, 33), (7, 129, 64), (16, 768, 768), (17, 130, 257), (29, 768, 2304), (32, 2048, 96), (33, 1000, 48),
    (64, 4096, 1024), (65, 512, 520), (127, 384, 131), (128, 1024, 640), (129, 128, 128), (200, 1001, 1537), (257, 1536, 1000), (300, 64, 4104), (513, 96, 200),
    (1000, 520, 72), (2100, 256, 1030), (2049, 1024, 1024),
])
@pytest.mark.parametrize("dtype", TYPES)
def test_product(rows, k, n, dtype):
    for bias, gelu in ((None, False), (dtype, True)):
        x, wq, ws, b = _problem(rows, k, n, dtype, bias, rows + k + n)
        out = ops.linear_int8(x, wq, ws, b, gelu=gelu)
        assert out.dtype == dtype and out.shape == (rows, n)
        xq, xs = ops.quantize_int8(x)
        _check(out, xq, xs, wq, ws, b, gelu)
        given = ops.linear_int8(xq, wq, ws, b, x_scale=xs, gelu=gelu, out_dtype=dtype)
        assert torch.equal(given, out)
    ops.check_status()


@pytest.mark.parametrize("rows,k,n", [(40, 1, 8), (100, 3, 40), (64, 96, 8), (50, 64, 1), (33, 17, 4), (90, 130, 12)])
@pytest.mark.parametrize("dtype", TYPES)
def test_product_of_few_features(rows, k, n, dtype):
    x, wq, ws, b = _problem(rows, k, n, dtype, dtype, rows + k + n)
    xq, xs = ops.quantize_int8(x)
    _check(ops.linear_int8(x, wq, ws, b), xq, xs, wq, ws, b, False)
    _check(ops.linear_int8(xq, wq, ws, b, x_scale=xs, out_dtype=dtype, gelu=True), xq, xs, wq, ws, b, True)
    ops.check_status()


@pytest.mark.parametrize("n", [1104, 1101, 1028])
@pytest.mark.parametrize("rows,k", [(9001, 2000), (5003, 300)])
def test_product_of_many_tiles(rows, k, n):
    """Every accumulator and stage used many times over, tiles that end inside the matrix, in every form of the store."""
    for dtype, gelu in ((torch.bfloat16, True), (torch.float32, False)):
        x, wq, ws, b = _problem(rows, k, n, dtype, torch.float32, n)
        xq, xs = ops.quantize_int8(x)
        acc = (xq.double() @ wq.double().t()).cpu()
        _check(ops.linear_int8(x, wq, ws, b, gelu=gelu), xq, xs, wq, ws, b, gelu, acc)
    ops.check_status()


@pytest.mark.parametrize("n", [1104, 1101, 1028])
@pytest.mark.parametrize("dtype,gelu", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float16, False), (torch.float32, True)])
def test_product_of_many_long_tiles(n, dtype, gelu):
    """The epilogue of few warps that long rows take, the last columns and rows of the matrix inside a tile."""
    x, wq, ws, b = _problem(7001, 2100, n, dtype, torch.float32, n + 1)
    xq, xs = ops.quantize_int8(x)
    acc = (xq.double() @ wq.double().t()).cpu()
    _check(ops.linear_int8(x, wq, ws, b, gelu=gelu), xq, xs, wq, ws, b, gelu, acc)
    ops.check_status()


@pytest.mark.parametrize("rows,k,n", [(5, 2000, 96), (70, 5000, 256), (300, 131071, 64), (1, 131071, 8)])
def test_largest_integers(rows, k, n):
    """Every product at its largest: the sums reach 2^31 - 2^14 and stay exact."""
    x = torch.full((rows, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    one = lambda m: torch.ones(m, device=DEV)
    out = ops.linear_int8(x, w, one(n), x_scale=one(rows), out_dtype=torch.float32)
    want = torch.tensor([16384 * k, -16256 * k], dtype=torch.int64).float().repeat(n // 2).to(DEV)  # (the sum rounded to fp32)
    assert torch.equal(out, want.expand(rows, n))


@pytest.mark.parametrize("rows", [3, 200])
def test_large_sums_through_the_gelu(rows):
    """Sums on either side of 2^24, where the conversion rounds, scaled to the GELU's range."""
    k, n = 4096, 72
    g = torch.Generator().manual_seed(rows)
    x = torch.randint(100, 128, (rows, k), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, 1), generator=g, dtype=torch.int8).expand(n, k).contiguous()
    xs, ws = torch.rand(rows, generator=g) * 1e-4, torch.rand(n, generator=g) * 1e-3
    for dtype in TYPES:
        out = ops.linear_int8(x.to(DEV), w.to(DEV), ws.to(DEV), x_scale=xs.to(DEV), gelu=True, out_dtype=dtype)
        _check(out, x, xs, w, ws, None, True)


def test_random_integers_and_signs_of_every_size():
    g = torch.Generator().manual_seed(5)
    x = torch.randint(-128, 128, (150, 777), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (90, 777), generator=g, dtype=torch.int8)
    xs, ws = torch.randn(150, generator=g), torch.randn(90, generator=g)
    out = ops.linear_int8(x.to(DEV), w.to(DEV), ws.to(DEV), x_scale=xs.to(DEV), out_dtype=torch.float32)
    _check(out, x, xs, w, ws, None, False)


def test_bias_in_fp32_leading_dimensions_and_other_output_types():
    x, wq, ws, _ = _problem(60, 192, 160, torch.bfloat16, None, 6)
    b = torch.randn(160, device=DEV)
    xq, xs = ops.quantize_int8(x)
    for t in TYPES:
        out = ops.linear_int8(x.view(3, 20, 192), wq, ws, b, out_dtype=t)
        assert out.shape == (3, 20, 160) and out.dtype == t
        _check(out.view(60, 160), xq, xs, wq, ws, b, False)
        assert torch.equal(ops.linear_int8(xq.view(3, 20, -1), wq, ws, b, x_scale=xs.view(3, 20), out_dtype=t), out)


def test_views_that_have_to_be_copied():
    x, wq, ws, b = _problem(40, 100, 56, torch.bfloat16, torch.bfloat16, 7)
    want = ops.linear_int8(x, wq, ws, b)
    dense = wq.contiguous()                                  # rows of 100 bytes
    assert dense.stride(0) == 100
    assert torch.equal(ops.linear_int8(x, dense, ws, b), want)
    assert torch.equal(ops.linear_int8(x, dense.t().contiguous().t(), ws, b), want)
    wide = torch.zeros(40, 300, dtype=torch.bfloat16, device=DEV)
    wide[:, 5:105] = x
    assert torch.equal(ops.linear_int8(wide[:, 5:105], wq, ws, b), want)
    two = torch.stack([ws, ws], 1)
    assert torch.equal(ops.linear_int8(x, wq, two[:, 0], torch.stack([b, b], 1)[:, 1]), want)
    off = torch.zeros(57, dtype=torch.bfloat16, device=DEV)
    off[1:] = b                                              # a bias that starts on two bytes
    assert torch.equal(ops.linear_int8(x, wq, ws, off[1:]), want)


@pytest.mark.parametrize("shape,expanded", [((1, 192), (6, 192)), ((2, 1, 192), (2, 4, 192)), ((1, 192), (300, 192)), ((5, 1, 192), (5, 40, 192)),
                                            ((1, 50, 192), (3, 50, 192))])
def test_expanded_integers_count_as_often_as_they_stand_for(shape, expanded):
    """x, its scales and the weight as views that repeat rows, against their copies."""
    g = torch.Generator().manual_seed(sum(expanded))
    x = torch.randint(-128, 128, shape, generator=g, dtype=torch.int8).to(DEV).expand(expanded)
    xs = torch.rand(shape[:-1], generator=g).to(DEV).expand(expanded[:-1])
    w = torch.randint(-128, 128, (72, 192), generator=g, dtype=torch.int8).to(DEV)
    ws = torch.rand(72, generator=g).to(DEV)
    want = ops.linear_int8(x.contiguous(), w, ws, x_scale=xs.contiguous(), out_dtype=torch.float32)
    _check(want.view(-1, 72), x.reshape(-1, 192), xs.reshape(-1), w, ws, None, False)
    assert torch.equal(ops.linear_int8(x, w, ws, x_scale=xs, out_dtype=torch.float32), want)
    one = w[:1].expand(72, 192)
    want = ops.linear_int8(x.contiguous(), one.contiguous(), ws, x_scale=xs.contiguous())
    assert torch.equal(ops.linear_int8(x, one, ws, x_scale=xs), want)
    ops.check_status()


def test_rows_that_are_not_finite_stay_apart():
    x, wq, ws, b = _problem(50, 300, 64, torch.bfloat16, torch.bfloat16, 8)
    want = ops.linear_int8(x, wq, ws, b, gelu=True)
    x[3, 17] = float("inf")
    x[30, 200] = float("nan")
    out = ops.linear_int8(x, wq, ws, b, gelu=True)
    bad = torch.zeros(50, dtype=torch.bool, device=DEV)
    bad[3] = bad[30] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], want[~bad])
    x[:] = 0
    assert torch.equal(ops.linear_int8(x, wq, ws, b), b.expand(50, 64))
    b[:] = float("inf")
    assert torch.isinf(ops.linear_int8(x, wq, ws, b, gelu=True)).all()


def test_gelu_over_its_range():
    """Through a weight of ones: the values are the tokens' own first elements, from far below zero to far above."""
    v = torch.linspace(-12, 12, 4001, device=DEV)
    x = torch.zeros(4001, 16, device=DEV)
    x[:, 0] = v
    w = torch.zeros(8, 16, dtype=torch.int8, device=DEV)
    w[:, 0] = 1
    out = ops.linear_int8(x, w, torch.ones(8, device=DEV), gelu=True)
    xq, xs = ops.quantize_int8(x)
    _check(out, xq, xs, w, torch.ones(8), None, True)


@pytest.mark.parametrize("rows", [1, 40, 3000])
def test_gelu_in_fp32_holds_what_fp32_holds(rows):
    """Values that reach the GELU unrounded (as the features' scales, everything else one).  Of q = |v| Phi(-|v|) the steps in fp32 leave
    5.8 * 2^-24 where reciprocal and exponential are correctly rounded (all of them simulated over 0 < |v| < 13); the approximate ones
    are documented to 2^-23 and 2^-22 relative, of which the reciprocal's counts at most twice and half a step of either is in the
    simulation already: 2 and 4 more, 12 in all.  Half a step of the result, and nothing below fp32's smallest normal number."""
    v = torch.cat([torch.linspace(-20, 20, 8001), -torch.logspace(-30, 1.1, 500), torch.logspace(-30, 30, 499)])
    x = torch.ones(rows, 16, dtype=torch.int8, device=DEV)
    w = torch.zeros(9000, 16, dtype=torch.int8, device=DEV)
    w[:, 3] = 1
    out = ops.linear_int8(x, w, v.to(DEV), x_scale=torch.ones(rows, device=DEV), gelu=True, out_dtype=torch.float32)
    assert (out == out[:1]).all()
    v = v.double()
    q = 0.5 * v.abs() * torch.special.erfc(v.abs() / 2 ** 0.5)
    want = v.clamp(min=0) - q
    allowed = 12 * 2.0 ** -24 * q + 2.0 ** -24 * want.abs() + torch.finfo(torch.float32).tiny
    worst = ((out[0].double().cpu() - want).abs() / allowed).max().item()
    assert worst <= 1.0, f"{worst:.3g} times what is allowed"


@pytest.mark.parametrize("rows", [2, 60])
@pytest.mark.parametrize("dtype", TYPES)
def test_gelu_of_what_is_not_finite_and_of_the_largest(rows, dtype):
    v = torch.tensor([float("inf"), -float("inf"), float("nan"), 3e38, -3e38, 0.0, -0.0, 1e-45]).to(DEV)
    x = torch.ones(rows, 16, dtype=torch.int8, device=DEV)
    w = torch.zeros(8, 16, dtype=torch.int8, device=DEV)
    w[:, 3] = 1
    out = ops.linear_int8(x, w, v, x_scale=torch.ones(rows, device=DEV), gelu=True, out_dtype=dtype)
    assert (out[:, 0] == float("inf")).all() and (out[:, 1] == 0).all() and torch.isnan(out[:, 2]).all()
    assert (out[:, 3] == v[3].to(dtype)).all() and (out[:, 4:7] == 0).all() and (out[:, 7].abs() <= 1e-45).all()


@pytest.mark.parametrize("cols", [(1 << 30) + 1, (1 << 31) + 8, (1 << 32) + 8])
def test_rows_that_are_too_long_are_refused(cols):
    """Before anything is read or copied, in the last case before 8 columns are left of them in 32 bits."""
    with pytest.raises(ValueError, match="elements"):
        ops.quantize_int8(torch.ones(1, 1, device=DEV).expand(1, cols))


def test_rows_behind_the_last_one_are_left_alone():
    import ctypes as C
    from flashdeberta_b200 import _lib
    for rows, k, n, t in [(5, 64, 40, torch.float32), (130, 256, 257, torch.bfloat16), (1, 128, 96, torch.float16)]:
        x, wq, ws, _ = _problem(rows, k, n, torch.float32, None, 9)
        xq, xs = ops.quantize_int8(x)
        out = torch.full((rows * n + 512,), 7.0, dtype=t, device=DEV)
        kind = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 3}[t]
        p = _lib.LinearInt8Params(C.sizeof(_lib.LinearInt8Params), _lib.FDB_INT8, xq.data_ptr(), xq.stride(0), xs.data_ptr(), wq.data_ptr(), wq.stride(0),
                                  ws.data_ptr(), None, out.data_ptr() + 256 * out.element_size(), rows, k, n, 0, kind, 0, 0, None, 0, None)
        if rows == 1:
            p.x_pitch = (k + 15) // 16 * 16
        _lib.check(_lib.load().fdb_linear_int8(C.byref(p), ops.raw_stream(x.device)))
        assert (out[:256] == 7).all() and (out[256 + rows * n:] == 7).all()
        assert torch.equal(out[256:256 + rows * n].view(rows, n), ops.linear_int8(x, wq, ws, out_dtype=t))


def test_streams_captures_and_many_calls():
    probs = [_problem(r, 512, 384, torch.bfloat16, torch.bfloat16, r) for r in (1, 30, 400)]
    want = [ops.linear_int8(*p, gelu=True) for p in probs]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            got.append([ops.linear_int8(*p, gelu=True) for p in probs])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))
    graphs, held = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append([ops.linear_int8(*p, gelu=True) for p in probs])
        graphs.append(g)
    others = [_problem(r, 512, 384, torch.bfloat16, torch.bfloat16, r + 77) for r in (1, 30, 400)]
    for p, o in zip(probs, others):
        p[0].copy_(o[0])
    want = [ops.linear_int8(*p, gelu=True) for p in probs]
    for g in graphs + graphs:
        g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in held for a, b in zip(r, want))
    ops.check_status()


def test_tracing_and_refusals():
    x, wq, ws, b = _problem(10, 64, 48, torch.bfloat16, torch.bfloat16, 10)
    fn = torch.compile(lambda x: ops.linear_int8(x, wq, ws, b), fullgraph=True, backend="aot_eager")
    assert torch.equal(fn(x), ops.linear_int8(x, wq, ws, b))
    torch.library.opcheck(torch.ops.flashdeberta_b200.linear_int8.default, (x, wq, ws, b, None, False, torch.bfloat16),
                          test_utils=("test_schema", "test_faketensor"))
    for bad, err in [(lambda: ops.linear_int8(x[:, :32], wq, ws), ValueError), (lambda: ops.linear_int8(x, wq.float(), ws), ValueError),
                     (lambda: ops.linear_int8(x, wq, ws.double()), ValueError), (lambda: ops.linear_int8(x.double(), wq, ws), TypeError),
                     (lambda: ops.linear_int8(wq, wq, ws), TypeError), (lambda: ops.linear_int8(x, wq, ws, b, x_scale=ws), TypeError),
                     (lambda: ops.linear_int8(wq, wq, ws, x_scale=ws[:4]), ValueError), (lambda: ops.linear_int8(x, wq, ws, b[:4]), ValueError),
                     (lambda: ops.linear_int8(x, wq, ws, b, out_dtype=torch.float16), ValueError), (lambda: ops.linear_int8(x, wq.cpu(), ws), ValueError),
                     (lambda: ops.linear_int8(x, wq, ws, out_dtype=torch.float64), TypeError), (lambda: ops.quantize_int8(x.double()), TypeError),
                     (lambda: ops.linear_int8(x.requires_grad_(), wq, ws), RuntimeError)]:
        with pytest.raises(err):
            bad()
    assert ops.linear_int8(x.detach()[:0], wq, ws).shape == (0, 48) and ops.quantize_int8(x.detach()[:0])[1].shape == (0,)
