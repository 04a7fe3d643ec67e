"""ops.grad_norm, ops.clip_grads_ and ops.clip_grad_norm_ against float64.

The norm adds 32 squares at a time in fp32 (each sum off by at most 32 * 2^-24 relative, all of one sign) and the rest in fp64, and is rounded
to fp32: 2^-18 relative covers it (half of it, the square root halves).  A scaled element is a product of fp32 numbers whose factor is off by
as much, rounded to its type."""
import math

import pytest
import torch

from flashdeberta_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _tensors(sizes, seed, types=TYPES, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*(s if isinstance(s, tuple) else (s,)), generator=g) * std).to(types[i % len(types)]).to(DEV) for i, s in enumerate(sizes)]


def _norm64(ts, p):
    flat = torch.cat([t.detach().double().flatten() for t in ts]) if ts else torch.zeros(1, dtype=torch.float64)
    return torch.linalg.vector_norm(flat, p).item()


def _check(got, want, factor):
    for a, t in zip(got, want):
        w = t.double() * factor
        info = torch.finfo(a.dtype)
        allowed = (info.eps / 2 + 2.0 ** -18) * w.abs() + (2.0 ** -25 if a.dtype == torch.float16 else info.tiny)
        assert ((a.double() - w).abs() <= allowed).all()


SIZES = [(1,), 7, (16384,), (16385,), (3, 5000), (257, 129), 0, (1000, 1000), 8, 2 ** 21 + 3]


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("types", [[t] for t in TYPES] + [TYPES], ids=["bf16", "fp16", "fp32", "mixed"])
def test_norm_and_scaling(p, types):
    ts = _tensors(SIZES, 1, types, std=0.1)
    want = _norm64(ts, p)
    norm = ops.grad_norm(ts, p)
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(norm.item() - want) <= 2.0 ** -18 * want
    for bound in (0.37 * want, 3 * want):
        factor = min(1.0, bound / (want + 1e-6))
        mine = [t.clone() for t in ts]
        got = ops.clip_grads_(mine, bound, norm_type=p)
        assert torch.equal(got, norm)
        _check(mine, ts, factor)
        if factor == 1.0:
            assert all(torch.equal(a, b) for a, b in zip(mine, ts))
        for t in TYPES:
            out = [torch.full_like(x, 7.0, dtype=t) for x in ts]
            given = [x.clone() for x in ts]
            assert torch.equal(ops.clip_grads_(given, bound, norm_type=p, out=out), norm)
            _check(out, ts, factor)
            assert all(torch.equal(a, b) for a, b in zip(given, ts))
            if t == types[0] and len(types) == 1:
                assert all(torch.equal(a, b) for a, b in zip(out, mine))


def test_against_torch():
    params = [torch.nn.Parameter(t) for t in _tensors([(300, 200), 300, (7, 11, 13)], 2, [torch.float32])]
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params] + [torch.nn.Parameter(torch.zeros(3, device=DEV))]
    for p, q in zip(params, twins):
        p.grad, q.grad = torch.sin(p.detach()), torch.sin(p.detach())
    mine, theirs = ops.clip_grad_norm_(params + [torch.nn.Parameter(torch.zeros(3, device=DEV))], 1.5), torch.nn.utils.clip_grad_norm_(twins, 1.5)
    torch.testing.assert_close(mine, theirs, rtol=1e-6, atol=0)
    for p, q in zip(params, twins):
        torch.testing.assert_close(p.grad, q.grad, rtol=1e-6, atol=0)
    ops.clip_grad_norm_(params[0], 0.0)
    assert params[0].grad.abs().max().item() == 0.0


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e18, 1e30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_squares_beyond_the_range_of_fp32(scale, dtype):
    ts = [(t.float() * scale).to(dtype) for t in _tensors([5000, (40, 50)], 3, [torch.float32])]
    want = _norm64(ts, 2.0)
    assert abs(ops.grad_norm(ts).item() - want) <= 2.0 ** -18 * want
    mine = [t.clone() for t in ts]
    ops.clip_grads_(mine, scale)
    _check(mine, ts, min(1.0, scale / (want + 1e-6)))


def test_mixed_magnitudes_and_zeros():
    t = torch.zeros(100000, device=DEV)
    assert ops.grad_norm([t, t[:0]]).item() == 0.0
    t[777], t[50000], t[99999] = 1e-25, 3e20, -4e20
    assert abs(ops.grad_norm([t]).item() / 5e20 - 1) < 1e-6


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_infinities_and_nan(p):
    ts = _tensors([100, 20000], 4, [torch.float32])
    ts[1][12345] = -math.inf
    mine = [t.clone() for t in ts]
    assert ops.clip_grads_(mine, 1.0, norm_type=p).item() == math.inf
    assert torch.isnan(mine[1][12345]) and mine[0].abs().max().item() == 0.0  # a factor of zero
    ts[0][3] = math.nan
    assert math.isnan(ops.clip_grads_(ts, 1.0, norm_type=p).item())
    assert all(torch.isnan(t).all() for t in ts)


def test_not_finite_raises_before_anything_is_scaled():
    params = [torch.nn.Parameter(torch.zeros(50, device=DEV)) for _ in range(2)]
    for q in params:
        q.grad = torch.ones(50, device=DEV)
    params[1].grad[7] = math.nan
    kept = params[0].grad.clone()
    with pytest.raises(RuntimeError, match="not finite"):
        ops.clip_grad_norm_(params, 0.1, error_if_nonfinite=True)
    assert torch.equal(params[0].grad, kept)
    params[1].grad[7] = 1.0
    assert abs(ops.clip_grad_norm_(params, 0.1, error_if_nonfinite=True).item() - 10.0) < 1e-5


@pytest.mark.parametrize("count", [119, 120, 121, 1000, 1001, 2300])
def test_many_tensors(count):
    """On either side of what one table of either size holds."""
    g = torch.Generator().manual_seed(count)
    sizes = torch.randint(0, 400, (count,), generator=g).tolist()
    sizes[5], sizes[-1] = 70000, 50001
    flat = torch.randn(sum(sizes), generator=g).to(DEV)
    ts = list(flat.split(sizes))
    want, kept = _norm64(ts, 2.0), flat.clone()
    assert abs(ops.grad_norm(ts).item() - want) <= 2.0 ** -18 * want
    assert abs(ops.clip_grads_(ts, 1.0).item() - want) <= 2.0 ** -18 * want
    _check([flat], [kept], 1.0 / (want + 1e-6))


@pytest.mark.parametrize("count,tables", [(1, 1), (1000, 1), (1001, 2), (2300, 3)])
def test_launches_are_counted(count, tables):
    """A launch takes a thousand tensors: that many for the norm, as many again to scale or one to join the norm."""
    ts = list(torch.ones(count * 3, device=DEV).split(3))
    before = ops.launch_count()
    ops.grad_norm(ts)
    assert ops.launch_count() - before == tables + 1
    ops.clip_grads_(ts, 1.0)
    assert ops.launch_count() - before == 3 * tables + 1


def test_tensors_that_start_anywhere():
    base = torch.randn(50000, device=DEV, generator=torch.Generator(DEV).manual_seed(6))
    for dtype in TYPES:
        flat = base.to(dtype)
        for off in range(1, 9):
            ts = [flat[off:20000 + off], flat[20011 + off:45000]]
            want = _norm64(ts, 2.0)
            assert abs(ops.grad_norm(ts).item() - want) <= 2.0 ** -18 * want
            out = [torch.empty(t.numel() + 3, dtype=torch.float32, device=DEV)[3:] for t in ts]
            ops.clip_grads_(ts, 1.0, out=out)
            _check(out, ts, 1.0 / (want + 1e-6))


def test_orders_strides_and_views():
    g = torch.Generator().manual_seed(7)
    a = torch.randn(60, 70, generator=g).to(DEV)
    ts = [a.t(), torch.randn(4, 5, 6, 7, generator=g).to(DEV).to(memory_format=torch.channels_last), torch.randn(30, 90, generator=g).to(DEV)[:, 3:80],
          torch.randn(9, generator=g).to(DEV)[::2]]
    kept = [t.clone() for t in ts]
    want = _norm64(ts, 2.0)
    assert abs(ops.grad_norm(ts).item() - want) <= 2.0 ** -18 * want
    out = [torch.zeros(t.shape, device=DEV) for t in ts]
    ops.clip_grads_(ts, 2.0, out=out)
    _check(out, kept, 2.0 / (want + 1e-6))
    strided = [torch.zeros(t.shape[::-1], device=DEV).permute(*range(t.dim() - 1, -1, -1)) for t in ts]
    ops.clip_grads_(ts, 2.0, out=strided)
    _check(strided, kept, 2.0 / (want + 1e-6))
    gaps = [torch.zeros(*t.shape, 2, device=DEV)[..., 0] for t in ts]
    ops.clip_grads_(ts, 2.0, out=gaps)
    _check(gaps, kept, 2.0 / (want + 1e-6))
    ops.clip_grads_(ts, 2.0)
    _check(ts, kept, 2.0 / (want + 1e-6))
    wide = torch.randn(1, 40, generator=g).to(DEV).expand(8, 40)  # (a gradient of a sum: its rows are one row)
    assert abs(ops.grad_norm([wide]).item() - _norm64([wide], 2.0)) <= 1e-5
    out = [torch.zeros(8, 40, device=DEV)]
    ops.clip_grads_([wide], 1.0, out=out)
    _check(out, [wide], 1.0 / (_norm64([wide], 2.0) + 1e-6))


def test_what_surrounds_a_strided_tensor_is_left_alone():
    base = torch.full((30, 90), 5.0, device=DEV)
    t = base[:, 3:80]
    ops.clip_grads_([t], 1.0)
    assert (base[:, :3] == 5).all() and (base[:, 80:] == 5).all() and (t < 5).all()
    flat = torch.full((1000,), 5.0, dtype=torch.bfloat16, device=DEV)
    ops.clip_grads_([flat[101:804]], 1.0)
    assert (flat[:101] == 5).all() and (flat[804:] == 5).all() and (flat[101:804] < 5).all()


def test_refusals():
    a, b = torch.ones(100, device=DEV), torch.ones(100, device=DEV)
    for bad, err in [(lambda: ops.clip_grads_([a, a], 1.0), ValueError), (lambda: ops.clip_grads_([a, a[50:]], 1.0), ValueError),
                     (lambda: ops.clip_grads_([a, b], 1.0, out=[b, a]), ValueError), (lambda: ops.clip_grads_([a], 1.0, out=[b, b]), ValueError),
                     (lambda: ops.clip_grads_([a], 1.0, out=[b[:50]]), ValueError), (lambda: ops.clip_grads_([a, b], 1.0, out=[b, b]), ValueError),
                     (lambda: ops.clip_grads_([a.double()], 1.0), TypeError), (lambda: ops.grad_norm([a.to_sparse()]), TypeError),
                     (lambda: ops.clip_grads_([a[:50]], 1.0, out=[a[20:70]]), ValueError), (lambda: ops.grad_norm([a], 0.5), ValueError),
                     (lambda: ops.clip_grads_([a.expand(2, 100)], 1.0), (ValueError, RuntimeError))]:
        with pytest.raises(err):
            bad()
    class Odd(torch.Tensor):
        pass

    with pytest.raises(TypeError, match="plain tensors"):
        ops.grad_norm([a.as_subclass(Odd)])
    assert (a == 1).all() and (b == 1).all()
    assert abs(ops.grad_norm([a, a]).item() - math.sqrt(200)) < 1e-4  # (read twice, counted twice)


def test_strided_tensors_that_overlap_are_refused():
    """As tensors without gaps are, and before anything is scaled."""
    m, other = torch.ones(30, 90, device=DEV), torch.full((30, 7), 3.0, device=DEV)
    out = torch.zeros(30, 90, device=DEV)
    t = m[:, 3:80]
    for bad in (lambda: ops.clip_grads_([t, t], 1.0), lambda: ops.clip_grads_([other, m[:, :10], m[:, 9:20]], 1.0), lambda: ops.clip_grads_([t, m], 1.0),
                lambda: ops.clip_grads_([other, other.clone()], 1.0, out=[out[:, :7], out[:, 5:12]]), lambda: ops.clip_grads_([m[:, ::2], m[:, ::3]], 1.0),
                lambda: ops.clip_grads_([m[:, :7], other], 1.0, out=[out[:, :7], m[:, 6:13]]), lambda: ops.clip_grads_([m[:1].expand(5, 90)], 1.0),
                lambda: ops.clip_grads_([m[:, :7].contiguous()], 1.0, out=[out[:1, :7].expand(30, 7)]),
                lambda: ops.clip_grads_([m.t()[:10], m.t()[9:]], 1.0)):
        with pytest.raises(ValueError, match="overlap"):
            bad()
    assert (m == 1).all() and (other == 3).all() and (out == 0).all()
    norm = ops.clip_grads_([m[:, :40], m[:, 40:41], m[:, 41:]], 1.0)  # slices beside one another
    assert abs(norm.item() - 2700 ** 0.5) < 1e-4 and (m == m[0, 0]).all() and abs(m[0, 0].item() - 2700 ** -0.5) < 1e-6
    m.fill_(1.0)
    assert abs(ops.clip_grads_([m[:, ::2], m[:, 1::2]], 1.0).item() - 2700 ** 0.5) < 1e-4 and (m == m[0, 0]).all()
    square = torch.arange(64.0, device=DEV).view(8, 8)  # its own output in another order
    want = square.t() / square.norm()
    ops.clip_grads_([square[:, :]], 1.0, out=[square.t()])
    torch.testing.assert_close(square, want, rtol=1e-5, atol=0)


def test_streams_and_captures():
    ts = _tensors([(500, 600), 333, (64, 64)], 8)
    kept = [t.clone() for t in ts]
    want = [t.clone() for t in ts]
    norm = ops.clip_grads_(want, 2.0)
    torch.cuda.synchronize()
    results = []
    for _ in range(3):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            out = [torch.empty_like(t) for t in ts]
            results.append((ops.clip_grads_(ts, 2.0, out=out), out))
    torch.cuda.synchronize()
    assert all(torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(o, want)) for n, o in results)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = ops.clip_grads_(ts, 2.0)
    for step in range(2):
        for t, k in zip(ts, kept):
            t.copy_(k * (step + 1))
        graph.replay()
        torch.cuda.synchronize()
        w = _norm64([k * (step + 1) for k in kept], 2.0)
        assert abs(held.item() - w) <= 2.0 ** -18 * w
        _check(ts, [k * (step + 1) for k in kept], 2.0 / (w + 1e-6))


def test_what_is_written_counts_as_modified():
    """Version counters move, as with torch's own in-place operators: autograd and this package's caches go by them."""
    ts = _tensors([(40, 50), 33], 9, [torch.float32])
    out = [torch.empty_like(t) for t in ts]
    before = [t._version for t in ts + out]
    ops.grad_norm(ts)
    assert [t._version for t in ts + out] == before
    ops.clip_grads_(ts, 1.0, out=out)
    assert [t._version for t in ts] == before[:2] and all(o._version > b for o, b in zip(out, before[2:]))
    ops.clip_grads_(ts, 1.0)
    assert all(t._version > b for t, b in zip(ts, before))
    w = torch.nn.Parameter(ts[0].clone())
    y = (w * w).sum()
    ops.clip_grads_([w.detach()], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_parameters_on_a_model_with_shared_and_frozen_ones():
    model = torch.nn.Sequential(torch.nn.Linear(40, 40), torch.nn.Linear(40, 40)).to(DEV)
    model[1].weight = model[0].weight
    model[1].bias.requires_grad_(False)
    model(torch.randn(8, 40, device=DEV)).square().sum().backward()
    want = _norm64([p.grad for p in model.parameters() if p.grad is not None], 2.0)
    got = ops.clip_grad_norm_(model.parameters(), 0.01)
    assert abs(got.item() - want) <= 2.0 ** -18 * want
    assert abs(ops.grad_norm([p.grad for p in model.parameters() if p.grad is not None]).item() - 0.01) < 1e-4
