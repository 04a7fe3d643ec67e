"""ops.residual_norm and its backward against the formulas in 64 bits.

Tolerances.  A result is rounded once to its type (half a step of it: finfo.eps / 2 relative).  Before that everything is fp32: a row's
sums add 8 elements per thread, then five shuffles, then up to 32 warps, so at most 45 roundings in a row, and the steps around them
a dozen: 64 roundings of 2^-24 of the largest magnitude that takes part.  What a norm makes of the rounding of its input grows with
max|row| / deviation (its condition).  A sum over rows adds at most `rows` terms one after another, each off by the same 64 roundings."""
import gc
import itertools

import pytest
import torch

from flashdeberta_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
NAMES = ("x", "residual", "weight", "bias", "post_weight", "post_bias", "gate")


def _inputs(shape, dtype, rms, post, gate, seed, residual=True, params=None):
    g = torch.Generator().manual_seed(seed)
    h = shape[-1]

    def normal(*s, std=1.0, mean=0.0, t=dtype):
        return (torch.randn(*s, generator=g) * std + mean).to(t).to(DEV)

    p = params or dtype
    t = dict.fromkeys(NAMES)
    t["x"] = normal(*shape, mean=0.3)
    t["residual"] = normal(*shape, std=2.0) if residual else None
    t["weight"] = normal(h, std=0.3, mean=1.0, t=p)
    t["bias"] = None if rms else normal(h, t=p)
    if post:
        t["post_weight"] = normal(h, std=0.3, mean=1.0, t=p)
        t["post_bias"] = None if rms else normal(h, t=p)
    if gate is not None:
        t["gate"] = normal(*gate, std=0.5, mean=0.5)
    return t, (normal(*shape), normal(*shape, std=0.5))


def _call(t, eps=1e-5, rms=False, scale=1.0):
    return ops.residual_norm(t["x"], t["residual"], t["weight"], t["bias"], eps, rms=rms, post_weight=t["post_weight"],
                             post_bias=t["post_bias"], gate=t["gate"], residual_scale=scale)


def _norm64(x, w, b, eps, rms):
    c = x if rms else x - x.mean(-1, keepdim=True)
    inv = (c.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    y = c * inv * w
    return (y if b is None else y + b), c * inv, inv


def _want(t, grads, eps, rms, scale):
    """Results and gradients in 64 bits, and for each the bound on what fp32 may lose."""
    v = {k: None if a is None else a.detach().double().cpu().requires_grad_() for k, a in t.items()}
    h, rows = v["x"].shape[-1], v["x"].numel() // v["x"].shape[-1]
    top = lambda a: a.detach().abs().amax(-1, keepdim=True)
    cond = 1.0
    u = v["x"]
    if v["post_weight"] is not None:
        u, hat1, inv1 = _norm64(v["x"], v["post_weight"], v["post_bias"], eps, rms)
        cond = 1.0 + top(v["x"]) * inv1.detach()
    gate = 1.0 if v["gate"] is None else v["gate"]
    stream = gate * u if v["residual"] is None else gate * u + scale * v["residual"]
    normed, hat2, inv2 = _norm64(stream, v["weight"], v["bias"], eps, rms)
    g64 = [a.double().cpu() for a in grads]
    leaves = [k for k in NAMES if v[k] is not None]
    got = dict(zip(leaves, torch.autograd.grad((normed, stream), [v[k] for k in leaves], g64, retain_graph=True)))
    a = lambda z: z.detach().abs() if torch.is_tensor(z) else abs(z)
    parts = a(gate) * a(u) + (0 if v["residual"] is None else abs(scale) * a(v["residual"]))
    m_stream = 64 * U * cond * parts.amax(-1, keepdim=True)
    cond2 = cond * (1.0 + parts.amax(-1, keepdim=True) * inv2.detach())
    m_normed = 64 * U * cond2 * (a(hat2).amax(-1, keepdim=True) * a(v["weight"]) + (0 if v["bias"] is None else a(v["bias"])))
    bound = {"normed": m_normed, "stream": m_stream}
    # gradients: the magnitudes of the terms, through both norms
    dn, ds = a(g64[0]), a(g64[1])
    y = dn * a(v["weight"])
    mean = lambda z: z.mean(-1, keepdim=True)
    dz = ds + inv2.detach() * (y + mean(y) + a(hat2) * mean(y * a(hat2)))
    err = 64 * U * cond2
    summed = lambda terms, like: (terms.expand(v["x"].shape) * (err * (1 + rows / 64.0))).sum_to_size(like.shape)
    bound["residual"] = err * abs(scale) * dz
    bound["weight"], bound["bias"] = summed(dn * a(hat2), v["weight"]), summed(dn, v["weight"])
    du = dz * a(gate)
    if v["post_weight"] is not None:
        p = du * a(v["post_weight"])
        bound["x"] = err * inv1.detach() * (p + mean(p) + a(hat1) * mean(p * a(hat1)))
        bound["post_weight"], bound["post_bias"] = summed(du * a(hat1), v["weight"]), summed(du, v["weight"])
        # (A and B are added up apart: their parts may be larger than what they come to)
        spread = a(hat1) * a(v["post_weight"]) + (0 if v["post_bias"] is None else a(v["post_bias"]))
    else:
        bound["x"], spread = err * du, a(u)
    if v["gate"] is not None:
        bound["gate"] = summed(dz * spread, v["gate"])
    return {"normed": normed.detach(), "stream": stream.detach(), **got}, bound


def _check(name, got, want, bound):
    assert got.shape == want.shape, name
    allowed = torch.finfo(got.dtype).eps / 2 * want.abs() + bound + torch.finfo(got.dtype).tiny
    if got.dtype == torch.float16:
        allowed = allowed + 2.0 ** -25  # half a step of its smallest numbers
    off = (got.double().cpu() - want).abs()
    worst = (off / allowed).max().item()
    assert worst <= 1.0, f"{name}: {worst:.3g} times what is allowed"


def _compare(t, grads, eps=1e-5, rms=False, scale=1.0):
    want, bound = _want(t, grads, eps, rms, scale)
    with torch.no_grad():
        plain = _call(t, eps, rms, scale)
    leaves = [k for k in NAMES if t[k] is not None]
    for k in leaves:
        t[k].requires_grad_()
    normed, stream = _call(t, eps, rms, scale)
    assert torch.equal(normed.detach(), plain[0]) and torch.equal(stream.detach(), plain[1])
    got = dict(zip(leaves, torch.autograd.grad((normed, stream), [t[k] for k in leaves], grads)))
    again = torch.autograd.grad(_call(t, eps, rms, scale), [t[k] for k in leaves], grads)
    for k, a in zip(leaves, again):
        assert torch.equal(got[k], a), k  # the same bits every time
        assert got[k].dtype == t[k].dtype
    _check("normed", normed.detach(), want["normed"], bound["normed"])
    _check("stream", stream.detach(), want["stream"], bound["stream"])
    for k in leaves:
        _check("d" + k, got[k], want[k], bound[k])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rms,post", list(itertools.product([False, True], [False, True])))
@pytest.mark.parametrize("gate", [None, "channel", "sequence", "element"])
@pytest.mark.parametrize("shape", [(3, 37, 264), (2, 5, 769)])
def test_every_form(dtype, rms, post, gate, shape):
    b, s, h = shape
    gate = {None: None, "channel": (h,), "sequence": (b, 1, h), "element": (b, s, h)}[gate]
    t, grads = _inputs(shape, dtype, rms, post, gate, 1)
    _compare(t, grads, rms=rms, scale=1.25)


@pytest.mark.parametrize("hidden", [1, 2, 7, 8, 31, 64, 255, 256, 512, 520, 1000, 1024, 1536, 2047, 4096, 4097, 5000, 8192])
@pytest.mark.parametrize("rows", [1, 3])
def test_widths(hidden, rows):
    t, grads = _inputs((rows, hidden), torch.bfloat16, False, True, (hidden,), 2)
    _compare(t, grads, eps=1e-3)


@pytest.mark.parametrize("dtype,hidden,gate", [(torch.bfloat16, 8192, "sequence"), (torch.float32, 8191, "element"), (torch.float16, 4104, "sequence")])
def test_long_rows_with_gates(dtype, hidden, gate):
    t, grads = _inputs((3, 4, hidden), dtype, False, True, (3, 1, hidden) if gate == "sequence" else (3, 4, hidden), 3)
    _compare(t, grads)


@pytest.mark.parametrize("batch,seqlen,hidden", [(1, 1, 64), (1, 4099, 40), (5, 1021, 96), (700, 3, 128), (2500, 2, 72), (3, 1, 256)])
@pytest.mark.parametrize("rms", [False, True])
def test_rows_and_groups(batch, seqlen, hidden, rms):
    """More groups than teams of warps, more teams than rows, groups that end inside a team's rows."""
    t, grads = _inputs((batch, seqlen, hidden), torch.float32, rms, True, (batch, 1, hidden), 4)
    _compare(t, grads, rms=rms, scale=0.7)


@pytest.mark.parametrize("dtype,rms,gate", [(torch.bfloat16, False, "sequence"), (torch.float16, True, "sequence"), (torch.float16, False, "element"),
                                            (torch.bfloat16, True, "element"), (torch.bfloat16, False, None)])
@pytest.mark.parametrize("batch,seqlen,hidden,residual", [(31, 331, 40, True), (7, 401, 1000, False), (3, 650, 2056, True), (2, 383, 4096, True)])
def test_many_rows_per_team(dtype, rms, gate, batch, seqlen, hidden, residual):
    """Rows on their way ahead of the one that is worked on, several times around, in groups that end in between."""
    gate = {None: None, "sequence": (batch, 1, hidden), "element": (batch, seqlen, hidden)}[gate]
    t, grads = _inputs((batch, seqlen, hidden), dtype, rms, True, gate, 11, residual=residual)
    _compare(t, grads, rms=rms, scale=0.7)


def test_without_residual_and_with_parameters_in_fp32():
    t, grads = _inputs((2, 33, 768), torch.bfloat16, False, True, (768,), 5, residual=False, params=torch.float32)
    t["gate"] = t["gate"].float()
    _compare(t, grads)
    t, grads = _inputs((2, 33, 200), torch.float16, True, False, (2, 33, 200), 6, residual=False, params=torch.float32)
    t["gate"] = t["gate"].float()
    _compare(t, grads, rms=True)


def test_gate_that_broadcasts_in_another_way():
    """A gate per position, shared by the sequences, and one number per row: taken as one per element; their gradients are summed."""
    for shape in [(1, 9, 136), (4, 9, 1), (9, 136), (1, 136), (1, 1, 136)]:
        t, grads = _inputs((4, 9, 136), torch.float32, False, True, shape, 7)
        _compare(t, grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 9, 136), (4, 9, 1), (9, 1), (4, 1, 1), (1,)])
def test_gradient_of_a_shared_gate_is_rounded_once(dtype, shape):
    """The sum over what shares a number of the gate, of parts that have not been rounded to the gate's type."""
    t, grads = _inputs((4, 9, 136), dtype, False, True, shape, 23)
    _compare(t, grads)


def test_one_gradient_and_only_what_is_asked_for():
    t, grads = _inputs((2, 17, 320), torch.float32, False, True, (320,), 8)
    want, bound = _want(t, (grads[0], torch.zeros_like(grads[1])), 1e-5, False, 1.0)
    t["weight"].requires_grad_()
    t["x"].requires_grad_()
    normed, stream = _call(t)
    got = torch.autograd.grad(normed, [t["x"], t["weight"]], grads[0])
    _check("dx", got[0], want["x"], bound["x"])
    _check("dweight", got[1], want["weight"], bound["weight"])
    want, bound = _want(t, (torch.zeros_like(grads[0]), grads[1]), 1e-5, False, 1.0)
    normed, stream = _call(t)
    got = torch.autograd.grad(stream, [t["x"], t["weight"]], grads[1])
    _check("dx", got[0], want["x"], bound["x"])
    assert got[1].abs().max().item() == 0.0


def test_gradient_against_differences():
    """sum(out * c) along a direction, by central differences of the kernel's own results.  Step 2^-7 of unit-variance inputs: the
    rounding of results of size 3 leaves sqrt(n) * 3 * 2^-24 / 2^-7 (n = 2 * 1320 terms: 1.2e-3), the third derivative of the norm
    (of order one per unit of the direction, its squared step 6e-5) less than that; the derivative is of order sqrt(n) = 50."""
    t, grads = _inputs((3, 5, 88), torch.float32, False, True, (3, 1, 88), 9)
    leaves = [k for k in NAMES if t[k] is not None]
    for k in leaves:
        t[k].requires_grad_()
    got = torch.autograd.grad(_call(t), [t[k] for k in leaves], grads)
    gen = torch.Generator().manual_seed(10)
    for k, g in zip(leaves, got):
        d = torch.randn(t[k].shape, generator=gen).to(DEV)
        step = 2.0 ** -7
        value = []
        for sign in (1, -1):
            moved = dict(t)
            moved[k] = (t[k] + sign * step * d).detach()
            with torch.no_grad():
                n, s = _call(moved)
            value.append((n.double() * grads[0].double()).sum() + (s.double() * grads[1].double()).sum())
        numeric = ((value[0] - value[1]) / (2 * step)).item()
        analytic = (g.double() * d.double()).sum().item()
        assert abs(numeric - analytic) <= 2e-2 + 2e-3 * (g.double().norm() * d.double().norm()).item(), k


def test_rows_far_from_zero_keep_their_deviation():
    """Mean 1000, deviation one: what a difference of summed squares would lose."""
    t, grads = _inputs((4, 512), torch.float32, False, False, None, 11)
    t["residual"] = t["residual"] + 1000.0
    _compare(t, grads)


def test_constant_rows_and_non_finite_rows_stay_apart():
    t, _ = _inputs((5, 256), torch.bfloat16, False, True, None, 12)
    t["x"][1] = 3.0                     # no deviation: the bias alone goes on
    t["x"][2, 7] = float("inf")
    t["x"][3, 9] = float("nan")
    clean, _ = _inputs((5, 256), torch.bfloat16, False, True, None, 12)
    normed, stream = _call(t)
    n0, s0 = _call(clean)
    for r in (0, 4):
        assert torch.equal(normed[r], n0[r]) and torch.equal(stream[r], s0[r])
    assert torch.isfinite(normed[1]).all()
    want = (t["post_bias"].float() + t["residual"][1].float()).to(torch.bfloat16)
    assert torch.equal(stream[1], want)
    assert torch.isnan(normed[2]).all() and torch.isnan(normed[3]).all()


def test_no_rows():
    t, grads = _inputs((0, 7, 64), torch.bfloat16, False, True, (64,), 13)
    leaves = [k for k in NAMES if t[k] is not None]
    for k in leaves:
        t[k].requires_grad_()
    n, s = _call(t)
    assert n.shape == s.shape == (0, 7, 64)
    got = torch.autograd.grad((n, s), [t[k] for k in leaves], grads)
    for k, g in zip(leaves, got):
        assert g.shape == t[k].shape and (g.numel() == 0 or g.abs().max().item() == 0.0)


def test_views_and_unaligned_rows():
    """Rows that are slices of wider ones, transposed gradients and tensors that start on two bytes."""
    t, grads = _inputs((2, 6, 128), torch.bfloat16, False, True, (2, 1, 128), 14)
    want, bound = _want(t, grads, 1e-5, False, 1.0)
    wide = torch.zeros(2, 6, 200, dtype=torch.bfloat16, device=DEV)
    wide[..., 3:131] = t["x"]
    odd = torch.zeros(2 * 6 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 6, 128)
    odd.copy_(t["residual"])
    t["x"], t["residual"] = wide[..., 3:131].requires_grad_(), odd.requires_grad_()
    n, s = _call(t)
    dn = grads[0].permute(1, 0, 2).contiguous().permute(1, 0, 2)
    got = torch.autograd.grad((n, s), [t["x"], t["residual"]], (dn, grads[1]))
    _check("normed", n.detach(), want["normed"], bound["normed"])
    _check("dx", got[0], want["x"], bound["x"])
    _check("dresidual", got[1], want["residual"], bound["residual"])


def test_side_stream_and_two_calls_at_once():
    t, grads = _inputs((8, 300, 512), torch.bfloat16, False, True, (8, 1, 512), 15)
    leaves = [k for k in NAMES if t[k] is not None]
    for k in leaves:
        t[k].requires_grad_()
    want = [*_call(t), *torch.autograd.grad(_call(t), [t[k] for k in leaves], grads)]
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    for st in streams:
        with torch.cuda.stream(st):
            out = _call(t)
            results.append([*out, *torch.autograd.grad(out, [t[k] for k in leaves], grads)])
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_captured_step_is_replayed():
    t, grads = _inputs((4, 50, 384), torch.bfloat16, True, True, (4, 1, 384), 16)
    leaves = [k for k in NAMES if t[k] is not None]
    for k in leaves:
        t[k].requires_grad_()

    def step():
        out = _call(t, rms=True)
        return [*out, *torch.autograd.grad(out, [t[k] for k in leaves], grads)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    gc.collect()  # no eager graph of these leaves lives while the capture runs
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    other, _ = _inputs((4, 50, 384), torch.bfloat16, True, True, (4, 1, 384), 17)
    with torch.no_grad():
        for k in leaves:
            t[k].copy_(other[k])
    graph.replay()
    torch.cuda.synchronize()
    kept = [h.detach().clone() for h in held]
    del held
    assert all(torch.equal(a, b.detach()) for a, b in zip(kept, step()))


def test_refusals():
    t, _ = _inputs((2, 3, 64), torch.bfloat16, False, True, (64,), 20)
    x, r, w, b, g = (t[k] for k in ("x", "residual", "weight", "bias", "gate"))
    for bad, err in [
            (lambda: ops.residual_norm(x.double(), None, w), TypeError), (lambda: ops.residual_norm(x, r[:1], w), ValueError),
            (lambda: ops.residual_norm(x, r.float(), w), ValueError), (lambda: ops.residual_norm(x, r, w[:8]), ValueError),
            (lambda: ops.residual_norm(x, r, w.half()), TypeError), (lambda: ops.residual_norm(x, r, w, b.float()), TypeError),
            (lambda: ops.residual_norm(x, r, w, b, rms=True), ValueError), (lambda: ops.residual_norm(x, r, w, post_bias=b), ValueError),
            (lambda: ops.residual_norm(x, r, w, post_weight=w[None]), ValueError), (lambda: ops.residual_norm(x, r, w, gate=g.double()), TypeError),
            (lambda: ops.residual_norm(x, r, w, gate=g[:8]), ValueError), (lambda: ops.residual_norm(x, r, w, gate=x[:, :2]), ValueError),
            (lambda: ops.residual_norm(x, r, w, gate=x[None]), ValueError), (lambda: ops.residual_norm(x, r, w.cpu()), ValueError),
            (lambda: ops.residual_norm(x, r.cpu(), w), ValueError), (lambda: ops.residual_norm(x, r, w, gate=g.cpu()), ValueError),
            (lambda: ops.residual_norm(torch.zeros(2, 8193, device=DEV), None, torch.zeros(8193, device=DEV)), ValueError),
            (lambda: ops.residual_norm(x[..., :0], None, w[:0]), ValueError)]:
        with pytest.raises(err):
            bad()


@pytest.mark.parametrize("gate,wanted,launches", [
    (None, ("x",), 1), (None, ("x", "bias"), 2), ((64,), ("gate",), 2), ((2, 1, 64), ("x", "gate"), 2), ((2, 3, 64), ("x", "gate"), 1),
    ((2, 3, 64), ("gate", "post_weight"), 2), ((2, 1, 64), ("residual",), 1)])
def test_launches_are_counted(gate, wanted, launches):
    """One for the rows, one more where a gradient is a sum over them."""
    t, grads = _inputs((2, 3, 64), torch.float32, False, True, gate, 21)
    for k in wanted:
        t[k].requires_grad_()
    before = ops.launch_count()
    out = _call(t)
    assert ops.launch_count() - before == 1
    torch.autograd.grad(out, [t[k] for k in wanted], grads)
    assert ops.launch_count() - before == 1 + launches


def test_in_a_layer_beside_add_layernorm():
    """The tail of this package's own output blocks: the same result as ops.add_layernorm up to the sum that it rounds first."""
    t, _ = _inputs((64, 768), torch.bfloat16, False, False, None, 18)
    normed, stream = _call(t, eps=1e-7)
    old = ops.add_layernorm(t["x"], t["residual"], t["weight"], t["bias"], 1e-7)
    # half a step of the sum (up to 8) through a deviation of 2.2 and a weight up to 2, and half a step of either result (up to 8)
    assert (normed.float() - old.float()).abs().max().item() <= 8 * 2.0 ** -8 * (1 / 2.0 * 2.0 + 2)
    assert torch.equal(stream, (t["x"].float() + t["residual"].float()).bfloat16())


def test_tracing_and_batched_gradients():
    t, grads = _inputs((2, 9, 64), torch.float32, False, True, (2, 1, 64), 19)
    leaves = [k for k in NAMES if t[k] is not None]
    for k in leaves:
        t[k].requires_grad_()
    want = torch.autograd.grad(_call(t), [t[k] for k in leaves], grads)
    fn = torch.compile(lambda t: _call(t), fullgraph=True, backend="aot_eager")
    got = torch.autograd.grad(fn(t), [t[k] for k in leaves], grads)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    args = (t["x"], t["residual"], t["weight"], t["bias"], t["post_weight"], t["post_bias"], t["gate"], 1e-5, False, 1.0)
    torch.library.opcheck(torch.ops.flashdeberta_b200.residual_norm.default, args,
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    normed, stream = _call(t)
    two = torch.stack([grads[0], 2 * grads[0]])
    got = torch.autograd.grad(normed, [t["x"], t["weight"]], two, is_grads_batched=True)
    one = torch.autograd.grad(_call(t)[0], [t["x"], t["weight"]], grads[0])
    for a, b in zip(got, one):
        assert torch.equal(a[0], b) and torch.equal(a[1], 2 * b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hidden", [1, 5, 9, 250, 257, 263, 767, 1023, 1027, 2050, 4099])
def test_16_bit_rows_that_start_anywhere(dtype, hidden):
    """Every shift of a row against 16 bytes, in results and gradients, with what lies around the tensors left alone."""
    for off in range(0, 8, 1 if hidden < 300 else 3):
        t, grads = _inputs((3, 5, hidden), dtype, False, True, (3, 5, hidden), hidden + off)
        want, bound = _want(t, grads, 1e-5, False, 1.0)
        hold = {}
        for k in ("x", "residual", "gate"):
            hold[k] = torch.full((15 * hidden + 24,), 9.0, dtype=dtype, device=DEV)
            v = hold[k][8 + off:8 + off + 15 * hidden].view(3, 5, hidden)
            v.copy_(t[k])
            t[k] = v
        for k in NAMES:
            t[k].requires_grad_()
        n, s = _call(t)
        got = torch.autograd.grad((n, s), [t[k] for k in NAMES], grads)
        _check("normed", n.detach(), want["normed"], bound["normed"])
        _check("stream", s.detach(), want["stream"], bound["stream"])
        for k, a in zip(NAMES, got):
            _check("d" + k, a, want[k], bound[k])
        for k, h in hold.items():
            assert (h[:8 + off] == 9).all() and (h[8 + off + 15 * hidden:] == 9).all()


def test_results_end_where_they_end():
    """Through the C entry, into the middle of larger buffers, at every shift."""
    import ctypes as C
    from flashdeberta_b200 import _lib
    for dtype, kind in ((torch.bfloat16, 0), (torch.float16, 3), (torch.float32, 1)):
        for rows, hidden in ((1, 3), (4, 33), (3, 515), (2, 1030)):
            t, _ = _inputs((rows, hidden), dtype, True, False, None, 30)
            want = ops.residual_norm(t["x"], t["residual"], t["weight"], eps=1e-5, rms=True)
            for off in range(8):
                out = [torch.full((rows * hidden + 32,), 7.0, dtype=dtype, device=DEV) for _ in range(2)]
                at = [o.data_ptr() + (16 + off) * o.element_size() for o in out]
                p = _lib.ResidualNormParams(C.sizeof(_lib.ResidualNormParams), kind, t["x"].data_ptr(), t["residual"].data_ptr(), t["weight"].data_ptr(), None, None,
                                            None, None, at[0], at[1], None, rows, 0, hidden, kind, 0, 1, 1.0, 1e-5)
                _lib.check(_lib.load().fdb_residual_norm(C.byref(p), ops.raw_stream(t["x"].device)))
                for o, w in zip(out, want):
                    assert (o[:16 + off] == 7).all() and (o[16 + off + rows * hidden:] == 7).all()
                    assert torch.equal(o[16 + off:16 + off + rows * hidden].view(rows, hidden), w)
