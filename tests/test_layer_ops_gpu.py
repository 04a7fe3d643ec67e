"""The operators around the attention together, as an encoder layer uses them."""
import copy
import threading

import pytest
import torch

from flashdeberta_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _block(h, f, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s, std: (torch.randn(*s, generator=g) * std).to(DEV)
    return {"wi": normal(f, h, std=h ** -0.5), "bi": normal(f, std=0.1).to(dtype), "wd": normal(h, f, std=f ** -0.5), "bd": normal(h, std=0.1).to(dtype),
            "gamma": (1 + normal(h, std=0.1)).to(dtype), "beta": normal(h, std=0.1).to(dtype)}


@pytest.mark.parametrize("rows,dtype", [(1, torch.bfloat16), (29, torch.float16), (777, torch.bfloat16)])
def test_feed_forward_block_in_8_bits(rows, dtype):
    """linear + GELU, linear, residual + LayerNorm, against the same block in float64 over unrounded weights.  8 bits of uniform steps leave
    a product of random factors off by about (1/127) * amax / rms / sqrt(12) = 0.9 % of its size for each factor (amax of a few hundred
    normal numbers is four times their rms): 1.3 % per layer, 1.9 % behind two, of values of order one that the LayerNorm keeps so."""
    p = _block(512, 2048, rows, dtype)
    x = torch.randn(rows, 512, generator=torch.Generator().manual_seed(rows + 1)).to(dtype).to(DEV)
    wi, si = ops.quantize_int8(p["wi"])
    wd, sd = ops.quantize_int8(p["wd"])
    hidden = ops.linear_int8(x, wi, si, p["bi"], gelu=True)
    out, stream = ops.residual_norm(ops.linear_int8(hidden, wd, sd, p["bd"]), x, p["gamma"], p["beta"], 1e-7)
    d = {k: v.double() for k, v in p.items()}
    want = torch.nn.functional.gelu(x.double() @ d["wi"].t() + d["bi"]) @ d["wd"].t() + d["bd"] + x.double()
    normed = torch.nn.functional.layer_norm(want, (512,), d["gamma"], d["beta"], 1e-7)
    assert ((stream.double() - want).norm() / want.norm()).item() < 0.02
    assert ((out.double() - normed).norm() / normed.norm()).item() < 0.02
    ops.check_status()


def test_training_steps_against_float64():
    """Three steps of gradient descent on a residual block with gated norms, its gradients clipped: parameters against the same steps in
    float64 by torch.  fp32 throughout, so what differs is rounding: a few hundred operations of 2^-24 each way, 2^-15 of the largest."""
    torch.manual_seed(0)
    h = 96
    mine = torch.nn.ParameterDict({
        "w": torch.nn.Parameter(torch.randn(h, h) / h ** 0.5), "gate": torch.nn.Parameter(torch.rand(4, 1, h)),
        "post": torch.nn.Parameter(1 + 0.1 * torch.randn(h)), "post_b": torch.nn.Parameter(0.1 * torch.randn(h)),
        "gamma": torch.nn.Parameter(1 + 0.1 * torch.randn(h)), "beta": torch.nn.Parameter(0.1 * torch.randn(h))}).to(DEV)
    theirs = copy.deepcopy(mine).double()
    x, y = torch.randn(4, 30, h, device=DEV), torch.randn(4, 30, h, device=DEV)
    prev = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        for _ in range(3):
            out, stream = ops.residual_norm(x @ mine["w"].t(), x, mine["gamma"], mine["beta"], 1e-5, post_weight=mine["post"], post_bias=mine["post_b"],
                                            gate=mine["gate"], residual_scale=0.9)
            ((out - y).square().mean() + stream.square().mean()).backward()
            u = torch.nn.functional.layer_norm(x.double() @ theirs["w"].t(), (h,), theirs["post"], theirs["post_b"], 1e-5)
            s = 0.9 * x.double() + theirs["gate"] * u
            o = torch.nn.functional.layer_norm(s, (h,), theirs["gamma"], theirs["beta"], 1e-5)
            ((o - y.double()).square().mean() + s.square().mean()).backward()
            got, want = ops.clip_grad_norm_(mine.parameters(), 0.05), torch.nn.utils.clip_grad_norm_(theirs.parameters(), 0.05)
            assert abs(got.item() / want.item() - 1) < 2.0 ** -15
            with torch.no_grad():
                for a, b in zip(mine.parameters(), theirs.parameters()):
                    a -= 10 * a.grad
                    b -= 10 * b.grad
                    a.grad = b.grad = None
        for (n, a), b in zip(mine.items(), theirs.values()):
            assert (a.double() - b).abs().max().item() <= 2.0 ** -15 * b.abs().max().item(), n
    finally:
        torch.backends.cuda.matmul.allow_tf32 = prev


def test_host_threads_at_once():
    """Four threads, each on its own stream, all operators: the results of one thread alone."""
    p = _block(256, 768, 3, torch.bfloat16)
    wi, si = ops.quantize_int8(p["wi"])
    xs = [torch.randn(40 + 30 * i, 256, device=DEV, dtype=torch.bfloat16) for i in range(4)]

    def work(x):
        a = ops.linear_int8(x, wi, si, p["bi"], gelu=True)
        n, s = ops.residual_norm(a[:, :256].contiguous(), x, p["gamma"], p["beta"])
        out = [torch.empty_like(n, dtype=torch.float32), torch.empty_like(s, dtype=torch.float32)]
        return [a, n, s, ops.clip_grads_([n, s], 0.5, out=out), *out]

    want = [work(x) for x in xs]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = work(xs[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype,gate", [(torch.bfloat16, "sequence"), (torch.float16, "element"), (torch.float32, "sequence")])
def test_backward_of_several_widths_on_host_threads_at_once(dtype, gate):
    """One form of the norms' backward, rows of four widths, a host thread and a stream for each, through the C entry: what one
    thread's launch needs of the kernel no other thread may take away."""
    from flashdeberta_b200 import _lib, norms
    lib = _lib.load()

    def problem(hidden):
        g = torch.Generator().manual_seed(hidden)
        normal = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)
        shape = (2, 3, hidden)
        tensors = [normal(*shape), normal(*shape), normal(hidden), normal(hidden), normal(hidden), normal(hidden),
                   normal(2, 1, hidden) if gate == "sequence" else normal(*shape)]
        grads = [normal(*shape), normal(*shape)]
        stats = norms._forward(*tensors, 1e-5, False, 1.0, True)[2]
        outs = [torch.empty_like(t) for t in tensors]
        head = norms._BWD.pack(norms._BWD.size + norms._FWD.size + norms._BWD_TAIL.size, 0) + norms._params(
            *tensors, tensors[0], None, stats, 1e-5, False, 1.0)
        at = [t.data_ptr() for t in grads + outs]
        need = lib.fdb_residual_norm_bwd_workspace_bytes(head + norms._BWD_TAIL.pack(*at, 0, 0))
        ws = torch.empty(need, dtype=torch.uint8, device=DEV)
        want = norms._backward(*grads, *tensors, stats, 1e-5, False, 1.0, (True,) * 7)
        return head + norms._BWD_TAIL.pack(*at, ws.data_ptr(), need), outs, want, (tensors, grads, stats, ws)

    problems = [problem(h) for h in (4096, 264, 2304, 1032)]
    torch.cuda.synchronize()
    streams, errors = [torch.cuda.Stream() for _ in problems], []

    def run(i):
        try:
            torch.cuda.set_device(0)
            for _ in range(400):
                _lib.check(lib.fdb_residual_norm_bwd(problems[i][0], streams[i].cuda_stream))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(problems))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for _, outs, want, _ in problems:
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_forward_mode_derivatives_are_refused():
    """Rather than lost: results of tensors with a tangent would have none."""
    import torch.autograd.forward_ad as fwd
    x, w = torch.randn(4, 64, device=DEV), torch.ones(64, device=DEV)
    q, s = ops.quantize_int8(torch.randn(48, 64, device=DEV))
    want = ops.residual_norm(x, x, w)
    one = torch.ones_like(x)
    with fwd.dual_level():
        dual, scale = fwd.make_dual(x, one), fwd.make_dual(s, torch.ones_like(s))
        for bad in (lambda: ops.residual_norm(dual, x, w), lambda: ops.residual_norm(x, dual, w), lambda: ops.residual_norm(x, x, fwd.make_dual(w, w)),
                    lambda: ops.quantize_int8(dual), lambda: ops.linear_int8(dual, q, s), lambda: ops.linear_int8(x, q, scale),
                    lambda: ops.grad_norm([x, dual]), lambda: ops.clip_grads_([dual], 1.0), lambda: ops.clip_grads_([x], 1.0, out=[dual])):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                bad()
        got = ops.residual_norm(x, x, w)  # (nothing here has a tangent)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert ops.linear_int8(x, q, s).shape == (4, 48) and abs(ops.grad_norm([x]).item() - x.norm().item()) < 1e-4
        leaf = x.clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.autograd.grad(ops.residual_norm(leaf, x, w)[0], leaf, fwd.make_dual(one, one))
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda v: ops.residual_norm(v, x, w), (x,), (one,))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements through each operator: the last rows as they come out alone."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of device memory")
    h, rows = 1000, 2200003
    gen = torch.Generator(DEV).manual_seed(0)
    rand = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
    x, r, dn, w, b = rand(rows, h).requires_grad_(), rand(rows, h), rand(rows, h), rand(h), rand(h)
    last = slice(rows - 777, rows)
    normed, stream = ops.residual_norm(x, r, w, b, post_weight=w, post_bias=b)
    dx, = torch.autograd.grad(normed, x, dn)
    x = x.detach()
    few = x[last].clone().requires_grad_()
    n, s = ops.residual_norm(few, r[last].clone(), w, b, post_weight=w, post_bias=b)
    assert torch.equal(normed[last], n) and torch.equal(stream[last], s) and torch.equal(dx[last], torch.autograd.grad(n, few, dn[last].clone())[0])
    few = few.detach()
    del normed, stream, dx, dn, r
    for n, dtype in ((1024, torch.bfloat16), (1001, torch.float32)):
        wq, ws = ops.quantize_int8(torch.randn(n, h, device=DEV))
        assert torch.equal(ops.linear_int8(x, wq, ws, out_dtype=dtype)[last], ops.linear_int8(few, wq, ws, out_dtype=dtype))
    assert all(torch.equal(a[last], c) for a, c in zip(ops.quantize_int8(x), ops.quantize_int8(few)))
    want = sum(c.double().square().sum() for c in x.split(100000)).sqrt().item()
    out = torch.zeros_like(x)
    assert abs(ops.clip_grads_([x.view(-1)[1:]], 1.0, out=[out.view(-1)[1:]]).item() - want) <= 2.0 ** -17 * want
    # (a factor of 1 / want up to 2^-18, and a rounding to bf16)
    assert ((out[last].double() * want - few.double()).abs() <= (2.0 ** -8 + 2.0 ** -17) * few.double().abs()).all()
    ops.check_status()
    del x, out
    torch.cuda.empty_cache()
