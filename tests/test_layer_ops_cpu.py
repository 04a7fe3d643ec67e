"""CPU-only checks of the operators around the attention: struct layouts, argument errors of the C entries and refusals of the Python
layer, all before anything is launched."""
import ctypes as C

import pytest
import torch

from flashdeberta_b200 import _lib, ops
from flashdeberta_b200.clip import _apart, _collide, _dense
from flashdeberta_b200.int8 import _rows, int8_rows
from flashdeberta_b200.norms import _gate_rows
from tests.test_abi_cpu import _refused, test_other_struct_layouts_match_the_header as _layout

STRUCTS = [("fdb_residual_norm_params", _lib.ResidualNormParams), ("fdb_residual_norm_bwd_params", _lib.ResidualNormBwdParams),
           ("fdb_linear_int8_params", _lib.LinearInt8Params), ("fdb_grad_tensor", _lib.GradTensor), ("fdb_clip_grads_params", _lib.ClipGradsParams)]
P = 0x1000


@pytest.mark.parametrize("name,struct", STRUCTS, ids=[n for n, _ in STRUCTS])
def test_struct_layouts_match_the_header(name, struct, tmp_path):
    _layout(name, struct, tmp_path)


def test_a_gradient_entry_is_four_words():
    """The table is built as rows of four 64-bit numbers, the two types in the last."""
    t = _lib.GradTensor(1, 2, 3, 4, 5)
    assert list((C.c_int64 * 4).from_buffer(t)) == [1, 2, 3, 4 | 5 << 32]


# ---- residual norm ---------------------------------------------------------------------------------------------------
def _norm(**kw):
    p = _lib.ResidualNormParams(C.sizeof(_lib.ResidualNormParams), _lib.FDB_BF16, P, P, P, P, P, P, P, P, P, P, 6, 3, 64, 0, 0, 0, 1.0, 1e-7)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(struct_bytes=0), -1), (dict(dtype=2), -1), (dict(param_dtype=3), -1), (dict(gate_dtype=3), -1), (dict(rows=-1), -1), (dict(hidden=0), -1),
    (dict(hidden=8193), -6), (dict(rows=1 << 31, gate_rows=1), -6), (dict(x=None), -1), (dict(weight=None), -1), (dict(normed=None), -1),
    (dict(rms=1), -1), (dict(rms=1, bias=None), -1), (dict(post_weight=None), -1), (dict(gate_rows=0), -1), (dict(gate_rows=4), -1),
    (dict(gate_rows=-3), -1), (dict(x=P + 1), -3), (dict(stream=P + 1), -3), (dict(bias=P + 1), -3), (dict(gate=P + 1), -3), (dict(stats=P + 8), -3),
    (dict(param_dtype=1, weight=P + 2), -3), (dict(gate_dtype=1, gate=P + 2), -3),
])
def test_residual_norm_argument_errors(change, code):
    p = _norm(**change)
    _refused(_lib.load().fdb_residual_norm(C.byref(p), None), code)


def test_residual_norm_without_rows_is_a_no_op():
    p = _norm(rows=0)
    assert _lib.load().fdb_residual_norm(C.byref(p), None) == 0


@pytest.mark.parametrize("change,fwd,code", [
    (dict(struct_bytes=0), {}, -1), (dict(dx=None), {}, -1), (dict(dnormed=None, dstream=None), {}, -1), ({}, dict(stats=None), -1),
    ({}, dict(residual=None), -1), ({}, dict(bias=None), -1), ({}, dict(gate=None), -1), ({}, dict(post_weight=None, post_bias=None), -1),
    ({}, dict(post_bias=None), -1), ({}, dict(hidden=9000), -6), (dict(dnormed=P + 1), {}, -3), (dict(dresidual=P + 1), {}, -3),
    (dict(dgate=P + 1), {}, -3), (dict(dweight=P + 1), {}, -3),
])
def test_residual_norm_backward_argument_errors(change, fwd, code):
    p = _norm(**fwd)
    b = _lib.ResidualNormBwdParams(C.sizeof(_lib.ResidualNormBwdParams), 0, p, *[P] * 10, 1 << 30)
    for k, v in change.items():
        setattr(b, k, v)
    lib = _lib.load()
    assert lib.fdb_residual_norm_bwd_workspace_bytes(C.byref(b)) == 0
    _refused(lib.fdb_residual_norm_bwd(C.byref(b), None), code)


def test_packed_parameters_have_the_structs_layout():
    from flashdeberta_b200 import int8, norms
    assert norms._FWD.size == C.sizeof(_lib.ResidualNormParams) and int8._PARAMS.size == C.sizeof(_lib.LinearInt8Params)
    assert norms._BWD.size + norms._FWD.size + norms._BWD_TAIL.size == C.sizeof(_lib.ResidualNormBwdParams)
    p = _lib.ResidualNormParams.from_buffer_copy(norms._FWD.pack(*range(1, 19), 0.5, 0.25))
    assert [getattr(p, f[0]) for f in p._fields_] == [*range(1, 19), 0.5, 0.25]
    b = _lib.ResidualNormBwdParams.from_buffer_copy(norms._BWD.pack(1, 2) + bytes(p) + norms._BWD_TAIL.pack(*range(3, 14)))
    assert [getattr(b, f[0]) for f in b._fields_ if f[0] != "fwd"] == [1, 2, *range(3, 14)] and b.fwd.eps == 0.25
    q = _lib.LinearInt8Params.from_buffer_copy(int8._PARAMS.pack(*range(1, 21)))
    assert [getattr(q, f[0]) for f in q._fields_] == [*range(1, 21)]


def test_gate_rows():
    assert _gate_rows(torch.empty(8), (3, 5, 8)) == 15
    assert _gate_rows(torch.empty(1, 1, 8), (3, 5, 8)) == 15
    assert _gate_rows(torch.empty(3, 1, 8), (3, 5, 8)) == 5
    assert _gate_rows(torch.empty(3, 5, 8), (3, 5, 8)) == 1
    assert _gate_rows(torch.empty(1, 8), (1, 8)) == 1
    assert _gate_rows(torch.empty(5, 8), (3, 5, 8)) is None
    assert _gate_rows(torch.empty(3, 5, 1), (3, 5, 8)) is None


# ---- 8-bit linear layer ------------------------------------------------------------------------------------------------
def _linear(**kw):
    p = _lib.LinearInt8Params(C.sizeof(_lib.LinearInt8Params), _lib.FDB_INT8, P, 64, P, P, 64, P, P, P, 100, 64, 32, 0, 0, 0, 0, None, 0, None)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,code", [
    (dict(struct_bytes=0), -1), (dict(x_dtype=2), -1), (dict(out_dtype=4), -1), (dict(bias_dtype=2), -1), (dict(bias_dtype=3), -1),
    (dict(rows=-1), -1), (dict(in_features=0), -1), (dict(out_features=0), -1), (dict(in_features=131072, x_pitch=1 << 18, weight_pitch=1 << 18), -6),
    (dict(rows=1 << 31), -6), (dict(x=None), -1), (dict(x_scale=None), -1), (dict(weight=None), -1), (dict(weight_scale=None), -1), (dict(out=None), -1),
    (dict(x_pitch=48), -1), (dict(weight_pitch=48), -1), (dict(x_pitch=72), -3), (dict(weight_pitch=72), -3), (dict(x=P + 8), -3), (dict(weight=P + 8), -3),
    (dict(x_scale=P + 2), -3), (dict(weight_scale=P + 2), -3), (dict(out=P + 1), -3), (dict(bias=P + 1), -3), (dict(status=P + 2), -3),
    (dict(x_dtype=0), -4), (dict(x_dtype=0, workspace=P, workspace_bytes=64), -4), (dict(x_dtype=0, workspace=P + 16, workspace_bytes=1 << 20), -4),
    (dict(x_dtype=0, x=P + 1), -3),
])
def test_linear_int8_argument_errors(change, code):
    p = _linear(**change)
    _refused(_lib.load().fdb_linear_int8(C.byref(p), None), code)


def test_linear_int8_sizes():
    lib = _lib.load()
    p = _linear(rows=0)
    assert lib.fdb_linear_int8(C.byref(p), None) == 0
    assert lib.fdb_linear_int8_workspace_bytes(C.byref(_linear())) == 0
    p = _linear(x_dtype=_lib.FDB_FP32, in_features=33, x_pitch=0)
    assert lib.fdb_linear_int8_workspace_bytes(C.byref(p)) >= 100 * (48 + 4)
    p.rows = 4  # a few tokens are rounded by the one kernel there is
    assert lib.fdb_linear_int8_workspace_bytes(C.byref(p)) == 0


@pytest.mark.parametrize("args,code", [
    ((P, 4, 2, 8, P, 16, P), -1), ((P, 0, -1, 8, P, 16, P), -1), ((P, 0, 2, 0, P, 16, P), -1), ((P, 0, 2, 18, P, 16, P), -1), ((None, 0, 2, 8, P, 16, P), -1),
    ((P, 0, 2, 8, None, 16, P), -1), ((P, 0, 2, 8, P, 16, None), -1), ((P + 1, 0, 2, 8, P, 16, P), -3), ((P + 2, 1, 2, 8, P, 16, P), -3),
    ((P, 0, 2, 8, P, 16, P + 2), -3), ((P, 0, 2, 8, P + 8, 16, P), -3), ((P, 0, 2, 8, P, 24, P), -3), ((P, 0, 1 << 31, 8, P, 16, P), -6),
])
def test_quantize_int8_argument_errors(args, code):
    _refused(_lib.load().fdb_quantize_int8(*args, None), code)


@pytest.mark.parametrize("cols", [(1 << 30) + 1, (1 << 31) - 1])
def test_quantize_int8_refuses_rows_that_it_cannot_count(cols):
    """A 32-bit column counter would pass its end."""
    _refused(_lib.load().fdb_quantize_int8(P, 0, 1, cols, P, 1 << 31, P, None), -6)


def test_quantize_int8_without_rows_is_a_no_op():
    assert _lib.load().fdb_quantize_int8(None, 0, 0, 8, None, 8, None, None) == 0


def test_int8_rows_layout():
    a = torch.randint(-128, 128, (5, 33), dtype=torch.int8)
    b = int8_rows(a)
    assert torch.equal(a, b) and b.stride() == (48, 1) and int8_rows(b) is b
    assert _rows(torch.zeros(3, 4, 48, dtype=torch.int8)[..., :33])[1] == 48
    assert _rows(torch.zeros(3, 5, 48, dtype=torch.int8)[:, :4]) is None       # rows of two strides
    assert _rows(torch.zeros(64, 32, dtype=torch.int8).t()) is None
    assert _rows(torch.zeros(1, 7, dtype=torch.int8))[1] == 16                    # one row: any pitch will do
    with pytest.raises(TypeError):
        int8_rows(torch.zeros(2, 2))


@pytest.mark.parametrize("shape,expanded", [((1, 16), (8, 16)), ((1, 64), (32, 64)), ((4, 1, 48), (4, 3, 48)), ((4, 1, 64), (4, 8, 64)), ((1, 5, 32), (6, 5, 32)),
                                            ((2, 1, 3, 16), (2, 4, 3, 16)), ((1, 1, 16), (2, 3, 16)), ((5, 1), (5, 16))])
def test_expanded_rows_of_integers_are_copied(shape, expanded):
    """A row that stands for several is in memory once: taken as rows behind one another it would be read far past its end."""
    a = torch.randint(-128, 128, shape, dtype=torch.int8).expand(expanded)
    assert _rows(a) is None
    b = int8_rows(a)
    at, pitch = _rows(b)
    assert torch.equal(a, b) and pitch >= expanded[-1]
    end = b.untyped_storage().data_ptr() + b.untyped_storage().nbytes()
    assert at + (a.numel() // expanded[-1] - 1) * pitch + expanded[-1] <= end


# ---- gradients ---------------------------------------------------------------------------------------------------------
def _clip(entry=(P, P, 5, 0, 0), **kw):
    t = (_lib.GradTensor * 2)(_lib.GradTensor(P, P, 3, 1, 1), _lib.GradTensor(*entry))
    p = _lib.ClipGradsParams(C.sizeof(_lib.ClipGradsParams), 2, C.addressof(t), 2, 1, 1.0, P, P, 1 << 30)
    for k, v in kw.items():
        setattr(p, k, v)
    return p, t


@pytest.mark.parametrize("change,code", [
    (dict(struct_bytes=0), -1), (dict(n_tensors=-1), -1), (dict(tensors=None), -1), (dict(norm_type=3), -1), (dict(max_norm=-1.0), -1),
    (dict(max_norm=float("nan")), -1), (dict(norm=None), -1), (dict(norm=P + 2), -3), (dict(workspace=None), -4), (dict(workspace=P + 8), -4),
    (dict(workspace_bytes=4), -4), (dict(entry=(None, P, 5, 0, 0)), -1), (dict(entry=(P, None, 5, 0, 0)), -1), (dict(entry=(P, P, -1, 0, 0)), -1),
    (dict(entry=(P, P, 5, 2, 0)), -1), (dict(entry=(P, P + 64, 5, 0, 4)), -1), (dict(entry=(P, P, 5, 0, 1)), -1), (dict(entry=(P + 1, P, 5, 0, 0)), -3),
    (dict(entry=(P, P + 2, 5, 0, 1)), -3), (dict(entry=(P, P, 1 << 45, 0, 0)), -6),
])
def test_clip_grads_argument_errors(change, code):
    p, keep = _clip(**change)
    _refused(_lib.load().fdb_clip_grads(C.byref(p), None), code)


def test_runs_of_memory_that_overlap():
    assert _apart([]) and _apart([(0, 4)]) and _apart([(8, 12), (0, 8)]) and _apart([], [(0, 4), (2, 6)])
    assert not _apart([(0, 4), (0, 4)]) and not _apart([(0, 9), (8, 9)])
    writes = [(40, 50), (10, 20)]
    assert _apart(writes, [(0, 10), (20, 40), (50, 60), (25, 35), (5, 8)])
    for read in [(0, 11), (19, 30), (12, 13), (0, 100), (30, 41), (49, 60), (10, 20), (45, 46)]:
        assert not _apart(writes, [read]), read


def test_tensors_that_fill_their_memory():
    t = torch.zeros(3, 4, 5)
    assert _dense(t) and _dense(t.permute(2, 0, 1)) and _dense(t[1:2]) and _dense(t[:, :1].contiguous().transpose(0, 1)) and _dense(torch.zeros(()))
    assert not _dense(t[:, 1:]) and not _dense(t[..., ::2]) and not _dense(torch.zeros(1, 4).expand(3, 4))


def test_elements_in_one_place():
    m = torch.zeros(12, 35)
    apart = [[m[:, :10], m[:, 10:20], m[:, 20:]], [m[:, ::2], m[:, 1::2]], [m[::2], m[1::2]], [m[::3, 1::2], m[1::3], m[2::3, ::7], m[::3, ::2]],
             [m[:6], m[6:, :4], m[6:, 4:]], [m.t()[:7], m[:, 7:].t()], [m.view(-1)[::6], m.view(-1)[1::6], m.view(-1)[2::3]], [m[:, 34], m[:, 0]],
             [m.view(3, 4, 35)[:, 1:3, 5], m.view(3, 4, 35)[:, 1:3, 6:9], m.view(3, 4, 35)[:, ::3]], [m.bfloat16(), m[:, 1:]], []]
    for ts in apart:
        assert not _collide(ts, []) and not _collide(ts[:1], ts[1:]) and not _collide([], ts + ts)
    together = [[m[:, 1:], m[:, 1:]], [m[:, :10], m[:, 9:20]], [m[:, ::2], m[:, ::3]], [m[:6, 1:], m[5:, ::2]], [m, m[3, 5:6]], [m[::2, :4], m.t()[3]],
                [m.view(-1)[::6], m.view(-1)[::4]], [m[:, 1:], m.view(torch.bfloat16)[7:9, 4:5]]]
    for a, b in together:
        assert _collide([a, b], []) and _collide([b], [a]) and _collide([a], [b]) and _collide([m.clone()[:, 2:], b, a], []) and not _collide([], [a, b])
    for t in (m[:1].expand(4, 35), m.view(-1).as_strided((5, 4), (3, 1)), m[:, :1].expand(12, 3)):
        assert _collide([t], []) and not _collide([], [t]) and not _collide([m.clone()], [t])
    for t in (m.as_strided((5, 4), (2, 3)), m.as_strided((3, 2), (2, 3))):  # 2 i + 3 j: twice six, or never twice
        places = {2 * i + 3 * j for i in range(t.shape[0]) for j in range(t.shape[1])}
        assert _collide([t], []) == (len(places) < t.numel())
    assert _collide([m.as_strided((5, 4), (2, 3))], []) and not _collide([m.as_strided((3, 2), (2, 3))], [])


def test_elements_that_stand_for_many_are_not_counted_out():
    m = torch.zeros(40)
    many = m[3:4].expand(10 ** 6, 10 ** 6)
    assert _collide([many], []) and _collide([m[::3]], [many]) and not _collide([m[::2]], [many])


def test_elements_in_one_place_against_a_list_of_them():
    gen = torch.Generator().manual_seed(0)
    pick = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=gen))
    base, seen = torch.zeros(400), set()
    for _ in range(400):
        views = []
        for _ in range(pick(1, 4)):
            shape = [pick(1, 5) for _ in range(pick(1, 4))]
            views.append(base.as_strided(shape, [pick(0 if pick(0, 6) == 0 else 1, 24) for _ in shape], pick(0, 60)))
        places = [torch.arange(400).as_strided(v.shape, v.stride(), v.storage_offset()).flatten().tolist() for v in views]
        cut = pick(1, len(views) + 1)
        written = sum(places[:cut], [])
        want = len(set(written)) < len(written) or bool(set(written) & set(sum(places[cut:], [])))
        assert _collide(views[:cut], views[cut:]) == want, [(v.shape, v.stride(), v.storage_offset()) for v in views]
        seen.add(want)
    assert seen == {True, False}


# ---- the Python layer ----------------------------------------------------------------------------------------------------
def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 8), torch.ones(8)
    for call in (lambda: ops.residual_norm(x, x, w, w), lambda: ops.quantize_int8(x), lambda: ops.grad_norm([x]), lambda: ops.clip_grads_([x], 1.0),
                 lambda: ops.linear_int8(x, torch.zeros(4, 8, dtype=torch.int8), torch.ones(4))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_forward_mode_derivatives_are_refused():
    import torch.autograd.forward_ad as fwd
    x = torch.ones(3)
    ops.refuse_tangents("it", (x, None))
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones(3))
        ops.refuse_tangents("it", (x, None))
        for bad in ((dual,), (None, x, dual)):
            with pytest.raises(RuntimeError, match="it has no forward-mode"):
                ops.refuse_tangents("it", bad)
    ops.refuse_tangents("it", (dual,))  # (the tangent ended with its level)
    with pytest.raises(RuntimeError, match="no forward-mode"):
        torch.func.jvp(lambda v: ops.refuse_tangents("it", (v,)) or v, (x,), (x,))


def test_empty_lists_of_gradients():
    assert ops.grad_norm([]).item() == 0.0 and ops.clip_grads_([], 1.0).item() == 0.0
    assert ops.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0).item() == 0.0  # no gradient there
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            ops.clip_grads_([], bad)
    with pytest.raises(ValueError):
        ops.grad_norm([], 3.0)
