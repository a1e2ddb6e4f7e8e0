"""Refusals of the operators that apply decoded weights, without a GPU: the C ABI looks at its arguments before it touches a
device, and the Python side before it calls."""
import copy
import ctypes as C
import pickle

import pytest
import torch

import ptwm_b200
from ptwm_b200 import _lib, operators
from ptwm_b200.operators import scaled_names

INVALID, SMALL, UNSUPPORTED = -1, -2, -5
A = 1 << 20  # an aligned address nobody reads


@pytest.fixture(scope="module")
def L():
    ptwm_b200.build()
    return _lib.lib()


def _weight(**over):
    a = dict(values=A, scales=A, global_scale=0, rows=64, cols=64, value_pitch=32, scale_pitch=16, group=32, reserved=0)
    a.update(over)
    return _lib.ScaledWeightArgs(**a)


@pytest.mark.parametrize("over, rc", [
    (dict(values=0), INVALID), (dict(scales=0), INVALID), (dict(group=8), INVALID), (dict(rows=0), INVALID), (dict(cols=0), INVALID), (dict(cols=48), INVALID),
    (dict(value_pitch=24), INVALID), (dict(values=A + 8), INVALID), (dict(scales=A + 4), INVALID), (dict(scale_pitch=8), INVALID), (dict(value_pitch=16), INVALID),
    (dict(cols=1024, value_pitch=512), INVALID), (dict(rows=(1 << 30) + 1), UNSUPPORTED)])
def test_matrices_that_are_none(L, over, rc):
    w = _weight(**over)
    assert L.ptwm_b200_matvec(C.addressof(w), A, 0, A, 1, 6, 0, 6, 0, 0, 0, 1) == rc
    assert L.ptwm_b200_matvec_grad(C.addressof(w), A, A, 1, 6, 0, 0, 0, 1) == rc
    assert _lib.last_error().startswith("scaled weight")


def test_tokens_that_are_none(L):
    w = _weight()
    p = C.addressof(w)
    nv = _weight(cols=48, group=16, value_pitch=32)
    for args, rc in [((p, A, 0, A, 1, 6, 0, 13), UNSUPPORTED), ((p, A, 0, A, 1, 13, 0, 6), UNSUPPORTED), ((p, A, A, A, 1, 6, 1, 6), UNSUPPORTED), ((p, A, 0, A, 1, 29, 1, 6), INVALID),
                     ((p, A, A, A, 1, 29, 0, 6), UNSUPPORTED), ((p, A, A, A, 1, 29, 3, 6), UNSUPPORTED), ((p, 0, 0, A, 1, 6, 0, 6), INVALID), ((p, A, 0, 0, 1, 6, 0, 6), INVALID),
                     ((p, A, 0, A, (1 << 19) + 1, 6, 0, 6), UNSUPPORTED), ((C.addressof(nv), A, A, A, 1, 29, 2, 6), INVALID), ((None, A, 0, A, 1, 6, 0, 6), INVALID)]:
        assert L.ptwm_b200_matvec(*args, 0, 0, 0, 1) == rc, args
    other = _weight(cols=96, value_pitch=48)
    refs, ys = (C.c_uint64 * 5)(p, C.addressof(other), p, p, p), (C.c_uint64 * 5)(A, A, 0, A, A)
    for count, at, rc in [(0, ys, INVALID), (2, ys, INVALID), (5, ys, UNSUPPORTED), (1, None, INVALID)]:
        assert L.ptwm_b200_matvec_group(refs, at, count, A, 0, 1, 6, 0, 6, 0, 0, 0, 1) == rc, count
    refs[1] = p
    assert L.ptwm_b200_matvec_group(refs, ys, 3, A, 0, 1, 6, 0, 6, 0, 0, 0, 1) == INVALID
    assert L.ptwm_b200_matvec(p, 0, 0, 0, 0, 6, 0, 6, 0, 0, 0, 1) == 0  # no tokens: nothing to do, on any machine
    assert L.ptwm_b200_matvec(p, 0, 0, 0, 0, 29, 2, 6, 0, 0, 0, 1) == 0
    for args, rc in [((p, A, A, 1, 29), UNSUPPORTED), ((p, 0, A, 1, 6), INVALID), ((p, A, 0, 1, 6), INVALID)]:
        assert L.ptwm_b200_matvec_grad(*args, 0, 0, 0, 1) == rc, args


def test_norms_that_are_none(L):
    for args, rc in [((A, 0, A, 0, A, 0, 4, 64, 29, 6, 0), UNSUPPORTED), ((A, 0, A, 0, A, 0, 4, 64, 6, 13, 0), UNSUPPORTED), ((A, 0, A, 0, A, A, 4, 64, 6, 6, 3), INVALID),
                     ((A, 0, A, 0, A, 0, 4, 0, 6, 6, 0), INVALID), ((A, 0, A, 0, A, A, 4, 48, 6, 6, 2), INVALID), ((0, 0, A, 0, A, 0, 4, 64, 6, 6, 0), INVALID),
                     ((A, 0, 0, 0, A, 0, 4, 64, 6, 6, 0), INVALID), ((A, 0, A, 0, 0, 0, 4, 64, 6, 6, 0), INVALID), ((A, A, A, 0, A, 0, 4, 64, 6, 6, 0), INVALID),
                     ((A, 0, A, 0, A, 0, 4, 64, 6, 6, 1), INVALID), ((A, 0, A, 0, A, 0, 1 << 31, 64, 6, 6, 0), UNSUPPORTED)]:
        assert L.ptwm_b200_rms_norm(*args, 1e-6, 0, 1) == rc, args
    assert L.ptwm_b200_rms_norm(0, 0, 0, 0, 0, 0, 0, 64, 6, 6, 0, 1e-6, 0, 1) == 0
    need = L.ptwm_b200_rms_norm_grad_scratch_bytes(1000, 64)
    assert need >= 64 * 4
    for args, rc in [((A, A, A, 0, A, 0, 0, 0, 4, 64, 29, 6), UNSUPPORTED), ((A, A, A, 0, 0, 0, 0, 0, 4, 64, 6, 6), INVALID), ((A, A, 0, 0, A, 0, 0, 0, 4, 64, 6, 6), INVALID),
                     ((A, A, A, 0, A, A, 0, 0, 1000, 64, 6, 6), SMALL), ((A, A, A, 0, A, A, A, need - 1, 1000, 64, 6, 6), SMALL), ((A, A, A, 0, A, 0, 0, 0, 4, 0, 6, 6), UNSUPPORTED)]:
        assert L.ptwm_b200_rms_norm_grad(*args, 1e-6, 0, 1) == rc, args


def test_addresses_that_no_value_of_the_type_has(L):
    w = _weight()
    p = C.addressof(w)
    for args in [(A + 1, 0, A, 0, A, 0, 4, 64, 6, 6, 0), (A + 2, 0, A, 0, A, 0, 4, 64, 1, 6, 0), (A, A + 1, A, A, A, 0, 4, 64, 6, 6, 0), (A, A, A, A + 1, A, 0, 4, 64, 6, 6, 0),
                 (A, 0, A + 2, 0, A, 0, 4, 64, 6, 1, 0), (A, 0, A, 0, A + 1, 0, 4, 64, 4, 6, 0), (A, 0, A, 0, A, A + 2, 4, 64, 6, 6, 1)]:
        assert L.ptwm_b200_rms_norm(*args, 1e-6, 0, 1) == INVALID, args
    need = L.ptwm_b200_rms_norm_grad_scratch_bytes(4, 64)
    for args in [(A, A, A + 1, 0, A, 0, 0, 0, 4, 64, 6, 6), (A, A, A, A + 1, A, 0, 0, 0, 4, 64, 6, 6), (A, A, A, 0, A, A + 2, A, need, 4, 64, 6, 1), (A, A, A, 0, A, A, A + 2, need, 4, 64, 6, 6)]:
        assert L.ptwm_b200_rms_norm_grad(*args, 1e-6, 0, 1) == INVALID, args
    for args in [(p, A + 1, 0, A, 1, 6, 0, 6), (p, A, 0, A + 2, 1, 6, 0, 1), (p, A, A + 2, A, 1, 29, 1, 6)]:
        assert L.ptwm_b200_matvec(*args, 0, 0, 0, 1) == INVALID, args
    for args in [(p, A + 1, A, 1, 6), (p, A, A + 2, 1, 1)]:
        assert L.ptwm_b200_matvec_grad(*args, 0, 0, 0, 1) == INVALID, args


def test_tensors_in_host_memory_are_refused():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="host memory"):
        ptwm_b200.rms_norm(x, torch.ones(64))
    with pytest.raises(ValueError, match="host memory"):
        ptwm_b200.ScaledWeight(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))
    with pytest.raises(ValueError, match="host memory"):
        ptwm_b200.ScaledActivations(x.to(torch.float8_e4m3fn), torch.zeros(2))
    with pytest.raises(TypeError, match="ScaledWeight"):
        ptwm_b200.matvec(x, torch.zeros(4, 32, dtype=torch.uint8))
    with pytest.raises(TypeError, match="tensor"):
        ptwm_b200.rms_norm([1.0], torch.ones(1))


def test_names_of_a_microscaled_matrix():
    def of(*names):
        return set(names).__contains__
    assert scaled_names("a", of("a.weight", "a.weight_scale", "a.weight_scale_2")) == ("a.weight", "a.weight_scale", "a.weight_scale_2")
    assert scaled_names("a", of("a.weight", "a.weight_scale")) == ("a.weight", "a.weight_scale", None)
    assert scaled_names("a", of("a_blocks", "a_scales", "a_bias")) == ("a_blocks", "a_scales", None)
    assert scaled_names("a", of("a", "a_scale", "a_scale_2")) == ("a", "a_scale", "a_scale_2")
    with pytest.raises(KeyError):
        scaled_names("a", of("a", "a_blocks", "b_scale"))


def test_gradients_of_two_types_that_are_none(L):
    p = C.addressof(_weight())
    for args, rc in [((p, A, A, 1, 29, 6), UNSUPPORTED), ((p, A, A, 1, 6, 29), UNSUPPORTED), ((p, A + 2, A, 1, 1, 6), INVALID), ((p, A, A + 2, 1, 6, 1), INVALID), ((p, 0, A, 1, 1, 6), INVALID),
                     ((p, A, 0, 1, 1, 6), INVALID), ((p, A, A, (1 << 19) + 1, 1, 6), UNSUPPORTED), ((None, A, A, 1, 1, 6), INVALID)]:
        assert L.ptwm_b200_matvec_grad_of(*args, 0, 0, 0, 1) == rc, args
    assert L.ptwm_b200_matvec_grad_of(p, 0, 0, 0, 1, 6, 0, 0, 0, 1) == 0


def _host_tensors(monkeypatch):
    """Handles on host memory, which nothing may be launched with."""
    monkeypatch.setattr(operators, "_on_cuda", lambda what, t, device=None: None)


def _own_addresses(w):
    assert w._ref == C.addressof(w._args)
    assert w._args.values == w._values.data_ptr() and w._args.scales == w._scales.data_ptr() and w._args.global_scale == (0 if w._global is None else w._global.data_ptr())


@pytest.mark.parametrize("kind", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("how", [copy.copy, copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o))])
def test_copies_of_handles_have_addresses_of_their_own(monkeypatch, kind, how):
    _host_tensors(monkeypatch)
    values = torch.arange(64 * 128, dtype=torch.int32).to(torch.uint8).reshape(64, 128)
    if kind == "mxfp4":
        w = ptwm_b200.ScaledWeight(values, torch.full((64, 16), 127, dtype=torch.uint8)[:, :8])
    else:
        w = ptwm_b200.ScaledWeight(values, torch.ones(64, 16).to(torch.float8_e4m3fn), torch.tensor([0.5]))
    _own_addresses(w)
    c = how(w)
    _own_addresses(c)
    assert c._ref != w._ref and (how is copy.copy or c._values.data_ptr() != w._values.data_ptr())
    assert c.kind == kind and c.shape == w.shape and torch.equal(c._values, w._values) and torch.equal(c._scales, w._scales)
    for field in ("rows", "cols", "value_pitch", "scale_pitch", "group"):
        assert getattr(c._args, field) == getattr(w._args, field)
    p = ptwm_b200.Projection(torch.ones(256), [w, w, c, w, c], eps=1e-3, quant="row")
    q = how(p)
    assert (q.eps, q.quant, len(q.weights)) == (1e-3, "row", 5) and torch.equal(q.norm, p.norm)
    refs = [r for call, _ in q._calls for r in call]
    assert refs == [m._ref for m in q.weights] and [len(ws) for _, ws in q._calls] == [4, 1]
    for m in q.weights:
        _own_addresses(m)
    assert how is copy.copy or not set(refs) & {w._ref, c._ref}


@pytest.mark.parametrize("cols, group, tokens, dtype, parts", [(954436352, 32, 2, 4, 2), (613565952, 16, 3, 4, 2), (858992640, 16, 1, 1, 3), (66587648, 32, 16, 1, 3)])
def test_rows_far_too_long_for_shared_memory_go_to_tiles(L, cols, group, tokens, dtype, parts):
    """What few tokens of such rows would want passes 2^32 bytes by a little: they are laid out for the kernel of many tokens instead."""
    pitch = (cols // group + 15) // 16 * 16
    w = _weight(rows=1, cols=cols, value_pitch=cols // 2, scale_pitch=pitch, group=group)
    assert L.ptwm_b200_matvec_scratch_bytes(C.addressof(w), A, tokens, dtype, 0) == parts * tokens * cols * 2


@pytest.mark.parametrize("cols", [(1 << 30) + 1, (1 << 31) - 8, (1 << 31) - 1])
def test_norms_of_rows_that_32_bits_do_not_count(L, cols):
    for quant in (0, 1):
        assert L.ptwm_b200_rms_norm(A, 0, A, 0, A, A, 1, cols, 6, 6, quant, 1e-6, 0, 1) == UNSUPPORTED
    assert L.ptwm_b200_rms_norm_grad(A, A, A, 0, A, 0, 0, 0, 1, cols, 6, 6, 1e-6, 0, 1) == UNSUPPORTED


def test_scratch_is_looked_at_before_any_launch(L):
    """A few rows of 8192 columns want none for 12 tokens, many do: a call for both says so before it touches the device."""
    few, many = _weight(rows=16, cols=8192, value_pitch=4096, scale_pitch=256), _weight(rows=14336, cols=8192, value_pitch=4096, scale_pitch=256)
    assert L.ptwm_b200_matvec_scratch_bytes(C.addressof(few), A, 12, 4, 0) == 0
    need = L.ptwm_b200_matvec_scratch_bytes(C.addressof(many), A, 12, 4, 0)
    assert need == 2 * 12 * 8192 * 2
    refs, ys = (C.c_uint64 * 2)(C.addressof(few), C.addressof(many)), (C.c_uint64 * 2)(A, A)
    for scratch, size, rc in [(0, 0, SMALL), (0, need, SMALL), (A, need - 1, SMALL), (A + 8, need, INVALID)]:
        assert L.ptwm_b200_matvec_group(refs, ys, 2, A, 0, 12, 4, 0, 4, scratch, size, 0, 1) == rc
    assert L.ptwm_b200_matvec(C.addressof(many), A, 0, A, 12, 4, 0, 4, 0, 0, 0, 1) == SMALL


def test_a_projection_keeps_its_norm_and_matrices(monkeypatch):
    _host_tensors(monkeypatch)
    given = [ptwm_b200.ScaledWeight(torch.zeros(n, 128, dtype=torch.uint8), torch.zeros(n, 16, dtype=torch.uint8)[:, :8]) for n in (16, 32)]
    p = ptwm_b200.Projection(torch.ones(256), given)
    kept = list(given)
    given.append(given[0])
    assert list(p.weights) == kept and not hasattr(p.weights, "append")
    for name, value in (("weights", given), ("norm", torch.ones(512))):
        with pytest.raises(AttributeError):
            setattr(p, name, value)
    assert [r for call, _ in p._calls for r in call] == [w._ref for w in p.weights]


def test_the_status_of_a_device_that_is_none(L):
    if torch.cuda.is_available():
        pytest.skip("there are devices")
    with pytest.raises(ptwm_b200.PtwmError):
        ptwm_b200.operator_status(0)
    with pytest.raises(ptwm_b200.PtwmError):
        ptwm_b200.operator_status("cuda:1")


def test_only_cuda_devices_have_a_status():
    with pytest.raises(ValueError, match="cpu"):
        ptwm_b200.operator_status("cpu")
