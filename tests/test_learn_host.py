"""The boundary of include/omk_learn.h without a GPU: what the library exports, and every refusal that its checks of arguments make
before anything is enqueued (the handle of these tests names no device: a call that got past its checks would have to
ask for one)."""
import ctypes as C
import math
import os
import re
import subprocess

import numpy as np
import pytest

from omoknuni_small_amd import learn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, CAPACITY, UNSUPPORTED = -1, -3, -5


def test_header_library_and_mirror_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "omk_learn.h")).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(omk_[a-z0-9_]+)\s*\(", text)))
    lib = learn._library()
    assert declared == sorted(learn.EXPORTS) == sorted(learn._ARGTYPES)
    for name in declared:
        assert hasattr(lib, name)


def test_header_is_c(tmp_path):
    """Both headers as C, and the structures as the mirror lays them out."""
    structs = [("omk_policy_rows", learn._Rows), ("omk_policy_samples", learn._Samples), ("omk_policy_loss_params", learn._PolicyParams),
               ("omk_policy_loss_out", learn._PolicyOut), ("omk_preference_params", learn._PreferenceParams),
               ("omk_preference_out", learn._PreferenceOut), ("omk_adamw_tensor", learn._AdamTensor), ("omk_adamw_desc", learn._AdamDesc)]
    lines = ["#include <stddef.h>", '#include "omk_learn.h"']
    for name, mirror in structs:
        names = [f[0] for f in mirror._fields_]
        lines.append("_Static_assert(sizeof(%s) == %d, \"%s\");" % (name, C.sizeof(mirror), name))
        lines += ["_Static_assert(offsetof(%s, %s) == %d, \"%s.%s\");" % (name, f, getattr(mirror, f).offset, name, f) for f in names]
    source = tmp_path / "header.c"
    source.write_text("\n".join(lines) + "\nint main(void) { return 0; }\n")
    subprocess.check_call(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(source)])


@pytest.fixture
def handle():
    # a learner as its calls see one, on device -1: zeroed memory with the ordinal in front
    return C.cast(C.create_string_buffer(b"\xff\xff\xff\xff" + bytes(252), 256), C.c_void_p)


def address(n):  # of no memory: a refused call reads nothing
    return 0x1000000 + 0x1000000 * n


def rows(**change):
    r = dict(d_logits=address(0), row_stride=225, rows=8, actions=225, type=1, d_legal=address(1), legal_stride=8)
    r.update(change)
    return learn._Rows(**r)


BAD_ROWS = [
    dict(type=3), dict(type=-1), dict(type=7), dict(rows=-1), dict(rows=1 << 31), dict(actions=0), dict(actions=-5),
    dict(actions=(1 << 24) + 1), dict(row_stride=224), dict(row_stride=-225), dict(legal_stride=7), dict(legal_stride=-8),
    dict(d_logits=None), dict(d_logits=address(0) + 1), dict(d_legal=address(1) + 2), dict(type=0, d_logits=address(0) + 2),
    dict(row_stride=1 << 61), dict(legal_stride=1 << 60),
]


def message():
    return learn._library().omk_last_error().decode()


@pytest.mark.parametrize("change", BAD_ROWS, ids=str)
def test_rows_are_refused(handle, change):
    lib, r = learn._library(), rows(**change)
    out = learn._PolicyOut(address(2), address(3), 225, address(4), None)
    samples = learn._Samples(*[address(5 + i) for i in range(5)])
    params = learn._PolicyParams(0.2, 0.2, 0.1, 1.0)
    pout = learn._PreferenceOut(address(2), address(3), 225, None, None, 0)
    pparams = learn._PreferenceParams(0.1, 0.0, 1.0)
    assert lib.omk_policy_priors(handle, C.byref(r), address(3), 225, None, 0) == INVALID
    assert message().startswith("omk_policy_priors: ")
    assert lib.omk_policy_logprobs(handle, C.byref(r), address(5), address(2), None, None, 0) == INVALID
    assert lib.omk_policy_loss(handle, C.byref(r), C.byref(samples), C.byref(params), C.byref(out), address(11), 1 << 20) == INVALID
    assert lib.omk_preference_loss(handle, C.byref(r), address(5), address(6), 2, None, C.byref(pparams), C.byref(pout),
                                   address(11), 1 << 20) == INVALID
    assert message().startswith("omk_preference_loss: ")


def policy(handle, samples=(), params=(), out=(), work=1 << 20, d_work=address(11), r=None):
    s = dict(d_moves=address(5), d_old_logprob=address(6), d_advantage=address(7), d_ref_logprob=address(8), d_weight=None)
    p = dict(clip_low=0.2, clip_high=0.2, kl_weight=0.1, scale=1.0)
    o = dict(d_loss=address(2), d_grad=address(3), grad_stride=225, d_logprob=address(4), d_kl=None)
    s.update(samples), p.update(params), o.update(out)
    r = r or rows()
    return learn._library().omk_policy_loss(handle, C.byref(r), C.byref(learn._Samples(**s)), C.byref(learn._PolicyParams(**p)),
                                            C.byref(learn._PolicyOut(**o)), d_work, work)


def test_policy_loss_refuses(handle):
    nan, inf = math.nan, math.inf
    for change in (dict(clip_low=-0.1), dict(clip_low=nan), dict(clip_high=-1.0), dict(clip_high=inf), dict(clip_high=nan),
                   dict(kl_weight=-1.0), dict(kl_weight=inf), dict(scale=nan), dict(scale=-inf)):
        assert policy(handle, params=change) == INVALID, change
    for change in (dict(d_moves=None), dict(d_old_logprob=None), dict(d_advantage=None), dict(d_ref_logprob=None),
                   dict(d_moves=address(5) + 2), dict(d_weight=address(9) + 1)):
        assert policy(handle, samples=change) == INVALID, change
    for change in (dict(d_loss=None), dict(d_logprob=None), dict(grad_stride=224), dict(d_grad=address(3) + 1),
                   dict(d_kl=address(8) + 2), dict(grad_stride=1 << 61),
                   dict(d_grad=address(0) + 2), dict(d_grad=address(0), grad_stride=226)):
        assert policy(handle, out=change) == INVALID, change
    for n in (5, 6, 7, 8):
        assert policy(handle, out=dict(d_logprob=address(n) + 4 * 7)) == INVALID and "across" in message()
        assert policy(handle, out=dict(d_kl=address(n) - 4 * 7)) == INVALID and "across" in message()
    needed = learn._library().omk_policy_loss_work(8, 225)
    assert needed > 0
    assert policy(handle, work=needed - 1) == CAPACITY
    assert policy(handle, d_work=None) == CAPACITY
    assert policy(handle, d_work=address(11) + 8) == INVALID
    assert policy(None) == INVALID


def test_priors_may_not_lie_across_the_logits(handle):
    lib, r = learn._library(), rows(type=0)
    for at in (address(0), address(0) + 4 * 225 * 8 - 4, address(0) - 4 * 225 * 8 + 4):
        assert lib.omk_policy_priors(handle, C.byref(r), at, 225, None, 0) == INVALID and "across" in message()


def test_wide_rows_need_work_space(handle):
    lib = learn._library()
    assert lib.omk_policy_work(100, 65528) == 0 and lib.omk_policy_work(0, 1 << 20) == 0
    needed = lib.omk_policy_work(8, 100000)
    assert needed > 0
    r = rows(actions=100000, row_stride=100000, d_legal=None)
    for d_work, n in ((None, needed), (address(11), needed - 1)):
        assert lib.omk_policy_priors(handle, C.byref(r), address(3), 100000, d_work, n) == CAPACITY
        assert lib.omk_policy_logprobs(handle, C.byref(r), address(5), address(2), None, d_work, n) == CAPACITY
    assert lib.omk_policy_priors(handle, C.byref(r), address(3), 100000, address(11) + 4, needed) == INVALID


def preference(handle, params=(), out=(), pairs=3, work=1 << 20, d_moves=address(5), d_begin=address(6), d_work=address(11)):
    p = dict(beta=0.1, label_smoothing=0.1, scale=1.0)
    o = dict(d_loss=address(2), d_grad=address(3), grad_stride=225, d_margin=None, d_line_logprob=None, zero_rest=0)
    p.update(params), o.update(out)
    r = rows()
    return learn._library().omk_preference_loss(handle, C.byref(r), d_moves, d_begin, pairs, None,
                                                C.byref(learn._PreferenceParams(**p)), C.byref(learn._PreferenceOut(**o)),
                                                d_work, work)


def test_preference_loss_refuses(handle):
    nan = math.nan
    for change in (dict(beta=nan), dict(beta=math.inf), dict(label_smoothing=-0.1), dict(label_smoothing=0.6),
                   dict(label_smoothing=nan), dict(scale=nan)):
        assert preference(handle, params=change) == INVALID, change
    for change in (dict(d_loss=None), dict(grad_stride=3), dict(d_grad=address(0) + 4), dict(d_margin=address(8) + 1)):
        assert preference(handle, out=change) == INVALID, change
    for change in (dict(d_margin=address(6) + 4), dict(d_line_logprob=address(6) + 24), dict(d_margin=address(6) - 8)):
        assert preference(handle, out=change) == INVALID and "across" in message(), change
    assert preference(handle, pairs=-1) == INVALID
    assert preference(handle, pairs=(1 << 23) + 1) == INVALID
    assert preference(handle, d_moves=None) == INVALID
    assert preference(handle, d_begin=None) == INVALID
    assert preference(handle, d_begin=address(6) + 1) == INVALID
    needed = learn._library().omk_preference_loss_work(8, 225, 3)
    assert preference(handle, work=needed - 1) == CAPACITY


def adamw(handle, tensor=(), **desc):
    t = dict(n=300, d_param=address(0), d_copy=None, d_m=address(1), d_v=address(2), d_m_scale=address(3),
             d_v_scale=address(4), lr_scale=1.0, weight_decay=0.0)
    t.update(tensor)
    tensors = (learn._AdamTensor * 1)(learn._AdamTensor(**t))
    d = dict(n_tensors=1, h_tensors=tensors, param_type=0, grad_type=0, copy_type=-1, state_type=0, beta1=0.9, beta2=0.999,
             eps=1e-8, seed=1)
    d.update(desc)
    got = C.c_void_p()
    rc = learn._library().omk_adamw_create(handle, C.byref(learn._AdamDesc(**d)), C.byref(got))
    assert not got
    return rc


def test_adamw_refuses(handle):
    for change in (dict(n=-1), dict(n=(1 << 40) + 1), dict(d_param=None), dict(d_m=None), dict(d_v=None),
                   dict(d_param=address(0) + 2), dict(d_m=address(1) + 1), dict(lr_scale=math.nan), dict(weight_decay=math.inf),
                   dict(d_copy=address(9))):
        assert adamw(handle, tensor=change) == INVALID, change
    for change in (dict(n_tensors=-1), dict(h_tensors=None), dict(param_type=3), dict(grad_type=-1), dict(copy_type=0),
                   dict(copy_type=3), dict(state_type=1), dict(state_type=-1), dict(beta1=1.0), dict(beta1=-0.1),
                   dict(beta2=math.nan), dict(eps=-1.0), dict(eps=math.nan), dict(eps=1e-40), dict(eps=1e39), dict(copy_type=1)):
        assert adamw(handle, **change) == INVALID, change
    for change in (dict(d_m_scale=None), dict(d_v_scale=None), dict(d_v_scale=address(4) + 2)):
        assert adamw(handle, tensor=change, state_type=3) == INVALID, change
    for change in (dict(d_m=address(0) + 4 * 299), dict(d_v=address(1)), dict(d_v=address(1) - 4 * 299)):
        assert adamw(handle, tensor=change) == INVALID and "overlap" in message(), change
    assert adamw(handle, tensor=dict(d_v_scale=address(3) + 4), state_type=3) == INVALID and "overlap" in message()
    assert adamw(handle, param_type=1, grad_type=2) == UNSUPPORTED
    assert adamw(handle, tensor=dict(d_copy=address(9)), param_type=1, grad_type=1, copy_type=1) == UNSUPPORTED
    assert adamw(None) == INVALID
    assert learn._library().omk_adamw_step(None, None, 0.1, None, None) == INVALID
    assert learn._library().omk_adamw_set_steps(None, 1) == INVALID


def test_a_learner_needs_a_device():
    lib, got = learn._library(), C.c_void_p()
    assert lib.omk_learner_create(1 << 20, C.byref(got)) in (INVALID, -2) and not got
    assert lib.omk_learner_create(0, None) == INVALID
    assert lib.omk_learner_set_stream(None, None) == INVALID
    assert lib.omk_learner_destroy(None) == 0 and lib.omk_adamw_destroy(None) == 0


def test_torch_without_a_gpu_is_named():
    import torch

    import omoknuni_small_amd as omk
    if torch.cuda.is_available():
        pytest.skip("a GPU is here")
    with pytest.raises(OSError, match="import torch before"):
        omk.Learner()


def test_masks_of_move_lists():
    begin, moves = [0, 3, 3, 6], [0, 31, 224, 32, -1, 300]
    mask = learn.legal_of_moves(begin, moves, 225)
    assert mask.shape == (3, 8) and mask.dtype == np.uint32
    bits = np.unpackbits(mask.view(np.uint8), axis=1, bitorder="little")
    assert [np.nonzero(b)[0].tolist() for b in bits] == [[0, 31, 224], [], [32]]


def test_pack_legal_on_the_host():
    torch = pytest.importorskip("torch")
    mask = torch.rand(5, 3, 70, generator=torch.Generator().manual_seed(1)) < 0.5
    packed = learn.pack_legal(mask)
    assert packed.shape == (5, 3, 3) and packed.dtype == torch.int32
    bits = np.unpackbits(packed.numpy().view(np.uint8), axis=-1, bitorder="little")[..., :70]
    assert (bits == mask.numpy()).all()
