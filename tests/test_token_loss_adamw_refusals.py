"""CPU checks of the token losses and AdamW: what the C entry points and their Python callers refuse before any
launch.  Pointers are numbers that nothing reads."""
import ctypes as C

import pytest
import torch

from renaissance_b200 import _lib, ops

A, B, D, E = 0x10000, 0x20000, 0x40000000, 0x50000000


@pytest.fixture(scope="module")
def lib():
    from renaissance_b200 import build
    build.build()
    return _lib.load()


def logp(lib, z=A, stride=16, labels=B, out=B, lse=None, rows=4, classes=16, dtype=0):
    return lib.trb200_token_logp(z, stride, labels, out, lse, rows, classes, dtype, None)


def policy(lib, z=A, stride=16, y=B, old=B, ref=None, adv=B, w=None, sc=B, lo=0.2, hi=0.2, kl=0.0, d=D, dstride=16,
           lp=B, part=B, loss=B, rows=4, classes=16, dtype=1):
    return lib.trb200_policy_loss_fused(z, stride, y, old, ref, adv, w, sc, lo, hi, kl, d, dstride, lp, part, loss, rows,
                                        classes, dtype, None)


def preference(lib, z=A, stride=16, y=B, starts=B, ref=None, sc=B, beta=0.1, eps=0.0, d=D, dstride=16, lp=B, seq=B,
               part=B, loss=B, rows=4, pairs=1, classes=16, dtype=2, ws=E, ws_bytes=None):
    if ws_bytes is None:
        ws_bytes = lib.trb200_preference_loss_workspace_bytes(rows)
    return lib.trb200_preference_loss_fused(z, stride, y, starts, ref, sc, beta, eps, d, dstride, lp, seq, part, loss,
                                            rows, pairs, classes, dtype, ws, ws_bytes, None)


@pytest.mark.parametrize("bad", [dict(z=None), dict(labels=None), dict(out=None), dict(rows=-1), dict(classes=0),
                                 dict(stride=15), dict(dtype=3), dict(dtype=-1), dict(z=A + 1), dict(z=A + 2, dtype=2)])
def test_token_logp_refuses(lib, bad):
    assert logp(lib, **bad) == _lib.ERR_INVALID_ARGUMENT
    assert b"token_logp" in lib.trb200_last_error()


def test_too_many_rows_or_classes_are_unsupported(lib):
    assert logp(lib, stride=1 << 31, classes=(1 << 30) + 1) == _lib.ERR_UNSUPPORTED
    assert logp(lib, rows=(1 << 30) + 1) == _lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("bad", [dict(z=None), dict(y=None), dict(old=None), dict(adv=None), dict(sc=None), dict(d=None),
                                 dict(lp=None), dict(part=None), dict(loss=None), dict(rows=-1), dict(classes=0),
                                 dict(stride=15), dict(dstride=15), dict(dtype=3), dict(d=D + 1), dict(kl=0.1),
                                 dict(kl=float("nan"), ref=B), dict(lo=-0.1), dict(lo=1.5), dict(hi=-1.0),
                                 dict(lo=float("nan")), dict(hi=float("nan")),
                                 dict(d=A), dict(d=A + 32), dict(d=A + 2 * 16 * 3 + 30), dict(d=A - 2)])
def test_policy_loss_refuses(lib, bad):
    assert policy(lib, **bad) == _lib.ERR_INVALID_ARGUMENT
    assert b"policy_loss" in lib.trb200_last_error()


@pytest.mark.parametrize("bad", [dict(z=None), dict(y=None), dict(starts=None), dict(sc=None), dict(d=None), dict(lp=None),
                                 dict(seq=None), dict(part=None), dict(loss=None), dict(rows=-1), dict(pairs=0),
                                 dict(pairs=-1), dict(pairs=1 << 30), dict(beta=float("inf")), dict(beta=float("nan")),
                                 dict(eps=-0.1), dict(eps=1.1), dict(eps=float("nan")), dict(d=A), dict(dtype=7)])
def test_preference_loss_refuses(lib, bad):
    assert preference(lib, **bad) == _lib.ERR_INVALID_ARGUMENT
    assert b"preference_loss" in lib.trb200_last_error()


def test_preference_loss_needs_its_workspace(lib):
    assert lib.trb200_preference_loss_workspace_bytes(0) == 0
    assert lib.trb200_preference_loss_workspace_bytes(1000) >= 12000
    assert preference(lib, ws=None) == _lib.ERR_WORKSPACE
    assert preference(lib, ws_bytes=lib.trb200_preference_loss_workspace_bytes(4) - 1) == _lib.ERR_WORKSPACE
    assert preference(lib, ws=E + 4) == _lib.ERR_WORKSPACE


@pytest.mark.parametrize("off", [1, 2, 3])
def test_arrays_of_four_byte_elements_have_to_be_aligned(lib, off):
    """A misaligned address would end in a fault of the GPU: refused before any launch."""
    calls = ((logp, "token_logp", ("labels", "out", "lse")),
             (policy, "policy_loss", ("y", "old", "ref", "adv", "w", "sc", "lp", "part", "loss")),
             (preference, "preference_loss", ("y", "starts", "ref", "sc", "lp", "seq", "part", "loss")))
    for call, name, fields in calls:
        for field in fields:
            assert call(lib, **{field: B + off}) == _lib.ERR_INVALID_ARGUMENT, field
            assert name.encode() in lib.trb200_last_error() and b"aligned" in lib.trb200_last_error(), field


# ------------------------------------------------------------------------------------------------ AdamW

def tensor(n=1000, at=0x100000, **kw):
    t = _lib.AdamWTensor(at, at + 0x100000, at + 0x200000, at + 0x300000, at + 0x400000, at + 0x500000, at + 0x600000, n, 0.1)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def write(lib, tensors, grad=2, copy=-1, bits=32, short=0, null_image=False):
    table = (_lib.AdamWTensor * max(1, len(tensors)))(*tensors)
    size = lib.trb200_adamw_plan_bytes(table, len(tensors))
    image = (C.c_char * max(1, size))()
    desc = _lib.AdamWPlanDesc()
    rc = lib.trb200_adamw_plan_write(table, len(tensors), grad, copy, bits, None if null_image else C.addressof(image),
                                     size - short, C.byref(desc))
    return rc, desc


def test_adamw_plan_counts_its_units(lib):
    rc, desc = write(lib, [tensor(1), tensor(0, 0x1100000), tensor(4097, 0x2100000)], copy=0, bits=8)
    assert rc == 0
    assert (desc.count, desc.units, desc.grad_dtype, desc.copy_dtype, desc.state_bits) == (3, 1 + 0 + 17, 2, 0, 8)
    assert write(lib, [])[0] == 0


@pytest.mark.parametrize("kw", [dict(grad=3), dict(grad=-1), dict(copy=2), dict(copy=-2), dict(bits=16), dict(null_image=True)])
def test_adamw_plan_refuses_kinds(lib, kw):
    assert write(lib, [tensor()], **kw)[0] == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("field", ["w", "g", "m", "v", "m_scale", "v_scale", "copy"])
def test_adamw_plan_refuses_null_and_misaligned(lib, field):
    assert write(lib, [tensor(**{field: None})], copy=0, bits=8)[0] == _lib.ERR_INVALID_ARGUMENT
    odd = {"m": 0, "v": 0}.get(field, 1)        # 8-bit states have no alignment
    if odd:
        assert write(lib, [tensor(**{field: 0x900001})], copy=0, bits=8)[0] == _lib.ERR_INVALID_ARGUMENT
    else:
        assert write(lib, [tensor(**{field: 0x900001})], copy=0, bits=8)[0] == 0
        assert write(lib, [tensor(**{field: 0x900001})])[0] == _lib.ERR_INVALID_ARGUMENT
    assert write(lib, [tensor(n=0, **{field: None})], copy=0, bits=8)[0] == 0       # nothing is read from an empty tensor


def test_adamw_plan_refuses_overlaps(lib):
    a = tensor()
    assert write(lib, [a, tensor()])[0] == _lib.ERR_INVALID_ARGUMENT                      # listed twice
    assert b"overlaps" in lib.trb200_last_error()
    assert write(lib, [a, tensor(at=0x2000000, w=a.w + 4 * 999)])[0] == _lib.ERR_INVALID_ARGUMENT
    assert write(lib, [a, tensor(at=0x2000000, w=a.w + 4 * 1000)])[0] == 0                # right behind
    assert write(lib, [a, tensor(at=0x2000000, v=a.m)])[0] == _lib.ERR_INVALID_ARGUMENT
    assert write(lib, [a, tensor(at=0x2000000, g=a.g)])[0] == 0                           # gradients may be shared
    assert write(lib, [tensor(g=a.w)])[0] == _lib.ERR_INVALID_ARGUMENT                    # a gradient that is a weight
    assert write(lib, [tensor(m_scale=a.v_scale)], bits=8)[0] == _lib.ERR_INVALID_ARGUMENT
    assert write(lib, [tensor(copy=a.w + 4 * 999)], copy=1)[0] == _lib.ERR_INVALID_ARGUMENT


def test_adamw_plan_refuses_sizes(lib):
    table = (_lib.AdamWTensor * 1)(tensor(n=-1))
    assert lib.trb200_adamw_plan_bytes(table, 1) == 0
    assert lib.trb200_adamw_plan_bytes(None, 1) == 0 and lib.trb200_adamw_plan_bytes(table, -1) == 0
    assert write(lib, [tensor()], short=1)[0] == _lib.ERR_WORKSPACE
    assert write(lib, [tensor(weight_decay=float("nan"))])[0] == _lib.ERR_INVALID_ARGUMENT
    assert write(lib, [tensor(weight_decay=-1.0)])[0] == _lib.ERR_INVALID_ARGUMENT


def test_adamw_step_refuses(lib):
    rc, good = write(lib, [tensor()])
    assert rc == 0
    good.image = 0x700000

    def step(plan=good, step=B, lr=0.1, b1=0.9, b2=0.99, eps=1e-8):
        return lib.trb200_adamw_step(C.byref(plan) if plan is not None else None, step, lr, None, b1, b2, eps, None, None, 0, None)

    assert step(plan=None) == _lib.ERR_INVALID_ARGUMENT
    for kw in (dict(step=None), dict(lr=float("inf")), dict(b1=1.0), dict(b1=-0.1), dict(b2=1.0), dict(b2=float("nan")),
               dict(eps=0.0), dict(eps=-1.0), dict(eps=float("nan"))):
        assert step(**kw) == _lib.ERR_INVALID_ARGUMENT, kw
    for field, value in (("image", None), ("image", 0x700008), ("count", -1), ("units", -1), ("grad_dtype", 5),
                         ("copy_dtype", 2), ("state_bits", 0)):
        bad = _lib.AdamWPlanDesc.from_buffer_copy(good)
        setattr(bad, field, value)
        assert step(plan=bad) == _lib.ERR_INVALID_ARGUMENT, field


@pytest.mark.parametrize("bits,power", [(32, -55), (8, -53)])
@pytest.mark.parametrize("beta2", [0.0, 0.99, 0.999, 0.999999])
def test_adamw_step_refuses_an_eps_below_what_v_holds(lib, bits, power, beta2):
    """Accepted values reach the next check (a misaligned image) and no launch."""
    rc, plan = write(lib, [tensor()], bits=bits)
    assert rc == 0
    plan.image = 0x700008
    least = 2.0 ** power / (1 - beta2) ** 0.5

    def step(eps):
        rc = lib.trb200_adamw_step(C.byref(plan), B, 0.1, None, 0.9, beta2, eps, None, None, 0, None)
        assert rc == _lib.ERR_INVALID_ARGUMENT
        return lib.trb200_last_error()

    for eps in (least * 0.99, least / 10, 1e-30, 1.2e-38, 1e-45, 0.0, -least * 2, float("nan"), float("inf"), 1e38):
        assert b"eps" in step(eps), eps
    for eps in (least * 1.01, 1e-8, 1.0, 8e37):
        assert b"image" in step(eps), eps


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("field", range(4))
def test_adamw_step_refuses_misaligned_scalars(lib, field, off):
    rc, plan = write(lib, [tensor()])
    assert rc == 0
    plan.image = 0x700000
    step, lr, scaling, skip = ((B + off if i == field else B) for i in range(4))
    assert lib.trb200_adamw_step(C.byref(plan), step, 0.1, lr, 0.9, 0.999, 1e-8, scaling, skip, 0, None) == _lib.ERR_INVALID_ARGUMENT
    assert b"aligned to 4 bytes" in lib.trb200_last_error()


# ------------------------------------------------------------------------------------------------ Python callers

def test_python_callers_refuse_cpu_tensors_and_shapes():
    z = torch.zeros(4, 16)
    y = torch.zeros(4, dtype=torch.int32)
    f = torch.zeros(4)
    with pytest.raises(TypeError):
        ops.token_logprobs(z, y)
    with pytest.raises(TypeError):
        ops.policy_loss_fused(z, y, f, f, f[:1])
    with pytest.raises(TypeError):
        ops.preference_loss_fused(z, y, torch.zeros(3, dtype=torch.int32), None, f[:1])
    with pytest.raises(TypeError):
        ops.AdamWPlan([f], [f], [f], [f])
    with pytest.raises(ValueError):
        ops.AdamWPlan([], [], [], [])
    with pytest.raises(ValueError):
        ops.AdamWPlan([f], [f], [f], [f], m_scales=[f])
    with pytest.raises(ValueError):
        ops.AdamWPlan([f], [f, f], [f], [f])
    with pytest.raises(ValueError):
        ops.AdamWPlan([f], [f], [f], [f], weight_decay=[0.1, 0.2])
    with pytest.raises(TypeError):
        ops.adamw_step(None, y, 0.1)
