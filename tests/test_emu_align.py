"""Host-emulation (CPU) runs of the alignment operators: index math, masks, refusals."""
import pytest
import torch

import align_cases as A
from emu_lib import emu_lib
from pcm_amd import capi


@pytest.fixture(autouse=True, params=["bf16", "f16"])
def _use_emu(request):
    """the formats are named per call: both builds of the library give the same results"""
    capi.set_lib(emu_lib(request.param))
    yield
    capi.set_lib(None)


@pytest.mark.parametrize("P,n,kw", [(1, 1, {}), (1, 3, dict(kind="square")), (2, 64, dict(eps=0.1, weighted=True)), (3, 255, dict(kind="hinge")),
                                    (2, 1023, dict(dtype="bf16", weighted=True)), (1, 2049, dict(dtype="f16", grad_scale=64.0)),
                                    (2, 1500, dict(reduce="sum", eps=0.2)), (1, 4100, dict(kind="square", dtype="bf16")), (2, 9000, dict(weighted=True, eps=0.1)), (1, 20001, dict(dtype="f16")), (40, 500, dict(kind="hinge"))])
def test_denoise_preference(P, n, kw):
    A.case_denoise_preference("cpu", P, n, **kw)


@pytest.mark.parametrize("P,T,kw", [(1, 1, {}), (1, 2, dict(kind="square")), (3, 63, dict(eps=0.1, masked=True)), (2, 65, dict(ragged=True, reduce="mean")),
                                    (3, 257, dict(masked=True, ragged=True, pad=3, dtype="bf16")), (2, 130, dict(dtype="f16", pad=8, masked=True, u8=True)),
                                    (1, 600, dict(kind="hinge", ragged=True, i64=True)), (4, 5, dict(masked=True, ragged=True, reduce="mean", pad=1)),
                                    (2500, 2, dict(masked=True)), (3, 11000, dict(masked=True, ragged=True))])
def test_preference(P, T, kw):
    A.case_preference("cpu", P, T, **kw)


@pytest.mark.parametrize("N,T,kw", [(1, 1, {}), (8, 4, dict(kl=0.04)), (3, 65, dict(masked=True, kl=0.1, reduce="row")), (5, 33, dict(ragged=True, per_step=True)),
                                    (4, 130, dict(masked=True, ragged=True, pad=5, dtype="bf16", kl=0.04)), (3, 77, dict(dtype="f16", reduce="sum", pad=8)),
                                    (2, 40, dict(with_old=False, kl=0.2)), (3, 17, dict(with_ref=True, i64=True, ragged=True, reduce="row")),
                                    (7, 1, dict(per_step=True, spread=3.0, kl=0.01)), (2, 300, dict(clip=(0.0, 0.0))),
                                    (3, 6000, dict(masked=True, ragged=True, kl=0.1)), (30, 600, dict(masked=True, reduce="row", kl=0.1, pad=1)),
                                    (4, 5000, dict(masked=True, reduce="row")), (6000, 3, dict(kl=0.1, ragged=True, masked=True)), (5000, 4, dict(reduce="row", masked=True)),
                                    (2100, 2, dict(per_step=True, pad=2)), (40, 500, dict(clip=(0.9, float("inf")), kl=0.1, spread=1.0))])
def test_policy(N, T, kw):
    A.case_policy("cpu", N, T, **kw)


def test_policy_where_nothing_counts():
    from pcm_amd import ops
    lp = torch.full((3, 9), float("nan"))
    for reduce in ("token", "row", "sum"):
        loss, grad, stats = ops.policy_loss(lp, torch.ones(3), old_logp=lp, ref_logp=lp, mask=torch.zeros(3, 9, dtype=torch.bool), kl_coef=0.1, reduce=reduce)
        assert loss.item() == 0.0 and not grad.any() and not stats.any()
        loss, grad, stats = ops.policy_loss(lp, torch.ones(3), old_logp=lp, lengths=torch.tensor([0, -3, 0]), reduce=reduce)
        assert loss.item() == 0.0 and not grad.any() and not stats.any()


@pytest.mark.parametrize("B,n,kw", [(1, 1, {}), (3, 63, dict(reduce="sum")), (2, 1025, dict(dtype="bf16")), (2, 700, dict(dtype="f16")), (1, 5000, {}), (1, 70001, {}), (40, 1500, dict(dtype="bf16"))])
def test_transition(B, n, kw):
    A.case_transition("cpu", B, n, **kw)


@pytest.mark.parametrize("kw", [{}, dict(max_norm=1e9), dict(where="apart"), dict(where="flat"), dict(where="apart", dtypes=("bf16", "f16"), out_dtypes=("f32",)),
                                dict(where="flat", dtypes=("f32",), out_dtypes=("bf16", "f16", "f32")), dict(sizes=[1], max_norm=1e-3), dict(scale=0.0)])
def test_clip(kw):
    A.case_clip("cpu", **kw)


def test_policy_run():
    A.case_policy_run("cpu")


@pytest.mark.slow
def test_preference_step():
    from pcm_amd import precision
    if capi.lib().act_dtype == 0:            # (the network's buffers are in the process's one 16-bit format, bfloat16)
        assert precision.precision() == "bf16"
        A.case_preference_step("cpu")


def test_deterministic():
    A.case_deterministic("cpu")


def test_not_a_number():
    A.case_not_a_number("cpu")


def test_without_gradient():
    A.case_without_gradient("cpu")


def test_infinite_margins():
    A.case_infinite_margins("cpu")


def test_refusals():
    A.case_refusals("cpu")


def test_dense_orders():
    A.case_dense_orders("cpu")


def test_separated_pairs():
    A.case_separated_pairs("cpu")


def test_far_reference():
    A.case_far_reference("cpu")


def test_monitored_kl():
    A.case_monitored_kl("cpu")


def test_zero_advantage():
    A.case_zero_advantage("cpu")


def test_student_near_base():
    A.case_student_near_base("cpu")


def test_lowest_reference():
    A.case_lowest_reference("cpu")


def test_launches_of_the_preference_loss():
    """a call launches what it needs: few elements one kernel; partial sums and gradient two; the loss of many pairs two of its own, and then none for a
    gradient that is not asked for"""
    import ctypes
    from pcm_amd import ops
    count = capi.lib().dll.pcm_emu_launches
    count.restype, count.argtypes = ctypes.c_long, []
    for P, T, want_grad, launches in ((4, 50, True, 1), (4, 50, False, 1), (100, 400, True, 2), (100, 400, False, 2), (2500, 2, True, 4), (2500, 2, False, 3)):
        lp = -torch.rand(2 * P, T)
        before = count()
        ops.preference_loss(lp, torch.zeros_like(lp), want_grad=want_grad)
        assert count() - before == launches, (P, T, want_grad)


def test_too_many_rows():
    A.case_too_many_rows("cpu")


def test_transition_scales():
    A.case_transition_scales("cpu")


def test_sampler_transition():
    A.case_sampler_transition("cpu")


def test_without_gradient_16bit():
    A.case_without_gradient_16bit("cpu")
