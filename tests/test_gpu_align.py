"""The alignment operators on the MI355X: parity with the 64-bit implementations at real sizes, hipGraph capture, streams."""
import pytest
import torch

import align_cases as A

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _product():
    from pcm_amd import capi
    assert torch.cuda.is_available()
    capi.set_lib(None)
    assert capi.lib().path == capi.DEFAULT_LIB
    yield
    torch.cuda.synchronize()


@pytest.mark.parametrize("P,n,kw", [(1, 1, {}), (1, 3, dict(kind="square")), (3, 255, dict(kind="hinge")), (1, 16384, {}), (24, 16384, dict(eps=0.1, weighted=True)),
                                    (5, 4 * 97 * 61, dict(dtype="bf16", weighted=True)), (2, 65536, dict(dtype="f16", grad_scale=64.0)),
                                    (3, 32769, dict(reduce="sum", eps=0.2)), (2, 262144, dict(kind="square")), (300, 1027, {}), (2, 40001, dict(dtype="bf16")),
                                    (257, 20001, dict(dtype="bf16"))])
def test_denoise_preference(P, n, kw):
    A.case_denoise_preference("cuda", P, n, **kw)


@pytest.mark.parametrize("P,T,kw", [(1, 1, {}), (1, 2, dict(kind="square")), (3, 63, dict(eps=0.1, masked=True)), (4, 50, {}), (300, 1, {}),
                                    (3, 257, dict(masked=True, ragged=True, pad=3, dtype="bf16")), (2, 4099, dict(dtype="f16", pad=8, masked=True, u8=True)),
                                    (1, 32768, dict(kind="hinge", ragged=True, i64=True)), (9, 1024, dict(masked=True, ragged=True, reduce="mean", pad=1)),
                                    (1, 70001, dict(masked=True, beta=0.1)), (2, 40000, dict(dtype="bf16", ragged=True)), (700, 40, dict(masked=True)),
                                    (2500, 2, dict(masked=True)), (20000, 1, dict(kind="square")), (3000, 1500, dict(dtype="bf16"))])
def test_preference(P, T, kw):
    A.case_preference("cuda", P, T, **kw)


@pytest.mark.parametrize("N,T,kw", [(1, 1, {}), (8, 4, dict(kl=0.04)), (3, 65, dict(masked=True, kl=0.1, reduce="row")), (5, 33, dict(ragged=True, per_step=True)),
                                    (64, 1027, dict(masked=True, ragged=True, pad=5, dtype="bf16", kl=0.04)), (33, 777, dict(dtype="f16", reduce="sum", pad=8)),
                                    (2, 40, dict(with_old=False, kl=0.2)), (30, 1700, dict(with_ref=True, i64=True, ragged=True, reduce="row")),
                                    (5000, 1, dict(per_step=True, spread=3.0, kl=0.01)), (2, 300, dict(clip=(0.0, 0.0))), (5000, 7, dict(ragged=True, masked=True, reduce="row")),
                                    (40, 500, dict(clip=(0.9, float("inf")), kl=0.1, spread=1.0)), (600, 5000, dict(reduce="row", masked=True, kl=0.1, pad=3)),
                                    (4, 50001, dict(reduce="row", masked=True, ragged=True)), (1, 20000, dict(reduce="row", masked=True, kl=0.1)), (2, 3000, dict(grad_scale=3.3e4, dtype="f16")), (9000, 3, dict(reduce="row", masked=True)), (9000, 2, dict(per_step=True, pad=2, dtype="bf16")),
                                    (6000, 100, dict(ragged=True, i64=True)), (512, 2048, dict(kl=0.04)), (1, 100003, dict(masked=True, kl=0.04, per_step=True))])
def test_policy(N, T, kw):
    A.case_policy("cuda", N, T, **kw)


@pytest.mark.parametrize("B,n,kw", [(1, 1, {}), (3, 63, dict(reduce="sum")), (16, 16384, {}), (2, 23668, dict(dtype="bf16")), (700, 1001, dict(dtype="f16")),
                                    (2, 262144, dict(reduce="sum")), (1, 1048583, {})])
def test_transition(B, n, kw):
    A.case_transition("cuda", B, n, **kw)


@pytest.mark.parametrize("kw", [{}, dict(max_norm=1e9), dict(where="apart"), dict(where="flat"), dict(where="apart", dtypes=("bf16", "f16"), out_dtypes=("f32",)),
                                dict(where="flat", dtypes=("f32",), out_dtypes=("bf16", "f16", "f32")), dict(sizes=[1], max_norm=1e-3), dict(scale=0.0),
                                dict(sizes=[3000001, 5, 700000] + [321] * 600, where="flat"), dict(sizes=[64 * 320] * 300, dtypes=("f32",))])
def test_clip(kw):
    A.case_clip("cuda", **kw)


def test_policy_run():
    A.case_policy_run("cuda")
    A.case_policy_run("cuda", B=5, steps=8, n=256, seed=1)


def test_preference_step():
    A.case_preference_step("cuda", hw=16)


def test_deterministic():
    A.case_deterministic("cuda", big=True)


def test_not_a_number():
    A.case_not_a_number("cuda")


def test_without_gradient():
    A.case_without_gradient("cuda")


def test_infinite_margins():
    A.case_infinite_margins("cuda")


def test_separated_pairs():
    A.case_separated_pairs("cuda")


def test_far_reference():
    A.case_far_reference("cuda")


def test_monitored_kl():
    A.case_monitored_kl("cuda")


def test_zero_advantage():
    A.case_zero_advantage("cuda")


def test_student_near_base():
    A.case_student_near_base("cuda")


def test_lowest_reference():
    A.case_lowest_reference("cuda")


def test_too_many_rows():
    A.case_too_many_rows("cuda")


def test_transition_scales():
    A.case_transition_scales("cuda")


def test_sampler_transition():
    A.case_sampler_transition("cuda")


def test_without_gradient_16bit():
    A.case_without_gradient_16bit("cuda")


def test_refusals():
    A.case_refusals("cuda")
    from pcm_amd import ops
    x = torch.zeros(4, 6)
    for call in (lambda: ops.preference_loss(x, x), lambda: ops.preference_loss(x.cuda(), x), lambda: ops.GradSet([x]), lambda: ops.GradSet([x.cuda()], out=[x]),
                 lambda: ops.policy_loss(x.cuda(), torch.ones(4)), lambda: ops.transition_logprob(x, x, torch.ones(4))):
        with pytest.raises(ValueError):
            call()


def test_dense_orders():
    A.case_dense_orders("cuda")


class _Everything:
    """one pass of every operator over buffers that stay where they are, so that it can be captured"""

    def __init__(self, seed, P=6, n=20000, N=40, T=333):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.shapes = dict(t=(2 * P, n), r=(2 * P, n), p=(2 * P, n), lp=(N, T), old=(N, T), ref=(N, T), adv=(N,), g0=(70000,), g1=(33,))
        self.buf = {k: torch.empty(s, device="cuda") for k, s in self.shapes.items()}
        self.mask = torch.rand(N, T, device="cuda", generator=g) < 0.8
        self.std = torch.full((2 * P,), 0.7, device="cuda")
        self.out = [torch.empty_like(self.buf["g0"]), torch.empty_like(self.buf["g1"])]
        from pcm_amd import ops
        self.ops, self.set = ops, ops.GradSet([self.buf["g0"], self.buf["g1"]], out=self.out)
        self.fill(seed)

    def fill(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        for k, s in self.shapes.items():
            self.buf[k].copy_(torch.randn(s, device="cuda", generator=g) * (0.2 if k in ("lp", "old", "ref") else 1.0))

    def run(self):
        b, ops = self.buf, self.ops
        res = list(ops.denoise_preference_loss(b["p"], b["r"], b["t"], beta=10.0))
        res += ops.preference_loss(b["lp"], b["ref"], mask=self.mask)
        res += ops.policy_loss(b["lp"], b["adv"], old_logp=b["old"], ref_logp=b["ref"], mask=self.mask, kl_coef=0.05)
        logp = ops.transition_logprob(b["p"], b["t"], self.std)
        res += [logp, ops.transition_logprob_bwd(b["p"], b["t"], self.std, logp), self.set.clip(1.0)]
        return res + self.out


def test_captured_and_replayed():
    """two graphs of all operators, replayed in turn and side by side with eager work between: every replay has the eager call's bits"""
    from pcm_amd import ops  # noqa: F401
    runs, graphs, outs = [_Everything(1), _Everything(2)], [], []
    for e in runs:
        e.run()
    torch.cuda.synchronize()
    for e in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(e.run())
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for i, e in enumerate(runs):
            e.fill(10 * rep + i)
        torch.cuda.synchronize()
        if rep < 2:
            for g in graphs:
                g.replay()
        else:
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for i, e in enumerate(runs):
            for a, b in zip(got[i], e.run()):
                assert torch.equal(a, b), (rep, i)


def test_on_another_stream():
    """the operators run on the current stream, after the work that is queued there"""
    e = _Everything(3)
    want = [t.clone() for t in e.run()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for k in e.buf:
        e.buf[k].zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        e.fill(3)
        got = e.run()
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", ["bf16", "f16"])
def test_both_builds_give_the_same_bits(fmt):
    from pcm_amd import capi
    e = _Everything(4)
    want = [t.clone() for t in e.run()]
    capi.set_lib(capi.Lib(capi.DEFAULT_LIB if fmt == "bf16" else capi.F16_LIB))
    for a, b in zip(e.run(), want):
        assert torch.equal(a, b)


def test_offsets_past_32_bits():
    """rows whose elements lie past 2^31: a column slice of rows that are far apart, at both ends of the buffer"""
    from pcm_amd import ops
    far = (1 << 31) + 5
    wide = torch.zeros(far + 4096, device="cuda", dtype=torch.bfloat16)
    lp = wide.as_strided((2, 1000), (far, 1))
    lp.copy_(-torch.rand(2, 1000, device="cuda"))
    ref = (lp + 0.1).contiguous()
    loss, grad, ratio = ops.preference_loss(lp, ref)
    want = (lp.double() - ref.double()).sum(1)
    A.close(ratio, want.cpu(), (20 * A.U * want.abs()).cpu(), "log ratios")
    _, grad, stats = ops.policy_loss(lp, torch.ones(2, device="cuda"), old_logp=ref)
    assert stats[3].item() == 2000 and grad.abs().sum().item() > 0
    big = wide[:far]
    big.fill_(2.0 ** -15)
    norm = ops.GradSet([big]).clip(1e-9)
    A.close(norm, torch.tensor([2.0 ** -15 * far ** 0.5], dtype=torch.float64), 2 * A.U, "norm")
    f = 1e-9 / (2.0 ** -15 * far ** 0.5 + 1e-6) * 2.0 ** -15
    for t in (big[:9], big[far // 2:far // 2 + 9], big[-9:]):
        A.close(t, torch.full((9,), f, dtype=torch.float64), f * 2.0 ** -8, "clipped")
