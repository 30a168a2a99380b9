"""Parity cases of the alignment operators (pcm_amd.ops: preference losses, clipped policy loss, transition log-probability, GradSet) against plain
64-bit implementations on the CPU; run by test_emu_align.py (host emulation) and test_gpu_align.py (MI355X).

Tolerances come from the arithmetic: u = 2^-24 is half a step of fp32, H(dtype) half a step of the output's format.  Elements are formed in fp32 and
summed in fp64 (at most eight of them are added in fp32 first)."""
import math

import pytest
import torch

from pcm_amd import ops

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def close(got, want, tol, what):
    """|got - want| <= tol elementwise; NaNs and infinities have to agree"""
    got, want = got.detach().double().cpu(), want.double().cpu()
    tol = tol if isinstance(tol, torch.Tensor) else torch.full_like(want, float(tol))
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol.cpu()))
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], tol[bad][:4])


def out_tol(want, tol, dtype):
    """fp32 error ``tol`` plus the rounding to the output's format (relative half step; absolute half step of its subnormals)"""
    tol = tol + U * want.abs() + 2.0 ** -149
    if dtype != torch.float32:
        tol = tol + half_step(dtype) * (want.abs() + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return tol


# ---- plain implementations ----
def pair_ref(ratio, P, beta, kind, eps):
    h = ratio[:P] - ratio[P:]
    if kind == "sigmoid":
        s = beta * h
        loss = -(1 - eps) * torch.nn.functional.logsigmoid(s) - eps * torch.nn.functional.logsigmoid(-s)
        slope = beta * (eps * torch.sigmoid(s) - (1 - eps) * torch.sigmoid(-s))
        curve = torch.full_like(s, beta * beta / 4)
    elif kind == "hinge":
        loss, slope, curve = (1 - beta * h).clamp(min=0), torch.where(beta * h < 1, -beta, 0.0).double(), torch.zeros_like(h)
    else:
        loss, slope, curve = (h - 0.5 / beta) ** 2, 2 * (h - 0.5 / beta), torch.full_like(h, 2.0)
    return loss, torch.cat([slope, -slope]) / P, torch.cat([curve, curve]) / P, slope.abs()


def check_pair(out, ratio, drho, beta, kind, eps, P, grad, dgrad_by_rho, grad_tol, dtype):
    """loss, log ratios and gradient of a pair loss: ``drho`` bounds the error of the log ratios before their rounding, ``grad`` = d ratio / d input,
    ``grad_tol`` the relative error of the gradient apart from that of the slope"""
    loss, slope, curve, steep = pair_ref(ratio, P, beta, kind, eps)
    close(out[2], ratio, drho + U * ratio.abs(), "log ratios")
    dh = drho[:P] + drho[P:]
    dh = torch.cat([dh, dh])
    # fp64 evaluation of the pair's loss adds nothing that counts; its slope times the error of the margin does
    close(out[0], loss.mean().reshape(1), (steep * dh[:P]).mean() + curve[:P].max() * P * (dh ** 2).max() + 2 * U * loss.mean().abs(), "loss")
    want = slope[:, None] * dgrad_by_rho
    if grad is not None:
        tol = (curve * dh)[:, None] * dgrad_by_rho.abs() + grad_tol * want.abs()
        close(grad, want, out_tol(want, tol, dtype), "gradient")


def case_denoise_preference(device, P, n, dtype="f32", kind="sigmoid", eps=0.0, weighted=False, reduce="mean", beta=None, grad_scale=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    beta = beta if beta is not None else {"sigmoid": 200.0, "hinge": 200.0, "square": 2.0}[kind] / (n if reduce == "sum" else 1)
    t = torch.randn(2 * P, n, generator=g)
    r = t + 0.3 * torch.randn(2 * P, n, generator=g)
    p = r + 0.05 * torch.randn(2 * P, n, generator=g)
    t, r, p = t.to(dt), r.to(dt), p.to(dt)
    w = torch.rand(2 * P, generator=g) + 0.5 if weighted else None
    out = ops.denoise_preference_loss(p.to(device), r.to(device), t.to(device), weight=w.to(device) if weighted else None, beta=beta, kind=kind,
                                      label_smoothing=eps, reduce=reduce, grad_scale=grad_scale)
    a, b = t.double() - p.double(), t.double() - r.double()
    k = (w.double() if weighted else torch.ones(2 * P, dtype=torch.float64)) / (n if reduce == "mean" else 1)
    ratio = -k * (a * a - b * b).sum(1)
    # a and b carry one rounding, their squares three, the difference one more; up to eight fp32 additions
    drho = 12 * U * k * (a * a + b * b).sum(1)
    assert out[1].dtype == dt and out[1].shape == p.shape
    check_pair(out, ratio, drho, beta, kind, eps, P, out[1], 2 * grad_scale * k[:, None] * a, 3 * U, dt)
    if kind == "sigmoid" and n <= 64:      # the formula's gradient against differences of the formula itself
        def f(pp):
            rho = -k * ((t.double() - pp) ** 2 - b * b).sum(1)
            return pair_ref(rho, P, beta, kind, eps)[0].mean()
        q, h = p.double(), 1e-6
        for i in (0, P * n, 2 * P * n - 1):
            e = torch.zeros(2 * P * n, dtype=torch.float64)
            e[i] = h
            e = e.view(2 * P, n)
            fd = ((f(q + e) - f(q - e)) / (2 * h) * grad_scale).item()
            assert abs(out[1].double().cpu().flatten()[i].item() - fd) <= 1e-4 * abs(fd) + half_step(dt) * abs(fd) * 2 + 1e-9, (i, fd)


def draw_places(R, T, g, masked, ragged, i64=False):
    mask = lengths = None
    where = torch.ones(R, T, dtype=torch.bool)
    if masked:
        mask = torch.rand(R, T, generator=g) < 0.7
        mask[R // 2] = False                     # a row whose mask leaves nothing
        where &= mask
    if ragged:
        lengths = (torch.rand(R, generator=g) * (T + 1)).long().clamp(max=T)
        lengths[0] = T
        if R > 2:
            lengths[1], lengths[2] = 0, T + 5     # no places; a length beyond the row counts as the row
        lengths = lengths if i64 else lengths.int()
        where &= torch.arange(T)[None] < lengths[:, None]
    return mask, lengths, where


def spoil(t, where):
    """what stands in places that do not count: NaN, infinities and the format's lowest value in turn"""
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(t.dtype).min], dtype=t.dtype)
    fill = bad[torch.arange(t.numel()).view(t.shape) % 4]
    return torch.where(where, t, fill)


def rows_apart(t, device, pad):
    """the tensor on the device as a view of rows ``pad`` elements longer, the gaps holding NaN"""
    if not pad:
        return t.to(device)
    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan") if t.is_floating_point() else 1, device=device).to(t.dtype)
    wide[:, 1:1 + t.shape[1]] = t.to(device)
    return wide[:, 1:1 + t.shape[1]]


def case_preference(device, P, T, dtype="f32", kind="sigmoid", eps=0.0, masked=False, ragged=False, reduce="sum", pad=0, beta=0.5, grad_scale=1.0,
                    i64=False, u8=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    mask, lengths, where = draw_places(2 * P, T, g, masked, ragged, i64)
    lp = -4 * torch.rand(2 * P, T, generator=g)
    rf = (lp + torch.randn(2 * P, T, generator=g) / math.sqrt(T)).to(dt)
    lp = lp.to(dt)
    dmask = None if mask is None else rows_apart(mask.to(torch.uint8) * 7 if u8 else mask, device, pad)
    out = ops.preference_loss(rows_apart(spoil(lp, where), device, pad), rows_apart(spoil(rf, where), device, 2 * pad), mask=dmask,
                              lengths=None if lengths is None else lengths.to(device), beta=beta, kind=kind, label_smoothing=eps, reduce=reduce,
                              grad_scale=grad_scale)
    gap = torch.where(where, lp.double() - rf.double(), 0.0)
    share = 1.0 / where.sum(1).clamp(min=1).double() if reduce == "mean" else torch.ones(2 * P, dtype=torch.float64)
    ratio = gap.sum(1) * share
    drho = 9 * U * gap.abs().sum(1) * share              # one rounding of each difference, up to eight fp32 additions
    assert out[1].dtype == dt and out[1].shape == lp.shape
    check_pair(out, ratio, drho, beta, kind, eps, P, out[1], grad_scale * share[:, None] * where.double(), 2 * U, dt)
    assert not out[1].cpu()[~where].any(), "gradient outside the places that count"


def case_policy(device, N, T, dtype="f32", masked=False, ragged=False, per_step=False, kl=0.0, with_ref=None, with_old=True, reduce="token", pad=0,
                clip=(0.2, 0.28), grad_scale=1.0, spread=0.3, i64=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    mask, lengths, where = draw_places(N, T, g, masked, ragged, i64)
    lp = -4 * torch.rand(N, T, generator=g)
    old = (lp + spread * torch.randn(N, T, generator=g)).to(dt)
    ref = (lp + spread * torch.randn(N, T, generator=g)).to(dt)
    lp = lp.to(dt)
    adv = torch.randn(N, T, generator=g) if per_step else torch.randn(N, generator=g)
    adv.view(-1)[0] = 0.0
    with_ref = kl != 0.0 if with_ref is None else with_ref

    def put(t):
        return rows_apart(spoil(t, where), device, pad)
    out = ops.policy_loss(put(lp), put(adv) if per_step else adv.to(device), old_logp=put(old) if with_old else None, ref_logp=put(ref) if with_ref else None,
                          mask=None if mask is None else rows_apart(mask, device, pad), lengths=None if lengths is None else lengths.to(device),
                          clip_low=clip[0], clip_high=clip[1], kl_coef=kl, reduce=reduce, grad_scale=grad_scale)
    a = (adv if per_step else adv[:, None].expand(N, T)).double()
    x = (lp.double() - old.double()) if with_old else torch.zeros(N, T, dtype=torch.float64)
    r, d = torch.exp(x), (ref.double() - lp.double()) if with_ref else torch.zeros(N, T, dtype=torch.float64)
    held = (a > 0) & (x > (math.log1p(clip[1]) if clip[1] < math.inf else math.inf)) | (a < 0) & (x < math.log1p(-clip[0]))
    obj = -torch.minimum(r * a, r.clamp(1 - clip[0], 1 + clip[1]) * a)
    k = torch.special.expm1(d) - d
    slope = torch.where(held, 0.0, -r * a) - kl * torch.special.expm1(d)
    count = where.sum()
    per_row = where.sum(1).clamp(min=1).double()
    w = {"token": torch.full((N, T), 1.0 / max(1, int(count)), dtype=torch.float64), "row": (1 / (per_row * N))[:, None].expand(N, T),
         "sum": torch.ones(N, T, dtype=torch.float64)}[reduce]
    w = torch.where(where, w, 0.0)
    # r: the argument's rounding and three steps of expf; obj: one product (the clip's bound: one rounding)
    t_obj = (x.abs() + 10) * U * (r * a).abs() + 2 * U * obj.abs()
    # the KL estimate: d rounded once, the series' or the difference's roundings (above 1/2: exp, 1 and d to half a step of the largest)
    t_kl = U * (d.abs() * torch.special.expm1(d).abs() + 16 * k + torch.where(d.abs() >= 0.49, 8 * torch.exp(d) + 2 * d.abs() + 2, 0.0))
    t_slope = t_obj + kl * (t_kl + 2 * U * d.abs()) + 2 * U * (slope.abs() + kl * (k + d).abs())
    want = w * grad_scale * slope
    assert out[1].dtype == dt and out[1].shape == lp.shape
    close(out[1], want, out_tol(want, w * grad_scale * t_slope + 3 * U * want.abs(), dt), "gradient")
    assert not out[1].cpu()[~where].any(), "gradient outside the places that count"
    so, sk = (w * obj).sum(), (w * k).sum()
    to, tk = (w * t_obj).sum(), (w * t_kl).sum()
    stats = torch.stack([so, sk, (held & where).sum().double() / max(1, int(count)), count.double()])
    close(out[2], stats, torch.stack([to + 9 * U * (w * obj.abs()).sum(), tk + 9 * U * sk, 2 * U * stats[2], torch.zeros((), dtype=torch.float64)]), "stats")
    close(out[0], (so + kl * sk).reshape(1), (to + 9 * U * (w * obj.abs()).sum() + kl * (tk + 10 * U * sk) + U * (so + kl * sk).abs()).item(), "loss")


def case_transition(device, B, n, dtype="f32", reduce="mean", seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = DTYPES[dtype]
    mean = torch.randn(B, n, generator=g)
    std = 0.05 + torch.rand(B, generator=g)
    x = (mean + std[:, None] * torch.randn(B, n, generator=g)).to(dt)
    mean = mean.to(dt)
    dlogp = torch.randn(B, generator=g)
    got = ops.transition_logprob(x.to(device), mean.to(device), std.to(device), reduce=reduce)
    grad = ops.transition_logprob_bwd(x.to(device), mean.to(device), std.to(device), dlogp.to(device), reduce=reduce)
    s, d = std.double()[:, None], x.double() - mean.double()
    k = 1.0 / n if reduce == "mean" else 1.0
    want = torch.distributions.Normal(mean.double(), s.expand_as(d)).log_prob(x.double()).sum(1) * k
    # differences one rounding, squares three, up to eight fp32 additions; the terms without x in fp64
    close(got, want, 11 * U * 0.5 * ((d / s) ** 2).sum(1) * k + U * want.abs(), "log-probability")
    want = dlogp.double()[:, None] * k * d / (s * s)
    assert grad.dtype == dt and grad.shape == x.shape
    close(grad, want, out_tol(want, 3 * U * want.abs(), dt), "gradient")


CLIP_SIZES = [1, 2, 3, 0, 7, 64, 255, 1000, 16384, 16385, 40001]


def case_clip(device, sizes=CLIP_SIZES, dtypes=("f32", "bf16", "f16"), out_dtypes=None, max_norm=1.0, scale=0.05, where="in place", seed=0):
    """where: "in place", "apart", or "flat" (slices of one flat buffer per format, at odd offsets)"""
    g = torch.Generator().manual_seed(seed)
    src = [(scale * torch.randn(n, generator=g)).to(DTYPES[dtypes[i % len(dtypes)]]) for i, n in enumerate(sizes)]
    out_dtypes = out_dtypes or dtypes
    dts = [s.dtype if where == "in place" else DTYPES[out_dtypes[i % len(out_dtypes)]] for i, s in enumerate(src)]
    dev = [s.clone().to(device) for s in src]
    if where == "in place":
        gs, out = ops.GradSet(dev), dev
    elif where == "apart":
        out = [torch.full(s.shape, float("nan"), dtype=d, device=device) for s, d in zip(src, dts)]
        gs = ops.GradSet(dev, out=out)
    else:
        out, used = [], {d: 1 for d in dts}
        flat = {d: torch.full((3 + sum(s.numel() + 1 for s in src),), float("nan"), dtype=d, device=device) for d in set(dts)}
        for s, d in zip(src, dts):
            out.append(flat[d][used[d]:used[d] + s.numel()])
            used[d] += s.numel() + 1
        gs = ops.GradSet(dev, out=out)
    total = sum((s.double() ** 2).sum().item() for s in src)
    norm = math.sqrt(total)
    sumsq = torch.empty(1, dtype=torch.float64, device=device)
    for first in (gs.norm(sumsq=sumsq), gs.clip(max_norm)):
        # fp64 throughout, one rounding to fp32
        close(first, torch.tensor([norm], dtype=torch.float64), 2 * U * norm, "norm")
    # 1000 fp64 additions at the most in any one chain, each half a step of fp64
    close(sumsq, torch.tensor([total], dtype=torch.float64), 1000 * 2.0 ** -53 * total, "sum of squares")
    f = min(1.0, max_norm / (norm + 1e-6)) if total else 1.0
    for s, o in zip(src, out):
        want = s.double() * f
        if f == 1.0 and o.dtype == s.dtype:
            assert torch.equal(o.cpu(), s), "nothing to clip: the bits stay"
        close(o, want, out_tol(want, 2 * U * want.abs(), o.dtype), "clipped gradient")
    if where == "flat":
        for d, t in flat.items():
            assert int(t.isnan().sum()) == t.numel() - sum(o.numel() for o in out if o.dtype == d), "written outside the outputs"


def case_policy_run(device, B=3, steps=4, n=24, seed=0):
    """the operators as they are used together: a sampler whose transition means are theta[step] * x, old and new policy, the clipped loss over the
    transitions' log-probabilities, back to the means, to theta, and the clipped gradient -- against autograd in 64 bits"""
    g = torch.Generator().manual_seed(seed)
    theta = 0.9 + 0.05 * torch.randn(steps, generator=g)
    old_theta, ref_theta = theta + 0.02 * torch.randn(steps, generator=g), theta + 0.02 * torch.randn(steps, generator=g)
    std = 0.2 + torch.rand(steps, generator=g)
    adv = torch.randn(B, generator=g)
    lengths = torch.tensor([steps, 0, steps - 1][:B] + [steps] * max(0, B - 3), dtype=torch.int32)
    xs = [torch.randn(B, n, generator=g)]
    for t in range(steps):
        xs.append(old_theta[t] * xs[-1] + std[t] * torch.randn(B, n, generator=g))
    xs = [x.to(device) for x in xs]
    sd = [std[t].expand(B).contiguous().to(device) for t in range(steps)]

    def logps(th):
        return torch.stack([ops.transition_logprob(xs[t + 1], (th[t].to(device) * xs[t]).contiguous(), sd[t], reduce="sum") for t in range(steps)], 1)
    lp, old, ref = logps(theta), logps(old_theta), logps(ref_theta)
    loss, dlp, stats = ops.policy_loss(lp, adv.to(device), old_logp=old, ref_logp=ref, lengths=lengths.to(device), kl_coef=0.1)
    grads = []
    for t in range(steps):
        dmean = ops.transition_logprob_bwd(xs[t + 1], (theta[t].to(device) * xs[t]).contiguous(), sd[t], dlp[:, t].contiguous(), reduce="sum")
        grads.append((dmean * xs[t]).sum().reshape(1))
    norm = ops.GradSet(grads).clip(0.5)

    th = theta.double().requires_grad_()

    def logps64(v):
        return torch.stack([torch.distributions.Normal(v[t] * xs[t].double().cpu(), std[t].double())
                            .log_prob(xs[t + 1].double().cpu()).sum(1) for t in range(steps)], 1)
    l64, o64, r64 = logps64(th), logps64(old_theta.double()).detach(), logps64(ref_theta.double()).detach()
    where = (torch.arange(steps)[None] < lengths[:, None])
    r = torch.exp(l64 - o64)
    a = adv.double()[:, None]
    term = -torch.minimum(r * a, r.clamp(0.8, 1.2) * a) + 0.1 * (torch.exp(r64 - l64) - (r64 - l64) - 1)
    want = (term * where).sum() / where.sum()
    want.backward()
    # the sums' size times a few half steps moves every exponent; the tolerance follows from |logp| <= 200 here: 200 * 16 u relative on r and exp(d)
    rel = 200 * 16 * U
    big = ((r * a).abs() + 0.1 * torch.exp(r64 - l64)).detach()
    close(loss, want.detach().reshape(1), rel * (big * where).sum().item() / int(where.sum()), "loss")
    full = th.grad.norm().item()
    dlogp_tol = rel * big.max().item() / int(where.sum())
    reach = sum(((xs[t + 1] - theta[t].to(device) * xs[t]).double() * xs[t].double()).abs().sum().item() / float(std[t]) ** 2 for t in range(steps))
    close(norm, torch.tensor([full], dtype=torch.float64), dlogp_tol * reach + 64 * U * reach, "norm")
    f = min(1.0, 0.5 / (full + 1e-6))
    close(torch.cat(grads), th.grad * f, 2 * (dlogp_tol * reach + 64 * U * reach), "gradient of theta")


def case_preference_step(device, hw=8, seed=0):
    """the operators as they are used together: one preference step of the student against its own frozen base -- forward of preferred and rejected
    samples, loss and gradient, LoRA backward, global norm over the factors' gradients, AdamW on it, clipping of a copy -- against the oracle's autograd"""
    from oracle import unet_sd15 as O
    from pcm_amd.model import LoraState, UNet, UNetWeights
    from pcm_amd.unet_spec import UNetConfig
    kw = dict(block_out_channels=(64, 128, 128), cross_attention_dim=64, heads=2, norm_num_groups=32)
    oc, pc = O.UNetConfig(**kw), UNetConfig(**kw)
    sd = O.init_state_dict(oc, 0)
    g = torch.Generator().manual_seed(seed)
    latents, noise = torch.randn(2, 4, hw, hw, generator=g), torch.randn(2, 4, hw, hw, generator=g)
    ctx, t, beta = torch.randn(2, 7, 64, generator=g), torch.tensor([419, 419]), 1.0
    W, lora = UNetWeights(pc, sd, device), LoraState(pc, 64, 8.0, device, seed=1, b_std=0.05)
    olora = {k: (lora.A_peft(m).detach().cpu().clone().requires_grad_(), m.B.detach().cpu().clone().requires_grad_()) for k, m in lora.modules.items()}
    x, dev = (0.6 * latents + 0.8 * noise), lambda v: v.to(device)      # noqa: E731
    student, base = UNet(W, lora), UNet(W, None)
    eps, tape = student.forward(dev(x), dev(t), dev(ctx), save=True)
    ref = base.forward(dev(x), dev(t), dev(ctx))
    loss, d_eps, ratio = ops.denoise_preference_loss(eps, ref, dev(noise), beta=beta)
    lora.zero_grad()
    student.backward(d_eps, tape)

    oeps, oref = O.unet_forward(oc, sd, x, t, ctx, olora, 8.0), O.unet_forward(oc, sd, x, t, ctx).detach()
    n = oeps[0].numel()
    rho = -(((noise - oeps).double() ** 2 - (noise - oref).double() ** 2).flatten(1).sum(1)) / n
    oloss = -torch.nn.functional.logsigmoid(beta * (rho[0] - rho[1]))
    oloss.backward()
    rho, oloss = rho.detach(), oloss.detach()
    # the operator on the predictions it was given, exactly; against the oracle's predictions, by how far the log ratios are apart
    e, r, no = eps.double().cpu(), ref.double().cpu(), noise.double()
    own = -(((no - e) ** 2 - (no - r) ** 2).flatten(1).sum(1)) / n
    close(ratio, own, 12 * U * ((no - e) ** 2 + (no - r) ** 2).flatten(1).sum(1) / n + U * own.abs(), "log ratios")
    gap = float(((own[0] - own[1]) - (rho[0] - rho[1])).abs())
    assert abs(loss.item() - oloss.item()) <= beta * gap + 1e-6, (loss.item(), oloss.item(), gap)
    # the slope is off by at most beta gap / 4 of beta; the network's bf16 backward by 5 % (the bound of its own test on this width)
    slope = float(torch.sigmoid(-beta * (rho[0] - rho[1])))
    num = sum(float(((got.cpu() - want.grad.view_as(got)) ** 2).sum()) for k, m in lora.modules.items()
              for got, want in ((lora.gA_peft(m), olora[k][0]), (m.gB, olora[k][1])))
    den = sum(float((want.grad ** 2).sum()) for pair in olora.values() for want in pair)
    print("preference step: LoRA gradient rel err %.3e, margin off by %.3e" % ((num / den) ** 0.5, gap))
    assert (num / den) ** 0.5 < 0.05 + beta * gap / 4 / slope
    # norm over the factors' gradients (views of the flat buffer), and the optimizer step that takes its square
    factors = [t for m in lora.modules.values() for t in (m.gA, m.gB)]
    copies = [torch.empty_like(t) for t in factors]
    gs = ops.GradSet(factors, out=copies)
    flat = (lora.grads.double() ** 2).sum().item()
    norm = gs.norm(sumsq=lora.gradsq)
    close(lora.gradsq, torch.tensor([flat], dtype=torch.float64), 1e-12 * flat, "sum of squares")
    norm2, c = gs.clip(0.5 * flat ** 0.5), 0.5 * flat ** 0.5 / (flat ** 0.5 + 1e-6)
    assert torch.equal(norm, norm2)
    for a, b in zip(copies, factors):
        want = b.double().cpu() * c
        close(a, want, out_tol(want, 2 * U * want.abs(), torch.float32), "clipped factor gradient")
    before, max_norm, lr, wd = lora.params.clone(), 0.5 * flat ** 0.5, 1e-4, 1e-2
    ops.adamw_clip_step(lora.params, lora.grads, lora.exp_avg, lora.exp_avg_sq, lora.gradsq, max_norm, lr, 0.9, 0.999, 1e-8, wd, 1)
    clipped = lora.grads.double().cpu() * c
    want = before.double().cpu() * (1 - lr * wd) - lr * clipped / (clipped.abs() + 1e-8)      # the first step: m / bc1 = g, sqrt(v / bc2) = |g|
    # g / (|g| + eps) to a few fp32 roundings where |g| is not lost against eps
    close(lora.params, want, 16 * U * (before.double().cpu().abs() + lr) + lr * 64 * U, "parameters after the step")


def case_deterministic(device, big=False):
    """the same call twice gives the same bits"""
    g = torch.Generator().manual_seed(5)
    n, N, T = (70000, 300, 1111) if big else (3000, 6, 70)
    t, r, p = (torch.randn(4, n, generator=g).to(device) for _ in range(3))
    lp, old, ref = (-torch.rand(N, T, generator=g).to(device) for _ in range(3))
    adv = torch.randn(N, generator=g).to(device)
    grads = [torch.randn(k, generator=g).to(device) for k in (5, 20000, 333, n)]
    outs = [torch.empty_like(x) for x in grads]
    gs = ops.GradSet(grads, out=outs)

    def run():
        a = ops.denoise_preference_loss(p, r, t) + ops.preference_loss(lp, ref) + ops.policy_loss(lp, adv, old_logp=old, ref_logp=ref, kl_coef=0.1)
        return [x.clone() for x in a + (ops.transition_logprob(t, r, adv[:4].abs().contiguous() + 0.1), gs.clip(1.0), *outs)]
    for x, y in zip(run(), run()):
        assert torch.equal(x, y)


def case_not_a_number(device):
    """a non-finite norm reaches the gradients as the formula has it"""
    a, b = torch.ones(5, device=device), torch.full((3,), float("inf"), device=device)
    norm = ops.GradSet([a, b]).clip(1.0)
    assert math.isinf(norm.item()) and not a.cpu().any() and b.cpu().isnan().all()
    a, b = torch.ones(5, device=device), torch.full((3,), float("nan"), device=device)
    norm = ops.GradSet([a, b]).clip(1.0)
    assert math.isnan(norm.item()) and a.cpu().isnan().all()
    # a large finite gradient does not overflow the sum of squares
    a = torch.full((4,), 1e38, device=device)
    norm = ops.GradSet([a]).clip(1.0)
    close(norm, torch.tensor([2e38], dtype=torch.float64), 4 * U * 2e38, "norm")
    close(a, torch.full((4,), 0.5).double(), 4 * U, "clipped")
    # NaN where it counts shows in the loss
    lp = torch.zeros(2, 3, device=device)
    lp[0, 1] = float("nan")
    loss, grad, ratio = ops.preference_loss(lp, torch.zeros_like(lp))
    assert math.isnan(loss.item()) and math.isnan(ratio[0].item()) and ratio[1].item() == 0.0
    for kind in ("hinge", "square"):
        assert math.isnan(ops.preference_loss(lp, torch.zeros_like(lp), kind=kind)[0].item())
    assert math.isnan(ops.policy_loss(lp, torch.ones(2, device=device), old_logp=torch.zeros_like(lp))[0].item())
    # an advantage of zero takes a place out of the objective, however far the policy has moved
    far = torch.full((1, 2), 200.0, device=device)
    loss, grad, _ = ops.policy_loss(far, torch.zeros(1, device=device), old_logp=torch.zeros_like(far))
    assert loss.item() == 0.0 and not grad.cpu().any()


def case_without_gradient(device):
    """want_grad=False: no gradient, the same loss, log ratios and statistics -- in one launch and in several"""
    g = torch.Generator().manual_seed(9)
    for P, n, N, T in ((2, 40, 5, 7), (5, 9000, 70, 300)):
        t, r, p = (torch.randn(2 * P, 4, n, generator=g).to(device) for _ in range(3))
        lp, ref = (-torch.rand(N // 2 * 2, T, generator=g).to(device) for _ in range(2))
        adv = torch.randn(N // 2 * 2, generator=g).to(device)
        for f in (lambda w: ops.denoise_preference_loss(p, r, t, want_grad=w), lambda w: ops.preference_loss(lp, ref, want_grad=w),
                  lambda w: ops.policy_loss(lp, adv, old_logp=ref, ref_logp=ref, kl_coef=0.1, want_grad=w),
                  lambda w: ops.policy_loss(lp, adv, reduce="row", want_grad=w)):
            a, b = f(True), f(False)
            assert b[1] is None and a[1].abs().sum().item() > 0 and torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    # the sampler's four-dimensional latents, and an infinite bound
    x = torch.randn(3, 4, 16, 16, generator=g).to(device)
    s = torch.full((3,), 0.5, device=device)
    assert torch.equal(ops.transition_logprob(x, x * 0.5, s), ops.transition_logprob(x.flatten(1), (x * 0.5).flatten(1), s))
    assert ops.transition_logprob_bwd(x, x * 0.5, s, s).shape == x.shape
    before = x.clone()
    norm = ops.GradSet([x]).clip(float("inf"))
    assert torch.equal(x, before) and abs(norm.item() - before.double().norm().item()) <= 2 * U * norm.item()


def case_infinite_margins(device):
    """a sample the policy or the reference rules out: the pair's loss is 0 or infinite, its gradient that of the limit, and no 0 times infinity"""
    inf = float("inf")
    lp, ref = torch.zeros(4, 3, device=device), torch.zeros(4, 3, device=device)
    lp[2, 1] = -inf                                   # the rejected sample of pair 0: s = inf
    lp[1, 0] = -inf                                   # the preferred sample of pair 1: s = -inf
    loss, grad, ratio = ops.preference_loss(lp, ref, beta=0.5)
    assert loss.item() == inf and ratio.tolist() == [0.0, -inf, -inf, 0.0]
    # pair 0: slope 0; pair 1: slope -beta, over two pairs
    assert grad.cpu().tolist() == [[0.0] * 3, [-0.25] * 3, [0.0] * 3, [0.25] * 3]
    loss, grad, _ = ops.preference_loss(lp[::2].contiguous(), ref[::2].contiguous(), beta=0.5)
    assert loss.item() == 0.0 and not grad.cpu().any()


def case_refusals(device):
    x = torch.zeros(4, 6, device=device)
    half = x.to(torch.bfloat16)
    one = torch.ones(4, device=device)
    refused = [
        (TypeError, lambda: ops.preference_loss(x, half)),
        (TypeError, lambda: ops.preference_loss(x.double(), x.double())),
        (TypeError, lambda: ops.preference_loss(x, x, mask=x)),
        (TypeError, lambda: ops.preference_loss(x, x, lengths=one)),
        (ValueError, lambda: ops.preference_loss(x[:3], x[:3])),
        (ValueError, lambda: ops.preference_loss(x[:0], x[:0])),
        (ValueError, lambda: ops.preference_loss(x[:, :0], x[:, :0])),
        (ValueError, lambda: ops.preference_loss(x, x[:, :5])),
        (ValueError, lambda: ops.preference_loss(x, x, mask=torch.ones(4, 5, dtype=torch.bool, device=device))),
        (ValueError, lambda: ops.preference_loss(x, x, lengths=torch.ones(3, dtype=torch.int32, device=device))),
        (ValueError, lambda: ops.preference_loss(x.t().contiguous().t(), x)),
        (ValueError, lambda: ops.preference_loss(x[:1].expand(4, 6), x)),
        (ValueError, lambda: ops.preference_loss(x, x, kind="other")),
        (ValueError, lambda: ops.preference_loss(x, x, reduce="token")),
        (RuntimeError, lambda: ops.preference_loss(x, x, beta=0.0)),
        (RuntimeError, lambda: ops.preference_loss(x, x, beta=float("nan"))),
        (RuntimeError, lambda: ops.preference_loss(x, x, kind="hinge", label_smoothing=0.1)),
        (RuntimeError, lambda: ops.preference_loss(x, x, label_smoothing=0.5)),
        (TypeError, lambda: ops.denoise_preference_loss(x, half, x)),
        (ValueError, lambda: ops.denoise_preference_loss(x, x, x[:2])),
        (ValueError, lambda: ops.denoise_preference_loss(x[:3], x[:3], x[:3])),
        (ValueError, lambda: ops.denoise_preference_loss(x, x, x, weight=one[:2])),
        (ValueError, lambda: ops.denoise_preference_loss(x, x, x, weight=one.to(torch.bfloat16))),
        (ValueError, lambda: ops.denoise_preference_loss(x.t().contiguous().t(), x, x)),
        (RuntimeError, lambda: ops.denoise_preference_loss(x, x, x, beta=-1.0)),
        (TypeError, lambda: ops.policy_loss(x, one.to(torch.bfloat16), old_logp=x)),
        (ValueError, lambda: ops.policy_loss(x, one[:3], old_logp=x)),
        (ValueError, lambda: ops.policy_loss(x, one, old_logp=x, kl_coef=0.1)),
        (ValueError, lambda: ops.policy_loss(x, one, old_logp=x, reduce="mean")),
        (RuntimeError, lambda: ops.policy_loss(x, one, old_logp=x, clip_low=1.0)),
        (RuntimeError, lambda: ops.policy_loss(x, one, old_logp=x, clip_high=-0.1)),
        (ValueError, lambda: ops.policy_loss(x[0], one, old_logp=x[0])),
        (TypeError, lambda: ops.policy_loss([1.0], one)),
        (ValueError, lambda: ops.transition_logprob(x, x[:2], one)),
        (ValueError, lambda: ops.transition_logprob(x, x, one[:3])),
        (ValueError, lambda: ops.transition_logprob(x, x, one.double())),
        (TypeError, lambda: ops.transition_logprob(x, half, one)),
        (ValueError, lambda: ops.transition_logprob(x, x, one, reduce="token")),
        (ValueError, lambda: ops.transition_logprob_bwd(x, x, one, one[:3])),
        (ValueError, lambda: ops.GradSet([])),
        (ValueError, lambda: ops.GradSet([x, x])),                                  # the same gradient twice
        (ValueError, lambda: ops.GradSet([x.view(-1)[:10], x.view(-1)[9:]])),        # overlapping
        (ValueError, lambda: ops.GradSet([x], out=[x.view(-1)[:12]])),
        (ValueError, lambda: ops.GradSet([x[:2]], out=[x[1:3]])),                    # an output over its own gradient, shifted
        (ValueError, lambda: ops.GradSet([x[:2], x[2:]], out=[x[2:], x[:2]])),       # outputs over other gradients
        (ValueError, lambda: ops.GradSet([x[:, :3]])),                               # gaps
        (ValueError, lambda: ops.GradSet([x], out=[x.clone().t().contiguous().t()])),  # another element order
        (TypeError, lambda: ops.GradSet([x.double()])),
        (TypeError, lambda: ops.GradSet([None])),
        (ValueError, lambda: ops.GradSet([x]).clip(0.0)),
        (ValueError, lambda: ops.GradSet([x]).clip(float("nan"))),
        (ValueError, lambda: ops.GradSet([x]).norm(sumsq=one)),
    ]
    for i, (kind, call) in enumerate(refused):
        with pytest.raises(kind):
            call()
            raise AssertionError(f"call {i} was not refused")


def case_dense_orders(device):
    """gradients whose elements are dense but not row-major, and a set that holds nothing"""
    a = torch.randn(5, 7).t()
    b = torch.randn(2, 3, 4, 5).to(memory_format=torch.channels_last)
    want = math.sqrt((a.double() ** 2).sum().item() + (b.double() ** 2).sum().item())
    da, db = torch.empty(5, 7, device=device).t().copy_(a), b.clone().to(device)
    norm = ops.GradSet([da, db]).clip(0.5)
    close(norm, torch.tensor([want], dtype=torch.float64), 2 * U * want, "norm")
    f = 0.5 / (want + 1e-6)
    for got, x in ((da, a), (db, b)):
        close(got, x.double() * f, 3 * U * x.double().abs() * f, "clipped")
    empty = ops.GradSet([torch.empty(0, device=device)])
    sumsq = torch.ones(1, dtype=torch.float64, device=device)
    assert empty.clip(1.0, sumsq=sumsq).item() == 0.0 and sumsq.item() == 0.0


# ---- where terms cancel, overflow or reach a limit: bounds relative to the 64-bit value ----
def case_separated_pairs(device):
    """the slope of pairs that are far apart keeps its digits down to the smallest number of fp32: margins s = beta * h with beta = 1, so that the
    margin itself is exact"""
    for eps in (0.0, 0.1):
        for s in (-60.0, -25.0, 0.0, 5.0, 17.0, 25.0, 30.0, 36.0, 38.0, 60.0, 85.0):
            lp = torch.tensor([[s], [0.0]], device=device)
            loss, grad, ratio = ops.preference_loss(lp, torch.zeros_like(lp), beta=1.0, label_smoothing=eps)
            down = math.exp(-s) / (1 + math.exp(-s)) if s >= 0 else 1 / (1 + math.exp(s))      # sig(-s) and sig(s), each without a difference
            up = math.exp(s) / (1 + math.exp(s)) if s < 0 else 1 / (1 + math.exp(-s))
            want = eps * up - (1 - eps) * down
            # fp64 throughout (its roundings, of what is subtracted, do not count), rounded once to the factor and once to the output
            close(grad, torch.tensor([[want], [-want]], dtype=torch.float64), 3 * U * abs(want) + 16 * 2.0 ** -53 + 2.0 ** -149 if eps else 3 * U * abs(want), (eps, s))
    # the same through the launches of many pairs
    P = 200
    s = torch.linspace(-20.0, 80.0, P).float()
    lp = torch.cat([s, torch.zeros(P)])[:, None]
    _, grad, _ = ops.preference_loss(lp.to(device), torch.zeros_like(lp).to(device), beta=1.0)
    want = -torch.sigmoid(-s.double()) / P
    close(grad[:P, 0], want, 4 * U * want.abs(), "many pairs")
    close(grad[P:, 0], -want, 4 * U * want.abs(), "many pairs")


def case_far_reference(device):
    """the KL term and its gradient, 1 - exp(d), where policy and reference are far apart, up to a reference that rules a place out (d = -inf) and a
    policy that does (d = inf)"""
    inf = float("inf")
    for dtype in ("f32", "bf16", "f16"):
        dt = DTYPES[dtype]
        ds = torch.tensor([-inf, torch.finfo(dt).min, -3e4, -1e4, -300.0, -20.0, -10.0, -2.5, -0.75, -0.5, -0.25, -2.0 ** -9, 0.0, 2.0 ** -9, 0.25, 0.5, 0.75, 2.5, 10.0, inf],
                          dtype=dt)
        # in one launch (rows of one place, of three, of nine), in several, and a row to a workgroup
        for rows, cols, reduce in ((1, 1, "sum"), (7, 3, "sum"), (3, 9, "sum"), (40, 500, "sum"), (32, 520, "row")):
            for d0 in range(len(ds)) if cols == 1 else (0,):
                ref = ds[(torch.arange(rows * cols) + d0) % len(ds)].view(rows, cols)
                lp = torch.zeros(rows, cols, dtype=dt)
                lp[ref == inf] = -inf                                        # the policy rules the place out: d = inf
                ref[ref == inf] = 0.0
                d = ref.double() - lp.double()
                for kl, a in ((1.0, 0.0), (0.04, 1.0)):
                    scale = float(rows * cols) if reduce == "row" else 1.0
                    old = torch.zeros_like(lp)
                    loss, grad, stats = ops.policy_loss(lp.to(device), torch.full((rows,), a, device=device), old_logp=old.to(device), ref_logp=ref.to(device),
                                                        kl_coef=kl, reduce=reduce, grad_scale=scale)
                    rise, r = torch.special.expm1(d), torch.exp(lp.double())
                    want = -a * r - kl * rise
                    # the exponential's four half steps, the difference's one, the product's and the sum's one each; the weight's one
                    tol = U * (6 * kl * torch.where(d.abs() < 0.5, rise.abs(), torch.exp(d)) + kl * rise.abs() + 4 * a * r + 3 * want.abs())
                    if a:                                                    # (advantage 0 and lp = -inf: 0 * (-inf - 0), no number)
                        close(grad, want, out_tol(want, tol, dt), (dtype, rows, cols, a, d0))
                    else:
                        fine = lp > -inf
                        close(grad[fine.to(device)], want[fine], out_tol(want, tol, dt)[fine], (dtype, rows, cols, a, d0))
                    kd = torch.where(d == inf, inf, rise - d)
                    w = scale if reduce == "row" else 1.0
                    t_kl = U * torch.where(d.abs() < 0.5, 16 * kd, 8 * torch.exp(d) + 3 * d.abs() + 2)
                    close(stats[1].reshape(1), (kd.sum() / w).reshape(1), (t_kl.sum() / w + 9 * U * kd.sum() / w).reshape(1), "KL")


def case_monitored_kl(device):
    """kl_coef = 0 with a reference: the KL is in the statistics, loss and gradient are those of the call without reference, also where the KL is infinite"""
    inf = float("inf")
    for rows, cols, reduce in ((1, 1, "token"), (3, 9, "token"), (40, 500, "token"), (32, 520, "row"), (6000, 3, "sum")):
        g = torch.Generator().manual_seed(rows)
        lp = -torch.rand(rows, cols, generator=g)
        old, adv = lp + 0.1 * torch.randn(rows, cols, generator=g), torch.randn(rows, generator=g)
        for d in (1.0, 95.0, inf, -inf):
            ref = lp.clone()
            ref[0, 0] += d
            lp, old, ref, adv = (t.to(device) for t in (lp, old, ref, adv))
            with_ref = ops.policy_loss(lp, adv, old_logp=old, ref_logp=ref, kl_coef=0.0, reduce=reduce)
            without = ops.policy_loss(lp, adv, old_logp=old, reduce=reduce)
            assert torch.isfinite(without[0]).all() and torch.equal(with_ref[0], without[0]), (rows, cols, d)
            assert torch.equal(with_ref[1], without[1]), (rows, cols, d)
            kl = with_ref[2][1].item()
            assert (kl == inf) if d != 1.0 else 0.0 < kl < 1.0, (rows, cols, d, kl)
            assert torch.equal(with_ref[2][[0, 2, 3]], without[2][[0, 2, 3]])
            lp, old, adv = lp.cpu(), old.cpu(), adv.cpu()


def case_zero_advantage(device):
    """an advantage of zero takes a place out of the objective, also where old or new policy rule it out; a NaN stays one"""
    inf, nan = float("inf"), float("nan")
    for rows, cols in ((1, 2), (5, 7), (40, 500)):
        for lp0, old0, want in ((-inf, 0.0, 0.0), (0.0, -inf, 0.0), (200.0, -200.0, 0.0), (nan, 0.0, nan), (-inf, -inf, nan)):
            lp, old, adv = torch.zeros(rows, cols), torch.zeros(rows, cols), torch.ones(rows, cols)
            lp[0, 1], old[0, 1], adv[0, 1] = lp0, old0, 0.0
            loss, grad, stats = ops.policy_loss(lp.to(device), adv.to(device), old_logp=old.to(device), reduce="sum")
            wl = torch.tensor([-(rows * cols - 1.0) + want], dtype=torch.float64)
            close(loss, wl, 0.0, ("loss", lp0, old0))
            wg = torch.full((rows, cols), -1.0, dtype=torch.float64)
            wg[0, 1] = want
            close(grad, wg, 0.0, ("gradient", lp0, old0))
            assert stats[2].item() == 0.0


def case_student_near_base(device):
    """the log ratios of a student close to its frozen base, as at the start of every run: exactly 0 where the predictions agree, and with an error that
    shrinks with their distance"""
    for P, n in ((1, 16384), (8, 500), (200, 300), (2, 20001)):
        for dtype in ("f32", "bf16", "f16"):
            dt = DTYPES[dtype]
            g = torch.Generator().manual_seed(n)
            t = torch.randn(2 * P, n, generator=g).to(dt)
            r = (t.float() + 0.3 * torch.randn(2 * P, n, generator=g)).to(dt)
            for away in (0.0, 1e-6, 1e-5, 1e-3):
                p = (r.float() + away * torch.randn(2 * P, n, generator=g)).to(dt)
                beta = 200.0
                loss, grad, ratio = ops.denoise_preference_loss(p.to(device), r.to(device), t.to(device), beta=beta)
                a, b, d = t.double() - p.double(), t.double() - r.double(), r.double() - p.double()
                want = -(d * (a + b)).mean(1)
                # differences, their sum and the product one rounding each, up to eight fp32 additions
                tol = 12 * U * (d.abs() * (a.abs() + b.abs())).mean(1)
                close(ratio, want, tol + U * want.abs(), (P, n, dtype, away))
                s = beta * (want[:P] - want[P:])
                close(loss, -torch.nn.functional.logsigmoid(s).mean().reshape(1), beta * (tol[:P] + tol[P:]).mean() + 2 * U, (P, n, dtype, away))
                if away == 0.0:
                    assert not ratio.cpu().any()


def case_lowest_reference(device):
    """log-probabilities of the format's lowest number at places that count: their sums leave fp32 but not the margin of a pair whose rows both hold them"""
    for dtype in ("f32", "bf16"):
        dt = DTYPES[dtype]
        low = torch.finfo(dt).min
        for P, T in ((1, 2), (2, 8), (3, 1500), (100, 400)):
            lp, ref = torch.zeros(2 * P, T, dtype=dt), torch.full((2 * P, T), low, dtype=dt)
            for reduce in ("mean", "sum"):
                loss, grad, ratio = ops.preference_loss(lp.to(device), ref.to(device), beta=0.5, reduce=reduce)
                close(loss, torch.tensor([math.log(2.0)], dtype=torch.float64), 2 * U, (dtype, P, T, reduce))
                close(ratio, torch.full((2 * P,), -low if reduce == "mean" else math.inf).double(), 2 * U * -low, (dtype, P, T, reduce))
                g = -0.25 / P / (T if reduce == "mean" else 1)
                want = torch.cat([torch.full((P, T), g), torch.full((P, T), -g)]).double()
                close(grad, want, out_tol(want, 2 * U * want.abs(), dt), (dtype, P, T, reduce))


def case_too_many_rows(device):
    """a launch has fewer than 2^32 threads: rows that would need more are refused before anything is read or launched"""
    import ctypes as C
    from pcm_amd import capi
    x = torch.zeros(64, device=device)
    p = x.data_ptr()
    lib = capi.lib()
    for rows, n in ((1 << 24, 2000), ((1 << 24) - 1, 2000), ((1 << 24) + 1, 1), (1 << 40, 1), (1 << 62, 2000)):
        with pytest.raises(RuntimeError):
            lib.call("pcm_transition_logprob", p, p, p, 0, 1, p, rows, n, p, 1 << 50, None)
        with pytest.raises(RuntimeError):
            lib.call("pcm_transition_logprob_bwd", p, p, p, p, 0, 1, p, rows, n, None)
    for pairs, n in ((1 << 23, 2000), ((1 << 23) + 1, 1), (1 << 40, 1), (1 << 62, 2000)):
        a = capi.DenoisePreferenceArgs(p, p, p, None, None, p, p, p, 1 << 50, pairs, n, 1.0, 0.0, 1.0, 0, 0, 0)
        with pytest.raises(RuntimeError):
            lib.call("pcm_denoise_preference_loss", C.byref(a), None)
        a = capi.PreferenceArgs(p, p, None, None, None, p, p, p, 1 << 50, pairs, n, n, n, 0, n, 1.0, 0.0, 1.0, 0, 0, 0, 0)
        with pytest.raises(RuntimeError):
            lib.call("pcm_preference_loss", C.byref(a), None)
    assert not x.cpu().any()


def case_transition_scales(device):
    """deviations far from 1: squares and the gradient's factor leave fp32 before their results do"""
    for B, n, dtype in ((4, 40, "f32"), (4, 3000, "bf16"), (4, 70000, "f32"), (2, 140000, "bf16")):
        dt = DTYPES[dtype]
        g = torch.Generator().manual_seed(n)
        for s, dl in ((1e-22, 1.0), (1e-19, 1e-3), (1e18, 1e-10), (1e25, 1e20)):
            std = torch.full((B,), s)
            x = (std[:, None] * torch.randn(B, n, generator=g)).to(dt)
            mean, dlogp = torch.zeros(B, n, dtype=dt), torch.full((B,), dl)
            sd, d = std.double()[:, None], x.double()
            for reduce, k in (("mean", 1.0 / n), ("sum", 1.0)):
                args = [t.to(device) for t in (x, mean, std)]
                want = torch.distributions.Normal(mean.double(), sd.expand_as(d)).log_prob(d).sum(1) * k
                # differences exact here, all else in fp64
                close(ops.transition_logprob(*args, reduce=reduce), want, 2 * U * want.abs(), (B, n, s, reduce))
                want = -dlogp.double()[:, None] * k * (mean.double() - d) / (sd * sd)
                close(ops.transition_logprob_bwd(*args, dlogp.to(device), reduce=reduce), want, out_tol(want, 2 * U * want.abs(), dt), (B, n, s, reduce))


def case_sampler_transition(device):
    """the stochastic flow-matching sampler's step from sigma to sigma_next as a transition: mean (1 - sigma_next) (x - sigma v), deviation sigma_next; the
    gradient by the model's output v follows with the factor -(1 - sigma_next) sigma"""
    from pcm_amd.fm import PCMFMSampler
    g = torch.Generator().manual_seed(3)
    sampler = PCMFMSampler(shift=3.0, stochastic=True)
    sampler.set_timesteps(4)
    x = torch.randn(2, 4, 8, 8, generator=g).to(device)
    for t, s, s_next in zip(sampler.timesteps, sampler.sigmas_[:-1].tolist(), sampler.sigmas_[1:].tolist()):
        v, noise = (torch.randn(x.shape, generator=g).to(device) for _ in range(2))
        out = sampler.step(v, t, x, noise=noise)
        mean = (1.0 - s_next) * (x - s * v)
        if s_next == 0.0:                            # the last step draws nothing: no density
            close(out, mean.cpu(), 8 * U * (x.abs() + v.abs()).cpu().double(), "last step")
            break
        close(out, (mean + s_next * noise).cpu(), 8 * U * (x.abs() + v.abs() + noise.abs()).cpu().double(), "step")
        std = torch.full((2,), s_next, device=device)
        logp = ops.transition_logprob(out, mean, std)
        dlogp = torch.tensor([0.5, -2.0], device=device)
        dv = -(1.0 - s_next) * s * ops.transition_logprob_bwd(out, mean, std, dlogp)
        v64 = v.double().cpu().requires_grad_()
        m64 = (1.0 - s_next) * (x.double().cpu() - s * v64)
        want = torch.distributions.Normal(m64, s_next).log_prob(out.double().cpu()).flatten(1).mean(1)
        (want * dlogp.double().cpu()).sum().backward()
        # mean and step are rounded to fp32: up to eight half steps of the largest of their terms, divided by the deviation
        off = 16 * U * (x.abs() + v.abs() + noise.abs()).double().cpu() / s_next
        z = ((out.double().cpu() - m64) / s_next).detach()
        close(logp, want.detach(), (z.abs() * off + off ** 2).flatten(1).mean(1) + 2 * U * want.detach().abs(), "log-probability")
        n = x[0].numel()
        tol = dlogp.double().cpu().abs()[:, None, None, None] * s * (1.0 - s_next) / s_next / n * off
        close(dv, v64.grad, tol + 8 * U * v64.grad.abs(), "gradient by the model's output")
        x = out


def case_without_gradient_16bit(device):
    """want_grad=False in the 16-bit formats, over every launch form"""
    for dtype in ("bf16", "f16"):
        dt = DTYPES[dtype]
        g = torch.Generator().manual_seed(4)
        for P, T in ((2, 40), (5, 9000), (300, 130), (2500, 3)):
            a, b, c = (torch.randn(2 * P, T, generator=g).to(dt).to(device) for _ in range(3))
            adv = torch.randn(2 * P, generator=g).to(device)
            mask = (torch.rand(2 * P, T, generator=g) < 0.7).to(device)
            for f in (lambda w: ops.denoise_preference_loss(a, b, c, want_grad=w, beta=1.0), lambda w: ops.preference_loss(a, b, mask=mask, want_grad=w),
                      lambda w: ops.policy_loss(a, adv, old_logp=b, ref_logp=c, mask=mask, kl_coef=0.1, want_grad=w), lambda w: ops.policy_loss(a, adv, old_logp=b, reduce="row", want_grad=w)):
                x, y = f(True), f(False)
                assert y[1] is None and torch.isfinite(x[0]).all() and torch.equal(x[0], y[0]) and torch.equal(x[2], y[2]), (dtype, P, T)
