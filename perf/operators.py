"""The alignment operators of pcm_amd.ops as a benchmark: preference losses over paired log ratios, the clipped policy loss with its KL term,
the log-probability of a sampler transition, and the global gradient norm with clipping.

``run`` computes them from elementary torch operations (``own`` false) or through pcm_amd.ops (``own`` true); ``exact`` gives the same outputs in
64 bits from the definitions.  Latent sizes are those of the framework's configurations (4 x 64 x 64, 4 x 128 x 128, 16 x 128 x 128)."""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _ops():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "phased-consistency-model_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from pcm_amd import ops
    return ops


# ---- cases ------------------------------------------------------------------------------------------------------------------------------
def _denoise(pairs, n, dtype, kind, smoothing=0.0, weighted=False, reduce="mean"):
    # with "sum" the mean's strength is kept by dividing beta by n
    beta = 2000.0 if reduce == "mean" else 2000.0 / n
    if kind == "square":
        beta = beta / 1000.0
    # half-precision gradients are loss-scaled so that they stay in the format's range, as half-precision training does
    scale = pairs * n / (2.0 if kind == "square" else 2000.0) if dtype == "f16" else 1.0
    return {"op": "denoise_preference", "pairs": pairs, "n": n, "dtype": dtype, "kind": kind, "smoothing": smoothing, "weighted": weighted,
            "reduce": reduce, "beta": beta, "scale": scale}


def _preference(pairs, steps, dtype, kind, smoothing=0.0, masked=False, ragged=False, reduce="sum", pad=0):
    return {"op": "preference", "pairs": pairs, "steps": steps, "dtype": dtype, "kind": kind, "smoothing": smoothing, "masked": masked,
            "ragged": ragged, "reduce": reduce, "pad": pad, "beta": 0.1 if reduce == "sum" else 2.0,
            "scale": 1.0 if dtype != "f16" else float(pairs * (steps if reduce == "mean" else 1))}


def _policy(rows, steps, dtype, masked=False, ragged=False, per_step=False, kl=0.0, reduce="token", pad=0):
    return {"op": "policy", "rows": rows, "steps": steps, "dtype": dtype, "masked": masked, "ragged": ragged, "per_step": per_step, "kl": kl,
            "reduce": reduce, "pad": pad, "scale": float(rows * steps) if dtype == "f16" and reduce != "sum" else 1.0}


def _logprob(direction, rows, n, dtype, reduce="mean"):
    return {"op": "transition_" + direction, "rows": rows, "n": n, "dtype": dtype, "reduce": reduce}


def _clip(count, smallest, largest, dtype, multiple=1):
    return {"op": "clip", "count": count, "smallest": smallest, "largest": largest, "dtype": dtype, "multiple": multiple}


def listed():
    return [
        # one preference pair of 64 x 64 latents: the call of a step at batch size one, where latency counts
        dict(_denoise(1, 4 * 64 * 64, "f32", "sigmoid"), name="denoise_one_pair"),
        # an ordinary batch at an odd resolution, 16-bit predictions, timestep weights
        dict(_denoise(24, 4 * 97 * 61, "bf16", "square", weighted=True), name="denoise_odd_bf16"),
        # the largest batch of 16-channel 128 x 128 latents that a card steps through at once
        dict(_denoise(64, 16 * 128 * 128, "f32", "sigmoid", smoothing=0.1), name="denoise_large"),
        # log-probabilities of the 50 transitions of a full sampler run, four pairs
        dict(_preference(4, 50, "f32", "sigmoid"), name="preference_sampler"),
        # long ragged sequences of odd length with a mask, some rows empty
        dict(_preference(96, 4099, "f32", "sigmoid", smoothing=0.05, masked=True, ragged=True, reduce="mean"), name="preference_long"),
        # eight samples of a four-step sampler with one reward each: the smallest policy step
        dict(_policy(8, 4, "f32", kl=0.04), name="policy_four_steps"),
        # an ordinary batch: 16-bit log-probabilities, a mask, an advantage per step, every row with the same weight
        dict(_policy(512, 1027, "bf16", masked=True, per_step=True, kl=0.02, reduce="row"), name="policy_rows_bf16"),
        # a large ragged batch with reference log-probabilities
        dict(_policy(2048, 8192, "f32", ragged=True, kl=0.04), name="policy_large"),
        # the log-probabilities of one transition of a batch of sixteen 64 x 64 latents
        dict(_logprob("forward", 16, 4 * 64 * 64, "f32"), name="transition_forward"),
        # its gradient for sixty-four 16-channel 128 x 128 latents
        dict(_logprob("backward", 64, 16 * 128 * 128, "f32"), name="transition_backward"),
        # the few small gradients of an embedding and its norm
        dict(_clip(12, 64, 4096, "f32"), name="clip_few"),
        # the gradients of low-rank factors on every layer of a denoiser, 16-bit and 32-bit ones side by side
        dict(_clip(556, 20000, 600000, "mixed", multiple=64), name="clip_low_rank_factors"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["denoise", "preference", "policy", "policy", "forward", "backward", "clip"])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    kind = rng.choice(["sigmoid", "sigmoid", "hinge", "square"])
    smoothing = rng.choice([0.0, 0.1]) if kind == "sigmoid" else 0.0
    masked, ragged, pad = rng.random() < 0.5, rng.random() < 0.5, rng.choice([0, 0, 0, 1, 8, 13])
    if op == "denoise":
        n = rng.choice([4 * 64 * 64, 4 * 128 * 128, 16 * 128 * 128, 16 * 64 * 64, _log(rng, 1000, 262144), _log(rng, 1000, 262144)])
        return _denoise(_log(rng, 1, max(1, min(256, 64 * 262144 // n))), n, dtype, kind, smoothing, rng.random() < 0.5, rng.choice(["mean", "sum"]))
    if op == "preference":
        steps = _log(rng, 1, 32768)
        return _preference(_log(rng, 1, max(1, min(1024, (1 << 22) // steps))), steps, dtype, kind, smoothing, masked, ragged,
                           rng.choice(["sum", "mean"]), pad)
    if op == "policy":
        steps = _log(rng, 1, 32768)
        return _policy(_log(rng, 1, max(1, min(16384, (1 << 24) // steps))), steps, dtype, masked, ragged, rng.random() < 0.5,
                       rng.choice([0.0, 0.04]), rng.choice(["token", "row", "sum"]), pad)
    if op == "clip":
        largest = _log(rng, 100, 2000000)
        return _clip(_log(rng, 1, max(1, min(900, 64000000 // largest))), max(1, largest // rng.choice([1, 10, 300])), largest,
                     rng.choice(["f32", "bf16", "mixed"]), rng.choice([1, 8, 64]))
    n = rng.choice([4 * 64 * 64, 4 * 128 * 128, 16 * 128 * 128, _log(rng, 1000, 262144), _log(rng, 1000, 262144)])
    return _logprob(op, _log(rng, 1, max(1, min(512, 64 * 262144 // n))), n, dtype, rng.choice(["mean", "sum"]))


def _clip_tensors(case):
    """sizes spread evenly in the logarithm from smallest to largest, in a fixed shuffled order, and their formats"""
    count, lo, hi = case["count"], case["smallest"], case["largest"]
    out = []
    for i in range(count):
        j = (i * 7919) % count
        size = int(round(lo * (hi / lo) ** (j / max(1, count - 1)) / case["multiple"])) * case["multiple"]
        size = max(size, case["multiple"])
        dtype = case["dtype"] if case["dtype"] != "mixed" else ("f32", "bf16", "f32", "f16")[i % 4]
        out.append((size, dtype))
    return out


# ---- inputs -----------------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _valid(case, rows, g):
    """mask (a prompt in front and a few dropped places), lengths (some zero) and where both count a place; None for what the case has not"""
    steps = case["steps"]
    places = torch.arange(steps, device="cuda")
    mask = lengths = None
    where = torch.ones(rows, steps, dtype=torch.bool, device="cuda")
    if case["masked"]:
        prompt = (torch.rand(rows, 1, device="cuda", generator=g) * steps * 0.4).long()
        wide = torch.zeros(rows, steps + case["pad"], dtype=torch.bool, device="cuda")
        mask = wide[:, :steps]
        mask.copy_((places >= prompt) & (torch.rand(rows, steps, device="cuda", generator=g) < 0.95))
        where = where & mask
    if case["ragged"]:
        lengths = (steps * (0.3 + 0.7 * torch.rand(rows, device="cuda", generator=g))).round().to(torch.int32)
        lengths = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.03, torch.zeros_like(lengths), lengths)
        where = where & (places < lengths[:, None])
    return mask, lengths, where


def _rows_like(value, where, case):
    """value in the case's format, with the format's lowest number where nothing counts, as a view of rows ``pad`` places longer"""
    dtype = DTYPES[case["dtype"]]
    value = value.to(dtype)
    value = torch.where(where, value, torch.full_like(value, torch.finfo(dtype).min))
    wide = torch.zeros(value.shape[0], value.shape[1] + case["pad"], dtype=dtype, device="cuda")
    wide[:, :value.shape[1]] = value
    return wide[:, :value.shape[1]]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    state = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if op == "denoise_preference":
        dtype, shape = DTYPES[case["dtype"]], (2 * case["pairs"], case["n"])
        target = normal(*shape)
        reference = target + 0.3 * normal(*shape)
        state["pred"] = (reference + 0.03 * normal(*shape)).to(dtype)
        state["ref"], state["target"] = reference.to(dtype), target.to(dtype)
        state["weight"] = torch.rand(shape[0], device="cuda", generator=g) + 0.5 if case["weighted"] else None
    elif op == "preference":
        rows = 2 * case["pairs"]
        state["mask"], state["lengths"], where = _valid(case, rows, g)
        logp = -torch.rand(rows, case["steps"], device="cuda", generator=g) * 4.0
        spread = 1.0 / math.sqrt(case["steps"]) if case["reduce"] == "sum" else 0.5
        state["logp"] = _rows_like(logp, where, case)
        state["ref"] = _rows_like(logp + spread * normal(rows, case["steps"]), where, case)
    elif op == "policy":
        rows, steps = case["rows"], case["steps"]
        state["mask"], state["lengths"], where = _valid(case, rows, g)
        logp = -torch.rand(rows, steps, device="cuda", generator=g) * 4.0
        state["logp"] = _rows_like(logp, where, case)
        state["old"] = _rows_like(logp + 0.15 * normal(rows, steps), where, case)
        state["ref"] = _rows_like(logp + 0.3 * normal(rows, steps), where, case) if case["kl"] else None
        state["advantages"] = normal(rows, steps) if case["per_step"] else normal(rows)
    elif op in ("transition_forward", "transition_backward"):
        dtype, rows = DTYPES[case["dtype"]], case["rows"]
        std = 0.05 + 0.5 * torch.rand(rows, device="cuda", generator=g)
        mean = normal(rows, case["n"])
        state["x"] = (mean + std[:, None] * normal(rows, case["n"])).to(dtype)
        state["mean"], state["std"] = mean.to(dtype), std
        state["dlogp"] = normal(rows) * (1.0 if case["reduce"] == "mean" else 1.0 / case["n"])
        if dtype == torch.float16:
            state["dlogp"] = state["dlogp"] * case["n"]      # loss-scaled
    else:
        grads = [(0.01 * normal(size)).to(DTYPES[d]) for size, d in _clip_tensors(case)]
        # clipped gradients go to one flat buffer of each format, in order: what an optimizer or a gradient exchange reads
        state["flat"] = {d: torch.empty(sum(t.numel() for t in grads if t.dtype == DTYPES[d]), dtype=DTYPES[d], device="cuda")
                         for d in sorted({d for _, d in _clip_tensors(case)})}
        used, out = {d: 0 for d in DTYPES.values()}, []
        for (size, d), t in zip(_clip_tensors(case), grads):
            out.append(state["flat"][d][used[t.dtype]:used[t.dtype] + size])
            used[t.dtype] += size
        state["grads"], state["out"] = grads, out
        state["max_norm"] = 0.004 * math.sqrt(sum(t.numel() for t in grads))
        if own:
            state["set"] = _ops().GradSet(grads, out=state["out"])
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)(case["op"], case, state)


def _run_own(op, case, s):
    ops = _ops()
    if op == "denoise_preference":
        loss, grad, ratio = ops.denoise_preference_loss(s["pred"], s["ref"], s["target"], weight=s["weight"], beta=case["beta"], kind=case["kind"],
                                                        label_smoothing=case["smoothing"], reduce=case["reduce"], grad_scale=case["scale"])
        return {"loss": loss, "grad": grad, "ratio": ratio}
    if op == "preference":
        loss, grad, ratio = ops.preference_loss(s["logp"], s["ref"], mask=s["mask"], lengths=s["lengths"], beta=case["beta"], kind=case["kind"],
                                                label_smoothing=case["smoothing"], reduce=case["reduce"], grad_scale=case["scale"])
        return {"loss": loss, "grad": grad, "ratio": ratio}
    if op == "policy":
        loss, grad, stats = ops.policy_loss(s["logp"], s["advantages"], old_logp=s["old"], ref_logp=s["ref"], mask=s["mask"], lengths=s["lengths"],
                                            clip_low=0.2, clip_high=0.28, kl_coef=case["kl"], reduce=case["reduce"], grad_scale=case["scale"])
        return {"loss": loss, "grad": grad, "stats": stats}
    if op == "transition_forward":
        return {"logp": ops.transition_logprob(s["x"], s["mean"], s["std"], reduce=case["reduce"])}
    if op == "transition_backward":
        return {"grad": ops.transition_logprob_bwd(s["x"], s["mean"], s["std"], s["dlogp"], reduce=case["reduce"])}
    norm = s["set"].clip(s["max_norm"])
    return {"norm": norm, "grads": s["flat"]}


def _counted(s, like):
    where = torch.ones(like.shape, dtype=torch.bool, device=like.device)
    if s["mask"] is not None:
        where = where & s["mask"]
    if s["lengths"] is not None:
        where = where & (torch.arange(like.shape[1], device=like.device) < s["lengths"][:, None])
    return where


def _pair_terms(ratio, case):
    """loss and its derivative by each row's log ratio, in 64 bits: there is one value per row"""
    pairs, beta, eps = case["pairs"], case["beta"], case["smoothing"]
    h = ratio[:pairs] - ratio[pairs:]
    if case["kind"] == "sigmoid":
        s = beta * h
        soft = torch.log1p(torch.exp(-s.abs()))
        loss = (1 - eps) * (soft + (-s).clamp(min=0)) + eps * (soft + s.clamp(min=0))
        slope = beta * (1 / (1 + torch.exp(-s)) - (1 - eps))
    elif case["kind"] == "hinge":
        s = beta * h
        loss = (1 - s).clamp(min=0)
        slope = torch.where(s < 1, torch.full_like(s, -beta), torch.zeros_like(s))
    else:
        gap = h - 1 / (2 * beta)
        loss, slope = gap * gap, 2 * gap
    slope = slope / pairs
    return loss.mean().reshape(1), torch.cat([slope, -slope])


def _run_plain(op, case, s):
    if op == "denoise_preference":
        dtype = s["pred"].dtype
        miss = s["target"].float() - s["pred"].float()
        ref_miss = s["target"].float() - s["ref"].float()
        scale = -(1.0 / case["n"] if case["reduce"] == "mean" else 1.0)
        if s["weight"] is not None:
            scale = scale * s["weight"].double()
        ratio = scale * (miss * miss - ref_miss * ref_miss).sum(dim=1, dtype=torch.float64)
        loss, slope = _pair_terms(ratio, case)
        grad = (-2 * slope * scale * case["scale"]).float()[:, None] * miss
        return {"loss": loss.float(), "grad": grad.to(dtype), "ratio": ratio.float()}
    if op == "preference":
        where = _counted(s, s["logp"])
        gap = torch.where(where, s["logp"].float() - s["ref"].float(), torch.zeros((), device=where.device))
        ratio = gap.sum(dim=1, dtype=torch.float64)
        share = torch.ones_like(ratio)
        if case["reduce"] == "mean":
            share = 1.0 / where.sum(dim=1).clamp(min=1).double()
        ratio = ratio * share
        loss, slope = _pair_terms(ratio, case)
        grad = torch.where(where, (slope * share * case["scale"]).float()[:, None], torch.zeros((), device=where.device))
        return {"loss": loss.float(), "grad": grad.to(s["logp"].dtype), "ratio": ratio.float()}
    if op == "policy":
        where = _counted(s, s["logp"])
        zero = torch.zeros((), device=where.device)
        logp = torch.where(where, s["logp"].float(), zero)
        # the border of the clipping is decided in 64 bits
        log_ratio = logp.double() - torch.where(where, s["old"].float(), zero).double()
        over, under = log_ratio > math.log1p(0.28), log_ratio < math.log1p(-0.2)
        ratio = torch.exp(log_ratio.float())
        adv = s["advantages"] if case["per_step"] else s["advantages"][:, None]
        adv = torch.where(where, adv, zero)
        clipped = ((adv > 0) & over) | ((adv < 0) & under)
        bound = torch.where(over, torch.full_like(ratio, 1.28), torch.full_like(ratio, 0.8))
        term = -adv * torch.where(clipped, bound, ratio)
        slope = torch.where(clipped, zero, -adv * ratio)
        kl = torch.zeros_like(term)
        if case["kl"]:
            d = torch.where(where, s["ref"].float() - s["logp"].float(), zero)
            # exp(d) - d - 1 of a small d is lost in 32 bits
            kl = (torch.expm1(d.double()) - d.double()).float()
            slope = slope - case["kl"] * torch.expm1(d)
        count = where.sum()
        if case["reduce"] == "token":
            weight = (1.0 / count.clamp(min=1).double()).expand(where.shape[0])
        elif case["reduce"] == "row":
            weight = 1.0 / (where.sum(dim=1).clamp(min=1).double() * where.shape[0])
        else:
            weight = torch.ones(where.shape[0], dtype=torch.float64, device=where.device)
        objective = (torch.where(where, term, zero).sum(dim=1, dtype=torch.float64) * weight).sum()
        divergence = (torch.where(where, kl, zero).sum(dim=1, dtype=torch.float64) * weight).sum()
        loss = objective + case["kl"] * divergence
        share = (clipped & where).sum().double() / count.clamp(min=1).double()
        stats = torch.stack([objective, divergence, share, count.double()])
        grad = torch.where(where, slope * (weight * case["scale"]).float()[:, None], zero)
        return {"loss": loss.reshape(1).float(), "grad": grad.to(s["logp"].dtype), "stats": stats.float()}
    if op == "transition_forward":
        z = (s["x"].float() - s["mean"].float()) / s["std"][:, None]
        n = case["n"]
        logp = -0.5 * (z * z).sum(dim=1, dtype=torch.float64) - n * torch.log(s["std"].double()) - 0.5 * n * math.log(2 * math.pi)
        return {"logp": (logp / n if case["reduce"] == "mean" else logp).float()}
    if op == "transition_backward":
        factor = s["dlogp"] / (s["std"] * s["std"])
        if case["reduce"] == "mean":
            factor = factor / case["n"]
        return {"grad": ((s["x"].float() - s["mean"].float()) * factor[:, None]).to(s["mean"].dtype)}
    total = torch.stack([(t.float() * t.float()).sum(dtype=torch.float64) for t in s["grads"]]).sum()
    norm = torch.sqrt(total)
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * factor)
    return {"norm": norm.reshape(1).float(), "grads": s["flat"]}


def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2, "f16": 2}.get(case["dtype"])
    if op == "denoise_preference":
        n = 2 * case["pairs"] * case["n"]
        return {"bytes": 4 * n * size + 8 * case["pairs"], "flops": 8 * n}
    if op in ("preference", "policy"):
        rows = 2 * case["pairs"] if op == "preference" else case["rows"]
        places = rows * case["steps"]
        # the share of places that count: what a mask or a length leaves out need not be read
        fill = (0.76 if case["masked"] else 1.0) * (0.63 if case["ragged"] else 1.0)
        inputs = 2 if op == "preference" or not case["kl"] else 3
        read = fill * places * (inputs * size + (4 if case.get("per_step") else 0))
        return {"bytes": int(read + places * (size + (1 if case["masked"] else 0)) + 8 * rows),
                "flops": int(fill * places * (3 if op == "preference" else 30))}
    if op == "transition_forward":
        n = case["rows"] * case["n"]
        return {"bytes": 2 * n * size + 8 * case["rows"], "flops": 4 * n}
    if op == "transition_backward":
        n = case["rows"] * case["n"]
        return {"bytes": 3 * n * size + 8 * case["rows"], "flops": 2 * n}
    tensors = _clip_tensors(case)
    return {"bytes": sum(2 * n * (4 if d == "f32" else 2) for n, d in tensors), "flops": sum(3 * n for n, _ in tensors)}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------------
def _pair_exact(ratios, case):
    """mean loss and slopes, pair by pair with Python's floats"""
    pairs, beta, eps = case["pairs"], case["beta"], case["smoothing"]
    total, up = [], []
    for a, b in zip(ratios[:pairs], ratios[pairs:]):
        s = beta * (a - b)
        if case["kind"] == "sigmoid":
            def nls(v):                                # minus the logarithm of the logistic function
                return math.log1p(math.exp(-v)) if v > -30 else -v + math.log1p(math.exp(v))
            total.append((1 - eps) * nls(s) + eps * nls(-s))
            up.append(beta * (-(1 - eps) * math.exp(-nls(-s)) + eps * math.exp(-nls(s))))
        elif case["kind"] == "hinge":
            total.append(max(0.0, 1 - s))
            up.append(-beta if s < 1 else 0.0)
        else:
            total.append((a - b - 0.5 / beta) ** 2)
            up.append(2 * (a - b - 0.5 / beta))
    up = [u / pairs for u in up]
    return math.fsum(total) / pairs, up + [-u for u in up]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    double = {"dtype": torch.float64, "device": "cuda"}
    if op == "denoise_preference":
        factors = [(1.0 if s["weight"] is None else s["weight"][r].item()) / (case["n"] if case["reduce"] == "mean" else 1)
                   for r in range(2 * case["pairs"])]
        ratios = []
        for r, f in enumerate(factors):
            t, p, q = (s[k][r].double() for k in ("target", "pred", "ref"))
            ratios.append(f * ((p - q) * (2 * t - p - q)).sum().item())
        loss, slopes = _pair_exact(ratios, case)
        grad = torch.stack([2 * u * f * case["scale"] * (s["target"][r].double() - s["pred"][r].double())
                            for r, (u, f) in enumerate(zip(slopes, factors))])
        return {"loss": torch.tensor([loss], **double), "grad": grad, "ratio": torch.tensor(ratios, **double)}
    if op == "preference":
        rows, steps = s["logp"].shape
        grad, ratios, places = torch.zeros(rows, steps, **double), [], []
        for r in range(rows):
            keep = s["mask"][r].clone() if s["mask"] is not None else torch.ones(steps, dtype=torch.bool, device="cuda")
            if s["lengths"] is not None:
                keep[int(s["lengths"][r]):] = False
            places.append(keep)
            gaps = s["logp"][r][keep].double() - s["ref"][r][keep].double()
            ratios.append(gaps.sum().item() / (max(1, gaps.numel()) if case["reduce"] == "mean" else 1))
        loss, slopes = _pair_exact(ratios, case)
        for r, keep in enumerate(places):
            grad[r][keep] = case["scale"] * slopes[r] / (max(1, int(keep.sum())) if case["reduce"] == "mean" else 1)
        return {"loss": torch.tensor([loss], **double), "grad": grad, "ratio": torch.tensor(ratios, **double)}
    if op == "policy":
        rows, steps = s["logp"].shape
        keep = torch.ones(rows, steps, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"].clone()
        if s["lengths"] is not None:
            keep[torch.arange(steps, device="cuda").expand(rows, steps) >= s["lengths"][:, None].expand(rows, steps)] = False
        row, place = keep.nonzero(as_tuple=True)
        lp, old = s["logp"][row, place].double(), s["old"][row, place].double()
        a = (s["advantages"][row, place] if case["per_step"] else s["advantages"][row]).double()
        r = torch.exp(lp - old)
        free, held = r * a, r.clamp(0.8, 1.28) * a
        objective = -torch.minimum(free, held)
        slope = torch.where(held < free, torch.zeros_like(free), -free)
        kl = torch.zeros_like(a)
        if case["kl"]:
            d = s["ref"][row, place].double() - lp
            kl = torch.special.expm1(d) - d
            slope = slope + case["kl"] * (1 - torch.exp(d))
        per_row = torch.bincount(row, minlength=rows).double()
        n = row.numel()
        if case["reduce"] == "token":
            w = torch.full_like(a, 1.0 / max(1, n))
        elif case["reduce"] == "row":
            w = 1.0 / (per_row[row] * rows)
        else:
            w = torch.ones_like(a)
        grad = torch.zeros(rows, steps, **double)
        grad[row, place] = w * slope * case["scale"]
        parts = [(w * objective).sum().item(), (w * kl).sum().item(), (held < free).sum().item() / max(1, n), float(n)]
        return {"loss": torch.tensor([parts[0] + case["kl"] * parts[1]], **double), "grad": grad, "stats": torch.tensor(parts, **double)}
    if op == "transition_forward":
        out = []
        for x, mean, std in zip(s["x"], s["mean"], s["std"].tolist()):
            value = -((x.double() - mean.double()) ** 2).sum().item() / (2 * std * std) - case["n"] * math.log(std * math.sqrt(2 * math.pi))
            out.append(value / (case["n"] if case["reduce"] == "mean" else 1))
        return {"logp": torch.tensor(out, **double)}
    if op == "transition_backward":
        variance = s["std"].double() ** 2 * (case["n"] if case["reduce"] == "mean" else 1)
        return {"grad": s["dlogp"].double()[:, None] / variance[:, None] * (s["x"].double() - s["mean"].double())}
    norm = math.sqrt(math.fsum((t.double() ** 2).sum().item() for t in s["grads"]))
    factor = min(1.0, s["max_norm"] / (norm + 1e-6))
    flat = {d: torch.cat([t.double() * factor for t in s["grads"] if t.dtype == DTYPES[d]]) for d in s["flat"]}
    return {"norm": torch.tensor([norm], **double), "grads": flat}
