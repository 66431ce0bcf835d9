"""Cases of the losses on a classifier's log-probabilities: policy, preference and distillation.

Three operators, each differentiable, stand beside the fused linear
cross-entropy:

* ``policy_loss``: the clipped policy loss of tokens with a KL term to a
  reference policy, on per-token log-probabilities; ``linear_policy_loss``
  computes it from hidden states, classifier and token ids;
* ``preference_loss``: the preference loss of pairs of sequences (chosen,
  rejected) from the log-ratios of their tokens; ``linear_preference_loss``
  from hidden states;
* ``linear_distillation_loss``: the KL divergence from a teacher known by its
  top K log-probabilities per token to the student's full softmax.

Every case is one training pass: the loss and its gradients.  Sizes of the
linear forms are those of the workloads of ``mlx_cce.synthetic``, or generic.
"""

import math
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}

# What a float16 program scales its mean losses by, so that small gradients are not lost.
LOSS_SCALE = 256.0

# Share of the tokens of a sequence that its prompt takes, on average (masked).
PROMPT = 0.3


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # a few rollouts of one prompt, packed: launch latency is all there is
        dict(name="policy_group", op="policy", tokens=413, seqs=8, padded=False, dtype="float32",
             per_token=False, ref=True, reduction="sequence"),
        # an ordinary padded batch of rollouts
        dict(name="policy_batch", op="policy", tokens=64 * 1000, seqs=64, padded=True, dtype="float32",
             per_token=False, ref=True, reduction="mean"),
        # a whole collection of long rollouts in one pass, token advantages
        dict(name="policy_collection", op="policy", tokens=8388593, seqs=2048, padded=False, dtype="float32",
             per_token=True, ref=True, reduction="mean"),
        # the head of an 8-billion-parameter model: the loss from hidden states
        dict(name="linear_policy_head", op="linear_policy", tokens=4096, seqs=8, D=4096, V=128256,
             dtype="bfloat16", bias=False, ref=True, reduction="mean"),
        # a small head in 16-bit floats, odd number of rows
        dict(name="linear_policy_small", op="linear_policy", tokens=331, seqs=5, D=1024, V=32000,
             dtype="float16", bias=False, ref=False, reduction="sequence"),
        # one small batch of pairs: latency
        dict(name="preference_batch", op="preference", tokens=1543, pairs=4, dtype="float32", kind="sigmoid"),
        # a large batch of long pairs, stored in bfloat16
        dict(name="preference_collection", op="preference", tokens=6291437, pairs=1024, dtype="bfloat16",
             kind="ipo"),
        # pairs through a head with a bias and the largest vocabulary
        dict(name="linear_preference_head", op="linear_preference", tokens=2048, pairs=4, D=2304, V=256000,
             dtype="bfloat16", bias=True, kind="sigmoid"),
        # a small float32 student
        dict(name="distill_float32", op="distill", tokens=512, K=16, D=512, V=32000, dtype="float32", bias=False,
             T=1.0, tail=False, padding=0.0, reduction="mean"),
        # an ordinary student, softened teacher
        dict(name="distill_student", op="distill", tokens=1024, K=64, D=2048, V=128256, dtype="bfloat16",
             bias=False, T=2.0, tail=False, padding=0.0, reduction="mean"),
        # the largest: many teacher entries and the mass that they leave over
        dict(name="distill_tail", op="distill", tokens=4096, K=128, D=4096, V=128256, dtype="bfloat16", bias=False,
             T=1.0, tail=True, padding=0.0, reduction="mean"),
        # ragged sizes, a bias, absent entries, a weight of its own for every token
        dict(name="distill_ragged", op="distill", tokens=777, K=19, D=1032, V=50021, dtype="float16", bias=True,
             T=1.5, tail=True, padding=0.1, reduction="none"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["policy", "linear_policy", "preference", "linear_preference", "distill", "distill"])
    if op == "policy":
        n = _log(rng, 64, 8000000)
        padded = rng.random() < 0.3
        s = max(1, min(_log(rng, 1, 4096), n // 8))
        return dict(op=op, tokens=n // s * s if padded else n, seqs=s, padded=padded,
                    dtype=rng.choice(["float32", "float32", "bfloat16"]), per_token=rng.random() < 0.5,
                    ref=rng.random() < 0.7, reduction=rng.choice(["mean", "sequence", "sum"]))
    if op == "preference":
        n = _log(rng, 64, 6000000)
        return dict(op=op, tokens=n, pairs=max(1, min(_log(rng, 1, 2048), n // 16)),
                    dtype=rng.choice(["float32", "bfloat16", "float16"]), kind=rng.choice(["sigmoid", "hinge", "ipo"]))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float16", "float16", "float32"])
    D = 8 * _log(rng, 8, 512)
    V = _log(rng, 512, 128256)
    most = 4096 * 4096 * 128256 if dtype != "float32" else 1024 * 1024 * 32000
    n = _log(rng, 16, max(17, min(4096, most // (D * V))))
    c = dict(op=op, tokens=n, D=D, V=V, dtype=dtype, bias=rng.random() < 0.3)
    if op == "linear_policy":
        c.update(seqs=max(1, min(_log(rng, 1, 64), n // 8)), ref=rng.random() < 0.7,
                 reduction=rng.choice(["mean", "sequence", "sum"]))
    elif op == "linear_preference":
        c.update(pairs=max(1, min(_log(rng, 1, 32), n // 16)), kind=rng.choice(["sigmoid", "hinge"]))
    else:
        c.update(K=_log(rng, 1, 256), T=rng.choice([1.0, 1.5, 2.0, 4.0]), tail=rng.random() < 0.4,
                 padding=rng.choice([0.0, 0.1]), reduction=rng.choice(["mean", "sum", "none"]))
    return c


def work(case):
    n = case["tokens"]
    it = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "policy":
        # log-probabilities, their old and reference values, advantages, mask; the gradient
        b = n * (it * (3 if case["ref"] else 2) + 1 + it)
        b += 4 * (n if case["per_token"] else case["seqs"])
        return {"bytes": b, "flops": 30 * n}
    if case["op"] == "preference":
        return {"bytes": n * (2 * it + 1 + it), "flops": 6 * n}
    D, V = case["D"], case["V"]
    rows = n if case["op"] == "distill" else int(n * (1 - PROMPT))
    b = 2 * it * (n * D + V * D) + 8 * n
    if case["bias"]:
        b += 2 * it * V
    if case["op"] == "distill":
        b += n * case["K"] * 12
    return {"bytes": b, "flops": 6 * rows * D * V}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _cut(n, s, g):
    """Offsets of s sequences of random lengths that hold n tokens."""
    at = torch.randint(0, n + 1, (s - 1,), generator=g, device="cuda").sort().values
    edge = at.new_tensor([0]), at.new_tensor([n])
    return torch.cat([edge[0], at, edge[1]]).to(torch.int32)


def _prompt_mask(cu, n, g):
    """True for the tokens of the answers: each sequence begins with a prompt."""
    length = (cu[1:] - cu[:-1]).long()
    share = torch.rand(length.shape, generator=g, device="cuda") * (2 * PROMPT)
    first = cu[:-1].long() + (length * share).long()
    seq = torch.repeat_interleave(torch.arange(length.numel(), device="cuda"), length, output_size=n)
    return torch.arange(n, device="cuda") >= first[seq]


def _logp(n, g):
    """Log-probabilities of sampled tokens: many near 0, a long tail."""
    u = torch.rand(n, generator=g, device="cuda")
    return -(u.pow(4) * 6 + 1e-3 * torch.rand(n, generator=g, device="cuda"))


def _near(x, g, width, wide):
    """Another policy's log-probabilities: near those of x, a few of them far away."""
    n = x.numel()
    far = (torch.rand(n, generator=g, device="cuda") < 0.05).float()
    d = torch.randn(n, generator=g, device="cuda")
    return torch.clamp(x + d * (width + wide * far), max=0.0)


def _head(case, g):
    """Hidden states, classifier and bias with peaked softmaxes, and the tokens at the peaks."""
    n, D, V = case["tokens"], case["D"], case["V"]
    dt = DTYPES[case["dtype"]]
    c = torch.randn(V, D, generator=g, device="cuda") * 0.02
    e = torch.randn(n, D, generator=g, device="cuda")
    # four preferred tokens per row, small ids more often (as in a frequency-sorted vocabulary)
    u = torch.rand(n, 4, generator=g, device="cuda")
    ids = ((V + 1.0) ** u - 1).long().clamp(0, V - 1)
    high = 6 + 6 * torch.rand(n, 4, generator=g, device="cuda")
    for j in range(4):
        ct = c[ids[:, j]]
        e = e + ct * (high[:, j] / ct.square().sum(1)).unsqueeze(1)
    bias = torch.randn(V, generator=g, device="cuda") * 0.1 if case["bias"] else None
    return e.to(dt), c.to(dt), None if bias is None else bias.to(dt), ids


def _leaf(x):
    return None if x is None else x.detach().requires_grad_(True)


def prepare(case, seed):
    g = _gen(seed)
    n, op = case["tokens"], case["op"]
    s = dict(case)
    if op in ("policy", "preference"):
        dt = DTYPES[case["dtype"]]
        logp = _logp(n, g)
        seqs = case["seqs"] if op == "policy" else 2 * case["pairs"]
        if case.get("padded"):
            cu = torch.arange(seqs + 1, device="cuda", dtype=torch.int32) * (n // seqs)
        else:
            cu = _cut(n, seqs, g)
        s.update(cu=cu, mask=_prompt_mask(cu, n, g))
        if op == "policy":
            s["old"] = _near(logp, g, 0.05, 0.5).to(dt)
            s["ref_logp"] = _near(logp, g, 0.2, 1.0).to(dt) if case["ref"] else None
            s["adv"] = torch.randn(n if case["per_token"] else seqs, generator=g, device="cuda")
            if case["padded"]:
                shape = (seqs, n // seqs)
                s["mask"] = s["mask"].view(shape)
                s["old"] = s["old"].view(shape)
                s["ref_logp"] = None if s["ref_logp"] is None else s["ref_logp"].view(shape)
                s["adv"] = s["adv"].view(shape) if case["per_token"] else s["adv"]
                logp = logp.view(shape)
        else:
            s["ref_logp"] = _near(logp, g, 0.1, 0.5).to(dt)
        s["logp"] = _leaf(logp.to(dt))
        return s
    e, c, bias, ids = _head(case, g)
    s.update(e=_leaf(e), c=_leaf(c), bias=_leaf(bias), grad=None)
    if case["dtype"] == "float16" and case.get("reduction") != "sum":
        s["grad"] = torch.tensor(LOSS_SCALE, device="cuda")
    if op == "distill":
        K, V, T = min(case["K"], case["V"]), case["V"], case["T"]
        top, where = [], []
        for r in range(0, n, 256):  # the teacher: the student's logits, sharpened and disturbed
            z = (e[r:r + 256] @ c.t()).float()
            z = 1.1 * z + 0.5 * torch.randn(z.shape, generator=g, device="cuda")
            v, i = z.log_softmax(1).topk(K, dim=1)
            top.append(v)
            where.append(i)
        s["teacher_logp"], s["teacher_ids"] = torch.cat(top), torch.cat(where)
        if case["padding"]:
            gone = torch.rand(n, K, generator=g, device="cuda") < case["padding"]
            gone[:, 0] = False
            s["teacher_ids"] = torch.where(gone, torch.full_like(s["teacher_ids"], -1), s["teacher_ids"])
        s["mask"] = torch.rand(n, generator=g, device="cuda") >= 0.05
        if case["reduction"] == "none":
            s["grad"] = torch.randn(n, generator=g, device="cuda")
        return s
    seqs = case["seqs"] if op == "linear_policy" else 2 * case["pairs"]
    cu = _cut(n, seqs, g)
    mask = _prompt_mask(cu, n, g)
    pick = torch.randint(0, 4, (n, 1), generator=g, device="cuda")
    targets = ids.gather(1, pick).squeeze(1)
    logp, cf = torch.empty(n, device="cuda"), c.float()
    for r in range(0, n, 256):
        z = e[r:r + 256].float() @ cf.t()
        if bias is not None:
            z = z + bias.float()
        logp[r:r + 256] = z.log_softmax(1).gather(1, targets[r:r + 256].unsqueeze(1)).squeeze(1)
    s.update(cu=cu, mask=mask, targets=torch.where(mask, targets, torch.full_like(targets, -100)))
    if op == "linear_policy":
        # log-probabilities from 16-bit products carry errors of 1e-6: no token
        # lies so near to the clipping border that these decide its gradient
        old = _near(logp, g, 0.05, 0.5)
        for border in (math.log(1.0 - CLIP_LOW), math.log(1.0 + CLIP_HIGH)):
            old = torch.where((logp - old - border).abs() < 1e-4, old - 1e-3, old)
        s["old"] = old
        s["ref_logp"] = _near(logp, g, 0.2, 1.0) if case["ref"] else None
        s["adv"] = torch.randn(seqs, generator=g, device="cuda")
    else:
        s["ref_logp"] = _near(logp, g, 0.1, 0.5)
    return s


# ---------------------------------------------------------------------------
# the operators in plain form
# ---------------------------------------------------------------------------

CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.28, 0.04
BETA = 0.1


def _seq_of(cu, n):
    """The sequence of each token."""
    return torch.searchsorted(cu[1:].contiguous(), torch.arange(n, device=cu.device, dtype=cu.dtype), right=True)


def _plain_policy(logp, old, ref, adv, mask, seq, seqs, reduction):
    """Loss, its gradient by logp, mean KL and share of clipped tokens.  The
    differences and the ratios next to the clipping border are taken in 64 bits."""
    m = mask.reshape(-1)
    x = logp.reshape(-1).double()
    a = adv.reshape(-1) if adv.numel() == x.numel() else adv[seq]
    d = x - old.reshape(-1).double()
    ratio = torch.exp(d)
    pos = a > 0
    open_ = torch.where(pos, ratio <= 1.0 + CLIP_HIGH, ratio >= 1.0 - CLIP_LOW) | (a == 0)
    bounded = torch.where(pos, torch.clamp(ratio, max=1.0 + CLIP_HIGH), torch.clamp(ratio, min=1.0 - CLIP_LOW))
    loss = -(bounded.float() * a)
    grad = torch.where(open_, -(ratio.float() * a), torch.zeros_like(a))
    kl = torch.zeros_like(loss)
    if ref is not None:
        q = ref.reshape(-1).double() - x
        kl = (torch.expm1(q) - q).float()
        loss = loss + KL * kl
        grad = grad - KL * torch.expm1(q).float()
    zero = torch.zeros_like(loss)
    loss, grad, kl = torch.where(m, loss, zero), torch.where(m, grad, zero), torch.where(m, kl, zero)
    count = m.sum().clamp(min=1)
    if reduction == "mean":
        weight = (1.0 / count).expand_as(loss)
    elif reduction == "sum":
        weight = torch.ones_like(loss)
    else:
        per = torch.zeros(seqs, device=m.device).index_add_(0, seq, m.float())
        weight = (1.0 / (per.clamp(min=1) * (per > 0).sum().clamp(min=1)))[seq]
    total = (loss.double() * weight.double()).sum().float()
    clipped = ((~open_) & m).sum() / count
    return total, grad * weight, (kl.double().sum() / count).float(), clipped.float()


def _plain_preference(logp, ref, mask, seq, pairs, kind):
    m = mask.reshape(-1)
    d = torch.where(m, logp.reshape(-1).float() - ref.reshape(-1).float(), torch.zeros(m.numel(), device=m.device))
    per = torch.zeros(2 * pairs, device=m.device, dtype=torch.float64).index_add_(0, seq, d.double())
    ratio = (per[:pairs] - per[pairs:]).float()
    h = BETA * ratio
    if kind == "sigmoid":
        loss = torch.clamp(-h, min=0) + torch.log1p(torch.exp(-h.abs()))
        slope = -BETA / (1 + torch.exp(h))
    elif kind == "hinge":
        loss = torch.clamp(1 - h, min=0)
        slope = torch.where(h < 1, -BETA, 0.0)
    else:
        loss = (ratio - 0.5 / BETA).square()
        slope = 2 * (ratio - 0.5 / BETA)
    slope = slope / pairs
    grad = torch.cat([slope, -slope])[seq] * m
    rewards = BETA * per.float()
    return loss.mean(), grad, rewards[:pairs], rewards[pairs:]


def _plain_logits(s):
    z = s["e"].float() @ s["c"].float().t()
    return z if s["bias"] is None else z + s["bias"].float()


def _plain_grads(s, dz):
    if s["grad"] is not None:
        dz = dz.mul_(s["grad"].reshape(-1, 1))
    out = {"grad_e": (dz @ s["c"].float()).to(s["e"].dtype), "grad_c": (dz.t() @ s["e"].float()).to(s["c"].dtype)}
    if s["bias"] is not None:
        out["grad_bias"] = dz.sum(0).to(s["bias"].dtype)
    return out


def _plain_token_logp(z, targets):
    """Log-probabilities of the targets (0 where there is none), and the softmax in z's place."""
    at = targets.clamp(min=0).unsqueeze(1)
    top = z.max(1, keepdim=True).values
    lse = (z - top).exp_().sum(1, keepdim=True).log_() + top
    logp = (z.gather(1, at) - lse).squeeze(1)
    return logp, z.sub_(lse).exp_(), at


def _plain_softmax_grad(q, at, g):
    """d(sum g logp)/dz = g (onehot - softmax), in q's place."""
    q.mul_(-g.unsqueeze(1))
    return q.scatter_add_(1, at, g.unsqueeze(1))


def _plain_distill(s):
    T, V = s["T"], s["V"]
    z = _plain_logits(s)
    if T != 1.0:
        z = z.div_(T)
    ids, t = s["teacher_ids"], s["teacher_logp"]
    there = ids >= 0
    at = ids.clamp(min=0)
    if s["tail"]:
        p = torch.where(there, t.double().exp(), 0.0)
        rest = (1 - p.sum(1)).clamp(min=0).float()
        p = p.float()
        logt = t
    else:
        logt = torch.where(there, t / T, -math.inf)
        logt = logt - logt.max(1, keepdim=True).values
        logt = logt - logt.exp().sum(1, keepdim=True).log()
        p = logt.exp()
        rest = torch.zeros_like(p[:, 0])
    top = z.max(1, keepdim=True).values
    lse = (z - top).exp_().sum(1, keepdim=True).log_() + top
    logq = z.gather(1, at) - lse
    zero = torch.zeros_like(p)
    loss = torch.where(p > 0, p * (logt - logq), zero).sum(1)
    whole = p.sum(1) + rest
    dz = z.sub_(lse).exp_()
    if s["tail"]:
        other = dz.clone()  # the student's mass outside of the teacher's entries
        rows = torch.arange(ids.shape[0], device=ids.device).unsqueeze(1).expand_as(ids)
        other[rows[there], at[there]] = 0.0
        qrest = other.sum(1)
        has = rest > 0
        loss = loss + torch.where(has, rest * (rest.log() - qrest.log()), 0.0)
        dz.mul_(whole.unsqueeze(1)).sub_(other.mul_(torch.where(has, rest / qrest, 0.0).unsqueeze(1)))
    dz.scatter_add_(1, at, -torch.where(there, p, zero))
    m = s["mask"]
    loss = torch.where(m, loss, 0.0)
    if s["reduction"] == "mean":
        count = m.sum().clamp(min=1)
        weight = m / count
        total = (loss.double().sum() / count).float()
    elif s["reduction"] == "sum":
        weight, total = m.float(), loss.double().sum().float()
    else:
        weight, total = m.float(), loss
    return {"loss": total, **_plain_grads(s, dz.mul_((weight / T).unsqueeze(1)))}


@torch.no_grad()
def _plain(s):
    op = s["op"]
    if op == "distill":
        return _plain_distill(s)
    seq = _seq_of(s["cu"], s["tokens"])
    if op == "policy":
        loss, grad, kl, clipped = _plain_policy(s["logp"], s["old"], s["ref_logp"], s["adv"], s["mask"], seq,
                                                s["seqs"], s["reduction"])
        return {"loss": loss, "grad": grad.to(s["logp"].dtype).view_as(s["logp"]), "kl": kl, "clipped": clipped}
    if op == "preference":
        loss, grad, chosen, rejected = _plain_preference(s["logp"], s["ref_logp"], s["mask"], seq, s["pairs"],
                                                         s["kind"])
        return {"loss": loss, "grad": grad.to(s["logp"].dtype), "chosen": chosen, "rejected": rejected}
    logp, q, at = _plain_token_logp(_plain_logits(s), s["targets"])
    m = s["targets"] >= 0
    if op == "linear_policy":
        loss, grad, kl, clipped = _plain_policy(logp, s["old"], s["ref_logp"], s["adv"], m, seq, s["seqs"],
                                                s["reduction"])
        out = {"loss": loss, "kl": kl, "clipped": clipped}
    else:
        loss, grad, chosen, rejected = _plain_preference(logp, s["ref_logp"], m, seq, s["pairs"], s["kind"])
        out = {"loss": loss}
    return {**out, **_plain_grads(s, _plain_softmax_grad(q, at, grad))}


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------

def _framework():
    if "mlx-cross-entropy_b200" not in sys.path:
        sys.path.insert(1, "mlx-cross-entropy_b200")
    import mlx_cce
    return mlx_cce


def _own_grads(s, out, loss, upstream=None):
    leaves = [("grad_e", s["e"]), ("grad_c", s["c"])] + ([] if s["bias"] is None else [("grad_bias", s["bias"])])
    grads = torch.autograd.grad(loss, [x for _, x in leaves], upstream)
    return {**out, **{k: g for (k, _), g in zip(leaves, grads)}}


def _own(s):
    cce = _framework()
    op = s["op"]
    if op == "policy":
        loss, stats = cce.policy_loss(s["logp"], s["old"], s["adv"], ref_logp=s["ref_logp"], mask=s["mask"],
                                      cu_seqlens=None if s["padded"] else s["cu"], clip=CLIP_LOW,
                                      clip_high=CLIP_HIGH, kl_coef=KL if s["ref"] else 0.0,
                                      reduction=s["reduction"], return_stats=True)
        (grad,) = torch.autograd.grad(loss, [s["logp"]])
        return {"loss": loss.detach(), "grad": grad, "kl": stats.kl, "clipped": stats.clip_fraction}
    if op == "preference":
        loss, rewards = cce.preference_loss(s["logp"], s["ref_logp"], mask=s["mask"], cu_seqlens=s["cu"], beta=BETA,
                                            loss_type=s["kind"], return_rewards=True)
        (grad,) = torch.autograd.grad(loss, [s["logp"]])
        return {"loss": loss.detach(), "grad": grad, "chosen": rewards.chosen, "rejected": rewards.rejected}
    if op == "linear_policy":
        loss, stats = cce.linear_policy_loss(s["e"], s["c"], s["targets"], s["old"], s["adv"], s["bias"],
                                             ref_logp=s["ref_logp"], cu_seqlens=s["cu"], clip=CLIP_LOW,
                                             clip_high=CLIP_HIGH, kl_coef=KL if s["ref"] else 0.0,
                                             reduction=s["reduction"], return_stats=True)
        return _own_grads(s, {"loss": loss.detach(), "kl": stats.kl, "clipped": stats.clip_fraction}, loss, s["grad"])
    if op == "linear_preference":
        loss = cce.linear_preference_loss(s["e"], s["c"], s["targets"], s["ref_logp"], s["bias"],
                                          cu_seqlens=s["cu"], beta=BETA, loss_type=s["kind"])
        return _own_grads(s, {"loss": loss.detach()}, loss, s["grad"])
    loss = cce.linear_distillation_loss(s["e"], s["c"], s["teacher_ids"], s["teacher_logp"], s["bias"],
                                        temperature=s["T"], tail=s["tail"], mask=s["mask"], reduction=s["reduction"])
    return _own_grads(s, {"loss": loss.detach()}, loss, s["grad"])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# 64 bits, from the definitions, differentiated by autograd
# ---------------------------------------------------------------------------

def _f64_policy(x, s, m, seq, seqs):
    """Sum of weight * loss over the tokens x, with the statistics."""
    a = s["adv"].reshape(-1).double()
    a = a if a.numel() == x.numel() else a[seq]
    old = s["old"].reshape(-1).double()
    r = torch.exp(x - old)
    token = -torch.minimum(r * a, torch.clamp(r, 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * a)
    kl = torch.zeros_like(x)
    if s["ref"]:
        q = s["ref_logp"].reshape(-1).double() - x
        kl = torch.exp(q) - 1 - q
        token = token + KL * kl
    count = max(int(m.sum()), 1)
    if s["reduction"] == "sequence":
        per = torch.bincount(seq[m], minlength=seqs)
        w = 1.0 / (per[seq].double() * int((per > 0).sum()))
    else:
        w = torch.full_like(x, 1.0 if s["reduction"] == "sum" else 1.0 / count)
    cut = ((a > 0) & (r > 1.0 + CLIP_HIGH)) | ((a < 0) & (r < 1.0 - CLIP_LOW))
    return (token * w)[m].sum(), kl[m].sum().detach() / count, (cut & m).double().sum() / count


def _f64_preference(x, s, m, seq):
    pairs = s["pairs"]
    d = torch.where(m, x - s["ref_logp"].reshape(-1).double(), torch.zeros_like(x))
    per = torch.zeros(2 * pairs, dtype=torch.float64, device=x.device).index_add(0, seq, d)
    gap = per[:pairs] - per[pairs:]
    if s["kind"] == "sigmoid":
        loss = -torch.nn.functional.logsigmoid(BETA * gap)
    elif s["kind"] == "hinge":
        loss = torch.relu(1 - BETA * gap)
    else:
        loss = (gap - 1 / (2 * BETA)) ** 2
    return loss.mean(), (BETA * per[:pairs]).detach(), (BETA * per[pairs:]).detach()


def _f64_tokens(s, x, m):
    cu = s["cu"].long()
    seq = torch.repeat_interleave(torch.arange(cu.numel() - 1, device=cu.device), cu[1:] - cu[:-1])
    if "policy" in s["op"]:
        loss, kl, cut = _f64_policy(x, s, m, seq, s["seqs"])
        return loss, {"kl": kl, "clipped": cut}
    loss, chosen, rejected = _f64_preference(x, s, m, seq)
    return loss, {"chosen": chosen, "rejected": rejected}


def exact(case, seed):
    s = prepare(case, seed)
    op, n = case["op"], case["tokens"]
    if op in ("policy", "preference"):
        x = s["logp"].detach().reshape(-1).double().requires_grad_(True)
        loss, more = _f64_tokens(s, x, s["mask"].reshape(-1))
        (grad,) = torch.autograd.grad(loss, [x])
        return {"loss": loss.detach(), "grad": grad.view_as(s["logp"]), **more}
    e, c = s["e"].detach().double(), s["c"].detach().double()
    b = None if s["bias"] is None else s["bias"].detach().double()
    T = case.get("T", 1.0)
    step = 512

    def logits(r):
        z = e[r:r + step] @ c.t()
        return (z if b is None else z + b) / T

    out = {}
    if op == "distill":
        m = s["mask"]
        weight = m.double() / (max(int(m.sum()), 1) if case["reduction"] == "mean" else 1)
        rows = torch.empty(n, dtype=torch.float64, device="cuda")

        def block(r, z):
            ids, t = s["teacher_ids"][r:r + step], s["teacher_logp"][r:r + step].double()
            there = ids >= 0
            lq = torch.log_softmax(z, 1)
            if case["tail"]:
                p = torch.where(there, t.exp(), 0.0)
                rest = (1 - p.sum(1)).clamp(min=0)
            else:
                p = torch.softmax(torch.where(there, t / T, -math.inf), 1)
                rest = torch.zeros_like(p[:, 0])
            per = torch.special.xlogy(p, p).sum(1) - (p * lq.gather(1, ids.clamp(min=0))).sum(1)
            if case["tail"]:
                inside = torch.zeros_like(lq, dtype=torch.bool)
                i, k = there.nonzero(as_tuple=True)
                inside[i, ids[i, k]] = True
                outside = torch.where(inside, -math.inf, lq).logsumexp(1)
                per = per + torch.where(rest > 0, torch.special.xlogy(rest, rest) - rest * outside, 0.0)
            rows[r:r + step] = torch.where(m[r:r + step], per, 0.0).detach()
            return (torch.where(m[r:r + step], per, 0.0) * weight[r:r + step]).sum()
    else:
        at = s["targets"].clamp(min=0)
        x = torch.cat([torch.log_softmax(logits(r), 1).gather(1, at[r:r + step, None])[:, 0]
                       for r in range(0, n, step)]).requires_grad_(True)
        loss, out = _f64_tokens(s, x, s["targets"] >= 0)
        out = out if op == "linear_policy" else {}
        out["loss"] = loss.detach()
        (gx,) = torch.autograd.grad(loss, [x])

        def block(r, z):
            return (torch.log_softmax(z, 1).gather(1, at[r:r + step, None])[:, 0] * gx[r:r + step]).sum()

    ge, gc, gb = torch.empty_like(e), torch.zeros_like(c), torch.zeros(case["V"], dtype=torch.float64, device="cuda")
    for r in range(0, n, step):
        z = logits(r).requires_grad_(True)
        (dz,) = torch.autograd.grad(block(r, z), [z])
        dz = dz / T
        if s["grad"] is not None:
            dz = dz * (s["grad"][r:r + step, None] if s["grad"].dim() else s["grad"]).double()
        ge[r:r + step] = dz @ c
        gc.addmm_(dz.t(), e[r:r + step])
        gb += dz.sum(0)
    if op == "distill":
        out["loss"] = rows if case["reduction"] == "none" else (rows * weight).sum()
    out.update(grad_e=ge, grad_c=gc)
    if b is not None:
        out["grad_bias"] = gb
    return out
