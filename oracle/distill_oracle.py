"""CPU oracle: distillation of a retriever's softmax from a teacher's top list, in 64 bits (no counterpart in the reference).

TEST INFRASTRUCTURE ONLY -- see oracle/__init__.py.
"""
from __future__ import annotations

import torch

__all__ = ["distill_ref", "distill_bounds"]


def _shares(index, score, teacher_temp):
    live = (index >= 0) & (score != float("-inf"))
    v = torch.where(live, score.double() / teacher_temp, torch.tensor(float("-inf"), dtype=torch.float64))
    some = live.any(1)
    v = torch.where(some[:, None], v, 0.0)
    t = torch.softmax(v, 1) * live * some[:, None]
    return live, some, t


def distill_ref(q, cand, temp, index, score, teacher_temp, n_local, grad_out=1.0):
    """dict of loss, agree, dq, dp (the first n_local candidates), dtemp, and what the bounds need (z, p, t, g), from the closed form."""
    q, c = q.double(), cand.double()
    B, T = q.shape[0], c.shape[0]
    s = q @ c.t()
    z = s / temp
    lse = torch.logsumexp(z, 1)
    live, some, t = _shares(index, score, teacher_temp)
    rows = max(1, int(some.sum()))
    target = torch.zeros(B, T, dtype=torch.float64)
    for b in range(B):
        for i in torch.nonzero(live[b])[:, 0].tolist():
            target[b, int(index[b, i])] += t[b, i]
    ent = torch.where(t > 0, t * torch.log(torch.where(t > 0, t, 1.0)), 0.0).sum(1)
    row = torch.where(some, ent - (target * (z - lse[:, None])).sum(1), 0.0)
    best = torch.where(live, score.double(), float("-inf")).argmax(1)
    pick = index[torch.arange(B), best]
    agree = float(((z.argmax(1) == pick) & some).sum()) / rows
    p = torch.exp(z - lse[:, None])
    g = (p - target) * some[:, None] * (grad_out / rows)
    return {"loss": row.sum() / rows, "agree": agree, "dq": g @ c / temp, "dp": (g.t() @ q)[:n_local] / temp,
            "dtemp": -(g * z).sum() / temp, "z": z, "lse": lse, "p": p, "target": target, "g": g, "some": some, "rows": rows}


def distill_bounds(r, q, cand, temp, score, teacher_temp, n_local, k, bf16, grad_out=1.0):
    """How far fp32 arithmetic can be from `r`: u = 2^-24 is half a step of fp32; a sum of n terms in any order is off by at most n u times the
    sum of the terms' magnitudes; what the products of bf16 parts leave out is below 2^-21 of a product (mid lo + lo mid + lo lo with
    |mid| <= 2^-7, |lo| <= 2^-15 of the value), what the products of fp16 parts leave out is at most 2^-21 (each value is off by 2^-23 of it and
    by 2^-36, lo lo is 2^-22 of a product); exp and log are off by at most 4 steps (8 u).  `cand` rows of magnitude 2^-10 and more carry
    the 2^-36 as 2^-26 of the row's largest value: `floor` below."""
    u, lost = 2.0 ** -24, 0.0 if bf16 else 2.0 ** -21
    floor = 0.0 if bf16 else 2.0 ** -26
    q, c = q.double().abs(), cand.double().abs()
    B, D = q.shape
    T = c.shape[0]
    qm, cm = q.amax(1, keepdim=True), c.amax(1, keepdim=True)
    dz = (((D + 16) * u + lost) * (q @ c.t()) + floor * (qm @ c.sum(1, keepdim=True).t() + q.sum(1, keepdim=True) @ cm.t())) / temp \
        + 3 * u * r["z"].abs()
    worst = dz.max(1)[0]
    l_err = worst + (T + 20) * u + 8 * u * r["lse"].abs()
    live = torch.isfinite(score)
    span = torch.where(live, score.double(), 0.0)
    span = (span.amax(1) - span.amin(1)).abs() / teacher_temp + 1.0
    t_rel = (3 * u * span + (k + 24) * u)[:, None]
    p_rel = (dz + l_err[:, None]) + 2 * u * (r["z"].abs() + r["lse"].abs()[:, None]) + 16 * u
    row = l_err + worst + t_rel[:, 0] * (span + r["z"].abs().amax(1) + r["lse"].abs()) * 2 + (k + 8) * u * (r["z"].abs().amax(1) + span + r["lse"].abs())
    loss = float((row * r["some"]).sum() / r["rows"]) + (B + 4) * u * float(r["loss"].abs())
    scale = abs(grad_out) / r["rows"]
    dg = (r["p"] * p_rel + r["target"] * t_rel + 6 * u * (r["p"] + r["target"])) * r["some"][:, None] * scale
    ga = r["g"].abs()
    cut = 2.0 ** -15 if bf16 else lost                            # g in two parts: hi 8 bits, mid 8 bits
    dq = (dg @ c + ((T + 16) * u + cut) * (ga @ c)) / temp
    dp = (dg.t() @ q + ((B + 16) * u + cut) * (ga.t() @ q))[:n_local] / temp
    if not bf16:
        # fp16 parts: a gradient of the logits is carried to 2^-50 of 1, a candidate or query to 2^-26 of its row's largest value
        w = r["some"][:, None] * scale
        dq = dq + ((2.0 ** -50) * w * c.sum(0, keepdim=True) + floor * (ga @ cm)) / temp
        dp = dp + ((2.0 ** -50) * (w * q).sum(0, keepdim=True) + floor * (ga.t() @ qm)[:n_local]) / temp
    if bf16:
        dq, dp = dq * 1.01 + 2.0 ** -8 * r["dq"].abs(), dp * 1.01 + 2.0 ** -8 * r["dp"].abs()
    dt = ((dg * r["z"].abs() + ga * dz).sum() + (B * T + 16) * u * (ga * r["z"].abs()).sum()) / temp
    return {"loss": loss, "dq": dq, "dp": dp, "dtemp": float(dt)}
