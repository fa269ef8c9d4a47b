"""Layer normalisation, candidate routing and distillation from top logits: the cases they are measured on, and the
operators in their plain form (elementary torch operations), beside the calls a program makes of this package.

The three belong to one training step: a latent or a batch of tokens is normalised, a head scores candidates (poses of
an object, views of a grid), routing picks the few that are rendered and their weights, and the scores learn from the
rendered ones (a teacher that knows the logits of its top candidates only)."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
INF = float("inf")


# ---- cases ---------------------------------------------------------------------------------------------------------

def _ln(rows, cols, dtype, params, step, affine="both", pad=0):
    return {"op": "layer_norm", "rows": rows, "cols": cols, "dtype": dtype, "params": params, "step": step,
            "affine": affine, "pad": pad}


def _route(rows, cands, top_k, dtype, score, step, bias=False, groups=1, top_groups=1, group_score="max",
           renormalize=True, scale=1.0, masked=0.0):
    return {"op": "route", "rows": rows, "cands": cands, "top_k": top_k, "dtype": dtype, "score": score, "step": step,
            "bias": bias, "groups": groups, "top_groups": top_groups, "group_score": group_score,
            "renormalize": renormalize, "scale": scale, "masked": masked}


def _distill(rows, cols, top, dtype, step, temperature=1.0, reduction="mean", empty=0.0, teacher="f32"):
    return {"op": "distill", "rows": rows, "cols": cols, "top": top, "dtype": dtype, "step": step,
            "temperature": temperature, "reduction": reduction, "empty": empty, "teacher": teacher}


def listed():
    return [
        # the latent of one batch of 32 images (examples/train_step.py), at inference: one small launch
        dict(_ln(32, 128, "f32", "f32", False), name="norm_latent_forward"),
        # the latents of 32 images under 6 candidate poses each, in training
        dict(_ln(192, 512, "f32", "f32", True), name="norm_candidates_step"),
        # per-vertex offsets of the 642-vertex icosphere (642 * 3 columns) in rows cut out of a wider head's output
        dict(_ln(6151, 1926, "f16", "f32", True, pad=35), name="norm_offsets_step"),
        # few, very long rows: feature maps normalised over channels and pixels together
        dict(_ln(129, 65536, "f32", "f32", False), name="norm_maps_forward"),
        # a large batch of image tokens in training
        dict(_ln(65536, 1024, "bf16", "bf16", True), name="norm_tokens_step"),
        # two of six candidate poses for each of 32 images, in training: the smallest call there is
        dict(_route(32, 6, 2, "f32", "softmax", True), name="route_poses_step"),
        # choosing among 64 candidates in groups of 8, some of them ruled out; the choice alone
        dict(_route(4099, 64, 6, "bf16", "sigmoid", False, True, 8, 3, "max", True, 2.5, 0.1), name="route_groups_forward"),
        # every token of a large batch among 256 candidates, in training
        dict(_route(131072, 256, 8, "bf16", "sigmoid", True, True, 8, 4, "top2", True, 2.5), name="route_tokens_step"),
        # the scores of six poses learn from the two rendered ones
        dict(_distill(32, 6, 2, "f32", True), name="distill_poses_step"),
        # a grid of viewpoints as classes, an odd number of them (rows start at any 2-byte address), some slots empty
        dict(_distill(4096, 8101, 32, "f16", True, 2.0, "none", 0.1), name="distill_views_step"),
        # three rows over many classes, the loss alone: too few rows to fill the card by rows
        dict(_distill(3, 131071, 100, "bf16", False, 1.5, "none"), name="distill_few_rows_forward"),
        # a large batch over many classes, in training
        dict(_distill(8192, 32768, 64, "bf16", True), name="distill_wide_step"),
    ]


def _log_int(rng, lo, hi):
    """a whole number between lo and hi, spread over the logarithm"""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16"])
    step = rng.random() < 0.6
    op = rng.choice(["layer_norm", "route", "distill"])
    if op == "layer_norm":
        cols = _log_int(rng, 32, 65536)
        rows = _log_int(rng, 1, min(65536, (1 << 25) // cols))
        return _ln(rows, cols, dtype, rng.choice([dtype, "f32"]), step, rng.choice(["both", "both", "weight", "none"]),
                   rng.choice([0, 0, rng.randint(1, 64)]))
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = _log_int(rng, 2, 1024 // groups)
        cands = groups * per
        rows = _log_int(rng, 1, min(131072, (1 << 24) // cands))
        top_groups = rng.randint(1, groups)
        return _route(rows, cands, rng.randint(1, min(32, top_groups * per)), dtype, rng.choice(["softmax", "sigmoid"]),
                      step, rng.random() < 0.6, groups, top_groups, rng.choice(["max", "top2"]), rng.random() < 0.8,
                      rng.choice([1.0, 2.5]), rng.choice([0.0, 0.0, 0.2]))
    cols = _log_int(rng, 6, 131072)
    rows = _log_int(rng, 1, min(32768, (1 << 26) // cols))
    return _distill(rows, cols, rng.randint(1, min(128, cols)), dtype, step, rng.choice([0.7, 1.0, 2.0, 4.0]),
                    rng.choice(["mean", "sum", "none"]), rng.choice([0.0, 0.0, 0.3]), rng.choice(["f32", dtype]))


# ---- inputs --------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = TYPES[case["dtype"]]
    M = case["rows"]
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    uniform = lambda *shape: torch.rand(*shape, generator=g, device=dev)  # noqa: E731
    s = {"case": dict(case)}
    if case["op"] == "layer_norm":
        D, wt = case["cols"], TYPES[case["params"]]
        wide = normal(M, D + case["pad"]) * (0.5 + uniform(M, 1)) + normal(M, 1)  # rows of differing mean and spread
        s["x"] = wide.to(dt)[:, :D].requires_grad_(case["step"])
        s["w"] = (1.0 + 0.2 * normal(D)).to(wt).requires_grad_(case["step"]) if case["affine"] != "none" else None
        s["b"] = (0.2 * normal(D)).to(wt).requires_grad_(case["step"]) if case["affine"] == "both" else None
        s["dy"] = normal(M, D).to(dt) if case["step"] else None
    elif case["op"] == "route":
        E = case["cands"]
        logits = 1.5 * normal(M, E) + 0.5 * normal(E)  # some candidates are liked by most rows
        if case["masked"] > 0:
            logits = logits.masked_fill(uniform(M, E) < case["masked"], -INF)
            logits = logits.masked_fill(uniform(M, 1) < 0.05, -INF)  # rows that nothing is left for
        s["logits"] = logits.to(dt).requires_grad_(case["step"])
        s["bias"] = 0.1 * normal(E) if case["bias"] else None
        s["dw"] = normal(M, case["top_k"]) if case["step"] else None
    else:
        V, k = case["cols"], case["top"]
        z = 2.0 * normal(M, V)
        s["logits"] = z.to(dt).requires_grad_(case["step"])
        z = z + 1.5 * normal(M, V)  # the teacher agrees with the student in part
        top = z.topk(k, dim=1)
        index = top.indices
        if case["empty"] > 0:
            index = index.masked_fill(uniform(M, k) < case["empty"], -1)
            index = index.masked_fill(uniform(M, 1) < 0.05, -1)  # rows without a teacher
        s["teacher"], s["index"] = top.values.to(TYPES[case["teacher"]]), index
        s["g"] = normal(M) if case["step"] and case["reduction"] == "none" else None
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _own_layer_norm, "route": _own_route, "distill": _own_distill}[op](state, state["case"])
    with torch.no_grad():
        return {"layer_norm": _plain_layer_norm, "route": _plain_route, "distill": _plain_distill}[op](state, state["case"])


def _own_layer_norm(s, c):
    from unicorn_amd.normalization import layer_norm
    y = layer_norm(s["x"], s["w"], s["b"], eps=1e-5)
    if not c["step"]:
        return {"y": y}
    wanted = [t for t in (s["x"], s["w"], s["b"]) if t is not None]
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, wanted, s["dy"]))}


def _own_route(s, c):
    from unicorn_amd.routing import route_candidates
    r = route_candidates(s["logits"], c["top_k"], bias=s["bias"], score=c["score"], groups=c["groups"],
                         top_groups=c["top_groups"], group_score=c["group_score"], renormalize=c["renormalize"],
                         scale=c["scale"])
    out = {"weights": r.weights.detach(), "indices": r.indices, "counts": r.counts}
    if c["step"]:
        out["grad"] = torch.autograd.grad(r.weights, s["logits"], s["dw"])[0]
    return out


def _own_distill(s, c):
    from unicorn_amd.distillation import distill_top_logits
    loss = distill_top_logits(s["logits"], s["teacher"], s["index"], temperature=c["temperature"],
                              reduction=c["reduction"])
    out = {"loss": loss.detach()}
    if c["step"]:
        out["grad"] = torch.autograd.grad(loss, s["logits"], s["g"])[0]
    return out


# ---- the plain forms: 32 bits, rounded once at the end ----------------------------------------------------------------

def _plain_layer_norm(s, c):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    r = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + 1e-5)
    xh = centred * r
    w = s["w"].float() if s["w"] is not None else None
    y = xh * w if w is not None else xh
    if s["b"] is not None:
        y = y + s["b"].float()
    y = y.to(s["x"].dtype)
    if not c["step"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w if w is not None else dy
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    grads = [dx.to(s["x"].dtype)]
    if w is not None:  # sums over many rows: in 64 bits
        grads.append((dy * xh).sum(0, dtype=torch.float64).to(s["w"].dtype))
    if s["b"] is not None:
        grads.append(dy.sum(0, dtype=torch.float64).to(s["b"].dtype))
    return {"y": y, "grads": grads}


def _plain_route(s, c):
    logits, (M, E), k, G = s["logits"], s["logits"].shape, c["top_k"], c["groups"]
    masked = logits == -INF
    wide = logits.double()  # which of two close scores is the larger is decided in 64 bits
    if s["bias"] is None:
        key = wide  # the scores' order is the logits' order
        value = _scores(wide, c["score"])
    else:
        key = value = (_scores(wide, c["score"]) + s["bias"].double()).masked_fill(masked, -INF)
    if G > 1:
        value = value.masked_fill(masked, -INF).view(M, G, E // G)
        best = value.topk(min(2 if c["group_score"] == "top2" else 1, E // G), dim=2).values
        best = best[..., 0] + best[..., 1:].masked_fill(best[..., 1:] == -INF, 0.0).sum(2)  # (one, where there is no second)
        order = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        kept = torch.zeros(M, G, dtype=torch.bool, device=logits.device).scatter_(1, order, True)
        key = key.masked_fill(~kept[:, :, None].expand(M, G, E // G).reshape(M, E), -INF)
    top = torch.sort(key, dim=1, descending=True, stable=True)
    indices = top.indices[:, :k]
    empty = top.values[:, :k] == -INF
    score = _scores(logits.float(), c["score"])
    a = score.gather(1, indices).masked_fill(empty, 0.0)
    total = a.sum(1, keepdim=True) if c["renormalize"] else torch.ones_like(a[:, :1])
    total = total.masked_fill(total == 0.0, 1.0)
    weights = c["scale"] * a / total
    chosen = indices.masked_fill(empty, -1)
    counts = torch.bincount(chosen.reshape(-1) + 1, minlength=E + 1)[1:].to(torch.int32)
    out = {"weights": weights, "indices": chosen, "counts": counts}
    if c["step"]:
        da = c["scale"] * s["dw"].masked_fill(empty, 0.0)
        if c["renormalize"]:  # a difference of nearly equal numbers where one choice has most of the weight: in 64 bits
            a64, dw = a.double(), s["dw"].double()
            total = a64.sum(1, keepdim=True)
            total = total.masked_fill(total == 0.0, 1.0)
            da = (c["scale"] * (dw * total - (dw * a64).sum(1, keepdim=True)) / (total * total)).float()
            da = da.masked_fill(empty, 0.0)
        ds = torch.zeros_like(score).scatter_add_(1, indices, da)
        if c["score"] == "softmax":
            grad = score * (ds - (da * a).sum(1, keepdim=True))
        else:
            grad = ds * score * (1.0 - score)
        out["grad"] = grad.masked_fill(masked, 0.0).to(logits.dtype)
    return out


def _scores(logits, kind):
    """scores of the candidates; a row that is masked everywhere scores 0 everywhere"""
    if kind == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    top = logits.amax(1, keepdim=True)
    e = torch.exp(logits - top.masked_fill(top == -INF, 0.0))
    total = e.sum(1, keepdim=True)
    return e / total.masked_fill(total == 0.0, 1.0)


def _plain_distill(s, c):
    T = c["temperature"]
    z = s["logits"].float()
    top = z.amax(1, keepdim=True)
    e = torch.exp((z - top) / T)
    total = e.sum(1, keepdim=True)
    # the student's logarithms at the teacher's classes, and the teacher's distribution over its filled slots
    filled = s["index"] >= 0
    index = s["index"].clamp(min=0)
    t = s["teacher"].float().masked_fill(~filled, -INF)
    most = t.amax(1, keepdim=True)
    has = most > -INF
    et = torch.exp((t - most.masked_fill(~has, 0.0)) / T)
    st = et.sum(1, keepdim=True)
    p = et / st.masked_fill(~has, 1.0)
    # differences of logarithms: in 64 bits, the two are close where the student has learnt
    log_q = (z.gather(1, index).double() - top.double()) / T - torch.log(total.double())
    log_p = (t.double() - most.masked_fill(~has, 0.0).double()) / T - torch.log(st.masked_fill(~has, 1.0).double())
    rows = T * T * torch.where(p > 0, p.double() * (log_p - log_q), 0.0).sum(1)
    teachers = has.sum().clamp(min=1)
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / teachers}[c["reduction"]].float()
    if not c["step"]:
        return {"loss": loss}
    scale = {"none": s["g"], "sum": 1.0, "mean": 1.0 / teachers}[c["reduction"]]
    scale = (T * scale * torch.ones_like(z[:, 0])).masked_fill(~has[:, 0], 0.0)[:, None]
    q = e / total
    grad = scale * q.scatter_add_(1, index, -p)
    return {"loss": loss, "grad": grad.to(s["logits"].dtype)}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    size, M = BYTES[case["dtype"]], case["rows"]
    if case["op"] == "layer_norm":
        D, affine = case["cols"], {"both": 2, "weight": 1, "none": 0}[case["affine"]]
        params = affine * D * BYTES[case["params"]]
        if case["step"]:
            return {"bytes": 4 * M * D * size + 2 * params, "flops": 20 * M * D}
        return {"bytes": 2 * M * D * size + params, "flops": 7 * M * D}
    if case["op"] == "route":
        E, k = case["cands"], case["top_k"]
        read = M * E * size + (4 * E if case["bias"] else 0)
        written = M * k * 12 + 4 * E
        if case["step"]:
            return {"bytes": read + written + M * k * 4 + M * E * size, "flops": 10 * M * E}
        return {"bytes": read + written, "flops": 6 * M * E}
    V, k = case["cols"], case["top"]
    read = M * V * size + M * k * (8 + BYTES[case["teacher"]])
    losses = 4 * (M if case["reduction"] == "none" else 1)
    if case["step"]:
        return {"bytes": read + losses + M * V * size + (4 * M if case["reduction"] == "none" else 0), "flops": 8 * M * V}
    return {"bytes": read + losses, "flops": 4 * M * V}


# ---- the definitions in 64 bits, on their own ---------------------------------------------------------------------------

def exact(case, seed):
    def largest(values, n):
        """the n largest of each row, one after the other, the first of equal ones first: (places, values)"""
        left, places, highs = values.clone(), [], []
        free = torch.ones_like(values, dtype=torch.bool)
        at = torch.arange(values.shape[1], device=values.device)
        for _ in range(n):
            high = left.amax(1, keepdim=True)
            place = torch.where((left == high) & free, at, values.shape[1]).amin(1, keepdim=True)
            places.append(place)
            highs.append(high)
            left.scatter_(1, place, -INF)
            free.scatter_(1, place, False)
        return torch.cat(places, 1), torch.cat(highs, 1)

    s = {k: (v.detach() if torch.is_tensor(v) else v) for k, v in prepare(case, seed).items()}
    if case["op"] == "route":
        return _exact_route(s, case, largest)
    return {"layer_norm": _exact_layer_norm, "distill": _exact_distill}[case["op"]](s, case)


def _exact_layer_norm(s, c):
    x = s["x"].double()
    D = x.shape[1]
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    sd = (var + 1e-5).sqrt()
    w = torch.ones(D, dtype=torch.float64, device=x.device) if s["w"] is None else s["w"].double()
    b = torch.zeros(D, dtype=torch.float64, device=x.device) if s["b"] is None else s["b"].double()
    xh = (x - mean) / sd
    y = torch.addcmul(b, xh, w)
    if not c["step"]:
        return {"y": y}
    # the Jacobian of a row is (I - 1 1'/D - xh xh'/D) / sd, applied to dy w
    dy = s["dy"].double()
    v = dy * w
    dx = (v - v.sum(1, keepdim=True) / D - xh * torch.linalg.vecdot(v, xh)[:, None] / D) / sd
    grads = [dx]
    if s["w"] is not None:
        grads.append(torch.linalg.vecdot(dy, xh, dim=0))
    if s["b"] is not None:
        grads.append(dy.sum(0))
    return {"y": y, "grads": grads}


def _exact_route(s, c, largest):
    logits = s["logits"].double()
    M, E = logits.shape
    barred = torch.isneginf(logits)
    if c["score"] == "sigmoid":
        score = torch.sigmoid(logits)
    else:
        score = torch.softmax(logits, 1).masked_fill(barred.all(1, keepdim=True), 0.0)
    rank_by = logits.clone() if s["bias"] is None else score + s["bias"].double()
    by_group = score if s["bias"] is None else rank_by
    rank_by = rank_by.masked_fill(barred, -INF)
    if c["groups"] > 1:
        blocks = by_group.masked_fill(barred, -INF).reshape(M, c["groups"], -1)
        n = blocks.shape[2]
        ordered = blocks.sort(2).values
        group = ordered[:, :, n - 1].clone()
        if c["group_score"] == "top2" and n > 1:
            group += torch.where(torch.isneginf(ordered[:, :, n - 2]), 0.0, ordered[:, :, n - 2])
        picked = largest(group, c["top_groups"])[0]
        allowed = torch.zeros_like(group).scatter(1, picked, 1.0).repeat_interleave(n, 1) > 0
        rank_by = rank_by.masked_fill(~allowed, -INF)
    indices, highs = largest(rank_by, c["top_k"])
    indices = torch.where(torch.isneginf(highs), -1, indices)
    real = indices >= 0
    a = torch.where(real, score.gather(1, indices.clamp(min=0)), 0.0)
    weights = c["scale"] * a
    if c["renormalize"]:
        total = torch.where(real.any(1, keepdim=True), a.sum(1, keepdim=True), 1.0)
        weights = weights / total
    counts = torch.stack([(indices == e).sum() for e in range(E)]).to(torch.int32)
    out = {"weights": weights, "indices": indices, "counts": counts}
    if c["step"]:
        dw = torch.where(real, s["dw"].double(), 0.0)
        if c["renormalize"]:
            da = c["scale"] * (dw * total - (dw * a).sum(1, keepdim=True)) / total ** 2
        else:
            da = c["scale"] * dw
        da = torch.where(real, da, 0.0)
        spread = torch.zeros_like(score).scatter_add(1, indices.clamp(min=0), da)
        if c["score"] == "sigmoid":
            grad = spread * score * torch.sigmoid(-logits)
        else:
            grad = spread * score - score * (spread * score).sum(1, keepdim=True)
        out["grad"] = grad.masked_fill(barred, 0.0)
    return out


def _exact_distill(s, c):
    T = c["temperature"]
    z = s["logits"].double() / T
    log_q = torch.log_softmax(z, 1)
    del z
    here = s["index"] >= 0
    at = torch.where(here, s["index"], 0)
    t = torch.where(here, s["teacher"].double() / T, -INF)
    taught = here.any(1)
    log_p = torch.log_softmax(torch.where(taught[:, None], t, 0.0), 1)
    p = torch.where(here, log_p.exp(), 0.0)
    rows = T * T * torch.where(here, p * (log_p - log_q.gather(1, at)), 0.0).sum(1)
    n = max(1, int(taught.sum()))
    loss = rows if c["reduction"] == "none" else rows.sum() / (n if c["reduction"] == "mean" else 1)
    if not c["step"]:
        return {"loss": loss}
    up = s["g"].double() if c["reduction"] == "none" else torch.full_like(rows, 1.0 / n if c["reduction"] == "mean" else 1.0)
    grad = log_q.exp_().scatter_add_(1, at, -p)
    return {"loss": loss, "grad": grad.mul_((T * up * taught)[:, None])}
