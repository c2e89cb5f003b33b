"""Cases for the learning operators on heat maps and tours: what a heat map (or an autoregressive decoder's
logits) says about the tours that were drawn from it, and the two losses that turn tour lengths into a gradient.

``own = False`` computes them from elementary torch operations, ``own = True`` calls ``ml4tspbench_amd``:

* ``tour_log_probs``: step log-probabilities of tours, softmax over the nodes not yet visited;
* ``clipped_policy_loss``: clipped importance ratios times advantages, with a KL term towards a reference;
* ``preference_loss``: logistic loss on log-ratio differences of the tours of one instance, shorter preferred.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------- the cases
def _logp(name, maps, per, n, rows, dtype, train, knn=0, fill="none"):
    case = {"op": "tour_log_probs", "maps": maps, "per": per, "n": n, "rows": rows, "dtype": dtype, "train": train,
            "knn": knn, "fill": fill}
    return {"name": name, **case} if name else case


def _policy(name, tours, steps, dtype, ratio, average, ref, mask, per_step=False):
    case = {"op": "clipped_policy_loss", "tours": tours, "steps": steps, "dtype": dtype, "ratio": ratio,
            "average": average, "ref": ref, "mask": mask, "per_step": per_step}
    return {"name": name, **case} if name else case


def _preference(name, inst, per, steps, dtype, pairs, ref, mask, per_step=False, smoothing=0.0):
    case = {"op": "preference_loss", "inst": inst, "per": per, "steps": steps, "dtype": dtype, "pairs": pairs,
            "ref": ref, "mask": mask, "per_step": per_step, "smoothing": smoothing}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one TSP-50 instance whose 16 samples are scored while its heat map is tuned: latency
        _logp("score one tsp50 x16", 1, 16, 50, "node", "f32", False),
        # the sampled TSP-500 batch (128 instances x 16 tours) scored under its heat maps
        _logp("score tsp500 128x16", 128, 16, 500, "node", "f32", False),
        # ... and its training step in bf16: values and the heat maps' gradient
        _logp("train tsp500 128x16 bf16", 128, 16, 500, "node", "bf16", True),
        # odd sizes, float16, k nearest neighbours with -inf elsewhere: rows that run out of neighbours are empty
        _logp("train tsp333 7x5 knn f16", 7, 5, 333, "node", "f16", True, 20, "-inf"),
        # one tour a map, k = 50 neighbours with the type's lowest value elsewhere
        _logp("train tsp1000 128x1 knn", 128, 1, 1000, "node", "f32", True, 50, "lowest"),
        # the largest maps
        _logp("train tsp10000 16x1", 16, 1, 10000, "node", "f32", True),
        # an autoregressive decoder's logits, a row for every step
        _logp("train steps tsp100 10000 bf16", 10000, 1, 100, "step", "bf16", True),
        # one instance's samples: latency
        _policy("policy 16x49", 16, 49, "f32", "step", "step", False, False),
        # the TSP-100 batch with a KL term; instances of fewer nodes are padded
        _policy("policy 10000x99 kl masked", 10000, 99, "f32", "step", "step", True, True),
        # whole-tour ratios over the sampled TSP-500 batch, bf16
        _policy("policy tour 2048x499 bf16", 2048, 499, "bf16", "tour", "tour", True, False),
        # every pair of the 16 samples of 128 TSP-500 instances
        _preference("preference 128x16x499", 128, 16, 499, "f32", "all", True, False),
        # an odd small batch: latency
        _preference("preference 5x7x37 best", 5, 7, 37, "bf16", "best", False, True, True, 0.1),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["node", "node", "step", "policy", "preference"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "node":
        n = _spread(rng, 5, 2000)
        per = _spread(rng, 1, 40)
        room = max(1, 200_000_000 // (per * n * n))
        maps = _spread(rng, 1, min(room, 300))
        fill = rng.choice(["none", "-inf", "lowest"])
        knn = 0 if fill == "none" else rng.randint(3, 60)
        return _logp(None, maps, per, n, "node", dtype, rng.random() < 0.7, knn, fill)
    if op == "step":
        n = _spread(rng, 3, 700)
        tours = _spread(rng, 1, min(5000, max(1, 200_000_000 // (n * n))))
        return _logp(None, tours, 1, n, "step", dtype, rng.random() < 0.7, 0, rng.choice(["none", "-inf"]))
    if op == "policy":
        steps = _spread(rng, 1, 10000)
        tours = _spread(rng, 1, min(10000, 10_000_000 // steps))
        ratio = rng.choice(["step", "tour"])
        average = "tour" if ratio == "tour" else rng.choice(["step", "tour"])
        return _policy(None, tours, steps, dtype, ratio, average, rng.random() < 0.6, rng.random() < 0.6,
                       ratio == "step" and rng.random() < 0.3)
    steps = _spread(rng, 1, 10000)
    per = _spread(rng, 2, 100)
    inst = _spread(rng, 1, max(1, min(1000, 10_000_000 // (steps * per))))
    return _preference(None, inst, per, steps, dtype, rng.choice(["all", "best"]), rng.random() < 0.6,
                       rng.random() < 0.6, rng.random() < 0.5, rng.choice([0.0, 0.1]))


# ---------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def rand(*shape):
        return torch.rand(shape, generator=gen, device=dev)

    def randn(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    if case["op"] == "tour_log_probs":
        n, maps, per = case["n"], case["maps"], case["per"]
        T = maps * per
        if case["rows"] == "node":
            # the logarithm of a "near edges are hot" heat map: -distance / tau plus noise
            pts = rand(maps, n, 2)
            logits = torch.cdist(pts, pts, compute_mode="donot_use_mm_for_euclid_dist").mul_(-math.sqrt(n) / 0.35)
            if case["knn"]:
                far = logits < logits.topk(min(case["knn"] + 1, n), dim=-1).values[..., -1:]
            logits.add_(torch.empty_like(logits).uniform_(-0.5, 0.35, generator=gen))
            if case["knn"]:
                logits.masked_fill_(far, -math.inf if case["fill"] == "-inf" else torch.finfo(dtype).min)
                del far
            logits = logits.to(dtype)
            tours = torch.zeros((T, n + 1), dtype=torch.int64, device=dev)
            if n <= 2000:           # drawn from the maps, one node after the other
                open_ = torch.ones((T, n), dtype=torch.bool, device=dev)
                open_[:, 0] = False
                cur = torch.zeros(T, dtype=torch.int64, device=dev)
                row = torch.arange(T, device=dev)
                for k in range(1, n):
                    u = rand(T, n).clamp_(1e-20, 1 - 1e-7)
                    score = logits[row // per, cur].float().clamp_(min=-1e30) - u.log_().neg_().log_()
                    cur = score.masked_fill_(~open_, -math.inf).argmax(-1)
                    tours[:, k] = cur
                    open_[row, cur] = False
            else:                   # up and down in strips, with some disorder
                strips = max(1, int(math.sqrt(n / 3)))
                p = pts.repeat_interleave(per, 0) + 0.3 / math.sqrt(n) * randn(T, n, 2)
                s = (p[..., 0] * strips).floor()
                key = s + torch.where(s % 2 == 0, p[..., 1], 1 - p[..., 1]).clamp(0, 0.999)
                order = key.argsort(-1)
                first = (order == 0).to(torch.int8).argmax(-1, keepdim=True)
                tours[:, :n] = order.gather(1, (torch.arange(n, device=dev) + first) % n)
        else:
            # decoder logits in (-10, 10); a decoder that masks its visited nodes itself leaves -inf there
            tours = torch.zeros((T, n + 1), dtype=torch.int64, device=dev)
            if n > 1:
                tours[:, 1:n] = rand(T, n - 1).argsort(-1) + 1
            logits = randn(T, n - 1, n).tanh_().mul_(10)
            if case["fill"] == "-inf":
                pos = torch.empty((T, n), dtype=torch.int64, device=dev)
                pos.scatter_(1, tours[:, :n], torch.arange(n, device=dev).expand(T, n))
                logits.masked_fill_(pos[:, None, :] <= torch.arange(n - 1, device=dev)[None, :, None], -math.inf)
            logits = logits.to(dtype)
        # a policy gradient's weights: the same advantage for every step of a tour
        g = randn(T, 1).expand(T, n - 1).contiguous() if case["train"] else None
        return {"case": case, "logits": logits, "tours": tours, "g": g}

    if case["op"] == "clipped_policy_loss":
        T, S = case["tours"], case["steps"]
    else:
        T, S = case["inst"] * case["per"], case["steps"]
    old = -2.0 * rand(T, S) ** 2 - 0.01
    state = {"case": case, "mask": None, "ref": None}
    small = 0.15 if case.get("ratio") != "tour" else 0.15 / math.sqrt(S)
    state["lp"] = (old + small * randn(T, S)).to(dtype)
    state["old"] = old.to(dtype)
    if case["ref"]:
        state["ref"] = (old + 0.2 * randn(T, S)).to(dtype)
    if case["mask"]:                # ragged: the steps behind a shorter tour's end do not count, some rows are empty
        keep = (rand(T, 1) * (S + 1) * 1.2).floor()
        keep = torch.where(rand(T, 1) < 0.05, torch.zeros_like(keep), keep)
        state["mask"] = torch.arange(S, device=dev)[None, :] < keep
        hidden = torch.full((), math.nan, dtype=dtype, device=dev)
        for k in ("lp", "old", "ref"):
            if state[k] is not None:
                state[k] = torch.where(state["mask"], state[k], hidden)
    if case["op"] == "clipped_policy_loss":
        state["adv"] = randn(T, S) if case["per_step"] else randn(T)
    else:
        state["len"] = (16.5 + 0.5 * rand(T).double())
        state["len"][:: 11] = 16.75                             # equal lengths: no preference between them
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_tour_log_probs(s):
    case, tours, g = s["case"], s["tours"], s["g"]
    n, M, P = case["n"], case["maps"], case["per"]
    T, dev = M * P, tours.device
    order = tours[:, :n]
    steps = torch.arange(n, device=dev)
    pos = torch.empty_like(order).scatter_(1, order, steps.expand(T, n))
    if case["rows"] == "node":
        when = pos                                              # the step at which a row (a node) is left
        after = tours.gather(1, pos + 1)
    else:
        when = steps[: n - 1].expand(T, n - 1)
        after = tours[:, 1:n]
    when, after = when.view(M, P, -1, 1), after.view(M, P, -1, 1)
    keep = pos.to(torch.int32).view(M, P, 1, n) > when.to(torch.int32)
    z = torch.where(keep, s["logits"].float().unsqueeze(1), -math.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    chosen = z.gather(-1, after) - top
    e = z.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    lp = torch.where(total > 0, chosen - total.log(), -math.inf).view(T, -1)
    lp = lp.gather(1, order[:, : n - 1]) if case["rows"] == "node" else lp
    if g is None:
        return lp
    w = torch.zeros_like(when, dtype=torch.float32)
    if case["rows"] == "node":
        w = torch.cat([g, g.new_zeros(T, 1)], 1).gather(1, pos).view_as(w)
    else:
        w = g.view_as(w)
    w = torch.where(total > 0, w, 0.0)
    d = e.mul_(-w / torch.where(total > 0, total, 1.0)).scatter_add_(-1, after, w)
    return lp, d.sum(1).to(s["logits"].dtype)


def _weights(kept, average):
    """The weight of every step in the averages: 1 / all kept steps, or 1 / (a tour's kept steps * tours with any)."""
    if average == "step":
        return kept / kept.sum().clamp(min=1)
    count = kept.sum(1, keepdim=True)
    return kept / count.clamp(min=1) / (count > 0).sum().clamp(min=1)


LOW, HIGH, KL = 0.2, 0.28, 0.04


def _plain_policy(s):
    case, mask = s["case"], s["mask"]
    lp = s["lp"].double()
    kept = torch.ones_like(lp) if mask is None else mask.double()
    x = lp - s["old"].double()
    x = x if mask is None else torch.where(mask, x, 0.0)
    adv = s["adv"].float() if s["adv"].dim() == 2 else s["adv"].float()[:, None]
    w = _weights(kept, case["average"])
    if case["ratio"] == "tour":
        x = x.sum(1, keepdim=True)
        wx = w.sum(1, keepdim=True)
    else:
        wx = w
    # which side of the border a ratio is on is decided in 64 bits: the gradient jumps there
    low, high = math.log1p(-LOW), math.log1p(HIGH)
    cut = ((adv > 0) & (x > high)) | ((adv < 0) & (x < low))
    r = x.float().exp()
    term = -adv * torch.where(cut, torch.where(x > high, 1 + HIGH, 1 - LOW), r)
    loss = (term * wx).sum()
    clip = (cut * wx).sum()
    dx = torch.where(cut, 0.0, -adv * r) * (wx if case["ratio"] == "step" else 1.0 / (kept.sum(1) > 0).sum().clamp(min=1) * kept)
    kl = torch.zeros_like(loss)
    if s["ref"] is not None:
        d = s["ref"].double() - lp
        d = d if mask is None else torch.where(mask, d, 0.0)
        kl = ((d.expm1() - d) * w).sum()                        # exp(d) - 1 - d, which 32 bits lose for small d
        loss = loss + KL * kl
        dx = dx - KL * w * d.expm1()
    return loss.float(), kl.float(), clip.float(), dx.to(s["lp"].dtype)


BETA = 0.5


def _plain_preference(s):
    case, mask = s["case"], s["mask"]
    I, P = case["inst"], case["per"]
    x = s["lp"].double() if s["ref"] is None else s["lp"].double() - s["ref"].double()
    kept = torch.ones_like(x) if mask is None else mask.double()
    x = x if mask is None else torch.where(mask, x, 0.0)
    scale = BETA / kept.sum(1).clamp(min=1) if case["per_step"] else torch.full_like(kept[:, 0], BETA)
    score = (x.sum(1) * scale).view(I, P)
    length = s["len"].view(I, P)
    wins = length[:, :, None] < length[:, None, :]
    if case["pairs"] == "best":                                 # the first of the shortest against every longer one
        first = length.argmin(1)
        wins = wins & (torch.arange(P, device=first.device)[None, :, None] == first[:, None, None])
    count = wins.sum()
    z = score[:, :, None] - score[:, None, :]
    soft = torch.clamp(-z, min=0) + torch.log1p(torch.exp(-z.abs()))        # -log sigmoid(z)
    eps = case["smoothing"]
    share = wins / count.clamp(min=1)
    loss = ((soft + eps * z) * share).sum()                     # (1-eps) softplus(-z) + eps softplus(z)
    dz = (eps - 1 / (1 + torch.exp(z))) * share
    dscore = (dz.sum(2) - dz.sum(1)).reshape(-1)
    grad = (dscore * scale)[:, None] * kept
    return loss.float(), count, grad.to(s["lp"].dtype)


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "tour_log_probs":
            return _plain_tour_log_probs(state)
        return _plain_policy(state) if case["op"] == "clipped_policy_loss" else _plain_preference(state)
    import ml4tspbench_amd as amd
    if case["op"] == "tour_log_probs":
        logits = state["logits"]
        if not case["train"]:
            return amd.tour_log_probs(logits, state["tours"], tours_per_map=case["per"], rows=case["rows"])
        logits = logits.detach().requires_grad_()
        lp = amd.tour_log_probs(logits, state["tours"], tours_per_map=case["per"], rows=case["rows"])
        return lp.detach(), torch.autograd.grad(lp, logits, state["g"])[0]
    lp = state["lp"].detach().requires_grad_()
    if case["op"] == "clipped_policy_loss":
        res = amd.clipped_policy_loss(lp, state["old"], state["adv"], ref_log_probs=state["ref"], mask=state["mask"],
                                      clip_low=LOW, clip_high=HIGH, kl_coef=KL if case["ref"] else 0.0,
                                      ratio=case["ratio"], average=case["average"])
        return res.loss.detach(), res.kl, res.clip_fraction, torch.autograd.grad(res.loss, lp)[0]
    res = amd.preference_loss(lp, state["len"], tours_per_instance=case["per"], ref_log_probs=state["ref"],
                              mask=state["mask"], beta=BETA, label_smoothing=case["smoothing"], pairs=case["pairs"],
                              per_step=case["per_step"])
    return res.loss.detach(), res.num_pairs, torch.autograd.grad(res.loss, lp)[0]


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] == "tour_log_probs":
        n, M, P = case["n"], case["maps"], case["per"]
        T, rows = M * P, n if case["rows"] == "node" else n - 1
        values = M * rows * n
        once = values * (4 + 2 * P)                             # maximum, exponential; a masked sum for every tour
        moved = values * size + T * (n + 1) * 8 + T * (n - 1) * 4
        if case["train"]:
            return {"bytes": moved + T * (n - 1) * 4 + values * size, "flops": once + values * (2 + 2 * P)}
        return {"bytes": moved, "flops": once}
    T = case["tours"] if "tours" in case else case["inst"] * case["per"]
    values = T * case["steps"]
    arrays = (3 if case["op"] == "clipped_policy_loss" else 2) + (1 if case["ref"] else 0)
    moved = values * (arrays * size + (1 if case["mask"] else 0))
    if case["op"] == "clipped_policy_loss":
        return {"bytes": moved + 4 * (values if case["per_step"] else T) + 12, "flops": 30 * values}
    return {"bytes": moved + 8 * T + 12, "flops": 3 * values + 20 * T * case["per"]}


# ---------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tour_log_probs":
        return _exact_tour_log_probs(s)
    lp = s["lp"].double()
    mask = s["mask"] if s["mask"] is not None else torch.ones_like(lp, dtype=torch.bool)
    lp = torch.where(mask, lp, 0.0).requires_grad_()
    rest = {k: torch.where(mask, s[k].double(), 0.0) if s[k] is not None else None for k in ("old", "ref")}
    count = mask.sum(1)
    if case["op"] == "clipped_policy_loss":
        tours = (count > 0).sum().clamp(min=1)

        def mean(v):
            if case["average"] == "step":
                return (v * mask).sum() / mask.sum().clamp(min=1)
            return ((v * mask).sum(1) / count.clamp(min=1)).sum() / tours

        adv = s["adv"].double()
        if case["ratio"] == "tour":
            r = ((lp - rest["old"]) * mask).sum(1).exp()
            term = torch.minimum(r * adv, r.clamp(1 - LOW, 1 + HIGH) * adv)
            full = count > 0
            loss = -(term * full).sum() / tours
            clip = ((r * adv > r.clamp(1 - LOW, 1 + HIGH) * adv) * full).sum() / tours
        else:
            adv = adv if adv.dim() == 2 else adv[:, None]
            r = (lp - rest["old"]).exp()
            term = torch.minimum(r * adv, r.clamp(1 - LOW, 1 + HIGH) * adv)
            loss, clip = -mean(term), mean((r * adv > r.clamp(1 - LOW, 1 + HIGH) * adv).double())
        kl = torch.zeros_like(loss)
        if rest["ref"] is not None:
            d = rest["ref"] - lp
            kl = mean(torch.expm1(d) - d)
        loss = loss + KL * kl
        (grad,) = torch.autograd.grad(loss, lp)
        return loss.detach(), kl.detach(), clip.detach(), grad
    x = (lp - rest["ref"] if rest["ref"] is not None else lp) * mask
    score = BETA * (x.sum(1) / count.clamp(min=1) if case["per_step"] else x.sum(1))
    length = s["len"].cpu().numpy().reshape(case["inst"], case["per"])
    win, lose = np.nonzero(np.ones((case["per"], case["per"]), dtype=bool))
    a, b = [], []
    for i, row in enumerate(length):
        ok = row[win] < row[lose]
        if case["pairs"] == "best":
            ok &= win == int(np.argmin(row))
        a.append(win[ok] + i * case["per"])
        b.append(lose[ok] + i * case["per"])
    a, b = (torch.from_numpy(np.concatenate(v)).to(lp.device) for v in (a, b))
    z, eps = score[a] - score[b], case["smoothing"]
    each = -(1 - eps) * torch.nn.functional.logsigmoid(z) - eps * torch.nn.functional.logsigmoid(-z)
    loss = each.sum() / max(1, len(a))
    (grad,) = torch.autograd.grad(loss, lp)
    return loss.detach(), None, grad


def _exact_tour_log_probs(s):
    """Tour by tour in the tour's own order: step t sees the places t + 1 .. n - 1 of its row."""
    case, tours, g = s["case"], s["tours"], s["g"]
    n, per = case["n"], case["per"]
    if tours.shape[0] * n * n > 1_700_000_000:
        return None
    lps = torch.empty((tours.shape[0], n - 1), dtype=torch.float64, device=tours.device)
    grad = torch.zeros(s["logits"].shape, dtype=torch.float64, device=tours.device) if g is not None else None
    block = max(1, min(512, 200_000_000 // (n * n)))
    for a in range(0, tours.shape[0], block):
        t = tours[a: a + block]
        T = t.shape[0]
        which = (torch.arange(a, a + T, device=t.device) // per)[:, None]
        row = t[:, : n - 1] if case["rows"] == "node" else torch.arange(n - 1, device=t.device).expand(T, n - 1)
        x = s["logits"][which, row].double()                                # (T, n - 1, n), a row for every step
        seen = t[:, None, :n].expand(T, n - 1, n)
        x = x.gather(2, seen).masked_fill_(torch.ones((n - 1, n), dtype=torch.bool, device=t.device).tril(), -math.inf)
        top = x.amax(2, keepdim=True)                                       # first: lowest values swallow a logarithm
        x = x.sub_(top.masked_fill(top == -math.inf, 0.0))
        lse = x.logsumexp(2)
        dead = lse == -math.inf
        lps[a: a + T] = (x.diagonal(1, 1, 2) - lse).masked_fill_(dead, -math.inf)
        if grad is None:
            continue
        gt = g[a: a + T].double().masked_fill(dead, 0.0)
        p = (x - lse.masked_fill(dead, 0.0)[..., None]).exp_().mul_(-gt[..., None])
        p.diagonal(1, 1, 2).add_(gt)
        back = torch.empty_like(p).scatter_(2, seen, p)
        grad.index_put_((which.expand(T, n - 1), row), back, accumulate=True)
    return lps if grad is None else (lps, grad)
