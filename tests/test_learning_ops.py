"""tour_log_probs, clipped_policy_loss, preference_loss: the kernels against the formulas in 64 bits (computed on the
CPU), their refusals, and a run of them together with the decoder, 2-opt and the evaluator.

Tolerances count roundings.  u = 2^-24 is half a step of float32 relative to the value; storing to a type costs
finfo(type).eps / 2 of the value.  A log-probability h - m - log S (m: the row's largest entry) rounds h - m and log S
and carries the relative error of S, a sum of exponentials exp(h - m) whose argument was rounded (u |h - m|, times
log2 e) and which the hardware's exponential gives to 2 ulp: all in all below 8 u (4 + |h - m|), with |h - m| the
largest that matters to the sum."""
import ctypes
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


# ------------------------------------------------------------------------------------------ formulas in 64 bits
def ref_log_probs(logits, tours, per, rows, g=None):
    """(lp, tolerance) and with g (grad, tolerance); logits any float type on the CPU, everything in float64."""
    h = logits.double()
    T, n = tours.shape[0], tours.shape[1] - 1
    lp = torch.zeros((T, n - 1), dtype=torch.float64)
    tol = torch.zeros_like(lp)
    grad, gtol = torch.zeros_like(h), torch.zeros_like(h)
    later = torch.ones((n - 1, n), dtype=torch.bool).triu(1)
    for k in range(T):
        order = tours[k, :n]
        m = k // per if rows == "node" else k
        row = order[:-1] if rows == "node" else torch.arange(n - 1)
        if sorted(order.tolist()) != list(range(n)):
            lp[k] = math.nan
            continue
        full = h[m][row].clone()
        full[torch.arange(n - 1), order[:-1]] = -math.inf        # the node that is left is never open
        full = torch.where(full.isfinite(), full, -math.inf)     # what a row maximum may be
        x = h[m][row][:, order].masked_fill(~later, -math.inf)
        top = x.amax(1, keepdim=True)
        dead = top[:, 0] == -math.inf
        s = torch.where(top == -math.inf, x, x - top)
        lse = s.logsumexp(1)
        chosen = s.diagonal(1)
        lp[k] = torch.where(dead, -math.inf, chosen - lse)
        # what the spread of a row costs: against the row's own largest entry, as far as the sum sees it (at most 64)
        high = torch.maximum(full.amax(1, keepdim=True), top).nan_to_num(0, 0, 0)
        far = (high - x).nan_to_num(0, 0, 0)
        near = (high - top).nan_to_num(0, 0, 0).clamp(max=64)[:, 0]
        tol[k] = 8 * U * (4 + near + far.diagonal(1))
        if g is None:
            continue
        gk = torch.where(dead, 0.0, g[k].double())
        p = torch.where(dead[:, None], 0.0, (s - lse[:, None]).exp()).masked_fill(~later, 0.0)
        p = torch.where((gk == 0)[:, None], 0.0, p)
        d = -gk[:, None] * p
        e = gk.abs()[:, None] * p * (4 + near[:, None] + torch.where(p > 0, far, 0.0))
        d.diagonal(1).add_(gk)
        e.diagonal(1).add_(gk.abs())
        for t in range(n - 1):
            grad[m, row[t], order] += d[t]
            gtol[m, row[t], order] += 8 * U * e[t]
    eps = torch.finfo(logits.dtype).eps / 2
    gtol = gtol + eps * grad.abs() + torch.finfo(logits.dtype).smallest_normal * eps
    return lp, tol, grad, gtol


def ref_policy(lp, old, adv, ref, mask, low, high, kl_coef, ratio, average):
    """Loss, kl, clip fraction and the gradient in lp, all in float64; also the sum of magnitudes of the loss terms."""
    mask = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask
    leaf = torch.where(mask, lp.double(), 0.0).requires_grad_()
    x0 = torch.where(mask, leaf, 0.0)           # a step that does not count has no gradient
    diff = x0 - torch.where(mask, old.double(), 0.0)
    count = mask.sum(1)
    has = count > 0

    def mean(v):
        if average == "step":
            return torch.where(mask, v, 0.0).sum() / max(1, int(mask.sum()))
        return (torch.where(mask, v, 0.0).sum(1) / count.clamp(min=1)).sum() / max(1, int(has.sum()))

    A = adv.double()
    if ratio == "tour":
        r = diff.sum(1).exp()
        low_, high_ = r * A, r.clamp(1 - low, 1 + high) * A
        term = torch.where(has, -torch.minimum(low_, high_), 0.0)
        size = float(term.detach().abs().sum()) / max(1, int(has.sum()))
        loss = term.sum() / max(1, int(has.sum()))
        clip = ((low_ > high_) & has).sum() / max(1, int(has.sum()))
    else:
        A = A if A.dim() == 2 else A[:, None]
        r = diff.exp()
        low_, high_ = r * A, r.clamp(1 - low, 1 + high) * A
        loss = mean(-torch.minimum(low_, high_))
        size = float(mean(torch.minimum(low_, high_).detach().abs()))
        clip = mean((low_ > high_).double())
    kl = torch.zeros((), dtype=torch.float64)
    if ref is not None:
        d = torch.where(mask, ref.double(), 0.0) - x0
        kl = mean(torch.expm1(d) - d)
        if kl_coef:
            loss = loss + kl_coef * kl
    grad = torch.autograd.grad(loss, leaf)[0] if lp.numel() else torch.zeros_like(leaf)
    return loss.detach(), kl.detach(), torch.as_tensor(clip).double(), grad, size


def ref_preference(lp, length, per, ref, mask, beta, eps, pairs, per_step):
    mask = torch.ones_like(lp, dtype=torch.bool) if mask is None else mask
    leaf = torch.where(mask, lp.double(), 0.0).requires_grad_()
    x0 = torch.where(mask, leaf, 0.0)           # a step that does not count has no gradient
    x = x0 if ref is None else x0 - torch.where(mask, ref.double(), 0.0)
    score = beta * x.sum(1) / (mask.sum(1).clamp(min=1) if per_step else 1)
    terms = []
    for i in range(lp.shape[0] // per):
        ls = [float(v) for v in length[i * per:(i + 1) * per]]
        best = min((v, k) for k, v in enumerate(ls) if v == v)[1] if any(v == v for v in ls) else -1
        for a in range(per):
            for b in range(per):
                if ls[a] < ls[b] and (pairs == "all" or a == best):
                    z = score[i * per + a] - score[i * per + b]
                    terms.append(-(1 - eps) * torch.nn.functional.logsigmoid(z)
                                 - eps * torch.nn.functional.logsigmoid(-z))
    if not terms:
        return torch.zeros((), dtype=torch.float64), 0, torch.zeros_like(leaf)
    loss = torch.stack(terms).mean()
    return loss.detach(), len(terms), torch.autograd.grad(loss, leaf)[0]


# ------------------------------------------------------------------------------------------ inputs
def make_tours(gen, T, n, start=False):
    t = torch.zeros((T, n + 1), dtype=torch.int64)
    for k in range(T):
        t[k, :n] = torch.randperm(n, generator=gen) if start else torch.cat(
            [torch.zeros(1, dtype=torch.int64), torch.randperm(n - 1, generator=gen) + 1])
        t[k, n] = t[k, 0]
    return t


def rows_of(gen, M, R, n, dtype, kind="plain"):
    """Rows of logits: plain; with forbidden entries; a wide range; poison where every tour has been; decoder's mask."""
    h = torch.randn((M, R, n), generator=gen) * 3
    if kind == "wide":          # a few entries far above all others: most steps see only what is 100 and more below
        h = h - 120.0
        h[..., :: 7] += 120.0
    elif kind == "inf":
        h[torch.rand((M, R, n), generator=gen) < 0.6] = -math.inf
        h[:, 0] = -math.inf
    elif kind == "lowest":
        h = h.to(dtype)
        h[torch.rand((M, R, n), generator=gen) < 0.6] = torch.finfo(dtype).min
        h[:, 0] = torch.finfo(dtype).min
    return h.to(dtype)


def compare(name, got, want, tol):
    got, want = got.detach().double().cpu(), want.detach().double()
    assert got.shape == want.shape, name
    fine = want.isfinite()
    assert torch.equal(got.isfinite(), fine), (name, "finite places")
    assert torch.equal(got[~fine].nan_to_num(7, 8, 9), want[~fine].nan_to_num(7, 8, 9)), (name, "infinities and NaN")
    off = (got - want)[fine].abs() - torch.as_tensor(tol, dtype=torch.float64).expand_as(want)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (name, float(off.max()), float((got - want)[fine].abs().max()))


def check_log_probs(logits, tours, per, rows, gen, view=lambda x: x):
    import ml4tspbench_amd as amd
    g = torch.randn((tours.shape[0], tours.shape[1] - 2), generator=gen)
    g[torch.rand(g.shape, generator=gen) < 0.1] = 0.0
    lp, tol, grad, gtol = ref_log_probs(logits, tours, per, rows, g)
    x = view(logits.cuda()).detach().requires_grad_()
    got = amd.tour_log_probs(x, tours.cuda(), tours_per_map=per, rows=rows)
    assert got.dtype == torch.float32
    (dx,) = torch.autograd.grad(got, x, g.cuda())
    assert dx.dtype == logits.dtype
    compare("log-probabilities", got, lp, tol)
    compare("gradient", dx, grad, gtol)
    return got.detach(), dx


# ------------------------------------------------------------------------------------------ CPU: refusals
def test_argument_checks_without_gpu():
    import ml4tspbench_amd as amd
    h, t = torch.zeros(2, 5, 5), make_tours(torch.Generator().manual_seed(0), 4, 5)
    lp = torch.zeros(4, 6)
    adv, length = torch.zeros(4), torch.zeros(4)
    for exc, what, call in [
        (TypeError, "float32, bfloat16 or float16", lambda: amd.tour_log_probs(h.double(), t, tours_per_map=2)),
        (TypeError, "integers", lambda: amd.tour_log_probs(h, t.float(), tours_per_map=2)),
        (ValueError, "rows must be", lambda: amd.tour_log_probs(h, t, tours_per_map=2, rows="edge")),
        (ValueError, "expected logits", lambda: amd.tour_log_probs(h, t)),
        (ValueError, "expected logits", lambda: amd.tour_log_probs(h, t[:3], tours_per_map=2)),
        (ValueError, "expected logits", lambda: amd.tour_log_probs(h[..., :4], t, tours_per_map=2)),
        (ValueError, "expected logits", lambda: amd.tour_log_probs(h, t, tours_per_map=0)),
        (ValueError, "tours_per_map must be 1", lambda: amd.tour_log_probs(torch.zeros(4, 4, 5), t, tours_per_map=2, rows="step")),
        (ValueError, "expected logits", lambda: amd.tour_log_probs(torch.zeros(4, 5, 5), t, rows="step")),
        (ValueError, "same HIP device", lambda: amd.tour_log_probs(h, t, tours_per_map=2)),
        (TypeError, "float32, bfloat16 or float16", lambda: amd.clipped_policy_loss(lp.double(), lp.double(), adv)),
        (ValueError, "expected log_probs", lambda: amd.clipped_policy_loss(lp[0], lp[0], adv)),
        (TypeError, "type of log_probs", lambda: amd.clipped_policy_loss(lp, lp.half(), adv)),
        (ValueError, "shape of log_probs", lambda: amd.clipped_policy_loss(lp, lp[:, :5], adv)),
        (TypeError, "boolean", lambda: amd.clipped_policy_loss(lp, lp, adv, mask=lp)),
        (ValueError, "shape of log_probs", lambda: amd.clipped_policy_loss(lp, lp, adv, mask=torch.ones(4, 5, dtype=torch.bool))),
        (ValueError, "advantages", lambda: amd.clipped_policy_loss(lp, lp, torch.zeros(6))),
        (ValueError, "advantages", lambda: amd.clipped_policy_loss(lp, lp, lp, ratio="tour")),
        (TypeError, "advantages", lambda: amd.clipped_policy_loss(lp, lp, adv.long())),
        (ValueError, "averaged over tours", lambda: amd.clipped_policy_loss(lp, lp, adv, ratio="tour", average="step")),
        (ValueError, "'step' or 'tour'", lambda: amd.clipped_policy_loss(lp, lp, adv, ratio="edge")),
        (ValueError, "clip_low", lambda: amd.clipped_policy_loss(lp, lp, adv, clip_low=1.0)),
        (ValueError, "clip_low", lambda: amd.clipped_policy_loss(lp, lp, adv, clip_high=math.nan)),
        (ValueError, "needs ref_log_probs", lambda: amd.clipped_policy_loss(lp, lp, adv, kl_coef=0.1)),
        (ValueError, "same HIP device", lambda: amd.clipped_policy_loss(lp, lp, adv)),
        (ValueError, "tours_per_instance", lambda: amd.preference_loss(lp, length, tours_per_instance=3)),
        (ValueError, "tours_per_instance", lambda: amd.preference_loss(lp, length, tours_per_instance=0)),
        (ValueError, "lengths", lambda: amd.preference_loss(lp, length[:3], tours_per_instance=2)),
        (TypeError, "lengths", lambda: amd.preference_loss(lp, length.long(), tours_per_instance=2)),
        (ValueError, "'all' or 'best'", lambda: amd.preference_loss(lp, length, tours_per_instance=2, pairs="worst")),
        (ValueError, "beta", lambda: amd.preference_loss(lp, length, tours_per_instance=2, beta=0.0)),
        (ValueError, "beta", lambda: amd.preference_loss(lp, length, tours_per_instance=2, label_smoothing=0.5)),
        (ValueError, "beta", lambda: amd.preference_loss(lp, length, tours_per_instance=2, beta=math.inf)),
        (ValueError, "kl_coef", lambda: amd.clipped_policy_loss(lp, lp, adv, ref_log_probs=lp, kl_coef=math.inf)),
        (ValueError, "same HIP device", lambda: amd.preference_loss(lp, length, tours_per_instance=2)),
    ]:
        with pytest.raises(exc, match=what):
            call()


def test_c_abi_checks_without_gpu():
    from ml4tspbench_amd import _lib
    L = _lib.lib()
    at, at2 = ctypes.c_void_p(256), ctypes.c_void_p(258)

    def logp(logits=at, tours=at, out=at, state=at, nbytes=1 << 30, T=4, n=10, per=2, rows=0, ms=100, rs=10, dt=0):
        return L.tsp2opt_tour_logprobs(logits, tours, out, state, nbytes, T, n, per, rows, ms, rs, dt, 0, None)

    assert L.tsp2opt_tour_logprobs_state_bytes(4, 10, 2, 0) >= 3 * 4 * 40
    assert L.tsp2opt_tour_logprobs_state_bytes(5, 10, 2, 0) == -1 and L.tsp2opt_tour_logprobs_state_bytes(4, 0, 2, 0) == -1
    assert logp(n=0) == -1 and logp(T=-2) == -1 and logp(T=3) == -1 and logp(per=0) == -1
    assert logp(n=70000) == -2 and logp(T=1 << 31, per=1) == -2
    assert logp(T=1 << 26, per=1) == -2 and logp(T=1 << 25, n=200, per=2) == -2      # launches of 2^32 threads
    assert logp(rows=2) == -1 and logp(rows=1) == -1 and logp(dt=1) == -1 and logp(ms=-1) == -1
    assert logp(logits=None) == -1 and logp(state=None) == -1
    assert logp(logits=at2) == -1 and b"misaligned" in L.tsp2opt_last_error()
    assert logp(tours=at2) == -1 and logp(state=at2) == -1 and logp(out=at2) == -1
    assert logp(nbytes=8) == -3
    assert logp(T=0) == 0 and logp(n=1) == 0                                    # nothing to choose
    assert L.tsp2opt_tour_logprobs_grad(at, at, at, 1 << 30, None, at, 4, 10, 2, 0, 100, 10, 0, 0, None) == -1
    assert L.tsp2opt_tour_logprobs_grad(at, at, at, 8, at, at, 4, 10, 2, 0, 100, 10, 0, 0, None) == -3

    def policy(lp=at, old=at, ref=None, adv=at, mask=None, loss=at, stats=at, state=at, nbytes=1 << 30, T=4, S=6, ps=0,
               rt=0, avg=0, lo=0.2, hi=0.2, kl=0.0, dt=0):
        return L.tsp2opt_policy_loss(lp, old, ref, adv, mask, loss, stats, state, nbytes, T, S, ps, rt, avg, lo, hi, kl, dt,
                                     0, None)

    assert L.tsp2opt_policy_loss_state_bytes(-1) == -1 and L.tsp2opt_policy_loss_state_bytes(4) > 0
    assert policy(T=-1) == -1 and policy(S=-1) == -1 and policy(dt=1) == -1 and policy(lp=None) == -1
    assert policy(loss=None) == -1 and policy(stats=None) == -1 and policy(state=None) == -1 and policy(state=at2) == -1
    assert policy(old=at2) == -1 and policy(lo=1.0) == -1 and policy(hi=-0.1) == -1 and policy(hi=math.nan) == -1
    assert policy(kl=0.1) == -1 and policy(kl=-1.0, ref=at) == -1
    assert policy(rt=1) == -1 and policy(rt=1, avg=1, ps=1) == -1 and policy(nbytes=8) == -3 and policy(T=1 << 32) == -2

    def pref(lp=at, ref=None, ln=at, mask=None, loss=at, pairs=at, state=at, nbytes=1 << 30, T=4, S=6, per=2, beta=1.0,
             eps=0.0, dt=0):
        return L.tsp2opt_preference_loss(lp, ref, ln, mask, loss, pairs, state, nbytes, T, S, per, 0, 0, beta, eps, dt, 0,
                                         None)

    assert L.tsp2opt_preference_loss_state_bytes(-1) == -1
    assert pref(per=0) == -1 and pref(per=3) == -1 and pref(beta=0.0) == -1 and pref(eps=0.5) == -1 and pref(dt=1) == -1
    assert pref(beta=math.inf) == -1 and policy(kl=math.inf, ref=at) == -1
    assert L.tsp2opt_tour_logprobs_state_bytes(1 << 60, 10, 2, 0) == -2
    assert pref(lp=None) == -1 and pref(ln=None) == -1 and pref(ln=at2) == -1 and pref(pairs=None) == -1
    assert pref(nbytes=8) == -3 and pref(S=1 << 32) == -2
    assert L.tsp2opt_preference_loss_grad(None, at, 1 << 30, None, at, 4, 6, 0, 0, None) == -1
    assert L.tsp2opt_preference_loss_grad(None, at, 8, at, at, 4, 6, 0, 0, None) == -3


def test_c_abi_wants_advantages_of_tours_without_steps():
    """One advantage a tour is read for every tour, also where no tour has a step."""
    from ml4tspbench_amd import _lib
    L, at = _lib.lib(), ctypes.c_void_p(256)

    def policy(adv, T, S, per_step=0, ratio=0, average=0):
        return L.tsp2opt_policy_loss(at, at, None, adv, None, at, at, at, 1 << 30, T, S, per_step, ratio, average, 0.2, 0.2,
                                     0.0, 0, 0, None)

    for ratio, average in ((0, 0), (0, 1), (1, 1)):
        assert policy(None, 4, 0, 0, ratio, average) == -1 and b"null pointer" in L.tsp2opt_last_error()
        assert policy(None, 4, 6, 0, ratio, average) == -1
    assert policy(None, 4, 6, 1) == -1


def test_errors_of_the_library_keep_their_code():
    """Tsp2optError.code is the library's return code, as for the operators that call it through _lib.check()."""
    from ml4tspbench_amd import _lib
    ext = _lib.learning_ext()
    with pytest.raises(_lib.Tsp2optError, match="65535") as e:
        ext.tour_log_probs(torch.zeros(1, 2, 2), torch.zeros((1, 70001), dtype=torch.int64), 1, 0)
    assert e.value.code == _lib.E_UNSUPPORTED
    with pytest.raises(_lib.Tsp2optError, match="bad size") as e:
        ext.tour_log_probs(torch.zeros(1, 2, 2), torch.zeros((3, 11), dtype=torch.int64), 2, 0)
    assert e.value.code == _lib.E_ARG


def test_sizes_beyond_32_bits_are_refused_before_anything_is_copied():
    """2^32 + 2 nodes are 2 in 32 bits; tours that share one element stand for such an array."""
    from ml4tspbench_amd import _lib
    ext, one = _lib.learning_ext(), torch.zeros((1, 1), dtype=torch.int64)
    for nodes in (1 << 16, (1 << 31) + 5, (1 << 32) + 2):
        with pytest.raises(_lib.Tsp2optError, match="65535") as e:
            ext.tour_log_probs(torch.zeros(1, 2, 2), one.expand(1, nodes + 1), 1, 0)
        assert e.value.code == _lib.E_UNSUPPORTED


def test_reference_gradient_matches_differences():
    """The formula the kernels are held to, against central differences in 64 bits."""
    gen = torch.Generator().manual_seed(3)
    h = torch.randn((2, 7, 7), generator=gen)
    tours = make_tours(gen, 6, 7)
    g = torch.randn((6, 6), generator=gen)
    _, _, grad, _ = ref_log_probs(h, tours, 3, "node", g)
    for _ in range(20):
        i = tuple(int(torch.randint(0, s, (1,), generator=gen)) for s in h.shape)
        vals = []
        for step in (1e-4, -1e-4):
            x = h.double()
            x[i] += step
            vals.append(float((ref_log_probs(x, tours, 3, "node")[0] * g.double()).sum()))
        assert abs((vals[0] - vals[1]) / 2e-4 - float(grad[i])) < 1e-6


# ------------------------------------------------------------------------------------------ GPU: log-probabilities
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,per,n", [(1, 1, 2), (3, 1, 3), (2, 3, 5), (2, 1, 33), (1, 2, 64), (3, 5, 65), (2, 16, 50),
                                     (1, 17, 100), (2, 4, 129), (1, 40, 37), (1, 3, 333), (2, 1, 257), (1, 2, 512),
                                     (1, 1, 1025), (1, 3, 1100), (1, 2, 13), (1, 18, 16), (2, 3, 17), (1, 33, 96), (2, 2, 190),
                                     (1, 2, 256), (1, 17, 300), (2, 2, 700), (1, 2, 1024), (1, 2, 2048), (1, 2, 2049),
                                     (1, 17, 2053), (1, 1, 4097)])
def test_gpu_log_probs_of_heat_maps(M, per, n, dtype):
    gen = torch.Generator().manual_seed(n * 100 + per)
    check_log_probs(rows_of(gen, M, n, n, dtype), make_tours(gen, M * per, n, start=True), per, "node", gen)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,n", [(1, 2), (3, 3), (5, 20), (2, 65), (4, 100), (1, 301), (2, 513), (1, 1026), (17, 8), (3, 17),
                                 (2, 193), (1, 255), (2, 257), (1, 769), (1, 2049)])
def test_gpu_log_probs_of_decoder_rows(T, n, dtype):
    gen = torch.Generator().manual_seed(n)
    check_log_probs(rows_of(gen, T, n - 1, n, dtype), make_tours(gen, T, n), 1, "step", gen)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("per", [1, 2, 7])
@pytest.mark.parametrize("kind", ["wide", "inf", "lowest"])
@pytest.mark.parametrize("n", [31, 140, 270, 1030, 2070])
def test_gpu_log_probs_of_masked_and_wide_rows(n, kind, per, dtype):
    """Rows that run out of entries, entries of the type's lowest value, steps whose open entries all lie far below the
    row's largest: where an exponential relative to the row's largest entry has nothing left."""
    gen = torch.Generator().manual_seed(n + per)
    check_log_probs(rows_of(gen, 1, n, n, dtype, kind), make_tours(gen, per, n), per, "node", gen)


@gpu
@pytest.mark.parametrize("dtype", DTYPES[:2], ids=["f32", "bf16"])
@pytest.mark.parametrize("layout,per,n,levels", [                       # spread: one column in seven is high
    ("spread", 2, 15, (0, -90)), ("spread", 18, 140, (0, -90)), ("spread", 3, 140, (0, -35, -90)),
    ("spread", 2, 270, (0, -90)), ("spread", 17, 270, (0, -90)), ("spread", 2, 1030, (0, -90)), ("spread", 2, 2070, (0, -90)),
    ("parts", 1, 1030, (0, -90)), ("parts", 1, 1030, (0, -35)), ("parts", 2, 1030, (0, -35)), ("parts", 2, 1030, (0, -60)),
    ("parts", 1, 2070, (0, -35, -90)), ("parts", 2, 2070, (0, -35, -60)), ("parts", 2, 2070, (0, -60, -90)),
    ("parts", 2, 2070, (-60, 0, -90)), ("parts", 2, 3100, (0, -60, -90, -35))])
def test_gpu_log_probs_of_steps_whose_sum_is_tiny(layout, per, n, levels, dtype):
    """Steps whose open entries lie 35 .. 90 below their row's maximum and still are in its sum, which then is around
    2^-50 .. 2^-130: what long tours end with where a map is sure of its first edges.  The high nodes are visited
    first.  With the levels in blocks of columns every part of a long row has a maximum of its own, far from the
    others'.  The tolerance is the formula's: exponentials at a distance of 100 carry 100 u of the difference and 100 u
    of the argument, the logarithm of such a sum and the difference that is left round 100 u each, below the 8 u (64 + 90)
    that it allows for.  A tour's term g p of the gradient, p = exp(h - m) / S with S >= 1, is lost where the hardware's
    exponential is below 2^-126, the smallest number that it gives (e^-90 is 2^-130): off by |g| 2^-126 a tour."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(n + per)
    j = torch.arange(n)
    parts = (n + 1023) // 1024
    width = (-(-n // parts) + 63) // 64                     # entries a lane, in the steps of 12 and 16 that these sizes take
    width = 64 * (12 if width <= 12 else 16)
    level = torch.tensor(levels, dtype=torch.float32)
    which = (j // width).clamp(max=len(levels) - 1) if layout == "parts" else torch.where(j % 7 == 0, 0, 1 + j % (len(levels) - 1))
    logits = (torch.randn((1, n, n), generator=gen) + level[which]).to(dtype)
    tours = torch.zeros((per, n + 1), dtype=torch.int64)
    for k in range(per):
        noise = torch.rand(n, generator=gen)
        tours[k, :n] = (-level[which] + 0.5 * noise).argsort()
        tours[k, n] = tours[k, 0]
    # such sums are there: base two, relative to the row's maximum without its diagonal
    x = logits[0][tours[0, :-2]].double()
    x[torch.arange(n - 1), tours[0, :-2]] = -math.inf
    top = x.amax(1, keepdim=True)
    seen = (x - top).gather(1, tours[0, None, :n].expand(n - 1, n)).masked_fill_(torch.ones((n - 1, n), dtype=torch.bool).tril(), -math.inf)
    size = seen.logsumexp(1) / math.log(2)
    deep = min(levels)
    assert int(((size < (deep + 6) / math.log(2)) & (size > -139)).sum()) >= 3
    if deep == -90:
        assert int(((size < -121) & (size > -139)).sum()) >= 3
    g = torch.randn((per, n - 1), generator=gen)
    g[torch.rand(g.shape, generator=gen) < 0.1] = 0.0
    lp, tol, grad, gtol = ref_log_probs(logits, tours, per, "node", g)
    heat = logits.cuda().requires_grad_()
    got = amd.tour_log_probs(heat, tours.cuda(), tours_per_map=per)
    (dx,) = torch.autograd.grad(got, heat, g.cuda())
    compare("log-probabilities", got, lp, tol)
    compare("gradient", dx, grad, gtol + per * float(g.abs().max()) * 2.0 ** -126)


@gpu
@pytest.mark.parametrize("per", [1, 3])
@pytest.mark.parametrize("n", [6, 70, 300, 1031, 2060])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 3.0e38])
def test_gpu_log_probs_never_use_visited_entries(value, n, per):
    """The diagonal, and every entry that all tours of the map have visited when its row is read, hold poison."""
    gen = torch.Generator().manual_seed(n)
    tours = make_tours(gen, per, n)
    logits = rows_of(gen, 1, n, n, torch.float32)
    seen = torch.ones((n, n), dtype=torch.bool)
    for t in tours:
        pos = torch.empty(n, dtype=torch.int64)
        pos[t[:n]] = torch.arange(n)
        seen &= pos[None, :] <= pos[:, None]
    assert int(seen.sum()) >= n
    clean, _ = check_log_probs(logits.masked_fill(seen, -5.0), tours, per, "node", gen)
    got, _ = check_log_probs(logits.masked_fill(seen, value), tours, per, "node", gen)
    assert torch.allclose(clean, got, rtol=0, atol=8 * U * (8 + 64))


@gpu
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_gpu_log_probs_pass_on_open_nan_and_inf(value):
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(9)
    n, per = 40, 3
    tours = make_tours(gen, per, n)
    logits = rows_of(gen, 1, n, n, torch.float32)
    logits[0, tours[1, 4], tours[1, 20]] = value            # open for tour 1 at step 4
    got = amd.tour_log_probs(logits.cuda(), tours.cuda(), tours_per_map=per).cpu()
    lp, tol, _, _ = ref_log_probs(logits, tours, per, "node")
    assert math.isnan(float(lp[1, 4])) and math.isnan(float(got[1, 4]))
    keep = lp.isfinite()
    assert torch.equal(keep, got.isfinite()) and bool(((got.double() - lp).abs() <= tol)[keep].all())


@gpu
@pytest.mark.parametrize("rows,per,n", [("node", 1, 40), ("node", 3, 40), ("node", 3, 256), ("node", 3, 300), ("step", 1, 40),
                                        ("node", 2, 1100)])
def test_gpu_log_probs_do_not_depend_on_the_closing_entry(rows, per, n):
    gen = torch.Generator().manual_seed(n)
    tours = make_tours(gen, 2 * per, n)
    logits = rows_of(gen, 2 if rows == "node" else 2 * per, n if rows == "node" else n - 1, n, torch.float32)
    want = check_log_probs(logits, tours, per, rows, torch.Generator().manual_seed(1))
    tours[:, n] = torch.tensor([1 << 40, -1, n, 7])[torch.arange(2 * per) % 4]
    got = check_log_probs(logits, tours, per, rows, torch.Generator().manual_seed(1))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("rows", ["node", "step"])
def test_gpu_log_probs_of_broken_tours(rows):
    """A tour with an index out of range or a repeated node gets NaN and leaves the gradient alone."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(4)
    n, T = 67, 6
    per = 3 if rows == "node" else 1
    tours = make_tours(gen, T, n)
    tours[1, 5] = n
    tours[2, 9] = tours[2, 10]
    tours[4, 3] = -1
    tours[5, n - 1] = 1 << 40
    logits = rows_of(gen, T // per, n if rows == "node" else n - 1, n, torch.float32)
    _, dx = check_log_probs(logits, tours, per, rows, gen)
    got = amd.tour_log_probs(logits.cuda(), tours.cuda(), tours_per_map=per, rows=rows)
    assert got.isnan().all(1).tolist() == [False, True, True, False, True, True]
    assert dx.isfinite().all()


@gpu
def test_gpu_log_probs_layouts_and_small_forms():
    """Padded rows, every other map, transposed maps (copied), one map without its axis, int32 tours, one tour; n = 1."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(8)
    M, n, per = 3, 45, 2
    tours = make_tours(gen, M * per, n)
    logits = rows_of(gen, M, n, n, torch.bfloat16)

    def padded(x):
        big = torch.full((M, n + 2, n + 5), math.nan, dtype=x.dtype, device=x.device)
        big[:, 1:n + 1, 3:n + 3] = x
        return big[:, 1:n + 1, 3:n + 3]

    def spread(x):
        big = torch.full((2 * M, n, n), math.nan, dtype=x.dtype, device=x.device)
        big[::2] = x
        return big[::2]

    plain, dplain = check_log_probs(logits, tours, per, "node", torch.Generator().manual_seed(1))
    for view in (padded, spread, lambda x: x.transpose(1, 2).contiguous().transpose(1, 2)):
        got, dx = check_log_probs(logits, tours, per, "node", torch.Generator().manual_seed(1), view)
        assert torch.equal(got, plain) and torch.equal(dx, dplain)
    one = amd.tour_log_probs(logits[1].cuda(), tours[2].to(torch.int32).cuda())
    assert one.shape == (1, n - 1)
    x = torch.zeros((4, 1, 1), device="cuda", requires_grad=True)
    none = amd.tour_log_probs(x, torch.zeros((4, 2), dtype=torch.int64, device="cuda"))
    assert none.shape == (4, 0)
    none.sum().backward()
    assert torch.equal(x.grad, torch.zeros_like(x))
    empty = amd.tour_log_probs(torch.zeros((0, 5, 5), device="cuda"), torch.zeros((0, 6), dtype=torch.int64, device="cuda"))
    assert empty.shape == (0, 4)


@gpu
@pytest.mark.parametrize("per,n", [(1, 60), (5, 60)])
def test_gpu_log_probs_gradient_against_differences(per, n):
    """Directional differences of the kernel's own values.  They are off by the values' rounding, below 8 u * 30 each
    and added up over the steps by the root of their number, over twice the step, and by step^2 |d3| / 6, where a third
    derivative along a direction of entries at most 1 is below 8 times the sum of |g|."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(n + per)
    tours = make_tours(gen, per, n).cuda()
    h = rows_of(gen, 1, n, n, torch.float32).cuda().requires_grad_()
    g = torch.randn((per, n - 1), generator=gen).cuda()
    (grad,) = torch.autograd.grad(amd.tour_log_probs(h, tours, tours_per_map=per), h, g)
    step = 0.02
    for _ in range(4):
        way = torch.sign(torch.randn((1, n, n), generator=gen)).cuda()
        f = [(amd.tour_log_probs(h.detach() + s * way, tours, tours_per_map=per).double() * g).sum() for s in (step, -step)]
        size = float(g.abs().sum())
        tol = 8 * U * 30 * size / step + step ** 2 / 6 * 8 * size
        assert abs(float((f[0] - f[1]) / (2 * step) - (grad.double() * way).sum())) < tol


@gpu
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -60, 2.0 ** 40, 2.0 ** 90])
@pytest.mark.parametrize("per,n", [(1, 40), (3, 40), (3, 300), (20, 300), (2, 1100), (2, 2100)])
def test_gpu_log_probs_gradients_of_any_size(per, n, size):
    """Incoming gradients far from 1 (a saturated preference loss sends such): a power of two passes through exactly,
    entries of 2^-20 of it and more stay normal numbers."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(n + per)
    tours = make_tours(gen, per, n)
    h = torch.rand((1, n, n), generator=gen)
    g = torch.randn((per, n - 1), generator=gen)
    x = h.cuda().requires_grad_()
    lp = amd.tour_log_probs(x, tours.cuda(), tours_per_map=per)
    (grad,) = torch.autograd.grad(lp, x, g.cuda() * size)
    _, _, want, tol = ref_log_probs(h, tours, per, "node", g)
    compare("gradient", grad.double().cpu() / size, want, tol)


@gpu
def test_gpu_log_probs_large_offsets():
    """Rows behind 2^31 bytes and behind 2^31 elements of a batch of maps."""
    import ml4tspbench_amd as amd
    n, M = 4096, 130
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    logits = torch.zeros((M, n, n), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(2)
    last = rows_of(gen, 1, n, n, torch.bfloat16)
    logits[M - 1] = last[0].cuda()
    tours = make_tours(gen, 1, n).expand(M, n + 1).contiguous()
    x = logits.requires_grad_()
    lp = amd.tour_log_probs(x, tours.cuda())
    (grad,) = torch.autograd.grad(lp, x, torch.ones_like(lp))
    want, tol, wgrad, wtol = ref_log_probs(last, tours[:1], 1, "node", torch.ones((1, n - 1)))
    compare("log-probabilities", lp[M - 1:], want, tol)
    compare("gradient", grad[M - 1:], wgrad, wtol)
    flat = -torch.log(torch.arange(n - 1, 0, -1, dtype=torch.float64))
    compare("flat rows", lp[M - 2:M - 1], flat[None], 8 * U * 12)


# ------------------------------------------------------------------------------------------ GPU: losses
def policy_inputs(gen, T, S, dtype, per_step, with_ref, with_mask):
    old = -2 * torch.rand((T, S), generator=gen) ** 2 - 0.01
    lp = (old + 0.3 * torch.randn((T, S), generator=gen)).to(dtype)
    ref = (old + 0.7 * torch.randn((T, S), generator=gen)).to(dtype) if with_ref else None
    old = old.to(dtype)
    adv = torch.randn((T, S) if per_step else (T,), generator=gen)
    adv.view(-1)[:: 5] = 0.0
    mask = None
    if with_mask:
        mask = torch.rand((T, S), generator=gen) < 0.7
        mask[0] = False
        for x in (lp, old, ref):
            if x is not None:
                x[~mask] = math.nan
    return lp, old, ref, adv, mask


def check_policy(lp, old, ref, adv, mask, ratio, average, kl_coef, low=0.2, high=0.3):
    import ml4tspbench_amd as amd
    x = lp.cuda().requires_grad_()
    dev = [None if v is None else v.cuda() for v in (old, adv, ref, mask)]
    res = amd.clipped_policy_loss(x, dev[0], dev[1], ref_log_probs=dev[2], mask=dev[3], clip_low=low, clip_high=high,
                                  kl_coef=kl_coef, ratio=ratio, average=average)
    (dx,) = torch.autograd.grad(res.loss, x, torch.tensor(1.5, device="cuda"))
    loss, kl, clip, grad, size = ref_policy(lp, old, adv, ref, mask, low, high, kl_coef, ratio, average or ratio)
    # the float exponential is good to 2 ulp of a rounded argument (|x| below 8 here: 2 u + 8 u), advantages and clip
    # borders round once each; the KL series and its coefficient the same; sums are in double
    compare("kl", res.kl, kl, 16 * U * float(kl))
    compare("clip fraction", res.clip_fraction, clip, 2 * U * float(clip))
    compare("loss", res.loss, loss, 16 * U * (size + kl_coef * float(kl)))
    count = max(1, int(mask.sum()) if mask is not None else lp.numel())
    part = 1.5 * kl_coef * 16 * U * 8 * max(1.0 / count, 1.0 / max(1, lp.shape[0]))      # KL and ratio parts may cancel
    eps = torch.finfo(lp.dtype).eps / 2
    compare("gradient", dx, 1.5 * grad, 24 * U * 1.5 * grad.abs() + part + eps * 1.5 * grad.abs() +
            torch.finfo(lp.dtype).smallest_normal * eps)
    assert dx.dtype == lp.dtype


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("ratio,average,per_step", [("step", None, False), ("step", "step", True), ("step", "tour", False),
                                                    ("step", "tour", True), ("tour", None, False)])
@pytest.mark.parametrize("T,S,ref,mask", [(1, 1, False, False), (3, 1, True, True), (16, 49, False, False),
                                          (7, 130, True, True), (5, 64, True, False), (300, 9, False, True),
                                          (1, 3000, True, True), (2, 9000, False, False), (4500, 3, True, True)])
def test_gpu_policy_loss(T, S, ref, mask, ratio, average, per_step, dtype):
    gen = torch.Generator().manual_seed(T * 31 + S)
    lp, old, r, adv, m = policy_inputs(gen, T, S, dtype, per_step, ref, mask)
    if ratio == "tour":         # whole-tour differences of the size of a step's
        lp = (torch.where(lp.isnan(), lp, old) + (0.3 / math.sqrt(S) * torch.randn((T, S), generator=gen)).to(dtype)).to(dtype)
    check_policy(lp, old, r, adv, m, ratio, average, 0.05 if ref else 0.0)


@gpu
def test_gpu_policy_loss_edges():
    """Nothing kept, no steps, no tours, a ratio on the border, impossible steps, KL of equal policies, strides."""
    import ml4tspbench_amd as amd
    lp = torch.zeros((3, 4), device="cuda", requires_grad=True)
    adv = torch.ones(3, device="cuda")
    none = torch.zeros((3, 4), dtype=torch.bool, device="cuda")
    for kind in ("step", "tour"):
        res = amd.clipped_policy_loss(lp, lp, adv, ref_log_probs=lp, mask=none, kl_coef=1.0, ratio=kind)
        assert [float(v.detach()) for v in (res.loss, res.kl, res.clip_fraction)] == [0.0, 0.0, 0.0]
        assert torch.equal(torch.autograd.grad(res.loss, lp)[0], torch.zeros_like(lp))
        for shape in ((3, 0), (0, 4)):
            e = torch.zeros(shape, device="cuda", requires_grad=True)
            r = amd.clipped_policy_loss(e, e, torch.zeros(shape[0], device="cuda"), ratio=kind)
            assert float(r.loss.detach()) == 0.0 and torch.autograd.grad(r.loss, e)[0].shape == shape
        res = amd.clipped_policy_loss(lp, lp, adv, ref_log_probs=lp, kl_coef=1.0, ratio=kind)
        assert float(res.kl) == 0.0 and float(res.loss.detach()) == -1.0
    x = torch.tensor([[-math.inf, -1.0]], device="cuda", requires_grad=True)      # ruled out since it was drawn: r = 0
    old = torch.tensor([[-2.0, -1.0]], device="cuda")
    res = amd.clipped_policy_loss(x, old, torch.ones(1, device="cuda"))
    assert float(res.loss.detach()) == -0.5 and torch.autograd.grad(res.loss, x)[0].tolist() == [[0.0, -0.5]]
    gen = torch.Generator().manual_seed(12)
    lp, old, ref, adv, mask = policy_inputs(gen, 9, 31, torch.float32, True, True, True)
    wide = torch.zeros((9, 62))
    wide[:, ::2] = lp
    a = amd.clipped_policy_loss(wide.cuda()[:, ::2], old.cuda(), adv.cuda(), ref_log_probs=ref.cuda(), mask=mask.cuda())
    b = amd.clipped_policy_loss(lp.cuda(), old.t().contiguous().t().cuda(), adv.cuda(), ref_log_probs=ref.cuda(),
                                mask=mask.cuda())
    assert torch.equal(a.loss, b.loss) and torch.equal(a.kl, b.kl)


@gpu
@pytest.mark.parametrize("ratio,average,per_step", [("step", "step", False), ("step", "step", True), ("step", "tour", False),
                                                    ("tour", "tour", False)])
def test_gpu_policy_loss_of_zero_advantages_and_far_ratios(ratio, average, per_step):
    """A tour of advantage 0 (an instance whose tours are equally long) adds nothing, however far its ratio has gone:
    e^100 is past the range of float, its product with 0 is 0."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(17)
    T, S = 6, 50
    old = -torch.rand((T, S), generator=gen) - 0.5
    lp = old + 0.02 * torch.randn((T, S), generator=gen)
    adv = torch.randn(T, generator=gen)
    old[1, 7] -= 100.0
    old[2] -= 2.5                       # 125 for the tour
    old[3, 0] = -math.inf               # e^inf is no number that 0 would win over: masked
    adv[1:4] = 0.0
    mask = torch.ones((T, S), dtype=torch.bool)
    mask[3, 0] = False
    if per_step:
        adv = adv[:, None].expand(T, S).contiguous()
    check_policy(lp, old, None, adv, mask, ratio, average, 0.0)
    x = lp.cuda().requires_grad_()
    res = amd.clipped_policy_loss(x, old.cuda(), torch.zeros_like(adv).cuda(), mask=mask.cuda(), ratio=ratio, average=average)
    assert float(res.loss.detach()) == 0.0 and float(res.clip_fraction) == 0.0
    assert not torch.autograd.grad(res.loss, x)[0].any()
    lost = amd.clipped_policy_loss(x, old.cuda(), adv.cuda(), ratio=ratio, average=average)      # and unmasked it is NaN
    assert math.isnan(float(lost.loss.detach()))


@gpu
@pytest.mark.parametrize("ratio,average,per_step", [("step", "step", False), ("step", "step", True), ("step", "tour", False),
                                                    ("tour", "tour", False)])
@pytest.mark.parametrize("T,S", [(200, 50), (3, 5000)])
def test_gpu_policy_loss_of_terms_past_the_range_of_float(T, S, ratio, average, per_step):
    """Single terms above 3.4e38 in averages below it: sums are in double, so are such terms.  e^95 carries the rounding
    of its argument, 95 u, the exponential's own 2 ulp and a handful of products: below 8 u (4 + 95) of it."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(18)
    lp = -torch.rand((T, S), generator=gen) - 0.5
    old = lp - 0.01 * torch.randn((T, S), generator=gen) / math.sqrt(S)
    ref = lp + 0.3 * torch.randn((T, S), generator=gen)
    adv = torch.randn(T, generator=gen)
    adv[1:] = -adv[1:].abs()                # where the ratio may grow
    far = 95.0 if average == "step" else 89.5           # averages of tours divide by less
    old[1, 3] -= far
    ref[T - 1, S // 2] += far               # another tour: the gradient's parts do not cancel
    lp[2, 0] += 60.0                        # far, and within the range
    adv_in = adv[:, None].expand(T, S).contiguous() if per_step else adv
    x = lp.cuda().requires_grad_()
    coef = 0.1 if average == "step" else 0.01
    res = amd.clipped_policy_loss(x, old.cuda(), adv_in.cuda(), ref_log_probs=ref.cuda(), kl_coef=coef, ratio=ratio,
                                  average=average)
    (dx,) = torch.autograd.grad(res.loss, x, torch.tensor(0.001, device="cuda"))
    loss, kl, clip, grad, size = ref_policy(lp, old, adv_in, ref, None, 0.2, 0.2, coef, ratio, average)
    share = 8 * U * (4 + 95)
    for name, got, want in (("loss", res.loss, loss), ("kl", res.kl, kl), ("gradient", dx, 0.001 * grad)):
        ok = want.abs() <= torch.finfo(torch.float32).max           # a result past it is inf
        assert torch.equal(got.detach().isfinite().cpu(), ok), name
        compare(name, got.detach().cpu()[ok], want[ok], share * want.abs()[ok] + share * 0.001 * coef)
    assert float(loss) > 1e30


@gpu
def test_gpu_policy_loss_small_kl_keeps_its_digits():
    """d of 1e-4: exp(d) - 1 - d is 5e-9, of which float32 subtraction would leave nothing."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(1)
    lp = -torch.rand((8, 50), generator=gen) - 0.5
    ref = lp + 1e-4 * torch.randn((8, 50), generator=gen)
    d = ref.double() - lp.double()
    res = amd.clipped_policy_loss(lp.cuda(), lp.cuda(), torch.zeros(8, device="cuda"), ref_log_probs=ref.cuda())
    want = (torch.expm1(d) - d).mean()
    compare("kl", res.kl, want, 8 * U * float(want))


def check_preference(lp, length, per, ref, mask, beta, eps, pairs, per_step):
    import ml4tspbench_amd as amd
    x = lp.cuda().requires_grad_()
    dev = [None if v is None else v.cuda() for v in (ref, mask)]
    res = amd.preference_loss(x, length.cuda(), tours_per_instance=per, ref_log_probs=dev[0], mask=dev[1], beta=beta,
                              label_smoothing=eps, pairs=pairs, per_step=per_step)
    (dx,) = torch.autograd.grad(res.loss, x, torch.tensor(0.5, device="cuda"))
    loss, count, grad = ref_preference(lp, length, per, ref, mask, beta, eps, pairs, per_step)
    assert int(res.num_pairs) == count and res.num_pairs.dtype == torch.int64
    # a score difference z is rounded to float once (u |z|; |z| <= loss + 1 where it is felt), the exponential and the
    # logarithm cost 4 u; a pair's derivative is at most 1, off by 9 u, and a tour is in at most `per` pairs
    compare("loss", res.loss, loss, 16 * U * (float(loss) + 1))
    half = torch.finfo(lp.dtype).eps / 2
    compare("gradient", dx, 0.5 * grad, 0.5 * ((half + 16 * U) * grad.abs() + 16 * U * beta * per / max(count, 1)) +
            torch.finfo(lp.dtype).smallest_normal * half)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("pairs,per_step,eps", [("all", False, 0.0), ("best", True, 0.1), ("all", True, 0.2)])
@pytest.mark.parametrize("I,per,S,ref,mask", [(1, 2, 1, False, False), (3, 1, 5, True, True), (5, 7, 37, False, True),
                                              (2, 16, 130, True, False), (40, 3, 9, True, True), (1, 70, 3, False, False),
                                              (1, 300, 2, True, True), (700, 2, 20, False, False), (2, 2, 2500, True, True)])
def test_gpu_preference_loss(I, per, S, ref, mask, pairs, per_step, eps, dtype):
    gen = torch.Generator().manual_seed(I + 10 * per + S)
    T = I * per
    lp = (-torch.rand((T, S), generator=gen)).to(dtype)
    r = (-torch.rand((T, S), generator=gen)).to(dtype) if ref else None
    m = None
    if mask:
        m = torch.rand((T, S), generator=gen) < 0.6
        m[0] = False
        for x in (lp, r):
            if x is not None:
                x[~m] = math.nan
    length = torch.rand(T, generator=gen, dtype=torch.float64) + 5
    length[:: 3] = 5.5                                  # ties
    if T > 5:
        length[4] = math.nan
    check_preference(lp, length, per, r, m, 0.7, eps, pairs, per_step)


@gpu
def test_gpu_preference_loss_edges():
    """Equal lengths, one tour an instance, NaN lengths, float32 lengths, far scores, no tours, no steps."""
    import ml4tspbench_amd as amd
    lp = torch.randn((4, 3), device="cuda", requires_grad=True)
    for length, per in ((torch.ones(4), 4), (torch.arange(4.0), 1), (torch.full((4,), math.nan), 2)):
        res = amd.preference_loss(lp, length.cuda(), tours_per_instance=per)
        assert float(res.loss.detach()) == 0.0 and int(res.num_pairs) == 0
        assert torch.equal(torch.autograd.grad(res.loss, lp)[0], torch.zeros_like(lp))
    a = amd.preference_loss(lp, torch.tensor([1.0, 2, 3, 4]).cuda(), tours_per_instance=2)
    b = amd.preference_loss(lp, torch.tensor([1.0, 2, 3, 4], dtype=torch.float64).cuda(), tours_per_instance=2)
    assert torch.equal(a.loss, b.loss) and int(a.num_pairs) == 2
    never = torch.tensor([[-math.inf], [1.0], [2.0], [-math.inf]], device="cuda", requires_grad=True)
    for order, eps, want in (([1.0, 2, 2, 1], 0.0, math.inf), ([2.0, 1, 1, 2], 0.0, 0.0), ([1.0, 2, 2, 1], 0.1, math.inf),
                             ([2.0, 1, 1, 2], 0.1, math.inf)):
        res = amd.preference_loss(never, torch.tensor(order).cuda(), tours_per_instance=2, label_smoothing=eps)
        assert float(res.loss.detach()) == want
        assert torch.autograd.grad(res.loss, never)[0].isfinite().all()
    far = torch.tensor([[-300.0], [300.0], [200.0], [-200.0]])
    check_preference(far, torch.tensor([1.0, 2, 1, 2]), 2, None, None, 1.0, 0.0, "all", False)
    for shape in ((0, 3), (4, 0)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        res = amd.preference_loss(x, torch.arange(float(shape[0])).cuda(), tours_per_instance=2)
        assert int(res.num_pairs) == (0 if shape[0] == 0 else 2)
        assert abs(float(res.loss.detach()) - (0.0 if shape[0] == 0 else math.log(2))) < 1e-6
        assert torch.autograd.grad(res.loss, x)[0].shape == shape


@gpu
@pytest.mark.parametrize("pairs", ["all", "best"])
@pytest.mark.parametrize("per", [1, 64, 65, 100, 1 << 33])
def test_gpu_preference_loss_of_no_tours(per, pairs):
    """An empty batch has no pair, however many tours an instance would have."""
    import ml4tspbench_amd as amd
    for steps in (0, 3, 20000):
        x = torch.zeros((0, steps), device="cuda", requires_grad=True)
        res = amd.preference_loss(x, torch.zeros(0, device="cuda"), tours_per_instance=per, pairs=pairs)
        assert float(res.loss.detach()) == 0.0 and int(res.num_pairs) == 0
        assert torch.autograd.grad(res.loss, x)[0].shape == x.shape


# ------------------------------------------------------------------------------------------ GPU: streams, graphs, runs
def whole_step(heat, tours, old, adv, length, per):
    """One training step's worth of calls: value, both losses, the heat maps' gradient."""
    import ml4tspbench_amd as amd
    lp = amd.tour_log_probs(heat, tours, tours_per_map=per)
    res = amd.clipped_policy_loss(lp, old, adv, ref_log_probs=old, kl_coef=0.1, ratio="tour")
    pref = amd.preference_loss(lp, length, tours_per_instance=per, beta=0.05)
    (grad,) = torch.autograd.grad(res.loss + 0.3 * pref.loss, heat)
    return lp.detach(), res.loss.detach(), pref.loss.detach(), grad


def step_inputs(seed, M=4, per=6, n=75):
    gen = torch.Generator().manual_seed(seed)
    heat = rows_of(gen, M, n, n, torch.float32).cuda()
    tours = make_tours(gen, M * per, n).cuda()
    import ml4tspbench_amd as amd
    old = amd.tour_log_probs(heat, tours, tours_per_map=per) + 0.02 * torch.randn((M * per, n - 1), generator=gen).cuda()
    return heat, tours, old, torch.randn(M * per, generator=gen).cuda(), torch.rand(M * per, generator=gen).double().cuda(), per


@gpu
def test_gpu_runs_are_bit_identical_and_streams_do_not_share():
    a, b = step_inputs(1), step_inputs(2)
    want = [whole_step(x[0].requires_grad_(), *x[1:]) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(whole_step(x[0], *x[1:]))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(p, q) for p, q in zip(run, want[i]))


@gpu
def test_gpu_captured_step_replays_like_the_eager_one():
    """Two captured steps, forward and backward, replayed in turn with new inputs in their buffers and eager calls and
    synchronisations in between."""
    fixed = [[t.clone() if isinstance(t, torch.Tensor) else t for t in step_inputs(s)] for s in (3, 4)]
    for f in fixed:
        f[0].requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for f in fixed:
            whole_step(*f)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for f in fixed:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(whole_step(*f))
        graphs.append(graph)
    for seed in range(10, 14):
        fresh = [step_inputs(seed), step_inputs(seed + 100)]
        want = [whole_step(x[0].requires_grad_(), *x[1:]) for x in fresh]
        for f, x in zip(fixed, fresh):
            with torch.no_grad():
                for p, q in zip(f[:5], x[:5]):
                    p.copy_(q)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(o, w))


@gpu
def test_gpu_without_gradients():
    """no_grad, inference mode and inputs that need none: the same values, nothing kept."""
    import ml4tspbench_amd as amd
    heat, tours, old, adv, length, per = step_inputs(6)
    want = amd.tour_log_probs(heat.clone().requires_grad_(), tours, tours_per_map=per)
    pol, pref = amd.clipped_policy_loss(want, old, adv), amd.preference_loss(want, length, tours_per_instance=per)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            got = amd.tour_log_probs(heat.clone(), tours.clone(), tours_per_map=per)
            a = amd.clipped_policy_loss(got, old.clone(), adv.clone(), mask=torch.ones_like(got, dtype=torch.bool))
            b = amd.preference_loss(got, length.clone(), tours_per_instance=per)
        assert not got.requires_grad and torch.equal(got, want.detach())
        assert torch.equal(a.loss, pol.loss.detach()) and torch.equal(b.loss, pref.loss.detach())
    assert not amd.tour_log_probs(heat, tours, tours_per_map=per).requires_grad


@gpu
def test_gpu_broadcast_maps_and_graph_kept_for_two_backwards():
    """One heat map expanded over several entries of the batch: its gradient is their sum; a graph used twice."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(14)
    n, M, per = 55, 3, 2
    tours = make_tours(gen, M * per, n).cuda()
    one = rows_of(gen, 1, n, n, torch.float32).cuda()
    a, b = one.clone().requires_grad_(), one.expand(M, n, n).contiguous().requires_grad_()
    g = torch.randn((M * per, n - 1), generator=gen).cuda()
    lp = amd.tour_log_probs(a.expand(M, n, n), tours, tours_per_map=per)
    first = torch.autograd.grad(lp, a, g, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(lp, a, g)[0])
    want = amd.tour_log_probs(b, tours, tours_per_map=per)
    assert torch.equal(lp.detach(), want.detach())
    (each,) = torch.autograd.grad(want, b, g)
    assert torch.allclose(first, each.sum(0, keepdim=True), rtol=4 * U * M, atol=4 * U * M * float(each.abs().max()))


@gpu
def test_gpu_second_derivative_and_changed_input_are_refused():
    import ml4tspbench_amd as amd
    heat, tours, *_, per = step_inputs(5)
    heat.requires_grad_()
    lp = amd.tour_log_probs(heat, tours, tours_per_map=per)
    (g,) = torch.autograd.grad(lp.sum(), heat, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    lp = amd.tour_log_probs(heat, tours, tours_per_map=per)
    with torch.no_grad():
        heat.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lp.sum().backward()


@gpu
@pytest.mark.parametrize("op", ["log_probs", "log_probs_strided", "policy", "preference", "one_node"])
def test_gpu_second_derivatives_raise_and_are_not_dropped(op):
    """With create_graph the gradient requires grad, and whatever derivative needs its own raises: alone, mixed with the
    operator's value (as a gradient penalty is), by backward() and by grad() in the leaf or in the incoming gradient."""
    import ml4tspbench_amd as amd
    heat, tours, old, adv, length, per = step_inputs(7, M=2, per=2, n=20)
    x = (heat if op.startswith("log") else torch.zeros((3, 1, 1), device="cuda") if op == "one_node" else old.detach()
         ).clone().requires_grad_()

    def value(x):
        if op == "policy":
            return amd.clipped_policy_loss(x, old, adv).loss
        if op == "preference":
            return amd.preference_loss(x, length, tours_per_instance=per).loss
        if op == "one_node":
            return amd.tour_log_probs(x, torch.zeros((3, 2), dtype=torch.int64, device="cuda")).sum()
        return amd.tour_log_probs(x.transpose(1, 2) if op.endswith("strided") else x, tours, tours_per_map=per).sum()

    weight = torch.ones((), device="cuda", requires_grad=True)
    (plain,) = torch.autograd.grad(value(x), x)
    for ask in (lambda g: torch.autograd.grad(value(x) + g.pow(2).sum(), x), lambda g: g.sum().backward(),
                lambda g: (value(x) + g.pow(2).sum()).backward(), lambda g: torch.autograd.grad(g.sum() + weight, weight)):
        (g,) = torch.autograd.grad(value(x) * weight, x, create_graph=True)
        assert g.requires_grad and torch.equal(g.detach(), plain) and not plain.requires_grad
        with pytest.raises(RuntimeError, match="no second derivative"):
            ask(g)
    (g,) = torch.autograd.grad(value(x) * weight, x, create_graph=True)         # not reached: nothing raises
    assert torch.equal(torch.autograd.grad(value(x) + g.detach().sum(), x)[0], plain)


@gpu
def test_gpu_refusals_of_the_library_keep_their_code():
    import ml4tspbench_amd as amd
    from ml4tspbench_amd import _lib
    n = 70000                                               # rows that share their memory
    heat = torch.zeros(n, device="cuda").as_strided((1, n, n), (0, 0, 1)).requires_grad_()
    with pytest.raises(_lib.Tsp2optError, match="65535") as e:
        amd.tour_log_probs(heat, torch.arange(n + 1, device="cuda")[None])
    assert e.value.code == _lib.E_UNSUPPORTED


@gpu
@pytest.mark.parametrize("op", ["log_probs", "policy", "preference"])
def test_gpu_function_transforms_and_forward_mode_raise(op):
    """vmap, torch.func.grad and forward-mode derivatives are not offered: they raise instead of giving something else."""
    import ml4tspbench_amd as amd
    heat, tours, old, adv, length, per = step_inputs(8, M=2, per=2, n=20)
    x = heat if op == "log_probs" else old.detach()

    def value(x):
        if op == "policy":
            return amd.clipped_policy_loss(x, old, adv).loss
        if op == "preference":
            return amd.preference_loss(x, length, tours_per_instance=per).loss
        return amd.tour_log_probs(x, tours, tours_per_map=per).sum()

    value(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(value)(x)
    with pytest.raises(RuntimeError):
        torch.func.vmap(value)(torch.stack([x, x]))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(value, (x,), (torch.ones_like(x),))
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        value(fwd.make_dual(x, torch.ones_like(x)))
    value(x)


@gpu
def test_gpu_run_of_decoder_two_opt_evaluation_and_losses():
    """As they are used: tours of heat maps are scored, improved, measured, and the losses' gradient comes back to the
    maps; every value against the formulas, chained in 64 bits on the CPU."""
    import ml4tspbench_amd as amd
    gen = torch.Generator().manual_seed(21)
    I, per, n = 3, 4, 48
    pts = torch.rand((I, n, 2), generator=gen, dtype=torch.float64)
    heat = (-torch.cdist(pts, pts) * math.sqrt(n) / 0.35).float()
    maps = heat.repeat_interleave(per, 0).exp() * (0.5 + torch.rand((I * per, n, n), generator=gen))
    start = amd.greedy_decode_device(maps.cuda(), pts.cuda(), maps_per_instance=per)
    better = amd.two_opt_device(pts.cuda(), start, tours_per_instance=per).tours
    tours = torch.stack([start.view(I, per, -1), better.view(I, per, -1)], 2).reshape(I * per * 2, n + 1)
    ev = amd.evaluate_tours(pts.cuda(), tours, tours_per_instance=2 * per)
    x = heat.cuda().requires_grad_()
    lp = amd.tour_log_probs(x, tours, tours_per_map=2 * per)
    length = ev.lengths.view(I, -1)
    adv = (length.mean(1, keepdim=True) - length).flatten()
    pol = amd.clipped_policy_loss(lp, lp.detach(), adv)
    pref = amd.preference_loss(lp, ev.lengths, tours_per_instance=2 * per, beta=0.1)
    (grad,) = torch.autograd.grad(pol.loss + pref.loss, x)
    want, tol, _, _ = ref_log_probs(heat, tours.cpu(), 2 * per, "node")
    compare("log-probabilities", lp.detach(), want, tol)
    y = lp.detach().cpu()
    l1, _, _, g1, _ = ref_policy(y, y, adv.cpu().float(), None, None, 0.2, 0.2, 0.0, "step", "step")
    l2, count, g2 = ref_preference(y, ev.lengths.cpu(), 2 * per, None, None, 0.1, 0.0, "all", False)
    assert int(pref.num_pairs) == count > 0
    compare("losses", pol.loss.detach() + pref.loss.detach(), l1 + l2, 32 * U * (float(adv.abs().mean()) + float(l2) + 1))
    _, _, g, gtol = ref_log_probs(heat, tours.cpu(), 2 * per, "node", (g1 + g2).float())
    slack = 64 * U * float((g1.abs() + g2.abs()).max()) * 2 * per
    compare("gradient", grad, g, gtol + slack)
