"""What is measured of the fine-tuning operators (token log-probabilities, clipped policy loss, preference loss, gradient
norm and clipped Adam step): the cases, their inputs, each operator in its plain form in elementary torch operations,
and the calls of include/znn_cuda.h that a user makes instead.  Logits, log-probabilities and gradients are float32,
targets int32, as everywhere in this framework."""
import math

import torch

own = False


def _f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


# Clip range, coefficients, optimizer settings: usual ones of such training runs, as the float arguments that calls take.
CLIP_LOW, CLIP_HIGH, KL_COEF, ENTROPY_COEF = map(_f32, (0.2, 0.28, 0.04, 0.01))
BETA, SMOOTHING = map(_f32, (0.1, 0.05))
LR, BETA1, BETA2, EPS, STEP = map(_f32, (3e-4, 0.9, 0.95, 1e-8, 100.0))


def listed():
    return [
        # scoring one step of a small batch of generated sequences: latency counts
        {"name": "logprob 8 x 8192", "op": "logprob", "rows": 8, "vocab": 8192, "pad": 0, "temp": 1.0, "entropy": False, "left_out": 0.0},
        # scoring a packed batch under a vocabulary of odd size: rows start at every alignment; prompts are left out
        {"name": "logprob 2045 x 50257", "op": "logprob", "rows": 2045, "vocab": 50257, "pad": 0, "temp": 0.7, "entropy": True, "left_out": 0.2},
        # gradient of a handful of short answers, added to what the logits' gradient already holds
        {"name": "logprob_grad 300 x 32003", "op": "logprob_grad", "rows": 300, "vocab": 32003, "pad": 0, "temp": 1.0, "entropy": False,
         "left_out": 0.3, "accumulate": True},
        # the GPT of the benchmark: 8 sequences of 1024, vocabulary 8192
        {"name": "logprob_grad 8192 x 8192", "op": "logprob_grad", "rows": 8192, "vocab": 8192, "pad": 0, "temp": 1.0, "entropy": True,
         "left_out": 0.1, "accumulate": False},
        # a policy step on one short answer of the GPT
        {"name": "policy 61 x 8192", "op": "policy", "rows": 61, "vocab": 8192, "pad": 0, "temp": 1.0, "kl": True, "entropy": False, "left_out": 0.1,
         "weighted": False},
        # a policy step over long answers with a large vocabulary whose rows are padded; the largest logits
        {"name": "policy 2048 x 131000", "op": "policy", "rows": 2048, "vocab": 131000, "pad": 72, "temp": 0.8, "kl": True, "entropy": True,
         "left_out": 0.15, "weighted": True},
        # four pairs of short answers
        {"name": "preference 4 pairs", "op": "preference", "pairs": 4, "rows": 163, "reference": True, "by_length": False, "left_out": 0.0},
        # a large batch of ragged long pairs, prompts left out
        {"name": "preference 700 pairs", "op": "preference", "pairs": 700, "rows": 1400021, "reference": True, "by_length": True, "left_out": 0.3},
        # the six tensors of the 784-128-64-10 network
        {"name": "grad_norm mlp", "op": "grad_norm", "layers": 0, "width": 128, "vocab": 784},
        # every tensor of a 12-layer transformer of width 640
        {"name": "grad_norm 12 layers", "op": "grad_norm", "layers": 12, "width": 640, "vocab": 8192},
        # the whole optimizer step of a small network: one slab
        {"name": "clip_adam 109 k", "op": "clip_adam", "count": 109386, "clipped": True},
        # the optimizer step of a model of the benchmark's class
        {"name": "clip_adam 98 M", "op": "clip_adam", "count": 98304007, "clipped": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprob", "logprob_grad", "policy", "preference", "grad_norm", "clip_adam"])
    if op in ("logprob", "logprob_grad", "policy"):
        vocab = _log(rng, 10, 140000)
        rows = _log(rng, 1, max(2, min(65536, 250000000 // (vocab + 64))))
        case = {"op": op, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, 3, 64]), "temp": rng.choice([1.0, 0.7, 1.25]),
                "entropy": rng.random() < 0.5, "left_out": rng.choice([0.0, 0.1, 0.5])}
        if op == "logprob_grad":
            case["accumulate"] = rng.random() < 0.5
        if op == "policy":
            case["kl"] = rng.random() < 0.6
            case["weighted"] = rng.random() < 0.4
        return case
    if op == "preference":
        return {"op": op, "pairs": _log(rng, 1, 2000), "rows": _log(rng, 2, 8000000), "reference": rng.random() < 0.8,
                "by_length": rng.random() < 0.5, "left_out": rng.choice([0.0, 0.2, 0.6])}
    if op == "grad_norm":
        return {"op": op, "layers": rng.randrange(0, 25), "width": rng.randrange(33, 1025), "vocab": _log(rng, 100, 40000)}
    return {"op": op, "count": _log(rng, 1, 98000000), "clipped": rng.random() < 0.7}


def _shapes(case):
    """The tensors' sizes of a model: an input matrix, per layer two gains, four square and two 2-fold products with
    biases, an output matrix with bias; no layers: a three-layer network on `vocab` inputs."""
    w, v = case["width"], case["vocab"]
    if case["layers"] == 0:
        return [v * w, w, w * (w // 2), w // 2, (w // 2) * 10, 10]
    layer = [w, w] + [w * w, w] * 4 + [2 * w * w, 2 * w, 2 * w * w, w]
    return [v * w, 1024 * w] + layer * case["layers"] + [w, w * v, v]


def _policy_inputs(case, g):
    """Logits as a language model gives them: noise plus a raised logit at the token that was taken, and a band of
    columns that are switched off (-inf) in every row; rows of prompts and padding carry target -1."""
    M, N, ld = case["rows"], case["vocab"], case["vocab"] + case["pad"]
    buf = torch.randn(M, ld, device="cuda", generator=g)
    x = buf[:, :N]
    x.mul_(2.0)
    targets = torch.randint(0, N, (M,), device="cuda", generator=g)
    taken = targets.unsqueeze(1)
    if N > 64:
        x[:, N // 2:N // 2 + N // 50] = -math.inf
    raised = 6.0 + 2.0 * torch.randn(M, 1, device="cuda", generator=g)
    x.scatter_(1, taken, raised)
    keep = torch.rand(M, device="cuda", generator=g) >= case["left_out"]
    keep[0] = True
    return buf, torch.where(keep, targets, -1).to(torch.int32)


def _off_border(ratio):
    """Moves ratios that lie within 1e-4 of a clip border away from it: there the gradient jumps, and rounding would
    decide between two right answers."""
    for border in (1.0 - CLIP_LOW, 1.0 + CLIP_HIGH):
        near = (ratio - border).abs() < 1e-4
        ratio = torch.where(near, border + 3e-4, ratio)
    return ratio


def _rows_logp(x, targets, inv_temp):
    """log-probabilities of the taken tokens, 256 rows at a time"""
    out = []
    for r in range(0, x.shape[0], 256):
        z = x[r:r + 256].double() * inv_temp
        out.append(z.gather(1, targets[r:r + 256].long().clamp(min=0).unsqueeze(1)).squeeze(1) - torch.logsumexp(z, 1))
    return torch.cat(out)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    st = {"case": case}
    if op in ("logprob", "logprob_grad", "policy"):
        M, N = case["rows"], case["vocab"]
        st["buf"], st["targets"] = _policy_inputs(case, g)
        st["inv_temp"] = _f32(1.0 / case["temp"])
        st["ld"] = N + case["pad"]
        st["logp"] = torch.empty(M, device="cuda")
        st["entropy"] = torch.empty(M, device="cuda") if case["entropy"] else None
    if op == "logprob":
        st["stats"] = torch.empty(M, 2, device="cuda")
    if op == "logprob_grad":
        # what the forward of the same step left
        x = st["buf"][:, :N]
        st["stats"], st["entropy"] = _saved(x, st["targets"], st["inv_temp"], case["entropy"])
        st["dlogp"] = torch.randn(M, device="cuda", generator=g) / M
        st["dentropy"] = torch.randn(M, device="cuda", generator=g) * (0.01 / M) if case["entropy"] else None
        # another loss's gradient is there already, and the operator adds to it
        st["dlogits"] = torch.randn(M, N, device="cuda", generator=g) / (M * 50.0) if case["accumulate"] else torch.empty(M, N, device="cuda")
    if op == "policy":
        x = st["buf"][:, :N]
        logp = _rows_logp(x, st["targets"], st["inv_temp"])
        ratio = _off_border(torch.exp(0.2 * torch.randn(M, device="cuda", generator=g, dtype=torch.float64)))
        st["old"] = (logp - torch.log(ratio)).float()
        st["ref"] = (logp + 0.3 * torch.randn(M, device="cuda", generator=g, dtype=torch.float64)).float() if case["kl"] else None
        st["advantages"] = torch.randn(M, device="cuda", generator=g)
        # mean over the sequences of each sequence's mean: rows of a long sequence weigh less
        st["weights"] = torch.rand(M, device="cuda", generator=g) * (2.0 / M) if case["weighted"] else None
        st["loss"] = torch.empty(2, device="cuda")
        st["token_loss"] = torch.empty(M, device="cuda")
        st["dlogits"] = torch.empty(M, N, device="cuda")
    if op == "preference":
        # answers of very different lengths, some empty, one after the other; a few rows at the end belong to none
        P, M = case["pairs"], case["rows"]
        cuts = torch.randint(0, M - M // 50 + 1, (2 * P,), device="cuda", generator=g).sort().values
        st["offsets"] = torch.cat([cuts.new_zeros(1), cuts]).to(torch.int32)
        st["logp_in"] = -2.0 * torch.rand(M, device="cuda", generator=g) - 0.01
        st["ref"] = st["logp_in"] + 0.2 * torch.randn(M, device="cuda", generator=g) if case["reference"] else None
        keep = torch.rand(M, device="cuda", generator=g) >= case["left_out"]
        st["targets"] = torch.where(keep, 7, -1).to(torch.int32)
        st["sequence"] = torch.searchsorted(cuts, torch.arange(M, device="cuda"), right=True)
        st["margin"] = 0.0 if case["reference"] else 0.02
        st["loss"] = torch.empty(1, device="cuda")
        st["pair_loss"] = torch.empty(P, device="cuda")
        st["rewards"] = torch.empty(2 * P, device="cuda")
        st["dlogp"] = torch.zeros(M, device="cuda")
    if op == "grad_norm":
        sizes = _shapes(case)
        flat = torch.randn(sum(sizes) + 4 * len(sizes), device="cuda", generator=g) * 1e-2
        st["grads"] = list(flat.split([s + 4 for s in sizes]))
        st["grads"] = [t[:s] for t, s in zip(st["grads"], sizes)]  # tensors one after the other, at any alignment
        st["max_norm"] = 1.0
        st["result"] = torch.empty(4096, device="cuda")
    if op == "clip_adam":
        n = case["count"]
        st["g"] = torch.randn(n, device="cuda", generator=g) * 1e-3
        st["w"] = torch.randn(n, device="cuda", generator=g) * 0.05
        st["m"] = torch.randn(n, device="cuda", generator=g) * 1e-4
        st["v"] = torch.rand(n, device="cuda", generator=g) * 1e-6
        st["max_norm"] = _f32(0.3 * 1e-3 * math.sqrt(n) if case["clipped"] else 3.0 * 1e-3 * math.sqrt(n) + 1e-2)
        st["result"] = torch.empty(4096, device="cuda")
    if own:
        import ctypes

        from znn_b200 import ops
        from znn_b200._lib import lib
        ops.init(torch.cuda.current_device())
        st["lib"] = lib()
        # the shim launches where torch's work is: the handle 1 names the legacy default stream
        st["lib"].call("znn_set_stream", torch.cuda.current_stream().cuda_stream or 1)
        if op == "grad_norm":
            st["pointers"] = (ctypes.c_void_p * len(st["grads"]))(*[t.data_ptr() for t in st["grads"]])
            st["counts"] = (ctypes.c_size_t * len(st["grads"]))(*[t.numel() for t in st["grads"]])
        if op == "clip_adam":
            st["pointers"] = (ctypes.c_void_p * 1)(st["g"].data_ptr())
            st["counts"] = (ctypes.c_size_t * 1)(case["count"])
    return st


def _saved(x, targets, inv_temp, entropy):
    """The forward's row statistics and entropies, 256 rows at a time in 64 bits"""
    tops, sums, ents = [], [], []
    for r in range(0, x.shape[0], 256):
        z = x[r:r + 256].double()
        top = z.amax(1, keepdim=True)
        d = (z - top) * inv_temp
        e = torch.exp(d)
        s = e.sum(1)
        tops.append(top.squeeze(1))
        sums.append(s)
        ents.append(torch.log(s) - torch.where(e > 0, d * e, 0.0).sum(1) / s)
    left = targets < 0
    stats = torch.stack([torch.cat(tops), torch.cat(sums)], 1).masked_fill(left.unsqueeze(1), 0.0).float().contiguous()
    return stats, torch.cat(ents).masked_fill(left, 0.0).float() if entropy else None


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _at(t):
    return None if t is None else t.data_ptr()


def _run_own(st):
    case, L = st["case"], st["lib"]
    op = case["op"]
    if op == "logprob":
        L.call("znn_token_logprob_fwd", _at(st["buf"]), st["ld"], _at(st["targets"]), st["inv_temp"], _at(st["logp"]), _at(st["entropy"]),
               _at(st["stats"]), case["rows"], case["vocab"])
        return {"logp": st["logp"], "entropy": st["entropy"], "stats": st["stats"]}
    if op == "logprob_grad":
        L.call("znn_token_logprob_bwd", _at(st["buf"]), st["ld"], _at(st["targets"]), st["inv_temp"], _at(st["stats"]), _at(st["entropy"]),
               _at(st["dlogp"]), _at(st["dentropy"]), _at(st["dlogits"]), case["vocab"], int(case["accumulate"]), case["rows"], case["vocab"])
        return {"dlogits": st["dlogits"]}
    if op == "policy":
        L.call("znn_policy_loss", _at(st["buf"]), st["ld"], _at(st["targets"]), st["inv_temp"], _at(st["old"]), _at(st["ref"]),
               _at(st["advantages"]), _at(st["weights"]), CLIP_LOW, CLIP_HIGH, KL_COEF if case["kl"] else 0.0,
               ENTROPY_COEF if case["entropy"] else 0.0, _at(st["loss"]), _at(st["token_loss"]), _at(st["logp"]), _at(st["entropy"]),
               _at(st["dlogits"]), case["vocab"], case["rows"], case["vocab"])
        return {"loss": st["loss"], "token_loss": st["token_loss"], "logp": st["logp"], "entropy": st["entropy"], "dlogits": st["dlogits"]}
    if op == "preference":
        L.call("znn_preference_loss", _at(st["logp_in"]), _at(st["ref"]), _at(st["targets"]), _at(st["offsets"]), BETA, SMOOTHING, st["margin"],
               int(case["by_length"]), _at(st["loss"]), _at(st["pair_loss"]), _at(st["rewards"]), _at(st["dlogp"]), case["pairs"], case["rows"])
        return {"loss": st["loss"], "pair_loss": st["pair_loss"], "rewards": st["rewards"], "dlogp": st["dlogp"]}
    if op == "grad_norm":
        L.call("znn_grad_norm", st["pointers"], st["counts"], len(st["grads"]), 1.0, st["max_norm"], _at(st["result"]))
        return {"norm": st["result"][:2]}
    L.call("znn_grad_norm", st["pointers"], st["counts"], 1, 1.0, st["max_norm"], _at(st["result"]))
    L.call("znn_adam_step_clipped", _at(st["w"]), _at(st["g"]), _at(st["m"]), _at(st["v"]), LR, BETA1, BETA2, EPS, STEP, 1.0, _at(st["result"]),
           case["count"])
    return {"norm": st["result"][:2], "w": st["w"], "m": st["m"], "v": st["v"]}


# ---- the plain forms -----------------------------------------------------------------------------------------------
def _plain_rows(x, targets, inv_temp):
    """row maximum, scaled distances from it, their exponentials, their sum, the taken token's log-probability"""
    top = x.amax(1, keepdim=True)
    d = (x - top) * inv_temp
    e = torch.exp(d)
    s = e.sum(1, dtype=torch.float64)
    taken = targets.long().clamp(min=0).unsqueeze(1)
    logp = d.gather(1, taken).squeeze(1).double() - torch.log(s)
    return top.squeeze(1), d, e, s, taken, logp


def _plain_entropy(d, e, s):
    return torch.log(s) - torch.where(e > 0, d * e, 0.0).sum(1, dtype=torch.float64) / s


def _plain_grad(d, e, s, taken, entropy, g, h, inv_temp):
    """inv_temp * (g * (onehot - p) - h * p * (log p + entropy)), rows of g and h in 64 bits"""
    p = e / s.unsqueeze(1).float()
    grad = -g.unsqueeze(1).float() * p
    if h is not None:
        log_p = d - torch.log(s).unsqueeze(1).float()
        grad = grad - h.unsqueeze(1).float() * torch.where(p > 0, p * (log_p + entropy.unsqueeze(1).float()), 0.0)
    grad.scatter_add_(1, taken, g.unsqueeze(1).float())
    return grad * inv_temp


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op in ("logprob", "logprob_grad", "policy"):
        x, inv_temp, targets = st["buf"][:, :case["vocab"]], st["inv_temp"], st["targets"]
        left = targets < 0
    if op == "logprob":
        top, d, e, s, _, logp = _plain_rows(x, targets, inv_temp)
        entropy = _plain_entropy(d, e, s).masked_fill(left, 0.0).float() if case["entropy"] else None
        stats = torch.stack([top, s.float()], 1).masked_fill(left.unsqueeze(1), 0.0)
        return {"logp": logp.masked_fill(left, 0.0).float(), "entropy": entropy, "stats": stats}
    if op == "logprob_grad":
        d = (x - st["stats"][:, :1]) * inv_temp
        e = torch.exp(d)
        taken = targets.long().clamp(min=0).unsqueeze(1)
        grad = _plain_grad(d, e, st["stats"][:, 1].double(), taken, st["entropy"], st["dlogp"], st["dentropy"], inv_temp)
        grad = grad.masked_fill(left.unsqueeze(1), 0.0)
        return {"dlogits": st["dlogits"].add_(grad) if case["accumulate"] else grad}
    if op == "policy":
        _, d, e, s, taken, logp = _plain_rows(x, targets, inv_temp)
        w = torch.where(left, 0.0, st["weights"].double() if case["weighted"] else 1.0 / (~left).sum().double())
        a = st["advantages"].double()
        ratio = torch.exp(logp - st["old"].double())
        bounded = ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH)
        token = -torch.minimum(ratio * a, bounded * a)
        slope = torch.where(ratio * a <= bounded * a, -a * ratio, 0.0)
        if case["kl"]:
            q = st["ref"].double() - logp
            token = token + KL_COEF * (torch.exp(q) - q - 1.0)
            slope = slope + KL_COEF * (1.0 - torch.exp(q))
        entropy, h = None, None
        if case["entropy"]:
            entropy = _plain_entropy(d, e, s)
            token = token - ENTROPY_COEF * entropy
            h = -ENTROPY_COEF * w
        token = torch.where(left, 0.0, token)
        counted = (~left & (w != 0)).sum().double()
        loss = torch.stack([(w * token).sum(), counted])
        grad = _plain_grad(d, e, s, taken, entropy, w * slope, h, inv_temp)
        return {"loss": loss.float(), "token_loss": token.float(), "logp": logp.masked_fill(left, 0.0).float(),
                "entropy": entropy.masked_fill(left, 0.0).float() if case["entropy"] else None, "dlogits": grad}
    if op == "preference":
        P = case["pairs"]
        kept = (st["targets"] >= 0) & (st["sequence"] < 2 * P)
        ratios = torch.where(kept, st["logp_in"].double() - (st["ref"].double() if case["reference"] else 0.0), 0.0)
        zeros = torch.zeros(2 * P + 1, device=ratios.device, dtype=torch.float64)
        sums = zeros.index_add(0, st["sequence"], ratios)[:-1]
        share = torch.full((2 * P,), BETA, device=ratios.device, dtype=torch.float64)
        if case["by_length"]:
            lens = zeros.index_add(0, st["sequence"], kept.double())[:-1]
            share = share / lens.clamp(min=1.0)
        rewards = sums * share
        m = rewards[0::2] - rewards[1::2] - st["margin"]
        pair = (1.0 - SMOOTHING) * torch.log1p(torch.exp(-m.abs())) + SMOOTHING * torch.log1p(torch.exp(-m.abs()))
        pair = pair + (1.0 - SMOOTHING) * (-m).clamp(min=0.0) + SMOOTHING * m.clamp(min=0.0)
        slope = (SMOOTHING - 1.0 + 1.0 / (1.0 + torch.exp(-m))) / P
        slopes = torch.stack([slope, -slope], 1).reshape(-1) * share
        return {"loss": pair.mean().reshape(1).float(), "pair_loss": pair.float(), "rewards": rewards.float(),
                "dlogp": torch.where(kept, slopes[st["sequence"].clamp(max=2 * P - 1)], 0.0).float()}
    grads = st["grads"] if op == "grad_norm" else [st["g"]]
    norm = torch.stack([(t * t).sum(dtype=torch.float64) for t in grads]).sum().sqrt()
    share = torch.where(norm > st["max_norm"], st["max_norm"] / norm, 1.0)
    result = torch.stack([norm, share]).float()
    if op == "grad_norm":
        return {"norm": result}
    g = st["g"] * result[1]
    lr = LR * math.sqrt(1.0 - BETA2 ** STEP) / (1.0 - BETA1 ** STEP)
    st["m"].mul_(BETA1).add_(g * (1.0 - BETA1))
    st["v"].mul_(BETA2).add_(g * g * (1.0 - BETA2))
    st["w"].sub_(st["m"] * lr / (torch.sqrt(st["v"]) + EPS))
    return {"norm": result, "w": st["w"], "m": st["m"], "v": st["v"]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("logprob", "logprob_grad", "policy"):
        M, N, it = case["rows"], case["vocab"], st["inv_temp"]
        targets = st["targets"].long()
        col = torch.arange(N, device="cuda")
        count = float((targets >= 0).sum())
        outs = {"logp": [], "entropy": [], "stats": [], "dlogits": [], "token_loss": []}
        total, counted = 0.0, 0
        for r in range(0, M, 256):
            rows = slice(r, min(r + 256, M))
            z = st["buf"][rows, :N].double() * it
            lse = torch.logsumexp(z, 1, keepdim=True)
            lp = z - lse
            p = lp.exp()
            t = targets[rows]
            in_use = t >= 0
            is_taken = col.unsqueeze(0) == t.unsqueeze(1)
            own_lp = torch.where(is_taken, lp, 0.0).sum(1)
            ent = -torch.special.xlogy(p, p).sum(1)
            raw = st["buf"][rows, :N].double().amax(1)
            outs["stats"].append(torch.where(in_use.unsqueeze(1), torch.stack([raw, torch.exp(lse.squeeze(1) - raw * it)], 1), 0.0))
            outs["logp"].append(torch.where(in_use, own_lp, 0.0))
            outs["entropy"].append(torch.where(in_use, ent, 0.0))
            if op == "logprob":
                continue
            if op == "logprob_grad":
                gp = st["dlogp"][rows].double()
                gh = st["dentropy"][rows].double() if case["entropy"] else torch.zeros_like(gp)
            else:
                a, old = st["advantages"][rows].double(), st["old"][rows].double()
                w = st["weights"][rows].double() if case["weighted"] else torch.full_like(a, 1.0 / count)
                w = torch.where(in_use, w, 0.0)
                rat = torch.exp(own_lp - old)
                hi, lo = 1.0 + CLIP_HIGH, 1.0 - CLIP_LOW
                # a gain counts up to the upper border, a loss down to the lower one
                reach = torch.where(a >= 0, rat.clamp(max=hi), rat.clamp(min=lo))
                val = -a * reach
                gp = torch.where(reach == rat, val, 0.0)
                if case["kl"]:
                    q = st["ref"][rows].double() - own_lp
                    val = val + KL_COEF * (torch.expm1(q) - q)
                    gp = gp - KL_COEF * torch.expm1(q)
                gh = torch.zeros_like(a)
                if case["entropy"]:
                    val = val - ENTROPY_COEF * ent
                    gh = gh - ENTROPY_COEF
                gp, gh = gp * w, gh * w
                val = torch.where(in_use, val, 0.0)
                outs["token_loss"].append(val)
                total += float((w * val).sum())
                counted += int((in_use & (w != 0)).sum())
            inner = torch.where(p > 0, p * (lp + ent.unsqueeze(1)), 0.0)
            dz = gp.unsqueeze(1) * (is_taken.double() - p) - gh.unsqueeze(1) * inner
            dx = torch.where(in_use.unsqueeze(1), dz * it, 0.0)
            if op == "logprob_grad" and case["accumulate"]:
                dx = dx + st["dlogits"][rows].double()
            outs["dlogits"].append(dx)
        cat = {k: torch.cat(v) if v else None for k, v in outs.items()}
        if not case["entropy"]:
            cat["entropy"] = None
        if op == "logprob":
            return {k: cat[k] for k in ("logp", "entropy", "stats")}
        if op == "logprob_grad":
            return {"dlogits": cat["dlogits"]}
        loss = torch.tensor([total, float(counted)], dtype=torch.float64, device="cuda")
        return {"loss": loss, **{k: cat[k] for k in ("token_loss", "logp", "entropy", "dlogits")}}
    if op == "preference":
        kept = (st["targets"] >= 0).cpu()
        diff = st["logp_in"].double().cpu()
        if case["reference"]:
            diff = diff - st["ref"].double().cpu()
        off = st["offsets"].tolist()
        rewards, pairs = [], []
        dlogp = torch.zeros(case["rows"], dtype=torch.float64)
        for p in range(case["pairs"]):
            parts = []
            for k in (2 * p, 2 * p + 1):
                sl = slice(off[k], off[k + 1])
                n = int(kept[sl].sum())
                parts.append((sl, BETA / max(n, 1) if case["by_length"] else BETA, float(diff[sl][kept[sl]].sum())))
            rc, rr = parts[0][1] * parts[0][2], parts[1][1] * parts[1][2]
            m = rc - rr - st["margin"]
            rewards += [rc, rr]
            up, down = 1.0 / (1.0 + math.exp(-m)), 1.0 / (1.0 + math.exp(m))
            pairs.append(-(1.0 - SMOOTHING) * math.log(up) - SMOOTHING * math.log(down))
            slope = ((SMOOTHING - 1.0) * down + SMOOTHING * up) / case["pairs"]
            for (sl, share, _), sign in zip(parts, (1.0, -1.0)):
                dlogp[sl] = torch.where(kept[sl], sign * slope * share, 0.0)
        pairs = torch.tensor(pairs, dtype=torch.float64)
        return {"loss": pairs.mean().reshape(1), "pair_loss": pairs, "rewards": torch.tensor(rewards, dtype=torch.float64), "dlogp": dlogp}
    grads = st["grads"] if op == "grad_norm" else [st["g"]]
    square = 0.0
    for t in grads:
        square += float(t.double().square().sum())
    norm = math.sqrt(square)
    share = st["max_norm"] / norm if norm > st["max_norm"] else 1.0
    result = torch.tensor([norm, share], dtype=torch.float64)
    if op == "grad_norm":
        return {"norm": result}
    b1, b2, eps, lr = BETA1, BETA2, EPS, LR
    g = st["g"].double() * share
    m = b1 * st["m"].double() + (1.0 - b1) * g
    v = b2 * st["v"].double() + (1.0 - b2) * g * g
    step = lr * math.sqrt(1.0 - b2 ** STEP) / (1.0 - b1 ** STEP)
    return {"norm": result, "w": st["w"].double() - step * m / (v.sqrt() + eps), "m": m, "v": v}


def work(case):
    """Each input read once, each output written once; operations as the formulas count them."""
    op = case["op"]
    if op in ("logprob", "logprob_grad", "policy"):
        M, N = case["rows"], case["vocab"]
        used = M * (1.0 - case["left_out"])
        cells = used * N
        if op == "logprob":
            return {"bytes": 4 * cells + 4 * M * (4 + case["entropy"]), "flops": (5 + 2 * case["entropy"]) * cells}
        if op == "logprob_grad":
            written = 8 * cells if case["accumulate"] else 4.0 * M * N
            return {"bytes": 4 * cells + written + 4 * M * 6, "flops": (6 + 4 * case["entropy"]) * cells}
        return {"bytes": 4 * cells + 4.0 * M * N + 4 * M * 8, "flops": (9 + 6 * case["entropy"]) * cells}
    if op == "preference":
        M = case["rows"]
        return {"bytes": M * (12 + 4 * case["reference"]) + 32 * case["pairs"], "flops": 4 * M}
    if op == "grad_norm":
        n = sum(_shapes(case))
        return {"bytes": 4 * n, "flops": 2 * n}
    n = case["count"]
    return {"bytes": 28 * n, "flops": 16 * n}
