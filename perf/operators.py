"""Workloads of the training-loss and optimizer operators.

Four groups: the log-probabilities of chosen classes, the clipped policy loss with its gradient, the paired
preference loss with its gradient, and the AdamW step over many tensors (states in 32 or in 8 bits).  `run` computes
them in elementary torch operations, or, where `own` is set, with the entry points of `renaissance_b200.ops`; `exact`
gives the same outputs from the definitions in 64 bits.
"""
import math
import random
from functools import reduce

import torch

own = False

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04
BETA, SMOOTHING = 0.1, 0.05
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.05
SEED = 1234567
BLOCK = 128                 # elements that share one scale of an 8-bit state
E4M3_MAX, E4M3_MIN_NORMAL = 448.0, 2.0 ** -6
SMALLEST = 2.0 ** -116      # a block whose largest state is below this is stored as zeros


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one batch of the 1000-class head that the networks here end in: latency counts
        {"name": "logp 48x1000", "op": "logp", "rows": 48, "classes": 1000, "dtype": "float16", "pad": 0,
         "masked": 0.1, "banned": 0},
        # the reference policy's pass over a rollout, an odd number of classes, rows that start anywhere
        {"name": "logp 6000x50021", "op": "logp", "rows": 6000, "classes": 50021, "dtype": "bfloat16", "pad": 0,
         "masked": 0.2, "banned": 0},
        # a small discrete action space
        {"name": "policy 64x1000", "op": "policy", "rows": 64, "classes": 1000, "dtype": "float16", "pad": 24,
         "masked": 0.0, "banned": 0, "kl": False},
        # an ordinary minibatch, a quarter of it padding, with the penalty against a reference policy
        {"name": "policy 4096x32000", "op": "policy", "rows": 4096, "classes": 32000, "dtype": "bfloat16", "pad": 0,
         "masked": 0.25, "banned": 0, "kl": True},
        # the largest: a big class table whose last columns are padding (minus infinity)
        {"name": "policy 8192x131072", "op": "policy", "rows": 8192, "classes": 131072, "dtype": "bfloat16", "pad": 0,
         "masked": 0.1, "banned": 77, "kl": True},
        # four short pairs
        {"name": "preference 4 pairs x1000", "op": "preference", "pairs": 4, "longest": 16, "prompt": 4,
         "classes": 1000, "dtype": "float16", "pad": 0, "behind": 3},
        # an ordinary minibatch: ragged answers behind prompts that do not count
        {"name": "preference 16 pairs x32000", "op": "preference", "pairs": 16, "longest": 256, "prompt": 32,
         "classes": 32000, "dtype": "bfloat16", "pad": 0, "behind": 100},
        # long answers over a big class table
        {"name": "preference 4 pairs x131072", "op": "preference", "pairs": 4, "longest": 1024, "prompt": 100,
         "classes": 131072, "dtype": "bfloat16", "pad": 0, "behind": 0},
        # a small perceptron: six tensors, latency counts
        {"name": "adamw32 mlp", "op": "adamw", "bits": 32, "params": "mlp", "grad": "float32", "copy": "none",
         "step": 10},
        # the parameters of VGG16-BN with float gradients and a half working copy
        {"name": "adamw32 vgg16bn", "op": "adamw", "bits": 32, "params": "vgg16bn", "grad": "float32",
         "copy": "float16", "step": 1000},
        # the parameters of ResNet-50 with bfloat16 gradients and working copy: 161 tensors, many of them tiny
        {"name": "adamw8 resnet50", "op": "adamw", "bits": 8, "params": "resnet50", "grad": "bfloat16",
         "copy": "bfloat16", "step": 0},
        # VGG16-BN again, states in 8 bits
        {"name": "adamw8 vgg16bn", "op": "adamw", "bits": 8, "params": "vgg16bn", "grad": "float32",
         "copy": "float16", "step": 1000},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["logp", "policy", "policy", "preference", "preference", "adamw", "adamw"])
    if op == "adamw":
        return {"op": op, "bits": rng.choice([32, 8]), "params": "drawn", "count": _log_int(rng, 1, 160),
                "total": _log_int(rng, 1000, 100_000_000), "sizes": rng.randrange(1 << 30),
                "grad": rng.choice(["float32", "float16", "bfloat16"]),
                "copy": rng.choice(["none", "float16", "bfloat16"]), "step": _log_int(rng, 1, 100_000)}
    dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
    most = (1 << 27) if dtype == "float32" else (1 << 28)
    classes = _log_int(rng, 8, 131072)
    if rng.random() < 0.5:
        classes = max(8, classes // 64 * 64)
    pad = rng.choice([0, 0, 1, 8, 40])
    if op == "preference":
        pairs = _log_int(rng, 1, 64)
        longest = _log_int(rng, 2, 1024)
        longest = max(2, min(longest, most // (2 * pairs * classes)))
        return {"op": op, "pairs": pairs, "longest": longest, "prompt": rng.randrange(0, max(1, longest // 2)),
                "classes": classes, "dtype": dtype, "pad": pad, "behind": rng.choice([0, 0, 1, 7])}
    rows = max(1, min(_log_int(rng, 1, 8192), most // classes))
    case = {"op": op, "rows": rows, "classes": classes, "dtype": dtype, "pad": pad,
            "masked": round(rng.choice([0.0, rng.uniform(0, 0.5)]), 3),
            "banned": rng.choice([0, rng.randrange(0, max(1, classes // 16))])}
    if op == "policy":
        case["kl"] = rng.random() < 0.5
    return case


# ------------------------------------------------------------------------------------------------ parameter lists

def _sizes(case):
    """(elements, decayed) of each parameter tensor; vectors (normalisation, biases) take no weight decay."""
    if case["params"] == "mlp":
        dims = [784, 512, 256, 10]
        return [x for i in range(3) for x in ((dims[i] * dims[i + 1], True), (dims[i + 1], False))]
    if case["params"] == "vgg16bn":
        out, c = [], 4
        for k in (64, 64, 128, 128, 256, 256, 256, 512, 512, 512, 512, 512, 512):
            out += [(k * 9 * c, True), (k, False), (k, False)]
            c = k
        for i, o in ((25088, 4096), (4096, 4096), (4096, 1000)):
            out += [(i * o, True), (o, False)]
        return out
    if case["params"] == "resnet50":
        out, c = [(64 * 49 * 4, True), (64, False), (64, False)], 64
        for mid, blocks in ((64, 3), (128, 4), (256, 6), (512, 3)):
            for b in range(blocks):
                for n, k in ((c * mid, mid), (mid * 9 * mid, mid), (mid * mid * 4, mid * 4)):
                    out += [(n, True), (k, False), (k, False)]
                if b == 0:
                    out += [(c * mid * 4, True), (mid * 4, False), (mid * 4, False)]
                c = mid * 4
        return out + [(2048 * 1000, True), (1000, False)]
    rng = random.Random(case["sizes"])
    parts = [rng.expovariate(1.0) ** 2 + 1e-3 for _ in range(case["count"])]
    scale = case["total"] / sum(parts)
    return [(max(1, int(p * scale)), rng.random() < 0.7) for p in parts]


def _offsets(sizes):
    """Every tensor starts at a whole block of the flat buffers, as the trainers lay their slots out."""
    offs, at = [], 0
    for n, _ in sizes:
        offs.append(at)
        at += -(-n // BLOCK) * BLOCK
    return offs, at


# ------------------------------------------------------------------------------------------------ inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _logits(rows, classes, pad, dtype, gen):
    full = torch.randn((rows, classes + pad), generator=gen, device="cuda", dtype=DTYPES[dtype])
    full.mul_(2.5)
    return full[:, :classes]


def _logp_of(logits, labels):
    """Log-probabilities of the labels in double, a band of rows at a time."""
    rows, classes = logits.shape
    band = max(1, (1 << 26) // classes)
    out = []
    for r in range(0, rows, band):
        z = logits[r:r + band].double()
        at = labels[r:r + band].long().clamp(0, classes - 1)
        out.append(z.gather(1, at[:, None])[:, 0] - torch.logsumexp(z, 1))
    return torch.cat(out)


def _labels(logits, gen):
    """A class for each row, of above-average probability as a sampled one is: the best of sixteen picks."""
    rows, classes = logits.shape
    picks = torch.randint(0, classes, (rows, 16), generator=gen, device="cuda")
    best = logits.gather(1, picks).float().argmax(1)
    return picks[torch.arange(rows, device="cuda"), best].int()


def _noise_off_the_borders(rows, gen):
    """How far the policy has moved from the one that acted, in log-probability.  No row lies within 1e-3 of a border
    of the clipping interval, where the gradient jumps."""
    d = torch.randn(rows, generator=gen, device="cuda", dtype=torch.float64) * 0.2
    for border in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
        d = torch.where((d - border).abs() < 1e-3, torch.full_like(d, border + 2e-3), d)
    return d


def prepare(case, seed):
    gen = _generator(seed)
    op = case["op"]
    if op == "adamw":
        return _prepare_adamw(case, gen)
    if op == "preference":
        return _prepare_preference(case, gen)
    rows, classes = case["rows"], case["classes"]
    logits = _logits(rows, classes, case["pad"], case["dtype"], gen)
    labels = _labels(logits[:, :classes - case["banned"]], gen)
    if case["banned"]:
        logits[:, classes - case["banned"]:] = -math.inf
    off = torch.rand(rows, generator=gen, device="cuda") < case["masked"]
    off[0] = False
    if op == "logp":
        labels[off] = -1
        return {"op": op, "logits": logits, "labels": labels}
    logp = _logp_of(logits, labels)
    keep = (~off).float()
    s = {"op": op, "logits": logits, "actions": labels,
         "old_logp": (logp - _noise_off_the_borders(rows, gen)).float(),
         "advantages": torch.randn(rows, generator=gen, device="cuda"),
         "weights": keep / keep.sum(),
         "scaling": torch.full((1,), 65536.0, device="cuda"),
         "ref_logp": None, "kl_coef": 0.0}
    if case["kl"]:
        s["ref_logp"] = (logp + 0.3 * torch.randn(rows, generator=gen, device="cuda", dtype=torch.float64)).float()
        s["kl_coef"] = KL_COEF
    return s


def _lengths(case):
    """Rows of each sequence; the shapes go by the case, not by the seed."""
    rng = random.Random(case["pairs"] * 7919 + case["longest"])
    return [rng.randint(max(1, case["longest"] // 2), case["longest"]) for _ in range(2 * case["pairs"])]


def _prepare_preference(case, gen):
    lens = _lengths(case)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    rows = starts[-1] + case["behind"]
    logits = _logits(rows, case["classes"], case["pad"], case["dtype"], gen)
    labels = _labels(logits, gen)
    logp = _logp_of(logits, labels)
    ref = []
    for s, (a, n) in enumerate(zip(starts, lens)):
        quiet = min(case["prompt"], n - 1)          # prompt rows carry no label that counts
        labels[a:a + quiet] = -1
        ref.append(logp[a + quiet:a + n].sum())
    ref = torch.stack(ref)
    ref = ref + 5.0 * torch.randn(ref.shape, generator=gen, device="cuda", dtype=torch.float64)
    return {"op": "preference", "logits": logits, "labels": labels,
            "seq_starts": torch.tensor(starts, dtype=torch.int32, device="cuda"), "ref_logp": ref.float(),
            "scaling": torch.full((1,), 65536.0, device="cuda")}


def _prepare_adamw(case, gen):
    sizes = _sizes(case)
    offs, total = _offsets(sizes)
    live = torch.zeros(total, dtype=torch.bool, device="cuda")
    blocks = total // BLOCK
    tensor_of = torch.empty(blocks, dtype=torch.int64, device="cuda")
    block_of = torch.empty(blocks, dtype=torch.int64, device="cuda")
    decay = torch.empty(blocks, dtype=torch.float32, device="cuda")
    for i, ((n, decayed), o) in enumerate(zip(sizes, offs)):
        live[o:o + n] = True
        b0, b1 = o // BLOCK, (o + n + BLOCK - 1) // BLOCK
        tensor_of[b0:b1] = i
        block_of[b0:b1] = torch.arange(b1 - b0, device="cuda")
        decay[b0:b1] = DECAY if decayed else 0.0
    randn = lambda: torch.randn(total, generator=gen, device="cuda")
    # gradients of one block differ by a good order of magnitude; the loss scale is still on them
    spread = torch.exp(randn())
    grad = (randn() * spread * 0.05).mul_(live).to(DTYPES[case["grad"]])
    s = {"op": "adamw", "bits": case["bits"], "w": (randn() * 0.05).mul_(live), "g": grad,
         "scaling": torch.full((1,), 64.0, device="cuda"), "skip": torch.zeros(1, dtype=torch.int32, device="cuda"),
         "step": torch.full((1,), case["step"], dtype=torch.int32, device="cuda"),
         "tensor_of": tensor_of, "block_of": block_of, "decay": decay,
         "copy": None if case["copy"] == "none" else torch.zeros(total, dtype=DTYPES[case["copy"]], device="cuda")}
    started = 1.0 if case["step"] else 0.0
    m = (randn() * spread * 3e-4 * started).mul_(live)
    v = (spread * 8e-4 * (1.0 + 0.1 * randn())).square_().mul_(live * started)
    del spread
    if case["bits"] == 32:
        s["m"], s["v"] = m, v
    else:
        s["m"], s["m_scale"] = _pack_nearest(m)
        s["v"], s["v_scale"] = _pack_nearest(v)
    if own:         # the plan that a program builds once over its tensors and keeps
        from renaissance_b200 import ops
        cut = lambda t: [t[o:o + n] for (n, _), o in zip(sizes, offs)]
        scales = lambda t: [t[o // BLOCK:(o + n + BLOCK - 1) // BLOCK] for (n, _), o in zip(sizes, offs)]
        more = {} if case["bits"] == 32 else {"m_scales": scales(s["m_scale"]), "v_scales": scales(s["v_scale"])}
        s["plan"] = ops.AdamWPlan(cut(s["w"]), cut(grad), cut(s["m"]), cut(s["v"]),
                                  copies=None if s["copy"] is None else cut(s["copy"]),
                                  weight_decay=[DECAY if d else 0.0 for _, d in sizes], **more)
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _plain_logp(logits, labels):
    """exp(z - max) and its row sums, the log-probability of the labels and which rows have one."""
    classes = logits.shape[1]
    valid = (labels >= 0) & (labels < classes)
    at = labels.long().clamp(0, classes - 1)[:, None]
    z = logits.float()
    top = z.amax(1, keepdim=True)
    z = z - top
    chosen = z.gather(1, at)[:, 0]
    e = z.exp_()
    total = e.sum(1)
    log_total = total.log()
    return e, total, chosen - log_total, log_total + top[:, 0], valid, at


def _plain_dlogits(e, total, coef, at, dtype):
    """coef * (onehot - p) for every row, rounded once."""
    e.mul_((-coef / total)[:, None])
    e.scatter_add_(1, at, coef[:, None])
    return e.masked_fill_((coef == 0)[:, None], 0.0).to(dtype)


def _run_logp(s):
    if own:
        from renaissance_b200 import ops
        r = ops.token_logprobs(s["logits"], s["labels"])
        return {"logp": r["logp"], "lse": r["lse"]}
    _, _, logp, lse, valid, _ = _plain_logp(s["logits"], s["labels"])
    zero = torch.zeros_like(logp)
    return {"logp": torch.where(valid, logp, zero), "lse": torch.where(valid, lse, zero)}


def _run_policy(s):
    if own:
        from renaissance_b200 import ops
        r = ops.policy_loss_fused(s["logits"], s["actions"], s["old_logp"], s["advantages"], s["scaling"],
                                  clip_low=CLIP_LOW, clip_high=CLIP_HIGH, ref_logp=s["ref_logp"],
                                  kl_coef=s["kl_coef"], weights=s["weights"])
        return {"loss": r["loss"], "loss_partial": r["loss_partial"], "logp": r["logp"], "dlogits": r["dlogits"]}
    e, total, logp, _, valid, at = _plain_logp(s["logits"], s["actions"])
    valid = valid & (s["weights"] != 0)
    zero = torch.zeros_like(logp)
    w = torch.where(valid, s["weights"], zero)
    adv = s["advantages"]
    ratio = (logp - s["old_logp"]).exp()
    kept = ratio * adv
    cut = ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv
    loss = -torch.minimum(kept, cut)
    slope = torch.where(kept <= cut, -kept, zero)
    if s["ref_logp"] is not None:
        gap = s["ref_logp"] - logp
        odds = gap.exp()
        loss = loss + s["kl_coef"] * (odds - gap - 1.0)
        slope = slope + s["kl_coef"] * (1.0 - odds)
    part = torch.where(valid, loss * w, zero)
    coef = torch.where(valid, slope * w, zero) * s["scaling"]
    return {"loss": part.sum().reshape(1), "loss_partial": part, "logp": torch.where(valid, logp, zero),
            "dlogits": _plain_dlogits(e, total, coef, at, s["logits"].dtype)}


def _run_preference(s):
    if own:
        from renaissance_b200 import ops
        r = ops.preference_loss_fused(s["logits"], s["labels"], s["seq_starts"], s["ref_logp"], s["scaling"],
                                      beta=BETA, label_smoothing=SMOOTHING)
        return {"loss": r["loss"], "loss_partial": r["loss_partial"], "seq_logp": r["seq_logp"], "logp": r["logp"],
                "dlogits": r["dlogits"]}
    e, total, logp, _, valid, at = _plain_logp(s["logits"], s["labels"])
    rows = logp.numel()
    starts = s["seq_starts"].long()
    seqs = starts.numel() - 1
    seq = torch.searchsorted(starts[1:], torch.arange(rows, device=logp.device), right=True)
    valid = valid & (seq < seqs)
    logp = torch.where(valid, logp, torch.zeros_like(logp))
    run_up = torch.cat([torch.zeros(1, dtype=torch.float64, device=logp.device), logp.double().cumsum(0)])
    seq_logp = run_up[starts[1:]] - run_up[starts[:-1]]
    margin = (seq_logp - s["ref_logp"].double()).view(-1, 2)
    x = BETA * (margin[:, 0] - margin[:, 1])
    soft = torch.log1p(torch.exp(-x.abs()))
    pairs = x.numel()
    # -log sigmoid(x) = max(-x, 0) + log(1 + exp(-|x|))
    part = ((1 - SMOOTHING) * ((-x).clamp_min(0) + soft) + SMOOTHING * (x.clamp_min(0) + soft)) / pairs
    pull = BETA * (SMOOTHING / (1 + torch.exp(-x)) - (1 - SMOOTHING) / (1 + torch.exp(x))) / pairs
    coef = torch.stack([pull, -pull], 1).reshape(-1) * s["scaling"].double()
    coef = torch.where(valid, coef[seq.clamp_max(seqs - 1)], torch.zeros_like(run_up[1:])).float()
    return {"loss": part.sum().float().reshape(1), "loss_partial": part.float(), "seq_logp": seq_logp.float(),
            "logp": logp, "dlogits": _plain_dlogits(e, total, coef, at, s["logits"].dtype)}


def _philox_round(x, k0, k1):
    low = 0xFFFFFFFF
    a, b, c, d = x
    # the high half of a 32 x 32 bit product from two products that fit 64 bits; the low half survives the wrap
    high = lambda v, f: ((((v >> 16) * f) + (((v & 0xFFFF) * f) >> 16)) >> 16) & low
    return (high(c, 0xCD9E8D57) ^ b ^ (k0 & low), (c * 0xCD9E8D57) & low,
            high(a, 0xD2511F53) ^ d ^ (k1 & low), (a * 0xD2511F53) & low)


def _philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32-10 on int64 tensors that hold 32-bit words."""
    return reduce(lambda x, i: _philox_round(x, k0 + i * 0x9E3779B9, k1 + i * 0xBB67AE85), range(10), (c0, c1, c2, c3))


def _random16(tensor_of, block_of, step):
    """16 random bits for every element.  A counter serves eight elements: four at 4 * lane of an even block of its
    tensor (the low halves, then the high halves of the words) and four at the same place of the block behind it."""
    lane = torch.arange(32, device=block_of.device)
    group = ((block_of >> 1)[:, None] * 32 + lane).reshape(-1)
    zero = torch.zeros_like(group)
    x = _philox(group & 0xFFFFFFFF, zero + tensor_of[:, None].expand(-1, 32).reshape(-1), zero + step.long(),
                group >> 32, SEED & 0xFFFFFFFF, SEED >> 32)
    words = torch.stack(x, 1)                                               # [blocks * 32, 4]
    odd = (block_of & 1).bool()[:, None].expand(-1, 32).reshape(-1)[:, None]
    return torch.where(odd, words >> 16, words & 0xFFFF).view(-1, BLOCK)


def _scale_of(x):
    top = x.abs().amax(1, keepdim=True)
    small = top < SMALLEST
    return torch.where(small, torch.zeros_like(top), top * (1.0 / E4M3_MAX)), \
        torch.where(small, torch.zeros_like(top), top.reciprocal() * E4M3_MAX)


def _pack_nearest(x):
    x = x.view(-1, BLOCK)
    scale, up = _scale_of(x)
    return (x * up).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _pack_stochastic(x, bits):
    """e4m3 codes of non-negative values: rounded up with the probability of what is cut off, and never to zero."""
    scale, up = _scale_of(x)
    y = (x * up).clamp_max(E4M3_MAX)
    normal = y >= E4M3_MIN_NORMAL
    raw = torch.where(normal, y, y + E4M3_MIN_NORMAL).view(torch.int32)     # steps of 2^20 in either range
    code = ((raw + (bits << 4).int()) >> 20) - torch.where(normal, 960, 968)
    code = torch.maximum(code, (y > 0).int())
    return code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _run_adamw(s):
    out = ["w", "m", "v"] + (["m_scale", "v_scale"] if s["bits"] == 8 else []) + (["copy"] if s["copy"] is not None else [])
    if own:
        from renaissance_b200 import ops
        ops.adamw_step(s["plan"], s["step"], lr=LR, beta1=BETA1, beta2=BETA2, eps=EPS, scaling=s["scaling"],
                       skip_flag=s["skip"], seed=SEED)
        return {**{k: s[k] for k in out}, "step": s["step"]}
    live = s["skip"] == 0                                                   # a step with a raised flag changes nothing
    t = (s["step"] + 1).double()
    unbias1, unbias2 = 1 - BETA1 ** t, 1 - BETA2 ** t
    rate = (LR / unbias1).float()
    widen = unbias2.rsqrt().float()
    g = s["g"].float() * s["scaling"].reciprocal()
    if s["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (s["v"].float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    w = (s["w"].view(-1, BLOCK) * (1.0 - LR * s["decay"])[:, None]).view(-1) - rate * m / (v.sqrt() * widen + EPS)
    s["w"].copy_(torch.where(live, w, s["w"]))
    if s["copy"] is not None:
        s["copy"].copy_(torch.where(live, w.to(s["copy"].dtype), s["copy"]))
    if s["bits"] == 32:
        s["m"].copy_(torch.where(live, m, s["m"]))
        s["v"].copy_(torch.where(live, v, s["v"]))
    else:
        m, m_scale = _pack_nearest(m)
        v, v_scale = _pack_stochastic(v.view(-1, BLOCK), _random16(s["tensor_of"], s["block_of"], s["step"]))
        byte = lambda x: x.view(torch.uint8)
        byte(s["m"]).copy_(torch.where(live, byte(m), byte(s["m"])))
        byte(s["v"]).copy_(torch.where(live, byte(v), byte(s["v"])))
        s["m_scale"].copy_(torch.where(live, m_scale, s["m_scale"]))
        s["v_scale"].copy_(torch.where(live, v_scale, s["v_scale"]))
    s["step"].add_(live.int())
    return {**{k: s[k] for k in out}, "step": s["step"]}


def run(state):
    return {"logp": _run_logp, "policy": _run_policy, "preference": _run_preference,
            "adamw": _run_adamw}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ cost and definition

def work(case):
    """Each input once, each output once.  A masked row's logits are not an input; its gradient is an output."""
    if case["op"] == "adamw":
        n = sum(k for k, _ in _sizes(case))
        grad = DTYPES[case["grad"]].itemsize
        copy = 0 if case["copy"] == "none" else DTYPES[case["copy"]].itemsize
        state = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK
        return {"bytes": n * (8 + grad + copy + state), "flops": 16.0 * n}
    item, classes = DTYPES[case["dtype"]].itemsize, case["classes"]
    if case["op"] == "preference":
        lens = _lengths(case)
        rows = sum(lens) + case["behind"]
        live = sum(n - min(case["prompt"], n - 1) for n in lens)
        return {"bytes": (live + rows) * classes * item + rows * 8 + case["pairs"] * 32, "flops": 6.0 * live * classes}
    live = case["rows"] * (1 - case["masked"])
    if case["op"] == "logp":
        return {"bytes": live * classes * item + case["rows"] * 12, "flops": 4.0 * live * classes}
    return {"bytes": (live + case["rows"]) * classes * item + case["rows"] * 28, "flops": 6.0 * live * classes}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    if case["op"] == "logp":
        rows = _ExactRows(s["logits"], s["labels"])
        return {"logp": rows.logp, "lse": rows.lse}
    if case["op"] == "policy":
        rows = _ExactRows(s["logits"], s["actions"], s["weights"] != 0)
        w, adv = s["weights"].double() * rows.counts, s["advantages"].double()
        ratio = torch.exp(rows.logp - s["old_logp"].double())
        outside = ((adv > 0) & (ratio > 1 + CLIP_HIGH)) | ((adv < 0) & (ratio < 1 - CLIP_LOW))
        bound = torch.where(adv > 0, torch.full_like(adv, 1 + CLIP_HIGH), torch.full_like(adv, 1 - CLIP_LOW))
        part = -torch.where(outside, bound, ratio) * adv
        slope = torch.where(outside, torch.zeros_like(adv), -ratio * adv)
        if s["ref_logp"] is not None:
            gap = s["ref_logp"].double() - rows.logp
            part = part + KL_COEF * (torch.expm1(gap) - gap)
            slope = slope - KL_COEF * torch.expm1(gap)
        part = torch.where(rows.counts, part * w, torch.zeros_like(part))
        return {"loss": part.sum().reshape(1), "loss_partial": part, "logp": rows.logp,
                "dlogits": rows.gradient(torch.where(rows.counts, slope * w, torch.zeros_like(slope)) * 65536.0)}
    starts = s["seq_starts"].tolist()
    inside = torch.zeros(s["labels"].numel(), dtype=torch.bool, device="cuda")
    inside[starts[0]:starts[-1]] = True
    rows = _ExactRows(s["logits"], s["labels"], inside)
    seq_logp = torch.stack([rows.logp[a:b].sum() for a, b in zip(starts, starts[1:])])
    rel = seq_logp - s["ref_logp"].double()
    x = BETA * (rel[0::2] - rel[1::2])
    part = -((1 - SMOOTHING) * torch.nn.functional.logsigmoid(x)
             + SMOOTHING * torch.nn.functional.logsigmoid(-x)) / x.numel()
    pull = BETA * (SMOOTHING * torch.sigmoid(x) - (1 - SMOOTHING) * torch.sigmoid(-x)) / x.numel()
    coef = torch.zeros_like(rows.logp)
    for i, (a, b) in enumerate(zip(starts, starts[1:])):
        coef[a:b] = pull[i // 2] * (1 if i % 2 == 0 else -1)
    return {"loss": part.sum().reshape(1), "loss_partial": part, "seq_logp": seq_logp, "logp": rows.logp,
            "dlogits": rows.gradient(torch.where(rows.counts, coef, torch.zeros_like(coef)) * 65536.0)}


class _ExactRows:
    """log softmax of the chosen classes in double and coef * d logp / d logits, a band of rows at a time."""

    def __init__(self, logits, labels, counts=None):
        self.z, self.labels = logits, labels.long()
        self.counts = (labels >= 0) & (labels < logits.shape[1])
        if counts is not None:
            self.counts = self.counts & counts
        self.band = max(1, (1 << 27) // logits.shape[1])
        lse = torch.cat([torch.logsumexp(z.double(), 1) for z in logits.split(self.band)])
        rows = torch.arange(logits.shape[0], device=logits.device)
        picked = logits[rows, self.labels.clamp(0, logits.shape[1] - 1)].double()
        zero = torch.zeros_like(lse)
        self.raw = lse
        self.lse = torch.where(self.counts, lse, zero)
        self.logp = torch.where(self.counts, picked - lse, zero)

    def gradient(self, coef):
        out = torch.empty(self.z.shape, dtype=torch.float32 if self.z.dtype != torch.float32 else torch.float64,
                          device=self.z.device)
        for r in range(0, self.z.shape[0], self.band):
            z, c = self.z[r:r + self.band], coef[r:r + self.band]
            g = -torch.softmax(z.double(), 1) * c[:, None]
            live = torch.nonzero(c != 0)[:, 0]
            g[live, self.labels[r:r + self.band][live]] += c[live]
            out[r:r + self.band] = g
        return out


def _exact_adamw(case, s):
    sizes = _sizes(case)
    offs, total = _offsets(sizes)
    if total > 200_000_000:
        return None
    t = case["step"] + 1
    lift = lambda x, sc: (x.to(torch.float64).view(-1, BLOCK) * sc.double()[:, None]).view(-1)
    m, v = (s["m"].double(), s["v"].double()) if case["bits"] == 32 else \
        (lift(s["m"], s["m_scale"]), lift(s["v"], s["v_scale"]))
    g = s["g"].double() / 64.0
    m.mul_(BETA1).add_(g, alpha=1 - BETA1)
    v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
    del g
    w = s["w"].double()
    for (n, decayed), o in zip(sizes, offs):
        if decayed:
            w[o:o + n] *= 1 - LR * DECAY
    w -= LR / (1 - BETA1 ** t) * m / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out = {"w": w, "step": torch.tensor([t], dtype=torch.int32)}
    if s["copy"] is not None:
        out["copy"] = w
    if case["bits"] == 32:
        return {**out, "m": m, "v": v}
    bits = _random16(s["tensor_of"], s["block_of"], s["step"]).view(-1, BLOCK)
    for name, x in (("m", m.view(-1, BLOCK)), ("v", v.view(-1, BLOCK))):
        top = x.abs().amax(1, keepdim=True)
        x = torch.where(top < SMALLEST, torch.zeros_like(x), x * E4M3_MAX / top.clamp_min(SMALLEST))
        # the spacing of e4m3 numbers around x: eight to a factor of two, and 2^-9 below 2^-6
        gap = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(E4M3_MIN_NORMAL)))) / 8
        if name == "m":
            q = torch.round(x / gap) * gap
        else:
            q = torch.floor(x / gap + bits.double() / 65536) * gap
            q = torch.where((x > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
        out[name] = q.view(-1)
        out[name + "_scale"] = torch.where(top < SMALLEST, torch.zeros_like(top), top / E4M3_MAX).view(-1)
    return out
