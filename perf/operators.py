"""Cases that measure the operators over distributions of classes (disparity bins or tokens):
log probabilities of given classes with entropy and top alternatives, and distillation from a
teacher's top entries, forward and backward.

Definitions, for a row of V classes x_j and z_j = scale * x_j, lse = log sum_j exp z_j,
p_j = exp(z_j - lse):

log_probs      log_prob = z_t - lse of the given class t (0 where t lies outside [0, V): no class is
               given there); entropy = - sum_j p_j log p_j; the `top` classes of largest z (ties: the
               lowest index first) as log-probabilities and indices.
distill_loss   the teacher lists k classes i_1..i_k with log-probabilities l_1..l_k (an index outside
               [0, V) is padding).  renormalise = False: q = exp l, everything not listed is one further
               class with r = max(0, 1 - sum q) against the student's P = sum of the unlisted p_j;
               loss = sum q (l - log p_i) + r (log r - log P).  renormalise = True: q = softmax of the
               list, r = 0.

Layouts: "rows" (rows, V); "volume" (B, V, H, W); "last" the same volume in torch's channels_last
memory format (the classes of a pixel lie together).
"""
import math

import torch
import torch.nn.functional as F

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# --------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one newly predicted row, scored and listed with its alternatives: latency counts
        dict(name="lp_one_row", op="log_probs", layout="rows", batch=1, classes=32768, height=1, width=1,
             dtype="bf16", scale=1.0, top=20, train=False, holes=0.0, masked=0.0),
        # scoring a ragged batch of predicted rows; odd number of classes, rows not aligned
        dict(name="lp_rows_odd", op="log_probs", layout="rows", batch=1023, classes=50001, height=1, width=1,
             dtype="f16", scale=1.0, top=5, train=False, holes=0.1, masked=0.0),
        # the teacher's pass at the stereo head's own size: 256 bins of a 256 x 512 map, costs (scale -1),
        # eight alternatives a pixel kept, scored where the ground truth has a value
        dict(name="lp_volume_teacher", op="log_probs", layout="volume", batch=1, classes=256, height=256, width=512,
             dtype="f32", scale=-1.0, top=8, train=False, holes=0.7, masked=0.0),
        # training a half-resolution head on sparse ground truth, costs under autocast
        dict(name="lp_volume_train", op="log_probs", layout="volume", batch=12, classes=64, height=96, width=320,
             dtype="bf16", scale=-1.0, top=0, train=True, holes=0.7, masked=0.05),
        # the same head in channels_last, an odd number of bins, a softened distribution
        dict(name="lp_last_train", op="log_probs", layout="last", batch=4, classes=193, height=96, width=320,
             dtype="f16", scale=0.5, top=0, train=True, holes=0.3, masked=0.0),
        # policy-gradient step over long rows: log-probabilities and entropy, both with gradients
        dict(name="lp_rows_train", op="log_probs", layout="rows", batch=4096, classes=32768, height=1, width=1,
             dtype="bf16", scale=1.0, top=0, train=True, holes=0.05, masked=0.0),
        # distilling a small student at an eighth of 192 x 640: a call of a few microseconds
        dict(name="ds_volume_small", op="distill", layout="volume", batch=1, classes=64, height=24, width=80,
             dtype="f32", scale=-1.0, k=4, renormalise=False, train=True, holes=0.0),
        # distilling the full-resolution head under autocast from eight entries a pixel
        dict(name="ds_volume_train", op="distill", layout="volume", batch=4, classes=256, height=192, width=640,
             dtype="bf16", scale=-1.0, k=8, renormalise=False, train=True, holes=0.1),
        # validating a student in channels_last: the loss map alone
        dict(name="ds_last_eval", op="distill", layout="last", batch=12, classes=128, height=96, width=320,
             dtype="f16", scale=1.0, k=8, renormalise=False, train=False, holes=0.2),
        # few rows, long ones, in full precision
        dict(name="ds_few_long_rows", op="distill", layout="rows", batch=5, classes=131072, height=1, width=1,
             dtype="f32", scale=1.0, k=32, renormalise=False, train=True, holes=0.0),
        # odd sizes, the teacher's list renormalised at a temperature of two
        dict(name="ds_rows_odd", op="distill", layout="rows", batch=333, classes=50001, height=1, width=1,
             dtype="f32", scale=0.5, k=20, renormalise=True, train=True, holes=0.05),
        # the largest: a training step over long rows with a long teacher's list
        dict(name="ds_rows_train", op="distill", layout="rows", batch=2048, classes=131072, height=1, width=1,
             dtype="bf16", scale=1.0, k=64, renormalise=False, train=True, holes=0.02),
    ]


def draw(rng):
    def log_uniform(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["log_probs", "distill"])
    layout = rng.choice(["rows", "volume", "last"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.6
    budget = 2048 * 131072 // 8          # elements of logits a drawn case may have
    if layout == "rows":
        classes = log_uniform(1000, 131072)
        batch = log_uniform(1, min(4096, budget // classes))
        height = width = 1
    else:
        classes = rng.randint(48, 256)
        height, width = rng.randint(20, 256), rng.randint(60, 640)
        batch = rng.randint(1, max(1, min(12, budget // (classes * height * width))))
    case = dict(op=op, layout=layout, batch=batch, classes=classes, height=height, width=width, dtype=dtype,
                scale=rng.choice([1.0, 1.0, 0.5] if layout == "rows" else [-1.0, -1.0, 1.0, 0.5]), train=train,
                holes=rng.choice([0.0, 0.1, 0.7]))
    if op == "log_probs":
        # training scores classes; scoring without gradients lists alternatives too
        case["top"] = 0 if train else rng.choice([1, 4, 5, 8, 16, 20])
        case["masked"] = rng.choice([0.0, 0.05])
    else:
        case["k"] = rng.choice([1, 4, 8, 16] if layout != "rows" else [4, 16, 20, 33, 64])
        case["renormalise"] = rng.random() < 0.3
    return case


def _shapes(case):
    """Shape of the logits, of a map without the class axis."""
    if case["layout"] == "rows":
        return (case["batch"], case["classes"]), (case["batch"],)
    return ((case["batch"], case["classes"], case["height"], case["width"]),
            (case["batch"], case["height"], case["width"]))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    shape, rows = _shapes(case)
    dtype = DTYPES[case["dtype"]]
    V = case["classes"]
    sign = 1.0 if case["scale"] > 0 else -1.0
    # z of a spread a trained head has; the stored logits are costs where the scale is negative
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(2.0)
    state = {"case": case}
    if case["op"] == "log_probs":
        # bins that leave the image (or classes that are not allowed) are the last ones of a masked case
        allowed = V - (max(1, int(case["masked"] * V)) if case["masked"] else 0)
        peak = torch.randint(0, allowed, rows, generator=gen, device="cuda")
        x.scatter_add_(1, peak.unsqueeze(1), torch.full_like(peak, 6.0, dtype=torch.float32).unsqueeze(1))
        # the given class is the peak in half of the rows, any class in the others
        other = torch.randint(0, allowed, rows, generator=gen, device="cuda")
        coin = torch.rand(rows, generator=gen, device="cuda")
        index = torch.where(coin < 0.5, peak, other)
        hole = torch.rand(rows, generator=gen, device="cuda") < case["holes"]
        state["index"] = index.masked_fill(hole, -1)
        if allowed < V:
            x[:, allowed:] = torch.finfo(dtype).min   # (the highest cost, where the scale is negative)
        if case["train"]:
            state["g_log_prob"] = torch.rand(rows, generator=gen, device="cuda") - 1.0
            state["g_entropy"] = torch.rand(rows, generator=gen, device="cuda") * 0.1
    else:
        k = case["k"]
        start = torch.randint(0, V, rows, generator=gen, device="cuda")
        step = torch.randint(1, max(2, V // k), rows, generator=gen, device="cuda")
        ar = torch.arange(k, device="cuda").view((1, k) + (1,) * (len(rows) - 1))
        idx = (start.unsqueeze(1) + step.unsqueeze(1) * ar) % V
        t = torch.randn((rows[0], k + 1) + rows[1:], generator=gen, device="cuda") * 2.0
        t = t.sort(dim=1, descending=True).values
        x.scatter_add_(1, idx, t[:, :k] + 3.0)
        lt = torch.log_softmax(t, 1)[:, :k]
        # the list of a row may be shorter than k (padding), or empty (a pixel outside the teacher's map)
        hole = torch.rand(rows, generator=gen, device="cuda") < case["holes"]
        keep = torch.randint(1, k + 1, rows, generator=gen, device="cuda")
        keep = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.8, torch.full_like(keep, k), keep)
        pad = hole.unsqueeze(1) | (ar >= keep.unsqueeze(1))
        state["teacher_index"] = idx.masked_fill(pad, -1).int()
        state["teacher"] = lt.contiguous()
        if case["train"]:
            state["g_loss"] = torch.rand(rows, generator=gen, device="cuda") + 0.5
    x = (x if sign > 0 else x.neg_()).to(dtype)
    if case["layout"] == "last":
        x = x.contiguous(memory_format=torch.channels_last)
    state["logits"] = x.requires_grad_(case["train"])
    return state


# --------------------------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        if state["case"]["op"] == "log_probs":
            return _plain_log_probs(state)
        return _plain_distill(state)


def _run_own(state):
    from depth_estimation_amd.distribution import distill_loss, log_probs
    case, x = state["case"], state["logits"]
    if case["op"] == "log_probs":
        out = log_probs(x, state["index"], scale=case["scale"], top=case["top"])
        if case["train"]:
            grad, = torch.autograd.grad([out.log_prob, out.entropy], [x], [state["g_log_prob"], state["g_entropy"]])
            return {"log_prob": out.log_prob.detach(), "entropy": out.entropy.detach(), "grad": grad}
        if case["top"]:
            return {"log_prob": out.log_prob, "entropy": out.entropy, "top_log_prob": out.top_log_prob,
                    "top_index": out.top_index}
        return {"log_prob": out.log_prob, "entropy": out.entropy}
    loss = distill_loss(x, state["teacher"], state["teacher_index"], scale=case["scale"],
                        renormalise=case["renormalise"])
    if case["train"]:
        grad, = torch.autograd.grad([loss], [x], [state["g_loss"]])
        return {"loss": loss.detach(), "grad": grad}
    return {"loss": loss}


def _plain_softmax(x, scale):
    """z - max, its exponential, and the sum over the classes, in 32 bits."""
    z = x.float() * scale
    t = z - z.amax(1, keepdim=True)
    e = t.exp()
    return t, e, e.sum(1, keepdim=True)


def _plain_log_probs(state):
    case, x, index = state["case"], state["logits"].detach(), state["index"]
    V, scale = case["classes"], case["scale"]
    t, e, s = _plain_softmax(x, scale)
    log_s = s.log()
    given = (index >= 0) & (index < V)
    at = index.clamp(0, V - 1).unsqueeze(1)
    log_prob = torch.where(given, (t.gather(1, at) - log_s).squeeze(1), 0.0)
    entropy = (log_s - (e * t.clamp_min(-1e30)).sum(1, keepdim=True) / s)
    out = {"log_prob": log_prob, "entropy": entropy.squeeze(1)}
    if case["top"]:
        # one unique whole number a class: the value in an order-keeping form above, the index below,
        # so that ties go to the lowest index
        v = x.float() if scale > 0 else -x.float()
        bits = (v + 0.0).view(torch.int32)
        order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long()
        ar = torch.arange(V, device=x.device).view((1, V) + (1,) * (x.dim() - 2))
        key = order * (1 << 32) + (V - 1 - ar)
        top = key.topk(case["top"], dim=1).values
        top_index = V - 1 - (top & 0xFFFFFFFF)
        out["top_log_prob"] = t.gather(1, top_index) - log_s
        out["top_index"] = top_index.int()
    if case["train"]:
        p = e / s
        g = torch.where(given, state["g_log_prob"], 0.0).unsqueeze(1)
        grad = -p * (g + state["g_entropy"].unsqueeze(1) * ((t - log_s).clamp_min(-1e30) + entropy))
        grad.scatter_add_(1, at, g)
        out["grad"] = (grad * scale).to(x.dtype)
    return out


def _plain_distill(state):
    case, x = state["case"], state["logits"].detach()
    scale, l, idx = case["scale"], state["teacher"].float(), state["teacher_index"].long()
    t, e, s = _plain_softmax(x, scale)
    valid = (idx >= 0) & (idx < case["classes"])
    at = idx.clamp(0, case["classes"] - 1)
    any_valid = valid.any(1, keepdim=True)
    if case["renormalise"]:
        u = torch.where(valid, l, -math.inf)
        u = u - torch.where(any_valid, u.amax(1, keepdim=True), 0.0)
        w = u.exp()
        total = torch.where(any_valid, w.sum(1, keepdim=True), 1.0)
        q, log_q = w / total, torch.where(valid, u - total.log(), 0.0)
        r = torch.zeros_like(total)
    else:
        log_q = torch.where(valid, l, 0.0)
        q = torch.where(valid, l.exp(), 0.0)
        r = torch.where(any_valid, (1.0 - q.sum(1, keepdim=True)).clamp_min(0.0), 0.0)
    loss = (q * (log_q - (t.gather(1, at) - s.log()))).sum(1, keepdim=True)
    # the classes the teacher does not list (padding is sent to a class of its own behind the last)
    marks = torch.zeros((x.shape[0], x.shape[1] + 1) + tuple(x.shape[2:]), device=x.device)
    marks.scatter_(1, torch.where(valid, idx, x.shape[1]), 1.0)
    unlisted = 1.0 - marks[:, :-1]
    rest = (e * unlisted).sum(1, keepdim=True)
    has = (r > 0) & (rest > 0)
    loss = loss + torch.where(has, r * (r.clamp_min(1e-38).log() - (rest / s).clamp_min(1e-38).log()), 0.0)
    out = {"loss": loss.squeeze(1)}
    if case["train"]:
        r = torch.where(has, r, 0.0)
        mass = q.sum(1, keepdim=True) + r
        grad = (e / s) * (mass - unlisted * torch.where(has, r * s / rest, 0.0))
        grad.scatter_add_(1, at, -q)
        out["grad"] = (grad * (state["g_loss"].unsqueeze(1) * scale)).to(x.dtype)
    return out


# ------------------------------------------------------------------------- work and 64 bits

def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    rows = case["batch"] * case["height"] * case["width"]
    n = rows * case["classes"]
    nbytes, flops = n * size, 6 * n                    # shift, exp, two sums with a product
    if case["op"] == "log_probs":
        nbytes += rows * (8 + 8 + 8 * case["top"])     # index in; log_prob, entropy, list out
        if case["train"]:
            nbytes += n * size + 8 * rows
            flops += 6 * n
    else:
        nbytes += rows * (8 * case["k"] + 4)           # the teacher's list in, the loss out
        if case["train"]:
            nbytes += n * size + 4 * rows
            flops += 4 * n
    return {"bytes": nbytes, "flops": flops}


def exact(case, seed):
    state = prepare(case, seed)
    z = (state["logits"].detach().double() * case["scale"]).requires_grad_(case["train"])
    logp = F.log_softmax(z, dim=1)
    V = case["classes"]
    if case["op"] == "log_probs":
        index = state["index"]
        given = (index >= 0) & (index < V)
        log_prob = torch.where(given, logp.gather(1, index.clamp(0, V - 1).unsqueeze(1)).squeeze(1), 0.0)
        entropy = -(logp.exp() * logp).sum(1)
        out = {"log_prob": log_prob.detach(), "entropy": entropy.detach()}
        if case["top"]:
            order = z.detach().sort(dim=1, descending=True, stable=True).indices[:, :case["top"]]
            out["top_log_prob"] = logp.detach().gather(1, order)
            out["top_index"] = order.int()
        outputs, ups = [log_prob, entropy], [state.get("g_log_prob"), state.get("g_entropy")]
    else:
        idx, l = state["teacher_index"].long(), state["teacher"].double()
        on = (idx >= 0) & (idx < V)
        alive = on.any(1)
        if case["renormalise"]:
            l = F.log_softmax(l.masked_fill(~on, -1e300), dim=1)
        q = l.exp() * on
        at = idx.clamp(0, V - 1)
        loss = (q * (torch.where(on, l, 0.0) - logp.gather(1, at))).sum(1)
        if not case["renormalise"]:
            mass = q.sum(1)
            listed_class = torch.zeros(z.shape, dtype=torch.uint8, device=z.device)
            listed_class.scatter_reduce_(1, at, on.to(torch.uint8), "amax")
            log_rest = logp.masked_fill(listed_class.bool(), -math.inf).logsumexp(1)
            r = (1.0 - mass).clamp_min(0.0)
            there = alive & (r > 0) & (listed_class == 0).any(1)
            log_rest = torch.where(there, log_rest, torch.zeros_like(log_rest))
            loss = loss + torch.where(there, r * (r.clamp_min(1e-300).log() - log_rest), 0.0)
        out = {"loss": loss.detach()}
        outputs, ups = [loss], [state.get("g_loss")]
    if case["train"]:
        grad, = torch.autograd.grad(outputs, [z], [g.double() for g in ups])
        out["grad"] = grad * case["scale"]
    return out
