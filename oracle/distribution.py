"""CPU restatement, in float64, of the operators over distributions of classes.

TEST INFRASTRUCTURE ONLY (see `oracle/__init__.py`).  The reference contains neither operator; the
definitions are the ones written out below (the usual soft-max, Shannon entropy and Kullback-Leibler
divergence), stated with the rules for masked classes and empty rows the kernels promise.  Every
function takes the class axis last.
"""
import torch

INF = float("inf")


def softmax(logits, scale):
    """(z, log p, p, empty): an empty row (every class at -inf) has log p = -inf and p = 0."""
    z = logits.double() * scale
    m = z.amax(-1, keepdim=True)
    empty = m == -INF
    t = z - torch.where(empty, 0.0, m)
    log_s = t.exp().sum(-1, keepdim=True).log()
    logp = torch.where((z == -INF) & ~log_s.isnan(), -INF, t - log_s)
    return z, logp, logp.exp(), empty[..., 0]


def _xlogx(p, logp):
    return torch.where(p == 0, 0.0, p * logp)


def log_probs(logits, index, scale=1.0, top=0):
    z, logp, p, _ = softmax(logits, scale)
    V = z.shape[-1]
    out = {"entropy": -_xlogx(p, logp).sum(-1)}
    if index is not None:
        given = (index >= 0) & (index < V)
        at = index.clamp(0, V - 1).long()[..., None]
        out["log_prob"] = torch.where(given, logp.gather(-1, at)[..., 0], 0.0)
    # the order of the classes is the order of the logits as they are stored (scale * x may round
    # different logits to one value); NaN first, equal values by lowest index
    v = logits.double() if scale > 0 else -logits.double()
    order = v.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    out["top_index"] = order.int()
    out["top_log_prob"] = logp.gather(-1, order)
    return out


def log_probs_grad(logits, index, scale, g_log_prob, g_entropy):
    """d (g_log_prob . log_prob + g_entropy . entropy) / d logits from the formula."""
    z, logp, p, empty = softmax(logits, scale)
    V = z.shape[-1]
    given = (index >= 0) & (index < V)
    gl = torch.where(given, g_log_prob.double(), 0.0)
    gh = g_entropy.double()
    H = -_xlogx(p, logp).sum(-1, keepdim=True)
    g = -gl[..., None] * p - gh[..., None] * (_xlogx(p, logp) + p * H)
    g.scatter_add_(-1, index.clamp(0, V - 1).long()[..., None], gl[..., None])
    quiet = empty | ((gl == 0) & (gh == 0))
    return torch.where(quiet[..., None], 0.0, g * scale)


def teacher(values, index, V, renormalise):
    """(valid, log q, q, r) of a teacher's list."""
    valid = (index >= 0) & (index < V)
    l = torch.where(valid, values.double(), -INF)
    if renormalise:
        m = l.amax(-1, keepdim=True)
        m = torch.where(m == -INF, 0.0, m)
        s = (l - m).exp().sum(-1, keepdim=True)
        l = torch.where(l == -INF, -INF, l - m - s.log())
    q = l.exp()
    r = torch.zeros_like(q[..., 0]) if renormalise else (1.0 - q.sum(-1)).clamp_min(0.0)
    return valid, l, q, torch.where(valid.any(-1), r, 0.0)


def _listed(index, valid, V):
    hits = torch.zeros(index.shape[:-1] + (V + 1,), dtype=torch.bool)
    hits.scatter_(-1, torch.where(valid, index.long(), V), True)
    return hits[..., :V]


def distill(logits, values, index, scale=1.0, renormalise=False):
    """dict: loss, gradient for an upstream gradient of 1, and the sizes rounding errors go by."""
    z, logp, p, empty = softmax(logits, scale)
    V = z.shape[-1]
    valid, l, q, r = teacher(values, index, V, renormalise)
    at = index.clamp(0, V - 1).long()
    listed = _listed(index, valid, V)
    lp_at = logp.gather(-1, at)
    live = q != 0
    loss = torch.where(live, q * (l - lp_at), 0.0).sum(-1)
    rest = torch.where(listed, -INF, z)
    m = rest.amax(-1)
    r = torch.where(m == -INF, 0.0, r)      # nothing unlisted is left of the student
    mz = torch.where(m == -INF, 0.0, m)
    e = (rest - mz[..., None]).exp()
    zm = z.amax(-1)
    zm = torch.where(zm == -INF, 0.0, zm)
    # the two maxima before the two logarithms: next to float32's largest values the logarithms would vanish
    log_P = (mz - zm) + (e.sum(-1).log() - (z - zm[..., None]).exp().sum(-1).log())
    loss = loss + torch.where(r > 0, r * (r.clamp_min(1e-300).log() - log_P), 0.0)
    alive = valid.any(-1)
    mass = q.sum(-1) + r
    share = torch.where((r > 0)[..., None], e / e.sum(-1, keepdim=True), 0.0)   # p_j / P, unlisted classes
    g = p * mass[..., None] - r[..., None] * share
    g.scatter_add_(-1, at, torch.where(valid, -q, 0.0))
    quiet = ~alive | empty | (mass == 0)
    size = torch.where(live, q * (l.abs() + lp_at.abs() + 1), 0.0).sum(-1) + \
        torch.where(r > 0, (r + 1e-6) * (r.clamp_min(1e-300).log().abs() + log_P.abs() + 1), 0.0)
    g_size = p * mass[..., None] + (r + 2e-7)[..., None] * share
    g_size.scatter_add_(-1, at, torch.where(valid, q, 0.0))
    return {"loss": torch.where(alive, loss, 0.0), "grad": torch.where(quiet[..., None], 0.0, g * scale),
            "size": size, "grad_size": g_size * abs(scale)}
