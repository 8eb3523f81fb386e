"""Plain 64-bit forms of the row operators (counter-based dropout, layer norm of a residual sum, token log probabilities), with a
first-order bound of what fp32 arithmetic may add to each value.  CPU only; test infrastructure.

The bounds count roundings: ``U`` = 2^-24 is half a step of fp32 relative to the value, a sum of n terms taken by at least 32
threads adds at most (n / 32 + 40) roundings of the terms' absolute sum, and ``half_step`` is the one rounding to the output's
type.  ``SLACK`` covers second-order terms."""
import numpy as np
import torch

U = 2.0 ** -24
SLACK = 1.05
# fp32's smallest normal number: an exponential below it may be taken as zero.  Where it enters by itself that is TINY at most,
# where it is multiplied by a logarithm 100 * TINY (the logarithm of TINY is -87.3).
TINY = 2.0 ** -126


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def philox4x32_10(counter, key):
    """Words [n, 4] (uint64 holding 32 bits) of the given counters [n, 4] under one key (2 words)."""
    x = [counter[:, i].astype(np.uint64) for i in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> np.uint64(32)) ^ x[1] ^ np.uint64(k0), b & low, (a >> np.uint64(32)) ^ x[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(x, 1)


def words(seed: int, call: int, n: int, first: int = 0):
    """The random words of elements first .. first + n - 1 of a call."""
    blocks = np.arange(first // 4, (first + n + 3) // 4, dtype=np.uint64)
    seed, call = seed & (2 ** 64 - 1), call & (2 ** 64 - 1)
    c = np.stack([blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32), np.full_like(blocks, call & 0xFFFFFFFF),
                  np.full_like(blocks, call >> 32)], 1)
    w = philox4x32_10(c, (seed & 0xFFFFFFFF, seed >> 32)).reshape(-1)
    return w[first % 4:first % 4 + n]


def keep_mask(seed: int, call: int, p: float, shape, first: int = 0):
    n = int(np.prod(shape)) if len(shape) else 1
    border = round(p * 2 ** 32)
    return torch.from_numpy(words(seed, call, n, first) >= np.uint64(border)).reshape(shape)


def dropped(x, p, keep):
    """dropout(x) in 64 bits, what is dropped selected away."""
    if p >= 1.0:
        return torch.zeros_like(x)
    return torch.where(keep, x / (1.0 - p), torch.zeros_like(x))


def dropout(x, p, keep, residual=None):
    """(y, bound): float64 tensors."""
    v = dropped(x.double(), p, keep)
    y = v if residual is None else v + residual.double()
    return y, SLACK * (half_step(x.dtype) * y.abs() + U * (2 * v.abs() + y.abs()))


def layer_norm(x, weight, bias, eps, residual=None, p=0.0, keep=None):
    """((y, z, mean, rstd), bounds of each)."""
    cols = x.shape[-1]
    v = dropped(x.double(), p, keep) if p else x.double()
    z = v if residual is None else v + residual.double()
    w = torch.ones(cols, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(cols, dtype=torch.float64) if bias is None else bias.double()
    chain = cols / 32 + 40
    mean = z.mean(-1, keepdim=True)
    d = z - mean
    var = d.square().mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    y = d * rstd * w + b
    dz = U * (2 * v.abs() + z.abs())
    dmean = dz.mean(-1, keepdim=True) + chain * U * z.abs().mean(-1, keepdim=True) + 2 * U * mean.abs()
    dd = dz + dmean + U * d.abs()
    dvar = (2 * d.abs() * dd + dd.square()).mean(-1, keepdim=True) + (chain + 4) * U * var
    drstd = 0.5 * dvar / (var + eps) + 6 * U                     # relative; rsqrtf is off by at most 2 ulp = 4 U
    dy = w.abs() * rstd * (dd + d.abs() * drstd) + 3 * U * ((w * d * rstd).abs() + y.abs()) + half_step(x.dtype) * y.abs()
    return (y, z, mean[..., 0], rstd[..., 0]), (SLACK * dy, SLACK * (dz + half_step(x.dtype) * z.abs()), SLACK * dmean[..., 0],
                                                SLACK * (drstd * rstd)[..., 0])


def layer_norm_bwd(dy, z, weight, mean, rstd, p=0.0, keep=None, dz=None, param_dtype=None):
    """((dx, dresidual, dweight, dbias), bounds of each) from the stored z, mean and rstd."""
    cols, kind = dy.shape[-1], dy.dtype
    dy, z = dy.double().reshape(-1, cols), z.double().reshape(-1, cols)
    r, m = rstd.double().reshape(-1, 1), mean.double().reshape(-1, 1)
    w = torch.ones(cols, dtype=torch.float64) if weight is None else weight.double()
    chain, rows = cols / 32 + 40, dy.shape[0]
    u, g = (z - m) * r, dy * w
    c1, c2 = (g * u).mean(1, keepdim=True), g.mean(1, keepdim=True)
    t = (g - c2 - u * c1) * r
    out = t if dz is None else t + dz.double().reshape(-1, cols)
    du, dg = 3 * U * u.abs(), U * g.abs()
    dc2 = (chain + 3) * U * g.abs().mean(1, keepdim=True)
    dc1 = (chain + 8) * U * (g * u).abs().mean(1, keepdim=True)
    size = g.abs() + c2.abs() + (u * c1).abs()
    bound = r * (dg + dc2 + u.abs() * dc1 + c1.abs() * du + 5 * U * size) + 2 * U * out.abs()
    dx = out if not p else dropped(out, p, keep.reshape(-1, cols))
    dxb = bound if not p else dropped(bound, p, keep.reshape(-1, cols)) + 2 * U * dx.abs()
    dw, db = (dy * u).sum(0), dy.sum(0)
    ph = half_step(param_dtype or kind)
    dwb = (rows + 12) * U * (dy * u).abs().sum(0) + ph * dw.abs()
    dbb = (rows + 8) * U * dy.abs().sum(0) + ph * db.abs()
    h = half_step(kind)
    return (dx, out, dw, db), (SLACK * (dxb + h * dx.abs()), SLACK * (bound + h * out.abs()), SLACK * dwb, SLACK * dbb)


def _rel_exp(d):
    # the argument's roundings (in base 2: 3 of them) and the exponential's own error, 2^-22 or better
    return (8 + 4 * d.abs().clamp_max(200.0)) * U


def token_logprobs(logits, targets, ignore_index=-100, top=0):
    """dict of logprob, entropy, top_index, top_logprob, stats and a dict of bounds, for rows [rows, vocab] without NaN or +inf."""
    x = logits.double()
    vocab = x.shape[1]
    m = x.amax(1, keepdim=True)
    none = m[:, 0] == -np.inf
    d = torch.where(none[:, None], torch.zeros_like(x), x - m)
    e = d.exp()
    ed = torch.where(e > 0, e * d, torch.zeros_like(e))
    first = (d == 0)
    rest = torch.where(first, torch.zeros_like(e), e).sum(1)
    count = first.sum(1).double()
    total = count + rest
    logz = torch.where(none, torch.zeros_like(rest), torch.where(count == 1, rest.log1p(), total.log()))
    chain = vocab / 32 + 40
    finite_d = torch.where(e > 0, d, torch.zeros_like(d))
    others = torch.where(first, torch.zeros_like(e), e)
    drest = (others * _rel_exp(finite_d)).sum(1) + chain * U * rest
    dlogz = drest / total + 3 * U * logz.abs() + vocab * TINY
    entropy = torch.where(none, torch.zeros_like(rest), logz - ed.sum(1) / total)
    ted = ed.abs().sum(1)
    dentropy = dlogz + ((ed.abs() * (_rel_exp(finite_d) + 2 * U)).sum(1) + chain * U * ted) / total + ted / total * (drest / total + 4 * U) + 100 * vocab * TINY
    out, bound = {}, {}

    def logp_at(index):
        at = d.gather(1, index)
        lp = at - logz[:, None]
        lp = torch.where(none[:, None], torch.full_like(lp, -np.inf), lp)
        return lp, U * at.abs() + dlogz[:, None] + 2 * U * lp.abs()

    if targets is not None:
        counted = targets != ignore_index
        lp, b = logp_at(torch.where(counted, targets, torch.zeros_like(targets))[:, None])
        out["logprob"] = torch.where(counted, lp[:, 0], torch.zeros_like(logz))
        bound["logprob"] = SLACK * torch.where(counted, b[:, 0], torch.zeros_like(logz))
    out["entropy"], bound["entropy"] = entropy, SLACK * (dentropy + 3 * U * entropy.abs())
    if top:
        out["top_index"] = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        lp, b = logp_at(out["top_index"])
        out["top_logprob"], bound["top_logprob"] = lp, SLACK * b
    out["stats"] = torch.stack((m[:, 0], logz), 1)
    bound["stats"] = torch.stack((torch.zeros_like(logz), SLACK * dlogz), 1)
    return out, bound


def token_logprobs_bwd(logits, stats, targets=None, d_logprob=None, ignore_index=-100, entropy=None, d_entropy=None, top_index=None, d_top=None):
    """(grad, bound) from the stored statistics, for rows without NaN or +inf and targets inside the vocabulary."""
    x, kind = logits.double(), logits.dtype
    m, logz = stats[:, :1].double(), stats[:, 1:].double()
    none = m == -np.inf
    d = torch.where(none, torch.zeros_like(x), x - m)
    lp = d - logz
    p = lp.exp()
    share, dshare = torch.zeros_like(x), torch.zeros_like(x)
    whole, size = torch.zeros_like(m), torch.zeros_like(m)
    if d_logprob is not None:
        counted = targets != ignore_index
        a = torch.where(counted, d_logprob.double(), torch.zeros_like(d_logprob.double()))[:, None]
        share = share.scatter_add(1, torch.where(counted, targets, torch.zeros_like(targets))[:, None], a)
        whole, size = whole + a, size + a.abs()
    if d_top is not None:
        share = share.scatter_add(1, top_index, d_top.double())
        dshare = dshare.scatter_add(1, top_index, d_top.double().abs())
        whole, size = whole + d_top.double().sum(1, keepdim=True), size + d_top.double().abs().sum(1, keepdim=True)
    terms = 34                                                            # most summands of a share or of the whole
    live = p > 1e-60                                                      # below this fp32 has long flushed p to zero
    relp = torch.where(live, (8 + 4 * lp.abs().clamp_max(200.0)) * U + 2 * U * (d.abs() + logz.abs()).clamp_max(400.0), torch.zeros_like(p))
    grad = -share * torch.expm1(lp) + (share - whole) * p
    bound = (whole.abs() + 2 * share.abs()) * p * relp + terms * U * (size * p + dshare + share.abs()) * 1.0 + 4 * U * grad.abs()
    if d_entropy is not None:
        dh, h = d_entropy.double()[:, None], entropy.double()[:, None]
        part = torch.where(live, dh * p * (lp + h), torch.zeros_like(p))
        grad = grad - part
        bound = bound + torch.where(live, dh.abs() * p * ((lp + h).abs() * (relp + 4 * U) + 2 * U * (d.abs() + logz.abs() + lp.abs() + h.abs())),
                                    torch.zeros_like(p)) + 2 * U * (grad.abs() + part.abs())
    grad = torch.where(none, torch.zeros_like(grad), grad)
    bound = torch.where(none, torch.zeros_like(bound), bound)
    flushed = 1 + size + (100 * d_entropy.double().abs()[:, None] if d_entropy is not None else 0)
    return grad, SLACK * (bound + half_step(kind) * grad.abs()) + 2 * TINY * flushed
