"""The row operators of a fine-tuning step around the compressed sites: what is measured of them.

dropout   y = residual + keep * x / (1 - p), with the mask drawn from a counter-based generator (Philox4x32-10: element i of
          call c takes word i % 4 of the block with counter (i // 4, c) under the key `seed`), so that no mask is ever stored;
          its backward pass draws the same mask again
norm      layer norm of a residual sum, y = LN(residual + dropout(x)) * weight + bias, and its backward pass with the
          gradients of weight and bias
logprob   log probabilities of given tokens under a row of logits, with the entropy of the row and its `top` best
          alternatives, and the gradient of all three with respect to the logits

Sizes are those of this repository's hosts (hidden 768 and 4096, 11008 channels of the feed-forward layer, vocabularies of 32000
and 50265) or generic ones around them."""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp32": 4}
IGNORE = -100


def listed():
    return [
        # the hidden dropout of an encoder's block in front of a norm that compresses its input: 16 sequences of 128 tokens
        dict(name="dropout_add_2048x768", op="dropout", way="forward", rows=2048, cols=768, type="bf16", p=0.1, residual=True),
        # a full-precision head's dropout, a width that no vector divides
        dict(name="dropout_fp32_1537x1001", op="dropout", way="forward", rows=1537, cols=1001, type="fp32", p=0.5, residual=False),
        # backward through the dropout in front of an adapter on the feed-forward activation of a long batch
        dict(name="dropout_grad_16384x11008", op="dropout", way="backward", rows=16384, cols=11008, type="bf16", p=0.05, residual=False),
        # one token through a norm, where launch latency is all there is
        dict(name="norm_1x768", op="norm", way="forward", rows=1, cols=768, type="bf16", params="bf16", p=0.0, residual=False, stream=False),
        # the end of an encoder's sublayer in training: dropout, residual, norm; 32 sequences of 128 tokens
        dict(name="norm_add_4096x768", op="norm", way="forward", rows=4096, cols=768, type="bf16", params="bf16", p=0.1, residual=True, stream=False),
        # its backward pass at the width and token count of a large model's step
        dict(name="norm_grad_65536x4096", op="norm", way="backward", rows=65536, cols=4096, type="bf16", params="fp32", p=0.1, residual=True, stream=False),
        # full precision, odd sizes, the sum also used behind the norm (a pre-norm residual stream)
        dict(name="norm_grad_fp32_3001x1003", op="norm", way="backward", rows=3001, cols=1003, type="fp32", params="fp32", p=0.0, residual=True, stream=True),
        # the answer of a served model: eight sequences, one token each, with its alternatives
        dict(name="logprob_top_8x32000", op="logprob", way="forward", rows=8, vocab=32000, type="bf16", top=20, entropy=True, ignored=0.0, masked=0.0),
        # scoring a batch of prompts and completions, prompts without a target
        dict(name="logprob_score_4096x32000", op="logprob", way="forward", rows=4096, vocab=32000, type="bf16", top=5, entropy=True, ignored=0.3, masked=0.0),
        # a large vocabulary, most of it closed by a mask of -inf and of the type's lowest value
        dict(name="logprob_masked_96x200001", op="logprob", way="forward", rows=96, vocab=200001, type="bf16", top=1, entropy=True, ignored=0.0, masked=0.6),
        # the gradient of the language-model loss of a training step
        dict(name="logprob_grad_8192x32000", op="logprob", way="backward", rows=8192, vocab=32000, type="bf16", top=0, entropy=False, ignored=0.25, masked=0.0),
        # a policy's gradient with an entropy bonus and distilled alternatives, full precision, an odd vocabulary
        dict(name="logprob_grad_fp32_513x50265", op="logprob", way="backward", rows=513, vocab=50265, type="fp32", top=4, entropy=True, ignored=0.1, masked=0.0),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op, way, kind = rng.choice(["dropout", "norm", "logprob"]), rng.choice(["forward", "backward"]), rng.choice(["bf16", "bf16", "fp32"])
    limit = 1 << 27                                                     # elements
    if op == "logprob":
        vocab = rng.choice([_spread(rng, 100, 200001), 32000, 50265])
        rows = _spread(rng, 1, max(1, min(8192, limit // vocab)))
        return dict(op=op, way=way, rows=rows, vocab=vocab, type=kind, top=rng.choice([0, 1, 5, _spread(rng, 1, 32)]), entropy=rng.random() < 0.5,
                    ignored=rng.choice([0.0, rng.uniform(0.0, 0.9)]), masked=rng.choice([0.0, rng.uniform(0.0, 0.9)]))
    cols = rng.choice([_spread(rng, 8, 16384), 8 * _spread(rng, 1, 2048), 768, 4096])
    rows = _spread(rng, 1, max(1, min(65536, limit // cols)))
    p = rng.choice([0.0, 0.1, rng.uniform(0.01, 0.9)]) if op == "norm" else rng.choice([0.1, rng.uniform(0.01, 0.9)])
    case = dict(op=op, way=way, rows=rows, cols=cols, type=kind, p=p, residual=rng.random() < 0.5)
    if op == "dropout":
        case["residual"] = case["residual"] and way == "forward"        # the residual's gradient is the arriving one
        return case
    return dict(case, params=rng.choice([kind, "fp32"]), stream=way == "backward" and rng.random() < 0.3)


# ---------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = _TYPES[case["type"]]
    state = {"case": case}

    def normal(*shape, scale=1.0):
        return torch.randn(shape, device="cuda", generator=gen).mul_(scale)

    def uniform(*shape):
        return torch.rand(shape, device="cuda", generator=gen)

    if case["op"] in ("dropout", "norm"):
        rows, cols = case["rows"], case["cols"]
        # activations: a few channels far larger than the others
        wide = torch.where(uniform(cols) < 0.01, 20.0, 1.0)
        seed_and_call = torch.randint(0, 1 << 62, (2,), device="cuda", generator=gen)
        state["rng"] = seed_and_call
    if case["op"] == "dropout":
        state["x"] = (normal(rows, cols) * wide).to(kind)
        state["residual"] = (normal(rows, cols) * wide).to(kind) if case["residual"] else None
    elif case["op"] == "norm":
        params = _TYPES[case["params"]]
        state["weight"] = (1 + normal(cols, scale=0.1)).to(params)
        state["bias"] = normal(cols, scale=0.1).to(params)
        x = (normal(rows, cols) * wide + 0.1).to(kind)
        if case["way"] == "forward":
            state["x"] = x
            state["residual"] = (normal(rows, cols) * wide).to(kind) if case["residual"] else None
        else:
            # what the forward pass keeps: the sum in front of the norm, its row means and reciprocal deviations
            state["z"] = x
            mean, rstd = [], []
            for part in x.split(4096):
                wide_part = part.double()
                m = wide_part.mean(1)
                mean.append(m.float())
                rstd.append(torch.rsqrt((wide_part - m[:, None]).square().mean(1) + 1e-5).float())
            state["mean"], state["rstd"] = torch.cat(mean), torch.cat(rstd)
            state["dy"] = normal(rows, cols).to(kind)
            state["dz"] = normal(rows, cols).to(kind) if case["stream"] else None
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab, scale=2.0)
        targets = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
        # trained models: the token that came is often the likely one, by a margin of its own in each row
        boost = uniform(rows) * 24.0
        logits[torch.arange(rows, device="cuda"), targets] += boost
        if case["masked"]:
            closed = uniform(vocab) < case["masked"]
            lowest = torch.finfo(kind).min
            shut = torch.where(uniform(vocab) < 0.5, float("-inf"), lowest)
            closed[: min(vocab, 40)] = False
            logits = torch.where(closed, shut, logits)
            targets = torch.where(closed[targets], targets % min(vocab, 40), targets)
        state["logits"] = logits.to(kind)
        del logits
        if case["ignored"]:
            targets = torch.where(uniform(rows) < case["ignored"], IGNORE, targets)
        state["targets"] = targets
        if case["way"] == "backward":
            # what the forward pass keeps of each row: its largest logit, the logarithm of the sum of exp(x - largest), entropy
            stats, entropy = [], []
            for part in state["logits"].split(256):
                d = part.double()
                top = d.amax(1, keepdim=True)
                d = d - top
                e = torch.exp(d)
                total = e.sum(1)
                stats.append(torch.stack((top[:, 0].float(), total.log().float()), 1))
                entropy.append((total.log() - torch.where(e > 0, e * d, 0.0).sum(1) / total).float())
            state["stats"] = torch.cat(stats)
            state["entropy"] = torch.cat(entropy) if case["entropy"] else None
            counted = max(1, int((targets != IGNORE).sum()))
            state["d_logprob"] = normal(rows) / counted
            state["d_entropy"] = normal(rows) / counted if case["entropy"] else None
            if case["top"]:
                k = min(case["top"], vocab)
                state["top_index"] = torch.topk(state["logits"].float(), k, dim=1).indices
                state["d_top"] = normal(rows, k) / counted
    return state


# ---------------------------------------------------------------------------------------------------- plain forms

def _philox(rng, blocks):
    """The four words of counter blocks 0 .. blocks - 1 of call rng[1] under the key rng[0], as int64 [blocks, 4]."""
    low = 0xFFFFFFFF
    i = torch.arange(blocks, device=rng.device)
    c0, c1 = i & low, i >> 32
    c2, c3 = (rng[1] & low).expand_as(i), (rng[1] >> 32 & low).expand_as(i)
    k0, k1 = rng[0] & low, rng[0] >> 32 & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57        # the 64 bits of each product
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    return torch.stack((c0, c1, c2, c3), 1)


def _keep(rng, p, shape):
    n = shape[0] * shape[1]
    words = _philox(rng, (n + 3) // 4).reshape(-1)[:n].reshape(shape)
    return words >= round(p * 4294967296.0)


def _plain_dropout(s, case):
    x = s["x"].float()
    y = torch.where(_keep(s["rng"], case["p"], x.shape), x * (1.0 / (1.0 - case["p"])), 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _plain_norm(s, case):
    z = s["x"].float()
    if case["p"]:
        z = torch.where(_keep(s["rng"], case["p"], z.shape), z * (1.0 / (1.0 - case["p"])), 0.0)
    if s["residual"] is not None:
        z = z + s["residual"].float()
    mean = z.mean(1, keepdim=True)
    d = z - mean
    rstd = torch.rsqrt(d.square().mean(1, keepdim=True) + 1e-5)
    y = d * rstd * s["weight"].float() + s["bias"].float()
    kind = s["x"].dtype
    return y.to(kind), z.to(kind), mean[:, 0], rstd[:, 0]


def _plain_norm_grad(s, case):
    kind, params = s["z"].dtype, s["weight"].dtype
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xhat = (s["z"].float() - s["mean"][:, None]) * rstd
    wdy = dy * s["weight"].float()
    dz = (wdy - xhat * (xhat * wdy).mean(1, keepdim=True) - wdy.mean(1, keepdim=True)) * rstd
    if s["dz"] is not None:
        dz = dz + s["dz"].float()
    dweight, dbias = (dy * xhat).sum(0).to(params), dy.sum(0).to(params)
    if not case["p"]:
        return dz.to(kind), dweight, dbias
    dx = torch.where(_keep(s["rng"], case["p"], dz.shape), dz * (1.0 / (1.0 - case["p"])), 0.0)
    return dx.to(kind), dz.to(kind), dweight, dbias


def _plain_logprob(s, case):
    x = s["logits"].float()
    largest = x.amax(1, keepdim=True)
    d = x - largest
    e = torch.exp(d)
    # the sums in 64 bits: behind the 1 of a row's largest logit, 32 lose all that makes a confident row's result
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    logz = total.log()
    counted = s["targets"] != IGNORE
    at = torch.where(counted, s["targets"], 0)[:, None]
    out = {"logprob": torch.where(counted, (d.gather(1, at) - logz)[:, 0], 0.0).float()}
    if case["entropy"]:
        out["entropy"] = (logz - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True, dtype=torch.float64) / total)[:, 0].float()
    if case["top"]:
        # largest value first, the lower index first among equals: both in one integer
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        index = torch.arange(x.shape[1], device=x.device)
        best = torch.topk(order * 4294967296 + (4294967295 - index), min(case["top"], x.shape[1]), dim=1).values
        out["top_index"] = 4294967295 - (best & 4294967295)
        out["top_logprob"] = (d.gather(1, out["top_index"]) - logz).float()
    return out


def _plain_logprob_grad(s, case):
    logp = s["logits"].float() - s["stats"][:, :1] - s["stats"][:, 1:]
    counted = s["targets"] != IGNORE
    # the tokens that a gradient arrives for, with the sum of what arrives for each of them
    index = torch.where(counted, s["targets"], 0)[:, None]
    arrives = torch.where(counted, s["d_logprob"], 0.0)[:, None]
    if case["top"]:
        index, arrives = torch.cat((index, s["top_index"]), 1), torch.cat((arrives, s["d_top"]), 1)
    whole = arrives.sum(1, keepdim=True)
    own_share = torch.where(index[:, :, None] == index[:, None, :], arrives[:, None, :], 0.0).sum(2)
    there = logp.gather(1, index)
    # share - whole * prob, with 1 - prob taken as expm1 where prob is near one
    value = (own_share - whole) * torch.exp(there) - own_share * torch.expm1(there)
    prob = torch.exp(logp)
    grad = (-whole * prob).scatter(1, index, value)
    if case["entropy"]:
        grad = grad - s["d_entropy"][:, None] * torch.where(prob > 0, prob * (logp + s["entropy"][:, None]), 0.0)
    return grad.to(s["logits"].dtype)


def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    if case["op"] == "dropout":
        return _plain_dropout(state, case)
    if case["op"] == "norm":
        return _plain_norm(state, case) if case["way"] == "forward" else _plain_norm_grad(state, case)
    return _plain_logprob(state, case) if case["way"] == "forward" else _plain_logprob_grad(state, case)


def _own(s, case):
    from hyc_lora_b200 import rowops

    if case["op"] == "dropout":
        return rowops.dropout(s["x"], case["p"], s["rng"], residual=s["residual"])
    if case["op"] == "norm":
        if case["way"] == "forward":
            out = rowops.layer_norm(s["x"], s["weight"], s["bias"], 1e-5, residual=s["residual"], p=case["p"], rng=s["rng"])
            return out.y, out.z, out.mean, out.rstd
        dx, dresidual, dweight, dbias = rowops.layer_norm_bwd(s["dy"], s["z"], s["weight"], s["mean"], s["rstd"], p=case["p"], rng=s["rng"], dz=s["dz"])
        return (dx, dresidual, dweight, dbias) if case["p"] else (dresidual, dweight, dbias)
    if case["way"] == "forward":
        got = rowops.token_logprobs(s["logits"], s["targets"], ignore_index=IGNORE, entropy=case["entropy"], top=min(case["top"], case["vocab"]))
        out = {"logprob": got.logprob}
        if case["entropy"]:
            out["entropy"] = got.entropy
        if case["top"]:
            out["top_index"], out["top_logprob"] = got.top_index, got.top_logprob
        return out
    return rowops.token_logprobs_bwd(s["logits"], s["stats"], s["targets"], s["d_logprob"], ignore_index=IGNORE, entropy=s["entropy"],
                                     d_entropy=s["d_entropy"], top_index=s.get("top_index"), d_top=s.get("d_top"))


# ---------------------------------------------------------------------------------------------------- least work

def work(case):
    size = _BYTES[case["type"]]
    if case["op"] == "logprob":
        n, rows = case["rows"] * case["vocab"], case["rows"]
        if case["way"] == "forward":
            out = 4 * (1 + case["entropy"]) + 12 * min(case["top"], case["vocab"])
            return {"bytes": n * size + rows * (8 + out), "flops": n * (3 + 2 * case["entropy"])}
        # rows without a target and without any other gradient are zeros: their logits need not be read
        read = n if case["entropy"] or case["top"] else n * (1 - case["ignored"])
        into = 8 + 8 + 4 + 8 * case["entropy"] + 12 * min(case["top"], case["vocab"])
        return {"bytes": int((read + n) * size + rows * into), "flops": int(read * (3 + 3 * case["entropy"]))}
    n, rows, cols = case["rows"] * case["cols"], case["rows"], case["cols"]
    if case["op"] == "dropout":
        return {"bytes": n * size * (3 if case["residual"] else 2), "flops": n * 2}
    drop = case["p"] > 0
    if case["way"] == "forward":
        tensors = 2 + case["residual"] + (1 if drop or case["residual"] else 0)
        return {"bytes": n * size * tensors + 8 * rows + 2 * cols * _BYTES[case["params"]], "flops": n * 8}
    tensors = 3 + drop + case["stream"]
    return {"bytes": n * size * tensors + 8 * rows + 3 * cols * _BYTES[case["params"]], "flops": n * 13}


# ---------------------------------------------------------------------------------------------------- 64 bits

def _exact_keep(rng, p, shape):
    """Philox4x32-10 from its definition, products taken in 16-bit pieces."""
    n, full = shape[0] * shape[1], (1 << 32) - 1
    seed, call = (int(v) for v in rng.tolist())

    def product(word, factor):
        upper, lower = word * (factor >> 16), word * (factor & 0xFFFF)
        middle = upper + lower.bitwise_right_shift(16)
        return middle.bitwise_right_shift(16), (middle.bitwise_and(0xFFFF) * 65536) + lower.bitwise_and(0xFFFF)

    block = torch.arange((n + 3) // 4, device=rng.device)
    x = [block % (1 << 32), block // (1 << 32), torch.full_like(block, call & full), torch.full_like(block, call >> 32 & full)]
    key = [seed & full, seed >> 32 & full]
    for turn in range(10):
        h0, l0 = product(x[0], 0xD2511F53)
        h1, l1 = product(x[2], 0xCD9E8D57)
        x = [h1.bitwise_xor(x[1]).bitwise_xor(key[0]), l1, h0.bitwise_xor(x[3]).bitwise_xor(key[1]), l0]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    border = round(p * (1 << 32))
    keep = torch.empty((block.numel(), 4), dtype=torch.bool, device=rng.device)
    for word in range(4):
        keep[:, word] = x[word] >= border
    return keep.view(-1)[:n].view(shape)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "dropout":
        y = s["x"].double() / (1.0 - case["p"])
        y = y.masked_fill_(~_exact_keep(s["rng"], case["p"], y.shape), 0.0)
        return y if s["residual"] is None else y.add_(s["residual"])
    if case["op"] == "norm":
        return _exact_norm(s, case) if case["way"] == "forward" else _exact_norm_grad(s, case)
    return _exact_logprob(s, case) if case["way"] == "forward" else _exact_logprob_grad(s, case)


def _exact_norm(s, case):
    z = s["x"].double()
    if case["p"]:
        z = (z / (1.0 - case["p"])).masked_fill_(~_exact_keep(s["rng"], case["p"], z.shape), 0.0)
    if s["residual"] is not None:
        z = z + s["residual"].double()
    mean = z.sum(1) / z.shape[1]
    variance = (z - mean[:, None]).pow_(2).sum(1) / z.shape[1]
    deviation = (variance + 1e-5).sqrt()
    y = (z - mean[:, None]).div_(deviation[:, None]).mul_(s["weight"].double()).add_(s["bias"].double())
    return y, z, mean, 1.0 / deviation


def _exact_norm_grad(s, case):
    weight, n = s["weight"].double(), s["z"].shape[1]
    keep = _exact_keep(s["rng"], case["p"], s["z"].shape) if case["p"] else None
    dweight, dbias = torch.zeros_like(weight), torch.zeros_like(weight)
    dx, dz = [], []
    for first in range(0, s["z"].shape[0], 8192):
        part = slice(first, first + 8192)
        dy, rstd = s["dy"][part].double(), s["rstd"][part].double()[:, None]
        unit = (s["z"][part].double() - s["mean"][part].double()[:, None]) * rstd
        dweight += torch.einsum("rc,rc->c", dy, unit)
        dbias += dy.sum(0)
        g = dy * weight
        g = rstd * (g - g.sum(1, keepdim=True) / n - unit * ((g * unit).sum(1, keepdim=True) / n))
        if s["dz"] is not None:
            g = g + s["dz"][part].double()
        dz.append(g)
        if keep is not None:
            dx.append((g / (1.0 - case["p"])).masked_fill_(~keep[part], 0.0))
    dz = torch.cat(dz)
    return (torch.cat(dx), dz, dweight, dbias) if keep is not None else (dz, dweight, dbias)


def _exact_logprob(s, case):
    parts = []
    for first in range(0, case["rows"], 512):
        x, t = s["logits"][first:first + 512].double(), s["targets"][first:first + 512]
        logp = x - torch.logsumexp(x, 1, keepdim=True)
        out = {"logprob": torch.where(t == IGNORE, 0.0, logp.gather(1, t.clamp_min(0)[:, None])[:, 0])}
        if case["entropy"]:
            out["entropy"] = -torch.special.xlogy(logp.exp(), logp.exp()).sum(1)
        if case["top"]:
            k = min(case["top"], case["vocab"])
            out["top_index"] = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
            out["top_logprob"] = logp.gather(1, out["top_index"])
        parts.append(out)
    return {name: torch.cat([p[name] for p in parts]) for name in parts[0]}


def _exact_logprob_grad(s, case):
    grads = []
    for first in range(0, case["rows"], 512):
        part = slice(first, first + 512)
        logp = s["logits"][part].double() - s["stats"][part].double().sum(1, keepdim=True)
        prob = logp.exp()
        t = s["targets"][part]
        d = s["d_logprob"][part].double().masked_fill(t == IGNORE, 0.0)[:, None]
        hot = torch.zeros_like(prob).scatter_(1, t.clamp_min(0)[:, None], 1.0)
        grad = d * (hot - prob)
        if case["entropy"]:
            grad -= s["d_entropy"][part].double()[:, None] * (torch.special.xlogy(prob, prob) + prob * s["entropy"][part].double()[:, None])
        if case["top"]:
            for k in range(s["top_index"].shape[1]):
                hot = torch.zeros_like(prob).scatter_(1, s["top_index"][part, k:k + 1], 1.0)
                grad += s["d_top"][part, k:k + 1].double() * (hot - prob)
        grads.append(grad)
    return torch.cat(grads)
