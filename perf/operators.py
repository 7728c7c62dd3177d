"""The two ends of a language model over its vocabulary table, as measured workloads.

take        out[i] = scale * table[index[i]]; an index outside the table gives a row of zeros
take_grad   grad[r] = scale * sum of g[i] over the i with index[i] == r; rows never named are zero
score       loss[i] and lse[i] of softmax cross entropy over logits = data . weight^T
train       the same loss with its gradients for data and weight

A row whose label is the ignored one, or lies outside the vocabulary, contributes nothing: its
loss, lse and gradients are zero.  Label smoothing spreads `smooth` evenly over the other classes.
"""
import math

import torch

own = False

IGNORED = -1
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token scored against the whole vocabulary: the last step of decoding with log-probabilities
        {"name": "score_1_bf16", "kind": "score", "n": 1, "v": 32000, "h": 1024, "dtype": "bf16", "ignored": 0.0, "smooth": 0.0},
        # a small batch of candidates, vocabulary of odd size
        {"name": "score_48_f16", "kind": "score", "n": 48, "v": 100003, "h": 2000, "dtype": "f16", "ignored": 0.1, "smooth": 0.0},
        # evaluation (perplexity) of a sequence
        {"name": "score_2048_bf16", "kind": "score", "n": 2048, "v": 32000, "h": 4096, "dtype": "bf16", "ignored": 0.0, "smooth": 0.0},
        # a small ragged training batch
        {"name": "train_257_f16", "kind": "train", "n": 257, "v": 32000, "h": 1024, "dtype": "f16", "ignored": 0.0, "smooth": 0.0},
        # a padded batch in which most tokens carry no loss, with label smoothing; nothing is a power of two
        {"name": "train_4096_padded_bf16", "kind": "train", "n": 4096, "v": 50021, "h": 1000, "dtype": "bf16", "ignored": 0.6, "smooth": 0.1},
        # a full training batch over a large vocabulary
        {"name": "train_8192_bf16", "kind": "train", "n": 8192, "v": 131072, "h": 4096, "dtype": "bf16", "ignored": 0.02, "smooth": 0.0},
        # one token on its way into a decoding step
        {"name": "take_1_bf16", "kind": "take", "n": 1, "v": 131072, "h": 4096, "dtype": "bf16", "scale": 1.0, "padding": 0.0},
        # an odd width: rows that start at any 2-byte address
        {"name": "take_4099_f16", "kind": "take", "n": 4099, "v": 50021, "h": 1001, "dtype": "f16", "scale": 0.5, "padding": 0.05},
        # a prompt batch with the embedding scaled by the square root of its width
        {"name": "take_32768_bf16", "kind": "take", "n": 32768, "v": 131072, "h": 4096, "dtype": "bf16", "scale": 64.0, "padding": 0.02},
        # the gradient of a few tokens
        {"name": "take_grad_64_f16", "kind": "take_grad", "n": 64, "v": 32000, "h": 1024, "dtype": "f16", "scale": 1.0, "padding": 0.0},
        # the gradient of a training batch
        {"name": "take_grad_16384_bf16", "kind": "take_grad", "n": 16384, "v": 131072, "h": 2048, "dtype": "bf16", "scale": 45.25, "padding": 0.02},
        # the repository's embedding configuration: 2^20 Zipf(1.1) tokens into a 262144 x 1024 table
        {"name": "take_grad_1048576_f32", "kind": "take_grad", "n": 1 << 20, "v": 262144, "h": 1024, "dtype": "f32", "scale": 1.0, "padding": 0.0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    h = _log_int(rng, low, high)
    step = rng.choice([1, 8, 64])
    return max(step, h // step * step)


def draw(rng):
    kind = rng.choice(["score", "train", "take", "take_grad"])
    if kind in ("score", "train"):
        return {"kind": kind, "n": _log_int(rng, 1, 8192), "v": _log_int(rng, 1000, 131072), "h": _width(rng, 64, 4096),
                "dtype": rng.choice(["f16", "bf16"]), "ignored": rng.choice([0.0, 0.05, 0.6]), "smooth": rng.choice([0.0, 0.0, 0.1])}
    wide = _width(rng, 64, 4096)
    return {"kind": kind, "n": _log_int(rng, 1, min(1 << 20, (1 << 30) // wide)), "v": _log_int(rng, 1000, 131072), "h": wide,
            "dtype": rng.choice(["f32", "f16", "bf16"]), "scale": rng.choice([1.0, 0.5, round(math.sqrt(wide), 3)]),
            "padding": rng.choice([0.0, 0.02])}


def _tokens(n, v, gen):
    """Zipf(1.1) tokens over [0, v), frequent ones scattered over the table."""
    mass = torch.arange(1, v + 1, device="cuda", dtype=torch.float64).pow_(-1.1).cumsum_(0)
    rank = torch.searchsorted(mass, torch.rand(n, device="cuda", dtype=torch.float64, generator=gen) * mass[-1]).clamp_(max=v - 1)
    return torch.randperm(v, device="cuda", generator=gen)[rank].to(torch.int32)


def _rows(n, share, gen):
    return torch.rand(n, device="cuda", generator=gen) < share


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    n, v, h = case["n"], case["v"], case["h"]
    dtype = DTYPES[case["dtype"]]
    state = dict(case)
    tokens = _tokens(n, v, gen)
    if case["kind"] in ("score", "train"):
        # logits of a model that has learnt something: standard deviation 2, the label's raised by 6
        weight = torch.randn(v, h, device="cuda", generator=gen).mul_(2.0 / math.sqrt(h))
        data = torch.randn(n, h, device="cuda", generator=gen)
        data += weight[tokens.long()] * 1.5
        tokens[_rows(n, case["ignored"], gen)] = IGNORED
        state.update(data=data.to(dtype), weight=weight.to(dtype), label=tokens,
                     loss=torch.empty(n, device="cuda"), lse=torch.empty(n, device="cuda"))
        live = int((tokens != IGNORED).sum())
        state["scale"] = 1.0 / max(live, 1)  # the mean over the tokens that count
        if case["kind"] == "train":
            state.update(gdata=torch.empty(n, h, device="cuda", dtype=dtype), gweight=torch.empty(v, h, device="cuda", dtype=dtype))
    else:
        tokens[_rows(n, case["padding"], gen)] = IGNORED
        state["index"] = tokens
        if case["kind"] == "take":
            state.update(table=torch.randn(v, h, device="cuda", generator=gen).mul_(0.02).to(dtype),
                         out=torch.empty(n, h, device="cuda", dtype=dtype))
        else:
            state.update(g=torch.randn(n, h, device="cuda", generator=gen).mul_(1e-3).to(dtype),
                         grad=torch.empty(v, h, device="cuda", dtype=dtype))
    if own:
        state["lib"], state["workspace"] = _workspace(case)
    return state


def _workspace(case):
    """The library and the scratch memory that a program allocates once for its batch size."""
    import mshadow_b200
    lib = mshadow_b200.load()
    n, v, h, dtype = case["n"], case["v"], case["h"], DTYPES[case["dtype"]]
    if case["kind"] == "take":
        return lib, None
    if case["kind"] == "take_grad":
        size = lib.embed_take_grad_workspace(n, v, h, dtype)
    else:
        size = lib.linear_softmax_loss_workspace(n, v, h, dtype, gradient=case["kind"] == "train")
    return lib, torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")


def _run_own(s):
    lib, stream = s["lib"], torch.cuda.current_stream().cuda_stream
    if s["kind"] == "take":
        return lib.embed_take(s["out"], s["table"], s["index"], scale=s["scale"], stream=stream)
    if s["kind"] == "take_grad":
        return lib.embed_take_grad(s["grad"], s["g"], s["index"], scale=s["scale"], workspace=s["workspace"], stream=stream)
    lib.linear_softmax_loss(s["loss"], s["lse"], s["data"], s["weight"], s["label"], ignore_label=IGNORED, smooth=s["smooth"],
                            workspace=s["workspace"], stream=stream)
    if s["kind"] == "score":
        return {"loss": s["loss"], "lse": s["lse"]}
    lib.linear_softmax_loss_grad(s["gdata"], s["gweight"], s["data"], s["weight"], s["label"], s["lse"], scale=s["scale"],
                                 ignore_label=IGNORED, smooth=s["smooth"], workspace=s["workspace"], stream=stream)
    return {"loss": s["loss"], "gdata": s["gdata"], "gweight": s["gweight"]}


def _run_plain(s):
    n, v = s["n"], s["v"]
    if s["kind"] in ("take", "take_grad"):
        index = s["index"].long()
        inside = (index >= 0) & (index < v)
        safe = torch.where(inside, index, 0)
        if s["kind"] == "take":
            return (s["table"][safe].float() * s["scale"] * inside[:, None]).to(s["table"].dtype)
        total = torch.zeros(v, s["h"], device="cuda").index_add_(0, safe, s["g"].float() * inside[:, None])
        return (total * s["scale"]).to(s["g"].dtype)
    data, weight, label = s["data"].float(), s["weight"].float(), s["label"].long()
    live = (label != IGNORED) & (label >= 0) & (label < v)
    safe = torch.where(live, label, 0)[:, None]
    other = s["smooth"] / (v - 1)
    logits = data @ weight.t()
    top = logits.amax(1)
    z = torch.gather(logits, 1, safe)[:, 0]
    lse = top + torch.exp(logits - top[:, None]).sum(1).log()
    loss = lse - (1.0 - s["smooth"]) * z
    if s["smooth"]:
        loss = loss - other * (logits.sum(1) - z)
    loss = torch.where(live, loss, 0.0)
    if s["kind"] == "score":
        return {"loss": loss, "lse": torch.where(live, lse, 0.0)}
    g = torch.exp(logits - lse[:, None])
    if s["smooth"]:
        g -= other
    g.scatter_add_(1, safe, torch.full((n, 1), other - (1.0 - s["smooth"]), device="cuda"))
    g *= (s["scale"] * live)[:, None]
    return {"loss": loss, "gdata": (g @ weight).to(s["data"].dtype), "gweight": (g.t() @ data).to(s["weight"].dtype)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    n, v, h = case["n"], case["v"], case["h"]
    e = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "take":
        kept = n * (1.0 - case["padding"])
        return {"bytes": int(kept * h * e + n * h * e + n * 4), "flops": int(kept * h)}
    if case["kind"] == "take_grad":
        kept = n * (1.0 - case["padding"])
        return {"bytes": int(kept * h * e + v * h * e + n * 4), "flops": int(2 * kept * h)}
    kept = n * (1.0 - case["ignored"])
    if case["kind"] == "score":
        return {"bytes": int((kept + v) * h * e + n * 12), "flops": int(2 * kept * v * h)}
    return {"bytes": int(2 * (kept + v) * h * e + n * 12), "flops": int(6 * kept * v * h)}


def exact(case, seed):
    """In 64 bits, a block of rows at a time."""
    s = prepare(case, seed)
    n, v, h = case["n"], case["v"], case["h"]
    if case["kind"] == "take":
        out = torch.zeros(n, h, dtype=torch.float64, device="cuda")
        rows = torch.nonzero((s["index"] >= 0) & (s["index"] < v))[:, 0]
        out[rows] = s["table"].index_select(0, s["index"][rows].long()).double() * s["scale"]
        return out
    if case["kind"] == "take_grad":
        rows = torch.nonzero((s["index"] >= 0) & (s["index"] < v))[:, 0]
        order = rows[torch.argsort(s["index"][rows], stable=True)]
        grad = torch.zeros(v, h, dtype=torch.float64, device="cuda")
        for part in torch.split(order, 1 << 17):
            grad.index_add_(0, s["index"][part].long(), s["g"][part].double() * s["scale"])
        return grad
    weight = s["weight"].double()
    loss = torch.zeros(n, dtype=torch.float64, device="cuda")
    lse = torch.zeros_like(loss)
    train = case["kind"] == "train"
    gdata = torch.zeros(n, h, dtype=torch.float64, device="cuda") if train else None
    gweight = torch.zeros(v, h, dtype=torch.float64, device="cuda") if train else None
    target = torch.full((v,), case["smooth"] / (v - 1), dtype=torch.float64, device="cuda")
    kept = torch.nonzero((s["label"] >= 0) & (s["label"] < v))[:, 0]
    for rows in torch.split(kept, 1024):
        if rows.numel() == 0:
            continue
        x = s["data"][rows].double()
        label = s["label"][rows].long()
        logp = torch.log_softmax(x.mm(weight.t()), 1)
        q = target.expand(rows.numel(), v).clone()
        q[torch.arange(rows.numel(), device="cuda"), label] = 1.0 - case["smooth"]
        loss[rows] = -(q * logp).sum(1)
        # the row's normaliser, from the label's own logit
        picked = (x * weight[label]).sum(1)
        lse[rows] = picked - logp[torch.arange(rows.numel(), device="cuda"), label]
        if train:
            d = (logp.exp() - q) * s["scale"]
            gdata[rows] = d.mm(weight)
            gweight += d.t().mm(x)
    if train:
        return {"loss": loss, "gdata": gdata, "gweight": gweight}
    return {"loss": loss, "lse": lse}
