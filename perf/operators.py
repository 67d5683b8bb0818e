"""Timed cases of three operators beside the FP8 linear layers: low-rank adapters of many requests beside a shared
projection (forward, and forward + backward), a whole mixture-of-experts layer for a few tokens, and the global gradient
norm over many tensors with clipping.

``own`` chooses between the plain forms written here in elementary torch operations and the framework's kernels.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one request's next token through a projection with its adapter: latency
        {"name": "adapter 1 token", "op": "lora", "t": 1, "k": 4096, "o": 4096, "r": 16, "n": 8, "dtype": "bf16", "order": "mixed"},
        # a decode batch: every row another request, half as many adapters as rows, some rows without one
        {"name": "adapter 96 requests", "op": "lora", "t": 96, "k": 4096, "o": 14336, "r": 16, "n": 48, "dtype": "bf16",
         "order": "mixed"},
        # prompts of a few requests back to back; odd row count, output width and rank
        {"name": "adapter ragged prompts", "op": "lora", "t": 2931, "k": 2056, "o": 2731, "r": 20, "n": 5, "dtype": "fp16",
         "order": "runs"},
        # fine-tuning one adapter beside the 4096 -> 14336 projection on 8192 tokens
        {"name": "adapter training", "op": "lora_train", "t": 8192, "k": 4096, "o": 14336, "r": 32, "n": 1, "dtype": "bf16",
         "order": "runs"},
        # several adapters trained in one batch of ragged rows
        {"name": "adapter training ragged", "op": "lora_train", "t": 1777, "k": 1160, "o": 904, "r": 8, "n": 6, "dtype": "fp16",
         "order": "mixed"},
        # one token through 2 of 8 large experts
        {"name": "experts 1 token", "op": "moe", "t": 1, "h": 4096, "f": 14336, "e": 8, "topk": 2, "dtype": "bf16",
         "weights": "bf16"},
        # a small decode batch over many small experts, FP8 weights with one scale per expert
        {"name": "experts many small fp8", "op": "moe", "t": 5, "h": 2048, "f": 1408, "e": 64, "topk": 8, "dtype": "bf16",
         "weights": "fp8"},
        # a full decode batch that reaches every expert, FP8 weights
        {"name": "experts 64 tokens fp8", "op": "moe", "t": 64, "h": 4096, "f": 14336, "e": 8, "topk": 2, "dtype": "bf16",
         "weights": "fp8"},
        # odd sizes, half precision
        {"name": "experts odd fp16", "op": "moe", "t": 23, "h": 1096, "f": 712, "e": 16, "topk": 4, "dtype": "fp16",
         "weights": "fp16"},
        # adapter gradients of a whole model: many small tensors, latency of a few launches
        {"name": "clip adapter gradients", "op": "clip", "tensors": 56, "numel": 65536, "ragged": False, "dtype": "bf16",
         "out": "bf16"},
        # a bucket of full weight gradients
        {"name": "clip weight gradients", "op": "clip", "tensors": 9, "numel": 58720256, "ragged": False, "dtype": "bf16",
         "out": "bf16"},
        # ragged odd lengths, half-precision gradients clipped into fp32 ones
        {"name": "clip ragged fp16", "op": "clip", "tensors": 37, "numel": 300007, "ragged": True, "dtype": "fp16",
         "out": "fp32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lora", "lora", "lora_train", "moe", "moe", "clip"])
    if op in ("lora", "lora_train"):
        t = _log(rng, 1, 8192) if op == "lora" else _log(rng, 64, 8192)
        k, o = _log(rng, 256, 8192 if op == "lora" else 4096), _log(rng, 256, 14336)
        if rng.random() < 0.7:
            k, o = k // 8 * 8, o // 8 * 8
        r = rng.choice([4, 8, 12, 16, 20, 32, 48, 64])
        return {"op": op, "t": t, "k": k, "o": o, "r": r, "n": rng.randint(1, 512 // r if op == "lora" else 8), "dtype": rng.choice(["bf16", "fp16"]),
                "order": rng.choice(["runs", "mixed"])}
    if op == "moe":
        weights = rng.choice(["same", "fp8"])
        dtype = rng.choice(["bf16", "bf16", "fp16"]) if weights == "same" else "bf16"
        e = rng.choice([4, 8, 16, 32, 64])
        k = rng.randint(1, min(8, e))
        h, f = _log(rng, 512, 4096) // 16 * 16, _log(rng, 512, 14336 if e <= 8 else 2048) // 16 * 16
        if weights == "same" and rng.random() < 0.3:
            h, f = h + 8, f + 8
        return {"op": op, "t": _log(rng, 1, 64), "h": h, "f": f, "e": e, "topk": k, "dtype": dtype,
                "weights": dtype if weights == "same" else "fp8"}
    n = _log(rng, 1, 300)
    return {"op": op, "tensors": n, "numel": _log(rng, 100, 120_000_000 // n), "ragged": rng.random() < 0.5,
            "dtype": rng.choice(["bf16", "fp16", "fp32"]), "out": rng.choice(["same", "fp32"])}


# ------------------------------------------------------------------------------------------------ inputs
def _adapter_ids(c, g):
    """Per token the adapter it uses, -1 = none (about one row in 16 where the batch is a mix of requests)."""
    t, n = c["t"], c["n"]
    if t == 1:
        return torch.randint(0, n, (1,), generator=g, device="cuda", dtype=torch.int32)
    if c["order"] == "runs":  # requests back to back: ids rise along the batch, runs of uneven length
        cut = torch.rand(n, generator=g, device="cuda").sort().values
        pos = torch.arange(t, device="cuda", dtype=torch.float32) / t
        ids = (pos[:, None] > cut[None, :]).sum(1).clamp(max=n - 1)
        return ids.to(torch.int32)
    ids = torch.randint(0, n, (t,), generator=g, device="cuda", dtype=torch.int32)
    none = torch.rand(t, generator=g, device="cuda") < 1 / 16
    return torch.where(none, -1, ids)


def _lengths(c):
    if not c["ragged"]:
        return [c["numel"]] * c["tensors"]
    return [max(1, c["numel"] * (1 + (7 * i) % 11) // 11 - i % 3) for i in range(c["tensors"])]


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    if c["op"] in ("lora", "lora_train"):
        dt = _DT[c["dtype"]]
        s = {"case": c, "x": randn(c["t"], c["k"], dtype=dt), "a": randn(c["n"], c["r"], c["k"], dtype=dt, std=c["k"] ** -0.5),
             "b": randn(c["n"], c["o"], c["r"], dtype=dt, std=c["r"] ** -0.5), "base": randn(c["t"], c["o"], dtype=dt),
             "scaling": 0.5 + torch.rand(c["n"], generator=g, device="cuda"), "ids": _adapter_ids(c, g)}
        if c["op"] == "lora_train":
            s["dy"] = randn(c["t"], c["o"], dtype=dt, std=0.1)
            s["base_grad"] = randn(c["t"], c["k"], dtype=dt, std=0.1)
        return s
    if c["op"] == "moe":
        dt = _DT[c["dtype"]]
        e, h, f = c["e"], c["h"], c["f"]
        s = {"case": c, "x": randn(c["t"], h, dtype=dt), "logits": randn(c["t"], e, dtype=torch.float32, std=1.5)}
        for name, shape, std in (("fc1", (2 * f, h), h ** -0.5), ("fc2", (h, f), f ** -0.5)):
            fp8 = c["weights"] == "fp8"
            w = torch.empty(e, *shape, dtype=torch.float8_e4m3fn if fp8 else dt, device="cuda")
            scale_inv = torch.ones(e, dtype=torch.float32, device="cuda")
            for i in range(e):
                wi = torch.randn(*shape, generator=g, device="cuda").mul_(std)
                if fp8:
                    scale_inv[i] = wi.abs().max() / 448
                    wi.div_(scale_inv[i])
                w[i] = wi.to(w.dtype)
            s[name], s[name + "_scale_inv"] = w, scale_inv if fp8 else None
        return s
    dt = _DT[c["dtype"]]
    lengths = _lengths(c)
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + (n + 63) // 64 * 64)
    flat = torch.empty(starts[-1], dtype=dt, device="cuda")
    flat.normal_(generator=g)
    flat.mul_(0.02)
    out = torch.zeros(starts[-1], dtype=dt if c["out"] == "same" else _DT[c["out"]], device="cuda")
    return {"case": c, "grads": [flat[i:i + n] for i, n in zip(starts, lengths)],
            "outs": [out[i:i + n] for i, n in zip(starts, lengths)], "out": out, "max_norm": 1.0}


# ------------------------------------------------------------------------------------------------ one pass
def _own_lora(s):
    from transformer_engine_amd.lora import lora_backward, lora_forward
    train = "dy" in s
    y, saved = lora_forward(s["x"], s["a"], s["b"], s["ids"], scaling=s["scaling"], base=s["base"], needs_backward=train)
    if not train:
        return y
    return (y, *lora_backward(s["dy"], saved, base_grad=s["base_grad"]))


def _own_moe(s):
    from transformer_engine_amd.moe import moe_forward, moe_topk
    ids, weights = moe_topk(s["logits"], s["case"]["topk"], renormalize=True)
    out = moe_forward(s["x"], s["fc1"], s["fc2"], ids, weights, fc1_scale_inv=s["fc1_scale_inv"],
                      fc2_scale_inv=s["fc2_scale_inv"])
    return ids, weights, out


def _own_clip(s):
    from transformer_engine_amd.weight_update import clip_grad_norm
    return clip_grad_norm(s["grads"], s["max_norm"], outs=s["outs"]), s["out"]


def _plain_lora(s):
    """All adapters' rank vectors of all tokens in two dense products, those of other tokens' adapters set to zero."""
    x, a, b, ids = s["x"].float(), s["a"].float(), s["b"].float(), s["ids"]
    n, r, k = a.shape
    o = b.shape[1]
    pick = ((ids[:, None] == torch.arange(n, device=ids.device)) * s["scaling"])[:, :, None]
    a2, b2 = a.reshape(n * r, k), b.permute(1, 0, 2).reshape(o, n * r)
    v = ((x @ a2.t()).view(-1, n, r) * pick).view(-1, n * r)
    y = (s["base"].float() + v @ b2.t()).to(s["x"].dtype)
    if "dy" not in s:
        return y
    dy = s["dy"].float()
    u = ((dy @ b2).view(-1, n, r) * pick).view(-1, n * r)
    dx = (s["base_grad"].float() + u @ a2).to(s["x"].dtype)
    da = (u.t() @ x).view(n, r, k).to(s["a"].dtype)
    db = (dy.t() @ v).view(o, n, r).permute(1, 0, 2).contiguous().to(s["b"].dtype)
    return y, dx, da, db


def _weights(s, name, at=None):
    w, scale_inv = s[name], s[name + "_scale_inv"]
    if at is not None:
        w = (w.view(torch.uint8)[at]).view(w.dtype) if scale_inv is not None else w[at]
        scale_inv = None if scale_inv is None else scale_inv[at]
    w = w.float()
    return w if scale_inv is None else w * scale_inv.view(*scale_inv.shape, 1, 1)


def _plain_moe(s):
    c, x = s["case"], s["x"].float()
    t, h, f, e = c["t"], c["h"], c["f"], c["e"]
    p = torch.softmax(s["logits"], dim=-1)
    ids = s["logits"].sort(dim=-1, descending=True, stable=True).indices[:, :c["topk"]]
    weights = p.gather(1, ids)
    weights = weights / weights.sum(-1, keepdim=True)
    if t * c["topk"] < e:  # the chosen experts' weights, one copy per token and choice
        z = torch.matmul(_weights(s, "fc1", ids), x[:, None, :, None])[..., 0]
        z = torch.sigmoid(z[..., :f]) * z[..., :f] * z[..., f:]
        y = torch.matmul(_weights(s, "fc2", ids), z[..., None])[..., 0]
        out = (y * weights[..., None]).sum(1)
    else:                  # every expert on every token, weighted by zero where it was not chosen
        z = (x @ _weights(s, "fc1").view(e * 2 * f, h).t()).view(t, e, 2 * f)
        z = torch.sigmoid(z[..., :f]) * z[..., :f] * z[..., f:]
        gate = torch.zeros(t, e, device=x.device).scatter_(1, ids, weights)
        z = (z * gate[..., None]).view(t, e * f)
        out = z @ _weights(s, "fc2").permute(0, 2, 1).reshape(e * f, h)
    return ids.to(torch.int32), weights, out.to(s["x"].dtype)


def _plain_clip(s):
    total = torch.stack([g.double().square().sum() for g in s["grads"]]).sum()
    norm = total.sqrt()
    factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    for g, o in zip(s["grads"], s["outs"]):
        o.copy_(g.float() * factor.float())
    return norm.float().view(1), s["out"]


def run(state):
    op = state["case"]["op"]
    if op in ("lora", "lora_train"):
        return _own_lora(state) if own else _plain_lora(state)
    if op == "moe":
        return _own_moe(state) if own else _plain_moe(state)
    return _own_clip(state) if own else _plain_clip(state)


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    c = case
    if c["op"] in ("lora", "lora_train"):
        t, k, o, r = c["t"], c["k"], c["o"], c["r"]
        used = min(c["n"], t)
        pools = used * r * (k + o)
        fwd = 2 * (t * k + pools + 2 * t * o) + 4 * t
        flops = 2 * t * r * (k + o)
        if c["op"] == "lora":
            return {"bytes": fwd, "flops": flops}
        # x once for both directions; dy, the shared projection's gradient, dx, and the adapters' gradients
        return {"bytes": fwd + 2 * (t * o + 2 * t * k + pools), "flops": 3 * flops}
    if c["op"] == "moe":
        t, h, f, e, k = c["t"], c["h"], c["f"], c["e"], c["topk"]
        hit = e * (1 - (1 - k / e) ** t)  # expected number of experts that some token chose
        return {"bytes": hit * 3 * f * h * (1 if c["weights"] == "fp8" else 2) + 4 * t * h + 4 * t * e,
                "flops": 6 * t * k * f * h}
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    n = sum(_lengths(c))
    return {"bytes": n * (size[c["dtype"]] + size[c["dtype"] if c["out"] == "same" else c["out"]]), "flops": 3 * n}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] in ("lora", "lora_train"):
        train = c["op"] == "lora_train"
        y = s["base"].double()
        if train:
            dx = s["base_grad"].double()
            da, db = torch.zeros(s["a"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["b"].shape, dtype=torch.float64, device="cuda")
        for i in range(c["n"]):
            rows = (s["ids"] == i).nonzero()[:, 0]
            if rows.numel() == 0:
                continue
            x, a, b = s["x"][rows].double(), s["a"][i].double(), s["b"][i].double()
            scale = s["scaling"][i].double()
            v = x @ a.t()
            y[rows] += scale * (v @ b.t())
            if train:
                dy = s["dy"][rows].double()
                u = scale * (dy @ b)
                dx[rows] += u @ a
                da[i] = u.t() @ x
                db[i] = scale * (dy.t() @ v)
        return (y, dx, da, db) if train else y
    if c["op"] == "moe":
        logits = s["logits"].double()
        order = torch.argsort(-logits, dim=-1, stable=True)[:, :c["topk"]]
        z = torch.exp(logits - logits.max(-1, keepdim=True).values)
        w = z.gather(1, order)
        w = w / w.sum(-1, keepdim=True)
        x, f = s["x"].double(), c["f"]
        out = torch.zeros_like(x)
        for i in range(c["e"]):
            row, col = (order == i).nonzero(as_tuple=True)
            if row.numel() == 0:
                continue
            w1, w2 = s["fc1"][i].double(), s["fc2"][i].double()
            if s["fc1_scale_inv"] is not None:
                w1, w2 = w1 * s["fc1_scale_inv"][i].double(), w2 * s["fc2_scale_inv"][i].double()
            gate, up = x[row] @ w1[:f].t(), x[row] @ w1[f:].t()
            out[row] += w[row, col][:, None] * ((gate / (1 + torch.exp(-gate)) * up) @ w2.t())
        return order.to(torch.int32), w, out
    total = 0.0
    for g in s["grads"]:
        total = total + torch.dot(g.double(), g.double())
    norm = torch.sqrt(total)
    factor = min(1.0, s["max_norm"] / (norm.item() + 1e-6))
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for g in s["grads"]:
        out[start:start + g.numel()] = g.double() * factor
        start += (g.numel() + 63) // 64 * 64
    return norm.view(1), out
