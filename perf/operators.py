"""Cases of the training-block operators: dropout, block norms and bucketed-bias softmax, with their gradients.

``run`` computes a case in plain torch (32-bit arithmetic, rounded once at the end) or, with ``own`` set, through
ask_b200 plans.  ``exact`` gives the same outputs from the definitions in 64 bits.

The dropout generator is Philox4x32-10 (Salmon, Moraes, Dror and Shaw, SC'11): element i takes word i % 4 of the
block with counter (lo(offset + i/4), hi(offset + i/4), stream, 1) under key (lo(seed), hi(seed)) and is kept when
that word is at least floor(p * 2^32); a kept element is scaled by 1 / (1 - p).
"""
import json
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
MASK32 = 0xFFFFFFFF


# ---- the cases --------------------------------------------------------------------------
def _dropout(name, dtype, count, p, residual):
    return {"name": name, "op": "dropout", "dtype": dtype, "count": count, "p": p, "residual": residual}


def _norm(name, op, dtype, rows, cols, norm="rms", branch=True, post=True, pre=True, bias=False, groups=0, alpha=1.0,
          p=0.0, params="f32"):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "cols": cols, "norm": norm, "branch": branch,
            "post": post, "pre": pre, "bias": bias, "groups": groups, "alpha": alpha, "p": p, "params": params}


def _softmax(name, op, dtype, batch, heads, queries, keys, buckets=32, distance=128, both=True, scale=1.0, causal=False,
             lengths=False, offsets=False, p=0.0, table="f32"):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "heads": heads, "queries": queries, "keys": keys,
            "buckets": buckets, "distance": distance, "both": both, "scale": scale, "causal": causal,
            "lengths": lengths, "offsets": offsets, "p": p, "table": table}


def listed():
    return [
        # fine-tuning with one short sequence: the call's latency is the time
        _dropout("dropout_small", "bf16", 16 * 1024, 0.1, False),
        # a residual stream in f32 whose size is no multiple of a vector, at a higher rate
        _dropout("dropout_residual_odd", "f32", 17_000_051, 0.25, True),
        # the activations of a training step, [32768, 4096]
        _dropout("dropout_train", "bf16", 32768 * 4096, 0.1, False),
        # serving: the norms between two blocks for a batch of eight single tokens
        _norm("norm_decode", "norm", "bf16", 8, 4096, groups=1, params="bf16"),
        # training: both norms, a gate for each of eight samples, dropout on the branch
        _norm("norm_train", "norm", "bf16", 32768, 4096, groups=8, p=0.1),
        # layer norms with biases of an odd width in f32, a scaled residual and no gate
        _norm("norm_layer_odd", "norm", "f32", 5003, 1023, norm="layer", bias=True, alpha=1.5),
        _norm("norm_grad_train", "norm_grad", "bf16", 32768, 4096, groups=8, p=0.1),
        # a prompt's worth of rows, layer norms with biases and one gate for all rows
        _norm("norm_grad_layer", "norm_grad", "f16", 4099, 1000, norm="layer", bias=True, groups=1, alpha=0.5),
        # serving: one token for each of 64 sequences against ragged caches of up to 4096 keys
        _softmax("softmax_decode", "softmax", "f16", 64, 32, 1, 4096, both=False, lengths=True, offsets=True),
        # an encoder layer in training: padded batch, dropout on the probabilities
        _softmax("softmax_train", "softmax", "bf16", 8, 16, 1024, 1024, lengths=True, p=0.1),
        _softmax("softmax_grad_train", "softmax_grad", "bf16", 8, 16, 1024, 1024, lengths=True, p=0.1),
        # a decoder layer in f32 with an odd length and scaled scores
        _softmax("softmax_grad_causal_odd", "softmax_grad", "f32", 3, 12, 1021, 1021, both=False, scale=0.125,
                 causal=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["dropout", "norm", "norm_grad", "softmax", "softmax_grad"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    most = 1 << (25 if dtype == "f32" else 26)
    rate = round(rng.uniform(0.05, 0.5), 3)
    if op == "dropout":
        case = _dropout("", dtype, _log(rng, 1000, most), rate, rng.random() < 0.5)
    elif op in ("norm", "norm_grad"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            cols = (cols + 7) // 8 * 8
        rows = _log(rng, 1, min(32768, most // cols))
        divisors = [g for g in (1, 2, 4, 8) if rows % g == 0]
        branch = rng.random() < 0.85
        post, pre = branch and rng.random() < 0.8, not branch or rng.random() < 0.8
        layer = rng.random() < 0.5
        case = _norm("", op, dtype, rows, cols, norm="layer" if layer else "rms", branch=branch, post=post, pre=pre,
                     bias=layer and (post or pre), groups=rng.choice([0] + divisors) if branch else 0,
                     alpha=rng.choice([1.0, round(rng.uniform(0.5, 3.0), 2)]) if branch else 1.0,
                     p=rate if branch and rng.random() < 0.5 else 0.0, params=rng.choice(["f32", dtype]))
    else:
        both, buckets = rng.random() < 0.6, rng.choice([16, 32, 64])
        common = dict(buckets=buckets, distance=rng.choice([64, 128, 200, 512]), both=both,
                      scale=rng.choice([1.0, 0.125, 0.0884]), table=rng.choice(["f32", dtype]))
        if op == "softmax" and rng.random() < 0.4:  # single tokens
            keys = _log(rng, 16, 65536)
            heads = rng.randint(1, 40)
            batch = _log(rng, 1, max(1, min(128, most // (keys * heads))))
            case = _softmax("", op, dtype, batch, heads, 1, keys, lengths=True, offsets=True,
                            **dict(common, both=False))
        else:
            queries = _log(rng, 2, 2048)
            keys = queries if rng.random() < 0.7 else _log(rng, 2, 4096)
            heads = max(1, min(rng.randint(1, 32), most // (queries * keys)))
            batch = max(1, min(_log(rng, 1, 16), most // (queries * keys * heads)))
            case = _softmax("", op, dtype, batch, heads, queries, keys, causal=not both and rng.random() < 0.7,
                            lengths=rng.random() < 0.5, p=rate if rng.random() < 0.5 else 0.0, **common)
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------------
def _lengths(case):
    """Keys in use for each sequence: between half of the keys and all of them, and an empty slot in a batch of four or more."""
    b, k = case["batch"], case["keys"]
    lens = [k - (i * k) // (2 * b) for i in range(b)]
    if b >= 4:
        lens[-1] = 0
    return lens


def _bucket_thresholds(case):
    """Distances at which the bucket index grows by one: single distances up to half of a side's buckets, then steps
    growing geometrically to `distance`, found in whole numbers."""
    side = case["buckets"] // 2 if case["both"] else case["buckets"]
    exact_ones = side // 2
    steps = side - exact_ones
    thresholds = list(range(1, exact_ones + 1))
    n = exact_ones
    for j in range(1, steps):  # least n with (n / exact)^steps >= (distance / exact)^j
        while n**steps * exact_ones**j < case["distance"]**j * exact_ones**steps:
            n += 1
        thresholds.append(n)
    return thresholds


def _elements(case):
    if case["op"] == "dropout":
        return case["count"]
    if case["op"].startswith("norm"):
        return case["rows"] * case["cols"]
    return case["batch"] * case["heads"] * case["queries"] * case["keys"]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, dtype=dt, mean=0.0, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    def empty(*shape, dtype=dt):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    op, f32 = case["op"], torch.float32
    s = {"case": case, "in": {}, "out": {}}
    i, o = s["in"], s["out"]
    if op == "dropout":
        i["x"] = normal(case["count"])
        if case["residual"]:
            i["residual"] = normal(case["count"], std=2.0)
        o["y"] = empty(case["count"])
    elif op.startswith("norm"):
        rows, cols, layer = case["rows"], case["cols"], case["norm"] == "layer"
        pt = TYPES[case["params"]]

        def stats(v):  # what the forward pass saves: (mean,) 1 / sqrt(variance + eps)
            v = v.float()
            mean = v.mean(1, keepdim=True) if layer else 0.0
            rstd = torch.rsqrt((v - mean).square().mean(1, keepdim=True) + 1e-6)
            return torch.cat([mean, rstd], 1) if layer else rstd

        grad = op == "norm_grad"
        h = normal(rows, cols, mean=0.1, std=2.0)
        y = normal(rows, cols, mean=-0.2, std=0.7) if case["branch"] else None
        if grad:
            if case["branch"]:
                i["dh"] = normal(rows, cols, std=0.1)
            if case["pre"]:
                i["du"] = normal(rows, cols, std=0.1)
                i["h"] = h
            if case["post"] or case["groups"]:
                i["y"] = y
        else:
            i["x"] = h
            if case["branch"]:
                i["y"] = y
        if case["post"]:
            i["w_post"] = normal(cols, dtype=pt, mean=1.0, std=0.2)
            if case["bias"]:
                i["b_post"] = normal(cols, dtype=pt, std=0.2)
        if case["groups"]:
            i["gate"] = normal(case["groups"], cols, dtype=pt, mean=0.5, std=0.3)
        if case["pre"]:
            i["w_pre"] = normal(cols, dtype=pt, mean=1.0, std=0.2)
            if case["bias"]:
                i["b_pre"] = normal(cols, dtype=pt, std=0.2)
        width = 2 if layer else 1
        if grad:
            if case["bias"]:
                i.pop("b_pre", None)  # the gradient does not depend on it
                if not case["groups"]:
                    i.pop("b_post", None)
            if case["post"]:
                i["stats_post"] = stats(y)
            if case["pre"]:
                i["stats_pre"] = stats(h)
            o["dx"] = empty(rows, cols)
            if case["branch"]:
                o["dy"] = empty(rows, cols)
            if case["post"]:
                o["dw_post"] = empty(cols, dtype=f32)
                if case["bias"]:
                    o["db_post"] = empty(cols, dtype=f32)
            if case["groups"]:
                o["dgate"] = empty(case["groups"], cols, dtype=f32)
            if case["pre"]:
                o["dw_pre"] = empty(cols, dtype=f32)
                if case["bias"]:
                    o["db_pre"] = empty(cols, dtype=f32)
        else:
            if case["branch"]:
                o["h"] = empty(rows, cols)
            if case["pre"]:
                o["u"] = empty(rows, cols)
            if case["post"]:
                o["stats_post"] = empty(rows, width, dtype=f32)
            if case["pre"]:
                o["stats_pre"] = empty(rows, width, dtype=f32)
    else:
        b, h, q, k = case["batch"], case["heads"], case["queries"], case["keys"]
        i["s"] = normal(b, h, q, k, std=2.0 / case["scale"])
        i["table"] = normal(case["buckets"], h, dtype=TYPES[case["table"]])
        if case["lengths"]:
            lens = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
            i["lengths"] = lens[torch.randperm(b, generator=g, device="cuda")].contiguous()
        if case["offsets"]:
            i["offsets"] = (i["lengths"] - 1).contiguous()
        if op == "softmax":
            o["p"] = empty(b, h, q, k)
            o["lse"] = empty(b, h, q, dtype=f32)
        else:
            s["in"]["lse"] = _lse(case, i)
            i["dp"] = normal(b, h, q, k, std=0.1)
            o["ds"] = empty(b, h, q, k)
            o["dtable"] = empty(case["buckets"], h, dtype=f32)
    if case["p"]:
        i["seed"] = torch.tensor([seed * 0x9E3779B97F4A7C15 % (1 << 62), seed * 1000003], dtype=torch.int64,
                                 device="cuda")
    return s


# ---- the plain forms ----------------------------------------------------------------------
def _mulhilo(a, m):
    """High and low words of the 64-bit product of 32-bit words held in int64 (the product's bits survive the wrap)."""
    v = a * m
    return (v >> 32) & MASK32, v & MASK32


def _keep(case, seed):
    """Which elements are kept, as 0 or 1 / (1 - p) in 32 bits."""
    n = _elements(case)
    block = torch.arange((n + 3) // 4, device="cuda") + seed[1]
    k0, k1 = seed[0] & MASK32, (seed[0] >> 32) & MASK32
    c0, c1 = block & MASK32, (block >> 32) & MASK32
    c2, c3 = torch.zeros_like(c0), torch.ones_like(c0)
    for r in range(10):  # the generator's rounds
        h0, l0 = _mulhilo(c0, 0xD2511F53)
        h1, l1 = _mulhilo(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ ((k0 + r * 0x9E3779B9) & MASK32), l1, h0 ^ c3 ^ ((k1 + r * 0xBB67AE85) & MASK32), l0
    words = torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]
    return (words >= int(case["p"] * 4294967296.0)).float() * (1.0 / (1.0 - case["p"]))


def _dropped(case, i, v):
    return v * _keep(case, i["seed"]).view(v.shape) if case["p"] else v


def _group_rows(case, gate):
    """The gate of each row's group, [rows, cols]."""
    return gate.float().repeat_interleave(case["rows"] // case["groups"], 0)


def _plain_norm(case, i):
    layer = case["norm"] == "layer"
    out = {}

    def normed(v, w, b):
        mean = v.mean(1, keepdim=True) if layer else 0.0
        rstd = torch.rsqrt((v - mean).square().mean(1, keepdim=True) + 1e-6)
        n = (v - mean) * rstd * w.float()
        return n + b.float() if b is not None else n, torch.cat([mean, rstd], 1) if layer else rstd

    h = i["x"].float()
    if case["branch"]:
        n = i["y"].float()
        if case["post"]:
            n, out["stats_post"] = normed(n, i["w_post"], i.get("b_post"))
        if case["groups"]:
            n = n * _group_rows(case, i["gate"])
        h = case["alpha"] * h + _dropped(case, i, n)
        out["h"] = h.to(i["x"].dtype)
    if case["pre"]:
        u, out["stats_pre"] = normed(h, i["w_pre"], i.get("b_pre"))
        out["u"] = u.to(i["x"].dtype)
    return out


def _plain_norm_grad(case, i):
    layer = case["norm"] == "layer"
    out = {}

    def hat(v, stats):
        return (v.float() - stats[:, :1]) * stats[:, 1:] if layer else v.float() * stats

    def through(a, xhat, stats):  # the norm's gradient to its input, `a` the gradient to xhat
        rstd = stats[:, 1:] if layer else stats
        mean = a.mean(1, keepdim=True) if layer else 0.0
        return rstd * (a - mean - xhat * (a * xhat).mean(1, keepdim=True))

    dt = (i["dh"] if case["branch"] else i["du"]).dtype
    grad = i["dh"].float() if case["branch"] else 0.0
    if case["pre"]:
        xhat, du = hat(i["h"], i["stats_pre"]), i["du"].float()
        grad = grad + through(du * i["w_pre"].float(), xhat, i["stats_pre"])
        out["dw_pre"] = (du * xhat).sum(0)
        if case["bias"]:
            out["db_pre"] = du.sum(0)
    out["dx"] = ((case["alpha"] if case["branch"] else 1.0) * grad).to(dt)
    if case["branch"]:
        d = _dropped(case, i, grad)
        if case["post"]:
            yhat = hat(i["y"], i["stats_post"])
        if case["groups"]:
            n = i["y"].float()
            if case["post"]:
                n = yhat * i["w_post"].float()
                n = n + i["b_post"].float() if case["bias"] else n
            out["dgate"] = (d * n).view(case["groups"], -1, case["cols"]).sum(1)
            d = d * _group_rows(case, i["gate"])
        if case["post"]:
            out["dw_post"] = (d * yhat).sum(0)
            if case["bias"]:
                out["db_post"] = d.sum(0)
            d = through(d * i["w_post"].float(), yhat, i["stats_post"])
        out["dy"] = d.to(dt)
    return out


def _relative(case, i):
    """Key position minus query position, [batch or 1, queries, keys]."""
    rel = torch.arange(case["keys"], device="cuda")[None, :] - torch.arange(case["queries"], device="cuda")[:, None]
    return rel[None] - i["offsets"].long()[:, None, None] if case["offsets"] else rel[None]


def _buckets(case, rel):
    side = case["buckets"] // 2 if case["both"] else case["buckets"]
    n = rel.abs() if case["both"] else (-rel).clamp(min=0)
    thresholds = torch.tensor(_bucket_thresholds(case), device="cuda")
    by_distance = (torch.arange(case["distance"] + 1, device="cuda")[:, None] >= thresholds).sum(1)
    b = by_distance[n.clamp(max=case["distance"])]
    return b + side * (rel > 0) if case["both"] else b


def _logits(case, i):
    """scale * s + bias, with -inf where a key is masked."""
    rel = _relative(case, i)
    bias = i["table"].float()[_buckets(case, rel)].permute(0, 3, 1, 2)
    logits = i["s"].float() * case["scale"] + bias
    if case["causal"]:
        logits = logits.masked_fill((rel > 0)[:, None], -math.inf)
    if case["lengths"]:
        past = torch.arange(case["keys"], device="cuda") >= i["lengths"].long()[:, None]
        logits = logits.masked_fill(past[:, None, None, :], -math.inf)
    return logits


def _lse(case, i):
    logits = _logits(case, i)
    top = logits.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    return ((logits - top).exp().sum(3).log() + top[..., 0]).contiguous()


def _plain_softmax(case, i):
    logits = _logits(case, i)
    top = logits.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    e = (logits - top).exp()
    total = e.sum(3, keepdim=True)
    p = torch.where(total > 0, e / total, 0.0)
    return {"p": _dropped(case, i, p).to(i["s"].dtype), "lse": (total.log() + top)[..., 0]}


def _plain_softmax_grad(case, i):
    logits = _logits(case, i)
    p = torch.where(logits == -math.inf, 0.0, (logits - i["lse"][..., None]).exp())
    d = _dropped(case, i, i["dp"].float())
    dl = p * (d - (p * d).sum(3, keepdim=True))
    buckets = _buckets(case, _relative(case, i))[:, None]
    by_place = dl.sum(0, keepdim=True) if buckets.shape[0] == 1 else dl
    dtable = torch.stack([torch.where(buckets == b, by_place, 0.0).sum((0, 2, 3)) for b in range(case["buckets"])])
    return {"ds": (dl * case["scale"]).to(i["s"].dtype), "dtable": dtable}


def run(state):
    if own:
        return _run_own(state)
    case, i = state["case"], state["in"]
    if case["op"] == "dropout":
        y = _dropped(case, i, i["x"].float())
        return {"y": (y + i["residual"].float() if case["residual"] else y).to(i["x"].dtype)}
    return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "softmax": _plain_softmax,
            "softmax_grad": _plain_softmax_grad}[case["op"]](case, i)


# ---- the framework's calls -------------------------------------------------------------------
_plans = {}  # a program keeps the plans of the steps that it runs


def _recipe(case):
    from ask_b200 import recipes as R

    op = case["op"]
    if op == "dropout":
        return R.dropout(case["dtype"], case["count"], case["p"], residual=case["residual"])
    if op.startswith("norm"):
        make = R.block_norm if op == "norm" else R.block_norm_grad
        return make(case["dtype"], case["rows"], case["cols"], norm=case["norm"], eps=1e-6, branch=case["branch"],
                    post=case["post"], pre=case["pre"], bias=case["bias"], gate_groups=case["groups"],
                    residual_scale=case["alpha"], dropout=case["p"], param_dtype=case["params"])
    make = R.bias_softmax if op == "softmax" else R.bias_softmax_grad
    thresholds = R.bucket_thresholds(case["buckets"], case["distance"], case["both"])
    return make(case["dtype"], case["batch"], case["heads"], case["queries"], case["keys"], thresholds,
                bidirectional=case["both"], scale=case["scale"], causal=case["causal"], lengths=case["lengths"],
                offsets=case["offsets"], dropout=case["p"], table_dtype=case["table"])


#: Ports in the plans' order; a case has those that its inputs and outputs name.
_INPUTS = {"dropout": ["x", "residual", "seed"],
           "norm": ["x", "y", "w_post", "b_post", "gate", "w_pre", "b_pre", "seed"],
           "norm_grad": ["dh", "du", "h", "y", "w_post", "b_post", "gate", "w_pre", "stats_post", "stats_pre", "seed"],
           "softmax": ["s", "table", "lengths", "offsets", "seed"],
           "softmax_grad": ["s", "dp", "lse", "table", "lengths", "offsets", "seed"]}
_OUTPUTS = {"dropout": ["y"], "norm": ["h", "u", "stats_post", "stats_pre"],
            "norm_grad": ["dx", "dy", "dw_post", "db_post", "dgate", "dw_pre", "db_pre"],
            "softmax": ["p", "lse"], "softmax_grad": ["ds", "dtable"]}


def _run_own(state):
    call = state.get("call")
    if call is None:
        import ask_b200

        case = state["case"]
        key = json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True)
        plan = _plans.get(key)
        if plan is None:
            plan = _plans[key] = ask_b200.Plan(_recipe(case), device=torch.cuda.current_device())
        if plan.scratch_bytes:
            state["scratch"] = torch.empty(plan.scratch_bytes, dtype=torch.uint8, device="cuda")
        call = state["call"] = plan.bind([state["in"][n] for n in _INPUTS[case["op"]] if n in state["in"]],
                                         [state["out"][n] for n in _OUTPUTS[case["op"]] if n in state["out"]],
                                         state.get("scratch"), torch.cuda.current_stream())
    call()
    return state["out"]


# ---- what a pass cannot do without --------------------------------------------------------------
def work(case):
    n, e, op = _elements(case), SIZE[case["dtype"]], case["op"]
    if op == "dropout":
        return {"bytes": n * e * (3 if case["residual"] else 2), "flops": n * 2}
    if op.startswith("norm"):
        rows, cols, pe = case["rows"], case["cols"], SIZE[case["params"]]
        branch, post, pre, gated = case["branch"], case["post"], case["pre"], bool(case["groups"])
        stats = (post + pre) * rows * 4 * (2 if case["norm"] == "layer" else 1)
        params = cols * ((post + pre) * (2 if case["bias"] else 1) + case["groups"])
        if op == "norm":
            return {"bytes": n * e * (1 + 2 * branch + pre) + stats + params * pe, "flops": n * (6 * post + 6 * pre + 4)}
        arrays = branch + 2 * pre + (post or gated) + 1 + branch
        return {"bytes": n * e * arrays + stats + params * (pe + 4), "flops": n * (10 * post + 10 * pre + 4)}
    used = n
    per_head = case["heads"]
    if case["lengths"] or case["causal"]:
        q, lens = case["queries"], _lengths(case) if case["lengths"] else [case["keys"]] * case["batch"]
        # a causal query i sees min(i + 1, length) keys
        used = per_head * sum((min(q, ln) * (min(q, ln) + 1) // 2 + max(0, q - ln) * ln) if case["causal"] else q * ln
                              for ln in lens)
    rows = case["batch"] * per_head * case["queries"]
    small = case["buckets"] * per_head * SIZE[case["table"]] + rows * 4
    if op == "softmax":
        return {"bytes": used * e + n * e + small, "flops": used * 6}
    return {"bytes": 2 * used * e + n * e + small + case["buckets"] * per_head * 4, "flops": used * 9}


# ---- the definitions in 64 bits --------------------------------------------------------------------
def _words64(blocks, key, stream):
    """Philox words of the blocks, [blocks, 4], by 16-bit halves: no product leaves 48 bits."""
    def product(m, v):
        low, high = (m & 0xFFFF) * v, (m >> 16) * v
        total_low = low + ((high & 0xFFFF) << 16)
        return (high >> 16) + (total_low >> 32), total_low % (1 << 32)

    x = [blocks % (1 << 32), (blocks >> 32) % (1 << 32), torch.full_like(blocks, stream), torch.full_like(blocks, 1)]
    ka, kb = key % (1 << 32), (key >> 32) % (1 << 32)
    for _ in range(10):
        (ha, la), (hb, lb) = product(0xD2511F53, x[0]), product(0xCD9E8D57, x[2])
        x = [hb ^ x[1] ^ ka, lb, ha ^ x[3] ^ kb, la]
        ka, kb = (ka + 0x9E3779B9) % (1 << 32), (kb + 0xBB67AE85) % (1 << 32)
    return torch.stack(x, dim=-1)


def _factors64(case, i, shape):
    if not case["p"]:
        return 1.0
    n = _elements(case)
    seed, offset = i["seed"].tolist()
    kept = _words64(torch.arange(offset, offset + -(-n // 4), device="cuda"), seed, 0).flatten()[:n]
    kept = kept >= math.floor(case["p"] * 2**32)
    return torch.where(kept, 1.0 / (1.0 - case["p"]), torch.zeros((), dtype=torch.float64, device="cuda")).view(shape)


def _exact_norm(case, i):
    f64, layer = torch.float64, case["norm"] == "layer"

    def moments(v):
        mu = v.sum(1) / case["cols"] if layer else torch.zeros(case["rows"], dtype=f64, device="cuda")
        var = (v * v).sum(1) / case["cols"] - mu * mu
        return mu, 1.0 / (var + 1e-6).sqrt()

    def affine(v, mu, r, w, b):
        z = torch.einsum("rc,r,c->rc", v - mu[:, None], r, i[w].to(f64))
        return z + i[b].to(f64) if b in i else z

    out, h = {}, i["x"].to(f64)
    if case["branch"]:
        z = i["y"].to(f64)
        if case["post"]:
            mu, r = moments(z)
            out["stats_post"] = torch.stack([mu, r], 1) if layer else r[:, None]
            z = affine(z, mu, r, "w_post", "b_post")
        if case["groups"]:
            z = (z.view(case["groups"], -1, case["cols"]) * i["gate"].to(f64)[:, None]).view(z.shape)
        h = h * case["alpha"] + z * _factors64(case, i, z.shape)
        out["h"] = h
    if case["pre"]:
        mu, r = moments(h)
        out["stats_pre"] = torch.stack([mu, r], 1) if layer else r[:, None]
        out["u"] = affine(h, mu, r, "w_pre", "b_pre")
    return out


def _exact_norm_grad(case, i):
    f64, layer, n = torch.float64, case["norm"] == "layer", case["cols"]
    shape = (case["rows"], n)

    def split(v, stats):
        mu = stats[:, 0].to(f64)[:, None] if layer else 0.0
        r = stats[:, -1].to(f64)[:, None]
        return (v.to(f64) - mu) * r, r

    def back(a, z, r):  # sum over columns of (identity - 1/n [- z z^T / n]) a
        t = a - z * (torch.einsum("rc,rc->r", a, z) / n)[:, None]
        return r * (t - (a.sum(1) / n)[:, None] if layer else t)

    out = {}
    g = i["dh"].to(f64) if case["branch"] else torch.zeros(shape, dtype=f64, device="cuda")
    if case["pre"]:
        du = i["du"].to(f64)
        z, r = split(i["h"], i["stats_pre"])
        out["dw_pre"] = torch.einsum("rc,rc->c", du, z)
        if case["bias"]:
            out["db_pre"] = du.sum(0)
        g = g + back(du * i["w_pre"].to(f64), z, r)
        del z, du
    out["dx"] = g * (case["alpha"] if case["branch"] else 1.0)
    if case["branch"]:
        g = g * _factors64(case, i, shape)
        gate = i["gate"].to(f64)[:, None] if case["groups"] else None
        folded = (case["groups"], -1, n)
        w = i["w_post"].to(f64) if case["post"] else 1.0
        z, r = split(i["y"], i["stats_post"]) if case["post"] else (i["y"].to(f64), 1.0) if case["groups"] else (0, 1.0)
        if case["groups"]:
            b = i["b_post"].to(f64) if "b_post" in i else 0.0
            out["dgate"] = torch.einsum("grc,grc->gc", g.view(folded), (z * w + b).view(folded))
            g = (g.view(folded) * gate).view(shape)
        if case["post"]:
            out["dw_post"] = torch.einsum("rc,rc->c", g, z)
            if case["bias"]:
                out["db_post"] = g.sum(0)
            g = back(g * w, z, r)
        out["dy"] = g
    return out


def _exact_softmax(case, i):
    f64 = torch.float64
    b, h, q, k = case["batch"], case["heads"], case["queries"], case["keys"]
    thresholds, side = _bucket_thresholds(case), case["buckets"] // (2 if case["both"] else 1)
    grad = case["op"] == "softmax_grad"
    factors = _factors64(case, i, (b, h, q, k))
    out = {n: [] for n in (("ds",) if grad else ("p", "lse"))}
    dtable = torch.zeros(case["buckets"], h, dtype=f64, device="cuda")
    key = torch.arange(k, device="cuda").expand(q, k)
    for j in range(b):
        place = torch.arange(q, device="cuda")[:, None] + (int(i["offsets"][j]) if case["offsets"] else 0)
        dist = place - key  # how far the key lies behind the query
        far = dist.abs() if case["both"] else dist.clamp(min=0)
        bucket = torch.bucketize(far, torch.tensor(thresholds, device="cuda"), right=True)
        if case["both"]:
            bucket = torch.where(dist < 0, bucket + side, bucket)
        seen = key < (int(i["lengths"][j]) if case["lengths"] else k)
        if case["causal"]:
            seen = seen & (dist >= 0)
        logits = i["s"][j].to(f64) * case["scale"] + i["table"].to(f64).t()[:, bucket]
        logits = torch.where(seen, logits, -math.inf)
        f = factors[j] if case["p"] else 1.0
        if not grad:
            lse = torch.logsumexp(logits, 2)
            out["lse"].append(lse)
            out["p"].append(torch.where(seen, (logits - lse[..., None]).exp(), 0.0) * f)
            continue
        p = torch.where(seen, (logits - i["lse"][j].to(f64)[..., None]).exp(), 0.0)
        d = i["dp"][j].to(f64) * f
        dl = p * d - p * torch.einsum("hqk,hqk->hq", p, d)[..., None]
        out["ds"].append(dl * case["scale"])
        for head in range(h):
            dtable[:, head] += torch.bincount(bucket.flatten(), weights=dl[head].flatten(), minlength=case["buckets"])
    out = {n: torch.stack(v) for n, v in out.items()}
    if grad:
        out["dtable"] = dtable
    return out


def exact(case, seed):
    i = prepare(case, seed)["in"]
    if case["op"] == "dropout":
        y = i["x"].double() * _factors64(case, i, i["x"].shape)
        return {"y": y + i["residual"].double() if case["residual"] else y}
    return {"norm": _exact_norm, "norm_grad": _exact_norm_grad, "softmax": _exact_softmax,
            "softmax_grad": _exact_softmax}[case["op"]](case, i)
