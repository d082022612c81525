"""The operators around a model's experts and vocabulary, as they are timed and compared.

Products of a sparse matrix that is made at run time and used once: the one-hot matrix of an embedding lookup, the
k entries a token has in the matrix a router makes, the block-diagonal matrix of the experts' weights.  A case is a
dict of plain values; ``prepare`` makes what a program holds before the call, ``run`` makes one pass (the plain form
in elementary operations, or the calls of ``alsparse_b200.spblas`` where ``own`` is set), ``exact`` gives the result
in 64 bits, ``work`` counts what the operation cannot do without.
"""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "i64": 8}


def _lookup(name, tokens, vocab, width, dtype, index, scale):
    return {"name": name, "op": "lookup", "tokens": tokens, "vocab": vocab, "width": width, "dtype": dtype, "index": index, "scale": scale}


def _lookup_grad(name, tokens, vocab, width, dtype, out, index, alpha, beta):
    return {"name": name, "op": "lookup_grad", "tokens": tokens, "vocab": vocab, "width": width, "dtype": dtype, "out": out, "index": index,
            "alpha": alpha, "beta": beta}


def _route(name, tokens, experts, k, dtype, score, bias, groups, top_groups, renorm, scale, grad):
    return {"name": name, "op": "route_grad" if grad else "route", "tokens": tokens, "experts": experts, "k": k, "dtype": dtype, "score": score,
            "bias": bias, "groups": groups, "top_groups": top_groups, "renorm": renorm, "scale": scale}


def _rows(name, op, tokens, experts, k, width, dtype):
    return {"name": name, "op": op, "tokens": tokens, "experts": experts, "k": k, "width": width, "dtype": dtype}


def _mm(name, op, rows, experts, inner, outer, dtype):
    return {"name": name, "op": op, "rows": rows, "experts": experts, "inner": inner, "outer": outer, "dtype": dtype}


def listed():
    return [
        # Serving: the rows of one token each of a few running sequences; what counts is what a call costs.
        _lookup("lookup_step", 24, 65536, 2048, "bf16", "i64", 1.0),
        # A long prompt (or a batch of them) of ragged sizes, rows scaled by the root of the width as some models have it.
        _lookup("lookup_prompt_ragged", 16383, 50001, 1001, "f32", "i32", 31.639),
        # Training: the gradient of the table, all of it written; a few tokens make up most of a text.
        _lookup_grad("lookup_grad_train", 16384, 65536, 2048, "bf16", "f32", "i64", 1.0, 0.0),
        # Serving: a decoding step of a few dozen sequences, sigmoid scores with a bias for balance, groups of experts.
        _route("route_step", 32, 256, 8, "f32", "sigmoid", True, 8, 4, True, 2.5, False),
        # A long prompt through the same router ...
        _route("route_prompt", 32768, 256, 8, "f32", "sigmoid", True, 8, 4, True, 2.5, False),
        # ... and the gradient of softmax scores over an odd number of experts.
        _route("route_grad_train", 20001, 60, 4, "bf16", "softmax", False, 1, 1, False, 1.0, True),
        # The rows of a decoding step put in the order of their experts, and of a long prompt.
        _rows("dispatch_step", "dispatch", 32, 256, 8, 2048, "bf16"),
        _rows("dispatch_prompt", "dispatch", 16384, 64, 8, 2048, "bf16"),
        # The experts' answers summed up for each token: a decoding step, and training with the gradients.
        _rows("combine_step", "combine", 48, 64, 6, 2048, "bf16"),
        _rows("combine_train", "combine_train", 12001, 64, 6, 2048, "f16"),
        # The experts' products: a decoding step, where the weights of every expert that has a token are read once, and
        # a training step with both gradients.
        _mm("experts_step", "experts", 256, 64, 2048, 1408, "bf16"),
        _mm("experts_train", "experts_train", 32768, 64, 2048, 1408, "bf16"),
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "route", "route_grad", "dispatch", "combine", "combine_train", "experts", "experts_train"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op in ("lookup", "lookup_grad"):
        vocab = _between(rng, 500, 131072)
        width = _between(rng, 32, min(4096, (1 << 27) // vocab))
        width = width if rng.random() < 0.4 else max(32, width // 32 * 32)
        tokens = _between(rng, 1, min(32768, (1 << 26) // width))
        index = rng.choice(["i32", "i64"])
        if op == "lookup":
            c = _lookup("", tokens, vocab, width, dtype, index, rng.choice([1.0, round(math.sqrt(width), 3)]))
        else:
            c = _lookup_grad("", tokens, vocab, width, dtype, rng.choice([dtype, "f32"]), index, rng.choice([1.0, 0.125]), rng.choice([0.0, 0.0, 1.0, 0.5]))
    elif op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _between(rng, 4, 512 // groups)
        k = rng.randint(1, min(8, experts // groups))
        c = _route("", _between(rng, 1, 32768), experts, k, dtype, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.5, groups,
                   rng.randint(max(1, groups // 2), groups), rng.random() < 0.5, rng.choice([1.0, 2.5]), op == "route_grad")
    elif op in ("dispatch", "combine", "combine_train"):
        experts = _between(rng, 4, 256)
        k = rng.randint(1, min(8, experts))
        width = _between(rng, 32, 4096)
        width = width if rng.random() < 0.4 else max(32, width // 32 * 32)
        c = _rows("", op, _between(rng, 1, min(16384, (1 << 28) // (width * k * (2 if dtype == "f32" else 1)))), experts, k, width, dtype)
    else:
        dtype = rng.choice(["f16", "bf16"])
        experts = _between(rng, 2, 128)
        inner, outer = (_between(rng, 64, 4096) for _ in range(2))
        if rng.random() < 0.7:
            inner, outer = max(64, inner // 64 * 64), max(64, outer // 64 * 64)
        elif rng.random() < 0.7:
            inner, outer = inner // 8 * 8, outer // 8 * 8
        experts = min(experts, max(2, (1 << 27) // (inner * outer)))
        most = min(32768, int(32768 * 2048 * 1408 / (inner * outer)))
        c = _mm("", op, _between(rng, 1, max(1, min(most, 512 if op == "experts" and rng.random() < 0.4 else most))), experts, inner, outer, dtype)
    c.pop("name")
    return c


def _normal(gen, *shape, dtype=torch.float32, by=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * by).to(dtype)


def _assign(gen, tokens, experts, k):
    """The experts of each token: k different ones, some experts in far greater demand than others, a few slots empty (padding)."""
    liking = torch.randn(experts, generator=gen, device="cuda")
    noise = -torch.log(-torch.log(torch.rand(tokens, experts, generator=gen, device="cuda").clamp(1e-9, 1 - 1e-7)))
    index = torch.topk(noise + liking, k, dim=1).indices.int()
    padding = torch.rand(tokens, generator=gen, device="cuda") < 0.01
    return torch.where(padding[:, None], torch.full_like(index, -1), index)


def prepare(case, seed):
    """The inputs a program holds before the call, the outputs it writes to and the workspace it keeps for the operator."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    dtype = DTYPE[case["dtype"]]
    if op in ("lookup", "lookup_grad"):
        T, V, D = case["tokens"], case["vocab"], case["width"]
        rank = torch.exp(torch.rand(T, generator=gen, device="cuda") * math.log(V)).long().clamp(max=V) - 1
        tokens = torch.randperm(V, generator=gen, device="cuda")[rank]
        tokens[torch.rand(T, generator=gen, device="cuda") < 0.02] = -1  # padding: an empty row
        s["tokens"] = tokens.to(torch.int32 if case["index"] == "i32" else torch.int64)
        if op == "lookup":
            s["table"] = _normal(gen, V, D, dtype=dtype, by=0.05)
            s["y"] = torch.empty(T, D, dtype=dtype, device="cuda")
        else:
            s["dy"] = _normal(gen, T, D, dtype=dtype)
            # beta != 0: what the pieces of the batch before this one have left; every pass adds to it
            s["dtable"] = _normal(gen, V, D, dtype=DTYPE[case["out"]])
            s["buffer"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    elif op in ("route", "route_grad"):
        T, E, k = case["tokens"], case["experts"], case["k"]
        logits = _normal(gen, T, E, by=1.5)
        logits[torch.rand(T, generator=gen, device="cuda") < 0.01] = -math.inf  # padding: nothing to choose from
        s["logits"] = logits.to(dtype)
        s["bias"] = _normal(gen, E, by=0.1) if case["bias"] else None
        s["index"] = torch.empty(T, k, dtype=torch.int32, device="cuda")
        s["weight"] = torch.empty(T, k, device="cuda")
        if op == "route_grad":
            s["index"] = _choose(case, s["logits"], s["bias"])
            s["dweight"] = _normal(gen, T, k)
            s["dlogits"] = torch.empty_like(s["logits"])
    elif op in ("dispatch", "combine", "combine_train"):
        T, E, k, D = case["tokens"], case["experts"], case["k"], case["width"]
        s["choice"] = _assign(gen, T, E, k)
        s["offsets"], s["slot"] = _plan(s["choice"], E)
        if op == "dispatch":
            s["x"] = _normal(gen, T, D, dtype=dtype)
            s["offsets"], s["slot"] = torch.empty_like(s["offsets"]), torch.empty_like(s["slot"])
            s["xs"] = torch.zeros(T * k, D, dtype=dtype, device="cuda")
            s["buffer"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
        else:
            s["y"] = _normal(gen, T * k, D, dtype=dtype)
            s["weight"] = torch.softmax(torch.randn(T, k, generator=gen, device="cuda"), dim=1)
            s["out"] = torch.empty(T, D, dtype=dtype, device="cuda")
            if op == "combine_train":
                s["dout"] = _normal(gen, T, D, dtype=dtype)
                s["dy"] = torch.zeros_like(s["y"])
                s["dweight"] = torch.empty_like(s["weight"])
    else:
        R, E, K, N = case["rows"], case["experts"], case["inner"], case["outer"]
        liking = torch.softmax(torch.randn(E, generator=gen, device="cuda") * 0.5, dim=0)
        count = torch.bincount(torch.multinomial(liking, R, replacement=True, generator=gen), minlength=E)
        s["offsets"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), count.cumsum(0)]).int()
        s["expert"] = torch.repeat_interleave(torch.arange(E, device="cuda"), count)
        s["most"] = int(count.max())
        s["x"] = _normal(gen, R, K, dtype=dtype)
        s["w"] = _normal(gen, E, N, K, dtype=dtype, by=1 / math.sqrt(K))
        s["y"] = torch.empty(R, N, dtype=dtype, device="cuda")
        if op == "experts_train":
            s["dy"] = _normal(gen, R, N, dtype=dtype)
            s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(s["w"])
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------


def _choose(case, logits, bias):
    """The experts of each token.  What is compared is compared in 64 bits: two keys may lie next to each other."""
    x = logits.double()
    masked = x == -math.inf
    key = x
    if bias is not None:
        score = torch.sigmoid(x) if case["score"] == "sigmoid" else torch.softmax(x, dim=1)
        key = torch.where(masked, -math.inf, score + bias.double())
    if case["groups"] > 1:
        by_group = key.view(key.shape[0], case["groups"], -1)
        best = by_group.sort(dim=2, descending=True).values
        group = best[:, :, 0]
        if bias is not None and best.shape[2] > 1:
            group = group + torch.where(best[:, :, 1] == -math.inf, 0.0, best[:, :, 1])
        order = group.sort(dim=1, descending=True, stable=True).indices
        kept = torch.zeros_like(group, dtype=torch.bool).scatter_(1, order[:, : case["top_groups"]], True)
        key = torch.where(kept[:, :, None], by_group, -math.inf).view_as(key)
    best = key.sort(dim=1, descending=True, stable=True)
    k = case["k"]
    return torch.where(best.values[:, :k] == -math.inf, -1, best.indices[:, :k]).int()


def _weights(case, logits, index):
    x = logits.float()
    some = index >= 0
    at = index.clamp(min=0).long()
    if case["score"] == "sigmoid":
        s = torch.sigmoid(x).gather(1, at)
    else:
        top = x.amax(dim=1, keepdim=True)
        e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        s = e.gather(1, at) / e.sum(dim=1, keepdim=True)
    s = torch.where(some, s, 0.0)
    if case["renorm"]:
        s = torch.where(some, s / s.sum(dim=1, keepdim=True), 0.0)
    return s * case["scale"]


def _route_grad(case, logits, index, dweight):
    x = logits.float()
    some = index >= 0
    at = index.clamp(min=0).long()
    top = x.amax(dim=1, keepdim=True)
    if case["score"] == "sigmoid":
        s = torch.sigmoid(x)
    else:
        e = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        total = e.sum(dim=1, keepdim=True)
        s = e / torch.where(total == 0, 1.0, total)
    ds = torch.where(some, dweight, 0.0) * case["scale"]
    if case["renorm"]:
        chosen = torch.where(some, s.gather(1, at), 0.0)
        total = chosen.sum(dim=1, keepdim=True)
        total = torch.where(total == 0, 1.0, total)
        ds = torch.where(some, (ds - (ds * chosen / total).sum(dim=1, keepdim=True)) / total, 0.0)
    full = torch.zeros_like(s).scatter_add_(1, at, ds)
    if case["score"] == "sigmoid":
        d = full * s * (1 - s)
    else:
        d = s * (full - (full * s).sum(dim=1, keepdim=True))
    return d.to(logits.dtype)


def _plan(index, experts):
    """Where each expert's rows begin, and the row of each (token, choice) pair in the experts' order; -1 for an empty slot."""
    flat = index.reshape(-1)
    key = torch.where(flat < 0, experts, flat).long()
    order = key.sort(stable=True).indices
    count = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([count.new_zeros(1), count[:experts].cumsum(0)]).int()
    slot = torch.empty_like(flat)
    slot[order] = torch.arange(flat.numel(), dtype=torch.int32, device=flat.device)
    return offsets, torch.where(flat < 0, -1, slot).view_as(index)


def _picked(y, slot):
    """Row slot[t, j] of y as 32 bits, zeros for an empty slot."""
    return torch.where((slot < 0)[:, :, None], 0.0, y[slot.clamp(min=0).long()].float())


def _by_expert(s, x):
    """The rows of x as (experts, longest, width), zeros behind an expert's last, and where each row stands there."""
    at = torch.arange(x.shape[0], device=x.device) - s["offsets"][:-1].long()[s["expert"]]
    padded = torch.zeros(s["w"].shape[0], s["most"], x.shape[1], device=x.device)
    padded[s["expert"], at] = x.float()
    return padded, at


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op in ("lookup", "lookup_grad"):
        tokens = s["tokens"].long()
        outside = ((tokens < 0) | (tokens >= case["vocab"]))[:, None]
        tokens = tokens.clamp(0, case["vocab"] - 1)
        if op == "lookup":
            return (torch.where(outside, 0.0, s["table"][tokens].float()) * case["scale"]).to(s["y"].dtype)
        # a word of a long text can occur thousands of times: its sum in 64 bits
        total = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
        total.index_add_(0, tokens, torch.where(outside, 0.0, s["dy"].double()))
        total = total.float() * case["alpha"]
        if case["beta"]:
            total = total + case["beta"] * s["dtable"].float()
        return s["dtable"].copy_(total)
    if op == "route":
        index = _choose(case, s["logits"], s["bias"])
        return index, _weights(case, s["logits"], index)
    if op == "route_grad":
        return _route_grad(case, s["logits"], s["index"], s["dweight"])
    if op == "dispatch":
        index = s["choice"]
        offsets, slot = _plan(index, case["experts"])
        # the row behind the last takes what goes nowhere
        to = torch.where(slot < 0, slot.numel(), slot).reshape(-1).long()
        xs = torch.zeros(slot.numel() + 1, case["width"], dtype=s["x"].dtype, device="cuda")
        xs[to] = s["x"].repeat_interleave(case["k"], dim=0)
        return offsets, slot, xs[:-1]
    if op in ("combine", "combine_train"):
        rows, w = _picked(s["y"], s["slot"]), torch.where(s["slot"] < 0, 0.0, s["weight"])
        out = (rows * w[:, :, None]).sum(dim=1).to(s["out"].dtype)
        if op == "combine":
            return out
        dout = s["dout"].float()[:, None, :]
        dweight = (rows * dout).sum(dim=2)
        to = torch.where(s["slot"] < 0, s["slot"].numel(), s["slot"]).reshape(-1).long()
        dy = torch.zeros(s["slot"].numel() + 1, case["width"], dtype=s["y"].dtype, device="cuda")
        dy[to] = (w[:, :, None] * dout).to(s["y"].dtype).reshape(-1, case["width"])
        return out, dy[:-1], dweight
    x, at = _by_expert(s, s["x"])
    w = s["w"].float()
    y = torch.bmm(x, w.transpose(1, 2))[s["expert"], at].to(s["y"].dtype)
    if op == "experts":
        return y
    dy, _ = _by_expert(s, s["dy"])
    dx = torch.bmm(dy, w)[s["expert"], at].to(s["x"].dtype)
    dw = torch.bmm(dy.transpose(1, 2), x).to(s["w"].dtype)
    return y, dx, dw


# ---- the framework's calls --------------------------------------------------------------------------------------


def _ok(status):
    if status != 0:
        raise RuntimeError("status %d" % status)


def _run_own(s):
    from alsparse_b200 import capi, spblas
    case = s["case"]
    op = case["op"]
    if op == "lookup":
        _ok(spblas.embedding(s["tokens"], s["table"], case["scale"], s["y"]))
        return s["y"]
    if op == "lookup_grad":
        _ok(spblas.embedding_grad(s["tokens"], s["dy"], case["alpha"], case["beta"], s["dtable"], s["buffer"]))
        return s["dtable"]
    if op in ("route", "route_grad"):
        score = capi.SCORE_SIGMOID if case["score"] == "sigmoid" else capi.SCORE_SOFTMAX
        if op == "route":
            _ok(spblas.route(score, s["logits"], s["bias"], case["groups"], case["top_groups"], case["renorm"], case["scale"], s["index"], s["weight"]))
            return s["index"], s["weight"]
        _ok(spblas.route_grad(score, s["logits"], s["index"], case["renorm"], case["scale"], s["dweight"], s["dlogits"]))
        return s["dlogits"]
    if op == "dispatch":
        _ok(spblas.expert_plan(s["choice"], s["offsets"], s["slot"], s["buffer"]))
        _ok(spblas.expert_dispatch(s["x"], s["slot"], s["xs"]))
        return s["offsets"], s["slot"], s["xs"]
    if op in ("combine", "combine_train"):
        _ok(spblas.expert_combine(s["y"], s["slot"], s["weight"], 0.0, s["out"]))
        if op == "combine":
            return s["out"]
        _ok(spblas.expert_combine_grad(s["dout"], s["y"], s["slot"], s["weight"], s["dy"], s["dweight"]))
        return s["out"], s["dy"], s["dweight"]
    _ok(spblas.expert_mm(capi.TRANSPOSE, s["offsets"], s["x"], s["w"], s["y"]))
    if op == "experts":
        return s["y"]
    _ok(spblas.expert_mm(capi.NON_TRANSPOSE, s["offsets"], s["dy"], s["w"], s["dx"]))
    _ok(spblas.expert_mm_grad(s["offsets"], s["dy"], s["x"], 0.0, s["dw"]))
    return s["y"], s["dx"], s["dw"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what cannot be done without --------------------------------------------------------------------------------


def work(case):
    op, b = case["op"], BYTES[case["dtype"]]
    if op in ("lookup", "lookup_grad"):
        T, V, D = case["tokens"], case["vocab"], case["width"]
        unique = min(T, V)
        # tokens come log-uniformly over the ranks: the number of different ones expected
        seen = sum((1 - (1 - math.log1p(1 / r) / math.log(V)) ** T) * n for r, n in _ranks(V))
        unique = min(unique, seen)
        if op == "lookup":
            return {"bytes": unique * D * b + T * D * b + T * BYTES[case["index"]], "flops": T * D}
        out = BYTES[case["out"]]
        moved = V if case["beta"] == 0 else 2 * unique if case["beta"] == 1 else 2 * V  # beta == 1: rows that do not occur stay
        return {"bytes": T * D * b + T * BYTES[case["index"]] + moved * D * out, "flops": 2 * T * D}
    if op in ("route", "route_grad"):
        T, E, k = case["tokens"], case["experts"], case["k"]
        more = T * E * b + T * k * 4 if op == "route_grad" else T * k * 4
        return {"bytes": T * E * b + T * k * 4 + more, "flops": 10 * T * E}
    if op in ("dispatch", "combine", "combine_train"):
        T, k, D = case["tokens"], case["k"], case["width"]
        n = T * k
        if op == "dispatch":
            return {"bytes": T * D * b + n * D * b + n * 8 + case["experts"] * 4, "flops": 0}
        forward = n * D * b + T * D * b + n * 8
        return {"bytes": forward + (T * D * b + n * D * b + n * 4 if op == "combine_train" else 0), "flops": 2 * n * D * (3 if op == "combine_train" else 1)}
    R, E, K, N = case["rows"], case["experts"], case["inner"], case["outer"]
    used = E * (1 - (1 - 1 / E) ** R)
    one = R * K * b + R * N * b + used * K * N * b
    if op == "experts":
        return {"bytes": one, "flops": 2 * R * K * N}
    return {"bytes": 2 * (R * K * b + R * N * b) + used * K * N * b + E * K * N * b, "flops": 6 * R * K * N}


def _ranks(vocab):
    """Ranks by which the number of different tokens is estimated, and how many ranks each stands for."""
    edges = sorted({min(vocab, int(1.3 ** i)) for i in range(1, 80)} | {1, vocab + 1})
    return [((lo + hi) / 2, hi - lo) for lo, hi in zip(edges, edges[1:])]


# ---- 64 bits ----------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        y = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        here = s["tokens"] >= 0
        y[here] = case["scale"] * s["table"].index_select(0, s["tokens"][here].long()).double()
        return y
    if op == "lookup_grad":
        here = s["tokens"] >= 0
        order = s["tokens"][here].long().argsort(stable=True)
        rows = s["dy"][here][order].double()
        word, count = torch.unique_consecutive(s["tokens"][here].long()[order], return_counts=True)
        d = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
        pieces = torch.split(rows, count.tolist()) if len(count) else []
        for i, piece in enumerate(pieces):
            d[word[i]] = piece.sum(0)
        return case["alpha"] * d + (case["beta"] * s["dtable"].double() if case["beta"] else 0.0)
    if op in ("route", "route_grad"):
        x = s["logits"].double()
        if op == "route":
            index = _exact_choice(case, x, None if s["bias"] is None else s["bias"].double())
        else:
            index = s["index"].long()
        some = index >= 0
        chosen = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
        chosen.scatter_(1, index.clamp(min=0), some)
        score = 1 / (1 + torch.exp(-x)) if case["score"] == "sigmoid" else torch.nan_to_num(torch.exp(x - torch.logsumexp(x, 1, keepdim=True)))
        weight = score * chosen
        if case["renorm"]:
            weight = torch.nan_to_num(weight / weight.sum(1, keepdim=True))
        if op == "route":
            return index.int(), torch.where(some, weight.gather(1, index.clamp(min=0)), 0.0) * case["scale"]
        dw = torch.zeros_like(x).scatter_(1, index.clamp(min=0), torch.where(some, s["dweight"].double(), 0.0)) * case["scale"]
        # through the logarithm of the scores: d weight_i / d log score_j = weight_i (i == j) - weight_i weight_j if renormalised
        dlog = weight * dw
        if case["renorm"]:
            dlog = dlog - weight * dlog.sum(1, keepdim=True)
        return dlog * (1 - score) if case["score"] == "sigmoid" else dlog - score * dlog.sum(1, keepdim=True)
    if op == "dispatch":
        flat = s["choice"].reshape(-1)
        at = torch.nonzero(flat >= 0)[:, 0]
        order = at[torch.argsort(flat[at].long() * flat.numel() + at)]
        offsets = torch.searchsorted(flat[order].contiguous(), torch.arange(case["experts"] + 1, device="cuda", dtype=flat.dtype)).int()
        slot = torch.full_like(flat, -1)
        slot[order] = torch.arange(order.numel(), device="cuda", dtype=slot.dtype)
        xs = torch.zeros(flat.numel(), case["width"], dtype=torch.float64, device="cuda")
        xs[: order.numel()] = s["x"].double()[order // case["k"]]
        return offsets, slot.view_as(s["choice"]), xs
    if op in ("combine", "combine_train"):
        T, k, D = case["tokens"], case["k"], case["width"]
        out = torch.zeros(T, D, dtype=torch.float64, device="cuda")
        dy = torch.zeros(T * k, D, dtype=torch.float64, device="cuda") if op == "combine_train" else None
        dweight = torch.zeros(T, k, dtype=torch.float64, device="cuda")
        for j in range(k):
            t = torch.nonzero(s["slot"][:, j] >= 0)[:, 0]
            at = s["slot"][t, j].long()
            y, w = s["y"][at].double(), s["weight"][t, j].double()[:, None]
            out[t] += w * y
            if dy is not None:
                dy[at] = w * s["dout"][t].double()
                dweight[t, j] = torch.einsum("td,td->t", y, s["dout"][t].double())
        return out if dy is None else (out, dy, dweight)
    y = torch.empty(s["y"].shape, dtype=torch.float64, device="cuda")
    train = op == "experts_train"
    dx = torch.empty(s["x"].shape, dtype=torch.float64, device="cuda") if train else None
    dw = torch.zeros(s["w"].shape, dtype=torch.float64, device="cuda") if train else None
    offsets = s["offsets"].tolist()
    for e in range(case["experts"]):
        rows = slice(offsets[e], offsets[e + 1])
        x, w = s["x"][rows].double(), s["w"][e].double()
        y[rows] = torch.einsum("rk,nk->rn", x, w)
        if train:
            dy = s["dy"][rows].double()
            dx[rows] = torch.einsum("rn,nk->rk", dy, w)
            dw[e] = torch.einsum("rn,rk->nk", dy, x)
    return (y, dx, dw) if train else y


def _exact_choice(case, x, bias):
    """Top-k by a stable sort of keys, one group limit before it: written with ranks instead of masks."""
    if bias is None:
        key = x.clone()
    else:
        score = x.sigmoid() if case["score"] == "sigmoid" else torch.nan_to_num(x.softmax(1))
        key = (score + bias).masked_fill(x.isneginf(), -math.inf)
    T, G = key.shape[0], case["groups"]
    if G > 1:
        each = key.reshape(T, G, -1)
        if bias is None:
            worth = each.amax(2)
        else:
            two = torch.topk(each, min(2, each.shape[2]), dim=2).values
            worth = two[..., 0] + (two[..., 1:].masked_fill(two[..., 1:].isneginf(), 0.0)).sum(-1)
        # the rank of a group: how many stand before it
        at = torch.arange(G, device=x.device)
        ahead = (worth[:, None, :] > worth[:, :, None]) | ((worth[:, None, :] == worth[:, :, None]) & (at[None, None, :] < at[None, :, None]))
        key = each.masked_fill((ahead.sum(2) >= case["top_groups"])[:, :, None], -math.inf).reshape(T, -1)
    value, index = torch.sort(-key, dim=1, stable=True)
    return index[:, : case["k"]].masked_fill(value[:, : case["k"]].isposinf(), -1)
